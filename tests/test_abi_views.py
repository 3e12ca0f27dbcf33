"""Columns of a wider tensor (q, k and v of one product's rows) handed to an entry point together with their row stride."""

import pytest
import torch

from dromos_amd.abi import BF16, F32, NORM_RMS, Kernels, hip_library_path


@pytest.fixture(scope="module")
def lx():
    return Kernels(hip_library_path(), "cpu")  # "cpu": no stream is asked of torch


def norm(lx, y, ld_y, h, ld_h, h_out, x, ld_x):
    """No rows: the arguments are looked at, nothing is read."""
    w = torch.ones(64, dtype=torch.bfloat16)
    return lx.status("block_norm", NORM_RMS, y, BF16, ld_y, None, None, None, 0, 1.0, 1.0, h, h_out, BF16, ld_h, w, None, BF16, x, BF16, ld_x, 1e-5, 0, 64, None)


def test_columns_with_their_stride(lx):
    wide = torch.zeros(5, 256, dtype=torch.bfloat16)
    y, h, x = wide[:, :64], wide[:, 64:128], wide[:, 128:192]
    assert norm(lx, y, 256, h, 256, h, x, 256) == 0
    assert lx.status("gemv_w", torch.zeros(2, 128)[:, :64], F32, 128, None, None, F32, torch.zeros(2, 96)[:, :8], F32, 96, 2, 8, 64, 1.0, 0.0, None) == 1  # no weight


def test_views_without_their_stride_refused(lx):
    wide = torch.zeros(5, 256, dtype=torch.bfloat16)
    y, h = wide[:, :64], wide[:, 64:128]
    whole = torch.zeros(5, 64, dtype=torch.bfloat16)
    assert norm(lx, whole, 64, whole, 64, whole, whole, 64) == 0
    for args in ((y, 64, whole, 64, whole, whole, 64), (whole, 64, h, 128, h, whole, 64), (whole, 64, whole, 64, h, whole, 64),
                 (wide[:, :128:2], 256, whole, 64, whole, whole, 64), (wide.t(), 1, whole, 64, whole, whole, 64)):
        with pytest.raises(ValueError):
            norm(lx, *args)
    with pytest.raises(ValueError):  # no stride is given for a weight
        lx.status("block_norm", NORM_RMS, whole, BF16, 64, wide[:, 0], None, None, 0, 1.0, 1.0, whole, whole, BF16, 64, None, None, BF16, None, BF16, 0, 1e-5, 0, 64, None)

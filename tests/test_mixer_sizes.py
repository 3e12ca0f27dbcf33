"""What lx_linear_attention_workspace_bytes answers for, and strides that lx_linear_attention refuses; no call here reaches the device."""

import ctypes

import pytest

from test_mixer_rules import HERE, batch, decay, linear, lx  # noqa: F401
from dromos_amd import abi
from dromos_amd.abi import F32


@pytest.mark.parametrize("heads,k_heads,dk,dv", [(1, 1, 64, 64), (4, 2, 64, 64), (32, 32, 128, 128), (128, 8, 128, 64), (3, 1, 256, 256), (6, 6, 8, 512), (2, 1, 256, 64), (4096, 4096, 8, 8)])
def test_a_workspace_answers_for_fewer_rows(lx, heads, k_heads, dk, dv):  # noqa: F811
    last = 0
    for T in [0, 1, 16, 17, 64, 127, 128, 129, 255, 256, 257, 300, 511, 512, 640, 1000, 1024, 2047, 2048, 4096, 10000, 32768, 1 << 17, 1 << 20, (1 << 30) - 1]:
        size = lx.size("linear_attention_workspace_bytes", batch(), T, heads, k_heads, dk, dv)
        assert size >= last, T
        last = size


@pytest.mark.parametrize("changes", [{"ld_q": (1 << 22) + 1}, {"ld_k": (1 << 22) + 8}, {"ld_v": 1 << 23}, {"ld_out": 1 << 30}, {"gate": HERE, "ld_gate": (1 << 22) + 1}])
def test_strides_refused(lx, changes):  # noqa: F811
    assert linear(lx, T=3, **changes) == 1


def test_a_workspace_is_asked_for(lx):  # noqa: F811
    """Rows enough for parts, and no workspace: refused before anything is launched."""
    assert linear(lx, T=4096, batch=ctypes.pointer(abi.LxKv8Batch(2, HERE, HERE, None, 0, 4096, 0)), decay=decay(abi.DECAY_STEP, HERE, F32, 4)) == 1


@pytest.mark.parametrize("over", ["q", "k", "v", "gate", "x"])
def test_results_over_an_input_refused(lx, over):  # noqa: F811
    """One row of a sequence, every tensor at a place of its own but for one."""
    places = {"q": HERE, "k": HERE + 256, "v": HERE + 512, "gate": HERE + 1024, "x": HERE + 1536}
    at = dict(places)
    x = at.pop("x")
    one = ctypes.pointer(abi.LxKv8Batch(1, HERE, HERE, None, 0, 1, 0))
    assert linear(lx, T=1, batch=one, states=None, decay=decay(abi.DECAY_STEP, x, F32, 4), out=places[over], **at) == 1

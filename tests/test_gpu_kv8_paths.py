"""Calls of lx_kv8_append and lx_kv8_attention that take the seldom kernels and loops: tiles of many rows over more tokens than a
workgroup looks up at a time, sums of few and of many parts at every head size, blocks of 128 tokens of wide heads, more
sequences than a wavefront has lanes."""

import ctypes

import pytest
import torch

from kv8 import Batch, Cache, attention
from test_gpu_kv8 import appended
from test_gpu_kv8_scales import check, spread_scales

pytestmark = pytest.mark.gpu


def attended(hip, fmt, batch, heads, group, dim, page=64, block=32, window=0, how=None, seed=0):
    """Checks the call's result; returns its plan (rows of a tile, parts, tokens of a part)."""
    cache = Cache(fmt, batch.pages, heads, page, block, dim).fill(seed + 1)
    if how:
        spread_scales(cache, batch, how)
    held, on = cache.to("cuda"), batch.to("cuda")
    q = torch.randn(batch.T, heads * group * dim, generator=torch.Generator().manual_seed(seed + 2)).to(torch.bfloat16)
    out = (ctypes.c_int64 * 7)()
    c, b = held.lx(), on.lx()
    assert hip.lib.dromos_kv8_plan(ctypes.pointer(c), ctypes.pointer(b), batch.T, heads * group, window, out) == 0
    got = attention(hip, q.cuda(), held, on, heads * group, dim**-0.5, window, out_dtype=torch.float32)
    check(got, q, cache, batch, heads * group, dim**-0.5, window)
    return out[0], out[2], out[3]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("how", [None, "rising", "falling", "mixed"])
def test_tiles_over_many_tokens_in_one_part(hip, fmt, dim, how):
    """9000 tokens in one part, looked up 4096 at a time; later ones with values much larger or smaller than earlier ones."""
    batch = Batch([130] + [1] * 400, [9000] + [1 + i % 40 for i in range(400)], 64)
    per, parts, _ = attended(hip, fmt, batch, 1, 1, dim, how=how)
    assert per == 128 and parts == 1


@pytest.mark.parametrize("dim", [64, 128])
def test_tiles_over_a_wide_window_in_one_part(hip, dim):
    batch = Batch([130] + [1] * 400, [12001] + [1 + i % 40 for i in range(400)], 48)
    per, parts, _ = attended(hip, "int8", batch, 1, 1, dim, page=48, block=16, window=5000, how="mixed")
    assert per == 128 and parts == 1


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("rows,group", [(1, 4), (5, 5), (110, 1)])
@pytest.mark.parametrize("length", [1500, 5000])
def test_sums_of_parts(hip, fmt, dim, rows, group, length):
    few = length < 2048
    _, parts, _ = attended(hip, fmt, Batch([rows], [length], 64), 1, group, dim)
    assert (2 <= parts <= 8) if few else parts > 8
    attended(hip, fmt, Batch([rows], [length], 64), 1, group, dim, how="mixed")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [192, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_long_blocks_of_wide_heads(hip, fmt, dim, dtype):
    """A block of 128 tokens of 192 or 256 values is the most a workgroup holds."""
    for rows, lengths in (([128], [128]), ([300], [333]), ([100, 0, 190, 1], [700, 5, 190, 129])):
        appended(hip, fmt, rows, lengths, dim=dim, page=256, block=128, dtype=dtype)


@pytest.mark.parametrize("seqs", [64, 65, 150])
def test_append_many_sequences(hip, seqs):
    appended(hip, "fp8", [1] * seqs, [1 + 7 * i % 90 for i in range(seqs)], dim=64)
    appended(hip, "int8", [i * 5 % 4 for i in range(seqs)], [3 + 7 * i % 90 for i in range(seqs)], dim=64, spare_rows=3)
    appended(hip, "int8", [1] * seqs, [i % 60 for i in range(seqs)], dim=64, single=True, spare_rows=2)


def test_attention_many_sequences(hip):
    attended(hip, "int8", Batch([i * 5 % 4 for i in range(150)], [3 + 7 * i % 90 for i in range(150)], 64), 2, 2, 64)

"""lx_kv8_attention where the scales of a sequence's value blocks lie far apart, or are 0: what a token weighs in the softmax
does not depend on its values. Against 64 bits, with a bound of every row's own."""

import math

import pytest
import torch

from kv8 import CODES, QMAX, Batch, Cache, append, attention

pytestmark = pytest.mark.gpu


def check(got, q, cache, batch, q_heads, scale, window=0):
    """out = sum a s code / sum a, with a = 2^(score - the largest). What may be off: a term's weight by half a step of f16
    (2^-11) and, where a s is 2^-21 of the row's largest a s or less, by half a step of f16's smallest numbers: 2^-25 where the
    row's largest is 2^7 or more, so 2^-32 of that one, times the code. Scores are f32 sums of dim products (in the terms and in
    the sum of a), 2^-20 covers exponentials, scales, sums and the division. The sum of a has no other error: none of its
    own from s. The result is rounded once. A weight under 2^-126 of the largest is no f32 number: 2^-101, as in kv8.py."""
    dim, group = cache.dim, q_heads // cache.heads
    raw, scales = cache.raw(), cache.scales.double().repeat_interleave(cache.block, -1)
    half = torch.finfo(got.dtype).eps / 2
    q = q.to(torch.bfloat16).double().view(-1, q_heads, dim)
    got = got.double().cpu().view_as(q)
    table, r0 = batch.table.tolist(), 0
    for s, (n, length) in enumerate(zip(batch.rows_of, batch.lengths_of)):
        if not n or not length:
            r0 += n
            continue
        t = torch.arange(length)
        p = torch.tensor(table[s])[t // cache.page].long()
        place = t % cache.page
        behind = (length - n + torch.arange(n))[:, None] - t[None]
        hidden = behind < 0
        if window:
            hidden |= behind >= window
        for h in range(q_heads):
            kh = h // group
            k = raw[0][p, kh, place] * scales[0][p, kh, place][:, None]
            code, vs = raw[1][p, kh, place], scales[1][p, kh, place]
            qh = q[r0:r0 + n, h]
            scores = (qh @ k.T * scale).masked_fill(hidden, -math.inf)
            a = (scores - scores.amax(1, keepdim=True)).exp()
            total, x = a.sum(1, keepdim=True), a * vs
            want, spread = x @ code / total, x @ code.abs() / total
            lost = 2.0**-32 * x.amax(1, keepdim=True) * ((~hidden).double() @ code.abs()) / total
            off = 2 * abs(scale) * (qh.abs() @ k.abs().T).masked_fill(hidden, 0.0).amax(1, keepdim=True) * dim * 2.0**-24
            bound = (spread * (2.0**-11 + off + 2.0**-20) + lost) * (1 + half) + half * want.abs() + 2.0**-101
            err = (got[r0:r0 + n, h] - want).abs()
            assert not bool(err.isnan().any()), f"NaN in sequence {s}, head {h}"
            worst = (err - bound).argmax()
            assert bool((err <= bound).all()), (f"sequence {s}, row {int(worst) // dim}, head {h}: off by {err.flatten()[worst]:.3e}, "
                                                f"allowed {bound.flatten()[worst]:.3e}, at {want.flatten()[worst]:.3e}")
        r0 += n


# The scale of a sequence's block b of `of`, as a factor.
SPREADS = {
    "every third 0": lambda b, of: 0.0 if b % 3 == 1 else 1.0,
    "one of seven": lambda b, of: 1.0 if b % 7 == 3 else 0.0,
    "the first": lambda b, of: float(b == 0),
    "the last": lambda b, of: float(b == of - 1),
    "none": lambda b, of: 0.0,
    "mixed": lambda b, of: (1.0, 2.0**-10, 2.0**-20, 0.0, 2.0**-30, 2.0**-50)[b * 7 % 6],
    "rising": lambda b, of: 2.0 ** (-60 + 60 * b // of),
    "falling": lambda b, of: 2.0 ** -(60 * b // of),
    "large": lambda b, of: 2.0 ** (100 - 190 * b // of),
    "small": lambda b, of: 2.0 ** (-70 - b % 11),
}


def spread_scales(cache, batch, how):
    for s, length in enumerate(batch.lengths_of):
        of = -(-length // cache.block)
        for b in range(of):
            t = b * cache.block
            cache.scales[1, batch.table[s, t // cache.page], :, t % cache.page // cache.block] *= SPREADS[how](b, of)


def attended(hip, fmt, rows, lengths, how, heads=2, group=2, dim=128, page=64, block=32, window=0, std=1.0, seed=0, out_dtype=torch.float32):
    batch = Batch(rows, lengths, page, seed)
    cache = Cache(fmt, batch.pages, heads, page, block, dim).fill(seed + 1)
    spread_scales(cache, batch, how)
    q = (torch.randn(batch.T, heads * group * dim, generator=torch.Generator().manual_seed(seed + 2)) * std).to(torch.bfloat16)
    got = attention(hip, q.cuda(), cache.to("cuda"), batch.to("cuda"), heads * group, dim**-0.5, window, out_dtype=out_dtype)
    check(got, q, cache, batch, heads * group, dim**-0.5, window)
    return got


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("how", SPREADS)
@pytest.mark.parametrize("dim,rows,lengths", [(64, [1, 1], [700, 90]), (128, [1, 5], [3000, 64]), (192, [1, 12], [2500, 400]), (256, [1, 3], [2500, 33]),
                                              (64, [150, 70], [700, 70]), (128, [150, 100], [3000, 400])])
def test_value_scales_far_apart(hip, fmt, how, dim, rows, lengths):
    """One part and several, tiles of few rows and of many; the scores near one another."""
    attended(hip, fmt, rows, lengths, how, dim=dim)


@pytest.mark.parametrize("std", [0.0, 6.0])
@pytest.mark.parametrize("how", ["one of seven", "mixed", "rising"])
@pytest.mark.parametrize("rows", [1, 150])
def test_value_scales_and_steep_or_equal_scores(hip, rows, how, std):
    attended(hip, "int8", [rows, rows], [900, 333], how, std=std)
    attended(hip, "fp8", [rows, rows], [900, 333], how, std=std, dim=64, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("how", ["every third 0", "mixed", "rising", "falling"])
@pytest.mark.parametrize("rows", [1, 6, 150])
@pytest.mark.parametrize("window", [17, 300])
def test_value_scales_and_windows(hip, rows, how, window):
    """Blocks that other rows of a tile see and a row does not have no part in its precision."""
    attended(hip, "int8", [rows, rows], [900, rows], how, window=window, dim=64, group=1)


@pytest.mark.parametrize("rows", [1, 150])
def test_a_quarter_of_ones(hip, rows):
    """Equal scores, a block of ones and three of zeros: a quarter."""
    batch = Batch([rows], [127 + rows], 32)
    batch.table[0] = torch.arange(batch.table.shape[1])
    cache = Cache("int8", batch.table.shape[1], 1, 32, 32, 64)
    cache.codes[1, 0], cache.scales[1, 0] = 127, 1.0 / 127
    q = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda")
    out = attention(hip, q, cache.to("cuda"), batch.to("cuda"), 1, 1.0, out_dtype=torch.float32)
    want = 32.0 / torch.arange(128, 128 + rows, dtype=torch.float64)
    assert bool(((out.double().cpu() - want[:, None]).abs() <= want[:, None] * 2.0**-10).all()), out[:, 0]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("rows", [1, 130])
def test_tokens_of_zeros_appended(hip, fmt, rows):
    """Padding: tokens whose values are zeros (and some whose values are infinite or no numbers, which become zeros), as
    lx_kv8_append writes them, keep their weight."""
    dim, heads, length = 64, 2, 400
    batch = Batch([length], [length], 64)
    cache = Cache(fmt, batch.pages, heads, 64, 32, dim).to("cuda")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(length, heads * dim, generator=g).to(torch.bfloat16) for _ in range(2))
    v[64:224], v[320:352] = 0, math.nan
    append(hip, cache, batch.to("cuda"), None, k.cuda(), v.cuda(), None, 0)
    batch = Batch([rows], [length], 64)
    q = torch.randn(rows, 4 * dim, generator=g).to(torch.bfloat16)
    got = attention(hip, q.cuda(), cache, batch.to("cuda"), 4, 0.1, out_dtype=torch.float32)
    after = cache.to("cpu")
    assert bool((after.scales[1] == 0).any())
    check(got, q, after, batch, 4, 0.1)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("rows,lengths", [([1, 6], [700, 90]), ([1, 6], [3000, 64]), ([150, 70], [700, 70]), ([150, 100], [3000, 400])])
def test_values_of_the_types_range(hip, fmt, rows, lengths):
    """Values up to 2^127, whose sum over the tokens is beyond f32 though their mean is not."""
    batch = Batch(rows, lengths, 64)
    cache = Cache(fmt, batch.pages, 2, 64, 32, 64).fill(1)
    cache.scales[1] *= 2.0**125
    cache.codes[1] = cache.codes[1] & 0x7F if fmt == "fp8" else cache.codes[1].view(torch.int8).abs().view(torch.uint8)
    q = torch.randn(batch.T, 4 * 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    got = attention(hip, q.cuda(), cache.to("cuda"), batch.to("cuda"), 4, 0.125, out_dtype=torch.float32)
    check(got, q, cache, batch, 4, 0.125)

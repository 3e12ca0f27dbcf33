"""The 8-bit paged cache on the GPU, through the C ABI, against the operators restated in 64 bits (kv8.py, where the
tolerances are derived): lx_kv8_append, lx_kv8_dequantize, lx_kv8_attention."""

import ctypes
import math

import pytest
import torch

from dromos_amd.abi import BF16, DTYPE
from kv8 import CODES, QMAX, Batch, Cache, append, attention, check_appended, check_attention, check_rotated

pytestmark = pytest.mark.gpu


def frequencies(rot, theta=1e4):
    return torch.tensor([theta ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float32)


def randn(seed, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def appended(hip, fmt, rows, lengths, heads=2, group=2, dim=128, page=64, block=32, rot=None, interleaved=False, dtype=torch.bfloat16, q_dtype=torch.bfloat16, single=False, seed=0,
             pad=0, offset=0, k=None, v=None, spare_rows=0, max_length=None):
    """One call on a cache that is full of codes, checked place by place; returns the cache after it."""
    rot = dim if rot is None else rot
    batch = Batch(rows, lengths, page, seed, single=single, max_length=max_length)
    cache = Cache(fmt, batch.pages, heads, page, block, dim).fill(seed + 1)
    T, kv, width = batch.T + spare_rows, heads * dim, heads * group * dim
    wide = torch.zeros(T * (width + 2 * kv + pad) + offset, dtype=dtype, device="cuda")[offset:].view(T, width + 2 * kv + pad)
    wide.copy_(randn(seed + 2, *wide.shape, dtype=dtype, std=1.3))
    if k is not None:
        wide[:, width:width + kv] = k.cuda()
    if v is not None:
        wide[:, width + kv:width + 2 * kv] = v.cuda()
    q, keys, values = wide[:, :width], wide[:, width:width + kv], wide[:, width + kv:width + 2 * kv]
    freq = frequencies(rot).cuda() if rot else None
    held, on = cache.to("cuda"), batch.to("cuda")
    q_out = torch.full((T, width), float("nan"), dtype=q_dtype, device="cuda")
    append(hip, held, on, q, keys, values, freq, rot, interleaved, q_out, heads * group, T=T)
    after = held.to("cpu")
    check_appended(cache, after, batch, keys.cpu()[:batch.T], values.cpu()[:batch.T], freq, rot, interleaved)
    check_rotated(q_out, q.cpu(), batch, heads * group, freq, rot, interleaved)
    return after


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("rows,lengths", [([1], [1]), ([1, 1, 1], [5, 64, 33]), ([37], [37]), ([0, 70, 3, 0, 1], [9, 203, 3, 0, 300])])
def test_append(hip, fmt, dim, rows, lengths):
    appended(hip, fmt, rows, lengths, dim=dim)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (96, 32), (64, 64), (384, 128), (4096, 128)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_pages_and_blocks(hip, fmt, page, block):
    appended(hip, fmt, [1, 150, 17, 300], [131, 150, 130, 555], page=page, block=block, dim=64, heads=3)


@pytest.mark.parametrize("rot", [0, 8, 64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
def test_append_rotations_and_types(hip, rot, interleaved, dtype, q_dtype):
    appended(hip, "int8", [3, 40], [50, 41], rot=rot, interleaved=interleaved, dtype=dtype, q_dtype=q_dtype)


# Rows off the 16 bytes that are moved at once: a stride, or the first row.
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (3, 5), (8, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_strides(hip, pad, offset, dtype):
    appended(hip, "fp8", [5, 1], [70, 1], pad=pad, offset=offset, dtype=dtype, heads=1, group=5)


def test_append_one_row_a_sequence_and_rows_behind_the_last(hip):
    appended(hip, "fp8", [1, 1, 1], [1, 40, 33], single=True, spare_rows=4)
    appended(hip, "int8", [2, 0, 35], [2, 7, 35], spare_rows=70)


def test_append_rows_without_a_token(hip):
    appended(hip, "int8", [3, 40, 2], [1, 33, 0])


def test_append_far_positions(hip):
    # 2^20 tokens in pages that the table names once: only the last ones are written.
    page, length, dim = 4096, (1 << 20) + 77, 64
    batch = Batch([80], [length], page)
    batch.pages = 3
    batch.table = torch.full((1, -(-length // page)), -1, dtype=torch.int32)
    batch.table[0, (length - 80) // page:] = torch.tensor([2, 0], dtype=torch.int32)[:batch.table.shape[1] - (length - 80) // page]
    cache = Cache("fp8", 3, 1, page, 32, dim).fill(5)
    x = randn(6, 80, 3 * dim).cuda()
    freq = frequencies(dim).cuda()
    held, on = cache.to("cuda"), batch.to("cuda")
    q_out = append(hip, held, on, x[:, :dim], x[:, dim:2 * dim], x[:, 2 * dim:], freq, dim, q_out=torch.full((80, dim), float("nan"), device="cuda"), q_heads=1)
    check_appended(cache, held.to("cpu"), batch, x[:, dim:2 * dim].cpu(), x[:, 2 * dim:].cpu(), freq, dim, False)
    check_rotated(q_out, x[:, :dim].cpu(), batch, 1, freq, dim, False)


def test_append_pages_that_are_none(hip):
    batch = Batch([50, 1], [100, 70], 32)
    batch.table[0, 2] = -1
    batch.table[1, 2] = batch.pages
    cache = Cache("int8", batch.pages, 2, 32, 32, 64).fill(3)
    x = randn(4, 51, 6 * 64).cuda()
    held, freq = cache.to("cuda"), frequencies(64).cuda()
    append(hip, held, batch.to("cuda"), None, x[:, :128], x[:, 128:256], freq, 64)
    check_appended(cache, held.to("cpu"), batch, x[:, :128].cpu(), x[:, 128:256].cpu(), freq, 64, False)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_zeros_infinities_and_nans(hip, fmt):
    k, v = randn(1, 40, 256), randn(2, 40, 256, std=100.0)
    k[:, 128:] = 0  # a head of zeros: scale 0
    v[3, 7], v[4, 8], v[5, 9] = math.inf, -math.inf, math.nan
    v[33:, :128] = 2e38  # the last block alone
    after = appended(hip, fmt, [40], [40], rot=0, k=k, v=v)
    assert bool((after.scales[0, :, 1] == 0).any())


def test_append_grows_a_scale_and_leaves_one(hip):
    """Token after token into one block: where a larger one comes the earlier codes are rescaled, where none comes they stay."""
    for fmt in ("int8", "fp8"):
        batch0 = Batch([1], [1], 32)
        cache = Cache(fmt, batch0.pages, 1, 32, 32, 64).fill(9)
        for t in range(34):
            b = Batch([1], [t + 1], 32)
            b.table = torch.tensor([[1, 0]], dtype=torch.int32)
            x = randn(20 + t, 1, 128, std=1.0 + 0.3 * (t % 7)).cuda()
            held = cache.to("cuda")
            append(hip, held, b.to("cuda"), None, x[:, :64], x[:, 64:], frequencies(64).cuda(), 64)
            after = held.to("cpu")
            check_appended(cache, after, b, x[:, :64].cpu(), x[:, 64:].cpu(), frequencies(64), 64, False)
            cache = after


def test_append_queries_in_place(hip):
    batch = Batch([9, 30], [20, 30], 32)
    cache = Cache("fp8", batch.pages, 2, 32, 16, 64).fill(1)
    x = randn(3, 39, 8 * 64).cuda()
    q, freq = x[:, :256].cpu().clone(), frequencies(64).cuda()
    out = append(hip, cache.to("cuda"), batch.to("cuda"), x[:, :256], x[:, 256:384], x[:, 384:], freq, 64, q_out=x[:, :256], q_heads=4)
    check_rotated(out, q, batch, 4, freq, 64, False)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("page,block,dim", [(16, 16, 64), (96, 32, 192), (256, 128, 256)])
def test_dequantize(hip, fmt, page, block, dim):
    cache = Cache(fmt, 7, 3, page, block, dim).fill(2)
    held = cache.to("cuda")
    out = torch.full((2, 7, 3, page, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    c = held.lx()
    hip("kv8_dequantize", ctypes.pointer(c), out[0], out[1])
    want = (cache.raw().float() * cache.scales.repeat_interleave(block, -1)[..., None]).to(torch.bfloat16)
    assert torch.equal(out.cpu(), want)
    out.fill_(7.0)
    hip("kv8_dequantize", ctypes.pointer(c), None, out[1])
    assert bool((out[0] == 7.0).all()) and torch.equal(out[1].cpu(), want[1])


# ---- attention --------------------------------------------------------------------------------------------------------------


def attended(hip, fmt, rows, lengths, heads=2, group=4, dim=128, page=64, block=32, window=0, q_dtype=torch.bfloat16, out_dtype=torch.bfloat16, single=False, seed=0, std=1.0, spare_rows=0,
             scale=None, max_length=None, spoil=True):
    batch = Batch(rows, lengths, page, seed, single=single, max_length=max_length)
    cache = Cache(fmt, batch.pages, heads, page, block, dim).fill(seed + 1)
    held, on = cache.to("cuda"), batch.to("cuda")
    if spoil:  # what lies where no token is must not matter: NaN codes, scales of NaN and infinity
        live = torch.zeros(batch.pages, page, dtype=torch.bool)
        for s, length in enumerate(lengths):
            for t in range(length):
                live[batch.table[s, t // page], t % page] = True
        bits = torch.where(live[None, :, None, :, None].cuda(), held.codes, torch.tensor(0x7F, dtype=torch.uint8, device="cuda"))
        held.codes.copy_(bits)
        dead = ~live.view(batch.pages, 1, page // block, block).any(-1).expand(-1, heads, -1).cuda()
        held.scales[0][dead], held.scales[1][dead] = math.nan, math.inf
    T = batch.T + spare_rows
    q = randn(seed + 2, T, heads * group * dim, dtype=q_dtype, std=std)
    scale = dim**-0.5 if scale is None else scale
    got = attention(hip, q.cuda(), held, on, heads * group, scale, window, out_dtype=out_dtype, T=T)
    assert bool(got[batch.T:].isnan().all()), "wrote rows behind the last sequence"
    check_attention(got[:batch.T], q[:batch.T], cache, batch, heads * group, scale, window)
    return got


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 4, 5, 16, 17])
def test_attention_single_rows(hip, fmt, dim, group):
    attended(hip, fmt, [1, 1, 1, 1], [1, 100, 517, 16], dim=dim, group=group)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("rows,lengths", [([3, 1, 8], [3, 64, 200]), ([5, 0, 17], [700, 80, 17]), ([130], [130]), ([40, 33], [333, 1000])])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_several_rows(hip, fmt, rows, lengths, dim):
    attended(hip, fmt, rows, lengths, dim=dim)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_lengths(hip, length, rows):
    attended(hip, "int8", [min(rows, length), 1], [length, length], heads=1, dim=64, page=32, block=16)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (80, 16), (96, 32), (128, 128), (4096, 64)])
@pytest.mark.parametrize("rows", [1, 50])
def test_attention_pages_and_blocks(hip, page, block, rows):
    attended(hip, "fp8", [rows, 1, rows], [777, 95, 129], page=page, block=block, dim=64)


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 300, 5000])
@pytest.mark.parametrize("rows", [1, 6, 90])
def test_attention_windows(hip, window, rows):
    attended(hip, "int8", [rows, rows], [400, rows], window=window, dim=64, page=32, block=32)


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 1 << 30])
def test_attention_windows_wider_than_anything(hip, window):
    for rows in ([5, 40], [1, 200]):
        attended(hip, "fp8", rows, [3, 150], window=window, dim=64)


def test_attention_windows_of_long_sequences(hip):
    """Parts of a window that lies far behind the first token; tiles of few and of many rows."""
    for rows in (1, 5, 150):
        attended(hip, "int8", [rows, rows, 0], [9000, 700 + rows, 50], window=2100, dim=64, heads=1, group=2, spoil=False)


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_types(hip, q_dtype, out_dtype, rows):
    attended(hip, "fp8", [rows, 1], [300, 64], q_dtype=q_dtype, out_dtype=out_dtype)


def test_attention_rows_without_a_token_are_zero(hip):
    got = attended(hip, "int8", [3, 1, 40], [1, 0, 20])
    assert bool((got[:2] == 0).all()) and bool((got[3:24] == 0).all())
    got = attended(hip, "fp8", [1, 1], [0, 5], single=True)
    assert bool((got[0] == 0).all())


def test_attention_rows_behind_the_last_sequence_stay(hip):
    attended(hip, "fp8", [1, 1], [50, 3], spare_rows=5)
    attended(hip, "int8", [60, 70], [80, 70], spare_rows=64)


@pytest.mark.parametrize("rows", [1, 33])
def test_attention_pages_that_are_none(hip, rows):
    batch = Batch([rows, rows], [300, 200], 32)
    batch.table[0, 0], batch.table[0, 3], batch.table[0, 9], batch.table[1, 6] = -1, batch.pages, 2**31 - 1, -2**31
    cache = Cache("fp8", batch.pages, 2, 32, 16, 128).fill(4)
    q = randn(5, 2 * rows, 8 * 128)
    got = attention(hip, q.cuda(), cache.to("cuda"), batch.to("cuda"), 8, 0.1)
    check_attention(got, q, cache, batch, 8, 0.1)
    batch.table[:] = -1  # no page at all: zeros
    got = attention(hip, q.cuda(), cache.to("cuda"), batch.to("cuda"), 8, 0.1)
    assert bool((got == 0).all())


@pytest.mark.parametrize("std", [8.0, 60.0])
@pytest.mark.parametrize("rows", [1, 48])
def test_attention_steep_softmax(hip, std, rows):
    attended(hip, "int8", [rows, rows], [900, 333], std=std)


def test_attention_scores_far_below_and_above(hip):
    """Scores of a thousand and more in both signs: only their differences matter."""
    for scale in (3.0, -3.0):
        attended(hip, "fp8", [1, 20], [500, 100], scale=scale, dim=64)


@pytest.mark.parametrize("length,heads,group", [(131072, 1, 4), (70001, 2, 1)])
def test_attention_long(hip, length, heads, group):
    attended(hip, "fp8", [1], [length], heads=heads, group=group, dim=64, spoil=False)


def test_attention_the_same_bits_again_and_on_another_stream(hip):
    batch = Batch([1, 1, 40, 0, 5], [1000, 17, 3000, 9, 2222], 64)
    cache = Cache("int8", batch.pages, 2, 64, 32, 128).fill(1).to("cuda")
    on, q = batch.to("cuda"), randn(2, 47, 1024).cuda()
    first = attention(hip, q, cache, on, 8, 0.09)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = attention(hip, q, cache, on, 8, 0.09)
    assert torch.equal(first.view(torch.int16), again.view(torch.int16))


def test_attention_output_strides(hip):
    """out as columns of something wider, rows off 16 bytes: what lies beside them stays."""
    batch = Batch([7, 1], [90, 33], 32)
    cache = Cache("fp8", batch.pages, 1, 32, 16, 64).fill(1)
    for pad in (1, 8):
        q = randn(2, 8, 256 + pad).cuda()
        out = torch.full((8, 256 + pad), 5.0, dtype=torch.bfloat16, device="cuda")
        attention(hip, q[:, :256], cache.to("cuda"), batch.to("cuda"), 4, 0.2, out=out[:, :256])
        check_attention(out[:, :256].contiguous(), q[:, :256].cpu().contiguous(), cache, batch, 4, 0.2)
        assert bool((out[:, 256:] == 5.0).all())


def test_attention_beyond_31_bits(hip):
    """A cache of more than 2^31 codes: pages at its end."""
    heads, page, dim = 8, 4096, 128
    pages = (1 << 31) // (heads * page * dim) + 6
    batch = Batch([1, 33], [5000, 4500], page)
    cache = Cache("int8", 6, heads, page, 32, dim).fill(3)
    big = Cache("int8", 1, heads, page, 32, dim)
    big.pages = pages
    big.codes = torch.zeros(2, pages, heads, page, dim, dtype=torch.uint8, device="cuda")
    big.scales = torch.zeros(2, pages, heads, page // 32, device="cuda")
    batch.table %= 6
    big.codes[:, pages - 6:], big.scales[:, pages - 6:] = cache.codes.cuda(), cache.scales.cuda()
    q = randn(4, 34, 16 * dim)
    on = batch.to("cuda")
    on.table = on.table + (pages - 6)
    got = attention(hip, q.cuda(), big, on, 16, 0.09)
    check_attention(got, q, cache, batch, 16, 0.09)
    x = randn(5, 34, 2 * heads * dim).cuda()
    append(hip, big, on, None, x[:, :heads * dim], x[:, heads * dim:], frequencies(dim).cuda(), dim)
    after = Cache("int8", 6, heads, page, 32, dim)
    after.codes, after.scales = big.codes[:, pages - 6:].cpu(), big.scales[:, pages - 6:].cpu()
    batch.pages = 6
    check_appended(cache, after, batch, x[:, :heads * dim].cpu(), x[:, heads * dim:].cpu(), frequencies(dim), dim, False)
    assert not bool(big.codes[:, :pages - 6].any())


# ---- numbers in device memory beyond what the caller has said -------------------------------------------------------------------


@pytest.mark.parametrize("group", [4, 40])
def test_no_table_at_all(hip, group):
    """ld_table 0: no sequence has a place for a token. Nothing is stored, rows attend to nothing."""
    batch = Batch([3, 1], [3, 40], 32)
    cache = Cache("fp8", batch.pages, 1, 32, 16, 64).fill(1).to("cuda")
    before, q = cache.codes.clone(), randn(2, 4, group * 64).cuda()
    on = batch.to("cuda")
    b = on.lx()
    b.table, b.ld_table = None, 0
    c = cache.lx()
    out = torch.full_like(q, 7.0)
    at = ctypes.pointer
    hip("kv8_attention", q, BF16, group * 64, at(c), at(b), out, BF16, group * 64, 4, group, 0.1, 0, None)
    assert bool((out == 0).all())
    k = randn(3, 4, 64).cuda()
    hip("kv8_append", at(c), at(b), None, k, k, BF16, 0, 64, 64, None, BF16, 0, None, 0, 0, 4, 0)
    assert torch.equal(cache.codes, before)


def test_lengths_beyond_the_callers_bound(hip):
    """Tokens behind max_length do not count: a sequence ends there, and its rows with it."""
    for rows in ([3, 5], [40, 70]):
        more, less = Batch(rows, [200, 300], 32), Batch(rows, [150, 150], 32)
        less.table, less.pages = more.table, more.pages
        more.max_length = 150
        cache = Cache("int8", more.pages, 2, 32, 16, 64).fill(1)
        q, kv = randn(2, more.T, 8 * 64), randn(3, 2, more.T, 2 * 64)
        got = attention(hip, q.cuda(), cache.to("cuda"), more.to("cuda"), 8, 0.1)
        check_attention(got, q, cache, less, 8, 0.1)
        held = cache.to("cuda")
        append(hip, held, more.to("cuda"), None, kv[0].cuda(), kv[1].cuda(), frequencies(64).cuda(), 64)
        check_appended(cache, held.to("cpu"), less, kv[0], kv[1], frequencies(64), 64, False)


def test_more_rows_than_the_callers_bound(hip):
    """Rows of a sequence behind max_rows are left alone; those in front of them are what they are without them."""
    more, less = Batch([3, 5], [200, 300], 32), Batch([3, 4], [200, 299], 32)
    less.table, less.pages = more.table, more.pages
    more.max_rows = 4
    cache = Cache("fp8", more.pages, 2, 32, 16, 64).fill(1)
    q, kv = randn(2, 8, 8 * 64), randn(3, 2, 8, 2 * 64)
    out = torch.full((8, 8 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    attention(hip, q.cuda(), cache.to("cuda"), more.to("cuda"), 8, 0.1, out=out)
    check_attention(out[:7], q[:7], cache, less, 8, 0.1)
    assert bool((out[7] == 7.0).all())
    held = cache.to("cuda")
    append(hip, held, more.to("cuda"), None, kv[0].cuda(), kv[1].cuda(), frequencies(64).cuda(), 64)
    check_appended(cache, held.to("cpu"), less, kv[0, :7], kv[1, :7], frequencies(64), 64, False)


@pytest.mark.parametrize("rows", [2, 60])
def test_pages_that_sequences_share(hip, rows):
    """A prefix of 96 tokens that three sequences have in common: read by all, written by none, each goes on in pages of its own."""
    batch = Batch([rows, rows, 1], [96 + rows, 130 + rows, 97], 32)
    batch.table[1, :3] = batch.table[2, :3] = batch.table[0, :3]
    cache = Cache("fp8", batch.pages, 2, 32, 16, 128).fill(1)
    held, on = cache.to("cuda"), batch.to("cuda")
    T = batch.T
    q, kv = randn(2, T, 8 * 128), randn(3, 2, T, 2 * 128)
    append(hip, held, on, None, kv[0].cuda(), kv[1].cuda(), frequencies(128).cuda(), 128)
    after = held.to("cpu")
    check_appended(cache, after, batch, kv[0], kv[1], frequencies(128), 128, False)
    got = attention(hip, q.cuda(), held, on, 8, 0.09)
    check_attention(got, q, after, batch, 8, 0.09)


def test_one_page_many_times(hip):
    """A table that names the same page again and again: its tokens count as often."""
    batch = Batch([3], [400], 32)
    batch.table[0, :] = batch.table[0, 0]
    cache = Cache("int8", batch.pages, 1, 32, 32, 64).fill(1)
    q = randn(2, 3, 4 * 64)
    check_attention(attention(hip, q.cuda(), cache.to("cuda"), batch.to("cuda"), 4, 0.1), q, cache, batch, 4, 0.1)

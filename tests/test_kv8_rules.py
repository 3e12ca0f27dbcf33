"""lx_kv8_* and lx_block_norm without a device: what they refuse, and how lx_kv8_append cuts a call's rows into pieces of
blocks whatever the numbers in device memory are (dromos_kv8_pieces walks them on host memory as the kernel does)."""

import ctypes
import random

import pytest
import torch

from dromos_amd.abi import BF16, F32, NORM_LAYER, NORM_RMS, NOT_SUPPORTED, W_BF16, W_BF16X, W_FP8, W_INT8, W_NVFP4, LxKv8, LxKv8Batch, Kernels, hip_library_path

SOME = 1 << 20  # an address that is never followed


@pytest.fixture(scope="module")
def lx():
    return Kernels(hip_library_path(), "cpu")  # "cpu": no stream is asked of torch


def cache(**over):
    f = dict(type=W_INT8, k=SOME, v=SOME, k_scale=SOME, v_scale=SOME, pages=4, heads=2, page=64, block=32, dim=128) | over
    return ctypes.pointer(LxKv8(*f.values()))


def batch(**over):
    f = dict(seqs=2, rows=SOME, lengths=SOME, table=SOME, ld_table=3, max_rows=1, max_length=192) | over
    return ctypes.pointer(LxKv8Batch(*f.values()))


BAD_CACHES = [(dict(type=W_BF16), NOT_SUPPORTED), (dict(type=W_NVFP4), NOT_SUPPORTED), (dict(type=W_BF16X), NOT_SUPPORTED), (dict(type=9), 1), (dict(k=None), 1), (dict(v=None), 1),
              (dict(k_scale=None), 1), (dict(v_scale=None), 1), (dict(k=SOME + 8), 1), (dict(v=SOME + 4), 1), (dict(pages=0), 1), (dict(heads=0), 1), (dict(heads=1025), 1),
              (dict(page=48), 1), (dict(page=16), 1), (dict(page=0), 1), (dict(page=4096 + 32), 1), (dict(block=8), 1), (dict(block=48), 1), (dict(block=256, page=256), 1),
              (dict(dim=80), 1), (dict(dim=0), 1), (dict(dim=512), 1), (dict(pages=1 << 30, page=4096), 1)]
BAD_BATCHES = [dict(lengths=None), dict(table=None), dict(seqs=-1), dict(ld_table=-1), dict(max_rows=-1), dict(max_length=-1)]


GIVEN = object()


def append(lx, c=GIVEN, b=GIVEN, q=SOME, k=SOME, v=SOME, dtype=BF16, ld_q=1024, ld_k=256, ld_v=256, q_out=SOME, out_dtype=BF16, ld_out=1024, freq=SOME, rot=128,
           T=2, q_heads=8):
    return lx.status("kv8_append", cache() if c is GIVEN else c, batch() if b is GIVEN else b, q, k, v, dtype, ld_q, ld_k, ld_v, q_out, out_dtype, ld_out, freq, rot, 0, T, q_heads, None)


def attention(lx, c=GIVEN, b=GIVEN, q=SOME, dtype=BF16, ld_q=1024, out=SOME, out_dtype=BF16, ld_out=1024, T=2, q_heads=8, window=0, workspace=SOME):
    return lx.status("kv8_attention", q, dtype, ld_q, cache() if c is GIVEN else c, batch() if b is GIVEN else b, out, out_dtype, ld_out, T, q_heads, 0.1, window, workspace, None)


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_caches_refused(lx, over, status):
    assert append(lx, c=cache(**over)) == status
    assert attention(lx, c=cache(**over)) == status
    assert lx.status("kv8_dequantize", cache(**over), SOME, SOME, None) == status


@pytest.mark.parametrize("over", BAD_BATCHES)
def test_batches_refused(lx, over):
    assert append(lx, b=batch(**over)) == 1
    assert attention(lx, b=batch(**over)) == 1


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(dtype=2), dict(out_dtype=7), dict(ld_q=1023), dict(ld_k=255), dict(ld_v=255),
                                  dict(ld_out=1023), dict(freq=None), dict(rot=136), dict(rot=12), dict(rot=-8), dict(T=-1), dict(q_heads=7), dict(q_heads=0)])
def test_append_arguments_refused(lx, over):
    assert append(lx, **over) == 1


@pytest.mark.parametrize("over", [dict(q=None), dict(out=None), dict(dtype=2), dict(out_dtype=-1), dict(ld_q=1023), dict(ld_out=1023), dict(T=-1), dict(q_heads=7), dict(q_heads=0), dict(window=-1)])
def test_attention_arguments_refused(lx, over):
    assert attention(lx, **over) == 1


def test_null_structs_refused(lx):
    assert append(lx, c=None) == 1 and attention(lx, c=None) == 1 and lx.status("kv8_dequantize", None, SOME, SOME, None) == 1
    assert append(lx, b=None) == 1 and attention(lx, b=None) == 1
    assert lx.size("kv8_attention_workspace_bytes", cache(), None, 2, 8) == 0
    assert lx.size("kv8_attention_workspace_bytes", cache(dim=80), batch(), 2, 8) == 0


def test_dequantize_arguments(lx):
    assert lx.status("kv8_dequantize", cache(), SOME + 2, None, None) == 1
    assert lx.status("kv8_dequantize", cache(), None, None, None) == 0


def test_nothing_to_do(lx):
    assert append(lx, T=0) == 0 and append(lx, b=batch(seqs=0)) == 0
    assert attention(lx, T=0) == 0 and attention(lx, b=batch(seqs=0)) == 0


def norm(lx, kind=NORM_RMS, y=SOME, y_dtype=BF16, ld_y=64, post=SOME, gate=SOME, ld_gate=64, beta=1.0, h=SOME, h_out=SOME, h_dtype=BF16, ld_h=64, weight=SOME,
         w_dtype=BF16, x=SOME, x_dtype=BF16, ld_x=64, T=2, H=64):
    return lx.status("block_norm", kind, y, y_dtype, ld_y, post, None, gate, ld_gate, 1.0, beta, h, h_out, h_dtype, ld_h, weight, None, w_dtype, x, x_dtype, ld_x, 1e-5,
                     T, H, None)


@pytest.mark.parametrize("over", [dict(kind=2), dict(kind=-1), dict(y_dtype=2), dict(h_dtype=2), dict(w_dtype=2), dict(x_dtype=2), dict(ld_y=63), dict(ld_h=63), dict(ld_x=63), dict(ld_gate=63),
                                  dict(h=None), dict(h_out=None), dict(x=None), dict(y=None, h=None), dict(y=None, weight=None), dict(T=-1), dict(H=-1), dict(H=32769, ld_y=40000, ld_h=40000, ld_x=40000, ld_gate=0)])
def test_norm_arguments_refused(lx, over):
    assert norm(lx, **over) == 1


def test_norm_nothing_to_do(lx):
    assert norm(lx, T=0) == 0 and norm(lx, kind=NORM_LAYER, H=0) == 0


def pieces(lx, page, block, pages, T, seqs, rows, lengths, table, max_length):
    c = cache(page=page, block=block, pages=pages)
    b = ctypes.pointer(LxKv8Batch(seqs, None if rows is None else rows.data_ptr(), lengths.data_ptr(), table.data_ptr(), table.shape[1], T, max_length))
    out = (ctypes.c_int * (5 * (T + 1)))()
    n = lx.lib.dromos_kv8_pieces(c, b, T, out, T + 1)
    return [tuple(out[5 * i:5 * i + 5]) for i in range(n)]


@pytest.mark.parametrize("seed", range(60))
def test_every_row_goes_with_one_piece(lx, seed):
    """Whole batches, rows without a token and rows behind the last sequence among them: the pieces cover every row that has
    a place in the cache once, and each lies in one block."""
    rng = random.Random(seed)
    block = rng.choice([16, 32, 64, 128])
    page = block * rng.choice([1, 2, 3])
    n = rng.randint(1, 9)
    rows = [rng.choice([0, 1, 1, 2, rng.randint(0, 5), rng.randint(0, 3 * block)]) for _ in range(n)]
    lengths = [rng.choice([0, 1, r, r + rng.randint(0, 400), max(0, r - 2)]) for r in rows]
    width = max(1, max(-(-length // page) for length in lengths))
    table = torch.tensor([[rng.choice([rng.randrange(50), rng.randrange(50), -1, 50, 2**31 - 1]) for _ in range(width)] for _ in rows], dtype=torch.int32)
    first = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    T = int(first[-1]) + rng.choice([0, 3, 70])
    got = pieces(lx, page, block, 50, T, n, first, torch.tensor(lengths, dtype=torch.int32), table, 10**6)
    seen = []
    for s, position, p, tokens, row in got:
        assert tokens > 0 and position // block == (position + tokens - 1) // block and position + tokens <= lengths[s]
        named = int(table[s, position // page])
        assert p == (named if 0 <= named < 50 else -1)
        assert row - int(first[s]) + lengths[s] - rows[s] == position
        seen += range(row, row + tokens)
    want = [int(first[s]) + i for s in range(n) for i in range(rows[s]) if lengths[s] - rows[s] + i >= 0]
    assert sorted(seen) == want


@pytest.mark.parametrize("seed", range(60))
def test_nonsense_stays_inside(lx, seed):
    """Rows out of order, lengths and pages that are no such thing: no piece leaves the rows, the table or the cache."""
    rng = random.Random(1000 + seed)
    block = rng.choice([16, 64])
    page, n, T, width = block * rng.choice([1, 3]), rng.randint(1, 6), rng.randint(1, 90), rng.randint(1, 4)
    wild = lambda: rng.choice([0, 1, -1, rng.randint(-200, 400), 2**31 - 1, -2**31])
    rows = torch.tensor([wild() for _ in range(n + 1)], dtype=torch.int32) if rng.random() < 0.8 else None
    lengths = torch.tensor([wild() for _ in range(n)], dtype=torch.int32)
    table = torch.tensor([[wild() for _ in range(width)] for _ in range(n)], dtype=torch.int32)
    limit = rng.choice([0, 5, 100, 2**31 - 1])
    for s, position, p, tokens, row in pieces(lx, page, block, 7, T, n, rows, lengths, table, limit):
        assert 0 <= s < n and tokens > 0 and 0 <= row and row + tokens <= T
        assert 0 <= position and position + tokens <= min(width * page, limit) and -1 <= p < 7
        assert position // block == (position + tokens - 1) // block


@pytest.mark.parametrize("seed", range(300))
def test_parts_cover_what_rows_see_and_fit_the_workspace(lx, seed):
    """How a call is cut up, on random sizes: every token that a row may see lies in one of the parts, whatever the window, and
    the partial sums fit the workspace, whose size does not ask for the window."""
    rng = random.Random(seed)
    log = lambda a, b: int(round(2 ** rng.uniform(a, b)))
    dim, block = rng.choice([64, 128, 192, 256]), rng.choice([16, 32, 64])
    page, heads, group = block * rng.choice([1, 2, 4]), log(0, 4), rng.choice([1, 2, 4, 5, 8, 16, 17])
    seqs, most, longest = log(0, 8), rng.choice([1, 1, log(0, 4), log(0, 13)]), log(0, 18)
    T = min(1 << 29, rng.randint(most, most * seqs))
    window = rng.choice([0, 0, log(0, 14), 2**31 - 1])
    ld = rng.choice([-(-longest // page), -(-longest // page) + 3, max(0, longest // page - 1)])
    c = cache(dim=dim, block=block, page=page, heads=heads)
    b = batch(seqs=seqs, ld_table=ld, max_rows=most, max_length=longest)
    out = (ctypes.c_int64 * 7)()
    assert lx.lib.dromos_kv8_plan(c, b, T, heads * group, window, out) == 0
    per, tiles, parts, chunk, workgroups, partial, workspace = out
    rows, length = min(most, T) * group, min(longest, ld * page)
    assert per in (16, 32, 128) and tiles * per >= rows and (tiles - 1) * per < rows
    seen = length if window == 0 else min(length, window + -(-per // group) + 16)  # the tile's rows and the run it begins in
    assert parts * chunk >= seen and chunk % 256 == 0 and (per == 128 or chunk <= 4096)
    assert workgroups == seqs * tiles * heads * parts and partial <= workspace
    assert parts == 1 or workspace > 0


def test_sequences_of_more_than_2_30_tokens_refused(lx):
    """A table may name one page many times, and so have room for more tokens than positions can count."""
    plan = lambda b: lx.lib.dromos_kv8_plan(cache(), b, 2, 8, 0, (ctypes.c_int64 * 7)())
    wide = (1 << 24) + 1  # pages of 64
    for call in (append, attention):
        assert call(lx, b=batch(ld_table=wide, max_length=2**31 - 1)) == 1
        assert call(lx, b=batch(ld_table=wide, max_length=(1 << 30) + 1)) == 1
    assert plan(batch(ld_table=wide, max_length=(1 << 30) + 1)) == 1
    assert plan(batch(ld_table=wide, max_length=1 << 30)) == 0 and plan(batch(ld_table=3, max_length=2**31 - 1)) == 0


@pytest.mark.parametrize("seqs,heads,group,T,rows,length", [(1 << 30, 1024, 1, 1 << 29, 1, 64), (1, 1, 65536, (1 << 30) - 1, 1 << 30, 64), (1 << 30, 1, 65536, (1 << 30) - 1, 1 << 30, 64),
                                                          (1 << 14, 1024, 1, 1 << 14, 1, 64), (1 << 22, 2, 8, 1 << 22, 1, 65536)])
def test_calls_of_more_workgroups_than_a_launch_refused(lx, seqs, heads, group, T, rows, length):
    """Not started, and never taken for a smaller one: neither a number of workgroups nor its bytes wraps around."""
    c, b = cache(heads=heads), batch(seqs=seqs, max_rows=rows, max_length=length, ld_table=1024)
    width = heads * group * 128
    assert lx.lib.dromos_kv8_plan(c, b, T, heads * group, 0, (ctypes.c_int64 * 7)()) == 1
    # The last would have its 16 parts of 4096 tokens (a window might make it fit); of the others no part fits.
    most = seqs * heads * 16 * 16 * (128 + 2) * 4 if length > 64 else 0
    assert lx.size("kv8_attention_workspace_bytes", c, b, T, heads * group) == most
    assert attention(lx, c=c, b=b, T=T, q_heads=heads * group, ld_q=width, ld_out=width) == 1

"""lx_kv8_attention_workspace_bytes on the CPU: a buffer for the largest call of a program holds what any smaller one needs, as
the library's other workspaces do. Fewer rows or sequences come in more parts, so their sums can want more than the largest's."""

import ctypes
import random

import pytest

from dromos_amd.abi import W_INT8, Kernels, LxKv8, LxKv8Batch, hip_library_path

SOME = 1 << 20  # an address that is never followed


@pytest.fixture(scope="module")
def lx():
    return Kernels(hip_library_path(), "cpu")  # "cpu": no stream is asked of torch


def cache(heads, dim, page=64, block=32):
    return ctypes.pointer(LxKv8(W_INT8, SOME, SOME, SOME, SOME, 1000, heads, page, block, dim))


def batch(seqs, max_rows, length, ld):
    return ctypes.pointer(LxKv8Batch(seqs, SOME, SOME, SOME, ld, max_rows, length))


def held(lx, c, b, T, q_heads):
    return lx.size("kv8_attention_workspace_bytes", c, b, T, q_heads)


def needed(lx, c, b, T, q_heads, window):
    """Bytes of partial sums that the call writes (0: refused, or none)."""
    out = (ctypes.c_int64 * 7)()
    return 0 if lx.lib.dromos_kv8_plan(c, b, T, q_heads, window, out) else out[5]


def test_a_token_after_a_prompt(lx):
    """One sequence of up to 131072 tokens, 8 heads of 128: a prompt's 4096 rows come in one part, a single row in 64."""
    c, ld = cache(8, 128), 131072 // 64
    prompt = held(lx, c, batch(1, 4096, 131072, ld), 4096, 32)
    assert needed(lx, c, batch(1, 4096, 131072, ld), 4096, 32, 0) == 0
    one = needed(lx, c, batch(1, 1, 131072, ld), 1, 32, 0)
    assert one == 8 * 64 * 16 * (128 + 2) * 4 and prompt >= one


def test_one_sequence_after_many(lx):
    c = cache(8, 128)
    one = needed(lx, c, batch(1, 1, 4096, 64), 1, 32, 0)
    assert one > 0 and held(lx, c, batch(256, 1, 4096, 64), 256, 32) >= one


@pytest.mark.parametrize("seed", range(400))
def test_the_largest_call_covers_smaller_ones(lx, seed):
    rng = random.Random(seed)
    log = lambda a, b: int(round(2 ** rng.uniform(a, b)))
    below = lambda n: rng.choice([1, n, rng.randint(1, n), min(n, log(0, max(0.1, n.bit_length() - 1)))])
    dim, heads, group = rng.choice([64, 128, 192, 256]), rng.choice([1, 2, 3, 8, 16, 64]), rng.choice([1, 2, 4, 5, 8, 16, 17, 128])
    seqs, most, length = log(0, 9), rng.choice([1, log(0, 4), log(0, 13)]), log(0, 18)
    T, ld = rng.randint(most, most * seqs), -(-length // 64) + rng.choice([0, 0, 3])
    c = cache(heads, dim)
    space = held(lx, c, batch(seqs, most, length, ld), T, heads * group)
    for _ in range(60):
        s, m, n, t = below(seqs), below(most), below(length), below(T)
        window = rng.choice([0, 0, log(0, 14)])
        assert needed(lx, c, batch(s, m, n, ld), t, heads * group, window) <= space, (s, m, n, t, window)
        assert held(lx, c, batch(s, m, n, ld), t, heads * group) <= space


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 5), (8, 4)])
def test_every_number_of_rows_and_sequences(lx, dim, heads, group):
    c, seqs, most, length = cache(heads, dim), 40, 300, 20000
    space = held(lx, c, batch(seqs, most, length, 400), seqs * most, heads * group)
    for s in range(1, seqs + 1, 3):
        for m in range(1, most + 1, 7):
            for t in (1, m, m + s, s * m):
                assert needed(lx, c, batch(s, m, length, 400), t, heads * group, 0) <= space, (s, m, t)


def test_the_answer_comes_quickly(lx):
    """A query of the largest sizes ends: it looks at cuts that differ, not at every number of rows."""
    for dim in (64, 256):
        c = cache(1, dim)
        for seqs in (1, 1 << 20):
            held(lx, c, batch(seqs, (1 << 30) - 1, 1 << 30, 1 << 24), (1 << 30) - 1, 1)

"""lx_rotate against the same in 64 bits.

Tolerance: cosine and sine are off by at most 2^-23 (the reduced angle's rounding, 2^-25, and the series'), times the amplitude a rounding
more; two products and their sum add three roundings. Together less than 2^-21 of |a| + |b| times the amplitude; then the result's own rounding."""

import pytest
import torch

from dromos_amd.abi import DTYPE
from mixer import HALF, UNTOUCHED, Rows, pointer, rotated

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def frequencies(rot, base=1e4):
    return torch.tensor([base ** (-2 * i / rot) for i in range(rot // 2)] or [0.0], dtype=F)


def check(got, x, positions, freq, amplitude, rot, interleaved, heads, dim, known=None):
    want, size = rotated(x, positions, freq[:rot // 2], amplitude, rot, interleaved, heads, dim)
    got = got.double().cpu()
    if known is None:
        known = torch.ones(x.shape[0], dtype=torch.bool)
    assert bool((got[~known] == UNTOUCHED).all()), "rows of nobody were written"
    error, share = (got - want).abs(), 2.0**-21 * size
    half = 0.0 if got.dtype == F else 1.0
    bound = share + HALF[check.out] * 1.01 * (want.abs() + share) * half
    assert bool((error <= bound + 1e-30)[known].all()), f"worst {(error / (bound + 1e-30))[known].max().item():.3g} of its bound"
    kept = torch.ones(heads, dim, dtype=torch.bool)
    kept[:, :rot] = False
    same = x.double().to(check.out).double()
    assert torch.equal(got[known][:, kept.flatten()], same[known][:, kept.flatten()]), "values behind the rotation are not as they were"


def turn(hip, x, rows, positions, freq, amplitude, rot, interleaved, heads, dim, out, ld=None, ld_out=None):
    wide = torch.zeros(x.shape[0], ld or x.shape[1], dtype=x.dtype, device="cuda")
    wide[:, :x.shape[1]] = x.cuda()
    y = torch.full((x.shape[0], ld_out or x.shape[1]), UNTOUCHED, dtype=out, device="cuda")
    batch = None if rows is None else rows.lx()
    hip("rotate", wide[:, :x.shape[1]], DTYPE[x.dtype], wide.shape[1], y[:, :x.shape[1]], DTYPE[out], y.shape[1], pointer(batch), positions, freq.cuda(),
        amplitude, rot, interleaved, x.shape[0], heads, dim)
    assert bool((y[:, x.shape[1]:] == UNTOUCHED).all())
    check.out = out
    return y[:, :x.shape[1]]


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("heads,dim,rot", [(1, 64, 64), (5, 128, 128), (40, 128, 64), (3, 256, 256), (7, 72, 40), (2, 80, 8), (3, 50, 26), (2, 33, 32), (1, 1, 0), (4, 128, 0),
                                           (1, 1024, 1024), (130, 16, 16), (9, 24, 24), (6, 64, 2)])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (F, BF), (F, F), (BF, F)])
def test_layouts_and_types(hip, dtype, out, heads, dim, rot, interleaved):
    T = 11
    x = torch.randn(T, heads * dim, generator=torch.Generator().manual_seed(dim)).to(dtype)
    positions = torch.tensor([0, 1, 2, 5, 77, 4095, 131071, 1 << 20, -3, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32)
    freq = frequencies(rot)
    got = turn(hip, x, None, positions.cuda(), freq, 1.25, rot, interleaved, heads, dim, out)
    check(got, x, positions, freq, 1.25, rot, interleaved, heads, dim)


@pytest.mark.parametrize("counts,lengths,T", [([1], [1], 1), ([3, 0, 1, 70, 0, 0, 5], [9, 4, 1, 70, 0, 3, 100000], 81), ([4, 6], [2, 0], 12), ([0, 0], [5, 0], 3),
                                              ([2] * 200, list(range(2, 202)), 400), ([1] * 5000, [7 * i % 9000 + 1 for i in range(5000)], 5000)])
def test_positions_of_a_batch(hip, counts, lengths, T):
    heads, dim, rot = 3, 64, 64
    rows = Rows(counts, lengths, T=T, device="cuda")
    x = torch.randn(T, heads * dim, generator=torch.Generator().manual_seed(T)).to(BF)
    positions, known = torch.zeros(T, dtype=torch.int32), torch.zeros(T, dtype=torch.bool)
    for _, begin, end, position, _, _ in rows.spans():
        positions[begin:end] = torch.arange(position, position + end - begin)
        known[begin:end] = True
    freq = frequencies(rot, 1e6)
    got = turn(hip, x, rows, None, freq, 1.0, rot, 0, heads, dim, BF)
    check(got, x, positions, freq, 1.0, rot, 0, heads, dim, known)


def test_bounds_of_a_batch(hip):
    # One row a sequence without a rows tensor; sequences behind the last row; rows beyond max_rows; numbers in device memory that are none.
    heads, dim, freq = 2, 32, frequencies(32)
    x = torch.randn(9, heads * dim, generator=torch.Generator().manual_seed(3)).to(BF)
    lengths = [5, 0, 1, 9, 3000]
    for seqs, T in ((5, 9), (5, 3)):
        got = turn(hip, x[:T], Rows(None, lengths, seqs=seqs, T=T, device="cuda"), None, freq, 1.0, 32, 1, heads, dim, BF)
        known = torch.tensor([n > 0 for n in lengths] + [False] * 4)[:T]
        check(got, x[:T], torch.tensor([n - 1 for n in lengths] + [0] * 4)[:T], freq, 1.0, 32, 1, heads, dim, known)
    got = turn(hip, x, Rows([4, 5], [4, 50], max_rows=3, device="cuda"), None, freq, 1.0, 32, 1, heads, dim, BF)
    known = torch.tensor([1, 1, 1, 0, 1, 1, 1, 0, 0]).bool()
    check(got, x, torch.tensor([0, 1, 2, 3, 45, 46, 47, 48, 49]), freq, 1.0, 32, 1, heads, dim, known)
    rows = Rows([4, 5], [1 << 31 - 1, -7], device="cuda")
    rows.rows_t.copy_(torch.tensor([-5, 100000, -(1 << 31)]))
    got = turn(hip, x, rows, None, freq, 1.0, 32, 1, heads, dim, BF)
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("offset", [0, 8, 4, 1])
def test_strides_alignment_and_in_place(hip, offset):
    heads, dim, rot, T = 5, 64, 32, 19
    whole = torch.randn(T, heads * dim + 24, generator=torch.Generator().manual_seed(offset)).to(BF).cuda()
    x = whole[:, offset:offset + heads * dim]
    before, freq = whole.cpu(), frequencies(rot)
    positions = torch.arange(100, 100 + T, dtype=torch.int32)
    hip("rotate", x, DTYPE[BF], whole.shape[1], x, DTYPE[BF], whole.shape[1], None, positions.cuda(), freq.cuda(), 0.5, rot, 0, T, heads, dim)
    check.out = BF
    check(x, before[:, offset:offset + heads * dim], positions, freq, 0.5, rot, 0, heads, dim)
    rest = torch.ones(whole.shape[1], dtype=torch.bool)
    rest[offset:offset + heads * dim] = False
    assert torch.equal(whole.cpu()[:, rest], before[:, rest])
    wide = turn(hip, before[:, :heads * dim], None, positions.cuda(), freq, 0.5, rot, 0, heads, dim, F, heads * dim + 3 * offset, heads * dim + 5 * offset)
    check(wide, before[:, :heads * dim], positions, freq, 0.5, rot, 0, heads, dim)


def test_equal_to_the_caches_rotation(hip):
    # lx_kv8_append's queries, turned by the same frequencies, bit for bit.
    from dromos_amd.abi import BF16, FORMATS, LxKv8, LxKv8Batch

    heads, dim, T = 4, 128, 37
    g = torch.Generator().manual_seed(9)
    x, freq = torch.randn(T, heads * dim, generator=g).to(BF).cuda(), frequencies(dim).cuda()
    rows, lengths, table = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, T], [T + 11], [0]))
    codes, scales = torch.zeros(2, 1, 1, 64, dim, dtype=torch.uint8, device="cuda"), torch.zeros(2, 1, 1, 4, device="cuda")
    cache = LxKv8(FORMATS["fp8"], codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), 1, 1, 64, 16, dim)
    batch = LxKv8Batch(1, rows.data_ptr(), lengths.data_ptr(), table.data_ptr(), 1, T, 64)
    k = torch.randn(T, dim, generator=g).to(BF).cuda()
    q, y = torch.empty_like(x), torch.empty_like(x)
    hip("kv8_append", pointer(cache), pointer(batch), x, k, k, BF16, heads * dim, dim, dim, q, BF16, heads * dim, freq, dim, 0, T, heads)
    hip("rotate", x, BF16, heads * dim, y, BF16, heads * dim, pointer(batch), None, freq, 1.0, dim, 0, T, heads, dim)
    assert torch.equal(q.view(torch.int16), y.view(torch.int16))

"""lx_causal_conv against the same in 64 bits.

Tolerance: W products and sums in f32, 2^-24 of the magnitudes each, W + 1 of them; silu's slope is at most 1.1, its own evaluation 2^-21 of its
value (exponential, sum, division); then the result's rounding. States are copies, bit for bit."""

import pytest
import torch

from dromos_amd.abi import ACT_NONE, ACT_SILU, DTYPE, LxStates
from mixer import HALF, UNTOUCHED, Rows, convolved, pointer

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def run(hip, x, weight, bias, silu, rows, state, out, keep="same", offset=0):
    """(y, states afterwards); ``offset``: x and y are columns of wider tensors from there on."""
    T, C = x.shape
    device = Rows(None if rows.plain else rows.counts, rows.lengths, rows.slots, rows.T, rows.max_rows, rows.seqs, "cuda")
    wide = torch.zeros(T, C + 2 * offset, dtype=x.dtype, device="cuda")
    wide[:, offset:offset + C] = x.cuda()
    y = torch.full((T, C + 3 * offset), UNTOUCHED, dtype=out, device="cuda")
    given = None if state is None else state.cuda()
    shape = (len(rows.counts) + 1, weight.shape[1] - 1, C) if state is None else state.shape
    kept = {"same": given, "other": torch.full(shape, UNTOUCHED, dtype=x.dtype, device="cuda"), "none": None}[keep]
    states = device.states(given, kept, shape[0])
    w, b = weight.cuda(), None if bias is None else bias.cuda()
    hip("causal_conv", wide[:, offset:offset + C], DTYPE[x.dtype], wide.shape[1], w, b, DTYPE[weight.dtype], weight.shape[1], ACT_SILU if silu else ACT_NONE,
        pointer(device.lx()), pointer(states), y[:, offset:offset + C], DTYPE[out], y.shape[1], T, C)
    mask = torch.ones(y.shape[1], dtype=torch.bool)
    mask[offset:offset + C] = False
    assert bool((y.cpu()[:, mask] == UNTOUCHED).all())
    return y[:, offset:offset + C], kept


def check(y, kept, x, weight, bias, silu, rows, state, before):
    want, size, states = convolved(x, weight, bias, silu, rows, state, before.shape[0])
    got, nobody = y.double().cpu(), want.isnan()
    assert bool((got[nobody] == UNTOUCHED).all()), "rows of nobody were written"
    share = 1.1 * (weight.shape[1] + 1) * 2.0**-24 * size + (2.0**-21 * want.abs() if silu else 0)
    bound = share + HALF[y.dtype] * 1.01 * (want.abs() + share) + 1e-30
    assert bool(((got - want).abs() <= bound)[~nobody].all()), f"worst {((got - want).abs() / bound)[~nobody].max().item():.3g} of its bound"
    if kept is None:
        return
    for slot in range(before.shape[0]):
        assert torch.equal(kept[slot].double().cpu(), states.get(slot, before[slot].double())), f"state {slot}"


def inputs(T, C, width, dtype, w_dtype, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, C, generator=g).to(dtype), (torch.randn(C, width, generator=g) * 0.5).to(w_dtype),
            torch.randn(C, generator=g).to(w_dtype) if bias else None, g)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("C", [8, 2050, 2048, 1, 37, 4104])
@pytest.mark.parametrize("width", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("dtype,out,w_dtype", [(BF, BF, BF), (F, F, F), (F, BF, BF), (BF, F, F)])
def test_sizes_and_types(hip, dtype, out, w_dtype, width, C, silu):
    rows = Rows([1, 0, 40, 16, 3, 17, 2], [5, 3, 40, 1000, 3, 17, 3], slots=[3, 1, 0, 7, 2, 5, 4])
    x, weight, bias, g = inputs(rows.T, C, width, dtype, w_dtype, silu, C)
    state = torch.randn(9, width - 1, C, generator=g).to(dtype)
    y, kept = run(hip, x, weight, bias, silu, rows, state, out)
    check(y, kept, x, weight, bias, silu, rows, state, state)


@pytest.mark.parametrize("C,offset", [(64, 0), (64, 4), (24, 8), (21, 1)])
@pytest.mark.parametrize("counts,lengths,slots,T,max_rows", [
    ([1] * 70, None, None, 70, None), ([5, 1, 33], None, [2, 0, 1], 45, None), ([40, 6], [40, 2], [0, 1], 50, None), ([4, 4], [0, 9], None, 8, None),
    ([40, 50], [100, 50], None, 90, 19), ([3] * 300, [i % 5 for i in range(300)], None, 900, None), ([2, 2, 2], [9, 9, 9], [1, -1, 99], 6, None),
    ([700], [700], [1], 700, None), ([16, 32, 48, 0, 64], [99] * 5, None, 160, None)])
def test_batches(hip, counts, lengths, slots, T, max_rows, C, offset):
    rows = Rows(counts, lengths, slots, T, max_rows)
    x, weight, bias, g = inputs(T, C, 4, BF, BF, True, T)
    count = max([1] + [s + 1 for s in slots or range(len(counts)) if s < 90]) + 1
    state = torch.randn(count, 3, C, generator=g).to(BF)
    y, kept = run(hip, x, weight, bias, True, rows, state, BF, offset=offset)
    check(y, kept, x, weight, bias, True, rows, state, state)
    y, kept = run(hip, x, weight, bias, True, rows, state, BF, "other", offset)
    check(y, kept, x, weight, bias, True, rows, state, torch.full_like(state, UNTOUCHED))
    y, kept = run(hip, x, weight, bias, True, rows, state, BF, "none", offset)
    check(y, kept, x, weight, bias, True, rows, state, state)


def test_without_states_or_rows(hip):
    x, weight, bias, _ = inputs(6, 40, 4, BF, BF, False)
    rows = Rows(None, [1, 5, 0, 2], seqs=4, T=6)
    y, kept = run(hip, x, weight, bias, False, rows, None, BF, "other")
    check(y, kept, x, weight, bias, False, rows, None, torch.full((5, 3, 40), UNTOUCHED, dtype=BF))
    y = torch.full_like(x, UNTOUCHED).cuda()
    rows = Rows([6], device="cuda")
    hip("causal_conv", x.cuda(), DTYPE[BF], 40, weight.cuda(), None, DTYPE[BF], 4, ACT_NONE, pointer(rows.lx()), None, y, DTYPE[BF], 40, 6, 40)
    check(y, None, x, weight, bias, False, Rows([6]), None, torch.zeros(0, 3, 40))


def test_pieces_equal_the_whole(hip):
    # A prompt in pieces gives the bits of the prompt at once.
    x, weight, bias, _ = inputs(90, 136, 4, BF, BF, True, 5)
    whole, _ = run(hip, x, weight, bias, True, Rows([90], [90]), torch.zeros(1, 3, 136, dtype=BF), BF)
    state, parts, at = torch.full((1, 3, 136), 9.0, dtype=BF), [], 0
    for n in (1, 2, 30, 1, 16, 40):
        at += n
        y, kept = run(hip, x[at - n:at], weight, bias, True, Rows([n], [at]), state, BF)
        parts.append(y)
        state = kept.cpu()
    assert torch.equal(torch.cat(parts).view(torch.int16), whole.contiguous().view(torch.int16))


def test_infinities_and_nans_stay_in_their_channel_and_reach(hip):
    x, weight, _, _ = inputs(50, 64, 4, BF, BF, False, 6)
    x[20, 5], x[30, 9] = float("nan"), float("inf")
    weight[9, 1] = 0.25
    y, _ = run(hip, x, weight, None, False, Rows([50], [50]), torch.zeros(1, 3, 64, dtype=BF), F, "none")
    odd = ~torch.isfinite(y.cpu())
    want = torch.zeros_like(odd)
    want[20:24, 5] = want[30:34, 9] = True
    assert torch.equal(odd, want)


def test_garbage_in_device_memory_stays_in_bounds(hip):
    x, weight, _, _ = inputs(20, 64, 4, BF, BF, False, 7)
    rows = torch.tensor([-9, 1 << 30, 3, -(1 << 31), 7], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([1 << 30, -4, 2, (1 << 31) - 1], dtype=torch.int32, device="cuda")
    slots = torch.tensor([-(1 << 31), (1 << 31) - 1, 1, 5], dtype=torch.int32, device="cuda")
    from dromos_amd.abi import LxKv8Batch

    state, y = torch.zeros(2, 3, 64, dtype=BF, device="cuda"), torch.zeros(20, 64, dtype=BF, device="cuda")
    batch = LxKv8Batch(4, rows.data_ptr(), lengths.data_ptr(), None, 0, 20, 0)
    states = LxStates(state.data_ptr(), state.data_ptr(), slots.data_ptr(), 2)
    hip("causal_conv", x.cuda(), DTYPE[BF], 64, weight.cuda(), None, DTYPE[BF], 4, ACT_NONE, pointer(batch), pointer(states), y, DTYPE[BF], 64, 20, 64)
    assert torch.isfinite(y.float()).all()

"""Edges of lx_rotate, lx_causal_conv and lx_linear_attention: places beyond 2^31, rows of nobody that hold NaNs, scales that are no part of an exponent,
steps of width zero, workspaces without a byte to spare. Tolerances as in those operators' own tests."""

import pytest
import torch

from dromos_amd.abi import ACT_NONE, BF16, F32, LxStates
from mixer import UNTOUCHED, Mixer, Rows, convolved, pointer, rotated

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
SHARE = 2.0**-14
FAR = 1 << 22  # a row's stride: 1100 rows end behind 2^32 values


def far_rows(T, width, dtype, values=None):
    """[T, width] at a stride of FAR."""
    whole = torch.empty((T - 1) * FAR + width, dtype=dtype, device="cuda")
    t = whole.as_strided((T, width), (FAR, 1))
    t.fill_(UNTOUCHED) if values is None else t.copy_(values)
    return t


def test_rows_beyond_32_bits(hip):
    T, g = 1100, torch.Generator().manual_seed(1)
    batch = Rows([T], [T + 3], [0], device="cuda")
    x = torch.randn(T, 64, generator=g).to(BF)
    freq = torch.tensor([0.5**i for i in range(32)], dtype=F)
    given, y = far_rows(T, 64, BF, x), far_rows(T, 64, BF)
    hip("rotate", given, BF16, FAR, y, BF16, FAR, pointer(batch.lx()), None, freq.cuda(), 1.0, 64, 0, T, 1, 64)
    want, size = rotated(x, torch.arange(3, T + 3), freq, 1.0, 64, False, 1, 64)
    assert bool(((y.double().cpu() - want).abs() <= 2.0**-21 * size + 2.0**-8 * 1.01 * (want.abs() + 2.0**-21 * size)).all())
    weight, kept = torch.randn(64, 4, generator=g), torch.randn(1, 3, 64, generator=g).to(BF)
    y.fill_(UNTOUCHED)
    w, held = weight.cuda(), kept.cuda()
    states = batch.states(held, held, 1)
    hip("causal_conv", given, BF16, FAR, w, None, F32, 4, ACT_NONE, pointer(batch.lx()), pointer(states), y, BF16, FAR, T, 64)
    want, size, after = convolved(x, weight, None, False, Rows([T], [T + 3], [0]), kept, 1)
    share = 1.1 * 5 * 2.0**-24 * size
    assert bool(((y.double().cpu() - want).abs() <= share + 2.0**-8 * 1.01 * (want.abs() + share)).all())
    assert torch.equal(held[0].double().cpu(), after[0])


@pytest.mark.parametrize("rows", [[3], [1100], [600, 500]])
def test_linear_attention_beyond_32_bits(hip, rows):
    T = sum(rows)
    batch = Rows(rows, [n + 5 for n in rows], list(range(len(rows))))
    m = Mixer(batch, 2, 1, 64, 64, "step", True, BF, seed=T)
    want = m.want()
    device = Rows(rows, batch.lengths, batch.slots, device="cuda")
    held = {}

    def call(args):
        args = list(args)
        for at, ld in ((0, 4), (1, 5), (2, 6), (9, 11), (14, 16)):
            held[at] = far_rows(T, args[at].shape[1], args[at].dtype, None if at == 14 else args[at])
            args[at], args[ld] = held[at], FAR
        hip("linear_attention", *args)

    _, kept = m.run(hip, call=call)
    m.check(held[14], kept, want, SHARE)
    assert device.T == T


@pytest.mark.parametrize("rows", [2, 70])
def test_slots_beyond_32_bits(hip, rows):
    # 256 KiB a slot of f32: slot 8200 begins behind 2^31 bytes, slot 33000 behind 2^31 values.
    heads, dk, dv, slots = 4, 128, 128, [33000, 8200]
    m = Mixer(Rows([rows, rows], [rows + 4] * 2, [0, 1]), heads, 2, dk, dv, "log", seed=rows)
    want = m.want()
    states = torch.empty(slots[0] + 1, heads, dk, dv, device="cuda")
    for i, slot in enumerate(slots):
        states[slot].copy_(m.state[i])
    at = torch.tensor(slots, dtype=torch.int32, device="cuda")

    def call(args):
        args = list(args)
        args[13] = pointer(LxStates(states.data_ptr(), states.data_ptr(), at.data_ptr(), states.shape[0]))
        hip("linear_attention", *args)

    out, _ = m.run(hip, call=call)
    m.count = 2
    m.check(out, torch.stack([states[slot] for slot in slots]), want, SHARE)


@pytest.mark.parametrize("max_rows", [4, 60, 300])
def test_nans_in_rows_of_nobody(hip, max_rows):
    """Rows in front of position 0, from max_rows on and behind the last sequence, and the states of sequences that begin."""
    counts = [max_rows + 2, 5, 1]
    rows = Rows(counts, [max_rows, 3, 1], [0, 1, 2], T=sum(counts) + 3, max_rows=max_rows)
    m = Mixer(rows, 4, 2, 64, 64, "step", True, BF, seed=max_rows)
    nobody = torch.ones(rows.T, dtype=torch.bool)
    for _, begin, end, _, _, _ in rows.spans():
        nobody[begin:end] = False
    assert bool(nobody.any())
    want = m.want()
    for t in (m.q, m.k, m.v, m.gate, m.x):
        t[nobody] = float("nan")
    m.state[:] = float("nan")
    before = torch.full_like(m.state, UNTOUCHED)
    out, kept = m.run(hip, keep="other")
    m.check(out, kept, want, SHARE, before)
    x = torch.randn(rows.T, 40).to(BF)
    x[nobody] = float("nan")
    weight, y = torch.randn(40, 4), torch.full((rows.T, 40), UNTOUCHED, dtype=BF, device="cuda")
    device = Rows(counts, rows.lengths, rows.slots, rows.T, max_rows, device="cuda")
    held, w = torch.full((3, 3, 40), float("nan"), dtype=BF, device="cuda"), weight.cuda()
    states = device.states(held, held, 3)
    hip("causal_conv", x.cuda(), BF16, 40, w, None, F32, 4, ACT_NONE, pointer(device.lx()), pointer(states), y, BF16, 40, rows.T, 40)
    want, size, after = convolved(x, weight, None, False, rows, None, 3)
    share = 1.1 * 5 * 2.0**-24 * size[~nobody]
    assert bool((y.cpu()[nobody] == UNTOUCHED).all())
    assert bool(((y.double().cpu()[~nobody] - want[~nobody]).abs() <= share + 2.0**-8 * 1.01 * (want[~nobody].abs() + share)).all())
    for slot, values in after.items():
        assert torch.equal(held[slot].double().cpu(), values)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-36, 3e33])
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_scales(hip, rows, scale):
    # f32 results: in bf16 the smallest ones would be subnormal.
    m = Mixer(Rows([rows], [rows + 2], [0]), 4, 2, 64, 64, "log", skip=scale == 0.0, out=F, seed=rows)
    m.scale = scale
    out, kept = m.run(hip)
    m.check(out, kept, m.want(), SHARE)


@pytest.mark.parametrize("rows", [4, 90, 400])
def test_steps_of_width_zero(hip, rows):
    """x = -infinity: a step of width 0 adds nothing and nothing fades; where g is x itself, all that was is forgotten."""
    for decay in ("step", "log"):
        m = Mixer(Rows([rows], [rows + 7], [0]), 4, 2, 64, 64, decay, out=F, seed=rows, rate=False)
        m.x[::3, 1], m.x[1, 2], m.x[rows - 1, 3] = (float("-inf"),) * 3
        out, kept = m.run(hip)
        m.check(out, kept, m.want(), SHARE)


@pytest.mark.parametrize("dk,dv,counts", [(64, 64, [300]), (128, 128, [129, 700, 2]), (256, 40, [1000, 260])])
def test_workspace_to_the_byte(hip, dk, dv, counts):
    m = Mixer(Rows(counts, counts, list(range(len(counts)))), 4, 2, dk, dv, "step", seed=dk)
    batch = m.rows.lx()
    need = int(hip.size("linear_attention_workspace_bytes", pointer(batch), m.rows.T, 4, 2, dk, dv))
    assert need > 0
    space = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    out, kept = m.run(hip, workspace=space)
    m.check(out, kept, m.want(), SHARE)
    assert bool((space[need:] == 0xFF).all())


@pytest.mark.parametrize("decay", ["log", "step"])
@pytest.mark.parametrize("rows,dk,dv", [(7, 128, 64), (64, 64, 64), (200, 128, 128), (200, 256, 72), (700, 128, 64)])
def test_states_and_f32_results_keep_their_precision(hip, rows, dk, dv, decay):
    """As a whole, by 2-norms. A token's factors are off by 2^-22 each (an exponent up to 4 rounded, its exponential), 2^-23 on average and on their own, terms
    and products by 2^-24, and twelve sums a chunk by 2^-24 each, 2^-22 together where they come as they like: under 2^-20."""
    for out in (F, BF):
        m = Mixer(Rows([rows], [rows + 9], [0]), 4, 2, dk, dv, decay, out=out, seed=rows + dk)
        want = m.want()
        got, kept = m.run(hip)
        assert (kept[0].double().cpu() - want["states"][0]).norm() <= 2.0**-20 * want["states"][0].norm()
        if out == F:
            assert (got.double().cpu() - want["out"]).norm() <= 2.0**-20 * want["out"].norm()


@pytest.mark.parametrize("counts", [[70, 3], [300, 0, 0, 400], [0, 0, 513, 0]])
def test_no_lengths(hip, counts):
    """No sequence begins with such a call."""
    m = Mixer(Rows(counts, None, list(range(len(counts)))), 2, 1, 64, 64, "step", seed=1)
    out, kept = m.run(hip)
    m.check(out, kept, m.want(), SHARE)


@pytest.mark.parametrize("most", [2, 8])
def test_thousands_of_sequences(hip, most):
    """More than the 64 x 64 that two turns of the search for a row's sequence tell apart; some are empty."""
    g = torch.Generator().manual_seed(most)
    counts = torch.randint(0, most + 1, (4200,), generator=g).tolist()
    slots = torch.randperm(4200, generator=g).tolist()
    rows = Rows(counts, [n + i % 3 for i, n in enumerate(counts)], slots)
    m = Mixer(rows, 1, 1, 8, 8, "log", seed=most)
    out, kept = m.run(hip)
    m.check(out, kept, m.want(), SHARE)
    x, weight, front = torch.randn(rows.T, 8, generator=g).to(BF), torch.randn(8, 4, generator=g), torch.randn(4200, 3, 8, generator=g).to(BF)
    device = Rows(counts, rows.lengths, slots, device="cuda")
    held, w, y = front.cuda(), weight.cuda(), torch.full((rows.T, 8), UNTOUCHED, dtype=BF, device="cuda")
    # Bounds far above the real rows: pieces, and a search among them.
    device.max_rows = 100
    states = device.states(held, held, 4200)
    hip("causal_conv", x.cuda(), BF16, 8, w, None, F32, 4, ACT_NONE, pointer(device.lx()), pointer(states), y, BF16, 8, rows.T, 8)
    want, size, after = convolved(x, weight, None, False, rows, front, 4200)
    share = 1.1 * 5 * 2.0**-24 * size
    assert bool(((y.double().cpu() - want).abs() <= share + 2.0**-8 * 1.01 * (want.abs() + share)).all())
    whole = front.double()
    for slot, values in after.items():
        whole[slot] = values
    assert torch.equal(held.double().cpu(), whole)


def test_bounds_above_the_real_rows(hip):
    """One captured size for anything up to it: the same results whatever max_rows says, as long as the same form is taken."""
    outs = []
    for most in (160, 700, 100000):
        m = Mixer(Rows([160, 5], [160, 30], [0, 1], T=700, max_rows=most), 4, 2, 128, 64, "step", True, BF, seed=3)
        out, kept = m.run(hip)
        m.check(out, kept, m.want(), SHARE)
        outs.append((out, kept))
    assert all(torch.equal(outs[0][i], o[i]) for o in outs[1:] for i in range(2))

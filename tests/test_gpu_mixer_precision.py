"""What lx_rotate, lx_causal_conv and lx_linear_attention keep of f32 where little things add up or sizes are extreme: slow decays, updates' weights,
gates, skips, infinities, far positions; and that a sequence's bits do not depend on how many others a call has."""

import math
from fractions import Fraction

import pytest
import torch

from dromos_amd.abi import ACT_SILU, BF16, DECAY_HEAD, DTYPE, F32, LxDecay, LxKv8Batch, LxStates
from mixer import UNTOUCHED, Mixer, Rows, pointer

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


class Fading:
    """Calls of `rows` rows whose keys are zero: a state of 64 x 64 that only fades, by a constant rate."""

    def __init__(self, hip, rows, rate, seed):
        self.hip, self.rows = hip, rows
        self.before = torch.rand(64, 64, generator=torch.Generator().manual_seed(seed)) + 0.5
        self.state, self.rate = self.before.cuda().view(1, 1, 64, 64), torch.tensor([rate], device="cuda")
        self.x, self.out = torch.zeros(rows, 64, dtype=BF, device="cuda"), torch.empty(rows, 64, dtype=BF, device="cuda")
        self.first = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        self.decay = LxDecay(DECAY_HEAD, None, F32, 1, self.rate.data_ptr(), None)
        self.batch, self.states = LxKv8Batch(1, self.first.data_ptr(), None, None, 0, rows, 0), LxStates(self.state.data_ptr(), self.state.data_ptr(), None, 1)
        need = int(hip.size("linear_attention_workspace_bytes", pointer(self.batch), rows, 1, 1, 64, 64))
        self.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

    def call(self):
        assert self.hip.status("linear_attention", self.x, self.x, self.x, BF16, 64, 64, 64, pointer(self.decay), None, None, BF16, 0, pointer(self.batch),
                               pointer(self.states), self.out, BF16, 64, self.rows, 1, 1, 64, 64, 0.125, self.workspace) == 0

    def errors(self, tokens):
        """The relative errors of the state's values."""
        want = self.before.double() * torch.exp(tokens * self.rate.double().cpu())
        return self.state[0, 0].double().cpu() / want - 1


@pytest.mark.parametrize("rate", [-1e-5, -1e-6])
@pytest.mark.parametrize("rows", [300, 131072])
def test_slow_decays_of_a_prompt(hip, rows, rate):
    """Up to 512 parts, a rounding of half a step, 2^-24, a part: at random 2^-24 sqrt(512 / 3) = 2^-20.3 of a value, and of 4096 values' mean a 64th of that, 2^-26.3,
    four times which is 2^-24.3. To one side: of each part's logarithm 2^-22 (its sum's rounding, the exponential's and a logarithm's), 2^-22 |n rate| together; a sum's
    last place, 2^-40 a token at most, 2^-23 of 131072 of them."""
    f = Fading(hip, rows, rate, 1)
    f.call()
    errors = f.errors(rows)
    assert abs(errors.mean().item()) <= 2.0**-22 * abs(rows * rate) + 2.0**-23
    assert errors.abs().max().item() <= 2.0**-22 * abs(rows * rate) + 2.0**-18


@pytest.mark.parametrize("rows,pieces", [(1, [1]), (6, [1] * 6), (7, [7]), (8, [8]), (64, [64]), (130, [128, 2])])
def test_slow_decays_of_many_short_calls(hip, rows, pieces):
    """8192 calls; a state is rounded once a piece. That is nothing random where a state falls by few steps at a time (6 rows: 4e-6 of a value, to one side), so what is
    compared with is the same in 64 bits rounded as often. Beside that the logarithms' errors, 2^-22 of them as in a prompt, and their last places, 2^-21 of all tokens."""
    calls, whole = 8192, -0.57
    f = Fading(hip, rows, whole / (calls * rows), 2)
    for _ in range(calls):
        f.call()
    rate, state = f.rate.double().item(), f.before.clone()
    fades = [math.exp(rate * n) for n in pieces]
    for _ in range(calls):
        for fade in fades:
            state = (state.double() * fade).float()
    apart = f.state[0, 0].double().cpu() / state.double() - 1
    assert abs(apart.mean().item()) <= 2.0**-22 * -whole + 2.0**-21
    assert apart.abs().max().item() <= 2.0**-22 * -whole + 2.0**-19


@pytest.mark.parametrize("rows", [1, 6, 7, 64, 300])
def test_strong_decays_of_a_state(hip, rows):
    """One factor, or some, down to the smallest normal number: each right to 2^-22 (an exponential and its correction) and a rounding of the state, of a token, or of a chunk or a
    part. A chunk's logarithm is a sum, a product and a part's sum, each of 24 bits: 3 2^-24 of itself."""
    for log in (-0.3, -0.6, -5.0, -40.0, -80.0, -86.5):
        f = Fading(hip, rows, log / rows, 3)
        f.call()
        assert f.errors(rows).abs().max().item() <= (2.0**-22 + 2.0**-24) * (rows if rows <= 6 else (rows + 63) // 64) + (3 * 2.0**-24 * -log if rows > 6 else 0)


def test_steps_of_any_width(hip):
    """softplus(x) from 1e-7 to 20, as the first update of a state of ones: an exponential right to 2^-23 and a rounding, a logarithm to 2^-22, two more roundings."""
    seqs, heads = 64, 64
    m = Mixer(Rows([1] * seqs, [1] * seqs), heads, 1, 8, 8, "step", seed=1, bias=False, spare=0)
    m.x = torch.linspace(-16, 20, seqs * heads).view(seqs, heads)
    m.k, m.v = torch.ones(seqs, 8, dtype=BF), torch.ones(seqs, heads * 8, dtype=BF)
    _, kept = m.run(hip)
    want = torch.log1p(torch.exp(m.x.double()))[:, :, None, None]
    assert ((kept.double().cpu() / want - 1).abs().max().item()) <= 2.0**-22 + 2.0**-23 + 3 * 2.0**-24


def relative(got, want):
    errors = got.double().cpu() / want - 1
    return errors.square().mean().sqrt().item(), errors.abs().max().item()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (256, 64)])
def test_updates_weights(hip, far, dk, dv):
    """A row of the state for each token, and a column of the values: states and results are single weights, e^{G - G_j} b_j. Steps that are their x as they stand
    (100 and more), decays of hardly anything. An exponential is right to 2^-23, a product to 2^-24: of a state one and one, and 2^-24 for terms and sums, 2^-22
    together, 2^-23.6 on average (each anywhere within its bound); of a result's weight two and five, 2^-20.8 and 2^-23. `far`: a token that all before it is forgotten at."""
    rows, heads = 64, 4
    m = Mixer(Rows([rows], [rows], [0]), heads, 1, dk, dv, "step", out=F, seed=dk, spare=0)
    g = torch.Generator().manual_seed(9)
    m.x = torch.rand(rows, heads, generator=g) * 1900 + 100
    m.bias, m.rate = None, -torch.rand(heads, generator=g) * 1e-5
    if far:
        m.x[0], m.rate[:] = 1e7, -1e-5
    m.k, m.q, m.v = torch.zeros(rows, dk, dtype=BF), torch.zeros(rows, dk, dtype=BF), torch.zeros(rows, heads, dv, dtype=BF)
    for t in range(rows):
        m.k[t, t % dk], m.v[t, :, t % dv] = 1.0, 1.0
    m.q[:] = 1.0
    m.v = m.v.view(rows, heads * dv)
    m.scale = 0.5
    b = m.x.double()
    sums = (b * m.rate.double()).cumsum(0)
    out, kept = m.run(hip)
    at = torch.arange(rows)
    state = kept[0].cpu()[:, at % dk, at % dv].t()  # [rows, heads]
    mean, worst = relative(state[1:], (torch.exp(sums[-1] - sums) * b)[1:])
    assert mean <= 2.0**-23.3 and worst <= 2.0**-22
    seen = out.cpu().view(rows, heads, dv)[:, :, at % dv]  # [row, head, token]
    want = 0.5 * torch.exp(sums[:, :, None] - sums.t()[None]) * b.t()[None]
    some = (at[:, None] >= at)[:, None].expand(-1, heads, -1) & (at > 0)
    mean, worst = relative(seen[some], want[some])
    assert mean <= 2.0**-22.9 and worst <= 2.0**-20.8
    assert bool((seen[(at[:, None] < at)[:, None].expand(-1, heads, -1)] == 0).all())


@pytest.mark.parametrize("heads,k_heads,dk,dv", [(32, 32, 128, 128), (32, 8, 256, 64), (64, 4, 72, 40), (32, 32, 64, 64)])
@pytest.mark.parametrize("rows", [1, 3])
def test_bits_do_not_depend_on_how_many_sequences(hip, rows, heads, k_heads, dk, dv):
    """f32 results and states, bit for bit, of the first sequence by itself, with one more, with 40 more."""
    alone = Mixer(Rows([rows], [rows + 2], [1], max_rows=rows), heads, k_heads, dk, dv, "step", True, BF, out=F, seed=4)
    first, state = alone.run(hip)
    for others in (1, 40):
        counts, slots = [rows] * (1 + others), [1, 0] + list(range(2, others + 1))
        more = Mixer(Rows(counts, [rows + 2] + [9] * others, slots, max_rows=rows), heads, k_heads, dk, dv, "step", True, BF, out=F, seed=5)
        for name in ("q", "k", "v", "x", "gate"):
            getattr(more, name)[:rows] = getattr(alone, name)
        more.rate, more.bias, more.skip, more.state[1] = alone.rate, alone.bias, alone.skip, alone.state[1]
        out, kept = more.run(hip)
        assert torch.equal(out[:rows], first) and torch.equal(kept[1], state[1]), others


@pytest.mark.parametrize("rate", [0.0, -1e-4, -0.3, -3.0])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 64), (256, 32)])
@pytest.mark.parametrize("rows", [1, 5, 70, 400])
def test_infinities_of_a_state(hip, rows, dk, dv, rate):
    """An infinity of a state stays one and where it is, unless all that a chunk leaves of a state is nothing in f32 (e^-192 < 2^-149), whose product with it is a NaN. Token by
    token its column's results are the sum's; by chunks they are no numbers (an infinity or a NaN). All others are as they are without it."""
    m = Mixer(Rows([rows], [rows + 7], [0]), 2, 1, dk, dv, "head", out=F, seed=rows + dk)
    m.rate[:] = rate
    clean, kept = m.run(hip)
    m.state[0, 0, 3, 5], m.state[0, 1, dk - 1, dv - 1] = float("inf"), float("-inf")
    out, after = m.run(hip)
    kept[0, 0, 3, 5], kept[0, 1, dk - 1, dv - 1] = float("inf"), float("-inf")
    if rows > 6 and 64 * rate < -150:
        for at in ((0, 0, 3, 5), (0, 1, dk - 1, dv - 1)):
            assert not math.isfinite(after[at].item())
            after[at] = kept[at]
    assert torch.equal(after, kept)
    clean, out = clean.view(rows, 2, dv), out.view(rows, 2, dv)
    for head, column, row, sign in ((0, 5, 3, 1.0), (1, dv - 1, dk - 1, -1.0)):
        seen = out[:, head, column].clone()
        assert not bool(torch.isfinite(seen).any())
        if rows <= 6:
            assert torch.equal(seen, sign * m.q[:, row].float().cuda().sign() * float("inf"))
        out[:, head, column] = clean[:, head, column]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("gate", [BF, F])
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_gates_of_f32_results(hip, rows, gate):
    """silu right to 2^-21 at any size, and to 2e-36 where it is less; keys and queries of zero, so that a result is its gate's factor (of two products, 2^-23)."""
    heads, dv = 2, 64
    m = Mixer(Rows([rows], [rows], [0]), heads, 1, 64, dv, "head", True, gate, out=F, seed=rows)
    m.k.zero_(), m.q.zero_(), m.v.fill_(1.0), m.skip.fill_(1.0)
    m.gate = ((torch.rand(rows, heads * dv, generator=torch.Generator().manual_seed(3)) - 0.5) * 176).to(gate)
    m.gate[0, :8] = torch.tensor([0.0, 1e30, -1e30, 3e38, -3e38, float("inf"), -90.0, -104.0]).to(gate)
    out, _ = m.run(hip)
    z = m.gate.double()
    want = z / (1 + torch.exp(-z))
    out = out.double().cpu()
    assert out[0, 5].item() == float("inf")
    out[0, 5] = want[0, 5] = 0.0
    assert bool(((out - want).abs() <= (2.0**-21 + 2.0**-23) * want.abs() + 2e-36).all())


@pytest.mark.parametrize("rows", [3, 64, 300])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (256, 72)])
def test_skips_of_bf16_results(hip, rows, dk, dv):
    """Queries of zero: a result is the skip's product, rounded to f32 and to bf16. The first rounding, 2^-24, moves the second one where a product is as near to a border, whose
    distances are 2^-8 or more: in 2^-15 of all. Twice that and a few."""
    m = Mixer(Rows([rows], [rows]), 4, 2, dk, dv, "step", True, seed=rows)
    m.q.zero_()
    out, _ = m.run(hip)
    want = (m.skip.double()[:, None] * m.v.double().view(rows, 4, dv)).view(rows, 4 * dv).to(BF)
    assert (out.cpu() != want).sum().item() <= 2.0**-14 * out.numel() + 4


@pytest.mark.parametrize("out", [F, BF])
def test_silu_of_a_convolution(hip, out):
    """As the gates', sums of f32 that are their last row as it stands; bf16 results' own rounding beside 2^-17."""
    C, z = 64, torch.cat([torch.linspace(-88, 88, 52), torch.tensor([1e30, -1e30, 3e38, -3e38, -90.0, -104.0, -1e5, 1e5, 0.0, -0.5, 300.0, float("inf")])])
    x = torch.zeros(2, C)
    x[1] = z
    weight, y = torch.tensor([[0.0, 1.0]] * C).cuda(), torch.full((2, C), UNTOUCHED, dtype=out, device="cuda")
    rows = Rows([2], [2], device="cuda")
    hip("causal_conv", x.cuda(), F32, C, weight, None, F32, 2, ACT_SILU, pointer(rows.lx()), None, y, DTYPE[out], C, 2, C)
    got, want = y[1].double().cpu(), z.double() / (1 + torch.exp(-z.double()))
    assert got[-1].item() == float("inf")
    share = 2.0**-21 if out == F else 2.0**-17 + 2.0**-8 * 1.01
    assert bool(((got - want).abs()[:-1] <= share * want.abs()[:-1] + 2e-36).all())


# pi to 60 places after the point.
PI = Fraction(3141592653589793238462643383279502884197169399375105820974944, 10**60)


def exact_turn(position, freq):
    """cos and sin of position * freq, the angle reduced in whole numbers."""
    angle = position * Fraction(freq)
    left = float(angle - round(angle / (2 * PI)) * 2 * PI)
    t = torch.tensor(left, dtype=torch.float64)
    return t.cos().item(), t.sin().item()


@pytest.mark.parametrize("interleaved", [0, 1])
def test_rotation_at_far_positions(hip, interleaved):
    """The angle is the product in 64 bits, off by 2^-53 twice: p f 2^-52; cosine and sine beside that by 2^-23 (the reduced angle's rounding, 2^-25, and the series');
    two products and a sum 2^-22 of |a| + |b|."""
    freq = torch.tensor([1.0, 0.7, 1e-2, 3.3e-5], dtype=F)
    positions = [0, 1, 131071, 1 << 20, (1 << 26) + 5, (1 << 30) - 1, (1 << 31) - 1, -(1 << 31), -77777777]
    T, rot = len(positions), 8
    x = torch.randn(T, rot, generator=torch.Generator().manual_seed(1))
    y = torch.full((T, rot), UNTOUCHED, device="cuda")
    hip("rotate", x.cuda(), F32, rot, y, F32, rot, None, torch.tensor(positions, dtype=torch.int32).cuda(), freq.cuda(), 1.0, rot, interleaved, T, 1, rot)
    got = y.double().cpu()
    for t, position in enumerate(positions):
        for i in range(rot // 2):
            c, s = exact_turn(position, freq[i].item())
            at = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            a, b = x[t, at[0]].item(), x[t, at[1]].item()
            bound = (abs(a) + abs(b)) * (abs(position * freq[i].item()) * 2.0**-52 + 2.0**-23 + 2.0**-22)
            assert abs(got[t, at[0]].item() - (a * c - b * s)) <= bound and abs(got[t, at[1]].item() - (b * c + a * s)) <= bound, (position, i)

"""lx_linear_attention against the recurrence in 64 bits, token by token.

Tolerance, as a share of the sum of the magnitudes that a result is made of. Token by token: exp(g) is off by 2^-22 (g's rounding included where |g|
is at most 4: beyond, what it multiplies has faded), a token's update by three roundings, so a state of n tokens by 2^-22 n + 2^-22 at most, n counted
up to the rows of these tests, 20: below 2^-17; an output adds dk products in f32, 256 of 2^-24 at most: 2^-16. Chunks: f32 factors enter products as
two bf16, which leaves 2^-16 of them (a first rounding's half step 2^-8, of what is left another 2^-8); a result passes through a state's update and its
use, or a weight of a token: 2^-15; sums of 64 + 256 products in f32 2^-15.7; exponentials 2^-20. Together below 2^-14, on both forms' account."""

import pytest
import torch

from dromos_amd.abi import BF16, DECAY_HEAD, F32, LxDecay, LxKv8Batch, LxStates
from mixer import UNTOUCHED, Mixer, Rows, pointer

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
SHARE = 2.0**-14


def check(hip, m, **options):
    want = m.want()
    out, kept = m.run(hip, **options)
    m.check(out, kept, want, SHARE)


@pytest.mark.parametrize("decay", ["head", "log", "step"])
@pytest.mark.parametrize("heads,k_heads,dk,dv", [(1, 1, 64, 64), (4, 2, 128, 64), (6, 6, 128, 128), (3, 1, 256, 256), (2, 2, 8, 8), (5, 5, 96, 80), (4, 1, 40, 200), (2, 1, 248, 136),
                                                 (1, 1, 64, 512), (16, 2, 128, 64), (9, 3, 136, 24)])
@pytest.mark.parametrize("counts,lengths", [([1], [1]), ([1, 1, 1], [9, 1, 3]), ([5, 0, 2], [7, 3, 2]), ([20], [20])])
def test_few_rows(hip, counts, lengths, heads, k_heads, dk, dv, decay):
    slots = [2 * i + 1 for i in range(len(counts))]
    check(hip, Mixer(Rows(counts, lengths, slots), heads, k_heads, dk, dv, decay, True, BF, seed=dk + dv))


@pytest.mark.parametrize("decay", ["head", "log", "step"])
@pytest.mark.parametrize("heads,k_heads,dk,dv", [(1, 1, 64, 64), (4, 2, 128, 64), (2, 2, 128, 128), (3, 1, 256, 256), (2, 2, 8, 8), (2, 2, 96, 80), (4, 1, 40, 200), (2, 1, 248, 136),
                                                 (1, 1, 64, 512), (16, 2, 128, 64), (9, 3, 136, 24), (3, 1, 64, 32), (6, 2, 128, 48)])
@pytest.mark.parametrize("counts,lengths", [([64], [64]), ([130, 0, 1, 63], [130, 3, 1, 90]), ([33], [40]), ([200], [1000])])
def test_many_rows(hip, counts, lengths, heads, k_heads, dk, dv, decay):
    slots = [2 * i + 1 for i in range(len(counts))]
    check(hip, Mixer(Rows(counts, lengths, slots), heads, k_heads, dk, dv, decay, seed=dk + dv))


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("dtype,out,gate,skip,step", [(BF, F, None, True, BF), (F, F, F, False, F), (F, BF, BF, True, BF), (BF, BF, F, True, F), (BF, F, BF, False, BF)])
@pytest.mark.parametrize("decay", ["log", "step"])
def test_types_skip_and_gate(hip, decay, dtype, out, gate, skip, step, rows):
    for heads, k_heads, dk, dv in ((4, 2, 128, 64), (3, 3, 72, 104)):
        m = Mixer(Rows([rows, 2], [rows, 9]), heads, k_heads, dk, dv, decay, skip, gate, dtype, out, step, seed=rows, bias=skip, rate=skip)
        check(hip, m)


@pytest.mark.parametrize("heads,k_heads,dk,dv", [(4, 2, 128, 64), (2, 2, 64, 128), (2, 1, 256, 64)])
@pytest.mark.parametrize("counts,lengths,slots,T,max_rows", [
    ([1] * 70, None, None, 70, None), ([5, 1, 90], None, [2, 0, 1], 100, None), ([70, 6], [40, 2], [0, 1], 80, None), ([4, 70], [0, 0], None, 74, None),
    ([100, 150], [100, 500], None, 250, 67), ([3] * 40, [i % 5 for i in range(40)], None, 120, None), ([2, 80, 2], [9, 99, 9], [1, -1, 99], 84, None),
    ([64, 128, 0, 192, 1, 65], [64, 999, 4, 192, 7, 65], None, 450, None), ([0, 0], [3, 0], None, 4, None)])
def test_batches(hip, counts, lengths, slots, T, max_rows, heads, k_heads, dk, dv):
    rows = Rows(counts, lengths, slots, T, max_rows)
    m = Mixer(rows, heads, k_heads, dk, dv, "step", True, BF, seed=T)
    if slots and 99 in slots:
        m.count, m.state = 3, m.state[:3].clone()
    want = m.want()
    out, kept = m.run(hip)
    m.check(out, kept, want, SHARE)
    out, kept = m.run(hip, keep="other")
    m.check(out, kept, want, SHARE, torch.full_like(m.state, UNTOUCHED))
    out, kept = m.run(hip, keep="none")
    m.check(out, kept, want, SHARE)
    want = m.want(None)
    out, kept = m.run(hip, give=False)
    m.check(out, kept, want, SHARE, torch.full_like(m.state, UNTOUCHED))


def test_one_row_a_sequence_without_rows(hip):
    m = Mixer(Rows(None, [1, 5, 0, 2], seqs=4, T=6), 4, 2, 128, 64, "step", seed=1)
    check(hip, m)
    check(hip, Mixer(Rows(None, None, seqs=4, T=3), 4, 2, 128, 64, "head", seed=2))


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("rows", [2, 90])
def test_columns_of_one_tensor(hip, rows, pad):
    check(hip, Mixer(Rows([rows], [rows + 7]), 4, 2, 128, 64, "log", True, seed=pad), mixed=True, pad=pad)


@pytest.mark.parametrize("decay", ["head", "log", "step"])
@pytest.mark.parametrize("rows", [7, 150])
def test_strong_decays(hip, rows, decay):
    # Sums of logarithms far below what a chunk's other tokens see.
    check(hip, Mixer(Rows([rows, 1], [rows + 5, 1]), 4, 2, 64, 64, decay, seed=rows, strong=True))


@pytest.mark.parametrize("rows", [9, 140])
def test_fresh_starts_within_a_sequence(hip, rows):
    # A decay of minus infinity forgets everything in front of its token, exactly.
    m = Mixer(Rows([rows], [rows + 3]), 2, 1, 64, 64, "log", seed=3, rate=False)
    for t in (0, 5, 6, rows - 2):
        m.x[t, 0] = -float("inf")
    m.x[4, 1] = -1e30
    check(hip, m)
    # An infinity or a NaN in a value stays in its column and in front of the next fresh start (in its chunk's products, nothing times it is one too, so
    # rows behind it in the chunk may hold it); the columns beside it are numbers.
    m.v[2, 7] = float("nan")
    out, _ = m.run(hip)
    out = out.float().cpu().view(rows, 2, 64)
    assert bool(torch.isfinite(out[:, 0, :7]).all() and torch.isfinite(out[:, 0, 8:]).all() and torch.isfinite(out[:, 1]).all())
    assert bool(torch.isfinite(out[:2]).all())


@pytest.mark.parametrize("rows", [12, 100])
def test_pieces_equal_the_whole(hip, rows):
    # A prompt in pieces, each going on from the state that the last one left, against the prompt at once.
    m = Mixer(Rows([rows], [rows], [0]), 4, 2, 128, 64, "step", True, BF, out=F, seed=rows, spare=0)
    want = m.want()
    state, parts, at = torch.full_like(m.state, 9.0), [], 0
    sizes = [1, 3, 8] if rows == 12 else [1, 64, 30, 5]
    whole = {name: getattr(m, name) for name in ("q", "k", "v", "gate", "x")}
    for n in sizes:
        piece = m
        piece.rows = Rows([n], [at + n], [0])
        for name, t in whole.items():
            setattr(piece, name, t[at:at + n])
        piece.state = state
        out, kept = piece.run(hip)
        parts.append(out)
        state = kept.cpu()
        at += n
    m.check(torch.cat(parts), state, want, 2 * SHARE)


@pytest.mark.parametrize("T,counts", [(2048, [2048]), (1500, [700, 800]), (4200, [3000, 1, 1199])])
@pytest.mark.parametrize("heads,k_heads,dk,dv", [(2, 1, 64, 64), (1, 1, 128, 128), (1, 1, 256, 72)])
def test_long_sequences(hip, heads, k_heads, dk, dv, T, counts):
    lengths = [n + 13 * i for i, n in enumerate(counts)]
    m = Mixer(Rows(counts, lengths), heads, k_heads, dk, dv, "step", False, BF, out=F, seed=T)
    check(hip, m)


@pytest.mark.parametrize("rows", [1, 16, 4096])
def test_slow_decays_over_many_calls(hip, rows):
    # A memory of 4096 tokens, filled call after call: roundings of the decay must not go to one side. A state that is rounded to half a step, 2^-24, a
    # token, at random, is off by 2^-24 sqrt(4096 / 2), 2.7e-6, of its size; 2^-23 of e^g on one side would be 5e-4.
    n = 8192
    m = Mixer(Rows([n], [n], [0]), 1, 1, 64, 64, "head", seed=6, spare=0)
    m.rate = torch.tensor([-(2.0**-12) * 1.07])
    k = m.k.double().abs()
    m.k = k.to(BF)
    m.v = m.v.abs()
    t = torch.arange(n, dtype=torch.float64)
    fades = torch.exp((n - 1 - t) * m.rate.double())
    want = (m.k.double() * fades[:, None]).t() @ m.v.double()
    whole = {name: getattr(m, name).cuda() for name in ("q", "k", "v")}
    state = torch.zeros(1, 1, 64, 64, device="cuda")
    out = torch.empty(rows, 64, dtype=BF, device="cuda")
    rate, first = m.rate.cuda(), torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    decay = LxDecay(DECAY_HEAD, None, F32, 1, rate.data_ptr(), None)
    batch, states = LxKv8Batch(1, first.data_ptr(), None, None, 0, rows, 0), LxStates(state.data_ptr(), state.data_ptr(), None, 1)
    need = int(hip.size("linear_attention_workspace_bytes", pointer(batch), rows, 1, 1, 64, 64))
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    for at in range(0, n, rows):
        q, k, v = (whole[name][at:at + rows] for name in ("q", "k", "v"))
        assert hip.status("linear_attention", q, k, v, BF16, 64, 64, 64, pointer(decay), None, None, BF16, 0, pointer(batch), pointer(states), out, BF16, 64, rows, 1, 1,
                          64, 64, 0.125, workspace) == 0
    assert ((state[0, 0].double().cpu() - want).norm() / want.norm()).item() < 1e-5


def test_the_same_call_gives_the_same_bits(hip):
    for rows in (4, 300):
        m = Mixer(Rows([rows, 3], [rows, 7]), 4, 2, 128, 64, "step", True, BF, seed=11)
        first, state = m.run(hip)
        for _ in range(3):
            out, kept = m.run(hip)
            assert torch.equal(out.view(torch.int16), first.view(torch.int16)) and torch.equal(kept, state)


@pytest.mark.parametrize("rows", [3, 130])
def test_a_sequence_does_not_depend_on_its_neighbours(hip, rows):
    alone = Mixer(Rows([rows], [rows + 2], [1], max_rows=rows), 2, 1, 128, 64, "log", seed=4)
    first, state = alone.run(hip)
    more = Mixer(Rows([rows, rows, 0, 1], [rows + 2, 500, 3, 1], [1, 0, 4, 3], max_rows=rows), 2, 1, 128, 64, "log", seed=5)
    for name in ("q", "k", "v", "x"):
        getattr(more, name)[:rows] = getattr(alone, name)
    more.rate, more.state[1] = alone.rate, alone.state[1]
    out, kept = more.run(hip)
    assert torch.equal(out[:rows].view(torch.int16), first.view(torch.int16)) and torch.equal(kept[1], state[1])


def test_garbage_in_device_memory_stays_in_bounds(hip):
    for T, most in ((20, 3), (200, 200)):
        m = Mixer(Rows([T], [T]), 4, 2, 64, 64, "step", seed=8)
        rows = torch.tensor([-9, 1 << 30, 3, -(1 << 31), 7], dtype=torch.int32, device="cuda")
        lengths = torch.tensor([1 << 30, -4, 2, (1 << 31) - 1], dtype=torch.int32, device="cuda")
        slots = torch.tensor([-(1 << 31), (1 << 31) - 1, 1, 5], dtype=torch.int32, device="cuda")

        def call(args):
            state = args[13].contents
            batch = LxKv8Batch(4, rows.data_ptr(), lengths.data_ptr(), None, 0, most, 0)
            states = LxStates(state.in_, state.out, slots.data_ptr(), state.count)
            hip("linear_attention", *args[:12], pointer(batch), pointer(states), *args[14:])

        out, kept = m.run(hip, call=call)
        assert torch.isfinite(out.float()).all() and torch.isfinite(kept).all()

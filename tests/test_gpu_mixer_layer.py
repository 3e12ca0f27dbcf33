"""The operators of a linear-attention mixer together, as a program uses them, through the C ABI: lx_block_norm, the product into the mixer
(lx_gemm_w / lx_gemv_w), lx_causal_conv over values, keys and queries, lx_rotate of keys and queries in place, lx_linear_attention with the
product's first columns as its gate and its last ones as step widths, the product out of it and lx_block_norm again.

Each operator's result is checked against the same in 64 bits of what stood in its input, so that its own tolerance holds: norms 2^-20 (sums of
256 squares, a root), products 2^-15 (256 terms of 2^-24 each) of the magnitudes, the others as in their own tests; each result's rounding beside."""

import ctypes

import pytest
import torch

from dromos_amd.abi import ACT_SILU, BF16, DECAY_STEP, F32, MATH_BF16, NORM_RMS, W_BF16, LxDecay, LxKv8Batch, LxStates
from dromos_amd.formats import master_weight, quantize_with
from mixer import HALF, UNTOUCHED, Mixer, Rows, convolved, pointer, rotated

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

HEADS, K_HEADS, DK, DV, HIDDEN, TAPS, ROT = 4, 2, 64, 64, 256, 4, 32
VALUES, KEYS = HEADS * DV, K_HEADS * DK
C = VALUES + 2 * KEYS  # values, keys, queries
STEP = VALUES + C      # where the step widths stand, behind the gate and those
WIDE = STEP + 8


class Layer:
    """Weights and buffers for up to `most` rows; step() issues one pass over a batch's rows on a stream."""

    def __init__(self, hip, most, slots, seed=0, skinny=False):
        g = torch.Generator().manual_seed(seed)
        self.hip, self.slots, self.skinny = hip, slots, skinny
        self.in_w = quantize_with(hip, master_weight(WIDE, HIDDEN, g).cuda(), W_BF16)
        self.out_w = quantize_with(hip, master_weight(HIDDEN, VALUES, g).cuda(), W_BF16)
        self.structs = self.in_w.lx(), self.out_w.lx()
        self.norms = [(torch.randn(n, generator=g) * 0.1 + 1).to(BF).cuda() for n in (HIDDEN, VALUES, HIDDEN, HIDDEN)]
        self.taps = (torch.randn(C, TAPS, generator=g) * 0.5).to(BF).cuda()
        self.tap_bias = torch.randn(C, generator=g).to(BF).cuda()
        self.freq = torch.tensor([1e4 ** (-2 * i / ROT) for i in range(ROT // 2)], dtype=torch.float32).cuda()
        self.skip, self.rate, self.bias = ((torch.rand(HEADS, generator=g) * a + b).cuda() for a, b in ((1.0, 0.5), (-4.0, -0.5), (0.6, -2.3)))
        self.inputs, self.states = torch.zeros(slots, TAPS - 1, C, dtype=BF, device="cuda"), torch.zeros(slots, HEADS, DK, DV, device="cuda")
        make = lambda n, dtype=BF: torch.zeros(most, n, dtype=dtype, device="cuda")  # noqa: E731
        self.h, self.x, self.z, self.mixed, self.o, self.n, self.y = make(HIDDEN, torch.float32), make(HIDDEN), make(WIDE), make(C), make(VALUES), make(VALUES), make(HIDDEN)

    def bind(self, batch, T, slots=None, to=None, workspace=None):
        """What one shape of step keeps: the structs and the workspace. ``to``: where states go, {inputs, states}, instead of where they come from."""
        inputs, states = to or (self.inputs, self.states)
        at = None if slots is None else slots.data_ptr()
        if workspace is None:
            need = int(self.hip.size("linear_attention_workspace_bytes", pointer(batch), T, HEADS, K_HEADS, DK, DV))
            workspace = torch.full((max(256, need),), 0xFF, dtype=torch.uint8, device="cuda")
        return {"batch": batch, "conv": LxStates(self.inputs.data_ptr(), inputs.data_ptr(), at, self.slots), "workspace": workspace,
                "mix": LxStates(self.states.data_ptr(), states.data_ptr(), at, self.slots), "held": (slots, to),
                "decay": LxDecay(DECAY_STEP, self.z.data_ptr() + 2 * STEP, BF16, WIDE, self.rate.data_ptr(), self.bias.data_ptr())}

    def product(self, x, w, k, y, n, T, stream):
        lib = self.hip.lib
        head, tail = (x.data_ptr(), BF16, k, pointer(w)), (None, F32, y.data_ptr(), BF16, n, T, n, k, 1.0, 0.0)
        if self.skinny:  # whose bits do not depend on the rows beside
            return lib.lx_gemm_skinny(*head, *tail, stream)
        return lib.lx_gemv_w(*head, *tail, stream) if T <= 8 else lib.lx_gemm_w(*head, MATH_BF16, *tail, None, stream)

    def step(self, bound, T, stream, after=None):
        """``after``: called with each operator's number, once it has been issued."""
        lib, at = self.hip.lib, lambda t: t.data_ptr()
        batch = pointer(bound["batch"])
        keys, queries = at(self.mixed) + 2 * VALUES, at(self.mixed) + 2 * (VALUES + KEYS)
        calls = [
            lambda: lib.lx_block_norm(NORM_RMS, None, BF16, 0, None, None, None, 0, 1.0, 1.0, at(self.h), None, F32, HIDDEN, at(self.norms[0]), None, BF16, at(self.x), BF16,
                                      HIDDEN, 1e-5, T, HIDDEN, stream),
            lambda: self.product(self.x, self.structs[0], HIDDEN, self.z, WIDE, T, stream),
            lambda: lib.lx_causal_conv(at(self.z) + 2 * VALUES, BF16, WIDE, at(self.taps), at(self.tap_bias), BF16, TAPS, ACT_SILU, batch, pointer(bound["conv"]),
                                       at(self.mixed), BF16, C, T, C, stream),
            lambda: lib.lx_rotate(keys, BF16, C, keys, BF16, C, batch, None, at(self.freq), 1.0, ROT, 0, T, 2 * K_HEADS, DK, stream),
            lambda: lib.lx_linear_attention(queries, keys, at(self.mixed), BF16, C, C, C, pointer(bound["decay"]), at(self.skip), at(self.z), BF16, WIDE, batch,
                                            pointer(bound["mix"]), at(self.o), BF16, VALUES, T, HEADS, K_HEADS, DK, DV, DK**-0.5, at(bound["workspace"]), stream),
            lambda: lib.lx_block_norm(NORM_RMS, None, BF16, 0, None, None, None, 0, 1.0, 1.0, at(self.o), None, BF16, VALUES, at(self.norms[1]), None, BF16, at(self.n), BF16,
                                      VALUES, 1e-5, T, VALUES, stream),
            lambda: self.product(self.n, self.structs[1], VALUES, self.y, HIDDEN, T, stream),
            lambda: lib.lx_block_norm(NORM_RMS, at(self.y), BF16, HIDDEN, at(self.norms[2]), None, None, 0, 0.5, 1.0, at(self.h), at(self.h), F32, HIDDEN, at(self.norms[3]), None,
                                      BF16, at(self.x), BF16, HIDDEN, 1e-5, T, HIDDEN, stream),
        ]
        for i, call in enumerate(calls):
            assert call() == 0, i
            if after:
                after(i)


def on_device(rows):
    return Rows(rows.counts, rows.lengths, rows.slots, rows.T, rows.max_rows, rows.seqs, "cuda")


def near(got, want, size, share, rows=slice(None)):
    got, rounding = got.double().cpu()[rows], HALF[got.dtype]
    bound = share * size + rounding * 1.01 * (want.abs() + share * size) + 1e-30
    error = (got - want).abs()
    assert bool((error <= bound).all()), f"worst {(error / bound).max().item():.3g} of its bound"


def normed(x, weight):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double().cpu()


class Checked:
    """Issues a step and checks each operator's output against what stood in its inputs."""

    def __init__(self, layer, rows, bound):
        self.layer, self.rows, self.T = layer, rows, rows.T
        self.inputs, self.states, self.h = layer.inputs.cpu(), layer.states.cpu(), layer.h[:self.T].cpu()
        self.positions = torch.zeros(self.T, dtype=torch.int64)
        self.known = torch.zeros(self.T, dtype=torch.bool)
        for _, begin, end, position, _, _ in rows.spans():
            self.positions[begin:end] = torch.arange(position, position + end - begin)
            self.known[begin:end] = True
        layer.step(bound, self.T, torch.cuda.current_stream().cuda_stream, self.after)

    def after(self, i):
        torch.cuda.synchronize()
        L, T, known = self.layer, self.T, self.known
        if i in (0, 5):
            source, weight, got = (self.h, L.norms[0], L.x) if i == 0 else (L.o[:T].cpu(), L.norms[1], L.n)
            want = normed(source, weight)
            near(got[:T], want, want.abs(), 2.0**-20)
        elif i in (1, 6):
            x, w, got = (L.x, L.in_w, L.z) if i == 1 else (L.n, L.out_w, L.y)
            x, w = x[:T].double().cpu(), w.to("cpu").dense().double()
            near(got[:T], x @ w.T, x.abs() @ w.abs().T, 2.0**-15)
        elif i == 2:
            x = L.z[:T, VALUES:STEP].cpu()
            want, size, kept = convolved(x, L.taps.cpu(), L.tap_bias.cpu(), True, self.rows, self.inputs, L.slots)
            near(L.mixed[:T], want[known], 1.1 * (TAPS + 1) * 2.0**-24 * size[known] + 2.0**-21 * want[known].abs(), 1.0, known)
            for slot in range(L.slots):
                assert torch.equal(L.inputs[slot].double().cpu(), kept.get(slot, self.inputs[slot].double()))
            self.before = L.mixed[:T].cpu()
        elif i == 3:
            want, size = rotated(self.before[:, VALUES:], self.positions, L.freq.cpu(), 1.0, ROT, False, 2 * K_HEADS, DK)
            near(L.mixed[:T, VALUES:], want[known], size[known], 2.0**-21, known)
            assert torch.equal(L.mixed[:T, :VALUES].cpu(), self.before[:, :VALUES])
        elif i == 4:
            m = Mixer(self.rows, HEADS, K_HEADS, DK, DV, "step", True, BF, step=BF)
            mixed, z = L.mixed[:T].cpu(), L.z[:T].cpu()
            m.v, m.k, m.q, m.gate, m.x = mixed[:, :VALUES], mixed[:, VALUES:VALUES + KEYS], mixed[:, VALUES + KEYS:], z[:, :VALUES], z[:, STEP:STEP + HEADS]
            m.skip, m.rate, m.bias, m.state, m.count = L.skip.cpu(), L.rate.cpu(), L.bias.cpu(), self.states, L.slots
            want = m.want()
            out = L.o[:T].clone()
            assert bool((out[~known.cuda()] == 1.0).all())
            out[~known.cuda()] = UNTOUCHED
            m.check(out, L.states, want, 2.0**-14)
        else:
            y = normed(L.y[:T].cpu(), L.norms[2])
            want = self.h.double() + 0.5 * y
            near(L.h[:T], want, self.h.double().abs() + y.abs(), 2.0**-20)
            x = normed(want, L.norms[3])
            near(L.x[:T], x, (self.h.double().abs() + y.abs()) / want.abs() * x.abs() + x.abs(), 2.0**-19)


def test_prompts_in_pieces_then_decode(hip):
    layer = Layer(hip, 450, 5)
    layer.inputs.fill_(3.0), layer.states.fill_(2.0)  # of sequences that were there before: not looked at
    g, held, slots = torch.Generator().manual_seed(5), [0, 0, 0], [4, 0, 2]
    # Pieces of the prompts (of one part and of several), a token each, drafted tokens, a padded call.
    for counts, T in (([300, 23, 0], 323), ([30, 0, 141], 175), ([1, 1, 1], 3), ([3, 1, 2], 8), ([18, 0, 40], 64)):
        held = [a + b for a, b in zip(held, counts)]
        rows = Rows(counts, held, slots, T)
        device = on_device(rows)
        layer.h[:T].copy_(torch.randn(T, HIDDEN, generator=g))
        layer.o.fill_(1.0)
        Checked(layer, rows, layer.bind(device.lx(), T, device.slots_t))


@pytest.mark.parametrize("most,steps", [
    (1, [([1, 1, 1], [30, 1, 900], [4, 0, 2]), ([1, 0, 1], [31, 1, 901], [4, 0, 2]), ([1, 1, 1], [1, 2, 5], [1, 0, 3]), ([0, 0, 0], [3, 4, 5], [0, 1, 2])]),
    (400, [([400, 40, 1], [400, 40, 9], [4, 0, 2]), ([1, 1, 1], [401, 41, 10], [4, 0, 2]), ([3, 400, 0], [404, 441, 10], [4, 0, 2]), ([129, 130, 128], [129, 999, 128], [0, 1, 3]),
           ([0, 0, 0], [1, 1, 1], [0, 1, 2])])])
def test_steps_in_a_graph(hip, most, steps):
    """One captured step, replayed as sequences come, grow and change slots, with eager work in between: every replay gives the bits of the same step
    issued eagerly, in the residual rows, the next input and the states."""
    T = 3 * most if most == 1 else 450
    layers = [Layer(hip, T, 5, seed=1) for _ in range(2)]
    g = torch.Generator().manual_seed(2)
    rows = torch.zeros(4, dtype=torch.int32, device="cuda")
    lengths, slots = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    batch = LxKv8Batch(3, rows.data_ptr(), lengths.data_ptr(), None, 0, most, 0)
    bound = [layer.bind(batch, T, slots) for layer in layers]
    stream, graph, lib = ctypes.c_void_p(), ctypes.c_void_p(), hip.lib
    assert lib.lx_rt_stream_create(ctypes.byref(stream)) == 0
    try:
        torch.cuda.synchronize()
        layers[0].step(bound[0], T, stream)  # first calls outside the capture; no sequence has a row
        assert lib.lx_rt_stream_sync(stream) == 0
        assert lib.lx_rt_capture_begin(stream) == 0
        layers[0].step(bound[0], T, stream)
        assert lib.lx_rt_capture_end(stream, ctypes.byref(graph)) == 0
        first = torch.randn(layers[0].inputs.shape, generator=g).to(BF), torch.randn(layers[0].states.shape, generator=g)
        for layer in layers:
            layer.inputs.copy_(first[0]), layer.states.copy_(first[1])
        for i, (counts, so_far, of) in enumerate(steps):
            rows.copy_(torch.tensor([0, counts[0], counts[0] + counts[1], sum(counts)], dtype=torch.int32))
            lengths.copy_(torch.tensor(so_far, dtype=torch.int32)), slots.copy_(torch.tensor(of, dtype=torch.int32))
            h = torch.randn(T, HIDDEN, generator=g)
            for layer in layers:
                layer.h.copy_(h), layer.mixed.zero_(), layer.o.zero_()
            torch.cuda.synchronize()
            assert lib.lx_rt_graph_launch(graph, stream) == 0
            assert lib.lx_rt_stream_sync(stream) == 0
            layers[1].step(bound[1], T, torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            for name in ("h", "x", "mixed", "o", "inputs", "states"):
                assert torch.equal(getattr(layers[0], name), getattr(layers[1], name)), f"replay {i}: {name}"
            assert bool(torch.isfinite(layers[0].h).all())
    finally:
        if graph:
            lib.lx_rt_graph_destroy(graph)
        lib.lx_rt_stream_destroy(stream)


def test_two_steps_at_once(hip):
    """Two layers' prompts on two streams, workspaces of their own: each as it is alone."""
    rows = Rows([400, 17], [400, 30], [1, 3])
    device, T = on_device(rows), rows.T
    layers = [Layer(hip, T, 5, seed=3 + i) for i in range(2)]
    bound = [layer.bind(device.lx(), T, device.slots_t) for layer in layers]
    hs = [torch.randn(T, HIDDEN, generator=torch.Generator().manual_seed(i)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in layers]

    def run(on):
        for layer, h in zip(layers, hs):
            layer.h.copy_(h), layer.inputs.fill_(0.5), layer.states.fill_(0.25)
        torch.cuda.synchronize()
        for _ in range(3):  # steps one after another on each stream, side by side with the other's
            for layer, b, stream in zip(layers, bound, on):
                layer.step(b, T, stream.cuda_stream)
        torch.cuda.synchronize()
        return [[t.clone() for t in (layer.h, layer.inputs, layer.states)] for layer in layers]

    alone = run([torch.cuda.current_stream()] * 2)
    together = run(streams)
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_drafted_tokens_are_committed_as_far_as_accepted(hip):
    """Five drafted tokens run with their states put elsewhere leave the sequences' own alone; the accepted ones, run again onto those, leave
    what token by token leaves."""
    layer, slots = Layer(hip, 10, 3, skinny=True), [2, 0]
    g = torch.Generator().manual_seed(8)
    layer.inputs.copy_(torch.randn(layer.inputs.shape, generator=g)), layer.states.copy_(torch.randn(layer.states.shape, generator=g))
    before = layer.inputs.clone(), layer.states.clone()
    apart = torch.full_like(layer.inputs, 7.0), torch.full_like(layer.states, 7.0)
    drafted = torch.randn(10, HIDDEN, generator=g)
    stream = torch.cuda.current_stream().cuda_stream

    def step(counts, lengths, h, to=None):
        rows = Rows(counts, lengths, slots)
        device = on_device(rows)
        layer.h[:rows.T].copy_(h)
        layer.step(layer.bind(device.lx(), rows.T, device.slots_t, to), rows.T, stream)
        torch.cuda.synchronize()

    step([5, 5], [25, 13], drafted, apart)
    assert torch.equal(layer.inputs, before[0]) and torch.equal(layer.states, before[1])
    assert bool((apart[1][1] == 7.0).all()) and not bool((apart[1][0] == 7.0).any())
    step([2, 4], [22, 12], torch.cat([drafted[:2], drafted[5:9]]))
    accepted = layer.inputs.clone(), layer.states.clone()
    layer.inputs.copy_(before[0]), layer.states.copy_(before[1])
    for i in range(4):
        counts = [1 if i < 2 else 0, 1]
        step(counts, [20 + min(i + 1, 2), 8 + i + 1], torch.cat([drafted[i:i + counts[0]], drafted[5 + i:6 + i]]))
    assert torch.equal(layer.inputs, accepted[0]) and torch.equal(layer.states, accepted[1])
    assert torch.equal(layer.states[1], before[1][1])

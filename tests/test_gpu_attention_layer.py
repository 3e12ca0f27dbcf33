"""The operators of an attention layer together, as a program uses them, through the C ABI: lx_block_norm, the QKV product
(lx_gemm_w / lx_gemv_w), lx_kv8_append, lx_kv8_attention, the output product and lx_block_norm again. A prompt in two pieces, then
decode steps captured once in a graph and replayed while lengths and inputs change on the device."""

import ctypes

import pytest
import torch

from conftest import rel_l2
from dromos_amd.abi import BF16, F32, MATH_BF16, NORM_RMS, W_FP8
from dromos_amd.formats import master_weight, quantize_with
from kv8 import Batch, Cache, attended, rotated

pytestmark = pytest.mark.gpu

Q_HEADS, HEADS, DIM, HIDDEN, PAGE, BLOCK = 8, 2, 64, 512, 32, 16
WIDTH, KV = Q_HEADS * DIM, HEADS * DIM


class Layer:
    """Weights and buffers for up to `most` rows; step() issues one pass over rows of a batch on a stream."""

    def __init__(self, hip, fmt, batch, most, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.hip, self.batch, self.most = hip, batch, most
        self.qkv_w = quantize_with(hip, master_weight(WIDTH + 2 * KV, HIDDEN, g).cuda(), W_FP8)
        self.out_w = quantize_with(hip, master_weight(HIDDEN, WIDTH, g).cuda(), W_FP8)
        self.norms = [(torch.randn(HIDDEN, generator=g) * 0.1 + 1).to(torch.bfloat16).cuda() for _ in range(3)]
        self.freq = torch.tensor([1e4 ** (-2 * i / DIM) for i in range(DIM // 2)], dtype=torch.float32).cuda()
        self.cache = Cache(fmt, batch.pages, HEADS, PAGE, BLOCK, DIM, "cuda")
        self.h = torch.zeros(most, HIDDEN, device="cuda")
        make = lambda n: torch.zeros(most, n, dtype=torch.bfloat16, device="cuda")
        self.x, self.qkv, self.q, self.o, self.y = make(HIDDEN), make(WIDTH + 2 * KV), make(WIDTH), make(WIDTH), make(HIDDEN)
        self.structs = self.qkv_w.lx(), self.out_w.lx()

    def product(self, x, w, k, y, n, T, stream):
        lib, weight = self.hip.lib, ctypes.pointer(w)
        head = (x.data_ptr(), BF16, k, weight)
        tail = (None, F32, y.data_ptr(), BF16, n, T, n, k, 1.0, 0.0)
        return lib.lx_gemv_w(*head, *tail, stream) if T <= 8 else lib.lx_gemm_w(*head, MATH_BF16, *tail, None, stream)

    def bind(self, on, T):
        """What one shape of step keeps: the structs and the workspace."""
        b, c = on.lx(), self.cache.lx()
        n = self.hip.size("kv8_attention_workspace_bytes", ctypes.pointer(c), ctypes.pointer(b), T, Q_HEADS)
        return b, c, torch.full((max(256, int(n)),), 0xFF, dtype=torch.uint8, device="cuda"), on

    def step(self, bound, T, stream, window=0):
        lib = self.hip.lib
        b, c, workspace, _ = bound
        b, c = ctypes.pointer(b), ctypes.pointer(c)
        at = lambda t: t.data_ptr()
        ld = WIDTH + 2 * KV
        qkv = at(self.qkv)
        status = [
            lib.lx_block_norm(NORM_RMS, None, BF16, 0, None, None, None, 0, 1.0, 1.0, at(self.h), None, F32, HIDDEN, at(self.norms[0]), None, BF16, at(self.x), BF16, HIDDEN,
                              1e-5, T, HIDDEN, stream),
            self.product(self.x, self.structs[0], HIDDEN, self.qkv, ld, T, stream),
            lib.lx_kv8_append(c, b, qkv, qkv + 2 * WIDTH, qkv + 2 * (WIDTH + KV), BF16, ld, ld, ld, at(self.q), BF16, WIDTH, at(self.freq), DIM, 0, T, Q_HEADS, stream),
            lib.lx_kv8_attention(at(self.q), BF16, WIDTH, c, b, at(self.o), BF16, WIDTH, T, Q_HEADS, DIM**-0.5, window, at(workspace), stream),
            self.product(self.o, self.structs[1], WIDTH, self.y, HIDDEN, T, stream),
            lib.lx_block_norm(NORM_RMS, at(self.y), BF16, HIDDEN, at(self.norms[1]), None, None, 0, 0.5, 1.0, at(self.h), at(self.h), F32, HIDDEN, at(self.norms[2]), None, BF16,
                              at(self.x), BF16, HIDDEN, 1e-5, T, HIDDEN, stream),
        ]
        assert status == [0] * 6, status


def batch_of(rows, lengths, table, pages):
    b = Batch(rows, lengths, PAGE)
    b.table, b.pages = table, pages
    return b


def rms(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()


def reference(layer, h, batch):
    """The same step in 64 bits from the residual rows h, on the cache as the step left it; rounded where the step's buffers
    round."""
    bf = lambda t: t.to(torch.bfloat16).double()
    qkv_w, out_w = (w.to("cpu").dense().double() for w in (layer.qkv_w, layer.out_w))
    x = bf(rms(h.double(), layer.norms[0].cpu()))
    qkv = bf(x @ qkv_w.T)
    positions = torch.tensor([p for _, _, p, _, _ in batch.places()])
    q = bf(rotated(qkv[:, :WIDTH].reshape(-1, Q_HEADS, DIM), positions, layer.freq.cpu(), DIM, False).flatten(1))
    keys = rotated(qkv[:, WIDTH:WIDTH + KV].reshape(-1, HEADS, DIM), positions, layer.freq.cpu(), DIM, False)
    cache = layer.cache.to("cpu")
    out, _, _ = attended(q, cache, batch, Q_HEADS, DIM**-0.5)
    y = bf(bf(out.flatten(1)) @ out_w.T)
    new = h.double() + 0.5 * rms(y, layer.norms[1].cpu())
    return new, rms(new, layer.norms[2].cpu()), keys, cache


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_prompt_in_pieces_then_decode(hip, fmt):
    lengths = [70, 23, 41]
    whole = Batch([0, 0, 0], [n + 16 for n in lengths], PAGE, seed=3)
    layer = Layer(hip, fmt, whole, 160)
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(5)
    held = [0, 0, 0]
    for rows in ([40, 23, 0], [30, 0, 41], [1, 1, 1], [3, 1, 2]):  # two pieces of the prompts, a token each, drafted tokens
        held = [a + b for a, b in zip(held, rows)]
        batch = batch_of(rows, held, whole.table, whole.pages)
        T = sum(rows)
        h = torch.randn(T, HIDDEN, generator=g)
        layer.h[:T].copy_(h)
        layer.step(layer.bind(batch.to("cuda"), T), T, stream)
        torch.cuda.synchronize()
        want_h, want_x, keys, cache = reference(layer, h, batch)
        assert rel_l2(layer.h[:T], want_h) <= 1e-2 and rel_l2(layer.x[:T], want_x) <= 1e-2
        # The cache holds this step's keys, to within its steps (int8: half of 1/127 of a block's largest; e4m3: 2^-4 of a value).
        values = cache.values()[0]
        for row, _, _, page, place in batch.places():
            got, exact = values[page, :, place], keys[row]
            assert rel_l2(got, exact) <= (0.03 if fmt == "int8" else 0.05), (row, rel_l2(got, exact))


def test_decode_steps_in_a_graph(hip):
    """One captured step, replayed as the sequences grow (over the edges of blocks and pages), with eager work in between: every
    replay gives the bits of the same step issued eagerly, in the residual rows, the next input and the cache."""
    seqs, start, steps = 5, [30, 1, 63, 95, 14], 6
    whole = Batch([1] * seqs, [n + steps for n in start], PAGE, seed=9, max_length=200)
    layers = [Layer(hip, "fp8", whole, seqs, seed=1) for _ in range(2)]
    lib = hip.lib
    stream = ctypes.c_void_p()
    assert lib.lx_rt_stream_create(ctypes.byref(stream)) == 0
    graph = ctypes.c_void_p()
    try:
        on = whole.to("cuda")
        on.lengths = torch.tensor(start, dtype=torch.int32, device="cuda")
        for layer in layers:
            layer.cache = Cache("fp8", whole.pages, HEADS, PAGE, BLOCK, DIM).fill(4).to("cuda")
        bound = [layer.bind(on, seqs) for layer in layers]
        torch.cuda.synchronize()
        layers[0].step(bound[0], seqs, stream)  # first calls outside the capture
        assert lib.lx_rt_stream_sync(stream) == 0
        layers[0].cache.codes.copy_(layers[1].cache.codes)
        layers[0].cache.scales.copy_(layers[1].cache.scales)
        torch.cuda.synchronize()
        assert lib.lx_rt_capture_begin(stream) == 0
        layers[0].step(bound[0], seqs, stream)
        assert lib.lx_rt_capture_end(stream, ctypes.byref(graph)) == 0
        g = torch.Generator().manual_seed(6)
        for i in range(steps):
            on.lengths += 1
            h = torch.randn(seqs, HIDDEN, generator=g)
            for layer in layers:
                layer.h.copy_(h)
            torch.cuda.synchronize()
            assert lib.lx_rt_graph_launch(graph, stream) == 0
            assert lib.lx_rt_stream_sync(stream) == 0
            layers[1].step(bound[1], seqs, torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            a, b = layers
            assert torch.equal(a.h, b.h) and torch.equal(a.x, b.x), f"step {i}"
            assert torch.equal(a.cache.codes, b.cache.codes) and torch.equal(a.cache.scales, b.cache.scales), f"step {i}"
    finally:
        if graph:
            lib.lx_rt_graph_destroy(graph)
        lib.lx_rt_stream_destroy(stream)


def test_parts_of_long_sequences_in_a_graph(hip):
    """A captured attention call whose sequences come in parts (partial sums in the workspace), replayed on other lengths: those
    that need one part, several or none."""
    whole = Batch([1, 1, 1], [5000, 5000, 5000], 64, seed=2)
    cache = Cache("int8", whole.pages, 1, 64, 32, 128).fill(3)
    held, on = cache.to("cuda"), whole.to("cuda")
    on.lengths = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4 * 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    out, again = (torch.zeros(3, 4 * 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c, b = held.lx(), on.lx()
    c, b = ctypes.pointer(c), ctypes.pointer(b)
    n = int(hip.size("kv8_attention_workspace_bytes", c, b, 3, 4))
    assert n > 0
    spaces = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.lib.lx_rt_stream_create(ctypes.byref(stream)) == 0
    try:
        torch.cuda.synchronize()
        call = lambda to, space, s: hip.lib.lx_kv8_attention(q.data_ptr(), BF16, 512, c, b, to.data_ptr(), BF16, 512, 3, 4, 0.09, 0, space.data_ptr(), s)
        assert call(out, spaces[0], stream) == 0
        assert hip.lib.lx_rt_stream_sync(stream) == 0
        assert hip.lib.lx_rt_capture_begin(stream) == 0
        assert call(out, spaces[0], stream) == 0
        assert hip.lib.lx_rt_capture_end(stream, ctypes.byref(graph)) == 0
        for lengths in ([5000, 1, 0], [0, 700, 4999], [256, 257, 3000], [5000, 5000, 5000]):
            on.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
            torch.cuda.synchronize()
            assert hip.lib.lx_rt_graph_launch(graph, stream) == 0
            assert hip.lib.lx_rt_stream_sync(stream) == 0
            assert call(again, spaces[1], torch.cuda.current_stream().cuda_stream) == 0
            torch.cuda.synchronize()
            assert torch.equal(out.view(torch.int16), again.view(torch.int16)), lengths
            for row, length in enumerate(lengths):
                assert bool((out[row] == 0).all()) == (length == 0)
    finally:
        if graph:
            hip.lib.lx_rt_graph_destroy(graph)
        hip.lib.lx_rt_stream_destroy(stream)


def test_two_streams_at_once(hip):
    """Two calls in flight at the same time, each with its own workspace, on one cache that both read."""
    batch = Batch([1] * 6, [3000, 17, 2500, 4096, 1, 900], 64, seed=1)
    cache = Cache("fp8", batch.pages, 2, 64, 32, 128).fill(2).to("cuda")
    on = batch.to("cuda")
    g = torch.Generator().manual_seed(3)
    qs = [torch.randn(6, 1024, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    outs = [[torch.zeros(6, 1024, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2)]
    c, b = cache.lx(), on.lx()
    c, b = ctypes.pointer(c), ctypes.pointer(b)
    n = max(256, int(hip.size("kv8_attention_workspace_bytes", c, b, 6, 8)))
    spaces = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    call = lambda i, to, s: hip.lib.lx_kv8_attention(qs[i].data_ptr(), BF16, 1024, c, b, to.data_ptr(), BF16, 1024, 6, 8, 0.09, 0, spaces[i].data_ptr(), s)
    torch.cuda.synchronize()
    for i in range(2):
        assert call(i, outs[0][i], torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for i in range(2):
            assert call(i, outs[1][i], streams[i].cuda_stream) == 0
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[0][i].view(torch.int16), outs[1][i].view(torch.int16))

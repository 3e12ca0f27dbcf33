"""Prompts' appends and attention (tiles of many rows, parts and their sums) captured into a graph and replayed on other rows,
lengths and inputs, with eager calls and synchronisations between."""

import ctypes

import pytest
import torch

from dromos_amd.abi import BF16
from kv8 import Batch, Cache, append, attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,group", [(64, 1, 2), (128, 2, 1), (256, 1, 2)])
def test_prompt_steps_in_a_graph(hip, dim, heads, group):
    most, longest, width, kv = 150, 3000, heads * group * dim, heads * dim
    T = 2 * most
    whole = Batch([most, most], [longest, longest], 64, seed=4)
    on = whole.to("cuda")
    caches = [Cache("fp8", whole.pages, heads, 64, 32, dim).fill(7).to("cuda") for _ in range(2)]
    qkv = torch.zeros(T, width + 2 * kv, dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv[:, :width], qkv[:, width:width + kv], qkv[:, width + kv:]
    freq = torch.tensor([1e4 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32, device="cuda")
    turned, out = (torch.zeros(T, width, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c, b = caches[0].lx(), on.lx()
    c, b = ctypes.pointer(c), ctypes.pointer(b)
    need = int(hip.size("kv8_attention_workspace_bytes", c, b, T, heads * group))
    assert need > 0
    space = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    at, ld = lambda t: t.data_ptr(), qkv.stride(0)

    def issue(stream):
        assert hip.lib.lx_kv8_append(c, b, at(q), at(k), at(v), BF16, ld, ld, ld, at(turned), BF16, width, at(freq), dim, 0, T, heads * group, stream) == 0
        assert hip.lib.lx_kv8_attention(at(turned), BF16, width, c, b, at(out), BF16, width, T, heads * group, dim**-0.5, 0, at(space), stream) == 0

    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.lib.lx_rt_stream_create(ctypes.byref(stream)) == 0
    try:
        torch.cuda.synchronize()
        assert hip.lib.lx_rt_capture_begin(stream) == 0
        issue(stream)
        assert hip.lib.lx_rt_capture_end(stream, ctypes.byref(graph)) == 0
        for i, (rows, lengths) in enumerate([([150, 150], [3000, 3000]), ([20, 0], [20, 9]), ([150, 97], [150, 2999]), ([0, 0], [5, 6]), ([1, 149], [1, 1000]), ([150, 150], [2000, 700])]):
            on.first.copy_(torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32))
            on.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
            qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)))
            turned.zero_()
            out.fill_(7.0)
            torch.cuda.synchronize()
            assert hip.lib.lx_rt_graph_launch(graph, stream) == 0
            assert hip.lib.lx_rt_stream_sync(stream) == 0
            want_turned, want = torch.zeros_like(turned), torch.full_like(out, 7.0)
            append(hip, caches[1], on, q, k, v, freq, dim, q_out=want_turned, q_heads=heads * group, T=T)
            attention(hip, want_turned, caches[1], on, heads * group, dim**-0.5, out=want, T=T)
            torch.cuda.synchronize()
            assert torch.equal(turned, want_turned), f"replay {i}"
            assert torch.equal(out.view(torch.int16), want.view(torch.int16)), f"replay {i}"
            assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales), f"replay {i}"
            assert bool((out[sum(rows):] == 7.0).all())
    finally:
        if graph:
            hip.lib.lx_rt_graph_destroy(graph)
        hip.lib.lx_rt_stream_destroy(stream)


def test_columns_of_one_tensor_by_name(hip):
    """q, k and v as columns of one product's rows, handed over with their row stride."""
    dim, heads, group, T = 64, 2, 2, 40
    batch = Batch([T], [T], 64)
    on, caches = batch.to("cuda"), [Cache("int8", batch.pages, heads, 64, 32, dim, "cuda") for _ in range(2)]
    width, kv = heads * group * dim, heads * dim
    qkv = torch.randn(T, width + 2 * kv, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    q, k, v = qkv[:, :width], qkv[:, width:width + kv], qkv[:, width + kv:]
    freq = torch.tensor([1e4 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32, device="cuda")
    want = append(hip, caches[0], on, q, k, v, freq, dim, q_heads=heads * group)
    got, ld = torch.empty_like(want), qkv.stride(0)
    c, b = caches[1].lx(), on.lx()
    hip("kv8_append", ctypes.pointer(c), ctypes.pointer(b), q, k, v, BF16, ld, ld, ld, got, BF16, width, freq, dim, 0, T, heads * group)
    assert torch.equal(got, want) and torch.equal(caches[0].codes, caches[1].codes)

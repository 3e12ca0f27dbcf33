"""lx_block_norm on the GPU, through the C ABI, against the same in 64 bits."""

import itertools

import pytest
import torch

from dromos_amd.abi import BF16, DTYPE, F32, NORM_LAYER, NORM_RMS

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


def randn(seed, *shape, dtype=H, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype)


def exact_norm(v, layer, w, b, eps):
    """The norm in 64 bits, and what an f32 sum's error (2^-18 relatively: at most 32 values a lane one after another, then a
    tree and sixteen wavefronts) makes of it: the mean off by that of the mean magnitude, the factor by that of itself."""
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros((), dtype=torch.float64)
    f = 1.0 / ((v - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    out = (v - mean) * f * w.double()
    off = out.abs() * 2.0**-17 + (v.abs().mean(-1, keepdim=True) * 2.0**-18 + v.abs() * 2.0**-23 if layer else 0.0) * f * w.double().abs()
    if b is not None:
        out = out + b.double()
        off = off + out.abs() * 2.0**-23
    return out, off, f


def call(hip, layer, y, post, post_b, gate, alpha, beta, h, w, b, x_dtype, eps, h_out=None, x=None, ld_gate=None):
    src = h if y is None else y
    T, width = src.shape
    h_dtype = h.dtype if h is not None else H
    if h_out is None and y is not None:
        h_out = torch.full((T, width), float("nan"), dtype=h_dtype, device="cuda")
    if x is None and w is not None:
        x = torch.full((T, width), float("nan"), dtype=x_dtype, device="cuda")
    at = lambda t: None if t is None else t.data_ptr()
    ld = lambda t: 0 if t is None else t.stride(0)
    weights = [t for t in (post, post_b, w, b) if t is not None]
    hip("block_norm", NORM_LAYER if layer else NORM_RMS, at(y), DTYPE[y.dtype] if y is not None else F32, ld(y), at(post), at(post_b), at(gate),
        (0 if gate is None or gate.shape[0] == 1 else gate.stride(0)) if ld_gate is None else ld_gate, alpha, beta, at(h), at(h_out), DTYPE[h_dtype],
        ld(h if h is not None else h_out), at(w), at(b), DTYPE[weights[0].dtype] if weights else BF16, at(x), DTYPE[x_dtype], ld(x), eps, T, width)
    return h_out, x


def check(hip, layer, y, post, post_b, gate, alpha, beta, h, w, b, x_dtype=H, eps=1e-5, **kw):
    cuda = lambda t: None if t is None else t.cuda()
    h_out, x = call(hip, layer, *(cuda(t) for t in (y, post, post_b, gate)), alpha, beta, cuda(h), cuda(w), cuda(b), x_dtype, eps, **kw)
    if y is None:
        s, off = h.double(), torch.zeros(1, dtype=torch.float64)
    else:
        r, off = y.double(), torch.zeros(1, dtype=torch.float64)
        if post is not None:
            r, off, _ = exact_norm(r, layer, post, post_b, eps)
        g = alpha * (1.0 if gate is None else gate.double())
        s, off = g * r, abs(g) * off
        off = off + s.abs() * 2.0**-22  # alpha, gate: a rounding each
        if beta:
            s = beta * h.double() + s
            off = off + (s.abs() + abs(beta) * h.double().abs()) * 2.0**-23
        half = torch.finfo(h_out.dtype).eps / 2
        err = (h_out.double().cpu() - s).abs()
        assert bool((err <= off * (1 + half) + half * s.abs()).all()), f"h off by {err.max():.3e}"
    if w is not None:
        want, by_norm, f = exact_norm(s, layer, w, b, eps)
        # What the sum's own error makes: its value's, and (through mean and factor) the row's largest.
        most = off.expand_as(s).amax(-1, keepdim=True)
        bound = by_norm + (off + most) * f * w.double().abs() + most * f * (want if b is None else want - b.double()).abs()
        half = torch.finfo(x_dtype).eps / 2
        err = (x.double().cpu() - want).abs()
        assert bool((err <= bound * (1 + half) + half * want.abs()).all()), f"x off by {err.max():.3e}"
    return h_out, x


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("width", [1, 7, 64, 256, 500, 511, 512, 520, 1000, 2048, 2056, 4096, 4100, 5120, 8192, 8200, 8191, 12288, 16384, 16392, 32768, 32767])
def test_widths(hip, layer, width):
    y, h = randn(1, 3, width, std=2.0, mean=0.3), randn(2, 3, width, std=3.0)
    check(hip, layer, y, randn(3, width, std=0.1, mean=1.0), None, None, 0.7, 1.0, h, randn(4, width, std=0.1, mean=1.0), None)


@pytest.mark.parametrize("y_dtype,h_dtype,x_dtype,w_dtype", itertools.product([F, H], repeat=4))
def test_types(hip, y_dtype, h_dtype, x_dtype, w_dtype):
    for width in (1024, 1025):
        check(hip, False, randn(1, 5, width, dtype=y_dtype), randn(2, width, dtype=w_dtype), randn(3, width, dtype=w_dtype), randn(4, 5, width, dtype=y_dtype), 1.3, 0.8,
              randn(5, 5, width, dtype=h_dtype), randn(6, width, dtype=w_dtype), randn(7, width, dtype=w_dtype), x_dtype)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("post,gate,pre,beta", itertools.product([False, True], ["none", "row", "one"], [False, True], [0.0, 1.0, -0.5]))
def test_parts(hip, layer, post, gate, pre, beta):
    width, T = 768, 9
    g = {"none": None, "row": randn(1, T, width), "one": randn(1, 1, width)}[gate]
    h_out, x = check(hip, layer, randn(2, T, width), randn(3, width) if post else None, randn(4, width) if post else None, g, 0.9, beta,
                     randn(5, T, width), randn(6, width) if pre else None, randn(7, width) if pre else None)
    assert pre or x is None


@pytest.mark.parametrize("layer", [False, True])
def test_before_the_first_block(hip, layer):
    for width in (640, 641):
        h_out, _ = check(hip, layer, None, None, None, None, 1.0, 1.0, randn(1, 4, width), randn(2, width), None)
        assert h_out is None


def test_no_residual_read(hip):
    """beta 0: h may be missing, or full of NaN."""
    y, w = randn(1, 4, 512), randn(2, 512)
    check(hip, False, y, None, None, None, 2.0, 0.0, None, w, None)
    check(hip, False, y, None, None, None, 2.0, 0.0, torch.full((4, 512), float("nan"), dtype=H), w, None)


@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 0), (0, 3), (0, 8)])
def test_strides_and_in_place(hip, pad, offset):
    T, width = 6, 1000
    def view(seed, dtype):
        flat = torch.zeros(T * (width + pad) + offset, dtype=dtype, device="cuda")[offset:].view(T, width + pad)
        flat.copy_(randn(seed, T, width + pad, dtype=dtype))
        return flat
    y, h, g = view(1, H), view(2, F), view(3, H)
    post, w = randn(4, width).cuda(), randn(5, width).cuda()
    want_h, want_x = call(hip, False, y[:, :width].contiguous(), post, None, g[:, :width].contiguous(), 0.5, 1.0, h[:, :width].contiguous(), w, None, H, 1e-6)
    beside_h, beside_y = h[:, width:].clone(), y[:, width:].clone()
    got_h, got_x = call(hip, False, y[:, :width], post, None, g[:, :width], 0.5, 1.0, h[:, :width], w, None, H, 1e-6, h_out=h[:, :width], x=y[:, :width])
    # Element by element a row is summed in another order: not the same bits, the same numbers.
    assert bool((got_h - want_h).abs().max() <= 2.0**-16 * want_h.abs().max())
    assert bool((got_x.float() - want_x.float()).abs().max() <= 2.0**-7 * want_x.float().abs().max())
    assert torch.equal(h[:, width:], beside_h) and torch.equal(y[:, width:], beside_y)


def test_zero_rows_and_extremes(hip):
    y, h = randn(1, 4, 512, dtype=F), randn(2, 4, 512, dtype=F)
    y[0], h[0] = 0, 0
    y[1] *= 1e-18
    h[2] *= 1e15
    for layer in (False, True):
        check(hip, layer, y, randn(3, 512, dtype=F), None, None, 1.0, 1.0, h, randn(4, 512, dtype=F), None, F)


@pytest.mark.parametrize("width", [2048, 2560, 4096, 4616, 8192])
def test_a_rows_bits_do_not_depend_on_how_many_there_are(hip, width):
    y, h, w = randn(1, 1100, width).cuda(), randn(2, 1100, width, dtype=F).cuda(), randn(3, width).cuda()
    for layer in (False, True):
        all_h, all_x = call(hip, layer, y, w, None, None, 1.0, 1.0, h, w, None, F, 1e-5)
        some_h, some_x = call(hip, layer, y[1000:1009], w, None, None, 1.0, 1.0, h[1000:1009], w, None, F, 1e-5)
        assert torch.equal(some_h, all_h[1000:1009]) and torch.equal(some_x, all_x[1000:1009])


def test_a_rows_bits_do_not_depend_on_the_others(hip):
    y, h = randn(1, 40, 4096).cuda(), randn(2, 40, 4096).cuda()
    w = randn(3, 4096).cuda()
    all_h, all_x = call(hip, True, y, w, None, None, 1.0, 1.0, h, w, None, H, 1e-5)
    for i in (0, 17, 39):
        one_h, one_x = call(hip, True, y[i:i + 1], w, None, None, 1.0, 1.0, h[i:i + 1], w, None, H, 1e-5)
        assert torch.equal(one_h[0], all_h[i]) and torch.equal(one_x[0], all_x[i])


def test_more_rows_than_a_launch_has_threads_for(hip):
    """Heads as rows: 2^26 + 5 rows of eight values, a wavefront each. The rows around the end of the first launch, and the last."""
    T, width = (1 << 26) + 5, 8
    y = torch.ones(T, width, dtype=H, device="cuda")
    edges = [slice(0, 9), slice((1 << 26) - 70, T)]
    for i, at in enumerate(edges):
        y[at] = randn(i, y[at].shape[0], width).cuda()
    w = randn(3, width).cuda()
    _, x = call(hip, False, None, None, None, None, 1.0, 1.0, y, w, None, H, 1e-5)
    for at in edges:
        _, some = call(hip, False, None, None, None, None, 1.0, 1.0, y[at].contiguous(), w, None, H, 1e-5)
        assert torch.equal(x[at], some)
    _, one = call(hip, False, None, None, None, None, 1.0, 1.0, y[1000:1001].contiguous(), w, None, H, 1e-5)
    assert bool((x[9:(1 << 26) - 70] == one).all())

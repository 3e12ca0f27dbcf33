"""The 8-bit paged cache for the tests: caches and batches to hand to the library, and its operators restated in 64 bits,
sequence by sequence and token by token."""

import ctypes
import math

import torch

from dromos_amd.abi import BF16, DTYPE, FORMATS, LxKv8, LxKv8Batch

QMAX = {"int8": 127.0, "fp8": 448.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


class Cache:
    """codes [2, pages, heads, page, dim] as bytes and scales [2, pages, heads, page / block], keys first."""

    def __init__(self, fmt, pages, heads, page, block, dim, device="cpu"):
        self.fmt, self.pages, self.heads, self.page, self.block, self.dim = fmt, pages, heads, page, block, dim
        self.codes = torch.zeros(2, pages, heads, page, dim, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(2, pages, heads, page // block, dtype=torch.float32, device=device)

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        q = QMAX[self.fmt]
        normal = torch.randn(self.codes.shape, generator=g) * (q / 3.5)
        self.codes = normal.round().clamp(-q, q).to(CODES[self.fmt]).view(torch.uint8).to(self.codes.device)
        self.scales = ((torch.rand(self.scales.shape, generator=g) + 0.5) * (2.3 / q)).to(self.scales.device)
        return self

    def to(self, device):
        c = Cache(self.fmt, 1, self.heads, self.page, self.block, self.dim)
        c.pages, c.codes, c.scales = self.pages, self.codes.to(device).clone(), self.scales.to(device).clone()
        return c

    def lx(self):
        return LxKv8(FORMATS[self.fmt], self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(),
                     self.scales[1].data_ptr(), self.pages, self.heads, self.page, self.block, self.dim)

    def raw(self):
        """The codes' numbers in 64 bits."""
        return self.codes.view(CODES[self.fmt]).double() if self.fmt == "int8" else self.codes.view(CODES["fp8"]).float().double()

    def values(self):
        s = self.scales.double().repeat_interleave(self.block, -1)
        return self.raw() * s[..., None]


class Batch:
    """rows: rows of every sequence; lengths: tokens of every sequence; pages are handed out in a shuffled order."""

    def __init__(self, rows, lengths, page, seed=0, spare=2, single=False, max_length=None):
        self.rows_of, self.lengths_of, self.page, self.single = list(rows), list(lengths), page, single
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.pages = max(1, len(order))
        self.table = torch.full((len(need), max(1, max(need, default=1))), 2**31 - 1, dtype=torch.int32)  # unused places hold no page
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.first = torch.tensor([0] + self.rows_of, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.lengths = torch.tensor(self.lengths_of, dtype=torch.int32)
        self.T = int(self.first[-1])
        self.max_rows, self.max_length = max(self.rows_of, default=0), max(self.lengths_of, default=0) if max_length is None else max_length

    def to(self, device):
        b = Batch.__new__(Batch)
        b.__dict__.update(self.__dict__)
        b.table, b.first, b.lengths = self.table.to(device), self.first.to(device), self.lengths.to(device)
        return b

    def lx(self):
        return LxKv8Batch(len(self.rows_of), None if self.single else self.first.data_ptr(), self.lengths.data_ptr(), self.table.data_ptr(),
                          self.table.shape[1], self.max_rows, self.max_length)

    def places(self):
        """[(row, sequence, position, page number, place in the page)] of every row, positions from -something on."""
        out, table = [], self.table.tolist()
        for s, (n, length) in enumerate(zip(self.rows_of, self.lengths_of)):
            for i in range(n):
                p = length - n + i
                out.append((sum(self.rows_of[:s]) + i, s, p, table[s][p // self.page] if p >= 0 else -1, p % self.page))
        return out


# ---- calls ------------------------------------------------------------------------------------------------------------


def append(lx, cache, batch, q, k, v, freq, rot, interleaved=False, q_out=None, q_heads=0, T=None, ld=None, status=False):
    """The views q, k, v may be columns of one wide tensor: rows are stride(0) apart. Returns q_out."""
    if q is not None and q_out is None:
        q_out = torch.full((q.shape[0], q.shape[1]), float("nan"), dtype=torch.bfloat16, device=q.device)
    c, b = cache.lx(), batch.lx()
    at = lambda t: None if t is None else t.data_ptr()
    args = (ctypes.pointer(c), ctypes.pointer(b), at(q), at(k), at(v), DTYPE[k.dtype], 0 if q is None else q.stride(0), k.stride(0),
            v.stride(0), at(q_out), BF16 if q_out is None else DTYPE[q_out.dtype], 0 if q_out is None else q_out.stride(0), at(freq), rot,
            int(interleaved), batch.T if T is None else T, q_heads)
    if status:
        return lx.status("kv8_append", *args)
    lx("kv8_append", *args)
    return q_out


def attention(lx, q, cache, batch, q_heads, scale, window=0, out=None, out_dtype=torch.bfloat16, T=None, workspace=None):
    if out is None:
        out = torch.full((q.shape[0], q_heads * cache.dim), float("nan"), dtype=out_dtype, device=q.device)
    c, b = cache.lx(), batch.lx()
    T = batch.T if T is None else T
    if workspace is None:
        n = int(lx.size("kv8_attention_workspace_bytes", ctypes.pointer(c), ctypes.pointer(b), T, q_heads))
        workspace = torch.full((n + 256,), 0xFF, dtype=torch.uint8, device=q.device)
        tail = n
    else:
        tail = None
    lx("kv8_attention", q.data_ptr(), DTYPE[q.dtype], q.stride(0), ctypes.pointer(c), ctypes.pointer(b), out.data_ptr(), DTYPE[out.dtype],
       out.stride(0), T, q_heads, scale, window, workspace.data_ptr())
    if tail is not None:
        assert bool((workspace[tail:] == 0xFF).all()), "wrote past its workspace"
    return out


# ---- the operators in 64 bits -------------------------------------------------------------------------------------------


def rotated(x, positions, freq, rot, interleaved):
    """x [rows, heads, dim] in 64 bits, turned by positions * freq."""
    x = x.double().clone()
    if rot == 0:
        return x
    angle = positions.double()[:, None, None] * freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    lo, hi = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = lo * c - hi * s, hi * c + lo * s
    return x


def attended(q, cache, batch, q_heads, scale, window=0):
    """(out, sum of weight * |value|, largest sum of |q k| of the row) for every row and query head, in 64 bits: what a
    tolerance is made from. q is rounded to bf16 first."""
    dim, group = cache.dim, q_heads // cache.heads
    values = cache.values()
    q = q.to(torch.bfloat16).double().view(-1, q_heads, dim)
    out, spread, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], q_heads, dtype=torch.float64)
    table = batch.table.tolist()
    for s, (n, length) in enumerate(zip(batch.rows_of, batch.lengths_of)):
        length = min(length, batch.max_length)
        tokens = [(t, table[s][t // cache.page]) for t in range(length)]
        tokens = [(t, p) for t, p in tokens if 0 <= p < cache.pages]
        if not tokens or not n:
            continue
        t = torch.tensor([t for t, _ in tokens])
        p = torch.tensor([p for _, p in tokens])
        k, v = (values[part][p, :, t % cache.page] for part in range(2))  # [tokens, heads, dim]
        r0 = sum(batch.rows_of[:s])
        pos = length - n + torch.arange(n)
        seen = t[None] <= pos[:, None]
        if window:
            seen &= t[None] > pos[:, None] - window
        for h in range(q_heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[r0:r0 + n, h]
            scores = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
            some = seen.any(1)
            w = torch.zeros_like(scores)
            w[some] = torch.softmax(scores[some], -1)
            out[r0:r0 + n, h], spread[r0:r0 + n, h] = w @ vh, w @ vh.abs()
            size[r0:r0 + n, h] = (qh.abs() @ kh.abs().T).masked_fill(~seen, 0.0).amax(1)
    return out, spread, size


def check_attention(got, q, cache, batch, q_heads, scale, window=0, rows=None):
    """The weights are rounded to f16 (half a step, 2^-11 of each, and one under 2^-29 of the row's largest perhaps to nothing); a score is an f32 sum of dim products, off by dim 2^-24
    of the sum of their magnitudes, and its exponential by as much relatively, in the weight and in the sum it is divided by;
    2^-20 covers the exponentials, the scales and the division; the result is rounded once to its type. A weight under 2^-126
    of the row's largest is no f32 number any more (a value of 1.5e-58 cannot come back): 2^17 tokens of such weights and
    values under 2^8 make 2^-101."""
    out, spread, size = attended(q, cache, batch, q_heads, scale, window)
    half = torch.finfo(got.dtype).eps / 2
    off = 2 * abs(scale) * size * cache.dim * 2.0**-24
    lost = max(batch.lengths_of, default=0) * 2.0**-29 * cache.values().abs().max()
    bound = (spread * (2.0**-11 + off[..., None] + 2.0**-20) + lost) * (1 + half) + half * out.abs() + 2.0**-101
    err = (got.double().cpu().view_as(out) - out).abs()
    assert not torch.isnan(err).any(), f"NaN in rows {torch.isnan(err).any(-1).any(-1).nonzero().flatten().tolist()[:8]}"
    worst = (err - bound).flatten().argmax()
    assert bool((err <= bound).all()), (f"off by {err.flatten()[worst]:.3e}, allowed {bound.flatten()[worst]:.3e}, at "
                                        f"{torch.unravel_index(worst, err.shape)}: {out.flatten()[worst]:.6f}")


def check_appended(before, after, batch, k, v, freq, rot, interleaved):
    """What lx_kv8_append wrote, place by place. A rotated value is off by (|a| + |b|) 2^-21 (sine and cosine by 2^-22, three
    roundings); a code is the nearest one to within that and 2^-22 of the block's largest value (the product with the
    inverse). Codes that stay follow from the scales by one f32 division, one product and one rounding: exactly. Everything
    else is as it was."""
    heads, dim, block, qmax = after.heads, after.dim, after.block, QMAX[after.fmt]
    places = [p for p in batch.places() if p[2] >= 0 and 0 <= p[3] < after.pages]
    touched = torch.zeros(after.codes.shape[1:4], dtype=torch.bool)
    scale_touched = torch.zeros(after.scales.shape[1:], dtype=torch.bool)
    raw = after.raw().cpu()
    scales = after.scales.cpu().double()
    was_codes, was_scales = before.codes.cpu(), before.scales.cpu()
    blocks = {}
    for row, s, p, page, place in places:
        blocks.setdefault((page, place // block), []).append((row, p, place % block))
    positions = torch.zeros(k.shape[0])
    for row, s, p, page, place in batch.places():
        positions[row] = p
    new = [rotated(k.cpu().reshape(-1, heads, dim), positions, freq.cpu() if rot else None, rot, interleaved), v.cpu().double().reshape(-1, heads, dim)]
    for part in range(2):
        x = new[part]
        mags = x.abs().where(x.isfinite(), torch.zeros(()).double())
        # what an element's rotation may be off by
        slack = torch.zeros_like(mags)
        if part == 0 and rot:
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
            raw_k = k.cpu().double().reshape(-1, heads, dim).abs().nan_to_num(0.0, 0.0, 0.0)
            both = (raw_k[..., a] + raw_k[..., b]) * 2.0**-21
            slack[..., a], slack[..., b] = both, both
        for (page, at), rows in blocks.items():
            lo = block * at
            first = min(place for _, _, place in rows)
            r = torch.tensor([row for row, _, _ in rows])
            in_page = torch.tensor([lo + place for _, _, place in rows])
            kept = first > 0
            old = was_scales[part, page, :, at].double() if kept else torch.zeros(heads, dtype=torch.float64)
            top = mags[r].amax((0, 2))
            want = torch.maximum(old, top / qmax)
            got = scales[part, page, :, at]
            off = slack[r].amax((0, 2)) / qmax + want * 2.0**-23 + 2.0**-126
            assert bool(((got - want).abs() <= off).all()), f"scale of page {page} block {at}: {got} against {want}"
            assert bool((got >= old).all())
            if not kept:
                assert bool((got[top == 0] == 0).all())
            codes = raw[part, page][:, in_page].permute(1, 0, 2)  # [rows, heads, dim]
            value = x[r]
            numbers = value.isfinite()
            held, limit = codes * got[None, :, None], got[None, :, None] * qmax
            if after.fmt == "int8":
                step = got[None, :, None].expand_as(held) * 0.5
            else:  # half a step of e4m3: 2^-4 of a normal code, 2^-10 below 2^-6
                step = got[None, :, None] * torch.maximum((value / got[None, :, None].clamp_min(1e-300)).abs() * 2.0**-4, torch.tensor(2.0**-10).double())
            err = (held - value.clamp(-limit, limit)).abs()
            bound = step + slack[r] + limit * 2.0**-22
            assert bool((err <= bound)[numbers].all()), f"page {page} block {at}: off by {(err - bound)[numbers].max():.3e}"
            infinite = value.isinf()
            live = (got > 0)[None, :, None].expand_as(infinite)
            assert bool((codes[infinite & live] == qmax * value.sign()[infinite & live]).all())
            nans = value.isnan()
            assert bool((codes[nans] == 0).all())
            touched[page, :, in_page] = True
            scale_touched[page, :, at] = True
            if first:
                front = slice(lo, lo + first)
                now = after.codes.cpu()[part, page, :, front]
                was = was_codes[part, page, :, front]
                grown = (got > old)
                factor = (old.float() / got.float())[:, None, None]
                again = was.view(CODES[after.fmt]).float() * factor
                again = again.round().clamp(-127, 127).to(torch.int8) if after.fmt == "int8" else again.clamp(-448, 448).to(torch.float8_e4m3fn)
                expect = torch.where(grown[:, None, None], again.view(torch.uint8), was)
                same = now == expect
                if after.fmt == "fp8":  # a zero may lose its sign
                    same |= ((now | expect) & 0x7F) == 0
                assert bool(same.all()), f"codes that stay in page {page} block {at}"
                touched[page, :, front] = True
        same = after.codes.cpu()[part] == was_codes[part]
        assert bool(same[~touched].all()), "wrote codes outside its tokens"
        keep = after.scales.cpu()[part].view(torch.int32) == was_scales[part].view(torch.int32)
        assert bool(keep[~scale_touched].all()), "wrote scales outside its blocks"


def check_rotated(got, q, batch, heads, freq, rot, interleaved):
    dim = q.shape[1] // heads
    rows = [(row, p) for row, _, p, _, _ in batch.places() if p >= 0]
    index, positions = torch.tensor([r for r, _ in rows], dtype=torch.long), torch.tensor([p for _, p in rows])
    x = q.cpu().reshape(-1, heads, dim)[index]
    want = rotated(x, positions, freq.cpu() if rot else None, rot, interleaved)
    slack = torch.zeros_like(want)
    if rot:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        both = (x.double()[..., a].abs() + x.double()[..., b].abs()) * 2.0**-21
        slack[..., a], slack[..., b] = both, both
    half = torch.finfo(got.dtype).eps / 2
    err = (got.cpu().double().view(q.shape[0], heads, dim)[index] - want).abs()
    assert bool((err <= slack * (1 + half) + half * want.abs()).all()), f"off by {err.max():.3e}"
    others = sorted(set(range(q.shape[0])) - set(index.tolist()))
    assert bool(got[others].isnan().all()), "wrote rows without a token"

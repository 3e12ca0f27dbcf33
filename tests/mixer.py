"""A linear-attention mixer's operators for the tests: batches to hand to the library, and the operators restated in 64 bits, sequence
by sequence and token by token. Beside a result stands what its error is measured in: the same sum over magnitudes."""

import ctypes
import math

import torch

from dromos_amd import abi
from dromos_amd.abi import BF16, DTYPE, F32, LxDecay, LxKv8Batch, LxStates

KINDS = {"head": abi.DECAY_HEAD, "log": abi.DECAY_LOG, "step": abi.DECAY_STEP}
# Half a step of a rounding, relative to the value.
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
UNTOUCHED = 77.0  # what outputs hold where nothing may be written


class Rows:
    """The rows of a call: ``counts`` of each sequence, tokens so far (``lengths``, None: not given), ``slots`` (None: sequence s has slot s),
    rows of the call (``T``, more than all of them together perhaps) and ``max_rows``. ``counts`` None: one row a sequence, no rows tensor."""

    def __init__(self, counts, lengths=None, slots=None, T=None, max_rows=None, seqs=None, device="cpu"):
        self.plain = counts is None
        self.counts = [1] * seqs if self.plain else list(counts)
        self.seqs = len(self.counts)
        self.first = [0]
        for n in self.counts:
            self.first.append(self.first[-1] + n)
        self.lengths, self.slots = lengths, slots
        self.T = self.first[-1] if T is None else T
        self.max_rows = max([0] + self.counts) if max_rows is None else max_rows
        self.device = device
        as_tensor = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.rows_t = None if self.plain else as_tensor(self.first)
        self.lengths_t, self.slots_t = as_tensor(lengths), as_tensor(slots)

    def lx(self):
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        return LxKv8Batch(self.seqs, at(self.rows_t), at(self.lengths_t), None, 0, self.max_rows, 0)

    def states(self, given, kept, count):
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        return LxStates(at(given), at(kept), at(self.slots_t), count)

    def spans(self):
        """[(sequence, first row of the call that counts, the one behind the last, position of that first row, whether it begins, slot)]"""
        found = []
        for s, n in enumerate(self.counts):
            lead = max(0, self.lengths[s]) - n if self.lengths is not None else 0
            first, stop = max(0, -lead), min(n, self.max_rows, self.T - self.first[s])
            if first < stop:
                found.append((s, self.first[s] + first, self.first[s] + stop, lead + first, self.lengths is not None and lead <= 0,
                              self.slots[s] if self.slots is not None else s))
        return found


def pointer(struct):
    return None if struct is None else ctypes.pointer(struct)


# ---- rotation ------------------------------------------------------------------------------------------------------------


def rotated(x, positions, freq, amplitude, rot, interleaved, heads, dim):
    """[T, heads * dim] in 64 bits, and the sum of the magnitudes that each value is made of."""
    x = x.double().view(x.shape[0], heads, dim)
    angle = positions.double()[:, None, None] * freq.double()
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    y, size = x.clone(), x.abs()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(amplitude)
    return y.flatten(1), size.flatten(1)


# ---- convolution ---------------------------------------------------------------------------------------------------------


def convolved(x, weight, bias, silu, rows, given, count):
    """y, its sums of magnitudes and the states afterwards ({slot: [width - 1, C]}); rows that belong to nobody are NaN."""
    T, C = x.shape
    width = weight.shape[1]
    y, size = (torch.full((T, C), math.nan, dtype=torch.float64) for _ in range(2))
    kept = {}
    w = weight.double()
    for s, begin, end, _, begins, slot in rows.spans():
        known = given is not None and not begins and 0 <= slot < count
        front = given[slot].double() if known else torch.zeros(width - 1, C, dtype=torch.float64)
        seen = torch.cat([front, x[begin:end].double()])
        n = end - begin
        part = sum(seen[j:j + n] * w[:, j] for j in range(width))
        magnitude = sum((seen[j:j + n] * w[:, j]).abs() for j in range(width))
        if bias is not None:
            part, magnitude = part + bias.double(), magnitude + bias.double().abs()
        y[begin:end] = part / (1 + torch.exp(-part)) if silu else part
        size[begin:end] = magnitude
        if 0 <= slot < count:
            kept[slot] = seen[n:]
    return y, size, kept


# ---- linear attention ----------------------------------------------------------------------------------------------------


class Mixer:
    """Inputs of a call of lx_linear_attention."""

    def __init__(self, rows, heads, k_heads, dk, dv, decay="head", skip=False, gate=None, dtype=torch.bfloat16, out=torch.bfloat16, step=torch.float32,
                 seed=0, strong=False, spare=1, bias=True, rate=True):
        self.rows, self.heads, self.k_heads, self.dk, self.dv, self.decay, self.dtype, self.out_dtype = rows, heads, k_heads, dk, dv, decay, dtype, out
        g = torch.Generator().manual_seed(seed)
        T = rows.T
        self.q, self.k = (torch.randn(T, k_heads * dk, generator=g).to(dtype) for _ in range(2))
        self.v = torch.randn(T, heads * dv, generator=g).to(dtype)
        self.scale = dk**-0.5
        self.skip = torch.rand(heads, generator=g) + 0.5 if skip else None
        self.gate = torch.randn(T, heads * dv, generator=g).to(gate) if gate else None
        self.x = self.rate = self.bias = None
        if decay == "head":
            self.rate = -torch.exp2(torch.rand(heads, generator=g) * 8 - (3 if strong else 9))
        elif decay == "log":
            self.x = (-torch.rand(T, heads, generator=g) * (6.0 if strong else 0.2)).to(step)
            self.rate = torch.rand(heads, generator=g) + 0.5 if rate else None
        else:
            self.x = (torch.randn(T, heads, generator=g) * (2.0 if strong else 0.7) - 2.0).to(step)
            self.bias = torch.randn(heads, generator=g) * 0.3 if bias else None
            self.rate = -(torch.rand(heads, generator=g) * 4 + 0.5) if rate else None
        slots = rows.slots if rows.slots is not None else range(rows.seqs)
        self.count = max([-1] + list(slots)) + 1 + spare
        self.state = torch.randn(self.count, heads, dk, dv, generator=g)

    def steps(self, t):
        """The decay's logarithm and the update's weight of row t, [heads] in 64 bits."""
        one = torch.ones(self.heads, dtype=torch.float64)
        if self.decay == "head":
            return self.rate.double(), one
        x = self.x[t].double()
        if self.decay == "log":
            return (x if self.rate is None else x * self.rate.double()), one
        d = torch.nn.functional.softplus(x if self.bias is None else x + self.bias.double(), threshold=1e9)
        return (-d if self.rate is None else d * self.rate.double()), d

    def want(self, state="own"):
        """{out, out_size, states {slot: S}, sizes {slot: sum of magnitudes}}; ``state``: what the call reads, None for nothing."""
        given = self.state if isinstance(state, str) else state
        T, heads, group = self.rows.T, self.heads, self.heads // self.k_heads
        out, size = (torch.full((T, heads, self.dv), math.nan, dtype=torch.float64) for _ in range(2))
        rounded = lambda x: x.to(torch.bfloat16).double()  # noqa: E731
        q, k = (rounded(x).view(T, self.k_heads, self.dk).repeat_interleave(group, 1) for x in (self.q, self.k))
        v = rounded(self.v).view(T, heads, self.dv)
        states, sizes = {}, {}
        for s, begin, end, _, begins, slot in self.rows.spans():
            known = given is not None and not begins and 0 <= slot < self.count
            S = given[slot].double().clone() if known else torch.zeros(heads, self.dk, self.dv, dtype=torch.float64)
            M = S.abs()
            for t in range(begin, end):
                log, weight = self.steps(t)
                fade = torch.exp(log)[:, None, None]
                new = k[t][:, :, None] * (v[t] * weight[:, None])[:, None, :]
                S, M = fade * S + new, fade * M + new.abs()
                out[t] = self.scale * (q[t][:, None] @ S)[:, 0]
                size[t] = abs(self.scale) * (q[t].abs()[:, None] @ M)[:, 0]
            if 0 <= slot < self.count:
                states[slot], sizes[slot] = S, M
        if self.skip is not None:
            more = self.skip.double()[:, None] * v
            out, size = out + more, size + more.abs()
        out, size = out.flatten(1), size.flatten(1)
        if self.gate is not None:
            z = self.gate.double()
            factor = z / (1 + torch.exp(-z))
            out, size = out * factor, size * factor.abs()
        return {"out": out, "out_size": size, "states": states, "sizes": sizes}

    def run(self, hip, give=True, keep="same", workspace=None, mixed=False, stream=None, call=None, pad=0):
        """(out, states afterwards) of the library's call, on the device. ``keep``: same (in place), other (a second tensor), none. ``mixed``: queries,
        keys and values are columns of one tensor, ``pad`` values behind them."""
        rows = Rows(None if self.rows.plain else self.rows.counts, self.rows.lengths, self.rows.slots, self.rows.T, self.rows.max_rows, self.rows.seqs, "cuda")
        cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
        q, k, v = cuda(self.q), cuda(self.k), cuda(self.v)
        if mixed:
            whole = torch.cat([v, k, q, torch.zeros(self.rows.T, pad, dtype=q.dtype, device="cuda")], 1)
            v, k, q = whole[:, :v.shape[1]], whole[:, v.shape[1]:v.shape[1] + k.shape[1]], whole[:, v.shape[1] + k.shape[1]:v.shape[1] + 2 * k.shape[1]]
        gate, x = cuda(self.gate), cuda(self.x)
        out = torch.full((self.rows.T, self.heads * self.dv), UNTOUCHED, dtype=self.out_dtype, device="cuda")
        given = cuda(self.state) if give else None
        kept = {"same": given if give else torch.full(self.state.shape, UNTOUCHED, device="cuda"),
                "other": torch.full(self.state.shape, UNTOUCHED, device="cuda"), "none": None}[keep]
        rate, bias, skip = cuda(self.rate), cuda(self.bias), cuda(self.skip)
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        decay = LxDecay(KINDS[self.decay], at(x), F32 if x is None else DTYPE[x.dtype], self.heads, at(rate), at(bias))
        batch, states = rows.lx(), rows.states(given, kept, self.count)
        sizes = (self.rows.T, self.heads, self.k_heads, self.dk, self.dv)
        if workspace is None:
            need = int(hip.size("linear_attention_workspace_bytes", pointer(batch), *sizes))
            assert need >= 0
            workspace = torch.randint(0, 256, (max(need, 16),), dtype=torch.uint8, device="cuda")
        args = (q, k, v, DTYPE[q.dtype], q.stride(0), k.stride(0), v.stride(0), pointer(decay), skip, gate, BF16 if gate is None else DTYPE[gate.dtype],
                self.heads * self.dv, pointer(batch), pointer(states), out, DTYPE[out.dtype], out.shape[1], *sizes, self.scale, workspace)
        self.held = (rows, decay, batch, states, rate, bias, skip, given, kept, x, q, k, v, gate, out, workspace, args)
        if call is None:
            hip("linear_attention", *args)
        else:
            call(args)
        return out, kept

    def check(self, out, kept, want, share, before=None):
        """Every output within ``share`` of the magnitudes it is a sum of, and its rounding; nothing else touched. ``before``: what the
        states' tensor held."""
        out, expected, size = out.double().cpu(), want["out"], want["out_size"]
        nobody = expected.isnan()
        assert bool((out[nobody] == UNTOUCHED).all()), "rows of nobody were written"
        error = (out - expected).abs()[~nobody]
        bound = (share * size + HALF[self.out_dtype] * 1.01 * (expected.abs() + share * size))[~nobody]
        assert bool((error <= bound + 1e-30).all()), f"out: worst {(error / (bound + 1e-30)).max().item():.3g} of its bound"
        if kept is None:
            return
        before = self.state if before is None else before
        for slot in range(self.count):
            got = kept[slot].double().cpu()
            if slot in want["states"]:
                error, bound = (got - want["states"][slot]).abs(), share * want["sizes"][slot] + 1e-30
                assert bool((error <= bound).all()), f"state {slot}: worst {(error / bound).max().item():.3g} of its bound"
            else:
                assert torch.equal(got, before[slot].double()), f"state {slot} was written"

"""The operators between the two products of a linear-attention mixer, as cases that can be timed and compared.

- ``rotate``: queries and keys of the call's rows turned by their positions, a part of each head or all of it, frequencies scaled
  for long contexts (lx_rotate).
- ``conv``: a short causal convolution along each sequence, a filter of its own for every channel, with the last inputs kept
  between calls (lx_causal_conv).
- ``linear``: linear attention with a decay for each head and a state kept between calls: prompts, drafted tokens, single tokens
  (lx_linear_attention).

With ``own`` false ``run`` computes the same by elementary torch operations. Which sequence has how many rows and tokens follows
from the case alone; values, slots and the order of things follow from the seed.
"""

import ctypes
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
CHUNK = 64
SPARE_SLOTS = 2


def _rotate(name, seqs, rows, longest, heads=40, dim=128, rot=128, interleaved=False, base=1e6, factor=1.0, explicit=False,
            dtype="bf16", out="bf16"):
    return {"name": name, "kind": "rotate", "seqs": seqs, "rows": rows, "longest": longest, "heads": heads, "dim": dim, "rot": rot,
            "interleaved": interleaved, "base": base, "factor": factor, "explicit": explicit, "dtype": dtype, "out": out}


def _conv(name, seqs, rows, longest, channels, width=4, silu=True, bias=True, dtype="bf16", out="bf16"):
    return {"name": name, "kind": "conv", "seqs": seqs, "rows": rows, "longest": longest, "channels": channels, "width": width,
            "silu": silu, "bias": bias, "dtype": dtype, "out": out}


def _linear(name, seqs, rows, longest, heads, k_heads, dk, dv, decay, skip=False, gate=False, out="bf16"):
    """``decay``: head (a constant for each head), log (one for every token and head), step (a step width for every token and
    head, which the update is multiplied by too)."""
    return {"name": name, "kind": "linear", "seqs": seqs, "rows": rows, "longest": longest, "heads": heads, "k_heads": k_heads,
            "dk": dk, "dv": dv, "decay": decay, "skip": skip, "gate": gate, "out": out}


def listed():
    return [
        # One stream decoding: its token's queries and keys. Latency counts.
        _rotate("rotate_s1", 1, 1, 8191),
        # Pieces of prompts far into long contexts: half of each head turned, neighbours paired, frequencies scaled.
        _rotate("rotate_pieces_scaled", 6, 2048, 131072, 36, 128, 64, True, 1e4, 8.0),
        # 64 streams decoding together through a wide mixer's convolution, each at a place of its own in its answer.
        _conv("conv_s64", 64, 1, 3001, 10240),
        # A prompt of 4096 tokens through the same.
        _conv("conv_prompt4096", 1, 4096, 4096, 10240),
        # Pieces of five prompts behind their earlier pieces; f32, three taps, no activation, an odd number of channels.
        _conv("conv_pieces_f32", 5, 611, 9001, 2050, 3, False, False, "f32", "f32"),
        # One stream decoding: the smallest state.
        _linear("linear_s1", 1, 1, 517, 32, 32, 128, 128, "head"),
        # 64 streams decoding together: 16 heads share a key, step widths, skip and gate; the states are what counts.
        _linear("linear_s64", 64, 1, 4096, 128, 8, 128, 64, "step", True, True),
        # Drafted tokens of eight streams verified together.
        _linear("linear_s8_verify5", 8, 5, 8191, 128, 8, 128, 64, "step", True, True),
        # A prompt of 4096 tokens through the same mixer.
        _linear("linear_prompt4096", 1, 4096, 4096, 128, 8, 128, 64, "step", True, True),
        # A long prompt, constant decays, few heads: work along a long axis.
        _linear("linear_prompt16384", 1, 16384, 16384, 16, 16, 128, 128, "head"),
        # Pieces of five prompts behind their earlier pieces; heads of odd sizes, f32 results.
        _linear("linear_pieces_odd", 5, 611, 9001, 12, 4, 96, 80, "log", out="f32"),
        # Eight prompts of up to 2048 tokens, a head of 256 keys' values.
        _linear("linear_prompts_wide", 8, 2048, 2048, 8, 8, 256, 256, "log", gate=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _lengths_of(rng, most):
    """(sequences, rows of the longest, its tokens): single tokens, a few, pieces, prompts."""
    seqs = _log_int(rng, 1, 64)
    rows = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, most)])
    return seqs, rows, max(rows, rng.choice([rows, _log_int(rng, 1, 131072)]))


def draw(rng):
    """One more case: from one row to a prompt, fresh sequences and ones far along, heads of every size, types."""
    kind = rng.choice(["rotate", "conv", "linear", "linear", "linear"])
    while True:
        seqs, rows, longest = _lengths_of(rng, 16384 if kind == "linear" else 8192)
        total = seqs * rows
        if kind == "rotate":
            dim = 8 * rng.randint(4, 32) if rng.random() < 0.7 else 2 * rng.randint(16, 128)
            heads = _log_int(rng, 1, 128)
            rot = rng.choice([dim, dim // 4 * 2, dim // 8 * 2])
            case = _rotate("", seqs, rows, longest, heads, dim, rot, rng.random() < 0.4, rng.choice([1e4, 5e5, 1e6]),
                           rng.choice([1.0, 1.0, 4.0, 32.0]), rng.random() < 0.3, rng.choice(["bf16", "bf16", "f32"]),
                           rng.choice(["bf16", "bf16", "f32"]))
            if total * heads * dim <= 8192 * 36 * 128:
                break
        elif kind == "conv":
            channels = _log_int(rng, 256, 16384)
            channels = channels if rng.random() < 0.2 else (channels + 63) // 64 * 64
            case = _conv("", seqs, rows, longest, channels, rng.randint(2, 4), rng.random() < 0.7, rng.random() < 0.7,
                         rng.choice(["bf16", "bf16", "f32"]), rng.choice(["bf16", "bf16", "f32"]))
            if total * channels <= 4096 * 10240:
                break
        else:
            dk, dv = rng.choice([(128, 128), (128, 64), (64, 64), (64, 128), (256, 256), (256, 512), (8 * rng.randint(2, 32), 8 * rng.randint(2, 40))])
            k_heads = _log_int(rng, 1, 32)
            heads = k_heads * rng.choice([1, 1, 2, 3, 8, 16])
            case = _linear("", seqs, rows, longest, heads, k_heads, dk, dv, rng.choice(["head", "log", "step"]), rng.random() < 0.4,
                           rng.random() < 0.4, rng.choice(["bf16", "bf16", "f32"]))
            if heads <= 128 and seqs * heads * dk * dv <= 64 * 128 * 128 * 64 and total * heads * max(dk, dv) <= 4096 * 128 * 128 \
                    and (total + 64 * seqs) * heads * dk * dv <= 4160 * 128 * 128 * 64:
                break
    del case["name"]
    return case


# ---- the inputs of a case ----------------------------------------------------------------------------------------------


def _sequences(case):
    """[(rows of this call, tokens so far with them)] of every sequence: the first has the most of both, the others have fewer,
    spread evenly; some of several begin with this call, and every seventh of those with more than one row has none."""
    found = []
    for i in range(case["seqs"]):
        rows, length = case["rows"], case["longest"]
        if i:
            length = max(1, int(length * ((i * 0.6180339887498949) % 1.0)))
            if rows > 16:
                rows = max(1, int(rows * ((i * 0.7548776662466927) % 1.0)))
            if rows > 1 and i % 7 == 6:
                rows = 0
            if i % 3 == 2:
                length = max(1, rows)
        found.append((min(rows, length), length))
    return found


class State:
    """Inputs, outputs and the arguments of the calls; what a program keeps between them too."""


def _frequencies(case):
    """Turned angles a position: base^(-2 i / rot), slowed by the factor where a wave is longer than the context the model was
    trained on, and in between by parts; their amplitude."""
    half, factor, original = case["rot"] // 2, case["factor"], 8192.0
    freq = [case["base"] ** (-i / half) for i in range(half)]
    if factor == 1.0:
        return freq, 1.0
    turns = [original * f / (2 * math.pi) for f in freq]
    kept = [min(1.0, max(0.0, (t - 1.0) / 31.0)) for t in turns]
    return [f * (k + (1 - k) / factor) for f, k in zip(freq, kept)], 0.1 * math.log(factor) + 1.0


def _inputs(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="f32", std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(TYPES[dtype])

    def uniform(*shape, low, high):
        return torch.rand(*shape, generator=g, device="cuda").mul_(high - low).add_(low)

    sequences = _sequences(case)
    s.lengths = torch.tensor([length for _, length in sequences], dtype=torch.int32, device="cuda")
    s.first = torch.tensor([0] + [rows for rows, _ in sequences], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    s.rows, s.most_rows = sum(rows for rows, _ in sequences), max(rows for rows, _ in sequences)
    s.slot_count = case["seqs"] + SPARE_SLOTS
    order = torch.randperm(s.slot_count, generator=torch.Generator().manual_seed(seed))
    s.slots = order[:case["seqs"]].to(torch.int32).cuda()
    if case["kind"] == "rotate":
        width = case["heads"] * case["dim"]
        # Queries and keys in front of the values, as the layer's first product writes them.
        s.qkv = normal(s.rows, width + 8 * case["dim"], dtype=case["dtype"])
        s.x = s.qkv[:, :width]
        freq, s.amplitude = _frequencies(case)
        s.freq = torch.tensor(freq, dtype=torch.float32, device="cuda")
        s.positions = None
        if case["explicit"]:
            s.positions = torch.cat([torch.arange(length - n, length, dtype=torch.int32) for n, length in sequences]).cuda()
        s.y = torch.empty(s.rows, width, dtype=TYPES[case["out"]], device="cuda")
    elif case["kind"] == "conv":
        channels, width = case["channels"], case["width"]
        s.x = normal(s.rows, channels, dtype=case["dtype"])
        s.weight = uniform(channels, width, low=-(width ** -0.5), high=width ** -0.5).to(torch.bfloat16)
        s.bias = uniform(channels, low=-0.5, high=0.5).to(torch.bfloat16) if case["bias"] else None
        s.state = normal(s.slot_count, width - 1, channels, dtype=case["dtype"])
        s.y = torch.empty(s.rows, channels, dtype=TYPES[case["out"]], device="cuda")
    else:
        heads, k_heads, dk, dv = (case[key] for key in ("heads", "k_heads", "dk", "dv"))
        # Values, keys and queries behind one another, as the convolution leaves them; gates and step widths likewise.
        mixed = heads * dv + 2 * k_heads * dk
        s.mixed = normal(s.rows, mixed, dtype="bf16")
        s.v, s.k, s.q = s.mixed.split([heads * dv, k_heads * dk, k_heads * dk], 1)
        s.scale = dk ** -0.5
        s.gates = normal(s.rows, heads * dv, dtype="bf16") if case["gate"] else None
        s.skip = uniform(heads, low=0.5, high=1.5) if case["skip"] else None
        s.bias = None
        if case["decay"] == "head":
            # Memories of 32 to 4096 tokens.
            s.step, s.rate = None, -torch.exp2(uniform(heads, low=-12.0, high=-5.0))
        elif case["decay"] == "log":
            s.step, s.rate = torch.nn.functional.logsigmoid(normal(s.rows, heads)) / 16.0, None
        else:
            # Step widths of 0.001 to 0.1 in the middle, decays of 1 to 16 a unit of them.
            s.step = normal(s.rows, heads, dtype="bf16", std=0.5)
            wide = torch.exp(uniform(heads, low=math.log(1e-3), high=math.log(0.1)))
            s.bias = wide + torch.log(-torch.expm1(-wide))
            s.rate = -uniform(heads, low=1.0, high=16.0)
        s.state = normal(s.slot_count, heads, dk, dv)
        s.out = torch.empty(s.rows, heads * dv, dtype=TYPES[case["out"]], device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _keep(s, case)
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------------


def _keep(s, case):
    """What a program that calls the library keeps: the library, the structs, the workspace, the call's arguments."""
    from dromos_amd import abi

    lx = abi.load_hip()
    stream = torch.cuda.current_stream().cuda_stream

    def call(name, *args):
        lowered = tuple(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args)
        return getattr(lx.lib, "lx_" + name), (*lowered, stream)

    s.batch = abi.LxKv8Batch(case["seqs"], s.first.data_ptr(), s.lengths.data_ptr(), None, 0, s.most_rows, case["longest"])
    batch = ctypes.pointer(s.batch)
    if case["kind"] == "rotate":
        s.call = call("rotate", s.x, abi.DTYPE[s.x.dtype], s.x.stride(0), s.y, abi.DTYPE[s.y.dtype], s.y.shape[1], batch, s.positions,
                      s.freq, s.amplitude, case["rot"], int(case["interleaved"]), s.rows, case["heads"], case["dim"])
        return
    s.states = abi.LxStates(s.state.data_ptr(), s.state.data_ptr(), s.slots.data_ptr(), s.slot_count)
    states = ctypes.pointer(s.states)
    if case["kind"] == "conv":
        channels = case["channels"]
        s.call = call("causal_conv", s.x, abi.DTYPE[s.x.dtype], channels, s.weight, s.bias, abi.BF16, case["width"],
                      abi.ACT_SILU if case["silu"] else abi.ACT_NONE, batch, states, s.y, abi.DTYPE[s.y.dtype], channels, s.rows, channels)
        return
    heads, k_heads, dk, dv = (case[key] for key in ("heads", "k_heads", "dk", "dv"))
    kind = {"head": abi.DECAY_HEAD, "log": abi.DECAY_LOG, "step": abi.DECAY_STEP}[case["decay"]]
    pointer = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    s.decay = abi.LxDecay(kind, pointer(s.step), abi.F32 if s.step is None else abi.DTYPE[s.step.dtype], heads, pointer(s.rate), pointer(s.bias))
    s.workspace = torch.empty(max(256, int(lx.size("linear_attention_workspace_bytes", batch, s.rows, heads, k_heads, dk, dv))),
                              dtype=torch.uint8, device="cuda")
    ld = s.mixed.shape[1]
    s.call = call("linear_attention", s.q, s.k, s.v, abi.BF16, ld, ld, ld, ctypes.pointer(s.decay), s.skip, s.gates, abi.BF16, heads * dv,
                  batch, states, s.out, abi.DTYPE[s.out.dtype], heads * dv, s.rows, heads, k_heads, dk, dv, s.scale, s.workspace)


def _own(s):
    entry, args = s.call
    status = entry(*args)
    if status != 0:
        raise RuntimeError(f"{entry.__name__} returned {status}")


# ---- the plain forms, in 32 bits ---------------------------------------------------------------------------------------


def _places(s):
    """Of every row: its sequence, its number among the sequence's rows, its position."""
    index = torch.arange(s.rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.first, index, right=True) - 1
    row = (index - s.first[seq]).long()
    return seq, row, (s.lengths[seq] - s.first[seq + 1] + index).long()


def _begins(s):
    """Whether a sequence begins with this call."""
    return s.lengths <= s.first[1:] - s.first[:-1]


def _rotate_plain(s):
    case = s.case
    position = _places(s)[2] if s.positions is None else s.positions
    x = s.x.float().reshape(s.rows, case["heads"], case["dim"])
    angle = position.double()[:, None, None] * s.freq.double()
    cos, sin = (angle.cos() * s.amplitude).float(), (angle.sin() * s.amplitude).float()
    turned, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s.y.copy_(torch.cat([turned, rest], -1).flatten(1))
    return {"y": s.y}


def _conv_plain(s):
    case = s.case
    channels, taps = case["channels"], case["width"]
    before = taps - 1
    seq, row, _ = _places(s)
    begins = _begins(s)
    # Row after row of what the filter sees: zeros, the kept rows of every slot, this call's rows.
    held = torch.cat([torch.zeros(1, channels, device="cuda", dtype=s.x.dtype), s.state.view(-1, channels), s.x])
    call = 1 + s.slot_count * before  # where this call's rows begin

    def at(seq, row):  # the place of row `row` of a sequence: before 0 the kept ones
        kept = 1 + s.slots[seq].long() * before + row + before
        kept = torch.where(begins[seq], torch.zeros_like(kept), kept)
        return torch.where(row < 0, kept, call + s.first[seq].long() + row)

    seen = at(seq[:, None].expand(-1, taps), row[:, None] + torch.arange(-before, 1, device="cuda"))
    y = (held[seen].float() * s.weight.float().t()).sum(1)
    if s.bias is not None:
        y = y + s.bias.float()
    s.y.copy_(y * torch.sigmoid(y) if case["silu"] else y)
    count = (s.first[1:] - s.first[:-1]).long()
    every = torch.arange(case["seqs"], device="cuda")
    last = held[at(every[:, None].expand(-1, before), count[:, None] + torch.arange(-before, 0, device="cuda"))]
    slots = s.slots.long()
    s.state[slots] = torch.where((count > 0)[:, None, None], last, s.state[slots])
    return {"y": s.y, "state": s.state}


def _steps(s):
    """The decay's logarithm and the update's weight of every row and head, in 64 bits."""
    heads = s.case["heads"]
    if s.case["decay"] == "head":
        return s.rate.double().expand(s.rows, heads), torch.ones(s.rows, heads, device="cuda", dtype=torch.float64)
    if s.case["decay"] == "log":
        return s.step.double(), torch.ones(s.rows, heads, device="cuda", dtype=torch.float64)
    x = s.step.double() + s.bias.double()
    step = x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))
    return step * s.rate.double(), step


def _linear_plain(s):
    """Chunk by chunk, all chunks at once: what a chunk's rows see of one another, what they see of the state in front of
    the chunk, and that state as the decayed sum of the chunks before."""
    case = s.case
    heads, k_heads, dk, dv = (case[key] for key in ("heads", "k_heads", "dk", "dv"))
    seqs, group = case["seqs"], heads // k_heads
    size = min(CHUNK, s.most_rows)
    chunks = -(-s.most_rows // size)
    seq, row, _ = _places(s)
    place = seq * (chunks * size) + row

    def laid(x, n, d):  # [seqs, heads, chunks, size, d], nothing where a sequence has no row
        out = torch.zeros(seqs * chunks * size, n, d, device="cuda", dtype=x.dtype)
        out[place] = x.reshape(s.rows, n, d)
        return out.view(seqs, chunks, size, n, d).permute(0, 3, 1, 2, 4)

    log, weight = (laid(x, heads, 1)[..., 0] for x in _steps(s))
    q, k = (laid(x.float(), k_heads, dk).contiguous() for x in (s.q, s.k))
    v = laid(s.v.float(), heads, dv).contiguous()
    total = log.cumsum(-1)  # up to and with each row of its chunk
    whole = total[..., -1]
    # Within a chunk.
    apart = torch.ones(size, size, device="cuda", dtype=torch.bool).tril()
    seen = torch.where(apart, total[..., :, None] - total[..., None, :], -math.inf).exp_().mul_(weight[..., None, :]).float()
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous())[:, :, None]
    scores = (seen.view(seqs, k_heads, group, chunks, size, size) * scores).view(seqs, heads, chunks, size, size)
    out = torch.matmul(scores, v)
    # A chunk's part of the state, and the state in front of every chunk (and behind the last).
    faded = ((whole[..., None] - total).exp() * weight).float()
    keys = k.transpose(-1, -2).contiguous()[:, :, None].expand(-1, -1, group, -1, -1, -1).reshape(seqs, heads, chunks, dk, size)
    part = torch.matmul(keys, v * faded[..., None]).view(seqs, heads, chunks, dk * dv)
    before = torch.nn.functional.pad(whole.cumsum(-1), (1, 0))
    between = before[..., :, None] - before[..., None, 1:]
    ahead = torch.ones(chunks + 1, chunks, device="cuda", dtype=torch.bool).tril(-1)
    state = torch.matmul(torch.where(ahead, between, -math.inf).exp_().float(), part)
    slots = s.slots.long()
    held = s.state[slots]
    start = torch.where(_begins(s)[:, None, None, None], torch.zeros_like(held), held).view(seqs, heads, 1, dk * dv)
    state = (state + before.exp().float()[..., None] * start).view(seqs, heads, chunks + 1, dk, dv)
    queries = q[:, :, None].expand(-1, -1, group, -1, -1, -1).reshape(seqs, heads, chunks, size, dk)
    out = out + torch.matmul(queries, state[:, :, :-1].contiguous()) * total.exp().float()[..., None]
    out = out.permute(0, 2, 3, 1, 4).reshape(-1, heads, dv)[place] * s.scale
    if s.skip is not None:
        out = out + s.skip[:, None] * s.v.float().reshape(s.rows, heads, dv)
    out = out.flatten(1)
    if s.gates is not None:
        gate = s.gates.float()
        out = out * (gate * torch.sigmoid(gate))
    s.out.copy_(out)
    some = (s.first[1:] > s.first[:-1])[:, None, None, None]
    s.state[slots] = torch.where(some, state[:, :, -1], held)
    return {"out": s.out, "state": s.state}


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"rotate": _rotate_plain, "conv": _conv_plain, "linear": _linear_plain}[kind](s)
    _own(s)
    return {"y": s.y} if kind == "rotate" else {"y": s.y, "state": s.state} if kind == "conv" else {"out": s.out, "state": s.state}


def work(case):
    """Every input read once and every output written once, states of sequences that begin with the call not read. Four
    operations per value of a state and token, two per tap, three per turned value."""
    sequences = _sequences(case)
    rows = sum(n for n, _ in sequences)
    held = sum(2 if length > n else 1 for n, length in sequences if n)
    if case["kind"] == "rotate":
        cells = rows * case["heads"] * case["dim"]
        return {"bytes": cells * (SIZE[case["dtype"]] + SIZE[case["out"]]) + 4.0 * rows * case["explicit"],
                "flops": 3.0 * rows * case["heads"] * case["rot"]}
    if case["kind"] == "conv":
        cells, kept = rows * case["channels"], (case["width"] - 1) * case["channels"]
        return {"bytes": cells * (SIZE[case["dtype"]] + SIZE[case["out"]]) + held * kept * SIZE[case["dtype"]]
                + 2.0 * case["channels"] * (case["width"] + case["bias"]), "flops": 2.0 * cells * case["width"]}
    values, keys = rows * case["heads"] * case["dv"], rows * case["k_heads"] * case["dk"]
    step = {"head": 0, "log": 4, "step": 2}[case["decay"]] * rows * case["heads"]
    return {"bytes": values * (2.0 + 2.0 * case["gate"] + SIZE[case["out"]]) + 4.0 * keys + step
            + 4.0 * held * case["heads"] * case["dk"] * case["dv"], "flops": 4.0 * values * case["dk"]}


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------------------


def _exact_rotate(s, case):
    """Every pair as a complex number times amplitude * e^(i position freq)."""
    parts, at = [], 0
    half, rot = case["rot"] // 2, case["rot"]
    for n, length in _sequences(case):
        x = s.x[at:at + n].double().reshape(n, case["heads"], case["dim"]).clone()
        angle = torch.arange(length - n, length, device="cuda").double()[:, None] * s.freq.double()
        turn = torch.polar(torch.full_like(angle, s.amplitude), angle)[:, None]
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, half), slice(half, rot))
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        parts.append(x.flatten(1))
        at += n
    return {"y": torch.cat(parts)}


def _exact_conv(s, case):
    """Sequence by sequence: the kept rows in front of its own, then tap by tap."""
    taps, parts, at = case["width"], [], 0
    state, slots = s.state.double().clone(), s.slots.tolist()
    for i, (n, length) in enumerate(_sequences(case)):
        front = state[slots[i]] if length > n else torch.zeros_like(state[0])
        x = torch.cat([front, s.x[at:at + n].double()])
        y = sum(x[j:j + n] * s.weight[:, j].double() for j in range(taps))
        if s.bias is not None:
            y = y + s.bias.double()
        parts.append(y / (1 + torch.exp(-y)) if case["silu"] else y)
        if n:
            state[slots[i]] = x[n:]
        at += n
    return {"y": torch.cat(parts), "state": state}


def _exact_linear(s, case):
    """Token by token, all sequences at once: the state decays, takes the token's product, and is read."""
    heads, k_heads, dk, dv = (case[key] for key in ("heads", "k_heads", "dk", "dv"))
    seqs, group, most = case["seqs"], heads // k_heads, s.most_rows
    if most > 1 and most * seqs * heads * dk * dv * 48 > 60e12:
        return None  # takes too long
    count = [n for n, _ in _sequences(case)]
    begins = torch.tensor([length <= n for n, length in _sequences(case)], device="cuda")
    index = torch.full((seqs, most), s.rows, dtype=torch.long)
    at = 0
    for i, n in enumerate(count):
        index[i, :n] = torch.arange(at, at + n)
        at += n
    index = index.cuda()

    def rows(x):  # one more row of zeros for those that a sequence does not have
        return torch.cat([x.double(), torch.zeros_like(x[:1], dtype=torch.float64)])

    q, k, v = rows(s.q), rows(s.k), rows(s.v)
    if case["decay"] == "head":
        log, weight = rows(s.rate.double().expand(s.rows, heads)), rows(torch.ones(s.rows, heads, device="cuda"))
    elif case["decay"] == "log":
        log, weight = rows(s.step), rows(torch.ones(s.rows, heads, device="cuda"))
    else:
        weight = torch.nn.functional.softplus(s.step.double() + s.bias.double(), threshold=1e9)
        log, weight = rows(weight * s.rate.double()), rows(weight)
    fade = log.exp()
    slots = s.slots.long()
    state = s.state.double()[slots]
    state[begins & torch.tensor([n > 0 for n in count], device="cuda")] = 0.0
    out = torch.zeros(s.rows + 1, heads, dv, dtype=torch.float64, device="cuda")
    for t in range(most):
        i = index[:, t]
        a, b = fade[i][..., None, None], weight[i][..., None]
        key = k[i].view(seqs, k_heads, 1, dk, 1).expand(-1, -1, group, -1, -1).reshape(seqs, heads, dk, 1)
        query = q[i].view(seqs, k_heads, 1, 1, dk).expand(-1, -1, group, -1, -1).reshape(seqs, heads, 1, dk)
        state.mul_(a).addcmul_(key, (v[i].view(seqs, heads, dv) * b)[:, :, None])
        out[i] = (query @ state)[:, :, 0]
    out = out[:-1] * s.scale
    if s.skip is not None:
        out = out + s.skip.double()[:, None] * s.v.double().reshape(s.rows, heads, dv)
    out = out.flatten(1)
    if s.gates is not None:
        out = out * torch.nn.functional.silu(s.gates.double())
    every = s.state.double().clone()
    every[slots] = state
    return {"out": out, "state": every}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "conv": _exact_conv, "linear": _exact_linear}[case["kind"]](s, case)

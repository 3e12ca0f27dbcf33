"""The operators between the products of an attention layer's step, as cases that can be timed and compared.

- ``append``: keys and values of this step's rows go into a paged cache of 8-bit codes with a scale per block of tokens
  and head; keys and queries are rotated by their positions on the way (lx_kv8_append). The cache's values are read back
  with lx_kv8_dequantize.
- ``attention``: the rows' queries against that cache, causal, over a window where the case has one (lx_kv8_attention).
- ``norm``: a block's output through its norm, gate and scale into the residual stream, and the norm in front of the next
  block (lx_block_norm).

With ``own`` false ``run`` computes the same by elementary torch operations in 32 bits. Which sequence has how many rows and
tokens follows from the case alone; values and the order of the pages follow from the seed.
"""

import ctypes
import math

import torch

own = False

QMAX = {"int8": 127.0, "fp8": 448.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
THETA = 1e6  # the rotation's base
SPARE_PAGES = 3


def _append(name, fmt, seqs, rows, longest, q_heads=32, heads=8, dim=128, page=64, block=32, rot=128, interleaved=False,
            dtype="bf16"):
    return {"name": name, "kind": "append", "format": fmt, "seqs": seqs, "rows": rows, "longest": longest, "q_heads": q_heads,
            "heads": heads, "dim": dim, "page": page, "block": block, "rot": rot, "interleaved": interleaved, "dtype": dtype}


def _attention(name, fmt, seqs, rows, longest, q_heads=32, heads=8, dim=128, page=64, block=32, window=0):
    return {"name": name, "kind": "attention", "format": fmt, "seqs": seqs, "rows": rows, "longest": longest,
            "q_heads": q_heads, "heads": heads, "dim": dim, "page": page, "block": block, "window": window}


def _norm(name, norm, rows, width, post, gate, stream="bf16", y="bf16", bias=False):
    """``gate``: none, row (a factor for every value) or broadcast (one row for all)."""
    return {"name": name, "kind": "norm", "norm": norm, "rows": rows, "width": width, "post": post, "gate": gate,
            "stream": stream, "y": y, "bias": bias}


def listed():
    return [
        # One stream decoding: its token's keys and values. Latency counts.
        _append("append_int8_s1", "int8", 1, 1, 101),
        # 64 streams decoding together, each at a place of its own in its answer.
        _append("append_fp8_s64", "fp8", 64, 1, 128),
        # A prompt of 4096 tokens.
        _append("append_fp8_prompt4096", "fp8", 1, 4096, 4096),
        # One stream early in its answer: the smallest attention.
        _attention("attention_int8_s1_517", "int8", 1, 1, 517),
        # 32 streams of ragged lengths: the decode step of a server.
        _attention("attention_fp8_s32_4096", "fp8", 32, 1, 4096),
        # One stream at the end of a long document: few rows over a long axis.
        _attention("attention_int8_s1_131072", "int8", 1, 1, 131072),
        # Drafted tokens of eight streams verified together.
        _attention("attention_fp8_s8_verify5", "fp8", 8, 5, 8191),
        # A prompt of 4096 tokens.
        _attention("attention_fp8_prompt4096", "fp8", 1, 4096, 4096),
        # Pieces of five prompts behind their earlier pieces, in small pages, over a window; a model with small heads.
        _attention("attention_int8_pieces_window", "int8", 5, 611, 9001, 16, 4, 64, 16, 16, 4096),
        # One stream: between two blocks of a layer.
        _norm("norm_rms_1x4096", "rms", 1, 4096, True, "none"),
        # 67 streams, the residual stream in f32, a gate for every value, norms with a mean and a bias.
        _norm("norm_layer_67x5120", "layer", 67, 5120, True, "row", "f32", "bf16", True),
        # A prompt of 8192 tokens, one gate for all of them.
        _norm("norm_rms_8192x4096", "rms", 8192, 4096, True, "broadcast"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: both formats, rows from one to a prompt, lengths to 131072 where the rows are few, head layouts with
    one to sixteen queries a key, pages of 16 to 256 tokens; norms from one row to 8192 and widths to 16384, odd ones too."""
    kind = rng.choice(["append", "attention", "attention", "norm"])
    if kind == "norm":
        while True:
            rows, width = _log_int(rng, 1, 8192), _log_int(rng, 512, 16384)
            width = width if rng.random() < 0.2 else (width + 63) // 64 * 64
            if rows * width <= 8192 * 4096:
                break
        post = rng.random() < 0.7
        case = _norm("", rng.choice(["rms", "layer"]), rows, width, post, rng.choice(["none", "row", "broadcast"]),
                     rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), rng.random() < 0.3)
    else:
        dim = rng.choice([64, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8]) if dim == 256 else rng.choice([1, 2, 4, 8, 16])
        q_heads = heads * rng.choice([1, 2, 4, 5, 8, 16])
        block = rng.choice([16, 32, 64])
        page = block * rng.choice([1, 2, 3, 4])
        fmt = rng.choice(["int8", "fp8"])
        if kind == "append":
            while True:
                seqs = _log_int(rng, 1, 64)
                rows = rng.choice([1, _log_int(rng, 1, 4096)])
                longest = max(rows, _log_int(rng, 1, 256))
                if seqs * rows * q_heads * dim <= 4096 * 4096 and seqs * longest * heads * dim <= 4096 * 1024:
                    break
            case = _append("", fmt, seqs, rows, longest, q_heads, heads, dim, page, block, rng.choice([dim, dim, dim // 2]),
                           rng.random() < 0.3, rng.choice(["bf16", "bf16", "f32"]))
        else:
            while True:
                seqs = _log_int(rng, 1, 64)
                rows = rng.choice([1, 1, _log_int(rng, 2, 8), _log_int(rng, 9, 4096)])
                longest = max(rows, _log_int(rng, 64, 131072))
                if seqs * rows * q_heads * dim * longest <= 4096 * 4096 * 4096 and seqs * longest * heads * dim <= 131072 * 1024:
                    break
            case = _attention("", fmt, seqs, rows, longest, q_heads, heads, dim, page, block,
                              _log_int(rng, 16, 8192) if rng.random() < 0.25 else 0)
    del case["name"]
    return case


# ---- the inputs of a case ----------------------------------------------------------------------------------------------


def _sequences(case):
    """[(rows, tokens in the cache, this call's rows among them)] of every sequence: the first has the most of both, the
    others have fewer, spread evenly; of several sequences with more than one row each, every fifth has none."""
    found = []
    for i in range(case["seqs"]):
        rows, length = case["rows"], case["longest"]
        if i:
            length = max(1, int(length * ((i * 0.6180339887498949) % 1.0)))
            if rows > 8:
                rows = max(1, int(rows * ((i * 0.7548776662466927) % 1.0)))
            if rows > 1 and i % 5 == 4:
                rows = 0
        found.append((min(rows, length), length))
    return found


class State:
    """Inputs, outputs and the arguments of the calls; what a program keeps between them too."""


def _paged(s, case, g):
    """The cache, the sequences' rows, lengths and page table."""
    sequences = _sequences(case)
    heads, dim, page, block, fmt = (case[key] for key in ("heads", "dim", "page", "block", "format"))
    need = [-(-length // page) for _, length in sequences]
    s.pages = sum(need) + SPARE_PAGES
    s.codes = torch.empty(2, s.pages, heads, page, dim, dtype=CODES[fmt], device="cuda")
    for part in s.codes:
        normal = torch.randn(part.shape, generator=g, device="cuda")
        part.copy_(normal.mul_(QMAX[fmt] / 3.5).round_().clamp_(-QMAX[fmt], QMAX[fmt]))
    s.scales = torch.rand(2, s.pages, heads, page // block, generator=g, device="cuda").add_(1.0).mul_(2.3 / QMAX[fmt])
    order = torch.randperm(s.pages, generator=torch.Generator().manual_seed(int(g.initial_seed()))).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s.table = table.cuda()
    s.lengths = torch.tensor([length for _, length in sequences], dtype=torch.int32, device="cuda")
    s.first = torch.tensor([0] + [rows for rows, _ in sequences], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    s.rows, s.most_rows, s.longest = sum(rows for rows, _ in sequences), max(rows for rows, _ in sequences), case["longest"]


def _inputs(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="f32", std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(TYPES[dtype])

    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        s.y, s.h = normal(rows, width, dtype=case["y"], std=2.0), normal(rows, width, dtype=case["stream"], std=3.0)
        s.gate = {"none": lambda: None, "row": lambda: normal(rows, width, dtype=case["y"]),
                  "broadcast": lambda: normal(1, width, dtype=case["y"])}[case["gate"]]()
        s.post = normal(width, dtype="bf16", std=0.1).add_(1.0) if case["post"] else None
        s.pre = normal(width, dtype="bf16", std=0.1).add_(1.0)
        s.post_bias = normal(width, dtype="bf16", std=0.1) if case["bias"] and case["post"] else None
        s.pre_bias = normal(width, dtype="bf16", std=0.1) if case["bias"] else None
        s.alpha, s.beta, s.eps = 0.7, 1.0, 1e-5
        s.h_out, s.x = torch.empty_like(s.h), torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    else:
        _paged(s, case, g)
        width = case["q_heads"] * case["dim"]
        if case["kind"] == "append":
            # One row of queries, keys and values behind one another, as the layer's first product writes it.
            kv = case["heads"] * case["dim"]
            s.qkv = normal(s.rows, width + 2 * kv, dtype=case["dtype"])
            s.q, s.k, s.v = s.qkv[:, :width], s.qkv[:, width:width + kv], s.qkv[:, width + kv:]
            half = case["rot"] // 2
            s.freq = torch.tensor([THETA ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")
            s.q_out = torch.empty(s.rows, width, dtype=torch.bfloat16, device="cuda")
            s.values = torch.empty(s.codes.shape, dtype=torch.bfloat16, device="cuda")
        else:
            s.q = normal(s.rows, width, dtype="bf16", std=1.5)
            s.scale = case["dim"] ** -0.5
            s.out = torch.empty(s.rows, width, dtype=torch.bfloat16, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _keep(s, case)
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------------


def _keep(s, case):
    """What a program that calls the library keeps: the library, the structs, the workspace, the calls' arguments."""
    from dromos_amd import abi

    lx = abi.load_hip()
    stream = torch.cuda.current_stream().cuda_stream

    def call(name, *args):
        lowered = tuple(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args)
        return getattr(lx.lib, "lx_" + name), (*lowered, stream)

    if case["kind"] == "norm":
        kind = abi.NORM_RMS if case["norm"] == "rms" else abi.NORM_LAYER
        rows, width = case["rows"], case["width"]
        ld_gate = width if case["gate"] == "row" else 0
        s.calls = [call("block_norm", kind, s.y, abi.DTYPE[s.y.dtype], width, s.post, s.post_bias, s.gate, ld_gate, s.alpha, s.beta,
                        s.h, s.h_out, abi.DTYPE[s.h.dtype], width, s.pre, s.pre_bias, abi.BF16, s.x, abi.BF16, width, s.eps, rows,
                        width)]
        return
    s.cache = abi.LxKv8(abi.FORMATS[case["format"]], s.codes[0].data_ptr(), s.codes[1].data_ptr(), s.scales[0].data_ptr(),
                        s.scales[1].data_ptr(), s.pages, case["heads"], case["page"], case["block"], case["dim"])
    s.batch = abi.LxKv8Batch(case["seqs"], s.first.data_ptr(), s.lengths.data_ptr(), s.table.data_ptr(), s.table.shape[1],
                             s.most_rows, s.longest)
    cache, batch = ctypes.pointer(s.cache), ctypes.pointer(s.batch)
    width = case["q_heads"] * case["dim"]
    if case["kind"] == "append":
        ld, dtype = s.qkv.shape[1], abi.DTYPE[s.qkv.dtype]
        s.calls = [call("kv8_append", cache, batch, s.q, s.k, s.v, dtype, ld, ld, ld, s.q_out, abi.BF16, width, s.freq, case["rot"],
                        int(case["interleaved"]), s.rows, case["q_heads"]),
                   call("kv8_dequantize", cache, s.values[0], s.values[1])]
        return
    s.workspace = torch.empty(max(256, int(lx.size("kv8_attention_workspace_bytes", cache, batch, s.rows, case["q_heads"]))),
                              dtype=torch.uint8, device="cuda")
    s.calls = [call("kv8_attention", s.q, abi.BF16, width, cache, batch, s.out, abi.BF16, width, s.rows, case["q_heads"], s.scale,
                    case["window"], s.workspace)]


def _own(s):
    for entry, args in s.calls:
        status = entry(*args)
        if status != 0:
            raise RuntimeError(f"{entry.__name__} returned {status}")


# ---- the plain forms, in 32 bits ---------------------------------------------------------------------------------------


def _places(s):
    """Of every row: its sequence, position, page and place in the page."""
    index = torch.arange(s.rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.first, index, right=True) - 1
    position = (s.lengths[seq] - s.first[seq + 1] + index).long()
    page = s.case["page"]
    return seq, position, s.table[seq, position // page].long(), position % page


def _rotated(x, heads, position, s):
    """[rows, heads, dim] in f32, rotated by the angles position * freq (the angles in 64 bits)."""
    case = s.case
    x = x.float().view(x.shape[0], heads, case["dim"])
    angle = position.double()[:, None, None] * s.freq.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    turned, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _coded(values, fmt):
    q = QMAX[fmt]
    return values.clamp(-q, q).to(CODES[fmt]) if fmt == "fp8" else values.round().clamp(-q, q).to(CODES[fmt])


def _appended(s, part, x, seq, position, page, place):
    """The rows x [rows, heads, dim] into part 0 (keys) or 1 (values) of the cache."""
    case = s.case
    fmt, block = case["format"], case["block"]
    codes, scales = s.codes[part], s.scales[part]
    pages, heads, blocks = scales.shape
    at = place // block
    # The largest magnitude that this call brings to each block, and the first place of it that it writes.
    top = torch.zeros(pages, blocks, heads, device="cuda")
    flat = (page * blocks + at)[:, None].expand(-1, heads)
    top = top.view(-1, heads).scatter_reduce(0, flat, x.abs().amax(-1), "amax").view(pages, blocks, heads).permute(0, 2, 1)
    begin = torch.full((pages * blocks,), block, device="cuda").scatter_reduce(0, page * blocks + at, place % block, "amin").view(pages, 1, blocks)
    touched, kept = begin < block, (begin > 0) & (begin < block)
    old = torch.where(kept, scales, torch.zeros_like(scales))
    new = torch.maximum(old, (top.double() / QMAX[fmt]).float())
    # Tokens in front of this call's, where the scale of their block grew.
    factor = torch.where(new > 0, (old.double() / new.double()).float(), torch.zeros_like(new))
    held = codes.view(pages, heads, blocks, block, -1)
    again = (kept & (new > old))[..., None, None] & (torch.arange(block, device="cuda")[:, None] < begin[..., None, None])
    held.copy_(torch.where(again, _coded(held.float() * factor[..., None, None], fmt).float(), held.float()).to(CODES[fmt]))
    scales.copy_(torch.where(touched, new, scales))
    inverse = torch.where(new > 0, (1.0 / new.double()).float(), torch.zeros_like(new))
    per_row = inverse[page, :, at]
    _as_bytes(codes)[page, :, place] = _as_bytes(_coded(x * per_row[..., None], fmt))


def _as_bytes(t):
    return t.view(torch.uint8)


def _values(s):
    """What the cache's codes stand for, [2, pages, heads, page, dim] in bf16."""
    two, pages, heads, blocks = s.scales.shape
    held = s.codes.float().view(two, pages, heads, blocks, s.case["block"], -1)
    return (held * s.scales[..., None, None]).view(s.codes.shape).to(torch.bfloat16)


def _append_plain(s):
    case = s.case
    seq, position, page, place = _places(s)
    q = _rotated(s.q, case["q_heads"], position, s).flatten(1).to(torch.bfloat16)
    _appended(s, 0, _rotated(s.k, case["heads"], position, s), seq, position, page, place)
    _appended(s, 1, s.v.float().view(s.rows, case["heads"], case["dim"]), seq, position, page, place)
    return {"q": q, "values": _values(s), "scales": s.scales}


def _attention_plain(s):
    case = s.case
    heads, dim, page, block = (case[key] for key in ("heads", "dim", "page", "block"))
    group = case["q_heads"] // heads
    token = torch.arange(s.longest, device="cuda")
    pages, place = s.table[:, token // page].long(), token % page
    index = torch.arange(s.rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.first, index, right=True) - 1
    row = index.long() - s.first[seq].long()
    inside = token < s.lengths[:, None]

    def held(part):  # [seqs, heads, longest, dim]
        scale = s.scales[part][pages, :, place // block].permute(0, 2, 1)[..., None]
        values = _as_bytes(s.codes[part])[pages, :, place].view(CODES[case["format"]]).permute(0, 2, 1, 3).float() * scale
        return torch.where(inside[:, None, :, None], values, torch.zeros((), device="cuda"))

    q = torch.zeros(case["seqs"], s.most_rows, case["q_heads"], dim, device="cuda")
    q[seq, row] = s.q.float().view(s.rows, case["q_heads"], dim)
    q = q.view(case["seqs"], s.most_rows, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(case["seqs"], heads, -1, dim)
    scores = torch.matmul(q, held(0).transpose(-1, -2).contiguous()).mul_(s.scale)
    scores = scores.view(case["seqs"], heads, s.most_rows, group, s.longest)
    last = (s.lengths - (s.first[1:] - s.first[:-1])).long()[:, None] + torch.arange(s.most_rows, device="cuda")
    seen = token <= last[..., None]
    if case["window"]:
        seen &= token > last[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), held(1).contiguous()).view(case["seqs"], heads, s.most_rows, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 2, 1, 3, 4).reshape(case["seqs"], s.most_rows, -1)
    return {"out": out[seq, row].to(torch.bfloat16)}


def _normed(x, norm, weight, bias, eps):
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    return x if bias is None else x + bias.float()


def _norm_plain(s):
    norm = s.case["norm"]
    r = s.y.float()
    if s.post is not None:
        r = _normed(r, norm, s.post, s.post_bias, s.eps)
    if s.gate is not None:
        r = r * s.gate.float()
    h = s.beta * s.h.float() + s.alpha * r
    return {"h": h.to(s.h.dtype), "x": _normed(h, norm, s.pre, s.pre_bias, s.eps).to(torch.bfloat16)}


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"append": _append_plain, "attention": _attention_plain, "norm": _norm_plain}[kind](s)
    _own(s)
    if kind == "append":
        return {"q": s.q_out, "values": s.values, "scales": s.scales}
    return {"out": s.out} if kind == "attention" else {"h": s.h_out, "x": s.x}


def work(case):
    """Every input read once and every output written once; of the cache, what the sequences hold (attention) or what is
    written and read back as values (append). Four operations per query value and attended key."""
    if case["kind"] == "norm":
        cells = case["rows"] * case["width"]
        gate = {"none": 0, "row": cells, "broadcast": case["width"]}[case["gate"]]
        return {"bytes": (cells + gate) * SIZE[case["y"]] + 2 * cells * SIZE[case["stream"]] + 2 * cells, "flops": 12.0 * cells}
    sequences = _sequences(case)
    rows, held = sum(n for n, _ in sequences), sum(length for _, length in sequences)
    kv, width = case["heads"] * case["dim"], case["q_heads"] * case["dim"]
    if case["kind"] == "append":
        pages = sum(-(-length // case["page"]) for _, length in sequences) + SPARE_PAGES
        cells = 2 * pages * case["page"] * kv
        return {"bytes": rows * (width + 2 * kv) * SIZE[case["dtype"]] + 2 * rows * width + 2 * rows * kv + 3 * cells,
                "flops": 3.0 * rows * (width + kv) + 2.0 * cells}
    window = case["window"] or case["longest"]
    seen, read = 0, 0
    for n, length in sequences:
        first = length - n + 1  # keys of the first row without a window
        seen += sum(range(first, length + 1)) if length <= window else sum(min(first + i, window) for i in range(n))
        read += min(length, window + n - 1) if n else 0
    return {"bytes": 2.0 * read * kv * (1 + 4.0 / (case["block"] * case["dim"])) + 4.0 * rows * width,
            "flops": 4.0 * case["q_heads"] * case["dim"] * seen}


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------------------


def _exact_append(s, case):
    """Sequence by sequence and block by block: the scale is the larger of the old one (while older tokens stay in the
    block) and the largest new magnitude over the largest code; codes are the nearest multiples. The plain values are
    what those codes stand for."""
    fmt, dim, heads, page, block = case["format"], case["dim"], case["heads"], case["page"], case["block"]
    sequences, half = _sequences(case), case["rot"] // 2

    def turned(x, n, position):
        x = x.double().reshape(x.shape[0], n, dim).clone()
        angle = position.double()[:, None] * s.freq.double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        a, b = (slice(0, case["rot"], 2), slice(1, case["rot"], 2)) if case["interleaved"] else (slice(0, half), slice(half, case["rot"]))
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    def nearest(v):
        if fmt == "int8":
            return v.round().clamp(-127, 127)
        v = v.clamp(-448, 448)
        exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0**-6)))
        step = torch.exp2(exponent - 3)
        return (v / step).round() * step

    codes, scales = s.codes.double(), s.scales.double()
    q, at = [], 0
    for i, (n, length) in enumerate(sequences):
        position = torch.arange(length - n, length, device="cuda")
        mine = slice(at, at + n)
        q.append(turned(s.q[mine], case["q_heads"], position).flatten(1))
        new = [turned(s.k[mine], heads, position), s.v[mine].double().view(n, heads, dim)]
        for part in range(2):
            t = length - n
            while t < length:
                end = min(length, (t // block + 1) * block)
                p, place = int(s.table_host[i][t // page]), t % page
                b, keep = place // block, place % block
                x = new[part][t - (length - n):end - (length - n)].permute(1, 0, 2)
                old = scales[part, p, :, b] if keep else torch.zeros(heads, dtype=torch.float64, device="cuda")
                scale = torch.maximum(old, x.abs().amax((1, 2)) / QMAX[fmt])
                front = codes[part, p, :, place - keep:place]
                grown = (scale > old)[:, None, None]
                codes[part, p, :, place - keep:place] = torch.where(grown, nearest(front * (old / scale)[:, None, None]), front)
                codes[part, p, :, place:place + end - t] = nearest(x / scale[:, None, None])
                scales[part, p, :, b] = scale
                t = end
        at += n
    values = codes.view(2, s.pages, heads, page // block, block, dim) * scales[..., None, None]
    return {"q": torch.cat(q), "values": values.view(s.codes.shape), "scales": scales}


def _exact_attention(s, case):
    heads, dim, page, block = case["heads"], case["dim"], case["page"], case["block"]
    group = case["q_heads"] // heads
    outs, at = [], 0
    for i, (n, length) in enumerate(_sequences(case)):
        if not n:
            continue
        pages = s.table[i, :-(-length // page)].long()
        keys, values = ((s.codes[part].view(torch.uint8)[pages].view(CODES[case["format"]]).double()
                         * s.scales[part][pages].double().repeat_interleave(block, -1)[..., None]).permute(1, 0, 2, 3)
                        .reshape(heads, -1, dim)[:, :length] for part in range(2))
        out = torch.empty(n, heads, group, dim, dtype=torch.float64, device="cuda")
        for begin in range(0, n, 512):  # so many rows at a time, for the scores' memory
            end = min(n, begin + 512)
            q = s.q[at + begin:at + end].double().view(end - begin, heads, group, dim).permute(1, 2, 0, 3).reshape(heads, -1, dim)
            scores = (q @ keys.transpose(1, 2).contiguous() * s.scale).view(heads, group, end - begin, length)
            behind = torch.arange(length, device="cuda") - (length - n + torch.arange(begin, end, device="cuda"))[:, None]
            hidden = behind > 0
            if case["window"]:
                hidden |= behind <= -case["window"]
            part = torch.softmax(scores.masked_fill(hidden, -math.inf), -1).view(heads, -1, length) @ values
            out[begin:end] = part.view(heads, group, end - begin, dim).permute(2, 0, 1, 3)
        outs.append(out.flatten(1))
        at += n
    return {"out": torch.cat(outs)}


def _exact_norm(s, case):
    def norm(x, weight, bias):
        mean = x.mean(-1, keepdim=True) if case["norm"] == "layer" else 0.0
        spread = ((x - mean) ** 2).sum(-1, keepdim=True) / case["width"]
        out = (x - mean) / (spread + s.eps).sqrt() * weight.double()
        return out if bias is None else out + bias.double()

    r = s.y.double() if s.post is None else norm(s.y.double(), s.post, s.post_bias)
    h = s.beta * s.h.double() + s.alpha * (r if s.gate is None else r * s.gate.double())
    return {"h": h, "x": norm(h, s.pre, s.pre_bias)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "append":
        s.table_host = s.table.tolist()
        return _exact_append(s, case)
    return (_exact_attention if case["kind"] == "attention" else _exact_norm)(s, case)

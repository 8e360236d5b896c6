"""The operators that a decoder layer needs between its quantised products, as measured cases.

Four operators of ``b200/linalg``: the root-mean-square norm with the residual's addition and an 8-bit output
(``tb200_rmsnorm_quant``), block tables and slot maps built from request lengths (``tb200_paged_plan``), rotary
positions with the write into the paged cache (``tb200_rope_append``) and the attention of new tokens over that cache
(``tb200_paged_attention``).  ``run`` computes them with elementary torch operations, or, where ``own`` is true, through
the library's entry points.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}          # tb200_type
FORMATS = {"int8": 0, "e4m3": 1, "e5m2": 2}      # tb200_quant_format
LARGEST = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DEVICE = "cuda"


# ---- cases ---------------------------------------------------------------------------------------------------------
def _norm(rows, cols, type, format, group):
    return {"op": "norm", "rows": rows, "cols": cols, "type": type, "format": format, "group": group}


def _plan(requests, cached, new, page, pad, lens):
    return {"op": "plan", "requests": requests, "cached": cached, "new": new, "page": page, "pad": pad, "lens": lens}


def _append(tokens, heads, kv_heads, dim, in_type, type, rot, interleaved, page, pad):
    return {"op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "in_type": in_type, "type": type,
            "rot": rot, "interleaved": interleaved, "page": page, "pad": pad}


def _attention(requests, cached, new, heads, kv_heads, dim, type, page, window, pad, lens):
    return {"op": "attention", "requests": requests, "cached": cached, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "type": type, "page": page, "window": window, "pad": pad, "lens": lens}


def listed():
    """``cached`` and ``new`` are the longest lengths of a case; ``lens`` seeds the lengths of its requests (0: all the longest)."""
    return [
        # one row before the projections of a decode step: int8 blocks of 32, the activations of the integer mat-vecs
        dict(_norm(1, 4096, "f32", "int8", 32), name="norm, one row"),
        # a prompt's rows before an fp8 product with one scale a row
        dict(_norm(8192, 4096, "bf16", "e4m3", 0), name="norm, 8192 rows"),
        # a wide, odd number of rows in groups of 128, as between the two products of a feed-forward block
        dict(_norm(333, 14336, "f16", "int8", 128), name="norm, 333 wide rows"),
        # the next token of 64 requests
        dict(_plan(64, 8191, 1, 16, 0, 11), name="plan, 64 decoding requests"),
        # a step that admits prompts: ragged chunks, some rows of the step empty
        dict(_plan(4000, 4000, 257, 16, 1000, 12), name="plan, 4000 ragged requests"),
        # one token's projections in fp32, as a quantised mat-vec leaves them
        dict(_append(1, 32, 8, 128, "f32", "bf16", 128, False, 16, 0), name="append, one token"),
        # a prompt's projections in one bf16 row a token, pairs next to one another
        dict(_append(8192, 32, 8, 128, "bf16", "bf16", 128, True, 16, 0), name="append, 8192 tokens"),
        # one request decoding after a short prompt: latency
        dict(_attention(1, 1000, 1, 32, 8, 128, "bf16", 16, 0, 0, 0), name="attention, one token"),
        # 64 decoding requests of ragged lengths: the cache's bandwidth
        dict(_attention(64, 8191, 1, 32, 8, 128, "f16", 16, 0, 0, 21), name="attention, 64 next tokens"),
        # two long contexts: few rows over a long axis
        dict(_attention(2, 131000, 1, 32, 8, 128, "bf16", 64, 0, 0, 22), name="attention, two long contexts"),
        # chunks of new tokens over what the cache holds already
        dict(_attention(4, 8000, 512, 32, 8, 128, "bf16", 16, 0, 5, 23), name="attention, four chunks"),
        # a whole prompt into an empty cache
        dict(_attention(1, 0, 8192, 32, 8, 128, "f16", 64, 0, 0, 0), name="attention, a prompt of 8192"),
    ]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(("norm", "plan", "append", "attention", "attention", "attention"))
    pad = rng.choice((0, 0, 3, 65))
    if op == "norm":
        group = rng.choice((0, 32, 64, 128))
        cols = _log_int(rng, 64, 16384)
        return _norm(_log_int(rng, 1, max(1, (32 << 20) // cols)), cols, rng.choice(("f32", "f16", "bf16")), rng.choice(("int8", "e4m3", "e5m2")), group)
    if op == "plan":
        new = _log_int(rng, 1, 4096)
        return _plan(_log_int(rng, 1, min(8192, (1 << 20) // new)), _log_int(rng, 1, 32768), new, rng.choice((8, 16, 20, 32, 64, 128)), pad, rng.randrange(1, 1 << 20))
    heads, kv_heads = rng.choice(((32, 8), (32, 32), (28, 4), (16, 1), (40, 8), (8, 8), (64, 8)))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    if op == "append":
        return _append(_log_int(rng, 1, (32 << 20) // ((heads + 2 * kv_heads) * dim)), heads, kv_heads, dim, rng.choice(("f32", "f16", "bf16")),
                       rng.choice(("f16", "bf16")), rng.choice((dim, dim, dim // 2)), rng.random() < 0.5, rng.choice((8, 16, 20, 32, 64, 128)), pad)
    page, window, kind = rng.choice((8, 16, 20, 32, 64, 128)), 0, rng.choice(("f16", "bf16"))
    if rng.random() < 0.5:  # next tokens, one or a few a request
        new = rng.choice((1, 1, 1, 2, 4))
        requests = _log_int(rng, 1, 128)
        cached = _log_int(rng, 16, max(16, min(131072, (1 << 28) // (requests * kv_heads * dim))))
    else:  # chunks
        new = _log_int(rng, 5, 4096)
        requests = _log_int(rng, 1, max(1, min(16, 4096 // new)))
        cached = _log_int(rng, 1, max(1, min(16384, (1 << 31) // (requests * heads * new))))
    if rng.random() < 0.25:
        window = _log_int(rng, 16, cached + new)
    return _attention(requests, cached, new, heads, kv_heads, dim, kind, page, window, pad, rng.randrange(1, 1 << 20))


def _lengths(case):
    """The cached and the new tokens of every request.  The first request has the longest lengths; the others are
    ragged, and one in sixteen of them adds nothing in this step."""
    n, cached, new = case["requests"], case["cached"], case["new"]
    if not case["lens"]:
        return [cached] * n, [new] * n
    rng = random.Random(case["lens"])
    c = [cached] + [rng.randint(cached // 8, cached) for _ in range(n - 1)]
    m = [new] + [0 if rng.random() < 1 / 16 else rng.randint((new + 1) // 2, new) for _ in range(n - 1)]
    return c, m


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if op == "norm":
        rows, cols, b = case["rows"], case["cols"], size[case["type"]]
        groups = -(-cols // case["group"]) if case["group"] else 1
        return {"bytes": rows * cols * (3 * b + 1) + rows * groups * 4 + cols * 4, "flops": 8 * rows * cols}
    if op == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        fresh = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        # lengths in, offsets and lengths out, a position and a slot for each token row, a free page in and an entry out for each fresh page
        return {"bytes": 16 * len(new) + 12 * (sum(new) + case["pad"]) + 8 * fresh, "flops": 0}
    if op == "append":
        t, rows = case["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": t * (rows * (size[case["in_type"]] + 2) + 4 * case["rot"] + 12), "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rot"]}
    cached, new = _lengths(case)
    window = case["window"]
    pairs = keys = 0
    for c, n in zip(cached, new):
        if window:
            pairs += sum(min(window, c + i + 1) for i in range(n))
            keys += min(c + n, window + n - 1) if n else 0
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n if n else 0
    pages = sum(-(-(c + n) // case["page"]) for c, n in zip(cached, new))
    return {"bytes": 4 * sum(new) * case["heads"] * case["dim"] + 4 * keys * case["kv_heads"] * case["dim"] + 4 * pages + 8 * len(new),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device=DEVICE)


def _offsets(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _tables(length, rot):
    """Cosine and sine of every position's angles, computed in 64 bits: [length][rot / 2]."""
    inverse = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    angles = torch.arange(length, dtype=torch.float64, device=DEVICE)[:, None] * inverse
    return angles.cos().float(), angles.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, type=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(type)

    def large(*shape, type):  # a cache: whatever earlier requests left lies behind the last token of a page
        return torch.empty(*shape, device=DEVICE, dtype=type).normal_(generator=gen)

    op, s = case["op"], {"case": case, "workspace": None}
    if op == "norm":
        rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
        group = case["group"] or cols
        # a residual stream: a few channels are much larger than the rest
        spread = torch.exp(0.5 * normal(cols)) * torch.where(torch.rand(cols, generator=gen, device=DEVICE) < 0.002, 30.0, 1.0)
        s.update(x=normal(rows, cols, type=kind), residual=(normal(rows, cols) * spread).to(kind), weight=1 + 0.2 * normal(cols), eps=1e-5)
        s.update(summed=torch.empty(rows, cols, device=DEVICE, dtype=kind), q=torch.empty(rows, cols, device=DEVICE, dtype=torch.uint8),
                 scales=torch.empty(rows, -(-cols // group), device=DEVICE))
        return s
    if op == "append":
        t, heads, kv_heads, dim, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        rows, pages = t + case["pad"], -(-t // page) + 3
        length = 2 * t + 4096
        cos, sin = _tables(length, case["rot"])
        slots = torch.randperm(pages * page, generator=gen, device=DEVICE)[:t].to(torch.int64)
        positions = torch.randint(0, length, (t,), generator=gen, device=DEVICE, dtype=torch.int32)
        fill = torch.full((case["pad"],), -1, device=DEVICE, dtype=torch.int64)
        s.update(qkv=normal(rows, (heads + 2 * kv_heads) * dim, type=TYPES[case["in_type"]]), cos=cos, sin=sin,
                 positions=torch.cat((positions, fill.to(torch.int32))), slots=torch.cat((slots, fill)),
                 q=large(rows, heads, dim, type=TYPES[case["type"]]), k_cache=large(pages, kv_heads, page, dim, type=TYPES[case["type"]]),
                 v_cache=large(pages, kv_heads, page, dim, type=TYPES[case["type"]]))
        return s
    cached, new = _lengths(case)
    page, tokens = case["page"], sum(new)
    before = [-(-c // page) for c in cached]
    after = [-(-(c + n) // page) for c, n in zip(cached, new)]
    width, pages = max(after), sum(after) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    starts, have = _ints(_offsets(after)[:-1], torch.int64), _ints(after)
    at = torch.arange(width, device=DEVICE)
    table = order[(starts[:, None] + at).clamp_(max=pages - 1)]
    s.update(cached=_ints(cached), new=_ints(new), width=width)
    if op == "plan":
        # pages held before this step stay in the table; the step's fresh pages come off the free list
        held = at < _ints(before)[:, None]
        fresh = (at < have[:, None]) & ~held
        s.update(table=torch.where(held, table, -1), free=table[fresh].contiguous(), rows=tokens + case["pad"],
                 counts=torch.zeros(4, device=DEVICE, dtype=torch.int32), offsets=torch.zeros(len(new) + 1, device=DEVICE, dtype=torch.int32),
                 kv_lens=torch.zeros(len(new), device=DEVICE, dtype=torch.int32), positions=torch.zeros(tokens + case["pad"], device=DEVICE, dtype=torch.int32),
                 slots=torch.zeros(tokens + case["pad"], device=DEVICE, dtype=torch.int64))
        return s
    heads, kv_heads, dim, kind = case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    s.update(table=torch.where(at < have[:, None], table, -1).contiguous(), offsets=_ints(_offsets(new)), tokens=tokens,
             kv_lens=_ints([c + n for c, n in zip(cached, new)]), scale=dim ** -0.5, longest=max(new),
             q=1.5 * normal(tokens + case["pad"], heads, dim, type=kind), k_cache=large(pages, kv_heads, page, dim, type=kind),
             v_cache=large(pages, kv_heads, page, dim, type=kind), out=normal(tokens + case["pad"], heads, dim, type=kind))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _values(q, case):
    """The numbers that the 8-bit output stands for, in units of their scales (which are an output of their own): fp8
    numbers as they are, whole numbers up to 127 in bf16, which holds them exactly."""
    return q.view(torch.int8).to(torch.bfloat16) if case["format"] == "int8" else q.view(FP8[case["format"]])


def _plain_norm(s):
    case = s["case"]
    rows, cols, group = case["rows"], case["cols"], case["group"] or case["cols"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + s["eps"]) * s["weight"]
    padded = torch.nn.functional.pad(y, (0, -cols % group)).view(rows, -1, group)
    top = padded.abs().amax(2)
    scales = torch.where(top == 0, 1.0, top / LARGEST[case["format"]])
    scaled = (padded * (1 / scales)[:, :, None]).view(rows, -1)[:, :cols]
    if case["format"] == "int8":
        q = torch.floor(scaled + 0.5).to(torch.int8)
    else:
        q = scaled.clamp(-LARGEST[case["format"]], LARGEST[case["format"]]).to(FP8[case["format"]])
    return {"values": _values(q.contiguous(), case), "scales": scales, "residual": h.to(s["x"].dtype)}


def _plain_plan(s):
    page, table, width = s["case"]["page"], s["table"], s["width"]
    cached, new = s["cached"].long(), s["new"].long()
    before, after = (cached + page - 1) // page, (cached + new + page - 1) // page
    offsets = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    fresh = torch.nn.functional.pad((after - before).cumsum(0), (1, 0))
    at = torch.arange(width, device=DEVICE)
    taken = fresh[:-1, None] + at - before[:, None]
    is_fresh = (at >= before[:, None]) & (at < after[:, None])
    table = torch.where(is_fresh, s["free"][taken.clamp(0, max(0, s["free"].numel() - 1))] if s["free"].numel() else table, table)
    row = torch.arange(s["rows"], device=DEVICE)
    used = row < offsets[-1]
    request = torch.searchsorted(offsets, row, right=True).clamp_(max=new.numel()) - 1
    position = cached[request] + row - offsets[request]
    entry = table[request, (position // page).clamp(0, width - 1)].long()
    counts = torch.stack((offsets[-1], offsets[-1], fresh[-1], fresh[-1]))
    return {"table": table, "offsets": offsets.to(torch.int32), "kv_lens": (cached + new).to(torch.int32), "counts": counts.to(torch.int32),
            "positions": torch.where(used, position, -1).to(torch.int32), "slots": torch.where(used, entry * page + position % page, -1)}


def _rotated(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_append(s):
    case = s["case"]
    t, heads, kv_heads, dim, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    kind = TYPES[case["type"]]
    qkv = s["qkv"][:t].float().view(t, heads + 2 * kv_heads, dim)
    position, slot = s["positions"][:t].long(), s["slots"][:t]
    turned = _rotated(qkv[:, :heads + kv_heads], s["cos"][position][:, None], s["sin"][position][:, None], case["interleaved"])
    s["q"][:t] = turned[:, :heads].to(kind)
    s["k_cache"][slot // page, :, slot % page] = turned[:, heads:].to(kind)
    s["v_cache"][slot // page, :, slot % page] = qkv[:, heads + kv_heads:].to(kind)
    return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim, window, longest = case["heads"], case["kv_heads"], case["dim"], case["window"], s["longest"]
    n, group, length = case["requests"], heads // kv_heads, s["width"] * case["page"]
    offsets, kv_lens, new = s["offsets"].long(), s["kv_lens"].long(), s["new"].long()
    pages = s["table"].clamp(min=0).long()
    at, key = torch.arange(longest, device=DEVICE), torch.arange(length, device=DEVICE)
    # rows of a request side by side: [request][kv head][head of the group, new token][dim]
    rows = (offsets[:-1, None] + at).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(n, longest, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * longest, dim)
    k = s["k_cache"][pages].float().transpose(1, 2).reshape(n, kv_heads, length, dim)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(n, kv_heads, group, longest, length)
    del k
    position = kv_lens[:, None] - new[:, None] + at
    seen = key <= position[:, :, None]
    if window:
        seen &= key > position[:, :, None] - window
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = s["v_cache"][pages].float().transpose(1, 2).reshape(n, kv_heads, length, dim)
    v.masked_fill_((key >= kv_lens[:, None])[:, None, :, None], 0)
    o = torch.matmul(scores.view(n, kv_heads, group * longest, length), v).view(n, kv_heads, group, longest, dim)
    o = (o / total.clamp(min=1e-30)).permute(0, 3, 1, 2, 4).reshape(n, longest, heads, dim)
    row = torch.arange(s["tokens"], device=DEVICE)
    request = torch.searchsorted(offsets, row, right=True) - 1
    s["out"][:s["tokens"]] = o[request, row - offsets[request]].to(s["out"].dtype)
    return s["out"]


_PLAIN = {"norm": _plain_norm, "plan": _plain_plan, "append": _plain_append, "attention": _plain_attention}


def _native():
    from tornadovm_b200 import B200Native
    return B200Native


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(s):
    case = s["case"]
    _native().call("tb200_rmsnorm_quant", case["rows"], case["cols"], CODES[case["type"]], s["x"].data_ptr(), case["cols"], s["residual"].data_ptr(),
                   s["summed"].data_ptr(), s["weight"].data_ptr(), s["eps"], FORMATS[case["format"]], case["group"], s["q"].data_ptr(),
                   s["scales"].data_ptr(), _stream())
    return {"values": _values(s["q"], case), "scales": s["scales"], "residual": s["summed"]}


def _own_plan(s):
    _native().call("tb200_paged_plan", s["new"].numel(), s["case"]["page"], s["width"], s["rows"], s["free"].numel(), s["cached"].data_ptr(),
                   s["new"].data_ptr(), s["free"].data_ptr(), s["table"].data_ptr(), s["offsets"].data_ptr(), s["kv_lens"].data_ptr(),
                   s["positions"].data_ptr(), s["slots"].data_ptr(), s["counts"].data_ptr(), _stream())
    return {k: s[k] for k in ("table", "offsets", "kv_lens", "counts", "positions", "slots")}


def _own_append(s):
    case = s["case"]
    heads, kv_heads, dim, width = case["heads"], case["kv_heads"], case["dim"], s["qkv"].shape[1]
    q = s["qkv"].data_ptr()
    k = q + heads * dim * s["qkv"].element_size()
    v = k + kv_heads * dim * s["qkv"].element_size()
    _native().call("tb200_rope_append", s["qkv"].shape[0], heads, kv_heads, dim, CODES[case["in_type"]], q, k, v, width, width, width,
                   s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], case["rot"], int(case["interleaved"]), s["positions"].data_ptr(),
                   CODES[case["type"]], s["q"].data_ptr(), case["page"], s["k_cache"].shape[0], s["slots"].data_ptr(), s["k_cache"].data_ptr(),
                   s["v_cache"].data_ptr(), _stream())
    return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    case, native = s["case"], _native()
    tokens, n, heads, kv_heads, dim = s["q"].shape[0], case["requests"], case["heads"], case["kv_heads"], case["dim"]
    if s["workspace"] is None:
        size = native.load().tb200_paged_attention_workspace_bytes(tokens, n, heads, kv_heads, dim)
        s["workspace"] = torch.empty(max(16, size), device=DEVICE, dtype=torch.uint8)
    native.call("tb200_paged_attention", tokens, n, s["longest"], heads, kv_heads, dim, CODES[case["type"]], s["q"].data_ptr(), heads * dim,
                s["offsets"].data_ptr(), s["kv_lens"].data_ptr(), s["table"].data_ptr(), s["width"], case["page"], s["k_cache"].shape[0],
                s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["scale"], case["window"], s["out"].data_ptr(), heads * dim,
                s["workspace"].data_ptr(), s["workspace"].numel(), _stream())
    return s["out"]


_OWN = {"norm": _own_norm, "plan": _own_plan, "append": _own_append, "attention": _own_attention}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "plan":
        return None  # whole numbers
    return _exact_append(s) if op == "append" else _exact_attention(s)


def _nearest(x, mantissa, lowest):
    """x at `mantissa` bits behind the leading one and steps of 2^lowest at least, half to even."""
    exponent = torch.frexp(x)[1] - 1
    step = torch.exp2((exponent - mantissa).clamp(min=lowest).double())
    return torch.round(x / step) * step


def _exact_norm(s):
    case, top = s["case"], LARGEST[s["case"]["format"]]
    group = case["group"] or case["cols"]
    h = s["x"].double() + s["residual"].double()
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + s["eps"]) * s["weight"].double()
    values, scales = [], []
    for part in y.split(group, dim=1):
        scale = part.abs().max(1, keepdim=True).values / top
        scale[scale == 0] = 1.0
        ratio = part / scale
        q = torch.floor(ratio + 0.5) if case["format"] == "int8" else _nearest(ratio, 3, -9) if case["format"] == "e4m3" else _nearest(ratio, 2, -16)
        values.append(q)
        scales.append(scale)
    return {"values": torch.cat(values, 1), "scales": torch.cat(scales, 1), "residual": h}


def _exact_append(s):
    case = s["case"]
    t, heads, kv_heads, dim, page, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page", "rot"))
    first = torch.arange(0, rot, 2, device=DEVICE) if case["interleaved"] else torch.arange(rot // 2, device=DEVICE)
    second = first + (1 if case["interleaved"] else rot // 2)
    qkv = s["qkv"].double()[:t].view(t, -1, dim)
    angle = s["positions"][:t].long()
    cos, sin = s["cos"].double()[angle].unsqueeze(1), s["sin"].double()[angle].unsqueeze(1)
    turned = qkv.clone()
    both = heads + kv_heads
    turned[:, :both, first] = qkv[:, :both, first] * cos - qkv[:, :both, second] * sin
    turned[:, :both, second] = qkv[:, :both, second] * cos + qkv[:, :both, first] * sin
    q, caches = s["q"].double(), [s["k_cache"].double(), s["v_cache"].double()]
    q[:t] = turned[:, :heads]
    for i, rows in enumerate((turned[:, heads:both], turned[:, both:])):
        flat = caches[i].transpose(1, 2).reshape(-1, kv_heads, dim).contiguous()
        flat[s["slots"][:t]] = rows
        caches[i] = flat.view(-1, page, kv_heads, dim).transpose(1, 2).contiguous()
    return {"q": q, "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attention(s):
    case = s["case"]
    heads, kv_heads, dim, page, window = (case[k] for k in ("heads", "kv_heads", "dim", "page", "window"))
    cached, new = _lengths(case)
    out, group, start = s["out"].double(), heads // kv_heads, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        if not n:
            continue
        total = c + n
        pages = s["table"][r, :-(-total // page)].long()
        last = torch.arange(c, total, device=DEVICE)
        keys = torch.arange(total, device=DEVICE)
        hidden = keys[None, :] > last[:, None]
        if window:
            hidden |= keys[None, :] <= last[:, None] - window
        for g in range(kv_heads):
            k = s["k_cache"][pages, g].reshape(-1, dim)[:total].double()
            v = s["v_cache"][pages, g].reshape(-1, dim)[:total].double()
            for h in range(g * group, (g + 1) * group):
                p = (s["q"][start:start + n, h].double() @ k.T) * s["scale"]
                p = torch.softmax(p.masked_fill(hidden, -math.inf), 1)
                out[start:start + n, h] = p @ v
        start += n
    return out

"""What the operators of a decode step over a 4-bit cache are measured on.

Three operators, each with its plain form (elementary torch operations) and the framework's call:

  write    rotary positions, then keys and values into the pages of a cache held in 4 bits
  attend   causal attention of decoded tokens or of prompt portions over such pages
  sample   the next token's draw: temperature, top-k, top-p, min-p, one given random number a row

The cache: 16 positions of a KV head form a block of bytes, [codes of the keys, 16 rows of D/2 bytes | codes of the values | (step, middle)
of the keys, 16 x D/64 pairs in the 16-bit type | the same of the values]; the low half of a byte is the earlier element; an element stands for
middle + step * (code - 8).  A plane is uint8 [pages, KV heads, page size / 16, bytes of a block].

Fields of a case: kind; dtype; Hq, Hkv, D; page (positions a page); window (0: all keys); requests, of which each has `past_lo` to `past_hi`
cached positions and brings `new_lo` to `new_hi` tokens (both spread evenly, so that lengths are ragged); rope, pairing (write);
rows, vocab, and which filters are set (sample).
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
GROUP = 64                     # elements that share a step and a middle


def _attend(name, dtype, Hq, Hkv, D, requests, past_lo, past_hi, new_lo=1, new_hi=1, page=16, window=0):
    return {"name": name, "kind": "attend", "dtype": dtype, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "window": window, "requests": requests,
            "past_lo": past_lo, "past_hi": past_hi, "new_lo": new_lo, "new_hi": new_hi}


def _write(name, dtype, Hq, Hkv, D, requests, past_lo, past_hi, new_lo, new_hi, page=16, rope=None, pairing=1):
    return {"name": name, "kind": "write", "dtype": dtype, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "requests": requests, "past_lo": past_lo,
            "past_hi": past_hi, "new_lo": new_lo, "new_hi": new_hi, "rope": D if rope is None else rope, "pairing": pairing}


def _sample(name, rows, vocab, top_k, top_p, min_p):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # one decoded token of an 8B model joins the cache: latency
        _write("write_token", "bfloat16", 32, 8, 128, 1, 700, 700, 1, 1),
        # 64 requests decode, half of each head rotated, adjacent pairs
        _write("write_batch64_half", "float16", 32, 8, 64, 64, 10, 5000, 1, 1, page=32, rope=32, pairing=0),
        # a whole prompt portion
        _write("write_prompt2048", "bfloat16", 32, 8, 128, 1, 0, 0, 2048, 2048),
        # one chat answer, short context: latency
        _attend("decode_1x700", "bfloat16", 32, 8, 128, 1, 700, 700),
        # one long document: the keys of eight heads have to be spread over the whole GPU
        _attend("decode_1x131000", "bfloat16", 32, 8, 128, 1, 131000, 131000, page=64),
        # every query head has a KV head of its own
        _attend("decode_8x2048_heads32", "float16", 32, 32, 128, 8, 1500, 2500),
        # ragged contexts, a window, small heads, three tokens a request (drafted tokens to be checked)
        _attend("decode_17_ragged_window", "float16", 32, 8, 64, 17, 0, 6000, new_lo=1, new_hi=4, window=2000),
        # a full batch at long contexts
        _attend("decode_64x8192", "bfloat16", 32, 8, 128, 64, 8192, 8192),
        # a prompt portion from the start
        _attend("prompt_2048", "bfloat16", 32, 8, 128, 1, 0, 0, new_lo=2048, new_hi=2048),
        # portions of five prompts behind what is cached already
        _attend("prompt_5_ragged", "float16", 24, 8, 128, 5, 0, 3500, new_lo=37, new_hi=500, page=32),
        # one request's draw
        _sample("sample_1x128256", 1, 128256, True, True, False),
        # a full batch's draws, each row with filters of its own
        _sample("sample_64x128256", 64, 128256, True, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "sample"])
    dtype = rng.choice(["bfloat16", "float16"])
    if kind == "sample":
        case = _sample("", _log(rng, 1, 64), _log(rng, 300, 150000), rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.5)
    else:
        D = rng.choice([64, 128])
        Hkv, G = rng.choice([1, 2, 3, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
        page = rng.choice([16, 16, 32, 48, 64])
        if kind == "write":
            requests = _log(rng, 1, 64)
            new = _log(rng, 1, max(1, 2048 // requests))
            past = _log(rng, 1, 8000)
            case = _write("", dtype, Hkv * G, Hkv, D, requests, rng.randrange(past), past, rng.randrange(new) + 1, new, page,
                          D // rng.choice([1, 1, 2, 4]), rng.choice([0, 1]))
        elif rng.random() < 0.7:                       # decoded tokens, or a few drafted ones
            requests = _log(rng, 1, 64)
            past = _log(rng, 1, min(100000, 64 * 8192 * 8 // (requests * Hkv)))
            new = 1 if rng.random() < 0.7 else max(1, 16 // G)
            case = _attend("", dtype, Hkv * G, Hkv, D, requests, rng.randrange(past), past, 1, new, page, rng.choice([0, 0, 0, _log(rng, 1, 4000)]))
        else:
            requests = rng.randrange(5) + 1
            new = _log(rng, 1, 1500 // requests)
            past = _log(rng, 1, 4000)
            case = _attend("", dtype, Hkv * G, Hkv, D, requests, rng.randrange(past), past, rng.randrange(new) + 1, new, page,
                           rng.choice([0, 0, _log(rng, 1, 4000)]))
    del case["name"]
    return case


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(cached positions, new tokens) of every request."""
    n = case["requests"]
    return _spread(case["past_lo"], case["past_hi"], n), _spread(case["new_lo"], case["new_hi"], n)


def _quantise(x, dtype):
    """x float32 [..., D] -> (codes uint8 [..., D/2], pairs (step, middle) of the 16-bit type [..., D/64, 2])."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = (hi / 15 - lo / 15).to(dtype)
    middle = (lo + 8 * step.float()).to(dtype)
    wrong = ~torch.isfinite(g).all(-1, keepdim=True)
    step, middle = (t.masked_fill(wrong, math.nan) for t in (step, middle))
    code = (torch.round((g - middle.float()) / step.float()) + 8).clamp(0, 15)
    code = torch.where((step == 0) | wrong, 8.0, code).to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.cat([step, middle], -1)


def _values(blocks, D, dtype):
    """uint8 [..., bytes of a block] -> float32 [..., 2 (keys, values), 16, D]."""
    codes = blocks[..., :16 * D].unflatten(-1, (2, 16, D // 2))
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8
    pairs = blocks[..., 16 * D:].contiguous().view(dtype).float().unflatten(-1, (2, 16, D // GROUP, 2))
    return (pairs[..., 1:] + pairs[..., :1] * code.unflatten(-1, (-1, GROUP))).flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    if case["kind"] == "sample":
        n, V = case["rows"], case["vocab"]
        # a language model's logits: most of the mass on some tokens, a long tail; whole steps of 1/16 make ties
        logits = torch.round((2.5 * rand(n, V) + 3.0 * rand(n, V).clamp(min=2.2)) * 16) / 16
        uni = lambda lo, hi: lo + (hi - lo) * torch.rand(n, device="cuda", generator=g)
        some = lambda t, off: torch.where(torch.rand(n, device="cuda", generator=g) < 0.8, t, torch.full_like(t, off))
        k = torch.exp(uni(0.0, math.log(min(V, 400)))).to(torch.int32)
        return {"case": case, "logits": logits, "temperature": uni(0.5, 1.5),
                "top_k": some(k, 0) if case["top_k"] else torch.zeros_like(k),
                "top_p": some(uni(0.5, 0.99), 1.0) if case["top_p"] else torch.ones(n, device="cuda"),
                "min_p": some(uni(0.0, 0.1), 0.0) if case["min_p"] else torch.zeros(n, device="cuda"),
                "uniform": torch.rand(n, device="cuda", generator=g, dtype=torch.float64),
                "ids": torch.empty(n, dtype=torch.int32, device="cuda"), "err": torch.zeros(1, dtype=torch.int32, device="cuda")}
    dtype, Hq, Hkv, D, page = DTYPES[case["dtype"]], case["Hq"], case["Hkv"], case["D"], case["page"]
    past, new = _lengths(case)
    total = [p + n for p, n in zip(past, new)]
    R, T = len(new), sum(new)
    held = [-(-n // page) for n in total]
    width = max(held)
    # the pages of a request lie scattered, as they do once requests have come and gone
    order = torch.randperm(sum(held), generator=torch.Generator().manual_seed(seed)).to(torch.int32).tolist()
    ends = torch.tensor(held).cumsum(0).tolist()
    tables = [order[e - n:e] for e, n in zip(ends, held)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    state = {"case": case, "qkv": rand(T, (Hq + 2 * Hkv) * D).to(dtype), "table": i32([t + [-1] * (width - len(t)) for t in tables]),
             "q_start": i32([0] + torch.tensor(new).cumsum(0).tolist()), "past": i32(past), "new": i32(new),
             "position": i32([p + i for p, n in zip(past, new) for i in range(n)]), "request": i32([r for r, n in enumerate(new) for _ in range(n)]),
             "err": torch.zeros(1, dtype=torch.int32, device="cuda")}
    n_blocks = page // 16
    if case["kind"] == "write":
        rope = case["rope"]
        angle = torch.arange(width * page, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, rope, 2, dtype=torch.float64, device="cuda") / rope)
        state["cos_sin"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        state["plane"] = torch.zeros(len(order), Hkv, n_blocks, 18 * D, dtype=torch.uint8, device="cuda")
        # the pages that receive tokens, as (request, page of the request)
        state["pages"] = i32([[r, j] for r, (p, n) in enumerate(zip(past, new)) for j in range(p // page, (p + n - 1) // page + 1)])
        state["q_out"] = torch.empty(T, Hq * D, dtype=dtype, device="cuda")
        state["values"] = torch.empty(state["pages"].shape[0], 2, Hkv, page, D, dtype=dtype, device="cuda")
        return state
    plane = torch.empty(len(order), Hkv, n_blocks, 18 * D, dtype=torch.uint8, device="cuda")
    kv = rand(len(order), Hkv, n_blocks, 2, 16, D)
    kv[..., 0, :, :] += rand(1, Hkv, 1, 1, D)                  # keys have channels that stand off for all positions
    codes, pairs = _quantise(kv, dtype)
    plane[..., :16 * D] = codes.flatten(-3)
    plane[..., 16 * D:] = pairs.flatten(-4).view(torch.uint8)
    state["plane"] = plane
    if own:
        from ferrum_b200.cache.storage import LayerCache
        from ferrum_b200.engine.batch import StepContext, StepEntry
        from ferrum_b200.parts.attention import PagedAttention
        mixer = PagedAttention(Hq * D, Hq, Hkv, D, None, dtype, window=case["window"])
        mixer.set_cache_bits(4)
        ctx = StepContext("cuda", T, R, [width])
        ctx.fill([StepEntry(r, p, [0] * n) for r, (p, n) in enumerate(zip(past, new))], [tables])
        cache = LayerCache(group=0, plane=plane, page_stride=plane.stride(0), page_size=page, writes=True, state=None)
        state.update(mixer=mixer, ctx=ctx, cache=cache, out=torch.empty(T, Hq * D, dtype=dtype, device="cuda"))
    return state


def run(state):
    case = state["case"]
    return {"write": _run_write, "attend": _run_attend, "sample": _run_sample}[case["kind"]](state, case)


def _run_write(s, case):
    Hq, Hkv, D, page, rope = case["Hq"], case["Hkv"], case["D"], case["page"], case["rope"]
    T, dtype, plane = s["qkv"].shape[0], s["qkv"].dtype, s["plane"]
    if own:
        from ferrum_b200.ops import lib as ops
        ops.rope_cache_write_packed(s["qkv"], T, s["position"], s["request"], s["table"], s["cos_sin"], plane, plane.stride(0), page, Hq, Hkv, D,
                                    rope, case["pairing"], s["err"], q_out=s["q_out"])
        ops.unpack_cache(plane, plane.stride(0), page, s["table"], s["pages"], s["values"], s["err"])
        return {"q": s["q_out"], "values": s["values"]}
    x = s["qkv"].float().view(T, Hq + 2 * Hkv, D)
    at = s["position"].long()
    cos, sin = s["cos_sin"][at][:, None].unbind(-1)
    turned = x[:, :Hq + Hkv, :rope]
    a, b = (turned[..., ::2], turned[..., 1::2]) if case["pairing"] == 0 else turned.chunk(2, -1)
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if case["pairing"] == 0 else torch.cat([a, b], -1)
    qk = torch.cat([turned, x[:, :Hq + Hkv, rope:]], -1)
    codes, pairs = _quantise(torch.stack([qk[:, Hq:], x[:, Hq + Hkv:]], 1), dtype)          # [T, 2, Hkv, ...]
    low, high = codes & 15, codes >> 4
    code = torch.stack([low, high], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float() - 8
    rows = (pairs[..., 1:].float() + pairs[..., :1].float() * code).flatten(-2).to(dtype)
    pages, values = s["pages"].long(), torch.zeros_like(s["values"])
    index = torch.full(s["table"].shape, -1, device="cuda")
    index[pages[:, 0], pages[:, 1]] = torch.arange(pages.shape[0], device="cuda")
    values[index[s["request"].long(), at // page], :, :, at % page] = rows
    return {"q": qk[:, :Hq].reshape(T, Hq * D).to(dtype), "values": values}


def _run_attend(s, case):
    if own:
        s["mixer"].attend(s["qkv"], s["out"], s["ctx"], s["cache"])
        return s["out"]
    Hq, Hkv, D, page, window = case["Hq"], case["Hkv"], case["D"], case["page"], case["window"]
    dtype, T, R = s["qkv"].dtype, s["qkv"].shape[0], s["past"].shape[0]
    kv = _values(s["plane"][s["table"].long().clamp(min=0)], D, dtype)                       # [R, pages, Hkv, blocks, 2, 16, D]
    kv = kv.permute(0, 4, 2, 1, 3, 5, 6).reshape(R, 2, Hkv, -1, D)
    K, V, L = kv[:, 0], kv[:, 1], kv.shape[3]
    most = int(case["new_hi"])
    slot = torch.arange(T, device="cuda") - s["q_start"].long()[s["request"].long()]
    q = torch.zeros(R, most, Hq, D, device="cuda")
    q[s["request"].long(), slot] = s["qkv"][:, :Hq * D].float().view(T, Hq, D)
    q = q.view(R, most, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, -1, D)     # rows: (head of the group, token)
    scores = (q @ K.transpose(-1, -2)).mul_(D ** -0.5).view(R, Hkv, -1, most, L)
    at = s["past"].long()[:, None] + torch.arange(most, device="cuda")                       # [R, tokens]
    key = torch.arange(L, device="cuda")
    hidden = key > at[..., None]
    if window:
        hidden |= key <= at[..., None] - window
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    out = (p.view(R, Hkv, -1, L) @ V) / p.sum(-1).view(R, Hkv, -1, 1)
    out = out.view(R, Hkv, -1, most, D).permute(0, 3, 1, 2, 4).reshape(R, most, Hq * D)
    return out[s["request"].long(), slot].to(dtype)


def _run_sample(s, case):
    if own:
        from ferrum_b200.ops import lib as ops
        ops.sample_filtered(s["logits"], case["rows"], s["ids"], s["err"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"])
        return s["ids"]
    V = case["vocab"]
    x, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    w = ((x.double() - x[:, :1].double()) / s["temperature"].double()[:, None]).exp()
    rank = torch.arange(V, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], V).long()[:, None]
    keep = rank < k
    before = (w * keep).cumsum(-1)
    total = before[:, -1:].clone()
    before = before - w
    p = s["top_p"].double()[:, None]
    keep &= (before < p * total) | (p >= 1)
    keep &= w >= s["min_p"].double()[:, None]
    mass = torch.zeros_like(w).scatter_(1, order, w * keep).cumsum(-1)
    return (mass > s["uniform"][:, None] * mass[:, -1:]).to(torch.uint8).argmax(-1).to(torch.int32)


def work(case):
    if case["kind"] == "sample":
        n, V = case["rows"], case["vocab"]
        return {"bytes": n * (V * 4 + 28), "flops": 12.0 * n * V}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    past, new = _lengths(case)
    T = sum(new)
    if case["kind"] == "write":
        return {"bytes": T * (2 * (2 * Hq + 2 * Hkv) * D + Hkv * 9 * D // 8 + 4 * case["rope"]), "flops": T * (3.0 * (Hq + Hkv) * case["rope"] + 12.0 * Hkv * D)}
    w = case["window"] or (1 << 40)
    keys = sum(min(p + n, w + n - 1) for p, n in zip(past, new))
    pairs = sum(min(p + i + 1, w) for p, n in zip(past, new) for i in range(n))
    return {"bytes": keys * Hkv * 9 * D // 8 + 4 * T * Hq * D, "flops": 4.0 * pairs * Hq * D}


def exact(case, seed):
    """The definitions in 64 bits, request by request; ids have no rounding to be held against, nor do stored values: each is one of 16 levels."""
    if case["kind"] == "sample":
        return None
    s = prepare(case, seed)
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    past, new = _lengths(case)
    if case["kind"] == "write":
        half, out, row = case["rope"] // 2, s["qkv"][:, :Hq * D].double().view(-1, Hq, D).clone(), 0
        at = s["position"].double()
        src = out.clone()
        for i in range(half):
            c, z = (t[:, None] for t in s["cos_sin"][s["position"].long(), i].double().unbind(-1))
            a, b = (2 * i, 2 * i + 1) if case["pairing"] == 0 else (i, i + half)
            out[:, :, a], out[:, :, b] = src[:, :, a] * c - src[:, :, b] * z, src[:, :, a] * z + src[:, :, b] * c
        return {"q": out.view(len(at), Hq * D), "values": None}
    n_blocks, row, outs = page // 16, 0, []
    for r, (p, n) in enumerate(zip(past, new)):
        L = p + n
        pages = s["plane"][s["table"][r, :-(-L // page)].long()]                             # [pages, Hkv, blocks, bytes]
        def plane_of(part):
            codes = pages[..., part * 8 * D:(part + 1) * 8 * D].reshape(-1, Hkv, n_blocks, 16, D // 2).to(torch.int16)
            level = torch.empty(codes.shape[:-1] + (D,), dtype=torch.float64, device="cuda")
            level[..., 0::2], level[..., 1::2] = (codes % 16 - 8).double(), (codes // 16 - 8).double()
            size = 16 * (D // GROUP) * 4
            start = 16 * D + part * size
            pair = pages[..., start:start + size].contiguous().view(s["qkv"].dtype).double().reshape(-1, Hkv, n_blocks, 16, D // GROUP, 2)
            level *= pair[..., 0].repeat_interleave(GROUP, -1)
            level += pair[..., 1].repeat_interleave(GROUP, -1)
            return level.permute(1, 0, 2, 3, 4).reshape(Hkv, -1, D)[:, :L]
        K, V = plane_of(0), plane_of(1)
        q = s["qkv"][row:row + n, :Hq * D].double().view(n, Hq, D)
        out = torch.empty(n, Hq, D, dtype=torch.float64, device="cuda")
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            dots = q[:, h] @ K[kv].T / math.sqrt(D)
            where = torch.arange(L, device="cuda")[None] - (p + torch.arange(n, device="cuda"))[:, None]
            seen = where <= 0
            if case["window"]:
                seen &= where > -case["window"]
            dots = torch.where(seen, dots, torch.full_like(dots, -math.inf))
            out[:, h] = torch.softmax(dots, -1) @ V[kv]
        outs.append(out.view(n, Hq * D))
        row += n
    return torch.cat(outs)

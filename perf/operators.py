"""The operators of serving from a paged 4-bit key/value cache, as they are measured: block tables and
slot maps from request lengths, the norms and rotation of queries and keys with the write into the
cache, and the attention that reads it. `run` computes them in elementary torch operations, or with
`own` through the framework's entry points (webpytorch_b200.kv4).

The cache is uint8 [pages, NKV, page / 16, block]: a block holds 16 positions of one key/value head,
    K codes [16][HD / 2] | K scales [16][HD / G] | V codes [16][HD / 2] | V scales [16][HD / G],
two codes to a byte (the lower nibble is the even element), and for each group of G elements a pair of
halves (s, m). A code n stands for half(s * n + m). Slot i is position i % page of page i / page.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small server: 8 requests, one new token each
        _plan("plan 8 decoding", 8, 4096, 16, 8, 0.0, 0.0),
        # a busy step: some requests end, some begin with prompts, the others decode
        _plan("plan 1000 mixed", 1000, 8192, 16, 20000, 0.1, 0.1),
        # a whole pool planned at once: long requests, a step of 256 Ki tokens, more asked than fits
        _plan("plan 6000 long", 6000, 32768, 64, 262144, 0.2, 0.05),
        # the decode step of the framework's 28-layer stack: fp32 activations, no norms of heads
        _rope("rope 1 token f32", 1, 28, 4, 128, 128, 16, 64, "f32", False, 0),
        # a step of 48 requests of a model with norms for each head, the finest groups
        _rope("rope 48 tokens bf16", 48, 32, 4, 128, 128, 16, 32, "bf16", True, 0),
        # small heads of which half the dimensions are rotated, rows wider than the heads
        _rope("rope 1999 half heads f16", 1999, 14, 2, 64, 32, 32, 64, "f16", True, 128),
        # a prompt of 16 Ki tokens
        _rope("rope 16384 tokens bf16", 16384, 32, 8, 128, 128, 64, 64, "bf16", True, 0),
        # one request in the middle of its answer, fp32 as in the decode stack
        _attn("attn 1 x 513 f32", "f32", 1, 28, 4, 128, 16, 64, 513, 513, 1, 1, 0),
        # a batch of requests of very different lengths
        _attn("attn 96 ragged bf16", "bf16", 96, 32, 8, 128, 16, 64, 200, 12000, 1, 1, 0),
        # one long document
        _attn("attn 1 x 131071 bf16", "bf16", 1, 28, 4, 128, 64, 128, 131071, 131071, 1, 1, 0),
        # many requests, a key/value head for each query head, a sliding window
        _attn("attn 250 windowed f16", "f16", 250, 16, 16, 64, 32, 32, 300, 4000, 1, 1, 1024),
        # chunks of two prompts on top of what is cached
        _attn("attn prompts bf16", "bf16", 2, 32, 4, 128, 64, 64, 2500, 6000, 900, 2000, 0),
    ]


def _plan(name, requests, longest, page, tokens, prompts, ended):
    return {"name": name, "op": "plan", "requests": requests, "longest": longest, "page": page, "tokens": tokens,
            "prompts": prompts, "ended": ended}


def _rope(name, tokens, nh, nkv, hd, rot, page, group, dtype, norm, pad):
    return {"name": name, "op": "rope", "tokens": tokens, "nh": nh, "nkv": nkv, "hd": hd, "rot": rot, "page": page,
            "group": group, "dtype": dtype, "norm": norm, "pad": pad}


def _attn(name, dtype, requests, nh, nkv, hd, page, group, len_lo, len_hi, q_lo, q_hi, window):
    return {"name": name, "op": "attn", "dtype": dtype, "requests": requests, "nh": nh, "nkv": nkv, "hd": hd,
            "page": page, "group": group, "len_lo": len_lo, "len_hi": len_hi, "q_lo": q_lo, "q_hi": q_hi,
            "window": window}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64])
    if op == "plan":
        n = _log(rng, 1, 6000)
        c = _plan("", n, _log(rng, 64, 32768), page, n + _log(rng, 1, 200000), rng.uniform(0, 0.3), rng.uniform(0, 0.2))
    else:
        nh, nkv = rng.choice([(28, 4), (32, 8), (32, 4), (14, 2), (16, 16), (16, 2), (8, 1), (40, 8), (64, 4)])
        hd = rng.choice([64, 128, 128, 256])
        group = rng.choice([g for g in (32, 64, 128) if g <= hd])
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        if op == "rope":
            c = _rope("", min(_log(rng, 1, 16384), (1 << 26) // ((nh + 2 * nkv) * hd)), nh, nkv, hd,
                      rng.choice([hd, hd, hd // 2]), page, group, dtype, rng.random() < 0.7, rng.choice([0, 0, 64]))
        else:
            kind = rng.choice(["decode", "decode", "decode", "few", "prompt"])
            if kind == "prompt":
                q_hi = _log(rng, 17, 2000)
                hi = min(_log(rng, q_hi, 6000), 250000 // (q_hi * nh * hd // 8192 + 40))
                hi = max(hi, q_hi)
                n = rng.randint(1, 2)
                q_lo = max(1, q_hi // 2)
            else:
                q_lo, q_hi = (1, 1) if kind == "decode" else (1, rng.randint(2, 16))
                hi = _log(rng, 16, 131071)
                n = max(1, min(_log(rng, 1, 250), 250000 * 1024 // (hi * nkv * hd)))
            c = _attn("", dtype, n, nh, nkv, hd, page, group, max(q_hi, hi // 20), hi, q_lo, q_hi,
                      rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------
# what a user's program has in hand
# --------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _lens(n, lo, hi, g):
    """n lengths of lo to hi, spread over their logarithm; the longest is hi."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    x = torch.exp(math.log(lo) + u * (math.log(hi) - math.log(lo))).round().to(torch.int32).clamp_(lo, hi)
    x[0] = hi
    return x


def _block_bytes(hd, group):
    return 16 * (hd + 8 * (hd // group))


def _tables(n, pages, held, width, g):
    """Block tables of n requests that hold held[b] of the pages in a shuffled pool, and the pages that are free."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    start = torch.cumsum(held, 0) - held
    col = torch.arange(width, device="cuda")
    mine = col[None, :] < held[:, None]
    at = (start[:, None] + col[None, :]).clamp(max=pages - 1)
    return torch.where(mine, order[at], torch.full_like(at, -1, dtype=torch.int32)).contiguous(), order


def prepare(case, seed):
    c, g = case, _gen(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn}[c["op"]](c, g)


def _prepare_plan(c, g):
    n, page = c["requests"], c["page"]
    prev = _lens(n, 1, c["longest"], g)
    kind = torch.rand(n, generator=g, device="cuda")
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    prompt = _lens(n, 1, max(1, c["longest"] // 2), g)
    first = kind < c["prompts"]
    prev = torch.where(first, torch.zeros_like(prev), prev)
    new = torch.where(first, prompt, new)
    new = torch.where(kind > 1 - c["ended"], torch.full_like(new, -1), new)
    held = ((prev + page - 1) // page).long()
    width = (c["longest"] + page - 1) // page + 1
    used, left = int(held.sum()), n // 2 + c["tokens"] // page // 2 + 1
    table, order = _tables(n, used + left, held, width, g)
    free = torch.zeros(n * width + left, dtype=torch.int32, device="cuda")
    free[:left] = order[used:]
    return {"case": c, "prev": prev, "new": new, "table": table, "free": free,
            "n_free": torch.tensor([left], dtype=torch.int32, device="cuda")}


def _rope_tables(lmax, rot):
    inv = 1.0 / (1e6 ** (torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
    ang = torch.arange(lmax, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()


def _prepare_rope(c, g):
    t, nh, nkv, hd, page = c["tokens"], c["nh"], c["nkv"], c["hd"], c["page"]
    width = (nh + 2 * nkv) * hd
    gain = torch.exp(0.4 * torch.randn(width, generator=g, device="cuda"))
    gain = torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, gain * 8, gain)   # outlier channels
    x = torch.randn(t, width + c["pad"], generator=g, device="cuda")
    x[:, :width] *= gain
    x = x.to(_T[c["dtype"]])[:, :width]
    cos, sin = _rope_tables(32768, c["rot"])
    pos = torch.randint(0, 32768, (t,), generator=g, device="cuda", dtype=torch.int32)
    pages = (t + page - 1) // page + 3
    slots = torch.randperm((pages - 1) * page, generator=g, device="cuda")[:t]
    if t > 16:                                    # the step's tail is padding
        slots[-5:] = -1
        pos[-5:] = -1
    weights = [(1 + 0.3 * torch.randn(hd, generator=g, device="cuda")) if c["norm"] else None for _ in range(2)]
    data = torch.zeros(pages, nkv, page // 16, _block_bytes(hd, c["group"]), dtype=torch.uint8, device="cuda")
    return {"case": c, "x": x, "cos": cos, "sin": sin, "pos": pos, "slots": slots, "wq": weights[0], "wk": weights[1],
            "data": data}


def _prepare_attn(c, g):
    n, nh, nkv, hd, page, group = (c[k] for k in ("requests", "nh", "nkv", "hd", "page", "group"))
    lens = _lens(n, c["len_lo"], c["len_hi"], g)
    ql = torch.linspace(c["q_lo"], c["q_hi"], n, device="cuda").round().to(torch.int32)
    ql = ql[torch.randperm(n, generator=g, device="cuda")]
    held = ((lens + page - 1) // page).long()
    pages = int(held.sum()) + 8
    table, _ = _tables(n, pages, held, int(held.max()) + 1, g)
    nb, half = page // 16, 8 * hd
    data = torch.randint(0, 256, (pages, nkv, nb, _block_bytes(hd, group)), generator=g, device="cuda",
                         dtype=torch.uint8)
    ng = hd // group
    for at in (half, 2 * half + 64 * ng):         # keys, then values: scales and minima of the groups
        s = 0.1 + 0.25 * torch.rand(pages, nkv, nb, 16 * ng, generator=g, device="cuda")
        m = -7.5 * s + 0.2 * torch.randn(pages, nkv, nb, 16 * ng, generator=g, device="cuda")
        data[..., at:at + 64 * ng] = torch.stack([s, m], -1).half().flatten(-2).view(torch.uint8)
    cu = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(ql, 0)
    q = (1.5 * torch.randn(int(cu[-1]), nh, hd, generator=g, device="cuda")).to(_T[c["dtype"]])
    return {"case": c, "q": q, "data": data, "table": table, "lens": lens, "cu": cu if c["q_hi"] > 1 else None,
            "q_max": int(ql.max()), "l_max": int(lens.max())}


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn}[c["op"]](c, state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn}[c["op"]](c, state)


def _cache(c, state):
    """The cache as the framework holds it, made once over the state's own memory."""
    if "cache" not in state:
        from webpytorch_b200 import kv4
        state["kv4"] = kv4
        state["cache"] = kv4.KV4Cache(state["data"].shape[0], c["nkv"], c["hd"], page=c["page"], group=c["group"],
                                      data=state["data"])
    return state["cache"]


def _own_plan(c, s):
    if "kv4" not in s:
        from webpytorch_b200 import kv4
        s["kv4"] = kv4
    p = s["kv4"].plan(s["prev"], s["new"], s["table"], s["free"], s["n_free"], c["page"], c["tokens"])
    return {"table": s["table"], "free": s["free"], "n_free": p.n_free, "lens": p.seq_lens, "cu": p.cu_new,
            "slots": p.slots, "positions": p.positions, "requests": p.requests}


def _own_rope(c, s):
    cache = _cache(c, s)
    q, _ = s["kv4"].qk_norm_rope(s["x"], c["nh"], c["nkv"], c["hd"], s["pos"], s["cos"], s["sin"], q_weight=s["wq"],
                                 k_weight=s["wk"], eps=1e-6, cache=cache, slots=s["slots"])
    k, v = cache.read(s["slots"])
    return {"q": q, "k": k, "v": v}


def _own_attn(c, s):
    cache = _cache(c, s)
    return {"o": s["kv4"].attention(s["q"], cache, s["table"], s["lens"], s["cu"], window=c["window"])}


# ---- plain: the plan ------------------------------------------------------------------------
def _plain_plan(c, s):
    page, cap = c["page"], c["tokens"]
    prev, new, table, free = s["prev"].long(), s["new"].long(), s["table"], s["free"]
    n, width = table.shape
    size = free.shape[0]
    n_free = s["n_free"].long()
    held = (prev + page - 1) // page
    over = new < 0
    want = torch.where(over, torch.zeros_like(new), prev + new)
    pages = (want + page - 1) // page
    fits = ~over & (pages <= width) & (held <= width)
    back = torch.where(over, held.clamp(max=width), torch.zeros_like(held))
    back_end = torch.cumsum(back, 0)
    avail = (n_free + back_end[-1:]).clamp(max=size)
    need = torch.where(fits, pages - held, torch.zeros_like(held))
    tok = torch.where(fits, new, torch.zeros_like(new))
    need_end, tok_end = torch.cumsum(need, 0), torch.cumsum(tok, 0)
    served = fits & (tok_end <= cap) & ((need == 0) | (need_end <= avail))
    put = torch.where(served, tok, torch.zeros_like(tok))
    cu = torch.cat([torch.zeros_like(put[:1]), torch.cumsum(put, 0)])
    lens = torch.where(over, torch.zeros_like(prev), torch.where(served, prev + new, prev))
    left = avail - torch.where(served, need, torch.zeros_like(need)).sum()
    # pages of requests that end go back on the stack, pages asked for come off its top
    col = torch.arange(width, device=table.device)[None, :]
    goes = over[:, None] & (col < back[:, None])
    to = torch.where(goes, n_free + (back_end - back)[:, None] + col, torch.full_like(col, size)).clamp(max=size)
    stack = torch.cat([free, free[:1]])
    stack[to.reshape(-1)] = table.reshape(-1)
    free.copy_(stack[:size])
    gets = served[:, None] & (col >= held[:, None]) & (col < pages[:, None])
    at = (avail - 1 - ((need_end - need) - held)[:, None] - col).clamp(0, size - 1)
    table.copy_(torch.where(gets, free[at], table))
    t = torch.arange(cap, device=table.device)
    r = torch.searchsorted(cu[1:], t, right=True)
    live = r < n
    r = r.clamp(max=n - 1)
    pos = prev[r] + t - cu[r]
    slot = table[r, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    none = torch.full_like(t, -1)
    return {"table": table, "free": free, "n_free": left.int(), "lens": lens.int(), "cu": cu.int(),
            "slots": torch.where(live, slot, none), "positions": torch.where(live, pos, none).int(),
            "requests": torch.where(live, r, none).int()}


# ---- plain: norms, rotation, and the write in 4 bits ------------------------------------------
def _tree_sum(x):
    """The sum over the last axis as a balanced tree of neighbours. Codes of 4 bits have to come out the same
    wherever they are made, so the order of the sum under them is part of the operator."""
    return x if x.shape[-1] == 1 else _tree_sum(x[..., 0::2] + x[..., 1::2])


def _norm_rotate(x, w, cos, sin, eps):
    if w is not None:
        r = 1.0 / torch.sqrt(_tree_sum(x * x) * (1.0 / x.shape[-1]) + eps)
        x = (x * r) * w
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _quantise(x, group):
    """Codes of x [..., HD] and the (s, m) of its groups."""
    y = x.unflatten(-1, (-1, group))
    lo, hi = y.amin(-1), y.amax(-1)
    s, m = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    d = (y - m.float()[..., None]) / torch.where(s == 0, torch.ones_like(s), s).float()[..., None]
    n = torch.where(s[..., None] == 0, torch.zeros_like(d), torch.round(d).clamp(0, 15))
    return n, s, m


def _values(n, s, m):
    return (s.float()[..., None] * n + m.float()[..., None]).half().flatten(-2)


def _parts(data, hd, group):
    """Views of the cache's keys and values: (codes [pages, NKV, blocks, 16, HD / 2], scales [..., 16, HD / G * 4] bytes)."""
    half, sc = 8 * hd, 64 * (hd // group)
    cut = lambda at, size: data[..., at:at + size].unflatten(-1, (16, size // 16))  # noqa: E731
    return (cut(0, half), cut(half, sc)), (cut(half + sc, half), cut(2 * half + sc, sc))


def _plain_rope(c, s):
    nh, nkv, hd, page, group = c["nh"], c["nkv"], c["hd"], c["page"], c["group"]
    x = s["x"].float().unflatten(-1, (nh + 2 * nkv, hd))
    pos = s["pos"].long()
    live = (pos >= 0)[:, None, None]
    cos, sin = s["cos"][pos.clamp(min=0)][:, None], s["sin"][pos.clamp(min=0)][:, None]
    q = _norm_rotate(x[:, :nh], s["wq"], cos, sin, 1e-6)
    k = _norm_rotate(x[:, nh:nh + nkv], s["wk"], cos, sin, 1e-6)
    # a row without a slot goes to the last page, which is nobody's
    slot = torch.where(s["slots"] < 0, torch.full_like(s["slots"], (s["data"].shape[0] - 1) * page), s["slots"])
    at = (slot // page, slice(None), slot % page // 16, slot % 16)
    out = {"q": torch.where(live, q, torch.zeros_like(q)).to(s["x"].dtype)}
    for name, y, (codes, scales) in zip("kv", (k, x[:, nh + nkv:]), _parts(s["data"], hd, group)):
        n, sc, m = _quantise(y, group)
        pair = n.flatten(-2).to(torch.uint8)
        codes[at] = pair[..., 0::2] | (pair[..., 1::2] << 4)
        scales[at] = torch.stack([sc, m], -1).flatten(-2).view(torch.uint8)
        out[name] = torch.where((s["slots"] >= 0)[:, None, None], _values(n, sc, m), torch.zeros((), dtype=torch.half,
                                                                                               device=y.device))
    return out


# ---- plain: attention -------------------------------------------------------------------------
def _decode(codes, scales):
    """The values that gathered codes [..., HD / 2] and their scales' bytes stand for, in 32 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    sm = scales.contiguous().view(torch.half).unflatten(-1, (-1, 2))
    n = n.unflatten(-1, (sm.shape[-2], -1)).float()
    return _values(n, sm[..., 0], sm[..., 1]).float()


def _plain_attn(c, s):
    nh, nkv, hd, page, group = c["nh"], c["nkv"], c["hd"], c["page"], c["group"]
    lens, dev = s["lens"].long(), s["q"].device
    b, width, qm = lens.shape[0], (s["l_max"] + page - 1) // page, s["q_max"]
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(b + 1, device=dev)
    table = s["table"][:, :width].long().clamp(min=0)
    kv = []
    for codes, scales in _parts(s["data"], hd, group):
        x = _decode(codes[table], scales[table])                      # [b, width, nkv, blocks, 16, hd]
        kv.append(x.permute(0, 2, 1, 3, 4, 5).reshape(b, nkv, width * page, hd))
    i = torch.arange(qm, device=dev)
    ql = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().unflatten(2, (nkv, nh // nkv)).permute(0, 2, 3, 1, 4)       # [b, nkv, group, qm, hd]
    z = torch.matmul(q.flatten(2, 3), kv[0].transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    z = z.unflatten(2, (nh // nkv, qm))
    at = (lens - ql)[:, None] + i                                      # positions of the queries
    p = torch.arange(width * page, device=dev)
    see = (p <= at[..., None]) & (p < lens[:, None, None])
    if c["window"]:
        see = see & (p > at[..., None] - c["window"])
    z = torch.where(see[:, None, None], z, torch.full((), -math.inf, device=dev))
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    den = e.sum(-1, keepdim=True)
    o = torch.matmul(e.flatten(2, 3), kv[1]).unflatten(2, (nh // nkv, qm)) / torch.where(den == 0, torch.ones_like(den),
                                                                                         den)
    t = torch.arange(s["q"].shape[0], device=dev)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, qm, nh, hd)
    return {"o": o[r, t - cu[r]].to(s["q"].dtype)}


# --------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "plan":
        # request lengths in and out, the offsets, one table entry and one stack entry for a page of new tokens
        t = c["tokens"]
        return {"bytes": c["requests"] * 16 + t * (8 + 4 + 4) + t // c["page"] * 8, "flops": 0}
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    size = _SIZE[c["dtype"]]
    if c["op"] == "rope":
        t = c["tokens"]
        cached = 2 * nkv * (hd // 2 + 4 * (hd // c["group"]))
        return {"bytes": t * ((nh + 2 * nkv) * hd * size + nh * hd * size + cached + 2 * nkv * hd * 2 + c["rot"] * 4 + 12),
                "flops": t * ((nh + nkv) * hd * 7 + 2 * nkv * hd * 5)}
    # lengths are spread over their logarithm
    lo, hi, n = c["len_lo"], c["len_hi"], c["requests"]
    mean = (hi - lo) / math.log(hi / lo) if hi > lo else hi
    ql = (c["q_lo"] + c["q_hi"]) / 2
    read = min(mean, c["window"] + ql) if c["window"] else mean
    seen = min(mean - ql / 2, c["window"]) if c["window"] else mean - (ql - 1) / 2
    return {"bytes": n * (read * nkv * (hd + 8 * (hd // c["group"])) + 2 * ql * nh * hd * size),
            "flops": 4 * n * ql * seen * nh * hd}


# --------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return None


def _exact_rope(c, s):
    nh, nkv, hd, group = c["nh"], c["nkv"], c["hd"], c["group"]
    x = s["x"].double().reshape(-1, nh + 2 * nkv, hd)
    t, rot = x.shape[0], c["rot"]
    pos = s["pos"].long().clamp(min=0)
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    heads = []
    for part, w in ((x[:, :nh], s["wq"]), (x[:, nh:nh + nkv], s["wk"])):
        if w is not None:
            part = part / (part.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        y = part.clone()
        pair = torch.complex(part[..., :rot // 2], part[..., rot // 2:rot]) * turn
        y[..., :rot // 2], y[..., rot // 2:rot] = pair.real, pair.imag
        heads.append(y)
    live, kept = (s["pos"] >= 0).double()[:, None, None], (s["slots"] >= 0).double()[:, None, None]
    out = {"q": heads[0] * live}
    for name, y in (("k", heads[1]), ("v", x[:, nh + nkv:])):
        y = y.reshape(t, nkv, hd // group, group)
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        sc, m = ((hi - lo) / 15).half().double(), lo.half().double()
        n = ((y - m) / sc).round().clamp(0, 15)
        n[(sc == 0).expand_as(n)] = 0
        out[name] = (sc * n + m).half().double().reshape(t, nkv, hd) * kept
    return out


def _exact_attn(c, s):
    nh, nkv, hd, page, group = c["nh"], c["nkv"], c["hd"], c["page"], c["group"]
    n, g = c["requests"], nh // nkv
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(n + 1))
    half, sc = 8 * hd, 64 * (hd // group)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(n):
        size, rows = lens[b], cu[b + 1] - cu[b]
        raw = s["data"][s["table"][b, :(size + page - 1) // page].long()]       # [pages, nkv, blocks, bytes]
        raw = raw.transpose(0, 1).reshape(nkv, -1, raw.shape[-1])
        kv = []
        for at in (0, half + sc):
            codes = raw[..., at:at + half].reshape(nkv, -1, hd // 2)[:, :size].int()
            sm = raw[..., at + half:at + half + sc].contiguous().view(torch.half).reshape(nkv, -1, hd // group, 2)
            sm = sm[:, :size].double().repeat_interleave(group, 2)
            codes = torch.stack([codes % 16, codes // 16], -1).reshape(nkv, size, hd).double()
            kv.append((sm[..., 0] * codes + sm[..., 1]).half().double())
        at = torch.arange(size - rows, size, device=out.device)[:, None]
        p = torch.arange(size, device=out.device)[None, :]
        hide = p > at
        if c["window"]:
            hide = hide | (p <= at - c["window"])
        for h in range(nkv):
            q = s["q"][cu[b]:cu[b + 1], h * g:(h + 1) * g].double().transpose(0, 1)
            z = (q @ kv[0][h].T / math.sqrt(hd)).masked_fill(hide, -math.inf)
            out[cu[b]:cu[b + 1], h * g:(h + 1) * g] = (torch.softmax(z, -1) @ kv[1][h]).transpose(0, 1)
    return {"o": out}

"""Oracle (numpy, 64 bits) for serving from the paged 4-bit cache — test infrastructure: the plan of a
step, norms and rotation, the 4-bit groups, and attention. The norm and rotation restate
webtorch/lm_engine.py:62-74, the attention webtorch/lm_engine.py:89-101; the cache and the plan have
no counterpart in the reference."""
import numpy as np


def plan(prev, new, table, free, n_free, page, max_tokens):
    """One request after the other. table and free are copied; returns (table, free, n_free, lens, cu, slots,
    positions, requests)."""
    table, free = table.copy(), free.copy()
    n, width = table.shape
    pages = lambda t: -(-int(t) // page)  # noqa: E731
    top = int(n_free)
    for b in range(n):
        if new[b] < 0:
            for i in range(min(pages(prev[b]), width)):
                if top < len(free):
                    free[top] = table[b, i]
                    top += 1
    avail, asked, tokens, taken = top, 0, 0, 0
    lens, cu, slots, positions, requests = [], [0], [], [], []
    for b in range(n):
        put = 0
        if new[b] >= 0 and pages(prev[b] + new[b]) <= width:
            need = pages(prev[b] + new[b]) - pages(prev[b])
            asked += need
            tokens += int(new[b])
            if tokens <= max_tokens and (need == 0 or asked <= avail):
                put = int(new[b])
                for i in range(need):
                    table[b, pages(prev[b]) + i] = free[avail - 1 - taken]
                    taken += 1
        for p in range(int(prev[b]), int(prev[b]) + put):
            slots.append(int(table[b, p // page]) * page + p % page)
            positions.append(p)
            requests.append(b)
        lens.append(0 if new[b] < 0 else int(prev[b]) + put)
        cu.append(cu[-1] + put)
    pad = [-1] * (max_tokens - len(slots))
    return (table, free, avail - taken, np.array(lens), np.array(cu), np.array(slots + pad, np.int64),
            np.array(positions + pad), np.array(requests + pad))


def norm_rotate(x, w, cos, sin, eps):
    """x [..., HD] in 64 bits; cos, sin [..., rot / 2] at the rows' positions."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    cos, sin = np.asarray(cos, np.float64), np.asarray(sin, np.float64)
    return np.concatenate([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def quantise(x, group):
    """(codes, s, m) of x [..., HD] fp32, step by step in IEEE fp32 as the kernel rounds."""
    y = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        lo, hi = y.min(-1), y.max(-1)
        s = ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
        m = lo.astype(np.float16)
        bad = ~(np.abs(y) <= 65504).all(-1)
        s[bad] = m[bad] = np.nan
        sf, mf = s.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
        n = np.clip(np.rint((y - mf) / np.where(sf == 0, np.float32(1), sf)), 0, 15)
        n = np.where((sf == 0) | bad[..., None], 0, n)
    return n.astype(np.uint8), s, m


def values(codes, s, m):
    """half(s n + m) of codes [..., groups, G], flattened to [..., HD]; float64 holds s n + m exactly."""
    v = (s.astype(np.float64)[..., None] * codes + m.astype(np.float64)[..., None]).astype(np.float16)
    return v.reshape(*v.shape[:-2], -1)


def attention(q, K, V, cu, lens, scale, window=0):
    """q [T, NH, HD]; K, V lists of [len, NKV, HD]; causal from the end of each request, in 64 bits."""
    out = np.zeros(q.shape)
    NH = q.shape[1]
    for b, (k, v) in enumerate(zip(K, V)):
        rows = cu[b + 1] - cu[b]
        grp = NH // k.shape[1]
        for i in range(rows):
            p = lens[b] - rows + i
            lo = max(0, p - window + 1) if window else 0
            if p < 0 or p + 1 <= lo:
                continue
            kk, vv = k[lo:p + 1].astype(np.float64), v[lo:p + 1].astype(np.float64)
            for h in range(NH):
                z = kk[:, h // grp] @ q[cu[b] + i, h].astype(np.float64) * scale
                e = np.exp(z - z.max())
                out[cu[b] + i, h] = e @ vv[:, h // grp] / e.sum()
    return out


def norm_rotate32(x, w, cos, sin, eps):
    """norm_rotate in IEEE fp32 steps, the sum of squares as a balanced tree of neighbours."""
    x = np.asarray(x, np.float32)
    if w is not None:
        s = x * x
        while s.shape[-1] > 1:
            s = s[..., 0::2] + s[..., 1::2]
        r = np.float32(1) / np.sqrt(s * np.float32(1.0 / x.shape[-1]) + np.float32(eps))
        x = (x * r) * np.asarray(w, np.float32)
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)

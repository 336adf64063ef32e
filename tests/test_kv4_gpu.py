"""Serving from the paged 4-bit cache on the GPU, against plain 64-bit restatements (oracle/kv4.py):
the plan of a step exactly, codes and scales bit for bit, attention within bounds derived from its
roundings."""
import numpy as np
import pytest
import torch

from oracle import kv4 as ok
from webpytorch_b200 import _ffi, kv4
from webpytorch_b200.decode import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


# ------------------------------------------------------------------------------------ plan
def run_plan(prev, new, table, free, n_free, page, cap, stride=None):
    n, width = table.shape
    wide = torch.full((n, stride or width), 99, dtype=torch.int32, device=DEV)
    wide[:, :width] = dev(table)
    t, f = wide[:, :width], dev(free)
    args = (dev(prev), dev(new), t, f, dev(np.array([n_free], np.int32)), page, cap)
    p = kv4.plan(*args)
    again = kv4.plan(*args)                       # the inputs are unchanged: the same answer
    for a, b in zip(p, again):
        assert torch.equal(a, b)
    got = [t, f, p.n_free, p.seq_lens, p.cu_new, p.slots, p.positions, p.requests]
    if stride:
        assert (wide[:, width:] == 99).all()
    return [x.cpu().numpy() for x in got]


def check_plan(prev, new, table, free, n_free, page, cap, stride=None):
    got = run_plan(prev, new, table, free, n_free, page, cap, stride)
    want = ok.plan(prev, new, table, free, n_free, page, cap)
    for name, g, w in zip(("table", "free", "n_free", "lens", "cu", "slots", "positions", "requests"), got, want):
        assert np.array_equal(g.reshape(-1), np.asarray(w).reshape(-1)), name
    return want


def make_plan(n, longest, page, spare, seed, ended=0.1, prompts=0.2, width_extra=1):
    rng = np.random.default_rng(seed)
    prev = rng.integers(0, longest + 1, n).astype(np.int32)
    new = np.ones(n, np.int32)
    u = rng.random(n)
    new[u < prompts] = rng.integers(0, longest + 1, n)[u < prompts]
    new[u > 1 - ended] = -1
    width = -(-longest // page) + width_extra
    held = -(-prev // page)
    order = rng.permutation(int(held.sum()) + spare).astype(np.int32)
    table = np.full((n, width), -7, np.int32)
    at = 0
    for b in range(n):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = np.full(len(order), -3, np.int32)
    free[:spare] = order[at:]
    return prev, new, table, free, spare


@pytest.mark.parametrize("n,longest,page,spare,cap", [
    (1, 40, 16, 3, 64), (1, 0, 16, 1, 0), (7, 100, 16, 40, 400), (33, 500, 32, 5, 300), (256, 60, 16, 1000, 20000),
    (1024, 90, 64, 200, 5000), (1025, 33, 16, 2000, 30000), (2500, 300, 128, 700, 100000), (5000, 200, 16, 30000, 1 << 19), (16385, 40, 16, 30000, 100000), (40000, 20, 16, 20000, 9000),
])
def test_plan(n, longest, page, spare, cap):
    check_plan(*make_plan(n, longest, page, spare, n), page, cap)


def test_plan_strided_table_and_rows_too_short():
    a = make_plan(50, 200, 16, 400, 3, width_extra=0)      # prompts on top of what is held overflow the row
    w = check_plan(*a, 16, 10000, stride=29)
    assert (w[3] == a[0]).any()


def test_plan_nothing_free_and_no_room():
    prev, new, table, free, _ = make_plan(64, 100, 16, 0, 5, ended=0.0, prompts=0.0)
    w = check_plan(prev, new, table, free if len(free) else np.zeros(1, np.int32), 0, 16, 64)
    assert (w[3] == prev)[prev % 16 == 0].all()            # no page for them
    assert (w[3] == prev + 1)[prev % 16 != 0].all()        # room in the page they hold
    w = check_plan(prev, new, table, np.zeros(8, np.int32), 0, 16, 0)
    assert (w[3] == prev).all()


def test_plan_pages_given_back_are_taken_in_the_same_step():
    prev = np.array([64, 10], np.int32)
    new = np.array([-1, 54], np.int32)
    table = np.array([[5, 6, 7, 8], [9, -1, -1, -1]], np.int32)
    w = check_plan(prev, new, table, np.zeros(6, np.int32), 0, 16, 64)
    assert list(w[0][1]) == [9, 8, 7, 6] and w[2] == 1 and list(w[3]) == [0, 64]


def test_plan_over_many_steps_keeps_every_page_once():
    rng = np.random.default_rng(11)
    n, page, width, pages = 37, 16, 12, 200
    prev, table = np.zeros(n, np.int32), np.full((n, width), -1, np.int32)
    free, n_free = rng.permutation(pages).astype(np.int32), pages
    for step in range(30):
        new = rng.integers(0, 20, n).astype(np.int32)
        new[(rng.random(n) < 0.1) & (prev > 0)] = -1
        new[prev == 0] = rng.integers(0, 60, (prev == 0).sum())
        table, free, n_free, prev = check_plan(prev, new, table, free, n_free, page, 500)[:4]
        prev = prev.astype(np.int32)
        owned = [p for b in range(n) for p in table[b, :-(-prev[b] // page)]] + list(free[:n_free])
        assert sorted(owned) == list(range(pages)), step


# ------------------------------------------------------------------------------------ norms, rotation, 4 bits
def rope_case(T, NH, NKV, HD, rot, dtype, norm, seed, pad=0, lmax=50):
    rng = np.random.default_rng(seed)
    W = (NH + 2 * NKV) * HD
    x = rng.standard_normal((T, W + pad)).astype(np.float32) * np.exp(rng.standard_normal(W + pad) * 0.5).astype(np.float32)
    xt = dev(x, TYPES[dtype])[:, :W]
    cos, sin = rope_tables(lmax, rot, 1e4)
    pos = rng.integers(0, lmax, T).astype(np.int32)
    w = [(1 + 0.2 * rng.standard_normal(HD)).astype(np.float32) if norm else None for _ in range(2)]
    return xt, xt.float().cpu().numpy().reshape(T, NH + 2 * NKV, HD), cos, sin, pos, w


def wt(w):
    return None if w is None else dev(w)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,NH,NKV,HD,rot,norm,pad", [
    (1, 28, 4, 128, 128, False, 0), (5, 4, 2, 64, 64, True, 3), (17, 3, 3, 128, 64, True, 0), (9, 8, 1, 256, 256, True, 16),
    (3, 2, 1, 64, 32, False, 0), (2, 5, 5, 128, 8, True, 1), (4, 2, 2, 256, 0, True, 0),
])
def test_norm_rope_without_cache(dtype, T, NH, NKV, HD, rot, norm, pad):
    xt, x, cos, sin, pos, (qw, kw) = rope_case(T, NH, NKV, HD, rot or 2, dtype, norm, T + HD, pad)
    if rot == 0:
        cos, sin = cos[:, :0], sin[:, :0]
    q, k = kv4.qk_norm_rope(xt, NH, NKV, HD, dev(pos), dev(cos), dev(sin), q_weight=wt(qw), k_weight=wt(kw), eps=1e-6)
    c, s = cos[pos][:, None], sin[pos][:, None]
    rq, rk = ok.norm_rotate(x[:, :NH], qw, c, s, 1e-6), ok.norm_rotate(x[:, NH:NH + NKV], kw, c, s, 1e-6)
    # about 10 fp32 roundings of values up to the row's largest, then one to the output's type
    eps = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for got, ref in ((q, rq), (k, rk)):
        got = got.float().cpu().numpy().astype(np.float64)
        bound = np.abs(ref) * eps + 10 * 2.0 ** -23 * np.abs(ref).max(-1, keepdims=True) * 2 + 1e-7
        assert (np.abs(got - ref) <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,NH,NKV,HD,group,page,norm", [
    (1, 4, 4, 128, 64, 16, False), (37, 8, 2, 128, 32, 32, True), (20, 2, 1, 128, 128, 64, True), (50, 14, 2, 64, 32, 16, True),
    (11, 2, 2, 64, 64, 128, False), (33, 4, 1, 256, 32, 16, True), (18, 4, 2, 256, 64, 64, True), (7, 4, 2, 256, 128, 32, False),
])
def test_cache_codes_bit_exact(dtype, T, NH, NKV, HD, group, page, norm):
    """Codes, scales and minima in the packed cache equal the IEEE fp32 steps of the definition, and the
    rest of the cache is not touched."""
    xt, x, cos, sin, pos, (qw, kw) = rope_case(T, NH, NKV, HD, HD, dtype, norm, T * HD + group)
    x[0, NH:, :] = x[0, NH:, :]
    if T > 4:                                  # a constant row, an infinity, a nan, a value past fp16
        xt[1] = 0.5
        xt[2, -1] = float("inf")
        xt[3, -HD] = float("nan")
        if dtype != "f16":
            xt[4, -1] = 1e5
        x = xt.float().cpu().numpy().reshape(T, NH + 2 * NKV, HD)
    rng = np.random.default_rng(T)
    pages = -(-T // page) + 2
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    if T > 6:
        slots[5], slots[6] = -1, pages * page
        pos[T - 1] = -1
    cache = kv4.KV4Cache(pages, NKV, HD, page=page, group=group)
    cache.data.fill_(0xA5)
    q, none = kv4.qk_norm_rope(xt, NH, NKV, HD, dev(pos), dev(cos), dev(sin), q_weight=wt(qw), k_weight=wt(kw), cache=cache,
                               slots=dev(slots))
    assert none is None
    if pos[-1] < 0:
        assert (q[-1] == 0).all()
    c, s = cos[np.maximum(pos, 0)][:, None], sin[np.maximum(pos, 0)][:, None]
    with np.errstate(all="ignore"):
        k = ok.norm_rotate32(x[:, NH:NH + NKV], kw, c, s, 1e-6)
    parts = [ok.quantise(y, group) for y in (k, x[:, NH + NKV:])]
    want = np.full(tuple(cache.data.shape), 0xA5, np.uint8)
    half, sc = 8 * HD, 64 * (HD // group)
    vals = [ok.values(*p) for p in parts]
    for t in range(T):
        if not 0 <= slots[t] < pages * page or pos[t] < 0:
            for w in vals:
                w[t] = 0
            continue
        p, r = divmod(int(slots[t]), page)
        blk, r = divmod(r, 16)
        for (n, ss, m), at in zip(parts, (0, half + sc)):
            for g in range(NKV):
                code = n[t, g].reshape(-1)
                want[p, g, blk, at + r * HD // 2:at + (r + 1) * HD // 2] = code[0::2] | code[1::2] << 4
                sm = np.stack([ss[t, g], m[t, g]], -1).astype(np.float16).reshape(-1)
                sm = np.where(np.isnan(sm), np.uint16(0x7fff), sm.view(np.uint16)).view(np.uint8)
                want[p, g, blk, at + half + r * sc // 16:at + half + (r + 1) * sc // 16] = sm
    assert np.array_equal(cache.data.cpu().numpy(), want)
    inside = np.where((slots >= pages * page) | (pos < 0), -1, slots)
    kk, vv = cache.read(dev(inside))
    for got, ref in zip((kk, vv), vals):
        got = got.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref)) and (got == ref)[~np.isnan(ref)].all()


@pytest.mark.parametrize("HD,rot,norm,pad", [(128, 128, False, 0), (128, 128, True, 0), (64, 32, True, 0), (256, 256, True, 0), (128, 128, True, 3)])
def test_norm_rope_is_the_ieee_steps_to_the_bit(HD, rot, norm, pad):
    """fp32 outputs equal the definition's steps, none of them fused with another, at sizes where one in a hundred
    elements would show it."""
    xt, x, cos, sin, pos, (qw, kw) = rope_case(300, 6, 2, HD, rot, "f32", norm, HD + rot, pad)
    q, k = kv4.qk_norm_rope(xt, 6, 2, HD, dev(pos), dev(cos), dev(sin), q_weight=wt(qw), k_weight=wt(kw), eps=1e-6)
    c, s = cos[pos][:, None], sin[pos][:, None]
    for got, ref in ((q, ok.norm_rotate32(x[:, :6], qw, c, s, 1e-6)), (k, ok.norm_rotate32(x[:, 6:8], kw, c, s, 1e-6))):
        assert np.array_equal(got.cpu().numpy(), ref)


def test_position_past_the_tables_gives_nan_and_is_not_cached():
    xt, _, cos, sin, _, _ = rope_case(2, 2, 1, 64, 64, "f32", False, 1, lmax=8)
    cache = kv4.KV4Cache(1, 1, 64, page=16, group=32)
    cache.data.zero_()
    q, _ = kv4.qk_norm_rope(xt, 2, 1, 64, dev(np.array([8, 7], np.int32)), dev(cos), dev(sin), cache=cache,
                            slots=dev(np.array([0, 1], np.int64)))
    assert q[0].isnan().all() and q[1].isfinite().all()
    k, v = cache.read(dev(np.array([0, 1], np.int64)))
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[1] != 0).any()


# ------------------------------------------------------------------------------------ attention
class Batch:
    """Requests with random keys and values in a shuffled pool whose unwritten bytes stand for nan."""

    def __init__(self, lens, NKV, HD, page, group, seed, first_page=0, amp=1.0, width_extra=2):
        rng = np.random.default_rng(seed)
        self.lens, self.HD, self.rng = np.asarray(lens, np.int32), HD, rng
        held = -(-self.lens.astype(np.int64) // page)
        pages = int(held.sum()) + 3
        self.cache = kv4.KV4Cache(first_page + pages, NKV, HD, page=page, group=group)
        self.cache.data[first_page:] = 0xFF
        order = rng.permutation(pages) + first_page
        table = np.full((len(lens), int(held.max(initial=0)) + width_extra), -1, np.int32)
        data = np.full((pages,) + tuple(self.cache.data.shape[1:]), 0xFF, np.uint8)
        half, sc = 8 * HD, 64 * (HD // group)
        self.K, self.V, at = [], [], 0
        for b, n in enumerate(self.lens):
            table[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
            vals = [np.zeros((0, NKV, HD), np.float16)] * 2 if n == 0 else []
            for off in (0, half + sc) if n else ():
                x = (rng.standard_normal((n, NKV, HD)) * amp + 0.3 * rng.standard_normal(HD)).astype(np.float32)
                codes, s, m = ok.quantise(x, group)
                vals.append(ok.values(codes, s, m))
                c = codes.reshape(n, NKV, HD)
                c = c[..., 0::2] | c[..., 1::2] << 4
                sm = np.ascontiguousarray(np.stack([s, m], -1).reshape(n, NKV, -1)).view(np.uint8)
                for p in range(n):
                    pg, r = table[b, p // page] - first_page, p % page
                    d = data[pg, :, r // 16]
                    r %= 16
                    d[:, off + r * HD // 2:off + (r + 1) * HD // 2] = c[p]
                    d[:, off + half + r * sc // 16:off + half + (r + 1) * sc // 16] = sm[p]
            self.K.append(vals[0])
            self.V.append(vals[1])
        self.cache.data[first_page:] = dev(data)
        self.table = dev(table)

    def queries(self, ql, NH, dtype, amp=1.5):
        cu = np.concatenate([[0], np.cumsum(ql)]).astype(np.int32)
        q = dev(self.rng.standard_normal((int(cu[-1]), NH, self.HD)) * amp, TYPES[dtype])
        return q, cu

    def check(self, q, cu, got, dtype, window=0, scale=None):
        ref = ok.attention(q.float().cpu().numpy(), self.K, self.V, cu, self.lens, scale or 1 / np.sqrt(self.HD), window)
        got = got.float().cpu().numpy().astype(np.float64)[:cu[-1]]
        vmax = max([np.abs(v).max() for v in self.V if v.size], default=0.0)
        # fp32: scores of |q||k| scale ~ 10 off by some 2^-21 of that, through exp, times |v| twice;
        # 16 bits: probabilities to 11 bits, and the output's own rounding
        if dtype == "f32":
            bound = 4e-5 * vmax
        else:
            bound = (2.0 ** -8 if dtype == "bf16" else 2.0 ** -11) * np.abs(ref) + 2.0 ** -10 * vmax
        err = np.abs(got - ref)
        assert (err <= bound).all(), (float(np.nanmax(err)), np.isnan(got).sum())


def attend(bt, q, cu, **kw):
    return kv4.attention(q, bt.cache, bt.table, dev(bt.lens), None if cu is None else dev(cu), **kw)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("HD,group,page", [(64, 32, 16), (64, 64, 64), (128, 32, 32), (128, 64, 16), (128, 128, 64),
                                           (256, 32, 16), (256, 64, 128), (256, 128, 16)])
@pytest.mark.parametrize("NH,NKV", [(7, 1), (4, 4), (8, 1), (24, 2), (16, 1)])
def test_decode_one_token(dtype, HD, group, page, NH, NKV):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 130]
    bt = Batch(lens, NKV, HD, page, group, HD + NH)
    q, cu = bt.queries([1] * len(lens), NH, dtype)
    bt.check(q, cu, attend(bt, q, None), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[0, 5, 0], [777], [3000, 1, 900], [31] * 40, [4097, 2049]])
def test_decode_lengths(dtype, lens):
    bt = Batch(lens, 2, 128, 16, 64, len(lens))
    q, cu = bt.queries([1] * len(lens), 14, dtype)
    got = attend(bt, q, None)
    bt.check(q, cu, got, dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("HD,NH,NKV", [(128, 28, 4), (64, 8, 8), (256, 6, 2)])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 33, 200])
def test_several_queries_and_windows(dtype, HD, NH, NKV, window):
    lens, ql = [1, 40, 7, 0, 150, 64], [1, 5, 7, 0, 33, 0]
    bt = Batch(lens, NKV, HD, 16, 32, window + HD)
    q, cu = bt.queries(ql, NH, dtype)
    bt.check(q, cu, attend(bt, q, cu, window=window), dtype, window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("HD,NH,NKV,page,group,lens,ql", [
    (128, 8, 2, 64, 64, [300], [300]), (128, 7, 1, 16, 128, [129, 513], [128, 130]), (64, 4, 4, 32, 32, [257, 90, 260], [200, 1, 129]),
    (256, 4, 1, 16, 64, [200], [77]), (128, 4, 4, 64, 32, [1, 400], [1, 399]), (64, 16, 1, 16, 64, [70, 70], [64, 65]),
])
@pytest.mark.parametrize("window", [0, 100])
def test_prompts(dtype, HD, NH, NKV, page, group, lens, ql, window):
    bt = Batch(lens, NKV, HD, page, group, sum(lens))
    q, cu = bt.queries(ql, NH, dtype)
    bt.check(q, cu, attend(bt, q, cu, window=window), dtype, window)

# calls with enough rows for the tensor-core kernel: long requests beside short, odd and empty ones
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("HD,NH,NKV,page,group,lens,ql", [
    (128, 32, 4, 64, 64, [300, 77, 17, 0, 129], [200, 1, 9, 0, 3]), (128, 28, 4, 16, 128, [513, 640], [130, 101]),
    (128, 40, 8, 32, 32, [1, 257, 128], [1, 193, 13]), (128, 8, 8, 16, 64, [900], [800]), (64, 64, 4, 32, 32, [257, 90, 260], [150, 1, 129]),
    (64, 16, 16, 16, 64, [1000], [800]), (64, 14, 2, 64, 32, [1023, 64], [900, 1]), (256, 16, 2, 16, 64, [333, 20], [200, 20]),
    (256, 16, 2, 32, 32, [70, 129, 5], [20, 129, 1]), (256, 40, 8, 16, 128, [400], [60]),
    (64, 32, 32, 16, 32, [700], [600]), (128, 16, 16, 16, 64, [300, 1200], [70, 1030]), (128, 32, 4, 64, 64, [2500, 100], [300, 9]),
])
@pytest.mark.parametrize("window", [0, 1, 130])
def test_many_rows(dtype, HD, NH, NKV, page, group, lens, ql, window):
    bt = Batch(lens, NKV, HD, page, group, sum(lens) + window)
    q, cu = bt.queries(ql, NH, dtype)
    bt.check(q, cu, attend(bt, q, cu, window=window), dtype, window)


@pytest.mark.parametrize("HD,NH,NKV", [(64, 64, 8), (128, 32, 8), (256, 16, 4)])
def test_many_rows_that_see_nothing_bad_pages_and_streams(HD, NH, NKV):
    """More query tokens than positions; a page that is not the cache's; a length past the table."""
    bt = Batch([100, 250, 250, 40], NKV, HD, 16, 64, HD)
    q, cu = bt.queries([200, 250, 250, 3], NH, "bf16")
    good = attend(bt, q, cu)
    bt.check(q, cu, good, "bf16")
    assert (good[:100] == 0).all() and (good[100:] != 0).any()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    again = attend(bt, q, cu, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(good, again)
    bt.table[1, 2] = -7
    lens = dev(np.array([100, 250, 16 * bt.table.shape[1] + 1, 40], np.int32))
    got = kv4.attention(q, bt.cache, bt.table, lens, dev(cu))
    # the other requests: the cut of the work depends on all lengths, so not to the bit
    bt.check(q, cu, torch.cat([got[:200], good[200:700], got[700:]]), "bf16")
    # a row that sees the page, or any of the too long request, is nan
    assert got[200 + 32:450].isnan().all() and got[450:700].isnan().all()


def test_strided_queries_padding_scale_and_offsets_past_32_bits_for_many_rows():
    first = (1 << 32) // (2304 * 4) + 5
    bt = Batch([300, 33], 4, 128, 16, 64, 12, first_page=first)
    q, cu = bt.queries([290, 4], 32, "f16")
    wide = torch.full((300, 32 * 128 + 24), float("nan"), dtype=torch.float16, device=DEV)
    wide[:294, :4096] = q.reshape(294, 4096)
    out = torch.full((300, 32, 128), 7.0, dtype=torch.float16, device=DEV)
    assert attend(bt, wide[:, :4096].unflatten(1, (32, 128)), cu, scale=-0.05, out=out) is out
    bt.check(q, cu, out, "f16", scale=-0.05)
    assert (out[294:] == 0).all()



def test_strided_queries_scale_padding_and_out():
    bt = Batch([20, 33], 2, 64, 16, 32, 5)
    q, cu = bt.queries([2, 3], 4, "bf16")
    wide = torch.full((9, 4 * 64 + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:5, :256] = q.reshape(5, 256)
    qs = wide[:, :256].unflatten(1, (4, 64))
    out = torch.full((9, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    assert attend(bt, qs, cu, scale=0.3, out=out) is out
    bt.check(q, cu, out, "bf16", scale=0.3)
    assert (out[5:] == 0).all()                  # rows of no request, whatever they hold


def test_more_rows_than_requests_are_zero_without_offsets():
    bt = Batch([20], 1, 128, 16, 64, 6)
    q, _ = bt.queries([3], 4, "f32")
    got = attend(bt, q, None)
    bt.check(q[:1], np.array([0, 1]), got, "f32")
    assert (got[1:] == 0).all()


def test_length_shorter_than_the_queries_leaves_rows_empty():
    bt = Batch([3], 1, 64, 16, 32, 7)
    q, cu = bt.queries([5], 2, "f32")
    got = attend(bt, q, cu)
    bt.check(q, cu, got, "f32")
    assert (got[:2] == 0).all() and (got[2:] != 0).any()


def test_bad_page_and_length_past_the_table_give_nan_for_that_request():
    bt = Batch([50, 50, 50], 1, 64, 16, 32, 8)
    q, cu = bt.queries([1, 1, 1], 2, "f32")
    good = attend(bt, q, None)
    bt.table[1, 2] = bt.cache.num_pages
    lens = dev(np.array([50, 50, 16 * bt.table.shape[1] + 1], np.int32))
    bt.table[2, 4:] = 0
    got = kv4.attention(q, bt.cache, bt.table, lens)
    assert torch.equal(got[0], good[0]) and got[1].isnan().all() and got[2].isnan().all()


def test_nan_in_what_a_query_sees_and_only_there():
    bt = Batch([64, 64], 1, 64, 16, 32, 9)
    q, cu = bt.queries([1, 1], 4, "f32")
    q[0, 1, 3] = float("nan")
    got = attend(bt, q, None)
    assert got[0, 1].isnan().all() and got[0, [0, 2, 3]].isfinite().all() and got[1].isfinite().all()


def test_extreme_scores():
    """One position takes all the weight, by scores far past exp's range."""
    bt = Batch([100], 1, 128, 16, 64, 10, amp=30.0)
    for dtype in ("f32", "bf16"):
        q, cu = bt.queries([1], 4, dtype, amp=60.0)
        got = attend(bt, q, None).float().cpu().numpy()
        K, V = bt.K[0][:, 0].astype(np.float64), bt.V[0][:, 0].astype(np.float64)
        z = q[0].double().cpu().numpy() @ K.T
        top = np.sort(z, -1)
        for h in range(4):
            if top[h, -1] - top[h, -2] > 2000:    # nothing else has weight
                want = V[z[h].argmax()]
                assert np.abs(got[0, h] - want).max() <= (2.0 ** -8 if dtype == "bf16" else 4e-5) * np.abs(want).max()
        assert np.isfinite(got).all()


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of the cache."""
    first = (1 << 32) // (2304 * 4) + 5
    bt = Batch([70, 33], 4, 128, 16, 64, 12, first_page=first)
    assert bt.cache.nbytes() > 1 << 32
    q, cu = bt.queries([1, 4], 8, "f32")
    bt.check(q, cu, attend(bt, q, cu), "f32")
    slots = dev(np.array([(bt.table[0, 0].item()) * 16 + 3], np.int64))
    k, v = bt.cache.read(slots)
    assert np.array_equal(k[0].cpu().numpy(), bt.K[0][3]) and np.array_equal(v[0].cpu().numpy(), bt.V[0][3])


def test_same_inputs_same_bits_on_any_stream():
    bt = Batch([5000, 3, 800, 0, 64], 4, 128, 16, 64, 13)
    q, cu = bt.queries([1] * 5, 28, "bf16")
    a = attend(bt, q, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = [attend(bt, q, None) for _ in range(5)]
    c = attend(bt, q, None, stream=s)
    torch.cuda.synchronize()
    for x in b + [c]:
        assert torch.equal(a, x)


def test_queries_that_another_stream_still_writes():
    """Unaligned queries are copied first: on the call's stream, behind what writes them."""
    bt = Batch([60, 33], 2, 64, 16, 32, 14)
    q, cu = bt.queries([1, 1], 4, "bf16")
    want = attend(bt, q, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    wide = torch.zeros((2, 1 + 4 * 64), dtype=torch.bfloat16, device=DEV)
    qs = wide[:, 1:].unflatten(1, (4, 64))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        qs.copy_(q)
    got = attend(bt, qs, None, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_step_in_a_graph():
    """plan, write and attention captured once and replayed with new inputs."""
    rng = np.random.default_rng(3)
    NH, NKV, HD, page, n, cap = 8, 2, 64, 16, 3, 8
    cache = kv4.KV4Cache(40, NKV, HD, page=page, group=32)
    cache.data.fill_(0xFF)
    cos, sin = (dev(x) for x in rope_tables(64, HD, 1e4))
    lens, new = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    table = torch.full((n, 4), -1, dtype=torch.int32, device=DEV)
    free, n_free = torch.arange(40, dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    x = torch.zeros(cap, (NH + 2 * NKV) * HD, device=DEV)

    def step():
        p = kv4.plan(lens, new, table, free, n_free, page, cap)
        q, _ = kv4.qk_norm_rope(x, NH, NKV, HD, p.positions, cos, sin, cache=cache, slots=p.slots)
        o = kv4.attention(q, cache, table, p.seq_lens, p.cu_new)
        lens.copy_(p.seq_lens)
        n_free.copy_(p.n_free)
        return q, o, p.cu_new

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            q, o, cu = step()
    torch.cuda.current_stream().wait_stream(s)
    K, V = [[] for _ in range(n)], [[] for _ in range(n)]
    c, sn = rope_tables(64, HD, 1e4)
    for counts in ([3, 5, 0], [1, 1, 1], [1, 0, 2], [1, 1, 1]):
        xs = rng.standard_normal((cap, NH + 2 * NKV, HD)).astype(np.float32)
        x.copy_(dev(xs).reshape(cap, -1))
        new.copy_(dev(np.array(counts, np.int32)))
        g.replay()
        at = 0
        for b, m in enumerate(counts):
            for _ in range(m):
                p = len(K[b])
                k = ok.norm_rotate32(xs[at, NH:NH + NKV], None, c[p], sn[p], 0.0)
                K[b].append(ok.values(*ok.quantise(k, 32)))
                V[b].append(ok.values(*ok.quantise(xs[at, NH + NKV:], 32)))
                at += 1
        offs = cu.cpu().numpy()
        assert list(np.diff(offs)) == counts
        ref = ok.attention(q.cpu().numpy(), [np.array(k).reshape(-1, NKV, HD) for k in K],
                           [np.array(w).reshape(-1, NKV, HD) for w in V], offs, [len(k) for k in K], HD ** -0.5)
        assert np.abs(o.cpu().numpy() - ref).max() <= 4e-5 * 5


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    bt = Batch([20], 2, 64, 16, 32, 1)
    q, cu = bt.queries([1], 4, "f32")
    lens = dev(bt.lens)
    with pytest.raises(ValueError):
        kv4.KV4Cache(4, 2, 96)
    with pytest.raises(ValueError):
        kv4.KV4Cache(4, 2, 64, page=24)
    with pytest.raises(ValueError):
        kv4.KV4Cache(4, 2, 64, data=torch.zeros(8, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        kv4.attention(q[:, :3], bt.cache, bt.table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q, bt.cache, bt.table, torch.cat([lens, lens]))
    with pytest.raises(TypeError):
        kv4.attention(q, bt.cache, bt.table.long(), lens)
    with pytest.raises(TypeError):
        kv4.attention(q.double(), bt.cache, bt.table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q, bt.cache, bt.table, lens.cpu())
    with pytest.raises(ValueError):
        kv4.attention(q, bt.cache, bt.table, lens, dev(np.array([0, 1, 1], np.int32)))
    with pytest.raises(_ffi.QLError):
        kv4.attention(q, bt.cache, bt.table, lens, window=-1)
    x = torch.zeros(1, 8 * 64, device=DEV)
    t = torch.zeros(4, 32, device=DEV)
    pos, slots = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        kv4.qk_norm_rope(x, 4, 3, 64, pos, t, t)
    with pytest.raises(ValueError):
        kv4.qk_norm_rope(x, 4, 2, 64, pos, t, t, q_weight=torch.ones(32, device=DEV))
    with pytest.raises(TypeError):
        kv4.qk_norm_rope(x, 4, 2, 64, pos.long(), t, t)
    with pytest.raises(TypeError):
        kv4.qk_norm_rope(x, 4, 2, 64, pos, t, t, cache=bt.cache)
    with pytest.raises(_ffi.QLError):
        kv4.qk_norm_rope(x, 4, 2, 64, pos, t[:, :31].contiguous(), t[:, :31].contiguous())
    with pytest.raises(ValueError):
        kv4.qk_norm_rope(x, 2, 3, 64, pos, t, t, cache=bt.cache, slots=slots)
    with pytest.raises(ValueError):
        kv4.plan(lens, torch.cat([lens, lens]), bt.table, lens, lens, 16, 4)
    with pytest.raises(_ffi.QLError):
        kv4.plan(lens, lens, bt.table, lens, lens.clone(), 20, 4)

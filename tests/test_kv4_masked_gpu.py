"""What a row of the attention does not see does not reach it: pages that are not the cache's, and keys and values
that stand for nan, at positions which other rows of the same tile see."""
import functools

import numpy as np
import pytest
import torch

from oracle import kv4 as ok
from test_kv4_gpu import Batch, attend

pytestmark = pytest.mark.gpu

# (dtype, HD, NH, NKV, page, group, lens, ql): tiles of the streaming kernel with 8 and 16 rows, the tensor-core kernel
# with positions cut over blocks and not
CASES = [
    ("f32", 128, 14, 2, 16, 64, [100, 300], [40, 5]), ("f32", 64, 4, 4, 32, 32, [200, 33], [120, 33]),
    ("f32", 256, 6, 2, 16, 32, [90], [90]), ("bf16", 128, 8, 4, 16, 32, [70, 40], [4, 3]), ("f16", 256, 16, 2, 16, 64, [150, 20], [100, 20]),
    ("bf16", 256, 8, 1, 64, 128, [400], [60]), ("bf16", 128, 32, 4, 16, 64, [300, 77, 129], [200, 1, 3]), ("f16", 64, 14, 2, 16, 32, [900, 64], [700, 1]),
    ("bf16", 128, 32, 32, 16, 128, [700, 150], [640, 100]), ("f16", 64, 64, 32, 32, 64, [400, 500], [300, 333]), ("bf16", 128, 28, 4, 64, 32, [700], [300]),
]


@functools.lru_cache(maxsize=None)
def make(at, window):
    """Requests, queries, and the 64-bit reference with the bound of Batch.check."""
    dtype, HD, NH, NKV, page, group, lens, ql = CASES[at]
    bt = Batch(lens, NKV, HD, page, group, 100 + window)
    q, cu = bt.queries(ql, NH, dtype)
    ref = ok.attention(q.float().cpu().numpy(), bt.K, bt.V, cu, bt.lens, HD ** -0.5, window)
    vmax = max(np.abs(v).max() for v in bt.V)
    bound = 4e-5 * vmax if dtype == "f32" else (2.0 ** -8 if dtype == "bf16" else 2.0 ** -11) * np.abs(ref) + 2.0 ** -10 * vmax
    return bt, q, cu, ref, bound


def seen_by(bt, cu, b, first, last, window):
    """Rows [T] that see one of the positions first .. last of request b."""
    out = torch.zeros(int(cu[-1]), dtype=torch.bool)
    n = cu[b + 1] - cu[b]
    for i in range(n):
        p = int(bt.lens[b]) - n + i
        lo = max(0, p - window + 1) if window else 0
        out[cu[b] + i] = bool(lo <= min(p, last) and first <= p)
    return out


def others_are_right(got, ref, bound, seen):
    """What `seen` [T, 1, 1] or [T, NH, HD] does not mark, against the reference."""
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - ref)
    assert (seen.numpy() | (err <= bound)).all()


@pytest.mark.parametrize("at", range(len(CASES)))
@pytest.mark.parametrize("window", [0, 50])
def test_a_page_that_is_not_the_caches(at, window):
    page, ql = CASES[at][4], CASES[at][7]
    bt, q, cu, ref, bound = make(at, window)
    others_are_right(attend(bt, q, cu, window=window), ref, bound, torch.zeros(1, 1, 1, dtype=torch.bool))
    for b, i, bad in ((0, (int(bt.lens[0]) - 1) // page, -7), (0, (int(bt.lens[0]) - ql[0] // 2) // page, 1 << 30),
                      (len(bt.lens) - 1, int(bt.lens[-1]) // page // 2, bt.cache.num_pages)):
        kept = bt.table[b, i].item()
        bt.table[b, i] = bad
        got = attend(bt, q, cu, window=window)
        bt.table[b, i] = kept
        seen = seen_by(bt, cu, b, i * page, i * page + page - 1, window)
        assert got[seen.to(got.device)].isnan().all()
        others_are_right(got, ref, bound, seen[:, None, None])


def edit(bt, b, p, kvh, group, what, value):
    """The bytes of (s, m) of one group of a cached position: keys ("k") or values ("v"). Returns the bytes before."""
    HD, G = bt.cache.HD, bt.cache.group
    half, sc, page = 8 * HD, 64 * (HD // G), bt.cache.page
    at = (0 if what == "k" else half + sc) + half + (p % 16) * (sc // 16) + 4 * group
    blk = bt.cache.data[bt.table[b, p // page].item(), kvh, p % page // 16]
    kept = blk[at:at + 4].clone()
    blk[at:at + 4] = torch.from_numpy(np.asarray(value, np.float16).view(np.uint8)) if not isinstance(value, torch.Tensor) else value
    return kept


@pytest.mark.parametrize("at", range(len(CASES)))
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("what,value", [("k", [np.nan, np.nan]), ("v", [np.nan, np.nan]), ("v", [1.0, np.inf])])
def test_a_group_that_stands_for_nan(at, window, what, value):
    dtype, HD, NH, NKV, page, group, lens, ql = CASES[at]
    bt, q, cu, ref, bound = make(at, window)
    grp, NG = NH // NKV, HD // group
    for b, p in ((0, lens[0] - 1), (0, lens[0] - 1 - ql[0] // 3), (0, lens[0] - ql[0]), (len(lens) - 1, lens[-1] - 1 - ql[-1] // 2),
                 (0, max(lens[0] - ql[0] - 20, 0))):
        kvh, n = (p * 7) % NKV, (p * 3) % NG
        kept = edit(bt, b, p, kvh, n, what, value)
        got = attend(bt, q, cu, window=window)
        edit(bt, b, p, kvh, n, what, kept)
        mark = torch.zeros(got.shape, dtype=torch.bool)
        els = slice(None) if what == "k" else slice(n * group, (n + 1) * group)
        for r in seen_by(bt, cu, b, p, p, window).nonzero()[:, 0].tolist():
            mark[r, kvh * grp:(kvh + 1) * grp, els] = True
        assert not got[mark.to(got.device)].isfinite().any()
        others_are_right(got, ref, bound, mark)


@pytest.mark.parametrize("dtype,NH,NKV,ql", [("f32", 4, 2, 20), ("bf16", 32, 4, 200)])
def test_values_past_fp16_are_not_finite_for_the_rows_that_see_them_alone(dtype, NH, NKV, ql):
    """A finite (s, m) whose last code stands for infinity: the codes below it are numbers."""
    HD, group, n, p = 128, 64, 300, 290
    bt = Batch([n], NKV, HD, 16, group, 3)
    q, cu = bt.queries([ql], NH, dtype)
    good = attend(bt, q, cu)
    edit(bt, 0, p, 1, 1, "v", [8736.0, -65504.0])
    half, at = 8 * HD, 8 * HD + 64 * (HD // group)
    codes = bt.cache.data[bt.table[0, p // 16].item(), 1, 0, at + p % 16 * HD // 2 + group // 2:][:group // 2].cpu().numpy()
    top = np.stack([codes & 15, codes >> 4], -1).reshape(-1) == 15
    assert top.any() and not top.all() and half < at
    got = attend(bt, q, cu)
    grp, first = NH // NKV, ql - (n - p)                   # row `first` is the first that sees the position
    assert torch.equal(got[:first], good[:first])
    assert torch.equal(got[:, :grp], good[:, :grp]) and torch.equal(got[:, grp:2 * grp, :group], good[:, grp:2 * grp, :group])
    finite = got[first:, grp:2 * grp, group:].isfinite().cpu().numpy()
    assert not finite[..., top].any() and finite[..., ~top].all()

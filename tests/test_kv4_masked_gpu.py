"""What a row of the attention does not see does not reach it: pages that are not the cache's, at positions which
other rows of the same tile see."""
import pytest
import torch

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


def make(case, seed):
    dtype, HD, NH, NKV, page, group, lens, ql = case
    bt = Batch(lens, NKV, HD, page, group, seed)
    q, cu = bt.queries(ql, NH, dtype)
    return bt, q, cu


def seen_by(bt, cu, b, first, last, window):
    """Rows [T] that see one of the positions first .. last of request b."""
    out = torch.zeros(int(cu[-1]), dtype=torch.bool)
    n = cu[b + 1] - cu[b]
    for i in range(n):
        p = int(bt.lens[b]) - n + i
        lo = max(0, p - window + 1) if window else 0
        out[cu[b] + i] = bool(lo <= min(p, last) and first <= p)
    return out


def others_as_before(bt, q, cu, got, good, seen, case, window):
    """got without what `seen` [T] or [T, NH] or [T, NH, HD] marks, against the 64-bit reference."""
    while seen.dim() < 3:
        seen = seen[..., None]
    bt.check(q, cu, torch.where(seen.to(got.device), good, got), case[0], window)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("window", [0, 50])
def test_a_page_that_is_not_the_caches(case, window):
    page = case[4]
    bt, q, cu = make(case, 100 + window)
    good = attend(bt, q, cu, window=window)
    bt.check(q, cu, good, case[0], window)
    for b, at, bad in ((0, (int(bt.lens[0]) - 1) // page, -7), (0, (int(bt.lens[0]) - case[7][0] // 2) // page, 1 << 30),
                       (len(bt.lens) - 1, max(int(bt.lens[-1]) // page // 2, 0), bt.cache.num_pages)):
        kept = bt.table[b, at].item()
        bt.table[b, at] = bad
        got = attend(bt, q, cu, window=window)
        bt.table[b, at] = kept
        seen = seen_by(bt, cu, b, at * page, at * page + page - 1, window)
        assert got[seen.to(got.device)].isnan().all()
        others_as_before(bt, q, cu, got, good, seen, case, window)

"""Arguments at the ends of their ranges: windows as long as any number, queries of one head with any stride."""
import numpy as np
import pytest
import torch

from test_kv4_gpu import Batch, attend, dev
from webpytorch_b200 import kv4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [64, 1 << 20, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 63])
@pytest.mark.parametrize("dtype,HD,NH,NKV,lens,ql", [
    ("f32", 64, 2, 1, [3, 40], [9, 40]), ("bf16", 128, 32, 4, [100, 250, 40], [200, 250, 3]), ("f16", 256, 4, 2, [5, 0], [8, 2]),
])
def test_a_window_past_every_position_hides_nothing(dtype, HD, NH, NKV, lens, ql, window):
    """Also where a length is shorter than the queries, so that the first of them are before position 0."""
    bt = Batch(lens, NKV, HD, 16, 32, 21)
    q, cu = bt.queries(ql, NH, dtype)
    want = attend(bt, q, cu)
    bt.check(q, cu, want, dtype)
    got = attend(bt, q, cu, window=window)
    if window > max(lens):
        assert torch.equal(got, want)
    else:
        bt.check(q, cu, got, dtype, window)


def test_one_head_in_rows_that_are_wider():
    bt = Batch([20, 33], 1, 64, 16, 32, 22)
    q, cu = bt.queries([2, 3], 1, "bf16")
    wide = torch.full((5, 64 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :64] = q[:, 0]
    want = attend(bt, q, cu)
    bt.check(q, cu, want, "bf16")
    for strided in (wide[:, None, :64], wide.as_strided((5, 1, 64), (88, 8, 1)), wide.as_strided((5, 1, 64), (88, 0, 1))):
        got = kv4.attention(strided, bt.cache, bt.table, dev(bt.lens), dev(cu))
        assert torch.equal(got, want) and np.isfinite(got.float().cpu().numpy()).all()

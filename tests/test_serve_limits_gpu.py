"""A request that grows to the end of its block table, where the page does not divide `lmax`."""
import numpy as np
import pytest
import torch

from conftest import max_rel_err
from test_decode_gpu import _model
from test_serve_gpu import EPS, THETA, TOL, Model
from webpytorch_b200.decode import rope_tables
from webpytorch_b200.serve import ServeStack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lmax,page,limit", [(100, 64, 128), (40, 16, 48), (48, 16, 48)])
def test_positions_up_to_the_table_are_served_right_and_no_more(lmax, page, limit):
    layers, refs, dims = _model(seed=2)
    H, NH, NKV, HD = dims
    st = ServeStack(layers, H, NH, NKV, HD, lmax, 2, 8, page=page, group=32, cap=16, theta=THETA, eps=EPS, graph=False)
    m = Model(st, refs, None, dims)
    m.cos, m.sin = rope_tables(limit, HD, THETA)
    rng = np.random.default_rng(lmax)
    for at in range(0, limit, 16):
        emb = rng.standard_normal((16, H)).astype(np.float32)
        h, p = st.step(torch.from_numpy(emb), [16, 0])
        assert st.lens.tolist() == [at + 16, 0] and int(p.cu_new[-1]) == 16
        got = h.cpu().numpy()
        assert np.isfinite(got).all()
        assert max_rel_err(got, m.step(emb, p)) < TOL
    emb = rng.standard_normal((2, H)).astype(np.float32)
    h, p = st.step(torch.from_numpy(emb), [1, 1])      # the first request is full: it waits, the other goes on
    assert st.lens.tolist() == [limit, 1] and p.requests[:2].tolist() == [1, -1]
    assert max_rel_err(h[:1].cpu().numpy(), m.step(emb[1:], p)) < TOL
    assert st.lmax == limit

"""Several requests through the layers over the paged 4-bit caches: prompts in chunks, decoding, requests that
end and begin, against the oracle's layer math on the values that the caches hold."""
import numpy as np
import pytest
import torch

from conftest import max_rel_err
from oracle import decode as odec
from oracle import kv4 as ok
from oracle.moe import silu
from test_decode_gpu import _model
from webpytorch_b200.decode import rope_tables
from webpytorch_b200.serve import ServeStack

pytestmark = pytest.mark.gpu
TOL = 2e-3
THETA, EPS = 1e6, 1e-6


def make(graph, norms, pages=12, requests=3, seed=0):
    layers, refs, (H, NH, NKV, HD) = _model(seed=seed)
    rng = np.random.default_rng(seed + 50)
    hn = [tuple(rng.uniform(0.5, 1.5, HD).astype(np.float32) for _ in range(2)) for _ in layers] if norms else None
    st = ServeStack(layers, H, NH, NKV, HD, 64, requests, pages, page=16, group=32, cap=16, theta=THETA, eps=EPS,
                    head_norms=None if hn is None else [tuple(torch.from_numpy(w) for w in p) for p in hn], graph=graph)
    return st, refs, hn, (H, NH, NKV, HD)


class Model:
    """The layers in numpy; keys and values are read back from the caches and checked to be within half a
    step of their own, so that rounding ties do not matter further on."""

    def __init__(self, st, refs, hn, dims):
        self.st, self.refs, self.hn = st, refs, hn
        self.H, self.NH, self.NKV, self.HD = dims
        self.kv = [[[[], []] for _ in range(st.requests)] for _ in refs]
        self.cos, self.sin = rope_tables(64, self.HD, THETA)

    def step(self, emb, p):
        n = int(p.cu_new[-1])
        req, pos, slots = (x[:n].cpu().numpy() for x in (p.requests, p.positions, p.slots))
        h = emb.astype(np.float32)
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        for i, lay in enumerate(self.refs):
            x = odec.rms(h, lay["in_ln"], EPS)
            q, k, v = (lay[m](x).reshape(n, -1, self.HD) for m in "qkv")
            qw, kw = self.hn[i] if self.hn else (None, None)
            q, k = ok.norm_rotate(q, qw, c, s, EPS), ok.norm_rotate(k, kw, c, s, EPS)
            got = [y.float().cpu().numpy() for y in self.st.caches[i].read(torch.from_numpy(slots).cuda())]
            for y, z in zip(got, (k, v)):
                _, sc, _ = ok.quantise(z.astype(np.float32), 32)
                step = np.repeat(sc.astype(np.float64), 32, -1).reshape(z.shape)
                assert (np.abs(y - z) <= step * 0.51 + 2e-3 * np.abs(z).max()).all()
            for t in range(n):
                for side, y in zip(self.kv[i][req[t]], got):
                    assert len(side) == pos[t]
                    side.append(y[t])
            o = np.zeros((n, self.NH * self.HD), np.float32)
            for t in range(n):
                K, V = (np.array(side[:pos[t] + 1]) for side in self.kv[i][req[t]])
                o[t] = ok.attention(q[t:t + 1], [K], [V], [0, 1], [pos[t] + 1], self.HD ** -0.5).reshape(-1)
            h = (h + lay["o"](o)).astype(np.float32)
            x = odec.rms(h, lay["post_ln"], EPS)
            h = (h + lay["down"](silu(lay["gate"](x)) * lay["up"](x))).astype(np.float32)
        return h

    def end(self, b):
        for layer in self.kv:
            layer[b] = [[], []]


@pytest.mark.parametrize("graph,norms", [(False, False), (True, True)])
def test_requests_that_begin_go_on_and_end(graph, norms):
    st, refs, hn, dims = make(graph, norms)
    m = Model(st, refs, hn, dims)
    rng = np.random.default_rng(7)
    length = [0, 0, 0]
    for counts in ([5, 0, 3], [1, 16 - 2, 1], [1, 1, 1], [-1, 2, 1], [7, 1, 1], [0, 0, 0], [1, -1, 9], [2, 4, 1]):
        total = sum(max(c, 0) for c in counts)
        emb = rng.standard_normal((total, dims[0])).astype(np.float32)
        h, p = st.step(torch.from_numpy(emb), counts)
        for b, c in enumerate(counts):
            if c < 0:
                m.end(b)
            length[b] = 0 if c < 0 else length[b] + c
        assert st.lens.tolist() == length and int(p.cu_new[-1]) == total
        if total:
            want = m.step(emb, p)
            assert max_rel_err(h[:total].cpu().numpy(), want) < TOL


def test_a_request_without_pages_waits_and_keeps_its_rows_out():
    """Three requests ask for more pages than there are: the last waits, and the others' rows stay theirs."""
    st, refs, hn, dims = make(False, False, pages=2)
    m = Model(st, refs, hn, dims)
    rng = np.random.default_rng(8)
    emb = rng.standard_normal((12, dims[0])).astype(np.float32)
    h, p = st.step(torch.from_numpy(emb), [5, 4, 3])
    assert st.lens.tolist() == [5, 4, 0] and int(p.cu_new[-1]) == 9
    assert max_rel_err(h[:9].cpu().numpy(), m.step(emb[:9], p)) < TOL
    h, p = st.step(torch.from_numpy(emb[9:]), [-1, 0, 3])        # the first ends, its page serves the last
    m.end(0)
    assert st.lens.tolist() == [0, 4, 3]
    assert max_rel_err(h[:3].cpu().numpy(), m.step(emb[9:], p)) < TOL


def test_graph_replay_equals_eager():
    a, b = make(False, True, seed=3)[0], make(True, True, seed=3)[0]
    rng = np.random.default_rng(4)
    for counts in ([4, 0, 6], [1, 3, 1], [1, 1, 1]):
        emb = torch.from_numpy(rng.standard_normal((sum(counts), a.H)).astype(np.float32))
        ha, pa = a.step(emb, counts)
        hb, pb = b.step(emb, counts)
        n = sum(counts)
        assert torch.equal(ha[:n], hb[:n])
        for x, y in zip(pa, pb):
            assert torch.equal(x, y)


def test_refusals():
    st, _, _, dims = make(False, False)
    with pytest.raises(ValueError):
        st.step(torch.zeros(3, dims[0]), [1, 1])
    with pytest.raises(ValueError):
        st.step(torch.zeros(3, dims[0]), [1, 1, 0])
    with pytest.raises(ValueError):
        st.step(torch.zeros(17, dims[0]), [17, 0, 0])
    with pytest.raises(ValueError):
        make(False, False)[0].__class__(st.layers, *dims, 64, 3, 4, cap=17)

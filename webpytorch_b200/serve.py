"""A decode stack that serves several requests at once: the layers of `decode.DecodeStack` over caches that are
shared in pages and held in 4 bits (`kv4`).

A step takes up to `cap` tokens of any mix: prompt chunks of requests that begin, the next tokens of those
that go on. Layer math as in decode.py (package `webtorch`, lm_engine.py:62-107), with norms of the query and
key heads where a layer has them:

    plan: block tables, slots and positions from the request lengths                  (kv4.plan, once a step)
    x = rms(h, in_ln); q | k | v = x @ Wqkv + b                                       one fused GEMV
    norms and rotation of q and k; k and v into the 4-bit pages                       (kv4.qk_norm_rope)
    o = softmax(q K^T / sqrt(HD)) V over the pages                                    (kv4.attention)
    h = h + o @ Wo;  h = h + (silu(g) * u) @ Wdown                                    three fused GEMVs

No length is read back to the host within a step, so it is captured in a CUDA graph and replayed.
"""
import torch

from . import _ffi, kv4
from .decode import fused_linear, rope_tables

__all__ = ["ServeStack"]


class ServeStack:
    """layers: DecodeLayers; head_norms: None, or for each layer (q_weight, k_weight) fp32 [HD].

    `requests` rows of lengths and block tables, `pages` pages of `page` positions in each layer's cache
    (4.5 bits a value at group 64), at most `lmax` positions a request (rounded up to whole pages: attribute `lmax`) and
    `cap` <= 16 tokens a step. A request that asks for more is not served and keeps its length."""

    def __init__(self, layers, H, NH, NKV, HD, lmax, requests, pages, page=64, group=64, cap=16, theta=1e6, eps=1e-6,
                 head_norms=None, device=None, graph=True):
        if not 1 <= cap <= 16:
            raise ValueError("cap must be 1 to 16 tokens a step, got %d" % cap)
        if head_norms is not None and len(head_norms) != len(layers):
            raise ValueError("head_norms must have an entry for each of the %d layers" % len(layers))
        self.layers, self.H, self.NH, self.NKV, self.HD = layers, H, NH, NKV, HD
        width = -(-lmax // page)
        lmax = width * page                        # what the plan serves, and so what the rotation's tables cover
        self.lmax, self.requests, self.cap, self.eps, self.page = lmax, requests, cap, float(eps), page
        dev = self.dev = layers[0].qkv.qweight.device if device is None else torch.device(device)
        self.head_norms = [(None, None)] * len(layers) if head_norms is None else [
            tuple(w.to(dev, torch.float32).contiguous() for w in pair) for pair in head_norms]
        self.caches = [kv4.KV4Cache(pages, NKV, HD, page=page, group=group, device=dev) for _ in layers]
        i32 = dict(dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, **i32)
        self.table = torch.full((requests, width), -1, **i32)
        self.free = torch.arange(pages - 1, -1, -1, **i32)
        self.n_free = torch.tensor([pages], **i32)
        self.new = torch.zeros(requests, **i32)
        self.emb = torch.zeros((cap, H), dtype=torch.float32, device=dev)
        self.first = torch.zeros(requests, dtype=torch.int64, device=dev)   # a request's first row of emb
        cos, sin = rope_tables(lmax, HD, theta)
        self.cos, self.sin = torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev)
        I = max(l.I for l in layers)
        self.h = torch.zeros((cap, H), dtype=torch.float32, device=dev)
        self.qkv = torch.empty((cap, (NH + 2 * NKV) * HD), dtype=torch.float32, device=dev)
        self.q = torch.empty((cap, NH, HD), dtype=torch.float32, device=dev)
        self.att = torch.empty((cap, NH, HD), dtype=torch.float32, device=dev)
        self.gu = torch.empty((cap, 2 * I), dtype=torch.float32, device=dev)
        need = max(int(_ffi.fn("ql_gptq_matmul_workspace")(cap, K)) for K in (H, NH * HD, I, 2 * I))
        self.ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        self.att_ws = torch.zeros(int(_ffi.fn("ql_kv4_attention_workspace")(NH, NKV, HD)), dtype=torch.uint8, device=dev)
        self.use_graph, self.graph, self.out = graph, None, None

    def _forward(self):
        p = kv4.plan(self.lens, self.new, self.table, self.free, self.n_free, self.page, self.cap)
        # row t of the step is the plan's token t: a request that is not served leaves no gap
        r = p.requests.clamp(min=0).long()
        src = (self.first[r] + p.positions - self.lens[r]).clamp(0, self.cap - 1)
        self.h.copy_(torch.where((p.requests >= 0)[:, None], self.emb[src], torch.zeros((), device=self.dev)))
        h, ws = self.h, self.ws
        for lay, cache, (qw, kw) in zip(self.layers, self.caches, self.head_norms):
            fused_linear(h, lay.qkv, norm_weight=lay.in_ln, norm_eps=self.eps, out=self.qkv, workspace=ws)
            kv4.qk_norm_rope(self.qkv, self.NH, self.NKV, self.HD, p.positions, self.cos, self.sin, q_weight=qw,
                             k_weight=kw, eps=self.eps, cache=cache, slots=p.slots, out=self.q)
            kv4.attention(self.q, cache, self.table, p.seq_lens, p.cu_new, out=self.att, workspace=self.att_ws)
            fused_linear(self.att.view(self.cap, -1), lay.o, residual=h, out=h, workspace=ws)
            fused_linear(h, lay.gate_up, norm_weight=lay.post_ln, norm_eps=self.eps, out=self.gu, workspace=ws)
            fused_linear(self.gu[:, :2 * lay.I], lay.down, glu=lay.I, residual=h, out=h, workspace=ws)
        self.lens.copy_(p.seq_lens)
        self.n_free.copy_(p.n_free)
        return p

    def step(self, embeddings, new_lens):
        """One step: new_lens[b] tokens of each request (0: none, negative: it ends), embeddings [sum, H] their
        rows in order. Returns (h [cap, H], plan): row t is the plan's token t (plan.requests, plan.positions; rows
        past plan.cu_new[-1] are padding). Requests are served as far as pages and `cap` go; lengths after the
        step are in `lens`. h and the plan are the step's own buffers, which the next step writes again."""
        new = torch.as_tensor(new_lens, dtype=torch.int32)
        if new.shape != (self.requests,):
            raise ValueError("new_lens must have %d entries" % self.requests)
        counts = new.clamp(min=0).long()
        total = int(counts.sum())
        if total > self.cap or embeddings.shape != (total, self.H):
            raise ValueError("embeddings must be [%d, %d], at most %d rows, got %s"
                             % (total, self.H, self.cap, tuple(embeddings.shape)))
        self.new.copy_(new)
        self.first.copy_(torch.cumsum(counts, 0) - counts)
        self.emb[:total].copy_(embeddings)
        if not self.use_graph:
            return self.h, self._forward()
        if self.graph is None:
            self._capture()
        self.graph.replay()
        return self.h, self.out

    def _capture(self):
        side = torch.cuda.Stream(self.dev)
        side.wait_stream(torch.cuda.current_stream(self.dev))
        state = (self.lens, self.table, self.free, self.n_free, self.new)
        kept = [t.clone() for t in state]
        with torch.cuda.stream(side):
            self.new.zero_()
            self._forward()                        # loads the kernels; no token, so no cache is written
            for t, k in zip(state, kept):
                t.copy_(k)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=side):
                self.out = self._forward()
        torch.cuda.current_stream(self.dev).wait_stream(side)

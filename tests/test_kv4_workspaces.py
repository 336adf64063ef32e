"""Which workspace an attention call uses: one for each stream, and one of its own for what a graph captures, since
a graph is replayed on any stream."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from webpytorch_b200 import _build, _ffi, kv4


def test_captured_calls_have_a_workspace_of_their_own(monkeypatch):
    _build.build()
    now = SimpleNamespace(stream=70, capture=0)
    size = _ffi.fn("ql_kv4_attention_workspace")
    monkeypatch.setattr(kv4, "_workspaces", {})
    monkeypatch.setattr(kv4, "_captured", {}, raising=False)
    monkeypatch.setattr(_ffi, "stream_ptr", lambda *a: now.stream)
    monkeypatch.setattr(_ffi, "fn", lambda name: size if name == "ql_kv4_attention_workspace" else lambda s: now.capture)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capture != 0)
    cache = SimpleNamespace(device=torch.device("cpu"), HD=64, NKV=2)

    def get(stream, capture):
        now.stream, now.capture = stream, capture
        return kv4._attention_workspace(cache, 4)

    eager = get(70, 0)
    first = get(70, 1)
    assert get(70, 1) is first                    # the layers of one graph
    second, other = get(70, 2), get(71, 2)
    all_ = [eager, first, second, other]
    assert len({w.data_ptr() for w in all_}) == 4
    assert get(70, 0) is eager
    for w in all_:
        assert w.numel() == size(4, 2, 64) and (w[:2048] == 0).all()


@pytest.mark.gpu
def test_two_graphs_and_eager_calls_at_the_same_time():
    """Two graphs captured on one stream are replayed on two others while calls run on the first: each gets the bits
    of a call that runs alone, call after call."""
    from test_kv4_gpu import Batch, attend, dev
    s = [torch.cuda.Stream() for _ in range(3)]
    sets = []
    for i, lens in enumerate(([9000, 300, 40], [5000, 5001], [700, 12000, 1])):
        bt = Batch(lens, 4, 128, 16, 64, 30 + i)
        q, cu = bt.queries([1] * len(lens), 28, "f32")
        want = attend(bt, q, None)
        bt.check(q, cu, want, "f32")
        sets.append((bt, q, dev(bt.lens), want))

    def call(i):
        bt, q, lens, _ = sets[i]
        return kv4.attention(q, bt.cache, bt.table, lens)

    torch.cuda.synchronize()
    with torch.cuda.stream(s[0]):
        call(0)
        call(1)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for i in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s[0]):
                outs.append([call(i) for _ in range(8)])
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            for x in o:
                x.fill_(-1)
        torch.cuda.synchronize()
        eager = []
        for g, stream in zip(graphs, s[1:]):
            with torch.cuda.stream(stream):
                g.replay()
        with torch.cuda.stream(s[0]):
            eager = [call(2) for _ in range(6)]
        torch.cuda.synchronize()
        for got, (_, _, _, want) in zip(outs + [eager], sets):
            for x in got:
                assert torch.equal(x, want)


@pytest.mark.gpu
def test_a_first_call_may_be_a_captured_one():
    """No call on the stream before: the graph brings its own workspace, and its counters start at zero each time."""
    from test_kv4_gpu import Batch, attend, dev
    bt = Batch([6000, 17], 2, 64, 16, 32, 44)
    q, cu = bt.queries([1, 1], 14, "f16")
    want, lens = attend(bt, q, None), dev(bt.lens)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = kv4.attention(q, bt.cache, bt.table, lens)
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, want)
    assert np.isfinite(want.float().cpu().numpy()).all()

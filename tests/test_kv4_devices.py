"""Tensors on the wrong device are refused before any kernel sees their address: on the host with tensors that
have a device and no memory, and on the GPU with one CPU tensor in each place in turn."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from webpytorch_b200 import _build, _ffi, kv4

NH, NKV, HD, T, B = 4, 2, 64, 3, 2


def tensors(device):
    e = lambda shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device=device)  # noqa: E731
    return dict(
        lens=e(B, torch.int32), new=e(B, torch.int32), table=e((B, 4), torch.int32), free=e(8, torch.int32),
        n_free=e(1, torch.int32), qkv=e((T, (NH + 2 * NKV) * HD)), positions=e(T, torch.int32), cos=e((16, HD // 2)),
        sin=e((16, HD // 2)), qw=e(HD), kw=e(HD), slots=e(T, torch.int64), q=e((T, NH, HD)), cu=e(B + 1, torch.int32),
        out=e((T, NH, HD)), ws=e(1 << 26, torch.uint8), data=e((8, NKV, 1, 1280), torch.uint8))


def calls(t):
    cache = kv4.KV4Cache.__new__(kv4.KV4Cache)
    cache.data, cache.device = t["data"], t["data"].device
    cache.num_pages, cache.NKV, cache.HD, cache.page, cache.group = 8, NKV, HD, 16, 32
    return {
        "plan": lambda: kv4.plan(t["lens"], t["new"], t["table"], t["free"], t["n_free"], 16, T),
        "rope": lambda: kv4.qk_norm_rope(t["qkv"], NH, NKV, HD, t["positions"], t["cos"], t["sin"], q_weight=t["qw"],
                                         k_weight=t["kw"], cache=cache, slots=t["slots"], out=t["out"]),
        "attention": lambda: kv4.attention(t["q"], cache, t["table"], t["lens"], t["cu"], out=t["out"], workspace=t["ws"]),
        "read": lambda: cache.read(t["slots"]),
    }


PLACES = [(c, n) for c, names in dict(
    plan=("lens", "new", "table", "free", "n_free"), rope=("qkv", "positions", "cos", "sin", "qw", "kw", "slots", "out", "data"),
    attention=("q", "table", "lens", "cu", "out", "ws", "data"), read=("slots", "data")).items() for n in names]


@pytest.mark.parametrize("call,name", PLACES)
@pytest.mark.parametrize("other", ["cpu", "cuda:1"])
def test_refused_on_the_host(monkeypatch, call, name, other):
    _build.build()

    def reached(fn, *a):
        raise AssertionError("%s was called" % fn)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_ffi, "call", reached)
    with FakeTensorMode(allow_non_fake_inputs=True):
        t = tensors("cuda:0")
        t[name] = tensors(other)[name]
        with pytest.raises(ValueError, match="cuda:0"):
            calls(t)[call]()


@pytest.mark.gpu
@pytest.mark.parametrize("call,name", PLACES)
def test_refused_on_the_gpu(call, name):
    t = tensors("cuda")
    calls(t)[call]()                              # as it should be
    t[name] = t[name].cpu()
    with pytest.raises(ValueError, match="cuda:0"):
        calls(t)[call]()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_workspace_with_gaps_is_refused_and_another_type_is_counted_in_bytes():
    t = tensors("cuda")
    t["ws"] = t["ws"][::2]
    with pytest.raises(ValueError, match="contiguous"):
        calls(t)["attention"]()
    need = int(_ffi.fn("ql_kv4_attention_workspace")(NH, NKV, HD))
    t["ws"] = torch.zeros(-(-need // 4), dtype=torch.int32, device="cuda")
    calls(t)["attention"]()
    t["ws"] = t["ws"][:need // 4 - 4].contiguous()
    with pytest.raises(_ffi.QLError):
        calls(t)["attention"]()

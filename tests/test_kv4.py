"""Serving from the paged 4-bit cache, on the host: the C ABI refuses what it does not support before
any CUDA call, and the oracle's 4-bit groups keep what they promise."""
import ctypes

import numpy as np
import pytest

from oracle import kv4 as ok
from webpytorch_b200 import _build, _ffi


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _ffi.load()


v = ctypes.c_void_p


def _plan(lib, **kw):
    a = dict(prev=16, new=32, n=4, table=64, stride=8, width=8, free=128, cap=32, n_free=256, page=16, max_tokens=8,
             lens=512, cu=1024, slots=2048, pos=4096, req=8192, left=16384, ws=32768, ws_bytes=1 << 12)
    a.update(kw)
    return lib.ql_kv_plan(v(a["prev"]), v(a["new"]), a["n"], v(a["table"]), a["stride"], a["width"], v(a["free"]),
                          a["cap"], v(a["n_free"]), a["page"], a["max_tokens"], v(a["lens"]), v(a["cu"]), v(a["slots"]),
                          v(a["pos"]), v(a["req"]), v(a["left"]), v(a["ws"]), a["ws_bytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), 1), (dict(page=8), 1), (dict(page=24), 1), (dict(page=8192), 1), (dict(stride=4), 1), (dict(width=0), 1),
    (dict(cap=0), 1), (dict(max_tokens=-1), 1), (dict(slots=0), 1), (dict(prev=0), 1), (dict(lens=16), 1),
    (dict(left=256), 1), (dict(n=20000, ws=0), 1), (dict(n=20000, ws_bytes=8), 1), (dict(width=1 << 20, stride=1 << 20, page=4096), 3),
])
def test_plan_refuses(lib, kw, code):
    assert _plan(lib, **kw) == code
    assert lib.ql_last_error()


def _rope(lib, **kw):
    a = dict(qkv=16, dtype=0, ld=768, T=2, NH=4, NKV=1, HD=128, pos=16, cos=16, sin=16, lmax=8, rot=128, qw=None, kw=None,
             eps=1e-6, q=16, k=None, cache=16, pages=4, page=16, group=64, slots=16)
    a.update(kw)
    return lib.ql_qk_norm_rope(v(a["qkv"]), a["dtype"], a["ld"], a["T"], a["NH"], a["NKV"], a["HD"], v(a["pos"]),
                               v(a["cos"]), v(a["sin"]), a["lmax"], a["rot"], a["qw"], a["kw"], a["eps"], v(a["q"]),
                               v(a["k"]), v(a["cache"]), a["pages"], a["page"], a["group"], v(a["slots"]), None)


@pytest.mark.parametrize("kw", [
    dict(HD=96, ld=4096), dict(ld=767), dict(dtype=3), dict(rot=124), dict(rot=136), dict(rot=-8), dict(lmax=0),
    dict(k=16), dict(cache=None), dict(slots=None), dict(group=16), dict(group=256), dict(page=48), dict(pages=0),
    dict(cache=24), dict(NKV=0), dict(T=-1), dict(qkv=0), dict(HD=64, group=128),
])
def test_qk_norm_rope_refuses(lib, kw):
    assert _rope(lib, **kw) == 1
    assert lib.ql_last_error()


def _attn(lib, **kw):
    a = dict(q=16, dtype=2, ldq=512, T=4, NH=4, NKV=2, HD=128, cache=16, pages=4, page=16, group=64, table=16, stride=4,
             width=4, lens=16, cu=None, B=4, scale=1.0, window=0, out=16, ws=256, ws_bytes=1 << 30)
    a.update(kw)
    return lib.ql_kv4_attention(v(a["q"]), a["dtype"], a["ldq"], a["T"], a["NH"], a["NKV"], a["HD"], v(a["cache"]),
                                a["pages"], a["page"], a["group"], v(a["table"]), a["stride"], a["width"], v(a["lens"]),
                                v(a["cu"]), a["B"], a["scale"], a["window"], v(a["out"]), v(a["ws"]), a["ws_bytes"], None)


@pytest.mark.parametrize("kw", [
    dict(HD=80, ldq=4096), dict(NH=5), dict(NKV=0), dict(dtype=-1), dict(ldq=511), dict(T=3), dict(B=0), dict(window=-1),
    dict(stride=3), dict(width=0), dict(page=17), dict(group=33), dict(pages=0), dict(cache=8), dict(q=0), dict(lens=0),
    dict(out=0), dict(page=4096, width=1 << 20, stride=1 << 20),
])
def test_attention_refuses(lib, kw):
    assert _attn(lib, **kw) == 1
    assert lib.ql_last_error()


def test_read_refuses(lib):
    good = [v(16), 4, 2, 128, 16, 64, v(16), 3, v(16), v(16), None]
    for i, x in ((0, v(0)), (0, v(8)), (1, 0), (3, 72), (4, 20), (5, 48), (6, v(0)), (7, -1), (8, v(0))):
        a = list(good)
        a[i] = x
        assert lib.ql_kv4_read(*a) == 1, i


def test_empty_calls_are_noops(lib):
    assert _rope(lib, T=0) == 0
    assert _attn(lib, T=0) == 0
    assert lib.ql_kv4_read(v(16), 4, 2, 128, 16, 64, v(16), 0, v(16), v(16), None) == 0


def test_block_bytes(lib):
    assert lib.ql_kv4_block_bytes(128, 64) == 2304
    assert lib.ql_kv4_block_bytes(64, 32) == 1280
    assert lib.ql_kv4_block_bytes(64, 128) == lib.ql_kv4_block_bytes(100, 32) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
def test_oracle_groups_are_within_half_a_step(group):
    """|x - value| <= s / 2 plus the roundings: m to 11 bits, and the value to 11 bits."""
    x = np.random.default_rng(group).standard_normal((40, 128)).astype(np.float32) * 3
    n, s, m = ok.quantise(x, group)
    err = np.abs(ok.values(n, s, m) - x).reshape(40, -1, group)
    # the scale's rounding moves the last code by at most 15 * 2^-11 of a step
    bound = s.astype(np.float64) * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -10 * np.abs(x).max()
    assert (err <= bound[..., None]).all()


def test_oracle_groups_that_are_not_finite_or_constant():
    x = np.zeros((3, 64), np.float32)
    x[0, 5] = np.inf
    x[1, 40] = 70000.0
    x[2] = 1.5
    val = ok.values(*ok.quantise(x, 32))
    assert np.isnan(val[0, :32]).all() and (val[0, 32:] == 0).all()
    assert np.isnan(val[1, 32:]).all() and (val[2] == 1.5).all()

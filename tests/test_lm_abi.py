"""CPU: the language-model entry points check their arguments on the host (fake aligned
device addresses, never dereferenced) and their schemas have Meta kernels."""
from __future__ import annotations

import ctypes
import math

import torch


def _rows(rows, cols, dtype=1, data=1 << 20, strides=None):
    from thintnpu_b200 import _lib
    d = _lib.TtnTensor()
    d.data, d.ndim, d.dtype = data, 2, dtype
    d.sizes[0], d.sizes[1] = rows, cols
    d.strides[0], d.strides[1] = strides or (cols, 1)
    return d


def test_route_argument_errors():
    from thintnpu_b200 import _lib
    lib = _lib.lib()
    W, I = 2 << 20, 3 << 20

    def route(d, k=2, groups=1, top=1, gt=1, flags=0, scale=1.0, bias=None, w=W, i=I):
        return lib.ttn_route_experts(ctypes.byref(d) if d else None, bias, k, groups, top, gt, flags, scale, w, i, None)

    assert route(None) == 1 and b"null descriptor" in lib.ttn_last_error()
    assert route(_rows(4, 16, dtype=3)) == 2 and b"dtype" in lib.ttn_last_error()
    assert route(_rows(-1, 16)) == 1
    assert route(_rows(4, 16, data=None)) == 1 and b"null data" in lib.ttn_last_error()
    assert route(_rows(4, 16, data=(1 << 20) + 2)) == 1 and b"aligned" in lib.ttn_last_error()
    assert route(_rows(4, 0)) == 2 and route(_rows(4, 1025)) == 2 and b"1024" in lib.ttn_last_error()
    assert route(_rows(4, 16), k=0) == 2 and route(_rows(4, 16), k=17) == 2 and route(_rows(4, 64), k=17) == 2
    assert route(_rows(4, 16), groups=3) == 1 and route(_rows(4, 64), groups=64) == 1 and route(_rows(4, 16), groups=0) == 1
    assert route(_rows(4, 16), groups=4, top=5) == 1 and route(_rows(4, 16), groups=4, top=0) == 1
    assert route(_rows(4, 16), gt=3) == 1 and route(_rows(4, 16), flags=4) == 1
    assert route(_rows(4, 16), scale=math.nan) == 1 and route(_rows(4, 16), scale=math.inf) == 1
    assert route(_rows(4, 16), w=None) == 1 and route(_rows(4, 16), i=None) == 1
    assert route(_rows(4, 16), bias=(1 << 20) + 1) == 1
    three = _rows(4, 16)
    three.ndim = 3
    assert route(three) == 1 and b"two dims" in lib.ttn_last_error()
    assert route(_rows(0, 16), w=None, i=None) == 0  # nothing to do


def test_logprobs_argument_errors():
    from thintnpu_b200 import _lib
    lib = _lib.lib()
    A = [i << 20 for i in range(2, 8)]

    def lp(d, tokens=A[0], scale=1.0, top=2, out=A[1], ent=A[2], tl=A[3], tt=A[4]):
        return lib.ttn_token_logprobs(ctypes.byref(d) if d else None, tokens, scale, top, out, ent, tl, tt, None)

    assert lp(None) == 1
    assert lp(_rows(4, 50, dtype=7)) == 2
    assert lp(_rows(4, 0)) == 2 and lp(_rows(4, (1 << 20) + 1)) == 2 and b"2^20" in lib.ttn_last_error()
    assert lp(_rows(4, 50, strides=(1, 4))) == 2 and b"stride" in lib.ttn_last_error()
    assert lp(_rows(4, 50), top=33) == 2 and lp(_rows(4, 50), top=-1) == 2 and lp(_rows(4, 5), top=6) == 2
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert lp(_rows(4, 50), scale=scale) == 1 and b"scale" in lib.ttn_last_error()
    assert lp(_rows(4, 50), tl=None) == 1 and lp(_rows(4, 50), tt=None) == 1
    assert lp(_rows(4, 50), tokens=None) == 1 and lp(_rows(4, 50), out=None) == 1
    assert lp(_rows(4, 50), tokens=A[0] + 4) == 1
    assert lp(_rows(0, 50), tl=None, tt=None) == 0


def test_expert_mlp_argument_errors_and_workspace():
    from thintnpu_b200 import _lib
    lib = _lib.lib()
    size = lib.ttn_expert_mlp_workspace_size
    base = dict(dtype=2, x=1 << 20, xs=64, t=4, h=64, ids=2 << 20, w=3 << 20, k=2, gu=4 << 20, dn=5 << 20, e=8, f=32,
                out=6 << 20, os=64, ws=7 << 20, bytes=1 << 30)

    def mlp(**kw):
        a = dict(base, **kw)
        return lib.ttn_expert_mlp(a["dtype"], a["x"], a["xs"], a["t"], a["h"], a["ids"], a["w"], a["k"], a["gu"],
                                  a["dn"], a["e"], a["f"], a["out"], a["os"], a["ws"], a["bytes"], None)

    assert mlp(dtype=1) == 2 and b"float16" in lib.ttn_last_error()
    for bad in (dict(t=-1), dict(h=0), dict(f=0), dict(e=0), dict(e=1025), dict(k=0), dict(k=33), dict(t=1 << 40)):
        assert mlp(**bad) == 1, bad
        full = dict(base, **bad)
        assert size(full["t"], full["h"], full["f"], full["e"], full["k"]) == 0
    assert mlp(h=68, xs=72, os=72) == 2 and mlp(f=40) == 2 and b"multiple" in lib.ttn_last_error()
    for name in ("x", "ids", "w", "gu", "dn", "out"):
        assert mlp(**{name: None}) == 1 and b"null" in lib.ttn_last_error()
    for name in ("x", "gu", "dn", "out"):
        assert mlp(**{name: base[name] + 8}) == 1 and b"16-byte" in lib.ttn_last_error()
    assert mlp(ids=base["ids"] + 2) == 1 and mlp(w=base["w"] + 2) == 1
    assert mlp(xs=68) == 1 and mlp(os=56) == 1 and mlp(xs=0) == 1 and b"strides" in lib.ttn_last_error()
    assert mlp(bytes=16) == 1 and mlp(ws=None) == 1 and mlp(ws=base["ws"] + 16) == 1 and b"workspace" in lib.ttn_last_error()
    assert mlp(t=0, x=None, out=None, ws=None, bytes=0) == 0
    assert 0 < size(1, 64, 32, 8, 2) <= size(64, 64, 32, 8, 2) <= size(4096, 64, 32, 8, 2)
    assert size(64, 64, 32, 8, 2) % 256 == 0


def test_other_entry_points_still_refuse_bf16():
    from thintnpu_b200 import _lib
    lib = _lib.lib()
    d = _rows(4, 16, dtype=2)
    assert lib.ttn_silu(ctypes.byref(d), ctypes.byref(d), None) == 2 and b"float16/float32" in lib.ttn_last_error()


def test_meta_shapes():
    from thintnpu_b200 import library  # noqa: F401
    nf = torch.ops.thin_native_flow
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)
    w, ids = nf.route_experts(meta(5, 64), 8, "sigmoid", meta(64, dtype=torch.float32), 8, 4, 2, True, 2.5)
    assert w.shape == ids.shape == (5, 8) and w.dtype == torch.float32 and ids.dtype == torch.int32
    y = nf.expert_mlp(meta(5, 64), ids, w, meta(8, 64, 64), meta(8, 64, 32))
    assert y.shape == (5, 64) and y.dtype == torch.bfloat16
    out = nf.token_logprobs(meta(5, 1000), meta(5, dtype=torch.int64), 3, 1.0)
    assert [tuple(t.shape) for t in out] == [(5,), (5,), (5, 3), (5, 3)]
    assert out[3].dtype == torch.int32 and out[0].dtype == torch.float32
    for op in ("route_experts", "expert_mlp", "token_logprobs"):
        for key in ("CUDA", "AutogradCUDA", "Meta"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key("thin_native_flow::" + op, key), (op, key)

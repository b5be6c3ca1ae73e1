"""Refusals of the four-bit and mixture-of-experts calls; they run before any CUDA call, so
fake pointers do. Also the plain 64-bit forms against known answers."""
import numpy as np
import pytest

import mx4_reference as R
from swiglu_b200 import _lib

F = 0x7F0000000000  # never dereferenced


def L():
    return _lib.lib()


def test_reference_known_answers():
    x = np.zeros((1, 33))
    x[0, :12] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.2, -0.25, -6.9, 4.0]
    codes, scales = R.quantize(x)
    assert scales.tolist() == [[127, 0]]
    v = R.values(codes, scales, 33)[0]
    # ties go to the even code; 7 lies beyond 6
    assert v[:12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, 0, -6, 4]
    x[0, 32] = np.inf
    codes, scales = R.quantize(x)
    assert scales.tolist() == [[127, 255]] and np.isnan(R.values(codes, scales, 33)[0, 32])
    assert R.quantize(np.full((1, 1), 2.0 ** -130))[1].tolist() == [[0]]
    assert R.select(np.array([[1., 2., 2., np.nan, -np.inf]]), 4).tolist() == [[3, 1, 2, 0]]


def test_quantize_guards():
    q, d = L().swb_mx4_quantize, L().swb_mx4_dequantize
    a, b, c = F, F + (1 << 30), F + (2 << 30)
    assert q(3, a, 32, b, c, 1, 32, None) == _lib.SWB_E_TYPE
    assert q(-1, a, 32, b, c, 1, 32, None) == _lib.SWB_E_TYPE
    assert q(0, a, 31, b, c, 1, 32, None) == _lib.SWB_E_SHAPE      # rows overlap
    assert q(0, a, 32, b, c, -1, 32, None) == _lib.SWB_E_SHAPE
    assert q(0, None, 32, b, c, 1, 32, None) == _lib.SWB_E_INPUT
    assert q(0, a, 32, None, c, 1, 32, None) == _lib.SWB_E_INPUT
    assert q(0, a, 32, b, None, 1, 32, None) == _lib.SWB_E_INPUT
    assert q(0, a, 32, a + 60, c, 1, 32, None) == _lib.SWB_E_OVERLAP_INPUT
    assert q(0, a, 32, b, b + 15, 1, 32, None) == _lib.SWB_E_OVERLAP_OUTPUT
    # nothing to do: no launch, so it succeeds without a GPU
    assert q(0, a, 32, b, c, 0, 32, None) == _lib.SWB_OK and q(0, a, 0, b, c, 4, 0, None) == _lib.SWB_OK
    assert d(5, b, c, a, 32, 1, 32, None) == _lib.SWB_E_TYPE
    assert d(0, b, c, a, 8, 1, 32, None) == _lib.SWB_E_SHAPE
    assert d(0, b, c, None, 32, 1, 32, None) == _lib.SWB_E_INPUT
    assert d(0, b, c, b, 32, 1, 32, None) == _lib.SWB_E_OVERLAP_INPUT
    assert d(2, b, c, a, 32, 0, 32, None) == _lib.SWB_OK


def test_project_guards():
    f = L().swb_mx4_project
    w, s, x, o, e = (F + k * (1 << 30) for k in range(5))
    ok = dict(type=0, w=w, s=s, x=x, pitch=64, bias=None, res=None, out=o, tokens=2, rows=8, cols=64, flags=0)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["type"], a["w"], a["s"], a["x"], a["pitch"], a["bias"], a["res"], a["out"], a["tokens"], a["rows"],
                 a["cols"], a["flags"], None)
    assert call(type=2) == _lib.SWB_E_TYPE
    assert call(flags=4) == _lib.SWB_E_INPUT
    assert call(tokens=-1) == _lib.SWB_E_SHAPE and call(rows=0) == _lib.SWB_E_SHAPE
    assert call(cols=0) == _lib.SWB_E_SHAPE and call(cols=_lib.SWB_MX4_MAX_DIM + 1) == _lib.SWB_E_SHAPE
    assert call(pitch=63) == _lib.SWB_E_SHAPE and call(tokens=_lib.SWB_MX4_MAX_TOKENS + 1) == _lib.SWB_E_SHAPE
    assert call(tokens=0, out=None) == _lib.SWB_OK
    assert call(w=None) == _lib.SWB_E_INPUT and call(x=None) == _lib.SWB_E_INPUT and call(s=None) == _lib.SWB_E_INPUT
    assert call(out=None) == _lib.SWB_E_FLOAT_OUTPUT
    assert call(out=None, flags=_lib.SWB_HALF_OUT) == _lib.SWB_E_HALF_OUTPUT
    assert call(flags=_lib.SWB_RESIDUAL) == _lib.SWB_E_RESIDUAL
    assert call(w=w + 8) == _lib.SWB_E_ALIGNMENT
    assert call(out=x) == _lib.SWB_E_OVERLAP_INPUT and call(out=w) == _lib.SWB_E_OVERLAP_INPUT
    assert call(out=s) == _lib.SWB_E_OVERLAP_INPUT and call(bias=o + 4) == _lib.SWB_E_OVERLAP_INPUT
    # the residual may be the output itself only when both have one type
    assert call(res=o, flags=_lib.SWB_RESIDUAL) == _lib.SWB_E_OVERLAP_INPUT
    assert call(res=o + 2, flags=_lib.SWB_RESIDUAL | _lib.SWB_HALF_OUT) == _lib.SWB_E_OVERLAP_INPUT


def test_matmul_guards():
    f = L().swb_mx4_matmul
    xc, xs, w, s, o, e = (F + k * (1 << 30) for k in range(6))
    ok = dict(type=0, xc=xc, xs=xs, w=w, s=s, bias=None, res=None, out=o, tokens=2, rows=8, cols=64, flags=0)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["type"], a["xc"], a["xs"], a["w"], a["s"], a["bias"], a["res"], a["out"], a["tokens"], a["rows"],
                 a["cols"], a["flags"], None)
    assert call(type=2) == _lib.SWB_E_TYPE and call(flags=_lib.SWB_HALF_OUT) == _lib.SWB_E_INPUT
    assert call(tokens=-1) == _lib.SWB_E_SHAPE and call(rows=0) == _lib.SWB_E_SHAPE and call(cols=0) == _lib.SWB_E_SHAPE
    assert call(rows=_lib.SWB_MX4_MAX_DIM + 1) == _lib.SWB_E_SHAPE
    assert call(tokens=0, out=None) == _lib.SWB_OK
    for name in ("xc", "xs", "w", "s"):
        assert call(**{name: None}) == _lib.SWB_E_INPUT, name
    assert call(out=None) == _lib.SWB_E_HALF_OUTPUT
    assert call(flags=_lib.SWB_RESIDUAL) == _lib.SWB_E_RESIDUAL
    assert call(xc=xc + 8) == _lib.SWB_E_ALIGNMENT and call(w=w + 4) == _lib.SWB_E_ALIGNMENT
    for name in ("xc", "xs", "w", "s"):
        assert call(out=ok[name]) == _lib.SWB_E_OVERLAP_INPUT, name
    assert call(bias=o + 4) == _lib.SWB_E_OVERLAP_INPUT
    assert call(res=o + 2, flags=_lib.SWB_RESIDUAL) == _lib.SWB_E_OVERLAP_INPUT


def test_moe_guards():
    f = L().swb_moe
    x, r, g, u, d, y, ws, gs, us, ds, ids, wt = (F + k * (1 << 30) for k in range(12))
    ok = dict(type=0, flags=0, x=x, pitch=64, r=r, g=g, u=u, d=d, gs=None, us=None, ds=None, y=y, ids=None, wt=None,
              tokens=2, hidden=64, inter=96, experts=4, topk=2, ws=ws, bytes=1 << 20)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["type"], a["flags"], a["x"], a["pitch"], a["r"], a["g"], a["u"], a["d"], a["gs"], a["us"], a["ds"],
                 a["y"], a["ids"], a["wt"], a["tokens"], a["hidden"], a["inter"], a["experts"], a["topk"], a["ws"],
                 a["bytes"], None)
    assert call(type=2) == _lib.SWB_E_TYPE and call(flags=4) == _lib.SWB_E_INPUT
    for bad in (dict(tokens=-1), dict(tokens=65), dict(hidden=0), dict(hidden=100001), dict(inter=0),
                dict(inter=100001), dict(experts=0), dict(experts=257), dict(topk=0), dict(topk=5), dict(pitch=63),
                dict(experts=32, topk=17)):
        assert call(**bad) == _lib.SWB_E_SHAPE, bad
    assert call(tokens=0, y=None) == _lib.SWB_OK
    for name in ("x", "r", "g", "u", "d"):
        assert call(**{name: None}) == _lib.SWB_E_INPUT, name
    assert call(flags=_lib.SWB_MOE_MX4) == _lib.SWB_E_INPUT                       # no scales
    assert call(flags=_lib.SWB_MOE_MX4, gs=gs, us=us) == _lib.SWB_E_INPUT
    assert call(y=None) == _lib.SWB_E_HALF_OUTPUT
    need = L().swb_moe_workspace_bytes(2, 4, 2, 96)
    assert need > 0
    assert call(bytes=need - 1) == _lib.SWB_E_WORKSPACE and call(ws=None) == _lib.SWB_E_WORKSPACE
    assert call(ws=ws + 16) == _lib.SWB_E_ALIGNMENT
    assert call(flags=_lib.SWB_MOE_MX4, gs=gs, us=us, ds=ds, u=u + 4) == _lib.SWB_E_ALIGNMENT
    assert call(y=x) == _lib.SWB_E_OVERLAP_INPUT and call(ids=d) == _lib.SWB_E_OVERLAP_INPUT
    assert call(flags=_lib.SWB_MOE_MX4, gs=gs, us=us, ds=ds, wt=ds) == _lib.SWB_E_OVERLAP_INPUT
    assert call(ids=ids, wt=ids + 8) == _lib.SWB_E_OVERLAP_OUTPUT and call(y=ws + 64) == _lib.SWB_E_OVERLAP_OUTPUT


def test_values_off_their_size_are_refused():
    """Addresses that no value of the type can have, which a kernel could not read."""
    P, E = _lib.SWB_RESIDUAL, _lib.SWB_E_ALIGNMENT
    x, c, s, o, b, r = (F + k * (1 << 30) for k in range(6))
    for kind, off in ((0, 1), (1, 1), (2, 2)):
        assert L().swb_mx4_quantize(kind, x + off, 64, c, s, 2, 64, None) == E
        assert L().swb_mx4_dequantize(kind, c, s, o + off, 64, 2, 64, None) == E
    for a in ((x + 1, b, r, o), (x, b + 1, r, o), (x, b, r + 1, o), (x, b, r, o + 2)):
        assert L().swb_mx4_project(0, c, s, a[0], 64, a[1], a[2], a[3], 2, 32, 64, P, None) == E
    assert L().swb_mx4_project(0, c, s, x, 64, b, r, o + 1, 2, 32, 64, P | _lib.SWB_HALF_OUT, None) == E
    for a in ((b + 1, r, o), (b, r + 1, o), (b, r, o + 1)):
        assert L().swb_mx4_matmul(0, x, x + (1 << 29), c, s, *a, 2, 32, 64, P, None) == E
    q = [F + k * (1 << 30) for k in range(8)]
    for i in range(8):  # x, router, gate, up, down, y, ids, weights
        v = list(q)
        v[i] += 2 if i > 5 else 1
        assert L().swb_moe(0, 0, v[0], 64, *v[1:5], None, None, None, *v[5:8], 2, 64, 96, 4, 2, F + (1 << 35), 1 << 20,
                           None) == E, i


def test_moe_workspace_sizes():
    w = L().swb_moe_workspace_bytes
    assert w(0, 8, 2, 64) > 0 and w(64, 256, 16, 100000) > 64 * 16 * 100000 * 2
    for bad in ((-1, 8, 2, 64), (65, 8, 2, 64), (1, 0, 1, 64), (1, 257, 2, 64), (1, 8, 0, 64), (1, 8, 9, 64),
                (1, 32, 17, 64), (1, 8, 2, 0), (1, 8, 2, 100001)):
        assert w(*bad) == 0, bad


def test_python_refusals_without_a_gpu():
    torch = pytest.importorskip("torch")
    import swiglu_b200 as S
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.mx4_quantize(x)
    q, s = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.mx4_project(x, q, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.moe_out(x, x, x, x, x, x, x, 1)
    with pytest.raises(RuntimeError, match="invalid shape"):
        S.moe_workspace(65, 8, 2, 64, device="cpu")

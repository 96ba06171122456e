"""Microscaled 4-bit rows on the CPU: the C ABI's refusals (no kernel is launched: every call here fails a host check) and
the Python wrappers'."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import _lib, elementwise, projection

P = 1 << 20  # a fake, aligned device address; operands lie 2^32 apart
BF16, F32, F16 = 0, 1, 2
NULL, SHAPE, DTYPE, STRIDE, EPS = 1, 2, 3, 7, 10


def addr(i: int) -> int:
    return P + (i << 32)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def quant_rows(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=64, q=addr(1), qs=32, s=addr(2), ss=2, N=4, C=64), **kw}
    return lib.hb_quant_rows_mx4(0, a["x"], a["dtype"], a["xs"], a["q"], a["qs"], a["s"], a["ss"], a["N"], a["C"])


def rms(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=64, w=addr(3), eps=1e-5, scale=addr(4), shift=addr(5), ms=64, L=2, q=addr(1),
                qs=32, s=addr(2), ss=2, N=4, C=64), **kw}
    return lib.hb_rms_modulate_mx4(0, a["x"], a["dtype"], a["xs"], a["w"], a["eps"], a["scale"], a["shift"], a["ms"],
                                   a["L"], a["q"], a["qs"], a["s"], a["ss"], a["N"], a["C"])


def residual(lib, **kw):
    a = {**dict(h=addr(6), hs=64, x=addr(0), dtype=BF16, xs=64, xb=addr(7), gate=addr(8), gs=64, local=addr(9),
                memory=1, w=addr(3), eps=1e-5, scale=addr(4), shift=addr(5), ms=64, L=2, oh=addr(10), os=64, q=addr(1),
                qs=32, s=addr(2), ss=2, N=4, C=64), **kw}
    return lib.hb_residual_rms_mx4(0, a["h"], a["dtype"], a["hs"], a["x"], a["xs"], a["xb"], a["gate"], a["gs"],
                                   a["local"], a["memory"], a["w"], a["eps"], a["scale"], a["shift"], a["ms"], a["L"],
                                   a["oh"], a["os"], a["q"], a["qs"], a["s"], a["ss"], a["N"], a["C"])


def glu(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=128, bias=addr(3), q=addr(1), qs=32, s=addr(2), ss=2, N=4, C=64), **kw}
    return lib.hb_glu_mx4(0, a["x"], a["dtype"], a["xs"], a["bias"], a["q"], a["qs"], a["s"], a["ss"], a["N"], a["C"])


@pytest.mark.parametrize("call", [quant_rows, rms, residual, glu])
@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, DTYPE), ({"N": 0}, SHAPE), ({"N": 1 << 31}, SHAPE), ({"C": 0}, SHAPE), ({"C": 48}, SHAPE),
    ({"x": 0}, NULL), ({"q": 0}, NULL), ({"s": 0}, NULL), ({"x": addr(0) + 8}, STRIDE), ({"q": addr(1) + 8}, STRIDE),
    ({"xs": 56}, STRIDE), ({"xs": 132}, STRIDE), ({"qs": 16}, STRIDE), ({"qs": 40}, STRIDE), ({"ss": 1}, STRIDE),
    ({"xs": 1 << 61}, STRIDE), ({"qs": 1 << 61}, STRIDE), ({"ss": 1 << 61}, STRIDE), ({"q": addr(0) + 64}, STRIDE),
    ({"s": addr(0) + 17}, STRIDE), ({"s": addr(1) + 17}, STRIDE), ({"xs": -64}, STRIDE), ({"ss": -2}, STRIDE),
])
def test_row_refusals(lib, call, kw, status):
    assert call(lib, **kw) == status
    assert lib.hb_last_error()


@pytest.mark.parametrize("call", [rms, residual])
@pytest.mark.parametrize("kw,status", [
    ({"w": 0}, NULL), ({"eps": -1.0}, EPS), ({"eps": float("nan")}, EPS), ({"scale": 0}, NULL), ({"shift": 0}, NULL),
    ({"w": addr(3) + 2}, STRIDE), ({"L": 3}, SHAPE), ({"L": 0}, SHAPE), ({"ms": 32}, STRIDE), ({"q": addr(3)}, STRIDE),
    ({"s": addr(3) + 255}, STRIDE), ({"q": addr(4) + 128}, STRIDE), ({"C": 16416, "xs": 40000, "qs": 20000}, SHAPE),
])
def test_norm_refusals(lib, call, kw, status):
    assert call(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    ({"h": 0}, NULL), ({"oh": 0}, NULL), ({"memory": -1}, SHAPE), ({"oh": addr(6)}, STRIDE),
    ({"oh": addr(0) + 128}, STRIDE), ({"oh": addr(1)}, STRIDE), ({"os": 60}, STRIDE), ({"q": addr(9) + 16}, STRIDE),
])
def test_residual_refusals(lib, kw, status):
    assert residual(lib, **kw) == status


def test_glu_refusals(lib):
    assert glu(lib, q=addr(3)) == STRIDE
    assert glu(lib, s=addr(3) + 511) == STRIDE
    assert glu(lib, xs=64) == STRIDE
    assert glu(lib, bias=addr(3) + 2) == STRIDE
    assert glu(lib, C=(1 << 24) + 32, xs=1 << 26, qs=1 << 24, ss=1 << 20) == SHAPE


def proj(lib, **kw):
    a = {**dict(x=addr(0), xs=32, sx=addr(1), sxs=2, w=addr(2), ws=32, sw=addr(3), sws=2, bias=addr(4), out=addr(5),
                dtype=BF16, os=24, M=4, K=64, F=24), **kw}
    return lib.hb_proj_mx4(0, a["x"], a["xs"], a["sx"], a["sxs"], a["w"], a["ws"], a["sw"], a["sws"], a["bias"],
                           a["out"], a["dtype"], a["os"], a["M"], a["K"], a["F"])


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, DTYPE), ({"M": 0}, SHAPE), ({"F": 0}, SHAPE), ({"K": 0}, SHAPE), ({"K": 48}, SHAPE),
    ({"M": (1 << 21) + 1}, SHAPE), ({"F": (1 << 21) + 1}, SHAPE), ({"K": (1 << 23) + 32}, SHAPE), ({"x": 0}, NULL),
    ({"sx": 0}, NULL), ({"w": 0}, NULL), ({"sw": 0}, NULL), ({"out": 0}, NULL), ({"x": addr(0) + 8}, STRIDE),
    ({"w": addr(2) + 8}, STRIDE), ({"bias": addr(4) + 2}, STRIDE), ({"xs": (1 << 22) + 16}, STRIDE),
    ({"ws": (1 << 22) + 16}, STRIDE), ({"xs": 16}, STRIDE), ({"ws": 16}, STRIDE), ({"xs": 40}, STRIDE),
    ({"ws": 40}, STRIDE), ({"sxs": 1}, STRIDE), ({"sws": 1}, STRIDE), ({"os": 23}, STRIDE), ({"out": addr(5) + 1}, STRIDE),
    ({"dtype": F32, "out": addr(5) + 2}, STRIDE), ({"xs": 1 << 61}, STRIDE), ({"sxs": 1 << 61}, STRIDE),
    ({"sws": 1 << 61}, STRIDE), ({"os": 1 << 61}, STRIDE), ({"out": addr(0) + 64}, STRIDE), ({"out": addr(2)}, STRIDE),
    ({"out": addr(1) + 6}, STRIDE), ({"out": addr(3) + 46}, STRIDE), ({"out": addr(4) + 8}, STRIDE),
])
def test_proj_refusals(lib, kw, status):
    assert proj(lib, **kw) == status


def test_wrappers_refuse_cpu_tensors():
    x, w = torch.zeros(2, 3, 64), torch.zeros(64)
    b = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    for call in (lambda: elementwise.quantize_rows_mx4(x), lambda: elementwise.glu_mx4(x),
                 lambda: elementwise.rms_modulate_mx4(x, w, 1e-5), lambda: elementwise.residual_rms_mx4(x, x, w, 1e-5),
                 lambda: projection.linear_mx4(b(2, 32), b(2, 2), b(8, 32), b(8, 2))):
        with pytest.raises(ValueError, match="ROCm device"):
            call()

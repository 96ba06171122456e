"""The 8-bit and 4-bit operators on the CPU: the C ABI's refusals (no kernel is launched: every call here fails a host
check), the Python wrappers' refusal of CPU tensors, and the weights' 4-bit form against a search for the nearest code
in fp64."""
from __future__ import annotations

import numpy as np
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
    a = {**dict(x=addr(0), dtype=BF16, xs=64, q=addr(1), qs=64, s=addr(2), N=4, C=64), **kw}
    return lib.hb_quant_rows(0, a["x"], a["dtype"], a["xs"], a["q"], a["qs"], a["s"], a["N"], a["C"])


def rms_q8(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=64, w=addr(3), eps=1e-5, scale=addr(4), shift=addr(5), ms=64, L=2, q=addr(1),
                qs=64, s=addr(2), N=4, C=64), **kw}
    return lib.hb_rms_modulate_q8(0, a["x"], a["dtype"], a["xs"], a["w"], a["eps"], a["scale"], a["shift"], a["ms"],
                                  a["L"], a["q"], a["qs"], a["s"], a["N"], a["C"])


def residual_q8(lib, **kw):
    a = {**dict(h=addr(6), hs=64, x=addr(0), dtype=BF16, xs=64, xb=addr(7), gate=addr(8), gs=64, local=addr(9),
                memory=1, w=addr(3), eps=1e-5, scale=addr(4), shift=addr(5), ms=64, L=2, oh=addr(10), os=64, q=addr(1),
                qs=64, s=addr(2), N=4, C=64), **kw}
    return lib.hb_residual_rms_q8(0, a["h"], a["dtype"], a["hs"], a["x"], a["xs"], a["xb"], a["gate"], a["gs"],
                                  a["local"], a["memory"], a["w"], a["eps"], a["scale"], a["shift"], a["ms"], a["L"],
                                  a["oh"], a["os"], a["q"], a["qs"], a["s"], a["N"], a["C"])


def glu_q8(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=128, bias=addr(3), q=addr(1), qs=64, s=addr(2), N=4, C=64), **kw}
    return lib.hb_glu_q8(0, a["x"], a["dtype"], a["xs"], a["bias"], a["q"], a["qs"], a["s"], a["N"], a["C"])


ROW_CASES = [
    ({"dtype": 3}, DTYPE), ({"N": 0}, SHAPE), ({"N": 1 << 31}, SHAPE), ({"C": 0}, SHAPE), ({"C": 60}, SHAPE),
    ({"C": 16392, "xs": 40000, "qs": 40000}, SHAPE), ({"x": 0}, NULL), ({"q": 0}, NULL), ({"s": 0}, NULL),
    ({"x": addr(0) + 8}, STRIDE), ({"q": addr(1) + 4}, STRIDE), ({"s": addr(2) + 2}, STRIDE),
    ({"xs": 56}, STRIDE), ({"qs": 56}, STRIDE), ({"qs": 68}, STRIDE), ({"xs": 1 << 61}, STRIDE),
    ({"qs": 1 << 61}, STRIDE), ({"q": addr(0) + 64}, STRIDE), ({"s": addr(0) + 16}, STRIDE),
    ({"s": addr(1) + 16}, STRIDE), ({"xs": -64}, STRIDE),
]


@pytest.mark.parametrize("call", [quant_rows, rms_q8, residual_q8, glu_q8])
@pytest.mark.parametrize("kw,status", ROW_CASES)
def test_row_refusals(lib, call, kw, status):
    if call is glu_q8 and kw.get("xs") == 56:
        kw = {"xs": 120}
    assert call(lib, **kw) == status
    assert lib.hb_last_error()


@pytest.mark.parametrize("kw,status", [
    ({"w": 0}, NULL), ({"eps": -1.0}, EPS), ({"eps": float("nan")}, EPS), ({"scale": 0}, NULL), ({"shift": 0}, NULL),
    ({"w": addr(3) + 2}, STRIDE), ({"L": 3}, SHAPE), ({"L": 0}, SHAPE), ({"ms": 32}, STRIDE), ({"q": addr(3)}, STRIDE), ({"s": addr(3) + 252}, STRIDE),
    ({"q": addr(4) + 128}, STRIDE), ({"scale": addr(4) + 2}, STRIDE),
])
@pytest.mark.parametrize("call", [rms_q8, residual_q8])
def test_norm_refusals(lib, call, kw, status):
    assert call(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    ({"h": 0}, NULL), ({"oh": 0}, NULL), ({"memory": -1}, SHAPE), ({"oh": addr(6)}, STRIDE), ({"oh": addr(0) + 128}, STRIDE),
    ({"oh": addr(1)}, STRIDE), ({"os": 60}, STRIDE), ({"xb": addr(7) + 2}, STRIDE), ({"oh": addr(7)}, STRIDE),
    ({"gs": 60}, STRIDE), ({"q": addr(9) + 16}, STRIDE), ({"os": 1 << 61}, STRIDE),
])
def test_residual_refusals(lib, kw, status):
    assert residual_q8(lib, **kw) == status


def test_glu_refusals(lib):
    assert glu_q8(lib, q=addr(3)) == STRIDE
    assert glu_q8(lib, s=addr(3) + 508) == STRIDE
    assert glu_q8(lib, xs=64) == STRIDE
    assert glu_q8(lib, bias=addr(3) + 2) == STRIDE


def proj_q8(lib, **kw):
    a = {**dict(x=addr(0), xs=64, sx=addr(1), w=addr(2), ws=64, sw=addr(3), bias=addr(4), out=addr(5), dtype=BF16, os=24,
                M=4, K=64, F=24), **kw}
    return lib.hb_proj_q8(0, a["x"], a["xs"], a["sx"], a["w"], a["ws"], a["sw"], a["bias"], a["out"], a["dtype"],
                          a["os"], a["M"], a["K"], a["F"])


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, DTYPE), ({"M": 0}, SHAPE), ({"F": 0}, SHAPE), ({"K": 0}, SHAPE), ({"K": 40}, SHAPE),
    ({"M": (1 << 21) + 1}, SHAPE), ({"F": (1 << 21) + 1}, SHAPE), ({"x": 0}, NULL), ({"sx": 0}, NULL), ({"w": 0}, NULL),
    ({"sw": 0}, NULL), ({"out": 0}, NULL), ({"x": addr(0) + 8}, STRIDE), ({"w": addr(2) + 8}, STRIDE),
    ({"sx": addr(1) + 2}, STRIDE), ({"sw": addr(3) + 2}, STRIDE), ({"bias": addr(4) + 2}, STRIDE),
    ({"xs": (1 << 23) + 16}, STRIDE), ({"ws": (1 << 23) + 16}, STRIDE), ({"K": (1 << 23) + 16}, SHAPE),
    ({"xs": 48}, STRIDE), ({"ws": 48}, STRIDE), ({"xs": 72}, STRIDE), ({"ws": 72}, STRIDE), ({"os": 23}, STRIDE),
    ({"out": addr(5) + 1}, STRIDE), ({"dtype": F32, "out": addr(5) + 2}, STRIDE), ({"xs": 1 << 61}, STRIDE),
    ({"ws": 1 << 61}, STRIDE), ({"os": 1 << 61}, STRIDE), ({"out": addr(0) + 128}, STRIDE), ({"out": addr(2)}, STRIDE),
    ({"out": addr(1) + 8}, STRIDE), ({"out": addr(3) + 8}, STRIDE), ({"out": addr(4) + 8}, STRIDE),
])
def test_proj_q8_refusals(lib, kw, status):
    assert proj_q8(lib, **kw) == status


def proj_q4(lib, **kw):
    a = {**dict(x=addr(0), dtype=BF16, xs=64, w=addr(1), ws=32, sc=addr(2), ss=2, bias=addr(3), silu=0, out=addr(4),
                os=24, N=4, K=64, F=24), **kw}
    return lib.hb_proj_q4(0, a["x"], a["dtype"], a["xs"], a["w"], a["ws"], a["sc"], a["ss"], a["bias"], a["silu"],
                          a["out"], a["os"], a["N"], a["K"], a["F"])


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, DTYPE), ({"N": 0}, SHAPE), ({"N": (1 << 16) + 1}, SHAPE), ({"F": 0}, SHAPE), ({"K": 0}, SHAPE),
    ({"K": 48}, SHAPE), ({"x": 0}, NULL), ({"w": 0}, NULL), ({"sc": 0}, NULL), ({"out": 0}, NULL),
    ({"bias": addr(3) + 2}, STRIDE), ({"x": addr(0) + 8}, STRIDE), ({"xs": 56}, STRIDE), ({"xs": 68}, STRIDE), ({"w": addr(1) + 8}, STRIDE),
    ({"ws": 16}, STRIDE), ({"ws": 40}, STRIDE), ({"ss": 1}, STRIDE), ({"os": 23}, STRIDE), ({"out": addr(4) + 1}, STRIDE),
    ({"dtype": F32, "out": addr(4) + 2}, STRIDE), ({"xs": 1 << 61}, STRIDE), ({"ws": 1 << 61}, STRIDE),
    ({"ss": 1 << 61}, STRIDE), ({"os": 1 << 61}, STRIDE), ({"out": addr(0) + 128}, STRIDE), ({"out": addr(1)}, STRIDE),
    ({"out": addr(2) + 8}, STRIDE), ({"out": addr(3) + 8}, STRIDE),
])
def test_proj_q4_refusals(lib, kw, status):
    assert proj_q4(lib, **kw) == status


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 3, 64)
    q = x.to(torch.float8_e4m3fn)
    w = torch.zeros(64)
    for call in (lambda: elementwise.quantize_rows(x), lambda: elementwise.glu_q8(x),
                 lambda: elementwise.rms_modulate_q8(x, w, 1e-5), lambda: elementwise.residual_rms_q8(x, x, w, 1e-5),
                 lambda: projection.linear_q8(q, x[..., 0], q[0], w[:3]),
                 lambda: projection.linear_q4(x, torch.zeros(8, 32, dtype=torch.uint8),
                                              torch.zeros(8, 2, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def dequant_q4(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)
    v = E2M1[c & 7] * np.where(c & 8, -1.0, 1.0)
    return v * np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, axis=1)


@pytest.mark.parametrize("case", ["normal", "ties", "zeros", "tiny", "huge"])
def test_quantize_q4_is_the_nearest_code(case):
    rng = np.random.default_rng(3)
    w = rng.standard_normal((5, 96))
    if case == "ties":  # 6 in every group, then values on the middles, both signs
        w = np.tile(np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 0] * 2),
                    (5, 3))
    if case == "zeros":
        w[:, 32:64] = 0
        w[2] = 0
    if case == "tiny":
        w *= 2.0 ** -121
    if case == "huge":
        w *= 2.0 ** 115
    w = w.astype(np.float32)
    codes, scales = projection.quantize_q4(torch.from_numpy(w))
    assert codes.shape == (5, 48) and scales.shape == (5, 3) and codes.dtype == scales.dtype == torch.uint8
    s = scales.numpy().astype(np.float64)
    assert s.min() >= 8 and s.max() <= 250
    w64 = w.astype(np.float64)
    amax = np.abs(w64.reshape(5, 3, 32)).max(-1)
    step = np.exp2(s - 127)
    assert (amax <= 6 * step).all()
    assert ((amax > 3 * step) | (s == 8) | (amax == 0)).all()  # a power less would not hold it
    got = dequant_q4(codes.numpy(), scales.numpy())
    rep = np.repeat(step, 32, axis=1)
    near = np.abs(np.abs(w64)[..., None] / rep[..., None] - E2M1).min(-1) * rep
    np.testing.assert_array_equal(np.abs(np.abs(got) - np.abs(w64)), near)
    assert (np.sign(got) * np.sign(w64) >= 0).all()
    if case == "ties":
        np.testing.assert_array_equal(np.abs(got[0, :8]), [6, 0, 1, 1, 2, 2, 4, 4])


def test_quantize_q4_refusals():
    for bad in (torch.zeros(4, 40), torch.zeros(32), torch.zeros(0, 32), torch.full((1, 32), float("inf")),
                torch.full((1, 32), float("nan")), torch.full((1, 32), 1e38)):
        with pytest.raises(ValueError):
            projection.quantize_q4(bad)

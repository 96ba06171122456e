"""Attention over packed sequences on the CPU: the C ABI's refusals (no kernel is launched: every call here fails a host
check) and the Python wrapper's."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import _lib
from hummingbird_amd.packed_attention import packed_attention

P = 1 << 20  # a fake, aligned device address; operands lie 2^32 apart
BF16, F32, F16 = 0, 1, 2
NULL, SHAPE, DTYPE, HEAD_DIM, STRIDE, WORKSPACE, EPS = 1, 2, 3, 4, 7, 8, 10


def addr(i: int) -> int:
    return P + (i << 32)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def attend(lib, **kw):
    a = {**dict(q=addr(0), qt=256, qh=64, k=addr(1), kt=128, kh=64, v=addr(2), vt=128, vh=64, dtype=BF16, off=addr(3),
                koff=addr(4), klen=addr(5), causal=1, scale=0.125, out=addr(6), ot=256, oh=64, zero=1, T=300, Tk=300, N=2,
                H=4, G=2, D=64, ws=0, wb=0), **kw}
    return lib.hb_packed_attention(0, a["q"], a["qt"], a["qh"], a["k"], a["kt"], a["kh"], a["v"], a["vt"], a["vh"],
                                   a["dtype"], a["off"], a["koff"], a["klen"], a["causal"], a["scale"], a["out"], a["ot"],
                                   a["oh"], a["zero"], a["T"], a["Tk"], a["N"], a["H"], a["G"], a["D"], a["ws"], a["wb"])


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, DTYPE), ({"D": 32}, HEAD_DIM), ({"D": 96}, HEAD_DIM), ({"T": 0}, SHAPE), ({"Tk": -1}, SHAPE),
    ({"N": 0}, SHAPE), ({"H": 0}, SHAPE), ({"G": 0}, SHAPE), ({"G": 3}, SHAPE), ({"T": 1 << 31}, SHAPE),
    ({"Tk": 1 << 31}, SHAPE), ({"N": 1 << 21}, SHAPE), ({"H": 1 << 16, "G": 1 << 16}, SHAPE),
    ({"T": 1 << 30, "H": 4, "G": 1}, SHAPE), ({"q": 0}, NULL), ({"k": 0}, NULL), ({"v": 0}, NULL), ({"out": 0}, NULL),
    ({"off": 0}, NULL), ({"koff": 0}, NULL), ({"scale": 0.0}, EPS), ({"scale": -1.0}, EPS),
    ({"scale": float("nan")}, EPS), ({"scale": float("inf")}, EPS), ({"scale": 3e38}, EPS), ({"q": addr(0) + 8}, STRIDE),
    ({"k": addr(1) + 2}, STRIDE), ({"v": addr(2) + 4}, STRIDE), ({"out": addr(6) + 8}, STRIDE), ({"qt": 260}, STRIDE),
    ({"qh": 68}, STRIDE), ({"kt": 132}, STRIDE), ({"vh": 62}, STRIDE), ({"ot": 252}, STRIDE), ({"kt": -128}, STRIDE),
    ({"dtype": F32, "qt": 258}, STRIDE), ({"kt": (1 << 23) + 8}, STRIDE), ({"vt": (1 << 23) + 8}, STRIDE),
    ({"qt": 1 << 61}, STRIDE), ({"ot": 1 << 61}, STRIDE), ({"ot": 128}, STRIDE), ({"oh": 56}, STRIDE), ({"oh": 0}, STRIDE),
    ({"out": addr(0) + 64}, STRIDE), ({"out": addr(1)}, STRIDE), ({"out": addr(2) + 1024}, STRIDE),
    ({"out": addr(3) - 153600 + 16}, STRIDE), ({"koff": addr(6) + 32}, STRIDE), ({"klen": addr(6) + 32}, STRIDE),
    ({"off": addr(3) + 2}, STRIDE), ({"koff": addr(4) + 1}, STRIDE), ({"klen": addr(5) + 2}, STRIDE),
])
def test_refusals(lib, kw, status):
    assert attend(lib, **kw) == status
    assert lib.hb_last_error()


def test_workspace(lib):
    few = dict(T=2, Tk=9000, N=2, H=4, G=2)
    need = lib.hb_packed_workspace_size(BF16, 2, 9000, 2, 4, 2, 64)
    assert need > 0 and need % (2 * 4 * 66 * 4) == 0
    assert lib.hb_packed_workspace_size(BF16, 100000, 100000, 2, 4, 2, 64) == 0
    assert lib.hb_packed_workspace_size(3, 2, 9000, 2, 4, 2, 64) == 0
    assert attend(lib, **few) == WORKSPACE
    assert attend(lib, **few, ws=addr(7), wb=need - 1) == WORKSPACE
    assert attend(lib, **few, ws=addr(7) + 8, wb=need) == WORKSPACE
    assert attend(lib, **few, ws=addr(6), wb=need) == STRIDE
    assert attend(lib, **few, ws=addr(1) + 256, wb=need) == STRIDE
    assert attend(lib, **few, ws=addr(5) - 64, wb=need) == STRIDE


def test_strides_of_one_token_and_one_head_are_not_looked_at(lib):
    """They step to nothing: each of these calls gets as far as the missing workspace."""
    one = dict(T=1, N=1, Tk=9000, H=4, G=2)
    assert attend(lib, **one, qt=3, ot=-5) == WORKSPACE
    assert attend(lib, **one, qt=1 << 61, ot=0) == WORKSPACE
    assert attend(lib, T=2, N=1, Tk=9000, H=1, G=1, qh=7, kh=-1, vh=1 << 62, oh=0) == WORKSPACE
    assert attend(lib, T=1, N=1, Tk=1, H=1, G=1, kt=5, vt=1 << 40, q=addr(0) + 2) == STRIDE


def test_wrapper_refuses_cpu_tensors():
    q = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="ROCm device"):
        packed_attention(q, q, q, torch.tensor([0, 3], dtype=torch.int32))

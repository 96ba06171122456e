"""8-bit rows to the bit: `quantize_rows` computes nothing but s = max(max |x| / 448, 2^-100) and q = e4m3(x / s), each
operation correctly rounded, so its scales and codes are compared for equality with torch's division and conversion on
the CPU."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def check_codes(x: torch.Tensor) -> None:
    """`x` (..., C) on the CPU, finite."""
    q, s = ew.quantize_rows(x.to(DEV))
    f = x.float()
    s_ref = (f.abs().amax(-1) / 448).clamp_min(2.0 ** -100)
    q_ref = (f / s_ref[..., None]).to(torch.float8_e4m3fn)
    assert torch.equal(s.cpu(), s_ref)
    differ = q.cpu().view(torch.uint8) != q_ref.view(torch.uint8)
    assert not differ.any(), f"{int(differ.sum())} of {differ.numel()} codes, first at {differ.nonzero()[0].tolist()}"


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("rows,C", [(4000, 1536), (300, 16384), (1, 8), (1300, 64)])
def test_codes_of_normal_rows(name, rows, C):
    announce("codes", name, rows, C)
    gen = torch.Generator().manual_seed(rows + C)
    check_codes(torch.randn(rows, C, generator=gen).to(DTYPES[name]))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("exponent", [-126, -112, -101, -95, -91, -89, -65, -63, 0, 100, 126])
def test_codes_of_rows_of_any_size(name, exponent):
    """Rows whose largest value is about 2^exponent, the values spread over the codes' whole range and below it."""
    dtype = DTYPES[name]
    if dtype is torch.float16 and not -14 <= exponent <= 14:
        exponent = max(-14, min(14, exponent))
    announce("codes", name, "2^", exponent)
    gen = torch.Generator().manual_seed(exponent + 200)
    size = torch.exp2(-20 * torch.rand(400, 512, generator=gen) + exponent)
    x = torch.where(torch.rand(400, 512, generator=gen) < 0.5, -size, size) * (1 + torch.rand(400, 1, generator=gen) / 2)
    check_codes(x.to(dtype))


def test_codes_on_and_beside_the_borders():
    """fp32 rows whose quotients by the row's scale are a border between two codes, and an fp32 unit to both sides."""
    announce("codes at borders")
    codes = torch.arange(0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    border = (codes[1:] + codes[:-1]) / 2  # exact: 5 significant bits
    gen = torch.Generator().manual_seed(7)
    rows = []
    for e in (-99, -90, -80, -64, 0, 60):
        for _ in range(20):
            s = torch.exp2(torch.tensor(float(e))) * (1 + torch.rand((), generator=gen))
            amax = s * 448
            s = amax / 448
            y = border * s  # rounded: on the border or beside it
            up, down = torch.nextafter(y, torch.full_like(y, 3e38)), torch.nextafter(y, torch.zeros_like(y))
            rows.append(torch.cat([amax[None], y, up, -down, -y, up, torch.zeros(1), torch.tensor([-0.0])]))
    x = torch.stack(rows)
    x = torch.cat([x, torch.zeros(x.shape[0], -x.shape[1] % 4)], dim=1)
    assert (x.abs().amax(-1) == x[:, 0]).all()
    check_codes(x)

"""The quantised products at the ends of their operands' ranges, on the GPU: any fp32 scales of `linear_q8` and any scale
bytes of `linear_q4` against fp64."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import projection as pr

pytestmark = pytest.mark.gpu
DEV = "cuda"


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


# rows, columns, features: the few-row kernel, both of its row tiles, and tiles of every kind
SHAPES = [(7, 512, 100), (24, 256, 200), (70, 1536, 64), (40, 48, 200), (300, 256, 1600), (1000, 896, 1500), (2048, 144, 5120),
          (4000, 208, 1501), (1300, 272, 1600)]
F32_MAX = torch.finfo(torch.float32).max


def integers(gen, n, k):
    return torch.randint(-4, 5, (n, k), device=DEV, generator=gen).float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_linear_q8_of_any_scales(M, K, F, dtype):
    """Scales of every exponent, denormal ones too, rows and features against each other. Integer products below 2^24 are
    summed exactly; each scale then costs at most one fp32 rounding (2^-24) and the output its own, the least steps of
    fp32 and of the output's type where the result is below the normal range. Results beyond the largest value are
    infinite."""
    announce("linear_q8 any scales", M, K, F, dtype)
    gen = torch.Generator(device=DEV).manual_seed(M + K + F)
    x, w = integers(gen, M, K), integers(gen, F, K)

    def scales(n):
        e = torch.randint(-149, 128, (n,), device=DEV, generator=gen)
        e[::3] = torch.randint(-20, 20, (e[::3].numel(),), device=DEV, generator=gen)
        return torch.ldexp(1 + torch.rand(n, device=DEV, generator=gen), e.float()).clamp_max(3e38)
    sx, sw = scales(M), scales(F)
    sw[1::7] *= -1
    assert (sw != 0).all() and (sx != 0).all()
    ref = (x.double() @ w.double().t()) * sw.double() * sx.double()[:, None]
    got = pr.linear_q8(x.to(torch.float8_e4m3fn), sx, w.to(torch.float8_e4m3fn), sw, dtype=dtype).double()
    half_step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    least = 2.0 ** -149 + (2.0 ** -134 if dtype == torch.bfloat16 else 0.0)
    inside = ref.abs() <= F32_MAX * (1 - 2.0 ** -7)
    assert ((got - ref).abs() <= (half_step * (1 + 2.0 ** -8) + 3 * 2.0 ** -24) * ref.abs() + 2 * least)[inside].all()
    beyond = ref.abs() > F32_MAX * (1 + 2.0 ** -7)
    assert (got[beyond] == torch.sign(ref[beyond]) * float("inf")).all()
    assert beyond.any() and inside.any()


@pytest.mark.parametrize("M,K,F", SHAPES)
def test_linear_q8_of_large_weights_and_small_rows(M, K, F):
    """Weights near the largest value: the result is in range where the sum times a weight's scale alone is not, beside
    features of ordinary scales. Powers of two: the same bits."""
    announce("linear_q8 large weights", M, K, F)
    gen = torch.Generator(device=DEV).manual_seed(M + K + F + 1)
    x = torch.randn(M, K, device=DEV, generator=gen).mul(60).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = torch.randn(F, K, device=DEV, generator=gen).mul(60).clamp(-448, 448).to(torch.float8_e4m3fn)
    sx, sw = torch.rand(M, device=DEV, generator=gen) + 1, torch.rand(F, device=DEV, generator=gen) + 1
    bias = torch.randn(F, device=DEV, generator=gen)
    large = torch.arange(F, device=DEV) % 5 == 2
    up = torch.where(large, 2.0 ** 120, 2.0 ** 20)
    for dtype in (torch.bfloat16, torch.float32):
        got = pr.linear_q8(x, sx * 2.0 ** -60, w, sw * up, dtype=dtype)
        ref = pr.linear_q8(x, sx, w, sw, dtype=dtype)
        assert torch.equal(got, (ref.double() * (up.double() * 2.0 ** -60)).to(dtype))
        with_bias = pr.linear_q8(x, sx * 2.0 ** -120, w, sw * 2.0 ** 120, bias, dtype=dtype).double()
        again = pr.linear_q8(x, sx, w, sw, bias, dtype=dtype).double()
        half_step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        prod = ref.double().abs() * (1 + 2 * half_step)
        # the two round the product before the bias, or not: an fp32 step of the product, two half steps of the output
        assert ((with_bias - again).abs() <= 2.0 ** -22 * (prod + bias.double().abs()) + 2 * half_step * again.abs() * 1.01).all()


@pytest.mark.parametrize("M,K,F", [(7, 512, 100), (70, 1536, 64), (300, 256, 1600)])
def test_linear_q8_of_scales_that_are_no_numbers(M, K, F):
    announce("linear_q8 scales nan, inf, 0", M, K, F)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x, w = integers(gen, M, K).abs() + 1, integers(gen, F, K).abs() + 1
    sx, sw = torch.ones(M, device=DEV), torch.ones(F, device=DEV)
    sw[3], sw[40], sw[41] = float("nan"), float("inf"), 0.0
    sx[2], sx[5] = float("nan"), float("inf")
    got = pr.linear_q8((x).to(torch.float8_e4m3fn), sx, w.to(torch.float8_e4m3fn), sw, dtype=torch.float32)
    ref = ((x.double() @ w.double().t()) * sw.double() * sx.double()[:, None]).float()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got.nan_to_num(0.0, 1.0, -1.0), ref.nan_to_num(0.0, 1.0, -1.0))


@pytest.mark.parametrize("name", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("x", [1.0, 2.0 ** -14, 1.75 * 2.0 ** 14])
def test_linear_q4_of_every_scale_byte(name, x):
    """Every code under every byte, picked out by one value of x (both nibbles, first and later groups): the product of
    a power of two times 1.75 and a code of at most 2 bits is exact, so it comes back rounded once. Weights of 2^128 and
    more are infinite, a group of byte 255 is NaN whatever x is."""
    announce("linear_q4 every byte", name, x)
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV, dtype=torch.float64)
    levels = torch.cat([levels, -levels])
    for column in (0, 1, 32 * 5 + 7, 32 * 5 + 30):
        codes = torch.zeros(256 * 16, 96, dtype=torch.uint8, device=DEV)
        codes[:, column // 2] = torch.arange(16, device=DEV, dtype=torch.uint8).repeat(256) << (4 * (column % 2))
        byte = torch.arange(256, device=DEV).repeat_interleave(16)
        scales = torch.full((256 * 16, 6), 127, dtype=torch.uint8, device=DEV)
        scales[:, column // 32] = byte.to(torch.uint8)
        v = torch.zeros(2, 192, dtype=dtype, device=DEV)
        v[1, column] = x
        w = levels.repeat(256) * torch.exp2(byte.double() - 127)
        held = torch.where(w.abs() >= 2.0 ** 128, torch.sign(w) * float("inf"), w)
        held[byte == 255] = float("nan")
        got = pr.linear_q4(v, codes, scales)
        for row, value in ((0, 0.0), (1, x)):
            ref = (held * value).float().to(dtype)
            assert torch.equal(torch.isnan(got[row]), torch.isnan(ref)), (column, row)
            assert torch.equal(got[row].nan_to_num(0.5), ref.nan_to_num(0.5)), (column, row)


def test_linear_q4_silu_over_its_range():
    """One weight of 1 per feature hands fp32 values to the activation as they are. The exponent's factor (log2(e) to 2^-26
    of itself) and its product (2^-24) are rounded, which is |z| (2^-24 + 2^-26) of e^-z; the exponential, the sum, the
    reciprocal and the product add up to 5 further units and the output's half: (1.3 |z| + 6) 2^-24. Where the sigmoid is
    below 2^-126 it may be zero."""
    announce("linear_q4 silu range")
    K = 256
    codes = torch.zeros(K, K // 2, dtype=torch.uint8, device=DEV)
    for f in range(K):
        codes[f, f // 2] = 2 << (4 * (f % 2))  # e2m1 code 2: 1.0
    scales = torch.full((K, K // 32), 127, dtype=torch.uint8, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.cat([torch.linspace(-90, 90, 4 * K, device=DEV), 100 * (torch.rand(4 * K, device=DEV, generator=gen) - 0.9),
                   torch.randn(2 * K, device=DEV, generator=gen)]).reshape(-1, K)
    got = pr.linear_q4(x, codes, scales, silu=True).double()
    z = x.double()
    ref = z * torch.sigmoid(z)
    bound = (1.3 * torch.clamp(-z, min=0) + 6) * 2.0 ** -24 * ref.abs() + z.abs() * 2.0 ** -126
    assert ((got - ref).abs() <= bound).all()

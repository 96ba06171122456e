"""The 8-bit rows and the 8-bit and 4-bit projections on the GPU against plain fp64 implementations.

Row operators. Every step is one fp32 operation (relative error 2^-24) but the hardware sigmoid (an exponential whose
argument, up to 12 here, is rounded: 12 log2(e) 2^-24 < 2^-19) and the mean of squares (a sum of C <= 16384 terms in
lanes of at most 32 and trees: < 2^-18, halved by the root). So y is within 2^-16 of M, the value that the magnitudes of
its operands give through the same formula; s within 2^-16 max M / 448; and q s within half an e4m3 step of y (2^-4 |y|,
2^-10 s below the normal range) and that error again. h' is within half a step of its type and 2^-18 of its operands'
magnitudes.

Products. Integer operands whose products span fewer than 13 bits and whose sums stay under 2^24 are added exactly by
every kind of matrix core, so the result is the correctly rounded one: compared for equality, which an element read or
written in the wrong place cannot pass. On normal operands: fp32 sums of n terms are within n 2^-24 sum |x w|; the e4m3
cores drop what lies 13 bits below the largest of 16 products, at most 2^-13 of it for each, 16 2^-13 max <= 2^-9
sum |x w| in all, and in the 2-norm over many outputs far less (2^-13 of the result is allowed there, 8 times the
1.5e-5 that random dropped parts give).
"""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew
from hummingbird_amd import projection as pr

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def generator(*key) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def rand(gen, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (mean + std * torch.randn(shape, device=DEV, generator=gen)).to(dtype)


def check_q8(q, s, y, mag, what):
    """8-bit rows against y (fp64) of operands' magnitude `mag` >= |y|."""
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    assert q.shape == y.shape and s.shape == y.shape[:-1]
    s64 = s.double()
    top = torch.clamp(y.abs().amax(-1) / 448, min=2.0 ** -100)
    err = 2.0 ** -16 * mag.amax(-1) / 448
    assert ((s64 - top).abs() <= err + 2.0 ** -23 * top).all(), f"{what}: scale"
    got = q.double() * s64[..., None]
    bound = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s64[..., None]) + 2.0 ** -15 * mag
    bad = (got - y).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}"


WIDTHS = [64, 8, 1536, 520, 8192, 12288, 16384]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("C", WIDTHS)
def test_quantize_rows(name, C):
    announce("quantize_rows", name, C)
    gen = generator(1, C)
    x = rand(gen, 5, 3, C, std=3.0, dtype=DTYPES[name])
    q, s = ew.quantize_rows(x)
    check_q8(q, s, x.double(), x.double().abs(), "quantize_rows")


@pytest.mark.parametrize("name", list(DTYPES))
def test_quantize_rows_special_rows(name):
    """Zeros, the least values, the largest ones, one large among small, a NaN, infinities, negative zero."""
    announce("quantize_rows special", name)
    dtype = DTYPES[name]
    x = rand(generator(5), 9, 128, dtype=dtype)
    big = torch.finfo(dtype).max
    x[0] = 0
    x[1] = torch.finfo(dtype).tiny
    x[2] = big * torch.sign(x[2].float()).to(dtype)
    x[3, 5] = 1e4
    x[4, 100] = float("nan")
    x[5, 1] = float("inf")
    x[6, 127] = float("-inf")
    x[7] = -0.0
    q, s = ew.quantize_rows(x)
    rows = [0, 1, 2, 3, 7, 8]
    check_q8(q[rows], s[rows], x[rows].double(), x[rows].double().abs(), "special rows")
    assert (q[[0, 7]].float() == 0).all() and (s[[0, 7]] == 2.0 ** -100).all()
    stands_for = q.float() * s[:, None]
    assert torch.isnan(stands_for[4:7]).all()
    assert torch.isnan(s[4]) and torch.isinf(s[5:7]).all()


@pytest.mark.parametrize("name", list(DTYPES))
def test_rows_of_a_wider_tensor(name):
    """Column slices (a row stride above the width) and leading axes."""
    announce("slices", name)
    dtype, gen = DTYPES[name], generator(9)
    wide = rand(gen, 2, 7, 320, dtype=dtype)
    x = wide[..., 64:192]
    for got, ref in zip(ew.quantize_rows(x), ew.quantize_rows(x.contiguous())):
        assert torch.equal(got.float(), ref.float())
    w = rand(gen, 128, std=0.1, mean=1.0)
    for got, ref in zip(ew.rms_modulate_q8(x, w, 1e-5), ew.rms_modulate_q8(x.contiguous(), w, 1e-5)):
        assert torch.equal(got.float(), ref.float())
    h = wide[..., 192:]
    for got, ref in zip(ew.residual_rms_q8(h, x, w, 1e-5), ew.residual_rms_q8(h.contiguous(), x.contiguous(), w, 1e-5)):
        assert torch.equal(got.float(), ref.float())
    p = wide[..., 64:]
    for got, ref in zip(ew.glu_q8(p), ew.glu_q8(p.contiguous())):
        assert torch.equal(got.float(), ref.float())


def norm_reference(v, mag, weight, eps, scale, shift):
    w = weight.double()
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    y, m = v * r * w, mag * r * w.abs()
    if scale is not None:
        s, t = scale.double()[:, None], shift.double()[:, None]
        y, m = y * (1 + s) + t, m * (1 + s.abs()) + t.abs()
    return y, m


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("B,L,C,mod", [(1, 1, 64, False), (2, 37, 1536, True), (3, 5, 264, True), (1, 129, 8192, False),
                                       (2, 3, 16384, True), (1, 2000, 1024, True)])
def test_rms_modulate_q8(name, B, L, C, mod):
    announce("rms_modulate_q8", name, B, L, C, mod)
    dtype, gen = DTYPES[name], generator(B, L, C)
    x = rand(gen, B, L, C, std=2.0, dtype=dtype)
    w = rand(gen, C, std=0.1, mean=1.0)
    rows = rand(gen, B, 6 * C, std=0.3, dtype=dtype)  # scale and shift are views into the adaLN row
    scale, shift = (rows[:, C:2 * C], rows[:, :C]) if mod else (None, None)
    q, s = ew.rms_modulate_q8(x, w, 1e-5, scale, shift)
    y, m = norm_reference(x.double(), x.double().abs(), w, 1e-5, scale, shift)
    check_q8(q, s, y, m, "rms_modulate_q8")


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("B,L,C,operands", [
    (1, 1, 64, "g"), (2, 37, 1536, "gb m"), (2, 37, 1536, "l m"), (1, 91, 1536, "g"), (3, 5, 264, "gblm"),
    (1, 129, 8192, ""), (2, 3, 16384, "gblm"), (1, 2000, 1024, "g")])
def test_residual_rms_q8(name, B, L, C, operands):
    announce("residual_rms_q8", name, B, L, C, operands)
    dtype, gen = DTYPES[name], generator(B, L, C, len(operands))
    h, x = rand(gen, B, L, C, std=3.0, dtype=dtype), rand(gen, B, L, C, dtype=dtype)
    w = rand(gen, C, std=0.1, mean=1.0)
    rows = rand(gen, B, 6 * C, std=0.5, dtype=dtype)
    gate = rows[:, 2 * C:3 * C] if "g" in operands else None
    scale, shift = (rows[:, :C], rows[:, C:2 * C]) if "m" in operands else (None, None)
    bias = rand(gen, C, std=0.2, dtype=dtype) if "b" in operands else None
    local = rand(gen, C, std=0.2, dtype=dtype) if "l" in operands else None
    memory = L // 2
    out, q, s = ew.residual_rms_q8(h, x, w, 1e-5, gate=gate, x_bias=bias, local=local, memory=memory, scale=scale,
                                   shift=shift)
    v, m = x.double(), x.double().abs()
    if bias is not None:
        v, m = v + bias.double(), m + bias.double().abs()
    if gate is not None:
        g = torch.sigmoid(1 - gate.double())[:, None]
        v, m = v * g, m * g
    v, m = h.double() + v, h.double().abs() + m
    if local is not None:
        v[:, memory:] += local.double()
        m[:, memory:] += local.double().abs()
    assert out.dtype == dtype
    half_step = torch.finfo(dtype).eps / 2
    assert ((out.double() - v).abs() <= half_step * v.abs() + 2.0 ** -18 * m).all(), "h'"
    y, ym = norm_reference(v, m, w, 1e-5, scale, shift)
    check_q8(q, s, y, ym, "residual_rms_q8")


def test_residual_rms_q8_local_from_token_zero_and_past_the_end():
    announce("residual_rms_q8 memory")
    gen = generator(3)
    h, x, w = rand(gen, 2, 4, 64), rand(gen, 2, 4, 64), rand(gen, 64, mean=1.0)
    local = rand(gen, 64)
    everywhere = ew.residual_rms_q8(h, x, w, 1e-5, local=local, memory=0)[0]
    nowhere = ew.residual_rms_q8(h, x, w, 1e-5, local=local, memory=4)[0]
    assert torch.equal(nowhere, h + x)
    assert torch.equal(everywhere, (h + x) + local)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("N,F,bias", [(1, 8, True), (5, 64, False), (154, 4096, True), (33, 6144, True), (3, 16384, False),
                                      (700, 1000, True)])
def test_glu_q8(name, N, F, bias):
    announce("glu_q8", name, N, F, bias)
    dtype, gen = DTYPES[name], generator(N, F)
    p = rand(gen, N, 2 * F, std=2.0, dtype=dtype)
    b = rand(gen, 2 * F, std=0.1) if bias else None
    q, s = ew.glu_q8(p, b)
    z, m = p.double(), p.double().abs()
    if bias:
        z, m = z + b.double(), m + b.double().abs()
    act = torch.sigmoid(z[:, F:])
    # an error of the gate's sum passes through silu with a slope of at most 1.1
    check_q8(q, s, z[:, :F] * z[:, F:] * act, m[:, :F] * m[:, F:] * torch.clamp(act + 0.1, max=1.0) * 1.1, "glu_q8")


def q8_rows(gen, n, k, spread=1.0):
    x = rand(gen, n, k) * torch.exp(spread * rand(gen, n, 1))
    s = x.abs().amax(-1) / 448
    return (x / s[:, None]).to(torch.float8_e4m3fn), s


# rows, columns, features: one of each, few rows, tiles' edges on both sides, a short and a long reduction, odd sizes
Q8_SHAPES = [(1, 16, 1), (1, 1536, 7680), (7, 1536, 512), (16, 64, 100), (17, 80, 33), (33, 256, 257), (64, 6144, 96),
             (65, 144, 64), (128, 128, 128), (129, 1536, 255), (257, 1040, 513), (300, 6144, 320), (1000, 512, 1536),
             # several tiles a workgroup, of 128 x 128 and 128 x 256, one and several steps of K, odd features
             (1300, 272, 1600), (2600, 144, 2570), (5000, 128, 2600), (2048, 144, 5120), (4100, 640, 2817),
             (8200, 64, 8197), (16500, 128, 4104),  # outputs past 128 MB
             # 64 x 64, 128 x 64 and 128 x 128 tiles with three or four stages: fewer steps than stages, and more
             (40, 48, 200), (100, 1296, 70), (1300, 112, 1000), (1290, 256, 1030), (1000, 896, 1500), (2000, 96, 2000),
             (1990, 272, 1990), (2040, 1168, 1537), (1290, 272, 3060), (1300, 80, 6100),
             (4000, 208, 1501), (1291, 400, 12200), (700, 128, 7600), (3990, 1040, 1410)]  # 128 x 192 tiles


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("M,K,F", Q8_SHAPES)
def test_linear_q8_integers_exactly(name, M, K, F):
    """Integers of at most 4 with unit scales and an integer bias: sums below 2^24, products within 5 bits."""
    announce("linear_q8 integers", name, M, K, F)
    dtype, gen = DTYPES[name], generator(M, K, F)
    x = torch.randint(-4, 5, (M, K), device=DEV, generator=gen).float()
    w = torch.randint(-4, 5, (F, K), device=DEV, generator=gen).float()
    b = torch.randint(-64, 65, (F,), device=DEV, generator=gen).float()
    ones = torch.ones(max(M, F), device=DEV)
    ref = x.double() @ w.double().t()
    q, wq = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    got = pr.linear_q8(q, ones[:M], wq, ones[:F], dtype=dtype)
    assert got.shape == (M, F) and got.dtype == dtype
    assert torch.equal(got, ref.to(dtype))
    got = pr.linear_q8(q, 2 * ones[:M], wq, 0.5 * ones[:F], b, dtype=dtype)
    assert torch.equal(got, (ref + b.double()).to(dtype))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("M,K,F", Q8_SHAPES)
def test_linear_q8_normal_operands(name, M, K, F):
    announce("linear_q8 normal", name, M, K, F)
    dtype, gen = DTYPES[name], generator(M, K, F, 1)
    (x, sx), (w, sw) = q8_rows(gen, M, K), q8_rows(gen, F, K, 0.3)
    b = rand(gen, F) * sw * 448
    got = pr.linear_q8(x, sx, w, sw, b, dtype=dtype).double()
    a, c = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
    prod = a @ c.t()
    ref, mag = prod + b.double(), a.abs() @ c.abs().t()
    half_step = torch.finfo(dtype).eps / 2
    fp32 = (K + 4) * 2.0 ** -24 * mag + 2.0 ** -22 * (prod.abs() + b.double().abs())
    cores = 0.0 if name == "fp32" else 2.0 ** -9
    assert ((got - ref).abs() <= half_step * ref.abs() * (1 + 2.0 ** -8) + fp32 + cores * mag
            + torch.finfo(dtype).tiny).all()
    if M * F >= 4096:
        rel = ((got - ref).norm() / ref.norm()).item()
        assert rel <= half_step + (2.0 ** -20 if name == "fp32" else 2.0 ** -13), rel


@pytest.mark.parametrize("M,K,F", [(7, 512, 100), (70, 1536, 64), (300, 256, 1600), (2048, 256, 5120)])
def test_linear_q8_of_large_rows_and_small_weights(M, K, F):
    """Rows near the largest value: the result is in range where the sum times a row's scale alone is not."""
    announce("linear_q8 large rows", M, K, F)
    gen = generator(M, K, F, 2)
    (x, sx), (w, sw) = q8_rows(gen, M, K, 0.1), q8_rows(gen, F, K, 0.1)
    sx, sw = sx * 2.0 ** 115, sw * 2.0 ** -20
    assert (x.float() @ w.float().t()).abs().amax() * sx.amin() > torch.finfo(torch.float32).max
    for dtype in (torch.bfloat16, torch.float32):
        got = pr.linear_q8(x, sx, w, sw, dtype=dtype)
        ref = pr.linear_q8(x, sx * 2.0 ** -115, w, sw * 2.0 ** 20, dtype=dtype)
        assert torch.equal(got, ref * 2.0 ** 95)  # powers of two: the same bits


def test_quantize_rows_of_many_rows():
    """More rows than one dimension of a grid holds."""
    announce("quantize_rows, many rows")
    x = rand(generator(11), 2 ** 21 + 5, 8, dtype=torch.bfloat16)
    q, s = ew.quantize_rows(x)
    for rows in (slice(0, 7), slice(2 ** 21 - 3, None)):
        got = ew.quantize_rows(x[rows])
        assert torch.equal(q[rows].float(), got[0].float()) and torch.equal(s[rows], got[1])
    check_q8(q, s, x.double(), x.double().abs(), "many rows")


def test_linear_q8_rows_behind_and_beside_are_left():
    """The output's surroundings keep their values at odd sizes (the C entry with a wider output)."""
    from hummingbird_amd import _lib
    announce("linear_q8 surroundings")
    for M, K, F in ((5, 64, 33), (130, 144, 131), (70, 1536, 260)):
        gen = generator(M, K, F)
        (x, sx), (w, sw) = q8_rows(gen, M, K), q8_rows(gen, F, K)
        for dtype, code in ((torch.bfloat16, 0), (torch.float32, 1), (torch.float16, 2)):
            out = torch.full((M + 3, F + 21), 77.0, device=DEV, dtype=dtype)
            st = _lib.load().hb_proj_q8(_lib.current_stream(x.device), x.data_ptr(), K, sx.data_ptr(), w.data_ptr(), K,
                                        sw.data_ptr(), 0, out.data_ptr(), code, F + 21, M, K, F)
            assert st == 0
            assert torch.equal(out[:M, :F], pr.linear_q8(x, sx, w, sw, dtype=dtype))
            assert (out[M:] == 77).all() and (out[:, F:] == 77).all()


def test_linear_q4_and_rows_leave_their_surroundings():
    """As above for the 4-bit product and the row operators (the C entries with wider outputs)."""
    from hummingbird_amd import _lib
    announce("linear_q4, rows: surroundings")
    lib = _lib.load()
    for N, K, F in ((3, 64, 33), (7, 160, 130), (17, 96, 8193)):
        gen = generator(N, K, F)
        codes, scales = pr.quantize_q4(rand(gen, F, K))
        for dtype, code in ((torch.bfloat16, 0), (torch.float32, 1), (torch.float16, 2)):
            x = rand(gen, N, K, dtype=dtype)
            out = torch.full((N + 2, F + 5), 77.0, device=DEV, dtype=dtype)
            st = lib.hb_proj_q4(_lib.current_stream(x.device), x.data_ptr(), code, K, codes.data_ptr(), K // 2,
                                scales.data_ptr(), K // 32, 0, 0, out.data_ptr(), F + 5, N, K, F)
            assert st == 0
            assert torch.equal(out[:N, :F], pr.linear_q4(x, codes, scales))
            assert (out[N:] == 77).all() and (out[:, F:] == 77).all()
    for N, C in ((5, 72), (3, 2056)):
        x = rand(generator(N, C), N, C, dtype=torch.bfloat16)
        q = torch.full((N + 1, C + 8), 1.0, device=DEV).to(torch.float8_e4m3fn)
        s = torch.full((N + 2,), 77.0, device=DEV)
        assert lib.hb_quant_rows(_lib.current_stream(x.device), x.data_ptr(), 0, C, q.data_ptr(), C + 8, s.data_ptr(), N,
                                 C) == 0
        ref = ew.quantize_rows(x)
        assert torch.equal(q[:N, :C].float(), ref[0].float()) and torch.equal(s[:N], ref[1])
        assert (q[N:].float() == 1).all() and (q[:, C:].float() == 1).all() and (s[N:] == 77).all()


def test_linear_q8_slices_and_special_values():
    """Row slices of wider tensors; a NaN or infinite row reaches its own outputs alone."""
    announce("linear_q8 slices, NaN rows")
    gen = generator(8)
    (x, sx), (w, sw) = q8_rows(gen, 40, 256), q8_rows(gen, 70, 256)
    xs, ws = x[:, 64:192], w[:, 128:]
    got = pr.linear_q8(xs, sx, ws, sw)
    assert torch.equal(got, pr.linear_q8(xs.contiguous(), sx, ws.contiguous(), sw))
    y = rand(gen, 40, 256)
    y[3, 7], y[9, 200], y[20] = float("nan"), float("inf"), 0.0
    q, s = ew.quantize_rows(y)
    out = pr.linear_q8(q, s, w, sw)
    assert torch.isnan(out[3]).all() and torch.isnan(out[9]).all() and (out[20] == 0).all()
    rest = [i for i in range(40) if i not in (3, 9)]
    assert torch.isfinite(out[rest]).all()
    assert torch.equal(out[rest], pr.linear_q8(q[rest].contiguous(), s[rest], w, sw))


def dequant_q4(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).long()
    v = torch.tensor(E2M1, dtype=torch.float64, device=DEV)[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


# rows, columns, features: every count of columns about a tile, one group, chunks' ends, one feature
Q4_SHAPES = [(1, 32, 1), (1, 256, 1536), (2, 1536, 9216), (3, 96, 17), (5, 160, 48), (6, 128, 31), (8, 544, 64),
             (9, 2048, 40), (10, 4128, 33), (11, 224, 16), (16, 6144, 100), (17, 512, 129), (20, 64, 64), (32, 1536, 65),
             (33, 1536, 65), (64, 1568, 130), (65, 96, 130), (150, 256, 70),
             (1, 96, 4113), (7, 160, 8190), (18, 64, 8209), (35, 128, 12275), (12, 192, 12305)]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("N,K,F", Q4_SHAPES)
def test_linear_q4_integers_exactly(name, N, K, F):
    """Integers of at most 8 and every code under scales of 2 to 8: sums are multiples of 1 under 2^24."""
    announce("linear_q4 integers", name, N, K, F)
    dtype, gen = DTYPES[name], generator(N, K, F)
    x = torch.randint(-8, 9, (N, K), device=DEV, generator=gen)
    codes = torch.randint(0, 256, (F, K // 2), device=DEV, generator=gen, dtype=torch.uint8)
    scales = torch.randint(128, 131, (F, K // 32), device=DEV, generator=gen, dtype=torch.uint8)
    b = torch.randint(-64, 65, (F,), device=DEV, generator=gen).float()
    x = x.to(dtype)
    ref = x.double() @ dequant_q4(codes, scales).t()
    got = pr.linear_q4(x, codes, scales)
    assert got.shape == (N, F) and got.dtype == dtype
    assert torch.equal(got, ref.to(dtype))
    assert torch.equal(pr.linear_q4(x, codes, scales, b), (ref + b.double()).to(dtype))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("N,K,F", Q4_SHAPES)
@pytest.mark.parametrize("silu", [False, True])
def test_linear_q4_normal_operands(name, N, K, F, silu):
    announce("linear_q4 normal", name, N, K, F, silu)
    dtype, gen = DTYPES[name], generator(N, K, F, 2)
    x = rand(gen, N, K, dtype=dtype)
    codes, scales = pr.quantize_q4(rand(gen, F, K, std=K ** -0.5))
    w = dequant_q4(codes, scales)
    b = rand(gen, F, std=0.1)
    got = pr.linear_q4(x, codes, scales, b, silu=silu).double()
    z = x.double() @ w.t() + b.double()
    err = (3 * K + 16) * 2.0 ** -24 * (x.double().abs() @ w.abs().t() + b.double().abs())
    ref = z * torch.sigmoid(z) if silu else z
    if silu:  # slope at most 1.1; the hardware sigmoid
        err = 1.1 * err + 2.0 ** -18 * ref.abs()
    assert ((got - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + err
            + torch.finfo(dtype).tiny).all()


@pytest.mark.parametrize("name", list(DTYPES))
def test_linear_q4_keeps_all_bits_of_x(name):
    """One weight of 1 per row picks x's elements out: they come back unchanged, from the least normal value to the
    largest, with an infinity and a NaN, which reach the outputs of their row."""
    announce("linear_q4 bits", name)
    dtype = DTYPES[name]
    K = 128
    codes = torch.zeros(K, K // 2, dtype=torch.uint8, device=DEV)
    for f in range(K):
        codes[f, f // 2] = 2 << (4 * (f % 2))  # e2m1 code 2: 1.0
    scales = torch.full((K, K // 32), 127, dtype=torch.uint8, device=DEV)
    x = rand(generator(4), 6, K)
    x[1] *= 1e3
    x[2] = torch.finfo(dtype).max * torch.sign(x[2])
    x[3] *= 1e-3
    x = x.to(dtype)
    assert torch.equal(pr.linear_q4(x, codes, scales), x)
    x[4, 3], x[5, 9] = float("inf"), float("nan")
    out = pr.linear_q4(x, codes, scales)
    assert torch.equal(out[:4], x[:4])
    assert out[4, 3] == float("inf") and torch.isnan(out[4, :3]).all()  # 0 * inf elsewhere
    assert torch.isnan(out[5]).all()


@pytest.mark.parametrize("exponent", [-100, -115, -125])
def test_linear_q4_of_small_fp32_rows(exponent):
    """fp32 rows keep their bits down to 2^-133: off by at most 2^-133 a value beyond the sum's rounding."""
    announce("linear_q4 small rows", exponent)
    gen = generator(13)
    x = rand(gen, 5, 256, std=2.0 ** exponent)
    codes, scales = pr.quantize_q4(rand(gen, 64, 256, std=2.0 ** 60))
    w = dequant_q4(codes, scales)
    got, ref = pr.linear_q4(x, codes, scales).double(), x.double() @ w.t()
    bound = (256 + 4) * 2.0 ** -24 * (x.double().abs() @ w.abs().t()) + 2.0 ** -133 * w.abs().sum(-1)
    assert ((got - ref).abs() <= bound).all()


@pytest.mark.parametrize("code", [8, 9, 64, 127, 200, 249, 250])
def test_linear_q4_scales(code):
    announce("linear_q4 scale", code)
    gen = generator(code)
    codes = torch.randint(0, 256, (20, 16), device=DEV, generator=gen, dtype=torch.uint8)
    scales = torch.full((20, 1), code, dtype=torch.uint8, device=DEV)
    x = torch.zeros(1, 32, device=DEV)
    x[0, 5] = 1.0
    w = dequant_q4(codes, scales)
    assert torch.equal(pr.linear_q4(x, codes, scales)[0].double(), w[:, 5])


def spread(t, stride):
    """`t`'s rows `stride` elements apart in memory that nothing else is written to."""
    rows, width = t.shape
    out = torch.empty((rows - 1) * stride + width, dtype=t.dtype, device=DEV).as_strided((rows, width), (stride, 1))
    out.copy_(t)
    return out


def test_offsets_past_32_bits():
    """Rows, weights and outputs that end past 2^32 bytes and elements: equal to those next to each other."""
    announce("offsets past 32 bits: rows")
    gen = generator(12)
    x = rand(gen, 4, 256, dtype=torch.bfloat16)
    far = spread(x, 3 << 29)
    for got, ref in zip(ew.quantize_rows(far), ew.quantize_rows(x)):
        assert torch.equal(got.float(), ref.float())
    announce("offsets past 32 bits: linear_q4")
    codes, scales = pr.quantize_q4(rand(gen, 600, 256))
    ref = pr.linear_q4(x, codes, scales)
    assert torch.equal(pr.linear_q4(far, spread(codes, 1 << 23), spread(scales, 1 << 23)), ref)
    del far
    announce("offsets past 32 bits: linear_q8")
    for M, F in ((1100, 700), (16, 1100), (2000, 3000)):
        (q, s), (w, sw) = q8_rows(gen, M, 144), q8_rows(gen, F, 144)
        ref = pr.linear_q8(q, s, w, sw)
        far_q = spread(q.view(torch.uint8), 1 << 22).view(torch.float8_e4m3fn)
        far_w = spread(w.view(torch.uint8), 1 << 22).view(torch.float8_e4m3fn)
        assert torch.equal(pr.linear_q8(far_q, s, far_w, sw), ref)
        del far_q, far_w
    (q, s), (w, sw) = q8_rows(gen, 70000, 64), q8_rows(gen, 32768, 64)
    out = pr.linear_q8(q, s, w, sw)
    assert torch.equal(out[69000:], pr.linear_q8(q[69000:], s[69000:].contiguous(), w, sw))


def test_refusals_of_devices_types_and_shapes():
    announce("refusals")
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    q, s = ew.quantize_rows(x)
    with pytest.raises(TypeError):
        ew.quantize_rows(x.double())
    with pytest.raises(ValueError):
        ew.quantize_rows(x[:, ::2])
    with pytest.raises(ValueError):
        ew.quantize_rows(x[:, :60])
    with pytest.raises(ValueError):
        ew.quantize_rows(x[:0])
    with pytest.raises(ValueError):
        ew.rms_modulate_q8(x[None], torch.ones(64), 1e-5)  # a weight on the host
    with pytest.raises(ValueError):
        ew.rms_modulate_q8(x[None], torch.ones(32, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        ew.residual_rms_q8(x[None], x[None, :2], torch.ones(64, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        ew.residual_rms_q8(x[None], x[None], torch.ones(64, device=DEV), 1e-5, memory=-1)
    with pytest.raises(ValueError):
        ew.glu_q8(x, torch.ones(64, device="cpu"))
    with pytest.raises(TypeError):
        pr.linear_q8(x, s, q, s)
    with pytest.raises(ValueError):
        pr.linear_q8(q, s[:3], q, s)
    with pytest.raises(ValueError):
        pr.linear_q8(q, s, q, s.cpu())
    with pytest.raises(ValueError):
        pr.linear_q8(q[:, :40], s, q[:, :40], s)
    with pytest.raises(TypeError):
        pr.linear_q8(q, s, q, s, dtype=torch.float64)
    codes, scales = pr.quantize_q4(torch.ones(8, 64, device=DEV))
    with pytest.raises(TypeError):
        pr.linear_q4(x, codes.to(torch.int8), scales)
    with pytest.raises(ValueError):
        pr.linear_q4(x, codes, scales[:, :1])
    with pytest.raises(ValueError):
        pr.linear_q4(x[:, :32], codes, scales)
    with pytest.raises(ValueError):
        pr.linear_q4(x, codes.cpu(), scales)
    with pytest.raises(ValueError):
        pr.linear_q4(x, codes, scales, torch.ones(7, device=DEV))


def test_chain_graph_and_streams():
    """A feed-forward of the operators together (norm, glu_proj, SwiGLU, proj_out): on a stream of its own and captured,
    every replay gives the eager result, with eager work between the replays."""
    announce("chain")
    gen = generator(77)
    B, L, C, F = 2, 150, 256, 512
    h, x = rand(gen, B, L, C, dtype=torch.bfloat16), rand(gen, B, L, C, dtype=torch.bfloat16)
    nw = rand(gen, C, std=0.1, mean=1.0)
    w1, s1 = ew.quantize_rows(rand(gen, 2 * F, C, std=C ** -0.5))
    w2, s2 = ew.quantize_rows(rand(gen, C, F, std=F ** -0.5))
    b1 = rand(gen, 2 * F, std=0.1)
    cond, cs = pr.quantize_q4(rand(gen, 6 * C, C, std=C ** -0.5))
    g = rand(gen, B, C, dtype=torch.bfloat16)

    def chain():
        ada = pr.linear_q4(g, cond, cs)
        scale, shift, gate = ada[:, :C], ada[:, C:2 * C], ada[:, 2 * C:3 * C]
        out, q, s = ew.residual_rms_q8(h, x, nw, 1e-5, gate=gate, scale=scale, shift=shift)
        f, fs = ew.glu_q8(pr.linear_q8(q, s, w1, s1), b1)
        return out, pr.linear_q8(f, fs, w2, s2)
    ref = [t.clone() for t in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = chain()
    torch.cuda.synchronize()
    for a, b in zip(again, ref):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = chain()
    for i in range(4):
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, ref):
            assert torch.equal(a, b), f"replay {i}"
        for a, b in zip(chain(), ref):
            assert torch.equal(a, b), f"eager after replay {i}"
    x.mul_(-1.5)  # the graph reads the inputs' present values
    new = chain()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, new):
        assert torch.equal(a, b)

"""Microscaled 4-bit rows and their product on the GPU against plain fp64 implementations.

Row operators. `quantize_rows_mx4` is exact arithmetic: codes and scale bytes are compared for equality. The others compute
y in fp32 as the 8-bit forms do, within 2^-16 of M, the value that the magnitudes of its operands give through the same
formula (tests/test_quant_gpu.py derives it). So a group's scale is the least that holds its largest magnitude, or its
neighbour where that magnitude lies within 2^-16 M of the border, and each value is within 2^-15 M of the distance that
the nearest of the codes has.

Products. Codes are multiples of 1/2 up to 6, and with scales of 1/2, 1 and 2 for each operand a product is a multiple of
2^-4 up to 144, so sums of K <= 4128 terms (and a bias of multiples of 1/4) are below 2^24 of these: every order adds them
exactly in fp32 and the result is the correctly rounded one, compared for equality, which an element read or written in the
wrong place cannot pass.
"""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew
from hummingbird_amd import projection as pr

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def generator(*key) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def rand(gen, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (mean + std * torch.randn(shape, device=DEV, generator=gen)).to(dtype)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What 4-bit rows stand for, in fp64."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*codes.shape[:-1], -1).long()
    v = VALUES.to(codes.device)[c & 7] * torch.where(c > 7, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return v * s.repeat_interleave(32, dim=-1)


def check_rows(q, s, y, mag, what):
    """4-bit rows against y (fp64) of operands' magnitude `mag` >= |y|."""
    assert q.dtype == s.dtype == torch.uint8
    assert q.shape == (*y.shape[:-1], y.shape[-1] // 2) and s.shape == (*y.shape[:-1], y.shape[-1] // 32)
    group = lambda t: t.reshape(*y.shape[:-1], -1, 32)  # noqa: E731
    step = torch.exp2(s.double() - 127)
    top, err = group(y).abs().amax(-1), 2.0 ** -16 * group(mag).amax(-1)
    assert (s >= 8).all() and (s <= 253).all()
    assert (top - err <= 6 * step).all(), f"{what}: scale too small"
    assert ((top + err > 3 * step) | (s == 8) | (top <= err)).all(), f"{what}: scale too large"
    got = values(q, s)
    near = (group(y).abs()[..., None] / step[..., None, None] - VALUES.to(y.device)).abs().amin(-1) * step[..., None]
    bad = (group(got) - group(y)).abs() > near + 2.0 ** -15 * group(mag)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("C", [32, 64, 96, 1536, 1056, 6144, 16416])
def test_quantize_rows(name, C):
    announce("quantize_rows_mx4", name, C)
    x = rand(generator(1, C), 5, 3, C, std=3.0, dtype=DTYPES[name])
    x[1, 1, 32:] = 0 if C > 32 else x[1, 1, 32:]
    q, s = ew.quantize_rows_mx4(x)
    wq, ws = pr.quantize_q4(x.reshape(15, C).float())
    assert torch.equal(q.reshape(15, -1), wq) and torch.equal(s.reshape(15, -1), ws)


@pytest.mark.parametrize("name", list(DTYPES))
def test_quantize_rows_every_border(name):
    """Every magnitude on and beside a border between codes, both signs, at scales over the type's range; the largest of a
    group on and beside the border of a scale."""
    announce("quantize_rows_mx4 borders", name)
    dtype = DTYPES[name]
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 1.5, 2, 3, 4, 0], device=DEV)
    eps = torch.finfo(dtype).eps
    near = torch.cat([base, base * (1 + eps), base * (1 - eps / 2), torch.tensor([0.1, 5.9], device=DEV)])
    near = torch.cat([near, -near])
    near = torch.nn.functional.pad(near, (0, -len(near) % 31)).reshape(-1, 31)
    tops = torch.tensor([6.0, 6 * (1 - eps / 2), 6 * (1 + eps), 3 * (1 + eps), 12 * (1 - eps / 2)], device=DEV)
    rows = torch.cat([torch.cat([near, t.expand(near.shape[0], 1)], dim=1) for t in tops])
    powers = (-13, 0, 12) if name == "fp16" else (-120, -20, 0, 20, 118)
    x = torch.cat([rows * 2.0 ** p for p in powers]).to(dtype)
    q, s = ew.quantize_rows_mx4(x)
    wq, ws = pr.quantize_q4(x.float())
    assert torch.equal(s, ws)
    assert torch.equal(q, wq)


@pytest.mark.parametrize("name", list(DTYPES))
def test_quantize_rows_special_groups(name):
    """The largest and least values, zeros of both signs, a NaN and infinities: their groups' bytes and nobody else's."""
    announce("quantize_rows_mx4 special", name)
    dtype = DTYPES[name]
    x = rand(generator(2), 6, 96, dtype=dtype)
    plain = ew.quantize_rows_mx4(x)
    y = x.clone()
    y[0, 32:64] = torch.finfo(dtype).max
    y[1, 32:64] = torch.finfo(dtype).smallest_normal
    y[2, 32:64] = -0.0
    y[3, 40] = float("nan")
    y[4, 63] = float("-inf")
    y[5, 32] = float("inf")
    q, s = ew.quantize_rows_mx4(y)
    assert torch.equal(q[:, :16], plain[0][:, :16]) and torch.equal(q[:, 32:], plain[0][:, 32:])
    assert torch.equal(s[:, 0], plain[1][:, 0]) and torch.equal(s[:, 2], plain[1][:, 2])
    assert (s[3:, 1] == 255).all() and int(s[2, 1]) == 127
    got = values(q, s)
    top = torch.finfo(dtype).max
    assert ((got[0, 32:64] - top).abs() <= top / 6 + 2.0 ** 104).all()  # half the step of 2 at 4 to 6, of 5 at least
    assert (got[1, 32:64] - torch.finfo(dtype).smallest_normal).abs().max() <= max(
        2.0 ** -121, torch.finfo(dtype).smallest_normal / 4)  # half a step at the least scale, or of 1 to 2's 4 codes
    assert (got[2, 32:64] == 0).all() and torch.isnan(got[3:, 32:64]).all()


def test_quantize_rows_strided():
    announce("quantize_rows_mx4 strides")
    wide = rand(generator(3), 4, 6, 256, dtype=torch.bfloat16)
    for x in (wide[..., 64:192], wide[:, 2], wide[:1], wide[:, :, 8:40]):
        q, s = ew.quantize_rows_mx4(x)
        wq, ws = ew.quantize_rows_mx4(x.contiguous())
        assert torch.equal(q, wq) and torch.equal(s, ws)


OPTIONS = [dict(), dict(gate=True), dict(mod=True), dict(gate=True, bias=True, mod=True), dict(local=True, mod=True),
           dict(gate=True, bias=True, local=True, mod=True)]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("C", [32, 1536, 1056, 4128, 16384])
@pytest.mark.parametrize("opt", range(len(OPTIONS)))
def test_residual_rms(name, C, opt):
    announce("residual_rms_mx4", name, C, OPTIONS[opt])
    o, dtype, B, L = OPTIONS[opt], DTYPES[name], 2, 3
    gen = generator(4, C, opt)
    h, x = rand(gen, B, L, C, dtype=dtype), rand(gen, B, L, C, dtype=dtype)
    w = rand(gen, C, std=0.1, mean=1.0)
    gate = rand(gen, B, C, dtype=dtype) if o.get("gate") else None
    xb = rand(gen, C, std=0.1, dtype=dtype) if o.get("bias") else None
    local = rand(gen, C, std=0.1, dtype=dtype) if o.get("local") else None
    scale, shift = (rand(gen, B, C, std=0.2, dtype=dtype), rand(gen, B, C, std=0.2, dtype=dtype)) if o.get("mod") else (
        None, None)
    oh, q, s = ew.residual_rms_mx4(h, x, w, 1e-5, gate=gate, x_bias=xb, local=local, memory=1, scale=scale, shift=shift)
    v, m = x.double(), x.double().abs()
    if xb is not None:
        v, m = v + xb.double(), m + xb.double().abs()
    if gate is not None:
        g = torch.sigmoid(1 - gate.double())[:, None]
        v, m = v * g, m * g
    v, m = h.double() + v, h.double().abs() + m
    if local is not None:
        v, m = v.clone(), m.clone()
        v[:, 1:] += local.double()
        m[:, 1:] += local.double().abs()
    half = torch.finfo(dtype).eps / 2
    assert ((oh.double() - v).abs() <= half * v.abs() + 2.0 ** -18 * m + 2.0 ** -24 * (dtype == torch.float16)).all()
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5)
    y, m = v * r * w.double(), m * r * w.double().abs()
    if scale is not None:
        y = y * (1 + scale.double())[:, None] + shift.double()[:, None]
        m = m * (1 + scale.double().abs())[:, None] + shift.double().abs()[:, None]
    check_rows(q, s, y, m, "residual_rms_mx4")
    if not any(o.get(k) for k in ("gate", "bias", "local")):
        q2, s2 = ew.rms_modulate_mx4(h, w, 1e-5, scale, shift)
        y = h.double() * torch.rsqrt((h.double() ** 2).mean(-1, keepdim=True) + 1e-5) * w.double()
        m = y.abs()
        if scale is not None:
            y = y * (1 + scale.double())[:, None] + shift.double()[:, None]
            m = m * (1 + scale.double().abs())[:, None] + shift.double().abs()[:, None]
        check_rows(q2, s2, y, m, "rms_modulate_mx4")


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("F", [32, 96, 4096, 6144, 16416])
@pytest.mark.parametrize("biased", [False, True])
def test_glu(name, F, biased):
    announce("glu_mx4", name, F, biased)
    gen = generator(5, F)
    p = rand(gen, 7, 2 * F, std=2.0, dtype=DTYPES[name])
    b = rand(gen, 2 * F, std=0.5) if biased else None
    q, s = ew.glu_mx4(p, b)
    p64, m = p.double(), p.double().abs()
    if biased:
        p64, m = p64 + b.double(), m + b.double().abs()
    v, g = p64.chunk(2, dim=-1)
    mv, mg = m.chunk(2, dim=-1)
    check_rows(q, s, v * g * torch.sigmoid(g), mv * mg * torch.sigmoid(g), "glu_mx4")


def codes(gen, rows, k, low=126, high=128):
    """Random 4-bit rows: all codes, scale bytes of [low, high]."""
    return (torch.randint(0, 256, (rows, k // 2), generator=gen, device=DEV, dtype=torch.uint8),
            torch.randint(low, high + 1, (rows, k // 32), generator=gen, device=DEV, dtype=torch.uint8))


def check_exact(x, xs, w, ws, bias, dtype, out):
    ref = values(x, xs) @ values(w, ws).t().contiguous()
    if bias is not None:
        ref = ref + bias.double()
    assert out.dtype == dtype and out.shape == ref.shape
    bad = out != ref.to(dtype)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}"


# rows, columns, features: few rows; one tile; tiles of each size, whole and partly empty; K inside a stage, over its end
SHAPES = [(1, 32, 1), (7, 1536, 7680), (16, 96, 17), (17, 64, 15), (31, 1056, 513), (33, 256, 64), (64, 512, 64),
          (65, 288, 65), (100, 2048, 129), (129, 1536, 257), (257, 1024, 1001), (700, 1536, 1536), (700, 1056, 1537),
          (1422, 1536, 1536), (1300, 512, 4096), (2584, 800, 1536), (2049, 1536, 7680), (1025, 1504, 12288),
          (3900, 4096, 3300), (3841, 4128, 3329), (24, 4096, 1000), (300, 2048, 1000), (4000, 1536, 8190),
          (4001, 1568, 8190), (2900, 4096, 3000),
          (90, 4128, 200), (1400, 544, 1500)]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_product(name, M, K, F):
    announce("linear_mx4", name, M, K, F)
    gen = generator(6, M, K, F)
    x, xs = codes(gen, M, K)
    w, ws = codes(gen, F, K)
    bias = torch.randint(-64, 65, (F,), generator=gen, device=DEV).float() / 4 if (M + F) % 2 else None
    out = pr.linear_mx4(x, xs, w, ws, bias, dtype=DTYPES[name])
    check_exact(x, xs, w, ws, bias, DTYPES[name], out)


def test_product_beyond_the_caches():
    """An output of more than 128 MB, whose stores take another way."""
    announce("linear_mx4 large output")
    for K in (256, 288):
        gen = generator(7, K)
        x, xs = codes(gen, 5601, K)
        w, ws = codes(gen, 12288, K)
        check_exact(x, xs, w, ws, None, torch.bfloat16, pr.linear_mx4(x, xs, w, ws))


@pytest.mark.parametrize("M", [5, 40, 300])
def test_product_strides(M):
    """Rows of wider tensors, scales at every alignment, a batch of rows, a strided bias."""
    announce("linear_mx4 strides", M)
    gen = generator(8, M)
    K, F = 1536, 200
    wide, wides = codes(gen, M, 2048)
    w, ws = codes(gen, F, 2048)
    for at in (0, 1, 2, 3, 5):
        x, xs = wide[:, 16 * at:16 * at + K // 2], wides[:, at:at + K // 32]
        y, ys = w[:, 16 * at:16 * at + K // 2], ws[:, at:at + K // 32]
        check_exact(x, xs, y, ys, None, torch.float32, pr.linear_mx4(x, xs, y, ys, dtype=torch.float32))
        check_exact(x.contiguous(), xs.contiguous(), y, ys, None, torch.bfloat16,
                    pr.linear_mx4(x.contiguous(), xs.contiguous(), y, ys))
    batch, scales = wide[:, :K // 2].reshape(M, 1, K // 2).expand(M, 1, K // 2), wides[:, :K // 32].reshape(M, 1, K // 32)
    out = pr.linear_mx4(batch, scales, w[:, :K // 2], ws[:, :K // 32])
    assert out.shape == (M, 1, F)
    check_exact(wide[:, :K // 2], wides[:, :K // 32], w[:, :K // 2], ws[:, :K // 32], None, torch.bfloat16, out[:, 0])


@pytest.mark.parametrize("M", [3, 70])
def test_product_of_every_scale(M):
    """One group per operand with every scale byte in turn: with 2^e the scales' product, sums (up to 192 2^e) are exact
    while they are normal numbers, not finite where every product is beyond the range, tiny where they are below it, and
    NaN under the byte 255."""
    announce("linear_mx4 scales", M)
    gen = generator(9, M)
    x = torch.full((M, 16), 0x22, dtype=torch.uint8, device=DEV)  # ones
    w, _ = codes(gen, 256, 32)
    ws = torch.arange(256, device=DEV, dtype=torch.int32).to(torch.uint8)[:, None].contiguous()
    for sx in (0, 1, 60, 127, 200, 253, 254):
        xs = torch.full((M, 1), sx, dtype=torch.uint8, device=DEV)
        out = pr.linear_mx4(x, xs, w, ws, dtype=torch.float32).double()
        assert torch.isnan(out[:, 255]).all()
        ref = values(x, xs) @ values(w, ws).t().contiguous()
        e = torch.arange(255, device=DEV) + sx - 254
        normal, low, high = (e >= -120) & (e <= 119), e < -120, e >= 130
        out, ref = out[:, :255], ref[:, :255]
        assert torch.equal(out[:, normal], ref[:, normal])
        assert ((out - ref)[:, low].abs() <= 2.0 ** -112).all()
        assert not torch.isfinite(out[:, high][ref[:, high] != 0]).any()
    xs = torch.full((M, 1), 127, dtype=torch.uint8, device=DEV)
    xs[1] = 255
    ws = torch.full_like(ws, 127)
    out = pr.linear_mx4(x, xs, w, ws, dtype=torch.float32)
    assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any() and not torch.isnan(out[2]).any()


@pytest.mark.parametrize("M", [9, 200])
def test_product_sums_are_fp32(M):
    """Normal rows of ordinary layers, fp32 outputs: n additions of relative error 2^-24."""
    announce("linear_mx4 sums", M)
    gen = generator(10, M)
    K, F = 6144, 300
    x, xs = ew.quantize_rows_mx4(rand(gen, M, K))
    w, ws = pr.quantize_q4(rand(gen, F, K, std=K ** -0.5))
    out = pr.linear_mx4(x, xs, w, ws, dtype=torch.float32).double()
    a, b = values(x, xs), values(w, ws)
    err, mag = (out - a @ b.t().contiguous()).abs(), a.abs() @ b.abs().t().contiguous()
    assert (err <= K * 2.0 ** -24 * mag).all()
    assert float((err / mag).mean()) < 2.0 ** -21


@pytest.mark.parametrize("M", [4, 64, 300])
def test_product_sums_across_scales(M):
    """Groups of very different scales: nothing of the small ones is cut off before the sum is rounded. A large and a small
    product in two groups give their sum exactly while it has 24 bits; random rows, whose groups' own sums are exact, are
    within a rounding per group."""
    announce("linear_mx4 sums across scales", M)
    gen = generator(15, M)
    for big, low in ((0, 4), (0, 1), (0, 2), (1, 5), (4, 0), (7, 3)):
        for d in range(19):
            x, xs = torch.zeros(M, 128, dtype=torch.uint8, device=DEV), torch.full((M, 8), 127, dtype=torch.uint8, device=DEV)
            w, ws = torch.zeros(64, 128, dtype=torch.uint8, device=DEV), torch.full((64, 8), 127, dtype=torch.uint8, device=DEV)
            x[:, 16 * big], w[:, 16 * big], x[:, 16 * low], w[:, 16 * low], xs[:, low] = 7, 7, 2, 2, 127 - d
            assert (pr.linear_mx4(x, xs, w, ws, dtype=torch.float32) == 36 + 2.0 ** -d).all(), (big, low, d)
    K = 256
    for spread in (0, 5, 10, 16, 30):
        x, xs = codes(gen, M, K, 127 - spread, 127)
        w, ws = codes(gen, 64, K, 127 - spread, 127)
        out = pr.linear_mx4(x, xs, w, ws, dtype=torch.float32).double()
        a, b = values(x, xs), values(w, ws)
        err, mag = (out - a @ b.t().contiguous()).abs(), a.abs() @ b.abs().t().contiguous()
        assert (err <= (K // 32 + 1) * 2.0 ** -24 * mag).all(), spread


def test_captured_and_on_another_stream():
    """Two graphs of one layer, replayed in turn with eager calls between, and a call on a stream of its own."""
    announce("mx4 graphs")
    gen = generator(11)
    w, ws = pr.quantize_q4(rand(gen, 512, 1536))
    xs = [rand(gen, n, 1536, dtype=torch.bfloat16) for n in (9, 400)]
    layer = lambda x: pr.linear_mx4(*ew.quantize_rows_mx4(x), w, ws)  # noqa: E731
    want = [layer(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(xs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[1])
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(x)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), x, ref in zip(graphs, xs, want):
            out.zero_()
            g.replay()
            assert torch.equal(layer(x), ref)
            torch.cuda.synchronize()
            assert torch.equal(out, ref)


def test_rows_past_32_bits():
    """Rows of an input, codes and an output whose places pass 2^32 bytes, the last of them checked."""
    announce("mx4 past 32 bits")
    gen = generator(12)
    C, N = 8192, 270000
    x = torch.empty(N, C, dtype=torch.bfloat16, device=DEV)
    last = rand(gen, 50, C, dtype=torch.bfloat16)
    x[-50:] = last
    x[:50] = last
    q, s = ew.quantize_rows_mx4(x)
    wq, ws = ew.quantize_rows_mx4(last)
    for part in (slice(0, 50), slice(N - 50, N)):
        assert torch.equal(q[part], wq) and torch.equal(s[part], ws)
    weight, bias = rand(gen, C, std=0.1, mean=1.0), rand(gen, C, std=0.1)
    q, s = ew.rms_modulate_mx4(x[None], weight, 1e-5)
    wq, ws = ew.rms_modulate_mx4(last[None], weight, 1e-5)
    assert torch.equal(q[0, -50:], wq[0]) and torch.equal(s[0, -50:], ws[0])
    h, q, s = ew.residual_rms_mx4(x[None], x[None], weight, 1e-5)
    wh, wq, ws = ew.residual_rms_mx4(last[None], last[None], weight, 1e-5)
    assert torch.equal(h[0, -50:], wh[0]) and torch.equal(q[0, -50:], wq[0]) and torch.equal(s[0, -50:], ws[0])
    del h
    q, s = ew.glu_mx4(x, bias)
    wq, ws = ew.glu_mx4(last, bias)
    assert torch.equal(q[-50:], wq) and torch.equal(s[-50:], ws)
    del x
    M, F, K = 140001, 16000, 64
    x, xs = codes(gen, M, K)
    w, ws = codes(gen, F, K)
    out = pr.linear_mx4(x, xs, w, ws)
    for part in (slice(0, 300), slice(M - 300, M)):
        check_exact(x[part], xs[part], w, ws, None, torch.bfloat16, out[part])
    del out
    for rows in (7, 40, 300):  # rows 4 MB apart
        far, fars = codes(gen, rows, K)
        buf = torch.empty(rows * (1 << 22) + 64, dtype=torch.uint8, device=DEV)
        y = buf.as_strided((rows, K // 2), (1 << 22, 1))
        y.copy_(far)
        check_exact(far, fars, w, ws, None, torch.bfloat16, pr.linear_mx4(y, fars, w, ws))
        check_exact(w, ws, far, fars, None, torch.bfloat16, pr.linear_mx4(w, ws, y, fars))
        fs = buf.as_strided((rows, K // 32), (1 << 22, 1), 33)
        fs.copy_(fars)
        check_exact(far, fars, w, ws, None, torch.bfloat16, pr.linear_mx4(far, fs, w, ws))
        check_exact(w, ws, far, fars, None, torch.bfloat16, pr.linear_mx4(w, ws, far, fs))


def test_wrapper_refusals():
    announce("mx4 refusals")
    gen = generator(13)
    x, w = rand(gen, 2, 5, 64, dtype=torch.bfloat16), rand(gen, 64)
    mod = rand(gen, 2, 64, dtype=torch.bfloat16)
    refused = [(ew.quantize_rows_mx4, (x[..., :40],)), (ew.quantize_rows_mx4, (x[..., :0],)),
               (ew.quantize_rows_mx4, (x.int(),)), (ew.quantize_rows_mx4, (x[..., ::2],)),
               (ew.quantize_rows_mx4, (x.transpose(0, 1),)), (ew.glu_mx4, (x[..., :32],)), (ew.glu_mx4, (x[..., :63],)),
               (ew.glu_mx4, (x, w[:32])), (ew.glu_mx4, (x, w.cpu())), (ew.rms_modulate_mx4, (x[0], w, 1e-5)),
               (ew.rms_modulate_mx4, (x, w[:32], 1e-5)), (ew.rms_modulate_mx4, (x, w, -1.0)),
               (ew.rms_modulate_mx4, (x, w, 1e-5, mod)), (ew.rms_modulate_mx4, (x, w, 1e-5, mod, mod.float())),
               (ew.rms_modulate_mx4, (x, w, 1e-5, mod[:1], mod[:1])), (ew.rms_modulate_mx4, (x, w.cpu(), 1e-5)),
               (ew.rms_modulate_mx4, (rand(gen, 1, 2, 16416), rand(gen, 16416), 1e-5)),
               (ew.residual_rms_mx4, (x, x[:1], w, 1e-5)), (ew.residual_rms_mx4, (x, x.float(), w, 1e-5)),
               (ew.residual_rms_mx4, (x, x.cpu(), w, 1e-5)), (ew.residual_rms_mx4, (x, x, w[:32], 1e-5))]
    q, s = ew.quantize_rows_mx4(x)
    a, b = codes(gen, 24, 64)
    refused += [(pr.linear_mx4, args) for args in (
        (q.int(), s, a, b), (q, s.int(), a, b), (q, s, a.char(), b), (q, s, a, b.float()), (q, s, a[:, :16], b),
        (q[..., :16], s, a, b), (q[..., :24], s, a[:, :24], b), (q, s[..., :1], a, b), (q, s[:1], a, b),
        (q, s, a, b[:, :1]), (q, s, a, b[:20]), (q, s, a.cpu(), b), (q, s.cpu(), a, b), (q.cpu(), s.cpu(), a.cpu(), b.cpu()),
        (q, s, a, b, w), (q, s, a, b, w[:24].cpu()), (q, s, a, b, None, torch.int8), (q, s, a, b, None, torch.float64),
        (q, s, a[None], b[None]), (q, s, a.t().contiguous().t(), b))]
    for i, (call, args) in enumerate(refused):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call(*args)
            pytest.fail(f"call {i} ({call.__name__}) was taken")


def test_no_rows_and_one():
    """Empty batches are refused, as by the 8-bit forms; one row of one group is a row."""
    announce("mx4 no rows")
    x = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16)
    for call in (ew.quantize_rows, ew.quantize_rows_mx4, ew.glu_mx4):
        with pytest.raises(ValueError):
            call(x)
    u = torch.zeros(0, 32, device=DEV, dtype=torch.uint8)
    a, b = codes(generator(14), 24, 64)
    with pytest.raises(ValueError):
        pr.linear_mx4(u, u[:, :2], a, b)
    q, s = ew.quantize_rows_mx4(torch.full((1, 32), 6.0, device=DEV))
    check_exact(q, s, q, s, None, torch.float32, pr.linear_mx4(q, s, q, s, dtype=torch.float32))

"""The denoiser on microscaled 4-bit rows and weights (`dit_forward(projections="mx4")`) on the GPU.

* The layers' order and operands: with every 4-bit operator replaced by its value before any rounding to 4 bits, under the
  fp32 preset, the path is the unquantised denoiser up to fp32 rounding: 2e-5 of the output's largest magnitude, as the
  unquantised one against its oracle.
* Each operator on the operands that the path gives it, against plain fp64 operations: a norm's and a GLU's rows as
  tests/test_mx4_gpu.py checks them; a product's sum of K terms within K 2^-24 of the magnitudes' product and one rounding.
* Against the unquantised denoiser: a rounding to e2m1 is off by at most 1/4 of the value (above the scale's 1), 1/4 /
  sqrt(3) = 14 % on average, on both operands of a product, 20 % of its result, and a branch holds up to three products in
  a row, 35 %. The branches' errors are independent and smaller than the residual stream they are added to: half of the
  output's norm is allowed, and the error must not vanish.
* The sampler's graph against the eager loop, replayed with other work in between: equal bits.
"""
from __future__ import annotations

import dataclasses

import pytest
import torch

from hummingbird_amd import dit, elementwise, projection, sampling
from hummingbird_amd.dtypes import BF16, FP16, FP32_PARITY
from tests.test_mx4_gpu import check_rows, values
from tests.test_quant_denoiser_gpu import SMALL, rel
from tests.test_sampler_gpu import MEDIUM2, case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def announce(name: str) -> None:
    print(f"\n[case] {name}", flush=True)


def norm64(v, weight, eps, scale, shift, mag=None):
    """The modulated norm of v and the same formula on magnitudes (of v's own, or `mag`), in fp64."""
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * weight.double()
    y, m = v * r, (v.abs() if mag is None else mag) * r.abs()
    if scale is not None:
        s, b = scale.double()[:, None], shift.double()[:, None]
        y, m = y * (1 + s) + b, m * (1 + s.abs()) + b.abs()
    return y, m


def residual64(h, x, gate, x_bias, local, memory):
    """The gated residual and the same formula on magnitudes, in fp64."""
    v, m = x.double(), x.double().abs()
    if x_bias is not None:
        v, m = v + x_bias.double(), m + x_bias.double().abs()
    if gate is not None:
        g = torch.sigmoid(1 - gate.double())[:, None]
        v, m = v * g, m * g
    v, m = h.double() + v, h.double().abs() + m
    if local is not None:
        v = torch.cat([v[:, :memory], v[:, memory:] + local.double()], dim=1)
        m = torch.cat([m[:, :memory], m[:, memory:] + local.double().abs()], dim=1)
    return v, m


def glu64(proj, bias):
    p = proj.double() if bias is None else proj.double() + bias.double()
    value, gate = p.chunk(2, dim=-1)
    return value * gate * torch.sigmoid(gate)


def small(tokens, batch):
    params, cond, mask, x = case(SMALL, FP32_PARITY, batch, tokens)
    params = dit.quantize_params(params, conditioning="keep", weights="mx4")
    static = dit.prepare_static(params, cond, mask, SMALL, FP32_PARITY)
    return params, static, x, torch.linspace(0.9, 0.3, batch, device=DEV)


@pytest.mark.parametrize("batch,tokens", [(2, 45), (1, 7)])
def test_the_path_without_roundings_is_the_unquantised_one(monkeypatch, batch, tokens):
    announce(f"dit_forward mx4 without roundings B={batch} T={tokens}")
    params, static, x, t = small(tokens, batch)
    want = dit.dit_forward(params, x, t, static, SMALL, FP32_PARITY)
    weights = {}
    for b in static["blocks"]:
        for part in ("self_attn", "cross_attn", "ff"):
            for layer in b[part].values():
                if "mx4" in layer:
                    weights[layer["mx4"][0].data_ptr()] = layer["weight"]

    def norm(x, w, eps, scale=None, shift=None):
        return norm64(x.double(), w, eps, scale, shift)[0].float(), None

    def residual(h, x, w, eps, gate=None, x_bias=None, local=None, memory=0, scale=None, shift=None):
        v, _ = residual64(h, x, gate, x_bias, local, memory)
        return v.to(h.dtype), norm64(v, w, eps, scale, shift)[0].float(), None

    monkeypatch.setattr(elementwise, "quantize_rows_mx4", lambda x: (x, None))
    monkeypatch.setattr(elementwise, "rms_modulate_mx4", norm)
    monkeypatch.setattr(elementwise, "residual_rms_mx4", residual)
    monkeypatch.setattr(elementwise, "glu_mx4", lambda p, b=None: (glu64(p, b).float(), None))
    monkeypatch.setattr(projection, "linear_mx4", lambda x, s, w, ws, bias=None, dtype=None: (
        x.double() @ weights[w.data_ptr()].double().t().contiguous()).to(dtype))
    got = dit.dit_forward(params, x, t, static, SMALL, FP32_PARITY, projections="mx4")
    assert (got - want).abs().max() <= 2e-5 * want.abs().max()


@pytest.mark.parametrize("batch,tokens", [(2, 45), (1, 7)])
def test_each_operator_of_the_path(monkeypatch, batch, tokens):
    announce(f"dit_forward mx4 operators B={batch} T={tokens}")
    params, static, x, t = small(tokens, batch)
    calls = {n: 0 for n in ("quantize_rows_mx4", "rms_modulate_mx4", "residual_rms_mx4", "glu_mx4", "linear_mx4")}
    kernels = {n: getattr(projection if n == "linear_mx4" else elementwise, n) for n in calls}

    def quantize(x):
        calls["quantize_rows_mx4"] += 1
        q, s = kernels["quantize_rows_mx4"](x)
        wq, ws = projection.quantize_q4(x.reshape(-1, x.shape[-1]).float())
        assert torch.equal(q.reshape(wq.shape), wq) and torch.equal(s.reshape(ws.shape), ws)
        return q, s

    def norm(x, w, eps, scale=None, shift=None):
        calls["rms_modulate_mx4"] += 1
        q, s = kernels["rms_modulate_mx4"](x, w, eps, scale, shift)
        check_rows(q, s, *norm64(x.double(), w, eps, scale, shift), "rms_modulate_mx4")
        return q, s

    def residual(h, x, w, eps, gate=None, x_bias=None, local=None, memory=0, scale=None, shift=None):
        calls["residual_rms_mx4"] += 1
        oh, q, s = kernels["residual_rms_mx4"](h, x, w, eps, gate=gate, x_bias=x_bias, local=local, memory=memory,
                                               scale=scale, shift=shift)
        v, m = residual64(h, x, gate, x_bias, local, memory)
        assert ((oh.double() - v).abs() <= 2.0 ** -24 * v.abs() + 2.0 ** -18 * m).all()
        check_rows(q, s, *norm64(v, w, eps, scale, shift, m), "residual_rms_mx4")
        return oh, q, s

    def glu(p, bias=None):
        calls["glu_mx4"] += 1
        q, s = kernels["glu_mx4"](p, bias)
        m = p.double().abs() if bias is None else p.double().abs() + bias.double().abs()
        mv, mg = m.chunk(2, dim=-1)
        gate = (p.double() if bias is None else p.double() + bias.double()).chunk(2, dim=-1)[1]
        check_rows(q, s, glu64(p, bias), mv * mg * torch.sigmoid(gate), "glu_mx4")
        return q, s

    def linear(x, s, w, ws, bias=None, dtype=torch.bfloat16):
        calls["linear_mx4"] += 1
        out = kernels["linear_mx4"](x, s, w, ws, bias, dtype=dtype)
        a, b = values(x, s), values(w, ws).t().contiguous()
        tol = a.shape[-1] * 2.0 ** -24 * (a.abs() @ b.abs()) + torch.finfo(dtype).eps / 2 * (a @ b).abs()
        assert ((out.double() - a @ b).abs() <= tol).all()
        return out

    for name, f in zip(calls, (quantize, norm, residual, glu, linear)):
        monkeypatch.setattr(projection if name == "linear_mx4" else elementwise, name, f)
    got = dit.dit_forward(params, x, t, static, SMALL, FP32_PARITY, projections="mx4")
    assert torch.isfinite(got).all()
    # two blocks: six products each; the first norm, three residuals less the last; two attention outputs; one GLU
    assert calls == dict(quantize_rows_mx4=4, rms_modulate_mx4=1, residual_rms_mx4=5, glu_mx4=2, linear_mx4=12)


@pytest.mark.parametrize("preset", ["bf16", "fp16"])
def test_dit_forward_mx4_is_near_the_unquantised_one(preset):
    announce(f"dit_forward medium mx4 vs {preset}")
    dtype = {"bf16": BF16, "fp16": FP16}[preset]
    params, cond, mask, x = case(MEDIUM2, dtype, 2, 300, seed=24, ctx_tokens=257)
    params = dit.quantize_params(params, weights="mx4")
    static = dit.prepare_static(params, cond, mask, MEDIUM2, dtype)
    t = torch.tensor([0.9, 0.35], device=DEV)
    got = dit.dit_forward(params, x, t, static, MEDIUM2, dtype, projections="mx4")
    off = rel(got, dit.dit_forward(params, x, t, static, MEDIUM2, dtype))
    print(f"off by {off:.3f} of the output's norm")
    assert 1e-3 < off <= 0.5


def test_sampler_mx4_graph_replays_equal_the_eager_loop():
    announce("PingpongGraph vs eager pingpong (mx4)")
    params, cond, mask, x = case(MEDIUM2, BF16, 1, 200, seed=25, ctx_tokens=257)
    params = dit.quantize_params(params, weights="mx4")
    static = dit.prepare_static(params, cond, mask, MEDIUM2, BF16)
    gen = torch.Generator().manual_seed(26)
    noise = torch.randn((3, 1, MEDIUM2.io_channels, 200), generator=gen).to(DEV)
    graph = sampling.PingpongGraph(params, static, MEDIUM2, BF16, x, noise, projections="mx4")
    schedule = sampling.build_schedule(3, device=DEV)
    for rep in range(3):
        x_r = torch.randn(x.shape, generator=gen).to(DEV)
        n_r = torch.randn(noise.shape, generator=gen).to(DEV)
        got = graph(x_r, n_r).clone()
        torch.cuda.synchronize()
        ref, _ = sampling.pingpong(params, x_r, schedule, n_r, static, MEDIUM2, BF16, trajectory=False, projections="mx4")
        torch.cuda.synchronize()
        assert torch.equal(got, ref), f"replay {rep}"
        _ = (torch.randn(1000, device=DEV) * 2).sum().item()  # unrelated eager work between replays


def test_refusals():
    announce("mx4 refusals")
    params, cond, mask, x = case(SMALL, BF16, 1, 20)
    t = torch.tensor([0.5], device=DEV)
    q8 = dit.quantize_params(params)
    static = dit.prepare_static(q8, cond, mask, SMALL, BF16)
    with pytest.raises(ValueError, match="quantize_params"):  # 8-bit weights
        dit.dit_forward(q8, x, t, static, SMALL, BF16, projections="mx4")
    both = dit.quantize_params(q8, weights="mx4")
    with pytest.raises(ValueError, match="prepare_static"):
        dit.dit_forward(both, x, t, static, SMALL, BF16, projections="mx4")
    with pytest.raises(ValueError, match="weights"):
        dit.quantize_params(params, weights="q4")
    plain = dataclasses.replace(SMALL, differential=False)
    few = dit.quantize_params(dit.init_params(plain, BF16, device=DEV), weights="mx4")
    with pytest.raises(ValueError, match="differential"):
        dit.dit_forward(few, x, t, dit.prepare_static(few, cond, mask, plain, BF16), plain, BF16, projections="mx4")
    # parameters with both forms serve every path as before
    static = dit.prepare_static(both, cond, mask, SMALL, BF16)
    for form, of in (("torch", params), ("q8", q8)):
        a = dit.dit_forward(both, x, t, static, SMALL, BF16, projections=form)
        b = dit.dit_forward(of, x, t, dit.prepare_static(of, cond, mask, SMALL, BF16), SMALL, BF16, projections=form)
        assert torch.equal(a, b)

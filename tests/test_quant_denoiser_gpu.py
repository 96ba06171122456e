"""The denoiser on 8-bit rows and 8- and 4-bit weights (`dit_forward(projections="q8")`) on the GPU.

* Against the same path with every quantised operator replaced by plain fp32 torch operations, under the fp32 preset.
  The two differ by fp32 rounding, about 1e-6 of a value, and where that moves a value over a border between two 8-bit
  codes, by one step. A border is within 1e-6 of a fraction 1e-6 / 2^-4 of the values, and a step is at most 2^-3 of the
  value, so a quantised tensor differs by about sqrt(1.6e-5) 2^-3 = 5e-4 of its norm; 12 of them follow each other in two
  blocks: 1e-2 is allowed.
* Against the unquantised denoiser, bf16 and half: a rounding to e4m3 is off by at most 2^-4, 2^-4 / sqrt(3) = 3.6 % on average,
  on both operands of a product, 5 % of its result, and a branch holds up to three products in a row, 9 %. The branches'
  errors are independent and smaller than the residual stream they are added to: 25 % of the output's norm is allowed,
  and the error must not vanish.
* The sampler's graph against the eager loop, replayed with other work in between: equal bits.
"""
from __future__ import annotations

import dataclasses

import pytest
import torch

from hummingbird_amd import dit, elementwise, projection, sampling
from hummingbird_amd.config import MEDIUM_DIT
from hummingbird_amd.dtypes import BF16, FP16, FP32_PARITY
from tests.test_sampler import TINY
from tests.test_sampler_gpu import MEDIUM2, case

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = dataclasses.replace(TINY, attention="hip", fourier_dim=32)


def announce(name: str) -> None:
    print(f"\n[case] {name}", flush=True)


def plain_rows(y):
    s = (y.float().abs().amax(-1) / 448).clamp_min(2.0 ** -100)
    return (y.float() / s[..., None]).to(torch.float8_e4m3fn), s


def plain_norm(v, weight, eps, scale, shift):
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * weight.float()
    if scale is not None:
        y = y * (1 + scale.float()[:, None]) + shift.float()[:, None]
    return plain_rows(y)


def plain_residual(h, x, weight, eps, gate=None, x_bias=None, local=None, memory=0, scale=None, shift=None):
    v = x.float()
    if x_bias is not None:
        v = v + x_bias.float()
    if gate is not None:
        v = v * torch.sigmoid(1 - gate.float())[:, None]
    v = h.float() + v
    if local is not None:
        v = torch.cat([v[:, :memory], v[:, memory:] + local.float()], dim=1)
    return (v.to(h.dtype), *plain_norm(v, weight, eps, scale, shift))


def plain_glu(proj, bias=None):
    value, gate = (proj.float() + bias.float()).chunk(2, dim=-1)
    return plain_rows(value * gate * torch.sigmoid(gate))


def plain_linear_q8(x, x_scale, weight, weight_scale, bias=None, dtype=torch.bfloat16):
    assert bias is None
    return ((x.float() @ weight.float().t()) * x_scale[..., None] * weight_scale).to(dtype)


def plain_linear_q4(x, weight, weight_scale, bias=None, silu=False):
    code = torch.stack([weight & 15, weight >> 4], dim=-1).reshape(weight.shape[0], -1).long()
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)[code & 7]
    w = level * torch.where(code >= 8, -1.0, 1.0) * torch.exp2(weight_scale.float() - 127).repeat_interleave(32, dim=1)
    y = x.float() @ w.t() + bias.float()
    return (y * torch.sigmoid(y) if silu else y).to(x.dtype)


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("batch,tokens", [(2, 45), (1, 7)])
def test_dit_forward_q8_vs_plain_operations(monkeypatch, batch, tokens):
    announce(f"dit_forward q8 vs plain operations B={batch} T={tokens}")
    params, cond, mask, x = case(SMALL, FP32_PARITY, batch, tokens)
    params = dit.quantize_params(params)
    static = dit.prepare_static(params, cond, mask, SMALL, FP32_PARITY)
    t = torch.linspace(0.9, 0.3, batch, device=DEV)
    got = dit.dit_forward(params, x, t, static, SMALL, FP32_PARITY, projections="q8")
    monkeypatch.setattr(elementwise, "quantize_rows", plain_rows)
    monkeypatch.setattr(elementwise, "rms_modulate_q8", lambda x, w, e, s=None, h=None: plain_norm(x.float(), w, e, s, h))
    monkeypatch.setattr(elementwise, "residual_rms_q8", plain_residual)
    monkeypatch.setattr(elementwise, "glu_q8", plain_glu)
    monkeypatch.setattr(projection, "linear_q8", plain_linear_q8)
    monkeypatch.setattr(projection, "linear_q4", plain_linear_q4)
    ref = dit.dit_forward(params, x, t, static, SMALL, FP32_PARITY, projections="q8")
    assert torch.isfinite(got).all()
    assert rel(got, ref) <= 1e-2, rel(got, ref)


@pytest.mark.parametrize("preset", ["bf16", "fp16"])
def test_dit_forward_q8_is_near_the_unquantised_one(preset):
    announce(f"dit_forward medium q8 vs {preset}")
    dtype = {"bf16": BF16, "fp16": FP16}[preset]
    params, cond, mask, x = case(MEDIUM2, dtype, 2, 300, seed=24, ctx_tokens=257)
    params = dit.quantize_params(params)
    static = dit.prepare_static(params, cond, mask, MEDIUM2, dtype)
    t = torch.tensor([0.9, 0.35], device=DEV)
    got = dit.dit_forward(params, x, t, static, MEDIUM2, dtype, projections="q8")
    ref = dit.dit_forward(params, x, t, static, MEDIUM2, dtype)
    off = rel(got, ref)
    print(f"off by {off:.3f} of the output's norm")
    assert 1e-4 < off <= 0.25


def test_sampler_q8_graph_replays_equal_the_eager_loop():
    announce("PingpongGraph vs eager pingpong (q8)")
    params, cond, mask, x = case(MEDIUM2, BF16, 1, 200, seed=25, ctx_tokens=257)
    params = dit.quantize_params(params)
    static = dit.prepare_static(params, cond, mask, MEDIUM2, BF16)
    gen = torch.Generator().manual_seed(26)
    noise = torch.randn((3, 1, MEDIUM2.io_channels, 200), generator=gen).to(DEV)
    graph = sampling.PingpongGraph(params, static, MEDIUM2, BF16, x, noise, projections="q8")
    schedule = sampling.build_schedule(3, device=DEV)
    for rep in range(3):
        x_r = torch.randn(x.shape, generator=gen).to(DEV)
        n_r = torch.randn(noise.shape, generator=gen).to(DEV)
        got = graph(x_r, n_r).clone()
        torch.cuda.synchronize()
        ref, _ = sampling.pingpong(params, x_r, schedule, n_r, static, MEDIUM2, BF16, trajectory=False, projections="q8")
        torch.cuda.synchronize()
        assert torch.equal(got, ref), f"replay {rep}"
        _ = (torch.randn(1000, device=DEV) * 2).sum().item()  # unrelated eager work between replays


def test_q8_refusals():
    announce("q8 refusals")
    params, cond, mask, x = case(SMALL, BF16, 1, 20)
    static = dit.prepare_static(params, cond, mask, SMALL, BF16)
    t = torch.tensor([0.5], device=DEV)
    with pytest.raises(ValueError, match="quantize_params"):
        dit.dit_forward(params, x, t, static, SMALL, BF16, projections="q8")
    quantized = dit.quantize_params(params)
    with pytest.raises(ValueError, match="quantize_params"):  # the static state of the plain parameters
        dit.dit_forward(quantized, x, t, static, SMALL, BF16, projections="q8")
    xla = dataclasses.replace(SMALL, attention="xla")
    with pytest.raises(ValueError, match="hip"):
        dit.dit_forward(quantized, x, t, dit.prepare_static(quantized, cond, mask, xla, BF16), xla, BF16,
                        projections="q8")
    # the quantised parameters serve the other paths as before
    a = dit.dit_forward(params, x, t, static, SMALL, BF16)
    b = dit.dit_forward(quantized, x, t, dit.prepare_static(quantized, cond, mask, SMALL, BF16), SMALL, BF16)
    assert torch.equal(a, b)
    assert "q8" not in params["transformer"]["blocks"][0]["ff"]["proj_out"]
    with pytest.raises(ValueError):
        dit.quantize_params(dit.init_params(dataclasses.replace(SMALL, fourier_dim=16), BF16, device=DEV))
    assert MEDIUM_DIT.fourier_dim % 32 == 0 and MEDIUM_DIT.embed_dim % 32 == 0

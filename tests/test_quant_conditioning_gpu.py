"""The quantised denoiser operator by operator, and with its conditioning layers on 16-bit weights
(`quantize_params(conditioning="keep")`), on the GPU.

Inside `dit_forward(projections="q8")` at the medium widths every call of a quantised operator is compared with fp64 on
the operands that it was given, so that no error can hide in what the roundings to 8 bits leave anyway. (Whole passes
cannot be compared as closely: an error of d in a row moves some 11 d of its values over a border, each by a step of 2^-3,
which is sqrt(11 d) 2^-3.5 of its norm. From 1e-6 that makes 3e-4, and what follows in the same pass 5e-3 and 2e-2 of it:
plain operations on an input 1e-6 off differ by up to 1.2e-2 themselves.) Row operators and `linear_q4`: the bounds
derived in test_quant_gpu.py, and equality for `quantize_rows`. `linear_q8`: an output is the fp64 value, off by the
matrix cores' part c (2^-13 of the product's norm is allowed for 16-bit outputs, 2^-20 for fp32 ones) and rounded to the
output type: the squares of the two, independent, add up, with 2 % for the sample.

Against the 16-bit denoiser: an e4m3 value of mantissa m in [1, 2) is off by a uniform part of its step of 2^-3, in the
mean 2^-3 / sqrt(12) sqrt(mean(1 / m^2)) = 2.55 %; a product of two such operands by 3.6 %; three products in a row (a
feed-forward, an attention) by 6.25 %. The branches' errors are independent, as the branches are, and are added to a
stream that is not quantised: 6.25 % of the output's norm is allowed.
"""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import dit, elementwise, projection, sampling
from hummingbird_amd.dtypes import BF16, FP16, FP32_PARITY
from tests.test_quant_denoiser_gpu import rel
from tests.test_quant_gpu import check_q8, dequant_q4, norm_reference
from tests.test_sampler_gpu import MEDIUM2, case

pytestmark = pytest.mark.gpu
DEV = "cuda"
PRESETS = {"bf16": BF16, "fp16": FP16, "fp32": FP32_PARITY}


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def checked(monkeypatch) -> dict:
    """Every quantised operator wrapped by its comparison; the counts of their calls."""
    calls = {}
    real = {n: getattr(m, n) for m, names in ((elementwise, ("quantize_rows", "rms_modulate_q8", "residual_rms_q8", "glu_q8")),
                                              (projection, ("linear_q8", "linear_q4"))) for n in names}

    def quantize_rows(x):
        q, s = real["quantize_rows"](x)
        f = x.cpu().float()
        s_ref = (f.abs().amax(-1) / 448).clamp_min(2.0 ** -100)
        assert torch.equal(s.cpu(), s_ref)
        assert torch.equal(q.cpu().view(torch.uint8), (f / s_ref[..., None]).to(torch.float8_e4m3fn).view(torch.uint8))
        return q, s

    def rms_modulate_q8(x, weight, eps, scale=None, shift=None):
        q, s = real["rms_modulate_q8"](x, weight, eps, scale, shift)
        check_q8(q, s, *norm_reference(x.double(), x.double().abs(), weight, eps, scale, shift), "rms_modulate_q8")
        return q, s

    def residual_rms_q8(h, x, weight, eps, gate=None, x_bias=None, local=None, memory=0, scale=None, shift=None):
        out, q, s = real["residual_rms_q8"](h, x, weight, eps, gate, x_bias, local, memory, scale, shift)
        v, m = x.double(), x.double().abs()
        if x_bias is not None:
            v, m = v + x_bias.double(), m + x_bias.double().abs()
        if gate is not None:
            g = torch.sigmoid(1 - gate.double())[:, None]
            v, m = v * g, m * g
        v, m = h.double() + v, h.double().abs() + m
        if local is not None:
            v[:, memory:] += local.double()
            m[:, memory:] += local.double().abs()
        # rounded to half a step of the value, and of the type's least values (half: 2^-24 apart below 2^-14, so 2^-25)
        info = torch.finfo(h.dtype)
        assert ((out.double() - v).abs() <= info.eps / 2 * torch.clamp(v.abs(), min=info.tiny) + 2.0 ** -18 * m).all()
        check_q8(q, s, *norm_reference(v, m, weight, eps, scale, shift), "residual_rms_q8")
        return out, q, s

    def glu_q8(proj, bias=None):
        q, s = real["glu_q8"](proj, bias)
        z, m = proj.double() + bias.double(), proj.double().abs() + bias.double().abs()
        f = z.shape[-1] // 2
        act = torch.sigmoid(z[..., f:])
        check_q8(q, s, z[..., :f] * z[..., f:] * act, m[..., :f] * m[..., f:] * torch.clamp(act + 0.1, max=1.0) * 1.1, "glu")
        return q, s

    def linear_q8(x, x_scale, weight, weight_scale, bias=None, dtype=torch.bfloat16):
        got = real["linear_q8"](x, x_scale, weight, weight_scale, bias, dtype=dtype)
        ref = (x.double() * x_scale.double()[..., None]) @ (weight.double() * weight_scale.double()[:, None]).t()
        rounding = (ref.to(dtype).double() - ref).square().sum()
        core = (2.0 ** (-20 if dtype == torch.float32 else -13) * ref.norm()).square()
        assert (got.double() - ref).square().sum() <= 1.02 * rounding + core
        return got

    def linear_q4(x, weight, weight_scale, bias=None, silu=False):
        got = real["linear_q4"](x, weight, weight_scale, bias, silu)
        w = dequant_q4(weight, weight_scale)
        z = x.double() @ w.t() + bias.double()
        err = (3 * x.shape[-1] + 16) * 2.0 ** -24 * (x.double().abs() @ w.abs().t() + bias.double().abs())
        ref = z * torch.sigmoid(z) if silu else z
        err = 1.1 * err + 2.0 ** -18 * ref.abs() if silu else err
        assert ((got.double() - ref).abs() <= torch.finfo(x.dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + err
                + torch.finfo(x.dtype).tiny).all()
        return got
    wrapped = locals()

    def counted(name):
        def call(*args, **kw):
            calls[name] = calls.get(name, 0) + 1
            return wrapped[name](*args, **kw)
        return call
    for name in real:
        monkeypatch.setattr(projection if name.startswith("linear") else elementwise, name, counted(name))
    return calls


@pytest.mark.parametrize("preset", list(PRESETS))
@pytest.mark.parametrize("conditioning", ["q4", "keep"])
def test_every_operator_of_the_denoiser(monkeypatch, preset, conditioning):
    announce("denoiser operator by operator", preset, conditioning)
    dtype = PRESETS[preset]
    params, cond, mask, x = case(MEDIUM2, dtype, 2, 300, seed=41, ctx_tokens=257)
    params = dit.quantize_params(params, conditioning=conditioning)
    static = dit.prepare_static(params, cond, mask, MEDIUM2, dtype)
    calls = checked(monkeypatch)
    out = dit.dit_forward(params, x, torch.tensor([0.9, 0.35], device=DEV), static, MEDIUM2, dtype, projections="q8")
    assert torch.isfinite(out).all()
    depth = MEDIUM2.depth
    want = {"quantize_rows": 2 * depth, "rms_modulate_q8": 1, "residual_rms_q8": 3 * depth - 1, "glu_q8": depth,
            "linear_q8": 6 * depth}
    assert calls == (want if conditioning == "keep" else {**want, "linear_q4": 4})


@pytest.mark.parametrize("preset", ["bf16", "fp16"])
def test_kept_conditioning_is_near_the_unquantised_denoiser(preset):
    announce("denoiser, conditioning kept, vs", preset)
    dtype = PRESETS[preset]
    params, cond, mask, x = case(MEDIUM2, dtype, 2, 300, seed=24, ctx_tokens=257)
    quantized = dit.quantize_params(params, conditioning="keep")
    static = dit.prepare_static(quantized, cond, mask, MEDIUM2, dtype)
    t = torch.tensor([0.9, 0.35], device=DEV)
    ref = dit.dit_forward(quantized, x, t, static, MEDIUM2, dtype)
    off = rel(dit.dit_forward(quantized, x, t, static, MEDIUM2, dtype, projections="q8"), ref)
    print(f"off by {off:.4f} of the output's norm")
    assert 1e-4 < off <= 0.0625, off


def test_kept_conditioning_in_a_graph_and_refusals():
    announce("denoiser, conditioning kept: graph, refusals")
    params, cond, mask, x = case(MEDIUM2, BF16, 1, 100, seed=42, ctx_tokens=257)
    quantized = dit.quantize_params(dit.quantize_params(params), conditioning="keep")  # of a quantised model: 4 bits left out
    assert "q4" not in quantized["to_timestep_embed"]["in"]
    static = dit.prepare_static(quantized, cond, mask, MEDIUM2, BF16)
    noise = torch.randn((2, 1, MEDIUM2.io_channels, 100), device=DEV)
    graph = sampling.PingpongGraph(quantized, static, MEDIUM2, BF16, x, noise, projections="q8")
    ref, _ = sampling.pingpong(quantized, x, sampling.build_schedule(2, device=DEV), noise, static, MEDIUM2, BF16,
                               trajectory=False, projections="q8")
    for _ in range(3):
        got = graph(x, noise).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, ref)
    with pytest.raises(ValueError, match="conditioning"):
        dit.quantize_params(params, conditioning="q8")
    with pytest.raises(ValueError, match="quantize_params"):
        dit.dit_forward(params, x, torch.tensor([0.5], device=DEV), static, MEDIUM2, BF16, projections="q8")


@pytest.mark.parametrize("conditioning", ["q4", "keep"])
def test_16_bit_weights_can_be_let_go(conditioning):
    """The "q8" path reads no `weight` of a layer that has a `q8`: without them it gives the same bits."""
    announce("denoiser without the 16-bit weights", conditioning)
    params, cond, mask, x = case(MEDIUM2, BF16, 1, 100, seed=43, ctx_tokens=257)
    quantized = dit.quantize_params(params, conditioning=conditioning)
    t = torch.tensor([0.5], device=DEV)
    ref = dit.dit_forward(quantized, x, t, dit.prepare_static(quantized, cond, mask, MEDIUM2, BF16), MEDIUM2, BF16,
                          projections="q8")
    deleted = 0
    for block in quantized["transformer"]["blocks"]:
        for part in block.values():
            for layer in part.values() if isinstance(part, dict) else ():
                if isinstance(layer, dict) and "q8" in layer:
                    del layer["weight"]
                    deleted += 1
    assert deleted == 6 * MEDIUM2.depth
    assert "weight" in params["transformer"]["blocks"][0]["ff"]["proj_out"]  # the caller's own stay
    got = dit.dit_forward(quantized, x, t, dit.prepare_static(quantized, cond, mask, MEDIUM2, BF16), MEDIUM2, BF16,
                          projections="q8")
    assert torch.equal(got, ref)

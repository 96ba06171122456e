"""The denoiser without the second attention branch (`DiTConfig.differential=False`, sa3jax/dit.py:131-176) on the GPU, its
attentions on `packed_attention`.

* In fp32 against the same layers on the CPU with plain attention: 2e-5 of the output's largest magnitude, as the
  differential denoiser against its oracle.
* The medium width under the 16-bit presets against plain attention on the same device, at the bf16 contract applied to the
  output divided by its largest magnitude, as the differential denoiser.
* The sampler's graph against the eager loop, replayed with other work in between: equal bits.
"""
from __future__ import annotations

import dataclasses

import pytest
import torch

from hummingbird_amd import dit, sampling, xla_chain
from hummingbird_amd.dtypes import BF16, FP16, FP32_PARITY
from tests.test_sampler_gpu import HIP_TINY, MEDIUM2, case
from tests.util import assert_bf16_parity

pytestmark = pytest.mark.gpu
DEV = "cuda"
PLAIN = dataclasses.replace(HIP_TINY, differential=False)


def announce(name: str) -> None:
    print(f"\n[case] {name}", flush=True)


def host(tree):
    if isinstance(tree, dict):
        return {k: host(v) for k, v in tree.items()}
    if isinstance(tree, list):
        return [host(v) for v in tree]
    return tree.cpu()


def plain_attention(monkeypatch):
    """`dit`'s attentions as plain torch operations: one softmax, no second branch."""
    def split(t, cfg):
        return xla_chain.heads(t, cfg.num_heads, cfg.head_dim)

    def attend(q, k, v, cfg):
        out = [xla_chain.sdpa(*(t[:, h] for t in (q, k, v)), cfg.head_dim ** -0.5, q.dtype) for h in range(cfg.num_heads)]
        return xla_chain.merge(torch.stack(out, dim=1))

    def self_attention(h, block, static, cfg, lam=None, dtype=None, projections="torch"):
        attn = block["self_attn"]
        q, k, v = (split(t, cfg) for t in (h @ attn["to_qkv"]["weight"].to(h.dtype).t()).chunk(3, dim=-1))
        cos, sin = xla_chain.rope_tables(h.shape[1], static["inv_freq"])
        q, k = (xla_chain.rope(xla_chain.rms(t, attn[n]["weight"], cfg.qk_norm_eps), cos, sin, h.dtype)
                for t, n in ((q, "q_norm"), (k, "k_norm")))
        out = attend(q, k, v * static["valid"].to(h.dtype)[:, None, :, None], cfg)
        return out @ attn["to_out"]["weight"].to(h.dtype).t()

    def cross_context(block, ctx, cfg):
        attn = block["cross_attn"]
        k, v = (split(t, cfg) for t in (ctx @ attn["to_kv"]["weight"].to(ctx.dtype).t()).chunk(2, dim=-1))
        return xla_chain.rms(k, attn["k_norm"]["weight"], cfg.qk_norm_eps), v

    def cross_attention(h, block, context, cfg, lam=None, offsets=None):
        attn = block["cross_attn"]
        q = split(h @ attn["to_q"]["weight"].to(h.dtype).t(), cfg)
        out = attend(xla_chain.rms(q, attn["q_norm"]["weight"], cfg.qk_norm_eps), *context, cfg)
        return out @ attn["to_out"]["weight"].to(h.dtype).t()

    for f in (self_attention, cross_context, cross_attention):
        monkeypatch.setattr(dit, f.__name__, f)


def scrambled(params, seed):
    """`params` with norm weights of other values than one."""
    gen = torch.Generator().manual_seed(seed)
    for b in params["transformer"]["blocks"]:
        for part in ("self_attn", "cross_attn"):
            for n in ("q_norm", "k_norm"):
                w = b[part][n]["weight"]
                b[part][n]["weight"] = (1 + 0.3 * torch.randn(w.shape, generator=gen)).to(w)
    return params


@pytest.mark.parametrize("batch,tokens", [(2, 40), (1, 1), (3, 129)])
def test_fp32_vs_plain_operations(monkeypatch, batch, tokens):
    announce(f"dit_forward plain model fp32 B={batch} T={tokens}")
    params, cond, mask, x = case(PLAIN, FP32_PARITY, batch, tokens)
    params = scrambled(params, 5)
    t = torch.linspace(0.9, 0.3, batch, device=DEV)
    static = dit.prepare_static(params, cond, mask, PLAIN, FP32_PARITY)
    got = dit.dit_forward(params, x, t, static, PLAIN, FP32_PARITY).cpu()
    h = torch.randn(batch, tokens + PLAIN.num_memory_tokens, PLAIN.embed_dim, generator=torch.Generator().manual_seed(6))
    block = params["transformer"]["blocks"][1]
    one = dit.cross_attention(h.to(DEV), block, static["cross"][1], PLAIN).cpu()
    plain_attention(monkeypatch)
    cfg = dataclasses.replace(PLAIN, attention="xla")
    params, cond, mask, x = (host(v) for v in (params, cond, mask, x))
    static = dit.prepare_static(params, cond, mask, cfg, FP32_PARITY)
    ref = dit.dit_forward(params, x, t.cpu(), static, cfg, FP32_PARITY)
    assert (got - ref).abs().max() <= 2e-5 * ref.abs().max()
    ref = dit.cross_attention(h, params["transformer"]["blocks"][1], static["cross"][1], cfg)
    assert (one - ref).abs().max() <= 2e-5 * ref.abs().max()


@pytest.mark.parametrize("preset", ["bf16", "fp16"])
def test_medium_width_vs_plain_operations(monkeypatch, preset):
    announce(f"dit_forward plain model medium width {preset}")
    dtype = {"bf16": BF16, "fp16": FP16}[preset]
    cfg = dataclasses.replace(MEDIUM2, differential=False)
    params, cond, mask, x = case(cfg, dtype, 2, 300, seed=24, ctx_tokens=257)
    t = torch.tensor([0.9, 0.35], device=DEV)
    got = dit.dit_forward(params, x, t, dit.prepare_static(params, cond, mask, cfg, dtype), cfg, dtype).float().cpu()
    plain_attention(monkeypatch)
    xcfg = dataclasses.replace(cfg, attention="xla")
    static = dit.prepare_static(params, cond, mask, xcfg, dtype)
    ref = dit.dit_forward(params, x, t, static, xcfg, dtype).float().cpu()
    scale = float(ref.abs().max())
    assert_bf16_parity(got.numpy() / scale, ref.numpy() / scale, f"plain dit_forward {preset} / max")


def test_sampler_graph_replays_equal_the_eager_loop():
    announce("PingpongGraph vs eager pingpong (plain model)")
    cfg = dataclasses.replace(MEDIUM2, differential=False)
    params, cond, mask, x = case(cfg, BF16, 1, 200, seed=25, ctx_tokens=257)
    static = dit.prepare_static(params, cond, mask, cfg, BF16)
    gen = torch.Generator().manual_seed(26)
    noise = torch.randn((3, 1, cfg.io_channels, 200), generator=gen).to(DEV)
    graph = sampling.PingpongGraph(params, static, cfg, BF16, x, noise)
    schedule = sampling.build_schedule(3, device=DEV)
    for rep in range(3):
        x_r = torch.randn(x.shape, generator=gen).to(DEV)
        n_r = torch.randn(noise.shape, generator=gen).to(DEV)
        got = graph(x_r, n_r).clone()
        torch.cuda.synchronize()
        ref, _ = sampling.pingpong(params, x_r, schedule, n_r, static, cfg, BF16, trajectory=False)
        torch.cuda.synchronize()
        assert torch.equal(got, ref), f"replay {rep}"
        _ = (torch.randn(1000, device=DEV) * 2).sum().item()  # unrelated eager work between replays


def test_refusals():
    announce("plain model refusals")
    params, cond, mask, x = case(PLAIN, BF16, 2, 20)
    static = dit.prepare_static(params, cond, mask, PLAIN, BF16)
    block = params["transformer"]["blocks"][0]
    h = torch.zeros(2, 24, PLAIN.embed_dim, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="lam"):
        dit.self_attention(h, block, static, PLAIN, lam=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="lam"):
        dit.cross_attention(h, block, static["cross"][0], PLAIN, lam=torch.ones(2, device=DEV))
    with pytest.raises(TypeError, match="cross_context"):
        dit.cross_attention(h, block, tuple(static["cross"][0]), PLAIN)
    with pytest.raises(ValueError, match="batch"):
        dit.cross_attention(h[:1], block, static["cross"][0], PLAIN)
    with pytest.raises(ValueError, match="ROCm device"):
        dit.use_packed(PLAIN, h.cpu())
    cpu = dataclasses.replace(PLAIN, attention="xla")
    with pytest.raises(NotImplementedError):  # without "hip" only the differential chain is there
        dit.self_attention(h, block, static, cpu)

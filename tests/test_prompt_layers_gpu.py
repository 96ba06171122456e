"""Two layers of a transformer over prompts of different lengths, as the 4-bit rows, their products and the packed attention
are used together: norm and rows, [q | k | v], attention, rows, product, residual, norm and rows, GLU, product. Then new
tokens, one a prompt, over caches whose slots have room behind the keys.

Each stage is compared on the operands that the run gave it, so that no stage's rounding counts for the next: rows and
attention as tests/test_mx4_gpu.py and tests/test_packed_gpu.py derive it, products within K 2^-24 of the magnitudes' product
and one rounding. The captured runs, eager ones of the same inputs: equal bits."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew
from hummingbird_amd import packed_attention as pa
from hummingbird_amd import projection as pr
from tests.test_mx4_denoiser_gpu import glu64, norm64, residual64
from tests.test_mx4_gpu import DTYPES, check_rows, generator, rand, values
from tests.test_packed_gpu import check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
E, H, G, D, F = 512, 8, 2, 64, 1024
WIDTH = (H + 2 * G) * D


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def layers(count: int, dtype: torch.dtype) -> list[dict]:
    gen = generator(20, count)

    def weight(out, k):
        return pr.quantize_q4(rand(gen, out, k, std=k ** -0.5))
    return [dict(norm=rand(gen, E, std=0.1, mean=1.0), qkv=weight(WIDTH, E), qkv_bias=rand(gen, WIDTH, std=0.1),
                 out=weight(E, H * D), ff_norm=rand(gen, E, std=0.1, mean=1.0), glu=weight(2 * F, E),
                 glu_bias=rand(gen, 2 * F, std=0.1), down=weight(E, F), down_bias=rand(gen, E, std=0.1, dtype=dtype))
            for _ in range(count)]


def run(h, net, attend, seen=None):
    """`h` `(T, E)` through `net`; `attend(i, q, k, v)` -> `(T, H, D)`. `seen` is called with each stage's operands."""
    dt, T = h.dtype, h.shape[0]
    seen = seen or (lambda *a, **k: None)

    def product(stage, rows, weight, bias=None):
        out = pr.linear_mx4(*rows, *weight, bias, dtype=dt)
        seen("product", stage, out, rows, weight, bias)
        return out

    rows = ew.rms_modulate_mx4(h[None], net[0]["norm"], 1e-6)
    seen("norm", "first", rows, h, net[0]["norm"])
    for i, layer in enumerate(net):
        qkv = product("qkv", [t.reshape(T, -1) for t in rows], layer["qkv"], layer["qkv_bias"])
        q, k, v = (t.reshape(T, -1, D) for t in qkv.split([H * D, G * D, G * D], dim=1))
        a = attend(i, q, k, v)
        rows = ew.quantize_rows_mx4(a.reshape(T, H * D))
        seen("rows", "attention", rows, a.reshape(T, H * D))
        o = product("out", rows, layer["out"])
        before = h
        h, *rows = (t[0] for t in ew.residual_rms_mx4(h[None], o[None], layer["ff_norm"], 1e-6))
        seen("residual", "attention", (h, rows), before, o, None, layer["ff_norm"])
        p = product("glu", rows, layer["glu"])
        rows = ew.glu_mx4(p, layer["glu_bias"])
        seen("glu", "glu", rows, p, layer["glu_bias"])
        f = product("down", rows, layer["down"])
        before = h
        if i + 1 < len(net):
            h, *rows = (t[0] for t in ew.residual_rms_mx4(h[None], f[None], net[i + 1]["norm"], 1e-6,
                                                          x_bias=layer["down_bias"]))
            seen("residual", "down", (h, rows), before, f, layer["down_bias"], net[i + 1]["norm"])
        else:
            h = ew.gated_residual(h[None], f[None], x_bias=layer["down_bias"])[0]
    return h


def comparing(name):
    half_step = torch.finfo(DTYPES[name]).eps / 2
    least = 2.0 ** -24 if name == "fp16" else 0.0  # half's subnormals

    def seen(what, stage, out, *args):
        if what == "product":
            (x, s), (w, ws), bias = args
            a, b = values(x, s), values(w, ws).t().contiguous()
            ref, mag = a @ b, a.abs() @ b.abs()
            if bias is not None:
                ref, mag = ref + bias.double(), mag + bias.double().abs()
            tol = (a.shape[-1] + 1) * 2.0 ** -24 * mag + half_step * ref.abs() + least
            assert ((out.double() - ref).abs() <= (1 + half_step) * tol).all(), stage
        elif what == "norm":
            check_rows(*out, *norm64(args[0].double()[None], args[1], 1e-6, None, None), stage)
        elif what == "rows":
            x = args[0]
            check_rows(*out, x.double(), x.double().abs(), stage)
        elif what == "residual":
            (h, rows), (before, x, bias, weight) = out, args
            v, m = residual64(before, x, None, bias, None, 0)
            assert ((h.double() - v).abs() <= half_step * v.abs() + 2.0 ** -18 * m + least).all(), stage
            check_rows(*rows, *norm64(v, weight, 1e-6, None, None, m), stage)
        else:
            p, bias = args
            m = p.double().abs() + bias.double().abs()
            mv, mg = m.chunk(2, dim=-1)
            gate = (p.double() + bias.double()).chunk(2, dim=-1)[1]
            check_rows(*out, glu64(p, bias), mv * mg * torch.sigmoid(gate), stage)
    return seen


@pytest.mark.parametrize("name", list(DTYPES))
def test_prompts_and_new_tokens(name):
    dtype, lengths, room = DTYPES[name], [70, 1, 0, 133], 6
    announce("prompts and new tokens", name, lengths)
    net, T, scale = layers(2, dtype), sum(lengths), D ** -0.5
    at = offsets(lengths)
    slots = [n + room for n in lengths]
    starts = [sum(slots[:i]) for i in range(len(slots))]
    where = torch.cat([torch.arange(n) + s for n, s in zip(lengths, starts)]).to(DEV)
    caches = [[torch.full((sum(slots), G, D), float("nan"), device=DEV, dtype=dtype) for _ in "kv"] for _ in net]

    def prompts(i, q, k, v):
        out = pa.packed_attention(q, k, v, at)
        first = [sum(lengths[:j]) for j in range(len(lengths))]
        check(out, q, k, v, lengths, lengths, first, True, scale, name, f"prompts, layer {i}")
        for cache, t in zip(caches[i], (k, v)):
            cache[where] = t
        return out

    h = run(rand(generator(21), T, E, dtype=dtype), net, prompts, comparing(name))
    assert torch.isfinite(h).all()
    slot_offsets, one_each = offsets(slots), offsets([1] * len(slots))
    for step in range(room):
        held = [n + step + 1 for n in lengths]
        lens = torch.tensor(held, dtype=torch.int32, device=DEV)
        place = torch.tensor([s + n - 1 for s, n in zip(starts, held)], device=DEV)

        def tokens(i, q, k, v):
            for cache, t in zip(caches[i], (k, v)):
                cache[place] = t
            out = pa.packed_attention(q, *caches[i], one_each, slot_offsets, lens)
            check(out, q, *caches[i], [1] * len(slots), held, starts, True, scale, name, f"token {step}, layer {i}")
            return out

        h = run(rand(generator(22, step), len(slots), E, dtype=dtype), net, tokens, comparing(name))
        assert torch.isfinite(h).all()


@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_captured_step_over_a_growing_cache(name):
    """One captured step for new tokens serves every step: lengths and places are read on the device."""
    dtype = DTYPES[name]
    announce("captured step", name)
    net, slots = layers(2, dtype), [900, 40, 3000]
    starts = torch.tensor([0, 900, 940], device=DEV)
    caches = [[rand(generator(23, i, j), sum(slots), G, D, dtype=dtype) for j in range(2)] for i in range(len(net))]
    slot_offsets, one_each = offsets(slots), offsets([1, 1, 1])
    lens = torch.tensor([5, 1, 2990], dtype=torch.int32, device=DEV)
    h = rand(generator(24), 3, E, dtype=dtype)

    def step(x):
        def tokens(i, q, k, v):
            for cache, t in zip(caches[i], (k, v)):
                cache.index_copy_(0, starts + lens - 1, t)
            return pa.packed_attention(q, *caches[i], one_each, slot_offsets, lens)
        return run(x, net, tokens)

    step(h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(h)
    for turn in range(4):
        h.copy_(rand(generator(25, turn), 3, E, dtype=dtype))
        lens.add_(torch.tensor([1, 9, 2], dtype=torch.int32, device=DEV))
        held = [[t.clone() for t in pair] for pair in caches]
        graph.replay()
        got, after = out.clone(), [[t.clone() for t in pair] for pair in caches]
        for pair, old in zip(caches, held):
            for t, o in zip(pair, old):
                t.copy_(o)
        want = step(h)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for p, r in zip(after, caches) for a, b in zip(p, r))

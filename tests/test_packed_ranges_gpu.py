"""Attention over packed sequences on the GPU where scores and values span the range of their types: scores far above those
that came first, alone and in parts that are joined, values whose sums pass the range, rows beside such ones. Against the
plain fp64 implementation of `test_packed_gpu`, with its tolerances."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import _lib
from hummingbird_amd import packed_attention as pa
from tests import test_packed_gpu as plain

pytestmark = pytest.mark.gpu
DEV, DTYPES, CODES = plain.DEV, plain.DTYPES, {"bf16": 0, "fp32": 1, "fp16": 2}


def scored(name, scores, D=64):
    """Keys `(n, 1, D)` whose products with queries of 4 in their first two values, scaled by 1/4, are `scores` `(n,)`
    exactly: multiples of 1/4 up to 128 in magnitude, a whole number and a fraction, each of 8 bits at most."""
    k = torch.zeros(scores.shape[0], 1, D, device=DEV)
    k[:, 0, 0] = torch.trunc(scores)
    k[:, 0, 1] = scores - k[:, 0, 0]
    return k.to(DTYPES[name])


def queries(name, n, D=64):
    q = torch.zeros(n, 1, D, device=DEV)
    q[..., :2] = 4.0
    return q.to(DTYPES[name])


def values(name, n, size, seed, D=64):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (size * (0.5 + 0.5 * torch.rand(n, 1, D, generator=gen, device=DEV))).to(DTYPES[name])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("size", [2.0 ** -10, 0.25, 1.0])
def test_scores_above_the_first_tile(name, size):
    """64 keys of score 0 and then 64 of x, x from 60 to 100 in quarters: totals that pass 2^128 in a lane's half of the
    keys, in the two halves together and not at all."""
    plain.announce("packed scores above the first tile", name, size)
    x = torch.arange(60, 100.25, 0.25, device=DEV)
    n = x.numel()
    k = scored(name, torch.stack([torch.zeros_like(x), x], dim=1).repeat_interleave(64, dim=1).reshape(-1))
    v = values(name, 128 * n, size, 1)
    lq, lk = [3] * n, [128] * n
    q, starts = queries(name, 3 * n), [128 * i for i in range(n)]
    for causal in (False, True):
        got = pa.packed_attention(q, k, v, plain.offsets(lq), plain.offsets(lk), causal=causal, scale=0.25)
        plain.check(got, q, k, v, lq, lk, starts, causal, 0.25, name, causal)


def split(name, T, Tk, N, D=64):
    """How many parts a call of one head has (0: one)."""
    return _lib.load().hb_packed_workspace_size(CODES[name], T, Tk, N, 1, 1, D) // (T * (D + 2) * 4)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("size", [2.0 ** -10, 1.0])
def test_parts_of_far_references(name, size):
    """One token over keys in parts, most of them x below, x from 60 to 100: of two keys that weigh alike one lies behind
    its part's first tile, which is x below it, and the other begins its part."""
    plain.announce("packed parts of far references", name, size)
    low = -torch.arange(60, 101, 1, device=DEV, dtype=torch.float32)
    n, keys = low.numel(), 5000
    assert split(name, n, n * keys, n)
    scores = low[:, None].repeat(1, keys)
    scores[:, 100], scores[:, 320] = -0.25, 0.0
    q, k, v = queries(name, n), scored(name, scores.reshape(-1)), values(name, n * keys, size, 2)
    starts = [keys * i for i in range(n)]
    got = pa.packed_attention(q, k, v, plain.offsets([1] * n), plain.offsets([keys] * n), scale=0.25)
    plain.check(got, q, k, v, [1] * n, [keys] * n, starts, True, 0.25, name, "far references")


@pytest.mark.parametrize("name", list(DTYPES))
def test_parts_that_weigh_little(name):
    """A part with a key of score 0 and others whose first tiles lie x below, x from 80 to 92, with one key each 69.25 above that (99.9
    binary orders): a weight of 2e-5 to 1e-10 each, under values so large that together they are seen."""
    plain.announce("packed parts that weigh little", name)
    low = -torch.arange(80, 92.25, 0.25, device=DEV)
    n, keys = low.numel(), 5000
    each = -(-keys // split(name, n, n * keys, n))
    each += -each % 64  # 16-bit parts' keys
    assert each >= 64
    scores = low[:, None].repeat(1, keys)
    scores[:, each + 150::each] = low[:, None] + 69.25
    scores[:, 0] = 0.0
    q, k, v = queries(name, n), scored(name, scores.reshape(-1)), values(name, n * keys, 1.0, 2)
    v.view(n, keys, 64)[:, each + 150::each] *= 2.0 ** (19 if name != "fp16" else 15)
    starts = [keys * i for i in range(n)]
    got = pa.packed_attention(q, k, v, plain.offsets([1] * n), plain.offsets([keys] * n), scale=0.25)
    plain.check(got, q, k, v, [1] * n, [keys] * n, starts, True, 0.25, name, "weigh little")


@pytest.mark.parametrize("name", list(DTYPES))
def test_parts_with_large_totals(name):
    """Parts that all begin with 64 keys of score 0 and go on with x, x from 60 to 100: totals of 2^100 to 2^128 each,
    which are added; parts that begin with scores of minus infinity; every row in one part, most of its keys low."""
    plain.announce("packed parts with large totals", name)
    x = torch.arange(60, 101, 1, device=DEV, dtype=torch.float32)
    n, keys = x.numel(), 5000
    assert split(name, n, n * keys, n)
    at = torch.arange(keys, device=DEV)
    q, v = queries(name, n), values(name, n * keys, 1.0, 3)
    starts = [keys * i for i in range(n)]
    for what, first in (("zero", 0.0), ("minus infinity", float("-inf"))):
        scores = torch.where(at % 64 % 5 == 0 if what == "zero" else at < 320, first, x[:, None].expand(n, keys))
        scores[:, :64] = first
        scores[:, at % 320 < 64] = first
        k = scored(name, torch.nan_to_num(scores, neginf=0.0).reshape(-1))
        k[..., 0].masked_fill_(torch.isinf(scores).reshape(-1, 1), float("-inf"))
        got = pa.packed_attention(q, k, v, plain.offsets([1] * n), plain.offsets([keys] * n), scale=0.25)
        plain.check(got, q, k, v, [1] * n, [keys] * n, starts, True, 0.25, name, what)


@pytest.mark.parametrize("name", list(DTYPES))
def test_bits_do_not_depend_on_the_neighbours(name):
    """Rows of the tile in which one is repeated (a NaN in a value that the others do not see, scores of another row that
    pass the range) have the bits that they have without it, whatever their own scores' range."""
    plain.announce("packed bits beside", name)
    n, D = 128, 64
    q, k, v = plain.make(name, n, n, 1, 1, D, 31)
    q, k = q * 0.5, k * 0.5
    q[..., 0] = 4.0
    at = plain.offsets([n])
    for x in (0.0, 3.0, 60.0, 70.0, 73.0, 76.0, 80.0, 83.0, 86.0, 88.0, 95.0):
        kk = k.clone()
        kk[:, :, 0] = 0.0
        kk[64:, :, 0] = x
        want = pa.packed_attention(q, kk, v, at, causal=True, scale=0.25)
        vv = v.clone()
        vv[127] = float("nan")
        got = pa.packed_attention(q, kk, vv, at, causal=True, scale=0.25)
        assert torch.equal(got[:127], want[:127]), x
        assert torch.isnan(got[127]).all() and torch.isfinite(want).all()
        qq = q.clone()
        qq[100, :, 0] = 400.0  # its scores pass the first tile's by a hundred times as much
        for causal in (False, True):
            want = pa.packed_attention(q, kk, v, at, causal=causal, scale=0.25)
            got = pa.packed_attention(qq, kk, v, at, causal=causal, scale=0.25)
            assert torch.equal(got[:100], want[:100]) and torch.equal(got[101:], want[101:]), (x, causal)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_large_values(name):
    """Values of 2^40 to 2^127 under scores that rise by 0 to 70 after the first tile: each result is a mean of values,
    and finite."""
    plain.announce("packed large values", name)
    x = torch.tensor([0.0, 5.0, 30.0, 42.0, 50.0, 55.0, 60.0, 65.0, 69.0, 70.0], device=DEV)
    n = x.numel()
    for keys, lq in ((192, 2), (3000, 1)):
        scores = torch.zeros(n, keys, device=DEV)
        scores[:, 64:] = x[:, None]
        k, q = scored(name, scores.reshape(-1)), queries(name, lq * n)
        starts = [keys * i for i in range(n)]
        for e in (40, 90, 119, 121, 127):
            v = values(name, n * keys, 2.0 ** e, 4)
            v[::4] = -v[::4]
            got = pa.packed_attention(q, k, v, plain.offsets([lq] * n), plain.offsets([keys] * n), scale=0.25)
            assert torch.isfinite(got).all(), (keys, e)
            plain.check(got, q, k, v, [lq] * n, [keys] * n, starts, True, 0.25, name, (keys, e))
        top = torch.full_like(v, torch.finfo(v.dtype).max * (1 - 2.0 ** -7))
        got = pa.packed_attention(q, k, top, plain.offsets([lq] * n), plain.offsets([keys] * n), scale=0.25)
        assert torch.isfinite(got).all()
        assert ((got.double() - top[:1].double()).abs() <= 2.0 ** -7 * top[:1].double()).all()


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("keys", [100, 5000])
def test_scores_past_two_to_the_24(name, keys):
    """Scores whose rounding in the exponent's units is whole binary orders: all are 251 x 239 x 2^e or, for every second
    key, half of that, exactly, so that the result is the mean of the values of the others. The tolerance of `check` without
    the scores' part: a probability's rounding twice, n steps of fp32 and the output's rounding."""
    plain.announce("packed scores past 2^24", name, keys)
    v = values(name, keys, 1.0, 5)
    tol = 2 * (2 * plain.HELD[name] + 2 * keys * 2.0 ** -24 + plain.HALF_STEP[name])
    for e in (4, 8, 10, 11, 12, 13, 14, 15, 16) + (() if name == "fp16" else (18, 20, 26, 50)):
        k = torch.zeros(keys, 1, 64, device=DEV)
        k[0::2, 0, 0], k[1::2, 0, 0] = 251 * 2.0 ** (e // 2), 251 * 2.0 ** (e // 2 - 1)
        for sign in (1.0, -1.0):
            q = torch.zeros(1, 1, 64, device=DEV)
            q[0, 0, 0] = sign * 239 * 2.0 ** (e - e // 2)
            for scale in (1.0, 0.3, 0.7, 0.11):
                got = pa.packed_attention(q.to(v.dtype), k.to(v.dtype), v, plain.offsets([1]), plain.offsets([keys]),
                                          scale=scale)
                want = v[0 if sign > 0 else 1::2].double().mean(0)
                assert ((got[0].double() - want).abs() <= tol * want).all(), (e, sign, scale)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_any_ranges(name, D):
    """Scores spread over 1 to 300 and values over 2^40 each way (half: 2^7), a key of minus infinity and a value of NaN in the
    middle of some sequences: each pass of the kernel for some rows of a tile and not for others, whole and in parts."""
    plain.announce("packed any ranges", name, D)
    gen = torch.Generator(device=DEV).manual_seed(6)
    for lq, lk, H, G in (([70, 5, 130], [70, 90, 130], 4, 2), ([3, 1], [3000, 2500], 8, 2), ([150], [1100], 3, 3)):
        T, Tk = sum(lq), sum(lk)
        starts = [sum(lk[:i]) for i in range(len(lk))]
        for spread in (1.0, 30.0, 100.0, 300.0):
            q, k, v = plain.make(name, T, Tk, H, G, D, int(spread))
            row = torch.rand(T, H, 1, generator=gen, device=DEV)  # some rows' scores spread less
            q = (q.float() * row * spread ** 0.5).to(q.dtype)
            k = (k.float() * spread ** 0.5).to(q.dtype)
            size = torch.rand(Tk, G, 1, generator=gen, device=DEV) * 2 - 1
            v = (v.float() * torch.exp2(size * (7 if name == "fp16" else 40))).to(q.dtype)
            for bad in (False, True):
                if bad:
                    k[starts[-1] + 7, 0] = 0
                    k[starts[-1] + 7, 0, 3] = float("-inf")
                    q[..., 3] = q[..., 3].abs() + 0.5
                    v[starts[0] + 40, G - 1, 5] = float("nan")
                for causal in (False, True):
                    got = pa.packed_attention(q, k, v, plain.offsets(lq), plain.offsets(lk), causal=causal)
                    plain.check(got, q, k, v, lq, lk, starts, causal, D ** -0.5, name, (lq, spread, bad, causal))

"""Attention over packed sequences on the GPU against a plain fp64 implementation.

Tolerance. With u the half step of the type that holds the probabilities (bf16 2^-8, half 2^-11; fp32: the hardware
exponential's 2^-22), each probability is off by u of itself, in the numerator and in the total: 2 u A, with A the
attention of |v|. A score is a sum of D products (D 2^-24 of scale |q| |k|), and the exponent's argument is rounded once at its
size: together e = (D + 4) 2^-24 max(scale |q| |k|) in the exponent, so 2 e A; the sums over n keys add n 2^-24 each,
2 n 2^-24 A; and the output is rounded once, u_out |out|, half's subnormals 2^-25. 16-bit probabilities below the type's least
are lost: half 2^-25 each of the largest, n 2^-25 max |v|. Everything is doubled for the second orders.
"""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import _lib
from hummingbird_amd import packed_attention as pa

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
HELD = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -22}


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


def offsets(lengths) -> torch.Tensor:
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=DEV)


def reference(q, k, v, lq, lk, starts, causal, scale):
    """(out, A, e) in fp64 for sequences of lq queries one after the other and lk keys from `starts` on."""
    T, H, D = q.shape
    per = H // k.shape[1]
    out, mag, e = (torch.zeros(T, H, n, dtype=torch.float64, device=q.device) for n in (D, D, 1))
    t = 0
    for a, b, at in zip(lq, lk, starts):
        for h in range(H):
            x, y, z = q[t:t + a, h].double(), k[at:at + b, h // per].double(), v[at:at + b, h // per].double()
            s = scale * (x @ y.t().contiguous())
            hidden = torch.zeros(a, b, dtype=torch.bool, device=q.device)
            if causal:
                hidden = torch.ones_like(hidden).triu(b - a + 1)
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), dim=1)
            p = torch.nan_to_num(p, nan=0.0) if hidden.any() or b == 0 else p
            out[t:t + a, h] = torch.where(hidden[:, :, None], 0.0, p[:, :, None] * z[None]).sum(1) if (
                a * b * D < 1 << 24) else p @ z
            mag[t:t + a, h] = p @ torch.nan_to_num(z, 0, 0, 0).abs()
            size = scale * (x.abs() @ y.abs().t().contiguous())
            e[t:t + a, h, 0] = torch.nan_to_num(size, 0, 0, 0).masked_fill(hidden, 0).amax(1) if b else 0
        t += a
    return out, mag, e


def check(got, q, k, v, lq, lk, starts, causal, scale, name, what):
    ref, mag, e = reference(q, k, v, lq, lk, starts, causal, scale)
    n, D = max(list(lk) + [1]), q.shape[2]
    tol = 2 * (2 * HELD[name] + 2 * (D + 4) * 2.0 ** -24 * e + 2 * n * 2.0 ** -24) * mag + 2 * HALF_STEP[name] * ref.abs()
    if name == "fp16":
        tol = tol + 2.0 ** -24 + n * 2.0 ** -24 * torch.nan_to_num(v.double(), 0, 0, 0).abs().max() / max(1, n)
    rows = sum(lq)
    bad = ~((got[:rows].double() - ref[:rows]).abs() <= tol[:rows]) & ~(
        (got[:rows].double() == ref[:rows]) | (torch.isnan(got[:rows]) & torch.isnan(ref[:rows])))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"


def make(name, T, Tk, H, G, D, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda n, h: torch.randn(n, h, D, generator=gen, device=DEV).to(DTYPES[name])  # noqa: E731
    return r(T, H), r(Tk, G), r(Tk, G)


LENGTHS = [[1], [64], [130], [63, 0, 65, 1, 128], [0, 0, 5], [200, 3, 129, 257], [31, 32, 33, 95, 96, 97, 2, 300]]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (6, 2), (8, 1), (5, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_packs(name, D, H, G, causal):
    for i, lengths in enumerate(LENGTHS):
        announce("packed", name, D, H, G, causal, lengths)
        q, k, v = make(name, sum(lengths), sum(lengths), H, G, D, 100 * D + H + i)
        got = pa.packed_attention(q, k, v, offsets(lengths), causal=causal)
        starts = [sum(lengths[:j]) for j in range(len(lengths))]
        check(got, q, k, v, lengths, lengths, starts, causal, D ** -0.5, name, lengths)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
def test_other_keys(name, causal):
    """More and fewer keys than queries, none, lengths inside slots; causal rows that see none give zeros."""
    lq, slots, lk = [3, 70, 1, 0, 40, 9], [200, 80, 65, 10, 64, 30], [130, 20, 65, 4, 0, 30]
    for D, H, G in ((64, 4, 2), (128, 3, 3)):
        announce("packed other keys", name, causal, D, H, G)
        q, k, v = make(name, sum(lq), sum(slots), H, G, D, 7)
        starts = [sum(slots[:j]) for j in range(len(slots))]
        lengths = torch.tensor(lk, dtype=torch.int32, device=DEV)
        got = pa.packed_attention(q, k, v, offsets(lq), offsets(slots), lengths, causal=causal, scale=0.3)
        check(got, q, k, v, lq, lk, starts, causal, 0.3, name, "slots")
        got = pa.packed_attention(q, k, v, offsets(lq), offsets(slots), causal=causal, scale=0.3)
        check(got, q, k, v, lq, slots, starts, causal, 0.3, name, "whole slots")
        no_keys = k[:0]
        got = pa.packed_attention(q, no_keys, no_keys, offsets(lq), offsets([0] * 6), causal=causal)
        assert torch.equal(got, torch.zeros_like(q))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("D,H,G", [(64, 4, 1), (128, 8, 2)])
def test_split_keys(name, D, H, G):
    """Few rows over many keys: the keys are split and the parts joined (some parts have none of a short sequence's)."""
    for lq, lk in (([1], [5000]), ([1, 1, 1], [3000, 1, 4100]), ([5, 0, 2], [4000, 700, 0]), ([40], [9001])):
        announce("packed split", name, D, H, G, lq, lk)
        need = _lib.load().hb_packed_workspace_size({"bf16": 0, "fp32": 1, "fp16": 2}[name], sum(lq), sum(lk), len(lq), H,
                                                    G, D)
        assert need > 0
        q, k, v = make(name, sum(lq), sum(lk), H, G, D, 8)
        starts = [sum(lk[:j]) for j in range(len(lk))]
        for causal in (False, True):
            got = pa.packed_attention(q, k, v, offsets(lq), offsets(lk), causal=causal)
            check(got, q, k, v, lq, lk, starts, causal, D ** -0.5, name, (lq, lk, causal))


@pytest.mark.parametrize("name", list(DTYPES))
def test_large_scores(name):
    """Scores of hundreds, rising along the keys (each tile has a new maximum) and falling."""
    announce("packed large scores", name)
    D, n = 64, 400
    q, k, v = make(name, n, n, 2, 2, D, 9)
    q = (q.abs() + 0.5).to(DTYPES[name])
    ramp = torch.linspace(-3, 3, n, device=DEV)[:, None, None]
    for slope in (ramp, -ramp):
        kk = (k * 0.1 + slope).to(DTYPES[name])
        for causal in (False, True):
            got = pa.packed_attention(q, kk, v, offsets([n]), causal=causal, scale=1.0)
            check(got, q, kk, v, [n], [n], [0], causal, 1.0, name, (float(slope[0]), causal))


@pytest.mark.parametrize("name", list(DTYPES))
def test_scores_far_above_the_first_ones(name):
    """Later keys whose scores pass the first tile's by more than any type's exponent range holds, in steps."""
    announce("packed far scores", name)
    D, n = 64, 330
    q, k, v = make(name, n, n, 2, 1, D, 17)
    q[..., 0] = 4.0
    for step in (30.0, 90.0, 126.0, 400.0):
        kk = (k * 0.1).contiguous()
        kk[..., 0] = torch.div(torch.arange(n, device=DEV), 64, rounding_mode="floor")[:, None] * step
        for causal in (False, True):
            got = pa.packed_attention(q, kk, v, offsets([n]), causal=causal, scale=0.25)
            check(got, q, kk, v, [n], [n], [0], causal, 0.25, name, (step, causal))


@pytest.mark.parametrize("name", list(DTYPES))
def test_scores_of_minus_infinity(name):
    """Keys whose scores are minus infinity weigh nothing, a first tile of them too, whatever the later scores are; a row of
    nothing else is zero."""
    announce("packed scores of minus infinity", name)
    D, n = 64, 200
    q, k, v = make(name, n, n, 2, 1, D, 19)
    q[..., :2] = 1.0
    for shift in (-300.0, 0.0, 300.0):
        kk = (k * 0.1).contiguous()
        kk[..., 1] = shift
        kk[:130, :, 0] = float("-inf")
        got = pa.packed_attention(q, kk, v, offsets([n]), causal=False, scale=1.0)
        check(got, q, kk[130:], v[130:], [n], [n - 130], [0], False, 1.0, name, shift)
        got = pa.packed_attention(q, kk, v, offsets([n]), causal=True, scale=1.0)
        assert (got[:130] == 0).all()
        check(got[130:], q[130:], kk[130:], v[130:], [n - 130], [n - 130], [0], True, 1.0, name, (shift, "causal"))


@pytest.mark.parametrize("name", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_enough_for_two_a_cu(name, D):
    """Sequences of very different lengths, enough tiles that fp32 ones are taken in another order; some empty, some equal."""
    announce("packed many tiles", name, D)
    for lengths in ([5, 0, 300, 131, 131, 0, 1, 250, 40, 129, 64, 128] * 2, [3] * 30 + [200] * 34, [70] * 65):
        H = 24
        q, k, v = make(name, sum(lengths), sum(lengths), H, H, D, 21)
        starts = [sum(lengths[:j]) for j in range(len(lengths))]
        for causal in (False, True):
            got = pa.packed_attention(q, k, v, offsets(lengths), causal=causal)
            check(got, q, k, v, lengths, lengths, starts, causal, D ** -0.5, name, (lengths[:3], causal))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_keys_that_are_not_seen(name, D):
    """NaN and infinities in keys and values that a row does not see (later ones of its own sequence, the next sequence's,
    a slot's room) leave it as it is; in those that it sees they reach it."""
    announce("packed hidden NaN", name, D)
    lengths, H, G = [70, 5, 130], 4, 2
    q, k, v = make(name, 205, 205, H, G, D, 10)
    clean = pa.packed_attention(q, k, v, offsets(lengths), causal=True)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for token, seq in ((40, 0), (72, 1), (75, 2), (204, 2), (139, 2)):
            for what in "kv":
                kk, vv = k.clone(), v.clone()
                (kk if what == "k" else vv)[token, 1, 3] = bad
                got = pa.packed_attention(q, kk, vv, offsets(lengths), causal=True)
                end = sum(lengths[:seq + 1])
                assert torch.equal(got[:token], clean[:token]), (bad, token, what)
                assert torch.equal(got[end:], clean[end:])
                assert torch.equal(got[:, :2], clean[:, :2])  # the other head of keys
                if what == "v":
                    seen = got[token:end, 2:, 3]
                    assert (torch.isnan(seen) if bad != bad else seen == bad).all()
                    assert torch.equal(got[token:end, 2:, 4:], clean[token:end, 2:, 4:])
    kk, vv = k.clone(), v.clone()
    kk[60:70], vv[60:70] = float("nan"), float("inf")  # a slot's room
    at, n = offsets(lengths), torch.tensor([60, 5, 130], dtype=torch.int32, device=DEV)
    for causal in (False, True):
        want = pa.packed_attention(q, k, v, at, at, n, causal=causal)
        assert torch.equal(pa.packed_attention(q, kk, vv, at, at, n, causal=causal), want)
        assert torch.isfinite(want).all()


@pytest.mark.parametrize("name", list(DTYPES))
def test_layouts(name):
    """Slices of one projection's rows, heads before tokens, padded rows, out with strides of its own."""
    announce("packed layouts", name)
    lengths, H, G, D = [50, 90, 7], 6, 3, 64
    T = sum(lengths)
    q, k, v = make(name, T, T, H, G, D, 11)
    want = pa.packed_attention(q, k, v, offsets(lengths))
    rows = torch.cat([t.reshape(T, -1) for t in (q, k, v)], dim=1)
    a, b, c = (t.reshape(T, -1, D) for t in rows.split([H * D, G * D, G * D], dim=1))
    assert torch.equal(pa.packed_attention(a, b, c, offsets(lengths)), want)
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(pa.packed_attention(*by_head, offsets(lengths)), want)
    room = torch.full((T, H, D + 16), 7.0, device=DEV, dtype=q.dtype)
    got = pa.packed_attention(q, k, v, offsets(lengths), out=room[..., :D])
    assert torch.equal(got, want) and (room[..., D:] == 7).all()
    by_head = torch.empty(H, T, D, device=DEV, dtype=q.dtype).transpose(0, 1)
    assert torch.equal(pa.packed_attention(q, k, v, offsets(lengths), out=by_head), want)


def test_strides_of_axes_of_one():
    announce("packed axes of one")
    q, k, v = make("bf16", 1, 70, 4, 1, 64, 18)
    at, koff = offsets([1]), offsets([70])
    want = pa.packed_attention(q, k, v, at, koff)
    odd = [q.as_strided(q.shape, (3, 64, 1)), k.as_strided(k.shape, (64, 5, 1)), v.as_strided(v.shape, (64, 1, 1))]
    out = torch.empty_like(q).as_strided(q.shape, (7, 64, 1))
    assert torch.equal(pa.packed_attention(*odd, at, koff, out=out), want)


def test_tokens_of_no_sequence():
    announce("packed rest")
    for H, G, D, split in ((4, 2, 64, False), (8, 2, 128, True)):
        T = 400 if not split else 12
        keys = T if not split else 6000
        q, k, v = make("bf16", T, keys, H, G, D, 12)
        at = torch.tensor([3, 3, 9], dtype=torch.int32, device=DEV)
        koff = at if not split else torch.tensor([0, 10, 6000], dtype=torch.int32, device=DEV)
        fresh = pa.packed_attention(q, k, v, at, koff)
        assert (fresh[:3] == 0).all() and (fresh[9:] == 0).all() and (fresh[3:9] != 0).any()
        out = torch.full_like(q, 5.0)
        got = pa.packed_attention(q, k, v, at, koff, out=out)
        assert got is out and (out[:3] == 5).all() and (out[9:] == 5).all() and torch.equal(out[3:9], fresh[3:9])
    assert torch.equal(pa.packed_attention(q, k, v, at[:1]), torch.zeros_like(q))
    assert pa.packed_attention(q[:0], k, v, torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (0, 8, 128)


def test_many_sequences():
    """More sequences than a wave looks at, most of them empty or of one token."""
    announce("packed many")
    lengths = [(7 * i) % 5 % 3 for i in range(333)] + [140]
    q, k, v = make("bf16", sum(lengths), sum(lengths), 2, 1, 64, 13)
    starts = [sum(lengths[:j]) for j in range(len(lengths))]
    for causal in (False, True):
        got = pa.packed_attention(q, k, v, offsets(lengths), causal=causal)
        check(got, q, k, v, lengths, lengths, starts, causal, 0.125, "bf16", causal)


def test_offsets_out_of_range_are_taken_as_the_nearest():
    announce("packed clamped offsets")
    q, k, v = make("bf16", 100, 100, 2, 2, 64, 14)
    want = pa.packed_attention(q, k, v, offsets([100]))
    wild = torch.tensor([-5, 1 << 30], dtype=torch.int32, device=DEV)
    assert torch.equal(pa.packed_attention(q, k, v, wild), want)
    down = torch.tensor([50, 20, 100], dtype=torch.int32, device=DEV)
    pa.packed_attention(q, k, v, down)  # (which values is not specified)
    torch.cuda.synchronize()


def test_captured_calls_follow_their_offsets():
    """Two graphs, one with split keys, replayed in turn with new lengths and eager calls between."""
    announce("packed graphs")
    sizes = [(300, 300, 4, 2), (2, 4000, 8, 2)]
    cases = []
    for T, Tk, H, G in sizes:
        q, k, v = make("fp16", T, Tk, H, G, 64, 15 + T)
        off, koff = offsets([T // 2, T - T // 2]), offsets([Tk // 2, Tk - Tk // 2])
        lens = (koff[1:] - koff[:-1]).contiguous()
        pa.packed_attention(q, k, v, off, koff, lens)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pa.packed_attention(q, k, v, off, koff, lens)
        cases.append((g, out, q, k, v, off, koff, lens))
    for step in range(4):
        for g, out, q, k, v, off, koff, lens in cases:
            T, half = q.shape[0], k.shape[0] // 2
            off[1] = [T // 2, 1, T - 1, T // 2][step]
            lens.copy_(torch.tensor([[half, half], [3, half], [half - 9, 1], [0, half]][step], dtype=torch.int32))
            out.fill_(3)
            g.replay()
            want = pa.packed_attention(q, k, v, off, koff, lens)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_on_another_stream():
    announce("packed stream")
    q, k, v = make("bf16", 3, 5000, 8, 2, 128, 16)
    off, koff = offsets([1, 2]), offsets([2000, 3000])
    want = pa.packed_attention(q, k, v, off, koff)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.packed_attention(q, k, v, off, koff)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    again = [pa.packed_attention(q, k, v, off, koff) for _ in range(3)]
    assert all(torch.equal(t, want) for t in again)


def test_tokens_and_heads_past_32_bits():
    """Keys, values, queries and outputs whose places pass 2^32 bytes: a token of each every 2 MB, heads 3 GB apart."""
    announce("packed past 32 bits")
    n, D, step = 2300, 64, 1 << 20
    for name in ("bf16", "fp32"):
        buf = torch.empty(n * step + 3 * D, dtype=DTYPES[name], device=DEV)
        q, k, v = make(name, n, n, 1, 1, D, 22)
        far = [buf.as_strided((n, 1, D), (step, D, 1), i * D) for i in range(3)]
        for f, t in zip(far, (q, k, v)):
            f.copy_(t)
        lengths = [1000, 1, 1299]
        want = pa.packed_attention(q, k, v, offsets(lengths))
        assert torch.equal(pa.packed_attention(*far, offsets(lengths)), want)
        few = [q[-3:], q[:3]]
        at, koff = offsets([1, 2]), offsets([1000, 1300])
        for rows in few:
            assert torch.equal(pa.packed_attention(rows, far[1], far[2], at, koff),
                               pa.packed_attention(rows, k, v, at, koff))
        far[0].fill_(5)
        got = pa.packed_attention(q, k, v, offsets(lengths), out=far[0])
        assert torch.equal(got.clone(), want) and torch.equal(far[1].clone(), k)
        wide = buf.as_strided((40, 2, D), (D, 800 * step, 1))
        x, y, z = make(name, 40, 40, 2, 2, D, 23)
        wide.copy_(y)
        assert torch.equal(pa.packed_attention(x, wide, z, offsets([40])), pa.packed_attention(x, y, z, offsets([40])))
        del buf, far, wide


def test_wrapper_refusals():
    announce("packed refusals")
    q, k, v = make("bf16", 10, 10, 4, 2, 64, 24)
    at = offsets([10])
    calls = [
        (ValueError, (q[0], k, v, at), {}), (ValueError, (q, k[..., 0], v, at), {}),
        (TypeError, (q, k.half(), v, at), {}), (TypeError, (q, k, v.float(), at), {}),
        (TypeError, (q, k.cpu(), v, at), {}), (ValueError, (q.cpu(), k.cpu(), v.cpu(), at.cpu()), {}),
        (TypeError, (q.int(), k.int(), v.int(), at), {}),
        (ValueError, (q[..., :32], k[..., :32], v[..., :32], at), {}), (ValueError, (q[:, :3], k, v, at), {}),
        (ValueError, (q, k, v[:9], at), {}), (ValueError, (q, k[:9], v[:9], at), {}),
        (ValueError, (q, k[:, :, ::2], v[:, :, ::2], at), {}), (ValueError, (q[:, :0], k, v, at), {}),
        (ValueError, (q, k[:, :0], v[:, :0], at), {}), (TypeError, (q, k, v, at.long()), {}),
        (TypeError, (q, k, v, at.cpu()), {}), (ValueError, (q, k, v, at[:0]), {}), (ValueError, (q, k, v, at[None]), {}),
        (ValueError, (q, k, v, torch.zeros(4, dtype=torch.int32, device=DEV)[::2]), {}),
        (ValueError, (q, k, v, at, offsets([5, 5])), {}), (TypeError, (q, k, v, at, at.float()), {}),
        (ValueError, (q, k, v, at, at, at), {}), (TypeError, (q, k, v, at, at, at[1:].long()), {}),
        (ValueError, (q, k, v, at), dict(out=q[:9])), (ValueError, (q, k, v, at), dict(out=torch.empty_like(q).half())),
        (ValueError, (q, k, v, at), dict(out=torch.empty(10, 4, 64, dtype=q.dtype))),
        (ValueError, (q, k, v, at), dict(out=torch.empty(10, 4, 128, device=DEV, dtype=q.dtype)[..., ::2])),
        (ValueError, (q, k, v, at), dict(out=q)), (ValueError, (q, k, v, at), dict(scale=0.0)),
        (ValueError, (q, k, v, at), dict(scale=-1.0)), (ValueError, (q, k, v, at), dict(scale=float("nan"))),
        (ValueError, (q, k, v, at), dict(out=torch.empty(1, 4, 64, device=DEV, dtype=q.dtype).expand(10, 4, 64))),
        (ValueError, (torch.empty(10, 4, 66, device=DEV, dtype=q.dtype)[..., 1:65], k, v, at), {}),
        (ValueError, (torch.empty(10, 4, 68, device=DEV, dtype=q.dtype)[..., :64], k, v, at), {}),
    ]
    for i, (error, args, more) in enumerate(calls):
        with pytest.raises(error):
            pa.packed_attention(*args, **more)
            pytest.fail(f"call {i} was taken")

"""Attention over packed sequences on MI355X (`hb_packed_attention`): prompts or clips of different lengths one after the
other in one tensor, causal or not, with heads of queries that share heads of keys, and new tokens over the keys of their
sequences. It is the plain softmax attention of the non-differential model (`DiTConfig.differential = False`,
sa3jax/dit.py:150-176) and of transformers beside the denoiser; `dense_attention`, `band_attention` and
`cross_attention` are the differential ones. Tensors are torch tensors on a ROCm device; work is enqueued on torch's
current stream.
"""
from __future__ import annotations

import torch

from hummingbird_amd import _lib
from hummingbird_amd.dense_attention import _require_gpu, dtype_code
from hummingbird_amd.elementwise import _new

SUPPORTED_HEAD_DIMS = (64, 128)


def _heads(t: torch.Tensor, name: str) -> None:
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name} must be (tokens, heads, head_dim) with unit stride on its last axis, got "
                         f"{tuple(t.shape)} with strides {t.stride()}")


def _table(t: torch.Tensor, name: str, entries: int, device: torch.device) -> torch.Tensor:
    """A table of int32 entries on `device`."""
    if t.dtype is not torch.int32 or t.device != device:
        raise TypeError(f"{name} must be int32 on {device}, got {t.dtype} on {t.device}")
    if t.shape != (entries,) or not t.is_contiguous():
        raise ValueError(f"{name} must have {entries} entries next to each other, got {tuple(t.shape)}")
    return t


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     key_offsets: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None, *,
                     causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """`q` `(T, H, D)`, `k` and `v` `(Tk, G, D)` -> `(T, H, D)` in `q.dtype`: softmax attention of N sequences, query head
    h over key head `h // (H // G)`.

    Sequence i has the queries `offsets[i]` to `offsets[i + 1]` and the keys `key_offsets[i]` to `key_offsets[i + 1]`
    (`offsets` where not given), the first `key_lengths[i]` of them where that is given: the keys of a cache whose slots
    have room behind them. `offsets` and `key_offsets` are `(N + 1,)` ascending, `key_lengths` `(N,)`, int32 on the device;
    they are read there, so nothing waits for them and a captured call follows their contents. With `causal` query a of
    lq sees the keys b <= a + lk - lq of lk: the queries are the last of the keys' tokens (one new token: lq = 1).
    A query that sees no key, or only keys of a score of minus infinity, gives zeros; keys that a query does not see take no
    part in it, whatever their values.
    `scale` (default `D ** -0.5`) is positive. bf16 and half inputs multiply on their own type's cores, with the probabilities
    rounded to that type; statistics and sums are fp32, and fp32 inputs are fp32 throughout.

    `out`, if given, is written and returned, its tokens of no sequence (before `offsets[0]`, from `offsets[N]` on) left as
    they are; a new output has zeros there. D 64 or 128; bf16, half or fp32; any strides of tokens and
    heads that are multiples of 16 bytes (of k's and v's tokens up to 2^23 values), every tensor 16-byte aligned."""
    if not q.is_cuda:
        _require_gpu(q, "q")
    dtype, dev = q.dtype, q.device
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    if k.dtype is not dtype or v.dtype is not dtype or k.device != dev or v.device != dev:
        raise TypeError(f"k and v must be {dtype} on {dev} as q, got {k.dtype} on {k.device} and {v.dtype} on {v.device}")
    code = dtype_code(dtype)
    tokens, heads, dim = q.shape
    keys, kv_heads, _ = k.shape
    (qt, qh, q1), (kt, kh, k1), (vt, vh, v1) = q.stride(), k.stride(), v.stride()
    if q1 != 1 or k1 != 1 or v1 != 1:
        _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    if dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"packed_attention needs head_dim in {SUPPORTED_HEAD_DIMS} (head_dim={dim})")
    if k.shape != v.shape or k.shape[2] != dim or kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"k and v must be (Tk, G, D) with H a multiple of G, got q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"offsets must be (N + 1,), got {tuple(offsets.shape)}")
    count = offsets.shape[0] - 1
    _table(offsets, "offsets", count + 1, dev)
    if key_offsets is None:
        if keys < tokens:
            raise ValueError(f"k and v have {keys} tokens, q {tokens}: without key_offsets they share q's sequences")
        key_offsets = offsets
    else:
        _table(key_offsets, "key_offsets", count + 1, dev)
    if key_lengths is not None:
        _table(key_lengths, "key_lengths", count, dev)
    fresh = out is None
    if fresh:
        out = _new((tokens, heads, dim), dtype, dev)
    else:
        _heads(out, "out")
        if out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
            raise ValueError(f"out must be {tuple(q.shape)} of {q.dtype} on {dev}, got {tuple(out.shape)} {out.dtype} on "
                             f"{out.device}")
    if tokens == 0 or count == 0:
        return out.zero_() if fresh else out
    lib = _lib.load()
    need = int(lib.hb_packed_workspace_size(code, tokens, keys, count, heads, kv_heads, dim))
    workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    ot, oh, _ = out.stride()
    _lib.launch(lib.hb_packed_attention, "packed_attention", dev, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(),
                vt, vh, code, offsets.data_ptr(), key_offsets.data_ptr(),
                0 if key_lengths is None else key_lengths.data_ptr(), int(bool(causal)),
                float(dim ** -0.5 if scale is None else scale), out.data_ptr(), ot, oh, int(fresh), tokens, keys, count,
                heads, kv_heads, dim, workspace.data_ptr() if need else 0, need)
    return out

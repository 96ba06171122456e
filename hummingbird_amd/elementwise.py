"""The elementwise steps of a SAME-L decoder block (`hb_dyt`, `hb_glu`) and of a DiT block (`hb_rms_modulate`,
`hb_gated_residual`) on MI355X: the `attention="hip"` counterparts of `same_l._dyt` followed by the block's cast to
the compute dtype (sa3jax/same_l.py:58-69, 191-192), of the GLU gate of `same_l._feed_forward`
(sa3jax/same_l.py:172-183; the DiT's SwiGLU, sa3jax/dit.py:218-221, is the same gate), and of the DiT block's
norms, adaLN modulations and residuals (sa3jax/dit.py:224-251). The `_q8` forms of the latter (`quantize_rows`,
`rms_modulate_q8`, `residual_rms_q8`, `glu_q8`) end in 8-bit rows, the inputs of `projection.linear_q8`, and the `_mx4`
forms in microscaled 4-bit rows, those of `projection.linear_mx4`. Tensors are torch tensors on a ROCm device; work is
enqueued on torch's current stream.
"""
from __future__ import annotations

import torch

from hummingbird_amd import _lib
from hummingbird_amd._derived import f32_vector
from hummingbird_amd.band_attention import pack_dyt
from hummingbird_amd.dense_attention import _f32_vector, _require_gpu, dtype_code


def _rows(t: torch.Tensor, name: str) -> tuple[int, int]:
    """(rows, row stride in elements) of a tensor whose leading axes flatten onto equally spaced rows: contiguous,
    a column slice of a wider contiguous tensor, or one token of each of its sequences."""
    if t.dim() < 1 or t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride on its last axis")
    axes = [(size, st) for size, st in zip(t.shape[:-1], t.stride()[:-1]) if size != 1]  # (one row's stride is any)
    stride = step = axes[-1][1] if axes else t.shape[-1]
    for size, st in reversed(axes):
        if st != step:
            raise ValueError(f"{name}'s leading axes must flatten onto rows of one stride")
        step *= size
    return t.numel() // t.shape[-1], stride


def dyt(x: torch.Tensor, norm: dict) -> torch.Tensor:
    """`cast(gamma * tanh(alpha * x) + beta)` over the last axis, computed in fp32 and returned in `x.dtype`
    (reference: same_l._dyt + `.astype(dtype.compute)`, same_l.py:58-69, 191-192). `norm` holds the DyT params
    `{alpha: scalar, gamma: (C,), beta: (C,)}`."""
    _require_gpu(x, "x")
    channels = x.shape[-1]
    params = pack_dyt(norm, channels, x.device)
    rows, stride = _rows(x, "x")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stream = _lib.current_stream(x.device)
    _lib.check(_lib.load().hb_dyt(stream, x.data_ptr(), dtype_code(x.dtype), stride, params.data_ptr(), out.data_ptr(),
                                  channels, rows, channels), "dyt")
    return out


def glu(proj: torch.Tensor, sinusoidal: bool, bias: torch.Tensor | None = None) -> torch.Tensor:
    """`value * act(gate)` for `[value | gate]` = the two halves of the last axis of the glu_proj output
    (reference: same_l._feed_forward, same_l.py:172-183); act = SiLU, or sin(pi * gate) when `sinusoidal`.
    `bias` (2F), if given, is the glu_proj layer's bias and `proj` the bare matmul: the bias is added in the
    compute dtype first (same_l._linear), in the same pass."""
    _require_gpu(proj, "proj")
    width = proj.shape[-1]
    if width % 2:
        raise ValueError(f"the glu_proj output width {width} is not even")
    inner = width // 2
    rows, stride = _rows(proj, "proj")
    bias_p = 0
    if bias is not None:
        bias = f32_vector(bias, proj.device)
        if bias.numel() != width:
            raise ValueError(f"bias must have {width} elements")
        bias_p = bias.data_ptr()
    out = torch.empty((*proj.shape[:-1], inner), dtype=proj.dtype, device=proj.device)
    stream = _lib.current_stream(proj.device)
    _lib.check(_lib.load().hb_glu(stream, proj.data_ptr(), dtype_code(proj.dtype), stride, bias_p,
                                  int(bool(sinusoidal)), out.data_ptr(), inner, rows, inner), "glu")
    return out


def residual_dyt(h: torch.Tensor, x: torch.Tensor, bias: torch.Tensor | None = None,
                 norm: dict | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """`(h + (x + bias), cast(DyT(h + (x + bias))))` in one pass: a residual add of the SAME-L block (reference:
    same_l._block, same_l.py:191-192) after the projection's bias add (same_l._linear), each sum held in the compute
    dtype, and with `norm` (DyT params) the DyT of the sum cast back, the next GEMM's input. `x` is the bare
    projection output; `bias` (C values) may be None. Without `norm` the second result is None."""
    _require_gpu(h, "h")
    if h.shape != x.shape or h.dtype != x.dtype or h.device != x.device:
        raise ValueError(f"h {tuple(h.shape)} {h.dtype} {h.device} and x {tuple(x.shape)} {x.dtype} {x.device} must match")
    channels = h.shape[-1]
    rows, hs = _rows(h, "h")
    _, xs = _rows(x, "x")
    bias_p = 0
    if bias is not None:
        bias = f32_vector(bias, h.device)
        if bias.numel() != channels:
            raise ValueError(f"bias must have {channels} elements")
        bias_p = bias.data_ptr()
    params = pack_dyt(norm, channels, h.device) if norm is not None else None
    out_h = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    out_y = torch.empty(h.shape, dtype=h.dtype, device=h.device) if norm is not None else None
    stream = _lib.current_stream(h.device)
    _lib.check(_lib.load().hb_residual_dyt(stream, h.data_ptr(), dtype_code(h.dtype), hs, x.data_ptr(), xs, bias_p,
                                           params.data_ptr() if params is not None else 0, out_h.data_ptr(),
                                           out_y.data_ptr() if out_y is not None else 0, channels, rows, channels),
               "residual_dyt")
    return out_h, out_y


def _per_batch(t: torch.Tensor | None, batch: int, channels: int, x: torch.Tensor, name: str):
    """(pointer, batch stride) of a `(B, C)` (or `(B, 1, C)`) per-batch row tensor of `x`'s dtype and device, possibly a
    view into a wider row (the adaLN chunks of `(B, 6 E)`); (0, 0) for None."""
    if t is None:
        return 0, 0
    if t.device != x.device:
        raise ValueError(f"{name} must be on {x.device}, got {t.device}")
    if t.dtype != x.dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")
    t2 = t.reshape(t.shape[0], t.shape[-1]) if t.dim() == 3 and t.shape[1] == 1 else t
    if t2.dim() != 2 or tuple(t2.shape) != (batch, channels) or t2.stride(-1) != 1:
        raise ValueError(f"{name} must be (B, C) = ({batch}, {channels}) with unit stride on C, got {tuple(t.shape)}")
    return t2.data_ptr(), (t2.stride(0) if batch > 1 else channels)


def _channel_vector(t: torch.Tensor | None, channels: int, x: torch.Tensor, name: str) -> int:
    """The pointer of `channels` values of `x`'s dtype and device next to each other, 0 for None. (A `(C, 1)` slice of a
    wider tensor has C values and a last stride of 1, but is not that.)"""
    if t is None:
        return 0
    if t.device != x.device:
        raise ValueError(f"{name} must be on {x.device}, got {t.device}")
    if t.dtype != x.dtype or t.numel() != channels or not t.is_contiguous():
        raise ValueError(f"{name} must be ({channels},) of {x.dtype} with unit stride")
    return t.data_ptr()


def _memory_tokens(memory: int, length: int) -> int:
    """The first token that takes `local`, of `length`: as a C int, which holds no more than 31 bits."""
    if memory < 0:
        raise ValueError(f"memory must be >= 0, got {memory}")
    return min(int(memory), length)


def rms_modulate(x: torch.Tensor, weight: torch.Tensor, eps: float, scale: torch.Tensor | None = None,
                 shift: torch.Tensor | None = None) -> torch.Tensor:
    """The DiT block norm on `(B, L, C)`: `cast(x * rsqrt(mean(x^2) + eps) * weight)` with an fp32 island
    (sa3jax/dit.py:44-57), then with `scale` / `shift` `(B, C)` the adaLN modulation `* (1 + scale) + shift`
    (sa3jax/dit.py:231-233, 246-247), each step in `x.dtype`. One pass (`hb_rms_modulate`)."""
    _require_gpu(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be (B, L, C), got {tuple(x.shape)}")
    batch, length, channels = x.shape
    rows, stride = _rows(x, "x")
    w = weight.to(device=x.device, dtype=torch.float32).contiguous().reshape(-1)
    if w.numel() != channels:
        raise ValueError(f"weight must have {channels} elements")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _per_batch(scale, batch, channels, x, "scale")
    hp, ms2 = _per_batch(shift, batch, channels, x, "shift")
    if scale is not None and ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stream = _lib.current_stream(x.device)
    _lib.check(_lib.load().hb_rms_modulate(stream, x.data_ptr(), dtype_code(x.dtype), stride, w.data_ptr(), float(eps),
                                           sp, hp, ms, length, out.data_ptr(), channels, rows, channels),
               "rms_modulate")
    return out


def gated_residual(h: torch.Tensor, x: torch.Tensor, gate: torch.Tensor | None = None,
                   x_bias: torch.Tensor | None = None, local: torch.Tensor | None = None,
                   memory: int = 0) -> torch.Tensor:
    """`h + (x + x_bias) * sigmoid(1 - gate)` on `(B, L, C)` (sa3jax/dit.py:234, 249-251), or `h + x` without
    `gate`, then `+ local` on the tokens at or past `memory` (sa3jax/dit.py:237-241); each step in `h.dtype`.
    `gate` is `(B, C)`, `x_bias` and `local` `(C,)`. One pass (`hb_gated_residual`)."""
    _require_gpu(h, "h")
    if h.dim() != 3 or x.shape != h.shape or x.dtype != h.dtype or x.device != h.device:
        raise ValueError(f"h and x must be (B, L, C) of one shape, dtype and device, got {tuple(h.shape)} {h.dtype} "
                         f"{h.device}, {tuple(x.shape)} {x.dtype} {x.device}")
    batch, length, channels = h.shape
    _, hs = _rows(h, "h")
    rows, xs = _rows(x, "x")
    gp, gs = _per_batch(gate, batch, channels, h, "gate")
    bp, lp = _channel_vector(x_bias, channels, h, "x_bias"), _channel_vector(local, channels, h, "local")
    out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    stream = _lib.current_stream(h.device)
    _lib.check(_lib.load().hb_gated_residual(stream, h.data_ptr(), dtype_code(h.dtype), hs, x.data_ptr(), xs,
                                             bp, gp, gs, lp, _memory_tokens(memory, length), length, out.data_ptr(),
                                             channels, rows, channels), "gated_residual")
    return out


def residual_rms(h: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float,
                 gate: torch.Tensor | None = None, x_bias: torch.Tensor | None = None,
                 local: torch.Tensor | None = None, memory: int = 0, scale: torch.Tensor | None = None,
                 shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`gated_residual(h, x, gate, x_bias, local, memory)` and then `rms_modulate` of its result with `weight`, `eps`,
    `scale`, `shift`, in one pass per row (`hb_residual_rms`; rows of at most 2048 values):
    returns `(h', norm(h'))`, the same values as the two calls. A DiT block's residuals each feed the next norm
    (sa3jax/dit.py:234-236, 237-247, 249-251 into the next block's 231-233)."""
    _require_gpu(h, "h")
    if h.dim() != 3 or x.shape != h.shape or x.dtype != h.dtype or x.device != h.device:
        raise ValueError(f"h and x must be (B, L, C) of one shape, dtype and device, got {tuple(h.shape)} {h.dtype} "
                         f"{h.device}, {tuple(x.shape)} {x.dtype} {x.device}")
    batch, length, channels = h.shape
    _, hs = _rows(h, "h")
    rows, xs = _rows(x, "x")
    gp, gs = _per_batch(gate, batch, channels, h, "gate")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _per_batch(scale, batch, channels, h, "scale")
    hp, ms2 = _per_batch(shift, batch, channels, h, "shift")
    if scale is not None and ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    w = weight.to(device=h.device, dtype=torch.float32).contiguous().reshape(-1)
    if w.numel() != channels:
        raise ValueError(f"weight must have {channels} elements")
    bp, lp = _channel_vector(x_bias, channels, h, "x_bias"), _channel_vector(local, channels, h, "local")
    out_h = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    out_y = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    stream = _lib.current_stream(h.device)
    _lib.check(_lib.load().hb_residual_rms(stream, h.data_ptr(), dtype_code(h.dtype), hs, x.data_ptr(), xs,
                                           bp, gp, gs, lp, _memory_tokens(memory, length), w.data_ptr(), float(eps), sp,
                                           hp, ms, length, out_h.data_ptr(), out_y.data_ptr(), channels, rows, channels),
               "residual_rms")
    return out_h, out_y


def residual_rms_supported(dtype: torch.dtype, channels: int) -> bool:
    """Whether `residual_rms` takes rows of `channels` values of `dtype` (held in registers)."""
    return channels <= 2048 and channels % (8 if dtype in (torch.bfloat16, torch.float16) else 4) == 0


# ---------------------------------------------------------------------------------------------------------------
# 8-bit rows: e4m3 values `q` with one fp32 scale `s` per row, standing for q * s.

Q8_DTYPE = torch.float8_e4m3fn
Q8_MAX_WIDTH = 16384  # values of a row, held in registers


def _layout(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, row stride, row width) of a device tensor of rows, as `_rows` with a quick way out for contiguous ones."""
    if not t.is_cuda:
        _require_gpu(t, name)
    width = t.shape[-1] if t.dim() else 0
    if not 0 < width < 1 << 31:
        raise ValueError(f"{name} must have rows of 1 to 2^31 - 1 values, got {tuple(t.shape)}")
    rows, stride = (t.numel() // width, width) if t.is_contiguous() else _rows(t, name)
    if rows >= 1 << 31:
        raise ValueError(f"{name} must have fewer than 2^31 rows, got {tuple(t.shape)}")
    return rows, stride, width


def _batch_rows(t: torch.Tensor | None, batch: int, channels: int, x: torch.Tensor, name: str) -> tuple[int, int]:
    """`_per_batch` of a tensor on `x`'s device, with a quick way out for None and for what is as it should be."""
    if t is None:
        return 0, 0
    if t.device != x.device:
        raise ValueError(f"{name} must be on {x.device}, got {t.device}")
    if t.dtype is x.dtype and t.shape == (batch, channels):
        step, unit = t.stride()
        if unit == 1:
            return t.data_ptr(), (step if batch > 1 else channels)
    return _per_batch(t, batch, channels, x, name)


def _f32_channels(t: torch.Tensor, channels: int, device: torch.device, name: str) -> torch.Tensor:
    """`t` as `channels` fp32 values on `device`, where it must live (converted where it is not fp32)."""
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype is torch.float32 and t.shape == (channels,) and t.is_contiguous():
        return t
    t = _f32_vector(t, device)
    if t.numel() != channels:
        raise ValueError(f"{name} must have {channels} elements")
    return t


def _new(shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """`torch.empty(shape, ...)`; with the strides spelt out it takes 1.3 us instead of 1.6 to 2.3."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 3:
        return torch.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _q8_out(like: torch.Tensor, width: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Contiguous 8-bit rows of `width` values and their scales, for the rows of `like`."""
    rows = tuple(like.shape[:-1])
    return _new((*rows, width), Q8_DTYPE, like.device), _new(rows, torch.float32, like.device)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """`x` `(..., C)` as 8-bit rows: `(q, s)`, q `(..., C)` e4m3 and s `(...)` fp32 with `s = max(max|x| / 448, 2^-100)`
    and `q = e4m3(x / s)`, in one pass (`hb_quant_rows`). A row with a NaN or an infinity stands for NaNs. C a multiple
    of 8 (fp32: 4), at most `Q8_MAX_WIDTH`."""
    rows, stride, channels = _layout(x, "x")
    code = dtype_code(x.dtype)
    q, s = _q8_out(x, channels)
    _lib.launch(_lib.load().hb_quant_rows, "quantize_rows", x.device, x.data_ptr(), code, stride, q.data_ptr(),
                channels, s.data_ptr(), rows, channels)
    return q, s


def rms_modulate_q8(x: torch.Tensor, weight: torch.Tensor, eps: float, scale: torch.Tensor | None = None,
                    shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`rms_modulate(x, weight, eps, scale, shift)` on `(B, L, C)` in fp32 throughout, as 8-bit rows `(q, s)` (see
    `quantize_rows`), in one pass (`hb_rms_modulate_q8`)."""
    rows, stride, channels = _layout(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be (B, L, C), got {tuple(x.shape)}")
    code = dtype_code(x.dtype)
    batch, length, _ = x.shape
    w = _f32_channels(weight, channels, x.device, "weight")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _batch_rows(scale, batch, channels, x, "scale")
    hp, ms2 = _batch_rows(shift, batch, channels, x, "shift")
    if ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    q, s = _q8_out(x, channels)
    _lib.launch(_lib.load().hb_rms_modulate_q8, "rms_modulate_q8", x.device, x.data_ptr(), code, stride, w.data_ptr(),
                float(eps), sp, hp, ms, length, q.data_ptr(), channels, s.data_ptr(), rows, channels)
    return q, s


def residual_rms_q8(h: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float,
                    gate: torch.Tensor | None = None, x_bias: torch.Tensor | None = None,
                    local: torch.Tensor | None = None, memory: int = 0, scale: torch.Tensor | None = None,
                    shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`residual_rms(h, x, weight, eps, gate, x_bias, local, memory, scale, shift)` with the norm as 8-bit rows, in one
    pass (`hb_residual_rms_q8`): `(h', q, s)`, h' in `h.dtype`, `(q, s)` as `quantize_rows` gives them. Both are
    rounded once, from fp32: the norm reads h' before its rounding."""
    rows, hs, channels = _layout(h, "h")
    if h.dim() != 3 or x.shape != h.shape or x.dtype != h.dtype or x.device != h.device:
        raise ValueError(f"h and x must be (B, L, C) of one shape, dtype and device, got {tuple(h.shape)} {h.dtype} "
                         f"{h.device}, {tuple(x.shape)} {x.dtype} {x.device}")
    xs = channels if x.is_contiguous() else _layout(x, "x")[1]
    code = dtype_code(h.dtype)
    batch, length, _ = h.shape
    gp, gs = _batch_rows(gate, batch, channels, h, "gate")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _batch_rows(scale, batch, channels, h, "scale")
    hp, ms2 = _batch_rows(shift, batch, channels, h, "shift")
    if ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    w = _f32_channels(weight, channels, h.device, "weight")
    bp, lp = _channel_vector(x_bias, channels, h, "x_bias"), _channel_vector(local, channels, h, "local")
    out_h = _new((batch, length, channels), h.dtype, h.device)
    q, s = _q8_out(h, channels)
    _lib.launch(_lib.load().hb_residual_rms_q8, "residual_rms_q8", h.device, h.data_ptr(), code, hs, x.data_ptr(), xs,
                bp, gp, gs, lp, _memory_tokens(memory, length), w.data_ptr(), float(eps), sp, hp, ms, length,
                out_h.data_ptr(), channels, q.data_ptr(), channels, s.data_ptr(), rows, channels)
    return out_h, q, s


def glu_q8(proj: torch.Tensor, bias: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`value * silu(gate)` for `[value | gate]` = the two halves of the last axis of `proj (+ bias)`, in fp32, as
    8-bit rows `(q, s)` (see `quantize_rows`), in one pass (`hb_glu_q8`): the DiT's SwiGLU (sa3jax/dit.py:218-221).
    `bias` `(2F,)` is the glu_proj layer's where `proj` is the bare product."""
    rows, stride, width = _layout(proj, "proj")
    code = dtype_code(proj.dtype)
    if width % 2:
        raise ValueError(f"the glu_proj output width {width} is not even")
    inner = width // 2
    bp = 0
    if bias is not None:
        bias = _f32_channels(bias, width, proj.device, "bias")
        bp = bias.data_ptr()
    q, s = _q8_out(proj, inner)
    _lib.launch(_lib.load().hb_glu_q8, "glu_q8", proj.device, proj.data_ptr(), code, stride, bp, q.data_ptr(), inner,
                s.data_ptr(), rows, inner)
    return q, s


# ---------------------------------------------------------------------------------------------------------------
# Microscaled 4-bit rows: e2m1 codes `q`, two per byte (the low nibble the even column), with one e8m0 scale byte `s` per
# 32 columns, standing for the code's value times 2^(s - 127): the form of `projection.quantize_q4`'s weights.

MX4_GROUP = 32  # columns that share a scale


def _mx4_out(like: torch.Tensor, width: int, what: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Contiguous 4-bit rows of `width` values and their scale bytes, for the rows of `like`."""
    if width % MX4_GROUP:
        raise ValueError(f"{what}: rows must be a multiple of {MX4_GROUP} values, got {width}")
    rows = tuple(like.shape[:-1])
    return (_new((*rows, width // 2), torch.uint8, like.device),
            _new((*rows, width // MX4_GROUP), torch.uint8, like.device))


def quantize_rows_mx4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """`x` `(..., C)` as 4-bit rows `(q, s)`, q `(..., C / 2)` and s `(..., C / 32)`, both uint8, in one pass
    (`hb_quant_rows_mx4`): per group of 32 columns the least s, from 8 on, that brings the largest magnitude to 6 or below
    (127 for a group of zeros), and e2m1(x 2^(127 - s)), to nearest, ties to the even code. A group with a NaN or an
    infinity stands for NaNs (s = 255). C a multiple of 32."""
    rows, stride, channels = _layout(x, "x")
    code = dtype_code(x.dtype)
    q, s = _mx4_out(x, channels, "quantize_rows_mx4")
    _lib.launch(_lib.load().hb_quant_rows_mx4, "quantize_rows_mx4", x.device, x.data_ptr(), code, stride, q.data_ptr(),
                channels // 2, s.data_ptr(), channels // MX4_GROUP, rows, channels)
    return q, s


def rms_modulate_mx4(x: torch.Tensor, weight: torch.Tensor, eps: float, scale: torch.Tensor | None = None,
                     shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`rms_modulate(x, weight, eps, scale, shift)` on `(B, L, C)` in fp32 throughout, as 4-bit rows `(q, s)` (see
    `quantize_rows_mx4`), in one pass (`hb_rms_modulate_mx4`). C a multiple of 32, at most `Q8_MAX_WIDTH`."""
    rows, stride, channels = _layout(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be (B, L, C), got {tuple(x.shape)}")
    code = dtype_code(x.dtype)
    batch, length, _ = x.shape
    w = _f32_channels(weight, channels, x.device, "weight")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _batch_rows(scale, batch, channels, x, "scale")
    hp, ms2 = _batch_rows(shift, batch, channels, x, "shift")
    if ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    q, s = _mx4_out(x, channels, "rms_modulate_mx4")
    _lib.launch(_lib.load().hb_rms_modulate_mx4, "rms_modulate_mx4", x.device, x.data_ptr(), code, stride, w.data_ptr(),
                float(eps), sp, hp, ms, length, q.data_ptr(), channels // 2, s.data_ptr(), channels // MX4_GROUP, rows,
                channels)
    return q, s


def residual_rms_mx4(h: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float,
                     gate: torch.Tensor | None = None, x_bias: torch.Tensor | None = None,
                     local: torch.Tensor | None = None, memory: int = 0, scale: torch.Tensor | None = None,
                     shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`residual_rms(h, x, weight, eps, gate, x_bias, local, memory, scale, shift)` with the norm as 4-bit rows, in one
    pass (`hb_residual_rms_mx4`): `(h', q, s)`, h' in `h.dtype`, `(q, s)` as `quantize_rows_mx4` gives them. Both are
    rounded once, from fp32: the norm reads h' before its rounding. C a multiple of 32, at most `Q8_MAX_WIDTH`."""
    rows, hs, channels = _layout(h, "h")
    if h.dim() != 3 or x.shape != h.shape or x.dtype != h.dtype or x.device != h.device:
        raise ValueError(f"h and x must be (B, L, C) of one shape, dtype and device, got {tuple(h.shape)} {h.dtype} "
                         f"{h.device}, {tuple(x.shape)} {x.dtype} {x.device}")
    xs = channels if x.is_contiguous() else _layout(x, "x")[1]
    code = dtype_code(h.dtype)
    batch, length, _ = h.shape
    gp, gs = _batch_rows(gate, batch, channels, h, "gate")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift are given together or not at all")
    sp, ms = _batch_rows(scale, batch, channels, h, "scale")
    hp, ms2 = _batch_rows(shift, batch, channels, h, "shift")
    if ms != ms2:
        raise ValueError("scale and shift must share their batch stride")
    w = _f32_channels(weight, channels, h.device, "weight")
    bp, lp = _channel_vector(x_bias, channels, h, "x_bias"), _channel_vector(local, channels, h, "local")
    q, s = _mx4_out(h, channels, "residual_rms_mx4")
    out_h = _new((batch, length, channels), h.dtype, h.device)
    _lib.launch(_lib.load().hb_residual_rms_mx4, "residual_rms_mx4", h.device, h.data_ptr(), code, hs, x.data_ptr(), xs,
                bp, gp, gs, lp, _memory_tokens(memory, length), w.data_ptr(), float(eps), sp, hp, ms, length,
                out_h.data_ptr(), channels, q.data_ptr(), channels // 2, s.data_ptr(), channels // MX4_GROUP, rows,
                channels)
    return out_h, q, s


def glu_mx4(proj: torch.Tensor, bias: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`value * silu(gate)` for `[value | gate]` = the two halves of the last axis of `proj (+ bias)`, in fp32, as
    4-bit rows `(q, s)` (see `quantize_rows_mx4`), in one pass (`hb_glu_mx4`): the DiT's SwiGLU
    (sa3jax/dit.py:218-221). `bias` `(2F,)` is the glu_proj layer's where `proj` is the bare product. F a multiple of 32."""
    rows, stride, width = _layout(proj, "proj")
    code = dtype_code(proj.dtype)
    if width % 2:
        raise ValueError(f"the glu_proj output width {width} is not even")
    inner = width // 2
    bp = 0
    if bias is not None:
        bias = _f32_channels(bias, width, proj.device, "bias")
        bp = bias.data_ptr()
    q, s = _mx4_out(proj, inner, "glu_mx4")
    _lib.launch(_lib.load().hb_glu_mx4, "glu_mx4", proj.device, proj.data_ptr(), code, stride, bp, q.data_ptr(),
                inner // 2, s.data_ptr(), inner // MX4_GROUP, rows, inner)
    return q, s

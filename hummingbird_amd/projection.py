"""The projections around the attention kernels on MI355X. The DiT self-attention's: `to_qkv` with the dense
kernel's key preparation in its epilogue, and `to_out` (reference: sa3jax/dit.py:190 and 195, `_linear` without
bias). The SAME-L block's: `glu_proj` with the GLU in its epilogue, and `to_out` / `proj_out` with the residual add
and the next DyT in theirs (reference: sa3jax/same_l.py:161, 181-184, 191-192).

`qkv_projection` runs `hb_dit_qkv_proj`: one matrix-core GEMM `h @ W_qkv^T` that never stores `qkv`; it writes the
queries as rows `[q | q_diff]` and the prepared keys and values (RMSNorm, RoPE, value mask) into the attention
workspace. `attend_projected` runs the attention against them (`hb_dense_attend_qq`), and `linear` is `x @ W^T`
(`hb_proj`). Together they compute what `h @ W_qkv^T -> dense_attention -> @ W_o^T` computes, in the same cast points.

`linear_q8` multiplies 8-bit rows (`elementwise.quantize_rows` and its kin) with 8-bit weights (`hb_proj_q8`), and
`linear_q4` a few rows with 4-bit weights (`quantize_q4`, `hb_proj_q4`).
"""
from __future__ import annotations

import torch

from hummingbird_amd import _lib
from hummingbird_amd._derived import f32_vector
from hummingbird_amd.band_attention import pack_dyt
from hummingbird_amd.dense_attention import _f32, _f32_vector, _require_gpu, dtype_code
from hummingbird_amd.elementwise import _f32_channels, _layout, _new, _rows

FUSED_DTYPES = (torch.bfloat16, torch.float16)


def fused_supported(dtype: torch.dtype, num_heads: int, head_dim: int, embed_dim: int, half: int) -> bool:
    """Whether `qkv_projection` takes this geometry (bf16 or half, head_dim 64, heads a multiple of 4, model width a
    multiple of 64, rotary half-width a multiple of 8 up to 32)."""
    return (dtype in FUSED_DTYPES and head_dim == 64 and num_heads % 4 == 0 and embed_dim % 64 == 0
            and 0 <= half <= 32 and half % 8 == 0)


def linear_supported(dtype: torch.dtype, out_features: int, in_features: int) -> bool:
    """Whether `linear` takes this product (bf16 or half, out_features a multiple of 256, in_features of 64)."""
    return dtype in FUSED_DTYPES and out_features % 256 == 0 and in_features % 64 == 0 and out_features > 0


def qkv_projection(h: torch.Tensor, w_qkv: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor | None,
                   sin: torch.Tensor | None, mask: torch.Tensor | None, num_heads: int, head_dim: int, half: int,
                   eps: float, workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`(B, L, E)` block input -> (`qq` `(B, L, 2 H D)` = `[q | q_diff]` of `h @ W_qkv^T`, the attention workspace
    holding the prepared k, k_diff and v). `w_qkv` is the layer weight `(5 H D, E)` (out x in); `cos`, `sin`, `mask`
    come from `dense_attention.tables`. Raises ValueError for geometries outside `fused_supported`."""
    _require_gpu(h, "h")
    if h.dim() != 3:
        raise ValueError(f"h must be (B, L, E), got {tuple(h.shape)}")
    batch, length, width = h.shape
    if not fused_supported(h.dtype, num_heads, head_dim, width, half):
        raise ValueError(f"the fused projection does not take dtype {h.dtype}, H={num_heads}, D={head_dim}, E={width}, "
                         f"half={half}")
    dev = h.device
    w = w_qkv.to(device=dev, dtype=h.dtype)
    if tuple(w.shape) != (5 * num_heads * head_dim, width):
        raise ValueError(f"w_qkv must be (5*H*D, E) = ({5 * num_heads * head_dim}, {width}), got {tuple(w.shape)}")
    _, hs = _rows(h, "h")
    _, ws_ = _rows(w, "w_qkv")
    kw = _f32_vector(k_weight, dev)
    cos_p = sin_p = 0
    if half > 0:
        cos, sin = _f32(cos, dev), _f32(sin, dev)
        cos_p, sin_p = cos.data_ptr(), sin.data_ptr()
    mask_p = 0
    if mask is not None:
        mask = _f32(mask, dev)
        mask_p = mask.data_ptr()
    lib = _lib.load()
    code = dtype_code(h.dtype)
    need = int(lib.hb_dense_workspace_size(code, batch, length, num_heads, head_dim))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < need or workspace.device != dev:
        raise ValueError(f"workspace must hold {need} bytes on {dev}")
    qq = torch.empty((batch, length, 2 * num_heads * head_dim), dtype=h.dtype, device=dev)
    stream = _lib.current_stream(dev)
    _lib.check(lib.hb_dit_qkv_proj(stream, h.data_ptr(), code, hs, w.data_ptr(), ws_, width, kw.data_ptr(), cos_p,
                                   sin_p, half, mask_p, qq.data_ptr(), batch, length, num_heads, head_dim, float(eps),
                                   workspace.data_ptr(), workspace.numel() * workspace.element_size()), "qkv_projection")
    return qq, workspace


def attend_projected(qq: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor | None,
                     sin: torch.Tensor | None, num_heads: int, head_dim: int, half: int, eps: float,
                     workspace: torch.Tensor, lam: torch.Tensor | None = None) -> torch.Tensor:
    """The differential self-attention of `dense_attention` for queries in `qq` (from `qkv_projection`) against the
    workspace it filled: `(B, L, H D)` in `qq.dtype`."""
    _require_gpu(qq, "qq")
    batch, length, _ = qq.shape
    dev = qq.device
    _, rs = _rows(qq, "qq")
    qw, kw = _f32_vector(q_weight, dev), _f32_vector(k_weight, dev)
    cos_p = sin_p = 0
    if half > 0:
        cos, sin = _f32(cos, dev), _f32(sin, dev)
        cos_p, sin_p = cos.data_ptr(), sin.data_ptr()
    lam_p = 0
    if lam is not None:
        lam = _f32_vector(lam, dev)
        lam_p = lam.data_ptr()
    out = torch.empty((batch, length, num_heads * head_dim), dtype=qq.dtype, device=dev)
    lib = _lib.load()
    stream = _lib.current_stream(dev)
    _lib.check(lib.hb_dense_attend_qq(stream, qq.data_ptr(), dtype_code(qq.dtype), rs, qw.data_ptr(), kw.data_ptr(),
                                      cos_p, sin_p, half, lam_p, out.data_ptr(), batch, length, num_heads, head_dim,
                                      float(eps), workspace.data_ptr(), workspace.numel() * workspace.element_size()),
               "attend_projected")
    return out


def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """`x @ W^T` on the matrix cores (the reference's `_linear` without bias), fp32 accumulation, one rounding to
    `x.dtype`. `weight` is `(F, K)` (out x in) with F a multiple of 256 and K of 64."""
    _require_gpu(x, "x")
    if x.dtype not in FUSED_DTYPES:
        raise TypeError(f"linear takes bfloat16 or float16 inputs, got {x.dtype}")
    w = weight.to(device=x.device, dtype=x.dtype)
    n, xs = _rows(x, "x")
    _, wstride = _rows(w, "weight")
    f, k = w.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, weight {k}")
    out = torch.empty((*x.shape[:-1], f), dtype=x.dtype, device=x.device)
    stream = _lib.current_stream(x.device)
    _lib.check(_lib.load().hb_proj(stream, x.data_ptr(), dtype_code(x.dtype), xs, w.data_ptr(), wstride, out.data_ptr(),
                                   f, n, k, f), "linear")
    return out


def glu_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, sinusoidal: bool) -> torch.Tensor:
    """`value * act(gate)` of `[value | gate] = x @ W^T (+ bias)` without storing the product (`hb_proj_glu`): the
    SAME-L feed-forward's `glu_proj` and GLU (reference: same_l._feed_forward, same_l.py:181-183), with the cast
    points of `elementwise.glu` on the rounded product. `weight` is the layer's `(2F, K)` (out x in), `bias` `(2F,)`
    or None; act = sin(pi * gate) when `sinusoidal`, else SiLU. F a multiple of 128, K of 64."""
    _require_gpu(x, "x")
    if x.dtype not in FUSED_DTYPES:
        raise TypeError(f"glu_linear takes bfloat16 or float16 inputs, got {x.dtype}")
    w = weight.to(device=x.device, dtype=x.dtype)
    n, xs = _rows(x, "x")
    _, wstride = _rows(w, "weight")
    f2, k = w.shape
    if x.shape[-1] != k or f2 % 2:
        raise ValueError(f"x has {x.shape[-1]} columns, weight is {tuple(w.shape)}")
    f = f2 // 2
    bias_p = 0
    if bias is not None:
        bias = f32_vector(bias, x.device)
        if bias.numel() != f2:
            raise ValueError(f"bias must have {f2} elements")
        bias_p = bias.data_ptr()
    out = torch.empty((*x.shape[:-1], f), dtype=x.dtype, device=x.device)
    stream = _lib.current_stream(x.device)
    _lib.check(_lib.load().hb_proj_glu(stream, x.data_ptr(), dtype_code(x.dtype), xs, w.data_ptr(), wstride, bias_p,
                                       int(bool(sinusoidal)), out.data_ptr(), f, n, k, f), "glu_linear")
    return out


def residual_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, h: torch.Tensor,
                    norm: dict | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """`(h + (x @ W^T + bias), cast(DyT(...)))` with the residual add and the next DyT in the GEMM's epilogue
    (`hb_proj_residual`): the SAME-L `to_out` / `proj_out` and the residual add after them (reference:
    same_l._block, same_l.py:191-192, and same_l._linear), with the cast points of `elementwise.residual_dyt` on the
    rounded product. `weight` is `(F, K)` (out x in), `bias` `(F,)` or None, `h` the residual `(..., F)`; without
    `norm` (DyT params) the second result is None. F a multiple of 256, K of 64."""
    _require_gpu(x, "x")
    if x.dtype not in FUSED_DTYPES:
        raise TypeError(f"residual_linear takes bfloat16 or float16 inputs, got {x.dtype}")
    w = weight.to(device=x.device, dtype=x.dtype)
    n, xs = _rows(x, "x")
    _, wstride = _rows(w, "weight")
    f, k = w.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, weight {k}")
    if h.shape[:-1] != x.shape[:-1] or h.shape[-1] != f or h.dtype != x.dtype or h.device != x.device:
        raise ValueError(f"h must be {(*x.shape[:-1], f)} of {x.dtype} on {x.device}, got {tuple(h.shape)} {h.dtype} on "
                         f"{h.device}")
    _, hs = _rows(h, "h")
    bias_p = 0
    if bias is not None:
        bias = f32_vector(bias, x.device)
        if bias.numel() != f:
            raise ValueError(f"bias must have {f} elements")
        bias_p = bias.data_ptr()
    params = pack_dyt(norm, f, x.device) if norm is not None else None
    out_h = torch.empty(h.shape, dtype=x.dtype, device=x.device)
    out_y = torch.empty(h.shape, dtype=x.dtype, device=x.device) if norm is not None else None
    stream = _lib.current_stream(x.device)
    _lib.check(_lib.load().hb_proj_residual(stream, x.data_ptr(), dtype_code(x.dtype), xs, w.data_ptr(), wstride,
                                            bias_p, h.data_ptr(), hs, params.data_ptr() if params is not None else 0,
                                            out_h.data_ptr(), out_y.data_ptr() if out_y is not None else 0, f, n, k,
                                            f), "residual_linear")
    return out_h, out_y


def same_l_supported(dtype: torch.dtype, dim: int, ff_inner: int, qkv_width: int) -> bool:
    """Whether the SAME-L block's projections take the fused kernels: bf16 or half, model width a multiple of 256,
    feed-forward width a multiple of 256 (its GLU half of 128 and proj_out's reduction of 64), the to_qkv width a
    multiple of 256."""
    return (dtype in FUSED_DTYPES and dim % 256 == 0 and ff_inner % 256 == 0 and qkv_width % 256 == 0 and dim > 0
            and ff_inner > 0)


def linear_q8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """`(x * x_scale) @ (weight * weight_scale)^T (+ bias)` of 8-bit rows on the matrix cores (`hb_proj_q8`): `x`
    `(..., K)` e4m3 with `x_scale` `(...)` fp32, `weight` `(F, K)` e4m3 with `weight_scale` `(F,)` fp32 (both as
    `elementwise.quantize_rows` gives them), `bias` `(F,)`; the sum, the scales and the bias in fp32, one rounding to
    `dtype` (bf16, half or fp32). K a multiple of 16; up to 2^21 rows and 2^21 features."""
    n, xs, k = _layout(x, "x")
    dev = x.device
    if x.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise TypeError(f"linear_q8 takes float8_e4m3fn rows and weights, got {x.dtype} and {weight.dtype}")
    if x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise TypeError(f"the scales must be float32, got {x_scale.dtype} and {weight_scale.dtype}")
    if weight.dim() != 2 or weight.shape[1] != k:
        raise ValueError(f"x must be (..., K) and weight (F, K), got {tuple(x.shape)} and {tuple(weight.shape)}")
    code = dtype_code(dtype)
    f, ws, _ = _layout(weight, "weight")
    if weight.device != dev or x_scale.device != dev or weight_scale.device != dev:
        raise ValueError(f"weight and the scales must be on {dev}, got {weight.device}, {x_scale.device}, "
                         f"{weight_scale.device}")
    if x_scale.shape != x.shape[:-1]:
        raise ValueError(f"x_scale must be {tuple(x.shape[:-1])}, got {tuple(x_scale.shape)}")
    if weight_scale.shape != (f,):
        raise ValueError(f"weight_scale must be ({f},), got {tuple(weight_scale.shape)}")
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()  # (a slice's scales: copied)
    bp = 0
    if bias is not None:
        bias = _f32_channels(bias, f, dev, "bias")
        bp = bias.data_ptr()
    out = _new((*x.shape[:-1], f), dtype, dev)
    _lib.launch(_lib.load().hb_proj_q8, "linear_q8", dev, x.data_ptr(), xs, x_scale.data_ptr(), weight.data_ptr(), ws,
                weight_scale.data_ptr(), bp, out.data_ptr(), code, f, n, k, f)
    return out


Q4_GROUP = 32  # columns that share a scale
_E2M1_MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6


def quantize_q4(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """`(F, K)` weights as `(codes (F, K / 2) uint8, scales (F, K / 32) uint8)` for `linear_q4`: e2m1 codes, two per
    byte (the low nibble the even column), and per group of 32 columns the e8m0 scale 2^(s - 127), the least power of
    two that brings the group's largest magnitude to 6 or below, with s at least 8. Magnitudes round to the nearest, ties
    to the even code. Done once per weight, in torch operations on the weight's device. K a multiple of 32; magnitudes
    must be at most 6 * 2^123 (s = 250)."""
    if weight.dim() != 2 or weight.shape[1] % Q4_GROUP or weight.numel() == 0:
        raise ValueError(f"weight must be (F, K) with K a multiple of {Q4_GROUP}, got {tuple(weight.shape)}")
    f, k = weight.shape
    w = weight.to(torch.float32).reshape(f, k // Q4_GROUP, Q4_GROUP)
    amax = w.abs().amax(dim=-1)
    if not bool((amax <= 6 * 2.0 ** 123).all()):
        raise ValueError("quantize_q4 needs finite weights of magnitudes up to 6 * 2^123")
    mant, exp = torch.frexp(amax)  # amax = mant 2^exp, mant in [0.5, 1): above 6 2^(exp - 3) when mant > 0.75
    e = torch.where(mant > 0.75, exp - 2, exp - 3)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(8 - 127, 250 - 127)
    v = w * torch.exp2(-e[..., None].to(torch.float32))
    mag = v.abs()
    middles = torch.tensor(_E2M1_MIDDLES, device=weight.device)
    below, upto = torch.bucketize(mag, middles), torch.bucketize(mag, middles, right=True)
    code = torch.where(below % 2 == 0, below, upto)  # on a middle the two differ: the even one
    code = (code + 8 * torch.signbit(v)).reshape(f, k)
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8).contiguous(), (e + 127).to(torch.uint8).contiguous()


def linear_q4(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
              silu: bool = False) -> torch.Tensor:
    """`act(x @ W^T (+ bias))` for few rows `x` `(..., K)` and 4-bit weights (`hb_proj_q4`): `weight` `(F, K / 2)` and
    `weight_scale` `(F, K / 32)`, both uint8, as `quantize_q4` gives them (any bytes are taken: under a scale of 253 or 254
    weights of 2^128 and more are infinite, 255 makes its group NaN); `bias` `(F,)`; act = SiLU with `silu`. x
    keeps all of its bits (bf16, half or fp32, there those above 2^-133), the sum, bias and activation are fp32, rounded
    once to `x.dtype`. It serves the layers that see one row per batch entry; up to 2^16 rows are taken."""
    n, xs, k = _layout(x, "x")
    dev = x.device
    code = dtype_code(x.dtype)
    if weight.dtype != torch.uint8 or weight_scale.dtype != torch.uint8:
        raise TypeError(f"linear_q4 takes uint8 codes and scales, got {weight.dtype} and {weight_scale.dtype}")
    if weight.dim() != 2 or k != 2 * weight.shape[1] or k % Q4_GROUP:
        raise ValueError(f"x must be (..., K) and weight (F, K / 2), K a multiple of {Q4_GROUP}, got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    if weight.device != dev or weight_scale.device != dev:
        raise ValueError(f"weight and weight_scale must be on {dev}, got {weight.device} and {weight_scale.device}")
    f, ws, _ = _layout(weight, "weight")
    if weight_scale.shape != (f, k // Q4_GROUP):
        raise ValueError(f"weight_scale must be (F, K / {Q4_GROUP}) = ({f}, {k // Q4_GROUP}), got "
                         f"{tuple(weight_scale.shape)}")
    _, ss, _ = _layout(weight_scale, "weight_scale")
    bp = 0
    if bias is not None:
        bias = _f32_channels(bias, f, dev, "bias")
        bp = bias.data_ptr()
    out = _new((*x.shape[:-1], f), x.dtype, dev)
    _lib.launch(_lib.load().hb_proj_q4, "linear_q4", dev, x.data_ptr(), code, xs, weight.data_ptr(), ws,
                weight_scale.data_ptr(), ss, bp, int(bool(silu)), out.data_ptr(), f, n, k, f)
    return out

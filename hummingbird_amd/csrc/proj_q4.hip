// Products of few rows with 4-bit weights, for gfx950 (MI355X): the denoiser's conditioning layers (timestep embedding,
// global condition, adaLN rows; sa3jax/dit.py:37-41, 340-361), whose cost is the weights' bytes.
//
//   out[n, f] = act(sum_k x[n, k] e2m1(w[f, k]) 2^(ws[f, k / 32] - 127) + bias[f]),
//
// w two e2m1 codes per byte (low nibble: the even column), ws one e8m0 scale per 32 columns (the OCP MX format), so a
// weight is 4.25 bits. The weights go from memory to the matrix cores through one conversion: v_cvt_scalef32_pk_bf16_fp4
// turns two codes and their scale into two exact bf16 values. x keeps all of its bits as well: a half row is two bf16
// rows, an fp32 row three (each the next 8 bits of the value, the remainders exact), and those rows are further columns
// of the same MFMA, whose 16 columns a single row leaves empty anyway. Sums are fp32.
//
// One workgroup computes 16 features for all columns; its waves take the 128-column chunks of K in turns and their
// partial sums are added in the waves' order. On v_mfma_f32_16x16x32_bf16 a lane holds 8 consecutive columns of feature
// (or row) lane % 16; which 8 is free as long as both operands agree, so quarter lane / 16 takes columns 32 q + 8 i of
// the chunk in MFMA i: a lane's 16 bytes of codes are then one scale group, read in one load.
#include "api.h"
#include "common.h"

namespace hb {
namespace q4 {

constexpr int kChunk = 128;  // columns of K per step: four groups
constexpr int kGroup = 32;
constexpr int kMaxWaves = 16;

struct Args {
  const void* x;  // (N, K), row stride xs elements
  int64_t xs;
  const uint8_t* w;  // (F, K / 2), row stride w_rs bytes
  int64_t w_rs;
  const uint8_t* ws;  // (F, K / 32), row stride ws_rs bytes
  int64_t ws_rs;
  const float* bias;  // F values or null
  int silu;
  void* out;  // (N, F), row stride os elements
  int64_t os;
  int N, K, F;
};

// Rows of x as bf16 rows whose sum they are: P pieces, each the leading 8 bits of what the earlier ones leave
// (truncated, so that no piece overflows and every remainder is exact). An infinity or NaN is the first piece alone.
template <typename T>
struct Pieces;
template <>
struct Pieces<uint16_t> {  // bf16
  static constexpr int P = 1;
  __device__ static u32x4 load8(const uint16_t* p, int) { return ld16(p); }
};
__device__ __forceinline__ float piece_of(float x, int piece) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
  if (!finite) return piece == 0 ? round_bf16(x) : 0.f;
  if (piece == 0) return hi;
  const float r = x - hi, mid = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  return piece == 1 ? mid : r - mid;
}
__device__ __forceinline__ u32x4 pack_pieces(const float (&x)[8], int piece) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = piece_of(x[j], piece);
  return pack8(v);  // each value is a bf16 already
}
template <>
struct Pieces<_Float16> {
  static constexpr int P = 2;
  __device__ static u32x4 load8(const _Float16* p, int piece) {
    float x[8];
    F16Io::unpack8(ld16(p), x);
    return pack_pieces(x, piece);
  }
};
template <>
struct Pieces<float> {
  static constexpr int P = 3;
  __device__ static u32x4 load8(const float* p, int piece) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
    }
    return pack_pieces(x, piece);
  }
};

template <typename T>
__device__ __forceinline__ T cast_out(float v);
template <>
__device__ __forceinline__ uint16_t cast_out<uint16_t>(float v) { return f2bf(v); }
template <>
__device__ __forceinline__ _Float16 cast_out<_Float16>(float v) { return static_cast<_Float16>(v); }
template <>
__device__ __forceinline__ float cast_out<float>(float v) { return v; }

// The 8 codes of `c` as bf16, times the scale.
__device__ __forceinline__ u32x4 dequant8(uint32_t c, float scale) {
  u32x4 v;
  v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
  v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
  v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
  v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  return v;
}

__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// CT tiles of 16 columns (rows of x times pieces) starting at column blockIdx.y * 16 CT.
template <typename T, int CT>
__global__ __launch_bounds__(64 * kMaxWaves) void q4_kernel(const Args a) {
  constexpr int P = Pieces<T>::P;
  __shared__ float part[kMaxWaves][CT][16][17];  // [wave][tile][feature][column]
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4, wave = wave_id(), waves = blockDim.x >> 6;
  const int f0 = blockIdx.x * 16, f = f0 + lr < a.F ? f0 + lr : a.F - 1;  // features past the end are not stored
  const int rows = 16 * CT / P;  // whole rows per workgroup
  const int row0 = blockIdx.y * rows;
  const uint8_t* wrow = a.w + f * a.w_rs;
  const uint8_t* srow = a.ws + f * a.ws_rs;
  const T* xrow[CT];
  int piece[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int col = 16 * t + lr, r = col / P, row = row0 + r;
    piece[t] = col - r * P;
    xrow[t] = r < rows && row < a.N ? static_cast<const T*>(a.x) + row * a.xs : nullptr;
  }
  f32x4 acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = (a.K + kChunk - 1) / kChunk;
  for (int c = wave; c < chunks; c += waves) {
    const int k0 = c * kChunk + kGroup * lq;  // this lane's group
    const bool in = k0 < a.K;                 // K is a multiple of the group
    u32x4 code = u32x4{0, 0, 0, 0};
    float scale = 1.f;
    if (in) {
      code = ld16(wrow + (k0 >> 1));
      scale = __uint_as_float(static_cast<uint32_t>(srow[k0 / kGroup]) << 23);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 wv = dequant8(code[i], scale);
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        u32x4 xv = u32x4{0, 0, 0, 0};
        if (in && xrow[t]) xv = Pieces<T>::load8(xrow[t] + k0 + 8 * i, piece[t]);
        acc[t] = mfma_16x16x32(wv, xv, acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < CT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][4 * lq + i][lr] = acc[t][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * rows; e += blockDim.x) {
    const int r = e >> 4, fo = e & 15, row = row0 + r;
    if (row >= a.N || f0 + fo >= a.F) continue;
    float v = 0.f;
    for (int p = 0; p < P; ++p) {
      const int col = r * P + p;
      for (int w = 0; w < waves; ++w) v += part[w][col >> 4][fo][col & 15];
    }
    if (a.bias) v += a.bias[f0 + fo];
    if (a.silu) v = v * __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * v));
    static_cast<T*>(a.out)[row * a.os + f0 + fo] = cast_out<T>(v);
  }
}

template <typename T>
void launch(hipStream_t stream, const Args& a) {
  const int cols = a.N * Pieces<T>::P;  // N <= 2^20
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const dim3 block(64 * (chunks < kMaxWaves ? chunks : kMaxWaves));
  const unsigned fx = static_cast<unsigned>((a.F + 15) / 16);
  auto grid = [&](int ct) {
    const int rows = 16 * ct / Pieces<T>::P;
    return dim3(fx, static_cast<unsigned>((a.N + rows - 1) / rows));
  };
  if (cols <= 16 / Pieces<T>::P * Pieces<T>::P) hipLaunchKernelGGL((q4_kernel<T, 1>), grid(1), block, 0, stream, a);
  else hipLaunchKernelGGL((q4_kernel<T, 2>), grid(2), block, 0, stream, a);
}

}  // namespace q4
}  // namespace hb

using namespace hb;

extern "C" int hb_proj_q4(hipStream_t stream, const void* x, int dtype, int64_t x_row_stride, const void* w,
                          int64_t w_row_stride, const void* w_scale, int64_t w_scale_row_stride, const float* bias,
                          int silu, void* out, int64_t out_row_stride, int N, int K, int F) {
  clear_error();
  const char* what = "proj_q4";
  if (dtype != HB_BF16 && dtype != HB_F32 && dtype != HB_F16)
    return fail(HB_ERR_DTYPE, "%s: dtype %d is not HB_BF16 (0), HB_F32 (1) or HB_F16 (2)", what, dtype);
  if (N < 1 || N > (1 << 16) || F < 1 || F > (1 << 28) || K < q4::kGroup || K > (1 << 28) || K % q4::kGroup)
    return fail(HB_ERR_SHAPE, "%s needs 1 <= N <= 2^16, 1 <= F <= 2^28 and K a multiple of %d (N=%d, K=%d, F=%d)", what,
                q4::kGroup, N, K, F);
  if (!x || !w || !w_scale || !out) return fail(HB_ERR_NULL, "%s: x, w, w_scale and out must be non-NULL", what);
  const int es = dtype == HB_F32 ? 4 : 2, vec = 16 / es;
  auto misaligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (misaligned(x, 16) || x_row_stride < K || x_row_stride % vec)
    return fail(HB_ERR_STRIDE, "%s: x must be 16-byte aligned with a row stride >= K and a multiple of %d", what, vec);
  if (misaligned(w, 16) || w_row_stride < K / 2 || w_row_stride % 16)
    return fail(HB_ERR_STRIDE, "%s: w must be 16-byte aligned with a row stride >= K / 2 bytes, a multiple of 16", what);
  if (w_scale_row_stride < K / q4::kGroup)
    return fail(HB_ERR_STRIDE, "%s: w_scale's row stride must be >= K / %d", what, q4::kGroup);
  if (misaligned(out, es) || out_row_stride < F)
    return fail(HB_ERR_STRIDE, "%s: out must be aligned to its elements with a row stride >= F", what);
  int st;
  if ((st = check_extent(what, "x", N, x_row_stride, K)) || (st = check_extent(what, "w", F, w_row_stride, K / 2)) ||
      (st = check_extent(what, "w_scale", F, w_scale_row_stride, K / q4::kGroup)) ||
      (st = check_extent(what, "out", N, out_row_stride, F)))
    return st;
  const int64_t ob = rows_bytes(N, out_row_stride, F, es);
  if ((st = check_disjoint(what, "out", out, ob, "x", x, rows_bytes(N, x_row_stride, K, es))) ||
      (st = check_disjoint(what, "out", out, ob, "w", w, rows_bytes(F, w_row_stride, K / 2, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "w_scale", w_scale,
                           rows_bytes(F, w_scale_row_stride, K / q4::kGroup, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "bias", bias, static_cast<int64_t>(F) * 4)))
    return st;
  const q4::Args a = {x, x_row_stride, static_cast<const uint8_t*>(w), w_row_stride,
                      static_cast<const uint8_t*>(w_scale), w_scale_row_stride, bias, silu ? 1 : 0, out,
                      out_row_stride, N, K, F};
  if (dtype == HB_BF16) q4::launch<uint16_t>(stream, a);
  else if (dtype == HB_F16) q4::launch<_Float16>(stream, a);
  else q4::launch<float>(stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return HB_OK;
}

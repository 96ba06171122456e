// Products of 8-bit rows and 8-bit weights, for gfx950 (MI355X): the denoiser's projections (sa3jax/dit.py:31-34) on
// the e4m3 matrix cores, whose rate is twice the bf16 one's.
//
//   out[m, f] = (sum_k x[m, k] w[f, k]) sx[m] sw[f] + bias[f],   x, w e4m3, sx, sw, bias and the sum fp32,
//
// rounded once to the output type. C^T = W x^T as in the 16-bit projections: a lane of a 32x32 MFMA's result holds one
// row of x and 16 features, four of them consecutive.
//
// The e4m3 matrix cores (v_mfma_f32_32x32x64_f8f6f4, and v_mfma_f32_32x32x16_fp8_fp8 alike) do not add in full fp32:
// within 16 products, what lies more than 13 bits below the largest is dropped. On rows of normal values that is an
// error of 1.5e-5 of the result, whatever K, where rounding to half costs 2.1e-4 and to bf16 1.7e-3: taken for 16-bit
// outputs. For fp32 outputs the codes are converted to bf16 (exact) and multiplied on the bf16 cores, whose sums are
// fp32 (error 5e-8 at K = 1536, that of an fp32 product).
#include <type_traits>

#include "api.h"
#include "common.h"

namespace hb {
namespace q8 {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Args {
  const uint8_t* x;  // (M, K), row stride x_rs bytes
  int64_t x_rs;
  const float* sx;
  const uint8_t* w;  // (F, K), row stride w_rs bytes
  int64_t w_rs;
  const float* sw;
  const float* bias;  // F values or null
  void* out;          // (M, F), row stride os elements
  int64_t os;
  int64_t M;
  int K, F;
};

// e4m3 x e4m3 without block scales, fp32 accumulation.
__device__ __forceinline__ f32x16 mfma_32x32x64(i32x8 a, i32x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ T cast_out(float v);
template <>
__device__ __forceinline__ uint16_t cast_out<uint16_t>(float v) { return f2bf(v); }
template <>
__device__ __forceinline__ _Float16 cast_out<_Float16>(float v) { return static_cast<_Float16>(v); }
template <>
__device__ __forceinline__ float cast_out<float>(float v) { return v; }

// 32 columns of a row from column k on, zeros from column K on (K a multiple of 16).
__device__ __forceinline__ i32x8 load32(const uint8_t* row, int k, int K) {
  u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (k < K) lo = ld16(row + k);
  if (k + 16 < K) hi = ld16(row + k + 16);
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

// 8 e4m3 codes as bf16, exact.
__device__ __forceinline__ u32x4 widen8(u32x2 c) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, false));
    v[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, true));
  }
  return v;
}

// One 32-feature x 32-row tile per wave, a workgroup 64 x 64.
template <typename T>
__global__ __launch_bounds__(256) void q8_kernel(const Args a) {
  const int lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5, wave = wave_id();
  const int f0 = blockIdx.x * 64 + 32 * (wave & 1);
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64 + 32 * (wave >> 1);
  const int f = f0 + lr < a.F ? f0 + lr : a.F - 1;            // rows past an end read a real one;
  const int64_t m = m0 + lr < a.M ? m0 + lr : a.M - 1;        // their results are not stored
  const uint8_t* wrow = a.w + f * a.w_rs;
  const uint8_t* xrow = a.x + m * a.x_rs;
  f32x16 acc = {};
  if constexpr (std::is_same<T, float>::value) {
    auto load8 = [](const uint8_t* p) { return *reinterpret_cast<const u32x2*>(p); };
    for (int k = 8 * lh; k < a.K; k += 16)
      acc = mfma_bf16_32x32x16(widen8(load8(wrow + k)), widen8(load8(xrow + k)), acc);
  } else {
    for (int k = 0; k < a.K; k += 64)
      acc = mfma_32x32x64(load32(wrow, k + 32 * lh, a.K), load32(xrow, k + 32 * lh, a.K), acc);
  }
  if (m0 + lr >= a.M) return;
  const float sx = a.sx[m];
  T* orow = static_cast<T*>(a.out) + m * a.os;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int fo = f0 + 8 * (i >> 2) + 4 * lh + (i & 3);
    if (fo < a.F) {
      float v = (acc[i] * sx) * a.sw[fo];
      if (a.bias) v += a.bias[fo];
      orow[fo] = cast_out<T>(v);
    }
  }
}

template <typename T>
void launch(hipStream_t stream, const Args& a) {
  const dim3 grid(static_cast<unsigned>((a.F + 63) / 64), static_cast<unsigned>((a.M + 63) / 64));
  hipLaunchKernelGGL((q8_kernel<T>), grid, dim3(256), 0, stream, a);
}

}  // namespace q8
}  // namespace hb

using namespace hb;

extern "C" int hb_proj_q8(hipStream_t stream, const void* x, int64_t x_row_stride, const float* x_scale, const void* w,
                          int64_t w_row_stride, const float* w_scale, const float* bias, void* out, int out_dtype,
                          int64_t out_row_stride, int64_t M, int K, int F) {
  clear_error();
  const char* what = "proj_q8";
  if (out_dtype != HB_BF16 && out_dtype != HB_F32 && out_dtype != HB_F16)
    return fail(HB_ERR_DTYPE, "%s: dtype %d is not HB_BF16 (0), HB_F32 (1) or HB_F16 (2)", what, out_dtype);
  if (M < 1 || M > (1 << 21) || F < 1 || F > (1 << 21) || K < 16 || K > (1 << 24) || K % 16)
    return fail(HB_ERR_SHAPE, "%s needs 1 <= M, F <= 2^21 and K a multiple of 16 up to 2^24 (M=%lld, K=%d, F=%d)", what,
                static_cast<long long>(M), K, F);
  if (!x || !x_scale || !w || !w_scale || !out)
    return fail(HB_ERR_NULL, "%s: x, x_scale, w, w_scale and out must be non-NULL", what);
  const int es = out_dtype == HB_F32 ? 4 : 2;
  auto misaligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (misaligned(x, 16) || x_row_stride < K || x_row_stride % 16)
    return fail(HB_ERR_STRIDE, "%s: x must be 16-byte aligned with a row stride >= K, a multiple of 16", what);
  if (misaligned(w, 16) || w_row_stride < K || w_row_stride % 16)
    return fail(HB_ERR_STRIDE, "%s: w must be 16-byte aligned with a row stride >= K, a multiple of 16", what);
  if (misaligned(out, es) || out_row_stride < F)
    return fail(HB_ERR_STRIDE, "%s: out must be aligned to its elements with a row stride >= F", what);
  int st;
  if ((st = check_extent(what, "x", M, x_row_stride, K)) || (st = check_extent(what, "w", F, w_row_stride, K)) ||
      (st = check_extent(what, "out", M, out_row_stride, F)))
    return st;
  const int64_t ob = rows_bytes(M, out_row_stride, F, es);
  if ((st = check_disjoint(what, "out", out, ob, "x", x, rows_bytes(M, x_row_stride, K, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "w", w, rows_bytes(F, w_row_stride, K, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "x_scale", x_scale, M * 4)) ||
      (st = check_disjoint(what, "out", out, ob, "w_scale", w_scale, static_cast<int64_t>(F) * 4)) ||
      (st = check_disjoint(what, "out", out, ob, "bias", bias, static_cast<int64_t>(F) * 4)))
    return st;
  const q8::Args a = {static_cast<const uint8_t*>(x), x_row_stride, x_scale, static_cast<const uint8_t*>(w),
                      w_row_stride, w_scale, bias, out, out_row_stride, M, K, F};
  if (out_dtype == HB_BF16) q8::launch<uint16_t>(stream, a);
  else if (out_dtype == HB_F16) q8::launch<_Float16>(stream, a);
  else q8::launch<float>(stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return HB_OK;
}

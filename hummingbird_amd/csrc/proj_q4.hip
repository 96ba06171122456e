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
// A workgroup computes 16 to 64 features for up to 64 columns; its waves take the 128-column chunks of K in turns and
// their partial sums are added in the waves' order. On v_mfma_f32_16x16x32_bf16 a lane holds 8 consecutive columns of
// feature (or row) lane % 16; which 8 is free as long as both operands agree, so quarter lane / 16 takes columns
// 32 q + 8 i of the chunk in MFMA i: a lane's 16 bytes of codes are then one scale group, read in one load.
#include "api.h"
#include "common.h"

namespace hb {
namespace q4 {

constexpr int kGroup = 32;
constexpr int kChunk = 128;  // columns of K per step of a wave: a group for each quarter of the lanes
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

// Rows of x as bf16 rows whose sum they are: P pieces, each the leading 8 bits of what the earlier ones leave (truncated,
// so that no piece overflows and every remainder is exact; a bf16 value has no bits below 2^-133). Piece p is x after p
// times y -= y & 0xffff0000, cut to its upper half: a lane holds the masks of its piece, zero past it. An infinity or NaN
// leaves NaNs in the later pieces; what counts then is the first one's sum (see the end of the kernel).
template <typename T>
struct Pieces;
template <>
struct Pieces<uint16_t> {  // bf16
  static constexpr int P = 1;
  __device__ explicit Pieces(int) {}
  __device__ u32x4 load8(const uint16_t* p) const { return ld16(p); }
};
// The upper halves of eight fp32 values.
__device__ __forceinline__ u32x4 upper8(const float (&x)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
  return v;
}
// y - (y & mask): x itself where the mask is zero (a signalling NaN quieted, so that its upper half stays one).
__device__ __forceinline__ float without_upper(float y, uint32_t mask) {
  return __fsub_rn(y, __uint_as_float(__float_as_uint(y) & mask));
}
template <>
struct Pieces<_Float16> {
  static constexpr int P = 2;
  uint32_t m1;
  __device__ explicit Pieces(int piece) : m1(piece >= 1 ? 0xffff0000u : 0u) {}
  __device__ u32x4 load8(const _Float16* p) const {
    float x[8];
    F16Io::unpack8(ld16(p), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = without_upper(x[j], m1);
    return upper8(x);
  }
};
template <>
struct Pieces<float> {
  static constexpr int P = 3;
  uint32_t m1, m2;
  __device__ explicit Pieces(int piece)
      : m1(piece >= 1 ? 0xffff0000u : 0u), m2(piece >= 2 ? 0xffff0000u : 0u) {}
  __device__ u32x4 load8(const float* p) const {
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = without_upper(without_upper(v[j], m1), m2);
    }
    return upper8(x);
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

// A wave's sums over the chunks wave, wave + waves, ... for FT tiles of 16 features and CT tiles of 16 columns (rows of x
// times pieces), from feature 16 FT blockIdx.x and row `rows` blockIdx.y on. x is read once for the FT tiles.
// Waves of a workgroup: four per SIMD, and three or two where a wave has more tiles, whose registers then hold the loads of
// a whole chunk (bf16, 33 x 6144 -> 12288, nine tiles: 24.9 us with 12 waves, 27.4 with 8, 29.1 with 14; 64 x 4096 -> 6144,
// eight: 21.2, 21.5 and, with 16, 25.2). The sums of all waves, 1 KB for each tile of a wave, take at most 128 KB.
constexpr int max_waves(int tiles) { return tiles >= 12 ? 8 : tiles >= 6 ? 12 : kMaxWaves; }

template <typename T, int CT, int FT>
__global__ __launch_bounds__(64 * max_waves(CT * FT)) void q4_kernel(const Args a) {
  constexpr int P = Pieces<T>::P, R = 16 / P;  // whole rows per tile
  __shared__ __attribute__((aligned(16))) f32x4 sums[max_waves(CT * FT) * FT * CT * 64];  // [wave][FT][CT][64 lanes]
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4, wave = wave_id(), waves = blockDim.x >> 6;
  const int f0 = blockIdx.x * 16 * FT, row0 = blockIdx.y * R * CT;
  const uint8_t* wrow[FT];
  const uint8_t* srow[FT];
#pragma unroll
  for (int t = 0; t < FT; ++t) {
    const int f = f0 + 16 * t + lr < a.F ? f0 + 16 * t + lr : a.F - 1;  // features past the end are not stored
    wrow[t] = a.w + f * a.w_rs;
    srow[t] = a.ws + f * a.ws_rs;
  }
  const T* xrow[CT];
  const int r = lr / P, piece = lr - r * P;  // this lane's row in a tile and its piece
  const Pieces<T> pieces(piece);
#pragma unroll
  for (int u = 0; u < CT; ++u) {
    const int row = row0 + R * u + r;
    xrow[u] = r < R && row < a.N ? static_cast<const T*>(a.x) + row * a.xs : nullptr;
  }
  float bias[FT][4];  // of this lane's results, loaded here so that nothing waits for them at the end
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + 16 * t + 4 * lq + j;
      bias[t][j] = a.bias ? a.bias[f < a.F ? f : a.F - 1] : 0.f;
    }
  f32x4 acc[FT][CT];
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int u = 0; u < CT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = (a.K + kChunk - 1) / kChunk;
  for (int c = wave; c < chunks; c += waves) {
    const int k0 = c * kChunk + kGroup * lq;  // this lane's group
    u32x4 code[FT];
    uint32_t scale[FT];
#pragma unroll
    for (int t = 0; t < FT; ++t) {
      code[t] = u32x4{0, 0, 0, 0};
      scale[t] = 127;
      if (k0 < a.K) {  // K is a multiple of the group
        code[t] = ld16(wrow[t] + (k0 >> 1));
        scale[t] = srow[t][k0 / kGroup];
      }
    }
    u32x4 x[CT][4];
#pragma unroll
    for (int u = 0; u < CT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[u][i] = u32x4{0, 0, 0, 0};
        if (k0 < a.K && xrow[u]) x[u][i] = pieces.load8(xrow[u] + k0 + 8 * i);
      }
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 wv = dequant8(code[t][i], __uint_as_float(scale[t] << 23));
#pragma unroll
        for (int u = 0; u < CT; ++u) acc[t][u] = mfma_16x16x32(wv, x[u][i], acc[t][u]);
      }
  }
  if (waves > 1) {
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int u = 0; u < CT; ++u) sums[((wave * FT + t) * CT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
  }
  // Tile (t, u) is finished by wave (t CT + u) % waves: lane (lr, lq) has column lr and features 4 lq .. + 3.
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int u = 0; u < CT; ++u) {
      if ((t * CT + u) % waves != wave) continue;
      f32x4 v = acc[t][u];
      if (waves > 1) {
        v = sums[(t * CT + u) * 64 + lane];
        for (int i = 1; i < waves; ++i) {
          const f32x4 o = sums[((i * FT + t) * CT + u) * 64 + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += o[j];
        }
      }
      // A row's pieces are in P neighbouring columns: added where the row starts, unless the first sum is not finite.
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float mine = v[j];
        float sum = mine;
#pragma unroll
        for (int p = 1; p < P; ++p) sum += __shfl_down(mine, p, kWave);
        v[j] = __builtin_isfinite(mine) ? sum : mine;
      }
      const int row = row0 + R * u + r, f = f0 + 16 * t + 4 * lq;
      if (piece != 0 || r >= R || row >= a.N) continue;
      T y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float z = v[j] + bias[t][j];
        // off by up to (1.3 |z| + 6) 2^-24 of itself for negative z (the exponent is rounded first), zero below -87.3
        if (a.silu)
          z = z * __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z));
        y[j] = cast_out<T>(z);
      }
      T* o = static_cast<T*>(a.out) + row * a.os + f;
      if (f + 4 <= a.F) {
        __builtin_memcpy(o, y, sizeof(y));  // one store, of any alignment of the elements
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (f + j < a.F) o[j] = y[j];
      }
    }
}

template <typename T, int CT, int FT>
void launch_tiles(hipStream_t stream, const Args& a) {
  constexpr int R = 16 / Pieces<T>::P, kMax = max_waves(CT * FT);
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const dim3 grid(static_cast<unsigned>((a.F + 16 * FT - 1) / (16 * FT)),
                  static_cast<unsigned>((a.N + R * CT - 1) / (R * CT)));
  hipLaunchKernelGGL((q4_kernel<T, CT, FT>), grid, dim3(64 * (chunks < kMax ? chunks : kMax)), 0, stream, a);
}

template <typename T, int FT>
void launch_rows(hipStream_t stream, const Args& a) {
  constexpr int R = 16 / Pieces<T>::P;
  if (a.N <= R) launch_tiles<T, 1, FT>(stream, a);
  else if (a.N <= 2 * R) launch_tiles<T, 2, FT>(stream, a);
  else if (a.N <= 3 * R) launch_tiles<T, 3, FT>(stream, a);
  else launch_tiles<T, 4, FT>(stream, a);
}

// Tiles of features per wave: as few as let every workgroup run at once, one per CU, and four where none do. Fewer read x
// more often and leave a second, mostly empty round of workgroups; more leave CUs without work (bf16, kernel times with
// one, two, three and four: 1 x 6144 -> 12288 15.8, 17.8, 13.3 and 16.3 us, 1 x 1536 -> 9216 5.8, 6.1, 5.5 and 6.0,
// 33 x 6144 -> 12288, with as many waves as 128 KB of sums allow, 51, 41, 28 and 28; with one to three, 1 x 12288 -> 6144
// 18.8, 16.6 and 21.1). The conversions do not show: without them the kernel is no faster.
template <typename T>
void launch(hipStream_t stream, const Args& a) {
  constexpr int R = 16 / Pieces<T>::P;
  const int64_t tiles = static_cast<int64_t>((a.F + 15) / 16) * ((a.N + 4 * R - 1) / (4 * R)), cus = device_cus();
  if (tiles <= cus) launch_rows<T, 1>(stream, a);
  else if (tiles <= 2 * cus) launch_rows<T, 2>(stream, a);
  else if (tiles <= 3 * cus) launch_rows<T, 3>(stream, a);
  else launch_rows<T, 4>(stream, a);
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
  if (misaligned(bias, 4)) return fail(HB_ERR_STRIDE, "%s: bias must be 4-byte aligned", what);
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

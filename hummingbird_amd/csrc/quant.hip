// Rows as 8-bit values with one scale each, for gfx950 (MI355X): the inputs of the 8-bit projections.
//
//   quant_rows       y = x
//   rms_modulate_q8  y = x rsqrt(mean(x^2) + eps) w (1 + scale) + shift      (the DiT block norm, sa3jax/dit.py:44-57,
//                    231-233, 246-247; without scale and shift dit.py:236)
//   residual_rms_q8  h' = h + (x + bias) sigmoid(1 - gate) + local (dit.py:234, 237-241, 249-251), and y the norm of h'
//   glu_q8           y = value silu(gate), [value | gate] = proj + bias      (dit.py:218-221)
//
// followed by s = max(max_c |y| / 448, 2^-100) and q = e4m3(y / s): 448 is the largest e4m3 value, so the row's largest
// value meets it and no other saturates. The floor keeps 1 / s finite; a row of zeros gives zeros. A row that holds a
// NaN gets the scale NaN and one whose largest magnitude is infinite the scale inf, with finite values 0 and infinite
// ones NaN: every value the row stands for, q s, is then NaN.
//
// Everything between the inputs and the outputs is fp32, h' included: the norm reads the sum itself, not its value
// rounded to the compute dtype, so that each output is rounded once.
#include <cmath>

#include "api.h"
#include "common.h"

namespace hb {
namespace quant {

// V consecutive elements of a row as fp32.
template <typename T>
struct Vec;
template <>
struct Vec<uint16_t> {  // bf16
  static constexpr int N = 8;
  __device__ static void load(const uint16_t* p, float (&x)[8]) { unpack8(ld16(p), x); }
  __device__ static void store(uint16_t* p, const float (&x)[8]) { st16(p, pack8(x)); }
};
template <>
struct Vec<_Float16> {
  static constexpr int N = 8;
  __device__ static void load(const _Float16* p, float (&x)[8]) { F16Io::unpack8(ld16(p), x); }
  __device__ static void store(_Float16* p, const float (&x)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = F16Io::pack2(x[2 * i], x[2 * i + 1]);
    st16(p, v);
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void load(const float* p, float (&x)[4]) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
  __device__ static void store(float* p, const float (&x)[4]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  }
};

template <int N>
__device__ __forceinline__ void load_f32(const float* p, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4_align4*>(p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i + j] = v[j];
  }
}

// 1 / (1 + e^-u) with the hardware exponential and reciprocal. The exponent -log2(e) u is rounded before the exponential, so
// that for negative u the relative error grows with it: up to (1.3 |u| + 6) 2^-24 (6 2^-24 for positive u; 60 2^-24 at -40,
// far below an 8-bit code's step); where the value is below 2^-126 it is zero.
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * u)); }

// Four fp32 values as e4m3, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true));
}

constexpr int kMaxWaves = 16;
constexpr float kScaleFloor = 0x1p-100f;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
// `op` over a wave's 64 lanes, in one order, the result in every lane: pairs, quads, halves of 16 and rows of 16 by DPP,
// then the rows by lane swaps (against LDS permutations: residual_rms_q8 on 5168 x 1536 bf16 15.6 -> 14.6 us).
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, const F& op) {
  v = op(v, dpp<0xb1>(v));   // quad_perm 1, 0, 3, 2
  v = op(v, dpp<0x4e>(v));   // quad_perm 2, 3, 0, 1
  v = op(v, dpp<0x141>(v));  // row_half_mirror
  v = op(v, dpp<0x140>(v));  // row_mirror
  const u32x2 a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(a[0], a[1]);
  const u32x2 b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(b[0], b[1]);
}

// `op` over a row: of its wave, or (waves > 1) of the workgroup's waves in their order through `buf`, a slot per wave and
// free of reads on entry.
template <typename F>
__device__ __forceinline__ uint32_t row_reduce(uint32_t v, int waves, uint32_t* buf, const F& op) {
  v = wave_reduce(v, op);
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < waves; ++i) v = op(v, buf[i]);
  return v;
}
__device__ __forceinline__ float row_sum(float v, int waves, uint32_t* buf) {
  return __uint_as_float(row_reduce(__float_as_uint(v), waves, buf, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, int waves, uint32_t* buf) {
  return row_reduce(v, waves, buf, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// y / s, correctly rounded, for values |y| <= 448 s: y times the rounded reciprocal of s, off by an fp32 unit or two, and a
// step of the remainder, which is exact while s is at least 2^-90. Without the step one value in 2000 of bf16 rows (they
// often lie on a border between two codes) gets the wrong code; with the compiler's division instead the row operators
// take up to a third longer (quantize_rows on 5168 x 1536 bf16: 5.9 us without the step, 6.4 with it, 8.6 divided). The order
// of the operations keeps the sign of a zero.
struct Divisor {
  float s, inv;
  // (an infinite scale leaves finite values zero, and infinite ones NaN)
  __device__ explicit Divisor(float scale) : s(__builtin_isinf(scale) ? 0.f : scale), inv(__fdiv_rn(1.f, scale)) {}
  __device__ float quotient(float y) const {
    const float q = y * inv;
    return __fmaf_rn(-__fmaf_rn(q, s, -y), inv, q);
  }
};

// The row's scale and its values in 8 bits; y holds zeros past the row, `lane` of the row's `lanes`. Magnitudes are
// compared as their bits: a NaN's are above every number's, so it reaches the scale.
template <int V, int CH>
__device__ __forceinline__ void store_q8(float (&y)[CH][V], uint8_t* q, float* s, int C, int lane, int lanes,
                                         uint32_t* buf) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < CH; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t b = __float_as_uint(y[k][j]) & 0x7fffffffu;
      m = m > b ? m : b;
    }
  const float amax = __uint_as_float(row_max(m, lanes / 64, buf));
  float sc = __fdiv_rn(amax, 448.f);
  if (sc < kScaleFloor) sc = kScaleFloor;  // not for a NaN
  float up = 1.f;
  if (sc < 0x1p-64f) {  // so that no remainder falls below the fp32 range; a branch of the whole row
    up = 0x1p64f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) y[k][j] *= up;
  }
  const Divisor by(sc * up);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c0 = (k * lanes + lane) * V;
    if (c0 < C) {
      uint32_t w[V / 4];
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        w[i] = pack_e4m3x4(by.quotient(y[k][4 * i]), by.quotient(y[k][4 * i + 1]), by.quotient(y[k][4 * i + 2]),
                           by.quotient(y[k][4 * i + 3]));
      if constexpr (V == 8) *reinterpret_cast<u32x2*>(q + c0) = u32x2{w[0], w[1]};
      else *reinterpret_cast<uint32_t*>(q + c0) = w[0];
    }
  }
  if (lane == 0) *s = sc;
}

enum Kind { kQuant = 0, kNorm = 1, kResidualNorm = 2, kGlu = 3 };

template <typename T>
struct Args {
  const T* x;  // kGlu: the projection's output, values at column 0 and gates at column C
  int64_t xs;
  const T* h;  // kResidualNorm
  int64_t hs;
  const T* xbias;
  const T* gate;
  int64_t gate_stride;
  const T* local;
  int memory;
  const float* fbias;  // kGlu: 2 C values
  const float* w;      // norms
  float eps;
  const T* scale;
  const T* shift;
  int64_t mod_stride;
  int L;  // rows per batch
  T* out_h;
  int64_t os;
  uint8_t* q;
  int64_t qs;
  float* s;
  int64_t N;
  int C;
};

// A row per workgroup, held in registers: CH chunks of V values per lane, chunk k of lane t at column
// (k * lanes + t) * V. What bounds it is memory: residual_rms_q8 on 5168 x 1536 bf16 (55.6 MB) takes 13.7 us, 2.3 of them
// a launch's own, glu_q8 on 5168 x 6144 bf16 (159 MB) 31.9 us, the rate of a large copy (5.1 TB/s).
template <typename T, int KIND, int CH>
__global__ __launch_bounds__(64 * kMaxWaves) void row_kernel(const Args<T> a) {
  constexpr int V = Vec<T>::N;
  __shared__ uint32_t sum_buf[kMaxWaves], max_buf[kMaxWaves];
  const int C = a.C, lane = threadIdx.x, lanes = blockDim.x;
  const int64_t n = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  if (n >= a.N) return;
  const int64_t b = static_cast<uint32_t>(n) / static_cast<uint32_t>(a.L);  // N < 2^31
  const bool add_local = KIND == kResidualNorm && a.local && n - b * a.L >= a.memory;
  float y[CH][V];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c0 = (k * lanes + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) y[k][j] = 0.f;
    if (c0 < C) {
      Vec<T>::load(a.x + n * a.xs + c0, y[k]);
      if constexpr (KIND == kGlu) {
        float g[V], t[V];
        Vec<T>::load(a.x + n * a.xs + C + c0, g);
        if (a.fbias) {
          load_f32(a.fbias + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) y[k][j] += t[j];
          load_f32(a.fbias + C + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] += t[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) y[k][j] = y[k][j] * (g[j] * sigmoid(g[j]));
      }
      if constexpr (KIND == kResidualNorm) {
        float t[V];
        if (a.xbias) {
          Vec<T>::load(a.xbias + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) y[k][j] += t[j];
        }
        if (a.gate) {
          Vec<T>::load(a.gate + b * a.gate_stride + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) y[k][j] *= sigmoid(1.f - t[j]);
        }
        Vec<T>::load(a.h + n * a.hs + c0, t);
#pragma unroll
        for (int j = 0; j < V; ++j) y[k][j] = t[j] + y[k][j];
        if (add_local) {
          Vec<T>::load(a.local + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) y[k][j] += t[j];
        }
        Vec<T>::store(a.out_h + n * a.os + c0, y[k]);
      }
    }
  }
  if constexpr (KIND == kNorm || KIND == kResidualNorm) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) ss = __fmaf_rn(y[k][j], y[k][j], ss);
    const float inv = rsqrtf(row_sum(ss, lanes / 64, sum_buf) / static_cast<float>(C) + a.eps);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c0 = (k * lanes + lane) * V;
      if (c0 < C) {
        float w[V];
        load_f32(a.w + c0, w);
#pragma unroll
        for (int j = 0; j < V; ++j) y[k][j] = (y[k][j] * inv) * w[j];
        if (a.scale) {
          float s[V], t[V];
          Vec<T>::load(a.scale + b * a.mod_stride + c0, s);
          Vec<T>::load(a.shift + b * a.mod_stride + c0, t);
#pragma unroll
          for (int j = 0; j < V; ++j) y[k][j] = y[k][j] * (1.f + s[j]) + t[j];
        }
      }
    }
  }
  store_q8<V, CH>(y, a.q + n * a.qs, a.s + n, C, lane, lanes, max_buf);
}

// The longest row, in registers of 16 waves of 64 lanes: four chunks of fp32 values a lane, two of 16-bit ones.
constexpr int kMaxC = 16384;

template <typename T, int KIND, int CH>
void launch_ch(hipStream_t stream, const Args<T>& a) {
  const int lanes = (a.C / Vec<T>::N + CH - 1) / CH;
  constexpr int64_t kAcross = 1 << 21;  // a dimension of a grid has less than 2^32 threads
  const dim3 grid(static_cast<unsigned>(a.N < kAcross ? a.N : kAcross),
                  static_cast<unsigned>((a.N + kAcross - 1) / kAcross));
  hipLaunchKernelGGL((row_kernel<T, KIND, CH>), grid, dim3((lanes + 63) / 64 * 64), 0, stream, a);
}

// One chunk per lane is quickest while the card holds all waves at once (residual_rms_q8, bf16: 1292 x 1536 5.9 us against
// 7.4 with three), and for the GLU, whose lanes have two loads each anyway (5168 x 6144: 34.5 against 37.5); beyond that
// three (5168 x 1536: 14.6 against 15.4, 1000 x 8192: 15.2 against 17.2, fp32 rms_modulate_q8 on 8249 x 1024: 13.2 against
// 14.6, quantize_rows on 5168 x 1536: 6.5 against 6.9). Wider rows take what holds them.
template <typename T, int KIND>
void launch(hipStream_t stream, const Args<T>& a) {
  const int chunks = a.C / Vec<T>::N;
  const int64_t waves = a.N * ((chunks + 63) / 64);
  const bool many = KIND != kGlu && chunks > 64 && waves > 32 * static_cast<int64_t>(device_cus());
  constexpr int kLanes = 64 * kMaxWaves, kWidest = kMaxC / Vec<T>::N;
  static_assert(kWidest <= 4 * kLanes, "the widest row has a kernel that holds it");
  if constexpr (kWidest > 3 * kLanes) {  // fp32
    if (chunks > 3 * kLanes) return launch_ch<T, KIND, 4>(stream, a);
  }
  if (many || chunks > kLanes) launch_ch<T, KIND, 3>(stream, a);
  else launch_ch<T, KIND, 1>(stream, a);
}

}  // namespace quant
}  // namespace hb

using namespace hb;

namespace {

// The operands of a call as its checks see them, in elements but for `esize`.
struct Operand {
  const char* name;
  const void* p;
  int esize;
  int64_t rows, stride, cols;
};

int esize_of(int dtype) { return dtype == HB_F32 ? 4 : 2; }
int vec_of(int dtype) { return dtype == HB_F32 ? 4 : 8; }

int check_rows(const char* what, int dtype, int64_t N, int C, int L) {
  if (dtype != HB_BF16 && dtype != HB_F32 && dtype != HB_F16)
    return fail(HB_ERR_DTYPE, "%s: dtype %d is not HB_BF16 (0), HB_F32 (1) or HB_F16 (2)", what, dtype);
  if (N < 1 || N >= (int64_t(1) << 31) || L < 1)
    return fail(HB_ERR_SHAPE, "%s needs 1 <= N < 2^31 and rows_per_batch >= 1", what);
  if (C < 1 || C > quant::kMaxC || C % vec_of(dtype))
    return fail(HB_ERR_SHAPE, "%s needs rows of 1 to %d values, a multiple of %d (got %d)", what, quant::kMaxC,
                vec_of(dtype), C);
  return HB_OK;
}

// Pointer, alignment, stride and extent of every operand (NULL ones were accepted by the caller), then that no output
// shares an element with an input or another output.
int check_operands(const char* what, const Operand* outs, int n_out, const Operand* ins, int n_in, int64_t vec) {
  int st;
  for (int i = 0; i < n_out + n_in; ++i) {
    const Operand& o = i < n_out ? outs[i] : ins[i - n_out];
    if (!o.p) continue;
    const int align = o.cols > 1 ? 16 : 4;  // rows; a scale per row
    if (reinterpret_cast<uintptr_t>(o.p) % align)
      return fail(HB_ERR_STRIDE, "%s: %s must be %d-byte aligned", what, o.name, align);
    if (o.cols > 1 && (o.stride < o.cols || o.stride % vec))
      return fail(HB_ERR_STRIDE, "%s: %s stride %lld must be >= %lld and a multiple of %lld", what, o.name,
                  static_cast<long long>(o.stride), static_cast<long long>(o.cols), static_cast<long long>(vec));
    if ((st = check_extent(what, o.name, o.rows, o.stride, o.cols))) return st;
  }
  for (int i = 0; i < n_out; ++i) {
    const Operand& o = outs[i];
    const int64_t ob = rows_bytes(o.rows, o.stride, o.cols, o.esize);
    for (int j = 0; j < n_in + i; ++j) {
      const Operand& r = j < n_in ? ins[j] : outs[j - n_in];
      if (!r.p) continue;
      if (r.rows == o.rows && r.esize == o.esize) {
        if ((st = check_no_overlap(what, o.name, o.p, o.stride, o.cols, r.name, r.p, r.stride, r.cols, o.rows, o.esize,
                                   false)))
          return st;
      } else if ((st = check_disjoint(what, o.name, o.p, ob, r.name, r.p,
                                      rows_bytes(r.rows, r.stride, r.cols, r.esize)))) {
        return st;
      }
    }
  }
  return HB_OK;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return HB_OK;
}

template <int KIND, typename T, typename F>
int launch_as(hipStream_t stream, const F& fill) {
  quant::Args<T> a = {};
  fill(a);
  quant::launch<T, KIND>(stream, a);
  return 0;
}

// Runs row_kernel<KIND> for `dtype`; `fill` sets the arguments of any element type.
template <int KIND, typename F>
int launch_kind(const char* what, hipStream_t stream, int dtype, const F& fill) {
  if (dtype == HB_BF16) launch_as<KIND, uint16_t>(stream, fill);
  else if (dtype == HB_F16) launch_as<KIND, _Float16>(stream, fill);
  else launch_as<KIND, float>(stream, fill);
  return launched(what);
}

// `p` as the pointer type of `field`.
template <typename T>
void set(const T*& field, const void* p) { field = static_cast<const T*>(p); }
template <typename T>
void set(T*& field, void* p) { field = static_cast<T*>(p); }

}  // namespace

extern "C" {

int hb_quant_rows(hipStream_t stream, const void* x, int dtype, int64_t x_row_stride, void* q, int64_t q_row_stride,
                  float* q_scale, int64_t N, int C) {
  clear_error();
  const char* what = "quant_rows";
  int st = check_rows(what, dtype, N, C, 1);
  if (st) return st;
  if (!x || !q || !q_scale) return fail(HB_ERR_NULL, "%s: x, q and q_scale must be non-NULL", what);
  const Operand outs[] = {{"q", q, 1, N, q_row_stride, C}, {"q_scale", q_scale, 4, N, 1, 1}};
  const Operand ins[] = {{"x", x, esize_of(dtype), N, x_row_stride, C}};
  if ((st = check_operands(what, outs, 2, ins, 1, vec_of(dtype)))) return st;
  return launch_kind<quant::kQuant>(what, stream, dtype, [&](auto& a) {
    set(a.x, x), a.xs = x_row_stride, a.L = 1;
    set(a.q, q), a.qs = q_row_stride, a.s = q_scale, a.N = N, a.C = C;
  });
}

int hb_rms_modulate_q8(hipStream_t stream, const void* x, int dtype, int64_t x_row_stride, const float* weight,
                       float eps, const void* scale, const void* shift, int64_t mod_batch_stride, int rows_per_batch,
                       void* q, int64_t q_row_stride, float* q_scale, int64_t N, int C) {
  clear_error();
  const char* what = "rms_modulate_q8";
  int st = check_rows(what, dtype, N, C, rows_per_batch);
  if (st) return st;
  if (!x || !weight || !q || !q_scale)
    return fail(HB_ERR_NULL, "%s: x, weight, q and q_scale must be non-NULL", what);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(HB_ERR_EPS, "%s: eps %g must be finite and >= 0", what, eps);
  if (reinterpret_cast<uintptr_t>(weight) % 4) return fail(HB_ERR_STRIDE, "%s: weight must be 4-byte aligned", what);
  if (!scale != !shift) return fail(HB_ERR_NULL, "%s: scale and shift are given together or not at all", what);
  if (scale && N % rows_per_batch) return fail(HB_ERR_SHAPE, "%s: N must be a multiple of rows_per_batch", what);
  const int64_t nb = scale ? N / rows_per_batch : 1, ms = nb > 1 ? mod_batch_stride : C;
  const int es = esize_of(dtype);
  const Operand outs[] = {{"q", q, 1, N, q_row_stride, C}, {"q_scale", q_scale, 4, N, 1, 1}};
  const Operand ins[] = {{"x", x, es, N, x_row_stride, C},
                         {"scale", scale, es, nb, ms, C},
                         {"shift", shift, es, nb, ms, C}};
  if ((st = check_operands(what, outs, 2, ins, 3, vec_of(dtype)))) return st;
  for (const Operand& o : outs)
    if ((st = check_disjoint(what, o.name, o.p, rows_bytes(o.rows, o.stride, o.cols, o.esize), "weight", weight,
                             static_cast<int64_t>(C) * 4)))
      return st;
  return launch_kind<quant::kNorm>(what, stream, dtype, [&](auto& a) {
    set(a.x, x), a.xs = x_row_stride, a.w = weight, a.eps = eps;
    set(a.scale, scale), set(a.shift, shift), a.mod_stride = ms, a.L = rows_per_batch;
    set(a.q, q), a.qs = q_row_stride, a.s = q_scale, a.N = N, a.C = C;
  });
}

int hb_residual_rms_q8(hipStream_t stream, const void* h, int dtype, int64_t h_row_stride, const void* x,
                       int64_t x_row_stride, const void* x_bias, const void* gate, int64_t gate_batch_stride,
                       const void* local, int memory, const float* weight, float eps, const void* scale,
                       const void* shift, int64_t mod_batch_stride, int rows_per_batch, void* out_h,
                       int64_t out_h_row_stride, void* q, int64_t q_row_stride, float* q_scale, int64_t N, int C) {
  clear_error();
  const char* what = "residual_rms_q8";
  int st = check_rows(what, dtype, N, C, rows_per_batch);
  if (st) return st;
  if (!h || !x || !weight || !out_h || !q || !q_scale)
    return fail(HB_ERR_NULL, "%s: h, x, weight, out_h, q and q_scale must be non-NULL", what);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(HB_ERR_EPS, "%s: eps %g must be finite and >= 0", what, eps);
  if (reinterpret_cast<uintptr_t>(weight) % 4) return fail(HB_ERR_STRIDE, "%s: weight must be 4-byte aligned", what);
  if (!scale != !shift) return fail(HB_ERR_NULL, "%s: scale and shift are given together or not at all", what);
  if (memory < 0) return fail(HB_ERR_SHAPE, "%s: memory must be >= 0", what);
  if ((gate || scale) && N % rows_per_batch)
    return fail(HB_ERR_SHAPE, "%s: N must be a multiple of rows_per_batch", what);
  const int64_t nb = gate || scale ? N / rows_per_batch : 1;
  const int64_t gs = nb > 1 ? gate_batch_stride : C, ms = nb > 1 ? mod_batch_stride : C;
  const int es = esize_of(dtype);
  const Operand outs[] = {{"out_h", out_h, es, N, out_h_row_stride, C},
                          {"q", q, 1, N, q_row_stride, C},
                          {"q_scale", q_scale, 4, N, 1, 1}};
  const Operand ins[] = {{"h", h, es, N, h_row_stride, C},   {"x", x, es, N, x_row_stride, C},
                         {"x_bias", x_bias, es, 1, C, C},    {"local", local, es, 1, C, C},
                         {"gate", gate, es, nb, gs, C},      {"scale", scale, es, nb, ms, C},
                         {"shift", shift, es, nb, ms, C}};
  if ((st = check_operands(what, outs, 3, ins, 7, vec_of(dtype)))) return st;
  for (const Operand& o : outs)
    if ((st = check_disjoint(what, o.name, o.p, rows_bytes(o.rows, o.stride, o.cols, o.esize), "weight", weight,
                             static_cast<int64_t>(C) * 4)))
      return st;
  return launch_kind<quant::kResidualNorm>(what, stream, dtype, [&](auto& a) {
    set(a.h, h), a.hs = h_row_stride, set(a.x, x), a.xs = x_row_stride, set(a.xbias, x_bias);
    set(a.gate, gate), a.gate_stride = gs, set(a.local, local), a.memory = memory;
    a.w = weight, a.eps = eps, set(a.scale, scale), set(a.shift, shift), a.mod_stride = ms, a.L = rows_per_batch;
    set(a.out_h, out_h), a.os = out_h_row_stride;
    set(a.q, q), a.qs = q_row_stride, a.s = q_scale, a.N = N, a.C = C;
  });
}

int hb_glu_q8(hipStream_t stream, const void* proj, int dtype, int64_t proj_row_stride, const float* bias, void* q,
              int64_t q_row_stride, float* q_scale, int64_t N, int F) {
  clear_error();
  const char* what = "glu_q8";
  int st = check_rows(what, dtype, N, F, 1);
  if (st) return st;
  if (!proj || !q || !q_scale) return fail(HB_ERR_NULL, "%s: proj, q and q_scale must be non-NULL", what);
  if (reinterpret_cast<uintptr_t>(bias) % 4) return fail(HB_ERR_STRIDE, "%s: bias must be 4-byte aligned", what);
  const Operand outs[] = {{"q", q, 1, N, q_row_stride, F}, {"q_scale", q_scale, 4, N, 1, 1}};
  const Operand ins[] = {{"proj", proj, esize_of(dtype), N, proj_row_stride, 2 * static_cast<int64_t>(F)}};
  if ((st = check_operands(what, outs, 2, ins, 1, vec_of(dtype)))) return st;
  for (const Operand& o : outs)
    if ((st = check_disjoint(what, o.name, o.p, rows_bytes(o.rows, o.stride, o.cols, o.esize), "bias", bias,
                             static_cast<int64_t>(F) * 8)))
      return st;
  return launch_kind<quant::kGlu>(what, stream, dtype, [&](auto& a) {
    set(a.x, proj), a.xs = proj_row_stride, a.fbias = bias, a.L = 1;
    set(a.q, q), a.qs = q_row_stride, a.s = q_scale, a.N = N, a.C = F;
  });
}

}  // extern "C"

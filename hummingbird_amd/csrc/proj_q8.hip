// Products of 8-bit rows and 8-bit weights, for gfx950 (MI355X): the denoiser's projections (sa3jax/dit.py:31-34) on
// the e4m3 matrix cores, whose rate is twice the bf16 one's.
//
//   out[m, f] = (sum_k x[m, k] w[f, k]) sx[m] sw[f] + bias[f],   x, w e4m3, sx, sw, bias and the sum fp32,
//
// rounded once to the output type, for any scales (see `scaled_any`). C^T = W x^T as in the 16-bit projections: a lane of a
// 32x32 MFMA's result holds one row of x and 16 features, four of them consecutive.
//
// The e4m3 matrix cores (v_mfma_f32_32x32x64_f8f6f4, and v_mfma_f32_32x32x16_fp8_fp8 alike) do not add in full fp32:
// in 8 consecutive columns each product is cut towards zero to a multiple of 2^(E - 13), E the largest sum of the two
// operands' exponents; the rest is fp32. On rows of normal values that is an error of 1.5e-5 of the result, whatever K
// (7e-5 with one channel in a hundred 100 times as large), where rounding to half costs 2.1e-4 and to bf16 1.7e-3: taken
// for 16-bit outputs, some of which it moves to the neighbouring value. For fp32 outputs the codes are converted to bf16
// (exact) and multiplied on the bf16 cores, whose sums are fp32 (error 5e-8 at K = 1536, that of an fp32 product).
#include <type_traits>

#include "api.h"
#include "common.h"
#include "rows_tile.h"
#include "tiles.h"

namespace hb {
namespace q8 {

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

// acc sw sx + bias for any scales, whatever the range of the products on the way. A sum of e4m3 products is 0 or of a
// magnitude from 2^-18 to 2^41 (K <= 2^23). With a feature's scale of 2^-100 to 2^86 it stays in the fp32 range, and one
// FMA does the rest. (The row's scale first would overflow for rows of 1e34 and weights of 1e-4.) Other scales, which
// weights of 1e30 have, would overflow or lose bits where the result does not (weights of 1e33 and rows of 1e-10): they
// are multiplied as mantissas and their exponents added.
__device__ __forceinline__ bool ordinary(float sw) {
  return __float_as_uint(sw) - __float_as_uint(0x1p-100f) <= __float_as_uint(0x1p86f) - __float_as_uint(0x1p-100f);
}
__device__ __forceinline__ float scaled_ordinary(float acc, float sw, float sx, float bias) {
  return __fmaf_rn(acc * sw, sx, bias);
}
__device__ __forceinline__ float scaled_any(float acc, float sw, float sx, float bias) {
  const float m = acc * __builtin_amdgcn_frexp_mantf(sw) * __builtin_amdgcn_frexp_mantf(sx);
  return ldexpf(m, __builtin_amdgcn_frexp_expf(sw) + __builtin_amdgcn_frexp_expf(sx)) + bias;
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

// ---- Tiled product ------------------------------------------------------------------------------------------
// A workgroup of WF x WM waves computes FT features x MT rows in steps of 128 columns of K, which stream through
// kStages LDS stages: rows of 128 bytes whose 16-byte chunks are XOR-swizzled, filled by global_load_lds. A wave
// multiplies NF x NM tiles of 32 x 32. Two stages suffice where a CU has two workgroups or a step takes longer than a
// copy; a workgroup that has its CU to itself waits for its copies with two (0.5 us a step, whatever the tile) and gains
// from three or four (2584 x 6144 -> 1536, Medium, 27.5 -> 25.3 us; 400 x 6144 -> 1536, Small, 14.5 -> 12.3).
template <int FT_, int MT_, int WF_, int WM_, int WAVES_, int STAGES_ = 2>
struct Tile {
  static constexpr int FT = FT_, MT = MT_, WF = WF_, WM = WM_;
  static constexpr int NW = WF * WM, NF = FT / WF / 32, NM = MT / WM / 32;
  static constexpr int kWaves = WAVES_;  // per SIMD, of the workgroups that share a CU
  static constexpr int kStages = STAGES_;
  static constexpr int kStage = (FT + MT) * kStep;
  static constexpr int kBlocksA = FT / 8 / NW, kBlocksB = MT / 8 / NW;  // 1 KB copies per wave and stage
  static_assert(FT % (8 * NW) == 0 && MT % (8 * NW) == 0 && NF >= 1 && NM >= 1, "whole copies and tiles per wave");
};

// The copies of a stage by one wave: blocks wv, wv + NW, ... of the A rows (features), then of the B rows. Lane i's 16
// bytes land at byte 16 i of a block, row i / 8, position i % 8, so it fetches the chunk that the swizzle puts there.
// RAGGED: K may end inside a stage; chunks from column K on come from `zeros`.

template <class TL, bool RAGGED>
struct StageCopy {
  const uint8_t* w0;
  const uint8_t* x0;
  uint32_t aoff[TL::kBlocksA], boff[TL::kBlocksB];
  const int wv = wave_id() % TL::NW, r8 = (threadIdx.x & 63) >> 3, chunk = (threadIdx.x & 7) ^ r8 ^ (wv & 1);

  // Aims the copies at the tile of feature f0 and row m0.
  __device__ __forceinline__ void aim(const Args& a, int f0, int64_t m0) {
    w0 = a.w + f0 * a.w_rs;
    x0 = a.x + m0 * a.x_rs;
    const int lastf = a.F - 1 - f0;
    const int64_t lastm = a.M - 1 - m0;
#pragma unroll
    for (int u = 0; u < TL::kBlocksA; ++u) {  // rows past an end read the last one; their results are not stored
      const int r = 8 * (wv + TL::NW * u) + r8;
      aoff[u] = static_cast<uint32_t>((r < lastf ? r : lastf) * a.w_rs) + 16 * chunk;
    }
#pragma unroll
    for (int u = 0; u < TL::kBlocksB; ++u) {
      const int r = 8 * (wv + TL::NW * u) + r8;
      boff[u] = static_cast<uint32_t>((r < lastm ? r : lastm) * a.x_rs) + 16 * chunk;
    }
  }
  // Copy u of a stage whose columns start at k, to the stage at LDS byte address `stage`.
  __device__ __forceinline__ void one(int u, int k, int K, uint32_t stage) const {
    const bool a = u < TL::kBlocksA;
    const uint8_t* base = (a ? w0 : x0) + k;
    const uint32_t off = a ? aoff[a ? u : 0] : boff[a ? 0 : u - TL::kBlocksA];
    const uint32_t to = stage + (a ? 0 : TL::FT * kStep) + (wv + TL::NW * (a ? u : u - TL::kBlocksA)) * 1024;
    if constexpr (RAGGED) lds_dma16_any(k + 16 * chunk < K ? base + off : zeros, to);
    else lds_dma16(base, off, to);
  }
  static constexpr int kCopies = TL::kBlocksA + TL::kBlocksB;
};

// Half a stage (64 columns) of a wave's operands: 32 bytes of each of its rows, lane half lh the chunks 4 kk + 2 lh + 0, 1.
template <class TL>
struct Frags {
  u32x4 a[TL::NF][2], b[TL::NM][2];
  static constexpr int kReads = 2 * (TL::NF + TL::NM);
  __device__ __forceinline__ void read(int i, const uint8_t* st, int fw, int mw, int kk) {
    const int lr = threadIdx.x & 31, lh = (threadIdx.x & 63) >> 5;
    const int c = 4 * kk + 2 * lh + (i & 1), t = i >> 1;
    if (t < TL::NF) a[t][i & 1] = *reinterpret_cast<const u32x4*>(st + swz_byte(fw + 32 * t + lr, c));
    else
      b[t - TL::NF][i & 1] =
          *reinterpret_cast<const u32x4*>(st + TL::FT * kStep + swz_byte(mw + 32 * (t - TL::NF) + lr, c));
  }
};

__device__ __forceinline__ i32x8 join(const u32x4 (&v)[2]) {
  return i32x8{static_cast<int>(v[0][0]), static_cast<int>(v[0][1]), static_cast<int>(v[0][2]),
               static_cast<int>(v[0][3]), static_cast<int>(v[1][0]), static_cast<int>(v[1][1]),
               static_cast<int>(v[1][2]), static_cast<int>(v[1][3])};
}

// One tile's 64 columns: on the e4m3 cores, or (WIDE) as four 16-column products of widened codes on the bf16 cores.
template <bool WIDE>
__device__ __forceinline__ f32x16 multiply(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x16 c) {
  if constexpr (!WIDE) return mfma_32x32x64(join(a), join(b), c);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const u32x2 ga = {a[g >> 1][2 * (g & 1)], a[g >> 1][2 * (g & 1) + 1]};
    const u32x2 gb = {b[g >> 1][2 * (g & 1)], b[g >> 1][2 * (g & 1) + 1]};
    c = mfma_bf16_32x32x16(widen8(ga), widen8(gb), c);
  }
  return c;
}

// A wave's results, scaled and stored (see `store_32x32`). `sw`, `bias`, `sx`: the scales of this wave's features and
// rows, in LDS.
template <typename T, class TL, bool STREAM>
__device__ __forceinline__ void store_tile(const Args& a, const f32x16 (&acc)[TL::NF][TL::NM], int f0, int64_t m0,
                                           const float* sw_, const float* bias_, const float* sx_) {
  const int lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5;
  float sx[TL::NM];
#pragma unroll
  for (int t = 0; t < TL::NM; ++t) sx[t] = sx_[32 * t + lr];
  bool odd = false;  // any scale of the wave's features that is not ordinary: a branch of the whole wave
#pragma unroll
  for (int n = 0; n < TL::NF; ++n) odd |= !ordinary(sw_[32 * n + lr]);
  odd = __any(odd);
#pragma unroll
  for (int n = 0; n < TL::NF; ++n) {
    const int fn = f0 + 32 * n;
    __builtin_amdgcn_sched_barrier(0);  // the scales of one n at a time: registers
    float sw[16], bias[16];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 s4 = *reinterpret_cast<const f32x4*>(sw_ + 32 * n + 8 * g + 4 * lh);
      const f32x4 b4 = *reinterpret_cast<const f32x4*>(bias_ + 32 * n + 8 * g + 4 * lh);
#pragma unroll
      for (int j = 0; j < 4; ++j) sw[4 * g + j] = s4[j], bias[4 * g + j] = b4[j];
    }
#pragma unroll
    for (int t = 0; t < TL::NM; ++t) {
      float v[16];
      if (__builtin_expect(odd, 0)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = scaled_any(acc[n][t][i], sw[i], sx[t], bias[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = scaled_ordinary(acc[n][t][i], sw[i], sx[t], bias[i]);
      }
      store_32x32<T, STREAM>(static_cast<T*>(a.out), a.os, a.M, a.F, m0 + 32 * t, fn, v);
    }
  }
}

template <class TL>
int64_t tiles_of(const Args& a) {
  return static_cast<int64_t>((a.F + TL::FT - 1) / TL::FT) * ((a.M + TL::MT - 1) / TL::MT);
}

// Workgroups stay: each takes every gridDim.x-th tile, and its copies run kStages steps ahead of the products across
// the tiles' ends, so that a tile's first steps land while the one before it is finished and stored. Past the last tile they
// copy that tile's columns again, for nothing: the loop has no branch around a copy, and the kernel waits for them
// before it ends.
template <typename T, class TL, bool RAGGED, bool STREAM>
__global__ __launch_bounds__(64 * TL::NW) __attribute__((amdgpu_waves_per_eu(TL::kWaves, TL::kWaves))) void tiled_kernel(
    const Args a) {
  constexpr bool WIDE = std::is_same<T, float>::value;
  __shared__ __attribute__((aligned(16))) uint8_t smem[TL::kStages * TL::kStage];
  // the scales and biases of a tile and of the next: features' scales, biases, rows' scales
  __shared__ __attribute__((aligned(16))) float scales[2][2 * TL::FT + TL::MT];
  const int nf = (a.F + TL::FT - 1) / TL::FT, nm = static_cast<int>((a.M + TL::MT - 1) / TL::MT), tiles = nf * nm;
  // Groups of eight feature tiles walk the row tiles together (of four: 8249 x 1536 -> 12288 177 against 172 us), and the
  // workgroups of an XCD take consecutive tiles, so that both operands are read from its L2.
  auto origin = [&](int p, int& f0, int64_t& m0) {
    constexpr int GF = 8;
    const int id = xcd_remap(p, tiles), g = id / (GF * nm), gs = nf - g * GF < GF ? nf - g * GF : GF;
    const int in = id - g * GF * nm;
    f0 = (g * GF + in % gs) * TL::FT;
    m0 = static_cast<int64_t>(in / gs) * TL::MT;
  };
  const int wv = wave_id(), fw = wv % TL::WF * (32 * TL::NF), mw = wv / TL::WF * (32 * TL::NM);
  const uint32_t lds0 = lds_addr(smem);
  const int nk = (a.K + kStep - 1) / kStep;

  // What is copied next: step `cs` of tile `ct` (in the order of p).
  StageCopy<TL, RAGGED> copy;
  int ct = blockIdx.x, cs = 0;
  auto aim = [&]() {
    int f0;
    int64_t m0;
    origin(ct, f0, m0);
    copy.aim(a, f0, m0);
  };
  auto advance = [&]() {
    if (++cs < nk) return;
    cs = 0;
    if (ct + static_cast<int>(gridDim.x) >= tiles) return;
    ct += gridDim.x;
    aim();
  };
  constexpr int kTiles = TL::NF * TL::NM, kReads = Frags<TL>::kReads, kCopies = StageCopy<TL, RAGGED>::kCopies;
  // A tile's scales, 64 of each kind by a wave, copied while its first step runs; tiles alternate between the sets.
  auto copy_scales = [&](int f0, int64_t m0, int set) {
    const uint32_t to = lds_addr(scales[set]) + 256 * wv;
    const int lane = threadIdx.x & 63, i = 64 * wv + lane;
    if (64 * wv < TL::FT) {
      const int f = i < a.F - 1 - f0 ? i : a.F - 1 - f0;
      lds_dma4(a.sw + f0, 4 * f, to);
      if (a.bias) lds_dma4(a.bias + f0, 4 * f, to + 4 * TL::FT);
    }
    if (64 * wv < TL::MT) {
      const int64_t last = a.M - 1 - m0;
      lds_dma4(a.sx + m0, static_cast<uint32_t>(4 * (i < last ? i : last)), to + 8 * TL::FT);
    }
  };
  if (!a.bias && threadIdx.x < TL::FT) scales[0][TL::FT + threadIdx.x] = scales[1][TL::FT + threadIdx.x] = 0.f;
  aim();
#pragma unroll
  for (int i = 0; i < TL::kStages; ++i) {
#pragma unroll
    for (int u = 0; u < kCopies; ++u) copy.one(u, cs * kStep, a.K, lds0 + i * TL::kStage);
    advance();
  }
  wait_copies<(TL::kStages - 1) * kCopies>();
  wait_lds();
  barrier();
  Frags<TL> lo, hi;
#pragma unroll
  for (int i = 0; i < kReads; ++i) lo.read(i, smem, fw, mw, 0);

  // A step of a wave is 2 kTiles products, lo's and hi's. In the first kFree the operands of hi are read; then every wave
  // has the whole stage in registers (barrier) and the step kStages on is copied into it, over kTiles products: faster,
  // the copies wait for the address unit and hold up the products. Before hi's products the next step's copies, issued
  // kStages - 1 steps ago, have landed (barrier), and its lo is read during them.
  constexpr int kFree = kTiles / 2;                                    // 0: one barrier does for both
  constexpr int kEarly = (kTiles - kFree) * kCopies / kTiles;          // copies issued before the second barrier
  constexpr int kLater = (TL::kStages - 2) * kCopies;                  // copies of the steps between the next and that one
  uint32_t b = 0;                                                      // byte offset of the step's stage
  int set = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, set ^= 1) {
    int f0;
    int64_t m0;
    origin(tile, f0, m0);
    copy_scales(f0, m0, set);
    f32x16 acc[TL::NF][TL::NM];
#pragma unroll
    for (int i = 0; i < TL::NF; ++i)
#pragma unroll
      for (int j = 0; j < TL::NM; ++j) acc[i][j] = f32x16{};
    for (int s = 0; s < nk; ++s) {
      const uint32_t stage = __builtin_amdgcn_readfirstlane(lds0 + b);
      const int k = cs * kStep;
      auto copies = [&](int j) {  // those of product j past the barrier
#pragma unroll
        for (int u = j * kCopies / kTiles; u < (j + 1) * kCopies / kTiles; ++u) copy.one(u, k, a.K, stage);
      };
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (kFree == 0 || i < kFree) {
          constexpr int n = kFree == 0 ? kTiles : kFree;
#pragma unroll
          for (int r = i * kReads / n; r < (i + 1) * kReads / n; ++r) hi.read(r, smem + b, fw, mw, 1);
        }
        if (kFree > 0 && i == kFree) {
          wait_lds();
          barrier();
        }
        if (kFree > 0 && i >= kFree) copies(i - kFree);
        acc[i / TL::NM][i % TL::NM] = multiply<WIDE>(lo.a[i / TL::NM], lo.b[i % TL::NM], acc[i / TL::NM][i % TL::NM]);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_copies<kLater + (kFree == 0 ? 0 : kEarly)>();
      if (kFree == 0) wait_lds();
      barrier();
      b = b == (TL::kStages - 1) * TL::kStage ? 0 : b + TL::kStage;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (kFree == 0) copies(i);
        else if (i < kFree) copies(kTiles - kFree + i);
        // (after the very last step, of a stage that nothing needs)
#pragma unroll
        for (int r = i * kReads / kTiles; r < (i + 1) * kReads / kTiles; ++r) lo.read(r, smem + b, fw, mw, 0);
        acc[i / TL::NM][i % TL::NM] = multiply<WIDE>(hi.a[i / TL::NM], hi.b[i % TL::NM], acc[i / TL::NM][i % TL::NM]);
        __builtin_amdgcn_sched_barrier(0);
      }
      advance();
    }
    if (nk < TL::kStages - 1) {  // the scales' copies are among those that the last wait left
      wait_copies<0>();
      barrier();
    }
    const float* sc = scales[set];
    store_tile<T, TL, STREAM>(a, acc, f0 + fw, m0 + mw, sc + fw, sc + TL::FT + fw, sc + 2 * TL::FT + mw);
  }
  wait_copies<0>();
}

template <typename T, class TL>
void launch_tiled(hipStream_t stream_, const Args& a) {
  const int64_t tiles = tiles_of<TL>(a), slots = static_cast<int64_t>(TL::kWaves) * 4 / TL::NW * device_cus();
  const dim3 grid(static_cast<unsigned>(tiles < slots ? tiles : slots)), block(64 * TL::NW);
  auto with = [&](auto ragged, auto stream) {
    hipLaunchKernelGGL((tiled_kernel<T, TL, decltype(ragged)::value, decltype(stream)::value>), grid, block, 0, stream_, a);
  };
  const std::true_type yes;
  const std::false_type no;
  if constexpr (TL::FT * TL::MT >= 128 * 128 && TL::kStages == 2) {  // (the others are for small outputs)
    if (a.M * a.F * static_cast<int64_t>(sizeof(T)) > kStreamBytes) return a.K % kStep ? with(yes, yes) : with(no, yes);
  }
  a.K % kStep ? with(yes, no) : with(no, no);
}

// ---- Few tiles ------------------------------------------------------------------------------------------------
// A product of fewer tiles than CUs, split along K inside the workgroup: kGroups groups of waves, each with stages of its
// own, take consecutive steps of one tile, and their sums are added in the groups' order through LDS.
constexpr int kGroups = 4;

template <typename T, class TL, bool RAGGED>
__global__ __launch_bounds__(64 * TL::NW * kGroups) void split_kernel(const Args a) {
  static_assert(TL::NF == 1 && TL::NM == 1, "a 32 x 32 tile per wave");
  constexpr bool WIDE = std::is_same<T, float>::value;
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * kGroups * TL::kStage];
  __shared__ __attribute__((aligned(16))) float scales[2 * TL::FT + TL::MT];
  static_assert((kGroups - 1) * TL::NW * 4096 <= 2 * kGroups * TL::kStage, "the groups' sums fit the stages");
  const int nf = (a.F + TL::FT - 1) / TL::FT;
  const int f0 = static_cast<int>(blockIdx.x) % nf * TL::FT;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / nf) * TL::MT;
  const int group = wave_id() / TL::NW, wv = wave_id() % TL::NW, lane = threadIdx.x & 63;
  const int fw = wv % TL::WF * 32, mw = wv / TL::WF * 32;
  const int nk = (a.K + kStep - 1) / kStep, per = (nk + kGroups - 1) / kGroups, first = group * per;
  const int mine = nk - first < per ? nk - first : per;  // steps of this group, possibly none; barriers are for `per`
  uint8_t* const stages = smem + 2 * group * TL::kStage;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem) + 2 * group * TL::kStage);
  if (threadIdx.x < TL::FT) {
    const int f = f0 + static_cast<int>(threadIdx.x) < a.F ? f0 + static_cast<int>(threadIdx.x) : a.F - 1;
    scales[threadIdx.x] = a.sw[f];
    scales[TL::FT + threadIdx.x] = a.bias ? a.bias[f] : 0.f;
  }
  if (threadIdx.x < TL::MT) {
    const int64_t m = m0 + threadIdx.x < a.M ? m0 + threadIdx.x : a.M - 1;
    scales[2 * TL::FT + threadIdx.x] = a.sx[m];
  }
  StageCopy<TL, RAGGED> copy;
  copy.aim(a, f0, m0);
  constexpr int kReads = Frags<TL>::kReads, kCopies = StageCopy<TL, RAGGED>::kCopies;
  auto fill = [&](int s) {  // the group's step s into stage s % 2
    if (s >= mine) return;
    const int k = (first + s) * kStep;
#pragma unroll
    for (int u = 0; u < kCopies; ++u) copy.one(u, k, a.K, lds0 + (s & 1) * TL::kStage);
  };
  fill(0);
  fill(1);
  f32x16 acc[1][1] = {{f32x16{}}};
  for (int s = 0; s < per; ++s) {
    // step s has landed: all copies but those of step s + 1
    if (s + 1 < mine) wait_copies<kCopies>();
    else wait_copies<0>();
    wait_lds();
    barrier();
    Frags<TL> lo, hi;
    if (s < mine) {
      const uint8_t* st = stages + (s & 1) * TL::kStage;
#pragma unroll
      for (int i = 0; i < kReads; ++i) lo.read(i, st, fw, mw, 0);
#pragma unroll
      for (int i = 0; i < kReads; ++i) hi.read(i, st, fw, mw, 1);
    }
    wait_lds();
    barrier();  // the stage is free
    fill(s + 2);
    if (s < mine) {
      acc[0][0] = multiply<WIDE>(lo.a[0], lo.b[0], acc[0][0]);
      acc[0][0] = multiply<WIDE>(hi.a[0], hi.b[0], acc[0][0]);
    }
  }
  // (every wave's reads ended before the last barrier, and no copy is in flight)
  f32x4* const sums = reinterpret_cast<f32x4*>(smem);  // [group - 1][wave][4][64 lanes]
  if (group > 0) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      sums[(((group - 1) * TL::NW + wv) * 4 + g) * 64 + lane] =
          f32x4{acc[0][0][4 * g], acc[0][0][4 * g + 1], acc[0][0][4 * g + 2], acc[0][0][4 * g + 3]};
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int o = 0; o < kGroups - 1; ++o)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = sums[((o * TL::NW + wv) * 4 + g) * 64 + lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[0][0][4 * g + j] += v[j];
    }
  store_tile<T, TL, false>(a, acc, f0 + fw, m0 + mw, scales + fw, scales + TL::FT + fw, scales + 2 * TL::FT + mw);
}

template <typename T, class TL>
void launch_split(hipStream_t stream, const Args& a) {
  const dim3 grid(static_cast<unsigned>(tiles_of<TL>(a))), block(64 * TL::NW * kGroups);
  if (a.K % kStep) hipLaunchKernelGGL((split_kernel<T, TL, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((split_kernel<T, TL, false>), grid, block, 0, stream, a);
}

// ---- Few rows -----------------------------------------------------------------------------------------------
// Up to 16 CT rows, where the weights' bytes are the cost: each is read once, straight into the registers of the wave that
// multiplies it. A workgroup computes 16 features for all rows; its waves take the 128-column chunks of K in turns and
// their partial sums are added in the waves' order. On v_mfma_f32_16x16x128_f8f6f4 a lane holds 32 consecutive columns
// of feature (or row) lane % 16.
constexpr int kMaxWaves = 16;

__device__ __forceinline__ f32x4 mfma_16x16x128(i32x8 a, i32x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

template <bool WIDE>
__device__ __forceinline__ f32x4 multiply16(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4 c) {
  if constexpr (!WIDE) return mfma_16x16x128(join(a), join(b), c);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const u32x2 ga = {a[g >> 1][2 * (g & 1)], a[g >> 1][2 * (g & 1) + 1]};
    const u32x2 gb = {b[g >> 1][2 * (g & 1)], b[g >> 1][2 * (g & 1) + 1]};
    c = mfma_bf16_16x16x32(widen8(ga), widen8(gb), c);
  }
  return c;
}

// 32 columns of a row from column k on, zeros from column K on (K a multiple of 16).
__device__ __forceinline__ void load32(const uint8_t* row, int k, int K, u32x4 (&v)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = u32x4{0, 0, 0, 0};
    if (k + 16 * i < K) v[i] = ld16(row + k + 16 * i);
  }
}

template <typename T, int CT>
__global__ __launch_bounds__(64 * kMaxWaves) void few_rows_kernel(const Args a) {
  constexpr bool WIDE = std::is_same<T, float>::value;
  __shared__ float part[kMaxWaves][CT][16][17];  // [wave][row tile][row][feature]
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4, wave = wave_id(), waves = blockDim.x >> 6;
  const int f0 = blockIdx.x * 16, M = static_cast<int>(a.M);
  const uint8_t* wrow = a.w + (f0 + lr < a.F ? f0 + lr : a.F - 1) * a.w_rs;  // past the end: not stored
  const uint8_t* xrow[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) xrow[t] = a.x + (16 * t + lr < M ? 16 * t + lr : M - 1) * a.x_rs;
  f32x4 acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = (a.K + kStep - 1) / kStep;
  u32x4 w[2][2], x[2][CT][2];
  auto load = [&](int c, int buf) {
    const int k = c * kStep + 32 * lq;
    load32(wrow, k, a.K, w[buf]);
#pragma unroll
    for (int t = 0; t < CT; ++t) load32(xrow[t], k, a.K, x[buf][t]);
  };
  // The loads of a wave's next chunk are in flight while it multiplies this one.
  int c = wave;
  load(c, 0);
  for (; c < chunks; c += 2 * waves) {
    if (c + waves < chunks) load(c + waves, 1);
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = multiply16<WIDE>(w[0], x[0][t], acc[t]);
    if (c + waves >= chunks) break;
    if (c + 2 * waves < chunks) load(c + 2 * waves, 0);
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = multiply16<WIDE>(w[1], x[1][t], acc[t]);
  }
#pragma unroll
  for (int t = 0; t < CT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][lr][4 * lq + i] = acc[t][i];
  __syncthreads();
  T* const out = static_cast<T*>(a.out);
  for (int e = threadIdx.x; e < 256 * CT; e += blockDim.x) {
    const int r = e >> 4, fo = e & 15;
    if (r >= M || f0 + fo >= a.F) continue;
    float v = 0.f;
    for (int i = 0; i < waves; ++i) v += part[i][r >> 4][r & 15][fo];
    const float sw = a.sw[f0 + fo], bias = a.bias ? a.bias[f0 + fo] : 0.f;
    v = ordinary(sw) ? scaled_ordinary(v, sw, a.sx[r], bias) : scaled_any(v, sw, a.sx[r], bias);
    out[r * a.os + f0 + fo] = cast_out<T>(v);
  }
}

template <typename T, int CT>
void launch_few_rows(hipStream_t stream, const Args& a) {
  const int chunks = (a.K + kStep - 1) / kStep;
  hipLaunchKernelGGL((few_rows_kernel<T, CT>), dim3(static_cast<unsigned>((a.F + 15) / 16)),
                     dim3(64 * (chunks < kMaxWaves ? chunks : kMaxWaves)), 0, stream, a);
}

// Which kernel, as measured (times in us, with the 2.5 of a launch; K = 1536 unless said). In order:
//   few rows   up to 16 rows (7 x 7680: 5.3 against 7.9 Small), and up to 32 of a narrow product (24 x 1536: 4.1 against
//              5.0, K = 6144 9.4 against 11.6; but 24 x 7680: 5.8 against 5.3);
//   Small      at most one per CU, with four stages from more than 8 steps on (400 x 1536, K = 6144: 12.3 against 14.0
//              with three and 16.5 Half; 100 x 1536, K = 256: 3.6 against 3.3 with two);
//   Half       at most one per CU (1292 x 1536, K = 6144: 16.8 against 21.4 Medium with three stages, 25.0 Small with two);
//   Medium     at most one per CU, with three stages (2584 x 1536, K = 6144: 25.3 against 27.5 with two); beyond that two
//              workgroups share a CU, one's epilogue beside the other's products (2584 x 12288: 53 against 56 with three
//              stages, one per CU, and 61 Large);
//   then what takes the least time, in rounds of Medium: a round of Large (one per CU) takes 0.95 of one of Medium (two
//              per CU; 5168 x 7680: 61.0 against 62.0; 5168 x 1536, K = 6144: 41.1 against 44.6) and one of Half 0.7
//              (504 tiles of Half, 11.3, against the same product's 264 of Medium, 13.9), and a last round of at most
//              one workgroup per CU 0.65 and 0.5. Tall, three stages and one per CU, takes 0.74 where one round of it
//              does (4000 x 1536: 12.4 against 14.4 Medium; 700 x 7680: 12.7 against 14.3); beyond one round it gains
//              in a loop over one product (1292 x 12288: 28.4 against 30.4) and loses in a render (39.7 against 38.9 ms).
// fp32 outputs are bound by the bf16 cores and the conversions, not by copies: two stages but for Half's and, with a tile
// per CU and more than 8 steps, K split among 16 waves (400 x 1536, K = 6144: 17.7 against 19.6); Small up to 3/4 Medium
// tiles per CU (154 x 12288: 13.1 against 14.7 Half); 257 x 12288: 16.3 Half against 21.8 Medium.
template <typename T>
void launch(hipStream_t stream, const Args& a) {
  using Small = Tile<64, 64, 2, 2, 3>;
  using Half = Tile<128, 64, 2, 2, 2, 3>;
  using Medium = Tile<128, 128, 2, 2, 2>;
  constexpr bool wide = sizeof(T) == 4;
  const int64_t cus = device_cus(), small = tiles_of<Small>(a), half = tiles_of<Half>(a), medium = tiles_of<Medium>(a);
  const bool is_long = a.K > 8 * kStep;
  if (a.M <= 16) return launch_few_rows<T, 1>(stream, a);
  if (a.M <= 32 && small <= cus / 4) return launch_few_rows<T, 2>(stream, a);
  if constexpr (wide) {
    if (small <= cus && is_long) return launch_split<T, Small>(stream, a);
    if (medium <= cus * 3 / 4) return launch_tiled<T, Small>(stream, a);
  } else {
    if (small <= cus && is_long) return launch_tiled<T, Tile<64, 64, 2, 2, 1, 4>>(stream, a);
    if (small <= cus) return launch_tiled<T, Small>(stream, a);
    if (half <= cus) return launch_tiled<T, Half>(stream, a);
    if (medium <= cus) return launch_tiled<T, Tile<128, 128, 2, 2, 1, 3>>(stream, a);
  }
  auto rounds = [&](int64_t tiles, double whole, double last) {  // two tiles per CU and round
    const int64_t rest = tiles % (2 * cus);
    return static_cast<double>(tiles / (2 * cus)) * whole + (rest > cus ? whole : rest > 0 ? last : 0.0);
  };
  const double m = rounds(medium, 1.0, 0.65), h = rounds(half, 0.7, 0.5);
  if constexpr (!wide) {
    using Large = Tile<128, 256, 2, 2, 1>;
    using Tall = Tile<128, 192, 2, 2, 1, 3>;
    const double l = 0.95 * static_cast<double>((tiles_of<Large>(a) + cus - 1) / cus);
    if (tiles_of<Tall>(a) <= cus && h > 0.74) return launch_tiled<T, Tall>(stream, a);
    if (l <= m && l <= h) return launch_tiled<T, Large>(stream, a);
  }
  if (h < m) return launch_tiled<T, Half>(stream, a);
  launch_tiled<T, Medium>(stream, a);
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
  if (M < 1 || M > (1 << 21) || F < 1 || F > (1 << 21) || K < 16 || K > (1 << 23) || K % 16)
    return fail(HB_ERR_SHAPE, "%s needs 1 <= M, F <= 2^21 and K a multiple of 16 up to 2^23 (M=%lld, K=%d, F=%d)", what,
                static_cast<long long>(M), K, F);
  if (!x || !x_scale || !w || !w_scale || !out)
    return fail(HB_ERR_NULL, "%s: x, x_scale, w, w_scale and out must be non-NULL", what);
  const int es = out_dtype == HB_F32 ? 4 : 2;
  auto misaligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  // A tile's rows are addressed by 32-bit offsets from its first.
  auto bad_rows = [&](const void* p, int64_t rs) { return misaligned(p, 16) || rs < K || rs % 16 || rs > (1 << 23); };
  const char* rows_of = bad_rows(x, x_row_stride) ? "x" : bad_rows(w, w_row_stride) ? "w" : nullptr;
  if (rows_of)
    return fail(HB_ERR_STRIDE, "%s: %s must be 16-byte aligned with a row stride >= K, a multiple of 16 up to 2^23", what,
                rows_of);
  if (misaligned(x_scale, 4) || misaligned(w_scale, 4) || misaligned(bias, 4))
    return fail(HB_ERR_STRIDE, "%s: x_scale, w_scale and bias must be 4-byte aligned", what);
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

// Products of microscaled 4-bit rows and weights, for gfx950 (MI355X).
//
//   out[m, f] = sum_k x[m, k] w[f, k] + bias[f],   x and w e2m1 codes with one e8m0 scale (a byte, 2^(s - 127)) per 32
//   columns, the sum and bias fp32, rounded once to the output type.
//
// C^T = W x^T on v_mfma_scale_f32_32x32x64_f8f6f4, whose 4-bit rate is twice the 8-bit one's and which applies the scales:
// lane half lh holds 32 columns of its row, and a byte of a register of its own is their scale. A stage is 256 columns, 128
// bytes of codes and 8 of scales per row: lane half lh takes blocks 4 lh .. 4 lh + 3 of the eight, one per product, so
// that one dword of a row holds its scales for the four (the order of K's blocks is free, as long as both operands share
// it). The products of e2m1 values are multiples of 1/4 up to 36, so the cores add a block's exactly; the rest is fp32.
#include <type_traits>

#include "api.h"
#include "common.h"
#include "rows_tile.h"
#include "tiles.h"

namespace hb {
namespace mx4 {

constexpr int kGroup = 32;        // columns that share a scale
constexpr int kCols = 2 * kStep;  // columns of a stage

struct Args {
  const uint8_t* x;  // (M, K / 2), row stride x_rs bytes
  int64_t x_rs;
  const uint8_t* sx;  // (M, K / 32), row stride sx_rs
  int64_t sx_rs;
  const uint8_t* w;  // (F, K / 2), row stride w_rs
  int64_t w_rs;
  const uint8_t* sw;  // (F, K / 32), row stride sw_rs
  int64_t sw_rs;
  const float* bias;  // F values or null
  void* out;          // (M, F), row stride os elements
  int64_t os;
  int64_t M;
  int K, F;
};

// 32 columns of each lane half (of each quarter of the wave for 16x16x128), scaled by byte J of the lanes' registers.
template <int J>
__device__ __forceinline__ f32x16 mfma_32x32x64(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 wa = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3])};
  const i32x8 wb = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, J, static_cast<int>(sa), J,
                                                         static_cast<int>(sb));
}
__device__ __forceinline__ f32x4 mfma_16x16x128(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 wa = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3])};
  const i32x8 wb = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, static_cast<int>(sa), 0,
                                                          static_cast<int>(sb));
}

// As lds_dma4 with an address per lane.
__device__ __forceinline__ void lds_dma4_any(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "m0");
}

// ---- Tiled product ------------------------------------------------------------------------------------------
// A workgroup of WF x WM waves computes FT features x MT rows in steps of 256 columns, which stream through kStages LDS
// stages: code rows of 128 bytes whose 16-byte chunks are XOR-swizzled, then the rows' scales. A wave multiplies NF x NM
// tiles of 32 x 32.
// RAGGED: K ends inside a stage, or scale rows that are not whole dwords. A row's eight scales of a stage then lie in two
// or three dwords, the first with up to three bytes of what is before them: the dwords are copied whole (each holds at
// least a byte of the row), 16 bytes a row, and shifted when they are used.
template <int FT_, int MT_, int WF_, int WM_, int WAVES_, int STAGES_ = 2>
struct Tile {
  static constexpr int FT = FT_, MT = MT_, WF = WF_, WM = WM_;
  static constexpr int NW = WF * WM, NF = FT / WF / 32, NM = MT / WM / 32;
  static constexpr int kWaves = WAVES_;  // per SIMD, of the workgroups that share a CU
  static constexpr int kStages = STAGES_;
  static constexpr int kBlocksA = FT / 8 / NW, kBlocksB = MT / 8 / NW;  // 1 KB copies per wave and stage
  static_assert(FT % (8 * NW) == 0 && MT % (8 * NW) == 0 && FT % 32 == 0 && NF >= 1 && NM >= 1,
                "whole copies and tiles per wave");
};
template <class TL, bool RAGGED>
struct Stage {
  static constexpr int kRows = TL::FT + TL::MT;
  static constexpr int kScaleRow = RAGGED ? 16 : 8;  // bytes
  static constexpr int kScales = kRows * kStep;      // where the scales start
  static constexpr int kBytes = kRows * (kStep + kScaleRow);
  static constexpr int kScaleBlocks = kRows * kScaleRow / 256;  // copies of 256 bytes; a wave's past the last repeat it
  static constexpr int kBlocksS = (kScaleBlocks + TL::NW - 1) / TL::NW;
};

// The copies of a stage by one wave: of the codes, blocks wv, wv + NW, ... of the A rows (features), then of the B rows,
// then of the scales. Lane i's 16 bytes of codes land at byte 16 i of a block, row i / 8, position i % 8, so it fetches
// the chunk that the swizzle puts there.
template <class TL, bool RAGGED>
struct StageCopy {
  using St = Stage<TL, RAGGED>;
  const uint8_t* w0;
  const uint8_t* x0;
  uint32_t aoff[TL::kBlocksA], boff[TL::kBlocksB];
  const uint8_t* sp[St::kBlocksS];  // this lane's dword of step 0
  int srem[St::kBlocksS];           // bytes from it to its row's end
  const int wv = wave_id() % TL::NW, r8 = (threadIdx.x & 63) >> 3, chunk = (threadIdx.x & 7) ^ r8 ^ (wv & 1);

  // Aims the copies at the tile of feature f0 and row m0. Rows past an end read the last one; their results are not stored.
  __device__ __forceinline__ void aim(const Args& a, int f0, int64_t m0) {
    w0 = a.w + f0 * a.w_rs;
    x0 = a.x + m0 * a.x_rs;
    const int lastf = a.F - 1 - f0;
    const int64_t lastm = a.M - 1 - m0;
#pragma unroll
    for (int u = 0; u < TL::kBlocksA; ++u) {
      const int r = 8 * (wv + TL::NW * u) + r8;
      aoff[u] = static_cast<uint32_t>((r < lastf ? r : lastf) * a.w_rs) + 16 * chunk;
    }
#pragma unroll
    for (int u = 0; u < TL::kBlocksB; ++u) {
      const int r = 8 * (wv + TL::NW * u) + r8;
      boff[u] = static_cast<uint32_t>((r < lastm ? r : lastm) * a.x_rs) + 16 * chunk;
    }
    constexpr int kDwords = St::kScaleRow / 4, kPer = 64 / kDwords;  // dwords a row, rows a block
    const int lane = threadIdx.x & 63, d = lane % kDwords;
#pragma unroll
    for (int u = 0; u < St::kBlocksS; ++u) {
      int block = wv + TL::NW * u;
      if (block > St::kScaleBlocks - 1) block = St::kScaleBlocks - 1;
      const bool isa = block * kPer < TL::FT;
      const int r = block * kPer + lane / kDwords - (isa ? 0 : TL::FT);
      const int64_t last = isa ? lastf : lastm, rr = r < last ? r : last;
      const uint8_t* row = isa ? a.sw + (f0 + rr) * a.sw_rs : a.sx + (m0 + rr) * a.sx_rs;
      const int ahead = RAGGED ? static_cast<int>(reinterpret_cast<uintptr_t>(row) & 3) : 0;
      sp[u] = row - ahead + 4 * d;
      srem[u] = 4 * d < ahead + 8 ? a.K / kGroup + ahead - 4 * d : 0;
    }
  }
  // Copy u of step s, to the stage at LDS byte address `stage`.
  __device__ __forceinline__ void one(int u, int s, int K, uint32_t stage) const {
    const int k = s * kStep;  // byte of the rows
    if (u < TL::kBlocksA + TL::kBlocksB) {
      const bool a = u < TL::kBlocksA;
      const uint8_t* base = (a ? w0 : x0) + k;
      const uint32_t off = a ? aoff[a ? u : 0] : boff[a ? 0 : u - TL::kBlocksA];
      const uint32_t to = stage + (a ? 0 : TL::FT * kStep) + (wv + TL::NW * (a ? u : u - TL::kBlocksA)) * 1024;
      if constexpr (RAGGED) lds_dma16_any(k + 16 * chunk < K / 2 ? base + off : zeros, to);
      else lds_dma16(base, off, to);
    } else {
      const int i = u - TL::kBlocksA - TL::kBlocksB;
      int block = wv + TL::NW * i;
      if (block > St::kScaleBlocks - 1) block = St::kScaleBlocks - 1;
      const uint32_t to = stage + St::kScales + 256 * block;
      if constexpr (RAGGED) lds_dma4_any(8 * s < srem[i] ? sp[i] + 8 * s : zeros, to);
      else lds_dma4_any(sp[i] + 8 * s, to);
    }
  }
  static constexpr int kCopies = TL::kBlocksA + TL::kBlocksB + St::kBlocksS;
};

// Half a stage of a wave's operands: two blocks of 32 columns of each of its rows, lane half lh the blocks
// 4 lh + 2 kk + 0, 1, and the scales of lane half lh's four.
template <class TL, bool RAGGED>
struct Frags {
  using St = Stage<TL, RAGGED>;
  u32x4 a[TL::NF][2], b[TL::NM][2];
  uint32_t sa[TL::NF][RAGGED ? 2 : 1], sb[TL::NM][RAGGED ? 2 : 1];
  static constexpr int kTwo = 2 * (TL::NF + TL::NM), kReads = kTwo + TL::NF + TL::NM;
  __device__ __forceinline__ void read(int i, const uint8_t* st, int fw, int mw, int kk) {
    const int lr = threadIdx.x & 31, lh = (threadIdx.x & 63) >> 5;
    if (i < kTwo) {
      const int c = 4 * lh + 2 * kk + (i & 1), t = i >> 1;
      if (t < TL::NF) a[t][i & 1] = *reinterpret_cast<const u32x4*>(st + swz_byte(fw + 32 * t + lr, c));
      else
        b[t - TL::NF][i & 1] =
            *reinterpret_cast<const u32x4*>(st + TL::FT * kStep + swz_byte(mw + 32 * (t - TL::NF) + lr, c));
      return;
    }
    const int t = i - kTwo;
    const int row = t < TL::NF ? fw + 32 * t + lr : TL::FT + mw + 32 * (t - TL::NF) + lr;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(st + St::kScales + St::kScaleRow * row + 4 * lh);
#pragma unroll
    for (int j = 0; j < (RAGGED ? 2 : 1); ++j) {
      if (t < TL::NF) sa[t][j] = p[j];
      else sb[t - TL::NF][j] = p[j];
    }
  }
};

// The scales of a lane half's four blocks out of the dwords that hold them: `shift` bytes in, those past K left out.
__device__ __forceinline__ uint32_t scale_of(const uint32_t (&d)[1], uint32_t, uint32_t) { return d[0]; }
__device__ __forceinline__ uint32_t scale_of(const uint32_t (&d)[2], uint32_t shift, uint32_t mask) {
  return __builtin_amdgcn_alignbyte(d[1], d[0], shift) & mask;
}

template <class TL>
int64_t tiles_of(const Args& a) {
  return static_cast<int64_t>((a.F + TL::FT - 1) / TL::FT) * ((a.M + TL::MT - 1) / TL::MT);
}

// The loop of the 8-bit product (proj_q8.hip), with steps of 256 columns: workgroups stay and their copies run kStages
// steps ahead across the tiles' ends.
template <typename T, class TL, bool RAGGED, bool STREAM>
__global__ __launch_bounds__(64 * TL::NW) __attribute__((amdgpu_waves_per_eu(TL::kWaves, TL::kWaves))) void tiled_kernel(
    const Args a) {
  using St = Stage<TL, RAGGED>;
  __shared__ __attribute__((aligned(16))) uint8_t smem[TL::kStages * St::kBytes];
  __shared__ __attribute__((aligned(16))) float bias[2][TL::FT];  // of a tile and of the next
  const int nf = (a.F + TL::FT - 1) / TL::FT, nm = static_cast<int>((a.M + TL::MT - 1) / TL::MT), tiles = nf * nm;
  // Groups of eight feature tiles walk the row tiles together, and the workgroups of an XCD take consecutive tiles, so
  // that both operands are read from its L2.
  auto origin = [&](int p, int& f0, int64_t& m0) {
    constexpr int GF = 8;
    const int id = xcd_remap(p, tiles), g = id / (GF * nm), gs = nf - g * GF < GF ? nf - g * GF : GF;
    const int in = id - g * GF * nm;
    f0 = (g * GF + in % gs) * TL::FT;
    m0 = static_cast<int64_t>(in / gs) * TL::MT;
  };
  const int lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5;
  const int wv = wave_id(), fw = wv % TL::WF * (32 * TL::NF), mw = wv / TL::WF * (32 * TL::NM);
  const uint32_t lds0 = lds_addr(smem);
  const int nk = (a.K + kCols - 1) / kCols;

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
  using Fr = Frags<TL, RAGGED>;
  constexpr int kTiles = TL::NF * TL::NM, kReads = Fr::kReads, kCopies = StageCopy<TL, RAGGED>::kCopies;
  auto copy_bias = [&](int f0, int set) {  // 64 features by a wave, copied while the tile's first step runs
    if (!a.bias || 64 * wv >= TL::FT) return;
    const int i = 64 * wv + lane, f = i < a.F - 1 - f0 ? i : a.F - 1 - f0;
    lds_dma4(a.bias + f0, 4 * f, lds_addr(bias[set]) + 256 * wv);
  };
  if (!a.bias && threadIdx.x < TL::FT) bias[0][threadIdx.x] = bias[1][threadIdx.x] = 0.f;
  aim();
#pragma unroll
  for (int i = 0; i < TL::kStages; ++i) {
#pragma unroll
    for (int u = 0; u < kCopies; ++u) copy.one(u, cs, a.K, lds0 + i * St::kBytes);
    advance();
  }
  wait_copies<(TL::kStages - 1) * kCopies>();
  wait_lds();
  barrier();
  Fr lo, hi;
#pragma unroll
  for (int i = 0; i < kReads; ++i) lo.read(i, smem, fw, mw, 0);

  // A step of a wave is 2 kTiles pairs of products, lo's and hi's. In the first kFree the operands of hi are read; then
  // every wave has the whole stage in registers (barrier) and the step kStages on is copied into it, over kTiles pairs.
  // Before hi's products the next step's copies, issued kStages - 1 steps ago, have landed (barrier), and its lo is read
  // during them.
  constexpr int kFree = kTiles / 2;                            // 0: one barrier does for both
  constexpr int kEarly = (kTiles - kFree) * kCopies / kTiles;  // copies issued before the second barrier
  constexpr int kLater = (TL::kStages - 2) * kCopies;          // copies of the steps between the next and that one
  uint32_t b = 0;                                              // byte offset of the step's stage
  int set = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, set ^= 1) {
    int f0;
    int64_t m0;
    origin(tile, f0, m0);
    copy_bias(f0, set);
    uint32_t sha[TL::NF] = {}, shb[TL::NM] = {};  // where in its first dword a row's scales start
    if constexpr (RAGGED) {
#pragma unroll
      for (int t = 0; t < TL::NF; ++t) {
        const int f = f0 + fw + 32 * t + lr;
        sha[t] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.sw) + (f < a.F ? f : a.F - 1) * a.sw_rs) & 3;
      }
#pragma unroll
      for (int t = 0; t < TL::NM; ++t) {
        const int64_t m = m0 + mw + 32 * t + lr;
        shb[t] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.sx) + (m < a.M ? m : a.M - 1) * a.sx_rs) & 3;
      }
    }
    f32x16 acc[TL::NF][TL::NM];
#pragma unroll
    for (int i = 0; i < TL::NF; ++i)
#pragma unroll
      for (int j = 0; j < TL::NM; ++j) acc[i][j] = f32x16{};
    for (int s = 0; s < nk; ++s) {
      const uint32_t stage = __builtin_amdgcn_readfirstlane(lds0 + b);
      const int step = cs;
      uint32_t mask = ~0u;  // the bytes of a lane half's scales that lie before K
      if constexpr (RAGGED) {
        const int n = a.K / kGroup - 8 * s - 4 * lh;
        mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
      }
      auto copies = [&](int j) {  // those of product j past the barrier
#pragma unroll
        for (int u = j * kCopies / kTiles; u < (j + 1) * kCopies / kTiles; ++u) copy.one(u, step, a.K, stage);
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
        const int ti = i / TL::NM, tj = i % TL::NM;
        const uint32_t sa = scale_of(lo.sa[ti], sha[ti], mask), sb = scale_of(lo.sb[tj], shb[tj], mask);
        acc[ti][tj] = mfma_32x32x64<0>(lo.a[ti][0], lo.b[tj][0], acc[ti][tj], sa, sb);
        acc[ti][tj] = mfma_32x32x64<1>(lo.a[ti][1], lo.b[tj][1], acc[ti][tj], sa, sb);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_copies<kLater + (kFree == 0 ? 0 : kEarly)>();
      if (kFree == 0) wait_lds();
      barrier();
      b = b == (TL::kStages - 1) * St::kBytes ? 0 : b + St::kBytes;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (kFree == 0) copies(i);
        else if (i < kFree) copies(kTiles - kFree + i);
        // (after the very last step, of a stage that nothing needs)
#pragma unroll
        for (int r = i * kReads / kTiles; r < (i + 1) * kReads / kTiles; ++r) lo.read(r, smem + b, fw, mw, 0);
        const int ti = i / TL::NM, tj = i % TL::NM;
        const uint32_t sa = scale_of(hi.sa[ti], sha[ti], mask), sb = scale_of(hi.sb[tj], shb[tj], mask);
        acc[ti][tj] = mfma_32x32x64<2>(hi.a[ti][0], hi.b[tj][0], acc[ti][tj], sa, sb);
        acc[ti][tj] = mfma_32x32x64<3>(hi.a[ti][1], hi.b[tj][1], acc[ti][tj], sa, sb);
        __builtin_amdgcn_sched_barrier(0);
      }
      advance();
    }
    if (nk < TL::kStages - 1) {  // the bias's copy is among those that the last wait left
      wait_copies<0>();
      barrier();
    }
#pragma unroll
    for (int n = 0; n < TL::NF; ++n) {
      __builtin_amdgcn_sched_barrier(0);  // the biases of one n at a time: registers
      float bs[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 b4 = *reinterpret_cast<const f32x4*>(bias[set] + fw + 32 * n + 8 * g + 4 * lh);
#pragma unroll
        for (int j = 0; j < 4; ++j) bs[4 * g + j] = b4[j];
      }
#pragma unroll
      for (int t = 0; t < TL::NM; ++t) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[n][t][i] + bs[i];
        store_32x32<T, STREAM>(static_cast<T*>(a.out), a.os, a.M, a.F, m0 + mw + 32 * t, f0 + fw + 32 * n, v);
      }
    }
  }
  wait_copies<0>();
}

// Whether the scale rows are whole dwords and K whole stages.
bool is_ragged(const Args& a) {
  auto odd = [](const uint8_t* p, int64_t rs) { return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(rs)) & 3; };
  return a.K % kCols || odd(a.sx, a.sx_rs) || odd(a.sw, a.sw_rs);
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
  const bool ragged = is_ragged(a);
  if constexpr (TL::FT * TL::MT >= 128 * 128 && TL::kStages == 2) {  // (the others are for small outputs)
    if (a.M * a.F * static_cast<int64_t>(sizeof(T)) > kStreamBytes) return ragged ? with(yes, yes) : with(no, yes);
  }
  ragged ? with(yes, no) : with(no, no);
}

// ---- Few rows -----------------------------------------------------------------------------------------------
// Up to 16 CT rows, where the weights' bytes are the cost: each is read once, straight into the registers of the wave that
// multiplies it. A workgroup computes 16 features for all rows; its waves take the 128-column chunks of K in turns and
// their partial sums are added in the waves' order. On v_mfma_f32_16x16x128_f8f6f4 a lane holds 32 consecutive columns
// of feature (or row) lane % 16, and their scale.
constexpr int kMaxWaves = 16;

template <typename T, int CT>
__global__ __launch_bounds__(64 * kMaxWaves) void few_rows_kernel(const Args a) {
  __shared__ float part[kMaxWaves][CT][16][17];  // [wave][row tile][row][feature]
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4, wave = wave_id(), waves = blockDim.x >> 6;
  const int f0 = blockIdx.x * 16, M = static_cast<int>(a.M), groups = a.K / kGroup;
  const int64_t f = f0 + lr < a.F ? f0 + lr : a.F - 1;  // past the end: not stored
  const uint8_t *wrow = a.w + f * a.w_rs, *wsc = a.sw + f * a.sw_rs, *xrow[CT], *xsc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int64_t m = 16 * t + lr < M ? 16 * t + lr : M - 1;
    xrow[t] = a.x + m * a.x_rs, xsc[t] = a.sx + m * a.sx_rs;
  }
  f32x4 acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = (groups + 3) / 4;
  u32x4 w[2], x[2][CT];
  uint32_t ws[2], xs[2][CT];
  auto load = [&](int c, int buf) {  // zeros past K
    const int g = 4 * c + lq;
    w[buf] = u32x4{0, 0, 0, 0}, ws[buf] = 0;
#pragma unroll
    for (int t = 0; t < CT; ++t) x[buf][t] = u32x4{0, 0, 0, 0}, xs[buf][t] = 0;
    if (g < groups) {
      w[buf] = ld16(wrow + 16 * static_cast<int64_t>(g)), ws[buf] = wsc[g];
#pragma unroll
      for (int t = 0; t < CT; ++t) x[buf][t] = ld16(xrow[t] + 16 * static_cast<int64_t>(g)), xs[buf][t] = xsc[t][g];
    }
  };
  // The loads of a wave's next chunk are in flight while it multiplies this one.
  int c = wave;
  load(c, 0);
  for (; c < chunks; c += 2 * waves) {
    if (c + waves < chunks) load(c + waves, 1);
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = mfma_16x16x128(w[0], x[0][t], acc[t], ws[0], xs[0][t]);
    if (c + waves >= chunks) break;
    if (c + 2 * waves < chunks) load(c + 2 * waves, 0);
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = mfma_16x16x128(w[1], x[1][t], acc[t], ws[1], xs[1][t]);
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
    out[r * a.os + f0 + fo] = cast_out<T>(v + (a.bias ? a.bias[f0 + fo] : 0.f));
  }
}

template <typename T, int CT>
void launch_few_rows(hipStream_t stream, const Args& a) {
  const int chunks = (a.K + 127) / 128;
  hipLaunchKernelGGL((few_rows_kernel<T, CT>), dim3(static_cast<unsigned>((a.F + 15) / 16)),
                     dim3(64 * (chunks < kMaxWaves ? chunks : kMaxWaves)), 0, stream, a);
}

// Which kernel: few rows up to 16 (up to 32 of a narrow product); then tiles by how many the product has for the card's
// CUs.
template <typename T>
void launch(hipStream_t stream, const Args& a) {
  using Small = Tile<64, 64, 2, 2, 3>;
  using Half = Tile<128, 64, 2, 2, 2, 3>;
  using Medium = Tile<128, 128, 2, 2, 2>;
  using Large = Tile<128, 256, 2, 2, 1>;
  const int64_t cus = device_cus(), small = tiles_of<Small>(a), half = tiles_of<Half>(a), medium = tiles_of<Medium>(a);
  if (a.M <= 16) return launch_few_rows<T, 1>(stream, a);
  if (a.M <= 32 && small <= cus / 4) return launch_few_rows<T, 2>(stream, a);
  if (small <= cus && a.K > 4 * kCols) return launch_tiled<T, Tile<64, 64, 2, 2, 1, 4>>(stream, a);
  if (small <= cus) return launch_tiled<T, Small>(stream, a);
  if (half <= cus) return launch_tiled<T, Half>(stream, a);
  if (medium <= 2 * cus) return launch_tiled<T, Medium>(stream, a);
  launch_tiled<T, Large>(stream, a);
}

}  // namespace mx4
}  // namespace hb

using namespace hb;

extern "C" int hb_proj_mx4(hipStream_t stream, const void* x, int64_t x_row_stride, const void* x_scale,
                           int64_t x_scale_row_stride, const void* w, int64_t w_row_stride, const void* w_scale,
                           int64_t w_scale_row_stride, const float* bias, void* out, int out_dtype,
                           int64_t out_row_stride, int64_t M, int K, int F) {
  clear_error();
  const char* what = "proj_mx4";
  if (out_dtype != HB_BF16 && out_dtype != HB_F32 && out_dtype != HB_F16)
    return fail(HB_ERR_DTYPE, "%s: dtype %d is not HB_BF16 (0), HB_F32 (1) or HB_F16 (2)", what, out_dtype);
  if (M < 1 || M > (1 << 21) || F < 1 || F > (1 << 21) || K < mx4::kGroup || K > (1 << 23) || K % mx4::kGroup)
    return fail(HB_ERR_SHAPE, "%s needs 1 <= M, F <= 2^21 and K a multiple of 32 up to 2^23 (M=%lld, K=%d, F=%d)", what,
                static_cast<long long>(M), K, F);
  if (!x || !x_scale || !w || !w_scale || !out)
    return fail(HB_ERR_NULL, "%s: x, x_scale, w, w_scale and out must be non-NULL", what);
  const int es = out_dtype == HB_F32 ? 4 : 2, groups = K / mx4::kGroup;
  auto misaligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  // A tile's rows are addressed by 32-bit offsets from its first.
  auto bad_rows = [&](const void* p, int64_t rs) { return misaligned(p, 16) || rs < K / 2 || rs % 16 || rs > (1 << 22); };
  const char* rows_of = bad_rows(x, x_row_stride) ? "x" : bad_rows(w, w_row_stride) ? "w" : nullptr;
  if (rows_of)
    return fail(HB_ERR_STRIDE, "%s: %s must be 16-byte aligned with a row stride >= K / 2, a multiple of 16 up to 2^22",
                what, rows_of);
  if (x_scale_row_stride < groups || w_scale_row_stride < groups)
    return fail(HB_ERR_STRIDE, "%s: the scales' row strides must be >= K / 32", what);
  if (misaligned(bias, 4)) return fail(HB_ERR_STRIDE, "%s: bias must be 4-byte aligned", what);
  if (misaligned(out, es) || out_row_stride < F)
    return fail(HB_ERR_STRIDE, "%s: out must be aligned to its elements with a row stride >= F", what);
  int st;
  if ((st = check_extent(what, "x", M, x_row_stride, K / 2)) || (st = check_extent(what, "w", F, w_row_stride, K / 2)) ||
      (st = check_extent(what, "x_scale", M, x_scale_row_stride, groups)) ||
      (st = check_extent(what, "w_scale", F, w_scale_row_stride, groups)) ||
      (st = check_extent(what, "out", M, out_row_stride, F)))
    return st;
  const int64_t ob = rows_bytes(M, out_row_stride, F, es);
  if ((st = check_disjoint(what, "out", out, ob, "x", x, rows_bytes(M, x_row_stride, K / 2, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "w", w, rows_bytes(F, w_row_stride, K / 2, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "x_scale", x_scale, rows_bytes(M, x_scale_row_stride, groups, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "w_scale", w_scale, rows_bytes(F, w_scale_row_stride, groups, 1))) ||
      (st = check_disjoint(what, "out", out, ob, "bias", bias, static_cast<int64_t>(F) * 4)))
    return st;
  const mx4::Args a = {static_cast<const uint8_t*>(x), x_row_stride, static_cast<const uint8_t*>(x_scale),
                       x_scale_row_stride, static_cast<const uint8_t*>(w), w_row_stride,
                       static_cast<const uint8_t*>(w_scale), w_scale_row_stride, bias, out, out_row_stride, M, K, F};
  if (out_dtype == HB_BF16) mx4::launch<uint16_t>(stream, a);
  else if (out_dtype == HB_F16) mx4::launch<_Float16>(stream, a);
  else mx4::launch<float>(stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return HB_OK;
}

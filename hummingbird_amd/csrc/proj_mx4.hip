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

// A pointer that is the same in every lane, in scalar registers.
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uintptr_t>(p);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32)));
  return reinterpret_cast<const uint8_t*>(hi << 32 | lo);
}

// ---- Tiled product ------------------------------------------------------------------------------------------
// A workgroup of WF x WM waves computes FT features x MT rows in steps of 256 columns, which stream through kStages LDS
// stages: code rows of 128 bytes whose 16-byte chunks are XOR-swizzled, then the rows' scales. A wave multiplies NF x NM
// tiles of 32 x 32, of one 64-column block after the other, and reads the next block's operands meanwhile.
// The scales are copied for kChunk steps at once, 32 bytes a row, into kBufs buffers of their own: blocks of 32 rows, the
// rows' first 16 bytes and then their second ones, so that 32 rows' reads meet on a bank in twos (as rows of 32 bytes in fours:
// 8249 x 1536 -> 12288 8.5 million conflict cycles, 3.6 so).
// RAGGED: K ends inside two steps, or scale rows that are not aligned to 16 bytes. The scales of two steps then lie in two
// 16-byte pieces, which are copied whole (each holds at least a byte of the row) and read from where they start.
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
  static constexpr int kRows = TL::FT + TL::MT, kBytes = kRows * kStep;
  static constexpr int kChunk = RAGGED ? 2 : 4;  // steps whose scales are copied together
  static constexpr int kScaleBytes = kRows * 32;
  // A chunk's copies start kStages steps before it, when the last reads of the chunk whose buffer it takes are over:
  // kBufs - 1 chunks, of two steps or (RAGGED) one where they are K's last, are kStages - 1 steps at least.
  static constexpr int kBufs = RAGGED ? TL::kStages : (TL::kStages + 2) / 2;
  static constexpr int kScaleBlocks = kScaleBytes / 1024;  // copies; a wave's past the last repeat it
  static constexpr int kBlocksS = (kScaleBlocks + TL::NW - 1) / TL::NW;
  static constexpr int kLds = TL::kStages * kBytes + kBufs * kScaleBytes;
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
  const uint8_t* sp[St::kBlocksS];  // this lane's 16 bytes of the first chunk
  int srem[St::kBlocksS];           // bytes from it to its row's end
  const int wv = wave_id() % TL::NW, r8 = (threadIdx.x & 63) >> 3, chunk = (threadIdx.x & 7) ^ r8 ^ (wv & 1);

  // Aims the copies at the tile of feature f0 and row m0. Rows past an end read the last one; their results are not stored.
  __device__ __forceinline__ void aim(const Args& a, int f0, int64_t m0) {
    w0 = uniform(a.w + f0 * a.w_rs);
    x0 = uniform(a.x + m0 * a.x_rs);
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
    constexpr int kPer = 32;  // rows a block
    const int lane = threadIdx.x & 63, piece = lane / kPer;
#pragma unroll
    for (int u = 0; u < St::kBlocksS; ++u) {
      const int block = scale_block(u);
      const bool isa = block * kPer < TL::FT;
      const int r = block * kPer + lane % kPer - (isa ? 0 : TL::FT);
      const int64_t last = isa ? lastf : lastm, rr = r < last ? r : last;
      const uint8_t* row = isa ? a.sw + (f0 + rr) * a.sw_rs : a.sx + (m0 + rr) * a.sx_rs;
      const int ahead = RAGGED ? static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) : 0;
      sp[u] = row - ahead + 16 * piece;
      srem[u] = a.K / kGroup + ahead - 16 * piece;
    }
  }
  __device__ __forceinline__ int scale_block(int u) const {
    const int block = wv + TL::NW * u;
    return block < St::kScaleBlocks ? block : St::kScaleBlocks - 1;
  }
  // Copy u of step s's codes, to the stage at LDS byte address `stage`.
  __device__ __forceinline__ void one(int u, int s, int K, uint32_t stage) const {
    const int k = s * kStep;  // byte of the rows
    const bool a = u < TL::kBlocksA;
    const uint8_t* base = (a ? w0 : x0) + k;
    const uint32_t off = a ? aoff[a ? u : 0] : boff[a ? 0 : u - TL::kBlocksA];
    const uint32_t to = stage + (a ? 0 : TL::FT * kStep) + (wv + TL::NW * (a ? u : u - TL::kBlocksA)) * 1024;
    if constexpr (RAGGED) lds_dma16_any(k + 16 * chunk < K / 2 ? base + off : zeros, to);
    else lds_dma16(base, off, to);
  }
  // The scales of the chunk that starts at step s to the buffer at LDS byte address `buf`. Pieces past a row's end come from
  // `zeros` (without RAGGED K is a multiple of 512: a piece lies before the end or past it).
  __device__ __forceinline__ void scales(int s, uint32_t buf) const {
#pragma unroll
    for (int u = 0; u < St::kBlocksS; ++u)
      lds_dma16_any(8 * s < srem[u] ? sp[u] + 8 * s : zeros, buf + 1024 * scale_block(u));
  }
  static constexpr int kCopies = TL::kBlocksA + TL::kBlocksB;
};

// A wave's operands of block J of a stage: lane half lh's 32 columns of each of its rows, chunk 4 lh + J.
template <class TL>
struct Block {
  u32x4 a[TL::NF], b[TL::NM];
  static constexpr int kReads = TL::NF + TL::NM;
  __device__ __forceinline__ void read(int t, const uint8_t* st, int fw, int mw, int j) {
    const int lr = threadIdx.x & 31, lh = (threadIdx.x & 63) >> 5, c = 4 * lh + j;
    if (t < TL::NF) a[t] = *reinterpret_cast<const u32x4*>(st + swz_byte(fw + 32 * t + lr, c));
    else b[t - TL::NF] = *reinterpret_cast<const u32x4*>(st + TL::FT * kStep + swz_byte(mw + 32 * (t - TL::NF) + lr, c));
  }
};

// The scales of a step: of lane half lh's four blocks, a byte each.
template <class TL, bool RAGGED>
struct Scales {
  using St = Stage<TL, RAGGED>;
  static constexpr int kDwords = RAGGED ? 2 : 1;
  uint32_t raw[TL::NF + TL::NM][kDwords];
  // From the buffer `buf`, of the chunk's step `at`; `ahead`: where in its first piece the row starts.
  __device__ __forceinline__ void read(int t, const uint8_t* buf, int at, int fw, int mw, uint32_t ahead) {
    const int lr = threadIdx.x & 31, lh = (threadIdx.x & 63) >> 5;
    const int first = t < TL::NF ? fw + 32 * t : TL::FT + mw + 32 * (t - TL::NF);  // of its block's rows
#pragma unroll
    for (int j = 0; j < kDwords; ++j) {
      const int o = 8 * at + 4 * lh + (RAGGED ? static_cast<int>(ahead & ~3u) : 0) + 4 * j;  // byte of the row's 32
      raw[t][j] = *reinterpret_cast<const uint32_t*>(buf + 32 * first + 512 * (o >> 4) + 16 * lr + (o & 15));
    }
  }
  // Out of the dwords that hold them, those past K (`mask`) left out.
  __device__ __forceinline__ uint32_t get(int t, uint32_t ahead, uint32_t mask) const {
    if constexpr (RAGGED) return __builtin_amdgcn_alignbyte(raw[t][1], raw[t][0], ahead & 3) & mask;
    else return raw[t][0];
  }
};

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
  using St = Stage<TL, RAGGED>;
  __shared__ __attribute__((aligned(16))) uint8_t smem[St::kLds];
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
  constexpr uint32_t kScales0 = TL::kStages * St::kBytes, kScalesEnd = St::kLds;
  const int nk = (a.K + kCols - 1) / kCols;

  // What is copied next: step `cs` of tile `ct` (in the order of p), its scales to the buffer at `cbuf`.
  StageCopy<TL, RAGGED> copy;
  int ct = blockIdx.x, cs = 0;
  uint32_t cbuf = kScales0;
  auto next_buf = [](uint32_t x) { return x + St::kScaleBytes == kScalesEnd ? kScales0 : x + St::kScaleBytes; };
  auto aim = [&]() {
    int f0;
    int64_t m0;
    origin(ct, f0, m0);
    copy.aim(a, f0, m0);
  };
  auto advance = [&]() {
    if (++cs < nk) {
      if (cs % St::kChunk == 0) cbuf = next_buf(cbuf);
      return;
    }
    cs = 0;
    cbuf = next_buf(cbuf);
    if (ct + static_cast<int>(gridDim.x) >= tiles) return;
    ct += gridDim.x;
    aim();
  };
  constexpr int kTiles = TL::NF * TL::NM, kReads = Block<TL>::kReads, kCopies = StageCopy<TL, RAGGED>::kCopies;
  // A step has four blocks of kTiles products. With one product a block (kWhole) a step's products take less time than a read
  // from LDS, so all of a step's operands are in registers when it begins: the barrier comes first, the stage is free for
  // the step kStages on, and each block's registers take the next step's operands behind its product (in a graph, 154 x
  // 4096 -> 1024: 9.1 -> 8.6 us, 400 x 6144 -> 1536: 12.6 -> 11.7).
  // With more, the reads run a block ahead of the products. When a step's last block is in registers everywhere and the next
  // step's copies have landed (the one barrier of a step, before the last block's products), the stage is free: the step
  // kStages on is copied into it, kFirst copies among the last block's products and the others among the next step's first.
  constexpr bool kWhole = kTiles == 1;
  constexpr int kFirst = kWhole ? kCopies : 3 * kCopies / 4;
  auto chunk = [&]() {
    if (cs % St::kChunk == 0) copy.scales(cs, __builtin_amdgcn_readfirstlane(lds0 + cbuf));
  };
  aim();
#pragma unroll
  for (int i = 0; i < TL::kStages; ++i) {
#pragma unroll
    for (int u = 0; u < (i == TL::kStages - 1 ? kFirst : kCopies); ++u) {
      if (u == 0 && (kWhole || i < TL::kStages - 1)) chunk();
      copy.one(u, cs, a.K, lds0 + i * St::kBytes);
    }
    if (kWhole || i < TL::kStages - 1) advance();
  }
  wait_copies<(TL::kStages - 2) * kCopies + kFirst>();
  wait_lds();
  barrier();
  uint32_t ahead[kReads] = {};  // where in its first piece a row's scales start, of the tile whose scales are read next
  auto find_ahead = [&](int tile) {
    if constexpr (RAGGED) {
      int f0;
      int64_t m0;
      origin(tile, f0, m0);
#pragma unroll
      for (int t = 0; t < kReads; ++t) {
        const int f = f0 + fw + 32 * t + lr;
        const int64_t m = m0 + mw + 32 * (t - TL::NF) + lr;
        const uint64_t at = t < TL::NF
                                ? reinterpret_cast<uintptr_t>(a.sw) + static_cast<int64_t>(f < a.F ? f : a.F - 1) * a.sw_rs
                                : reinterpret_cast<uintptr_t>(a.sx) + (m < a.M ? m : a.M - 1) * a.sx_rs;
        ahead[t] = static_cast<uint32_t>(at) & 15;
      }
    }
  };
  find_ahead(blockIdx.x);
  uint32_t sbuf = kScales0;  // the buffer of the next scales
  Block<TL> blk[kWhole ? 4 : 2];
  Scales<TL, RAGGED> next;
#pragma unroll
  for (int i = 0; i < kReads; ++i) {
#pragma unroll
    for (int j = 0; j < (kWhole ? 4 : 1); ++j) blk[j].read(i, smem, fw, mw, j);
    next.read(i, smem + sbuf, 0, fw, mw, ahead[i]);
  }

  uint32_t b = 0;                                                                     // byte offset of the step's stage
  uint32_t late = __builtin_amdgcn_readfirstlane(lds0 + (TL::kStages - 1) * St::kBytes);  // the stage whose copies go on
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int f0;
    int64_t m0;
    origin(tile, f0, m0);
    f32x16 acc[TL::NF][TL::NM];
    auto step = [&](int s, auto first) {
      if constexpr (kWhole) {
        wait_copies<(TL::kStages - 2) * kCopies>();
        wait_lds();
        barrier();
      }
      chunk();  // with the copies that go on among the first block's products
      uint32_t mask = ~0u;  // the bytes of a lane half's scales that lie before K
      if constexpr (RAGGED) {
        const int n = a.K / kGroup - 8 * s - 4 * lh;
        mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
      }
      uint32_t sc[kReads];
#pragma unroll
      for (int t = 0; t < kReads; ++t) sc[t] = next.get(t, ahead[t], mask);
      // the next step's scales: the chunk's next ones, or a new chunk's first
      const bool over = s + 1 == nk;
      const int at = over ? 0 : (s + 1) % St::kChunk;
      if (!at) sbuf = next_buf(sbuf);
      if (RAGGED && over) find_ahead(tile + gridDim.x < static_cast<unsigned>(tiles) ? tile + gridDim.x : tile);
      const uint8_t* const here = smem + b;
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + b);
      b = b == (TL::kStages - 1) * St::kBytes ? 0 : b + St::kBytes;
      auto block = [&](auto which) {
        constexpr int J = decltype(which)::value;
        if constexpr (kWhole) {
          if constexpr (J == 0) {
#pragma unroll
            for (int u = 0; u < kCopies; ++u) copy.one(u, cs, a.K, to);
            advance();
          }
          acc[0][0] = mfma_32x32x64<J>(blk[J].a[0], blk[J].b[0], J == 0 && decltype(first)::value ? f32x16{} : acc[0][0],
                                       sc[0], sc[1]);
#pragma unroll
          for (int r = 0; r < kReads; ++r) {
            blk[J].read(r, smem + b, fw, mw, J);
            if constexpr (J == 0) next.read(r, smem + sbuf, at, fw, mw, ahead[r]);
          }
          return;
        }
        if constexpr (J == 3) {
          wait_copies<(TL::kStages - 2) * kCopies>();
          wait_lds();
          barrier();
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
#pragma unroll
          for (int r = i * kReads / kTiles; r < (i + 1) * kReads / kTiles; ++r) {
            // (after the very last step, of a stage that nothing needs)
            blk[(J + 1) & 1].read(r, J == 3 ? smem + b : here, fw, mw, (J + 1) & 3);
            if constexpr (J == 3) next.read(r, smem + sbuf, at, fw, mw, ahead[r]);
          }
          if constexpr (J == 0 || J == 3) {
            constexpr int kFrom = J == 3 ? 0 : kFirst, kNum = J == 3 ? kFirst : kCopies - kFirst;
#pragma unroll
            for (int u = i * kNum / kTiles; u < (i + 1) * kNum / kTiles; ++u)
              copy.one(kFrom + u, cs, a.K, J == 3 ? to : late);
          }
          const int ti = i / TL::NM, tj = i % TL::NM;
          acc[ti][tj] = mfma_32x32x64<J>(blk[J & 1].a[ti], blk[J & 1].b[tj],
                                         J == 0 && decltype(first)::value ? f32x16{} : acc[ti][tj], sc[ti],
                                         sc[TL::NF + tj]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (J == 0) advance();
      };
      block(std::integral_constant<int, 0>{});
      block(std::integral_constant<int, 1>{});
      block(std::integral_constant<int, 2>{});
      block(std::integral_constant<int, 3>{});
      late = to;
    };
    // the first step's products start from zero (8249 x 1536 -> 12288: 116 us with registers to clear, 114 so)
    step(0, std::true_type{});
#pragma unroll 1
    for (int s = 1; s < nk; ++s) step(s, std::false_type{});
#pragma unroll
    for (int n = 0; n < TL::NF; ++n) {
      __builtin_amdgcn_sched_barrier(0);  // the biases of one n at a time: registers
      float bs[16] = {};
      if (a.bias) {
        const int fn = f0 + fw + 32 * n;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int f = fn + 8 * g + 4 * lh;
          if (fn + 32 <= a.F) {
            const f32x4 b4 = *reinterpret_cast<const f32x4_align4*>(a.bias + f);
#pragma unroll
            for (int j = 0; j < 4; ++j) bs[4 * g + j] = b4[j];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) bs[4 * g + j] = a.bias[f + j < a.F ? f + j : a.F - 1];
          }
        }
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

// Whether K ends inside two stages, or the scale rows are not 16-byte aligned.
bool is_ragged(const Args& a) {
  auto odd = [](const uint8_t* p, int64_t rs) { return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(rs)) & 15; };
  return a.K % 512 || odd(a.sx, a.sx_rs) || odd(a.sw, a.sw_rs);
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

// Which kernel, as measured (us, of which a call's host part is 7.7; K = 1536 unless said). In order:
//   few rows  up to 16 rows, and up to 32 of a narrow product (24 x 1536, K = 6144: 9.5 against 11.0 Small);
//   Small     up to 3/4 Medium tiles a CU (1422 x 1536, K = 6144: 18.8 against 21.3; but 2584 x 1536, K = 6144: 30.9 against
//             23.1), with three stages where a CU has one such tile and K is 4096 or more (400 x 1536, K = 6144, in a graph:
//             11.5 against 12.2; 333 x 1001, K = 1056: 6.1 and 5.9);
//   Huge      K of 4096 and more, and a tile for half of the CUs: eight waves that share their copies and read a quarter
//             less from LDS (8192^3: 245 against 316, 20000 x 4096 -> 1536: 69 and 79, 3000 x 6144 -> 3000: 42 and 48); from
//             K = 1536 on where they fill their rounds to seven eighths (8249 x 12288: 115 against 119, 5168 x 12288: 66 and
//             73; but after a norm, at a higher clock, 5168 x 7680, 630 tiles: 56 and 53, 2584 x 12288, 528: 42.5 and 37.9), as
//             one workgroup has the CU and little runs beside its epilogue (8192 x 512 -> 8192: 53 and 40);
//   Medium    the rest, two workgroups a CU, or one of eight waves where that is all there is (in a graph, 2584 x 1536: 9.3
//             against 9.7; 1422 x 2600: 9.3 and 9.6) (against 128 x 64 tiles 2584 x 12288: 42.1 and 48.6, 5168 x 7680: 49.7 and 58.7).
template <typename T>
void launch(hipStream_t stream, const Args& a) {
  using Small = Tile<64, 64, 2, 2, 3>;
  using Medium = Tile<128, 128, 2, 2, 2>;
  using Huge = Tile<256, 256, 4, 2, 2>;
  const int64_t cus = device_cus(), small = tiles_of<Small>(a);
  if (a.M <= 16) return launch_few_rows<T, 1>(stream, a);
  if (a.M <= 32 && small <= cus / 4) return launch_few_rows<T, 2>(stream, a);
  if (small <= cus && a.K >= 4096) return launch_tiled<T, Tile<64, 64, 2, 2, 1, 3>>(stream, a);
  if (tiles_of<Medium>(a) <= cus * 3 / 4) return launch_tiled<T, Small>(stream, a);
  const int64_t huge = tiles_of<Huge>(a), places = (huge + cus - 1) / cus * cus;
  if (a.K >= 4096 ? huge >= cus / 2 : a.K >= 1536 && huge >= places * 7 / 8) return launch_tiled<T, Huge>(stream, a);
  if (tiles_of<Medium>(a) <= cus) return launch_tiled<T, Tile<128, 128, 4, 2, 2>>(stream, a);
  launch_tiled<T, Medium>(stream, a);
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

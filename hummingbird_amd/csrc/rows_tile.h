// Pieces of the products of quantised rows (proj_q8.hip, proj_mx4.hip): tiles of 128-byte rows in LDS, their copies and
// waits, and the stores of a 32 x 32 tile of results.
#pragma once

#include "common.h"
#include "tiles.h"

namespace hb {

// Outputs of more bytes than half of the last cache (256 MB) are stored past it: what reads them next would not find
// them there, and they would drive the operands out (8249 x 1536 -> 12288, 203 MB: 172 -> 160 us). Smaller ones stay:
// without, the denoiser's 120 s render, whose norms read them at once, takes 40.6 ms instead of 40.0.
constexpr int64_t kStreamBytes = int64_t(128) << 20;

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;  // bytes of a row per stage

// As lds_dma16 with 4 bytes per lane: 256 bytes at LDS byte address `lds`.
__device__ __forceinline__ void lds_dma4(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(voff), "s"(sbase) : "m0");
}

// As lds_dma16 with an address per lane.
__device__ __forceinline__ void lds_dma16_any(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "m0");
}

// Byte of logical 16-byte chunk `chunk` of row `row` in a stage: the reads of a fragment (one chunk of consecutive
// rows) then spread over the banks.
__device__ __forceinline__ int swz_byte(int row, int chunk) {
  return row * kStep + 16 * (chunk ^ (row & 7) ^ ((row >> 3) & 1));
}

// All but the newest N of this wave's copies have landed (older loads and stores too).
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// This wave's LDS reads and writes are done.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What a copy reads in the place of columns past the last one.
__device__ __attribute__((aligned(16))) const uint8_t zeros[16] = {};

template <typename T>
__device__ __forceinline__ T cast_out(float v);
template <>
__device__ __forceinline__ uint16_t cast_out<uint16_t>(float v) { return f2bf(v); }
template <>
__device__ __forceinline__ _Float16 cast_out<_Float16>(float v) { return static_cast<_Float16>(v); }
template <>
__device__ __forceinline__ float cast_out<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<uint16_t>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<_Float16>(float lo, float hi) { return F16Io::pack2(lo, hi); }

// A lane half's registers exchanged: `x`'s upper half of the wave (or of each 32 lanes) against `y`'s lower one.
__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = r[0], y = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {
  const u32x2 r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  x = r[0], y = r[1];
}

// 16 bytes of consecutive results from feature f of a row on, those past the last feature left out. Rows of any stride and
// width: the 16-byte store takes any alignment of its elements.
// STREAM: past the caches (see kStreamBytes).
typedef u32x4 u32x4_align2 __attribute__((aligned(2)));
template <bool STREAM, typename T>
__device__ __forceinline__ void store16(T* row, int f, int F, u32x4 v) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));
  if (f + N <= F) {
    u32x4_align2* p = reinterpret_cast<u32x4_align2*>(row + f);
    if constexpr (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
  } else if (f < F) {
#pragma unroll
    for (int j = 0; j < N - 1; ++j) {
      if (f + j >= F) continue;
      if constexpr (sizeof(T) == 4) row[f + j] = __uint_as_float(v[j]);
      else row[f + j] = __builtin_bit_cast(T, static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1))));
    }
  }
}

// The results of a 32 x 32 tile: `v`, in registers 4 g .. 4 g + 3, features 8 g + 4 lh .. + 3 of row lr of the tile at
// feature f0 and row m0, for lane (lr, lh). They leave in stores of 16 rows of 64 bytes: for 16-bit types the wave's
// halves exchange so that a lane holds eight consecutive features, and then its 16-lane rows so that four lanes hold 64
// bytes of a row (through LDS a tile waits for its own round trip: 8-bit 5168 x 6144 -> 1536 54 against 43 us).
template <typename T, bool STREAM>
__device__ __forceinline__ void store_32x32(T* out, int64_t os, int64_t M, int F, int64_t m0, int f0,
                                            const float (&v)[16]) {
  const int lr = threadIdx.x & 31, lh = (threadIdx.x & 63) >> 5;
  if constexpr (sizeof(T) == 4) {
    uint32_t w[4][4];  // [g]: features 8 g + 4 lh .. + 3
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[g][j] = __float_as_uint(v[4 * g + j]);
#pragma unroll
    for (int p = 0; p < 2; ++p)  // 64 bytes of a row: groups 2 p and 2 p + 1
#pragma unroll
      for (int j = 0; j < 4; ++j) swap16(w[2 * p][j], w[2 * p + 1][j]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // rows 16 (q % 2) .. of the tile
      const int64_t m = m0 + 16 * (q & 1) + (lr & 15);
      const int f = f0 + 16 * (q >> 1) + 8 * (lr >> 4) + 4 * lh;
      if (m < M) store16<STREAM>(out + m * os, f, F, u32x4{w[q][0], w[q][1], w[q][2], w[q][3]});
    }
  } else {
    uint32_t w[4][2];  // [g]: features 8 g + 4 lh .. + 3
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      w[g][0] = pack2<T>(v[4 * g], v[4 * g + 1]);
      w[g][1] = pack2<T>(v[4 * g + 2], v[4 * g + 3]);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)  // lane half lh: the eight features of group 2 p + lh
#pragma unroll
      for (int j = 0; j < 2; ++j) swap32(w[2 * p][j], w[2 * p + 1][j]);
#pragma unroll
    for (int p = 0; p < 2; ++p)  // rows 16 p .. of the tile, 16 lanes of groups 0, 1 and 16 of 2, 3 in each half
#pragma unroll
      for (int j = 0; j < 2; ++j) swap16(w[p][j], w[2 + p][j]);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t m = m0 + 16 * p + (lr & 15);
      const int f = f0 + 16 * (lr >> 4) + 8 * lh;
      if (m < M)
        store16<STREAM>(out + m * os, f, F,
                        u32x4{w[2 * p][0], w[2 * p][1], w[2 * p + 1][0], w[2 * p + 1][1]});
    }
  }
}

}  // namespace hb

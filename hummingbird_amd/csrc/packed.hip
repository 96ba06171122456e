// Attention over packed sequences for gfx950 (MI355X): queries of N sequences one after the other in q, the keys of each in
// k and v, H heads of queries to G of keys.
//
//   out[t, h] = sum_b softmax_b(scale q[t, h] . k[b, h / gs]) v[b, h / gs],   gs = H / G,
//
// over the keys b of t's sequence, those at or before t's place at the end of them when `causal`. A row with no key, or
// with nothing but scores of minus infinity, is zero.
//
// A workgroup computes a tile of rows of one sequence for one head of keys; a row is one query's one head, the gs heads that
// share the keys next to each other, so that a tile reads its keys once whatever gs is and one new token fills gs rows.
// Keys pass through LDS in tiles of KT, two stages, by global_load_lds; a wave holds 32 NCT rows as MFMA columns:
//   S^T = K Q^T, P = exp2(c S^T - m) with the running maximum m, O^T += V^T P^T,
// so that the probabilities go from the accumulators of S^T into the operands of O^T as they are (attn_tile.h), and
// statistics are a lane's own but for the exchange with its other half. 16-bit inputs multiply on their own type's cores,
// with P rounded to it (its sum is of the rounded values): against fp64 an output of norm 1 is off by 2.3e-3 in bf16 and
// 2.8e-4 in half, where its own rounding is 1.7e-3 and 2.1e-4. (P in two parts, the second what the first leaves, gives the
// latter two but takes 41 % longer: 496 -> 700 us and 50 -> 70 in the first two cases below.) fp32 on the fp32 cores with P in
// fp32. Statistics and sums are fp32.
//
// Bound by the matrix cores and, at 64 dims, the exponentials beside them: bf16, 8249 and 7001 tokens, causal, 16 heads of
// 128 to 4 494 us (1.03 PFLOP/s), 4 x 1300 tokens, 16 heads of 64 43 us (670 TFLOP/s); one new token by the keys' bytes: 16
// sequences, 287 MB 65 us (4.4 TB/s).
//
// The lengths are read on the device: the grid has a slot for every tile that the rows could need (a sequence wastes less
// than one), and each workgroup finds its sequence in the offsets; no launch waits for the host to know them. The search is
// linear, 64 sequences a turn, and of thousands of short ones it is most of the time (prompts of 20 to 200 tokens, 4 heads of
// 64: 512 of them 48 us, 4096 975, 16384 12400).
#include <cmath>
#include <type_traits>

#include "api.h"
#include "attn_tile.h"
#include "common.h"
#include "tiles.h"

namespace hb {
namespace packed {

struct Args {
  const uint8_t *q, *k, *v;                    // strides in bytes, of tokens and of heads
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  uint8_t* out;
  int64_t o_ts, o_hs;
  const int *off, *koff, *klen;                // N + 1 offsets of queries and of keys; N lengths of keys, or null
  int causal, zero_rest;
  float c;                                     // scale log2(e)
  int T, Tk, N, H, G, gs;
  int slots, splits;                           // tiles of rows, parts of the keys
  float* part_o;                               // splits > 1: (splits, T, H, D) sums, not yet divided
  float* part_ml;                              // and (splits, T, H, 2) maxima and totals
};

// The element type's arithmetic. KT: keys per LDS tile.
template <class IO>
struct E16 {
  static constexpr int ES = 2, KT = 64;
  using Io = IO;
};
struct E32 {
  static constexpr int ES = 4, KT = 32;
};

__device__ __forceinline__ int clamp_to(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

struct Tile {
  bool found;
  int index;       // of the sequence's tiles, or of the slots without one
  int idle;        // slots without a tile
  int q0, lq;      // the sequence's first query and queries
  int k0, lk;      // and keys
};

// Slot u's tile of R rows. Lane i of a wave looks at sequence 64 n + i. `sorted`: up to 64 sequences in the order of their
// lengths, the longest first.
__device__ __forceinline__ Tile find_tile(const Args& a, int u, int R, bool sorted) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int i0 = 0; i0 < a.N; i0 += 64) {
    const int i = i0 + lane;
    int number = i, q0 = 0, lq = 0;
    if (i < a.N) {
      q0 = clamp_to(a.off[i], 0, a.T);
      lq = clamp_to(a.off[i + 1], q0, a.T) - q0;
    }
    if (sorted) {
      int rank = 0;
      for (int j = 0; j < a.N; ++j) {
        const int other = __builtin_amdgcn_readlane(lq, j);
        rank += other > lq || (other == lq && j < lane);
      }
      if (lane >= a.N) rank = lane;  // 0 to N - 1 are the sequences'
      number = __builtin_amdgcn_ds_permute(4 * rank, number);
      q0 = __builtin_amdgcn_ds_permute(4 * rank, q0);
      lq = __builtin_amdgcn_ds_permute(4 * rank, lq);
    }
    const int tiles = static_cast<int>((static_cast<int64_t>(lq) * a.gs + R - 1) / R);
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(upto, d, kWave);
      if (lane >= d) upto += x;
    }
    const uint64_t past = __ballot(before + upto > u);
    if (past) {
      const int who = __ffsll(static_cast<unsigned long long>(past)) - 1;
      Tile t;
      t.found = true;
      const int seq = __builtin_amdgcn_readfirstlane(__shfl(number, who, kWave));
      t.q0 = __builtin_amdgcn_readfirstlane(__shfl(q0, who, kWave));
      t.lq = __builtin_amdgcn_readfirstlane(__shfl(lq, who, kWave));
      const int n = __builtin_amdgcn_readfirstlane(__shfl(tiles, who, kWave));
      t.index = u - before - (__builtin_amdgcn_readfirstlane(__shfl(upto, who, kWave)) - n);
      if (a.causal) t.index = n - 1 - t.index;  // the longest first
      t.k0 = clamp_to(a.koff[seq], 0, a.Tk);
      t.lk = clamp_to(a.koff[seq + 1], t.k0, a.Tk) - t.k0;
      if (a.klen) t.lk = clamp_to(a.klen[seq], 0, t.lk);
      t.idle = 0;
      return t;
    }
    before += __builtin_amdgcn_readfirstlane(__shfl(upto, 63, kWave));
  }
  return Tile{false, u - before, a.slots - before, 0, 0, 0, 0};
}

// Byte of logical 16-byte chunk `chunk` of row `row` of a K or V tile, such that the reads spread over the banks: K's of one
// chunk of 32 consecutive rows; V's, transposing ones of 64 bytes of 8 rows or (fp32) of 128 bytes of rows 4 apart.
template <class E, int D>
__device__ __forceinline__ int k_byte(int row, int chunk) {
  constexpr int RB = D * E::ES;
  if constexpr (RB == 128) return row * RB + 16 * (chunk ^ (row & 7) ^ ((row >> 3) & 1));
  else return row * RB + 16 * (chunk ^ (row & 15));
}
template <class E, int D>
__device__ __forceinline__ int v_chunk(int row, int chunk) {
  if constexpr (E::ES == 4) return chunk ^ (8 * ((row >> 2) & 1));
  else if constexpr (D == 64) return chunk ^ (4 * ((row >> 1) & 1));
  else return chunk ^ (4 * (row & 3));
}

template <class E, int D>
struct Lds {
  static constexpr int kTile = E::KT * D * E::ES;  // bytes of a K or a V tile
  static constexpr int kStage = 2 * kTile;
};

// The copies of a key tile by one of NW waves: 1 KB blocks wv, wv + NW, ... of K, then of V.
template <class E, int D, int NW>
struct KeyCopy {
  static constexpr int RB = D * E::ES, kRows = 1024 / RB, kBlocks = E::KT * RB / 1024 / NW;
  const uint8_t *k, *v;
  uint32_t koff[kBlocks], voff[kBlocks];
  int lk;
  int64_t k_ts, v_ts;

  __device__ __forceinline__ int row(int u) const {
    return kRows * (wave_id() % NW + NW * u) + (threadIdx.x & 63) / (64 / kRows);
  }
  __device__ __forceinline__ void offsets(int u, int r, uint32_t& ko, uint32_t& vo) const {
    const int chunk = threadIdx.x & (64 / kRows - 1), at = row(u);
    ko = static_cast<uint32_t>(r * k_ts) + (k_byte<E, D>(at, chunk) - at * RB);
    vo = static_cast<uint32_t>(r * v_ts) + 16 * v_chunk<E, D>(at, chunk);
  }
  __device__ __forceinline__ KeyCopy(const Args& a, const Tile& t, int g)
      : k(a.k + t.k0 * a.k_ts + g * a.k_hs), v(a.v + t.k0 * a.v_ts + g * a.v_hs), lk(t.lk), k_ts(a.k_ts), v_ts(a.v_ts) {
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) offsets(u, row(u), koff[u], voff[u]);
  }
  // The keys from k0 on into the stage at LDS byte address `stage`; past the last key, that one again (it is masked).
  __device__ __forceinline__ void operator()(int k0, uint32_t stage) const {
    const uint8_t *kb = k + k0 * k_ts, *vb = v + k0 * v_ts;
    const int wv = wave_id() % NW;
    const bool whole = k0 + E::KT <= lk;
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
      uint32_t ko = koff[u], vo = voff[u];
      if (!whole) {
        const int r = row(u), last = lk - 1 - k0;
        offsets(u, r < last ? r : last, ko, vo);
      }
      lds_dma16(kb, ko, stage + (wv + NW * u) * 1024);
      lds_dma16(vb, vo, stage + Lds<E, D>::kTile + (wv + NW * u) * 1024);
    }
  }
};

template <class IO>
__device__ __forceinline__ float add_pair(uint32_t p, float acc);
template <>
__device__ __forceinline__ float add_pair<Bf16Io>(uint32_t p, float acc) { return add_bf16_pair(p, acc); }
template <>
__device__ __forceinline__ float add_pair<F16Io>(uint32_t p, float acc) {
  const uint32_t ones = 0x3c003c00u;
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), __builtin_bit_cast(f16x2, ones), acc, false);
}

// V^T for dims 32 dt + lr and keys {16 g + 8 (j / 4) + 4 lh + j % 4 : j < 8}, by transposing reads (attn_tile.h's v_frag on
// swizzled rows).
template <class E, int D>
__device__ __forceinline__ u32x4 v_operand(const uint8_t* sV, int dt, int g) {
  const int lane = threadIdx.x & 63, grp = lane >> 4, m = lane & 15;
  const int row = 16 * g + 4 * (grp >> 1) + (m >> 2), chunk = 4 * dt + 2 * (grp & 1) + ((m & 3) >> 1);
  const uint8_t* p = sV + row * (2 * D) + 8 * (m & 1);
  lds_i16x4* p0 = (lds_i16x4*)(p + 16 * v_chunk<E, D>(row, chunk));
  lds_i16x4* p1 = (lds_i16x4*)(p + 8 * (2 * D) + 16 * v_chunk<E, D>(row + 8, chunk));
  const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p0);
  const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p1);
  const u32x2 ux = __builtin_bit_cast(u32x2, x), uy = __builtin_bit_cast(u32x2, y);
  return u32x4{ux[0], ux[1], uy[0], uy[1]};
}

// How a tile's rows are computed. kPlain takes every sum as it comes. Rows that come out with a NaN or in need of range
// (Rows::again) are computed again by themselves: kApart the same way but that a NaN or an infinity in the values of a key
// reaches only the rows that see it (else its product with their probability of zero is a NaN), and those that still are out
// of range kExact, from the largest score of each row. Both are rare, and the other rows keep what they have: no row's bits
// depend on its neighbours, or on keys that it does not see.
enum Pass { kPlain, kApart, kExact };

// The rows of a wave, NCT times 32 of them, MFMA columns: what it holds between key tiles.
template <class E, int D, int NCT>
struct Rows {
  static constexpr int RT = E::KT / 32, kQ = D * E::ES / 32;  // 16-byte pieces of a query per lane
  u32x4 q[NCT][kQ];
  f32x16 o[NCT][D / 32];
  float m[NCT], l[NCT];
  int lim[NCT];  // keys that this lane's row sees
  uint64_t taken[NCT] = {};  // which of o's values took a NaN or an infinity of V's in the rows computed again: 16 dt + i

  __device__ __forceinline__ void clear(int ct) {
    m[ct] = -INFINITY, l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[ct][dt] = f32x16{};
  }
  // Clears the rows that are to be computed again, and lets the others see no key, so that they stay as they are. Whether this
  // wave has one. They are those with a NaN, a total of 2^100 or more (the whole row's, of both halves of the wave) or a sum of
  // 2^120 or more that it did not take from V, so that what is added to the others later (the parts' totals and sums) stays in
  // range; and of the rows that see a key those with a reference of 2^24 or more, whose rounding is whole binary orders of
  // every probability, or of minus infinity. `begin`: the first key.
  __device__ __forceinline__ bool again(int begin) {
    const int lane = threadIdx.x & 63;
    bool any = false;
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      bool found = !(l[ct] + __shfl_xor(l[ct], 32, kWave) < 0x1p100f) || (begin < lim[ct] && !(fabsf(m[ct]) < 0x1p24f));
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) found |= !(fabsf(o[ct][dt][i]) < 0x1p120f) && !(taken[ct] >> (16 * dt + i) & 1);
      const uint64_t lanes = __ballot(found);
      any |= lanes != 0;
      if (((lanes >> 32 | lanes) >> (lane & 31)) & 1) clear(ct);
      else lim[ct] = 0;
    }
    return any;
  }

  // The scores of 32 RT keys.
  __device__ __forceinline__ void scores(const uint8_t* sK, f32x16 (&sc)[NCT][RT]) const {
    const int lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) sc[ct][rt] = f32x16{};
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(sK + k_byte<E, D>(32 * rt + lr, 2 * i + lh));
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          if constexpr (E::ES == 2) {
            sc[ct][rt] = mfma_io_32x32x16<typename E::Io>(kf, q[ct][i], sc[ct][rt]);
          } else {
            const f32x4 x = __builtin_bit_cast(f32x4, kf), y = __builtin_bit_cast(f32x4, q[ct][i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[ct][rt] = mfma_f32_32x32x2(x[j], y[j], sc[ct][rt]);
          }
        }
      }
    }
  }

  // The scores' probabilities: 16-bit ones in p, fp32 ones in the scores' place. The reference m is a row's maximum over the
  // first tile, and follows the maximum only where that has passed it by 2^kSlack: larger probabilities lose nothing while
  // they are in range, and o is seldom multiplied. bf16 ones are to 2^127: the maximum of the tiles after the first is not
  // looked at (causal, 8192 tokens, 24 heads of 64: 246 -> 233 us).
  static constexpr bool kWide = std::is_same<E, E16<Bf16Io>>::value;
  static constexpr float kSlack = kWide ? 100.f : 8.f;
  __device__ __forceinline__ void softmax(int ct, f32x16 (&sc)[RT], u32x4 (&p)[RT][2], int k0, float c, bool masked,
                                          bool first) {
    const int lh = (threadIdx.x & 63) >> 5;
    if (masked) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[rt][r] = k0 + acc_key(rt, r, lh) < lim[ct] ? sc[rt][r] : -INFINITY;
    }
    if (!kWide || first) {
      float top = -INFINITY;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[rt][r]);
      const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * c;
      const bool passed = top > m[ct] + kSlack;
      if (__any(passed)) {
        const float alpha = passed ? fast_exp2(m[ct] - top) : 1.f;
        m[ct] = passed ? top : m[ct];
        l[ct] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) o[ct][dt] *= alpha;
      }
    }
    const float base = m[ct] == -INFINITY ? 0.f : m[ct];  // every key so far masked: nothing to add up
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float e0 = fast_exp2(__fmaf_rn(sc[rt][r], c, -base));
        const float e1 = fast_exp2(__fmaf_rn(sc[rt][r + 1], c, -base));
        if constexpr (E::ES == 2) {
          const uint32_t w = E::Io::pack2(e0, e1);
          p[rt][r >> 3][(r & 7) >> 1] = w;
          l[ct] = add_pair<typename E::Io>(w, l[ct]);
        } else {
          sc[rt][r] = e0, sc[rt][r + 1] = e1;
          l[ct] += e0 + e1;
        }
      }
  }

  // The same by the largest score so far, whose distances are taken before they are multiplied by c. The probabilities are
  // 2^-order() at most, so that no sum of them and values passes the largest value; half's, whose values are below 2^16, are
  // not scaled. m: that score itself.
  __device__ __forceinline__ int order(int ct) const {
    if constexpr (std::is_same<E, E16<F16Io>>::value) return 0;
    else return 33 - __clz(lim[ct]);  // 2^order > 2 lim
  }
  __device__ __forceinline__ void softmax_exact(int ct, f32x16 (&sc)[RT], u32x4 (&p)[RT][2], int k0, float c) {
    const int lh = (threadIdx.x & 63) >> 5;
    float top = -INFINITY;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[rt][r] = k0 + acc_key(rt, r, lh) < lim[ct] ? sc[rt][r] : -INFINITY;
        top = fmaxf(top, sc[rt][r]);
      }
    const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    if (top > m[ct]) {
      const float alpha = fast_exp2((m[ct] - top) * c);
      m[ct] = top;
      l[ct] *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[ct][dt] *= alpha;
    }
    const float base = m[ct] == -INFINITY ? 0.f : m[ct], down = static_cast<float>(-order(ct));
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float e0 = fast_exp2(__fmaf_rn(sc[rt][r] - base, c, down));
        const float e1 = fast_exp2(__fmaf_rn(sc[rt][r + 1] - base, c, down));
        if constexpr (E::ES == 2) {
          const uint32_t w = E::Io::pack2(e0, e1);
          p[rt][r >> 3][(r & 7) >> 1] = w;
          l[ct] = add_pair<typename E::Io>(w, l[ct]);
        } else {
          sc[rt][r] = e0, sc[rt][r + 1] = e1;
          l[ct] += e0 + e1;
        }
      }
  }
  // After kExact: its rows' references in binary orders, as the others'. Where c m is rounded by no more than an order the
  // sums take the rest; a larger m is one of scores that are rounded by as much.
  __device__ __forceinline__ void to_orders(float c) {
    constexpr float kMost = 0x1.fffffep127f;
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      if (lim[ct] == 0 || m[ct] == -INFINITY) continue;
      const float base = fminf(fmaxf(m[ct] * c, -kMost), kMost), up = static_cast<float>(order(ct)), ref = base + up;
      const float rest = __fmaf_rn(m[ct], c, -base) + (base - (ref - up));
      const float f = fabsf(rest) <= 1.f ? fast_exp2(rest) : 1.f;
      m[ct] = ref;
      l[ct] *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[ct][dt] *= f;
    }
  }

  // One key tile; `masked`: some row does not see all of its keys from k0 on.
  template <int PASS>
  __device__ __forceinline__ void step(const uint8_t* sK, const uint8_t* sV, int k0, float c, bool masked, bool first) {
    f32x16 sc[NCT][RT];
    u32x4 p[NCT][RT][2];
    scores(sK, sc);
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      if constexpr (PASS == kExact) softmax_exact(ct, sc[ct], p[ct], k0, c);
      else softmax(ct, sc[ct], p[ct], k0, c, masked || PASS != kPlain, first);
    }
    if constexpr (PASS != kPlain) return add_apart(sV, k0, sc, p);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      if constexpr (E::ES == 2) {
#pragma unroll
        for (int g = 0; g < 2 * RT; ++g) {
          const u32x4 vf = v_operand<E, D>(sV, dt, g);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
            o[ct][dt] = mfma_io_32x32x16<typename E::Io>(vf, p[ct][g >> 1][g & 1], o[ct][dt]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float vf = v_value(sV, dt, r);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) o[ct][dt] = mfma_f32_32x32x2(vf, sc[ct][0][r], o[ct][dt]);
        }
      }
    }
  }

  // fp32: V of key acc_key(0, r, lh), dim 32 dt + lr.
  __device__ __forceinline__ float v_value(const uint8_t* sV, int dt, int r) const {
    const int lane = threadIdx.x & 63, lr = lane & 31, key = acc_key(0, r, lane >> 5);
    return *reinterpret_cast<const float*>(sV + key * (D * 4) + 16 * v_chunk<E, D>(key, 8 * dt + (lr >> 2)) + 4 * (lr & 3));
  }

  // The same sums from V's finite values, in the same order, and then those of its NaNs and infinities, one key at a time,
  // added to the rows that see it.
  __device__ __forceinline__ void add_apart(const uint8_t* sV, int k0, const f32x16 (&sc)[NCT][RT],
                                            const u32x4 (&p)[NCT][RT][2]) {
    const int lh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      auto add = [&](int key, int ct, const f32x16& x) {
        const bool seen = k0 + key < lim[ct];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (!seen || x[i] == 0.f) continue;
          o[ct][dt][i] += x[i];
          taken[ct] |= uint64_t(1) << (16 * dt + i);
        }
      };
      if constexpr (E::ES == 2) {
        u32x4 wild[2 * RT];
        bool any = false;
#pragma unroll
        for (int g = 0; g < 2 * RT; ++g) {
          u32x4 vf = v_operand<E, D>(sV, dt, g);
          constexpr uint32_t kExp = std::is_same<typename E::Io, Bf16Io>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = ((vf[i] & kExp) == kExp ? 0xffffu : 0u) |
                                ((vf[i] & (kExp << 16)) == kExp << 16 ? 0xffff0000u : 0u);
            wild[g][i] = vf[i] & at;
            vf[i] &= ~at;
            any |= at != 0;
          }
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
            o[ct][dt] = mfma_io_32x32x16<typename E::Io>(vf, p[ct][g >> 1][g & 1], o[ct][dt]);
        }
        if (!__any(any)) continue;
#pragma unroll
        for (int g = 0; g < 2 * RT; ++g) {
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {  // key 16 g + j: element 4 (j / 8) + j % 4 of lane half (j / 4) % 2
            u32x4 one;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              one[i] = lh == ((j >> 2) & 1) && i == 2 * (j >> 3) + ((j & 3) >> 1)
                           ? wild[g][i] & (j & 1 ? 0xffff0000u : 0xffffu)
                           : 0u;
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
              add(16 * g + j, ct, mfma_io_32x32x16<typename E::Io>(one, p[ct][g >> 1][g & 1], f32x16{}));
          }
        }
      } else {
        auto is_wild = [](float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; };
        bool any = false;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float vf = v_value(sV, dt, r);
          any |= is_wild(vf);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) o[ct][dt] = mfma_f32_32x32x2(is_wild(vf) ? 0.f : vf, sc[ct][0][r], o[ct][dt]);
        }
        if (!__any(any)) continue;
#pragma unroll 1
        for (int n = 0; n < 32; ++n) {  // register n / 2 of lane half n % 2
          const int r = n >> 1;
          const float vf = v_value(sV, dt, r), wild = lh == (n & 1) && is_wild(vf) ? vf : 0.f;
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            float one = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) one = r == i ? sc[ct][0][i] : one;
            add(acc_key(0, r, n & 1), ct, mfma_f32_32x32x2(wild, one, f32x16{}));
          }
        }
      }
    }
  }
};

template <class E, int D, int NCT, int NW, int WAVES>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES))) void attend_kernel(const Args a) {
  using L = Lds<E, D>;
  constexpr int R = 32 * NCT * NW;
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * L::kStage];
  const int lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5, wv = wave_id();
  // consecutive workgroups: the parts of one tile's keys, then the heads of keys, then the slots. fp32 tiles are bound by the
  // matrix cores, and the CU with the longest ones ends last: where there are two a CU, the longest sequences come first and
  // every other 256 workgroups (a CU has one of each) go the other way round, so that a long tile meets a short one (24
  // prompts of up to 256 tokens, 16 heads of 64: 46 -> 41 us; 16-bit tiles gain nothing, and short ones lose a third).
  int b = blockIdx.x;
  const bool sorted = E::ES == 4 && a.N <= 64 && gridDim.x >= 512;
  if (sorted && (b & 256) && (b | 255) < static_cast<int>(gridDim.x)) b ^= 255;
  const int part = b % a.splits, rest = b / a.splits, g = rest % a.G, u = rest / a.G;
  const Tile t = find_tile(a, u, R, sorted);
  const int row_bytes = D * E::ES;
  if (!t.found) {
    if (!a.zero_rest || part) return;
    // the rows of no sequence, shared by the slots without a tile (one at least: every sequence fills the most of its last)
    const int first = clamp_to(a.off[0], 0, a.T), end = clamp_to(a.off[a.N], first, a.T), spare = a.T - (end - first);
    const int pieces = a.gs * row_bytes / 16;  // 16-byte ones of this head's rows of a token
    for (int i = t.index; i < spare; i += t.idle) {
      uint8_t* row = a.out + static_cast<int64_t>(i < first ? i : end + i - first) * a.o_ts;
      for (int j = threadIdx.x; j < pieces; j += 64 * NW)
        st16(row + (g * a.gs + j / (row_bytes / 16)) * a.o_hs + 16 * (j % (row_bytes / 16)), u32x4{0, 0, 0, 0});
    }
    return;
  }
  const int rows = t.lq * a.gs, r0 = t.index * R + wv * 32 * NCT;
  // the keys that row r sees; rows past the last as that one
  auto sees = [&](int r) {
    const int at = (r < rows ? r : rows - 1) / a.gs;
    return a.causal ? clamp_to(at + (t.lk - t.lq) + 1, 0, t.lk) : t.lk;
  };
  const int all = __builtin_amdgcn_readfirstlane(sees(t.index * R + R - 1));  // of the workgroup's rows
  int most = r0 < rows ? __builtin_amdgcn_readfirstlane(sees(r0 + 32 * NCT - 1)) : 0;  // of the wave's: the last
  const int least = __builtin_amdgcn_readfirstlane(sees(r0));                               // and the first one
  const int each = ((all + a.splits - 1) / a.splits + E::KT - 1) / E::KT * E::KT;
  const int begin = part * each, end = begin + each < all ? begin + each : all;

  Rows<E, D, NCT> w;
  int64_t token[NCT];
  int head[NCT];
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const int r = r0 + 32 * ct + lr, rc = r < rows ? r : rows - 1, at = rc / a.gs;
    token[ct] = t.q0 + at;
    head[ct] = g * a.gs + rc - at * a.gs;
    w.lim[ct] = r0 < rows ? sees(r) : 0;  // (a wave past the last row sees nothing)
    const uint8_t* p = a.q + token[ct] * a.q_ts + head[ct] * a.q_hs;
#pragma unroll
    for (int i = 0; i < Rows<E, D, NCT>::kQ; ++i) w.q[ct][i] = ld16(p + 32 * i + 16 * lh);
  }
  const uint32_t lds0 = lds_addr(smem);
  auto run = [&](auto pass) {
    if (begin >= end) return;
    const KeyCopy<E, D, NW> copy(a, t, g);
    copy(begin, lds0);
    int stage = 0;
    for (int k0 = begin; k0 < end; k0 += E::KT, stage ^= 1) {
      // vmcnt(0): this wave's copies of the tile. As the builtin, which the compiler counts: after assembly it would wait for
      // the queries' loads inside the loop, and with them for the copies of the next tile (one token 89 -> 65 us).
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();  // everybody's, and the other stage is free
      if (k0 + E::KT < end) copy(k0 + E::KT, lds0 + (stage ^ 1) * L::kStage);
      const uint8_t* s = smem + stage * L::kStage;
      if (k0 < most) w.template step<decltype(pass)::value>(s, s + L::kTile, k0, a.c, k0 + E::KT > least, k0 == begin);
    }
  };
  // Whether the workgroup has rows to compute again (and once all know it the stages are free).
  auto again = [&]() {
    const bool here = w.again(begin);
    if (!here) most = 0;
    return __syncthreads_or(here);
  };
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) w.clear(ct);
  run(std::integral_constant<int, kPlain>{});
  if (again()) {
    run(std::integral_constant<int, kApart>{});
    if (again()) {
      run(std::integral_constant<int, kExact>{});
      if (a.splits > 1) w.to_orders(a.c);
    }
  }

#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const float total = w.l[ct] + __shfl_xor(w.l[ct], 32, kWave);
    if (r0 + 32 * ct + lr >= rows) continue;
    if (a.splits > 1) {
      const int64_t at = (static_cast<int64_t>(part) * a.T + token[ct]) * a.H + head[ct];
      float* po = a.part_o + at * D;
      // The join weighs a part by 2^(its reference - the largest one), which is lost where it is no normal number. A
      // reference under a total of 2^32 and more is raised by the total's exponent (the factor is exact); under a smaller
      // one a lost part is less than 2^-90 of the result's weights.
      const bool raise = total >= 0x1p32f && total < INFINITY;
      const int up = raise ? static_cast<int>(__float_as_uint(total) >> 23) - 127 : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(po + 32 * dt + 8 * i + 4 * lh) =
              f32x4{w.o[ct][dt][4 * i] * down, w.o[ct][dt][4 * i + 1] * down, w.o[ct][dt][4 * i + 2] * down,
                    w.o[ct][dt][4 * i + 3] * down};
      if (lh == 0) a.part_ml[2 * at] = w.m[ct] + static_cast<float>(up), a.part_ml[2 * at + 1] = total * down;
      continue;
    }
    const float inv = total == 0.f ? 0.f : __frcp_rn(total);
    uint8_t* orow = a.out + token[ct] * a.o_ts + head[ct] * a.o_hs;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = w.o[ct][dt][4 * i + j] * inv;
        uint8_t* p = orow + (32 * dt + 8 * i + 4 * lh) * E::ES;
        if constexpr (E::ES == 2)
          *reinterpret_cast<u32x2*>(p) = u32x2{E::Io::pack2(x[0], x[1]), E::Io::pack2(x[2], x[3])};
        else
          *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
      }
  }
}

// The parts of each row's keys joined, in their order: a wave per row.
template <class E, int D>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + wave_id(), all = static_cast<int64_t>(a.T) * a.H;
  if (n >= all) return;
  const int token = static_cast<int>(n / a.H), head = static_cast<int>(n - static_cast<int64_t>(token) * a.H);
  const int first = clamp_to(a.off[0], 0, a.T);
  if (token < first || token >= clamp_to(a.off[a.N], first, a.T)) return;  // of no sequence
  // lane i: part i's maximum and total (64 parts at most)
  float top = -INFINITY, total = 0.f;
  if (lane < a.splits) top = a.part_ml[2 * (lane * all + n)], total = a.part_ml[2 * (lane * all + n) + 1];
  const float best = wave_max(top), f = fast_exp2(top - (best == -INFINITY ? 0.f : best));
  total *= f;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d, kWave);
  constexpr int N = D / 64, kAtOnce = 8;
  float sum[N] = {};
  for (int s0 = 0; s0 < a.splits; s0 += kAtOnce) {
    float o[kAtOnce][N];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = (s0 + i < a.splits ? s0 + i : a.splits - 1) * all + n;
#pragma unroll
      for (int j = 0; j < N; ++j) o[i][j] = a.part_o[at * D + N * lane + j];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float fi = __shfl(f, s0 + i, kWave);
      if (s0 + i < a.splits)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = __fmaf_rn(fi, o[i][j], sum[j]);
    }
  }
  const float inv = total == 0.f ? 0.f : __frcp_rn(total);
  uint8_t* p = a.out + token * a.o_ts + head * a.o_hs + N * lane * E::ES;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (E::ES == 4) reinterpret_cast<float*>(p)[j] = sum[j] * inv;
    else reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(E::Io::pack2(sum[j] * inv, 0.f));
  }
}

constexpr int kWaves = 4, kColumns = 1, kTileRows = 32 * kColumns * kWaves;

// Slots: a sequence of n rows takes at most (n + kTileRows - 1) / kTileRows tiles.
int64_t slots_of(int64_t T, int N, int gs) { return (T * gs + kTileRows - 1) / kTileRows + N; }

// Parts of the keys: where the tiles do not give every CU three workgroups, as many as do (16 new tokens, 8 heads of keys of
// 128: 58 us against 63 with two a CU), of 256 keys in the mean at least; 64 for fp32, whose 32 keys take 1.7 to 3.4 us where
// 16-bit ones' 64 take 0.5 (7 sequences of new tokens over 2093 keys of 128: 49 -> 20 us; 16-bit parts of 128 keys cost up to
// twice what they save). For balance as many as give six a CU, of 512 keys: fp32 tiles (3223 tokens: 424 -> 377 us) and
// those of a wave's rows or fewer, which read at the memory's rate (one token of 16 sequences of up to 8249 keys, not in any
// cache: 16 heads of 64 83 -> 72 us, 8 of 128 72 -> 69; other 16-bit tiles lose to it, 5828 tokens 121 -> 138).
int splits_of(int dtype, int64_t T, int64_t Tk, int N, int H, int G) {
  const int64_t tiles = slots_of(T, N, H / G) * G, mean = Tk / N, cus = device_cus();
  auto smaller = [](int64_t x, int64_t y) { return x < y ? x : y; };
  int64_t s = smaller(3 * cus / tiles, mean / (dtype == HB_F32 ? 64 : 256));
  if (dtype == HB_F32 || T * (H / G) <= 32 * static_cast<int64_t>(N)) {
    const int64_t even = smaller(6 * cus / tiles, mean / 512);
    if (even > s) s = even;
  }
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}

size_t workspace_of(int dtype, int64_t T, int64_t Tk, int N, int H, int G, int D) {
  const int s = splits_of(dtype, T, Tk, N, H, G);
  return s == 1 ? 0 : static_cast<size_t>(s) * static_cast<size_t>(T) * H * (D + 2) * 4;
}

template <class E, int D>
void launch(hipStream_t stream, const Args& a) {
  const unsigned grid = static_cast<unsigned>(a.slots) * a.G * a.splits;
  auto attend = [&](auto per_simd) {
    hipLaunchKernelGGL((attend_kernel<E, D, kColumns, kWaves, decltype(per_simd)::value>), dim3(grid), dim3(64 * kWaves), 0,
                       stream, a);
  };
  // fp32 heads of 128 do without spills with a wave a SIMD (12 prompts of 161 to 312 tokens, 32 heads: 171 -> 147 us), but
  // tiles of one wave's rows leave the other SIMDs to a second workgroup, where there is one (29 sequences of 1 to 5 new
  // tokens over 63 keys, 16 heads: 18.6 us, 28 with one).
  if constexpr (D == 64) attend(std::integral_constant<int, 3>{});
  else if (E::ES == 2 || (grid > static_cast<unsigned>(device_cus()) && static_cast<int64_t>(a.T) * a.gs <= 32ll * a.N))
    attend(std::integral_constant<int, 2>{});
  else if constexpr (E::ES == 4) attend(std::integral_constant<int, 1>{});
  if (a.splits > 1)
    hipLaunchKernelGGL((join_kernel<E, D>), dim3(static_cast<unsigned>((static_cast<int64_t>(a.T) * a.H + 3) / 4)),
                       dim3(256), 0, stream, a);
}

int check_sizes(const char* what, int dtype, int64_t T, int64_t Tk, int N, int H, int G, int D) {
  if (dtype != HB_BF16 && dtype != HB_F32 && dtype != HB_F16)
    return fail(HB_ERR_DTYPE, "%s: dtype %d is not HB_BF16 (0), HB_F32 (1) or HB_F16 (2)", what, dtype);
  if (D != 64 && D != 128) return fail(HB_ERR_HEAD_DIM, "%s: head_dim %d is not 64 or 128", what, D);
  constexpr int64_t kMost = int64_t(1) << 30;
  if (T < 1 || Tk < 0 || N < 1 || H < 1 || G < 1 || H % G || H > 65535 || N > (1 << 20) || T > kMost || Tk > kMost ||
      T * (H / G) > kMost || slots_of(T, N, H / G) * G >= (int64_t(1) << 24))
    return fail(HB_ERR_SHAPE, "%s: T=%lld, Tk=%lld, N=%d, H=%d, G=%d out of range", what, static_cast<long long>(T),
                static_cast<long long>(Tk), N, H, G);
  return HB_OK;
}

}  // namespace packed
}  // namespace hb

using namespace hb;

extern "C" {

size_t hb_packed_workspace_size(int dtype, int64_t T, int64_t Tk, int N, int H, int G, int D) {
  clear_error();
  if (packed::check_sizes("packed_workspace_size", dtype, T, Tk, N, H, G, D)) return 0;
  return packed::workspace_of(dtype, T, Tk, N, H, G, D);
}

int hb_packed_attention(hipStream_t stream, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                        int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                        int64_t v_head_stride, int dtype, const int* offsets, const int* key_offsets,
                        const int* key_lengths, int causal, float scale, void* out, int64_t out_token_stride,
                        int64_t out_head_stride, int zero_rest, int64_t T, int64_t Tk, int N, int H, int G, int D,
                        void* workspace, size_t workspace_bytes) {
  clear_error();
  const char* what = "packed_attention";
  int st = packed::check_sizes(what, dtype, T, Tk, N, H, G, D);
  if (st) return st;
  if (!q || !offsets || !key_offsets || !out || (Tk > 0 && (!k || !v)))
    return fail(HB_ERR_NULL, "%s: q, k, v, offsets, key_offsets and out must be non-NULL", what);
  if (!(scale > 0.0f) || !std::isfinite(scale) || !std::isfinite(scale * kLog2e))
    return fail(HB_ERR_EPS, "%s: scale %g must be finite and > 0", what, scale);
  const int es = dtype == HB_F32 ? 4 : 2, vec = 16 / es;
  struct Operand {
    const char* name;
    const void* p;
    int64_t ts, hs, tokens;
    int heads;
    int64_t bytes;
  } ops[] = {{"out", out, out_token_stride, out_head_stride, T, H, 0}, {"q", q, q_token_stride, q_head_stride, T, H, 0},
             {"k", k, k_token_stride, k_head_stride, Tk, G, 0},       {"v", v, v_token_stride, v_head_stride, Tk, G, 0}};
  for (Operand& o : ops) {
    if (!o.tokens) continue;
    if (o.tokens == 1) o.ts = 0;  // never stepped by, whatever the caller's tensor has there
    if (o.heads == 1) o.hs = 0;
    if (reinterpret_cast<uintptr_t>(o.p) % 16 || o.ts % vec || o.hs % vec || o.ts < 0 || o.hs < 0)
      return fail(HB_ERR_STRIDE, "%s: %s must be 16-byte aligned with strides that are multiples of %d, not negative", what,
                  o.name, vec);
    // a key tile's rows are addressed by 32-bit offsets from its first
    if ((o.name[0] == 'k' || o.name[0] == 'v') && o.ts > (1 << 23))
      return fail(HB_ERR_STRIDE, "%s: %s token stride must be at most 2^23", what, o.name);
    if ((st = check_extent(what, o.name, o.tokens, o.ts, D)) || (st = check_extent(what, o.name, o.heads, o.hs, D)))
      return st;
    o.bytes = ((o.tokens - 1) * o.ts + (o.heads - 1) * o.hs + D) * es;
  }
  // the output's rows share no element: heads within tokens or tokens within heads
  const Operand &oo = ops[0], &oq = ops[1], &ok = ops[2], &ov = ops[3];
  const bool inside = H == 1 || oo.hs >= D, outside = T == 1 || oo.ts >= D;
  if (!inside || !outside ||
      !(T == 1 || H == 1 || oo.ts >= (H - 1) * oo.hs + D || oo.hs >= (T - 1) * oo.ts + D))
    return fail(HB_ERR_STRIDE, "%s: the rows of out overlap", what);
  const int64_t ob = oo.bytes, table = (static_cast<int64_t>(N) + 1) * 4;
  const size_t need = packed::workspace_of(dtype, T, Tk, N, H, G, D);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(HB_ERR_WORKSPACE, "%s needs %zu bytes of workspace, 16-byte aligned", what, need);
  auto misaligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0; };
  if (misaligned(offsets) || misaligned(key_offsets) || misaligned(key_lengths))
    return fail(HB_ERR_STRIDE, "%s: offsets, key_offsets and key_lengths must be 4-byte aligned", what);
  const int64_t wb = static_cast<int64_t>(need);
  for (const Operand& o : ops)
    if ((o.name[0] != 'o' && (st = check_disjoint(what, "out", out, ob, o.name, o.p, o.bytes))) ||
        (st = check_disjoint(what, "workspace", workspace, wb, o.name, o.p, o.bytes)))
      return st;
  const struct {
    const char* name;
    const void* p;
    int64_t bytes;
  } tables[] = {{"offsets", offsets, table}, {"key_offsets", key_offsets, table}, {"key_lengths", key_lengths, table - 4}};
  for (const auto& o : tables)
    if ((st = check_disjoint(what, "out", out, ob, o.name, o.p, o.bytes)) ||
        (st = check_disjoint(what, "workspace", workspace, wb, o.name, o.p, o.bytes)))
      return st;
  packed::Args a = {};
  a.q = static_cast<const uint8_t*>(q), a.q_ts = oq.ts * es, a.q_hs = oq.hs * es;
  a.k = static_cast<const uint8_t*>(k), a.k_ts = ok.ts * es, a.k_hs = ok.hs * es;
  a.v = static_cast<const uint8_t*>(v), a.v_ts = ov.ts * es, a.v_hs = ov.hs * es;
  a.out = static_cast<uint8_t*>(out), a.o_ts = oo.ts * es, a.o_hs = oo.hs * es;
  a.off = offsets, a.koff = key_offsets, a.klen = key_lengths;
  a.causal = causal != 0, a.zero_rest = zero_rest != 0, a.c = scale * kLog2e;
  a.T = static_cast<int>(T), a.Tk = static_cast<int>(Tk), a.N = N, a.H = H, a.G = G, a.gs = H / G;
  a.slots = static_cast<int>(packed::slots_of(T, N, H / G)), a.splits = packed::splits_of(dtype, T, Tk, N, H, G);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o ? a.part_o + static_cast<int64_t>(a.splits) * T * H * D : nullptr;
  auto run = [&](auto e) {
    using E = decltype(e);
    if (D == 64) packed::launch<E, 64>(stream, a);
    else packed::launch<E, 128>(stream, a);
  };
  if (dtype == HB_BF16) run(packed::E16<Bf16Io>{});
  else if (dtype == HB_F16) run(packed::E16<F16Io>{});
  else run(packed::E32{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return HB_OK;
}

}  // extern "C"

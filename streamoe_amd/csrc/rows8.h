// rows8.h — quantized products of 8-bit rows on the int8 matrix cores (one
// translation unit per weight width includes it: rows8_q4.hip, rows8_q3.hip,
// rows8_q8.hip).
//
//   y[t, o] = sum_g sx[t, g] (s[o, g] sum_{c in g} q[o, c] x[t, c]
//                             + b[o, g] sum_{c in g} x[t, c])
//
// The codes enter as they are (8-bit ones less 128, with 128 s added to b), so
// a group's sums are exact int32: |sum| <= 128 * 128 * 128. They are turned
// into f32 and accumulated there, in one rounding each; with one scale per row
// (x_group 0) sx multiplies the finished sum.
//
// Operands: lane (c, kb) of a wave holds 16 inputs of row c in each of two
// operands per step of 128 inputs. Of 4- and 3-bit weights it loads the chunk
// of 32 codes kb of the step; for groups of 64 the halves of two lanes' chunks
// are exchanged, for groups of 32 the four lanes' chunks are transposed by
// their words, so that an operand lies in one group (or two halves of it do,
// in groups of 32). The rows' inputs are loaded from the matching places and
// put in the codes' byte order, evens before odds of eight.
#pragma once

#include "common.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace smoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kQ8Step = 128;

// Rows' scales per group enter times 2^-24 and the finished sums leave times
// 2^24: a group's sum (up to 2^21, and 1.5 2^23 in the kernels that read it from
// a float's bits) times the largest scale then stays in f32's range. Both are
// exact but for scales below 2^-102.
constexpr float kQ8Down = 0x1p-24f, kQ8Up = 0x1p24f;

__device__ __forceinline__ i32x4 q8_mfma(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 q8_mfma32(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x32_i8((long)(((uint64_t)a1 << 32) | a0), (long)(((uint64_t)b1 << 32) | b0), c, 0, 0, 0);
}

// The 4 x 4 words (lane block of 16, register) transposed.
__device__ __forceinline__ void q8_transpose4(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  const auto ac = __builtin_amdgcn_permlane32_swap(a, c, false, false);
  const auto bd = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  const auto ab = __builtin_amdgcn_permlane16_swap(ac[0], bd[0], false, false);
  const auto cd = __builtin_amdgcn_permlane16_swap(ac[1], bd[1], false, false);
  a = ab[0], b = ab[1], c = cd[0], d = cd[1];
}

// Chunks of 32 bytes, one per lane block, to operands of one group each: the
// halves of two lanes' chunks exchanged (groups of 64), the four lanes' chunks
// transposed by their eights (of 32).
template <int G>
__device__ __forceinline__ void q8_exchange(uint32_t (&q)[8]) {
  if constexpr (G == 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto r = __builtin_amdgcn_permlane32_swap(q[i], q[i + 4], false, false);
      q[i] = r[0];
      q[i + 4] = r[1];
    }
  }
  if constexpr (G == 32) {
    q8_transpose4(q[0], q[2], q[4], q[6]);
    q8_transpose4(q[1], q[3], q[5], q[7]);
  }
}

// The loaded codes of a step (chunks of 32) as operands.
template <int BITS, int G>
__device__ __forceinline__ void q8_operands(const uint32_t (&d)[BITS == 8 ? 8 : BITS], u32x4 (&b)[2]) {
  uint32_t q[8];
  if constexpr (BITS == 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = d[i] ^ 0x80808080u;
    q8_exchange<G>(q);
  } else {
    Raw<BITS> w;
#pragma unroll
    for (int i = 0; i < BITS; ++i) w.d[i] = d[i];
    if constexpr (BITS == 4) {  // the same exchange while it is half the words
      if constexpr (G == 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto r = __builtin_amdgcn_permlane32_swap(w.d[i], w.d[i + 2], false, false);
          w.d[i] = r[0];
          w.d[i + 2] = r[1];
        }
      }
      if constexpr (G == 32) q8_transpose4(w.d[0], w.d[1], w.d[2], w.d[3]);
    }
    unpack_bytes(w, q);
    if constexpr (BITS == 3) q8_exchange<G>(q);
  }
  b[0] = u32x4{q[0], q[1], q[2], q[3]};
  b[1] = u32x4{q[4], q[5], q[6], q[7]};
}

// Sums of group g of a step, from z on.
template <int G>
__device__ __forceinline__ i32x4 q8_sums(const u32x4 (&x)[2], const u32x4 (&b)[2], uint32_t g, i32x4 z = {0, 0, 0, 0}) {
  if constexpr (G == 64) {
    return q8_mfma(x[g], b[g], z);
  } else if constexpr (G == 32) {
    const uint32_t h = g / 2, o = g % 2 * 2;
    return q8_mfma32(x[h][o], x[h][o + 1], b[h][o], b[h][o + 1], z);
  } else {
    return q8_mfma(x[1], b[1], q8_mfma(x[0], b[0], z));
  }
}

// ---------------------------------------------------------------------------
// Few rows or columns: a block's waves share MT tiles of 16 rows x NT tiles of
// 16 columns and take the steps of 128 inputs in turn (up to 16 waves: a small
// call is one round trip to memory), a step ahead. Loads are made in memory
// order: lane 4 r + p takes part p (32 inputs) of row r, one cache access per
// four lanes where the operand order would take one per lane, and a lane
// permute brings the parts to the operand's lanes (4 rows 2048 -> 4096 took
// 5.9 us in operand order, 3.4 now). Rows are the A operand: lane (c, kb) ends
// with column c of rows 4 kb .. 4 kb + 3. The sums of inputs come from a product
// with ones; the waves' parts are added in LDS.
// ---------------------------------------------------------------------------
template <int BITS, int G, bool XG, int MT, int NT>
__global__ __launch_bounds__(MT * NT == 1 ? 1024 : 512) void k_q8_few(Q8Args a) {
  constexpr uint32_t GS = kQ8Step / G, W = BITS == 8 ? 8 : BITS, SW = (GS + 1) / 2;
  extern __shared__ __attribute__((aligned(16))) f32x4 red[];  // [wave][MT * NT][64]
  const uint32_t lane = threadIdx.x & 63, c16 = lane & 15, kb = lane >> 4, lr = lane >> 2, lp = lane & 3;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const uint32_t K = a.K, O = a.O, gpr = K / G, steps = (K + kQ8Step - 1) / kQ8Step;
  const uint32_t col0 = blockIdx.x * (NT * 16), row0 = blockIdx.y * (MT * 16);
  const uint32_t row_bytes = K / 32 * (BITS * 4);
  const int8_t* xr[MT];
  const float* sxr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    xr[m] = a.x + (uint64_t)min(row0 + m * 16 + lr, a.n - 1) * K;
    sxr[m] = a.sx + (uint64_t)min(row0 + m * 16 + c16, a.n - 1) * (XG ? gpr : 1u);
  }
  const uint8_t* wr[NT];
  const uint16_t *sr[NT], *br[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    wr[t] = a.w + (uint64_t)min(col0 + t * 16 + lr, O - 1) * row_bytes;
    const uint64_t c = (uint64_t)min(col0 + t * 16 + c16, O - 1) * gpr;
    sr[t] = a.s + c;
    br[t] = a.b + c;
  }
  struct Step {
    u32x4 x[MT][2];
    uint32_t w[NT][W], s[NT][SW], b[NT][SW];  // pairs of groups
    float sx[MT][GS];
  };
  auto load = [&](uint32_t st, Step& v) {
    const uint32_t k0 = st * kQ8Step;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* const p = wr[t] + min(k0 / 32 + lp, K / 32 - 1) * (BITS * 4);
      if constexpr (BITS == 8) {
        const u32x4 lo = *reinterpret_cast<const u32x4*>(p), hi = *reinterpret_cast<const u32x4*>(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[t][i] = lo[i], v.w[t][4 + i] = hi[i];
      } else {
        const Raw<BITS> r = load_raw<BITS, false>(p);
#pragma unroll
        for (int i = 0; i < BITS; ++i) v.w[t][i] = r.d[i];
      }
#pragma unroll
      for (uint32_t j = 0; j < SW; ++j) {
        const uint32_t g = st * GS + 2 * j;
        if (GS > 1 && a.even) {
          v.s[t][j] = *reinterpret_cast<const uint32_t*>(sr[t] + min(g, gpr - 2));
          v.b[t][j] = *reinterpret_cast<const uint32_t*>(br[t] + min(g, gpr - 2));
        } else {
          const uint32_t g0 = min(g, gpr - 1), g1 = min(g + 1, gpr - 1);
          v.s[t][j] = sr[t][g0] | (GS > 1 ? (uint32_t)sr[t][g1] << 16 : 0u);
          v.b[t][j] = br[t][g0] | (GS > 1 ? (uint32_t)br[t][g1] << 16 : 0u);
        }
      }
    }
    const uint32_t at = min(k0 + lp * 32, K - 32);  // K is a multiple of 32
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      v.x[m][0] = *reinterpret_cast<const u32x4*>(xr[m] + at);
      v.x[m][1] = *reinterpret_cast<const u32x4*>(xr[m] + at + 16);
      if constexpr (XG)
#pragma unroll
        for (uint32_t j = 0; j < GS; ++j) v.sx[m][j] = sxr[m][min(st * GS + j, gpr - 1)];
    }
  };
  const int psrc = (int)((c16 * 4 + kb) * 4);
  auto from = [&](int src, uint32_t x) { return (uint32_t)__builtin_amdgcn_ds_bpermute(src, (int)x); };
  const u32x4 one = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
  const u32x4 ones[2] = {one, one};
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](uint32_t st, const Step& v) {
    const bool in = st * kQ8Step + lp * 32 < K;
    u32x4 x[MT][2], w[NT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = from(psrc, in ? v.x[m][i / 4][i % 4] : 0u);
      q8_exchange<G>(d);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t* const e = d + 4 * h;
        if (BITS == 8)
          x[m][h] = u32x4{e[0], e[1], e[2], e[3]};
        else  // evens before odds, as the codes unpack
          x[m][h] = u32x4{__builtin_amdgcn_perm(e[1], e[0], 0x06040200u), __builtin_amdgcn_perm(e[1], e[0], 0x07050301u),
                          __builtin_amdgcn_perm(e[3], e[2], 0x06040200u), __builtin_amdgcn_perm(e[3], e[2], 0x07050301u)};
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint32_t d[W];
#pragma unroll
      for (uint32_t i = 0; i < W; ++i) d[i] = from(psrc, v.w[t][i]);
      q8_operands<BITS, G>(d, w[t]);
    }
#pragma unroll
    for (uint32_t j = 0; j < GS; ++j) {
      f32x4 xf[MT], sx[MT];  // of rows 4 kb ..
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const i32x4 X = q8_sums<G>(x[m], ones, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (XG) sx[m][i] = __shfl(v.sx[m][j], 4 * (int)kb + i, kWave) * kQ8Down;
          xf[m][i] = XG ? (float)X[i] * sx[m][i] : (float)X[i];
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        auto half = [&](uint32_t p) { return __uint_as_float(j & 1 ? p & 0xFFFF0000u : p << 16); };
        const float s = half(v.s[t][j / 2]);
        float b = half(v.b[t][j / 2]);
        if (BITS == 8) b = __builtin_fmaf(s, 128.f, b);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const i32x4 S = q8_sums<G>(x[m], w[t], j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f = (float)S[i];
            if constexpr (XG) f *= sx[m][i];
            acc[m][t][i] = __builtin_fmaf(s, f, acc[m][t][i]);
            acc[m][t][i] = __builtin_fmaf(b, xf[m][i], acc[m][t][i]);
          }
        }
      }
    }
  };
  f32x4 scale[MT];  // of the rows that the wave ends
  if (!XG && wave < MT * NT) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) scale[m][i] = a.sx[min(row0 + m * 16 + 4 * kb + i, a.n - 1)];
  }
  // Every path to a use of a step has the same loads behind it, or the wait
  // would be for all of them.
  Step v[2];
  uint32_t st = wave;  // there are no more waves than steps
  load(st, v[0]);
  while (st + nw < steps) {
    load(st + nw, v[1]);
    compute(st, v[0]);
    st += nw;
    if (st + nw >= steps) {
      v[0] = v[1];
      break;
    }
    load(st + nw, v[0]);
    compute(st, v[1]);
    st += nw;
  }
  compute(st, v[0]);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) red[(wave * MT * NT + m * NT + t) * 64 + lane] = acc[m][t];
  __syncthreads();
  for (uint32_t mt = wave; mt < MT * NT; mt += nw) {
    f32x4 sum = red[mt * 64 + lane], by = scale[0];
#pragma unroll
    for (uint32_t m = 1; m < MT; ++m)
      if (mt / NT == m) by = scale[m];
    for (uint32_t w = 1; w < nw; ++w) sum += red[(w * MT * NT + mt) * 64 + lane];
    const uint32_t col = col0 + mt % NT * 16 + c16;
    if (col >= O) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = row0 + mt / NT * 16 + 4 * kb + i;
      if (r < a.n) a.y[(uint64_t)r * O + col] = sum[i] * (XG ? kQ8Up : by[i]);
    }
  }
}

constexpr uint32_t kMagicBits = 0x4B400000u;  // 1.5 * 2^23
constexpr float kMagic = 12582912.f;

typedef __bf16 qbf16x8 __attribute__((ext_vector_type(8)));

// sx to 22 significant bits.
__device__ __forceinline__ float q8_round22(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7F800000u) == 0x7F800000u) return v;
  return __uint_as_float((u + 1u + ((u >> 2) & 1u)) & ~3u);
}

// Three bf16 of a and three of b, each the rest of those before it.
__device__ __forceinline__ qbf16x8 q8_parts(float a, float b) {
  auto top = [](float v) { return __float_as_uint(v) & 0xFFFF0000u; };
  const uint32_t ah = top(a), bh = top(b);
  const float ar = a - __uint_as_float(ah), br = b - __uint_as_float(bh);
  const uint32_t am = top(ar), bm = top(br);
  const uint32_t al = __float_as_uint(ar - __uint_as_float(am)), bl = __float_as_uint(br - __uint_as_float(bm));
  return __builtin_bit_cast(qbf16x8, u32x4{ah >> 16 | am, al >> 16 | bh, bm >> 16 | (bl & 0xFFFF0000u), 0u});
}

// ---------------------------------------------------------------------------
// Few rows, many columns: the rows stay in LDS, as operands, and the waves
// stream the weights, a tile of 16 columns after another, four steps (a round)
// at a time. A wave's load takes four rows' codes of those steps, whole lines
// (256 bytes a row with 4 bits), and its own part of LDS hands them to the
// operands' lanes. The loads are non-temporal: weights that a step reads once
// come from HBM (16 rows 2048 -> 151936, three sets of weights in turn: 40 us,
// 4.6 TB/s, temporal 42.5; the same set again and again 39 and, from the
// memory-side cache, 34). Two rounds are in flight while one is computed (one:
// 43, three: 41, five: 42), for which nothing between them may branch. Rows
// are the A operand: lane (c, kb) ends with column c of rows 4 kb .. 4 kb + 3,
// and needs the scales of one column only.
// ---------------------------------------------------------------------------
constexpr uint32_t kWideSteps = 4;  // per round of loads

// Where piece p (16 inputs) of a row's step lies among its operands: place of
// its e-th eight, in 8-byte units of [h][kb][row][e]; rows are exchanged by
// 4 h + kb so that the pieces of a row fall in different banks.
template <int G>
__device__ __forceinline__ uint32_t q8_slot(uint32_t p, uint32_t e, uint32_t row) {
  const uint32_t h = G == 128 ? p & 1 : p >> 2;
  const uint32_t kb = G == 32 ? (p & 1) * 2 + e : G == 64 ? ((p & 1) << 1) | ((p >> 1) & 1) : p >> 1;
  const uint32_t f = G == 32 ? (p >> 1) & 1 : e;
  return ((h * 4 + kb) * 16 + (row ^ (h * 4 + kb))) * 2 + f;
}

__host__ __device__ constexpr uint32_t q8_wide_steps(uint32_t K) {
  return (K + kWideSteps * kQ8Step - 1) / (kWideSteps * kQ8Step) * kWideSteps;
}
// LDS: operands, the bias term's operands per eight groups, the rows' scales,
// each wave's 16 x 16 chunks of a round.
__host__ __device__ constexpr uint32_t q8_wide_lds(uint32_t bits, uint32_t K, uint32_t G, uint32_t mt, bool xg) {
  const uint32_t steps = q8_wide_steps(K), groups = steps * (kQ8Step / G);
  return mt * (steps * 2048 + (groups + 7) / 8 * 1024 + (xg ? groups * 64 : 0)) + 4 * 256 * (bits == 8 ? 32 : 16);
}

template <int BITS, int G, bool XG, int MT>
__global__ __launch_bounds__(256, 2) void k_q8_wide(Q8Args a, uint32_t tiles) {
  constexpr uint32_t GS = kQ8Step / G, W = BITS == 8 ? 8 : BITS, GC = GS * kWideSteps;  // groups per round
  constexpr uint32_t PW = GC >= 8 ? GC / 8 : 1;  // pairs of scales a lane loads per round (G = 128: two lanes the same)
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const uint32_t tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t K = a.K, O = a.O, gpr = K / G, row_bytes = K / 32 * (BITS * 4);
  const uint32_t steps = q8_wide_steps(K), groups = steps * GS, octets = (groups + 7) / 8, rounds = steps / kWideSteps;
  u32x4* const xl = reinterpret_cast<u32x4*>(lds_raw);                 // [step][m][h][64]
  u32x4* const parts = xl + steps * MT * 128;                          // [octet][m][64]
  float* const sxl = reinterpret_cast<float*>(parts + octets * MT * 64);  // [group][m][16]
  // The wave's chunks of a round: chunk p of row r at place 16 r + (p ^ r), so
  // that the rows' reads of one chunk fall in different banks.
  constexpr uint32_t CW = BITS == 8 ? 2 : 1;  // 16-byte words per chunk
  u32x4* const mine = reinterpret_cast<u32x4*>(sxl + (XG ? groups * MT * 16 : 0)) + wave * 256 * CW;

  // The loads of a round: chunk lp of rows lr, lr + 4, .. of the tile.
  const uint32_t lr = lane >> 4, lp = lane & 15;
  struct Round {
    uint32_t w[kWideSteps][W];
    uint32_t s[PW], b[PW];
  };
  auto group_of = [&](uint32_t rd, uint32_t i) { return rd * GC + 8 * i + 2 * (GC < 8 ? kb & 1 : kb); };
  auto load = [&](uint32_t tile, uint32_t rd, Round& v) {
    const uint32_t col = min(tile * 16 + c16, O - 1);
    const uint32_t chunk = min(rd * kWideSteps * 4 + lp, K / 32 - 1) * (BITS * 4);
#pragma unroll
    for (uint32_t i = 0; i < kWideSteps; ++i) {
      const uint8_t* const p = a.w + (uint64_t)min(tile * 16 + 4 * i + lr, O - 1) * row_bytes + chunk;
      if constexpr (BITS == 8) {
        const u32x4 lo = ld_w<true>(reinterpret_cast<const u32x4*>(p)), hi = ld_w<true>(reinterpret_cast<const u32x4*>(p + 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) v.w[i][j] = lo[j], v.w[i][4 + j] = hi[j];
      } else {
        const Raw<BITS> r = load_raw<BITS, true>(p);
#pragma unroll
        for (int j = 0; j < BITS; ++j) v.w[i][j] = r.d[j];
      }
    }
    // Pairs of groups: lane block kb those of pair kb (and 4 + kb); the last
    // two again past the end.
#pragma unroll
    for (uint32_t i = 0; i < PW; ++i) {
      const uint32_t g = group_of(rd, i);
      const uint64_t e = (uint64_t)col * gpr + min(g, gpr - 2);
      __builtin_memcpy(&v.s[i], a.s + e, 4);  // on two bytes
      __builtin_memcpy(&v.b[i], a.b + e, 4);
    }
  };
  const uint32_t stride = gridDim.x * 4;
  uint32_t tile = blockIdx.x * 4 + wave;
  uint32_t rd = 0, lt = tile, ld = 0;  // computed next, loaded next
  auto next = [&](uint32_t& t, uint32_t& r) {
    if (++r == rounds) r = 0, t += stride;
  };
  // Without a branch, or the waits for a round would be for all of them; past
  // the last tile the first again.
  constexpr int D = BITS == 8 ? 2 : 3;
  Round v[D];
  auto ahead = [&](Round& v) {
    load(lt < tiles ? lt : min(tile, tiles - 1), ld, v);
    next(lt, ld);
  };
#pragma unroll
  for (int k = 0; k < D - 1; ++k) ahead(v[k]);

  // The rows as operands; rows past the last and inputs from K on are zero.
  for (uint32_t i = tid; i < steps * 8 * MT * 16; i += 256) {
    const uint32_t p = i % (steps * 8), r = i / (steps * 8);
    u32x4 q = {0u, 0u, 0u, 0u};
    if (r < a.n && p * 16 < K) q = *reinterpret_cast<const u32x4*>(a.x + (uint64_t)r * K + p * 16);
    uint2* const to = reinterpret_cast<uint2*>(xl + ((p / 8) * MT + r / 16) * 128);
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
      uint2 o = make_uint2(q[2 * e], q[2 * e + 1]);
      if (BITS != 8) o = make_uint2(__builtin_amdgcn_perm(o.y, o.x, 0x06040200u), __builtin_amdgcn_perm(o.y, o.x, 0x07050301u));
      to[q8_slot<G>(p % 8, e, r % 16)] = o;
    }
  }
  if constexpr (XG)
    for (uint32_t i = tid; i < groups * MT * 16; i += 256) {
      const uint32_t r = i % (MT * 16), g = i / (MT * 16);
      sxl[i] = r < a.n ? q8_round22(a.sx[(uint64_t)r * gpr + min(g, gpr - 1)] * kQ8Down) : 0.f;
    }
  __syncthreads();
  const uint32_t at[2] = {kb * 16 + (c16 ^ kb), 64 + kb * 16 + (c16 ^ (4 + kb))};
  const u32x4 one = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
  const u32x4 ones[2] = {one, one};
  for (uint32_t i = wave; i < octets * MT; i += 4) {
    const uint32_t o = i / MT, m = i % MT;
    float xs[2] = {0.f, 0.f};
    // All eight, the last group in the place of those behind it (no branch: out
    // of the middle of these the compiler (7.2.0) read the last product's result
    // one instruction after it, where the matrix cores need eight).
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const bool in = o * 8 + j < gpr;
      const uint32_t g = in ? o * 8 + j : gpr - 1;
      const u32x4* const xo = xl + (g / GS * MT + m) * 128;
      const u32x4 x[2] = {xo[at[0]], xo[at[1]]};
      i32x4 S;
      if constexpr (GS == 1)
        S = q8_sums<G>(ones, x, 0);
      else if constexpr (GS == 2)
        S = j & 1 ? q8_sums<G>(ones, x, 1) : q8_sums<G>(ones, x, 0);
      else
        S = j % 4 == 0 ? q8_sums<G>(ones, x, 0) : j % 4 == 1 ? q8_sums<G>(ones, x, 1) : j % 4 == 2 ? q8_sums<G>(ones, x, 2) : q8_sums<G>(ones, x, 3);
      float f = (float)S[0];
      if constexpr (XG) f *= sxl[g * MT * 16 + m * 16 + c16];
      xs[j & 1] = in && kb == j / 2 ? f : xs[j & 1];
    }
    parts[i * 64 + lane] = __builtin_bit_cast(u32x4, q8_parts(xs[0], xs[1]));
  }
  __syncthreads();

  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kStart = XG ? (int)kMagicBits : 0;
  const i32x4 start = {kStart, kStart, kStart, kStart};
  auto from = [&](int src, uint32_t x) { return (uint32_t)__builtin_amdgcn_ds_bpermute(src, (int)x); };
  auto compute = [&](uint32_t rd, Round& v) {
    static_assert(kWideSteps == 4, "16 chunks of a row, four rows per load");
    wave_lds();  // the last round's reads come first
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t r = 4 * i + lr;
#pragma unroll
      for (uint32_t c = 0; c < CW; ++c) {
        u32x4 q = {v.w[i][4 * c], v.w[i][4 * c + 1], v.w[i][4 * c + 2], 0u};
        if (BITS != 3) q.w = v.w[i][(4 * c + 3) % W];
        mine[(r * 16 + (lp ^ r)) * CW + c] = q;
      }
    }
    wave_lds();
    if (gpr & 1) {  // the last group alone, loaded behind the one before
#pragma unroll
      for (uint32_t i = 0; i < PW; ++i)
        if (group_of(rd, i) == gpr - 1) v.s[i] >>= 16, v.b[i] >>= 16;
    }
    // The bias term of this round's eights (G = 128: a round is half of one).
#pragma unroll
    for (uint32_t i = 0; i < PW; ++i) {
      const uint32_t o = rd * GC / 8 + i;
      uint32_t p = v.b[i], q = v.s[i];
      if (GC < 8 && (kb >> 1) != (rd & 1)) p = q = 0;  // the other half's pairs
      auto term = [&](uint32_t p, float f) {
        const u32x4 t = {__builtin_amdgcn_perm(p, p, 0x01000100u), p, __builtin_amdgcn_perm(p, p, 0x03020302u), 0u};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f32x4 z = acc[m];
          if (f != 1.f) z = f32x4{0.f, 0.f, 0.f, 0.f};
          z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, parts[(o * MT + m) * 64 + lane]),
                                                      __builtin_bit_cast(qbf16x8, t), z, 0, 0, 0);
          acc[m] = f != 1.f ? acc[m] + z * f : z;
        }
      };
      term(p, 1.f);
      if (BITS == 8) term(q, 128.f);  // 8-bit codes enter less 128
    }
    uint32_t sw[GC / 2];  // the column's pairs of scales
#pragma unroll
    for (uint32_t i = 0; i < GC / 2; ++i) sw[i] = from((int)(((i % 4) * 16 + c16) * 4), v.s[i / 4]);
#pragma unroll
    for (uint32_t i = 0; i < kWideSteps; ++i) {
      uint32_t d[W];
#pragma unroll
      for (uint32_t c = 0; c < CW; ++c) {
        const u32x4 q = mine[(c16 * 16 + ((i * 4 + kb) ^ c16)) * CW + c];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (4 * c + j < W) d[4 * c + j] = q[j];
      }
      u32x4 w[2];
      q8_operands<BITS, G>(d, w);
      const uint32_t st = rd * kWideSteps + i;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const u32x4* const xo = xl + (st * MT + m) * 128;
        const u32x4 x[2] = {xo[at[0]], xo[at[1]]};
#pragma unroll
        for (uint32_t j = 0; j < GS; ++j) {
          const uint32_t g = i * GS + j, p = sw[g / 2];
          const float s = __uint_as_float(g & 1 ? p & 0xFFFF0000u : p << 16);
          const i32x4 S = q8_sums<G>(x, w, j, start);
          f32x4 sx;
          if constexpr (XG) sx = *reinterpret_cast<const f32x4*>(sxl + (st * GS + j) * MT * 16 + m * 16 + 4 * kb);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float f = XG ? __builtin_fmaf(__int_as_float(S[k]), sx[k], -kMagic * sx[k]) : (float)S[k];
            acc[m][k] = __builtin_fmaf(s, f, acc[m][k]);
          }
        }
      }
    }
  };
  f32x4 sxr[MT];  // the rows' scales
  if constexpr (!XG) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) sxr[m][k] = a.sx[min((uint32_t)(m * 16 + 4 * kb + k), a.n - 1)];
  }
  auto finish = [&](uint32_t tile) {
    const uint32_t col = tile * 16 + c16;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t r = m * 16 + 4 * kb + k;
        if (r < a.n && col < O) a.y[(uint64_t)r * O + col] = acc[m][k] * (XG ? kQ8Up : sxr[m][k]);
      }
      acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  // Rounds of all of the wave's tiles in one sequence.
  while (tile < tiles) {
#pragma unroll
    for (int k = 0; k < D; ++k) {
      ahead(v[(k + D - 1) % D]);
      compute(rd, v[k]);
      if (rd + 1 == rounds) finish(tile);
      next(tile, rd);
      if (tile >= tiles) return;
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: four waves take WM MT tiles of 16 rows x WN NT tiles of 16 columns,
// step after step of 128 inputs; a block is KS of them, each over its share of
// the steps with LDS of its own, for calls of few tiles (one wave per SIMD is
// the latency of its steps, 0.9 us each). 1000 rows 4096 -> 7168 with scales per
// group take 76 us, 775 TOPS. A step's rows go straight into LDS, its codes
// through registers, where they are unpacked once per block instead of once per
// wave; the next step's loads are in flight while a step is computed. Weights
// are the A operand, so a lane ends with four neighbouring columns of one row.
//
// The fold of a group's sums is the largest part of it: two VALU instructions
// per value, 8 per lane and 16 x 16 x 64 product (34 cycles, and the product
// keeps the VALU from issuing for 10 of its 16), 36 of the 76 us. Matrix cores
// are busy 20 % and the VALU 52 % of the time; what the two waves of a SIMD
// wait for beside that (a step's end waits for all its copies and the barrier)
// has not been taken apart. Groups of 128, half the folds, take 67 us, groups of
// 32 126. With scales per group the sums come
// out of the MFMA as floats, 1.5 2^23 + S, by an accumulator that starts as
// that number's bits (|S| < 2^22), and fma(f, sx, -1.5 2^23 sx) = sx S in one
// rounding: the product in the constant is exact for an sx of 22 bits, so sx is
// rounded to those (by 2^-23 of it).
//
// The bias term: a product with ones leaves a group's sum of inputs X in every
// lane of a row, and eight groups' sums times biases are one bf16 MFMA, lane
// block kb holding groups 2 kb and 2 kb + 1 as sx X = h + m + l in three bf16
// (exact: 24 bits) against the bias three times. (v_mfma_f32_16x16x4_f32 on the
// sums as they are takes 64 cycles for four groups: 9 us of 87 at 1000 rows
// 4096 -> 7168.)
// ---------------------------------------------------------------------------
// LDS place (16 bytes) of piece p (16 inputs) of a row's step: the eight pieces
// of a row side by side, exchanged by the row so that eight rows' reads of one
// piece fall in different banks.
__device__ __forceinline__ uint32_t q8_place(uint32_t row, uint32_t p) { return row * 8 + (p ^ (row & 7)); }

template <int BITS, bool XG, int WM, int WN, int MT, int NT>
struct Q8Tile {
  static constexpr uint32_t BM = WM * MT * 16, BN = WN * NT * 16;
  struct Buf {
    u32x4 x[BM * 8], w[BN * 8];
  };
  struct Lds {
    Buf buf[2];
    // Of two fours of groups, by group mod 8: scales, rows' scales; of eight:
    // the packed biases and scales (pairs of groups) of a column.
    float s[2][4][BN], sx[XG ? 2 : 1][XG ? 4 : 1][XG ? BM : 1];
    uint32_t pair[2][BITS == 8 ? 2 : 1][4][BN];  // [octet mod 2][bias, scale][pair][column]
  };
};

template <int BITS, int G, bool XG, int WM, int WN, int MT, int NT, int KS>
__global__ __launch_bounds__(256 * KS, KS == 1 ? 2 : KS) void k_q8_tile(Q8Args a, uint32_t nrb, uint32_t units) {
  using T = Q8Tile<BITS, XG, WM, WN, MT, NT>;
  constexpr uint32_t BM = T::BM, BN = T::BN, GS = kQ8Step / G;
  static_assert(WM * WN == 4, "four waves");
  static_assert(BN % 64 == 0 && BM % 64 == 0, "a wave stages one kind");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const uint32_t share = KS == 1 ? 0u : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  typename T::Lds& lds = reinterpret_cast<typename T::Lds*>(lds_raw)[share];
  const uint32_t tid = KS == 1 ? threadIdx.x : threadIdx.x & 255, lane = tid & 63, c16 = lane & 15, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  // XCD x = blockIdx % 8 takes a contiguous range of the units (rows fastest),
  // so the row blocks of some columns share their weights in one L2.
  const uint32_t per = (units + 7) / 8, u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || u >= units) return;
  const uint32_t row0 = u % nrb * BM, col0 = u / nrb * BN;
  const uint32_t K = a.K, O = a.O, gpr = K / G, steps = (K + kQ8Step - 1) / kQ8Step;
  const uint32_t row_bytes = K / 32 * (BITS * 4);
  const uint32_t rows = min(BM, a.n - row0), cols = min(BN, O - col0);

  // What a thread stages: pieces of 16 inputs of rows, chunks of weight rows
  // (32 codes; 8 bits: 16) and, per eight groups, the scales or biases of a
  // column and half of a row's scales (read step by step, each of these small
  // reads would fetch its line again). Scalar bases of the block and 32-bit
  // offsets of the lane.
  constexpr uint32_t XP = BM * 8 / 256;
  constexpr uint32_t WC = BITS == 8 ? 8 : 4, WP = BN * WC / 256;
  constexpr uint32_t CB = BITS == 8 ? 16 : chunk_bytes<BITS>(), CI = BITS == 8 ? 16 : 32;  // bytes, codes of a chunk
  constexpr uint32_t SP = (2 * BN + 255) / 256, XS = (2 * BM + 255) / 256;
  const int8_t* const xb = a.x + (uint64_t)row0 * K;
  const uint8_t* const wb = a.w + (uint64_t)col0 * row_bytes;
  const uint16_t* const sb = a.s + (uint64_t)col0 * gpr;
  const uint16_t* const bb = a.b + (uint64_t)col0 * gpr;
  const float* const sxb = a.sx + (uint64_t)row0 * (XG ? gpr : 0);
  uint32_t xo[XP], wo[WP], so[SP], sxo[XS];
  const uint32_t xp = (tid & 7) ^ ((tid >> 3) & 7);  // the piece whose place is tid mod 8 (256 threads are whole eights of rows)
#pragma unroll
  for (uint32_t i = 0; i < XP; ++i) xo[i] = min((tid + 256 * i) / 8, rows - 1) * K + xp * 16;
#pragma unroll
  for (uint32_t i = 0; i < WP; ++i) wo[i] = min((tid + 256 * i) / WC, cols - 1) * row_bytes + tid % WC * CB;
  auto s_part = [&](uint32_t i) { return (wave * 64 + 256 * i) / BN; };  // 0: scales, 1: biases
  auto x_part = [&](uint32_t i) { return (wave * 64 + 256 * i) / BM; };  // half of eight groups
#pragma unroll
  for (uint32_t i = 0; i < SP; ++i) so[i] = min((tid + 256 * i) % BN, cols - 1) * gpr;
#pragma unroll
  for (uint32_t i = 0; i < XS; ++i) sxo[i] = min((tid + 256 * i) % BM, rows - 1) * gpr;

  u32x4 wr[WP], sr[SP];
  f32x4 sxr[XS];
  auto load_scales = [&](uint32_t g0) {  // of groups g0 .. g0 + 7, the last repeated behind it
#pragma unroll
    for (uint32_t i = 0; i < SP; ++i) {
      if (s_part(i) > 1) continue;
      const uint16_t* const p = s_part(i) ? bb : sb;
      if (a.svec) {  // gpr is a multiple of 8
        sr[i] = *reinterpret_cast<const u32x4*>(p + g0 + lane_off(so[i]));
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint32_t lo = p[lane_off(so[i] + min(g0 + 2 * j, gpr - 1))], hi = p[lane_off(so[i] + min(g0 + 2 * j + 1, gpr - 1))];
          sr[i][j] = lo | hi << 16;
        }
      }
    }
    if constexpr (XG) {
#pragma unroll
      for (uint32_t i = 0; i < XS; ++i) {
        if (x_part(i) > 1) continue;
        const uint32_t g = g0 + 4 * x_part(i);
        if (a.xvec && g + 4 <= gpr) {
          sxr[i] = *reinterpret_cast<const f32x4*>(sxb + g + lane_off(sxo[i]));
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) sxr[i][j] = sxb[lane_off(sxo[i] + min(g + j, gpr - 1))];
        }
      }
    }
  };
  // TAIL: the step that K ends in. Loads past the end step back into the row
  // (by as many pieces or chunks as they are past it); the codes there become
  // zero in store.
  const uint32_t whole = K / kQ8Step;
  auto load = [&](uint32_t st, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    const uint32_t k0 = st * kQ8Step;
    const int8_t* const x = xb + k0;
    const uint8_t* const w = wb + k0 / 32 * (BITS * 4);
    auto back = [&](uint32_t at, uint32_t n) { return TAIL && at >= n ? at - (n - 1) : 0u; };
    u32x4* const xl = lds.buf[st & 1].x + wave * 64;
#pragma unroll
    for (uint32_t i = 0; i < XP; ++i) dma16(x + lane_off(xo[i] - back(xp, TAIL ? (K - k0) / 16 : 8u) * 16), xl + 256 * i);
#pragma unroll
    for (uint32_t i = 0; i < WP; ++i) {
      const uint8_t* const q = w + lane_off(wo[i] - back(tid % WC, TAIL ? (K - k0) / CI : WC) * CB);
      if constexpr (BITS == 8) {
        wr[i] = *reinterpret_cast<const u32x4*>(q);
      } else {
        const Raw<BITS> r = load_raw<BITS, false>(q);
#pragma unroll
        for (int j = 0; j < BITS; ++j) wr[i][j] = r.d[j];
      }
    }
    if (st * GS % 8 == 0) load_scales(st * GS);
  };
  auto fetch = [&](uint32_t st) {
    if (st < whole)
      load(st, std::false_type{});
    else if (st < steps)
      load(st, std::true_type{});
  };
  auto store = [&](uint32_t st) {
    u32x4* const wl = lds.buf[st & 1].w;
    const bool past = st >= whole && tid % WC >= (K - st * kQ8Step) / CI;
#pragma unroll
    for (uint32_t i = 0; i < WP; ++i) {
      const uint32_t col = (tid + 256 * i) / WC, c = tid % WC;
      if constexpr (BITS == 8) {
        wl[q8_place(col, c)] = past ? u32x4{0u, 0u, 0u, 0u} : wr[i] ^ 0x80808080u;
      } else {
        Raw<BITS> r;
#pragma unroll
        for (int j = 0; j < BITS; ++j) r.d[j] = past ? 0u : wr[i][j];
        uint32_t q[8];  // evens and odds of eight codes
        unpack_bytes(r, q);
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = __builtin_amdgcn_perm(q[2 * j + 1], q[2 * j], 0x05010400u);
          v[2 * j + 1] = __builtin_amdgcn_perm(q[2 * j + 1], q[2 * j], 0x07030602u);
        }
        wl[q8_place(col, 2 * c)] = u32x4{v[0], v[1], v[2], v[3]};
        wl[q8_place(col, 2 * c + 1)] = u32x4{v[4], v[5], v[6], v[7]};
      }
    }
    if (st * GS % 4) return;
    const uint32_t half = st * GS / 4 & 1, octet = st * GS / 8 & 1;
#pragma unroll
    for (uint32_t i = 0; i < SP; ++i) {
      if (s_part(i) > 1) continue;
      const uint32_t col = (tid + 256 * i) % BN;
      if (s_part(i) == 0) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint32_t v = half ? sr[i][2 + j / 2] : sr[i][j / 2];
          lds.s[half][j][col] = __uint_as_float(j & 1 ? v & 0xFFFF0000u : v << 16);
        }
      }
      if (half == 0 && (BITS == 8 || s_part(i) == 1)) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) lds.pair[octet][1 - s_part(i)][j][col] = sr[i][j];
      }
    }
    if constexpr (XG) {
#pragma unroll
      for (uint32_t i = 0; i < XS; ++i) {
        if (x_part(i) != half) continue;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) lds.sx[half][j][(tid + 256 * i) % BM] = q8_round22(sxr[i][j] * kQ8Down);
      }
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kStart = XG ? (int)kMagicBits : 0;
  const i32x4 start = {kStart, kStart, kStart, kStart};
  const u32x4 one = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
  float xs[MT][2];  // sx X of groups 2 kb and 2 kb + 1 of the eight
#pragma unroll
  for (int m = 0; m < MT; ++m) xs[m][0] = xs[m][1] = 0.f;

  auto compute = [&](uint32_t st, bool last) {
    const typename T::Buf& B = lds.buf[st & 1];
    const uint32_t half = st * GS / 4 & 1, g0 = st * GS % 4;
    struct Op {
      u32x4 v[2];  // groups of 128: both operands; of 32: the group's half of one
    };
    // Operand of group j of the step: 16 inputs at 64 h + 16 kb, of groups of 32
    // eight at 32 j + 8 kb.
    auto read = [&](const u32x4* rows16, uint32_t j) {
      Op o;
      if constexpr (G == 32) {
        const uint2 v = reinterpret_cast<const uint2*>(rows16 + q8_place(c16, 2 * j + kb / 2))[kb & 1];
        o.v[0] = u32x4{v.x, v.y, 0u, 0u};
      } else {
        o.v[0] = rows16[q8_place(c16, (G == 64 ? 4 * j : 0u) + kb)];
        if (G == 128) o.v[1] = rows16[q8_place(c16, 4 + kb)];
      }
      return o;
    };
    auto product = [&](const Op& w, const Op& x) {
      if constexpr (G == 128)
        return q8_mfma(w.v[1], x.v[1], q8_mfma(w.v[0], x.v[0], start));
      else if constexpr (G == 64)
        return q8_mfma(w.v[0], x.v[0], start);
      else
        return q8_mfma32(w.v[0].x, w.v[0].y, x.v[0].x, x.v[0].y, start);
    };
    const Op ones{{one, one}};
#pragma unroll
    for (uint32_t j = 0; j < GS; ++j) {
      Op x[MT], w[2];
      float sx[MT], cx[MT];
      f32x4 s[2];
      i32x4 S[2];
      // The sum S times the row's scale of this group.
      auto value = [&](int32_t v, int m) {
        if constexpr (XG)
          return __builtin_fmaf(__int_as_float(v), sx[m], cx[m]);
        else
          return (float)v;
      };
      auto read_w = [&](int t) {
        w[t & 1] = read(B.w + (wn * NT + t) * 128, j);
        s[t & 1] = *reinterpret_cast<const f32x4*>(&lds.s[half][g0 + j][(wn * NT + t) * 16 + 4 * kb]);
      };
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        x[m] = read(B.x + (wm * MT + m) * 128, j);
        if constexpr (XG) {
          sx[m] = lds.sx[half][g0 + j][(wm * MT + m) * 16 + c16];
          cx[m] = -kMagic * sx[m];
        }
      }
      read_w(0);
      // Units (column tile t, row tile m), m fastest, the product with ones
      // behind them: a unit's product is issued ahead of the fold of the one
      // before it.
      constexpr int UNITS = (NT + 1) * MT;
      auto issue = [&](int u) {
        const int t = u / MT, m = u % MT;
        S[u & 1] = product(t < NT ? w[t & 1] : ones, x[m]);
      };
      issue(0);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int t = u / MT, m = u % MT;
        if (m == 0 && t + 1 < NT) read_w(t + 1);
        if (u + 1 < UNITS) {
          issue(u + 1);
          // Holds the product ahead of this fold (it would be placed at its
          // use, with the fold waiting for it).
          asm volatile("" : "+v"(S[0]), "+v"(S[1]));
        }
        if (t < NT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][t][i] = __builtin_fmaf(s[t & 1][i], value(S[u & 1][i], m), acc[m][t][i]);
        } else {
          const uint32_t g = st * GS + j;
          const float v = g < gpr ? value(S[u & 1][0], m) : 0.f;
          const bool mine = kb == (g / 2 & 3);
          if (g & 1)
            xs[m][1] = mine ? v : xs[m][1];
          else
            xs[m][0] = mine ? v : xs[m][0];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const uint32_t g1 = (st + 1) * GS;  // groups done
    if (g1 % 8 == 0 || last) {
      const uint32_t octet = (g1 - 1) / 8 & 1;
      auto term = [&](uint32_t which, float f) {
        qbf16x8 xv[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xv[m] = q8_parts(xs[m][0] * f, xs[m][1] * f);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t p = lds.pair[octet][which][kb][(wn * NT + t) * 16 + c16];
          const uint32_t lo = __builtin_amdgcn_perm(p, p, 0x01000100u), hi = __builtin_amdgcn_perm(p, p, 0x03020302u);
          const qbf16x8 bv = __builtin_bit_cast(qbf16x8, u32x4{lo, p, hi, 0u});
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv, xv[m], acc[m][t], 0, 0, 0);
        }
      };
      term(0, 1.f);
      if (BITS == 8) term(1, 128.f);  // 8-bit codes entered less 128
#pragma unroll
      for (int m = 0; m < MT; ++m) xs[m][0] = xs[m][1] = 0.f;
    }
  };

  // A share starts with a whole eight of groups.
  constexpr uint32_t ALIGN = GS >= 8 ? 1 : 8 / GS;
  const uint32_t each = KS == 1 ? steps : ((steps + KS - 1) / KS + ALIGN - 1) / ALIGN * ALIGN;
  const uint32_t first = KS == 1 ? 0u : share * each, end = KS == 1 ? steps : min(first + each, steps);
  if (KS == 1 || first < end) {
    fetch(first);
    store(first);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows' copies into LDS
  __syncthreads();
  for (uint32_t i = 0; i < each; ++i) {  // as many barriers in every share
    const uint32_t st = first + i;
    if (KS == 1 || st + 1 < end) fetch(st + 1);  // nothing past the last step
    if (KS == 1 || st < end) compute(st, st + 1 == end);
    if (st + 1 < end) store(st + 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  if constexpr (KS > 1) {  // the shares' parts, over their LDS
    f32x4* const part = reinterpret_cast<f32x4*>(lds_raw);
    if (share) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[((share - 1) * MT * NT + m * NT + t) * 256 + tid] = acc[m][t];
    }
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < KS - 1; ++k) acc[m][t] += part[(k * MT * NT + m * NT + t) * 256 + tid];
  }

  float scale[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) scale[m] = XG ? kQ8Up : a.sx[min(row0 + (wm * MT + m) * 16 + c16, a.n - 1)];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t r = row0 + (wm * MT + m) * 16 + c16;
    if (r >= a.n) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t col = col0 + (wn * NT + t) * 16 + 4 * kb;
      float* const y = a.y + (uint64_t)r * O + col;
      const f32x4 v = acc[m][t] * scale[m];
      if (a.vec) {
        if (col < O) *reinterpret_cast<f32x4*>(y) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < O) y[i] = v[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
template <int BITS, int G, bool XG, int WM, int WN, int MT, int NT, int KS>
static hipError_t q8_tile(const Q8Args& a, hipStream_t st) {
  using T = Q8Tile<BITS, XG, WM, WN, MT, NT>;
  const uint32_t nrb = (a.n + T::BM - 1) / T::BM, units = nrb * ((a.O + T::BN - 1) / T::BN);
  constexpr uint32_t lds = KS * sizeof(typename T::Lds);
  static_assert(lds <= 160 * 1024 && (KS - 1) * MT * NT * 4096 <= lds, "the shares' LDS");
  auto fn = k_q8_tile<BITS, G, XG, WM, WN, MT, NT, KS>;
  if (lds > 64 * 1024) {
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(fn), lds, raised);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3((units + 7) / 8 * 8), dim3(256 * KS), lds, st, a, nrb, units);
  return hipGetLastError();
}

template <int BITS, int G, bool XG, int MT, int NT>
static hipError_t q8_few(const Q8Args& a, uint32_t waves, hipStream_t st) {
  const dim3 grid((a.O + NT * 16 - 1) / (NT * 16), (a.n + MT * 16 - 1) / (MT * 16));
  hipLaunchKernelGGL((k_q8_few<BITS, G, XG, MT, NT>), grid, dim3(waves * 64), waves * MT * NT * 1024, st, a);
  return hipGetLastError();
}

template <int BITS, int G, bool XG, int MT>
static hipError_t q8_wide(const Q8Args& a, hipStream_t st) {
  const uint32_t lds = q8_wide_lds(BITS, a.K, G, MT, XG), tiles = (a.O + 15) / 16;
  auto fn = k_q8_wide<BITS, G, XG, MT>;
  if (lds > 64 * 1024) {
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(fn), 160 * 1024, raised);
    if (e != hipSuccess) return e;
  }
  // Two blocks on each CU (one where the rows fill its LDS), every wave as
  // many tiles.
  const uint32_t slots = 256 * (lds > 80 * 1024 ? 1 : 2) * 4, rounds = (tiles + slots - 1) / slots;
  const uint32_t blocks = (tiles + 4 * rounds - 1) / (4 * rounds);
  hipLaunchKernelGGL(fn, dim3(blocks), dim3(256), lds, st, a, tiles);
  return hipGetLastError();
}

// Which kernel, by how many blocks there are for the 256 CUs. Times in us, 4
// bits, groups of 64, row scales, graph replays; n rows K -> O. Over 630 calls
// of all bits and groups drawn from 1 to 1000 rows, 150 to 60000 columns, 512
// to 7168 inputs the chosen kernel took 1.03 times the fastest one's time; of the
// two tiles of 64 and 128, over 235 calls of 17 to 1000 rows and 4000 to 152000
// columns, 1.01 times.
template <int BITS, int G, bool XG>
static hipError_t q8_go(const Q8Args& a, hipStream_t st) {
  const uint32_t steps = (a.K + kQ8Step - 1) / kQ8Step;
  const uint64_t rt = (a.n + 15) / 16, ct = (a.O + 15) / 16;  // row and column tiles
  auto units = [&](uint32_t m, uint32_t n) { return (uint64_t)((a.n + m - 1) / m) * ((a.O + n - 1) / n); };
  const uint64_t u64 = units(64, 64), u128 = units(128, 128);
  // Whether s shares of the steps all have some (they start on eight groups).
  auto shares = [&](uint32_t s) { return steps >= s * (8 * G / kQ8Step); };
  // One tile a block, all steps at once (16 rows 2048 -> 4096: 5.1, two column
  // tiles a block 6.3; 32 rows: 7.2 and, two row tiles a block, 6.1).
  if (rt * ct <= 256) return q8_few<BITS, G, XG, 1, 1>(a, std::min(steps, 16u), st);
  if (rt == 1) {
    // 16 rows 2048 -> 16384, weights from HBM: 10.0, rows in LDS 10.1; -> 24576:
    // 13.7 and 12.6; -> 32768: 16.8 and 13.5. Rows that do not fit a CU's LDS
    // fall back (8192 -> 151936: 277 with scales per group, which do not, 154
    // with scales per row, which do).
    if (ct <= 1024 || a.K < 2 * G || q8_wide_lds(BITS, a.K, G, 1, XG) > 160 * 1024)
      return q8_few<BITS, G, XG, 1, 2>(a, std::min(steps, 8u), st);
    return q8_wide<BITS, G, XG, 1>(a, st);
  }
  // Two tiles a block, side by side where that wastes less (64 rows 7168 ->
  // 2048: 11.0, four tiles 14.3; 45 rows 2048 -> 2560: 6.5 and 8.1), or four
  // (64 rows 2048 -> 4096: 7.8, two tiles 8.3).
  const uint64_t b21 = (rt + 1) / 2 * ct, b12 = rt * ((ct + 1) / 2), b22 = (rt + 1) / 2 * ((ct + 1) / 2);
  if (b21 <= 256 && b21 <= b12) return q8_few<BITS, G, XG, 2, 1>(a, std::min(steps, 8u), st);
  if (b12 <= 256) return q8_few<BITS, G, XG, 1, 2>(a, std::min(steps, 8u), st);
  if (b22 <= 256) return q8_few<BITS, G, XG, 2, 2>(a, std::min(steps, 8u), st);
  // Fewer waves each for somewhat more blocks, while 64 x 64 tiles would leave
  // CUs idle (200 rows 7168 -> 2048, 448 blocks: 24.3, staged 27.7), and for
  // short sums, which have no steps to share (200 rows 512 -> 2048: 5.4, staged
  // 7.1; 400 rows: 7.6 and 7.1).
  if (b22 <= (steps < 8 ? 640u : 448u)) return q8_few<BITS, G, XG, 2, 2>(a, std::min(steps, 4u), st);
  // 64 x 64 tiles, four shares while their blocks fit the chip at once, then
  // two (200 rows 2048 -> 4096, 256 tiles: 11.1, two shares 12.7, one 17.5; 400
  // rows, 448: 19.5, 17.2, 20.4).
  if (u64 <= 256 && shares(4)) return q8_tile<BITS, G, XG, 2, 2, 2, 2, 4>(a, st);
  if (u64 <= 512 && shares(2)) return q8_tile<BITS, G, XG, 2, 2, 2, 2, 2>(a, st);
  // 128 x 128 where they fill the chip with two shares each (1000 rows 2048 ->
  // 4096, 256 tiles: 27.0, 64 x 64 29.9) or two blocks on most CUs (1000 rows
  // 4096 -> 7168, 448: 78 and 89; 600 rows 4096 -> 8192, 320: 70 and 64), but
  // for short sums (140 rows 512 -> 43682: 32 and 25) that 64 x 64 tiles have
  // blocks for, and where they hold fewer rows or columns than they have room
  // for: a tile of 128 takes 3.4 times one of 64 (64 rows 2048 -> 151936: 88 and
  // 64; 65 rows: 89 and 110; 130 rows: 169 and 153).
  if (u128 > 192 && u128 <= 256 && shares(2)) return q8_tile<BITS, G, XG, 2, 2, 4, 4, 2>(a, st);
  if (u128 > 384 && ((steps >= 8 && 10 * u64 >= 34 * u128) || u64 > kQ8MaxBlocks)) return q8_tile<BITS, G, XG, 2, 2, 4, 4, 1>(a, st);
  return q8_tile<BITS, G, XG, 2, 2, 2, 2, 1>(a, st);
}

template <int BITS>
hipError_t q8_launch(const Q8Args& a, uint32_t group, bool x_grouped, hipStream_t st) {
  if (x_grouped)
    return group == 32 ? q8_go<BITS, 32, true>(a, st) : group == 64 ? q8_go<BITS, 64, true>(a, st) : q8_go<BITS, 128, true>(a, st);
  return group == 32 ? q8_go<BITS, 32, false>(a, st) : group == 64 ? q8_go<BITS, 64, false>(a, st) : q8_go<BITS, 128, false>(a, st);
}

}  // namespace smoe

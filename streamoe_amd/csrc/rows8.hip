// rows8.hip — quantized products of 8-bit rows on the int8 matrix cores.
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
#include "common.h"
#include "kernels.h"

#include <type_traits>

namespace smoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kQ8Step = 128;

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

// First input (of a step) of the e-th eight of operand h at lane block kb.
template <int BITS, int G>
__device__ __forceinline__ uint32_t q8_pos(uint32_t h, uint32_t e, uint32_t kb) {
  if (G == 32) return 64 * h + 8 * kb + 32 * e;
  if (BITS == 8) return 64 * h + 16 * kb + 8 * e;
  if (G == 64) return 64 * h + 32 * (kb & 1) + 16 * (kb >> 1) + 8 * e;
  return 32 * kb + 16 * h + 8 * e;
}

// The rows' operands of a step; inputs from K on are zero.
template <int BITS, int G>
__device__ __forceinline__ void q8_load_x(const int8_t* row, uint32_t k0, uint32_t K, uint32_t kb, u32x4 (&x)[2]) {
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    uint2 v[2];
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
      const uint32_t at = k0 + q8_pos<BITS, G>(h, e, kb);
      v[e] = make_uint2(0u, 0u);
      if (at < K) v[e] = *reinterpret_cast<const uint2*>(row + at);
      if (BITS != 8) {
        const uint2 n = v[e];
        v[e].x = __builtin_amdgcn_perm(n.y, n.x, 0x06040200u);
        v[e].y = __builtin_amdgcn_perm(n.y, n.x, 0x07050301u);
      }
    }
    x[h] = u32x4{v[0].x, v[0].y, v[1].x, v[1].y};
  }
}

// The codes of weight row `row` of a step as operands (past K: any codes).
template <int BITS, int G>
__device__ __forceinline__ void q8_load_w(const uint8_t* row, uint32_t k0, uint32_t K, uint32_t kb, u32x4 (&b)[2]) {
  if constexpr (BITS == 8) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      uint2 v[2];
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e)
        v[e] = *reinterpret_cast<const uint2*>(row + min(k0 + q8_pos<BITS, G>(h, e, kb), K - 8));
      b[h] = u32x4{v[0].x, v[0].y, v[1].x, v[1].y} ^ 0x80808080u;
    }
  } else {
    Raw<BITS> w = load_raw<BITS, false>(row + min(k0 / 32 + kb, K / 32 - 1) * chunk_bytes<BITS>());
    if constexpr (G == 64 && BITS == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(w.d[i], w.d[i + 2], false, false);
        w.d[i] = r[0];
        w.d[i + 2] = r[1];
      }
    }
    if constexpr (G == 32 && BITS == 4) q8_transpose4(w.d[0], w.d[1], w.d[2], w.d[3]);
    uint32_t q[8];
    unpack_bytes(w, q);
    if constexpr (G == 64 && BITS == 3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(q[i], q[i + 4], false, false);
        q[i] = r[0];
        q[i + 4] = r[1];
      }
    }
    if constexpr (G == 32 && BITS == 3) {
      q8_transpose4(q[0], q[2], q[4], q[6]);
      q8_transpose4(q[1], q[3], q[5], q[7]);
    }
    b[0] = u32x4{q[0], q[1], q[2], q[3]};
    b[1] = u32x4{q[4], q[5], q[6], q[7]};
  }
}

// Sums of group g of a step.
template <int G>
__device__ __forceinline__ i32x4 q8_sums(const u32x4 (&x)[2], const u32x4 (&b)[2], uint32_t g) {
  const i32x4 z = {0, 0, 0, 0};
  if constexpr (G == 64) {
    return q8_mfma(x[g], b[g], z);
  } else if constexpr (G == 32) {
    const uint32_t h = g / 2, o = g % 2 * 2;
    return q8_mfma32(x[h][o], x[h][o + 1], b[h][o], b[h][o + 1], z);
  } else {
    return q8_mfma(x[1], b[1], q8_mfma(x[0], b[0], z));
  }
}

// A block: 16 rows x NT tiles of 16 columns, its four waves taking the steps
// in turn; the sums of the inputs come from a product with ones.
template <int BITS, int G, bool XG, int NT>
__global__ __launch_bounds__(256) void k_q8(Q8Args a) {
  constexpr uint32_t GS = kQ8Step / G;
  __shared__ f32x4 red[4][NT][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, kb = lane >> 4;
  const uint32_t K = a.K, O = a.O, gpr = K / G, steps = (K + kQ8Step - 1) / kQ8Step;
  const uint32_t col0 = blockIdx.x * (NT * 16), row0 = blockIdx.y * 16;
  const uint32_t row_bytes = K / 32 * (BITS * 4);
  const int8_t* const xr = a.x + (uint64_t)min(row0 + c16, a.n - 1) * K;
  const uint8_t* wr[NT];
  const uint16_t *sr[NT], *br[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t c = min(col0 + t * 16 + c16, O - 1);
    wr[t] = a.w + (uint64_t)c * row_bytes;
    sr[t] = a.s + (uint64_t)c * gpr;
    br[t] = a.b + (uint64_t)c * gpr;
  }
  const float* sx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sx[i] = a.sx + (uint64_t)min(row0 + 4 * kb + i, a.n - 1) * (XG ? gpr : 1u);
  const u32x4 one = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
  const u32x4 ones[2] = {one, one};
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t st = wave; st < steps; st += 4) {
    const uint32_t k0 = st * kQ8Step;
    u32x4 x[2], w[NT][2];
    q8_load_x<BITS, G>(xr, k0, K, kb, x);
#pragma unroll
    for (int t = 0; t < NT; ++t) q8_load_w<BITS, G>(wr[t], k0, K, kb, w[t]);
#pragma unroll
    for (uint32_t j = 0; j < GS; ++j) {
      const uint32_t g = min(st * GS + j, gpr - 1);
      const i32x4 X = q8_sums<G>(x, ones, j);
      f32x4 xf, xs;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xs[i] = XG ? sx[i][g] : 1.f;
        xf[i] = xs[i] * (float)X[i];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float s = bf16f(sr[t][g]);
        float b = bf16f(br[t][g]);
        if (BITS == 8) b = __builtin_fmaf(s, 128.f, b);
        const i32x4 S = q8_sums<G>(x, w[t], j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[t][i] = __builtin_fmaf(s * xs[i], (float)S[i], acc[t][i]);
          acc[t][i] = __builtin_fmaf(b, xf[i], acc[t][i]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  for (uint32_t t = wave; t < NT; t += 4) {
    const f32x4 v = (red[0][t][lane] + red[1][t][lane]) + (red[2][t][lane] + red[3][t][lane]);
    const uint32_t col = col0 + t * 16 + c16;
    if (col >= O) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = row0 + 4 * kb + i;
      if (r < a.n) a.y[(uint64_t)r * O + col] = XG ? v[i] : v[i] * sx[i][0];
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: a block of four waves takes WM MT tiles of 16 rows x WN NT tiles
// of 16 columns, step after step of 128 inputs. A step's rows and codes go
// through registers into LDS in operand order (a wave's operand is 1 KB that
// the lanes read in lane order), the codes unpacked and the rows' bytes put in
// their order once per block instead of once per wave; the next step's loads
// are in flight while a step is computed. Weights are the A operand, so a lane
// ends with four neighbouring columns of one row.
//
// The fold of a group's sums is what bounds it: two VALU instructions per
// value (16 x 16 x 64: 8 per lane, 32 cycles, against 16 on the matrix cores).
// With scales per group the sums come out of the MFMA as floats, 1.5 2^23 + S,
// by an accumulator that starts as that number's bits (|S| < 2^22), and
// fma(f, sx, -1.5 2^23 sx) = sx S in one rounding: the product in the constant
// is exact for an sx of 22 bits, so sx is rounded to those (by 2^-23 of it).
// The bias term runs on v_mfma_f32_16x16x4_f32, four groups at a time, over the
// rows' group sums, which a product with ones leaves in every lane of a row.
// ---------------------------------------------------------------------------
constexpr uint32_t kMagicBits = 0x4B400000u;  // 1.5 * 2^23
constexpr float kMagic = 12582912.f;

// sx to 22 significant bits.
__device__ __forceinline__ float q8_round22(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7F800000u) == 0x7F800000u) return v;
  return __uint_as_float((u + 1u + ((u >> 2) & 1u)) & ~3u);
}

// Where the e-th eight of piece p (16 inputs) of a row's step lies in operand
// order: [h][kb][row][e], 8-byte units for rows of 16 (see q8_pos). The row's
// place is exchanged by 4 h + kb, so that the pieces of a row, which
// neighbouring lanes write, fall in different banks (8 writes to one: 33 of
// 54 % of the LDS cycles were conflicts).
template <int BITS, int G>
__device__ __forceinline__ uint32_t q8_slot(uint32_t p, uint32_t e, uint32_t row) {
  uint32_t h, kb, f = e;
  if (G == 32) {
    h = p >> 2, kb = (p & 1) * 2 + e, f = (p >> 1) & 1;
  } else if (BITS == 8) {
    h = p >> 2, kb = p & 3;
  } else if (G == 64) {
    h = p >> 2, kb = ((p & 1) << 1) | ((p >> 1) & 1);
  } else {
    h = p & 1, kb = p >> 1;
  }
  return ((h * 4 + kb) * 16 + (row ^ (h * 4 + kb))) * 2 + f;
}

template <int BITS, int G, bool XG, int WM, int WN, int MT, int NT>
struct Q8Tile {
  static constexpr uint32_t BM = WM * MT * 16, BN = WN * NT * 16, GS = kQ8Step / G;
  struct Buf {
    u32x4 x[BM * 8], w[BN * 8];
    float s[GS][BN];
    float sx[XG ? 2 * GS : 1][XG ? BM : 1];  // sx, then -1.5 2^23 sx
  };
  struct Lds {
    Buf buf[2];
    float b[2][4][BN];  // biases, by group mod 4
  };
};

template <int BITS, int G, bool XG, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(256, 2) void k_q8_tile(Q8Args a, uint32_t nrb, uint32_t units) {
  using T = Q8Tile<BITS, G, XG, WM, WN, MT, NT>;
  constexpr uint32_t BM = T::BM, BN = T::BN, GS = T::GS;
  static_assert(WM * WN == 4, "four waves");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  typename T::Lds& lds = *reinterpret_cast<typename T::Lds*>(lds_raw);
  const uint32_t tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  // XCD x = blockIdx % 8 takes a contiguous range of the units (rows fastest),
  // so the row blocks of some columns share their weights in one L2.
  const uint32_t per = (units + 7) / 8, u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || u >= units) return;
  const uint32_t row0 = u % nrb * BM, col0 = u / nrb * BN;
  const uint32_t K = a.K, O = a.O, gpr = K / G, steps = (K + kQ8Step - 1) / kQ8Step;
  const uint32_t row_bytes = K / 32 * (BITS * 4);

  // What a thread stages: pieces of 16 inputs of rows, chunks of weight rows
  // (32 codes; 8 bits: 16), scales and biases, rows' scales.
  constexpr uint32_t XP = BM * 8 / 256;
  constexpr uint32_t WC = BITS == 8 ? 8 : 4, WP = BN * WC / 256;
  constexpr uint32_t SP = (GS * BN + 255) / 256, XS = XG ? (GS * BM + 255) / 256 : 1;
  static_assert(BM * 8 % 256 == 0 && BN * WC % 256 == 0, "whole pieces per thread");
  // A wave's 16 cols x 4 chunks in an order whose eights of lanes write to
  // different banks (columns c and c + 2 side by side).
  auto w_col = [](uint32_t id) {
    const uint32_t c = id / WC;
    return BITS == 8 ? c : (c & ~3u) | ((c & 1) << 1) | ((c >> 1) & 1);
  };
  // Scalar bases of the block and 32-bit offsets of the lane.
  const int8_t* const xb = a.x + (uint64_t)row0 * K;
  const uint8_t* const wb = a.w + (uint64_t)col0 * row_bytes;
  const uint16_t* const sb = a.s + (uint64_t)col0 * gpr;
  const uint16_t* const bb = a.b + (uint64_t)col0 * gpr;
  const float* const sxb = a.sx + (uint64_t)row0 * (XG ? gpr : 0);
  const uint32_t rows = min(BM, a.n - row0), cols = min(BN, O - col0);
  uint32_t xo[XP], wo[WP], so[SP], sxo[XS];
#pragma unroll
  for (uint32_t i = 0; i < XP; ++i) xo[i] = min((tid + 256 * i) / 8, rows - 1) * K + (tid & 7) * 16;
#pragma unroll
  for (uint32_t i = 0; i < WP; ++i) {
    const uint32_t id = tid + 256 * i;
    wo[i] = min(w_col(id), cols - 1) * row_bytes + id % WC * (BITS == 8 ? 16 : chunk_bytes<BITS>());
  }
#pragma unroll
  for (uint32_t i = 0; i < SP; ++i) {
    const uint32_t id = tid + 256 * i;
    so[i] = min(id % BN, cols - 1) * gpr + min(id / BN, GS - 1);
  }
#pragma unroll
  for (uint32_t i = 0; i < XS; ++i) {
    const uint32_t id = tid + 256 * i;
    sxo[i] = min(id % BM, rows - 1) * gpr + min(id / BM, GS - 1);
  }
  u32x4 xr[XP], wr[WP];
  float sr[SP], br[SP], sxr[XS];
  // TAIL: the step that K ends in. Loads past the end step back into the row
  // (by as many pieces, chunks or groups as they are past it); inputs there
  // are zero.
  auto load = [&](uint32_t st, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    const uint32_t k0 = st * kQ8Step, g0 = st * GS, ng = TAIL ? gpr - g0 : GS;
    const int8_t* const x = xb + k0;
    const uint8_t* const w = wb + k0 / 32 * (BITS * 4);
    auto back = [&](uint32_t at, uint32_t n) { return TAIL && at >= n ? at - (n - 1) : 0u; };
#pragma unroll
    for (uint32_t i = 0; i < XP; ++i) {
      const uint32_t p = tid & 7, np = TAIL ? (K - k0) / 16 : 8u;
      xr[i] = *reinterpret_cast<const u32x4*>(x + lane_off(xo[i] - back(p, np) * 16));
      if (TAIL && p >= np) xr[i] = u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (uint32_t i = 0; i < WP; ++i) {
      constexpr uint32_t CB = BITS == 8 ? 16 : chunk_bytes<BITS>(), CI = BITS == 8 ? 16 : 32;
      const uint8_t* const q = w + lane_off(wo[i] - back(tid % WC, TAIL ? (K - k0) / CI : WC) * CB);
      if constexpr (BITS == 8) {
        wr[i] = *reinterpret_cast<const u32x4*>(q);
      } else {
        const Raw<BITS> r = load_raw<BITS, false>(q);
#pragma unroll
        for (int j = 0; j < BITS; ++j) wr[i][j] = r.d[j];
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < SP; ++i) {
      const uint32_t o = lane_off(so[i] - back(min((tid + 256 * i) / BN, GS - 1), ng));
      sr[i] = bf16f((sb + g0)[o]);
      br[i] = bf16f((bb + g0)[o]);
    }
    if constexpr (XG) {
#pragma unroll
      for (uint32_t i = 0; i < XS; ++i)
        sxr[i] = (sxb + g0)[lane_off(sxo[i] - back(min((tid + 256 * i) / BM, GS - 1), ng))];
    }
  };
  auto store = [&](uint32_t st) {
    typename T::Buf& B = lds.buf[st & 1];
    uint2* const x8 = reinterpret_cast<uint2*>(B.x);
    uint2* const w8 = reinterpret_cast<uint2*>(B.w);
#pragma unroll
    for (uint32_t i = 0; i < XP; ++i) {
      const uint32_t id = tid + 256 * i, row = id / 8, p = id % 8;
      uint2 v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t lo = xr[i][2 * e], hi = xr[i][2 * e + 1];
        v[e] = BITS == 8 ? make_uint2(lo, hi)
                         : make_uint2(__builtin_amdgcn_perm(hi, lo, 0x06040200u), __builtin_amdgcn_perm(hi, lo, 0x07050301u));
      }
      const uint32_t tile = row / 16 * 256, r16 = row % 16;
      if constexpr (G == 32) {
        x8[tile + q8_slot<BITS, G>(p, 0, r16)] = v[0];
        x8[tile + q8_slot<BITS, G>(p, 1, r16)] = v[1];
      } else {
        B.x[(tile + q8_slot<BITS, G>(p, 0, r16)) / 2] = u32x4{v[0].x, v[0].y, v[1].x, v[1].y};
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < WP; ++i) {
      const uint32_t id = tid + 256 * i, col = w_col(id), c = id % WC;
      const uint32_t tile = col / 16 * 256, r16 = col % 16;
      if constexpr (BITS == 8) {
        const u32x4 v = wr[i] ^ 0x80808080u;
        if constexpr (G == 32) {
          w8[tile + q8_slot<BITS, G>(c, 0, r16)] = make_uint2(v.x, v.y);
          w8[tile + q8_slot<BITS, G>(c, 1, r16)] = make_uint2(v.z, v.w);
        } else {
          B.w[(tile + q8_slot<BITS, G>(c, 0, r16)) / 2] = v;
        }
      } else {
        Raw<BITS> r;
#pragma unroll
        for (int j = 0; j < BITS; ++j) r.d[j] = wr[i][j];
        uint32_t q[8];
        unpack_bytes(r, q);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          if constexpr (G == 32) {
            w8[tile + q8_slot<BITS, G>(2 * c + h, 0, r16)] = make_uint2(q[4 * h], q[4 * h + 1]);
            w8[tile + q8_slot<BITS, G>(2 * c + h, 1, r16)] = make_uint2(q[4 * h + 2], q[4 * h + 3]);
          } else {
            B.w[(tile + q8_slot<BITS, G>(2 * c + h, 0, r16)) / 2] = u32x4{q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]};
          }
        }
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < SP; ++i) {
      const uint32_t id = tid + 256 * i, col = id % BN, j = id / BN, g = st * GS + j;
      if (GS * BN % 256 && j >= GS) continue;
      B.s[j][col] = sr[i];
      lds.b[(g >> 2) & 1][g & 3][col] = BITS == 8 ? __builtin_fmaf(sr[i], 128.f, br[i]) : br[i];
    }
    if constexpr (XG) {
#pragma unroll
      for (uint32_t i = 0; i < XS; ++i) {
        const uint32_t id = tid + 256 * i, row = id % BM, j = id / BM;
        if (GS * BM % 256 && j >= GS) continue;
        const float sx = q8_round22(sxr[i]);
        B.sx[j][row] = sx;
        B.sx[GS + j][row] = -kMagic * sx;
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
  float xs[MT];  // the row's group sums, lane block kb that of group 4 q + kb
#pragma unroll
  for (int m = 0; m < MT; ++m) xs[m] = 0.f;
  auto compute = [&](uint32_t st) {
    const typename T::Buf& B = lds.buf[st & 1];
    // The lane's place in operand h (q8_slot).
    const uint32_t at[2] = {kb * 16 + (c16 ^ kb), 64 + kb * 16 + (c16 ^ (4 + kb))};
    const u32x4* const xt = B.x + wm * MT * 128;
    const u32x4* const wt = B.w + wn * NT * 128;
#pragma unroll
    for (uint32_t j = 0; j < GS; ++j) {
      u32x4 x[MT][2];  // G = 128: both operands
      float sx[MT], cx[MT];
      auto product = [&](const u32x4 (&w)[2], int m) {
        if constexpr (G == 128)
          return q8_mfma(w[1], x[m][1], q8_mfma(w[0], x[m][0], start));
        else if constexpr (G == 64)
          return q8_mfma(w[0], x[m][0], start);
        else
          return q8_mfma32(w[0].x, w[0].y, x[m][0].x, x[m][0].y, start);
      };
      // The sum S times the row's scale of this group.
      auto value = [&](int32_t S, int m) {
        if constexpr (XG)
          return __builtin_fmaf(__int_as_float(S), sx[m], cx[m]);
        else
          return (float)S;
      };
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (G == 128) {
          x[m][0] = xt[m * 128 + at[0]];
          x[m][1] = xt[m * 128 + at[1]];
        } else if constexpr (G == 64) {
          x[m][0] = xt[m * 128 + at[j]];
        } else {
          const uint2 v = reinterpret_cast<const uint2*>(xt + m * 128 + at[j / 2])[j % 2];
          x[m][0].x = v.x;
          x[m][0].y = v.y;
        }
        if constexpr (XG) {
          sx[m] = B.sx[j][wm * MT * 16 + m * 16 + c16];
          cx[m] = B.sx[GS + j][wm * MT * 16 + m * 16 + c16];
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&B.s[j][wn * NT * 16 + t * 16 + 4 * kb]);
        u32x4 w[2];
        if constexpr (G == 128) {
          w[0] = wt[t * 128 + at[0]];
          w[1] = wt[t * 128 + at[1]];
        } else if constexpr (G == 64) {
          w[0] = wt[t * 128 + at[j]];
        } else {
          const uint2 v = reinterpret_cast<const uint2*>(wt + t * 128 + at[j / 2])[j % 2];
          w[0].x = v.x;
          w[0].y = v.y;
        }
        i32x4 S[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) S[m] = product(w, m);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][t][i] = __builtin_fmaf(s[i], value(S[m][i], m), acc[m][t][i]);
      }
      const u32x4 ones[2] = {one, one};
      const bool mine = kb == ((st * GS + j) & 3);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float v = value(product(ones, m)[0], m);
        xs[m] = mine ? v : xs[m];
      }
    }
    const uint32_t g1 = (st + 1) * GS;  // groups staged so far
    if ((g1 & 3) == 0 || st + 1 == steps) {
      const uint32_t ring = ((g1 - 1) >> 2) & 1;
      // In the last four, groups that do not exist count nothing.
      const bool live = g1 - ((g1 - 1) & 3) - 1 + kb < g1;
      float b[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b[t] = lds.b[ring][kb][wn * NT * 16 + t * 16 + c16];
        b[t] = live ? b[t] : 0.f;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[t], xs[m], acc[m][t], 0, 0, 0);
        xs[m] = 0.f;
      }
    }
  };

  const uint32_t whole = K / kQ8Step;  // steps without a tail
  auto fetch = [&](uint32_t st) {
    if (st < whole)
      load(st, std::false_type{});
    else if (st < steps)
      load(st, std::true_type{});
  };
  fetch(0);
  store(0);
  __syncthreads();
  for (uint32_t st = 0; st < steps; ++st) {
    fetch(st + 1);
    compute(st);
    if (st + 1 < steps) store(st + 1);
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t r = row0 + (wm * MT + m) * 16 + c16;
    if (r >= a.n) continue;
    const float sx = XG ? 1.f : a.sx[r];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t col = col0 + (wn * NT + t) * 16 + 4 * kb;
      float* const y = a.y + (uint64_t)r * O + col;
      const f32x4 v = acc[m][t] * sx;
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
template <int BITS, int G, bool XG, int WM, int WN, int MT, int NT>
static hipError_t q8_tile(const Q8Args& a, hipStream_t st) {
  using T = Q8Tile<BITS, G, XG, WM, WN, MT, NT>;
  const uint32_t nrb = (a.n + T::BM - 1) / T::BM, units = nrb * ((a.O + T::BN - 1) / T::BN);
  constexpr uint32_t lds = sizeof(typename T::Lds);
  auto fn = k_q8_tile<BITS, G, XG, WM, WN, MT, NT>;
  if (lds > 64 * 1024) {
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(fn), lds, raised);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3((units + 7) / 8 * 8), dim3(256), lds, st, a, nrb, units);
  return hipGetLastError();
}

template <int BITS, int G, bool XG>
static hipError_t q8_go(const Q8Args& a, hipStream_t st) {
  if (a.n > 64) return q8_tile<BITS, G, XG, 2, 2, 4, 4>(a, st);
  constexpr int NT = 4;
  const dim3 grid((a.O + NT * 16 - 1) / (NT * 16), (a.n + 15) / 16);
  hipLaunchKernelGGL((k_q8<BITS, G, XG, NT>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int BITS, bool XG>
static hipError_t q8_group(const Q8Args& a, uint32_t group, hipStream_t st) {
  return group == 32 ? q8_go<BITS, 32, XG>(a, st) : group == 64 ? q8_go<BITS, 64, XG>(a, st) : q8_go<BITS, 128, XG>(a, st);
}

hipError_t launch_qmm_i8(const Q8Args& a, uint32_t bits, uint32_t group, bool x_grouped, hipStream_t st) {
  if (bits == 8) return x_grouped ? q8_group<8, true>(a, group, st) : q8_group<8, false>(a, group, st);
  if (bits == 4) return x_grouped ? q8_group<4, true>(a, group, st) : q8_group<4, false>(a, group, st);
  return x_grouped ? q8_group<3, true>(a, group, st) : q8_group<3, false>(a, group, st);
}

}  // namespace smoe

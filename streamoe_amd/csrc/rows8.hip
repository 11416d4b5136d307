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
// Host side.
// ---------------------------------------------------------------------------
template <int BITS, int G, bool XG>
static hipError_t q8_go(const Q8Args& a, hipStream_t st) {
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

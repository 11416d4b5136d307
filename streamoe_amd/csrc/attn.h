// attn.h — attention of new tokens over a paged cache (one unit per cache type
// includes this; attn_join.hip has the second launch).
//
//   s_p = scale q . k_p,  m = max s,  out = sum e^(s_p - m) v_p / sum e^(s_p - m)
//
// One pass over the positions: the running maximum m, the sum l and the
// unscaled output of every column (a token's head) stay in registers; a larger
// maximum scales l and the output by e^(old - new).
//
// Work is a list of units of 128 positions: for every group of up to 16 columns
// (tokens of one sequence next to each other times the query heads of one key
// head) the units its positions touch, group after group. Block b takes the
// units [b per, (b + 1) per), so batches of any lengths are split evenly and one
// long row over the whole chip; a group cut between blocks leaves each one's m,
// l and output in the workspace, which k_attn_join adds up. Nothing is decided
// on the host, whose knowledge of lengths would need a wait.
//
// A wave has 32 positions of a unit. S^T = K Q^T: A the keys (a row per lane of
// 16, 8 dims per lane sixteen), B the queries out of LDS; the result has a
// column per lane of 16 and positions 4 g + r of both halves in lane sixteen g.
// O^T = V^T P^T takes P as it lies there: contraction slot j of lane sixteen g is
// position 16 (j / 4) + 4 g + j % 4, and V is loaded in that order, whole rows
// by 16 lanes, and turned in registers (one byte permute per two values). So
// nothing passes between lanes but the maximum.
#pragma once

#include <type_traits>

#include "kv.h"

namespace smoe {

typedef __bf16 abf16x8 __attribute__((ext_vector_type(8)));
typedef float af32x8 __attribute__((ext_vector_type(8), aligned(16)));

constexpr uint32_t kAttnUnit = 128;     // positions of a unit: 32 of each wave
constexpr float kAttnNone = -3.0e38f;   // maximum of no scores

// Positions that token (seq, pos) sees.
__device__ __forceinline__ void attn_range(const AttnArgs& a, int32_t seq, int32_t pos, int32_t* lo, int32_t* hi) {
  bool wrong;
  const bool in = kv_token(a.t, seq, pos, &wrong);
  *hi = in ? pos : -1;
  *lo = in && a.window && (uint32_t)pos >= a.window ? pos - (int32_t)a.window + 1 : 0;
}

// The tokens that share a tile with token r: up to `together` of one sequence at
// positions that follow one another, from a multiple of it on. A block keeps the
// call's first tokens in LDS: what it asks again and again of them is a chain of
// loads otherwise.
struct AttnGroup {
  uint32_t n;        // tokens; 0: r is not the first of its group
  int32_t lo, hi;    // positions that one of them sees; hi < lo: none
  uint32_t units;
};
constexpr uint32_t kAttnHeld = 1024;
struct AttnTokens {
  const AttnArgs& a;
  const int32_t *held_seq, *held_pos;
  __device__ int32_t seq(uint32_t r) const { return r < kAttnHeld ? held_seq[r] : a.t.seq[r]; }
  __device__ int32_t pos(uint32_t r) const { return r < kAttnHeld ? held_pos[r] : a.t.pos[r]; }
  __device__ bool follows(uint32_t r) const {
    return r % a.together && seq(r) == seq(r - 1) && (uint32_t)pos(r) == (uint32_t)pos(r - 1) + 1u;
  }
  __device__ AttnGroup group(uint32_t r) const {
    AttnGroup g = {0, 0, -1, 0};
    if (follows(r)) return g;
    const int32_t s = seq(r);
    uint32_t lo = ~0u;
    do {
      int32_t l, h;
      attn_range(a, s, pos(r + g.n), &l, &h);
      if (h >= 0) lo = min(lo, (uint32_t)l), g.hi = max(g.hi, h);
      ++g.n;
    } while (r + g.n < a.t.n && follows(r + g.n));
    if (g.hi >= 0) {
      g.lo = (int32_t)lo;
      g.units = (uint32_t)g.hi / kAttnUnit - lo / kAttnUnit + 1;
    }
    return g;
  }
};

// Waves per SIMD that the kernel's registers leave room for, so blocks per CU:
// keys, values and outputs of dims up to 256 alone take 192 of a wave's.
constexpr uint32_t attn_blocks_per_cu(uint32_t d) { return d == 256 ? 1 : 2; }
constexpr uint32_t kAttnCus = 256;

template <int D, bool I8>
constexpr int attn_dim(int c, int j) {  // dim of output j of lane c of 16
  return I8 || D < 128 ? c * (D / 16) + j : (j / 8) * 128 + c * 8 + j % 8;
}

__device__ __forceinline__ f32x4 attn_mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(abf16x8, a), __builtin_bit_cast(abf16x8, b), c, 0, 0, 0);
}
// The upper halves of two words, of floats that are bf16 values: both of them.
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
// Eight floats as the sum of three bf16 vectors, each the rest's upper half.
__device__ __forceinline__ void attn_split(const float (&x)[8], u32x4 (&p)[3]) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x[j];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#pragma unroll
    for (int w = 0; w < 4; ++w) p[i][w] = upper_halves(__float_as_uint(v[2 * w]), __float_as_uint(v[2 * w + 1]));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] -= __uint_as_float(__float_as_uint(v[j]) & 0xFFFF0000u);
  }
}
__device__ __forceinline__ float code_f(uint32_t word, int byte) { return (float)(int8_t)(word >> (8 * byte)); }

// Largest (sum) over the four lanes of a column.
__device__ __forceinline__ float column_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float v) { return swap32_add(swap16_add(v, v), swap16_add(v, v)); }

typedef const __attribute__((address_space(4))) int32_t* const_ints;

// Units of a block.
__device__ __forceinline__ uint64_t attn_per(uint64_t units, uint32_t blocks_log) {
  return (units + (1u << blocks_log) - 1) >> blocks_log;
}

// D: head_dim up to it (FULL: equal). QP: parts of a query value (1: bf16 rows,
// 3: f32).
template <int D, bool I8, bool FULL, int QP>
__global__ __launch_bounds__(256, attn_blocks_per_cu(D)) void k_attn(AttnArgs a) {
  constexpr int KS = D / 32;                    // key steps of 32 dims
  constexpr int VJ = D / 16;                    // dims per lane of a value row
  constexpr int KW = I8 ? 2 : 4, VW = I8 ? VJ / 4 : VJ / 2;  // words of a lane: a key step, a value row
  constexpr int kSwap = 2 * VJ * 64 * 16, kQ = QP * KS * 64 * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kSwap > kQ ? kSwap : kQ];
  __shared__ float ml[4][16][2];
  __shared__ uint64_t sums[4];
  __shared__ uint32_t start_row;
  __shared__ uint64_t start_units;
  __shared__ int32_t held_seq[kAttnHeld], held_pos[kAttnHeld];
  const uint32_t t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t n = a.t.n, tiles = a.c.heads * a.parts, hd = a.c.dim;

  for (uint32_t r = t; r < min(n, kAttnHeld); r += 256) held_seq[r] = a.t.seq[r], held_pos[r] = a.t.pos[r];
  __syncthreads();
  const AttnTokens tokens = {a, held_seq, held_pos};

  // Units before every token, and where this block's begin.
  const uint32_t each = (n + 255) / 256, r0 = t * each;
  uint64_t own = 0;
  for (uint32_t r = r0; r < min(n, r0 + each); ++r) own += tokens.group(r).units;
  uint64_t upto = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t v = __shfl_up((unsigned long long)upto, o, kWave);
    if (lane >= (uint32_t)o) upto += v;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint64_t all = 0, skip = 0;
#pragma unroll
  for (uint32_t w = 0; w < 4; ++w) {
    if (w < wave) skip += sums[w];
    all += sums[w];
  }
  const uint64_t mine = skip + upto - own;
  if (blockIdx.x == 0) {
    uint64_t u = mine;
    for (uint32_t r = r0; r < min(n, r0 + each); ++r) {
      a.before[r] = u;
      u += tokens.group(r).units;
      bool wrong;
      kv_token(a.t, tokens.seq(r), tokens.pos(r), &wrong);
      if (wrong) *a.err = 2u;
    }
    if (t == 0) a.before[n] = all;
  }
  all *= tiles;
  const uint64_t per = attn_per(all, a.blocks_log);
  uint64_t x = blockIdx.x * per;
  const uint64_t end = min(all, x + per);
  if (x >= end) return;
  if (mine * tiles <= x && x < (mine + own) * tiles) {
    uint64_t u = mine;
    for (uint32_t r = r0;; ++r) {
      const uint64_t more = tokens.group(r).units;
      if (x < (u + more) * tiles) {
        start_row = r;
        start_units = u;
        break;
      }
      u += more;
    }
  }
  __syncthreads();

  uint32_t row = __builtin_amdgcn_readfirstlane(start_row);
  uint64_t base = start_units * tiles;
  const uint64_t block_x = x;
  while (x < end) {
    const AttnGroup grp = tokens.group(row);
    const uint32_t units = __builtin_amdgcn_readfirstlane(grp.units);
    if (x >= base + (uint64_t)units * tiles) {  // another group's token, or padding
      base += (uint64_t)units * tiles;
      ++row;
      continue;
    }
    const uint32_t together = __builtin_amdgcn_readfirstlane(grp.n);
    const int32_t lo = __builtin_amdgcn_readfirstlane(grp.lo), hi = __builtin_amdgcn_readfirstlane(grp.hi);
    const int32_t seq = __builtin_amdgcn_readfirstlane(tokens.seq(row));
    const uint32_t tile = (uint32_t)(x - base) / units, first = (uint32_t)(x - base) - tile * units;
    const uint32_t count = (uint32_t)min((uint64_t)(units - first), end - x);
    const uint32_t kvh = tile / a.parts, part = tile - kvh * a.parts;
    const uint32_t head0 = kvh * a.group + part * 16, heads = min(16u, a.group - part * 16);
    const uint32_t cols = together * heads;

    // This lane's column: its token and what it sees.
    const uint32_t my_token = min(col / heads, together - 1);
    int32_t see_lo, see_hi;
    attn_range(a, seq, tokens.pos(row + my_token), &see_lo, &see_hi);
    // What all see.
    int32_t all_lo = 0, all_hi = 0x7FFFFFFF;
    for (uint32_t i = 0; i < together; ++i) {
      int32_t l, h;
      attn_range(a, seq, __builtin_amdgcn_readfirstlane(tokens.pos(row + i)), &l, &h);
      all_lo = max(all_lo, l);
      all_hi = min(all_hi, h);
    }

    // The queries as operands: part, step, lane.
    for (uint32_t i = t; i < (uint32_t)KS * 64; i += 256) {
      const uint32_t c = i & 15, lg = (i >> 4) & 3, step = i >> 6;
      const uint32_t d = I8 ? (step >> 1) * 64 + lg * 16 + (step & 1) * 8 : step * 32 + lg * 8;
      const uint32_t token = c / heads;
      u32x4* const to = reinterpret_cast<u32x4*>(lds) + i;
      const bool in = c < cols && d < hd;
      const uint64_t at = in ? (row + token) * a.q_stride + (head0 + c - token * heads) * hd + d : 0;
      if constexpr (QP == 1) {
        const u32x4 v = *reinterpret_cast<const u32x4*>((const uint16_t*)a.q + at);
        to[0] = in ? v : u32x4{0, 0, 0, 0};
      } else {
        const af32x8 v = *reinterpret_cast<const af32x8*>((const float*)a.q + at);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = in ? v[j] : 0.f;
        u32x4 p[3];
        attn_split(f, p);
#pragma unroll
        for (int j = 0; j < 3; ++j) to[j * KS * 64] = p[j];
      }
    }
    __syncthreads();

    f32x4 acc[VJ];
#pragma unroll
    for (int j = 0; j < VJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
    float m = kAttnNone, l = 0.f;

    // This wave's tiles: the units' 32 positions that overlap [lo, hi].
    const uint32_t unit0 = (uint32_t)lo / kAttnUnit + first;
    uint32_t p0 = unit0 * kAttnUnit + wave * 32;  // first position of a tile
    uint32_t left = count;
    if ((int32_t)p0 + 31 < lo) p0 += kAttnUnit, --left;
    if (left && (int32_t)(p0 + (left - 1) * kAttnUnit) > hi) --left;

    const const_ints table = (const_ints)a.t.table + (uint64_t)seq * a.t.width;
    const uint32_t slot_stride = (uint32_t)a.c.slot;
    const uint32_t k_off = col * slot_stride + g * 16;
    const uint32_t v_off = g * 4 * slot_stride;
    // Dims past head_dim are read as the row's first; their queries are zero,
    // their outputs are not written.
    auto k_dim = [&](int s) -> uint32_t {  // bytes from the lane's offset to step s (I8: two steps)
      const uint32_t at = s * 64;
      return FULL || at + g * 16 < hd * (I8 ? 1 : 2) ? at : 0u - g * 16;
    };
    auto v_dim = [&](int half) -> uint32_t {
      const uint32_t at = half * 256 + col * (VW < 4 ? VW * 4 : 16);
      return FULL || at < hd * (I8 ? 1 : 2) ? at : 0u;
    };
    struct Page {
      uint64_t at;     // bytes from the cache's start to the half tile's first row
      uint64_t scale;  // index of its first scale
      bool ok;
    };
    auto page = [&](uint32_t pos) {
      Page p;
      const uint32_t i = kv_page_of(a.c, pos >> 4);
      // The second half of the last tile may lie past the table.
      const int32_t id = pos < a.t.positions ? table[i] : -1;
      const uint32_t slot = pos - i * a.c.page_size;
      p.ok = (uint32_t)id < a.c.n_pages;
      const uint32_t use = p.ok ? (uint32_t)id : 0u;
      p.at = use * a.c.page + kvh * a.c.head + (p.ok ? slot : 0u) * a.c.slot;
      p.scale = ((uint64_t)use * a.c.heads + kvh) * a.c.page_size + (p.ok ? slot : 0u);
      return p;
    };

    uint32_t kr[2][KS][KW];
    uint32_t vr[8][VW];
    f32x4 ks[2], vs[2];
    auto load_k = [&](const Page (&pg)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const gbytes p = as_global(a.c.k + pg[u].at);
#pragma unroll
        for (int s = 0; s < KS / (I8 ? 2 : 1); ++s) {
          const u32x4 w = gld<false, u32x4>(p + (k_off + k_dim(s)));
          if constexpr (I8) {
            kr[u][2 * s][0] = w.x, kr[u][2 * s][1] = w.y, kr[u][2 * s + 1][0] = w.z, kr[u][2 * s + 1][1] = w.w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) kr[u][s][i] = w[i];
          }
        }
        if constexpr (I8) ks[u] = *reinterpret_cast<const f32x4*>(a.c.ks + pg[u].scale + g * 4);
      }
    };
    auto load_v = [&](const Page (&pg)[2]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const gbytes p = as_global(a.c.v + pg[j >> 2].at + (uint64_t)(j & 3) * slot_stride);
        if constexpr (VW >= 4) {
#pragma unroll
          for (int h = 0; h < VW / 4; ++h) {
            const u32x4 w = gld<false, u32x4>(p + (v_off + v_dim(h)));
#pragma unroll
            for (int i = 0; i < 4; ++i) vr[j][4 * h + i] = w[i];
          }
        } else if constexpr (VW == 2) {
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 w = gld<false, u32x2>(p + (v_off + v_dim(0)));
          vr[j][0] = w.x, vr[j][1] = w.y;
        } else {
          vr[j][0] = gld<false, uint32_t>(p + (v_off + v_dim(0)));
        }
      }
      if constexpr (I8) {
#pragma unroll
        for (int u = 0; u < 2; ++u) vs[u] = *reinterpret_cast<const f32x4*>(a.c.vs + pg[u].scale + g * 4);
      }
    };
    // O^T += V^T P^T; SOME: of this lane's column only where it is `mine`, and with
    // values whose mask is 0 as zeros.
    auto add_pv = [&](const u32x4 (&p)[3], const uint32_t (&mask)[4], bool mine, auto some) {
      constexpr bool SOME = decltype(some)::value;
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        u32x4 f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (I8) {
            f[w] = upper_halves(__float_as_uint(code_f(vr[2 * w][j / 4], j % 4)),
                                __float_as_uint(code_f(vr[2 * w + 1][j / 4], j % 4)));
          } else {
            f[w] = __builtin_amdgcn_perm(vr[2 * w + 1][j / 2], vr[2 * w][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
          }
          if constexpr (SOME) f[w] &= mask[w];
        }
        f32x4 sum = acc[j];
#pragma unroll
        for (int i = 0; i < 3; ++i) sum = attn_mfma(f, p[i], sum);
        if constexpr (SOME) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][r] = mine ? sum[r] : acc[j][r];
        } else {
          acc[j] = sum;
        }
      }
    };

    if (left) {
      Page now[2] = {page(p0), page(p0 + 16)};
      load_k(now);
      load_v(now);
      for (; left; --left, p0 += kAttnUnit) {
        Page next[2] = {now[0], now[1]};
        if (left > 1) next[0] = page(p0 + kAttnUnit), next[1] = page(p0 + kAttnUnit + 16);
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < KS; ++st) {
          u32x4 q[QP];
#pragma unroll
          for (int i = 0; i < QP; ++i) q[i] = reinterpret_cast<const u32x4*>(lds)[(i * KS + st) * 64 + lane];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            u32x4 k;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (I8)
                k[w] = upper_halves(__float_as_uint(code_f(kr[u][st][w / 2], 2 * (w % 2))),
                                    __float_as_uint(code_f(kr[u][st][w / 2], 2 * (w % 2) + 1)));
              else
                k[w] = kr[u][st][w];
            }
#pragma unroll
            for (int i = 0; i < QP; ++i) s[u] = attn_mfma(k, q[i], s[u]);
          }
        }
        float y[8];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[4 * u + r] = s[u][r] * a.scale * (I8 ? ks[u][r] : 1.f);
        load_k(next);
        const bool whole = (int32_t)p0 >= all_lo && (int32_t)p0 + 31 <= all_hi && now[0].ok && now[1].ok;
        if (!whole) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int32_t pos = (int32_t)(p0 + (j >> 2) * 16 + g * 4 + (j & 3));
            y[j] = pos >= see_lo && pos <= see_hi && now[j >> 2].ok ? y[j] : -INFINITY;
          }
          if (!(now[0].ok && now[1].ok) && lane == 0) {
            const bool bad = (!now[0].ok && (int32_t)p0 + 15 >= lo && (int32_t)p0 <= hi) ||
                             (!now[1].ok && (int32_t)p0 + 31 >= lo && (int32_t)p0 + 16 <= hi);
            if (bad) *a.err = 2u;
          }
        }
        float top = y[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, y[j]);
        const float bigger = fmaxf(m, column_max(top));
        if (__any(bigger > m)) {
          const float f = __builtin_amdgcn_exp2f(m - bigger);
          l *= f;
#pragma unroll
          for (int j = 0; j < VJ; ++j) acc[j] *= f;
          m = bigger;
        }
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          w[j] = __builtin_amdgcn_exp2f(y[j] - m);
          l += w[j];
          if constexpr (I8) w[j] = whole || y[j] > -INFINITY || y[j] != y[j] ? w[j] * vs[j >> 2][j & 3] : 0.f;
        }
        u32x4 p[3];
        attn_split(w, p);
        uint32_t mask[4] = {0, 0, 0, 0};
        if (whole) {
          add_pv(p, mask, true, std::false_type{});
        } else {
          // A position that only some of the tokens see may hold anything, a NaN
          // too, which no weight of zero keeps out: each token's columns by
          // themselves.
          for (uint32_t i = 0; i < together; ++i) {
            int32_t tl, th;
            attn_range(a, seq, __builtin_amdgcn_readfirstlane(tokens.pos(row + i)), &tl, &th);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              uint32_t both = 0;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = 2 * h + e;
                const int32_t pos = (int32_t)(p0 + (j >> 2) * 16 + g * 4 + (j & 3));
                if (pos >= tl && pos <= th && now[j >> 2].ok) both |= e ? 0xFFFF0000u : 0xFFFFu;
              }
              mask[h] = both;
            }
            add_pv(p, mask, my_token == i, std::true_type{});
          }
        }
        load_v(next);
        now[0] = next[0], now[1] = next[1];
      }
    }

    // The four waves' columns into one.
    l = column_sum(l);
    if (g == 0) ml[wave][col][0] = m, ml[wave][col][1] = l;
    __syncthreads();  // ends the use of the queries, too
    const float m0 = ml[0][col][0], m1 = ml[1][col][0], m2 = ml[2][col][0], m3 = ml[3][col][0];
    const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
    const float total = ml[0][col][1] * __builtin_amdgcn_exp2f(m0 - top) + ml[1][col][1] * __builtin_amdgcn_exp2f(m1 - top) +
                        ml[2][col][1] * __builtin_amdgcn_exp2f(m2 - top) + ml[3][col][1] * __builtin_amdgcn_exp2f(m3 - top);
    const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int j = 0; j < VJ; ++j) acc[j] *= f;
    f32x4* const swap = reinterpret_cast<f32x4*>(lds) + (wave & 1) * VJ * 64 + lane;
    if (wave >= 2) {
#pragma unroll
      for (int j = 0; j < VJ; ++j) swap[j * 64] = acc[j];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
      for (int j = 0; j < VJ; ++j) acc[j] += swap[j * 64];
    }
    __syncthreads();
    if (wave == 1) {
#pragma unroll
      for (int j = 0; j < VJ; ++j) swap[j * 64] = acc[j];
    }
    __syncthreads();
    if (wave == 0) {
      const bool done = first == 0 && count == units;
      const uint64_t slot = 2 * blockIdx.x + (base + (uint64_t)tile * units > block_x ? 1 : 0);
      // A column without weights (nothing seen): zeros.
      const float scale = done ? (total == 0.f ? 0.f : 1.f / total) : 1.f;
#pragma unroll
      for (int j = 0; j < VJ; ++j) acc[j] = (acc[j] + swap[VJ * 64 + j * 64]) * scale;
      if (col < cols) {
        const uint32_t token = col / heads;
        const uint64_t at = done ? (uint64_t)(row + token) * a.heads * hd + (head0 + col - token * heads) * hd
                                 : (slot * 16 + col) * D;
        float* const to = (done ? (float*)a.out : a.acc) + at;
        constexpr int RUN = VJ < 8 ? VJ : 8;  // dims next to each other
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int b = 0; b < VJ; b += RUN) {
            const uint32_t d = attn_dim<D, I8>(g * 4 + r, b);
            if (done && !FULL && d >= hd) continue;
            if (done && a.out_bf16) {
#pragma unroll
              for (int j = 0; j < RUN; j += 4) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                const f32x4 v = {acc[b + j][r], acc[b + j + 1][r], acc[b + j + 2][r], acc[b + j + 3][r]};
                *reinterpret_cast<bf16x4*>((uint16_t*)a.out + at + d + j) = __builtin_convertvector(v, bf16x4);
              }
            } else {
#pragma unroll
              for (int j = 0; j < RUN; j += 4)
                *reinterpret_cast<f32x4*>(to + d + j) = f32x4{acc[b + j][r], acc[b + j + 1][r], acc[b + j + 2][r], acc[b + j + 3][r]};
            }
          }
        if (!done && g == 0) {
          float* const s = a.ml + (slot * 16 + col) * 2;
          s[0] = top;
          s[1] = total;
        }
      }
    }
    x += count;
    if (x == base + (uint64_t)units * tiles) base = x, ++row;
    if (x < end) __syncthreads();
  }
}

template <int D, bool I8>
static hipError_t attn_go(const AttnArgs& a, bool q_bf16, hipStream_t st) {
  const auto fn = a.c.dim == D ? (q_bf16 ? k_attn<D, I8, true, 1> : k_attn<D, I8, true, 3>)
                               : (q_bf16 ? k_attn<D, I8, false, 1> : k_attn<D, I8, false, 3>);
  hipLaunchKernelGGL(fn, dim3(1u << a.blocks_log), dim3(256), 0, st, a);
  return hipGetLastError();
}
template <bool I8>
static hipError_t launch_attn(const AttnArgs& a, bool q_bf16, hipStream_t st) {
  if (a.c.dim <= 64) return attn_go<64, I8>(a, q_bf16, st);
  if (a.c.dim <= 128) return attn_go<128, I8>(a, q_bf16, st);
  return attn_go<256, I8>(a, q_bf16, st);
}

}  // namespace smoe

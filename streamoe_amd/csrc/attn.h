// attn.h — attention of new tokens over a paged cache (one unit per cache type
// includes this; attn_join.hip has the second launch).
//
//   s_p = scale q . k_p,  m = max s,  out = sum e^(s_p - m) v_p / sum e^(s_p - m)
//
// One pass over the positions: the running maximum m, the sum l and the
// unscaled output of every column (a token's head) stay in registers; a larger
// maximum scales l and the output by e^(old - new).
//
// Work is a list of units of 32 positions: for every group of up to 16 columns
// (tokens of one sequence next to each other times the query heads of one key
// head) the units its positions touch, group after group, with kAttnOver more
// in front of each that stand for what a group costs by itself. Block b takes
// an equal part of them, so batches of any lengths are split evenly and
// one long row over the whole chip; a group cut between blocks leaves each one's
// m, l and output in the workspace, which k_attn_join adds up. Nothing is
// decided on the host, whose knowledge of lengths would need a wait.
//
// A block's four waves take its units in turn. S^T = K Q^T: A the keys (a row per
// lane of 16, 8 dims per lane sixteen), B the queries out of LDS; the result has
// a column per lane of 16 and positions 4 g + r of both halves in lane sixteen g.
// O^T = V^T P^T takes P as it lies there: contraction slot j of lane sixteen g is
// position 16 (j / 4) + 4 g + j % 4, and V is loaded in that order, whole rows
// by 16 lanes, and turned in registers (one byte permute per two values). So
// nothing passes between lanes but the maximum.
//
// Memory bounds long rows: one row of 131001 positions of 2 key heads of 256 in
// bf16, 268 MB, takes 52 us, 5.2 TB/s (a large read 5.8, a copy 5.0), 48 rows of
// 16 heads of 128, 233 MB, 50; the matrix cores are busy 6 and 8 % of that, the
// vector units 14 and 19. 61 rows of up to 9001 positions in 8 bits, 154 MB, take
// 39 us, 3.9 TB/s: twice the positions to a byte (vector units 32 %) and a part
// more per row. Short ones are bound by the chain plan, table, keys, values,
// exchange: 700 positions 9.6 us, a window of 1000 in 8 sequences 15.
#pragma once

#include <type_traits>

#include "kv.h"

#include "attn_plan.h"

namespace smoe {

typedef __bf16 abf16x8 __attribute__((ext_vector_type(8)));
typedef float af32x8 __attribute__((ext_vector_type(8), aligned(16)));

constexpr float kAttnNone = -3.0e38f;   // maximum of no scores

// Waves per SIMD that the kernel's registers leave room for, so blocks per CU:
// keys, values and outputs of dims up to 256 alone take 192 of a wave's in bf16; 128
// in 8 bits, where the kernel as a whole still has 380 to 392. No vector register is
// spilled; 112 to 143 scalars (the plan, spans, arguments) lie in vector lanes.
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

// D: head_dim up to it (FULL: equal). QP: parts of a query value (1: bf16 rows,
// 3: f32).
//
// The next tile's keys are asked for when this one's are used up, its values
// likewise, over the end of a part of a group into the next: their loads are
// always in flight.
template <int D, bool I8, int QP>
constexpr uint32_t attn_lds() {  // two parts' queries; four waves' outputs
  return (2 * QP * (D / 32) + 4 * (D / 16)) * 1024;
}
template <int D, bool I8, bool FULL, int QP>
__global__ __launch_bounds__(256, attn_blocks_per_cu(D)) void k_attn(AttnArgs a) {
  constexpr int KS = D / 32;                    // key steps of 32 dims
  constexpr int VJ = D / 16;                    // dims per lane of a value row
  constexpr int KW = I8 ? 2 : 4, VW = I8 ? VJ / 4 : VJ / 2;  // words of a lane: a key step, a value row
  constexpr int QN = KS < 4 ? 1 : KS / 4;       // pieces of eight query values per thread
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  u32x4* const q_lds = reinterpret_cast<u32x4*>(lds);
  f32x4* const o_lds = reinterpret_cast<f32x4*>(lds + 2 * QP * KS * 1024);
  __shared__ float2 ml[4][16];
  __shared__ attn_u64 chunk_units[kKvMaxTokens / 64];
  const uint32_t t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t hd = a.c.dim, blk = blockIdx.x;

  AttnPlan plan;
  if (!plan.begin(a, chunk_units)) return;

  // What the group's tokens see: one of them, and all.
  struct Span {
    int32_t lo, hi, all_lo, all_hi;
  };
  auto span_of = [&](const AttnPart& p) {
    Span s;
    const int32_t last = p.pos + (int32_t)p.n - 1, top = (int32_t)a.t.positions - 1;
    int32_t unused;
    attn_range(a, true, max(p.pos, 0), &s.lo, &unused);
    s.hi = min(last, top);
    attn_range(a, true, s.hi, &s.all_lo, &unused);
    s.all_hi = p.pos < 0 || last > top ? -1 : p.pos;
    return s;
  };
  // This wave's units of a part, every fourth: where its first begins, how many.
  uint32_t turn = wave;  // units until this wave's next
  auto tiles_of = [&](const AttnPart& p, const Span& s, uint32_t* p0, uint32_t* left) {
    *p0 = ((uint32_t)s.lo / kAttnUnit + p.first + turn) * kAttnUnit;
    *left = p.count > turn ? (p.count - turn + 3) / 4 : 0u;
    turn = (turn - p.count) & 3;
  };

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
  auto page = [&](int32_t seq, uint32_t kvh, uint32_t pos) {
    Page p;
    const uint32_t i = kv_page_of(a.c, pos >> 4);
    // The second half of the last tile may lie past the table.
    const int32_t id = pos < a.t.positions ? ((const_ints)a.t.table)[(uint64_t)seq * a.t.width + i] : -1;
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
  // on: whether there is a tile to load; else all lanes read its first bytes.
  auto load_k = [&](const Page (&pg)[2], bool on) {
    const uint32_t off = on ? k_off : 0u;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const gbytes p = as_global(a.c.k + pg[u].at);
#pragma unroll
      for (int s = 0; s < KS / (I8 ? 2 : 1); ++s) {
        const u32x4 w = gld<false, u32x4>(p + (off + (FULL || on ? k_dim(s) : 0u)));
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
  auto load_v = [&](const Page (&pg)[2], bool on) {
    const uint32_t off = on ? v_off : 0u, step = on ? slot_stride : 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const gbytes p = as_global(a.c.v + pg[j >> 2].at + (uint64_t)(j & 3) * step);
      if constexpr (VW >= 4) {
#pragma unroll
        for (int h = 0; h < VW / 4; ++h) {
          const u32x4 w = gld<false, u32x4>(p + (off + v_dim(h)));
#pragma unroll
          for (int i = 0; i < 4; ++i) vr[j][4 * h + i] = w[i];
        }
      } else if constexpr (VW == 2) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 w = gld<false, u32x2>(p + (off + v_dim(0)));
        vr[j][0] = w.x, vr[j][1] = w.y;
      } else {
        vr[j][0] = gld<false, uint32_t>(p + (off + v_dim(0)));
      }
    }
    if constexpr (I8) {
#pragma unroll
      for (int u = 0; u < 2; ++u) vs[u] = *reinterpret_cast<const f32x4*>(a.c.vs + pg[u].scale + g * 4);
    }
  };
  f32x4 acc[VJ];
  // O^T += V^T P^T; SOME: of this lane's column only where it is `mine`, and with
  // values whose mask is 0 as zeros.
  auto add_pv = [&](const u32x4 (&p)[3], const uint32_t (&mask)[4], bool mine, auto some) {
    constexpr bool SOME = decltype(some)::value;
    // (A zero that the compiler does not know, so that it does not form the
    // operands of all tokens' rounds ahead, in as many registers again.)
    uint32_t zero = 0;
    if constexpr (SOME) asm volatile("" : "+v"(zero));
    auto v = [&](int j, int i) { return SOME ? vr[j][i] ^ zero : vr[j][i]; };
#pragma unroll
    for (int j = 0; j < VJ; ++j) {
      u32x4 f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (I8) {
          f[w] = upper_halves(__float_as_uint(code_f(v(2 * w, j / 4), j % 4)),
                              __float_as_uint(code_f(v(2 * w + 1, j / 4), j % 4)));
        } else {
          f[w] = __builtin_amdgcn_perm(v(2 * w + 1, j / 2), v(2 * w, j / 2), j % 2 ? 0x07060302u : 0x05040100u);
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

  // The queries of a part, as operands: part of the value, step, lane.
  struct Heads {
    uint32_t kvh, first, n, cols;
  };
  auto heads_of = [&](const AttnPart& p) {
    Heads h;
    h.kvh = p.tile / a.parts;
    const uint32_t part = p.tile - h.kvh * a.parts;
    h.first = h.kvh * a.group + part * 16;
    h.n = min(16u, a.group - part * 16);
    h.cols = p.n * h.n;
    return h;
  };
  std::conditional_t<QP == 1, u32x4, af32x8> qv[QN];
  auto load_q = [&](const AttnPart& p, const Heads& h) {
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const uint32_t i = t + j * 256, c = i & 15, lg = (i >> 4) & 3, step = i >> 6;
      const uint32_t d = I8 ? (step >> 1) * 64 + lg * 16 + (step & 1) * 8 : step * 32 + lg * 8;
      const uint32_t token = c / h.n;
      const uint64_t at = c < h.cols && d < hd ? (p.row + token) * a.q_stride + (h.first + c - token * h.n) * hd + d : 0;
      if constexpr (QP == 1)
        qv[j] = *reinterpret_cast<const u32x4*>((const uint16_t*)a.q + at);
      else
        qv[j] = *reinterpret_cast<const af32x8*>((const float*)a.q + at);
    }
  };
  uint32_t q_at = 0;  // this part's queries in LDS: of two places in turn
  auto store_q = [&](const Heads& h, uint32_t to) {
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const uint32_t i = t + j * 256, c = i & 15, lg = (i >> 4) & 3, step = i >> 6;
      const uint32_t d = I8 ? (step >> 1) * 64 + lg * 16 + (step & 1) * 8 : step * 32 + lg * 8;
      const bool in = c < h.cols && d < hd;
      if (i >= (uint32_t)KS * 64) continue;
      if constexpr (QP == 1) {
        q_lds[to + i] = in ? qv[j] : u32x4{0, 0, 0, 0};
      } else {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = in ? qv[j][e] : 0.f;
        u32x4 s[3];
        attn_split(f, s);
#pragma unroll
        for (int e = 0; e < 3; ++e) q_lds[to + e * KS * 64 + i] = s[e];
      }
    }
  };

  AttnPart cur;
  if (!plan.next(a, cur)) return;
  Span see = span_of(cur);
  Heads heads = heads_of(cur);
  uint32_t p0, left;  // this wave's next tile, and how many it has
  tiles_of(cur, see, &p0, &left);
  load_q(cur, heads);
  Page now[2];
  auto load_first = [&] {
    now[0] = page(cur.seq, heads.kvh, p0), now[1] = page(cur.seq, heads.kvh, p0 + 16);
    load_k(now, true);
    load_v(now, true);
  };
  if (left) load_first();
  for (bool begin = true;; begin = false) {
    // The part behind this one.
    AttnPart then = cur;
    const bool more = plan.next(a, then);
    Span then_see = see;
    Heads then_heads = heads;
    uint32_t then_p0 = 0, then_left = 0;
    if (more) {
      then_see = span_of(then);
      then_heads = heads_of(then);
      tiles_of(then, then_see, &then_p0, &then_left);
    }
    if (begin) {  // the first part's queries, its loads still on their way
      store_q(heads, 0);
      __syncthreads();
    }
    load_q(then, then_heads);
    bool loaded = false;  // the part behind's first tile

    // This lane's column: its token and what it sees.
    const uint32_t my_token = min(col / heads.n, cur.n - 1);
    int32_t see_lo, see_hi;
    attn_range(a, true, cur.pos + (int32_t)my_token, &see_lo, &see_hi);
#pragma unroll
    for (int j = 0; j < VJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
    float m = kAttnNone, l = 0.f;

    for (; left; --left, p0 += 4 * kAttnUnit) {
      // The tile to ask for next: this part's, or the first of the one behind it.
      const bool same = left > 1, on = same || then_left;
      Page next[2] = {now[0], now[1]};
      if (on) {
        const int32_t seq = same ? cur.seq : then.seq;
        const uint32_t kvh = same ? heads.kvh : then_heads.kvh, at = same ? p0 + 4 * kAttnUnit : then_p0;
        next[0] = page(seq, kvh, at), next[1] = page(seq, kvh, at + 16);
      }
      f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        u32x4 q[QP];
#pragma unroll
        for (int i = 0; i < QP; ++i) q[i] = q_lds[q_at + (i * KS + st) * 64 + lane];
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
        // Else all of the queries are read at once, into registers that are not there.
        if (st % 2) __builtin_amdgcn_sched_barrier(0);
      }
      float y[8];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) y[4 * u + r] = s[u][r] * a.scale * (I8 ? ks[u][r] : 1.f);
      load_k(next, on);
      const bool whole = (int32_t)p0 >= see.all_lo && (int32_t)p0 + 31 <= see.all_hi && now[0].ok && now[1].ok;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int32_t pos = (int32_t)(p0 + (j >> 2) * 16 + g * 4 + (j & 3));
          y[j] = pos >= see_lo && pos <= see_hi && now[j >> 2].ok ? y[j] : -INFINITY;
        }
        if (!(now[0].ok && now[1].ok) && lane == 0) {
          const bool bad = (!now[0].ok && (int32_t)p0 + 15 >= see.lo && (int32_t)p0 <= see.hi) ||
                           (!now[1].ok && (int32_t)p0 + 31 >= see.lo && (int32_t)p0 + 16 <= see.hi);
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
        for (uint32_t i = 0; i < cur.n; ++i) {
          int32_t tl, th;
          attn_range(a, true, cur.pos + (int32_t)i, &tl, &th);
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
      load_v(next, on);
      now[0] = next[0], now[1] = next[1];
      loaded = on && !same;
    }
    store_q(then_heads, q_at ^ (QP * KS * 64));

    // The four waves' columns into one, a quarter of the dims in each.
    l = column_sum(l);
    if (g == 0) ml[wave][col] = float2{m, l};
#pragma unroll
    for (int j = 0; j < VJ; ++j) o_lds[(wave * VJ + j) * 64 + lane] = acc[j];
    __syncthreads();  // the next queries are there, too
    const float2 s0 = ml[0][col], s1 = ml[1][col], s2 = ml[2][col], s3 = ml[3][col];
    const float top = fmaxf(fmaxf(s0.x, s1.x), fmaxf(s2.x, s3.x));
    float f[4] = {__builtin_amdgcn_exp2f(s0.x - top), __builtin_amdgcn_exp2f(s1.x - top), __builtin_amdgcn_exp2f(s2.x - top),
                  __builtin_amdgcn_exp2f(s3.x - top)};
    const float total = s0.y * f[0] + s1.y * f[1] + s2.y * f[2] + s3.y * f[3];
    const attn_u64 slot = 2 * blk + (cur.begun ? 0 : 1);
    // A column without weights (nothing seen): zeros.
    const float scale = !cur.whole ? 1.f : total == 0.f ? 0.f : 1.f / total;
    constexpr int RUN = VJ / 4;  // dims next to each other
    float o[RUN][4];
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += o_lds[(w * VJ + wave * RUN + j) * 64 + lane] * f[w];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[j][r] = sum[r] * scale;
    }
    if (more) __syncthreads();  // the outputs' place is free
    if (col < heads.cols) {
      const uint32_t token = col / heads.n;
      const uint64_t at = cur.whole ? ((uint64_t)(cur.row + token) * a.heads + heads.first + col - token * heads.n) * hd
                                    : (slot * 16 + col) * D;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t d = attn_dim<D, I8>(g * 4 + r, wave * RUN);
        if (cur.whole && !FULL && d >= hd) continue;
        typedef float run_f __attribute__((ext_vector_type(RUN < 2 ? 2 : RUN)));
        typedef __bf16 run_b __attribute__((ext_vector_type(RUN < 2 ? 2 : RUN)));
        if constexpr (RUN == 1) {
          if (cur.whole && a.out_bf16)
            ((__bf16*)a.out)[at + d] = (__bf16)o[0][r];
          else
            (cur.whole ? (float*)a.out : a.acc)[at + d] = o[0][r];
        } else {
          run_f v;
#pragma unroll
          for (int j = 0; j < RUN; ++j) v[j] = o[j][r];
          if (cur.whole && a.out_bf16)
            *reinterpret_cast<run_b*>((uint16_t*)a.out + at + d) = __builtin_convertvector(v, run_b);
          else
            *reinterpret_cast<run_f*>((cur.whole ? (float*)a.out : a.acc) + at + d) = v;
        }
      }
      if (!cur.whole && wave == 0 && g == 0) *reinterpret_cast<float2*>(a.ml + (slot * 16 + col) * 2) = float2{top, total};
    }
    if (!more) return;
    cur = then, see = then_see, heads = then_heads, p0 = then_p0, left = then_left;
    q_at ^= QP * KS * 64;
    if (left && !loaded) load_first();
  }
}

template <int D, bool I8, bool FULL, int QP>
static hipError_t attn_go(const AttnArgs& a, hipStream_t st) {
  static std::atomic<uint64_t> raised{0};
  constexpr uint32_t bytes = attn_lds<D, I8, QP>();
  const hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(&k_attn<D, I8, FULL, QP>), bytes, raised);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_attn<D, I8, FULL, QP>), dim3(1u << a.blocks_log), dim3(256), bytes, st, a);
  return hipGetLastError();
}
template <int D, bool I8>
static hipError_t attn_of(const AttnArgs& a, bool q_bf16, hipStream_t st) {
  if (a.c.dim == D) return q_bf16 ? attn_go<D, I8, true, 1>(a, st) : attn_go<D, I8, true, 3>(a, st);
  return q_bf16 ? attn_go<D, I8, false, 1>(a, st) : attn_go<D, I8, false, 3>(a, st);
}
template <bool I8>
static hipError_t launch_attn(const AttnArgs& a, bool q_bf16, hipStream_t st) {
  if (a.c.dim <= 64) return attn_of<64, I8>(a, q_bf16, st);
  if (a.c.dim <= 128) return attn_of<128, I8>(a, q_bf16, st);
  return attn_of<256, I8>(a, q_bf16, st);
}

}  // namespace smoe

// beam.hip — one step of a beam search behind the LM head.
//
//   k_beam_slice  a slice of one beam's logits: each wave's largest value and
//                 sum of exponentials, and the n_picks largest logits in order
//   k_beam_pick   one request: log-sum-exp of every beam, and the n_picks
//                 largest of score + logit - log-sum-exp among the slices' own
//   k_beam_copy   dst row i = src row rows[i] of a list of state tensors
//
// A logit becomes 32 bits in an order that integers compare, and a key with the
// complement of its token below it, so keys are unique, equal logits fall in
// token order and sorting needs no tie rules.
#include "common.h"
#include "kernels.h"

#include <type_traits>

namespace smoe {

typedef unsigned long long u64;

constexpr uint32_t kBeamTile = 4096;          // logits per block and round: 16 per thread
constexpr uint32_t kOrdNegInf = 0x007FFFFFu;  // beam_ord(-inf)

// Order of floats as unsigned integers; -0 as +0, NaN as -inf.
__device__ __forceinline__ uint32_t beam_ord(float v) {
  const uint32_t b = __float_as_uint(v == v ? v + 0.f : -INFINITY);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// e^x for x <= 0, from below -87 on 2^-126 (nothing beside a sum of at least
// one): 2^p with p = x log2 e rounded, times 1 + r ln 2 for what the rounding
// left, r = x log2 e - p; off by two ulp and |x| 1.4e-8 (log2 e in 24 bits).
__device__ __forceinline__ float beam_exp(float x) {
  constexpr float kLog2e = 1.44269502f, kLn2 = 0.693147182f;
  x = fmaxf(x, -87.3f);
  const float p = x * kLog2e;
  const float r = __builtin_fmaf(x, kLog2e, -p);
  const float e = __builtin_amdgcn_exp2f(p);
  return __builtin_fmaf(e, r * kLn2, e);
}

// Wave reductions on DPP (row shifts, then row broadcasts: complete in lane
// 63), the result in every lane. A shuffle is an LDS permute, 100 cycles each.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp_u32<0x111, 0xF>(v));
  v = max(v, dpp_u32<0x112, 0xF>(v));
  v = max(v, dpp_u32<0x114, 0xF>(v));
  v = max(v, dpp_u32<0x118, 0xF>(v));
  v = max(v, dpp_u32<0x142, 0xA>(v));
  v = max(v, dpp_u32<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add_f64(double v) {
  const u64 b = (u64)__double_as_longlong(v);
  const u64 o = (u64)dpp_u32<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp_u32<CTRL, ROWS>((uint32_t)b);
  return v + __longlong_as_double((long long)o);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v = dpp_add_f64<0x111, 0xF>(v);
  v = dpp_add_f64<0x112, 0xF>(v);
  v = dpp_add_f64<0x114, 0xF>(v);
  v = dpp_add_f64<0x118, 0xF>(v);
  v = dpp_add_f64<0x142, 0xA>(v);
  v = dpp_add_f64<0x143, 0xC>(v);
  const u64 b = (u64)__double_as_longlong(v);
  const u64 hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63), lo = (uint32_t)__builtin_amdgcn_readlane((int)b, 63);
  return __longlong_as_double((long long)(hi << 32 | lo));
}
__device__ __forceinline__ float wave_max_f32(float v) { return readlane_f(wave_max_last(v), 63); }

__device__ __forceinline__ uint32_t count_below(u64 mask) {  // set bits of the lanes below this one
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Whether a beam still takes part with its own logits.
__device__ __forceinline__ bool beam_open(const BeamArgs& a, uint32_t row) {
  return a.scores[row] > -INFINITY && !(a.done && a.done[row]);
}

// Each wave collects what of its 1024 logits can be among the P largest: with
// T the P-th largest of the largest logits of some groups of lanes, at least P
// logits are >= T. Groups of four or two lanes do where there are twice P of
// them (16 lane reads instead of 64), with little more than P logits >= T as a
// rule. Where those are over 17 P, T is the P-th largest of single lanes: those
// above it lie in fewer than P lanes, and of those equal to it the P of lowest
// tokens suffice. The block's list is ranked by counting.
__global__ __launch_bounds__(256) void k_beam_slice(BeamArgs a) {
  extern __shared__ __attribute__((aligned(16))) u64 list[];  // [68 P], then twice [P] of the tiles before
  __shared__ uint32_t count;
  const uint32_t t = threadIdx.x, lane = t & 63, P = a.picks;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  u64* const top = list + 4 * 17 * P;
  const uint64_t first = (uint64_t)row * a.vocab, total = (uint64_t)a.rows * a.vocab;
  const uint32_t shift = (uint32_t)(first & 3);  // tiles start on 16 bytes, up to three logits ahead of the row
  float m = -INFINITY;
  double sum = 0.0;
  if (t < P) top[t] = 0;
  const uint32_t tile0 = slice * a.tiles;
  for (uint32_t tile = tile0; tile < tile0 + a.tiles; ++tile) {
    const int64_t tok0 = (int64_t)tile * kBeamTile - shift;
    if (tok0 >= (int64_t)a.vocab) break;
    // Value 4 j + c is token tok + 1024 j + c. A NaN counts as -inf, and so do
    // places outside the row, which must not be taken.
    const int64_t tok = tok0 + t * 4;
    const bool whole = tok0 >= 0 && tok0 + kBeamTile <= (int64_t)a.vocab;
    float v[16];
    if (whole) {
      const float* const p = a.logits + first + tok;
      f32x4 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const f32x4*>(p + 1024 * j);
      if (tile == tile0 && !beam_open(a, row)) return;  // under the loads
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = fmaxf(q[i / 4][i % 4], -INFINITY);
    } else {
      if (tile == tile0 && !beam_open(a, row)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t k = tok + 1024 * j, e = (int64_t)first + k;
        f32x4 q = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (k < (int64_t)a.vocab) {
          if (e + 4 <= (int64_t)total) {
            q = *reinterpret_cast<const f32x4*>(a.logits + e);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (e + c < (int64_t)total) q[c] = a.logits[e + c];
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) v[4 * j + c] = k + c >= 0 && k + c < (int64_t)a.vocab ? fmaxf(q[c], -INFINITY) : -INFINITY;
      }
    }
    float tm = v[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) tm = fmaxf(tm, v[i]);
    // Sum of exponentials below the thread's running maximum.
    const float nm = fmaxf(m, tm);
    if (nm > -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += beam_exp(v[i] - nm);
      sum = sum * (double)(m > -INFINITY ? beam_exp(m - nm) : 0.f) + (double)s;
      m = nm;
    }
    // The P-th largest of the groups' largest: the smallest of those that fewer
    // than P are above.
    auto threshold = [&](float g, auto lanes) {
      uint32_t higher = 0;
#pragma unroll
      for (int l = 0; l < 64; l += decltype(lanes)::value) higher += readlane_f(g, l) > g ? 1u : 0u;
      return -wave_max_f32(higher < P ? -g : -INFINITY);
    };
    const float two = fmaxf(tm, dpp_f<0xB1>(tm, tm)), four = fmaxf(two, dpp_f<0x4E>(two, two));
    // What is not above the P-th largest of the tiles before has no place.
    const float floor = tile == tile0 ? -INFINITY : beam_value((uint32_t)(top[P - 1] >> 32));
    float least = fmaxf(floor, P <= 8    ? threshold(four, std::integral_constant<int, 4>{})
                               : P <= 16 ? threshold(two, std::integral_constant<int, 2>{})
                                         : threshold(tm, std::integral_constant<int, 1>{}));
    auto key = [&](int i) { return (u64)beam_ord(v[i]) << 32 | (uint32_t)~(uint32_t)(tok + 1024 * (i / 4) + i % 4); };
    u64* const out = top + P;  // beside the tops, which are still read
    if (t == 0) count = 0;
    if (t < P) out[t] = 0;
    __syncthreads();
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) mine += v[i] >= least ? 1u : 0u;
    uint32_t upto = mine;
    upto += dpp_u32<0x111, 0xF>(upto);
    upto += dpp_u32<0x112, 0xF>(upto);
    upto += dpp_u32<0x114, 0xF>(upto);
    upto += dpp_u32<0x118, 0xF>(upto);
    upto += dpp_u32<0x142, 0xA>(upto);
    upto += dpp_u32<0x143, 0xC>(upto);
    const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    // Few enough, and none of them a place outside the row.
    if (n <= 17 * P && (whole || least > -INFINITY)) {
      uint32_t base = 0;
      if (lane == 0) base = atomicAdd(&count, n);
      uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)base) + upto - mine;
      if (mine) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (v[i] >= least) list[at++] = key(i);
      }
    } else {
      // Those above the single lanes' threshold, then the first P of the equal
      // ones.
      least = fmaxf(floor, threshold(tm, std::integral_constant<int, 1>{}));
      uint32_t above = 0, met = 0;
      u64 mask[16];
      bool same[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t k = tok + 1024 * (i / 4) + i % 4;
        above += (uint32_t)__popcll(__ballot(v[i] > least));
        same[i] = v[i] == least && k >= 0 && k < (int64_t)a.vocab;
        mask[i] = __ballot(same[i]);
        met += (uint32_t)__popcll(mask[i]);
      }
      met = min(met, P);
      uint32_t base = 0;
      if (lane == 0) base = atomicAdd(&count, above + met);
      base = (uint32_t)__builtin_amdgcn_readfirstlane((int)base);
      uint32_t seen = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // tokens ascend over j, then the lanes, then c
        uint32_t at = seen;
#pragma unroll
        for (int c = 0; c < 4; ++c) at += count_below(mask[4 * j + c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (same[4 * j + c]) {
            if (at < P) list[base + at] = key(4 * j + c);
            ++at;
          }
          seen += (uint32_t)__popcll(mask[4 * j + c]);
        }
      }
      base += met;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const u64 m1 = __ballot(v[i] > least);
        if (v[i] > least) list[base + count_below(m1)] = key(i);
        base += (uint32_t)__popcll(m1);
      }
    }
    __syncthreads();
    const uint32_t all = count, before = tile > tile0 ? P : 0u;
    for (uint32_t e = t; e < all + before; e += 256) {
      const u64 k = e < all ? list[e] : top[e - all];
      if (!k) continue;
      uint32_t r = 0, i = 0;
      for (; i + 4 <= all; i += 4) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list + i), y = *reinterpret_cast<const ulonglong2*>(list + i + 2);
        r += (x.x > k ? 1u : 0u) + (x.y > k ? 1u : 0u) + (y.x > k ? 1u : 0u) + (y.y > k ? 1u : 0u);
      }
      for (; i < all; ++i) r += list[i] > k ? 1u : 0u;
      for (i = 0; i < before; ++i) r += top[i] > k ? 1u : 0u;
      if (r < P) out[r] = k;
    }
    __syncthreads();
    if (t < P) top[t] = out[t];
    if (a.tiles > 1) __syncthreads();
  }
  const float wm = wave_max_f32(m);
  const double ws = wave_sum_f64(m > -INFINITY ? sum * (double)beam_exp(m - wm) : 0.0);
  if (lane == 0) a.stats[(uint64_t)blockIdx.x * 4 + wave] = BeamStat{ws, wm, 0u};
  if (t < P) a.cand[(uint64_t)blockIdx.x * P + t] = top[t];
}

struct BeamKey {
  u64 hi, lo;  // value; beam, logit, token
};
__device__ __forceinline__ bool above(const BeamKey& x, const BeamKey& y) {
  return x.hi > y.hi || (x.hi == y.hi && x.lo > y.lo);
}
__device__ __forceinline__ BeamKey beam_key(double v, uint32_t beam, uint32_t ord, uint32_t token) {
  v = v == v ? v + 0.0 : -INFINITY;
  const u64 b = (u64)__double_as_longlong(v);
  return {b >> 63 ? ~b : b | 1ull << 63,
          (u64)(kBeamMaxBeams - 1 - beam) << 60 | (u64)ord << 28 | (kBeamMaxVocab - 1 - token)};
}

// A wave per beam: lane s holds the head of slice s's list (at most 64 slices);
// the largest head, of equal ones the lowest lane's (slices are in token
// order), is taken P times. The beams' P each are ranked by counting.
__global__ __launch_bounds__(256) void k_beam_pick(BeamArgs a) {
  extern __shared__ __attribute__((aligned(16))) BeamKey best[];  // [beams * P], then [4][P][64] u64
  const uint32_t t = threadIdx.x, lane = t & 63, P = a.picks, W = a.beams, S = a.slices;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6), row0 = blockIdx.x * W;
  u64* const held = reinterpret_cast<u64*>(best + W * P) + wave * P * 64;
  for (uint32_t b = wave; b < W; b += 4) {
    const uint32_t row = row0 + b;
    // Loads together; of a beam that is not open they may hold anything.
    BeamStat s[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      s[i] = BeamStat{0.0, -INFINITY, 0u};
      if (i * 64 + lane < 4 * S) s[i] = a.stats[(uint64_t)row * S * 4 + i * 64 + lane];
    }
    if (lane < S) {
      const u64* const from = a.cand + ((uint64_t)row * S + lane) * P;
      for (uint32_t j = 0; j < P; ++j) held[j * 64 + lane] = from[j];
    }
    const float sc = a.scores[row];
    BeamKey* const to = best + b * P;
    bool open = beam_open(a, row);
    double lse = 0.0;
    if (open) {
      const float m = wave_max_f32(fmaxf(fmaxf(s[0].max, s[1].max), fmaxf(s[2].max, s[3].max)));
      double sum = 0.0;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sum += s[i].max > -INFINITY ? s[i].sum * (double)beam_exp(s[i].max - m) : 0.0;
      sum = wave_sum_f64(sum);
      // All logits masked, or an infinity among them: no token has a value.
      open = m > -INFINITY && m < INFINITY;
      if (open) lse = (double)m + log(sum);
    }
    if (open) {
      u64 head = lane < S ? held[lane] : 0;
      uint32_t at = 0;
      for (uint32_t j = 0; j < P; ++j) {
        const uint32_t o = (uint32_t)(head >> 32), mo = wave_max_u32(o);
        if (!mo) {  // no more tokens than picks
          if (lane == 0) to[j] = BeamKey{0, 0};
          continue;
        }
        const uint32_t from = (uint32_t)__ffsll((long long)__ballot(o == mo)) - 1;
        if (lane == from) {
          to[j] = beam_key((double)sc + ((double)beam_value(o) - lse), b, o, ~(uint32_t)head);
          ++at;
          head = at < P ? held[at * 64 + lane] : 0;
        }
      }
    } else if (lane < P) {
      // Ended: the pad token keeps the score, then the others in order; nothing
      // left: the first tokens.
      const bool ended = a.done && a.done[row] && sc > -INFINITY;
      const uint32_t tok = !ended ? lane : lane == 0 ? a.pad : lane - 1 < a.pad ? lane - 1 : lane;
      to[lane] = tok < a.vocab ? beam_key(ended && lane == 0 ? (double)sc : -INFINITY, b, kOrdNegInf, tok) : BeamKey{0, 0};
    }
  }
  __syncthreads();
  const uint32_t n = W * P;
  for (uint32_t c = t; c < n; c += 256) {
    const BeamKey k = best[c];
    if (!k.hi) continue;
    uint32_t r = 0;
    for (uint32_t i = 0; i < n; ++i) r += above(best[i], k) ? 1u : 0u;
    if (r >= P) continue;
    const uint64_t o = (uint64_t)blockIdx.x * P + r;
    const double v = __longlong_as_double((long long)(k.hi >> 63 ? k.hi & ~(1ull << 63) : ~k.hi));
    a.out_scores[o] = (float)v;
    a.out_rows[o] = (int32_t)(row0 + kBeamMaxBeams - 1 - (uint32_t)(k.lo >> 60));
    a.out_tokens[o] = (int32_t)(kBeamMaxVocab - 1 - (uint32_t)(k.lo & (kBeamMaxVocab - 1)));
  }
}

// ---------------------------------------------------------------------------
// Reordering.
// ---------------------------------------------------------------------------
constexpr uint32_t kCopyChunk = 16384;  // bytes per block
constexpr uint32_t kCopyStates = 32;    // states per launch (by value: 2.5 KB of arguments)

struct CopyArgs {
  BeamCopy s[kCopyStates];
  uint64_t end[kCopyStates];  // blocks of the states up to and with this one
  uint32_t n;
  const int32_t* rows;
  uint32_t n_rows, src_rows;
  uint32_t* err;
};

template <typename T>
__device__ __forceinline__ void copy_units(const uint8_t* src, uint8_t* dst, uint32_t bytes) {
  const uint32_t n = bytes / sizeof(T);
  for (uint32_t i = threadIdx.x; i < n; i += 256)
    reinterpret_cast<T*>(dst)[i] = reinterpret_cast<const T*>(src)[i];
  for (uint32_t i = n * sizeof(T) + threadIdx.x; i < bytes; i += 256) dst[i] = src[i];
}

__global__ __launch_bounds__(256) void k_beam_copy(CopyArgs a) {
  uint64_t u = blockIdx.x;
  uint32_t k = 0;
  while (k + 1 < a.n && u >= a.end[k]) ++k;
  if (k) u -= a.end[k - 1];
  const BeamCopy& s = a.s[k];
  const uint64_t chunks = (s.bytes + kCopyChunk - 1) / kCopyChunk;
  const uint64_t c = u % chunks, pr = u / chunks;
  const uint64_t piece = pr % s.pieces, row = pr / s.pieces;
  const int32_t from = a.rows[row];
  if (from < 0 || (uint32_t)from >= a.src_rows) {
    if (threadIdx.x == 0) *a.err = 2u;
    return;
  }
  const uint64_t at = c * kCopyChunk;
  const uint32_t bytes = (uint32_t)(s.bytes - at < kCopyChunk ? s.bytes - at : kCopyChunk);
  const uint8_t* src = s.src + (uint64_t)from * s.src_row + piece * s.src_piece + at;
  uint8_t* dst = s.dst + row * s.dst_row + piece * s.dst_piece + at;
  if (s.unit == 16)
    copy_units<u32x4>(src, dst, bytes);
  else if (s.unit == 4)
    copy_units<uint32_t>(src, dst, bytes);
  else
    copy_units<uint8_t>(src, dst, bytes);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
static uint64_t al256(uint64_t n) { return (n + 255) & ~255ull; }

uint64_t beam_workspace(uint32_t requests, uint32_t beams, uint32_t vocab, uint32_t picks, BeamArgs* a, uint8_t* base) {
  // Tiles of a row start up to three logits ahead of it.
  const uint32_t tiles = (vocab + 3 + kBeamTile - 1) / kBeamTile;
  const uint32_t per = (tiles + kBeamMaxSlices - 1) / kBeamMaxSlices, slices = (tiles + per - 1) / per;
  const uint64_t lists = (uint64_t)requests * beams * slices;
  const uint64_t sb = al256(lists * 4 * sizeof(BeamStat));
  if (a) {
    a->slices = slices;
    a->tiles = per;
    a->stats = reinterpret_cast<BeamStat*>(base);
    a->cand = reinterpret_cast<unsigned long long*>(base + sb);
  }
  return sb + al256(lists * picks * 8);
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(k_beam_slice, dim3(a.rows * a.slices), dim3(256), (4 * 17 + 2) * a.picks * 8, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t lds = a.beams * a.picks * sizeof(BeamKey) + 4 * a.picks * 64 * 8;
  if (lds > 64 * 1024) {
    static std::atomic<uint64_t> raised{0};
    e = raise_lds_limit(reinterpret_cast<const void*>(k_beam_pick), 160 * 1024, raised);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k_beam_pick, dim3(a.rows / a.beams), dim3(256), lds, st, a);
  return hipGetLastError();
}

uint64_t beam_copy_blocks(const BeamCopy& s, uint32_t n_rows) {
  return (s.bytes + kCopyChunk - 1) / kCopyChunk * s.pieces * n_rows;
}

hipError_t launch_beam_copy(const BeamCopy* states, uint32_t n, const int32_t* rows, uint32_t n_rows,
                            uint32_t src_rows, uint32_t* err, hipStream_t st) {
  uint32_t i = 0;
  while (i < n) {
    CopyArgs a{};
    uint64_t blocks = 0;
    for (; i < n && a.n < kCopyStates; ++i) {
      const uint64_t b = beam_copy_blocks(states[i], n_rows);
      if (b == 0) continue;
      if (a.n && blocks + b > kMaxBlocks) break;
      a.s[a.n] = states[i];
      a.end[a.n++] = blocks += b;
    }
    if (!a.n) break;
    a.rows = rows;
    a.n_rows = n_rows;
    a.src_rows = src_rows;
    a.err = err;
    hipLaunchKernelGGL(k_beam_copy, dim3((uint32_t)blocks), dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace smoe

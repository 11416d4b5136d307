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

#include <algorithm>
#include <type_traits>

namespace smoe {

typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kBeamBlocks = 512;         // two per CU, if rows and tiles allow
constexpr uint32_t kBeamTile = 4096;          // logits per block and round: 16 per thread

// e^x for x <= 0, from below -87 on (and for a NaN) 2^-126 (nothing beside a
// sum of at least one): 2^p with p = x log2 e rounded, times 1 + r ln 2 for what the rounding
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
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp_u32<0x111, 0xF>(v));
  v = max(v, dpp_u32<0x112, 0xF>(v));
  v = max(v, dpp_u32<0x114, 0xF>(v));
  v = max(v, dpp_u32<0x118, 0xF>(v));
  v = max(v, dpp_u32<0x142, 0xA>(v));
  v = max(v, dpp_u32<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max_f32(float v) { return readlane_f(wave_max_last(v), 63); }

__device__ __forceinline__ uint32_t count_below(u64 mask) {  // set bits of the lanes below this one
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Whether a beam still takes part with its own logits.
__device__ __forceinline__ bool beam_open(const BeamArgs& a, uint32_t row) {
  return a.scores[row] > -INFINITY && !(a.done && a.done[row]);
}

// Keys that a wave may hold: its P largest and what one tile can add, 17 P.
__host__ __device__ constexpr uint32_t beam_held(uint32_t picks) { return 18 * picks; }

// Each wave goes through its 1024 logits of every tile by itself and keeps what
// can be among the P largest: with T the least of the largest logits of at
// least P groups of lanes (over all tiles so far), or the P-th largest of more
// groups, at least P logits are >= T, and few more as a rule. Where a tile has
// more of them than there is room for, the wave's list is cut to its P largest
// and T becomes the P-th largest of the tile's single lanes: those above it lie
// in fewer than P lanes, and of those equal to it the P of lowest tokens
// suffice. In the end the block ranks what is >= the waves' largest T by
// counting.
//
// Four rows of 151936 (one tile a block) take 7.5 us, of which the loads are
// 2.0, threshold 0.7, list and ranks 1.7; 64 rows 13.1 us for 39 MB: loads 5.2,
// the exponentials 2.5, thresholds 2.4, lists 1.5, one after another (two blocks
// per CU are two waves per SIMD; the VALU is busy a quarter of the time). One
// tile a block took 14 us there (each with a threshold, a list to rank and its
// reductions). Peeling the last tile off, so that no branch stands between a
// tile's loads and its use, gained nothing.
__global__ __launch_bounds__(256) void k_beam_slice(BeamArgs a) {
  extern __shared__ __attribute__((aligned(16))) u64 lists[];  // per wave [19 P]; all waves' [72 P]
  __shared__ __attribute__((aligned(16))) float held[256 * 16];  // logits of threads that have one for the list
  __shared__ float least_of[4];
  __shared__ uint32_t count;
  const uint32_t t = threadIdx.x, lane = t & 63, P = a.picks;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  u64* const list = lists + wave * (beam_held(P) + P);
  const uint64_t first = (uint64_t)row * a.vocab;
  // Thread t's fours j of a tile: tokens start + 1024 j + 4 t on, counted from
  // the row's first, whatever its address: rows of the same logits are added up
  // the same way, so they tie. Fours lie on 4 bytes.
  auto load = [&](uint32_t tile, f32x4 (&q)[4]) {
    const uint32_t tok0 = tile * kBeamTile, tok = tok0 + t * 4;
    const float* const p = a.logits + first + tok;
    if (tok0 + kBeamTile <= a.vocab) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const f32x4u*>(p + 1024 * j);
      return;
    }
    // Places behind the row are -inf.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = tok + 1024 * j;
      q[j] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (k + 4 <= a.vocab) {
        q[j] = *reinterpret_cast<const f32x4u*>(p + 1024 * j);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (k + c < a.vocab) q[j][c] = p[1024 * j + c];
      }
    }
  };
  const uint32_t tile0 = slice * a.tiles;
  uint32_t tiles = a.tiles;
  while (tiles && (tile0 + tiles - 1) * kBeamTile >= a.vocab) --tiles;
  f32x4 q[4], ahead[4];
  if (tiles) load(tile0, q);
  if (!beam_open(a, row)) return;  // under the loads
  float m = -INFINITY, least = -INFINITY, most = -INFINITY;
  double sum = 0.0;
  uint32_t used = 0;
  for (uint32_t i = 0; i < tiles; ++i) {
    if (i + 1 < tiles) load(tile0 + i + 1, ahead);
    const uint32_t tok0 = (tile0 + i) * kBeamTile;
    // A NaN counts as -inf: maxima pass it over, and so does beam_exp.
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = __builtin_canonicalizef(q[e / 4][e % 4]);
    float tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) tm = fmaxf(tm, v[e]);
    // Sum of exponentials below the thread's running maximum.
    const float nm = fmaxf(m, tm);
    if (nm > -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) s += beam_exp(v[e] - nm);
      sum = sum * (double)(m > -INFINITY ? beam_exp(m - nm) : 0.f) + (double)s;
      m = nm;
    }
    // The P-th largest of the groups' largest: the smallest of those that fewer
    // than P are above.
    auto threshold = [&](float g, auto lanes) {
      uint32_t higher = 0;
#pragma unroll 16
      for (int l = 0; l < 64; l += decltype(lanes)::value) higher += readlane_f(g, l) > g ? 1u : 0u;
      return -wave_max_f32(higher < P ? -g : -INFINITY);
    };
    most = fmaxf(most, tm);
    if (i % 2 == 0) {  // every time: 64 beams 18.0 us, so 17.6
      const float two = fmaxf(most, dpp_f<0xB1>(most, most)), four = fmaxf(two, dpp_f<0x4E>(two, two));
      least = P <= 8    ? threshold(four, std::integral_constant<int, 4>{})
              : P <= 16 ? threshold(two, std::integral_constant<int, 2>{})
                        : threshold(most, std::integral_constant<int, 1>{});
    }
    // Bit 15 - e: v[e] >= least, as the sign of what is next below least minus v.
    const uint32_t lb = __float_as_uint(least + 0.f);
    const float below = least > -INFINITY ? __uint_as_float(lb == 0u ? 0x80000001u : (int32_t)lb > 0 ? lb - 1 : lb + 1) : least;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) bits = __builtin_amdgcn_alignbit(bits, __float_as_uint(below - v[e]), 31);
    const uint32_t mine = (uint32_t)__popc(bits);
    uint32_t upto = mine;
    upto += dpp_u32<0x111, 0xF>(upto);
    upto += dpp_u32<0x112, 0xF>(upto);
    upto += dpp_u32<0x114, 0xF>(upto);
    upto += dpp_u32<0x118, 0xF>(upto);
    upto += dpp_u32<0x142, 0xA>(upto);
    upto += dpp_u32<0x143, 0xC>(upto);
    const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    auto key = [&](float x, uint32_t token) { return (u64)float_ord(x) << 32 | ~token; };
    auto hold = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(held + t * 16 + 4 * j) = f32x4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
    };
    if (used + n <= beam_held(P) && least > -INFINITY) {
      if (bits) {
        hold();
        uint32_t at = used + upto - mine;
        do {
          const uint32_t e = (uint32_t)__clz((int)bits) - 16;
          list[at++] = key(held[t * 16 + e], tok0 + t * 4 + 1024 * (e / 4) + e % 4);
          bits &= ~(0x8000u >> e);
        } while (bits);
      }
      used += n;
    } else {
      if (used > P) {  // the P largest, by way of the places behind the list
        wave_lds();
        u64* const best = list + beam_held(P);
        for (uint32_t e = lane; e < used; e += 64) {
          const u64 k = list[e];
          uint32_t r = 0;
          for (uint32_t o = 0; o < used; ++o) r += list[o] > k ? 1u : 0u;
          if (r < P) best[r] = k;
        }
        wave_lds();
        if (lane < P) list[lane] = best[lane];
        used = P;
      }
      // 64 logits at a time in token order: the fours 0 of all lanes, the fours
      // 1, ..
      const float edge = fmaxf(least, threshold(tm, std::integral_constant<int, 1>{}));
      hold();
      wave_lds();
      auto look = [&](uint32_t r, uint32_t& token) {
        const uint32_t from = wave * 64 + r % 4 * 16 + lane / 4;
        token = tok0 + from * 4 + 1024 * (r / 4) + lane % 4;
        return fmaxf(held[from * 16 + 4 * (r / 4) + lane % 4], -INFINITY);
      };
      uint32_t token, met = 0;
      for (uint32_t r = 0; r < 16; ++r) {
        const float x = look(r, token);
        const bool same = x == edge && token < a.vocab;
        const u64 m1 = __ballot(x > edge), m2 = __ballot(same);
        if (x > edge) list[used + count_below(m1)] = key(x, token);
        used += (uint32_t)__popcll(m1);
        const uint32_t at = met + count_below(m2);
        if (same && at < P) list[used + at - met] = key(x, token);
        const uint32_t more = min((uint32_t)__popcll(m2), P - met);
        used += more;
        met += more;
      }
      wave_lds();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = ahead[j];
  }
  // What is >= the waves' largest T, then ranks by counting, a quarter of those
  // per lane of a quad.
  u64* const all = lists + 4 * (beam_held(P) + P);
  if (lane == 0) least_of[wave] = least;
  if (t == 0) count = 0;
  __syncthreads();
  const float floor = fmaxf(fmaxf(least_of[0], least_of[1]), fmaxf(least_of[2], least_of[3]));
  const u64 from = (u64)float_ord(floor) << 32;
  for (uint32_t e = lane; e < used + lane; e += 64) {
    const u64 k = e < used ? list[e] : 0;
    const u64 mask = __ballot(k >= from && k);
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&count, (uint32_t)__popcll(mask));
    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    if (k >= from && k) all[at + count_below(mask)] = k;
  }
  __syncthreads();
  u64* const out = a.cand + (uint64_t)blockIdx.x * P;
  const uint32_t n = count, part = t & 3, per = (n + 15) / 16 * 4;
  for (uint32_t e = t / 4; e < (n + 15) / 16 * 16; e += 64) {
    const u64 k = e < n ? all[e] : 0;
    uint32_t r = 0, i = part * per;
    const uint32_t last = min(i + per, n);
    for (; i + 4 <= last; i += 4) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(all + i), y = *reinterpret_cast<const ulonglong2*>(all + i + 2);
      r += (x.x > k ? 1u : 0u) + (x.y > k ? 1u : 0u) + (y.x > k ? 1u : 0u) + (y.y > k ? 1u : 0u);
    }
    for (; i < last; ++i) r += all[i] > k ? 1u : 0u;
    r += dpp_u32<0xB1, 0xF>(r);
    r += dpp_u32<0x4E, 0xF>(r);
    if (part == 0 && k && r < P) out[r] = k;
  }
  if (t >= n && t < P) out[t] = 0;
  const float wm = wave_max_f32(m);
  const double ws = wave_sum_f64(m > -INFINITY ? sum * (double)beam_exp(m - wm) : 0.0);
  if (lane == 0) a.stats[(uint64_t)blockIdx.x * 4 + wave] = BeamStat{ws, wm, 0u};
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
// order), is taken P times. The beams' P each are ranked by counting, each by eight
// lanes. 4.4 us for one request of four beams and 8 picks, 4.8 for 16: a chain
// of one load, P rounds of a wave's maximum (0.1 us each) and the ranks (one
// lane per pick: 0.8 us more).
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
          to[j] = beam_key((double)sc + ((double)ord_float(o) - lse), b, o, ~(uint32_t)head);
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
  for (uint32_t c = t / 8; c < (n + 31) / 32 * 32; c += 32) {
    const BeamKey k = c < n ? best[c] : BeamKey{0, 0};
    uint32_t r = 0;
    for (uint32_t i = t & 7; i < n; i += 8) r += above(best[i], k) ? 1u : 0u;
    r += dpp_u32<0xB1, 0xF>(r);
    r += dpp_u32<0x4E, 0xF>(r);
    r += dpp_u32<0x141, 0xF>(r);
    if ((t & 7) || !k.hi || r >= P) continue;
    const uint64_t o = (uint64_t)blockIdx.x * P + r;
    const double v = __longlong_as_double((long long)(k.hi >> 63 ? k.hi & ~(1ull << 63) : ~k.hi));
    a.out_scores[o] = (float)v;
    a.out_rows[o] = (int32_t)(row0 + kBeamMaxBeams - 1 - (uint32_t)(k.lo >> 60));
    a.out_tokens[o] = (int32_t)(kBeamMaxVocab - 1 - (uint32_t)(k.lo & (kBeamMaxVocab - 1)));
  }
}

// ---------------------------------------------------------------------------
// Reordering: a block per 16 KiB of a piece; a launch takes up to 32 states, so
// a cache of many layers needs few. 2.3 GB (40 states of 64 rows, four pieces
// of 150 KB, each source row taken twice) in 457 us, 5.0 TB/s, a large copy's
// rate; eight states of four rows of 64 KiB in 4.1 us. Addresses or strides that
// 4 does not divide go byte by byte (16 rows of 4 MiB, from the caches: 44 us, 18
// on 16 bytes and 20 on 4).
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
  const uint32_t tiles = (vocab + kBeamTile - 1) / kBeamTile;
  const uint64_t rows = (uint64_t)requests * beams;
  const uint32_t per = (uint32_t)std::max<uint64_t>((tiles + kBeamMaxSlices - 1) / kBeamMaxSlices,
                                                    std::min<uint64_t>((rows * tiles + kBeamBlocks - 1) / kBeamBlocks, tiles));
  const uint32_t slices = (tiles + per - 1) / per;
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
  hipLaunchKernelGGL(k_beam_slice, dim3(a.rows * a.slices), dim3(256), (4 * (beam_held(a.picks) + a.picks) + 4 * beam_held(a.picks)) * 8, st, a);
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

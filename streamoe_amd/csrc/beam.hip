// beam.hip — one step of a beam search behind the LM head.
//
//   k_beam_slice  a slice of one beam's logits: largest value, sum of
//                 exponentials, and its n_picks largest logits in order
//   k_beam_pick   one request: log-sum-exp of every beam, and the n_picks
//                 largest of score + logit - log-sum-exp among the slices' own
//   k_beam_copy   dst row i = src row rows[i] of a list of state tensors
//
// A logit becomes a 64-bit key, its bits in an order that integers compare
// (above) over the complement of its token (below), so keys are unique, equal
// logits fall in token order and selection needs no tie rules. To find the P
// largest of a block's values: the P-th largest T of the 256 threads' own
// largest is no larger than the P-th largest of all, and at most P threads
// hold keys >= T, so at most 16 P keys are collected and ranked by counting.
#include "common.h"
#include "kernels.h"

namespace smoe {

typedef unsigned long long u64;

constexpr uint32_t kBeamTile = 4096;  // logits per block and round: 16 per thread
constexpr uint32_t kBeamList = kBeamMaxPicks * 16 + kBeamMaxPicks;
constexpr uint32_t kOrdNegInf = 0x007FFFFFu;  // beam_ord(-inf)

// Order of floats as unsigned integers; -0 as +0, NaN as -inf.
__device__ __forceinline__ uint32_t beam_ord(float v) {
  const uint32_t b = __float_as_uint(v == v ? v + 0.f : -INFINITY);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// Whether a beam still takes part with its own logits.
__device__ __forceinline__ bool beam_open(const BeamArgs& a, uint32_t row) {
  return a.scores[row] > -INFINITY && !(a.done && a.done[row]);
}

__global__ __launch_bounds__(256) void k_beam_slice(BeamArgs a) {
  __shared__ __attribute__((aligned(16))) u64 heads[256];
  __shared__ u64 list[kBeamList], top[kBeamMaxPicks], thresh;
  __shared__ uint32_t count;
  __shared__ float red[4];
  __shared__ double redd[4];
  const uint32_t t = threadIdx.x, P = a.picks;
  const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  if (!beam_open(a, row)) return;
  const uint64_t first = (uint64_t)row * a.vocab, total = (uint64_t)a.rows * a.vocab;
  const uint32_t shift = (uint32_t)(first & 3);  // tiles start on 16 bytes, up to three logits ahead of the row
  float m = -INFINITY;
  double sum = 0.0;
  if (t < P) top[t] = 0;
  for (uint32_t tile = slice * a.tiles; tile < (slice + 1) * a.tiles; ++tile) {
    const int64_t tok0 = (int64_t)tile * kBeamTile - shift;
    if (tok0 >= (int64_t)a.vocab) break;
    float v[16];
    int64_t tok[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      tok[j] = tok0 + (j * 256 + t) * 4;
      const int64_t e = (int64_t)first + tok[j];
      f32x4 q = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (tok[j] < (int64_t)a.vocab) {
        if (e + 4 <= (int64_t)total) {
          q = *reinterpret_cast<const f32x4*>(a.logits + e);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (e + c < (int64_t)total) q[c] = a.logits[e + c];
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) v[4 * j + c] = q[c];
    }
    u64 key[16], best = 0;
    float tm = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t k = tok[i / 4] + i % 4;
      const bool in = k >= 0 && k < (int64_t)a.vocab;
      const uint32_t o = beam_ord(v[i]);
      key[i] = in ? (u64)o << 32 | (uint32_t)~(uint32_t)k : 0;
      v[i] = in ? beam_value(o) : -INFINITY;
      best = key[i] > best ? key[i] : best;
      tm = fmaxf(tm, v[i]);
    }
    // Sum of exponentials below the thread's running maximum.
    const float nm = fmaxf(m, tm);
    if (nm > -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += expf(v[i] - nm);
      sum = sum * (double)expf(m - nm) + (double)s;
      m = nm;
    }
    heads[t] = best;
    if (t == 0) thresh = 0, count = 0;
    __syncthreads();
    uint32_t rank = 0;
    for (uint32_t i = 0; i < 256; ++i) rank += heads[i] > best ? 1u : 0u;
    if (best && rank == P - 1) thresh = best;
    __syncthreads();
    const u64 floor = top[P - 1], T = thresh > floor ? thresh : floor;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (key[i] && key[i] >= T) list[atomicAdd(&count, 1u)] = key[i];
    if (t < P && top[t]) list[atomicAdd(&count, 1u)] = top[t];
    __syncthreads();
    const uint32_t n = count;
    if (t < P) top[t] = 0;
    __syncthreads();
    for (uint32_t c = t; c < n; c += 256) {
      const u64 k = list[c];
      uint32_t r = 0;
      for (uint32_t i = 0; i < n; ++i) r += list[i] > k ? 1u : 0u;
      if (r < P) top[r] = k;
    }
    __syncthreads();
  }
  const float bm0 = wave_max(m);
  if ((t & 63) == 0) red[t >> 6] = bm0;
  __syncthreads();
  const float bm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const double ws = wave_sum_f64(m > -INFINITY ? sum * (double)expf(m - bm) : 0.0);
  if ((t & 63) == 0) redd[t >> 6] = ws;
  __syncthreads();
  if (t == 0) a.stats[blockIdx.x] = BeamStat{(redd[0] + redd[1]) + (redd[2] + redd[3]), bm, 0u};
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

__global__ __launch_bounds__(256) void k_beam_pick(BeamArgs a) {
  __shared__ BeamKey heads[kBeamMaxBeams * kBeamMaxSlices], list[kBeamMaxPicks * kBeamMaxPicks];
  __shared__ double lse[kBeamMaxBeams], score[kBeamMaxBeams];
  __shared__ uint32_t open[kBeamMaxBeams];  // 1 by its logits, 2 ended (the pad token keeps the score), 0 nothing left
  __shared__ BeamKey thresh;
  __shared__ uint32_t count;
  const uint32_t t = threadIdx.x, lane = t & 63, P = a.picks, W = a.beams, S = a.slices;
  const uint32_t row0 = blockIdx.x * W;
  for (uint32_t b = t >> 6; b < W; b += 4) {
    const uint32_t row = row0 + b;
    const float sc = a.scores[row];
    const bool ended = a.done && a.done[row];
    uint32_t st = ended && sc > -INFINITY ? 2u : 0u;
    double l = 0.0;
    if (beam_open(a, row)) {
      BeamStat s{0.0, -INFINITY, 0u};
      if (lane < S) s = a.stats[(uint64_t)row * S + lane];
      const float m = wave_max(s.max);
      const double sum = wave_sum_f64(s.max > -INFINITY ? s.sum * exp((double)s.max - (double)m) : 0.0);
      // All logits masked, or an infinity among them: no token has a value.
      if (m > -INFINITY && m < INFINITY) st = 1u, l = (double)m + log(sum);
    }
    if (lane == 0) lse[b] = l, score[b] = (double)sc, open[b] = st;
  }
  if (t == 0) thresh = BeamKey{0, 0}, count = 0;
  __syncthreads();
  // Entry j of list (beam b, slice s), in falling order; none: {0, 0}.
  auto entry = [&](uint32_t b, uint32_t s, uint32_t j) {
    BeamKey none{0, 0};
    if (open[b] == 1u) {
      const u64 k = a.cand[((uint64_t)(row0 + b) * S + s) * P + j];
      if (!k) return none;
      const uint32_t o = (uint32_t)(k >> 32);
      return beam_key(score[b] + ((double)beam_value(o) - lse[b]), b, o, ~(uint32_t)k);
    }
    if (s) return none;
    if (open[b] == 2u) {
      if (j == 0) return beam_key(score[b], b, kOrdNegInf, a.pad);
      const uint32_t tok = j - 1 < a.pad ? j - 1 : j;
      return tok < a.vocab ? beam_key(-INFINITY, b, kOrdNegInf, tok) : none;
    }
    return j < a.vocab ? beam_key(-INFINITY, b, kOrdNegInf, j) : none;
  };
  const uint32_t L = W * S;
  for (uint32_t i = t; i < L; i += 256) heads[i] = entry(i / S, i % S, 0);
  __syncthreads();
  for (uint32_t i = t; i < L; i += 256) {
    const BeamKey h = heads[i];
    uint32_t rank = 0;
    for (uint32_t k = 0; k < L; ++k) rank += above(heads[k], h) ? 1u : 0u;
    if (h.hi && rank == P - 1) thresh = h;
  }
  __syncthreads();
  const BeamKey T = thresh;
  for (uint32_t i = t; i < L; i += 256) {
    if (!heads[i].hi || above(T, heads[i])) continue;
    for (uint32_t j = 0; j < P; ++j) {
      const BeamKey k = entry(i / S, i % S, j);
      if (!k.hi || above(T, k)) break;
      list[atomicAdd(&count, 1u)] = k;
    }
  }
  __syncthreads();
  const uint32_t n = count;
  for (uint32_t c = t; c < n; c += 256) {
    const BeamKey k = list[c];
    uint32_t r = 0;
    for (uint32_t i = 0; i < n; ++i) r += above(list[i], k) ? 1u : 0u;
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
  const uint64_t sb = al256(lists * sizeof(BeamStat));
  if (a) {
    a->slices = slices;
    a->tiles = per;
    a->stats = reinterpret_cast<BeamStat*>(base);
    a->cand = reinterpret_cast<unsigned long long*>(base + sb);
  }
  return sb + al256(lists * picks * 8);
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(k_beam_slice, dim3(a.rows * a.slices), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_beam_pick, dim3(a.rows / a.beams), dim3(256), 0, st, a);
  return hipGetLastError();
}

// Blocks of one state, and whether a launch can hold them.
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
      if (a.n && blocks + b > kBeamCopyMaxBlocks) break;
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

// sample.hip — one token per row of logits, drawn from the filtered
// distribution.
//
//   k_sample_top   a slice's largest key; clears the row's sums
//   k_sample_bins  the row's logits by their distance from its largest: counts
//                  and masses per bin, of the row and (masses) of the slice
//   k_sample_list  the keys of the bins in which a border lies, and each slice's
//                  mass of what is kept for certain
//   k_sample_pick  the borders themselves, the sum, and the token
//
// A logit becomes 32 bits in an order that integers compare, and a key with the
// complement of its token below it, so keys are unique and the order of the
// filters is that of falling keys. Bins are by the distance d from the row's
// largest logit (a rounded difference, but it never falls as logits fall): 64 to
// every power of two of d from 1/16 to 64, so that they are finest where the
// mass is. All three filters keep a first part of the order: what decides is one
// key, and only the bins around it have to be looked into.
// (1536 finer bins cost more than their shorter lists save: 16 rows of wide
// nuclei 35 us instead of 30; of 64 mixed rows they save 2 of 68.)
//
// A mass e^((logit - max) / T) is f64 and then an integer of 2^-s: sums of
// integers are the same in any order, so atomics may form them. Masses of whole
// bins are formed once. A row with a small top-k needs no masses but of those
// tokens: all of them are listed, the list is sorted and the token found in it
// (one row of 151936 with top-k 20: 19 us, with bins of masses and the slice gone
// through again 24). A larger top-k alone needs the masses of what it keeps.
//
// The reads (39 MB of 64 rows of 151936: 8 us) are what a call cannot do without;
// later passes find most of them in the memory-side cache. What bounds the four
// is: top, the reads, 9 us at 64 rows; bins, the series in f64 and the additions
// in LDS, 14; list, three comparisons a logit, 13; pick, one block's chain of
// loads, scans and selections, 16 (one row: 2.7, 4.4, 5.5 and 6.5).
#include "common.h"
#include "kernels.h"

namespace smoe {

typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kSampleThreads = 256, kPickThreads = 512;
constexpr uint32_t kSampleSlices = 128;  // of a row at most
constexpr uint32_t kCountStride = kSampleBins + 4;
constexpr uint32_t kNoBin = kSampleBins;
// Longer lists are not sorted but selected from (16 rows of wide nuclei, lists of
// 360 to 770: 27 us; with up to 512 sorted 30; up to 64 as here).
constexpr uint32_t kSort = 256;
constexpr uint32_t kSmallK = 448;  // with the tokens that share its bin, mostly, a block's threads

// Bin of a logit, 0 the largest's; least distance of a bin (not of 0).
constexpr uint32_t kFirst = (127 - 4) << 6;  // the upper bits of 1/16
__device__ __forceinline__ float sample_bin_from(uint32_t bin) { return __uint_as_float((kFirst + bin) << 17); }
__device__ __forceinline__ uint32_t sample_bin(float max, float l) {
  const float d = max - l;                     // NaN where both are infinite: 0
  const uint32_t b = d > 0.f ? __float_as_uint(d) >> 17 : 0u;
  return b < kFirst ? 0u : min(b - kFirst, kSampleBins - 1);
}

// 2^(t + up) for -70 <= t <= 0, to 2^-44 of it: t = n + f, and (2^f - 1) / f as
// the polynomial that agrees with it at nine Chebyshev points of [-1/2, 1/2]. n
// is the lower word of t + 1.5 2^52 and goes into the exponent: conversions and
// the scaling instruction take four times as long as an addition.
__device__ __forceinline__ double sample_exp2(double t, int up) {
  constexpr double c[9] = {0.6931471805599453,     0.2402265069581299,      0.055504108664760424,
                           0.009618129159402558,   0.0013333558179043112,   0.00015403455852453838,
                           1.525268684626772e-05,  1.3255224878668817e-06,  1.0203121063391729e-07};
  const double whole = t + 0x1.8p52, f = t - (whole - 0x1.8p52);
  double e = c[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) e = __builtin_fma(e, f, c[i]);
  const u64 bits = (u64)__double_as_longlong(__builtin_fma(e, f, 1.0));
  const uint32_t n = (uint32_t)__double_as_longlong(whole) + (uint32_t)up;
  return __longlong_as_double((long long)(bits + ((u64)(n << 20) << 32)));
}

struct SampleRow {
  bool good, greedy;
  uint32_t k;              // kept at most; 0: all
  double inv_t, top_p, min_p, u;
  __device__ bool by_mass() const { return top_p < 1.0; }
  __device__ bool small() const { return k && k <= kSmallK; }
  __device__ bool masses() const { return !small() && (by_mass() || !k); }  // of all bins
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, uint32_t row) {
  SampleRow r;
  const float t = a.temperature ? a.temperature[row] : 1.f, p = a.top_p ? a.top_p[row] : 1.f;
  const float m = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
  const int32_t k = a.top_k ? a.top_k[row] : 0;
  r.good = t >= 0.f && t < INFINITY && p >= 0.f && m >= 0.f && m <= 1.f && u >= 0.f && u < 1.f;
  r.greedy = t == 0.f;
  r.k = k <= 0 || (uint32_t)k >= a.vocab ? 0u : (uint32_t)k;
  r.inv_t = 1.0 / (double)t;
  r.top_p = p;
  r.min_p = m;
  r.u = u;
  return r;
}

// What a row's largest logit makes of the others.
struct SampleScale {
  float top;
  bool infinite;            // +inf: 0 beside the others' -inf
  double max, inv_t, inv_t2, least;  // 1 / T, also for powers of two; what min_p keeps, in units
  int up;                   // a mass of 1 is 2^up
  __device__ SampleScale(const SampleArgs& a, const SampleRow& r, uint32_t o)
      : top(ord_float(o)), infinite(o == 0xFF800000u), max(infinite ? 0.0 : (double)top), inv_t(r.inv_t),
        inv_t2(r.inv_t * 1.4426950408889634), least(__builtin_ldexp(r.min_p, a.up)), up(a.up) {}
  __device__ float finite(float l) const { return infinite ? (l == INFINITY ? 0.f : -INFINITY) : l; }
  __device__ double log_mass(float l) const { return ((double)finite(l) - max) * inv_t; }
  // The mass as an integer; *kept: whether min_p keeps it. 0 below 2^-70, as for
  // -inf and NaN. No branches, so that several logits' series are formed side by
  // side.
  __device__ u64 mass(float l, bool* kept) const {
    const double e = sample_exp2(fmax(((double)finite(l) - max) * inv_t2, -70.0), up);
    *kept = e >= least;
    // The sum's last place is 1: its lower bits are the rounded product.
    return (u64)__double_as_longlong(e + 0x1p52) - 0x4330000000000000ull;
  }
  // Of four logits; 0 where min_p does not keep it (if `kept_only`).
  __device__ void masses(f32x4 l, u64 (&m)[4], bool kept_only) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bool kept;
      m[j] = mass(l[j], &kept);
      m[j] = kept || !kept_only ? m[j] : 0ull;
    }
  }
};

__device__ __forceinline__ u64 sample_key(float l, uint32_t token) { return (u64)float_ord(l) << 32 | (uint32_t)~token; }
__device__ __forceinline__ uint32_t key_token(u64 key) { return ~(uint32_t)key; }

// Over the block's T threads; lds: T / 64 words. Every thread gets the result.
template <uint32_t T>
__device__ __forceinline__ u64 block_max(u64 v, u64* lds) {
  v = wave_max_last_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (uint32_t w = 1; w < T / 64; ++w) v = max(v, lds[w]);
  return v;
}
// Sums of the threads before this one, of two values (lds: 2 T / 64 words);
// all: of all.
template <uint32_t T, uint32_t N>
__device__ __forceinline__ void block_before(u64 (&v)[N], u64 (&all)[N], u64* lds) {
  u64 s[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) s[i] = wave_scan_u64(v[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) lds[(threadIdx.x >> 6) * N + i] = s[i];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    u64 skip = 0, sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < T / 64; ++w) {
      const u64 x = lds[w * N + i];
      if (w < threadIdx.x >> 6) skip += x;
      sum += x;
    }
    all[i] = sum;
    v[i] = skip + s[i] - v[i];
  }
}
template <uint32_t T>
__device__ __forceinline__ u64 block_sum(u64 v, u64* lds) {
  u64 a[1] = {v}, s[1];
  block_before<T, 1>(a, s, lds);
  return s[0];
}
template <uint32_t T>
__device__ __forceinline__ u64 block_before(u64 v, u64* all, u64* lds) {
  u64 a[1] = {v}, s[1];
  block_before<T, 1>(a, s, lds);
  *all = s[0];
  return a[0];
}

// Thread t's four logits of a thousand from `first` on, -inf behind the row.
__device__ __forceinline__ f32x4 sample_load(const float* row, uint32_t at, uint32_t vocab) {
  if (at + 4 <= vocab) return *reinterpret_cast<const f32x4u*>(row + at);
  f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    if (at + j < vocab) v[j] = row[at + j];
  return v;
}

// A thread's fours of a slice, a thousand logits of the block at a time, two of
// these on their way. Kernels that follow one another go through a slice in
// turns (BACK: from its end): what an XCD's L2 still holds is what the one before
// read last.
template <bool BACK>
struct SampleFours {
  static constexpr uint32_t kAhead = 2, kStep = kSampleThreads * 4;
  const float* row;
  uint32_t vocab, first, steps, at;  // this thread's place in the first step; steps of the slice
  f32x4 next[kAhead];
  __device__ __forceinline__ uint32_t place(uint32_t i) const { return first + (BACK ? steps - 1 - i : i) * kStep; }
  __device__ __forceinline__ SampleFours(const SampleArgs& a, uint32_t r, uint32_t slice)
      : row(a.logits + (uint64_t)r * a.vocab), vocab(a.vocab), first(slice * a.slice + threadIdx.x * 4),
        steps((min(a.slice, a.vocab - slice * a.slice) + kStep - 1) / kStep), at(0) {
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) next[j] = load(j);
  }
  __device__ __forceinline__ f32x4 load(uint32_t i) const {
    return i < steps ? sample_load(row, place(i), vocab) : f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  }
  template <class F>
  __device__ __forceinline__ void go(F each) {  // each(logits, first token)
    for (; at < steps; at += kAhead) {
      f32x4 v[kAhead];
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        v[j] = next[j];
        next[j] = load(at + kAhead + j);
      }
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j)
        if (at + j < steps) each(v[j], place(at + j));
    }
  }
};

// What a thread asks for first: all of it is on its way at once.
__device__ __forceinline__ u64 slice_top(const SampleArgs& a, uint32_t row) {
  return threadIdx.x < a.slices ? a.tops[row * a.slices + threadIdx.x] : 0ull;
}

__global__ __launch_bounds__(kSampleThreads) void k_sample_top(SampleArgs a) {
  __shared__ u64 lds[4];
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  u64 top = 0;
  SampleFours<false> fours(a, row, slice);
  fours.go([&](f32x4 v, uint32_t i) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const u64 key = sample_key(v[j], i + j);
      if (v[j] > -INFINITY && key > top) top = key;
    }
  });
  top = block_max<kSampleThreads>(top, lds);
  if (t == 0) a.tops[blockIdx.x] = top;
  for (uint32_t i = slice * kSampleThreads + t; i < kCountStride; i += a.slices * kSampleThreads) {
    a.count[(uint64_t)row * kCountStride + i] = 0;
    if (i < kSampleBins) a.mass[(uint64_t)row * kSampleBins + i] = 0;
  }
}

__global__ __launch_bounds__(kSampleThreads) void k_sample_bins(SampleArgs a) {
  __shared__ u64 mass[kSampleBins];
  __shared__ uint32_t count[kSampleBins];
  __shared__ u64 lds[4];
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const SampleRow r = sample_row(a, row);
  u64 top = slice_top(a, row);
  SampleFours<true> fours(a, row, slice);
  if (!r.good || r.greedy) return;
  for (uint32_t i = t; i < kSampleBins; i += kSampleThreads) mass[i] = 0, count[i] = 0;
  top = block_max<kSampleThreads>(top, lds);
  if (!top) return;
  const SampleScale scale(a, r, (uint32_t)(top >> 32));
  const bool counts = r.k, masses = r.masses();
  fours.go([&](f32x4 v, uint32_t) {
    u64 m[4] = {0, 0, 0, 0};
    if (masses) scale.masses(v, m, false);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t bin = sample_bin(scale.top, v[j]);
      if (counts && v[j] > -INFINITY) atomicAdd(&count[bin], 1u);
      if (m[j]) atomicAdd(&mass[bin], m[j]);
    }
  });
  __syncthreads();
  u64* const own = a.slice_mass + (uint64_t)blockIdx.x * kSampleBins;
  for (uint32_t i = t; i < kSampleBins; i += kSampleThreads) {
    if (count[i]) atomicAdd(a.count + (uint64_t)row * kCountStride + i, count[i]);
    if (mass[i]) atomicAdd(a.mass + (uint64_t)row * kSampleBins + i, mass[i]);
    if (masses) own[i] = mass[i];
  }
}

// The bins in which the borders lie (kNoBin: there is none).
struct SampleBorder {
  uint32_t k_bin, k_before;     // top-k's, and tokens before it
  u64 k_mass;                   // mass before it, or of all
  uint32_t p_first, p_last;     // top-p's is one of these
  u64 p_before;                 // mass before the first of them
  uint32_t m_first, m_last;     // min-p's is one of these
  bool small;                   // all of top-k is listed
  __device__ uint32_t certain() const { return small ? 0u : min(min(k_bin, p_first), m_first); }  // bins below it are kept
  // Bins from it on are neither kept nor listed.
  __device__ uint32_t end() const {
    if (k_bin == kNoBin && p_first == kNoBin) return m_first == kNoBin ? kNoBin : m_last + 1;
    const uint32_t e = k_bin == kNoBin ? p_last + 1 : k_bin + 1;  // top-p's border is not behind top-k's
    return min(max(e, m_first == kNoBin ? 0u : m_last + 1), kNoBin);
  }
  __device__ bool listed(uint32_t bin) const {
    if (small) return bin <= k_bin;
    return bin == k_bin || (bin >= p_first && bin <= p_last) || (bin >= m_first && bin <= m_last);
  }
};
struct SampleBorderLds {
  u64 part[2 * kPickThreads / 64];
  SampleBorder b;
  u64 k_own;
};
__device__ __forceinline__ u64 share_of(double p, u64 of) {  // at least one
  const double v = __builtin_ceil(p * (double)of);
  return v >= 1.0 ? (u64)v : 1ull;
}
// Thread t of T has the B bins from B t on.
template <uint32_t T>
struct SampleShare {
  static constexpr uint32_t B = (kSampleBins + T - 1) / T;
  uint32_t c[B];
  u64 m[B], before;  // counts; masses; mass of the bins ahead
  __device__ __forceinline__ void load(const SampleArgs& a, uint32_t row) {
#pragma unroll
    for (uint32_t j = 0; j < B; ++j) {
      const uint32_t i = B * threadIdx.x + j;
      c[j] = i < kSampleBins ? a.count[(uint64_t)row * kCountStride + i] : 0u;
      m[j] = i < kSampleBins ? a.mass[(uint64_t)row * kSampleBins + i] : 0ull;
    }
  }
};
template <uint32_t T>
__device__ __forceinline__ SampleBorder sample_border(const SampleRow& r, const SampleScale& scale, SampleBorderLds* lds,
                                                      SampleShare<T>& share) {
  constexpr uint32_t B = SampleShare<T>::B;
  const uint32_t t = threadIdx.x;
  u64 own[2] = {0, 0}, all[2];
#pragma unroll
  for (uint32_t j = 0; j < B; ++j) {
    own[0] += share.c[j];
    own[1] += share.m[j];
  }
  block_before<T, 2>(own, all, lds->part);
  const auto& c = share.c;
  const auto& m = share.m;
  u64 n = own[0];
  share.before = own[1];
  if (t == 0) {
    lds->b = SampleBorder{kNoBin, 0, all[1], kNoBin, kNoBin, 0, kNoBin, kNoBin, r.small()};
    lds->k_own = 0;
    if (!r.small() && r.min_p > 0.0 && !scale.infinite) {
      // The last logit that min-p keeps, to within more than its roundings.
      const double x = log(r.min_p), at = scale.max + x / r.inv_t, off = (fabs(scale.max) + fabs(at)) * 0x1p-22 + fabs(x / r.inv_t) * 0x1p-40;
      lds->b.m_first = sample_bin(scale.top, (float)(at + off));
      lds->b.m_last = sample_bin(scale.top, (float)(at - off));
    }
  }
  __syncthreads();
  if (r.k) {
    u64 w = share.before;
#pragma unroll
    for (uint32_t j = 0; j < B; ++j) {
      if (n < r.k && r.k <= n + c[j]) {
        lds->b.k_bin = B * t + j;
        lds->b.k_before = (uint32_t)n;
        lds->b.k_mass = w;
        lds->k_own = m[j];
      }
      n += c[j];
      w += m[j];
    }
    __syncthreads();
  }
  if (r.by_mass() && !r.small()) {
    const u64 lo = share_of(r.top_p, lds->b.k_mass), hi = share_of(r.top_p, lds->b.k_mass + lds->k_own);
    u64 w = share.before;
#pragma unroll
    for (uint32_t j = 0; j < B; ++j) {
      if (w < lo && lo <= w + m[j]) {
        lds->b.p_first = B * t + j;
        lds->b.p_before = w;
      }
      if (w < hi && hi <= w + m[j]) lds->b.p_last = B * t + j;
      w += m[j];
    }
  }
  __syncthreads();
  SampleBorder b = lds->b;
  // Behind the other borders min-p's does not count.
  if (b.m_first > min(b.k_bin, b.p_last)) b.m_first = b.m_last = kNoBin;
  return b;
}

// A block gathers in LDS the keys of all distances that it has to look at, three
// comparisons a logit, and sorts them out afterwards, a key per thread: masses
// of what is kept for certain (top-k alone), the list, one addition to the row's
// count per block (thousands to one place are one after another). Bins, masses
// and lists a step at a time took 10 us of blocks of wide nuclei (10 thousand
// logits) instead of 5.
constexpr uint32_t kListHeld = 2048;
__global__ __launch_bounds__(kSampleThreads) void k_sample_list(SampleArgs a) {
  __shared__ u64 lds[2 * kSampleThreads / 64];
  __shared__ SampleBorderLds border_lds;
  __shared__ u64 held[kListHeld];
  __shared__ uint32_t n_held, list_at;
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const SampleRow r = sample_row(a, row);
  u64 top = slice_top(a, row);
  SampleShare<kSampleThreads> share;
  share.load(a, row);
  SampleFours<false> fours(a, row, slice);
  if (!r.good || r.greedy) return;
  top = block_max<kSampleThreads>(top, lds);
  if (!top) return;
  const SampleScale scale(a, r, (uint32_t)(top >> 32));
  const SampleBorder b = sample_border<kSampleThreads>(r, scale, &border_lds, share);
  if (t == 0) n_held = 0;
  __syncthreads();
  uint32_t* const count = a.count + (uint64_t)row * kCountStride + kSampleBins;
  u64* const list = a.list + (uint64_t)row * a.vocab;
  const uint32_t certain = b.certain();
  u64 sum = 0;
  const bool masses = r.masses();
  if (masses) {
    const u64* const own = a.slice_mass + (uint64_t)blockIdx.x * kSampleBins;
    for (uint32_t i = t; i < certain; i += kSampleThreads) sum += own[i];
  }
  // Distances of what has to be looked at (most logits are behind it). A NaN
  // bounds none: distances of finite logits may be infinite, those beside +inf
  // are infinity and NaN.
  const uint32_t last = b.end();
  const float near = !masses || certain == 0 || scale.infinite ? -INFINITY : sample_bin_from(certain);
  const bool no_far = scale.infinite || last == kNoBin || (b.small && b.k_bin == kNoBin);
  const float far = no_far ? __builtin_nanf("") : sample_bin_from(last);
  // Nothing to list, and masses of bins: the slice need not be read. (Without them
  // the masses of all that is kept are formed here, also where no border was found:
  // a top-k of more than there are.)
  if (certain < kNoBin || !masses) fours.go([&](f32x4 v, uint32_t i) {
    u64 hits[4];
    uint32_t n = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const float d = scale.top - v[j];
      hits[j] = __ballot(!(d < near) && !(d >= far) && v[j] > -INFINITY);
      n += (uint32_t)__popcll(hits[j]);
    }
    if (!n) return;
    // A place for each, one addition per wave.
    uint32_t at = 0;
    if ((t & 63) == 0) at = atomicAdd(&n_held, n);
    at = __builtin_amdgcn_readfirstlane(at);
    if (at + n <= kListHeld) {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        if (hits[j] >> (t & 63) & 1)
          held[__builtin_amdgcn_mbcnt_hi((uint32_t)(hits[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits[j], at))] = sample_key(v[j], i + j);
        at += (uint32_t)__popcll(hits[j]);
      }
      return;
    }
    // No room.
    u64 m[4] = {0, 0, 0, 0};
    if (!masses && certain) scale.masses(v, m, false);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t place = __builtin_amdgcn_mbcnt_hi((uint32_t)(hits[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits[j], at));
      if (hits[j] >> (t & 63) & 1) {
        const uint32_t bin = sample_bin(scale.top, v[j]);
        if (place < kListHeld)
          held[place] = sample_key(v[j], i + j);
        else if (bin < certain)
          sum += m[j];
        else if (b.listed(bin))
          list[atomicAdd(count, 1u)] = sample_key(v[j], i + j);
      }
      at += (uint32_t)__popcll(hits[j]);
    }
  });
  __syncthreads();
  const uint32_t n = min(n_held, kListHeld);
  // Where no bin between the first and the last listed one is not, all are.
  const bool plain = !scale.infinite && (b.small || (masses && (b.k_bin != kNoBin) + (b.p_first != kNoBin) + (b.m_first != kNoBin) == 1));
  u64 own[2] = {sum, 0}, all[2];
  if (plain) {
    if (t == 0 && n) list_at = atomicAdd(count, n);
  } else {
    for (uint32_t i = t; i < n; i += kSampleThreads) {
      const float l = ord_float((uint32_t)(held[i] >> 32));
      const uint32_t bin = sample_bin(scale.top, l);
      bool kept;
      if (bin < certain)
        own[0] += scale.mass(l, &kept);
      else
        own[1] += b.listed(bin);
    }
  }
  block_before<kSampleThreads, 2>(own, all, lds);
  if (t == 0) a.kept[blockIdx.x] = all[0];
  if (plain) {
    for (uint32_t i = t; i < n; i += kSampleThreads) list[list_at + i] = held[i];
    return;
  }
  if (!all[1]) return;
  if (t == 0) list_at = atomicAdd(count, (uint32_t)all[1]);
  __syncthreads();
  uint32_t to = list_at + (uint32_t)own[1];
  for (uint32_t i = t; i < n; i += kSampleThreads) {
    const uint32_t bin = sample_bin(scale.top, ord_float((uint32_t)(held[i] >> 32)));
    if (bin >= certain && b.listed(bin)) list[to++] = held[i];
  }
}

// The row's list: with their masses in registers, up to eight keys of a thread;
// a longer one (ties, logits past 64 from the largest) out of memory, again and
// again.
constexpr uint32_t kPickEach = 8, kPickBins = (kSampleBins + kPickThreads - 1) / kPickThreads;
struct SampleList {
  const u64* list;
  uint32_t n;
  u64 keys[kPickEach], masses[kPickEach];
  __device__ static float logit(u64 key) { return ord_float((uint32_t)(key >> 32)); }
  __device__ bool held() const { return n <= kPickEach * kPickThreads; }
  __device__ __forceinline__ void hold(const SampleScale& scale) {  // keys[0] is there
    if (!held()) return;
#pragma unroll
    for (uint32_t h = 0; h < kPickEach; h += 4) {
      if (n <= h * kPickThreads) break;
#pragma unroll
      for (uint32_t j = h ? h : 1; j < h + 4; ++j) keys[j] = threadIdx.x + j * kPickThreads < n ? list[threadIdx.x + j * kPickThreads] : 0ull;
      u64 m[4];
      scale.masses(f32x4{logit(keys[h]), logit(keys[h + 1]), logit(keys[h + 2]), logit(keys[h + 3])}, m, false);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) masses[h + j] = m[j];
    }
  }
  // f(key, mass) of this thread's.
  template <class F>
  __device__ __forceinline__ void each(const SampleScale& scale, F f) const {
    if (held()) {
#pragma unroll
      for (uint32_t j = 0; j < kPickEach; ++j)
        if (threadIdx.x + j * kPickThreads < n) f(keys[j], masses[j]);
    } else {
      for (uint32_t i = threadIdx.x; i < n; i += kPickThreads) {
        bool kept;
        f(list[i], scale.mass(logit(list[i]), &kept));
      }
    }
  }
};

// Its entries of one bin, in order; a place is the distance from `first` (in
// steps of the order) and the token in one number, the first of the order the
// smallest.
struct SamplePlaces {
  u64 thr;              // only keys from it on
  float max;
  uint32_t bin, end;    // kNoBin: all of them, up to bin end; else the same
  uint32_t first, token_bits;
  __device__ bool in(u64 key) const { return bin == kNoBin || (key >= thr && sample_bin(max, ord_float((uint32_t)(key >> 32))) == bin); }
  __device__ u64 place(u64 key) const { return (u64)(first - (uint32_t)(key >> 32)) << token_bits | key_token(key); }
  __device__ u64 key(u64 p) const {
    return (u64)(first - (uint32_t)(p >> token_bits)) << 32 | (uint32_t)~(uint32_t)(p & ((1ull << token_bits) - 1));
  }
};

constexpr int kDigit = 9;
static_assert(1u << kDigit == kPickThreads, "a digit's value per thread");
struct SelectLds {
  u64 weight[1u << kDigit];
  uint32_t count[1u << kDigit];
  u64 part[kPickThreads / 64];
  u64 prefix, rest, found;
  u64 few[64], few_weight[64];
  uint32_t left, n_few;
};
// Key of the first place up to which the weights (masses, or 1 each) add up to
// `target` or more, digit after digit of the places from the top; there is one.
// When 64 keys or fewer share the digits, a wave compares them with one another:
// two digits less, 1.2 us each, for 1.
__device__ __forceinline__ u64 sample_select(const SampleList& list, SamplePlaces s, const SampleScale& scale, u64 target, bool by_mass,
                                             SelectLds* lds) {
  const uint32_t t = threadIdx.x;
  // The values that the bins may hold, to within more than a distance's rounding.
  s.first = float_ord(s.max);
  uint32_t last = kOrdNegInf;
  if (!scale.infinite) {
    if (s.bin != kNoBin && s.bin) s.first = float_ord((float)(scale.max - sample_bin_from(s.bin) * (1 - 0x1p-22))) + 1;
    if (s.end < kSampleBins - 1) last = float_ord((float)(scale.max - sample_bin_from(s.end + 1) * (1 + 0x1p-22))) - 1;
  }
  const uint32_t span = s.first - last;
  int shift = (int)((span ? 32 - __builtin_clz(span) : 0) + s.token_bits);
  u64 prefix = 0;  // the digits above shift
  for (;;) {
    const int width = min(shift, kDigit);
    shift -= width;
    lds->weight[t] = 0;
    lds->count[t] = 0;
    if (t == 0) lds->n_few = 0;
    __syncthreads();
    list.each(scale, [&](u64 key, u64 mass) {
      const u64 p = s.place(key);
      if (!s.in(key) || p >> (shift + width) != prefix) return;
      const uint32_t digit = (uint32_t)(p >> shift) & ((1u << width) - 1);
      atomicAdd(&lds->count[digit], 1u);
      if (by_mass) atomicAdd(&lds->weight[digit], mass);
    });
    __syncthreads();
    const u64 w = by_mass ? lds->weight[t] : lds->count[t];
    u64 all;
    const u64 before = block_before<kPickThreads>(w, &all, lds->part);
    if (before < target && target <= before + w) {
      lds->prefix = prefix << width | t;
      lds->rest = target - before;
      lds->left = lds->count[t];
    }
    __syncthreads();
    prefix = lds->prefix;
    target = lds->rest;
    if (shift == 0) return s.key(prefix);
    if (lds->left <= 64) break;
    __syncthreads();
  }
  list.each(scale, [&](u64 key, u64 mass) {
    if (!s.in(key) || s.place(key) >> shift != prefix) return;
    const uint32_t i = atomicAdd(&lds->n_few, 1u);
    if (i < 64) lds->few[i] = key, lds->few_weight[i] = by_mass ? mass : 1ull;
  });
  __syncthreads();
  if (t < 64) {
    const uint32_t n = min(lds->n_few, 64u);
    const u64 key = lds->few[t], w = lds->few_weight[t];
    u64 before = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) before += lds->few[i] > key ? lds->few_weight[i] : 0ull;
    if (t < n && before < target && target <= before + w) lds->found = key;
  }
  __syncthreads();
  return lds->found;
}

// u of the total; u < 1 and total >= 2^s: the product stays below the total.
__device__ __forceinline__ u64 sample_target(const SampleRow& r, u64 total) {
  return min((u64)(r.u * (double)total), total - 1);
}
__device__ __forceinline__ void sample_out(const SampleArgs& a, uint32_t row, const SampleScale& scale, float l, uint32_t token, u64 total) {
  a.tokens[row] = (int32_t)token;
  if (a.logprobs) a.logprobs[row] = (float)(scale.log_mass(l) - log(__builtin_ldexp((double)total, -a.up)));
}

__global__ __launch_bounds__(kPickThreads) void k_sample_pick(SampleArgs a) {
  constexpr uint32_t kStep = 256, kScan = 8;  // of the last part
  __shared__ alignas(16) u64 keys[kPickThreads];
  __shared__ u64 masses[kPickThreads];
  __shared__ u64 scan[kPickThreads / 64][kScan][64];
  __shared__ u64 lds[kPickThreads / 64];
  __shared__ SampleBorderLds border_lds;
  __shared__ SelectLds select_lds;
  __shared__ u64 kept_of[kSampleSlices];
  __shared__ uint32_t the_one;
  __shared__ u64 the_rest;
  const uint32_t t = threadIdx.x, row = blockIdx.x;
  const SampleRow r = sample_row(a, row);
  SampleList list;
  list.list = a.list + (uint64_t)row * a.vocab;
  list.n = a.count[(uint64_t)row * kCountStride + kSampleBins];
  const u64 kept_own = t < a.slices ? a.kept[(uint64_t)row * a.slices + t] : 0ull;
  list.keys[0] = t < a.vocab ? list.list[t] : 0ull;  // if it is one
  SampleShare<kPickThreads> share;
  share.load(a, row);
  const u64 top = block_max<kPickThreads>(slice_top(a, row), lds);
  if (!r.good || !top || r.greedy) {
    if (t == 0) {
      if (!r.good) *a.err = 2u;
      const bool any = r.good && top;
      a.tokens[row] = any ? (int32_t)key_token(top) : -1;
      if (a.logprobs) a.logprobs[row] = any ? 0.f : __builtin_nanf("");
    }
    return;
  }
  const SampleScale scale(a, r, (uint32_t)(top >> 32));
  u64 thr = 0;  // keys from it on are kept
  if (t < a.slices) kept_of[t] = kept_own;
  const SampleBorder b = sample_border<kPickThreads>(r, scale, &border_lds, share);
  if (b.certain() == kNoBin) list.n = 0;
  list.hold(scale);
  SamplePlaces s;
  s.thr = 0;
  s.max = scale.top;
  s.token_bits = a.vocab > 1 ? 32 - __builtin_clz(a.vocab - 1) : 0;
  // Of more keys than are sorted: top-k's last (of all where all of top-k are
  // listed), then top-p's.
  const bool border = b.small || b.k_bin != kNoBin || b.p_first != kNoBin;  // but min-p's
  bool by_k = b.small || b.k_bin != kNoBin;
  u64 own_k = 0;  // mass of top-k's bin that is kept
  const bool sort = b.small || list.n <= kSort;
#pragma unroll 1
  for (bool more = border && (!sort || list.n > kPickThreads); more;) {
    u64 target = b.small ? r.k : r.k - b.k_before;
    s.bin = b.small ? kNoBin : b.k_bin;
    s.end = b.k_bin;
    if (!by_k) {
      target = share_of(r.top_p, b.k_mass + own_k);
      u64 w = share.before;
#pragma unroll
      for (uint32_t j = 0; j < kPickBins; ++j) {
        const uint32_t bin = kPickBins * t + j;
        const u64 mass = bin == b.k_bin ? own_k : share.m[j];
        if (w < target && target <= w + mass) {
          the_one = bin;
          the_rest = target - w;
        }
        w += mass;
      }
      __syncthreads();
      s.bin = s.end = the_one;
      target = the_rest;
    }
    thr = sample_select(list, s, scale, target, !by_k, &select_lds);
    more = by_k && r.by_mass() && !b.small;
    if (by_k && b.small) {
      // The k largest alone.
      if (t == 0) the_one = 0;
      __syncthreads();
      list.each(scale, [&](u64 key, u64) {
        if (key >= thr) keys[atomicAdd(&the_one, 1u)] = key;
      });
      __syncthreads();
      list.n = r.k;
      list.keys[0] = t < list.n ? keys[t] : 0ull;
      bool kept;
      list.masses[0] = scale.mass(SampleList::logit(list.keys[0]), &kept);
    } else if (more) {
      s.thr = thr;
      u64 sum = 0;
      list.each(scale, [&](u64 key, u64 mass) { sum += s.in(key) ? mass : 0ull; });
      own_k = block_sum<kPickThreads>(sum, lds);
    }
    by_k = false;
  }
  if (border && sort) {
    // Few keys: sorted by counting the larger ones, which puts the bins in order
    // and top-k's last.
    const u64 key = t < list.n ? list.keys[0] : 0ull;
    __syncthreads();
    keys[t] = key;
    __syncthreads();
    uint32_t rank = 0;
    if ((t & ~63u) < list.n) {
#pragma unroll 4
      for (uint32_t i = 0; i < list.n; i += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + i);
        rank += (two.x > key) + (two.y > key);
      }
    }
    __syncthreads();
    if (t < list.n) {
      keys[rank] = key;
      masses[rank] = list.masses[0];
    }
    __syncthreads();
    const u64 mine = t < list.n ? keys[t] : 0ull, here = t < list.n ? masses[t] : 0ull;
    const uint32_t bin = t < list.n ? sample_bin(scale.top, SampleList::logit(mine)) : kNoBin;
    // Keys from `last` on are not top-k's.
    const uint32_t k_from = b.small ? 0u : (uint32_t)block_sum<kPickThreads>(bin < b.k_bin, lds);
    uint32_t last = b.small ? min(r.k, list.n) : b.k_bin != kNoBin ? k_from + (r.k - b.k_before) : list.n;
    const bool in_k = t < last && t >= k_from && (b.small || b.k_bin != kNoBin);
    u64 sums[2] = {b.small || (bin >= b.p_first && bin <= b.p_last) ? here : 0ull, in_k ? here : 0ull}, all[2];
    block_before<kPickThreads, 2>(sums, all, border_lds.part);
    if (r.by_mass()) {
      // Kept: with less mass before it than top-p asks for.
      const u64 target = share_of(r.top_p, (b.small ? 0ull : b.k_mass) + all[1]);
      const bool under = (b.small ? 0ull : b.p_before) + sums[0] < target;
      const bool kept = t < last && (b.small ? under : bin < b.p_first || (bin <= b.p_last && under));
      last = (uint32_t)block_sum<kPickThreads>(kept, lds);
    }
    thr = keys[last - 1];  // the first key of top-k's or top-p's bin is kept
    if (b.small) {
      // All that may be kept is here: the token by the masses of lower tokens.
      bool kept;
      if (r.min_p > 0.0) scale.mass(SampleList::logit(mine), &kept);
      const u64 w = t < last && (r.min_p <= 0.0 || kept) ? here : 0ull;
      masses[t] = w;
      __syncthreads();
      u64 before = 0, total = 0;
#pragma unroll 4
      for (uint32_t i = 0; i < last; ++i) {
        const u64 m = masses[i];
        total += m;
        before += key_token(keys[i]) < key_token(mine) ? m : 0ull;
      }
      const u64 target = sample_target(r, total);
      if (before <= target && target < before + w) sample_out(a, row, scale, SampleList::logit(mine), key_token(mine), total);
      return;
    }
  }
  // Every slice's kept mass: what is certain, and what of the list is kept. (The
  // slice and the rest are numbers whatever happens: logits that another stream
  // writes meanwhile give a wrong token, not a read outside of the row.)
  if (t == 0) the_one = 0, the_rest = 0;
  __syncthreads();
  list.each(scale, [&](u64 key, u64 mass) {
    bool kept = true;
    if (key >= thr && scale.least > 0.0) scale.mass(SampleList::logit(key), &kept);  // min-p
    if (key >= thr && kept && mass) atomicAdd(&kept_of[key_token(key) / a.slice], mass);
  });
  __syncthreads();
  const u64 own = t < a.slices ? kept_of[t] : 0ull;
  u64 total;
  u64 before = block_before<kPickThreads>(own, &total, lds);
  u64 target = sample_target(r, total);
  if (before <= target && target < before + own) {
    the_one = t;
    the_rest = target - before;
  }
  __syncthreads();
  const uint32_t slice = the_one;
  target = the_rest;
  // Each wave has a stretch of the slice, 256 tokens a step; then the wave in
  // whose stretch the sum passes u looks for the step and the token. The masses
  // of the first steps stay in LDS.
  const float* const l = a.logits + (uint64_t)row * a.vocab;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const uint32_t stretch = (a.slice / (kPickThreads / 64) + kStep - 1) / kStep * kStep;
  const uint32_t begin = slice * a.slice, from = begin + min(a.slice, wave * stretch);
  const uint32_t to = min(min(a.vocab, begin + a.slice), from + stretch);
  // Kept masses of this lane's four tokens from i on.
  auto masses_at = [&](f32x4 v, uint32_t i, u64 (&m)[4]) {
    bool in[4], any = false;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) any |= in[j] = i + j < to && sample_key(v[j], i + j) >= thr;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) m[j] = 0;
    if (!__any(any)) return;
    scale.masses(v, m, true);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) m[j] = in[j] ? m[j] : 0ull;
  };
  u64 sum = 0;
  f32x4 next = sample_load(l, from + lane * 4, a.vocab);
#pragma unroll 1
  for (uint32_t i = from, step = 0; i < to; i += kStep, ++step) {
    const f32x4 v = next;
    next = sample_load(l, i + kStep + lane * 4, a.vocab);
    u64 m[4];
    masses_at(v, i + lane * 4, m);
    const u64 own4 = m[0] + m[1] + m[2] + m[3];
    if (step < kScan) scan[wave][step][lane] = own4;
    sum += own4;
  }
  sum = wave_scan_u64(sum);
  if (lane == 63) lds[wave] = sum;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) {
    const u64 m = lds[w];
    if (target < m) return;  // another wave's
    target -= m;
  }
  if (target >= lds[wave]) return;
#pragma unroll 1
  for (uint32_t i = from, step = 0; i < to; i += kStep, ++step) {
    const f32x4 v = sample_load(l, i + lane * 4, a.vocab);
    u64 m[4], own4;
    if (step < kScan) {
      own4 = scan[wave][step][lane];
    } else {
      masses_at(v, i + lane * 4, m);
      own4 = m[0] + m[1] + m[2] + m[3];
    }
    const u64 upto = wave_scan_u64(own4), here = __ballot(target < upto);
    if (!here) {
      target -= (u64)(uint32_t)__builtin_amdgcn_readlane((int)(upto >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
      continue;
    }
    masses_at(v, i + lane * 4, m);
    if (lane == (uint32_t)__builtin_ctzll(here)) {
      u64 before4 = upto - own4;
      float l_at = 0.f;
      uint32_t token = 0;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        if (target >= before4 && target < before4 + m[j]) l_at = v[j], token = i + lane * 4 + j;
        before4 += m[j];
      }
      sample_out(a, row, scale, l_at, token, total);
    }
    return;
  }
}

// Slices of whole thousands (of 1024), for about a thousand blocks in all but
// not above five each: longer ones leave the pick much to go through alone and
// the CUs with blocks that end far apart (10 thousands: 64 rows of 151936 62 us
// instead of 54; 38: 256 rows 209 instead of 124), shorter ones are mostly
// prologue (one thousand instead of two: 64 rows of 32000 37 us instead of 34;
// two instead of five: 64 rows of 151936 61).
static void sample_slices(uint32_t n, uint32_t vocab, uint32_t* slice, uint32_t* slices) {
  const uint32_t want = n >= 1024 ? 1 : min(kSampleSlices, 1024 / n), most = max(5u, (vocab + kSampleSlices * 1024 - 1) / (kSampleSlices * 1024));
  *slice = min(most, ((vocab + want - 1) / want + 1023) / 1024) * 1024;
  *slices = (vocab + *slice - 1) / *slice;
}

uint64_t sample_workspace(uint32_t n, uint32_t vocab, SampleArgs* a, uint8_t* base) {
  uint32_t slice, slices;
  sample_slices(n, vocab, &slice, &slices);
  auto al = [](uint64_t b) { return (b + 255) & ~(uint64_t)255; };
  const uint64_t rows = n, tops = al(rows * slices * 8), mass = al(rows * kSampleBins * 8);
  const uint64_t count = al(rows * kCountStride * 4), list = al(rows * vocab * 8);
  const uint64_t slice_mass = rows * slices * kSampleBins * 8;
  if (a) {
    uint32_t bits = 0;
    while (((uint64_t)1 << bits) < vocab) ++bits;
    a->slice = slice;
    a->slices = slices;
    a->up = bits < 11 ? 51 : 62 - (int)bits;
    a->tops = (u64*)base;
    a->kept = (u64*)(base + tops);
    a->mass = (u64*)(base + 2 * tops);
    a->list = (u64*)(base + 2 * tops + mass);
    a->count = (uint32_t*)(base + 2 * tops + mass + list);
    a->slice_mass = (u64*)(base + 2 * tops + mass + list + count);
  }
  return 2 * tops + mass + list + count + slice_mass;
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(a.n * a.slices), block(kSampleThreads);
  hipLaunchKernelGGL(k_sample_top, grid, block, 0, st, a);
  hipLaunchKernelGGL(k_sample_bins, grid, block, 0, st, a);
  hipLaunchKernelGGL(k_sample_list, grid, block, 0, st, a);
  hipLaunchKernelGGL(k_sample_pick, dim3(a.n), dim3(kPickThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace smoe

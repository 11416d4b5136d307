// sample.hip — one token per row of logits, drawn from the filtered
// distribution.
//
//   k_sample_top   a slice's largest key; clears the row's sums
//   k_sample_bins  the row's logits by their distance from its largest: counts
//                  and masses per bin (rows with top-k or top-p)
//   k_sample_list  the keys of the bins in which a border lies, and each slice's
//                  mass of what is kept for certain
//   k_sample_pick  the borders themselves, the sum, and the token
//
// A logit becomes 32 bits in an order that integers compare, and a key with the
// complement of its token below it, so keys are unique and the order of the
// filters is that of falling keys. Its distance from the row's largest is an
// integer too; bins are 32 to every power of two of it, so that they are finest
// where the mass is. All three filters keep a first part of the order: what
// decides is one key, and only the bins around it have to be looked into.
//
// A mass e^((logit - max) / T) is f64 and then an integer of 2^-s: sums of
// integers are the same in any order, so atomics may form them.
#include "common.h"
#include "kernels.h"

namespace smoe {

typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kSampleThreads = 256;
constexpr uint32_t kSampleSlices = 128;  // of a row at most
constexpr uint32_t kCountStride = kSampleBins + 4;
constexpr uint32_t kNoBin = kSampleBins;

// Bin of a distance: itself below 32, else 32 to a power of two.
__device__ __forceinline__ uint32_t sample_bin(uint32_t d) {
  if (d < 32) return d;
  const uint32_t e = 31 - __builtin_clz(d);
  return (e - 4) * 32 + ((d >> (e - 5)) & 31);
}
// First distance of a bin, and the binary digits that its distances differ in.
__device__ __forceinline__ void sample_bin_range(uint32_t bin, uint32_t* first, uint32_t* bits) {
  if (bin < 32) {
    *first = bin;
    *bits = 0;
    return;
  }
  *bits = bin / 32 - 1;
  *first = (32 + bin % 32) << *bits;
}

// e^x for -46 <= x <= 0: x = n ln 2 + r, the series of e^r to r^11 (what is left
// out is below 2^-47 of it).
__device__ __forceinline__ double sample_exp(double x) {
  const double n = __builtin_rint(x * 1.4426950408889634), r = __builtin_fma(n, -0.6931471805599453, x);
  double e = 1.0 / 39916800;
  constexpr double c[11] = {1, 1, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800};
#pragma unroll
  for (int i = 10; i >= 0; --i) e = __builtin_fma(e, r, c[i]);
  return __builtin_ldexp(e, (int)n);
}

struct SampleRow {
  bool good, greedy;
  uint32_t k;              // kept at most; 0: all
  double inv_t, top_p, min_p, u;
  __device__ bool by_mass() const { return top_p < 1.0; }
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
  uint32_t top;       // its order
  double max, inv_t, unit, least, min_p;
  bool infinite;
  __device__ SampleScale(const SampleArgs& a, const SampleRow& r, uint32_t o)
      : top(o), max(ord_float(o)), inv_t(r.inv_t), unit(a.unit), min_p(r.min_p), infinite(o == 0xFF800000u) {
    // Below it a mass rounds to zero.
    least = -0.6931471805599453 * (2 + __builtin_amdgcn_frexp_exp(a.unit));
  }
  __device__ double log_mass(float l) const {
    if (infinite) return l == INFINITY ? 0.0 : -INFINITY;
    return ((double)l - max) * inv_t;
  }
  // The mass as an integer; *kept: whether min_p keeps it.
  __device__ u64 mass(float l, bool* kept) const {
    const double x = log_mass(l);
    const double e = x > least ? sample_exp(x) : 0.0;
    *kept = e >= min_p;
    return (u64)__builtin_rint(e * unit);
  }
};

__device__ __forceinline__ u64 sample_key(float l, uint32_t token) { return (u64)float_ord(l) << 32 | (uint32_t)~token; }
__device__ __forceinline__ uint32_t key_token(u64 key) { return ~(uint32_t)key; }

// Over the block's 256 threads; lds: 4 of T. Every thread gets the result.
__device__ __forceinline__ u64 block_max(u64 v, u64* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (u64)__shfl_xor(v, o, kWave));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}
// Sum of the threads before this one; *all: of all.
__device__ __forceinline__ u64 block_before(u64 v, u64* all, u64* lds) {
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(s, o, kWave);
    if ((threadIdx.x & 63) >= (uint32_t)o) s += w;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  u64 skip = 0;
  *all = 0;
#pragma unroll
  for (uint32_t w = 0; w < 4; ++w) {
    if (w < threadIdx.x >> 6) skip += lds[w];
    *all += lds[w];
  }
  return skip + s - v;
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

__device__ __forceinline__ u64 row_top(const SampleArgs& a, uint32_t row, u64* lds) {
  return block_max(threadIdx.x < a.slices ? a.tops[row * a.slices + threadIdx.x] : 0ull, lds);
}

__global__ __launch_bounds__(kSampleThreads) void k_sample_top(SampleArgs a) {
  __shared__ u64 lds[4];
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const float* const l = a.logits + (uint64_t)row * a.vocab;
  u64 top = 0;
  const uint32_t from = slice * a.slice, to = min(a.vocab, from + a.slice);
  for (uint32_t i = from + t * 4; i < to; i += kSampleThreads * 4) {
    const f32x4 v = sample_load(l, i, a.vocab);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const u64 key = sample_key(v[j], i + j);
      if (v[j] > -INFINITY && key > top) top = key;
    }
  }
  top = block_max(top, lds);
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
  if (!r.good || r.greedy || !(r.k || r.by_mass())) return;
  const u64 top = row_top(a, row, lds);
  if (!top) return;
  for (uint32_t i = t; i < kSampleBins; i += kSampleThreads) mass[i] = 0, count[i] = 0;
  __syncthreads();
  const SampleScale scale(a, r, (uint32_t)(top >> 32));
  const float* const l = a.logits + (uint64_t)row * a.vocab;
  const uint32_t from = slice * a.slice, to = min(a.vocab, from + a.slice);
  for (uint32_t i = from + t * 4; i < to; i += kSampleThreads * 4) {
    const f32x4 v = sample_load(l, i, a.vocab);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (!(v[j] > -INFINITY)) continue;
      const uint32_t bin = sample_bin(scale.top - float_ord(v[j]));
      atomicAdd(&count[bin], 1u);
      if (r.by_mass()) {
        bool kept;
        const u64 m = scale.mass(v[j], &kept);
        if (m) atomicAdd(&mass[bin], m);
      }
    }
  }
  __syncthreads();
  for (uint32_t i = t; i < kSampleBins; i += kSampleThreads) {
    if (!count[i]) continue;
    atomicAdd(a.count + (uint64_t)row * kCountStride + i, count[i]);
    if (mass[i]) atomicAdd(a.mass + (uint64_t)row * kSampleBins + i, mass[i]);
  }
}

// The bins in which the borders lie (kNoBin: there is none).
struct SampleBorder {
  uint32_t k_bin, k_before;     // top-k's, and tokens before it
  u64 k_mass;                   // mass before it, or of all
  uint32_t p_first, p_last;     // top-p's is one of these
  __device__ bool certain(uint32_t bin) const { return bin < min(k_bin, p_first); }
  __device__ bool listed(uint32_t bin) const { return bin == k_bin || (bin >= p_first && bin <= p_last); }
};
struct SampleBorderLds {
  u64 part[4];
  SampleBorder b;
  u64 k_own;
};
__device__ __forceinline__ u64 share_of(double p, u64 of) {  // at least one
  const double v = __builtin_ceil(p * (double)of);
  return v >= 1.0 ? (u64)v : 1ull;
}
// Thread t has bins 4 t .. 4 t + 3; before: mass ahead of its first, m: of each.
__device__ __forceinline__ SampleBorder sample_border(const SampleArgs& a, const SampleRow& r, uint32_t row,
                                                      SampleBorderLds* lds, u64* before, u64 (&m)[4]) {
  const uint32_t t = threadIdx.x;
  uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) m[j] = 0;
  if (4 * t < kSampleBins) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = a.count[(uint64_t)row * kCountStride + 4 * t + j];
      m[j] = a.mass[(uint64_t)row * kSampleBins + 4 * t + j];
    }
  }
  u64 all, all_count;
  u64 n = block_before((u64)c[0] + c[1] + c[2] + c[3], &all_count, lds->part);
  *before = block_before(m[0] + m[1] + m[2] + m[3], &all, lds->part);
  if (t == 0) {
    lds->b = SampleBorder{kNoBin, 0, all, kNoBin, kNoBin};
    lds->k_own = 0;
  }
  __syncthreads();
  if (r.k) {
    u64 w = *before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n < r.k && r.k <= n + c[j]) {
        lds->b.k_bin = 4 * t + j;
        lds->b.k_before = (uint32_t)n;
        lds->b.k_mass = w;
        lds->k_own = m[j];
      }
      n += c[j];
      w += m[j];
    }
    __syncthreads();
  }
  if (r.by_mass()) {
    const u64 lo = share_of(r.top_p, lds->b.k_mass), hi = share_of(r.top_p, lds->b.k_mass + lds->k_own);
    u64 w = *before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (w < lo && lo <= w + m[j]) lds->b.p_first = 4 * t + j;
      if (w < hi && hi <= w + m[j]) lds->b.p_last = 4 * t + j;
      w += m[j];
    }
  }
  __syncthreads();
  return lds->b;
}

__global__ __launch_bounds__(kSampleThreads) void k_sample_list(SampleArgs a) {
  __shared__ u64 lds[4];
  __shared__ SampleBorderLds border_lds;
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const SampleRow r = sample_row(a, row);
  if (!r.good || r.greedy) return;
  const u64 top = row_top(a, row, lds);
  if (!top) return;
  const SampleScale scale(a, r, (uint32_t)(top >> 32));
  SampleBorder b = {kNoBin, 0, 0, kNoBin, kNoBin};
  if (r.k || r.by_mass()) {
    u64 before, m[4];
    b = sample_border(a, r, row, &border_lds, &before, m);
  }
  const float* const l = a.logits + (uint64_t)row * a.vocab;
  const uint32_t from = slice * a.slice, to = min(a.vocab, from + a.slice);
  u64 sum = 0;
  for (uint32_t i = from + t * 4; i < to; i += kSampleThreads * 4) {
    const f32x4 v = sample_load(l, i, a.vocab);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (!(v[j] > -INFINITY)) continue;
      const uint32_t bin = sample_bin(scale.top - float_ord(v[j]));
      if (b.certain(bin)) {
        bool kept;
        const u64 m = scale.mass(v[j], &kept);
        if (kept) sum += m;
      } else if (b.listed(bin)) {
        const uint32_t at = atomicAdd(a.count + (uint64_t)row * kCountStride + kSampleBins, 1u);
        a.list[(uint64_t)row * a.vocab + at] = sample_key(v[j], i + j);
      }
    }
  }
  u64 all;
  block_before(sum, &all, lds);
  if (t == 0) a.kept[blockIdx.x] = all;
}

// The list's entries of one bin, in order; a place is distance and token in one
// number, the first of the order the smallest.
struct SamplePlaces {
  u64 thr;        // only keys from it on
  uint32_t bin, top, first, bits, token_bits;
  __device__ bool place(u64 key, u64* p) const {
    const uint32_t d = top - (uint32_t)(key >> 32);
    if (key < thr || sample_bin(d) != bin) return false;
    *p = (u64)(d - first) << token_bits | key_token(key);
    return true;
  }
  __device__ u64 key(u64 p) const {
    const uint32_t d = first + (uint32_t)(p >> token_bits), token = (uint32_t)(p & ((1ull << token_bits) - 1));
    return (u64)(top - d) << 32 | (uint32_t)~token;
  }
};

constexpr uint32_t kDigit = 10;
struct SelectLds {
  u64 weight[1u << kDigit];
  uint32_t count[1u << kDigit];
  u64 part[4];
  u64 prefix, rest, found;
  uint32_t left;
};
// Key of the first place up to which the weights (masses, or 1 each) add up to
// `target` or more, digit after digit of the places from the top; there is one.
template <bool MASS>
__device__ u64 sample_select(const u64* list, uint32_t n, const SamplePlaces& s, const SampleScale& scale, u64 target,
                             SelectLds* lds) {
  const uint32_t t = threadIdx.x;
  int shift = (int)(s.bits + s.token_bits);
  u64 prefix = 0;  // the digits above shift
  for (;;) {
    const int width = min(shift, (int)kDigit);
    shift -= width;
    for (uint32_t i = t; i < 1u << kDigit; i += kSampleThreads) lds->weight[i] = 0, lds->count[i] = 0;
    __syncthreads();
    for (uint32_t i = t; i < n; i += kSampleThreads) {
      u64 p;
      if (!s.place(list[i], &p) || p >> (shift + width) != prefix) continue;
      const uint32_t digit = (uint32_t)(p >> shift) & ((1u << width) - 1);
      atomicAdd(&lds->count[digit], 1u);
      if constexpr (MASS) {
        bool kept;
        atomicAdd(&lds->weight[digit], scale.mass(ord_float((uint32_t)(list[i] >> 32)), &kept));
      }
    }
    __syncthreads();
    u64 w[4], all, sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += w[j] = MASS ? lds->weight[4 * t + j] : lds->count[4 * t + j];
    u64 before = block_before(sum, &all, lds->part);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (before < target && target <= before + w[j]) {
        lds->prefix = prefix << width | (4 * t + j);
        lds->rest = target - before;
        lds->left = lds->count[4 * t + j];
      }
      before += w[j];
    }
    __syncthreads();
    prefix = lds->prefix;
    target = lds->rest;
    if (shift == 0) return s.key(prefix);
    if (lds->left == 1) break;
    __syncthreads();
  }
  // One place has these digits.
  for (uint32_t i = t; i < n; i += kSampleThreads) {
    u64 p;
    if (s.place(list[i], &p) && p >> shift == prefix) lds->found = list[i];
  }
  __syncthreads();
  return lds->found;
}

__global__ __launch_bounds__(kSampleThreads) void k_sample_pick(SampleArgs a) {
  __shared__ u64 lds[4];
  __shared__ SampleBorderLds border_lds;
  __shared__ SelectLds select_lds;
  __shared__ u64 kept_of[kSampleSlices];
  __shared__ uint32_t the_slice;
  __shared__ u64 the_rest;
  const uint32_t t = threadIdx.x, row = blockIdx.x;
  const SampleRow r = sample_row(a, row);
  const u64 top = row_top(a, row, lds);
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
  const u64* const list = a.list + (uint64_t)row * a.vocab;
  uint32_t n = 0;
  if (r.k || r.by_mass()) {
    u64 before, m[4];
    const SampleBorder b = sample_border(a, r, row, &border_lds, &before, m);
    n = a.count[(uint64_t)row * kCountStride + kSampleBins];
    SamplePlaces s;
    s.thr = 0;
    s.top = scale.top;
    s.token_bits = a.vocab > 1 ? 32 - __builtin_clz(a.vocab - 1) : 0;
    u64 own = 0;  // mass of top-k's bin that is kept
    if (b.k_bin != kNoBin) {
      s.bin = b.k_bin;
      sample_bin_range(s.bin, &s.first, &s.bits);
      thr = s.thr = sample_select<false>(list, n, s, scale, r.k - b.k_before, &select_lds);
      if (r.by_mass()) {
        u64 sum = 0;
        for (uint32_t i = t; i < n; i += kSampleThreads) {
          u64 p;
          bool kept;
          if (s.place(list[i], &p)) sum += scale.mass(ord_float((uint32_t)(list[i] >> 32)), &kept);
        }
        block_before(sum, &own, lds);
      }
    }
    if (r.by_mass()) {
      const u64 target = share_of(r.top_p, b.k_mass + own);
      u64 w = before;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 mass = 4 * t + j == b.k_bin ? own : m[j];
        if (w < target && target <= w + mass) {
          the_slice = 4 * t + j;
          the_rest = target - w;
        }
        w += mass;
      }
      __syncthreads();
      s.bin = the_slice;
      sample_bin_range(s.bin, &s.first, &s.bits);
      thr = sample_select<true>(list, n, s, scale, the_rest, &select_lds);
    }
  }
  // Every slice's kept mass: what is certain, and what of the list is kept.
  if (t < a.slices) kept_of[t] = a.kept[(uint64_t)row * a.slices + t];
  __syncthreads();
  for (uint32_t i = t; i < n; i += kSampleThreads) {
    const u64 key = list[i];
    bool kept;
    const u64 m = scale.mass(ord_float((uint32_t)(key >> 32)), &kept);
    if (key >= thr && kept && m) atomicAdd(&kept_of[key_token(key) / a.slice], m);
  }
  __syncthreads();
  const u64 own = t < a.slices ? kept_of[t] : 0ull;
  u64 total;
  u64 before = block_before(own, &total, lds);
  // u < 1 and total >= 2^s: the product stays below the total.
  u64 target = (u64)(r.u * (double)total);
  target = min(target, total - 1);
  if (before <= target && target < before + own) {
    the_slice = t;
    the_rest = target - before;
  }
  __syncthreads();
  const uint32_t slice = the_slice;
  target = the_rest;
  const float* const l = a.logits + (uint64_t)row * a.vocab;
  const uint32_t run = a.slice / kSampleThreads, from = slice * a.slice + t * run;
  auto mass_at = [&](float v, uint32_t token) -> u64 {
    if (!(v > -INFINITY) || sample_key(v, token) < thr) return 0;
    bool kept;
    const u64 m = scale.mass(v, &kept);
    return kept ? m : 0ull;
  };
  u64 sum = 0;
  for (uint32_t i = from; i < min(a.vocab, from + run); i += 4) {
    const f32x4 v = sample_load(l, i, a.vocab);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) sum += mass_at(v[j], i + j);
  }
  u64 all;
  before = block_before(sum, &all, lds);
  if (before <= target && target < before + sum) {
    for (uint32_t i = from;; ++i) {
      const u64 m = mass_at(l[i], i);
      if (target < before + m) {
        a.tokens[row] = (int32_t)i;
        if (a.logprobs) a.logprobs[row] = (float)(scale.log_mass(l[i]) - log((double)total / a.unit));
        break;
      }
      before += m;
    }
  }
}

// Slices of whole thousands, about a thousand blocks in all.
static void sample_slices(uint32_t n, uint32_t vocab, uint32_t* slice, uint32_t* slices) {
  const uint32_t want = n >= 1024 ? 1 : n * kSampleSlices <= 1024 ? kSampleSlices : 1024 / n;
  *slice = ((vocab + want - 1) / want + 1023) / 1024 * 1024;
  *slices = (vocab + *slice - 1) / *slice;
}

uint64_t sample_workspace(uint32_t n, uint32_t vocab, SampleArgs* a, uint8_t* base) {
  uint32_t slice, slices;
  sample_slices(n, vocab, &slice, &slices);
  auto al = [](uint64_t b) { return (b + 255) & ~(uint64_t)255; };
  const uint64_t rows = n, tops = al(rows * slices * 8), mass = al(rows * kSampleBins * 8);
  const uint64_t count = al(rows * kCountStride * 4), list = al(rows * vocab * 8);
  if (a) {
    uint32_t bits = 0;
    while (((uint64_t)1 << bits) < vocab) ++bits;
    a->slice = slice;
    a->slices = slices;
    a->unit = (double)((uint64_t)1 << (62 - bits));
    a->tops = (u64*)base;
    a->kept = (u64*)(base + tops);
    a->mass = (u64*)(base + 2 * tops);
    a->list = (u64*)(base + 2 * tops + mass);
    a->count = (uint32_t*)(base + 2 * tops + mass + list);
  }
  return 2 * tops + mass + list + count;
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(a.n * a.slices), block(kSampleThreads);
  hipLaunchKernelGGL(k_sample_top, grid, block, 0, st, a);
  if (a.top_k || a.top_p) hipLaunchKernelGGL(k_sample_bins, grid, block, 0, st, a);
  hipLaunchKernelGGL(k_sample_list, grid, block, 0, st, a);
  hipLaunchKernelGGL(k_sample_pick, dim3(a.n), block, 0, st, a);
  return hipGetLastError();
}

}  // namespace smoe

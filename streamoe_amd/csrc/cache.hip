// cache.hip — rows into and out of a paged key / value cache.
//
//   k_kv_append  cache row (seq, pos, head) = k or v of a token: bf16 to nearest
//                even; 8 bits: scale = max |x| / 127, code = rint(x / scale)
//   k_kv_gather  the other way round, code * scale in f32
//
// Both move rows of head_dim values between places that a table gives: bytes
// bound many rows (gathered prefixes of four requests, 8 key heads of 128 out of
// 8 bits into bf16, 80 MB: 17 us, 4.6 TB/s of a large copy's 5.0), the chain seq
// and pos -> table -> row a few (100 tokens of 2 heads of 256 gathered 2.9 us, one
// appended 1.8, a thousand of 2 heads of 256 to 8 bits 4.8).
#include <type_traits>

#include "kv.h"

namespace smoe {

typedef __bf16 kbf16x8 __attribute__((ext_vector_type(8)));
typedef float kf32x8 __attribute__((ext_vector_type(8), aligned(16)));
typedef int32_t ki32x4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kKvThreads = 256;
constexpr uint32_t kKvPerBlock = 8;  // tokens of an append's block at most
static_assert(kKvMaxTokens <= 2048 * kKvPerBlock, "two thousand blocks");

__device__ __forceinline__ uint64_t kv_row(const KvView& c, uint32_t page, uint32_t head, uint32_t slot) {
  return page * c.page + head * c.head + slot * c.slot;
}
__device__ __forceinline__ uint64_t kv_scale(const KvView& c, uint32_t page, uint32_t head, uint32_t slot) {
  return ((uint64_t)page * c.heads + head) * c.page_size + slot;
}

// A block has up to 8 tokens (per_block) with all of their rows: a key and a
// value row per head, 2^lanes_log lanes each, eight values per lane. Of tokens
// with the same sequence and position the last is written: the block looks for
// its own among all behind them, 8 bytes each out of L2 (16384 tokens: 64 KB a
// block on average, beside 32 KB or more of rows), sixteen of a thread on their
// way at once where there are so many, and compares only those between the least
// and the greatest of its own, which are few of a prompt's or a batch's (16384
// tokens of 64 sequences, 2 heads of 256 in bf16, 67 MB: 20 us; all compared 86).
template <bool XBF16, bool I8>
__global__ __launch_bounds__(kKvThreads) void k_kv_append(KvRowsArgs a) {
  __shared__ int32_t seqs[kKvPerBlock], poss[kKvPerBlock];
  __shared__ uint32_t dead[kKvPerBlock], ids[kKvPerBlock];
  const uint32_t t = threadIdx.x, first = blockIdx.x * a.per_block, n = a.t.n;
  const uint32_t mine = min(a.per_block, n - first);
  bool in = false;
  uint32_t id = 0;
  if (t < mine) {
    const int32_t s = a.t.seq[first + t], p = a.t.pos[first + t];
    bool wrong;
    in = kv_token(a.t, s, p, &wrong);
    if (wrong) *a.err = 2u;
    seqs[t] = s;
    poss[t] = p;
    dead[t] = !in;
    if (in) id = (uint32_t)a.t.table[(uint64_t)s * a.t.width + kv_page_of(a.c, (uint32_t)p >> 4)];
  }
  __syncthreads();
  if (first + 1 < n) {
    int32_t s0 = 0x7FFFFFFF, s1 = -1, p0 = 0x7FFFFFFF, p1 = -1;
    for (uint32_t i = 0; i < mine; ++i) {
      if (dead[i]) continue;
      s0 = min(s0, seqs[i]), s1 = max(s1, seqs[i]);
      p0 = min(p0, poss[i]), p1 = max(p1, poss[i]);
    }
    __syncthreads();
    const auto look = [&](uint32_t j, int32_t s, int32_t p) {
      if (s < s0 || s > s1 || p < p0 || p > p1) return;
      for (uint32_t i = 0; i < mine; ++i)
        if (first + i < j && seqs[i] == s && poss[i] == p) dead[i] = 1;
    };
    if (n < 4) {
      for (uint32_t j = first + 1; j < n; ++j) look(j, a.t.seq[j], a.t.pos[j]);
    } else {
      const auto some = [&](uint32_t j, auto count) {
        constexpr uint32_t B = decltype(count)::value;
        ki32x4 s[B], p[B];
#pragma unroll
        for (uint32_t b = 0; b < B; ++b) {  // the last four for those behind the end
          const uint32_t at = min(j + b * 4 * kKvThreads, n - 4);
          s[b] = *reinterpret_cast<const ki32x4*>(a.t.seq + at);
          p[b] = *reinterpret_cast<const ki32x4*>(a.t.pos + at);
        }
#pragma unroll
        for (uint32_t b = 0; b < B; ++b) {
          const uint32_t at = min(j + b * 4 * kKvThreads, n - 4);
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) look(at + e, s[b][e], p[b][e]);
        }
      };
      uint32_t j = first + 1 + 4 * t;
      if (n - first > 4 * kKvThreads) {
        for (; j < n; j += 16 * kKvThreads) some(j, std::integral_constant<uint32_t, 4>{});
      } else if (j < n) {
        some(j, std::integral_constant<uint32_t, 1>{});
      }
    }
  }
  if (t < mine) {
    if (in && id >= a.c.n_pages) {
      *a.err = 2u;
      dead[t] = 1;
    }
    ids[t] = id;
  }
  __syncthreads();
  const uint32_t lanes = 1u << a.lanes_log, lane = t & (lanes - 1), heads2 = 2 * a.c.heads;
  const uint32_t e = lane * 8;
  const bool has = e < a.c.dim;
  for (uint32_t r = t >> a.lanes_log; r < mine * heads2; r += kKvThreads >> a.lanes_log) {
    const uint32_t i = r / heads2, kv = r - i * heads2;
    if (dead[i]) continue;
    const bool is_v = kv >= a.c.heads;
    const uint32_t head = is_v ? kv - a.c.heads : kv;
    kf32x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (has) {
      const uint64_t at = (first + i) * a.stride + head * a.c.dim + e;
      const void* const src = is_v ? a.v : a.k;
      if constexpr (XBF16)
        x = __builtin_convertvector(*reinterpret_cast<const kbf16x8*>((const uint16_t*)src + at), kf32x8);
      else
        x = *reinterpret_cast<const kf32x8*>((const float*)src + at);
    }
    const uint32_t pos = (uint32_t)poss[i], id = ids[i];
    const uint32_t slot = pos - kv_page_of(a.c, pos >> 4) * a.c.page_size;
    uint8_t* const to = (is_v ? a.c.v : a.c.k) + kv_row(a.c, id, head, slot);
    if constexpr (!I8) {
      if (has) *reinterpret_cast<kbf16x8*>(to + 2 * e) = __builtin_convertvector(x, kbf16x8);
    } else {
      float top = 0.f, fin = 0.f;  // fin: 0 while all are finite, else NaN
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(x[j]));
        fin = __builtin_fmaf(x[j], 0.f, fin);
      }
      top = fin == 0.f ? top : INFINITY;
      for (uint32_t o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor(top, (int)o, kWave));
      const bool ok = top >= kQuantFloor && top < INFINITY;
      const float s = top < INFINITY ? (ok ? top / 127.f : 0.f) : __builtin_nanf("");
      int32_t c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = ok ? (int32_t)__builtin_rintf(x[j] / s) : 0;
      if (has)
        *reinterpret_cast<uint2*>(to + e) = uint2{pack_bytes(c[0], c[1], c[2], c[3]), pack_bytes(c[4], c[5], c[6], c[7])};
      if (lane == 0) (is_v ? a.c.vs : a.c.ks)[kv_scale(a.c, id, head, slot)] = s;
    }
  }
}

// One row per 2^lanes_log lanes, 16 bytes of the cache per lane (8 bf16 or 16
// codes).
template <bool OBF16, bool I8>
__global__ __launch_bounds__(kKvThreads) void k_kv_gather(KvRowsArgs a) {
  const uint32_t heads2 = 2 * a.c.heads;
  const uint32_t r = blockIdx.x * (kKvThreads >> a.lanes_log) + (threadIdx.x >> a.lanes_log);
  const uint32_t e = (threadIdx.x & ((1u << a.lanes_log) - 1)) * (I8 ? 16 : 8);
  const uint32_t i = r / heads2, kv = r - i * heads2;
  if (i >= a.t.n || e >= a.c.dim) return;
  const bool is_v = kv >= a.c.heads;
  const uint32_t head = is_v ? kv - a.c.heads : kv;
  const int32_t s = a.t.seq[i], p = a.t.pos[i];
  bool wrong;
  bool in = kv_token(a.t, s, p, &wrong);
  const uint32_t n = in ? kv_page_of(a.c, (uint32_t)p >> 4) : 0u;
  const int32_t id = in ? a.t.table[(uint64_t)s * a.t.width + n] : 0;
  if (in && (uint32_t)id >= a.c.n_pages) in = false, wrong = true;
  if (wrong) *a.err = 2u;
  const uint32_t slot = (uint32_t)p - n * a.c.page_size;
  const uint8_t* const from = (is_v ? a.c.v : a.c.k) + (in ? kv_row(a.c, id, head, slot) : 0);
  const uint64_t at = i * a.stride + head * a.c.dim + e;
  void* const out = is_v ? a.vo : a.ko;
  auto put = [&](kf32x8 x, uint64_t o) {
    if constexpr (OBF16)
      *reinterpret_cast<kbf16x8*>((uint16_t*)out + o) = __builtin_convertvector(x, kbf16x8);
    else
      *reinterpret_cast<kf32x8*>((float*)out + o) = x;
  };
  const kf32x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
  if constexpr (I8) {
    kf32x8 lo = zero, hi = zero;
    if (in) {
      const u32x4 c = *reinterpret_cast<const u32x4*>(from + e);
      const float sc = (is_v ? a.c.vs : a.c.ks)[kv_scale(a.c, id, head, slot)];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = (float)(int8_t)(c[j >> 2] >> (8 * (j & 3))) * sc;
        hi[j] = (float)(int8_t)(c[2 + (j >> 2)] >> (8 * (j & 3))) * sc;
      }
    }
    put(lo, at);
    put(hi, at + 8);
  } else {
    kf32x8 x = zero;
    if (in) x = __builtin_convertvector(*reinterpret_cast<const kbf16x8*>(from + 2 * e), kf32x8);
    put(x, at);
  }
}

static uint32_t lanes_log(uint32_t dim, uint32_t per) {
  uint32_t l = 0;
  while ((per << l) < dim) ++l;
  return l;
}

// Blocks of one token up to 2048 (more would search as long for fewer rows: 16384
// tokens of 4 30 us instead of 20, 4096 of one 9.4 instead of 7.1), two thousand beyond
// (one thousand: 23 and 7.3).
hipError_t launch_kv_append(KvRowsArgs a, bool x_bf16, bool i8, hipStream_t st) {
  a.lanes_log = lanes_log(a.c.dim, 8);
  a.per_block = (a.t.n + 2047) / 2048;
  const auto fn = x_bf16 ? (i8 ? k_kv_append<true, true> : k_kv_append<true, false>)
                         : (i8 ? k_kv_append<false, true> : k_kv_append<false, false>);
  hipLaunchKernelGGL(fn, dim3((a.t.n + a.per_block - 1) / a.per_block), dim3(kKvThreads), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_kv_gather(KvRowsArgs a, bool out_bf16, bool i8, hipStream_t st) {
  a.lanes_log = lanes_log(a.c.dim, i8 ? 16 : 8);
  const uint32_t rows = kKvThreads >> a.lanes_log;
  const auto fn = out_bf16 ? (i8 ? k_kv_gather<true, true> : k_kv_gather<true, false>)
                           : (i8 ? k_kv_gather<false, true> : k_kv_gather<false, false>);
  hipLaunchKernelGGL(fn, dim3((a.t.n * 2 * a.c.heads + rows - 1) / rows), dim3(kKvThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace smoe

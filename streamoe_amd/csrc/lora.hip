// lora.hip — low-rank adapters of many requests beside a shared projection.
//
//   y[t] = base[t] + scale[a] B_a (A_a x[t]),  a = ids[t]
//
//   k_lora_plan    rows sorted by adapter, items of up to 16 rows of one, for
//                  more rows or adapters than the next kernel sorts by itself
//   k_lora_down    u = A x of an item's rows on bf16 MFMA, one share of the
//                  inputs per block, partial sums in f32; leaves the items
//   k_lora_up      the shares added, scaled, times B on bf16 MFMA, plus base
//   k_lora_one     the last two for few rows and little of A
//
// f32 values enter the matrix cores as three bf16, eight bits of the value each:
// nothing is lost. A and B are bf16, so the products are exact and the sums f32.
// An infinity leaves a NaN in the second part, so its row's outputs are NaN.
#include "common.h"
#include "kernels.h"

#include <type_traits>

namespace smoe {

typedef __bf16 lbf16x8 __attribute__((ext_vector_type(8)));
typedef float lf32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kLoraM = 16;  // rows per item

__device__ __forceinline__ f32x4 mfma_bf16(lbf16x8 a, lbf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// v = p[0] + p[1] + p[2], each the rest's upper half.
__device__ __forceinline__ void split_bf16(lf32x8 v, lbf16x8 (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = __builtin_amdgcn_perm(__float_as_uint(v[2 * j + 1]), __float_as_uint(v[2 * j]), 0x07060302u);
    p[i] = __builtin_bit_cast(lbf16x8, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] -= __uint_as_float(__float_as_uint(v[j]) & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void split_bf16(float v, uint16_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t top = __float_as_uint(v) & 0xFFFF0000u;
    p[i] = (uint16_t)(top >> 16);
    v -= __uint_as_float(top);
  }
}

// The first n of eight bf16, zeros behind (n may be <= 0 or >= 8).
__device__ __forceinline__ lbf16x8 first_of(lbf16x8 v, int n) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = n >= 2 * j + 2 ? w[j] : n == 2 * j + 1 ? w[j] & 0xFFFFu : 0u;
  return __builtin_bit_cast(lbf16x8, w);
}

__device__ __forceinline__ uint32_t lora_rank(const LoraArgs& a, uint32_t ad) {
  if (!a.ranks) return a.max_rank;
  const int32_t r = a.ranks[ad];
  return r < 0 ? 0u : min((uint32_t)r, a.max_rank);
}

// Inclusive sums over the wave: DPP row shifts, then row broadcasts.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lora_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t lora_scan(uint32_t v) {
  v += lora_dpp<0x111, 0xF>(v);
  v += lora_dpp<0x112, 0xF>(v);
  v += lora_dpp<0x114, 0xF>(v);
  v += lora_dpp<0x118, 0xF>(v);
  v += lora_dpp<0x142, 0xA>(v);
  v += lora_dpp<0x143, 0xC>(v);
  return v;
}

// One block: counts per adapter, their items, each item's rows. Rows without
// an adapter (-1, or an id that does not exist, which is reported as a rank out
// of range is) come last, as items of adapter n_adapters. An item holds all
// that the other kernels need to know of its adapter.
__global__ __launch_bounds__(1024) void k_lora_plan(LoraArgs a) {
  extern __shared__ uint32_t sh[];  // [n_adapters + 1] counts, then taken; [n_adapters + 1] first items
  __shared__ uint32_t wrow[16], witem[16], base_row, base_item;
  const uint32_t t = threadIdx.x, N = a.n_adapters + 1;
  uint32_t* const first = sh + N;
  const int32_t id0 = t < a.n ? a.ids[t] : -1;  // the first 1024 rows' stay in registers
  for (uint32_t i = t; i < N; i += 1024) sh[i] = 0;
  if (t == 0) base_row = base_item = 0;
  __syncthreads();
  bool bad = false;
  auto adapter = [&](uint32_t row) {
    const int32_t id = row < 1024 ? id0 : a.ids[row];
    bad |= id < -1 || id >= (int32_t)a.n_adapters;
    return id < 0 || id >= (int32_t)a.n_adapters ? a.n_adapters : (uint32_t)id;
  };
  for (uint32_t r = t; r < a.n; r += 1024) atomicAdd(&sh[adapter(r)], 1u);
  for (uint32_t i0 = 0; i0 < N; i0 += 1024) {
    const uint32_t ad = i0 + t;
    uint32_t rank = 0;
    float scale = 0.f;
    if (ad < a.n_adapters) {
      rank = lora_rank(a, ad);
      scale = a.scale[ad];
      if (a.ranks) bad |= a.ranks[ad] < 0 || a.ranks[ad] > (int32_t)a.max_rank;
    }
    __syncthreads();  // the counts; the bases of the 1024 before
    const uint32_t c = ad < N ? sh[ad] : 0u, it = (c + kLoraM - 1) / kLoraM;
    const uint32_t pr = lora_scan(c), pi = lora_scan(it);
    if ((t & 63) == 63) wrow[t >> 6] = pr, witem[t >> 6] = pi;
    __syncthreads();
    uint32_t row = base_row + pr - c, item = base_item + pi - it;
    for (uint32_t w = 0; w < (t >> 6); ++w) row += wrow[w], item += witem[w];
    if (ad < N) {
      sh[ad] = 0;
      first[ad] = item;
      for (uint32_t j = 0; j < it; ++j)
        a.items[item + j] = LoraItem{ad, row + j * kLoraM, min(kLoraM, c - j * kLoraM), rank, scale};
    }
    __syncthreads();
    if (t == 1023) base_row = row + c, base_item = item + it;
  }
  __syncthreads();
  if (bad) *a.err = 2u;
  for (uint32_t i = base_item + t; i < a.n_items; i += 1024) a.items[i] = LoraItem{0u, 0u, 0u, 0u, 0.f};
  // Which row of an adapter takes which place does not touch any result.
  for (uint32_t r = t; r < a.n; r += 1024) {
    const uint32_t ad = adapter(r);
    a.rows[first[ad] * kLoraM + atomicAdd(&sh[ad], 1u)] = r;
  }
}

constexpr uint32_t kLoraSmall = 64;  // rows whose items need no plan: one per lane

// Item blockIdx.x of a call of up to 64 rows, by every wave for itself: the
// rows' ids, one per lane, the lanes of the same id from ballots of its bits;
// every 16th of them starts an item, items are in the order of those lanes.
// `rows` receives the item's rows (kLoraM per wave). (Adapter after adapter in a
// loop a call of 64 rows of 64 adapters took 18 us, 9.5 so.)
__device__ __forceinline__ LoraItem lora_wave_item(const LoraArgs& a, uint32_t lane, uint32_t* rows) {
  const bool there = lane < a.n;
  const int32_t id = a.ids[min(lane, a.n - 1)];
  const bool bad = there && (id < -1 || id >= (int32_t)a.n_adapters);
  const uint32_t ad = bad || id < 0 ? a.n_adapters : (uint32_t)id;
  uint32_t rank = 0;  // of the lane's adapter
  float scale = 0.f;
  if (ad < a.n_adapters) rank = lora_rank(a, ad), scale = a.scale[ad];
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    bool wrong = bad;
    if (a.ranks)
      for (uint32_t i = lane; i < a.n_adapters; i += 64) wrong |= a.ranks[i] < 0 || a.ranks[i] > (int32_t)a.max_rank;
    if (wrong) *a.err = 2u;
  }
  uint64_t same = __ballot(there);
  for (uint32_t bit = 0; a.n_adapters >> bit; ++bit) {
    const bool set = ad >> bit & 1;
    const uint64_t m = __ballot(set);
    same &= set ? m : ~m;
  }
  auto below = [](uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
  const uint32_t place = below(same), all = (uint32_t)__popcll(same);
  const bool first = there && place % kLoraM == 0;
  const uint64_t firsts = __ballot(first);
  const uint32_t count = first ? min(kLoraM, all - place) : 0u, upto = lora_scan(count);
  const uint64_t which = __ballot(first && below(firsts) == blockIdx.x);
  LoraItem it{0u, 0u, 0u, 0u, 0.f};
  if (which) {
    const int lead = __ffsll((long long)which) - 1;
    auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lead); };
    it = LoraItem{of(ad), of(upto - count), of(count), of(rank), readlane_f(scale, lead)};
    const uint32_t at = place - of(place);
    if (there && ad == it.adapter && at < kLoraM) rows[at] = lane;
  }
  // The rows are in LDS: no other wave writes or reads this part.
  wave_lds();
  return it;
}

constexpr uint32_t kLoraMid = 1024;  // rows, and adapters and one: four of each per thread

struct LoraFind {
  uint32_t count[kLoraMid];
  uint32_t sums[4], of[4][4];
  LoraItem item;
  uint32_t nth;  // of the adapter's items
  uint32_t rows[kLoraM];
};

// Item blockIdx.x of a call of up to 1024 rows and 1023 adapters, by the block:
// counts per adapter, their items (the adapters t, t + 256, .. of thread 0, of
// thread 1, ..), then the places of the item's adapter's rows in the rows'
// order.
__device__ __forceinline__ LoraItem lora_block_item(const LoraArgs& a, LoraFind& f) {
  const uint32_t t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), N = a.n_adapters;
  int32_t id[4], rk[4];
  float sc[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t row = 256 * j + t;
    id[j] = -1;
    if (256 * j < a.n) id[j] = a.ids[min(row, a.n - 1)];
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    rk[j] = (int32_t)a.max_rank;
    sc[j] = 0.f;
    if (256 * j < N) {
      sc[j] = a.scale[min(256 * j + t, N - 1)];
      if (a.ranks) rk[j] = a.ranks[min(256 * j + t, N - 1)];
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    if (256 * j <= N) f.count[256 * j + t] = 0;
  if (t == 0) f.item = LoraItem{0u, 0u, 0u, 0u, 0.f};
  __syncthreads();
  uint32_t ad[4];  // ~0: no row
  bool bad = false;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    ad[j] = ~0u;
    if (256 * j >= a.n) continue;
    const bool in = 256 * j + t < a.n, is = id[j] >= 0 && id[j] < (int32_t)N;
    bad |= in && !is && id[j] != -1;
    if (in) ad[j] = is ? (uint32_t)id[j] : N;
    // Those of the first lane's adapter in one, the others one by one (64 adds
    // to one address are 64 turns).
    const uint32_t lead = (uint32_t)__builtin_amdgcn_readfirstlane((int)ad[j]);
    const uint64_t same = __ballot(ad[j] == lead);
    if (ad[j] != lead || lane == 0)
      if (ad[j] != ~0u) atomicAdd(&f.count[ad[j]], lane == 0 ? (uint32_t)__popcll(same) : 1u);
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) bad |= rk[j] < 0 || rk[j] > (int32_t)a.max_rank;
  if (bad && blockIdx.x == 0 && blockIdx.y == 0) *a.err = 2u;
  __syncthreads();
  // Items in the upper half, rows in the lower.
  uint32_t own[4], sum = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    own[j] = 0;
    if (256 * j > N) continue;
    const uint32_t c = f.count[256 * j + t];
    own[j] = (c + kLoraM - 1) / kLoraM << 16 | c;
    sum += own[j];
  }
  uint32_t before = lora_scan(sum);
  if (lane == 63) f.sums[wave] = before;
  __syncthreads();
  before -= sum;
  for (uint32_t w = 0; w < wave; ++w) before += f.sums[w];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t nth = blockIdx.x - (before >> 16), i = 256 * j + t;
    if (nth < own[j] >> 16) {
      const uint32_t rank = i < N ? (uint32_t)min(max(rk[j], 0), (int32_t)a.max_rank) : 0u;
      f.item = LoraItem{i, (before & 0xFFFFu) + nth * kLoraM, min(kLoraM, (own[j] & 0xFFFFu) - nth * kLoraM), rank,
                        i < N ? sc[j] : 0.f};
      f.nth = nth;
    }
    before += own[j];
  }
  __syncthreads();
  const LoraItem it = f.item;
  if (it.count == 0) return it;  // the whole block
  uint64_t of[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    of[j] = __ballot(ad[j] == it.adapter);
    if (lane == 0) f.of[j][wave] = (uint32_t)__popcll(of[j]);
  }
  __syncthreads();
  uint32_t at = 0u - f.nth * kLoraM;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    uint32_t place = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(of[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)of[j], 0u));
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const uint32_t c = f.of[j][w];
      at += c;
      if (w < wave) place += c;
    }
    if (ad[j] == it.adapter && place < kLoraM) f.rows[place] = 256 * j + t;
  }
  __syncthreads();
  return it;
}

// The item of this block as k_lora_plan or k_lora_down left it, and row
// min(c, count - 1) of it.
__device__ __forceinline__ LoraItem lora_item(const LoraArgs& a, uint32_t lane, uint32_t& row) {
  const LoraItem it = a.items[blockIdx.x];
  const uint32_t r = a.rows[blockIdx.x * kLoraM + (lane & 15)];  // unset past the count: replaced
  const uint32_t last = (uint32_t)__shfl((int)r, (int)(it.count ? it.count - 1 : 0u), kWave);
  row = (lane & 15) < it.count ? r : last;
  return it;
}

// Who finds the items: k_lora_plan, k_lora_down's waves, its blocks.
enum LoraBy { kByPlan, kByWave, kByBlock };

// u[share][place][j] = sum over the share's inputs of A[j] x. Four waves take
// steps of 32 inputs in turn; lane (c, kb) holds eight inputs kb of row c. A
// share per block makes blocks of few rows: 200 rows, 40 adapters of rank 64,
// 4096 inputs 10.5 us for 24 MB, of which finding the items is about 3.
template <bool XBF16, LoraBy BY, int MT>
__global__ __launch_bounds__(256) void k_lora_down(LoraArgs a) {
  __shared__ f32x4 red[4][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, kb = lane >> 4;
  uint32_t row;
  LoraItem it;
  if constexpr (BY == kByPlan) {
    it = lora_item(a, lane, row);
  } else {
    const uint32_t* rows;
    if constexpr (BY == kByWave) {
      __shared__ uint32_t of_wave[4][kLoraM];
      it = lora_wave_item(a, lane, of_wave[wave]);
      rows = of_wave[wave];
    } else {
      __shared__ LoraFind f;
      it = lora_block_item(a, f);
      rows = f.rows;
    }
    row = it.count ? rows[min(c16, it.count - 1)] : 0u;
    if (blockIdx.y == 0 && threadIdx.x < kLoraM) {
      a.rows[blockIdx.x * kLoraM + threadIdx.x] = row;
      if (threadIdx.x == 0) a.items[blockIdx.x] = it;
    }
  }
  if (it.count == 0 || it.adapter >= a.n_adapters) return;
  const uint32_t K = a.in_dim, share = blockIdx.y;
  const uint32_t rank = it.rank, nt = (rank + 15) / 16;
  const uint16_t* const A = (const uint16_t*)(a.a + (uint64_t)it.adapter * a.a_stride);
  const uint32_t steps = (K + 31) / 32, s0 = steps * share / a.shares, s1 = steps * (share + 1) / a.shares;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Two steps' loads at once.
  using X = std::conditional_t<XBF16, lbf16x8, lf32x8>;
  struct Step {
    X x;
    lbf16x8 w[MT];
  };
  auto load = [&](uint32_t s, Step& v) {
    const uint32_t k = s * 32 + kb * 8, kc = k < K ? k : 0;  // K is a multiple of 8
    v.x = *reinterpret_cast<const X*>(reinterpret_cast<const uint8_t*>(a.x) + ((uint64_t)row * K + kc) * (sizeof(X) / 8));
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (i < (int)nt) v.w[i] = *reinterpret_cast<const lbf16x8*>(A + (uint64_t)min(i * 16 + c16, rank - 1) * K + kc);
  };
  auto compute = [&](uint32_t s, const Step& v) {
    const bool in = s * 32 + kb * 8 < K;
    lbf16x8 x[3];
    if constexpr (XBF16)
      x[0] = first_of(v.x, in ? 8 : 0);
    else
      split_bf16(in ? v.x : lf32x8{0, 0, 0, 0, 0, 0, 0, 0}, x);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i >= (int)nt) break;
      const lbf16x8 w = first_of(v.w[i], in && i * 16 + c16 < rank ? 8 : 0);
#pragma unroll
      for (int k = 0; k < (XBF16 ? 1 : 3); ++k) acc[i] = mfma_bf16(x[k], w, acc[i]);
    }
  };
  for (uint32_t s = s0 + wave; s < s1; s += 8) {
    Step v[2];
    load(s, v[0]);
    if (s + 4 < s1) load(s + 4, v[1]);
    compute(s, v[0]);
    if (s + 4 < s1) compute(s + 4, v[1]);
  }
  for (uint32_t i = 0; i < nt; ++i) {
    f32x4 v = acc[0];
#pragma unroll
    for (int j = 1; j < MT; ++j)
      if ((int)i == j) v = acc[j];
    red[wave][lane] = v;
    __syncthreads();
    if (wave == 0) {
      const f32x4 s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
      float* const u = a.u + ((uint64_t)share * a.n + it.start) * a.max_rank + i * 16 + c16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * kb + r < it.count && i * 16 + c16 < a.max_rank) u[(uint64_t)(4 * kb + r) * a.max_rank] = s[r];
    }
    __syncthreads();
  }
}

// D = B (outputs) x u (rows): lane (c, kb) ends with outputs 4 kb .. of row c.
// A block takes 64 NT outputs of an item; it adds the shares once, into LDS, as
// the bf16 parts that its waves read as operands (added by every wave for
// itself the shares were 22 of 33 us: 200 rows, 40 adapters of rank 64, 4096 ->
// 4096). The products go through LDS too, so that base and y move in whole rows
// of the block (in the products' order each lane touches a line of its own).
// B's and base's loads go out ahead of everything. 200 rows of rank 64 -> 4096
// 10.1 us for 28 MB, 1000 rows of rank 32 -> 4096 12.6 us for 33 MB of base and
// y. With NT = 4 the 162 to 198 registers and 16 accumulators leave two blocks
// per CU, so these 848 and 1056 blocks run in two to three rounds, each the
// chain of its loads: items, shares and base, products, stores.
template <int KT, int NT>
__global__ __launch_bounds__(256) void k_lora_up(LoraArgs a) {
  constexpr uint32_t RP = KT * 32 + 8;  // bf16 per row in LDS: rows apart by 16 bytes of banks
  constexpr uint32_t OB = 64 * NT, OP = OB + 4;  // outputs of the block; floats per row in LDS, apart by 16 bytes of banks
  __shared__ __attribute__((aligned(16))) uint16_t up[3][kLoraM * RP];
  __shared__ __attribute__((aligned(16))) float prod[kLoraM * OP];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, kb = lane >> 4;
  uint32_t row;
  const LoraItem it = lora_item(a, lane, row);
  if (it.count == 0) return;
  const uint32_t O = a.out_dim, R = a.max_rank;
  const uint32_t o0 = (blockIdx.y * 4 + wave) * NT * 16;
  const bool none = it.adapter >= a.n_adapters;
  if (none && a.base == a.y) return;
  const uint32_t rank = none ? 0u : it.rank;
  lbf16x8 w[KT][NT];
  if (rank) {
    const uint16_t* const B = (const uint16_t*)(a.b + (uint64_t)it.adapter * a.b_stride);
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const uint32_t k = s * 32 + kb * 8;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (s * 32 < (int)rank)
          w[s][i] = *reinterpret_cast<const lbf16x8*>(B + (uint64_t)min(o0 + i * 16 + c16, O - 1) * R + (k < R ? k : 0));  // R is a multiple of 8
    }
  }
  // Fours of outputs of whole rows: thread i's are i, i + 256, ..
  const uint32_t ob = blockIdx.y * OB;
  auto place = [&](int i, uint32_t& r, uint32_t& o) {
    const uint32_t f = threadIdx.x + 256 * i;
    r = f / (OB / 4);
    o = f % (OB / 4) * 4;
    return (uint64_t)(uint32_t)__shfl((int)row, (int)r, kWave) * O + ob + o;
  };
  f32x4 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t r, o;
    const uint64_t e = place(i, r, o);
    if (!a.base || r >= it.count) continue;
    if (a.vec) {
      if (ob + o < O) acc[i] = *reinterpret_cast<const f32x4*>(a.base + e);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (ob + o + c < O) acc[i][c] = a.base[e + c];
    }
  }
  f32x4 low[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) low[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (rank) {  // the same for the whole block
    const float scale = it.scale;
    const uint32_t q = R / 4;  // quarters of eights: a thread adds four values
    for (uint32_t i = threadIdx.x; i < kLoraM * KT * 8; i += 256) {
      const uint32_t r = i / (KT * 8), k = i % (KT * 8) * 4;
      f32x4 u = {0.f, 0.f, 0.f, 0.f};
      if (r < it.count && k < R) {
        const f32x4* const p = reinterpret_cast<const f32x4*>(a.u) + ((uint64_t)it.start + r) * q + k / 4;
        const uint64_t apart = (uint64_t)a.n * q;
        // Loads of up to eight shares at once, added in order.
        auto add = [&](uint32_t s0, auto count) {
          constexpr int C = decltype(count)::value;
          f32x4 v[C];
#pragma unroll
          for (int s = 0; s < C; ++s) v[s] = p[(s0 + s) * apart];
#pragma unroll
          for (int s = 0; s < C; ++s) u += v[s];
        };
        if (a.shares >= 8) {
          for (uint32_t s = 0; s < a.shares; s += 8) add(s, std::integral_constant<int, 8>{});
        } else if (a.shares == 4) {
          add(0, std::integral_constant<int, 4>{});
        } else {
          add(0, std::integral_constant<int, 1>{});
        }
      }
      uint16_t p[4][3];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_bf16(k + j < rank ? u[j] * scale : 0.f, p[j]);  // nothing was written behind the rank
#pragma unroll
      for (int j = 0; j < 3; ++j)
        *reinterpret_cast<uint2*>(up[j] + r * RP + k) =
            make_uint2(p[0][j] | (uint32_t)p[1][j] << 16, p[2][j] | (uint32_t)p[3][j] << 16);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const uint32_t k = s * 32 + kb * 8;
      if (s * 32 >= (int)rank) break;
      const int left = k < rank ? (int)(rank - k) : 0;
      lbf16x8 v[3];
#pragma unroll
      for (int j = 0; j < 3; ++j) v[j] = *reinterpret_cast<const lbf16x8*>(up[j] + c16 * RP + k);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const lbf16x8 b = first_of(w[s][i], left);
#pragma unroll
        for (int j = 0; j < 3; ++j) low[i] = mfma_bf16(b, v[j], low[i]);
      }
    }
  }
  if (rank) {
#pragma unroll
    for (int i = 0; i < NT; ++i) *reinterpret_cast<f32x4*>(prod + c16 * OP + (wave * NT + i) * 16 + 4 * kb) = low[i];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    uint32_t r, o;
    const uint64_t e = place(i, r, o);
    if (r >= it.count) continue;
    f32x4 v = acc[i];
    if (rank) v += *reinterpret_cast<const f32x4*>(prod + r * OP + o);
    if (a.vec) {
      if (ob + o < O) *reinterpret_cast<f32x4*>(a.y + e) = v;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (ob + o + c < O) a.y[e + c] = v[c];
    }
  }
}

// Both products of a small item in one launch: sixteen waves share the inputs
// (step s is wave s mod 16's), their parts are added in LDS, and each wave takes
// 16 outputs. Every block of 256 outputs forms u for itself, from the caches (8
// rows, 4 adapters of rank 16, 2048 -> 2048: 6.7 us, the two kernels 6.2). A CU
// loads a block's 64 KB of A and 16 KB of x in some 0.6 us; the rest is one
// wave's chain (ids, rows, loads, the joins' barriers, the second product), not
// taken apart.
template <bool XBF16, int MT>
__global__ __launch_bounds__(1024) void k_lora_one(LoraArgs a) {
  constexpr int KT = (MT + 1) / 2, U = MT <= 2 ? 4 : 2;  // steps of 32 ranks; steps of inputs in flight
  constexpr uint32_t RP = KT * 32 + 8;                   // as in k_lora_up
  __shared__ __attribute__((aligned(16))) float red[16][256];
  __shared__ __attribute__((aligned(16))) uint16_t up[3][kLoraM * RP];
  __shared__ uint32_t of_wave[16][kLoraM];
  const uint32_t lane = threadIdx.x & 63, c16 = lane & 15, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraItem it = lora_wave_item(a, lane, of_wave[wave]);
  if (it.count == 0) return;
  const bool none = it.adapter >= a.n_adapters;
  if (none && a.base == a.y) return;
  const uint32_t row = of_wave[wave][min(c16, it.count - 1)];
  const uint32_t K = a.in_dim, O = a.out_dim, R = a.max_rank, rank = none ? 0u : it.rank, steps = (K + 31) / 32;
  const uint32_t o0 = (blockIdx.y * 16 + wave) * 16, o = o0 + 4 * kb;
  // B's rows and base first: they are needed last.
  lbf16x8 b[KT];
  if (rank) {
    const uint16_t* const B = (const uint16_t*)(a.b + (uint64_t)it.adapter * a.b_stride) + (uint64_t)min(o0 + c16, O - 1) * R;
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const uint32_t k = s * 32 + kb * 8;
      b[s] = *reinterpret_cast<const lbf16x8*>(B + (k < R ? k : 0));  // R is a multiple of 8
    }
  }
  const bool mine = c16 < it.count;
  const uint64_t e = (uint64_t)row * O + o;
  f32x4 base = {0.f, 0.f, 0.f, 0.f};
  if (a.base && mine) {
    if (a.vec) {
      if (o < O) base = *reinterpret_cast<const f32x4*>(a.base + e);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (o + c < O) base[c] = a.base[e + c];
    }
  }
  f32x4 low = {0.f, 0.f, 0.f, 0.f};
  if (rank) {  // the same for the whole block
    const uint32_t nt = (rank + 15) / 16;
    const uint16_t* const A = (const uint16_t*)(a.a + (uint64_t)it.adapter * a.a_stride);
    using X = std::conditional_t<XBF16, lbf16x8, lf32x8>;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = wave; s0 < steps; s0 += 16 * U) {
      X x[U];
      lbf16x8 w[U][MT];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const uint32_t k = (s0 + 16 * j) * 32 + kb * 8, kc = k < K ? k : 0;  // K is a multiple of 8
        if (s0 + 16 * j >= steps) continue;
        x[j] = X{};
        if (mine) x[j] = *reinterpret_cast<const X*>(reinterpret_cast<const uint8_t*>(a.x) + ((uint64_t)row * K + kc) * (sizeof(X) / 8));
#pragma unroll
        for (int i = 0; i < MT; ++i)
          if (i < (int)nt) w[j][i] = *reinterpret_cast<const lbf16x8*>(A + (uint64_t)min(i * 16 + c16, rank - 1) * K + kc);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (s0 + 16 * j >= steps) break;
        const bool in = (s0 + 16 * j) * 32 + kb * 8 < K;
        lbf16x8 p[3];
        if constexpr (XBF16)
          p[0] = first_of(x[j], in ? 8 : 0);
        else
          split_bf16(in ? x[j] : lf32x8{0, 0, 0, 0, 0, 0, 0, 0}, p);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (i >= (int)nt) break;
          const lbf16x8 v = first_of(w[j][i], in && i * 16 + c16 < rank ? 8 : 0);
#pragma unroll
          for (int k = 0; k < (XBF16 ? 1 : 3); ++k) acc[i] = mfma_bf16(p[k], v, acc[i]);
        }
      }
    }
    const uint32_t t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 2 * KT; ++i) {  // tiles behind the rank leave zeros
      const f32x4 v = i < MT ? acc[i < MT ? i : 0] : f32x4{0.f, 0.f, 0.f, 0.f};
      if (i) __syncthreads();
      *reinterpret_cast<f32x4*>(&red[wave][lane * 4]) = v;
      __syncthreads();
      // Value 4 l + r: row 4 (l / 16) + r, rank 16 i + l % 16.
      if (t < 256) {
        float sum = red[0][t];
#pragma unroll
        for (int w = 1; w < 16; ++w) sum += red[w][t];
        const uint32_t j = i * 16 + (t >> 2 & 15), at = ((t >> 6) * 4 + (t & 3)) * RP + j;
        uint16_t p[3];
        split_bf16(j < rank ? sum * it.scale : 0.f, p);
#pragma unroll
        for (int k = 0; k < 3; ++k) up[k][at] = p[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const uint32_t k = s * 32 + kb * 8;
      const lbf16x8 v = first_of(b[s], k < rank ? (int)(rank - k) : 0);
#pragma unroll
      for (int j = 0; j < 3; ++j) low = mfma_bf16(v, *reinterpret_cast<const lbf16x8*>(up[j] + c16 * RP + k), low);
    }
  }
  if (!mine) return;
  const f32x4 y = base + low;
  if (a.vec) {
    if (o < O) *reinterpret_cast<f32x4*>(a.y + e) = y;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (o + c < O) a.y[e + c] = y[c];
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
static uint64_t al256(uint64_t n) { return (n + 255) & ~255ull; }

// Shares of the inputs: enough blocks for few rows, none to spare for many
// (k_lora_up adds 16, 8, 4 or 1).
static uint32_t lora_shares(uint32_t n) { return n <= 64 ? 16u : n <= 1024 ? 8u : n <= 4096 ? 4u : 1u; }

uint64_t lora_workspace(uint32_t n_adapters, uint32_t max_rank, uint32_t n, LoraArgs* a, uint8_t* base) {
  const uint32_t shares = lora_shares(n);
  // Every adapter in use leaves at most one item short of 16 rows.
  const uint32_t items = n / kLoraM + (n < n_adapters + 1 ? n : n_adapters + 1);
  const uint64_t ib = al256((uint64_t)items * sizeof(LoraItem)), pb = al256((uint64_t)items * kLoraM * 4);
  if (a) {
    a->n_items = items;
    a->shares = shares;
    a->items = reinterpret_cast<LoraItem*>(base);
    a->rows = reinterpret_cast<uint32_t*>(base + ib);
    a->u = reinterpret_cast<float*>(base + ib + pb);
  }
  return ib + pb + al256((uint64_t)shares * n * max_rank * 4);
}

template <LoraBy BY>
static hipError_t lora_go(const LoraArgs& a, bool x_bf16, hipStream_t st) {
  auto down = [&](auto fn) {
    hipLaunchKernelGGL(fn, dim3(a.n_items, a.shares), dim3(256), 0, st, a);
    return hipGetLastError();
  };
  const uint32_t mt = (a.max_rank + 15) / 16;  // tiles of 16 ranks
  const hipError_t e = x_bf16 ? (mt <= 1   ? down(k_lora_down<true, BY, 1>)
                                 : mt <= 2 ? down(k_lora_down<true, BY, 2>)
                                 : mt <= 4 ? down(k_lora_down<true, BY, 4>)
                                           : down(k_lora_down<true, BY, 8>))
                              : (mt <= 1   ? down(k_lora_down<false, BY, 1>)
                                 : mt <= 2 ? down(k_lora_down<false, BY, 2>)
                                 : mt <= 4 ? down(k_lora_down<false, BY, 4>)
                                           : down(k_lora_down<false, BY, 8>));
  if (e != hipSuccess) return e;
  // Outputs per block: as many as leave two blocks for every CU.
  auto up = [&](auto fn, uint32_t nt) {
    hipLaunchKernelGGL(fn, dim3(a.n_items, (a.out_dim + 64 * nt - 1) / (64 * nt)), dim3(256), 0, st, a);
    return hipGetLastError();
  };
  const bool wide = (uint64_t)a.n_items * ((a.out_dim + 255) / 256) >= 512;
  if (a.max_rank <= 32) return wide ? up(k_lora_up<1, 4>, 4) : up(k_lora_up<1, 1>, 1);
  if (a.max_rank <= 64) return wide ? up(k_lora_up<2, 4>, 4) : up(k_lora_up<2, 1>, 1);
  return wide ? up(k_lora_up<4, 4>, 4) : up(k_lora_up<4, 1>, 1);
}

// One launch where what a block reads of A and x is little: us on the device,
// f32 rows, 4 adapters, one launch and two: 8 rows 512 -> 512 rank 16 4.0 and
// 6.3, rank 64 7.0 and 7.4; 2048 -> 2048 rank 16 6.7 and 6.2 (131 KB), 16 rows
// 7.1 and 6.4 (197 KB), 64 rows 9.6 and 6.7; rank 32 8.6 and 6.6; 4096 -> 512
// rank 16 9.8 and 6.5. Over 1500 calls of 1 to 64 rows and as many adapters, 256
// to 4096 inputs, 64 to 4096 outputs, ranks 8 to 64 the chosen took 1.007 times
// the faster one's time (135 or 165 KB: 1.008). A caller without a graph pays
// 2.5 for the second launch.
constexpr uint64_t kOneBlocks = 512, kOneBytes = 150 * 1000;

hipError_t launch_lora(const LoraArgs& a, bool x_bf16, hipStream_t st) {
  const uint64_t blocks = (uint64_t)a.n_items * ((a.out_dim + 255) / 256);
  const uint32_t mt = (a.max_rank + 15) / 16;  // tiles of 16 ranks
  if (a.n <= kLoraSmall && mt <= 4 && blocks <= kOneBlocks &&
      (uint64_t)a.in_dim * (kLoraM * 2 * mt + (a.n < kLoraM ? a.n : kLoraM) * (x_bf16 ? 2 : 4)) <= kOneBytes) {
    auto one = [&](auto fn) {
      hipLaunchKernelGGL(fn, dim3(a.n_items, (a.out_dim + 255) / 256), dim3(1024), 0, st, a);
      return hipGetLastError();
    };
    if (mt <= 1) return x_bf16 ? one(k_lora_one<true, 1>) : one(k_lora_one<false, 1>);
    if (mt <= 2) return x_bf16 ? one(k_lora_one<true, 2>) : one(k_lora_one<false, 2>);
    return x_bf16 ? one(k_lora_one<true, 4>) : one(k_lora_one<false, 4>);
  }
  if (a.n <= kLoraSmall) return lora_go<kByWave>(a, x_bf16, st);
  if (a.n <= kLoraMid && a.n_adapters < kLoraMid) return lora_go<kByBlock>(a, x_bf16, st);
  hipLaunchKernelGGL(k_lora_plan, dim3(1), dim3(1024), (a.n_adapters + 1) * 8, st, a);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : lora_go<kByPlan>(a, x_bf16, st);
}

}  // namespace smoe

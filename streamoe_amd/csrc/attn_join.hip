// attn_join.hip — the rows of the attention that several blocks had a part of,
// and the rows that see nothing.
#include "attn.h"

namespace smoe {

// A block joins a share (blockIdx.y) of one group's columns: fours of dims, each
// by 256 / lanes threads that go through the parts in turn and are added up at
// the end. Parts are added in their order, so a call gives the same bits again.
// 4 to 5 us: the launch and a chain of three loads (the units before the group,
// then m, l and the outputs of its parts, a few MB); where a row is cut into 128
// parts, 64 blocks share its columns. The last block of a group joining them would
// need counters that start at zero: the workspace holds anything, the handle's
// memory could have them if each group's last block put its own back.
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, uint32_t pad) {
  __shared__ f32x4 sum[256];
  __shared__ float2 stat[256];
  const uint32_t tiles = a.c.heads * a.parts, row = blockIdx.x / tiles, tile = blockIdx.x - row * tiles;
  const uint32_t t = threadIdx.x, fours = a.c.dim / 4;
  const uint64_t before = a.before[row], units = a.before[row + 1] - before, all_units = a.before[a.t.n];
  // The group, all of its tokens at once.
  const uint32_t i = t & 15, r = min(row + i, a.t.n - 1), r1 = r ? r - 1 : 0;
  const bool follows = attn_follows(a, r, a.t.seq[r], a.t.pos[r], a.t.seq[r1], a.t.pos[r1]);
  const uint32_t mask = (uint32_t)__ballot(follows && row + i < a.t.n) & 0xFFFFu;
  if (mask & 1) return;  // another group's token
  const uint32_t n = __builtin_ctz(~(mask >> 1)) + 1;
  const uint32_t kvh = tile / a.parts, part = tile - kvh * a.parts;
  const uint32_t head0 = kvh * a.group + part * 16, heads = min(16u, a.group - part * 16);
  const uint32_t all = n * heads * fours, share = (all + gridDim.y - 1) / gridDim.y;
  const uint32_t from = blockIdx.y * share, to = min(all, from + share);
  auto put = [&](uint32_t e, f32x4 v) {
    const uint32_t col = e / fours, token = col / heads;
    const uint64_t at = ((uint64_t)(row + token) * a.heads + head0 + col - token * heads) * a.c.dim + (e - col * fours) * 4;
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    if (a.out_bf16)
      *reinterpret_cast<bf16x4*>((uint16_t*)a.out + at) = __builtin_convertvector(v, bf16x4);
    else
      *reinterpret_cast<f32x4*>((float*)a.out + at) = v;
  };
  if (!units) {
    for (uint32_t e = from + t; e < to; e += 256) put(e, f32x4{0, 0, 0, 0});
    return;
  }
  const uint64_t total = all_units * tiles, x = before * tiles + tile * units + kAttnOver, last = x + units - kAttnOver - 1;
  const uint32_t b0 = attn_block_of(x, total, a.blocks_log), b1 = attn_block_of(last, total, a.blocks_log);
  if (b0 == b1) return;
  const uint32_t parts = b1 - b0 + 1;
  uint32_t lanes = 8;
  while (lanes < 256 && lanes < share) lanes *= 2;
  const uint32_t turns = 256 / lanes, turn = t / lanes;
  for (uint32_t e0 = from; e0 < to; e0 += lanes) {
    const uint32_t e = e0 + t % lanes, in = min(e, all - 1), col = in / fours, d = (in - col * fours) * 4;
    float m = kAttnNone, l = 0.f;
    f32x4 acc = {0, 0, 0, 0};
    // K parts of this turn from p on, their loads together.
    auto take = [&](uint32_t p0, auto count) {
      constexpr uint32_t K = decltype(count)::value;
      float2 s[K];
      f32x4 v[K];
#pragma unroll
      for (uint32_t i = 0; i < K; ++i) {
        const uint32_t p = min(p0 + i * turns, parts - 1);
        const uint64_t slot = 2 * (uint64_t)(b0 + p) + (p == 0 ? 1 : 0);
        s[i] = *reinterpret_cast<const float2*>(a.ml + (slot * 16 + col) * 2);
        v[i] = *reinterpret_cast<const f32x4*>(a.acc + (slot * 16 + col) * pad + d);
      }
      float top = m;
#pragma unroll
      for (uint32_t i = 0; i < K; ++i) top = fmaxf(top, s[i].x);
      const float f = __builtin_amdgcn_exp2f(m - top);
      l *= f;
      acc *= f;
      m = top;
#pragma unroll
      for (uint32_t i = 0; i < K; ++i) {
        if (p0 + i * turns >= parts) continue;
        const float w = __builtin_amdgcn_exp2f(s[i].x - top);
        l += s[i].y * w;
        acc += v[i] * w;
      }
    };
    if (parts <= turns) {
      if (turn < parts) take(turn, std::integral_constant<uint32_t, 1>{});
    } else {
      for (uint32_t p = turn; p < parts; p += 4 * turns) take(p, std::integral_constant<uint32_t, 4>{});
    }
    auto add = [&](float om, float ol, f32x4 oacc) {
      const float top = fmaxf(m, om), f = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(om - top);
      l = l * f + ol * w;
      acc = acc * f + oacc * w;
      m = top;
    };
    // Turns of one wave, then of the waves.
    for (uint32_t o = lanes; o < 64; o <<= 1) {
      f32x4 other;
#pragma unroll
      for (int j = 0; j < 4; ++j) other[j] = __shfl_xor(acc[j], (int)o, kWave);
      add(__shfl_xor(m, (int)o, kWave), __shfl_xor(l, (int)o, kWave), other);
    }
    sum[t] = acc;
    stat[t] = float2{m, l};
    __syncthreads();
    if (turn == 0 && e < to) {
      for (uint32_t i = max(64u, lanes); i < 256; i += max(64u, lanes)) add(stat[t + i].x, stat[t + i].y, sum[t + i]);
      put(e, acc * (l == 0.f ? 0.f : 1.f / l));
    }
    __syncthreads();
  }
}

hipError_t launch_attn_join(const AttnArgs& a, hipStream_t st) {
  const uint32_t items = a.t.n * a.c.heads * a.parts;
  // A share of eight fours where there are few rows to join, whole groups where
  // there are many; a thousand blocks in all (captured calls of 61 rows of 2
  // key heads 48.8 us, with two thousand 49.4, 500 48.9; 48 rows of 16 key heads
  // 55.6, 56.6 and 55.7; 8 sequences' 4 tokens each of 8 key heads 20.6, 22.0 and 22.3).
  const uint32_t most = (min(16u, a.group) * a.together * a.c.dim / 4 + 7) / 8, y = min(most, max(1u, 1024 / items));
  const uint32_t pad = a.c.dim <= 64 ? 64 : a.c.dim <= 128 ? 128 : 256;
  hipLaunchKernelGGL(k_attn_join, dim3(items, y), dim3(256), 0, st, a, pad);
  return hipGetLastError();
}

uint64_t attn_workspace(uint32_t dim, uint32_t n, AttnArgs* a, uint8_t* base) {
  const uint32_t pad = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  auto al = [](uint64_t b) { return (b + 255) & ~(uint64_t)255; };
  const uint32_t blocks = kAttnCus * attn_blocks_per_cu(pad);
  const uint64_t before = al((uint64_t)(n + 1) * 8), ml = al((uint64_t)blocks * 2 * 16 * 2 * 4);
  if (a) {
    a->blocks_log = 31 - __builtin_clz(blocks);
    a->before = (uint64_t*)base;
    a->ml = (float*)(base + before);
    a->acc = (float*)(base + before + ml);
  }
  return before + ml + (uint64_t)blocks * 2 * 16 * pad * 4;
}

}  // namespace smoe

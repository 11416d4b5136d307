// attn_plan.h — which part of a call's attention each block takes.
//
// Integers only, so that a host program can run it against its definition with a
// block's waves in any order: the exchange between lanes (common.h) is the
// includer's.
#pragma once

#include "kernels.h"

namespace smoe {

constexpr uint32_t kAttnUnit = 32;  // positions of a unit
// What a group costs by itself (queries, first loads, the exchange between the
// waves, a part for the join), in units: calls of 61 rows of very different lengths
// in 8 bits, captured, take 58 us with 0, 50 with 2, 50 with 4, 49 with 6, 47 with
// 8, 47 with 12; 48 rows of 16 key heads 89, 62, 56, 56, 56 and 59; 8 sequences'
// windows of 1000 25, 24, 21, 21, 20 and 20.
constexpr uint32_t kAttnOver = 6;

typedef unsigned long long attn_u64;

// Positions [lo, hi] that position pos of a sequence sees; hi < lo: none.
__device__ __forceinline__ void attn_range(const AttnArgs& a, bool seq_in, int32_t pos, int32_t* lo, int32_t* hi) {
  const bool in = seq_in && (uint32_t)pos < a.t.positions;
  *hi = in ? pos : -1;
  *lo = in && a.window && (uint32_t)pos >= a.window ? pos - (int32_t)a.window + 1 : 0;
}
// Whether token r goes on where the one before it ends, and shares its tile.
__device__ __forceinline__ bool attn_follows(const AttnArgs& a, uint32_t r, int32_t seq, int32_t pos, int32_t seq_before,
                                             int32_t pos_before) {
  return (r & (a.together - 1)) && seq == seq_before && pos_before != 0x7FFFFFFF && pos == pos_before + 1;
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, uint32_t lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}
__device__ __forceinline__ attn_u64 lane_u64(attn_u64 v, uint32_t lane) {
  return (attn_u64)lane_u32((uint32_t)(v >> 32), lane) << 32 | lane_u32((uint32_t)v, lane);
}

// Sixty-four tokens, one per lane. Tokens of one sequence at positions that
// follow one another share a tile, up to `together` (a power of two) from a
// multiple of it on: the lane of the first has their number and their units.
struct AttnChunk {
  uint32_t first;    // token of lane 0
  int32_t seq, pos;
  uint32_t n, units;  // kAttnOver among them; 0: sees nothing
  attn_u64 before;   // units of the lanes before, from the chunk's start
  bool wrong;        // out of range
  __device__ void load(const AttnArgs& a, uint32_t from) {
    const uint32_t lane = threadIdx.x & 63, r = from + lane;
    const bool in = r < a.t.n;
    first = from;
    seq = in ? a.t.seq[r] : -1;
    pos = in ? a.t.pos[r] : 0;
    const int32_t s = __shfl_up(seq, 1, kWave), p = __shfl_up(pos, 1, kWave);
    const bool follows = in && attn_follows(a, r, seq, pos, s, p);
    const attn_u64 mask = __ballot(follows);
    n = follows || !in ? 0u : (uint32_t)__builtin_ctzll(~((mask >> 1) >> lane)) + 1;
    const bool seq_in = (uint32_t)seq < a.t.n_seqs;
    wrong = in && seq != -1 && !(seq_in && (uint32_t)pos < a.t.positions);
    int32_t lo, hi;
    attn_range(a, seq_in && n, max(pos, 0), &lo, &hi);
    hi = min((int32_t)((uint32_t)pos + n - 1), (int32_t)a.t.positions - 1);  // pos + n may pass 2^31
    units = seq_in && n && hi >= max(pos, 0) ? (uint32_t)hi / kAttnUnit - (uint32_t)lo / kAttnUnit + 1 + kAttnOver : 0u;
    before = wave_scan_u64(units) - units;
  }
  __device__ attn_u64 all() const { return lane_u64(before + units, 63); }
};

// One block's part of a group's tile: units [first, first + count) of its positions'.
struct AttnPart {
  uint32_t row, n, tile, first, count;
  int32_t seq, pos;
  bool whole, begun;  // all of the group's units; units before them are another block's
};

// Block b takes the units from attn_from(all, b) to attn_from(all, b + 1): as many
// as the others or one more, one each where there are fewer than blocks.
__device__ __forceinline__ attn_u64 attn_from(attn_u64 units, uint32_t block, uint32_t blocks_log) {
  return units >> blocks_log ? (units * block) >> blocks_log : min((attn_u64)block, units);
}
// The block that has unit x: the last that begins at or before it.
__device__ __forceinline__ uint32_t attn_block_of(attn_u64 x, attn_u64 units, uint32_t blocks_log) {
  if (!(units >> blocks_log)) return (uint32_t)x;
  const attn_u64 y = ((x + 1) << blocks_log) - 1;
  return (y | units) >> 32 ? (uint32_t)(y / units) : (uint32_t)y / (uint32_t)units;
}

// A block's place in the list of units, the same in all of its waves.
struct AttnPlan {
  AttnChunk chunk;    // of tokens, in which unit x lies
  attn_u64 chunk_at;  // units before it
  attn_u64 x, end;    // the block's units (times tiles) still to come
  uint32_t tiles;     // of a group

  // All waves of a block: whether the block has any units. chunk_units: LDS, one per
  // chunk. Block 0 also leaves the units before every token, and finds tokens out
  // of range.
  __device__ __forceinline__ bool begin(const AttnArgs& a, attn_u64* chunk_units) {
    const uint32_t t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t n = a.t.n, blk = blockIdx.x;
    tiles = a.c.heads * a.parts;
    chunk_at = 0;
    attn_u64 all;
    if (n <= 64) {
      chunk.load(a, 0);
      all = chunk.all();
      x = attn_from(all * tiles, blk, a.blocks_log);
      end = attn_from(all * tiles, blk + 1, a.blocks_log);
      if (blk == 0 && wave == 0) {
        if (lane < n) a.before[lane] = chunk.before;
        if (lane == 0) a.before[n] = all;
        if (chunk.wrong) *a.err = 2u;
      }
      return x < end;
    }
    const uint32_t chunks = (n + 63) / 64;
    for (uint32_t c = wave; c < chunks; c += 4) {
      chunk.load(a, c * 64);
      const attn_u64 units = chunk.all();
      if (lane == 0) chunk_units[c] = units;
      if (blk == 0 && chunk.wrong) *a.err = 2u;
    }
    __syncthreads();
    attn_u64 u[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += u[j] = 4 * lane + j < chunks ? chunk_units[4 * lane + j] : 0ull;
    const attn_u64 upto = wave_scan_u64(sum);
    all = lane_u64(upto, 63);
    x = attn_from(all * tiles, blk, a.blocks_log);
    end = attn_from(all * tiles, blk + 1, a.blocks_log);
    // Lane l has the units before chunks 4 l to 4 l + 3. (Not written over
    // chunk_units, which other waves may still be reading.)
    attn_u64 before = upto - sum, own = 0;  // own: before chunk 4 l + wave
    uint32_t c = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (j == wave) own = before;
      const attn_u64 here = __ballot(before * tiles <= x && x < (before + u[j]) * tiles);
      if (here) {
        const uint32_t l = (uint32_t)__builtin_ctzll(here);
        c = 4 * l + j;
        chunk_at = lane_u64(before, l);
      }
      before += u[j];
    }
    if (blk == 0) {
      for (uint32_t i = wave; i < chunks; i += 4) {
        chunk.load(a, i * 64);
        const attn_u64 at = lane_u64(own, i / 4);
        if (i * 64 + lane < n) a.before[i * 64 + lane] = at + chunk.before;
      }
      if (t == 0) a.before[n] = all;
    }
    if (x >= end) return false;
    chunk.load(a, c * 64);
    return true;
  }

  // The next part from unit x on, x then behind it; false: there is none.
  __device__ __forceinline__ bool next(const AttnArgs& a, AttnPart& p) {
    while (x < end) {
      const attn_u64 at = (chunk_at + chunk.before) * tiles;
      const attn_u64 here = __ballot(at <= x && x < at + (attn_u64)chunk.units * tiles);
      if (!here) {
        // (Not behind the last token, should positions change meanwhile.)
        if (chunk.first + 64 >= a.t.n) return false;
        chunk_at += chunk.all();
        chunk.load(a, chunk.first + 64);
        continue;
      }
      const uint32_t l = (uint32_t)__builtin_ctzll(here), units = lane_u32(chunk.units, l);
      const attn_u64 off = x - lane_u64(at, l);
      p.tile = off >> 32 ? (uint32_t)(off / units) : (uint32_t)off / units;
      const uint32_t from = (uint32_t)(off - (attn_u64)p.tile * units);
      const uint32_t to = (uint32_t)min((attn_u64)units, from + (end - x));
      x += to - from;
      if (to <= kAttnOver) continue;
      p.row = chunk.first + l;
      p.n = lane_u32(chunk.n, l);
      p.seq = (int32_t)lane_u32((uint32_t)chunk.seq, l);
      p.pos = (int32_t)lane_u32((uint32_t)chunk.pos, l);
      p.begun = from > kAttnOver;
      p.first = p.begun ? from - kAttnOver : 0u;
      p.count = to - kAttnOver - p.first;
      p.whole = !p.begun && to == units;
      return true;
    }
    return false;
  }
};

}  // namespace smoe

// The attention's plan (streamoe_amd/csrc/attn_plan.h) on the host: what every
// wave of every block takes, against the definition — groups of tokens, their
// units of 32 positions, block after block an equal part of the list.
#include "block_emu.h"

#include "../../streamoe_amd/csrc/attn_plan.h"

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <map>
#include <random>

using namespace smoe;

static int failures = 0;
#define CHECK(c, ...)                      \
  do {                                     \
    if (!(c)) {                            \
      if (++failures <= 20) {              \
        printf("%s:%d %s: ", __func__, __LINE__, #c); \
        printf(__VA_ARGS__);               \
        printf("\n");                      \
      }                                    \
    }                                      \
  } while (0)

struct Group {
  uint32_t row, n;
  int64_t lo, hi;  // of the positions that its tokens see; hi < lo: none
  uint64_t positions_units() const { return hi < lo ? 0 : hi / kAttnUnit - lo / kAttnUnit + 1; }
};

static std::vector<Group> groups_of(const AttnArgs& a) {
  std::vector<Group> out;
  for (uint32_t r = 0; r < a.t.n;) {
    uint32_t n = 1;
    while (r + n < a.t.n && (r + n) % a.together && a.t.seq[r + n] == a.t.seq[r] && (int64_t)a.t.pos[r + n] == (int64_t)a.t.pos[r] + n) ++n;
    Group g{r, n, INT64_MAX, -1};
    for (uint32_t i = r; i < r + n; ++i) {
      const int64_t s = a.t.seq[i], p = a.t.pos[i];
      if (s < 0 || s >= a.t.n_seqs || p < 0 || p >= a.t.positions) continue;
      g.lo = std::min(g.lo, a.window ? std::max<int64_t>(0, p - a.window + 1) : 0);
      g.hi = std::max(g.hi, p);
    }
    out.push_back(g);
    r += n;
  }
  return out;
}

struct Taken {
  uint32_t block;
  AttnPart p;
};
static bool same(const AttnPart& a, const AttnPart& b) {
  return a.row == b.row && a.n == b.n && a.tile == b.tile && a.first == b.first && a.count == b.count && a.seq == b.seq &&
         a.pos == b.pos && a.whole == b.whole && a.begun == b.begun;
}

static void check_plan(const char* what, AttnArgs a, const std::vector<int32_t>& seq, const std::vector<int32_t>& pos,
                       const int (&waves)[4]) {
  a.t.seq = seq.data();
  a.t.pos = pos.data();
  a.t.n = (uint32_t)seq.size();
  std::vector<uint64_t> before(a.t.n + 1, ~0ull);
  uint32_t err = 0;
  a.before = before.data();
  a.err = &err;
  const std::vector<Group> groups = groups_of(a);
  const uint64_t tiles = a.c.heads * a.parts;
  uint64_t all = 0;
  for (const Group& g : groups) all += g.positions_units() ? g.positions_units() + kAttnOver : 0;
  std::map<std::pair<uint32_t, uint32_t>, std::vector<Taken>> taken;  // by row and tile
  for (uint32_t b = 0; b < 1u << a.blocks_log; ++b) {
    emu::block_id.x = b;
    std::vector<AttnPart> parts[emu::kThreads];
    attn_u64 chunk_units[kKvMaxTokens / 64];
    memset(chunk_units, 0xFF, sizeof chunk_units);
    const bool ok = emu::run(waves, [&] {
      AttnPlan plan;
      if (!plan.begin(a, chunk_units)) return;
      const uint32_t t = threadIdx.x;
      AttnPart p;
      while (parts[t].size() < 100000 && plan.next(a, p)) parts[t].push_back(p);
    });
    CHECK(ok, "%s block %u: barriers or exchanges that do not match", what, b);
    if (!ok) return;
    for (int t = 1; t < emu::kThreads; ++t) {
      bool eq = parts[t].size() == parts[0].size();
      for (size_t i = 0; eq && i < parts[0].size(); ++i) eq = same(parts[t][i], parts[0][i]);
      CHECK(eq, "%s block %u: thread %d has other parts than thread 0", what, b, t);
      if (!eq) return;
    }
    for (const AttnPart& p : parts[0]) taken[{p.row, p.tile}].push_back({b, p});
  }
  uint64_t at = 0;
  size_t used = 0;
  bool wrong = false;
  for (uint32_t r = 0; r < a.t.n; ++r) {
    const int64_t s = seq[r], p = pos[r];
    wrong |= s != -1 && (s < 0 || s >= a.t.n_seqs || p < 0 || p >= a.t.positions);
  }
  CHECK((err == 2) == wrong, "%s: error word %u", what, err);
  for (const Group& g : groups) {
    const uint64_t units = g.positions_units();
    CHECK(before[g.row] == at, "%s: units before row %u: %llu, not %llu", what, g.row, (unsigned long long)before[g.row], (unsigned long long)at);
    if (!units) continue;
    for (uint32_t tile = 0; tile < tiles; ++tile) {
      const auto i = taken.find({g.row, tile});
      CHECK(i != taken.end(), "%s: row %u tile %u is nobody's", what, g.row, tile);
      if (i == taken.end()) return;
      ++used;
      const std::vector<Taken>& list = i->second;
      const uint64_t x = at * tiles + tile * (units + kAttnOver) + kAttnOver, total = all * tiles;
      CHECK(list.front().block == attn_block_of(x, total, a.blocks_log) && list.back().block == attn_block_of(x + units - 1, total, a.blocks_log),
            "%s: row %u tile %u: other blocks than the join's", what, g.row, tile);
      uint64_t from = 0;
      for (size_t j = 0; j < list.size(); ++j) {
        const AttnPart& p = list[j].p;
        CHECK(p.first == from && p.count && p.n == g.n && p.seq == seq[g.row] && p.pos == pos[g.row] && p.begun == (j > 0) &&
                  p.whole == (list.size() == 1) && list[j].block == list[0].block + j,
              "%s: row %u tile %u part %zu", what, g.row, tile, j);
        from += p.count;
      }
      CHECK(from == units, "%s: row %u tile %u: %llu units of %llu", what, g.row, tile, (unsigned long long)from, (unsigned long long)units);
    }
    at += units + kAttnOver;
  }
  CHECK(used == taken.size(), "%s: parts of rows that are no group's first or see nothing", what);
  CHECK(before[a.t.n] == at && at == all, "%s: all units", what);
}

static void plans(unsigned seed) {
  std::mt19937 rng(seed);
  auto in = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
  const int orders[][4] = {{0, 1, 2, 3}, {1, 0, 3, 2}, {3, 2, 1, 0}, {2, 3, 0, 1}};
  const uint32_t sizes[] = {1, 3, 64, 65, 129, 330};
  for (uint32_t n : sizes) {
    AttnArgs a{};
    a.blocks_log = (uint32_t)in(2, 3);
    const uint32_t group = (uint32_t)in(1, 40);
    a.c.heads = (uint32_t)in(1, 2);
    a.parts = (group + 15) / 16;
    a.together = 1;
    while (a.together * 2 * group <= 16) a.together *= 2;
    a.t.n_seqs = 6;
    a.t.positions = 5000;
    a.window = in(0, 1) ? 0 : (uint32_t)in(1, 900);
    std::vector<int32_t> seq(n), pos(n);
    for (uint32_t r = 0; r < n; ++r) {
      if (r && in(0, 9) < 7) {  // a run
        seq[r] = seq[r - 1];
        pos[r] = pos[r - 1] + 1;
        continue;
      }
      const int64_t kind = in(0, 19);
      seq[r] = kind == 0 ? -1 : kind == 1 ? (int32_t)in(6, 9) : kind == 2 ? -5 : (int32_t)in(0, 5);
      pos[r] = kind == 3 ? -2 : kind == 4 ? 4998 : (int32_t)in(0, in(0, 1) ? 40 : 4999);
    }
    char what[64];
    for (const auto& order : orders) {
      if (n > 300 && order[0] > 0) break;
      snprintf(what, sizeof what, "seed %u, %u tokens, wave %d first", seed, n, order[0]);
      check_plan(what, a, seq, pos, order);
    }
  }
  // Positions next to the largest number, alone, in runs, and before others.
  for (uint32_t together : {1u, 2u, 16u}) {
    AttnArgs a{};
    a.blocks_log = 2;
    a.c.heads = a.parts = 1;
    a.together = together;
    a.t.n_seqs = 2;
    a.t.positions = 1u << 30;
    const std::vector<int32_t> seq = {0, 0, 0, 1, 1, 1, 1, -1, 0, 0, 1};
    const std::vector<int32_t> pos = {INT32_MAX, INT32_MAX - 1, INT32_MAX, 100, INT32_MIN, INT32_MIN + 1, INT32_MAX, 0, -1, 0, (1 << 30) - 1};
    check_plan("positions that are far", a, seq, pos, orders[0]);
    a.t.positions = 4096;
    a.window = 100;
    check_plan("positions that are far, a window", a, seq, pos, orders[0]);
  }
  // Nothing but padding, and one row that sees something behind it.
  for (uint32_t n : {5u, 64u, 65u, 300u}) {
    AttnArgs a{};
    a.blocks_log = 3;
    a.c.heads = 2;
    a.parts = a.together = 1;
    a.t.n_seqs = 2;
    a.t.positions = 4096;
    std::vector<int32_t> seq(n, -1), pos(n, 0);
    check_plan("padding", a, seq, pos, orders[0]);
    seq[n - 1] = 1;
    pos[n - 1] = 3000;
    check_plan("padding but for the last", a, seq, pos, orders[0]);
  }
}

// attn_block_of against attn_from, whose blocks are wide integers' quotients: units
// next to the blocks' borders and far from them, totals of few units to the most
// that a call can have (16384 rows of 2^30 positions and 482 tiles each, below 2^49).
static void blocks() {
  std::mt19937_64 rng(1);
  std::vector<uint64_t> totals = {1, 255, 256, 257, 511, 512, 513, 70001, (1ull << 32) + 786432, (1ull << 32) + 5000};
  for (int bit = 20; bit <= 48; ++bit)
    for (int64_t off : {-513, -1, 0, 1, 2, 511, 512}) totals.push_back((1ull << bit) + (uint64_t)off);
  for (int i = 0; i < 500; ++i) totals.push_back(1 + (rng() >> (15 + rng() % 48)));
  for (uint64_t total : totals)
    for (uint32_t log : {8u, 9u}) {
      const uint32_t n = 1u << log;
      std::vector<uint64_t> units;
      for (uint32_t b = 0; b <= n; ++b) {
        const uint64_t from = attn_from(total, b, log);
        const uint64_t want = total < n ? std::min<uint64_t>(b, total) : (uint64_t)((unsigned __int128)total * b >> log);
        CHECK(from == want, "total %llu block %u", (unsigned long long)total, b);
        for (uint64_t x : {from - 1, from, from + 1}) units.push_back(x);
      }
      for (int i = 0; i < 2000; ++i) units.push_back(rng() >> (rng() % 64));
      for (uint64_t x : units) {
        if (x >= total) continue;
        const uint32_t b = attn_block_of(x, total, log);
        CHECK(b < n && attn_from(total, b, log) <= x && x < attn_from(total, b + 1, log), "unit %llu of %llu: block %u of %u",
              (unsigned long long)x, (unsigned long long)total, b, n);
      }
    }
}

int main(int argc, char** argv) {
  for (int i = 1; i < argc; ++i) {
    if (!strcmp(argv[i], "blocks"))
      blocks();
    else
      plans((unsigned)atoi(argv[i]));
  }
  printf("failures=%d\n", failures);
  return failures != 0;
}

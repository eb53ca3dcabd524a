// Host checks of the paged cache's index arithmetic (csrc/paged_model.hpp): page numbers against plain
// division, and a sequence's rows and visible keys under offsets and lengths of any value.
#include "paged_model.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#define CHECK(x)                                                        \
  do {                                                                  \
    if (!(x)) {                                                         \
      std::printf("line %d: %s\n", __LINE__, #x);                       \
      std::exit(1);                                                     \
    }                                                                   \
  } while (0)

static uint32_t rnd() {
  static uint64_t s = 88172645463325252ull;
  s ^= s << 13, s ^= s >> 7, s ^= s << 17;
  return (uint32_t)(s >> 16);
}

// Every step of every tile belongs to exactly one workgroup, in order; a tile's parts after its first are the
// first segments of the workgroups that follow, as the join of partial results takes them.
static void check_work() {
  for (int round = 0; round < 3000; ++round) {
    const int group = 1 + rnd() % 20, rows = 16 << rnd() % 4, seqs = 1 + rnd() % 12, kv_heads = 1 + rnd() % 4;
    const int capacity = 1 + rnd() % 3000, n = 1 + rnd() % 40, min_units = 128;
    const bool causal = rnd() % 2, whole = rnd() % 4 == 0, wild = rnd() % 8 == 0;
    const pa::TileShape tiles = pa::make_tiles(group, rows);
    CHECK(tiles.heads * tiles.tokens <= rows && tiles.heads * tiles.splits >= group);
    pa::SeqRows seq[12];
    int first = 0;
    for (int s = 0; s < seqs; ++s) {
      const int count = rnd() % 3 == 0 ? 0 : rnd() % 3 ? 1 : rnd() % 300;
      const int length = wild ? rnd() % 2000 : count + rnd() % 2500;
      seq[s] = {first, count, length};
      first += count;
    }
    const int heads = kv_heads * tiles.splits;
    int64_t total = 0;
    for (int s = 0; s < seqs; ++s) total += heads * pa::tiles_cost(seq[s], tiles, causal, pa::tiles_of(seq[s], tiles));
    const int active = (int)(total / min_units < 1 ? 1 : total / min_units < n ? total / min_units : n);
    // the tile that the next segment must continue or begin
    int s = 0, head = 0, tile = 0, step = 0;
    auto skip_empty = [&] { while (s < seqs && seq[s].count == 0) ++s; };
    skip_empty();
    for (int w = 0; w < active; ++w) {
      const int64_t at = pa::share_of(total, active, w), end = pa::share_of(total, active, w + 1);
      pa::WorkWalk walk{tiles, seqs, heads, capacity, causal, whole, at, end, 0, 0};
      for (int i = 0; i < seqs; ++i) {   // the sequence that holds `at`
        const int64_t all = heads * pa::tiles_cost(seq[i], tiles, causal, pa::tiles_of(seq[i], tiles));
        if (walk.begin + all > at) break;
        walk.begin += all;
        walk.seq = i + 1;
      }
      pa::Segment g;
      bool head_of_list = true;
      while (walk.next([&](int i) { return seq[i]; }, g)) {
        CHECK(g.seq == s && g.head == head && g.tile == tile && g.from == step && g.from < g.to && g.to <= g.steps);
        CHECK(g.steps == pa::tile_steps(seq[s], tiles, tile, capacity, causal));
        CHECK(g.from == 0 || (head_of_list && !whole));
        head_of_list = false;
        step = g.to;
        if (step == g.steps) {
          step = 0;
          if (++tile == pa::tiles_of(seq[s], tiles)) {
            tile = 0;
            if (++head == heads) head = 0, ++s, skip_empty();
          }
        }
      }
      CHECK(step == 0 || !head_of_list);   // an unfinished tile is continued by the very next workgroup
    }
    CHECK(s == seqs && head == 0 && tile == 0 && step == 0);
  }
}

int main() {
  const uint32_t top = 1u << 30;
  auto check_div = [&](uint32_t d) {
    const pa::PageDiv p = pa::make_page_div(d);
    auto one = [&](uint64_t n) { CHECK(n >= 2ull * top || pa::page_of((uint32_t)n, p) == n / d); };
    for (uint64_t n = 0; n < 200; ++n) one(n);
    for (uint64_t q = 1; q * d < 2ull * top && q < 300; ++q) one(q * d - 1), one(q * d), one(q * d + 1);
    for (int i = 0; i < 200; ++i) one(rnd() % (2ull * top));
    one(2ull * top - 1), one(2ull * top - 2), one((2ull * top - 1) / d * d), one((2ull * top - 1) / d * d - 1);
  };
  for (uint32_t d = 1; d < 5000; ++d) check_div(d);
  for (int i = 0; i < 5000; ++i) check_div(rnd() % top + 1);
  for (uint32_t d : {top, top - 1, top / 2, top / 2 + 1, 65535u, 65536u, 65537u}) check_div(d);

  const int odd[] = {INT32_MIN, INT32_MIN + 1, -1000, -1, 0, 1, 2, 7, 63, 64, 1000, (1 << 30) - 1, 1 << 30, INT32_MAX};
  for (int tokens : {1, 2, 64, 1000, 1 << 30})
    for (int b : odd)
      for (int e : odd)
        for (int len : odd) {
          const pa::SeqRows s = pa::seq_rows(b, e, len, tokens);
          CHECK(s.first >= 0 && s.count >= 0 && (int64_t)s.first + s.count <= tokens && s.length >= 0);
          for (int cap : {1, 64, 1 << 30})
            for (int i : {0, s.count / 2, s.count - 1}) {
              if (i < 0) continue;
              const int64_t pos = (int64_t)s.length - s.count + i;
              CHECK(pa::new_token_pos(s, i) == pos);
              const int64_t c = pos + 1 < 0 ? 0 : pos + 1 > cap ? cap : pos + 1;
              CHECK(pa::keys_seen(s, i, cap, true) == c);
              CHECK(pa::keys_seen(s, i, cap, false) == (s.length < cap ? s.length : cap));
            }
        }
  check_work();
  std::printf("ok\n");
  return 0;
}

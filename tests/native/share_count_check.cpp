// The workgroups that take shares of a call (csrc/paged_model.hpp), and what they get, on the host.
#include <cstdio>
#include <random>
#include <vector>

#include "paged_model.hpp"

using namespace pa;

static bool fail(const char* what, int64_t a, int64_t b) { return std::printf("%s: %lld %lld\n", what, (long long)a, (long long)b), false; }

// Every tile's steps are taken once; returns the most units of a workgroup and the number of tiles that are cut.
static bool divide(const std::vector<SeqRows>& seqs, int heads, const TileShape& t, int capacity, bool whole, int min_units, int grid,
                   int& active, int64_t& most, int& cut) {
  int64_t total = 0, tiles = 0;
  std::vector<int64_t> begins;
  for (const SeqRows& r : seqs) {
    begins.push_back(total);
    total += heads * tiles_cost(r, t, false, tiles_of(r, t)), tiles += (int64_t)heads * tiles_of(r, t);
  }
  active = share_count(total, tiles, min_units, grid);
  int64_t steps = 0, want = 0;
  for (const SeqRows& r : seqs)
    for (int i = 0; i < tiles_of(r, t); ++i) want += heads * (int64_t)tile_steps(r, t, i, capacity, false);
  most = 0, cut = 0;
  for (int w = 0; w < active; ++w) {
    const int64_t at = share_of(total, active, w), end = share_of(total, active, w + 1);
    int seq = 0;
    while (seq + 1 < (int)seqs.size() && begins[seq + 1] <= at) ++seq;
    WorkWalk walk{t, (int)seqs.size(), heads, capacity, false, whole, at, end, begins[seq], seq};
    Segment s;
    int64_t units = 0;
    while (walk.next([&](int i) { return seqs[i]; }, s)) {
      steps += s.to - s.from;
      cut += s.from == 0 && s.to < s.steps;
      units += (s.from == 0 ? kTileCost : 0) + (s.to - s.from) * kStep;
    }
    most = units > most ? units : most;
  }
  return steps == want || fail("steps", steps, want);
}

int main() {
  // At least one workgroup, at most the grid, one for each tile whatever min_units is, min_units each where tiles are large.
  for (int grid : {1, 7, 256, 512})
    for (int64_t tiles : {0, 1, 5, 114, 256, 100000})
      for (int64_t each : {256, 300, 456, 1023, 5000})
        for (int least : {128, 512, 1024}) {
          const int64_t total = tiles * each, n = share_count(total, tiles, least, grid);
          const int64_t want = std::max<int64_t>(1, std::min<int64_t>(grid, std::max(tiles, total / least)));
          if (n != want) return fail("count", n, want), 1;
        }
  if (share_count((int64_t)1 << 62, 1 << 30, 1024, 512) != 512) return fail("large", 0, 0), 1;
  // 32 sequences of 48 tokens and 200 keys, 8 heads of 4: 256 tiles of 256 rows, one a workgroup, none cut.
  int active, cut;
  int64_t most;
  if (!divide(std::vector<SeqRows>(32, SeqRows{0, 48, 200}), 8, make_tiles(4, 256), 8192, false, 1024, 256, active, most, cut)) return 1;
  if (active != 256 || cut != 0 || most != kTileCost + 7 * kStep) return fail("short", active, most), 1;
  // Short ones of any lengths: no workgroup has more than the longest tile and a step.
  std::mt19937 rng(1);
  for (int n = 0; n < 200; ++n) {
    std::vector<SeqRows> seqs(1 + rng() % 40);
    int64_t longest = 0;
    for (SeqRows& r : seqs) {
      r = {0, (int)(rng() % 65), (int)(rng() % 700)};
      r.length = std::max(r.length, r.count);
      if (r.count) longest = std::max<int64_t>(longest, kTileCost + (r.length + kStep - 1) / kStep * kStep);
    }
    const int heads = 1 + rng() % 6;
    for (bool whole : {false, true}) {
      if (!divide(seqs, heads, make_tiles(4, 256), 8192, whole, 1024, 256, active, most, cut)) return 1;
      if (active < 256 && !whole && most > longest + kTileCost + 2 * kStep) return fail("share", most, longest), 1;
      if (whole && cut) return fail("whole", cut, 0), 1;
    }
  }
  std::puts("ok");
}

// The index arithmetic of the paged key/value cache, shared by the kernels, the launchers and the host
// tests: page numbers by multiplication, and a sequence's rows and visible keys under the clamps that keep
// every access inside its tensor whatever the page table, lengths and offsets hold.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

// Sizes the launchers admit: capacities, rows of new tokens and page sizes are at most 2^30, so that one of them and
// a tile's more fits 31 bits (two of 2^30 do not); the rows of a cache (pages x heads x page size) stay below 2^31.
constexpr int64_t kPagedMaxPos = 1ll << 30;

// pos / page_size as a multiplication: with L = ceil(log2 d) and magic = floor(2^(31+L) / d) + 1,
// (pos * magic) >> (31 + L) is the quotient for every pos < 2^31 (the excess of magic * d over 2^(31+L) is
// at most 2^L).
struct PageDiv {
  uint32_t magic;
  int shift;
};
__host__ inline PageDiv make_page_div(uint32_t d) {
  int shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {(uint32_t)(((1ull << (31 + shift)) / d) + 1), shift};
}
__host__ __device__ __forceinline__ uint32_t page_of(uint32_t pos, PageDiv p) {
  return (uint32_t)(((uint64_t)(pos << 1) * p.magic) >> 32) >> p.shift;
}

__host__ __device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// A sequence's new tokens: rows [first, first + count) of the packed tensors, the cache's capacity for it
// and its length after the call. Offsets outside [0, tokens] or out of order give fewer rows, never others
// than the tensor has; a negative length counts as 0.
struct SeqRows {
  int first, count, length;
};
__host__ __device__ __forceinline__ SeqRows seq_rows(int begin, int end, int length, int tokens) {
  const int b = clamp_int(begin, 0, tokens), e = clamp_int(end, b, tokens);
  return {b, e - b, clamp_int(length, 0, (int)kPagedMaxPos)};
}
// The rows as the work is counted and divided by: a longer sequence has its new tokens past the capacity too, and every
// key that it sees below it, at the length capacity + count: the same rows and keys, but no more work than the launcher
// admits. (Compared by the difference: both summands may be 2^30.)
__host__ __device__ __forceinline__ SeqRows held_rows(SeqRows s, int capacity) {
  if (s.length - s.count > capacity) s.length = capacity + s.count;
  return s;
}
// Position in the cache of the sequence's new token i; below 0 or past the table's columns it has none.
__host__ __device__ __forceinline__ int new_token_pos(const SeqRows& s, int i) { return s.length - s.count + i; }
// Keys that new token i sees: those up to its own position (causal) or the sequence's, and never more than
// the table has columns for.
__host__ __device__ __forceinline__ int keys_seen(const SeqRows& s, int i, int capacity, bool causal) {
  return clamp_int(causal ? new_token_pos(s, i) + 1 : s.length, 0, capacity);
}

// 32 bits of a mask over a sequence's new tokens from its bit j0 on, bit i for new token j0 + i: ones before the first (the
// sequence's earlier keys, which all of them see), zeros past its `words` words. word(i) gives word i.
template <typename Word>
__host__ __device__ __forceinline__ uint32_t mask_window(int j0, int words, Word word) {
  const int i = j0 >> 5;   // (rounded down)
  const uint32_t lo = i < 0 ? ~0u : i < words ? word(i) : 0u, hi = i + 1 < 0 ? ~0u : i + 1 < words ? word(i + 1) : 0u;
  return (uint32_t)(((uint64_t)hi << 32 | lo) >> (j0 & 31));
}

// ---- Work of an attention call, and its division over workgroups ----
//
// A tile is up to `rows` query rows that read the same keys: `heads` query heads of one key/value head times
// `tokens` consecutive new tokens of one sequence. Tiles are counted sequence by sequence, head by head, token
// by token; each costs about as many units as it has keys to read (closed forms, so that a workgroup finds its
// place without a list). Workgroup w of n takes the units [share(w), share(w + 1)): the same number for every
// workgroup whatever the lengths are, cut at steps of kStep keys. What a cut leaves of a tile are partial
// results, joined afterwards.
constexpr int kStep = 32;       // keys of a step
// Units a tile costs beside its keys: its queries, its first keys on their way, its result, in the time of keys.
// Counted as 64, 256 and 512 keys: 24 x 700 tokens over 4096 keys, D = 128, e4m3 595, 520 and 531 us; 16 x 16 over
// 4096, D = 64, int8 37, 34 and 32; 256 x 1 over 1000 144, 126 and 130; one over 1031 does not see it.
constexpr int kTileCost = 256;
// Least units of a workgroup: a step for each of four waves. With 64 and 256, 2 x 5 tokens over 4096 take 27 and 22
// us, 2 x 100 over 900 take 32 and 31 (128: 22 and 27), one over 1031 the same.
constexpr int kMinUnits = 128;

struct TileShape {
  int group, heads, tokens, splits;   // query heads per key/value head; of a tile; tokens of a tile; tiles that cover the group
};
__host__ __device__ __forceinline__ TileShape make_tiles(int group, int rows) {
  const int heads = group < rows ? group : rows;
  return {group, heads, rows / heads, (group + heads - 1) / heads};
}
__host__ __device__ __forceinline__ int tiles_of(const SeqRows& s, const TileShape& t) {
  return (s.count + t.tokens - 1) / t.tokens;
}
// Units of a sequence's first n tiles (n at most tiles_of) of one head. A causal tile counts the keys up to its
// last token's; only the last tile can have fewer tokens than the others.
__host__ __device__ __forceinline__ int64_t tiles_cost(const SeqRows& s, const TileShape& t, bool causal, int64_t n) {
  const int before = s.length - s.count;
  int64_t cost = n * (kTileCost + (causal ? (before > 0 ? before : 0) : s.length));
  if (causal) {
    const int64_t full = n < s.count / t.tokens ? n : s.count / t.tokens;
    cost += t.tokens * (full * (full + 1) / 2) + (n > full ? s.count : 0);
  }
  return cost;
}
// Steps of a tile: those with a key that its last token sees, and one if there is none.
__host__ __device__ __forceinline__ int tile_steps(const SeqRows& s, const TileShape& t, int tile, int capacity, bool causal) {
  const int last = (tile + 1) * (int64_t)t.tokens < s.count ? (tile + 1) * t.tokens - 1 : s.count - 1;
  const int keys = keys_seen(s, last, capacity, causal);
  return keys == 0 ? 1 : (keys - 1) / kStep + 1;
}
// Workgroups of `grid` that take shares: as many as have min_units units each, but one for each of `tiles` tiles in any case
// (a share of that size cuts none where they are alike).
__host__ __device__ __forceinline__ int share_count(int64_t total, int64_t tiles, int min_units, int grid) {
  const int64_t by_units = total / min_units, most = by_units > tiles ? by_units : tiles;
  return most < 1 ? 1 : most < grid ? (int)most : grid;
}
__host__ __device__ __forceinline__ int64_t share_of(int64_t total, int n, int w) {
  const int64_t each = total / n, rest = total % n;
  return each * w + (w < rest ? w : rest);
}

// A workgroup's part of one tile: steps [from, to) of `steps`; `head` counts key/value heads times splits.
struct Segment {
  SeqRows rows;
  int seq, head, tile, from, to, steps;
};
// The segments of units [at, end). Starts at sequence `seq`, whose units begin at `begin`; load(s) gives a
// sequence's rows. The first segment is searched for, each next one follows from the last without a division.
// whole: tiles are not cut, one belongs to the workgroup whose units hold its first.
struct WorkWalk {
  TileShape tiles;
  int seqs, heads, capacity;   // heads: key/value heads times splits
  bool causal, whole;
  int64_t at, end, begin;      // begin: of the current tile (before the first segment, of the sequence)
  int seq;
  int head = 0, tile = -1, count = 0;   // the current tile, and the sequence's tiles; -1: before the first
  SeqRows rows = {0, 0, 0};

  template <typename Load>
  __host__ __device__ __forceinline__ bool next(Load load, Segment& out) {
    while (at < end) {
      if (tile < 0) {
        rows = load(seq);
        count = tiles_of(rows, tiles);
        if (count == 0) return false;   // (no sequence holds `at`)
        const int64_t per_head = tiles_cost(rows, tiles, causal, count), r = at - begin;
        head = (int)(r / per_head);
        const int64_t in_head = r - head * per_head;
        tile = 0;   // the last tile that begins at or before in_head
        for (int hi = count - 1; tile < hi;) {
          const int mid = tile + (hi - tile + 1) / 2;
          if (tiles_cost(rows, tiles, causal, mid) <= in_head) tile = mid; else hi = mid - 1;
        }
        begin += head * per_head + tiles_cost(rows, tiles, causal, tile);
      } else if (++tile == count) {
        tile = 0;
        if (++head == heads) {
          head = 0;
          do {
            if (++seq >= seqs) return false;
            rows = load(seq);
            count = tiles_of(rows, tiles);
          } while (count == 0);
        }
      }
      const int64_t t0 = begin, last = (int64_t)(tile + 1) * tiles.tokens;
      const int before = rows.length - rows.count;
      const int64_t t1 = t0 + kTileCost + (causal ? (before > 0 ? before : 0) + (last < rows.count ? last : rows.count) : rows.length);
      const int steps = tile_steps(rows, tiles, tile, capacity, causal);
      const int64_t from = at == t0 ? 0 : whole ? steps : (at - t0) / kStep;
      const int64_t to = end >= t1 || whole ? steps : (end - t0) / kStep;
      at = t1 < end ? t1 : end;
      begin = t1;
      if (from < to && from < steps) {
        out = {rows, seq, head, tile, (int)from, (int)(to < steps ? to : steps), steps};
        return true;
      }
    }
    return false;
  }
};

}  // namespace pa

// The index arithmetic of the paged key/value cache, shared by the kernels, the launchers and the host
// tests: page numbers by multiplication, and a sequence's rows and visible keys under the clamps that keep
// every access inside its tensor whatever the page table, lengths and offsets hold.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

// Sizes the launchers admit: positions, rows of new tokens and page sizes stay below 2^30, so sums of two
// fit 32 bits; the rows of a cache (pages x heads x page size) stay below 2^31.
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
// Position in the cache of the sequence's new token i; below 0 or past the table's columns it has none.
__host__ __device__ __forceinline__ int new_token_pos(const SeqRows& s, int i) { return s.length - s.count + i; }
// Keys that new token i sees: those up to its own position (causal) or the sequence's, and never more than
// the table has columns for.
__host__ __device__ __forceinline__ int keys_seen(const SeqRows& s, int i, int capacity, bool causal) {
  return clamp_int(causal ? new_token_pos(s, i) + 1 : s.length, 0, capacity);
}

}  // namespace pa

// The paged key/value cache: rows written into pages (as they are, or in 8 bits with a scale for each token
// and head) and read back.
//
// A cache is [pages][heads][page_size][d]: a page holds page_size tokens of one sequence, and the rows of one
// head in a page are contiguous, which is what attention reads. Position p of sequence s is row p % page_size
// of page page_table[s][p / page_size]. A table entry outside [0, pages) is an absent page: nothing is written
// there, its rows read as zeros and attention does not see its keys.
//
// 8-bit rows: scale = amax / L with L the type's largest value (int8: 127, e4m3: 448), code =
// round(x * (L / amax)) to nearest even, amax the row's largest magnitude; all in fp32. A row below 2^-100 is
// held as zeros (L / amax would leave fp32's range). A row with an element that is not finite gets a NaN
// scale, so it reads as NaN.
#pragma once

#include "../paged_model.hpp"
#include "common.hpp"

namespace pa {

struct i8 { int8_t bits; };       // storage types of the 8-bit caches
struct e4m3 { uint8_t bits; };

template <typename C> struct cache_type {
  static constexpr bool k8bit = false;
  static constexpr float kLargest = 0.f;
};
template <> struct cache_type<i8> {
  static constexpr bool k8bit = true;
  static constexpr float kLargest = 127.f;
};
template <> struct cache_type<e4m3> {
  static constexpr bool k8bit = true;
  static constexpr float kLargest = 448.f;
};

struct PagedCache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int* table;
  const int* lengths;
  const int* cu;          // null: every sequence has `per_seq` new tokens
  int pages, page_size, heads, seqs, cols;
  int tokens, per_seq;    // new tokens of the call
  int capacity;           // cols * page_size
  int64_t table_stride;
  PageDiv div;
};

__device__ __forceinline__ SeqRows load_seq(const PagedCache& c, int s) {
  const int begin = c.cu ? c.cu[s] : s * c.per_seq;
  const int end = c.cu ? c.cu[s + 1] : begin + c.per_seq;
  return held_rows(seq_rows(begin, end, c.lengths[s], c.tokens), c.capacity);
}
// Cache row of position pos (0 <= pos < capacity) of sequence s for head h, -1 if its page is absent.
__device__ __forceinline__ int cache_row(const PagedCache& c, int s, int h, int pos) {
  const int col = (int)page_of((uint32_t)pos, c.div);
  const int page = c.table[s * c.table_stride + col];
  if ((unsigned)page >= (unsigned)c.pages) return -1;
  return (page * c.heads + h) * c.page_size + (pos - col * c.page_size);
}

// The first sequence that has row t, by all lanes of a wave together (t wave-uniform): the first offset at or before t
// whose next one is past it, among 64 offsets a load, against log2(seqs) dependent loads of a search, which offsets out of
// order would mislead. seqs if none has it.
__device__ __forceinline__ int find_seq(const PagedCache& c, int t) {
  if (!c.cu) return t / c.per_seq;
  for (int s0 = 0; s0 < c.seqs; s0 += kWave - 1) {
    const uint64_t begun = __builtin_amdgcn_ballot_w64(c.cu[min(s0 + (int)threadIdx.x % kWave, c.seqs)] <= t);
    const uint64_t has = begun & ~(begun >> 1) & ~(1ull << (kWave - 1));
    if (has) return s0 + __builtin_ctzll(has);
  }
  return c.seqs;
}

// Eight consecutive elements of a cache row in fp32. (A row in 16 bits has no scale.)
__device__ __forceinline__ void cached8(const f16* row, int at, float, float (&x)[8]) {
  const f16x8 v = *reinterpret_cast<const f16x8*>(row + at);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
}
__device__ __forceinline__ void cached8(const bf16* row, int at, float, float (&x)[8]) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(row + at);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
}
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void cached8(const i8* row, int at, float scale, float (&x)[8]) {
  const u32x2 v = *reinterpret_cast<const u32x2*>(row + at);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)(v[j / 4] >> (8 * (j % 4))) * scale;
}
__device__ __forceinline__ void cached8(const e4m3* row, int at, float scale, float (&x)[8]) {
  const u32x2 v = *reinterpret_cast<const u32x2*>(row + at);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[j], false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[j], true);
    x[4 * j] = a[0] * scale, x[4 * j + 1] = a[1] * scale, x[4 * j + 2] = b[0] * scale, x[4 * j + 3] = b[1] * scale;
  }
}

// Eight codes of x * inv.
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], float inv, i8*) {
  u32x2 w = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j / 4] |= ((unsigned)(int)rintf(x[j] * inv) & 0xffu) << (8 * (j % 4));
  return w;
}
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], float inv, e4m3*) {
  u32x2 w;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
    w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, p, true);
  }
  return w;
}

struct RowsIn {
  const void* p;
  int64_t token, head;   // strides in elements
};

// One row (a new token's key or value of one head) per LPR lanes, 16 bytes a lane. Rows of a wave run over
// (token, K or V, head): a token's heads are near each other in the inputs. A row's largest magnitude is a maximum
// over its lanes, without LDS. Small calls are bound by the chain from offsets over lengths
// and page table to the store (32 single tokens: 3.3 us), large ones by bytes: 8 x up to 2048 tokens, 16 heads, D = 64,
// f16, 17.2 us, 4.3 TB/s; 4 x up to 4096, 8 heads, D = 128, bf16 to int8 21.4 us, 2.8 TB/s: the scales of a page and head
// come from as many workgroups, each 4 bytes as a write of 32 (25.0 MB written for 20.6). (Two to eight groups of rows a wave,
// their loads on their way together, are no faster: 18.2 to 24 us and 24 to 27.)
template <typename T, typename C, int D>
__global__ void __launch_bounds__(256) cache_write_rows(PagedCache c, RowsIn kin, RowsIn vin) {
  constexpr int LPR = D / 8, RPW = kWave / LPR;
  const int lane = (int)threadIdx.x % kWave, sub = lane % LPR;
  const int64_t wave = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  const int64_t row0 = wave * RPW, rows = (int64_t)c.tokens * 2 * c.heads;
  int seq = 0, tok = 0, h = 0;
  bool is_v = false, mine = false;
  typedef typename vec8<T>::type V8;
  V8 x;
  // The rows of a wave lie in a few tokens: find each token's sequence with the whole wave.
  {
    const int64_t row = min(row0 + lane / LPR, rows - 1);
    tok = (int)(row / (2 * c.heads));
    const int rest = (int)(row - (int64_t)tok * 2 * c.heads);
    is_v = rest >= c.heads;
    h = is_v ? rest - c.heads : rest;
    mine = row0 + lane / LPR < rows;
    // (Every row may be read, also one that no sequence has: on its way before its place is known.)
    const RowsIn& in = is_v ? vin : kin;
    x = *reinterpret_cast<const V8*>(static_cast<const T*>(in.p) + tok * in.token + h * in.head + 8 * sub);
    int last = -1;
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
      const int t = __builtin_amdgcn_readlane(tok, r * LPR);
      const int s = t == last ? -1 : find_seq(c, t);
      if (s >= 0 && tok == t) seq = s;
      last = t;
    }
  }
  if (!mine || seq >= c.seqs) return;
  const SeqRows s = load_seq(c, seq);
  const int i = tok - s.first;
  if (i < 0 || i >= s.count) return;
  const int pos = new_token_pos(s, i);
  if (pos < 0 || pos >= c.capacity) return;
  const int at = cache_row(c, seq, h, pos);
  if (at < 0) return;
  C* out = static_cast<C*>(is_v ? c.v : c.k) + (int64_t)at * D + 8 * sub;
  if constexpr (!cache_type<C>::k8bit) {
    *reinterpret_cast<V8*>(out) = x;
  } else {
    float f[8], amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = (float)x[j];
      amax = fmaxf(amax, fabsf(f[j]));
      finite = finite && __builtin_isfinite(f[j]);
    }
    // A row's lanes are neighbours: the NaN that marks a row goes through the max as an infinity.
    amax = finite ? amax : INFINITY;
    amax = fmaxf(amax, dpp_move<0xB1>(amax));
    amax = fmaxf(amax, dpp_move<0x4E>(amax));
    amax = fmaxf(amax, dpp_move<0x141>(amax));
    if constexpr (LPR == 16) amax = fmaxf(amax, dpp_move<0x140>(amax));
    const bool some = amax >= 0x1p-100f, ok = amax < INFINITY;
    const float inv = some && ok ? cache_type<C>::kLargest / amax : 0.f;
    if (!ok)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    *reinterpret_cast<u32x2*>(out) = codes8(f, inv, static_cast<C*>(nullptr));
    if (sub == 0) (is_v ? c.v_scale : c.k_scale)[at] = !ok ? NAN : some ? amax / cache_type<C>::kLargest : 0.f;
  }
}

// Rows read back as (seqs, heads, n, D), one row per LPR lanes; zeros from a sequence's length on and for
// absent pages. Grid: x over (sequence, head), y over blocks of rows. Bytes are all it does: 16 sequences of 1 to 8192
// tokens, 8 heads, D = 128, e4m3 (537 MB of results): 148 us, 4.75 TB/s; 102 where the codes are in the memory-side cache.
// STREAM: results past kStreamBytes go by the caches, which could not hold them for a reader: that case took 164 us
// through them with the codes in there, 32 full sequences 350 for 329. Fewer stay in: 67 MB and a sum over them 31 us, past the caches 33.
constexpr int64_t kStreamBytes = 256ll << 20;   // the memory-side cache
template <typename T, typename C, int D, bool STREAM>
__global__ void __launch_bounds__(256) cache_read_rows(PagedCache c, T* k, T* v, int n) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;
  const int s = (int)blockIdx.x / c.heads, h = (int)blockIdx.x % c.heads;
  const int sub = (int)threadIdx.x % LPR;
  typedef typename vec8<T>::type V8;
  const int length = clamp_int(c.lengths[s], 0, c.capacity);
  for (int pos = (int)blockIdx.y * RPB + (int)threadIdx.x / LPR; pos < n; pos += (int)gridDim.y * RPB) {
    const int at = pos < length ? cache_row(c, s, h, pos) : -1;
    const int64_t to = ((int64_t)blockIdx.x * n + pos) * D + 8 * sub;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      V8 o = {};
      if (at >= 0) {
        float x[8], scale = 1.f;
        if constexpr (cache_type<C>::k8bit) scale = (m ? c.v_scale : c.k_scale)[at];
        cached8(static_cast<const C*>(m ? c.v : c.k) + (int64_t)at * D, 8 * sub, scale, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = from_f32<T>(x[j]);
      }
      V8* out = reinterpret_cast<V8*>((m ? v : k) + to);
      if constexpr (STREAM) __builtin_nontemporal_store(o, out); else *out = o;
    }
  }
}

}  // namespace pa

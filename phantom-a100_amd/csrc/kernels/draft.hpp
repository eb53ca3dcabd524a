// Trees of drafted tokens: their masks and positions, their verification against the target's probabilities, and the
// cache rows of the accepted ones.
//
// A sequence's new tokens of a step are a tree: token 0 is the root, which is certain, parents[i] < i is the token that
// token i was drafted behind (-1, or anything that is no earlier token: none). A chain of drafts has parents i - 1. At
// most kTreeMax tokens of a sequence make its tree.
#pragma once

#include "paged_cache.hpp"

namespace pa {

constexpr int kTreeMax = 1024;

// ---- Masks and positions ----
//
// Bit j % 32 of word j / 32 of a token's mask row is set if j is the token itself or one of its ancestors; its position is
// that of the sequence's first new token plus its depth. A thread takes a word of a row and walks up from the token through
// the parents in LDS, as far as nodes of the word can be (parents come before their children).
struct TreeArgs {
  const int* parents;
  const int* lengths;
  const int* cu;             // null: per_seq tokens each
  int tokens, per_seq, most, words;
  int* mask;                 // [token][words]
  int* positions;
};
__global__ void __launch_bounds__(256) draft_tree_rows(TreeArgs a) {
  __shared__ int parent[kTreeMax];
  const int s = (int)blockIdx.x;
  const int begin = a.cu ? a.cu[s] : s * a.per_seq, end = a.cu ? a.cu[s + 1] : begin + a.per_seq;
  const SeqRows r = seq_rows(begin, end, a.lengths[s], a.tokens);
  const int tree = min(r.count, a.most);
  for (int i = (int)threadIdx.x; i < tree; i += 256) {
    const int p = a.parents[r.first + i];
    parent[i] = p < i && p >= 0 ? p : -1;
  }
  __syncthreads();
  const int64_t items = (int64_t)r.count * a.words;
  for (int64_t item = (int64_t)blockIdx.y * 256 + threadIdx.x; item < items; item += (int64_t)gridDim.y * 256) {
    const int i = (int)(item / a.words), w = (int)(item - (int64_t)i * a.words);
    unsigned bits = 0;
    int depth = 0;
    if (i < tree)   // (tokens behind the tree's most see no new token)
      for (int at = i; at >= 32 * w; at = parent[at], ++depth)
        if (at / 32 == w) bits |= 1u << at % 32;
    a.mask[(int64_t)(r.first + i) * a.words + w] = (int)bits;
    if (w == 0) a.positions[r.first + i] = r.length - r.count + max(depth - 1, 0);
  }
}

// ---- Verification ----
//
// From the root on, the drafts behind the current token are tried in order; the first accepted one becomes the current
// token. p and q are the current token's rows of the target's and the draft's probabilities (an element that is not a
// positive finite number counts as 0), u the draft's own random number, t its token:
//   q given: accepted iff u q(t) S(c) < max(p(t) - c q(t), 0), with c = 0 and S(0) = 1 at first; else c grows by S(c), the
//     sum of max(p - c q, 0) over the vocabulary. (After a rejection the target's distribution is max(p - q, 0) / S(1); after
//     the next, max(p / S(1) - (1 / S(1) + 1) q, 0) up to its sum, and so on: always max(p - c q, 0) / S(c).)
//   drafts that are no samples (q null): accepted iff u m < p(t), m = 1 at first; else m falls by p(t), and p(t) is 0 from
//     then on.
// Where no draft is left, the next token is the first one whose sum of weights up to it exceeds u S, u the root's random
// number, S the sum of the weights max(p - c q, 0) (or p without the rejected tokens); if S is 0, p's.
// Sums, products and comparisons are in 64 bits: the next token lies between sums over the whole vocabulary, and in 32 bits
// one draw in a hundred would miss it.
struct VerifyArgs {
  const int64_t* tokens;
  const int* parents;
  const float* p;
  const float* q;            // null: the drafts are no samples
  const float* u;
  const int* cu;
  int64_t p_stride, q_stride;
  int n_tokens, vocab, most, splits;
  int* path;                 // [seqs][most]
  int* accepted;
  int64_t* next;
  struct VerifyState* states;   // [seqs]
  double* sums;              // [seqs][splits]
};
// Where a sequence's path ended: the row of probabilities, c, and the sequence's rows.
struct VerifyState {
  double off;
  int first, tree, node, pad;
};
constexpr int kVerifyChunk = 4096;   // elements of a row that a workgroup sums

__device__ __forceinline__ double weight_of(float x) { return x > 0.f && x < INFINITY ? (double)x : 0.0; }

// What is left of p after `off` times q. (The product is rounded by itself: p - off q is 0 where the two are equal.)
__device__ __forceinline__ double left_of(double p, double off, double q) {
#pragma clang fp contract(off)
  const double x = p - off * q;
  return x > 0 ? x : 0.0;
}

// The sum of x over the workgroup's threads, the same in all of them and in the same order always. lds: 16 numbers.
__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
  const int waves = (int)blockDim.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
  __syncthreads();
  double sum = 0;
  for (int i = 0; i < waves; ++i) sum += lds[i];
  return sum;
}

// What the walk needs of each draft. 20 KB of LDS.
struct Drafts {
  int parent[kTreeMax];      // -1: no draft
  int token[kTreeMax];
  float p[kTreeMax], q[kTreeMax], u[kTreeMax];
};

// The walk of one sequence, by all threads of a workgroup alike. path: where the path goes, null if nowhere. Returns the
// number of accepted tokens.
template <bool DRAWN>
__device__ __forceinline__ int verify_walk(const VerifyArgs& a, int s, Drafts& d, double* lds, int* path, VerifyState& st) {
  const SeqRows r = seq_rows(a.cu[s], a.cu[s + 1], 0, a.n_tokens);
  const int tree = min(r.count, a.most), tid = (int)threadIdx.x, lane = tid % kWave;
  for (int i = tid; i < tree; i += (int)blockDim.x) {
    const int up = a.parents[r.first + i];
    const int64_t t = a.tokens[r.first + i];
    const bool draft = up >= 0 && up < i && t >= 0 && t < a.vocab;
    d.parent[i] = draft ? up : -1;
    d.token[i] = draft ? (int)t : -1;
    d.u[i] = a.u[r.first + i];
    const int64_t row = r.first + (draft ? up : 0);
    const int64_t col = draft ? t : 0;
    d.p[i] = a.p[row * a.p_stride + col];
    if constexpr (DRAWN) d.q[i] = a.q[row * a.q_stride + col];
  }
  __syncthreads();
  if constexpr (!DRAWN) {
    // A token that an earlier draft behind the same token had is rejected already where it is tried.
    for (int i = tid; i < tree; i += (int)blockDim.x)
      if (d.parent[i] >= 0)
        for (int j = d.parent[i] + 1; j < i; ++j)
          if (d.parent[j] == d.parent[i] && d.token[j] == d.token[i]) {
            d.p[i] = 0.f;
            break;
          }
    __syncthreads();
  }
  st = {0.0, r.first, tree, 0, 0};
  if (tree == 0) return 0;
  int accepted = 1;
  double mass = 1.0;
  if (path && tid == 0) path[0] = 0;
  for (int i0 = 0; i0 < tree; i0 += kWave) {
    const int i = i0 + lane, up = i < tree ? d.parent[i] : -1;
    uint64_t left = ~0ull;   // drafts of these 64 that have not been passed
    while (true) {
      const uint64_t tried = __builtin_amdgcn_ballot_w64(up == st.node && i > st.node) & left;
      if (!tried) break;
      const int bit = __builtin_ctzll(tried), child = i0 + bit;
      left = bit == 63 ? 0 : ~0ull << (bit + 1);
      const double p = weight_of(d.p[child]), u = (double)d.u[child];
      bool yes;
      if constexpr (DRAWN) {
        const double q = weight_of(d.q[child]);
        double size = 1.0;
        if (st.off != 0.0) {   // (another draft behind a rejected one)
          const float* pr = a.p + (r.first + st.node) * a.p_stride;
          const float* qr = a.q + (r.first + st.node) * a.q_stride;
          double sum = 0;
          for (int v = tid; v < a.vocab; v += (int)blockDim.x) sum += left_of(weight_of(pr[v]), st.off, weight_of(qr[v]));
          size = block_sum(sum, lds);
        }
        yes = u * q * size < left_of(p, st.off, q);
        if (!yes) st.off += size;
      } else {
        yes = u * mass < p;
        if (!yes) mass = mass > p ? mass - p : 0.0;
      }
      if (yes) {
        if (path && tid == 0) path[accepted] = child;
        ++accepted;
        st.node = child;
        st.off = 0.0;
        mass = 1.0;
      }
    }
  }
  return accepted;
}

// Bits of the tokens from v0 on, a chunk of them, that the drafts behind `node` had. All threads; bits: a chunk's.
__device__ __forceinline__ void rejected_bits(const VerifyArgs& a, const VerifyState& st, int v0, unsigned* bits) {
  for (int i = (int)threadIdx.x; i < kVerifyChunk / 32; i += (int)blockDim.x) bits[i] = 0;
  __syncthreads();
  for (int i = st.node + 1 + (int)threadIdx.x; i < st.tree; i += (int)blockDim.x)
    if (a.parents[st.first + i] == st.node) {
      const int64_t t = a.tokens[st.first + i];
      if (t >= v0 && t - v0 < kVerifyChunk) atomicOr(&bits[(t - v0) / 32], 1u << (t - v0) % 32);
    }
  __syncthreads();
}

// A sequence whose drafts were drawn: its walk, which may have to sum rows.
__global__ void __launch_bounds__(1024) verify_drawn(VerifyArgs a) {
  __shared__ Drafts d;
  __shared__ double lds[16];
  const int s = (int)blockIdx.x;
  VerifyState st;
  int* path = a.path + (int64_t)s * a.most;
  const int accepted = verify_walk<true>(a, s, d, lds, path, st);
  for (int i = accepted + (int)threadIdx.x; i < a.most; i += 1024) path[i] = -1;
  if (threadIdx.x == 0) {
    a.accepted[s] = accepted;
    a.states[s] = st;
  }
}

// The sum of a chunk of the last row's weights. Where the drafts are no samples, each workgroup walks its sequence by itself
// (no row has to be summed for it), and that of the first chunk writes the path. Grid: chunks, sequences.
template <bool DRAWN>
__global__ void __launch_bounds__(256) verify_sums(VerifyArgs a) {
  __shared__ Drafts d;
  __shared__ double lds[16];
  __shared__ unsigned bits[kVerifyChunk / 32];
  const int s = (int)blockIdx.y, v0 = (int)blockIdx.x * kVerifyChunk;
  VerifyState st;
  if constexpr (DRAWN) {
    st = a.states[s];
  } else {
    int* path = blockIdx.x == 0 ? a.path + (int64_t)s * a.most : nullptr;
    const int accepted = verify_walk<false>(a, s, d, lds, path, st);
    if (path) {
      for (int i = accepted + (int)threadIdx.x; i < a.most; i += 256) path[i] = -1;
      if (threadIdx.x == 0) {
        a.accepted[s] = accepted;
        a.states[s] = st;
      }
    }
  }
  if (st.tree == 0) return;
  if constexpr (!DRAWN) rejected_bits(a, st, v0, bits);
  const int64_t row = st.first + st.node;
  double sum = 0;
#pragma unroll
  for (int k = 0; k < kVerifyChunk / 256; ++k) {
    const int e = k * 256 + (int)threadIdx.x, v = v0 + e;
    if (v >= a.vocab) break;
    double x = weight_of(a.p[row * a.p_stride + v]);
    if constexpr (DRAWN) {
      if (st.off != 0.0) x = left_of(x, st.off, weight_of(a.q[row * a.q_stride + v]));
    } else {
      x = bits[e / 32] >> e % 32 & 1 ? 0.0 : x;
    }
    sum += x;
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) a.sums[(int64_t)s * a.splits + blockIdx.x] = sum;
}

// The next token of a sequence: the chunk that u S falls into by the chunks' sums, then the element. Dynamic LDS: the
// chunks' sums.
template <bool DRAWN>
__global__ void __launch_bounds__(256) verify_pick(VerifyArgs a) {
  extern __shared__ double sums[];
  __shared__ double lds[16];
  __shared__ double upto[256];
  __shared__ unsigned bits[kVerifyChunk / 32];
  __shared__ int found, last;
  __shared__ double before;
  const int s = (int)blockIdx.x, tid = (int)threadIdx.x;
  const VerifyState st = a.states[s];
  if (st.tree == 0) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
  const int64_t row = st.first + st.node;
  const float* pr = a.p + row * a.p_stride;
  const float* qr = DRAWN ? a.q + row * a.q_stride : nullptr;
  double off = st.off;
  bool whole = false;   // p as it is
  for (int i = tid; i < a.splits; i += 256) sums[i] = a.sums[(int64_t)s * a.splits + i];
  __syncthreads();
  double total = 0;
  for (int i = 0; i < a.splits; ++i) total += sums[i];
  if (!(total > 0)) {   // nothing is left of p: p itself
    whole = true;
    off = 0.0;
    for (int c = 0; c < a.splits; ++c) {
      double sum = 0;
      for (int v = c * kVerifyChunk + tid; v < min(a.vocab, (c + 1) * kVerifyChunk); v += 256) sum += weight_of(pr[v]);
      sum = block_sum(sum, lds);
      if (tid == 0) sums[c] = sum;
    }
    __syncthreads();
    total = 0;
    for (int i = 0; i < a.splits; ++i) total += sums[i];
    if (!(total > 0)) {
      if (tid == 0) a.next[s] = -1;
      return;
    }
  }
  const double theta = (double)a.u[st.first] * total;
  if (tid == 0) {
    // The first chunk whose sum up to it exceeds theta; else (rounding, or u from 1 on) the last that has any weight.
    double sum = 0, at = 0;
    int chunk = 0;
    for (int i = 0; i < a.splits; ++i) {
      if (sums[i] > 0) chunk = i, at = sum;
      sum += sums[i];
      if (sums[i] > 0 && sum > theta) break;
    }
    found = chunk, before = at;
  }
  __syncthreads();
  const int chunk = found, v0 = chunk * kVerifyChunk;
  const double rest = theta - before;
  if (!DRAWN && !whole) rejected_bits(a, st, v0, bits);
  // Each thread a run of elements.
  constexpr int RUN = kVerifyChunk / 256;
  double x[RUN], mine = 0;
#pragma unroll
  for (int k = 0; k < RUN; ++k) {
    const int e = tid * RUN + k, v = v0 + e;
    double w = v < a.vocab ? weight_of(pr[v]) : 0.0;
    if (DRAWN) {
      if (off != 0.0 && v < a.vocab) w = left_of(w, off, weight_of(qr[v]));
    } else if (!whole) {
      w = bits[e / 32] >> e % 32 & 1 ? 0.0 : w;
    }
    x[k] = w;
    mine += w;
  }
  upto[tid] = mine;
  if (tid == 0) found = kVerifyChunk, last = -1;
  __syncthreads();
  double sum = 0;
  for (int i = 0; i < tid; ++i) sum += upto[i];
  int here = kVerifyChunk, latest = -1;
#pragma unroll
  for (int k = 0; k < RUN; ++k) {
    sum += x[k];
    if (x[k] > 0) {
      latest = tid * RUN + k;
      if (sum > rest && here == kVerifyChunk) here = latest;
    }
  }
  if (here < kVerifyChunk) atomicMin(&found, here);
  if (latest >= 0) atomicMax(&last, latest);
  __syncthreads();
  if (tid == 0) a.next[s] = v0 + (found < kVerifyChunk ? found : last);
}

// ---- The accepted tokens' rows ----
//
// Row path[j] of a sequence's new tokens becomes row j, j = 0 .. accepted - 1. A thread takes 16 bytes of each row, keys or
// values, of one head, and every j in order: rows never move up, so that a row is read before another one replaces it,
// and kKeepAhead rows are read before the first of them is written.
struct KeepArgs {
  const int* path;           // [seqs][width]
  const int* accepted;
  int* lengths;              // after the call
  int64_t path_stride;
  int width;
};
constexpr int kKeepAhead = 8;
template <int CB>   // bytes of a row
__global__ void __launch_bounds__(256) cache_keep_rows(PagedCache c, KeepArgs a) {
  constexpr int LPR = CB / 16;
  const int s = (int)blockIdx.x;
  const SeqRows r = seq_rows(c.cu[s], c.cu[s + 1], c.lengths[s], c.tokens);
  const int kept = clamp_int(a.accepted[s], 0, min(r.count, a.width)), before = r.length - r.count;
  if (blockIdx.y == 0 && threadIdx.x == 0) a.lengths[s] = max(before + kept, 0);
  const int64_t col = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (col >= (int64_t)2 * c.heads * LPR) return;
  const int chunk = (int)(col % LPR), which = (int)(col / LPR), h = which % c.heads;
  unsigned char* rows = static_cast<unsigned char*>(which >= c.heads ? c.v : c.k);
  float* scale = chunk == 0 ? (which >= c.heads ? c.v_scale : c.k_scale) : nullptr;
  const int* path = a.path + s * a.path_stride;
  auto row_at = [&](int i) {   // of the sequence's new token i, -1 if it has no place
    const int64_t pos = (int64_t)before + i;
    return i >= 0 && i < r.count && pos >= 0 && pos < c.capacity ? cache_row(c, s, h, (int)pos) : -1;
  };
  for (int j0 = 0; j0 < kept; j0 += kKeepAhead) {
    u32x4 x[kKeepAhead];
    float f[kKeepAhead];
    int to[kKeepAhead];
#pragma unroll
    for (int k = 0; k < kKeepAhead; ++k) {
      to[k] = -1;
      const int j = j0 + k, from = j < kept ? path[j] : j;
      if (from == j) continue;
      const int src = row_at(from);
      to[k] = src < 0 ? -1 : row_at(j);
      if (to[k] < 0) continue;
      x[k] = *reinterpret_cast<const u32x4*>(rows + (int64_t)src * CB + chunk * 16);
      if (scale) f[k] = scale[src];
    }
#pragma unroll
    for (int k = 0; k < kKeepAhead; ++k)
      if (to[k] >= 0) {
        *reinterpret_cast<u32x4*>(rows + (int64_t)to[k] * CB + chunk * 16) = x[k];
        if (scale) scale[to[k]] = f[k];
      }
  }
}

}  // namespace pa

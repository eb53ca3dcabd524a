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
// the parents in LDS, as far as nodes of the word can be (parents come before their children). What bounds it is latency:
// offsets, parents, the way up; a tree of 26 tokens takes 1.8 us, 64 of up to 256 2.9.
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
//
// The weights of a row are summed in runs of 1024 elements, each by a wave, and the next token is looked for among the
// runs' sums first and in one run then. Short vocabularies go in one workgroup a sequence and one launch, long ones in as
// many waves as the rows have runs, a launch behind the walk. What bounds them: 48 chains of up to 8 of 128000 tokens, latency in
// the walk (4.9 us) and the choice (4.6), bytes between (8.8 us, 45 MB); one chain of 32000 in one workgroup, latency (9.4);
// 16 trees of 21 of 65537 tokens, three drafts behind a token, the walk's own sums, up to four behind one another (26 us).
struct VerifyState;
struct VerifyArgs {
  const int64_t* tokens;
  const int* parents;
  const float* p;
  const float* q;            // null: the drafts are no samples
  const float* u;
  const int* cu;
  int64_t p_stride, q_stride;
  int n_tokens, vocab, most, runs;
  int* path;                 // [seqs][most]
  int* accepted;
  int64_t* next;
  VerifyState* states;       // [seqs]
  double* sums;              // [seqs][runs]
};
// Where a sequence's path ended: its row of probabilities is first + node.
struct VerifyState {
  double off;                // c
  int first, tree, node, pad;
};
constexpr int kRun = 1024, kRunEach = kRun / kWave;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // four elements of a row, wherever it begins

// An element as it counts, and what is left of it after `off` times q's.
// (0x180: positive and finite, by v_cmp_class.)
__device__ __forceinline__ double weight_of(float x) { return __builtin_amdgcn_classf(x, 0x180) ? (double)x : 0.0; }
__device__ __forceinline__ double left_of(double p, double off, double q) { return fmax(fma(-off, q, p), 0.0); }

// x of another lane, by a move of its halves (common.hpp).
template <typename Move>
__device__ __forceinline__ double move_halves(double x, Move move) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = __builtin_bit_cast(unsigned, move(__builtin_bit_cast(float, (unsigned)u)));
  const unsigned hi = __builtin_bit_cast(unsigned, move(__builtin_bit_cast(float, (unsigned)(u >> 32))));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sums over 16 lanes that follow each other, and over the wave; the same in all lanes (a tree of the same pairs for each).
__device__ __forceinline__ double row_sum16(double x) {
  x += move_halves(x, [](float y) { return dpp_move<0xB1>(y); });
  x += move_halves(x, [](float y) { return dpp_move<0x4E>(y); });
  x += move_halves(x, [](float y) { return dpp_move<0x141>(y); });
  return x + move_halves(x, [](float y) { return dpp_move<0x140>(y); });
}
__device__ __forceinline__ double wave_sum(double x) {
  x = row_sum16(x);
  x += move_halves(x, [](float y) { return partner16(y); });
  return x + move_halves(x, [](float y) { return partner32(y); });
}
// The sum of x over a workgroup of 1024 threads, the same in all of them and in the same order always. lds: 16 numbers.
__device__ __forceinline__ double block_sum(double x, double* lds) {
  x = wave_sum(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
  __syncthreads();
  return row_sum16(lds[threadIdx.x % 16]);
}

// What the walk needs of each draft. 20 KB of LDS.
struct Drafts {
  int parent[kTreeMax];      // -1: no draft
  int token[kTreeMax];
  float p[kTreeMax], q[kTreeMax], u[kTreeMax];
};

// Adds what is left of N elements to a sum. Where none of the wave's is negative or not finite, which their bits show for half an
// operation an element, without the weights' own tests (16 trees of 21 of 65537 tokens 42 us and 34).
template <int N>
__device__ __forceinline__ void add_left(const float (&p)[N], const float (&q)[N], double off, double& sum) {
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) top = max(top, max(__builtin_bit_cast(unsigned, p[k]), __builtin_bit_cast(unsigned, q[k])));
  if (__builtin_amdgcn_ballot_w64(top >= 0x7f800000u) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) sum += left_of((double)p[k], off, (double)q[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) sum += left_of(weight_of(p[k]), off, weight_of(q[k]));
  }
}
// S(off) of a row, by a workgroup of 1024 threads, 8 elements a thread and step, the next step's and the rest's on their way
// meanwhile. What bounds it is the VALU of the one CU (66 % busy), six operations in 64 bits or on their way there a pair of elements: rows
// of p and q of 256 KB each take 5 us. (Each element tested by its class, 16 a step and nothing ahead, 7.5; loads of single
// elements and comparisons for the class, 10 to 12.)
__device__ __forceinline__ double row_left(const VerifyArgs& a, int64_t row, double off, double* lds) {
  constexpr int EACH = 2, N = 4 * EACH, STEP = N * 1024;
  const float* pr = a.p + row * a.p_stride;
  const float* qr = a.q + row * a.q_stride;
  const int steps = a.vocab / STEP;
  float p0[N], q0[N], p1[N], q1[N], p[N], q[N];
  auto load = [&](int step, float (&ps)[N], float (&qs)[N]) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int v = step * STEP + 4 * ((int)threadIdx.x + 1024 * k);
      const f32x4u x = *reinterpret_cast<const f32x4u*>(pr + v), y = *reinterpret_cast<const f32x4u*>(qr + v);
#pragma unroll
      for (int j = 0; j < 4; ++j) ps[4 * k + j] = x[j], qs[4 * k + j] = y[j];
    }
  };
  if (steps > 0) load(0, p0, q0);
#pragma unroll
  for (int k = 0; k < N; ++k) {   // the rest
    const int v = steps * STEP + (int)threadIdx.x + 1024 * k;
    p[k] = v < a.vocab ? pr[v] : 0.f, q[k] = v < a.vocab ? qr[v] : 0.f;
  }
  double sum = 0;
  for (int i = 0; i < steps; i += 2) {
    if (i + 1 < steps) load(i + 1, p1, q1);
    add_left(p0, q0, off, sum);
    if (i + 1 == steps) break;
    if (i + 2 < steps) load(i + 2, p0, q0);
    add_left(p1, q1, off, sum);
  }
  add_left(p, q, off, sum);
  return block_sum(sum, lds);
}

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
        // (S(0) is 1; another draft behind a rejected one needs a row's sum)
        const double size = st.off != 0.0 ? row_left(a, r.first + st.node, st.off, lds) : 1.0;
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
__device__ __forceinline__ void write_walk(const VerifyArgs& a, int s, int* path, int accepted, const VerifyState& st) {
  for (int i = accepted + (int)threadIdx.x; i < a.most; i += (int)blockDim.x) path[i] = -1;
  if (threadIdx.x == 0) a.accepted[s] = accepted, a.states[s] = st;
}

// Weights of a wave's elements of a run that starts at v0, 16 a lane: element e(k) = kRunEach * lane + k (by_lane) or
// 4 * lane + 256 * (k / 4) + k % 4. out: bits of the run's tokens that count as 0, null if none do.
__device__ __forceinline__ int run_element(bool by_lane, int k) {
  const int lane = (int)threadIdx.x % kWave;
  return by_lane ? kRunEach * lane + k : 4 * lane + 256 * (k / 4) + k % 4;
}
template <bool DRAWN>
__device__ __forceinline__ void run_weights(const VerifyArgs& a, int64_t row, double off, int v0, bool by_lane, const unsigned* out,
                                            double (&x)[kRunEach]) {
  const float* pr = a.p + row * a.p_stride + v0;
  const float* qr = DRAWN && off != 0.0 ? a.q + row * a.q_stride + v0 : pr;
  float p[kRunEach], q[kRunEach];
  if (v0 + kRun <= a.vocab) {
#pragma unroll
    for (int k = 0; k < kRunEach; k += 4) {
      const f32x4u y = *reinterpret_cast<const f32x4u*>(pr + run_element(by_lane, k));
      const f32x4u z = DRAWN ? *reinterpret_cast<const f32x4u*>(qr + run_element(by_lane, k)) : y;
#pragma unroll
      for (int j = 0; j < 4; ++j) p[k + j] = y[j], q[k + j] = z[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kRunEach; ++k) {
      const int e = run_element(by_lane, k);
      p[k] = v0 + e < a.vocab ? pr[e] : 0.f;
      q[k] = DRAWN && v0 + e < a.vocab ? qr[e] : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < kRunEach; ++k) {
    double w = weight_of(p[k]);
    if constexpr (DRAWN) w = off != 0.0 ? left_of(w, off, weight_of(q[k])) : w;
    if (out) {
      const int e = run_element(by_lane, k);
      w = out[e / 32] >> e % 32 & 1 ? 0.0 : w;
    }
    x[k] = w;
  }
}
template <bool DRAWN>
__device__ __forceinline__ double run_sum(const VerifyArgs& a, int64_t row, double off, int v0, const unsigned* out) {
  double x[kRunEach], sum = 0;
  run_weights<DRAWN>(a, row, off, v0, false, out, x);
#pragma unroll
  for (int k = 0; k < kRunEach; ++k) sum += x[k];
  return wave_sum(sum);
}
// Bits of the tokens of a run from v0 on that the drafts behind the last token had, by one wave (a run's bits are its own).
__device__ __forceinline__ void rejected_bits(const VerifyArgs& a, const VerifyState& st, int v0, unsigned* bits) {
  const int lane = (int)threadIdx.x % kWave;
  if (lane < kRun / 32) bits[lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int i = st.node + 1 + lane; i < st.tree; i += kWave)
    if (a.parents[st.first + i] == st.node) {
      const int64_t t = a.tokens[st.first + i];
      if (t >= v0 && t - v0 < kRun) atomicOr(&bits[(t - v0) / 32], 1u << (t - v0) % 32);
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// The next token, by one wave: `sums` are those of the row's runs. Lane l takes the runs l G to (l + 1) G - 1, then 16
// elements of the run that was found.
template <bool DRAWN>
__device__ __forceinline__ int64_t pick_token(const VerifyArgs& a, const VerifyState& st, const double* sums, unsigned* bits) {
  const int lane = (int)threadIdx.x % kWave;
  const int64_t row = st.first + st.node;
  const int group = (a.runs + kWave - 1) / kWave, r0 = lane * group, r1 = min(r0 + group, a.runs);
  double off = st.off, mine = 0;
  bool whole = false;   // p as it is
  for (int r = r0; r < r1; ++r) mine += sums[r];
  if (!(wave_sum(mine) > 0)) {   // nothing is left of it
    whole = true;
    off = 0.0;
    mine = 0;
    for (int r = 0; r < a.runs; ++r) {
      const double sum = run_sum<DRAWN>(a, row, 0.0, r * kRun, nullptr);
      mine += r >= r0 && r < r1 ? sum : 0.0;
    }
  }
  auto scan = [&](double x) {   // sums up to the lane's
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const double other = __shfl_up(x, d);
      if (lane >= d) x += other;
    }
    return x;
  };
  // The first lane with weight whose sum up to it exceeds theta; else (rounding, or u from 1 on) the last with weight.
  auto choose = [&](double x, double upto, double theta) {
    const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0), over = __builtin_amdgcn_ballot_w64(x > 0 && upto > theta);
    return over ? __builtin_ctzll(over) : some ? kWave - 1 - __builtin_clzll(some) : -1;
  };
  double upto = scan(mine);
  double theta = (double)a.u[st.first] * __shfl(upto, kWave - 1);
  int at = choose(mine, upto, theta);
  if (at < 0) return -1;
  theta -= __shfl(upto - mine, at);   // (the lane's own runs)
  int run = 0;
  {
    double sum = 0, before = 0;
    for (int r = at * group; r < min((at + 1) * group, a.runs); ++r) {
      const double x = whole ? run_sum<DRAWN>(a, row, 0.0, r * kRun, nullptr) : sums[r];
      if (x > 0) run = r, before = sum;
      sum += x;
      if (x > 0 && sum > theta) break;
    }
    theta -= before;
  }
  const int v0 = run * kRun;
  if (!DRAWN && !whole) rejected_bits(a, st, v0, bits);
  double x[kRunEach];
  run_weights<DRAWN>(a, row, off, v0, true, !DRAWN && !whole ? bits : nullptr, x);
  mine = 0;
#pragma unroll
  for (int k = 0; k < kRunEach; ++k) mine += x[k];
  upto = scan(mine);
  at = choose(mine, upto, theta);
  double sum = upto - mine;
  int here = -1, last = -1;
#pragma unroll
  for (int k = 0; k < kRunEach; ++k) {
    sum += x[k];
    if (x[k] > 0) last = k;
    if (x[k] > 0 && here < 0 && sum > theta) here = k;
  }
  here = __shfl(here < 0 ? last : here, at < 0 ? 0 : at);
  return at < 0 ? -1 : v0 + kRunEach * at + here;
}

// The whole of a sequence in one workgroup. Dynamic LDS: the runs' sums.
template <bool DRAWN>
__global__ void __launch_bounds__(1024) verify_whole(VerifyArgs a) {
  extern __shared__ double sums[];
  __shared__ Drafts d;
  __shared__ double lds[16];
  __shared__ unsigned bits[16][kRun / 32];
  const int s = (int)blockIdx.x, wave = (int)threadIdx.x / kWave;
  VerifyState st;
  int* path = a.path + (int64_t)s * a.most;
  const int accepted = verify_walk<DRAWN>(a, s, d, lds, path, st);
  for (int i = accepted + (int)threadIdx.x; i < a.most; i += 1024) path[i] = -1;
  if (threadIdx.x == 0) a.accepted[s] = accepted;
  if (st.tree == 0) {
    if (threadIdx.x == 0) a.next[s] = -1;
    return;
  }
  for (int r = wave; r < a.runs; r += 16) {
    if constexpr (!DRAWN) rejected_bits(a, st, r * kRun, bits[wave]);
    const double sum = run_sum<DRAWN>(a, st.first + st.node, st.off, r * kRun, DRAWN ? nullptr : bits[wave]);
    if (threadIdx.x % kWave == 0) sums[r] = sum;
  }
  __syncthreads();
  if (wave == 0) {
    const int64_t token = pick_token<DRAWN>(a, st, sums, bits[0]);
    if (threadIdx.x == 0) a.next[s] = token;
  }
}

// The walk alone, of a sequence whose drafts were drawn (it may have to sum rows).
__global__ void __launch_bounds__(1024) verify_drawn(VerifyArgs a) {
  __shared__ Drafts d;
  __shared__ double lds[16];
  VerifyState st;
  int* path = a.path + (int64_t)blockIdx.x * a.most;
  const int accepted = verify_walk<true>(a, (int)blockIdx.x, d, lds, path, st);
  write_walk(a, (int)blockIdx.x, path, accepted, st);
}

// The runs' sums of the last row, one a wave. Where the drafts are no samples, each workgroup walks its sequence by itself
// (no row has to be summed for that), and the first one writes the path. Grid: four runs, sequences.
template <bool DRAWN>
__global__ void __launch_bounds__(256) verify_sums(VerifyArgs a) {
  __shared__ Drafts d;
  __shared__ double lds[16];
  __shared__ unsigned bits[4][kRun / 32];
  const int s = (int)blockIdx.y, wave = (int)threadIdx.x / kWave, r = (int)blockIdx.x * 4 + wave;
  VerifyState st;
  if constexpr (DRAWN) {
    st = a.states[s];
  } else {
    int* path = blockIdx.x == 0 ? a.path + (int64_t)s * a.most : nullptr;
    const int accepted = verify_walk<false>(a, s, d, lds, path, st);
    if (path) write_walk(a, s, path, accepted, st);
  }
  if (st.tree == 0 || r >= a.runs) return;
  if constexpr (!DRAWN) rejected_bits(a, st, r * kRun, bits[wave]);
  const double sum = run_sum<DRAWN>(a, st.first + st.node, st.off, r * kRun, DRAWN ? nullptr : bits[wave]);
  if (threadIdx.x % kWave == 0) a.sums[(int64_t)s * a.runs + r] = sum;
}

// The next token of a sequence, behind the runs' sums.
template <bool DRAWN>
__global__ void __launch_bounds__(kWave) verify_pick(VerifyArgs a) {
  __shared__ unsigned bits[kRun / 32];
  const int s = (int)blockIdx.x;
  const VerifyState st = a.states[s];
  const int64_t token = st.tree == 0 ? -1 : pick_token<DRAWN>(a, st, a.sums + (int64_t)s * a.runs, bits);
  if (threadIdx.x == 0) a.next[s] = token;
}

// ---- The accepted tokens' rows ----
//
// Row path[j] of a sequence's new tokens becomes row j, j = 0 .. accepted - 1. A thread takes 16 bytes of each row, keys or
// values, of one head, and every j in order: rows never move up, so that a row is read before another one replaces it,
// and kKeepAhead rows are read before the first of them is written. A chain of four loads (offsets, path, page table, row) and
// the store: 4 sequences, 8 heads of 128 in bf16, 4.1 us; 64 in int8 5.8.
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

// Attention of each sequence's new tokens over its pages.
//
// New token i of a sequence of `length` tokens, count of them new, sees the keys at positions up to
// length - count + i (causal) or all of them: O = sum_j softmax_j(q . k_j / sqrt(D)) v_j. Query head h reads
// key/value head h / group. A token that sees no key gets zeros.
#pragma once

#include "paged_cache.hpp"

namespace pa {

struct RowsQ {
  const void* q;
  void* o;
  int64_t q_token, q_head, o_token, o_head;   // strides in elements
  int group, heads;                            // query heads per key/value head, and query heads
};

// One workgroup per (new token, query head): 256 / (D / 8) keys at a time, 8 dims a lane, each group of D / 8
// lanes with a running maximum and sum of its own; the groups are joined through LDS at the end.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(256) paged_attn_rows(PagedCache c, RowsQ a, float scale_log2, int causal) {
  constexpr int LPR = D / 8, KPB = 256 / LPR;
  __shared__ float acc_s[KPB][D];
  __shared__ float m_s[KPB], l_s[KPB];
  const int t = (int)blockIdx.x / a.heads, hq = (int)blockIdx.x % a.heads, h = hq / a.group;
  const int sub = (int)threadIdx.x % LPR, kg = (int)threadIdx.x / LPR;
  const int seq = find_seq(c, t);
  if (seq >= c.seqs) return;
  const SeqRows s = load_seq(c, seq);
  if (t < s.first || t >= s.first + s.count) return;
  const int seen = keys_seen(s, t - s.first, c.capacity, causal);
  float q[8], o[8] = {}, m = -INFINITY, l = 0.f;
  cached8(static_cast<const T*>(a.q) + t * a.q_token + hq * a.q_head, 8 * sub, 1.f, q);
  for (int pos = kg; pos < seen; pos += KPB) {
    const int at = cache_row(c, seq, h, pos);
    if (at < 0) continue;
    float x[8], ks = 1.f, vs = 1.f, dot = 0.f;
    if constexpr (cache_type<C>::k8bit) ks = c.k_scale[at], vs = c.v_scale[at];
    cached8(static_cast<const C*>(c.k) + (int64_t)at * D, 8 * sub, ks, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) dot = fmaf(q[j], x[j], dot);
    dot += dpp_move<0xB1>(dot);
    dot += dpp_move<0x4E>(dot);
    dot += dpp_move<0x141>(dot);
    if constexpr (LPR == 16) dot += dpp_move<0x140>(dot);
    dot *= scale_log2;
    const float mn = fmaxf(m, dot);
    const float old = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
    const float p = mn == -INFINITY ? 0.f : exp2_fast(dot - mn);
    cached8(static_cast<const C*>(c.v) + (int64_t)at * D, 8 * sub, vs, x);
    m = mn;
    l = fmaf(l, old, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = fmaf(p, x[j], o[j] * old);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc_s[kg][8 * sub + j] = o[j];
  if (sub == 0) m_s[kg] = m, l_s[kg] = l;
  __syncthreads();
  if ((int)threadIdx.x < D) {
    float mx = -INFINITY, sum = 0.f, out = 0.f;
    for (int g = 0; g < KPB; ++g) mx = fmaxf(mx, m_s[g]);
    for (int g = 0; g < KPB; ++g) {
      const float w = m_s[g] == -INFINITY ? 0.f : exp2_fast(m_s[g] - mx);
      sum = fmaf(w, l_s[g], sum);
      out = fmaf(w, acc_s[g][threadIdx.x], out);
    }
    static_cast<T*>(a.o)[t * a.o_token + hq * a.o_head + threadIdx.x] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
  }
}

}  // namespace pa

// Rotary positions: pairs of a head's first `pairs` x 2 elements turned by angles that grow with the token's position.
//
// Pair p of a token at position n is turned by the angle n f[p] (inverse: by its negative, which is the turn's gradient
// and its undoing where the factor is 1): (x, y) -> s (x cos - y sin, x sin + y cos). The pairs are (p, p + pairs), the
// halves of the turned part, or (2 p, 2 p + 1), interleaved. Elements behind the turned part pass as they are.
#pragma once

#include "../paged_model.hpp"
#include "common.hpp"

namespace pa {

constexpr int kRopeMaxDim = 1024;

struct RopeRows {
  const void* in;
  void* out;
  int64_t in_b, in_n, in_h, out_b, out_n, out_h;   // strides in elements; a head's elements are contiguous
  int heads;
};
struct RopeArgs {
  RopeRows x[2];
  const void* positions;      // int32 or int64
  const double* freqs;
  int64_t pos_b, pos_n;
  int64_t tokens;             // b * n
  int n, d, pairs, pos64, inverse;
  int units;                  // of a head: W pairs or up to 2 W elements that pass each; interleaved, W elements (at least 2)
  int heads, group;           // q's and k's heads, and the tokens that a workgroup takes at a time
  int heads_outer;            // units follow each other token by token within a head, else head by head within a token
  PageDiv by_n, by_pairs, by_units, by_inner;   // by_inner: units of a head's tokens, or of a token's heads
  float scale;
};
constexpr int kRopeTurns = 1024;   // angles of a group

// cos and sin of n f in fp32. The angle in turns is n f / (2 pi), of which a fraction counts: products and fraction in 64
// bits with the products' rounding carried along, so that it is right to about 2^-50 of a turn at any 32-bit position (in
// 32 bits position 10^6 would be off by 0.06 rad). An eighth of a turn either side of a quarter goes to the fp32 functions.
__device__ __forceinline__ float2 rope_turn(double pos, double f, bool inverse, float scale) {
  constexpr double kInv2Pi = 0.15915494309189535, kInv2PiLow = -9.839338337591243e-18;   // 1 / (2 pi) in two parts
  const double g = f * kInv2Pi, g_low = fma(f, kInv2Pi, -g) + f * kInv2PiLow;
  const double t = pos * g, t_low = fma(pos, g, -t) + pos * g_low;
  const double part = (t - rint(t)) + t_low, quarter = rint(4.0 * part);
  const float rest = 2.0f * (float)(part - 0.25 * quarter);   // in half turns
  float s, c;
  sincospif(rest, &s, &c);
  const int q = (int)quarter & 3;
  float cq = q & 1 ? -s : c, sq = q & 1 ? c : s;
  if (q & 2) cq = -cq, sq = -sq;
  return {cq * scale, (inverse ? -sq : sq) * scale};
}

// A workgroup takes a few tokens: their angles once, in LDS, for all heads of q and k; then units over the threads, in the
// order of memory. A unit is read whole before it is written, by one thread: in and out may be the same rows. W is the widest
// that sizes, strides and addresses allow. Bytes are what bounds it: gradients of 4 x 4096 tokens, (B, H, N, d) with 64 heads of
// 128, half of each turned, interleaved, 102 us, 5.3 TB/s (in units of two loads side by side 120: each load then takes every
// other 16 bytes); 32768 packed tokens of 40 heads 120 us, 5.6 TB/s. 64 single tokens of 40 heads are latency: 4.4 us.
template <typename T, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_rows(RopeArgs a) {
  __shared__ float2 turn[kRopeTurns];
  const int turned = INTERLEAVED && W > 1 ? 2 * a.pairs / W : a.pairs / W, inner = (a.heads_outer ? a.group : a.heads) * a.units;
  for (int64_t t0 = (int64_t)blockIdx.x * a.group; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.group) {
    const int here = (int)min((int64_t)a.group, a.tokens - t0);
    __syncthreads();
    for (int i = (int)threadIdx.x; i < here * a.pairs; i += 256) {
      const int t = (int)page_of(i, a.by_pairs), token = (int)t0 + t, b = (int)page_of(token, a.by_n);
      const int64_t at = b * a.pos_b + (token - b * a.n) * a.pos_n;
      const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[at] : (double)static_cast<const int*>(a.positions)[at];
      turn[i] = rope_turn(pos, a.freqs[i - t * a.pairs], a.inverse != 0, a.scale);
    }
    __syncthreads();
    const int items = (a.heads_outer ? a.heads : here) * inner;
    for (int i = (int)threadIdx.x; i < items; i += 256) {
      const int outer = (int)page_of(i, a.by_inner), rest = i - outer * inner;
      const int mid = (int)page_of(rest, a.by_units), u = rest - mid * a.units;
      const int t = a.heads_outer ? mid : outer;
      int h = a.heads_outer ? outer : mid;
      if (t >= here) continue;
      const int token = (int)t0 + t, b = (int)page_of(token, a.by_n), n = token - b * a.n;
      const RopeRows& x = a.x[h < a.x[0].heads ? 0 : 1];
      h -= h < a.x[0].heads ? 0 : a.x[0].heads;
      const T* in = static_cast<const T*>(x.in) + b * x.in_b + n * x.in_n + h * x.in_h;
      T* out = static_cast<T*>(x.out) + b * x.out_b + n * x.out_n + h * x.out_h;
      // Two loads of W elements a lane, each of them side by side over the lanes: the pairs' halves, or halves of what passes;
      // interleaved: one of W (at least a pair), wherever it lies.
      constexpr int E = INTERLEAVED && W == 1 ? 2 : W;
      typedef T TE __attribute__((ext_vector_type(E), aligned(sizeof(T) * W)));
      if constexpr (INTERLEAVED) {
        const int e = u * E;
        if (e + E > a.d) {   // (an odd head's last element)
          out[e] = in[e];
          continue;
        }
        TE v = *reinterpret_cast<const TE*>(in + e);
        if (u < turned) {
#pragma unroll
          for (int k = 0; k < E; k += 2) {
            const float2 angle = turn[t * a.pairs + (e + k) / 2];
            const float xv = to_f32(v[k]), yv = to_f32(v[k + 1]);
            v[k] = from_f32<T>(fmaf(xv, angle.x, -(yv * angle.y))), v[k + 1] = from_f32<T>(fmaf(xv, angle.y, yv * angle.x));
          }
        }
        *reinterpret_cast<TE*>(out + e) = v;
      } else {
        const bool turns = u < turned;
        const int e0 = turns ? u * W : 2 * a.pairs + (u - turned) * W, e1 = e0 + (turns ? a.pairs : (a.units - turned) * W);
        const bool both = e1 < a.d;
        TE v0 = *reinterpret_cast<const TE*>(in + e0), v1 = {};
        if (both) v1 = *reinterpret_cast<const TE*>(in + e1);
        if (turns) {
#pragma unroll
          for (int k = 0; k < W; ++k) {
            const float2 angle = turn[t * a.pairs + u * W + k];
            const float xv = to_f32(v0[k]), yv = to_f32(v1[k]);
            v0[k] = from_f32<T>(fmaf(xv, angle.x, -(yv * angle.y))), v1[k] = from_f32<T>(fmaf(xv, angle.y, yv * angle.x));
          }
        }
        *reinterpret_cast<TE*>(out + e0) = v0;
        if (both) *reinterpret_cast<TE*>(out + e1) = v1;
      }
    }
  }
}

}  // namespace pa

// Rotary positions: pairs of a head's first `pairs` x 2 elements turned by angles that grow with the token's position.
//
// Pair p of a token at position n is turned by the angle n f[p] (inverse: by its negative, which is the turn's gradient
// and its undoing where the factor is 1): (x, y) -> s (x cos - y sin, x sin + y cos). The pairs are (p, p + pairs), the
// halves of the turned part, or (2 p, 2 p + 1), interleaved. Elements behind the turned part pass as they are.
#pragma once

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
  int n, d, pairs, pos64, inverse, units;   // units: of a head, each `W` pairs or `W` elements that pass
  float scale;
};

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

// A workgroup takes one token: its angles once, in LDS, for all heads of q and k; then units of W pairs (two loads of W
// elements), or of W elements that pass, over the threads. A unit is read whole before it is written, by one thread: in
// and out may be the same rows. W is the widest that sizes, strides and addresses allow.
template <typename T, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_rows(RopeArgs a) {
  typedef T TW __attribute__((ext_vector_type(W)));
  __shared__ float2 turn[kRopeMaxDim / 2];
  for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const int64_t b = token / a.n, n = token - b * a.n;
    const int64_t at = b * a.pos_b + n * a.pos_n;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[at] : (double)static_cast<const int*>(a.positions)[at];
    __syncthreads();
    for (int p = (int)threadIdx.x; p < a.pairs; p += 256) turn[p] = rope_turn(pos, a.freqs[p], a.inverse != 0, a.scale);
    __syncthreads();
    const int turned = a.pairs / W, first = a.x[0].heads * a.units, all = first + a.x[1].heads * a.units;
    for (int i = (int)threadIdx.x; i < all; i += 256) {
      const RopeRows& x = a.x[i < first ? 0 : 1];
      const int j = i < first ? i : i - first, h = j / a.units, u = j - h * a.units;
      const T* in = static_cast<const T*>(x.in) + b * x.in_b + n * x.in_n + h * x.in_h;
      T* out = static_cast<T*>(x.out) + b * x.out_b + n * x.out_n + h * x.out_h;
      if (u >= turned) {
        const int e = 2 * a.pairs + (u - turned) * W;
        *reinterpret_cast<TW*>(out + e) = *reinterpret_cast<const TW*>(in + e);
        continue;
      }
      const int e0 = INTERLEAVED ? 2 * u * W : u * W, e1 = INTERLEAVED ? e0 + W : e0 + a.pairs;
      const TW v0 = *reinterpret_cast<const TW*>(in + e0), v1 = *reinterpret_cast<const TW*>(in + e1);
      TW w0, w1;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float2 t = turn[u * W + k];
        // interleaved: the unit's 2 W elements are x, y, x, y, ...
        const int xe = INTERLEAVED ? 2 * k : k, ye = INTERLEAVED ? 2 * k + 1 : W + k;
        const float xv = to_f32(xe < W ? v0[xe % W] : v1[xe % W]), yv = to_f32(ye < W ? v0[ye % W] : v1[ye % W]);
        const T xo = from_f32<T>(fmaf(xv, t.x, -(yv * t.y))), yo = from_f32<T>(fmaf(xv, t.y, yv * t.x));
        if (xe < W) w0[xe % W] = xo; else w1[xe % W] = xo;
        if (ye < W) w0[ye % W] = yo; else w1[ye % W] = yo;
      }
      *reinterpret_cast<TW*>(out + e0) = w0;
      *reinterpret_cast<TW*>(out + e1) = w1;
    }
  }
}

}  // namespace pa

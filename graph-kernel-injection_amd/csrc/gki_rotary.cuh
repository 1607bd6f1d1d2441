// Rows turned by rotary positions (RotaryArgs), for the kernels that do it.
#pragma once

#include "gki_paged.cuh"

namespace gki {
namespace {

// cos and sin of pair j at a token. The angle is made and reduced in 64 bits (turns, then the
// quarter it lies in: at most an eighth of a turn from it, which fp32 holds to 2^-28 of a
// turn). The turns of a position and their product with it are rounded, by about 3.3 units of 2^-53
// of the angle together: up to 2^-21.2 of a radian at position 2^30 and frequency 1, against exact
// angles 2^-21.9 at most.
__device__ inline float2 rotary_turn(const RotaryArgs& a, int64_t t, int j) {
  const int64_t at = a.axis[j] * a.pa + t / a.n * a.pb + t % a.n * a.pn;
  const double p = a.wide ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
  double r = p * a.turns[j];
  r -= rint(r);
  const double quarter = rint(4.0 * r);
  float s, c;
  sincospif((float)(2.0 * (r - 0.25 * quarter)), &s, &c);
  const int k = (int)quarter & 3;
  const float cs = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s;
  const float sn = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
  return make_float2(cs, sn * a.sign);
}

// 16 bytes of a row as floats, and back.
template <typename T> constexpr int kPer16 = T::is_f32 ? 4 : 8;
template <typename T>
__device__ inline void unpack16(const uint4& w, float (&f)[kPer16<T>]) {
  if constexpr (T::is_f32) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  } else {
    const uint16_t* h = (const uint16_t*)&w;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = T::to_float(h[i]);
  }
}
template <typename T>
__device__ inline uint4 pack16(const float (&f)[kPer16<T>]) {
  if constexpr (T::is_f32)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// Items of a row: a thread turns E pairs (two chunks of 16 bytes, or one where the pairs
// are interleaved) or copies a chunk behind them.
template <typename T, bool INTER>
__device__ inline int rotary_items(int pairs, int D) {
  constexpr int E = kPer16<T>;
  return INTER ? D / E : pairs / E + (D - 2 * pairs) / E;
}
// Item i of the row at src, to dst; cs: the token's cosines and sines.
template <typename T, bool INTER>
__device__ inline void rotary_item(const RotaryArgs& a, const float2* cs, int i, const typename T::storage* src,
                                   typename T::storage* dst) {
  constexpr int E = kPer16<T>;
  const int np = a.pairs / E;
  if (INTER ? i >= 2 * np : i >= np) {                   // behind the pairs
    const int c = INTER ? i : i + np;
    *(uint4*)(dst + c * E) = *(const uint4*)(src + c * E);
    return;
  }
  if constexpr (INTER) {
    float f[E], g[E];
    unpack16<T>(*(const uint4*)(src + i * E), f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 w = cs[(i * E + e) / 2];
      g[e] = f[e] * w.x - f[e + 1] * w.y;
      g[e + 1] = f[e] * w.y + f[e + 1] * w.x;
    }
    *(uint4*)(dst + i * E) = pack16<T>(g);
  } else {
    float f[E], h[E], u[E], v[E];
    unpack16<T>(*(const uint4*)(src + i * E), f);
    unpack16<T>(*(const uint4*)(src + a.pairs + i * E), h);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 w = cs[i * E + e];
      u[e] = f[e] * w.x - h[e] * w.y;
      v[e] = f[e] * w.y + h[e] * w.x;
    }
    *(uint4*)(dst + i * E) = pack16<T>(u);
    *(uint4*)(dst + a.pairs + i * E) = pack16<T>(v);
  }
}

}  // namespace
}  // namespace gki

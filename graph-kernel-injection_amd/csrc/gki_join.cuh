// The states (largest score, sum, accumulator) that slices of a row's keys leave, joined.
#pragma once

#include "gki_common.cuh"

namespace gki {
namespace {

// O = sum_p f_p acc_p / sum_p f_p l_p and LSE = M + ln(sum_p f_p l_p) with f_p the
// exponential of m_p - M, M the largest m_p (NATURAL: in natural units, else base 2):
// a wave per row, the parts in order; L2 holds what the slices wrote. A row without
// keys has O = 0, LSE = 0. Sums in fp32: n parts add n roundings of 2^-24 to the thousands
// that the parts hold. 1024 rows of 11 parts, D128: 4 us.
template <typename T, int D, bool NATURAL>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ acc, const float* __restrict__ ml,
                                                   typename T::storage* __restrict__ O, float* __restrict__ LSE,
                                                   int64_t n_rows, int n_parts) {
  constexpr int E = D >= 64 ? D / 64 : 1;      // elements per lane
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= n_rows || (D < 64 && lane >= D)) return;
  const float2* st = (const float2*)ml + row * n_parts;
  const float* x = acc + row * n_parts * D + E * lane;
  float M = kNegInf;
#pragma unroll 4
  for (int p = 0; p < n_parts; ++p) M = fmaxf(M, st[p].x);
  const float Mu = M == kNegInf ? 0.f : M;
  float L = 0.f, a[E];
#pragma unroll
  for (int e = 0; e < E; ++e) a[e] = 0.f;
#pragma unroll 4
  for (int p = 0; p < n_parts; ++p) {
    const float f = __builtin_amdgcn_exp2f(NATURAL ? (st[p].x - Mu) * kLog2e : st[p].x - Mu);
    L += st[p].y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] += x[(size_t)p * D + e] * f;
  }
  typename T::storage* dst = O + row * D + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = T::from_float(a[e] / (L == 0.f ? 1.f : L));
  if (lane == 0) LSE[row] = L == 0.f ? 0.f : NATURAL ? (float)((double)M + log((double)L)) : lse_natural(M, L);
}

template <typename T, int D, bool NATURAL>
void launch_join(const float* acc, const float* ml, void* o, float* lse, int64_t n_rows, int n_parts,
                 hipStream_t stream) {
  hipLaunchKernelGGL((join_kernel<T, D, NATURAL>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, stream, acc, ml,
                     (typename T::storage*)o, lse, n_rows, n_parts);
}

}  // namespace
}  // namespace gki

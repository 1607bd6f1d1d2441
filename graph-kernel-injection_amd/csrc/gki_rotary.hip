// Rotary positions of queries and keys in one launch, forward and (by the opposite
// angle) backward.
//
// Bound by HBM: every row is read once and written once. A workgroup takes up to four
// tokens: their cosines and sines once into LDS (64-bit angles, two orders of magnitude
// dearer than an element's products), then all heads of both tensors. Turned rows are rounded
// once, to their type. 16384 tokens of 32 + 8 heads (D128 bf16, 335 MB both ways) 69 us, 4.85 TB/s, what
// a large copy reaches (4.97); 64 tokens 4.3.
#include "gki_rotary.cuh"

namespace gki {
namespace {

constexpr int kMaxPairs = 64;
// From kManyTokens on, us, 1 / 4 tokens a group: 2048 (H32/8 D128) 9.6 / 10.9, 4096 17.0 / 16.8, 4096
// (H4/4 D64 fp32) 6.7 / 5.3, 16384 (H32/8) 70.8 / 67.9.
constexpr int kTokensPerGroup = 4, kManyTokens = 4096;

template <typename T, int D, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, HeadRows q, HeadRows k, int tokens_per_group) {
  using S = typename T::storage;
  __shared__ float2 cs[kTokensPerGroup * kMaxPairs];
  const int64_t t0 = (int64_t)blockIdx.x * tokens_per_group;
  const int n_tok = (int)min((int64_t)tokens_per_group, a.tokens - t0);
  for (int i = threadIdx.x; i < n_tok * a.pairs; i += 256)
    cs[(i / a.pairs) * kMaxPairs + i % a.pairs] = rotary_turn(a, t0 + i / a.pairs, i % a.pairs);
  __syncthreads();
  const int per_row = rotary_items<T, INTER>(a.pairs, D), heads = q.heads + k.heads;
  for (int x = threadIdx.x; x < n_tok * heads * per_row; x += 256) {
    const int i = x % per_row, y = x / per_row, tok = y / heads, hh = y % heads;
    const bool is_k = hh >= q.heads;
    const HeadRows& r = is_k ? k : q;
    const int h = is_k ? hh - q.heads : hh;
    const int64_t t = t0 + tok, b = t / a.n, j = t % a.n;
    rotary_item<T, INTER>(a, cs + tok * kMaxPairs, i, (const S*)r.src + b * r.sb + j * r.sn + h * r.sh,
                          (S*)r.dst + b * r.db + j * r.dn + h * r.dh);
  }
}

template <typename T, int D>
int rotary(const RotaryArgs& a, const HeadRows& q, const HeadRows& k, hipStream_t stream) {
  const int per = a.tokens >= kManyTokens ? kTokensPerGroup : 1;
  const dim3 grid((unsigned)((a.tokens + per - 1) / per));
  if (a.interleaved) hipLaunchKernelGGL((rotary_kernel<T, D, true>), grid, dim3(256), 0, stream, a, q, k, per);
  else hipLaunchKernelGGL((rotary_kernel<T, D, false>), grid, dim3(256), 0, stream, a, q, k, per);
  return check_launch("gki_rotary");
}

template <int D>
int rotary_of(int dtype, const RotaryArgs& a, const HeadRows& q, const HeadRows& k, hipStream_t stream) {
  if (dtype == kF32) return rotary<F32, D>(a, q, k, stream);
  return dtype == kF16 ? rotary<F16, D>(a, q, k, stream) : rotary<BF16, D>(a, q, k, stream);
}

}  // namespace

int rotary_dispatch(int dtype, int head_dim, const RotaryArgs& a, const HeadRows& q, const HeadRows& k,
                    hipStream_t stream) {
  switch (head_dim) {
    case 16: return rotary_of<16>(dtype, a, q, k, stream);
    case 32: return rotary_of<32>(dtype, a, q, k, stream);
    case 64: return rotary_of<64>(dtype, a, q, k, stream);
    default: return rotary_of<128>(dtype, a, q, k, stream);
  }
}

}  // namespace gki

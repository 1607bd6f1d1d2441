// Attention of few query rows over long streams of keys and values (the rolling cache
// held in 8 bits, cross attention of single tokens), for gfx950.
//
// A stream is the K / V rows of one (b, kv head); the rows that read it are the
// group * n_q query rows of that head's group. For each of them
//   S_t = scale * q . k_t,  O = sum_t exp(S_t - m) v_t / sum_t exp(S_t - m),
//   LSE = m + ln(sum),  m the largest S_t,
// over the stream's visible tokens t; a row that sees none has O = 0, LSE = 0.
// The work is bound by reading K and V once (HBM): a workgroup takes an equal
// slice of a stream's tokens for up to 32 of its rows, and the slices' states
// (max, sum, accumulator, all fp32) are joined by join_kernel when there are
// several.
//
// 8-bit rows. A row x of D values is stored as D e4m3 codes and one byte e + 127:
// e is the smallest integer (at least -117) with max |x_i| <= 448 * 2^e, code i the
// e4m3 number nearest to x_i * 2^-e (ties to even). The scale is a power of two
// so that the division is exact and the codes do not depend on how it is carried
// out, and so that a stored value, code * 2^e, is a bfloat16: it enters the matrix
// cores as it is, whatever the type of the queries. An e4m3 number has 4 significant
// bits whatever its exponent, so a scale closer to the row's maximum would gain
// nothing above the subnormal codes (below 2^-14.8 of the maximum). Infinities and
// NaN are stored as NaN; the scale is that of the finite values.
#include <algorithm>
#include <string>

#include "gki_join.cuh"
#include "gki_rows16.cuh"

namespace gki {
namespace {

constexpr int kMinExponent = -117;           // 2^-9 (the smallest code) * 2^-117 is a normal float
constexpr float kStreamSlack = 8.f;          // log2 units the lazy reference max may lag (p <= 2^8)

// ---------------------------------------------------------------------------
// Writing and reading back.
// ---------------------------------------------------------------------------
// Eight consecutive elements as floats, and back.
template <typename T>
__device__ inline void load8(const typename T::storage* p, float (&f)[8]) {
  if constexpr (T::is_f32) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 w = *(const uint4*)p;
    const uint16_t* h = (const uint16_t*)&w;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = T::to_float(h[i]);
  }
}

// Rows that a launch writes into a rolling cache: of n_new from position start on, the
// first n_a and n_b from the i_b-th on (surviving_rows).
struct AppendRows {
  int n_new, n_a, i_b, n_b, start, sink, ring;
  __device__ inline int source(int r) const { return r < n_a ? r : i_b + (r - n_a); }
  __device__ inline int slot(int i) const {
    const int p = start + i;
    return p < sink ? p : sink + (p - sink) % ring;
  }
};
struct AppendArgs {
  void *kc, *vc;
  uint8_t *ks, *vs;            // exponents of the 8-bit rows
  const void *kn, *vn;
  int BH;
  AppendRows rows;
  int n_blocks;                // workgroups that write (0: none)
};

// Eight elements of a row, and the largest finite magnitude among them.
template <typename T>
__device__ inline float load8_top(const typename T::storage* p, float (&f)[8]) {
  load8<T>(p, f);
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = fabsf(f[j]);
    top = fmaxf(top, x < __builtin_huge_valf() ? x : 0.f);     // false for NaN too
  }
  return top;
}
// The exponent of a row: top = (1 + m / 2^23) 2^k <= 448 * 2^e = 1.75 * 2^(8 + e).
__device__ inline int exponent_of(float top) {
  const uint32_t bits = __float_as_uint(top);
  return max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0), kMinExponent);
}
// The codes of eight elements of a row of exponent e.
__device__ inline uint2 codes8(const float (&f)[8], int e) {
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = fabsf(f[j]) < __builtin_huge_valf() ? f[j] * inv : __builtin_nanf("");
  int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
  int w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
  return make_uint2((uint32_t)w0, (uint32_t)w1);
}

// D / 8 lanes per row of K or V, eight elements each; in 8 bits the largest magnitude
// goes round among them. Bound by HBM: reads the rows once, writes them once.
template <typename T, int D, bool EIGHT>
__device__ inline void append_rows(const AppendArgs& a, int block) {
  using S = typename T::storage;
  constexpr int LPR = D / 8;                   // lanes per row
  const int rows = a.rows.n_a + a.rows.n_b;
  const int ch = threadIdx.x % LPR;
  const int64_t n = (int64_t)a.BH * rows;
  // whole rows: the lanes of a row leave together
  for (int64_t row = ((int64_t)block * 256 + threadIdx.x) / LPR; row < 2 * n; row += (int64_t)a.n_blocks * (256 / LPR)) {
    const bool is_v = row >= n;
    const int64_t rr = is_v ? row - n : row;
    const int bh = (int)(rr / rows), i = a.rows.source((int)(rr % rows));
    const S* src = (const S*)(is_v ? a.vn : a.kn) + ((size_t)bh * a.rows.n_new + i) * D + 8 * ch;
    const size_t dst = (size_t)bh * (a.rows.sink + a.rows.ring) + a.rows.slot(i);
    if constexpr (EIGHT) {
      float f[8];
      float top = load8_top<T>(src, f);
#pragma unroll
      for (int off = 1; off < LPR; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
      const int e = exponent_of(top);
      *(uint2*)((uint8_t*)(is_v ? a.vc : a.kc) + dst * D + 8 * ch) = codes8(f, e);
      if (ch == 0) (is_v ? a.vs : a.ks)[dst] = (uint8_t)(e + 127);
    } else {
      static_assert(!T::is_f32 || EIGHT, "16-bit rows");
      *(uint4*)((S*)(is_v ? a.vc : a.kc) + dst * D + 8 * ch) = *(const uint4*)src;
    }
  }
}
template <typename T, int D>
__global__ __launch_bounds__(256) void append8_kernel(AppendArgs a) {
  append_rows<T, D, true>(a, blockIdx.x);
}

// Two e4m3 codes of a word (its low or high half) times 2^e: exact in fp32.
__device__ inline f32x2 codes2(uint32_t w, bool high, float scale) {
  const auto x = high ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  return f32x2{x[0] * scale, x[1] * scale};
}
__device__ inline float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

// The held rows in ascending order of position, as values of the cache's type, and
// the positions. Row r < n_sink is position r, any other lo + r - n_sink. Eight
// values per lane; bound by HBM.
struct HeldRows {
  int n, n_sink, lo, sink, ring;
  __device__ inline int position(int r) const { return r < n_sink ? r : lo + (r - n_sink); }
  __device__ inline int slot(int r) const {
    const int p = position(r);
    return p < sink ? p : sink + (p - sink) % ring;
  }
};
template <typename T, int D, bool EIGHT>
__global__ __launch_bounds__(256) void held_rows_kernel(
    const void* __restrict__ kc, const void* __restrict__ vc, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, typename T::storage* __restrict__ ko, typename T::storage* __restrict__ vo,
    int64_t* __restrict__ positions, int BH, HeldRows a) {
  using S = typename T::storage;
  constexpr int LPR = D / 8;
  const int ch = threadIdx.x % LPR;
  const int64_t n = (int64_t)BH * a.n;
  for (int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR; row < 2 * n;
       row += (int64_t)gridDim.x * (256 / LPR)) {
    const bool is_v = row >= n;
    const int64_t rr = is_v ? row - n : row;
    const int bh = (int)(rr / a.n), r = (int)(rr % a.n);
    if (row < a.n && ch == 0) positions[r] = a.position(r);
    const size_t src = (size_t)bh * (a.sink + a.ring) + a.slot(r);
    S* dst = (is_v ? vo : ko) + (size_t)rr * D + 8 * ch;
    if constexpr (EIGHT) {
      const float s = scale_of((is_v ? vs : ks)[src]);
      const uint2 w = *(const uint2*)((const uint8_t*)(is_v ? vc : kc) + src * D + 8 * ch);
      const f32x2 x[4] = {codes2(w.x, false, s), codes2(w.x, true, s), codes2(w.y, false, s), codes2(w.y, true, s)};
      if constexpr (T::is_f32) {
        *(float4*)dst = make_float4(x[0][0], x[0][1], x[1][0], x[1][1]);
        *(float4*)(dst + 4) = make_float4(x[2][0], x[2][1], x[3][0], x[3][1]);
      } else {
        *(uint4*)dst = make_uint4(pack2<T>(x[0][0], x[0][1]), pack2<T>(x[1][0], x[1][1]), pack2<T>(x[2][0], x[2][1]),
                                  pack2<T>(x[3][0], x[3][1]));
      }
    } else {
      const S* from = (const S*)(is_v ? vc : kc) + src * D + 8 * ch;
      *(uint4*)dst = *(const uint4*)from;
      if constexpr (T::is_f32) *(uint4*)(dst + 4) = *(const uint4*)(from + 4);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------
// The tokens of a rolling cache that some of its n_q last positions see: sinks
// 0 .. n_sink - 1, then positions w_lo .. length - 1.
struct RingStream {
  static constexpr bool kSteps = true;         // a step's own tokens may be among them
  int n_tokens, n_sink, w_lo, sink, ring, base, q_off, window;   // base: (w_lo - sink) mod ring
  __device__ inline int count(int) const { return n_tokens; }
  __device__ inline int row(int t) const {
    if (t < n_sink) return t;
    const int j = base + (t - n_sink);
    return sink + (j >= ring ? j - ring : j);
  }
  __device__ inline int position(int t) const { return t < n_sink ? t : w_lo + (t - n_sink); }
  // Do tokens t .. t + n - 1 lie in consecutive rows (all sinks, or window tokens that
  // the ring does not turn between)?
  __device__ inline bool consecutive(int t, int n) const {
    return t + n <= n_sink || (t >= n_sink && (base + (t - n_sink) >= ring || base + (t - n_sink) + n <= ring));
  }
  // Does some row not see some of them?
  __device__ inline bool partly_hidden(int t, int n) const {
    const int p0 = position(t), p1 = position(t + n - 1);
    return p1 > q_off || (p1 >= sink && max(p0, sink) <= n_tok_last() - window);
  }
  __device__ inline int n_tok_last() const { return w_lo + (n_tokens - n_sink) - 1; }   // the last query's position
  // token rule of query position i
  __device__ inline bool visible(int i, int t) const {
    const int p = position(t), qa = q_off + i;
    return (p <= qa) & ((p < sink) | (p > qa - window));
  }
};

// A contiguous stream per (b, kv head): all its rows, or the first len[b] of them (a
// length outside 0 .. n counts as the nearest).
struct DenseStream {
  static constexpr bool kSteps = false;
  const int32_t* len;
  int n, H_kv;
  __device__ inline int count(int s) const {
    return len == nullptr ? n : max(0, min(__builtin_amdgcn_readfirstlane(len[s / H_kv]), n));
  }
  __device__ inline int row(int t) const { return t; }
  __device__ inline int position(int t) const { return t; }
  __device__ inline bool consecutive(int, int) const { return true; }
  __device__ inline bool partly_hidden(int, int) const { return false; }
  __device__ inline bool visible(int, int) const { return true; }
};

struct StreamArgs {
  const void *q, *k, *v;
  const uint8_t *ks, *vs;      // exponents of the 8-bit rows
  void* o;
  float* lse;
  float *acc, *ml;             // states of the slices: [rows][n_parts][D] and [rows][n_parts][2]
  int H_kv, rb;                // rb = group * n_q: rows of Q that one (b, kv head) has, one after another
  int n_q, q_stride;           // q_stride = H * n_q rows of Q between batch entries
  int kv_rows;                 // rows that K and V hold per stream
  int n_rows, row_tiles;       // query rows of a stream, and tiles of them
  int n_blocks;                // workgroups: streams * n_splits * row_tiles
  int n_splits;                // slices here: parts part0 .. of the n_parts states that a row has in the
  int part0, n_parts;          // workspace (n_parts 1: O and LSE are written here)
  float scale_log2;            // |scale| log2 e (log2 e for scale 0), the sign in q_sign
  float q_sign;                // 1, -1, or 0: the scores are those of q_sign * q
  // A step's own tokens, positions start .. of which each stream has n_new rows here, are
  // taken from these rows: the cache's are being written by the same launch. (Their
  // slots held positions at least `ring` older, which no row of the step sees.)
  const void *k_new, *v_new;
  int n_new, start;            // no such tokens: start past every position
};

// Queries as 1, 2 or 3 bfloat16 pieces whose sum they are (8, 11 and 24 significant
// bits), so that products with the stored values are those of the queries themselves.
template <typename T> constexpr int kPieces = std::is_same<T, BF16>::value ? 1 : std::is_same<T, F16>::value ? 2 : 3;

template <typename C, int NPC>
__device__ inline void split8(float (&f)[8], uint4 (&piece)[NPC]) {
#pragma unroll
  for (int n = 0; n < NPC; ++n) {
    piece[n] = make_uint4(pack2<C>(f[0], f[1]), pack2<C>(f[2], f[3]), pack2<C>(f[4], f[5]), pack2<C>(f[6], f[7]));
    if (n + 1 < NPC) {
      const uint16_t* h = (const uint16_t*)&piece[n];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] -= C::to_float(h[i]);
    }
  }
}

// Where a workgroup works: 16 NB query rows (from row0 on) of stream s against the
// slice [g0, g1) of its tokens. Row tiles of a slice are neighbours on one XCD.
struct StreamPlace {
  int s, row0, split, g0, g1;
  size_t q_row0, kb;           // the stream's first row of Q, of K and V
  template <class Src>
  __device__ inline StreamPlace(const StreamArgs& a, const Src& src, int rows_tile, int block) {
    int lb = xcd_remap(block, a.n_blocks);
    row0 = lb % a.row_tiles * rows_tile;
    lb /= a.row_tiles;
    split = lb % a.n_splits;
    s = lb / a.n_splits;
    q_row0 = (size_t)(s / a.H_kv) * a.q_stride + (size_t)(s % a.H_kv) * a.rb;
    kb = (size_t)s * a.kv_rows;
    const int n_tok = src.count(s);
    g0 = (int)(((int64_t)n_tok * split) / a.n_splits);
    g1 = (int)(((int64_t)n_tok * (split + 1)) / a.n_splits);
  }
  // Row r of the stream in Q: a shared prefix is read by rb rows of each sequence.
  __device__ inline size_t q_row(const StreamArgs& a, int r) const {
    return a.n_rows == a.rb ? q_row0 + r : q_row0 + (size_t)(r / a.rb) * a.q_stride + r % a.rb;
  }
  __device__ inline int steps(int tokens) const { return (g1 - g0 + tokens - 1) / tokens; }
};

// A step's 128 rows of D codes in LDS: row-major, 16-byte chunks XOR-swizzled so that both
// kinds of reads are free of conflicts: 16 bytes of rows {0-3, 8-11, 16-19, 24-27} (+ 4)
// at one chunk, and transposed reads of 16 consecutive rows at one chunk.
constexpr int kStep8 = 128;
template <int D>
__device__ inline int code_swz(int row) {
  const int b3 = (row >> 3) & 1, b24 = ((row >> 2) ^ (row >> 4)) & 1;
  return D >= 128 ? ((row >> 1) & 1) | b3 << 1 | b24 << 2 : b3 | b24 << 1;
}
template <int D>
__device__ inline int code_off(int row, int byte) {
  return row * D + (((byte >> 4) ^ code_swz<D>(row)) << 4) + (byte & 15);
}
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
// Eight codes times a power of two, as bfloat16 (exact).
__device__ inline uint4 bf16x8_of(uint32_t lo, uint32_t hi, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)));
}
// One byte per lane to LDS dwords, lane i at lds + 4 i.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void dma_load1(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_ubyte %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

// One transposed read as lds_tr4's, of the rows rho(t, 4 g + e) that lane group g's
// scores of subtile t belong to.
template <int D>
__device__ inline uint2 lds_tr4_rho(const uint16_t* tile, int t, int n0, int lane) {
  const int g = lane >> 4, l = lane & 15;
  const uint16_t* p = tile + lds_off<D>(rho(t, 4 * g + (l >> 2)), n0 + 4 * (l & 3));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)p));
}

// A wave's share of a workgroup of four: 16 NB query rows, as columns of S^T = K Q^T on
// v_mfma_f32_16x16x32, against 16 of the 64 tokens of each step (tiles of element
// type C in LDS; the wave's tokens are those of subtile rho(wave, .), whose rows the
// swizzle serves without conflicts), with a softmax state of its own. NPC: pieces of the queries and of
// the probabilities. The reference max is lazy: it moves when a score exceeds it by
// the slack, so that the rescale almost never runs.
template <typename T, typename C, int D, int NB, int NPC, bool RULE, bool EIGHT>
struct StreamWave {
  static constexpr int KS = D / 32, DT = D / 16;
  uint4 qf[NB][KS][NPC];
  floatx4 o[NB][DT];
  float lsum[NB], m[NB];
  int my_q[NB], wave, lane, grp, col;

  __device__ inline StreamWave(const StreamArgs& a, const StreamPlace& at) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    grp = lane >> 4, col = lane & 15;
    // Q^T operand of column block h: lane (grp, col) holds elements 32 ks + 8 grp .. +7
    // (EIGHT: 64 (ks / 2) + 16 grp + 8 (ks % 2) .. +7) of row row0 + 16 h + col
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      const int r = at.row0 + 16 * h + col;
      my_q[h] = r % a.n_q;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float f[8];
        load8<T>((const typename T::storage*)a.q + at.q_row(a, r < a.n_rows ? r : 0) * D +
                     (EIGHT ? 64 * (ks >> 1) + 16 * grp + 8 * (ks & 1) : 32 * ks + 8 * grp), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = r < a.n_rows && a.q_sign != 0.f ? f[i] * a.q_sign : 0.f;
        split8<C>(f, qf[h][ks]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[h][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
      lsum[h] = 0.f;
      m[h] = kNegInf;
    }
  }

  // The reference max follows the rows' largest score (scaled, the lane's mx) where some
  // row's exceeds it by the slack.
  __device__ inline void move_max(int h, float mx) {
    if (__any(mx > m[h] + kStreamSlack)) {
      mx = wave_max16x4(mx);
      const bool grow = mx > m[h] + kStreamSlack;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m[h] - mx) : 1.f;
      m[h] = grow ? mx : m[h];
      lsum[h] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[h][dt] *= alpha;
    }
  }

  // The wave's 16 tokens of the step of 64 that starts at token t; g1 ends the slice.
  template <class Src>
  __device__ inline void step(const StreamArgs& a, const Src& src, const uint16_t* ck, const uint16_t* cv, int t, int g1) {
    floatx4 s[NB];
#pragma unroll
    for (int h = 0; h < NB; ++h) s[h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 x = lds_row8<D>(ck, rho(wave, col), 32 * ks + 8 * grp);
#pragma unroll
      for (int h = 0; h < NB; ++h) s[h] = C::mfma(x, qf[h][ks][0], s[h]);
    }
    // lane (grp, col): s[h][i] = score of token t + rho(wave, 4 grp + i) for row row0 + 16 h + col
    if (t + kTileN > g1 || (RULE && src.partly_hidden(t, kTileN))) {
      const int t0 = t + rho(wave, 4 * grp);
#pragma unroll
      for (int h = 0; h < NB; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bool ok = t0 + i < g1;
          if constexpr (RULE) ok = ok && src.visible(my_q[h], t0 + i);
          s[h][i] = ok ? s[h][i] : kNegInf;
        }
    }
    uint2 pb[NB];
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      move_max(h, fmaxf(fmaxf(s[h][0], s[h][1]), fmaxf(s[h][2], s[h][3])) * a.scale_log2);
      const float m_use = m[h] == kNegInf ? 0.f : m[h];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i], a.scale_log2, -m_use));
      lsum[h] += (s[h][0] + s[h][1]) + (s[h][2] + s[h][3]);
      pb[h] = make_uint2(pack2<C>(s[h][0], s[h][1]), pack2<C>(s[h][2], s[h][3]));
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint2 x = lds_tr4_rho<D>(cv, wave, 16 * dt, lane);
#pragma unroll
      for (int h = 0; h < NB; ++h) o[h][dt] = mfma16k<C>(x, pb[h], o[h][dt]);
    }
  }

  // The wave's 32 tokens (tile rows 32 wave ..) of the step of 128 over 8-bit rows that
  // starts at token t. A lane's 16 codes of a K row feed two products (the queries list
  // their elements in the same order), its scores belong to tokens 8 grp + 4 u + i: with
  // their V row's power of two they are the operand of V^T, eight tokens of a column by
  // one transposed read.
  template <class Src>
  __device__ inline void step8(const StreamArgs& a, const Src& src, const uint8_t* ck, const uint8_t* cv,
                               const uint32_t* ks, const uint32_t* vs, int t, int g1) {
    floatx4 s[NB][2];
#pragma unroll
    for (int h = 0; h < NB; ++h) s[h][0] = s[h][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 32 * wave + rho(u, col);
      const float scale = scale_of(ks[row]);
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const uint4 w = *(const uint4*)(ck + code_off<D>(row, 64 * j + 16 * grp));
        const uint4 x = bf16x8_of(w.x, w.y, scale), y = bf16x8_of(w.z, w.w, scale);
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int n = 0; n < NPC; ++n) {
            s[h][u] = C::mfma(x, qf[h][2 * j][n], s[h][u]);
            s[h][u] = C::mfma(y, qf[h][2 * j + 1][n], s[h][u]);
          }
      }
    }
    const int t0 = t + 32 * wave + 8 * grp;
    if (t + kStep8 > g1 || (RULE && src.partly_hidden(t, kStep8))) {
#pragma unroll
      for (int h = 0; h < NB; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool ok = t0 + 4 * u + i < g1;
            if constexpr (RULE) ok = ok && src.visible(my_q[h], t0 + 4 * u + i);
            s[h][u][i] = ok ? s[h][u][i] : kNegInf;
          }
    }
    floatx4 sv[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint4 e = *(const uint4*)(vs + 32 * wave + 8 * grp + 4 * u);
      sv[u] = floatx4{scale_of(e.x), scale_of(e.y), scale_of(e.z), scale_of(e.w)};
    }
    uint4 pb[NB][NPC];
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[h][u][i]);
      move_max(h, mx * a.scale_log2);
      const float m_use = m[h] == kNegInf ? 0.f : m[h];
      float f[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[h][u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][u][i], a.scale_log2, -m_use));
          f[4 * u + i] = s[h][u][i] * sv[u][i];
        }
        lsum[h] += (s[h][u][0] + s[h][u][1]) + (s[h][u][2] + s[h][u][3]);
      }
      split8<C>(f, pb[h]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int l = lane & 15;
      const uint8_t* v = cv + code_off<D>(32 * wave + 8 * grp + (l >> 1), 16 * dt + 8 * (l & 1));
      const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)v);
      const uint4 x = bf16x8_of((uint32_t)w.x, (uint32_t)w.y, 1.f);
#pragma unroll
      for (int h = 0; h < NB; ++h)
#pragma unroll
        for (int n = 0; n < NPC; ++n) o[h][dt] = C::mfma(x, pb[h][n], o[h][dt]);
    }
  }

  // The four waves' states meet in LDS (wacc: 64 D floats, wml: 128), one column block
  // at a time: lane (grp, col) holds O^T rows 16 dt + 4 grp + i of row row0 + 16 h + col.
  __device__ inline void finish(const StreamArgs& a, const StreamPlace& at, float* wacc, float* wml) {
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      const float lw = wave_sum16x4(lsum[h]);
      __syncthreads();                         // the tiles' (or the previous block's) readers are done
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *(floatx4*)(wacc + (wave * 16 + col) * D + 16 * dt + 4 * grp) = o[h][dt];
      if (grp == 0) {
        wml[(wave * 16 + col) * 2] = m[h];
        wml[(wave * 16 + col) * 2 + 1] = lw;
      }
      __syncthreads();
      const int rows_h = min(16, a.n_rows - at.row0 - 16 * h);
      for (int idx = threadIdx.x; idx < rows_h * (D / 4); idx += 256) {
        const int rl = idx / (D / 4), d = 4 * (idx % (D / 4));
        const size_t row = at.q_row(a, at.row0 + 16 * h + rl);
        float M = kNegInf;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, wml[(w * 16 + rl) * 2]);
        const float Mu = M == kNegInf ? 0.f : M;
        float L = 0.f;
        floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = __builtin_amdgcn_exp2f(wml[(w * 16 + rl) * 2] - Mu);
          L += wml[(w * 16 + rl) * 2 + 1] * f;
          x += *(const floatx4*)(wacc + (w * 16 + rl) * D + d) * f;
        }
        if (a.n_parts == 1) {
          x = x / (L == 0.f ? 1.f : L);        // no visible token: 0; NaN stays NaN
          typename T::storage* dst = (typename T::storage*)a.o + row * D + d;
          if constexpr (T::is_f32) *(floatx4*)dst = x;
          else *(uint2*)dst = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
          if (d == 0) a.lse[row] = L == 0.f ? 0.f : lse_natural(M, L);
        } else {
          *(floatx4*)(a.acc + (row * a.n_parts + a.part0 + at.split) * D + d) = x;
          if (d == 0) *(float2*)(a.ml + (row * a.n_parts + a.part0 + at.split) * 2) = make_float2(M, L);
        }
      }
    }
  }
};

// Over 8-bit rows: codes and exponents gathered into LDS by LDS-DMA as they are, two
// steps of 128 tokens in flight (non-temporal: 6.6 against 5.9 TB/s on 1.08 GB; staged
// through registers, half as much in flight, 256 streams of 2048 took 34 us for 23), turned into bfloat16 as operands
// (v_cvt_scalef32_pk_bf16_fp8). fp16 and fp32 queries, and their probabilities, are 2 and
// 3 bfloat16 pieces: 2 and 3 times the products, for which the memory-bound stream
// leaves room. bf16: P is rounded to bfloat16 for P V, as in the 16-bit decode (half a
// unit of 2^-8 of each weight, averaged over the keys); the row sums add the fp32 P.
template <typename T, int D, int NB, bool RULE, class Src>
__device__ inline void stream8_rows(const StreamArgs& a, const Src& src, int block, uint16_t* sk, uint16_t* sv,
                                    uint32_t* sc) {
  using S = typename T::storage;
  constexpr int NP = kStep8 * D / 4096;        // 1 KB LDS blocks per wave and tensor
  constexpr int TILE = kStep8 * D;
  constexpr int UPR = D / 16;                  // 16-byte units per row
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const StreamPlace at(a, src, 16 * NB, block);
  const bool once = a.row_tiles == 1;          // no other workgroup reads these rows
  const int n_steps = at.steps(kStep8);
  const uint8_t *K = (const uint8_t*)a.k + at.kb * D, *V = (const uint8_t*)a.v + at.kb * D;
  const uint8_t* E = (wave < 2 ? a.ks : a.vs) + at.kb;     // exponents: waves 0, 1 K's, 2, 3 V's, 64 rows each
  uint8_t *rk = (uint8_t*)sk, *rv = (uint8_t*)sv;
  StreamWave<T, BF16, D, NB, kPieces<T>, RULE, true> w(a, at);
  dma_wait();   // the Q loads are complete before any LDS-DMA is in flight

  int drow[NP], doff[NP];                      // the lane's row of its LDS blocks, and where its codes are in a tile
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int e = (4 * p + wave) * 1024 + 16 * lane;
    drow[p] = e / D;
    doff[p] = (((e % D) >> 4) ^ code_swz<D>(drow[p])) << 4;
  }
  const int erow = 64 * (wave & 1) + lane;
  auto first_token = [&](int c) { return at.g0 + c * kStep8; };
  // Does a step hold tokens that the step writes, or rows past the slice that the loads
  // do not leave out? These are put right in LDS.
  auto whole = [&](int t, int n) { return src.consecutive(t, n) && src.position(t + n - 1) < a.start; };
  auto issue = [&](int c, int b) {
    const int t = first_token(c), n = min(kStep8, at.g1 - t);
    const uint32_t lk = lds_addr(rk + b * TILE), lv = lds_addr(rv + b * TILE);
    const uint32_t le = lds_addr(sc + (2 * b + (wave >> 1)) * kStep8 + 64 * (wave & 1));
    if (whole(t, n)) {
      // rows one after another: resources over those that the slice has (past them zeros),
      // the lane's offsets the same for every step
      const size_t row = (size_t)src.row(t);
      const i32x4 qk = buffer_rsrc(K + row * D, n * D), qv = buffer_rsrc(V + row * D, n * D);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        dma_buf16(qk, drow[p] * D + doff[p], lk + (4 * p + wave) * 1024, once);
        dma_buf16(qv, drow[p] * D + doff[p], lv + (4 * p + wave) * 1024, once);
      }
      dma_load1(E + row + min(erow, n - 1), le);
    } else {
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const size_t row = (size_t)src.row(min(t + drow[p], at.g1 - 1));
        dma_load16(K + row * D + doff[p], lk + (4 * p + wave) * 1024, once);
        dma_load16(V + row * D + doff[p], lv + (4 * p + wave) * 1024, once);
      }
      dma_load1(E + src.row(min(t + erow, at.g1 - 1)), le);
    }
  };
  // A step that is not whole: rows past the slice zeros, and the step's own tokens
  // quantised here as append_rows quantises them (16 codes of K or V per lane).
  auto mend = [&](int c, int b) {
    const int t = first_token(c), n = min(kStep8, at.g1 - t);
    for (int i = tid; i < (kStep8 - n) * UPR; i += 256) {
      const int row = n + i / UPR;
      *(uint4*)(rk + b * TILE + row * D + 16 * (i % UPR)) = make_uint4(0, 0, 0, 0);
      *(uint4*)(rv + b * TILE + row * D + 16 * (i % UPR)) = make_uint4(0, 0, 0, 0);
    }
    const int fresh = min(n, src.position(t + n - 1) - a.start + 1);     // the last ones of the step
    if (fresh > 0) {
      const int x = tid / UPR, row = n - fresh + x / 2, is_v = x & 1, ch = tid % UPR;
      const int i = src.position(t + min(row, n - 1)) - a.start;
      const bool mine = x < 2 * fresh && i >= 0;
      const S* p = (const S*)(is_v ? a.v_new : a.k_new) + ((size_t)at.s * a.n_new + max(i, 0)) * D + 16 * ch;
      float lo[8], hi[8];
      float top = fmaxf(load8_top<T>(p, lo), load8_top<T>(p + 8, hi));
#pragma unroll
      for (int o = 1; o < UPR; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
      const int e = exponent_of(top);
      const uint2 u = codes8(lo, e), v = codes8(hi, e);
      if (mine) {
        *(uint4*)((is_v ? rv : rk) + b * TILE + code_off<D>(row, 16 * ch)) = make_uint4(u.x, u.y, v.x, v.y);
        if (ch == 0) sc[(2 * b + is_v) * kStep8 + row] = (uint32_t)(e + 127);
      }
    }
  };
  if (n_steps > 0) issue(0, 0);
  if (n_steps > 1) issue(1, 1);
  for (int c = 0; c < n_steps; ++c) {
    const int b = c & 1, t = first_token(c);
    if (c + 1 < n_steps) vm_wait<2 * NP + 1>();   // step c has landed, the next may be in flight
    else vm_wait<0>();
    __syncthreads();
    if (!whole(t, min(kStep8, at.g1 - t))) {
      mend(c, b);
      __syncthreads();
    }
    w.step8(a, src, rk + b * TILE, rv + b * TILE, sc + 2 * b * kStep8, sc + (2 * b + 1) * kStep8, t, at.g1);
    __syncthreads();                           // every wave is done with buffer b
    if (c + 2 < n_steps) issue(c + 2, b);
  }
  w.finish(a, at, (float*)sk, (float*)sv);
}

// Over 16-bit rows: gathered into LDS by LDS-DMA, two steps in flight, so that no
// registers hold loads (non-temporal: 6.9 against 6.2 TB/s on 4.2 GB of D128 keys and
// values, 6.6 against 5.9 on 0.8 GB of D64).
template <typename T, int D, int NB, bool RULE, class Src>
__device__ inline void stream16_rows(const StreamArgs& a, const Src& src, int block, uint16_t* sk, uint16_t* sv) {
  constexpr int NP = D / 32;                   // 1 KB LDS blocks per wave and 64-row tile
  constexpr int TILE = kTileN * D;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const StreamPlace at(a, src, 16 * NB, block);
  const bool once = a.row_tiles == 1;
  const int n_chunks = at.steps(kTileN);
  const uint16_t *K = (const uint16_t*)a.k + at.kb * D, *V = (const uint16_t*)a.v + at.kb * D;
  StreamWave<T, T, D, NB, 1, RULE, false> w(a, at);
  dma_wait();   // the Q loads are complete before any LDS-DMA is in flight

  // the lane's chunk of LDS block 4 p + wave of a tile: row, swizzled column
  int drow[NP], dcol[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int e = (4 * p + wave) * 512 + 8 * lane;
    drow[p] = e / D;
    dcol[p] = (((e % D) >> 3) ^ lds_swz<D>(drow[p])) << 3;
  }
  auto issue = [&](int c, int b) {
    const uint32_t lk = lds_addr(sk + b * TILE), lv = lds_addr(sv + b * TILE);
    const int t = at.g0 + c * kTileN, n = min(kTileN, at.g1 - t);
    if (src.consecutive(t, n) && src.position(t + n - 1) < a.start) {
      // rows one after another: resources over those that the slice has (past them zeros),
      // the lane's offsets the same for every step
      const size_t row = (size_t)src.row(t) * D;
      const i32x4 rk = buffer_rsrc(K + row, n * D * 2), rv = buffer_rsrc(V + row, n * D * 2);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int off = 2 * (drow[p] * D + dcol[p]);
        dma_buf16(rk, off, lk + (4 * p + wave) * 1024, once);
        dma_buf16(rv, off, lv + (4 * p + wave) * 1024, once);
      }
      return;
    }
    // tokens past the slice repeat its last one and are masked when consumed
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int x = min(t + drow[p], at.g1 - 1);
      const uint16_t *kt = K + (size_t)src.row(x) * D, *vt = V + (size_t)src.row(x) * D;
      if constexpr (Src::kSteps) {
        const int i = src.position(x) - a.start;
        if (i >= 0) {
          const size_t own = ((size_t)at.s * a.n_new + i) * D;
          kt = (const uint16_t*)a.k_new + own, vt = (const uint16_t*)a.v_new + own;
        }
      }
      dma_load16(kt + dcol[p], lk + (4 * p + wave) * 1024, once);
      dma_load16(vt + dcol[p], lv + (4 * p + wave) * 1024, once);
    }
  };
  if (n_chunks > 0) issue(0, 0);
  if (n_chunks > 1) issue(1, 1);
  for (int c = 0; c < n_chunks; ++c) {
    const int b = c & 1;
    wait_chunks<NP, 2>(min(1, n_chunks - 1 - c));   // chunk c has landed
    __syncthreads();
    w.step(a, src, sk + b * TILE, sv + b * TILE, at.g0 + c * kTileN, at.g1);
    __syncthreads();                           // every wave is done with buffer b
    if (c + 2 < n_chunks) issue(c + 2, b);
  }
  w.finish(a, at, (float*)sk, (float*)sv);
}

template <typename T, int D, int NB, bool RULE, bool EIGHT, class Src>
__device__ inline void stream_rows(const StreamArgs& a, const Src& src, int block, uint16_t* sk, uint16_t* sv) {
  __shared__ __align__(16) uint32_t sc[2][2][kStep8];      // 8-bit: exponents of K and V rows
  if constexpr (EIGHT) stream8_rows<T, D, NB, RULE>(a, src, block, sk, sv, &sc[0][0][0]);
  else stream16_rows<T, D, NB, RULE>(a, src, block, sk, sv);
}

// Waves per SIMD that the registers must leave room for: as many workgroups per CU as
// their LDS allows (two at head_dim 128, four at 64, one less there with two row blocks
// or three pieces).
template <typename T, int D, int NB> constexpr int kStreamWaves = D >= 128 ? 2 : NB == 1 && !T::is_f32 ? 4 : 3;

// Streams, then the workgroups that write a step's tokens into the cache.
template <typename T, int D, int NB, bool RULE, bool EIGHT, class Src>
__global__ __launch_bounds__(256, (kStreamWaves<T, D, NB>)) void stream_kernel(StreamArgs a, Src src, AppendArgs ap) {
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];
  if constexpr (Src::kSteps) {
    if ((int)blockIdx.x >= a.n_blocks) {
      append_rows<T, D, EIGHT>(ap, blockIdx.x - a.n_blocks);
      return;
    }
  }
  stream_rows<T, D, NB, RULE, EIGHT>(a, src, blockIdx.x, &sk[0][0], &sv[0][0]);
}

// The sequences' own streams in a launch with the shared prefix's workgroups, which come
// first: with about one of those per CU each CU gets one of the matrix cores' kind and
// one of the memory's (in turn, they went by two of a kind to each CU).
template <typename T, int D, int NB, bool EIGHT>
struct OwnStreams {
  StreamArgs a;
  RingStream src;
  AppendArgs ap;
  int shared_blocks;           // a multiple of the XCDs
  // Is the workgroup one of these? Its index among its kind.
  __device__ inline bool takes(int& block) const {
    const int own = block - shared_blocks;
    block = own >= 0 ? own : block;
    return own >= 0;
  }
  __device__ inline void run(int block, uint16_t* sk, uint16_t* sv) const {
    if (block < a.n_blocks) stream_rows<T, D, NB, true, EIGHT>(a, src, block, sk, sv);
    else if (block < a.n_blocks + ap.n_blocks) append_rows<T, D, EIGHT>(ap, block - a.n_blocks);
  }
};

// A shared prefix of few rows as streams, and the sequences' own.
template <typename T, int D, class Beside>
__global__ __launch_bounds__(256, (kStreamWaves<T, D, 2>)) void prefix_streams_kernel(StreamArgs a, DenseStream src, Beside beside) {
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];
  int block = blockIdx.x;
  if (beside.takes(block)) beside.run(block, &sk[0][0], &sv[0][0]);
  else if (block < a.n_blocks) stream_rows<T, D, 2, false, false>(a, src, block, &sk[0][0], &sv[0][0]);
}

// A workgroup per 256 lanes of work, up to a grid whose lanes a launch can count.
inline dim3 row_grid(int64_t lanes) { return dim3((unsigned)std::min<int64_t>((lanes + 255) / 256, 1 << 20)); }

// Workgroups that write the rows of `a`.
inline int append_blocks(const AppendArgs& a, int head_dim) {
  const int64_t lanes = 2 * (int64_t)a.BH * (a.rows.n_a + a.rows.n_b) * (head_dim / 8);
  return (int)row_grid(lanes).x;
}

inline void set_rows(StreamArgs& a, int n_streams, int tile) {
  a.row_tiles = (a.n_rows + tile - 1) / tile;
  a.n_blocks = n_streams * a.n_splits * a.row_tiles;
}

// The streams of a launch in row tiles of the size that their rows take.
template <typename T, int D, bool EIGHT, class Src>
void launch_streams(StreamArgs a, const Src& src, int n_streams, const AppendArgs& ap, hipStream_t stream) {
  const int tile = stream_rows_tile(EIGHT && kPieces<T> > 1, a.n_rows);
  set_rows(a, n_streams, tile);
#define GKI_STREAM(NB, RULE)                                                                              \
  hipLaunchKernelGGL((stream_kernel<T, D, NB, RULE, EIGHT, Src>), dim3(a.n_blocks + ap.n_blocks), dim3(256), \
                     0, stream, a, src, ap)
  if constexpr (!Src::kSteps) {     // every token is visible to every row
    if (tile == 32) GKI_STREAM(2, false);
    else GKI_STREAM(1, false);
  } else if constexpr (kPieces<T> > 1) {
    if (a.n_q == 1) GKI_STREAM(1, false);
    else GKI_STREAM(1, true);
  } else {
    if (a.n_q == 1 && tile == 32) GKI_STREAM(2, false);
    else if (a.n_q == 1) GKI_STREAM(1, false);
    else if (tile == 32) GKI_STREAM(2, true);
    else GKI_STREAM(1, true);
  }
#undef GKI_STREAM
}

template <typename T, int D>
int cross_stream(const StreamArgs& a, const DenseStream& src, int n_streams, hipStream_t stream) {
  launch_streams<T, D, false>(a, src, n_streams, AppendArgs{}, stream);
  if (a.n_parts > 1) launch_join<T, D, false>(a.acc, a.ml, a.o, a.lse, (int64_t)n_streams * a.rb, a.n_parts, stream);
  return check_launch("gki_cross_fwd");
}

template <typename T, int D>
int attend8(const StreamArgs& a, const RingStream& src, int n_streams, const AppendArgs& ap, hipStream_t stream) {
  launch_streams<T, D, true>(a, src, n_streams, ap, stream);
  if (a.n_parts > 1) launch_join<T, D, false>(a.acc, a.ml, a.o, a.lse, (int64_t)n_streams * a.rb, a.n_parts, stream);
  return check_launch("gki_rolling8_decode");
}

template <typename T, int D, int NB, bool EIGHT>
void launch_prefix(const Geom& g, OwnStreams<T, D, NB, EIGHT> own, StreamArgs shared, int n_prefix, hipStream_t stream) {
  set_rows(own.a, g.B * g.H_kv, 16 * NB);
  const int n_own = own.a.n_blocks + own.ap.n_blocks;
  if (prefix_as_streams(shared.n_rows)) {
    set_rows(shared, g.H_kv, 32);
    own.shared_blocks = kXcd * ((shared.n_blocks + kXcd - 1) / kXcd);
    hipLaunchKernelGGL((prefix_streams_kernel<T, D, OwnStreams<T, D, NB, EIGHT>>), dim3(own.shared_blocks + n_own), dim3(256), 0,
                       stream, shared, DenseStream{nullptr, n_prefix, g.H_kv}, own);
    return;
  }
  Geom pg = g;
  pg.n_q = shared.n_rows;
  pg.n_kv = n_prefix;
  pg.causal = 0;
  const SharedRows sh{shared.n_rows, shared.rb, shared.q_stride, shared.n_splits, shared.part0, shared.n_parts,
                      shared.acc, shared.ml};
  const int n_qt = (shared.n_rows + kTileMF - 1) / kTileMF;
  own.shared_blocks = kXcd * ((n_qt * sh.n_splits * g.H_kv + kXcd - 1) / kXcd);
  hipLaunchKernelGGL((fwd_kernel_16<T, D, kFwdPipe<D>, kShared, OwnStreams<T, D, NB, EIGHT>>), dim3(own.shared_blocks + n_own),
                     dim3(kFwdThreads), 0, stream, pg, (const uint16_t*)shared.q, (const uint16_t*)shared.k,
                     (const uint16_t*)shared.v, (uint16_t*)nullptr, (float*)nullptr, (const int32_t*)nullptr,
                     (const int32_t*)nullptr, n_qt, (const int32_t*)nullptr, sh, own);
}

// A prefix that the sequences share and each sequence's own cache in one launch, then
// their states joined. `own` and `shared` differ in the rows, the keys and the parts.
template <typename T, int D>
int prefix_decode(const Geom& g, const StreamArgs& own, const RingStream& ring, const AppendArgs& ap,
                  const StreamArgs& shared, int n_prefix, hipStream_t stream) {
#define GKI_PREFIX(NB, EIGHT) \
  launch_prefix<T, D, NB, EIGHT>(g, OwnStreams<T, D, NB, EIGHT>{own, ring, ap, 0}, shared, n_prefix, stream)
  const bool wide = stream_rows_tile(own.ks && kPieces<T> > 1, own.n_rows) == 32;
  if (own.ks) {
    if constexpr (kPieces<T> == 1) {
      if (wide) GKI_PREFIX(2, true);
      else GKI_PREFIX(1, true);
    } else {
      GKI_PREFIX(1, true);
    }
  } else if (wide) GKI_PREFIX(2, false);
  else GKI_PREFIX(1, false);
#undef GKI_PREFIX
  launch_join<T, D, false>(own.acc, own.ml, own.o, own.lse, (int64_t)g.B * g.H * g.n_q, own.n_parts, stream);
  return check_launch("gki_rolling_prefix_decode");
}

template <typename T, int D>
int append8(AppendArgs a, hipStream_t stream) {
  a.n_blocks = append_blocks(a, D);
  if (a.n_blocks == 0) return 0;
  hipLaunchKernelGGL((append8_kernel<T, D>), dim3(a.n_blocks), dim3(256), 0, stream, a);
  return check_launch("gki_rolling8_append");
}

template <typename T, int D>
int held_rows(const void* kc, const void* vc, const uint8_t* ks, const uint8_t* vs, void* ko, void* vo,
              int64_t* positions, int BH, const HeldRows& a, hipStream_t stream) {
  using S = typename T::storage;
  const int64_t lanes = 2 * (int64_t)BH * a.n * (D / 8);
  const dim3 grid = row_grid(lanes);
  if (ks) hipLaunchKernelGGL((held_rows_kernel<T, D, true>), grid, dim3(256), 0, stream, kc, vc, ks, vs, (S*)ko, (S*)vo, positions, BH, a);
  else hipLaunchKernelGGL((held_rows_kernel<T, D, false>), grid, dim3(256), 0, stream, kc, vc, ks, vs, (S*)ko, (S*)vo, positions, BH, a);
  return check_launch("gki_rolling_read");
}

}  // namespace

#define GKI_BY_TYPE(FN, ...)                                                        \
  if (head_dim == 64) {                                                             \
    if (dtype == kF32) return FN<F32, 64>(__VA_ARGS__);                             \
    if (dtype == kF16) return FN<F16, 64>(__VA_ARGS__);                             \
    return FN<BF16, 64>(__VA_ARGS__);                                               \
  }                                                                                 \
  if (dtype == kF32) return FN<F32, 128>(__VA_ARGS__);                              \
  if (dtype == kF16) return FN<F16, 128>(__VA_ARGS__);                              \
  return FN<BF16, 128>(__VA_ARGS__);

namespace {
StreamArgs stream_args(const Geom& g, const void* q, const void* k, const void* v, const uint8_t* ks,
                       const uint8_t* vs, void* o, float* lse, int kv_rows, float* ws, int n_splits, int head_dim) {
  StreamArgs a{};
  a.q = q, a.k = k, a.v = v, a.ks = ks, a.vs = vs, a.o = o, a.lse = lse;
  a.H_kv = g.H_kv;
  a.rb = a.n_rows = g.group * g.n_q;
  a.n_q = g.n_q;
  a.q_stride = g.H * g.n_q;
  a.kv_rows = kv_rows;
  a.n_splits = a.n_parts = n_splits;
  a.acc = ws;
  a.ml = ws + (size_t)g.B * g.H * g.n_q * n_splits * head_dim;
  a.scale_log2 = g.qk_scale_log2;
  a.q_sign = g.scale == 0.f ? 0.f : g.scale < 0.f ? -1.f : 1.f;
  a.start = 1 << kPartialBit;
  return a;
}

AppendArgs append_args(void* kc, void* vc, uint8_t* ks, uint8_t* vs, const void* kn, const void* vn, int BH, int n_new,
                       int start, int sink, int ring) {
  AppendArgs a{kc, vc, ks, vs, kn, vn, BH, AppendRows{n_new, 0, 0, 0, start, sink, ring}, 0};
  surviving_rows(start, n_new, sink, ring, &a.rows.n_a, &a.rows.i_b, &a.rows.n_b);
  return a;
}

// A step: its n_q tokens (k_new, v_new) are written by the launch that attends them.
void set_step(const Geom& g, StreamArgs& a, AppendArgs& ap, const void* k_new, const void* v_new, int ring, int head_dim) {
  if (!k_new) return;
  a.k_new = k_new;
  a.v_new = v_new;
  a.n_new = g.n_q;
  a.start = g.q_off;
  ap = append_args((void*)a.k, (void*)a.v, (uint8_t*)a.ks, (uint8_t*)a.vs, k_new, v_new, g.B * g.H_kv, g.n_q, g.q_off,
                   g.sink, ring);
  ap.n_blocks = append_blocks(ap, head_dim);
}
RingStream ring_args(const Geom& g, int ring) {
  RingStream src;
  ring_stream(g.n_kv, g.n_q, g.sink, g.window, ring, &src.n_sink, &src.w_lo, &src.base, &src.n_tokens);
  src.sink = g.sink;
  src.ring = ring;
  src.q_off = g.q_off;
  src.window = g.window;
  return src;
}
}  // namespace

int append8_dispatch(int dtype, int head_dim, uint8_t* kc, uint8_t* vc, uint8_t* ks, uint8_t* vs, const void* kn,
                     const void* vn, int BH, int n_new, int start, int sink, int ring, hipStream_t stream) {
  const AppendArgs a = append_args(kc, vc, ks, vs, kn, vn, BH, n_new, start, sink, ring);
  GKI_BY_TYPE(append8, a, stream)
}

int read_dispatch(int dtype, int head_dim, const void* kc, const void* vc, const uint8_t* ks, const uint8_t* vs,
                  void* ko, void* vo, int64_t* positions, int BH, int length, int sink, int ring,
                  hipStream_t stream) {
  HeldRows a{};
  a.n_sink = length < sink ? length : sink;
  a.lo = length - ring > sink ? length - ring : sink;
  a.n = a.n_sink + (length > a.lo ? length - a.lo : 0);
  a.sink = sink;
  a.ring = ring;
  if (a.n == 0) return 0;
  GKI_BY_TYPE(held_rows, kc, vc, ks, vs, ko, vo, positions, BH, a, stream)
}

int attend8_dispatch(int dtype, int head_dim, const Geom& g, const void* q, const void* k, const void* v,
                     const uint8_t* ks, const uint8_t* vs, const void* k_new, const void* v_new, void* o, float* lse,
                     int ring, float* ws, int n_splits, hipStream_t stream) {
  const RingStream src = ring_args(g, ring);
  StreamArgs a = stream_args(g, q, k, v, ks, vs, o, lse, g.sink + ring, ws, n_splits, head_dim);
  AppendArgs ap{};
  set_step(g, a, ap, k_new, v_new, ring, head_dim);
  GKI_BY_TYPE(attend8, a, src, g.B * g.H_kv, ap, stream)
}

int cross_stream_dispatch(int dtype, int head_dim, const Geom& g, const void* q, const void* k, const void* v, void* o,
                          float* lse, float* ws, int n_splits, hipStream_t stream) {
  const DenseStream src{g.kv_len, g.n_kv, g.H_kv};
  const StreamArgs a = stream_args(g, q, k, v, nullptr, nullptr, o, lse, g.n_kv, ws, n_splits, head_dim);
  const int n = g.B * g.H_kv;
#define GKI_CROSS_STREAM(DD) \
  return dtype == kF16 ? cross_stream<F16, DD>(a, src, n, stream) : cross_stream<BF16, DD>(a, src, n, stream)
  if (head_dim == 32) GKI_CROSS_STREAM(32);
  if (head_dim == 64) GKI_CROSS_STREAM(64);
  GKI_CROSS_STREAM(128);
#undef GKI_CROSS_STREAM
}

int prefix_decode_dispatch(int dtype, int head_dim, const Geom& g, const void* q, const void* k, const void* v,
                           const uint8_t* ks, const uint8_t* vs, const void* k_new, const void* v_new,
                           const void* prefix_k, const void* prefix_v, int n_prefix, void* o, float* lse, int ring,
                           float* ws, int n_prefix_splits, int n_splits, hipStream_t stream) {
  const int n_parts = n_prefix_splits + n_splits;
  StreamArgs own = stream_args(g, q, k, v, ks, vs, o, lse, g.sink + ring, ws, n_parts, head_dim);
  own.n_splits = n_splits;
  own.part0 = n_prefix_splits;
  AppendArgs ap{};
  set_step(g, own, ap, k_new, v_new, ring, head_dim);
  StreamArgs shared = stream_args(g, q, prefix_k, prefix_v, nullptr, nullptr, o, lse, n_prefix, ws, n_parts, head_dim);
  shared.n_splits = n_prefix_splits;
  shared.n_rows = g.B * shared.rb;
  const RingStream src = ring_args(g, ring);
  if (dtype == kF16)
    return head_dim == 64 ? prefix_decode<F16, 64>(g, own, src, ap, shared, n_prefix, stream)
                          : prefix_decode<F16, 128>(g, own, src, ap, shared, n_prefix, stream);
  return head_dim == 64 ? prefix_decode<BF16, 64>(g, own, src, ap, shared, n_prefix, stream)
                        : prefix_decode<BF16, 128>(g, own, src, ap, shared, n_prefix, stream);
}

}  // namespace gki

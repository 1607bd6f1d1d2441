// A wave's part in attention of few query rows over a stream of keys and values: the
// streams of rolling caches, cross attention and paged caches.
#pragma once

#include "gki_common.cuh"

namespace gki {
namespace {

constexpr float kStreamSlack = 8.f;          // log2 units the lazy reference max may lag (p <= 2^8)

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

__device__ inline float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

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
// Row: what the token rule wants to know of a row (RULE). ROUNDED: the row sums add the
// probabilities as they are rounded for P V (16-bit rows), so that a part of their errors cancels.
template <typename T, typename C, int D, int NB, int NPC, bool RULE, bool EIGHT, typename Row = int, bool ROUNDED = false>
struct StreamWave {
  static constexpr int KS = D / 32, DT = D / 16;
  uint4 qf[NB][KS][NPC];
  floatx4 o[NB][DT];
  float lsum[NB], m[NB];
  Row my_q[NB];
  int wave, lane, grp, col;

  // Rows row0 .. n_rows - 1 of a stream: row_of(r) is where row r's elements are, rule_of(r) its Row.
  template <class Rows, class Rules>
  __device__ inline StreamWave(int row0, int n_rows, float q_sign, Rows row_of, Rules rule_of, int tid = threadIdx.x) {
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    grp = lane >> 4, col = lane & 15;
    // Q^T operand of column block h: lane (grp, col) holds elements 32 ks + 8 grp .. +7
    // (EIGHT: 64 (ks / 2) + 16 grp + 8 (ks % 2) .. +7) of row row0 + 16 h + col
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      const int r = row0 + 16 * h + col;
      my_q[h] = rule_of(r);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float f[8];
        load8<T>(row_of(r < n_rows ? r : 0) + (EIGHT ? 64 * (ks >> 1) + 16 * grp + 8 * (ks & 1) : 32 * ks + 8 * grp), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = r < n_rows && q_sign != 0.f ? f[i] * q_sign : 0.f;
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
  template <class Args, class Src>
  __device__ inline void step(const Args& a, const Src& src, const uint16_t* ck, const uint16_t* cv, int t, int g1) {
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
      pb[h] = make_uint2(pack2<C>(s[h][0], s[h][1]), pack2<C>(s[h][2], s[h][3]));
      if constexpr (ROUNDED) {
        const uint16_t* r = (const uint16_t*)&pb[h];
        lsum[h] += (C::to_float(r[0]) + C::to_float(r[1])) + (C::to_float(r[2]) + C::to_float(r[3]));
      } else {
        lsum[h] += (s[h][0] + s[h][1]) + (s[h][2] + s[h][3]);
      }
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
  template <class Args, class Src>
  __device__ inline void step8(const Args& a, const Src& src, const uint8_t* ck, const uint8_t* cv,
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
  // write(r, d, x, M, L): elements d .. d + 3 of the r-th row's sum, its largest score, its row
  // sum; n_rows: the rows from row0 on.
  template <class Write>
  __device__ inline void finish(int n_rows, float* wacc, float* wml, Write write, int tid = threadIdx.x) {
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
      const int rows_h = min(16, n_rows - 16 * h);
      for (int idx = tid; idx < rows_h * (D / 4); idx += 256) {
        const int rl = idx / (D / 4), d = 4 * (idx % (D / 4));
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
        write(16 * h + rl, d, x, M, L);
      }
    }
  }
};

}  // namespace
}  // namespace gki

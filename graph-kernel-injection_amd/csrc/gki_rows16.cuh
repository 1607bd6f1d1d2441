// The 16-bit forward's row tile: 128 query rows of one head against the kv tiles of a
// list (block-sparse prefill), of a batch entry's own keys (cross attention) or of a
// slice of a prefix that the rows share (decode behind a shared prefix).
#pragma once

#include "gki_common.cuh"

namespace gki {
namespace {

struct Alone {};      // nothing beside the row tiles

// Online-softmax reference max moves only when a tile's row max exceeds it by
// more than this many log2 units, so p = exp2(s - m) stays below 2^8 and the O
// rescale is almost never needed. O = acc / l and LSE = m + ln(l) are exact for
// any reference max.
constexpr float kRescaleSlack = 8.f;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Issue order of the skewed (PIPE) loop, imposed with sched_group_barrier
// (masks: 0x008 MFMA, 0x100 LDS read, 0x002 VALU). S_{j+1}: kPipeAheadS K
// reads first, then per MFMA one more read and kPipeValuS VALU ops of the exp
// work. O += V P: kPipeAheadO V^T reads first, then two reads and kPipeValuO
// VALU ops (the maxima of S_{j+1}) per MFMA. On a B1 H32 N16384 W2048 bf16
// forward: 3 VALU ops 0.542 ms, 5 or 6 0.552-0.557, reads 2 / 4 ahead 0.546,
// 8 / 12 0.557, no imposed order 0.560.
constexpr int kPipeAheadS = 4, kPipeAheadO = 8, kPipeValuS = 3, kPipeValuO = 1;
constexpr int kFwdThreads = 256;
// Waves per SIMD the compiler must fit in registers (HIP's second launch
// bound): 4 (up to 128 VGPRs) for head_dim <= 64, whose 32 KB of K / V buffers
// allow four workgroups per CU; 2 for head_dim 128 (64 KB of buffers, two
// workgroups per CU).
//
// PIPE selects the tile schedule. Without it every kv tile runs S = K Q^T,
// then mask / max / exp, then O += V P in turn, and the matrix cores idle
// through the softmax unless another wave of the SIMD has MFMAs to issue. With
// it the loop is skewed by one tile: iteration j runs S_{j+1} = K_{j+1} Q^T
// while it exponentiates S_j (MFMA and VALU of one wave in one straight-line
// block, interleaved in the order kPipe* describes), then O += V_j P_j while
// it takes the row maxima of S_{j+1}. K is therefore read one tile ahead of V:
// at iteration j the LDS holds K_{j+1} and V_j while K_{j+2} and V_{j+1} land
// in the other halves of the two double buffers (the same 2 x 2 tiles of LDS).
// Either loop is unrolled by two: the buffers are then constants of the LDS
// instructions, and the two score tiles of PIPE swap roles without copies.
// P_j is pinned (an empty asm that takes it) inside the S_{j+1} block:
// otherwise the compiler sinks the exp work past the mask branch into the
// O += V P block and no MFMA of S_{j+1} overlaps it.
//
// Against four waves of 16x16x32 MFMAs on the same tiles (ms, same card, three
// interleaved rounds): B1 H32 N16384 D128 W2048 bf16 0.530 -> 0.523, B4 H16
// N8192 D64 W1024 fp16 0.174 -> 0.168, B1 H16 N131072 D64 W4096 bf16 2.20 ->
// 2.16, 500 queries behind 8500 keys D128 0.0525 -> 0.0467, B4 H8 N2000 D32
// 0.0177 -> 0.0150.
// SHARED (a prefix that the rows of a batch share): a slice of the keys for 128 rows
// (SharedRows), and the workgroups of `beside` in the same launch.
template <typename T, int D, bool PIPE, int WALK, class Beside>
__global__ __launch_bounds__(kFwdThreads, D <= 64 && WALK != kShared ? 4 : 2) void fwd_kernel_16(
    Geom g, const uint16_t* __restrict__ Q, const uint16_t* __restrict__ K,
    const uint16_t* __restrict__ V, uint16_t* __restrict__ O, float* __restrict__ LSE,
    const int32_t* __restrict__ row_ptr, const int32_t* __restrict__ row_idx, int n_qt,
    const int32_t* __restrict__ wg_order, SharedRows sh, Beside beside) {
  constexpr bool DENSE = WALK != kListed, SHARED = WALK == kShared;
  constexpr int KS = D / 16;                   // k-steps of the QK^T contraction
  constexpr int DT = D >= 32 ? D / 32 : 1;     // 32-row tiles of O^T
  constexpr int NW = 4;
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];

  int block = blockIdx.x, n_wg = n_qt * g.B * g.H;
  if constexpr (SHARED) {
    if (beside.takes(block)) {
      beside.run(block, &sk[0][0], &sv[0][0]);
      return;
    }
    n_wg = n_qt * sh.n_splits * g.H_kv;
    if (block >= n_wg) return;
  }
  const int wg = work_of(block, n_wg, wg_order, entries_of<WALK == kDense>(g));
  if (wg < 0) return;
  // SHARED: the row tiles of a slice are neighbours, its head is bh / n_splits
  const int bh = wg / n_qt, qt = wg - bh * n_qt;
  const size_t qb = (size_t)bh * g.n_q * D;
  const size_t kb = (size_t)(SHARED ? bh / sh.n_splits : kv_bh(g, bh)) * g.n_kv * D;
  if constexpr (WALK == kDense) g.n_kv = own_keys(g, bh / g.H);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, hi = lane >> 5, col = lane & 31;
  const Lane32<D> at(lane);
  const int qw = qt * kTileMF + wave * 32;     // first row of this wave

  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    if constexpr (SHARED) {
      const int r = min(qw + col, g.n_q - 1), d = 16 * ks + 8 * hi;
      qf[ks] = q_words(g, *(const uint4*)(Q + sh.row(bh / sh.n_splits, r) * D + d));
    } else {
      const uint4 v = q_words(g, row16_or_zero<D>(Q + qb, qw + col, g.n_q, 16 * ks + 8 * hi));
      qf[ks] = qw + col < g.n_q ? v : make_uint4(0, 0, 0, 0);
    }
  }

  floatx16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = splat16(0.f);
  // Row sums on the MFMA pipe: 16x16x32 reads the P operand of a 32x32x16 as
  // (lane groups 0 and 2: rows 0-15, groups 1 and 3: rows 16-31), so a selector
  // of ones that pairs result row group g with the operand groups of g's parity
  // leaves lane l the sum of row l & 31 (over the same 16-bit P that
  // multiplies V) in every component.
  floatx4 lsum = floatx4{0.f, 0.f, 0.f, 0.f};
  const uint4 ones = ((lane >> 2) & 1) == ((lane >> 4) & 1) ? T::ones8() : make_uint4(0, 0, 0, 0);
  // nm: minus the row's reference max (scaled, log2 units), so P = exp2(S c + nm); thr: the unscaled score
  // above which it must move, (max + slack) / c, -inf until the row has seen a visible key.
  const float slack = kRescaleSlack * __builtin_amdgcn_rcpf(g.qk_scale_log2);   // a trigger: approximate is fine
  float nm = 0.f, thr = kNegInf;

  DmaTile<D, NW, true> dma;
  dma.init(tid);
  auto stage = [&](const uint16_t* src, int k0, uint16_t* dst) { dma.load(src + kb, k0, g.n_kv, dst); };
  auto tile_k0 = [&](int ent) { return (ent & kIdxMask) * kTileN; };

  // S^T of one kv tile: the 32 query rows of the wave against its 64 keys.
  auto scores = [&](const uint16_t* ck, floatx16 (&s)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[t] = T::mfma32(at.rows(ck, t, ks), qf[ks], ks == 0 ? splat16(0.f) : s[t]);
    }
  };
  // Token mask of a tile (only where some element of it can be hidden).
  auto apply_mask = [&](int ent, floatx16 (&s)[2]) {
    const int k0 = tile_k0(ent);
    const bool partial = (ent >> kPartialBit) & 1;
    const bool need_mask = partial || (qw + 31 >= g.n_q) || (k0 + kTileN > g.n_kv) ||
                           !tile_all_visible(g, qw, min(qw + 31, g.n_q - 1), k0, k0 + kTileN - 1);
    if (need_mask) {
      const uint64_t bits = row_valid_bits(g, qw + col, k0, partial);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const LaneBits32 vis((uint32_t)(bits >> (32 * t)), hi);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = vis.pick(r, s[t][r], kNegInf);
      }
    }
  };
  auto lane_max = [&](const floatx16 (&s)[2]) {
    float mx = kNegInf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
    return mx;
  };
  // The reference moves (to the row's max) only when some score exceeds it by
  // the slack: p stays below 2^8 and the rescale of O and the row sums almost
  // never runs. Each lane tests its own half of the row; the cross-lane max
  // runs only then. Runs after every product of the tiles before.
  auto move_max = [&](float mx) {
    if (__any(mx > thr)) {
      const float mr = half_max(mx);
      const bool grow = mr > thr;
      const float nm1 = grow ? -mr * g.qk_scale_log2 : nm;
      // a first reference below zero scales nothing yet (o = lsum = 0)
      const float alpha = __builtin_amdgcn_exp2f(fminf(nm1 - nm, 0.f));
      nm = nm1;
      thr = grow ? mr + slack : thr;
      lsum[0] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
  };
  // P = exp2(S c + nm) packed to 16-bit MFMA operands (16 keys each).
  auto probs = [&](floatx16 (&s)[2], uint4 (&p)[4]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], g.qk_scale_log2, nm));
      p[2 * t] = pack8<T>(s[t], 0);
      p[2 * t + 1] = pack8<T>(s[t], 1);
    }
  };
  // O^T += V^T P^T and the row sums.
  auto accumulate = [&](const uint16_t* cv, const uint4 (&p)[4]) {
#pragma unroll
    for (int st = 0; st < 4; ++st) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma32(at.cols(cv, st, dt), p[st], o[dt]);
      lsum = T::mfma(ones, p[st], lsum);
    }
  };
  const int n_kt = kv_tiles_of(g), slice = SHARED ? bh % sh.n_splits : 0;
  const int e_beg = SHARED ? (int)((int64_t)n_kt * slice / sh.n_splits) : DENSE ? 0 : row_ptr[qt];
  const int e_end = SHARED ? (int)((int64_t)n_kt * (slice + 1) / sh.n_splits) : DENSE ? n_kt : row_ptr[qt + 1];
  auto entry = [&](int e) { return walk_entry<DENSE>(row_idx, e); };
  if constexpr (!PIPE) {
    if (e_beg < e_end) {
      stage(K, tile_k0(entry(e_beg)), sk[0]);
      stage(V, tile_k0(entry(e_beg)), sv[0]);
    }
    dma_wait();
    __syncthreads();

    // unrolled by two so that the buffers are constants of the instructions
    auto step = [&](int e, int buf) {
      const int ent = entry(e);
      if (e + 1 < e_end) {
        const int k1 = tile_k0(entry(e + 1));
        stage(K, k1, sk[buf ^ 1]);
        stage(V, k1, sv[buf ^ 1]);
      }
      // Left out where no row of this wave sees a key of the tile (a listed tile
      // is one that some of the workgroup's 128 rows sees): 2.5% of a forward
      // over 18-tile rows, 0.7% over 67 (head_dim 64).
      if (!tile_unseen(g, qw, qw + 31, tile_k0(ent), kTileN)) {
        floatx16 s[2];
        uint4 p[4];
        mfma_priority_hi<true>();
        scores(sk[buf], s);
        mfma_priority_lo<true>();
        apply_mask(ent, s);
        move_max(lane_max(s));
        probs(s, p);
        mfma_priority_hi<true>();
        accumulate(sv[buf], p);
        mfma_priority_lo<true>();
      }
      dma_wait();        // the next tile's LDS-DMA has landed before the barrier
      __syncthreads();
    };
    int e = e_beg;
    for (; e + 1 < e_end; e += 2) {
      step(e, 0);
      step(e + 1, 1);
    }
    if (e < e_end) step(e, 0);
  } else {
    const int n = e_end - e_beg;
    floatx16 sa[2], sb[2];
    // Prologue: K_0, V_0 and K_1 in LDS, S_0 with its maxima.
    if (n > 0) {
      const int k0 = tile_k0(entry(e_beg));
      stage(K, k0, sk[0]);
      stage(V, k0, sv[0]);
      if (n > 1) stage(K, tile_k0(entry(e_beg + 1)), sk[1]);
    }
    dma_wait();
    __syncthreads();
    if (n > 0) {
      scores(sk[0], sa);
      apply_mask(entry(e_beg), sa);
      move_max(lane_max(sa));
    }
    __syncthreads();   // every wave is done with K_0 before iteration 0 refills its buffer

    // Iteration j (j + 1 < n): S_{j+1} from K_{j+1} into sn while s = S_j
    // becomes P_j; O += V_j P_j while sn's maxima are taken.
    auto step = [&](int j, int par, floatx16 (&s)[2], floatx16 (&sn)[2]) {   // par = j & 1
      const int e = e_beg + j;
      const int ent1 = entry(e + 1);
      // LDS: K_{j+1} in sk[(j+1)&1], V_j in sv[j&1]; refill the other halves
      if (j + 2 < n) stage(K, tile_k0(entry(e + 2)), sk[par]);
      stage(V, tile_k0(ent1), sv[par ^ 1]);

      uint4 p[4];
      scores(sk[par ^ 1], sn);   // MFMA ...
      probs(s, p);                   // ... under VALU
      // P is formed here, not sunk past the mask branch into the next block
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        u32x4 w = __builtin_bit_cast(u32x4, p[st]);
        asm volatile("" : "+v"(w));
        p[st] = __builtin_bit_cast(uint4, w);
      }
      // issue order: the 2 KS MFMAs of S_{j+1} between the exp work
      __builtin_amdgcn_sched_group_barrier(0x100, kPipeAheadS, 0);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + kPipeAheadS < 2 * KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, kPipeValuS, 0);
      }
      apply_mask(ent1, sn);
      accumulate(sv[par], p);           // MFMA ...
      const float mx = lane_max(sn);      // ... under VALU
      // issue order: the 4 DT MFMAs of O += V P (two V^T reads each) with the
      // maxima of S_{j+1} between them
      __builtin_amdgcn_sched_group_barrier(0x100, kPipeAheadO, 1);
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        if (2 * i + kPipeAheadO < 8 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        __builtin_amdgcn_sched_group_barrier(0x002, kPipeValuO, 1);
      }
      move_max(mx);
      dma_wait();
      __syncthreads();
    };
    auto last = [&](floatx16 (&s)[2], int par) {
      uint4 p[4];
      probs(s, p);
      accumulate(sv[par], p);
    };
    // Unrolled by two so that the score buffers swap roles without copies.
    int j = 0;
    for (; j + 2 < n; j += 2) {
      step(j, 0, sa, sb);
      step(j + 1, 1, sb, sa);
    }
    if (j + 1 < n) {
      step(j, 0, sa, sb);
      last(sb, 1);
    } else if (n > 0) {
      last(sa, 0);
    }
  }

  // The epilogue's row offsets from the lane index afresh (mbcnt: not provably
  // the one above), not the prologue's Q offsets held across the loop.
  const int lane_e = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const int hi_e = lane_e >> 5;
  const int my_q = qw + (lane_e & 31);
  const float l_tot = lsum[0];
  if constexpr (SHARED) {
    if (my_q >= g.n_q) return;
    const size_t at = sh.row(bh / sh.n_splits, my_q) * sh.n_parts + sh.part0 + slice;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(floatx4*)(sh.acc + at * D + 32 * dt + 8 * r + 4 * hi_e) =
            floatx4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
    if (hi_e == 0) *(float2*)(sh.ml + at * 2) = make_float2(l_tot == 0.f ? kNegInf : -nm, l_tot);
    return;
  }
  const bool valid = l_tot > 0.f;
  const float inv = valid ? 1.f / l_tot : 1.f;
  if (my_q < g.n_q) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < (D >= 32 ? 4 : 2); ++r) {     // D = 16: rows past 15 do not exist
        uint2 w;
        w.x = pack2<T>(o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv);
        w.y = pack2<T>(o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv);
        *(uint2*)(O + qb + (size_t)my_q * D + 32 * dt + 8 * r + 4 * hi_e) = w;
      }
    if (hi_e == 0) LSE[(size_t)bh * g.n_q + my_q] = valid ? lse_natural(-nm, l_tot) : 0.f;
  }
}

// The skewed schedule holds two score tiles (32 more VGPRs): head_dim 128
// has them within its 256 (without it 2% slower); at head_dim 64 it would cost
// the fourth workgroup per CU.
template <int D>
constexpr bool kFwdPipe = D >= 128;

}  // namespace
}  // namespace gki

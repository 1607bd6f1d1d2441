// What the paged cache's entry points and kernels share.
#pragma once

#include "gki_common.cuh"

namespace gki {

// Sum of lanes 0 .. l, by DPP.
template <int CTRL, int ROWS>
__device__ inline uint32_t dpp_or_zero(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}
__device__ inline uint32_t wave_prefix(uint32_t x) {
  x += dpp_or_zero<0x111, 0xF>(x);     // row_shr 1, 2, 4, 8
  x += dpp_or_zero<0x112, 0xF>(x);
  x += dpp_or_zero<0x114, 0xF>(x);
  x += dpp_or_zero<0x118, 0xF>(x);
  x += dpp_or_zero<0x142, 0xA>(x);     // lane 15 of a row to the next, for rows 1 and 3
  x += dpp_or_zero<0x143, 0xC>(x);     // lane 31 to rows 2 and 3
  return x;
}

// Rotary positions with several axes: pair j of a row's P pairs of elements turns by
//   angle = position[axis_j] * frequency_j,  (a, b) -> (a cos - b sin, a sin + b cos),
// pairs (j, j + P) or, interleaved, (2 j, 2 j + 1); elements from 2 P on stay as they are.
struct RotaryArgs {
  const double* turns;         // [P] frequency / (2 pi): turns per position
  const int32_t* axis;         // [P]
  const void* positions;       // int32 or int64, axis a of token (b, i) at a * pa + b * pb + i * pn
  int64_t pa, pb, pn;
  int wide;                    // positions are int64
  int pairs, interleaved;
  float sign;                  // -1: the gradient's turn
  int64_t tokens;              // B * n
  int n;
};

// Rows of heads, D elements each: token (b, i), head h at b * sb + i * sn + h * sh of the
// source, with the d strides of the destination.
struct HeadRows {
  const void* src;
  void* dst;
  int heads;
  int64_t sb, sn, sh, db, dn, dh;
};

// Tables of requests: position p of request r lies in page table[r][p >> shift].
struct PageTables {
  int32_t *lengths, *pages, *kept;     // [R] positions held, pages taken so far, first page behind the sinks not given back
  int32_t *table;                      // [R][max_pages], -1: none
  int32_t *ring, *queue;               // free pages: [num_pages]; {head, count}
  int32_t* status;
  int R, max_pages, shift, num_pages, sink, window;
};

// A step's tokens: counts[r] of each request, one request's rows after the other's.
struct PageStep {
  const int32_t *counts, *parents;
  int rows, max_count, words;
  int32_t *row_starts, *base, *positions;
  int64_t* slots;
  uint64_t* ancestors;
  int4* requests;                      // [R + 1] {requests with tokens, rows}, then of each {request, first row, rows, base}
};

// Rows of keys and values and the pool that they go to: [num_pages][H_kv][page_size][D].
struct PageRows {
  const void *k, *v;
  int64_t k_stride, v_stride;          // elements between rows; heads lie D apart
  void *k_pages, *v_pages;
  const int64_t* slots;
  int64_t n_slots;                     // of the pool
  int rows, H_kv, shift;
  // element of the pool where head h of a row at `slot` starts
  __device__ inline size_t at(int64_t slot, int h, int D) const {
    return ((((size_t)(slot >> shift) * H_kv + h) << shift) + (slot & ((1 << shift) - 1))) * D;
  }
};

// How attention over pages is shared out; us with the join at bf16 D128, H32/8 (H64/8: trees of 60),
// and fp16 D64 H16 ("mixed").
//
// Workgroups that take shares: as many as the card holds at once. 256 / 512 / 768 / 1024 at
// D128: 32 decodes over up to 4096 keys 52 / 44 / 49 / 48, chunks of 512 129 / 108 / 124 / 119, trees of 60
// 145 / 121 / 137 / 133; 512 / 768 / 1024 / 1536 at D64: mixed 54 / 51 / 50 / 55.
inline int paged_groups(int head_dim) { return head_dim >= 128 ? 512 : 1024; }
// What a walk's prologue and epilogue count, in 64-key steps: 0 / 2 / 4 / 6: decodes 52.9 / 43.9 / 45.1 /
// 45.1, chunks 111 / 108 / 110 / 109, mixed 53.3 / 49.8 / 51.6 / 50.7, trees of 60 120 / 121 / 122 / 123.
constexpr int kPagedPieceCost = 2;
// Steps that a share has at least: a walk as long as the longest gets about kPagedPieces pieces,
// whose join costs as much as they save from there on. One decode over 768 / 4096 / 16384 keys:
// 2 steps at least 13.1 / 20.5 / 29.5, 4 15.3 / 17.7 / 29.5, 8 18.8 / 20.1 / 28.1, 16 26.1 / 25.9 /
// 28.5; this rule 13.2 / 17.7 / 28.0.
constexpr int kPagedMinShare = 2, kPagedMostShare = 8, kPagedPieces = 16;
// Walks shorter than this are not cut: the join is another launch, and below there is little to win
// (one decode of 8 heads, replayed: 9 key tiles cut 10.1, whole 10.6 to 10.9; 13 tiles cut 13.2, whole 17.4).
constexpr int kPagedCutSteps = 16;

struct PagedArgs {
  const uint16_t *q, *k_pages, *v_pages;
  uint16_t* o;
  float* lse;                          // [rows][H] or null
  const int4* requests;                // PageStep's
  const int32_t *positions, *table;
  const uint64_t* ancestors;           // [rows][words], null: no trees
  int64_t q_stride;                    // elements between rows of q; heads lie D apart
  int rows, H, H_kv, group, max_pages, shift, num_pages, sink, window, words;
  float scale_log2, q_sign;            // as StreamArgs': the sign of the scale, or zero, goes to q
  uint32_t q_and, q_xor;               // the same as words of Q
  int groups;                          // workgroups that share the work
  int least;                           // steps that a share has at least
  int coarse;                          // a step of the work is 2^coarse key tiles, so that 31 bits count them all
  // the states of row tiles that the shares' ends cut, of `cap` rows each; acc null: none is cut
  int cap;
  float *acc, *ml;
  struct CutTile* cuts;                // [groups]
};

// A row tile that ends a workgroup's share unfinished: its request's rows, its pieces (0: none).
struct CutTile {
  int first, n, h, tile, pieces;
};

// Rows of a piece's state, and the floats of all states and cuts (0 where no row tile's walk, by what
// the host knows, is long enough to be cut). States are in 32 bits.
inline int paged_cap(int64_t max_count, int group) { return (int)std::min<int64_t>(128, max_count * group); }
inline int64_t paged_workspace(int groups, int head_dim, int64_t max_count, int group, int64_t sink, int64_t window,
                               int64_t max_length) {
  const int64_t seen = std::min(max_length, sink + window + max_count + 64);
  if ((seen + 63) / 64 + 2 < kPagedCutSteps) return 0;
  return (int64_t)groups * (2 * paged_cap(max_count, group) * (head_dim + 2) + 5);
}

}  // namespace gki

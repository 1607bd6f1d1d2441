// Attention of requests of different lengths over paged keys and values, with sinks and a
// sliding window (the StreamingLLM rule), for gfx950.
//
// Request r has `base` keys and brings n rows, which stand behind them at places base + i.
// A row at position p sees the keys x <= p with x < S or x > p - W:
//   S_x = scale * q . k_x,  O = sum_x exp(S_x - m) v_x / sum_x exp(S_x - m),  LSE = m + ln(sum).
// Drafted trees: row i stands at p = base + depth_i; of the keys from base on it sees those
// that its word of ancestors names (which has the rule in it already).
//
// The rows of a request that read one kv head, (token, q head of the group) token by token,
// are its rows here. Up to 32 of them run as a stream (four waves share out the keys of a
// step), more as tiles of 128 (four waves of 32 rows). Either walks the 64-key tiles of the
// sinks and of its rows' windows once, whatever lies between, or a slice of them; slices'
// states are joined. Pages are addressed a 1 KB LDS block at a time, each of which lies in
// one page; keys past the request's last, and pages that it does not have, are zeros
// without being read: what another request left in a page is never seen. (A NaN or
// infinity among the request's own values reaches every row of a tile that reads it.)
#include "gki_paged.cuh"
#include "gki_stream_wave.cuh"

namespace gki {
namespace {

constexpr int kRowTile = 128;          // rows of a tile: four waves of 32
constexpr int kFewRows = 32;           // up to as many run as a stream
constexpr int kIds = 1024;             // page ids held in LDS at a time

// The 64-key tiles that rows at positions lo_pos .. see of keys 0 .. end - 1: the sinks',
// then the window's.
struct KeyTiles {
  int n_sink, w0, n;
  __device__ inline KeyTiles(const PagedArgs& a, int lo_pos, int end) {
    const int lo = max(0, lo_pos - a.window + 1);
    n_sink = (min(a.sink, end) + 63) >> 6;
    w0 = max(lo >> 6, n_sink);
    n = n_sink + (lo < end ? max(0, ((end + 63) >> 6) - w0) : 0);
  }
  __device__ inline int first_key(int i) const { return (i < n_sink ? i : w0 + (i - n_sink)) << 6; }
};

// ---------------------------------------------------------------------------
// Which unit of work a workgroup takes. A unit is a slice of the keys of a row tile of one
// request and kv head. Lengths are known on the device only, so every workgroup counts
// for itself, a wave 64 requests at a time: the key tiles of all row tiles, from them the
// length of a slice that fills the card, from it the units. The units of a (request, head)
// are neighbours on one XCD, a slice's row tiles side by side.
// ---------------------------------------------------------------------------
struct Request {
  int first, n, base, tiles, keys;     // first row of the step's, rows, keys before them; row tiles, key tiles
  __device__ inline Request(const PagedArgs& a, int r) {
    const bool ok = r < a.R;
    r = ok ? r : a.R - 1;
    first = a.row_starts[r];
    n = ok ? a.row_starts[r + 1] - first : 0;
    base = a.base[r];
    const int rows = n * a.group;
    tiles = rows <= kFewRows ? (rows + kFewRows - 1) / kFewRows : (rows + kRowTile - 1) / kRowTile;
    keys = n ? KeyTiles(a, base, base + n).n : 0;
  }
  // Slices of about `length` key tiles.
  __device__ inline int slices(const PagedArgs& a, int length) const {
    return keys < a.whole ? 1 : min(a.max_slices, (keys + length - 1) / length);
  }
};

__device__ inline int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);       // the same everywhere: scalar
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | lo);
}
// Sum of lanes 0 .. l.
__device__ inline int wave_prefix(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}
__device__ inline int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

struct Unit {
  int r, first, n, base;               // the request
  int h, tile, slice, n_slices;
};

__device__ inline bool find_unit(const PagedArgs& a, int block, Unit& u) {
  const int lane = threadIdx.x & 63;
  int64_t all = 0;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const Request q(a, r0 + lane);
    all += (int64_t)q.tiles * q.keys;
  }
  all = wave_sum64(all) * a.H_kv;
  const int length = (int)max((int64_t)a.min_slice, (all + a.target - 1) / a.target);
  int units = 0;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const Request q(a, r0 + lane);
    units += q.tiles * q.slices(a, length);
  }
  units = (int)wave_sum64(units) * a.H_kv;
  if (block >= units) return false;
  int t = xcd_remap(block, units);
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const Request q(a, r0 + lane);
    const int mine = q.tiles * q.slices(a, length) * a.H_kv, sum = wave_prefix(mine);
    const uint64_t past = __ballot(sum > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      u.r = r0 + l;
      u.first = lane_value(q.first, l), u.n = lane_value(q.n, l), u.base = lane_value(q.base, l);
      u.n_slices = lane_value(q.slices(a, length), l);
      const int tiles = lane_value(q.tiles, l);
      t -= lane_value(sum - mine, l);
      u.tile = t % tiles;
      t /= tiles;
      u.slice = t % u.n_slices;
      u.h = t / u.n_slices;
      return true;
    }
    t -= lane_value(sum, 63);
  }
  return false;
}

// Keys of the 64 from x0 on that the i-th of a request's tokens sees.
__device__ inline uint64_t seen_bits(const PagedArgs& a, const Unit& u, uint32_t i, int x0) {
  const bool tree = a.ancestors != nullptr;
  const int pos = tree ? (a.positions + u.first)[i] : u.base + (int)i;
  const uint64_t rule = bit_range(pos - a.window + 1 - x0, 63) | bit_range(0, a.sink - 1 - x0);
  uint64_t bits = bit_range(0, (tree ? u.base - 1 : pos) - x0) & rule;
  const int from = x0 - u.base;        // number of the node at x0
  if (tree && from > -64) {
    const uint64_t* word = a.ancestors + (int64_t)u.first * a.words;
    const int w = from >> 6, sh = from & 63;                 // from < 0: w = -1
    if (w >= 0 && w < a.words) bits |= word[i * a.words + w] >> sh;
    if (sh && w + 1 < a.words) bits |= word[i * a.words + w + 1] << (64 - sh);
  }
  return bits;
}

// The key tiles of a unit, into LDS by LDS-DMA: a wave's 1 KB blocks, each from one page.
// The page ids of up to 1024 / (pages per tile) tiles ahead are held in LDS.
template <int D, bool ROW32>
struct PageTiles {
  static constexpr int NB = D / 8, NP = NB / 4;          // 1 KB blocks of a tile, of a wave
  // byte offset of the lane's 16 bytes in a block of a page; where 32 consecutive rows are read
  // (ROW32) the swizzle is that of the wave for each of its blocks
  int voff[ROW32 ? 1 : NP], wave;
  KeyTiles keys;
  const int32_t* table;                // the request's pages
  int* ids;
  int end, h, c0, c1, filled;          // its keys, the kv head; the unit's tiles; those from `filled` - span on are held
  int per, span;                       // pages per tile (at least one), tiles that `ids` holds
  bool once;                           // no other workgroup reads these rows

  __device__ inline PageTiles(const PagedArgs& a, const Unit& u, const KeyTiles& k, int* lds_ids, bool read_once)
      : keys(k), ids(lds_ids), once(read_once) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < (ROW32 ? 1 : NP); ++p) {
      const int e = (4 * p + wave) * 512 + 8 * lane, row = e / D;
      voff[p] = 2 * (row * D + ((((e % D) >> 3) ^ lds_swz<D, ROW32>(row)) << 3) - (4 * p + wave) * 512);
    }
    table = a.table + (int64_t)u.r * a.max_pages;
    end = u.base + u.n;
    h = u.h;
    c0 = __builtin_amdgcn_readfirstlane((int)((int64_t)k.n * u.slice / u.n_slices));
    c1 = __builtin_amdgcn_readfirstlane((int)((int64_t)k.n * (u.slice + 1) / u.n_slices));
    per = max(1, kTileN >> a.shift);
    span = kIds / per;
    filled = c0;
  }
  // The ids of tiles c .. c + span - 1; every wave comes here at the same tile.
  __device__ inline void fill(const PagedArgs& a, int c) {
    __syncthreads();                   // the ids before have been read
    for (int i = threadIdx.x; i < min(span, c1 - c) * per; i += 256) {
      const int x = keys.first_key(c + i / per) + (i % per << a.shift);
      const int id = table[min(x, end - 1) >> a.shift];
      ids[i] = x < end && (unsigned)id < (unsigned)a.num_pages ? id : -1;
    }
    __syncthreads();
    filled = c + span;
  }
  __device__ inline void before(const PagedArgs& a, int c) {
    if (c >= filled) fill(a, c);
  }
  __device__ inline void load(const PagedArgs& a, const uint16_t* pool, int c, const uint16_t* lds) const {
    const uint32_t l0 = lds_addr(lds);
    const int x0 = keys.first_key(c), i0 = (c - (filled - span)) * per;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int blk = 4 * p + wave, row = blk * (512 / D), x = x0 + row;      // the block's first row
      const int id = __builtin_amdgcn_readfirstlane(ids[i0 + (a.shift < 6 ? row >> a.shift : 0)]);
      const int in_page = x & ((1 << a.shift) - 1);
      const int64_t first = (((int64_t)max(id, 0) * a.H_kv + h) << a.shift) + in_page;
      const int rows = id < 0 ? 0 : max(0, min(512 / D, end - x));
      dma_buf16(buffer_rsrc(pool + first * D, rows * D * 2), voff[ROW32 ? 0 : p], l0 + blk * 1024, once);
    }
  }
};

// ---------------------------------------------------------------------------
// Up to 32 rows.
// ---------------------------------------------------------------------------
struct StreamRow {
  int pos;
  uint64_t word;                       // ancestors
};
// The token rule for StreamWave: token t is key t of the request.
struct PagedRule {
  int base, last, sink, window;        // last: of the rows' positions, or above it
  bool tree;
  __device__ inline bool partly_hidden(int t, int n) const {
    return t + n > base || (t + n > sink && max(t, sink) <= last - window);
  }
  __device__ inline bool visible(const StreamRow& r, int t) const {
    const bool rule = (t < sink) | (t > r.pos - window);
    if (!tree) return (t <= r.pos) & rule;
    return t < base ? rule : (r.word >> ((t - base) & 63)) & 1;
  }
};

// The states that slices leave: acc [rows][max_slices][D], ml [rows][max_slices][2] for
// rows = (token, q head), and how many a token has.
__device__ inline float* slice_acc(const PagedArgs& a, int64_t row, int slice, int D) {
  return a.acc + (row * a.max_slices + slice) * D;
}
__device__ inline float2* slice_ml(const PagedArgs& a, int64_t row, int slice) {
  return (float2*)a.ml + row * a.max_slices + slice;
}

// As the streams of the other caches: two key tiles in flight, so that no registers hold
// loads. Bound by HBM.
template <typename T, int D, int NB>
__device__ inline void paged_stream(const PagedArgs& a, const Unit& u, uint16_t* sk, uint16_t* sv, int* ids) {
  constexpr int TILE = kTileN * D;
  const int rows = u.n * a.group;
  auto token = [&](int r) { return u.first + min(r, rows - 1) / a.group; };
  StreamWave<T, T, D, NB, 1, true, false, StreamRow> w(
      0, rows, a.q_sign,
      [&](int r) { return a.q + (int64_t)token(r) * a.q_stride + (u.h * a.group + r % a.group) * D; },
      [&](int r) {
        const int t = token(r);
        return StreamRow{a.positions[t], a.ancestors ? a.ancestors[(int64_t)t * a.words] : 0};
      });
  const PagedRule rule{u.base, u.base + u.n - 1, a.sink, a.window, a.ancestors != nullptr};
  PageTiles<D, false> page(a, u, KeyTiles(a, u.base, u.base + u.n), ids, true);
  dma_wait();   // the loads above are complete before any LDS-DMA is in flight
  auto issue = [&](int c) {
    const int b = (c - page.c0) & 1;
    page.before(a, c);
    page.load(a, a.k_pages, c, sk + b * TILE);
    page.load(a, a.v_pages, c, sv + b * TILE);
  };
  if (page.c0 < page.c1) issue(page.c0);
  if (page.c0 + 1 < page.c1) issue(page.c0 + 1);
  for (int c = page.c0; c < page.c1; ++c) {
    const int b = (c - page.c0) & 1;
    wait_chunks<page.NP, 2>(min(1, page.c1 - 1 - c));     // tile c has landed
    __syncthreads();
    w.step(a, rule, sk + b * TILE, sv + b * TILE, page.keys.first_key(c), page.end);
    __syncthreads();                             // every wave is done with buffer b
    if (c + 2 < page.c1) issue(c + 2);
  }
  w.finish(rows, (float*)sk, (float*)sv, [&](int r, int d, floatx4 x, float M, float L) {
    const int64_t row = (int64_t)token(r) * a.H + u.h * a.group + r % a.group;
    if (u.n_slices == 1) {
      x = x / (L == 0.f ? 1.f : L);              // no visible key: 0; NaN stays NaN
      *(uint2*)(a.o + row * D + d) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
      if (d == 0 && a.lse) a.lse[row] = L == 0.f ? 0.f : lse_natural(M, L);
    } else {
      *(floatx4*)(slice_acc(a, row, u.slice, D) + d) = x;
      if (d == 0) *slice_ml(a, row, u.slice) = make_float2(M, L);
    }
  });
}

// ---------------------------------------------------------------------------
// Tiles of 128 rows.
// ---------------------------------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16, a wave's 32 rows as columns, the
// row sums on the matrix pipe too. At head_dim 128 the loop is skewed by one key tile, as
// in the prefill forward: S of tile c + 1 (matrix cores) while tile c's probabilities are
// formed (VALU), then O of tile c while the maxima of S are taken, the two interleaved by
// sched_group_barrier. K is read one tile ahead of V.
template <int D> constexpr bool kPagedSkew = D >= 128;
constexpr int kAheadS = 4, kAheadO = 8, kValuS = 3, kValuO = 1;

template <typename T, int D>
__device__ inline void paged_tile(const PagedArgs& a, const Unit& u, uint16_t* sk, uint16_t* sv, int* ids) {
  constexpr int KS = D / 16, DT = D / 32, TILE = kTileN * D;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = u.n * a.group, row0 = u.tile * kRowTile, roww = row0 + wave * 32;
  const int hi = lane >> 5, col = lane & 31;
  const Lane32<D> lanes(lane);
  const bool mine = roww + col < rows;                     // the lane's row of the request's
  const uint32_t token = mine ? (roww + col) / a.group : 0;      // the request's
  const int head = u.h * a.group + (mine ? (roww + col) % a.group : 0);
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint4 w = *(const uint4*)(a.q + (int64_t)(u.first + token) * a.q_stride + head * D + 16 * ks + 8 * hi);
    w = make_uint4((w.x & a.q_and) ^ a.q_xor, (w.y & a.q_and) ^ a.q_xor, (w.z & a.q_and) ^ a.q_xor, (w.w & a.q_and) ^ a.q_xor);
    qf[ks] = mine ? w : make_uint4(0, 0, 0, 0);
  }
  dma_wait();   // these loads are complete before any LDS-DMA is in flight

  const bool tree = a.ancestors != nullptr;
  const int last_token = min(row0 + kRowTile - 1, rows - 1) / a.group;
  // an ancestor has a lower number, a node's position is at least base
  const KeyTiles keys(a, u.base + (tree ? 0 : row0 / a.group), u.base + last_token + 1);
  PageTiles<D, true> page(a, u, keys, ids, rows <= kRowTile);
  // the wave's rows see all keys up to all_to that no window hides: it reaches from above last_pos - W
  const bool active = roww < rows;
  const int all_to = tree ? u.base - 1 : u.base + min(roww, rows - 1) / a.group;
  const int hidden_to = u.base + min(roww + 31, rows - 1) / a.group - a.window;

  floatx16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = splat16(0.f);
  floatx4 lsum = floatx4{0.f, 0.f, 0.f, 0.f};
  // row sums on the matrix pipe: lane l gets that of row l & 31 of the operand of 32 rows
  const uint32_t one = ((lane >> 2) & 1) == ((lane >> 4) & 1) ? T::ones8().x : 0u;
  const float slack = kStreamSlack / a.scale_log2;
  float nm = 0.f, thr = kNegInf;

  auto scores = [&](const uint16_t* ck, floatx16 (&s)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[t] = T::mfma32(lanes.rows(ck, t, ks), qf[ks], ks == 0 ? splat16(0.f) : s[t]);
  };
  auto mask = [&](int c, floatx16 (&s)[2]) {
    const int x0 = keys.first_key(c);
    if (x0 + kTileN - 1 <= all_to && (x0 > hidden_to || x0 + kTileN <= a.sink)) return;
    const uint64_t bits = seen_bits(a, u, token, x0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const LaneBits32 vis((uint32_t)(bits >> (32 * t)), hi);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = vis.pick(r, s[t][r], kNegInf);
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
  // the reference follows the row's largest score where this exceeds it by the slack
  auto move_max = [&](float mx) {
    if (__any(mx > thr)) {
      const float mr = half_max(mx);
      const bool grow = mr > thr;
      const float nm1 = grow ? -mr * a.scale_log2 : nm;
      // a first reference below zero scales nothing yet (o = lsum = 0)
      const float alpha = __builtin_amdgcn_exp2f(fminf(nm1 - nm, 0.f));
      nm = nm1;
      thr = grow ? mr + slack : thr;
      lsum[0] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
  };
  auto probs = [&](floatx16 (&s)[2], uint4 (&p)[4]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], a.scale_log2, nm));
      p[2 * t] = pack8<T>(s[t], 0);
      p[2 * t + 1] = pack8<T>(s[t], 1);
    }
  };
  auto pin = [&](uint4 (&p)[4]) {
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      u32x4 w = __builtin_bit_cast(u32x4, p[st]);
      asm volatile("" : "+v"(w));
      p[st] = __builtin_bit_cast(uint4, w);
    }
  };
  auto accumulate = [&](const uint16_t* cv, const uint4 (&p)[4]) {
    uint32_t w = one;                  // the operand is made here: four registers fewer while P is formed
    asm volatile("" : "+v"(w));
    const uint4 ones = make_uint4(w, w, w, w);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma32(lanes.cols(cv, st, dt), p[st], o[dt]);
      lsum = T::mfma(ones, p[st], lsum);
    }
  };
  auto stage_k = [&](int c, int b) {
    page.before(a, c);
    page.load(a, a.k_pages, c, sk + b * TILE);
  };
  auto stage_v = [&](int c, int b) { page.load(a, a.v_pages, c, sv + b * TILE); };
  const int c0 = page.c0, n = page.c1 - page.c0;
  if constexpr (!kPagedSkew<D>) {
    if (n > 0) {
      stage_k(c0, 0);
      stage_v(c0, 0);
    }
    dma_wait();
    __syncthreads();
    // unrolled by two so that the buffers are constants of the instructions
    auto step = [&](int j, int buf) {
      if (j + 1 < n) {
        stage_k(c0 + j + 1, buf ^ 1);
        stage_v(c0 + j + 1, buf ^ 1);
      }
      if (active) {
        floatx16 s[2];
        uint4 p[4];
        mfma_priority_hi<true>();
        scores(sk + buf * TILE, s);
        mfma_priority_lo<true>();
        mask(c0 + j, s);
        move_max(lane_max(s));
        probs(s, p);
        mfma_priority_hi<true>();
        accumulate(sv + buf * TILE, p);
        mfma_priority_lo<true>();
      }
      dma_wait();
      __syncthreads();
    };
    int j = 0;
    for (; j + 1 < n; j += 2) {
      step(j, 0);
      step(j + 1, 1);
    }
    if (j < n) step(j, 0);
  } else {
    // prologue: K_0, V_0 and K_1 in LDS, S_0 with its maxima
    floatx16 sa[2], sb[2];
    if (n > 0) {
      stage_k(c0, 0);
      stage_v(c0, 0);
      if (n > 1) stage_k(c0 + 1, 1);
    }
    dma_wait();
    __syncthreads();
    if (n > 0 && active) {
      scores(sk, sa);
      mask(c0, sa);
      move_max(lane_max(sa));
    }
    __syncthreads();   // every wave is done with K_0 before iteration 0 refills its buffer
    auto step = [&](int j, int par, floatx16 (&s)[2], floatx16 (&sn)[2]) {   // par = j & 1
      stage_v(c0 + j + 1, par ^ 1);
      if (j + 2 < n) stage_k(c0 + j + 2, par);
      if (active) {
        uint4 p[4];
        scores(sk + (par ^ 1) * TILE, sn);
        probs(s, p);
        pin(p);                        // P is formed here, not sunk past the mask branch into the next block
        __builtin_amdgcn_sched_group_barrier(0x100, kAheadS, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (i + kAheadS < 2 * KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, kValuS, 0);
        }
        mask(c0 + j + 1, sn);
        accumulate(sv + par * TILE, p);
        const float mx = lane_max(sn);
        __builtin_amdgcn_sched_group_barrier(0x100, kAheadO, 1);
#pragma unroll
        for (int i = 0; i < 4 * DT; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
          if (2 * i + kAheadO < 8 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
          __builtin_amdgcn_sched_group_barrier(0x002, kValuO, 1);
        }
        move_max(mx);
      }
      dma_wait();
      __syncthreads();
    };
    // unrolled by two so that the score buffers swap roles without copies
    int j = 0;
    for (; j + 2 < n; j += 2) {
      step(j, 0, sa, sb);
      step(j + 1, 1, sb, sa);
    }
    if (j + 1 < n) {
      step(j, 0, sa, sb);
      sa[0] = sb[0], sa[1] = sb[1];
    }
    if (n > 0 && active) {
      uint4 p[4];
      probs(sa, p);
      pin(p);
      accumulate(sv + ((n - 1) & 1) * TILE, p);
    }
  }

  // the row afresh, not held through the loop
  const int lane_e = lane_now(), hi_e = lane_e >> 5, my = roww + (lane_e & 31);
  if (my >= rows) return;
  const float l = lsum[0];
  const int64_t row = (int64_t)(u.first + my / a.group) * a.H + u.h * a.group + my % a.group;
  if (u.n_slices > 1) {
    float* dst = slice_acc(a, row, u.slice, D);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(floatx4*)(dst + 32 * dt + 8 * r + 4 * hi_e) =
            floatx4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
    if (hi_e == 0) *slice_ml(a, row, u.slice) = make_float2(l == 0.f ? kNegInf : -nm, l);
    return;
  }
  const float inv = l > 0.f ? 1.f / l : 1.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(uint2*)(a.o + row * D + 32 * dt + 8 * r + 4 * hi_e) =
          make_uint2(pack2<T>(o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv), pack2<T>(o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv));
  if (hi_e == 0 && a.lse) a.lse[row] = l > 0.f ? lse_natural(-nm, l) : 0.f;
}

template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void paged_kernel(PagedArgs a) {
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];
  __shared__ int ids[kIds];
  // rows behind the last request have no output: zeros
  for (int64_t x = (int64_t)a.row_starts[a.R] * a.H * (D / 8) + (int64_t)blockIdx.x * 256 + threadIdx.x;
       x < (int64_t)a.rows * a.H * (D / 8); x += (int64_t)gridDim.x * 256) {
    *(uint4*)(a.o + 8 * x) = make_uint4(0, 0, 0, 0);
    if (a.lse && x % (D / 8) == 0) a.lse[x / (D / 8)] = 0.f;
  }
  Unit u;
  if (!find_unit(a, blockIdx.x, u)) return;
  const int rows = u.n * a.group;
  if (a.max_slices > 1 && u.h == 0 && u.slice == 0) {       // for the join
    const int t0 = rows <= kFewRows ? 0 : u.tile * kRowTile / a.group;
    for (int t = t0 + threadIdx.x; t < u.n && t * a.group < (u.tile + 1) * kRowTile; t += 256) a.parts[u.first + t] = u.n_slices;
  }
  if (rows <= 16) paged_stream<T, D, 1>(a, u, sk[0], sv[0], ids);
  else if (rows <= kFewRows) paged_stream<T, D, 2>(a, u, sk[0], sv[0], ids);
  else paged_tile<T, D>(a, u, sk[0], sv[0], ids);
}

// The slices of a row joined, a wave per (token, q head): as join_kernel, with the slices
// that the token has. Rows of one slice are done.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  constexpr int E = D / 64;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= (int64_t)a.row_starts[a.R] * a.H) return;
  const int n = a.parts[row / a.H];
  if (n == 1) return;
  const float2* st = slice_ml(a, row, 0);
  const float* x = slice_acc(a, row, 0, D) + E * lane;
  float M = kNegInf;
#pragma unroll 4
  for (int p = 0; p < n; ++p) M = fmaxf(M, st[p].x);
  const float Mu = M == kNegInf ? 0.f : M;
  float L = 0.f, s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.f;
#pragma unroll 4
  for (int p = 0; p < n; ++p) {
    const float f = __builtin_amdgcn_exp2f(st[p].x - Mu);
    L += st[p].y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] += x[(size_t)p * D + e] * f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.o[row * D + E * lane + e] = T::from_float(s[e] / (L == 0.f ? 1.f : L));
  if (lane == 0 && a.lse) a.lse[row] = L == 0.f ? 0.f : lse_natural(M, L);
}

template <typename T, int D>
int paged_attend(const PagedArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((paged_kernel<T, D>), dim3((unsigned)paged_units(a)), dim3(256), 0, stream, a);
  if (a.max_slices > 1)
    hipLaunchKernelGGL((paged_join_kernel<T, D>), dim3((unsigned)(((int64_t)a.rows * a.H + 3) / 4)), dim3(256), 0, stream, a);
  return check_launch("gki_paged_attend");
}

}  // namespace

int paged_attend_dispatch(int dtype, int head_dim, const PagedArgs& a, hipStream_t stream) {
  if (dtype == kF16) return head_dim == 64 ? paged_attend<F16, 64>(a, stream) : paged_attend<F16, 128>(a, stream);
  return head_dim == 64 ? paged_attend<BF16, 64>(a, stream) : paged_attend<BF16, 128>(a, stream);
}

}  // namespace gki

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
// are its rows here. Up to 16 of them run as a stream (four waves share out the keys of a
// step), more as tiles of 128 (four waves of 32 rows). Either walks the 64-key tiles of the
// sinks and of its rows' windows once, whatever lies between, or a piece of them; pieces'
// states are joined. Pages are addressed a 1 KB LDS block at a time, each of which lies in
// one page; keys past the request's last, and pages that it does not have, are zeros
// without being read: what another request left in a page is never seen. (A NaN or
// infinity among the request's own values reaches every row of a tile that reads it.)
#include "gki_paged.cuh"
#include "gki_stream_wave.cuh"

namespace gki {
namespace {

constexpr int kRowTile = 128;          // rows of a tile: four waves of 32
// Up to as many run as a stream, us with the join, stream / tile: 32 requests' decodes of 4 rows over
// 4096 keys (D128) 90 / 104, 64 of 16 rows over 2048 95 / 103, 16 of 16 rows over 4096 54 / 51, one
// over 512 (D64) 10.8 / 12.7; with two blocks of 16 rows: 16 of 32 rows over 4096 63 / 55, 32 of 32
// rows over 1024 (D64) 31 / 26.
constexpr int kFewRows = 16;
// A cut closer than this many steps to a row tile's ends moves there (half a share at most), us with
// the join for 1 / 2 / 3 / 4 / 6 / 8: 32 decodes 44.7 / 45.0 / 43.7 / 43.8 / 44.2 / 46.7, chunks of 512
// 110 / 110 / 109 / 108 / 107 / 107, mixed 51.7 / 51.2 / 48.7 / 49.8 / 48.2 / 48.0, trees of 26 36.1 /
// 36.1 / 34.3 / 34.4 / 34.4 / 34.4, of 60 121 for all. In shares above 64 steps, closer than a 16th: four
// times 2048 rows behind 4000 keys (H32/8 D128) 587, with a 4th / an 8th / 4 steps 600 / 596 / 594.
constexpr uint32_t kCutEdge = 4;
constexpr int kPagePieces = 512;       // pieces of pages whose places are held in LDS at a time

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
// Which work a workgroup takes. The key tiles of all row tiles of all requests and kv heads,
// one after the other (request, head, row tile, key tile), are cut into equal shares, a
// workgroup each. A row tile counts as many key tiles as its request's rows see together: requests of
// any lengths load the card evenly, but the row tiles of a chunk longer than the keys before it do
// not, as the first of them walk less than they count (four prompts of 2048 tokens, H32/8 D128: 0.52
// PFLOP/s at the start, 0.93 behind 4000 keys). A row tile that a cut
// divides leaves the states of its pieces, which are joined; a cut close to its ends
// moves there. Lengths are known on the device only, so every workgroup counts for
// itself, a wave 64 requests at a time (`extend` lists those that have tokens: 32 of 4096
// requests cost what 32 of 32 do, 47 us), once: it goes from one row tile of its share to the
// next without counting again (single tokens of 8192 requests over 100 keys, 8 heads, D128: 4.46 ms
// with a count for each, 1.00 so). Neighbours work on one XCD: row tiles of a (request, head) meet
// their keys in its L2.
// ---------------------------------------------------------------------------
__device__ inline uint32_t lane_of(uint32_t x, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)x, l); }
__device__ inline uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

struct Request {
  uint32_t r, first, n, base;          // the request, first row of the step's, rows, keys before them
  uint32_t tiles, keys;                // row tiles, the steps of each
  // Number i of those that have tokens, `end` of them (a load of number 0, which may be none, is harmless).
  __device__ inline Request(const PagedArgs& a, int i, int end) {
    const int4 x = a.requests[1 + (i < end ? i : 0)];
    r = x.x, first = x.y, base = x.w;
    n = i < end ? x.z : 0;
    const uint32_t rows = n * a.group;
    tiles = (rows + kRowTile - 1) / kRowTile;
    // a walk's prologue and epilogue cost about as much as kPagedPieceCost key tiles
    const uint32_t k = KeyTiles(a, base, base + n).n + kPagedPieceCost;
    keys = max((uint32_t)kPagedMinShare, (k + (1u << a.coarse) - 1) >> a.coarse);
  }
  __device__ inline uint32_t steps(const PagedArgs& a) const { return tiles * a.H_kv * keys; }
};

// The row tile that holds a step: its request (`index` in the list), which of the request's it is
// (head by head), its first step.
struct Place {
  uint32_t first, n, base, tiles, keys, number, start;
  int r, index;
  __device__ inline void set(const Request& q, int l, int list_index, uint32_t before, uint32_t step) {
    index = list_index;
    r = lane_of(q.r, l);
    first = lane_of(q.first, l), n = lane_of(q.n, l), base = lane_of(q.base, l);
    tiles = lane_of(q.tiles, l), keys = lane_of(q.keys, l);
    number = scalar((step - before) / keys);
    start = before + number * keys;
  }
  // Row tile `number` of the request at `index`, whose first step is `start`.
  __device__ inline Place(const PagedArgs& a, int index, uint32_t number, uint32_t start)
      : number(number), start(start), index(index) {
    const Request q(a, index, index + 1);
    r = scalar(q.r);
    first = scalar(q.first), n = scalar(q.n), base = scalar(q.base);
    tiles = scalar(q.tiles), keys = scalar(q.keys);
  }
  __device__ inline Place() {}
};

struct Shares {
  Request q;                           // the lane's (its first of `run`)
  int run;                             // requests per lane
  uint32_t sum;                        // steps of lanes 0 .. this one
  uint32_t all, share;                 // steps in all, of a workgroup
  uint32_t edge;                       // cuts this close to a row tile's ends move there
  int lane;
  int n;                               // requests that have tokens
  __device__ inline Shares(const PagedArgs& a, int tid, int active)
      : q(a, (tid & 63) * ((active + 63) >> 6), active), run((active + 63) >> 6), lane(tid & 63), n(active) {
    uint32_t mine = q.steps(a);
    for (int i = 1; i < run; ++i) mine += Request(a, lane * run + i, n).steps(a);
    sum = wave_prefix(mine);
    all = lane_of(sum, 63);
    share = scalar(max((uint32_t)a.least, (all + a.groups - 1) / a.groups));
    edge = max(min(kCutEdge, share / 2), share / 16);
  }
  __device__ inline Place place(const PagedArgs& a, uint32_t step) const {      // step < all
    Place p;
    const int l = __builtin_ctzll(__ballot(sum > step));
    uint32_t before = l ? lane_of(sum, l - 1) : 0;
    if (run == 1) {
      p.set(q, l, l, before, step);
      return p;
    }
    const int end = min((l + 1) * run, n);
    for (int r0 = l * run;; r0 += 64) {
      const Request x(a, r0 + lane, end);
      const uint32_t upto = wave_prefix(x.steps(a));
      const uint64_t past = __ballot(before + upto > step);
      if (past || r0 + 64 >= end) {
        const int m = past ? __builtin_ctzll(past) : 0;
        p.set(x, m, r0 + m, before + (m ? lane_of(upto, m - 1) : 0), step);
        return p;
      }
      before += lane_of(upto, 63);
    }
  }
  // Where the cut at step c goes: it stays inside a row tile that is long enough.
  __device__ inline uint32_t cut(const PagedArgs& a, uint32_t c) const {
    if (c == 0 || c >= all) return min(c, all);
    const Place p = place(a, c);
    const uint32_t off = c - p.start;
    if (off == 0 || (a.acc && off >= edge && p.keys - off >= edge)) return c;
    return 2 * off < p.keys ? p.start : p.start + p.keys;
  }
};

// A piece of a row tile's walk: steps s0 .. s1 - 1 of `steps`. Of the pieces of a row tile that
// is cut the first is the last of its workgroup's share, any other the first of its own: the
// first of c workgroups from w on has state 2 w + 1, the others 2 (w + 1), 2 (w + 2), ...
struct Unit {
  int r, first, n, base;               // the request
  int h, tile, state;                  // state -1: all of the walk
  uint32_t s0, s1, steps;
  __device__ inline Unit(const Place& p, uint32_t lo, uint32_t hi, int w) {
    r = p.r, first = p.first, n = p.n, base = p.base;
    h = scalar(p.number / p.tiles), tile = p.number - h * p.tiles;
    steps = p.keys;
    s0 = lo - p.start;
    s1 = min(p.keys, hi - p.start);
    state = s0 > 0 ? 2 * w : s1 < steps ? 2 * w + 1 : -1;
  }
  // The first of a walk's n key tiles that belongs to step s or a later one.
  __device__ inline int tile_of(int n, uint32_t s) const {
    if (s == 0 || s == steps || (uint32_t)n == steps) return s == steps ? n : s;
    if ((n | s) < 65536) return scalar((uint32_t)n * s / steps);
    return scalar((uint32_t)((uint64_t)n * s / steps));
  }
};

// The arguments of the running kernel, whose first they are, read anew where they are needed
// once or seldom: they are not held in registers through the loops (scalar ones that do
// not fit would take vector ones).
__device__ inline PagedArgs fresh_args() {
#ifdef __HIP_DEVICE_COMPILE__          // the host's pass does not know the builtin
  const __attribute__((address_space(4))) PagedArgs* p =
      (const __attribute__((address_space(4))) PagedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
#else
  return PagedArgs{};
#endif
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
// Where the tiles' pieces (64 keys, or a page of 16 or 32) start in the pool is held in LDS
// for up to kPieces of them at a time. ONCE: no other workgroup reads these keys.
template <int D, bool ROW32, bool ONCE>
struct PageTiles {
  static constexpr int NB = D / 8, NP = NB / 4, RB = 512 / D;      // 1 KB blocks of a tile, of a wave; rows of a block
  // byte offset of the lane's 16 bytes in a block of a page; where 32 consecutive rows are read
  // (ROW32) the swizzle is that of the wave for each of its blocks
  int voff[ROW32 ? 1 : NP], wave;
  KeyTiles keys;
  int64_t* pieces;                     // bytes from the pool's start, -1: no such page
  int r, h, end, c0, c1, filled;       // its request, kv head, keys; the unit's tiles; those before `filled` are held
  int piece, per, span;                // log2 of a piece's keys, pieces of a tile, tiles that `pieces` holds

  __device__ inline PageTiles(const PagedArgs& a, const Unit& u, const KeyTiles& k, int64_t* lds, int tid)
      : keys(k), pieces(lds), r(u.r), h(u.h), end(u.base + u.n) {
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
#pragma unroll
    for (int p = 0; p < (ROW32 ? 1 : NP); ++p) {
      const int e = (4 * p + wave) * 512 + 8 * lane, row = e / D;
      voff[p] = 2 * (row * D + ((((e % D) >> 3) ^ lds_swz<D, ROW32>(row)) << 3) - (4 * p + wave) * 512);
    }
    c0 = u.tile_of(k.n, u.s0);
    c1 = u.tile_of(k.n, u.s1);
    piece = min(a.shift, 6);
    per = 64 >> piece;
    span = kPagePieces / per;
    filled = c0;
  }
  // The pieces of tiles c .. c + span - 1; every wave comes here at the same tile.
  __device__ inline void fill(int c) {
    const PagedArgs a = fresh_args();
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int32_t* table = a.table + (int64_t)r * a.max_pages;
    __syncthreads();                   // the pieces before have been read
    for (int i = tid; i < min(span, c1 - c) * per; i += 256) {
      const int x = keys.first_key(c + i / per) + (i % per << piece);
      const int id = table[min(x, end - 1) >> a.shift];
      const int64_t row = (((int64_t)id * a.H_kv + h) << a.shift) + (x & ((1 << a.shift) - 1));
      pieces[i] = x < end && (unsigned)id < (unsigned)a.num_pages ? row * (2 * D) : -1;
    }
    __syncthreads();
    filled = c + span;
  }
  __device__ inline void load(const uint16_t* pool, int c, const uint16_t* lds) {
    if (c >= filled) fill(c);
    int wave = this->wave;             // the wave's constants are made here, not held: scalars are short in the loops
    asm volatile("" : "+s"(wave));
    const uint32_t l0 = scalar(lds_addr(lds) + wave * 1024);
    const int i0 = (c - (filled - span)) * per, x0 = keys.first_key(c);
    if (per == 1) {
      const int64_t at = scalar64(pieces[i0]);
      const char* base = (const char*)pool + at + wave * 1024;
      const int left = scalar(at < 0 ? 0 : end - x0);      // keys from the tile's first on
#pragma unroll
      for (int p = 0; p < NP; ++p)
        dma_buf16(buffer_rsrc(base + p * 4096, rows_left<RB>(left - (4 * p + wave) * RB) * D * 2), voff[ROW32 ? 0 : p],
                  l0 + p * 4096, ONCE);
    } else {
      int64_t held[NP];                // all read before the first load is issued
#pragma unroll
      for (int p = 0; p < NP; ++p) held[p] = pieces[i0 + ((4 * p + wave) * RB >> piece)];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int row = (4 * p + wave) * RB;
        const int64_t at = scalar64(held[p]);
        const char* base = (const char*)pool + at + (row & ((1 << piece) - 1)) * (2 * D);
        const int left = scalar(at < 0 ? 0 : end - x0 - row);
        dma_buf16(buffer_rsrc(base, rows_left<RB>(left) * D * 2), voff[ROW32 ? 0 : p], l0 + p * 4096, ONCE);
      }
    }
  }
  __device__ static inline int64_t scalar64(int64_t x) {
    return (int64_t)((uint64_t)scalar((uint32_t)((uint64_t)x >> 32)) << 32 | scalar((uint32_t)x));
  }
};

// ---------------------------------------------------------------------------
// Up to 16 rows.
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

// Row r of a piece's state: acc [2 groups][cap][D], ml [2 groups][cap][2].
__device__ inline float* piece_acc(const PagedArgs& a, int state, int r, int D) { return a.acc + ((int64_t)state * a.cap + r) * D; }
__device__ inline float2* piece_ml(const PagedArgs& a, int state, int r) { return (float2*)a.ml + (int64_t)state * a.cap + r; }

// As the streams of the other caches: two key tiles in flight by LDS-DMA, so that no registers
// hold loads. P is rounded to T for the matrix pipe, and the sums are those of the rounded P, so
// that what rounding adds to a row's weights it adds to their sum (fp16: 2.8e-4 of the result, 3.2e-4
// with sums before rounding). Bound by HBM: 32 decodes over 4096 keys, D128 H32/8, 537 MB in
// 90 us with the join, 6.0 TB/s.
template <typename T, int D>
__device__ inline void paged_stream(const PagedArgs& a, const Unit& u, uint16_t* sk, uint16_t* sv, int64_t* pieces, int tid) {
  constexpr int TILE = kTileN * D;
  const int rows = u.n * a.group;
  auto token = [&](int r) { return u.first + min(r, rows - 1) / a.group; };
  // the first keys are on their way while the queries are read
  PageTiles<D, false, true> page(a, u, KeyTiles(a, u.base, u.base + u.n), pieces, tid);
  auto issue = [&](int c) {
    const int b = (c - page.c0) & 1;
    page.load(a.k_pages, c, sk + b * TILE);
    page.load(a.v_pages, c, sv + b * TILE);
  };
  if (page.c0 < page.c1) issue(page.c0);
  if (page.c0 + 1 < page.c1) issue(page.c0 + 1);
  StreamWave<T, T, D, 1, 1, true, false, StreamRow, true> w(
      0, rows, a.q_sign,
      [&](int r) { return a.q + (int64_t)token(r) * a.q_stride + (u.h * a.group + r % a.group) * D; },
      [&](int r) {
        const int t = token(r);
        return StreamRow{a.positions[t], a.ancestors ? a.ancestors[(int64_t)t * a.words] : 0};
      }, tid);
  const PagedRule rule{u.base, u.base + u.n - 1, a.sink, a.window, a.ancestors != nullptr};
  dma_wait();
  for (int c = page.c0; c < page.c1; ++c) {
    const int b = (c - page.c0) & 1;
    wait_chunks<page.NP, 2>(min(1, page.c1 - 1 - c));     // tile c has landed
    __syncthreads();
    w.step(a, rule, sk + b * TILE, sv + b * TILE, page.keys.first_key(c), page.end);
    __syncthreads();                             // every wave is done with buffer b
    if (c + 2 < page.c1) issue(c + 2);
  }
  w.finish(rows, (float*)sk, (float*)sv, [&, a = fresh_args()](int r, int d, floatx4 x, float M, float L) {
    if (u.state < 0) {
      const int64_t row = (int64_t)token(r) * a.H + u.h * a.group + r % a.group;
      x = x / (L == 0.f ? 1.f : L);              // no visible key: 0; NaN stays NaN
      *(uint2*)(a.o + row * D + d) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
      if (d == 0 && a.lse) a.lse[row] = L == 0.f ? 0.f : lse_natural(M, L);
    } else if (r < a.cap) {
      *(floatx4*)(piece_acc(a, u.state, r, D) + d) = x;
      if (d == 0) *piece_ml(a, u.state, r) = make_float2(M, L);
    }
  }, tid);
}

// ---------------------------------------------------------------------------
// Tiles of 128 rows.
// ---------------------------------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16, a wave's 32 rows as columns, the
// row sums on the matrix pipe too. At head_dim 128 the loop is skewed by one key tile, as
// in the prefill forward: S of tile c + 1 (matrix cores) while tile c's probabilities are
// formed (VALU), then O of tile c while the maxima of S are taken, the two interleaved by
// sched_group_barrier. K is read one tile ahead of V. P is rounded to T, as are the outputs; S, the
// maxima, the sums and O are in 32 bits. Two workgroups of a CU take 2.0 us for a 64-key step of
// each (1.07 PFLOP/s on 256 CUs), one alone 1.25 to 1.43. Chunks of 512 (4 requests, H32/8, W4096) 101
// us of kernel for 68 GFLOP: 1.4 of two waves a SIMD on average, as shares are uneven and pieces have
// their ends, the matrix cores busy for 33% of it, the VALU for 26%. Trees of 60 (8 requests, H64/8,
// W8192) 114 us: the row tiles of a (request, head) read its keys apart in time, 591 MB past L2 for 200
// MB of keys and values, 5.2 TB/s.
template <int D> constexpr bool kPagedSkew = D >= 128;
constexpr int kAheadS = 4, kAheadO = 8, kValuS = 3, kValuO = 1;

template <typename T, int D>
__device__ inline void paged_tile(const PagedArgs& a, const Unit& u, uint16_t* sk, uint16_t* sv, int64_t* pieces, int tid) {
  constexpr int KS = D / 16, DT = D / 32, TILE = kTileN * D;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = u.n * a.group, row0 = u.tile * kRowTile, roww = row0 + wave * 32;
  const int hi = lane >> 5, col = lane & 31;
  const Lane32<D> lanes(lane);
  const bool mine = roww + col < rows;                     // the lane's row of the request's
  const uint32_t token = mine ? (roww + col) / a.group : 0;      // the request's
  const bool tree = a.ancestors != nullptr;
  // quotients as scalars, and with them the walk
  const int last_token = scalar(min(row0 + kRowTile - 1, rows - 1) / a.group);
  // an ancestor has a lower number, a node's position is at least base
  const KeyTiles keys(a, u.base + (tree ? 0 : (int)scalar(row0 / a.group)), u.base + last_token + 1);
  PageTiles<D, true, false> page(a, u, keys, pieces, tid);
  // the wave's rows see all keys up to all_to that no window hides: it reaches from above last_pos - W
  const bool active = roww < rows;
  const int all_to = tree ? u.base - 1 : u.base + (int)scalar(min(roww, rows - 1) / a.group);
  const int hidden_to = u.base + (int)scalar(min(roww + 31, rows - 1) / a.group) - a.window;

  auto stage_k = [&](int c, int b) { page.load(a.k_pages, c, sk + b * TILE); };
  auto stage_v = [&](int c, int b) { page.load(a.v_pages, c, sv + b * TILE); };
  // the first tiles are on their way while the queries are read
  const int c0 = page.c0, n = page.c1 - page.c0;
  if (n > 0) {
    stage_k(c0, 0);
    stage_v(c0, 0);
    if (kPagedSkew<D> && n > 1) stage_k(c0 + 1, 1);
  }
  const int head = u.h * a.group + (mine ? (roww + col) % a.group : 0);
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint4 w = *(const uint4*)(a.q + (int64_t)(u.first + token) * a.q_stride + head * D + 16 * ks + 8 * hi);
    w = make_uint4((w.x & a.q_and) ^ a.q_xor, (w.y & a.q_and) ^ a.q_xor, (w.z & a.q_and) ^ a.q_xor, (w.w & a.q_and) ^ a.q_xor);
    qf[ks] = mine ? w : make_uint4(0, 0, 0, 0);
  }
  floatx16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = splat16(0.f);
  // row sums on the matrix pipe: lane l gets that of row l & 31 of the operand of 32 rows
  floatx4 lsum = floatx4{0.f, 0.f, 0.f, 0.f};
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
    int l = threadIdx.x & 31;
    asm volatile("" : "+v"(l));
    const PagedArgs e = fresh_args();
    const uint64_t bits = seen_bits(e, u, min(roww + l, rows - 1) / e.group, x0);
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
    int l = threadIdx.x;               // the operand is made here: five registers fewer while P is formed
    asm volatile("" : "+v"(l));
    const uint32_t w = ((l >> 2) & 1) == ((l >> 4) & 1) ? T::ones8().x : 0u;
    const uint4 ones = make_uint4(w, w, w, w);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma32(lanes.cols(cv, st, dt), p[st], o[dt]);
      lsum = T::mfma(ones, p[st], lsum);
    }
  };
  if constexpr (!kPagedSkew<D>) {
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
    dma_wait();
    __syncthreads();
    if (!active) {     // a wave without rows brings its part of the tiles
      __syncthreads();
      for (int j = 0; j + 1 < n; ++j) {
        stage_v(c0 + j + 1, (j & 1) ^ 1);
        if (j + 2 < n) stage_k(c0 + j + 2, j & 1);
        dma_wait();
        __syncthreads();
      }
      return;
    }
    if (n > 0) {
      scores(sk, sa);
      mask(c0, sa);
      move_max(lane_max(sa));
    }
    __syncthreads();   // every wave is done with K_0 before iteration 0 refills its buffer
    auto step = [&](int j, int par, floatx16 (&s)[2], floatx16 (&sn)[2]) {   // par = j & 1
      stage_v(c0 + j + 1, par ^ 1);
      if (j + 2 < n) stage_k(c0 + j + 2, par);
      {
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
    if (n > 0) {
      uint4 p[4];
      probs(sa, p);
      pin(p);
      accumulate(sv + ((n - 1) & 1) * TILE, p);
    }
  }

  // the row afresh, not held through the loop
  int lane_e = threadIdx.x & 63;
  asm volatile("" : "+v"(lane_e));
  const PagedArgs e = fresh_args();
  const int hi_e = lane_e >> 5, my = roww + (lane_e & 31);
  if (my >= rows) return;
  const float l = lsum[0];
  if (u.state >= 0) {
    if (my - row0 >= e.cap) return;
    float* dst = piece_acc(e, u.state, my - row0, D);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(floatx4*)(dst + 32 * dt + 8 * r + 4 * hi_e) =
            floatx4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
    if (hi_e == 0) *piece_ml(e, u.state, my - row0) = make_float2(l == 0.f ? kNegInf : -nm, l);
    return;
  }
  const int64_t row = (int64_t)(u.first + my / e.group) * e.H + u.h * e.group + my % e.group;
  const float inv = l == 0.f ? 1.f : 1.f / l;              // no visible key: 0; NaN stays NaN
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(uint2*)(e.o + row * D + 32 * dt + 8 * r + 4 * hi_e) =
          make_uint2(pack2<T>(o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv), pack2<T>(o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv));
  if (hi_e == 0 && e.lse) e.lse[row] = l == 0.f ? 0.f : lse_natural(-nm, l);
}

template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 4 : 2) void paged_kernel(PagedArgs args) {
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];
  __shared__ int64_t pieces[kPagePieces];
  __shared__ uint32_t todo[2][4];
  __shared__ uint32_t cut[3];
  // rows behind the last request have no output: zeros
  for (int64_t x = (int64_t)args.requests[0].y * args.H * (D / 8) + (int64_t)blockIdx.x * 256 + threadIdx.x;
       x < (int64_t)args.rows * args.H * (D / 8); x += (int64_t)gridDim.x * 256) {
    *(uint4*)(args.o + 8 * x) = make_uint4(0, 0, 0, 0);
    if (args.lse && x % (D / 8) == 0) args.lse[x / (D / 8)] = 0.f;
  }
  // One piece of the share after the other. Only the rest of the share (steps lo .. hi - 1, the row
  // tile at lo) and how shares are cut are kept between two, in LDS (the rest by turns, as a wave may
  // read it late), so that the row tiles have their registers.
  for (int turn = 0;; ++turn) {
    const PagedArgs a = fresh_args();
    int tid = threadIdx.x;             // not an invariant: nothing made from it is held either
    asm volatile("" : "+v"(tid));
    uint32_t lo, hi, share, edge;
    int w;
    Place p;
    if (turn == 0) {
      const Shares s(a, tid, a.requests[0].x);
      const int used = (int)((s.all + s.share - 1) / s.share);
      const bool idle = (int)blockIdx.x >= used;
      w = idle ? (int)blockIdx.x : xcd_remap(blockIdx.x, used);
      if (a.acc && tid == 0) a.cuts[w].pieces = 0;
      if (idle) return;
      lo = s.cut(a, w * s.share), hi = s.cut(a, (w + 1) * s.share);
      if (lo >= hi) return;
      p = s.place(a, lo);
      share = s.share, edge = s.edge;
      if (tid == 0) cut[0] = share, cut[1] = edge, cut[2] = w;
    } else {
      const uint32_t* rest = todo[turn & 1];
      lo = scalar(rest[0]), hi = scalar(rest[1]);
      if (lo >= hi) return;
      p = Place(a, (int)scalar(rest[2]), scalar(rest[3]), lo);
      share = scalar(cut[0]), edge = scalar(cut[1]), w = (int)scalar(cut[2]);
    }
    const Unit u(p, lo, hi, w);
    if (tid == 0) {
      // of the row tiles of all heads of all requests of the list the next
      const bool more = p.number + 1 < p.tiles * a.H_kv;
      uint32_t* rest = todo[(turn + 1) & 1];
      rest[0] = lo + (u.s1 - u.s0);
      rest[1] = hi;
      rest[2] = more ? p.index : p.index + 1;
      rest[3] = more ? p.number + 1 : 0;
      if (u.state == 2 * w + 1)        // for the join: cuts at the shares' ends up to the edge
        a.cuts[w] = CutTile{u.first, u.n, u.h, u.tile, 2 + (int)((p.start + p.keys - edge) / share - (w + 1))};
    }
    const int rows = u.n * a.group;
    if (rows <= kFewRows) paged_stream<T, D>(a, u, sk[0], sv[0], pieces, tid);
    else paged_tile<T, D>(a, u, sk[0], sv[0], pieces, tid);
    __syncthreads();                   // LDS is read no more
  }
}

// The pieces of the row tile that workgroup blockIdx.x's share ends in, if it is cut, joined: a
// thread for four elements of a row, pieces in order. As join_kernel: O = sum_p f_p acc_p / sum_p
// f_p l_p, f_p = exp2(m_p - M). Bound by latency (the cut, the maxima, the sums): many small
// workgroups, most of which leave at once. 4.5 us for 32 decodes, 12 for trees of 60
// (19 where a thread had more of a row), 13 where 128 rows of every share are cut (67 MB of states).
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedArgs a) {
  constexpr int RPG = kJoinThreads / (D / 4);
  const CutTile c = a.cuts[blockIdx.x];
  if (c.pieces == 0) return;
  const int rows = c.n * a.group, row0 = c.tile * kRowTile;
  const int r = blockIdx.y * RPG + threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
  if (r >= min(min(rows - row0, kRowTile), a.cap)) return;
  auto state = [&](int p) { return p == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + p); };
  float M = kNegInf;
#pragma unroll 4
  for (int p = 0; p < c.pieces; ++p) M = fmaxf(M, piece_ml(a, state(p), r)->x);
  const float Mu = M == kNegInf ? 0.f : M;
  float L = 0.f;
  floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < c.pieces; ++p) {
    const float2 ml = *piece_ml(a, state(p), r);
    const float f = __builtin_amdgcn_exp2f(ml.x - Mu);
    L += ml.y * f;
    x += *(const floatx4*)(piece_acc(a, state(p), r, D) + d) * f;
  }
  x = x / (L == 0.f ? 1.f : L);
  const int64_t row = (int64_t)(c.first + (row0 + r) / a.group) * a.H + c.h * a.group + (row0 + r) % a.group;
  *(uint2*)(a.o + row * D + d) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
  if (d == 0 && a.lse) a.lse[row] = L == 0.f ? 0.f : lse_natural(M, L);
}

template <typename T, int D>
int paged_attend(const PagedArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((paged_kernel<T, D>), dim3(a.groups), dim3(256), 0, stream, a);
  const dim3 grid(a.groups, (a.cap * (D / 4) + kJoinThreads - 1) / kJoinThreads);
  if (a.acc) hipLaunchKernelGGL((paged_join_kernel<T, D>), grid, dim3(kJoinThreads), 0, stream, a);
  return check_launch("gki_paged_attend");
}

}  // namespace

int paged_attend_dispatch(int dtype, int head_dim, const PagedArgs& a, hipStream_t stream) {
  if (dtype == kF16) return head_dim == 64 ? paged_attend<F16, 64>(a, stream) : paged_attend<F16, 128>(a, stream);
  return head_dim == 64 ? paged_attend<BF16, 64>(a, stream) : paged_attend<BF16, 128>(a, stream);
}

}  // namespace gki

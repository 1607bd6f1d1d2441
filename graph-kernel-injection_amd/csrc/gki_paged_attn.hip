// Attention of requests of different lengths over paged keys and values, with sinks and a
// sliding window (the StreamingLLM rule), for gfx950.
//
// Request r has `base` keys and brings n rows, which stand behind them at places base + i.
// A row at position p sees the keys x <= p with x < S or x > p - W:
//   S_x = scale * q . k_x,  O = sum_x exp(S_x - m) v_x / sum_x exp(S_x - m),  LSE = m + ln(sum).
// Drafted trees: row i stands at p = base + depth_i; of the keys from base on it sees those
// that its word of ancestors names (which has the rule in it already).
//
// The rows of a request that read one kv head, (token, q head of the group) token by
// token, are cut into tiles; a tile walks the 64-key tiles of the sinks and of its rows'
// windows once, whatever lies between. Pages are addressed a 1 KB LDS block at a time, each
// of which lies in one page; keys past the request's last, and pages that it does not have,
// are zeros without being read: what another request left in a page is never seen. (A NaN or
// infinity among the request's own values reaches every row of a tile that reads it.)
#include "gki_paged.cuh"

namespace gki {
namespace {

constexpr float kSlack = 8.f;          // log2 units that the reference max may lag
constexpr int kTile = 128;             // rows of a tile: four waves of 32

// What a workgroup works on: rows row0 .. row0 + n_rows - 1 of those that request r has of
// a kv head.
struct PagedPlace {
  int r, tile, first, n, base;         // first row of the request in the step, its rows, its keys before them
};

// The place of tile number t over all requests: a wave counts 64 requests at a time.
__device__ inline bool find_place(const PagedArgs& a, int t, PagedPlace& at) {
  const int lane = threadIdx.x & 63;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const int r = min(r0 + lane, a.R - 1);
    const int s = a.row_starts[r], n = r0 + lane < a.R ? a.row_starts[r + 1] - s : 0;
    const int tiles = (n * a.group + kTile - 1) / kTile;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum, o);
      if (lane >= o) sum += y;
    }
    const uint64_t past = __ballot(sum > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      at.r = r0 + l;
      at.tile = t - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
      at.first = __builtin_amdgcn_readlane(s, l);
      at.n = __builtin_amdgcn_readlane(n, l);
      at.base = __builtin_amdgcn_readfirstlane(a.base[at.r]);
      return true;
    }
    t -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

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

// Keys of the 64 from x0 on that a row sees.
__device__ inline uint64_t seen_bits(const PagedArgs& a, int row, int pos, int base, int x0) {
  const uint64_t rule = bit_range(pos - a.window + 1 - x0, 63) | bit_range(0, a.sink - 1 - x0);
  if (a.ancestors == nullptr) return bit_range(0, pos - x0) & rule;
  uint64_t bits = bit_range(0, base - 1 - x0) & rule;
  const uint64_t* word = a.ancestors + (int64_t)row * a.words;
  const int from = x0 - base;          // number of the node at x0
  if (from > -64) {
    if (from < 0) {
      bits |= word[0] << -from;
    } else if ((from >> 6) < a.words) {
      const int w = from >> 6, sh = from & 63;
      bits |= word[w] >> sh;
      if (sh && w + 1 < a.words) bits |= word[w + 1] << (64 - sh);
    }
  }
  return bits;
}

// A tile of 64 keys or values into LDS: the wave's 1 KB blocks, each from one page.
template <int D>
struct PageTile {
  DmaTile<D, 4, true> dma;
  const int32_t* table;                // the request's pages
  int end, h;                          // its keys, the kv head
  __device__ inline void load(const PagedArgs& a, const uint16_t* pool, int x0, const uint16_t* lds) const {
    const uint32_t l0 = lds_addr(lds);
#pragma unroll
    for (int p = 0; p < dma.NP; ++p) {
      const int blk = 4 * p + dma.wave;
      if (dma.NB % 4 == 0 || blk < dma.NB) {
        const int row = blk * (512 / D), x = x0 + row;               // the block's first row; its page
        const int id = x < end ? __builtin_amdgcn_readfirstlane(table[x >> a.shift]) : -1;
        const bool there = (unsigned)id < (unsigned)a.num_pages;
        const int in_page = x & ((1 << a.shift) - 1);
        // as if the tile's row 0 lay in this page too: the lane's offsets are those of whole tiles
        const int64_t row0 = ((((int64_t)(there ? id : 0) * a.H_kv + h) << a.shift) + in_page) - row;
        const int rows = there ? row + min((1 << a.shift) - in_page, end - x) : 0;
        dma_buf16(buffer_rsrc(pool + row0 * D, rows * D * 2), 2 * dma.off[p], l0 + blk * 1024);
      }
    }
  }
};

template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void paged_tiles_kernel(PagedArgs a) {
  constexpr int KS = D / 16, DT = D / 32;
  __shared__ __align__(16) uint16_t sk[2][kTileN * D];
  __shared__ __align__(16) uint16_t sv[2][kTileN * D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y;

  // rows behind the last request have no output: zeros
  for (int64_t x = (int64_t)a.row_starts[a.R] * a.H * (D / 8) + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + tid;
       x < (int64_t)a.rows * a.H * (D / 8); x += (int64_t)gridDim.x * gridDim.y * 256) {
    *(uint4*)(a.o + 8 * x) = make_uint4(0, 0, 0, 0);
    if (a.lse && x % (D / 8) == 0) a.lse[x / (D / 8)] = 0.f;
  }
  PagedPlace at;
  if (!find_place(a, blockIdx.x, at)) return;
  const int rows = at.n * a.group, row0 = at.tile * kTile;
  const int hi = lane >> 5, col = lane & 31;
  const Lane32<D> lanes(lane);
  const int my = row0 + wave * 32 + col;                   // the lane's row of the request's
  const bool mine = my < rows;
  const int token = at.first + (mine ? my / a.group : 0), head = h * a.group + (mine ? my % a.group : 0);
  const int pos = a.positions[token];
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint4 w = *(const uint4*)(a.q + (int64_t)token * a.q_stride + head * D + 16 * ks + 8 * hi);
    w = make_uint4((w.x & a.q_and) ^ a.q_xor, (w.y & a.q_and) ^ a.q_xor, (w.z & a.q_and) ^ a.q_xor, (w.w & a.q_and) ^ a.q_xor);
    qf[ks] = mine ? w : make_uint4(0, 0, 0, 0);
  }
  dma_wait();   // these loads are complete before any LDS-DMA is in flight

  const bool tree = a.ancestors != nullptr;
  const int last_token = min(row0 + kTile - 1, rows - 1) / a.group;
  const int end = at.base + last_token + 1;                // an ancestor has a lower number
  const KeyTiles keys(a, at.base + (tree ? 0 : row0 / a.group), end);
  PageTile<D> page;
  page.dma.init(tid);
  page.table = a.table + (int64_t)at.r * a.max_pages;
  page.end = at.base + at.n;
  page.h = h;

  floatx16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = splat16(0.f);
  floatx4 lsum = floatx4{0.f, 0.f, 0.f, 0.f};
  // row sums on the matrix pipe: lane l gets that of row l & 31 of the operand of 32 rows
  const uint4 ones = ((lane >> 2) & 1) == ((lane >> 4) & 1) ? T::ones8() : make_uint4(0, 0, 0, 0);
  const float slack = kSlack / a.scale_log2;
  float nm = 0.f, thr = kNegInf;

  if (keys.n > 0) {
    page.load(a, a.k_pages, keys.first_key(0), sk[0]);
    page.load(a, a.v_pages, keys.first_key(0), sv[0]);
  }
  dma_wait();
  __syncthreads();
  auto step = [&](int i, int buf) {
    const int x0 = keys.first_key(i);
    if (i + 1 < keys.n) {
      page.load(a, a.k_pages, keys.first_key(i + 1), sk[buf ^ 1]);
      page.load(a, a.v_pages, keys.first_key(i + 1), sv[buf ^ 1]);
    }
    floatx16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[t] = T::mfma32(lanes.rows(sk[buf], t, ks), qf[ks], ks == 0 ? splat16(0.f) : s[t]);
    const uint64_t bits = mine ? seen_bits(a, token, pos, at.base, x0) : 0;
    float mx = kNegInf;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const LaneBits32 vis((uint32_t)(bits >> (32 * t)), hi);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = vis.pick(r, s[t][r], kNegInf);
        mx = fmaxf(mx, s[t][r]);
      }
    }
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
    uint4 p[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], a.scale_log2, nm));
      p[2 * t] = pack8<T>(s[t], 0);
      p[2 * t + 1] = pack8<T>(s[t], 1);
    }
#pragma unroll
    for (int st = 0; st < 4; ++st) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma32(lanes.cols(sv[buf], st, dt), p[st], o[dt]);
      lsum = T::mfma(ones, p[st], lsum);
    }
    dma_wait();
    __syncthreads();
  };
  int i = 0;
  for (; i + 1 < keys.n; i += 2) {
    step(i, 0);
    step(i + 1, 1);
  }
  if (i < keys.n) step(i, 0);

  if (!mine) return;
  const float l = lsum[0], inv = l > 0.f ? 1.f / l : 1.f;
  uint16_t* dst = a.o + ((int64_t)token * a.H + head) * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(uint2*)(dst + 32 * dt + 8 * r + 4 * hi) =
          make_uint2(pack2<T>(o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv), pack2<T>(o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv));
  if (hi == 0 && a.lse) a.lse[(int64_t)token * a.H + head] = l > 0.f ? lse_natural(-nm, l) : 0.f;
}

}  // namespace

// `tiles`: an upper bound of the requests' row tiles.
int paged_attend_dispatch(int dtype, int head_dim, const PagedArgs& a, hipStream_t stream) {
  const int64_t tiles = (int64_t)a.rows * a.group / kTile + std::min(a.R, a.rows);
  const dim3 grid((unsigned)tiles, (unsigned)a.H_kv);
#define GKI_PAGED(T, D) hipLaunchKernelGGL((paged_tiles_kernel<T, D>), grid, dim3(256), 0, stream, a)
  if (dtype == kF16) {
    if (head_dim == 64) GKI_PAGED(F16, 64);
    else GKI_PAGED(F16, 128);
  } else if (head_dim == 64) GKI_PAGED(BF16, 64);
  else GKI_PAGED(BF16, 128);
#undef GKI_PAGED
  return check_launch("gki_paged_attend");
}

}  // namespace gki

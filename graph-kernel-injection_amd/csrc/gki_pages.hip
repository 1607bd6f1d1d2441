// Page tables of requests, built on the GPU, and the rows that go to pages.
//
// A request's position p lies in its page p / page_size (a power of two), which the pool
// holds as [num_pages][H_kv][page_size][D]. Free pages are a queue (a ring of num_pages
// ids): pages are taken from its head and come back at its end, both in the order of
// requests and positions, so that the same calls give the same tables. A page that no
// later query of a request can see (behind its window, no sinks in it) goes back when the
// request is extended: a request holds O(sinks + window) pages however long it gets.
#include "gki_rotary.cuh"

namespace gki {
namespace {

constexpr int kBookThreads = 1024;
// Rows that the book-keeping workgroup places itself; more have a launch of their own. extend and
// accept of 64 requests, us, placed by it / by a launch: 1024 rows 7.3 / 9.2, 4096 9.7 / 9.4, 8192
// 12.7 / 9.3, 16384 19.2 / 9.4.
constexpr int kBookRows = 4096;
constexpr int kMaxDraft = 256;

enum Refusal : int { kOutOfPages = 1, kTooManyRows = 2, kBadCount = 4 };

// Exclusive prefix of x over the workgroup, and the total; `part` holds one sum per wave.
__device__ inline int block_scan(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = (int)wave_prefix((uint32_t)x);
  __syncthreads();                     // `part` of the scan before has been read
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kBookThreads / 64; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + s - x;
}

// Adds the lanes' x to a sum in LDS: its low 15 bits and the rest apart, as 64 of these fit.
__device__ inline void add_to(unsigned long long* sum, uint32_t x) {
  const uint32_t lo = wave_prefix(x & 0x7FFF), hi = wave_prefix(x >> 15);
  if ((threadIdx.x & 63) == 63 && (lo | hi)) atomicAdd(sum, ((unsigned long long)hi << 15) + lo);
}

// The last r of 0 .. n - 1 with start[r] <= i (start ascending, start[0] <= i): where
// several requests start at i (empty ones), the one that holds it.
__device__ inline int locate(const int32_t* start, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ inline int sink_pages(const PageTables& t) { return (int)(((int64_t)t.sink + (1 << t.shift) - 1) >> t.shift); }

// What a request's step takes: the first page that is kept after it, and pages to add.
struct Need {
  int kept, pages;
  __device__ inline Need(const PageTables& t, int r, int count) {
    const int len = t.lengths[r];
    kept = t.kept[r];
    pages = t.pages[r];
    if (count > 0) {
      // the next token sees positions above len - window; its own page stays
      const int64_t oldest = max((int64_t)0, (int64_t)len - t.window + 1);
      kept = max(kept, (int)(min(oldest, (int64_t)len) >> t.shift));
      pages = max(pages, (len + count + (1 << t.shift) - 1) >> t.shift);
    }
  }
};

// Slot and position of a row that is number i of request r's.
__device__ inline void place_row(const PageTables& t, const PageStep& s, int row, int r, int i) {
  const int x = s.base[r] + i;
  s.slots[row] = ((int64_t)t.table[(int64_t)r * t.max_pages + (x >> t.shift)] << t.shift) + (x & ((1 << t.shift) - 1));
  s.positions[row] = x;
}
__device__ inline void no_row(const PageStep& s, int row) {
  s.slots[row] = -1;
  s.positions[row] = 0;
}

// One workgroup: checks the step, gives pages back, takes pages, and (PLACE) places the
// rows. A step that does not fit changes nothing and leaves no rows. Bound by latency (three
// passes over the requests, flat loops over pages and rows): 5.3 us for 8 requests, 6.1 for 512.
// One workgroup, since pages are given out in order; sums and prefixes by DPP (8.8 -> 5.6 us).
template <bool PLACE>
__global__ __launch_bounds__(kBookThreads) void extend_kernel(PageTables t, PageStep s) {
  __shared__ int part[kBookThreads / 64];
  __shared__ int first[kBookThreads], from[kBookThreads], starts[kBookThreads];
  __shared__ unsigned long long sums[3];
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid < 3) sums[tid] = 0;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int head = t.queue[0], count = t.queue[1];
  for (int r0 = 0; r0 < t.R; r0 += kBookThreads) {
    const int r = r0 + tid;
    int c = 0, new_pages = 0, dead = 0;
    if (r < t.R) {
      c = s.counts[r];
      if (c < 0 || c > s.max_count || (int64_t)t.lengths[r] + c > ((int64_t)t.max_pages << t.shift)) {
        bad = 1;
        c = 0;
      }
      const Need n(t, r, c);
      new_pages = n.pages - t.pages[r];
      dead = n.kept - t.kept[r];
    }
    add_to(&sums[0], c);
    add_to(&sums[1], new_pages);
    add_to(&sums[2], dead);
  }
  __syncthreads();
  const int why = bad ? kBadCount : (sums[0] > (unsigned long long)s.rows ? kTooManyRows : 0) |
                                        (sums[1] > (unsigned long long)count + sums[2] ? kOutOfPages : 0);
  if (why) {
    if (tid == 0) {
      *t.status |= why;
      s.requests[0] = make_int4(0, 0, 0, 0);
    }
    for (int r = tid; r <= t.R; r += kBookThreads) {
      s.row_starts[r] = 0;
      if (r < t.R) s.base[r] = t.lengths[r];
    }
    if constexpr (PLACE)
      for (int row = tid; row < s.rows; row += kBookThreads) no_row(s, row);
    return;
  }
  // pages that go back
  int given = 0;
  if (sums[2]) {
    for (int r0 = 0; r0 < t.R; r0 += kBookThreads) {
      const int r = r0 + tid, kept = r < t.R ? t.kept[r] : 0;
      const int next = r < t.R ? Need(t, r, s.counts[r]).kept : 0;
      int total;
      first[tid] = block_scan(next - kept, part, total);
      from[tid] = kept;
      if (r < t.R) t.kept[r] = next;
      __syncthreads();
      for (int i = tid; i < total; i += kBookThreads) {
        const int x = locate(first, kBookThreads, i);
        int32_t* e = t.table + (int64_t)(r0 + x) * t.max_pages + from[x] + (i - first[x]);
        t.ring[((int64_t)head + count + given + i) % t.num_pages] = *e;
        *e = -1;
      }
      given += total;
      __syncthreads();
    }
  }
  // pages that are taken, the rows' starts, lengths
  int taken = 0, rows = 0, active = 0;
  for (int r0 = 0; r0 < t.R; r0 += kBookThreads) {
    const int r = r0 + tid, c = r < t.R ? s.counts[r] : 0;
    const int had = r < t.R ? t.pages[r] : 0, len = r < t.R ? t.lengths[r] : 0;
    const int pages = r < t.R && c > 0 ? max(had, (len + c + (1 << t.shift) - 1) >> t.shift) : had;
    int total_rows, total;
    const int start = rows + block_scan(c, part, total_rows);
    int total_active;
    const int place = active + block_scan(c > 0 ? 1 : 0, part, total_active);
    if (c > 0) s.requests[1 + place] = make_int4(r, start, c, len);
    active += total_active;
    first[tid] = block_scan(pages - had, part, total);
    from[tid] = had;
    starts[tid] = start;
    if (r < t.R) {
      s.row_starts[r] = start;
      s.base[r] = len;
      t.lengths[r] = len + c;
      t.pages[r] = pages;
    }
    __syncthreads();
    for (int i = tid; i < total; i += kBookThreads) {
      const int x = locate(first, kBookThreads, i);
      t.table[(int64_t)(r0 + x) * t.max_pages + from[x] + (i - first[x])] = t.ring[((int64_t)head + taken + i) % t.num_pages];
    }
    taken += total;
    rows += total_rows;
    __syncthreads();
  }
  if (tid == 0) {
    s.row_starts[t.R] = rows;
    s.requests[0] = make_int4(active, rows, 0, 0);
    t.queue[0] = (int)(((int64_t)head + taken) % t.num_pages);
    t.queue[1] = count + given - taken;
  }
  if constexpr (PLACE) {
    __syncthreads();
    for (int row = tid; row < s.rows; row += kBookThreads) {
      if (row >= rows) {
        no_row(s, row);
        continue;
      }
      // the starts of up to a workgroup's threads are in LDS
      const bool held = t.R <= kBookThreads;
      const int r = held ? locate(starts, t.R, row) : locate(s.row_starts, t.R, row);
      place_row(t, s, row, r, row - (held ? starts[r] : s.row_starts[r]));
    }
  }
}

// The rows of a step, by a thread each.
__global__ __launch_bounds__(256) void place_kernel(PageTables t, PageStep s) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= s.rows) return;
  if (row >= s.row_starts[t.R]) {
    no_row(s, row);
    return;
  }
  const int r = locate(s.row_starts, t.R, row);
  place_row(t, s, row, r, row - s.row_starts[r]);
}

// The nodes of a request's tree, by a thread each: node i stands at position base + depth
// and sees its ancestors and itself where these are sinks or in its window. A parent that
// is not an earlier node counts as none. The last workgroup writes the rows behind the
// trees.
__global__ __launch_bounds__(kMaxDraft) void tree_kernel(PageTables t, PageStep s) {
  __shared__ int up[kMaxDraft];
  const int r = blockIdx.x, i = threadIdx.x;
  if (r == t.R) {
    for (int row = s.row_starts[t.R] + i; row < s.rows; row += kMaxDraft) {
      no_row(s, row);
      for (int w = 0; w < s.words; ++w) s.ancestors[(int64_t)row * s.words + w] = 0;
    }
    return;
  }
  const int row0 = s.row_starts[r], n = s.row_starts[r + 1] - row0;      // at most max_count <= kMaxDraft
  if (i < n) {
    const int p = s.parents[row0 + i];
    up[i] = p >= 0 && p < i ? p : -1;
  }
  __syncthreads();
  if (i >= n) return;
  int depth = 0;
  for (int j = up[i]; j >= 0; j = up[j]) ++depth;
  const int base = s.base[r];
  uint64_t bits[kMaxDraft / 64] = {0, 0, 0, 0};
  for (int j = i, d = depth; j >= 0; j = up[j], --d) {
    const uint64_t bit = base + d < t.sink || depth - d < t.window ? 1ull << (j & 63) : 0;
#pragma unroll
    for (int w = 0; w < kMaxDraft / 64; ++w) bits[w] |= (j >> 6) == w ? bit : 0;
  }
  place_row(t, s, row0 + i, r, i);
  s.positions[row0 + i] = base + depth;
#pragma unroll
  for (int w = 0; w < kMaxDraft / 64; ++w)
    if (w < s.words) s.ancestors[(int64_t)(row0 + i) * s.words + w] = bits[w];
}

// Requests marked in `done` give all their pages back and hold nothing.
__global__ __launch_bounds__(kBookThreads) void release_kernel(PageTables t, const uint8_t* done) {
  __shared__ int part[kBookThreads / 64];
  __shared__ int first[kBookThreads], skip[kBookThreads];
  const int tid = threadIdx.x, head = t.queue[0], count = t.queue[1], n_sink = sink_pages(t);
  int given = 0;
  for (int r0 = 0; r0 < t.R; r0 += kBookThreads) {
    const int r = r0 + tid;
    const bool go = r < t.R && done[r];
    const int pages = go ? t.pages[r] : 0, kept = go ? t.kept[r] : 0;
    int total;
    first[tid] = block_scan(min(pages, n_sink) + max(0, pages - kept), part, total);
    skip[tid] = kept - n_sink;                 // pages behind the sinks that are gone already
    if (go) {
      t.lengths[r] = 0;
      t.pages[r] = 0;
      t.kept[r] = n_sink;
    }
    __syncthreads();
    for (int i = tid; i < total; i += kBookThreads) {
      const int x = locate(first, kBookThreads, i), j = i - first[x];
      int32_t* e = t.table + (int64_t)(r0 + x) * t.max_pages + (j < n_sink ? j : j + skip[x]);
      t.ring[((int64_t)head + count + given + i) % t.num_pages] = *e;
      *e = -1;
    }
    given += total;
    __syncthreads();
  }
  if (tid == 0) t.queue[1] = count + given;
}

// lengths = base + what is accepted of the step's tokens, if less than they are: a request
// that was released since holds no pages, and must not be long again.
__global__ __launch_bounds__(256) void accept_kernel(int32_t* lengths, const int32_t* base, const int32_t* row_starts,
                                                     const int32_t* accepted, int R) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= R) return;
  const int n = row_starts[r + 1] - row_starts[r];
  if (n > 0) lengths[r] = min(lengths[r], base[r] + max(0, min(accepted[r], n)));
}

// ---------------------------------------------------------------------------
// Rows into pages.
// ---------------------------------------------------------------------------
// D / 8 lanes per head of a row; rows without a slot are left out. Bound by HBM, small steps by
// latency: 3.8 k rows of 16 heads (D64, 32 MB both ways) 6.8 us, 8 of 8 heads 1.8.
template <int D>
__global__ __launch_bounds__(256) void append_kernel(PageRows p) {
  constexpr int LPR = D / 8;
  const int ch = threadIdx.x % LPR;
  const int64_t n = (int64_t)p.rows * p.H_kv;
  for (int64_t x = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR; x < 2 * n; x += (int64_t)gridDim.x * (256 / LPR)) {
    const bool is_v = x >= n;
    const int64_t y = is_v ? x - n : x;
    const int row = (int)(y / p.H_kv), h = (int)(y % p.H_kv);
    const int64_t slot = p.slots[row];
    if (slot < 0 || slot >= p.n_slots) continue;
    const uint16_t* src = (const uint16_t*)(is_v ? p.v : p.k) + (int64_t)row * (is_v ? p.v_stride : p.k_stride) + h * D;
    *(uint4*)((uint16_t*)(is_v ? p.v_pages : p.k_pages) + p.at(slot, h, D) + 8 * ch) = *(const uint4*)(src + 8 * ch);
  }
}

// The same with the keys turned by their positions, and the queries turned into q_out
// ([rows][H][D]), also those of rows without a slot: a workgroup per row, whose cosines and sines are
// made once for all heads (rotary_turn). Turned rows are rounded once, to T. Bound by HBM, small
// steps by latency: 1.7 k rows of 32 + 2 * 8 heads (D128, 43 MB both ways) 9.2 us, 32 rows 4.0;
// apart, the turn and the append are two launches, and the keys are read twice.
template <typename T, int D>
__global__ __launch_bounds__(256) void append_rotated_kernel(PageRows p, RotaryArgs a, HeadRows q) {
  __shared__ float2 cs[64];
  const int row = blockIdx.x;
  for (int j = threadIdx.x; j < a.pairs; j += 256) cs[j] = rotary_turn(a, row, j);
  const int64_t slot = p.slots[row];
  const bool placed = slot >= 0 && slot < p.n_slots;
  __syncthreads();
  auto turn = [&](int i, const uint16_t* src, uint16_t* dst) {
    if (a.interleaved) rotary_item<T, true>(a, cs, i, src, dst);
    else rotary_item<T, false>(a, cs, i, src, dst);
  };
  const int per_row = a.interleaved ? rotary_items<T, true>(a.pairs, D) : rotary_items<T, false>(a.pairs, D);
  const uint16_t* k = (const uint16_t*)p.k + (int64_t)row * p.k_stride;
  const uint16_t* v = (const uint16_t*)p.v + (int64_t)row * p.v_stride;
  for (int x = threadIdx.x; x < (q.heads + p.H_kv) * per_row; x += 256) {
    const int hh = x / per_row, i = x % per_row, h = hh - q.heads;
    if (h < 0)
      turn(i, (const uint16_t*)q.src + (int64_t)row * q.sn + hh * q.sh, (uint16_t*)q.dst + (int64_t)row * q.dn + hh * q.dh);
    else if (placed) turn(i, k + h * D, (uint16_t*)p.k_pages + p.at(slot, h, D));
  }
  if (placed)
    for (int x = threadIdx.x; x < p.H_kv * (D / 8); x += 256) {
      const int h = x / (D / 8), c = 8 * (x % (D / 8));
      *(uint4*)((uint16_t*)p.v_pages + p.at(slot, h, D) + c) = *(const uint4*)(v + h * D + c);
    }
}

// Rows of each request's accepted path to the slots of its first tokens. Node i of a path is
// number path[i] > i of the request's rows, or moves nothing. A thread has 16 bytes of every
// row of a (request, head): it reads eight rows before it writes them, and what a later one
// reads has a higher number than all that were written. Bound by latency (paths, slots, rows, one
// after the other): 16 requests' paths of up to 26 nodes, 8 heads 5.4 us (a row at a time 9.6).
template <int D>
__global__ __launch_bounds__(256) void move_kernel(PageRows p, const int32_t* row_starts, const int32_t* paths,
                                                   const int32_t* accepted, int R, int path_len) {
  constexpr int LPR = D / 8, N = 8;
  const int64_t x = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int ch = threadIdx.x % LPR;
  if (x >= 2ll * R * p.H_kv) return;
  const bool is_v = x >= (int64_t)R * p.H_kv;
  const int64_t y = is_v ? x - (int64_t)R * p.H_kv : x;
  const int r = (int)(y / p.H_kv), h = (int)(y % p.H_kv);
  const int row0 = row_starts[r], n = row_starts[r + 1] - row0;
  const int last = min(min(accepted[r], n), path_len);
  uint16_t* pool = (uint16_t*)(is_v ? p.v_pages : p.k_pages) + 8 * ch;
  for (int i0 = 0; i0 < last; i0 += N) {
    int node[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      node[e] = paths[(int64_t)r * path_len + min(i0 + e, last - 1)];
      if (i0 + e >= last || node[e] <= i0 + e || node[e] >= n) node[e] = -1;
    }
    int64_t from[N], to[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      from[e] = p.slots[row0 + max(node[e], 0)];
      to[e] = p.slots[row0 + min(i0 + e, last - 1)];
      if (from[e] < 0 || from[e] >= p.n_slots || to[e] < 0 || to[e] >= p.n_slots) node[e] = -1;
    }
    u32x4 w[N];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = *(const u32x4*)(pool + (node[e] < 0 ? 0 : p.at(from[e], h, D)));
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (node[e] >= 0) *(u32x4*)(pool + p.at(to[e], h, D)) = w[e];
  }
}

inline dim3 lanes_grid(int64_t lanes) { return dim3((unsigned)std::min<int64_t>((lanes + 255) / 256, 1 << 20)); }

}  // namespace

int page_extend_dispatch(const PageTables& t, const PageStep& s, hipStream_t stream) {
  const bool place = s.parents == nullptr && s.rows <= kBookRows;
  if (place) hipLaunchKernelGGL(extend_kernel<true>, dim3(1), dim3(kBookThreads), 0, stream, t, s);
  else hipLaunchKernelGGL(extend_kernel<false>, dim3(1), dim3(kBookThreads), 0, stream, t, s);
  if (s.parents) hipLaunchKernelGGL(tree_kernel, dim3(t.R + 1), dim3(kMaxDraft), 0, stream, t, s);
  else if (!place) hipLaunchKernelGGL(place_kernel, dim3((s.rows + 255) / 256), dim3(256), 0, stream, t, s);
  return check_launch("gki_page_extend");
}

int page_release_dispatch(const PageTables& t, const uint8_t* done, hipStream_t stream) {
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kBookThreads), 0, stream, t, done);
  return check_launch("gki_page_release");
}

int page_accept_dispatch(int32_t* lengths, const int32_t* base, const int32_t* row_starts, const int32_t* accepted,
                         int R, hipStream_t stream) {
  hipLaunchKernelGGL(accept_kernel, dim3((R + 255) / 256), dim3(256), 0, stream, lengths, base, row_starts, accepted, R);
  return check_launch("gki_page_accept");
}

int paged_append_dispatch(int head_dim, const PageRows& p, hipStream_t stream) {
  const dim3 grid = lanes_grid(2ll * p.rows * p.H_kv * (head_dim / 8));
  if (head_dim == 64) hipLaunchKernelGGL(append_kernel<64>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(append_kernel<128>, grid, dim3(256), 0, stream, p);
  return check_launch("gki_paged_append");
}

int paged_append_rotated_dispatch(int dtype, int head_dim, const PageRows& p, const RotaryArgs& a, const HeadRows& q,
                                  hipStream_t stream) {
#define GKI_ROT(T, D) hipLaunchKernelGGL((append_rotated_kernel<T, D>), dim3(p.rows), dim3(256), 0, stream, p, a, q)
  if (dtype == kF16) {
    if (head_dim == 64) GKI_ROT(F16, 64);
    else GKI_ROT(F16, 128);
  } else if (head_dim == 64) GKI_ROT(BF16, 64);
  else GKI_ROT(BF16, 128);
#undef GKI_ROT
  return check_launch("gki_paged_append_rotated");
}

int paged_move_dispatch(int head_dim, const PageRows& p, const int32_t* row_starts, const int32_t* paths,
                        const int32_t* accepted, int R, int path_len, hipStream_t stream) {
  const int64_t lanes = 2ll * R * p.H_kv * (head_dim / 8);
  const dim3 grid((unsigned)((lanes + 255) / 256));
  if (head_dim == 64) hipLaunchKernelGGL(move_kernel<64>, grid, dim3(256), 0, stream, p, row_starts, paths, accepted, R, path_len);
  else hipLaunchKernelGGL(move_kernel<128>, grid, dim3(256), 0, stream, p, row_starts, paths, accepted, R, path_len);
  return check_launch("gki_paged_accept");
}

}  // namespace gki

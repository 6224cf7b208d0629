// A cache's pages: shared, copied before a write, freed, compacted, and positions moved.
#include "host_common.h"
#include "decode_common.h"
#include "tf_search.h"

using namespace tfd;
using namespace tfd_host;

namespace {

constexpr int kErrPos = 2, kErrPage = 4, kErrRow = TFD_ERR_ROW_RANGE, kErrNone = TFD_ERR_NO_PAGES;
constexpr int kOne = 1024;                   // threads of the kernels of one block
constexpr int kMaxRows = TFD_PAGES_MAX_ROWS;

// scratch: per page the entries that want it and, as its complement, the lowest of them (zero
// between calls); a list of pages; per entry a decision; per row a copy
struct Scratch {
  int *writers, *first, *list, *entry, *src, *dst, *head;
};
__host__ __device__ inline Scratch scratch_of(const TfdPages& p) {
  Scratch s;
  s.writers = p.scratch;
  s.first = s.writers + p.num_pages;
  s.list = s.first + p.num_pages;
  s.entry = s.list + p.num_pages;
  s.src = s.entry + (int64_t)p.rows * p.max_pages;
  s.dst = s.src + p.rows;
  s.head = s.dst + p.rows;
  return s;
}

__device__ __forceinline__ int pages_for(int64_t positions) {
  return (int)((positions + kPage - 1) / kPage);
}

// Sum of a value over the block's threads before this one, and over all of them.
__device__ __forceinline__ int block_scan(int v, int* wave_s, int& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  if (lane == kWave - 1) wave_s[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
  const int waves = blockDim.x / kWave;
  for (int w = 0; w < waves; ++w) {
    const int y = wave_s[w];
    if (w < wave) before += y;
    all += y;
  }
  __syncthreads();
  total = all;
  return before + x - v;
}

// ---------------------------------------------------------------------------
// Fork and free: a block takes some columns of the table for all rows, so that it may write
// in place what it has read; references change by one for each entry that does.  A launch and two
// rounds of loads: 2.3 us for 16 rows of 45 pages, 4.7 for 24 rows.
// ---------------------------------------------------------------------------
constexpr int kForkCols = 16;

__global__ __launch_bounds__(kBlock) void k_pages_fork(TfdPages p, const int* __restrict__ parents,
                                                       const uint8_t* __restrict__ which,
                                                       const int* __restrict__ lengths,
                                                       int* __restrict__ lengths_out) {
  extern __shared__ int old_s[];             // [rows][kForkCols]
  const int tid = threadIdx.x, c0 = blockIdx.x * kForkCols, items = p.rows * kForkCols;
  for (int i = tid; i < items; i += kBlock) {
    const int c = c0 + i % kForkCols;
    old_s[i] = c < p.max_pages ? p.table[(int64_t)(i / kForkCols) * p.max_pages + c] : -1;
  }
  __syncthreads();
  for (int i = tid; i < items; i += kBlock) {
    const int r = i / kForkCols, c = c0 + i % kForkCols;
    int from = parents ? parents[r] : which[r] ? -1 : r;
    if (from < -1 || from >= p.rows) {
      if (c == c0) raise_error(p.err, kErrRow);
      from = r;
    }
    const int len = parents && from >= 0 ? lengths[from] : 0;
    if (c == 0 && parents) lengths_out[r] = len;
    if (c >= p.max_pages) continue;
    const int was = old_s[i];
    int now = -1;
    if (from == r) now = was;
    else if (from >= 0 && c < pages_for(len)) now = old_s[from * kForkCols + i % kForkCols];
    if (now == was) continue;
    if (was >= 0 && was < p.num_pages) atomicSub(&p.refs[was], 1);
    if (now >= 0 && now < p.num_pages) atomicAdd(&p.refs[now], 1);
    p.table[(int64_t)r * p.max_pages + c] = now;
  }
}

// ---------------------------------------------------------------------------
// Take, in one block: every step is a few thousand entries at most, and their order (rows,
// then positions) has to hold.  An entry's decision waits for all entries' counts, and the
// table changes after all have decided.  Bound by latency, eight barriers and five rounds of
// loads: 7.5 us for a position of each of 16 rows, 8.2 for all pages of 24 rows of 611.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kOne) void k_pages_take(TfdPages p, const int* __restrict__ lengths,
                                                     const int* __restrict__ counts, int n_all) {
  __shared__ int wave_s[kOne / kWave];
  __shared__ int start_s[kMaxRows + 1], page0_s[kMaxRows];
  const Scratch s = scratch_of(p);
  const int tid = threadIdx.x;
  // the wanted entries of each row
  int want = 0;
  if (tid < p.rows) {
    const int len = lengths[tid];
    const int64_t n = counts ? counts[tid] : n_all;
    int first = 0;
    if (len < 0) raise_error(p.err, kErrPos);
    else if (n > 0) {
      first = len / kPage;
      int64_t last = (len + n + kPage - 1) / kPage;
      if (last > p.max_pages) {
        raise_error(p.err, kErrPos);
        last = p.max_pages;
      }
      want = last > first ? (int)(last - first) : 0;
    }
    page0_s[tid] = first;
    s.src[tid] = -1;
  }
  int total;
  const int before = block_scan(want, wave_s, total);
  if (tid < p.rows) start_s[tid] = before;
  if (tid == 0) start_s[p.rows] = total;
  __syncthreads();
  auto row_of = [&](int e) {                 // the row whose entries hold e
    int lo = 0, hi = p.rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (start_s[mid] <= e) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto at_of = [&](int e, int r) { return r * (int64_t)p.max_pages + page0_s[r] + e - start_s[r]; };
  // who wants the shared pages
  for (int e = tid; e < total; e += kOne) {
    const int r = row_of(e);
    const int64_t at = at_of(e, r);
    const int page = p.table[at];
    if (page >= 0 && page < p.num_pages && p.refs[page] > 1) {
      atomicAdd(&s.writers[page], 1);
      atomicMax(&s.first[page], 0x7fffffff - e);   // the lowest entry
    }
  }
  // the lowest free pages, as many as could be wanted
  int free_pages = 0;
  for (int i0 = 0; i0 < p.num_pages && free_pages < total; i0 += 4 * kOne) {
    int v[4];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 4 * tid + j;
      v[j] = i < p.num_pages ? p.refs[i] : 1;
      mine += v[j] == 0;
    }
    int found;
    int rank = free_pages + block_scan(mine, wave_s, found);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v[j] == 0) s.list[rank++] = i0 + 4 * tid + j;
    free_pages += found;
  }
  __syncthreads();
  // decisions: -2 the entry stays, -1 no page was left, else its new page
  int taken = 0;
  for (int e0 = 0; e0 < total; e0 += kOne) {
    const int e = e0 + tid;
    int fresh = 0;
    if (e < total) {
      const int page = p.table[at_of(e, row_of(e))];
      if (page < 0 || page >= p.num_pages) fresh = 1;
      else {
        const int refs = p.refs[page];
        // (counted by atomics: read where those are)
        fresh = refs > 1 && !(coh_ldi(&s.writers[page]) == refs &&
                              coh_ldi(&s.first[page]) == 0x7fffffff - e);
      }
    }
    int found;
    const int rank = taken + block_scan(fresh, wave_s, found);
    if (e < total) s.entry[e] = !fresh ? -2 : rank < free_pages ? s.list[rank] : -1;
    taken += found;
  }
  if (tid == 0 && taken > free_pages) raise_error(p.err, kErrNone);
  __syncthreads();
  for (int e = tid; e < total; e += kOne) {
    const int r = row_of(e);
    const int64_t at = at_of(e, r);
    const int page = p.table[at], now = s.entry[e];
    const bool held = page >= 0 && page < p.num_pages;
    if (!held && page != -1) raise_error(p.err, kErrPage);
    if (held) s.writers[page] = 0, s.first[page] = 0;
    if (now == -2) continue;
    if (held) {
      atomicSub(&p.refs[page], 1);
      if (e == start_s[r] && lengths[r] % kPage && now >= 0) {
        s.src[r] = page;
        s.dst[r] = now;
      }
    }
    if (now >= 0) atomicAdd(&p.refs[now], 1);
    p.table[at] = now;
  }
}

// ---------------------------------------------------------------------------
// Copies: a block takes 32 KiB of one page of one pool at a time, all its loads before its
// stores; the blocks walk the items, whose number (of pairs) may lie on the device.  kHoles: -1
// in src is a place without a copy (take's list, a place for every row).  Bound by memory: 1.6 GB
// in 310 us, 5.1 TB/s; a page of each of 8 rows 4.4 us.
// ---------------------------------------------------------------------------
constexpr int kCopyLoads = 8;
constexpr int64_t kCopyBytes = kBlock * 16 * kCopyLoads;

template <bool kHoles>
__global__ __launch_bounds__(kBlock) void k_pages_copy(TfdPages p, const int* __restrict__ src,
                                                       const int* __restrict__ dst, int n,
                                                       const int* __restrict__ n_dev,
                                                       int pieces) {
  if (n_dev) n = min(n, *n_dev);
  const uint32_t per = (uint32_t)p.n_pools * pieces, items = n * per;
#pragma unroll 1
  for (uint32_t it = blockIdx.x; it < items; it += gridDim.x) {
    const uint32_t pair = it / per, pool = it % per / pieces, piece = it % pieces;
    const int a = src[pair];
    if (kHoles && a == -1) continue;
    const int b = dst[pair];
    if (a < 0 || a >= p.num_pages || b < 0 || b >= p.num_pages) {
      if (threadIdx.x == 0) raise_error(p.err, kErrPage);
      continue;
    }
    const TfdPool t = p.pools[pool];
    const uint8_t* from = (const uint8_t*)t.base + a * t.page_bytes;
    uint8_t* to = (uint8_t*)t.base + b * t.page_bytes;
    const int64_t at0 = piece * kCopyBytes + threadIdx.x * 16;
    u32x4 v[kCopyLoads];
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
      v[i] = *(g_u32x4*)(from + min(at0 + i * kBlock * 16, t.page_bytes - 16));
    }
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
      const int64_t at = at0 + i * kBlock * 16;
      if (at < t.page_bytes) *reinterpret_cast<u32x4*>(to + at) = v[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Keep: a thread takes 16 bytes of a head's positions along the path, in order.  The path
// rises, so what a position moves to lies before everything that is still to be read.  Rounds of
// loads (path, pages, values) bound it: 10 us for 32 rows of 28 layers, 2.2 TB/s.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kBlock) void k_pages_keep(TfdPages p, const int* __restrict__ lengths,
                                                       const int* __restrict__ path,
                                                       const int* __restrict__ counts, int nodes,
                                                       int* __restrict__ lengths_out) {
  const int row = blockIdx.x, len = lengths[row], n = counts[row], tid = threadIdx.x;
  const int64_t room = (int64_t)p.max_pages * kPage;
  const int* const way = path + (int64_t)row * nodes;
  bool bad = n < 0 || n > nodes, far = len < 0;
  for (int i = tid; !bad && !far && i < n; i += kBlock) {
    const int t = way[i];
    bad |= t < i || t >= nodes || (i > 0 && t <= way[i - 1]);
    far |= (int64_t)len + t >= room;
  }
  const bool any_bad = __syncthreads_or(bad), any_far = __syncthreads_or(far);
  if (blockIdx.y == 0 && tid == 0) {
    if (any_bad) raise_error(p.err, kErrRow);
    if (any_far) raise_error(p.err, kErrPos);
    lengths_out[row] = any_bad || any_far ? len : len + n;
  }
  if (any_bad || any_far) return;
  const TfdPool t = p.pools[blockIdx.y];
  const int per = t.row_bytes / 16;          // columns of a head
  const int* const table = p.table + (int64_t)row * p.max_pages;
  auto place = [&](int pos, int h, int c) -> uint8_t* {
    const int page = table[pos / kPage];
    if (page < 0 || page >= p.num_pages) {
      raise_error(p.err, kErrPage);
      return nullptr;
    }
    return (uint8_t*)t.base + page * t.page_bytes +
           ((int64_t)h * kPage + pos % kPage) * t.row_bytes + c * 16;
  };
  for (int i = tid; i < t.heads * per; i += kBlock) {
    const int h = i / per, c = i % per;
    constexpr int kMoves = 4;
    for (int k0 = 0; k0 < n; k0 += kMoves) {
      u32x4 v[kMoves];
      uint8_t* to[kMoves];
#pragma unroll
      for (int k = 0; k < kMoves; ++k) {
        to[k] = nullptr;
        if (k0 + k >= n) continue;
        const int f = way[k0 + k];
        if (f == k0 + k) continue;
        const uint8_t* from = place(len + f, h, c);
        if (from) {
          v[k] = *(g_u32x4*)from;
          to[k] = place(len + k0 + k, h, c);
        }
      }
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if (to[k]) *reinterpret_cast<u32x4*>(to[k]) = v[k];
    }
  }
}

// ---------------------------------------------------------------------------
// Compact: one block pairs the pages in use from `live` on with the free ones below; the
// copies follow, and then the table's entries and the references (6.8, 4.7 and 4.8 us beside
// the copies' 310 of 24 rows of 28 layers).  writers holds the moved
// pages' new numbers, plus one, until the last launch, which leaves zeros.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kOne) void k_pages_pair(TfdPages p, int* __restrict__ live) {
  __shared__ int wave_s[kOne / kWave];
  const Scratch s = scratch_of(p);
  const int tid = threadIdx.x;
  int used = 0;
  for (int i = tid; i < p.num_pages; i += kOne) used += p.refs[i] > 0;
  int n;
  block_scan(used, wave_s, n);
  // holes: list from the front; movers: first from the front (both ordered)
  int holes = 0, movers = 0;
  for (int i0 = 0; i0 < p.num_pages; i0 += kOne) {
    const int i = i0 + tid;
    const bool in = i < p.num_pages && p.refs[i] > 0;
    const bool hole = i < n && !in, move = i >= n && in;
    int found;
    const int rank = block_scan(hole ? 1 : 0, wave_s, found);
    if (hole) s.list[holes + rank] = i;
    holes += found;
    const int rank2 = block_scan(move ? 1 : 0, wave_s, found);
    if (move) s.first[movers + rank2] = i;
    movers += found;
  }
  __syncthreads();
  for (int k = tid; k < movers; k += kOne) s.writers[s.first[k]] = s.list[k] + 1;
  if (tid == 0) {
    *s.head = movers;
    if (live) *live = n;
  }
}

__global__ __launch_bounds__(kBlock) void k_pages_rename(TfdPages p) {
  const Scratch s = scratch_of(p);
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i < (int64_t)p.rows * p.max_pages) {
    const int page = p.table[i];
    if (page >= 0 && page < p.num_pages) {
      const int now = s.writers[page];
      if (now) p.table[i] = now - 1;
    }
  }
}

__global__ __launch_bounds__(kBlock) void k_pages_settle(TfdPages p) {
  const Scratch s = scratch_of(p);
  const int k = blockIdx.x * kBlock + threadIdx.x;
  if (k >= *s.head) return;
  const int from = s.first[k], to = s.list[k];
  p.refs[to] = p.refs[from];
  p.refs[from] = 0;
  s.writers[from] = 0;
  s.first[k] = 0;
}

int check_pages(const TfdPages* p, const char* what) {
  if (!p) return fail(kBadArg, "%s: null args", what);
  if (p->rows < 1 || p->rows > kMaxRows || p->max_pages < 1 || p->num_pages < 1 ||
      p->max_pages > (1 << 22) || (int64_t)p->rows * p->max_pages > (1 << 30) || p->n_pools < 0 ||
      p->n_pools > 65535 || p->max_page_bytes < 0)
    return fail(kBadShape, "%s: rows=%d (1..%d) max_pages=%d num_pages=%d pools=%d", what, p->rows,
                kMaxRows, p->max_pages, p->num_pages, p->n_pools);
  if (!p->table || !p->refs || !p->scratch || (p->n_pools && !p->pools))
    return fail(kBadArg, "%s: null pointer", what);
  return 0;
}

// Blocks of a walk over `items`: enough to fill the chip a few times over.
unsigned walk_blocks(int64_t items) {
  const int64_t most = 16 * (int64_t)compute_units();
  return (unsigned)(items < most ? items < 1 ? 1 : items : most);
}

int64_t copy_pieces(const TfdPages& p) { return (p.max_page_bytes + kCopyBytes - 1) / kCopyBytes; }

// Refused before a call's first launch: what a call has decided it also copies.
int check_copies(const TfdPages& p, int n) {
  const int64_t pieces = copy_pieces(p);
  if (pieces > (1 << 20) || n * pieces * p.n_pools >= (1ll << 31))
    return fail(kUnsupported, "pages: copies of %d pages of %lld bytes in %d pools in one call", n,
                (long long)p.max_page_bytes, p.n_pools);
  return 0;
}

// Up to n pairs (n_dev: their number on the device) of the lists copied in every pool.
template <bool kHoles>
void copy_pairs(const TfdPages& p, const int* src, const int* dst, int n, const int* n_dev,
                hipStream_t s) {
  if (n == 0 || p.n_pools == 0) return;
  const int64_t pieces = copy_pieces(p);
  k_pages_copy<kHoles><<<walk_blocks(n * pieces * p.n_pools), kBlock, 0, s>>>(p, src, dst, n, n_dev,
                                                                              (int)pieces);
}

}  // namespace

extern "C" {

int tfd_pages_fork(const TfdPages* pages, const int32_t* parents, const uint8_t* which,
                   const int32_t* lengths, int32_t* lengths_out, void* stream) {
  if (const int rc = check_pages(pages, "pages_fork")) return rc;
  if (parents ? !lengths || !lengths_out : !which)
    return fail(kBadArg, "pages_fork: null pointer");
  const TfdPages& p = *pages;
  const int lds = p.rows * kForkCols * 4;    // 64 KiB at most
  k_pages_fork<<<(p.max_pages + kForkCols - 1) / kForkCols, kBlock, lds, (hipStream_t)stream>>>(
      p, parents, which, lengths, lengths_out);
  return launched("pages_fork");
}

int tfd_pages_take(const TfdPages* pages, const int32_t* lengths, const int32_t* counts,
                   int n_all, void* stream) {
  if (const int rc = check_pages(pages, "pages_take")) return rc;
  if (!lengths) return fail(kBadArg, "pages_take: null pointer");
  const TfdPages& p = *pages;
  if (const int rc = check_copies(p, p.rows)) return rc;
  auto s = (hipStream_t)stream;
  k_pages_take<<<1, kOne, 0, s>>>(p, lengths, counts, n_all);
  const Scratch t = scratch_of(p);
  copy_pairs<true>(p, t.src, t.dst, p.rows, nullptr, s);
  return launched("pages_take");
}

int tfd_pages_copy(const TfdPages* pages, const int32_t* src, const int32_t* dst, int n,
                   void* stream) {
  if (const int rc = check_pages(pages, "pages_copy")) return rc;
  if (n < 0) return fail(kBadShape, "pages_copy: n=%d", n);
  const TfdPages& p = *pages;
  if (n == 0 || p.n_pools == 0) return 0;
  if (!src || !dst) return fail(kBadArg, "pages_copy: null pointer");
  if (const int rc = check_copies(p, n)) return rc;
  copy_pairs<false>(p, src, dst, n, nullptr, (hipStream_t)stream);
  return launched("pages_copy");
}

int tfd_pages_keep(const TfdPages* pages, const int32_t* lengths, const int32_t* path,
                   const int32_t* counts, int nodes, int32_t* lengths_out, void* stream) {
  if (const int rc = check_pages(pages, "pages_keep")) return rc;
  if (nodes < 1) return fail(kBadShape, "pages_keep: nodes=%d", nodes);
  if (!lengths || !path || !counts || !lengths_out)
    return fail(kBadArg, "pages_keep: null pointer");
  const TfdPages& p = *pages;
  if (p.n_pools < 1) return fail(kBadShape, "pages_keep: no pools");
  k_pages_keep<<<dim3(p.rows, p.n_pools), kBlock, 0, (hipStream_t)stream>>>(
      p, lengths, path, counts, nodes, lengths_out);
  return launched("pages_keep");
}

int tfd_pages_compact(const TfdPages* pages, int32_t* live, void* stream) {
  if (const int rc = check_pages(pages, "pages_compact")) return rc;
  const TfdPages& p = *pages;
  const int most = (p.num_pages + 1) / 2;    // pairs
  if (const int rc = check_copies(p, most)) return rc;
  const Scratch t = scratch_of(p);
  auto s = (hipStream_t)stream;
  k_pages_pair<<<1, kOne, 0, s>>>(p, live);
  copy_pairs<false>(p, t.first, t.list, most, t.head, s);
  const int64_t entries = (int64_t)p.rows * p.max_pages;
  k_pages_rename<<<(unsigned)((entries + kBlock - 1) / kBlock), kBlock, 0, s>>>(p);
  k_pages_settle<<<(most + kBlock - 1) / kBlock, kBlock, 0, s>>>(p);
  return launched("pages_compact");
}

}  // extern "C"

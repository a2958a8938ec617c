// Pages of a KV cache: rows of a table name pages of a pool, refs counts the rows that name a page.
//
// A page is free while its count is zero.  All but the last page of a row are full, and only full pages are shared:
// a fork copies the partly filled last page, so a row may always write behind its last token.  Pages are given out the
// lowest first, in the order of the request, so that equal requests give equal tables.
//
// The bookkeeping (whole numbers, a few KB to a few hundred KB) is a chain of short phases.  The scans run in one CTA; what goes
// cell by cell (new table rows, places of tokens) runs in the same CTA up to kFewCells cells, which saves a launch, and
// beyond over all SMs: 2048 rows x 40 tokens take 22 us in eight CTAs, most of it waiting for dependent loads.
#pragma once

#include "vk_common.cuh"

namespace vk {
namespace pages {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kFewCells = 4096;

struct Pool {
  int32_t* table;  // [rows, max_pages], -1 behind a row's last page
  int32_t* lens;   // [rows] tokens
  int32_t* refs;   // [n_pages]
  int rows, max_pages, n_pages, page_shift;
};

struct Move {
  int32_t src, dst, tokens;  // tokens 0: nothing to copy
};

// Exclusive prefix sum of one value per thread over the block; *total gets the sum.  All threads of the block call it.
VK_DEV int block_scan(int v, int* total) {
  __shared__ int warp_sums[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const int s = warp_sums[w];
    before += w < warp ? s : 0;
    all += s;
  }
  __syncthreads();  // warp_sums may be written again
  *total = all;
  return before + x - v;
}

constexpr int kPer = 16;  // pages a thread looks at in one step of a scan

// Writes the numbers i of lo .. hi - 1 for which refs[i] > 0 is `used`, in ascending order, through put(place, i) for places
// below `want`; returns how many there are, or some number of at least `want`.  Called by all threads of a block.
template <typename Put>
VK_DEV int scan_pages(const int32_t* refs, int lo, int hi, bool used, int want, Put put) {
  int found = 0;
  for (int64_t base = lo; base < hi && found < want; base += kPlanThreads * kPer) {
    const int64_t first = base + static_cast<int64_t>(threadIdx.x) * kPer;
    uint32_t is = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (first + i < hi && (refs[first + i] > 0) == used) is |= 1u << i;
    int n;
    int at = found + block_scan(__popc(is), &n);
    for (; is; is &= is - 1, ++at)
      if (at < want) put(at, static_cast<int>(first) + __ffs(is) - 1);
    found += n;
  }
  __syncthreads();
  return found;
}

// The lowest `want` free pages into list; returns how many there are (at most want).
VK_DEV int free_pages(const Pool& p, int want, int32_t* list) {
  const int found = scan_pages(p.refs, 0, p.n_pages, false, want, [&](int at, int i) { list[at] = i; });
  return found < want ? found : want;
}

// Which of the items naming row (one item per thread) has it: the first in the list.  claim: [rows] scratch.
VK_DEV void claim_rows(const int32_t* list, int n, int rows, int32_t* claim) {
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (list[i] >= 0 && list[i] < rows) claim[list[i]] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (list[i] >= 0 && list[i] < rows) atomicMin(&claim[list[i]], i);
  __syncthreads();
}

// The tokens of a row, -1 where its length or its partly filled last page is out of range.
VK_DEV int row_len(const Pool& p, int row) {
  const int len = p.lens[row];
  if (len < 0 || len > p.max_pages << p.page_shift) return -1;
  if ((len & ((1 << p.page_shift) - 1)) == 0) return len;
  const int last = p.table[static_cast<int64_t>(row) * p.max_pages + (len >> p.page_shift)];
  return last >= 0 && last < p.n_pages ? len : -1;
}
// Of a length a row can have: at most max_pages whole pages, so the sum stays below 2^31.
VK_DEV int pages_of(const Pool& p, int len) { return (len + (1 << p.page_shift) - 1) >> p.page_shift; }

struct ExtendArgs {
  Pool p;
  const int32_t* list;  // [n] rows, or NULL: all rows
  int n, count;
  int32_t* page;        // [n, count] out
  int32_t* slot;
  int32_t* claim;       // [rows] scratch
  int32_t* first;       // [n] scratch: place of the item's first new page in the free list, -1: not served
  int32_t* len;         // [n] scratch: tokens before the call
  int32_t* free_list;   // [n_pages] scratch
};

// Tables, counts and places of the cells (item, token) x0, x0 + step, ...
VK_DEV void extend_cells(const ExtendArgs& a, uint32_t x0, uint32_t step) {
  const Pool& p = a.p;
  const uint32_t cells = static_cast<uint32_t>(a.n) * a.count;  // below 2^31
  for (uint32_t x = x0; x < cells; x += step) {
    const uint32_t i = x / a.count;
    const int j = static_cast<int>(x - i * a.count), at = a.first[i];
    int pg = -1, slot = -1;
    if (at >= 0) {
      const int row = a.list ? a.list[i] : i, len = a.len[i], pos = len + j;
      const int c = pos >> p.page_shift, old = pages_of(p, len);
      int32_t* cell = p.table + static_cast<int64_t>(row) * p.max_pages + c;
      slot = pos & ((1 << p.page_shift) - 1);
      if (c < old) {
        pg = *cell;
      } else {
        pg = a.free_list[at + c - old];
        if (slot == 0) {  // a new page's first token
          *cell = pg;
          p.refs[pg] = 1;
        }
      }
      if (j == 0) p.lens[row] = len + a.count;
    }
    a.page[x] = pg;
    a.slot[x] = slot;
  }
}

// Room for `count` more tokens in each listed row.  cells: the cells are written here.
__global__ void __launch_bounds__(kPlanThreads) extend_kernel(ExtendArgs a, bool cells) {
  const Pool& p = a.p;
  pdl_wait();
  pdl_launch_dependents();
  if (a.list) claim_rows(a.list, a.n, p.rows, a.claim);
  int want = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    bool ok = i < a.n;
    if (ok) {
      const int row = a.list ? a.list[i] : i;
      ok = row >= 0 && row < p.rows && (!a.list || a.claim[row] == i);
      if (ok) {
        const int len = row_len(p, row);
        a.len[i] = len;
        ok = len >= 0 && a.count <= (p.max_pages << p.page_shift) - len;  // (their sum may pass 2^31)
        if (ok) need = pages_of(p, len + a.count) - pages_of(p, len);
      }
      if (!ok) raise_error(ERR_BOUNDS);
    }
    int n;
    const int at = want + block_scan(need, &n);
    if (i < a.n) a.first[i] = ok ? at : -1;
    want += n;
  }
  const int got = free_pages(p, want < p.n_pages ? want : p.n_pages, a.free_list);
  // a row that is refused keeps its places in the list, so that no later row takes a page that an earlier one lacked
  if (got < want)
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
      const int at = a.first[i];
      if (at < 0) continue;
      const int need = pages_of(p, a.len[i] + a.count) - pages_of(p, a.len[i]);
      if (need && at + need > got) {
        raise_error(ERR_PAGES);
        a.first[i] = -1;
      }
    }
  __syncthreads();
  if (cells) extend_cells(a, threadIdx.x, kPlanThreads);
}

__global__ void __launch_bounds__(256) extend_cells_kernel(ExtendArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  extend_cells(a, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

struct ForkArgs {
  Pool p;
  const int32_t* src;
  const int32_t* dst;
  int n;
  int32_t* claim;      // [rows] scratch
  int32_t* state;      // [n] scratch: place in the free list, -1: not served or nothing to do
  int32_t* len;        // [n] scratch: the new length
  int32_t* stage;      // [n, max_pages] scratch: the new table rows
  int32_t* free_list;  // [n] scratch
  Move* moves;         // [n] out
};

// The new table rows' cells (item, column) x0, x0 + step, ...: put down before any table row is written, since a row may be
// source and target at once.
VK_DEV void fork_stage(const ForkArgs& a, uint32_t x0, uint32_t step) {
  const Pool& p = a.p;
  const int mask = (1 << p.page_shift) - 1;
  const uint32_t cells = static_cast<uint32_t>(a.n) * p.max_pages;  // below 2^31
  for (uint32_t x = x0; x < cells; x += step) {
    const uint32_t i = x / p.max_pages;
    const int c = static_cast<int>(x - i * p.max_pages), at = a.state[i];
    if (at < 0) continue;
    const int full = a.len[i] >> p.page_shift;
    int v = -1;
    if (c < full)
      v = p.table[static_cast<int64_t>(a.src[i]) * p.max_pages + c];
    else if (c == full && (a.len[i] & mask))
      v = a.free_list[at];
    a.stage[x] = v;
  }
}

// Tables, lengths and counts from the new rows.
VK_DEV void fork_write(const ForkArgs& a, uint32_t x0, uint32_t step) {
  const Pool& p = a.p;
  const uint32_t cells = static_cast<uint32_t>(a.n) * p.max_pages;
  for (uint32_t x = x0; x < cells; x += step) {
    const uint32_t i = x / p.max_pages;
    const int c = static_cast<int>(x - i * p.max_pages);
    if (a.state[i] < 0) continue;
    int32_t* cell = p.table + static_cast<int64_t>(a.dst[i]) * p.max_pages + c;
    const int old = *cell, now = a.stage[x];
    if (old != now) {
      if (old >= 0 && old < p.n_pages) atomicSub(&p.refs[old], 1);
      if (now >= 0 && now < p.n_pages) atomicAdd(&p.refs[now], 1);
      *cell = now;
    }
    if (c == 0) p.lens[a.dst[i]] = a.len[i];
  }
}

// Rows dst[i] become copies of the rows src[i] as they were before the call.  cells: the table rows are written here.
__global__ void __launch_bounds__(kPlanThreads) fork_kernel(ForkArgs a, bool cells) {
  const Pool& p = a.p;
  const int mask = (1 << p.page_shift) - 1;
  pdl_wait();
  pdl_launch_dependents();
  claim_rows(a.dst, a.n, p.rows, a.claim);
  int want = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    bool ok = i < a.n;
    if (ok) {
      const int s = a.src[i], t = a.dst[i];
      ok = s >= 0 && s < p.rows && t >= 0 && t < p.rows && a.claim[t] == i;
      const int len = ok ? row_len(p, s) : -1;
      if (len < 0) raise_error(ERR_BOUNDS);
      ok = len >= 0 && s != t;
      if (ok) {
        a.len[i] = len;
        need = (len & mask) != 0;
      }
    }
    int n;
    const int at = want + block_scan(need, &n);
    if (i < a.n) a.state[i] = ok ? at : -1;
    want += n;
  }
  const int got = free_pages(p, want, a.free_list);
  // what is copied
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    Move m{0, 0, 0};
    const int at = a.state[i];
    if (at >= 0) {
      const int part = a.len[i] & mask, full = a.len[i] >> p.page_shift;
      if (part && at >= got) {
        raise_error(ERR_PAGES);
        a.state[i] = -1;
      } else if (part) {
        m = Move{p.table[static_cast<int64_t>(a.src[i]) * p.max_pages + full], a.free_list[at], part};
      }
    }
    a.moves[i] = m;
  }
  __syncthreads();
  if (!cells) return;
  fork_stage(a, threadIdx.x, kPlanThreads);
  __syncthreads();
  fork_write(a, threadIdx.x, kPlanThreads);
}

__global__ void __launch_bounds__(256) fork_stage_kernel(ForkArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  fork_stage(a, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// The listed rows (NULL: all) give their pages up.  One warp per row; a row named twice is empty the second time.
__global__ void __launch_bounds__(256) free_kernel(Pool p, const int32_t* list, int n) {
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  if (i >= n) return;
  const int row = list ? list[i] : i;
  if (row < 0 || row >= p.rows) {
    if (lane == 0) raise_error(ERR_BOUNDS);
    return;
  }
  if (lane == 0) p.lens[row] = 0;
  for (int c = lane; c < p.max_pages; c += 32) {
    const int old = atomicExch(&p.table[static_cast<int64_t>(row) * p.max_pages + c], -1);
    if (old >= 0 && old < p.n_pages) atomicSub(&p.refs[old], 1);
  }
}

struct CompactArgs {
  Pool p;
  int32_t* holes;   // [n_pages] scratch
  int32_t* goes;    // [n_pages] scratch, from number `live` on: where a moved page goes, -1: it was free
  Move* moves;      // [n_pages / 2] out
  int32_t* counts;  // [2] out: moves, pages in use
  int32_t* live;    // [1] out: pages in use
};

// The live pages from number `live` on go into the free pages below it, both in ascending order.
__global__ void __launch_bounds__(kPlanThreads) compact_kernel(CompactArgs a) {
  const Pool& p = a.p;
  pdl_wait();
  pdl_launch_dependents();
  const int live = scan_pages(p.refs, 0, p.n_pages, true, p.n_pages, [](int, int) {});
  scan_pages(p.refs, 0, live, false, live, [&](int at, int i) { a.holes[at] = i; });
  for (int i = live + threadIdx.x; i < p.n_pages; i += kPlanThreads) a.goes[i] = -1;
  __syncthreads();
  const int moved = scan_pages(p.refs, live, p.n_pages, true, p.n_pages, [&](int at, int i) {
    const int to = a.holes[at];
    a.moves[at] = Move{i, to, 1 << p.page_shift};
    a.goes[i] = to;
    p.refs[to] = p.refs[i];
    p.refs[i] = 0;
  });
  if (threadIdx.x == 0) {
    a.counts[0] = moved;
    a.counts[1] = live;
    a.live[0] = live;
  }
}

struct CopyArgs {
  uint8_t* k;          // [layers, n_pages, page_bytes]
  uint8_t* v;
  const Move* moves;
  const int32_t* count;  // moves to make, or NULL: n
  int n, layers;
  int64_t page_bytes, layer_bytes;
  int token_bytes;     // a multiple of 16
};

// What the copying kernel does besides: nothing, the new table rows of a fork, or the new page numbers of a compaction.
struct JustCopy {
  VK_DEV void operator()(uint32_t, uint32_t) const {}
};
struct ForkWrite {
  ForkArgs a;
  VK_DEV void operator()(uint32_t x0, uint32_t step) const { fork_write(a, x0, step); }
};
struct Renumber {
  Pool p;
  const int32_t* goes;
  const int32_t* live;
  VK_DEV void operator()(uint32_t x0, uint32_t step) const {
    const int from = *live;
    const uint32_t cells = static_cast<uint32_t>(p.rows) * p.max_pages;  // below 2^31
    for (uint32_t x = x0; x < cells; x += step) {
      const int old = p.table[x];
      if (old < from || old >= p.n_pages) continue;
      const int to = goes[old];
      if (to >= 0)
        p.table[x] = to;
      else
        raise_error(ERR_BOUNDS);  // the table names a page that refs holds for free
    }
  }
};

// Copies each move's tokens in every layer of K and V.  Bound by HBM: 16 bytes per thread and load, a unit (one page of one layer
// of K or V) per CTA at a time, eight CTAs an SM; 1485 moves of 262 KB (8 layers): 111 us, 7.0 TB/s.
template <typename Also>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(CopyArgs a, Also also) {
  pdl_wait();
  pdl_launch_dependents();
  also(blockIdx.x * kCopyThreads + threadIdx.x, gridDim.x * kCopyThreads);
  const int n = a.count ? *a.count : a.n;
  const int64_t units = static_cast<int64_t>(n) * a.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const Move m = a.moves[u / (a.layers * 2)];
    const int layer = static_cast<int>(u / 2 % a.layers);
    uint8_t* base = (u & 1 ? a.v : a.k) + layer * a.layer_bytes;
    const uint4* from = reinterpret_cast<const uint4*>(base + m.src * a.page_bytes);
    uint4* to = reinterpret_cast<uint4*>(base + m.dst * a.page_bytes);
    const int64_t words = static_cast<int64_t>(m.tokens) * a.token_bytes / 16;
    for (int64_t i = threadIdx.x; i < words; i += kCopyThreads) to[i] = from[i];
  }
}

}  // namespace pages
}  // namespace vk

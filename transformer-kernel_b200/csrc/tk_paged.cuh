// Bookkeeping and data movement of a paged key-value cache.
//
// A cache is one fp16 pool [layers, num_pages, 2 (k, v), Hkv, page_size, hd]
// and its books, all int32 on the device: a page table [max_seqs, width], the
// sequences' lengths, a reference count per page and a bit per page that is
// set while the page is free. The state a call leaves depends on the books
// and the call alone: pages are always taken lowest first, in the order of
// the call's entries, and reference counts move by integer atomics, whose
// order does not show. A partial last page has one holder (fork copies it),
// so appending to a sequence never writes a page that another one reads.
//
// A call applies whole or not at all: its entries are checked before anything
// is written, a refused call sets a bit of the status word and the device
// error word, and while the status word is set later calls on the cache
// change nothing. The pages that a table names are not among what is checked
// first: one outside the pool, which these calls never leave there, is skipped
// and reported by fork and store when they reach it, with the rest of the call
// applied or not. Entries with slot -1 are padding and are skipped.
//
// These kernels are bound by latency (integer work on a few kB, one CTA that
// scans the free bits: 7 us for 640 pages of 8 prompts) and, where data moves,
// by HBM, 2 bytes of traffic per byte: store of 45,000 tokens x 16 heads of 64
// in 64 us (5.8 TB/s), a compaction that moves 0.37 GB in 127 us (5.8), 1000
// pages of 0.5 MB copied in 177 us (5.9).
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

#include "tk_ptx.cuh"

namespace tk {
namespace paged {

// Bits of the status word.
enum : int {
  kOutOfPages = 1,  // fewer free pages than the call needs
  kBadSlot = 2,     // a slot out of range or named twice, or a negative count
  kTooLong = 4,     // a sequence longer than its row of the page table
  kBadPage = 8,     // the page table or a list of pages names one outside the pool
  kNotEmpty = 16,   // a slot that has to be empty is not
  kTimedOut = 32,   // a wait inside an attention call gave up
};

struct Books {
  int* table;           // [max_seqs, width]
  int* lens;            // [max_seqs]
  int* refs;            // [num_pages]
  uint32_t* free_mask;  // [mask_words]: bit set = page free; padded with zeros to 4 words
  int* status;
  int* live;            // pages in use after a compaction
  int* scratch;         // [3 * num_pages]
  int64_t width;
  int max_seqs, num_pages, mask_words;
  int page_shift;
};

constexpr int kPlanThreads = 512;  // single-CTA kernels
constexpr int kMaxEntries = 8192;  // entries of one call (their prefix sums stay in shared memory)

__device__ __forceinline__ void refuse(const Books& b, int why, unsigned where) {
  atomicOr(b.status, why);
  report_error(kDevCacheRefused, where);
}

// Exclusive prefix sum of one value per thread; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[wid] = x;
  __syncthreads();
  int before = 0, all = 0;
  const int nw = blockDim.x >> 5;
  for (int w = 0; w < nw; ++w) {
    const int s = warp_sums[w];
    before += w < wid ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// Ids of the lowest `want` free pages into `list`, ascending; returns how
// many there are (at least `want`, or fewer when the pool has no more).
__device__ __forceinline__ int lowest_free(const Books& b, int want, int* list, int* warp_sums) {
  int found = 0;
  for (int base = 0; base < b.mask_words && found < want; base += static_cast<int>(blockDim.x) * 4) {
    const int w0 = base + static_cast<int>(threadIdx.x) * 4;
    uint4 m = make_uint4(0u, 0u, 0u, 0u);
    if (w0 < b.mask_words) m = *reinterpret_cast<const uint4*>(b.free_mask + w0);
    const uint32_t words[4] = {m.x, m.y, m.z, m.w};
    int total;
    int r = found + block_scan(__popc(m.x) + __popc(m.y) + __popc(m.z) + __popc(m.w), warp_sums, &total);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = words[i];
      while (w != 0u && r < want) {
        list[r++] = (w0 + i) * 32 + __ffs(w) - 1;
        w &= w - 1u;
      }
    }
    found += total;
  }
  __syncthreads();
  return found;
}

// Entry that owns page number r of the call: the last i with first[i] <= r
// among entries that need pages (first is the exclusive prefix sum).
__device__ __forceinline__ int owner_of(const int* first, int n, int r) {
  int lo = 0, hi = n;  // first[lo] <= r < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void take_page(const Books& b, int page) {
  b.refs[page] = 1;
  atomicAnd(b.free_mask + (page >> 5), ~(1u << (page & 31)));
}

// Appends counts[i] tokens to sequence slots[i]: lengths grow, and the pages
// that they reach into are taken.
__global__ void __launch_bounds__(kPlanThreads)
    reserve_kernel(Books b, const int* slots, const int* counts, int n, int require_empty) {
  extern __shared__ int sh[];
  int* first = sh;                                          // [n]
  uint32_t* seen = reinterpret_cast<uint32_t*>(sh + n);     // [max_seqs / 32]
  __shared__ int warp_sums[32];
  for (int i = threadIdx.x; i < (b.max_seqs + 31) / 32; i += blockDim.x) seen[i] = 0u;
  grid_dep_wait();
  if (*b.status != 0) return;
  __syncthreads();
  const int ps = 1 << b.page_shift;
  int bad = 0, total = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n && slots[i] != -1) {
      const int s = slots[i], c = counts[i];
      if (s < 0 || s >= b.max_seqs || c < 0) {
        bad |= kBadSlot;
      } else {
        if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad |= kBadSlot;
        const int64_t len = b.lens[s], want = len + c;
        if (len < 0 || want > b.width * ps) bad |= kTooLong;
        if (require_empty && len != 0) bad |= kNotEmpty;
        if (bad == 0)
          need = static_cast<int>(((want + ps - 1) >> b.page_shift) - ((len + ps - 1) >> b.page_shift));
      }
    }
    int sum;
    const int before = block_scan(need, warp_sums, &sum);
    if (i < n) first[i] = total + before;
    // more pages than the pool has is refused below, whatever the excess
    total = static_cast<int>(min(static_cast<int64_t>(total) + sum, static_cast<int64_t>(1) << 30));
  }
  if (total > b.num_pages) bad |= kOutOfPages;
  if (__syncthreads_or(bad)) {
    if (bad) refuse(b, bad, 0xB100u);
    return;
  }
  if (total > 0) {
    if (lowest_free(b, total, b.scratch, warp_sums) < total) {
      if (threadIdx.x == 0) refuse(b, kOutOfPages, 0xB101u);
      return;
    }
    for (int r = threadIdx.x; r < total; r += blockDim.x) {
      const int i = owner_of(first, n, r);
      const int s = slots[i], page = b.scratch[r];
      const int64_t have = (b.lens[s] + ps - 1) >> b.page_shift;
      b.table[s * b.width + have + (r - first[i])] = page;
      take_page(b, page);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (slots[i] != -1) b.lens[slots[i]] += counts[i];
}

// First half of a fork: checks the pairs, gives each child its length and,
// where the parent's last page is partial, a page of its own for it.
__global__ void __launch_bounds__(kPlanThreads)
    fork_plan_kernel(Books b, const int* src, const int* dst, int n) {
  extern __shared__ int sh[];
  int* first = sh;
  uint32_t* seen = reinterpret_cast<uint32_t*>(sh + n);
  __shared__ int warp_sums[32];
  for (int i = threadIdx.x; i < (b.max_seqs + 31) / 32; i += blockDim.x) seen[i] = 0u;
  grid_dep_wait();
  if (*b.status != 0) return;
  __syncthreads();
  const int ps = 1 << b.page_shift;
  int bad = 0, total = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n && src[i] != -1 && dst[i] != -1) {
      const int s = src[i], d = dst[i];
      if (s < 0 || s >= b.max_seqs || d < 0 || d >= b.max_seqs) {
        bad |= kBadSlot;
      } else {
        if (atomicOr(&seen[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) bad |= kBadSlot;
        if (b.lens[d] != 0) bad |= kNotEmpty;
        if (b.lens[s] < 0 || b.lens[s] > b.width * ps) bad |= kTooLong;
        if (bad == 0) need = (b.lens[s] & (ps - 1)) != 0;
      }
    }
    int sum;
    const int before = block_scan(need, warp_sums, &sum);
    if (i < n) first[i] = total + before;
    total += sum;
  }
  if (__syncthreads_or(bad)) {
    if (bad) refuse(b, bad, 0xB200u);
    return;
  }
  if (total > b.num_pages || (total > 0 && lowest_free(b, total, b.scratch, warp_sums) < total)) {
    if (threadIdx.x == 0) refuse(b, kOutOfPages, 0xB201u);
    return;
  }
  for (int r = threadIdx.x; r < total; r += blockDim.x) {
    const int i = owner_of(first, n, r), page = b.scratch[r];
    b.table[dst[i] * b.width + (b.lens[src[i]] >> b.page_shift)] = page;
    take_page(b, page);
  }
  __syncthreads();  // the owners have been looked up: `first` now takes the lengths
  // a child may be another pair's (empty) parent: every length is read before any is written
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    if (i < n) first[i] = (src[i] != -1 && dst[i] != -1) ? b.lens[src[i]] : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (src[i] != -1 && dst[i] != -1) b.lens[dst[i]] = first[i];
}

// Where the pages' numbers are: page p of layer l is one contiguous block of
// page_vecs 16-byte vectors, [2, Hkv, page_size, hd].
struct Pool {
  uint4* base;
  int64_t layer_vecs, page_vecs;
  int layers, row_vecs;  // 16-byte vectors of one token's row of one head
};

__device__ __forceinline__ bool page_ok(const Books& b, int page) { return page >= 0 && page < b.num_pages; }

// Second half of a fork: grid (pairs, chunks). Shares the full pages and
// copies the used rows of the partial one, over every layer.
__global__ void __launch_bounds__(256) fork_apply_kernel(Books b, Pool pool, const int* src, const int* dst) {
  grid_dep_wait();
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s == -1 || d == -1 || *b.status != 0) return;
  const int len = b.lens[d], ps = 1 << b.page_shift;
  const int full = len >> b.page_shift, rows = len & (ps - 1);
  const int step = gridDim.y * blockDim.x, t0 = blockIdx.y * blockDim.x + threadIdx.x;
  const int* from = b.table + s * b.width;
  int* to = b.table + d * b.width;
  for (int k = t0; k < full; k += step) {
    const int page = from[k];
    to[k] = page;
    if (page_ok(b, page)) atomicAdd(b.refs + page, 1);
    else refuse(b, kBadPage, 0xB202u);
  }
  if (rows == 0) return;
  const int p0 = from[full], p1 = to[full];
  if (!page_ok(b, p0) || !page_ok(b, p1)) {
    if (t0 == 0) refuse(b, kBadPage, 0xB203u);
    return;
  }
  const int head_vecs = ps * pool.row_vecs, used = rows * pool.row_vecs;
  const int heads = static_cast<int>(pool.page_vecs / head_vecs);  // k and v heads together
  const int64_t total = static_cast<int64_t>(pool.layers) * heads * used;
  for (int64_t v = t0; v < total; v += step) {
    const int64_t block = v / used;
    const int64_t at = (block / heads) * pool.layer_vecs + (block % heads) * head_vecs + v % used;
    pool.base[at + p1 * pool.page_vecs] = pool.base[at + p0 * pool.page_vecs];
  }
}

// One CTA per entry: its pages lose a reference, those without any become
// free. Every CTA checks the whole list, so that all agree whether it applies.
__global__ void __launch_bounds__(256) release_kernel(Books b, const int* slots, int n) {
  extern __shared__ int sh[];
  uint32_t* seen = reinterpret_cast<uint32_t*>(sh);
  for (int i = threadIdx.x; i < (b.max_seqs + 31) / 32; i += blockDim.x) seen[i] = 0u;
  grid_dep_wait();
  const int status = *b.status;  // only a refusal of this very list can set it meanwhile
  if (__syncthreads_or(status)) return;
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = slots[i];
    if (s == -1) continue;
    if (s < 0 || s >= b.max_seqs) bad = kBadSlot;
    else if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad = kBadSlot;
  }
  if (__syncthreads_or(bad)) {
    if (bad && blockIdx.x == 0) refuse(b, bad, 0xB300u);
    return;
  }
  const int s = slots[blockIdx.x];
  if (s == -1) return;
  const int64_t len = max(0, b.lens[s]);
  const int64_t pages = min(b.width, (len + (1 << b.page_shift) - 1) >> b.page_shift);
  __syncthreads();
  int* row = b.table + s * b.width;
  for (int64_t k = threadIdx.x; k < pages; k += blockDim.x) {
    const int page = row[k];
    row[k] = -1;
    if (!page_ok(b, page)) continue;  // reported where the page was to be used
    if (atomicSub(b.refs + page, 1) == 1) atomicOr(b.free_mask + (page >> 5), 1u << (page & 31));
  }
  if (threadIdx.x == 0) b.lens[s] = 0;
}

// First half of a compaction: pairs the k-th free page below the number of
// live pages with the k-th live page at or above it, moves the reference
// counts and rewrites the free bits. scratch = [pages to fill][pages to
// empty][new id of every emptied page].
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(Books b, int* moved) {
  __shared__ int warp_sums[32];
  grid_dep_wait();
  if (*b.status != 0) {
    if (threadIdx.x == 0) *moved = 0;
    return;
  }
  int* fill = b.scratch;
  int* empty = b.scratch + b.num_pages;
  int* new_id = b.scratch + 2 * static_cast<int64_t>(b.num_pages);
  int free_here = 0;
  for (int w = threadIdx.x; w < b.mask_words; w += blockDim.x) free_here += __popc(b.free_mask[w]);
  int free_pages;
  block_scan(free_here, warp_sums, &free_pages);
  const int live = b.num_pages - free_pages;
  int fills = 0, empties = 0;
  for (int base = 0; base < b.mask_words; base += blockDim.x) {
    const int w = base + threadIdx.x, p0 = w * 32;
    uint32_t free_w = 0u, valid = 0u, below = 0u;
    if (w < b.mask_words) {
      free_w = b.free_mask[w];
      const int in_pool = min(32, max(0, b.num_pages - p0)), low = min(32, max(0, live - p0));
      valid = in_pool == 32 ? ~0u : (1u << in_pool) - 1u;
      below = low == 32 ? ~0u : (1u << low) - 1u;
    }
    uint32_t f = free_w & below, e = ~free_w & valid & ~below;
    int sum;
    // both counts fit one scan: a chunk has 32 * kPlanThreads = 2^14 pages
    const int before = block_scan(__popc(f) | (__popc(e) << 16), warp_sums, &sum);
    int rf = fills + (before & 0xffff), re = empties + (before >> 16);
    while (f != 0u) {
      fill[rf++] = p0 + __ffs(f) - 1;
      f &= f - 1u;
    }
    while (e != 0u) {
      empty[re++] = p0 + __ffs(e) - 1;
      e &= e - 1u;
    }
    fills += sum & 0xffff;
    empties += sum >> 16;
    __syncthreads();
    if (w < b.mask_words) b.free_mask[w] = valid & ~below;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < empties; k += blockDim.x) {
    const int to = fill[k], from = empty[k];
    b.refs[to] = b.refs[from];
    b.refs[from] = 0;
    new_id[from] = to;
  }
  if (threadIdx.x == 0) {
    *b.live = live;
    *moved = empties;
  }
}

// Second half: renames the moved pages in the tables and copies their data
// over every layer. Sources and destinations are disjoint sets, so the copies
// need no order.
__global__ void __launch_bounds__(256) compact_apply_kernel(Books b, Pool pool, const int* moved) {
  grid_dep_wait();
  if (*b.status != 0) return;
  const int m = *moved, live = *b.live;
  if (m == 0) return;
  const int* fill = b.scratch;
  const int* empty = b.scratch + b.num_pages;
  const int* new_id = b.scratch + 2 * static_cast<int64_t>(b.num_pages);
  for (int s = blockIdx.x; s < b.max_seqs; s += gridDim.x) {
    const int64_t len = max(0, b.lens[s]);
    const int64_t pages = min(b.width, (len + (1 << b.page_shift) - 1) >> b.page_shift);
    int* row = b.table + s * b.width;
    for (int64_t k = threadIdx.x; k < pages; k += blockDim.x) {
      const int page = row[k];
      if (page_ok(b, page) && page >= live) row[k] = new_id[page];
    }
  }
  constexpr int kUnroll = 8;  // four: 133 us for 0.37 GB moved, against 127
  const int64_t chunk = 256 * kUnroll;  // vectors a CTA copies at a time
  const int64_t chunks = (pool.page_vecs + chunk - 1) / chunk;
  const int64_t units = static_cast<int64_t>(m) * pool.layers * chunks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t c = u % chunks, kl = u / chunks;
    const int64_t layer = kl % pool.layers;
    const int k = static_cast<int>(kl / pool.layers);
    const uint4* from = pool.base + layer * pool.layer_vecs + empty[k] * pool.page_vecs;
    uint4* to = pool.base + layer * pool.layer_vecs + fill[k] * pool.page_vecs;
    uint4 v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t at = c * chunk + i * 256 + threadIdx.x;
      if (at < pool.page_vecs) v[i] = from[at];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t at = c * chunk + i * 256 + threadIdx.x;
      if (at < pool.page_vecs) to[at] = v[i];
    }
  }
}

// Rebuilds the free bits from the reference counts.
__global__ void __launch_bounds__(256) free_mask_kernel(Books b) {
  grid_dep_wait();
  const int w = blockIdx.x * blockDim.x + threadIdx.x;
  if (w >= b.mask_words) return;
  uint32_t bits = 0u;
  for (int i = 0; i < 32; ++i) {
    const int page = w * 32 + i;
    if (page < b.num_pages && b.refs[page] <= 0) bits |= 1u << i;
  }
  b.free_mask[w] = bits;
}

// Whole pages src[i] -> dst[i] of every layer; grid (pairs, chunks). Every CTA
// checks the whole list, so that all agree whether it applies.
__global__ void __launch_bounds__(256) copy_pages_kernel(Books b, Pool pool, const int* src, const int* dst) {
  grid_dep_wait();
  const int status = *b.status;  // only a refusal of this very list can set it meanwhile
  if (__syncthreads_or(status)) return;
  int bad = 0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += blockDim.x)
    if (!page_ok(b, src[i]) || !page_ok(b, dst[i])) bad = kBadPage;
  if (__syncthreads_or(bad)) {
    if (bad && blockIdx.x == 0 && blockIdx.y == 0) refuse(b, bad, 0xB400u);
    return;
  }
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  const int64_t total = pool.layers * pool.page_vecs;
  for (int64_t v = static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x; v < total;
       v += static_cast<int64_t>(gridDim.y) * blockDim.x) {
    const int64_t at = (v / pool.page_vecs) * pool.layer_vecs + v % pool.page_vecs;
    pool.base[at + d * pool.page_vecs] = pool.base[at + s * pool.page_vecs];
  }
}

// Keys and values of the last counts[b] tokens of sequence slots[b] into
// their pages of one layer. k, v: logically [B, Hkv, S, hd]; a thread moves
// one 16-byte piece of a key row and of the value row. Reads run along the
// rows of the projection, writes are the hd * 2 contiguous bytes of a head's
// row in its page.
struct StoreParams {
  const __half* k;
  const __half* v;
  int64_t stride_b, stride_h, stride_s;
  const int* slots;
  const int* counts;  // null: every row has S tokens
  uint4* pages;       // this layer's pages
  int64_t page_vecs;
  int S, heads, row_vecs;
};

__global__ void __launch_bounds__(256) store_kernel(Books b, StoreParams p) {
  extern __shared__ int sh[];
  uint32_t* seen = reinterpret_cast<uint32_t*>(sh);  // [max_seqs / 32]
  for (int i = threadIdx.x; i < (b.max_seqs + 31) / 32; i += blockDim.x) seen[i] = 0u;
  grid_dep_wait();
  const int status = *b.status;  // a refusal of this very list, or a page outside the pool, can set it meanwhile
  if (__syncthreads_or(status)) return;
  const int ps = 1 << b.page_shift;
  // every CTA checks every row, so that all agree whether the call applies
  int bad = 0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.y); i += blockDim.x) {
    const int s = p.slots[i];
    if (s == -1) continue;
    if (s < 0 || s >= b.max_seqs) {
      bad |= kBadSlot;
      continue;
    }
    if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad |= kBadSlot;
    const int count = p.counts == nullptr ? p.S : p.counts[i];
    const int64_t len = b.lens[s];
    if (count < 0 || count > p.S || count > len || len > b.width * ps) bad |= kTooLong;
  }
  if (__syncthreads_or(bad)) {
    if (bad && blockIdx.x == 0 && blockIdx.y == 0) refuse(b, bad, 0xB500u);
    return;
  }
  const int row = blockIdx.y;
  const int s = p.slots[row];
  if (s == -1) return;
  const int count = p.counts == nullptr ? p.S : p.counts[row];
  const int64_t len = b.lens[s];
  const int per_token = p.heads * p.row_vecs;
  const int64_t total = static_cast<int64_t>(count) * per_token;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int t = static_cast<int>(i / per_token);
    const int within = static_cast<int>(i % per_token);
    const int h = within / p.row_vecs, c = within % p.row_vecs;
    const int64_t pos = len - count + t;
    const int page = b.table[s * b.width + (pos >> b.page_shift)];
    if (!page_ok(b, page)) {
      refuse(b, kBadPage, 0xB501u);
      continue;
    }
    const int64_t from = row * p.stride_b + h * p.stride_h + t * p.stride_s + c * 8;
    uint4* to = p.pages + page * p.page_vecs + (static_cast<int64_t>(h) * ps + (pos & (ps - 1))) * p.row_vecs + c;
    const uint4 kv = *reinterpret_cast<const uint4*>(p.k + from);
    const uint4 vv = *reinterpret_cast<const uint4*>(p.v + from);
    to[0] = kv;
    to[p.page_vecs / 2] = vv;
  }
}

}  // namespace paged
}  // namespace tk

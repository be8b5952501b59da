// Attention of one new token per sequence over a paged key-value cache.
//
//   out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j   over the visible
//   keys j < len:  len - 1 - j < window  or  j < sinks   (window 0: all)
//
// k_j and v_j live in pages of page_size tokens, [Hkv, page_size, hd] each,
// named by a page table; H / Hkv query heads share a key-value head. With
// k_new / v_new the last key is the new token's: it is written into its page
// here and read from the argument, so a decode step needs no store launch.
//
// Bound by HBM: every visible key and value is read once, 4 * hd bytes per
// key and key-value head, against 4 * G * hd operations (G = H / Hkv). The
// tensor cores take the products because the FMA pipe could not at G >= 4:
// one m16n8k16 product handles up to 16 query heads of a group. These are the
// warp-level mma.sync products on purpose: a decode step has 1 to 16 query
// rows per key-value head, so a 128-row tcgen05 tile would idle at least 7/8
// of its rows and its operands' way through TMEM would only add latency,
// while the warp-level rate is several times what HBM can feed.
//
// Each warp works alone: it walks its keys KS at a time through its own ring
// of NST shared-memory stages, filled by TMA (a 4-D map over the pages, boxes
// of 16 or KS rows that never cross a page, swizzled so that ldmatrix reads
// without bank conflicts) and one mbarrier per stage. S = Q K^T and O = P V
// keep their accumulators, the running maximum and the sum in registers in
// fp32; P is rounded to fp16 for the second product (half a step, 2^-11
// relative, as in the prompt kernel). No barrier joins the warps until their
// results are merged.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "tk_paged.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace decode {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;  // query heads of one m16n8k16 tile

template <int HD>
struct Cfg {
  static_assert(HD == 16 || HD == 32 || HD == 64 || HD == 128 || HD == 256, "head_dim");
  static constexpr int KS = HD <= 32 ? 32 : 16;                 // keys per step
  static constexpr int NST = HD >= 128 ? 3 : 4;                 // stages per warp
  static constexpr int SPAN = HD >= 64 ? 128 : HD * 2;          // swizzle span, bytes
  static constexpr int COLS = HD >= 64 ? 64 : HD;               // columns of a TMA box
  static constexpr int CHUNKS = HD / COLS;                      // boxes per row
  static constexpr int CHUNK_BYTES = KS * SPAN;                 // [KS, COLS]
  static constexpr int TILE_BYTES = CHUNKS * CHUNK_BYTES;       // K or V of one step
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int WARP_BYTES = NST * STAGE_BYTES;
  static constexpr int SMEM_BYTES = kWarps * WARP_BYTES + 1024;
  static_assert(CHUNK_BYTES % 1024 == 0, "swizzle atoms");
};

struct Params {
  const __half* q;        // [B, H, hd]
  const __half* k_new;    // optional [B, Hkv, hd]: the token at position len - 1
  const __half* v_new;
  __half* k_pages;        // [P, Hkv, page_size, hd] with the strides below
  __half* v_pages;
  const int* table;       // [max_seqs, width]
  const int* lens;        // [max_seqs]
  const int* slots;       // optional [B]; absent: row b is sequence b; -1: padding
  int* status;            // optional status word of the cache
  __half* out;            // [B, ld_out], head h at columns [h * hd, h * hd + hd)
  int64_t q_stride_b, q_stride_h, new_stride_b, new_stride_h, page_stride, head_stride, width, ld_out;
  int B, H, Hkv, G, gtiles, max_seqs, num_pages, page_shift, box_rows;
  int hd;                 // head_dim of the data: HD, or 8 in the HD = 16 kernel (zero-padded by TMA)
  int window, sinks;      // window 0: every key
  float scale_log2;
  uint64_t wait_limit_ns;
};

// The visible keys of a sequence as a list of KS-key steps: the first
// `sink_steps` steps start at key 0, the others at `lo`, a multiple of KS.
template <int KS>
struct Span {
  int len, first, lo, sinks, sink_steps, steps;  // first = first key of the window

  __device__ __forceinline__ Span(const Params& p, int n) {
    len = n;
    first = (p.window > 0 && n > p.window) ? n - p.window : 0;
    sinks = p.sinks;
    lo = first / KS * KS;
    sink_steps = min((min(sinks, n) + KS - 1) / KS, lo / KS);
    steps = n > 0 ? sink_steps + (n - lo + KS - 1) / KS : 0;
  }
  __device__ __forceinline__ int key0(int step) const {
    return step < sink_steps ? step * KS : lo + (step - sink_steps) * KS;
  }
  __device__ __forceinline__ bool visible(int key) const { return key < len && (key >= first || key < sinks); }
  // every key of the step is visible
  __device__ __forceinline__ bool whole(int key) const {
    return key + KS <= len && (key >= first || key + KS <= sinks);
  }
};

// Byte offset of 16-byte piece c of row r in a swizzled [rows, SPAN] tile.
template <int SPAN>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  if (SPAN == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  if (SPAN == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  return r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}

// The same for a K or V tile of CHUNKS such tiles side by side.
template <int HD>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  using C = Cfg<HD>;
  constexpr int per = C::COLS / 8;
  return (c / per) * C::CHUNK_BYTES + swz<C::SPAN>(r, c % per);
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

enum : unsigned { kSiteFull = 1, kSitePage = 2, kSiteSlot = 3, kSiteLen = 4 };

// One warp's share of a (sequence, key-value head, tile of query heads):
// running maximum (raw scores), this lane's part of the sum, and O. Lane
// 4 g + t holds rows g and g + 8, columns 8 n + 2 t and the next.
template <int HD>
struct State {
  float m[2], l[2];
  float o[HD / 8][4];

  __device__ __forceinline__ void reset() {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  }
};

// Page numbers of the steps ahead, one step (or half a step, KS = 32 over
// pages of 16) per lane; a page outside the pool is replaced by -1, where TMA
// reads zeros.
template <int HD>
struct Pages {
  static constexpr int KS = Cfg<HD>::KS;
  int ids[KS / 16];
  bool bad;

  // pages of steps first, first + stride, ..., one per lane
  __device__ __forceinline__ void load(const Params& p, const Span<KS>& sp, const int* row, int first, int stride,
                                       int end) {
    const int step = first + static_cast<int>(lane_id()) * stride;
    bad = false;
#pragma unroll
    for (int i = 0; i < KS / 16; ++i) {
      ids[i] = -1;
      if (step < end) {
        const int key = sp.key0(step) + i * 16;
        if (key < sp.len) {
          ids[i] = row[key >> p.page_shift];
          if (ids[i] < 0 || ids[i] >= p.num_pages) {
            ids[i] = -1;
            bad = true;
          }
        }
      }
    }
  }
};

// Loads step `step` (its pages in lane `src` of pg) into `stage`.
template <int HD>
__device__ __forceinline__ void load_step(const Params& p, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                          const Span<Cfg<HD>::KS>& sp, const Pages<HD>& pg, int src, int step, int kvh,
                                          uint8_t* stage, uint64_t* bar) {
  using C = Cfg<HD>;
  int ids[C::KS / 16];
#pragma unroll
  for (int i = 0; i < C::KS / 16; ++i) ids[i] = __shfl_sync(0xffffffffu, pg.ids[i], src);
  if (lane_id() == 0) {
    mbar_arrive_expect_tx(bar, C::STAGE_BYTES);
    const int key = sp.key0(step), in_page = (1 << p.page_shift) - 1;
#pragma unroll
    for (int r = 0; r < C::KS; r += 16) {
      if (r != 0 && p.box_rows != 16) break;  // one box holds the whole step
      const int page = ids[r / 16];
      const int slot = (key + r) & in_page;
#pragma unroll
      for (int c = 0; c < C::CHUNKS; ++c) {
        uint8_t* dst = stage + c * C::CHUNK_BYTES + r * C::SPAN;
        tma_load_4d(dst, map_k, bar, c * C::COLS, slot, kvh, page);
        tma_load_4d(dst + C::TILE_BYTES, map_v, bar, c * C::COLS, slot, kvh, page);
      }
    }
  }
}

// Q rows of query heads [h0, h0 + rows) as m16n8k16 A operands; rows past
// `rows` and columns past the data's head_dim are zero.
template <int HD>
__device__ __forceinline__ void load_q(const Params& p, int b, int h0, int rows, uint32_t (&a)[HD / 16][4]) {
  const int g = static_cast<int>(lane_id()) >> 2, t = static_cast<int>(lane_id()) & 3;
  const __half* base = p.q + b * p.q_stride_b + h0 * p.q_stride_h;
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = g + (i & 1) * 8, c = kk * 16 + (i >> 1) * 8 + t * 2;
      a[kk][i] = (r < rows && c < p.hd) ? *reinterpret_cast<const uint32_t*>(base + r * p.q_stride_h + c) : 0u;
    }
}

// Prepares a step that is not wholly visible or holds the new token: the new
// row goes into the tile, and the value rows of hidden keys become zero, so
// that whatever lies there (never written, or not finite) meets P = 0 as 0.
template <int HD>
__device__ __forceinline__ void patch_step(const Params& p, const Span<Cfg<HD>::KS>& sp, int key0, int b, int kvh,
                                           uint8_t* stage) {
  using C = Cfg<HD>;
  const int lane = static_cast<int>(lane_id());
  const int last = sp.len - 1 - key0;
  if (p.k_new != nullptr && last >= 0 && last < C::KS) {
    for (int c = lane; c < p.hd / 8; c += 32) {
      const int64_t from = b * p.new_stride_b + kvh * p.new_stride_h + c * 8;
      *reinterpret_cast<uint4*>(stage + tile_at<HD>(last, c)) = *reinterpret_cast<const uint4*>(p.k_new + from);
      *reinterpret_cast<uint4*>(stage + C::TILE_BYTES + tile_at<HD>(last, c)) =
          *reinterpret_cast<const uint4*>(p.v_new + from);
    }
  }
  for (int i = lane; i < C::KS * (HD / 8); i += 32) {
    const int r = i / (HD / 8);
    if (!sp.visible(key0 + r))
      *reinterpret_cast<uint4*>(stage + C::TILE_BYTES + tile_at<HD>(r, i % (HD / 8))) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();  // before TMA fills the stage again
  __syncwarp();
}

// One step of KS keys in `stage`. TWO: the tile has more than 8 query heads.
template <int HD, bool TWO>
__device__ __forceinline__ void do_step(const Params& p, const Span<Cfg<HD>::KS>& sp, int key0, bool whole,
                                        uint32_t stage, const uint32_t (&qa)[HD / 16][4], State<HD>& st) {
  using C = Cfg<HD>;
  constexpr int NB = C::KS / 8;
  const int lane = static_cast<int>(lane_id());
  float s[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
  // the four 8x8 tiles of an ldmatrix: keys +0 / +8, columns +0 / +8
  const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
    for (int n = 0; n < NB; n += 2) {
      uint32_t b0, b1, b2, b3;
      ldsm4(stage + tile_at<HD>(n * 8 + kr, kk * 2 + kc), b0, b1, b2, b3);
      mma_16816(s[n], qa[kk], b0, b1);
      mma_16816(s[n + 1], qa[kk], b2, b3);
    }
  if (!whole) {
    const int t = (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!sp.visible(key0 + n * 8 + t + (i & 1))) s[n][i] = -INFINITY;
  }
  constexpr int R = TWO ? 2 : 1;
  float mx[2] = {st.m[0], st.m[1]};
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int n = 0; n < NB; ++n) mx[r] = fmaxf(mx[r], fmaxf(s[n][2 * r], s[n][2 * r + 1]));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
  }
  const bool grew = mx[0] > st.m[0] || (TWO && mx[1] > st.m[1]);
  if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float alpha = st.m[r] == -INFINITY ? 0.f : ex2_approx((st.m[r] - mx[r]) * p.scale_log2);
      st.l[r] *= alpha;
      st.m[r] = mx[r];
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        st.o[n][2 * r] *= alpha;
        st.o[n][2 * r + 1] *= alpha;
      }
    }
  }
  uint32_t pa[NB / 2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r >= R) {
#pragma unroll
      for (int n = 0; n < NB; ++n) pa[n / 2][(n & 1) * 2 + r] = 0u;
      continue;
    }
    const float c = st.m[r] == -INFINITY ? 0.f : -st.m[r] * p.scale_log2;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float p0 = ex2_approx(fmaf(s[n][2 * r], p.scale_log2, c));
      const float p1 = ex2_approx(fmaf(s[n][2 * r + 1], p.scale_log2, c));
      st.l[r] += p0 + p1;
      pa[n / 2][(n & 1) * 2 + r] = pack_half2(p0, p1);
    }
  }
  const int vr = lane & 15, vc = lane >> 4;
#pragma unroll
  for (int n = 0; n < HD / 8; n += 2)
#pragma unroll
    for (int kk = 0; kk < NB / 2; ++kk) {
      uint32_t b0, b1, b2, b3;
      ldsm4_t(stage + C::TILE_BYTES + tile_at<HD>(kk * 16 + vr, n + vc), b0, b1, b2, b3);
      mma_16816(st.o[n], pa[kk], b0, b1);
      mma_16816(st.o[n + 1], pa[kk], b2, b3);
    }
}

// Sequence of batch row b and its length; false when the row is left as it
// is (padding, a bad slot, a refused cache).
__device__ __forceinline__ bool row_of(const Params& p, int b, int* slot, int* len) {
  *slot = p.slots == nullptr ? b : p.slots[b];
  *len = 0;
  if (*slot == -1) return false;
  if (*slot < 0 || *slot >= p.max_seqs) {
    if (threadIdx.x == 0) {
      if (p.status != nullptr) atomicOr(p.status, paged::kBadSlot);
      report_error(kDevCacheRefused, 0xB600u + kSiteSlot);
    }
    return false;
  }
  *len = p.lens[*slot];
  if (*len < 0 || *len > (p.width << p.page_shift)) {
    if (threadIdx.x == 0) {
      if (p.status != nullptr) atomicOr(p.status, paged::kTooLong);
      report_error(kDevCacheRefused, 0xB600u + kSiteLen);
    }
    return false;
  }
  return true;
}

// Writes the new token's key and value of head kvh into its page.
__device__ __forceinline__ void store_new(const Params& p, const int* row, int len, int b, int kvh) {
  const int pos = len - 1, page = row[pos >> p.page_shift];
  if (page < 0 || page >= p.num_pages) return;  // reported by the load of that step
  const int64_t at = page * p.page_stride + kvh * p.head_stride +
                     static_cast<int64_t>(pos & ((1 << p.page_shift) - 1)) * p.hd;
  for (int c = static_cast<int>(lane_id()); c < p.hd / 8; c += 32) {
    const int64_t from = b * p.new_stride_b + kvh * p.new_stride_h + c * 8;
    *reinterpret_cast<uint4*>(p.k_pages + at + c * 8) = *reinterpret_cast<const uint4*>(p.k_new + from);
    *reinterpret_cast<uint4*>(p.v_pages + at + c * 8) = *reinterpret_cast<const uint4*>(p.v_new + from);
  }
}

// One CTA per (b, kv head, tile of up to 16 query heads): warp w takes steps
// w, w + 4, ... and the four results meet in shared memory.
template <int HD, bool TWO>
__global__ void __launch_bounds__(kThreads)
    decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Params p) {
  using C = Cfg<HD>;
  constexpr int KS = C::KS, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kWarps][NST];
  __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = warp_id_uniform(), lane = static_cast<int>(lane_id());
  if (lane == 0) {
    for (int s = 0; s < NST; ++s) mbar_init(&full[warp][s], 1);
    fence_barrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  __syncwarp();
  grid_dep_wait();
  int item = blockIdx.x;
  const int gt = item % p.gtiles;
  item /= p.gtiles;
  const int kvh = item % p.Hkv, b = item / p.Hkv;
  int slot, len;
  const int status = p.status == nullptr ? 0 : *p.status;
  const bool live = row_of(p, b, &slot, &len) && status == 0;
  // status may be set by another CTA of this launch: one answer for the CTA
  if (!__syncthreads_and(live)) return;
  const int h0 = kvh * p.G + gt * kRows, rows = min(kRows, p.G - gt * kRows);
  const int* row = p.table + slot * p.width;
  const Span<KS> sp(p, len);

  uint32_t qa[HD / 16][4];
  load_q<HD>(p, b, h0, rows, qa);
  State<HD> st;
  st.reset();
  uint8_t* ring = smem + warp * C::WARP_BYTES;
  const int mine = sp.steps > warp ? (sp.steps - warp + kWarps - 1) / kWarps : 0;  // steps of this warp
  Pages<HD> pg;
  bool bad = false, ok = true;
  int loaded = 0;  // steps requested so far
  auto request = [&]() {
    if (loaded % 32 == 0) {
      pg.load(p, sp, row, warp + loaded * kWarps, kWarps, sp.steps);
      bad |= pg.bad;
    }
    load_step<HD>(p, &map_k, &map_v, sp, pg, loaded % 32, warp + loaded * kWarps, kvh,
                  ring + (loaded % NST) * C::STAGE_BYTES, &full[warp][loaded % NST]);
    ++loaded;
  };
  for (int i = 0; i < NST && i < mine; ++i) request();
  if (p.k_new != nullptr && gt == 0 && warp == 0 && len > 0) store_new(p, row, len, b, kvh);
  for (int i = 0; i < mine; ++i) {
    const int s = i % NST;
    if (!mbar_wait_warp(&full[warp][s], (i / NST) & 1, nullptr, p.wait_limit_ns)) {
      if (lane == 0) report_error(kDevWaitTimeout, 0xB600u + kSiteFull);
      ok = false;
      break;
    }
    uint8_t* stage = ring + s * C::STAGE_BYTES;
    const int key0 = sp.key0(warp + i * kWarps);
    const bool whole = sp.whole(key0);
    if (!whole || (p.k_new != nullptr && key0 + KS >= sp.len)) patch_step<HD>(p, sp, key0, b, kvh, stage);
    do_step<HD, TWO>(p, sp, key0, whole, smem_u32(stage), qa, st);
    __syncwarp();
    if (loaded < mine) request();
  }
  if (!ok) {
    // let copies already in flight land before the CTA can exit
    for (int i = max(0, loaded - NST); i < loaded; ++i)
      mbar_wait_warp(&full[warp][i % NST], (i / NST) & 1, nullptr, kDrainLimitNs);
  }
  grid_dep_launch();
  if (__any_sync(0xffffffffu, bad) && lane == 0) {
    if (p.status != nullptr) atomicOr(p.status, paged::kBadPage);
    report_error(kDevCacheRefused, 0xB600u + kSitePage);
  }

  // merge: each warp's maximum and sum, then O scaled to the common maximum
  const int g = lane >> 2, t = lane & 3;
  constexpr int R = TWO ? 2 : 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    if (t == 0) {
      sh_m[warp][g + 8 * r] = st.m[r];
      sh_l[warp][g + 8 * r] = st.l[r];
    }
  }
  __syncthreads();  // also: every warp is done with its ring, which O reuses
  float* sh_o = reinterpret_cast<float*>(smem);  // [kWarps][8 R][HD]
  static_assert(kWarps * 8 * 2 * HD * 4 <= C::SMEM_BYTES - 1024, "merge buffer");
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int rr = g + 8 * r;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_m[w][rr]);
    const float f = st.m[r] == -INFINITY ? 0.f : ex2_approx((st.m[r] - top) * p.scale_log2);
    float* dst = sh_o + (warp * 8 * R + rr) * HD;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
      *reinterpret_cast<float2*>(dst + n * 8 + t * 2) = make_float2(st.o[n][2 * r] * f, st.o[n][2 * r + 1] * f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (p.hd / 2); i += kThreads) {
    const int rr = i / (p.hd / 2), c = (i % (p.hd / 2)) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_m[w][rr]);
    float l = 0.f;
    float2 o = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (sh_m[w][rr] != -INFINITY) l += sh_l[w][rr] * ex2_approx((sh_m[w][rr] - top) * p.scale_log2);
      const float2 x = *reinterpret_cast<const float2*>(sh_o + (w * 8 * R + rr) * HD + c);
      o.x += x.x;
      o.y += x.y;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;  // no visible key: zeros
    *reinterpret_cast<uint32_t*>(p.out + b * p.ld_out + (h0 + rr) * p.hd + c) = pack_half2(o.x * inv, o.y * inv);
  }
}

}  // namespace decode
}  // namespace tk

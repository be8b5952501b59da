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
// results are merged. Measured: 4 x 100,000 keys, 16 heads of 64: 264 us (6.2
// TB/s, 0.95 of the copy's rate); 64 sequences, 32 / 8 heads of 128, window
// 2000: 79 us (5.9 TB/s); one sequence of 97 tokens: 3.1 us in a graph.
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

// Tiles of a kernel: KS keys a step, NST stages a warp.
template <int HD_, int KS_, int NST_>
struct Tiles {
  static constexpr int HD = HD_, KS = KS_, NST = NST_;
  static_assert(HD == 16 || HD == 32 || HD == 64 || HD == 128 || HD == 256, "head_dim");
  static constexpr int SPAN = HD >= 64 ? 128 : HD * 2;          // swizzle span, bytes
  static constexpr int COLS = HD >= 64 ? 64 : HD;               // columns of a TMA box
  static constexpr int CHUNKS = HD / COLS;                      // boxes per row
  static constexpr int CHUNK_BYTES = KS * SPAN;                 // [KS, COLS]
  static constexpr int TILE_BYTES = CHUNKS * CHUNK_BYTES;       // K or V of one step
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int SMEM_BYTES = kWarps * NST * STAGE_BYTES + 1024;
  static_assert(CHUNK_BYTES % 1024 == 0, "swizzle atoms");
};

// A step's latency (barrier, products, two shuffles, exponentials: 0.5 us at
// 16 keys, 0.7 at 32, 0.9 at 64, hd 64) is what a lone warp is bound by, so
// steps are as large as leaves the rings room for several warps an SM: 12 with
// 192 KB in flight at hd 64, 4 with 128 KB at hd 128 and 192 KB at hd 256, 16
// with 64 and 128 KB at hd 16 and 32. 32 keys against 16: 8 x 16,384 keys, 16
// heads of 64, one CTA each, 98 us against 150; 8 x 1024, 8 groups of hd 128,
// 11.7 against 16.2; 64 keys lose where CTAs are many (256 short sequences, 48
// us against 29).
template <int HD>
struct Cfg : Tiles<HD, HD == 256 ? 16 : 32, HD == 256 ? 3 : 2> {
  using Base = Tiles<HD, HD == 256 ? 16 : 32, HD == 256 ? 3 : 2>;
  // CTAs per SM: shared memory (the split kernel's other needs are under
  // 10 KB) and 65,536 registers
  static constexpr int BY_SMEM = 228 * 1024 / (Base::SMEM_BYTES + 10 * 1024);
  static constexpr int CTAS = BY_SMEM < 4 ? BY_SMEM : 4;
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
  int* status;            // the cache's status word
  __half* out;            // [B, ld_out], head h at columns [h * hd, h * hd + hd)
  int64_t q_stride_b, q_stride_h, new_stride_b, new_stride_h, page_stride, head_stride, width, ld_out;
  int B, H, Hkv, G, gtiles, max_seqs, num_pages, page_shift;
  int hd;                 // head_dim of the data: HD, or 8 in the HD = 16 kernel (zero-padded by TMA)
  int window, sinks;      // window 0: every key
  float scale_log2;
  uint64_t wait_limit_ns; // 0: every wait for keys gives up at once
  int store_ctas;         // first CTAs of decode_kernel: they store the new tokens (none without k_new)
  // split over the grid (decode_split_kernel)
  int ctas, min_steps;    // CTAs of the grid; fewest steps one takes
  int2* info;             // [B * Hkv * gtiles]: first CTA and number of parts of a split result, (0, 0) if whole
  float* part_ml;         // [2 * ctas][2][kRows]: maximum and sum of a part
  float* part_o;          // [2 * ctas][kRows][HD]
};

// The visible keys of a sequence as a list of KS-key steps: the first
// `sink_steps` steps start at key 0, the others at `lo`, a multiple of KS.
template <int KS>
struct Span {
  int len, first, lo, sinks, sink_steps, steps;  // first = first key of the window

  Span() = default;
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
template <class C>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
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

// Page numbers of the steps ahead, one step per lane, a number for every 16
// keys; a page outside the pool is replaced by -1, where TMA reads zeros.
template <class C>
struct Pages {
  static constexpr int KS = C::KS;
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
template <class C>
__device__ __forceinline__ void load_step(const Params& p, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                          const Span<C::KS>& sp, const Pages<C>& pg, int src, int step, int kvh,
                                          uint8_t* stage, uint64_t* bar) {
  int ids[C::KS / 16];
#pragma unroll
  for (int i = 0; i < C::KS / 16; ++i) ids[i] = __shfl_sync(0xffffffffu, pg.ids[i], src);
  if (lane_id() == 0) {
    mbar_arrive_expect_tx(bar, C::STAGE_BYTES);
    const int key = sp.key0(step), in_page = (1 << p.page_shift) - 1;
#pragma unroll
    for (int r = 0; r < C::KS; r += 16) {
      if (((key + r) & in_page) != 0 && r != 0) continue;  // in the box before: boxes have min(KS, page size) rows
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

// The new token's key and value row of one head, 16 bytes each in lanes
// below hd / 8; loaded before the keys of its step arrive.
struct NewRow {
  uint4 k, v;

  __device__ __forceinline__ void load(const Params& p, int b, int kvh) {
    const int c = static_cast<int>(lane_id());
    if (c >= p.hd / 8) return;
    const int64_t from = b * p.new_stride_b + kvh * p.new_stride_h + c * 8;
    k = *reinterpret_cast<const uint4*>(p.k_new + from);
    v = *reinterpret_cast<const uint4*>(p.v_new + from);
  }
  // into its page; `page` as the table names it
  __device__ __forceinline__ void store(const Params& p, int page, int len, int kvh) const {
    const int c = static_cast<int>(lane_id());
    if (page < 0 || page >= p.num_pages || c >= p.hd / 8) return;  // reported by the load of that step
    const int64_t at = page * p.page_stride + kvh * p.head_stride +
                       static_cast<int64_t>((len - 1) & ((1 << p.page_shift) - 1)) * p.hd + c * 8;
    *reinterpret_cast<uint4*>(p.k_pages + at) = k;
    *reinterpret_cast<uint4*>(p.v_pages + at) = v;
  }
};

// Prepares a step that is not wholly visible or holds the new token: the new
// row goes into the tile, and the value rows of hidden keys become zero, so
// that whatever lies there (never written, or not finite) meets P = 0 as 0.
template <class C>
__device__ __forceinline__ void patch_step(const Params& p, const Span<C::KS>& sp, int key0, const NewRow& row,
                                           uint8_t* stage) {
  constexpr int HD = C::HD;
  const int lane = static_cast<int>(lane_id());
  const int last = sp.len - 1 - key0;
  if (p.k_new != nullptr && last >= 0 && last < C::KS && lane < p.hd / 8) {
    *reinterpret_cast<uint4*>(stage + tile_at<C>(last, lane)) = row.k;
    *reinterpret_cast<uint4*>(stage + C::TILE_BYTES + tile_at<C>(last, lane)) = row.v;
  }
  for (int i = lane; i < C::KS * (HD / 8); i += 32) {
    const int r = i / (HD / 8);
    if (!sp.visible(key0 + r))
      *reinterpret_cast<uint4*>(stage + C::TILE_BYTES + tile_at<C>(r, i % (HD / 8))) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();  // before TMA fills the stage again
  __syncwarp();
}

// One step of KS keys in `stage`. TWO: the tile has more than 8 query heads.
template <class C, bool TWO>
__device__ __forceinline__ void do_step(const Params& p, const Span<C::KS>& sp, int key0, bool whole, uint32_t stage,
                                        const uint32_t (&qa)[C::HD / 16][4], State<C::HD>& st) {
  constexpr int HD = C::HD;
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
      ldsm4(stage + tile_at<C>(n * 8 + kr, kk * 2 + kc), b0, b1, b2, b3);
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
      ldsm4_t(stage + C::TILE_BYTES + tile_at<C>(kk * 16 + vr, n + vc), b0, b1, b2, b3);
      mma_16816(st.o[n], pa[kk], b0, b1);
      mma_16816(st.o[n + 1], pa[kk], b2, b3);
    }
}

// Sequence of batch row b and its length; false when the row is left as it
// is (padding, a bad slot or length, which `report` reports).
__device__ __forceinline__ bool row_ok(const Params& p, int b, int* slot, int* len, bool report) {
  *slot = p.slots == nullptr ? b : p.slots[b];
  *len = 0;
  if (*slot == -1) return false;
  const bool slot_ok = *slot >= 0 && *slot < p.max_seqs;
  if (slot_ok) *len = p.lens[*slot];
  if (slot_ok && *len >= 0 && *len <= (p.width << p.page_shift)) return true;
  if (report) {
    atomicOr(p.status, slot_ok ? paged::kTooLong : paged::kBadSlot);
    report_error(kDevCacheRefused, 0xB600u + (slot_ok ? kSiteLen : kSiteSlot));
  }
  return false;
}

// Merge of the four warps' results. put_state leaves a warp's maximum, sum
// and O (fp32, unnormalised) in shared memory; take_states hands each thread
// its rows' common maximum, sum and column pairs of O.
template <class C, bool TWO>
__device__ __forceinline__ void put_state(State<C::HD>& st, float* o, float* m, float* l) {
  static_assert(kRows * C::HD * 4 <= C::STAGE_BYTES, "a stage holds a warp's O");
  const int g = static_cast<int>(lane_id()) >> 2, t = static_cast<int>(lane_id()) & 3;
#pragma unroll
  for (int r = 0; r < (TWO ? 2 : 1); ++r) {
    float sum = st.l[r];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t == 0) {
      m[g + 8 * r] = st.m[r];
      l[g + 8 * r] = sum;
    }
#pragma unroll
    for (int n = 0; n < C::HD / 8; ++n)
      *reinterpret_cast<float2*>(o + (g + 8 * r) * C::HD + n * 8 + t * 2) =
          make_float2(st.o[n][2 * r], st.o[n][2 * r + 1]);
  }
}

// Warp w's O lies at base + w * pitch + at[w] bytes (at null: 0).
template <class C, class F>
__device__ __forceinline__ void take_states(const Params& p, const uint8_t* base, int pitch, const int* at,
                                            const float (&m)[kWarps][kRows], const float (&l)[kWarps][kRows], int rows,
                                            F&& emit) {
  const int pairs = p.hd / 2;
  for (int i = threadIdx.x; i < rows * pairs; i += kThreads) {
    const int rr = i / pairs, c = (i % pairs) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m[w][rr]);
    float sum = 0.f;
    float2 o = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (m[w][rr] == -INFINITY) continue;  // saw no key (and may not have written its O)
      const float f = ex2_approx((m[w][rr] - top) * p.scale_log2);
      const float2 x = *reinterpret_cast<const float2*>(
          reinterpret_cast<const float*>(base + w * pitch + (at == nullptr ? 0 : at[w])) + rr * C::HD + c);
      sum = fmaf(l[w][rr], f, sum);
      o.x = fmaf(x.x, f, o.x);
      o.y = fmaf(x.y, f, o.y);
    }
    emit(rr, c, top, sum, o);
  }
}

// A wait gave up: the call's output and new tokens are not what they should be,
// so later calls stop at the status word until the caller has put things right.
__device__ __forceinline__ void report_timeout(const Params& p) {
  atomicOr(p.status, paged::kTimedOut);
  report_error(kDevWaitTimeout, 0xB600u + kSiteFull);
}

// The new tokens of a call are stored whole or not at all, by CTAs of their own:
// each looks at every row first -- a slot or a length that cannot be, a sequence
// that two rows name (two new tokens for one place) -- so that all agree, and no
// segment waits for that. The segments take the new token from the argument and
// never see what its place in the page holds. `seen`: a bit per sequence.
// (Checks in every segment's CTA instead: 256 short sequences, 16 heads of 64,
// 29.4 us against 28.6; 1000 of 30 tokens, 4 heads of 32, 15.0 against 7.3.)
__device__ __forceinline__ void store_new_rows(const Params& p, uint32_t* seen) {
  for (int i = threadIdx.x; i < (p.max_seqs + 31) / 32; i += kThreads) seen[i] = 0u;
  grid_dep_wait();
  const int status = *p.status;
  if (__syncthreads_or(status)) return;
  int bad = 0;
  for (int i = threadIdx.x; i < p.B; i += kThreads) {
    const int s = p.slots == nullptr ? i : p.slots[i];
    if (s == -1) continue;
    if (s < 0 || s >= p.max_seqs) {
      bad |= paged::kBadSlot;
      continue;
    }
    if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad |= paged::kBadSlot;
    const int len = p.lens[s];
    if (len < 0 || len > (p.width << p.page_shift)) bad |= paged::kTooLong;
  }
  if (__syncthreads_or(bad)) {
    if (bad) {
      atomicOr(p.status, bad);
      report_error(kDevCacheRefused, 0xB600u + ((bad & paged::kBadSlot) ? kSiteSlot : kSiteLen));
    }
    return;
  }
  const int vecs = p.hd / 8, per_row = p.Hkv * vecs, in_page = (1 << p.page_shift) - 1;
  const int64_t total = static_cast<int64_t>(p.B) * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(p.store_ctas) * kThreads) {
    const int b = static_cast<int>(i / per_row), within = static_cast<int>(i % per_row);
    const int h = within / vecs, c = within % vecs;
    const int s = p.slots == nullptr ? b : p.slots[b];
    if (s == -1) continue;
    const int last = p.lens[s] - 1;
    if (last < 0) continue;
    const int page = p.table[s * p.width + (last >> p.page_shift)];
    if (page < 0 || page >= p.num_pages) continue;  // reported by the segment that reads it
    const int64_t from = b * p.new_stride_b + h * p.new_stride_h + c * 8;
    const int64_t to = page * p.page_stride + h * p.head_stride + static_cast<int64_t>(last & in_page) * p.hd + c * 8;
    *reinterpret_cast<uint4*>(p.k_pages + to) = *reinterpret_cast<const uint4*>(p.k_new + from);
    *reinterpret_cast<uint4*>(p.v_pages + to) = *reinterpret_cast<const uint4*>(p.v_new + from);
  }
}

// WPS warps per segment (b, kv head, tile of up to 16 query heads): with 4 a
// CTA has one segment, warp w takes steps w, w + 4, ... and the four results
// meet in shared memory; with 1 each warp has its own and nothing is merged.
// With new tokens the grid's first store_ctas CTAs store them.
template <int HD, bool TWO, int WPS>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::CTAS)
    decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Params p) {
  using C = Cfg<HD>;
  constexpr int KS = C::KS, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  if (blockIdx.x < static_cast<unsigned>(p.store_ctas)) {
    store_new_rows(p, reinterpret_cast<uint32_t*>(smem_raw));
    return;
  }
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
  const int cta = static_cast<int>(blockIdx.x) - p.store_ctas;
  int item = WPS == 1 ? cta * kWarps + warp : cta;
  const int gt = item % p.gtiles;
  item /= p.gtiles;
  const int kvh = item % p.Hkv, b = item / p.Hkv;
  int slot = -1, len = 0;
  bool live = false;
  if (b < p.B && *p.status == 0) live = row_ok(p, b, &slot, &len, WPS == 1 ? lane == 0 : threadIdx.x == 0);
  // status may be set by another CTA of this launch: one answer for the segment
  if (WPS == 1 ? !__all_sync(0xffffffffu, live) : !__syncthreads_and(live)) return;
  const int h0 = kvh * p.G + gt * kRows, rows = min(kRows, p.G - gt * kRows);
  const int* row = p.table + slot * p.width;
  const Span<KS> sp(p, len);
  const int first = WPS == 1 ? 0 : warp;
  const int mine = sp.steps > first ? (sp.steps - first + WPS - 1) / WPS : 0;  // steps of this warp

  uint8_t* ring = smem + warp * NST * C::STAGE_BYTES;
  Pages<C> pg;
  bool bad = false, ok = mine == 0 || p.wait_limit_ns != 0;
  int loaded = 0;  // steps requested so far
  auto request = [&]() {
    if (loaded % 32 == 0) {
      pg.load(p, sp, row, first + loaded * WPS, WPS, sp.steps);
      bad |= pg.bad;
    }
    load_step<C>(p, &map_k, &map_v, sp, pg, loaded % 32, first + loaded * WPS, kvh,
                 ring + (loaded % NST) * C::STAGE_BYTES, &full[warp][loaded % NST]);
    ++loaded;
  };
  for (int i = 0; i < NST && i < mine; ++i) request();
  uint32_t qa[HD / 16][4];
  load_q<HD>(p, b, h0, rows, qa);
  NewRow new_row;
  const bool has_new = p.k_new != nullptr && mine > 0 && (sp.steps - 1) % WPS == first;  // the last step is mine
  if (has_new) new_row.load(p, b, kvh);
  State<HD> st;
  st.reset();
  for (int i = 0; ok && i < mine; ++i) {
    const int s = i % NST;
    ok = mbar_wait_warp(&full[warp][s], (i / NST) & 1, nullptr, p.wait_limit_ns);
    if (!ok) break;
    uint8_t* stage = ring + s * C::STAGE_BYTES;
    const int key0 = sp.key0(first + i * WPS);
    const bool whole = sp.whole(key0);
    if (!whole || (has_new && i + 1 == mine)) patch_step<C>(p, sp, key0, new_row, stage);
    do_step<C, TWO>(p, sp, key0, whole, smem_u32(stage), qa, st);
    __syncwarp();
    if (loaded < mine) request();
  }
  if (!ok) {
    if (lane == 0) report_timeout(p);
    // let copies already in flight land before the CTA can exit
    for (int i = max(0, loaded - NST); i < loaded; ++i)
      mbar_wait_warp(&full[warp][i % NST], (i / NST) & 1, nullptr, kDrainLimitNs);
  }
  grid_dep_launch();
  if (__any_sync(0xffffffffu, bad) && lane == 0) {
    atomicOr(p.status, paged::kBadPage);
    report_error(kDevCacheRefused, 0xB600u + kSitePage);
  }
  if (WPS == 1) {
    if (!ok) return;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < (TWO ? 2 : 1); ++r) {
      float l = st.l[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const float inv = l > 0.f ? 1.f / l : 0.f;  // no visible key: zeros
      const int rr = g + 8 * r;
      __half* dst = p.out + b * p.ld_out + (h0 + rr) * p.hd + t * 2;
      if (rr < rows) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
          if (n * 8 < p.hd)
            *reinterpret_cast<uint32_t*>(dst + n * 8) = pack_half2(st.o[n][2 * r] * inv, st.o[n][2 * r + 1] * inv);
      }
    }
    return;
  }
  // every warp is done with its ring, which the merge reuses, and has seen all its keys
  if (!__syncthreads_and(ok)) return;
  put_state<C, TWO>(st, reinterpret_cast<float*>(ring), sh_m[warp], sh_l[warp]);
  __syncthreads();
  take_states<C>(p, smem, NST * C::STAGE_BYTES, nullptr, sh_m, sh_l, rows, [&](int rr, int c, float, float l, float2 o) {
    const float inv = l > 0.f ? 1.f / l : 0.f;  // no visible key: zeros
    *reinterpret_cast<uint32_t*>(p.out + b * p.ld_out + (h0 + rr) * p.hd + c) = pack_half2(o.x * inv, o.y * inv);
  });
}

// ----------------------------------------------------------------------------
// Long caches, ragged lengths: the steps of all (b, kv head, query-head tile)
// segments, in that order, are one list, cut into equal ranges for the CTAs of
// a grid that fills the GPU. A CTA walks the parts of segments in its range;
// its four warps take every fourth step of a part, so that together they read
// neighbouring keys (DRAM pages), and their rings run on from part to part.
// After a part the warps merge; a segment that lies inside a range is done
// then, one that crosses a border leaves a part (maximum, sum, unnormalised O,
// fp32) per CTA in the workspace -- slot 0 of a CTA for a segment that began
// before its range, slot 1 for one that begins in it -- and join_kernel adds
// the parts in order, so the result does not depend on which CTA ends first.
// ----------------------------------------------------------------------------
constexpr int kMaxRows = 512;  // rows whose lengths a CTA keeps in shared memory

// A part: steps [s0, s1) of segment sg of row b; `left` steps of the CTA's
// range follow it.
template <class C>
struct Part {
  Span<C::KS> sp;
  int b, sg, s0, s1;
  int64_t left;

  __device__ __forceinline__ void enter(const Params& p, const int* sh_len) { sp = Span<C::KS>(p, sh_len[b]); }
  __device__ __forceinline__ void cut(int from, int64_t steps) {
    s0 = from;
    s1 = sp.steps - from < steps ? sp.steps : from + static_cast<int>(steps);
    left = steps - (s1 - s0);
  }
  __device__ __forceinline__ bool last() const { return s1 == sp.steps; }
  // the part that follows; false at the end of the range
  __device__ __forceinline__ bool next(const Params& p, const int* sh_len, int segs) {
    if (left == 0) return false;
    if (++sg == segs) {
      sg = 0;
      do ++b;
      while (sh_len[b] <= 0);
      enter(p, sh_len);
    }
    cut(0, left);
    return true;
  }
};

template <int HD, bool TWO>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::CTAS)
    decode_split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        Params p) {
  using C = Cfg<HD>;
  constexpr int KS = C::KS, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kWarps][NST];
  __shared__ int64_t sh_first[kMaxRows + 1];  // steps of one segment each of the rows before
  __shared__ int sh_len[kMaxRows], sh_slot[kMaxRows];
  __shared__ uint32_t sh_seen[paged::kMaxEntries / 32];  // sequences that get a new token
  __shared__ int64_t sh_sum[kWarps];
  __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
  __shared__ int sh_at[kWarps];
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
  const int status = *p.status;
  if (__syncthreads_or(status)) return;  // join_kernel then returns as well
  const int segs = p.Hkv * p.gtiles;
  const bool check_twice = p.k_new != nullptr && p.slots != nullptr;
  if (check_twice) {
    for (int i = threadIdx.x; i < (p.max_seqs + 31) / 32; i += kThreads) sh_seen[i] = 0u;
    __syncthreads();
  }
  bool twice = false, wrong = false;

  // lengths and the exclusive prefix sum of the rows' steps
  int64_t carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int slot = -1, len = 0;
    int64_t x = 0;
    if (b < p.B) {
      if (!row_ok(p, b, &slot, &len, blockIdx.x == 0)) {
        len = -1;  // left as it is
        wrong |= slot != -1;
      } else if (check_twice) twice |= atomicOr(&sh_seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1u;
      x = len > 0 ? Span<KS>(p, len).steps : 0;
      sh_len[b] = len;
      sh_slot[b] = slot;
    }
    const int64_t own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sh_sum[warp] = x;
    __syncthreads();
    int64_t before = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh_sum[w];
      carry += sh_sum[w];
    }
    if (b < p.B) sh_first[b] = before + x - own;
    __syncthreads();
  }
  // in every CTA: a row that cannot be, two new tokens for one place
  if (p.k_new != nullptr && __syncthreads_or(twice || wrong)) {
    if (twice && blockIdx.x == 0) {
      atomicOr(p.status, paged::kBadSlot);
      report_error(kDevCacheRefused, 0xB600u + kSiteSlot);
    }
    return;
  }
  const int64_t total = carry * segs;
  // rows without keys: zeros for an empty sequence, nothing for the others
  for (int b = blockIdx.x; b < p.B; b += p.ctas) {
    if (sh_len[b] > 0) continue;
    for (int i = threadIdx.x; i < segs; i += kThreads) p.info[b * segs + i] = make_int2(0, 0);
    if (sh_len[b] == 0)
      for (int i = threadIdx.x; i < p.H * p.hd / 2; i += kThreads)
        *reinterpret_cast<uint32_t*>(p.out + b * p.ld_out + 2 * i) = 0u;
  }
  const int64_t even = (total + p.ctas - 1) / p.ctas;
  const int64_t per = even > p.min_steps ? even : p.min_steps;
  const int64_t r0 = blockIdx.x * per, r1 = r0 + per < total ? r0 + per : total;
  if (r0 >= r1) return;

  Part<C> use;  // the part that the warps work on
  {
    int lo = 0, hi = p.B;  // sh_first[lo] * segs <= r0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh_first[mid] * segs <= r0) lo = mid;
      else hi = mid;
    }
    use.b = lo;  // a row without keys shares its start with the row behind it, so this one has some
    use.enter(p, sh_len);
    const int64_t within = r0 - sh_first[use.b] * segs;
    use.sg = static_cast<int>(within / use.sp.steps);
    use.cut(static_cast<int>(within % use.sp.steps), r1 - r0);
  }
  Part<C> get = use;  // the part of the next step that this warp requests
  int get_step = get.s0 + warp;
  bool more = true;
  auto settle = [&]() {  // short parts may have no step for this warp
    while (more && get_step >= get.s1) {
      more = get.next(p, sh_len, segs);
      get_step = warp;
    }
  };
  settle();
  uint8_t* ring = smem + warp * NST * C::STAGE_BYTES;
  Pages<C> pg;
  int pg_b = -1, pg_step = 0;  // row and first step whose pages pg holds (every fourth step)
  bool bad = false, ok = p.wait_limit_ns != 0;
  int loaded = 0, used = 0;
  auto request = [&]() {
    const int ahead = get_step - pg_step;
    if (get.b != pg_b || ahead < 0 || ahead >= 32 * kWarps || ahead % kWarps != 0) {
      pg_b = get.b;
      // from the row's start where that holds this step too: its next segments begin there
      pg_step = get_step < 16 * kWarps ? get_step % kWarps : get_step;
      pg.load(p, get.sp, p.table + sh_slot[get.b] * p.width, pg_step, kWarps, get.sp.steps);
      bad |= pg.bad;
    }
    load_step<C>(p, &map_k, &map_v, get.sp, pg, (get_step - pg_step) / kWarps, get_step, get.sg / p.gtiles,
                 ring + (loaded % NST) * C::STAGE_BYTES, &full[warp][loaded % NST]);
    ++loaded;
    get_step += kWarps;
    settle();
  };
  for (int i = 0; i < NST && more; ++i) request();

  uint32_t qa[HD / 16][4];
  State<HD> st;
  NewRow new_row;
  int64_t done = r0;  // steps of the list before the current part
  for (bool go = true; go; go = use.next(p, sh_len, segs)) {
    const int kvh = use.sg / p.gtiles, gt = use.sg % p.gtiles;
    const int h0 = kvh * p.G + gt * kRows, rows = min(kRows, p.G - gt * kRows);
    load_q<HD>(p, use.b, h0, rows, qa);
    // the new token is in the last step, which one of the warps has
    const bool has_new = p.k_new != nullptr && use.last() && (use.s1 - 1 - use.s0) % kWarps == warp;
    int page = -1;
    if (has_new) {
      new_row.load(p, use.b, kvh);
      page = p.table[sh_slot[use.b] * p.width + ((use.sp.len - 1) >> p.page_shift)];
    }
    st.reset();
    int held = 0;  // stage of this warp's last step, which holds its O during the merge
    bool hold = false;
    for (int step = use.s0 + warp; step < use.s1; step += kWarps) {
      const int s = used % NST;
      // a warp that gave up only keeps the others company at the barriers
      if (ok) ok = mbar_wait_warp(&full[warp][s], (used / NST) & 1, nullptr, p.wait_limit_ns);
      if (!ok) continue;
      ++used;
      uint8_t* stage = ring + s * C::STAGE_BYTES;
      const int key0 = use.sp.key0(step);
      const bool whole = use.sp.whole(key0), last = step + kWarps >= use.s1;
      if (!whole || (has_new && last)) patch_step<C>(p, use.sp, key0, new_row, stage);
      do_step<C, TWO>(p, use.sp, key0, whole, smem_u32(stage), qa, st);
      __syncwarp();
      if (last) {
        held = s * C::STAGE_BYTES;
        hold = true;
      } else if (more) {
        request();
      }
    }
    if (has_new && ok && gt == 0) new_row.store(p, page, use.sp.len, kvh);
    // merge; a warp without a step has maximum -inf and leaves the ring alone
    if (hold) {
      put_state<C, TWO>(st, reinterpret_cast<float*>(ring + held), sh_m[warp], sh_l[warp]);
      fence_proxy_async_smem();  // before TMA fills the stage again
    } else if (lane < kRows) {
      sh_m[warp][lane] = -INFINITY;
    }
    if (lane == 0) sh_at[warp] = held;
    const bool all_ok = __syncthreads_and(ok);
    const bool begins = use.s0 == 0, ends = use.last();
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (begins ? 1 : 0);
    if (all_ok)
      take_states<C>(p, smem, NST * C::STAGE_BYTES, sh_at, sh_m, sh_l, rows,
                     [&](int rr, int c, float m, float l, float2 o) {
                       if (begins && ends) {
                         const float inv = l > 0.f ? 1.f / l : 0.f;
                         *reinterpret_cast<uint32_t*>(p.out + use.b * p.ld_out + (h0 + rr) * p.hd + c) =
                             pack_half2(o.x * inv, o.y * inv);
                       } else {
                         if (c == 0) {
                           p.part_ml[slot * 2 * kRows + rr] = m;
                           p.part_ml[slot * 2 * kRows + kRows + rr] = l;
                         }
                         *reinterpret_cast<float2*>(p.part_o + (slot * kRows + rr) * HD + c) = o;
                       }
                     });
    if (begins && threadIdx.x == 0) {
      const int parts = static_cast<int>((done + use.sp.steps - r0 + per - 1) / per);
      p.info[use.b * segs + use.sg] = ends ? make_int2(0, 0) : make_int2(blockIdx.x, parts);
    }
    done += use.s1 - use.s0;
    __syncthreads();  // the merge has read the held stages
    if (hold && ok && more) request();
  }
  if (!ok) {
    if (lane == 0) report_timeout(p);  // join_kernel returns: parts are missing
    // let copies already in flight land before the CTA can exit
    for (int i = max(0, loaded - NST); i < loaded; ++i)
      mbar_wait_warp(&full[warp][i % NST], (i / NST) & 1, nullptr, kDrainLimitNs);
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) {
    atomicOr(p.status, paged::kBadPage);
    report_error(kDevCacheRefused, 0xB600u + kSitePage);
  }
}

// One CTA per segment and query head: the parts of a split result, scaled to
// their common maximum and added in order. Threads take a column pair each;
// the parts are spread over the remaining threads. blockDim is 1024 where few
// segments have many parts, else 256.
constexpr int kJoinThreads = 1024;

template <int HD>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(Params p) {
  constexpr int PAIRS = HD / 2;
  __shared__ float2 sh_o[kJoinThreads];  // [LANES][PAIRS]
  __shared__ float sh_m[kJoinThreads / 32], sh_l[kJoinThreads / PAIRS];
  const int LANES = blockDim.x / PAIRS;
  grid_dep_wait();
  if (*p.status != 0) return;
  const int2 info = p.info[blockIdx.x];
  const int n = info.y;
  if (n == 0) return;
  const int segs = p.Hkv * p.gtiles;
  const int b = blockIdx.x / segs, sg = blockIdx.x % segs;
  const int rr = blockIdx.y, h = (sg / p.gtiles) * p.G + (sg % p.gtiles) * kRows + rr;
  if ((sg % p.gtiles) * kRows + rr >= p.G) return;
  // part i: slot 1 of the first CTA, slot 0 of those after it
  auto slot_of = [&](int i) { return 2 * static_cast<int64_t>(info.x + i) + (i == 0 ? 1 : 0); };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < n; i += blockDim.x) top = fmaxf(top, p.part_ml[slot_of(i) * 2 * kRows + rr]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sh_m[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) top = fmaxf(top, sh_m[w]);
  const int c = threadIdx.x % PAIRS, k = threadIdx.x / PAIRS;
  float2 o = make_float2(0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int i = k; i < n; i += LANES) {
    const int64_t slot = slot_of(i);
    const float m = p.part_ml[slot * 2 * kRows + rr];
    const float f = m == -INFINITY ? 0.f : ex2_approx((m - top) * p.scale_log2);
    const float2 x = *reinterpret_cast<const float2*>(p.part_o + (slot * kRows + rr) * HD + 2 * c);
    l = fmaf(p.part_ml[slot * 2 * kRows + kRows + rr], f, l);
    o.x = fmaf(x.x, f, o.x);
    o.y = fmaf(x.y, f, o.y);
  }
  sh_o[threadIdx.x] = o;
  if (c == 0) sh_l[k] = l;
  __syncthreads();
  if (threadIdx.x < PAIRS && 2 * static_cast<int>(threadIdx.x) < p.hd) {
    o = make_float2(0.f, 0.f);
    l = 0.f;
    for (int i = 0; i < LANES; ++i) {
      o.x += sh_o[i * PAIRS + threadIdx.x].x;
      o.y += sh_o[i * PAIRS + threadIdx.x].y;
      l += sh_l[i];
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    *reinterpret_cast<uint32_t*>(p.out + b * p.ld_out + h * p.hd + 2 * threadIdx.x) =
        pack_half2(o.x * inv, o.y * inv);
  }
}

}  // namespace decode
}  // namespace tk

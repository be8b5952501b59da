// Causal attention of a prompt with a sliding window and a few first tokens
// that stay visible.
//
//   out[b, i, h] = sum_j softmax_j(scale * q_i . k_j) v_j  over the keys
//   j <= i, j < kv_len[b], and i - j < window or j < sinks
//
// q [B, H, S, hd], k and v [B, Hkv, S, hd] (query head h reads key-value head
// h / (H / Hkv)), out [B, S, H * hd]; a row that sees no key is zero.
//
// The work is the band's: a query tile of 128 rows reads the key tiles of
// [tile - window, tile] and those of the first tokens, 4 * hd operations per
// visible pair, and never touches the tiles in between. Same roles, barriers
// and softmax as attn_fwd_kernel (tk_attn.cuh): persistent CTAs, 12 warps --
// TMA, MMA issuer, one that cleans partial value tiles, one idle, then two
// softmax groups of four warps with one query row per thread, each group on
// one of the item's two query tiles, sharing every key and value tile. What
// differs:
//  - an item's steps are the tiles of the first tokens, then the tiles from
//    the window's start; the second query tile's window starts one tile
//    later, so its group skips the first window tile (unless it holds first
//    tokens);
//  - a score row is masked by three bounds (causal and length from above, the
//    window from below, the first tokens), combined into one bit per column;
//    tiles inside the band take the unmasked path;
//  - keys and values move through one ring of tile slots (K_j, V_j, K_j+1,
//    ...), each released on its own;
//  - hd 128: the score and output tiles of two groups fill TMEM, so P_g
//    overwrites the first half of S_g, and S_g of the next step is issued once
//    P_g's product is complete; hd 256: one query tile per item.
// Bound by the softmax warps' latency (hd <= 64: the SFU, the busiest pipe, is
// at 56%, the tensor pipe at 37%; a quarter of the exponentials go on the FMA
// pipe, none cost +2%, half +12%) and by the chain scores -> softmax -> product
// of a group (hd 128: tensor pipe 48%, SFU 37%). Measured under steady load, in
// brackets ten calls after a pause, before the clock falls: one prompt of
// 100,000 tokens, 16 heads of 64, window 4096: 2.48 ms, 673 TFLOP/s of visible
// pairs (2.21, 755); 4 x 8191, 32 / 8 heads of 128, window 1024: 0.74 ms, 707
// (0.64, 815); 4 x 8191, 16 / 4 heads of 256, window 1024: 0.83 ms, 630 (0.76).
//
// Value rows at and past kv_len are zeroed in shared memory before the product
// reads them: their P is 0, but 0 times what they hold may not be (keys need
// no such care, masked scores are never used).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "tk_attn.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace attn {
namespace win {

struct Params {
  __half* out;          // [B, S, ld_out] fp16, head h at columns [h * hd, h * hd + hd)
  int64_t ld_out;
  int B, S, H, G;       // G = H / Hkv
  int window, sinks;    // window >= 1
  int pair_heads;       // the groups of an item take two heads of one tile (G even), else two tiles of one head
  float scale_log2;
  const int* kv_len;    // optional [B]
  int q_heads_inner, kv_heads_inner;  // tensor-map dim order, as attn::Params
  int hd;               // head_dim of the data: HD, or 8 in the HD = 16 kernel (zero-padded by TMA)
  uint64_t wait_limit_ns;
};

template <int HD>
struct Cfg {
  static_assert(HD == 16 || HD == 32 || HD == 64 || HD == 128 || HD == 256, "head_dim");
  static constexpr int GROUPS = HD == 256 ? 1 : 2;              // query tiles of an item
  static constexpr bool P_OVER_S = HD == 128;
  static constexpr int COLS = HD >= 64 ? 64 : HD;               // columns of a TMA box
  static constexpr int NC = HD / COLS;                          // boxes (chunks) of a tile
  static constexpr int ROW_BYTES = COLS * 2;                    // swizzle span
  static constexpr SmemLayout LAYOUT = COLS == 64 ? kLayoutSW128 : COLS == 32 ? kLayoutSW64 : kLayoutSW32;
  static constexpr int SBO = 8 * ROW_BYTES;
  static constexpr int CHUNK_BYTES = kBM * ROW_BYTES;
  static constexpr int TILE_BYTES = NC * CHUNK_BYTES;           // Q, K or V tile
  static constexpr int QSETS = HD >= 128 ? 1 : 2;
  static constexpr int SLOTS = HD == 256 ? 2 : HD == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int SMEM_BYTES = TILE_BYTES * (QSETS * GROUPS + SLOTS) + 1024;
  static_assert(SMEM_BYTES <= 232448, "shared memory");
  // TMEM columns of group g: S, P (packed fp16 pairs), O
  static constexpr int col_s(int g) { return g * kBN; }
  static constexpr int col_p(int g) { return P_OVER_S ? g * kBN : HD == 256 ? 128 : 256 + 64 * g; }
  static constexpr int col_o(int g) { return P_OVER_S ? 256 + 128 * g : HD == 256 ? 192 : 384 + 64 * g; }
};

enum : unsigned { kSiteQ = 1, kSiteSlot = 2, kSiteS = 3, kSiteP = 4, kSiteO = 5, kSiteEmpty = 6, kSiteOFree = 7,
                  kSiteQEmpty = 8, kSitePv = 9, kSiteSFree = 10, kSiteClean = 11 };

// One work item: group 0 takes head h of sequence b and query tile tq0, group 1
// (has1) head h + dh and tile tq0 + dq, one of them 0 and the other 1. Two heads
// of one key-value head need the same key tiles; two tiles of one head need one
// tile more than either.
// Step j works on key tile tile(j); group 0 takes steps j < n0, group 1 all
// but `skip`.
struct Item {
  int b, h, tq0, dh, dq, kv_bound;
  int n_sink, lo;       // steps of the first tokens' tiles; first window tile
  int n, n0, n1, skip;
  int dirty;            // step whose value tile reaches past kv_len (-1: none)
  bool has1;

  __device__ __forceinline__ int tile(int j) const { return j < n_sink ? j : lo + j - n_sink; }
  __device__ __forceinline__ bool uses(int g, int j) const { return g == 0 ? j < n0 : (has1 && j != skip); }
};

template <int GROUPS>
__device__ __forceinline__ Item make_item(const Params& p, int idx, int q_tiles, int q_items) {
  Item it;
  const bool pair = GROUPS == 2 && p.pair_heads;
  it.dh = pair ? 1 : 0;
  it.dq = 1 - it.dh;
  const int heads = p.H >> it.dh, bh_count = p.B * heads;
  const int bh = idx % bh_count;
  it.b = bh / heads;
  it.h = (bh % heads) << it.dh;
  // full windows first, the first rows' short ones last
  it.tq0 = (pair ? 1 : GROUPS) * (q_items - 1 - idx / bh_count);
  it.has1 = pair || (GROUPS == 2 && it.tq0 + 1 < q_tiles);
  it.kv_bound = p.S;
  if (p.kv_len != nullptr) it.kv_bound = max(0, min(p.S, p.kv_len[it.b]));
  const int n_kv = (it.kv_bound + kBN - 1) / kBN;
  const int sink_tiles = (min(p.sinks, it.kv_bound) + kBN - 1) / kBN;
  it.lo = max(0, it.tq0 * kBM - p.window + 1) / kBN;
  const int lo1 = max(0, (it.tq0 + it.dq) * kBM - p.window + 1) / kBN;
  const int hi0 = min(it.tq0, n_kv - 1), hi1 = it.has1 ? min(it.tq0 + it.dq, n_kv - 1) : hi0;
  it.n_sink = min(sink_tiles, it.lo);
  it.n = it.n_sink + max(0, hi1 - it.lo + 1);
  it.n0 = it.n - (hi1 - hi0);
  it.skip = (it.has1 && lo1 > it.lo && it.lo >= sink_tiles && it.lo <= hi1) ? it.n_sink : -1;
  it.n1 = it.has1 ? it.n - (it.skip >= 0 ? 1 : 0) : 0;
  it.dirty = -1;
  if (it.kv_bound < p.S && it.kv_bound % kBN != 0) {
    const int t = n_kv - 1;  // kv_bound > 0 here
    if (t < it.n_sink) it.dirty = t;
    else if (t >= it.lo && t <= hi1) it.dirty = it.n_sink + t - it.lo;
  }
  return it;
}

template <int HD>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int heads_inner,
                                          int row, int h, int b) {
  using C = Cfg<HD>;
#pragma unroll
  for (int c = 0; c < C::NC; ++c) {
    if (heads_inner)
      tma_load_4d(dst + c * C::CHUNK_BYTES, map, bar, c * C::COLS, h, row, b);
    else
      tma_load_4d(dst + c * C::CHUNK_BYTES, map, bar, c * C::COLS, row, h, b);
  }
}

// Shared-memory matrix descriptor whose start moves by constants: only its low
// word changes (addresses stay below 2^18, so the 14-bit field never carries).
// One thread issues every product, and what it executes between two of them
// adds up: rebuilding both descriptors each time and splitting P V into 64
// columns made the issuer the slowest role at hd 128.
struct Desc {
  uint32_t lo, hi;

  __device__ __forceinline__ Desc(uint32_t addr, uint32_t lbo, uint32_t sbo, SmemLayout layout) {
    const uint64_t d = smem_desc(addr, lbo, sbo, layout);
    lo = static_cast<uint32_t>(d);
    hi = static_cast<uint32_t>(d >> 32);
  }
  __device__ __forceinline__ uint64_t at(int bytes) const {
    return (static_cast<uint64_t>(hi) << 32) | (lo + static_cast<uint32_t>(bytes >> 4));
  }
};

// Whether phase `parity` of `bar` is complete, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// The lowest n bits of a word (n clamped to 0..32).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attn_window_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, Params p) {
  using C = Cfg<HD>;
  constexpr int SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[C::QSETS];
  __shared__ __align__(8) uint64_t q_empty[C::QSETS];
  __shared__ __align__(8) uint64_t slot_full[SLOTS];
  __shared__ __align__(8) uint64_t slot_empty[SLOTS];
  __shared__ __align__(8) uint64_t s_full[2];      // per softmax group
  __shared__ __align__(8) uint64_t p_full[2];
  __shared__ __align__(8) uint64_t o_full[2];
  __shared__ __align__(8) uint64_t o_free[2];
  __shared__ __align__(8) uint64_t pv_done[2];
  __shared__ __align__(8) uint64_t s_free[2];
  __shared__ __align__(8) uint64_t v_dirty;
  __shared__ __align__(8) uint64_t v_clean;
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_flag;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                           // QSETS x GROUPS tiles
  uint8_t* sR = smem + C::QSETS * C::GROUPS * C::TILE_BYTES;    // SLOTS tiles

  const int warp = warp_id_uniform();
  const uint32_t lane = lane_id();
  const int q_tiles = (p.S + kBM - 1) / kBM;
  const bool pair = C::GROUPS == 2 && p.pair_heads;
  const int q_items = pair ? q_tiles : (q_tiles + C::GROUPS - 1) / C::GROUPS;
  const int n_items = q_items * p.B * (pair ? p.H / 2 : p.H);
  const unsigned kid = 0xC0u + HD / 16;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::QSETS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&slot_full[s], 1);
      mbar_init(&slot_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
      mbar_init(&o_full[g], 1);
      mbar_init(&o_free[g], 4);
      mbar_init(&pv_done[g], 1);
      mbar_init(&s_free[g], 4);
    }
    mbar_init(&v_dirty, 1);
    mbar_init(&v_clean, 1);
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  grid_dep_wait();  // the previous kernel's outputs are complete and visible

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    if (warp == 0) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        prefetch_tensormap(&map_q);
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        int n = 0;   // tiles loaded so far (ring position): K of a step, then its V
        int qn = 0;  // items with work loaded so far
        bool ok = true;
        for (int idx = blockIdx.x; idx < n_items && ok; idx += gridDim.x) {
          const Item it = make_item<C::GROUPS>(p, idx, q_tiles, q_items);
          if (it.n == 0) continue;
          const int qs = qn % C::QSETS;
          const uint32_t q_phase = (qn / C::QSETS) & 1;
          ++qn;
          if (!mbar_wait(&q_empty[qs], q_phase ^ 1u, &abort_flag, p.wait_limit_ns)) {
            report_error(kDevWaitTimeout, kid * 256 + kSiteQEmpty);
            abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t* q_dst = sQ + qs * C::GROUPS * C::TILE_BYTES;
          mbar_arrive_expect_tx(&q_full[qs], C::TILE_BYTES * (it.has1 ? 2 : 1));
          load_tile<HD>(q_dst, &map_q, &q_full[qs], p.q_heads_inner, it.tq0 * kBM, it.h, it.b);
          if (it.has1)
            load_tile<HD>(q_dst + C::TILE_BYTES, &map_q, &q_full[qs], p.q_heads_inner, (it.tq0 + it.dq) * kBM,
                          it.h + it.dh, it.b);
          const int kvh = it.h / p.G;
          for (int j = 0; j < 2 * it.n; ++j, ++n) {
            const int s = n % SLOTS;
            if (!mbar_wait(&slot_empty[s], ((n / SLOTS) & 1) ^ 1u, &abort_flag, p.wait_limit_ns)) {
              report_error(kDevWaitTimeout, kid * 256 + kSiteEmpty);
              abort_flag = 1;
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&slot_full[s], C::TILE_BYTES);
            load_tile<HD>(sR + s * C::TILE_BYTES, (j & 1) ? &map_v : &map_k, &slot_full[s], p.kv_heads_inner,
                          it.tile(j >> 1) * kBN, kvh, it.b);
          }
        }
        // all of this CTA's loads are issued: the next kernel may be scheduled
        grid_dep_launch();
        if (!ok) {
          // let copies already in flight land before the CTA can exit
          for (int t = max(0, n - SLOTS); t < n; ++t)
            mbar_wait(&slot_full[t % SLOTS], (t / SLOTS) & 1, nullptr, kDrainLimitNs);
          for (int t = max(0, qn - C::QSETS); t < qn; ++t)
            mbar_wait(&q_full[t % C::QSETS], (t / C::QSETS) & 1, nullptr, kDrainLimitNs);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      if (lane == 0) {
        constexpr uint32_t idesc_s = idesc_f16_f32(kBM, kBN, false, false);
        constexpr uint32_t idesc_o = idesc_f16_f32(kBM, HD, false, true);
        struct Group {
          int tiles = 0;     // products P V issued (p_full, pv_done phases)
          int o_uses = 0;    // items in which O_g was accumulated (o_full / o_free phases)
          int s_issued = 0;  // S_g issued (s_free phases)
          int in_item = 0;   // products of the current item
        };
        Group grp0, grp1;
        int base = 0;      // ring position of the item's first tile
        int qn = 0;
        int turns = 0, taken = 0;  // cleaner's turns given (v_dirty) and seen ended (v_clean)
        bool ok = true;
        auto fail = [&](unsigned site) {
          report_error(kDevWaitTimeout, kid * 256 + site);
          ok = false;
        };
        auto wait_tile = [&](int t) -> bool {
          if (mbar_wait(&slot_full[t % SLOTS], (t / SLOTS) & 1, &abort_flag, p.wait_limit_ns)) return true;
          fail(kSiteSlot);
          return false;
        };
        for (int idx = blockIdx.x; idx < n_items && ok; idx += gridDim.x) {
          const Item it = make_item<C::GROUPS>(p, idx, q_tiles, q_items);
          if (it.n == 0) continue;
          const int qs = qn % C::QSETS;
          const uint32_t q_phase = (qn / C::QSETS) & 1;
          ++qn;
          grp0.in_item = grp1.in_item = 0;
          if (!mbar_wait(&q_full[qs], q_phase, &abort_flag, p.wait_limit_ns)) {
            fail(kSiteQ);
            break;
          }
          // S_g = Q_g K_j^T. It overwrites the previous scores (and P_g, where
          // that lies over them): the softmax has pulled those into registers
          // (s_free), P_g's product is complete (pv_done).
          auto issue_s = [&](Group& gs, const int g, int j, bool last_reader) {
            if (!ok || !wait_tile(base + 2 * j)) return;
            if (C::P_OVER_S) {
              if (gs.tiles > 0 && !mbar_wait(&pv_done[g], (gs.tiles - 1) & 1, &abort_flag, p.wait_limit_ns)) {
                fail(kSitePv);
                return;
              }
            } else if (gs.s_issued > 0 &&
                       !mbar_wait(&s_free[g], (gs.s_issued - 1) & 1, &abort_flag, p.wait_limit_ns)) {
              fail(kSiteSFree);
              return;
            }
            ++gs.s_issued;
            tc_fence_after();
            const Desc dq(smem_u32(sQ + (qs * C::GROUPS + g) * C::TILE_BYTES), 16, C::SBO, C::LAYOUT);
            const Desc dk(smem_u32(sR + ((base + 2 * j) % SLOTS) * C::TILE_BYTES), 16, C::SBO, C::LAYOUT);
#pragma unroll(HD == 256 ? 4 : HD / 16)
            for (int kk = 0; kk < HD / 16; ++kk) {
              const int at = kk / (C::COLS / 16) * C::CHUNK_BYTES + kk % (C::COLS / 16) * 32;
              mma_f16_ss(tmem_base + C::col_s(g), dq.at(at), dk.at(at), idesc_s, kk != 0 ? 1u : 0u);
            }
            mma_commit(&s_full[g]);
            if (last_reader) mma_commit(&slot_empty[(base + 2 * j) % SLOTS]);
          };
          // O_g += P_g V_j once group g has written P_g (p_full).
          auto issue_pv = [&](Group& gs, const int g, int j, int n_g, bool last_reader) {
            if (!ok || !wait_tile(base + 2 * j + 1)) return;
            if (!mbar_wait(&p_full[g], gs.tiles & 1, &abort_flag, p.wait_limit_ns)) {
              fail(kSiteP);
              return;
            }
            ++gs.tiles;
            if (gs.in_item == 0 && gs.o_uses > 0 &&
                !mbar_wait(&o_free[g], (gs.o_uses - 1) & 1, &abort_flag, p.wait_limit_ns)) {
              // the previous item's epilogue of group g must be done reading O_g
              fail(kSiteOFree);
              return;
            }
            tc_fence_after();
            // V is MN-major: 8 keys x COLS columns a swizzle atom, CHUNK_BYTES to
            // the next COLS columns, so one product spans the whole head
            const Desc dv(smem_u32(sR + ((base + 2 * j + 1) % SLOTS) * C::TILE_BYTES), C::CHUNK_BYTES, C::SBO,
                          C::LAYOUT);
#pragma unroll
            for (int ks = 0; ks < kBN / 16; ++ks)
              mma_f16_ts(tmem_base + C::col_o(g), tmem_base + C::col_p(g) + ks * 8, dv.at(ks * 16 * C::ROW_BYTES),
                         idesc_o, (gs.in_item > 0 || ks > 0) ? 1u : 0u);
            mma_commit(&pv_done[g]);
            if (last_reader) mma_commit(&slot_empty[(base + 2 * j + 1) % SLOTS]);
            if (++gs.in_item == n_g) {
              mma_commit(&o_full[g]);
              ++gs.o_uses;
            }
          };
          auto next_s = [&](const int g, int j) {
            if (g == 0 && it.uses(0, j)) issue_s(grp0, 0, j, !it.uses(1, j));
            if (g == 1 && j < it.n && it.uses(1, j)) issue_s(grp1, 1, j, true);
          };
          auto next_pv = [&](const int g, int j) {
            if (g == 0 && it.uses(0, j)) issue_pv(grp0, 0, j, it.n0, !it.uses(1, j));
            if (g == 1 && it.uses(1, j)) issue_pv(grp1, 1, j, it.n1, true);
          };
          next_s(0, 0);
          next_s(1, 0);
          for (int j = 0; j < it.n && ok; ++j) {
            if (p.kv_len != nullptr && j == max(0, it.dirty)) {
              // once an item the cleaner gets its turn: when the partial value
              // tile has landed and before its products, or at once
              if (it.dirty >= 0 && !wait_tile(base + 2 * j + 1)) break;
              if (turns > taken && !mbar_wait(&v_clean, taken++ & 1, &abort_flag, p.wait_limit_ns)) {
                fail(kSiteClean);
                break;
              }
              mbar_arrive(&v_dirty);
              ++turns;
              if (it.dirty >= 0 && !mbar_wait(&v_clean, taken++ & 1, &abort_flag, p.wait_limit_ns)) {
                fail(kSiteClean);
                break;
              }
            }
            if (C::P_OVER_S) {
              next_pv(0, j);
              next_s(0, j + 1);
              next_pv(1, j);
              next_s(1, j + 1);
            } else {
              // the next scores are computed during this step's exponentials
              next_s(0, j + 1);
              next_s(1, j + 1);
              next_pv(0, j);
              next_pv(1, j);
            }
          }
          if (!ok) break;
          mma_commit(&q_empty[qs]);  // every S of this item read its Q set
          base += 2 * it.n;
        }
        // everything issued is complete before TMEM can be released
        mma_commit(&drain_bar);
        mbar_wait(&drain_bar, 0, nullptr, ok ? p.wait_limit_ns : kDrainLimitNs);
        if (!ok) abort_flag = 1;
      }
      __syncwarp();
    } else if (warp == 2 && p.kv_len != nullptr) {
      // ---------------- cleaner: value rows at and past kv_len become zero ----------------
      // The issuer gives it one turn an item (v_dirty, ended by v_clean), so
      // that both barriers advance in step with the items.
      int base = 0, turns = 0;
      for (int idx = blockIdx.x; idx < n_items; idx += gridDim.x) {
        const Item it = make_item<C::GROUPS>(p, idx, q_tiles, q_items);
        if (it.n == 0) continue;
        if (!mbar_wait_warp(&v_dirty, turns++ & 1, &abort_flag, p.wait_limit_ns)) {
          if (lane == 0) report_error(kDevWaitTimeout, kid * 256 + kSiteClean);
          abort_flag = 1;
          break;
        }
        if (it.dirty >= 0) {
          const int t = base + 2 * it.dirty + 1;
          uint8_t* tile = sR + (t % SLOTS) * C::TILE_BYTES;
          // whole rows: the swizzle permutes 16-byte pieces within a row
          const int from = (it.kv_bound % kBN) * C::ROW_BYTES;
          for (int c = 0; c < C::NC; ++c)
            for (int o = from + static_cast<int>(lane) * 16; o < C::CHUNK_BYTES; o += 32 * 16)
              *reinterpret_cast<uint4*>(tile + c * C::CHUNK_BYTES + o) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clean);
        base += 2 * it.n;
      }
    }  // warp 3: no role
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------- softmax, group g, one query row per thread ----------------
    const int g = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + static_cast<int>(lane);
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_s = t_lane + (g == 0 ? C::col_s(0) : C::col_s(1));
    const uint32_t t_p = t_lane + (g == 0 ? C::col_p(0) : C::col_p(1));
    const uint32_t t_o = t_lane + (g == 0 ? C::col_o(0) : C::col_o(1));
    const float sl = p.scale_log2;
    int tiles = 0, o_uses = 0;
    bool ok = true;
    // Whether the previous product and the next scores are there, asked among
    // a tile's last exponentials, where the answer's latency costs nothing (a
    // wait that finds its phase complete still takes 150 clocks: 100,000 tokens
    // of window 4096, 2290 -> 2195 us).
    bool pv_ready = false, s_ready = false;
    for (int idx = blockIdx.x; idx < n_items && ok; idx += gridDim.x) {
      const Item it = make_item<C::GROUPS>(p, idx, q_tiles, q_items);
      if (g == 1 && !it.has1) continue;
      const int n_g = g == 0 ? it.n0 : it.n1;
      const int q_idx = (it.tq0 + g * it.dq) * kBM + r;
      float m = -INFINITY;  // running max, raw score units
      float l = 0.f;
      int done = 0;         // steps of this item so far
      for (int j = 0; j < it.n; ++j) {
        if (!it.uses(g, j)) continue;
        if (!__all_sync(0xffffffffu, s_ready) &&
            !mbar_wait_warp(&s_full[g], tiles & 1, &abort_flag, p.wait_limit_ns)) {
          report_error(kDevWaitTimeout, kid * 256 + kSiteS);
          abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const int k0 = it.tile(j) * kBN;
        // key k0 + c is visible iff c < lim and (c >= wlo or c < slim)
        const int lim = min(it.kv_bound, q_idx + 1) - k0;
        const int wlo = q_idx - p.window + 1 - k0;
        const int slim = p.sinks - k0;
        const bool full = lim >= kBN && (wlo <= 0 || slim >= kBN);
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, sv[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(sv[c]);
        if (!C::P_OVER_S) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[g]);
        }
        if (!full) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t seen = low_bits(lim - c * 32) & (~low_bits(wlo - c * 32) | low_bits(slim - c * 32));
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (!((seen >> t) & 1u)) sv[c][t] = 0xff800000u;  // -inf
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int t = 0; t < 32; t += 2)
            mx4[(t >> 1) & 3] = max3(mx4[(t >> 1) & 3], __uint_as_float(sv[c][t]), __uint_as_float(sv[c][t + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        float m_use = m;
        float alpha = 1.f;
        if (mx > m) {
          if (m == -INFINITY || (mx - m) * sl > kLazyRescaleLog2) {
            alpha = (m == -INFINITY) ? 0.f : ex2_approx((m - mx) * sl);
            m_use = mx;
          }
        }
        // a masked score is -inf and gives 0 (the FMA-pipe exponential clamps
        // it at 2^-126, which the fp16 P rounds to 0)
        const float neg_mc = (m_use == -INFINITY) ? 0.f : -m_use * sl;
        // Eight columns at a time, one group's exponentials between the next
        // one's scaling and the previous one's sums and packing: the SFU takes
        // a warp's exponential every 8 clocks, which leaves issue slots for
        // the other two.
        float rs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t pk[4][16];
        auto scale8 = [&](int u) {
#pragma unroll
          for (int t = (u & 3) * 8; t < (u & 3) * 8 + 8; t += 2) {
            float x0, x1;
            fma2(x0, x1, __uint_as_float(sv[u >> 2][t]), __uint_as_float(sv[u >> 2][t + 1]), sl, neg_mc);
            sv[u >> 2][t] = __float_as_uint(x0);
            sv[u >> 2][t + 1] = __float_as_uint(x1);
          }
        };
        auto exp8 = [&](int u) {
#pragma unroll
          for (int t = (u & 3) * 8; t < (u & 3) * 8 + 8; t += 2) exp2_cols(sv[u >> 2][t], sv[u >> 2][t + 1], t);
        };
        auto pack8 = [&](int u) {
#pragma unroll
          for (int t = (u & 3) * 8; t < (u & 3) * 8 + 8; t += 2) {
            const float p0 = __uint_as_float(sv[u >> 2][t]), p1 = __uint_as_float(sv[u >> 2][t + 1]);
            const int a = ((t >> 1) & 3) * 2;
            add2(rs[a], rs[a + 1], p0, p1);
            pk[u >> 2][t / 2] = pack_half2(p0, p1);
          }
        };
        scale8(0);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          if (u < 15) scale8(u + 1);
          exp8(u);
          if (!C::P_OVER_S && u == 12) {
            pv_ready = tiles == 0 || mbar_test(&pv_done[g], (tiles - 1) & 1);
            s_ready = mbar_test(&s_full[g], (tiles + 1) & 1);
          }
          if (u > 0) pack8(u - 1);
        }
        pack8(15);
        // The previous step's product reads P_g and writes O_g: complete before
        // P_g is overwritten or O_g rescaled. (Where P_g lies over S_g, this
        // step's scores were only issued after it.)
        auto wait_pv = [&]() -> bool {
          if (C::P_OVER_S) return true;
          if (!__all_sync(0xffffffffu, pv_ready) && !mbar_wait_warp(&pv_done[g], (tiles - 1) & 1, &abort_flag, p.wait_limit_ns)) {
            report_error(kDevWaitTimeout, kid * 256 + kSitePv);
            abort_flag = 1;
            return false;
          }
          tc_fence_after();
          return true;
        };
        ok = wait_pv();
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st16(t_p + c * 16, pk[c]);
        const float row_sum = ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
        const bool need = (done > 0) && (alpha != 1.f);
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + c, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int t = 0; t < 16; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * alpha);
            tmem_st16(t_o + c, o);
          }
        }
        l = l * alpha + row_sum;
        m = m_use;
        ++tiles;
        ++done;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      if (!ok) break;
      // epilogue: O / l -> fp16 [b, q, h*hd + c]
      if (n_g > 0) {
        if (!mbar_wait_warp(&o_full[g], o_uses & 1, &abort_flag, p.wait_limit_ns)) {
          report_error(kDevWaitTimeout, kid * 256 + kSiteO);
          abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
      }
      // a row that sees no key has m = -inf: zeros
      const float inv_l = (m != -INFINITY) ? 1.f / l : 0.f;
      __half* dst = p.out + (static_cast<int64_t>(it.b) * p.S + q_idx) * p.ld_out + (it.h + g * it.dh) * p.hd;
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        if (n_g > 0) {
          tmem_ld16(t_o + c, o);
          tmem_ld_wait(o);
        } else {
#pragma unroll
          for (int t = 0; t < 16; ++t) o[t] = 0u;
        }
        if (q_idx < p.S) {
          uint4 w0, w1;
          w0.x = pack_half2(__uint_as_float(o[0]) * inv_l, __uint_as_float(o[1]) * inv_l);
          w0.y = pack_half2(__uint_as_float(o[2]) * inv_l, __uint_as_float(o[3]) * inv_l);
          w0.z = pack_half2(__uint_as_float(o[4]) * inv_l, __uint_as_float(o[5]) * inv_l);
          w0.w = pack_half2(__uint_as_float(o[6]) * inv_l, __uint_as_float(o[7]) * inv_l);
          w1.x = pack_half2(__uint_as_float(o[8]) * inv_l, __uint_as_float(o[9]) * inv_l);
          w1.y = pack_half2(__uint_as_float(o[10]) * inv_l, __uint_as_float(o[11]) * inv_l);
          w1.z = pack_half2(__uint_as_float(o[12]) * inv_l, __uint_as_float(o[13]) * inv_l);
          w1.w = pack_half2(__uint_as_float(o[14]) * inv_l, __uint_as_float(o[15]) * inv_l);
          reinterpret_cast<uint4*>(dst + c)[0] = w0;
          if (c + 16 <= p.hd) reinterpret_cast<uint4*>(dst + c)[1] = w1;  // head_dim 8: columns 8..15 are padding
        }
      }
      if (n_g > 0) {
        ++o_uses;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[g]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, kTmemCols);
}

}  // namespace win
}  // namespace attn
}  // namespace tk

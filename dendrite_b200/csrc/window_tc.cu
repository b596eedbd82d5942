// Sliding-window attention of chunks of new tokens on tcgen05 (TMEM
// accumulators): bf16 queries over bf16 / E4M3 / MXFP8 pages, head dims 64
// and 128.
//
// A work item is (sequence, KV head, 256 query rows): the rows of 256 / g new
// tokens, so the visible pages of an item are those of its first row's window
// up to its last row's position, plus the pages of the first tokens. Persistent
// CTAs, one per SM, take the items in a fixed order, long ones (late rows)
// first, the direction of every second round reversed; nothing is planned on
// the host. The rows form two 128-row sub-tiles A and B that share each K/V
// tile of 128 tokens (8 pages of the item's list):
//   warp 0       TMA producer, two boxes a page into the K/V ring (FP8 codes:
//                into a staging ring); lane p < 8 looks page p of a tile up
//   warp 1       issues the products, per tile P_A.V, Q_A.K', P_B.V, Q_B.K'
//                (the tensor core works on one sub-tile while the softmax of
//                the other runs)
//   warps 2-9    softmax, a thread per row: scores from TMEM, one pass per 64
//                tokens, weights written over them
//   warps 10-13  FP8: codes widened into the K/V ring
// The tensor pipe and the exponential unit bound it together: 256 rows x 128
// tokens are 2048 cycles of products at D = 128 and 2048 of exponentials.
//
// Types. bf16 and MXFP8 pages take bf16 products; a code times its power of
// two is exact in bf16. E4M3 pages take f16 products on the bare codes (exact,
// one conversion for two codes): Q's rows are scaled by a power of two into
// f16's range and the per-head scales go into the score scale and the epilogue.
// The softmax weights are rounded once (to nearest) to the products' type, 8
// bits in bf16 and 11 in f16: a second bf16 term would cost half as many
// products again, and the output is rounded to bf16's 8 bits anyway. Row sums
// and references are f32.
//
// Masks. The item's page list is a virtual axis x (first-token pages, then
// window pages); a row of position p sees x in [p - window + 1 - shift, p -
// shift] and x < sinks. Only tiles that some row does not see whole are masked;
// V of slots that no row of the item sees is zeroed before the product (zero
// times NaN is not zero).
#include <algorithm>

#include "tc_common.cuh"
#include "window.cuh"

namespace dd {

constexpr int kWtRows = 256;
constexpr int kWtConvWarps = 4;
constexpr int kWtStages = 3;

template <int D, int KV>
struct WtCfg {
  static constexpr bool kFp8 = KV != DD_DTYPE_BF16;
  static constexpr bool kF16 = KV == DD_DTYPE_E4M3;
  static constexpr int kHalves = D / 64;                 // 64-dim halves of a row
  static constexpr int kHalfBytes = kTcTok * 128;        // [128 rows][128 B], 128-byte swizzle
  static constexpr int kTileBytes = kHalves * kHalfBytes;  // a Q sub-tile, or a K or V tile
  static constexpr int kSlots = kFp8 ? 3 : 4;
  static constexpr int kCodes = kTcTok * D;              // staged codes of a tile
  static constexpr int kExps = kTcTok * (D / 32);        // MXFP8 exponents of a tile
  static constexpr int kThreads = kFp8 ? 320 + 32 * kWtConvWarps : 320;
  static constexpr int kSmem = (2 + kSlots) * kTileBytes +
                               (kFp8 ? kWtStages * (kCodes + kExps) : 0) + 1024;
  // D f32, M = 128; A / B type in bits 7 and 10 (0 f16, 1 bf16); N in bits 17-22.
  static constexpr uint32_t kType = kF16 ? 0u : (1u << 7) | (1u << 10);
  static constexpr uint32_t kIdQK = (1u << 4) | kType | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t kIdPV = (1u << 4) | kType | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24) | (1u << 16);
  // How far a score may pass the reference, and the shift of the weights
  // (log2): f16 weights stay below 2^16 and normal down to 2^-21.
  static constexpr float kStep = kF16 ? 8.f : 16.f;
  static constexpr float kShift = kF16 ? 7.f : 0.f;
};

struct WtBars {
  uint64_t kv_full[4], kv_empty[4];
  uint64_t st_full[kWtStages], st_empty[kWtStages];
  uint64_t s_full[2], p_full[2];
  uint64_t item_done, q_ready;
  uint32_t tmem_base;
  int abort;
};

struct WtItem {
  int32_t h, nrows;       // nrows <= 0: no such item
  int32_t t0, table;      // the sequence's page table
  int32_t r0;             // first row of the sequence
  int64_t row0;           // first of the item's rows, counted from the sequence's first
  int32_t pos0;           // position of the sequence's first row
  int32_t p_lo, p_hi;
  WinPages wp;
  int32_t shift, ntiles;
};

// Item `i` of this CTA (all roles walk the same list); false past the end.
__device__ __forceinline__ bool wt_item(const WinArgs& a, int64_t units, int i, WtItem& it) {
  const int64_t n = gridDim.x;
  const int64_t u = i * n + ((i & 1) ? n - 1 - blockIdx.x : blockIdx.x);
  if (i * n >= units) return false;
  it.nrows = 0;
  if (u >= units) return true;
  const int64_t unit = units - 1 - u;
  it.h = (int32_t)(unit % a.Hkv);
  int32_t s, tile;
  win_tile(a, kWtRows, unit / a.Hkv, s, tile);
  const SeqRows sr = seq_rows(a.row_indptr, a.num_tokens, a.num_rows, s);
  it.row0 = (int64_t)tile * kWtRows;
  it.nrows = (int32_t)min((int64_t)kWtRows, max((int64_t)sr.m * a.g - it.row0, (int64_t)0));
  if (tile < 0) it.nrows = 0;
  if (it.nrows <= 0) return true;
  it.r0 = sr.r0;
  it.pos0 = sr.pos0;
  it.p_lo = sr.pos0 + (int32_t)(it.row0 / a.g);
  it.p_hi = sr.pos0 + (int32_t)((it.row0 + it.nrows - 1) / a.g);
  it.t0 = a.page_indptr[s];
  it.table = a.page_indptr[s + 1] - it.t0;
  it.wp = win_pages(a.window, a.sinks, it.p_lo, it.p_hi);
  it.shift = (it.wp.wp - it.wp.ns) * kPageSize;
  it.ntiles = (it.wp.count + kTcPagesPerTile - 1) / kTcPagesPerTile;
  return true;
}
// Pool page of page v of the item's list; 0xFFFFFFFF past its end or where
// there is no such page.
__device__ __forceinline__ uint32_t wt_page(const WinArgs& a, const WtItem& it, int32_t v, bool report) {
  if (v >= it.wp.count) return 0xFFFFFFFFu;
  const int32_t idx = it.wp.page(v);
  const uint32_t id = idx < it.table ? (uint32_t)a.page_indices[it.t0 + idx] : 0xFFFFFFFFu;
  if (id < (uint32_t)a.num_pages) return id;
  if (report) win_report(a.status, kDevErrBadPage, idx < it.table ? id : (uint32_t)idx);
  return 0xFFFFFFFFu;
}
// Whether some row of the item sees virtual token x.
__device__ __forceinline__ bool wt_seen(const WinArgs& a, const WtItem& it, int32_t x) {
  return x <= it.p_hi - it.shift && (a.window == 0 || x > it.p_lo - a.window - it.shift || x < a.sinks);
}
// Whether every row of the item sees all of virtual tokens [x, x + n).
__device__ __forceinline__ bool wt_whole(const WinArgs& a, const WtItem& it, int32_t x, int32_t n) {
  return x + n - 1 <= it.p_lo - it.shift &&
         (a.window == 0 || x > it.p_hi - a.window - it.shift || x + n <= a.sinks);
}

// Weights of 64 scores, to the products' type, over the chunk's half of the
// score columns; their f32 sum is added to acc.
template <bool kF16>
__device__ __forceinline__ void wt_weights(float (&s)[64], uint64_t sc2, uint64_t nm2, uint64_t& acc, uint32_t taddr) {
  uint64_t a0 = 0ull, a1 = 0ull;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const int k = 32 * half + i;
      const uint64_t x0 = f2_fma(f2_pack(s[k], s[k + 1]), sc2, nm2);
      const uint64_t x1 = f2_fma(f2_pack(s[k + 2], s[k + 3]), sc2, nm2);
      const float e0 = fast_exp2(f2_lo(x0)), e1 = fast_exp2(f2_hi(x0));
      const float e2 = fast_exp2(f2_lo(x1)), e3 = fast_exp2(f2_hi(x1));
      a0 = f2_add(a0, f2_pack(e0, e1));
      a1 = f2_add(a1, f2_pack(e2, e3));
      w[i / 2] = kF16 ? pack_f16x2(e0, e1) : pack_bf16x2(e0, e1);
      w[i / 2 + 1] = kF16 ? pack_f16x2(e2, e3) : pack_bf16x2(e2, e3);
    }
    tmem_st16u(taddr + 16 * half, w);
  }
  acc = f2_add(acc, f2_add(a0, a1));
}

// `cols` columns of packed f16 pairs of this thread's TMEM lane, times f.
__device__ __noinline__ void tmem_scale_f16(uint32_t taddr, int cols, float f) {
  for (int c = 0; c < cols; c += 16) {
    uint32_t v[16];
    tmem_ld16u(taddr + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      v[i] = pack_f16x2(x.x * f, x.y * f);
    }
    tmem_st16u(taddr + c, v);
  }
  tmem_wait_st();
}

template <int D, int KV>
__global__ void __launch_bounds__(WtCfg<D, KV>::kThreads, 1)
    win_tc_kernel(const __grid_constant__ CUtensorMap kv_map, WinArgs a, int64_t units) {
  using Cfg = WtCfg<D, KV>;
  constexpr bool kFp8 = Cfg::kFp8, kF16 = Cfg::kF16;
  constexpr int kSlots = Cfg::kSlots, kTile = Cfg::kTileBytes, kHalf = Cfg::kHalfBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ WtBars bars;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_s = smem;                        // [sub-tile][half][128 rows][128 B]
  uint8_t* slots = smem + 2 * kTile;          // [slot][half][128 rows][128 B]
  uint8_t* stages = slots + kSlots * kTile;   // FP8: [stage][128 rows][D]
  uint8_t* stage_exps = stages + kWtStages * Cfg::kCodes;  // [stage][128 rows][D / 32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WsHeader* err = reinterpret_cast<WsHeader*>(a.status);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars.kv_full[s], kFp8 ? 32 * kWtConvWarps : 1);
      mbar_init(&bars.kv_empty[s], 1);
    }
    for (int s = 0; s < kWtStages; ++s) {
      mbar_init(&bars.st_full[s], 1);
      mbar_init(&bars.st_empty[s], 32 * kWtConvWarps);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars.s_full[x], 1);
      mbar_init(&bars.p_full[x], 128);
    }
    mbar_init(&bars.item_done, 1);
    mbar_init(&bars.q_ready, 256);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&bars.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 64) prefetch_tmap(&kv_map);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars.tmem_base;
  volatile int* abort = &bars.abort;
  WtItem it;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    const int64_t rows_total = (int64_t)a.num_pages * 2 * a.Hkv * kPageSize;
    const int pj = lane & (kTcPagesPerTile - 1);
    const bool mine = lane < kTcPagesPerTile;
    int gidx = 0;
    bool ok = true;
    for (int i = 0; ok && wt_item(a, units, i, it); ++i) {
      if (it.nrows <= 0) continue;
      uint32_t cur = mine ? wt_page(a, it, pj, true) : 0xFFFFFFFFu;
      uint32_t nxt = 0xFFFFFFFFu;
      for (int idx = 0; idx < 2 * it.ntiles; ++idx, ++gidx) {
        const int j = idx >> 1, kv = idx & 1;
        if (kv == 0 && mine) nxt = wt_page(a, it, (j + 1) * kTcPagesPerTile + pj, true);
        // A missing page reads past the pool's end: zeros.
        const bool have = mine && cur != 0xFFFFFFFFu;
        const int y = have ? (int)((((int64_t)cur * 2 + kv) * a.Hkv + it.h) * kPageSize) : (int)rows_total;
        if constexpr (kFp8) {
          const int su = gidx % kWtStages;
          ok = __all_sync(0xffffffffu, gidx < kWtStages ||
                                           mbar_wait(&bars.st_empty[su], ((gidx / kWtStages) - 1) & 1, abort, err));
          if (!ok) break;
          const uint32_t present = __ballot_sync(0xffffffffu, have);
          if (lane == 0)
            mbar_arrive_expect_tx(&bars.st_full[su],
                                  Cfg::kCodes + (KV == DD_DTYPE_MXFP8 ? __popc(present) * (Cfg::kExps / 8) : 0));
          __syncwarp();
          if (mine) {
            tma_load_2d(stages + su * Cfg::kCodes + pj * kPageSize * D, &kv_map, 0, y, &bars.st_full[su]);
            if (KV == DD_DTYPE_MXFP8 && have)
              bulk_load(stage_exps + su * Cfg::kExps + pj * (Cfg::kExps / 8),
                        reinterpret_cast<const uint8_t*>(a.scales) + (int64_t)y * (D / 32), Cfg::kExps / 8,
                        &bars.st_full[su]);
          }
        } else {
          const int s = gidx % kSlots;
          ok = __all_sync(0xffffffffu, gidx < kSlots ||
                                           mbar_wait(&bars.kv_empty[s], ((gidx / kSlots) - 1) & 1, abort, err));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bars.kv_full[s], kTile);
          __syncwarp();
          if (mine) {
            uint8_t* dst = slots + s * kTile + pj * 2048;
#pragma unroll
            for (int hf = 0; hf < Cfg::kHalves; ++hf) tma_load_2d(dst + hf * kHalf, &kv_map, 64 * hf, y, &bars.kv_full[s]);
          }
        }
        if (kv == 1) cur = nxt;
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      const uint64_t q_desc0 = umma_desc(smem_u32(q_s), 16, 1024);
      const uint64_t k_desc0 = umma_desc(smem_u32(slots), 16, 1024);
      const uint64_t v_desc0 = umma_desc(smem_u32(slots), kHalf, 1024);
      int g0 = 0;            // ring index of the item's first K tile
      int seen[2] = {0, 0};  // tiles each sub-tile's softmax has handed over
      int n = 0;             // items so far
      bool ok = true;
      for (int i = 0; ok && wt_item(a, units, i, it); ++i) {
        if (it.nrows <= 0) continue;
        const int ntiles = it.ntiles;
        const int nsub = it.nrows > 128 ? 2 : 1;
        auto wait_slot = [&](int idx) {
          return mbar_wait(&bars.kv_full[(g0 + idx) % kSlots], ((g0 + idx) / kSlots) & 1, abort, err);
        };
        auto issue_qk = [&](int x, int j) {
          const uint64_t kd = k_desc0 + (uint64_t)((((g0 + 2 * j) % kSlots) * kTile) >> 4);
          const uint64_t qd = q_desc0 + (uint64_t)((x * kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4);
            umma_ss(tbase + col_s(x), qd + off, kd + off, Cfg::kIdQK, kk > 0 ? 1u : 0u);
          }
          umma_commit(&bars.s_full[x]);
        };
        ok = mbar_wait(&bars.q_ready, n & 1, abort, err);
        ++n;
        if (!ok || ntiles == 0) continue;
        ok = wait_slot(0);
        if (!ok) break;
        tc_fence_after();
        for (int x = 0; x < nsub; ++x) issue_qk(x, 0);
        umma_commit(&bars.kv_empty[g0 % kSlots]);
        for (int j = 0; ok && j < ntiles; ++j) {
          const int sv = (g0 + 2 * j + 1) % kSlots;
          const uint64_t vd = v_desc0 + (uint64_t)((sv * kTile) >> 4);
          for (int x = 0; ok && x < nsub; ++x) {
            if (!mbar_wait(&bars.p_full[x], (seen[x] + j) & 1, abort, err)) { ok = false; break; }
            if (x == 0 && !wait_slot(2 * j + 1)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kt = 0; kt < 8; ++kt)
              umma_ts(tbase + col_o(x), tbase + col_s(x) + kt * 8, vd + (uint64_t)((kt * 2048) >> 4), Cfg::kIdPV,
                      (j > 0 || kt > 0) ? 1u : 0u);
            if (j + 1 < ntiles) {
              if (x == 0) {
                if (!wait_slot(2 * j + 2)) { ok = false; break; }
                tc_fence_after();
              }
              issue_qk(x, j + 1);
              if (x == nsub - 1) umma_commit(&bars.kv_empty[(g0 + 2 * j + 2) % kSlots]);
            }
          }
          if (ok) umma_commit(&bars.kv_empty[sv]);
        }
        if (ok) umma_commit(&bars.item_done);
        seen[0] += ntiles;
        if (nsub > 1) seen[1] += ntiles;
        g0 += 2 * ntiles;
      }
    }
  } else if (kFp8 && warp >= 10) {
    // -------------------------------------------------------------- converters
    // A thread widens 16 codes of one token at a time; eight neighbouring
    // threads cover two rows, so their stores fall into eight bank groups.
    const int t = threadIdx.x - 320;
    constexpr int kConvThreads = 32 * kWtConvWarps;
    constexpr int kChunks = kTcTok * D / 16;
    int gidx = 0;
    bool ok = true;
    for (int i = 0; ok && wt_item(a, units, i, it); ++i) {
      if (it.nrows <= 0) continue;
      const int pj = lane & (kTcPagesPerTile - 1);
      uint32_t page = wt_page(a, it, pj, false), pages = 0;
      for (int idx = 0; idx < 2 * it.ntiles; ++idx, ++gidx) {
        const int su = gidx % kWtStages, s = gidx % kSlots;
        if ((idx & 1) == 0) {  // the tile's pages that exist; the next tile's ids on their way
          pages = __ballot_sync(0xffffffffu, page != 0xFFFFFFFFu);
          page = wt_page(a, it, ((idx >> 1) + 1) * kTcPagesPerTile + pj, false);
        }
        ok = mbar_wait(&bars.st_full[su], (gidx / kWtStages) & 1, abort, err) &&
             (gidx < kSlots || mbar_wait(&bars.kv_empty[s], ((gidx / kSlots) - 1) & 1, abort, err));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* src = stages + su * Cfg::kCodes;
        const uint8_t* exps = stage_exps + su * Cfg::kExps;
        uint8_t* dst = slots + s * kTile;
        const int32_t x0 = (idx >> 1) * kTcTok;
        const bool clean = wt_whole(a, it, x0, kTcTok);
#pragma unroll 4
        for (int id = t; id < kChunks; id += kConvThreads) {
          int row, c;  // token, 16-dim chunk
          uint4 codes;
          if constexpr (D == 128) {
            const int half = (id >> 3) & 1;
            row = ((id >> 4) << 1) | ((id >> 2) & 1);
            c = half * 4 + (id & 3);
            codes = *reinterpret_cast<const uint4*>(src + row * 128 + ((c ^ (row & 7)) << 4));
          } else {
            row = id >> 2;
            c = id & 3;
            codes = *reinterpret_cast<const uint4*>(src + row * 64 + (c << 4));
          }
          uint32_t o[8];
          if constexpr (kF16) {
            const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              o[2 * k] = e4m3_f16(w[k], 0);
              o[2 * k + 1] = e4m3_f16(w[k], 1);
            }
          } else {
            e4m3x16_to_bf16(codes, e8m0_to_float(exps[row * (D / 32) + (c >> 1)]), o);
          }
          // Slots that no row sees, and missing pages (their exponents are stale).
          if (!((pages >> (row >> 4)) & 1) || (!clean && !wt_seen(a, it, x0 + row))) {
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = 0;
          }
          uint8_t* drow = dst + (c >> 2) * kHalf + row * 128;
          const int cl = c & 3;
          *reinterpret_cast<uint4*>(drow + (((2 * cl) ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(drow + (((2 * cl + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars.kv_full[s]);
        mbar_arrive(&bars.st_empty[su]);
      }
    }
  } else if (warp >= 2 && warp < 10) {
    // ----------------------------------------------------------------- softmax
    const int x = (warp - 2) >> 2;  // sub-tile
    const int quarter = warp & 3;   // TMEM lanes [32 * quarter, + 32)
    const int r = quarter * 32 + lane, row = x * 128 + r;
    const uint32_t lane_base = tbase + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_col = lane_base + col_s(x), o_col = lane_base + col_o(x);
    float scale_log2 = a.scale_log2, v_scale = 1.f;  // of the current item
    int seen = 0, done = 0, g0 = 0;
    // Row of q and out that this thread holds of an item.
    auto place = [&](const WtItem& q, int64_t& token) {
      const int64_t rr = q.row0 + row;
      token = q.r0 + rr / a.g;
      return qo_head_of(a.gqa_map, q.h, (int)(rr % a.g), a.Hkv, a.g);
    };
    // Q row -> the sub-tile's swizzled K-major tile, handed to the MMA warp.
    // Returns the power of two by which the stored row must be multiplied back.
    auto write_q = [&](const WtItem& q) {
      const uint4* src = nullptr;
      if (row < q.nrows) {
        int64_t token;
        const int hq = place(q, token);
        src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + token * a.q_stride + (int64_t)hq * D);
      }
      int up = 0;
      if constexpr (kF16) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = src ? src[c] : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
        }
        up = f16_row_shift(top);
      }
      const float by = __uint_as_float((uint32_t)(127 + up) << 23);
      uint8_t* qx = q_s + x * kTile + r * 128;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 v = src ? src[c] : make_uint4(0, 0, 0, 0);
        if constexpr (kF16) {
          v.x = bf16x2_to_f16x2(v.x, by);
          v.y = bf16x2_to_f16x2(v.y, by);
          v.z = bf16x2_to_f16x2(v.z, by);
          v.w = bf16x2_to_f16x2(v.w, by);
        }
        *reinterpret_cast<uint4*>(qx + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      mbar_arrive(&bars.q_ready);
      return up;
    };
    int i = 0;
    bool have = false;
    while (wt_item(a, units, i, it)) {
      if (it.nrows > 0) {
        have = true;
        break;
      }
      ++i;
    }
    int up = 0;
    if (have) up = write_q(it);
    while (have) {
      const WtItem cur = it;
      const bool live = row < cur.nrows, active = x == 0 || cur.nrows > 128;
      // The next item with rows, if any.
      have = false;
      while (wt_item(a, units, ++i, it)) {
        if (it.nrows > 0) {
          have = true;
          break;
        }
      }
      if constexpr (kF16) {
        scale_log2 = f16_score_scale(a.scale_log2, up) * reinterpret_cast<const float*>(a.scales)[cur.h];
        v_scale = reinterpret_cast<const float*>(a.scales)[a.Hkv + cur.h];
      }
      const int32_t p = cur.pos0 + (int32_t)((cur.row0 + row) / a.g);
      const int32_t hi = p - cur.shift, lo = a.window ? p - a.window + 1 - cur.shift : 0;
      const int ntiles = cur.ntiles;
      // Which of a tile's pages exist: looked up a tile ahead, as the producer does.
      const int pj = lane & (kTcPagesPerTile - 1);
      uint32_t page = active && ntiles > 0 ? wt_page(a, cur, pj, false) : 0xFFFFFFFFu;
      float m_used = -INFINITY;
      uint64_t lsum = 0ull;
      bool ok = true;
      const uint64_t sc2 = f2_pack(scale_log2, scale_log2);
      for (int j = 0; active && j < ntiles; ++j) {
        const int32_t x0 = j * kTcTok;
        const uint32_t pages = __ballot_sync(0xffffffffu, page != 0xFFFFFFFFu) & 0xffu;
        page = wt_page(a, cur, (j + 1) * kTcPagesPerTile + pj, false);
        const bool whole = pages == 0xffu && wt_whole(a, cur, x0, kTcTok);
        ok = ok && mbar_wait(&bars.s_full[x], (seen + j) & 1, abort, err);
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float s[64];
          {
            float t[32];
            tmem_ld32(s_col + c * 64, t);
#pragma unroll
            for (int k = 0; k < 32; ++k) s[k] = t[k];
            tmem_ld32(s_col + c * 64 + 32, t);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) s[32 + k] = t[k];
          }
          if (!whole) {
            // Bit k: the row sees token x0 + 64 c + k.
            const int32_t b = x0 + 64 * c;
            auto below = [](int32_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
            uint64_t see = below(hi - b + 1) & (~below(lo - b) | below(a.sinks - b));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (!((pages >> (4 * c + k)) & 1)) see &= ~(0xffffull << (16 * k));
            const uint32_t see0 = (uint32_t)see, see1 = (uint32_t)(see >> 32);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (!((see0 >> k) & 1)) s[k] = -INFINITY;
              if (!((see1 >> k) & 1)) s[32 + k] = -INFINITY;
            }
          }
          float m0 = s[0], m1 = s[1];
#pragma unroll
          for (int k = 2; k < 62; k += 4) {
            m0 = max3f(m0, s[k], s[k + 1]);
            m1 = max3f(m1, s[k + 2], s[k + 3]);
          }
          const float mt = ok ? max3f(m0, m1, fmaxf(s[62], s[63])) * scale_log2 : m_used;
          if (__any_sync(0xffffffffu, mt > m_used + Cfg::kStep)) {
            const float m_new = mt > m_used + Cfg::kStep ? ceilf(mt) : m_used;
            const float f = m_used == m_new ? 1.f : exp2f(m_used - m_new);  // a power of two
            if (j > 0) tmem_scale_cols<false>(o_col, D, f);
            if (c == 1) {
              if constexpr (kF16)
                tmem_scale_f16(s_col, 32, f);
              else
                tmem_scale_cols<true>(s_col, 32, f);
            }
            lsum = f2_fma(lsum, f2_pack(f, f), 0ull);
            m_used = m_new;
          }
          const float ref = (m_used == -INFINITY ? 0.f : m_used) - Cfg::kShift;
          wt_weights<kF16>(s, sc2, f2_pack(-ref, -ref), lsum, s_col + c * 32);
        }
        // bf16 pages: V of slots that no row sees (sub-tile A's 128 threads, a
        // token each, before they hand the weights over).
        if (!kFp8 && x == 0 && !wt_whole(a, cur, x0, kTcTok)) {
          const int vi = g0 + 2 * j + 1;
          ok = mbar_wait(&bars.kv_full[vi % kSlots], (vi / kSlots) & 1, abort, err) && ok;
          if (!wt_seen(a, cur, x0 + r)) {
            uint8_t* v = slots + (vi % kSlots) * kTile + r * 128;
#pragma unroll
            for (int hf = 0; hf < Cfg::kHalves; ++hf)
#pragma unroll
              for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(v + hf * kHalf + 16 * k) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars.p_full[x]);
      }
      if (active) seen += ntiles;
      g0 += 2 * ntiles;
      if (ntiles > 0) {
        ok = mbar_wait(&bars.item_done, done & 1, abort, err) && ok;
        ++done;
        tc_fence_after();
      }
      // The next item's Q before this epilogue: its first scores overlap it
      // (its first P.V, which overwrites O, waits for this thread's weights).
      const int up_next = have && __all_sync(0xffffffffu, ok) ? write_q(it) : 0;
      if (active) {
        const float L = f2_lo(lsum) + f2_hi(lsum);
        const float inv = L == 0.f ? 0.f : v_scale / L;
        int64_t token = 0;
        const int hq = live ? place(cur, token) : 0;
        const int64_t dst = token * a.Hq + hq;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (ntiles > 0) {
            tmem_ld32(o_col + c * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.f;
          }
          if (live) {
            uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + dst * D + c * 32);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              out[k] = make_uint4(pack_bf16x2(o[8 * k] * inv, o[8 * k + 1] * inv),
                                  pack_bf16x2(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                                  pack_bf16x2(o[8 * k + 4] * inv, o[8 * k + 5] * inv),
                                  pack_bf16x2(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
          }
        }
        if (live && a.lse)
          a.lse[dst] = L == 0.f ? -INFINITY : (m_used - Cfg::kShift + log2f(L)) * kLn2;
      }
      up = up_next;
      tc_fence_before();
      if (!__all_sync(0xffffffffu, ok)) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kTmemCols)
                 : "memory");
  }
}

int make_kv_tensor_map(CUtensorMap* map, const void* kv, int64_t num_pages, int Hkv, int D,
                       int elem_bytes, int two_halves);

template <int D, int KV>
static cudaError_t launch_win_tc_t(const CUtensorMap& map, const WinArgs& a, int64_t units, int sms, cudaStream_t st) {
  using Cfg = WtCfg<D, KV>;
  cudaError_t e = cudaFuncSetAttribute(win_tc_kernel<D, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  ProfScope ps(kProfTc, st);
  win_tc_kernel<D, KV><<<(unsigned)std::min<int64_t>(units, sms), Cfg::kThreads, Cfg::kSmem, st>>>(map, a, units);
  return cudaGetLastError();
}
template <int D>
static cudaError_t launch_win_tc_kv(const CUtensorMap& map, const WinArgs& a, int64_t units, int sms, cudaStream_t st) {
  switch (a.kv_dtype) {
    case DD_DTYPE_BF16: return launch_win_tc_t<D, DD_DTYPE_BF16>(map, a, units, sms, st);
    case DD_DTYPE_E4M3: return launch_win_tc_t<D, DD_DTYPE_E4M3>(map, a, units, sms, st);
    default: return launch_win_tc_t<D, DD_DTYPE_MXFP8>(map, a, units, sms, st);
  }
}

int launch_win_tc(const WinArgs& a, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  CUtensorMap map;
  const int rc = make_kv_tensor_map(&map, a.kv, a.num_pages, a.Hkv, a.D, a.kv_dtype == DD_DTYPE_BF16 ? 2 : 1, 0);
  if (rc) return rc;
  const int64_t units = (a.num_seqs + (int64_t)a.num_rows * a.g / kWtRows) * a.Hkv;
  const cudaError_t e = a.D == 64 ? launch_win_tc_kv<64>(map, a, units, sms, st) : launch_win_tc_kv<128>(map, a, units, sms, st);
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("window attention launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

}  // namespace dd

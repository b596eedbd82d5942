// Sliding-window attention of chunks of new tokens on tcgen05 (TMEM
// accumulators): bf16 queries over bf16 / E4M3 / MXFP8 pages, head dims 64
// and 128.
//
// A work item is (sequence, KV head, two sub-tiles of 128 / g new tokens), a
// sub-tile's rows being (token, query head of the group): up to 128 rows of Q,
// which one TMA box brings. The item's pages are those that its first token's
// window up to its last token's position reach, plus those of the first tokens.
// The launch has a CTA per item, long ones (late tokens) first. Each CTA that
// has started (one per SM) claims further ones in place of their starting, as
// it comes near the end of its item; nothing is planned on the host. (A fixed
// share of the items for each CTA took 291 us in place of 270 for 4 chunks of 1000
// tokens, E4M3, window 2048, and with weights of one bf16 term 908 in place of 799
// for 16 chunks of 200 to 2000, bf16, window 4096.) Where the items are few, a cluster of 2 to 8 CTAs
// shares one: each takes some of its tiles, and the outputs are joined through
// shared memory. K and V come in tiles of 128 tokens (8 pages of the item's list):
//   softmax      warps 0-3 sub-tile A, 4-7 B, a thread per row: the maximum of
//                128 scores in TMEM, then the weights of the tile's second and
//                first 64 tokens, each written over its scores and handed over
//                by itself
//   converters   warps 8-11 (FP8): codes widened into the K/V ring
//   producer     TMA boxes of K and V into the ring (FP8 codes: into a staging
//                ring); lane p < 8 looks page p of a tile up
//   issuers      one per sub-tile: per tile P.V by halves, then the next Q.K
//   scheduler    claims the items, into a small ring that the others read
//                (finding an item is a chain of dependent loads and divisions),
//                and an item's Q once the previous item's last scores are done
// The tensor core works on one sub-tile while the softmax of the other runs.
// A tile of 256 rows at D = 128 is 3120 cycles of products (65 each, their
// shared-memory operands keeping that memory busy throughout; E4M3, whose weights
// are one term, 2080) and 2048 of exponentials.
//
// Types. bf16 and MXFP8 pages take bf16 products; a code times its power of
// two is exact in bf16. E4M3 pages take f16 products on the bare codes (exact,
// one conversion for two codes): Q's rows are scaled by a power of two into
// f16's range and the per-head scales go into the score scale and the epilogue.
// The softmax weights are two bf16 terms (16 bits, as in the streaming kernel and
// the plans' kernels: with one, 1.1e-3 off on average, a prompt of 8191 tokens takes
// 394 us in place of 495) or one f16 term, rounded to nearest (11 bits, 2^-32 of the
// largest weight at worst). Row sums and references are f32.
//
// Masks. The item's page list is a virtual axis x (first-token pages, then
// window pages); a row of position p sees x in [p - window + 1 - shift, p -
// shift] and x < sinks. Only chunks that some row does not see whole are
// masked; V of slots that no row of the item sees is zeroed before the product
// (zero times NaN is not zero).
#include <algorithm>
#include <cfloat>

#include "tc_common.cuh"
#include "window.cuh"

namespace dd {

constexpr int kWtConvWarps = 4;
constexpr int kWtStages = 3;
constexpr int kWtChunk = 64;  // tokens of a half tile

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
  static constexpr int kProducer = kFp8 ? 12 : 8;        // then two issuers and the scheduler
  static constexpr int kThreads = 32 * (kProducer + 4);
  // FP8: the softmax takes registers over from the other warps and holds a
  // tile's scores, in place of reading their first half again (8 chunks of 200
  // to 700 tokens, window 1024, MXFP8: 109 us -> 102; 4 of 1000, window 2048,
  // E4M3: 309 -> 306; bf16, 16 of 200 to 2000, window 4096: 1011 -> 1013, 64 of 16:
  // 285 -> 296, so not there).
  // Together no more than the block's at launch.
  static constexpr bool kHeld = kFp8;
  static constexpr int kRegs = kFp8 ? 128 : 168, kRegsSoftmax = 184, kRegsConvert = 80, kRegsRest = 64;
  static_assert(256 * kRegsSoftmax + 128 * kRegsConvert + 128 * kRegsRest <= 512 * 128);
  static constexpr int kSmem = (2 + kSlots) * kTileBytes + (kFp8 ? kWtStages * (kCodes + kExps) : 0) + 1024;
  // D f32, M = 128; A / B type in bits 7 and 10 (0 f16, 1 bf16); N in bits 17-22.
  static constexpr uint32_t kType = kF16 ? 0u : (1u << 7) | (1u << 10);
  static constexpr uint32_t kIdQK = (1u << 4) | kType | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t kIdPV = (1u << 4) | kType | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24) | (1u << 16);
  // How far a score may pass the reference, and the shift of the weights
  // (log2): f16 weights stay below 2^16 and normal down to 2^-21.
  static constexpr float kStep = kF16 ? 8.f : 16.f;
  static constexpr float kShift = kF16 ? 7.f : 0.f;
};

struct WtItem {
  int32_t ntok;           // new tokens; 0: no such item, -1 in the ring: no more
  int32_t h;
  int32_t t0, table;      // the sequence's page table
  int32_t row;            // first row of q and out
  int32_t p_lo, p_hi;     // positions of its first and last token
  WinPages wp;
  int32_t shift, nchunks;
  int32_t first;          // pages [first, wp.count) of the list are this CTA's
};

constexpr int kWtItems = 2;  // items of the ring
constexpr int kWtSplit = 8;  // CTAs that share an item at most
constexpr int kWtAhead = 2;  // tiles of an item still to be asked for when the next is claimed
struct WtBars {
  uint64_t kv_full[4], kv_empty[4];
  uint64_t st_full[kWtStages], st_empty[kWtStages];
  uint64_t s_full[2];                   // per sub-tile: scores ready (and the previous P.V in O)
  uint64_t p_full[2][2];                // and half of the tile: weights ready
  uint64_t o_full[2];                   // once an item: its last P.V is in O
  uint64_t turn[2];                     // the other sub-tile's products of a tile are issued
  uint64_t q_raw[2];                    // f16: bf16 rows of Q in place, to be converted
  uint64_t q_full[2], q_empty[2];       // Q ready / the item's last scores done
  uint64_t item_full[kWtItems], item_empty[kWtItems];
  uint64_t late;                        // an item's last tiles are being asked for
  uint64_t claim;                       // the answer to a claim has come
  uint64_t join;                        // split: both sub-tiles' last P.V are in O
  WtItem items[kWtItems];
  alignas(16) uint4 answer;
  uint32_t tmem_base;
  int abort;
};

// Unit `u` of the launch, late tokens first; ntok = 0 for a surplus one. Tiles
// are counted in tokens: `per` of them make an item. The launch keeps units and
// rows * g below 2^31.
// An item split over a cluster is cut at whole tiles: share `rank` of `nsplit`.
__device__ __forceinline__ void wt_item(const WinArgs& a, int32_t per, int32_t u, int rank, int nsplit, WtItem& it) {
  const uint32_t unit = gridDim.x / nsplit - 1 - (uint32_t)u, tile_id = unit / (uint32_t)a.Hkv;
  it.ntok = 0;
  it.h = (int32_t)(unit - tile_id * (uint32_t)a.Hkv);
  int32_t s, tile;
  win_tile(a, 1, per, tile_id, s, tile);
  const SeqRows sr = seq_rows(a.row_indptr, a.num_tokens, a.num_rows, s);
  if (tile < 0 || tile > sr.m / per) return;
  it.ntok = min(per, sr.m - tile * per);
  if (it.ntok <= 0) return;
  it.row = sr.r0 + tile * per;
  it.p_lo = sr.pos0 + tile * per;
  it.p_hi = it.p_lo + it.ntok - 1;
  it.t0 = a.page_indptr[s];
  it.table = a.page_indptr[s + 1] - it.t0;
  it.wp = win_pages(a.window, a.sinks, it.p_lo, it.p_hi);
  it.shift = (it.wp.wp - it.wp.ns) * kPageSize;
  const int32_t tiles = (it.wp.count + kTcPagesPerTile - 1) / kTcPagesPerTile;
  it.first = (int32_t)((int64_t)tiles * rank / nsplit) * kTcPagesPerTile;
  it.wp.count = min(it.wp.count, (int32_t)((int64_t)tiles * (rank + 1) / nsplit) * kTcPagesPerTile);
  it.nchunks = (it.wp.count - it.first + kWtChunk / kPageSize - 1) / (kWtChunk / kPageSize);
}
// Table entry of page v of the CTA's share of the list as it stands (0xFFFFFFFF past the
// list or the table): looked up a tile ahead, and judged when it is used, so
// that nobody waits for it.
__device__ __forceinline__ uint32_t wt_entry(const WinArgs& a, const WtItem& it, int32_t v) {
  const int32_t idx = it.wp.page(it.first + v);
  return it.first + v < it.wp.count && idx < it.table ? (uint32_t)a.page_indices[it.t0 + idx] : 0xFFFFFFFFu;
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

// One arrival for a warp that is through with something (32 would queue up at
// the barrier's address).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The same value in every lane, known as such.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ int32_t uniform(int32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// Whole-warp forms: one elected lane (the same for every call) issues.
__device__ __forceinline__ void umma_commit_one(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred l;\n elect.sync _|l, 0xffffffff;\n"
      " @l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
      : "memory");
}
// Shared-memory descriptors: 128-byte swizzle, 1024 bytes from 8 rows to the
// next 8; the leading offset and the start address, in 16-byte units, make the
// low word.
constexpr uint32_t kWtDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// S = Q K^T: D / 16 products, 16 dims (32 bytes) apart, 64-dim halves `half` apart.
template <int D, uint32_t kId>
__device__ __forceinline__ void umma_qk(uint32_t d, uint32_t a, uint32_t b, uint32_t half) {
  a |= 1u << 16;
  b |= 1u << 16;
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
    asm volatile(
        "{\n .reg .pred l, t, f;\n .reg .b64 da, db;\n .reg .b32 a, b;\n"
        " elect.sync _|l, 0xffffffff;\n setp.ne.b32 f, %5, 0;\n setp.eq.b32 t, 0, 0;\n"
        " mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
        " @l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, f;\n"
        " add.u32 a, %1, 2;\n add.u32 b, %2, 2;\n mov.b64 da, {a, %3};\n mov.b64 db, {b, %3};\n"
        " @l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, t;\n"
        " add.u32 a, %1, 4;\n add.u32 b, %2, 4;\n mov.b64 da, {a, %3};\n mov.b64 db, {b, %3};\n"
        " @l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, t;\n"
        " add.u32 a, %1, 6;\n add.u32 b, %2, 6;\n mov.b64 da, {a, %3};\n mov.b64 db, {b, %3};\n"
        " @l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, t;\n}" ::"r"(d),
        "r"(a + h * half), "r"(b + h * half), "n"(kWtDescHi), "n"(kId), "r"(h));
}
// O += P V over 64 tokens: 4 products, P 8 TMEM columns and V 16 rows (2 KB) apart.
template <uint32_t kId>
__device__ __forceinline__ void umma_pv(uint32_t d, uint32_t p, uint32_t b, uint32_t half, uint32_t acc) {
  b |= half << 16;
  asm volatile(
      "{\n .reg .pred l, t, f;\n .reg .b64 db;\n .reg .b32 b, p;\n"
      " elect.sync _|l, 0xffffffff;\n setp.ne.b32 f, %5, 0;\n setp.eq.b32 t, 0, 0;\n"
      " mov.b64 db, {%2, %3};\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, f;\n"
      " add.u32 p, %1, 8;\n add.u32 b, %2, 128;\n mov.b64 db, {b, %3};\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [p], db, %4, t;\n"
      " add.u32 p, %1, 16;\n add.u32 b, %2, 256;\n mov.b64 db, {b, %3};\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [p], db, %4, t;\n"
      " add.u32 p, %1, 24;\n add.u32 b, %2, 384;\n mov.b64 db, {b, %3};\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [p], db, %4, t;\n}" ::"r"(d),
      "r"(p), "r"(b), "n"(kWtDescHi), "n"(kId), "r"(acc));
}
// Claims a CTA of this launch that has not started yet (16 bytes at `answer`,
// counted by `bar`), and its index; -1 if there is none left.
__device__ __forceinline__ void claim_cta(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int32_t claimed_cta(const uint4* answer) {
  int32_t u;
  asm volatile(
      "{\n .reg .b128 r;\n .reg .pred p;\n ld.shared.b128 r, [%1];\n mov.b32 %0, -1;\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n}"
      : "=r"(u)
      : "r"(smem_u32(answer))
      : "memory");
  return u;
}
// 4-D TMA load (Q rows: dims, heads, head groups, tokens).
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                                            int32_t w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_tma_4d(const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(x), "r"(y),
               "r"(z), "r"(w)
               : "memory");
}

// 64 bytes of this thread's row of out: whole 32-byte sectors at a time where
// the address allows (16 bytes at a time are twice the requests, and the rows
// of a warp are as many lines apart).
__device__ __forceinline__ void store16(uint16_t* out, const uint32_t (&w)[16], bool wide) {
  if (wide) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + 16 * k), "r"(w[8 * k]),
                   "r"(w[8 * k + 1]), "r"(w[8 * k + 2]), "r"(w[8 * k + 3]), "r"(w[8 * k + 4]), "r"(w[8 * k + 5]),
                   "r"(w[8 * k + 6]), "r"(w[8 * k + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      reinterpret_cast<uint4*>(out)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  }
}

__device__ __forceinline__ void tmem_st8u(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// This thread's O row times f (rare: kept small rather than fast).
template <int D>
__device__ __forceinline__ void wt_rescale(uint32_t taddr, float f) {
#pragma unroll 1
  for (int c = 0; c < D; c += 16) {
    uint32_t v[16];
    tmem_ld16u(taddr + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    tmem_st16u(taddr + c, v);
  }
  tmem_wait_st();
}

// Weights of 32 scores, to the products' type (bf16: the second terms 32 columns
// on); their f32 sum is added to acc.
template <bool kF16>
__device__ __forceinline__ void wt_weights(const float (&s)[32], uint64_t sc2, uint64_t nm2, uint64_t& acc, uint32_t taddr) {
#pragma unroll
  for (int j = 0; j < 32; j += 16) {  // eight columns at a time: sixteen cost registers (MXFP8 chunks 107 us, 102)
    uint32_t w[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t x = f2_fma(f2_pack(s[j + 2 * i], s[j + 2 * i + 1]), sc2, nm2);
      const uint64_t e = f2_pack(fast_exp2(f2_lo(x)), fast_exp2(f2_hi(x)));
      acc = f2_add(acc, e);
      if constexpr (kF16)
        w[i] = pack_f16x2(f2_lo(e), f2_hi(e));
      else
        split_bf16x2_packed(e, w[i], lo[i]);
    }
    tmem_st8u(taddr + j / 2, w);
    if constexpr (!kF16) tmem_st8u(taddr + 32 + j / 2, lo);
  }
}

// kSplit false: nsplit is 1, known as such (the code of the shares cost the
// others 1 to 3%).
template <int D, int KV, bool kSplit>
__global__ void __maxnreg__((WtCfg<D, KV>::kRegs))
    win_tc_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map, WinArgs a,
                  int cluster) {
  const int nsplit = kSplit ? cluster : 1;
  using Cfg = WtCfg<D, KV>;
  constexpr bool kFp8 = Cfg::kFp8, kF16 = Cfg::kF16, kHeld = Cfg::kHeld;
  constexpr int kSlots = Cfg::kSlots, kTile = Cfg::kTileBytes, kHalf = Cfg::kHalfBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ WtBars bars;
  __shared__ float join_m[256], join_l[256];  // split: the rows' references and sums
  __shared__ float join_w[kWtSplit][256];     // and the weights of their shares
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_s = smem;                        // [sub-tile][half][128 rows][128 B]
  uint8_t* slots = smem + 2 * kTile;          // [slot][half][128 rows][128 B]
  uint8_t* stages = slots + kSlots * kTile;   // FP8: [stage][128 rows][D]
  uint8_t* stage_exps = stages + kWtStages * Cfg::kCodes;  // [stage][128 rows][D / 32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = 128 / a.g;  // tokens of a sub-tile
  WsHeader* err = reinterpret_cast<WsHeader*>(a.status);
  const int rank = blockIdx.x % nsplit;
  constexpr int kPitch = D + 4;  // of a row of the outputs that are joined, f32, in place of Q, K and V
  static_assert(256 * kPitch * 4 <= (2 + kSlots) * kTile);
  float* join_o = reinterpret_cast<float*>(smem);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars.kv_full[s], kFp8 ? kWtConvWarps : 1);
      mbar_init(&bars.kv_empty[s], 2);  // both sub-tiles' issuers
    }
    for (int s = 0; s < kWtStages; ++s) {
      mbar_init(&bars.st_full[s], 1);
      mbar_init(&bars.st_empty[s], kWtConvWarps);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars.s_full[x], 1);
      for (int h = 0; h < 2; ++h) mbar_init(&bars.p_full[x][h], 4);
      mbar_init(&bars.o_full[x], 1);
      mbar_init(&bars.turn[x], 1);
      mbar_init(&bars.q_raw[x], 1);
      mbar_init(&bars.q_full[x], kF16 ? 4 : 1);
      mbar_init(&bars.q_empty[x], 1);
    }
    for (int s = 0; s < kWtItems; ++s) {
      mbar_init(&bars.item_full[s], 1);
      mbar_init(&bars.item_empty[s], 8 + (kFp8 ? kWtConvWarps : 0) + 3);
    }
    mbar_init(&bars.late, 1);
    mbar_init(&bars.claim, 1);
    mbar_init(&bars.join, 8);
    bars.items[0].ntok = 0;
    bars.abort = 0;
    fence_mbar_init();
    mbar_arrive(&bars.turn[0]);  // sub-tile A begins
  }
  if (warp == Cfg::kProducer + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&bars.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == Cfg::kProducer * 32) {
    prefetch_tmap(&kv_map);
    prefetch_tmap(&q_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars.tmem_base;
  volatile int* abort = &bars.abort;
  // A warp's view of the item ring: the next item, or ntok = -1 after the last
  // one (and after an abort). The slot is given back once the warp has copied it.
  int item_k = 0;
  auto next_item = [&](WtItem& it) {
    const int s = item_k % kWtItems;
    const bool got = __all_sync(0xffffffffu, mbar_wait(&bars.item_full[s], (item_k / kWtItems) & 1, abort, err));
    it = bars.items[s];
    if (!got) it.ntok = -1;
    __syncwarp();
    if (got && lane == 0) mbar_arrive(&bars.item_empty[s]);
    ++item_k;
    return it.ntok > 0;
  };
  WtItem it;

  if (warp < 8) {
    // ----------------------------------------------------------------- softmax
    if constexpr (kHeld) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoftmax) : "memory");
    const int x = warp >> 2;        // sub-tile
    const int quarter = warp & 3;   // TMEM lanes [32 * quarter, + 32)
    const int r = quarter * 32 + lane;
    const int tok = x * sub + r / a.g, head = r % a.g;  // this thread's token of an item, head of the group
    const uint32_t lane_base = tbase + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_col = lane_base + col_s(x), o_col = lane_base + col_o(x);
    float scale_log2 = a.scale_log2, v_scale = 1.f;  // of the current item
    int g0 = 0;                // ring index of the item's first K tile
    int n = 0;                 // items of this sub-tile so far
    int tiles = 0;             // its tiles so far
    bool ok = true;
    // f16: this thread's row of the item's Q, bf16 as loaded, to f16 in place;
    // returns the power of two that it was multiplied by. The sign of the head's
    // K scale goes into the row, and so does NaN: the maximum is taken before the
    // scale, and a masked score, -inf, has to stay that.
    auto convert_q = [&]() {
      int up = 0;
      if constexpr (kF16) {
        ok = mbar_wait(&bars.q_raw[x], n & 1, abort, err) && ok;
        uint8_t* qx = q_s + x * kTile + r * 128;
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(qx + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
        }
        up = f16_row_shift(top);
        float by = __uint_as_float((uint32_t)(127 + up) << 23);
        const float k_scale = reinterpret_cast<const float*>(a.scales)[it.h];
        if (!(k_scale >= 0.f)) by = k_scale < 0.f ? -by : k_scale;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4* at = reinterpret_cast<uint4*>(qx + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4));
          uint4 v = *at;
          v.x = bf16x2_to_f16x2(v.x, by);
          v.y = bf16x2_to_f16x2(v.y, by);
          v.z = bf16x2_to_f16x2(v.z, by);
          v.w = bf16x2_to_f16x2(v.w, by);
          *at = v;
        }
        fence_proxy_async_smem();
        warp_arrive(&bars.q_full[x]);
      }
      return up;
    };
    auto is_active = [&](const WtItem& q) { return q.nchunks > 0 && q.ntok > x * sub; };
    bool have = next_item(it);
    int up = have && is_active(it) ? convert_q() : 0;
    while (have) {
      const WtItem cur = it;
      const bool active = is_active(cur);
      if constexpr (kF16) {
        // Above zero, which would make NaN of the -inf of a masked score (the
        // scores of a row of zeros, whose power of two is the largest, stay zero).
        scale_log2 = fmaxf(f16_score_scale(a.scale_log2, up) * fabsf(reinterpret_cast<const float*>(a.scales)[cur.h]), FLT_MIN);
        v_scale = reinterpret_cast<const float*>(a.scales)[a.Hkv + cur.h];
      }
      const int32_t p = cur.p_lo + tok;
      const int32_t hi = p - cur.shift, lo = a.window ? p - a.window + 1 - cur.shift : 0;
      const int nchunks = active ? cur.nchunks : 0;
      const int pj = lane & (kTcPagesPerTile - 1);
      uint32_t entry = nchunks > 0 ? wt_entry(a, cur, pj) : 0xFFFFFFFFu;
      float m_used = -INFINITY;
      uint64_t lsum = 0ull;
      const uint64_t sc2 = f2_pack(scale_log2, scale_log2);
      for (int c = 0; c < nchunks; c += 2) {
        const int32_t x0 = cur.first * kPageSize + c * kWtChunk;
        const bool two = c + 1 < nchunks;
        // Which of the tile's pages exist.
        const uint32_t pages = __ballot_sync(0xffffffffu, entry < (uint32_t)a.num_pages) & 0xffu;
        entry = wt_entry(a, cur, (c / 2 + 1) * kTcPagesPerTile + pj);
        const bool seen_whole = wt_whole(a, cur, x0, kTcTok), whole = pages == 0xffu && seen_whole;
        float s[kHeld ? 4 : 2][32];
        // Scores of half h, those that the row does not see as -inf.
        auto load = [&](int h) {
          float(*sh)[32] = s + (kHeld ? 2 * h : 0);
          tmem_ld32(s_col + kWtChunk * h, sh[0]);
          tmem_ld32(s_col + kWtChunk * h + 32, sh[1]);
          if (!kHeld || h == 1 || !two) tmem_wait_ld();
        };
        auto mask = [&](int h) {
          float(*sh)[32] = s + (kHeld ? 2 * h : 0);
          if (whole) return;
          auto below = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // bit k: the row sees token x0 + 64 h + 32 i + k
            const int32_t b = x0 + kWtChunk * h + 32 * i;
            uint32_t see = below(hi - b + 1) & (~below(lo - b) | below(a.sinks - b));
            if (!((pages >> (4 * h + 2 * i)) & 1)) see &= 0xffff0000u;
            if (!((pages >> (4 * h + 2 * i + 1)) & 1)) see &= 0x0000ffffu;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1)) sh[i][k] = -INFINITY;
          }
        };
        // (A NaN or infinite score passes the maximum by or makes it infinite;
        // its exponential is NaN either way, and with it the row's sum.)
        auto row_max = [&](int h) {
          const float(*sh)[32] = s + (kHeld ? 2 * h : 0);
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* v = &sh[i / 2][16 * (i % 2)];
            mx[i] = fmaxf(v[0], v[1]);
#pragma unroll
            for (int k = 2; k < 16; k += 2) mx[i] = max3f(mx[i], v[k], v[k + 1]);
          }
          return max3f(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
        };
        ok = ok && mbar_wait(&bars.s_full[x], tiles & 1, abort, err);
        ++tiles;
        tc_fence_after();
        load(0);
        if (kHeld && two) load(1);
        mask(0);
        float mt = row_max(0);
        if (two) {
          if (!kHeld) load(1);
          mask(1);
          mt = fmaxf(mt, row_max(1));
        }
        mt = ok ? mt * scale_log2 : m_used;
        if (__any_sync(0xffffffffu, mt > m_used + Cfg::kStep)) {
          const float m_new = mt > m_used + Cfg::kStep ? ceilf(mt) : m_used;
          const float f = m_used == m_new ? 1.f : exp2f(m_used - m_new);  // a power of two
          if (c > 0) wt_rescale<D>(o_col, f);
          lsum = f2_fma(lsum, f2_pack(f, f), 0ull);
          m_used = m_new;
        }
        // bf16 pages: V of slots that no row sees, before any of the tile's
        // products (each sub-tile's threads for itself, a token each).
        if (!kFp8 && !seen_whole) {
          const int vi = g0 + c + 1;
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
        const float ref = (m_used == -INFINITY ? 0.f : m_used) - Cfg::kShift;
        const uint64_t nm2 = f2_pack(-ref, -ref);
        auto hand_over = [&](int h) {
          float(*sh)[32] = s + (kHeld ? 2 * h : 0);
          wt_weights<kF16>(sh[0], sc2, nm2, lsum, s_col + kWtChunk * h);
          wt_weights<kF16>(sh[1], sc2, nm2, lsum, s_col + kWtChunk * h + 16);
          tmem_wait_st();
          tc_fence_before();
          warp_arrive(&bars.p_full[x][h]);
        };
        if (two) {
          hand_over(1);
          if (!kHeld) {  // again
            load(0);
            mask(0);
          }
        }
        hand_over(0);
      }
      g0 += 2 * ((cur.nchunks + 1) / 2);
      if (active) ++n;
      have = next_item(it);
      // The next item's Q before this epilogue: its first scores overlap it
      // (its first P.V, which overwrites O, waits for this thread's weights).
      const int up_next = have && is_active(it) ? convert_q() : 0;
      if (active) {
        ok = mbar_wait(&bars.o_full[x], (n - 1) & 1, abort, err) && ok;
        __syncwarp();
        tc_fence_after();
      }
      {
        const bool live = r < sub * a.g && tok < cur.ntok, wide = ((uintptr_t)a.out & 31) == 0;
        const float L = f2_lo(lsum) + f2_hi(lsum);
        const float inv = L == 0.f ? 0.f : v_scale / L;
        const int64_t dst = (int64_t)(cur.row + tok) * a.Hq + qo_head_of(a.gqa_map, cur.h, head, a.Hkv, a.g);
        if (nsplit > 1) {  // both sub-tiles' products are done: their operands' place is free
          warp_arrive(&bars.join);
          ok = mbar_wait(&bars.join, 0, abort, err) && ok;
          __syncwarp();
          join_m[x * 128 + r] = m_used - Cfg::kShift;
          join_l[x * 128 + r] = L;
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (active) {
            tmem_ld32(o_col + c * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.f;
          }
          if (nsplit > 1) {
            float4* to = reinterpret_cast<float4*>(join_o + (x * 128 + r) * kPitch + c * 32);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              to[k] = make_float4(o[4 * k] * inv, o[4 * k + 1] * inv, o[4 * k + 2] * inv, o[4 * k + 3] * inv);
          } else if (live) {
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + dst * D + c * 32;
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = pack_bf16x2(o[2 * k] * inv, o[2 * k + 1] * inv);
            store16(out, w, wide);
          }
        }
        if (nsplit == 1 && live && a.lse)
          a.lse[dst] = L == 0.f ? -INFINITY : (m_used - Cfg::kShift + log2f(L)) * kLn2;
      }
      up = up_next;
      tc_fence_before();
      if (!__all_sync(0xffffffffu, ok)) break;
    }
  } else if (kFp8 && warp < 12) {
    // -------------------------------------------------------------- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsConvert) : "memory");
    // A thread widens 16 codes of one token at a time; eight neighbouring
    // threads cover two rows, so their stores fall into eight bank groups.
    const int t = threadIdx.x - 256;
    constexpr int kConvThreads = 32 * kWtConvWarps;
    constexpr int kChunks = kTcTok * D / 16;
    int gidx = 0;
    bool ok = true;
    while (ok && next_item(it)) {
      const int pj = lane & (kTcPagesPerTile - 1);
      uint32_t entry = wt_entry(a, it, pj), pages = 0;
      const int ntiles = (it.nchunks + 1) / 2;
      for (int idx = 0; idx < 2 * ntiles; ++idx, ++gidx) {
        const int su = gidx % kWtStages, s = gidx % kSlots;
        if ((idx & 1) == 0) {  // the tile's pages that exist; the next tile's ids on their way
          pages = __ballot_sync(0xffffffffu, entry < (uint32_t)a.num_pages);
          entry = wt_entry(a, it, ((idx >> 1) + 1) * kTcPagesPerTile + pj);
        }
        ok = mbar_wait(&bars.st_full[su], (gidx / kWtStages) & 1, abort, err) &&
             (gidx < kSlots || mbar_wait(&bars.kv_empty[s], ((gidx / kSlots) - 1) & 1, abort, err));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* src = stages + su * Cfg::kCodes;
        const uint8_t* exps = stage_exps + su * Cfg::kExps;
        uint8_t* dst = slots + s * kTile;
        const int32_t x0 = it.first * kPageSize + (idx >> 1) * kTcTok;
        const bool clean = (pages & 0xffu) == 0xffu && wt_whole(a, it, x0, kTcTok);
        // Two chunks at a time, both read before the first is stored: no load
        // may pass a store that could be to its address, so one at a time each
        // waits for the one before (the calls named at kHeld, with weights of one
        // term: MXFP8 92 us -> 84, E4M3 306 -> 292, as long as without any widening;
        // four: 84, 295).
        constexpr int kBatch = 2;
#pragma unroll 1
        for (int i0 = 0; i0 < kChunks / kConvThreads; i0 += kBatch) {
          uint4 codes[kBatch];
          uint8_t ex[kBatch];
          auto where = [&](int i, int& row, int& c) {  // token, 16-dim chunk
            const int id = t + (i0 + i) * kConvThreads;
            if constexpr (D == 128) {
              row = ((id >> 4) << 1) | ((id >> 2) & 1);
              c = ((id >> 3) & 1) * 4 + (id & 3);
            } else {
              row = id >> 2;
              c = id & 3;
            }
          };
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            int row, c;
            where(i, row, c);
            codes[i] = *reinterpret_cast<const uint4*>(D == 128 ? src + row * 128 + ((c ^ (row & 7)) << 4)
                                                                : src + row * 64 + (c << 4));
            if constexpr (!kF16) ex[i] = exps[row * (D / 32) + (c >> 1)];
          }
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            int row, c;
            where(i, row, c);
            uint32_t o[8];
            if constexpr (kF16) {
              const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) e4m3x4_f16(w[k], o[2 * k], o[2 * k + 1]);
            } else {
              e4m3x16_to_bf16(codes[i], e8m0_to_float(ex[i]), o);
            }
            // Slots that no row sees, and missing pages (their exponents are stale).
            if (!clean && (!((pages >> (row >> 4)) & 1) || !wt_seen(a, it, x0 + row))) {
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = 0;
            }
            uint8_t* drow = dst + (c >> 2) * kHalf + row * 128;
            const int cl = c & 3;
            *reinterpret_cast<uint4*>(drow + (((2 * cl) ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(drow + (((2 * cl + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&bars.kv_full[s]);
        if (lane == 0) mbar_arrive(&bars.st_empty[su]);
      }
    }
  } else {
    if constexpr (kHeld) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsRest) : "memory");
    if (warp == Cfg::kProducer) {
      // ---------------------------------------------------------------- producer
      const int64_t rows_total = (int64_t)a.num_pages * 2 * a.Hkv * kPageSize;
      const int pj = lane & (kTcPagesPerTile - 1);
      const bool mine = lane < kTcPagesPerTile;
      int gidx = 0;
      bool ok = true;
      while (ok && next_item(it)) {
        uint32_t cur = wt_entry(a, it, pj), nxt = 0xFFFFFFFFu;
        const int ntiles = (it.nchunks + 1) / 2, late = 2 * max(ntiles - kWtAhead, 0);
        if (ntiles == 0 && lane == 0) mbar_arrive(&bars.late);
        for (int idx = 0; idx < 2 * ntiles; ++idx, ++gidx) {
          const int j = idx >> 1, kv = idx & 1;
          if (idx == late && lane == 0) mbar_arrive(&bars.late);
          // A missing page reads past the pool's end: zeros.
          const bool have = mine && cur < (uint32_t)a.num_pages;
          const int32_t v = it.first + j * kTcPagesPerTile + pj;
          if (kv == 0 && mine && !have && v < it.wp.count) {
            const int32_t at = it.wp.page(v);
            win_report(a.status, kDevErrBadPage, at < it.table ? cur : (uint32_t)at);
          }
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
          if (kv == 0)
            nxt = wt_entry(a, it, (j + 1) * kTcPagesPerTile + pj);
          else
            cur = nxt;
        }
      }
    } else if (warp <= Cfg::kProducer + 2) {
      // ----------------------------------------------------------------- issuers
      // A warp for each sub-tile: a product is accepted only when the one before
      // it has all but run, and even a wait for a barrier that is already complete
      // costs 85 cycles, so one warp for both left the tensor core idle at every
      // wait. The whole warp walks the list, every branch taken on a vote, and one
      // elected lane issues, several products to an asm block.
      const int x = warp - Cfg::kProducer - 1;
      // 16-byte units; in a cluster the address also names the CTA, above bit 17.
      const uint32_t q_addr = ((smem_u32(q_s) + x * kTile) & 0x3ffff) >> 4, s_addr = (smem_u32(slots) & 0x3ffff) >> 4;
      const uint32_t tb = uniform(tbase);
      int g0 = 0;              // ring index of the item's first K tile
      int n = 0;               // items of this sub-tile
      int turns = 0;           // turns taken
      int used[2] = {0, 0};    // its first and second halves of tiles
      bool ok = true;
      auto wait = [&](uint64_t* bar, int phase) {
        const bool all = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort, err));
        tc_fence_after();
        return all;
      };
      while (ok) {
        next_item(it);
        const int nchunks = uniform(it.nchunks), ntok = uniform(it.ntok);
        if (ntok <= 0) break;
        const int ntiles = (nchunks + 1) / 2;
        if (ntok <= x * sub) {
          // Nothing to issue here: the tiles are given back as they come.
          for (int i = g0; ok && i < g0 + 2 * ntiles; ++i) {
            ok = wait(&bars.kv_full[i % kSlots], i / kSlots);
            if (ok && lane == 0) mbar_arrive(&bars.kv_empty[i % kSlots]);
            __syncwarp();
          }
          g0 += 2 * ntiles;
          continue;
        }
        if (nchunks == 0) continue;
        // With both sub-tiles at work their products are issued in turn, a tile's
        // last P.V and the next Q.K together: issued as they come, both sub-tiles
        // fall into step, their softmaxes share the exponential unit and then
        // their products the tensor core (4650 cycles a tile).
        const bool both = ntok > sub;
        auto my_turn = [&]() { return !both || wait(&bars.turn[x], turns++); };
        auto your_turn = [&]() {
          if (both && lane == 0) mbar_arrive(&bars.turn[1 - x]);
          __syncwarp();
        };
        // Scores of tile j; what is free after them.
        auto issue_qk = [&](int j) {
          const int slot = (g0 + 2 * j) % kSlots;
          umma_qk<D, Cfg::kIdQK>(tb + col_s(x), q_addr, s_addr + (slot * kTile >> 4), kHalf >> 4);
          umma_commit_one(&bars.s_full[x]);
          umma_commit_one(&bars.kv_empty[slot]);
          if (j == ntiles - 1) umma_commit_one(&bars.q_empty[x]);
        };
        ok = wait(&bars.q_full[x], n++) && wait(&bars.kv_full[g0 % kSlots], g0 / kSlots) && my_turn();
        if (!ok) break;
        issue_qk(0);
        your_turn();
        for (int j = 0; ok && j < ntiles; ++j) {
          const int vi = g0 + 2 * j + 1, ki = vi + 1, slot = vi % kSlots;
          const uint32_t o = tb + col_o(x), p = tb + col_s(x), v = s_addr + (slot * kTile >> 4);
          const bool two = 2 * j + 1 < nchunks, more = j + 1 < ntiles;
          auto product = [&](uint32_t pt, uint32_t vt, uint32_t acc) {  // of 64 tokens; bf16: of both terms
            umma_pv<Cfg::kIdPV>(o, pt, vt, kHalf >> 4, acc);
            if constexpr (!kF16) umma_pv<Cfg::kIdPV>(o, pt + 32, vt, kHalf >> 4, 1u);
          };
          ok = wait(&bars.kv_full[slot], vi / kSlots) && (!more || wait(&bars.kv_full[ki % kSlots], ki / kSlots));
          if (two) {
            ok = ok && wait(&bars.p_full[x][1], used[1]++);
            if (!ok) break;
            product(p + kWtChunk, v + (kWtChunk * 128 >> 4), j > 0 ? 1u : 0u);
          }
          ok = ok && my_turn() && wait(&bars.p_full[x][0], used[0]++);
          if (!ok) break;
          product(p, v, j > 0 || two ? 1u : 0u);
          umma_commit_one(&bars.kv_empty[slot]);
          if (more)
            issue_qk(j + 1);
          else
            umma_commit_one(&bars.o_full[x]);
          your_turn();
        }
        g0 += 2 * ntiles;
      }
    } else {
      // --------------------------------------------------- scheduler and Q loader
      // Publishes an item, loads its Q once the scores of the one before are
      // done, and claims the next when the item's last tiles are asked for.
      int n[2] = {0, 0}, claims = 0;
      int32_t u = (int32_t)blockIdx.x / nsplit;
      bool ok = true;
      const bool tiled = a.gqa_map == DD_GQA_TILED;
      auto claim = [&]() {
        if (nsplit > 1) {  // as many CTAs as the GPU has room for: one item each
          u = -1;
          return;
        }
        __syncwarp();
        if (lane == 0) {
          fence_proxy_async_smem();  // the last answer has been read
          mbar_arrive_expect_tx(&bars.claim, 16);
          claim_cta(&bars.answer, &bars.claim);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.claim, claims++ & 1, abort, err));
        u = ok && lane == 0 ? claimed_cta(&bars.answer) : -1;
        u = __shfl_sync(0xffffffffu, u, 0);
      };
      for (int k = 0;; ++k) {
        it.ntok = -1;
        while (u >= 0) {
          wt_item(a, 2 * sub, u, rank, nsplit, it);
          if (it.ntok > 0) break;
          it.ntok = -1;
          claim();
        }
        const int s = k % kWtItems;
        ok = ok && __all_sync(0xffffffffu, k < kWtItems || mbar_wait(&bars.item_empty[s], ((k / kWtItems) - 1) & 1, abort, err));
        if (!ok) break;
        if (lane == 0) {
          bars.items[s] = it;
          mbar_arrive(&bars.item_full[s]);
        }
        __syncwarp();
        if (u < 0) break;
        // Into L2 first, while the buffers are still in use.
        if (lane == 0 && it.nchunks > 0)
          for (int x = 0; x < 2 && it.ntok > x * sub; ++x)
            for (int hf = 0; hf < Cfg::kHalves; ++hf)
              prefetch_tma_4d(&q_map, 64 * hf, tiled ? it.h : 0, tiled ? 0 : it.h, it.row + x * sub);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (it.nchunks == 0 || it.ntok <= x * sub) break;
          ok = __all_sync(0xffffffffu, n[x] == 0 || mbar_wait(&bars.q_empty[x], (n[x] - 1) & 1, abort, err));
          if (!ok) break;
          ++n[x];
          if (lane == 0) {
            uint64_t* bar = kF16 ? &bars.q_raw[x] : &bars.q_full[x];
            mbar_arrive_expect_tx(bar, Cfg::kHalves * sub * a.g * 128);
#pragma unroll
            for (int hf = 0; hf < Cfg::kHalves; ++hf)
              tma_load_4d(q_s + x * kTile + hf * kHalf, &q_map, 64 * hf, tiled ? it.h : 0, tiled ? 0 : it.h,
                          it.row + x * sub, bar);
          }
          __syncwarp();
        }
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars.late, k & 1, abort, err));
        if (!ok) break;
        claim();
        if (!ok) break;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort) {  // a wait ran out: what is still in flight lands before the CTA leaves
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 200000) {
    }
  }
  if (nsplit > 1) {  // the shares of an item's rows: their weights, then their sum
    cluster_barrier();
    const WtItem& one = bars.items[0];
    const int rows = one.ntok > sub ? 128 + (one.ntok - sub) * a.g : max(one.ntok, 0) * a.g;
    auto place = [&](int row) {  // in out, -1 for a row of the tile that stands for nothing
      const int x = row >> 7, r = row & 127;
      if (row >= rows || r >= sub * a.g) return (int64_t)-1;
      return (int64_t)(one.row + x * sub + r / a.g) * a.Hq + qo_head_of(a.gqa_map, one.h, r % a.g, a.Hkv, a.g);
    };
    if (threadIdx.x < 256) {
      const int row = threadIdx.x;
      const int64_t dst = place(row);
      const uint32_t am = smem_u32(&join_m[row]), al = smem_u32(&join_l[row]);
      float m[kWtSplit], l[kWtSplit], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWtSplit; ++k) {
        m[k] = dst >= 0 && k < nsplit ? cluster_ld(am, k) : -INFINITY;
        l[k] = dst >= 0 && k < nsplit ? cluster_ld(al, k) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < kWtSplit; ++k) top = fmaxf(top, m[k]);
#pragma unroll
      for (int k = 0; k < kWtSplit; ++k) {
        l[k] *= exp2f(m[k] - (top == -INFINITY ? 0.f : top));
        sum += l[k];
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < kWtSplit; ++k) join_w[k][row] = l[k] * inv;
      if (dst >= 0 && rank == 0 && a.lse) a.lse[dst] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
    __syncthreads();
    constexpr int kVecs = D / 4, kStep = 4;  // 16 bytes of four rows at a time
    const int quads = (rows + kStep - 1) / kStep * kVecs;
    for (int i = threadIdx.x + rank * Cfg::kThreads; i < quads; i += nsplit * Cfg::kThreads) {
      const int row = i / kVecs * kStep, d = i % kVecs * 4;
      const uint32_t ao = smem_u32(join_o + row * kPitch + d);
      float4 acc[kStep];
#pragma unroll
      for (int t = 0; t < kStep; ++t) acc[t] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < nsplit; ++k) {
        float4 y[kStep];
#pragma unroll
        for (int t = 0; t < kStep; ++t) y[t] = cluster_ld4(ao + t * kPitch * 4, k);
#pragma unroll
        for (int t = 0; t < kStep; ++t) {
          const float w = join_w[k][row + t];
          acc[t].x = fmaf(w, y[t].x, acc[t].x), acc[t].y = fmaf(w, y[t].y, acc[t].y);
          acc[t].z = fmaf(w, y[t].z, acc[t].z), acc[t].w = fmaf(w, y[t].w, acc[t].w);
        }
      }
#pragma unroll
      for (int t = 0; t < kStep; ++t) {
        const int64_t dst = place(row + t);
        if (dst >= 0)
          *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + dst * D + d) =
              make_uint2(pack_bf16x2(acc[t].x, acc[t].y), pack_bf16x2(acc[t].z, acc[t].w));
      }
    }
    cluster_barrier();  // no CTA leaves while another reads its rows
  }
  if (warp == Cfg::kProducer + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kTmemCols)
                 : "memory");
  }
}

int make_kv_tensor_map(CUtensorMap* map, const void* kv, int64_t num_pages, int Hkv, int D,
                       int elem_bytes, int two_halves);
int make_q_tensor_map(CUtensorMap* map, const void* q, int64_t rows, int64_t row_stride, int Hq, int Hkv, int D,
                      int gqa_map, int tokens);

template <int D, int KV, bool kSplit>
static cudaError_t launch_win_tc_t(const CUtensorMap& kv, const CUtensorMap& q, const WinArgs& a, int32_t units,
                                   int nsplit, cudaStream_t st) {
  using Cfg = WtCfg<D, KV>;
  cudaError_t e = cudaFuncSetAttribute(win_tc_kernel<D, KV, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  if (Cfg::kHeld) {
    // setmaxnreg.inc waits for registers that the block does not have if it
    // was launched with fewer.
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, win_tc_kernel<D, KV, kSplit>);
    if (e != cudaSuccess) return e;
    if (fa.numRegs < Cfg::kRegs) return cudaErrorLaunchOutOfResources;
  }
  ProfScope ps(kProfTc, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * nsplit));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = nsplit;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = nsplit > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, win_tc_kernel<D, KV, kSplit>, kv, q, a, nsplit);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
template <int D, bool kSplit>
static cudaError_t launch_win_tc_kv(const CUtensorMap& kv, const CUtensorMap& q, const WinArgs& a, int32_t units,
                                    int nsplit, cudaStream_t st) {
  switch (a.kv_dtype) {
    case DD_DTYPE_BF16: return launch_win_tc_t<D, DD_DTYPE_BF16, kSplit>(kv, q, a, units, nsplit, st);
    case DD_DTYPE_E4M3: return launch_win_tc_t<D, DD_DTYPE_E4M3, kSplit>(kv, q, a, units, nsplit, st);
    default: return launch_win_tc_t<D, DD_DTYPE_MXFP8, kSplit>(kv, q, a, units, nsplit, st);
  }
}

static int64_t win_tc_units(const WinArgs& a) {
  return ((int64_t)a.num_seqs + a.num_rows / (2 * (128 / a.g))) * a.Hkv;
}

// A group has to fit a sub-tile, and the kernel's 32-bit item arithmetic and
// TMA coordinates have to hold the batch and the pool.
bool win_tc_fits(const WinArgs& a) {
  const int64_t pool_rows = (int64_t)a.num_pages * 2 * a.Hkv * kPageSize;
  return a.D <= 128 && a.g <= 128 && pool_rows > 0 && pool_rows <= 0x7FFFFFFF &&
         win_tc_units(a) < (1ll << 31) - 1024;
}

// CTAs of a cluster that share an item's tiles: where the items leave most of
// the GPU idle, as long as a share is four tiles or more. Eight CTAs, which take
// an SM each, have to fit one group of SMs: such clusters fill some three
// quarters of the GPU. (16,000 tokens, window 0, 8 heads, bf16, 32 / 256 new
// ones: 45 / 94 us, against 76 / 557 of the streaming kernel.)
int win_tc_split(int64_t items, int64_t pages, int sms) {
  int n = 1;
  while (n < kWtSplit && items * n * 2 * (n == 4 ? 4 : 3) <= sms * 3 && pages >= 4 * kTcPagesPerTile * 2 * n) n *= 2;
  return n;
}

// DD_ERR_NOT_AVAILABLE: not launched, the registers do not hold it.
int launch_win_tc(const WinArgs& a, int nsplit, cudaStream_t st) {
  CUtensorMap kv, q;
  int rc = make_kv_tensor_map(&kv, a.kv, a.num_pages, a.Hkv, a.D, a.kv_dtype == DD_DTYPE_BF16 ? 2 : 1, 0);
  if (!rc) rc = make_q_tensor_map(&q, a.q, a.num_rows, a.q_stride, a.Hq, a.Hkv, a.D, a.gqa_map, 128 / a.g);
  if (rc) return rc;
  const int32_t units = (int32_t)win_tc_units(a);
  const auto launch = a.D == 64 ? (nsplit > 1 ? launch_win_tc_kv<64, true> : launch_win_tc_kv<64, false>)
                                : (nsplit > 1 ? launch_win_tc_kv<128, true> : launch_win_tc_kv<128, false>);
  const cudaError_t e = launch(kv, q, a, units, nsplit, st);
  if (e == cudaErrorLaunchOutOfResources) {
    cudaGetLastError();
    return DD_ERR_NOT_AVAILABLE;
  }
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("window attention launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

}  // namespace dd

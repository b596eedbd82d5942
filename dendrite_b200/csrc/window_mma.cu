// Sliding-window attention for few query rows per sequence (decode, guessed
// tokens): bf16 queries over bf16 / E4M3 / MXFP8 pages, head dims 64-256.
//
// Few rows read many tokens, so HBM bounds it: the kernel's work is to keep
// loads in flight and to spend few instructions on each byte.
//  - A warp takes one 16-token page at a time and waits for no other warp. bf16
//    pages go straight from global memory into the fragment registers of its
//    products, every 32-byte sector read whole by one instruction. FP8 pages
//    hold half as many bytes for as many instructions, so registers keep too
//    little in flight: they come through a ring in shared memory, three pages or
//    more for each warp (128 x 2048 tokens of E4M3: 89 us, 5.5 TB/s, against 103
//    through the registers).
//  - The products are transposed, S^T = K Q^T and O^T = V^T P^T (m16n8k16), so
//    the page's tokens (and V's head dims) are the 16-row side and the 8-column
//    side holds NT x 8 query rows: a GQA group of up to 8 wastes no second half.
//    The head dims of K are contracted in an order in which a lane's share of
//    a token is contiguous (Q is loaded in the same order); V's dims are dealt
//    to the product's rows the same way, two tokens' words being interleaved
//    with byte permutes.
//  - bf16: K of the next page is requested as soon as S is formed, V of the next
//    as soon as O is: half to all of a page is in flight for every warp.
//  - S^T and O^T have their query row in the same lane, so the softmax state
//    (reference, sum) and a rescale need no exchange; the reference moves only
//    when a score passes it by 8 (log2 units), found by one vote a page.
//  - FP8 codes are exact in f16, so the scores take f16 products on the codes
//    themselves: a row of Q is scaled by a power of two into f16's range, E4M3's
//    per-head scale is folded into the score scale, MXFP8's exponents of K scale
//    S per 32-dim block. E4M3's V is taken the same way, its scale in the
//    epilogue. MXFP8's V is widened to bf16, where a code times its power of two
//    is exact whatever the other tokens' exponents are.
//  - The warps of a CTA take pages in turn, the CTAs of a cluster (1 to 16)
//    split the visible pages; the states are joined through shared memory and
//    the cluster's shared memory, so a call is one launch without workspace.
// Weights are rounded to two bf16 terms for bf16 and MXFP8 pages (bf16's products
// take both operands in bf16; two terms keep 16 bits) and to f16 for E4M3 pages
// (11 bits, 2^-32 of the largest weight at worst, V of a head having one scale);
// sums and references are f32.
#include <algorithm>

#include "window.cuh"

namespace dd {

constexpr int kWinWarps = 4;
constexpr float kWinStep = 8.0f;     // how far a score may pass the reference (log2 units)
constexpr float kWinF16Shift = 7.0f; // f16 weights are held as 2^7 w: below 2^16, normal down to 2^-21

enum { kWinBf16 = 0, kWinE4m3 = 1, kWinMx = 2 };

__device__ __forceinline__ uint4 ldg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t movm_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool kF16>
__device__ __forceinline__ void win_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  if (kF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A page's K or V share of a lane, in the order of the products.
//  K: token g + 8 * half, dims 32 i + 8 c .. + 8 (i < D / 32)
//  V: bf16: token t(j), dims 64 i + 8 g .. + 8 (i < D / 64);
//     FP8:  token t(j), dims 32 i + 4 g .. + 4 (i < D / 32);   t = 2c, 2c+1, 2c+8, 2c+9
template <int D, int KV>
struct WinFrag;
template <int D>
struct WinFrag<D, kWinBf16> {
  uint4 k[D / 32][2];
  uint4 v[D / 64][4];
};
template <int D, int KV>
struct WinFrag {
  uint2 k[D / 32][2];
  uint32_t v[D / 32][4];
  // MXFP8: exponent bytes (D / 32 of them each) of K's tokens g, g + 8 and V's tokens t(j)
  uint32_t ek[2][(D + 127) / 128], ev[4][(D + 127) / 128];
};

// ---- bf16: straight from global memory.
template <int D>
__device__ __forceinline__ void load_k(WinFrag<D, kWinBf16>& f, const WinArgs& a, uint32_t page, int h, int g, int c) {
  const int64_t row = ((int64_t)page * 2 * a.Hkv + h) * kPageSize + g;
  const uint16_t* p = reinterpret_cast<const uint16_t*>(a.kv) + row * D + 8 * c;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) f.k[i][half] = ldg128(p + half * 8 * D + 32 * i);
}
template <int D>
__device__ __forceinline__ void load_v(WinFrag<D, kWinBf16>& f, const WinArgs& a, uint32_t page, int h, int g, int c) {
  const int64_t slice = (((int64_t)page * 2 + 1) * a.Hkv + h) * kPageSize;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = slice + 2 * c + (j & 1) + 8 * (j >> 1);
    const uint16_t* p = reinterpret_cast<const uint16_t*>(a.kv) + row * D + 8 * g;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) f.v[i][j] = ldg128(p + 64 * i);
  }
}
// ---- FP8: a warp's pages come through a ring in shared memory of its own.
// A slice (16 tokens of K or V of a head) lies there in units of 32 bytes, placed
// so that the words of eight dims of tokens t .. t + 3 (t = 0, 4; K) and of
// tokens t, t + 2, t + 4, t + 6 (V) fall into different banks.
template <int D>
__device__ __forceinline__ int ring_unit(int t, int b) {
  if (D == 64) return (t ^ ((t >> 2) & 1)) * 2 + (b ^ ((t >> 1) & 1));
  return t * (D / 32) + (b ^ ((t >> 1) & 3) ^ ((t & 1) << 1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Asks for a page: K, V, then MXFP8's exponents of both.
template <int D, int KV>
__device__ __forceinline__ void ring_load(uint32_t stage, const WinArgs& a, uint32_t page, int h, int lane) {
  const int64_t krow = ((int64_t)page * 2 * a.Hkv + h) * kPageSize, vrow = krow + (int64_t)a.Hkv * kPageSize;
  const uint8_t* kv = reinterpret_cast<const uint8_t*>(a.kv);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int q = lane + 32 * i, t = q / (D / 16), cc = q % (D / 16);
    const uint32_t dst = stage + ring_unit<D>(t, cc >> 1) * 32 + (cc & 1) * 16;
    cp_async16(dst, kv + krow * D + q * 16);
    cp_async16(dst + kPageSize * D, kv + vrow * D + q * 16);
  }
  if (KV == kWinMx && lane < 2 * (D / 32)) {
    const int q = lane % (D / 32);
    cp_async16(stage + 2 * kPageSize * D + lane * 16,
               reinterpret_cast<const uint8_t*>(a.scales) + (lane < D / 32 ? krow : vrow) * (D / 32) + q * 16);
  }
}
template <int D>
__device__ __forceinline__ void ring_exps(const uint8_t* p, uint32_t (&e)[(D + 127) / 128]) {
  if (D == 64) {
    e[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i) e[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}
template <int D, int KV>
__device__ __forceinline__ void ring_k(WinFrag<D, KV>& f, const uint8_t* stage, int g, int c) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      f.k[i][half] = *reinterpret_cast<const uint2*>(stage + ring_unit<D>(g + 8 * half, i) * 32 + 8 * c);
  if constexpr (KV == kWinMx) {
    const uint8_t* e = stage + 2 * kPageSize * D;
    ring_exps<D>(e + g * (D / 32), f.ek[0]);
    ring_exps<D>(e + (g + 8) * (D / 32), f.ek[1]);
  }
}
template <int D, int KV>
__device__ __forceinline__ void ring_v(WinFrag<D, KV>& f, const uint8_t* stage, int g, int c) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f.v[i][j] = *reinterpret_cast<const uint32_t*>(stage + kPageSize * D +
                                                     ring_unit<D>(2 * c + (j & 1) + 8 * (j >> 1), i) * 32 + 4 * g);
  if constexpr (KV == kWinMx) {
    const uint8_t* e = stage + 2 * kPageSize * D + kPageSize * (D / 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) ring_exps<D>(e + (2 * c + (j & 1) + 8 * (j >> 1)) * (D / 32), f.ev[j]);
  }
}
// Byte b of a word of E8M0 exponents as a power of two (0: 0 in place of
// 2^-127, which no sum of scores sees; 255: infinity).
__device__ __forceinline__ float exp_byte(uint32_t w, int b) {
  return __uint_as_float(__byte_perm(w, 0u, 0x0444u | (b << 12)) >> 1);
}
template <int N>
__device__ __forceinline__ bool has_nan_exp(const uint32_t (&e)[N]) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) any |= (~e[i] - 0x01010101u) & e[i] & 0x80808080u;  // a zero byte of ~e
  return any != 0;
}
// Byte b of two words of E8M0 exponents as a bf16 pair of powers of two (0: 2^-127; 255: infinity).
__device__ __forceinline__ uint32_t exp_pair(uint32_t w0, uint32_t w1, int b) {
  return __vmaxu2((__byte_perm(w0, w1, b | (b + 4) << 8) & 0xff00ffu) << 7, 0x00400040u);
}
// Four E4M3 codes (a word) as two bf16 pairs, exact, each pair times `by`.
__device__ __forceinline__ void e4m3x4_bf16_by(uint32_t codes, uint32_t by, uint32_t& lo, uint32_t& hi) {
  const float2 a = e4m3x2_to_float2((uint16_t)(codes & 0xffffu)), b = e4m3x2_to_float2((uint16_t)(codes >> 16));
  auto times = [&](float2 x) {
    const uint32_t w = pack_bf16x2(x.x, x.y);
    const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&by));
    return *reinterpret_cast<const uint32_t*>(&y);
  };
  lo = times(a);
  hi = times(b);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2& v, int i) { return i == 0 ? v.x : v.y; }

template <int D, int NT>
struct WinShared {
  float o[kWinWarps][NT * 8][D + 4];  // per warp: its output, normalised by its own sum
  float m[kWinWarps][NT * 8], l[kWinWarps][NT * 8];
  float cm[NT * 8], cl[NT * 8];       // the CTA's joined state (o[0] holds its output)
};

// CTAs that an SM holds, as far as the registers go. FP8 pages are half the
// bytes of bf16 ones and need the fourth (128 x 2048 tokens of E4M3: 89 us, in
// three 97).
template <int D, int KV, int NT>
constexpr int kWinCtas = D * NT >= 256 ? 2 : KV == kWinBf16 && D == 128 ? 3 : 4;

// FP8: bytes of a page in the ring, and the pages that a warp's share of the
// SM's shared memory holds.
template <int D, int KV, int NT>
struct WinRing {
  static constexpr bool kUsed = KV != kWinBf16;
  static constexpr int kPage = 2 * kPageSize * D + (KV == kWinMx ? 2 * kPageSize * (D / 32) : 0);
  static constexpr int kPages = kUsed ? (208 * 1024 / kWinCtas<D, KV, NT> / kWinWarps) / kPage : 0;
  static constexpr int kRing = kWinWarps * kPages * kPage, kState = sizeof(WinShared<D, NT>);
  static constexpr int kSmem = kRing > kState ? kRing : kState;
};

template <int D, int KV, int NT>
__global__ void __launch_bounds__(kWinWarps * 32, kWinCtas<D, KV, NT>) win_mma_kernel(WinArgs a, int nsplit) {
  constexpr int R = NT * 8;
  constexpr bool kF16 = KV != kWinBf16;    // Q, K
  constexpr bool kF16V = KV == kWinE4m3;  // weights, V
  constexpr int kBlocks = D / 32;
  using Ring = WinRing<D, KV, NT>;
  constexpr bool kRing = Ring::kUsed;
  extern __shared__ __align__(16) uint8_t win_smem[];
  WinShared<D, NT>& sh = *reinterpret_cast<WinShared<D, NT>*>(win_smem);  // once the ring is done
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % nsplit;
  const int64_t unit = blockIdx.x / nsplit;
  const int h = (int)(unit % a.Hkv);
  int32_t s, tile;
  win_tile(a, a.g, R, unit / a.Hkv, s, tile);
  const SeqRows sr = seq_rows(a.row_indptr, a.num_tokens, a.num_rows, s);
  const int64_t rows = (int64_t)sr.m * a.g, row0 = (int64_t)tile * R;
  const int nrows = (int)min((int64_t)R, rows - row0);
  if (tile < 0 || nrows <= 0) return;  // the whole cluster
  const int32_t p_lo = sr.pos0 + (int32_t)(row0 / a.g);
  const int32_t p_hi = sr.pos0 + (int32_t)((row0 + nrows - 1) / a.g);
  const WinPages wp = win_pages(a.window, a.sinks, p_lo, p_hi);
  // This CTA's pages [v0, v1) of the visible ones; its warps take them in turn.
  const int32_t v0 = (int32_t)((int64_t)rank * wp.count / nsplit), v1 = (int32_t)((int64_t)(rank + 1) * wp.count / nsplit);
  const int32_t t0 = a.page_indptr[s], table = a.page_indptr[s + 1] - t0;

  // Query row r of the tile -> its row of q and out.
  auto q_row = [&](int r, int64_t& token) {
    const int64_t rr = row0 + r;
    token = sr.r0 + rr / a.g;
    return qo_head_of(a.gqa_map, h, (int)(rr % a.g), a.Hkv, a.g);
  };
  // Page id of the lane's next page: one read for the warp's next 32.
  int32_t base_v = v0 + warp;
  auto read_ids = [&](int32_t v) {
    const int32_t vv = v + kWinWarps * lane;
    if (vv >= v1) return 0xFFFFFFFFu;
    const int32_t idx = wp.page(vv);
    const uint32_t id = idx < table ? (uint32_t)a.page_indices[t0 + idx] : 0xFFFFFFFFu;
    if (id < (uint32_t)a.num_pages) return id;
    win_report(a.status, kDevErrBadPage, idx < table ? id : (uint32_t)idx);
    return 0xFFFFFFFFu;
  };
  uint32_t ids = read_ids(base_v);
  int32_t at = 0;  // pages handed out of this read
  // Pages v0 + warp, + kWinWarps, ... one call after another; 0xFFFFFFFF for a bad one.
  auto take = [&](int32_t v) {
    if (v >= v1) return 0xFFFFFFFFu;
    if (at == 32) {
      base_v = v;
      ids = read_ids(base_v);
      at = 0;
    }
    return __shfl_sync(0xffffffffu, ids, at++);
  };
  WinFrag<D, KV> f;
  uint32_t now = 0xFFFFFFFFu;
  uint8_t* ring = win_smem + warp * Ring::kPages * Ring::kPage;
  int32_t ahead = v0 + warp;  // FP8: the next page to be asked for
  int ask = 0, slot = 0;      // the ring's places for it and for the current one
  uint32_t there = 0;         // places that hold a page
  auto ask_next = [&]() {
    const uint32_t id = take(ahead);
    ahead += kWinWarps;
    there &= ~(1u << ask);
    if (id != 0xFFFFFFFFu) {
      ring_load<D, KV>(smem_u32(ring) + ask * Ring::kPage, a, id, h, lane);
      there |= 1u << ask;
    }
    cp_async_commit();
    ask = ask + 1 == Ring::kPages ? 0 : ask + 1;
  };
  if constexpr (kRing) {
    for (int i = 0; i < Ring::kPages - 1; ++i) ask_next();
  } else {
    now = take(v0 + warp);
    if (now != 0xFFFFFFFFu) {
      load_k(f, a, now, h, g, c);
      load_v(f, a, now, h, g, c);
    }
  }

  // Q fragments: lane (g, c) holds row 8 n + g, dims 32 i + 8 c .. + 8.
  uint32_t q[NT][D / 32][4];
  float scale[NT][2];   // score scale of columns 2c, 2c + 1
  int32_t pos[NT][2];   // their positions
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    int64_t token = 0;
    const int hq = r < nrows ? q_row(r, token) : 0;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) +
                                                      token * a.q_stride + (int64_t)hq * D + 8 * c);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 x = r < nrows ? src[4 * i] : make_uint4(0, 0, 0, 0);
      q[n][i][0] = x.x, q[n][i][1] = x.y, q[n][i][2] = x.z, q[n][i][3] = x.w;
    }
    float row_scale = a.scale_log2;
    if (kF16) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max(top, max(q[n][i][w] & 0x7fffu, (q[n][i][w] >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = f16_row_shift(top);
      const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          q[n][i][w] = bf16x2_to_f16x2(q[n][i][w], by);
      row_scale = f16_score_scale(row_scale, up);
      if (KV == kWinE4m3) row_scale *= reinterpret_cast<const float*>(a.scales)[h];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      scale[n][e] = kF16 ? __shfl_sync(0xffffffffu, row_scale, (2 * c + e) * 4) : row_scale;
      pos[n][e] = sr.pos0 + (int32_t)((row0 + 8 * n + 2 * c + e) / a.g);
    }
  }

  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
  }

  // Page v of the list, pool page `now`; the loads of the next one go out as
  // f's registers come free.
  for (int32_t v = v0 + warp; v < v1; v += kWinWarps) {
    const uint8_t* stage = ring + slot * Ring::kPage;
    uint32_t next = 0xFFFFFFFFu;
    if constexpr (kRing) {
      const bool bad = !((there >> slot) & 1);
      __syncwarp();  // every lane is through with the place that is asked for next
      ask_next();
      cp_async_wait<Ring::kPages - 1>();
      __syncwarp();  // every lane's part of this page has come
      slot = slot + 1 == Ring::kPages ? 0 : slot + 1;
      if (bad) continue;
      ring_k<D, KV>(f, stage, g, c);
    } else {
      next = take(v + kWinWarps);
      if (now == 0xFFFFFFFFu) {  // a bad page: skipped
        now = next;
        if (now != 0xFFFFFFFFu) {
          load_k(f, a, now, h, g, c);
          load_v(f, a, now, h, g, c);
        }
        continue;
      }
    }
    // ---- S^T = K Q^T
    float x[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if constexpr (KV == kWinBf16) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            win_mma<false>(x[n], word(f.k[i][0], 2 * u), word(f.k[i][1], 2 * u), word(f.k[i][0], 2 * u + 1),
                           word(f.k[i][1], 2 * u + 1), q[n][i][2 * u], q[n][i][2 * u + 1]);
      } else {
        float y[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[n][e] = KV == kWinMx ? 0.f : x[n][e];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_f16(word(f.k[i][0], u), a0, a2);
          e4m3x4_f16(word(f.k[i][1], u), a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) win_mma<true>(y[n], a0, a1, a2, a3, q[n][i][2 * u], q[n][i][2 * u + 1]);
        }
        if constexpr (KV == kWinMx) {
          const float e0 = exp_byte(f.ek[0][i / 4], i % 4), e1 = exp_byte(f.ek[1][i / 4], i % 4);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            x[n][0] = fmaf(y[n][0], e0, x[n][0]);
            x[n][1] = fmaf(y[n][1], e0, x[n][1]);
            x[n][2] = fmaf(y[n][2], e1, x[n][2]);
            x[n][3] = fmaf(y[n][3], e1, x[n][3]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = y[n][e];
        }
      }
    }
    if constexpr (KV == kWinMx) {
      // exp_byte takes the NaN exponent for infinity.
      const bool n0 = has_nan_exp(f.ek[0]), n1 = has_nan_exp(f.ek[1]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < 2 ? n0 : n1) x[n][e] = NAN;
    }
    if constexpr (kRing) {
      ring_v<D, KV>(f, stage, g, c);
    } else {
      now = next;
      if (now != 0xFFFFFFFFu) load_k(f, a, now, h, g, c);
    }
    // ---- mask. Most pages are seen whole by every row.
    const int32_t j0 = wp.page(v) * kPageSize;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] *= scale[n][e & 1];
    const bool whole = j0 + kPageSize - 1 <= p_lo &&
                       (a.window == 0 || j0 > p_hi - a.window || j0 + kPageSize <= a.sinks);
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!win_sees(a.window, a.sinks, pos[n][e & 1], j0 + g + 8 * (e >> 1))) x[n][e] = -INFINITY;
      // Slots that no row of the tile sees may hold anything: their V (and
      // exponents) become zero, as zero times NaN is not.
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t t = j0 + 2 * c + (j & 1) + 8 * (j >> 1);
        const bool seen = t <= p_hi && (a.window == 0 || t > p_lo - a.window || t < a.sinks);
        if (!seen) {
          if constexpr (KV == kWinBf16) {
#pragma unroll
            for (int i = 0; i < D / 64; ++i) f.v[i][j] = make_uint4(0, 0, 0, 0);
          } else {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) f.v[i][j] = 0;
            if constexpr (KV == kWinMx) {
#pragma unroll
              for (int i = 0; i < (D + 127) / 128; ++i) f.ev[j][i] = 0;
            }
          }
        }
      }
    }
    if constexpr (KV == kWinMx) {
      // exp_pair takes the NaN exponent for infinity: NaN codes make it NaN.
      bool some = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) some |= has_nan_exp(f.ev[j]);
      if (__any_sync(0xffffffffu, some)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < kBlocks; ++i)
            if (((f.ev[j][i / 4] >> (8 * (i % 4))) & 255) == 255) f.v[i][j] = 0x7f7f7f7f;
      }
    }
    // ---- references: moved for all rows once some score passes its own by
    // more than kWinStep (the first page always).
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) over |= fmaxf(x[n][e], x[n][e + 2]) > m[n][e] + kWinStep;
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = fmaxf(x[n][e], x[n][e + 2]);
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, b));
          t = fmaxf(t, m[n][e]);
          const float by = m[n][e] == t ? 1.f : exp2f(m[n][e] - t);
          m[n][e] = t;
          l[n][e] *= by;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[n][i][e] *= by;
            o[n][i][e + 2] *= by;
          }
        }
    }
    // ---- weights
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ref = (m[n][e] == -INFINITY ? 0.f : m[n][e]) - (kF16V ? kWinF16Shift : 0.f);
        x[n][e] = fast_exp2(x[n][e] - ref);
        x[n][e + 2] = fast_exp2(x[n][e + 2] - ref);
        l[n][e] += x[n][e] + x[n][e + 2];
      }
    }
    // ---- O^T += V^T P^T
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if constexpr (kF16V) {
          hi[n][half] = movm_trans(pack_f16x2(x[n][2 * half], x[n][2 * half + 1]));
        } else {
          uint32_t a_hi, a_lo;
          split_bf16x2(x[n][2 * half], x[n][2 * half + 1], a_hi, a_lo);
          hi[n][half] = movm_trans(a_hi);
          lo[n][half] = movm_trans(a_lo);
        }
      }
    auto product = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        win_mma<kF16V>(o[n][i], a0, a1, a2, a3, hi[n][0], hi[n][1]);
        if constexpr (!kF16V) win_mma<false>(o[n][i], a0, a1, a2, a3, lo[n][0], lo[n][1]);
      }
    };
    if constexpr (KV == kWinBf16) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t w0 = word(f.v[i][0], u), w1 = word(f.v[i][1], u), w2 = word(f.v[i][2], u), w3 = word(f.v[i][3], u);
          product(4 * i + u, __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410),
                  __byte_perm(w2, w3, 0x7632));
        }
    } else {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint32_t l0 = __byte_perm(f.v[i][0], f.v[i][1], 0x5140), h0 = __byte_perm(f.v[i][0], f.v[i][1], 0x7362);
        const uint32_t l1 = __byte_perm(f.v[i][2], f.v[i][3], 0x5140), h1 = __byte_perm(f.v[i][2], f.v[i][3], 0x7362);
        uint32_t by0 = 0, by1 = 0;
        if constexpr (KV == kWinMx) {
          by0 = exp_pair(f.ev[0][i / 4], f.ev[1][i / 4], i % 4);
          by1 = exp_pair(f.ev[2][i / 4], f.ev[3][i / 4], i % 4);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a0, a1, a2, a3;
          if constexpr (KV == kWinMx) {
            e4m3x4_bf16_by(u ? h0 : l0, by0, a0, a1);
            e4m3x4_bf16_by(u ? h1 : l1, by1, a2, a3);
          } else {
            e4m3x4_f16(u ? h0 : l0, a0, a1);
            e4m3x4_f16(u ? h1 : l1, a2, a3);
          }
          product(2 * i + u, a0, a1, a2, a3);
        }
      }
    }
    if constexpr (!kRing) {
      if (now != 0xFFFFFFFFu) load_v(f, a, now, h, g, c);
    }
  }
  if constexpr (kRing) __syncthreads();  // the state takes the ring's place

  // ---- the warp's state, normalised by its own sum
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float t = l[n][e];
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) t += __shfl_xor_sync(0xffffffffu, t, b);
      const int r = 8 * n + 2 * c + e;
      const float v_scale = KV == kWinE4m3 ? reinterpret_cast<const float*>(a.scales)[a.Hkv + h] : 1.f;
      const float inv = t == 0.f ? 0.f : v_scale * (1.f / t);
      if (g == 0) {
        sh.m[warp][r] = m[n][e] - (kF16V ? kWinF16Shift : 0.f);
        sh.l[warp][r] = t;
      }
      if constexpr (KV == kWinBf16) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          float4* dst = reinterpret_cast<float4*>(&sh.o[warp][r][64 * i + 8 * g]);
          dst[0] = make_float4(o[n][4 * i][e] * inv, o[n][4 * i][e + 2] * inv, o[n][4 * i + 1][e] * inv, o[n][4 * i + 1][e + 2] * inv);
          dst[1] = make_float4(o[n][4 * i + 2][e] * inv, o[n][4 * i + 2][e + 2] * inv, o[n][4 * i + 3][e] * inv, o[n][4 * i + 3][e + 2] * inv);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
          *reinterpret_cast<float4*>(&sh.o[warp][r][32 * i + 4 * g]) =
              make_float4(o[n][2 * i][e] * inv, o[n][2 * i][e + 2] * inv, o[n][2 * i + 1][e] * inv, o[n][2 * i + 1][e + 2] * inv);
      }
    }
  __syncthreads();

  // ---- join the warps (into o[0]), then the CTAs of the cluster
  constexpr int kVec = D / 4;
  auto weights = [](float mm, float ll, float top) { return ll * exp2f(mm - (top == -INFINITY ? 0.f : top)); };
  for (int idx = threadIdx.x; idx < nrows * kVec; idx += kWinWarps * 32) {
    const int r = idx / kVec, d = idx % kVec * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) top = fmaxf(top, sh.m[w][r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) {
      const float wt = weights(sh.m[w][r], sh.l[w][r], top);
      const float4 y = *reinterpret_cast<const float4*>(&sh.o[w][r][d]);
      sum += wt;
      acc.x = fmaf(wt, y.x, acc.x), acc.y = fmaf(wt, y.y, acc.y);
      acc.z = fmaf(wt, y.z, acc.z), acc.w = fmaf(wt, y.w, acc.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<float4*>(&sh.o[0][r][d]) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (d == 0) {
      sh.cm[r] = top;
      sh.cl[r] = sum;
    }
  }
  if (nsplit > 1)
    cluster_barrier();
  else
    __syncthreads();
  for (int idx = threadIdx.x + rank * kWinWarps * 32; idx < nrows * kVec; idx += nsplit * kWinWarps * 32) {
    const int r = idx / kVec, d = idx % kVec * 4;
    float top, sum;
    float4 acc;
    if (nsplit == 1) {
      acc = *reinterpret_cast<const float4*>(&sh.o[0][r][d]);
      top = sh.cm[r];
      sum = sh.cl[r];
    } else {
      const uint32_t am = smem_u32(&sh.cm[r]), al = smem_u32(&sh.cl[r]), ao = smem_u32(&sh.o[0][r][d]);
      top = -INFINITY;
      sum = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < nsplit; ++k) top = fmaxf(top, cluster_ld(am, k));
      for (int k = 0; k < nsplit; ++k) {
        const float wt = weights(cluster_ld(am, k), cluster_ld(al, k), top);
        const float4 y = cluster_ld4(ao, k);
        sum += wt;
        acc.x = fmaf(wt, y.x, acc.x), acc.y = fmaf(wt, y.y, acc.y);
        acc.z = fmaf(wt, y.z, acc.z), acc.w = fmaf(wt, y.w, acc.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
    int64_t token;
    const int hq = q_row(r, token);
    const int64_t dst = token * a.Hq + hq;
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + dst * D + d) =
        make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
    if (d == 0 && a.lse) a.lse[dst] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
  if (nsplit > 1) cluster_barrier();  // no CTA leaves while another reads its state
}

// ------------------------------------------------------------------ host side
// CTAs of a cluster. A CTA costs some 6 us of dependent loads and joining
// besides its pages, so no more than one wave of them is launched, down to a
// page for each warp; but where the units (tile, KV head) alone are a little
// more than whole waves and have pages enough, they are split to even the last
// one out. (4096-token windows, bf16: 64 sequences of 8 heads, 512 units for
// 444 places: 220 us whole, 187 in two, 177 in four; 4 sequences: 67 us whole,
// 17 in eight.) Sixteen CTAs have to fit one group of SMs, so such clusters
// fill some 0.6 of the places in one wave, and joining them costs a microsecond
// that few pages do not repay (a decode step of 1 / 2 / 3 sequences of 8 heads,
// bf16, 8192-token windows, eight and sixteen: 17.9, 14.8; 21.8, 20.3; 25.6,
// 35.4 us; 1024-token windows 8.2, 8.7; 8.8, 10.1; 9.1, 17.4).
static int win_split(int64_t units, int64_t places, int64_t pages) {
  int n = 1;
  while (n < 8 && units * n * 2 <= places && pages >= 2 * n * kWinWarps) n *= 2;
  if (n == 8 && units * 16 * 5 <= places * 3 && pages >= 128) n = 16;
  auto last_wave_idle = [&]() {
    const int64_t waves = (units * n + places - 1) / places;
    return units * n * 100 < waves * places * 85;
  };
  if (units > places)
    while (n < 8 && last_wave_idle() && pages >= 128 * n) n *= 2;
  return n;
}

template <int D, int KV, int NT>
static int launch_win_mma_t(const WinArgs& a, int max_pages, int sms, cudaStream_t st) {
  constexpr int R = 8 * NT;
  const int64_t tiles = a.row_indptr ? a.num_seqs + (int64_t)a.num_rows * a.g / R
                                     : (int64_t)a.num_seqs * ((a.g + R - 1) / R);
  const int64_t full = a.row_indptr ? win_tiles_expected(a, R) : tiles;  // tiles that have rows
  int64_t pages = max_pages > 0 ? max_pages : INT64_MAX;
  if (a.window > 0) pages = std::min(pages, ((int64_t)a.window + a.sinks) / kPageSize + 2);
  const int nsplit = win_split(full * a.Hkv, (int64_t)sms * kWinCtas<D, KV, NT>, pages);
  const int64_t blocks = tiles * a.Hkv * nsplit;
  if (blocks > 0x7FFFFFFF) return fail(DD_ERR_INVALID_ARGUMENT, "too many rows");
  using Ring = WinRing<D, KV, NT>;
  cudaError_t e = cudaSuccess;
  if (Ring::kSmem > 48 * 1024)
    e = cudaFuncSetAttribute(win_mma_kernel<D, KV, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring::kSmem);
  if (e == cudaSuccess && nsplit > 8)
    e = cudaFuncSetAttribute(win_mma_kernel<D, KV, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kWinWarps * 32);
    cfg.dynamicSmemBytes = Ring::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = nsplit;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = nsplit > 1 ? 1 : 0;
    ProfScope ps(kProfMma, st);
    e = cudaLaunchKernelEx(&cfg, win_mma_kernel<D, KV, NT>, a, nsplit);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("window attention launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

template <int D, int KV>
static int launch_win_mma_nt(const WinArgs& a, int max_pages, int sms, cudaStream_t st) {
  // Rows of an average sequence: one column block of 8 where they fit it, or
  // where two of head_dim 256 would not fit the registers.
  const int64_t rows = ((int64_t)a.num_rows * a.g + a.num_seqs - 1) / a.num_seqs;
  if constexpr (D < 256)
    if (rows > 8) return launch_win_mma_t<D, KV, 2>(a, max_pages, sms, st);
  return launch_win_mma_t<D, KV, 1>(a, max_pages, sms, st);
}
template <int D>
static int launch_win_mma_kv(const WinArgs& a, int max_pages, int sms, cudaStream_t st) {
  switch (a.kv_dtype) {
    case DD_DTYPE_BF16: return launch_win_mma_nt<D, kWinBf16>(a, max_pages, sms, st);
    case DD_DTYPE_E4M3: return launch_win_mma_nt<D, kWinE4m3>(a, max_pages, sms, st);
    default: return launch_win_mma_nt<D, kWinMx>(a, max_pages, sms, st);
  }
}

// max_pages: pages of the longest table, 0 if not known.
int launch_win_mma(const WinArgs& a, int max_pages, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  switch (a.D) {
    case 64: return launch_win_mma_kv<64>(a, max_pages, sms, st);
    case 128: return launch_win_mma_kv<128>(a, max_pages, sms, st);
    default: return launch_win_mma_kv<256>(a, max_pages, sms, st);
  }
}

}  // namespace dd

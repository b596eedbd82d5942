// Shared pieces of the sliding-window attention kernels (window.cu,
// window_mma.cu, window_tc.cu): arguments, the rows of a ragged batch and the
// pages that a range of query positions sees.
#pragma once
#include "dd_device.cuh"

namespace dd {

struct WinArgs {
  const void* q;       // [rows][Hq][D], q_stride elements from row to row
  int64_t q_stride;
  const void* kv;
  const void* scales;
  void* out;           // [rows][Hq][D] in q_dtype
  float* lse;          // [rows][Hq], natural log, or NULL
  uint32_t* status;    // 2 words, or NULL
  const int32_t* row_indptr;   // NULL: one row per sequence
  const int32_t* page_indptr;
  const int32_t* page_indices;
  const int32_t* num_tokens;
  int32_t num_seqs, num_rows;
  int32_t window, sinks;
  int32_t Hq, Hkv, g, D, kv_dtype, q_dtype, gqa_map, num_pages;
  float scale_log2;
};

// status: the first error's code and detail.
__device__ __forceinline__ void win_report(uint32_t* status, uint32_t code, uint32_t aux) {
  if (status && atomicCAS(status, 0u, code) == 0u) status[1] = aux;
}

// Rows [r0, r0 + m) of the batch belong to sequence s, whose row i has
// position pos0 + i (negative: a row without a token, which sees nothing).
// Row ranges are cut to the num_rows that the buffers hold.
struct SeqRows {
  int32_t r0, m, pos0, n;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* row_indptr, const int32_t* num_tokens,
                                            int32_t num_rows, int32_t s) {
  SeqRows q;
  q.n = max(num_tokens[s], 0);
  int32_t a = s, b = s + 1;
  if (row_indptr) {
    a = row_indptr[s];
    b = row_indptr[s + 1];
  }
  q.pos0 = q.n - (b - a);
  q.r0 = min(max(a, 0), num_rows);
  q.m = max(min(b, num_rows) - q.r0, 0);
  return q;
}

// The sequence that owns a row: the last s with row_indptr[s] <= row (empty
// sequences before it share its start), or -1 for a row behind the last one.
__device__ __forceinline__ int32_t seq_of_row(const int32_t* row_indptr, int32_t num_seqs,
                                              int32_t row) {
  if (!row_indptr) return row < num_seqs ? row : -1;
  if (num_seqs <= 0 || row < row_indptr[0] || row >= row_indptr[num_seqs]) return -1;
  int32_t lo = 0, hi = num_seqs;  // row_indptr[lo] <= row < row_indptr[hi]
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (row_indptr[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The pages that hold a token visible to some position of [p_lo, p_hi], in
// order: `ns` pages of first tokens, then the windows' pages from page `wp`.
// Page v of the list is table entry page(v).
struct WinPages {
  int32_t ns, wp, count;
  __device__ __forceinline__ int32_t page(int32_t v) const { return v < ns ? v : wp + v - ns; }
};
__device__ __forceinline__ WinPages win_pages(int32_t window, int32_t sinks, int32_t p_lo,
                                              int32_t p_hi) {
  WinPages w;
  if (p_hi < 0) {
    w.ns = w.wp = w.count = 0;
    return w;
  }
  const int32_t first = window > 0 ? max(0, max(p_lo, 0) - window + 1) : 0;
  w.wp = first / kPageSize;
  w.ns = min((int32_t)(((int64_t)min(sinks, first) + kPageSize - 1) / kPageSize), w.wp);
  w.count = w.ns + p_hi / kPageSize - w.wp + 1;
  return w;
}

// Whether position p sees token j (p >= 0 or nothing).
__device__ __forceinline__ bool win_sees(int32_t window, int32_t sinks, int32_t p, int32_t j) {
  return j <= p && (window == 0 || j > p - window || j < sinks);
}

// Four E4M3 codes (a word) as two f16x2, exact: bytes 0-1 -> lo, 2-3 -> hi.
__device__ __forceinline__ void e4m3x4_f16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A bf16 query row as f16: the row times 2^up, its largest element (bf16 bits
// `top`, sign off) just below 2^15. bf16's 8 bits then are exact down to 2^-29
// of that element; what is smaller is off by at most 2^-39 of it.
__device__ __forceinline__ int f16_row_shift(uint32_t top) {
  return max(-126, min(127, 14 - ((int)(top >> 7) - 127)));
}
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w, float by) {
  return pack_f16x2(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xffff0000u) * by);
}
// scale * 2^-up, in two exact steps (2^-up alone may be below f32's normal range).
__device__ __forceinline__ float f16_score_scale(float scale, int up) {
  return scale * __uint_as_float((uint32_t)(127 - up / 2) << 23) * __uint_as_float((uint32_t)(127 - (up - up / 2)) << 23);
}

// Tile t of the batch: sequence and tile within it, a tile being R of the
// sequence's m * g rows. Sequence s owns the tiles from s + floor(start(s) * g
// / R): at least the ceil(m * g / R) that it needs, so no prefix sum over the
// sequences is wanted; surplus tiles have no rows, and those before the first
// sequence's row come out as tile -1.
__device__ __forceinline__ void win_tile(const WinArgs& a, int g, int R, int64_t t, int32_t& s, int32_t& tile) {
  if (!a.row_indptr) {
    const int per = (g + R - 1) / R;
    s = (int32_t)(t / per);
    tile = (int32_t)(t % per);
    return;
  }
  int32_t lo = 0, hi = a.num_seqs;
  auto base = [&](int32_t i) { return i + (int64_t)min(max(a.row_indptr[i], 0), a.num_rows) * g / R; };
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (base(mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  s = lo;
  tile = (int32_t)max(t - base(lo), (int64_t)-1);
}

// Tiles of R rows that a chunk call's sequences fill, as far as the host knows:
// all of one length where that divides, else each with half a tile over.
inline int64_t win_tiles_expected(const WinArgs& a, int R) {
  const int64_t seqs = a.num_seqs, rows = (int64_t)a.num_rows * a.g;
  if (a.num_rows % a.num_seqs == 0) return seqs * ((rows / seqs + R - 1) / R);
  return seqs > rows / R + seqs / 2 ? seqs : rows / R + seqs / 2;
}

// Another CTA's shared memory: reads at the place that `addr` is in this one's.
__device__ __forceinline__ float cluster_ld(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_ld4(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}

// Kernel launches (each returns a dd_status).
int launch_win_simple(const WinArgs& a, cudaStream_t st);
int launch_win_mma(const WinArgs& a, int max_pages, cudaStream_t st);
bool win_tc_fits(const WinArgs& a);
int win_tc_split(int64_t items, int64_t pages, int sms);
int launch_win_tc(const WinArgs& a, int nsplit, cudaStream_t st);

}  // namespace dd

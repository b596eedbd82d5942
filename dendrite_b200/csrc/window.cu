// Sliding-window attention over the paged cache: C entry points, the choice of
// kernel, and the CUDA-core kernel.
//
// With x_j = scale * q.k_j over the tokens j that a query of position p sees
// (the last `window` up to p, and the first `sinks`), out = sum_j w_j v_j with
// w_j = exp(x_j - lse), lse = log sum_j exp(x_j). The kernels walk the visible
// pages once with a running maximum and sum (kept in f32, log2 domain); the
// page table is read on the device, and no entry outside the visible pages.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "window.cuh"

namespace dd {

// ------------------------------------------------------- CUDA-core kernel
// f32 queries or f32 pages. One warp per (row, query head): its lanes share
// the head dims, a page's 16 scores are reduced across the warp, and the
// running maximum moves once per page. Bound by its shuffles and exponentials,
// not by memory: it is the parity path.
template <int E>  // elements per lane
__device__ __forceinline__ void win_load(const WinArgs& a, int which, int h, uint32_t page, int t,
                                         int lane, float (&x)[E]) {
  constexpr int D = E * 32;
  const int64_t row = (((int64_t)page * 2 + which) * a.Hkv + h) * kPageSize + t;
  const int d = lane * E;
  if (a.kv_dtype == DD_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = reinterpret_cast<const float*>(a.kv)[row * D + d + e];
  } else if (a.kv_dtype == DD_DTYPE_BF16) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      x[e] = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(a.kv)[row * D + d + e]);
  } else {
    const float s = a.kv_dtype == DD_DTYPE_E4M3
                        ? reinterpret_cast<const float*>(a.scales)[which * a.Hkv + h]
                        : e8m0_to_float(reinterpret_cast<const uint8_t*>(a.scales)[row * (D / 32) + d / 32]);
#pragma unroll
    for (int e = 0; e < E; ++e)
      x[e] = e4m3_to_float(reinterpret_cast<const uint8_t*>(a.kv)[row * D + d + e]) * s;
  }
}

template <int E>
__global__ void __launch_bounds__(128) win_simple_kernel(WinArgs a) {
  constexpr int D = E * 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.num_rows * a.Hq) return;
  const int32_t row = (int32_t)(w / a.Hq);
  const int hq = (int)(w % a.Hq);
  const int h = a.gqa_map == DD_GQA_TILED ? hq % a.Hkv : hq / a.g;
  const int32_t s = seq_of_row(a.row_indptr, a.num_seqs, row);
  if (s < 0) return;
  const SeqRows sr = seq_rows(a.row_indptr, a.num_tokens, a.num_rows, s);
  const int32_t p = sr.pos0 + row - sr.r0;
  const int64_t qoff = (int64_t)row * a.q_stride + (int64_t)hq * D + lane * E;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = a.q_dtype == DD_DTYPE_F32 ? reinterpret_cast<const float*>(a.q)[qoff + e]
                                     : bf16_bits_to_float(reinterpret_cast<const uint16_t*>(a.q)[qoff + e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const WinPages wp = win_pages(a.window, a.sinks, p, p);
  const int32_t t0 = a.page_indptr[s], table = a.page_indptr[s + 1] - t0;
  for (int v = 0; v < wp.count; ++v) {
    const int32_t idx = wp.page(v);
    const uint32_t page = idx < table ? (uint32_t)a.page_indices[t0 + idx] : 0xFFFFFFFFu;
    if (page >= (uint32_t)a.num_pages) {
      if (lane == 0) win_report(a.status, kDevErrBadPage, idx < table ? page : (uint32_t)idx);
      continue;
    }
    float x[kPageSize];
    float mx = m;
#pragma unroll
    for (int t = 0; t < kPageSize; ++t) {
      float k[E], acc = 0.f;
      win_load<E>(a, 0, h, page, t, lane, k);
#pragma unroll
      for (int e = 0; e < E; ++e) acc = fmaf(q[e], k[e], acc);
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, i);
      x[t] = win_sees(a.window, a.sinks, p, idx * kPageSize + t) ? acc * a.scale_log2 : -INFINITY;
      mx = fmaxf(mx, x[t]);
    }
    // Nothing but -inf so far: any finite reference gives weights of zero (and
    // a NaN score stays NaN; fmaxf passes it over).
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float f = exp2f(m - ref);
    l *= f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
    for (int t = 0; t < kPageSize; ++t) {
      if (!win_sees(a.window, a.sinks, p, idx * kPageSize + t)) continue;  // its V is not looked at
      const float wgt = exp2f(x[t] - ref);
      float val[E];
      win_load<E>(a, 1, h, page, t, lane, val);
      l += wgt;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(wgt, val[e], o[e]);
    }
    m = mx;
  }
  // l is NaN where a visible score is: the row is NaN then, not zero.
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t ooff = ((int64_t)row * a.Hq + hq) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (a.q_dtype == DD_DTYPE_F32)
      reinterpret_cast<float*>(a.out)[ooff + e] = o[e] * inv;
    else
      reinterpret_cast<__nv_bfloat16*>(a.out)[ooff + e] = __float2bfloat16_rn(o[e] * inv);
  }
  if (lane == 0 && a.lse) a.lse[(int64_t)row * a.Hq + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

int launch_win_simple(const WinArgs& a, cudaStream_t st) {
  const int64_t warps = (int64_t)a.num_rows * a.Hq;
  const int64_t blocks = (warps + 3) / 4;
  if (blocks > 0x7FFFFFFF) return fail(DD_ERR_INVALID_ARGUMENT, "too many rows");
  {
    ProfScope ps(kProfSimple, st);
    switch (a.D) {
      case 64: win_simple_kernel<2><<<(unsigned)blocks, 128, 0, st>>>(a); break;
      case 128: win_simple_kernel<4><<<(unsigned)blocks, 128, 0, st>>>(a); break;
      default: win_simple_kernel<8><<<(unsigned)blocks, 128, 0, st>>>(a); break;
    }
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("window attention launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

// Chunks: which of the two tensor-core kernels, and in how many CTAs the tcgen05
// one splits an item. Both walk the visible pages of every KV head, the streaming
// kernel once for 16 rows (or a sequence's fewer), at a time for the whole GPU
// that goes by the page's bytes and their unpacking, the tcgen05 kernel once for up
// to 256, 8 pages after 8 on one SM a CTA, items in waves, with more to set up and
// shares to join. The constants are fitted to 1152 measured pairs (1 to 64
// sequences x 2 to 256 new tokens, windows of 16 to 4096 and none over 8000 tokens,
// 1, 4 and 8 heads a group, head dims 64 and 128): the choice is more than 1.2 times
// the better one in 2 of them, and in 4 of 400 ragged batches drawn from the same
// ranges. Around the border (streaming, tcgen05; us), head dim 128: bf16, 4 heads a
// group, window 1024, 16 sequences x 8 new tokens 28.1, 29.4; x 16 54.8, 29.3; 64 x 4
// 65.3, 93.0; x 8 113.9, 92.8; window 16, 64 x 4 19.5, 23.4; x 8 32.4, 23.6; no
// window, 1 x 8 26.7, 29.2; x 32 43.7, 30.9; E4M3, 8 heads, window 4096, 16 x 4 59.7,
// 68.7; x 8 114.2, 68.5; MXFP8, 4 heads, window 1024, 16 x 8 30.6, 32.3; x 16 56.9,
// 32.3; head dim 64: bf16 16 x 8 20.0, 25.4; x 16 29.8, 25.4; E4M3 16 x 4 42.9, 59.4;
// x 8 72.9, 59.7.
static bool tc_is_faster(const WinArgs& a, int max_pages, int& nsplit) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t tokens = a.num_rows / a.num_seqs;
  int64_t pages = max_pages > 0 ? max_pages : 256;
  if (a.window > 0) pages = std::min(pages, ((int64_t)a.window + a.sinks + tokens) / kPageSize + 2);
  const int64_t tiles16 = win_tiles_expected(a, 16) * a.Hkv;
  const int64_t items = win_tiles_expected(a, 2 * (128 / a.g) * a.g) * a.Hkv;
  nsplit = win_tc_split(items, pages, sms);
  const int64_t tiles = ((pages + 7) / 8 + nsplit - 1) / nsplit;  // of a CTA
  // A page's time in hundredths of a nanosecond.
  const int64_t page = a.kv_dtype == DD_DTYPE_BF16 ? (a.D == 64 ? 55 : 110) : a.kv_dtype == DD_DTYPE_E4M3 ? (a.D == 64 ? 45 : 80)
                                                                                                       : (a.D == 64 ? 75 : 100);
  const int64_t stream_ns = 5200 + tiles16 * (1500 + pages * page) / 100;
  const int64_t join_ns = nsplit == 1 ? 0 : tokens * a.g > 128 ? 10000 : 4000;
  const int64_t tc_ns = 7500 + (items * nsplit + sms - 1) / sms * (2300 + tiles * 1700) + join_ns;
  return tc_ns < stream_ns;
}

static int window_attention(const dd_attn_config* cfg, int32_t num_seqs, int32_t num_rows,
                            int32_t max_pages, int32_t window, int32_t sinks, const void* q,
                            int64_t q_stride, const void* kv, const void* scales,
                            const int32_t* q_indptr, const int32_t* page_indptr,
                            const int32_t* page_indices, const int32_t* num_tokens, void* out,
                            float* lse, uint32_t* status, cudaStream_t st) {
  if (window < 0 || sinks < 0) return fail(DD_ERR_INVALID_ARGUMENT, "window and sinks must be >= 0");
  if (max_pages < 0) return fail(DD_ERR_INVALID_ARGUMENT, "max_pages_per_seq must be >= 0");
  if (num_seqs == 0 || num_rows == 0) return DD_OK;
  if (!q || !out) return fail(DD_ERR_INVALID_ARGUMENT, "q / out is NULL");
  if (!page_indptr || !num_tokens)  // page_indices may be NULL when every table is empty
    return fail(DD_ERR_INVALID_ARGUMENT, "page table pointer is NULL");
  if (!kv && cfg->num_pages > 0) return fail(DD_ERR_INVALID_ARGUMENT, "kv_pages is NULL");
  const bool fp8 = cfg->kv_dtype == DD_DTYPE_E4M3 || cfg->kv_dtype == DD_DTYPE_MXFP8;
  if (fp8 && !scales) return fail(DD_ERR_INVALID_ARGUMENT, "FP8 KV pages need kv_scales");
  if (((uintptr_t)kv | (uintptr_t)q | (uintptr_t)out) & 15)
    return fail(DD_ERR_INVALID_ARGUMENT, "kv_pages, q and out must be 16-byte aligned");
  const int elem = cfg->q_dtype == DD_DTYPE_F32 ? 4 : 2;
  if (q_stride < (int64_t)cfg->num_qo_heads * cfg->head_dim || (q_stride * elem) % 16)
    return fail(DD_ERR_INVALID_ARGUMENT,
                "q_stride must cover a row's heads and be a multiple of 16 bytes");
  if (cfg->kv_dtype == DD_DTYPE_MXFP8 && ((uintptr_t)scales & 15))
    return fail(DD_ERR_INVALID_ARGUMENT, "MXFP8 kv_scales must be 16-byte aligned");
  WinArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = q;
  a.q_stride = q_stride;
  a.kv = kv;
  a.scales = scales;
  a.out = out;
  a.lse = lse;
  a.status = status;
  a.row_indptr = q_indptr;
  a.page_indptr = page_indptr;
  a.page_indices = page_indices;
  a.num_tokens = num_tokens;
  a.num_seqs = num_seqs;
  a.num_rows = num_rows;
  a.window = std::min(window, 1 << 30);  // no sequence is longer; keeps differences in 32 bits
  a.sinks = window > 0 ? sinks : 0;
  a.Hq = cfg->num_qo_heads;
  a.Hkv = cfg->num_kv_heads;
  a.g = cfg->num_qo_heads / cfg->num_kv_heads;
  a.D = cfg->head_dim;
  a.kv_dtype = cfg->kv_dtype;
  a.q_dtype = cfg->q_dtype;
  a.gqa_map = cfg->gqa_map;
  a.num_pages = cfg->num_pages;
  const float scale = cfg->scale > 0.f ? cfg->scale : 1.0f / std::sqrt((float)cfg->head_dim);
  a.scale_log2 = scale * kLog2e;
  if (cfg->q_dtype == DD_DTYPE_F32 || cfg->kv_dtype == DD_DTYPE_F32) return launch_win_simple(a, st);
  int nsplit = 1;
  if (q_indptr && win_tc_fits(a) && tc_is_faster(a, max_pages, nsplit)) {
    const int rc = launch_win_tc(a, nsplit, st);
    if (rc != DD_ERR_NOT_AVAILABLE) return rc;
  }
  return launch_win_mma(a, max_pages, st);
}

}  // namespace dd

using namespace dd;

extern "C" int dd_decode_paged_window(const dd_attn_config* cfg, int32_t batch_size,
                                      int32_t max_pages_per_seq, int32_t window, int32_t sinks,
                                      const void* q, int64_t q_stride, const void* kv_pages,
                                      const void* kv_scales, const int32_t* page_indptr,
                                      const int32_t* page_indices, const int32_t* num_tokens,
                                      void* out, float* lse, uint32_t* status, dd_stream_t stream) {
  const int rc = check_config(cfg);
  if (rc) return rc;
  if (batch_size < 0) return fail(DD_ERR_INVALID_ARGUMENT, "batch_size must be >= 0");
  return window_attention(cfg, batch_size, batch_size, max_pages_per_seq, window, sinks, q, q_stride,
                          kv_pages, kv_scales, nullptr, page_indptr, page_indices, num_tokens, out,
                          lse, status, (cudaStream_t)stream);
}

extern "C" int dd_prefill_paged_window(const dd_attn_config* cfg, int32_t num_seqs, int32_t num_rows,
                                       int32_t max_pages_per_seq, int32_t window, int32_t sinks,
                                       const void* q, int64_t q_stride, const void* kv_pages,
                                       const void* kv_scales, const int32_t* q_indptr,
                                       const int32_t* page_indptr, const int32_t* page_indices,
                                       const int32_t* num_tokens, void* out, float* lse,
                                       uint32_t* status, dd_stream_t stream) {
  const int rc = check_config(cfg);
  if (rc) return rc;
  if (num_seqs < 0 || num_rows < 0) return fail(DD_ERR_INVALID_ARGUMENT, "num_seqs and num_rows must be >= 0");
  if (num_seqs > 0 && num_rows > 0 && !q_indptr) return fail(DD_ERR_INVALID_ARGUMENT, "q_indptr is NULL");
  return window_attention(cfg, num_seqs, num_rows, max_pages_per_seq, window, sinks, q, q_stride,
                          kv_pages, kv_scales, q_indptr, page_indptr, page_indices, num_tokens, out,
                          lse, status, (cudaStream_t)stream);
}

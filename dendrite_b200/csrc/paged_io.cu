// Ragged writes and reads of the paged cache through device page tables: the
// append of a batch's new tokens, quantised as they are written, and the
// read-back of token ranges, dequantised. Both move every element once; what
// bounds them is HBM.
#include "window.cuh"

namespace dd {

struct PagedIo {
  void* kv;
  void* scales;
  const int32_t* row_indptr;
  const int32_t* page_indptr;
  const int32_t* page_indices;
  const int32_t* tokens;   // append: tokens per sequence; gather: first token (NULL: 0)
  uint32_t* status;
  int32_t num_seqs, num_rows, Hkv, num_pages, pool_dtype, ext_dtype;
  const void* k;           // append: sources; gather: destinations
  const void* v;
  int64_t k_stride, v_stride;
};

// Page and slot of the token that a row stands for; false (and the status
// words) where there is no such page. `live` is false for a row behind the
// last sequence.
template <bool kAppend>
__device__ __forceinline__ bool io_place(const PagedIo& a, int32_t row, bool report, uint32_t& page,
                                         int32_t& slot, bool& live) {
  const int32_t s = seq_of_row(a.row_indptr, a.num_seqs, row);
  live = s >= 0;
  if (!live) return false;
  int32_t pos;
  if (kAppend) {
    const int32_t end = a.row_indptr ? a.row_indptr[s + 1] : s + 1;
    pos = a.tokens[s] - (end - row);
  } else {
    pos = (a.tokens ? a.tokens[s] : 0) + row - a.row_indptr[s];
  }
  const int32_t t0 = a.page_indptr[s], table = a.page_indptr[s + 1] - t0;
  page = 0xFFFFFFFFu;
  if (pos >= 0 && pos / kPageSize < table) page = (uint32_t)a.page_indices[t0 + pos / kPageSize];
  slot = pos & (kPageSize - 1);
  if (page < (uint32_t)a.num_pages) return true;
  if (report) win_report(a.status, kDevErrBadPage, (uint32_t)row);
  return false;
}

// One warp per (row, K/V, head); lane owns E = D/32 consecutive elements.
template <int D>
__global__ void __launch_bounds__(256) append_paged_kernel(PagedIo a) {
  constexpr int E = D / 32;
  const int64_t w = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)a.num_rows * 2 * a.Hkv) return;
  const int32_t row = (int32_t)(w / (2 * a.Hkv));
  const int rest = (int)(w % (2 * a.Hkv));
  const int which = rest / a.Hkv, h = rest % a.Hkv;
  uint32_t page;
  int32_t slot;
  bool live;
  if (!io_place<true>(a, row, rest == 0 && lane == 0, page, slot, live)) return;
  const int64_t src = (int64_t)row * (which ? a.v_stride : a.k_stride) + (int64_t)h * D + lane * E;
  const void* from = which ? a.v : a.k;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    x[e] = a.ext_dtype == DD_DTYPE_F32 ? reinterpret_cast<const float*>(from)[src + e]
                                       : bf16_bits_to_float(reinterpret_cast<const uint16_t*>(from)[src + e]);
  const int64_t r = (((int64_t)page * 2 + which) * a.Hkv + h) * kPageSize + slot;
  const int64_t dst = r * D + lane * E;
  if (a.pool_dtype == DD_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<float*>(a.kv)[dst + e] = x[e];
  } else if (a.pool_dtype == DD_DTYPE_BF16) {
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<__nv_bfloat16*>(a.kv)[dst + e] = __float2bfloat16_rn(x[e]);
  } else if (a.pool_dtype == DD_DTYPE_E4M3) {
    const float sc = reinterpret_cast<const float*>(a.scales)[which * a.Hkv + h];
#pragma unroll
    for (int e = 0; e < E; ++e)
      reinterpret_cast<uint8_t*>(a.kv)[dst + e] = float_to_e4m3_satrn(__fdiv_rn(x[e], sc));
  } else {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, fabsf(x[e]));
#pragma unroll
    for (int o = 1; o < 32 / E; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int ex = m > 0.f ? max(floor_log2_pos(m) - 8, -127) : -127;
    const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);  // 2^-ex, a normal f32
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<uint8_t*>(a.kv)[dst + e] = float_to_e4m3_satrn(x[e] * inv);
    if ((lane * E) % 32 == 0)
      reinterpret_cast<uint8_t*>(a.scales)[r * (D / 32) + lane * E / 32] = (uint8_t)(ex + 127);
  }
}

template <int D>
__global__ void __launch_bounds__(256) gather_paged_kernel(PagedIo a) {
  constexpr int E = D / 32;
  const int64_t w = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)a.num_rows * 2 * a.Hkv) return;
  const int32_t row = (int32_t)(w / (2 * a.Hkv));
  const int rest = (int)(w % (2 * a.Hkv));
  const int which = rest / a.Hkv, h = rest % a.Hkv;
  uint32_t page;
  int32_t slot;
  bool live;
  const bool ok = io_place<false>(a, row, rest == 0 && lane == 0, page, slot, live);
  if (!live) return;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
  if (ok) {
    const int64_t r = (((int64_t)page * 2 + which) * a.Hkv + h) * kPageSize + slot;
    const int64_t src = r * D + lane * E;
    if (a.pool_dtype == DD_DTYPE_F32) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = reinterpret_cast<const float*>(a.kv)[src + e];
    } else if (a.pool_dtype == DD_DTYPE_BF16) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(a.kv)[src + e]);
    } else {
      const float s = a.pool_dtype == DD_DTYPE_E4M3
                          ? reinterpret_cast<const float*>(a.scales)[which * a.Hkv + h]
                          : e8m0_to_float(reinterpret_cast<const uint8_t*>(a.scales)[r * (D / 32) + lane * E / 32]);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = e4m3_to_float(reinterpret_cast<const uint8_t*>(a.kv)[src + e]) * s;
    }
  }
  void* to = const_cast<void*>(which ? a.v : a.k);
  const int64_t dst = ((int64_t)row * a.Hkv + h) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (a.ext_dtype == DD_DTYPE_F32)
      reinterpret_cast<float*>(to)[dst + e] = x[e];
    else
      reinterpret_cast<__nv_bfloat16*>(to)[dst + e] = __float2bfloat16_rn(x[e]);
  }
}

static int io_check(const dd_attn_config* cfg, const void* kv, const void* scales, int32_t num_rows,
                    const int32_t* page_indptr, const void* k, const void* v, int32_t ext_dtype) {
  if (!kv || !page_indptr || !k || !v) return fail(DD_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (ext_dtype != DD_DTYPE_F32 && ext_dtype != DD_DTYPE_BF16)
    return fail(DD_ERR_INVALID_ARGUMENT, "K/V outside the pool must be f32 or bf16");
  const bool fp8 = cfg->kv_dtype == DD_DTYPE_E4M3 || cfg->kv_dtype == DD_DTYPE_MXFP8;
  if (fp8 && !scales) return fail(DD_ERR_INVALID_ARGUMENT, "FP8 pages need kv_scales");
  if (((uintptr_t)kv | (uintptr_t)k | (uintptr_t)v) & 15)
    return fail(DD_ERR_INVALID_ARGUMENT, "kv_pages, k and v must be 16-byte aligned");
  if (fp8 && ((uintptr_t)scales & (cfg->kv_dtype == DD_DTYPE_MXFP8 ? 15 : 3)))
    return fail(DD_ERR_INVALID_ARGUMENT, "kv_scales not aligned");
  if ((int64_t)num_rows * 2 * cfg->num_kv_heads / 8 >= 0x7FFFFFFF)
    return fail(DD_ERR_INVALID_ARGUMENT, "too many rows");
  return DD_OK;
}

}  // namespace dd

using namespace dd;

extern "C" int dd_append_kv_paged(const dd_attn_config* cfg, void* kv_pages, void* kv_scales,
                                  int32_t num_seqs, int32_t num_rows, const int32_t* new_indptr,
                                  const int32_t* page_indptr, const int32_t* page_indices,
                                  const int32_t* num_tokens, const void* k, int64_t k_stride,
                                  const void* v, int64_t v_stride, int32_t src_dtype,
                                  uint32_t* status, dd_stream_t stream) {
  int rc = check_config(cfg);
  if (rc) return rc;
  if (num_seqs < 0 || num_rows < 0) return fail(DD_ERR_INVALID_ARGUMENT, "num_seqs and num_rows must be >= 0");
  if (num_seqs == 0 || num_rows == 0) return DD_OK;
  if (!new_indptr && num_rows != num_seqs)
    return fail(DD_ERR_INVALID_ARGUMENT, "without new_indptr there is one row per sequence");
  if (!num_tokens) return fail(DD_ERR_INVALID_ARGUMENT, "num_tokens is NULL");
  rc = io_check(cfg, kv_pages, kv_scales, num_rows, page_indptr, k, v, src_dtype);
  if (rc) return rc;
  const int64_t width = (int64_t)cfg->num_kv_heads * cfg->head_dim;
  const int elem = src_dtype == DD_DTYPE_F32 ? 4 : 2;
  if (k_stride < width || v_stride < width || (k_stride * elem) % 16 || (v_stride * elem) % 16)
    return fail(DD_ERR_INVALID_ARGUMENT,
                "k_stride and v_stride must cover a row's heads and be multiples of 16 bytes");
  const PagedIo a{kv_pages, kv_scales, new_indptr, page_indptr, page_indices, num_tokens, status,
                  num_seqs, num_rows, cfg->num_kv_heads, cfg->num_pages, cfg->kv_dtype, src_dtype,
                  k, v, k_stride, v_stride};
  const unsigned blocks = (unsigned)(((int64_t)num_rows * 2 * cfg->num_kv_heads + 7) / 8);
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps(kProfOther, st);
    switch (cfg->head_dim) {
      case 64: append_paged_kernel<64><<<blocks, 256, 0, st>>>(a); break;
      case 128: append_paged_kernel<128><<<blocks, 256, 0, st>>>(a); break;
      default: append_paged_kernel<256><<<blocks, 256, 0, st>>>(a); break;
    }
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("append_kv_paged launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

extern "C" int dd_gather_kv_paged(const dd_attn_config* cfg, const void* kv_pages,
                                  const void* kv_scales, int32_t num_seqs, int32_t num_rows,
                                  const int32_t* out_indptr, const int32_t* first_token,
                                  const int32_t* page_indptr, const int32_t* page_indices,
                                  void* k_out, void* v_out, int32_t out_dtype, uint32_t* status,
                                  dd_stream_t stream) {
  int rc = check_config(cfg);
  if (rc) return rc;
  if (num_seqs < 0 || num_rows < 0) return fail(DD_ERR_INVALID_ARGUMENT, "num_seqs and num_rows must be >= 0");
  if (num_seqs == 0 || num_rows == 0) return DD_OK;
  if (!out_indptr) return fail(DD_ERR_INVALID_ARGUMENT, "out_indptr is NULL");
  rc = io_check(cfg, kv_pages, kv_scales, num_rows, page_indptr, k_out, v_out, out_dtype);
  if (rc) return rc;
  const PagedIo a{const_cast<void*>(kv_pages), const_cast<void*>(kv_scales), out_indptr, page_indptr,
                  page_indices, first_token, status, num_seqs, num_rows, cfg->num_kv_heads,
                  cfg->num_pages, cfg->kv_dtype, out_dtype, k_out, v_out, 0, 0};
  const unsigned blocks = (unsigned)(((int64_t)num_rows * 2 * cfg->num_kv_heads + 7) / 8);
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps(kProfOther, st);
    switch (cfg->head_dim) {
      case 64: gather_paged_kernel<64><<<blocks, 256, 0, st>>>(a); break;
      case 128: gather_paged_kernel<128><<<blocks, 256, 0, st>>>(a); break;
      default: gather_paged_kernel<256><<<blocks, 256, 0, st>>>(a); break;
    }
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DD_ERR_CUDA, std::string("gather_kv_paged launch: ") + cudaGetErrorString(e));
  return DD_OK;
}

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
  int32_t log2_d;
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

// A row's K and V heads are one run of 2 * Hkv * D elements, cut into 16-byte
// chunks of the pool's type (kN elements). A warp takes 32 chunks of a row, a
// chunk a lane, or 128 in four rounds: the row's place in the page table is a
// chain of dependent reads, which a small call pays as few times as it can in
// turn (16 tokens: 2.7 us against 3.9) and a large one as few times as it can at
// all (95,000 MXFP8 tokens read back: 122 us against 97, 6.1 TB/s; 33,000
// tokens stored as E4M3 68 against 51, 4.0 TB/s, bound by its divisions' issue
// slots beside HBM). Four chunks of a lane in flight cost registers, so warps,
// and lost (119, 78). Pool-side accesses are
// whole 128-byte runs of one head.
template <int POOL>
struct IoPool {
  static constexpr int kN = POOL == DD_DTYPE_F32 ? 4 : POOL == DD_DTYPE_BF16 ? 8 : 16;
};
constexpr int kIoWarps = 4;

// kN consecutive elements as f32, from / to 16-byte aligned (8 bytes for the
// four bf16 of an f32 chunk) memory.
template <int EXT, int N>
__device__ __forceinline__ void io_load(const void* base, int64_t at, float (&x)[N]) {
  if constexpr (EXT == DD_DTYPE_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = p[i];
      x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
  } else {
    const uint2* p = reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(base) + at);
    uint32_t w[N / 2];
    if constexpr (N == 4) {
      const uint2 v = *p;
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int EXT, int N>
__device__ __forceinline__ void io_store(void* base, int64_t at, const float (&x)[N]) {
  if constexpr (EXT == DD_DTYPE_F32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    uint2* p = reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + at);
    if constexpr (N == 4) {
      *p = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 8; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
}

// Chunk c of a row: K or V, head, element; pool row of that (page, K/V, head, slot).
template <int N>
struct IoChunk {
  int which, h, d;
  int64_t ext, row;
  __device__ __forceinline__ IoChunk(const PagedIo& a, int c, int half, uint32_t page, int32_t slot) {
    which = c >= half;
    const int e = (which ? c - half : c) * N;
    h = e >> a.log2_d;
    d = e & ((1 << a.log2_d) - 1);
    ext = e;
    row = (((int64_t)page * 2 + which) * a.Hkv + h) * kPageSize + slot;
  }
};

// Warp's row and its chunks [c0, c1), 32 times kRounds of them at most.
template <int N, int kRounds>
__device__ __forceinline__ bool io_share(const PagedIo& a, int32_t& row, int& c0, int& c1) {
  const int64_t w = (int64_t)blockIdx.x * kIoWarps + (threadIdx.x >> 5);
  const int all = 2 * (a.Hkv << a.log2_d) / N, parts = (all + 32 * kRounds - 1) / (32 * kRounds);
  const int64_t r = parts == 1 ? w : w / parts;
  if (r >= a.num_rows) return false;
  row = (int32_t)r;
  c0 = (int)(w - r * parts) * 32 * kRounds;
  c1 = min(all, c0 + 32 * kRounds);
  return true;
}

template <int POOL, int EXT, int kRounds>
__global__ void __launch_bounds__(kIoWarps * 32) append_paged_kernel(PagedIo a) {
  constexpr int N = IoPool<POOL>::kN;
  const int lane = threadIdx.x & 31;
  int32_t row;
  int c0, c1;
  if (!io_share<N, kRounds>(a, row, c0, c1)) return;
  uint32_t page;
  int32_t slot;
  bool live;
  if (!io_place<true>(a, row, c0 == 0 && lane == 0, page, slot, live)) return;
  const int half = (a.Hkv << a.log2_d) / N;
#pragma unroll
  for (int u = 0; u < kRounds; ++u, c0 += 32) {
    if (c0 >= c1) break;
    const bool in = c0 + lane < c1;  // lanes past the end keep the warp's exchange whole
    const IoChunk<N> k(a, in ? c0 + lane : 0, half, page, slot);
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    if (in) io_load<EXT, N>(k.which ? a.v : a.k, (int64_t)row * (k.which ? a.v_stride : a.k_stride) + k.ext, x);
    const int64_t dst = (k.row << a.log2_d) + k.d;
    if constexpr (POOL == DD_DTYPE_F32 || POOL == DD_DTYPE_BF16) {
      if (in) io_store<POOL, N>(a.kv, dst, x);
    } else {
      if constexpr (POOL == DD_DTYPE_E4M3) {
        const float sc = reinterpret_cast<const float*>(a.scales)[k.which * a.Hkv + k.h];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __fdiv_rn(x[i], sc);
      } else {
        // 32 elements are two neighbouring lanes' chunks.
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const int ex = m > 0.f ? max(floor_log2_pos(m) - 8, -127) : -127;
        const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);  // 2^-ex, a normal f32
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= inv;
        if (in && !(lane & 1))
          reinterpret_cast<uint8_t*>(a.scales)[(k.row << (a.log2_d - 5)) + (k.d >> 5)] = (uint8_t)(ex + 127);
      }
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = e4m3x4_satrn(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      if (in) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.kv) + dst) = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
}

template <int POOL, int EXT, int kRounds>
__global__ void __launch_bounds__(kIoWarps * 32) gather_paged_kernel(PagedIo a) {
  constexpr int N = IoPool<POOL>::kN;
  const int lane = threadIdx.x & 31;
  int32_t row;
  int c0, c1;
  if (!io_share<N, kRounds>(a, row, c0, c1)) return;
  uint32_t page;
  int32_t slot;
  bool live;
  const bool ok = io_place<false>(a, row, c0 == 0 && lane == 0, page, slot, live);
  if (!live) return;
  const int half = (a.Hkv << a.log2_d) / N;
  const int64_t width = (int64_t)a.Hkv << a.log2_d;
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int c = c0 + lane + 32 * u;
    if (c >= c1) break;
    const IoChunk<N> k(a, c, half, ok ? page : 0, slot);
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    if (ok) {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.kv) +
                                                      ((k.row << a.log2_d) + k.d) * (16 / N));
      const uint32_t q[4] = {v.x, v.y, v.z, v.w};
      if constexpr (POOL == DD_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __uint_as_float(q[i]);
      } else if constexpr (POOL == DD_DTYPE_BF16) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          x[2 * i] = __uint_as_float(q[i] << 16);
          x[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
        }
      } else {
        const float sc = POOL == DD_DTYPE_E4M3
                             ? reinterpret_cast<const float*>(a.scales)[k.which * a.Hkv + k.h]
                             : e8m0_to_float(reinterpret_cast<const uint8_t*>(
                                   a.scales)[(k.row << (a.log2_d - 5)) + (k.d >> 5)]);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 y = e4m3x2_to_float2((uint16_t)(i & 1 ? q[i / 2] >> 16 : q[i / 2] & 0xffffu));
          x[2 * i] = y.x * sc;
          x[2 * i + 1] = y.y * sc;
        }
      }
    }
    io_store<EXT, N>(const_cast<void*>(k.which ? a.v : a.k), (int64_t)row * width + k.ext, x);
  }
}

template <int POOL, int EXT, int kRounds>
static void launch_io_t(bool append, const PagedIo& a, cudaStream_t st) {
  const int64_t all = 2 * ((int64_t)a.Hkv << a.log2_d) / IoPool<POOL>::kN;
  const int64_t parts = (all + 32 * kRounds - 1) / (32 * kRounds);
  const unsigned blocks = (unsigned)((a.num_rows * parts + kIoWarps - 1) / kIoWarps);
  ProfScope ps(kProfOther, st);
  if (append)
    append_paged_kernel<POOL, EXT, kRounds><<<blocks, kIoWarps * 32, 0, st>>>(a);
  else
    gather_paged_kernel<POOL, EXT, kRounds><<<blocks, kIoWarps * 32, 0, st>>>(a);
}
template <int POOL>
static void launch_io(bool append, const PagedIo& a, int sms, cudaStream_t st) {
  const int64_t all = 2 * ((int64_t)a.Hkv << a.log2_d) / IoPool<POOL>::kN;
  // One round a warp as long as these warps fit the GPU at once.
  const bool one = a.num_rows * ((all + 31) / 32) <= (int64_t)sms * 32;
  const bool f32 = a.ext_dtype == DD_DTYPE_F32;
  if (one)
    f32 ? launch_io_t<POOL, DD_DTYPE_F32, 1>(append, a, st) : launch_io_t<POOL, DD_DTYPE_BF16, 1>(append, a, st);
  else
    f32 ? launch_io_t<POOL, DD_DTYPE_F32, 4>(append, a, st) : launch_io_t<POOL, DD_DTYPE_BF16, 4>(append, a, st);
}
static int run_io(bool append, const PagedIo& a, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if ((int64_t)a.num_rows * a.Hkv >= (1ll << 31)) return fail(DD_ERR_INVALID_ARGUMENT, "too many rows");
  switch (a.pool_dtype) {
    case DD_DTYPE_F32: launch_io<DD_DTYPE_F32>(append, a, sms, st); break;
    case DD_DTYPE_BF16: launch_io<DD_DTYPE_BF16>(append, a, sms, st); break;
    case DD_DTYPE_E4M3: launch_io<DD_DTYPE_E4M3>(append, a, sms, st); break;
    default: launch_io<DD_DTYPE_MXFP8>(append, a, sms, st); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(DD_ERR_CUDA, std::string(append ? "append_kv_paged" : "gather_kv_paged") + " launch: " + cudaGetErrorString(e));
  return DD_OK;
}

static int log2_dim(int d) { return d == 64 ? 6 : d == 128 ? 7 : 8; }

static int io_check(const dd_attn_config* cfg, const void* kv, const void* scales, const int32_t* page_indptr,
                     const void* k, const void* v, int32_t ext_dtype) {
  if (!kv || !page_indptr || !k || !v) return fail(DD_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (ext_dtype != DD_DTYPE_F32 && ext_dtype != DD_DTYPE_BF16)
    return fail(DD_ERR_INVALID_ARGUMENT, "K/V outside the pool must be f32 or bf16");
  const bool fp8 = cfg->kv_dtype == DD_DTYPE_E4M3 || cfg->kv_dtype == DD_DTYPE_MXFP8;
  if (fp8 && !scales) return fail(DD_ERR_INVALID_ARGUMENT, "FP8 pages need kv_scales");
  if (((uintptr_t)kv | (uintptr_t)k | (uintptr_t)v) & 15)
    return fail(DD_ERR_INVALID_ARGUMENT, "kv_pages, k and v must be 16-byte aligned");
  if (fp8 && ((uintptr_t)scales & (cfg->kv_dtype == DD_DTYPE_MXFP8 ? 15 : 3)))
    return fail(DD_ERR_INVALID_ARGUMENT, "kv_scales not aligned");
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
  rc = io_check(cfg, kv_pages, kv_scales, page_indptr, k, v, src_dtype);
  if (rc) return rc;
  const int64_t width = (int64_t)cfg->num_kv_heads * cfg->head_dim;
  const int elem = src_dtype == DD_DTYPE_F32 ? 4 : 2;
  if (k_stride < width || v_stride < width || (k_stride * elem) % 16 || (v_stride * elem) % 16)
    return fail(DD_ERR_INVALID_ARGUMENT,
                "k_stride and v_stride must cover a row's heads and be multiples of 16 bytes");
  const PagedIo a{kv_pages, kv_scales, new_indptr, page_indptr, page_indices, num_tokens, status,
                  num_seqs, num_rows, cfg->num_kv_heads, cfg->num_pages, cfg->kv_dtype, src_dtype,
                  k, v, k_stride, v_stride, log2_dim(cfg->head_dim)};
  return run_io(true, a, (cudaStream_t)stream);
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
  rc = io_check(cfg, kv_pages, kv_scales, page_indptr, k_out, v_out, out_dtype);
  if (rc) return rc;
  const PagedIo a{const_cast<void*>(kv_pages), const_cast<void*>(kv_scales), out_indptr, page_indptr,
                  page_indices, first_token, status, num_seqs, num_rows, cfg->num_kv_heads,
                  cfg->num_pages, cfg->kv_dtype, out_dtype, k_out, v_out, 0, 0, log2_dim(cfg->head_dim)};
  return run_io(false, a, (cudaStream_t)stream);
}

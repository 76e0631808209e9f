// vqb_prefix_attention: attention of a batch over the paged cache.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j - m) in one pass over
// the keys: m is a running maximum, and what has been summed is scaled by
// exp(m_old - m_new) when it moves.
//
// A warp takes one (query, head) row and 32 keys at a time: a lane computes the
// score of one key, then the lanes share the value's dimensions.
#include "vqb_common.cuh"
#include "vqb_internal.h"

namespace vqb {
namespace {

struct AttnParams {
  vqb_attention_desc d;
  const uint16_t* q;
  const uint16_t* kc;
  const uint16_t* vc;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  const int32_t* prefix_pages;
  uint16_t* out;
  float* lse;
  int group;
  int page_shift;
  float scale_log2;  // scale * log2(e): scores in powers of two
};

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t h) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(__ushort_as_half(h));
}
template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

// The request whose queries include token n: the last r with cu_q[r] <= n (n < cu_q[R]).
__device__ __forceinline__ int request_of(const int32_t* cu_q, int R, int n) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(cu_q + mid) <= n) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(256) attention_rows_kernel(AttnParams p) {
  __shared__ float s_q[8][D];
  pdl_wait();
  pdl_trigger();
  const vqb_attention_desc& d = p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  const int n = static_cast<int>(row / d.heads), h = static_cast<int>(row - static_cast<int64_t>(n) * d.heads);
  if (n >= d.n_tokens || n >= __ldg(p.cu_q + d.n_requests)) return;
  const int r = request_of(p.cu_q, d.n_requests, n);
  const int q0 = __ldg(p.cu_q + r), nq = __ldg(p.cu_q + r + 1) - q0;
  int len = max(min(__ldg(p.kv_lens + r), d.max_kv_len), 0);
  len = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(d.table_width) << p.page_shift));
  const int seen = d.causal ? max(min(len - nq + (n - q0) + 1, len), 0) : len;
  const int kvh = h / p.group;
  const uint16_t* q = p.q + n * d.q_token_stride + h * d.q_head_stride;
  for (int e = lane; e < D; e += 32) s_q[warp][e] = widen<BF16>(q[e]);
  __syncwarp();

  float m = -INFINITY, l = 0.0f, acc[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
  for (int part = 0; part < 2; ++part) {
    const int32_t* pages = part == 0 ? p.prefix_pages : p.table + static_cast<int64_t>(r) * d.table_width;
    const int count = part == 0 ? d.prefix_len : seen;
    for (int j0 = 0; j0 < count; j0 += 32) {
      const int j = j0 + lane;
      int page = -1;
      float s = -INFINITY;
      if (j < count) {
        page = __ldg(pages + (j >> p.page_shift));
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(d.num_pages)) page = -1;
        s = 0.0f;
        if (page >= 0) {
          const uint16_t* k = p.kc + page * d.kc_page_stride + kvh * d.kc_head_stride +
                              (j & (d.page_size - 1)) * d.kc_token_stride;
          for (int e = 0; e < D; e += 8) {
            const uint4 w = *reinterpret_cast<const uint4*>(k + e);
            const uint16_t* x = reinterpret_cast<const uint16_t*>(&w);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(s_q[warp][e + i], widen<BF16>(x[i]), s);
          }
        }
        s *= p.scale_log2;
      }
      float top = s;
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m, top);
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float keep = exp2f(m - base);
      m = mn;
      const float w = j < count ? exp2f(s - base) : 0.0f;
      float sum = w;
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = l * keep + sum;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] *= keep;
      const int here = min(32, count - j0);
      for (int i = 0; i < here; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const int pg = __shfl_sync(0xffffffffu, page, i);
        if (pg < 0) continue;
        const uint16_t* v = p.vc + pg * d.vc_page_stride + kvh * d.vc_head_stride +
                            ((j0 + i) & (d.page_size - 1)) * d.vc_token_stride;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wi, widen<BF16>(v[lane + 32 * e]), acc[e]);
      }
    }
  }
  uint16_t* o = p.out + n * d.out_token_stride + h * d.out_head_stride;
  const bool empty = m == -INFINITY;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[lane + 32 * e] = narrow<BF16>(empty ? 0.0f : acc[e] / l);
  if (p.lse && lane == 0)
    p.lse[static_cast<int64_t>(n) * d.heads + h] = empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Everything about a call that does not need its pointers.
vqb_status check_desc(const vqb_attention_desc& d) {
  if (d.n_requests < 0 || d.n_tokens < 0 || d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads || d.max_q_len < 0 ||
      d.max_kv_len < 0 || d.prefix_len < 0 || d.num_pages < 0 || d.table_width < 0)
    return VQB_BAD_SHAPE;
  if (!(d.scale > 0.0f) || d.scale > 3.0e38f) return VQB_BAD_SHAPE;
  if (d.head_dim != 64 && d.head_dim != 128) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.page_size < 16 || d.page_size > 1024 || (d.page_size & (d.page_size - 1))) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.heads > 65535 || d.n_requests > 65535) return VQB_UNSUPPORTED_GEOMETRY;
  if (static_cast<int64_t>(d.table_width) * d.page_size < d.max_kv_len) return VQB_BAD_SHAPE;
  const int64_t strides[] = {d.q_token_stride, d.q_head_stride, d.out_token_stride, d.out_head_stride,
                             d.kc_page_stride, d.kc_head_stride, d.kc_token_stride,
                             d.vc_page_stride, d.vc_head_stride, d.vc_token_stride};
  for (int64_t s : strides) {
    if (s % 8) return VQB_BAD_ALIGNMENT;
    if (s < 0) return VQB_BAD_SHAPE;
  }
  return VQB_OK;
}

}  // namespace
}  // namespace vqb

using namespace vqb;

extern "C" size_t vqb_prefix_attention_workspace_size(const vqb_attention_desc* desc) {
  if (!desc || check_desc(*desc) != VQB_OK) return 0;
  return 256;
}

extern "C" vqb_status vqb_prefix_attention(const vqb_attention_desc* desc, vqb_dtype dtype, const void* q,
                                           const void* k_cache, const void* v_cache, const int32_t* block_table,
                                           const int32_t* kv_lens, const int32_t* cu_q, const int32_t* prefix_pages,
                                           void* out, float* lse, void* workspace, size_t workspace_bytes,
                                           vqb_stream_t stream) {
  if (!desc) return VQB_NULL_POINTER;
  const vqb_attention_desc& d = *desc;
  const vqb_status st = check_desc(d);
  if (st != VQB_OK) return st;
  if (dtype != VQB_F16 && dtype != VQB_BF16) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.n_tokens == 0 || d.n_requests == 0) return VQB_OK;
  if (!q || !k_cache || !v_cache || !kv_lens || !cu_q || !out || !workspace) return VQB_NULL_POINTER;
  if ((d.max_kv_len > 0 && !block_table) || (d.prefix_len > 0 && !prefix_pages)) return VQB_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return VQB_BAD_ALIGNMENT;
  if (workspace_bytes < vqb_prefix_attention_workspace_size(desc)) return VQB_WORKSPACE_TOO_SMALL;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  AttnParams p{d, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache),
               static_cast<const uint16_t*>(v_cache), block_table, kv_lens, cu_q, prefix_pages,
               static_cast<uint16_t*>(out), lse, d.heads / d.kv_heads, __builtin_ctz(d.page_size),
               d.scale * 1.4426950408889634f};
  const int64_t rows = static_cast<int64_t>(d.n_tokens) * d.heads;
  if ((rows + 7) / 8 > 0x7fffffff) return VQB_UNSUPPORTED_GEOMETRY;
  const unsigned blocks = static_cast<unsigned>((rows + 7) / 8);
  if (cudaMemsetAsync(workspace, 0, 16, s) != cudaSuccess) return VQB_CUDA_ERROR;
  cudaError_t ce;
  const bool bf = dtype == VQB_BF16;
  if (d.head_dim == 128)
    ce = bf ? launch_pdl(attention_rows_kernel<true, 128>, blocks, 256, 0, s, p)
            : launch_pdl(attention_rows_kernel<false, 128>, blocks, 256, 0, s, p);
  else
    ce = bf ? launch_pdl(attention_rows_kernel<true, 64>, blocks, 256, 0, s, p)
            : launch_pdl(attention_rows_kernel<false, 64>, blocks, 256, 0, s, p);
  if (ce != cudaSuccess) return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

// vqb_rotary_append: rotary positions on q and k, k and v into the paged cache.
//
// (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t), t = 2 pi pos f.
// f is given in turns per position with 64 fraction bits, so pos * f mod 2^64 is
// the exact fraction of a turn at any position and its upper 32 bits, as a signed
// number of half turns, go to sincospif.  The lower 32 cost up to 2^-32 turns and the
// rounding of the upper ones to fp32 up to 2^-26 (half a unit of a number below 1 half
// turn): 9.5e-8 radians at any position, where a product of fp32 numbers would lose
// 2^-24 of a million turns.
//
// Bound: bytes (each of q, k, v read once and written once).  A block takes a few
// tokens: it computes their rotary_dim / 2 sines and cosines once into shared
// memory, then streams all heads, a thread moving VEC pairs (two 16-byte loads
// and stores when the layout allows).  16385 tokens of 40 + 8 + 8 heads of 128:
// 80 us, 5.9 TB/s; one token 1.9 us in a captured graph.
#include "vqb_common.cuh"
#include "vqb_internal.h"

namespace vqb {
namespace {

constexpr int kThreads = 256;

struct RotaryParams {
  vqb_rotary_desc d;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* positions;
  const int64_t* freq;
  const int32_t* slots;
  uint16_t* q_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int tokens_per_block;
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

// N 16-bit elements, as one access of up to 16 bytes
template <int N>
struct alignas(2 * N < 16 ? 2 * N : 16) Pack {
  uint16_t e[N];
};

template <bool BF16, int VEC>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(RotaryParams p) {
  extern __shared__ float2 s_cs[];  // [tokens][rotary_dim / 2]
  const vqb_rotary_desc& d = p.d;
  const int half = d.rotary_dim / 2;
  const int n0 = blockIdx.x * p.tokens_per_block;
  const int nt = min(p.tokens_per_block, d.n_tokens - n0);
  pdl_wait();
  pdl_trigger();
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int t = i / half, f = i - t * half;
    const uint64_t phase = static_cast<uint64_t>(static_cast<int64_t>(__ldg(p.positions + n0 + t))) *
                           static_cast<uint64_t>(__ldg(p.freq + f));
    const float turns2 = static_cast<float>(static_cast<int32_t>(phase >> 32)) * 4.656612873077393e-10f;  // 2^-31
    float s, c;
    sincospif(turns2, &s, &c);
    s_cs[i] = make_float2(c * d.amplitude, s * d.amplitude);
  }
  __syncthreads();

  const int cpd = d.head_dim / (2 * VEC);      // chunks of VEC pairs in a head
  const int crot = half / VEC;                 // those that are rotated
  const int all_heads = d.heads + 2 * d.kv_heads;
  const int work = nt * all_heads * cpd;
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < work; i += gridDim.y * kThreads) {
    const int c = i % cpd, hn = i / cpd;
    const int h = hn % all_heads, t = hn / all_heads;
    const int64_t n = n0 + t;
    const uint16_t* src;
    uint16_t* dst;
    bool rotate = c < crot;
    if (h < d.heads) {
      src = p.q + n * d.q_token_stride + h * d.q_head_stride;
      dst = p.q_out + n * d.out_token_stride + h * d.out_head_stride;
    } else {
      const int slot = __ldg(p.slots + n);
      const int page = slot / d.page_size, off = slot - page * d.page_size;
      if (slot < 0 || page >= d.num_pages) continue;
      if (h < d.heads + d.kv_heads) {
        const int kh = h - d.heads;
        src = p.k + n * d.k_token_stride + kh * d.k_head_stride;
        dst = p.k_cache + page * d.kc_page_stride + kh * d.kc_head_stride + off * d.kc_token_stride;
      } else {
        const int vh = h - d.heads - d.kv_heads;
        src = p.v + n * d.v_token_stride + vh * d.v_head_stride;
        dst = p.v_cache + page * d.vc_page_stride + vh * d.vc_head_stride + off * d.vc_token_stride;
        rotate = false;
      }
    }
    // where the chunk's two runs of VEC elements start
    int e0 = 2 * VEC * c, e1 = e0 + VEC;
    if (c < crot && !d.interleaved) {
      e0 = VEC * c;
      e1 = e0 + half;
    }
    Pack<VEC> a = *reinterpret_cast<const Pack<VEC>*>(src + e0);
    Pack<VEC> b = *reinterpret_cast<const Pack<VEC>*>(src + e1);
    if (rotate) {
      const float2* cs = s_cs + t * half + VEC * c;
      if (d.interleaved) {
        uint16_t x[2 * VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { x[j] = a.e[j]; x[VEC + j] = b.e[j]; }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = widen<BF16>(x[2 * j]), w = widen<BF16>(x[2 * j + 1]);
          x[2 * j] = narrow<BF16>(u * cs[j].x - w * cs[j].y);
          x[2 * j + 1] = narrow<BF16>(w * cs[j].x + u * cs[j].y);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) { a.e[j] = x[j]; b.e[j] = x[VEC + j]; }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = widen<BF16>(a.e[j]), w = widen<BF16>(b.e[j]);
          a.e[j] = narrow<BF16>(u * cs[j].x - w * cs[j].y);
          b.e[j] = narrow<BF16>(w * cs[j].x + u * cs[j].y);
        }
      }
    }
    *reinterpret_cast<Pack<VEC>*>(dst + e0) = a;
    *reinterpret_cast<Pack<VEC>*>(dst + e1) = b;
  }
}

template <bool BF16>
cudaError_t launch(const RotaryParams& p, int vec, dim3 grid, size_t smem, cudaStream_t s) {
  if (vec == 8) return launch_pdl(rotary_append_kernel<BF16, 8>, grid, kThreads, smem, s, p);
  if (vec == 2) return launch_pdl(rotary_append_kernel<BF16, 2>, grid, kThreads, smem, s, p);
  return launch_pdl(rotary_append_kernel<BF16, 1>, grid, kThreads, smem, s, p);
}

}  // namespace
}  // namespace vqb

using namespace vqb;

extern "C" vqb_status vqb_rotary_append(const vqb_rotary_desc* desc, vqb_dtype dtype, const void* q, const void* k,
                                        const void* v, const int32_t* positions, const int64_t* freq,
                                        const int32_t* slots, void* q_out, void* k_cache, void* v_cache,
                                        vqb_stream_t stream) {
  if (!desc) return VQB_NULL_POINTER;
  const vqb_rotary_desc& d = *desc;
  if (dtype != VQB_F16 && dtype != VQB_BF16) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.n_tokens < 0 || d.heads < 0 || d.kv_heads < 0 || d.head_dim < 2 || d.head_dim % 2 || d.rotary_dim < 0 ||
      d.rotary_dim % 2 || d.rotary_dim > d.head_dim)
    return VQB_BAD_SHAPE;
  if (d.head_dim > 1024 || d.heads > 4096 || d.kv_heads > 4096) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.kv_heads > 0 && (d.page_size < 1 || d.num_pages < 1)) return VQB_BAD_SHAPE;
  if (d.n_tokens == 0 || d.heads + d.kv_heads == 0) return VQB_OK;
  if (!positions || (d.rotary_dim > 0 && !freq) || (d.heads > 0 && (!q || !q_out))) return VQB_NULL_POINTER;
  if (d.kv_heads > 0 && (!k || !v || !slots || !k_cache || !v_cache)) return VQB_NULL_POINTER;
  DeviceInfo di;
  if (device_info(&di) != VQB_OK) return VQB_CUDA_ERROR;

  // the widest access that every address, stride and run of pairs allows (in elements)
  uintptr_t bits = 0;
  auto ptr = [&](const void* x) { bits |= reinterpret_cast<uintptr_t>(x); };
  auto stride = [&](int64_t s) { bits |= static_cast<uintptr_t>(s) * 2; };
  if (d.heads > 0) {
    ptr(q); ptr(q_out);
    stride(d.q_token_stride); stride(d.q_head_stride); stride(d.out_token_stride); stride(d.out_head_stride);
  }
  if (d.kv_heads > 0) {
    ptr(k); ptr(v); ptr(k_cache); ptr(v_cache);
    stride(d.k_token_stride); stride(d.k_head_stride); stride(d.v_token_stride); stride(d.v_head_stride);
    stride(d.kc_page_stride); stride(d.kc_head_stride); stride(d.kc_token_stride);
    stride(d.vc_page_stride); stride(d.vc_head_stride); stride(d.vc_token_stride);
  }
  if (bits & 1) return VQB_BAD_ALIGNMENT;
  const int half = d.rotary_dim / 2;
  int vec = 1;
  if (bits % 16 == 0 && half % 8 == 0 && d.head_dim % 16 == 0) vec = 8;
  else if (bits % 4 == 0 && half % 2 == 0 && d.head_dim % 4 == 0) vec = 2;

  RotaryParams p{d, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                 positions, freq, slots, static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_cache),
                 static_cast<uint16_t*>(v_cache), 1};
  // many tokens: 4 a block, which amortises the block's start; few: a token's heads
  // are spread over up to 4 blocks so that one token does not wait for 2 loads in a row
  if (d.n_tokens > 4 * di.sms) p.tokens_per_block = 4;
  const unsigned gx = static_cast<unsigned>((d.n_tokens + p.tokens_per_block - 1) / p.tokens_per_block);
  unsigned gy = 1;
  const int64_t work = static_cast<int64_t>(d.heads + 2 * d.kv_heads) * (d.head_dim / (2 * vec));
  while (gy < 4 && static_cast<int64_t>(gx) * gy * 2 <= 2 * di.sms && work > static_cast<int64_t>(gy) * kThreads) gy *= 2;
  const size_t smem = sizeof(float2) * static_cast<size_t>(p.tokens_per_block) * (half > 0 ? half : 1);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t ce = dtype == VQB_BF16 ? launch<true>(p, vec, dim3(gx, gy), smem, s)
                                           : launch<false>(p, vec, dim3(gx, gy), smem, s);
  if (ce != cudaSuccess) return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

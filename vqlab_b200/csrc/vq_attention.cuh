// Shared pieces of the attention kernels (vq_attention*.cu).
#pragma once

#include "vqb_common.cuh"
#include "vqb_internal.h"
#include "vqb_tma.cuh"

namespace vqb {

// One attention call.  Partial results (a pass over some of a row's keys):
// part_o fp32 [parts][n_tokens * heads][D] is sum_j 2^(s_j - m) v_j, part_ml
// (m, sum_j 2^(s_j - m)) with scores s in powers of two.
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
  float* part_o;
  float2* part_ml;
  int* status;      // int32 [1] of the workspace
  uint32_t* note;   // behind the status block: `mark` once a masked value may have spoiled a row of this call
  uint32_t mark;    // this call's, not 0
  int group;
  int page_shift;
  float scale_log2;  // scale * log2(e): scores in powers of two
};

// One pass of a call: which keys, how many splits of them, where results go.
struct AttnPass {
  int joint;     // rows of all requests together, over the shared prefix alone
  int prefix;    // (not joint) the request's keys begin with the shared prefix
  int splits;    // 0: no such pass
  int rest;      // (joint) splits of the last pair of tiles, when only one of the two has rows; 0: as the others
  int part0;     // first partial result of the pass, one a split; -1: the pass writes out itself
  int cluster;   // decode kernel: blocks of a cluster, which share a split's keys
  int stage_keys;  // decode kernel: keys of a stage, 16 or 32 (D = 64 only)
  int row_tiles;   // of a block: 16 rows each (decode kernel) or 128 (tile kernel), one or two
  int first;     // the call's first pass: its first block clears the status block
};

// Rows of a key/value head that one block of the tile kernel takes in the pass over the prefix.
__host__ __device__ constexpr int tile_block_rows(int head_dim) { return head_dim == 128 ? 256 : 128; }

// Partial results of the pass over the prefix that a row has: `row` counts the
// rows of its key/value head (token * group + head of the group).
__device__ __forceinline__ int shared_parts(const AttnPass& shared, int block_rows, int rows, int64_t row) {
  return shared.rest && row >= static_cast<int64_t>(rows / block_rows) * block_rows ? shared.rest : shared.splits;
}

vqb_status launch_attention_tiles(const AttnParams& p, const AttnPass& pass, bool bf16, int64_t tiles, cudaStream_t s);
vqb_status launch_attention_decode(const AttnParams& p, const AttnPass& pass, const AttnPass& shared, bool bf16, cudaStream_t s);

constexpr float kLn2 = 0.6931471805599453f;
// A weight is 2^(s - m + kLift), m the running maximum, which follows the scores only
// when they pass it by more than kSlack powers of two: what has been summed is rescaled
// a few times in a long row.  The weights are rounded to the cache's type, and each has
// to keep its relative accuracy, since thousands of small ones may be all of a result (one
// key with a large score and a value of 0 beside them).  bf16 has fp32's exponents.  fp16 is
// accurate from 2^-14 to 2^16, so its weights are lifted to end below 2^15 and are
// good down to 2^-25 of the row's largest; below that a weight is off by at most 2^-36 of it.
// (Without the lift 699 weights of e^-17 came out 44 % too large, of e^-17.5 as 0.)  Partial
// results and the log-sum-exp carry m - kLift for m.
template <bool BF16>
constexpr float kSlack = BF16 ? 8.0f : 4.0f;
template <bool BF16>
constexpr float kLift = BF16 ? 0.0f : 11.0f;

template <bool BF16>
__device__ __forceinline__ uint16_t narrow16(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}
// (lo, hi) as two 16-bit numbers
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The status block starts at zero: written by the call's first block as it starts,
// 2 s before any wait can give up.  Nothing else of the call's first launch may write
// there: no order holds between its blocks.
__device__ __forceinline__ void clear_status(const AttnParams& p, const AttnPass& pass) {
  if (pass.first && (blockIdx.x | blockIdx.y | blockIdx.z) == 0 && threadIdx.x < 4) p.status[static_cast<int>(threadIdx.x) - 1] = 0;
}

// The MMAs multiply a masked value by a weight of 0, which is NaN where the value is
// not finite.  A pass that masks keys says here that a row of it came out not
// finite; a kernel after the passes then works such rows out again (vq_attention.cu).
// The note is the call's own mark, so that no one has to clear it before: whatever
// the word held, it says nothing of this call.  (A word that the first block sets to 0
// could lose another block's note.)
__device__ __forceinline__ void note_not_finite(const AttnParams& p) { *p.note = p.mark; }

// The queries of request r, as far as the call's bounds go.
struct RequestRows {
  int q0;   // first token
  int nq;   // tokens
  int len;  // keys of its own that count
  int at;   // place of its first query among all its keys (below 0: more queries than keys)
};
__device__ __forceinline__ RequestRows request_rows(const AttnParams& p, int r) {
  RequestRows x;
  const int end = __ldg(p.cu_q + r + 1);
  x.q0 = max(__ldg(p.cu_q + r), 0);
  x.nq = max(min(end, p.d.n_tokens) - x.q0, 0);
  const int held = max(__ldg(p.kv_lens + r), 0);
  x.len = min(held, p.d.max_kv_len);
  x.at = held - max(end - x.q0, 0);
  return x;
}
// Own keys that query i of the request sees.
__device__ __forceinline__ int visible(const AttnParams& p, const RequestRows& x, int i) {
  return p.d.causal ? max(min(x.at + i + 1, x.len), 0) : x.len;
}

// 1 / l, the sum of a row's weights.  l = 0: a row that sees no key is 0; one whose
// scores are all -inf is exp(-inf) / exp(-inf), NaN.  (Finite scores make l >= 1.)  own: keys of its
// request that the row sees.
__device__ __forceinline__ float reciprocal_sum(const AttnParams& p, float l, int own) {
  if (l != 0.0f) return 1.0f / l;
  return own > 0 || p.d.prefix_len > 0 ? __int_as_float(0x7FC00000) : 0.0f;
}

// The request whose queries include token n: the last r with cu_q[r] <= n.
__device__ __forceinline__ int request_of(const int32_t* cu_q, int R, int n) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(cu_q + mid) <= n) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      :: "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// A page pool as a tensor [pages][heads][page][D] with the caller's strides;
// a box is 64 elements (one 128-byte swizzle row) of `rows` tokens.
inline vqb_status encode_pool(CUtensorMap* map, const vqb_attention_desc& d, bool bf16, const void* base,
                              int64_t page_stride, int64_t head_stride, int64_t token_stride, int rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return VQB_CUDA_ERROR;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(d.head_dim), static_cast<cuuint64_t>(d.page_size),
                        static_cast<cuuint64_t>(d.kv_heads), static_cast<cuuint64_t>(d.num_pages)};
  int64_t st[3] = {token_stride, head_stride, page_stride};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] == 1) st[i] = d.head_dim;  // never stepped over
    if (st[i] <= 0) return VQB_BAD_SHAPE;
    strides[i] = static_cast<cuuint64_t>(st[i]) * 2;
    if (strides[i] >= (cuuint64_t(1) << 40)) return VQB_UNSUPPORTED_GEOMETRY;
  }
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? VQB_OK
             : VQB_CUDA_ERROR;
}

}  // namespace vqb

// Attention of many query rows over common keys on the 5th-generation tensor
// cores: a long prompt over its own cache, or the rows of a whole batch over the
// prefix that it shares (each prefix page is then read once for 256 rows
// instead of once a request).
//
// A block takes (256 rows of one key/value head and a run of keys): two tiles of
// 128 rows (a row = a token and a head of the group) that share every K and V
// tile of 128 keys; or one tile: at D = 64, and at D = 128 for requests of up to 128 rows
// that are with their heads more than SMs.  Roles:
//   * a TMA warp fills a ring of shared-memory stages with K and V tiles, one
//     box a page and 64 elements (a lane a page);
//   * one thread issues S = Q_t K^T (both from shared memory) into tensor memory,
//     another O_t += P_t V with P_t in tensor memory and V read along its other
//     dimension.  Issuing keeps step with the tensor cores, so one thread for both
//     left them idle while it went from one barrier to the next (3400 cycles a
//     key tile of two row tiles; now 2700);
//   * four softmax warps a tile, a thread a row: the row's 128 scores into
//     registers, running maximum and sum, weights as 16-bit numbers to tensor
//     memory.  O is rescaled in place, by the same thread, only when the maximum
//     has grown by more than 2^kSlack.
// Tensor memory's 512 columns (two tiles, D = 128) hold two O tiles (256), two weight tiles
// (128) and one score tile (128) that the two row tiles use in turn: it is free again as
// soon as the scores are in registers, so the next Q K^T runs beside this tile's
// exponentials and no score waits for a P V.  (With a score tile each, weights
// had to lie over scores, and each tile's chain of exponentials, P V and Q K^T was
// serial: 3900 cycles a key tile against 2100 of MMAs.)
// Bound: the MMAs and the softmax chain between them (2700 cycles a key tile, 2048 of MMAs), at the clock that the power cap
// leaves: 4096 tokens over up to 8192 keys (40 heads, D = 128) take 428 us as a single call at full clock (1.20
// PFLOP/s), 468 to 477 us back to back; at D = 64 the exponentials, which take longer than a key tile's MMAs.
// Scores, weights' sum and O are fp32; the weights are rounded once to the
// cache's type, which the MMA needs (their sum takes them as they were).
//
// Every wait is bounded (2 s): on expiry the block records VQB_TIMEOUT, waits for
// its copies and MMAs in flight, frees its tensor memory and returns.
#include "vq_attention.cuh"

namespace vqb {
namespace {

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
// NT row tiles a block.  Two (D = 128): one block an SM.  One (D = 64, and at D = 128 where the plan has many small requests): two
// blocks share an SM, 256 columns of tensor memory each, so that their starts and ends overlap and rows are dealt in 128s.
// At D = 128 a tile's weights then lie over its scores, the next Q K^T waits for P V, and the other block fills the gaps.
template <int NT>
constexpr int kSoftmaxWarps = 4 * NT;  // four a row tile; then a warp each for Q K^T, P V and the copies
template <int NT>
constexpr int kThreads = NT == 2 ? 352 : 256;
template <int NT>
constexpr int kTmemCols = NT == 2 ? 512 : 256;
// Registers a thread with one row tile: 256 x 128 at launch; the last four warps leave 72 each,
// which the softmax warps take: 128 x 200 + 128 x 56.
constexpr int kRegsSoftmax = 200, kRegsOther = 56;
constexpr int kPolyEvery = 4;  // every fourth pair of exponentials by polynomial
template <int D>
constexpr int kStageBytes = kTileKeys * D * 2;  // a K or a V tile
// Stages of the ring, of K and V tiles in turn.  Even: K and V then have stages of their own, and each stage's "full"
// barrier one issuer that waits for every one of its phases.  With an odd number a stage holds K and V in turn, each
// issuer waits for every second phase only, and a wait by parity takes the phase two before its own for its own
// when the copy between has not landed yet.  Four keep the MMAs as busy as five did (464 us of a 4096-token chunk either
// way) and leave room for two blocks an SM at D = 64.
template <int D, int NT>
constexpr int kStages = D == 128 && NT == 1 ? 2 : 4;
template <int D, int NT>
constexpr size_t tiles_smem() {
  return 1024 + size_t(NT) * kTileRows * D * 2 + size_t(kStages<D, NT>) * kStageBytes<D> + 256;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
               :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// D (+)= A B, A and B in shared memory
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// D (+)= A B, A in tensor memory
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
#define VQB_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define VQB_RW8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
#define VQB_S8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : VQB_R8(v, 0), VQB_R8(v, 8), VQB_R8(v, 16), VQB_R8(v, 24) : "r"(addr) : "memory");
}
// wait for the loads, and keep what uses these registers behind the wait
__device__ __forceinline__ void tc_wait_ld32(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : VQB_RW8(v, 0), VQB_RW8(v, 8), VQB_RW8(v, 16), VQB_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void tc_wait_ld16(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : VQB_RW8(v, 0), VQB_RW8(v, 8)::"memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :: "r"(addr), VQB_S8(v, 0), VQB_S8(v, 8) : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : VQB_R8(v, 0), VQB_R8(v, 8) : "r"(addr) : "memory");
}

// pairs of fp32 numbers
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// the largest, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest of 128 scores.
__device__ __forceinline__ float max128(const float* s) {
  float t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = max3(s[32 * k], s[32 * k + 1], s[32 * k + 2]);
#pragma unroll
  for (int e = 3; e < 31; e += 2)
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = max3(t[k], s[32 * k + e], s[32 * k + e + 1]);
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = max3(t[k], s[32 * k + 31], s[32 * k + 31]);
  return max3(max3(t[0], t[1], t[2]), t[3], t[3]);
}

// 2^x of two numbers on the FMA pipe: x = n + f with n the nearest integer (adding
// 1.5 * 2^23 leaves n in the sum's low bits), 2^f for f in [-1/2, 1/2] by a
// polynomial of degree 4 (least relative error with the constant 1: 2^-18.4, below
// the weights' 16 bits), n added to the exponent.  x is held to -127, for which the
// sum of the bits of 1 and of -127 in the exponent is 0: masked scores (-inf) get
// weight 0.
__device__ __forceinline__ float2 exp2_poly(uint64_t x2) {
  float2 x = unpair(x2);
  x2 = pair(fmaxf(x.x, -127.0f), fmaxf(x.y, -127.0f));
  const uint64_t magic = pair(12582912.0f, 12582912.0f), unmagic = pair(-12582912.0f, -12582912.0f);
  const uint64_t t = add2(x2, magic);
  const uint64_t f = fma2(add2(t, unmagic), pair(-1.0f, -1.0f), x2);
  uint64_t r = fma2(f, pair(0.009582818485796452f, 0.009582818485796452f), pair(0.05590637028217316f, 0.05590637028217316f));
  r = fma2(r, f, pair(0.24024099111557007f, 0.24024099111557007f));
  r = fma2(r, f, pair(0.6931241750717163f, 0.6931241750717163f));
  r = fma2(r, f, pair(1.0f, 1.0f));
  const float2 y = unpair(r), k = unpair(t);
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(k.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(k.y) << 23)));
}

// Weights 2^(score * scale - base) of 32 scores as 16-bit numbers; returns their
// sum.  Every kPolyEvery-th pair goes to the FMA pipe, which is otherwise little
// used, since the special function unit's 16 exponentials a cycle bound a tile as
// much as its MMAs do.
template <bool BF16>
__device__ __forceinline__ float weights32(uint32_t (&pk)[16], const float* s, uint64_t scale2, uint64_t base2) {
  uint64_t sum0 = pair(0.f, 0.f), sum1 = sum0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x2 = fma2(pair(s[2 * e], s[2 * e + 1]), scale2, base2);
    float2 w;
    if (e % kPolyEvery == kPolyEvery - 1) {
      w = exp2_poly(x2);
    } else {
      const float2 x = unpair(x2);
      w = make_float2(exp2_fast(x.x), exp2_fast(x.y));
    }
    if (e & 1) sum1 = add2(sum1, pair(w.x, w.y));
    else sum0 = add2(sum0, pair(w.x, w.y));
    pk[e] = pack16<BF16>(w.x, w.y);
  }
  const float2 t = unpair(add2(sum0, sum1));
  return t.x + t.y;
}

// Shared-memory matrix descriptors, 128-byte swizzle: start >> 4 at [0,14),
// leading byte offset >> 4 at [16,30), stride byte offset >> 4 at [32,46),
// version 1 at [46,48), layout type 2 at [61,64).  Q and K: the contracted
// dimension is contiguous, 8-row groups 1024 bytes apart.  V: the output
// dimension is contiguous, 64 elements a row; 8-key groups 1024 bytes apart
// (stride), the second 64 elements a whole half tile away (leading).
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t leading) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(leading >> 4) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) | (static_cast<uint64_t>(2u) << 61);
}
// kind::f16, fp32 accumulator, A and B of one 16-bit type, N >> 3 at [17,23),
// M >> 4 at [24,29); bit 16: B's output dimension is the contiguous one.
template <bool BF16>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool b_along_n) {
  return (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((b_along_n ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
}

// What a block works on.
struct TileWork {
  RequestRows rq;
  int request;
  int row0, rows;  // its first row, and rows of the request (tokens x group)
  int seg0, seg1;  // keys: of the prefix, of the request itself
};

// The block's request and rows, kRows at a time.  joint: all tokens are one run of rows.  Else
// blocks count pairs of tiles over the requests, the last first (a causal
// prompt's last tiles have the most keys).  false: nothing there.
template <int kRows>
__device__ __forceinline__ bool find_work(const AttnParams& p, const AttnPass& pass, int block, int lane, TileWork* w) {
  const vqb_attention_desc& d = p.d;
  if (pass.joint) {
    w->request = -1;
    w->rq.q0 = 0;
    w->rq.nq = min(__ldg(p.cu_q + d.n_requests), d.n_tokens);
    w->rq.len = w->rq.at = 0;
    w->row0 = block * kRows;
    w->rows = w->rq.nq * p.group;
    w->seg0 = d.prefix_len;
    w->seg1 = 0;
    return w->row0 < w->rows;
  }
  int before = 0;
  for (int base = d.n_requests; base > 0; base -= 32) {
    const int r = base - 1 - lane;
    RequestRows rq{0, 0, 0, 0};
    if (r >= 0) rq = request_rows(p, r);
    const int pairs = (min(rq.nq, d.max_q_len) * p.group + kRows - 1) / kRows;
    int inc = pairs;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + inc > block);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int first = before + __shfl_sync(0xffffffffu, inc - pairs, src);
      const int np = __shfl_sync(0xffffffffu, pairs, src);
      w->request = base - 1 - src;
      w->rq.q0 = __shfl_sync(0xffffffffu, rq.q0, src);
      w->rq.nq = __shfl_sync(0xffffffffu, rq.nq, src);
      w->rq.len = __shfl_sync(0xffffffffu, rq.len, src);
      w->rq.at = __shfl_sync(0xffffffffu, rq.at, src);
      w->rows = min(w->rq.nq, d.max_q_len) * p.group;
      w->row0 = (np - 1 - (block - first)) * kRows;
      w->seg0 = pass.prefix ? d.prefix_len : 0;
      const int last = min(w->row0 + kRows, w->rows) - 1;
      w->seg1 = visible(p, w->rq, last / p.group);
      return true;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}

template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kThreads<NT>, NT == 2 ? 1 : 2)
attention_tiles_kernel(AttnParams p, AttnPass pass, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ unsigned char smem_raw[];
  constexpr int NS = kStages<D, NT>;
  static_assert(NS % 2 == 0, "a stage must hold K tiles only or V tiles only");
  constexpr bool kOver = D == 128 && NT == 1;  // weights over scores
  constexpr int kWarpQk = kSoftmaxWarps<NT>, kWarpPv = kWarpQk + 1, kWarpTma = kWarpQk + 2;
  constexpr int kHalf = kTileKeys * 128;  // 64 elements of 128 rows
  constexpr int kQTile = kTileRows * D * 2;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_s = smem;
  unsigned char* ring = smem + NT * kQTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NS * kStageBytes<D>);
  uint64_t* kv_full = bars;            // [NS] the stage's copies landed
  uint64_t* kv_empty = bars + NS;      // [NS] the MMAs that read the stage are done
  uint64_t* s_full = kv_empty + NS;    // [2] a tile's scores are in tensor memory
  uint64_t* s_read = s_full + 2;       // [2] they are in registers (four warps)
  uint64_t* p_full = s_read + 2;       // [2] its weights are in tensor memory (four warps)
  uint64_t* o_full = p_full + 2;       // [2] its O has this key tile
  uint64_t* mma_done = o_full + 2;     // [2] teardown: an issuer's MMAs are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // values that every lane has alike are broadcast, so that the MMA warp's operands are uniform
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const vqb_attention_desc& d = p.d;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&mma_done[t], 1);
      mbar_init(&s_read[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  clear_status(p, pass);
  pdl_trigger();
  TileWork w;
  // block (tile pair, split): the splits of a pair are neighbours; a last pair of one tile may have fewer
  const int item = blockIdx.x / d.kv_heads, kvh = blockIdx.x % d.kv_heads;
  const int pairs_full = pass.rest ? (d.n_tokens * p.group) / (NT * kTileRows) : 0x7fffffff;
  const bool in_rest = item / pass.splits >= pairs_full;
  const int splits = in_rest ? pass.rest : pass.splits;
  const int tile_pair = in_rest ? pairs_full : item / pass.splits;
  const int split = in_rest ? item - pairs_full * pass.splits : item - tile_pair * pass.splits;
  if (!find_work<NT * kTileRows>(p, pass, tile_pair, lane, &w)) return;  // the same for every thread
  const int tiles0 = (w.seg0 + kTileKeys - 1) / kTileKeys, all = tiles0 + (w.seg1 + kTileKeys - 1) / kTileKeys;
  const int t0 = static_cast<int>(static_cast<int64_t>(all) * split / splits);
  const int n = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / splits) - t0;
  const int active = NT == 2 && w.rows - w.row0 > kTileRows ? 2 : 1;

  uint32_t tmem = 0;
  if (warp < kWarpTma) {
    if (warp == kWarpPv) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                   :: "r"(smem_u32(tmem_slot)), "r"(kTmemCols<NT>) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp < kWarpQk) {
      // Q into shared memory (128-byte swizzle), rows past the last as zeros; K's first tiles are on their way meanwhile
      // (a warp loads its 32 rows, a lane knowing where one of them is)
      const int g = w.row0 + warp * 32 + lane, gq = min(g, w.rows - 1), tok = gq / p.group;
      const unsigned long long mine = reinterpret_cast<unsigned long long>(
          p.q + (w.rq.q0 + tok) * d.q_token_stride + (kvh * p.group + (gq - tok * p.group)) * d.q_head_stride);
      constexpr int kChunks = D / 8, kAtOnce = 32 / kChunks;
      const int c = lane % kChunks;
      const int nlive = min(max(w.rows - (w.row0 + warp * 32), 0), 32);
      const uint32_t to = smem_u32(q_s + (warp >> 2) * kQTile + (c >> 3) * kHalf + (warp & 3) * 32 * 128);
      if (warp < 4 * active) {
#pragma unroll
        for (int r = 0; r < 32; r += kAtOnce) {
          const int row = r + lane / kChunks;
          const unsigned long long src = __shfl_sync(0xffffffffu, mine, row) + c * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                       :: "r"(to + row * 128 + (((c & 7) ^ (row & 7)) << 4)), "l"(src), "r"(row < nlive ? 16 : 0) : "memory");
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("barrier.cta.sync 1, %0;" :: "n"(kWarpTma * 32) : "memory");
    tc_fence_after();
    tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  }
  // columns: the scores of either tile, tile t's weights, its output
  const uint32_t s_col = tmem;
  auto p_col = [&](int t) { return kOver ? tmem : tmem + kTileKeys + t * (kTileKeys / 2); };
  auto o_col = [&](int t) { return tmem + kTileKeys + (kOver ? 0 : NT * (kTileKeys / 2)) + t * D; };

  if (warp >= kWarpQk) {
  if constexpr (NT == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsOther));
  if (warp == kWarpTma) {
    // ---------------- K and V tiles: a lane loads a page
    const int box = min(d.page_size, kTileKeys);
    auto page_of = [&](int i) -> int {  // the lane's page of the i-th tile (past the pool: read as zeros)
      if (i >= n) return d.num_pages;
      const bool own = t0 + i >= tiles0;
      const int start = (own ? t0 + i - tiles0 : t0 + i) * kTileKeys, key = start + lane * box;
      if (lane * box >= kTileKeys || key >= (own ? w.seg1 : w.seg0)) return d.num_pages;
      const int page = own ? __ldg(p.table + static_cast<int64_t>(w.request) * d.table_width + (key >> p.page_shift))
                           : __ldg(p.prefix_pages + (key >> p.page_shift));
      return static_cast<unsigned>(page) < static_cast<unsigned>(d.num_pages) ? page : d.num_pages;
    };
    int page = page_of(0);
    bool ok = true;
    int issued = 0;
    for (int i = 0; i < n && ok; ++i) {
      const int page_next = page_of(i + 1);
      const bool own = t0 + i >= tiles0;
      const int start = (own ? t0 + i - tiles0 : t0 + i) * kTileKeys;
      const int held = min((own ? w.seg1 : w.seg0) - start, kTileKeys);
      const int boxes = (held + box - 1) / box;
#pragma unroll
      for (int kv = 0; kv < 2 && ok; ++kv) {
        const int st = (2 * i + kv) % NS;
        if (!warp_wait(&kv_empty[st], (((2 * i + kv) / NS) & 1) ^ 1, abort_flag)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(&kv_full[st], static_cast<uint32_t>(boxes * box * D * 2));
        __syncwarp();
        ++issued;
        if (lane < boxes) {
          unsigned char* dst = ring + st * kStageBytes<D> + lane * box * 128;
          const int off = (start + lane * box) & (d.page_size - 1);
#pragma unroll
          for (int h = 0; h < D / 64; ++h)
            tma_load_4d(kv == 0 ? &kmap : &vmap, &kv_full[st], dst + h * kHalf, h * 64, off, kvh, page);
        }
      }
      page = page_next;
    }
    // no copy may still be writing shared memory when the block ends
    if (lane == 0)
      for (int k = max(issued - NS, 0); k < issued; ++k) mbar_drain(&kv_full[k % NS], (k / NS) & 1);
  } else if (warp == kWarpQk) {
    // ---------------- S = Q_t K^T for the two tiles in turn: 16 of D a step
    constexpr uint32_t idesc = idesc_f16<BF16>(kTileKeys, false);
    const bool issuer = elect_one();
    const uint64_t q0 = desc128(smem_u32(q_s), 16), k0 = desc128(smem_u32(ring), 16);
    bool ok = true;
    int st = 0, phase = 0;  // K's stage: every second one
    for (int i = 0; i < n && ok; ++i) {
      ok = mbar_wait(&kv_full[st], phase, abort_flag);
      const uint64_t b = k0 + static_cast<uint32_t>(st) * (kStageBytes<D> >> 4);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t == 1 && active < 2) break;
        // the score tile is free once the scores before are in registers (kOver: once their weights have met the values)
        if (t == 1) ok = ok && mbar_wait(&s_read[0], i & 1, abort_flag);
        else if (i > 0) ok = ok && mbar_wait(kOver ? &o_full[0] : &s_read[active - 1], (i - 1) & 1, abort_flag);
        tc_fence_after();
        __syncwarp();
        if (issuer && ok) {
          const uint64_t a = q0 + t * (kQTile >> 4);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
            tc_mma_ss(s_col, a + off, b + off, idesc, ks > 0);
          }
          tc_commit(&s_full[t]);
          if (t == active - 1) tc_commit(&kv_empty[st]);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      st += 2;
      if (st >= NS) {
        st -= NS;
        phase ^= 1;
      }
    }
    if (issuer) {
      tc_commit(&mma_done[0]);
      mbar_drain(&mma_done[0], 0);
    }
    __syncwarp();
  } else if (warp == kWarpPv) {
    // ---------------- O_t (+)= P_t V: 16 keys a step, up to the last that is held
    constexpr uint32_t idesc = idesc_f16<BF16>(D, true);
    const bool issuer = elect_one();
    const uint64_t v0 = desc128(smem_u32(ring), kHalf);
    bool ok = true;
    int st = 1, phase = 0;
    for (int i = 0; i < n && ok; ++i) {
      const bool own = t0 + i >= tiles0;
      const int held = (own ? w.seg1 : w.seg0) - (own ? t0 + i - tiles0 : t0 + i) * kTileKeys;
      const int steps = (min(held, kTileKeys) + 15) / 16;
      ok = mbar_wait(&kv_full[st], phase, abort_flag);
      const uint64_t b = v0 + static_cast<uint32_t>(st) * (kStageBytes<D> >> 4);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t == 1 && active < 2) break;
        ok = ok && mbar_wait(&p_full[t], i & 1, abort_flag);
        tc_fence_after();
        __syncwarp();
        if (issuer && ok) {
          if (steps == 8) {
            tc_mma_ts(o_col(t), p_col(t), b, idesc, i > 0);
#pragma unroll
            for (int ks = 1; ks < 8; ++ks) tc_mma_ts(o_col(t), p_col(t) + ks * 8, b + ks * (2048 >> 4), idesc, 1);
          } else {
            for (int ks = 0; ks < steps; ++ks)
              tc_mma_ts(o_col(t), p_col(t) + ks * 8, b + ks * (2048 >> 4), idesc, i > 0 || ks > 0);
          }
          tc_commit(&o_full[t]);
          if (t == active - 1) tc_commit(&kv_empty[st]);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      st += 2;
      if (st >= NS) {
        st -= NS;
        phase ^= 1;
      }
    }
    if (issuer) {
      tc_commit(&mma_done[1]);
      mbar_drain(&mma_done[1], 0);
    }
    __syncwarp();
  }
  } else {
    // ---------------- softmax: a thread a row
    if constexpr (NT == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kRegsSoftmax));
    const int t = warp >> 2;
    if (t < active) {
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const int g = w.row0 + t * kTileRows + (warp & 3) * 32 + lane;
      const int gv = min(g, w.rows - 1), tok = gv / p.group;
      const int vis = pass.joint ? 0 : visible(p, w.rq, tok);
      const uint32_t srow = s_col + lanes, prow = p_col(t) + lanes, orow = o_col(t) + lanes;
      const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int i = 0; i < n; ++i) {
        const bool own = t0 + i >= tiles0;
        const int start = (own ? t0 + i - tiles0 : t0 + i) * kTileKeys;
        const int held = min((own ? w.seg1 : w.seg0) - start, kTileKeys);
        const int lim = own ? vis - start : held;
        if (!(ok = warp_wait(&s_full[t], i & 1, abort_flag))) break;
        tc_fence_after();
        float s[128];
        uint32_t* u = reinterpret_cast<uint32_t*>(s);
#pragma unroll
        for (int c = 0; c < 4; ++c) tc_ld32(srow + c * 32, u + c * 32);
#pragma unroll
        for (int c = 0; c < 4; ++c) tc_wait_ld32(u + c * 32);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_read[t]);
        if (__any_sync(0xffffffffu, lim < kTileKeys)) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= lim) s[c] = -INFINITY;
        }
        const float mx = max128(s) * p.scale_log2;
        bool fresh = i == 0;
        if (__any_sync(0xffffffffu, mx > m + kSlack<BF16>)) {
          const float mn = fmaxf(m, mx);
          const float f = mn == -INFINITY ? 1.0f : exp2_fast(m - mn);
          m = mn;
          l *= f;
          if (i > 0) {
            if (!(ok = warp_wait(&o_full[t], (i - 1) & 1, abort_flag))) break;
            fresh = true;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tc_ld16(orow + c * 16, o);
              tc_wait_ld16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tc_st16(orow + c * 16, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m - kLift<BF16>;
        const uint64_t base2 = pair(-base, -base);
        uint32_t pk0[16], pk1[16];
        l += weights32<BF16>(pk0, s, scale2, base2);
        l += weights32<BF16>(pk1, s + 32, scale2, base2);
        // the weights of the key tile before have met their values once its MMAs are done
        if (!fresh) {
          if (!(ok = warp_wait(&o_full[t], (i - 1) & 1, abort_flag))) break;
          tc_fence_after();
        }
        tc_st16(prow, pk0);
        tc_st16(prow + 16, pk1);
        l += weights32<BF16>(pk0, s + 64, scale2, base2);
        tc_st16(prow + 32, pk0);
        l += weights32<BF16>(pk1, s + 96, scale2, base2);
        tc_st16(prow + 48, pk1);
        // NaN or inf among the scores: NaN, also where the polynomial clamped it
        if (!(mx < INFINITY)) l = __int_as_float(0x7FC00000);
        if (t == 0 && (warp & 3) == 0 && (held & 15)) {
          // what lies past the last key may be anything: its weight is 0, its value must be finite
          const int st = (2 * i + 1) % NS;
          if (!(ok = warp_wait(&kv_full[st], ((2 * i + 1) / NS) & 1, abort_flag))) break;
          const int first = held, rows = ((held + 15) & ~15) - held;
          for (int e = lane; e < rows * (D / 8); e += 32) {
            const int rr = first + e / (D / 8), c = e % (D / 8);
            *reinterpret_cast<uint4*>(ring + st * kStageBytes<D> + (c >> 3) * kHalf + rr * 128 + (c & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok && n > 0) ok = warp_wait(&o_full[t], (n - 1) & 1, abort_flag);
      if (!ok && lane == 0) *p.status = VQB_TIMEOUT;
      if (ok) {
        tc_fence_after();
        m -= kLift<BF16>;
        const int64_t token = w.rq.q0 + tok;
        const int head = kvh * p.group + (gv - tok * p.group);
        const int64_t grow = token * d.heads + head;
        const bool live = g < w.rows;
        const bool partial = pass.part0 >= 0;
        const int64_t at = (pass.part0 + split) * (static_cast<int64_t>(d.n_tokens) * d.heads) + grow;
        const float inv = reciprocal_sum(p, l, vis);
        // through shared memory (Q's, which no MMA reads any more), so that a row leaves as whole lines: D 16-bit
        // numbers, or half of its fp32 ones at a time
        constexpr int kRowBytes = D * 2, kRowChunks = kRowBytes / 16;
        unsigned char* stage = q_s + t * kQTile + (warp & 3) * 32 * kRowBytes;
        unsigned char* mine = partial ? reinterpret_cast<unsigned char*>(p.part_o + at * D)
                                      : reinterpret_cast<unsigned char*>(p.out + token * d.out_token_stride + head * d.out_head_stride);
        float zero = 0.0f;  // NaN once an element is not finite
        for (int pass2 = 0; pass2 < (partial ? 2 : 1); ++pass2) {
          const int cols = partial ? D / 2 : D;
#pragma unroll 1
          for (int c = 0; c < cols / 32; ++c) {
            uint32_t o[32];
            if (n > 0) {
              tc_ld32(orow + pass2 * (D / 2) + c * 32, o);
              tc_wait_ld32(o);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) zero = fmaf(__uint_as_float(o[e]), 0.0f, zero);
            if (partial) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(stage + lane * kRowBytes + (((c * 8 + e) ^ (lane & 7)) << 4)) =
                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 16; ++e)
                pk[e] = pack16<BF16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4*>(stage + lane * kRowBytes + (((c * 4 + e) ^ (lane & 7)) << 4)) =
                    make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
            }
            __syncwarp();
          }
          const int nlive = min(max(w.rows - (g - lane), 0), 32);  // rows of the warp that exist
#pragma unroll
          for (int r = 0; r < 32; r += 32 / kRowChunks) {
            const int rr = r + lane / kRowChunks, c = lane % kRowChunks;
            const unsigned long long to = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), rr);
            if (rr < nlive)
              *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(to) + pass2 * kRowBytes + c * 16) =
                  *reinterpret_cast<const uint4*>(stage + rr * kRowBytes + ((c ^ (rr & 7)) << 4));
          }
          __syncwarp();
        }
        if (live && vis < w.seg1 && zero != 0.0f) note_not_finite(p);
        if (live) {
          if (partial) p.part_ml[at] = make_float2(m, l);
          else if (p.lse) p.lse[grow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpPv)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(kTmemCols<NT>) : "memory");
}

template <int D, bool BF16, int NT>
vqb_status launch(const AttnParams& p, const AttnPass& pass, int64_t tiles, const CUtensorMap& km, const CUtensorMap& vm,
                  cudaStream_t s) {
  constexpr size_t smem = tiles_smem<D, NT>();
  static_assert((NT == 2 ? 1 : 2) * (smem + 1024) <= 233472, "over the opt-in shared memory of an SM");
  if (cudaFuncSetAttribute(attention_tiles_kernel<D, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return VQB_CUDA_ERROR;
  // the rows with the most keys first, over all heads
  const int64_t items = pass.rest ? static_cast<int64_t>(tiles - 1) * pass.splits + pass.rest
                                  : static_cast<int64_t>(tiles) * pass.splits;
  if (items * p.d.kv_heads > 0x7fffffff) return VQB_UNSUPPORTED_GEOMETRY;
  const dim3 grid(static_cast<unsigned>(items * p.d.kv_heads));
  if (launch_pdl(attention_tiles_kernel<D, BF16, NT>, grid, kThreads<NT>, smem, s, p, pass, km, vm) != cudaSuccess)
    return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

}  // namespace

// tiles: an upper bound of the blocks of rows (pass.row_tiles row tiles each) of the pass.
vqb_status launch_attention_tiles(const AttnParams& p, const AttnPass& pass, bool bf16, int64_t tiles, cudaStream_t s) {
  CUtensorMap km, vm;
  const vqb_attention_desc& d = p.d;
  const int box = d.page_size < kTileKeys ? d.page_size : kTileKeys;
  vqb_status st = encode_pool(&km, d, bf16, p.kc, d.kc_page_stride, d.kc_head_stride, d.kc_token_stride, box);
  if (st != VQB_OK) return st;
  st = encode_pool(&vm, d, bf16, p.vc, d.vc_page_stride, d.vc_head_stride, d.vc_token_stride, box);
  if (st != VQB_OK) return st;
  if (d.head_dim == 128 && pass.row_tiles == 2)
    return bf16 ? launch<128, true, 2>(p, pass, tiles, km, vm, s) : launch<128, false, 2>(p, pass, tiles, km, vm, s);
  if (d.head_dim == 128)
    return bf16 ? launch<128, true, 1>(p, pass, tiles, km, vm, s) : launch<128, false, 1>(p, pass, tiles, km, vm, s);
  return bf16 ? launch<64, true, 1>(p, pass, tiles, km, vm, s) : launch<64, false, 1>(p, pass, tiles, km, vm, s);
}

}  // namespace vqb

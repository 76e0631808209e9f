// Attention of requests with few query rows (tokens x heads of a group <= 16)
// over their own keys: one pass over the cache, bound by its bytes.
//
// A cluster of blocks takes (request, key/value head) and splits its keys evenly.
// A block's four warps are independent: each streams every fourth group of keys of
// the block's run through its own ring of shared-memory stages (8 KB of K and V in
// 2 KB TMA boxes of 16 keys; the warp's first lane refills a stage as soon as the warp has
// read it), with its own running maximum and sum.  A warp computes
// S = Q K^T and O += P V with m16n8k16 MMAs: Q and O stay in registers, P goes from
// the accumulator's layout, rounded to the cache's type, straight into the next MMA's operand.  Of 17 to 32 rows
// two warps take 16 each and share a ring, whose stages are refilled once both have
// read them.  Long runs of keys move at 6.0 TB/s at D = 128 (24 requests of up to 15000 keys
// and 5 rows, 8 heads: 115 us; the bytes take 105); with two row tiles the MMAs begin to bind (24 of up to 8000 keys
// and 20 rows, 4 heads: 66 us, 3.0 TB/s; the bytes take 30).
//
// The results are joined without leaving the kernel: the four warps' in shared
// memory, then the cluster's over distributed shared memory (each block joins its
// share of the rows), then, when the batch has a shared prefix, with the partial
// results of the pass over the prefix.  That pass is the kernel before this one on
// the stream; this one starts as its blocks end and waits for it only here.  Only
// where eight blocks for a (request, head) would leave most SMs idle do several
// clusters share it, and a join kernel follows.
#include "vq_attention.cuh"

namespace vqb {
namespace {

constexpr int kWarps = 4;
constexpr int kGroup = 16;  // keys of a box, which lies in one page
// RT warps share a ring, each with its own 16 rows (RT = 1 or 2: up to 16 or 32 rows a block); 4 / RT rings split
// the block's keys.  A stage holds U keys: 16 at D = 128, 32 at D = 64 -- or 16 there, with RT = 1 (the plan says when).
// Stages of a ring, and blocks an SM: of 64 KB and 168 registers, or (16 keys at D = 64) of 48 KB and 128 registers.
template <int D, int U, int RT>
constexpr int kStages = U * D == 1024 ? 3 : 2 * RT;
template <int D, int U>
constexpr int kResident = U * D == 1024 ? 4 : 3;
template <int D, int U>
constexpr int kHalfBytes = U * D * 2;  // K or V of a stage
template <int D, int U, int RT>
constexpr size_t kRingBytes = size_t(kStages<D, U, RT>) * 2 * kHalfBytes<D, U>;
template <int D, int U>
constexpr size_t kWarpBytes = U * D == 1024 ? 12288 : 16384;  // a warp's share of the rings; at the end it holds fp32 [16][D]

// A block's shared memory: the rings first (1024-byte aligned, as the copies'
// swizzle needs: the block has no other shared memory), then the small things.
template <int D, int U, int RT>
struct DecodeSmem {
  unsigned char rings[kWarps * kWarpBytes<D, U>];
  uint64_t full[kWarps / RT][kStages<D, U, RT>];   // a stage's copies have landed
  uint64_t empty[kWarps / RT][kStages<D, U, RT>];  // RT > 1: all its warps have read it
  float2 ml[16 * RT];  // the block's own
  float m[kWarps][16], l[kWarps][16];
  int abort;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// every thread of every block of the cluster, always the same number of times
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 ld_remote4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float2 ld_remote2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}

// A running join of partial results (m, l, four elements of O).
struct Joined {
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float pm, float pl, float4 po) {
    const float mn = fmaxf(m, pm), base = mn == -INFINITY ? 0.0f : mn;
    const float f = exp2_fast(m - base), g = exp2_fast(pm - base);
    m = mn;
    l = l * f + pl * g;
    o.x = o.x * f + po.x * g;
    o.y = o.y * f + po.y * g;
    o.z = o.z * f + po.z * g;
    o.w = o.w * f + po.w * g;
  }
};

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, bool BF16, int U, int RT>
__global__ void __launch_bounds__(kWarps * 32, kResident<D, U>)
attention_decode_kernel(AttnParams p, AttnPass pass, AttnPass shared, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ __align__(1024) unsigned char smem[];
  using Smem = DecodeSmem<D, U, RT>;
  Smem& sm = *reinterpret_cast<Smem*>(smem);
  auto& s_full = sm.full;
  auto& s_m = sm.m;
  auto& s_l = sm.l;
  auto& s_ml = sm.ml;
  int& s_abort = sm.abort;
  constexpr int NS = kStages<D, U, RT>, KW = kWarps / RT, kG = U / kGroup, kGroupBytes = kGroup * D * 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kw = warp / RT, rt = warp % RT;  // its ring, and which 16 of the block's rows
  const vqb_attention_desc& d = p.d;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int w = 0; w < KW; ++w)
      for (int i = 0; i < NS; ++i) {
        mbar_init(&s_full[w][i], 1);
        if (RT > 1) mbar_init(&sm.empty[w][i], RT);
      }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // With a pass over the prefix before this kernel, that pass's blocks have all
  // waited for what came before them by the time this one may start, and only its
  // results have to be waited for, below.
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
  }
  if (pass.first) pdl_wait();
  pdl_trigger();
  clear_status(p, pass);
  // the request's table row is on its way while its lengths are read (a call whose requests hold nothing may have no table)
  if (d.max_kv_len > 0 && static_cast<int>(threadIdx.x) * 32 < d.table_width)
    asm volatile("prefetch.global.L1 [%0];"
                 :: "l"(p.table + static_cast<int64_t>(blockIdx.z) * d.table_width + threadIdx.x * 32) : "memory");

  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int kvh = blockIdx.y, r = blockIdx.z;
  const int cluster = blockIdx.x / ranks;
  const RequestRows rq = request_rows(p, r);
  const int nrows = min(rq.nq * p.group, 16 * RT);
  // Whoever waits for this kernel also waits for the pass before it, through the
  // first block; the others may leave before that pass has ended.
  const bool waits = !pass.first && (blockIdx.x | blockIdx.y | blockIdx.z) == 0;
  if (nrows == 0) {  // the same for the whole cluster
    if (waits) pdl_wait();
    return;
  }
  const int seg0 = pass.prefix ? d.prefix_len : 0;
  const int seg1 = visible(p, rq, rq.nq - 1);
  const int tiles0 = (seg0 + U - 1) / U, tiles = tiles0 + (seg1 + U - 1) / U;
  const int split = cluster * ranks + rank, splits = gridDim.x;
  const int u0 = static_cast<int>(static_cast<int64_t>(tiles) * split / splits);
  const int u1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / splits);
  // this ring's stages: u0 + kw, then every KW-th
  const int n = u1 - u0 > kw ? (u1 - u0 - kw + KW - 1) / KW : 0;
  unsigned char* ring = smem + kw * kRingBytes<D, U, RT>;

  auto page_of = [&](int k) -> int {  // page of the ring's k-th group of 16 keys (past the end: read as zeros)
    const int u = u0 + kw + KW * (k / kG);
    const bool own = u >= tiles0;
    const int key = (own ? u - tiles0 : u) * U + (k % kG) * kGroup;
    if (k >= n * kG || key >= (own ? seg1 : seg0)) return d.num_pages;
    const int page = own ? __ldg(p.table + static_cast<int64_t>(r) * d.table_width + (key >> p.page_shift))
                         : __ldg(p.prefix_pages + (key >> p.page_shift));
    return static_cast<unsigned>(page) < static_cast<unsigned>(d.num_pages) ? page : d.num_pages;
  };
  // the ring's k-th stage, by its first warp; lane g copies its g-th group
  auto issue = [&](int k, int page) {
    const int u = u0 + kw + KW * k;
    const int key = (u < tiles0 ? u : u - tiles0) * U + lane * kGroup;
    const int off = key & (d.page_size - 1);
    uint64_t* bar = &s_full[kw][k % NS];
    unsigned char* dst = ring + (k % NS) * 2 * kHalfBytes<D, U> + lane * kGroupBytes;
    if (lane == 0) mbar_expect_tx(bar, 2 * kHalfBytes<D, U>);
    if constexpr (kG > 1) __syncwarp();
    if (lane < kG) {
#pragma unroll
      for (int h = 0; h < D / 64; ++h) tma_load_4d(&kmap, bar, dst + h * 2048, h * 64, off, kvh, page);
#pragma unroll
      for (int h = 0; h < D / 64; ++h) tma_load_4d(&vmap, bar, dst + kHalfBytes<D, U> + h * 2048, h * 64, off, kvh, page);
    }
  };

  // pages of 32 groups at a time, one a lane; the next 32 are fetched while these are used
  int pages = 0, pages_next = 0, issued = 0;
  if (rt == 0) {
    pages = page_of(lane);
    pages_next = page_of(32 + lane);
    for (; issued < NS && issued < n; ++issued) issue(issued, __shfl_sync(0xffffffffu, pages, issued * kG + lane % kG));
  }

  // Q as the first operand: rows lane / 4 and lane / 4 + 8
  const int row0 = lane >> 2, row1 = row0 + 8;  // of the warp's 16
  const int wrows = min(max(nrows - rt * 16, 0), 16), first = rt * 16;
  uint32_t qf[D / 16][4];
  {
    auto qrow = [&](int row) {
      const int g = first + row;
      return p.q + (rq.q0 + g / p.group) * d.q_token_stride + (kvh * p.group + g % p.group) * d.q_head_stride;
    };
    const uint16_t* a = qrow(row0 < wrows ? row0 : -rt * 16);
    const uint16_t* b = qrow(row1 < wrows ? row1 : -rt * 16);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int e = ks * 16 + (lane & 3) * 2;
      qf[ks][0] = row0 < wrows ? *reinterpret_cast<const uint32_t*>(a + e) : 0u;
      qf[ks][1] = row1 < wrows ? *reinterpret_cast<const uint32_t*>(b + e) : 0u;
      qf[ks][2] = row0 < wrows ? *reinterpret_cast<const uint32_t*>(a + e + 8) : 0u;
      qf[ks][3] = row1 < wrows ? *reinterpret_cast<const uint32_t*>(b + e + 8) : 0u;
    }
  }
  const int vis0 = visible(p, rq, min((first + row0) / p.group, rq.nq - 1));
  const int vis1 = visible(p, rq, min((first + row1) / p.group, rq.nq - 1));

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  // a lane's row address for the two kinds of 8x8 matrix loads
  const int krow = ((lane >> 4) << 3) + (lane & 7), kchunk = (lane >> 3) & 1;
  const int vrow = (((lane >> 3) & 1) << 3) + (lane & 7), vchunk = lane >> 4;
  for (int k = 0; k < n; ++k) {
    if (!warp_wait(&s_full[kw][k % NS], (k / NS) & 1, &s_abort)) {
      // gave up: copies in flight must land before the ring is used again
      for (int j = k; lane == 0 && j < issued; ++j) mbar_drain(&s_full[kw][j % NS], (j / NS) & 1);
      if (lane == 0) *p.status = VQB_TIMEOUT;
      break;
    }
    if (RT == 1 || wrows > 0) {
      const int u = u0 + kw + KW * k;
      const bool own = u >= tiles0;
      const int key = (own ? u - tiles0 : u) * U;
      const uint32_t kb = smem_u32(ring + (k % NS) * 2 * kHalfBytes<D, U>), vb = kb + kHalfBytes<D, U>;
      const int lim0 = min((own ? vis0 : seg0) - key, U), lim1 = min((own ? vis1 : seg0) - key, U);
      const int held = min((own ? seg1 : seg0) - key, U);
      if (held < U) {
        // what lies past the last key may be anything: its weight is 0, its value must be finite
        unsigned char* v = ring + (k % NS) * 2 * kHalfBytes<D, U> + kHalfBytes<D, U>;
        for (int i = lane; i < (U - held) * (D / 8); i += 32) {
          const int rr = held + i / (D / 8), c = i % (D / 8);
          *reinterpret_cast<uint4*>(v + (rr / kGroup) * kGroupBytes + (c >> 3) * 2048 + (rr % kGroup) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a copy reuses the stage
        __syncwarp();
      }
      float s[2 * kG][4];
#pragma unroll
      for (int t = 0; t < 2 * kG; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          uint32_t b[4];
          const int c = ks * 2 + kchunk;
          ldsm4(b, kb + g * kGroupBytes + (c >> 3) * 2048 + krow * 128 + (((c & 7) ^ (krow & 7)) << 4));
          mma16816<BF16>(s[2 * g], qf[ks], b[0], b[1]);
          mma16816<BF16>(s[2 * g + 1], qf[ks], b[2], b[3]);
        }
      if (__any_sync(0xffffffffu, lim0 < U || lim1 < U)) {
#pragma unroll
        for (int t = 0; t < 2 * kG; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = t * 8 + (lane & 3) * 2 + e;
            if (col >= lim0) s[t][e] = -INFINITY;
            if (col >= lim1) s[t][2 + e] = -INFINITY;
          }
      }
      float t0 = fmaxf(s[0][0], s[0][1]), t1 = fmaxf(s[0][2], s[0][3]);
#pragma unroll
      for (int t = 1; t < 2 * kG; ++t) {
        t0 = fmaxf(t0, fmaxf(s[t][0], s[t][1]));
        t1 = fmaxf(t1, fmaxf(s[t][2], s[t][3]));
      }
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)) * p.scale_log2;
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2)) * p.scale_log2;
      if (__any_sync(0xffffffffu, t0 > m0 + kSlack<BF16> || t1 > m1 + kSlack<BF16>)) {
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float f0 = n0 == -INFINITY ? 1.0f : exp2_fast(m0 - n0), f1 = n1 == -INFINITY ? 1.0f : exp2_fast(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= f0;
          o[i][1] *= f0;
          o[i][2] *= f1;
          o[i][3] *= f1;
        }
      }
      const float b0 = m0 == -INFINITY ? 0.0f : m0 - kLift<BF16>, b1 = m1 == -INFINITY ? 0.0f : m1 - kLift<BF16>;
#pragma unroll
      for (int t = 0; t < 2 * kG; ++t) {
        s[t][0] = exp2_fast(fmaf(s[t][0], p.scale_log2, -b0));
        s[t][1] = exp2_fast(fmaf(s[t][1], p.scale_log2, -b0));
        s[t][2] = exp2_fast(fmaf(s[t][2], p.scale_log2, -b1));
        s[t][3] = exp2_fast(fmaf(s[t][3], p.scale_log2, -b1));
        l0 += s[t][0] + s[t][1];
        l1 += s[t][2] + s[t][3];
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float(*w)[4] = s + 2 * g;
        const uint32_t pf[4] = {pack16<BF16>(w[0][0], w[0][1]), pack16<BF16>(w[0][2], w[0][3]),
                                pack16<BF16>(w[1][0], w[1][1]), pack16<BF16>(w[1][2], w[1][3])};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t b[4];
          const int c = i * 2 + vchunk;
          ldsm4_t(b, vb + g * kGroupBytes + (c >> 3) * 2048 + vrow * 128 + (((c & 7) ^ (vrow & 7)) << 4));
          mma16816<BF16>(o[2 * i], pf, b[0], b[1]);
          mma16816<BF16>(o[2 * i + 1], pf, b[2], b[3]);
        }
      }
    }
    __syncwarp();
    // the stage that is free: this one, or, where other warps may still read this one, the one before
    const int done = RT == 1 ? k : k - 1, next = done + NS;
    if constexpr (RT > 1) {
      if (lane == 0) mbar_arrive(&sm.empty[kw][k % NS]);
      if (rt != 0 || done < 0 || next >= n) continue;
      if (!warp_wait(&sm.empty[kw][done % NS], (done / NS) & 1, &s_abort)) {
        for (int j = k + 1; lane == 0 && j < issued; ++j) mbar_drain(&s_full[kw][j % NS], (j / NS) & 1);
        if (lane == 0) *p.status = VQB_TIMEOUT;
        break;
      }
    }
    if ((next * kG & 31) == 0) {
      pages = pages_next;
      pages_next = page_of(next * kG + 32 + lane);
    }
    const int pg = __shfl_sync(0xffffffffu, pages, (next * kG & 31) + lane % kG);
    if (next < n) {
      issue(next, pg);
      issued = next + 1;
    }
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  // ---- the results of the warps with the same rows, joined: each leaves its own where its ring, or a part of it, was
  if constexpr (RT > 1) __syncthreads();
  else __syncwarp();
  float* mine = reinterpret_cast<float*>(smem + warp * kWarpBytes<D, U>);  // [16][D]
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const int e = i * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2*>(mine + row0 * D + e) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(mine + row1 * D + e) = make_float2(o[i][2], o[i][3]);
  }
  if ((lane & 3) == 0) {
    s_m[warp][row0] = m0 - kLift<BF16>;
    s_l[warp][row0] = l0;
    s_m[warp][row1] = m1 - kLift<BF16>;
    s_l[warp][row1] = l1;
  }
  __syncthreads();
  constexpr int kPer = D / 4;  // threads of a row, four elements each
  constexpr size_t kShare = kWarpBytes<D, U> / sizeof(float);
  float* rings = reinterpret_cast<float*>(smem);
  for (int i = threadIdx.x; i < nrows * kPer; i += kWarps * 32) {
    const int row = i / kPer, e = (i % kPer) * 4;
    Joined j;
#pragma unroll
    for (int c = 0; c < KW; ++c) {
      const int w = c * RT + row / 16;
      j.add(s_m[w][row % 16], s_l[w][row % 16], *reinterpret_cast<const float4*>(rings + w * kShare + (row % 16) * D + e));
    }
    *reinterpret_cast<float4*>(rings + (row / 16) * kShare + (row % 16) * D + e) = j.o;  // this thread alone reads these elements
    if (e == 0) s_ml[row] = make_float2(j.m, j.l);
  }
  if (ranks > 1) cluster_sync();
  else __syncthreads();
  const bool partial = pass.part0 >= 0;
  if (!pass.first && !partial) pdl_wait();  // the prefix's partial results
  // ---- rows dealt over the cluster's blocks
  const int64_t all_rows = static_cast<int64_t>(d.n_tokens) * d.heads;
  for (int i = threadIdx.x; i < ((nrows - static_cast<int>(rank) + static_cast<int>(ranks) - 1) / static_cast<int>(ranks)) * kPer;
       i += kWarps * 32) {
    const int row = (i / kPer) * ranks + rank, e = (i % kPer) * 4;
    Joined j;
    for (uint32_t c = 0; c < ranks; ++c) {
      const float2 ml = ld_remote2(remote(&s_ml[row], c));
      j.add(ml.x, ml.y, ld_remote4(remote(rings + (row / 16) * kShare + (row % 16) * D + e, c)));
    }
    const int64_t tok = rq.q0 + row / p.group;
    const int head = kvh * p.group + row % p.group;
    const int64_t grow = tok * d.heads + head;
    if (visible(p, rq, row / p.group) < seg1 && (j.o.x + j.o.y + j.o.z + j.o.w) * 0.0f != 0.0f) note_not_finite(p);
    if (partial) {
      const int64_t at = (pass.part0 + cluster) * all_rows + grow;
      *reinterpret_cast<float4*>(p.part_o + at * D + e) = j.o;
      if (e == 0) p.part_ml[at] = make_float2(j.m, j.l);
    } else {
      const int joins = pass.first ? 0 : shared_parts(shared, tile_block_rows(D), d.n_tokens * p.group, tok * p.group + row % p.group);
#pragma unroll 4
      for (int i2 = 0; i2 < joins; ++i2) {
        const int64_t at = i2 * all_rows + grow;
        const float2 ml = __ldcg(p.part_ml + at);
        j.add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + e)));
      }
      const float inv = reciprocal_sum(p, j.l, visible(p, rq, row / p.group));
      const uint2 w = make_uint2(pack16<BF16>(j.o.x * inv, j.o.y * inv), pack16<BF16>(j.o.z * inv, j.o.w * inv));
      *reinterpret_cast<uint2*>(p.out + tok * d.out_token_stride + head * d.out_head_stride + e) = w;
      if (p.lse && e == 0) p.lse[grow] = j.l == 0.0f ? -INFINITY : (j.m + log2f(j.l)) * kLn2;
    }
  }
  if (ranks > 1) cluster_sync();  // no block leaves while another reads its memory
  if (waits) pdl_wait();
}

template <int D, bool BF16, int U, int RT>
vqb_status launch(const AttnParams& p, const AttnPass& pass, const AttnPass& shared, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  constexpr size_t smem = sizeof(DecodeSmem<D, U, RT>);
  if (cudaFuncSetAttribute(attention_decode_kernel<D, BF16, U, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return VQB_CUDA_ERROR;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pass.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pass.splits * pass.cluster, p.d.kv_heads, p.d.n_requests);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, attention_decode_kernel<D, BF16, U, RT>, p, pass, shared, km, vm) != cudaSuccess) return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

template <int D, bool BF16>
vqb_status launch_rows(const AttnParams& p, const AttnPass& pass, const AttnPass& shared, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  constexpr int U = 2048 / D;
  if (pass.row_tiles == 2) return launch<D, BF16, U, 2>(p, pass, shared, km, vm, s);
  if (pass.stage_keys < U) return launch<D, BF16, 16, 1>(p, pass, shared, km, vm, s);
  return launch<D, BF16, U, 1>(p, pass, shared, km, vm, s);
}

}  // namespace

vqb_status launch_attention_decode(const AttnParams& p, const AttnPass& pass, const AttnPass& shared, bool bf16, cudaStream_t s) {
  CUtensorMap km, vm;
  const vqb_attention_desc& d = p.d;
  vqb_status st = encode_pool(&km, d, bf16, p.kc, d.kc_page_stride, d.kc_head_stride, d.kc_token_stride, kGroup);
  if (st != VQB_OK) return st;
  st = encode_pool(&vm, d, bf16, p.vc, d.vc_page_stride, d.vc_head_stride, d.vc_token_stride, kGroup);
  if (st != VQB_OK) return st;
  if (d.head_dim == 128) return bf16 ? launch_rows<128, true>(p, pass, shared, km, vm, s) : launch_rows<128, false>(p, pass, shared, km, vm, s);
  return bf16 ? launch_rows<64, true>(p, pass, shared, km, vm, s) : launch_rows<64, false>(p, pass, shared, km, vm, s);
}

}  // namespace vqb

// vqb_paged_tables: one step's block tables, lengths and slot map from the
// requests' lengths.
//
// The mathematics is three running sums over the requests r (context c, new n,
// page size P): pages given back (n = -1: ceil(c / P)), new tokens, and pages
// needed (ceil((c + n) / P) - ceil(c / P)).  With them every output element has
// a closed form: request r's j-th new page is entry (start + need sum before r
// + j) of the ring of free pages, extended by the pages given back in this
// call, and token t belongs to the request whose token sum covers it.  So no
// element waits for another: every block computes the sums itself (a few
// thousand integers out of L2, about a microsecond) and then writes its share
// of the rows and tokens -- one launch and no grid-wide step.  In an in-place
// call the values that it overwrites and a block may still read (lengths,
// state, the rows of finished requests) are written by the block that arrives
// last.
//
// Bound: bytes (table rows in and out, 12 bytes a token); small steps are
// bound by the launch and a chain of latencies: lengths, sums, pages, stores.
// So what does not depend on the sums is fetched beside them, one warp takes
// the 64-bit remainders, page numbers are products instead of quotients, and
// rows and tokens are dealt to all SMs.  Per step in a captured graph: 8
// requests 5.0 -> 3.6 us, 1000 requests with 512-wide rows 9.2 -> 7.6 us (their
// 5.6 MB take 0.9), 300 prompts of up to 600 tokens 7.2 -> 5.4 us.  In place: 3.3,
// 9.1 and 6.3 us for steps without new tokens, 13 and 7.9 us for the latter two with
// (copies that restore the inputs taken off); the arrival of all blocks and the last
// one's writes are longer than the copies that it saves.
#include "vqb_common.cuh"
#include "vqb_internal.h"

namespace vqb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxRequests = 8192;

struct PagedParams {
  vqb_paged_desc d;
  const int32_t* context;
  const int32_t* fresh;
  const int32_t* table_in;
  const int32_t* ring_in;
  int64_t* state;
  int32_t* table;
  int32_t* ring;
  int64_t* state_out;
  int32_t* kv_lens;
  int32_t* cu_q;
  int32_t* slots;
  int32_t* positions;
  int32_t* requests;
  uint32_t per_page, shift;  // x / page_size of a non-negative x is x * per_page >> shift
};

// x / P for 0 <= x < 2^31 by a product: with l = ceil(log2 P) and M = floor(2^(31 + l) / P) + 1, M P = 2^(31 + l) + e with
// 0 < e <= P <= 2^l, so x M / 2^(31 + l) = x / P + x e / (P 2^(31 + l)) and the last term is below 1 / P.
__device__ __forceinline__ int page_of(const PagedParams& p, int x) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * p.per_page) >> p.shift);
}

// What a request that holds c tokens and gets n more holds and wants; lengths
// below zero count as zero and a row never holds more pages than it has places.
struct Request {
  int held;    // pages of its row in use
  int tokens;  // new tokens
  int need;    // pages it lacks
  int back;    // pages it gives back
  bool gone;   // it has finished
  bool fits;   // its row has places enough
};

__device__ __forceinline__ Request request(const PagedParams& p, int c, int n) {
  const vqb_paged_desc& d = p.d;
  Request q;
  c = max(c, 0);
  q.held = min(c > 0 ? page_of(p, c - 1) + 1 : 0, d.table_width);
  q.tokens = max(n, 0);
  const int64_t end = static_cast<int64_t>(c) + q.tokens;
  const int pages = end > 0 ? page_of(p, static_cast<int>(min(end, int64_t{0x7fffffff})) - 1) + 1 : 0;
  q.gone = n < 0;
  q.fits = pages <= d.table_width && end <= 0x7fffffff;
  q.need = q.gone || !q.fits ? 0 : max(pages - q.held, 0);
  q.back = q.gone ? q.held : 0;
  return q;
}

// The last index in [0, n) whose sum is <= v (sums[0] = 0, non-decreasing).
__device__ __forceinline__ int find(const int* sums, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= v) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void prefetch_l2(const void* a) { asm volatile("prefetch.global.L2 [%0];" ::"l"(a)); }

// VEC: table rows move as 16-byte vectors
template <bool VEC>
__global__ void __launch_bounds__(kThreads) paged_tables_kernel(PagedParams p) {
  extern __shared__ int s_sums[];
  const vqb_paged_desc& d = p.d;
  const int R = d.n_requests, W = d.table_width, P = d.page_size;
  int* s_tok = s_sums;               // [R + 1] new tokens before r
  int* s_need = s_tok + R + 1;       // [R + 1] pages needed before r
  int* s_back = s_need + R + 1;      // [R + 1] pages given back before r
  int* s_ctx = s_back + R + 1;       // [R] tokens held, [R] new tokens: read once, so that
  int* s_new = s_ctx + R;            //     every later step is free of their latency
  __shared__ int s_warp[3][kThreads / 32];
  __shared__ int s_refused, s_given, s_last;
  __shared__ uint32_t s_head_mod, s_tail_mod;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const uint32_t F = static_cast<uint32_t>(d.ring_size);
  const bool table_in_place = p.table == p.table_in, ring_in_place = p.ring == p.ring_in;
  const bool lens_in_place = p.kv_lens == p.context, state_in_place = p.state == p.state_out;
  // rows are dealt to the blocks in turn, from a block's first warp on, tokens and ring places 32 at a time from its last
  // warp down: every SM has its share, and in a small step other warps have the tokens than have the rows
  const int gwarp = warp * gridDim.x + blockIdx.x, gwarps = gridDim.x * (kThreads / 32);
  const int64_t gthreads = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t gthread = static_cast<int64_t>(kThreads / 32 - 1 - warp) * gridDim.x * 32 + blockIdx.x * 32 + lane;
  const int64_t head = __ldcg(p.state), tail = __ldcg(p.state + 1);
  // what does not depend on the sums is on its way while they are made: the warp's first row, the thread's first ring place
  if (gwarp < R && lane * 32 < W) prefetch_l2(p.table_in + static_cast<int64_t>(gwarp) * W + lane * 32);
  const int first_place = !ring_in_place && gthread < F ? __ldcg(p.ring_in + gthread) : 0;
  if (tid == 0) {
    s_refused = 0;
    s_given = 0;
  }

  // ---- the three sums: a thread adds up a run of requests, then the threads' totals are scanned
  for (int r = tid; r < R; r += kThreads) {
    s_ctx[r] = __ldcg(p.context + r);
    s_new[r] = __ldcg(p.fresh + r);
  }
  __syncthreads();
  if (warp == kThreads / 32 - 1) {
    // one warp divides for all (a 64-bit remainder is some 80 instructions), and fetches the ring's next pages
    const uint32_t hm = static_cast<uint32_t>(static_cast<uint64_t>(head) % F);
    if (lane == 0) {
      s_head_mod = hm;
      s_tail_mod = static_cast<uint32_t>(static_cast<uint64_t>(tail) % F);
    }
    prefetch_l2(p.ring_in + (hm + static_cast<uint32_t>(lane) * 32) % F);
  }
  auto load = [&](int r) { return request(p, s_ctx[r], s_new[r]); };
  const int per = (R + kThreads - 1) / kThreads;
  const int r0 = min(tid * per, R), r1 = min(r0 + per, R);
  int tot[3] = {0, 0, 0};
  for (int r = r0; r < r1; ++r) {
    const Request q = load(r);
    tot[0] += q.tokens;
    tot[1] += q.need;
    tot[2] += q.back;
  }
  int inc[3] = {tot[0], tot[1], tot[2]};
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int v = __shfl_up_sync(0xffffffffu, inc[k], o);
      if (lane >= o) inc[k] += v;
    }
  }
  if (lane == 31) {
#pragma unroll
    for (int k = 0; k < 3; ++k) s_warp[k][warp] = inc[k];
  }
  __syncthreads();
  {
    int at[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      at[k] = inc[k] - tot[k] + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[k][lane] : 0);
    }
    for (int r = r0; r < r1; ++r) {
      const Request q = load(r);
      s_tok[r] = at[0];
      s_need[r] = at[1];
      s_back[r] = at[2];
      at[0] += q.tokens;
      at[1] += q.need;
      at[2] += q.back;
    }
    if (r1 == R && (r0 < R || tid == 0)) {  // the thread with the last request (thread 0 when there is none)
      s_tok[R] = at[0];
      s_need[R] = at[1];
      s_back[R] = at[2];
    }
  }
  __syncthreads();

  const int returned = s_back[R], total = s_tok[R];
  const int64_t waiting = tail - head;  // entries of the ring before this call's returns
  const int64_t avail = waiting + returned;
  const uint32_t head_mod = s_head_mod, tail_mod = s_tail_mod;
  auto taken = [&](int r, const Request& q) {
    return !q.gone && q.fits && (q.need == 0 || static_cast<int64_t>(s_need[r]) + q.need <= avail);
  };
  // entry `i` from the ring's start: a free page, or one given back in this call
  auto page_at = [&](int i) -> int {
    if (i < waiting) return __ldcg(p.ring_in + (head_mod + static_cast<uint32_t>(i)) % F);
    const int b = i - static_cast<int>(waiting);
    if (b < 0 || b >= returned) return -1;
    // the last request whose sum is <= b gives it back: those after it with the same sum give nothing
    const int r = find(s_back, R, b);
    return __ldcg(p.table_in + static_cast<int64_t>(r) * W + (b - s_back[r]));
  };

  // ---- table rows and pages given back, a warp to a request
  for (int r = gwarp; r < R; r += gwarps) {
    const Request q = load(r);
    const bool ok = taken(r, q);
    const int32_t* in = p.table_in + static_cast<int64_t>(r) * W;
    int32_t* out = p.table + static_cast<int64_t>(r) * W;
    const int first_new = ok && lane < q.need ? page_at(s_need[r] + lane) : -1;  // beside the row's own loads
    if (q.gone) {
      for (int j = lane; j < q.held; j += 32)
        p.ring[(tail_mod + static_cast<uint32_t>(s_back[r] + j)) % F] = __ldcg(in + j);
    }
    const int keep = q.gone ? 0 : q.held;
    if (!table_in_place) {
      if constexpr (VEC) {
#pragma unroll 4
        for (int j = 4 * lane; j < W; j += 128) {
          int4 v = make_int4(-1, -1, -1, -1);
          if (j < keep) {
            v = __ldcg(reinterpret_cast<const int4*>(in + j));
            if (j + 1 >= keep) v.y = -1;
            if (j + 2 >= keep) v.z = -1;
            if (j + 3 >= keep) v.w = -1;
          }
          *reinterpret_cast<int4*>(out + j) = v;
        }
      } else {
#pragma unroll 4
        for (int j = lane; j < W; j += 32) out[j] = j < keep ? __ldcg(in + j) : -1;
      }
      __syncwarp();
    }
    if (ok)
      for (int j = lane; j < q.need; j += 32) out[q.held + j] = j == lane ? first_new : page_at(s_need[r] + j);
    if (!lens_in_place && lane == 0) p.kv_lens[r] = q.gone ? 0 : max(s_ctx[r], 0) + (ok ? q.tokens : 0);
  }
  // the ring's other places (those given back in this call were written above)
  if (!ring_in_place) {
    for (int64_t i = gthread; i < F; i += gthreads) {
      const uint32_t from_tail = (static_cast<uint32_t>(i) + F - tail_mod) % F;
      if (from_tail >= static_cast<uint32_t>(returned)) p.ring[i] = i == gthread ? first_place : __ldcg(p.ring_in + i);
    }
  }
  // ---- tokens
  for (int64_t t = gthread; t < d.max_tokens; t += gthreads) {
    int slot = -1, pos = 0, r = -1;
    if (t < total) {
      r = find(s_tok, R, static_cast<int>(t));
      const Request q = load(r);
      const int place = static_cast<int>(static_cast<uint32_t>(max(s_ctx[r], 0)) + static_cast<uint32_t>(t - s_tok[r]));
      pos = static_cast<int>(static_cast<uint32_t>(d.position_offset) + static_cast<uint32_t>(place));
      if (taken(r, q)) {
        const int col = page_of(p, place);
        const int page = col < q.held ? __ldcg(p.table_in + static_cast<int64_t>(r) * W + col)
                                      : page_at(s_need[r] + col - q.held);
        if (page >= 0) slot = static_cast<int>(static_cast<uint32_t>(page) * P + (place - col * P));
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.requests[t] = r;
  }
  if (blockIdx.x == 0)
    for (int r = tid; r <= R; r += kThreads) p.cu_q[r] = s_tok[r];

  // ---- what is written over what other blocks may still read: by the block that
  // arrives last (none but this one when the grid is one block)
  const bool over = table_in_place || lens_in_place || state_in_place;
  if (over && gridDim.x > 1) {
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      const unsigned long long n = atomicAdd(reinterpret_cast<unsigned long long*>(p.state + 3), 1ull);
      s_last = n == gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
  } else {
    if (blockIdx.x != 0) return;
    __syncthreads();
  }
  int refused = 0, given = 0;
  for (int r = tid; r < R; r += kThreads) {
    const Request q = load(r);
    const bool ok = taken(r, q);
    if (!q.gone && !ok) ++refused;
    if (ok) given += q.need;
    if (lens_in_place) p.kv_lens[r] = q.gone ? 0 : max(s_ctx[r], 0) + (ok ? q.tokens : 0);
  }
  if (refused) atomicAdd(&s_refused, refused);
  if (given) atomicAdd(&s_given, given);
  if (table_in_place) {
    for (int r = warp; r < R; r += kThreads / 32) {
      const int back = s_back[r + 1] - s_back[r];
      for (int j = lane; j < back; j += 32) p.table[static_cast<int64_t>(r) * W + j] = -1;
    }
  }
  __syncthreads();
  if (tid == 0) {
    if (over && gridDim.x > 1) p.state[3] = 0;
    p.state_out[0] = head + s_given;
    p.state_out[1] = tail + returned;
    p.state_out[2] = s_refused;
    p.state_out[3] = 0;
  }
}

}  // namespace
}  // namespace vqb

using namespace vqb;

extern "C" vqb_status vqb_paged_tables(const vqb_paged_desc* desc, const int32_t* context_lens, const int32_t* new_lens,
                                       const int32_t* block_table, const int32_t* free_pages, int64_t* state,
                                       int32_t* block_table_out, int32_t* free_pages_out, int64_t* state_out,
                                       int32_t* kv_lens, int32_t* cu_q, int32_t* slots, int32_t* positions,
                                       int32_t* requests, vqb_stream_t stream) {
  if (!desc) return VQB_NULL_POINTER;
  const vqb_paged_desc& d = *desc;
  if (d.n_requests < 0 || d.table_width < 1 || d.page_size < 1 || d.ring_size < 1 || d.max_tokens < 0)
    return VQB_BAD_SHAPE;
  if (d.n_requests > kMaxRequests) return VQB_UNSUPPORTED_GEOMETRY;
  if (!free_pages || !state || !free_pages_out || !state_out || !cu_q) return VQB_NULL_POINTER;
  if (d.n_requests > 0 && (!context_lens || !new_lens || !block_table || !block_table_out || !kv_lens))
    return VQB_NULL_POINTER;
  if (d.max_tokens > 0 && (!slots || !positions || !requests)) return VQB_NULL_POINTER;
  DeviceInfo di;
  if (device_info(&di) != VQB_OK) return VQB_CUDA_ERROR;
  PagedParams p{d, context_lens, new_lens, block_table, free_pages, state, block_table_out, free_pages_out, state_out,
                kv_lens, cu_q, slots, positions, requests, 0, 31};
  while ((1ull << (p.shift - 31)) < static_cast<uint64_t>(d.page_size)) ++p.shift;
  p.per_page = static_cast<uint32_t>((1ull << p.shift) / d.page_size + 1);
  // a block for every 16 rows (one a warp) or 512 tokens or ring places, one block an SM at most
  int64_t blocks = (static_cast<int64_t>(d.n_requests) + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t others = (static_cast<int64_t>(d.max_tokens) + kThreads - 1) / kThreads;
  const int64_t places = block_table == block_table_out ? 0 : (static_cast<int64_t>(d.ring_size) + kThreads - 1) / kThreads;
  blocks = blocks > others ? blocks : others;
  blocks = blocks > places ? blocks : places;
  blocks = blocks < 1 ? 1 : (blocks > di.sms ? di.sms : blocks);
  const size_t smem = sizeof(int) * (5 * static_cast<size_t>(d.n_requests) + 3);
  const bool vec = d.table_width % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(block_table_out)) & 15) == 0;
  const auto kern = vec ? paged_tables_kernel<true> : paged_tables_kernel<false>;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem)) != cudaSuccess)
    return VQB_CUDA_ERROR;
  if (launch_pdl(kern, static_cast<unsigned>(blocks), kThreads, smem, reinterpret_cast<cudaStream_t>(stream), p) !=
      cudaSuccess)
    return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

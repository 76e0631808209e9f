// vqb_prefix_attention: attention of a batch over the paged cache.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j,
// in one pass over the keys with a running maximum.  Sums over disjoint sets of
// a row's keys join exactly: with partial (m_i, l_i, O_i) and M = max m_i,
// o = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  So a call is a list of passes
// over parts of the keys, and a join when there are several partial results:
//   * rows of all requests together over the shared prefix
//     (vq_attention_tiles.cu): its pages are read once for 256 rows;
//   * each request's own keys: vq_attention_decode.cu for up to 16 rows a
//     key/value head (32 in batches of many requests), vq_attention_tiles.cu for more;
//   * both over splits of the keys where there are fewer blocks than SMs.
#include <atomic>

#include "vq_attention.cuh"

namespace vqb {
namespace {

struct AttnPlan {
  AttnPass shared;     // splits = 0: no pass over the prefix alone
  AttnPass own;
  bool decode;         // the own pass runs the decode kernel
  int64_t shared_tiles, own_tiles;  // pairs of row tiles (own: an upper bound)
  int parts;           // partial results in the workspace
  bool join;           // a join kernel follows (else the own pass writes out)
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Times in microseconds: a key tile of a block with two row tiles (D = 64: of one of
// two blocks on an SM), with one, and a block's start and end.
constexpr double kPairTile = 1.5, kOneTile = 1.2, kBlockEnds = 7.0;
constexpr int kMaxSplits = 64;

// Splits of `tiles` key tiles over the tile kernel's blocks: the fewest rounds of
// the longest block, and the join's traffic (`row_cost`: a partial result's).
int pick_splits(int64_t blocks, int64_t tiles, int slots, double row_cost, bool joined_anyway, double* time = nullptr) {
  int best = 1;
  double best_t = 1e30;
  for (int s = 1; s <= kMaxSplits && s <= tiles; ++s) {
    const double rounds = static_cast<double>(ceil_div(blocks * s, slots));
    double t = rounds * (static_cast<double>(ceil_div(tiles, s)) * kPairTile + kBlockEnds);
    if (s > 1 || joined_anyway) t += row_cost * s + 4.0;
    if (t < best_t * 0.98) {
      best_t = t;
      best = s;
    }
  }
  if (time) *time = best_t;
  return best;
}

// The decode kernel's time with `cluster` blocks a (request, head), in microseconds: what the blocks cost besides their keys,
// times the rounds (a third of one at least: a block an SM), and their meeting; and the longest run of keys, bound by its own copies, beside all keys, bound by memory (half of the
// shorter one still shows).  With one row tile a block (two) a round of blocks costs 5 us (10; 7.5 at D = 64) and a key of a
// run 11.3 ns (25), 0.6 of that at D = 64.  Lengths are taken to average 0.55 of the largest.  Fitted to 32 (14)
// batches of 1 to 200 requests with 200 to 15000 keys, each timed with 1, 2, 4 and 8 blocks: the choice costs 0.5 % on
// average against the best of the four.  (Two rounds of blocks with 512 keys or more cost 6 %: 8 requests of up
// to 900 keys 15.1 us in clusters of 8, 10.3 of 4; 64 of up to 600 28.2 us in clusters of 2, 23.5 without.)
double decode_time(const vqb_attention_desc& d, int row_tiles, int64_t keys, int cluster, int sms) {
  const double rh = static_cast<double>(d.n_requests) * d.kv_heads, half = d.head_dim == 64 ? 0.5 : 1.0;
  const double block = row_tiles == 1 ? 5.0 : d.head_dim == 64 ? 7.5 : 10.0;
  const double run = static_cast<double>(keys) / cluster * (row_tiles == 1 ? 0.0113 : 0.025) * (d.head_dim == 64 ? 0.6 : 1.0);
  const double all = 0.55 * keys * rh * 0.08e-3 * half * (row_tiles == 1 ? 1.0 : 1.25);
  const double rounds = rh * cluster / (3 * sms);
  const double meet = cluster == 1 ? 0.0 : cluster == 2 ? 0.95 : cluster == 4 ? 1.15 : 1.35;  // the cluster's blocks
  return meet + block * (rounds > 0.33 ? rounds : 0.33) + (run > all ? run + 0.5 * all : all + 0.5 * run);
}

int pick_cluster(const vqb_attention_desc& d, int row_tiles, int64_t keys, int sms, double* time) {
  int best = 1;
  *time = decode_time(d, row_tiles, keys, 1, sms);
  for (int c = 2; c <= 8; c *= 2) {
    const double t = decode_time(d, row_tiles, keys, c, sms);
    if (t < *time) {
      *time = t;
      best = c;
    }
  }
  return best;
}

// Splits of the pass over the prefix before a decode pass over the requests' own
// keys, which takes `alone` us by itself (bound by memory) and needs `other` SM
// microseconds.  Either it has all SMs first and the decode pass joins the partial
// results, or it leaves SMs on which the decode pass runs at the same time (one is
// bound by arithmetic, the other by memory), and a join kernel follows (about 9 us).
// Measured: 250 requests behind 32768 keys with up to 2000 of their own 306 us in
// turn, 274 us together (2 splits: 80 blocks); 64 requests behind 16421 keys with up
// to 500 of their own 52 us in turn, 56 us together.  Returns true for the latter.
bool pick_shared_splits(AttnPass* a, int64_t full, bool rest, int heads, int64_t tiles, int sms, double row_cost,
                        double other, double alone) {
  double best_t = 1e30;
  bool together = false;
  for (int s = 1; s <= kMaxSplits && s <= tiles; ++s) {
    const int s2 = rest ? static_cast<int>(s * kOneTile / kPairTile + 0.999) : 0;
    const int64_t n1 = full * s * heads, n2 = static_cast<int64_t>(s2) * heads;
    const double t1 = full ? kBlockEnds + kPairTile * ceil_div(tiles, s) : 0.0;
    const double t2 = rest ? kBlockEnds + kOneTile * ceil_div(tiles, s2) : 0.0;
    const double longest = t1 > t2 ? t1 : t2;
    for (int mode = 0; mode < 2; ++mode) {
      double t;
      if (mode == 0) {
        t = ceil_div(n1 + n2, sms) * longest + alone + row_cost * s;
      } else {
        if (n1 + n2 > sms) continue;  // none left
        t = (n1 * t1 + n2 * t2 + other) / sms;
        if (t < longest) t = longest;
        t += row_cost * (s + 1) + 9.0;
      }
      if (t < best_t * 0.98) {
        best_t = t;
        a->splits = s;
        a->rest = s2;
        together = mode == 1;
      }
    }
  }
  return together;
}

AttnPlan make_plan(const vqb_attention_desc& d, int sms) {
  AttnPlan a{};
  const int block_rows = tile_block_rows(d.head_dim);
  const int slots = d.head_dim == 128 ? sms : 2 * sms;  // blocks of the tile kernel at a time
  const int group = d.heads / d.kv_heads;
  const int64_t rows = static_cast<int64_t>(d.n_tokens) * group;  // of one key/value head
  const int64_t most = static_cast<int64_t>(d.max_q_len < d.n_tokens ? d.max_q_len : d.n_tokens) * group;
  // the prefix for all rows at once, unless a request fills tiles by itself
  const bool joint = d.prefix_len > 0 && d.n_requests > 1 && most <= 256;
  // a partial result written and read, at 4 TB/s
  const double row_cost = static_cast<double>(d.n_tokens) * d.heads * d.head_dim * 8.0 / 4.0e6;
  const int64_t keys = static_cast<int64_t>(d.max_kv_len) + (joint ? 0 : d.prefix_len);
  const int64_t requests_heads = static_cast<int64_t>(d.n_requests) * d.kv_heads;
  a.own.prefix = !joint && d.prefix_len > 0;
  // A request's own rows at D = 128: blocks of two row tiles, or, where requests have one tile and are more than SMs, blocks of
  // one, two an SM (86 requests of 40 rows and up to 64 keys 39 -> 27 us, 24 of 20 rows and up to 8000 keys 106 -> 95 us; 16
  // of 25 rows and up to 2000 keys on 128 blocks would take 32 us instead of 29).
  const int own_rows = d.head_dim == 128 && (most > 128 || requests_heads <= sms) ? 256 : 128;
  a.own_tiles = rows / own_rows + d.n_requests;
  const int64_t blocks = (rows / own_rows > d.n_requests ? rows / own_rows : d.n_requests) * d.kv_heads;
  double tiles_t, decode_t;
  a.own.splits = pick_splits(blocks, ceil_div(keys, 128), own_rows == 256 ? sms : 2 * sms, row_cost, joint, &tiles_t);
  // The decode kernel for up to 16 rows, and for up to 32 where it is the faster one: short contexts, and D = 64 (200 requests of
  // 25 rows and up to 300 keys 60 us, in tiles 73; 64 of 25 rows at D = 64 and up to 1000 keys 27 us, in tiles 32; but 64 of 25
  // rows and up to 2500 keys 91 us, in tiles 86, and 16 of up to 500 17 us, in tiles 13).  With 64 rows a block the tile kernel
  // had nearly every batch.
  const int decode_tiles = most <= 16 ? 1 : 2;
  a.own.cluster = pick_cluster(d, decode_tiles, keys, sms, &decode_t);
  a.decode = most <= 16 || (most <= 32 && decode_t < tiles_t);
  a.own.row_tiles = a.decode ? decode_tiles : own_rows / 128;
  if (a.decode) {
    a.own.splits = 1;
    // Several clusters a (request, head), of 256 keys a block or more, and a join kernel, where clusters of eight would leave most
    // SMs idle.  One request with 8 heads at D = 128: 4200 keys 11.7 us, 11.1 in one cluster; 5000 11.8 and 11.9; 6500 12.6 and
    // 14.1; 8200 12.7 and 16.6; with one head 4200 10.0 and 10.6, 16000 11.4 and 26.3; 8 heads at D = 64: 4200 8.7 and 7.9, 8000 9.5 and 10.0.
    if (most <= 16 && requests_heads * 8 < sms && keys > 8 * 512) {
      const int64_t fill = ceil_div(2 * sms, requests_heads * 8), most_k = keys / (8 * 256);
      a.own.cluster = 8;
      a.own.splits = static_cast<int>(fill < most_k ? fill : most_k);
    }
    // At D = 64 stages of 32 keys, which share a stage's fixed work: 24 requests of up to 15000 keys 68 -> 62 us, 250 of up
    // to 5000 214 -> 205 us.  They leave room for three blocks an SM, stages of 16 for four, which is better where that many
    // blocks are one round and have few keys each, or run beside the pass over the prefix for few; the rule asks for the round
    // alone.  16 against 32 keys, 8 heads: 74 requests of up to 300 8.6 and 10.9 us, of 2000 33.2 and 32.8; 33 of 2000 18.8 and 20.2; 60 of 1000 17.7
    // and 16.5; 4 heads: 140 of up to 100 6.0 and 8.9, of 1000 18.2 and 19.0, 117 of 2000 28.9 and 25.6; behind a prefix: 64 of 500
    // behind 16000 36.5 and 38.5, 30 of 300 behind 3000 12.8 and 14.3, 100 of 1500 behind 5000 49.1 and 45.6, 250 of 2500 behind 9000 145 and 140.
    const int64_t n = requests_heads * a.own.cluster * a.own.splits;
    a.own.stage_keys = d.head_dim == 64 && !joint && !(n > 3 * sms && n <= 4 * sms) ? 32 : 16;
  }
  bool together = !a.decode;  // the own pass leaves partial results too
  if (joint) {
    a.shared.joint = 1;
    a.shared.row_tiles = block_rows / 128;
    a.shared.first = 1;
    a.shared_tiles = ceil_div(rows, block_rows);
    // the last block has one row tile with rows, of two
    const bool rest = d.head_dim == 128 && rows % block_rows > 0 && rows % block_rows <= block_rows / 2;
    const int64_t tiles = ceil_div(d.prefix_len, 128);
    if (a.decode) {
      // an SM's time for the own keys: 100 GB/s and 2 us a block, with lengths that average 0.6 of the largest
      const double bytes = 0.6 * keys * requests_heads * d.head_dim * 4.0;
      const double other = bytes / 1.0e5 + 2.0 * requests_heads * a.own.cluster;
      const double alone = bytes / 6.4e6 > other / sms ? bytes / 6.4e6 : other / sms;
      together = pick_shared_splits(&a.shared, a.shared_tiles - rest, rest, d.kv_heads, tiles, slots, row_cost, other * slots / sms, alone);
    } else {
      a.shared.splits = pick_splits(a.shared_tiles * d.kv_heads, tiles, slots, row_cost, true);
    }
  }
  a.own.first = a.shared.splits == 0;
  a.join = a.own.splits > 1 || (a.shared.splits > 0 && together);
  a.own.part0 = a.join ? a.shared.splits : -1;
  a.parts = a.shared.splits + (a.join ? a.own.splits : 0);
  return a;
}

constexpr size_t kStatusBytes = 256;  // the status block (16 bytes), then the note

size_t part_rows(const vqb_attention_desc& d) { return static_cast<size_t>(d.n_tokens) * d.heads; }
size_t ml_bytes(const vqb_attention_desc& d, int parts) { return (parts * part_rows(d) * sizeof(float2) + 255) & ~size_t(255); }

// Joins a row's partial results, a warp a row: a lane weighs a part, then the
// parts' elements are read without waiting for one another.  Bound: the partial
// results' bytes, which are in L2 as a rule.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attention_join_kernel(AttnParams p, AttnPass shared, int own_parts) {
  pdl_wait();
  pdl_trigger();
  const vqb_attention_desc& d = p.d;
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(d.n_tokens) * d.heads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t n = row / d.heads;
  const int h = static_cast<int>(row - n * d.heads);
  if (n >= __ldg(p.cu_q + d.n_requests)) return;
  const int ns = shared.splits ? shared_parts(shared, tile_block_rows(D), d.n_tokens * p.group, n * p.group + h % p.group) : 0;
  const int parts = ns + own_parts;  // the own pass's follow the `splits` places of the shared one's
  constexpr int kPer = D / 32;
  float m = -INFINITY, l = 0.0f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const int i = i0 + lane;
    const int64_t at = (i < ns ? i : i - ns + shared.splits) * rows + row;
    const float2 ml = i < parts ? __ldcg(p.part_ml + at) : make_float2(-INFINITY, 0.0f);
    float top = ml.x;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
    const float keep = exp2_fast(m - base), w = exp2_fast(ml.x - base);
    m = mn;
    float sum = ml.y * w;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * keep + sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= keep;
    const int here = min(parts - i0, 32);
#pragma unroll 4
    for (int k = 0; k < here; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float* o = p.part_o + __shfl_sync(0xffffffffu, at, k) * D + lane * kPer;
      if constexpr (kPer == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(o));
        acc[0] += v.x * wk;
        acc[1] += v.y * wk;
        acc[2] += v.z * wk;
        acc[3] += v.w * wk;
      } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(o));
        acc[0] += v.x * wk;
        acc[1] += v.y * wk;
      }
    }
  }
  int own = 0;
  if (l == 0.0f) {
    const RequestRows rq = request_rows(p, request_of(p.cu_q, d.n_requests, static_cast<int>(n)));
    own = visible(p, rq, static_cast<int>(n) - rq.q0);
  }
  const float inv = reciprocal_sum(p, l, own);
  uint16_t* out = p.out + n * d.out_token_stride + h * d.out_head_stride + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack16<BF16>(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---- rows that a masked value has spoiled (0 times a value that is not finite)

template <bool BF16>
__device__ __forceinline__ float widen16(uint16_t h) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(__ushort_as_half(h));
}

// A row that is not finite, of a request whose later keys it does not see: worked out
// again, by a warp, over the keys that it does see -- if one of the values that it
// does not see is indeed not finite.  A row that is not finite by what it sees stays so.
// Scalar work, for what should not be there: a NaN in the last value of a chunk makes
// 512 tokens over 1024 keys take 3.1 ms instead of 0.04, 4096 over 8192 24 ms instead of 0.43 (40 heads, D = 128).
// The log-sum-exp stays as the passes wrote it: it has no values in it.
template <int D, bool BF16>
__device__ void exact_row(const AttnParams& p, int request, const RequestRows& rq, int64_t token, int head) {
  const vqb_attention_desc& d = p.d;
  const int lane = threadIdx.x & 31, kvh = head / p.group;
  const int seen = visible(p, rq, static_cast<int>(token) - rq.q0);
  auto page_of = [&](bool own, int j) {
    const int page = own ? __ldg(p.table + static_cast<int64_t>(request) * d.table_width + (j >> p.page_shift))
                         : __ldg(p.prefix_pages + (j >> p.page_shift));
    return static_cast<unsigned>(page) < static_cast<unsigned>(d.num_pages) ? page : -1;
  };
  auto value = [&](int page, int j) {
    return p.vc + page * d.vc_page_stride + kvh * d.vc_head_stride + (j & (d.page_size - 1)) * d.vc_token_stride;
  };
  bool fault = false;
  for (int j0 = seen; j0 < rq.len && !fault; j0 += 32) {
    const int j = j0 + lane;
    bool bad = false;
    const int page = j < rq.len ? page_of(true, j) : -1;
    if (page >= 0) {
      const uint16_t* v = value(page, j);
      for (int e = 0; e < D; ++e) bad = bad || !(fabsf(widen16<BF16>(v[e])) < INFINITY);
    }
    fault = __any_sync(0xffffffffu, bad);
  }
  if (!fault) return;
  const uint16_t* q = p.q + token * d.q_token_stride + head * d.q_head_stride;
  float acc[D / 32];
  float m = -INFINITY, l = 0.0f;
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
  bool nan = false;  // NaN the row stays, whatever follows
  for (int part = 0; part < 2; ++part) {
    const int end = part ? seen : d.prefix_len;
    for (int j0 = 0; j0 < end && !nan; j0 += 32) {
      const int j = j0 + lane;
      const int page = j < end ? page_of(part != 0, j) : -1;
      float s = j < end ? 0.0f : -INFINITY;
      if (page >= 0) {
        const uint16_t* k = p.kc + page * d.kc_page_stride + kvh * d.kc_head_stride + (j & (d.page_size - 1)) * d.kc_token_stride;
        for (int e = 0; e < D; ++e) s = fmaf(widen16<BF16>(q[e]), widen16<BF16>(k[e]), s);
      }
      s *= p.scale_log2;
      float top = s;
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
      const float keep = exp2f(m - base), w = j < end ? exp2f(s - base) : 0.0f;
      m = mn;
      float sum = w;
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = l * keep + sum;
      bool all_nan = true;
      for (int e = 0; e < D / 32; ++e) acc[e] *= keep;
      for (int i = 0; i < 32; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const int pg = __shfl_sync(0xffffffffu, page, i);
        if (pg < 0) continue;
        const uint16_t* v = value(pg, j0 + i);
        for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wi, widen16<BF16>(v[lane + 32 * e]), acc[e]);
      }
      for (int e = 0; e < D / 32; ++e) all_nan = all_nan && acc[e] != acc[e];
      nan = l != l || __all_sync(0xffffffffu, all_nan);
    }
  }
  uint16_t* out = p.out + token * d.out_token_stride + head * d.out_head_stride;
  const float inv = reciprocal_sum(p, l, seen);
  for (int e = 0; e < D / 32; ++e) out[lane + 32 * e] = narrow16<BF16>(acc[e] * inv);
}

// After the passes of a call that masks keys: nothing, unless a pass noted a row
// that is not finite.  The last block to end takes the note away, since a captured call
// has one mark for all its replays; status[1], which counts the blocks, was cleared in an earlier launch.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attention_exact_kernel(AttnParams p) {
  pdl_wait();
  pdl_trigger();
  if (__ldcg(p.note) != p.mark) return;
  const vqb_attention_desc& d = p.d;
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(min(__ldg(p.cu_q + d.n_requests), d.n_tokens)) * d.heads;
  for (int64_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8) {
    const int64_t n = row / d.heads;
    const int h = static_cast<int>(row - n * d.heads);
    const uint16_t* out = p.out + n * d.out_token_stride + h * d.out_head_stride;
    bool bad = false;
    for (int e = lane; e < D; e += 32) bad = bad || !(fabsf(widen16<BF16>(out[e])) < INFINITY);
    if (!__any_sync(0xffffffffu, bad)) continue;
    const int r = request_of(p.cu_q, d.n_requests, static_cast<int>(n));
    exact_row<D, BF16>(p, r, request_rows(p, r), n, h);
  }
  __syncthreads();
  if (threadIdx.x == 0 && atomicAdd(p.status + 1, 1) == static_cast<int>(gridDim.x) - 1) {
    *p.note = 0;
    p.status[1] = 0;
  }
}

vqb_status launch_join(const AttnParams& p, const AttnPass& shared, int own_parts, bool bf, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((part_rows(p.d) + 7) / 8);
  cudaError_t ce;
  if (p.d.head_dim == 128)
    ce = bf ? launch_pdl(attention_join_kernel<128, true>, blocks, 256, 0, s, p, shared, own_parts)
            : launch_pdl(attention_join_kernel<128, false>, blocks, 256, 0, s, p, shared, own_parts);
  else
    ce = bf ? launch_pdl(attention_join_kernel<64, true>, blocks, 256, 0, s, p, shared, own_parts)
            : launch_pdl(attention_join_kernel<64, false>, blocks, 256, 0, s, p, shared, own_parts);
  if (ce != cudaSuccess) return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

vqb_status launch_exact(const AttnParams& p, bool bf, cudaStream_t s) {
  const size_t rows = (part_rows(p.d) + 7) / 8;
  const unsigned blocks = static_cast<unsigned>(rows < 296 ? rows : 296);
  cudaError_t ce;
  if (p.d.head_dim == 128)
    ce = bf ? launch_pdl(attention_exact_kernel<128, true>, blocks, 256, 0, s, p)
            : launch_pdl(attention_exact_kernel<128, false>, blocks, 256, 0, s, p);
  else
    ce = bf ? launch_pdl(attention_exact_kernel<64, true>, blocks, 256, 0, s, p)
            : launch_pdl(attention_exact_kernel<64, false>, blocks, 256, 0, s, p);
  if (ce != cudaSuccess) return VQB_CUDA_ERROR;
  note_launch();
  return VQB_OK;
}

// Everything about a call that does not need its pointers.
vqb_status check_desc(const vqb_attention_desc& d) {
  if (d.n_requests < 0 || d.n_tokens < 0 || d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads || d.max_q_len < 0 ||
      d.max_kv_len < 0 || d.prefix_len < 0 || d.num_pages < 1 || d.table_width < 0)
    return VQB_BAD_SHAPE;
  if (!(d.scale > 0.0f) || d.scale > 3.0e38f) return VQB_BAD_SHAPE;
  if (d.head_dim != 64 && d.head_dim != 128) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.page_size < 16 || d.page_size > 1024 || (d.page_size & (d.page_size - 1))) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.heads > 65535 || d.n_requests > 65535) return VQB_UNSUPPORTED_GEOMETRY;
  if (static_cast<int64_t>(d.n_tokens) * d.heads > 0x7fffffff) return VQB_UNSUPPORTED_GEOMETRY;
  if (static_cast<int64_t>(d.table_width) * d.page_size < d.max_kv_len) return VQB_BAD_SHAPE;
  if (static_cast<int64_t>(d.prefix_len) + d.max_kv_len > 0x7fff0000) return VQB_UNSUPPORTED_GEOMETRY;
  const int64_t strides[] = {d.q_token_stride, d.q_head_stride, d.out_token_stride, d.out_head_stride,
                             d.kc_page_stride, d.kc_head_stride, d.kc_token_stride,
                             d.vc_page_stride, d.vc_head_stride, d.vc_token_stride};
  for (int64_t s : strides) {
    if (s % 8) return VQB_BAD_ALIGNMENT;
    if (s < 0) return VQB_BAD_SHAPE;
  }
  return VQB_OK;
}

// SMs the plan counts on: the plan must not depend on the device that happens
// to be current, so that the workspace's size fits the call.
constexpr int kPlanSms = 148;

}  // namespace
}  // namespace vqb

using namespace vqb;

extern "C" size_t vqb_prefix_attention_workspace_size(const vqb_attention_desc* desc) {
  if (!desc || check_desc(*desc) != VQB_OK) return 0;
  const AttnPlan a = make_plan(*desc, kPlanSms);
  return kStatusBytes + ml_bytes(*desc, a.parts) + a.parts * part_rows(*desc) * desc->head_dim * sizeof(float);
}

extern "C" vqb_status vqb_prefix_attention(const vqb_attention_desc* desc, vqb_dtype dtype, const void* q,
                                           const void* k_cache, const void* v_cache, const int32_t* block_table,
                                           const int32_t* kv_lens, const int32_t* cu_q, const int32_t* prefix_pages,
                                           void* out, float* lse, void* workspace, size_t workspace_bytes,
                                           vqb_stream_t stream) {
  if (!desc) return VQB_NULL_POINTER;
  const vqb_attention_desc& d = *desc;
  vqb_status st = check_desc(d);
  if (st != VQB_OK) return st;
  if (dtype != VQB_F16 && dtype != VQB_BF16) return VQB_UNSUPPORTED_GEOMETRY;
  if (d.n_tokens == 0 || d.n_requests == 0) return VQB_OK;
  if (!q || !k_cache || !v_cache || !kv_lens || !cu_q || !out || !workspace) return VQB_NULL_POINTER;
  if ((d.max_kv_len > 0 && !block_table) || (d.prefix_len > 0 && !prefix_pages)) return VQB_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return VQB_BAD_ALIGNMENT;
  if (workspace_bytes < vqb_prefix_attention_workspace_size(desc)) return VQB_WORKSPACE_TOO_SMALL;
  const AttnPlan a = make_plan(d, kPlanSms);
  static std::atomic<uint32_t> calls{0};
  uint32_t mark = ++calls;
  if (mark == 0) mark = ++calls;
  const bool bf = dtype == VQB_BF16;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  AttnParams p{d, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache),
               static_cast<const uint16_t*>(v_cache), block_table, kv_lens, cu_q, prefix_pages,
               static_cast<uint16_t*>(out), lse, reinterpret_cast<float*>(ws + kStatusBytes + ml_bytes(d, a.parts)),
               reinterpret_cast<float2*>(ws + kStatusBytes), reinterpret_cast<int*>(ws) + 1, reinterpret_cast<uint32_t*>(ws) + 4, mark, d.heads / d.kv_heads,
               __builtin_ctz(d.page_size), d.scale * 1.4426950408889634f};
  timer_before(s);
  if (a.shared.splits > 0) {
    st = launch_attention_tiles(p, a.shared, bf, a.shared_tiles, s);
    if (st != VQB_OK) return st;
  }
  st = a.decode ? launch_attention_decode(p, a.own, a.shared, bf, s) : launch_attention_tiles(p, a.own, bf, a.own_tiles, s);
  if (st != VQB_OK) return st;
  if (a.join) st = launch_join(p, a.shared, a.own.splits, bf, s);
  if (st == VQB_OK && d.causal && d.max_q_len > 1) st = launch_exact(p, bf, s);
  timer_after(s);
  return st;
}

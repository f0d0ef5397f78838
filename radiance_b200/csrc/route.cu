// Mixture-of-experts routing around the grouped expert GEMMs: top-k of the router's logits with
// per-expert counts, the row plan of the expert-sorted layout and the balance loss; the gradient of
// the logits; and the moves of token rows to their experts' rows and back, with their gradients.
//
// radiance routes with softmax and topk and gathers and scatters rows with index ops (MoEFeedForward,
// src/radiance/model/ffn.py:156-436).  Here one pass over the logits does the selection and the
// statistics, and every row is moved by one kernel each way.  All of it is bound by memory traffic
// (or, for few tokens, by launches); nothing uses floating-point atomics, so results repeat bit for bit.
#include <type_traits>

#include "common.cuh"
#include "../../include/radiance_nvfp4.h"

namespace rb {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxExperts = 256;   // the grouped GEMM's group limit
constexpr int kMaxTopK = 32;       // one lane keeps one pick
constexpr int kMaxPairs = 4096;    // (token, pick) pairs of one block, held in shared memory
constexpr int kGroupAlign = 128;   // every expert's rows end at a multiple of the GEMM's tile height

struct RouteArgs {
  const void* logits;   // tokens x experts, row stride ld
  int64_t tokens, ld;
  int experts, k;
  const float* bias;    // added to the logits for the selection only, or nullptr
  const uint8_t* valid; // tokens to route, or nullptr for all
  int renormalize;
  float* weights;       // tokens x k
  int32_t* picks;       // tokens x k, -1: none
  int32_t* rows;        // tokens x k
  int64_t* counts;      // experts
  int64_t* plan_counts; // the same again, or nullptr
  int64_t* offsets;     // experts + 1
  float* loss;
  float* share;         // experts: d loss / d (an expert's probability), of any routed token
  int64_t chunk;        // tokens per block
  int64_t blocks;
  // scratch, per block: pairs of each expert, sums of each expert's probability, routed tokens
  uint16_t* hist;       // blocks x experts (a block has at most kMaxPairs pairs)
  float* psum;          // blocks x experts
  int32_t* nrouted;     // blocks
};

template <typename T>
__device__ __forceinline__ float logit(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}

// Order-preserving unsigned key of a score: NaN above everything (as torch sorts it), -0 equal to +0,
// and 0 for -inf, which is never selected.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return 0xFFFFFFFFu;
  if (s == -INFINITY) return 0u;
  const uint32_t b = __float_as_uint(s + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <int LPT>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <int LPT>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Exclusive scan over the block's kRouteThreads values; `sm` holds kRouteWarps ints.
__device__ __forceinline__ int64_t block_exclusive_scan(int64_t v, int64_t* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sm[warp] = incl;
  __syncthreads();
  int64_t before = 0;
  for (int w = 0; w < warp; ++w) before += sm[w];
  return before + incl - v;
}

struct PlanSmem {
  int32_t tot[kRouteThreads], pre[kRouteThreads];
  float ps[kRouteThreads];
  int64_t base[kMaxExperts];
  int64_t warp_sum[kRouteWarps];
  double red[kRouteWarps];
  int32_t n[kRouteWarps];
};

// The second half of routing, by one block: the totals of every expert over all blocks' counts,
// then the final rows of the pairs of chunks [c0, c1); with `summary`, also counts, offsets and loss.
// As many threads as fit share an expert: thread s * experts + e adds the counts of blocks s, s + ns, ...,
// kAhead loads in flight, since nothing but their latency costs time here (one after the other: 14 us for 129
// blocks' counts of 160 experts).
__device__ __forceinline__ void plan_block(const RouteArgs& a, int64_t c0, int64_t c1, bool summary, PlanSmem& sm) {
  constexpr int kAhead = 16;
  const int ns = kRouteThreads / a.experts, s = (int)threadIdx.x / a.experts;
  const int e = (int)threadIdx.x - s * a.experts;
  int32_t tot = 0, pre = 0;
  float ps = 0.0f;
  if (s < ns) {
    // From chunk c0 on and round to it: started at chunk 0 by every block, they all ask for the same lines at
    // the same time.
    for (int64_t i0 = s; i0 < a.blocks; i0 += kAhead * ns) {
      int32_t h[kAhead];
      float p[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t i = i0 + u * ns, b = i + c0 < a.blocks ? i + c0 : i + c0 - a.blocks;
        h[u] = i < a.blocks ? (int32_t)__ldcg(a.hist + b * a.experts + e) : 0;
        p[u] = summary && i < a.blocks ? __ldcg(a.psum + b * a.experts + e) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        tot += h[u];
        if (i0 + u * ns + c0 >= a.blocks) pre += h[u];
        ps += p[u];
      }
    }
  }
  sm.tot[threadIdx.x] = tot;
  sm.pre[threadIdx.x] = pre;
  sm.ps[threadIdx.x] = ps;
  __syncthreads();
  const int x = threadIdx.x;
  int64_t total = 0, prefix = 0;
  double p = 0.0;
  if (x < a.experts) {
    for (int i = 0; i < ns; ++i) {
      total += sm.tot[i * a.experts + x];
      prefix += sm.pre[i * a.experts + x];  // 0 in a summary, which starts at chunk 0
      p += sm.ps[i * a.experts + x];
    }
  }
  const int64_t padded = (total + kGroupAlign - 1) / kGroupAlign * kGroupAlign;
  const int64_t offset = block_exclusive_scan(padded, sm.warp_sum);
  if (x < a.experts) sm.base[x] = offset + prefix;
  if (summary) {
    if (x < a.experts) {
      a.counts[x] = total;
      if (a.plan_counts != nullptr) a.plan_counts[x] = total;
      a.offsets[x] = offset;
      if (x == a.experts - 1) a.offsets[a.experts] = offset + padded;
    }
    // loss = sum_e share_e (sum of p_e), share_e = E (count_e / sum of counts) / n
    int32_t n = 0;
    for (int64_t b = x; b < a.blocks; b += kRouteThreads) n += __ldcg(a.nrouted + b);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    double fp = x < a.experts ? (double)total * p : 0.0, pairs = x < a.experts ? (double)total : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      fp += __shfl_xor_sync(0xFFFFFFFFu, fp, o);
      pairs += __shfl_xor_sync(0xFFFFFFFFu, pairs, o);
    }
    __shared__ double sfp[kRouteWarps];
    if ((x & 31) == 0) {
      sm.red[x >> 5] = pairs;
      sfp[x >> 5] = fp;
      sm.n[x >> 5] = n;
    }
    __syncthreads();
    if (x == 0) {
      for (int w = 1; w < kRouteWarps; ++w) {
        fp += sfp[w];
        pairs += sm.red[w];
        n += sm.n[w];
      }
      sm.red[0] = n > 0 ? (double)a.experts / (pairs * (double)n) : 0.0;
      *a.loss = (float)(sm.red[0] * fp);
    }
    __syncthreads();
    if (x < a.experts) a.share[x] = (float)(sm.red[0] * (double)total);
  }
  __syncthreads();
  for (int64_t ch = c0; ch < c1; ++ch) {
    const int64_t i0 = ch * a.chunk * a.k, i1 = min(a.tokens, (ch + 1) * a.chunk) * a.k;
    for (int64_t i = i0 + x; i < i1; i += 4 * kRouteThreads) {
      int32_t pick[4], rank[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t at = i + u * kRouteThreads;
        pick[u] = at < i1 ? __ldcg(a.picks + at) : -1;
        rank[u] = at < i1 ? __ldcg(a.rows + at) : 0;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t at = i + u * kRouteThreads;
        if (at < i1) a.rows[at] = pick[u] < 0 ? -1 : (int32_t)(sm.base[pick[u]] + rank[u]);
      }
    }
    if (ch + 1 < c1) {
      __syncthreads();
      if (x < a.experts) sm.base[x] += __ldcg(a.hist + ch * a.experts + x);
      __syncthreads();
    }
  }
}

// The best of a group's (key, expert) candidates: the largest key, ties to the lower expert.
template <int LPT>
__device__ __forceinline__ void group_best(uint32_t& key, int& expert) {
  if constexpr (LPT == 32) {  // whole warps have reductions in hardware
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, key);
    expert = (int)__reduce_min_sync(0xFFFFFFFFu, key == m ? (uint32_t)expert : 0x7FFFFFFFu);
    key = m;
  } else {
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
      const uint32_t ok = __shfl_xor_sync(0xFFFFFFFFu, key, o);
      const int oe = __shfl_xor_sync(0xFFFFFFFFu, expert, o);
      if (ok > key || (ok == key && oe < expert)) key = ok, expert = oe;
    }
  }
}

// One block takes `chunk` consecutive tokens.  LPT lanes hold one token's logits, ITEMS experts to a
// lane (expert e sits in lane e % LPT), so a warp works on 32 / LPT tokens and its loads of a row are
// contiguous.  First the tokens: softmax, the k picks one maximum at a time (a lane looks through its own
// experts again only when one of them was picked), weights, and each lane's sums of its experts' probabilities.
// Then the pairs, from shared memory: each warp ranks a run of them among the pairs of the same expert
// (match_any gives the lanes with the same pick), the warps' counts are scanned, and the block's ranks and
// counts go out for plan_block.
// What this costs is latency, a launch's and a block's: the tokens are spread over one block per SM, and a
// block of sixteen warps goes through its share in a step or two.  With plan_block, 16384 x 8, k = 2: 10.7 us;
// 4099 x 160, k = 6: 18.7 us (eight warps, five shuffles for each of two values a pick: 12.5 and 35 us).
template <typename T, int LPT, int ITEMS>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteArgs a) {
  constexpr int kGroups = kRouteThreads / LPT;
  __shared__ int16_t pair[kMaxPairs];
  __shared__ uint16_t rank[kMaxPairs];
  __shared__ union {
    float p[kRouteWarps][kMaxExperts];    // sums of probabilities, then
    int32_t n[kRouteWarps][kMaxExperts];  // counts of pairs
  } per_warp;
  __shared__ int32_t wn[kRouteWarps];
  __shared__ PlanSmem plan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane & (LPT - 1), gid = threadIdx.x / LPT;
  const int64_t t0 = (int64_t)blockIdx.x * a.chunk, t1 = min(a.tokens, t0 + a.chunk);
  float acc[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) acc[i] = 0.0f;
  int nrouted = 0;
  for (int64_t tb = t0; tb < t1; tb += kGroups) {
    const int64_t t = tb + gid;
    const bool live = t < t1 && (a.valid == nullptr || a.valid[t] != 0);
    float x[ITEMS];
    uint32_t key[ITEMS];
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = i * LPT + gl;
      const bool in = live && e < a.experts;
      x[i] = in ? logit<T>(a.logits, t * a.ld + e) : -INFINITY;
      key[i] = in ? score_key(a.bias != nullptr ? x[i] + a.bias[e] : x[i]) : 0u;
      m = fmaxf(m, x[i]);
      nan |= x[i] != x[i];
    }
    m = group_max<LPT>(m);
    const float top = m;
    if (nan) m = NAN;  // this lane's exponentials become NaN, and with them the sum
    float z = 0.0f, p[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      p[i] = expf(x[i] - m);
      if (i * LPT + gl >= a.experts) p[i] = 0.0f;  // not an expert (its -inf against m = -inf is no zero)
      z += p[i];
    }
    z = group_sum<LPT>(z);
    uint32_t lane_key = 0;  // the best of this lane's experts that are left
    int lane_best = 0x7FFFFFFF;
    const auto look = [&]() {
      lane_key = 0;
      lane_best = 0x7FFFFFFF;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (key[i] > lane_key) lane_key = key[i], lane_best = i * LPT + gl;
    };
    look();
    int mine = -1;  // lane j of the group keeps pick j
    for (int j = 0; j < a.k; ++j) {
      uint32_t bk = lane_key;
      int be = lane_best;
      group_best<LPT>(bk, be);
      if (bk == 0) be = -1;  // nothing selectable is left (the loop goes on: other groups of the warp need it)
      if (gl == j) mine = be;
      if (be == lane_best) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (be == i * LPT + gl) key[i] = 0;
        look();
      }
    }
    const bool routed = __shfl_sync(0xFFFFFFFFu, mine, lane & ~(LPT - 1)) >= 0;
    if (routed) {
      const float rz = 1.0f / z;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) acc[i] += p[i] * rz;
      nrouted += gl == 0;
    }
    // The weights: p of the picks, or their softmax among themselves.
    const float xs = mine >= 0 ? logit<T>(a.logits, t * a.ld + mine) : -INFINITY;
    float w;
    if (a.renormalize) {
      const float ms = group_max<LPT>(xs);
      w = mine >= 0 ? expf(xs - ms) : 0.0f;
      const float sum = group_sum<LPT>(w);
      w = mine >= 0 ? w / sum : 0.0f;
    } else {
      w = mine >= 0 ? expf(xs - top) / z : 0.0f;
    }
    if (t < t1 && gl < a.k) {
      a.weights[t * a.k + gl] = w;
      a.picks[t * a.k + gl] = mine;
      pair[(t - t0) * a.k + gl] = (int16_t)mine;
    }
  }
  // Sums of probabilities: lanes holding the same experts, then the warps, in order.
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
    for (int o = 16; o >= LPT; o >>= 1) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], o);
    if (lane < LPT && i * LPT + gl < kMaxExperts) per_warp.p[warp][i * LPT + gl] = acc[i];
  }
  nrouted = __reduce_add_sync(0xFFFFFFFFu, nrouted);
  if (lane == 0) wn[warp] = nrouted;
  __syncthreads();
  if ((int)threadIdx.x < a.experts) {
    float ps = 0.0f;
    for (int w = 0; w < kRouteWarps; ++w) ps += per_warp.p[w][threadIdx.x];
    a.psum[(int64_t)blockIdx.x * a.experts + threadIdx.x] = ps;
  }
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < kRouteWarps; ++w) n += wn[w];
    a.nrouted[blockIdx.x] = n;
  }
  __syncthreads();
  // Ranks within this warp's run of pairs.
  for (int i = lane; i < a.experts; i += 32) per_warp.n[warp][i] = 0;
  __syncwarp();
  const int pairs = t1 > t0 ? (int)((t1 - t0) * a.k) : 0;
  const int run = ((pairs + kRouteWarps - 1) / kRouteWarps + 31) & ~31;
  const int p0 = warp * run, p1 = min(pairs, p0 + run);
  for (int i0 = p0; i0 < p1; i0 += 32) {
    const int i = i0 + lane;
    const int e = i < p1 ? (int)pair[i] : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    int before = 0;
    if (e >= 0) before = per_warp.n[warp][e];
    __syncwarp();
    if (e >= 0) {
      rank[i] = (uint16_t)(before + __popc(same & ((1u << lane) - 1u)));
      if ((same >> lane) == 1u) per_warp.n[warp][e] = before + __popc(same);  // the last lane of its kind
    }
    __syncwarp();
  }
  __syncthreads();
  if ((int)threadIdx.x < a.experts) {
    const int e = threadIdx.x;
    int sum = 0;
    for (int w = 0; w < kRouteWarps; ++w) {
      const int h = per_warp.n[w][e];
      per_warp.n[w][e] = sum;  // pairs of this expert in earlier warps
      sum += h;
    }
    a.hist[(int64_t)blockIdx.x * a.experts + e] = (uint16_t)sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += kRouteThreads) {
    const int e = pair[i];
    a.rows[t0 * a.k + i] = e >= 0 ? per_warp.n[i / run][e] + rank[i] : 0;
  }
  if (gridDim.x == 1) {  // few tokens: this block finishes the plan itself
    __syncthreads();
    plan_block(a, 0, 1, true, plan);
  }
}

// The rows of all pairs: block b of gridDim.x - 1 finishes its share of the chunks, the last block
// writes counts, offsets and loss.
__global__ void __launch_bounds__(kRouteThreads) route_plan_kernel(const RouteArgs a) {
  __shared__ PlanSmem plan;
  const int64_t workers = gridDim.x - 1;
  if (blockIdx.x == workers) {
    plan_block(a, 0, 0, true, plan);
    return;
  }
  const int64_t per = (a.blocks + workers - 1) / workers;
  const int64_t c0 = min(a.blocks, per * blockIdx.x), c1 = min(a.blocks, c0 + per);
  plan_block(a, c0, c1, false, plan);
}

// ---------------------------------------------------------------------------------------------
// Gradient of the logits
// ---------------------------------------------------------------------------------------------
struct RouteBwdArgs {
  const void* logits;
  int64_t tokens, ld;
  int experts, k;
  int renormalize;
  const float* weights;
  const int32_t* picks;
  const float* share;      // experts
  const float* grad_w;     // tokens x k, or nullptr
  const float* grad_loss;  // scalar, or nullptr
  void* grad;              // tokens x experts, row stride ldo
  int64_t ldo;
};

// dl = p (c - <p, c>) + the picks' part, c_e = grad_loss share_e.  The probabilities are computed
// again from the logits instead of being stored by the forward pass.
template <typename T, int LPT, int ITEMS>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const RouteBwdArgs a) {
  constexpr int kGroups = kRouteThreads / LPT;
  const int lane = threadIdx.x & 31;
  const int gl = lane & (LPT - 1), gid = threadIdx.x / LPT;
  const float g = a.grad_loss != nullptr ? *a.grad_loss : 0.0f;
  float c[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int e = i * LPT + gl;
    c[i] = e < a.experts && g != 0.0f ? g * a.share[e] : 0.0f;
  }
  for (int64_t tb = (int64_t)blockIdx.x * kGroups; tb < a.tokens; tb += (int64_t)gridDim.x * kGroups) {
    const int64_t t = tb + gid;
    const bool in_t = t < a.tokens;
    int pick = -1;
    float w = 0.0f, gw = 0.0f;
    if (in_t && gl < a.k) {
      pick = a.picks[t * a.k + gl];
      if (pick >= a.experts) pick = -1;
      if (pick >= 0) {
        w = a.weights[t * a.k + gl];
        if (a.grad_w != nullptr) gw = a.grad_w[t * a.k + gl];
      }
    }
    const bool routed = __shfl_sync(0xFFFFFFFFu, pick, lane & ~(LPT - 1)) >= 0;
    float x[ITEMS], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = i * LPT + gl;
      x[i] = routed && e < a.experts ? logit<T>(a.logits, t * a.ld + e) : -INFINITY;
      m = fmaxf(m, x[i]);
    }
    m = group_max<LPT>(m);
    float z = 0.0f, p[ITEMS], pc = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      p[i] = i * LPT + gl < a.experts ? expf(x[i] - m) : 0.0f;
      z += p[i];
    }
    z = group_sum<LPT>(z);
    const float rz = 1.0f / z;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      p[i] *= rz;
      pc += p[i] * c[i];
    }
    pc = group_sum<LPT>(pc);
    const float wg = w * gw, wsum = group_sum<LPT>(wg);
    const float part = a.renormalize ? wg - w * wsum : wg;  // of this lane's pick
    float d[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) d[i] = p[i] * (c[i] - pc - (a.renormalize ? 0.0f : wsum));
    for (int j = 0; j < a.k; ++j) {
      const int pe = __shfl_sync(0xFFFFFFFFu, pick, (lane & ~(LPT - 1)) + j);
      const float pv = __shfl_sync(0xFFFFFFFFu, part, (lane & ~(LPT - 1)) + j);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (pe == i * LPT + gl) d[i] += pv;
    }
    if (in_t) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int e = i * LPT + gl;
        if (e >= a.experts) continue;
        const float v = routed ? d[i] : 0.0f;
        if constexpr (sizeof(T) == 2)
          reinterpret_cast<__nv_bfloat16*>(a.grad)[t * a.ldo + e] = __float2bfloat16_rn(v);
        else reinterpret_cast<float*>(a.grad)[t * a.ldo + e] = v;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Rows to the experts and back
// ---------------------------------------------------------------------------------------------
struct RowsArgs {
  const void* src;       // dispatch: tokens x d;  combine, combine backward: num_rows x d (expert rows)
  int64_t ld_src;
  const void* extra;     // combine: residual or nullptr;  combine backward: grad_y (tokens x d)
  int64_t ld_extra;
  const int32_t* rows;   // tokens x k
  const float* weights;  // tokens x k, or nullptr for ones
  void* out;             // dispatch, combine backward: num_rows x d;  combine: tokens x d
  int64_t ld_out;
  float* grad_w;         // combine backward: tokens x k
  int64_t tokens, d, num_rows;
  int k;
  int cx;                // threads to a token (a power of two, 32 .. 256)
  // dispatch and combine backward: the rows that no pair fills become zero
  const int64_t* counts;
  const int64_t* offsets;
  int experts, pad_slices;
};

// kVec elements of T as one load: 16 bytes, or one element where rows are not 16-byte aligned.  get and set
// turn them into fp32 and back (rounded).
template <typename T, int kVec>
struct Pack;
template <>
struct Pack<__nv_bfloat16, 8> {
  uint4 q;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Pack<float, 4> {
  uint4 q;
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(q.x), f[1] = __uint_as_float(q.y), f[2] = __uint_as_float(q.z), f[3] = __uint_as_float(q.w);
  }
  __device__ __forceinline__ void set(const float (&f)[4]) {
    q = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Pack<__nv_bfloat16, 1> {
  __nv_bfloat16 q;
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = __bfloat162float(q); }
  __device__ __forceinline__ void set(const float (&f)[1]) { q = __float2bfloat16_rn(f[0]); }
};
template <>
struct Pack<float, 1> {
  float q;
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = q; }
  __device__ __forceinline__ void set(const float (&f)[1]) { q = f[0]; }
};
template <typename T, int kVec>
__device__ __forceinline__ Pack<T, kVec> load_pack(const T* p) {
  Pack<T, kVec> r;
  if constexpr (kVec > 1) r.q = __ldg(reinterpret_cast<const uint4*>(p));
  else r.q = *p;
  return r;
}
template <typename T, int kVec>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, kVec>& r) {
  if constexpr (kVec > 1) *reinterpret_cast<uint4*>(p) = r.q;
  else *p = r.q;
}

// Up to kP pairs of a token: their rows (-1 without one; a row outside the layout is never touched) and weights.
template <int kP>
struct Pairs {
  int32_t row[kP];
  float w[kP];
};
template <int kP>
__device__ __forceinline__ Pairs<kP> load_pairs(const RowsArgs& a, int64_t t, int j0) {
  Pairs<kP> p;
#pragma unroll
  for (int u = 0; u < kP; ++u) {
    const bool in = t < a.tokens && j0 + u < a.k;
    const int32_t r = in ? __ldg(a.rows + t * a.k + j0 + u) : -1;
    p.row[u] = r < a.num_rows ? r : -1;
    p.w[u] = in && a.weights != nullptr ? __ldg(a.weights + t * a.k + j0 + u) : 1.0f;
  }
  return p;
}

// Zeroes the rows that hold no pair: the end of every expert's group and the rows past the last group.  Each
// is one run of consecutive rows.  A group's run is cut into `pad_slices` pieces, and the pieces of all
// groups are dealt to the blocks; the last run is dealt to all blocks row by row.
template <typename T, int kVec>
__device__ __forceinline__ void zero_unused_rows(const RowsArgs& a) {
  const int ty = (int)threadIdx.x / a.cx, ny = 256 / a.cx, x = (int)threadIdx.x % a.cx;
  T* out = reinterpret_cast<T*>(a.out);
  const float none[kVec] = {};
  Pack<T, kVec> zero;
  zero.set(none);
  const auto clear = [&](int64_t r0, int64_t r1, int64_t first, int64_t step) {
    r0 = max(r0, (int64_t)0);
    r1 = min(r1, a.num_rows);
    for (int64_t r = r0 + first; r < r1; r += step)
      for (int64_t c = (int64_t)x * kVec; c < a.d; c += (int64_t)a.cx * kVec)
        store_pack<T, kVec>(out + r * a.ld_out + c, zero);
  };
  for (int b = blockIdx.x; b < a.experts * a.pad_slices; b += gridDim.x) {
    const int e = b / a.pad_slices, slice = b % a.pad_slices;
    clear(a.offsets[e] + a.counts[e], a.offsets[e + 1], (int64_t)slice * ny + ty, (int64_t)a.pad_slices * ny);
  }
  clear(a.offsets[a.experts], a.num_rows, (int64_t)blockIdx.x * ny + ty, (int64_t)gridDim.x * ny);
}

// The three moves below share a shape: cx threads take a token (a warp when there are tokens for every
// resident warp, more for a few tokens), every thread kCols vectors of its row and kP of its pairs at a time, and
// the tokens are dealt to as many blocks as are resident.  A token's rows and weights are loaded while the
// token before it is moved, and a warp reads long pieces of a row (2 KB) with many loads in flight, two
// blocks to an SM: 16384 tokens x 2048, k = 2 with a residual, combine in 47 us (268 MB, 5.7 TB/s).  One
// vector a thread at higher occupancy, each token waiting for its rows and only then for its data: 96 us;
// four vectors but three blocks, with registers spilled: 75 us.
constexpr int kRowsBlocksPerSm = 2;
constexpr int kRowsCols2 = 4;  // vectors at a time for up to two pairs
constexpr int kRowsCols4 = 2;  // and for four pairs at a time

// x[t] to the row of each of its pairs: a token's row is read once and written k times.
template <typename T, int kVec, int kP, int kCols>
__global__ void __launch_bounds__(256, kRowsBlocksPerSm) token_dispatch_kernel(const RowsArgs a) {
  zero_unused_rows<T, kVec>(a);
  const int cx = a.cx, ny = 256 / cx, x = (int)threadIdx.x % cx;
  const int64_t step = (int64_t)gridDim.x * ny, wide = (int64_t)cx * kVec;
  T* out = reinterpret_cast<T*>(a.out);
  int64_t t = (int64_t)blockIdx.x * ny + (int)threadIdx.x / cx;
  Pairs<kP> next = load_pairs<kP>(a, t, 0);
  for (; t < a.tokens; t += step) {
    const Pairs<kP> first = next;
    next = load_pairs<kP>(a, t + step, 0);
    const T* src = reinterpret_cast<const T*>(a.src) + t * a.ld_src;
    for (int64_t c = (int64_t)x * kVec; c < a.d; c += kCols * wide) {
      Pack<T, kVec> v[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (c + i * wide < a.d) v[i] = load_pack<T, kVec>(src + c + i * wide);
      for (int j0 = 0; j0 < a.k; j0 += kP) {
        const Pairs<kP> p = j0 == 0 ? first : load_pairs<kP>(a, t, j0);
#pragma unroll
        for (int u = 0; u < kP; ++u)
          if (p.row[u] >= 0) {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
              if (c + i * wide < a.d) store_pack<T, kVec>(out + p.row[u] * a.ld_out + c + i * wide, v[i]);
          }
      }
    }
  }
}

// y[t] = residual[t] + sum_j w[t, j] rows[row(t, j)], in fp32 and in the order of j, rounded once.
// Without weights it is the dispatch's backward.
template <typename T, int kVec, int kP, int kCols>
__global__ void __launch_bounds__(256, kRowsBlocksPerSm) token_combine_kernel(const RowsArgs a) {
  const int cx = a.cx, ny = 256 / cx, x = (int)threadIdx.x % cx;
  const int64_t step = (int64_t)gridDim.x * ny, wide = (int64_t)cx * kVec;
  const T* src = reinterpret_cast<const T*>(a.src);
  int64_t t = (int64_t)blockIdx.x * ny + (int)threadIdx.x / cx;
  Pairs<kP> next = load_pairs<kP>(a, t, 0);
  for (; t < a.tokens; t += step) {
    const Pairs<kP> first = next;
    next = load_pairs<kP>(a, t + step, 0);
    const T* res = a.extra != nullptr ? reinterpret_cast<const T*>(a.extra) + t * a.ld_extra : nullptr;
    T* out = reinterpret_cast<T*>(a.out) + t * a.ld_out;
    for (int64_t c = (int64_t)x * kVec; c < a.d; c += kCols * wide) {
      float acc[kCols][kVec];
      Pack<T, kVec> rv[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        if (res != nullptr && c + i * wide < a.d) rv[i] = load_pack<T, kVec>(res + c + i * wide);
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[i][e] = 0.0f;
      }
      for (int j0 = 0; j0 < a.k; j0 += kP) {
        const Pairs<kP> p = j0 == 0 ? first : load_pairs<kP>(a, t, j0);
        Pack<T, kVec> v[kP][kCols];
#pragma unroll
        for (int u = 0; u < kP; ++u)
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            if (p.row[u] >= 0 && c + i * wide < a.d)
              v[u][i] = load_pack<T, kVec>(src + p.row[u] * a.ld_src + c + i * wide);
#pragma unroll
        for (int u = 0; u < kP; ++u) {
          if (p.row[u] < 0) continue;
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            float f[kVec];
            v[u][i].get(f);
#pragma unroll
            for (int e = 0; e < kVec; ++e) acc[i][e] = fmaf(p.w[u], f[e], acc[i][e]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        if (c + i * wide >= a.d) continue;
        if (res != nullptr) {
          float f[kVec];
          rv[i].get(f);
#pragma unroll
          for (int e = 0; e < kVec; ++e) acc[i][e] += f[e];
        }
        Pack<T, kVec> o;
        o.set(acc[i]);
        store_pack<T, kVec>(out + c + i * wide, o);
      }
    }
  }
}

// grad_rows[row(t, j)] = w[t, j] grad_y[t] and grad_w[t, j] = <grad_y[t], rows[row(t, j)]>.  grad_y's
// row is read once for kP pairs; each pair's product is summed over its cx threads in a fixed order.
template <typename T, int kVec, int kP, int kCols>
__global__ void __launch_bounds__(256, kRowsBlocksPerSm) token_combine_backward_kernel(const RowsArgs a) {
  __shared__ float red[2][8][kP];
  zero_unused_rows<T, kVec>(a);
  const int cx = a.cx, ny = 256 / cx, x = (int)threadIdx.x % cx, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * ny, wide = (int64_t)cx * kVec;
  const T* src = reinterpret_cast<const T*>(a.src);
  T* out = reinterpret_cast<T*>(a.out);
  int buf = 0;
  int64_t t = (int64_t)blockIdx.x * ny + (int)threadIdx.x / cx;
  Pairs<kP> next = load_pairs<kP>(a, t, 0);
  // Every thread of the block makes the same number of turns: they meet at the barrier below.
  for (int64_t tb = (int64_t)blockIdx.x * ny; tb < a.tokens; tb += step, t += step) {
    const Pairs<kP> first = next;
    next = load_pairs<kP>(a, t + step, 0);
    const bool in_t = t < a.tokens;
    const T* gy = reinterpret_cast<const T*>(a.extra) + (in_t ? t : 0) * a.ld_extra;
    for (int j0 = 0; j0 < a.k; j0 += kP) {
      const Pairs<kP> p = j0 == 0 ? first : load_pairs<kP>(a, t, j0);
      float dot[kP] = {};
      if (in_t) {
        for (int64_t c = (int64_t)x * kVec; c < a.d; c += kCols * wide) {
          Pack<T, kVec> g[kCols], v[kP][kCols];
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            if (c + i * wide >= a.d) continue;
            g[i] = load_pack<T, kVec>(gy + c + i * wide);
#pragma unroll
            for (int u = 0; u < kP; ++u)
              if (p.row[u] >= 0) v[u][i] = load_pack<T, kVec>(src + p.row[u] * a.ld_src + c + i * wide);
          }
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            if (c + i * wide >= a.d) continue;
            float gf[kVec];
            g[i].get(gf);
#pragma unroll
            for (int u = 0; u < kP; ++u) {
              if (p.row[u] < 0) continue;
              float f[kVec];
              v[u][i].get(f);
#pragma unroll
              for (int e = 0; e < kVec; ++e) {
                dot[u] = fmaf(gf[e], f[e], dot[u]);
                f[e] = p.w[u] * gf[e];
              }
              Pack<T, kVec> o;
              o.set(f);
              store_pack<T, kVec>(out + p.row[u] * a.ld_out + c + i * wide, o);
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kP; ++u) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[u] += __shfl_xor_sync(0xFFFFFFFFu, dot[u], o);
      }
      if (cx == 32) {  // a warp to a token
        float s = dot[0];
#pragma unroll
        for (int u = 1; u < kP; ++u)
          if (lane == u) s = dot[u];
        if (in_t && lane < kP && j0 + lane < a.k) a.grad_w[t * a.k + j0 + lane] = s;
        continue;
      }
      // The token's warps are consecutive, the first holding x = 0 .. 31.  Two buffers, one barrier a turn: a
      // buffer is written again only after the barrier that follows its reads.
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < kP; ++u) red[buf][warp][u] = dot[u];
      }
      __syncthreads();
      if (in_t && x < kP && j0 + x < a.k) {
        float s = red[buf][warp][x];
        for (int i = 1; i < cx / 32; ++i) s += red[buf][warp + i][x];
        a.grad_w[t * a.k + j0 + x] = s;
      }
      buf ^= 1;
    }
  }
}

}  // namespace rb

namespace {

int route_failed(int code, const char* fmt, const char* what, long long x = 0, long long y = 0) {
  rb_host::set_error(fmt, what, x, y);
  return code;
}

bool route_device(const char* what) { return rb_host::sm100(rb_host::current_device(), what); }

int route_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return RB_OK;
  rb_host::set_error("%s launch failed: %s", what, cudaGetErrorString(e));
  return RB_ERR_CUDA;
}

bool unaligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// Lanes per token: the power of two that holds the experts, a warp at most.
int route_lanes(int experts) {
  int l = 1;
  while (l < experts && l < 32) l <<= 1;
  return l;
}

// Tokens per block: the same for every SM, in whole steps of the block's token groups, and no more pairs than
// its shared memory holds.
int64_t route_chunk(int64_t tokens, int experts, int k, int64_t sms) {
  const int groups = rb::kRouteThreads / route_lanes(experts);
  const int64_t most = rb::kMaxPairs / k;
  const int64_t turns = (tokens + sms * most - 1) / (sms * most);  // blocks per SM
  int64_t c = turns > 0 ? (tokens + sms * turns - 1) / (sms * turns) : 1;
  c = (c + groups - 1) / groups * groups;
  if (c > most) c = most;
  return c < 1 ? 1 : c;
}

size_t route_scratch(int64_t blocks, int64_t experts) { return (size_t)(blocks * (6 * experts + 4)); }

// f(LPT, ITEMS) as integral constants for the number of experts.
template <typename F>
void route_shape(int experts, F&& f) {
  using std::integral_constant;
  const int l = route_lanes(experts);
  if (l == 1) f(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (l == 2) f(integral_constant<int, 2>(), integral_constant<int, 1>());
  else if (l == 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (l == 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (l == 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (experts <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (experts <= 64) f(integral_constant<int, 32>(), integral_constant<int, 2>());
  else if (experts <= 96) f(integral_constant<int, 32>(), integral_constant<int, 3>());
  else if (experts <= 128) f(integral_constant<int, 32>(), integral_constant<int, 4>());
  else if (experts <= 192) f(integral_constant<int, 32>(), integral_constant<int, 6>());
  else f(integral_constant<int, 32>(), integral_constant<int, 8>());
}

int check_route(const char* what, int dtype, int64_t tokens, int64_t experts, int64_t ld, int k) {
  if (dtype != RB_DTYPE_BF16 && dtype != RB_DTYPE_F32)
    return route_failed(RB_ERR_ARG, "%s: unsupported logits dtype %lld", what, dtype);
  if (experts < 1 || experts > rb::kMaxExperts || k < 1 || k > experts || k > rb::kMaxTopK)
    return route_failed(RB_ERR_SHAPE, "%s needs 1 <= experts <= 256 and 1 <= k <= min(experts, 32), got experts=%lld k=%lld",
                        what, experts, k);
  if (tokens < 0 || ld < experts || tokens * k + experts * 128 > 0x7FFFFFFF)
    return route_failed(RB_ERR_SHAPE, "%s: %lld tokens (row stride %lld) are out of range", what, tokens, ld);
  return RB_OK;
}

// Checks and the launch shape of the three row kernels.  Returns the elements per load, or 0 on an error.
int rows_shape(const char* what, rb::RowsArgs& a, int dtype, bool pads, int* rc) {
  if (dtype != RB_DTYPE_BF16 && dtype != RB_DTYPE_F32) {
    *rc = route_failed(RB_ERR_ARG, "%s: unsupported dtype %lld", what, dtype);
    return 0;
  }
  if (a.tokens < 0 || a.d < 1 || a.k < 1 || a.num_rows < 0 || a.num_rows > 0x7FFFFFFF || a.tokens > 0x3FFFFFFF ||
      a.ld_src < a.d || a.ld_out < a.d || (a.extra != nullptr && a.ld_extra < a.d) ||
      (pads && (a.experts < 1 || a.experts > rb::kMaxExperts))) {
    *rc = route_failed(RB_ERR_SHAPE, "%s: sizes out of range or a row stride below the width (tokens=%lld, width=%lld)",
                       what, a.tokens, a.d);
    return 0;
  }
  const int esize = dtype == RB_DTYPE_BF16 ? 2 : 4, lanes = 16 / esize;
  const bool vec = a.d % lanes == 0 && a.ld_src % lanes == 0 && a.ld_out % lanes == 0 && !unaligned(a.src, 16) &&
                   !unaligned(a.out, 16) && (a.extra == nullptr || (a.ld_extra % lanes == 0 && !unaligned(a.extra, 16)));
  const int per = vec ? lanes : 1;
  // Threads to a token: a warp, and twice that as long as warps would stay idle and the row has vectors for them.
  const int64_t packs = (a.d + per - 1) / per;
  const int64_t warps = (int64_t)rb_host::sm_budget(rb_host::current_device()) * 8 * rb::kRowsBlocksPerSm;
  a.cx = 32;
  while (a.cx < 256 && a.cx < packs && a.tokens * (a.cx / 32) < warps) a.cx <<= 1;
  if (pads) {  // about two thousand pieces to clear, at most 16 an expert
    a.pad_slices = 2048 / a.experts;
    if (a.pad_slices > 16) a.pad_slices = 16;
  }
  *rc = RB_OK;
  return per;
}

}  // namespace

// One wave of blocks, or as many as there are groups of tokens (and, with `pads`, pieces to clear) if that is
// less.
static unsigned rows_grid(const rb::RowsArgs& a, bool pads) {
  const int64_t ny = 256 / a.cx, most = (int64_t)rb_host::sm_budget(rb_host::current_device()) * rb::kRowsBlocksPerSm;
  int64_t want = (a.tokens + ny - 1) / ny;
  if (pads && want < (int64_t)a.experts * a.pad_slices) want = (int64_t)a.experts * a.pad_slices;
  return (unsigned)(want < most ? want : most);
}

#define RB_ROWS_LAUNCH_AS(kernel, T, vec)                                             \
  (a.k <= 2 ? rb::kernel<T, vec, 2, rb::kRowsCols2><<<rows_grid(a, pads), 256, 0, st>>>(a) \
            : rb::kernel<T, vec, 4, rb::kRowsCols4><<<rows_grid(a, pads), 256, 0, st>>>(a))
#define RB_ROWS_LAUNCH(kernel, clears)                                                \
  do {                                                                                \
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);                         \
    constexpr bool pads = clears;                                                     \
    if (dtype == RB_DTYPE_BF16) {                                                     \
      if (per == 8) RB_ROWS_LAUNCH_AS(kernel, __nv_bfloat16, 8);                      \
      else RB_ROWS_LAUNCH_AS(kernel, __nv_bfloat16, 1);                               \
    } else {                                                                          \
      if (per == 4) RB_ROWS_LAUNCH_AS(kernel, float, 4);                              \
      else RB_ROWS_LAUNCH_AS(kernel, float, 1);                                       \
    }                                                                                 \
  } while (0)

extern "C" {

size_t rb_nvfp4_route_workspace(int64_t tokens, int64_t experts, int k) {
  if (tokens < 0 || experts < 1 || experts > rb::kMaxExperts || k < 1 || k > rb::kMaxTopK) return 0;
  // Enough for every SM budget, which another thread may change before the call that uses it.  With s SMs a chunk
  // has at least tokens / (s turns) tokens, turns < tokens / (s most) + 1, or is `most`: never more than
  // s + tokens / most blocks.  And it is never below a step of the block's groups (or `most`).
  const int64_t most = rb::kMaxPairs / k, step = rb::kRouteThreads / route_lanes((int)experts);
  const int64_t least = step < most ? step : most;
  const int64_t a = rb_host::num_sms(rb_host::current_device()) + (tokens + most - 1) / most;
  const int64_t b = (tokens + least - 1) / least;
  const int64_t blocks = a < b ? a : b;
  return route_scratch(blocks > 1 ? blocks : 1, experts);
}

int rb_nvfp4_route_plan(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t ld, int k,
                        const float* expert_bias, const void* valid, int renormalize, float* weights, int32_t* picks,
                        int32_t* rows, int64_t* counts, int64_t* plan_counts, int64_t* offsets, float* loss,
                        float* share, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "nvfp4 route";
  if (const int rc = check_route(what, dtype, tokens, experts, ld, k)) return rc;
  if (counts == nullptr || offsets == nullptr || loss == nullptr || share == nullptr || workspace == nullptr ||
      (tokens > 0 && (logits == nullptr || weights == nullptr || picks == nullptr || rows == nullptr)) ||
      unaligned(counts, 8) || unaligned(plan_counts, 8) || unaligned(offsets, 8) || unaligned(workspace, 4))
    return route_failed(RB_ERR_ARG, "%s: null or misaligned pointer argument", what);
  if (!route_device(what)) return RB_ERR_DEVICE;
  const int64_t sms = rb_host::sm_budget(rb_host::current_device());
  const int64_t chunk = route_chunk(tokens, (int)experts, k, sms);
  const int64_t blocks = tokens > 0 ? (tokens + chunk - 1) / chunk : 1;
  if (workspace_bytes < route_scratch(blocks, experts))
    return route_failed(RB_ERR_ARG, "%s: a workspace of %lld bytes is too small", what, (long long)workspace_bytes);
  rb::RouteArgs a = {};
  a.logits = logits;
  a.tokens = tokens;
  a.ld = ld;
  a.experts = (int)experts;
  a.k = k;
  a.bias = expert_bias;
  a.valid = reinterpret_cast<const uint8_t*>(valid);
  a.renormalize = renormalize;
  a.weights = weights;
  a.picks = picks;
  a.rows = rows;
  a.counts = counts;
  a.plan_counts = plan_counts;
  a.offsets = offsets;
  a.loss = loss;
  a.share = share;
  a.chunk = chunk;
  a.blocks = blocks;
  a.psum = reinterpret_cast<float*>(workspace);
  a.nrouted = reinterpret_cast<int32_t*>(a.psum + a.blocks * experts);
  a.hist = reinterpret_cast<uint16_t*>(a.nrouted + a.blocks);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  route_shape(a.experts, [&](auto l, auto i) {
    if (dtype == RB_DTYPE_BF16)
      rb::route_kernel<__nv_bfloat16, decltype(l)::value, decltype(i)::value>
          <<<(unsigned)a.blocks, rb::kRouteThreads, 0, st>>>(a);
    else
      rb::route_kernel<float, decltype(l)::value, decltype(i)::value>
          <<<(unsigned)a.blocks, rb::kRouteThreads, 0, st>>>(a);
  });
  if (a.blocks > 1) {
    const unsigned workers = (unsigned)(a.blocks < sms ? a.blocks : sms);
    rb::route_plan_kernel<<<workers + 1, rb::kRouteThreads, 0, st>>>(a);
  }
  return route_launched(what);
}

int rb_nvfp4_route(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t ld, int k,
                   const float* expert_bias, const void* valid, int renormalize, float* weights, int32_t* picks,
                   int32_t* rows, int64_t* counts, int64_t* offsets, float* loss, float* share, void* workspace,
                   size_t workspace_bytes, void* stream) {
  return rb_nvfp4_route_plan(logits, dtype, tokens, experts, ld, k, expert_bias, valid, renormalize, weights, picks,
                             rows, counts, nullptr, offsets, loss, share, workspace, workspace_bytes, stream);
}

int rb_nvfp4_route_backward(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t ld, int k,
                            int renormalize, const float* weights, const int32_t* picks, const float* share,
                            const float* grad_weights, const float* grad_loss, void* grad_logits, int64_t ldo,
                            void* stream) {
  const char* what = "nvfp4 route_backward";
  if (const int rc = check_route(what, dtype, tokens, experts, ld, k)) return rc;
  if (ldo < experts) return route_failed(RB_ERR_SHAPE, "%s: the gradient's row stride %lld is below %lld experts", what, ldo, experts);
  if (tokens == 0) return RB_OK;
  if (logits == nullptr || weights == nullptr || picks == nullptr || share == nullptr ||
      grad_logits == nullptr)
    return route_failed(RB_ERR_ARG, "%s: null or misaligned pointer argument", what);
  if (!route_device(what)) return RB_ERR_DEVICE;
  rb::RouteBwdArgs a = {};
  a.logits = logits;
  a.tokens = tokens;
  a.ld = ld;
  a.experts = (int)experts;
  a.k = k;
  a.renormalize = renormalize;
  a.weights = weights;
  a.picks = picks;
  a.share = share;
  a.grad_w = grad_weights;
  a.grad_loss = grad_loss;
  a.grad = grad_logits;
  a.ldo = ldo;
  const int groups = rb::kRouteThreads / route_lanes(a.experts);
  const int64_t blocks = (tokens + groups - 1) / groups, most = (int64_t)8 * rb_host::sm_budget(rb_host::current_device());
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  route_shape(a.experts, [&](auto l, auto i) {
    if (dtype == RB_DTYPE_BF16)
      rb::route_backward_kernel<__nv_bfloat16, decltype(l)::value, decltype(i)::value>
          <<<grid, rb::kRouteThreads, 0, st>>>(a);
    else
      rb::route_backward_kernel<float, decltype(l)::value, decltype(i)::value><<<grid, rb::kRouteThreads, 0, st>>>(a);
  });
  return route_launched(what);
}

int rb_nvfp4_token_dispatch(const void* x, int dtype, int64_t tokens, int64_t d, int64_t ldx, const int32_t* rows,
                            int k, const int64_t* counts, const int64_t* offsets, int64_t experts, void* out,
                            int64_t num_rows, int64_t ldo, void* stream) {
  const char* what = "nvfp4 token_dispatch";
  rb::RowsArgs a = {};
  a.src = x;
  a.ld_src = ldx;
  a.rows = rows;
  a.k = k;
  a.counts = counts;
  a.offsets = offsets;
  a.experts = (int)(experts < 0 || experts > rb::kMaxExperts ? 0 : experts);
  a.out = out;
  a.num_rows = num_rows;
  a.ld_out = ldo;
  a.tokens = tokens;
  a.d = d;
  int rc;
  const int per = rows_shape(what, a, dtype, true, &rc);
  if (per == 0) return rc;
  if (num_rows == 0) return RB_OK;
  if (out == nullptr || counts == nullptr || offsets == nullptr || (tokens > 0 && (x == nullptr || rows == nullptr)) ||
      unaligned(counts, 8) || unaligned(offsets, 8))
    return route_failed(RB_ERR_ARG, "%s: null or misaligned pointer argument", what);
  if (!route_device(what)) return RB_ERR_DEVICE;
  RB_ROWS_LAUNCH(token_dispatch_kernel, true);
  return route_launched(what);
}

int rb_nvfp4_token_combine(const void* y, int dtype, int64_t num_rows, int64_t d, int64_t ldy, const int32_t* rows,
                           int k, const float* weights, const void* residual, int64_t ldr, void* out, int64_t tokens,
                           int64_t ldo, void* stream) {
  const char* what = "nvfp4 token_combine";
  rb::RowsArgs a = {};
  a.src = y;
  a.ld_src = ldy;
  a.extra = residual;
  a.ld_extra = ldr;
  a.rows = rows;
  a.weights = weights;
  a.k = k;
  a.out = out;
  a.num_rows = num_rows;
  a.ld_out = ldo;
  a.tokens = tokens;
  a.d = d;
  int rc;
  const int per = rows_shape(what, a, dtype, false, &rc);
  if (per == 0) return rc;
  if (tokens == 0) return RB_OK;
  if (out == nullptr || rows == nullptr || (num_rows > 0 && y == nullptr))
    return route_failed(RB_ERR_ARG, "%s: null pointer argument", what);
  if (!route_device(what)) return RB_ERR_DEVICE;
  RB_ROWS_LAUNCH(token_combine_kernel, false);
  return route_launched(what);
}

int rb_nvfp4_token_combine_backward(const void* grad_y, int64_t ldg, const void* y, int64_t ldy, int dtype,
                                    int64_t tokens, int64_t d, const int32_t* rows, int k, const float* weights,
                                    const int64_t* counts, const int64_t* offsets, int64_t experts, void* grad_rows,
                                    int64_t num_rows, int64_t ldo, float* grad_weights, void* stream) {
  const char* what = "nvfp4 token_combine_backward";
  rb::RowsArgs a = {};
  a.src = y;
  a.ld_src = ldy;
  a.extra = grad_y;
  a.ld_extra = ldg;
  a.rows = rows;
  a.weights = weights;
  a.k = k;
  a.counts = counts;
  a.offsets = offsets;
  a.experts = (int)(experts < 0 || experts > rb::kMaxExperts ? 0 : experts);
  a.out = grad_rows;
  a.num_rows = num_rows;
  a.ld_out = ldo;
  a.grad_w = grad_weights;
  a.tokens = tokens;
  a.d = d;
  int rc;
  const int per = rows_shape(what, a, dtype, true, &rc);
  if (per == 0) return rc;
  if (num_rows == 0 && tokens == 0) return RB_OK;
  if (counts == nullptr || offsets == nullptr || unaligned(counts, 8) || unaligned(offsets, 8) ||
      (num_rows > 0 && (grad_rows == nullptr || y == nullptr)) ||
      (tokens > 0 && (grad_y == nullptr || rows == nullptr || weights == nullptr || grad_weights == nullptr)))
    return route_failed(RB_ERR_ARG, "%s: null or misaligned pointer argument", what);
  if (!route_device(what)) return RB_ERR_DEVICE;
  RB_ROWS_LAUNCH(token_combine_backward_kernel, true);
  return route_launched(what);
}

}  // extern "C"

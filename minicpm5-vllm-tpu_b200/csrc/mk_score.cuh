// Scoring of given tokens: log-probability, entropy, rank and best alternatives from rows of logits, and the
// first two from hidden rows through the lm_head without the logits ever being in memory.
//
// With m = max x, u = x - m, z = sum e^u:   lse = m + ln z,   ln p_t = u_t - ln z,
//                                           entropy = -sum p ln p = ln z - (sum e^u u) / z
// Partial (m, z, w = sum e^u u) over disjoint parts join at m' = max m: with d = m - m',
//   z' += z e^d,   w' += (w + z d) e^d
#pragma once

#include "mk_common.cuh"

namespace mk {

// Running statistics of part of a row.  m = -inf: nothing seen (or only -inf); then z = w = 0.  A logit of
// -inf adds nothing; +inf and NaN make z NaN, and with it all that is computed from the row.  Differences that
// only multiply a weight of 0 are cut at kFar (e^-200 is 0 in f32), where 0 * inf would be NaN.
struct RowStats {
  float m, z, w;
};
constexpr float kFar = -200.f;
__device__ __forceinline__ RowStats stats_empty() { return {-INFINITY, 0.f, 0.f}; }
__device__ __forceinline__ RowStats stats_join(const RowStats& a, const RowStats& b) {
  RowStats r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = a.m - ref, db = b.m - ref, ea = __expf(da), eb = __expf(db);
  r.z = a.z * ea + b.z * eb;
  r.w = (a.w + a.z * fmaxf(da, kFar)) * ea + (b.w + b.z * fmaxf(db, kFar)) * eb;
  return r;
}
__device__ __forceinline__ void stats_add(RowStats& s, float x) {
  s = stats_join(s, {x, x == -INFINITY ? 0.f : x - x == 0.f ? 1.f : __int_as_float(0x7fffffff), 0.f});
}
__device__ __forceinline__ RowStats stats_warp(RowStats s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    RowStats t;
    t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
    t.z = __shfl_xor_sync(0xffffffffu, s.z, o);
    t.w = __shfl_xor_sync(0xffffffffu, s.w, o);
    s = stats_join(s, t);
  }
  return s;
}

// Order of the alternatives: value descending, then id ascending; zeros of either sign are equal and a NaN
// comes after every number.  An entry is one 64-bit number, larger = earlier.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_entry(uint32_t key, int id) {
  return static_cast<unsigned long long>(key) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int order_id(unsigned long long e) { return static_cast<int>(~static_cast<uint32_t>(e)); }

// ---------------------------------------------------------------------------------- from logits
// One CTA per row: one pass for the statistics and the rank, then one for each alternative, the largest entry
// that comes after the last pick.
constexpr int TL_THREADS = 1024;
constexpr int TL_TOPK_MAX = 64;

template <typename E>
__device__ __forceinline__ float logit_at(const E* p, size_t i);
template <>
__device__ __forceinline__ float logit_at<float>(const float* p, size_t i) { return p[i]; }
template <>
__device__ __forceinline__ float logit_at<__nv_bfloat16>(const __nv_bfloat16* p, size_t i) { return __bfloat162float(p[i]); }

template <typename E>
__global__ void __launch_bounds__(TL_THREADS)
    token_logprobs_kernel(const E* __restrict__ logits, int V, long long ld, const int32_t* __restrict__ targets, int k,
                          float* __restrict__ lp, float* __restrict__ ent, int32_t* __restrict__ rank,
                          int32_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  __shared__ RowStats rs[32];
  __shared__ int rc[32];
  __shared__ unsigned long long pick[32];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wp = tid >> 5;
  const E* row = logits + static_cast<long long>(b) * ld;
  const int t = targets[b];
  const bool given = t >= 0 && t < V;
  const float mine = given ? logit_at(row, t) : 0.f;
  RowStats s = stats_empty();
  int above = 0;
  for (int i = tid; i < V; i += TL_THREADS) {
    const float x = logit_at(row, i);
    stats_add(s, x);
    above += x > mine || (mine != mine && x == x);
  }
  s = stats_warp(s);
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) { rs[wp] = s; rc[wp] = above; }
  __syncthreads();
  s = rs[0];
  above = rc[0];
  for (int i = 1; i < 32; ++i) { s = stats_join(s, rs[i]); above += rc[i]; }
  const float lz = logf(s.z);
  if (tid == 0) {
    lp[b] = !given ? 0.f : s.z == 0.f ? -INFINITY : mine - s.m - lz;
    ent[b] = s.z == 0.f ? 0.f : lz - s.w / s.z;
    rank[b] = given ? above + 1 : 0;
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < k; ++r) {
    unsigned long long best = 0;
    for (int i = tid; i < V; i += TL_THREADS) {
      const unsigned long long e = order_entry(order_key(logit_at(row, i)), i);
      if (e < last && e > best) best = e;
    }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) pick[wp] = best;
    __syncthreads();
    for (int i = 0; i < 32; ++i) best = max(best, pick[i]);
    last = best;
    if (tid == 0) {
      const int id = order_id(best);
      top_ids[static_cast<size_t>(b) * k + r] = id;
      top_lp[static_cast<size_t>(b) * k + r] = s.z == 0.f ? -INFINITY : logit_at(row, id) - s.m - lz;
    }
  }
}

// ---------------------------------------------------------------------------------- from hidden rows
// Partial statistics of row t over one part of the vocabulary.
struct ScorePart {
  float m, z, w;
};

// SC_TOK hidden rows in shared memory as f32; a warp walks the part's vocabulary rows, its lanes split H.
constexpr int SC_TOK = 8;
constexpr int SC_THREADS = 256;
__global__ void __launch_bounds__(SC_THREADS)
    score_tokens_kernel(const __nv_bfloat16* __restrict__ h, int T, int H, long long ld, const __nv_bfloat16* __restrict__ W,
                        int V, const int32_t* __restrict__ targets, float scale, ScorePart* __restrict__ part,
                        float* __restrict__ target_logit) {
  extern __shared__ float hs[];  // [SC_TOK][H]
  __shared__ RowStats red[SC_THREADS / 32][SC_TOK];
  pdl_wait();
  pdl_trigger();
  const int tok0 = blockIdx.x * SC_TOK, lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < SC_TOK * H; i += SC_THREADS) {
    const int t = tok0 + i / H;
    hs[i] = t < T ? __bfloat162float(h[static_cast<long long>(t) * ld + i % H]) : 0.f;
  }
  __syncthreads();
  const int per = (V + gridDim.y - 1) / gridDim.y, v0 = blockIdx.y * per, v1 = min(V, v0 + per);
  RowStats s[SC_TOK];
  int tg[SC_TOK];
#pragma unroll
  for (int t = 0; t < SC_TOK; ++t) {
    s[t] = stats_empty();
    tg[t] = tok0 + t < T ? targets[tok0 + t] : -1;
  }
  for (int v = v0 + wp; v < v1; v += SC_THREADS / 32) {
    float acc[SC_TOK] = {};
    for (int c = lane; c < H; c += 32) {
      const float w = __bfloat162float(W[static_cast<size_t>(v) * H + c]);
#pragma unroll
      for (int t = 0; t < SC_TOK; ++t) acc[t] += w * hs[t * H + c];
    }
#pragma unroll
    for (int t = 0; t < SC_TOK; ++t) {
      for (int o = 16; o; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
      const float x = acc[t] * scale;
      stats_add(s[t], x);
      if (v == tg[t] && lane == 0) target_logit[tok0 + t] = x;
    }
  }
  if (lane == 0)
#pragma unroll
    for (int t = 0; t < SC_TOK; ++t) red[wp][t] = s[t];
  __syncthreads();
  if (threadIdx.x < SC_TOK && tok0 + threadIdx.x < T) {
    RowStats r = red[0][threadIdx.x];
    for (int i = 1; i < SC_THREADS / 32; ++i) r = stats_join(r, red[i][threadIdx.x]);
    part[static_cast<size_t>(tok0 + threadIdx.x) * gridDim.y + blockIdx.y] = {r.m, r.z, r.w};
  }
}

// Joins a row's parts in order.
__global__ void score_join_kernel(const ScorePart* __restrict__ part, int nparts, int T, int V,
                                  const int32_t* __restrict__ targets, const float* __restrict__ target_logit,
                                  float* __restrict__ lp, float* __restrict__ ent) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  RowStats s = stats_empty();
  for (int i = 0; i < nparts; ++i) {
    const ScorePart p = part[static_cast<size_t>(t) * nparts + i];
    s = stats_join(s, {p.m, p.z, p.w});
  }
  const int tg = targets[t];
  const float lz = logf(s.z);
  lp[t] = tg < 0 || tg >= V ? 0.f : s.z == 0.f ? -INFINITY : target_logit[t] - s.m - lz;
  ent[t] = s.z == 0.f ? 0.f : lz - s.w / s.z;
}

}  // namespace mk

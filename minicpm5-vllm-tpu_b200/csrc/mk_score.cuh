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
// Row statistics of logits = scale * h W^T, tile by tile.  D[token, v] is computed by tcgen05.mma with tokens on
// the TMEM lanes, so that an epilogue thread owns one token and walks its tile's 256 logits with (m, z, w) in
// registers: nothing crosses lanes, and what leaves the kernel is 12 bytes per (token, 256 logits) instead of
// 1024 (f32 logits of 8192 tokens over 73448 ids would be 2.4 GB written and read again).
//
// What bounds it: 2 H operations per logit against five instructions and one exponential in the epilogue; with
// H = 1536 the tensor cores take 12288 cycles for a 128 x 256 tile and the exponentials 2048, hidden behind the
// next tile's products (two accumulators fill the 512 TMEM columns).  With few tokens W's bytes are the bound.
//
// Layout.  PAIR (more than 128 tokens): two CTAs work on 256 tokens x 256 ids with 2-SM MMAs, each holding its 128
// tokens and half of the ids, which halves the operand bytes that each SM takes in per product.  Otherwise one
// CTA works on 128 tokens x 256 ids.  Tiles go out id-major: the CTAs at work share a few id tiles at a time, so W
// comes from HBM once and the token tiles stay in L2.
//   warp 0     TMA producer (64 of H per stage, 128-byte swizzle)
//   warp 1     TMEM allocator and MMA issuer (the even CTA's, for both of a pair)
//   warps 2-5  epilogue, one per 32-lane quarter of TMEM
constexpr int SC_M = 128;      // tokens per CTA
constexpr int SC_V = 256;      // ids per tile
constexpr int SC_K = 64;       // of H per stage
constexpr int SC_THREADS = 192;
constexpr uint32_t SC_A_BYTES = SC_M * SC_K * 2;
__host__ __device__ constexpr int sc_stages(bool pair) { return pair ? 6 : 4; }
__host__ __device__ constexpr int sc_b_rows(bool pair) { return pair ? SC_V / 2 : SC_V; }
__host__ __device__ constexpr uint32_t sc_stage_bytes(bool pair) { return SC_A_BYTES + sc_b_rows(pair) * SC_K * 2; }
__host__ __device__ constexpr size_t sc_smem_bytes(bool pair) { return 1024 + sc_stages(pair) * sc_stage_bytes(pair) + 256; }
constexpr float kLn2 = 0.693147180559945f;

struct ScoreArgs {
  int T, H, V, id_tiles, tok_tiles;
  const int32_t* targets;
  float scale;          // logit scale * log2 e: the statistics are in units of log 2
  float* part;          // [id tiles][3][ld_part]: m, z, w
  long long ld_part;    // T rounded up
  float* target_logit;  // [T]
  int* err;
};

template <bool PAIR>
__global__ void __launch_bounds__(SC_THREADS, 1)
    score_tokens_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
                        const ScoreArgs args) {
  constexpr int STAGES = sc_stages(PAIR), B_ROWS = sc_b_rows(PAIR);
  constexpr uint32_t STAGE = sc_stage_bytes(PAIR);
  extern __shared__ uint8_t sc_smem_raw[];
  const uint32_t raw = smem_u32(sc_smem_raw);
  uint8_t* base = sc_smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(base + STAGES * STAGE);  // [STAGES] both operands landed
  uint64_t* empty = full + STAGES;   // [STAGES] the MMAs that read the stage finished
  uint64_t* tfull = empty + STAGES;  // [2] accumulator ready
  uint64_t* tempty = tfull + 2;      // [2] accumulator drained
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = PAIR ? cluster_ctarank() : 0u;
  auto lead_bar = [&](uint64_t* b) { return PAIR ? mapa_cluster(smem_u32(b), 0) : smem_u32(b); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4 * (PAIR ? 2 : 1));
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmH);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();

  const int unit = PAIR ? static_cast<int>(blockIdx.x) >> 1 : static_cast<int>(blockIdx.x);
  const int units = PAIR ? static_cast<int>(gridDim.x) >> 1 : static_cast<int>(gridDim.x);
  const int tiles = args.id_tiles * args.tok_tiles, my_tiles = (tiles - unit + units - 1) / units;
  const int KT = (args.H + SC_K - 1) / SC_K;  // past H both operands read zeros
  auto id_tile = [&](int it) { return (unit + it * units) / args.tok_tiles; };
  // first token of this CTA's half of the tile
  auto tok0 = [&](int it) {
    return ((unit + it * units) % args.tok_tiles) * (PAIR ? 2 * SC_M : SC_M) + static_cast<int>(crank) * SC_M;
  };

  if (warp == 0) {
    const bool leader = elect_one();
    pdl_wait();
    uint32_t issued = 0, issued_par = 0;
    int idx = 0;
    bool ok = true;
    for (int it = 0; ok && it < my_tiles; ++it) {
      const int t0 = tok0(it), v0 = id_tile(it) * SC_V + static_cast<int>(crank) * (PAIR ? B_ROWS : 0);
      for (int kt = 0; kt < KT; ++kt, ++idx) {
        const int s = idx % STAGES;
        const uint32_t ph = (idx / STAGES) & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ph ^ 1u, abort_flag));
        if (!ok) break;
        if (leader) {
          uint8_t* at = base + s * STAGE;
          if constexpr (PAIR) {
            if (crank == 0) mbar_arrive_expect_tx(&full[s], 2 * STAGE);
            const uint32_t fb = lead_bar(&full[s]);
            tma_load_2d_pair(at, &tmH, fb, kt * SC_K, t0);
            tma_load_2d_pair(at + SC_A_BYTES, &tmW, fb, kt * SC_K, v0);
          } else {
            mbar_arrive_expect_tx(&full[s], STAGE);
            tma_load_2d(at, &tmH, &full[s], kt * SC_K, t0);
            tma_load_2d(at + SC_A_BYTES, &tmW, &full[s], kt * SC_K, v0);
          }
        }
        __syncwarp();
        issued |= 1u << s;
        issued_par = (issued_par & ~(1u << s)) | (ph << s);
      }
    }
    // every issued copy lands before the CTA may exit (a pair's on the even CTA's barriers)
    if (!PAIR || crank == 0)
      for (int s = 0; s < STAGES; ++s)
        if (issued & (1u << s)) mbar_wait_drain(&full[s], (issued_par >> s) & 1u);
  } else if (warp == 1) {
    if (!PAIR || crank == 0) {
      const bool leader = elect_one();
      const uint32_t idesc = idesc_bf16_f32(PAIR ? 2 * SC_M : SC_M, SC_V);
      auto commit_all = [&](uint64_t* b) {
        if constexpr (PAIR) {
          mma_commit_pair(smem_u32(b));
          mma_commit_pair(mapa_cluster(smem_u32(b), 1));
        } else {
          mma_commit(b);
        }
      };
      int idx = 0;
      bool ok = true;
      for (int it = 0; ok && it < my_tiles; ++it) {
        const int a = it & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&tempty[a], ((it >> 1) & 1) ^ 1u, abort_flag))) break;
        tc_fence_after();
        const uint32_t d = tmem_base + a * SC_V;
        for (int kt = 0; kt < KT; ++kt, ++idx) {
          const int s = idx % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (idx / STAGES) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = sdesc_kmajor_sw128(smem_u32(base + s * STAGE));
          const uint64_t db = sdesc_kmajor_sw128(smem_u32(base + s * STAGE + SC_A_BYTES));
          if (leader) {
#pragma unroll
            for (int k = 0; k < SC_K / 16; ++k) {
              if constexpr (PAIR)
                mma_f16_ss_pair(d, da + 2 * k, db + 2 * k, idesc, (kt | k) != 0 ? 1u : 0u);
              else
                mma_f16_ss(d, da + 2 * k, db + 2 * k, idesc, (kt | k) != 0 ? 1u : 0u);
            }
            commit_all(&empty[s]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) commit_all(&tfull[a]);
        __syncwarp();
      }
      if (leader) {
        if constexpr (PAIR)
          mma_commit_pair(smem_u32(drain));
        else
          mma_commit(drain);
      }
      __syncwarp();
      mbar_wait_drain(drain, 0);
    }
  } else {
    const int q = warp & 3;  // the TMEM quarter that this warp may read
    pdl_wait();
    for (int it = 0; it < my_tiles; ++it) {
      const int a = it & 1, vt = id_tile(it), t = tok0(it) + q * 32 + lane, v0 = vt * SC_V;
      const int tg = t < args.T ? args.targets[t] : -1;
      const int nv = min(SC_V, args.V - v0);
      if (!mbar_wait(&tfull[a], (it >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      float m = -INFINITY, z = 0.f, w = 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < nv; c0 += 32) {
        uint32_t acc[32];
        tmem_ld_32x32b_x32(tmem_base + a * SC_V + c0 + (static_cast<uint32_t>(q * 32) << 16), acc);
        tmem_ld_wait();
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(acc[j]) * args.scale;
        if (c0 + 32 > nv) {  // ids past the vocabulary weigh nothing
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c0 + j >= nv) y[j] = -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 32; j += 2) top = max3f(top, y[j], y[j + 1]);
        const float ref = top == -INFINITY ? 0.f : top, d = m - ref, f = ex2_approx(d);
        w = (w + z * fmaxf(d, kFar)) * f;
        z *= f;
        m = top;
        float z1 = 0.f, w1 = 0.f;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float ua = y[j] - ref, ub = y[j + 1] - ref, ea = ex2_approx(ua), eb = ex2_approx(ub);
          z += ea;
          z1 += eb;
          w = fmaf(ea, fmaxf(ua, kFar), w);
          w1 = fmaf(eb, fmaxf(ub, kFar), w1);
        }
        z += z1;
        w += w1;
        const int at = tg - v0 - c0;
        if (at >= 0 && at < 32) {
          float x = y[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) x = j == at ? y[j] : x;
          if (tg < args.V) args.target_logit[t] = x;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_cluster(lead_bar(&tempty[a]));
        else
          mbar_arrive(&tempty[a]);
      }
      if (t < args.T) {
        float* p = args.part + static_cast<long long>(vt) * 3 * args.ld_part + t;
        p[0] = m;
        p[args.ld_part] = z;
        p[2 * args.ld_part] = w;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if constexpr (PAIR) {
    cluster_sync();  // neither CTA frees its TMEM or leaves while the pair's MMAs may still read its operands
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
  } else {
    if (warp == 1) tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag && args.err) atomicCAS(args.err, 0, DEV_ERR_TIMEOUT_SCORE);
}

// Joins a token's id tiles: 32 tokens x SJ_SLICES slices of the tiles per CTA, then the slices in order.
constexpr int SJ_SLICES = 32;
__device__ __forceinline__ RowStats stats_join2(const RowStats& a, const RowStats& b) {  // units of log 2
  RowStats r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = a.m - ref, db = b.m - ref, ea = ex2_approx(da), eb = ex2_approx(db);
  r.z = a.z * ea + b.z * eb;
  r.w = (a.w + a.z * fmaxf(da, kFar)) * ea + (b.w + b.z * fmaxf(db, kFar)) * eb;
  return r;
}
__global__ void __launch_bounds__(32 * SJ_SLICES)
    score_join_kernel(const ScoreArgs args, float* __restrict__ lp, float* __restrict__ ent) {
  __shared__ RowStats s_p[SJ_SLICES][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, t = blockIdx.x * 32 + lane;
  RowStats s = stats_empty();
  if (t < args.T) {
#pragma unroll 4
    for (int vt = slice; vt < args.id_tiles; vt += SJ_SLICES) {
      const float* p = args.part + static_cast<long long>(vt) * 3 * args.ld_part + t;
      s = stats_join2(s, {p[0], p[args.ld_part], p[2 * args.ld_part]});
    }
  }
  s_p[slice][lane] = s;
  __syncthreads();
  if (slice || t >= args.T) return;
  for (int i = 1; i < SJ_SLICES; ++i) s = stats_join2(s, s_p[i][lane]);
  const int tg = args.targets[t];
  const float lz = log2f(s.z);
  lp[t] = tg < 0 || tg >= args.V ? 0.f : s.z == 0.f ? -INFINITY : (args.target_logit[t] - s.m - lz) * kLn2;
  ent[t] = s.z == 0.f ? 0.f : (lz - s.w / s.z) * kLn2;
}

}  // namespace mk

// Attention of new tokens over the 8-bit paged cache (layout in mk_cache.cuh).
//
//   s_j = softmax_scale * kscale * (q . kcode_j)   keys j <= the query's position
//   o   = sum_j exp(s_j - m) * vscale * vcode_j / sum_j exp(s_j - m),   lse = m + ln sum_j exp(s_j - m)
//
// A row that sees no key (an idle row of the batch) gives zeros and lse = -inf.
#pragma once

#include "mk_cache.cuh"

namespace mk {

struct PagedAttnArgs {
  const __nv_bfloat16* q;
  long long ld_q, hs_q;
  int n_q, rows, width;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  float scale;
  __nv_bfloat16* out;
  float* lse;
  int* err;
};

// One CTA per (token, query head): 128 keys at a time, one score per thread, then one channel per thread.
constexpr int PA_THREADS = 128;
__global__ void __launch_bounds__(PA_THREADS) attn_paged_kernel(KvPages c, PagedAttnArgs a) {
  __shared__ float qs[128], ps[PA_THREADS], red[PA_THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const int tok = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = c.head_dim;
  int row = tok, n = 1, first = tok;
  if (a.cu) {
    int lo = 0, hi = a.rows - 1;  // last row that begins at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= tok) lo = mid; else hi = mid - 1;
    }
    row = lo;
    first = a.cu[row];
    n = a.cu[row + 1] - first;
  }
  const int keys = a.lens[row] - n + (tok - first) + 1;  // keys this query sees
  const int kvh = h / (a.n_q / c.n_kv);
  if (tid < hd) qs[tid] = __bfloat162float(a.q[static_cast<long long>(tok) * a.ld_q + h * a.hs_q + tid]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int base = 0; base < keys; base += PA_THREADS) {
    const int j = base + tid;
    float s = -INFINITY;
    int page = -1;
    if (j < keys) page = kv_page_of(a.table, a.width, c.num_pages, row, j >> c.page_shift, a.err);
    if (page >= 0) {
      const int8_t* kp = kv_head_ptr(c, page, 0, kvh) + static_cast<size_t>(j & ((1 << c.page_shift) - 1)) * hd;
      float d = 0.f;
      for (int e = 0; e < hd; ++e) d += qs[e] * static_cast<float>(kp[e]);
      s = d * (*kv_scale_ptr(c, page, 0, kvh) * a.scale);
    }
    float mx = s;
    for (int w = 16; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = m;
    for (int w = 0; w < PA_THREADS / 32; ++w) mx = fmaxf(mx, red[w]);
    const float p = page >= 0 ? expf(s - mx) : 0.f;
    float sum = p;
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    ps[tid] = page >= 0 ? p * *kv_scale_ptr(c, page, 1, kvh) : 0.f;
    __syncthreads();
    const float keep = mx == m ? 1.f : expf(m - mx);
    l *= keep;
    for (int w = 0; w < PA_THREADS / 32; ++w) l += red[w];
    o *= keep;
    m = mx;
    if (tid < hd)
      for (int i = 0; i < min(PA_THREADS, keys - base); ++i) {
        const int pg = kv_page_of(a.table, a.width, c.num_pages, row, (base + i) >> c.page_shift, a.err);
        if (pg < 0) continue;
        const int in = (base + i) & ((1 << c.page_shift) - 1);
        o += ps[i] * static_cast<float>(kv_head_ptr(c, pg, 1, kvh)[(static_cast<size_t>(in >> 2) * hd + tid) * 4 + (in & 3)]);
      }
    __syncthreads();
  }
  if (tid < hd)
    a.out[(static_cast<size_t>(tok) * a.n_q + h) * hd + tid] = __float2bfloat16(l == 0.f ? 0.f : o / l);
  if (tid == 0 && a.lse) a.lse[static_cast<size_t>(tok) * a.n_q + h] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace mk

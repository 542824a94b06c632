// C ABI of token scoring: log-probabilities of given tokens from logits or from hidden rows.
// See include/minicpm5_mk.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "mk_host.cuh"
#include "mk_score.cuh"

namespace {

using mk::aligned16;
using mk::HostDevice;
using mk::launch_k;
using mk::launch_k_cluster;
using mk::launch_k_pair;

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// More than one CTA's tokens go to CTA pairs: up to 128 half of a pair's products would be with rows past the end.
bool in_pairs(int T) { return T > mk::SC_M; }
int64_t id_tiles(int T, int V) {
  const int ids = mk::sc_ids(in_pairs(T));
  return (static_cast<int64_t>(V) + ids - 1) / ids;
}
int64_t ld_part(int T) { return (static_cast<int64_t>(T) + 31) / 32 * 32; }
size_t part_bytes(int T, int V) { return align256(static_cast<size_t>(id_tiles(T, V)) * 3 * ld_part(T) * sizeof(float)); }

// bf16 rows [rows, ld], boxes of 64 columns x box_rows, 128-byte swizzle; zeros past the last row and column.
mk_status map_rows(const HostDevice& d, CUtensorMap* m, const void* p, int64_t rows, int cols, int64_t ld, int box_rows) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {mk::SC_K, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t es[2] = {1, 1};
  const CUresult r = d.encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, es,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MK_OK : MK_ERR_CUDA;
}

// Per-device set-up of the scoring kernels: shared memory limits and how many CTA pairs run at once.
constexpr int kMaxDevices = 64;
std::mutex g_mu;
int g_pairs[kMaxDevices];
bool g_ready[kMaxDevices];

mk_status score_pairs(int sms, int* pairs) {
  int dev = 0;
  MK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return MK_ERR_BAD_ARG;
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_ready[dev]) {
    MK_CUDA(cudaFuncSetAttribute(mk::score_tokens_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(mk::SC_SMEM_BYTES)));
    MK_CUDA(cudaFuncSetAttribute(mk::score_tokens_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(mk::SC_SMEM_BYTES)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (sms / 2));
    cfg.blockDim = dim3(mk::SC_THREADS);
    cfg.dynamicSmemBytes = mk::SC_SMEM_BYTES;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    MK_CUDA(cudaOccupancyMaxActiveClusters(&n, mk::score_tokens_kernel<true>, &cfg));
    if (n <= 0) return MK_ERR_CUDA;
    g_pairs[dev] = n;
    g_ready[dev] = true;
  }
  *pairs = g_pairs[dev];
  return MK_OK;
}

}  // namespace

extern "C" {

mk_status mk_token_logprobs(const void* logits, int32_t logits_bits, int32_t T, int32_t V, int64_t ld,
                            const int32_t* targets, int32_t top_k, float* logprobs, float* entropy, int32_t* ranks,
                            int32_t* top_ids, float* top_logprobs, void* stream) {
  if (logits_bits != 16 && logits_bits != 32) return MK_ERR_BAD_ARG;
  if (T < 0 || V <= 0 || ld < 0 || top_k < 0 || top_k > mk::TL_TOPK_MAX || top_k > V) return MK_ERR_BAD_SHAPE;
  if (T == 0) return MK_OK;
  if (!logits || !targets || !logprobs || !entropy || !ranks || (top_k && (!top_ids || !top_logprobs))) return MK_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(logits) % (logits_bits / 8)) return MK_ERR_BAD_ALIGN;
  HostDevice d;
  MK_TRY(mk::host_device(&d));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  mk::LogitsArgs a;
  a.logits = logits;
  a.V = V;
  a.k = top_k;
  a.ld = ld;
  a.targets = targets;
  a.lp = logprobs;
  a.ent = entropy;
  a.rank = ranks;
  a.top_ids = top_ids;
  a.top_lp = top_logprobs;
  // A row is shared by as many CTAs of 512 threads (up to eight) as still have half a step's 8192 logits each, while
  // there are SMs for them (us at 130560 f32, k = 5, with 1, 2, 4, 8 CTAs a row: 8 rows 21, 15, 11, 10; 74 rows 22, 18,
  // 23, 29; 148 rows 24, 22, 35, 48).  From there on a row has one CTA: of 512 threads while the rows are up to three an
  // SM (296 rows 32, with 128 threads 56; 400 rows 49 and 60; bf16 26 and 44, 40 and 47), then of 128, eight to an SM
  // (1184 rows 125 with 512 threads, 101 with 128; bf16 94 and 74).
  int cluster = 1;
  while (cluster < mk::TL_CLUSTER_MAX && static_cast<int64_t>(T) * cluster * 2 <= d.sm_count && V / (cluster * 2) >= 8192)
    cluster *= 2;
  const bool many = cluster > 1 || (T <= static_cast<int64_t>(d.sm_count) * 3 && V >= mk::TL_MANY * mk::TL_VALUES);
  if (many) {
    void (*k)(mk::LogitsArgs, int) = logits_bits == 32 ? mk::token_logprobs_kernel<float, mk::TL_MANY>
                                                       : mk::token_logprobs_kernel<__nv_bfloat16, mk::TL_MANY>;
    if (cluster == 1) return launch_k(k, dim3(static_cast<unsigned>(T)), dim3(mk::TL_MANY), 0, st, true, a, 1);
    return launch_k_cluster(cluster, k, dim3(static_cast<unsigned>(T) * cluster), dim3(mk::TL_MANY), 0, st, true, a, cluster);
  }
  void (*k)(mk::LogitsArgs, int) = logits_bits == 32 ? mk::token_logprobs_kernel<float, mk::TL_FEW>
                                                     : mk::token_logprobs_kernel<__nv_bfloat16, mk::TL_FEW>;
  return launch_k(k, dim3(static_cast<unsigned>(T)), dim3(mk::TL_FEW), 0, st, true, a, 1);
}

mk_status mk_score_tokens_workspace(int32_t T, int32_t H, int32_t V, size_t* bytes) {
  if (!bytes) return MK_ERR_BAD_ARG;
  if (T < 0 || H <= 0 || H % 8 || V <= 0) return MK_ERR_BAD_SHAPE;
  *bytes = part_bytes(T, V) + static_cast<size_t>(T) * sizeof(float);
  return MK_OK;
}

mk_status mk_score_tokens(const void* h, int32_t T, int32_t H, int64_t ld, const void* lm_head, int32_t V,
                          const int32_t* targets, float logit_scale, float* logprobs, float* entropy, void* workspace,
                          size_t workspace_bytes, void* stream) {
  size_t need = 0;
  MK_TRY(mk_score_tokens_workspace(T, H, V, &need));
  if (ld < H) return MK_ERR_BAD_SHAPE;
  if (T == 0) return MK_OK;
  if (!h || !lm_head || !targets || !logprobs || !entropy || !workspace) return MK_ERR_BAD_ARG;
  if (workspace_bytes < need) return MK_ERR_WORKSPACE;
  if (!aligned16(h) || !aligned16(lm_head) || !aligned16(workspace) || ld % 8) return MK_ERR_BAD_ALIGN;
  HostDevice d;
  MK_TRY(mk::host_device(&d));
  int pairs = 0;
  MK_TRY(score_pairs(d.sm_count, &pairs));
  const bool pair = in_pairs(T);
  const int tok_tile = pair ? 2 * mk::SC_M : mk::SC_M;
  const int64_t tok_tiles = (static_cast<int64_t>(T) + tok_tile - 1) / tok_tile, ids = id_tiles(T, V);
  if (tok_tiles * ids > INT_MAX / 2) return MK_ERR_TOO_LARGE;
  CUtensorMap mh, mw;
  const int rows = pair ? mk::SC_M : (T + 7) / 8 * 8;
  MK_TRY(map_rows(d, &mh, h, T, H, ld, rows));
  MK_TRY(map_rows(d, &mw, lm_head, V, H, H, mk::SC_B_ROWS));
  mk::ScoreArgs a;
  a.T = T;
  a.H = H;
  a.V = V;
  a.id_tiles = static_cast<int>(ids);
  a.tok_tiles = static_cast<int>(tok_tiles);
  a.rows = rows;
  a.targets = targets;
  a.scale = static_cast<float>(logit_scale * 1.4426950408889634 * (1.0 + mk::kTruncPerStep * ((H + 15) / 16)));
  a.part = static_cast<float*>(workspace);
  a.ld_part = ld_part(T);
  a.target_logit = reinterpret_cast<float*>(static_cast<char*>(workspace) + part_bytes(T, V));
  a.err = d.err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tiles = a.id_tiles * a.tok_tiles, units = std::min(pair ? pairs : d.sm_count, tiles);
  a.parts = a.tok_tiles == 1 ? units : a.id_tiles;
  if (pair)
    MK_TRY(launch_k_pair(mk::score_tokens_kernel<true>, dim3(2 * units), dim3(mk::SC_THREADS),
                         mk::SC_SMEM_BYTES, st, true, mh, mw, a));
  else
    MK_TRY(launch_k(mk::score_tokens_kernel<false>, dim3(units), dim3(mk::SC_THREADS),
                    mk::SC_SMEM_BYTES, st, true, mh, mw, a));
  // (many tokens fill the GPU with fewer slices each: 8192 tokens' 287 parts join in 11 us
  // with 256 threads a CTA, in 13.5 with 512, 19 with 1024, 16 with 128)
  const int join = T > d.sm_count * 16 ? 256 : mk::SJ_THREADS;
  return launch_k(mk::score_join_kernel, dim3((T + mk::SJ_TOKENS - 1) / mk::SJ_TOKENS), dim3(join), 0, st, true, a, logprobs,
                  entropy);
}

}  // extern "C"

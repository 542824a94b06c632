// C ABI of token scoring: log-probabilities of given tokens from logits or from hidden rows.
// See include/minicpm5_mk.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "mk_host.cuh"
#include "mk_score.cuh"

namespace {

using mk::aligned16;
using mk::HostDevice;
using mk::launch_k;

constexpr int kScoreParts = 16;

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

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
  if (logits_bits == 32)
    return launch_k(mk::token_logprobs_kernel<float>, dim3(T), dim3(mk::TL_THREADS), 0, st, true,
                    static_cast<const float*>(logits), V, static_cast<long long>(ld), targets, top_k, logprobs, entropy,
                    ranks, top_ids, top_logprobs);
  return launch_k(mk::token_logprobs_kernel<__nv_bfloat16>, dim3(T), dim3(mk::TL_THREADS), 0, st, true,
                  static_cast<const __nv_bfloat16*>(logits), V, static_cast<long long>(ld), targets, top_k, logprobs,
                  entropy, ranks, top_ids, top_logprobs);
}

mk_status mk_score_tokens_workspace(int32_t T, int32_t H, int32_t V, size_t* bytes) {
  if (!bytes) return MK_ERR_BAD_ARG;
  if (T < 0 || H <= 0 || H % 8 || V <= 0) return MK_ERR_BAD_SHAPE;
  *bytes = align256(static_cast<size_t>(T) * kScoreParts * sizeof(mk::ScorePart)) + static_cast<size_t>(T) * sizeof(float);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  mk::ScorePart* part = static_cast<mk::ScorePart*>(workspace);
  float* tl = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                       align256(static_cast<size_t>(T) * kScoreParts * sizeof(mk::ScorePart)));
  const size_t smem = static_cast<size_t>(mk::SC_TOK) * H * sizeof(float);
  MK_CUDA(cudaFuncSetAttribute(mk::score_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  MK_TRY(launch_k(mk::score_tokens_kernel, dim3((T + mk::SC_TOK - 1) / mk::SC_TOK, kScoreParts), dim3(mk::SC_THREADS), smem,
                  st, true, static_cast<const __nv_bfloat16*>(h), T, H, static_cast<long long>(ld),
                  static_cast<const __nv_bfloat16*>(lm_head), V, targets, logit_scale, part, tl));
  return launch_k(mk::score_join_kernel, dim3((T + 127) / 128), dim3(128), 0, st, true,
                  static_cast<const mk::ScorePart*>(part), kScoreParts, T, V, targets, static_cast<const float*>(tl),
                  logprobs, entropy);
}

}  // extern "C"

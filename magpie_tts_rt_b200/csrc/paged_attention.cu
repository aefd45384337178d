// Attention over the paged key/value cache (include/magpie_tts_rt_b200.h,
// group 7): checks of the calls, and the choice of kernel.  Single tokens go
// to the step kernel (paged_step.cu), runs of tokens to the tensor-core
// kernel (paged_prompt.cu).
#include <cmath>

#include "paged_attention.cuh"

namespace mtt {

size_t paged_attention_workspace(const mtt_b200_paged_cache_t& c, int q_heads, int rows) {
  return step_workspace(c, q_heads) + prompt_workspace(c, q_heads, rows);
}

}  // namespace mtt

using namespace mtt;

extern "C" {

int mtt_b200_launch_paged_attention(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  PagedCache c;
  void* space = nullptr;
  if (args == nullptr || !paged_cache_view(cache, &c) || args->layer < 0 || args->layer >= c.layers ||
      args->q_heads < 1 || args->q_heads % c.kv_heads != 0 || args->q_heads / c.kv_heads > kCacheMaxGroup ||
      args->rows < 0 || args->rows > kCacheMaxRows || args->window < 0 || args->sinks < 0 ||
      !(args->scale > 0.f) || !std::isfinite(args->scale))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (args->rows == 0) return MTT_B200_STATUS_OK;
  if (args->q == nullptr || args->out == nullptr || !aligned16(args->q) || !aligned16(args->out) ||
      args->q_row_stride % 8 != 0 || args->out_row_stride % 8 != 0 ||
      (args->offsets == nullptr && args->rows > c.slots) ||
      (args->key_mask != nullptr && args->mask_stride < static_cast<int64_t>(c.table_pages) * c.page_size) ||
      (space = paged_attention_space(*cache, args->q_heads, args->rows, workspace, workspace_bytes)) == nullptr)
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  Attend a{args->layer, args->q_heads, args->q_heads / c.kv_heads, args->rows, args->window, args->sinks, args->scale * 1.4426950408889634f,
           static_cast<const uint16_t*>(args->q), args->q_row_stride, static_cast<uint16_t*>(args->out),
           args->out_row_stride, args->lse, args->offsets, args->key_mask, args->mask_stride};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.offsets == nullptr) return cache_call_status(launch_step(c, cache->dtype, a, space, s));
  return cache_call_status(
      launch_prompt(c, cache->dtype, a, static_cast<char*>(space) + step_workspace(*cache, args->q_heads), s));
}

}  // extern "C"

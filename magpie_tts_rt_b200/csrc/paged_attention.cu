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

namespace {

// Checks what every attention call's arguments have to fulfil.
bool attend_args(const PagedCache& c, const mtt_b200_cache_attention_t* args, Attend* a) {
  if (args == nullptr || args->layer < 0 || args->layer >= c.layers || args->q_heads < 1 ||
      args->q_heads % c.kv_heads != 0 || args->q_heads / c.kv_heads > kCacheMaxGroup || args->rows < 0 ||
      args->rows > kCacheMaxRows || args->window < 0 || args->sinks < 0 || !(args->scale > 0.f) ||
      !std::isfinite(args->scale))
    return false;
  if (args->rows > 0 &&
      (args->q == nullptr || args->out == nullptr || !aligned16(args->q) || !aligned16(args->out) ||
       args->q_row_stride % 8 != 0 || args->out_row_stride % 8 != 0 ||
       (args->offsets == nullptr && args->rows > c.slots) ||
       (args->key_mask != nullptr && args->mask_stride < static_cast<int64_t>(c.table_pages) * c.page_size)))
    return false;
  *a = Attend{args->layer, args->q_heads, args->q_heads / c.kv_heads, args->rows, args->window, args->sinks,
              args->scale * 1.4426950408889634f, static_cast<const uint16_t*>(args->q), args->q_row_stride,
              static_cast<uint16_t*>(args->out), args->out_row_stride, args->lse, args->offsets, args->key_mask,
              args->mask_stride};
  return true;
}

// Keys and values of all members' prefixes from which on the prefix pass pays:
// it adds about 20 us of launches and dependent steps, while those bytes read
// slot by slot come at 4 to 9 TB/s, mostly from L2.  Measured, each slot on its
// own against shared: 101 MB (12 heads of 64, 1024 tokens, 32 slots) 19 against
// 30 us; 134 MB (8 of 128, 16384, 2) 38 / 62; 302 MB (12 of 64, 192, 512) 43 / 34;
// 403 MB (12 of 64, 16384, 8) 66 / 60; 2.1 GB (8 of 128, 4096, 128) 244 / 43.
constexpr double kSharedBytesWorth = 220e6;

// Bytes of the prefix pass's results: base and state (SharedPrefix).
size_t base_bytes(const mtt_b200_paged_cache_t& c) { return (4 * static_cast<size_t>(c.slots) + 255) / 256 * 256; }
size_t state_bytes(const mtt_b200_paged_cache_t& c, int q_heads) {
  return (static_cast<size_t>(c.slots) * q_heads * (c.head_dim + 4) * 4 + 255) / 256 * 256;
}

int attend(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args, void* workspace,
           size_t workspace_bytes, const Waits& waits, void* stream) {
  PagedCache c;
  Attend a;
  if (!paged_cache_view(cache, &c) || !attend_args(c, args, &a)) return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (a.rows == 0) return MTT_B200_STATUS_OK;
  void* space = paged_attention_space(*cache, a.q_heads, a.rows, workspace, workspace_bytes);
  if (space == nullptr) return MTT_B200_STATUS_INVALID_ARGUMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.offsets == nullptr) return cache_call_status(launch_step(c, cache->dtype, a, SharedPrefix{}, space, s));
  return cache_call_status(
      launch_prompt(c, cache->dtype, a, static_cast<char*>(space) + step_workspace(*cache, a.q_heads), waits, s));
}

int attend_shared(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                  const mtt_b200_prefix_groups_t* groups, void* workspace, size_t workspace_bytes,
                  const Waits& waits, void* stream) {
  PagedCache c;
  Attend a;
  if (!paged_cache_view(cache, &c) || !attend_args(c, args, &a) || a.offsets != nullptr || a.key_mask != nullptr ||
      groups == nullptr || groups->n_groups < 0 || groups->n_groups > c.slots || groups->n_members < 0 ||
      groups->n_members > kCacheMaxRows)
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (a.rows == 0) return MTT_B200_STATUS_OK;
  void* space = paged_attention_space(*cache, a.q_heads, groups->n_members, workspace, workspace_bytes);
  const size_t plain = (mtt_b200_paged_cache_workspace_size(cache, a.q_heads, groups->n_members) + 255) / 256 * 256;
  if (space == nullptr || workspace_bytes < plain + base_bytes(*cache) + state_bytes(*cache, a.q_heads))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  SharedPrefix shared{};
  const double shared_bytes = 4.0 * groups->shared_tokens * c.kv_heads * c.head_dim;
  if (groups->n_groups > 0 && groups->n_members > 0 &&
      (groups->shared_tokens <= 0 || shared_bytes >= kSharedBytesWorth)) {
    if (groups->voice == nullptr || groups->tokens == nullptr || groups->offsets == nullptr ||
        groups->members == nullptr)
      return MTT_B200_STATUS_INVALID_ARGUMENT;
    int32_t* base = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + plain);
    float* state = reinterpret_cast<float*>(static_cast<char*>(workspace) + plain + base_bytes(*cache));
    const cudaError_t e = launch_prefix(c, cache->dtype, a, *groups, base, state,
                                        static_cast<char*>(space) + step_workspace(*cache, a.q_heads), waits, s);
    if (e != cudaSuccess) return cache_call_status(e);
    shared.base = base;
    shared.state = state;
  }
  return cache_call_status(launch_step(c, cache->dtype, a, shared, space, s));
}

}  // namespace

extern "C" {

int mtt_b200_launch_paged_attention(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  return attend(cache, args, workspace, workspace_bytes, Waits{}, stream);
}

size_t mtt_b200_paged_shared_workspace_size(const mtt_b200_paged_cache_t* cache, int32_t q_heads, int32_t n_members) {
  const size_t plain = mtt_b200_paged_cache_workspace_size(cache, q_heads, n_members);
  return plain == 0 ? 0 : (plain + 255) / 256 * 256 + base_bytes(*cache) + state_bytes(*cache, q_heads);
}

int mtt_b200_launch_paged_attention_shared(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                                           const mtt_b200_prefix_groups_t* groups, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  return attend_shared(cache, args, groups, workspace, workspace_bytes, Waits{}, stream);
}

int mtt_b200_launch_test_paged_attention(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                                         const mtt_b200_prefix_groups_t* groups, uint32_t wait_ns, int32_t starve,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  const Waits waits{wait_ns, Waits{}.tile_ns, starve != 0};
  return groups == nullptr ? attend(cache, args, workspace, workspace_bytes, waits, stream)
                           : attend_shared(cache, args, groups, workspace, workspace_bytes, waits, stream);
}

}  // extern "C"

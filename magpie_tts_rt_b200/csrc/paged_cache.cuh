// Device view of the paged key/value cache (include/magpie_tts_rt_b200.h,
// group 7) and the helpers its upkeep and attention kernels share.
#pragma once

#include <cuda_fp16.h>

#include "../../include/magpie_tts_rt_b200.h"
#include "common.cuh"

namespace mtt {

constexpr int kCacheMaxSlots = 16384;
constexpr int kCacheMaxGroup = 64;  // query heads per key head
constexpr int kCacheMaxRows = 1 << 22;  // query rows of a call

struct PagedCache {
  int pages, layers, kv_heads, page_size, page_shift, head_dim, slots, table_pages;
  int64_t kv_elems;  // elements of one layer's keys (or values) in a page
  uint16_t* pool;
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int32_t* status;
  int32_t* live;
  int32_t* refused;

  // tokens of a slot, as far as its table can hold them
  __device__ __forceinline__ int length(int slot) const {
    const int n = lengths[slot];
    return max(0, min(n, table_pages << page_shift));
  }
  __device__ __forceinline__ bool is_page(int p) const {
    return static_cast<unsigned>(p) < static_cast<unsigned>(pages);
  }
  // first element of (page, layer, keys or values)
  __device__ __forceinline__ int64_t block(int page, int layer, int kv) const {
    return ((static_cast<int64_t>(page) * layers + layer) * 2 + kv) * kv_elems;
  }
};

// The first statement of every kernel here (before its first global access):
// the next launch on the stream may be scheduled from now on, and waits in
// turn for this grid; this one waits for the launch before it.
__device__ __forceinline__ void take_turn() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  wait_prior_grid();
}

// Checks a caller's cache and fills the device view; false for bad arguments.
bool paged_cache_view(const mtt_b200_paged_cache_t* c, PagedCache* out);

// Workspace bytes of the attention calls (they follow the upkeep's words).
size_t paged_attention_workspace(const mtt_b200_paged_cache_t& c, int q_heads, int rows);

// Start of the attention's part of a workspace; null when the workspace is too small.
void* paged_attention_space(const mtt_b200_paged_cache_t& c, int q_heads, int rows, void* workspace, size_t bytes);

// SMs of the current device (0: cannot be queried).
int cache_sm_count();

// MTT_B200_STATUS_* of a sequence of launches.
int cache_call_status(cudaError_t e);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace mtt

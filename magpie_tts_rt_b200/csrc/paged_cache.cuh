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
  int dtype, bits;   // MTT_B200_DTYPE_*; bits a value in the pool: 16 or 4
  int64_t kv_elems;  // one layer's keys (or values) in a page, in units of 16 bits
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
  // first unit of (page, layer, keys or values)
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

// Where row `row` of a call's rows belongs: rows [offsets[i], offsets[i + 1])
// are the last tokens of slot i, or, without offsets, row i that of slot i.
struct RowPlace {
  int slot, pos;  // pos -1: it has no token
  int unfit;      // the slot's offsets: 0 fit, 1 name more rows than it has tokens, 2 lead out of the rows
  // For all lanes of a warp.  32 offsets are looked at in each step of the search:
  // 512 slots take two dependent loads, not nine.
  __device__ __forceinline__ RowPlace(const PagedCache& c, const int32_t* offsets, int rows, int row)
      : slot(row), pos(-1), unfit(0) {
    int count = 1, first = row;
    if (offsets != nullptr) {
      // the slot with offsets[slot] <= row < offsets[slot + 1]
      const int lane = threadIdx.x & 31;
      int lo = 0, hi = c.slots;
      while (lo < hi) {
        const int step = (hi - lo + 31) >> 5, at = lo + (lane + 1) * step;
        const uint32_t past = __ballot_sync(0xffffffffu, at > hi || offsets[at] > row);
        if (past == 0) {
          lo = hi;
          break;
        }
        const int k = __ffs(past) - 1;
        hi = min(hi, lo + (k + 1) * step - 1);
        lo += k * step;
      }
      slot = lo;
      if (slot >= c.slots) return;
      first = offsets[slot];
      const int end = offsets[slot + 1];
      count = end - first;
      if (first < 0 || first > row || end > rows) {
        unfit = 2;
        return;
      }
    }
    const int len = c.length(slot);
    if (offsets == nullptr && len == 0) return;
    if (count > len) {
      unfit = 1;
      return;
    }
    pos = len - count + row - first;
  }
};

// Checks a caller's cache and fills the device view; false for bad arguments.
bool paged_cache_view(const mtt_b200_paged_cache_t* c, PagedCache* out);

// Whether the rows of a store or load fit the cache and the calls' rules.
bool rows_checked(const PagedCache& c, const mtt_b200_cache_rows_t* rows);

// store of a 4-bit cache, with arguments that have been checked.
int store4(const PagedCache& c, const mtt_b200_cache_rows_t& rows, cudaStream_t stream);

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

// What the attention kernels over the paged cache share: arguments, 16-bit
// type helpers, and the base-2 softmax arithmetic.
#pragma once

#include "paged_cache.cuh"
#include "ptx.cuh"

namespace mtt {

struct Attend {
  int layer, q_heads, group, rows, window, sinks;
  float scale2;  // scale * log2(e): scores are kept in base 2
  const uint16_t* q;
  int64_t q_row;
  uint16_t* out;
  int64_t out_row;
  float* lse;
  const int32_t* offsets;
  const bool* key_mask;
  int64_t mask_stride;
};

// What the prefix pass leaves for the step kernel.
struct SharedPrefix {
  const int32_t* base;  // [rows] tokens of the slot's prefix that are already attended to (0: none); null: no groups
  const float* state;   // [slots][q_heads][head_dim + 4]: weighted values, maximum (base 2), sum
};

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // the pair, and what its rounding leaves of the two
  static __device__ __forceinline__ uint2 split(float lo, float hi) {
    const uint32_t h = pack(lo, hi);
    return make_uint2(h, pack(lo - __uint_as_float(h << 16), hi - __uint_as_float(h & 0xffff0000u)));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Half16<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint2 split(float lo, float hi) {
    const uint32_t h = pack(lo, hi);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return make_uint2(h, pack(lo - f.x, hi - f.y));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Transpose of an 8 x 8 matrix of 16-bit values held one row pair per thread.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The 16-key tiles of a slot that a query at its last token may see, from
// token `base` (a multiple of 16) on: first the tiles with sinks, then the
// window's.
struct SeenTiles {
  int len, low;             // keys >= low or < sinks are in reach
  int sink0, sink_n, win0;  // tile numbers
  int n;                    // tiles in all
  __device__ __forceinline__ SeenTiles(int length, int window, int sinks, int base) {
    len = length;
    low = window > 0 && window < len ? len - window : 0;
    sink0 = base >> 4;
    const int end = (len + 15) >> 4;
    const int sink_end = low > base ? (min(sinks, len) + 15) >> 4 : sink0;
    sink_n = max(0, min(sink_end, end) - sink0);
    win0 = max(max(low, base) >> 4, sink0 + sink_n);
    n = len > base ? sink_n + max(0, end - win0) : 0;
  }
  __device__ __forceinline__ int tile(int t) const { return t < sink_n ? sink0 + t : win0 + t - sink_n; }
};

// Workspace of the single-token attention.
size_t step_workspace(const mtt_b200_paged_cache_t& c, int q_heads);
cudaError_t launch_step(const PagedCache& c, int dtype, const Attend& a, const SharedPrefix& shared, void* space,
                        cudaStream_t stream);

// How long the prompt kernel's waits may last: ns, and tile_ns for each key tile
// of a CTA's share (which takes it some 2 us).
struct Waits {
  uint32_t ns = 200000000, tile_ns = 50000;
  bool starve = false;  // tests: no key tile ever arrives
};

// Workspace of the prompt attention for calls of up to `rows` query rows.
size_t prompt_workspace(const mtt_b200_paged_cache_t& c, int q_heads, int rows);
cudaError_t launch_prompt(const PagedCache& c, int dtype, const Attend& a, void* space, const Waits& waits,
                          cudaStream_t stream);

// The prefix pass of the shared-prefix attention: fills base and state.
cudaError_t launch_prefix(const PagedCache& c, int dtype, const Attend& a, const mtt_b200_prefix_groups_t& groups,
                          int32_t* base, float* state, void* space, const Waits& waits, cudaStream_t stream);

}  // namespace mtt

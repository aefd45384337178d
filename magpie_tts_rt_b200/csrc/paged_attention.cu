// Attention over the paged key/value cache (include/magpie_tts_rt_b200.h, group 7).
#include "paged_attention.cuh"

namespace mtt {
namespace {

// One warp per (row, query head): keys one after the other, a running
// maximum and sum, the head's dimensions over the lanes.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(PagedCache c, Attend a) {
  wait_prior_grid();
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int row = static_cast<int>(w / a.q_heads), h = static_cast<int>(w % a.q_heads);
  if (row >= a.rows) return;
  int slot = row, count = 1, first = row;
  bool ok = true;
  if (a.offsets != nullptr) {
    int lo = 0, hi = c.slots;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    slot = lo;
    ok = slot < c.slots;
    if (ok) {
      first = a.offsets[slot];
      count = a.offsets[slot + 1] - first;
      ok = first >= 0 && first <= row && a.offsets[slot + 1] <= a.rows;
    }
  }
  const int len = ok ? c.length(slot) : 0;
  if (count > len) ok = false;
  const int p = len - count + row - first;
  float q[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = Half16<T>::to_f(a.q[row * a.q_row + static_cast<int64_t>(h) * D + lane * E + e]);
    acc[e] = 0.f;
  }
  float m = -CUDART_INF_F, l = 0.f;
  for (int j = 0; ok && j <= p; ++j) {
    if (a.window > 0 && p - j >= a.window && j >= a.sinks) continue;
    if (a.key_mask != nullptr && !a.key_mask[slot * a.mask_stride + j]) continue;
    const int page = c.table[static_cast<int64_t>(slot) * c.table_pages + (j >> c.page_shift)];
    if (!c.is_page(page)) continue;
    const int64_t at = (static_cast<int64_t>(h / a.group) * c.page_size + (j & (c.page_size - 1))) * D + lane * E;
    const uint16_t* k = c.pool + c.block(page, a.layer, 0) + at;
    const uint16_t* v = c.pool + c.block(page, a.layer, 1) + at;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], Half16<T>::to_f(k[e]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale2;
    const float mn = fmaxf(m, s);
    const float keep = m == mn ? 1.f : ex2(m - mn), x = ex2(s - mn);
    l = l * keep + x;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(x, Half16<T>::to_f(v[e]), acc[e] * keep);
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[row * a.out_row + static_cast<int64_t>(h) * D + lane * E + e] = Half16<T>::one(acc[e] * inv);
  if (lane == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(row) * a.q_heads + h] = (m + log2f(l)) * kLn2;
}

}  // namespace

size_t paged_attention_workspace(const mtt_b200_paged_cache_t& c, int q_heads) { return step_workspace(c, q_heads); }

}  // namespace mtt

using namespace mtt;

extern "C" {

int mtt_b200_launch_paged_attention(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_attention_t* args,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  PagedCache c;
  void* space = nullptr;
  if (args == nullptr || !paged_cache_view(cache, &c) || args->layer < 0 || args->layer >= c.layers ||
      args->q_heads < 1 || args->q_heads % c.kv_heads != 0 || args->q_heads / c.kv_heads > kCacheMaxGroup ||
      args->rows < 0 || args->window < 0 || args->sinks < 0)
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (args->rows == 0) return MTT_B200_STATUS_OK;
  if (args->q == nullptr || args->out == nullptr || !aligned16(args->q) || !aligned16(args->out) ||
      args->q_row_stride % 8 != 0 || args->out_row_stride % 8 != 0 ||
      (args->offsets == nullptr && args->rows > c.slots) ||
      (args->key_mask != nullptr && args->mask_stride < static_cast<int64_t>(c.table_pages) * c.page_size) ||
      (space = paged_attention_space(*cache, args->q_heads, workspace, workspace_bytes)) == nullptr)
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  Attend a{args->layer, args->q_heads, args->q_heads / c.kv_heads, args->rows, args->window, args->sinks, args->scale * 1.4426950408889634f,
           static_cast<const uint16_t*>(args->q), args->q_row_stride, static_cast<uint16_t*>(args->out),
           args->out_row_stride, args->lse, args->offsets, args->key_mask, args->mask_stride};
  if (a.offsets == nullptr)
    return cache_call_status(launch_step(c, cache->dtype, a, space, static_cast<cudaStream_t>(stream)));
  const int64_t warps = static_cast<int64_t>(args->rows) * args->q_heads;
  auto* kernel = cache->dtype == MTT_B200_DTYPE_BF16
                     ? (c.head_dim == 64 ? attend_rows_kernel<__nv_bfloat16, 64> : attend_rows_kernel<__nv_bfloat16, 128>)
                     : (c.head_dim == 64 ? attend_rows_kernel<__half, 64> : attend_rows_kernel<__half, 128>);
  return cache_call_status(launch_serialized(kernel, dim3(static_cast<unsigned>((warps + 3) / 4)), dim3(128), 0,
                                             static_cast<cudaStream_t>(stream), c, a));
}

}  // extern "C"

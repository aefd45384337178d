// Rows into and out of the paged cache beside paged_cache.cu's 16-bit store:
// store4 writes them in 4 bits, load reads them back.
//
// A token's head is held by head_dim / 16 lanes, 16 dims each as two 16-byte
// pieces, so that a group's 64 dims lie in 4 lanes (head_dim 64: all of them) or
// one piece of each of 8: minimum and maximum take two or three shuffles in
// packed 16-bit pairs.  HBM bounds both kernels.
#include "cache4.cuh"

namespace mtt {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;

struct RowsArgs {
  int layer, n_layers, rows, chunks;
  uint16_t *k, *v;
  int64_t k_row, v_row, k_layer, v_layer;
  const int32_t* offsets;
};

// A warp's unit: part `chunk` of a row's (layer, keys or values, head) items.
template <int D>
struct RowUnit {
  static constexpr int L = D / 16, H = 32 / L;  // lanes of a head, heads of a warp
  int row, i0, i1;
  __device__ __forceinline__ RowUnit(const PagedCache& c, const RowsArgs& in) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
    row = static_cast<int>(unit / in.chunks);
    const int chunk = static_cast<int>(unit % in.chunks);
    const int items = 2 * in.n_layers * c.kv_heads, each = ((items + in.chunks - 1) / in.chunks + H - 1) / H * H;
    i0 = chunk * each;
    i1 = min(items, i0 + each);
  }
};

// An item's first element in k or v, and its place in the cache.
struct RowItem {
  int kv, layer, head;
  uint16_t* at;
  __device__ __forceinline__ RowItem(const PagedCache& c, const RowsArgs& in, int row, int item) {
    const int b = item / c.kv_heads;
    head = item - b * c.kv_heads;
    kv = b & 1;
    layer = b >> 1;
    at = (kv ? in.v + row * in.v_row + layer * in.v_layer : in.k + row * in.k_row + layer * in.k_layer) +
         static_cast<int64_t>(head) * c.head_dim;
    layer += in.layer;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowsThreads) store4_kernel(PagedCache c, RowsArgs in) {
  using U = RowUnit<D>;
  take_turn();
  const U u(c, in);
  if (u.row >= in.rows) return;
  const int lane = threadIdx.x & 31, t = lane % U::L;
  const RowPlace at(c, in.offsets, in.rows, u.row);
  if (at.pos < 0 && at.unfit == 0) return;
  if (at.unfit != 2 && c.refused != nullptr && c.refused[at.slot] != 0) return;  // its last tokens are not the rows'
  int bad = at.unfit != 0 ? 1 : 0, page = -1;
  if (bad == 0) {
    page = c.table[static_cast<int64_t>(at.slot) * c.table_pages + (at.pos >> c.page_shift)];
    if (!c.is_page(page) || c.refs[page] > 1) bad = 3;
  }
  if (bad != 0) {
    if (lane == 0 && c.status != nullptr) c.status[at.slot] = bad;
    return;
  }
  const int in_page = at.pos & (c.page_size - 1);
  for (int i0 = u.i0; i0 < u.i1; i0 += U::H) {
    const int i = i0 + lane / U::L;
    const bool on = i < u.i1;
    const RowItem item(c, in, u.row, on ? i : i0);
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(item.at) + t);
    const uint4 b = __ldcs(reinterpret_cast<const uint4*>(item.at) + t + U::L);
    unsigned char* block = block4(c, page, item.layer, item.kv, item.head);
    Extent4<T> e = Extent4<T>::of(a);
    if constexpr (D == 64) {
      e.take(b);
      e.join(U::L);
      const Pair4<T> p(e);
      if (on) {
        *codes_at(c, block, in_page, t) = p.codes(a);
        *codes_at(c, block, in_page, t + U::L) = p.codes(b);
        if (t == 0) *pair_at(c, block, in_page, 0) = p.bits;
      }
    } else {
      Extent4<T> f = Extent4<T>::of(b);
      e.join(U::L);
      f.join(U::L);
      const Pair4<T> p(e), q(f);
      if (on) {
        *codes_at(c, block, in_page, t) = p.codes(a);
        *codes_at(c, block, in_page, t + U::L) = q.codes(b);
        if (t < 2) *pair_at(c, block, in_page, t) = t == 0 ? p.bits : q.bits;
      }
    }
  }
}

template <typename T, int D, int Bits>
__global__ void __launch_bounds__(kRowsThreads) load_kernel(PagedCache c, RowsArgs in) {
  using U = RowUnit<D>;
  take_turn();
  const U u(c, in);
  if (u.row >= in.rows) return;
  const int lane = threadIdx.x & 31, t = lane % U::L;
  const RowPlace at(c, in.offsets, in.rows, u.row);
  const int page = at.pos < 0 ? -1 : c.table[static_cast<int64_t>(at.slot) * c.table_pages + (at.pos >> c.page_shift)];
  const bool there = c.is_page(page);
  const int in_page = at.pos & (c.page_size - 1);
  for (int i = u.i0 + lane / U::L; i < u.i1; i += U::H) {
    const RowItem item(c, in, u.row, i);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (there) {
      if constexpr (Bits == 4) {
        unsigned char* block = block4(c, page, item.layer, item.kv, item.head);
        a = values4<T>(*codes_at(c, block, in_page, t), *pair_at(c, block, in_page, t / 8));
        b = values4<T>(*codes_at(c, block, in_page, t + U::L), *pair_at(c, block, in_page, (t + U::L) / 8));
      } else {
        const uint16_t* src = c.pool + c.block(page, item.layer, item.kv) +
                              (static_cast<int64_t>(item.head) * c.page_size + in_page) * D;
        a = *(reinterpret_cast<const uint4*>(src) + t);
        b = *(reinterpret_cast<const uint4*>(src) + t + U::L);
      }
    }
    __stcs(reinterpret_cast<uint4*>(item.at) + t, a);
    __stcs(reinterpret_cast<uint4*>(item.at) + t + U::L, b);
  }
}

template <typename Run>
cudaError_t for_type_and_dim(const PagedCache& c, Run run) {
  using std::integral_constant;
  auto dim = [&](auto type) {
    return c.head_dim == 64 ? run(type, integral_constant<int, 64>{}) : run(type, integral_constant<int, 128>{});
  };
  return c.dtype == MTT_B200_DTYPE_BF16 ? dim(__nv_bfloat16{}) : dim(__half{});
}

RowsArgs rows_args(const PagedCache& c, const mtt_b200_cache_rows_t& r) {
  RowsArgs in{r.layer, r.n_layers, r.rows, 1, static_cast<uint16_t*>(const_cast<void*>(r.k)),
              static_cast<uint16_t*>(const_cast<void*>(r.v)), r.k_row_stride, r.v_row_stride, r.k_layer_stride,
              r.v_layer_stride, r.offsets};
  // few rows: a row's items are dealt to several warps
  const int heads = 32 / (c.head_dim / 16), passes = (2 * r.n_layers * c.kv_heads + heads - 1) / heads;
  const int sms = cache_sm_count();
  in.chunks = std::max(1, std::min(passes, (sms * 16 + r.rows - 1) / r.rows));
  return in;
}

dim3 rows_grid(const RowsArgs& in) {
  return dim3(static_cast<unsigned>((static_cast<int64_t>(in.rows) * in.chunks + kRowsWarps - 1) / kRowsWarps));
}

}  // namespace

int store4(const PagedCache& c, const mtt_b200_cache_rows_t& rows, cudaStream_t stream) {
  const RowsArgs in = rows_args(c, rows);
  return cache_call_status(for_type_and_dim(c, [&](auto type, auto dim) {
    return launch_serialized(store4_kernel<decltype(type), decltype(dim)::value>, rows_grid(in), dim3(kRowsThreads), 0, stream,
                             c, in);
  }));
}

bool rows_checked(const PagedCache& c, const mtt_b200_cache_rows_t* rows) {
  return rows->rows >= 0 && rows->layer >= 0 && rows->n_layers >= 1 && rows->n_layers <= c.layers - rows->layer &&
         (rows->rows == 0 ||
          (rows->k != nullptr && rows->v != nullptr && aligned16(rows->k) && aligned16(rows->v) &&
           (rows->k_row_stride | rows->v_row_stride | rows->k_layer_stride | rows->v_layer_stride) % 8 == 0 &&
           (rows->offsets != nullptr || rows->rows <= c.slots)));
}

}  // namespace mtt

using namespace mtt;

extern "C" {

int mtt_b200_launch_paged_cache_load(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_rows_t* rows, void* stream) {
  PagedCache c;
  if (rows == nullptr || !paged_cache_view(cache, &c) || !rows_checked(c, rows)) return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (rows->rows == 0) return MTT_B200_STATUS_OK;
  const RowsArgs in = rows_args(c, *rows);
  return cache_call_status(for_type_and_dim(c, [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    return launch_serialized(c.bits == 4 ? load_kernel<T, D, 4> : load_kernel<T, D, 16>, rows_grid(in), dim3(kRowsThreads), 0,
                             static_cast<cudaStream_t>(stream), c, in);
  }));
}

}  // extern "C"

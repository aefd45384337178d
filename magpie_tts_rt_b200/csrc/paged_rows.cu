// Rows into and out of the paged cache beside paged_cache.cu's 16-bit store:
// store4 writes them in 4 bits, load reads them back.
//
// A token's head is held by head_dim / 16 lanes, 16 dims each (32 bytes, in one
// load where the rows allow it), so that a group's 64 dims lie in 4 lanes: minimum and
// maximum take two shuffles in packed 16-bit pairs.  HBM bounds both kernels as long
// as instructions stay few (store4: the schedulers are busy 78% of the time), and a
// load's as long as enough of them are on their way.  16,892 rows (prompts of 96 slots) of 8
// layers, 8 heads of 128, in a graph: stored in 142 us (709 MB, 5.0 TB/s), loaded in 120
// (5.9 TB/s; one head of a lane ahead instead of four 141), from 16 bits 173 (1.11 GB, 6.4
// TB/s; one ahead 172, four 179).
#include "cache4.cuh"

namespace mtt {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;
template <int Bits>
constexpr int kLoadAhead = Bits == 4 ? 4 : 2;  // heads of a load that a lane has on their way

struct RowsArgs {
  int layer, n_layers, rows, chunks;
  bool wide;  // rows of k and v are 32-byte aligned
  uint16_t *k, *v;
  int64_t k_row, v_row, k_layer, v_layer;
  const int32_t* offsets;
};

// A warp's unit: part `chunk` of a row's (layer, keys or values, head) items, a head
// for each D / 16 lanes at a time.
template <int D>
struct RowUnit {
  static constexpr int L = D / 16, H = 32 / L;  // lanes of a head, heads of a warp
  int row, i, end;                              // the lane's item
  int block, head;                              // item i: 2 * layer + (keys or values), and head
  int blocks_on, heads_on;                      // from an item to the lane's next
  __device__ __forceinline__ RowUnit(const PagedCache& c, const RowsArgs& in) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
    row = static_cast<int>(unit / in.chunks);
    const int chunk = static_cast<int>(unit % in.chunks);
    const int items = 2 * in.n_layers * c.kv_heads, each = ((items + in.chunks - 1) / in.chunks + H - 1) / H * H;
    i = chunk * each + (threadIdx.x & 31) / L;
    end = min(items, (chunk + 1) * each);
    block = i / c.kv_heads;
    head = i - block * c.kv_heads;
    blocks_on = H / c.kv_heads;
    heads_on = H - blocks_on * c.kv_heads;
  }
  __device__ __forceinline__ bool on() const { return i < end; }
  __device__ __forceinline__ void next(const PagedCache& c) {
    i += H;
    block += blocks_on;
    head += heads_on;
    if (head >= c.kv_heads) {
      head -= c.kv_heads;
      ++block;
    }
  }
  // the lane's 16 dims of the item in k or v (`k`, `v`: those of the row's first head and layer)
  __device__ __forceinline__ uint16_t* at(uint16_t* k, uint16_t* v, const RowsArgs& in) const {
    return ((block & 1) != 0 ? v + (block >> 1) * in.v_layer : k + (block >> 1) * in.k_layer) + static_cast<int64_t>(head) * D;
  }
  // the item's keys or values in its page (`first`: those of the call's first layer), all heads
  __device__ __forceinline__ unsigned char* place(const PagedCache& c, unsigned char* first) const {
    return first + static_cast<uint64_t>(static_cast<uint32_t>(block)) * static_cast<uint64_t>(2 * c.kv_elems);
  }
};

struct Piece {
  uint4 a, b;  // 16 values
  __device__ __forceinline__ void load(const uint16_t* p, bool wide) {
    if (wide) {
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                   : "l"(p));
    } else {
      a = __ldcs(reinterpret_cast<const uint4*>(p));
      b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
    }
  }
  __device__ __forceinline__ void store(uint16_t* p, bool wide) const {
    if (wide) {
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                   "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                   : "memory");
    } else {
      __stcs(reinterpret_cast<uint4*>(p), a);
      __stcs(reinterpret_cast<uint4*>(p) + 1, b);
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowsThreads) store4_kernel(PagedCache c, RowsArgs in) {
  using U = RowUnit<D>;
  take_turn();
  U u(c, in);
  if (u.row >= in.rows) return;
  const int lane = threadIdx.x & 31, t = lane % U::L;
  uint16_t *k = in.k + u.row * in.k_row + 16 * t, *v = in.v + u.row * in.v_row + 16 * t;
  Piece next{};
  if (u.on()) next.load(u.at(k, v, in), in.wide);
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
  const int in_page = at.pos & (c.page_size - 1), head_bytes = block4_bytes(c);
  const int codes = in_page * (D / 2) + 8 * t, pair = block4_codes(c) + (in_page * (D / kGroup4) + t / 4) * 4;
  unsigned char* first = reinterpret_cast<unsigned char*>(c.pool + c.block(page, in.layer, 0));
  while (__any_sync(0xffffffffu, u.on())) {
    const Piece x = next;
    const bool on = u.on();
    unsigned char* to = u.place(c, first) + static_cast<int64_t>(u.head) * head_bytes;
    u.next(c);
    if (u.on()) next.load(u.at(k, v, in), in.wide);
    Extent4<T> e = Extent4<T>::of(x.a);
    e.take(x.b);
    e.join(4);
    const Pair4<T> p(e);
    if (on) {
      *reinterpret_cast<uint2*>(to + codes) = make_uint2(p.codes(x.a), p.codes(x.b));
      if (t % 4 == 0) *reinterpret_cast<uint32_t*>(to + pair) = p.bits;
    }
  }
}

template <typename T, int D, int Bits>
__global__ void __launch_bounds__(kRowsThreads) load_kernel(PagedCache c, RowsArgs in) {
  using U = RowUnit<D>;
  take_turn();
  U u(c, in);
  if (u.row >= in.rows) return;
  const int t = (threadIdx.x & 31) % U::L;
  const RowPlace at(c, in.offsets, in.rows, u.row);
  const int page = at.pos < 0 ? -1 : c.table[static_cast<int64_t>(at.slot) * c.table_pages + (at.pos >> c.page_shift)];
  const bool there = c.is_page(page);
  const int in_page = at.pos & (c.page_size - 1);
  uint16_t *k = in.k + u.row * in.k_row + 16 * t, *v = in.v + u.row * in.v_row + 16 * t;
  unsigned char* first = reinterpret_cast<unsigned char*>(c.pool + c.block(page, in.layer, 0));
  U ahead = u;  // the item that is asked for next
  if constexpr (Bits == 4) {
    const int head_bytes = block4_bytes(c);
    const int codes = in_page * (D / 2) + 8 * t, pair = block4_codes(c) + (in_page * (D / kGroup4) + t / 4) * 4;
    uint2 w[kLoadAhead<Bits>];
    uint32_t p[kLoadAhead<Bits>];
    auto load = [&](int n) {
      if (there && ahead.on()) {
        const unsigned char* from = ahead.place(c, first) + static_cast<int64_t>(ahead.head) * head_bytes;
        w[n] = __ldcs(reinterpret_cast<const uint2*>(from + codes));
        p[n] = __ldcs(reinterpret_cast<const uint32_t*>(from + pair));
      }
      ahead.next(c);
    };
#pragma unroll
    for (int n = 0; n < kLoadAhead<Bits>; ++n) {
      w[n] = make_uint2(0, 0);
      p[n] = 0;
      load(n);
    }
    while (u.on()) {
#pragma unroll
      for (int n = 0; n < kLoadAhead<Bits>; ++n) {
        if (!u.on()) break;
        const Piece x{values4<T>(w[n].x, p[n]), values4<T>(w[n].y, p[n])};
        uint16_t* to = u.at(k, v, in);
        u.next(c);
        load(n);
        x.store(to, in.wide);
      }
    }
  } else {
    Piece x[kLoadAhead<Bits>];
    auto load = [&](int n) {
      if (there && ahead.on())
        x[n].load(reinterpret_cast<const uint16_t*>(ahead.place(c, first)) +
                      (static_cast<int64_t>(ahead.head) * c.page_size + in_page) * D + 16 * t, true);
      ahead.next(c);
    };
#pragma unroll
    for (int n = 0; n < kLoadAhead<Bits>; ++n) {
      x[n] = Piece{};
      load(n);
    }
    while (u.on()) {
#pragma unroll
      for (int n = 0; n < kLoadAhead<Bits>; ++n) {
        if (!u.on()) break;
        const Piece y = x[n];
        uint16_t* to = u.at(k, v, in);
        u.next(c);
        load(n);
        y.store(to, in.wide);
      }
    }
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
  const auto aligned32 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; };
  const bool wide = aligned32(r.k) && aligned32(r.v) &&
                    (r.k_row_stride | r.v_row_stride | r.k_layer_stride | r.v_layer_stride) % 16 == 0;
  RowsArgs in{r.layer, r.n_layers, r.rows, 1, wide, static_cast<uint16_t*>(const_cast<void*>(r.k)),
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

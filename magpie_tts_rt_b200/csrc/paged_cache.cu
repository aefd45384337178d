// Upkeep of the paged key/value cache: extend, fork, free, compact, store.
//
// Every operator is a plan (which pages go where: integers, scanned over the
// slots and over the pool's reference counts by one CTA, so the result does
// not depend on timing) followed by the movement of whole pages or rows,
// which is bound by HBM: each byte is read once and written once with
// 16-byte accesses, enough of them in flight to cover the latency.
// Measured: 16,800 rows of 32 KB stored in 174 us (6.3 TB/s read and written);
// 96 pages of 2.1 MB copied from 4 in 37 us (5.4 TB/s written); the plans 4 to 6 us.
#include <algorithm>
#include <atomic>

#include "paged_cache.cuh"

namespace mtt {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;

// Workspace of one upkeep call, in 32-bit words.
struct UpkeepSpace {
  int32_t* free_list;  // [pages] free pages, ascending
  int32_t* rank;       // [slots] index of the slot's first new page in free_list; -1 not granted
  int32_t* len;        // [slots] forked lengths
  int32_t* rows;       // [slots][table_pages] forked rows
  int32_t* src;        // [pages] page copies: from
  int32_t* dst;        // [pages] to
  int32_t* map;        // [pages] compact: new number of each page
  int32_t* counts;     // [4] 0 page copies
};

size_t upkeep_words(int64_t pages, int64_t slots, int64_t table_pages) {
  return static_cast<size_t>(4 * pages + 2 * slots + slots * table_pages + 64);
}

UpkeepSpace upkeep_space(const PagedCache& c, void* ws) {
  int32_t* p = static_cast<int32_t*>(ws);
  UpkeepSpace u;
  u.counts = p;
  p += 64;
  u.free_list = p;
  p += c.pages;
  u.src = p;
  p += c.pages;
  u.dst = p;
  p += c.pages;
  u.map = p;
  p += c.pages;
  u.rank = p;
  p += c.slots;
  u.len = p;
  p += c.slots;
  u.rows = p;
  return u;
}

// Exclusive prefix sum over the block's threads; `total` gets the sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int warp_sum[kPlanThreads / 32];
  __shared__ int all;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += n;
    }
    warp_sum[lane] = s;
    if (lane == 31) all = s;
  }
  __syncthreads();
  const int before = (warp > 0 ? warp_sum[warp - 1] : 0) + inc - v;
  *total = all;
  __syncthreads();
  return before;
}

// Lists the free pages in ascending order, at least `want` of them if there
// are that many; returns how many were found.  A thread looks at 16 pages a
// round: what a round costs is its latency, and a pool may have 100,000s.
__device__ int list_free(const PagedCache& c, int32_t* list, int want) {
  constexpr int kEach = 16;
  int found = 0;
  for (int64_t base = 0; base < c.pages && found < want; base += kEach * kPlanThreads) {
    const int64_t p0 = base + kEach * threadIdx.x;
    uint32_t free = 0;
    if (p0 + kEach <= c.pages) {
      int4 r[kEach / 4];
#pragma unroll
      for (int j = 0; j < kEach / 4; ++j) r[j] = *reinterpret_cast<const int4*>(c.refs + p0 + 4 * j);
#pragma unroll
      for (int j = 0; j < kEach / 4; ++j)
        free |= ((r[j].x == 0 ? 1u : 0u) | (r[j].y == 0 ? 2u : 0u) | (r[j].z == 0 ? 4u : 0u) | (r[j].w == 0 ? 8u : 0u))
                << (4 * j);
    } else {
      for (int j = 0; j < kEach; ++j)
        if (p0 + j < c.pages && c.refs[p0 + j] == 0) free |= 1u << j;
    }
    int total;
    int at = found + block_scan(__popc(free), &total);
    for (; free != 0; free &= free - 1) list[at++] = static_cast<int32_t>(p0) + __ffs(free) - 1;
    found += total;
  }
  __syncthreads();
  return found;
}

// What each slot asks for, and the sum over the slots before it (at most
// INT_MAX): of the thread's first slot in registers, of further ones (more than
// kPlanThreads slots) in the workspace.
struct Asked {
  int need, rank, all;
  template <typename Need>
  __device__ __forceinline__ Asked(const PagedCache& c, const UpkeepSpace& u, Need need_of) {
    int64_t before = 0;
    for (int base = 0; base < c.slots; base += kPlanThreads) {
      const int i = base + threadIdx.x;
      const int n = i < c.slots ? need_of(i) : -1;
      int total;
      const int r = static_cast<int>(min(before + block_scan(max(n, 0), &total), static_cast<int64_t>(INT32_MAX)));
      if (base == 0) {
        need = n;
        rank = r;
      } else if (i < c.slots) {
        u.rank[i] = r;
        u.len[i] = n;
      }
      before += total;
    }
    all = static_cast<int>(min(before, static_cast<int64_t>(INT32_MAX)));
  }
  __device__ __forceinline__ void load(const UpkeepSpace& u, int i) {
    if (i < kPlanThreads) return;
    need = u.len[i];
    rank = u.rank[i];
  }
  // whether its pages are among the `free` ones; no more are granted after one is not
  __device__ __forceinline__ bool granted(int free) const {
    return need == 0 || (need > 0 && static_cast<int64_t>(rank) + need <= free);
  }
};

// One CTA.  Grants the slots' new pages and writes them into the tables.
__global__ void __launch_bounds__(kPlanThreads) extend_kernel(PagedCache c, const int32_t* counts, UpkeepSpace u) {
  take_turn();
  Asked a(c, u, [&](int i) {  // pages; -1: the count is out of range
    const int len = c.length(i), add = counts[i];
    // the sum is taken in 64 bits: a count near 2^31 is refused, not wrapped
    const int64_t want = (static_cast<int64_t>(len) + add + c.page_size - 1) >> c.page_shift;
    if (add < 0 || want > c.table_pages) return -1;
    return static_cast<int>(want) - ((len + c.page_size - 1) >> c.page_shift);
  });
  const int free_pages = list_free(c, u.free_list, a.all);
  for (int i = threadIdx.x; i < c.slots; i += kPlanThreads) {
    a.load(u, i);
    const int len = c.length(i), add = counts[i];
    const bool ok = a.granted(free_pages);
    if (ok && add > 0) {
      int32_t* row = c.table + static_cast<int64_t>(i) * c.table_pages + ((len + c.page_size - 1) >> c.page_shift);
      for (int j = 0; j < a.need; ++j) {
        const int p = u.free_list[a.rank + j];
        row[j] = p;
        c.refs[p] = 1;
      }
      c.lengths[i] = len + add;
    }
    if (c.status != nullptr && add != 0) c.status[i] = ok ? 0 : (a.need < 0 ? 1 : 2);
    if (c.refused != nullptr) c.refused[i] = add != 0 && !ok;
  }
}

// One CTA: which slots are forked, and their first private page's rank.
__global__ void __launch_bounds__(kPlanThreads)
    fork_plan_kernel(PagedCache c, const int32_t* source, int deep, UpkeepSpace u) {
  __shared__ int copies;
  if (threadIdx.x == 0) copies = 0;
  take_turn();
  Asked a(c, u, [&](int i) {  // pages; -1: it stays as it is; -2: no such source
    const int s = source[i];
    if (s == -1 || s == i) return -1;
    if (s < 0 || s >= c.slots) return -2;
    const int len = c.length(s);
    return deep ? (len + c.page_size - 1) >> c.page_shift : ((len & (c.page_size - 1)) != 0 ? 1 : 0);
  });
  const int free_pages = list_free(c, u.free_list, a.all);
  for (int i = threadIdx.x; i < c.slots; i += kPlanThreads) {
    a.load(u, i);
    const bool ok = a.granted(free_pages);
    u.rank[i] = ok ? a.rank : -1;
    if (ok && a.need > 0) atomicMax(&copies, a.rank + a.need);
    if (a.need != -1 && c.status != nullptr) c.status[i] = a.need == -2 ? 1 : (ok ? 0 : 2);
  }
  __syncthreads();
  if (threadIdx.x == 0) u.counts[0] = copies;
}

// Slot d (one CTA each): its new row, from its source's old one, and the page copies it asks for.
__global__ void __launch_bounds__(kMoveThreads) fork_rows_kernel(PagedCache c, const int32_t* source, int deep,
                                                                 UpkeepSpace u) {
  take_turn();
  const int d = blockIdx.x;
  const int rank = u.rank[d];
  if (rank < 0) return;
  const int s = source[d];
  const int len = c.length(s);
  const int used = (len + c.page_size - 1) >> c.page_shift;
  const int first_copy = deep ? 0 : len >> c.page_shift;
  const int32_t* old = c.table + static_cast<int64_t>(s) * c.table_pages;
  int32_t* row = u.rows + static_cast<int64_t>(d) * c.table_pages;
  for (int j = threadIdx.x; j < c.table_pages; j += kMoveThreads) {
    int p = j < used ? old[j] : -1;
    if (j < used && j >= first_copy) {
      const int to = u.free_list[rank + j - first_copy];
      u.src[rank + j - first_copy] = p;
      u.dst[rank + j - first_copy] = to;
      p = to;
    }
    row[j] = p;
    if (c.is_page(p)) atomicAdd(&c.refs[p], 1);
  }
  if (threadIdx.x == 0) u.len[d] = len;
}

// Part `part` of `parts` of one page, all layers.  kAgain: other copies read the
// same page (a voice's partial page goes to every session forked from it), so
// it stays in L2.
template <bool kAgain>
__device__ __forceinline__ void copy_page(const PagedCache& c, int from, int to, int part, int parts) {
  const int64_t vecs = static_cast<int64_t>(c.layers) * 2 * c.kv_elems / 8;
  const int64_t lo = vecs * part / parts, hi = vecs * (part + 1) / parts;
  const uint4* s = reinterpret_cast<const uint4*>(c.pool) + from * vecs;
  uint4* d = reinterpret_cast<uint4*>(c.pool) + to * vecs;
  int64_t v = lo + threadIdx.x;
  for (; v + 3 * kMoveThreads < hi; v += 4 * kMoveThreads) {
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = kAgain ? __ldcg(s + v + j * kMoveThreads) : __ldcs(s + v + j * kMoveThreads);
#pragma unroll
    for (int j = 0; j < 4; ++j) __stcs(d + v + j * kMoveThreads, x[j]);
  }
  for (; v < hi; v += kMoveThreads) __stcs(d + v, __ldcs(s + v));
}

// The plan's page copies, `parts` pieces each, dealt over the grid.
template <bool kAgain>
__device__ __forceinline__ void copy_pairs(const PagedCache& c, const UpkeepSpace& u, int parts) {
  const int64_t items = static_cast<int64_t>(u.counts[0]) * parts;
  for (int64_t w = blockIdx.x; w < items; w += gridDim.x) {
    const int pair = static_cast<int>(w / parts);
    const int from = u.src[pair], to = u.dst[pair];
    if (c.is_page(from) && c.is_page(to)) copy_page<kAgain>(c, from, to, static_cast<int>(w % parts), parts);
  }
}

// The forked rows and lengths become the slots', the pages they had are released, partial pages copied.
__global__ void __launch_bounds__(kMoveThreads) fork_commit_kernel(PagedCache c, UpkeepSpace u, int parts) {
  take_turn();
  for (int d = blockIdx.x; d < c.slots; d += gridDim.x) {
    if (u.rank[d] < 0) continue;
    int32_t* row = c.table + static_cast<int64_t>(d) * c.table_pages;
    const int32_t* next = u.rows + static_cast<int64_t>(d) * c.table_pages;
    for (int j = threadIdx.x; j < c.table_pages; j += kMoveThreads) {
      const int p = row[j];
      if (c.is_page(p)) atomicSub(&c.refs[p], 1);
      row[j] = next[j];
    }
    if (threadIdx.x == 0) {
      c.lengths[d] = u.len[d];
      if (c.refused != nullptr) c.refused[d] = 0;
    }
  }
  copy_pairs<true>(c, u, parts);
}

// One warp per slot.
__global__ void __launch_bounds__(kMoveThreads) free_kernel(PagedCache c, const bool* mask) {
  take_turn();
  const int i = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
  if (i >= c.slots || !mask[i]) return;
  int32_t* row = c.table + static_cast<int64_t>(i) * c.table_pages;
  for (int j = threadIdx.x & 31; j < c.table_pages; j += 32) {
    const int p = row[j];
    if (c.is_page(p)) atomicSub(&c.refs[p], 1);
    row[j] = -1;
  }
  if ((threadIdx.x & 31) == 0) {
    c.lengths[i] = 0;
    if (c.refused != nullptr) c.refused[i] = 0;
  }
}

// One CTA: live pages, and where those past the live count go.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(PagedCache c, UpkeepSpace u) {
  take_turn();
  const int live = c.pages - list_free(c, u.free_list, INT32_MAX);  // free pages below `live` come first in the list
  int moved = 0;
  for (int base = live & ~(4 * kPlanThreads - 1); base < c.pages; base += 4 * kPlanThreads) {
    const int p0 = base + 4 * threadIdx.x;
    bool f[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = p0 + j >= live && p0 + j < c.pages && c.refs[p0 + j] != 0;
      n += f[j];
    }
    int total;
    int at = moved + block_scan(n, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (f[j]) {
        const int to = u.free_list[at];
        u.src[at] = p0 + j;
        u.dst[at] = to;
        u.map[p0 + j] = to;
        ++at;
      }
    }
    moved += total;
  }
  if (threadIdx.x == 0) {
    u.counts[0] = moved;
    u.counts[1] = live;
    if (c.live != nullptr) c.live[0] = live;
  }
}

__global__ void __launch_bounds__(kMoveThreads) compact_move_kernel(PagedCache c, UpkeepSpace u, int parts) {
  take_turn();
  const int moved = u.counts[0], live = u.counts[1];
  if (moved == 0) return;
  const int64_t entries = static_cast<int64_t>(c.slots) * c.table_pages;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kMoveThreads;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x;
  for (int64_t e = me; e < entries; e += stride) {
    const int p = c.table[e];
    if (p >= live && p < c.pages) c.table[e] = u.map[p];
  }
  for (int64_t m = me; m < moved; m += stride) {
    c.refs[u.dst[m]] = c.refs[u.src[m]];
    c.refs[u.src[m]] = 0;
  }
  copy_pairs<false>(c, u, parts);
}

struct Rows {
  int layer, n_layers, rows;
  const uint16_t *k, *v;
  int64_t k_row, v_row, k_layer, v_layer;
  const int32_t* offsets;
};

// Row blockIdx.x: its keys and values of every given layer to its slot's page.
__global__ void __launch_bounds__(kMoveThreads) store_kernel(PagedCache c, Rows in) {
  take_turn();
  const int row = blockIdx.x;
  int slot = row, count = 1, first = row;
  if (in.offsets != nullptr) {
    // the slot with offsets[slot] <= row < offsets[slot + 1]
    int lo = 0, hi = c.slots;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (in.offsets[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    slot = lo;
    if (slot >= c.slots) return;
    first = in.offsets[slot];
    count = in.offsets[slot + 1] - first;
    if (first < 0 || first > row || in.offsets[slot + 1] > in.rows) {
      if (threadIdx.x == 0 && c.status != nullptr) c.status[slot] = 1;
      return;
    }
  }
  const int len = c.length(slot);
  if (in.offsets == nullptr && len == 0) return;
  if (c.refused != nullptr && c.refused[slot] != 0) return;  // its last tokens are not the rows'
  if (count > len) {
    if (threadIdx.x == 0 && c.status != nullptr) c.status[slot] = 1;
    return;
  }
  const int t = len - count + row - first;
  const int page = c.table[static_cast<int64_t>(slot) * c.table_pages + (t >> c.page_shift)];
  if (!c.is_page(page) || c.refs[page] > 1) {
    if (threadIdx.x == 0 && c.status != nullptr) c.status[slot] = 3;
    return;
  }
  // A thread keeps its piece of the heads and walks over (layer, keys or
  // values), several rows of threads side by side where the heads are few.
  const int hv = c.kv_heads * c.head_dim / 8;  // 16-byte pieces of one layer's keys
  const int dv_shift = c.head_dim == 64 ? 3 : 4;
  const int side = max(1, kMoveThreads / hv), blocks = 2 * in.n_layers;
  const int mine = static_cast<int>(threadIdx.x) / min(hv, kMoveThreads);
  if (mine >= side) return;
  const int64_t in_page = static_cast<int64_t>(t & (c.page_size - 1)) * c.head_dim;
  for (int piece = hv < kMoveThreads ? threadIdx.x - mine * hv : threadIdx.x; piece < hv; piece += kMoveThreads) {
    const int h = piece >> dv_shift, e = piece & ((1 << dv_shift) - 1);
    uint16_t* dst = c.pool + c.block(page, in.layer, 0) + static_cast<int64_t>(h) * c.page_size * c.head_dim + in_page + 8 * e;
    const uint16_t* k = in.k + row * in.k_row + 8 * piece;
    const uint16_t* v = in.v + row * in.v_row + 8 * piece;
    constexpr int kAhead = 4;
    for (int b = mine; b < blocks; b += kAhead * side) {
      uint4 x[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int at = b + n * side, l = at >> 1;
        if (at < blocks) x[n] = __ldcs(reinterpret_cast<const uint4*>((at & 1) ? v + l * in.v_layer : k + l * in.k_layer));
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int at = b + n * side;
        if (at < blocks) *reinterpret_cast<uint4*>(dst + at * c.kv_elems) = x[n];
      }
    }
  }
}

// Pieces a page copy is cut into: about 32 KB each, so that few large pages still occupy every SM.
int copy_parts(const PagedCache& c) {
  const int64_t bytes = static_cast<int64_t>(c.layers) * 4 * c.kv_elems;
  return static_cast<int>(std::min<int64_t>(std::max<int64_t>((bytes + 32767) / 32768, 1), 4096));
}

}  // namespace

int cache_sm_count() {
  static std::atomic<int> known[64];  // by device ordinal; 0 not asked yet
  int dev = -1, sms = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    if (dev >= 0 && dev < 64 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) {
      if (dev >= 0 && dev < 64) known[dev].store(sms, std::memory_order_relaxed);
      return sms;
    }
  }
  cudaGetLastError();
  return 0;
}

int cache_call_status(cudaError_t e) {
  if (e == cudaSuccess) e = cudaPeekAtLastError();
  return e == cudaSuccess ? MTT_B200_STATUS_OK : MTT_B200_STATUS_CUDA_ERROR;
}

bool paged_cache_view(const mtt_b200_paged_cache_t* c, PagedCache* out) {
  if (c == nullptr || c->pages < 1 || c->layers < 1 || c->kv_heads < 1 || c->slots < 1 || c->slots > kCacheMaxSlots ||
      c->table_pages < 1 || (c->head_dim != 64 && c->head_dim != 128) ||
      (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) ||
      (c->dtype != MTT_B200_DTYPE_BF16 && c->dtype != MTT_B200_DTYPE_F16))
    return false;
  // rows of the pool (one token's keys or values of one head) and tokens of a slot are counted in 31 bits
  const double rows = static_cast<double>(c->pages) * c->layers * 2 * c->kv_heads * c->page_size;
  if (rows >= 2147483648.0 || static_cast<int64_t>(c->table_pages) * c->page_size >= (int64_t{1} << 30) ||
      static_cast<double>(c->slots) * c->table_pages * (c->page_size / 16) >= 2147352576.0)
    return false;
  if (c->pool == nullptr || c->page_table == nullptr || c->lengths == nullptr || c->refs == nullptr ||
      (reinterpret_cast<uintptr_t>(c->pool) & 127u) != 0 || !aligned16(c->refs))
    return false;
  out->pages = c->pages;
  out->layers = c->layers;
  out->kv_heads = c->kv_heads;
  out->page_size = c->page_size;
  out->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  out->head_dim = c->head_dim;
  out->slots = c->slots;
  out->table_pages = c->table_pages;
  out->kv_elems = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  out->pool = static_cast<uint16_t*>(c->pool);
  out->table = c->page_table;
  out->lengths = c->lengths;
  out->refs = c->refs;
  out->status = c->status;
  out->live = c->live;
  out->refused = c->refused;
  return true;
}

}  // namespace mtt

using namespace mtt;

namespace {

size_t upkeep_bytes(const mtt_b200_paged_cache_t& c) {
  return (4 * upkeep_words(c.pages, c.slots, c.table_pages) + 255) / 256 * 256;
}

// The upkeep words lie at the workspace's start.
bool upkeep_checked(const mtt_b200_paged_cache_t* cache, void* ws, size_t bytes, PagedCache* c, UpkeepSpace* u) {
  if (!paged_cache_view(cache, c) || ws == nullptr || !aligned16(ws) || bytes < upkeep_bytes(*cache)) return false;
  *u = upkeep_space(*c, ws);
  return true;
}

}  // namespace

void* mtt::paged_attention_space(const mtt_b200_paged_cache_t& c, int q_heads, int rows, void* workspace, size_t bytes) {
  const size_t up = upkeep_bytes(c);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 ||
      bytes < up + paged_attention_workspace(c, q_heads, rows))
    return nullptr;
  return static_cast<char*>(workspace) + up;
}

extern "C" {

size_t mtt_b200_paged_cache_workspace_size(const mtt_b200_paged_cache_t* cache, int32_t q_heads, int32_t rows) {
  PagedCache c;
  if (!paged_cache_view(cache, &c) || q_heads < 1 || q_heads % c.kv_heads != 0 ||
      q_heads / c.kv_heads > kCacheMaxGroup || rows < 0 || rows > kCacheMaxRows)
    return 0;
  return upkeep_bytes(*cache) + paged_attention_workspace(*cache, q_heads, rows);
}

int mtt_b200_launch_paged_cache_extend(const mtt_b200_paged_cache_t* cache, const int32_t* counts, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  PagedCache c;
  UpkeepSpace u;
  if (counts == nullptr || !upkeep_checked(cache, workspace, workspace_bytes, &c, &u))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  return cache_call_status(launch_serialized(extend_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), c,
                                  counts, u));
}

int mtt_b200_launch_paged_cache_fork(const mtt_b200_paged_cache_t* cache, const int32_t* source, int32_t deep,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  PagedCache c;
  UpkeepSpace u;
  const int sms = cache_sm_count();
  if (source == nullptr || sms <= 0 || !upkeep_checked(cache, workspace, workspace_bytes, &c, &u))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_serialized(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, source, deep, u);
  if (e == cudaSuccess)
    e = launch_serialized(fork_rows_kernel, dim3(c.slots), dim3(kMoveThreads), 0, s, c, source, deep, u);
  if (e == cudaSuccess)
    e = launch_serialized(fork_commit_kernel, dim3(8 * sms), dim3(kMoveThreads), 0, s, c, u, copy_parts(c));
  return cache_call_status(e);
}

int mtt_b200_launch_paged_cache_free(const mtt_b200_paged_cache_t* cache, const bool* mask, void* stream) {
  PagedCache c;
  if (mask == nullptr || !paged_cache_view(cache, &c)) return MTT_B200_STATUS_INVALID_ARGUMENT;
  constexpr int per = kMoveThreads / 32;
  return cache_call_status(launch_serialized(free_kernel, dim3((c.slots + per - 1) / per), dim3(kMoveThreads), 0,
                                  static_cast<cudaStream_t>(stream), c, mask));
}

int mtt_b200_launch_paged_cache_compact(const mtt_b200_paged_cache_t* cache, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  PagedCache c;
  UpkeepSpace u;
  const int sms = cache_sm_count();
  if (sms <= 0 || !upkeep_checked(cache, workspace, workspace_bytes, &c, &u)) return MTT_B200_STATUS_INVALID_ARGUMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_serialized(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, u);
  if (e == cudaSuccess)
    e = launch_serialized(compact_move_kernel, dim3(8 * sms), dim3(kMoveThreads), 0, s, c, u, copy_parts(c));
  return cache_call_status(e);
}

int mtt_b200_launch_paged_cache_store(const mtt_b200_paged_cache_t* cache, const mtt_b200_cache_rows_t* rows,
                                      void* stream) {
  PagedCache c;
  if (rows == nullptr || !paged_cache_view(cache, &c) || rows->rows < 0 || rows->layer < 0 || rows->n_layers < 1 ||
      rows->n_layers > c.layers - rows->layer)
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  if (rows->rows == 0) return MTT_B200_STATUS_OK;
  if (rows->k == nullptr || rows->v == nullptr || !aligned16(rows->k) || !aligned16(rows->v) ||
      (rows->k_row_stride | rows->v_row_stride | rows->k_layer_stride | rows->v_layer_stride) % 8 != 0 ||
      (rows->offsets == nullptr && rows->rows > c.slots))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  Rows in{rows->layer, rows->n_layers, rows->rows, static_cast<const uint16_t*>(rows->k),
          static_cast<const uint16_t*>(rows->v), rows->k_row_stride, rows->v_row_stride, rows->k_layer_stride,
          rows->v_layer_stride, rows->offsets};
  return cache_call_status(launch_serialized(store_kernel, dim3(rows->rows), dim3(kMoveThreads), 0,
                                  static_cast<cudaStream_t>(stream), c, in));
}

}  // extern "C"

// Attention of runs of query rows over the paged cache on the tensor cores:
// the prompt form (slot i's rows are its newest tokens, causal, with window,
// sinks and key mask) and the prefix pass of groups of slots that share a
// prefix (every member's newest token over the voice's pages).
//
//   S = Q K^T,  P = e^{scale S - m},  l += P 1,  O += P V     per 128-key tile
//
// A unit is a key head and two Q tiles of 128 rows; a tile's rows are the
// group's query heads of consecutive tokens (128 / group of them), so shared
// key heads fill the MMA's 128 rows and every key tile in shared memory is
// used by both Q tiles.  Warp roles (384 threads, one CTA per SM):
//   warps 0-3, 4-7  softmax of Q tile 0 / 1: one thread per row reads S from
//                   tensor memory, writes P over it in 16 bits (the A operand
//                   of the second product), half a tile at a time, and stores
//                   the result;
//   warp 8          issues the MMAs: S0, S1, then P0 V, next S0, P1 V, next S1,
//                   ... so that one tile's products run under the other tile's
//                   softmax;
//   warp 9          TMA: the pages of each key tile into a ring of stages
//                   (128-byte swizzle);
//   warp 10         clears value rows that no query of the unit may see (page
//                   tails, masked keys, later keys, those that the window has left
//                   behind), whose probability of 0 must not meet a NaN;
//   warp 11         TMA: the next unit's queries, as soon as the last scores
//                   of this one are done (the prefix pass's rows lie apart, so
//                   there the softmax warps copy them).
// Tensor memory: S0, S1 (128 columns each), O0, O1 (head_dim each), which at
// head_dim 128 is all of it.
//
// m is not the maximum so far, but one found when it was last needed: as long
// as a half tile's probabilities stay below 2^15 (where f16 ends; f32 sums and
// any 16-bit type keep their relative precision up to there) nothing is
// compared or rescaled.  (For f16 they are held 2^8 times as large from the start,
// so that what is small beside the largest stays in that type's range too.)  Only
// when they do not, or when a row has seen no key yet, is the maximum looked for, O
// and l rescaled, and the half taken again.
//
// The units' key tiles form one line that is cut into equal parts, one per
// CTA; a unit cut by a boundary leaves (m, l, O) in the workspace for a
// second kernel that joins the parts in order.
//
// Every wait is bounded.  Some last as long as a unit's part in a share (the
// next unit's queries wait for this one's last scores, a Q tile without rows
// for the next unit), so the bound grows with the key tiles of the CTA's share:
// 50 us for each, some twenty times what it takes, and 0.2 s beside.  A CTA in
// which a wait gives up says so in the workspace and leaves; the join marks the
// slots of its share with status 4 (and lets the members of a prefix pass be
// attended on their own).
//
// Probabilities are rounded once to the cache's type because P is the tensor
// core's A operand: to multiply the rounding's remainder as well would take a key
// tile's MMAs from 2048 to 3072 cycles of the 3100 that it takes.
//
// Measured: 8192 tokens, 32/8 heads of 128, causal, 484 us alone and 550 to 562 us
// back to back, where the board's power holds the clock near 1.4 GHz (1.14 and
// 0.99 PFLOP/s); the tensor pipe and the special function unit are each busy 59% of
// the time.  A key tile takes both Q tiles about 3100 SM cycles: 2048 of MMA, as
// many of exponentials, and what bounds it is a softmax warp's own chain: 500
// cycles for a half's 64 exponentials a row, 300 for loads, packing, stores and
// barriers, while the other tile's warp shares its scheduler.  Tried and slower:
// 64-key tiles with two score buffers (N = 64 MMAs cost 47 cycles, not 32), one
// issuing warp per Q tile, two threads per row, a register split with setmaxnreg
// (230 bytes spilled in the loop), a quarter of the exponentials as polynomials on
// the FMA pipe (5 to 10%: it is instructions that bound the loop).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gemm_tc.cuh"
#include "paged_attention.cuh"

namespace mtt {
namespace {

constexpr int kTile = 128;          // rows of a Q tile
constexpr int kKeys = 128;          // keys of a key tile
constexpr int kHalf = kKeys / 2;    // keys whose probabilities are handed over together
constexpr int kPairRows = 2 * kTile;
constexpr int kPromptThreads = 384;
constexpr int kPromptPlanThreads = 1024;
// e^{scale S - m} is held times 2^this (see above); l and O share the factor
template <typename T>
constexpr float kPromptBias = std::is_same_v<T, __half> ? 8.f : 0.f;
constexpr int kMinShare = 2;        // key tiles a CTA takes at least
constexpr int kMaxSms = 160;        // workspaces are sized for the largest device

template <int D>
struct PromptCfg {
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr uint32_t kQBytes = kTile * D * 2;
  static constexpr uint32_t kTileBytes = kKeys * D * 2;
  static constexpr uint32_t kOutBytes = 8 * 32 * 128;  // a 32 x 64 block of results per softmax warp, on its way out
  static constexpr size_t kSmem =
      1024 + 2 * static_cast<size_t>(kQBytes) + kStages * static_cast<size_t>(kTileBytes) + kOutBytes;
};

// Rows of the attention: tokens of slots, or members of prefix groups.
struct PromptRows {
  int n;                     // slots, or groups
  int n_rows;                // rows in all (tokens, or members)
  const int32_t* offsets;    // [n + 1]
  const int32_t* members;    // prefix pass: slot of each member; null for prompts
  const int32_t* voice;      // prefix pass: [n] slot that holds the prefix
  const int32_t* tokens;     // prefix pass: [n] its length
  int longest;               // prefix pass: longer prefixes are not shared (the window hides some of them)
  int32_t* base;             // prefix pass: [slots] out, SharedPrefix::base
  bool own_plan;             // each CTA of the kernel makes the plan
  bool q_mapped;             // the query map describes q: tiles come by TMA
  float* state;              // prefix pass: [slots][q_heads][D + 4]: O, m, l of each member
};

// A unit's place on the line: its key tiles, and before them what entering and
// leaving it costs, in key tiles.
constexpr int kPairCost = 2;

struct PromptSpace {
  int64_t* head;       // [0] pairs, [1] length of one key head's line, [2] length of a share
  int32_t* cta_pair;   // [kMaxSms + 1] the pair that holds the start of CTA c's share
  int32_t* first;      // [n + 1] pairs of the slots before
  int32_t* gave_up;    // [kMaxSms] whether a wait of CTA c ran out
  int4* rec;           // [2 * pairs]: first token (or member), place (high), key tiles, place (low); then Geom
  float* part;         // [CTAs][2][D + 2][256]
  Waits waits;
};

// A pair's place on its key head's line.
__device__ __forceinline__ int64_t pair_place(const int4& rec) {
  return static_cast<int64_t>(rec.y) << 32 | static_cast<uint32_t>(rec.w);
}

// Where a pair's rows and keys are: rows [row0, row0 + count) are the slot's
// (or group's), its keys the first len tokens of key_slot.
struct Geom {
  int row0, count, len, key_slot;
};

struct PairGeom : Geom {
  bool ok;
  __device__ __forceinline__ PairGeom(const PagedCache& c, const PromptRows& r, int i) {
    const int a = r.offsets[i], b = r.offsets[i + 1];
    ok = a >= 0 && a <= b && b <= r.n_rows;
    row0 = ok ? a : 0;
    count = ok ? b - a : 0;
    if (r.members != nullptr) {
      key_slot = r.voice[i];
      len = r.tokens[i];
      ok = ok && key_slot >= 0 && key_slot < c.slots && len > 0 && len <= r.longest && (len & (c.page_size - 1)) == 0;
      ok = ok && c.length(ok ? key_slot : 0) >= len;
    } else {
      key_slot = i;
      len = c.length(i);
      ok = ok && count <= len;
    }
    if (!ok) {
      len = 0;
      key_slot = 0;
    }
  }
};

// The key tiles that queries at positions [p0, p1] may see.
struct KeySpan {
  int sink_n, win0, n;
  __device__ __forceinline__ KeySpan(int p0, int p1, int window, int sinks) {
    const int low = window > 0 ? max(0, p0 - window + 1) : 0;
    const int end = p1 / kKeys + 1;
    sink_n = low > 0 && sinks > 0 ? min((min(sinks - 1, p1)) / kKeys + 1, end) : 0;
    win0 = max(low / kKeys, sink_n);
    n = sink_n + max(0, end - win0);
  }
  __device__ __forceinline__ int tile(int t) const { return t < sink_n ? t : win0 + t - sink_n; }
};

// The key tiles of which a query at positions [p0, p1] sees anything.
struct TilesSeen {
  int low, high, sink;
  __device__ __forceinline__ TilesSeen(int p0, int p1, int window, int sinks) {
    low = window > 0 ? max(0, p0 - window + 1) / kKeys : 0;
    high = p0 <= p1 ? p1 / kKeys : -1;
    sink = (sinks > 0 ? (sinks - 1) / kKeys : -1);
  }
  __device__ __forceinline__ bool at(int j) const { return j <= high && (j >= low || j <= sink); }
};
// Whether every one of them sees every key of it.
__device__ __forceinline__ bool tile_full(int j, int p0, int p1, int window, int sinks) {
  return kKeys * j + kKeys - 1 <= p0 && (window == 0 || kKeys * j > p1 - window || kKeys * (j + 1) <= sinks);
}

// Positions [p0, p1] of the rows of tokens [t0, t1); empty when p1 < p0.  In
// the prefix pass every row stands at the prefix's end.
__device__ __forceinline__ void positions(const Geom& g, bool prefix, int t0, int t1, int* p0, int* p1) {
  t1 = min(t1, g.count);
  if (prefix) {
    *p1 = g.len - 1;
    *p0 = t0 < t1 && g.len > 0 ? g.len - 1 : g.len;
  } else {
    *p0 = g.len - g.count + t0;
    *p1 = g.len >= g.count ? g.len - g.count + t1 - 1 : *p0 - 1;  // a slot with more rows than tokens: none
  }
}

// ---------------------------------------------------------------------------
// plan: lists the pairs and cuts the line of key tiles.  One CTA's work, ahead
// of the kernel; where every pair has a thread of its own each CTA of the kernel
// does it for itself instead: 1.5 to 3 us less a call (one prompt of 218 tokens
// 18.2 -> 16.3 us, 2048 slots over four voices 90.9 -> 88.0 us).
// ---------------------------------------------------------------------------

template <int Threads>
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* total) {
  constexpr int kWarps = Threads / 32;
  __shared__ int64_t warp_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int64_t s = lane < kWarps ? warp_sum[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t n = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += n;
    }
    if (lane < kWarps) warp_sum[lane] = s;
  }
  __syncthreads();
  const int64_t before = (warp > 0 ? warp_sum[warp - 1] : 0) + inc - v;
  *total = warp_sum[kWarps - 1];
  __syncthreads();
  return before;
}

// Fills first and rec; the length of a share.  Of `ctas` CTAs those from c0 on,
// one a thread, get their first pair.
template <int Threads>
__device__ void make_plan(const PagedCache& c, const PromptRows& rows, const PromptSpace& ws, int window, int sinks,
                          int tokens_per_pair, int ctas, int c0, int c1) {
  const int tid = threadIdx.x;
  const bool prefix = rows.members != nullptr;
  // slots whose offsets overlap could ask for more pairs than there is room for
  const int most = rows.n_rows / tokens_per_pair + rows.n;
  int pairs = 0;
  for (int base = 0; base < rows.n; base += Threads) {
    const int i = base + tid;
    int n = 0;
    if (i < rows.n) n = (PairGeom(c, rows, i).count + tokens_per_pair - 1) / tokens_per_pair;
    int64_t total;
    const int64_t before = pairs + plan_scan<Threads>(n, &total);
    if (i < rows.n) ws.first[i] = static_cast<int>(min(before, static_cast<int64_t>(most)));
    pairs = static_cast<int>(min(pairs + total, static_cast<int64_t>(most)));
  }
  if (tid == 0) ws.first[rows.n] = pairs;
  __syncthreads();
  int64_t tiles = 0;
  for (int base = 0; base < pairs; base += Threads) {
    const int k = base + tid;
    int n = 0, tok0 = 0;
    Geom geom{0, 0, 0, 0};
    if (k < pairs) {
      int lo = 0, hi = rows.n;  // the last slot whose pairs begin at or before k
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ws.first[mid] <= k) lo = mid; else hi = mid;
      }
      tok0 = (k - ws.first[lo]) * tokens_per_pair;
      geom = PairGeom(c, rows, lo);
      int p0, p1;
      positions(geom, prefix, tok0, tok0 + tokens_per_pair, &p0, &p1);
      // rows that see nothing still need their zeros written: one tile without keys
      n = p0 <= p1 ? KeySpan(p0, p1, window, sinks).n : (prefix ? 0 : 1);
    }
    int64_t total;
    const int64_t before = tiles + plan_scan<Threads>(n > 0 ? n + kPairCost : 0, &total);
    if (k < pairs) {
      ws.rec[2 * k] = make_int4(tok0, static_cast<int>(before >> 32), n, static_cast<int>(before));
      ws.rec[2 * k + 1] = make_int4(geom.row0, geom.count, geom.len, geom.key_slot);
    }
    tiles += total;
  }
  __syncthreads();
  const int64_t all = tiles * c.kv_heads;
  const int64_t per = max((all + ctas - 1) / ctas, static_cast<int64_t>(kMinShare + kPairCost));
  if (tid == 0) {
    ws.head[0] = pairs;
    ws.head[1] = tiles;
    ws.head[2] = per;
  }
  const int cta = c0 + tid;
  if (cta < c1 && cta * per < all) {
    const int64_t x = cta * per % tiles;
    int lo = 0, hi = pairs;  // the last pair that begins at or before x (pairs without tiles are never last)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pair_place(ws.rec[2 * mid]) <= x) lo = mid; else hi = mid;
    }
    ws.cta_pair[cta] = lo;
  }
}

__global__ void __launch_bounds__(kPromptPlanThreads)
    prompt_plan_kernel(PagedCache c, PromptRows rows, PromptSpace ws, int window, int sinks, int tokens_per_pair,
                       int ctas) {
  take_turn();
  if (rows.members != nullptr)
    for (int i = threadIdx.x; i < c.slots; i += kPromptPlanThreads) rows.base[i] = 0;
  make_plan<kPromptPlanThreads>(c, rows, ws, window, sinks, tokens_per_pair, ctas, 0, ctas);
}

// ---------------------------------------------------------------------------
// a CTA's share, unit by unit
// ---------------------------------------------------------------------------

// Places are counted from the start of the CTA's share.
struct Walk {
  int end;          // of the share
  int place;        // where the unit begins (before the share, when another CTA holds its beginning)
  int pairs, head, pair;
  int tok0, n;      // the unit's first token (or member) and key tiles
  Geom g;
  int t0, t1;       // its key tiles in this share

  __device__ __forceinline__ bool begin(const PromptSpace& ws, int kv_heads, int cta) {
    pairs = static_cast<int>(ws.head[0]);
    const int64_t line = ws.head[1], per = ws.head[2], x = cta * per;
    if (x >= line * kv_heads) return false;
    end = static_cast<int>(min(line * kv_heads - x, per));
    head = static_cast<int>(x / line);
    pair = ws.cta_pair[cta];
    place = static_cast<int>(pair_place(ws.rec[2 * pair]) - (x - head * line));
    return load(ws);
  }
  __device__ __forceinline__ bool next(const PromptSpace& ws) {
    place += kPairCost + n;
    if (place >= end) return false;
    ++pair;
    return load(ws);
  }
  // false when the share ends before the unit's first key tile
  __device__ __forceinline__ bool load(const PromptSpace& ws) {
    int4 rec;
    while (true) {
      if (pair >= pairs) {
        pair = 0;
        ++head;
      }
      rec = ws.rec[2 * pair];
      if (rec.z > 0) break;
      ++pair;
    }
    const int4 at = ws.rec[2 * pair + 1];
    tok0 = rec.x;
    n = rec.z;
    g = Geom{at.x, at.y, at.z, at.w};
    t0 = max(-place - kPairCost, 0);
    t1 = min(n, end - place - kPairCost);
    return t1 > 0;
  }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == n; }
  // which of its CTA's two parts a cut unit leaves
  __device__ __forceinline__ int part() const { return place <= 0 ? 0 : 1; }
};

// 128-byte-swizzled MN-major operand (values: [keys][64 dims] rows of 128
// bytes): 8-key groups 1024 bytes apart, the next 64 dims one block of kKeys rows on.
__device__ __forceinline__ uint64_t value_desc(uint32_t a) {
  uint64_t d = static_cast<uint64_t>((a & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((kKeys * 128) >> 4) << 16;  // leading byte offset: 64 dims on
  d |= static_cast<uint64_t>(1024 >> 4) << 32;           // stride byte offset: 8 keys on
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <typename T>
__host__ __device__ constexpr uint32_t prompt_idesc(int n, bool b_mn_major);
template <>
__host__ __device__ constexpr uint32_t prompt_idesc<__nv_bfloat16>(int n, bool b_mn_major) {
  return umma_idesc_bf16(kTile, n) | (b_mn_major ? 1u << 16 : 0u);
}
template <>
__host__ __device__ constexpr uint32_t prompt_idesc<__half>(int n, bool b_mn_major) {
  return (umma_idesc_bf16(kTile, n) & ~((1u << 7) | (1u << 10))) | (b_mn_major ? 1u << 16 : 0u);
}

// One thread of a converged warp, the same one every time: what it issued is
// tracked by the commits it issues.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// The high words of the two descriptor forms: stride 1024 bytes (8 rows of
// 128), descriptor version 1, 128-byte swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// D[tmem] (+)= A[smem desc] x B[smem desc]^T, given the descriptors' low words.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                        bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %5, 0;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(kDescHigh), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// D[tmem] (+)= A[tmem] x B[smem desc].
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc,
                                        bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n mov.b64 db, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(kDescHigh), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t bits2(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 pair2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}

// NaN if any of the three is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// A wait of up to *limit ns, for all lanes of the warp or none.
struct Patience {
  const volatile unsigned long long* limit;  // in shared memory: looked at only by a wait that has to
  __device__ __forceinline__ bool wait(unsigned long long* bar, uint32_t parity) const {
    const uint32_t at = smem_addr(bar);
    bool ok = mbar_try_cta(at, parity);
    if (!ok) {
      const unsigned long long end = global_ns() + *limit;
      do ok = mbar_try_cta(at, parity);
      while (!ok && global_ns() <= end);
    }
    return __all_sync(0xffffffffu, ok);
  }
};

// For what is certain to come, before the CTA leaves: its own copies in flight, its MMAs.
constexpr unsigned long long kDrainNs = 1000000000ull;
__device__ __forceinline__ void drain(unsigned long long* bar, uint32_t parity) { mbar_wait_cta(bar, parity, kDrainNs); }

__device__ __forceinline__ bool alive(const volatile int* err) { return __all_sync(0xffffffffu, *err == 0); }

// bits [lo, hi) of a 32-bit word
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (lo >= hi) return 0u;
  const uint32_t up = hi == 32 ? 0xffffffffu : (1u << hi) - 1u;
  return up & ~((1u << lo) - 1u);
}

// The key tiles of a unit: those that either of its Q tiles may see.
__device__ __forceinline__ KeySpan unit_span(const Walk& w, bool prefix, int tq, const Attend& a) {
  int p0, p1;
  positions(w.g, prefix, w.tok0, w.tok0 + 2 * tq, &p0, &p1);
  return KeySpan(p0, max(p0, p1), a.window, a.sinks);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap pool_map, const __grid_constant__ CUtensorMap q_map, PagedCache c, Attend a, PromptRows rows,
                  PromptSpace ws) {
  using C = PromptCfg<D>;
  constexpr int S = C::kStages;
  constexpr int DB = D / 64;  // 64-dim blocks of a tile
  constexpr uint32_t kSCol = 0, kOCol = 2 * kKeys;  // S of Q tile i: column i kKeys, O: kOCol + i D
  extern __shared__ unsigned char prompt_smem[];
  __shared__ unsigned long long kv_full[S], kv_empty[S], ready[S], q_ready[2], s_full[2], p_full[2][2], half_done[2],
      o_full[2], q_free[2], fin;
  __shared__ uint32_t tmem_base;
  __shared__ unsigned long long wait_limit;
  __shared__ int err;
  const uint32_t pad = (1024u - (smem_addr(prompt_smem) & 1023u)) & 1023u;
  unsigned char* q_smem = prompt_smem + pad;
  unsigned char* ring = q_smem + 2 * C::kQBytes;
  unsigned char* out_smem = ring + static_cast<size_t>(S) * C::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const bool prefix = rows.members != nullptr;
  const int tq = kTile / a.group;  // tokens of a Q tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&ready[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_ready[i], rows.q_mapped ? 1 : 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i][0], 4);
      mbar_init(&p_full[i][1], 4);
      mbar_init(&half_done[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&q_free[i], 1);
    }
    mbar_init(&fin, 1);
    err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    tmem_alloc(&tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 9 && lane == 0)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&pool_map)) : "memory");
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = tmem_base;
  volatile int* errv = &err;
  take_turn();
  if (rows.own_plan) {  // all CTAs write the same plan
    if (prefix)
      for (int k = blockIdx.x * kPromptThreads + threadIdx.x; k < c.slots; k += gridDim.x * kPromptThreads) rows.base[k] = 0;
    make_plan<kPromptThreads>(c, rows, ws, a.window, a.sinks, 2 * tq, gridDim.x, blockIdx.x, blockIdx.x + 1);
    __syncthreads();
  }

  Walk w;
  const bool any = w.begin(ws, c.kv_heads, blockIdx.x);
  const Patience patience{&wait_limit};
  if (threadIdx.x == 0) wait_limit = ws.waits.ns + static_cast<unsigned long long>(ws.waits.tile_ns) * (any ? w.end : 0);
  __syncthreads();

  if (warp == 9) {
    // ---- TMA producer.  Order: keys 0, then values t, keys t + 1, as they are used.
    int it = 0;
    const int rows_per_box = min(kKeys, c.page_size), boxes = kKeys / rows_per_box;
    const int beyond = c.pages * c.layers * 2 * c.kv_heads * c.page_size;  // a row past the pool: reads zeros
    for (bool more = any && !ws.waits.starve; more && alive(errv); more = w.next(ws)) {
      const Geom g = w.g;
      const KeySpan span = unit_span(w, prefix, tq, a);
      const int32_t* table = c.table + static_cast<int64_t>(g.key_slot) * c.table_pages;
      // the row of the pool, before the choice of keys or values, where lane's box of tile t begins
      auto page_of = [&](int t) {
        const int key = kKeys * span.tile(t) + lane * rows_per_box;
        return lane < boxes && t < w.t1 && key < g.len ? table[key >> c.page_shift] : -1;
      };
      auto copy = [&](int t, int page, int kv) {
        const int s = it % S;
        if (it >= S && !patience.wait(&kv_empty[s], ((it / S) - 1) & 1)) return false;
        ++it;
        if (lane == 0) mbar_expect_tx(&kv_full[s], C::kTileBytes);
        __syncwarp();
        if (lane < boxes) {
          const int in_page = (kKeys * span.tile(t) + lane * rows_per_box) & (c.page_size - 1);
          const int y = c.is_page(page) ? (((page * c.layers + a.layer) * 2 + kv) * c.kv_heads + w.head) * c.page_size + in_page
                                        : beyond;
          unsigned char* dst = ring + static_cast<size_t>(s) * C::kTileBytes + lane * rows_per_box * 128;
#pragma unroll
          for (int b = 0; b < DB; ++b) tma_load_2d(dst + b * (kKeys * 128), &pool_map, 64 * b, y, &kv_full[s]);
        }
        return true;
      };
      int page = page_of(w.t0), next_page = page_of(w.t0 + 1);
      bool ok = copy(w.t0, page, 0);
      for (int t = w.t0; ok && t < w.t1; ++t) {
        const int ahead = page_of(t + 2);  // on its way while the copies wait for their stages
        ok = copy(t, page, 1);
        if (ok && t + 1 < w.t1) ok = copy(t + 1, next_page, 0);
        page = next_page;
        next_page = ahead;
      }
      if (!ok) *errv = 1;
    }
    // no copy may still be landing in shared memory when the CTA leaves
    if (lane == 0)
      for (int k = max(0, it - S); k < it; ++k) drain(&kv_full[k % S], (k / S) & 1);
  } else if (warp == 10) {
    // ---- value rows that no query of the unit may see are cleared before the MMA warp may use the tile.  Key tiles pass
    // through too: so neither this warp nor the MMA warp is ever a round of the ring away from the other.
    int it = 0;
    for (bool more = any; more && alive(errv); more = w.next(ws)) {
      const Geom g = w.g;
      const KeySpan span = unit_span(w, prefix, tq, a);
      const bool* mask = a.key_mask != nullptr ? a.key_mask + g.key_slot * a.mask_stride : nullptr;
      int p0, p1;
      positions(g, prefix, w.tok0, w.tok0 + 2 * tq, &p0, &p1);
      const bool zero_tail = p1 + 1 == g.len && (g.len & (c.page_size - 1)) == 0;  // keys past it came as zeros
      auto pass = [&](int t) {  // the ring's next tile: values of tile t, or keys (t < 0)
        const int s = it % S;
        if (!patience.wait(&kv_full[s], (it / S) & 1)) return false;
        ++it;
        const int base = t < 0 ? 0 : kKeys * span.tile(t);
        if (t >= 0 && (mask != nullptr || (base + kKeys > p1 + 1 && !zero_tail) ||
                       (a.window > 0 && base <= p0 - a.window && base + kKeys > a.sinks))) {
          unsigned char* v = ring + static_cast<size_t>(s) * C::kTileBytes;
          for (int r = lane; r < kKeys; r += 32) {
            const int j = base + r;
            const bool keep =
                j <= p1 && (a.window == 0 || j > p0 - a.window || j < a.sinks) && (mask == nullptr || mask[j]);
            if (!keep) {
#pragma unroll
              for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  *reinterpret_cast<uint4*>(v + b * (kKeys * 128) + r * 128 + 16 * k) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&ready[s]);
        return true;
      };
      bool ok = pass(-1);
      for (int t = w.t0; ok && t < w.t1; ++t) {
        ok = pass(t);
        if (ok && t + 1 < w.t1) ok = pass(-1);
      }
      if (!ok) *errv = 1;
    }
  } else if (warp == 11) {
    // ---- queries: a box of 64 dims x the group's heads x the tile's tokens, whose rows are the tile's
    int units[2] = {0, 0};  // whose queries have been asked for
    for (bool more = any && rows.q_mapped; more && alive(errv); more = w.next(ws)) {
      bool ok = true;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (units[i] > 0) ok = ok && patience.wait(&q_free[i], (units[i] - 1) & 1);
        if (ok) ++units[i];
        if (ok && lane == 0) {
          mbar_expect_tx(&q_ready[i], static_cast<uint32_t>(tq * a.group * D * 2));
#pragma unroll
          for (int b = 0; b < DB; ++b)
            tma_load_3d(q_smem + i * C::kQBytes + b * (kTile * 128), &q_map, 64 * b, w.head * a.group,
                        w.g.row0 + w.tok0 + i * tq, &q_ready[i]);
        }
        __syncwarp();
      }
      if (!ok) *errv = 1;
    }
    // no copy may still be landing in shared memory when the CTA leaves
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (units[i] > 0) drain(&q_ready[i], (units[i] - 1) & 1);
    }
  } else if (warp == 8) {
    // ---- MMA issuer.  The whole warp walks along, so that what the
    // instructions are given stays in uniform registers (from a single thread's
    // branch an MMA took 89 cycles to issue instead of 64); one elected thread
    // issues them.  Only the descriptors' low words change.
    int it = 0;  // ring position
    int p_uses[2] = {0, 0}, q_uses = 0;
    const uint32_t q_lo = static_cast<uint32_t>(umma_desc_sw128(q_smem));
    const uint32_t k_lo = static_cast<uint32_t>(umma_desc_sw128(ring));
    const uint32_t v_lo = static_cast<uint32_t>(value_desc(smem_addr(ring)));
    constexpr uint32_t kTileStep = C::kTileBytes >> 4, kBlock = (kTile * 128) >> 4;
    auto scores = [&](int i, int s) {  // S_i = Q_i K^T
      const uint32_t qd = q_lo + i * (C::kQBytes >> 4), kd = k_lo + s * kTileStep;
      if (elect_one()) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ss(tmem + kSCol + i * kKeys, qd + d * kBlock + 2 * kk, kd + d * kBlock + 2 * kk,
                    prompt_idesc<T>(kKeys, false), (d | kk) != 0);
        umma_commit(&s_full[i]);
      }
      __syncwarp();
    };
    auto commit = [&](unsigned long long* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    bool more = any;
    while (more && alive(errv)) {
      int q0[2], q1[2];
      positions(w.g, prefix, w.tok0, w.tok0 + tq, &q0[0], &q1[0]);
      positions(w.g, prefix, w.tok0 + tq, w.tok0 + 2 * tq, &q0[1], &q1[1]);
      const KeySpan span = unit_span(w, prefix, tq, a);
      const TilesSeen seen[2] = {TilesSeen(q0[0], q1[0], a.window, a.sinks), TilesSeen(q0[1], q1[1], a.window, a.sinks)};
      bool started[2] = {false, false};
      const int t0 = w.t0, t1 = w.t1;
      int last[2];  // each Q tile's last key tile in this share
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        last[i] = seen[i].high < 0 ? t0 - 1 : t1 - 1;
        while (last[i] >= t0 && !seen[i].at(span.tile(last[i]))) --last[i];
      }
      more = w.next(ws);  // its loads are on their way while this unit runs
      bool ok = patience.wait(&ready[it % S], (it / S) & 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ok = ok && patience.wait(&q_ready[i], q_uses & 1);
        if (ok) {
          tmem_fence_after_sync();
          if (seen[i].at(span.tile(t0))) scores(i, it % S);
          if (last[i] <= t0) commit(&q_free[i]);  // (a Q tile without key tiles in this share: at once)
        }
      }
      ++q_uses;
      if (ok) commit(&kv_empty[it % S]);
      ++it;
      for (int t = t0; ok && t < t1; ++t) {
        const int vs = it % S, ks = (it + 1) % S;
        const bool next = t + 1 < t1;
        ok = patience.wait(&ready[vs], (it / S) & 1);
        if (next) ok = ok && patience.wait(&ready[ks], ((it + 1) / S) & 1);
        const int j = span.tile(t), j1 = next ? span.tile(t + 1) : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (seen[i].at(j)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ok = ok && patience.wait(&p_full[i][h], p_uses[i] & 1);
              if (ok) {
                tmem_fence_after_sync();
                const uint32_t vd = v_lo + vs * kTileStep + h * (kHalf * 128 >> 4);
                if (elect_one()) {
#pragma unroll
                  for (int kk = 0; kk < kHalf / 16; ++kk)
                    umma_ts(tmem + kOCol + i * D, tmem + kSCol + i * kKeys + h * (kHalf / 2) + 8 * kk, vd + kk * (2048 >> 4),
                            prompt_idesc<T>(D, true), started[i] || (h | kk) != 0);
                  if (h == 0) umma_commit(&half_done[i]);
                }
                __syncwarp();
              }
            }
            ++p_uses[i];
            started[i] = true;
            if (ok && t == last[i]) commit(&o_full[i]);
          }
          if (ok && next && seen[i].at(j1)) {
            scores(i, ks);
            if (t + 1 == last[i]) commit(&q_free[i]);
          }
        }
        if (ok) {
          commit(&kv_empty[vs]);
          if (next) commit(&kv_empty[ks]);
          it += next ? 2 : 1;
        }
      }
      if (!ok) *errv = 1;
    }
    // every MMA this warp issued has completed before tensor memory is freed
    commit(&fin);
    drain(&fin, 0);
  } else {
    // ---- softmax of Q tile i: thread r is its row r
    const int i = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_col = tmem + kSCol + i * kKeys + lanes, o_col = tmem + kOCol + i * D + lanes;
    const int tok_in_tile = r / a.group, head_in_group = r % a.group;
    // Whole rows go to global memory: 8 lanes a 128-byte piece, 4 rows at a time (a thread per row would touch 32
    // sectors with every instruction, which took longer than several key tiles).
    const int piece = lane & 7, sub_row = lane >> 3;
    int s_uses = 0, o_uses = 0, unit = 0;
    // this thread's row of unit u: q and out row, or -1
    auto row_of = [&](const Walk& u) {
      const int tok = u.tok0 + i * tq + tok_in_tile;
      if (tok_in_tile >= tq || tok >= u.g.count) return -1;
      const int row = prefix ? rows.members[u.g.row0 + tok] : u.g.row0 + tok;
      return row >= 0 && row < a.rows ? row : -1;
    };
    // without a query map: the warp's 32 rows of queries into shared memory
    auto load_q = [&](const Walk& u, int row) {
      const uint16_t* src = a.q + static_cast<int64_t>(u.head * a.group) * D + 8 * piece;
      unsigned char* dst = q_smem + i * C::kQBytes + 32 * (warp & 3) * 128;
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int from = 4 * k + sub_row;
          const int q_row = __shfl_sync(0xffffffffu, row, from), h = __shfl_sync(0xffffffffu, head_in_group, from);
          v[k] = q_row >= 0 ? *reinterpret_cast<const uint4*>(src + q_row * a.q_row + h * D + 64 * b)
                            : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int to = 4 * k + sub_row;
          *reinterpret_cast<uint4*>(dst + b * (kTile * 128) + to * 128 + 16 * (piece ^ (to & 7))) = v[k];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[i]);
    };
    int q_row = -1;
    if (any) {
      q_row = row_of(w);
      if (!rows.q_mapped) load_q(w, q_row);
    }
    for (bool more = any; more && alive(errv); ++unit) {
      int q0, q1;
      positions(w.g, prefix, w.tok0 + i * tq, w.tok0 + (i + 1) * tq, &q0, &q1);
      const TilesSeen seen(q0, q1, a.window, a.sinks);
      const KeySpan span = unit_span(w, prefix, tq, a);
      const int len = w.g.len, t0 = w.t0, t1 = w.t1, q_head = w.head * a.group + head_in_group;
      const int pos = prefix ? len - 1 : len - w.g.count + w.tok0 + i * tq + tok_in_tile;
      const bool* mask = a.key_mask != nullptr ? a.key_mask + w.g.key_slot * a.mask_stride : nullptr;
      const bool whole = w.whole();
      const int part_at = 2 * static_cast<int>(blockIdx.x) + w.part();
      more = w.next(ws);  // from here on w is the next unit: its loads are on their way while this one runs
      const int next_row = more ? row_of(w) : -1;
      float m = -CUDART_INF_F, l = 0.f;
      bool ok = true, started = false;
      for (int t = t0; t < t1; ++t) {
        const int j = span.tile(t);
        if (!seen.at(j)) continue;
        const int base = kKeys * j;
        const bool all = mask == nullptr && tile_full(j, q0, q1, a.window, a.sinks) && base + kKeys <= len;
        uint32_t kept[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (mask != nullptr) {  // before the wait, which covers the loads
          bool on[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) on[x] = base + 32 * x + lane < len && mask[base + 32 * x + lane];
#pragma unroll
          for (int x = 0; x < 4; ++x) kept[x] = __ballot_sync(0xffffffffu, on[x]);
        }
        ok = patience.wait(&s_full[i], s_uses & 1);
        if (!ok) break;
        tmem_fence_after_sync();
        // One half after the other, so that 64 scores are held and not 128: P of
        // the first half goes over the first half's scores alone.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t s[kHalf];
          tmem_ld64(s, s_col + kHalf * h);
          if (!all) {
            const int from = base + kHalf * h;
            const int hi = min(pos + 1, len) - from;
            const int lo = a.window > 0 ? max(max(pos + 1 - from, 0) - a.window, 0) : 0;
            const int sk = min(a.sinks, from + kHalf) - from;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t see = kept[2 * h + x] & bit_range(0, hi - 32 * x) &
                                   (bit_range(lo - 32 * x, 32) | bit_range(0, sk - 32 * x));
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((see >> k) & 1u)) s[32 * x + k] = 0xff800000u;
            }
          }
          float sum;
          auto probabilities = [&] {
            const float off = m == -CUDART_INF_F ? 0.f : fmaf(-m, a.scale2, kPromptBias<T>);
            const float2 scale = make_float2(a.scale2, a.scale2), offs = make_float2(off, off);
            float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t p[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int e = 32 * x + 2 * k;
                float2 v = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale, offs);
                v.x = ex2(v.x);
                v.y = ex2(v.y);
                // the sum keeps the unrounded probabilities; the values' weights are rounded to 16 bits once
                sums[k & 1] = add2(sums[k & 1], v);
                p[k] = Half16<T>::pack(v.x, v.y);
              }
              tmem_st16(s_col + (kHalf / 2) * h + 16 * x, p);
            }
            sums[0] = add2(sums[0], sums[1]);
            sum = sums[0].x + sums[0].y;
          };
          bool find = h == 0 && !started;
          while (true) {
            if (find) {
              float top = m;
#pragma unroll
              for (int k = 0; k < kHalf; k += 2) top = max_nan(top, __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
              if (started || h == 1) {
                // the products so far must be in O: those of the tiles before are (these scores came after them)
                if (h == 1) ok = patience.wait(&half_done[i], s_uses & 1);
                if (!ok) break;
                tmem_fence_after_sync();
                const float f = m == -CUDART_INF_F ? 1.f : ex2((m - top) * a.scale2);
                l *= f;
#pragma unroll 1
                for (int b = 0; b < D / 16; ++b) {
                  uint32_t o[16];
                  tmem_ld16(o, o_col + 16 * b);
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                  tmem_st16(o_col + 16 * b, o);
                }
              }
              m = top;
            }
            probabilities();
            if (find || !__any_sync(0xffffffffu, q_row >= 0 && (!(sum <= 32768.f) || m == -CUDART_INF_F))) break;
            find = true;
          }
          if (!ok) break;
          l += sum;
          tmem_wait_st();
          tmem_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[i][h]);
        }
        if (!ok) break;
        ++s_uses;
        started = true;
      }
      if (ok && more && !rows.q_mapped) {  // before this unit's result comes out
        ok = patience.wait(&q_free[i], unit & 1);
        if (ok) load_q(w, next_row);
      }
      if (ok && started) ok = patience.wait(&o_full[i], o_uses++ & 1);
      if (!ok) {
        *errv = 1;
        break;
      }
      tmem_fence_after_sync();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float m2 = m == -CUDART_INF_F ? m : fmaf(m, a.scale2, -kPromptBias<T>);
      const bool there = q_row >= 0;
      float* part = ws.part + static_cast<int64_t>(part_at) * (D + 2) * kPairRows + i * kTile + r;
      float* state = prefix && there ? rows.state + (static_cast<int64_t>(q_row) * a.q_heads + q_head) * (D + 4) : nullptr;
      unsigned char* stage = out_smem + warp * (32 * 128);
      // where the 8 rows whose pieces this lane stores go (null: nowhere)
      uint16_t* to[8];
      {
        uint16_t* mine = there ? a.out + q_row * a.out_row + static_cast<int64_t>(q_head) * D : nullptr;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          to[k] = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), 4 * k + sub_row));
      }
#pragma unroll
      for (int b = 0; b < DB; ++b) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t o[32];
          tmem_ld32(o, o_col + 64 * b + 32 * half);
          if (!started) {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0u;
          }
          if (!whole) {
            if (there) {
#pragma unroll
              for (int k = 0; k < 32; ++k) part[(64 * b + 32 * half + k) * kPairRows] = __uint_as_float(o[k]);
            }
          } else if (prefix) {
            if (there) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                *reinterpret_cast<uint4*>(state + 64 * b + 32 * half + 4 * k) =
                    make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint4 y;
              y.x = Half16<T>::pack(__uint_as_float(o[8 * k]) * inv, __uint_as_float(o[8 * k + 1]) * inv);
              y.y = Half16<T>::pack(__uint_as_float(o[8 * k + 2]) * inv, __uint_as_float(o[8 * k + 3]) * inv);
              y.z = Half16<T>::pack(__uint_as_float(o[8 * k + 4]) * inv, __uint_as_float(o[8 * k + 5]) * inv);
              y.w = Half16<T>::pack(__uint_as_float(o[8 * k + 6]) * inv, __uint_as_float(o[8 * k + 7]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * 128 + 16 * ((4 * half + k) ^ (lane & 7))) = y;
            }
          }
          __syncwarp();
        }
        if (whole && !prefix) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int from = 4 * k + sub_row;
            const uint4 y = *reinterpret_cast<const uint4*>(stage + from * 128 + 16 * (piece ^ (from & 7)));
            if (to[k] != nullptr) *reinterpret_cast<uint4*>(to[k] + 64 * b + 8 * piece) = y;
          }
          __syncwarp();
        }
      }
      if (there) {
        if (!whole) {
          part[D * kPairRows] = m2;
          part[(D + 1) * kPairRows] = l;
        } else if (prefix) {
          *reinterpret_cast<float2*>(state + D) = make_float2(m2, l);
        } else if (a.lse != nullptr) {
          a.lse[static_cast<int64_t>(q_row) * a.q_heads + q_head] = (m2 + log2f(l)) * kLn2;
        }
      }
      tmem_fence_before_sync();
      q_row = next_row;
    }
    tmem_wait_st();  // also where a wait ran out between a store and its use
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    tmem_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) ws.gave_up[blockIdx.x] = *errv;
}

// Prefix pass: how many of each member's tokens it has attended to (base is 0 so far).
__device__ void member_bases(const PagedCache& c, const PromptRows& rows) {
  for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < rows.n_rows; k += gridDim.x * blockDim.x) {
    int lo = 0, hi = rows.n;  // the group whose members begin at or before k
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (rows.offsets[mid] <= k) lo = mid; else hi = mid;
    }
    const PairGeom g(c, rows, lo);
    const int slot = rows.members[k];
    if (!g.ok || k < g.row0 || k >= g.row0 + g.count || slot < 0 || slot >= c.slots || c.length(slot) < g.len) continue;
    const int last = (g.len >> c.page_shift) - 1;
    if (c.table[static_cast<int64_t>(slot) * c.table_pages + last] ==
        c.table[static_cast<int64_t>(g.key_slot) * c.table_pages + last])
      rows.base[slot] = g.len;
  }
}

// Status 4: of a prompt's slots, those with units in the shares of the CTAs that
// gave up (thread c's says whether CTA c did); of a prefix pass, all members.
__device__ void mark_lost(const PagedCache& c, const PromptRows& rows, const PromptSpace& ws, bool gave_up) {
  if (rows.members != nullptr) {
    for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < rows.n_rows; k += gridDim.x * blockDim.x) {
      const int slot = rows.members[k];
      if (slot >= 0 && slot < c.slots) c.status[slot] = 4;
    }
  } else if (gave_up && blockIdx.x == 0) {
    Walk w;
    for (bool more = w.begin(ws, c.kv_heads, threadIdx.x); more; more = w.next(ws)) c.status[w.g.key_slot] = 4;
  }
}

// Joins the parts of the units that a boundary between CTAs cut.  Every CTA
// lists these units (by the CTA in whose share the first boundary between their
// key tiles falls) and takes its share of their blocks of 32 rows and 32 dims.
// Also gives rows that no slot has their zeros.
// (A CTA for each boundary and block, most without work: 65 slots over
// 32,768 tokens 111.0 us a call instead of 106.7.)
constexpr int kJoinParts = 8;  // parts on their way at a time
constexpr int kJoinThreads = 256;  // more than there are boundaries
static_assert(kJoinThreads >= kMaxSms);

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    prompt_join_kernel(PagedCache c, Attend a, PromptRows rows, PromptSpace ws, int ctas) {
  __shared__ int cut[kJoinThreads], warp_cuts[kJoinThreads / 32];
  take_turn();
  const bool prefix = rows.members != nullptr;
  const bool mine_gave_up = threadIdx.x < ctas && ws.gave_up[threadIdx.x] != 0;
  const int row0 = rows.offsets[0], row1 = rows.offsets[rows.n];  // slots have the rows between
  const int64_t line = ws.head[1], per = ws.head[2];
  int cuts = 0;
  {
    const int cta = threadIdx.x + 1, warp = threadIdx.x >> 5;
    const int64_t x = cta * per;
    bool mine = false;
    if (cta < ctas && x < line * c.kv_heads) {
      const int4 rec = ws.rec[2 * ws.cta_pair[cta]];
      const int64_t tile_x = x / line * line + pair_place(rec) + kPairCost;
      mine = x > tile_x && x - per <= tile_x;
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0) warp_cuts[warp] = __popc(votes);
    const bool gave_up = __syncthreads_or(mine_gave_up);
    if (prefix && !gave_up) member_bases(c, rows);
    if (gave_up && c.status != nullptr) mark_lost(c, rows, ws, mine_gave_up);
    int before = 0;
#pragma unroll
    for (int k = 0; k < kJoinThreads / 32; ++k) {
      if (k < warp) before += warp_cuts[k];
      cuts += warp_cuts[k];
    }
    if (mine) cut[before + __popc(votes & ((1u << (threadIdx.x & 31)) - 1u))] = cta;
    __syncthreads();
  }
  const int tq = kTile / a.group;
  constexpr int kBlocks = (kPairRows / 32) * (D / 32);
  for (int item = blockIdx.x; item < cuts * kBlocks; item += gridDim.x) {
    const int cta = cut[item / kBlocks];
    const int64_t x = cta * per;
    const int head = static_cast<int>(x / line);
    const int pair = ws.cta_pair[cta];
    const int4 rec = ws.rec[2 * pair], at = ws.rec[2 * pair + 1];
    const Geom g{at.x, at.y, at.z, at.w};
    const int64_t unit_x = head * line + pair_place(rec), tile_x = unit_x + kPairCost;
    const int n = static_cast<int>((tile_x + rec.z - 1) / per) - cta + 2;  // parts, from CTA cta - 1 on
    const int r = 32 * (item % kBlocks / (D / 32)) + (threadIdx.x & 31);
    const int i = r / kTile, rr = r % kTile;
    const int tok = rec.x + i * tq + rr / a.group;
    if (rr / a.group >= tq || tok >= g.count) continue;
    int q_row = g.row0 + tok;
    if (prefix) {
      q_row = rows.members[q_row];
      if (q_row < 0 || q_row >= a.rows) continue;
    }
    const int q_head = head * a.group + rr % a.group;
    constexpr int E = 4;  // dims per thread
    const int d0 = 32 * (item % (D / 32)) + E * (threadIdx.x >> 5);
    const int64_t stride = static_cast<int64_t>(D + 2) * kPairRows;
    const float* parts = ws.part + 2 * (cta - 1) * stride + r;
    const int64_t first = ((cta - 1) * per >= unit_x ? 0 : 1) * stride;
    float top = -CUDART_INF_F, l = 0.f, o[E] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += kJoinParts) {
      float m[kJoinParts], s[kJoinParts], y[kJoinParts][E];
  #pragma unroll
      for (int k = 0; k < kJoinParts; ++k) {
        const bool on = k0 + k < n;
        const float* p = parts + (k0 + k == 0 ? first : 2 * (k0 + k) * stride);
        m[k] = on ? __ldcg(p + D * kPairRows) : -CUDART_INF_F;
        s[k] = on ? __ldcg(p + (D + 1) * kPairRows) : 0.f;
  #pragma unroll
        for (int e = 0; e < E; ++e) y[k][e] = on ? __ldcg(p + (d0 + e) * kPairRows) : 0.f;
      }
      float most = top;
  #pragma unroll
      for (int k = 0; k < kJoinParts; ++k) most = fmaxf(most, m[k]);
      const float z = most == -CUDART_INF_F ? 0.f : most;
      const float keep = ex2(top - z);
      top = most;
      l *= keep;
  #pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= keep;
  #pragma unroll
      for (int k = 0; k < kJoinParts; ++k) {
        const float f = ex2(m[k] - z);
        l = fmaf(f, s[k], l);
  #pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(f, y[k][e], o[e]);
      }
    }
    if (prefix) {
      float* state = rows.state + (static_cast<int64_t>(q_row) * a.q_heads + q_head) * (D + 4);
      *reinterpret_cast<float4*>(state + d0) = make_float4(o[0], o[1], o[2], o[3]);
      if (d0 == 0) *reinterpret_cast<float2*>(state + D) = make_float2(top, l);
      continue;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(a.out + q_row * a.out_row + static_cast<int64_t>(q_head) * D + d0) =
        make_uint2(Half16<T>::pack(o[0] * inv, o[1] * inv), Half16<T>::pack(o[2] * inv, o[3] * inv));
    if (d0 == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(q_row) * a.q_heads + q_head] = (top + log2f(l)) * kLn2;
  }
  // rows that no slot has see nothing
  if (!prefix && row0 >= 0 && row0 <= row1 && row1 <= a.rows && row1 - row0 < a.rows) {
    const int64_t pieces = static_cast<int64_t>(a.q_heads) * (D / 8), all = (row0 + a.rows - row1) * pieces;
    for (int64_t e = blockIdx.x * kJoinThreads + threadIdx.x; e < all; e += gridDim.x * kJoinThreads) {
      const int k = static_cast<int>(e / pieces), at = static_cast<int>(e % pieces);
      const int64_t row = k < row0 ? k : row1 + k - row0;
      *reinterpret_cast<uint4*>(a.out + row * a.out_row + 8 * at) = make_uint4(0, 0, 0, 0);
      if (at % (D / 8) == 0 && a.lse != nullptr) a.lse[row * a.q_heads + at / (D / 8)] = -CUDART_INF_F;
    }
  }
}

// Bytes of the parts of a prompt call's workspace.
struct PromptLayout {
  size_t cta_pair, gave_up, first, rec, part, bytes;
  PromptLayout(int n, int rows, int group, int head_dim) {
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t pairs = static_cast<size_t>(rows) / (2 * (kTile / group)) + n + 1;
    cta_pair = 256;
    gave_up = cta_pair + up(4 * (kMaxSms + 1));
    first = gave_up + up(4 * kMaxSms);
    rec = first + up(4 * (static_cast<size_t>(n) + 1));
    part = rec + up(32 * pairs);
    bytes = part + up(static_cast<size_t>(kMaxSms) * 2 * (head_dim + 2) * kPairRows * 4);
  }
};

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn find_encode() {
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q{};
  const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                  q == cudaDriverEntryPointSuccess;
  cudaGetLastError();
  return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
}

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = find_encode();
  return fn;
}

// The pool as a matrix of rows (one token's keys or values of one head); a
// box is one page's rows of one head (at most a key tile's), 64 dims wide.
bool pool_map(const PagedCache& c, int dtype, CUtensorMap* map) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t rows = static_cast<cuuint64_t>(c.pages) * c.layers * 2 * c.kv_heads * c.page_size;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(c.head_dim), rows};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(c.head_dim) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(std::min(c.page_size, kKeys))};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map,
            dtype == MTT_B200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
            c.pool, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The queries as [rows][heads][head_dim]; a box is a Q tile's tokens, its group's heads and 64 dims.
bool query_map(const PagedCache& c, int dtype, const Attend& a, CUtensorMap* map) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(a.q_heads),
                              static_cast<cuuint64_t>(a.rows)};
  const cuuint64_t row = static_cast<cuuint64_t>(a.rows == 1 ? static_cast<int64_t>(a.q_heads) * c.head_dim : a.q_row) * 2;
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.head_dim) * 2, row};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(kTile / a.group)};
  const cuuint32_t elem[3] = {1, 1, 1};
  return row >= dims[0] * dims[1] * 2 &&
         fn(map, dtype == MTT_B200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<uint16_t*>(a.q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
             CUDA_SUCCESS;
}

cudaError_t run_prompt(const PagedCache& c, int dtype, const Attend& a, PromptRows rows, void* space,
                       const Waits& waits, cudaStream_t stream) {
  const int sms = cache_sm_count();
  CUtensorMap map, q_map;
  if (sms <= 0 || sms > kMaxSms || !pool_map(c, dtype, &map)) return cudaErrorInvalidValue;
  rows.q_mapped = rows.members == nullptr && query_map(c, dtype, a, &q_map);
  if (!rows.q_mapped) q_map = map;  // not read
  const int tokens_per_pair = 2 * (kTile / a.group);
  rows.own_plan = rows.n_rows / tokens_per_pair + rows.n <= kPromptThreads;
  const PromptLayout at(rows.n, rows.n_rows, a.group, c.head_dim);
  char* base = static_cast<char*>(space);
  PromptSpace ws;
  ws.head = reinterpret_cast<int64_t*>(base);
  ws.cta_pair = reinterpret_cast<int32_t*>(base + at.cta_pair);
  ws.gave_up = reinterpret_cast<int32_t*>(base + at.gave_up);
  ws.first = reinterpret_cast<int32_t*>(base + at.first);
  ws.rec = reinterpret_cast<int4*>(base + at.rec);
  ws.part = reinterpret_cast<float*>(base + at.part);
  ws.waits = waits;
  auto go = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    const auto kernel = prompt_kernel<T, D>;
    constexpr size_t smem = PromptCfg<D>::kSmem;
    static std::atomic<uint64_t> opted_in;  // devices on which this kernel has its shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1))) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e == cudaSuccess && dev < 64) opted_in.fetch_or(uint64_t{1} << dev, std::memory_order_relaxed);
    }
    if (e == cudaSuccess && !rows.own_plan)
      e = launch_serialized(prompt_plan_kernel, dim3(1), dim3(kPromptPlanThreads), 0, stream, c, rows, ws, a.window,
                            a.sinks, tokens_per_pair, sms);
    if (e == cudaSuccess) e = launch_serialized(kernel, dim3(sms), dim3(kPromptThreads), smem, stream, map, q_map, c, a, rows, ws);
    if (e == cudaSuccess)
      e = launch_serialized(prompt_join_kernel<T, D>, dim3(4 * sms), dim3(kJoinThreads), 0, stream, c, a, rows, ws, sms);
    return e;
  };
  auto pick = [&](auto type) {
    return c.head_dim == 64 ? go(type, std::integral_constant<int, 64>{}) : go(type, std::integral_constant<int, 128>{});
  };
  return dtype == MTT_B200_DTYPE_BF16 ? pick(__nv_bfloat16{}) : pick(__half{});
}

}  // namespace

size_t prompt_workspace(const mtt_b200_paged_cache_t& c, int q_heads, int rows) {
  return PromptLayout(c.slots, rows, q_heads / c.kv_heads, c.head_dim).bytes;
}

cudaError_t launch_prompt(const PagedCache& c, int dtype, const Attend& a, void* space, const Waits& waits,
                          cudaStream_t stream) {
  PromptRows rows{};
  rows.n = c.slots;
  rows.n_rows = a.rows;
  rows.offsets = a.offsets;
  return run_prompt(c, dtype, a, rows, space, waits, stream);
}

cudaError_t launch_prefix(const PagedCache& c, int dtype, const Attend& a, const mtt_b200_prefix_groups_t& groups,
                          int32_t* base, float* state, void* space, const Waits& waits, cudaStream_t stream) {
  PromptRows rows{};
  rows.n = groups.n_groups;
  rows.n_rows = groups.n_members;
  rows.offsets = groups.offsets;
  rows.members = groups.members;
  rows.voice = groups.voice;
  rows.tokens = groups.tokens;
  rows.longest = a.window > 0 ? a.sinks : INT32_MAX;
  rows.base = base;
  rows.state = state;
  Attend all = a;  // every member sees the whole prefix
  all.window = all.sinks = 0;
  return run_prompt(c, dtype, all, rows, space, waits, stream);
}

}  // namespace mtt

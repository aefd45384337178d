// Attention of one new token per slot over the paged cache.
//
//   out = sum_j e^{s q.k_j} v_j / sum_j e^{s q.k_j} over the keys the window,
//   the sinks and the mask leave: one pass with a running maximum and sum.
//
// Every key and value is used for one query row of each query head that
// shares the key head, so HBM bounds it: 4 x head_dim bytes per key and key
// head.  The design keeps those bytes in flight and everything else cheap:
//  * Keys and values go from global memory straight into the registers that
//    mma.sync reads, 16 bytes a load, with no shared memory between.  A
//    warp's step is 16 keys (32 with head_dim 64).  Scores are S^T = K Q^T
//    with the keys on the MMA's 16-row side and up to 8 query heads on its
//    8-column side (a step of one query head costs no more).  The
//    contraction's order is free, so a thread's A fragment is simply its 16
//    bytes of the key row; matrix transposes turn P^T into the B operand of
//    O^T += V^T P^T (once for its 16-bit rounding, once for the rest), and
//    V^T's fragments are byte permutes of two keys' 16-byte pieces.  (tcgen05 would want the same bytes staged in shared
//    memory for a tile of 128 rows of which 1 to 16 are real.)
//  * The work is one line of 16-key tiles over all (slot, key head) units,
//    cut into equal parts for the warps of a grid that fills the device, so
//    ragged lengths balance by themselves and no warp waits for another.  A
//    unit that a cut divides leaves (maximum, sum, weighted values) of each
//    part in the workspace; a second kernel joins the parts in their order,
//    so the result does not depend on timing.
//  * Few slots, whose call is launches and latency, take clusters instead
//    (step_few_kernel): one launch.
// Measured, line and join: 512 slots of 12 heads of 64, up to 1242 of 2048 keys in
// reach, 164 us (974 MB from DRAM, where masked keys are not read: 5.9 TB/s); 8
// slots of 30,001 to 65,536 keys, 32/8 heads of 128, 239 to 251 us from one GPU to
// another (6.3 to 6.0 TB/s).  Clusters: 2 slots of 467 keys, 12 heads of 64, 5.4 us
// (9.0 us as a line).  What bounds the line is DRAM; where sequences are short (1
// to 249 keys) a unit's chain of dependent loads (65 us for 275 MB).  The second
// product of the values costs 1%.  Tried, before it: shares per CTA with the four
// warps of a CTA side by side in a unit (187 and 247 us, 389 us for the short ones,
// when the line took 162 and 238); a unit's further tiles prefetched into L2 when
// it is entered (249 -> 253 us, the short ones 10 us more).
//
// A pool in 4 bits (attend_tiles4) takes 9/32 of the bytes: the same 512 slots 108 us
// (306 MB, 2.8 TB/s), the same 8 slots in f16 135 us (422 MB, 3.1 TB/s).  Nothing is full
// there: the logic pipe is busy 66 and 64% of the time, the schedulers 51 and 52, with 13
// and 10 warps an SM (128 and 168 registers) to cover a step's chain of load, score,
// maximum and weight.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cache4.cuh"

namespace mtt {
namespace {

constexpr int kStepWarps = 4;
constexpr int kStepThreads = 32 * kStepWarps;

// Forms of the kernels: 16 for a pool in 16 bits; for one in 4 bits how many query
// heads a key head has at most: 1, 2, 4, 8 or more (9).  (Two heads of 128 dims take
// form 4, whose two tiles a step leave registers: 16 slots of 16,384 keys, 8 key
// heads, 101 us instead of 107.  Heads of 64 dims: 115 instead of 99.)
constexpr int step_form(int bits, int head_dim, int group) {
  if (bits == 16) return 16;
  if (group > 4) return group > 8 ? 9 : 8;
  return group > 2 || (group == 2 && head_dim == 128) ? 4 : group;
}

// 16-key tiles per warp and step.  (4 bits, the same keys, or twice as many with 64
// dims, in us with 4 / 2 / 1 tiles: 4 heads of 64 116 / 113 / -, 8 of 64 177 / 129 /
// 143, 8 of 128 - / 124 / 129, 16 of 64 490 / 190 / 191, 16 of 128 - / 263 / 185:
// what does not fit the registers is what costs.  Since bf16's off is held as an eighth
// 16 of 64 take 196 us and 16 of 128 191, the others within 1% of these.)
constexpr int step_tiles(int head_dim, int form) {
  if (form == 16) return head_dim == 64 ? 2 : 1;
  return form == 9 ? 1 : form >= 4 ? 2 : 4;
}
constexpr int step_ctas(int head_dim, int nb) {  // per SM (registers)
  return (head_dim == 64 ? 4 : 3) - (nb == 2 ? 1 : 0);
}

// A unit's place on the line: its tiles, and before them what entering and
// leaving it costs, in tiles.  (2052 slots with 1 to 249 keys each, prefix pass
// included: 134 us with 0, 96 with 2, 104 with 4, 116 with 8.)
// (512 sessions over a 4-bit pool: 113 us with 2, 109 with 4.)
constexpr int unit_cost(int form) { return form == 16 ? 2 : 4; }

// Probabilities are held 2^15 times as large where the cache is f16, so that what
// is small beside the largest (1) stays in that type's range; sums and weighted
// values share the factor, and the maximum that goes with them is less by 15.
template <typename T>
constexpr float kStepBias = std::is_same_v<T, __half> ? 15.f : 0.f;

struct StepSpace {
  int4* cut;    // [warps]: the cut unit that begins in the warp's share: slot, unit, warps that hold it (0: none)
  float* part;  // [warps][2][queries][D + 2]: of the share's first unit, and of a later one
};

// E consecutive dims of a row: weighted values, maximum (base 2) and sum.
template <int E>
struct RowPart {
  float m, l, o[E];
  __device__ __forceinline__ void none() {
    m = -CUDART_INF_F;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
  }
  __device__ __forceinline__ void join(const RowPart& x) {
    const float top = fmaxf(m, x.m);
    const float z = top == -CUDART_INF_F ? 0.f : top;
    const float f0 = ex2(m - z), f1 = ex2(x.m - z);
    m = top;
    l = fmaf(f0, l, f1 * x.l);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(f0, o[e], f1 * x.o[e]);
  }
  // what the prefix pass left for this row (nothing where `there` is false)
  template <int D>
  __device__ __forceinline__ void prefix(const SharedPrefix& s, int q_heads, int slot, int h, int d, bool there) {
    none();
    if (!there) return;
    const float* st = s.state + (static_cast<int64_t>(slot) * q_heads + h) * (D + 4);
    const float2 ml = *reinterpret_cast<const float2*>(st + D);
    m = ml.x;
    l = ml.y;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 y = *reinterpret_cast<const float2*>(st + d + e);
      o[e] = y.x;
      o[e + 1] = y.y;
    }
  }
  template <typename T, int D>
  __device__ __forceinline__ void store(const Attend& a, int slot, int h, int d) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t y[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) y[e] = Half16<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
    uint16_t* out = a.out + slot * a.out_row + static_cast<int64_t>(h) * D + d;
    if constexpr (E == 8) {
      *reinterpret_cast<uint4*>(out) = make_uint4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) *reinterpret_cast<uint32_t*>(out + 2 * e) = y[e];
    }
    if (d == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(slot) * a.q_heads + h] = (m + log2f(l)) * kLn2;
  }
};

// Waits for the cluster's CTAs; what they wrote to shared memory before is visible.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float2 load_cluster(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
  return v;
}

// Not the read-only path: the launch before this one may have written the
// cache, and this kernel may already have been scheduled by then.
__device__ __forceinline__ uint4 load16(const uint16_t* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

// A thread's running maximum (base 2), sum and weighted values: queries 2t, 2t + 1
// of each 8, dims 8g .. 8g + 7 of each 64.
template <int D, int NB>
struct StepSums {
  float m[NB][2], l[NB][2], acc[NB][D / 64][4][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b][0] = m[b][1] = -CUDART_INF_F;
      l[b][0] = l[b][1] = 0.f;
#pragma unroll
      for (int v = 0; v < D / 64; ++v)
#pragma unroll
        for (int w = 0; w < 4; ++w) acc[b][v][w][0] = acc[b][v][w][1] = acc[b][v][w][2] = acc[b][v][w][3] = 0.f;
    }
  }
};

// A warp's tiles t0 .. t1 - 1 of a unit.  `page` holds the pages of the first
// step's tiles.  Called once for `sums`.
template <typename T, int D, int NB>
__device__ __forceinline__ void attend_tiles(const PagedCache& c, const Attend& a, const SeenTiles& seen,
                                             const int32_t* row, const bool* mask, int64_t head_at, int t0, int t1,
                                             const uint4 (&q)[NB][D / 32], int (&page)[step_tiles(D, 16)],
                                             StepSums<D, NB>& sums) {
  constexpr int NT = step_tiles(D, 16);
  constexpr int KC = D / 32;  // 16-byte pieces of a key row per thread
  constexpr int VC = D / 64;  // of a value row
  const int lane = threadIdx.x & 31, t = lane & 3, g = lane >> 2;
  auto& [m, l, acc] = sums;
      for (int base = t0; base < t1; base += NT) {
        // keys in reach: one per lane
        const int my_tile = base + (lane >> 4);
        bool in = my_tile < t1 && (lane >> 4) < NT;
        {
          const int j = 16 * seen.tile(my_tile) + (lane & 15);
          in = in && j < seen.len && (j >= seen.low || j < a.sinks);
          if (in && mask != nullptr) in = mask[j];
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, in);
        uint4 kr[NT][2][KC], vr[NT][4][VC];
        uint32_t on[NT];
  #pragma unroll
        for (int u = 0; u < NT; ++u) {
          on[u] = c.is_page(page[u]) ? (bits >> (16 * u)) & 0xffffu : 0u;
          const int in_page = (16 * seen.tile(base + u)) & (c.page_size - 1);
          const uint16_t* kp = c.pool + c.block(page[u], a.layer, 0) + head_at + static_cast<int64_t>(in_page) * D;
  #pragma unroll
          for (int h = 0; h < 2; ++h)
  #pragma unroll
            for (int k = 0; k < KC; ++k)
              kr[u][h][k] = load16(kp + (g + 8 * h) * D + 8 * (t + 4 * k), (on[u] >> (g + 8 * h)) & 1u);
          const uint16_t* vp = kp + c.kv_elems;
  #pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 2 * t + (i & 1) + 8 * (i >> 1);
  #pragma unroll
            for (int v = 0; v < VC; ++v) vr[u][i][v] = load16(vp + key * D + 8 * (g + 8 * v), (on[u] >> key) & 1u);
          }
        }
        // the next step's pages, while this step's keys arrive
  #pragma unroll
        for (int u = 0; u < NT; ++u) {
          const int tt = base + NT + u;
          page[u] = tt < t1 ? row[(16 * seen.tile(tt)) >> c.page_shift] : -1;
        }
  #pragma unroll
        for (int b = 0; b < NB; ++b) {
          float s[NT][4];
          float top0 = m[b][0], top1 = m[b][1];
  #pragma unroll
          for (int u = 0; u < NT; ++u) {
            s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
  #pragma unroll
            for (int k = 0; k < KC; ++k) {
              Half16<T>::mma(s[u], kr[u][0][k].x, kr[u][1][k].x, kr[u][0][k].y, kr[u][1][k].y, q[b][k].x, q[b][k].y);
              Half16<T>::mma(s[u], kr[u][0][k].z, kr[u][1][k].z, kr[u][0][k].w, kr[u][1][k].w, q[b][k].z, q[b][k].w);
            }
            const bool lo = (on[u] >> g) & 1u, hi = (on[u] >> (g + 8)) & 1u;
            s[u][0] = lo ? s[u][0] * a.scale2 : -CUDART_INF_F;
            s[u][1] = lo ? s[u][1] * a.scale2 : -CUDART_INF_F;
            s[u][2] = hi ? s[u][2] * a.scale2 : -CUDART_INF_F;
            s[u][3] = hi ? s[u][3] * a.scale2 : -CUDART_INF_F;
            top0 = fmaxf(top0, fmaxf(s[u][0], s[u][2]));
            top1 = fmaxf(top1, fmaxf(s[u][1], s[u][3]));
          }
  #pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
          }
          const float z0 = top0 == -CUDART_INF_F ? 0.f : top0, z1 = top1 == -CUDART_INF_F ? 0.f : top1;
          const float y0 = z0 - kStepBias<T>, y1 = z1 - kStepBias<T>;
          const float keep0 = ex2(m[b][0] - z0), keep1 = ex2(m[b][1] - z1);
          m[b][0] = top0;
          m[b][1] = top1;
          l[b][0] *= keep0;
          l[b][1] *= keep1;
  #pragma unroll
          for (int v = 0; v < VC; ++v)
  #pragma unroll
            for (int w = 0; w < 4; ++w) {
              acc[b][v][w][0] *= keep0;
              acc[b][v][w][1] *= keep1;
              acc[b][v][w][2] *= keep0;
              acc[b][v][w][3] *= keep1;
            }
  #pragma unroll
          for (int u = 0; u < NT; ++u) {
            const float p0 = ex2(s[u][0] - y0), p1 = ex2(s[u][1] - y1), p2 = ex2(s[u][2] - y0), p3 = ex2(s[u][3] - y1);
            // the sum keeps the unrounded probabilities; the values' weights are two 16-bit numbers each, of whose sum
            // 16 bits (bf16) or 22 (f16) are right: the second products cost no bytes, and HBM is what bounds this
            l[b][0] += p0 + p2;
            l[b][1] += p1 + p3;
            const uint2 w0 = Half16<T>::split(p0, p1), w1 = Half16<T>::split(p2, p3);
            const uint32_t b0 = transpose8x8(w0.x), b1 = transpose8x8(w1.x);
            const uint32_t rest0 = transpose8x8(w0.y), rest1 = transpose8x8(w1.y);
  #pragma unroll
            for (int v = 0; v < VC; ++v) {
              const uint4 &x0 = vr[u][0][v], &x1 = vr[u][1][v], &x2 = vr[u][2][v], &x3 = vr[u][3][v];
              const uint32_t vt[4][4] = {
                  {__byte_perm(x0.x, x1.x, 0x5410), __byte_perm(x0.x, x1.x, 0x7632), __byte_perm(x2.x, x3.x, 0x5410),
                   __byte_perm(x2.x, x3.x, 0x7632)},
                  {__byte_perm(x0.y, x1.y, 0x5410), __byte_perm(x0.y, x1.y, 0x7632), __byte_perm(x2.y, x3.y, 0x5410),
                   __byte_perm(x2.y, x3.y, 0x7632)},
                  {__byte_perm(x0.z, x1.z, 0x5410), __byte_perm(x0.z, x1.z, 0x7632), __byte_perm(x2.z, x3.z, 0x5410),
                   __byte_perm(x2.z, x3.z, 0x7632)},
                  {__byte_perm(x0.w, x1.w, 0x5410), __byte_perm(x0.w, x1.w, 0x7632), __byte_perm(x2.w, x3.w, 0x5410),
                   __byte_perm(x2.w, x3.w, 0x7632)}};
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                Half16<T>::mma(acc[b][v][w], vt[w][0], vt[w][1], vt[w][2], vt[w][3], b0, b1);
                Half16<T>::mma(acc[b][v][w], vt[w][0], vt[w][1], vt[w][2], vt[w][3], rest0, rest1);
              }
            }
          }
        }
      }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b][0] -= kStepBias<T>;
    m[b][1] -= kStepBias<T>;
  }
}

// 4 or 8 bytes, as load16, without a condition: a register that a load may leave as it is costs an instruction to clear.
__device__ __forceinline__ uint32_t load4(const unsigned char* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const unsigned char* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// The first of the 8 dims that piece k of a thread's queries holds, as its keys do.
template <int Form>
__device__ __forceinline__ int step_dims(int t, int k) {
  return Form == 16 ? 32 * k + 8 * t : 64 * (k >> 1) + 16 * t + 8 * (k & 1);
}
// The query of a product's column.
template <int Form>
__device__ __forceinline__ int step_column(int g) {
  return Form >= 8 ? g : g & (Form == 1 ? 1 : Form - 1);  // (with one query the odd columns are empty)
}

// attend_tiles for a pool in 4 bits.  Nothing is rounded on the way into the
// products: a code is a small whole number, exact in either 16-bit type, and the
// pairs come in afterwards, in f32,
//   q.k = sum over groups: step (q.(16 + c)) + off sum q,   off = low - 16 step;
// the values' weights are p step, in two bf16 numbers each (their range is not
// f16's), and p off is summed by itself.  A weight is so right to 2^-16, and a value
// to 2^-16 of p 31 step.  Of bf16's largest groups 16 and 31 steps would leave f32:
// there off, and the values, are an eighth of themselves.
//
// What is busiest is the logic and shift unit: the codes' way into 16 bits takes two
// instructions for each pair of codes, 64 a tile of 16 keys and 64 dims, and so the
// rest has to be few; the other bound is registers, and with them warps.
//  * A product has 8 columns.  Few queries take them several times, each time for
//    another tile: with one or two queries (Form 1, 2) a thread's two columns are
//    those of tile t of four, with up to four of tile t / 2 of two.  Scores of the
//    other tiles are passed over, so that a thread has two scores a query in four
//    (two) tiles, and loads, weighs and masks two pairs instead of eight.  For the
//    values the weights go through one transposition for all of them and are
//    cleared outside the tile's own columns; the columns are added up at the end.
//    With one query the second column holds what the first one's rounding leaves.
//  * Addresses are 64-byte units in 32 bits, found by one lane a tile.
//  * All 16 keys of a tile are loaded; a key that is not in reach counts by its
//    weight of zero alone (its pair, which may be anything, is taken as zero).
//  * The maximum is looked after only when a key passes it.
//  * A step's keys are loaded under the softmax of the one before, its values under
//    the next scores (113 -> 109 and 147 -> 136 us of the head comment's cases).
// Tried and slower: shifts as high halves of products, for another pipe (118, 152
// us), another number of tiles a step or CTAs an SM.
template <typename T, int D, int NB, int Form>
__device__ __forceinline__ void attend_tiles4(const PagedCache& c, const Attend& a, const SeenTiles& seen,
                                              const int32_t* row, const bool* mask, int head, int t0, int t1,
                                              const uint4 (&q)[NB][D / 32], StepSums<D, NB>& sums) {
  using B = __nv_bfloat16;
  constexpr int NT = step_tiles(D, Form);
  constexpr int G = D / kGroup4;
  constexpr int QC = Form == 1 ? 1 : 2;                        // queries of a thread
  constexpr int TP = Form <= 2 ? 4 : Form == 4 ? 2 : 1;        // tiles that share the columns
  constexpr int NP = NT / TP, kTileShift = TP == 4 ? 0 : TP == 2 ? 1 : 2;
  const int lane = threadIdx.x & 31, t = lane & 3, g = lane >> 2;
  const int my = t >> kTileShift;         // the thread's tile of each TP
  const int col_tile = g >> (kTileShift + 1);  // the tile of column g
  auto &m = sums.m, &l = sums.l;
  auto& acc = sums.acc;
  constexpr float kPart = std::is_same_v<T, B> ? 0.125f : 1.f;  // of off, and of the values
  auto step_part = [](uint32_t bits) {  // step, and the part of off
    const float2 pair = unpack2<T>(bits);
    return make_float2(pair.x, fmaf(-16.f * kPart, pair.x, kPart * pair.y));
  };
  // the queries' sums over each group, times the scale
  float qs[NB][G][QC], rest[NB][G][QC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int v = 0; v < G; ++v) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4& x = q[b][2 * v + k];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2<T>(w[i]);
          sum += f.x + f.y;
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int i = 0; i < QC; ++i) {
        qs[b][v][i] = __shfl_sync(0xffffffffu, sum, 4 * (2 * t + i)) * (a.scale2 / kPart);
        rest[b][v][i] = 0.f;
      }
    }
  // the thread's bytes in page 0's block: codes of keys g (and g + 8), of values 2t (2t + 1, 2t + 8, 2t + 9), pairs of keys g
  const unsigned char* k_base = block4(c, 0, a.layer, 0, head);
  const unsigned char* p_base = k_base + block4_codes(c) + g * (4 * G);
  const unsigned char* vp_base = p_base + 2 * c.kv_elems;
  const unsigned char* v_base = k_base + 2 * c.kv_elems + 2 * t * (D / 2) + 4 * g;
  k_base += g * (D / 2) + 8 * t;
  const uint32_t page_units = static_cast<uint32_t>(c.layers * c.kv_elems / 16);  // of 64 bytes: a pool of 256 GB at most
  // Lane u (of each NT) looks up tile u of a step: its first key, its place in its page in tiles (-1: there is none), and
  // where its codes begin.
  const int mine = lane & (NT - 1);
  auto lookup = [&](int base) { return base + mine < t1 ? row[(16 * seen.tile(base + mine)) >> c.page_shift] : -1; };
  struct Place {
    int key, in;
    uint32_t at;
  };
  auto place = [&](int base, int page) {
    Place p;
    p.key = 16 * seen.tile(base + mine);
    p.in = c.is_page(page) ? (p.key & (c.page_size - 1)) >> 4 : -1;
    p.at = page * page_units + p.in * (D / 8);
    return p;
  };
  auto at64 = [](const unsigned char* from, uint32_t units) {  // from + 64 units
    uint64_t r;
    asm("mad.wide.u32 %0, %1, 64, %2;" : "=l"(r) : "r"(units), "l"(from));
    return reinterpret_cast<const unsigned char*>(r);
  };
  // (a tile that is not there leaves its registers as they are: codes are numbers whatever they are, pairs are looked at
  // only where a key is in reach)
  uint2 kr[NT][2][G] = {};
  uint32_t vr[NT][4][G] = {}, kp[NP][2][G] = {}, vp[NP][2][G] = {};
  auto load_pair = [](uint32_t (&to)[G], const unsigned char* at) {
    if constexpr (G == 1) {
      to[0] = load4(at);
    } else {
      const uint2 x = load8(at);
      to[0] = x.x;
      to[1] = x.y;
    }
  };
  auto load_keys = [&](const Place& p, bool (&on)[NP][2]) {  // on: whether the thread's keys g, g + 8 of its tiles are in reach
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const bool there = __shfl_sync(0xffffffffu, p.in, u) >= 0;
      const unsigned char* at = at64(k_base, __shfl_sync(0xffffffffu, p.at, u));
      if (there) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int v = 0; v < G; ++v) kr[u][h][v] = load8(at + 8 * h * (D / 2) + 32 * v);
      }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int u = n * TP + my;
      const int key = TP == 4 ? p.key : __shfl_sync(0xffffffffu, p.key, u), in = TP == 4 ? p.in : __shfl_sync(0xffffffffu, p.in, u);
      const uint32_t first = TP == 4 ? p.at : __shfl_sync(0xffffffffu, p.at, u);
      const unsigned char* at = at64(p_base, first - in * (D / 8 - G));  // pairs lie in 64-byte units, too
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = key + g + 8 * h;
        on[n][h] = in >= 0 && j < seen.len && (j >= seen.low || j < a.sinks);
        if (in >= 0) load_pair(kp[n][h], at + 32 * G * h);
      }
      if (mask != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (on[n][h]) on[n][h] = mask[key + g + 8 * h];
      }
    }
  };
  auto load_values = [&](const Place& p) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const bool there = __shfl_sync(0xffffffffu, p.in, u) >= 0;
      const unsigned char* at = at64(v_base, __shfl_sync(0xffffffffu, p.at, u));
      if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < G; ++v) vr[u][i][v] = load4(at + ((i & 1) + 8 * (i >> 1)) * (D / 2) + 32 * v);
      }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int u = n * TP + my;
      const int in = TP == 4 ? p.in : __shfl_sync(0xffffffffu, p.in, u);
      const uint32_t first = TP == 4 ? p.at : __shfl_sync(0xffffffffu, p.at, u);
      const unsigned char* at = at64(vp_base, first - in * (D / 8 - G));
      if (in >= 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) load_pair(vp[n][h], at + 32 * G * h);
      }
    }
  };
  bool on[NP][2];
  Place here = place(t0, lookup(t0));
  int next_page = lookup(t0 + NT);
  load_keys(here, on);
  load_values(here);
  for (int base = t0; base < t1; base += NT) {
    const Place next = place(base + NT, next_page);
    next_page = lookup(base + 2 * NT);
    float s[NB][NP][2][QC], top[NB][QC];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int i = 0; i < QC; ++i) top[b][i] = -CUDART_INF_F;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        float x[G][4];
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int v = 0; v < G; ++v) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint2 &r0 = kr[n * TP + u][0][v], &r1 = kr[n * TP + u][1][v];
              const uint32_t w0 = k == 0 ? r0.x : r0.y, w1 = k == 0 ? r1.x : r1.y;
              const uint4& z = q[b][2 * v + k];
              if (k == 0)
                Half16<T>::mma0(y, codes2<T, 0>(w0), codes2<T, 0>(w1), codes2<T, 1>(w0), codes2<T, 1>(w1), z.x, z.y);
              else
                Half16<T>::mma(y, codes2<T, 0>(w0), codes2<T, 0>(w1), codes2<T, 1>(w0), codes2<T, 1>(w1), z.x, z.y);
              Half16<T>::mma(y, codes2<T, 2>(w0), codes2<T, 2>(w1), codes2<T, 3>(w0), codes2<T, 3>(w1), z.z, z.w);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (QC == 2 || i % 2 == 0) x[v][i] = u == 0 || my == u ? y[i] : x[v][i];
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int v = 0; v < G; ++v) {
            const float2 so = step_part(kp[n][h][v]);
            const float step = so.x * a.scale2;
#pragma unroll
            for (int i = 0; i < QC; ++i)
              s[b][n][h][i] = fmaf(step, x[v][2 * h + i], v == 0 ? so.y * qs[b][0][i] : fmaf(so.y, qs[b][v][i], s[b][n][h][i]));
          }
#pragma unroll
          for (int i = 0; i < QC; ++i) {
            s[b][n][h][i] = on[n][h] ? s[b][n][h][i] : -CUDART_INF_F;
            top[b][i] = fmaxf(top[b][i], s[b][n][h][i]);
          }
        }
      }
    }
    bool next_on[NP][2];
    load_keys(next, next_on);  // under the softmax and the values' product
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      bool more = false;
#pragma unroll
      for (int i = 0; i < QC; ++i) more = more || top[b][i] > m[b][i];
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int i = 0; i < QC; ++i) {
          // over the keys and, where the columns are shared, over the tiles
#pragma unroll
          for (int o = TP == 4 ? 1 : TP == 2 ? 2 : 4; o < 32; o <<= 1) top[b][i] = fmaxf(top[b][i], __shfl_xor_sync(0xffffffffu, top[b][i], o));
          top[b][i] = fmaxf(top[b][i], m[b][i]);
          const float keep = top[b][i] == -CUDART_INF_F ? 1.f : ex2(m[b][i] - top[b][i]);
          m[b][i] = top[b][i];
          l[b][i] *= keep;
#pragma unroll
          for (int v = 0; v < G; ++v) {
            rest[b][v][i] *= keep;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              acc[b][v][w][i] *= keep;
              acc[b][v][w][2 + i] *= keep;
              if constexpr (QC == 1) {
                acc[b][v][w][1] *= keep;
                acc[b][v][w][3] *= keep;
              }
            }
          }
        }
      }
      float z[QC];
#pragma unroll
      for (int i = 0; i < QC; ++i) z[i] = m[b][i] == -CUDART_INF_F ? 0.f : m[b][i];
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        float w[2][QC];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < QC; ++i) {
            w[h][i] = ex2(s[b][n][h][i] - z[i]);
            l[b][i] += w[h][i];
          }
#pragma unroll
        for (int v = 0; v < G; ++v) {
          uint32_t first[2], second[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2 so = step_part(on[n][h] ? vp[n][h][v] : 0u);
            so.x *= kPart;
#pragma unroll
            for (int i = 0; i < QC; ++i) rest[b][v][i] = fmaf(w[h][i], so.y, rest[b][v][i]);
            const float x0 = w[h][0] * so.x;
            if constexpr (QC == 1) {
              first[h] = transpose8x8(Half16<B>::pack(x0, x0 - unpack2<B>(Half16<B>::pack(x0, 0.f)).x));
            } else {
              const uint2 x = Half16<B>::split(x0, w[h][1] * so.x);
              first[h] = transpose8x8(x.x);
              second[h] = transpose8x8(x.y);
            }
          }
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            const uint32_t(&r)[4][G] = vr[n * TP + u];
            const uint32_t near[2] = {__byte_perm(r[0][v], r[1][v], 0x5410), __byte_perm(r[0][v], r[1][v], 0x7632)};
            const uint32_t far[2] = {__byte_perm(r[2][v], r[3][v], 0x5410), __byte_perm(r[2][v], r[3][v], 0x7632)};
            const bool mine = TP == 1 || col_tile == u;
            const uint32_t b0 = mine ? first[0] : 0u, b1 = mine ? first[1] : 0u;
            auto dims = [&](auto which) {  // 8g + 2w (row g of the product) and 8g + 2w + 1 (row g + 8)
              constexpr int W = decltype(which)::value;
              const uint32_t v0 = codes2<B, W>(near[0]), v1 = codes2<B, W>(near[1]);
              const uint32_t v2 = codes2<B, W>(far[0]), v3 = codes2<B, W>(far[1]);
              Half16<B>::mma(acc[b][v][W], v0, v1, v2, v3, b0, b1);
              if constexpr (QC == 2) Half16<B>::mma(acc[b][v][W], v0, v1, v2, v3, mine ? second[0] : 0u, mine ? second[1] : 0u);
            };
            dims(std::integral_constant<int, 0>{});
            dims(std::integral_constant<int, 1>{});
            dims(std::integral_constant<int, 2>{});
            dims(std::integral_constant<int, 3>{});
          }
        }
      }
    }
    load_values(next);  // under the next step's scores
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) on[n][h] = next_on[n][h];
  }
  // shared columns are added up; the weights' part that belongs to no code is the same for all dims of a group
  auto over_tiles = [&](float x) {
    if constexpr (TP == 4) x += __shfl_xor_sync(0xffffffffu, x, 1);
    if constexpr (TP >= 2) x += __shfl_xor_sync(0xffffffffu, x, 2);
    return x;
  };
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      l[b][i] = over_tiles(l[b][i]);
#pragma unroll
      for (int v = 0; v < G; ++v) {
        float x = rest[b][v][i];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x = over_tiles(x);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float& o = acc[b][v][w][2 * k + i];
            o = (over_tiles(QC == 1 ? o + acc[b][v][w][2 * k + 1] : o) + x) * (1.f / kPart);
          }
      }
    }
}

template <typename T, int D, int NB, int Form>
__device__ __forceinline__ void attend_tiles_of(const PagedCache& c, const Attend& a, const SeenTiles& seen,
                                                const int32_t* row, const bool* mask, int head, int t0, int t1,
                                                const uint4 (&q)[NB][D / 32], int (&page)[step_tiles(D, Form)],
                                                StepSums<D, NB>& sums) {
  if constexpr (Form != 16)
    attend_tiles4<T, D, NB, Form>(c, a, seen, row, mask, head, t0, t1, q, sums);
  else
    attend_tiles<T, D, NB>(c, a, seen, row, mask, static_cast<int64_t>(head) * c.page_size * D, t0, t1, q, page, sums);
}

template <typename T, int D, int NB, int Form>
__global__ void __launch_bounds__(kStepThreads, step_ctas(D, NB))
    step_kernel(PagedCache c, Attend a, SharedPrefix shared, StepSpace ws, int blocks, int min_tiles) {
  constexpr int NT = step_tiles(D, Form), kUnitCost = unit_cost(Form);
  constexpr int NQ = 8 * NB;   // query rows of a unit
  constexpr int KC = D / 32, VC = D / 64;
  extern __shared__ int tiles_before[];  // [rows + 1]: tiles of a key head of the slots before
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = lane & 3, g = lane >> 2;
  take_turn();

  auto tiles_of = [&](int i) {
    return SeenTiles(c.length(i), a.window, a.sinks, shared.base != nullptr ? shared.base[i] : 0);
  };
  // tiles of every slot, scanned: a thread's slots lie side by side
  {
    __shared__ int warp_sum[kStepWarps];
    const int each = (a.rows + kStepThreads - 1) / kStepThreads;
    const int i0 = min(a.rows, tid * each), i1 = min(a.rows, i0 + each);
    int n = 0;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) {
      const int tiles = tiles_of(i).n;
      const int x = tiles > 0 ? tiles + kUnitCost : 0;
      tiles_before[i] = x;
      n += x;
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int before = inc - n, all = 0;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    for (int i = i0; i < i1; ++i) {
      const int x = tiles_before[i];
      tiles_before[i] = before;
      before += x;
    }
    if (tid == 0) tiles_before[a.rows] = all;
    __syncthreads();
  }
  const int units = c.kv_heads * blocks;
  const int64_t total = static_cast<int64_t>(tiles_before[a.rows]) * units;
  const int shares = gridDim.x * kStepWarps, me = blockIdx.x * kStepWarps + warp;
  const int64_t per = max((total + shares - 1) / shares, static_cast<int64_t>(min_tiles));

  // slots without a key in reach here
  for (int i = blockIdx.x; i < a.rows; i += gridDim.x) {
    if (tiles_before[i + 1] != tiles_before[i]) continue;
    const bool there = shared.base != nullptr && shared.base[i] > 0;
    for (int e = tid; e < a.q_heads * (D / 8); e += kStepThreads) {
      RowPart<8> r;
      r.prefix<D>(shared, a.q_heads, i, e / (D / 8), 8 * (e % (D / 8)), there);
      r.store<T, D>(a, i, e / (D / 8), 8 * (e % (D / 8)));
    }
  }

  int64_t x = me * per;
  const int64_t x_end = min(total, x + per);
  if (lane == 0) ws.cut[me] = make_int4(0, 0, 0, 0);
  if (x >= x_end) return;
  const int64_t x_first = x;
  int slot, head, block, t0, t1;
  int64_t unit_x;  // where the unit begins on the line; its tile i lies at unit_x + kUnitCost + i
  {
    int lo = 0, hi = a.rows;  // the last slot whose tiles begin at or before x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(tiles_before[mid]) * units <= x) lo = mid; else hi = mid;
    }
    slot = lo;
    const int64_t slot_x = static_cast<int64_t>(tiles_before[slot]) * units;
    const int n = tiles_before[slot + 1] - tiles_before[slot];
    const int unit = static_cast<int>((x - slot_x) / n);
    head = unit / blocks;
    block = unit - head * blocks;
    unit_x = slot_x + static_cast<int64_t>(unit) * n;
  }
  SeenTiles seen = tiles_of(slot);
  int base_tokens = shared.base != nullptr ? shared.base[slot] : 0;
  uint4 q[NB][KC];
  int page[NT];  // (16 bits; attend_tiles4 looks its tiles' up by itself)
  // the unit's share, its queries and its first pages
  auto enter = [&] {
    t0 = static_cast<int>(max(x - unit_x - kUnitCost, static_cast<int64_t>(0)));
    t1 = static_cast<int>(max(min(static_cast<int64_t>(seen.n), x_end - unit_x - kUnitCost), static_cast<int64_t>(0)));
    const int queries = min(NQ, a.group - block * NQ);
    const int col = step_column<Form>(g);
    const int64_t q_at = slot * a.q_row + static_cast<int64_t>(head * a.group + block * NQ + col) * D;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int k = 0; k < KC; ++k) q[b][k] = load16(a.q + q_at + 8 * b * D + step_dims<Form>(t, k), 8 * b + col < queries);
    if constexpr (Form == 16) {
      const int32_t* row = c.table + static_cast<int64_t>(slot) * c.table_pages;
#pragma unroll
      for (int u = 0; u < NT; ++u) page[u] = t0 + u < t1 ? row[(16 * seen.tile(t0 + u)) >> c.page_shift] : -1;
    }
  };
  enter();
  while (true) {
    const int queries = min(NQ, a.group - block * NQ);
    const int q_head = head * a.group + block * NQ;
    const int32_t* row = c.table + static_cast<int64_t>(slot) * c.table_pages;
    const bool* mask = a.key_mask != nullptr ? a.key_mask + slot * a.mask_stride : nullptr;
    StepSums<D, NB> sums;
    sums.clear();
    attend_tiles_of<T, D, NB, Form>(c, a, seen, row, mask, head, t0, t1, q, page, sums);
    auto& [m, l, acc] = sums;

    // a thread holds queries 2t, 2t + 1 and dims 8g .. 8g + 7 of each 64
    const bool whole = t0 == 0 && t1 == seen.n, some = t0 < t1;
    const bool there = base_tokens > 0 && whole;
    RowPart<8> before[2][VC];  // of the first 8 queries: on their way while the next unit is entered
    if (NB == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < VC; ++v)
          before[i][v].template prefix<D>(shared, a.q_heads, slot, q_head + 2 * t + i, 64 * v + 8 * g,
                                          there && 2 * t + i < queries);
    }
    // of a cut unit: the share's part 0 when the unit is its first, else part 1
    const int my_part = x_first >= unit_x ? 0 : 1;
    float* part = ws.part + (2 * static_cast<int64_t>(me) + my_part) * NQ * (D + 2);
    if (t0 == 0 && some && !whole && lane == 0)
      ws.cut[me] = make_int4(slot, head * blocks + block,
                             static_cast<int>((unit_x + kUnitCost + seen.n - 1) / per) - me + 1, my_part);
    const int my_slot = slot;
    x = unit_x + kUnitCost + seen.n;
    const bool more = x < x_end;
    if (more) {
      unit_x = x;
      if (++block == blocks) {
        block = 0;
        if (++head == c.kv_heads) {
          head = 0;
          do ++slot; while (tiles_before[slot + 1] == tiles_before[slot]);
          seen = tiles_of(slot);
          base_tokens = shared.base != nullptr ? shared.base[slot] : 0;
        }
      }
      enter();
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[b][0] += __shfl_xor_sync(0xffffffffu, l[b][0], o);
        l[b][1] += __shfl_xor_sync(0xffffffffu, l[b][1], o);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int qi = 8 * b + 2 * t + i;
        if (qi < queries && some) {
#pragma unroll
          for (int v = 0; v < VC; ++v) {
            const int d = 64 * v + 8 * g;
            RowPart<8> r;
            r.m = m[b][i];
            r.l = l[b][i];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              r.o[2 * w] = acc[b][v][w][i];
              r.o[2 * w + 1] = acc[b][v][w][2 + i];
            }
            if (whole) {
              if (there) {
                if (NB > 1) before[i][v].template prefix<D>(shared, a.q_heads, my_slot, q_head + qi, d, true);
                r.join(before[i][v]);
              }
              r.template store<T, D>(a, my_slot, q_head + qi, d);
            } else {
#pragma unroll
              for (int w = 0; w < 4; ++w)
                *reinterpret_cast<float2*>(part + qi * (D + 2) + d + 2 * w) = make_float2(r.o[2 * w], r.o[2 * w + 1]);
              if (d == 0) *reinterpret_cast<float2*>(part + qi * (D + 2) + D) = make_float2(r.m, r.l);
            }
          }
        }
      }
    }
    if (!more) break;
  }
}

// Joins the parts of the units that a cut divided.  `threads` threads (32, 64
// or 128) look after the unit that begins in one warp's share, a pair of dims of
// one query each; CTA y after the y-th 128 of them.
constexpr int kJoinChunk = 16;  // parts on their way at a time

template <typename T, int D>
__global__ void __launch_bounds__(kStepThreads)
    step_join_kernel(Attend a, SharedPrefix shared, StepSpace ws, int nq, int blocks, int threads) {
  take_turn();
  const int me = (blockIdx.x * kStepThreads + threadIdx.x) / threads;
  const int e = blockIdx.y * kStepThreads + threadIdx.x % threads;
  const int qi = e / (D / 2), d = 2 * (e % (D / 2));
  const int64_t stride = static_cast<int64_t>(nq) * (D + 2);
  const int4 cut = ws.cut[me];
  const int head = cut.y / blocks, block = cut.y % blocks;
  if (cut.z > 0 && qi < min(nq, a.group - block * nq)) {
    // the first part lies where the warp left it, the others are their warps' first units
    const float* parts = ws.part + 2 * static_cast<int64_t>(me) * stride + qi * (D + 2);
    RowPart<2> r, before;
    const int h = head * a.group + block * nq + qi;
    before.prefix<D>(shared, a.q_heads, cut.x, h, d, shared.base != nullptr && shared.base[cut.x] > 0);
    r.none();
    for (int k0 = 0; k0 < cut.z; k0 += kJoinChunk) {
      float2 ml[kJoinChunk], y[kJoinChunk];
#pragma unroll
      for (int k = 0; k < kJoinChunk; ++k) {
        const float* p = parts + (k0 + k == 0 ? cut.w : 2 * (k0 + k)) * stride;
        const bool on = k0 + k < cut.z;
        ml[k] = on ? __ldcg(reinterpret_cast<const float2*>(p + D)) : make_float2(-CUDART_INF_F, 0.f);
        y[k] = on ? __ldcg(reinterpret_cast<const float2*>(p + d)) : make_float2(0.f, 0.f);
      }
      float top = r.m;
#pragma unroll
      for (int k = 0; k < kJoinChunk; ++k) top = fmaxf(top, ml[k].x);
      const float z = top == -CUDART_INF_F ? 0.f : top;
      const float keep = ex2(r.m - z);
      r.m = top;
      r.l *= keep;
      r.o[0] *= keep;
      r.o[1] *= keep;
#pragma unroll
      for (int k = 0; k < kJoinChunk; ++k) {
        const float f = ex2(ml[k].x - z);
        r.l = fmaf(f, ml[k].y, r.l);
        r.o[0] = fmaf(f, y[k].x, r.o[0]);
        r.o[1] = fmaf(f, y[k].y, r.o[1]);
      }
    }
    r.join(before);
    r.store<T, D>(a, cut.x, h, d);
  }
}

// Few slots: a cluster of 1 to 8 CTAs for each unit, its tiles dealt to the
// cluster's warps, which join their parts through shared memory: one launch and
// no workspace.  The largest cluster is taken with which all units run at once
// (8 CTAs of 8 warps only where a slot can have more than one step for each of 32
// warps), if a slot cannot be longer than few_steps steps of each of its warps.
// There this saves the scan, the second launch and the parts' way through L2;
// past either limit the line of tiles is faster, as it fills the device and
// balances it.  How long a slot can be is the table's width, which the host knows,
// not its length, which it does not: a short slot in a wide table takes the line.
// GPU time of a call in us, line / clusters, bf16, all slots of the
// same length (in brackets what is not taken, as it was with one product of the
// values):
//   heads  dim  slots    128 keys      467         1000         2000         8000
//   12/12   64    2     8.5 /  5.6   9.2 /  5.8  11.9 /  7.4  14.3 /  7.5  20.8 / 16.0
//   12/12   64    9    10.5 /  6.3  13.4 /  8.2  15.6 / 12.0  20.2 / 18.2
//   12/12   64   24    12.0 /  6.7  13.6 / 12.2  21.8 / 19.0 (32.6 / 29.4)
//   32/8   128    4    12.6 /  6.2  14.0 /  8.2  16.6 / 10.1  20.8 / 13.5 (36.0 / 34.8)
//   32/8   128   16    14.5 /  7.4  17.8 / 12.0  23.7 / 18.3 (34.8 / 30.8)
//   32/8   128   48    18.3 / 12.5 (29.1 / 27.4) (45.9 / 48.6)
//   16/1   128    6    21.2 /  7.9  21.8 /  8.1  22.8 /  9.9  27.1 / 14.8
// Over 4 bits twice as many steps are taken (in brackets what is not):
//   heads  dim  slots    128 keys      467         1000         2000         4000         8000
//   12/12   64    2     8.0 /  4.7  10.2 /  4.8  11.8 /  5.0  12.4 /  5.7  13.9 /  7.2  15.3 /  9.7
//   12/12   64   24    10.8 /  5.2  13.6 /  7.1  15.8 /  9.8  19.7 / 14.7  31.8 / 26.6 (54.3 / 48.7)
//   32/8   128    4    11.8 /  6.8  12.2 /  7.6  13.3 /  8.5  15.0 / 11.4  19.2 / 17.0  25.0 / 27.3
//   32/8   128   16    12.3 /  7.3  14.5 /  9.5  18.4 / 13.0  23.3 / 19.6  35.4 / 34.9 (58.4 / 66.0)
//   16/1   128    6    19.4 /  5.9  20.1 /  6.0  20.7 /  7.5  21.9 /  8.8  23.9 / 11.3  29.3 / 16.4
constexpr int kMaxSpread = 8;
constexpr int few_steps(int form) { return form == 16 ? 4 : 8; }

// 4 CTAs of 4 warps an SM, as head_dim 64 has by itself: 132 registers instead of
// 128 would let one cluster in four go.
template <typename T, int D, int NB, int W, int Form>
__global__ void __launch_bounds__(32 * W, D == 128 && NB == 1 && W == 4 ? 4 : 0) step_few_kernel(PagedCache c, Attend a, int blocks, int spread) {
  constexpr int NT = step_tiles(D, Form);
  constexpr int NQ = 8 * NB, KC = D / 32, VC = D / 64;
  constexpr int kRow = D + 2;  // weighted values, maximum, sum
  extern __shared__ float few_smem[];
  auto parts = reinterpret_cast<float (*)[NQ][kRow]>(few_smem);  // [W]
  auto& joined = parts[W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = lane & 3, g = lane >> 2;
  const int rank = blockIdx.x % spread, unit = blockIdx.x / spread;
  const int block = unit % blocks, head = unit / blocks % c.kv_heads, slot = unit / blocks / c.kv_heads;
  const int queries = min(NQ, a.group - block * NQ), q_head = head * a.group + block * NQ;
  take_turn();

  const SeenTiles seen(c.length(slot), a.window, a.sinks, 0);
  // steps of NT tiles, dealt evenly
  const int warps = spread * W;
  const int steps = (seen.n + NT - 1) / NT, me = rank * W + warp;
  const int t0 = NT * static_cast<int>(static_cast<int64_t>(steps) * me / warps);
  const int t1 = min(seen.n, NT * static_cast<int>(static_cast<int64_t>(steps) * (me + 1) / warps));
  const int32_t* row = c.table + static_cast<int64_t>(slot) * c.table_pages;
  uint4 q[NB][KC];
  int page[NT];
  if constexpr (Form == 16) {
#pragma unroll
    for (int u = 0; u < NT; ++u) page[u] = t0 + u < t1 ? row[(16 * seen.tile(t0 + u)) >> c.page_shift] : -1;
  }
  const int col = step_column<Form>(g);
  const int64_t q_at = slot * a.q_row + static_cast<int64_t>(q_head + col) * D;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int k = 0; k < KC; ++k) q[b][k] = load16(a.q + q_at + 8 * b * D + step_dims<Form>(t, k), 8 * b + col < queries);
  StepSums<D, NB> sums;
  sums.clear();
  attend_tiles_of<T, D, NB, Form>(c, a, seen, row, a.key_mask != nullptr ? a.key_mask + slot * a.mask_stride : nullptr, head,
                                  t0, t1, q, page, sums);
  auto& [m, l, acc] = sums;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[b][i] += __shfl_xor_sync(0xffffffffu, l[b][i], o);
      float* part = parts[warp][8 * b + 2 * t + i];
#pragma unroll
      for (int v = 0; v < VC; ++v)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float2*>(part + 64 * v + 8 * g + 2 * w) = make_float2(acc[b][v][w][i], acc[b][v][w][2 + i]);
      if (g == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m[b][i], l[b][i]);
    }
  __syncthreads();
  const int pairs = queries * (D / 2);  // of dims
  auto join = [&](int n, auto at) {  // of n parts, in order
    RowPart<2> r;
    r.none();
    float2 ml[kMaxSpread], y[kMaxSpread];
#pragma unroll
    for (int k = 0; k < kMaxSpread; ++k)
      if (k < n) at(k, &ml[k], &y[k]);
#pragma unroll
    for (int k = 0; k < kMaxSpread; ++k)
      if (k < n) {
        RowPart<2> x;
        x.m = ml[k].x;
        x.l = ml[k].y;
        x.o[0] = y[k].x;
        x.o[1] = y[k].y;
        r.join(x);
      }
    return r;
  };
  for (int e = tid; e < pairs; e += 32 * W) {
    const int qi = e / (D / 2), d = 2 * (e % (D / 2));
    const RowPart<2> r = join(W, [&](int k, float2* ml, float2* y) {
      *ml = *reinterpret_cast<const float2*>(&parts[k][qi][D]);
      *y = *reinterpret_cast<const float2*>(&parts[k][qi][d]);
    });
    *reinterpret_cast<float2*>(&joined[qi][d]) = make_float2(r.o[0], r.o[1]);
    if (d == 0) *reinterpret_cast<float2*>(&joined[qi][D]) = make_float2(r.m, r.l);
  }
  cluster_sync();
  const int each = pairs / spread;  // D / 2 is a multiple of it
  for (int e = rank * each + tid; e < (rank + 1) * each; e += 32 * W) {
    const int qi = e / (D / 2), d = 2 * (e % (D / 2));
    const RowPart<2> r = join(spread, [&](int k, float2* ml, float2* y) {
      *ml = load_cluster(cluster_addr(&joined[qi][D], k));
      *y = load_cluster(cluster_addr(&joined[qi][d], k));
    });
    r.store<T, D>(a, slot, q_head + qi, d);
  }
  cluster_sync();  // the others may still be reading this CTA's shared memory
}

constexpr size_t few_bytes(int head_dim, int nb, int warps) {
  return static_cast<size_t>(warps + 1) * 8 * nb * (head_dim + 2) * 4;
}

// Launch of step_few_kernel with clusters of `spread` CTAs.
struct FewLaunch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg{};
  FewLaunch(int units, int spread, int warps, size_t smem, cudaStream_t stream) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = spread;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(units * spread);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
};

// Clusters of `Spread` CTAs of the kernel that the current device runs at once
// (0: cannot be queried).  Nothing here allocates or throws.
template <typename T, int D, int NB, int W, int Spread, int Form>
int few_clusters() {
  static std::atomic<int> known[64];  // by device ordinal, plus 1; the opt-in below is per device
  int dev = -1, clusters = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    if (dev >= 0 && dev < 64 && (clusters = known[dev].load(std::memory_order_relaxed)) > 0) return clusters - 1;
    const auto kernel = step_few_kernel<T, D, NB, W, Form>;
    FewLaunch launch(1, Spread, W, few_bytes(D, NB, W), nullptr);
    launch.cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(few_bytes(D, NB, W))) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &launch.cfg) == cudaSuccess) {
      if (dev >= 0 && dev < 64) known[dev].store(clusters + 1, std::memory_order_relaxed);
      return clusters;
    }
  }
  cudaGetLastError();
  return 0;
}

// 8-query blocks of a unit, and units per key head
void step_blocks(int group, int* nb, int* blocks) {
  *nb = group <= 8 ? 1 : 2;
  *blocks = (group + 8 * *nb - 1) / (8 * *nb);
}

}  // namespace

// cut records, then parts; sized for the largest device this library runs on
// (kMaxSms SMs), so that the size does not depend on the current one
constexpr int kMaxSms = 160;
size_t cut_bytes(int head_dim, int nb) {
  return static_cast<size_t>(kMaxSms) * step_ctas(head_dim, nb) * kStepWarps * sizeof(int4);
}

size_t step_workspace(const mtt_b200_paged_cache_t& c, int q_heads) {
  int nb, blocks;
  step_blocks(q_heads / c.kv_heads, &nb, &blocks);
  const size_t shares = static_cast<size_t>(kMaxSms) * step_ctas(c.head_dim, nb) * kStepWarps;
  return cut_bytes(c.head_dim, nb) + (shares * 2 * 8 * nb * (c.head_dim + 2) * 4 + 255) / 256 * 256;
}

cudaError_t launch_step(const PagedCache& c, int dtype, const Attend& a, const SharedPrefix& shared, void* space,
                        cudaStream_t stream) {
  int nb, blocks;
  step_blocks(a.group, &nb, &blocks);
  const int form = step_form(c.bits, c.head_dim, a.group);
  StepSpace ws;
  ws.cut = static_cast<int4*>(space);
  ws.part = reinterpret_cast<float*>(static_cast<char*>(space) + cut_bytes(c.head_dim, nb));
  const int sms = cache_sm_count();
  if (sms <= 0 || sms > kMaxSms) return cudaErrorInvalidValue;
  const size_t smem = 4 * (static_cast<size_t>(a.rows) + 1);
  const int grid = sms * step_ctas(c.head_dim, nb), shares = grid * kStepWarps;
  const int min_tiles = unit_cost(form) + step_tiles(c.head_dim, form);
  const int pairs = std::min(8 * nb, a.group) * c.head_dim / 2;
  auto go = [&](auto kernel, auto join) {
    if (smem > 40 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 4 * (kCacheMaxSlots + 1));
      if (e != cudaSuccess) return e;
    }
    cudaError_t e = launch_serialized(kernel, dim3(grid), dim3(kStepThreads), smem, stream, c, a, shared, ws, blocks,
                                      min_tiles);
    if (e != cudaSuccess) return e;
    const int threads = pairs <= 32 ? 32 : pairs <= 64 ? 64 : kStepThreads;
    return launch_serialized(join, dim3(shares / (kStepThreads / threads), (pairs + kStepThreads - 1) / kStepThreads),
                             dim3(kStepThreads), 0, stream, a, shared, ws, 8 * nb, blocks, threads);
  };
  const int64_t units = static_cast<int64_t>(a.rows) * c.kv_heads * blocks;
  // the most keys that a row can see (a run of tiles has up to 15 keys more at each end)
  int64_t reach = static_cast<int64_t>(c.table_pages) * c.page_size;
  if (a.window > 0) reach = std::min(reach, static_cast<int64_t>(a.window) + a.sinks + 32);
  auto few = [&](auto kernel, int warps, int spread) {
    const FewLaunch launch(static_cast<int>(units), spread, warps, few_bytes(c.head_dim, nb, warps), stream);
    return cudaLaunchKernelEx(&launch.cfg, kernel, c, a, blocks, spread);
  };
  auto with_form = [&](auto type, auto dim, auto bs, auto f) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, NB = decltype(bs)::value, Form = decltype(f)::value;
    auto fits = [&](int warps, int clusters) {
      return units <= clusters && reach <= static_cast<int64_t>(few_steps(Form)) * warps * 16 * step_tiles(D, Form);
    };
    if (shared.base == nullptr) {
      if (reach > 32 * 16 * step_tiles(D, Form) && fits(64, few_clusters<T, D, NB, 8, 8, Form>()))
        return few(step_few_kernel<T, D, NB, 8, Form>, 8, 8);
      if (fits(32, few_clusters<T, D, NB, 4, 8, Form>())) return few(step_few_kernel<T, D, NB, 4, Form>, 4, 8);
      if (fits(16, few_clusters<T, D, NB, 4, 4, Form>())) return few(step_few_kernel<T, D, NB, 4, Form>, 4, 4);
      if (fits(8, few_clusters<T, D, NB, 4, 2, Form>())) return few(step_few_kernel<T, D, NB, 4, Form>, 4, 2);
      if (fits(4, few_clusters<T, D, NB, 4, 1, Form>())) return few(step_few_kernel<T, D, NB, 4, Form>, 4, 1);
    }
    return go(step_kernel<T, D, NB, Form>, step_join_kernel<T, D>);
  };
  auto run = [&](auto type, auto dim, auto bs) {
    using std::integral_constant;
    if (form == 16) return with_form(type, dim, bs, integral_constant<int, 16>{});
    if constexpr (decltype(bs)::value == 1) {
      if (form == 1) return with_form(type, dim, bs, integral_constant<int, 1>{});
      if constexpr (decltype(dim)::value == 64) {
        if (form == 2) return with_form(type, dim, bs, integral_constant<int, 2>{});
      }
      if (form == 4) return with_form(type, dim, bs, integral_constant<int, 4>{});
    }
    return with_form(type, dim, bs, integral_constant<int, decltype(bs)::value == 1 ? 8 : 9>{});
  };
  auto pick = [&](auto type) {
    using std::integral_constant;
    if (c.head_dim == 64)
      return nb == 1 ? run(type, integral_constant<int, 64>{}, integral_constant<int, 1>{})
                     : run(type, integral_constant<int, 64>{}, integral_constant<int, 2>{});
    return nb == 1 ? run(type, integral_constant<int, 128>{}, integral_constant<int, 1>{})
                   : run(type, integral_constant<int, 128>{}, integral_constant<int, 2>{});
  };
  return dtype == MTT_B200_DTYPE_BF16 ? pick(__nv_bfloat16{}) : pick(__half{});
}

}  // namespace mtt

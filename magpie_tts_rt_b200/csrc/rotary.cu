// Norm and position rotation of query and key heads, alone (rotate) or on the
// way into the paged cache (append).
//
//   y = x w / sqrt(mean x^2 + eps);  (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)
//
// Every element is read and written once: HBM bounds many rows, latency few, and a
// prompt's append (offsets, length, table and reference count follow one another
// before a row's first use, one pass of loads on its way).  A head is held by
// head_dim / 16 lanes as two 16-byte pieces each, chosen so that both dims of
// every pair lie in the same lane and a lane has the same 8 pairs in every head.  A
// warp takes a row's heads, a few at a time, and finds the row's cosines and sines
// once (each lane a pair or two, exchanged through shared memory); a lane keeps
// their products with the weights, so that norm and rotation are two products an
// element, in pairs of f32, and a factor for the head.  The mean takes two or three
// shuffles.  What hides the loads is warps: 32 an SM, for which a lane's coefficients
// lie in shared memory (in registers, 16 warps with four passes' loads in flight
// each: 45 us instead of 32 for 8192 rows of 32 and 8 heads of 128, which is 5.3
// TB/s; the append of 7105 such rows, prompts of 24 slots, 39 us (4.5 TB/s), into 4 bits
// 48 (3.2 TB/s), where 111 registers leave 16 warps).
//
// The angle is position x turns in 64 bits, of which only the part past whole
// turns is kept: exact to 2^-22 of a turn at positions up to 2^31, where a 32-bit
// product would be off by whole turns.
#include <cmath>

#include "cache4.cuh"

namespace mtt {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRotWarps = kRotThreads / 32;
// Passes whose loads are on their way while another is turned.  (With the loops over it written out for one the compiler
// spills 24 bytes instead of 0 to 16: 8192 rows 34 us instead of 32.)
constexpr int kRotAhead = 1;

enum class Into { kRows, kCache16, kCache4 };

struct RotArgs {
  int rotary_dim, interleaved, rows, q_heads, kv_heads, layer, chunks;
  float eps;
  const double* turns;
  const float *q_weight, *k_weight;
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_out;
  int64_t q_row, k_row, v_row, q_out_row, k_out_row;
  const int32_t *positions, *offsets;
};

// A lane's share of a head is 16 values, 8 pairs y that lie beside each other, and
// what turns them: z = y own + other (another pair).  Interleaved, y is a pair of the
// rotation and the other one itself, swapped,
//   own = (w0 c, w1 c),  other = (-w1 s, w0 s);
// else the lane's first piece (pairs 0 to 3) is turned against the second,
//   own = w c,  other = -+ its w s.
// They lie in shared memory, for queries and for keys: in registers they would halve
// the number of warps.  [own 0-1 .. own 6-7, other 0-1 .. other 6-7][lane of a head]
template <int L>
using Coefficients = float4[8][L];

template <bool Interleaved, int L>
__device__ __forceinline__ void make_coefficients(Coefficients<L>& to, int t, const float2* turn, const float* weight, int pa, int pb) {
  float2 own[8], other[8];
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 x = weight == nullptr ? make_float4(1.f, 1.f, 1.f, 1.f)
                                       : *reinterpret_cast<const float4*>(weight + 8 * (i < 8 ? pa : pb) + i % 8);
    w[i] = x.x;
    w[i + 1] = x.y;
    w[i + 2] = x.z;
    w[i + 3] = x.w;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = turn[i];  // cosine, sine of the lane's pair i
    if constexpr (Interleaved) {
      own[i] = make_float2(w[2 * i] * v.x, w[2 * i + 1] * v.x);
      other[i] = make_float2(-w[2 * i + 1] * v.y, w[2 * i] * v.y);
    } else {
      float2 &a = own[i / 2], &b = own[4 + i / 2], &c = other[i / 2], &d = other[4 + i / 2];
      (i % 2 ? a.y : a.x) = w[i] * v.x;
      (i % 2 ? b.y : b.x) = w[8 + i] * v.x;
      (i % 2 ? c.y : c.x) = -w[8 + i] * v.y;
      (i % 2 ? d.y : d.x) = w[i] * v.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    to[i][t] = make_float4(own[2 * i].x, own[2 * i].y, own[2 * i + 1].x, own[2 * i + 1].y);
    to[4 + i][t] = make_float4(other[2 * i].x, other[2 * i].y, other[2 * i + 1].x, other[2 * i + 1].y);
  }
}

template <typename T, int D, Into To, bool Interleaved>
__global__ void __launch_bounds__(kRotThreads, To == Into::kCache4 ? 4 : 8) rotate_kernel(PagedCache c, RotArgs in) {
  constexpr int L = D / 16, H = 32 / L;  // lanes of a head, heads of a pass
  __shared__ float2 turn[kRotWarps][D / 2];
  __shared__ Coefficients<L> coefficients[kRotWarps][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane % L, j = lane / L;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp;
  const int row = static_cast<int>(unit / in.chunks), chunk = static_cast<int>(unit % in.chunks);
  take_turn();
  if (row >= in.rows) return;
  // passes of H heads: queries', keys', then (append) values'
  const int qp = (in.q_heads + H - 1) / H, kp = (in.kv_heads + H - 1) / H;
  const int passes = qp + kp + (To == Into::kRows ? 0 : kp);
  const int p0 = static_cast<int>(static_cast<int64_t>(passes) * chunk / in.chunks);
  const int p1 = static_cast<int>(static_cast<int64_t>(passes) * (chunk + 1) / in.chunks);
  // the lane's pieces of a query or key head
  const bool turned = t < in.rotary_dim / 16, all_turned = in.rotary_dim == D;
  const int pa = turned && !Interleaved ? t : 2 * t;
  const int pb = turned && !Interleaved ? t + in.rotary_dim / 16 : 2 * t + 1;
  const uint16_t* q_src = in.q + row * in.q_row + j * D + 8 * pa;
  const uint16_t* k_src = in.k + row * in.k_row + j * D + 8 * pa;
  const uint16_t* v_src = in.v + row * in.v_row + j * D + 8 * t;
  const int second = 8 * (pb - pa);  // from the first piece to the other

  uint4 x[kRotAhead][2];
  auto load = [&](int n, int p) {
    if (p >= p1) return;
    const bool is_v = To != Into::kRows && p >= qp + kp, is_q = p < qp;
    const int h = (is_q ? p : is_v ? p - qp - kp : p - qp) * H;
    if (h + j >= (is_q ? in.q_heads : in.kv_heads)) return;
    const uint16_t* src = (is_q ? q_src : is_v ? v_src : k_src) + h * D;
    x[n][0] = *reinterpret_cast<const uint4*>(src);
    x[n][1] = *reinterpret_cast<const uint4*>(src + (is_v ? 8 * L : second));
  };
#pragma unroll
  for (int n = 0; n < kRotAhead; ++n) {
    x[n][0] = x[n][1] = make_uint4(0, 0, 0, 0);
    load(n, p0 + n);
  }

  // where the row goes
  int page = -1, in_page = 0, position = 0;
  bool known = true;  // append: the row is a token of a slot
  if constexpr (To == Into::kRows) {
    position = in.positions[row];
  } else {
    const RowPlace at(c, in.offsets, in.rows, row);
    const bool refused = at.slot < c.slots && c.refused != nullptr && c.refused[at.slot] != 0;
    known = at.pos >= 0 && !refused;
    int bad = at.unfit == 2 || (at.unfit == 1 && !refused) ? 1 : 0;
    if (known) {
      page = c.table[static_cast<int64_t>(at.slot) * c.table_pages + (at.pos >> c.page_shift)];
      if (!c.is_page(page) || c.refs[page] > 1) {
        page = -1;
        bad = 3;
      }
      in_page = at.pos & (c.page_size - 1);
      position = in.positions != nullptr ? in.positions[row] : at.pos;
    }
    if (bad != 0 && chunk == 0 && lane == 0 && c.status != nullptr) c.status[at.slot] = bad;
  }
#pragma unroll
  for (int k = 0; k < D / 64; ++k) {
    const int i = lane + 32 * k;  // pairs past rotary_dim: no turn
    const double turns = i < in.rotary_dim / 2 ? position * in.turns[i] : 0.;
    float sn, cs;
    // within half a turn the fast functions are right to 2^-21, where the result is rounded to 2^-12 at best
    __sincosf(6.283185307f * static_cast<float>(turns - rint(turns)), &sn, &cs);
    turn[warp][i] = make_float2(cs, sn);
  }
  __syncwarp();

  // the lanes of the pass's first head for the queries, of its second for the keys
  if (j < 2) make_coefficients<Interleaved, L>(coefficients[warp][j], t, &turn[warp][8 * t], j == 0 ? in.q_weight : in.k_weight, pa, pb);
  __syncwarp();
  // head h: what becomes of it, in 16 bits
  auto turn_head = [&](bool is_q, uint4& a, uint4& b) {
    const float* weight = is_q ? in.q_weight : in.k_weight;
    const Coefficients<L>& with = coefficients[warp][is_q ? 0 : 1];
    float2 y[8];
    {
      const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = unpack2<T>(u[i]);
    }
    float inv = 1.f;  // of the norm
    if (weight != nullptr) {
      float2 sums = mul2(y[0], y[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) sums = fma2(y[i], y[i], sums);
      float sum = sums.x + sums.y;
#pragma unroll
      for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      inv = rsqrtf(sum * (1.f / D) + in.eps);
    }
    uint32_t z[8];
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 own = with[i][t], other = with[4 + i][t];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 mine = y[2 * i + k], far = Interleaved ? make_float2(mine.y, mine.x) : y[(2 * i + k + 4) % 8];
        const float2 kept = mul2(mine, k == 0 ? make_float2(own.x, own.y) : make_float2(own.z, own.w));
        float2 v = fma2(far, k == 0 ? make_float2(other.x, other.y) : make_float2(other.z, other.w), kept);
        // a dim past rotary_dim is not turned: not by 0 either, which an infinite neighbour would make a NaN
        if (!all_turned) v = turned ? v : kept;
        if (weight != nullptr) v = mul2(v, inv2);
        z[2 * i + k] = Half16<T>::pack(v.x, v.y);
      }
    }
    if (turned || weight != nullptr) {  // else it keeps its bits
      a = make_uint4(z[0], z[1], z[2], z[3]);
      b = make_uint4(z[4], z[5], z[6], z[7]);
    }
  };
  // keys or values of the row's token into the cache
  auto put = [&](int kv, int h, int qa, int qb, const uint4& a, const uint4& b, bool on) {
    if constexpr (To == Into::kCache16) {
      if (on) {
        uint4* out = reinterpret_cast<uint4*>(c.pool + c.block(page, in.layer, kv) +
                                              (static_cast<int64_t>(h) * c.page_size + in_page) * D);
        out[qa] = a;
        out[qb] = b;
      }
    } else {
      unsigned char* block = block4(c, page, in.layer, kv, on ? h : 0);
      if constexpr (D == 64) {
        Extent4<T> e = Extent4<T>::of(a);
        e.take(b);
        e.join(L);
        const Pair4<T> g(e);
        if (on) {
          *codes_at(c, block, in_page, qa) = g.codes(a);
          *codes_at(c, block, in_page, qb) = g.codes(b);
          if (t == 0) *pair_at(c, block, in_page, 0) = g.bits;
        }
      } else {
        // either piece may belong to either group: where a lane has none, an extent that changes nothing
        const Extent4<T> ea = Extent4<T>::of(a), eb = Extent4<T>::of(b);
        constexpr uint32_t kMost = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
        const Extent4<T> none{kMost, kMost | 0x80008000u};
        Extent4<T> e0 = qa < 8 ? ea : none, e1 = qa < 8 ? none : ea;
        if (qb < 8) {
          e0 = {min2<T>(e0.low, eb.low), max2<T>(e0.high, eb.high)};
        } else {
          e1 = {min2<T>(e1.low, eb.low), max2<T>(e1.high, eb.high)};
        }
        e0.join(L);
        e1.join(L);
        const Pair4<T> g0(e0), g1(e1);
        if (on) {
          *codes_at(c, block, in_page, qa) = (qa < 8 ? g0 : g1).codes(a);
          *codes_at(c, block, in_page, qb) = (qb < 8 ? g0 : g1).codes(b);
          if (t < 2) *pair_at(c, block, in_page, t) = t == 0 ? g0.bits : g1.bits;
        }
      }
    }
  };
  for (int base = p0; base < p1; base += kRotAhead) {
#pragma unroll
    for (int n = 0; n < kRotAhead; ++n) {
      const int p = base + n;
      if (p >= p1) break;
      uint4 a = x[n][0], b = x[n][1];
      load(n, p + kRotAhead);
      if (To != Into::kRows && p >= qp + kp) {
        const int h = (p - qp - kp) * H + j;
        if (page >= 0) put(1, h, t, t + L, a, b, h < in.kv_heads);
        continue;
      }
      const bool is_q = p < qp;
      const int h = (is_q ? p : p - qp) * H + j;
      const bool on = h < (is_q ? in.q_heads : in.kv_heads);
      turn_head(is_q, a, b);
      if (is_q || To == Into::kRows) {
        if (!known) a = b = make_uint4(0, 0, 0, 0);
        if (on) {
          uint4* out = reinterpret_cast<uint4*>((is_q ? in.q_out + row * in.q_out_row : in.k_out + row * in.k_out_row) +
                                                static_cast<int64_t>(h) * D);
          out[pa] = a;
          out[pb] = b;
        }
      } else if (page >= 0) {
        put(0, h, pa, pb, a, b, on);
      }
    }
  }
}

bool rotation_checked(const mtt_b200_rotation_t* r) {
  return r != nullptr && (r->head_dim == 64 || r->head_dim == 128) && r->rotary_dim >= 16 && r->rotary_dim <= r->head_dim &&
         r->rotary_dim % 16 == 0 && (r->dtype == MTT_B200_DTYPE_BF16 || r->dtype == MTT_B200_DTYPE_F16) &&
         r->turns != nullptr && (reinterpret_cast<uintptr_t>(r->turns) & 7u) == 0 && aligned16(r->q_weight) &&
         aligned16(r->k_weight) && r->eps >= 0.f && std::isfinite(r->eps);
}

bool rows_ok(const void* p, int64_t stride) { return p != nullptr && aligned16(p) && stride % 8 == 0; }

bool rotate_rows_checked(const mtt_b200_rotate_rows_t* r) {
  return r != nullptr && r->rows >= 0 && r->rows <= kCacheMaxRows && r->q_heads >= 0 && r->q_heads <= 65536 &&
         r->kv_heads >= 0 && r->kv_heads <= 65536 &&
         (r->rows == 0 || r->q_heads == 0 || (rows_ok(r->q, r->q_row_stride) && rows_ok(r->q_out, r->q_out_row_stride))) &&
         (r->rows == 0 || r->kv_heads == 0 || rows_ok(r->k, r->k_row_stride));
}

int run(const PagedCache& c, const mtt_b200_rotation_t& rot, const mtt_b200_rotate_rows_t& r, Into to, cudaStream_t stream) {
  RotArgs in{rot.rotary_dim, rot.interleaved != 0, r.rows, r.q_heads, r.kv_heads, r.layer, 1, rot.eps, rot.turns,
             rot.q_weight, rot.k_weight, static_cast<const uint16_t*>(r.q), static_cast<const uint16_t*>(r.k),
             static_cast<const uint16_t*>(r.v), static_cast<uint16_t*>(r.q_out), static_cast<uint16_t*>(r.k_out),
             r.q_row_stride, r.k_row_stride, r.v_row_stride, r.q_out_row_stride, r.k_out_row_stride, r.positions, r.offsets};
  const int heads = 32 / (rot.head_dim / 16), qp = (r.q_heads + heads - 1) / heads, kp = (r.kv_heads + heads - 1) / heads;
  const int passes = qp + (to == Into::kRows ? 1 : 2) * kp;
  if (r.rows == 0 || passes == 0) return MTT_B200_STATUS_OK;
  // few rows: a row's heads are dealt to several warps
  const int sms = cache_sm_count();
  in.chunks = std::max(1, std::min(passes, (sms * 16 + r.rows - 1) / r.rows));
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(r.rows) * in.chunks + kRotWarps - 1) / kRotWarps));
  auto go = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    auto kernel = [&](auto interleaved) {
      constexpr bool I = decltype(interleaved)::value;
      return to == Into::kRows      ? rotate_kernel<T, D, Into::kRows, I>
             : to == Into::kCache16 ? rotate_kernel<T, D, Into::kCache16, I>
                                    : rotate_kernel<T, D, Into::kCache4, I>;
    };
    return launch_serialized(in.interleaved != 0 ? kernel(std::true_type{}) : kernel(std::false_type{}), grid, dim3(kRotThreads),
                             0, stream, c, in);
  };
  auto pick = [&](auto type) {
    return rot.head_dim == 64 ? go(type, std::integral_constant<int, 64>{}) : go(type, std::integral_constant<int, 128>{});
  };
  return cache_call_status(rot.dtype == MTT_B200_DTYPE_BF16 ? pick(__nv_bfloat16{}) : pick(__half{}));
}

}  // namespace
}  // namespace mtt

using namespace mtt;

extern "C" {

int mtt_b200_launch_rotate_heads(const mtt_b200_rotation_t* rotation, const mtt_b200_rotate_rows_t* rows, void* stream) {
  if (!rotation_checked(rotation) || !rotate_rows_checked(rows) ||
      (rows->rows > 0 && (rows->positions == nullptr || (rows->kv_heads > 0 && !rows_ok(rows->k_out, rows->k_out_row_stride)))))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  return run(PagedCache{}, *rotation, *rows, Into::kRows, static_cast<cudaStream_t>(stream));
}

int mtt_b200_launch_paged_cache_append(const mtt_b200_paged_cache_t* cache, const mtt_b200_rotation_t* rotation,
                                       const mtt_b200_rotate_rows_t* rows, void* stream) {
  PagedCache c;
  if (!paged_cache_view(cache, &c) || !rotation_checked(rotation) || !rotate_rows_checked(rows) ||
      rotation->head_dim != c.head_dim || rotation->dtype != c.dtype || rows->kv_heads != c.kv_heads || rows->layer < 0 ||
      rows->layer >= c.layers ||
      (rows->rows > 0 && (!rows_ok(rows->v, rows->v_row_stride) || (rows->offsets == nullptr && rows->rows > c.slots))))
    return MTT_B200_STATUS_INVALID_ARGUMENT;
  return run(c, *rotation, *rows, c.bits == 4 ? Into::kCache4 : Into::kCache16, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

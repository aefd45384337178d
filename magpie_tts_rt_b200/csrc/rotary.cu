// Norm and position rotation of query and key heads, alone (rotate) or on the
// way into the paged cache (append).
//
//   y = x w / sqrt(mean x^2 + eps);  (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)
//
// HBM bounds it: every element is read and written once.  A head is held by
// head_dim / 16 lanes as two 16-byte pieces each, chosen so that both dims of
// every pair lie in the same lane and a lane has the same 8 pairs in every head:
// a warp, which takes heads of one row, finds its row's cosines and sines once
// (each lane a pair or two, exchanged through shared memory) and keeps them in
// registers, as it does the weights.  The mean takes two or three shuffles.
//
// The angle is position x turns in 64 bits, of which only the part past whole
// turns is kept: exact to 2^-22 of a turn at positions up to 2^31, where a 32-bit
// product would be off by whole turns.
#include <cmath>

#include "cache4.cuh"

namespace mtt {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotAhead = 4;  // passes whose loads are in flight together

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

template <typename T, int D, Into To>
__global__ void __launch_bounds__(kRotThreads) rotate_kernel(PagedCache c, RotArgs in) {
  constexpr int L = D / 16, H = 32 / L;  // lanes of a head, heads of a pass
  __shared__ float2 turn[kRotWarps][D / 2];
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
  const bool turned = t < in.rotary_dim / 16;
  const int pa = turned && !in.interleaved ? t : 2 * t;
  const int pb = turned && !in.interleaved ? t + in.rotary_dim / 16 : 2 * t + 1;

  uint4 x[kRotAhead][2];
  auto load = [&](int n, int p) {
    const bool is_q = p < qp, is_k = !is_q && p < qp + kp;
    const int h = (is_q ? p : is_k ? p - qp : p - qp - kp) * H + j;
    if (p >= p1 || h >= (is_q ? in.q_heads : in.kv_heads)) {
      x[n][0] = x[n][1] = make_uint4(0, 0, 0, 0);
      return;
    }
    const uint16_t* src = is_q ? in.q + row * in.q_row : is_k ? in.k + row * in.k_row : in.v + row * in.v_row;
    src += static_cast<int64_t>(h) * D;
    x[n][0] = *(reinterpret_cast<const uint4*>(src) + (is_q || is_k ? pa : t));
    x[n][1] = *(reinterpret_cast<const uint4*>(src) + (is_q || is_k ? pb : t + L));
  };
#pragma unroll
  for (int n = 0; n < kRotAhead; ++n) load(n, p0 + n);

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
  for (int i = lane; i < in.rotary_dim / 2; i += 32) {
    const double turns = position * in.turns[i];
    float s, cs;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &cs);
    turn[warp][i] = make_float2(cs, s);
  }
  __syncwarp();
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = turned ? turn[warp][8 * t + i] : make_float2(1.f, 0.f);
    cs[i] = v.x;
    sn[i] = v.y;
  }

  float w[16];
  const float* weight = nullptr;
  for (int base = p0; base < p1; base += kRotAhead) {
#pragma unroll
    for (int n = 0; n < kRotAhead; ++n) {
      const int p = base + n;
      if (p >= p1) break;
      const bool is_q = p < qp, is_k = !is_q && p < qp + kp;
      const int h = (is_q ? p : is_k ? p - qp : p - qp - kp) * H + j;
      const bool on = h < (is_q ? in.q_heads : in.kv_heads);
      uint4 a = x[n][0], b = x[n][1];
      if (is_q || is_k) {
        const float* mine = is_q ? in.q_weight : in.k_weight;
        float y[16];
        {
          const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = unpack2<T>(u[i]);
            y[2 * i] = v.x;
            y[2 * i + 1] = v.y;
          }
        }
        if (mine != nullptr) {
          if (mine != weight) {  // once for the queries, once for the keys
            weight = mine;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              *reinterpret_cast<float4*>(w + 4 * i) = *(reinterpret_cast<const float4*>(mine + 8 * pa) + i);
              *reinterpret_cast<float4*>(w + 8 + 4 * i) = *(reinterpret_cast<const float4*>(mine + 8 * pb) + i);
            }
          }
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum = fmaf(y[i], y[i], sum);
#pragma unroll
          for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = rsqrtf(sum * (1.f / D) + in.eps);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = y[i] * inv * w[i];
        }
        float z[16];
        if (in.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[2 * i] = fmaf(y[2 * i], cs[i], -y[2 * i + 1] * sn[i]);
            z[2 * i + 1] = fmaf(y[2 * i + 1], cs[i], y[2 * i] * sn[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[i] = fmaf(y[i], cs[i], -y[8 + i] * sn[i]);
            z[8 + i] = fmaf(y[8 + i], cs[i], y[i] * sn[i]);
          }
        }
        // a dim past rotary_dim is not turned: not by 0 either, which an infinite neighbour would make a NaN
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = turned ? z[i] : y[i];
        if (turned || mine != nullptr) {  // else it keeps its bits
          a = make_uint4(Half16<T>::pack(z[0], z[1]), Half16<T>::pack(z[2], z[3]), Half16<T>::pack(z[4], z[5]),
                         Half16<T>::pack(z[6], z[7]));
          b = make_uint4(Half16<T>::pack(z[8], z[9]), Half16<T>::pack(z[10], z[11]), Half16<T>::pack(z[12], z[13]),
                         Half16<T>::pack(z[14], z[15]));
        }
      }
      if (is_q) {
        if (!known) a = b = make_uint4(0, 0, 0, 0);
        if (on) {
          uint4* out = reinterpret_cast<uint4*>(in.q_out + row * in.q_out_row + static_cast<int64_t>(h) * D);
          out[pa] = a;
          out[pb] = b;
        }
      } else if constexpr (To == Into::kRows) {
        if (on) {
          uint4* out = reinterpret_cast<uint4*>(in.k_out + row * in.k_out_row + static_cast<int64_t>(h) * D);
          out[pa] = a;
          out[pb] = b;
        }
      } else if (page >= 0) {
        const int qa = is_k ? pa : t, qb = is_k ? pb : t + L;  // the pieces' numbers
        if constexpr (To == Into::kCache16) {
          if (on) {
            uint4* out = reinterpret_cast<uint4*>(c.pool + c.block(page, in.layer, is_k ? 0 : 1) +
                                                  (static_cast<int64_t>(h) * c.page_size + in_page) * D);
            out[qa] = a;
            out[qb] = b;
          }
        } else {
          unsigned char* block = block4(c, page, in.layer, is_k ? 0 : 1, on ? h : 0);
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
      }
    }
#pragma unroll
    for (int n = 0; n < kRotAhead; ++n) load(n, base + kRotAhead + n);
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
    const auto kernel = to == Into::kRows      ? rotate_kernel<T, D, Into::kRows>
                        : to == Into::kCache16 ? rotate_kernel<T, D, Into::kCache16>
                                               : rotate_kernel<T, D, Into::kCache4>;
    return launch_serialized(kernel, grid, dim3(kRotThreads), 0, stream, c, in);
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

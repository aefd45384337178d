// The 4-bit form of the paged cache's pool (MTT_B200_CACHE_4BIT): where a
// token's codes and (step, low) pairs lie, and how they are made from 16-bit
// values and turned back into them.
#pragma once

#include "paged_attention.cuh"

namespace mtt {

constexpr int kGroup4 = 64;  // dims that share a pair

// Bytes of one head's block in a page; of them the codes' come first.
__device__ __forceinline__ int block4_bytes(const PagedCache& c) { return c.page_size * 9 * c.head_dim / 16; }
__device__ __forceinline__ int block4_codes(const PagedCache& c) { return c.page_size * c.head_dim / 2; }

// The block of (page, layer, keys or values, head).
__device__ __forceinline__ unsigned char* block4(const PagedCache& c, int page, int layer, int kv, int head) {
  return reinterpret_cast<unsigned char*>(c.pool + c.block(page, layer, kv)) + static_cast<int64_t>(head) * block4_bytes(c);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Two 16-bit minima or maxima; NaN if either is.
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t min2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t min2<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Smallest and largest of a group so far, in two lanes of 16 bits each.
template <typename T>
struct Extent4 {
  uint32_t low, high;
  __device__ __forceinline__ void take(const uint4& x) {
    low = min2<T>(low, min2<T>(min2<T>(x.x, x.y), min2<T>(x.z, x.w)));
    high = max2<T>(high, max2<T>(max2<T>(x.x, x.y), max2<T>(x.z, x.w)));
  }
  __device__ __forceinline__ void join(int lanes) {  // with the lanes that differ in these bits of their number
    for (int o = 1; o < lanes; o <<= 1) {
      low = min2<T>(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = max2<T>(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
  }
  static __device__ __forceinline__ Extent4 of(const uint4& x) {
    return {min2<T>(min2<T>(x.x, x.y), min2<T>(x.z, x.w)), max2<T>(max2<T>(x.x, x.y), max2<T>(x.z, x.w))};
  }
};

// A group's pair, and what its codes are chosen with.  Every operation is
// rounded as the format says (no contraction): the codes do not depend on which
// kernel stores a token.
template <typename T>
struct Pair4 {
  float low, inverse;
  uint32_t bits;  // step, low
  __device__ __forceinline__ explicit Pair4(const Extent4<T>& e) {
    low = unpack2<T>(min2<T>(e.low, e.low >> 16 | e.low << 16)).x;
    const float high = unpack2<T>(max2<T>(e.high, e.high >> 16 | e.high << 16)).x;
    const float spread = __fsub_rn(high, low);
    // not finite: the whole group reads as NaN
    const float wide = spread <= 3.402823466e38f ? fifteenth(spread) : CUDART_NAN_F;
    bits = Half16<T>::pack(wide, low);
    const float step = unpack2<T>(bits).x;
    inverse = step >= 1.17549435e-38f ? __frcp_rn(step) : 0.f;
  }
  // x / 15 rounded to nearest: the product with the rounded reciprocal, and one step with what is left (Markstein 1990);
  // numbers so small that what is left could be lost are divided
  static __device__ __forceinline__ float fifteenth(float x) {
    constexpr float kBy = 1.f / 15.f;
    if (x < 1e-25f) return __fdiv_rn(x, 15.f);
    const float q = x * kBy;
    return fmaf(fmaf(-15.f, q, x), kBy, q);
  }
  // The codes of 8 values.  1.5 * 2^23 is added, which rounds to a whole number, half to even, and leaves the code in the
  // lowest bits of 0x4b400000 + code; eight of them are put together by products, whose constant parts add up to one.
  // (The minimum holds back what a step far below f16's normal range asks for, and keeps product and sum two operations.)
  __device__ __forceinline__ uint32_t codes(const uint4& x) const {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    const float2 less = make_float2(-low, -low), by = make_float2(inverse, inverse), whole = make_float2(12582912.f, 12582912.f);
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v = mul2(add2(unpack2<T>(w[i]), less), by);
      v = add2(make_float2(fminf(v.x, 15.f), fminf(v.y, 15.f)), whole);
      r += __float_as_uint(v.x) * (1u << (4 * i)) + __float_as_uint(v.y) * (1u << (4 * i + 16));
    }
    return inverse == 0.f ? 0u : r - 0x4b400000u * 0x11111111u;  // (no step: the group is constant, or not finite)
  }
};

// Codes of dims 2 I and 2 I + 1 of the eight in w, as 16 + code in 16 bits each:
// the code goes into the upper mantissa bits of 16.0, so that it takes a shift and
// one three-input operation, and nothing is rounded.
template <typename T, int I>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) {
    const uint32_t x = I == 0 ? w << 6 : I == 1 ? w << 2 : w >> (4 * I - 6);
    return (x & 0x03c003c0u) | 0x4c004c00u;
  } else {
    const uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3);
    return (x & 0x00780078u) | 0x41804180u;
  }
}

// step, and what belongs to 16 + code: value = step (16 + code) + off
__device__ __forceinline__ float2 step_off(float2 pair) { return make_float2(pair.x, fmaf(-16.f, pair.x, pair.y)); }

// value = low + step * (codes2 - 16), two at a time: the subtraction is exact, the
// rest rounded once.  step2, low2: step and low twice.
template <typename T>
__device__ __forceinline__ uint32_t value2(uint32_t c16, uint32_t step2, uint32_t low2);
template <>
__device__ __forceinline__ uint32_t value2<__nv_bfloat16>(uint32_t c16, uint32_t step2, uint32_t low2) {
  uint32_t r;
  asm("{\n .reg .b32 c;\n add.rn.bf16x2 c, %1, %4;\n fma.rn.bf16x2 %0, c, %2, %3;\n}\n"
      : "=r"(r) : "r"(c16), "r"(step2), "r"(low2), "r"(0xc180c180u));
  return r;
}
template <>
__device__ __forceinline__ uint32_t value2<__half>(uint32_t c16, uint32_t step2, uint32_t low2) {
  uint32_t r;
  asm("{\n .reg .b32 c;\n add.rn.f16x2 c, %1, %4;\n fma.rn.f16x2 %0, c, %2, %3;\n}\n"
      : "=r"(r) : "r"(c16), "r"(step2), "r"(low2), "r"(0xcc00cc00u));
  return r;
}

// The values of 8 codes, rounded to 16 bits.
template <typename T>
__device__ __forceinline__ uint4 values4(uint32_t codes, uint32_t pair) {
  const uint32_t step2 = __byte_perm(pair, 0, 0x1010), low2 = __byte_perm(pair, 0, 0x3232);
  return make_uint4(value2<T>(codes2<T, 0>(codes), step2, low2), value2<T>(codes2<T, 1>(codes), step2, low2),
                    value2<T>(codes2<T, 2>(codes), step2, low2), value2<T>(codes2<T, 3>(codes), step2, low2));
}

// Where a token's 8 dims from 8 * piece on, and the pair of its group, lie in its block.
__device__ __forceinline__ uint32_t* codes_at(const PagedCache& c, unsigned char* block, int in_page, int piece) {
  return reinterpret_cast<uint32_t*>(block + in_page * (c.head_dim / 2)) + piece;
}
__device__ __forceinline__ uint32_t* pair_at(const PagedCache& c, unsigned char* block, int in_page, int group) {
  return reinterpret_cast<uint32_t*>(block + block4_codes(c)) + in_page * (c.head_dim / kGroup4) + group;
}

}  // namespace mtt

// 4-bit matrix with group scales: storage order and the decoding of its
// codes into 16-bit tensor-core fragments.
//
// W^[n,k] = s[n, k / G] c[n,k], c in -8..7, G in {32, 64, 128}. A matrix is
// cut into blocks of 16 rows by 128 columns (zero padded), 1 KB each, in the
// order in which a warp's lanes want them: lane 4 g + t holds rows g and g + 8
// as 16 bytes each, the bytes of row half h at h * 512 + lane * 16. Word w of
// those 16 bytes holds the eight codes k = 32 w + 8 t + i; code i sits, biased
// by 8, in nibble i / 2 (i even) or 4 + i / 2 (i odd), so that
// (word >> 4 j) & 0x000f000f is the pair (2 j, 2 j + 1) as two 16-bit lanes.
// A warp so reads a block with two fully coalesced 16-byte loads a lane, and
// the k order of a fragment (any order serves that the other operand shares)
// keeps eight neighbouring k in a lane, which x is read by.
// Scales: [row tile][k block][128 / G][16 rows], bf16 or fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace tt {
namespace q4 {

constexpr int kRows = 16;     // rows of a block
constexpr int kCols = 128;    // columns of a block
constexpr int kBlockBytes = kRows * kCols / 2;

enum Type : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// (x & m) | o in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(m), "r"(o));
  return r;
}

// A pair of biased codes (bits 0-3 and 16-19 of x) as two exact 16-bit
// floats. The code goes into the mantissa of 128 (bf16, whose unit in the
// last place there is 1) or 1024 (fp16), and 128 + 8 or 1024 + 8 comes off.
template <bool kHalf>
__device__ __forceinline__ uint32_t decode_pair(uint32_t x) {
  if constexpr (kHalf) {
    const uint32_t v = and_or(x, 0x000f000fu, 0x64006400u);
    const __half2 r = __hsub2(reinterpret_cast<const __half2&>(v), __half2half2(__ushort_as_half(0x6408)));
    return reinterpret_cast<const uint32_t&>(r);
  } else {
    const uint32_t v = and_or(x, 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162&>(v),
                                     __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
    return reinterpret_cast<const uint32_t&>(r);
  }
}

// Two fp16 pairs at a time, from nibbles 0 and 1 of each half of x: the second
// stands 16 times too high in the mantissa, which the fused multiply-add that
// takes the bias off puts right, instead of a shift.
__device__ __forceinline__ void decode_two_pairs(uint32_t x, uint32_t& first, uint32_t& second) {
  const uint32_t a = and_or(x, 0x000f000fu, 0x64006400u), b = and_or(x, 0x00f000f0u, 0x64006400u);
  const __half2 ra = __hsub2(reinterpret_cast<const __half2&>(a), __half2half2(__ushort_as_half(0x6408)));  // 1032
  const __half2 rb = __hfma2(reinterpret_cast<const __half2&>(b), __half2half2(__ushort_as_half(0x2c00)),   // 1 / 16
                             __half2half2(__ushort_as_half(0xd480)));                                       // -72
  first = reinterpret_cast<const uint32_t&>(ra);
  second = reinterpret_cast<const uint32_t&>(rb);
}

// The same for either type (bf16's mantissa is too short for the second form).
template <bool kHalf>
__device__ __forceinline__ void decode_four(uint32_t x, uint32_t& first, uint32_t& second) {
  if constexpr (kHalf) {
    decode_two_pairs(x, first, second);
  } else {
    first = decode_pair<false>(x);
    second = decode_pair<false>(x >> 4);
  }
}

// Not volatile: the compiler moves it past the loads.
template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kHalf) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}

// Two floats as kTerms bf16 pairs that add up to them. Each term but the last
// takes the value's next 8 bits as they stand (so fp32's largest value does
// not round up to infinity) and the last is rounded: two terms leave 2^-16 of
// the value, three nothing. An infinity stays in the first term alone.
template <int kTerms>
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t (&out)[kTerms]) {
#pragma unroll
  for (int i = 0; i + 1 < kTerms; ++i) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    out[i] = __byte_perm(ua, ub, 0x7632);
    a = (ua << 1) == 0xff000000u ? 0.f : a - __uint_as_float(ua & 0xffff0000u);
    b = (ub << 1) == 0xff000000u ? 0.f : b - __uint_as_float(ub & 0xffff0000u);
  }
  out[kTerms - 1] = pack_bf16(a, b);
}

// Plain loads, volatile: moved towards their use, or with a conversion beside
// them, they would make the warp wait there and then. Callers give an address
// that holds, and drop what they did not want when they use it.
__device__ __forceinline__ uint4 ldg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg64(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ldg32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ldg16(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
// The word that holds scale i (bf16: with its neighbour), and the scale in it.
__device__ __forceinline__ uint32_t scale_word(const void* scales, bool f32, long long i) {
  return ldg32(static_cast<const char*>(scales) + (f32 ? 4 * i : (2 * i & ~3LL)));
}
__device__ __forceinline__ float scale_value(uint32_t word, bool f32, int odd) {
  return __uint_as_float(f32 ? word : odd ? word & 0xffff0000u : word << 16);
}

}  // namespace q4
}  // namespace tt

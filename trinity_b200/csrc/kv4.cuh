// Reading the 4-bit form of a cache row: eight codes and their group's (s, lo) into eight 16-bit values.
#pragma once

#include "common.cuh"

namespace tb200 {

template <typename T> struct Kv4Decode;

// A code in the low mantissa bits of a 16-bit float whose exponent makes one mantissa step a 1: 1024 + c in fp16,
// 128 + c in bf16.  Subtracting the offset is exact, and lo + c s is one fused multiply-add: rounded once.  s is rounded, so
// lo + 15 s may pass the type's largest number where max x is next to it: such a value is read as that number (a NaN stays one).
template <> struct Kv4Decode<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;
  static __device__ __forceinline__ uint32_t pair(uint32_t two_codes, __half2 s, __half2 lo) {
    uint32_t u = two_codes | kMagic;
    __half2 c = __hsub2(*reinterpret_cast<__half2*>(&u), __float2half2_rn(1024.f));
    __half2 v = __hmin2_nan(__hfma2(c, s, lo), __half2half2(__ushort_as_half(0x7bffu)));
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint4 decode8(uint32_t word, uint32_t meta) {
    uint32_t sb = __byte_perm(meta, meta, 0x1010), lb = __byte_perm(meta, meta, 0x3232);
    const __half2 s = *reinterpret_cast<__half2*>(&sb), lo = *reinterpret_cast<__half2*>(&lb);
    // pairs (0,4) (1,5) (2,6) (3,7)
    const uint32_t a = pair(word & 0x000f000fu, s, lo), b = pair((word >> 4) & 0x000f000fu, s, lo);
    const uint32_t c = pair((word >> 8) & 0x000f000fu, s, lo), d = pair((word >> 12) & 0x000f000fu, s, lo);
    return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632));
  }
};

template <> struct Kv4Decode<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;
  static __device__ __forceinline__ uint32_t pair(uint32_t two_codes, __nv_bfloat162 s, __nv_bfloat162 lo) {
    uint32_t u = two_codes | kMagic;
    __nv_bfloat162 c = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), __float2bfloat162_rn(128.f));
    __nv_bfloat162 v = __hmin2_nan(__hfma2(c, s, lo), __bfloat162bfloat162(__ushort_as_bfloat16(0x7f7fu)));
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint4 decode8(uint32_t word, uint32_t meta) {
    uint32_t sb = __byte_perm(meta, meta, 0x1010), lb = __byte_perm(meta, meta, 0x3232);
    const __nv_bfloat162 s = *reinterpret_cast<__nv_bfloat162*>(&sb), lo = *reinterpret_cast<__nv_bfloat162*>(&lb);
    const uint32_t a = pair(word & 0x000f000fu, s, lo), b = pair((word >> 4) & 0x000f000fu, s, lo);
    const uint32_t c = pair((word >> 8) & 0x000f000fu, s, lo), d = pair((word >> 12) & 0x000f000fu, s, lo);
    return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632));
  }
};

}  // namespace tb200

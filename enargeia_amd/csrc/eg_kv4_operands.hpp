// Matrix operands from the paged 4-bit cache, for the attentions that read it (the forms that K and V codes
// take in the products, and why, stand in eg_kv4_attention.hip). Not part of the ABI.
#pragma once

#include "eg_kv4.hpp"

namespace eg_kv4 {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
using egd::u32x4;

constexpr float kLargest = 0x1p20f;
constexpr float kLog2e = 1.44269504088896340736f;
// slot of an 8-deep operand -> nibble of a word, as the two masks below deliver them
constexpr uint32_t kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};

// Max over the 4 lanes that hold a head (lane % 16).
__device__ __forceinline__ float max_of_head(float x) {
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto t = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}
__device__ __forceinline__ half2v halves(uint32_t v) { return __builtin_bit_cast(half2v, v); }
__device__ __forceinline__ uint32_t bits(half2v v) { return __builtin_bit_cast(uint32_t, v); }

// Bits put over four of a word's nibbles: one v_and_or_b32 where they are in a register (as a literal,
// beside the mask, they take an instruction of their own).
struct Magic {
  uint32_t lo, hi;  // f16 1024 (a nibble at the bottom: 1024 + code), f16 64 (the next one: 64 + code)
};
__device__ __forceinline__ Magic magic() {
  Magic m{0x64006400u, 0x54005400u};
  asm("" : "+v"(m.lo), "+v"(m.hi));
  return m;
}

// 8 codes as the first product takes them: slots 0, 1, 4, 5 code * 2^-24, slots 2, 3, 6, 7 code * 2^-20
// (code is value + 8 here); or, kSigned, the values -7 .. 7 themselves.
template <bool kSigned>
__device__ __forceinline__ half8 codes(uint32_t w, const Magic& m) {
  const uint32_t y = w >> 8;
  if constexpr (kSigned) {
    const half2v lo = {(_Float16)-1032.f, (_Float16)-1032.f}, hi = {(_Float16)-72.f, (_Float16)-72.f};
    return as_half8(bits(halves((w & 0x000F000Fu) | m.lo) + lo), bits(halves((w & 0x00F000F0u) | m.hi) + hi),
                    bits(halves((y & 0x000F000Fu) | m.lo) + lo), bits(halves((y & 0x00F000F0u) | m.hi) + hi));
  } else {
    return as_half8(w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u);
  }
}

// 8 codes of one dim at 8 positions, times the positions' scales (pairs in kOrder's order).
__device__ __forceinline__ half8 values(uint32_t w, const half2v (&s)[4], const Magic& m) {
  const uint32_t y = w >> 8;
  const half2v lo = {(_Float16)-1032.f, (_Float16)-1032.f}, hi = {(_Float16)-72.f, (_Float16)-72.f};
  const half2v a = (halves((w & 0x000F000Fu) | m.lo) + lo) * s[0];  // 1024 + code
  const half2v b = (halves((w & 0x00F000F0u) | m.hi) + hi) * s[1];  // 64 + code
  const half2v c = (halves((y & 0x000F000Fu) | m.lo) + lo) * s[2];
  const half2v d = (halves((y & 0x00F000F0u) | m.hi) + hi) * s[3];
  return as_half8(bits(a), bits(b), bits(c), bits(d));
}

// 8 consecutive scales as pairs in kOrder's order.
__device__ __forceinline__ void scale_pairs(const u32x4& s, half2v (&pairs)[4]) {
  pairs[0] = halves(__builtin_amdgcn_perm(s.z, s.x, 0x05040100u));
  pairs[1] = halves(__builtin_amdgcn_perm(s.z, s.x, 0x07060302u));
  pairs[2] = halves(__builtin_amdgcn_perm(s.w, s.y, 0x05040100u));
  pairs[3] = halves(__builtin_amdgcn_perm(s.w, s.y, 0x07060302u));
}

__device__ __forceinline__ float half_of(const u32x4& s, uint32_t i) {
  const half2v h = halves(s[i / 2]);
  return (float)(i % 2 ? h.y : h.x);
}

// The first `n` (0..8) of 8 halves, the others zero.
__device__ __forceinline__ u32x4 first_halves(u32x4 v, int n) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] &= n >= 2 * i + 2 ? 0xFFFFFFFFu : n == 2 * i + 1 ? 0xFFFFu : 0u;
  return v;
}

}  // namespace eg_kv4

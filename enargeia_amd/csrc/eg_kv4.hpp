// What the kernels over the paged 4-bit cache share (format and page layout: enargeia_hip.h).
// Not part of the ABI.
#pragma once

#include <type_traits>

#include "eg_internal.hpp"

namespace eg_kv4 {

// Where a kv head's four streams lie in its block of a page, in bytes.
struct Layout {
  uint32_t head_bytes, v_codes, k_scales, v_scales;
};
template <int D>
__host__ __device__ __forceinline__ Layout layout(uint32_t page) {
  return Layout{page * (D + D / 8), page * (D / 2), page * D, page * D + page * (D / 16)};
}

// The pool and its page table as the kernels take them.
struct Pool {
  uint8_t* base;
  const uint32_t* table;
  uint64_t stride;
  uint32_t pages, max_pages, page_shift, kv_heads, sequences;
  // The page of a sequence's position; `pages` or more where there is none.
  __device__ __forceinline__ uint32_t page_of(uint32_t seq, uint32_t position) const {
    const uint32_t i = position >> page_shift;
    return i < max_pages ? table[(size_t)seq * max_pages + i] : 0xFFFFFFFFu;
  }
  __device__ __forceinline__ uint8_t* block(uint32_t page, uint32_t kv, uint32_t head_bytes) const {
    return base + (uint64_t)page * stride + (uint64_t)kv * head_bytes;
  }
};

inline uint32_t log2_of(uint32_t v) { return 31u - (uint32_t)__builtin_clz(v); }

inline Pool pool_of(const eg_kv4_dims& d, const void* pool, const uint32_t* table) {
  return Pool{const_cast<uint8_t*>(static_cast<const uint8_t*>(pool)), table, d.page_stride, d.pages, d.max_pages,
              log2_of(d.page_size), d.kv_heads, d.sequences};
}

inline uint64_t page_bytes(const eg_kv4_dims& d) {
  return (uint64_t)d.kv_heads * d.page_size * (d.head_dim + d.head_dim / 8);
}

// The context's device as the current one while a call launches.
class OnDevice {
 public:
  explicit OnDevice(const eg_context* ctx) {
    int now = ctx->device;
    if (hipGetDevice(&now) == hipSuccess && now != ctx->device && hipSetDevice(ctx->device) == hipSuccess) before_ = now;
  }
  ~OnDevice() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int before_ = -1;
};

// The checks every entry point over a pool makes.
int check_dims(eg_context* ctx, const char* op, const eg_kv4_dims* dims, const void* pool);

// Rows as memory holds them.
struct bf16 {
  uint16_t bits;
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, bf16>::value) return bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};
  else return (T)v;
}

// f with T one of float, _Float16, bf16 for an eg_element.
template <class F>
void with_type(int element, F&& f) {
  if (element == EG_ELEMENT_F32) f(float{});
  else if (element == EG_ELEMENT_F16) f(_Float16{});
  else f(bf16{});
}

inline bool known_type(int element) { return element >= EG_ELEMENT_F32 && element <= EG_ELEMENT_BF16; }

// The sequence that packed row r belongs to: the last s with offsets[s] <= r, `sequences` or more
// (or none) where r is in no sequence. The wave reads 64 offsets at a time: one memory latency where
// a bisection has log2(sequences).
__device__ __forceinline__ bool find_sequence(const uint32_t* offsets, uint32_t sequences, uint32_t r, uint32_t& seq,
                                              uint32_t& first, uint32_t& end) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t below = 0;  // offsets at most r
  for (uint32_t i0 = 0; i0 <= sequences; i0 += 64) {
    const uint32_t i = i0 + lane;
    const uint32_t n = (uint32_t)__builtin_popcountll(__ballot(i <= sequences && offsets[min(i, sequences)] <= r));
    below += n;
    if (n < 64) break;
  }
  if (below == 0 || below > sequences) return false;
  seq = below - 1;
  first = offsets[seq];
  end = offsets[seq + 1];
  return first <= r && r < end;  // (always, of ascending offsets)
}

// A sequence's first position, kept where adding any row index to it stays past every table's reach.
__device__ __forceinline__ uint32_t start_of(const uint32_t* starts, uint32_t seq) { return min(starts[seq], 1u << 31); }

}  // namespace eg_kv4

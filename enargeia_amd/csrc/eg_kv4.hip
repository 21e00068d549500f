// The paged 4-bit cache (enargeia_hip.h): rows appended, rows read back, pages copied. All three move
// bytes: their floor is what they read and write once at the memory's rate.
//
// Append and read go by blocks of positions of a page (8, or 32): a V code word holds 8 positions of one
// dim, so a block's V words are written by one wave from its 8 rows, whole - or, where the batch has
// only some of the 8, merged into what is there (one wave per block and kv head: no race). Packed rows
// and blocks do not align, so a wave that owns `span` packed rows takes the blocks whose first row
// of this call lies among them, rows past its span included.
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256;

// The runs of rows that lie in one block of kBlock positions, for the packed rows [r0, r0 + span):
// f(sequence, first row, its position, rows).
template <uint32_t kBlock, class F>
__device__ __forceinline__ void for_blocks(const uint32_t* offsets, const uint32_t* starts, uint32_t sequences,
                                           uint32_t rows, uint32_t r0, uint32_t span, F&& f) {
  uint32_t r = r0, seq = 0, first = 0, end = 0, start = 0;
  bool have = false;
  const uint32_t stop = min(r0 + span, rows);
  while (r < stop) {
    if (!have || r >= end) {
      // rows before the first sequence are in none: go on with the next row of the span
      if (!find_sequence(offsets, sequences, r, seq, first, end)) {
        if (r >= offsets[sequences]) return;
        r++;
        continue;
      }
      have = true;
      start = start_of(starts, seq);
    }
    const uint32_t position = start + (r - first), in_block = position & (kBlock - 1u);
    const uint32_t n = min(min(kBlock - in_block, end - r), rows - r);
    if (in_block == 0 || r == first) f(seq, r, position, n);
    r += n;
  }
}

// Max over aligned groups of 32 lanes, in every lane.
__device__ __forceinline__ uint32_t max_of_32(uint32_t v) {
  const auto step = [&](int o) { v = max(v, (uint32_t)o); };
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
  step(__builtin_amdgcn_ds_swizzle((int)v, 0x401F));
  return v;
}

// OR over aligned groups of 8 lanes, in every lane.
__device__ __forceinline__ uint32_t or_of_8(uint32_t v) {
  v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
  v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
  v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);
  return v;
}

// The code (0..15) of this lane's value and the f16 bits of its group's scale; a group is 32 lanes.
// The absmax is taken over the values' bits, which order magnitudes and put infinities and NaN on top.
// Products with reciprocals, not divisions: they are what the format says (a division of f32 is some ten
// instructions, and takes a value halfway between two codes to the other one now and then).
__device__ __forceinline__ uint32_t quantize(float x, uint32_t& scale) {
#pragma clang fp contract(off)
  const uint32_t top = max_of_32(__float_as_uint(x) & 0x7FFFFFFFu);
  if (top >= 0x7F800000u) {
    scale = 0x7E00u;
    return 8u;
  }
  const float t = fminf(__uint_as_float(top) * (1.0f / 7.0f), 9344.0f);
  scale = (egd::float_to_half(t) + 4u) & 0xFFF8u;
  const float s = egd::half_to_float((uint16_t)scale);
  const float r = s > 0.f ? 1.0f / s : 0.f;
  return (uint32_t)((int)fminf(fmaxf(rintf(x * r), -7.f), 7.f) + 8);
}

struct AppendArgs {
  const void *q, *k, *v;
  const float2* rope;
  const uint32_t *offsets, *starts;
  void *q_out, *k_out, *v_out;
  uint32_t rows, heads, q_stride, k_stride, v_stride, rope_positions;
  uint32_t span, q_span;          // packed rows per wave of a kv head, per workgroup of queries
  uint32_t kv_groups, kv_blocks;  // workgroups of the kv heads: per span, in all; those of the queries follow
};

// The positions of rows r0 + lane (kNowhere for those of no sequence).
constexpr uint32_t kNowhere = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t position_of(const uint32_t* offsets, const uint32_t* starts, uint32_t sequences,
                                                uint32_t r) {
  uint32_t lo = 0, hi = sequences + 1, first = 0;  // offsets[lo - 1] <= r < offsets[hi], as far as known
  if (sequences < 64) {  // all offsets in the wave's lanes
    const uint32_t mine = offsets[min(threadIdx.x & 63u, sequences)];
    while (__ballot(lo < hi)) {
      const uint32_t mid = (lo + hi) / 2, v = (uint32_t)__shfl((int)mine, (int)min(mid, sequences), 64);
      if (lo < hi) {
        if (v <= r) {
          lo = mid + 1;
          first = v;
        } else {
          hi = mid;
        }
      }
    }
  } else {
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2, v = offsets[mid];
      if (v <= r) {
        lo = mid + 1;
        first = v;
      } else {
        hi = mid;
      }
    }
  }
  return lo == 0 || lo > sequences ? kNowhere : start_of(starts, lo - 1) + (r - first);
}

// 4 consecutive elements.
template <class T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (std::is_same<T, float>::value) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    struct alignas(8) Four {
      T v[4];
    };
    const Four f = *reinterpret_cast<const Four*>(p);
    return make_float4(to_f32(f.v[0]), to_f32(f.v[1]), to_f32(f.v[2]), to_f32(f.v[3]));
  }
}
template <class T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  if constexpr (std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    struct alignas(8) Four {
      T v[4];
    };
    *reinterpret_cast<Four*>(p) = Four{{from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)}};
  }
}

// The queries of `rows` packed rows from r0 on, rotated: a thread has 4 dims of a head's first half and the
// 4 of its second that pair with them. A row is skipped where its position is out of reach.
template <int D, class TI, class TO>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, const Pool& pool, uint32_t r0, uint32_t rows) {
#pragma clang fp contract(off)
  constexpr uint32_t kQuads = D / 8, kAhead = 2;
  __shared__ uint32_t position[64];
  const uint32_t tid = threadIdx.x;
  const TI* q = static_cast<const TI*>(a.q);
  TO* out = static_cast<TO*>(a.q_out);
  const uint32_t per_row = a.heads * kQuads, items = rows * per_row;
  const auto at_of = [&](uint32_t i) { return (i % per_row) / kQuads * D + 4 * (i % kQuads); };  // (kQuads divides per_row)
  const auto read = [&](uint32_t i, float4& u, float4& w) {
    const TI* src = q + (size_t)(r0 + i / per_row) * a.q_stride + at_of(i);
    u = load4(src);
    w = load4(src + D / 2);
  };
  const auto finish = [&](uint32_t i, float4 u, float4 w) {
    const uint32_t r = i / per_row, p = position[r];
    if (p == kNowhere) return;
    if (a.rope) {
      const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)p * (D / 2) + 4 * (i % kQuads));
      const float4 x = cs[0], y = cs[1];  // (cos, sin) of two pairs each
      const float4 s = u;
      u = make_float4(s.x * x.x - w.x * x.y, s.y * x.z - w.y * x.w, s.z * y.x - w.z * y.y, s.w * y.z - w.w * y.w);
      w = make_float4(w.x * x.x + s.x * x.y, w.y * x.z + s.y * x.w, w.z * y.x + s.z * y.y, w.w * y.z + s.w * y.w);
    }
    TO* to = out + (size_t)(r0 + r) * (a.heads * D) + at_of(i);
    store4(to, u);
    store4(to + D / 2, w);
  };
  // What a thread takes first is under way while the positions are found.
  float4 u[kAhead], w[kAhead];
#pragma unroll
  for (uint32_t j = 0; j < kAhead; j++) read(min(tid + j * kThreads, items - 1), u[j], w[j]);
  if (tid < 64) {
    uint32_t p = position_of(a.offsets, a.starts, pool.sequences, r0 + tid);
    if (p != kNowhere && ((p >> pool.page_shift) >= pool.max_pages || (a.rope && p >= a.rope_positions))) p = kNowhere;
    position[tid] = p;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < kAhead; j++)
    if (tid + j * kThreads < items) finish(tid + j * kThreads, u[j], w[j]);
  for (uint32_t i = tid + kAhead * kThreads; i < items; i += kThreads) {
    read(i, u[0], w[0]);
    finish(i, u[0], w[0]);
  }
}

// The first kv_blocks workgroups: a wave per (span of packed rows, kv head's K or V). A lane holds dim
// `lane` of up to 8 rows (and dim lane + 64 at head_dim 128), all read at once. The others: the span's
// queries. Bound by latency where the rows are few, by memory where they are many.
template <int D, class TI, class TO>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, Pool pool) {
  constexpr int kPer = D / 64;  // dims per lane
  const uint32_t kvh = pool.kv_heads;
  if (blockIdx.x >= a.kv_blocks) {
    const uint32_t r0 = (blockIdx.x - a.kv_blocks) * a.q_span;
    rotate_queries<D, TI, TO>(a, pool, r0, min(a.q_span, a.rows - r0));
    return;
  }
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t task = blockIdx.x % a.kv_groups * 4 + wave, r0 = blockIdx.x / a.kv_groups * a.span;
  if (task >= 2 * kvh) return;
  const bool is_k = task < kvh;
  const uint32_t head = is_k ? task : task - kvh;
  const TI* src = static_cast<const TI*>(is_k ? a.k : a.v);
  TO* dst = static_cast<TO*>(is_k ? a.k_out : a.v_out);
  const uint32_t stride = is_k ? a.k_stride : a.v_stride, out_stride = kvh * D;
  const Layout at = layout<D>(1u << pool.page_shift);
  const uint32_t scales_at = is_k ? at.k_scales : at.v_scales;  // (chosen in the lambda it goes through memory)

  for_blocks<8>(a.offsets, a.starts, pool.sequences, a.rows, r0, a.span,
                [&](uint32_t seq, uint32_t row, uint32_t position, uint32_t n) {
    if ((position >> pool.page_shift) >= pool.max_pages) return;
    const uint32_t page = pool.page_of(seq, position);
    if (a.rope) {  // rows that the rope does not reach are skipped
      if (position >= a.rope_positions) return;
      n = min(n, a.rope_positions - position);
    }
    float x[8][kPer];
    float2 cs[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
      const uint32_t r = row + min(i, n - 1);  // (rows past n are read as the last one: never used)
#pragma unroll
      for (int j = 0; j < kPer; j++) x[i][j] = to_f32(src[(size_t)r * stride + head * D + 64 * j + lane]);
      cs[i] = make_float2(1.f, 0.f);
      if (a.rope && is_k)
        cs[i] = a.rope[(size_t)(position + min(i, n - 1)) * (D / 2) + (D == 64 ? lane & 31u : lane)];
    }
    if (a.rope && is_k) {
#pragma clang fp contract(off)
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        if constexpr (D == 64) {  // the pair's other half is 32 lanes away
          const float y = __shfl_xor(x[i][0], 32, 64);
          const float p = x[i][0] * cs[i].x, t = y * cs[i].y;
          x[i][0] = lane < 32 ? p - t : p + t;
        } else {
          const float u = x[i][0], w = x[i][1];
          x[i][0] = u * cs[i].x - w * cs[i].y;
          x[i][1] = w * cs[i].x + u * cs[i].y;
        }
      }
    }
    if (dst) {
#pragma unroll
      for (uint32_t i = 0; i < 8; i++)
        if (i < n) {
#pragma unroll
          for (int j = 0; j < kPer; j++)
            dst[(size_t)(row + i) * out_stride + head * D + 64 * j + lane] = from_f32<TO>(x[i][j]);
        }
    }
    if (page >= pool.pages) return;
    uint8_t* block = pool.block(page, head, at.head_bytes);
    const uint32_t slot = position & ((1u << pool.page_shift) - 1u), mine = lane & 7u;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      uint32_t kword = 0, vword = 0, my_scale = 0;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        uint32_t s;
        const uint32_t u = quantize(x[i][j], s);
        if ((lane & 31u) == i) my_scale = s;  // lane i of a group keeps row i's scale
        if (is_k) {
          const uint32_t w = or_of_8(u << (4 * mine));
          if (mine == i) kword = w;  // lane i of eight keeps row i's word
        } else if (i < n) {
          vword |= u << (4 * ((slot + i) & 7u));
        }
      }
      const uint32_t group = 2 * j + (lane >> 5);
      if (is_k) {
        if (mine < n)
          reinterpret_cast<uint32_t*>(block)[(slot + mine) * (D / 8) + ((lane >> 3) & 3u) * (D / 32) + group] = kword;
      } else {
        uint32_t* word = reinterpret_cast<uint32_t*>(block + at.v_codes) + (slot >> 3) * D + 64 * j + lane;
        if (n < 8) {
          const uint32_t mask = ((1u << (4 * n)) - 1u) << (4 * (slot & 7u));
          vword |= *word & ~mask;
        }
        *word = vword;
      }
      if ((lane & 31u) < n)
        reinterpret_cast<uint16_t*>(block + scales_at)
            [(group << pool.page_shift) + slot + (lane & 31u)] = (uint16_t)my_scale;
    }
  });
}

struct ReadArgs {
  const uint32_t *offsets, *starts;
  void *k_out, *v_out;
  uint32_t rows, span;
};

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    struct alignas(16) Eight {
      T v[8];
    };
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; i++) e.v[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Eight*>(p) = e;
  }
}
template <class T>
__device__ __forceinline__ void store2(T* p, float a, float b) {
  struct alignas(2 * sizeof(T)) Two {
    T v[2];
  };
  *reinterpret_cast<Two*>(p) = Two{{from_f32<T>(a), from_f32<T>(b)}};
}

// A wave per (span of packed rows, kv head's K or V), blocks of kBlock positions. K: a lane dequantizes
// words, 8 dims of a row each, stored in one. V: a lane has 2 dims (the wave 128: a block's 8 rows, or at
// head_dim 64 every other one). All of a block's words are read before any value is stored. 16 x 4096 rows of 8 heads
// of 128 (bf16) 74.0 us (4.65 TB/s) in blocks of 32, 88.6 of 16, 123.8 of 8. (Stored past the caches' retention they
// take 55.1, but the attention that reads the rows next pays for it: 512 queries each over them 570 us in all for 556,
// 500 each over 4 x 2000 rows of 2 heads of 64 39.3 for 34.3.) Of few kv heads blocks of 32 are few waves: 16384 rows of
// 2 heads of 64 are one block for each of two waves a SIMD, so one latency is the launch: 7.1 us for 11 MB.
template <int D, uint32_t kBlock, class TO>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a, Pool pool) {
  constexpr uint32_t kGroups = D / 32, kWords = D / 8;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t task = blockIdx.y * 4 + wave, kvh = pool.kv_heads;
  if (task >= 2 * kvh) return;
  const bool is_k = task < kvh;
  const uint32_t head = is_k ? task : task - kvh;
  TO* dst = static_cast<TO*>(is_k ? a.k_out : a.v_out);
  const Layout at = layout<D>(1u << pool.page_shift);
  const auto value = [](uint32_t word, uint32_t i, float s) { return (float)((int)((word >> (4 * i)) & 15u) - 8) * s; };
  for_blocks<kBlock>(a.offsets, a.starts, pool.sequences, a.rows, blockIdx.x * a.span, a.span,
                     [&](uint32_t seq, uint32_t row, uint32_t position, uint32_t n) {
    const uint32_t page = pool.page_of(seq, position);
    const bool have = page < pool.pages;
    const uint8_t* block = pool.block(have ? page : 0, head, at.head_bytes);
    const uint32_t slot = position & ((1u << pool.page_shift) - 1u);
    const uint16_t* scales = reinterpret_cast<const uint16_t*>(block + (is_k ? at.k_scales : at.v_scales));
    TO* out = dst + ((size_t)row * kvh + head) * D;
    if (is_k) {
      constexpr uint32_t kEach = kBlock * kWords / 64;
      uint32_t word[kEach];
      float s[kEach];
      const uint32_t w = lane % kWords, group = w / 4, part = w % 4;  // dims 8 w .. +8
#pragma unroll
      for (uint32_t j = 0; j < kEach; j++) {
        const uint32_t i = min((64 * j + lane) / kWords, n - 1);  // (rows past n: the last one, not stored)
        word[j] = reinterpret_cast<const uint32_t*>(block)[(slot + i) * kWords + part * kGroups + group];
        s[j] = egd::half_to_float(scales[(group << pool.page_shift) + slot + i]);
      }
#pragma unroll
      for (uint32_t j = 0; j < kEach; j++) {
        const uint32_t i = (64 * j + lane) / kWords;
        if (i >= n) continue;
        float v[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) v[e] = have ? value(word[j], e, s[j]) : 0.f;
        store8(out + (size_t)i * kvh * D + 8 * w, v);
      }
    } else {
      constexpr uint32_t kRows = 128 / D;  // rows at a time
      const uint32_t p = lane % (D / 2), first = slot >> 3;
      uint2 word[kBlock / 8];
      uint4 s[kBlock / 8];
#pragma unroll
      for (uint32_t j = 0; j < kBlock / 8; j++) {
        const uint32_t b = min(first + j, (slot + n - 1) >> 3);
        word[j] = reinterpret_cast<const uint2*>(block + at.v_codes)[b * (D / 2) + p];
        s[j] = *reinterpret_cast<const uint4*>(scales + ((p / 16) << pool.page_shift) + 8 * b);
      }
#pragma unroll
      for (uint32_t j = 0; j < kBlock / 8; j++)
#pragma unroll
        for (uint32_t e = 0; e < 8; e += kRows) {
          const uint32_t f = e + (D == 64 ? lane >> 5 : 0);  // position of the 8
          const uint32_t i = 8 * (first + j) + f - slot;     // row (before the first: past n)
          const uint32_t pair[4] = {s[j].x, s[j].y, s[j].z, s[j].w};
          const float scale = egd::half_to_float((uint16_t)(pair[e / 2] >> (16 * (f & 1u))));
          if (i < n)
            store2(out + (size_t)i * kvh * D + 2 * p, have ? value(word[j].x, f, scale) : 0.f,
                   have ? value(word[j].y, f, scale) : 0.f);
        }
    }
  });
}

// A part of a page per workgroup, kCopyWords 16-byte words a thread, all read before any is written, past the
// caches' retention. 2000 pages of 221,184 bytes: 167.2 us (5.29 TB/s; 175.4 with ordinary accesses; with 4
// words a thread 168.9 and with 8 172.2).
constexpr uint32_t kCopyWords = 2, kCopyBytes = kThreads * kCopyWords * 16;
__global__ __launch_bounds__(256) void copy_pages_kernel(uint8_t* pool, const uint32_t* pairs, uint32_t pages,
                                                         uint64_t stride, uint32_t parts) {
  const uint32_t pair = blockIdx.x / parts, part = blockIdx.x % parts;
  const uint32_t from = pairs[2 * (size_t)pair], to = pairs[2 * (size_t)pair + 1];
  if (from >= pages || to >= pages) return;
  const uint64_t begin = (uint64_t)part * kCopyBytes + 16u * threadIdx.x;
  const uint8_t* src = pool + from * stride;
  uint8_t* dst = pool + to * stride;
  egd::u32x4 v[kCopyWords];
#pragma unroll
  for (uint32_t i = 0; i < kCopyWords; i++) {  // (past the page: its last word again, not written)
    const uint64_t o = begin + 16u * kThreads * i;
    v[i] = __builtin_nontemporal_load(reinterpret_cast<const egd::u32x4*>(src + (o < stride ? o : stride - 16)));
  }
#pragma unroll
  for (uint32_t i = 0; i < kCopyWords; i++) {
    const uint64_t o = begin + 16u * kThreads * i;
    if (o < stride) __builtin_nontemporal_store(v[i], reinterpret_cast<egd::u32x4*>(dst + o));
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Where the rows are at most this many a wave has one row (a decode batch's rows are blocks of their own, and
// a wave would take them one after another) and a workgroup one row's queries; else a block.
constexpr uint32_t kFewRows = 2048;

// Rows of queries per workgroup of a long append: about two items of 8 elements a thread, what it reads
// ahead. 16384 rows of 14 heads of 64 (f32 to f16, with the read back) 29.1 us in 4s, 30.8 in 2s, 30.2 in 8s; 4000
// of 40 heads of 128 (bf16) 35.2 us in 1s, 38.7 in 4s.
uint32_t query_span(uint32_t rows, uint32_t width) {
  return rows <= kFewRows || width == 0 ? 1u : std::max(1u, std::min(8u, 4096u / width));
}

}  // namespace

// What a page's size follows from.
static int check_format(eg_context* ctx, const char* op, const eg_kv4_dims* d) {
  if (d->head_dim != 64 && d->head_dim != 128)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: head_dim %u is not supported (64, 128)", op, d->head_dim);
  if (d->page_size != 32 && d->page_size != 64 && d->page_size != 128 && d->page_size != 256)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: page_size %u is not supported (32, 64, 128, 256)", op, d->page_size);
  if (d->kv_heads == 0 || d->kv_heads > 1024)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: %u kv heads (1 to 1024)", op, d->kv_heads);
  return EG_OK;
}

int eg_kv4::check_dims(eg_context* ctx, const char* op, const eg_kv4_dims* d, const void* pool) {
  if (!d || !pool) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const int st = check_format(ctx, op, d);
  if (st != EG_OK) return st;
  if (d->pages == 0) return eg::fail(ctx, EG_ERR_INVALID, "%s: a pool of no pages", op);
  if (d->page_stride % 16 != 0 || d->page_stride < eg_kv4::page_bytes(*d))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: page_stride %llu is not a multiple of 16 of at least %llu bytes", op,
                    (unsigned long long)d->page_stride, (unsigned long long)eg_kv4::page_bytes(*d));
  if (!aligned(pool)) return eg::fail(ctx, EG_ERR_INVALID, "%s: the pool must be 16-byte aligned", op);
  if ((uint64_t)d->max_pages * d->page_size >= (1ull << 31))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u pages of %u positions per sequence (under 2^31 positions)", op,
                    d->max_pages, d->page_size);
  if (d->sequences > (1u << 20))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences (at most 2^20)", op, d->sequences);
  return EG_OK;
}

extern "C" {

int eg_kv4_page_bytes(const eg_kv4_dims* dims, uint64_t* out_bytes) {
  if (!dims || !out_bytes) return eg::fail(nullptr, EG_ERR_INVALID, "kv4_page_bytes: NULL argument");
  const int st = check_format(nullptr, "kv4_page_bytes", dims);
  if (st != EG_OK) return st;
  *out_bytes = eg_kv4::page_bytes(*dims);
  return EG_OK;
}

int eg_kv4_append(eg_context* ctx, const void* q, const void* k, const void* v, const float* rope,
                  const uint32_t* offsets, const uint32_t* starts, const uint32_t* table, void* pool, void* q_out,
                  void* k_out, void* v_out, const eg_kv4_dims* dims, const eg_kv4_append_dims* append) {
  const char* op = "kv4_append";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  const bool some = append && append->rows != 0 && dims->sequences != 0;
  if (!append || (some && (!k || !v || !offsets || !starts || !table)))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_kv4_append_dims& d = *append;
  if (!known_type(d.in_type) || !known_type(d.out_type))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: in_type %d, out_type %d (eg_element)", op, d.in_type, d.out_type);
  if (some && ((q == nullptr) != (q_out == nullptr) || (q == nullptr) != (d.heads == 0)))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q, q_out and heads go together", op);
  if (d.heads > 65535) return eg::fail(ctx, EG_ERR_RANGE, "%s: %u heads (at most 65535)", op, d.heads);
  const uint32_t width = dims->kv_heads * dims->head_dim, q_width = d.heads * dims->head_dim;
  AppendArgs a{q, k, v, reinterpret_cast<const float2*>(rope), offsets, starts, q_out, k_out, v_out, d.rows, d.heads,
               d.q_stride ? d.q_stride : q_width, d.k_stride ? d.k_stride : width,
               d.v_stride ? d.v_stride : width, d.rope_positions, d.rows <= kFewRows ? 1u : 8u, query_span(d.rows, q_width),
               (2 * dims->kv_heads + 3) / 4, 0};
  if (a.q_stride < q_width || a.k_stride < width || a.v_stride < width || (a.q_stride | a.k_stride | a.v_stride) % 4)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: row strides %u, %u, %u (multiples of 4, at least a row)", op, a.q_stride,
                    a.k_stride, a.v_stride);
  if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(rope) || !aligned(q_out) || !aligned(k_out) ||
      !aligned(v_out))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q, k, v, rope and the outputs must be 16-byte aligned", op);
  if (!some) return EG_OK;
  if (d.rows >= (1u << 30)) return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows (under 2^30)", op, d.rows);
  const eg_kv4::Pool p = eg_kv4::pool_of(*dims, pool, table);
  const uint64_t kv_blocks = (uint64_t)((d.rows + a.span - 1) / a.span) * a.kv_groups;
  const uint64_t blocks = kv_blocks + (d.heads ? (d.rows + a.q_span - 1) / a.q_span : 0);
  if (blocks >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows of %u kv heads over the grid limit", op, d.rows, dims->kv_heads);
  a.kv_blocks = (uint32_t)kv_blocks;
  const dim3 grid((uint32_t)blocks);
  const OnDevice on(ctx);
  with_type(d.in_type, [&](auto ti) {
    with_type(d.out_type, [&](auto to) {
      if (dims->head_dim == 64)
        hipLaunchKernelGGL((append_kernel<64, decltype(ti), decltype(to)>), grid, dim3(kThreads), 0, ctx->stream, a, p);
      else
        hipLaunchKernelGGL((append_kernel<128, decltype(ti), decltype(to)>), grid, dim3(kThreads), 0, ctx->stream, a, p);
    });
  });
  return eg::check_launch(ctx, op);
}

int eg_kv4_read(eg_context* ctx, const uint32_t* offsets, const uint32_t* starts, const uint32_t* table,
                const void* pool, void* k_out, void* v_out, uint32_t rows, int out_type, const eg_kv4_dims* dims) {
  const char* op = "kv4_read";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  const bool some = rows != 0 && dims->sequences != 0;
  if (some && (!offsets || !starts || !table || !k_out || !v_out))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  if (!known_type(out_type)) return eg::fail(ctx, EG_ERR_INVALID, "%s: out_type %d (eg_element)", op, out_type);
  if (!aligned(k_out) || !aligned(v_out))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: the outputs must be 16-byte aligned", op);
  if (!some) return EG_OK;
  if (rows >= (1u << 30)) return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows (under 2^30)", op, rows);
  const bool few = rows <= kFewRows;
  const ReadArgs a{offsets, starts, k_out, v_out, rows, few ? 1u : 32u};
  const eg_kv4::Pool p = eg_kv4::pool_of(*dims, pool, table);
  const dim3 grid((rows + a.span - 1) / a.span, (2 * dims->kv_heads + 3) / 4);
  if (grid.x >= (1u << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows over the grid limit", op, rows);
  const OnDevice on(ctx);
  with_type(out_type, [&](auto to) {
    using TO = decltype(to);
    const auto kernel = dims->head_dim == 64 ? (few ? read_kernel<64, 8, TO> : read_kernel<64, 32, TO>)
                                             : (few ? read_kernel<128, 8, TO> : read_kernel<128, 32, TO>);
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, ctx->stream, a, p);
  });
  return eg::check_launch(ctx, op);
}

int eg_kv4_copy_pages(eg_context* ctx, void* pool, const uint32_t* pairs, uint32_t count, const eg_kv4_dims* dims) {
  const char* op = "kv4_copy_pages";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  if (count == 0) return EG_OK;
  if (!pairs) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const uint64_t parts = (dims->page_stride + kCopyBytes - 1) / kCopyBytes;
  if (parts > ((1ull << 31) / kThreads - 1) / count)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u pages of %llu bytes over the grid limit", op, count,
                    (unsigned long long)dims->page_stride);
  const OnDevice on(ctx);
  hipLaunchKernelGGL(copy_pages_kernel, dim3((uint32_t)(parts * count)), dim3(kThreads), 0, ctx->stream,
                     static_cast<uint8_t*>(pool), pairs, dims->pages, dims->page_stride, (uint32_t)parts);
  return eg::check_launch(ctx, op);
}

}  // extern "C"

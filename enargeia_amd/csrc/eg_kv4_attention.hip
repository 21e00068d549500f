// Attention of one token per sequence over the paged 4-bit cache (eg_attention_decode_kv4).
//
//   out[s][h] = sum_j p_j V[j] / sum_j p_j,  p_j = exp(scale q[s][h] . K[j] - max_j),  j < lengths[s]
//
// One pass over the cache with the running max and sum of the softmax. A workgroup takes one kv head, up to
// 16 (8) of its query heads and one chunk of a sequence's positions; its four waves take the chunk's
// tiles in turn and meet in LDS at the end; chunks meet in a second launch.
//
// Both products run on v_mfma_f32_16x16x32_f16 in the transposed form S^T = K Q^T, O^T = V^T P^T:
// the accumulators of the first (a lane holds one head's scores of 8 positions) are the second's B
// operand where they lie. Row r = 4 g + e of key block n (of 2 in a tile of 32) is position 8 g +
// kOrder[4 n + e], so lane group g's eight scores are positions 8 g .. +8: one V code word of a dim is
// one lane's A operand, and one 16-byte read its positions' scales.
//
// K codes go into the first product as they are: four bits at the bottom of an f16 are a denormal,
// code * 2^-24 (2^-20 for the nibble above, whose queries are divided by 16), which the matrix cores
// multiply exactly. (For f32 rows as code - 8 in f16, 9 instructions per word: what the sum and its start
// at -8 times the queries leave of each other is off by 2e-6 of the result, these by 2e-7.) A group of
// 32 dims is one product's depth, so its accumulator, started at -8 times the sum of the queries, is
// sum q (code - 8), and the scale is applied to it: 5 vector instructions per word of 8 codes. V's scale
// differs along the second product's depth, so V is dequantized: (1024 + code) - 1032 in f16, times the
// scale - exact by the format - 13 instructions per word.
//
// Queries are scaled by a power of two that puts a head's largest into [2^14, 2^15), weights by 2^15:
// an f16 and the f16 of what it leaves (kParts 2, for f32 rows) then hold 22 bits of them.
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
using egd::u32x4;

constexpr uint32_t kThreads = 256, kWaves = 4;
constexpr uint64_t kInfinityCache = 256u << 20;  // bytes
constexpr float kLargest = 0x1p20f;
constexpr float kLog2e = 1.44269504088896340736f;
// slot of an 8-deep operand -> nibble of a word, as the two masks below deliver them
constexpr uint32_t kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};

struct Args {
  const void* q;
  const uint32_t* lengths;
  void* out;
  float* o;   // partials [sequence][head][split][D], unnormalised; NULL without a split
  float* ml;  // [sequence][head][split] (max, sum)
  uint32_t heads, group, head_tiles, q_stride, out_stride, splits, min_chunk, capacity;
  float scale;  // times log2 e
};

// Positions per chunk: the same in the attention and the launch that joins its partials.
__device__ __forceinline__ uint32_t chunk_of(const Args& a, uint32_t length) {
  const uint32_t even = (length + a.splits - 1) / a.splits;
  return max(a.min_chunk, (even + 63u) & ~63u);
}

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

// D: head_dim. T: key tiles of 32 per step. At T = 2 a lane's column (lane % 16) is head lane % 8 of
// tile lane / 8 % 2: each tile's product has zeros in the other's columns, both add into the same
// accumulators, and the softmax of two tiles costs one's instructions - for groups of up to 8 heads, where half
// of the columns would be empty. T = 1: 16 heads. kParts: f16 parts of a query and of a weight.
// (Two waves per SIMD: their registers hold two steps' operands each, one step's loads under way while
// the other is multiplied.)
// kStream: codes are read past the caches' retention (non-temporal), where the call's reach is larger than the
// Infinity Cache: 32 sequences of 16384 (32 / 8 heads of 128) 94.4 us for 106.5, but 16 of up to 8192 26.0 for
// 24.6 (calls on one layer that follow each other: what lies in the caches is from the call before).
template <int D, int T, int kParts, bool kStream, class TQ>
__global__ __launch_bounds__(256, 2) void decode_kernel(Args a, Pool pool) {
  constexpr int kGroups = D / 32, kBlocks = D / 16;  // dim groups of K; blocks of 16 dims of O^T
  constexpr bool kSigned = kParts == 2;
  constexpr int kAux = kStream ? egd::kNonTemporal : 0;
  constexpr uint32_t kTile = 32 * T, kHeads = 16 / T;
  constexpr int kVWords = D / 16;  // V words of a lane: its dims D / 16 * (lane % 16) + 0 ..
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lr = lane & 15u, lg = lane >> 4;
  const uint32_t col = lr % kHeads, half = T == 2 ? lr >> 3 : 0;

  uint32_t id = blockIdx.x;
  const uint32_t split = id % a.splits;
  id /= a.splits;
  const uint32_t ht = id % a.head_tiles;
  id /= a.head_tiles;
  const uint32_t kv = id % pool.kv_heads, seq = id / pool.kv_heads;

  const uint32_t length = min(a.lengths[seq], a.capacity), chunk = chunk_of(a, length);
  const uint32_t begin = split * chunk, end = min(length, begin + chunk);
  if (split != 0 && begin >= length) return;
  const uint32_t heads = min(kHeads, a.group - ht * kHeads), head0 = kv * a.group + ht * kHeads;
  const Magic bits_over = magic();

  const uint32_t page_size = 1u << pool.page_shift;
  const Layout at = layout<D>(page_size);
  const uint32_t k_off = (8 * (lr >> 2) + kOrder[0]) * (D / 2) + lg * (kGroups * 4);
  const uint32_t e_off = lr & 3u;  // row e of a lane's K operand: positions kOrder[e] and kOrder[4 + e]
  const uint32_t k_row0 = k_off + (e_off == 0 ? 0u : e_off == 1 ? 4u : e_off == 2 ? 1u : 5u) * (D / 2);
  const uint32_t v_off = at.v_codes + (lg * D + lr * kVWords) * 4;
  const uint32_t ks_off = at.k_scales + (32 * half + 8 * lg) * 2;
  const uint32_t vs_off = at.v_scales + (((lr * kVWords) / 32) << (pool.page_shift + 1)) + 16 * lg;

  // A step's operands as they come from memory.
  struct Tile {
    uint32_t k[T][2][kGroups];
    uint32_t v[T][kVWords];
    u32x4 ks[kGroups], vs[T];
    bool have;
  };
  const auto load = [&](Tile& t, uint32_t page, uint32_t slot) {
    t.have = page < pool.pages;
    // (no page: a resource of no bytes, whose loads return zeros)
    const auto r = egd::buffer(pool.block(t.have ? page : 0, kv, at.head_bytes), t.have ? at.head_bytes : 0);
#pragma unroll
    for (int i = 0; i < T; i++) {
      const uint32_t s = slot + 32 * i;
#pragma unroll
      for (int n = 0; n < 2; n++) {  // positions 2 apart: kOrder[4 + e] = kOrder[e] + 2
        const uint32_t o = k_row0 + 2 * n * (D / 2);
        if constexpr (kGroups == 2) {
          const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, o, s * (D / 2), kAux);
          t.k[i][n][0] = w[0];
          t.k[i][n][1] = w[1];
        } else {
          const u32x4 w = egd::load_b128_p<kAux>(r, o, s * (D / 2));
#pragma unroll
          for (int g = 0; g < kGroups; g++) t.k[i][n][g] = w[g];
        }
      }
#pragma unroll
      for (int j = 0; j < kVWords; j += 4) {
        const u32x4 w = egd::load_b128_p<kAux>(r, v_off + 4 * j, (s / 8) * (D * 4));
#pragma unroll
        for (int e = 0; e < 4; e++) t.v[i][j + e] = w[e];
      }
      t.vs[i] = egd::load_b128(r, vs_off, s * 2);
    }
#pragma unroll
    for (int g = 0; g < kGroups; g++) t.ks[g] = egd::load_b128(r, ks_off, ((g << pool.page_shift) + slot) * 2);
  };

  const uint32_t steps = begin < end ? (end - begin + kTile - 1) / kTile : 0;
  const uint32_t mine = steps > wave ? (steps - wave + kWaves - 1) / kWaves : 0;  // steps of this wave
  // The pages of this wave's next 64 steps, one a lane, from its step i0 on.
  const auto pages_of = [&](uint32_t i0) {
    const uint32_t step = wave + kWaves * (i0 + lane);
    return step < steps ? pool.page_of(seq, begin + step * kTile) : 0xFFFFFFFFu;
  };
  const auto fetch = [&](Tile& t, uint32_t ids, uint32_t i0, uint32_t i) {
    load(t, (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)i),
         (begin + (wave + kWaves * (i0 + i)) * kTile) & (page_size - 1u));
  };
  uint32_t ids = pages_of(0);

  // The queries, B operand: lane group g has dims 32 grp + 8 g + kOrder[slot] of head `col`.
  half8 qf[T][kGroups][kParts];
  f32x4 start[kGroups];  // -8 sum q per group: what makes codes of code - 8
  float f;
  {
    float x[kGroups][8], top = 0.f;
    const bool in = col < heads;
    const TQ* src = static_cast<const TQ*>(a.q) + (size_t)seq * a.q_stride + (size_t)(head0 + (in ? col : 0)) * D;
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
      struct alignas(16) Eight {
        TQ v[8];
      };
      const Eight e = *reinterpret_cast<const Eight*>(src + 32 * g + 8 * lg);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[g][i] = in ? to_f32(e.v[kOrder[i]]) : 0.f;
        top = fmaxf(top, fabsf(x[g][i]));
      }
    }
    top = max_of_head(top);
    int e = top > 0.f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
    e = max(-100, min(110, e));
    f = fmaxf(ldexpf(a.scale, kSigned ? -e : 24 - e), 0x1p-126f);  // (not 0: -inf times it is -inf)
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
      half8 part[kParts];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float y = ldexpf(x[g][i], e);
#pragma unroll
        for (int p = 0; p < kParts; p++) {
          const _Float16 h = (_Float16)y;
          y -= (float)h;
          part[p][i] = !kSigned && (i & 2) ? h * (_Float16)0.0625f : h;
        }
      }
      const half8 eight = as_half8(0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u);
      start[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < kParts; p++) {
        if constexpr (!kSigned) start[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight, part[p], start[g], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < T; i++)
          qf[i][g][p] = T == 1 || half == (uint32_t)i ? part[p] : half8{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
  }

  f32x4 o[kBlocks];
#pragma unroll
  for (int n = 0; n < kBlocks; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // running max of the scores before f; this lane's share of the sum

  const auto compute = [&](Tile& t, uint32_t i) {
    const uint32_t j0 = begin + (wave + kWaves * i) * kTile;
    f32x4 s[2];
#pragma unroll
    for (int n = 0; n < 2; n++) {
      s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        f32x4 acc = start[g];
#pragma unroll
        for (int b = 0; b < T; b++) {
          const half8 kc = codes<kSigned>(t.k[b][n][g], bits_over);
#pragma unroll
          for (int p = 0; p < kParts; p++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qf[b][g][p], acc, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] = fmaf(half_of(t.ks[g], kOrder[4 * n + e]), acc[e], s[n][e]);
      }
    }
    if (j0 + kTile > end || !t.have) {  // positions past the end: no score, values of zero
      const int seen = t.have ? (int)end - (int)(j0 + 32 * half + 8 * lg) : 0;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if ((int)kOrder[4 * n + e] >= seen) s[n][e] = -INFINITY;
#pragma unroll
      for (int b = 0; b < T; b++) t.vs[b] = first_halves(t.vs[b], t.have ? (int)end - (int)(j0 + 32 * b + 8 * lg) : 0);
    }
    float top = m;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) top = fmaxf(top, s[n][e]);
    top = max_of_head(top);
    float shift = top == -INFINITY ? 0.f : fmaf(top, f, -15.f);
    // (past kLargest the max's own rounding would put weights out of f16's range: there it is taken from the
    // scores instead, which leaves the largest exactly 0)
    if (__builtin_amdgcn_ballot_w64(fabsf(shift) > kLargest) != 0) {
      const float from = top == -INFINITY ? 0.f : top;  // (a half without a position yet)
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] -= from;
      shift = -15.f;
    }
    if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
      const float alpha = top > m ? __builtin_amdgcn_exp2f((m - top) * f) : 1.f;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < kBlocks; n++) o[n] *= alpha;
      m = top;
    }
    half8 pb[kParts];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float p = __builtin_amdgcn_exp2f(fmaf(s[n][e], f, -shift));
        l += p;
#pragma unroll
        for (int k = 0; k < kParts; k++) {
          const _Float16 h = (_Float16)p;
          pb[k][4 * n + e] = h;
          p -= (float)h;
        }
      }
#pragma unroll
    for (int b = 0; b < T; b++) {
      half2v pairs[4];
      scale_pairs(t.vs[b], pairs);
      half8 w[kParts];
#pragma unroll
      for (int k = 0; k < kParts; k++)
        w[k] = T == 1 || half == (uint32_t)b ? pb[k] : half8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < kBlocks; n++) {
        const half8 va = values(t.v[b][n], pairs, bits_over);
#pragma unroll
        for (int k = 0; k < kParts; k++) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, w[k], o[n], 0, 0, 0);
      }
    }
  };

  // (The page ids are read outside the loop over their 64 steps: a wait for them inside would be a wait
  // for the tiles under way.)
  for (uint32_t i0 = 0; i0 < mine; i0 += 64) {
    if (i0) ids = pages_of(i0);
    const uint32_t n = min(64u, mine - i0);
    Tile tiles[2];
    fetch(tiles[0], ids, i0, 0);
    for (uint32_t i = 0; i < n; i += 2) {
      if (i + 1 < n) fetch(tiles[1], ids, i0, i + 1);
      compute(tiles[0], i0 + i);
      if (i + 1 < n) {
        if (i + 2 < n) fetch(tiles[0], ids, i0, i + 2);
        compute(tiles[1], i0 + i + 1);
      }
    }
  }

  // The waves (and at T = 2 each wave's two halves) meet in LDS.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __shared__ float top_of[kWaves * T][kHeads], sum_of[kWaves * T][kHeads];
  __shared__ __attribute__((aligned(16))) float part_of[kWaves * T][kHeads][D];
  const uint32_t source = wave * T + half;
  if (lg == 0) {
    top_of[source][col] = m == -INFINITY ? -INFINITY : m * f;
    sum_of[source][col] = l;
  }
  // row 4 lg + e of block n is dim D / 16 (4 lg + e) + n
#pragma unroll
  for (int e = 0; e < 4; e++)
#pragma unroll
    for (int n = 0; n < kBlocks; n += 4)
      *reinterpret_cast<float4*>(&part_of[source][col][kBlocks * (4 * lg + e) + n]) =
          make_float4(o[n][e], o[n + 1][e], o[n + 2][e], o[n + 3][e]);
  __syncthreads();
  const bool whole = chunk >= length;  // no other chunk: the result itself
  for (uint32_t i = tid; i < heads * (D / 4); i += kThreads) {
    const uint32_t h = i / (D / 4), d = 4 * (i % (D / 4));
    float top = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < kWaves * T; w++) top = fmaxf(top, top_of[w][h]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves * T; w++) {
      const float c = top_of[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top_of[w][h] - top);
      const float4 v = *reinterpret_cast<const float4*>(&part_of[w][h][d]);
      sum = fmaf(c, sum_of[w][h], sum);
      acc = make_float4(fmaf(c, v.x, acc.x), fmaf(c, v.y, acc.y), fmaf(c, v.z, acc.z), fmaf(c, v.w, acc.w));
    }
    const size_t row = (size_t)seq * a.heads + head0 + h;
    if (whole) {
      const float r = sum == 0.f ? 0.f : 1.f / sum;
      TQ* to = static_cast<TQ*>(a.out) + (size_t)seq * a.out_stride + (size_t)(head0 + h) * D + d;
      to[0] = from_f32<TQ>(acc.x * r);
      to[1] = from_f32<TQ>(acc.y * r);
      to[2] = from_f32<TQ>(acc.z * r);
      to[3] = from_f32<TQ>(acc.w * r);
    } else {
      *reinterpret_cast<float4*>(a.o + (row * a.splits + split) * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.ml + 2 * (row * a.splits + split)) = make_float2(top, sum);
    }
  }
}

// A sequence's chunks joined: a workgroup per (sequence, head), its waves taking the chunks in turn.
template <int D, class TQ>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  constexpr uint32_t kPer = D / 64;
  const uint32_t head = blockIdx.x % a.heads, seq = blockIdx.x / a.heads, tid = threadIdx.x;
  const uint32_t lane = tid & 63u, wave = tid >> 6;
  const uint32_t length = min(a.lengths[seq], a.capacity), chunk = chunk_of(a, length);
  if (chunk >= length) return;  // one chunk: it wrote the result
  const uint32_t count = (length + chunk - 1) / chunk;
  const size_t row = ((size_t)seq * a.heads + head) * a.splits;
  const float* ml = a.ml + 2 * row;
  float top = -INFINITY;
  for (uint32_t c = lane; c < count; c += 64) top = fmaxf(top, ml[2 * c]);
  top = egd::team_allmax<64>(top);
  float acc[kPer] = {}, sum = 0.f;
#pragma unroll 4
  for (uint32_t c = wave; c < count; c += kWaves) {
    const float w = ml[2 * c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[2 * c] - top);
    sum = fmaf(w, ml[2 * c + 1], sum);
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) acc[j] = fmaf(w, a.o[(row + c) * D + 64 * j + lane], acc[j]);
  }
  __shared__ float part[kWaves][D], sums[kWaves];
#pragma unroll
  for (uint32_t j = 0; j < kPer; j++) part[wave][64 * j + lane] = acc[j];
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (tid < D) {
    const float total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const float v = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    static_cast<TQ*>(a.out)[(size_t)seq * a.out_stride + (size_t)head * D + tid] =
        from_f32<TQ>(total == 0.f ? 0.f : v / total);
  }
}

template <int D, int T, class TQ>
void launch(eg_context* ctx, const Args& a, const Pool& p, bool stream, uint64_t blocks) {
  constexpr int kParts = std::is_same<TQ, float>::value ? 2 : 1;
  const dim3 grid((uint32_t)blocks), threads(kThreads);
  if (stream) hipLaunchKernelGGL((decode_kernel<D, T, kParts, true, TQ>), grid, threads, 0, ctx->stream, a, p);
  else hipLaunchKernelGGL((decode_kernel<D, T, kParts, false, TQ>), grid, threads, 0, ctx->stream, a, p);
  if (a.splits > 1)
    hipLaunchKernelGGL((join_kernel<D, TQ>), dim3(p.sequences * a.heads), threads, 0, ctx->stream, a);
}

}  // namespace

extern "C" int eg_attention_decode_kv4(eg_context* ctx, const void* q, const uint32_t* lengths, const uint32_t* table,
                                       const void* pool, void* out, const eg_kv4_dims* dims,
                                       const eg_attention_kv4_dims* attention) {
  const char* op = "attention_decode_kv4";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  if (!attention || (dims->sequences != 0 && (!q || !lengths || !out || (dims->max_pages != 0 && !table))))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_attention_kv4_dims& d = *attention;
  if (!known_type(d.type)) return eg::fail(ctx, EG_ERR_INVALID, "%s: type %d (eg_element)", op, d.type);
  if (d.heads == 0 || d.heads % dims->kv_heads != 0 || d.heads > 65535)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: heads %u are not a multiple of kv_heads %u (at most 65535)", op, d.heads,
                    dims->kv_heads);
  if (!(d.scale >= 0.f) || d.scale > 1e6f) return eg::fail(ctx, EG_ERR_INVALID, "%s: scale %g (0 to 1e6)", op, d.scale);
  const uint32_t width = d.heads * dims->head_dim;
  Args a{};
  a.q = q;
  a.lengths = lengths;
  a.out = out;
  a.heads = d.heads;
  a.group = d.heads / dims->kv_heads;
  a.q_stride = d.q_stride ? d.q_stride : width;
  a.out_stride = d.out_stride ? d.out_stride : width;
  if (a.q_stride < width || a.out_stride < width || (a.q_stride | a.out_stride) % 8)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: strides %u, %u (multiples of 8, at least a row)", op, a.q_stride,
                    a.out_stride);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q and out must be 16-byte aligned", op);
  if (dims->sequences == 0) return EG_OK;
  a.scale = (d.scale > 0.f ? d.scale : 1.0f / sqrtf((float)dims->head_dim)) * kLog2e;
  a.capacity = dims->max_pages * dims->page_size;
  // Two key tiles a step where the heads leave room for them (and a step's 64 positions lie in one page).
  const bool pair = a.group <= 8 && dims->page_size >= 64;
  a.head_tiles = pair ? 1 : (a.group + 15) / 16;
  // Splits, none for tables that reach 1024: chunks of at least two steps a wave. A workgroup's first loads wait for
  // each other (length, page, rows) and the join is a launch, so shorter chunks cost more than they balance: 48
  // sequences of 2048 (14 / 2 heads of 64) 11.1 us in chunks of 512, 13.9 in 1024, 13.1 in 256; 5 of 4000 (32 / 2 of 64,
  // f16) 9.2 in 256, 9.9 in 512, 11.6 in 1024; 1 of 517 6.5 whole, 9.0 in two. Workgroups: two a CU, as the device
  // holds at once (16 of up to 8192, 28 / 4 of 128, f32: 24.6 us, in twice as many 29.7), but of T = 1's one where the
  // tables do not reach 1024 positions for each of two (4 of 65536, 16 / 1 of 128: 19.5 us, in a few more 21.8).
  // All of this goes by counts, the lengths being on the device: with more (sequence, kv head) rows than CUs nothing
  // is split, and a sequence far longer than the others holds the launch up (one of 65536 beside 63 of 512, 32 / 8 of
  // 128, bf16: 340 us, alone 24; 64 of 512: 12.5).
  a.min_chunk = pair ? 512 : 256;
  const uint64_t rows = (uint64_t)dims->sequences * dims->kv_heads * a.head_tiles, twice = 2ull * ctx->cu_count / rows;
  const uint64_t room = pair || a.capacity >= 1024 * twice ? twice : ctx->cu_count / rows;
  const uint64_t most = (a.capacity + a.min_chunk - 1) / a.min_chunk;
  uint64_t splits = a.capacity <= 1024 ? 1 : std::max<uint64_t>(1, std::min(room, most));
  const uint64_t per_split = (uint64_t)dims->sequences * d.heads * (dims->head_dim + 2) * 4;
  splits = std::max<uint64_t>(1, std::min<uint64_t>(splits, (eg::kPartialsBytes - 64) / per_split));
  a.splits = (uint32_t)splits;
  if (rows * splits >= (1ull << 31) / kThreads || (uint64_t)dims->sequences * d.heads >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences of %u heads over the grid limit", op, dims->sequences, d.heads);
  a.ml = reinterpret_cast<float*>(eg::partials(ctx));
  a.o = a.ml + (((size_t)dims->sequences * d.heads * splits * 2 + 3) & ~(size_t)3);
  const Pool p = eg_kv4::pool_of(*dims, pool, table);
  // The most that the call can read: what the tables reach, and what the pool holds, of its one layer. (The other
  // layers of a step are not counted, though they too pass through the caches before this one is read again.)
  const uint64_t reach = std::min<uint64_t>((uint64_t)dims->sequences * dims->max_pages, dims->pages) * eg_kv4::page_bytes(*dims);
  const bool stream = reach > kInfinityCache;
  const OnDevice on(ctx);
  with_type(d.type, [&](auto t) {
    using TQ = decltype(t);
    const uint64_t blocks = rows * splits;
    if (dims->head_dim == 64)
      pair ? launch<64, 2, TQ>(ctx, a, p, stream, blocks) : launch<64, 1, TQ>(ctx, a, p, stream, blocks);
    else
      pair ? launch<128, 2, TQ>(ctx, a, p, stream, blocks) : launch<128, 1, TQ>(ctx, a, p, stream, blocks);
  });
  return eg::check_launch(ctx, op);
}

// Attention of a tree of drafted rows per sequence over the paged 4-bit cache (eg_attention_tree_kv4).
//
//   out[r][h] = sum_j p_j V[j] / sum_j p_j,  p_j = exp(scale q[r][h] . K[j] - max_j),  j of those that row r sees
//
// The decode attention (eg_kv4_attention.hip) with more columns: a kv head's columns are all its query heads of all
// the sequence's rows, in blocks of 16, and a tile of positions serves as many of them as there are. One pass over the
// cache with the running max and sum of the softmax; chunks of a sequence's positions meet in a second launch. Which of
// the last positions a column sees is its row's ancestors, as 64 bits; tiles before them have no mask. Two kernels: few
// columns bind by what a wave waits for and unpacks, many by issue (products and vector instructions hardly overlap).
//
// Maxima, sums and results are f32. A weight enters the second product as f16: f32 rows' in two parts, 22 bits; 16-bit rows' in one, 11
// bits, while the sum that divides has all of them. Results of 16-bit rows are then off, relative to their norm, by 2.5e-4 to 2.9e-4 in
// f16, whose own rounding is 2.1e-4, and by 1.67e-3 in bf16 for 1.66e-3; two parts take 126 us where one takes 80 (8 sequences of 64 rows
// at up to 8192, 32 / 8 heads of 128, f32 and bf16).
#include <algorithm>

#include "eg_kv4_operands.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256, kMostRows = 64;

struct Args {
  const void* q;
  const uint32_t *offsets, *parents, *lengths;
  void* out;
  float* o;   // partials [row][head][split][D], unnormalised
  float* ml;  // [row][head][split] (max, sum)
  uint32_t rows, max_rows, heads, group, tiles, q_stride, out_stride, splits, min_chunk, capacity;
  float scale;  // times log2 e
};

// Positions per chunk: the same in the attention and the launch that joins its partials.
__device__ __forceinline__ uint32_t chunk_of(const Args& a, uint32_t length) {
  const uint32_t even = (length + a.splits - 1) / a.splits;
  return max(a.min_chunk, (even + 63u) & ~63u);
}

// Whether a sequence's rows, packed rows first .. last, are computed.
__device__ __forceinline__ bool computed(const Args& a, uint32_t first, uint32_t last) {
  return first <= last && last <= a.rows && last - first <= a.max_rows;
}

// What a row of a sequence sees of its rows, itself among them: lane i of a wave, with row i's parent, gets row i's bits. Each turn
// adds what the row at the end of the chain so far has, and moves that end to its own: 6 turns reach 64.
__device__ __forceinline__ uint64_t ancestors(bool tree, uint32_t parent) {
  const uint32_t lane = threadIdx.x & 63u;
  if (!tree) return ~0ull >> (63u - lane);
  uint32_t end = parent < lane ? parent : lane;
  uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
  for (int i = 0; i < 6; i++) {
    lo |= (uint32_t)__shfl((int)lo, (int)end, 64);
    hi |= (uint32_t)__shfl((int)hi, (int)end, 64);
    end = (uint32_t)__shfl((int)end, (int)end, 64);
  }
  return (uint64_t)hi << 32 | lo;
}

// Those bits of a row.
__device__ __forceinline__ uint64_t of_row(uint64_t all, uint32_t row) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)(all >> 32), (int)row, 64) << 32 |
         (uint32_t)__shfl((int)(uint32_t)all, (int)row, 64);
}

// A column's query as it comes from memory: lane group g has dims 32 grp + 8 g .. +8.
template <class TQ>
struct alignas(16) Eight {
  TQ v[8];
};
template <int D, class TQ>
__device__ __forceinline__ void load_query(const Args& a, uint32_t row, uint32_t head, uint32_t lg, Eight<TQ> (&raw)[D / 32]) {
  const TQ* src = static_cast<const TQ*>(a.q) + (size_t)row * a.q_stride + (size_t)head * D;
#pragma unroll
  for (int g = 0; g < D / 32; g++) raw[g] = *reinterpret_cast<const Eight<TQ>*>(src + 32 * g + 8 * lg);
}

// And as the first product's B operand: slots in kOrder's order, times the power of two that puts the largest of the
// column's into [2^14, 2^15), whose exponent is returned.
template <int D, int kParts, class TQ>
__device__ __forceinline__ int make_query(const Eight<TQ> (&raw)[D / 32], bool in, half8 (&qf)[D / 32][kParts]) {
  float x[D / 32][8], top = 0.f;
#pragma unroll
  for (int g = 0; g < D / 32; g++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[g][i] = in ? to_f32(raw[g].v[kOrder[i]]) : 0.f;
      top = fmaxf(top, fabsf(x[g][i]));
    }
  top = max_of_head(top);
  const int up = max(-100, min(110, top > 0.f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0));
#pragma unroll
  for (int g = 0; g < D / 32; g++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float y = ldexpf(x[g][i], up);
#pragma unroll
      for (int p = 0; p < kParts; p++) {
        const _Float16 h = (_Float16)y;
        y -= (float)h;
        qf[g][p][i] = h;
      }
    }
  return up;
}

// Few columns: 16 a workgroup, whose waves take a chunk's tiles of 32 positions in turn and meet in LDS. D: head_dim. kWaves: 4, or
// 8 where a CU has one workgroup, so that one wave's work is beside another's waits (16 sequences of 16 rows at up to 2048, 14 / 2
// heads of 64: f32 15.3 us for 17.5, bf16 13.4 for 16.0; 1 of 5 rows at 517 7.3 for 7.4). kParts: f16 parts of a query and of a
// weight (2 for f32 rows). (With two blocks of columns a wave, 32 / 8 heads of 128 in
// bf16: 16 sequences of up to 2048 with 8 rows 35.1 us for 22.9, 32 of up to 4096 62.3 for 54.8: half as many workgroups,
// and no registers left for the next tile's words.)
template <int D, int kWaves, int kParts, class TQ>
__global__ __launch_bounds__(64 * kWaves, 2) void few_kernel(Args a, Pool pool) {
  constexpr int kGroups = D / 32, kDims = D / 16;  // dim groups of K; blocks of 16 dims of O^T
  constexpr bool kSigned = kParts == 2;
  constexpr uint32_t kTile = 32, kColumns = 16;
  constexpr int kVWords = D / 16;  // V words of a lane: its dims D / 16 * (lane % 16) + 0 ..
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lr = lane & 15u, lg = lane >> 4;

  uint32_t id = blockIdx.x;
  const uint32_t split = id % a.splits;
  id /= a.splits;
  const uint32_t tile = id % a.tiles;
  id /= a.tiles;
  const uint32_t kv = id % pool.kv_heads, seq = id / pool.kv_heads;

  const uint32_t first = a.offsets[seq], last = a.offsets[seq + 1], n = last - first, length = a.lengths[seq];
  const uint32_t reach = min(length, a.capacity), chunk = chunk_of(a, reach), begin = split * chunk;
  if (!computed(a, first, last) | (tile * kColumns >= n * a.group) | ((split != 0) & (begin >= reach))) return;  // (read at once)
  const bool fits = n <= length;  // (else the rows give zeros)
  const uint32_t base = fits ? length - n : 0, end = fits ? min(reach, begin + chunk) : 0;
  const Magic bits_over = magic();

  // This lane's column.
  const uint32_t c0 = tile * kColumns, column = c0 + lr;
  const bool in = column < n * a.group;
  const uint32_t row = in ? column / a.group : 0, head = kv * a.group + (in ? column % a.group : 0);

  const uint32_t page_size = 1u << pool.page_shift;
  const Layout at = layout<D>(page_size);
  const uint32_t e_off = lr & 3u;  // row e of a lane's K operand: positions kOrder[e] and kOrder[4 + e]
  const uint32_t k_row0 = (8 * (lr >> 2) + (e_off == 0 ? 0u : e_off == 1 ? 4u : e_off == 2 ? 1u : 5u)) * (D / 2) +
                          lg * (kGroups * 4);
  const uint32_t v_off = at.v_codes + (lg * D + lr * kVWords) * 4;
  const uint32_t ks_off = at.k_scales + 8 * lg * 2;
  const uint32_t vs_off = at.v_scales + (((lr * kVWords) / 32) << (pool.page_shift + 1)) + 16 * lg;

  // A step's operands as they come from memory.
  struct Tile {
    uint32_t k[2][kGroups];
    uint32_t v[kVWords];
    u32x4 ks[kGroups], vs;
    bool have;
  };
  const auto load = [&](Tile& t, uint32_t page, uint32_t slot) {
    t.have = page < pool.pages;
    // (no page: a resource of no bytes, whose loads return zeros)
    const auto r = egd::buffer(pool.block(t.have ? page : 0, kv, at.head_bytes), t.have ? at.head_bytes : 0);
#pragma unroll
    for (int m = 0; m < 2; m++) {  // positions 2 apart: kOrder[4 + e] = kOrder[e] + 2
      const uint32_t o = k_row0 + 2 * m * (D / 2);
      if constexpr (kGroups == 2) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, o, slot * (D / 2), 0);
        t.k[m][0] = w[0];
        t.k[m][1] = w[1];
      } else {
        const u32x4 w = egd::load_b128(r, o, slot * (D / 2));
#pragma unroll
        for (int g = 0; g < kGroups; g++) t.k[m][g] = w[g];
      }
    }
#pragma unroll
    for (int j = 0; j < kVWords; j += 4) {
      const u32x4 w = egd::load_b128(r, v_off + 4 * j, (slot / 8) * (D * 4));
#pragma unroll
      for (int e = 0; e < 4; e++) t.v[j + e] = w[e];
    }
    t.vs = egd::load_b128(r, vs_off, slot * 2);
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
  // Reads that wait for nothing but offsets and lengths first, then the first tile's; the rest goes on beside those.
  uint32_t ids = pages_of(0);
  const bool tail = end > base;
  const uint32_t parent = tail && a.parents && lane < n ? a.parents[first + lane] : 0xFFFFFFFFu;
  Eight<TQ> raw[kGroups];
  load_query<D, TQ>(a, first + row, head, lg, raw);
  Tile tiles[2];
  if (mine != 0) fetch(tiles[0], ids, 0, 0);
  const uint64_t sees = tail ? of_row(ancestors(a.parents != nullptr, parent), row) : 0;

  half8 qf[kGroups][kParts];
  f32x4 start[kGroups];  // -8 sum q per group: what makes codes of code - 8
  const int up = make_query<D, kParts, TQ>(raw, in, qf);
  const float f = fmaxf(ldexpf(a.scale, kSigned ? -up : 24 - up), 0x1p-126f);  // (not 0: -inf times it is -inf)
#pragma unroll
  for (int g = 0; g < kGroups; g++) {
    start[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (!kSigned) {
      const half8 eight = as_half8(0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u);
#pragma unroll
      for (int p = 0; p < kParts; p++) {
#pragma unroll
        for (int i = 2; i < 8; i++)
          if (i & 2) qf[g][p][i] *= (_Float16)0.0625f;
        start[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight, qf[g][p], start[g], 0, 0, 0);
      }
    }
  }

  f32x4 o[kDims];
#pragma unroll
  for (int i = 0; i < kDims; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // running max of the scores before f; this lane's share of the sum

  const auto compute = [&](Tile& t, uint32_t i) {
    const uint32_t j0 = begin + (wave + kWaves * i) * kTile;
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        const half8 kc = codes<kSigned>(t.k[k][g], bits_over);
        f32x4 acc = start[g];
#pragma unroll
        for (int p = 0; p < kParts; p++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qf[g][p], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++) s[k][e] = fmaf(half_of(t.ks[g], kOrder[4 * k + e]), acc[e], s[k][e]);
      }
    bool poison = false;  // the column sees a value that is not a number
    if (j0 + kTile > base || !t.have) {
      // positions past the end: no score, values of zero; of the sequence's rows what the column sees
      const int seen = t.have ? (int)(end - j0) : 0;  // of the tile
      t.vs = first_halves(t.vs, max(0, min(8, seen - (int)(8 * lg))));
      uint32_t visible = 0xFFFFFFFFu;  // of the tile's 32 positions
      if (j0 >= base) visible = (uint32_t)(sees >> (j0 - base));
      else if (base - j0 < 32) visible = (uint32_t)(sees << (base - j0)) | ((1u << (base - j0)) - 1u);
      if (seen < 32) visible &= seen <= 0 ? 0u : (1u << seen) - 1u;
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (!(visible >> (8 * lg + kOrder[4 * k + e]) & 1u)) s[k][e] = -INFINITY;
      // A scale that is not a number (its values are none then) would reach, times a weight of 0, the columns that do
      // not see its position: it is taken out of the product, and put into the sums of those that do.
      uint32_t bad = 0;  // of this lane's 8 positions
#pragma unroll
      for (int h = 0; h < 8; h++) {
        const uint32_t x = t.vs[h / 2] >> (16 * (h & 1)) & 0x7FFFu;
        if (x >= 0x7C00u) bad |= 1u << h;
      }
      if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) {
#pragma unroll
        for (int h = 0; h < 8; h++)
          if (bad >> h & 1u) t.vs[h / 2] &= h & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        // The dims of this lane's sums (D / 16 (4 lg + e) + n) are all of group D lg / 128, whose scales the lanes of
        // columns 2 D lg / 128 * 16 / D .. hold: the first of them, of each four positions' lane group.
        const uint32_t holder = lg * D / 128 * 32 / kVWords;
        uint32_t mask = 0;
#pragma unroll
        for (uint32_t x = 0; x < 4; x++) mask |= (uint32_t)__shfl((int)bad, (int)(16 * x + holder), 64) << (8 * x);
        poison = (visible & mask) != 0;
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) top = fmaxf(top, s[k][e]);
    top = max_of_head(top);
    float shift = top == -INFINITY ? 0.f : fmaf(top, f, -15.f);
    // (past kLargest the max's own rounding would put weights out of f16's range: there it is taken from the
    // scores instead, which leaves the largest exactly 0)
    if (__builtin_amdgcn_ballot_w64(fabsf(shift) > kLargest) != 0) {
      const float from = top == -INFINITY ? 0.f : top;  // (a column without a position yet)
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[k][e] -= from;
      shift = -15.f;
    }
    if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
      const float alpha = top > m ? __builtin_amdgcn_exp2f((m - top) * f) : 1.f;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < kDims; i++) o[i] *= alpha;
      m = top;
    }
    half8 pb[kParts];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float p = __builtin_amdgcn_exp2f(fmaf(s[k][e], f, -shift));
        l += p;
#pragma unroll
        for (int x = 0; x < kParts; x++) {
          const _Float16 h = (_Float16)p;
          pb[x][4 * k + e] = h;
          p -= (float)h;
        }
      }
    if (poison) {
#pragma unroll
      for (int i = 0; i < kDims; i++) o[i] += __builtin_nanf("");
    }
    half2v pairs[4];
    scale_pairs(t.vs, pairs);
#pragma unroll
    for (int i = 0; i < kDims; i++) {
      const half8 va = values(t.v[i], pairs, bits_over);
#pragma unroll
      for (int x = 0; x < kParts; x++) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[x], o[i], 0, 0, 0);
    }
  };

  // (The page ids are read outside the loop over their 64 steps: a wait for them inside would be a wait
  // for the tiles under way.)
  for (uint32_t i0 = 0; i0 < mine; i0 += 64) {
    if (i0) {
      ids = pages_of(i0);
      fetch(tiles[0], ids, i0, 0);
    }
    const uint32_t count = min(64u, mine - i0);
    for (uint32_t i = 0; i < count; i += 2) {
      if (i + 1 < count) fetch(tiles[1], ids, i0, i + 1);
      compute(tiles[0], i0 + i);
      if (i + 1 < count) {
        if (i + 2 < count) fetch(tiles[0], ids, i0, i + 2);
        compute(tiles[1], i0 + i + 1);
      }
    }
  }

  // The waves meet in LDS. (A lane's rows there are D floats apart, so the 16 columns' stores meet in the same banks: 1,536 cycles a
  // workgroup, 60% of the kernel's LDS cycles with 16 sequences of 16 rows.)
  __shared__ float top_of[kWaves][16], sum_of[kWaves][16];
  __shared__ __attribute__((aligned(16))) float part_of[kWaves][16][D];
  const bool whole = chunk >= reach;  // no other chunk: the result itself
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (lg == 0) {
    top_of[wave][lr] = m == -INFINITY ? -INFINITY : m * f;
    sum_of[wave][lr] = l;
  }
  // row 4 lg + e of block i is dim D / 16 (4 lg + e) + i
#pragma unroll
  for (int e = 0; e < 4; e++)
#pragma unroll
    for (int i = 0; i < kDims; i += 4)
      *reinterpret_cast<float4*>(&part_of[wave][lr][kDims * (4 * lg + e) + i]) =
          make_float4(o[i][e], o[i + 1][e], o[i + 2][e], o[i + 3][e]);
  __syncthreads();
  const uint32_t columns = min(16u, n * a.group - c0);
  for (uint32_t i = tid; i < columns * (D / 4); i += 64 * kWaves) {
    const uint32_t h = i / (D / 4), d = 4 * (i % (D / 4));
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, top_of[w][h]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float c = top_of[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top_of[w][h] - top);
      const float4 v = *reinterpret_cast<const float4*>(&part_of[w][h][d]);
      sum = fmaf(c, sum_of[w][h], sum);
      acc = make_float4(fmaf(c, v.x, acc.x), fmaf(c, v.y, acc.y), fmaf(c, v.z, acc.z), fmaf(c, v.w, acc.w));
    }
    const uint32_t r = first + (c0 + h) / a.group, hd = kv * a.group + (c0 + h) % a.group;
    if (whole) {
      const float x = sum == 0.f ? 0.f : 1.f / sum;
      TQ* to = static_cast<TQ*>(a.out) + (size_t)r * a.out_stride + (size_t)hd * D + d;
      to[0] = from_f32<TQ>(acc.x * x);
      to[1] = from_f32<TQ>(acc.y * x);
      to[2] = from_f32<TQ>(acc.z * x);
      to[3] = from_f32<TQ>(acc.w * x);
    } else {
      const size_t at_row = ((size_t)r * a.heads + hd) * a.splits + split;
      *reinterpret_cast<float4*>(a.o + at_row * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.ml + 2 * at_row) = make_float2(top, sum);
    }
  }
}

// Many columns: the waves share the tiles instead of taking them in turn. A step of 64 positions is dequantized
// once, by all four waves, into LDS - K as what the first product takes (8 dims of a position), V as what the second takes
// (8 positions of a dim), each code times its scale, exact in f16 - and each wave multiplies it with its own kBlocks
// blocks of columns. So a word is unpacked once for 64 kBlocks columns, columns never meet, and one step's words are under
// way and the next one's in the other half of LDS while this one is multiplied. Scores need no scale of their own.
//
// K lies as [8 dims][position], V as [8 positions][dim], so that a product's 16 rows are 16 consecutive operands of
// 16 bytes; positions in the order of the first product's rows (row 16 k + 4 a + e of 32: position 8 a + kOrder[4 k + e]),
// dims 4 q + j (2 q + j at head_dim 64) at 32 j + q, so that V's stores follow each other. K's do
// not: of eight lanes that store together two positions share two slots of four, and conflicts are 4.4 of the 13.2 million LDS
// cycles of 8 sequences of 64 rows at up to 8192.
//
// kHalves 2, for up to 64 columns: two waves share 32 columns, each with half of a step's positions, and meet at the end. (Four
// waves of 16 columns each read all of a step from LDS: 64 KB more a step, which is what bound them.)
//
// kWaves 8, for more than 128 columns: a word is unpacked once for 256, two steps between barriers (8 sequences of 64 rows at up
// to 8192, 32 / 8 heads of 128, bf16: 81 us for 87). Eight waves that share positions, for up to 128 and up to 64 columns,
// were as fast as four with the sequences in twice as many chunks.
template <int D, int kWaves, int kHalves, int kParts, class TQ>
__global__ __launch_bounds__(64 * kWaves, 2) void wide_kernel(Args a, Pool pool) {
  constexpr int kBlocks = 2, kGroups = D / 32, kDims = D / 16, kWords = D / 32;  // kWords: of K and of V, a thread and step
  constexpr uint32_t kSub = kWaves / 4;  // steps between barriers
  // The max is taken up only where it has grown by kLag (in powers of two): with 16-bit rows, whose weights are scaled by
  // that much less, a column's sums are then rescaled about once (8 of up to 8192, 64 rows, 32 / 8 heads of 128, bf16, in eights:
  // 92.6 us, rescaled at every new max 98).
  constexpr float kLag = kParts == 2 ? 0.f : 3.f, kShift = 15.f - kLag;
  constexpr uint32_t kStep = 64, kColumns = 16 * kBlocks * kWaves / kHalves, kPad = kStep + 1;
  constexpr int kKeys = 4 / kHalves;  // blocks of 16 positions of a step and wave
  __shared__ half8 k_of[2 * kSub][D / 8][kPad], v_of[2 * kSub][8][D];
  // of a tail step's V: positions (8 a byte) whose scale is no number
  __shared__ __attribute__((aligned(8))) uint8_t bad_of[2 * kSub][kGroups][8];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lr = lane & 15u, lg = lane >> 4;
  // the step and the 32 positions of it that this wave unpacks
  const uint32_t sub = kSub == 1 ? 0 : wave >> 2, half_step = kSub == 1 ? wave >> 1 : (wave >> 1) & 1u;

  uint32_t id = blockIdx.x;
  const uint32_t split = id % a.splits;
  id /= a.splits;
  const uint32_t tile = id % a.tiles;
  id /= a.tiles;
  const uint32_t kv = id % pool.kv_heads, seq = id / pool.kv_heads;

  const uint32_t first = a.offsets[seq], last = a.offsets[seq + 1], n = last - first, length = a.lengths[seq];
  const uint32_t reach = min(length, a.capacity), chunk = chunk_of(a, reach), begin = split * chunk;
  if (!computed(a, first, last) | (tile * kColumns >= n * a.group) | ((split != 0) & (begin >= reach))) return;  // (read at once)
  const bool fits = n <= length;  // (else the rows give zeros)
  const uint32_t base = fits ? length - n : 0, end = fits ? min(reach, begin + chunk) : 0;
  const Magic bits_over = magic();
  const uint32_t half = kHalves == 1 ? 0 : wave >> 1, of_half = kHalves == 1 ? wave : wave & 1u;  // the wave's half of a step
  const uint32_t c0 = tile * kColumns + 16 * kBlocks * of_half;                   // the first of its columns
  const bool active = c0 < n * a.group;

  const uint32_t page_size = 1u << pool.page_shift;
  const Layout at = layout<D>(page_size);
  // K: a thread has position tid / 4 and words (tid % 4, 0 ..) of its row, and the scale of group tid % 4; V: 8
  // positions tid / 32 and kWords dims.
  const uint32_t position = (tid >> 2) & 31u, quad = tid & 3u, pairs_at = tid & 31u, eight = (tid >> 5) & 3u;
  const uint32_t k_off = position * (D / 2) + quad * (kGroups * 4);
  const uint32_t ks_off = at.k_scales + ((quad % kGroups) << (pool.page_shift + 1)) + position * 2;
  const uint32_t v_off = at.v_codes + (eight * D + pairs_at * kWords) * 4;
  const uint32_t v_group = pairs_at * kWords / 32;
  const uint32_t vs_off = at.v_scales + (v_group << (pool.page_shift + 1)) + eight * 16;
  const uint32_t j = ((position & 3u) << 1) | ((position >> 2) & 1u);  // kOrder[j] = position % 8
  const uint32_t k_to = 32 * half_step + 16 * (j >> 2) + 4 * (position >> 3) + (j & 3u);

  const uint32_t steps = begin < end ? (end - begin + kStep - 1) / kStep : 0;
  // The pages of 64 halves of steps, one a lane, from step s0 on.
  const auto pages_of = [&](uint32_t s0) {
    const uint32_t p = begin + s0 * kStep + 32 * lane;
    return p < end ? pool.page_of(seq, p) : 0xFFFFFFFFu;
  };
  uint32_t ids = pages_of(0), later = 0;  // `later`: of the 32 steps after those
  const auto page_at = [&](uint32_t s, uint32_t half) {  // (ids of the step's 32; the next ones' from the second on)
    return (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(2 * (s & 31u) + half));
  };

  struct Stage {
    uint32_t k[kWords], v[kWords];
    u32x4 vs;
    uint32_t ks;
  };
  const auto load = [&](Stage& t, uint32_t page, uint32_t s) {
    const bool have = page < pool.pages;
    // (no page: a resource of no bytes, whose loads return zeros)
    const auto r = egd::buffer(pool.block(have ? page : 0, kv, at.head_bytes), have ? at.head_bytes : 0);
    const uint32_t slot = (begin + s * kStep + 32 * half_step) & (page_size - 1u);
    if constexpr (kWords == 4) {
      const u32x4 k = egd::load_b128(r, k_off, slot * (D / 2)), v = egd::load_b128(r, v_off, (slot / 8) * (D * 4));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        t.k[i] = k[i];
        t.v[i] = v[i];
      }
    } else {
      const uint64_t k = egd::load_b64(r, k_off, slot * (D / 2)), v = egd::load_b64(r, v_off, (slot / 8) * (D * 4));
      t.k[0] = (uint32_t)k;
      t.k[1] = (uint32_t)(k >> 32);
      t.v[0] = (uint32_t)v;
      t.v[1] = (uint32_t)(v >> 32);
    }
    t.ks = __builtin_amdgcn_raw_buffer_load_b16(r, ks_off, slot * 2, 0);
    t.vs = egd::load_b128(r, vs_off, slot * 2);
  };
  const auto put = [&](Stage& t, uint32_t s) {
    const uint32_t buffer = s & (2 * kSub - 1);
    const uint32_t two = t.ks * 0x00010001u;  // (each group's by its quad of lanes)
    const uint32_t scale[4] = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)two, 0x00, 0xF, 0xF, true),
                               (uint32_t)__builtin_amdgcn_update_dpp(0, (int)two, 0x55, 0xF, 0xF, true),
                               (uint32_t)__builtin_amdgcn_update_dpp(0, (int)two, 0xAA, 0xF, 0xF, true),
                               (uint32_t)__builtin_amdgcn_update_dpp(0, (int)two, 0xFF, 0xF, 0xF, true)};
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
      const half2v x = halves(scale[g]);
      const half2v same[4] = {x, x, x, x};
      k_of[buffer][4 * g + quad][k_to] = values(t.k[g], same, bits_over);
    }
    const uint32_t j0 = begin + s * kStep + 32 * half_step + 8 * eight;  // of this thread's V
    if (begin + (s + 1) * kStep > base) {
      // positions past the end: values of zero. Scales that are no numbers (their values are none then) would reach, times
      // a weight of 0, the columns that do not see their position: they are taken out of the product, and noted for the
      // sums of those that do.
      t.vs = first_halves(t.vs, max(0, min(8, (int)(end - j0))));
      uint32_t bad = 0;
#pragma unroll
      for (int h = 0; h < 8; h++)
        if ((t.vs[h / 2] >> (16 * (h & 1)) & 0x7FFFu) >= 0x7C00u) {
          bad |= 1u << h;
          t.vs[h / 2] &= h & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        }
      if (pairs_at % (32 / kWords) == 0) bad_of[buffer][v_group][4 * half_step + eight] = (uint8_t)bad;
    }
    half2v pairs[4];
    scale_pairs(t.vs, pairs);
#pragma unroll
    for (int w = 0; w < kWords; w++) v_of[buffer][4 * half_step + eight][32 * w + pairs_at] = values(t.v[w], pairs, bits_over);
  };

  // This lane's columns, and what each sees of the sequence's rows.
  half8 qf[kBlocks][kGroups][kParts];
  float f[kBlocks];
  uint64_t sees[kBlocks];
  Stage stage;
  // (reads that wait for nothing but offsets and lengths first, then the first step's; the rest goes on beside those)
  const bool tail_of = end > base;
  const uint32_t parent = tail_of && a.parents && lane < n ? a.parents[first + lane] : 0xFFFFFFFFu;
  Eight<TQ> raw[kBlocks][kGroups];
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const uint32_t c = min(c0 + 16 * b + lr, n * a.group - 1);
    load_query<D, TQ>(a, first + c / a.group, kv * a.group + c % a.group, lg, raw[b]);
  }
  if (sub < steps) load(stage, page_at(sub, half_step), sub);
  const uint64_t all = tail_of ? ancestors(a.parents != nullptr, parent) : 0;
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const uint32_t c = min(c0 + 16 * b + lr, n * a.group - 1);
    const bool in = c0 + 16 * b + lr < n * a.group;
    sees[b] = of_row(all, c / a.group);
    const int up = make_query<D, kParts, TQ>(raw[b], in, qf[b]);
    f[b] = fmaxf(ldexpf(a.scale, -up), 0x1p-126f);  // (not 0: -inf times it is -inf)
  }

  f32x4 o[kBlocks][kDims];
  float m[kBlocks], l[kBlocks];  // running max of the scores before f; this lane's share of the sum
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int i = 0; i < kDims; i++) o[b][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto compute = [&](uint32_t step) {
    const uint32_t buffer = step & (2 * kSub - 1), j0 = begin + step * kStep;
    f32x4 s[kBlocks][kKeys];
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
#pragma unroll
      for (int k = 0; k < kKeys; k++) s[b][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < kGroups; g++)
#pragma unroll
      for (int k = 0; k < kKeys; k++) {
        const half8 kc = k_of[buffer][4 * g + lg][32 * half + 16 * k + lr];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
          for (int p = 0; p < kParts; p++) s[b][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qf[b][g][p], s[b][k], 0, 0, 0);
      }
    const bool have0 = page_at(step, 0) < pool.pages, have1 = page_at(step, 1) < pool.pages;
    if (j0 + kStep > base || !have0 || !have1) {
      // of the sequence's rows what the column sees; nothing past the end or on no page
      uint64_t real = end - j0 >= 64 ? ~0ull : (1ull << (end - j0)) - 1u;
      if (!have0) real &= 0xFFFFFFFF00000000ull;
      if (!have1) real &= 0x00000000FFFFFFFFull;
      const bool tail = j0 + kStep > base;
#pragma unroll
      for (int b = 0; b < kBlocks; b++) {
        uint64_t visible = j0 >= base ? sees[b] >> (j0 - base) : ~0ull;
        if (j0 < base && tail) visible = sees[b] << (base - j0) | ((1ull << (base - j0)) - 1u);
        visible &= real;
        if (kHalves == 2) visible &= 0xFFFFFFFFull << (32 * half);  // (the other half's are the other wave's)
        const uint64_t mine = visible >> (32 * half + 8 * lg);
#pragma unroll
        for (int k = 0; k < kKeys; k++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (!(mine >> (32 * (k >> 1) + kOrder[4 * (k & 1) + e]) & 1u)) s[b][k][e] = -INFINITY;
        if (tail) {
          // this lane's sums are of dims 64 i + 16 lg .. +16 (32 i + 8 lg .. +8 at head_dim 64), i < 2
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const uint32_t group = D == 128 ? 2 * i + (lg >> 1) : i;
            if (visible & *reinterpret_cast<const uint64_t*>(bad_of[buffer][group])) {
#pragma unroll
              for (int x = i; x < kDims; x += 2) o[b][x] += __builtin_nanf("");
            }
          }
        }
      }
    }
    half8 pb[kBlocks][kKeys / 2][kParts];
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      float top = m[b];
#pragma unroll
      for (int k = 0; k < kKeys; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, s[b][k][e]);
      top = max_of_head(top);
      if (__builtin_amdgcn_ballot_w64((top - m[b]) * f[b] > kLag) != 0) {
        const float alpha = top > m[b] ? __builtin_amdgcn_exp2f((m[b] - top) * f[b]) : 1.f;
        l[b] *= alpha;
#pragma unroll
        for (int i = 0; i < kDims; i++) o[b][i] *= alpha;
        m[b] = top;
      }
      float shift = m[b] == -INFINITY ? 0.f : fmaf(m[b], f[b], -kShift);
      // (past kLargest the max's own rounding would put weights out of f16's range: there it is taken from the
      // scores instead, which leaves the largest exactly 0)
      if (__builtin_amdgcn_ballot_w64(fabsf(shift) > kLargest) != 0) {
        const float from = m[b] == -INFINITY ? 0.f : m[b];  // (a column without a position yet)
#pragma unroll
        for (int k = 0; k < kKeys; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[b][k][e] -= from;
        shift = -kShift;
      }
#pragma unroll
      for (int k = 0; k < kKeys; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float p = __builtin_amdgcn_exp2f(fmaf(s[b][k][e], f[b], -shift));
          l[b] += p;
#pragma unroll
          for (int x = 0; x < kParts; x++) {
            const _Float16 h = (_Float16)p;
            pb[b][k >> 1][x][4 * (k & 1) + e] = h;
            p -= (float)h;
          }
        }
    }
#pragma unroll
    for (int h = 0; h < kKeys / 2; h++)
#pragma unroll
      for (int i = 0; i < kDims; i++) {
        const half8 va = v_of[buffer][4 * (half + h) + lg][16 * i + lr];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
          for (int x = 0; x < kParts; x++)
            o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[b][h][x], o[b][i], 0, 0, 0);
      }
  };

  if (sub < steps) put(stage, sub);
  if (kSub + sub < steps) load(stage, page_at(kSub + sub, half_step), kSub + sub);
  __syncthreads();
  for (uint32_t s = 0; s < steps; s += kSub) {
    if (active) compute(s);  // (both in a loop take 24 registers more)
    if (kSub == 2 && active && s + 1 < steps) compute(s + 1);
    if (s + kSub + sub < steps) put(stage, s + kSub + sub);
    if ((s & 31u) == 32u - kSub) ids = later;  // (the next steps')
    if ((s & 31u) == 32u - 3 * kSub) later = pages_of(s + 3 * kSub);
    const uint32_t next = s + 2 * kSub + sub;
    if (next < steps) {
      const uint32_t page = (next & 31u) == sub && (s & 31u) == 32u - 2 * kSub
                                ? (uint32_t)__builtin_amdgcn_readlane((int)later, (int)(2 * sub + half_step))
                                : page_at(next, half_step);
      load(stage, page, next);
    }
    __syncthreads();
  }

#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    l[b] += __shfl_xor(l[b], 16, 64);
    l[b] += __shfl_xor(l[b], 32, 64);
  }
  if constexpr (kHalves == 2) {  // the other half's wave has the same columns and dims in the same lanes
    f32x4* const sums = reinterpret_cast<f32x4*>(v_of) + of_half * (kBlocks * kDims * 64) + lane;
    float2* const stats = reinterpret_cast<float2*>(k_of) + of_half * (kBlocks * 64) + lane;
    if (half == 1) {
#pragma unroll
      for (int b = 0; b < kBlocks; b++) {
        stats[64 * b] = make_float2(m[b], l[b]);
#pragma unroll
        for (int i = 0; i < kDims; i++) sums[64 * (kDims * b + i)] = o[b][i];
      }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      const float2 other = stats[64 * b];
      const float top = fmaxf(m[b], other.x), from = top == -INFINITY ? 0.f : top;
      const float x = __builtin_amdgcn_exp2f((m[b] - from) * f[b]), y = __builtin_amdgcn_exp2f((other.x - from) * f[b]);
      l[b] = l[b] * x + other.y * y;
#pragma unroll
      for (int i = 0; i < kDims; i++) o[b][i] = o[b][i] * x + sums[64 * (kDims * b + i)] * y;
      m[b] = top;
    }
  }
  if (!active) return;
  const bool whole = chunk >= reach;  // no other chunk: the result itself
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const uint32_t c = c0 + 16 * b + lr;
    const float sum = l[b];
    if (c >= n * a.group) continue;
    const uint32_t r = first + c / a.group, hd = kv * a.group + c % a.group;
    const size_t at_row = ((size_t)r * a.heads + hd) * a.splits + split;
    const float x = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
    const float top = m[b] == -INFINITY ? -INFINITY : m[b] * f[b];
    if (!whole && lg == 0) *reinterpret_cast<float2*>(a.ml + 2 * at_row) = make_float2(top, sum);
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float y[kWords];
#pragma unroll
        for (int w = 0; w < kWords; w++) y[w] = o[b][i + 2 * w][e] * x;
        const uint32_t d = (D / 2) * i + (4 * lg + e) * kWords;
        if (whole) {
          struct alignas(sizeof(TQ) * kWords) Several {
            TQ v[kWords];
          } to;
#pragma unroll
          for (int w = 0; w < kWords; w++) to.v[w] = from_f32<TQ>(y[w]);
          *reinterpret_cast<Several*>(static_cast<TQ*>(a.out) + (size_t)r * a.out_stride + (size_t)hd * D + d) = to;
        } else {
          struct alignas(4 * kWords) Several {
            float v[kWords];
          } to;
#pragma unroll
          for (int w = 0; w < kWords; w++) to.v[w] = y[w];
          *reinterpret_cast<Several*>(a.o + at_row * D + d) = to;
        }
      }
  }
}

// The chunks of kTogether (row, head) joined by a workgroup, D / 4 threads each.
template <int D, class TQ>
__global__ __launch_bounds__(256) void join_kernel(Args a, uint32_t sequences) {
  constexpr uint32_t kEach = D / 4, kTogether = kThreads / kEach;
  const uint32_t i = blockIdx.x * kTogether + threadIdx.x / kEach, d = 4 * (threadIdx.x % kEach);
  const uint32_t r = i / a.heads, head = i % a.heads;
  if (r >= a.rows) return;
  uint32_t lo = 0, hi = sequences;  // the sequence: the last that begins at r or before
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.offsets[mid] <= r) lo = mid;
    else hi = mid;
  }
  const uint32_t first = a.offsets[lo], last = a.offsets[lo + 1];
  if (r < first || r >= last || !computed(a, first, last)) return;
  const uint32_t reach = min(a.lengths[lo], a.capacity), chunk = chunk_of(a, reach);
  if (chunk >= reach) return;  // (one chunk: it wrote the result)
  const uint32_t count = (reach + chunk - 1) / chunk;
  const size_t at_row = (size_t)i * a.splits;
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + at_row;
  const float* o = a.o + at_row * D + d;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (uint32_t c = 0; c < count; c++) {
    const float2 s = ml[c];
    const float4 v = *reinterpret_cast<const float4*>(o + (size_t)c * D);
    const float to = fmaxf(top, s.x), from = to == -INFINITY ? 0.f : to;
    const float x = __builtin_amdgcn_exp2f(top - from), y = __builtin_amdgcn_exp2f(s.x - from);
    sum = fmaf(sum, x, s.y * y);
    acc = make_float4(fmaf(acc.x, x, v.x * y), fmaf(acc.y, x, v.y * y), fmaf(acc.z, x, v.z * y), fmaf(acc.w, x, v.w * y));
    top = to;
  }
  const float x = sum == 0.f ? 0.f : 1.f / sum;
  struct alignas(4 * sizeof(TQ)) Four {
    TQ v[4];
  };
  *reinterpret_cast<Four*>(static_cast<TQ*>(a.out) + (size_t)r * a.out_stride + (size_t)head * D + d) =
      Four{{from_f32<TQ>(acc.x * x), from_f32<TQ>(acc.y * x), from_f32<TQ>(acc.z * x), from_f32<TQ>(acc.w * x)}};
}

struct Plan {
  uint32_t per_tile, waves, tiles, splits, min_chunk;  // per_tile: blocks of 16 columns a workgroup
};

template <int D, class TQ>
void launch(eg_context* ctx, const Args& a, const Pool& p, const Plan& plan, uint64_t blocks) {
  constexpr int kParts = std::is_same<TQ, float>::value ? 2 : 1;
  const dim3 grid((uint32_t)blocks), threads(kThreads);
  const auto kernel = plan.per_tile == 1   ? (plan.waves == 4 ? few_kernel<D, 4, kParts, TQ> : few_kernel<D, 8, kParts, TQ>)
                      : plan.per_tile == 4 ? wide_kernel<D, 4, 2, kParts, TQ>
                      : plan.per_tile == 8 ? wide_kernel<D, 4, 1, kParts, TQ>
                                           : wide_kernel<D, 8, 1, kParts, TQ>;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * plan.waves), 0, ctx->stream, a, p);
  if (a.splits > 1)
    hipLaunchKernelGGL((join_kernel<D, TQ>), dim3((a.rows * a.heads * (D / 4) + kThreads - 1) / kThreads), threads, 0,
                       ctx->stream, a, p.sequences);
}

// The kernel and the chunks of a sequence's positions: what the times below add up to least by. Lengths are on the device, so
// it goes by what the tables reach less a page, whose last ones are seldom full, and by a page at least (of no positions all kinds
// cost the same: 32 and 64 sequences of 32 rows in a page of 256 each, 32 / 8 heads of 128, bf16, took 30.8 and 57.0 us for 14.5
// and 21.5). The times of a step of a workgroup alone on its CU and of one of several, in us: measured with each kernel of four
// waves - at up to 4096 positions 32 sequences of 16 rows, 32 / 8 heads of 128, bf16, took 100 us in single blocks, 85 in fours
// and 76 with positions halved, 107 and 85 in eights; 64 of 16 / 4 heads of 64 54, 62 and 49, 81 and 63. Of eight waves, fitted:
// single blocks by two shared steps of four waves; sixteens (256 columns), alone or not, by what they gain on eights over sizes of
// the whole range, whose sequences differ in length, which a workgroup alone on its CU has to wait for - of 32 rows of 64 / 8
// heads they take 149 us for 173 (128, bf16), 243 for 269 (f32), 100 for 116 and 168 for 176 (64). A launch, its chain of reads
// and the waves' meeting take 6 us, a join 4.5 and its partials a us for 4 MB written and read.
Plan plan_of(uint32_t cus, uint64_t pairs, uint64_t columns, uint32_t reach, uint64_t outputs, uint32_t head_dim, bool f32) {
  struct Kind {
    uint32_t per_tile, waves, step;
    double alone[2][2], shared[2][2];  // [head_dim 128][f32]
  };
  constexpr Kind kKinds[] = {{1, 4, 128, {{0.55, 0.75}, {1.0, 1.25}}, {{0.38, 0.52}, {0.74, 0.93}}},
                             {1, 8, 256, {{0.76, 1.04}, {1.48, 1.86}}, {{0.76, 1.04}, {1.48, 1.86}}},
                             {4, 4, 64, {{0.87, 1.16}, {1.22, 1.70}}, {{0.54, 0.78}, {0.88, 1.22}}},
                             {8, 4, 64, {{1.17, 1.84}, {1.59, 2.46}}, {{0.75, 1.23}, {1.03, 1.74}}},
                             {16, 8, 64, {{1.45, 2.40}, {2.00, 3.45}}, {{1.45, 2.40}, {2.00, 3.45}}}};
  const uint64_t per_split = outputs * (head_dim + 2) * 4, room = (eg::kPartialsBytes - 64) / per_split;
  Plan best{};
  double least = -1.0;
  for (const Kind& kind : kKinds) {
    const uint64_t width = 16 * kind.per_tile, tiles = (columns + width - 1) / width, all = pairs * tiles;
    const double alone = kind.alone[head_dim == 128][f32], shared = kind.shared[head_dim == 128][f32];
    if (kind.per_tile != 1 && 2 * columns < width) continue;
    const uint64_t most = std::min<uint64_t>({std::max<uint64_t>(1, (reach + 255) / 256), std::max<uint64_t>(1, 4ull * cus / all),
                                              std::max<uint64_t>(1, room)});
    // (each number of chunks up to 8; of more, those that give a CU 1 to 4 workgroups. All of them, where tables are long, are
    // microseconds of the host's time.)
    for (uint64_t i = 1, last = 0; i <= 12; i++) {
      const uint64_t s = std::min(most, i <= 8 ? i : (i - 8) * cus / all);
      if (s <= last) continue;
      last = s;
      const uint64_t even = (reach + s - 1) / s, chunk = s == 1 ? reach : std::max<uint64_t>(256, (even + 63) & ~63ull);
      const uint64_t chunks = s == 1 ? 1 : (reach + chunk - 1) / chunk, steps = (chunk + kind.step - 1) / kind.step;
      const uint64_t each = (all * chunks + cus - 1) / cus;  // workgroups of the busiest CU
      double us = (kind.waves == 8 ? 6.6 : 6.0) + steps * (each == 1 ? alone : each * shared);
      if (chunks > 1) us += 4.5 + chunks * per_split * 2 / 4e6;
      if (least < 0.0 || us < least) {
        least = us;
        best = Plan{kind.per_tile, kind.waves, (uint32_t)tiles, (uint32_t)s, 256};
      }
    }
  }
  if (best.splits == 1) best.min_chunk = 0x7FFFFFC0u;  // (whole, however long)
  return best;
}

}  // namespace

extern "C" int eg_attention_tree_kv4(eg_context* ctx, const void* q, const uint32_t* offsets, const uint32_t* parents,
                                     const uint32_t* lengths, const uint32_t* table, const void* pool, void* out,
                                     const eg_kv4_dims* dims, const eg_attention_tree_dims* attention) {
  const char* op = "attention_tree_kv4";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  const bool some = attention && attention->rows != 0 && attention->max_rows != 0 && dims->sequences != 0;
  if (!attention || (some && (!q || !offsets || !lengths || !out || (dims->max_pages != 0 && !table))))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_attention_tree_dims& d = *attention;
  if (!known_type(d.type)) return eg::fail(ctx, EG_ERR_INVALID, "%s: type %d (eg_element)", op, d.type);
  if (d.heads == 0 || d.heads % dims->kv_heads != 0 || d.heads > 65535)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: heads %u are not a multiple of kv_heads %u (at most 65535)", op, d.heads,
                    dims->kv_heads);
  if (d.max_rows > kMostRows) return eg::fail(ctx, EG_ERR_RANGE, "%s: max_rows %u (at most %u)", op, d.max_rows, kMostRows);
  if (!(d.scale >= 0.f) || d.scale > 1e6f) return eg::fail(ctx, EG_ERR_INVALID, "%s: scale %g (0 to 1e6)", op, d.scale);
  const uint32_t width = d.heads * dims->head_dim;
  Args a{};
  a.q = q;
  a.offsets = offsets;
  a.parents = parents;
  a.lengths = lengths;
  a.out = out;
  a.rows = d.rows;
  a.max_rows = d.max_rows;
  a.heads = d.heads;
  a.group = d.heads / dims->kv_heads;
  a.q_stride = d.q_stride ? d.q_stride : width;
  a.out_stride = d.out_stride ? d.out_stride : width;
  if (a.q_stride < width || a.out_stride < width || (a.q_stride | a.out_stride) % 8)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: strides %u, %u (multiples of 8, at least a row)", op, a.q_stride,
                    a.out_stride);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q and out must be 16-byte aligned", op);
  if (!some) return EG_OK;
  a.scale = (d.scale > 0.f ? d.scale : 1.0f / sqrtf((float)dims->head_dim)) * kLog2e;
  a.capacity = dims->max_pages * dims->page_size;
  const uint64_t pairs = (uint64_t)dims->sequences * dims->kv_heads, columns = (uint64_t)std::min(d.max_rows, d.rows) * a.group;
  const uint32_t page = std::min(a.capacity, dims->page_size), reach = std::max(page, a.capacity - page);
  const Plan plan = plan_of(ctx->cu_count, pairs, columns, reach, (uint64_t)d.rows * d.heads, dims->head_dim,
                            d.type == EG_ELEMENT_F32);
  const uint64_t tiles = pairs * plan.tiles, splits = plan.splits;
  a.tiles = plan.tiles;
  a.splits = plan.splits;
  a.min_chunk = plan.min_chunk;
  if (tiles * splits >= (1ull << 31) / kThreads || (uint64_t)d.rows * d.heads >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows of %u heads in %u sequences over the grid limit", op, d.rows, d.heads,
                    dims->sequences);
  // A workgroup writes the columns that it alone uses, after their queries are read: the result may take q's place, row by row. What the
  // others read of all else it would overwrite.
  const uint64_t size = d.type == EG_ELEMENT_F32 ? 4 : 2, n = dims->sequences;
  const Extent result{out, d.rows, size * a.out_stride, size * width}, queries{q, d.rows, size * a.q_stride, size * width};
  bool apart = (q == out && a.q_stride == a.out_stride) || !overlap(result, queries);
  for (const Extent& in : {words(offsets, n + 1), words(parents, d.rows), words(lengths, n), words(table, n * dims->max_pages),
                           Extent{pool, dims->pages, dims->page_stride, eg_kv4::page_bytes(*dims)}})
    apart = apart && !overlap(result, in);
  if (!apart) return eg::fail(ctx, EG_ERR_INVALID, "%s: out lies in an input (it may be q, row by row)", op);
  a.ml = reinterpret_cast<float*>(eg::partials(ctx));
  a.o = a.ml + (((size_t)d.rows * d.heads * splits * 2 + 3) & ~(size_t)3);
  const Pool p = eg_kv4::pool_of(*dims, pool, table);
  const OnDevice on(ctx);
  with_type(d.type, [&](auto t) {
    using TQ = decltype(t);
    if (dims->head_dim == 64) launch<64, TQ>(ctx, a, p, plan, tiles * splits);
    else launch<128, TQ>(ctx, a, p, plan, tiles * splits);
  });
  return eg::check_launch(ctx, op);
}

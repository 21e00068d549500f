// Causal attention over packed sequences of different lengths (eg_attention_packed).
//
//   out[i][h] = sum_j p_j V[j] / sum_j p_j,  p_j = exp(scale q[i][h] . K[j] - max_j),  j <= nk - nq + i
//
// One pass over the keys with the running max and sum of the softmax. A workgroup takes 128 queries of
// one head, a wave 32 of them; key tiles of 64 go through LDS, the next one's loads under way while
// this one is multiplied. Both products run on v_mfma_f32_32x32x16 in the transposed form S^T = K Q^T,
// O^T = V^T P^T: a lane holds one query's scores (rows of S^T: 4 consecutive keys of every 8), which
// are the second product's B operand where they lie, with V^T read from LDS transposed.
//
// Bound by the SIMDs' issue of both units, and at length by power: the clock falls from 2.4 to 1.9 GHz. A wave and
// tile of 64 keys take 1024 (head_dim 128) or 512 (64) cycles of the matrix cores and about 750 of vector
// instructions (32 exponentials of 8 cycles, the rest 4 each), together 2050 (two waves a SIMD) and 1220 (three).
// MI355X: a prompt of 8192, 32 / 8 heads of 128, bf16: 514 us, 1070 TFLOP/s (a library product of 8192 reaches 1435
// on the card), the matrix cores busy 55% of 956,000 cycles; 14 heads of 64, f16: 147 us, 820 TFLOP/s; 8 prompts of
// up to 2048, 14 heads of 64: 49 us. Tried and slower at 8192: two groups of four waves half a step apart, one at its
// products while the other is at its softmax (550 us); the next tile's scores among this one's softmax (832, and 950
// with one wave a SIMD); 64 queries a wave (head_dim 64, 206 us); row sums by a product with ones or by dot products
// (528, 518). Reading V before the softmax, or keeping the reads of V from waiting for the other buffer's loads,
// changes 1% either way.
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using eg_kv4::bf16;
using eg_kv4::from_f32;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
using egd::u32x4;

constexpr uint32_t kThreads = 256, kWaves = 4;
constexpr uint32_t kQueries = 32 * kWaves;  // per workgroup
constexpr uint32_t kKeys = 64;              // per tile
constexpr uint32_t kSplitTiles = 6, kLeastSplits = 3;
constexpr float kLag = 8.f, kLargest = 0x1p20f;
constexpr float kLog2e = 1.44269504088896340736f;

struct Args {
  const void *q, *k, *v;
  void* out;
  const uint32_t *q_offsets, *k_offsets;
  uint32_t sequences, rows, key_rows, heads, group, q_stride, k_stride, v_stride, out_stride;
  uint32_t xcds;  // XCDs a kv head, where kv heads are 1, 2 or 4; else 0
  // Keys split over workgroups: partials [row][head][split][D], unnormalised, and (max times scale, sum).
  uint32_t splits, items;
  uint32_t xcd_cus;  // CUs of an XCD
  float *o, *ml;
  float scale;  // times log2 e
};

template <class T>
__device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (std::is_same<T, _Float16>::value) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
  } else {
    return egd::pack_bf16(a, b);
  }
}

// Max over the 2 lanes that hold a query (lane % 32).
__device__ __forceinline__ float max_of_query(float x) {
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <class T>
constexpr uint32_t kExponent = std::is_same<T, _Float16>::value ? 0x7C00u : 0x7F80u;

// Infinities and NaN among 8 values replaced by zeros.
template <class T>
__device__ __forceinline__ void clean(u32x4& v) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const bool lo = (v[i] & kExponent<T>) == kExponent<T>, hi = ((v[i] >> 16) & kExponent<T>) == kExponent<T>;
    v[i] &= (lo ? 0xFFFF0000u : 0xFFFFFFFFu) & (hi ? 0xFFFFu : 0xFFFFFFFFu);
  }
}

// Sum over the wave, in every lane, by DPP.
__device__ __forceinline__ uint32_t sum_of_wave(uint32_t v) {
  const auto add = [&](int moved) { v += (uint32_t)moved; };
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));   // row_half_mirror
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));   // row_mirror
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Query block `id` of all sequences' blocks, those with the most blocks of their sequence before them (so,
// about, the most keys) first: ranks go down through the levels, a level being the sequences' blocks of one
// index. The level is the largest with no more than `id` blocks above it, by bisection; the sequences' counts
// are in the wave's lanes. More than 64 sequences: from the last one's last block on. False past the last.
__device__ __forceinline__ bool find_block(const Args& a, uint32_t id, uint32_t& seq, uint32_t& block) {
  const uint32_t lane = threadIdx.x & 63u;
  const auto blocks_of = [&](uint32_t s) {
    if (s >= a.sequences) return 0u;
    const uint32_t b = min(a.q_offsets[s], a.rows), e = min(a.q_offsets[s + 1], a.rows);
    return e > b ? (e - b + kQueries - 1) / kQueries : 0u;
  };
  if (a.sequences <= 64) {
    const uint32_t n = blocks_of(lane);
    const auto from_level = [&](uint32_t level) {  // blocks of this level and above
      return sum_of_wave(n > level ? n - level : 0u);
    };
    uint32_t lo = 0, hi = a.rows / kQueries + 1;  // from_level(lo) > id >= from_level(hi)
    if (from_level(0) <= id) return false;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (from_level(mid) > id) lo = mid;
      else hi = mid;
    }
    uint64_t have = __ballot(n > lo);
    for (uint32_t skip = id - from_level(lo + 1); skip; skip--) have &= have - 1;
    seq = (uint32_t)__builtin_ctzll(have);
    block = lo;
    return true;
  }
  const uint32_t last = (a.sequences - 1) / 64 * 64;
  for (uint32_t i0 = last;; i0 -= 64) {
    uint32_t upto = blocks_of(i0 + (63u - lane));  // blocks of lanes 0 .. this one, later sequences in lower lanes
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
      const uint32_t t = __shfl_up(upto, d, 64);
      if (lane >= d) upto += t;
    }
    const uint64_t past = __ballot(upto > id);
    if (past) {
      const int l = __builtin_ctzll(past);
      const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, l);
      seq = i0 + (63u - (uint32_t)l);
      block = total - 1 - id;  // the sequence's last block first
      return true;
    }
    id -= (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if (i0 == 0) return false;
  }
}

// The query block (its rank) and head of this workgroup. Workgroups go to the 8 XCDs in turn, each with its own L2:
// a kv head's keys and values are read by one XCD (of fewer than 8 kv heads, by 8 / kv_heads), its query
// heads and blocks in ranks' order there - but for the first, one a CU, which go the other way: the workgroups after
// them go to the same CUs in the same order, so the CU with the fewest keys of the first gets the most of the
// second. A prompt of 8192, 14 heads of 64: 147 us for 157, 32 heads of 128 and 2048: 46.9 for 50.0.
__device__ __forceinline__ void work_of(const Args& a, uint32_t id, uint32_t& rank, uint32_t& h) {
  const uint32_t kv_heads = a.heads / a.group, xcd = id % 8u;
  uint32_t turn = id / 8u;
  if (turn < a.xcd_cus && a.items >= 8u * a.xcd_cus) turn = a.xcd_cus - 1 - turn;
  if (a.xcds) {
    const uint32_t item = turn * a.xcds + xcd % a.xcds;
    rank = item / a.group;
    h = xcd / a.xcds * a.group + item % a.group;
  } else if (kv_heads % 8u == 0) {
    const uint32_t mine = a.heads / 8u, i = turn % mine;
    rank = turn / mine;
    h = (xcd + 8u * (i / a.group)) * a.group + i % a.group;
  } else {
    rank = (8u * turn + xcd) / a.heads;
    h = (8u * turn + xcd) % a.heads;
  }
}

// A workgroup's queries and keys.
struct Work {
  uint32_t head, split, q0, nq, q_begin, k_begin;
  int shift;          // query i sees the keys below shift + i
  uint32_t key_end;   // of the workgroup's last query
  uint32_t first, stop;  // its key tiles [first, stop)
  uint32_t per_split;    // key tiles of a split
};
// (The splits of an item lie `items` apart: an item's workgroups are on one XCD, items being a multiple of 8.)
__device__ __forceinline__ bool find_work(const Args& a, uint32_t id, Work& w) {
  uint32_t rank, seq, block;
  w.split = a.splits > 1 ? id / a.items : 0;
  work_of(a, a.splits > 1 ? id % a.items : id, rank, w.head);
  if (!find_block(a, rank, seq, block)) return false;
  w.q_begin = min(a.q_offsets[seq], a.rows);
  w.nq = min(a.q_offsets[seq + 1], a.rows) - w.q_begin;
  w.k_begin = min(a.k_offsets[seq], a.key_rows);
  const uint32_t nk = max(min(a.k_offsets[seq + 1], a.key_rows), w.k_begin) - w.k_begin;
  w.q0 = block * kQueries;
  w.shift = (int)(nk - w.nq) + 1;
  const int last = w.shift + (int)min(w.q0 + kQueries, w.nq) - 1;
  w.key_end = last > 0 ? min((uint32_t)last, nk) : 0;
  const uint32_t tiles = (w.key_end + kKeys - 1) / kKeys;
  w.per_split = ((nk + kKeys - 1) / kKeys + a.splits - 1) / a.splits;
  w.first = min(w.split * w.per_split, tiles);
  w.stop = min(w.first + w.per_split, tiles);
  return true;
}

// LDS is one array: with a second one the compiler has the reads of K wait for the loads into the other
// buffer (as it does with stores to LDS in the loop). The reads run two steps ahead of their products.
template <int D, bool kSplit, class T, class TO>
__global__ __launch_bounds__(256, 2) void packed_kernel(Args a) {
  constexpr uint32_t kSlots = D / 8;                  // 16-byte slots of a row
  constexpr uint32_t kRow = D * 2, kTile = kKeys * kRow;  // bytes
  constexpr int kSteps = D / 16, kBlocks = D / 32;    // depth steps of S^T; blocks of 32 dims of O^T
  constexpr uint32_t kLoads = kTile / (kThreads * 16);
  __shared__ __attribute__((aligned(16))) uint8_t tiles[4 * kTile];  // [buffer][K or V]
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lq = lane & 31u, lh = lane >> 5;  // MFMA lane coordinates
  Work w;
  if (!find_work(a, blockIdx.x, w)) return;
  if (kSplit && w.split != 0 && w.first >= w.stop) return;
  const uint32_t h = w.head, kv = h / a.group, q_begin = w.q_begin, nq = w.nq, key_end = w.key_end;
  const uint32_t query = w.q0 + wave * 32 + lq;
  const T* q = static_cast<const T*>(a.q);
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.k) + (size_t)w.k_begin * a.k_stride + kv * D);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.v) + (size_t)w.k_begin * a.v_stride + kv * D);
  const int limit = w.shift + (int)query;                 // the keys this lane's query sees are below
  const int open = w.shift + (int)(w.q0 + wave * 32);     // and those the wave's first query does
  const uint32_t first = kSplit ? w.first : 0, stop = kSplit ? w.stop : (key_end + kKeys - 1) / kKeys;

  // Q^T, B operand: query lq, dims 16 s + 8 lh .. +8.
  u32x4 qf[kSteps];
  {
    const bool in = query < nq;
    const u32x4* src = reinterpret_cast<const u32x4*>(q + (size_t)(q_begin + (in ? query : 0)) * a.q_stride + h * D + 8 * lh);
#pragma unroll
    for (int s = 0; s < kSteps; s++) qf[s] = in ? src[2 * s] : u32x4{0, 0, 0, 0};
  }
  // K's and V's rows go to LDS 16 bytes a lane, row r's slot j at j ^ swizzle(r): 16 rows of K's
  // operand reads, and the 4 rows of V's transposed ones, then lie in different banks.
  const uint32_t lrow = tid / kSlots, slot = tid % kSlots;
  const auto kswz = [](uint32_t r) { return D == 64 ? (r >> 1) & 7u : r & 15u; };
  const auto vswz = [](uint32_t r) { return D == 64 ? 4u * ((r >> 1) & 1u) : 4u * (r & 3u); };
  uint32_t kfrom[kLoads], vfrom[kLoads];  // byte offsets in a tile, of rows kThreads / kSlots apart
#pragma unroll
  for (uint32_t i = 0; i < kLoads; i++) {
    const uint32_t r = lrow + i * (kThreads / kSlots);
    kfrom[i] = r * a.k_stride * 2 + 16 * (slot ^ kswz(r));
    vfrom[i] = r * a.v_stride * 2 + 16 * (slot ^ vswz(r));
  }
  const auto load_tile = [&](uint32_t t, uint32_t buf) {
    const uint32_t j0 = t * kKeys, left = min(kKeys, key_end - j0);
    // (the resources end with the last key's row: past it, zeros)
    const auto kr = egd::buffer(kbase + (size_t)j0 * a.k_stride * 2, (left - 1) * a.k_stride * 2 + kRow);
    const auto vr = egd::buffer(vbase + (size_t)j0 * a.v_stride * 2, (left - 1) * a.v_stride * 2 + kRow);
#pragma unroll
    for (uint32_t i = 0; i < kLoads; i++) {
      uint8_t* at = tiles + 2 * kTile * buf + (i * kThreads + wave * 64) * 16;
      egd::load_to_lds(kr, at, kfrom[i]);
      egd::load_to_lds(vr, at + kTile, vfrom[i]);
    }
  };
  const auto settle = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0: the memory-to-LDS loads have landed
    __syncthreads();
  };
  // V^T operand reads: 4 keys x 16 dims a group of 16 lanes; lane i points at key i / 4, dims 4 (i % 4).
  const uint32_t li = lane & 15u, vrow = 4 * lh + (li >> 2);
  constexpr uint32_t kVTile = kTile;
  uint32_t vat[kBlocks];
#pragma unroll
  for (uint32_t n = 0; n < (uint32_t)kBlocks; n++)
    vat[n] = kVTile + vrow * kRow + 16 * ((4 * n + 2 * ((lane >> 4) & 1u) + ((li & 3u) >> 1)) ^ vswz(vrow)) + 8 * (li & 1u);

  f32x16 o[kBlocks];
  float m, l, off;  // running max before the scale; this lane's share of the sum; the max after the scale
  bool large;       // some query's is past kLargest: off is 0
  const auto run = [&](auto careful) {
#pragma unroll
  for (int n = 0; n < kBlocks; n++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[n][e] = 0.f;
  m = -INFINITY;
  l = off = 0.f;
  large = false;
  if (first < stop) load_tile(first, first & 1u);
  settle();
  for (uint32_t t = first; t < stop; t++) {
    const uint32_t j0 = t * kKeys, buf = t & 1u;
    const uint8_t* tile = tiles + 2 * kTile * buf;
    if (t + 1 < stop) load_tile(t + 1, buf ^ 1u);
    // (a wave whose queries all end before this tile has nothing to do in it)
    if ((int)j0 < open + 31) {
      f32x16 s[2];
#pragma unroll
      for (uint32_t n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[n][e] = 0.f;
      const auto key = [&](uint32_t d, uint32_t n) {
        const uint32_t r = 32 * n + lq;
        return *reinterpret_cast<const u32x4*>(tile + r * kRow + 16 * ((2 * d + lh) ^ kswz(r)));
      };
      u32x4 ka[3][2];
#pragma unroll
      for (uint32_t d = 0; d < 2; d++)
#pragma unroll
        for (uint32_t n = 0; n < 2; n++) ka[d][n] = key(d, n);
#pragma unroll
      for (uint32_t d = 0; d < (uint32_t)kSteps; d++) {
        if (d + 2 < (uint32_t)kSteps)
#pragma unroll
          for (uint32_t n = 0; n < 2; n++) ka[(d + 2) % 3][n] = key(d + 2, n);
#pragma unroll
        for (uint32_t n = 0; n < 2; n++) s[n] = multiply<T>(ka[d % 3][n], qf[d], s[n]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (uint32_t d = 0; d < (uint32_t)kSteps; d++) {
        if (d + 2 < (uint32_t)kSteps) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      }
      // register e of block n is key j0 + 32 n + 8 (e / 4) + 4 lh + e % 4
      const bool masked = (int)(j0 + kKeys) > open;
      if (masked) {
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 16; e++)
            if ((int)(j0 + 32 * n + 8 * (e / 4) + 4 * lh + e % 4) >= limit) s[n][e] = -INFINITY;
      }
      // The weights are relative to a max that may lag 2^kLag behind: it is taken up, and the accumulators
      // rescaled, only where a score passes that (or is a query's first).
      float top = m;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, s[n][e]);
      if (__builtin_amdgcn_ballot_w64((top - m) * a.scale > kLag) != 0) {
        top = max_of_query(top);
        const float alpha = top > m ? __builtin_amdgcn_exp2f((m - top) * a.scale) : 1.f;
        l *= alpha;
#pragma unroll
        for (int n = 0; n < kBlocks; n++) o[n] *= alpha;
        m = top;
        off = m == -INFINITY ? 0.f : m * a.scale;
        large = __builtin_amdgcn_ballot_w64(fabsf(off) > kLargest) != 0;
        if (large) off = 0.f;
      }
      // (past kLargest the max's own rounding would put weights out of range: there it is taken from the scores
      // instead)
      if (large) {
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 16; e++) s[n][e] -= from;
      }
      const auto add_values = [&](auto cleaned) {
        const auto weights = [&](int k) {  // of keys 16 k .. +16 of the tile, as far as this lane has them
          u32x4 p;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[k / 2][8 * (k & 1) + e], a.scale, -off));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[k / 2][8 * (k & 1) + e + 1], a.scale, -off));
            l += x + y;
            p[e / 2] = pack<T>(x, y);
          }
          return p;
        };
        const auto value = [&](int k, int b) {
          const uint8_t* at = tile + vat[b] + 16 * k * kRow;
          const egd::s16x4 lo = egd::lds_read_transposed(at), hi = egd::lds_read_transposed(at + 8 * kRow);
          u32x4 va = __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (decltype(cleaned)::value) clean<T>(va);
          return va;
        };
        u32x4 va[2][kBlocks], p[2];
        p[0] = weights(0);
#pragma unroll
        for (int b = 0; b < kBlocks; b++) va[0][b] = value(0, b);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if (k < 3) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++) va[(k + 1) & 1][b] = value(k + 1, b);
            p[(k + 1) & 1] = weights(k + 1);
          }
#pragma unroll
          for (int b = 0; b < kBlocks; b++) o[b] = multiply<T>(va[k & 1][b], p[k & 1], o[b]);
        }
      };
      if (!decltype(careful)::value || !masked) {
        add_values(std::false_type{});
      } else if constexpr (decltype(careful)::value) {
        add_values(std::true_type{});
        for (uint32_t j = 0; j < kKeys && (int)(j0 + j) < limit && j0 + j < key_end; j++) {
          const T* row = reinterpret_cast<const T*>(vbase) + (size_t)(j0 + j) * a.v_stride;
#pragma unroll
          for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const float v = eg_kv4::to_f32(row[32 * n + 8 * (e / 4) + 4 * lh + e % 4]);
              if (!(fabsf(v) < INFINITY)) o[n][e] += v;
            }
        }
      }
    }
    settle();
  }

  l += __shfl_xor(l, 32, 64);
  };
  run(std::false_type{});
  // A masked weight is 0, but 0 times an infinity or NaN in V is NaN: where a result is not finite the
  // workgroup goes through its keys again, with care in the tiles that have masked ones.
  float check = 0.f;
#pragma unroll
  for (int n = 0; n < kBlocks; n++)
#pragma unroll
    for (int e = 0; e < 16; e++) check = fmaf(o[n][e], 0.f, check);
  const bool again = __builtin_amdgcn_ballot_w64(query < nq && check != 0.f) != 0;
  uint32_t* votes = reinterpret_cast<uint32_t*>(tiles);  // (the tiles have been read)
  votes[wave] = again;
  __syncthreads();
  if (votes[0] | votes[1] | votes[2] | votes[3]) {
    __syncthreads();
    run(std::true_type{});
  }
  if (query >= nq) return;
  if constexpr (kSplit) {
    const size_t row = ((size_t)(q_begin + query) * a.heads + h) * a.splits + w.split;
#pragma unroll
    for (int n = 0; n < kBlocks; n++)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(a.o + row * D + 32 * n + 8 * (e / 4) + 4 * lh) =
            make_float4(o[n][e], o[n][e + 1], o[n][e + 2], o[n][e + 3]);
    if (lh == 0) *reinterpret_cast<float2*>(a.ml + 2 * row) = make_float2(m * a.scale, l);
    return;
  }
  const float r = limit > 0 ? 1.0f / l : 0.f;  // (no key seen: zeros)
  TO* out = static_cast<TO*>(a.out) + (size_t)(q_begin + query) * a.out_stride + h * D;
#pragma unroll
  for (int n = 0; n < kBlocks; n++)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      TO* to = out + 32 * n + 8 * (e / 4) + 4 * lh;
      if constexpr (std::is_same<TO, float>::value)
        *reinterpret_cast<float4*>(to) = make_float4(o[n][e] * r, o[n][e + 1] * r, o[n][e + 2] * r, o[n][e + 3] * r);
      else
        *reinterpret_cast<uint2*>(to) = make_uint2(pack<TO>(o[n][e] * r, o[n][e + 1] * r), pack<TO>(o[n][e + 2] * r, o[n][e + 3] * r));
    }
}

// The splits of a query block joined, in their order: 4 dims of a query a thread, kThreads / (D / 4) queries a
// workgroup.
template <int D, class T, class TO>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  constexpr uint32_t kEach = kThreads / (D / 4), kParts = kQueries / kEach;
  Args all = a;
  all.splits = 1;
  Work w;
  if (!find_work(all, blockIdx.x / kParts, w)) return;
  const uint32_t per_split = (w.per_split + a.splits - 1) / a.splits;  // (of one split: all the sequence's tiles)
  const uint32_t count = max(1u, per_split ? (w.stop + per_split - 1) / per_split : 1u);
  const uint32_t query = w.q0 + blockIdx.x % kParts * kEach + threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
  if (query < w.nq) {
    const size_t row = ((size_t)(w.q_begin + query) * a.heads + w.head) * a.splits;
    float top = -INFINITY;
    for (uint32_t c = 0; c < count; c++) top = fmaxf(top, a.ml[2 * (row + c)]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (uint32_t c = 0; c < count; c++) {
      const float2 ml = *reinterpret_cast<const float2*>(a.ml + 2 * (row + c));
      const float4 v = *reinterpret_cast<const float4*>(a.o + (row + c) * D + d);
      // (a split of which the query sees no key has nothing but zeros; its max, of none, is below all)
      const float f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
      sum = fmaf(f, ml.y, sum);
      acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
    }
    const float r = w.shift + (int)query > 0 ? 1.0f / sum : 0.f;
    TO* to = static_cast<TO*>(a.out) + (size_t)(w.q_begin + query) * a.out_stride + w.head * D + d;
    if constexpr (std::is_same<TO, float>::value)
      *reinterpret_cast<float4*>(to) = make_float4(acc.x * r, acc.y * r, acc.z * r, acc.w * r);
    else
      *reinterpret_cast<uint2*>(to) = make_uint2(pack<TO>(acc.x * r, acc.y * r), pack<TO>(acc.z * r, acc.w * r));
  }
}

}  // namespace

extern "C" int eg_attention_packed(eg_context* ctx, const void* q, const void* k, const void* v,
                                   const uint32_t* q_offsets, const uint32_t* k_offsets, void* out,
                                   const eg_attention_packed_dims* dims) {
  const char* op = "attention_packed";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const bool some = dims && dims->rows != 0 && dims->sequences != 0;
  if (!dims || (some && (!q || !q_offsets || !k_offsets || !out || (dims->key_rows != 0 && (!k || !v)))))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_attention_packed_dims& d = *dims;
  if (d.head_dim != 64 && d.head_dim != 128)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: head_dim %u is not supported (64, 128)", op, d.head_dim);
  if (d.kv_heads == 0 || d.heads == 0 || d.heads % d.kv_heads != 0 || d.heads > 65535)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: heads %u are not a multiple of kv_heads %u (at most 65535)", op, d.heads,
                    d.kv_heads);
  if (d.type != EG_ELEMENT_F16 && d.type != EG_ELEMENT_BF16)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: type %d (f16 or bf16)", op, d.type);
  if (d.out_type != d.type && d.out_type != EG_ELEMENT_F32)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: out_type %d (the type %d, or f32)", op, d.out_type, d.type);
  if (!(d.scale >= 0.f) || d.scale > 1e6f) return eg::fail(ctx, EG_ERR_INVALID, "%s: scale %g (0 to 1e6)", op, d.scale);
  const uint32_t width = d.heads * d.head_dim, kv_width = d.kv_heads * d.head_dim;
  Args a{q, k, v, out, q_offsets, k_offsets, d.sequences, d.rows, d.key_rows, d.heads, d.heads / d.kv_heads,
         d.q_stride ? d.q_stride : width, d.k_stride ? d.k_stride : kv_width, d.v_stride ? d.v_stride : kv_width,
         d.out_stride ? d.out_stride : width,
         d.kv_heads <= 4 && d.kv_heads != 3 ? 8 / d.kv_heads : 0, 1, 0, (uint32_t)ctx->cu_count / 8, nullptr, nullptr,
         std::max((d.scale > 0.f ? d.scale : 1.0f / sqrtf((float)d.head_dim)) * kLog2e, 0x1p-126f)};
  if (a.q_stride < width || a.out_stride < width || a.k_stride < kv_width || a.v_stride < kv_width ||
      (a.q_stride | a.k_stride | a.v_stride | a.out_stride) % 8)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: strides %u, %u, %u, %u (multiples of 8, at least a row)", op, a.q_stride,
                    a.k_stride, a.v_stride, a.out_stride);
  if (a.k_stride > (1u << 23) || a.v_stride > (1u << 23))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: key strides %u, %u (at most 2^23 elements)", op, a.k_stride, a.v_stride);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15u)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q, k, v and out must be 16-byte aligned", op);
  if (d.sequences > (1u << 20))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences (at most 2^20)", op, d.sequences);
  if (d.rows >= (1u << 30) || d.key_rows >= (1u << 30))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows, %u key rows (under 2^30)", op, d.rows, d.key_rows);
  if (!some) return EG_OK;
  // at most this many query blocks, whatever the lengths
  const uint64_t blocks = (uint64_t)d.rows / kQueries + std::min<uint64_t>(d.sequences, d.rows);
  // (a kv head's items rounded up to its XCDs)
  const uint64_t items = a.xcds ? (blocks * a.group + a.xcds - 1) / a.xcds * 8 : blocks * d.heads;
  if (items >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows of %u heads over the grid limit", op, d.rows, d.heads);
  // Few query blocks leave the device idle over long keys: each block's keys are then split over workgroups, as
  // many as make two workgroups a CU, of at least kSplitTiles of a sequence's tiles. 14 / 2 heads of 64: 256
  // queries after 1792 rows 28.9 -> 15.7 us, twice 64 after 6000 75 -> 21.6 (of at least 8 tiles 23.0; of 4 the first
  // takes 16.6, and a prompt of 1024 18.8 for 15.9). Two splits, where no more fit, cost more in the join than they
  // gain: 4 of 500 after 2000 37.6 for 33.9. What stays: a workgroup is 128 queries of one head, so of 64 queries two
  // of its waves go through all keys for none, and every head of a kv head loads the same keys (twice 64 after 6000:
  // 21.3 us with 4.6 in the join, where the products they need take 1.8).
  const uint64_t resident = 2ull * ctx->cu_count;
  const uint64_t tiles = (uint64_t)d.key_rows / d.sequences / kKeys, row_bytes = (uint64_t)d.rows * d.heads * (d.head_dim + 2) * 4;
  const uint64_t splits = std::min({resident / (blocks * d.heads), tiles / kSplitTiles, (eg::kPartialsBytes - 64) / row_bytes});
  a.items = (uint32_t)((items + 7) / 8 * 8);
  if (splits >= kLeastSplits) {
    a.splits = (uint32_t)splits;
    a.ml = reinterpret_cast<float*>(eg::partials(ctx));
    a.o = a.ml + (((size_t)d.rows * d.heads * splits * 2 + 3) & ~(size_t)3);
  }
  const auto go = [&](auto t, auto to) {
    using T = decltype(t);
    using TO = decltype(to);
    const dim3 whole(a.items), threads(kThreads);
    if (a.splits > 1) {
      hipLaunchKernelGGL((d.head_dim == 64 ? packed_kernel<64, true, T, TO> : packed_kernel<128, true, T, TO>),
                         dim3(a.items * a.splits), threads, 0, ctx->stream, a);
      hipLaunchKernelGGL((d.head_dim == 64 ? join_kernel<64, T, TO> : join_kernel<128, T, TO>),
                         dim3(a.items * d.head_dim / 8), threads, 0, ctx->stream, a);
    } else {
      hipLaunchKernelGGL((d.head_dim == 64 ? packed_kernel<64, false, T, TO> : packed_kernel<128, false, T, TO>), whole,
                         threads, 0, ctx->stream, a);
    }
  };
  const eg_kv4::OnDevice on(ctx);
  if (d.type == EG_ELEMENT_F16) {
    if (d.out_type == EG_ELEMENT_F32) go(_Float16{}, float{});
    else go(_Float16{}, _Float16{});
  } else {
    if (d.out_type == EG_ELEMENT_F32) go(bf16{}, float{});
    else go(bf16{}, bf16{});
  }
  return eg::check_launch(ctx, op);
}

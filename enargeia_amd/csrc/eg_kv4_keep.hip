// Accepted rows of a speculative step moved together in the pages of the 4-bit cache (eg_kv4_keep_rows).
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256, kMostRows = 64;
constexpr uint32_t kNoRow = 0xFFFFFFFFu;

struct KeepArgs {
  const uint32_t *path, *counts, *offsets, *lengths;
  uint32_t* new_lengths;
  uint32_t layers, max_rows, each, blocks;  // each: (layer, kv head) pairs of a wave; blocks: workgroups of a sequence
  uint64_t layer_bytes;
};

// A wave per `each` (layer, kv head) of a sequence. All of a pair's rows are read before any is written: K words and
// scales into registers, V words (8 positions of a dim) into LDS, where each lane keeps those of its own dims and puts
// together the ones that rows go to. Which rows move is found once a workgroup. Bound by latency where the step is small:
// offsets, table, path, words (one of 16 rows, 24 layers, 2 heads of 64: 5 us); and by the partly used words of V where it is
// large: 64 of up to 32 rows, 32 layers, 8 heads of 128, 25 us for the 130 MB of words touched (39 MB of rows).
template <int D>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a, Pool pool) {
  constexpr uint32_t kGroups = D / 32, kWindow = kMostRows / 8 + 1, kLane = D / 64;  // kLane: dims a lane
  constexpr uint32_t kQuads = D / 32;                                               // 16-byte words of a K row
  constexpr uint32_t kRowsK = 64 / kQuads, kEachK = kMostRows / kRowsK;  // K rows a load; loads of 64 rows
  constexpr uint32_t kRowsS = 64 / (2 * kGroups), kEachS = kMostRows / kRowsS;
  typedef uint32_t dims __attribute__((ext_vector_type(kLane)));
  __shared__ uint32_t from[kMostRows], pages[4], moves[kMostRows], moved_of, used_of;
  __shared__ dims words_of[kThreads / 64][kWindow][64];
  const uint32_t seq = blockIdx.x / a.blocks, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = a.offsets[seq + 1] - a.offsets[seq], length = a.lengths[seq];
  const bool fits = n <= a.max_rows && n <= length;
  const uint32_t count = fits ? min(a.counts[seq], n) : 0;
  if (blockIdx.x % a.blocks == 0 && tid == 0) a.new_lengths[seq] = fits ? length - n + count : length;
  if (count == 0) return;
  const uint32_t base = length - n, shift = pool.page_shift, mask = (1u << shift) - 1u;
  if (wave == 0) {  // the rows that move: their places, and where they come from
    uint32_t j = lane < count ? a.path[(size_t)seq * a.max_rows + lane] : kNoRow;
    if (lane < 4) pages[lane] = pool.page_of(seq, ((base >> shift) + lane) << shift);
    __builtin_amdgcn_wave_barrier();
    if (j >= n || j == lane || pages[((base + j) >> shift) - (base >> shift)] >= pool.pages ||
        pages[((base + lane) >> shift) - (base >> shift)] >= pool.pages)
      j = kNoRow;
    from[lane] = j;
    const uint64_t moving = __ballot(j != kNoRow);
    if (j != kNoRow) moves[__builtin_popcountll(moving & ((1ull << lane) - 1u))] = lane;
    uint32_t used = 0;  // V words that rows come from or go to
#pragma unroll
    for (uint32_t b = 0; b < kWindow; b++) {
      const uint32_t w = (base >> 3) + b;
      if (__ballot(j != kNoRow && ((base + j) >> 3 == w || (base + lane) >> 3 == w)) != 0) used |= 1u << b;
    }
    if (lane == 0) {
      moved_of = (uint32_t)__builtin_popcountll(moving);
      used_of = used;
    }
  }
  __syncthreads();
  const uint32_t moved = __builtin_amdgcn_readfirstlane(moved_of), used = __builtin_amdgcn_readfirstlane(used_of);
  if (moved == 0) return;
  const auto page_at = [&](uint32_t slot) { return pages[(slot >> shift) - (base >> shift)]; };
  const Layout at = layout<D>(1u << shift);
  dims(*words)[64] = words_of[wave];
  const uint32_t first = base >> 3;
  const uint32_t my_to = moves[lane], my_from = from[lane < moved ? my_to : 0];  // of the lane's move
  const auto to_of = [&](uint32_t m) { return (uint32_t)__builtin_amdgcn_readlane((int)my_to, (int)m); };
  const auto from_of = [&](uint32_t m) { return (uint32_t)__builtin_amdgcn_readlane((int)my_from, (int)m); };
  const uint32_t pairs = a.layers * pool.kv_heads, begin = (blockIdx.x % a.blocks * (kThreads / 64) + wave) * a.each;
  for (uint32_t pair = begin; pair < min(begin + a.each, pairs); pair++) {
    const uint32_t layer = pair / pool.kv_heads, head = pair % pool.kv_heads;
    uint8_t* const place = pool.base + layer * a.layer_bytes + (uint64_t)head * at.head_bytes;
    const auto block = [&](uint32_t slot) { return place + (uint64_t)page_at(slot) * pool.stride; };
    const auto k_at = [&](uint32_t slot) {
      return reinterpret_cast<egd::u32x4*>(block(slot)) + (slot & mask) * kQuads + lane % kQuads;
    };
    const auto s_at = [&](uint32_t slot) {  // K's groups, then V's
      return reinterpret_cast<uint16_t*>(block(slot) + at.k_scales) + ((size_t)(lane % (2 * kGroups)) << shift) + (slot & mask);
    };
    const auto v_at = [&](uint32_t b) {
      const uint32_t slot = max(8 * (first + b), base);
      return reinterpret_cast<dims*>(block(slot) + at.v_codes) + ((slot & mask) >> 3) * 64 + lane;
    };
    egd::u32x4 k[kEachK];
    uint16_t s[kEachS];
#pragma unroll
    for (uint32_t e = 0; e < kEachK; e++) {
      const uint32_t m = e * kRowsK + lane / kQuads;
      if (m < moved) k[e] = *k_at(base + from[moves[m]]);
    }
#pragma unroll
    for (uint32_t e = 0; e < kEachS; e++) {
      const uint32_t m = e * kRowsS + lane / (2 * kGroups);
      if (m < moved) s[e] = *s_at(base + from[moves[m]]);
    }
    for (uint32_t m = used; m != 0; m &= m - 1) {
      const uint32_t b = (uint32_t)__builtin_ctz(m);
      words[b][lane] = *v_at(b);
    }
    egd::drain();  // (rows may go to where others come from)
#pragma unroll
    for (uint32_t e = 0; e < kEachK; e++) {
      const uint32_t m = e * kRowsK + lane / kQuads;
      if (m < moved) *k_at(base + moves[m]) = k[e];
    }
#pragma unroll
    for (uint32_t e = 0; e < kEachS; e++) {
      const uint32_t m = e * kRowsS + lane / (2 * kGroups);
      if (m < moved) *s_at(base + moves[m]) = s[e];
    }
    // A target word's rows follow each other: it is put together, then written.
    for (uint32_t m = 0; m < moved;) {
      const uint32_t b = ((base + to_of(m)) >> 3) - first;
      dims w = words[b][lane];
      for (; m < moved && ((base + to_of(m)) >> 3) - first == b; m++) {
        const uint32_t slot = base + from_of(m), e = 4 * ((base + to_of(m)) & 7u);
        const dims c = (words[(slot >> 3) - first][lane] >> (4 * (slot & 7u))) & 15u;
        w = (w & ~(15u << e)) | (c << e);
      }
      *v_at(b) = w;
    }
  }
}

}  // namespace

extern "C" int eg_kv4_keep_rows(eg_context* ctx, const uint32_t* path, const uint32_t* counts, const uint32_t* offsets,
                                const uint32_t* lengths, const uint32_t* table, void* pool, uint32_t* new_lengths,
                                const eg_kv4_dims* dims, uint32_t layers, uint32_t max_rows) {
  const char* op = "kv4_keep_rows";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  const int st = eg_kv4::check_dims(ctx, op, dims, pool);
  if (st != EG_OK) return st;
  if (max_rows > kMostRows) return eg::fail(ctx, EG_ERR_RANGE, "%s: max_rows %u (at most %u)", op, max_rows, kMostRows);
  const uint64_t layer_bytes = eg_kv4::page_bytes(*dims);
  if (layers == 0 || layers > dims->page_stride / layer_bytes)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: %u layers of %llu bytes in pages of %llu", op, layers,
                    (unsigned long long)layer_bytes, (unsigned long long)dims->page_stride);
  if (dims->sequences != 0 && (!offsets || !lengths || !new_lengths || !counts || (max_rows != 0 && !path) ||
                               (dims->max_pages != 0 && !table)))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  if (dims->sequences == 0) return EG_OK;
  const uint64_t n = dims->sequences;  // (a sequence's workgroups read its length at any time)
  const Extent made = words(new_lengths, n), held{pool, dims->pages, dims->page_stride, layers * layer_bytes};
  for (const Extent& in : {words(lengths, n), words(counts, n), words(offsets, n + 1), words(path, n * max_rows),
                           words(table, n * dims->max_pages)}) {
    if (overlap(made, in)) return eg::fail(ctx, EG_ERR_INVALID, "%s: new_lengths lie in an input", op);
    if (overlap(held, in)) return eg::fail(ctx, EG_ERR_INVALID, "%s: an input lies in the pool", op);
  }
  if (overlap(made, held)) return eg::fail(ctx, EG_ERR_INVALID, "%s: new_lengths lie in the pool", op);
  // A pair a wave, more where that would be more waves than the device holds at once.
  const uint64_t pairs = (uint64_t)layers * dims->kv_heads, room = (uint64_t)ctx->cu_count * 32;
  const uint64_t each = std::max<uint64_t>(1, pairs * dims->sequences / room), waves = (pairs + each - 1) / each;
  const uint64_t blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
  if (pairs >= (1ull << 32) || blocks * dims->sequences >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences of %u layers over the grid limit", op, dims->sequences, layers);
  const KeepArgs a{path, counts, offsets, lengths, new_lengths, layers, max_rows, (uint32_t)each, (uint32_t)blocks, layer_bytes};
  const eg_kv4::Pool p = eg_kv4::pool_of(*dims, pool, table);
  const dim3 grid((uint32_t)(blocks * dims->sequences));
  const OnDevice on(ctx);
  if (dims->head_dim == 64) hipLaunchKernelGGL(keep_kernel<64>, grid, dim3(kThreads), 0, ctx->stream, a, p);
  else hipLaunchKernelGGL(keep_kernel<128>, grid, dim3(kThreads), 0, ctx->stream, a, p);
  return eg::check_launch(ctx, op);
}

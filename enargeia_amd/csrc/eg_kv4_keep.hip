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
  uint32_t layers, max_rows;
  uint64_t layer_bytes;
};

// A workgroup per (sequence, layer, kv head). All of a head's rows are read before any is written: K words and
// scales into registers, V words (8 positions of a dim) into LDS, where the ones that rows go to are put together.
// Bound by latency: the rows of a step are few.
template <int D>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a, Pool pool) {
  constexpr uint32_t kRowWords = D / 8, kGroups = D / 32, kWindow = kMostRows / 8 + 1;
  constexpr uint32_t kEachWord = kMostRows * kRowWords / kThreads, kScales = kMostRows * 2 * kGroups;
  constexpr uint32_t kEachScale = (kScales + kThreads - 1) / kThreads;
  __shared__ uint32_t from[kMostRows], pages[4], words[kWindow][D];
  uint32_t id = blockIdx.x;
  const uint32_t head = id % pool.kv_heads;
  id /= pool.kv_heads;
  const uint32_t layer = id % a.layers, seq = id / a.layers, tid = threadIdx.x;
  const uint32_t n = a.offsets[seq + 1] - a.offsets[seq], length = a.lengths[seq];
  const bool fits = n <= a.max_rows && n <= length;
  const uint32_t count = fits ? min(a.counts[seq], n) : 0;
  if (layer == 0 && head == 0 && tid == 0) a.new_lengths[seq] = fits ? length - n + count : length;
  if (count == 0) return;
  const uint32_t base = length - n, shift = pool.page_shift, mask = (1u << shift) - 1u;
  if (tid < 4) pages[tid] = pool.page_of(seq, ((base >> shift) + tid) << shift);
  __syncthreads();
  const auto page_at = [&](uint32_t slot) { return pages[(slot >> shift) - (base >> shift)]; };
  if (tid < kMostRows) {
    uint32_t j = kNoRow;
    if (tid < count) {
      j = a.path[(size_t)seq * a.max_rows + tid];
      if (j >= n || j == tid || page_at(base + j) >= pool.pages || page_at(base + tid) >= pool.pages) j = kNoRow;
    }
    from[tid] = j;
  }
  if (__syncthreads_or(tid < kMostRows && from[tid < kMostRows ? tid : 0] != kNoRow) == 0) return;
  const Layout at = layout<D>(1u << shift);
  uint8_t* const layer_base = pool.base + layer * a.layer_bytes;
  const auto block = [&](uint32_t slot) {
    return layer_base + (uint64_t)page_at(slot) * pool.stride + (uint64_t)head * at.head_bytes;
  };
  uint32_t k[kEachWord];
  uint16_t s[kEachScale];
  const auto scale_at = [&](uint32_t slot, uint32_t which) {  // which: K's groups, then V's
    return reinterpret_cast<uint16_t*>(block(slot) + at.k_scales) + ((size_t)which << shift) + (slot & mask);
  };
#pragma unroll
  for (uint32_t e = 0; e < kEachWord; e++) {
    const uint32_t i = (e * kThreads + tid) / kRowWords, j = from[i];
    if (j != kNoRow)
      k[e] = reinterpret_cast<const uint32_t*>(block(base + j))[((base + j) & mask) * kRowWords + tid % kRowWords];
  }
#pragma unroll
  for (uint32_t e = 0; e < kEachScale; e++) {
    const uint32_t x = e * kThreads + tid, i = x / (2 * kGroups), j = x < kScales ? from[i] : kNoRow;
    if (j != kNoRow) s[e] = *scale_at(base + j, x % (2 * kGroups));
  }
  const uint32_t first = base >> 3, last = (base + n - 1) >> 3;
  const auto word_at = [&](uint32_t b, uint32_t d) {
    return reinterpret_cast<uint32_t*>(block(8 * b < base ? base : 8 * b) + at.v_codes) + ((8 * b & mask) >> 3) * D + d;
  };
  for (uint32_t x = tid; x < (last - first + 1) * D; x += kThreads) {
    const uint32_t b = first + x / D;
    if (page_at(8 * b < base ? base : 8 * b) < pool.pages) words[b - first][x % D] = *word_at(b, x % D);
  }
  __syncthreads();
#pragma unroll
  for (uint32_t e = 0; e < kEachWord; e++) {
    const uint32_t i = (e * kThreads + tid) / kRowWords;
    if (from[i] != kNoRow)
      reinterpret_cast<uint32_t*>(block(base + i))[((base + i) & mask) * kRowWords + tid % kRowWords] = k[e];
  }
#pragma unroll
  for (uint32_t e = 0; e < kEachScale; e++) {
    const uint32_t x = e * kThreads + tid, i = x / (2 * kGroups);
    if (x < kScales && from[i] != kNoRow) *scale_at(base + i, x % (2 * kGroups)) = s[e];
  }
  for (uint32_t x = tid; x < (last - first + 1) * D; x += kThreads) {
    const uint32_t b = first + x / D, d = x % D;
    if (8 * b >= base + count || page_at(8 * b < base ? base : 8 * b) >= pool.pages) continue;
    uint32_t w = words[b - first][d], moved = 0;
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) {
      const uint32_t i = 8 * b + e - base;  // (before the first row: past count)
      if (i >= count || from[i] == kNoRow) continue;
      const uint32_t slot = base + from[i];
      const uint32_t c = (words[(slot >> 3) - first][d] >> (4 * (slot & 7u))) & 15u;
      w = (w & ~(15u << (4 * e))) | (c << (4 * e));
      moved = 1;
    }
    if (moved) *word_at(b, d) = w;
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
  const uint64_t blocks = (uint64_t)dims->sequences * layers;
  if (blocks >= (1ull << 31) / kThreads / dims->kv_heads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences of %u layers over the grid limit", op, dims->sequences, layers);
  const KeepArgs a{path, counts, offsets, lengths, new_lengths, layers, max_rows, layer_bytes};
  const eg_kv4::Pool p = eg_kv4::pool_of(*dims, pool, table);
  const dim3 grid((uint32_t)blocks * dims->kv_heads);
  const OnDevice on(ctx);
  if (dims->head_dim == 64) hipLaunchKernelGGL(keep_kernel<64>, grid, dim3(kThreads), 0, ctx->stream, a, p);
  else hipLaunchKernelGGL(keep_kernel<128>, grid, dim3(kThreads), 0, ctx->stream, a, p);
  return eg::check_launch(ctx, op);
}

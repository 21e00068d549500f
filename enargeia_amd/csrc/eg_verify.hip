// Drafted tokens against the target's probabilities (eg_verify_drafts).
//
// Three quantities of a row of logits decide: its largest, Z = sum 2^((l - largest) log2(e) / temperature), and
// the running sum that the next token is drawn by. All three come from partials per chunk of kChunk ids, made for
// all rows at once by verify_stats: that pass reads the logits, and is what bounds the operator. Which rows the branch
// goes through then takes single logits (verify_walk, a workgroup per sequence), and the draw reads one chunk
// of one row again: the one in which the running sum passes the target. After a rejection by draft probabilities
// the sums are of max(p - q, 0), so that row's chunks are summed once more: there a workgroup per chunk finds the
// branch by itself, and sums its chunk (verify_draw then has the sums).
//
// Sums and exponentials are f64: of 151,936 running sums some lie within f32's rounding of the drawn target in one
// draw of a hundred, within these in none of 10^6. f64 vector instructions run at f32's rate, and an exponential is
// 15 of them. (The largest is taken from a logit before the product with the scale: the difference is exact, where products
// of large logits leave their rounding.)
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256, kMostRows = 64, kEach = 16, kChunk = kThreads * kEach;
constexpr uint32_t kWalkThreads = 512, kWalkEach = kChunk / kWalkThreads;
constexpr uint32_t kMostVocab = 1u << 20;  // 256 chunks: a thread each
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct VerifyArgs {
  const void* logits;
  const uint32_t *tokens, *offsets, *parents;
  const float *draft, *accept, *draws, *temperatures;
  uint32_t *path, *counts, *next;
  struct Stats* stats;       // [row][chunk]
  struct Residual* residual; // [sequence]
  double* masses;            // [sequence][chunk] of the residual
  uint32_t sequences, rows, max_rows, vocab, chunks;
  uint64_t stride, draft_stride;
};

struct Stats {
  double sum;  // of 2^((l - reference(top)) scale)
  float top;
  uint32_t id;  // the lowest of `top` (0 where that is -inf)
};

// A sequence whose next token is drawn from max(p - q, 0) of a row.
struct Residual {
  double scale, total;  // total: Z
  uint32_t row;         // kNone: no such draw
  float reference;
};

// What a row's exponents are taken from: its largest, and 0 for a row of -inf alone (its sum is then 0).
__device__ __forceinline__ float reference(float top) { return top == -INFINITY ? 0.f : top; }

// 2^x for x <= 0, to 1.1e-12 of it: 2^k times the polynomial that has 2^r's values at the 9 Chebyshev points of
// |r| <= 1/2 (1 at r = 0 but for its rounding: whole powers are exact). x + 1.5 * 2^52 has k in its low bits. Below -1100: 0.
// (Not a number: something else; see `broken`.)
__device__ __forceinline__ double exp2_of(double x) {
  constexpr double kRound = 0x1.8p52;
  x = fmax(x, -1100.0);
  const double t = x + kRound, r = x - (t - kRound);
  double p = 1.3255224878668817e-06;
  p = fma(p, r, 1.5310079402249296e-05);
  p = fma(p, r, 0.00015403455852453838);
  p = fma(p, r, 0.0013333450568000645);
  p = fma(p, r, 0.009618129159402558);
  p = fma(p, r, 0.05550410941205933);
  p = fma(p, r, 0.2402265069581299);
  p = fma(p, r, 0.6931471805459335);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)__double2loint(t));
}

// A logit of which there are no probabilities.
__device__ __forceinline__ bool broken(float l) { return !(l < INFINITY); }

__device__ __forceinline__ double scale_of(float temperature) { return 1.4426950408889634 / (double)temperature; }

// A sequence's temperature, 0 for greedy.
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, uint32_t seq) {
  const float t = a.temperatures ? a.temperatures[seq] : 0.f;
  return t > 0.f ? t : 0.f;
}

template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Several {
  T v[N];
};

// Ids i .. i + N of a row, `fill` past its end. (In one: a load behind a condition of its own waits for itself.)
template <int N, class T>
__device__ __forceinline__ void load_ids(const T* x, uint32_t i, uint32_t vocab, float fill, float (&v)[N]) {
  if (i + N <= vocab) {
    const Several<T, N> s = *reinterpret_cast<const Several<T, N>*>(x + i);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = to_f32(s.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = i + e < vocab ? to_f32(x[i + e]) : fill;
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Sum over a workgroup of kWaves waves, in every thread.
template <int kWaves>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kWaves];
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = part[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) sum += part[w];
  return sum;
}

// The sum over the threads before this one of a verify_walk's workgroup; `total` over all.
__device__ __forceinline__ double block_before(double v, double& total) {
  constexpr uint32_t kWaves = kWalkThreads / 64;
  __shared__ double part[kWaves];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  double run = v;
#pragma unroll
  for (uint32_t m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(run, m, 64);
    if (lane >= m) run += o;
  }
  __syncthreads();
  if (lane == 63) part[wave] = run;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; w++) {
    if (w == wave) before = total;
    total += part[w];
  }
  const double o = __shfl_up(run, 1, 64);
  return lane == 0 ? before : before + o;
}

// A workgroup per (chunk, row): its largest logit and its sum.
template <class T>
__global__ __launch_bounds__(256) void verify_stats(VerifyArgs a) {
  constexpr uint32_t kWide = 16 / sizeof(T);
  const uint32_t row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + (uint64_t)row * a.stride;
  const uint32_t begin = chunk * kChunk;
  float v[kEach];  // (under way while the row's sequence is found)
#pragma unroll
  for (uint32_t j = 0; j < kEach / kWide; j++) {
    float w[kWide];
    load_ids<kWide>(x, begin + kWide * (j * kThreads + tid), a.vocab, -INFINITY, w);
#pragma unroll
    for (uint32_t e = 0; e < kWide; e++) v[j * kWide + e] = w[e];
  }
  uint32_t seq, first, end;
  if (!find_sequence(a.offsets, a.sequences, row, seq, first, end)) return;
  const float temperature = temperature_of(a, seq);
  float top = -INFINITY;
  uint32_t id = 0;
#pragma unroll
  for (uint32_t j = 0; j < kEach; j++)
    if (v[j] > top) {
      top = v[j];
      id = begin + kWide * ((j / kWide) * kThreads + tid) + j % kWide;
    }
  egd::team_argmax<64>(top, id);
  __shared__ float tops[4];
  __shared__ uint32_t ids[4];
  if ((tid & 63u) == 0) {
    tops[tid >> 6] = top;
    ids[tid >> 6] = id;
  }
  __syncthreads();
  top = tops[0];
  id = ids[0];
#pragma unroll
  for (uint32_t w = 1; w < 4; w++)
    if (egd::better(tops[w], ids[w], top, id)) {
      top = tops[w];
      id = ids[w];
    }
  double sum = 0.0;
  if (temperature > 0.f) {
    const double scale = scale_of(temperature), from = reference(top);
    bool bad = false;
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) {
      sum += exp2_of(((double)v[j] - from) * scale);
      bad |= broken(v[j]);
    }
    sum = block_sum<4>(bad ? (double)NAN : sum);
  }
  if (tid == 0) a.stats[(uint64_t)row * a.chunks + chunk] = Stats{sum, top, id};
}

// Times a chunk's sum: from its reference to the row's.
__device__ __forceinline__ double rescaled(const Stats& s, float top, double scale) {
  return s.top == -INFINITY ? s.sum : s.sum * exp2_of(((double)s.top - (double)reference(top)) * scale);
}

// Of the threads that have a `first` (not kNone) the lowest one's; where there is none, of those that have a `last` the highest
// one's, or 0. Every thread gets it. (By ballots: an atomic minimum in LDS takes a wave's lanes one after another.)
__device__ __forceinline__ uint32_t first_or_last(uint32_t first, uint32_t last) {
  constexpr uint32_t kWaves = kWalkThreads / 64;
  __shared__ uint32_t firsts[kWaves], lasts[kWaves];
  const uint64_t have_first = __ballot(first != kNone), have_last = __ballot(last != kNone);
  if ((threadIdx.x & 63u) == 0) firsts[threadIdx.x >> 6] = lasts[threadIdx.x >> 6] = kNone;
  if (have_first != 0 && (threadIdx.x & 63u) == (uint32_t)__builtin_ctzll(have_first)) firsts[threadIdx.x >> 6] = first;
  if (have_last != 0 && (threadIdx.x & 63u) == 63u - (uint32_t)__builtin_clzll(have_last)) lasts[threadIdx.x >> 6] = last;
  __syncthreads();
  uint32_t got = kNone, highest = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; w++) {
    if (got == kNone) got = firsts[w];
    if (lasts[w] != kNone) highest = lasts[w];
  }
  __syncthreads();
  return got != kNone ? got : highest;
}

// The chunk in which the running sum of `mass` (a chunk per thread) exceeds draw * the whole sum, and what of that
// lies before it. False: there is nothing to draw from.
__device__ __forceinline__ bool find_chunk(double mass, float draw, uint32_t& chunk, double& target) {
  __shared__ double rest;
  double total;
  const double before = block_before(mass, total);
  if (!(total > 0.0) || !(total < (double)INFINITY)) return false;  // (the same in every thread)
  const double whole = (double)draw * total;
  chunk = first_or_last(mass > 0.0 && before + mass > whole ? threadIdx.x : kNone, mass > 0.0 ? threadIdx.x : kNone);
  if (threadIdx.x == chunk) rest = whole - before;
  __syncthreads();
  target = rest;
  return true;
}

// The lowest id at which the running sum of the chunk's values, from its beginning on, exceeds `target`; the last one
// of a value above 0 where rounding leaves none. values(first id, out) gives a thread's kWalkEach. Every thread gets it.
template <class F>
__device__ __forceinline__ uint32_t find_in_chunk(uint32_t chunk, double target, F&& values) {
  const uint32_t begin = chunk * kChunk + threadIdx.x * kWalkEach;
  double e[kWalkEach], sum = 0.0;
  values(begin, e);
  uint32_t last = kNone, hit = kNone;
#pragma unroll
  for (uint32_t j = 0; j < kWalkEach; j++) {
    sum += e[j];
    if (e[j] > 0.0) last = begin + j;
  }
  double total, run = block_before(sum, total);
#pragma unroll
  for (uint32_t j = 0; j < kWalkEach; j++) {
    run += e[j];
    if (e[j] > 0.0 && run > target && hit == kNone) hit = begin + j;
  }
  return first_or_last(hit, last);
}

// max(p - q, 0) of ids i .. of a sequence's last accepted row.
template <class T, int N>
__device__ __forceinline__ void left_over(const VerifyArgs& a, const Residual& r, uint32_t i, double (&e)[N]) {
  const T* x = static_cast<const T*>(a.logits) + (uint64_t)r.row * a.stride;
  const float* q = a.draft + (uint64_t)r.row * a.draft_stride;
  const double from = r.reference, to = 1.0 / r.total;
  float l[N], d[N];
  load_ids<N>(x, i, a.vocab, -INFINITY, l);
  load_ids<N>(q, i, a.vocab, 0.f, d);
#pragma unroll
  for (int j = 0; j < N; j++) e[j] = fmax(exp2_of(((double)l[j] - from) * r.scale) * to - (double)d[j], 0.0);
}

// A workgroup per sequence: its rows' sums from their chunks', the branch, and the next token. With draft
// probabilities (kDraft) one per (chunk, sequence): the first of them writes what that finds, and where the draw is from
// max(p - q, 0), each sums its chunk of that, for the launch after this one. A chain of dependent reads bounds it: offsets;
// rows and sums; single logits; the chunk.
template <bool kDraft, class T>
__global__ __launch_bounds__(kWalkThreads) void verify_walk(VerifyArgs a) {
  __shared__ float top_of[kMostRows], accept_of[kMostRows], q_of[kMostRows];
  __shared__ double sum_of[kMostRows], value_of[kMostRows];  // value_of: of a row's token where it was drafted
  __shared__ uint32_t id_of[kMostRows], token_of[kMostRows], path_of[kMostRows];
  __shared__ uint32_t count_of, row_of;
  __shared__ uint64_t rejected_of;  // rows, of the last row's children
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const bool writes = !kDraft || blockIdx.x == 0;
  const uint32_t first = a.offsets[seq], end = a.offsets[seq + 1], n = end - first;
  if (n == 0 || n > a.max_rows || first > end || end > a.rows) {
    if (!writes) return;
    if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = kNone;
    if (tid == 0) {
      a.counts[seq] = 0;
      a.next[seq] = kNone;
      if (kDraft) a.residual[seq].row = kNone;
    }
    return;
  }
  const float temperature = temperature_of(a, seq);
  const bool greedy = !(temperature > 0.f);
  const double scale = greedy ? 0.0 : scale_of(temperature);
  const T* logits = static_cast<const T*>(a.logits) + (uint64_t)first * a.stride;
  const Stats* stats = a.stats + (uint64_t)first * a.chunks;
  // The first wave has a row a lane: its parent, its token, and that token's logit and q at the parent, all under way
  // while the rows' sums are put together.
  Stats s[4];  // (256 chunks at most)
  const auto load_stats = [&](uint32_t r) {
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      const uint32_t c = lane + 64 * k;
      s[k] = Stats{0.0, -INFINITY, 0};
      if (c < a.chunks) s[k] = stats[(uint64_t)r * a.chunks + c];
    }
  };
  uint32_t parent = kNone, token = kNone;
  float logit = -INFINITY, q = 0.f, accept = 0.f;
  if (wave == 0) {
    const uint32_t mine = first + min(lane, n - 1);
    uint32_t p = lane - 1;
    if (a.parents) p = a.parents[mine];
    token = a.tokens[mine];
    if (!greedy) accept = a.accept[mine];
    load_stats(0);
    if (lane < n && p < lane) parent = p;
    if (lane >= n) token = kNone;
    if (!greedy) {
      const bool has = parent != kNone && token < a.vocab;
      const uint64_t from = has ? parent : 0, id = has ? token : 0;
      const float l = to_f32(logits[from * a.stride + id]);
      if (kDraft) q = a.draft[(first + from) * a.draft_stride + id];
      if (has) logit = l;
      else q = 0.f;
    }
  }
  for (uint32_t r = wave; r < n; r += kWalkThreads / 64) {
    float top = -INFINITY;
    uint32_t id = 0;
    if (r != 0) load_stats(r);
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
      if (egd::better(s[k].top, s[k].id, top, id)) {
        top = s[k].top;
        id = s[k].id;
      }
    egd::team_argmax<64>(top, id);
    double sum = 0.0;
    if (!greedy) {
#pragma unroll
      for (uint32_t k = 0; k < 4; k++)
        if (64 * k < a.chunks) sum += rescaled(s[k], top, scale);
      sum = wave_sum(sum);
    }
    if (lane == 0) {
      top_of[r] = top;
      id_of[r] = id;
      sum_of[r] = sum;
    }
  }
  __syncthreads();
  if (wave == 0) {  // (the whole wave takes the same steps)
    token_of[lane] = token;
    accept_of[lane] = accept;
    q_of[lane] = q;
    value_of[lane] = parent == kNone ? 0.0 : exp2_of(((double)logit - (double)reference(top_of[parent])) * scale);
    if (lane == 0) path_of[0] = 0;
    uint32_t at = 0, count = 1;
    uint64_t rejected = 0;
    for (;;) {
      uint64_t children = __ballot(parent == at);
      uint32_t to = kNone;
      double left = sum_of[at];
      rejected = 0;
      while (children != 0) {
        const uint32_t r = (uint32_t)__builtin_ctzll(children), x = token_of[r];
        children &= children - 1;
        bool ok;
        if (greedy) {
          ok = x == id_of[at];
        } else if (kDraft) {
          ok = (double)accept_of[r] * (double)q_of[r] * left < value_of[r];
        } else {
          const bool again = (__ballot(token == x) & rejected) != 0;
          ok = !again && (double)accept_of[r] * left < value_of[r];
          if (!ok && !again) left -= value_of[r];
        }
        if (ok) {
          to = r;
          break;
        }
        rejected |= 1ull << r;
      }
      if (to == kNone) break;
      at = to;
      if (lane == 0) path_of[count] = at;
      count++;
    }
    if (lane == 0) {
      count_of = count;
      row_of = at;
      rejected_of = rejected;
    }
  }
  __syncthreads();
  const uint32_t count = count_of, at = row_of;
  const uint64_t rejected = rejected_of;
  const double total = sum_of[at];
  const bool draws = !greedy && total > 0.0 && total < (double)INFINITY, from_rest = kDraft && draws && rejected != 0;
  if (writes) {
    if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = tid < count ? path_of[tid] : kNone;
    if (tid == 0) {
      a.counts[seq] = count;
      a.next[seq] = id_of[at];  // (unless one is drawn)
      if (kDraft) a.residual[seq] = Residual{scale, total, from_rest ? first + at : kNone, reference(top_of[at])};
    }
  }
  if (from_rest) {
    const Residual r{scale, total, first + at, reference(top_of[at])};
    double e[kWalkEach], sum = 0.0;
    left_over<T>(a, r, blockIdx.x * kChunk + tid * kWalkEach, e);
#pragma unroll
    for (uint32_t j = 0; j < kWalkEach; j++) sum += e[j];
    sum = block_sum<kWalkThreads / 64>(sum);
    if (tid == 0) a.masses[(uint64_t)seq * a.chunks + blockIdx.x] = sum;
    return;
  }
  if (!writes || !draws) return;
  double mass = 0.0;
  if (tid < a.chunks) {
    mass = rescaled(stats[(uint64_t)at * a.chunks + tid], top_of[at], scale);
    uint64_t seen = 0;  // (of a token that several rejected rows hold the first one counts)
    for (uint64_t m = rejected; m != 0; m &= m - 1) {
      const uint32_t r = (uint32_t)__builtin_ctzll(m);
      bool again = false;
      for (uint64_t o = seen; o != 0; o &= o - 1) again |= token_of[__builtin_ctzll(o)] == token_of[r];
      seen |= 1ull << r;
      if (!again && token_of[r] / kChunk == tid) mass -= value_of[r];
    }
    mass = fmax(mass, 0.0);
  }
  uint32_t chunk;
  double target;
  if (!find_chunk(mass, a.draws[seq], chunk, target)) return;
  const T* x = logits + at * a.stride;
  const double from = reference(top_of[at]);
  const uint32_t id = find_in_chunk(chunk, target, [&](uint32_t i, double (&e)[kWalkEach]) {
    float l[kWalkEach];
    load_ids<kWalkEach>(x, i, a.vocab, -INFINITY, l);
#pragma unroll
    for (uint32_t j = 0; j < kWalkEach; j++) e[j] = exp2_of(((double)l[j] - from) * scale);
    for (uint64_t m = rejected; m != 0; m &= m - 1) {
      const uint32_t gone = token_of[__builtin_ctzll(m)] - i;
#pragma unroll
      for (uint32_t j = 0; j < kWalkEach; j++)
        if (j == gone) e[j] = 0.0;
    }
  });
  if (tid == 0) a.next[seq] = id;
}

template <class T>
__global__ __launch_bounds__(kWalkThreads) void verify_draw(VerifyArgs a) {
  const uint32_t seq = blockIdx.x, tid = threadIdx.x;
  const Residual r = a.residual[seq];
  if (r.row == kNone) return;
  const double mass = tid < a.chunks ? a.masses[(uint64_t)seq * a.chunks + tid] : 0.0;
  uint32_t chunk;
  double target;
  if (!find_chunk(mass, a.draws[seq], chunk, target)) return;  // (p and q leave nothing)
  const uint32_t id = find_in_chunk(chunk, target, [&](uint32_t i, double (&e)[kWalkEach]) { left_over<T>(a, r, i, e); });
  if (tid == 0) a.next[seq] = id;
}

}  // namespace

extern "C" int eg_verify_drafts(eg_context* ctx, const void* logits, const uint32_t* tokens, const uint32_t* offsets,
                                const uint32_t* parents, const float* draft, const float* accept, const float* draws,
                                const float* temperatures, uint32_t* path, uint32_t* counts, uint32_t* next,
                                const eg_verify_dims* dims) {
  const char* op = "verify_drafts";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  if (!dims) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_verify_dims& d = *dims;
  if (!known_type(d.type)) return eg::fail(ctx, EG_ERR_INVALID, "%s: type %d (eg_element)", op, d.type);
  if (d.max_rows > kMostRows) return eg::fail(ctx, EG_ERR_RANGE, "%s: max_rows %u (at most %u)", op, d.max_rows, kMostRows);
  if (d.vocab == 0 || d.vocab > kMostVocab)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: vocab %u (1 to %u)", op, d.vocab, kMostVocab);
  if (draft && parents)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: draft probabilities go with chains (parents is not NULL)", op);
  VerifyArgs a{};
  a.stride = d.logits_stride ? d.logits_stride : d.vocab;
  a.draft_stride = d.draft_stride ? d.draft_stride : d.vocab;
  if (a.stride < d.vocab || a.draft_stride < d.vocab)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: strides %u, %u (at least vocab %u)", op, d.logits_stride, d.draft_stride,
                    d.vocab);
  if (d.sequences == 0) return EG_OK;
  if (!offsets || !counts || !next || (d.max_rows != 0 && !path) || (d.rows != 0 && (!logits || !tokens)) ||
      (temperatures && ((d.rows != 0 && !accept) || !draws)))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  if ((reinterpret_cast<uintptr_t>(logits) % (d.type == EG_ELEMENT_F32 ? 4 : 2)) != 0)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: logits are not aligned to their type", op);
  a.chunks = (d.vocab + kChunk - 1) / kChunk;
  const uint64_t stats = (uint64_t)d.rows * a.chunks * sizeof(Stats);
  const uint64_t residual = draft ? (uint64_t)d.sequences * (sizeof(Residual) + a.chunks * sizeof(double)) : 0;
  if (stats + residual > eg::kPartialsBytes || d.rows > 65535 || d.sequences > 65535)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences, %u rows of %u ids over the workspace or the grid limit", op, d.sequences, d.rows,
                    d.vocab);
  a.logits = logits;
  a.tokens = tokens;
  a.offsets = offsets;
  a.parents = parents;
  a.draft = draft;
  a.accept = accept;
  a.draws = draws;
  a.temperatures = temperatures;
  a.path = path;
  a.counts = counts;
  a.next = next;
  uint8_t* at = eg::partials(ctx);
  a.stats = reinterpret_cast<Stats*>(at);
  a.residual = reinterpret_cast<Residual*>(at + stats);
  a.masses = reinterpret_cast<double*>(at + stats + (uint64_t)d.sequences * sizeof(Residual));
  a.sequences = d.sequences;
  a.rows = d.rows;
  a.max_rows = d.max_rows;
  a.vocab = d.vocab;
  const OnDevice on(ctx);
  with_type(d.type, [&](auto t) {
    using T = decltype(t);
    const dim3 threads(kThreads);
    if (d.rows != 0) hipLaunchKernelGGL(verify_stats<T>, dim3(a.chunks, d.rows), threads, 0, ctx->stream, a);
    const dim3 walk(kWalkThreads);
    if (draft && temperatures) {
      hipLaunchKernelGGL((verify_walk<true, T>), dim3(a.chunks, d.sequences), walk, 0, ctx->stream, a);
      hipLaunchKernelGGL(verify_draw<T>, dim3(d.sequences), walk, 0, ctx->stream, a);
    } else {
      hipLaunchKernelGGL((verify_walk<false, T>), dim3(1, d.sequences), walk, 0, ctx->stream, a);
    }
  });
  return eg::check_launch(ctx, op);
}

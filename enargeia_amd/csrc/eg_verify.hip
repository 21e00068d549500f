// Drafted tokens against the target's probabilities (eg_verify_drafts).
//
// A row's largest logit and Z = sum 2^((l - largest) log2(e) / temperature) decide what is accepted. Both come from
// partials per chunk of kChunk ids, made for all rows at once by verify_stats: that pass reads the logits, and is what
// bounds the operator. Which rows the branch goes through then takes single logits. The next token's running sum goes
// over the branch's last row only: a workgroup per few chunks finds the branch by itself and sums its chunks (verify_walk),
// and the chunk in which the running sum passes the target is read once more (verify_draw; by the last workgroup to
// arrive instead of a launch of its own, both took 18.5 us for 9.2 and 4.9 with 16 sequences, and 19.5 for 14.4 and 5.7 with 48: one
// form for both, the one that never loses much).
//
// What is decided is decided in f64: of 151,936 running sums some lie within f32's rounding of the drawn target in one draw
// of a hundred, within these in none of 10^6. Exponentials in f64 are 15 f64 instructions, which over all rows take
// longer than reading them (48 sequences of up to 8 rows: 47 us, in f32 30.5): so Z is summed in f32 (kExact false),
// which is off by less than kMargin of it, and a row for which that could decide otherwise is summed again in f64 where it comes
// up. Draft probabilities are taken from p = e / Z itself, so their rows' Z are f64 from the start. (The largest is taken from a
// logit before the product with the scale: the difference is exact, where products of large logits leave their rounding.)
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256, kMostRows = 64, kEach = 16, kChunk = kThreads * kEach;
constexpr uint32_t kWalkThreads = 512, kWalkEach = kChunk / kWalkThreads;
constexpr uint32_t kMostVocab = 1u << 20;  // 256 chunks: a thread each
constexpr uint32_t kNone = 0xFFFFFFFFu;

// The error of a Z in f32, relative. Differences from the largest are rounded once, as is their product with the scale,
// itself rounded: 3 x 2^-24 of exponents that matter down to -30 (2^-30 of 2^20 ids are 2^-10 of Z, and their own errors no
// more than that times 1/8), so 6e-6 of an exponential, whose own error is 2^-23 and that of 16 added 2^-20.
constexpr double kMargin = 0x1p-16;
// Temperatures between which scales and exponents fit f32; beyond, Z is f64. (A difference of two logits that passes f32's
// largest is -inf there, its exponential 0: up to 2^120 that is an exponent under -2^8. A scale is a normal number to 2^126.)
constexpr float kColdest = 1e-30f, kHottest = 0x1p120f;
__device__ __forceinline__ bool fits_f32(float temperature) { return temperature >= kColdest && temperature <= kHottest; }

// What a sequence's next token is drawn from: a row's p, or (of > 0) max(p - q, 0).
struct Draw {
  double scale, of;     // of: Z, 0 for p
  uint64_t rejected;    // rows whose tokens p is without
  uint32_t row, first;  // row: kNone where none is drawn; first: the sequence's
  float reference;
};

struct VerifyArgs {
  const void* logits;
  const uint32_t *tokens, *offsets, *parents;
  const float *draft, *accept, *draws, *temperatures;
  uint32_t *path, *counts, *next;
  struct Stats* stats;  // [row][chunk]
  Draw* draw;           // [sequence]; NULL: all greedy
  double* masses;       // [sequence][chunk] of what is drawn from
  uint32_t sequences, rows, max_rows, vocab, chunks, together;  // together: chunks of a verify_walk's workgroup
  uint64_t stride, draft_stride;
};

struct Stats {
  double sum;  // of 2^((l - reference(top)) scale)
  float top;
  uint32_t id;  // the lowest of `top` (0 where that is -inf)
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

// Whether a sequence of packed rows first .. end is computed.
__device__ __forceinline__ bool computed(const VerifyArgs& a, uint32_t first, uint32_t end) {
  return first < end && end <= a.rows && end - first <= a.max_rows;
}

// The lowest sequence that is computed and holds `row`: by its own two offsets, as verify_walk has it, whatever the other
// sequences' are. (The walk reads the sums of every row of such a sequence: each is made in this call.) A wave looks at 64.
__device__ __forceinline__ bool find_computed(const VerifyArgs& a, uint32_t row, uint32_t& seq) {
  for (uint32_t i0 = 0; i0 < a.sequences; i0 += 64) {
    const uint32_t i = i0 + (threadIdx.x & 63u), s = min(i, a.sequences - 1);
    const uint32_t first = a.offsets[s], end = a.offsets[s + 1];
    const uint64_t holds = __ballot(i < a.sequences && computed(a, first, end) && first <= row && row < end);
    if (holds != 0) {
      seq = i0 + (uint32_t)__builtin_ctzll(holds);
      return true;
    }
  }
  return false;
}

// A workgroup per (chunk, row): its largest logit and its sum.
template <bool kExact, class T>
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
  uint32_t seq;
  if (!find_computed(a, row, seq)) return;
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
    for (uint32_t j = 0; j < kEach; j++) bad |= broken(v[j]);
    if (kExact || !fits_f32(temperature)) {
#pragma unroll
      for (uint32_t j = 0; j < kEach; j++) sum += exp2_of(((double)v[j] - from) * scale);
    } else {
      const float s = (float)scale, f = reference(top);
      float part[4] = {};
#pragma unroll
      for (uint32_t j = 0; j < kEach; j++) part[j % 4] += __builtin_amdgcn_exp2f((v[j] - f) * s);
      sum = (double)((part[0] + part[1]) + (part[2] + part[3]));
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

// What is drawn from, of ids i .. with logits l and draft probabilities q: p's exponentials without the rejected
// rows' tokens, or max(p - q, 0).
template <int N>
__device__ __forceinline__ void drawn_from(const Draw& r, const uint32_t* tokens, uint32_t i, const float (&l)[N],
                                           const float (&q)[N], double (&e)[N]) {
#pragma unroll
  for (int j = 0; j < N; j++) e[j] = exp2_of(((double)l[j] - (double)r.reference) * r.scale);
  if (r.of > 0.0) {
    const double to = 1.0 / r.of;
#pragma unroll
    for (int j = 0; j < N; j++) e[j] = fmax(e[j] * to - (double)q[j], 0.0);
  } else {
    for (uint64_t m = r.rejected; m != 0; m &= m - 1) {
      const uint32_t gone = tokens[__builtin_ctzll(m)] - i;
#pragma unroll
      for (uint32_t j = 0; j < N; j++)
        if (j == gone) e[j] = 0.0;
    }
  }
}

// A row's Z in f64, by the whole workgroup.
template <class T>
__device__ __forceinline__ double exact_sum(const VerifyArgs& a, const T* row, float top, double scale) {
  const double from = reference(top);
  double sum = 0.0;
  for (uint32_t i = threadIdx.x * kWalkEach; i < a.vocab; i += kChunk) {
    float l[kWalkEach];
    load_ids<kWalkEach>(row, i, a.vocab, -INFINITY, l);
#pragma unroll
    for (uint32_t j = 0; j < kWalkEach; j++) sum += exp2_of(((double)l[j] - from) * scale);
  }
  return block_sum<kWalkThreads / 64>(sum);
}

// A workgroup per (`together` chunks, sequence): the sequence's rows' sums from their chunks', the branch, and where a
// token is drawn the sums of its chunks of what it is drawn from, for verify_draw. The first of a sequence writes what it finds.
// A chain of dependent reads bounds it: offsets; rows and sums; single logits; the chunks.
// kBatch chunks of it at a time (1 or 4): all of their ids are under way before any is waited for.
template <bool kDraft, uint32_t kBatch, class T>
__global__ __launch_bounds__(kWalkThreads) void verify_walk(VerifyArgs a) {
  __shared__ float top_of[kMostRows], accept_of[kMostRows], q_of[kMostRows];
  __shared__ double sum_of[kMostRows], value_of[kMostRows];  // value_of: of a row's token where it was drafted
  __shared__ uint32_t id_of[kMostRows], token_of[kMostRows], path_of[kMostRows];
  __shared__ uint32_t count_of, row_of, unsure_of;
  __shared__ uint64_t rejected_of;  // rows, of the last row's children
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const bool writes = blockIdx.x == 0;
  const uint32_t first = a.offsets[seq], end = a.offsets[seq + 1], n = end - first;
  if (!computed(a, first, end)) {
    if (!writes) return;
    if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = kNone;
    if (tid == 0) {
      a.counts[seq] = 0;
      a.next[seq] = kNone;
      if (a.draw) a.draw[seq].row = kNone;
    }
    return;
  }
  const float temperature = temperature_of(a, seq);
  const bool greedy = !(temperature > 0.f), rough = !kDraft && fits_f32(temperature);
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
  uint32_t at = 0, count = 1;
  uint64_t rejected = 0, exact = rough ? 0 : ~0ull;  // exact: rows whose sum is
  if (wave == 0) {
    token_of[lane] = token;
    accept_of[lane] = accept;
    q_of[lane] = q;
    value_of[lane] = parent == kNone ? 0.0 : exp2_of(((double)logit - (double)reference(top_of[parent])) * scale);
    if (lane == 0) path_of[0] = 0;
  }
  for (;;) {
    if (wave == 0) {  // (the whole wave takes the same steps)
      uint32_t unsure = kNone;
      for (;;) {
        uint64_t children = __ballot(parent == at);
        uint32_t to = kNone;
        const double sum = sum_of[at];
        double left = sum;
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
            const double than = (double)accept_of[r] * left;
            if (!again && !(exact >> at & 1u) && fabs(than - value_of[r]) < (double)accept_of[r] * sum * kMargin) {
              unsure = at;
              break;
            }
            ok = !again && than < value_of[r];
            if (!ok && !again) left -= value_of[r];
          }
          if (ok) {
            to = r;
            break;
          }
          rejected |= 1ull << r;
        }
        if (unsure != kNone || to == kNone) break;
        at = to;
        if (lane == 0) path_of[count] = at;
        count++;
      }
      if (lane == 0) {
        count_of = count;
        row_of = at;
        rejected_of = rejected;
        unsure_of = unsure;
      }
    }
    __syncthreads();
    const uint32_t again = unsure_of;
    if (again == kNone) break;
    const double sum = exact_sum(a, logits + again * a.stride, top_of[again], scale);
    if (tid == 0) sum_of[again] = sum;
    exact |= 1ull << again;
    __syncthreads();
  }
  count = count_of;
  at = row_of;
  const double total = sum_of[at];
  const bool draws = !greedy && total > 0.0 && total < (double)INFINITY;
  const Draw from{scale, kDraft && rejected_of != 0 ? total : 0.0, kDraft ? 0 : rejected_of, draws ? first + at : kNone, first,
                  reference(top_of[at])};
  if (writes) {
    if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = tid < count ? path_of[tid] : kNone;
    if (tid == 0) {
      a.counts[seq] = count;
      a.next[seq] = id_of[at];  // (unless one is drawn)
      if (a.draw) a.draw[seq] = from;
    }
  }
  if (!draws) return;
  constexpr uint32_t kWaves = kWalkThreads / 64;
  __shared__ double part[kBatch][kWaves];
  const uint32_t last = min(a.chunks, (blockIdx.x + 1) * a.together);
  const T* row = logits + at * a.stride;
  const float* draft = a.draft + (uint64_t)(first + at) * a.draft_stride;
  double* masses = a.masses + (uint64_t)seq * a.chunks;
  for (uint32_t c0 = blockIdx.x * a.together; c0 < last; c0 += kBatch) {
    float l[kBatch][kWalkEach], q[kBatch][kWalkEach] = {};
    if (c0 + kBatch <= last && (c0 + kBatch) * kChunk <= a.vocab) {
#pragma unroll
      for (uint32_t b = 0; b < kBatch; b++) {
        const uint32_t i = (c0 + b) * kChunk + tid * kWalkEach;
        const Several<T, kWalkEach> x = *reinterpret_cast<const Several<T, kWalkEach>*>(row + i);
#pragma unroll
        for (uint32_t j = 0; j < kWalkEach; j++) l[b][j] = to_f32(x.v[j]);
        if (kDraft) {
          const Several<float, kWalkEach> y = *reinterpret_cast<const Several<float, kWalkEach>*>(draft + i);
#pragma unroll
          for (uint32_t j = 0; j < kWalkEach; j++) q[b][j] = y.v[j];
        }
      }
    } else {
#pragma unroll
      for (uint32_t b = 0; b < kBatch; b++) {
        const uint32_t i = (c0 + b) * kChunk + tid * kWalkEach, ids = c0 + b < last ? a.vocab : 0;
        load_ids<kWalkEach>(row, i, ids, -INFINITY, l[b]);
        if (kDraft) load_ids<kWalkEach>(draft, i, ids, 0.f, q[b]);
      }
    }
    double sum[kBatch];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; b++) {
      double e[kWalkEach];
      drawn_from(from, token_of, (c0 + b) * kChunk + tid * kWalkEach, l[b], q[b], e);
      sum[b] = 0.0;
#pragma unroll
      for (uint32_t j = 0; j < kWalkEach; j++) sum[b] += e[j];
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; b++) sum[b] = wave_sum(sum[b]);
    __syncthreads();
#pragma unroll
    for (uint32_t b = 0; b < kBatch; b++)
      if (lane == b) part[b][wave] = sum[b];
    __syncthreads();
    if (tid < kBatch && c0 + tid < last) {
      double all = part[tid][0];
#pragma unroll
      for (uint32_t w = 1; w < kWaves; w++) all += part[tid][w];
      masses[c0 + tid] = all;
    }
  }
}

// A workgroup per sequence: the chunk, and the id in it.
template <class T>
__global__ __launch_bounds__(kWalkThreads) void verify_draw(VerifyArgs a) {
  const uint32_t seq = blockIdx.x, tid = threadIdx.x;
  const Draw r = a.draw[seq];
  if (r.row == kNone) return;
  const double mass = tid < a.chunks ? a.masses[(uint64_t)seq * a.chunks + tid] : 0.0;
  uint32_t chunk;
  double target;
  if (!find_chunk(mass, a.draws[seq], chunk, target)) return;  // (nothing is left to draw from)
  const T* row = static_cast<const T*>(a.logits) + (uint64_t)r.row * a.stride;
  const uint32_t id = find_in_chunk(chunk, target, [&](uint32_t i, double (&e)[kWalkEach]) {
    float l[kWalkEach], q[kWalkEach] = {};
    load_ids<kWalkEach>(row, i, a.vocab, -INFINITY, l);
    if (r.of > 0.0) load_ids<kWalkEach>(a.draft + (uint64_t)r.row * a.draft_stride, i, a.vocab, 0.f, q);
    drawn_from(r, a.tokens + r.first, i, l, q, e);
  });
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
  const uint64_t draw = temperatures ? (uint64_t)d.sequences * (sizeof(Draw) + a.chunks * sizeof(double)) : 0;
  if (stats + draw > eg::kPartialsBytes || d.rows > 65535 || d.sequences > 65535)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences, %u rows of %u ids over the workspace or the grid limit", op, d.sequences,
                    d.rows, d.vocab);
  const uint64_t n = d.sequences;  // (a sequence's workgroups read its inputs at any time)
  const uint64_t size = d.type == EG_ELEMENT_F32 ? 4 : 2;
  const Extent outputs[] = {words(path, n * d.max_rows), words(counts, n), words(next, n)};
  const Extent inputs[] = {words(tokens, d.rows), words(offsets, n + 1), words(parents, d.rows), words(accept, d.rows),
                           words(draws, n), words(temperatures, n), {logits, d.rows, size * a.stride, size * d.vocab},
                           {draft, d.rows, 4 * a.draft_stride, 4ull * d.vocab}};
  for (const Extent& out : outputs) {
    for (const Extent& in : inputs)
      if (overlap(out, in)) return eg::fail(ctx, EG_ERR_INVALID, "%s: an output lies in an input", op);
    for (const Extent& other : outputs)
      if (&out != &other && overlap(out, other)) return eg::fail(ctx, EG_ERR_INVALID, "%s: an output lies in another", op);
  }
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
  a.draw = temperatures ? reinterpret_cast<Draw*>(at + stats) : nullptr;
  a.masses = reinterpret_cast<double*>(at + stats + (uint64_t)d.sequences * sizeof(Draw));
  // A chunk a workgroup where all are then under way at once, else four and more.
  const uint64_t all_chunks = (uint64_t)a.chunks * d.sequences, room = 4ull * ctx->cu_count;
  a.together = all_chunks <= room ? 1 : 4 * (uint32_t)((all_chunks + 4 * room - 1) / (4 * room));
  a.sequences = d.sequences;
  a.rows = d.rows;
  a.max_rows = d.max_rows;
  a.vocab = d.vocab;
  const OnDevice on(ctx);
  with_type(d.type, [&](auto t) {
    using T = decltype(t);
    const bool drafted = draft && temperatures;
    const dim3 threads(kThreads), walk(kWalkThreads);
    const dim3 grid(temperatures ? (a.chunks + a.together - 1) / a.together : 1, d.sequences);
    if (d.rows != 0) {
      if (drafted) hipLaunchKernelGGL((verify_stats<true, T>), dim3(a.chunks, d.rows), threads, 0, ctx->stream, a);
      else hipLaunchKernelGGL((verify_stats<false, T>), dim3(a.chunks, d.rows), threads, 0, ctx->stream, a);
    }
    const auto kernel = drafted ? (a.together == 1 ? verify_walk<true, 1, T> : verify_walk<true, 4, T>)
                                : (a.together == 1 ? verify_walk<false, 1, T> : verify_walk<false, 4, T>);
    hipLaunchKernelGGL(kernel, grid, walk, 0, ctx->stream, a);
    if (temperatures) hipLaunchKernelGGL(verify_draw<T>, dim3(d.sequences), walk, 0, ctx->stream, a);
  });
  return eg::check_launch(ctx, op);
}

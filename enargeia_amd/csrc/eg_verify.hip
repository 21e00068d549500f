// Drafted tokens against the target's probabilities (eg_verify_drafts).
//
// Three quantities of a row of logits decide: its largest, Z = sum 2^((l - largest) log2(e) / temperature), and
// the running sum that the next token is drawn by. All three come from partials per chunk of kChunk ids, made for
// all rows at once by verify_stats: that pass reads the logits, and is what bounds the operator. Which rows the branch
// goes through then takes single logits (verify_walk, a workgroup per sequence), and the draw reads one chunk
// of one row again: the one in which the running sum passes the target. After a rejection by draft probabilities
// the sums are of max(p - q, 0), so that row's chunks are summed once more (verify_residual, verify_draw).
//
// Sums and exponentials are f64: of 151,936 running sums some lie within f32's rounding of the drawn target in one
// draw of a hundred, within these in none of 10^6. f64 vector instructions run at f32's rate, and an exponential is
// about 16 of them, under the time of its logit's 4 bytes.
#include <algorithm>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256, kMostRows = 64, kEach = 16, kChunk = kThreads * kEach;
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

// 2^x for x <= 0, to 3e-13: 2^k times the Taylor polynomial of 2^r, |r| <= 1/2, whose next term is at most
// 0.347^11 / 11! = 2.2e-13. NaN stays NaN.
__device__ __forceinline__ double exp2_of(double x) {
  x = x < -1100.0 ? -1100.0 : x;
  const double k = rint(x), r = x - k;
  double p = 7.054911620801121e-09;
  p = fma(p, r, 1.01780860092396997e-07);
  p = fma(p, r, 1.3215486790144305e-06);
  p = fma(p, r, 1.5252733804059838e-05);
  p = fma(p, r, 0.0001540353039338161);
  p = fma(p, r, 0.0013333558146428443);
  p = fma(p, r, 0.009618129107628477);
  p = fma(p, r, 0.055504108664821576);
  p = fma(p, r, 0.24022650695910069);
  p = fma(p, r, 0.6931471805599453);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)k);
}

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

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 64];
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// The sum over the threads before this one; `total` over all.
__device__ __forceinline__ double block_before(double v, double& total) {
  __shared__ double part[kThreads / 64];
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
  for (uint32_t w = 0; w < wave; w++) before += part[w];
  total = (part[0] + part[1]) + (part[2] + part[3]);
  const double o = __shfl_up(run, 1, 64);
  return lane == 0 ? before : before + o;
}

// A workgroup per (chunk, row): its largest logit and its sum.
template <class T>
__global__ __launch_bounds__(256) void verify_stats(VerifyArgs a) {
  constexpr uint32_t kWide = 16 / sizeof(T);
  const uint32_t row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  uint32_t seq, first, end;
  if (!find_sequence(a.offsets, a.sequences, row, seq, first, end)) return;
  const float temperature = temperature_of(a, seq);
  const T* x = static_cast<const T*>(a.logits) + (uint64_t)row * a.stride;
  const uint32_t begin = chunk * kChunk;
  float v[kEach];
#pragma unroll
  for (uint32_t j = 0; j < kEach / kWide; j++) {
    const uint32_t i = begin + kWide * (j * kThreads + tid);
    if (i + kWide <= a.vocab) {
      const Several<T, kWide> s = *reinterpret_cast<const Several<T, kWide>*>(x + i);
#pragma unroll
      for (uint32_t e = 0; e < kWide; e++) v[j * kWide + e] = to_f32(s.v[e]);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < kWide; e++) v[j * kWide + e] = i + e < a.vocab ? to_f32(x[i + e]) : -INFINITY;
    }
  }
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
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) sum += exp2_of(((double)v[j] - from) * scale);
    sum = block_sum(sum);
  }
  if (tid == 0) a.stats[(uint64_t)row * a.chunks + chunk] = Stats{sum, top, id};
}

// Times a chunk's sum: from its reference to the row's.
__device__ __forceinline__ double rescaled(const Stats& s, float top, double scale) {
  return s.top == -INFINITY ? s.sum : s.sum * exp2_of(((double)s.top - (double)reference(top)) * scale);
}

// The lowest id at which the running sum of value(id), from this chunk's beginning on, exceeds `target`; the last one
// of a value above 0 where rounding leaves none. Every thread gets it.
template <class F>
__device__ __forceinline__ uint32_t find_in_chunk(uint32_t chunk, uint32_t vocab, double target, F&& value) {
  __shared__ uint32_t found, last;
  const uint32_t begin = chunk * kChunk + threadIdx.x * kEach;
  if (threadIdx.x == 0) {
    found = kNone;
    last = 0;
  }
  double e[kEach], sum = 0.0;
  uint32_t mine = 0;
#pragma unroll
  for (uint32_t j = 0; j < kEach; j++) {
    e[j] = begin + j < vocab ? value(begin + j) : 0.0;
    sum += e[j];
    if (e[j] > 0.0) mine = begin + j;
  }
  double total, run = block_before(sum, total);  // (its barriers order the two words above)
  uint32_t hit = kNone;
#pragma unroll
  for (uint32_t j = 0; j < kEach; j++) {
    run += e[j];
    if (e[j] > 0.0 && run > target && hit == kNone) hit = begin + j;
  }
  if (hit != kNone) atomicMin(&found, hit);
  if (mine != 0) atomicMax(&last, mine);
  __syncthreads();
  return found != kNone ? found : last;
}

// The chunk in which the running sum of `mass` (a chunk per thread) exceeds draw * the whole sum, and what of that
// lies before it. False: there is nothing to draw from.
__device__ __forceinline__ bool find_chunk(double mass, float draw, uint32_t& chunk, double& target) {
  __shared__ uint32_t at, last;
  __shared__ double rest;
  if (threadIdx.x == 0) {
    at = kNone;
    last = kNone;
  }
  double total;
  const double before = block_before(mass, total);
  if (!(total > 0.0) || !(total < (double)INFINITY)) return false;  // (the same in every thread)
  const double whole = (double)draw * total;
  if (mass > 0.0 && before + mass > whole) atomicMin(&at, threadIdx.x);
  __syncthreads();
  if (at == kNone && mass > 0.0) atomicMin(&last, kThreads - 1 - threadIdx.x);  // (of the last: the lowest of these)
  __syncthreads();
  chunk = at != kNone ? at : kThreads - 1 - last;
  if (threadIdx.x == chunk) rest = whole - before;
  __syncthreads();
  target = rest;
  return true;
}

// A workgroup per sequence: its rows' sums from their chunks', the branch, and the next token - but of a draw from
// max(p - q, 0), which is left to the launches after this one.
template <class T>
__global__ __launch_bounds__(256) void verify_walk(VerifyArgs a) {
  __shared__ float top_of[kMostRows], accept_of[kMostRows], q_of[kMostRows];
  __shared__ double sum_of[kMostRows], value_of[kMostRows];  // value_of: of a row's token where it was drafted
  __shared__ uint32_t id_of[kMostRows], parent_of[kMostRows], token_of[kMostRows], path_of[kMostRows];
  __shared__ uint32_t count_of, row_of;
  __shared__ uint64_t rejected_of;  // rows, of the last row's children
  const uint32_t seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t first = a.offsets[seq], end = a.offsets[seq + 1], n = end - first;
  if (a.draft && tid == 0) a.residual[seq].row = kNone;
  if (n == 0 || n > a.max_rows || first > end || end > a.rows) {
    if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = kNone;
    if (tid == 0) {
      a.counts[seq] = 0;
      a.next[seq] = kNone;
    }
    return;
  }
  const float temperature = temperature_of(a, seq);
  const bool greedy = !(temperature > 0.f);
  const double scale = greedy ? 0.0 : scale_of(temperature);
  const T* logits = static_cast<const T*>(a.logits) + (uint64_t)first * a.stride;
  const Stats* stats = a.stats + (uint64_t)first * a.chunks;
  for (uint32_t r = wave; r < n; r += kThreads / 64) {
    float top = -INFINITY;
    uint32_t id = 0;
    for (uint32_t c = lane; c < a.chunks; c += 64) {
      const Stats s = stats[(uint64_t)r * a.chunks + c];
      if (egd::better(s.top, s.id, top, id)) {
        top = s.top;
        id = s.id;
      }
    }
    egd::team_argmax<64>(top, id);
    double sum = 0.0;
    if (!greedy) {
      for (uint32_t c = lane; c < a.chunks; c += 64) sum += rescaled(stats[(uint64_t)r * a.chunks + c], top, scale);
      sum = wave_sum(sum);
    }
    if (lane == 0) {
      top_of[r] = top;
      id_of[r] = id;
      sum_of[r] = sum;
    }
  }
  if (tid < n) {
    uint32_t p = tid - 1;  // (of row 0: none)
    if (a.parents) p = a.parents[first + tid];
    parent_of[tid] = p < tid ? p : kNone;
    token_of[tid] = a.tokens[first + tid];
    accept_of[tid] = greedy ? 0.f : a.accept[first + tid];
  }
  __syncthreads();
  if (tid < n) {
    const uint32_t p = parent_of[tid], x = token_of[tid];
    double value = 0.0;
    float q = 0.f;
    if (p != kNone && x < a.vocab && !greedy) {
      value = exp2_of(((double)to_f32(logits[p * a.stride + x]) - (double)reference(top_of[p])) * scale);
      if (a.draft) q = a.draft[(uint64_t)(first + p) * a.draft_stride + x];
    }
    value_of[tid] = value;
    q_of[tid] = q;
  }
  __syncthreads();
  if (wave == 0) {  // (the whole wave takes the same steps)
    uint32_t at = 0, count = 1;
    uint64_t rejected = 0;
    if (lane == 0) path_of[0] = 0;
    const uint32_t my_parent = lane < n ? parent_of[lane] : kNone, my_token = lane < n ? token_of[lane] : kNone;
    for (;;) {
      uint64_t children = __ballot(my_parent == at);
      uint32_t to = kNone;
      double left = sum_of[at];
      rejected = 0;
      while (children != 0) {
        const uint32_t r = (uint32_t)__builtin_ctzll(children), token = token_of[r];
        children &= children - 1;
        bool ok;
        if (greedy) {
          ok = token == id_of[at];
        } else if (a.draft) {
          ok = (double)accept_of[r] * (double)q_of[r] * left < value_of[r];
        } else {
          const bool again = (__ballot(my_token == token) & rejected) != 0;
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
  if (tid < a.max_rows) a.path[(uint64_t)seq * a.max_rows + tid] = tid < count ? path_of[tid] : kNone;
  if (tid == 0) a.counts[seq] = count;
  const double total = sum_of[at];
  if (greedy || !(total > 0.0) || !(total < (double)INFINITY)) {
    if (tid == 0) a.next[seq] = id_of[at];
    return;
  }
  if (a.draft && rejected != 0) {
    if (tid == 0) {
      a.residual[seq] = Residual{scale, total, first + at, reference(top_of[at])};
      a.next[seq] = id_of[at];  // (what stays where p and q leave nothing)
    }
    return;
  }
  // Of a token that several rejected rows hold the first one counts.
  const auto gone = [&](uint32_t id) {
    bool is = false;
    for (uint64_t m = rejected; m != 0; m &= m - 1) is |= token_of[__builtin_ctzll(m)] == id;
    return is;
  };
  double mass = 0.0;
  if (tid < a.chunks) {
    mass = rescaled(stats[(uint64_t)at * a.chunks + tid], top_of[at], scale);
    uint64_t seen = 0;
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
  if (!find_chunk(mass, a.draws[seq], chunk, target)) {
    if (tid == 0) a.next[seq] = id_of[at];
    return;
  }
  const T* x = logits + at * a.stride;
  const double from = reference(top_of[at]);
  const uint32_t id = find_in_chunk(chunk, a.vocab, target, [&](uint32_t i) {
    return gone(i) ? 0.0 : exp2_of(((double)to_f32(x[i]) - from) * scale);
  });
  if (tid == 0) a.next[seq] = id;
}

// max(p - q, 0) of an id in a sequence's last accepted row.
template <class T>
__device__ __forceinline__ double left_over(const VerifyArgs& a, const Residual& r, uint32_t id) {
  const double l = to_f32((static_cast<const T*>(a.logits) + (uint64_t)r.row * a.stride)[id]);
  const double q = a.draft[(uint64_t)r.row * a.draft_stride + id];
  return fmax(exp2_of((l - (double)r.reference) * r.scale) / r.total - q, 0.0);
}

template <class T>
__global__ __launch_bounds__(256) void verify_residual(VerifyArgs a) {
  const uint32_t seq = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const Residual r = a.residual[seq];
  if (r.row == kNone) return;
  double sum = 0.0;
#pragma unroll
  for (uint32_t j = 0; j < kEach; j++) {
    const uint32_t i = chunk * kChunk + j * kThreads + tid;
    if (i < a.vocab) sum += left_over<T>(a, r, i);
  }
  sum = block_sum(sum);
  if (tid == 0) a.masses[(uint64_t)seq * a.chunks + chunk] = sum;
}

template <class T>
__global__ __launch_bounds__(256) void verify_draw(VerifyArgs a) {
  const uint32_t seq = blockIdx.x, tid = threadIdx.x;
  const Residual r = a.residual[seq];
  if (r.row == kNone) return;
  const double mass = tid < a.chunks ? a.masses[(uint64_t)seq * a.chunks + tid] : 0.0;
  uint32_t chunk;
  double target;
  if (!find_chunk(mass, a.draws[seq], chunk, target)) return;
  const uint32_t id = find_in_chunk(chunk, a.vocab, target, [&](uint32_t i) { return left_over<T>(a, r, i); });
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
  if (d.sequences > (1u << 20)) return eg::fail(ctx, EG_ERR_RANGE, "%s: %u sequences (at most 2^20)", op, d.sequences);
  const uint64_t stats = (uint64_t)d.rows * a.chunks * sizeof(Stats);
  const uint64_t residual = draft ? (uint64_t)d.sequences * (sizeof(Residual) + a.chunks * sizeof(double)) : 0;
  if (stats + residual > eg::kPartialsBytes || d.rows > 65535 || (draft && d.sequences > 65535))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows of %u ids over the workspace or the grid limit", op, d.rows, d.vocab);
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
    hipLaunchKernelGGL(verify_walk<T>, dim3(d.sequences), threads, 0, ctx->stream, a);
    if (draft && temperatures) {
      hipLaunchKernelGGL(verify_residual<T>, dim3(a.chunks, d.sequences), threads, 0, ctx->stream, a);
      hipLaunchKernelGGL(verify_draw<T>, dim3(d.sequences), threads, 0, ctx->stream, a);
    }
  });
  return eg::check_launch(ctx, op);
}

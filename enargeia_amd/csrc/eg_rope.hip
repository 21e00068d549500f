// Rotary positions (enargeia_hip.h): tables of (cos, sin) with scaled frequencies, and rows rotated at positions of
// their own. Both move bytes: their floor is what they read and write once at the memory's rate.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostDim = 512;

struct Frequencies {
  double f[kMostDim / 2];  // turns per position
};

// (cos, sin) of `turns` turns, to 2^-51: the nearest quarter is taken off exactly, what is left is at most an eighth of a turn,
// an angle of up to pi / 4, whose series' next terms are under 2^-54 ((pi / 4)^17 / 17! and ^18 / 18!).
__device__ __forceinline__ double2 turned(double turns) {
  const double r = turns - rint(turns), quarter = rint(4.0 * r);
  const double x = (r - 0.25 * quarter) * 6.283185307179586, y = x * x;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, y, 1.0 / 6227020800.0);
  c = fma(c, y, -1.0 / 87178291200.0);
  s = fma(s, y, -1.0 / 39916800.0);
  c = fma(c, y, 1.0 / 479001600.0);
  s = fma(s, y, 1.0 / 362880.0);
  c = fma(c, y, -1.0 / 3628800.0);
  s = fma(s, y, -1.0 / 5040.0);
  c = fma(c, y, 1.0 / 40320.0);
  s = fma(s, y, 1.0 / 120.0);
  c = fma(c, y, -1.0 / 720.0);
  s = fma(s, y, -1.0 / 6.0);
  c = fma(c, y, 1.0 / 24.0);
  s = fma(s * y, x, x);
  c = fma(c, y, -0.5);
  c = fma(c, y, 1.0);
  const int q = (int)quarter;  // -2 .. 2
  const double co = q & 1 ? s : c, si = q & 1 ? c : s;
  return make_double2(q == 1 || (q & 2 && !(q & 1)) ? -co : co, q < 0 || q == 2 ? -si : si);
}

// A thread makes two pairs, 16 bytes, of kRows positions that follow each other: the first's by series, the others' each
// from the one before, turned by one position (4 f64 instructions for 32, off by up to 2^-51 more with each). 131,072
// positions of 64 pairs 12.7 us, with a series each 19.3; stores alone 12.
constexpr uint32_t kRows = 8;
__global__ __launch_bounds__(256) void table_kernel(float4* table, Frequencies fs, uint32_t first, uint32_t positions,
                                                    uint32_t halves, uint32_t count, double amplitude) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  const uint32_t rows = i / halves, j = i - rows * halves;
  const double p = (double)(first + kRows * rows);
  const double2 step[2] = {turned(fs.f[2 * j]), turned(fs.f[2 * j + 1])};
  double2 at[2] = {turned(p * fs.f[2 * j]), turned(p * fs.f[2 * j + 1])};
#pragma unroll
  for (int e = 0; e < 2; e++) at[e] = make_double2(at[e].x * amplitude, at[e].y * amplitude);
#pragma unroll
  for (uint32_t k = 0; k < kRows; k++) {
    const uint32_t row = kRows * rows + k;
    if (row < positions)
      table[(uint64_t)row * halves + j] = make_float4((float)at[0].x, (float)at[0].y, (float)at[1].x, (float)at[1].y);
#pragma unroll
    for (int e = 0; e < 2; e++)
      at[e] = make_double2(fma(at[e].x, step[e].x, -at[e].y * step[e].y), fma(at[e].y, step[e].x, at[e].x * step[e].y));
  }
}

struct RopeArgs {
  const void *q, *k;
  const float2* table;
  const uint32_t *positions, *offsets, *starts;
  void *q_out, *k_out;
  uint32_t rows, heads, kv_heads, head_dim, rotary_dim;
  uint32_t q_stride, k_stride, q_out_stride, k_out_stride, table_positions, sequences;
};

template <class T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Several {
  T v[N];
};

// A workgroup per row, so that the position and its table row are found once; a unit is 8 elements of a head: 4 pairs,
// or 8 elements past the rotary part. Memory bounds it: 32,768 rows of 40 heads of 128, half rotated, bf16, in 116 us, 5.8 TB/s
// read and written; 16 rows of 16 heads of 64 in 2.8 us, a chain of offsets, position, table. Neighbours as pairs, f32 out: 4
// elements, so that a wave's 16-byte stores follow each other, and two units under way (16,384 rows of 40 heads of 128, f16 to f32,
// in 97 us for 107). Halves apart: the units that rotate first, so that a wave does one thing (half rotated, bf16, 59 us for 69).
template <bool kInterleaved, class TI, class TO>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
#pragma clang fp contract(off)
  const uint32_t r = blockIdx.x;
  uint64_t position = a.positions ? a.positions[r] : 0;
  if (a.offsets) {
    uint32_t seq, first, end;
    if (!find_sequence(a.offsets, a.sequences, r, seq, first, end)) return;
    if (!a.positions) position = r - first;
    if (a.starts) position += a.starts[seq];
  }
  if (position >= a.table_positions) return;
  const float2* cs = a.table + position * (a.rotary_dim / 2);
  constexpr uint32_t kUnit = kInterleaved && sizeof(TO) == 4 ? 4 : 8;
  const uint32_t per_head = a.head_dim / kUnit, turned = a.rotary_dim / kUnit;
  const uint32_t units = (a.heads + a.kv_heads) * per_head, half = a.rotary_dim / 2;
  const uint32_t split = (a.heads + a.kv_heads) * turned;  // halves apart: units before it rotate, so that waves do one or the other
  struct Unit {
    const TI* src;
    TO* dst;
    uint32_t u;
    Several<TI, kUnit> x;
    Several<TI, 4> y, z;
  };
  // (apart: a unit whose pairs lie half the rotary part from each other)
  const auto load = [&](auto apart, uint32_t i, Unit& t) {
    uint32_t head;
    if constexpr (!decltype(apart)::value) {
      const uint32_t first = kInterleaved ? 0 : turned, each = per_head - first, j = kInterleaved ? i : i - split;
      head = j / each;
      t.u = first + j % each;
    } else {
      head = i / turned;
      t.u = i % turned;
    }
    const bool is_q = head < a.heads;
    if (!is_q) head -= a.heads;
    t.src = static_cast<const TI*>(is_q ? a.q : a.k) + (size_t)r * (is_q ? a.q_stride : a.k_stride) + (size_t)head * a.head_dim;
    t.dst = static_cast<TO*>(is_q ? a.q_out : a.k_out) + (size_t)r * (is_q ? a.q_out_stride : a.k_out_stride) +
            (size_t)head * a.head_dim;
    if constexpr (decltype(apart)::value) {
      t.y = *reinterpret_cast<const Several<TI, 4>*>(t.src + 4 * t.u);
      t.z = *reinterpret_cast<const Several<TI, 4>*>(t.src + half + 4 * t.u);
    } else {
      t.x = *reinterpret_cast<const Several<TI, kUnit>*>(t.src + kUnit * t.u);
    }
  };
  const auto store = [&](auto apart, const Unit& t) {
    if constexpr (decltype(apart)::value) {
      Several<TO, 4> y, w;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 c = cs[4 * t.u + e];
        const float p = to_f32(t.y.v[e]), o = to_f32(t.z.v[e]);
        y.v[e] = from_f32<TO>(p * c.x - o * c.y);
        w.v[e] = from_f32<TO>(o * c.x + p * c.y);
      }
      *reinterpret_cast<Several<TO, 4>*>(t.dst + 4 * t.u) = y;
      *reinterpret_cast<Several<TO, 4>*>(t.dst + half + 4 * t.u) = w;
    } else {
      Several<TO, kUnit> y;
      if (kInterleaved && t.u < turned) {
#pragma unroll
        for (uint32_t e = 0; e < kUnit / 2; e++) {
          const float2 c = cs[kUnit / 2 * t.u + e];
          const float p = to_f32(t.x.v[2 * e]), w = to_f32(t.x.v[2 * e + 1]);
          y.v[2 * e] = from_f32<TO>(p * c.x - w * c.y);
          y.v[2 * e + 1] = from_f32<TO>(w * c.x + p * c.y);
        }
      } else {
#pragma unroll
        for (uint32_t e = 0; e < kUnit; e++) y.v[e] = from_f32<TO>(to_f32(t.x.v[e]));
      }
      *reinterpret_cast<Several<TO, kUnit>*>(t.dst + kUnit * t.u) = y;
    }
  };
  constexpr std::true_type apart{};
  constexpr std::false_type whole{};
  if constexpr (kInterleaved) {  // two units under way together (a load does not pass a store by itself: an output may be its input)
    for (uint32_t i = threadIdx.x; i < units; i += 2 * kThreads) {
      Unit one, two;
      load(whole, i, one);
      const bool more = i + kThreads < units;
      if (more) load(whole, i + kThreads, two);
      store(whole, one);
      if (more) store(whole, two);
    }
  } else {  // (which have two loads each)
    for (uint32_t i = threadIdx.x; i < units; i += kThreads) {
      Unit one;
      if (i < split) {
        load(apart, i, one);
        store(apart, one);
      } else {
        load(whole, i, one);
        store(whole, one);
      }
    }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool above_zero(double v) { return v > 0.0 && std::isfinite(v); }

}  // namespace

extern "C" {

int eg_rope_table(eg_context* ctx, float* table, const eg_rope_table_dims* dims) {
  const char* op = "rope_table";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  if (!dims || (!table && dims->positions != 0)) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_rope_table_dims& d = *dims;
  if (d.rotary_dim == 0 || d.rotary_dim % 8 != 0 || d.rotary_dim > kMostDim)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: rotary_dim %u (a multiple of 8, 8 to %u)", op, d.rotary_dim, kMostDim);
  if (d.scaling < EG_ROPE_PLAIN || d.scaling > EG_ROPE_LOG_TURNS)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: scaling %d (eg_rope_scaling)", op, d.scaling);
  if (!above_zero(d.theta)) return eg::fail(ctx, EG_ERR_INVALID, "%s: theta %g (above 0)", op, d.theta);
  if (d.scaling != EG_ROPE_PLAIN && !above_zero(d.factor))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: factor %g (above 0)", op, d.factor);
  const bool by_turns = d.scaling == EG_ROPE_TURNS || d.scaling == EG_ROPE_LOG_TURNS;
  if (by_turns && (!above_zero(d.context) || !above_zero(d.low) || !above_zero(d.high) || d.low >= d.high))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: context %g, low %g, high %g (above 0, low below high)", op, d.context, d.low,
                    d.high);
  if (!std::isfinite(d.amplitude)) return eg::fail(ctx, EG_ERR_INVALID, "%s: amplitude %g", op, d.amplitude);
  if ((uint64_t)d.first + d.positions > (1ull << 31))
    return eg::fail(ctx, EG_ERR_RANGE, "%s: positions %u from %u on (together under 2^31)", op, d.positions, d.first);
  if (!aligned(table)) return eg::fail(ctx, EG_ERR_INVALID, "%s: the table must be 16-byte aligned", op);
  const uint32_t pairs = d.rotary_dim / 2;
  const uint64_t count = (uint64_t)((d.positions + kRows - 1) / kRows) * (pairs / 2), blocks = (count + kThreads - 1) / kThreads;
  if (blocks >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u positions of %u over the grid limit", op, d.positions, d.rotary_dim);
  if (count == 0) return EG_OK;
  // Frequencies by one power and products of 64 bits of mantissa (256 of them stay under half a last place of a double:
  // a power each took 3 us of a call's 7).
  const long double r = d.rotary_dim, pi = 3.14159265358979323846264338327950288L;
  const long double theta = d.scaling == EG_ROPE_BASE ? d.theta * powl(d.factor, r / (r - 2.0L)) : d.theta;
  const long double step = powl(theta, -2.0L / r);
  const double log_step = d.scaling == EG_ROPE_LOG_TURNS ? std::log((double)step) : 0.0;
  const double log_low = d.scaling == EG_ROPE_LOG_TURNS ? std::log(d.context / (2.0 * (double)pi * d.low)) : 0.0;
  Frequencies fs;
  long double power = 1.0L;
  for (uint32_t i = 0; i < pairs; i++, power *= step) {
    long double f = power;
    if (d.scaling == EG_ROPE_LINEAR) f /= d.factor;
    if (by_turns) {
      const double turns = (double)(d.context * f / (2.0L * pi));
      double w = d.scaling == EG_ROPE_TURNS ? (turns - d.low) / (d.high - d.low)
                                            : (log_low + i * log_step) / std::log(d.high / d.low);
      w = std::min(1.0, std::max(0.0, w));
      f *= w + (1.0 - w) / d.factor;
    }
    fs.f[i] = (double)(f / (2.0L * pi));
  }
  const OnDevice on(ctx);
  hipLaunchKernelGGL(table_kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, ctx->stream,
                     reinterpret_cast<float4*>(table), fs, d.first, d.positions, pairs / 2, (uint32_t)count,
                     d.amplitude == 0.0 ? 1.0 : d.amplitude);
  return eg::check_launch(ctx, op);
}

int eg_rope(eg_context* ctx, const void* q, const void* k, const float* table, const uint32_t* positions,
            const uint32_t* offsets, const uint32_t* starts, void* q_out, void* k_out, const eg_rope_dims* dims) {
  const char* op = "rope";
  if (!ctx) return eg::fail(nullptr, EG_ERR_INVALID, "%s: ctx is NULL", op);
  if (!dims) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const eg_rope_dims& d = *dims;
  if (d.head_dim == 0 || d.head_dim % 8 != 0 || d.head_dim > kMostDim)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: head_dim %u (a multiple of 8, 8 to %u)", op, d.head_dim, kMostDim);
  const uint32_t rotary = d.rotary_dim ? d.rotary_dim : d.head_dim;
  if (rotary % 8 != 0 || rotary > d.head_dim)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: rotary_dim %u (a multiple of 8, to head_dim %u)", op, rotary, d.head_dim);
  if (d.layout != EG_ROPE_HALF && d.layout != EG_ROPE_INTERLEAVED)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: layout %d (eg_rope_layout)", op, d.layout);
  if (!known_type(d.in_type) || !known_type(d.out_type))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: in_type %d, out_type %d (eg_element)", op, d.in_type, d.out_type);
  if (d.heads > 65535 || d.kv_heads > 65535)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u and %u heads (at most 65535)", op, d.heads, d.kv_heads);
  const bool some = d.rows != 0 && (!offsets || d.sequences != 0);
  if (some && ((q == nullptr) != (d.heads == 0) || (q_out == nullptr) != (d.heads == 0) ||
               (k == nullptr) != (d.kv_heads == 0) || (k_out == nullptr) != (d.kv_heads == 0)))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q, q_out and heads go together, and k, k_out and kv_heads", op);
  if (!offsets && (starts || d.sequences != 0))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: starts and sequences go with offsets", op);
  if (some && (!table || (!offsets && !positions))) return eg::fail(ctx, EG_ERR_INVALID, "%s: NULL argument", op);
  const uint32_t width = d.heads * d.head_dim, kv_width = d.kv_heads * d.head_dim;
  const RopeArgs a{q, k, reinterpret_cast<const float2*>(table), positions, offsets, starts, q_out, k_out, d.rows,
                   d.heads, d.kv_heads, d.head_dim, rotary, d.q_stride ? d.q_stride : width,
                   d.k_stride ? d.k_stride : kv_width, d.q_out_stride ? d.q_out_stride : width,
                   d.k_out_stride ? d.k_out_stride : kv_width, d.table_positions, d.sequences};
  if (a.q_stride < width || a.k_stride < kv_width || a.q_out_stride < width || a.k_out_stride < kv_width ||
      (a.q_stride | a.k_stride | a.q_out_stride | a.k_out_stride) % 8)
    return eg::fail(ctx, EG_ERR_INVALID, "%s: strides %u, %u, %u, %u (multiples of 8, at least a row)", op, a.q_stride,
                    a.k_stride, a.q_out_stride, a.k_out_stride);
  if (!aligned(q) || !aligned(k) || !aligned(table) || !aligned(q_out) || !aligned(k_out))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: q, k, the table and the outputs must be 16-byte aligned", op);
  const auto in_place = [&](const void* in, const void* out, uint32_t from, uint32_t to) {
    return in == nullptr || in != out || (d.in_type == d.out_type && from == to);
  };
  if (!in_place(q, q_out, a.q_stride, a.q_out_stride) || !in_place(k, k_out, a.k_stride, a.k_out_stride))
    return eg::fail(ctx, EG_ERR_INVALID, "%s: an output that is its input has its type and stride", op);
  if (!some || (d.heads == 0 && d.kv_heads == 0)) return EG_OK;
  if (d.rows >= (1u << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u rows over the grid limit", op, d.rows);
  // An output is its input, row by row, or apart from all that other workgroups read and write.
  const auto rows_of = [&](const void* at, uint32_t stride, uint32_t row, int type) {
    const uint64_t size = type == EG_ELEMENT_F32 ? 4 : 2;
    return Extent{at, d.rows, size * stride, size * row};
  };
  const Extent outputs[] = {rows_of(q_out, a.q_out_stride, width, d.out_type), rows_of(k_out, a.k_out_stride, kv_width, d.out_type)};
  const Extent inputs[] = {rows_of(q, a.q_stride, width, d.in_type), rows_of(k, a.k_stride, kv_width, d.in_type),
                           words(table, (uint64_t)d.table_positions * rotary), words(positions, d.rows),
                           words(offsets, (uint64_t)d.sequences + 1), words(starts, d.sequences)};
  for (int o = 0; o < 2; o++)
    for (int i = 0; i < 6; i++)
      if (!(i == o && outputs[o].at == inputs[i].at) && overlap(outputs[o], inputs[i]))
        return eg::fail(ctx, EG_ERR_INVALID, "%s: an output lies in an input (it may be its own, row by row)", op);
  if (overlap(outputs[0], outputs[1])) return eg::fail(ctx, EG_ERR_INVALID, "%s: q_out and k_out overlap", op);
  const OnDevice on(ctx);
  with_type(d.in_type, [&](auto ti) {
    with_type(d.out_type, [&](auto to) {
      using TI = decltype(ti);
      using TO = decltype(to);
      const auto kernel = d.layout == EG_ROPE_HALF ? rope_kernel<false, TI, TO> : rope_kernel<true, TI, TO>;
      hipLaunchKernelGGL(kernel, dim3(d.rows), dim3(kThreads), 0, ctx->stream, a);
    });
  });
  return eg::check_launch(ctx, op);
}

}  // extern "C"

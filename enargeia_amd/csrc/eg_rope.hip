// Rotary positions (enargeia_hip.h): tables of (cos, sin) with scaled frequencies, and rows rotated at positions of
// their own. Both move bytes: their floor is what they read and write once at the memory's rate.
#include <algorithm>
#include <cmath>

#include "eg_kv4.hpp"

namespace {

using namespace eg_kv4;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostDim = 512;

struct Frequencies {
  double f[kMostDim / 2];  // radians per position
};

__global__ __launch_bounds__(256) void table_kernel(float2* table, Frequencies fs, uint32_t first, uint32_t pairs,
                                                    uint64_t count, double amplitude) {
  const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  const uint32_t p = (uint32_t)(i / pairs), j = (uint32_t)(i % pairs);
  double s, c;
  sincos((double)(first + p) * fs.f[j], &s, &c);
  table[i] = make_float2((float)(amplitude * c), (float)(amplitude * s));
}

struct RopeArgs {
  const void *q, *k;
  const float2* table;
  const uint32_t *positions, *offsets, *starts;
  void *q_out, *k_out;
  uint32_t rows, heads, kv_heads, head_dim, rotary_dim;
  uint32_t q_stride, k_stride, q_out_stride, k_out_stride, table_positions, sequences;
};

template <class T>
struct alignas(16) Eight {
  T v[8];
};
template <class T>
struct alignas(sizeof(T) * 4) Four {
  T v[4];
};

// A workgroup per row; a unit is 8 elements of a head: 4 pairs, or 8 elements past the rotary part.
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
  const uint32_t per_head = a.head_dim / 8, turned = a.rotary_dim / 8;
  const uint32_t units = (a.heads + a.kv_heads) * per_head;
  for (uint32_t i = threadIdx.x; i < units; i += kThreads) {
    uint32_t head = i / per_head;
    const uint32_t u = i % per_head;
    const bool is_q = head < a.heads;
    if (!is_q) head -= a.heads;
    const TI* src = static_cast<const TI*>(is_q ? a.q : a.k) + (size_t)r * (is_q ? a.q_stride : a.k_stride) +
                    (size_t)head * a.head_dim;
    TO* dst = static_cast<TO*>(is_q ? a.q_out : a.k_out) + (size_t)r * (is_q ? a.q_out_stride : a.k_out_stride) +
              (size_t)head * a.head_dim;
    if (kInterleaved || u >= turned) {
      const Eight<TI> x = *reinterpret_cast<const Eight<TI>*>(src + 8 * u);
      Eight<TO> y;
      if (u < turned) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 t = cs[4 * u + e];
          const float p = to_f32(x.v[2 * e]), w = to_f32(x.v[2 * e + 1]);
          y.v[2 * e] = from_f32<TO>(p * t.x - w * t.y);
          y.v[2 * e + 1] = from_f32<TO>(w * t.x + p * t.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) y.v[e] = from_f32<TO>(to_f32(x.v[e]));
      }
      *reinterpret_cast<Eight<TO>*>(dst + 8 * u) = y;
    } else {
      const uint32_t half = a.rotary_dim / 2;
      const Four<TI> x = *reinterpret_cast<const Four<TI>*>(src + 4 * u);
      const Four<TI> z = *reinterpret_cast<const Four<TI>*>(src + half + 4 * u);
      Four<TO> y, w;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 t = cs[4 * u + e];
        const float p = to_f32(x.v[e]), o = to_f32(z.v[e]);
        y.v[e] = from_f32<TO>(p * t.x - o * t.y);
        w.v[e] = from_f32<TO>(o * t.x + p * t.y);
      }
      *reinterpret_cast<Four<TO>*>(dst + 4 * u) = y;
      *reinterpret_cast<Four<TO>*>(dst + half + 4 * u) = w;
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
  const uint64_t count = (uint64_t)d.positions * pairs, blocks = (count + kThreads - 1) / kThreads;
  if (blocks >= (1ull << 31) / kThreads)
    return eg::fail(ctx, EG_ERR_RANGE, "%s: %u positions of %u over the grid limit", op, d.positions, d.rotary_dim);
  if (count == 0) return EG_OK;
  const double r = d.rotary_dim;
  const double theta = d.scaling == EG_ROPE_BASE ? d.theta * std::pow(d.factor, r / (r - 2.0)) : d.theta;
  Frequencies fs{};
  for (uint32_t i = 0; i < pairs; i++) {
    double f = std::pow(theta, -2.0 * i / r);
    if (d.scaling == EG_ROPE_LINEAR) f /= d.factor;
    if (by_turns) {
      const double turns = d.context * f / (2.0 * M_PI);
      double w = d.scaling == EG_ROPE_TURNS ? (turns - d.low) / (d.high - d.low)
                                            : std::log(turns / d.low) / std::log(d.high / d.low);
      w = std::min(1.0, std::max(0.0, w));
      f = f * (w + (1.0 - w) / d.factor);
    }
    fs.f[i] = f;
  }
  const OnDevice on(ctx);
  hipLaunchKernelGGL(table_kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, ctx->stream,
                     reinterpret_cast<float2*>(table), fs, d.first, pairs, count, d.amplitude == 0.0 ? 1.0 : d.amplitude);
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

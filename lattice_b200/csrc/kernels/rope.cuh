// Rotation of a token's rows, shared by the kernels that rotate them: into the 16-bit cache
// (kernels/rope.cu) and beside the 4-bit cache's append (kernels/kv4.cu).  kernels/rope.cu has the
// arithmetic.
#pragma once

#include <cuda_runtime.h>

#include "../launch.hpp"
#include "ptx.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kRopeThreads = 128;

__device__ __forceinline__ int pair_axis(const RopeAppendArgs &a, int i) {
  if (a.axes == 1) return 0;
  if (a.interleaved) {
    const int x = i % a.axes;
    return i < a.axes * a.sections[x] ? x : 0;
  }
  int x = 0;
  for (int end = a.sections[0]; i >= end && x + 1 < a.axes; end += a.sections[x]) ++x;
  return x;
}

// Cosine and sine of pair i's angle at a token.
__device__ __forceinline__ float2 cos_sin(const RopeAppendArgs &a, int token, int i) {
  const int64_t at = pair_axis(a, i) * a.positions_stride + token;
  double s, c;
  sincos(double(a.positions[at]) * double(a.inv_freq[i]), &s, &c);
  return make_float2(float(c), float(s));
}

template <int V>
struct Chunk {
  uint16_t e[V];
};
template <int V>
__device__ __forceinline__ Chunk<V> load(const uint16_t *p) {
  Chunk<V> c;
  if constexpr (V == 8) {
    *reinterpret_cast<uint4 *>(c.e) = *reinterpret_cast<const uint4 *>(p);
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2 *>(c.e) = *reinterpret_cast<const uint2 *>(p);
  } else {
    c.e[0] = p[0];
  }
  return c;
}
template <int V>
__device__ __forceinline__ void store(uint16_t *p, const Chunk<V> &c) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(c.e);
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(c.e);
  } else {
    p[0] = c.e[0];
  }
}

template <typename T>
__device__ __forceinline__ float widen(uint16_t v) {
  return ptx::to_f32<T>(*reinterpret_cast<T *>(&v));
}
template <typename T>
__device__ __forceinline__ uint16_t narrow(float v) {
  const T t = ptx::from_f32<T>(v);
  return *reinterpret_cast<const uint16_t *>(&t);
}
template <typename T>
__device__ __forceinline__ void turn(uint16_t &x1, uint16_t &x2, float2 cs) {
  const float a = widen<T>(x1), b = widen<T>(x2);
  x1 = narrow<T>(__fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y)));
  x2 = narrow<T>(__fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, cs.y)));
}

// A unit of work is V pairs of a head (two chunks of V values), V values past rotary_dim, or V
// values of the v row.
//
// All of a token's units, each loaded, turned and stored before the next: the fewest registers, for
// many tokens.  dst: the token's row in the pages (elements), or -1.
template <typename T, int V, bool WITH_KV>
__device__ __forceinline__ void rotate_token(const RopeAppendArgs &a, int token, const float2 *cs,
                                             int64_t dst) {
  const int half = a.rotary_dim / 2, D = a.head_dim;
  const int turned = half / V, per_head = turned + (D - a.rotary_dim) / V;
  const int rows = (a.num_q_heads + (WITH_KV ? a.kv_heads : 0)) * per_head;
  const int units = rows + (WITH_KV && dst >= 0 ? a.kv_heads * D / V : 0);
  for (int u = int(threadIdx.x); u < units; u += kRopeThreads) {
    if (u >= rows) {
      const int e = (u - rows) * V;
      store<V>(static_cast<uint16_t *>(a.va_v) + dst + e,
               load<V>(static_cast<const uint16_t *>(a.v) + token * a.v_stride + e));
      continue;
    }
    const int r = u / per_head, i = u % per_head;
    const bool is_k = r >= a.num_q_heads;
    const int h = is_k ? r - a.num_q_heads : r;
    const uint16_t *src =
        is_k ? static_cast<const uint16_t *>(a.k) + token * a.k_stride + int64_t(h) * D
             : static_cast<const uint16_t *>(a.q) + token * a.q_stride_token +
                   h * a.q_stride_head;
    uint16_t *out = is_k ? a.k_out ? static_cast<uint16_t *>(a.k_out) + token * a.k_out_stride +
                                         int64_t(h) * D
                                   : nullptr
                         : static_cast<uint16_t *>(a.q_out) + token * a.q_out_stride_token +
                               h * a.q_out_stride_head;
    uint16_t *page = is_k && dst >= 0
                         ? static_cast<uint16_t *>(a.va_k) + dst + int64_t(h) * D : nullptr;
    if (i >= turned) {  // past rotary_dim: as they are
      const int e = a.rotary_dim + (i - turned) * V;
      const Chunk<V> x = load<V>(src + e);
      if (out) store<V>(out + e, x);
      if (page) store<V>(page + e, x);
      continue;
    }
    const int e0 = a.neox ? i * V : 2 * i * V, e1 = e0 + (a.neox ? half : V);
    Chunk<V> x = load<V>(src + e0), y = load<V>(src + e1);
    if (a.neox) {
#pragma unroll
      for (int j = 0; j < V; ++j) turn<T>(x.e[j], y.e[j], cs[i * V + j]);
    } else if constexpr (V == 1) {
      turn<T>(x.e[0], y.e[0], cs[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        turn<T>(x.e[2 * j], x.e[2 * j + 1], cs[i * V + j]);
        turn<T>(y.e[2 * j], y.e[2 * j + 1], cs[i * V + V / 2 + j]);
      }
    }
    if (out) {
      store<V>(out + e0, x);
      store<V>(out + e1, y);
    }
    if (page) {
      store<V>(page + e0, x);
      store<V>(page + e1, y);
    }
  }
}

// The same unit with its loads apart from the rest, so that they are under way before the token's
// cosines are there.
template <int V>
struct Unit {
  Chunk<V> x, y;
  uint16_t *out;       // of the row (x at e0, y at e1), or null
  int e0, e1;          // of x and y in the row; e1 < 0: x alone, not turned
  int page;            // element of the row in the token's page row, or -1
  int pair;            // first pair of x
  bool is_v;
};
struct TokenUnits {
  int turned, per_head, rows, all;  // units of a head (turned ones first), of q and k, and in all
};
template <int V>
__device__ __forceinline__ TokenUnits token_units(const RopeAppendArgs &a) {
  TokenUnits t;
  t.turned = a.rotary_dim / 2 / V;
  t.per_head = t.turned + (a.head_dim - a.rotary_dim) / V;
  t.rows = (a.num_q_heads + a.kv_heads) * t.per_head;
  t.all = t.rows + a.kv_heads * a.head_dim / V;
  return t;
}
template <int V>
__device__ __forceinline__ void fetch(const RopeAppendArgs &a, const TokenUnits &t, int token,
                                      int u, Unit<V> *w) {
  const int D = a.head_dim;
  w->out = nullptr;
  w->e1 = -1;
  w->is_v = u >= t.rows;
  if (w->is_v) {
    w->e0 = (u - t.rows) * V;
    w->page = 0;
    w->x = load<V>(static_cast<const uint16_t *>(a.v) + token * a.v_stride + w->e0);
    return;
  }
  const int r = u / t.per_head, i = u - r * t.per_head;
  const bool is_k = r >= a.num_q_heads;
  const int h = is_k ? r - a.num_q_heads : r;
  const uint16_t *src;
  if (is_k) {
    src = static_cast<const uint16_t *>(a.k) + token * a.k_stride + int64_t(h) * D;
    if (a.k_out) w->out = static_cast<uint16_t *>(a.k_out) + token * a.k_out_stride + int64_t(h) * D;
  } else {
    src = static_cast<const uint16_t *>(a.q) + token * a.q_stride_token + h * a.q_stride_head;
    w->out = static_cast<uint16_t *>(a.q_out) + token * a.q_out_stride_token +
             h * a.q_out_stride_head;
  }
  w->page = is_k ? h * D : -1;
  if (i >= t.turned) {
    w->e0 = a.rotary_dim + (i - t.turned) * V;
  } else {
    w->pair = i * V;
    w->e0 = a.neox ? i * V : 2 * i * V;
    w->e1 = w->e0 + (a.neox ? a.rotary_dim / 2 : V);
    w->y = load<V>(src + w->e1);
  }
  w->x = load<V>(src + w->e0);
}
// page: the token's row in K's and V's pages, or null
template <typename T, int V>
__device__ __forceinline__ void finish(const RopeAppendArgs &a, const float2 *cs, Unit<V> &w,
                                       uint16_t *page_k, uint16_t *page_v) {
  uint16_t *page = w.page < 0 ? nullptr : w.is_v ? page_v : page_k;
  if (page) page += w.page;
  if (w.e1 >= 0) {
    if (a.neox) {
#pragma unroll
      for (int j = 0; j < V; ++j) turn<T>(w.x.e[j], w.y.e[j], cs[w.pair + j]);
    } else if constexpr (V == 1) {
      turn<T>(w.x.e[0], w.y.e[0], cs[w.pair]);
    } else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        turn<T>(w.x.e[2 * j], w.x.e[2 * j + 1], cs[w.pair + j]);
        turn<T>(w.y.e[2 * j], w.y.e[2 * j + 1], cs[w.pair + V / 2 + j]);
      }
    }
    if (w.out) store<V>(w.out + w.e1, w.y);
    if (page) store<V>(page + w.e1, w.y);
  }
  if (w.out) store<V>(w.out + w.e0, w.x);
  if (page) store<V>(page + w.e0, w.x);
}

}  // namespace
}  // namespace dev
}  // namespace kcmm

// Rotary positions with one or several axes, and the append that follows them, in one call.
//
// A row's pair i turns by p * inv_freq[i], p the token's position on the pair's axis:
//   x1' = x1 cos - x2 sin,  x2' = x2 cos + x1 sin
// The angle and its sine and cosine are computed in 64 bits (a position times a frequency of 24
// bits has up to 55) and rounded once to 32; the products and sums are 32-bit operations, each
// rounded, so that a row comes out the same wherever it is computed; x' is rounded once to the
// rows' 16-bit type.  The 4-bit cache quantises the rounded rows.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../launch.hpp"
#include "pdl.cuh"
#include "ptx.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kThreads = 128;

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

// Element offset of the token's row in its page, or -1 (nothing to write; a status as for the
// slot write where the slot is no row of the cache).
template <int V>
__device__ __forceinline__ int64_t page_row(const RopeAppendArgs &a, int token) {
  const int64_t slot = a.slot_mapping[token];
  if (slot < 0) return -1;
  const int64_t blk = slot / a.block_size, row = int64_t(a.kv_heads) * a.head_dim;
  int bad = 0;
  int64_t dst = -1;
  if (blk >= a.offsets_len) {
    bad = 1;
  } else if (a.valid && !a.valid[blk]) {
    bad = 2;
  } else {
    const uint64_t off = a.block_offsets[blk];
    dst = int64_t(off) + (slot - blk * a.block_size) * row;
    if (off > a.region_elems || uint64_t(dst + row) > a.region_elems || dst % V != 0) bad = 3;
  }
  if (bad == 0) return dst;
  if (a.status) atomicCAS(a.status, 0, bad);
  return -1;
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

// One CTA a token.  A unit of work is V pairs of a head (two chunks of V values), V values
// past rotary_dim, or V values of the v row.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeAppendArgs a) {
  __shared__ float2 s_cs[128];
  __shared__ int64_t s_dst;
  const int token = int(blockIdx.x), tid = int(threadIdx.x);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int half = a.rotary_dim / 2;
  if (tid < half) {
    const int64_t at = pair_axis(a, tid) * a.positions_stride + token;
    double s, c;
    sincos(double(a.positions[at]) * double(a.inv_freq[tid]), &s, &c);
    s_cs[tid] = make_float2(float(c), float(s));
  }
  if (tid == kThreads - 1) s_dst = a.va_k ? page_row<V>(a, token) : -1;
  __syncthreads();
  const int64_t dst = s_dst;
  const int D = a.head_dim;
  const int turned = half / V, per_head = turned + (D - a.rotary_dim) / V;
  const int rows = (a.num_q_heads + a.kv_heads) * per_head;
  const int units = rows + (dst >= 0 ? a.kv_heads * D / V : 0);
  for (int u = tid; u < units; u += kThreads) {
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
      for (int j = 0; j < V; ++j) turn<T>(x.e[j], y.e[j], s_cs[i * V + j]);
    } else if constexpr (V == 1) {
      turn<T>(x.e[0], y.e[0], s_cs[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        turn<T>(x.e[2 * j], x.e[2 * j + 1], s_cs[i * V + j]);
        turn<T>(y.e[2 * j], y.e[2 * j + 1], s_cs[i * V + V / 2 + j]);
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

// Values of an access: 8 or 4 where rows, heads and the halves of a rotated row allow it.
int vector_width(const RopeAppendArgs &a) {
  for (int v : {8, 4}) {
    const uint64_t bytes = uint64_t(v) * 2 - 1;
    uint64_t at = reinterpret_cast<uint64_t>(a.k) | reinterpret_cast<uint64_t>(a.v) |
                  reinterpret_cast<uint64_t>(a.k_out);
    int64_t strides = a.k_stride | a.v_stride | a.k_out_stride;
    if (a.num_q_heads) {
      at |= reinterpret_cast<uint64_t>(a.q) | reinterpret_cast<uint64_t>(a.q_out);
      strides |= a.q_stride_token | a.q_stride_head | a.q_out_stride_token | a.q_out_stride_head;
    }
    if ((at & bytes) == 0 && strides % v == 0 && a.head_dim % v == 0 && a.rotary_dim % (2 * v) == 0)
      return v;
  }
  return 1;
}

template <typename T>
cudaError_t launch(const RopeAppendArgs &a, cudaStream_t stream) {
  const int v = vector_width(a);
  auto fn = v == 8 ? rope_kernel<T, 8> : v == 4 ? rope_kernel<T, 4> : rope_kernel<T, 1>;
  return launch_pdl(fn, dim3(uint32_t(a.num_tokens)), dim3(kThreads), 0, stream, a);
}

}  // namespace

cudaError_t rope_append(const RopeAppendArgs &args, cudaStream_t stream) {
  RopeAppendArgs a = args;
  const bool bf16 = a.dtype == Dtype::BF16;
  auto rotate = [&] {
    return bf16 ? launch<__nv_bfloat16>(a, stream) : launch<__half>(a, stream);
  };
  if (!a.kv4) return rotate();
  // the 4-bit cache takes the rotated rows from k_out, or from scratch
  const int64_t row = int64_t(a.kv_heads) * a.head_dim;
  CallScratch scratch;
  if (!a.k_out) {
    const cudaError_t e = scratch.acquire(stream, size_t(a.num_tokens) * row * 2);
    if (e != cudaSuccess) return e;
    a.k_out = scratch.ptr;
    a.k_out_stride = row;
  }
  Kv4RowsArgs c = {};
  c.dtype = a.dtype;
  c.va_k = a.va_k;
  c.va_v = a.va_v;
  c.region_bytes = a.region_elems * 2;
  c.slot_mapping = a.slot_mapping;
  c.block_offsets = a.block_offsets;
  c.valid = a.valid;
  c.offsets_len = a.offsets_len;
  c.num_tokens = a.num_tokens;
  c.kv_heads = a.kv_heads;
  c.head_dim = a.head_dim;
  c.block_size = a.block_size;
  c.k = a.k_out;
  c.v = const_cast<void *>(a.v);
  c.k_stride = a.k_out_stride;
  c.v_stride = a.v_stride;
  c.status = a.status;
  c.vec = ((reinterpret_cast<uint64_t>(a.k_out) | reinterpret_cast<uint64_t>(a.v)) & 15) == 0 &&
          a.k_out_stride % 8 == 0 && a.v_stride % 8 == 0;
  a.va_k = a.va_v = nullptr;
  cudaError_t e = rotate();
  if (e == cudaSuccess) e = kv4_append(c, stream);
  const cudaError_t r = scratch.ptr ? scratch.release(stream) : cudaSuccess;
  return e != cudaSuccess ? e : r;
}

}  // namespace dev
}  // namespace kcmm

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
#include "rope.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kFewCtas = 4;  // an SM, up to which a token is cut into parts

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

// The cosines of the CTA's token and its row in the pages, seen by all threads afterwards.
template <int V>
__device__ __forceinline__ void token_setup(const RopeAppendArgs &a, float2 *s_cs,
                                            int64_t *s_dst) {
  const int token = int(blockIdx.x), tid = int(threadIdx.x);
  if (tid < a.rotary_dim / 2) s_cs[tid] = cos_sin(a, token, tid);
  if (tid == kRopeThreads - 1) *s_dst = a.va_k ? page_row<V>(a, token) : -1;
  __syncthreads();
}

// Many tokens, a CTA each: bound by HBM, for which the loads of many small CTAs suffice.
template <typename T, int V>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeAppendArgs a) {
  __shared__ float2 s_cs[128];
  __shared__ int64_t s_dst;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  token_setup<V>(a, s_cs, &s_dst);
  rotate_token<T, V, true>(a, int(blockIdx.x), s_cs, s_dst);
}

// A few tokens are bound by the latency of a CTA's steps (slot -> page; positions -> cosines;
// rows).  So CTAs (tokens, parts), a part of the token's units each, and a thread's first loads
// under way before the cosines: 64 tokens of 32 + 8 heads of 128 take 5.4 us, with the kernel above
// 7.0.  (Many tokens take longer so, since the loads' registers cost CTAs an SM: 16,384 take 84 us
// against 69.)
template <typename T, int V>
__global__ void __launch_bounds__(kRopeThreads) rope_few_kernel(const RopeAppendArgs a) {
  __shared__ float2 s_cs[128];
  __shared__ int64_t s_dst;
  const int token = int(blockIdx.x);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const TokenUnits t = token_units<V>(a);
  const int end = int(int64_t(t.all) * (blockIdx.y + 1) / gridDim.y);
  int u = int(int64_t(t.all) * blockIdx.y / gridDim.y) + int(threadIdx.x);
  Unit<V> w;
  if (u < end) fetch<V>(a, t, token, u, &w);
  token_setup<V>(a, s_cs, &s_dst);
  uint16_t *page_k = nullptr, *page_v = nullptr;
  if (s_dst >= 0) {
    page_k = static_cast<uint16_t *>(a.va_k) + s_dst;
    page_v = static_cast<uint16_t *>(a.va_v) + s_dst;
  }
  while (u < end) {
    finish<T, V>(a, s_cs, w, page_k, page_v);
    u += kRopeThreads;
    if (u < end) fetch<V>(a, t, token, u, &w);
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
  const int units = (a.num_q_heads + 2 * a.kv_heads) * a.head_dim / (2 * v);  // about
  const int parts = std::max(1, std::min(kFewCtas * device_sm_count() / a.num_tokens,
                                         (units + kRopeThreads - 1) / kRopeThreads));
  auto many = v == 8 ? rope_kernel<T, 8> : v == 4 ? rope_kernel<T, 4> : rope_kernel<T, 1>;
  auto few = v == 8   ? rope_few_kernel<T, 8>
             : v == 4 ? rope_few_kernel<T, 4>
                      : rope_few_kernel<T, 1>;
  return launch_pdl(parts > 1 ? few : many, dim3(uint32_t(a.num_tokens), uint32_t(parts)),
                    dim3(kRopeThreads), 0, stream, a);
}

}  // namespace

cudaError_t rope_append(const RopeAppendArgs &args, cudaStream_t stream) {
  RopeAppendArgs a = args;
  const bool bf16 = a.dtype == Dtype::BF16;
  auto rotate = [&] {
    return bf16 ? launch<__nv_bfloat16>(a, stream) : launch<__half>(a, stream);
  };
  if (!a.kv4) return rotate();
  const int64_t row = int64_t(a.kv_heads) * a.head_dim;
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
  c.k = const_cast<void *>(a.k);
  c.v = const_cast<void *>(a.v);
  c.k_stride = a.k_stride;
  c.v_stride = a.v_stride;
  c.status = a.status;
  c.vec = true;
  if (vector_width(a) == 8 && (a.k_out != a.k || 32 % (a.head_dim / 8) == 0)) {
    const cudaError_t e = kv4_rope_append(c, a, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  // Many tokens, and rows off their alignment: rotated first, to k_out or scratch, then appended.
  CallScratch scratch;
  if (!a.k_out) {
    const cudaError_t e = scratch.acquire(stream, size_t(a.num_tokens) * row * 2);
    if (e != cudaSuccess) return e;
    a.k_out = scratch.ptr;
    a.k_out_stride = row;
  }
  c.k = a.k_out;
  c.k_stride = a.k_out_stride;
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

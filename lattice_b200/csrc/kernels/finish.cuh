// Second pass of the split decodes that keep attention weights (kernels/decode.cu,
// kernels/kv4.cu): merges the splits' partial outputs through their log-sum-exp and, where
// the call asks for them, adds every cached token's softmax weight to its accumulated one:
//   w_out[b,g,t] = w_in[b,g,t] + sum over the query heads h of kv head g of
//                  exp2(score[b,h,t] - lse[b,h])
// The first pass leaves the scores (log2 units, 32 bits) in scratch, since a weight needs
// the whole row's sum: 8 bytes a head and token beside the 36 to 512 bytes of K and V
// that the row costs, instead of reading K a second time.  Bound by latency and the scores'
// traffic: 13 us for 64 sequences of 512 to 4096 tokens with 32 heads on 8 (19 MB of scores,
// 9 MB of weights both ways), where the first pass takes 116.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../launch.hpp"
#include "pdl.cuh"
#include "ptx.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kFinishThreads = 256;
constexpr int kFinishTokens = 1024;   // tokens of one CTA: 4 a thread
constexpr int kFinishMaxGroup = 256;  // query heads of one kv head

struct FinishParams {
  const int32_t *seq_lens;
  int max_tokens;  // seq_lens are capped to this
  int hq, hkv, head_dim;
  int num_splits, tokens_per_split;
  const float *part_o;    // [b * hq + h][num_splits][head_dim], each split normalised; null:
                          // the output is done, part_lse has the rows' own
  const float *part_lse;  // [b * hq + h][num_splits], log2 units
  void *out;
  int64_t o_sb, o_sh;
  const float *scores;  // [b * hq + h][score_stride], or null: no weights
  int64_t score_stride;
  const float *w_in;  // [b][hkv][w_stride]
  float *w_out;
  int64_t w_stride;
  bool w_vec;  // rows of weights start on 16 bytes
};

// Grid (token chunks, hkv, batch).  Every CTA computes the log-sum-exp of its group's
// heads from the splits' (at most num_splits values a head), the first chunk's CTA merges
// the outputs.  Sequences of length 0 are left untouched.  A split none of whose pages could be
// read has log-sum-exp and scores of -inf and weighs nothing; where that is so of all of a row's
// tokens its output is 0.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const FinishParams p) {
  __shared__ float s_lse[kFinishMaxGroup];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int len = min(p.seq_lens[b], p.max_tokens);
  const int t0 = int(blockIdx.x) * kFinishTokens;
  if (len <= 0 || (t0 >= len && blockIdx.x > 0)) return;
  const int lo = int((int64_t(kvh) * p.hq + p.hkv - 1) / p.hkv);
  const int G = int((int64_t(kvh + 1) * p.hq + p.hkv - 1) / p.hkv) - lo;
  const int ns = (len + p.tokens_per_split - 1) / p.tokens_per_split;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int h = warp; h < G; h += kFinishThreads / 32) {
    const float *lse = p.part_lse + (int64_t(b) * p.hq + lo + h) * p.num_splits;
    float M = -INFINITY;
    bool nan = false;
    for (int s = lane; s < ns; s += 32) {
      M = fmaxf(M, lse[s]);
      nan |= lse[s] != lse[s];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    nan = __any_sync(0xffffffffu, nan);
    float sum = 0.f;
    for (int s = lane; s < ns; s += 32) sum += ptx::fast_exp2(lse[s] - M);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // exp2(-inf - (+inf)) = 0
    const float total = M == -INFINITY && !nan ? INFINITY : M + log2f(sum);
    if (lane == 0) s_lse[h] = total;
  }
  __syncthreads();
  if (blockIdx.x == 0 && p.part_o) {
    const int D = p.head_dim, quads = D / 4;
    for (int i = threadIdx.x; i < G * quads; i += kFinishThreads) {
      const int h = i / quads, d = (i - h * quads) * 4;
      const int64_t row = (int64_t(b) * p.hq + lo + h) * p.num_splits;
      const float total = s_lse[h];
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < ns; ++s) {
        const float lse = p.part_lse[row + s];
        const float w = ptx::fast_exp2(lse - total);
        float4 v = *reinterpret_cast<const float4 *>(p.part_o + (row + s) * D + d);
        if (lse == -INFINITY) v = make_float4(0.f, 0.f, 0.f, 0.f);  // it normalised no tokens
        acc.x += v.x * w;
        acc.y += v.y * w;
        acc.z += v.z * w;
        acc.w += v.w * w;
      }
      T *dst = static_cast<T *>(p.out) + int64_t(b) * p.o_sb + int64_t(lo + h) * p.o_sh + d;
      dst[0] = ptx::from_f32<T>(acc.x);
      dst[1] = ptx::from_f32<T>(acc.y);
      dst[2] = ptx::from_f32<T>(acc.z);
      dst[3] = ptx::from_f32<T>(acc.w);
    }
  }
  if (!p.scores) return;
  const float *sc = p.scores + (int64_t(b) * p.hq + lo) * p.score_stride;
  const int64_t wrow = (int64_t(b) * p.hkv + kvh) * p.w_stride;
  // a weights row of w_stride entries holds the weights of the first w_stride tokens
  const int t1 = int(min(int64_t(min(len, t0 + kFinishTokens)), p.w_stride));
  const int t = t0 + int(threadIdx.x) * 4;
  if (t >= t1) return;
  __align__(16) float w[4] = {0.f, 0.f, 0.f, 0.f};
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  const float *w_in = p.w_in + wrow + t;
  float *w_out = p.w_out + wrow + t;
  const bool vec = p.w_vec && t + 4 <= t1;
  if (vec) {
    *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(w_in);
  } else {
    for (int i = 0; i < 4 && t + i < t1; ++i) w[i] = w_in[i];
  }
  // rows of scores are whole units long: reading past the last token stays inside
#pragma unroll 4
  for (int h = 0; h < G; ++h) {
    const float4 x = *reinterpret_cast<const float4 *>(sc + h * p.score_stride + t);
    const float lse = s_lse[h];
    sum[0] += ptx::fast_exp2(x.x - lse);
    sum[1] += ptx::fast_exp2(x.y - lse);
    sum[2] += ptx::fast_exp2(x.z - lse);
    sum[3] += ptx::fast_exp2(x.w - lse);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] += sum[i];
  if (vec) {
    *reinterpret_cast<float4 *>(w_out) = *reinterpret_cast<const float4 *>(w);
  } else {
    for (int i = 0; i < 4 && t + i < t1; ++i) w_out[i] = w[i];
  }
}

inline cudaError_t launch_finish(Dtype dtype, FinishParams f, int batch, cudaStream_t stream) {
  f.w_vec = ((reinterpret_cast<uintptr_t>(f.w_in) | reinterpret_cast<uintptr_t>(f.w_out)) & 15) == 0 &&
            f.w_stride % 4 == 0;
  const int chunks = f.scores ? (f.max_tokens + kFinishTokens - 1) / kFinishTokens : 1;
  return launch_pdl(dtype == Dtype::BF16 ? finish_kernel<__nv_bfloat16> : finish_kernel<__half>,
                    dim3(chunks, f.hkv, batch), dim3(kFinishThreads), 0, stream, f);
}

}  // namespace
}  // namespace dev
}  // namespace kcmm

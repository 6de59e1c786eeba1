// Beam search: the n best of beams x vocabulary, and the beams' states gathered by parent.
//
//   score(k, v) = scores_in[k] + logits[k,v] - max_k - log sum_v exp(logits[k,v] - max_k)
//   (scores_out, parents, tokens) = the n largest over (k, v), ties to the lowest (k, v)
// A NaN logit counts as -inf and +inf as the largest finite value; a beam without a finite
// logit scores -inf everywhere.  A finished beam has the one candidate (k, eos) of its own
// score; its other tokens score -inf.
//
// Pass 1 reads the logits once, 64 bytes a thread, and keeps of each chunk the running
// maximum and sum of the softmax and the n largest logits: the n-th largest of the threads'
// own maxima bounds them from below, so that a second look at the registers leaves little
// more than n to sort.  It is bound by HBM for large vocabularies and by latency for small
// ones.  Pass 2 scores and ranks a request's beams x chunks x n candidates.
#include <cuda_runtime.h>

#include <algorithm>

#include "../launch.hpp"
#include "pdl.cuh"
#include "ptx.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVecs = 4;                                // 16-byte loads of a thread
constexpr int kChunkBytes = kThreads * kVecs * 16;      // logits of one CTA of pass 1
constexpr int kMaxSelect = kBeamMaxSelect;

// (value, index) as one key: larger value first, then lower index.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long make_key(float x, uint32_t index) {
  return (static_cast<unsigned long long>(value_key(x)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) {
  return 0xffffffffu - uint32_t(k);
}
__device__ __forceinline__ float clean(float x) {
  return x == x ? fminf(x, 3.402823466e38f) : -INFINITY;
}

// The largest of the warp's keys (0 = none).
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

struct TopShared {
  unsigned long long warp_top[kWarps * kMaxSelect];
  unsigned long long bound;
  int count;
};

// The n-th largest of the CTA's per-thread maxima `mine` (0 = the thread has no key; keys
// differ), or 0 if there are fewer than n.  At least n keys of the CTA are >= it, and only
// threads whose maximum is >= it (at most n) hold such keys.
__device__ unsigned long long nth_maximum(unsigned long long mine, int n, TopShared *sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = min(n, 32);  // of a warp's 32 maxima at most 32 count
  unsigned long long k = mine;
  for (int r = 0; r < m; ++r) {
    const unsigned long long top = warp_max(k);
    if (lane == 0) sh->warp_top[warp * kMaxSelect + r] = top;
    if (k == top) k = 0;
  }
  __syncthreads();
  // rank of every warp's r-th maximum among all: how many are larger
  const int total = kWarps * m;
  if (threadIdx.x == 0) sh->bound = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const unsigned long long x = sh->warp_top[(i / m) * kMaxSelect + i % m];
    int larger = 0;
    for (int w = 0; w < kWarps; ++w) {
      // a warp's list descends: count its entries above x
      const unsigned long long *l = sh->warp_top + w * kMaxSelect;
      int lo = 0, hi = m;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (l[mid] > x) {
          lo = mid + 1;
        } else {
          hi = mid;
        }
      }
      larger += lo;
    }
    if (x != 0 && larger == n - 1) sh->bound = x;
  }
  __syncthreads();
  return sh->bound;
}

template <typename T>
__device__ __forceinline__ float widen(T x) {
  return ptx::to_f32(x);
}
template <>
__device__ __forceinline__ float widen<float>(float x) {
  return x;
}

// Grid (chunks, rows), a row being one beam of one request.
template <typename T>
__global__ void __launch_bounds__(kThreads) beam_chunk_kernel(const BeamArgs a) {
  constexpr int PER = 16 / sizeof(T);  // logits of a load
  constexpr int MOST = kVecs * PER;    // of a thread
  __shared__ TopShared sh;
  __shared__ unsigned long long s_list[kMaxSelect * MOST];
  __shared__ float s_red[kWarps];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31;
  if (a.finished && a.finished[row]) return;  // pass 2 knows its one candidate
  const T *base = static_cast<const T *>(a.logits) + int64_t(row) * a.row_stride;
  // 16-byte blocks counted from the one that holds the row's first logit
  const int lead = int((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  const int64_t first = int64_t(chunk) * (kChunkBytes / int(sizeof(T))) - lead;
  if (first >= a.vocab) {  // an aligned row needs no chunk for its lead
    if (tid == 0) a.part[int64_t(row) * a.chunks + chunk] = make_float2(-INFINITY, 0.f);
    if (tid < a.n) a.cand[(int64_t(row) * a.chunks + chunk) * a.n + tid] = 0ull;
    return;
  }
  alignas(16) T x[kVecs][PER];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int64_t at = first + (int64_t(i) * kThreads + tid) * PER;
    if (at >= 0 && at + PER <= a.vocab) {
      *reinterpret_cast<uint4 *>(x[i]) = __ldcs(reinterpret_cast<const uint4 *>(base + at));
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (at + e >= 0 && at + e < a.vocab) x[i][e] = base[at + e];
    }
  }
  unsigned long long mine = 0;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int64_t at = first + (int64_t(i) * kThreads + tid) * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (at + e < 0 || at + e >= a.vocab) continue;
      const float v = clean(widen(x[i][e]));
      mx = fmaxf(mx, v);
      const unsigned long long k = make_key(v, uint32_t(at + e));
      mine = k > mine ? k : mine;
    }
  }
  // maximum and sum of the chunk
  float m = mx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s_red[warp] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_red[w]);
  float sum = 0.f;
  if (m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int64_t at = first + (int64_t(i) * kThreads + tid) * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (at + e >= 0 && at + e < a.vocab) sum += __expf(clean(widen(x[i][e])) - m);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) s_red[warp] = sum;
  if (tid == 0) sh.count = 0;
  const unsigned long long bound = nth_maximum(mine, a.n, &sh);  // synchronises
  if (tid == 0) {
    float total = 0.f;
    for (int w = 0; w < kWarps; ++w) total += s_red[w];
    a.part[int64_t(row) * a.chunks + chunk] = make_float2(m, total);
  }
  if (mine != 0 && mine >= bound) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int64_t at = first + (int64_t(i) * kThreads + tid) * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (at + e < 0 || at + e >= a.vocab) continue;
        const unsigned long long k = make_key(clean(widen(x[i][e])), uint32_t(at + e));
        if (k >= bound) s_list[atomicAdd(&sh.count, 1)] = k;
      }
    }
  }
  __syncthreads();
  const int count = sh.count;
  unsigned long long *cand = a.cand + (int64_t(row) * a.chunks + chunk) * a.n;
  for (int i = tid; i < max(count, a.n); i += kThreads) {
    if (i >= count) {
      cand[i] = 0ull;  // fewer than n logits in the chunk
      continue;
    }
    const unsigned long long k = s_list[i];
    int larger = 0;
    for (int j = 0; j < count; ++j) larger += s_list[j] > k;
    if (larger < a.n) cand[larger] = k;
  }
}

constexpr int kBestThreads = 256;

// One CTA a request.
__global__ void __launch_bounds__(kBestThreads) beam_best_kernel(const BeamArgs a) {
  __shared__ TopShared sh;
  extern __shared__ float2 s_norm[];  // [beams]: max, log of the sum
  __shared__ unsigned long long s_best[kMaxSelect];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int k = warp; k < a.beams; k += kBestThreads / 32) {
    const int row = b * a.beams + k;
    if (a.finished && a.finished[row]) continue;
    const float2 *part = a.part + int64_t(row) * a.chunks;
    float M = -INFINITY;
    for (int i = lane; i < a.chunks; i += 32) M = fmaxf(M, part[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float sum = 0.f;
    if (M != -INFINITY)
      for (int i = lane; i < a.chunks; i += 32) sum += part[i].y * __expf(part[i].x - M);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_norm[k] = make_float2(M, logf(sum));
  }
  __syncthreads();
  // candidate i of the request: beam, then chunk, then rank; a finished beam's are its eos
  // and its lowest other tokens
  const int per_beam = a.chunks * a.n, total = a.beams * per_beam;
  auto candidate = [&](int i) -> unsigned long long {
    const int k = i / per_beam, r = i - k * per_beam, row = b * a.beams + k;
    float score = a.scores_in[row];
    uint32_t token;
    if (a.finished && a.finished[row]) {
      if (r >= a.n || r >= a.vocab) return 0ull;
      token = r == 0 ? a.eos : r <= a.eos ? r - 1 : r;
      if (r > 0) score = -INFINITY;
    } else {
      const unsigned long long c = a.cand[int64_t(row) * a.chunks * a.n + r];
      if (c == 0ull) return 0ull;
      token = key_index(c);
      const float x = key_value(uint32_t(c >> 32));
      score = x == -INFINITY ? -INFINITY : ((x - s_norm[k].x) - s_norm[k].y) + score;
    }
    if (!(score == score)) score = -INFINITY;
    return make_key(score, uint32_t(k) * uint32_t(a.vocab) + token);
  };
  // repeatedly the n-th largest of the threads' maxima bounds the result from below; the
  // keys at or above it fit n per thread, and the list is drained in rounds of one key a
  // thread in descending order
  unsigned long long cut = ~0ull;  // keys below it are left
  int done = 0;
  while (done < a.n) {
    unsigned long long mine = 0;
    for (int i = tid; i < total; i += kBestThreads) {
      const unsigned long long k = candidate(i);
      if (k < cut && k > mine) mine = k;
    }
    const int left = a.n - done;
    if (tid == 0) sh.count = 0;
    const unsigned long long bound = nth_maximum(mine, left, &sh);
    // Thread maxima at or above the bound are not yet the result: a thread may hold a second
    // key above another's maximum.  Those down to the largest second key are final.
    unsigned long long second = 0;
    if (mine != 0 && mine >= bound)
      for (int i = tid; i < total; i += kBestThreads) {
        const unsigned long long k = candidate(i);
        if (k < mine && k > second) second = k;
      }
    const unsigned long long top = warp_max(second);
    __syncthreads();
    if (lane == 0) sh.warp_top[warp] = top;
    __syncthreads();
    unsigned long long floor_key = 0;
    for (int w = 0; w < kBestThreads / 32; ++w)
      floor_key = sh.warp_top[w] > floor_key ? sh.warp_top[w] : floor_key;
    const unsigned long long take = bound > floor_key ? bound : floor_key + 1;
    __syncthreads();
    unsigned long long *maxima = sh.warp_top;  // [kBestThreads], reused
    maxima[tid] = mine != 0 && mine >= take ? mine : 0ull;
    __syncthreads();
    if (maxima[tid] != 0) {
      int larger = 0;
      for (int t = 0; t < kBestThreads; ++t) larger += maxima[t] > maxima[tid];
      if (larger < left) {
        s_best[done + larger] = maxima[tid];
        atomicAdd(&sh.count, 1);
      }
    }
    __syncthreads();
    if (sh.count == 0) break;  // no candidate is left
    done += sh.count;
    cut = s_best[done - 1];
    __syncthreads();
  }
  if (tid < done) {
    const unsigned long long k = s_best[tid];
    const uint32_t i = key_index(k);
    const int64_t at = int64_t(b) * a.n + tid;
    a.scores_out[at] = key_value(uint32_t(k >> 32));
    a.parents[at] = int32_t(i / uint32_t(a.vocab));
    a.tokens[at] = int32_t(i % uint32_t(a.vocab));
  }
}

// dst row (b, j) = src row (b, parents[b, j]); with tokens, its entry token_index = tokens[b, j].
// Grid (pieces, batch * n).
__global__ void beam_gather_kernel(const BeamGatherArgs a) {
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int row = blockIdx.y, b = row / a.n;
  const int parent = a.parents[row];
  if (parent < 0 || parent >= a.beams) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.diag, int32_t(kDiagBadLaunch));
    return;
  }
  const uint8_t *src = a.src + (int64_t(b) * a.beams + parent) * a.row_bytes;
  uint8_t *dst = a.dst + int64_t(row) * a.row_bytes;
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  const int64_t at = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t token_at = a.tokens ? a.token_index * 4 : -16;
  if (a.vec) {
    for (int64_t i = at * 16; i < a.row_bytes; i += step * 16) {
      uint4 v = *reinterpret_cast<const uint4 *>(src + i);
      if (token_at >= i && token_at < i + 16) {
        const uint32_t t = uint32_t(a.tokens[row]);
        const int e = int(token_at - i) / 4;
        v.x = e == 0 ? t : v.x;
        v.y = e == 1 ? t : v.y;
        v.z = e == 2 ? t : v.z;
        v.w = e == 3 ? t : v.w;
      }
      *reinterpret_cast<uint4 *>(dst + i) = v;
    }
  } else {
    for (int64_t i = at * 4; i < a.row_bytes; i += step * 4)
      *reinterpret_cast<uint32_t *>(dst + i) =
          i == token_at ? uint32_t(a.tokens[row]) : *reinterpret_cast<const uint32_t *>(src + i);
  }
}

}  // namespace

cudaError_t beam_select(const BeamArgs &args, cudaStream_t stream) {
  BeamArgs a = args;
  const int elem = a.type == 2 ? 4 : 2;
  const int64_t per = kChunkBytes / elem;
  // an unaligned row's first block starts before it
  const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
                       a.row_stride * elem % 16 == 0;
  a.chunks = int((a.vocab + (aligned ? 0 : 16 / elem - 1) + per - 1) / per);
  const int rows = a.batch * a.beams;
  const size_t cand_bytes = size_t(rows) * a.chunks * a.n * 8;
  CallScratch scratch;
  cudaError_t e = scratch.acquire(stream, cand_bytes + size_t(rows) * a.chunks * 8);
  if (e != cudaSuccess) return e;
  a.cand = static_cast<unsigned long long *>(scratch.ptr);
  a.part = reinterpret_cast<float2 *>(static_cast<char *>(scratch.ptr) + cand_bytes);
  const dim3 grid(a.chunks, rows);
  e = launch_pdl(a.type == 0   ? beam_chunk_kernel<__half>
                 : a.type == 1 ? beam_chunk_kernel<__nv_bfloat16>
                               : beam_chunk_kernel<float>,
                 grid, dim3(kThreads), 0, stream, a);
  if (e == cudaSuccess)
    e = launch_pdl(beam_best_kernel, dim3(a.batch), dim3(kBestThreads),
                   size_t(a.beams) * sizeof(float2), stream, a);
  const cudaError_t r = scratch.release(stream);
  return e != cudaSuccess ? e : r;
}

cudaError_t beam_gather(const BeamGatherArgs &a, cudaStream_t stream) {
  const int64_t items = a.row_bytes / (a.vec ? 16 : 4);
  const int threads = int(std::min<int64_t>(256, (items + 31) / 32 * 32));
  const int pieces = int(std::min<int64_t>((items + threads - 1) / threads, 64));
  return launch_pdl(beam_gather_kernel, dim3(pieces, a.batch * a.n), dim3(threads), 0, stream, a);
}

}  // namespace dev
}  // namespace kcmm

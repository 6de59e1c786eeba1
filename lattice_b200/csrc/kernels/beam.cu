// Beam search: the n best of beams x vocabulary, and the beams' states gathered by parent.
//
//   score(k, v) = scores_in[k] + logits[k,v] - max_k - log sum_v exp(logits[k,v] - max_k)
//   (scores_out, parents, tokens) = the n largest over (k, v), ties to the lowest (k, v)
// A NaN logit counts as -inf and +inf as the largest finite value; a beam without a finite
// logit scores -inf everywhere.  A finished beam has the one candidate (k, eos) of its own
// score; its other tokens score -inf.
//
// A CTA reads 16 KB of a beam's logits once, 64 bytes a thread, and keeps the chunk's
// maximum, its sum of exponentials and its n largest logits: the n-th largest of its warps'
// maxima (its threads', where n is above 8) bounds those from below, so that a second look at
// the registers leaves little more than n to sort.  The last CTA of a request scores and ranks
// its beams x chunks x n candidates in the same way.  Bounds from all threads' maxima cost a
// second pass wherever 16-bit maxima were equal: 7 us of the 24 that 16 requests of 4 beams over
// 128,256 bf16 logits took, the gathers of histories and tables included.
//
// Different logits can round to one score (scores of -inf, or large beside the logits' steps), and
// then the lower token comes first though its logit is the smaller one: each chunk also says how
// large its largest logit off the list is, and where that one's score equals the n-th best the
// last CTA looks the ties up in the logits themselves (the check is 2 of that call's 19.2 us).
//
// The sum takes __expf: 2 + 1.17 |x| units of 2^-23 off at x = logit - max, which a term's share
// exp(x) weighs, so that the sum is off by (2 + 1.17 ln vocab) 2^-23 at most, 2^-19, and its
// logarithm by 2e-6, a unit of a score of 20.
//
// That call is bound by the latency of a CTA's steps (load, maximum, exponentials, list,
// counter, then the ranking; 16 MB of logits would take 2.5 us): chunks of 8 and 32 KB took 3 and
// 19 us more.  So are small vocabularies.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

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
constexpr int kFewKeys = kThreads;  // ranked one against all

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
// NaN to -inf, +inf to the largest finite value, in the logits' own type.
__device__ __forceinline__ uint32_t clean(uint32_t x, float) {
  const float v = __uint_as_float(x);
  return __float_as_uint(fminf(fmaxf(v, -INFINITY), 3.402823466e38f));
}
__device__ __forceinline__ uint32_t clean(uint32_t x, __half) {
  asm("max.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xfc00fc00u));
  asm("min.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7bff7bffu));
  return x;
}
__device__ __forceinline__ uint32_t clean(uint32_t x, __nv_bfloat16) {
  asm("max.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0xff80ff80u));
  asm("min.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7f7f7f7fu));
  return x;
}

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half) {
  asm("max.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  asm("max.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
template <typename T>
__device__ __forceinline__ float half_of(uint32_t x, int e) {  // the low or high 16 bits
  if constexpr (std::is_same<T, __half>::value) {
    return __half2float(__ushort_as_half(uint16_t(x >> (16 * e))));
  } else {
    return __uint_as_float(e ? x & 0xffff0000u : x << 16);
  }
}

// The value of T next below x (a finite value of T); below the lowest one -inf.
template <typename T>
__device__ __forceinline__ float next_below(float x) {
  if constexpr (sizeof(T) == 4) {
    return key_value(value_key(x) - 1);
  } else if constexpr (std::is_same<T, __half>::value) {
    const uint32_t u = __half_as_ushort(__float2half_rn(x));
    const uint32_t y = (u & 0x7fffu) == 0 ? 0x8001u : u & 0x8000u ? u + 1 : u - 1;
    return __half2float(__ushort_as_half(uint16_t(y)));
  } else {
    const uint32_t u = __float_as_uint(x) >> 16;
    const uint32_t y = (u & 0x7fffu) == 0 ? 0x8001u : u & 0x8000u ? u + 1 : u - 1;
    return __uint_as_float(y << 16);
  }
}

// The n-th largest of the kWarps values of `top`, n <= kWarps.
template <typename K>
__device__ __forceinline__ K nth_of_warps(const K *top, int n) {
  const int lane = threadIdx.x & 31, me = lane % kWarps;
  const K x = top[me];
  int before = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) before += top[w] > x || (top[w] == x && w < me);
  const uint32_t is = __ballot_sync(0xffffffffu, before == n - 1);
  return __shfl_sync(0xffffffffu, x, __ffs(int(is)) - 1);
}

// The largest of the warp's keys (0 = none).
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

struct TopShared {
  unsigned long long warp_top[kThreads];  // kWarps lists of min(n, 32)
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
    if (lane == 0) sh->warp_top[warp * m + r] = top;
    if (k == top) k = 0;
  }
  if (threadIdx.x == 0) sh->bound = 0;
  __syncthreads();
  const int total = kWarps * m;
  if (int(threadIdx.x) < total) {  // the one that n - 1 others exceed
    const unsigned long long x = sh->warp_top[threadIdx.x];
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < total; ++i) larger += sh->warp_top[i] > x;
    if (x != 0 && larger == n - 1) sh->bound = x;
  }
  __syncthreads();
  return sh->bound;
}

// The n-th largest of the CTA's per-thread values, as its value_key (every thread has one,
// n <= kThreads; equal values count as often as they occur).
__device__ uint32_t nth_value(uint32_t mine, int n, TopShared *sh) {
  uint32_t *tops = reinterpret_cast<uint32_t *>(sh->warp_top);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = min(n, 32);
  uint32_t k = mine;
  for (int r = 0; r < m; ++r) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, k);
    if (lane == 0) tops[warp * m + r] = top;
    if (lane == __ffs(int(__ballot_sync(0xffffffffu, k == top))) - 1) k = 0;
  }
  __syncthreads();
  const int total = kWarps * m;
  if (int(threadIdx.x) < total) {  // fewer than n larger, n or more not smaller
    const uint32_t x = tops[threadIdx.x];
    int larger = 0, equal = 0;
#pragma unroll 8
    for (int i = 0; i < total; ++i) {
      larger += tops[i] > x;
      equal += tops[i] == x;
    }
    if (larger < n && larger + equal >= n) sh->bound = x;  // one value, of equal threads
  }
  __syncthreads();
  return uint32_t(sh->bound);
}

// 32-bit score of a logit x of a beam with (maximum, log of the sum) norm.
__device__ __forceinline__ float score_of(float x, float2 norm, float score_in) {
  const float s = x == -INFINITY ? -INFINITY : ((x - norm.x) - norm.y) + score_in;
  return s == s ? s : -INFINITY;
}

// best[above .. n): the lowest of request b's (beam, token) whose score's key is `want`, looked up
// in all its logits.  Rare: see the check in beam_best.
template <typename T>
__device__ __noinline__ void lowest_ties(const BeamArgs &a, int b, uint32_t want, int above,
                                         const float2 *norm, unsigned long long *best) {
  constexpr int kEach = 8;  // tokens of a thread at a time
  __shared__ int s_found[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int found = above;
  for (int k = 0; k < a.beams && found < a.n; ++k) {
    const int row = b * a.beams + k;
    const bool finished = a.finished && a.finished[row];
    const float score_in = a.scores_in[row];
    const float2 nrm = norm[k];
    if (!finished && value_key(score_of(nrm.x, nrm, score_in)) < want) continue;  // all lower
    const T *x = static_cast<const T *>(a.logits) + int64_t(row) * a.row_stride;
    for (int64_t base = 0; base < a.vocab && found < a.n; base += kThreads * kEach) {
      const int64_t v0 = base + tid * kEach;
      uint32_t hit = 0;
      for (int e = 0; e < kEach && v0 + e < a.vocab; ++e) {
        float s;
        if (finished) {
          s = uint32_t(v0 + e) == a.eos ? score_in : -INFINITY;
          s = s == s ? s : -INFINITY;
        } else {
          uint32_t bits;
          if constexpr (sizeof(T) == 4) {
            bits = reinterpret_cast<const uint32_t *>(x)[v0 + e];
          } else {
            bits = reinterpret_cast<const uint16_t *>(x)[v0 + e];
          }
          bits = clean(bits, T());
          float v;
          if constexpr (sizeof(T) == 4) {
            v = __uint_as_float(bits);
          } else {
            v = half_of<T>(bits, 0);
          }
          s = score_of(v, nrm, score_in);
        }
        hit |= value_key(s) == want ? 1u << e : 0u;
      }
      int sum = __popc(hit);
      const int mine = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      __syncthreads();  // the last round's reads
      if (lane == 31) s_found[warp] = sum;
      __syncthreads();
      int at = found + sum - mine, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        at += w < warp ? s_found[w] : 0;
        all += s_found[w];
      }
      for (; hit != 0 && at < a.n; hit &= hit - 1, ++at)
        best[at] = (static_cast<unsigned long long>(want) << 32) |
                   (0xffffffffu -
                    (uint32_t(k) * uint32_t(a.vocab) + uint32_t(v0) + __ffs(int(hit)) - 1));
      found += all;
    }
  }
  __syncthreads();
}

// One CTA's part of the choice: the last one of request b.
template <typename T>
__device__ void beam_best(const BeamArgs &a, int b, TopShared *sh, unsigned long long *list) {
  __shared__ float2 s_norm[kBeamMaxBeams];  // max, log of the sum
  __shared__ unsigned long long s_best[kMaxSelect];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the n-th listed and the largest unlisted logit of chunk i, for the check at the end; the
  // thread's first chunk's are loaded here, ahead of everything that waits
  const int64_t chunk0 = int64_t(b) * a.beams * a.chunks;
  auto nth_of = [&](int i) { return __ldcg(a.cand + (chunk0 + i) * a.n + a.n - 1); };
  auto rest_of = [&](int i) { return __ldcg(a.rest + chunk0 + i); };
  unsigned long long first_nth = 0;
  float first_rest = 0.f;
  if (tid < a.beams * a.chunks) {
    first_nth = nth_of(tid);
    first_rest = rest_of(tid);
  }
  for (int k = warp; k < a.beams; k += kWarps) {
    const int row = b * a.beams + k;
    if (a.finished && a.finished[row]) continue;
    const float2 *part = a.part + int64_t(row) * a.chunks;
    float M = -INFINITY, sum = 0.f;  // of this lane's chunks
    for (int i = lane; i < a.chunks; i += 32) {
      const float2 x = __ldcg(part + i);
      const float top = fmaxf(M, x.x);
      if (top != -INFINITY) sum = sum * __expf(M - top) + x.y * __expf(x.x - top);
      M = top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float M2 = __shfl_xor_sync(0xffffffffu, M, o);
      const float sum2 = __shfl_xor_sync(0xffffffffu, sum, o);
      const float top = fmaxf(M, M2);
      if (top != -INFINITY) sum = sum * __expf(M - top) + sum2 * __expf(M2 - top);
      M = top;
    }
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
      const unsigned long long c = __ldcg(a.cand + int64_t(row) * a.chunks * a.n + r);
      if (c == 0ull) return 0ull;
      token = key_index(c);
      const float x = key_value(uint32_t(c >> 32));
      score = score_of(x, s_norm[k], score);
    }
    if (!(score == score)) score = -INFINITY;
    return make_key(score, uint32_t(k) * uint32_t(a.vocab) + token);
  };
  // As for a chunk: the n-th largest of the warps' maxima bounds the n largest from below.
  int done = 0;
  bool ranked = false;
  if (a.n <= kWarps) {
    unsigned long long mine = 0, second = 0;
    for (int i = tid; i < total; i += kThreads) {
      const unsigned long long k = candidate(i);
      second = k > mine ? mine : k > second ? k : second;
      mine = k > mine ? k : mine;
    }
    const unsigned long long top = warp_max(mine);
    if (lane == 0) sh->warp_top[warp] = top;
    if (tid == 0) sh->count = 0;
    __syncthreads();
    unsigned long long bound = nth_of_warps(sh->warp_top, a.n);
    bound = bound == 0 ? 1 : bound;  // fewer warps have keys: all keys count
    auto put = [&](unsigned long long k) {
      const int at = atomicAdd(&sh->count, 1);
      if (at < kFewKeys) list[at] = k;
    };
    if (mine >= bound) put(mine);
    if (second >= bound) {
      for (int i = tid; i < total; i += kThreads) {
        const unsigned long long k = candidate(i);
        if (k >= bound && k != mine) put(k);
      }
    }
    __syncthreads();
    const int count = sh->count;
    ranked = count <= kFewKeys;
    if (ranked) {
      if (tid < count) {
        const unsigned long long x = list[tid];
        int larger = 0;
        for (int i = 0; i < count; ++i) larger += list[i] > x;
        if (larger < a.n) s_best[larger] = x;
      }
      done = min(count, a.n);
    }
    __syncthreads();
  }
  // Else in rounds: the n-th largest of the threads' maxima bounds what is left from below, and
  // the largest second key of a thread says down to where the maxima are final.
  unsigned long long cut = ~0ull;  // keys below it are left
  while (!ranked && done < a.n) {
    unsigned long long mine = 0, second = 0;
    for (int i = tid; i < total; i += kThreads) {
      const unsigned long long k = candidate(i);
      if (k >= cut) continue;
      if (k > mine) {
        second = mine;
        mine = k;
      } else if (k > second) {
        second = k;
      }
    }
    const int left = a.n - done;
    const unsigned long long bound = nth_maximum(mine, left, sh);
    if (mine < bound) second = 0;
    const unsigned long long top = warp_max(second);
    if (lane == 0) sh->warp_top[warp] = top;
    if (tid == 0) sh->count = 0;
    __syncthreads();
    unsigned long long floor_key = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) floor_key = max(floor_key, sh->warp_top[w]);
    const unsigned long long take = bound > floor_key ? bound : floor_key + 1;
    __syncthreads();
    // the final maxima, at most `left`, ranked among themselves
    if (mine != 0 && mine >= take) sh->warp_top[atomicAdd(&sh->count, 1)] = mine;
    __syncthreads();
    const int count = sh->count;
    if (count == 0) break;  // no candidate is left
    if (tid < count) {
      const unsigned long long x = sh->warp_top[tid];
      int larger = 0;
      for (int i = 0; i < count; ++i) larger += sh->warp_top[i] > x;
      if (larger < left) s_best[done + larger] = x;
    }
    __syncthreads();
    done += min(count, left);
    cut = s_best[done - 1];
  }
  // A chunk hides ties of the n-th best where its own n-th logit scores as much, and so does a
  // smaller one off the list; or, where an equal one is off the list (its index is higher than
  // those of its equals), a larger one on it does.
  const uint32_t last = uint32_t(s_best[a.n - 1] >> 32);
  bool hidden = false;
  for (int i = tid; i < a.beams * a.chunks; i += kThreads) {
    const int k = i / a.chunks, row = b * a.beams + k;
    if (a.finished && a.finished[row]) continue;
    const unsigned long long c = i == tid ? first_nth : nth_of(i);
    const float rest = i == tid ? first_rest : rest_of(i), score_in = a.scores_in[row];
    auto scores_last = [&](float x) {
      return value_key(score_of(x, s_norm[k], score_in)) == last;
    };
    if (c == 0ull) continue;  // all of the chunk is on its list
    const float nth = key_value(uint32_t(c >> 32));
    if (!scores_last(nth)) continue;
    if (rest < nth) {
      hidden |= scores_last(rest);
    } else {
      hidden |= nth != -INFINITY && scores_last(next_below<T>(nth));
      for (int j = a.n - 2; j >= 0; --j) {
        const float x = key_value(uint32_t(__ldcg(a.cand + (chunk0 + i) * a.n + j) >> 32));
        if (x == nth) continue;
        hidden |= scores_last(x);
        break;
      }
    }
  }
  if (__syncthreads_or(hidden)) {
    int above = 0;
    while (above < a.n && uint32_t(s_best[above] >> 32) != last) ++above;
    __syncthreads();
    lowest_ties<T>(a, b, last, above, s_norm, s_best);
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

// Grid (chunks, rows), a row being one beam of one request.
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) beam_select_kernel(const __grid_constant__ BeamArgs a) {
  constexpr int PER = 16 / sizeof(T);  // logits of a load
  constexpr int MOST = kVecs * PER;    // of a thread
  __shared__ TopShared sh;
  __shared__ unsigned long long s_list[kMaxSelect * MOST];
  __shared__ float s_red[kWarps], s_sum[kWarps];
  __shared__ uint32_t s_below[kWarps];
  __shared__ int s_last;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31, b = row / a.beams;
  const bool finished = a.finished && a.finished[row];  // beam_best knows its candidate
  if (!finished) {
    const T *base = static_cast<const T *>(a.logits) + int64_t(row) * a.row_stride;
    // 16-byte blocks counted from the one that holds the row's first logit
    const int lead = int((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
    const int64_t first = int64_t(chunk) * (kChunkBytes / int(sizeof(T))) - lead;
    uint32_t x[kVecs][4];
    const int64_t at0 = first + int64_t(tid) * PER;  // load i's first logit: + i * kThreads * PER
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int64_t at = at0 + int64_t(i) * kThreads * PER;
      if (at >= 0 && at + PER <= a.vocab) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(base + at));
        x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
      } else {  // the row's ends: logits outside it become NaN here, and -inf below
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          constexpr int PW = 4 / sizeof(T);
          x[i][w] = 0xffffffffu;
#pragma unroll
          for (int e = 0; e < PW; ++e) {
            const int64_t k = at + w * PW + e;
            if (k < 0 || k >= a.vocab) continue;
            if constexpr (PW == 1) {
              x[i][w] = reinterpret_cast<const uint32_t *>(base)[k];
            } else {
              const uint32_t bits = reinterpret_cast<const uint16_t *>(base)[k];
              x[i][w] = e ? (x[i][w] & 0xffffu) | (bits << 16) : (x[i][w] & 0xffff0000u) | bits;
            }
          }
        }
      }
    }
    auto value = [&](int i, int e) {  // logit e of load i
      if constexpr (sizeof(T) == 4) {
        return __uint_as_float(x[i][e]);
      } else {
        return half_of<T>(x[i][e / 2], e & 1);
      }
    };
    // the thread's maximum, the chunk's, and the chunk's sum
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
      for (int w = 0; w < 4; ++w) x[i][w] = clean(x[i][w], T());
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, value(i, e));
    } else {
      uint32_t two = x[0][0];
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) two = max2(two, x[i][w], T());
      mx = fmaxf(half_of<T>(two, 0), half_of<T>(two, 1));
    }
    float m = mx;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_red[warp] = m;
    if (tid == 0) sh.count = 0;
    // a bound of the n largest from below: n warps, or n threads, have a logit that reaches it
    float floor_value;
    if (a.n <= kWarps) {
      __syncthreads();
      floor_value = nth_of_warps(s_red, a.n);
    } else {
      floor_value = key_value(nth_value(value_key(mx), a.n, &sh));  // synchronises
    }
    m = s_red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_red[w]);
    // The logits that reach it: few, unless many are equal or fewer than n are finite.
    auto index = [&](int bit) {
      return at0 + int64_t(bit / PER) * kThreads * PER + bit % PER;
    };
    uint32_t reach = 0;  // bit i * PER + e
    if (mx >= floor_value) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e)
          reach |= value(i, e) >= floor_value ? 1u << (i * PER + e) : 0u;
    }
    auto each = [&](auto f) {  // f(key) of the thread's logits that reach the bound
      for (uint32_t left = reach; left != 0; left &= left - 1) {
        const int bit = __ffs(int(left)) - 1;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
          for (int e = 0; e < PER; ++e) v = bit == i * PER + e ? value(i, e) : v;
        const int64_t at = index(bit);
        if (at >= 0 && at < a.vocab) f(make_key(v, uint32_t(at)));
      }
    };
    if (floor_value == -INFINITY) {
      if (tid == 0) sh.count = kFewKeys + 1;  // logits outside the row would reach it as well
    } else if (reach != 0) {
      each([&](unsigned long long k) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kFewKeys) s_list[at] = k;
      });
    }
    float sum = 0.f;
    if (m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e) sum += __expf(value(i, e) - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      float total = 0.f;
      for (int w = 0; w < kWarps; ++w) total += s_sum[w];
      a.part[int64_t(row) * a.chunks + chunk] = make_float2(m, total);
    }
    int count = sh.count;
    const bool crowded = count > kFewKeys;
    if (crowded) {
      // the n-th largest of the threads' own largest keys is the bound: at most n threads, all
      // of whose logits fit, have keys that reach it
      __syncthreads();
      if (tid == 0) sh.count = 0;
      unsigned long long mine = 0ull;
      each([&](unsigned long long k) { mine = k > mine ? k : mine; });
      const unsigned long long bound = nth_maximum(mine, a.n, &sh);
      each([&](unsigned long long k) {
        if (k >= bound) s_list[atomicAdd(&sh.count, 1)] = k;
      });
      __syncthreads();
      count = sh.count;
    }
    unsigned long long *cand = a.cand + (int64_t(row) * a.chunks + chunk) * a.n;
    float *rest = a.rest + int64_t(row) * a.chunks + chunk;  // largest logit off the list, or more
    if (!crowded && count == a.n) {  // all that reach the bound are listed: the largest that does not
      uint32_t below = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (value(i, e) < floor_value) below = max(below, value_key(value(i, e)));
      below = __reduce_max_sync(0xffffffffu, below);
      if (lane == 0) s_below[warp] = below;
      __syncthreads();
      if (tid == 0) {
        for (int w = 0; w < kWarps; ++w) below = max(below, s_below[w]);
        *rest = key_value(below);
      }
    }
    for (int i = tid; i < max(count, a.n); i += kThreads) {
      if (i >= count) {
        cand[i] = 0ull;  // fewer than n logits in the chunk
        continue;
      }
      const unsigned long long k = s_list[i];
      int larger = 0;
      for (int j = 0; j < count; ++j) larger += s_list[j] > k;
      if (larger < a.n) cand[larger] = k;
      if (larger == (crowded ? a.n - 1 : a.n)) *rest = key_value(uint32_t(k >> 32));
    }
  }
  __syncthreads();
  if (tid == 0) {
    __threadfence();  // the CTA's candidates, which the barrier ordered before this
    s_last = atomicAdd(a.counters + b, 1) == a.beams * a.chunks - 1;
    if (s_last) a.counters[b] = 0;  // for the next call
    __threadfence();
  }
  __syncthreads();
  if (s_last) beam_best<T>(a, b, &sh, s_list);
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
  a.chunks = int((int64_t(a.vocab) + (aligned ? 0 : 16 / elem - 1) + per - 1) / per);
  const int rows = a.batch * a.beams;
  const size_t cand_bytes = size_t(rows) * a.chunks * a.n * 8;
  CallScratch scratch;
  cudaError_t e = scratch.acquire(stream, cand_bytes + size_t(rows) * a.chunks * 12);
  if (e != cudaSuccess) return e;
  a.cand = static_cast<unsigned long long *>(scratch.ptr);
  a.part = reinterpret_cast<float2 *>(static_cast<char *>(scratch.ptr) + cand_bytes);
  a.rest = reinterpret_cast<float *>(a.part + size_t(rows) * a.chunks);
  const dim3 grid(a.chunks, rows);
  a.counters = scratch.counters;
  e = launch_pdl(a.type == 0   ? beam_select_kernel<__half>
                 : a.type == 1 ? beam_select_kernel<__nv_bfloat16>
                               : beam_select_kernel<float>,
                 grid, dim3(kThreads), 0, stream, a);
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

// Attention over packed prompts on the sm_100a tensor cores (tcgen05).
//
// Sequence b has queries [q_start[b], q_start[b+1]) and keys [k_start[b], k_start[b+1]) in
// packed rows; query i of nq attends to the keys j <= i + nk - nq (all nk where not causal):
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(scale log2(e) q_i.k_j - m_i + kShift),
// with the running maximum m_i and sum of p in 32 bits over one pass of the keys.  A row that
// sees no key gives zeros.
//
// A CTA owns 128 NT consecutive rows of one sequence and kv head, row = query * G + head in
// the group of G, so that every K and V tile feeds the query heads of its group; groups need
// not divide the rows.  Keys go by in steps of 64.  Two score buffers a tile: QK(j+2) is
// issued as soon as P.V(j) has read the buffer, so that the softmax of a step never waits for
// the products of the step before it, and the tensor pipe not for the softmax.
//   warps 0 .. 4NT-1  softmax: thread = row.  S from TMEM, P back over it, output at the end
//   then one warp     MMA issue and TMEM
//   then one warp     K and V tiles by TMA: boxes of 64 values x 64 tokens, 128-byte swizzle,
//                     values past head_dim and tokens past the tensor zero-filled
// TMEM columns: score buffer (tile x, step parity) at 64 (2x + parity), P in its first 32;
// O of tile x at 128 NT + x DP.
//
// P is rounded to V's 16-bit type (both operands of a product have one type): an output is off
// by at most half a unit of that type times sum(p |v|) / sum(p) more than its own rounding.
// kShift places P in [2^-24, 2^15]: the maximum is raised when a step exceeds it by more than
// 2^8, and f16 then still holds weights of 2^-31 of the largest.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../launch.hpp"
#include "pdl.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr uint64_t kWaitNs = 1000000000ull;
constexpr int kKeys = 64;           // keys of a step
constexpr float kShift = 7.f;       // log2 of P where a score is the maximum
constexpr float kRaise = 8.f;       // log2 by which a step has to exceed the maximum to raise it
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kBlk = 128 * 128;         // 64 values of 128 rows
constexpr uint32_t kKvBlk = kKeys * 128;     // 64 values of a step's keys
constexpr size_t kMaxSmem = 227 * 1024;

template <int DP>
struct Shape {
  static constexpr int NT = DP <= 128 ? 2 : 1;  // tiles of 128 rows: O takes DP columns each
  static constexpr int kRows = 128 * NT;
  static constexpr int kBlocks = DP / 64;
  static constexpr uint32_t kTileQ = kBlocks * kBlk;
  static constexpr uint32_t kTileKv = kBlocks * kKvBlk;
  static constexpr uint32_t kFixed = NT * kTileQ + 1024 + 512;  // alignment, barriers
  static constexpr int kFit = int((kMaxSmem - kFixed) / (2 * kTileKv));
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static_assert(kStages >= 2, "two K and V tiles have to fit");
  static constexpr uint32_t kOffK = NT * kTileQ;
  static constexpr uint32_t kOffV = kOffK + kStages * kTileKv;
  static constexpr uint32_t kOffBar = kOffV + kStages * kTileKv;
  static constexpr size_t kSmem = kOffBar + 512 + 1024;
  static constexpr int kSoftmaxWarps = 4 * NT;
  static constexpr int kThreads = (kSoftmaxWarps + 2) * 32;
  static constexpr uint32_t kO = 128 * NT;  // TMEM column of O
  // barriers
  static constexpr int kQFull = 0, kKFull = 1, kKEmpty = kKFull + kStages,
                       kVFull = kKEmpty + kStages, kVEmpty = kVFull + kStages,
                       kVLast = kVEmpty + kStages, kSFull = kVLast + 1, kPFull = kSFull + 2 * NT,
                       kODone = kPFull + 2 * NT, kDrain = kODone + 2 * NT, kSlot = kDrain + 1;
  static_assert((kSlot + 1) * 8 <= 512, "barrier space");
  static_assert(kO + NT * DP <= kTmemCols, "TMEM");
};

struct Params {
  CUtensorMap tmk, tmv;
  PromptAttnArgs a;
  float scale_log2;
  uint32_t idesc_qk, idesc_pv;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return ptx::Mma<T>::pack(lo, hi);
}

// Bounded wait of a whole warp, which gives up as soon as another role has failed; every lane
// gets the same answer.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *fail) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  for (uint32_t n = 1;; ++n) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
    if ((n & 63) == 0) {
      const bool late = ptx::globaltimer_ns() - t0 > kWaitNs;
      if (late) *fail = 1;
      if (__any_sync(0xffffffffu, late || *fail)) return false;
    }
  }
}

struct Seq {
  int q0, nq, k0, nk;
};
// A sequence's rows, empty (and *bad set) where its starts are no ascending part of the rows.
__device__ __forceinline__ Seq load_seq(const PromptAttnArgs &a, int b, bool *bad) {
  const int q0 = a.q_start[b], q1 = a.q_start[b + 1], k0 = a.k_start[b], k1 = a.k_start[b + 1];
  Seq s = {q0, q1 - q0, k0, k1 - k0};
  if (q0 < 0 || q1 < q0 || q1 > a.num_q_tokens || k0 < 0 || k1 < k0 || k1 > a.num_k_tokens) {
    s.nq = 0;
    *bad = true;
  }
  return s;
}

struct Item {
  int b, h, t;  // sequence, kv head, row tile (from its start)
};
// Work item `i` of the list (sequence, kv head, row tiles from the last, which sees the most
// keys, to the first); false past the list's end.  One warp: lane l looks at sequence 32 n + l.
template <int ROWS>
__device__ __forceinline__ bool find_item(const PromptAttnArgs &a, int64_t i, Item *it) {
  const int lane = threadIdx.x & 31, G = a.group;
  bool bad = false, found = false;
  for (int b0 = 0; b0 < a.batch && !found; b0 += 32) {
    const int b = b0 + lane;
    int64_t nt = 0;
    if (b < a.batch) nt = (int64_t(load_seq(a, b, &bad).nq) * G + ROWS - 1) / ROWS;
    int64_t end = nt * a.kv_heads;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += o;
    }
    const uint32_t after = __ballot_sync(0xffffffffu, i < end);
    if (after) {
      const int l = __ffs(after) - 1;
      const int64_t rel = i - (__shfl_sync(0xffffffffu, end, l) -
                               __shfl_sync(0xffffffffu, nt, l) * a.kv_heads);
      const int64_t n = __shfl_sync(0xffffffffu, nt, l);
      it->b = b0 + l;
      it->h = int(rel / n);
      it->t = int(n - 1 - rel % n);
      found = true;
    } else {
      i -= __shfl_sync(0xffffffffu, end, 31);
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.diag, int32_t(kDiagBadLaunch));
  return found;
}

template <typename T, int DP>
__global__ void __launch_bounds__(Shape<DP>::kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ Params P) {
  using S = Shape<DP>;
  constexpr int NT = S::NT;
  const PromptAttnArgs &a = P.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t sb = (raw + 1023u) & ~1023u;
  unsigned char *smem = smem_raw + (sb - raw);
  __shared__ int s_fail;
  __shared__ Item s_item;
  __shared__ int s_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kMmaWarp = S::kSoftmaxWarps, kTmaWarp = kMmaWarp + 1;
  auto bar = [&](int i) { return sb + S::kOffBar + uint32_t(i) * 8; };

  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (warp == 0) {
    Item it = {0, 0, 0};
    const bool found = find_item<S::kRows>(a, int64_t(blockIdx.x), &it);
    if (lane == 0) {
      s_item = it;
      s_found = found;
      s_fail = 0;
    }
  } else if (warp == kTmaWarp) {
    if (lane == 0) {
      ptx::prefetch_tensormap(&P.tmk);
      ptx::prefetch_tensormap(&P.tmv);
      ptx::mbar_init(bar(S::kQFull), S::kSoftmaxWarps * 32);
      for (int i = 0; i < S::kStages; ++i) {
        ptx::mbar_init(bar(S::kKFull + i), 1);
        ptx::mbar_init(bar(S::kKEmpty + i), 1);
        ptx::mbar_init(bar(S::kVFull + i), 1);
        ptx::mbar_init(bar(S::kVEmpty + i), 1);
      }
      ptx::mbar_init(bar(S::kVLast), 1);
      ptx::mbar_init(bar(S::kDrain), 1);
      for (int i = 0; i < 2 * NT; ++i) {
        ptx::mbar_init(bar(S::kSFull + i), 1);
        ptx::mbar_init(bar(S::kPFull + i), 128);
        ptx::mbar_init(bar(S::kODone + i), 1);
      }
      ptx::fence_mbarrier_init();
    }
  } else if (warp == kMmaWarp) {
    tc::tmem_alloc(bar(S::kSlot), kTmemCols);
    tc::tmem_relinquish();
    tc::fence_before_sync();
  }
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::kOffBar + S::kSlot * 8);
  volatile int *fail = &s_fail;

  if (s_found) {
    const Item it = s_item;
    bool bad = false;
    const Seq s = load_seq(a, it.b, &bad);
    const int G = a.group;
    const int64_t rows = int64_t(s.nq) * G, row0 = int64_t(it.t) * S::kRows;
    const int past = s.nk - s.nq;  // keys before the first query
    // keys that tile x's last row sees, in steps
    auto steps = [&](int x) {
      const int64_t last = min(row0 + 128 * (x + 1), rows) - 1;
      if (last < row0 + 128 * x) return 0;
      const int64_t n = a.causal ? min(int64_t(s.nk), last / G + past + 1) : int64_t(s.nk);
      return n <= 0 ? 0 : int((n + kKeys - 1) / kKeys);
    };
    int n_steps[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) n_steps[x] = steps(x);
    int n_max = n_steps[0];
    if constexpr (NT == 2) n_max = max(n_steps[0], n_steps[1]);

    if (warp == kTmaWarp) {
      int issued_k = 0, issued_v = 0;  // steps whose copies have begun
      for (int j = 0; j < n_max; ++j) {
        const int st = j % S::kStages;
        const uint32_t ph = uint32_t((j / S::kStages - 1) & 1);
        const int key = s.k0 + j * kKeys;
        if (j >= S::kStages && !wait(bar(S::kKEmpty + st), ph, fail)) break;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(bar(S::kKFull + st), S::kTileKv);
#pragma unroll
          for (int c = 0; c < S::kBlocks; ++c)
            ptx::tma_load_3d(sb + S::kOffK + st * S::kTileKv + c * kKvBlk, &P.tmk, c * 64, it.h,
                             key, bar(S::kKFull + st));
        }
        __syncwarp();
        issued_k = j + 1;
        if (j >= S::kStages && !wait(bar(S::kVEmpty + st), ph, fail)) break;
        // Rows past the sequence are another's: P is 0 there, and V has to be finite.
        const int live = min(kKeys, s.nk - j * kKeys);
        const uint32_t full = bar(live < kKeys ? S::kVLast : S::kVFull + st);
        const uint32_t dst = sb + S::kOffV + st * S::kTileKv;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(full, S::kTileKv);
#pragma unroll
          for (int c = 0; c < S::kBlocks; ++c)
            ptx::tma_load_3d(dst + c * kKvBlk, &P.tmv, c * 64, it.h, key, full);
        }
        __syncwarp();
        if (live < kKeys) {  // the sequence's last step, once
          if (!wait(full, 0, fail)) break;
          const int words = (kKeys - live) * 8;  // 16-byte words of a block's rows
          for (int i = lane; i < words * S::kBlocks; i += 32) {
            const uint32_t at = dst + (i / words) * kKvBlk + live * 128 + (i % words) * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0) : "memory");
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(S::kVFull + st));
          __syncwarp();
        } else {
          issued_v = j + 1;
        }
      }
      if (*fail) {  // no copy may land after the CTA has gone
        for (int j = max(0, issued_k - S::kStages); j < issued_k; ++j)
          ptx::mbar_wait_bounded(bar(S::kKFull + j % S::kStages),
                                 uint32_t((j / S::kStages) & 1), kWaitNs);
        for (int j = max(0, issued_v - S::kStages); j < issued_v; ++j)
          ptx::mbar_wait_bounded(bar(S::kVFull + j % S::kStages),
                                 uint32_t((j / S::kStages) & 1), kWaitNs);
      }
    } else if (warp == kMmaWarp) {
      auto issue_qk = [&](int x, int j) {
        if (lane == 0) {
          const uint32_t qa = sb + uint32_t(x) * S::kTileQ;
          const uint32_t ka = sb + S::kOffK + (j % S::kStages) * S::kTileKv;
          const uint32_t tS = tmem + uint32_t(2 * x + (j & 1)) * kKeys;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            tc::mma_ss(tS, tc::sw128_desc(qa + (k >> 2) * kBlk + (k & 3) * 32, 16, 1024),
                       tc::sw128_desc(ka + (k >> 2) * kKvBlk + (k & 3) * 32, 16, 1024),
                       P.idesc_qk, k > 0);
          tc::commit(bar(S::kSFull + 2 * x + (j & 1)));
        }
        __syncwarp();
      };
      auto issue_pv = [&](int x, int j) {
        if (lane == 0) {
          const uint32_t va = sb + S::kOffV + (j % S::kStages) * S::kTileKv;
          const uint32_t tP = tmem + uint32_t(2 * x + (j & 1)) * kKeys;
          const uint32_t tO = tmem + S::kO + uint32_t(x) * DP;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            tc::mma_ts(tO, tP + k * 8, tc::sw128_desc(va + k * 2048, kKvBlk, 1024), P.idesc_pv,
                       j > 0 || k > 0);
          tc::commit(bar(S::kODone + 2 * x + (j & 1)));
        }
        __syncwarp();
      };
      auto release = [&](int b) {
        if (lane == 0) tc::commit(bar(b));
        __syncwarp();
      };
      bool ok = n_max == 0 || wait(bar(S::kQFull), 0, fail);
      for (int j = 0; ok && j < min(2, n_max); ++j) {
        ok = wait(bar(S::kKFull + j % S::kStages), 0, fail);
        if (!ok) break;
#pragma unroll
        for (int x = 0; x < NT; ++x)
          if (j < n_steps[x]) issue_qk(x, j);
        release(S::kKEmpty + j % S::kStages);
      }
      for (int j = 0; ok && j < n_max; ++j) {
        const int st = j % S::kStages, jn = j + 2, sn = jn % S::kStages;
        ok = wait(bar(S::kVFull + st), uint32_t((j / S::kStages) & 1), fail);
        if (ok && jn < n_max)
          ok = wait(bar(S::kKFull + sn), uint32_t((jn / S::kStages) & 1), fail);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          if (!ok || j >= n_steps[x]) continue;
          ok = wait(bar(S::kPFull + 2 * x + (j & 1)), uint32_t((j >> 1) & 1), fail);
          if (!ok) continue;
          issue_pv(x, j);
          if (jn < n_steps[x]) issue_qk(x, jn);
        }
        if (!ok) break;
        release(S::kVEmpty + st);
        if (jn < n_max) release(S::kKEmpty + sn);
      }
      if (!ok) {  // no product may run on after the CTA has gone
        release(S::kDrain);
        ptx::mbar_wait_bounded(bar(S::kDrain), 0, kWaitNs);
      }
    } else {
      // Q: 16 bytes a lane; rows and values past the end are zeros
      constexpr int kChunks = DP / 8;
      for (int i = tid; i < S::kRows * kChunks; i += S::kSoftmaxWarps * 32) {
        const int r = i / kChunks, c = i % kChunks;
        const int64_t row = row0 + r;
        const bool in = row < rows && c * 8 < a.head_dim;
        const int64_t tok = in ? row / G : 0;
        const int head = in ? it.h * G + int(row % G) : 0;
        const uint16_t *src = static_cast<const uint16_t *>(a.q) +
                              (in ? (s.q0 + tok) * a.q_stride_token +
                                        int64_t(head) * a.q_stride_head + c * 8
                                  : 0);
        const uint32_t dst = sb + uint32_t(r >> 7) * S::kTileQ + uint32_t(c >> 3) * kBlk +
                             uint32_t(r & 127) * 128 + uint32_t(((c & 7) ^ (r & 7)) * 16);
        ptx::cp_async16(dst, src, in ? 16u : 0u);
      }
      ptx::cp_async_commit();
      ptx::cp_async_wait<0>();
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(S::kQFull));

      const int x = warp >> 2, q4 = warp & 3;
      const int n = NT == 2 && x == 1 ? n_steps[NT - 1] : n_steps[0];
      const int64_t row = row0 + 128 * x + q4 * 32 + lane;
      const bool row_ok = row < rows;
      // last key that the row sees; rows past the end go as far as the last one
      const int tok = int(min(row, rows - 1) / G);
      const int lim = a.causal ? tok + past : s.nk - 1;
      const int lim0 = __shfl_sync(0xffffffffu, lim, 0);
      const uint32_t lanes = uint32_t(q4 * 32) << 16;
      const uint32_t tO = tmem + S::kO + uint32_t(x) * DP + lanes;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const uint32_t tS = tmem + uint32_t(2 * x + (j & 1)) * kKeys + lanes;
        if (!wait(bar(S::kSFull + 2 * x + (j & 1)), uint32_t((j >> 1) & 1), fail)) {
          ok = false;
          break;
        }
        // S(j) came after P.V(j-2), whose barrier is thus the one before P.V(j)'s
        if (j >= 2 &&
            !wait(bar(S::kODone + 2 * x + (j & 1)), uint32_t(((j - 2) >> 1) & 1), fail)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        float v[kKeys];
        tc::ld32(tS, v);
        tc::ld32(tS + 32, v + 32);
        tc::wait_ld();
        const int k0 = j * kKeys;
        if (k0 + kKeys - 1 > lim0) {
#pragma unroll
          for (int c = 0; c < kKeys; ++c) v[c] = k0 + c > lim ? -INFINITY : v[c];
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kKeys; c += 8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = ptx::max3(mx[i], v[c + 2 * i], v[c + 2 * i + 1]);
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * P.scale_log2;
        const bool raise = top > m + kRaise;  // the first step's m is -inf
        float f = 1.f;
        if (raise) {
          f = ptx::fast_exp2(m - top);  // 0 before the first key
          m = top;
          l *= f;
        }
        if (j > 0 && __any_sync(0xffffffffu, raise)) {
          // P.V(j-1) has to have added to O; P.V(j) has not begun
          if (!wait(bar(S::kODone + 2 * x + ((j - 1) & 1)), uint32_t(((j - 1) >> 1) & 1), fail)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            float o[32];
            tc::ld32(tO + c * 32, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tc::st32(tO + c * 32, o);
          }
          tc::wait_st();
        }
        const float sub = m == -INFINITY ? 0.f : m - kShift;  // nothing seen yet: P is 0
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w[kKeys / 2];
#pragma unroll
        for (int c = 0; c < kKeys; c += 2) {
          const float e0 = ptx::fast_exp2(fmaf(v[c], P.scale_log2, -sub));
          const float e1 = ptx::fast_exp2(fmaf(v[c + 1], P.scale_log2, -sub));
          sum[c & 2] += e0;
          sum[(c & 2) + 1] += e1;
          w[c / 2] = pack2<T>(e0, e1);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tc::st32u(tS, w);
        tc::wait_st();
        tc::fence_before_sync();
        ptx::mbar_arrive(bar(S::kPFull + 2 * x + (j & 1)));
      }
      if (ok && n > 0)
        ok = wait(bar(S::kODone + 2 * x + ((n - 1) & 1)), uint32_t(((n - 1) >> 1) & 1), fail);
      if (ok) {
        tc::fence_after_sync();
        const float inv = l > 0.f ? 1.f / l : l;  // l is 0, or a NaN that stays one
        const bool none = n == 0 || l == 0.f;
        uint16_t *dst = static_cast<uint16_t *>(a.out) +
                        (row_ok ? (s.q0 + row / G) * a.out_stride_token +
                                      (int64_t(it.h) * G + row % G) * a.out_stride_head
                                : 0);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          if (n > 0) {
            tc::ld32(tO + c * 32, o);
            tc::wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = none ? 0.f : o[e] * inv;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (!row_ok || c * 32 + q * 8 >= a.head_dim) continue;
            uint4 u;
            u.x = pack2<T>(o[q * 8], o[q * 8 + 1]);
            u.y = pack2<T>(o[q * 8 + 2], o[q * 8 + 3]);
            u.z = pack2<T>(o[q * 8 + 4], o[q * 8 + 5]);
            u.w = pack2<T>(o[q * 8 + 6], o[q * 8 + 7]);
            *reinterpret_cast<uint4 *>(dst + c * 32 + q * 8) = u;
          }
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (s_fail && tid == 0) atomicOr(a.diag, int32_t(kDiagWaitTimeout));
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int DP>
cudaError_t launch(const PromptAttnArgs &a, cudaStream_t stream) {
  using S = Shape<DP>;
  Params p;
  std::memset(static_cast<void *>(&p), 0, sizeof(p));
  std::memcpy(&p.tmk, a.k_map, sizeof(CUtensorMap));
  std::memcpy(&p.tmv, a.v_map, sizeof(CUtensorMap));
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  p.idesc_qk = tc::idesc_f16(bf16, 128, kKeys, false, false);
  p.idesc_pv = tc::idesc_f16(bf16, 128, DP, false, true);
  auto fn = prompt_attn_kernel<T, DP>;
  cudaError_t e =
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem));
  if (e != cudaSuccess) return e;
  // every sequence has at most one partly filled tile a kv head
  const int64_t tiles = int64_t(a.num_q_tokens) * a.group / S::kRows + a.batch;
  return launch_pdl(fn, dim3(uint32_t(tiles * a.kv_heads)), dim3(S::kThreads), S::kSmem, stream,
                    p);
}

}  // namespace

int prompt_attn_box_rows() { return kKeys; }

cudaError_t prompt_attn(const PromptAttnArgs &a, cudaStream_t stream) {
  const bool bf16 = a.dtype == Dtype::BF16;
#define KCMM_PROMPT(DP) \
  return bf16 ? launch<__nv_bfloat16, DP>(a, stream) : launch<__half, DP>(a, stream)
  if (a.head_dim <= 64) KCMM_PROMPT(64);
  if (a.head_dim <= 128) KCMM_PROMPT(128);
  if (a.head_dim <= 192) KCMM_PROMPT(192);
  KCMM_PROMPT(256);
#undef KCMM_PROMPT
}

}  // namespace dev
}  // namespace kcmm

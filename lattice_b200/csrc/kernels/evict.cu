// Eviction of cached tokens by accumulated attention weight.
//
// For every sequence b and kv head g with n > budget cached tokens, slot i of position
//   pos(i) = positions_in[i] for i < kept_lens[b], else i + next_positions[b] - n,
// stays if pos(i) < sinks or pos(i) >= next_positions[b] - recent; the rest of the budget
// goes to the other slots of largest weight (ties: the lowest slot; NaN counts as -inf).
// The kept slots past the budget move, in order, into the freed ones below it, so a source
// (>= budget) is never a destination (< budget): the moves need no order among themselves,
// and only the rows that have to move are touched.
//
// The selection narrows a range of 32-bit keys by histograms of 2048 equal bins, as wide as
// the range asks for: accumulated weights spread over a few octaves, and bins fixed to their
// leading bits would put half of them into 4 (measured: 72 us a call for 16 rows of 16,700
// tokens, the atomics on one bin serialised, against 25).  The last few keys are ranked one
// against all: another histogram or two took 2 to 5 us more.  A cluster of CTAs shares a long
// row.  It is bound by the latency of its passes, over keys in shared memory where they fit
// (128 rows of 3700 tokens: 11 us).  The moves are a copy of scattered rows:
// 105,000 of 2 x 256 bytes take 18.5 us, 5.8 TB/s read and written, half of it in L2 (58 MB of
// HBM traffic, 2.8 TB/s); the loads' latency bounds them, with 30 % of the warps that would fit.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../launch.hpp"
#include "kv4_layout.cuh"
#include "pdl.cuh"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace kcmm {
namespace dev {
namespace {

constexpr int kFewKeys = 256;  // ranked one against all instead of by another histogram
constexpr int kBins = 2048;
constexpr int kCopies = 4;  // slots of a thread in flight
constexpr int kMaxCluster = 8;
constexpr int kSliceTokens = 4096;
constexpr int kKeyCapacity = 49152;  // keys in shared memory: 192 KB

// One row's moves: count, then [most_moves] each of destination and source slots; its sequence's
// new length, which the move kernel passes on: here other CTAs still read the arrays that the
// caller may have given for it (kept_lens, seq_lens).
struct RowMoves {
  int32_t *count, *new_len, *dst, *src;
};
__device__ __forceinline__ RowMoves row_moves(const EvictArgs &a, int row) {
  const int64_t rows = int64_t(a.batch) * a.kv_heads, at = int64_t(row) * a.most_moves;
  RowMoves r;
  r.count = a.scratch + row;
  r.new_len = a.scratch + rows + row / a.kv_heads;
  r.dst = a.scratch + rows + a.batch + at;
  r.src = r.dst + rows * a.most_moves;
  return r;
}

// Larger key = kept first.  Finite weights keep their order, -0 and +0 are one value.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kHeldKey = 0xffffffffu;  // above every weight's

struct Counts {
  int gt, eq;        // keys above and at the threshold
  int gt_lo, eq_lo;  // those among the slots below the budget
};

// CLUSTER: several CTAs share a row; a single CTA's barriers cost a third of a cluster's.
template <int kSelectThreads, bool CLUSTER>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
  constexpr int kSelectWarps = kSelectThreads / 32;
  static_assert(kSelectWarps <= 32 && kBins % (2 * kSelectThreads) == 0, "a warp sums the warps");
  constexpr int kPairs = kBins / 2 / kSelectThreads;  // bin pairs of a thread
  __shared__ __align__(8) int s_hist[kBins];
  __shared__ int4 s_range[kSelectWarps], s_total;
  extern __shared__ uint32_t s_keys[];
  __shared__ Counts s_warp[kSelectWarps];
  __shared__ Counts s_cta;
  __shared__ int s_scan[kSelectWarps];
  __shared__ __align__(16) int4 s_bin;
  __shared__ int s_above, s_few;
  __shared__ __align__(16) uint32_t s_list[kFewKeys + 4], s_all[CLUSTER ? kFewKeys + 4 : 4];
  __shared__ uint32_t s_threshold;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int kMostRanks = CLUSTER ? kMaxCluster : 1;
  const int C = CLUSTER ? int(cluster.num_blocks()) : 1;
  const int rank = CLUSTER ? int(cluster.block_rank()) : 0;
  auto sync = [&] {
    if constexpr (CLUSTER) {
      cluster.sync();
    } else {
      __syncthreads();
    }
  };
  auto of_rank = [&](auto *x, int r) {  // CTA r's copy of a shared variable
    if constexpr (CLUSTER) {
      return cluster.map_shared_rank(x, r);
    } else {
      return x;
    }
  };
  const int b = blockIdx.z, g = blockIdx.y, row = b * a.kv_heads + g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = max(a.seq_lens[b], 0);
  const int kept_len = min(max(a.kept_lens[b], 0), n), next = a.next_positions[b];
  const float *w_in = a.w_in + int64_t(row) * a.w_stride;
  float *w_out = a.w_out + int64_t(row) * a.w_stride;
  const int32_t *p_in = a.p_in + int64_t(row) * a.w_stride;
  int32_t *p_out = a.p_out + int64_t(row) * a.w_stride;
  const RowMoves mv = row_moves(a, row);
  auto pos_of = [&](int i) { return i < kept_len ? p_in[i] : i + next - n; };

  if (n > a.max_tokens || n > a.w_stride) {  // more tokens than the arguments hold
    if (rank == 0 && tid == 0) {
      mv.count[0] = 0;
      if (g == 0) *mv.new_len = n;
      atomicOr(a.diag, int32_t(kDiagBadLaunch));
    }
    return;
  }
  if (rank == 0 && tid == 0) {
    mv.count[0] = 0;
    if (g == 0) *mv.new_len = min(n, a.budget);
  }
  if (n <= a.budget) {  // uniform over the cluster
    for (int i = rank * kSelectThreads + tid; i < n; i += C * kSelectThreads) {
      const float w = w_in[i];
      const int p = pos_of(i);
      w_out[i] = w;
      p_out[i] = p;
    }
    return;
  }
  const int slice = (n + C - 1) / C, begin = min(rank * slice, n), end = min(begin + slice, n);
  auto make_key = [&](int i) {
    const int p = pos_of(i);
    return p < a.sinks || p >= next - a.recent ? kHeldKey : weight_key(w_in[i]);
  };

  // ---- keys, their range, and how many slots are held -----------------------------------------
  // The keys of this CTA's slice stay in shared memory where it holds them.
  const bool staged = end - begin <= a.key_capacity;
  uint32_t kmin = 0xffffffffu, kmax = 0;
  int held = 0;
#pragma unroll 4
  for (int i = begin + tid; i < end; i += kSelectThreads) {
    const uint32_t k = make_key(i);
    if (staged) s_keys[i - begin] = k;
    held += k == kHeldKey;
    if (k != kHeldKey) {
      kmin = min(kmin, k);
      kmax = max(kmax, k);
    }
  }
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  held = __reduce_add_sync(0xffffffffu, held);
  if (lane == 0) s_range[warp] = make_int4(int(kmin), int(kmax), held, 0);
  for (int i = tid; i < kBins; i += kSelectThreads) s_hist[i] = 0;
  __syncthreads();
  if (warp == 0) {
    const int4 r = lane < kSelectWarps ? s_range[lane] : make_int4(-1, 0, 0, 0);
    kmin = __reduce_min_sync(0xffffffffu, uint32_t(r.x));
    kmax = __reduce_max_sync(0xffffffffu, uint32_t(r.y));
    held = __reduce_add_sync(0xffffffffu, r.z);
    if (lane == 0) s_total = make_int4(int(kmin), int(kmax), held, 0);
  }
  sync();
  kmin = 0xffffffffu;
  kmax = 0;
  held = 0;
#pragma unroll
  for (int r = 0; r < kMostRanks; ++r) {
    if (r >= C) continue;
    const int4 t = *of_rank(&s_total, r);
    kmin = min(kmin, uint32_t(t.x));
    kmax = max(kmax, uint32_t(t.y));
    held += t.z;
  }
  auto key_of = [&](int i) { return staged ? s_keys[i - begin] : make_key(i); };

  // ---- threshold: the budget-th largest key, and how many equal to it stay -------------
  uint32_t threshold = kHeldKey;
  int want = a.budget;  // keys at or below kmax to take, when the held ones are taken
  if (held < a.budget) {
    want -= held;
    uint32_t lo = kmin, hi = kmax;  // the wanted key lies in [lo, hi]; keys above hi are taken
#pragma unroll 1
    while (lo != hi) {
      const int bits = 32 - __clz(int(hi - lo));  // of the range
      const int shift = max(bits - 11, 0);
#pragma unroll 4
      for (int base = begin; base < end; base += kSelectThreads) {
        const int i = base + tid;
        const uint32_t k = i < end ? key_of(i) : 0;
        const bool in = i < end && k >= lo && k <= hi;
        const int bin = in ? int((k - lo) >> shift) : -1;
        // lanes that share the first live lane's bin count as one (equal weights would
        // otherwise serialise)
        const uint32_t live = __ballot_sync(0xffffffffu, in);
        if (live == 0) continue;
        const int first = __shfl_sync(0xffffffffu, bin, __ffs(int(live)) - 1);
        const uint32_t same = __ballot_sync(0xffffffffu, bin == first);
        if (bin == first) {
          if (lane == __ffs(int(same)) - 1) atomicAdd(&s_hist[bin], __popc(same));
        } else if (in) {
          atomicAdd(&s_hist[bin], 1);
        }
      }
      sync();
      // Bins from the top: thread t has the 2 kPairs bins below kBins - 2 kPairs t.  One CTA
      // adds up all the CTAs' and tells the others: each reading them all took 2 us longer.
      if (rank == 0) {
        const int top = kBins - 2 * kPairs * tid;
        int2 c[kPairs];  // c[i]: bins top - 2i - 2 (x) and top - 2i - 1 (y)
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          c[i] = make_int2(0, 0);
          int2 h[kMostRanks];  // all in flight together
#pragma unroll
          for (int r = 0; r < kMostRanks; ++r)
            h[r] = r < C ? *reinterpret_cast<const int2 *>(of_rank(s_hist, r) + top - 2 * i - 2)
                         : make_int2(0, 0);
#pragma unroll
          for (int r = 0; r < kMostRanks; ++r) {
            c[i].x += h[r].x;
            c[i].y += h[r].y;
          }
          mine += c[i].x + c[i].y;
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += x;
        }
        if (lane == 31) s_scan[warp] = sum;
        __syncthreads();
        int above = lane < warp ? s_scan[lane] : 0;
        above = __reduce_add_sync(0xffffffffu, above) + sum - mine;  // keys above these bins
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n_bin = e == 0 ? c[i].y : c[i].x;
            if (above < want && above + n_bin >= want) {
              const int4 x = make_int4(top - 2 * i - 1 - e, above, n_bin, 0);
#pragma unroll
              for (int r = 0; r < kMostRanks; ++r)
                if (r < C) *of_rank(&s_bin, r) = x;
            }
            above += n_bin;
          }
        }
      }
      if (tid == 0) s_few = 0;
      sync();
      for (int i = tid; i < kBins; i += kSelectThreads) s_hist[i] = 0;
      const int4 wanted = s_bin;  // bin, keys above it, keys in it
      __syncthreads();
      want -= wanted.y;
      const uint32_t base = lo + (uint32_t(wanted.x) << shift);
      hi = min(hi, base + ((1u << shift) - 1));
      lo = base;
      if (lo != hi && wanted.z <= kFewKeys) {
        // few keys are left: each is ranked against all
        for (int i = begin + tid; i < end; i += kSelectThreads) {
          const uint32_t k = key_of(i);
          if (k >= lo && k <= hi) s_list[atomicAdd(&s_few, 1)] = k;
        }
        sync();
        // every CTA's keys, then zeros, which are below any key, up to a multiple of 4
        const uint32_t *list = s_list;
        int few = s_few;
        if constexpr (CLUSTER) {
          few = 0;
#pragma unroll
          for (int r = 0; r < kMostRanks; ++r) {
            if (r >= C) continue;
            const int some = *of_rank(&s_few, r);
            if (tid < some) s_all[few + tid] = of_rank(s_list, r)[tid];
            few += some;
          }
          list = s_all;
          if (tid < 3) s_all[few + tid] = 0;
        } else {
          if (tid < 3) s_list[few + tid] = 0;
        }
        __syncthreads();
        if (tid < few) {
          const uint32_t k = list[tid];
          int larger = 0, equal = 0;
          for (int i = 0; i < few; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(list + i);
            larger += (x.x > k) + (x.y > k) + (x.z > k) + (x.w > k);
            equal += (x.x == k) + (x.y == k) + (x.z == k) + (x.w == k);
          }
          if (larger < want && larger + equal >= want) {  // equal keys write the same
            s_threshold = k;
            s_above = larger;
          }
        }
        __syncthreads();
        want -= s_above;
        lo = hi = s_threshold;
      }
    }
    threshold = lo;
  }
  // `want` keys equal to the threshold stay: the lowest slots

  // ---- counts per warp segment, then over the CTA and the cluster ------------------------
  const int seg = (end - begin + kSelectWarps - 1) / kSelectWarps;
  const int s0 = min(begin + warp * seg, end), s1 = min(s0 + seg, end);
  Counts c = {0, 0, 0, 0};
  for (int i = s0 + lane; i < s1; i += 32) {
    const uint32_t k = key_of(i);
    const bool lo = i < a.budget;
    c.gt += k > threshold;
    c.eq += k == threshold;
    c.gt_lo += k > threshold && lo;
    c.eq_lo += k == threshold && lo;
  }
  c.gt = __reduce_add_sync(0xffffffffu, c.gt);
  c.eq = __reduce_add_sync(0xffffffffu, c.eq);
  c.gt_lo = __reduce_add_sync(0xffffffffu, c.gt_lo);
  c.eq_lo = __reduce_add_sync(0xffffffffu, c.eq_lo);
  if (lane == 0) s_warp[warp] = c;
  __syncthreads();
  if (warp == 0) {
    const Counts w = lane < kSelectWarps ? s_warp[lane] : Counts{0, 0, 0, 0};
    const Counts t = {__reduce_add_sync(0xffffffffu, w.gt), __reduce_add_sync(0xffffffffu, w.eq),
                      __reduce_add_sync(0xffffffffu, w.gt_lo),
                      __reduce_add_sync(0xffffffffu, w.eq_lo)};
    if (lane == 0) s_cta = t;
  }
  sync();
  int gt = 0, eq = 0, gt_lo = 0, eq_lo = 0;  // gt, eq: before this warp's segment
#pragma unroll
  for (int r = 0; r < kMostRanks; ++r) {
    if (r >= C) continue;
    const Counts t = *of_rank(&s_cta, r);
    if (r < rank) {
      gt += t.gt;
      eq += t.eq;
    }
    gt_lo += t.gt_lo;
    eq_lo += t.eq_lo;
  }
  gt += __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane].gt : 0);
  eq += __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane].eq : 0);
  const int kept_lo = gt_lo + min(eq_lo, want);  // slots below the budget that stay
  const int moves = min(a.budget - kept_lo, a.most_moves);  // at most budget, and n - budget

  // ---- the lists of freed slots and of moving ones, by rank ------------------------------
  const uint32_t below = (1u << lane) - 1;
  for (int base = s0; base < s1; base += 32) {
    const int i = base + lane;
    const bool in = i < s1;
    const uint32_t k = in ? key_of(i) : 0;
    const uint32_t gts = __ballot_sync(0xffffffffu, in && k > threshold);
    const uint32_t eqs = __ballot_sync(0xffffffffu, in && k == threshold);
    const int eq_before = eq + __popc(eqs & below);
    const int kept_before = gt + __popc(gts & below) + min(eq_before, want);
    const bool keep = in && (k > threshold || (k == threshold && eq_before < want));
    const int at = i < a.budget ? i - kept_before : kept_before - kept_lo;
    if (in && keep == (i >= a.budget) && uint32_t(at) < uint32_t(a.most_moves))
      (keep ? mv.src : mv.dst)[at] = i;
    gt += __popc(gts);
    eq += __popc(eqs);
  }
  if (rank == 0 && tid == 0) mv.count[0] = moves;

  // ---- weights and positions of the slots below the budget, freed ones included ------------
  // (inputs and outputs may be the same memory: loads of several slots before their stores)
  const int low_end = min(end, a.budget);
  for (int base = begin + tid; base < low_end; base += kCopies * kSelectThreads) {
    float w[kCopies];
    int p[kCopies];
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      const int i = base + k * kSelectThreads;
      w[k] = i < low_end ? w_in[i] : 0.f;
      p[k] = i < low_end ? pos_of(i) : 0;
    }
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      const int i = base + k * kSelectThreads;
      if (i < low_end) {
        w_out[i] = w[k];
        p_out[i] = p[k];
      }
    }
  }
  sync();  // the lists are complete, and the freed slots may be filled
  for (int j = rank * kSelectThreads + tid; j < moves; j += C * kSelectThreads) {
    const int d = __ldcg(mv.dst + j), i = __ldcg(mv.src + j);
    const float w = w_in[i];
    const int p = pos_of(i);
    w_out[d] = w;
    p_out[d] = p;
  }
  sync();  // the moved slots' weights have been read; the slots past the budget weigh 0
  for (int i = max(begin, a.budget) + tid; i < end; i += kSelectThreads) w_out[i] = 0.f;
}

constexpr int kMoveThreads = 256;

// First byte of head g's row (16-bit cache) or chunk (4-bit cache) of slot i, and the
// token's place in its chunk; -1 where the slot, the table or the offset is bad.
__device__ __forceinline__ int64_t slot_bytes(const EvictArgs &a, int b, int g, int i, int *t) {
  if (uint32_t(i) >= uint32_t(a.max_tokens)) return -1;
  const int page = i / a.block_size, in = i - page * a.block_size;
  const int blk = a.tables[int64_t(b) * a.bt_stride + page];
  if (blk < 0) return -1;
  const uint64_t off = a.offsets[blk] * 2;
  const int64_t row = a.kv4 ? 9 * a.head_dim / 16 : 2 * a.head_dim;
  if ((off & 15) || off + uint64_t(a.block_size) * a.kv_heads * row > a.region_bytes) return -1;
  *t = in % kKv4Unit;
  if (a.kv4)
    return int64_t(off) + (int64_t(g) * (a.block_size / kKv4Unit) + in / kKv4Unit) * 9 * a.head_dim;
  return int64_t(off) + (int64_t(in) * a.kv_heads + g) * row;
}

// Up to 32 moves a warp: each lane resolves one (slot -> page -> offset, three loads deep), then
// the warp copies them, 8 vectors a lane in flight before their stores.
constexpr int kMovesInFlight = 8;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 31;
  const RowMoves mv = row_moves(a, b * a.kv_heads + g);
  const int moves = mv.count[0];
  if (blockIdx.x == 0 && g == 0 && threadIdx.x == 0) a.new_lens[b] = *mv.new_len;
  const int warps = int(gridDim.x) * (kMoveThreads / 32);
  for (int j0 = (int(blockIdx.x) * (kMoveThreads / 32) + int(threadIdx.x >> 5)) * a.warp_moves;
       j0 < moves; j0 += warps * a.warp_moves) {
    const int n = min(a.warp_moves, moves - j0);
    int64_t s = 0, d = -1;
    int ts = 0, td = 0;
    if (lane < n) {
      s = slot_bytes(a, b, g, mv.src[j0 + lane], &ts);
      d = slot_bytes(a, b, g, mv.dst[j0 + lane], &td);
      if (s < 0 || d < 0) {
        atomicOr(a.diag, int32_t(kDiagBadOffset));
        d = -1;
      }
    }
    if (!a.kv4) {
      const int pieces = a.head_dim / 8;  // of a row, 16 bytes each; K's, then V's
      const int all = 2 * pieces * n;
      for (int i0 = lane; i0 - lane < all; i0 += 32 * kMovesInFlight) {
        uint4 x[kMovesInFlight];
        uint8_t *to[kMovesInFlight];
#pragma unroll
        for (int k = 0; k < kMovesInFlight; ++k) {
          const int i = i0 + 32 * k, m = min(i / (2 * pieces), n - 1);
          const int64_t sm = __shfl_sync(0xffffffffu, s, m), dm = __shfl_sync(0xffffffffu, d, m);
          const int e = i - m * 2 * pieces;
          uint8_t *base = e < pieces ? a.va_k : a.va_v;
          const int at = (e < pieces ? e : e - pieces) * 16;
          to[k] = i < all && dm >= 0 ? base + dm + at : nullptr;
          if (to[k]) x[k] = __ldcs(reinterpret_cast<const uint4 *>(base + sm + at));
        }
#pragma unroll
        for (int k = 0; k < kMovesInFlight; ++k)
          if (to[k]) *reinterpret_cast<uint4 *>(to[k]) = x[k];
      }
      continue;
    }
    const int groups = a.head_dim / 32;
    for (int m = 0; m < n; ++m) {
      const int64_t sm = __shfl_sync(0xffffffffu, s, m), dm = __shfl_sync(0xffffffffu, d, m);
      const int tsm = __shfl_sync(0xffffffffu, ts, m), tdm = __shfl_sync(0xffffffffu, td, m);
      if (dm < 0) continue;
      for (int i = lane; i < 4 * groups; i += 32) {  // K: the 4 words of each group
        const int jg = i / 4, c = i % 4;
        *reinterpret_cast<uint32_t *>(
            a.va_k + dm + kv4_code_offset(groups, jg, (tdm & 7) * 4 + c, tdm >> 3)) =
            *reinterpret_cast<const uint32_t *>(
                a.va_k + sm + kv4_code_offset(groups, jg, (tsm & 7) * 4 + c, tsm >> 3));
      }
      for (int i = lane; i < 8 * groups; i += 32) {  // V: the 8 half words of each group
        const int jg = i / 8, q = i % 8;
        *reinterpret_cast<uint16_t *>(
            a.va_v + dm + kv4_code_offset(groups, jg, q * 4 + (tdm & 7) / 2, tdm >> 3) +
            (tdm & 1) * 2) =
            *reinterpret_cast<const uint16_t *>(
                a.va_v + sm + kv4_code_offset(groups, jg, q * 4 + (tsm & 7) / 2, tsm >> 3) +
                (tsm & 1) * 2);
      }
      for (int i = lane; i < 2 * groups; i += 32) {
        uint8_t *base = i < groups ? a.va_k : a.va_v;
        const int jg = i % groups;
        *reinterpret_cast<uint16_t *>(base + dm +
                                      kv4_scale_offset(i >= groups, groups, tdm, jg)) =
            *reinterpret_cast<const uint16_t *>(base + sm +
                                                kv4_scale_offset(i >= groups, groups, tsm, jg));
      }
    }
  }
}

}  // namespace

cudaError_t evict_tokens(const EvictArgs &args, cudaStream_t stream) {
  EvictArgs a = args;
  const int rows = a.batch * a.kv_heads;
  a.most_moves = std::min(a.budget, std::max(a.max_tokens - a.budget, 0));
  CallScratch scratch;
  cudaError_t e = scratch.acquire(
      stream, (size_t(rows) + a.batch + size_t(rows) * a.most_moves * 2) * 4);
  if (e != cudaSuccess) return e;
  a.scratch = static_cast<int32_t *>(scratch.ptr);
  // CTAs of a row's cluster: as many as leave each kSliceTokens, while they all run at once.
  // 16 rows of up to 16,900 tokens: slices of 2048 tokens (8 CTAs) 41 us, 4096 (4) 24.6, 8192
  // (2) 31, whole rows 43.  A whole row above it takes 1024 threads (32 rows of 8000 tokens:
  // 25.5 against 27.9 us), all else 512 (16 rows of 3700 in CTAs of their own 29.3 us both ways,
  // 512 of 1200 47 against 58; the clusters above 28.3, with registers spilled).
  int C = 1;
  while (C < kMaxCluster && a.max_tokens / (2 * C) >= kSliceTokens &&
         int64_t(rows) * 2 * C <= device_sm_count())
    C *= 2;
  a.key_capacity = std::min((a.max_tokens + C - 1) / C, kKeyCapacity);
  const int smem = a.key_capacity * 4;
  const int threads = C == 1 && a.max_tokens > kSliceTokens ? 1024 : 512;
  void (*fn)(const EvictArgs) = C > 1            ? evict_select_kernel<512, true>
                                : threads == 512 ? evict_select_kernel<512, false>
                                                 : evict_select_kernel<1024, false>;
  // The attribute belongs to the kernel, not to the launch: always the largest, so that a call of
  // another width on another thread does not lower it between here and the launch.
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeyCapacity * 4);
  if (e != cudaSuccess) {
    scratch.release(stream);
    return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, a.kv_heads, a.batch);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (C > 1 ? 1 : 0);
  e = cudaLaunchKernelEx(&cfg, fn, a);
  if (e == cudaSuccess) {
    // enough warps for every SM, none for moves that cannot be
    const int most = std::max(a.most_moves, 1);
    // 8 a warp while that leaves warps idle: 35.2 -> 30.8 us for one row of 16,384 tokens cut to
    // half; 32 where there are many: 40.3 -> 32.0 us for 128 rows of 3700 cut to 1024
    a.warp_moves = int64_t(rows) * most <= int64_t(device_sm_count()) * 64 * 8 ? 8 : 32;
    const int per = kMoveThreads / 32 * a.warp_moves;
    const int want = std::max(1, 8 * device_sm_count() / rows);
    const int grid = std::min((most + per - 1) / per, want);
    e = launch_pdl(evict_move_kernel, dim3(grid, a.kv_heads, a.batch), dim3(kMoveThreads), 0,
                   stream, a);
  }
  const cudaError_t r = scratch.release(stream);
  return e != cudaSuccess ? e : r;
}

}  // namespace dev
}  // namespace kcmm

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
// The selection is a radix select (11 + 11 + 10 bits) over 32-bit keys, a cluster of CTAs a
// row.  It is bound by the latency of its passes over the row's weights, which stay in L1
// and L2 after the first.  The moves are a copy, bound by HBM.
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

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;

// One row's moves: count, then [budget] each of destination slots, source slots and the
// weights and positions that move with them.
struct RowMoves {
  int32_t *count, *dst, *src, *pos;
  float *w;
};
__device__ __forceinline__ RowMoves row_moves(const EvictArgs &a, int row) {
  const int64_t rows = int64_t(a.batch) * a.kv_heads, at = int64_t(row) * a.budget;
  RowMoves r;
  r.count = a.scratch + row;
  r.dst = a.scratch + rows + at;
  r.src = r.dst + rows * a.budget;
  r.pos = r.src + rows * a.budget;
  r.w = reinterpret_cast<float *>(r.pos + rows * a.budget);
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

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ int s_hist[kBins];
  __shared__ Counts s_warp[kSelectWarps];
  __shared__ Counts s_cta;
  __shared__ int s_scan[kSelectWarps];
  __shared__ int s_digit, s_above;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
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
      if (g == 0) a.new_lens[b] = n;
      atomicOr(a.diag, int32_t(kDiagBadLaunch));
    }
    return;
  }
  if (rank == 0 && tid == 0) {
    mv.count[0] = 0;
    if (g == 0) a.new_lens[b] = min(n, a.budget);
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
  auto key_of = [&](int i) {
    const int p = pos_of(i);
    return p < a.sinks || p >= next - a.recent ? kHeldKey : weight_key(w_in[i]);
  };

  // ---- threshold: the budget-th largest key, and how many equal to it stay -------------
  uint32_t prefix = 0;
  int want = a.budget;  // keys to take among those that match the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int top = pass == 0 ? 32 : pass == 1 ? 21 : 10;  // bits below are undecided
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kSelectThreads) s_hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const uint32_t k = key_of(i);
      if (pass == 0 || (k >> top) == prefix) atomicAdd(&s_hist[(k >> shift) & mask], 1);
    }
    cluster.sync();
    // Bins from the top: thread t has bins 2047 - 2t and 2046 - 2t, all CTAs' sums.
    const int hi = kBins - 1 - 2 * tid;
    int c0 = 0, c1 = 0;
    for (int r = 0; r < C; ++r) {
      const int *h = cluster.map_shared_rank(s_hist, r);
      c0 += h[hi];
      c1 += h[hi - 1];
    }
    int sum = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += s_scan[w];
    before += sum - c0 - c1;  // keys above this thread's bins
    if (before < want && before + c0 >= want) {
      s_digit = hi;
      s_above = before;
    } else if (before + c0 < want && before + c0 + c1 >= want) {
      s_digit = hi - 1;
      s_above = before + c0;
    }
    cluster.sync();  // every CTA has read this one's histogram
    prefix = (prefix << (pass == 2 ? 10 : 11)) | uint32_t(s_digit);
    want -= s_above;
  }
  const uint32_t threshold = prefix;  // `want` keys equal to it stay: the lowest slots

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
  if (tid == 0) {
    Counts t = {0, 0, 0, 0};
    for (int w = 0; w < kSelectWarps; ++w) {
      t.gt += s_warp[w].gt;
      t.eq += s_warp[w].eq;
      t.gt_lo += s_warp[w].gt_lo;
      t.eq_lo += s_warp[w].eq_lo;
    }
    s_cta = t;
  }
  cluster.sync();
  int gt = 0, eq = 0, gt_lo = 0, eq_lo = 0;  // gt, eq: before this warp's segment
  for (int r = 0; r < C; ++r) {
    const Counts t = *cluster.map_shared_rank(&s_cta, r);
    if (r < rank) {
      gt += t.gt;
      eq += t.eq;
    }
    gt_lo += t.gt_lo;
    eq_lo += t.eq_lo;
  }
  for (int w = 0; w < warp; ++w) {
    gt += s_warp[w].gt;
    eq += s_warp[w].eq;
  }
  const int kept_lo = gt_lo + min(eq_lo, want);  // slots below the budget that stay
  const int moves = a.budget - kept_lo;

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
    if (in && i < a.budget && !keep) mv.dst[i - kept_before] = i;
    if (keep && i >= a.budget) {
      const int j = kept_before - kept_lo;
      mv.src[j] = i;
      mv.w[j] = w_in[i];
      mv.pos[j] = pos_of(i);
    }
    gt += __popc(gts);
    eq += __popc(eqs);
  }
  if (rank == 0 && tid == 0) mv.count[0] = moves;
  __threadfence();
  cluster.sync();  // the lists are complete, and nothing past the budget is read again

  // ---- weights and positions of the kept slots; the slots past them weigh 0 --------------
  for (int i = begin + tid; i < end; i += kSelectThreads) {
    if (i < a.budget) {
      const float w = w_in[i];
      const int p = pos_of(i);
      w_out[i] = w;
      p_out[i] = p;
    } else {
      w_out[i] = 0.f;
    }
  }
  cluster.sync();
  for (int j = rank * kSelectThreads + tid; j < moves; j += C * kSelectThreads) {
    const int d = __ldcg(mv.dst + j);
    w_out[d] = __ldcg(mv.w + j);
    p_out[d] = __ldcg(mv.pos + j);
  }
}

constexpr int kMoveThreads = 256;

// First byte of head g's row (16-bit cache) or chunk (4-bit cache) of slot i, and the
// token's place in its chunk; null where the table or the offset is bad.
__device__ __forceinline__ int64_t slot_bytes(const EvictArgs &a, int b, int g, int i, int *t) {
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

// One warp a move.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 31;
  const RowMoves mv = row_moves(a, b * a.kv_heads + g);
  const int moves = mv.count[0];
  const int warps = int(gridDim.x) * (kMoveThreads / 32);
  for (int j = int(blockIdx.x) * (kMoveThreads / 32) + (threadIdx.x >> 5); j < moves; j += warps) {
    int ts, td;
    const int64_t s = slot_bytes(a, b, g, mv.src[j], &ts), d = slot_bytes(a, b, g, mv.dst[j], &td);
    if (s < 0 || d < 0) {
      if (lane == 0) atomicOr(a.diag, int32_t(kDiagBadOffset));
      continue;
    }
    if (!a.kv4) {
      const int pieces = a.head_dim / 8;  // 16 bytes each; K's, then V's
      for (int i = lane; i < 2 * pieces; i += 32) {
        uint8_t *base = i < pieces ? a.va_k : a.va_v;
        const int at = (i < pieces ? i : i - pieces) * 16;
        *reinterpret_cast<uint4 *>(base + d + at) = *reinterpret_cast<const uint4 *>(base + s + at);
      }
    } else {
      const int groups = a.head_dim / 32;
      for (int i = lane; i < 4 * groups; i += 32) {  // K: the 4 words of each group
        const int jg = i / 4, c = i % 4;
        *reinterpret_cast<uint32_t *>(a.va_k + d + kv4_code_offset(groups, jg, (td & 7) * 4 + c, td >> 3)) =
            *reinterpret_cast<const uint32_t *>(
                a.va_k + s + kv4_code_offset(groups, jg, (ts & 7) * 4 + c, ts >> 3));
      }
      for (int i = lane; i < 8 * groups; i += 32) {  // V: the 8 half words of each group
        const int jg = i / 8, q = i % 8;
        *reinterpret_cast<uint16_t *>(a.va_v + d + kv4_code_offset(groups, jg, q * 4 + (td & 7) / 2, td >> 3) +
                                      (td & 1) * 2) =
            *reinterpret_cast<const uint16_t *>(
                a.va_v + s + kv4_code_offset(groups, jg, q * 4 + (ts & 7) / 2, ts >> 3) + (ts & 1) * 2);
      }
      for (int i = lane; i < 2 * groups; i += 32) {
        uint8_t *base = i < groups ? a.va_k : a.va_v;
        const int jg = i % groups;
        *reinterpret_cast<uint16_t *>(base + d + kv4_scale_offset(i >= groups, groups, td, jg)) =
            *reinterpret_cast<const uint16_t *>(base + s + kv4_scale_offset(i >= groups, groups, ts, jg));
      }
    }
  }
}

}  // namespace

cudaError_t evict_tokens(const EvictArgs &args, cudaStream_t stream) {
  EvictArgs a = args;
  const int rows = a.batch * a.kv_heads;
  CallScratch scratch;
  cudaError_t e = scratch.acquire(stream, (size_t(rows) + size_t(rows) * a.budget * 4) * 4);
  if (e != cudaSuccess) return e;
  a.scratch = static_cast<int32_t *>(scratch.ptr);
  // CTAs of a row's cluster: as many as leave each 2048 tokens, while they all run at once.
  int C = 1;
  while (C < kMaxCluster && a.max_tokens / (2 * C) >= 2048 &&
         int64_t(rows) * 2 * C <= device_sm_count())
    C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, a.kv_heads, a.batch);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
  if (e == cudaSuccess) {
    // a move is 1 to 2 KB each way: enough warps for every SM, none for moves that cannot be
    const int most = std::min(a.budget, std::max(a.max_tokens - a.budget, 1));
    const int per = kMoveThreads / 32;
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

// The 4-bit KV cache: quantising append, read-back, and paged decode attention over it.
//
// Format.  A row (one token, one kv head) of D values is cut into groups of 32:
//   s = bf16(max|x| / 7),  code = round-half-even(x / s) in [-7, 7],  value = code * s
// (codes 0 where s is 0; a group that holds an infinity or NaN stores s = NaN and reads as
// NaN).  4.5 bits a value, 9/32 of the 16-bit cache.
//
// Layout.  A page holds [kv head][16-token unit] chunks of 9 D bytes: 8 D of codes, then
// 16 D/32 scales.  Inside a chunk the codes lie in the order in which the lanes of a warp
// hold the operands of mma.m16n8k16, so a decode warp loads them straight from global
// memory into its operand registers, 16 bytes a lane, without shared memory or shuffles:
//   K (A operand, rows = tokens): lane (g, c) holds words of tokens g and g+8;
//     the word of group j has dims 32j+8c+{0..7}, dim 2i in nibble i and 2i+1 in nibble i+4;
//   V (A operand transposed, rows = dims): the lane's words are tokens (2c, 2c+1) and
//     (2c+8, 2c+9), the even token in the low half; nibble i is dim 32j+4g+i.
// No byte holds two tokens, so appends need no read-modify-write.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../launch.hpp"
#include "finish.cuh"
#include "kv4_layout.cuh"
#include "pdl.cuh"
#include "ptx.cuh"

namespace kcmm {
namespace dev {
namespace {

constexpr int kUnit = kKv4Unit;
constexpr int kGroup = kKv4Group;

// --- append and read -----------------------------------------------------------------

// First byte of the chunk that holds `slot`, or -1 (a status as for the 16-bit slot write).
__device__ __forceinline__ int64_t chunk_of(const Kv4RowsArgs &a, int64_t slot, int *t) {
  const int64_t blk = slot / a.block_size;
  const int in = int(slot - blk * a.block_size);
  *t = in % kUnit;
  if (blk >= a.offsets_len) {
    if (a.status) atomicCAS(a.status, 0, 1);
    return -1;
  }
  if (a.valid && !a.valid[blk]) {
    if (a.status) atomicCAS(a.status, 0, 2);
    return -1;
  }
  const uint64_t off = a.block_offsets[blk] * 2;
  const uint64_t page = uint64_t(a.block_size) / kUnit * a.kv_heads * 9 * a.head_dim;
  if ((off & 15) || off + page > a.region_bytes) {
    if (a.status) atomicCAS(a.status, 0, 1);
    return -1;
  }
  return int64_t(off) + int64_t(in / kUnit) * 9 * a.head_dim;
}

// Four consecutive values a thread; the 8 threads of a group share its maximum.
template <typename T>
__global__ void kv4_append_kernel(const Kv4RowsArgs a) {
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int row = blockIdx.x;
  const int64_t slot = a.slot_mapping[row];
  if (slot < 0) return;
  int t;
  const int64_t chunk0 = chunk_of(a, slot, &t);
  if (chunk0 < 0) return;
  const int D = a.head_dim, groups = D / kGroup, quads = a.kv_heads * D / 4;
  const int64_t head_stride = int64_t(a.block_size / kUnit) * 9 * D;
  // quads is a multiple of 8: the 8 threads of a group run or idle together
  for (int base = 0; base < 2 * quads; base += blockDim.x) {
    const int i0 = base + int(threadIdx.x);
    const bool live = i0 < 2 * quads;
    const int i = live ? i0 : 0;
    const bool is_v = i >= quads;
    const int e = (is_v ? i - quads : i) * 4, head = e / D, d = e - head * D;
    const T *src = static_cast<const T *>(is_v ? a.v : a.k) +
                   int64_t(row) * (is_v ? a.v_stride : a.k_stride) + e;
    __align__(8) T raw[4];
    if (a.vec) {
      *reinterpret_cast<uint2 *>(raw) = *reinterpret_cast<const uint2 *>(src);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) raw[k] = src[k];
    }
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = ptx::to_f32(raw[k]);
    float mx = 0.f;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mx = fmaxf(mx, fabsf(x[k]));
      bad |= !isfinite(x[k]);
    }
    if (bad) mx = INFINITY;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    // The 16-bit inputs and the 8-bit scale make x / s miss every rounding boundary by far
    // more than a 32-bit quotient's rounding, unless it lies on one: the codes are exact.
    __nv_bfloat16 s = __float2bfloat16_rn(__fdiv_rn(mx, 7.f));
    if (mx == INFINITY) s = __ushort_as_bfloat16(0x7fc0);
    const float sf = __bfloat162float(s);
    uint32_t n[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float q = sf > 0.f ? rintf(__fdiv_rn(x[k], sf)) : 0.f;
      q = fminf(fmaxf(q, -7.f), 7.f);
      n[k] = uint32_t(int(q) + 8);
    }
    const int j = d / kGroup, in = (d % kGroup) / 4;  // the thread's place in its group
    uint8_t *chunk = static_cast<uint8_t *>(is_v ? a.va_v : a.va_k) + chunk0 + head * head_stride;
    const uint32_t half = n[0] | (n[2] << 4) | (n[1] << 16) | (n[3] << 20);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, half, 1);
    if (!live) continue;
    if (is_v) {
      const int lane = in * 4 + (t & 7) / 2;
      *reinterpret_cast<uint16_t *>(chunk + kv4_code_offset(groups, j, lane, t >> 3) + (t & 1) * 2) =
          uint16_t(n[0] | (n[1] << 4) | (n[2] << 8) | (n[3] << 12));
    } else if ((in & 1) == 0) {
      const int lane = (t & 7) * 4 + in / 2;
      *reinterpret_cast<uint32_t *>(chunk + kv4_code_offset(groups, j, lane, t >> 3)) =
          half | (other << 8);
    }
    if (in == 0) *reinterpret_cast<__nv_bfloat16 *>(chunk + kv4_scale_offset(groups, t, j)) = s;
  }
}

template <typename T>
__global__ void kv4_read_kernel(const Kv4RowsArgs a) {
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int row = blockIdx.x;
  const int64_t slot = a.slot_mapping[row];
  if (slot < 0) return;
  int t;
  const int64_t chunk0 = chunk_of(a, slot, &t);
  if (chunk0 < 0) return;
  const int D = a.head_dim, groups = D / kGroup, quads = a.kv_heads * D / 4;
  const int64_t head_stride = int64_t(a.block_size / kUnit) * 9 * D;
  for (int i = threadIdx.x; i < 2 * quads; i += blockDim.x) {
    const bool is_v = i >= quads;
    const int e = (is_v ? i - quads : i) * 4, head = e / D, d = e - head * D;
    const int j = d / kGroup, in = (d % kGroup) / 4;
    const uint8_t *chunk =
        static_cast<const uint8_t *>(is_v ? a.va_v : a.va_k) + chunk0 + head * head_stride;
    uint32_t n[4];
    if (is_v) {
      const int lane = in * 4 + (t & 7) / 2;
      const uint32_t w = *reinterpret_cast<const uint16_t *>(
          chunk + kv4_code_offset(groups, j, lane, t >> 3) + (t & 1) * 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = (w >> (4 * k)) & 15u;
    } else {
      const int lane = (t & 7) * 4 + in / 2;
      const uint32_t w =
          *reinterpret_cast<const uint32_t *>(chunk + kv4_code_offset(groups, j, lane, t >> 3)) >>
          ((in & 1) * 8);
      n[0] = w & 15u;
      n[2] = (w >> 4) & 15u;
      n[1] = (w >> 16) & 15u;
      n[3] = (w >> 20) & 15u;
    }
    const float s = __bfloat162float(
        *reinterpret_cast<const __nv_bfloat16 *>(chunk + kv4_scale_offset(groups, t, j)));
    T *dst = static_cast<T *>(is_v ? a.v : a.k) +
             int64_t(row) * (is_v ? a.v_stride : a.k_stride) + e;
    __align__(8) T y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = ptx::from_f32<T>(float(int(n[k]) - 8) * s);
    if (a.vec) {
      *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(y);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[k] = y[k];
    }
  }
}

// --- decode ----------------------------------------------------------------------------

constexpr int kWarps = 4;

struct Kv4Params {
  const void *q;
  void *out;
  const int32_t *tables;
  const int32_t *seq_lens;
  const uint64_t *offsets;
  const uint8_t *va_k;
  const uint8_t *va_v;
  uint64_t region_bytes;
  int batch, hq, hkv, bs, max_bps;
  float scale_log2;
  int units_per_split, num_splits, n_head_tiles, heads_per_tile;
  float *part_o, *part_lse;
  float *scores;
  int64_t score_stride;
  int32_t *diag;
  int64_t q_sb, q_sh, o_sb, o_sh, bt_stride;
  bool q_vec;  // every query row starts on 16 bytes
};

// Two codes of a word to f16: 0x6400 is 1024 with a unit of 1 in its last place, so a
// nibble or-ed into bits 0-3 (4-7) adds n (16 n); the subtraction (multiply-add) that
// leaves n - 8 is exact.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  uint32_t x = (w & 0x000f000fu) | 0x64006400u;
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64086408u));
  return x;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
  uint32_t x = (w & 0x00f000f0u) | 0x64006400u;
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x) : "r"(0x2c002c00u), "r"(0xd480d480u));
  return x;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// One lane's share of a unit: K and V words and the scales of tokens g and g+8.
template <int D>
struct UnitRegs {
  static constexpr int NG = D / kGroup;  // pages are read through L2 alone, once each
  alignas(16) uint32_t k[2 * NG];
  alignas(16) uint32_t v[2 * NG];
  alignas(16) uint32_t ks[NG];
  alignas(16) uint32_t vs[NG];  // 2 NG bf16: token g's groups, then token g+8's

  __device__ __forceinline__ void load(const uint8_t *kc, const uint8_t *vc, int lane) {
    if constexpr (NG % 2 == 0) {
#pragma unroll
      for (int j = 0; j < NG / 2; ++j) {
        *reinterpret_cast<uint4 *>(k + 4 * j) =
            __ldcg(reinterpret_cast<const uint4 *>(kc + (j * 32 + lane) * 16));
        *reinterpret_cast<uint4 *>(v + 4 * j) =
            __ldcg(reinterpret_cast<const uint4 *>(vc + (j * 32 + lane) * 16));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        *reinterpret_cast<uint2 *>(k + 2 * j) =
            __ldcg(reinterpret_cast<const uint2 *>(kc + (j * 32 + lane) * 8));
        *reinterpret_cast<uint2 *>(v + 2 * j) =
            __ldcg(reinterpret_cast<const uint2 *>(vc + (j * 32 + lane) * 8));
      }
    }
    const uint8_t *kp = kc + NG * 256 + (lane >> 2) * (NG * 4);
    const uint8_t *vp = vc + NG * 256 + (lane >> 2) * (NG * 4);
    if constexpr (NG % 4 == 0) {
#pragma unroll
      for (int j = 0; j < NG; j += 4) {
        *reinterpret_cast<uint4 *>(ks + j) = __ldcg(reinterpret_cast<const uint4 *>(kp + 4 * j));
        *reinterpret_cast<uint4 *>(vs + j) = __ldcg(reinterpret_cast<const uint4 *>(vp + 4 * j));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        ks[j] = __ldcg(reinterpret_cast<const uint32_t *>(kp) + j);
        vs[j] = __ldcg(reinterpret_cast<const uint32_t *>(vp) + j);
      }
    }
  }
  // scale of token g (w = 0) or g + 8 (w = 1), group j
  __device__ __forceinline__ static float scale(const uint32_t *s, int w, int j) {
    const int i = w * NG + j;
    return i & 1 ? bf16_hi(s[i >> 1]) : bf16_lo(s[i >> 1]);
  }
};

template <typename T, int D, int NT, bool SCORES>
__global__ void __launch_bounds__(kWarps * 32) kv4_decode_kernel(const Kv4Params p) {
  constexpr int NG = D / kGroup;
  constexpr int HT = 8 * NT;  // heads of a tile
  extern __shared__ __align__(16) float kv4_smem[];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int b = blockIdx.z, split = blockIdx.x;
  const int kvh = int(blockIdx.y) / p.n_head_tiles, ht = int(blockIdx.y) % p.n_head_tiles;
  const int seq_len = min(p.seq_lens[b], p.max_bps * p.bs);
  if (seq_len <= 0) return;
  const int n_units = (seq_len + kUnit - 1) / kUnit;
  const int u_begin = split * p.units_per_split;
  if (u_begin >= n_units) return;
  const int u_end = min(u_begin + p.units_per_split, n_units);
  const int group_lo = int((int64_t(kvh) * p.hq + p.hkv - 1) / p.hkv);
  const int group_hi = int((int64_t(kvh + 1) * p.hq + p.hkv - 1) / p.hkv);
  const int lo = group_lo + ht * HT;
  const int G = min(group_hi - lo, HT);
  if (G <= 0) return;

  // ---- Q as the B operand (columns = heads), scaled per head by a power of two --------
  // f16 for both input types: with the row's largest magnitude brought into [64, 128) every
  // bf16 or f16 value is exact down to 2^-20 of that, and nothing overflows.
  uint32_t qb[NT][NG][4];
  float s_scale[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
    float x[NG][8];
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const T *src = static_cast<const T *>(p.q) + int64_t(b) * p.q_sb +
                     int64_t(lo + min(h, G - 1)) * p.q_sh + j * kGroup + c * 8;
      __align__(16) T tmp[8];
      if (p.q_vec) {
        *reinterpret_cast<uint4 *>(tmp) = *reinterpret_cast<const uint4 *>(src);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) tmp[e] = src[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[j][e] = h < G ? ptx::to_f32(tmp[e]) : 0.f;
        mx = fmaxf(mx, fabsf(x[j][e]));
      }
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int ex = max(int((__float_as_uint(mx) >> 23) & 255u) - 127, -100);
    const float up = __uint_as_float(uint32_t(127 + 6 - ex) << 23);
    const float down = __uint_as_float(uint32_t(127 - 6 + ex) << 23) * p.scale_log2;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qb[nt][j][i] = ptx::Mma<__half>::pack(x[j][2 * i] * up, x[j][2 * i + 1] * up);
    }
    // this lane's score columns are heads 2c and 2c+1
    s_scale[nt][0] = __shfl_sync(0xffffffffu, down, (2 * c) * 4);
    s_scale[nt][1] = __shfl_sync(0xffffffffu, down, (2 * c + 1) * 4);
  }

  const int n_w = (u_end - u_begin - warp + kWarps - 1) / kWarps;  // this warp's units
  const int64_t chunk_bytes = 9 * D;
  const int units_per_page = p.bs / kUnit;
  const int64_t page_bytes = int64_t(units_per_page) * p.hkv * chunk_bytes;

  float o[NT][2 * NG][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }
  float v_up = 0.f;  // power of two on the V scales inside P

  int64_t my_at = -1;  // lane i: byte offset of the chunk of unit i of the current 32
  auto resolve = [&](int k0) {
    my_at = -1;
    const int k = k0 + lane;
    if (k < n_w) {
      const int u = u_begin + warp + k * kWarps;
      const int page = u / units_per_page, in = u - page * units_per_page;
      const int blk = p.tables[int64_t(b) * p.bt_stride + page];
      if (blk >= 0) {
        const uint64_t off = p.offsets[blk] * 2;
        if ((off & 15) == 0 && off + page_bytes <= p.region_bytes)
          my_at = int64_t(off) + (int64_t(kvh) * units_per_page + in) * chunk_bytes;
      }
      if (my_at < 0) atomicOr(p.diag, int32_t(kDiagBadOffset));
    }
  };

  UnitRegs<D> cur, nxt;
  bool cur_ok = false, nxt_ok = false;
  auto fetch = [&](int k, UnitRegs<D> &r) {
    if ((k & 31) == 0) resolve(k);
    const int64_t at = __shfl_sync(0xffffffffu, my_at, k & 31);
    if (at >= 0) r.load(p.va_k + at, p.va_v + at, lane);
    return at >= 0;
  };
  if (n_w > 0) cur_ok = fetch(0, cur);

  for (int k = 0; k < n_w; ++k) {
    nxt_ok = k + 1 < n_w ? fetch(k + 1, nxt) : false;
    const int u = u_begin + warp + k * kWarps;
    const int nvalid = cur_ok ? min(kUnit, seq_len - u * kUnit) : 0;
    const bool in0 = g < nvalid, in1 = g + 8 < nvalid;
    if (nvalid > 0) {
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w0 = cur.k[2 * j], w1 = cur.k[2 * j + 1];
        const uint32_t a0[4] = {low_codes(w0), low_codes(w1), high_codes(w0), high_codes(w1)};
        const uint32_t a1[4] = {low_codes(w0 >> 8), low_codes(w1 >> 8), high_codes(w0 >> 8),
                                high_codes(w1 >> 8)};
        const float k0 = UnitRegs<D>::scale(cur.ks, 0, j), k1 = UnitRegs<D>::scale(cur.ks, 1, j);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          ptx::Mma<__half>::run(acc, a0, qb[nt][j][0], qb[nt][j][1]);
          ptx::Mma<__half>::run(acc, a1, qb[nt][j][2], qb[nt][j][3]);
          if (j == 0) {
            s[nt][0] = acc[0] * k0;
            s[nt][1] = acc[1] * k0;
            s[nt][2] = acc[2] * k1;
            s[nt][3] = acc[3] * k1;
          } else {
            s[nt][0] = fmaf(acc[0], k0, s[nt][0]);
            s[nt][1] = fmaf(acc[1], k0, s[nt][1]);
            s[nt][2] = fmaf(acc[2], k1, s[nt][2]);
            s[nt][3] = fmaf(acc[3], k1, s[nt][3]);
          }
        }
      }
      float v0[NG], v1[NG], vmx = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        // a slot past the context holds anything: its scales count as 0
        v0[j] = in0 ? UnitRegs<D>::scale(cur.vs, 0, j) : 0.f;
        v1[j] = in1 ? UnitRegs<D>::scale(cur.vs, 1, j) : 0.f;
        vmx = fmaxf(vmx, fmaxf(v0[j], v1[j]));
      }
      bool raise = vmx * v_up > 64.f || v_up == 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = i < 2 ? in0 : in1;
          s[nt][i] = in ? s[nt][i] * s_scale[nt][i & 1] : -INFINITY;
          raise |= s[nt][i] > m[nt][i & 1] + 8.f;
        }
        if constexpr (SCORES) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int h = nt * 8 + 2 * c + (i & 1);
            if (h < G)
              p.scores[(int64_t(b) * p.hq + lo + h) * p.score_stride + u * kUnit + g +
                       (i >> 1) * 8] = s[nt][i];
          }
        }
      }
      // The running maximum is raised only when a score exceeds it by more than 8 (a factor
      // of 256, which P's f16 range holds), the V normaliser only past a factor of 64: both
      // are rare after a warp's first unit, so most units skip the rescaling of O.
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int o2 = 1; o2 < 32; o2 <<= 1) vmx = fmaxf(vmx, __shfl_xor_sync(0xffffffffu, vmx, o2));
        float vr = 1.f;
        if (vmx * v_up > 64.f || v_up == 0.f) {
          const int ex = max(int(__float_as_uint(vmx) >> 23) - 127, -100);
          const float up = __uint_as_float(uint32_t(127 + 2 - ex) << 23);
          vr = v_up == 0.f ? 1.f : up / v_up;
          v_up = up;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(s[nt][i], s[nt][i + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[nt][i]);
            const float r = m[nt][i] == -INFINITY ? 0.f : ptx::fast_exp2(m[nt][i] - mx);
            m[nt][i] = mx;
            l[nt][i] *= r;
#pragma unroll
            for (int d = 0; d < 2 * NG; ++d) {
              o[nt][d][i] *= r * vr;
              o[nt][d][i + 2] *= r * vr;
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        v0[j] *= v_up;
        v1[j] *= v_up;
      }
      uint32_t pb[NT][NG][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[nt][i] = ptx::fast_exp2(s[nt][i] - m[nt][i & 1]);
          l[nt][i & 1] += s[nt][i];
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          // P in f16 carries 11 bits beside the scales' and codes' exact products
          pb[nt][j][0] = transpose8x8(ptx::Mma<__half>::pack(s[nt][0] * v0[j], s[nt][1] * v0[j]));
          pb[nt][j][1] = transpose8x8(ptx::Mma<__half>::pack(s[nt][2] * v1[j], s[nt][3] * v1[j]));
        }
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w0 = cur.v[2 * j], w1 = cur.v[2 * j + 1];
        const uint32_t a0[4] = {low_codes(w0), high_codes(w0), low_codes(w1), high_codes(w1)};
        const uint32_t a1[4] = {low_codes(w0 >> 8), high_codes(w0 >> 8), low_codes(w1 >> 8),
                                high_codes(w1 >> 8)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          ptx::Mma<__half>::run(o[nt][2 * j], a0, pb[nt][j][0], pb[nt][j][1]);
          ptx::Mma<__half>::run(o[nt][2 * j + 1], a1, pb[nt][j][0], pb[nt][j][1]);
        }
      }
    } else if constexpr (SCORES) {
      // a page that could not be read: its tokens weigh nothing
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        const int h = (i >> 2) * 8 + 2 * c + (i & 1);
        if (h < G)
          p.scores[(int64_t(b) * p.hq + lo + h) * p.score_stride + u * kUnit + g +
                   ((i >> 1) & 1) * 8] = -INFINITY;
      }
    }
    cur = nxt;
    cur_ok = nxt_ok;
  }

  // ---- merge the warps ----------------------------------------------------------------
  float *cO = kv4_smem;                 // [kWarps][HT][D]
  float *cm = cO + kWarps * HT * D;     // [kWarps][HT]
  float *cl = cm + kWarps * HT;         // [kWarps][HT]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[nt][i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int h = nt * 8 + 2 * c + i;
      if (g == 0) {
        cm[warp * HT + h] = m[nt][i];
        cl[warp * HT + h] = sum;
      }
      const float down = v_up == 0.f ? 0.f : 1.f / v_up;
      if (h < G) {
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          *reinterpret_cast<float4 *>(cO + (warp * HT + h) * D + j * kGroup + g * 4) =
              make_float4(o[nt][2 * j][i] * down, o[nt][2 * j][i + 2] * down,
                          o[nt][2 * j + 1][i] * down, o[nt][2 * j + 1][i + 2] * down);
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), d = (i % (D / 4)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, cm[w * HT + h]);
    float L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = cm[w * HT + h], lw = cl[w * HT + h];
      if (mw == -INFINITY && lw == 0.f) continue;  // the warp saw no token
      const float sc = ptx::fast_exp2(mw - M);
      const float4 v = *reinterpret_cast<const float4 *>(cO + (w * HT + h) * D + d);
      L += lw * sc;
      x.x += v.x * sc;
      x.y += v.y * sc;
      x.z += v.z * sc;
      x.w += v.w * sc;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (p.num_splits == 1 && !SCORES) {
      T *dst = static_cast<T *>(p.out) + int64_t(b) * p.o_sb + int64_t(lo + h) * p.o_sh + d;
      dst[0] = ptx::from_f32<T>(x.x * inv);
      dst[1] = ptx::from_f32<T>(x.y * inv);
      dst[2] = ptx::from_f32<T>(x.z * inv);
      dst[3] = ptx::from_f32<T>(x.w * inv);
    } else {
      const int64_t row = (int64_t(b) * p.hq + lo + h) * p.num_splits + split;
      *reinterpret_cast<float4 *>(p.part_o + row * D + d) =
          make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
      if (d == 0) p.part_lse[row] = M + log2f(L);
    }
  }
}

using Kv4Fn = void (*)(const Kv4Params);

template <typename T, int D, int NT>
Kv4Fn pick_scores(bool scores) {
  return scores ? kv4_decode_kernel<T, D, NT, true> : kv4_decode_kernel<T, D, NT, false>;
}
template <typename T, int D>
Kv4Fn pick_tiles(int nt, bool scores) {
  return nt == 1 ? pick_scores<T, D, 1>(scores) : pick_scores<T, D, 2>(scores);
}
template <typename T>
Kv4Fn pick(int D, int nt, bool scores) {
  switch (D) {
    case 32: return pick_tiles<T, 32>(nt, scores);
    case 64: return pick_tiles<T, 64>(nt, scores);
    case 96: return pick_tiles<T, 96>(nt, scores);
    case 128: return pick_tiles<T, 128>(nt, scores);
    case 160: return pick_tiles<T, 160>(nt, scores);
    case 192: return pick_tiles<T, 192>(nt, scores);
    case 224: return pick_tiles<T, 224>(nt, scores);
    case 256: return pick_tiles<T, 256>(nt, scores);
    default: return nullptr;
  }
}

}  // namespace

cudaError_t kv4_append(const Kv4RowsArgs &a, cudaStream_t stream) {
  const int items = 2 * a.kv_heads * a.head_dim / 4;
  const int threads = std::min(512, (items + 31) / 32 * 32);
  return launch_pdl(a.dtype == Dtype::BF16 ? kv4_append_kernel<__nv_bfloat16>
                                           : kv4_append_kernel<__half>,
                    dim3(a.num_tokens), dim3(threads), 0, stream, a);
}

cudaError_t kv4_read(const Kv4RowsArgs &a, cudaStream_t stream) {
  const int items = 2 * a.kv_heads * a.head_dim / 4;
  const int threads = std::min(512, (items + 31) / 32 * 32);
  return launch_pdl(a.dtype == Dtype::BF16 ? kv4_read_kernel<__nv_bfloat16>
                                           : kv4_read_kernel<__half>,
                    dim3(a.num_tokens), dim3(threads), 0, stream, a);
}

cudaError_t kv4_decode_attention(const DecodeArgs &a, const DecodeWeights &w,
                                 cudaStream_t stream) {
  const int D = a.head_dim;
  const int g_max = (a.num_q_heads + a.kv_heads - 1) / a.kv_heads;
  const int nt = g_max <= 8 ? 1 : 2;
  const bool scores = w.w_out != nullptr;
  const Kv4Fn fn = a.dtype == Dtype::BF16 ? pick<__nv_bfloat16>(D, nt, scores)
                                          : pick<__half>(D, nt, scores);
  if (!fn) return cudaErrorNotSupported;
  Kv4Params p = {};
  p.q = a.q;
  p.out = a.out;
  p.tables = a.block_tables;
  p.seq_lens = a.seq_lens;
  p.offsets = a.block_offsets;
  p.va_k = static_cast<const uint8_t *>(a.va_k);
  p.va_v = static_cast<const uint8_t *>(a.va_v);
  p.region_bytes = a.region_elems * 2;
  p.batch = a.batch;
  p.hq = a.num_q_heads;
  p.hkv = a.kv_heads;
  p.bs = a.block_size;
  p.max_bps = a.max_blocks_per_seq;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.diag = a.diag;
  const int64_t dense_row = int64_t(a.num_q_heads) * D;
  p.q_sb = a.q_stride_token ? a.q_stride_token : dense_row;
  p.q_sh = a.q_stride_head ? a.q_stride_head : D;
  p.o_sb = a.out_stride_token ? a.out_stride_token : dense_row;
  p.o_sh = a.out_stride_head ? a.out_stride_head : D;
  p.bt_stride = a.tables_stride ? a.tables_stride : a.max_blocks_per_seq;
  p.q_vec = ((reinterpret_cast<uintptr_t>(a.q) & 15) | (p.q_sb & 7) | (p.q_sh & 7)) == 0;
  p.n_head_tiles = (g_max + 8 * nt - 1) / (8 * nt);

  const int max_units = int((int64_t(a.max_blocks_per_seq) * a.block_size + kUnit - 1) / kUnit);
  const int64_t items = int64_t(a.batch) * a.kv_heads * p.n_head_tiles;
  const int64_t target = int64_t(device_sm_count()) * 4 * 4;
  const int64_t want = std::max<int64_t>(1, (target + items - 1) / items);
  int ups = int((max_units + want - 1) / want);
  ups = std::max(ups, 16);
  p.units_per_split = ups;
  p.num_splits = (max_units + ups - 1) / ups;

  const size_t rows = size_t(a.batch) * a.num_q_heads;
  const bool partial = p.num_splits > 1 || scores;
  p.score_stride = int64_t(max_units) * kUnit;
  size_t bytes = 0;
  if (partial) bytes = rows * p.num_splits * (size_t(D) + 1) * 4;
  bytes = (bytes + 15) & ~size_t(15);
  const size_t scores_at = bytes;
  if (scores) bytes += rows * size_t(p.score_stride) * 4;
  CallScratch scratch;
  if (bytes) {
    cudaError_t e = scratch.acquire(stream, bytes);
    if (e != cudaSuccess) return e;
    p.part_o = static_cast<float *>(scratch.ptr);
    p.part_lse = p.part_o + rows * p.num_splits * D;
    if (scores) p.scores = reinterpret_cast<float *>(static_cast<char *>(scratch.ptr) + scores_at);
  }
  const size_t smem = size_t(kWarps) * 8 * nt * (D + 2) * 4;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e == cudaSuccess)
    e = launch_pdl(fn, dim3(p.num_splits, a.kv_heads * p.n_head_tiles, a.batch),
                   dim3(kWarps * 32), smem, stream, p);
  if (e == cudaSuccess && partial) {
    FinishParams f = {};
    f.seq_lens = a.seq_lens;
    f.max_tokens = a.max_blocks_per_seq * a.block_size;
    f.hq = a.num_q_heads;
    f.hkv = a.kv_heads;
    f.head_dim = D;
    f.num_splits = p.num_splits;
    f.tokens_per_split = p.units_per_split * kUnit;
    f.part_o = p.part_o;
    f.part_lse = p.part_lse;
    f.out = a.out;
    f.o_sb = p.o_sb;
    f.o_sh = p.o_sh;
    f.scores = p.scores;
    f.score_stride = p.score_stride;
    f.w_in = w.w_in;
    f.w_out = w.w_out;
    f.w_stride = w.w_stride;
    const int chunks = scores ? (f.max_tokens + kFinishTokens - 1) / kFinishTokens : 1;
    e = launch_pdl(a.dtype == Dtype::BF16 ? finish_kernel<__nv_bfloat16> : finish_kernel<__half>,
                   dim3(chunks, a.kv_heads, a.batch), dim3(kFinishThreads), 0, stream, f);
  }
  const cudaError_t r = scratch.release(stream);
  return e != cudaSuccess ? e : r;
}

}  // namespace dev
}  // namespace kcmm

// The 4-bit KV cache: quantising append, read-back, and paged decode attention over it.
//
// Format.  A row (one token, one kv head) of D values is cut into groups of 32:
//   s = bf16(max|x| / 7),  code = round-half-even(x / s) in [-7, 7],  value = code * s
// (codes 0 where s is 0; a group that holds an infinity or NaN stores s = NaN and reads as
// NaN).  4.5 bits a value, 9/32 of the 16-bit cache.
//
// Layout.  A page holds [kv head][16-token unit] chunks of 9 D bytes: 8 D of codes, then
// 16 D/32 scales.  Inside a chunk the codes lie in the order in which the lanes of a warp
// hold the operands of the decode's mma, so that it reads them 16 bytes a lane and unpacks
// them in place, without shuffles or transposes:
//   K (A operand, rows = tokens): lane (g, c) holds words of tokens g and g+8;
//     the word of group j has dims 32j+8c+{0..7}, dim 2i in nibble i and 2i+1 in nibble i+4;
//   V (A operand transposed, rows = dims): the lane's words are tokens (2c, 2c+1) and
//     (2c+8, 2c+9), the even token in the low half; nibble i is dim 32j+4g+i.
// The scales lie in the order of the accumulators they meet: K's by token (g, g+8), V's by
// token pair as the codes.
// No byte holds two tokens, so appends need no read-modify-write.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

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
//
// One warp a head and K or V of a tile of rows.  Where the tile's 16 slots are one unit of a
// page (a prompt's chunk), lane (g, c) takes exactly the values whose codes it holds in the
// layout: its source loads are whole 32-byte sectors, its code stores one 16-byte vector a
// pair of groups, and no byte goes through shared memory.  Other tiles (decode steps, the
// ends of a chunk) go row by row, 8 values a lane.  16,384 tokens of 8 heads of 128 took 179 us
// row by row for both kernels and take 45 by units.  Neither HBM (1.9 TB/s of its 6.4 in the append)
// nor the issue slots (61 and 68 %) are full there: a warp waits for the loads of one pair of
// groups before it asks for the next one's.  Short inputs are bound by the latency of
// slot -> offset -> row (64 tokens: 4.4 us).

constexpr int kRowsThreads = 128;
// A tile has a unit's 16 rows where that leaves every SM kTileWarps warps, else kFewRows: at 8
// heads 16 rows take 9.2, 10.1, 11.1 and 45 us for 512, 1024, 2048 and 16,384 tokens, 2 rows
// 5.4, 8.1, 12.9 and 81.  1 and 4 rows take 4.5 and 5.6 us for 64 tokens, 2 rows 4.4.
constexpr int kTileWarps = 10;
constexpr int kFewRows = 2;

template <typename T>
__device__ __forceinline__ float widen16(uint32_t bits) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    return __half2float(__ushort_as_half(uint16_t(bits)));
  } else {
    return __uint_as_float(bits << 16);
  }
}

// The scale of a group from the largest magnitude bits among its values.
struct GroupScale {
  uint32_t bits;  // bf16
  float s, inv;
  int kind;  // 0: the codes are 0; 1: quotients through 1/s; 2: s is too small or large for that
};
// max / 7 by the reciprocal: the product's error is under half a unit of 24 bits, and a value
// of 11 bits over 7 lies 2^-13 or more from where bf16 rounding turns, unless it lies on it;
// then the product rounds to it.
template <typename T>
__device__ __forceinline__ GroupScale group_scale(uint32_t mag) {
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  GroupScale r;
  const float mx = widen16<T>(mag);
  const bool plain = mx > 1e-28f && mx < 1e30f;
  float s = mx * (1.f / 7.f);
  if (!plain) s = __fdiv_rn(mx, 7.f);
  const __nv_bfloat16 rounded = __float2bfloat16_rn(s);
  r.bits = mag >= kInf ? 0x7fc0u : uint32_t(__bfloat16_as_ushort(rounded));
  r.s = __bfloat162float(rounded);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv) : "f"(r.s));
  r.kind = mag >= kInf || r.s == 0.f ? 0 : plain ? 1 : 2;
  return r;
}

// code + 8 of N values, in the low 4 bits of 0x4b400000 + code + 8.  The quotient by the
// approximate reciprocal is corrected once by its exact remainder (Markstein's division step):
// half-way quotients come out exact, and all others of a value of 11 bits by a scale of 8 lie
// 2^-14 or more away from half-way, so that rounding to even on adding 1.5 2^23 gives the
// code of the exact quotient.
template <int N>
__device__ __forceinline__ void code_bits(const float *x, const GroupScale &r, uint32_t *n) {
  constexpr float kRound = 12582920.f;  // 1.5 2^23 + 8
  if (r.kind == 1) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float q = x[e] * r.inv;
      n[e] = __float_as_uint(fmaf(fmaf(-q, r.s, x[e]), r.inv, q) + kRound);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float q = r.kind == 0 ? 0.f : fminf(fmaxf(__fdiv_rn(x[e], r.s), -7.f), 7.f);
      n[e] = __float_as_uint(q + kRound);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void widen_all(const uint32_t *w, float *x) {
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = widen16<T>((w[e / 2] >> (16 * (e & 1))) & 0xffffu);
}

// Nibbles of 4 codes, code i at bit step * i, from code_bits' words.
template <int STEP>
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  constexpr uint32_t k = 0x4b400000u;
  return a + (b << STEP) + (c << (2 * STEP)) + (d << (3 * STEP)) -
         k * (1u + (1u << STEP) + (1u << (2 * STEP)) + (1u << (3 * STEP)));
}
// A K word: dims 8c + {0..7}, dim 2i in nibble i, 2i + 1 in nibble i + 4.
__device__ __forceinline__ uint32_t pack_k(const uint32_t *n) {
  return pack4<4>(n[0], n[2], n[4], n[6]) + (pack4<4>(n[1], n[3], n[5], n[7]) << 16);
}
__device__ __forceinline__ float code_value(uint32_t nibble, float s) {
  return (__uint_as_float(0x4b000000u | nibble) - 8388616.f) * s;  // (n - 8) s
}

// Byte offset of the first chunk (head 0) of the unit that holds `slot`, or -1 (with a status
// as for the 16-bit slot write); *t the slot's place in its unit.
__device__ __forceinline__ int64_t chunk_of(const Kv4RowsArgs &a, int64_t slot, int *t) {
  if (slot < 0) return -1;
  int64_t blk;
  int in;
  if (slot < 0x7fffffff) {
    blk = uint32_t(slot) / uint32_t(a.block_size);
    in = int(uint32_t(slot) - uint32_t(blk) * uint32_t(a.block_size));
  } else {
    blk = slot / a.block_size;
    in = int(slot - blk * a.block_size);
  }
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

// The rows of a warp's tile: lane i has row i's chunk; `unit` where they are one whole unit.
struct Tile {
  int row0, rows, head;
  bool is_v, unit;
  int64_t chunk;  // of row `lane`, at this head
  int t;
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const Kv4RowsArgs &a, Tile *tile) {
  const int lane = threadIdx.x & 31;
  const int w = int(blockIdx.y) * (kRowsThreads / 32) + int(threadIdx.x >> 5);
  if (w >= 2 * a.kv_heads) return false;
  tile->is_v = w >= a.kv_heads;
  tile->head = tile->is_v ? w - a.kv_heads : w;
  tile->row0 = int(blockIdx.x) * ROWS;
  tile->rows = min(ROWS, a.num_tokens - tile->row0);
  tile->chunk = -1;
  tile->t = 0;
  int64_t slot = -1;
  if (lane < tile->rows) {
    slot = a.slot_mapping[tile->row0 + lane];
    tile->chunk = chunk_of(a, slot, &tile->t);
    if (tile->chunk >= 0)
      tile->chunk += int64_t(tile->head) * (a.block_size / kUnit) * 9 * a.head_dim;
  }
  const int64_t first = __shfl_sync(0xffffffffu, slot, 0);
  const bool in_order = lane >= kUnit || (slot == first + lane && tile->chunk >= 0);
  tile->unit = ROWS == kUnit && first % kUnit == 0 && __all_sync(0xffffffffu, in_order);
  return true;
}

template <int N>
__device__ __forceinline__ void load_row(uint32_t *w, const uint16_t *src, bool vec) {
  if (vec) {
    if constexpr (N == 4) {
      *reinterpret_cast<uint4 *>(w) = __ldcs(reinterpret_cast<const uint4 *>(src));
    } else {
      *reinterpret_cast<uint2 *>(w) = __ldcs(reinterpret_cast<const uint2 *>(src));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = uint32_t(src[2 * i]) | (uint32_t(src[2 * i + 1]) << 16);
  }
}
template <int N>
__device__ __forceinline__ void store_row(uint16_t *dst, const uint32_t *w, bool vec) {
  if (vec) {
    if constexpr (N == 4) {
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(w);
    } else {
      *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      dst[2 * i] = uint16_t(w[i]);
      dst[2 * i + 1] = uint16_t(w[i] >> 16);
    }
  }
}
// Largest magnitude bits of N words' halves, by half.
template <int N>
__device__ __forceinline__ uint32_t magnitudes(const uint32_t *w) {
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < N; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return m;
}
__device__ __forceinline__ uint32_t larger_half(uint32_t m) { return max(m & 0xffffu, m >> 16); }

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kRowsThreads) kv4_append_kernel(const Kv4RowsArgs a) {
  constexpr int NG = D / kGroup, PAIR = NG % 2 == 0 ? 2 : 1;  // groups of a code vector
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  Tile tile;
  if (!find_tile<ROWS>(a, &tile)) return;
  const uint16_t *src = static_cast<const uint16_t *>(tile.is_v ? a.v : a.k) + tile.head * D;
  const int64_t stride = tile.is_v ? a.v_stride : a.k_stride;
  uint8_t *region = static_cast<uint8_t *>(tile.is_v ? a.va_v : a.va_k);
  src += int64_t(tile.row0) * stride;

  if (tile.unit) {
    uint8_t *chunk = region + __shfl_sync(0xffffffffu, tile.chunk, 0);
    alignas(16) uint32_t scales[2 * NG];
#pragma unroll
    for (int j0 = 0; j0 < NG; j0 += PAIR) {
      alignas(16) uint32_t codes[2 * PAIR];
#pragma unroll
      for (int jj = 0; jj < PAIR; ++jj) {
        const int j = j0 + jj;
        if (!tile.is_v) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {  // tokens g, g + 8: 8 values
            alignas(16) uint32_t x[4];
            load_row<4>(x, src + (g + 8 * w) * stride + j * kGroup + c * 8, a.vec);
            uint32_t m = magnitudes<4>(x);
            m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const GroupScale s = group_scale<T>(larger_half(m));
            uint32_t n[8];
            float f[8];
            widen_all<T, 8>(x, f);
            code_bits<8>(f, s, n);
            codes[jj * 2 + w] = pack_k(n);
            scales[w * NG + j] = s.bits;
          }
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w) {  // tokens 2c, 2c + 1 (+ 8): 4 values each
            alignas(8) uint32_t x0[2], x1[2];
            const uint16_t *at = src + (2 * c + 8 * w) * stride + j * kGroup + g * 4;
            load_row<2>(x0, at, a.vec);
            load_row<2>(x1, at + stride, a.vec);
            uint32_t m = larger_half(magnitudes<2>(x0)) | (larger_half(magnitudes<2>(x1)) << 16);
            m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const GroupScale s0 = group_scale<T>(m & 0xffffu), s1 = group_scale<T>(m >> 16);
            uint32_t n0[4], n1[4];
            float f[4];
            widen_all<T, 4>(x0, f);
            code_bits<4>(f, s0, n0);
            widen_all<T, 4>(x1, f);
            code_bits<4>(f, s1, n1);
            codes[jj * 2 + w] = pack4<4>(n0[0], n0[1], n0[2], n0[3]) |
                                (pack4<4>(n1[0], n1[1], n1[2], n1[3]) << 16);
            scales[2 * j + w] = s0.bits | (s1.bits << 16);
          }
        }
      }
      if constexpr (PAIR == 2) {
        *reinterpret_cast<uint4 *>(chunk + kv4_code_offset(NG, j0, lane, 0)) =
            *reinterpret_cast<const uint4 *>(codes);
      } else {
        *reinterpret_cast<uint2 *>(chunk + kv4_code_offset(NG, j0, lane, 0)) =
            *reinterpret_cast<const uint2 *>(codes);
      }
    }
    if (!tile.is_v && c == 0) {
#pragma unroll
      for (int i = 0; i < NG; ++i)
        *reinterpret_cast<uint32_t *>(chunk + NG * 256 + (g * NG + i) * 4) =
            scales[2 * i] | (scales[2 * i + 1] << 16);
    } else if (tile.is_v && g == 0) {
#pragma unroll
      for (int i = 0; i < 2 * NG; ++i)
        *reinterpret_cast<uint32_t *>(chunk + NG * 256 + (c * 2 * NG + i) * 4) = scales[i];
    }
    return;
  }

  constexpr int P = D / 8;  // lanes of a row
  for (int base = 0; base < tile.rows * P; base += 32) {
    const int i = base + lane, r = min(i / P, tile.rows - 1), piece = i % P;
    const int64_t at = __shfl_sync(0xffffffffu, tile.chunk, r);
    const int t = __shfl_sync(0xffffffffu, tile.t, r);
    const bool live = i < tile.rows * P && at >= 0;
    alignas(16) uint32_t x[4] = {0u, 0u, 0u, 0u};
    if (live) load_row<4>(x, src + r * stride + piece * 8, a.vec);
    uint32_t m = magnitudes<4>(x);  // P is a multiple of 4: the lanes of a group are one row's
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (!live) continue;
    const GroupScale s = group_scale<T>(larger_half(m));
    uint32_t n[8];
    float f[8];
    widen_all<T, 8>(x, f);
    code_bits<8>(f, s, n);
    const int j = piece / 4, q = piece % 4;
    uint8_t *chunk = region + at;
    if (!tile.is_v) {
      *reinterpret_cast<uint32_t *>(chunk + kv4_code_offset(NG, j, (t & 7) * 4 + q, t >> 3)) =
          pack_k(n);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint16_t *>(
            chunk + kv4_code_offset(NG, j, (2 * q + h) * 4 + (t & 7) / 2, t >> 3) + (t & 1) * 2) =
            uint16_t(pack4<4>(n[4 * h], n[4 * h + 1], n[4 * h + 2], n[4 * h + 3]));
    }
    if (q == 0)
      *reinterpret_cast<uint16_t *>(chunk + kv4_scale_offset(tile.is_v, NG, t, j)) =
          uint16_t(s.bits);
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return ptx::Mma<T>::pack(lo, hi);
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kRowsThreads) kv4_read_kernel(const Kv4RowsArgs a) {
  constexpr int NG = D / kGroup, PAIR = NG % 2 == 0 ? 2 : 1;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  Tile tile;
  if (!find_tile<ROWS>(a, &tile)) return;
  uint16_t *dst = static_cast<uint16_t *>(tile.is_v ? a.v : a.k) + tile.head * D;
  const int64_t stride = tile.is_v ? a.v_stride : a.k_stride;
  const uint8_t *region = static_cast<const uint8_t *>(tile.is_v ? a.va_v : a.va_k);
  dst += int64_t(tile.row0) * stride;

  if (tile.unit) {
    const uint8_t *chunk = region + __shfl_sync(0xffffffffu, tile.chunk, 0);
    uint32_t scales[2 * NG];  // K: two bf16 a word, token g's then token g + 8's; V: [group][w]
#pragma unroll
    for (int i = 0; i < (tile.is_v ? 2 * NG : NG); ++i)
      scales[i] = *reinterpret_cast<const uint32_t *>(
          chunk + NG * 256 + (tile.is_v ? c * 2 * NG + i : g * NG + i) * 4);
#pragma unroll
    for (int j0 = 0; j0 < NG; j0 += PAIR) {
      alignas(16) uint32_t codes[2 * PAIR];
      if constexpr (PAIR == 2) {
        *reinterpret_cast<uint4 *>(codes) = __ldcs(
            reinterpret_cast<const uint4 *>(chunk + kv4_code_offset(NG, j0, lane, 0)));
      } else {
        *reinterpret_cast<uint2 *>(codes) = __ldcs(
            reinterpret_cast<const uint2 *>(chunk + kv4_code_offset(NG, j0, lane, 0)));
      }
#pragma unroll
      for (int jj = 0; jj < PAIR; ++jj) {
        const int j = j0 + jj;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t x = codes[jj * 2 + w];
          if (!tile.is_v) {
            const int i = w * NG + j;
            const float s = __uint_as_float(i & 1 ? scales[i >> 1] & 0xffff0000u
                                                  : scales[i >> 1] << 16);
            alignas(16) uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              y[e] = pack16<T>(code_value((x >> (4 * e)) & 15u, s),
                               code_value((x >> (4 * e + 16)) & 15u, s));
            store_row<4>(dst + (g + 8 * w) * stride + j * kGroup + c * 8, y, a.vec);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float s = __uint_as_float(h ? scales[2 * j + w] & 0xffff0000u
                                                : scales[2 * j + w] << 16);
              const uint32_t z = x >> (16 * h);
              alignas(8) uint32_t y[2] = {
                  pack16<T>(code_value(z & 15u, s), code_value((z >> 4) & 15u, s)),
                  pack16<T>(code_value((z >> 8) & 15u, s), code_value((z >> 12) & 15u, s))};
              store_row<2>(dst + (2 * c + h + 8 * w) * stride + j * kGroup + g * 4, y, a.vec);
            }
          }
        }
      }
    }
    return;
  }

  constexpr int P = D / 8;
  for (int base = 0; base < tile.rows * P; base += 32) {
    const int i = base + lane, r = min(i / P, tile.rows - 1), piece = i % P;
    const int64_t at = __shfl_sync(0xffffffffu, tile.chunk, r);
    const int t = __shfl_sync(0xffffffffu, tile.t, r);
    if (i >= tile.rows * P || at < 0) continue;
    const int j = piece / 4, q = piece % 4;
    const uint8_t *chunk = region + at;
    const float s = __uint_as_float(
        uint32_t(*reinterpret_cast<const uint16_t *>(chunk + kv4_scale_offset(tile.is_v, NG, t, j)))
        << 16);
    alignas(16) uint32_t y[4];
    if (!tile.is_v) {
      const uint32_t x = *reinterpret_cast<const uint32_t *>(
          chunk + kv4_code_offset(NG, j, (t & 7) * 4 + q, t >> 3));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = pack16<T>(code_value((x >> (4 * e)) & 15u, s),
                         code_value((x >> (4 * e + 16)) & 15u, s));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t z = *reinterpret_cast<const uint16_t *>(
            chunk + kv4_code_offset(NG, j, (2 * q + h) * 4 + (t & 7) / 2, t >> 3) + (t & 1) * 2);
        y[2 * h] = pack16<T>(code_value(z & 15u, s), code_value((z >> 4) & 15u, s));
        y[2 * h + 1] = pack16<T>(code_value((z >> 8) & 15u, s), code_value((z >> 12) & 15u, s));
      }
    }
    store_row<4>(dst + r * stride + piece * 8, y, a.vec);
  }
}

// --- decode ----------------------------------------------------------------------------

constexpr int kWarps = 4;
// Query heads of a CTA, the columns of the mma.  More heads of a kv head become more CTAs, that
// unpack the same codes again, from L2: two tiles of 16 in a CTA's registers instead took a fifth
// longer for 16 sequences of up to 2000 tokens with 16 heads on 1 (now 19.4 us), 4 % for 32 of up
// to 4096 with 64 on 4 (38.0), a third at heads of 256 (28.6).
constexpr int kHeads = 8;
// Units of a CTA, at least.  8 leave more pieces to merge, 32 fewer CTAs: 13.2 and 14.6 us
// against 13.8 for 3 sequences of up to 777 tokens, 16.9 and 26.0 against 19.3 for 8 of up to
// 2000.
constexpr int kMinRange = 16;
// Pieces of a sequence, about, which its last CTA merges: 16 and 64 take 26.6 and 24.3 us
// against 22.1 for one of 32,768 tokens.
constexpr int kMaxPieces = 32;
// Pieces that the merge takes at a time: 4 and 16 take 30.8 and 28.4 us against 28.4 for 8
// sequences of 32,768 tokens and 8 heads on 1, and 13.6 and 14.2 against 13.8 for 3 of up to 777.  A
// first pass over their sums cost 2 us more.
constexpr int kMergeAtOnce = 8;
constexpr float kNoMax = -3e38f;  // a row's maximum before its first finite score
// The normaliser of a row lies kLift above its maximum (log2 units): probabilities are below
// 2^(kSlack - kLift), so that the sum of 2^18 values of bf16's largest stays below 32-bit's.
constexpr float kLift = 24.f, kSlack = 6.f;
constexpr int kStages = 3;  // steps of a warp's ring; 2 are as fast
constexpr uint64_t kWaitLimitNs = 1000000000ull;  // a chunk that has not landed in 1 s is
                                                  // reported, never waited on forever

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
  int n_head_tiles;
  float *part_o, *part_lse;  // two slots a CTA: [CTA][2][heads of a tile] rows
  int32_t *counters;         // a zero per CTA: pieces of a shared sequence that are done
  float *scores;             // SCORES: [batch * hq][score_stride], log2 units
  float *lse;                // SCORES: [batch * hq], log2 units
  int64_t score_stride;
  int32_t *diag;
  int64_t q_sb, q_sh, o_sb, o_sh, bt_stride;
  bool q_vec;  // every query row starts on 16 bytes
};

// The values of two of a word's codes, nibbles I and I + 4, exactly, in T.  f16: 0x6400 is 1024
// with a unit of 1 in its last place, so a nibble or-ed into bits 0-3 (4-7) adds n (16 n); the
// subtraction (multiply-add) that leaves n - 8 is exact.  bf16: 0x4300 is 128 alike, for bits 0-3
// alone.  `base` is that word in a register the compiler cannot see through: with both
// constants immediate the and-or takes two instructions instead of one.
template <typename T>
__device__ __forceinline__ uint32_t code_base() {
  uint32_t base;
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("mov.u32 %0, 0x64006400;" : "=r"(base));
  } else {
    asm volatile("mov.u32 %0, 0x43004300;" : "=r"(base));
  }
  return base;
}
template <typename T, int I>
__device__ __forceinline__ uint32_t codes_of(uint32_t w, uint32_t base) {
  constexpr bool kF16 = std::is_same<T, __half>::value;
  constexpr int kShift = kF16 ? I / 2 * 8 : I * 4;
  uint32_t x;
  if constexpr (kF16 && I % 2 == 1) {
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w >> kShift), "n"(0x00f000f0u), "r"(base));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x) : "r"(0x2c002c00u), "r"(0xd480d480u));
  } else {
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w >> kShift), "n"(0x000f000fu), "r"(base));
    if constexpr (kF16) {
      asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64086408u));
    } else {
      asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0x43084308u));
    }
  }
  return x;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// Units that a warp takes at a time: two give its loads, matrix products and shuffles
// something to overlap with (22.1 against 23.9 us for one sequence of 32,768 tokens, 8 kv
// heads of 128; equal for the batch below), as long as the registers of both fit.
__host__ __device__ constexpr int units_at_a_time(int D) { return D <= 128 ? 2 : 1; }
__host__ __device__ constexpr int ctas_per_sm(int D) { return D <= 128 ? 4 : 2; }

// The high halves of two floats, a's low; the low halves.
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __byte_perm(a, b, 0x7632);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
  return __byte_perm(a, b, 0x5410);
}

// K's scale of token g (w = 0) or g + 8 (w = 1), group j, of a lane's 2 NG scales
template <int NG>
__device__ __forceinline__ float k_scale(const uint32_t *ks, int w, int j) {
  const int i = w * NG + j;
  return i & 1 ? bf16_hi(ks[i >> 1]) : bf16_lo(ks[i >> 1]);
}

// N words from shared memory in the widest loads that N allows; step: 16-byte vectors (8
// where N is odd) lie this many bytes apart
template <int N>
__device__ __forceinline__ void load_words(uint32_t *r, const unsigned char *p, int step) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      *reinterpret_cast<uint4 *>(r + 4 * i) = *reinterpret_cast<const uint4 *>(p + i * step);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      *reinterpret_cast<uint2 *>(r + 2 * i) = *reinterpret_cast<const uint2 *>(p + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const uint32_t *>(p + i * step);
  }
}

// Work split.  The units of all sequences, end to end, are cut into equal ranges, one for each
// CTA x of a kv head (and head tile) y = blockIdx.y: lengths differ by a factor of 8 within
// a batch, and CTAs of one (sequence, split) each took 7 % longer for the Llama-3-8B decode batch
// (64 sequences of 512 to 4096 tokens, 8 kv heads of 128; now 65.9 us).  A sequence
// inside one range is finished there; the pieces of one that several CTAs share go to scratch
// and the last CTA to finish merges them.
//
// That batch fills neither HBM (2.6 TB/s) nor the issue slots (60 %): 16 tokens of a kv head cost
// about 480 warp instructions, more than half of them unpacking codes and forming their weights,
// in chains that 3.5 warps a scheduler do not cover (an issue finds 1.0 of them in a fixed
// latency, 0.85 at a busy pipe, 0.5 at a load).  Few sequences are bound by latency: lengths ->
// table -> offset -> chunk -> counter -> merge (13.8 us for 3 of up to 777 tokens).
//
// A CTA's warps take every kWarps-th step of NU units of its piece.  Each warp runs its own
// ring of kStages steps: a lane issues a unit's K and V chunks as two bulk copies, the whole
// warp reads its operands from shared memory.
template <typename T, int D, bool SCORES>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(D))
    kv4_decode_kernel(const Kv4Params p) {
  constexpr int NG = D / kGroup;
  constexpr int NU = units_at_a_time(D);
  constexpr uint32_t kChunk = 9 * D;
  extern __shared__ __align__(128) unsigned char kv4_smem[];
  __shared__ uint64_t s_bar[kWarps * kStages];
  __shared__ int s_fail, s_last;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = int(blockIdx.y) / p.n_head_tiles, ht = int(blockIdx.y) % p.n_head_tiles;
  // query heads h with h * hkv / hq == kvh
  const int group_lo = int((uint32_t(kvh) * uint32_t(p.hq) + p.hkv - 1) / uint32_t(p.hkv));
  const int group_hi = int((uint32_t(kvh + 1) * uint32_t(p.hq) + p.hkv - 1) / uint32_t(p.hkv));
  const int lo = group_lo + ht * kHeads;
  const int G = min(group_hi - lo, kHeads);
  if (G <= 0) return;

  // ---- this CTA's range of units, and the sequence it starts in ---------------------------
  const int cap = p.max_bps * p.bs;
  auto units_of = [&](int b) { return (min(max(p.seq_lens[b], 0), cap) + kUnit - 1) / kUnit; };
  // every warp for itself: lane i sums a run of sequences
  const int run = (p.batch + 31) / 32;
  const int b_lo = min(lane * run, p.batch), b_hi = min(b_lo + run, p.batch);
  int mine = 0;
#pragma unroll 4
  for (int i = b_lo; i < b_hi; ++i) mine += units_of(i);
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  const int total = __shfl_sync(0xffffffffu, incl, 31);
  // at least a step or two a warp, less only where the sequences themselves are shorter
  const int range = max((total + int(gridDim.x) - 1) / int(gridDim.x),
                        min(kMinRange, (total + p.batch - 1) / p.batch));
  const int r0 = int(blockIdx.x) * range, r1 = min(r0 + range, total);
  if (r0 >= total) return;
  int b_first = b_lo, before = incl - mine;  // units of the sequences before b
  const uint32_t found = __ballot_sync(0xffffffffu, before <= r0 && r0 < incl);
  if (before <= r0 && r0 < incl) {
    for (int n = units_of(b_first); before + n <= r0; n = units_of(b_first)) {
      before += n;
      ++b_first;
    }
  }
  b_first = __shfl_sync(0xffffffffu, b_first, __ffs(int(found)) - 1);
  before = __shfl_sync(0xffffffffu, before, __ffs(int(found)) - 1);
  uint64_t *bars = s_bar + warp * kStages;
  if (lane < kStages) ptx::mbar_init(ptx::smem_u32(bars + lane), 1);
  if (threadIdx.x == 0) s_fail = 0;
  ptx::fence_proxy_async_smem();
  __syncthreads();

  unsigned char *ring = kv4_smem + warp * kStages * NU * 2 * kChunk;
  const int units_per_page = p.bs / kUnit;
  int st = 0;  // stage and phase of the next step
  uint32_t parity = 0;
  auto advance = [&] {
    if (++st == kStages) {
      st = 0;
      parity ^= 1;
    }
  };
  // Count a finished piece of the sequence that starts in CTA `first`: true in the CTA that
  // finished last, which leaves the counter at zero for the next call.
  auto last_piece = [&](int first, int pieces) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();  // the CTA's pieces, which the barrier ordered before this
      int32_t *counter = p.counters + int64_t(blockIdx.y) * gridDim.x + first;
      s_last = atomicAdd(counter, 1) == pieces - 1;
      if (s_last) *counter = 0;
      __threadfence();
    }
    __syncthreads();
    return s_last != 0;
  };
  bool lost = false;      // a wait ran out: the rest of the range is given up (and reported)
  for (int b = b_first; before < r1; ++b) {
  const int n_units = units_of(b);
  if (n_units == 0) continue;
  const int seq_len = min(p.seq_lens[b], cap);
  const int u_begin = max(r0 - before, 0), u_end = min(r1 - before, n_units);
  const int x_first = before / range, x_last = (before + n_units - 1) / range;
  const int pieces = x_last - x_first + 1;  // CTAs that share the sequence
  const int slot = u_begin == 0 && before > r0 ? 1 : 0;
  const int at_first = before;
  before += n_units;
  if (lost) {
    if (pieces > 1) last_piece(x_first, pieces);
    continue;
  }

  // ---- Q as the B operand (columns = heads) -------------------------------------------------
  // In its own type, as it is: brought into f16's range by a power of two a row, as an earlier
  // form had it for 2.8 us of 63 less, it lost dims 2^-20 below the row's largest, however large
  // the keys there.  Loaded first: its latency overlaps the addresses'.
  __align__(16) T q_raw[NG][8];
  const T *src = static_cast<const T *>(p.q) + int64_t(b) * p.q_sb +
                 int64_t(lo + min(g, G - 1)) * p.q_sh + c * 8;
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (p.q_vec) {
      *reinterpret_cast<uint4 *>(q_raw[j]) =
          *reinterpret_cast<const uint4 *>(src + j * kGroup);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) q_raw[j][e] = src[j * kGroup + e];
    }
  }

  // ---- the warp's units and their first copies ------------------------------------------
  // step i of the warp: units first_unit + i * kWarps * NU + {0, .., NU - 1}; the addresses of
  // 32 units at a time, one a lane
  const int first_unit = u_begin + warp * NU;
  const int n_w = max(0, (u_end - first_unit + kWarps * NU - 1) / (kWarps * NU));
  int64_t my_at = -1;  // byte offset of the chunk of unit lane % NU of step k0 + lane / NU
  auto resolve = [&](int k0) {
    my_at = -1;
    const int i = k0 + lane / NU;
    const int u = first_unit + i * (kWarps * NU) + lane % NU;
    if (i < n_w && u < u_end) {
      const int page = u / units_per_page, in = u - page * units_per_page;
      const int blk = p.tables[int64_t(b) * p.bt_stride + page];
      if (blk >= 0) {
        const uint64_t off = p.offsets[blk] * 2;
        if ((off & 15) == 0 &&
            off + uint64_t(units_per_page) * p.hkv * kChunk <= p.region_bytes)
          my_at = int64_t(off) + (int64_t(kvh) * units_per_page + in) * kChunk;
      }
      if (my_at < 0) atomicOr(p.diag, int32_t(kDiagBadOffset));
    }
  };
  constexpr int kBatchSteps = 32 / NU;
  uint32_t readable = 0;  // bit st * NU + r: unit r of the step in stage st was copied
  // unit r of a stage: its K chunk, then its V chunk
  auto issue = [&](int k, int stage) {
    if (k % kBatchSteps == 0) resolve(k);
    int64_t at[NU];
    readable &= ~(((1u << NU) - 1) << (stage * NU));
#pragma unroll
    for (int r = 0; r < NU; ++r) {
      at[r] = __shfl_sync(0xffffffffu, my_at, (k % kBatchSteps) * NU + r);
      if (at[r] >= 0) readable |= 1u << (stage * NU + r);
    }
    if (lane == 0) {
      const uint32_t bar = ptx::smem_u32(bars + stage);
      const uint32_t dst = ptx::smem_u32(ring + stage * NU * 2 * kChunk);
      uint32_t bytes = 0;
#pragma unroll
      for (int r = 0; r < NU; ++r) bytes += at[r] >= 0 ? 2 * kChunk : 0u;
      ptx::mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
      for (int r = 0; r < NU; ++r) {
        if (at[r] >= 0) {
          ptx::bulk_g2s(dst + r * 2 * kChunk, p.va_k + at[r], kChunk, bar);
          ptx::bulk_g2s(dst + r * 2 * kChunk + kChunk, p.va_v + at[r], kChunk, bar);
        }
      }
    }
  };
  for (int k = 0; k < kStages && k < n_w; ++k) issue(k, (st + k) % kStages);

  uint32_t qb[NG][4];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qb[j][i] = g < G ? reinterpret_cast<const uint32_t *>(q_raw[j])[i] : 0u;
  }

  float o[2 * NG][4];  // O transposed: rows = dims, columns = heads
#pragma unroll
  for (int i = 0; i < 2 * NG; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2], l[2];
  m[0] = m[1] = kNoMax;
  l[0] = l[1] = 0.f;
  bool failed = false;
  using B = __nv_bfloat16;  // of the second product
  const uint32_t k_base = code_base<T>(), v_base = code_base<B>();

  for (int k = 0; k < n_w; ++k) {
    const int u = first_unit + k * (kWarps * NU);
    const bool landed = ptx::mbar_wait_bounded(ptx::smem_u32(bars + st), parity, kWaitLimitNs);
    if (!__all_sync(0xffffffffu, landed)) {
      failed = true;
      break;
    }
    const uint32_t units = (readable >> (st * NU)) & ((1u << NU) - 1);
    if (units == 0) {  // no page could be read: the tokens weigh nothing
      if constexpr (SCORES) {
        for (int i = lane; i < G * NU * kUnit; i += 32) {
          const int h = i / (NU * kUnit), t = u * kUnit + i % (NU * kUnit);
          if (t < u_end * kUnit)
            p.scores[(int64_t(b) * p.hq + lo + h) * p.score_stride + t] = -INFINITY;
        }
      }
      if (k + kStages < n_w) issue(k + kStages, st);
      advance();
      continue;
    }
    const unsigned char *chunk = ring + st * NU * 2 * kChunk;
    // ---- S = Q K^T, transposed: rows = tokens, columns = heads -----------------------------
    float s[NU][4];
#pragma unroll
    for (int r = 0; r < NU; ++r) {
      const unsigned char *kc = chunk + r * 2 * kChunk;
      alignas(16) uint32_t kw[2 * NG];
      alignas(16) uint32_t ks[NG];
      if constexpr (NG % 2 == 0) {
        load_words<2 * NG>(kw, kc + lane * 16, 512);
      } else {
#pragma unroll
        for (int j = 0; j < NG; ++j) load_words<2>(kw + 2 * j, kc + (j * 32 + lane) * 8, 0);
      }
      load_words<NG>(ks, kc + NG * 256 + g * (NG * 4), NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w0 = kw[2 * j], w1 = kw[2 * j + 1];
        const uint32_t a0[4] = {codes_of<T, 0>(w0, k_base), codes_of<T, 0>(w1, k_base),
                                codes_of<T, 1>(w0, k_base), codes_of<T, 1>(w1, k_base)};
        const uint32_t a1[4] = {codes_of<T, 2>(w0, k_base), codes_of<T, 2>(w1, k_base),
                                codes_of<T, 3>(w0, k_base), codes_of<T, 3>(w1, k_base)};
        const float k0 = k_scale<NG>(ks, 0, j), k1 = k_scale<NG>(ks, 1, j);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        ptx::Mma<T>::run(acc, a0, qb[j][0], qb[j][1]);
        ptx::Mma<T>::run(acc, a1, qb[j][2], qb[j][3]);
        float *sr = s[r];
        if (j == 0) {
          sr[0] = acc[0] * k0;
          sr[1] = acc[1] * k0;
          sr[2] = acc[2] * k1;
          sr[3] = acc[3] * k1;
        } else {
          sr[0] = fmaf(acc[0], k0, sr[0]);
          sr[1] = fmaf(acc[1], k0, sr[1]);
          sr[2] = fmaf(acc[2], k1, sr[2]);
          sr[3] = fmaf(acc[3], k1, sr[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][i] *= p.scale_log2;
    }
    alignas(16) uint32_t vs[NU][2 * NG];  // V's scales [group][token pair (2c, 2c+1) + 8 i]
#pragma unroll
    for (int r = 0; r < NU; ++r)
      load_words<2 * NG>(vs[r], chunk + r * 2 * kChunk + kChunk + NG * 256 + c * (NG * 8),
                         NG % 2 == 0 ? 16 : 8);

    // Slots past the context, and units whose page could not be read, hold anything: their
    // scores become -inf and their scales 0.
    if (units != (1u << NU) - 1 || seq_len - u * kUnit < NU * kUnit) {
#pragma unroll
      for (int r = 0; r < NU; ++r) {
        const int nvalid = (units >> r) & 1u ? seq_len - (u + r) * kUnit : 0;
        if (g >= nvalid) s[r][0] = s[r][1] = -INFINITY;
        if (g + 8 >= nvalid) s[r][2] = s[r][3] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) {
          const int t = 2 * c + (i & 1) * 8;
          vs[r][i] &= (t < nvalid ? 0x0000ffffu : 0u) | (t + 1 < nvalid ? 0xffff0000u : 0u);
        }
      }
    }
    if constexpr (SCORES) {
#pragma unroll
      for (int r = 0; r < NU; ++r) {
        if (u + r >= u_end) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = 2 * c + (i & 1);
          if (h < G)
            p.scores[(int64_t(b) * p.hq + lo + h) * p.score_stride + (u + r) * kUnit + g +
                     (i >> 1) * 8] = s[r][i];
        }
      }
    }
    // The normaliser m is raised only when a score exceeds the maximum that it was set for by more
    // than kSlack: rare after a warp's first step, so most steps skip the rescaling of O.
    bool raise = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float mx = fmaxf(s[0][i], s[0][i + 2]);
#pragma unroll
      for (int r = 1; r < NU; ++r) mx = fmaxf(mx, fmaxf(s[r][i], s[r][i + 2]));
      raise |= mx > m[i] + (kSlack - kLift);
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = kNoMax;
#pragma unroll
        for (int r = 0; r < NU; ++r) mx = fmaxf(mx, fmaxf(s[r][i], s[r][i + 2]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = fmaxf(m[i], mx + kLift);
        const float rr = ptx::fast_exp2(m[i] - mx);
        m[i] = mx;
        l[i] *= rr;
#pragma unroll
        for (int d = 0; d < 2 * NG; ++d) {
          o[d][i] *= rr;
          o[d][i + 2] *= rr;
        }
      }
    }
    // ---- O += V^T (P S)^T, S the scale of a token's group -------------------------------------
    // The codes are the A operand; the weight of a (token, head, group), the probability times
    // the scale in 32 bits, is the B operand (rows = tokens, columns = heads) as a pair of bf16,
    // its leading 8 bits and its remainder's: 16 bits, and the range of 32-bit floats.  One f16,
    // which took 57 us against 61 for the Llama-3-8B batch, rounds a probability of 11 bits twice
    // and loses groups and tokens whose scales lie far apart, since one range holds them all.
    float pt[NU][4];  // P transposed: head g, tokens (2c, 2c+1) + 8 i
#pragma unroll
    for (int r = 0; r < NU; ++r) {
      uint32_t x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = ptx::fast_exp2(s[r][i] - m[i & 1]);
        l[i & 1] += p;
        x[i] = __float_as_uint(p);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t hi = transpose8x8(high_halves(x[2 * i], x[2 * i + 1]));
        const uint32_t lo = transpose8x8(low_halves(x[2 * i], x[2 * i + 1]));
        pt[r][2 * i] = __uint_as_float(low_halves(lo, hi));
        pt[r][2 * i + 1] = __uint_as_float(high_halves(lo, hi));
      }
    }
#pragma unroll
    for (int r = 0; r < NU; ++r) {
      const unsigned char *vc = chunk + r * 2 * kChunk + kChunk;
      alignas(16) uint32_t vw[2 * NG];
      if constexpr (NG % 2 == 0) {
        load_words<2 * NG>(vw, vc + lane * 16, 512);
      } else {
#pragma unroll
        for (int j = 0; j < NG; ++j) load_words<2>(vw + 2 * j, vc + (j * 32 + lane) * 8, 0);
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w0 = vw[2 * j], w1 = vw[2 * j + 1];
        const uint32_t a0[4] = {codes_of<B, 0>(w0, v_base), codes_of<B, 1>(w0, v_base),
                                codes_of<B, 0>(w1, v_base), codes_of<B, 1>(w1, v_base)};
        const uint32_t a1[4] = {codes_of<B, 2>(w0, v_base), codes_of<B, 3>(w0, v_base),
                                codes_of<B, 2>(w1, v_base), codes_of<B, 3>(w1, v_base)};
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t sc = vs[r][2 * j + i];
          const float x0 = pt[r][2 * i] * bf16_lo(sc), x1 = pt[r][2 * i + 1] * bf16_hi(sc);
          const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
          hi[i] = high_halves(b0, b1);
          lo[i] = ptx::Mma<B>::pack(x0 - __uint_as_float(b0 & 0xffff0000u),
                                    x1 - __uint_as_float(b1 & 0xffff0000u));
        }
        ptx::Mma<B>::run(o[2 * j], a0, hi[0], hi[1]);
        ptx::Mma<B>::run(o[2 * j + 1], a1, hi[0], hi[1]);
        ptx::Mma<B>::run(o[2 * j], a0, lo[0], lo[1]);
        ptx::Mma<B>::run(o[2 * j + 1], a1, lo[0], lo[1]);
      }
    }
    __syncwarp();
    if (k + kStages < n_w) issue(k + kStages, st);
    advance();
  }
  if (failed) {
    // Let copies still in flight land before the shared memory is released (bounded as
    // well), then report.
    for (int st = 0; st < kStages; ++st) {
      ptx::mbar_wait_bounded(ptx::smem_u32(bars + st), 0, 1000000ull);
      ptx::mbar_wait_bounded(ptx::smem_u32(bars + st), 1, 1000000ull);
    }
    if (lane == 0) {
      atomicOr(p.diag, int32_t(kDiagWaitTimeout));
      s_fail = 1;
    }
  }
  __syncthreads();
  lost = s_fail;
  const bool whole = pieces == 1;
  float *part_o = p.part_o + (int64_t(blockIdx.y) * gridDim.x * 2) * kHeads * D;
  float *part_lse = p.part_lse + (int64_t(blockIdx.y) * gridDim.x * 2) * kHeads;
  auto store = [&](int h, int d, float4 x, float lse) {
    T *dst = static_cast<T *>(p.out) + int64_t(b) * p.o_sb + int64_t(lo + h) * p.o_sh + d;
    dst[0] = ptx::from_f32<T>(x.x);
    dst[1] = ptx::from_f32<T>(x.y);
    dst[2] = ptx::from_f32<T>(x.z);
    dst[3] = ptx::from_f32<T>(x.w);
    if constexpr (SCORES) {
      if (d == 0) p.lse[int64_t(b) * p.hq + lo + h] = lse;
    }
  };

  // ---- merge the warps (the rings are free) -----------------------------------------------
  float *cO = reinterpret_cast<float *>(kv4_smem);  // [kWarps][kHeads][D]
  float *cm = cO + kWarps * kHeads * D;                 // [kWarps][kHeads]
  float *cl = cm + kWarps * kHeads;                     // [kWarps][kHeads]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float sum = l[i];
    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    const int h = 2 * c + i;
    if (g == 0) {
      cm[warp * kHeads + h] = m[i];
      cl[warp * kHeads + h] = sum;
    }
    if (h < G) {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        *reinterpret_cast<float4 *>(cO + (warp * kHeads + h) * D + j * kGroup + g * 4) =
            make_float4(o[2 * j][i], o[2 * j][i + 2], o[2 * j + 1][i], o[2 * j + 1][i + 2]);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), d = (i % (D / 4)) * 4;
    float M = kNoMax;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, cm[w * kHeads + h]);
    float L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = cm[w * kHeads + h], lw = cl[w * kHeads + h];
      const float sc = ptx::fast_exp2(mw - M);
      const float4 v = *reinterpret_cast<const float4 *>(cO + (w * kHeads + h) * D + d);
      L += lw * sc;
      x.x += v.x * sc;
      x.y += v.y * sc;
      x.z += v.z * sc;
      x.w += v.w * sc;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L, lse = M + log2f(L);
    x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    if (whole) {
      if (!lost) store(h, d, x, lse);
    } else {
      const int64_t row = (int64_t(blockIdx.x) * 2 + slot) * kHeads + h;
      *reinterpret_cast<float4 *>(part_o + row * D + d) = x;
      if (d == 0) part_lse[row] = lse;
    }
  }
  // The next sequence's bulk copies refill what the merge wrote: a proxy of their own, which
  // only this orders after these threads' accesses (the barrier of either branch follows).
  ptx::fence_proxy_async_smem();
  if (whole) {
    __syncthreads();  // the rings' memory is free again
    continue;
  }
  // the last CTA of a shared sequence merges its pieces
  if (!last_piece(x_first, pieces) || lost) continue;
  // the first piece lies in its CTA's second slot unless it starts that CTA's range
  const int64_t first_row = (int64_t(x_first) * 2 + (at_first > x_first * range ? 1 : 0)) * kHeads;
  auto row_of = [&](int k) { return k == 0 ? first_row : int64_t(x_first + k) * 2 * kHeads; };
  for (int i = threadIdx.x; i < G * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), d = (i % (D / 4)) * 4;
    float M = -INFINITY, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    // kMergeAtOnce pieces at a time, their sums and rows in flight together
    for (int k0 = 0; k0 < pieces; k0 += kMergeAtOnce) {
      float lse[kMergeAtOnce], top = M;
      float4 v[kMergeAtOnce];
#pragma unroll
      for (int j = 0; j < kMergeAtOnce; ++j) {
        const int64_t row = row_of(min(k0 + j, pieces - 1)) + h;
        lse[j] = __ldcg(part_lse + row);
        v[j] = __ldcg(reinterpret_cast<const float4 *>(part_o + row * D + d));
        if (k0 + j >= pieces) lse[j] = -INFINITY;
        top = fmaxf(top, lse[j]);
      }
      const float r = top == -INFINITY ? 1.f : ptx::fast_exp2(M - top);
      M = top;
      L *= r;
      x = make_float4(x.x * r, x.y * r, x.z * r, x.w * r);
#pragma unroll
      for (int j = 0; j < kMergeAtOnce; ++j) {
        const float w = lse[j] == -INFINITY ? 0.f : ptx::fast_exp2(lse[j] - (M + kLift));
        L += w;
        x.x += v[j].x * w;
        x.y += v[j].y * w;
        x.z += v[j].z * w;
        x.w += v[j].w * w;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    store(h, d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv),
          M + kLift + log2f(L));
  }
  }
}

using Kv4Fn = void (*)(const Kv4Params);

template <typename T, int D>
Kv4Fn pick_scores(bool scores) {
  return scores ? kv4_decode_kernel<T, D, true> : kv4_decode_kernel<T, D, false>;
}
template <typename T>
Kv4Fn pick(int D, bool scores) {
  switch (D) {
    case 32: return pick_scores<T, 32>(scores);
    case 64: return pick_scores<T, 64>(scores);
    case 96: return pick_scores<T, 96>(scores);
    case 128: return pick_scores<T, 128>(scores);
    case 160: return pick_scores<T, 160>(scores);
    case 192: return pick_scores<T, 192>(scores);
    case 224: return pick_scores<T, 224>(scores);
    case 256: return pick_scores<T, 256>(scores);
    default: return nullptr;
  }
}

}  // namespace

namespace {

using Kv4RowsFn = void (*)(const Kv4RowsArgs);

template <typename T, int D>
Kv4RowsFn pick_rows(bool append, bool tiles) {
  return append ? tiles ? kv4_append_kernel<T, D, kUnit> : kv4_append_kernel<T, D, kFewRows>
                : tiles ? kv4_read_kernel<T, D, kUnit> : kv4_read_kernel<T, D, kFewRows>;
}
template <typename T>
Kv4RowsFn pick_rows(int D, bool append, bool tiles) {
  switch (D) {
    case 32: return pick_rows<T, 32>(append, tiles);
    case 64: return pick_rows<T, 64>(append, tiles);
    case 96: return pick_rows<T, 96>(append, tiles);
    case 128: return pick_rows<T, 128>(append, tiles);
    case 160: return pick_rows<T, 160>(append, tiles);
    case 192: return pick_rows<T, 192>(append, tiles);
    case 224: return pick_rows<T, 224>(append, tiles);
    case 256: return pick_rows<T, 256>(append, tiles);
    default: return nullptr;
  }
}

cudaError_t launch_rows(const Kv4RowsArgs &a, bool append, cudaStream_t stream) {
  const bool tiles =
      int64_t(a.num_tokens / kUnit) * 2 * a.kv_heads >= int64_t(kTileWarps) * device_sm_count();
  const Kv4RowsFn fn = a.dtype == Dtype::BF16
                           ? pick_rows<__nv_bfloat16>(a.head_dim, append, tiles)
                           : pick_rows<__half>(a.head_dim, append, tiles);
  if (!fn) return cudaErrorNotSupported;
  const int rows = tiles ? kUnit : kFewRows, per = kRowsThreads / 32;
  return launch_pdl(fn, dim3((a.num_tokens + rows - 1) / rows, (2 * a.kv_heads + per - 1) / per),
                    dim3(kRowsThreads), 0, stream, a);
}

}  // namespace

cudaError_t kv4_append(const Kv4RowsArgs &a, cudaStream_t stream) {
  return launch_rows(a, true, stream);
}

cudaError_t kv4_read(const Kv4RowsArgs &a, cudaStream_t stream) {
  return launch_rows(a, false, stream);
}

cudaError_t kv4_decode_attention(const DecodeArgs &a, const DecodeWeights &w,
                                 cudaStream_t stream) {
  const int D = a.head_dim;
  const int g_max = (a.num_q_heads + a.kv_heads - 1) / a.kv_heads;
  const bool scores = w.w_out != nullptr;
  const Kv4Fn fn = a.dtype == Dtype::BF16 ? pick<__nv_bfloat16>(D, scores)
                                          : pick<__half>(D, scores);
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
  p.n_head_tiles = (g_max + kHeads - 1) / kHeads;

  // One wave of CTAs, every one with its share of the units of one kv head's (head tile's)
  // tokens.  Four waves of smaller shares where those are many lost: 96 kv heads of 256, 4
  // sequences of 100 to 2000 tokens took 60 % longer (now 50 us), of 2000 to 6000 28 % (144).
  const int slots = device_sm_count() * ctas_per_sm(D), Y = a.kv_heads * p.n_head_tiles;
  const int X = int(std::min<int64_t>(std::max(1, slots / Y), int64_t(kMaxPieces) * a.batch));

  const size_t rows = size_t(a.batch) * a.num_q_heads, slots_used = size_t(X) * Y * 2 * kHeads;
  const int max_tokens = a.max_blocks_per_seq * a.block_size;
  p.score_stride = max_tokens;
  // piece outputs, their log-sum-exp, and for the weights the rows' own and the scores
  const size_t lse_at = slots_used * D * 4, row_at = lse_at + slots_used * 4;
  const size_t scores_at = (row_at + (scores ? rows * 4 : 0) + 15) & ~size_t(15);
  CallScratch scratch;
  cudaError_t e =
      scratch.acquire(stream, scores_at + (scores ? rows * size_t(max_tokens) * 4 : 0));
  if (e != cudaSuccess) return e;
  char *base = static_cast<char *>(scratch.ptr);
  p.part_o = reinterpret_cast<float *>(base);
  p.part_lse = reinterpret_cast<float *>(base + lse_at);
  p.lse = reinterpret_cast<float *>(base + row_at);
  p.scores = scores ? reinterpret_cast<float *>(base + scores_at) : nullptr;
  p.counters = scratch.counters;
  const int nu = units_at_a_time(D);
  const size_t smem = std::max(size_t(kWarps) * kStages * nu * 18 * D,  // rings
                               size_t(kWarps) * kHeads * (D + 2) * 4);  // warps' results
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e == cudaSuccess) e = launch_pdl(fn, dim3(X, Y), dim3(kWarps * 32), smem, stream, p);
  if (e == cudaSuccess && scores) {
    FinishParams f = {};
    f.seq_lens = a.seq_lens;
    f.max_tokens = max_tokens;
    f.hq = a.num_q_heads;
    f.hkv = a.kv_heads;
    f.num_splits = 1;
    f.tokens_per_split = max_tokens;
    f.part_lse = p.lse;
    f.scores = p.scores;
    f.score_stride = p.score_stride;
    f.w_in = w.w_in;
    f.w_out = w.w_out;
    f.w_stride = w.w_stride;
    e = launch_finish(a.dtype, f, a.batch, stream);
  }
  const cudaError_t r = scratch.release(stream);
  return e != cudaSuccess ? e : r;
}

}  // namespace dev
}  // namespace kcmm

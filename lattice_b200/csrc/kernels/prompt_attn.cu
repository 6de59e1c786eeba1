// Attention over packed prompts on the sm_100a tensor cores (tcgen05).
//
// Sequence b has queries [q_start[b], q_start[b+1]) and keys [k_start[b], k_start[b+1]) in
// packed rows; query i of nq attends to the keys j <= i + nk - nq (all nk where not causal):
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(scale log2(e) q_i.k_j - m_i + shift),
// with the running maximum m_i and sum of p in 32 bits over one pass of the keys.  A row that
// sees no key gives zeros.
//
// A work item is NT tiles of up to 128 rows of one sequence and kv head (row = query * G + head in
// the group of G, so that every K and V tile feeds the query heads of its group) over the keys
// that they see.  Persistent CTAs, one an SM, take items from a list; K and V go by in steps of 128
// keys (64 above head_dim 128) through a ring of shared memory tiles.
//   8 or 4 warps  softmax, thread = row of a tile: S from TMEM, P back to it, the output at the end
//   MMA warp      issue of QK and P.V, a whole warp in uniform control flow
//   TMA warp      K and V tiles: boxes of 64 values x a step's tokens, 128-byte swizzle, values past
//                 head_dim and tokens past the tensor zero-filled
//   Q warp        hands out the items and loads their Q tiles
//   checking warp V's tiles at the causal border
// TMEM holds O of both tiles and, in what is left, scores and P (enum Scores).  Two tiles take
// turns: the products of one run while the other's softmax does.  The scores stand in registers
// while P is computed, the maximum of a step is found beside its exponentials, which run on the
// maximum so far, and the first half of P goes to its product before the second is computed.
//
// What bounds it, by the clock in a CTA at head_dim 128 (a step of both tiles: 3000 cycles): the
// softmax, 2 x 128 keys for each of 128 threads, whose exponentials alone are 1536 cycles of the
// MUFU unit with a quarter of them computed otherwise; the products are 2200 (64 an MMA, Q's rows
// from shared memory).  At 64 the same softmax stands beside half the products.  The loops of all
// roles have to fit the SM's instruction cache: with some thousand instructions more they missed
// it and took up to a third longer.  Calls of few short items are bound by an item's chain of
// steps, some 10,000 cycles.
// Measured (device; one call after the other, inputs in L2 as far as they fit | L2 flushed, other
// kernels between the calls): 32,768 tokens of 8 heads on 1 of 128: 1.63 | 1.87 ms, 1350 | 1170
// TFLOP/s; 16 prompts of 1 to 2048 tokens, 32 heads on 8: 221 | 259 us, 860 | 730; 4
// chunks of 300 to 512 behind 2000 to 8192: 128 | 150 us, 1120 | 960; 8 prompts of 511 to 4001, 16
// heads on 4 of 64: 174 | 178 us, 600 | 590; 3 of 1025 to 5000, 8 on 2 of 256: 135 | 157 us, 1070 |
// 920; 32 single tokens over up to 4095: 54 | 63 us, and from HBM 4.3 TB/s.
//
// P is rounded to V's 16-bit type (both operands of a product have one type): an output is off
// by at most half a unit of that type times sum(p |v|) / sum(p) more than its own rounding.  (The
// remainder of P as a second product would add half of the products' 2200 cycles a step, which is
// 3300 beside the softmax's 3000.)
// m_i is raised when a step exceeds it by more than 2^8, so that P is at most 2^(shift + 8).  For
// f16 the shift is 7: P up to 2^15, and weights of 2^-31 of the largest are still held.  bf16's
// values reach 2^128, as 32 bits do, and the sum of P v must not pass that: there the shift lies so
// far below zero that the P of a row's keys add up to less than 1.  It goes by the item's keys and
// no further than they need, so that products of small values stay what they are as long as can be
// (down to 2^-93 in full for the largest weights of 32,768 keys).
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
constexpr float kShiftF16 = 7.f;    // log2 of P where a score is the maximum
constexpr float kRaise = 8.f;       // log2 by which a step has to exceed the maximum to raise it
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kQBlk = 128 * 128;  // 64 values of 128 rows
constexpr size_t kMaxSmem = 227 * 1024;
constexpr int kItemSlots = 2;

// How a tile's scores and P share the TMEM columns that O leaves.
enum class Scores {
  kInPlace,   // P over the scores: QK(j+1) after P.V(j)
  kSeparate,  // P beside the scores: QK(j+1) once the scores are in registers
  kDouble,    // two score buffers, P over each: QK(j+1) before P.V(j)
};

template <int DP>
struct Shape {
  static constexpr int NT = DP <= 128 ? 2 : 1;  // tiles of 128 rows: O takes DP columns each
  static constexpr Scores kScores = DP <= 64    ? Scores::kSeparate
                                    : DP <= 128 ? Scores::kInPlace
                                                : Scores::kDouble;
  static constexpr bool kAhead = kScores != Scores::kInPlace;  // QK(j+1) comes before P.V(j)
  static constexpr int kBufs = kScores == Scores::kDouble ? 2 : 1;
  static constexpr int kKeys = DP <= 128 ? 128 : 64;  // keys of a step
  static constexpr int kBlocks = DP / 64;
  static constexpr uint32_t kKvBlk = kKeys * 128;  // 64 values of a step's keys
  static constexpr uint32_t kTileQ = kBlocks * kQBlk;
  static constexpr uint32_t kTileKv = kBlocks * kKvBlk;
  static constexpr uint32_t kBars = 512, kMisc = 256, kPatch = 3 * DP * 2;
  static constexpr uint32_t kFixed = NT * kTileQ + kBars + kMisc + kPatch;
  static constexpr int kFit = int((kMaxSmem - kFixed) / kTileKv);
  static constexpr int kSlots = kFit > 10 ? 10 : kFit;  // K and V tiles in flight
  static_assert(kSlots >= 4, "K and V of two steps have to fit");
  static constexpr uint32_t kOffKv = NT * kTileQ;
  static constexpr uint32_t kOffBar = kOffKv + kSlots * kTileKv;
  static constexpr uint32_t kOffMisc = kOffBar + kBars, kOffPatch = kOffMisc + kMisc;
  static constexpr size_t kSmem = kOffPatch + kPatch;
  static constexpr int kSoftmaxWarps = 4 * NT;
  static constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
  // TMEM columns: scores, P where it is separate, O
  static constexpr uint32_t kS = 0;
  static constexpr uint32_t kP = kScores == Scores::kSeparate ? NT * kKeys : 0;
  static constexpr uint32_t kO = NT * kBufs * kKeys +
                                 (kScores == Scores::kSeparate ? NT * kKeys / 2 : 0);
  static_assert(kO + NT * DP <= kTmemCols, "TMEM");
  // barriers; those of a tile by [x][buffer]
  static constexpr int kQFull = 0, kQFree = 1, kKvFull = 2, kKvEmpty = kKvFull + kSlots,
                       kRaw = kKvEmpty + kSlots, kSFull = kRaw + kSlots,
                       kSFree = kSFull + NT * kBufs, kPFull = kSFree + NT,  // halves of P: + 1
                       kODone = kPFull + 2 * NT, kItemFull = kODone + 2 * NT,
                       kItemEmpty = kItemFull + kItemSlots, kChecked = kItemEmpty + kItemSlots,
                       kRead = kChecked + 2, kWant = kRead + 2, kDrain = kWant + 1, kSlot = kDrain + 1;
  static_assert((kSlot + 1) * 8 <= kBars, "barrier space");
  // Register split: the launch gives every thread kLaunchRegs; two softmax warpgroups then take
  // kSoftmaxRegs and the other one keeps kOtherRegs.  setmaxnreg.inc waits until the registers
  // are free in the CTA's pool, so that the split must not exceed it; the launcher checks the
  // compiled kernel's count too.
  static constexpr bool kSplitRegs = NT == 2;
  static constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
  static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= 384 * kLaunchRegs, "register pool");
};

struct Params {
  CUtensorMap tmk, tmv, tmq;
  PromptAttnArgs a;
  float scale_log2;
  uint32_t idesc_qk, idesc_pv;
  bool q_boxes;          // tmq holds: Q's tiles are boxes
  int tile_rows;         // of a tile's 128: whole tokens where Q's tiles are boxes
  uint32_t group_magic;  // ceil(2^32 / group), 0 for a group of 1
  int32_t *next_item;    // zero, and zero again after the call
  int parts;             // that an item is cut into, at most
  unsigned long long *merged;  // [item][softmax warp]: tickets that count the parts that are done
  unsigned long long ticket_base;
  float *part_o;         // [part][row of q][head][DP]: sums of P V
  float2 *part_ml;       // [part][row of q][head]: maximum (log2 units) and sum of P
};

template <typename T>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(uint16_t(bits)));
  return __uint_as_float(bits << 16);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return ptx::Mma<T>::pack(lo, hi);
}

// Bounded wait of a whole warp, which gives up as soon as another role has failed; every lane
// gets the same answer.  Short, since the roles' loops share the SM's instruction cache: the limit
// is 2^31 clock cycles, about a second.
// A wait that may SPAN an item, which takes some 60 cycles a key at most, has 2^38: more than the
// longest item.  A stall does not last that long: the copies and products of an item that does not
// go on are always waited for within a step too.  (A limit that starts anew with every step, tried
// instead, cost short prompts 2 to 4 %.)
template <bool SPAN>
__device__ __forceinline__ uint32_t wait_clock() {
  uint32_t t;
  if constexpr (SPAN) {
    asm volatile("mov.u32 %0, %%clock_hi;" : "=r"(t));
  } else {
    asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  }
  return t;
}
template <bool SPAN = false>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *fail) {
  constexpr uint32_t kLimit = SPAN ? 64 : 0x7fffffffu;
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  const uint32_t t0 = wait_clock<SPAN>();
  do {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  } while (!__any_sync(0xffffffffu, *fail != 0 || wait_clock<SPAN>() - t0 > kLimit));
  *fail = 1;
  return false;
}

// Pairs of 32-bit values and their operations, one instruction a pair.  Volatile like all of the
// softmax's arithmetic: exp_half says why.
struct Pair {
  uint64_t b;
};
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.b) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(Pair p, float &x, float &y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.b));
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.b) : "l"(a.b), "l"(b.b), "l"(c.b));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r.b) : "l"(a.b), "l"(b.b));
  return r;
}
__device__ __forceinline__ float exp2_mufu(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Three-input maximum that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm volatile("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_v(float a, float b) {
  float r;
  asm volatile("max.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// r's bits + (t << 23): a value of exponent 0 times 2^t, t in the low bits of a float.
__device__ __forceinline__ float scale_by(float r, float t) {
  int32_t y;
  asm volatile("mad.lo.s32 %0, %1, 8388608, %2;"
               : "=r"(y)
               : "r"(__float_as_int(t)), "r"(__float_as_int(r)));
  return __int_as_float(y);
}
template <typename T>
__device__ __forceinline__ uint32_t pack_v(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

// P of 8 G keys: w = pairs of 16-bit 2^(v scale + sub), their sums added to `sum`.  With MAX the
// maxima of v and of `more` (8 G values each) go to mx; more_ready waits for `more`, halfway.
//
// A warp issues in order, and the MUFU unit takes one of its exponentials every 8 cycles: the other
// instructions have to stand between those for the unit not to idle.  So by groups of 4 pairs (6
// exponentials; the next group's arguments, the sums and roundings of the one before, maxima), an
// order that volatile operations keep.  One pair of four is done on the FMA and integer pipes:
// 2^x with x = n + f, n from adding 1.5 2^23, 2^f on [-1/2, 1/2] as a polynomial of degree 4 with
// 2^0 exactly 1 (fitted for the least largest relative error, 3e-6, where f16 rounds to 2^-12), n
// added to its exponent.  Arguments below -127 give 0; those up to 127 are exact in n.
template <typename T, int G, bool MAX, typename Ready>
__device__ __forceinline__ void exp_half(const float *v, const float *more, uint32_t *w, Pair *sum,
                                         Pair scale, Pair sub, float *mx, Ready more_ready) {
  constexpr float kMagic = 12582912.f;
  const Pair magic = pair(kMagic, kMagic), unmagic = pair(-kMagic, -kMagic);
  const Pair minus = pair(-1.f, -1.f), one = pair(1.f, 1.f);
  const Pair c4 = pair(0x1.39f3a6p-7f, 0x1.39f3a6p-7f), c3 = pair(0x1.c9fb52p-5f, 0x1.c9fb52p-5f);
  const Pair c2 = pair(0x1.ec03b6p-3f, 0x1.ec03b6p-3f), c1 = pair(0x1.62e132p-1f, 0x1.62e132p-1f);
  Pair x[4];
  float e[2][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fma2(pair(v[2 * i], v[2 * i + 1]), scale, sub);
#pragma unroll
  for (int g = 0; g <= G; ++g) {
    float *E = e[g & 1], *D = e[(g & 1) ^ 1];  // this group's results, and the last one's
    const bool cur = g < G, next = g + 1 < G, prev = g > 0;
    if (MAX && g == G / 2) more_ready();
    Pair y[4], t, n, f, r;
    float a, b, x0, x1;
    // maxima: those of v in the first half of the groups, those of `more` in the second
    auto max_at = [&](int k) {
      if (!MAX || !cur) return;
      const int i = (g % (G / 2)) * 16 + 2 * k;
      const float *z = g < G / 2 ? v : more;
      mx[k & 3] = max3_nan(mx[k & 3], z[i], z[i + 1]);
    };
    auto arg = [&](int i) {
      if (next)
        y[i] = fma2(pair(v[8 * (g + 1) + 2 * i], v[8 * (g + 1) + 2 * i + 1]), scale, sub);
    };
    auto add = [&](int i) {
      if (prev) sum[i & 1] = add2(sum[i & 1], pair(D[2 * i], D[2 * i + 1]));
    };
    auto cvt = [&](int i) {
      if (prev) w[4 * (g - 1) + i] = pack_v<T>(D[2 * i], D[2 * i + 1]);
    };
    auto mufu = [&](int i) {
      if (!cur) return;
      unpair(x[i / 2], x0, x1);
      E[i] = exp2_mufu(i & 1 ? x1 : x0);
    };
    mufu(0);
    if (cur) {
      unpair(x[3], a, b);
      a = max_v(a, -127.f);
    }
    max_at(0);
    arg(0);
    add(0);
    mufu(1);
    if (cur) b = max_v(b, -127.f);
    max_at(1);
    cvt(0);
    if (cur) t = add2(pair(a, b), magic);
    mufu(2);
    max_at(2);
    arg(1);
    add(1);
    if (cur) n = add2(t, unmagic);
    max_at(3);
    cvt(1);
    mufu(3);
    if (cur) f = fma2(n, minus, pair(a, b));
    max_at(4);
    arg(2);
    add(2);
    if (cur) r = fma2(f, c4, c3);
    mufu(4);
    max_at(5);
    cvt(2);
    if (cur) r = fma2(r, f, c2);
    max_at(6);
    arg(3);
    add(3);
    mufu(5);
    if (cur) r = fma2(r, f, c1);
    max_at(7);
    cvt(3);
    if (cur) {
      r = fma2(r, f, one);
      float r0, r1, t0, t1;
      unpair(t, t0, t1);
      unpair(r, r0, r1);
      E[6] = scale_by(r0, t0);
      E[7] = scale_by(r1, t1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = y[i];
  }
}

struct Seq {
  int q0, nq, k0, nk;
};
// A sequence's rows; *bad set where its starts are no ascending part of the rows.
__device__ __forceinline__ Seq load_seq(const PromptAttnArgs &a, int b, bool *bad) {
  const int q0 = a.q_start[b], q1 = a.q_start[b + 1], k0 = a.k_start[b], k1 = a.k_start[b + 1];
  Seq s = {q0, q1 - q0, k0, k1 - k0};
  *bad = q0 < 0 || q1 < q0 || q1 > a.num_q_tokens || k0 < 0 || k1 < k0 || k1 > a.num_k_tokens;
  return s;
}

// A work item: the rows of one CTA, row = (token - tok0) * G + head in the group - in0.
struct Item {
  int rows;     // 1 to tile_rows NT; -1: no more items
  int h;        // kv head
  int tok0;     // token of the first row, within its sequence
  int in0;      // head in the group of the first row
  int q0;       // row of q and out that tok0 is
  int k0, nk;   // the sequence's keys
  int past;     // keys in front of its first query
  int keys[2];  // keys that each tile looks at: those that its last row sees
  int log_keys;  // the item's keys (all parts) are fewer than 2^log_keys
  int parts;    // of the item's keys, merged by the last to finish; 1: the output itself
  int part;     // k0, nk, past and keys are from this part's first key on
  int id;       // of the item, where it has parts
};
constexpr int kMinSteps = 4;  // of a part
constexpr int kMaxParts = 16;
// Work item `i` of the list (sequences, of every 32 the longest first; kv heads; row tiles from the
// last, which sees the most keys, to the first: the short items fill the end); rows = -1 past the
// list's end, and *total then its length.  One warp: lane l looks at sequence 32 n + l.  (In the
// order of the sequences 32 tokens over pasts of up to 4095 keys took 92 us, longest first 73.)
// The list ends at the first 32 that hold malformed starts: it is then no longer than the launch
// assumed, whatever the starts are.
template <int NT>
__device__ __forceinline__ Item find_item(const PromptAttnArgs &a, int tile_rows, int64_t i,
                                          int64_t *total) {
  const int lane = threadIdx.x & 31, G = a.group, ROWS = NT * tile_rows;
  const int64_t asked = i;
  bool bad = false;
  Item it;
  it.rows = -1;
  for (int b0 = 0; b0 < a.batch && it.rows < 0; b0 += 32) {
    const int b = b0 + lane;
    Seq s = {0, 0, 0, 0};
    if (b < a.batch) s = load_seq(a, b, &bad);
    if (__any_sync(0xffffffffu, bad)) break;
    if (a.batch > 1) {  // lane l takes the l-th longest of the 32
      int rank = 0, from = 0;
      for (int o = 0; o < 32; ++o) {
        const int nk = __shfl_sync(0xffffffffu, s.nk, o);
        rank += nk > s.nk || (nk == s.nk && o < lane);
      }
      for (int o = 0; o < 32; ++o)
        if (__shfl_sync(0xffffffffu, rank, o) == lane) from = o;
      s.q0 = __shfl_sync(0xffffffffu, s.q0, from);
      s.nq = __shfl_sync(0xffffffffu, s.nq, from);
      s.k0 = __shfl_sync(0xffffffffu, s.k0, from);
      s.nk = __shfl_sync(0xffffffffu, s.nk, from);
    }
    const int64_t nt = (int64_t(s.nq) * G + ROWS - 1) / ROWS;
    int64_t end = nt * a.kv_heads;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += o;
    }
    const uint32_t after = __ballot_sync(0xffffffffu, i < end);
    if (after) {
      const int l = __ffs(after) - 1;
      const int64_t n = __shfl_sync(0xffffffffu, nt, l);
      const int64_t rel = i - (__shfl_sync(0xffffffffu, end, l) - n * a.kv_heads);
      const int nq = __shfl_sync(0xffffffffu, s.nq, l);
      const int64_t rows = int64_t(nq) * G, row0 = (n - 1 - rel % n) * ROWS;
      it.h = int(rel / n);
      it.rows = int(min(int64_t(ROWS), rows - row0));
      it.tok0 = int(row0 / G);
      it.in0 = int(row0 % G);
      it.q0 = __shfl_sync(0xffffffffu, s.q0, l) + it.tok0;
      it.k0 = __shfl_sync(0xffffffffu, s.k0, l);
      it.nk = __shfl_sync(0xffffffffu, s.nk, l);
      it.past = it.nk - nq;
      for (int x = 0; x < 2; ++x) {
        const int last = min(tile_rows * (x + 1), it.rows) - 1;  // the tile's last row
        it.keys[x] = last < tile_rows * x ? 0
                     : a.causal
                         ? max(0, min(it.nk, it.tok0 + (it.in0 + last) / G + it.past + 1))
                         : it.nk;
      }
      it.log_keys = 32 - __clz(max(it.keys[0], it.keys[1]));
    } else {
      i -= __shfl_sync(0xffffffffu, end, 31);
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.diag, int32_t(kDiagBadLaunch));
  *total = asked - i;
  return it;
}

// Cut an item down to one of its parts: whole steps of keys; false where it has fewer parts.
template <int KEYS>
__device__ __forceinline__ bool take_part(Item *it, int part, int parts) {
  const int steps = (max(it->keys[0], it->keys[1]) + KEYS - 1) / KEYS;
  it->parts = max(1, min(parts, steps / kMinSteps));
  it->part = part;
  if (part >= it->parts) return false;
  const int lo = part * steps / it->parts * KEYS, n = (part + 1) * steps / it->parts * KEYS - lo;
  it->k0 += lo;
  it->nk -= lo;
  it->past -= lo;
  for (int x = 0; x < 2; ++x) it->keys[x] = max(0, min(it->keys[x] - lo, n));
  return true;
}

// The outputs of a row that sees infinities or NaN which the products did not (`sees` keys from the
// first hidden one).  Out of line: beside the loops its few instructions cost them 4 %.
template <typename T, int DP>
__device__ __noinline__ void patch_row(uint16_t *dst, const volatile uint16_t *patch, int sees,
                                       int head_dim) {
  __syncwarp();  // the row's other lanes have stored theirs
  if (!dst || sees <= 0) return;
  for (int c = 0; c < head_dim; ++c) {
    float y = widen<T>(__ldcg(reinterpret_cast<const unsigned short *>(dst) + c));
    if (patch[c] < sees) y = NAN;
    if (patch[DP + c] < sees) y += INFINITY;
    if (patch[2 * DP + c] < sees) y -= INFINITY;
    dst[c] = uint16_t(pack2<T>(y, 0.f));
  }
}

// PARTS: items are cut into P.parts.  A kernel of its own, since the merge's instructions beside
// the others cost calls without parts up to a third (the SM's instruction cache).
template <typename T, int DP, bool PARTS>
__global__ void __launch_bounds__(Shape<DP>::kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ Params P) {
  using S = Shape<DP>;
  constexpr int NT = S::NT, KEYS = S::kKeys, H = KEYS / 2;
  const PromptAttnArgs &a = P.a;
  extern __shared__ __align__(1024) unsigned char smem[];  // the swizzle goes by 1024 bytes
  const uint32_t sb = ptx::smem_u32(smem);
  if (sb & 1023u) {
    if (threadIdx.x == 0) atomicOr(a.diag, int32_t(kDiagBadLaunch));
    return;
  }
  Item *s_items = reinterpret_cast<Item *>(smem + S::kOffMisc);
  // by item parity: V held values that some rows must not see (see the checking warp)
  volatile int *s_patched = reinterpret_cast<volatile int *>(s_items + kItemSlots);
  int *s_fail = const_cast<int *>(s_patched) + 2;
  static_assert(kItemSlots * sizeof(Item) + 12 <= S::kMisc, "space");
  // first such key of each column, from the first key that a row does not see: NaN, inf, -inf
  volatile uint16_t *s_patch = reinterpret_cast<volatile uint16_t *>(smem + S::kOffPatch);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kMmaWarp = S::kSoftmaxWarps, kTmaWarp = kMmaWarp + 1, kQWarp = kMmaWarp + 2,
                kCheckWarp = kMmaWarp + 3;
  auto bar = [&](int i) { return sb + S::kOffBar + uint32_t(i) * 8; };

  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (warp == kTmaWarp) {
    if (lane == 0) {
      ptx::prefetch_tensormap(&P.tmk);
      ptx::prefetch_tensormap(&P.tmv);
      *s_fail = 0;
      ptx::mbar_init(bar(S::kQFull), 1);
      if (P.q_boxes) ptx::prefetch_tensormap(&P.tmq);
      ptx::mbar_init(bar(S::kQFree), 1);
      ptx::mbar_init(bar(S::kWant), 1);
      for (int i = 0; i < S::kSlots; ++i) {
        ptx::mbar_init(bar(S::kKvFull + i), 1);
        ptx::mbar_init(bar(S::kKvEmpty + i), 1);
        ptx::mbar_init(bar(S::kRaw + i), 1);
      }
      for (int i = 0; i < 2; ++i) {  // even and odd items: either side may be an item ahead
        ptx::mbar_init(bar(S::kChecked + i), 1);
        ptx::mbar_init(bar(S::kRead + i), S::kSoftmaxWarps);
      }
      ptx::mbar_init(bar(S::kDrain), 1);
      for (int i = 0; i < NT * S::kBufs; ++i) ptx::mbar_init(bar(S::kSFull + i), 1);
      for (int x = 0; x < NT; ++x) {
        ptx::mbar_init(bar(S::kSFree + x), 128);
        ptx::mbar_init(bar(S::kPFull + 2 * x), 128);
        ptx::mbar_init(bar(S::kPFull + 2 * x + 1), 128);
        ptx::mbar_init(bar(S::kODone + 2 * x), 1);
        ptx::mbar_init(bar(S::kODone + 2 * x + 1), 1);
      }
      for (int i = 0; i < kItemSlots; ++i) {
        ptx::mbar_init(bar(S::kItemFull + i), 1);
        ptx::mbar_init(bar(S::kItemEmpty + i), S::kSoftmaxWarps + 3);
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
  volatile int *fail = s_fail;

  // The CTA's k-th item, from the warp that hands them out; without rows it ends the role.
  auto next_item = [&](int k) {
    Item it;
    it.rows = -1;
    const int slot = k % kItemSlots;
    if (!wait<true>(bar(S::kItemFull + slot), uint32_t((k / kItemSlots) & 1), fail)) return it;
    it = s_items[slot];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(S::kItemEmpty + slot));
    return it;
  };
  // Row of an item, counted from its first token's first head -> token; below 2^16.
  auto token_of = [&](uint32_t at) {
    return P.group_magic ? __umulhi(at, P.group_magic) : at;
  };
  auto steps_of = [&](int keys) { return (keys + KEYS - 1) / KEYS; };
  // K and V tiles pass through the slots in the order in which the products need them:
  // K0 V0 K1 V1 .., or K0 K1 V0 K2 V1 .. where QK runs ahead.
  auto pos_k = [&](int j) { return S::kAhead ? (j == 0 ? 0 : 2 * j - 1) : 2 * j; };
  auto pos_v = [&](int j, int n) { return S::kAhead ? min(2 * j + 2, 2 * n - 1) : 2 * j + 1; };

  // Keys of an item from this one on are hidden from its first row, at least.
  auto hidden_from = [&](const Item &it) {
    return a.causal ? max(0, it.tok0 + it.past + 1) : it.nk;
  };
  // Whether V's tile j holds such keys, or rows past the sequence that a product reads: then it
  // goes through the checking warp.
  auto to_check = [&](const Item &it, int j) {
    const int end = (j + 1) * KEYS;
    return hidden_from(it) < min(end, it.nk) || (it.nk < end && it.nk % 16 != 0);
  };

  if (warp >= S::kSoftmaxWarps) {
  if constexpr (S::kSplitRegs)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegs));
  if (warp == kQWarp) {
    // ---------------- Q, and the items ----------------
    // The next item of the list.  Every CTA asks once past the end, and the last to do so leaves
    // the counter at zero.
    auto take = [&](bool *whole) {
      int32_t i = 0;
      if (lane == 0) i = atomicAdd(P.next_item, 1);
      i = __shfl_sync(0xffffffffu, i, 0);
      int64_t total = 0;
      const int parts = PARTS ? P.parts : 1;
      Item it = find_item<NT>(a, P.tile_rows, i / parts, &total);
      if (it.rows < 0 && lane == 0 && i == total * parts + int64_t(gridDim.x) - 1)
        atomicExch(P.next_item, 0);
      it.id = i / parts;
      it.parts = 1;
      *whole = !PARTS || it.rows < 0 || take_part<KEYS>(&it, i % parts, parts);
      return it;
    };
    // Parts that an item does not have are passed over.
    auto take_next = [&] {
      Item it;
      bool whole = false;
      while (!whole) it = take(&whole);
      return it;
    };
    bool ended = false;
    int q_begun = 0;  // items whose Q is copied as boxes
    for (int k = 0;; ++k) {
      const int slot = k % kItemSlots;
      if (k >= kItemSlots &&
          !wait(bar(S::kItemEmpty + slot), uint32_t((k / kItemSlots - 1) & 1), fail))
        break;
      // Taken when all copies of the last one have begun, not before: an SM with a long item leaves
      // the next to others (32 single tokens over pasts of up to 4095 keys: 77 us -> 61).  Up to four
      // steps earlier measures the same.
      if (k > 0 && !wait<true>(bar(S::kWant), uint32_t((k - 1) & 1), fail)) break;
      const Item it = take_next();
      ended = it.rows < 0;
      if (lane == 0) {
        s_items[slot] = it;
        ptx::mbar_arrive(bar(S::kItemFull + slot));
      }
      __syncwarp();
      if (it.rows < 0) break;
      if (k > 0 && !wait(bar(S::kQFree), uint32_t((k - 1) & 1), fail)) break;
      const int G = a.group;
      if (P.q_boxes) {
        // rows past the sequence are the next one's: their results are not stored
        if (lane == 0) {
          const int tiles = NT == 2 && it.rows > P.tile_rows ? 2 : 1;
          ptx::mbar_arrive_expect_tx(bar(S::kQFull),
                                     uint32_t(tiles * S::kBlocks * P.tile_rows) * 128);
          for (int x = 0; x < tiles; ++x) {
#pragma unroll
            for (int c = 0; c < S::kBlocks; ++c)
              ptx::tma_load_3d(sb + uint32_t(x) * S::kTileQ + c * kQBlk, &P.tmq, c * 64, it.h * G,
                               it.q0 + x * (128 / G), bar(S::kQFull));
          }
        }
        __syncwarp();
        q_begun = k + 1;
        continue;
      }
      // 16 bytes a lane; rows and values past the end are zeros
      constexpr int kChunks = DP / 8;
      const uint16_t *base = static_cast<const uint16_t *>(a.q) + int64_t(it.q0) * a.q_stride_token +
                             int64_t(it.h) * G * a.q_stride_head;
#pragma unroll 4
      for (int i = lane; i < NT * 128 * kChunks; i += 32) {
        const int r = i / kChunks, c = i % kChunks;
        const bool in = r < it.rows && c * 8 < a.head_dim;
        const uint32_t at = uint32_t(it.in0 + r), tok = token_of(at);
        const uint16_t *src = base + int64_t(tok) * a.q_stride_token +
                              int64_t(at - tok * G) * a.q_stride_head + c * 8;
        const uint32_t dst = sb + uint32_t(r >> 7) * S::kTileQ + uint32_t(c >> 3) * kQBlk +
                             uint32_t(r & 127) * 128 + uint32_t(((c & 7) ^ (r & 7)) * 16);
        ptx::cp_async16(dst, in ? src : static_cast<const uint16_t *>(a.q), in ? 16u : 0u);
      }
      ptx::cp_async_commit();
      ptx::cp_async_wait<0>();
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(S::kQFull));
    }
    if (*fail && q_begun)  // no copy may land after the CTA has gone
      ptx::mbar_wait_bounded(bar(S::kQFull), uint32_t((q_begun - 1) & 1), kWaitNs);
    while (!ended) ended = take_next().rows < 0;  // after a failure: the counter has to end at zero
  } else if (warp == kTmaWarp) {
    // ---------------- K and V ----------------
    int pos = 0;                   // tiles of the items before
    int begun = 0;                 // tiles whose copies have begun
    uint32_t raw_phase = 0, raw = 0;  // by slot: parity of its next unchecked tile; it holds one
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const Item it = next_item(k);
      if (it.rows < 0) break;
      const int n = steps_of(max(it.keys[0], it.keys[1]));
      auto slot_of = [&](int p) { return (pos + p) % S::kSlots; };
      auto free_slot = [&](int p) {
        const int q = pos + p;
        return q < S::kSlots ||
               wait(bar(S::kKvEmpty + q % S::kSlots), uint32_t((q / S::kSlots - 1) & 1), fail);
      };
      auto load = [&](const CUtensorMap *map, int p, int j, bool check) {
        if (!free_slot(p)) return false;
        const int slot = slot_of(p);
        if (lane == 0) {
          const uint32_t dst = sb + S::kOffKv + uint32_t(slot) * S::kTileKv;
          const uint32_t full = bar((check ? S::kRaw : S::kKvFull) + slot);
          ptx::mbar_arrive_expect_tx(full, S::kTileKv);
#pragma unroll
          for (int c = 0; c < S::kBlocks; ++c)
            ptx::tma_load_3d(dst + c * S::kKvBlk, map, c * 64, it.h, it.k0 + j * KEYS, full);
        }
        __syncwarp();
        begun = pos + p + 1;
        raw = check ? raw | 1u << slot : raw & ~(1u << slot);
        if (check) raw_phase ^= 1u << slot;
        return true;
      };
      auto load_k = [&](int j) { return load(&P.tmk, pos_k(j), j, false); };
      auto load_v = [&](int j) { return load(&P.tmv, pos_v(j, n), j, to_check(it, j)); };
      if (S::kAhead && n > 0) ok = load_k(0);
      for (int j = 0; ok && j < n; ++j) {
        if (S::kAhead) {
          ok = (j + 1 >= n || load_k(j + 1)) && load_v(j);
        } else {
          ok = load_k(j) && load_v(j);
        }
      }
      if (lane == 0) ptx::mbar_arrive(bar(S::kWant));
      __syncwarp();
      pos += 2 * n;
    }
    if (*fail) {  // no copy may land after the CTA has gone
      for (int q = max(0, begun - S::kSlots); q < begun; ++q) {
        const int slot = q % S::kSlots;
        if (raw >> slot & 1) {
          ptx::mbar_wait_bounded(bar(S::kRaw + slot), raw_phase >> slot & 1 ^ 1, kWaitNs);
        } else {
          ptx::mbar_wait_bounded(bar(S::kKvFull + slot), uint32_t((q / S::kSlots) & 1), kWaitNs);
        }
      }
    }
  } else if (warp == kCheckWarp) {
    // ---------------- V's tiles at the causal border ----------------
    // A product multiplies a key that a row does not see by P = 0, which an infinity or NaN in V
    // turns into NaN.  So where some row of the item does not see a key, the tile is looked
    // through before the products read it; what is not finite there becomes 0 and is noted by
    // column, and the rows that do see it get their infinity or NaN at the end.  Rows past the
    // sequence that a product reads (its last 16 keys) are another's, or nothing, and are cleared.
    constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
    int pos = 0;
    uint32_t raw_phase = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const Item it = next_item(k);
      if (it.rows < 0) break;
      const int n = steps_of(max(it.keys[0], it.keys[1])), hidden = hidden_from(it);
      // the flag of the item before last has been read
      if (k >= 2) ok = wait(bar(S::kRead + (k & 1)), uint32_t((k / 2 - 1) & 1), fail);
      if (!ok) break;
      if (lane == 0) s_patched[k & 1] = 0;
      __syncwarp();
      bool dirty = false;
      for (int j = 0; ok && j < n; ++j) {
        if (!to_check(it, j)) continue;
        const int slot = (pos + pos_v(j, n)) % S::kSlots;
        ok = wait<true>(bar(S::kRaw + slot), raw_phase >> slot & 1, fail);
        raw_phase ^= 1u << slot;
        if (!ok) break;
        const uint32_t tile = sb + S::kOffKv + uint32_t(slot) * S::kTileKv;
        // rows that a product reads (whole 16s of the keys that the item sees), and of these the
        // sequence's own
        const int seen = max(it.keys[0], it.keys[1]) - j * KEYS;
        const int end = min(KEYS, (seen + 15) / 16 * 16), live = min(end, it.nk - j * KEYS);
        const int from = max(0, hidden - j * KEYS);
        const auto at = [&](int row, int chunk) {  // 16 bytes of 8 columns
          return tile + (chunk >> 3) * S::kKvBlk + row * 128 + (((chunk & 7) ^ (row & 7)) * 16);
        };
        // kLanes lanes a row
        constexpr int kChunks = DP / 8, kLanes = kChunks > 16 ? 32 : kChunks;
        const int chunk = lane % kLanes, first_row = lane / kLanes;
        uint32_t odd = 0;
        if (chunk < kChunks) {
          for (int row = live + first_row; row < end; row += 32 / kLanes)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at(row, chunk)), "r"(0)
                         : "memory");
#pragma unroll 8
          for (int row = from + first_row; row < live; row += 32 / kLanes) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(at(row, chunk)));
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= (w[e] & kExp) + kOne;
          }
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, odd & 0x80008000u)) {
          if (!dirty) {
            // the notes of the item before have been read
            if (k > 0) ok = wait(bar(S::kRead + ((k - 1) & 1)), uint32_t((k - 1) / 2 & 1), fail);
            if (!ok) break;
            for (int i = lane; i < 3 * DP; i += 32) s_patch[i] = 0xffffu;
            if (lane == 0) s_patched[k & 1] = 1;
            __syncwarp();
            dirty = true;
          }
          // a lane has 8 columns to itself
          for (int row = from; row < live && lane < kChunks; ++row) {
            uint16_t h[8];
            uint4 *p = reinterpret_cast<uint4 *>(smem + (at(row, lane) - sb));
            *reinterpret_cast<uint4 *>(h) = *p;
            for (int e = 0; e < 8; ++e) {
              if ((h[e] & (kExp & 0xffffu)) != (kExp & 0xffffu)) continue;
              const int kind = (h[e] & 0x7fffu) > (kExp & 0xffffu) ? 0 : h[e] & 0x8000u ? 2 : 1;
              volatile uint16_t *first = s_patch + kind * DP + lane * 8 + e;
              if (*first == 0xffffu) *first = uint16_t(j * KEYS + row - hidden);
              h[e] = 0;
            }
            *p = *reinterpret_cast<uint4 *>(h);
          }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(S::kKvFull + slot));
        __syncwarp();
      }
      if (!ok) break;
      if (lane == 0) ptx::mbar_arrive(bar(S::kChecked + (k & 1)));
      __syncwarp();
      pos += 2 * n;
    }
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issue ----------------
    // Warp-uniform in the compiler's eyes too: see mma_ss_warp.
    const uint32_t base = __shfl_sync(0xffffffffu, sb, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    constexpr uint32_t kHi = tc::kDescHigh;
    int pos = 0, step[NT] = {};  // of the items before
    int issued = 0;              // items whose last commit is issued
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const Item it = next_item(k);
      if (it.rows < 0) break;
      int keys[NT], n[NT], n_max = 0;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        keys[x] = __shfl_sync(0xffffffffu, it.keys[x], 0);
        n[x] = steps_of(keys[x]);
        n_max = max(n_max, n[x]);
      }
      auto n_of = [&](int x) { return NT == 2 && x == 1 ? n[NT - 1] : n[0]; };
      auto keys_of = [&](int x) { return NT == 2 && x == 1 ? keys[NT - 1] : keys[0]; };
      auto step_of = [&](int x) { return NT == 2 && x == 1 ? step[NT - 1] : step[0]; };
      // Slot of a tile, once it is there.
      auto tile_at = [&](int p, uint32_t *at) {
        const int q = pos + p;
        *at = base + S::kOffKv + uint32_t(q % S::kSlots) * S::kTileKv;
        return wait(bar(S::kKvFull + q % S::kSlots), uint32_t((q / S::kSlots) & 1), fail);
      };
      auto release = [&](int p) { tc::commit_warp(bar(S::kKvEmpty + (pos + p) % S::kSlots)); };
      auto issue_qk = [&](int x, int j, uint32_t at) {
        const int g = step_of(x) + j;
        const uint32_t qa = tc::desc_low(base + uint32_t(x) * S::kTileQ, 16);
        const uint32_t ka = tc::desc_low(at, 16);
        const uint32_t tS = tm + S::kS + uint32_t(x * S::kBufs + g % S::kBufs) * KEYS;
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
          tc::mma_ss_warp(tS, qa + ((c >> 2) * kQBlk + (c & 3) * 32) / 16,
                          ka + ((c >> 2) * S::kKvBlk + (c & 3) * 32) / 16, kHi, P.idesc_qk, c > 0);
        tc::commit_warp(bar(S::kSFull + x * S::kBufs + g % S::kBufs));
      };
      // P.V of one half of a step's keys: the 16-key products that hold a key.
      auto issue_pv = [&](int x, int j, int half, uint32_t at) {
        const int g = step_of(x) + j;
        const uint32_t va = tc::desc_low(at, S::kKvBlk);
        const uint32_t tP = tm + (S::kScores == Scores::kSeparate
                                      ? S::kP + uint32_t(x) * (KEYS / 2)
                                      : S::kS + uint32_t(x * S::kBufs + g % S::kBufs) * KEYS);
        const uint32_t tO = tm + S::kO + uint32_t(x) * DP;
        const int live = keys_of(x) - j * KEYS;
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < KEYS / 32; ++c) {
          const int i = half * (KEYS / 32) + c;
          if (i * 16 < live)
            tc::mma_ts_warp(tO, tP + i * 8, va + i * 2048 / 16, kHi, P.idesc_pv, j > 0 || i > 0);
        }
      };
      ok = wait(bar(S::kQFull), uint32_t(k & 1), fail);
      uint32_t at_k = 0, at_v = 0;
      if (ok && n_max > 0) {
        ok = tile_at(pos_k(0), &at_k);
        if (!ok) break;
#pragma unroll 1
        for (int x = 0; x < NT; ++x)
          if (n_of(x) > 0) issue_qk(x, 0, at_k);
        release(pos_k(0));
      }
      for (int j = 0; ok && j < n_max; ++j) {
        const bool more = j + 1 < n_max;
        if (S::kAhead && more) {
          ok = tile_at(pos_k(j + 1), &at_k);
#pragma unroll 1
          for (int x = 0; x < NT; ++x) {
            if (!ok || j + 1 >= n_of(x)) continue;
            // the scores of step j (two buffers: P of step j - 1) have left their columns
            if (S::kScores == Scores::kSeparate)
              ok = wait(bar(S::kSFree + x), uint32_t((step_of(x) + j) & 1), fail);
            if (ok) issue_qk(x, j + 1, at_k);
          }
          if (!ok) break;
          release(pos_k(j + 1));
        }
        ok = tile_at(pos_v(j, n_max), &at_v);
        if (ok && !S::kAhead && more) ok = tile_at(pos_k(j + 1), &at_k);
#pragma unroll 1
        for (int x = 0; x < NT; ++x) {
          if (!ok || j >= n_of(x)) continue;
          const uint32_t ph = uint32_t((step_of(x) + j) & 1);
#pragma unroll
          for (int half = 0; ok && half < 2; ++half) {
            ok = wait(bar(S::kPFull + 2 * x + half), ph, fail);
            if (!ok) break;
            issue_pv(x, j, half, at_v);
          }
          if (!ok) continue;
          tc::commit_warp(bar(S::kODone + 2 * x + ((step_of(x) + j) & 1)));
          if (!S::kAhead && j + 1 < n_of(x)) issue_qk(x, j + 1, at_k);
        }
        if (!ok) break;
        release(pos_v(j, n_max));
        if (!S::kAhead && more) release(pos_k(j + 1));
      }
      tc::commit_warp(bar(S::kQFree));
      issued = k + 1;
      pos += 2 * n_max;
#pragma unroll
      for (int x = 0; x < NT; ++x) step[x] += n[x];
    }
    // No product may run on, and no arrival of a commit land, after the CTA has gone: the last
    // commits come after those that the softmax waits for.
    if (*fail) {
      tc::commit_warp(bar(S::kDrain));
      ptx::mbar_wait_bounded(bar(S::kDrain), 0, kWaitNs);
    } else if (issued > 0) {
      ptx::mbar_wait_bounded(bar(S::kQFree), uint32_t((issued - 1) & 1), kWaitNs);
    }
  }
  } else {
    // ---------------- softmax: thread = row of tile x ----------------
    if constexpr (S::kSplitRegs)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
    const int x = warp >> 2, q4 = warp & 3;
    const uint32_t lanes = uint32_t(q4 * 32) << 16;
    const uint32_t tO = tmem + S::kO + uint32_t(x) * DP + lanes;
    int step = 0;  // of the items before
    bool ok = true;
    // An output whose row sees infinities or NaN that the products did not.
    auto patch_of = [&](float y, int col, int sees) {
      const volatile uint16_t *first = s_patch + col;
      if (first[0] < sees) y = NAN;
      if (first[DP] < sees) y += INFINITY;
      if (first[2 * DP] < sees) y -= INFINITY;
      return y;
    };
    // The first `last` + 1 of 32 columns, as bits: they become predicates several at a time, where
    // a comparison a column took 2 % of a call of short prompts.
    auto seen_of = [](int last) {
      return last < 0 ? 0u : last > 30 ? ~0u : (2u << last) - 1;
    };
    auto o_done = [&](int g) {
      return wait(bar(S::kODone + 2 * x + (g & 1)), uint32_t((g >> 1) & 1), fail);
    };
    for (int k = 0; ok; ++k) {
      const Item it = next_item(k);
      if (it.rows < 0) break;
      const int warp_row = P.tile_rows * x + q4 * 32, r = warp_row + lane;
      const int rows_end = min(it.rows, P.tile_rows * (x + 1));  // of the tile
      // last key that the row sees; rows past the end go as far as the last one
      const int tok = int(token_of(uint32_t(it.in0 + min(r, rows_end - 1))));
      const int lim = a.causal ? it.tok0 + tok + it.past : it.nk - 1;
      const int lim0 = __shfl_sync(0xffffffffu, lim, 0);
      const int n = steps_of(x == 0 ? it.keys[0] : it.keys[1]);
      float m = -INFINITY, l = 0.f;
      const float shift = std::is_same<T, __half>::value ? kShiftF16 : -kRaise - float(it.log_keys);
      for (int j = 0; ok && j < n; ++j) {
        const int g = step + j, buf = g % S::kBufs;
        const uint32_t tS = tmem + S::kS + uint32_t(x * S::kBufs + buf) * KEYS + lanes;
        const uint32_t tP =
            S::kScores == Scores::kSeparate ? tmem + S::kP + uint32_t(x) * (KEYS / 2) + lanes : tS;
        ok = wait(bar(S::kSFull + x * S::kBufs + buf), uint32_t((g / S::kBufs) & 1), fail);
        if (!ok) break;
        tc::fence_after_sync();
        const int k0 = j * KEYS;
        const bool masked = k0 + KEYS - 1 > lim0;
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto row_max = [&] {
          return max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * P.scale_log2;
        };
        if (j == 0) {
#pragma unroll 1
          for (int c0 = 0; c0 < KEYS; c0 += 32) {
            float u[32];
            tc::ld32(tS + c0, u);
            tc::wait_ld();
            const uint32_t seen = seen_of(lim - k0 - c0);
#pragma unroll
            for (int c = 0; c < 32; c += 2)
              mx[c / 2 & 3] = max3_nan(mx[c / 2 & 3], seen >> c & 1 ? u[c] : -INFINITY,
                                       seen >> (c + 1) & 1 ? u[c + 1] : -INFINITY);
          }
          const float top = row_max();
          m = top == -INFINITY ? top : top + (top - top);  // NaN where it is infinite
        }
        // The first half's exponentials run on the maximum so far while the step's own is found;
        // where that exceeds it (seldom) they run again.
        float v[KEYS];
        uint32_t w[KEYS / 4];
        Pair sum[2];
        float sub;
        auto settle_half = [&](int half) {
          tc::wait_ld();
          if (masked) {
#pragma unroll
            for (int c0 = half * H; c0 < half * H + H; c0 += 32) {
              const uint32_t seen = seen_of(lim - k0 - c0);
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c0 + c] = seen >> c & 1 ? v[c0 + c] : -INFINITY;
            }
          }
        };
        for (bool again = false;;) {
#pragma unroll
          for (int c = 0; c < KEYS; c += 32) tc::ld32(tS + c, v + c);
          settle_half(0);
          sub = m == -INFINITY ? 0.f : shift - m;  // nothing seen yet: P is 0
          sum[0] = sum[1] = pair(0.f, 0.f);
          exp_half<T, KEYS / 16, true>(v, v + H, w, sum, pair(P.scale_log2, P.scale_log2),
                                       pair(sub, sub), mx, [&] { settle_half(1); });
          const float top = row_max();
          // a NaN or infinite maximum makes the row NaN, as its softmax is (what stands in rows
          // past the tile's is nobody's)
          const bool raise = !(top <= m + kRaise) && r < rows_end;
          if (S::kAhead && j > 0 && !again)  // P.V of the step before has added to O and read P
            ok = o_done(g - 1);
          if (!ok || j == 0 || again || !__any_sync(0xffffffffu, raise)) break;
          again = true;
          float f = 1.f;
          if (raise) {
            f = ptx::fast_exp2(m - top);  // 0 before the first key
            m = top + (top - top);
            l *= f;
          }
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            float o[32];
            tc::ld32(tO + c, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tc::st32(tO + c, o);
          }
          tc::wait_st();
        }
        if (!ok) break;
        if constexpr (S::kScores == Scores::kSeparate) {
          tc::fence_before_sync();
          ptx::mbar_arrive(bar(S::kSFree + x));
        }
        auto store_half = [&](int half) {
          if constexpr (H == 64) {
            tc::st32u(tP + half * 32, w);
          } else {
            tc::st16u(tP + half * 16, w);
          }
          tc::wait_st();
          tc::fence_before_sync();
          ptx::mbar_arrive(bar(S::kPFull + 2 * x + half));
        };
        store_half(0);
        exp_half<T, KEYS / 16, false>(v + H, v, w, sum, pair(P.scale_log2, P.scale_log2),
                                      pair(sub, sub), mx, [] {});
        store_half(1);
        // In place: S(j) came after P.V(j-1), whose phase has to be passed before P.V(j+1)'s.
        if (!S::kAhead && j > 0) {
          ok = o_done(g - 1);
          if (!ok) break;
        }
        float s0, s1;
        unpair(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }
      if (ok && n > 0) ok = o_done(step + n - 1);
      if (ok) ok = wait<true>(bar(S::kChecked + (k & 1)), uint32_t((k / 2) & 1), fail);
      if (!ok) break;
      const bool patched = s_patched[k & 1];
      step += n;
      tc::fence_after_sync();
      // The output, 8 rows of 64 bytes a store: rows g + 8 i lie with the four lanes of g, which
      // trade 8-column groups so that each stores 16 bytes.  (A row a lane touches 32 lines a store:
      // 5000 cycles an item where this takes 3400.)
      const int g8 = lane >> 2, c4 = lane & 3;
      // Four words of each of a row's lanes (u[q]: columns 8 q + 2 c4, + 1) -> lane c4 stores the
      // words of columns 8 c4 ..: a 4 x 4 transposition in two exchanges.
      auto store_row = [&](uint16_t *dst, uint32_t *u, int c) {
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (q & d) continue;
            const bool up = c4 & d;
            const uint32_t give = up ? u[q] : u[q | d];
            const uint32_t got = __shfl_xor_sync(0xffffffffu, give, d);
            u[q] = up ? got : u[q];
            u[q | d] = up ? u[q | d] : got;
          }
        }
        if (dst && c + 8 * c4 < a.head_dim)
          *reinterpret_cast<uint4 *>(dst + c + 8 * c4) = make_uint4(u[0], u[1], u[2], u[3]);
      };
      auto out_of = [&](int rr) {  // null past the tile
        const uint32_t at = uint32_t(it.in0 + rr), t = token_of(at);
        return rr < rows_end
                   ? static_cast<uint16_t *>(a.out) + (int64_t(it.q0) + t) * a.out_stride_token +
                         int64_t(it.h * a.group + int(at - t * a.group)) * a.out_stride_head
                   : nullptr;
      };
      // keys that a row sees of those hidden from the item's first
      auto sees_of = [&](int rr) {
        return it.tok0 + int(token_of(uint32_t(it.in0 + rr))) + it.past + 1 - hidden_from(it);
      };
      const float sum = n == 0 ? 0.f : l;
      const bool split = PARTS && it.parts > 1;
#pragma unroll 1
      for (int i = 0; !split && i < 4 && warp_row + 8 * i < rows_end; i += 2) {
        float scale[2];
        uint16_t *dst[2];
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int from = g8 + 8 * (i + e);
          scale[e] = __shfl_sync(0xffffffffu, inv, from);  // 0: nothing seen
          dst[e] = out_of(warp_row + from);
        }
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float o[16];
          if (n > 0) {
            tc::ld16x256b_x4(tO + (uint32_t(i * 8) << 16) + c, o);
            tc::wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t u[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float y0 = o[4 * q + 2 * e] * scale[e], y1 = o[4 * q + 2 * e + 1] * scale[e];
              u[q] = scale[e] == 0.f ? 0u : pack2<T>(y0, y1);
            }
            store_row(dst[e], u, c);
          }
        }
      }
      if (patched && !split)
        patch_row<T, DP>(out_of(warp_row + lane), s_patch, sum == 0.f ? 0 : sees_of(warp_row + lane),
                         a.head_dim);
      if constexpr (PARTS) {
        // row of q * heads + head of a row of the CTA
        auto row_of = [&](int rr) {
          const uint32_t at = uint32_t(it.in0 + rr), t = token_of(at);
          return (int64_t(it.q0) + t) * (a.kv_heads * a.group) + it.h * a.group +
                 int(at - t * a.group);
        };
        const int64_t all_rows = int64_t(a.num_q_tokens) * a.kv_heads * a.group;
        if (split && warp_row < rows_end) {
          // the part's sums as they are
          if (warp_row + lane < rows_end)
            __stcg(P.part_ml + it.part * all_rows + row_of(warp_row + lane), make_float2(m, sum));
#pragma unroll 1
          for (int i = 0; n > 0 && i < 4 && warp_row + 8 * i < rows_end; i += 2) {
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              float o[16];
              tc::ld16x256b_x4(tO + (uint32_t(i * 8) << 16) + c, o);
              tc::wait_ld();
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int rr = warp_row + g8 + 8 * (i + e);
                if (rr >= rows_end) continue;
                float *y = P.part_o + (it.part * all_rows + row_of(rr)) * DP + c + 2 * c4;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  __stcg(reinterpret_cast<float2 *>(y + 8 * q),
                         make_float2(o[4 * q + 2 * e], o[4 * q + 2 * e + 1]));
              }
            }
          }
          if (patched && n > 0) {
            __syncwarp();
            const int rr = warp_row + lane, sees = rr < rows_end && sum != 0.f ? sees_of(rr) : 0;
            float *y = P.part_o + (it.part * all_rows + row_of(min(rr, rows_end - 1))) * DP;
#pragma unroll 1
            for (int c = 0; sees > 0 && c < a.head_dim; ++c) y[c] = patch_of(__ldcg(y + c), c, sees);
          }
          // the last warp to have these rows' sums of a part merges all of them
          __threadfence();
          __syncwarp();
          uint32_t before = 0;
          if (lane == 0) {
            unsigned long long *done = P.merged + it.id * S::kSoftmaxWarps + warp;
            atomicMax(done, P.ticket_base);
            before = uint32_t(atomicAdd(done, 1ull) - P.ticket_base);
          }
          before = __shfl_sync(0xffffffffu, before, 0);
          __threadfence();
          if (before == uint32_t(it.parts - 1)) {
#pragma unroll 1
            for (int i = 0; i < 4 && warp_row + 8 * i < rows_end; ++i) {
              const int rr = warp_row + g8 + 8 * i;
              const int64_t row = row_of(min(rr, rows_end - 1));
              // all loads of a step before the first is used
              float2 ml[kMaxParts];
#pragma unroll
              for (int p = 0; p < kMaxParts; ++p)
                ml[p] = p < it.parts ? __ldcg(P.part_ml + p * all_rows + row)
                                     : make_float2(-INFINITY, 0.f);
              float top = -INFINITY, all = 0.f;
#pragma unroll
              for (int p = 0; p < kMaxParts; ++p)
                if (ml[p].y != 0.f) top = max3_nan(top, ml[p].x, ml[p].x);
#pragma unroll
              for (int p = 0; p < kMaxParts; ++p) {
                ml[p].x = ml[p].y == 0.f ? 0.f : ptx::fast_exp2(ml[p].x - top);
                all += ml[p].x * ml[p].y;
              }
              const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
              for (int c = 0; c < DP; c += 32) {
                float2 o[4] = {};
                const float *y = P.part_o + row * DP + c + 2 * c4;
#pragma unroll
                for (int p0 = 0; p0 < kMaxParts; p0 += 4) {
                  if (p0 >= it.parts) break;
                  float2 v[4][4];
#pragma unroll
                  for (int p = 0; p < 4; ++p) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                      v[p][q] = ml[p0 + p].y == 0.f
                                    ? make_float2(0.f, 0.f)
                                    : __ldcg(reinterpret_cast<const float2 *>(
                                          y + (p0 + p) * all_rows * DP + 8 * q));
                  }
#pragma unroll
                  for (int p = 0; p < 4; ++p) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                      o[q].x += ml[p0 + p].x * v[p][q].x;
                      o[q].y += ml[p0 + p].x * v[p][q].y;
                    }
                  }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  o[q].x *= inv;
                  o[q].y *= inv;
                }
                uint32_t u[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) u[q] = pack2<T>(o[q].x, o[q].y);
                __syncwarp();
                store_row(out_of(rr), u, c);
              }
            }
          }
        }
      }
      tc::fence_before_sync();  // before the next item's first P says that O may be overwritten
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(S::kRead + (k & 1)));
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (*s_fail && tid == 0) atomicOr(a.diag, int32_t(kDiagWaitTimeout));
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
  p.q_boxes = a.q_map != nullptr;
  if (p.q_boxes) std::memcpy(&p.tmq, a.q_map, sizeof(CUtensorMap));
  p.tile_rows = p.q_boxes ? 128 / a.group * a.group : 128;
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  p.idesc_qk = tc::idesc_f16(bf16, 128, S::kKeys, false, false);
  p.idesc_pv = tc::idesc_f16(bf16, 128, DP, false, true);
  p.group_magic = a.group == 1 ? 0 : uint32_t(((uint64_t(1) << 32) + a.group - 1) / a.group);
  // every sequence has at most one partly filled tile a kv head
  const int64_t items =
      (int64_t(a.num_q_tokens) * a.group / (S::NT * p.tile_rows) + a.batch) * a.kv_heads;
  const int sms = device_sm_count();
  // Two SMs or more an item: its keys in parts, as many as run at once.
  p.parts = 1;
  if (a.num_k_tokens >= 2 * kMinSteps * S::kKeys)
    p.parts = int(std::max<int64_t>(1, std::min<int64_t>(kMaxParts, sms / items)));
  if (items * S::kSoftmaxWarps > kTickets) p.parts = 1;
  static_assert(kMaxParts < kTicketRange, "parts of an item are counted by a ticket");
  const int64_t rows = int64_t(a.num_q_tokens) * a.group * a.kv_heads;
  CallScratch scratch;
  cudaError_t e = scratch.acquire(stream, p.parts > 1 ? size_t(rows) * p.parts * (DP + 2) * 4 : 16);
  if (e != cudaSuccess && p.parts > 1) {  // no room for the parts' sums
    cudaGetLastError();
    p.parts = 1;
    e = scratch.acquire(stream, 16);
  }
  if (e != cudaSuccess) return e;
  auto fn = p.parts > 1 ? prompt_attn_kernel<T, DP, true> : prompt_attn_kernel<T, DP, false>;
  if (S::kSplitRegs) {
    // with fewer registers at launch than the split was made for, setmaxnreg.inc would wait
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, fn);
    if (e == cudaSuccess &&
        fa.numRegs * S::kThreads < 256 * S::kSoftmaxRegs + 128 * S::kOtherRegs)
      e = cudaErrorInvalidConfiguration;
  }
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem));
  p.next_item = scratch.counters + kZeroedCounters / 2 - 1;
  p.merged = scratch.tickets;
  p.ticket_base = scratch.ticket_base;
  p.part_o = static_cast<float *>(scratch.ptr);
  p.part_ml = reinterpret_cast<float2 *>(p.part_o + rows * p.parts * DP);
  const int ctas = int(std::min<int64_t>(items * p.parts, sms));
  if (e == cudaSuccess)
    e = launch_pdl(fn, dim3(uint32_t(ctas)), dim3(S::kThreads), S::kSmem, stream, p);
  const cudaError_t r = scratch.release(stream);
  return e != cudaSuccess ? e : r;
}

}  // namespace

int prompt_attn_box_rows(int head_dim) {
  return head_dim <= 64    ? Shape<64>::kKeys
         : head_dim <= 128 ? Shape<128>::kKeys
         : head_dim <= 192 ? Shape<192>::kKeys
                           : Shape<256>::kKeys;
}

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

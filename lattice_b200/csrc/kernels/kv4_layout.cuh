// Where a token's codes and scales lie in a 4-bit chunk (16 tokens, one kv head, K or V);
// kernels/kv4.cu has the format.
#pragma once

namespace kcmm {
namespace dev {

constexpr int kKv4Unit = 16;   // tokens of a chunk
constexpr int kKv4Group = 32;  // values of a scale

// Byte offset of lane `lane`'s word w of group j.  Groups lie in pairs where their number is
// even, so that a lane's load is 16 bytes instead of 8.
__host__ __device__ constexpr int kv4_code_offset(int groups, int j, int lane, int w) {
  return groups % 2 == 0 ? ((j >> 1) * 32 + lane) * 16 + (j & 1) * 8 + w * 4
                         : (j * 32 + lane) * 8 + w * 4;
}
// Byte offset of the scale of token t (of 16), group j.  K's: token g's groups, then token
// g+8's, by g.  V's: by token pair c, then group, then half of the unit, a pair in one word.
__host__ __device__ constexpr int kv4_scale_offset(bool is_v, int groups, int t, int j) {
  return groups * 256 + (is_v ? ((t & 7) >> 1) * groups * 8 + j * 8 + (t >> 3) * 4 + (t & 1) * 2
                              : (((t & 7) * 2 + (t >> 3)) * groups + j) * 2);
}

}  // namespace dev
}  // namespace kcmm

// The 4-bit cache's page format (include/mi_kv4.h) and its quantiser.
//
// A page is one block of one KV head: codes [D/32][block_size][16 bytes], then parameter words
// [block_size][D/32], a word holding the group's step s (low 16 bits) and minimum m (high 16 bits) as
// bfloat16.  The codes of one group of eight consecutive tokens are 128 contiguous bytes, which is
// what one 8x8 ldmatrix reads: as it stands it yields an MMA operand whose rows are tokens (K), and
// transposed one whose rows are head_dim values (V), with no shuffle and no bank conflict.
#pragma once

#include "common.cuh"

namespace mi {

constexpr int kKv4Group = 32;  // values that share (s, m)

__host__ __device__ __forceinline__ int64_t kv4_page_bytes(int block_size, int head_dim) {
  return (int64_t)block_size * head_dim / 2 + (int64_t)block_size * (head_dim / kKv4Group) * 4;
}

__device__ __forceinline__ float kv4_step(uint32_t word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float kv4_min(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

// Bits of x rounded to bfloat16 (nearest even).
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  const __nv_bfloat16 b = __float2bfloat16_rn(x);
  return *reinterpret_cast<const uint16_t*>(&b);
}

// Quantise a group spread over four consecutive lanes (eight values each): this lane's eight codes,
// packed, and the group's parameter word.  `quad` is the mask of the four lanes.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[8], unsigned quad, uint32_t& word) {
  float lo = x[0], hi = x[0];
  bool finite = fabsf(x[0]) <= 3.402823466e38f;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) <= 3.402823466e38f;  // false for NaN too
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(quad, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(quad, hi, o));
  }
  const uint32_t mb = bf16_bits(lo);
  const float m = __uint_as_float(mb << 16);
  const uint32_t sb = bf16_bits(__fdiv_rn(hi - m, 15.f));
  const float s = __uint_as_float(sb << 16);
  // A group that no finite (s, m) describes reads back as NaN.
  if (!__all_sync(quad, finite) || (mb & 0x7f80u) == 0x7f80u || (sb & 0x7f80u) == 0x7f80u) {
    word = 0x7fc00000u;
    return 0u;
  }
  // hi - m can be negative (m rounded up past a constant group): s <= 0 then, and all codes are 0.
  word = (mb << 16) | (s > 0.f ? sb : 0u);
  if (!(s > 0.f)) return 0u;
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i] - m, s)), 0.f), 15.f);
    code |= (uint32_t)c << (4 * i);
  }
  return code;
}

}  // namespace mi

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
//
// The code is the exact quotient (x - m) / s rounded to nearest even.  An IEEE division per value would
// bound the store (90 us of a 20,000-token store against 17 us of traffic); a product with 1 / s is off
// by at most 15 * 2^-23, so only a quotient that lands within 2^-17 of a tie is decided by its residual
// (x - m) - c s, which one fma gives exactly.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[8], unsigned quad, uint32_t& word) {
  float lo = x[0], hi = x[0], poison = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    poison = fmaf(x[i], 0.f, poison);  // NaN from an infinity or a NaN
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
  if (!__all_sync(quad, poison == 0.f) || (mb & 0x7f80u) == 0x7f80u || (sb & 0x7f80u) == 0x7f80u) {
    word = 0x7fc00000u;
    return 0u;
  }
  // hi - m can be negative (m rounded up past a constant group): s <= 0 then, and all codes are 0.
  word = (mb << 16) | (s > 0.f ? sb : 0u);
  if (!(s > 0.f)) return 0u;
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, nearest even
  const bool normal = s >= 0x1p-126f && s <= 0x1p125f;
  const float inv = normal ? __frcp_rn(s) : 0.f;
  float c[8], worst = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fminf(fmaxf((x[i] - m) * inv, 0.f), 15.f);
    c[i] = (y + kRound) - kRound;
    worst = fmaxf(worst, fabsf(y - c[i]));
  }
  if (worst > 0.5f - 0x1p-17f || !normal) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = x[i] - m;
      if (normal) {
        const float e = fmaf(-c[i], s, d);  // residual against half a step; at a tie the even code
        const float half = 0.5f * s;
        const bool odd = ((int)c[i] & 1) != 0;
        if (e > half || (e == half && odd)) c[i] += 1.f;
        else if (e < -half || (e == -half && odd)) c[i] -= 1.f;
      } else {
        c[i] = rintf(__fdiv_rn(d, s));
      }
      c[i] = fminf(fmaxf(c[i], 0.f), 15.f);
    }
  }
  // four codes are the digits of a 16-bit integer, read out of a float's mantissa
  const float w0 = fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0]))) + 8388608.f;
  const float w1 = fmaf(c[7], 4096.f, fmaf(c[6], 256.f, fmaf(c[5], 16.f, c[4]))) + 8388608.f;
  return __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x5410);
}

}  // namespace mi

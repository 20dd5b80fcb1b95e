// The 4-bit cache's page format (include/mi_kv4.h) and its quantiser.
//
// A page is one block of one KV head: codes [D/32][block_size][16 bytes], then parameter words
// [block_size][D/32], a word holding the group's step s (low 16 bits) and minimum m (high 16 bits) as
// bfloat16.  The codes of one group of eight consecutive tokens are 128 contiguous bytes, which is
// what one 8x8 ldmatrix reads: as it stands it yields an MMA operand whose rows are tokens (K), and
// transposed one whose rows are head_dim values (V), with no shuffle and no bank conflict.
#pragma once

#include <type_traits>

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

// Eight consecutive values as they are in memory.
template <typename T> struct Raw8 {
  uint32_t w[8 * sizeof(T) / 4];
  __device__ __forceinline__ float at(int i) const { return Elem<T>::to_f(reinterpret_cast<const T*>(w)[i]); }
  // value i less m, rounded to fp32: one instruction for the 16-bit types
  __device__ __forceinline__ float less(int i, float m) const {
    if constexpr (sizeof(T) == 2) {
      const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      float d;
      if constexpr (std::is_same<T, __half>::value) asm("sub.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(h), "f"(m));
      else asm("sub.f32.bf16 %0, %1, %2;" : "=f"(d) : "h"(h), "f"(m));
      return d;
    } else {
      return at(i) - m;
    }
  }
};

// Smallest and largest of a group spread over two consecutive lanes, NaN where there is one: K's in the first
// of the two, V's in the second (a whole warp calls).
template <typename T>
__device__ __forceinline__ void kv4_range(const Raw8<T> (&k)[2], const Raw8<T> (&v)[2], bool second, float& lo, float& hi) {
  if constexpr (sizeof(T) == 2) {
    // two values an instruction; (lo, -hi) as one pair that a minimum reduces
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto least_most = [](const Raw8<T> (&x)[2]) {
      const T2* p = reinterpret_cast<const T2*>(x[0].w);
      const T2* q = reinterpret_cast<const T2*>(x[1].w);
      T2 least = __hmin2_nan(p[0], q[0]), most = __hmax2_nan(p[0], q[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        least = __hmin2_nan(least, __hmin2_nan(p[i], q[i]));
        most = __hmax2_nan(most, __hmax2_nan(p[i], q[i]));
      }
      most = __hneg2(most);
      const uint32_t a = *reinterpret_cast<const uint32_t*>(&least), b = *reinterpret_cast<const uint32_t*>(&most);
      const uint32_t low = __byte_perm(a, b, 0x5410), high = __byte_perm(a, b, 0x7632);
      const T2 both = __hmin2_nan(*reinterpret_cast<const T2*>(&low), *reinterpret_cast<const T2*>(&high));
      return *reinterpret_cast<const uint32_t*>(&both);
    };
    const uint32_t kr = least_most(k), vr = least_most(v);
    const uint32_t own = second ? vr : kr;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, second ? kr : vr, 1);
    const T2 both = __hmin2_nan(*reinterpret_cast<const T2*>(&own), *reinterpret_cast<const T2*>(&other));
    lo = Elem<T>::to_f(both.x);
    hi = -Elem<T>::to_f(both.y);
  } else {
    float l[2], h[2], poison[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      l[t] = h[t] = (t ? v : k)[0].at(0);
      poison[t] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float f = (t ? v : k)[i >> 3].at(i & 7);
        l[t] = fminf(l[t], f);
        h[t] = fmaxf(h[t], f);
        poison[t] = fmaf(f, 0.f, poison[t]);  // NaN from a NaN (or an infinity)
      }
    }
    const float nan = (second ? poison[1] : poison[0]) + __shfl_xor_sync(0xffffffffu, second ? poison[0] : poison[1], 1);
    lo = fminf(second ? l[1] : l[0], __shfl_xor_sync(0xffffffffu, second ? l[0] : l[1], 1)) + nan;
    hi = fmaxf(second ? h[1] : h[0], __shfl_xor_sync(0xffffffffu, second ? h[0] : h[1], 1));
  }
}

// x / 15, correctly rounded: one correction of the product with 1 / 15 (exact over all mantissas; tiny x,
// whose residual would be subnormal, by division).
__device__ __forceinline__ float div15(float x) {
  if (fabsf(x) < 0x1p-100f) return __fdiv_rn(x, 15.f);
  constexpr float r = 1.f / 15.f;
  const float q = x * r;
  return fmaf(fmaf(-15.f, q, x), r, q);
}

// A group's parameter word (s, m) from its smallest and largest value.
__device__ __forceinline__ uint32_t kv4_word(float lo, float hi) {
  uint32_t mb = bf16_bits(lo);
  if (mb == 0x8000u) mb = 0u;  // a zero minimum has no sign: which of +0 and -0 a reduction keeps is its own affair
  const uint32_t sb = bf16_bits(div15(hi - __uint_as_float(mb << 16)));
  // A group that no finite (s, m) describes reads back as NaN (an infinite hi makes an infinite s or a NaN).
  const bool spoiled = (mb & 0x7f80u) == 0x7f80u || (sb & 0x7f80u) == 0x7f80u;
  // hi - m can be negative (m rounded up past a constant group): s <= 0 then, and all codes are 0.
  return spoiled ? 0x7fc00000u : (mb << 16) | (sb & 0x8000u ? 0u : sb);
}

// What a group's quotients need.
struct Kv4Scale {
  float m, s;
  float inv, s16;  // 1 / (16 s) within 2^-23, 16 s
  bool any;        // false: all codes are 0
  bool fast;       // s is far from the ends of fp32's range
};
__device__ __forceinline__ Kv4Scale kv4_scale(uint32_t word) {
  Kv4Scale g;
  g.m = kv4_min(word);
  g.s = kv4_step(word);
  g.any = g.s > 0.f;
  g.fast = g.s >= 0x1p-110f && g.s <= 0x1p110f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g.inv) : "f"(g.s));
  g.inv *= 0.0625f;
  g.s16 = 16.f * g.s;
  return g;
}

// round((x - m) / s) clamped to 0..15 as the low bits of 1.5 * 2^23 + c, from d = x - m.
//
// An IEEE division per value would bound the store (90 us of a 20,000-token store against 17 us of
// traffic).  The quotient is the product with 1 / s, corrected once by its residual: it is then off by at
// most half a unit and 2^-22 of one, so half way points, which 16-bit values meet every few hundred, come
// out exact.  Clamped to [0, 1] in units of 16 on the way (at most 15 (1 + 2^-8) / 16 but for the lower end).
__device__ __forceinline__ uint32_t kv4_code(const Kv4Scale& g, float d) {
  const float y0 = d * g.inv;
  const float y = __saturatef(fmaf(fmaf(-y0, g.s16, d), g.inv, y0));
  return __float_as_uint(fmaf(y, 16.f, 12582912.f));  // rounded to an integer
}
constexpr uint32_t kKv4CodeBase = 0x4b400000u;  // 1.5 * 2^23

// The same for steps at the ends of fp32's range: 0..15.
__device__ __forceinline__ uint32_t kv4_code_slow(const Kv4Scale& g, float d) {
  return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(d, g.s)), 0.f), 15.f);
}

// Quantise a group of K and one of V, both spread over two consecutive lanes (twice eight values each), by a
// whole warp: this lane's codes of both, eight a word, and the parameter word of K in the first of the two
// lanes (`second` false), of V in the other: each lane works out one and is told the other.
template <typename T>
__device__ __forceinline__ void kv4_quantise(const Raw8<T> (&k)[2], const Raw8<T> (&v)[2], bool second, uint32_t (&kc)[2],
                                             uint32_t (&vc)[2], uint32_t& word) {
  float lo, hi;
  kv4_range<T>(k, v, second, lo, hi);
  word = kv4_word(lo, hi);
  const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
  const Kv4Scale gk = kv4_scale(second ? other : word), gv = kv4_scale(second ? word : other);
  const bool odd = (gk.any && !gk.fast) || (gv.any && !gv.fast);
  if (!__any_sync(0xffffffffu, odd)) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      kc[n] = vc[n] = 0u - kKv4CodeBase * 0x11111111u;  // less the digits' common part
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kc[n] += kv4_code(gk, k[n].less(i, gk.m)) << (4 * i);
        vc[n] += kv4_code(gv, v[n].less(i, gv.m)) << (4 * i);
      }
      if (!gk.any) kc[n] = 0u;
      if (!gv.any) vc[n] = 0u;
    }
    return;
  }
  auto digit = [](const Kv4Scale& g, float d) {
    return !g.any ? 0u : g.fast ? kv4_code(g, d) - kKv4CodeBase : kv4_code_slow(g, d);
  };
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    kc[n] = vc[n] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      kc[n] |= digit(gk, k[n].at(i) - gk.m) << (4 * i);
      vc[n] |= digit(gv, v[n].at(i) - gv.m) << (4 * i);
    }
  }
}

// Quantise a group spread over 32 / E consecutive lanes, E fp32 values each, by a whole warp: this lane's E
// codes, packed, and the group's parameter word.  The same bytes as above for the same values.
template <int E>
__device__ __forceinline__ uint32_t kv4_quantise_warp(const float (&x)[E], uint32_t& word) {
  float lo = x[0], hi = x[0], poison = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    poison = fmaf(x[i], 0.f, poison);  // NaN from a NaN (or an infinity)
  }
#pragma unroll
  for (int o = 1; o < 32 / E; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    poison += __shfl_xor_sync(0xffffffffu, poison, o);
  }
  word = kv4_word(lo + poison, hi);
  const Kv4Scale g = kv4_scale(word);
  uint32_t code = 0;
  if (g.any) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      code |= (g.fast ? kv4_code(g, x[i] - g.m) - kKv4CodeBase : kv4_code_slow(g, x[i] - g.m)) << (4 * i);
  }
  return code;
}

// The eight values that packed codes and a parameter word stand for, rounded to T: bf16 and fp32 once, fp16 by way of
// fp32 (the parameters are no halves), half a unit and 2^-24 of the value at most.
template <typename T>
__device__ __forceinline__ Raw8<T> kv4_values(uint32_t code, uint32_t par) {
  Raw8<T> v;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    // c as 128 + c in a bfloat16's mantissa, less 128; s c + m is one fused operation on the stored halves
    const uint32_t s2 = __byte_perm(par, par, 0x1010), m2 = __byte_perm(par, par, 0x3232);
    const uint32_t next = code >> 4;
    const __nv_bfloat162 base = __float2bfloat162_rn(128.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // byte i of the word holds codes 2i and 2i + 1
      const uint32_t pair = (__byte_perm(code, next, 0x0400 + 0x0101 * i) & 0x000f000fu) | 0x43004300u;
      const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair), base);
      const __nv_bfloat162 r =
          __hfma2(c, *reinterpret_cast<const __nv_bfloat162*>(&s2), *reinterpret_cast<const __nv_bfloat162*>(&m2));
      v.w[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  } else {
    const float s = kv4_step(par), m = kv4_min(par);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = __uint_as_float(0x4b000000u | ((code >> (4 * i)) & 15u)) - 8388608.f;  // 2^23 + c, less 2^23
      reinterpret_cast<T*>(v.w)[i] = Elem<T>::from_f(fmaf(c, s, m));
    }
  }
  return v;
}

}  // namespace mi

// Paged decode attention over the 4-bit cache (format: kv4_format.cuh), one query token per sequence.
//
// A row's output is sum_t p_t v_t / sum_t p_t, p_t = exp(scale * q.k_t), k_t and v_t the values their
// codes stand for.
//
// Generic kernel (any type, head_dim, block size and group count): one CTA per (sequence, query head);
// its warps take the pages in turn, a lane holding value lane of every group, with an online softmax in
// fp32, and merge in shared memory.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_format.cuh"

namespace mi {
namespace {

constexpr int kKv4Warps = 8;  // of the generic kernel's CTA

template <typename T>
__global__ void __launch_bounds__(kKv4Warps * 32) kv4_decode_generic_kernel(const Kv4DecodeArgs a) {
  constexpr int MAXG = 256 / kKv4Group;
  const int64_t b = blockIdx.x / a.hq;
  const int hq = (int)(blockIdx.x - b * a.hq);
  const int h = hq / a.groups;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int ng = a.head_dim / kKv4Group;
  int64_t ctx = max((int64_t)0, a.context_lens[b]);
  if (ctx > a.max_blocks * a.block_size) {
    if (threadIdx.x == 0) record_status(MI_STATUS_BAD_LENGTH);
    ctx = a.max_blocks * a.block_size;
  }
  const T* q = reinterpret_cast<const T*>(a.q + b * a.q_sb + (int64_t)hq * a.q_sh);
  float qv[MAXG], acc[MAXG];
#pragma unroll
  for (int g = 0; g < MAXG; ++g) {
    qv[g] = g < ng ? Elem<T>::to_f(q[g * kKv4Group + lane]) * a.scale_log2 : 0.f;
    acc[g] = 0.f;
  }
  float m_run = -INFINITY, l_run = 0.f;
  const int64_t pages = (ctx + a.block_size - 1) / a.block_size;
  for (int64_t p = warp; p < pages; p += kKv4Warps) {
    int64_t blk = a.block_tables[b * a.table_stride + p];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) record_status(MI_STATUS_BAD_BLOCK);
      blk = 0;
    }
    const int64_t page = (blk * a.hkv + h) * a.page_bytes;
    const int64_t par = page + (int64_t)a.block_size * (a.head_dim >> 1);
    const int n = (int)min((int64_t)a.block_size, ctx - p * a.block_size);
    for (int t = 0; t < n; ++t) {
      float x = 0.f;
#pragma unroll
      for (int g = 0; g < MAXG; ++g) {
        if (g >= ng) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(a.k_pool + par + ((int64_t)t * ng + g) * 4);
        const uint32_t byte = (uint8_t)a.k_pool[page + ((int64_t)g * a.block_size + t) * 16 + (lane >> 1)];
        x = fmaf(qv[g], fmaf((float)((byte >> (4 * (lane & 1))) & 15u), kv4_step(w), kv4_min(w)), x);
      }
      x = warp_sum(x);
      const float m_new = fmaxf(m_run, x);
      const float alpha = m_new == -INFINITY ? 1.f : exp2f(m_run - m_new);
      const float pr = m_new == -INFINITY ? 0.f : exp2f(x - m_new);
      l_run = l_run * alpha + pr;
      m_run = m_new;
#pragma unroll
      for (int g = 0; g < MAXG; ++g) {
        if (g >= ng) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(a.v_pool + par + ((int64_t)t * ng + g) * 4);
        const uint32_t byte = (uint8_t)a.v_pool[page + ((int64_t)g * a.block_size + t) * 16 + (lane >> 1)];
        acc[g] = acc[g] * alpha + pr * fmaf((float)((byte >> (4 * (lane & 1))) & 15u), kv4_step(w), kv4_min(w));
      }
    }
  }
  __shared__ float sm[kKv4Warps], sl[kKv4Warps], so[kKv4Warps][256];
  if (lane == 0) {
    sm[warp] = m_run;
    sl[warp] = l_run;
  }
#pragma unroll
  for (int g = 0; g < MAXG; ++g)
    if (g < ng) so[warp][g * kKv4Group + lane] = acc[g];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.head_dim) return;
  float m_all = -INFINITY;
  for (int w = 0; w < kKv4Warps; ++w) m_all = fmaxf(m_all, sm[w]);
  float o = 0.f, l = 0.f;
  for (int w = 0; w < kKv4Warps; ++w) {
    const float f = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - m_all);
    l += f * sl[w];
    o += f * so[w][d];
  }
  T* dst = reinterpret_cast<T*>(a.out + b * a.out_sb) + (int64_t)hq * a.head_dim;
  dst[d] = Elem<T>::from_f(l == 0.f ? 0.f : o / l);
}

}  // namespace

Kv4DecodePlan plan_kv4_decode(int64_t batch, int hq, int hkv, int head_dim, int64_t max_blocks, int block_size,
                              int dtype) {
  (void)batch, (void)hq, (void)hkv, (void)head_dim, (void)max_blocks, (void)block_size, (void)dtype;
  return Kv4DecodePlan{};
}

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, const Kv4DecodePlan& plan, int dtype, cudaStream_t s) {
  (void)plan;
  const unsigned grid = (unsigned)(a.batch * a.hq);
  if (dtype == MI_BF16) kv4_decode_generic_kernel<__nv_bfloat16><<<grid, kKv4Warps * 32, 0, s>>>(a);
  else if (dtype == MI_F16) kv4_decode_generic_kernel<__half><<<grid, kKv4Warps * 32, 0, s>>>(a);
  else kv4_decode_generic_kernel<float><<<grid, kKv4Warps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mi

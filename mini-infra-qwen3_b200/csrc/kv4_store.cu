// Store and gather of the 4-bit paged cache (format: kv4_format.cuh).
//
// * kv4_scatter_kernel / kv4_store_chunks_kernel — quantise tokens into their slots, K and V in one
//   launch; a thread takes eight values of K and the same eight of V, four lanes a group;
// * kv4_gather_kernel — pages back as dense blocks in the model's type: out = T(m + s * c).
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_format.cuh"

namespace mi {
namespace {

constexpr int kKv4Threads = 256;

// Eight consecutive elements as floats; one or two 16-byte loads when the host proved them aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void kv4_load8(const char* p, float (&x)[8]) {
  if constexpr (VEC) {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / N; ++j) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + j);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) x[j * N + i] = Elem<T>::to_f(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(reinterpret_cast<const T*>(p)[i]);
  }
}

// Unit u (eight values of head h = u / (D/8)) of one token into slot (block, offset).
template <typename T, bool VEC>
__device__ __forceinline__ void kv4_put(const Kv4StoreArgs& a, const char* k_row, const char* v_row, int64_t block,
                                        int offset, int u) {
  const int per_head = a.head_dim >> 3;
  const int h = u / per_head;
  const int w = u - h * per_head;  // 8-value unit of the head; group w / 4
  float k[8], v[8];
  kv4_load8<T, VEC>(k_row + h * a.k_sb[1] + (int64_t)w * 8 * (int)sizeof(T), k);
  kv4_load8<T, VEC>(v_row + h * a.v_sb[1] + (int64_t)w * 8 * (int)sizeof(T), v);
  const unsigned quad = 0xfu << (threadIdx.x & 28);
  uint32_t kw, vw;
  const uint32_t kc = kv4_quantise(k, quad, kw);
  const uint32_t vc = kv4_quantise(v, quad, vw);
  const int64_t page = (block * a.heads + h) * a.page_bytes;
  const int64_t code_at = page + ((int64_t)(w >> 2) * a.block_size + offset) * 16 + (w & 3) * 4;
  *reinterpret_cast<uint32_t*>(a.k_pool + code_at) = kc;
  *reinterpret_cast<uint32_t*>(a.v_pool + code_at) = vc;
  if ((w & 3) == 0) {
    const int64_t par_at = page + (int64_t)a.block_size * (a.head_dim >> 1) +
                           ((int64_t)offset * (a.head_dim / kKv4Group) + (w >> 2)) * 4;
    *reinterpret_cast<uint32_t*>(a.k_pool + par_at) = kw;
    *reinterpret_cast<uint32_t*>(a.v_pool + par_at) = vw;
  }
}

// Flat over (token, unit); the four lanes of a group always take the same path.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kKv4Threads) kv4_scatter_kernel(const Kv4StoreArgs a) {
  const int units = a.heads * (a.head_dim >> 3);
  const int64_t total = a.num_tokens * units;
  for (int64_t i = (int64_t)blockIdx.x * kKv4Threads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kKv4Threads) {
    const int64_t token = i / units;
    const int u = (int)(i - token * units);
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.num_blocks * a.block_size) {
      if (u == 0) record_status(MI_STATUS_BAD_SLOT);
      continue;
    }
    const int64_t row = a.rows ? a.rows[token] : token;
    const int64_t pos = a.positions ? a.positions[token] : 0;
    if (row < 0 || row >= a.src_rows || pos < 0 || pos >= a.src_positions) {
      if (u == 0) record_status(MI_STATUS_BAD_INDEX);
      continue;
    }
    const int64_t block = slot / a.block_size;
    kv4_put<T, VEC>(a, a.k_src + row * a.k_sb[0] + pos * a.k_sb[2], a.v_src + row * a.v_sb[0] + pos * a.v_sb[2], block,
                    (int)(slot - block * a.block_size), u);
  }
}

// Flat over (row, padded position, unit); padding positions are skipped.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kKv4Threads) kv4_store_chunks_kernel(const Kv4StoreArgs a) {
  const int units = a.heads * (a.head_dim >> 3);
  const int64_t total = a.batch * a.padded_len * units;
  for (int64_t i = (int64_t)blockIdx.x * kKv4Threads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kKv4Threads) {
    const int64_t item = i / units;  // row * padded_len + p
    const int u = (int)(i - item * units);
    const int64_t row = item / a.padded_len;
    const int64_t p = item - row * a.padded_len;
    const int64_t len = a.chunk_lens[row];
    const int64_t first = a.padded_len - len;
    if (first < 0 && p == 0 && u == 0) record_status(MI_STATUS_BAD_LENGTH);  // only the last padded_len exist
    if (p < first) continue;
    const int64_t pos = a.starts[row] + (p - first);
    const int64_t logical = pos / a.block_size;
    if (pos < 0 || logical >= a.table_width) {
      if (u == 0) record_status(MI_STATUS_BAD_LENGTH);
      continue;
    }
    const int64_t block = a.block_tables[row * a.table_stride + logical];
    if (block < 0 || block >= a.num_blocks) {
      if (u == 0) record_status(MI_STATUS_BAD_BLOCK);
      continue;
    }
    kv4_put<T, VEC>(a, a.k_src + row * a.k_sb[0] + p * a.k_sb[2], a.v_src + row * a.v_sb[0] + p * a.v_sb[2], block,
                    (int)(pos - logical * a.block_size), u);
  }
}

// One CTA per gathered block: flat over (token, head, 8-value unit) of K, then of V.
template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_gather_kernel(const Kv4GatherArgs a) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t item = blockIdx.x;  // b * blocks_per_row + j
  const int64_t b = item / a.blocks_per_row;
  const int64_t j = item - b * a.blocks_per_row;
  const int per_head = a.head_dim >> 3;
  const int units = a.heads * per_head;  // per token
  const int total = a.block_size * units;
  int64_t valid = a.block_size;  // tokens of this block that are read
  if (a.lengths) valid = min((int64_t)a.block_size, max((int64_t)0, a.lengths[b] - j * a.block_size));
  int64_t block = 0;
  if (valid > 0) {
    block = a.block_ids[b * a.id_stride + j];
    if (block < 0 || block >= a.num_blocks) {
      if (threadIdx.x == 0) record_status(MI_STATUS_BAD_BLOCK);
      valid = 0;
    }
  }
  const int ng = a.head_dim / kKv4Group;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const char* pool = kv ? a.v_pool : a.k_pool;
    T* out = reinterpret_cast<T*>(kv ? a.v_out : a.k_out) + item * total * 8;
    for (int i = threadIdx.x; i < total; i += kKv4Threads) {
      const int t = i / units;
      const int u = i - t * units;
      const int h = u / per_head;
      const int w = u - h * per_head;
      uint4 pk[8 / N];
      T* e = reinterpret_cast<T*>(pk);
      if (t < valid) {
        const char* page = pool + (block * a.heads + h) * a.page_bytes;
        const uint32_t code =
            __ldg(reinterpret_cast<const uint32_t*>(page + ((int64_t)(w >> 2) * a.block_size + t) * 16) + (w & 3));
        const uint32_t par = __ldg(
            reinterpret_cast<const uint32_t*>(page + (int64_t)a.block_size * (a.head_dim >> 1)) + t * ng + (w >> 2));
        const float s = kv4_step(par), m = kv4_min(par);
#pragma unroll
        for (int n = 0; n < 8; ++n) e[n] = Elem<T>::from_f(fmaf((float)((code >> (4 * n)) & 15u), s, m));
      } else {
#pragma unroll
        for (int n = 0; n < 8; ++n) e[n] = Elem<T>::from_f(0.f);
      }
#pragma unroll
      for (int n = 0; n < 8 / N; ++n) reinterpret_cast<uint4*>(out + (int64_t)i * 8)[n] = pk[n];
    }
  }
}

template <typename T>
cudaError_t launch_kv4_store_t(const Kv4StoreArgs& a, bool chunks, bool vec, cudaStream_t s) {
  const int64_t tokens = chunks ? a.batch * a.padded_len : a.num_tokens;
  const int64_t threads = tokens * a.heads * (a.head_dim >> 3);
  const unsigned grid = (unsigned)std::min<int64_t>((threads + kKv4Threads - 1) / kKv4Threads, 148 * 16);
  if (chunks) {
    if (vec) kv4_store_chunks_kernel<T, true><<<grid, kKv4Threads, 0, s>>>(a);
    else kv4_store_chunks_kernel<T, false><<<grid, kKv4Threads, 0, s>>>(a);
  } else {
    if (vec) kv4_scatter_kernel<T, true><<<grid, kKv4Threads, 0, s>>>(a);
    else kv4_scatter_kernel<T, false><<<grid, kKv4Threads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_store(const Kv4StoreArgs& a, bool chunks, bool vec, int dtype, cudaStream_t s) {
  if (dtype == MI_BF16) return launch_kv4_store_t<__nv_bfloat16>(a, chunks, vec, s);
  if (dtype == MI_F16) return launch_kv4_store_t<__half>(a, chunks, vec, s);
  return launch_kv4_store_t<float>(a, chunks, vec, s);
}

cudaError_t launch_kv4_gather(const Kv4GatherArgs& a, int dtype, cudaStream_t s) {
  const unsigned grid = (unsigned)(a.batch * a.blocks_per_row);
  if (dtype == MI_BF16) kv4_gather_kernel<__nv_bfloat16><<<grid, kKv4Threads, 0, s>>>(a);
  else if (dtype == MI_F16) kv4_gather_kernel<__half><<<grid, kKv4Threads, 0, s>>>(a);
  else kv4_gather_kernel<float><<<grid, kKv4Threads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mi

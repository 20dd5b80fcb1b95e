// Store and gather of the 4-bit paged cache (format: kv4_format.cuh).
//
// * kv4_store_kernel — quantises tokens into their slots, K and V in one launch: tokens at given slots or
//   right-aligned chunks through block tables;
// * kv4_gather_kernel — pages back as dense blocks in the model's type: out = T(m + s * c).
//
// Both move bytes: 16 histories of up to 16,383 tokens are gathered in 206 us (1.28 GB, 0.95 of the measured HBM
// rate); 22,300 tokens of 8 heads of 128 are stored in 27 us (18 us of traffic; 32,768 in 35, 27): about 13
// instructions a value of K and V, and the start and end of the grid, are what is left.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_format.cuh"

namespace mi {
namespace {

constexpr int kKv4Threads = 256;       // of a gathering CTA
constexpr int kKv4StoreThreads = 128;
constexpr int kKv4Tile = 16;  // tokens of a storing CTA

// Eight consecutive elements; 16-byte loads when the host proved them aligned.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> kv4_load8(const char* p) {
  Raw8<T> x;
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j)
      reinterpret_cast<uint4*>(x.w)[j] = __ldg(reinterpret_cast<const uint4*>(p) + j);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(x.w)[i] = reinterpret_cast<const T*>(p)[i];
  }
  return x;
}

// A CTA takes sixteen tokens (two lanes each: its slot is looked up once) and strides its warps over the
// (head, group) pairs, a lane quantising sixteen values of K and the same of V.  A warp's sixteen tokens of
// one group read 64-byte runs and, where the tokens share a page, write 256 contiguous bytes.  Four warps a
// CTA: 27 us where eight took 30, a CTA leaving its registers to the next sooner.  The next pair's loads are
// issued before this pair is quantised.  NG: groups of a head, 0 for any; it divides the stride, so that a warp
// keeps its group and its pointers move by fixed amounts.
template <typename T, bool VEC, bool CHUNKS, int NG>
__global__ void __launch_bounds__(kKv4StoreThreads) kv4_store_kernel(const Kv4StoreArgs a) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const unsigned tokens = (unsigned)(CHUNKS ? a.batch * a.padded_len : a.num_tokens);  // < 2^31
  const unsigned token = blockIdx.x * (unsigned)kKv4Tile + (lane >> 1);
  const bool tell = warp == 0 && blockIdx.y == 0 && (lane & 1) == 0;
  const int ng = NG ? NG : a.head_dim / kKv4Group;
  const int w = lane & 1;  // takes eight-value quarters w and w + 2 of the group
  const int pairs = a.heads * ng;
  static_assert(NG == 0 || kKv4StoreThreads / 32 % (NG ? NG : 1) == 0, "a warp keeps its group");
  const int step = gridDim.y * (kKv4StoreThreads / 32);
  int pair = blockIdx.y * (kKv4StoreThreads / 32) + warp;
  if (pair >= pairs) return;
  // where the token comes from; the loads below are in flight while its slot is looked up.  The lanes of a
  // token that is not stored stay for the warp's exchanges.
  bool live = token < tokens;
  int64_t row = 0, p = 0, pos = 0;
  if (live) {
    if constexpr (CHUNKS) {
      row = token / (unsigned)a.padded_len;
      p = token - (unsigned)row * (unsigned)a.padded_len;
      const int64_t first = a.padded_len - a.chunk_lens[row];
      pos = a.starts[row] + (p - first);
      if (first < 0 && p == 0 && tell) record_status(MI_STATUS_BAD_LENGTH);  // only the last padded_len exist
      live = p >= first;
    } else {
      row = a.rows ? a.rows[token] : token;
      p = a.positions ? a.positions[token] : 0;
      if (row < 0 || row >= a.src_rows || p < 0 || p >= a.src_positions) {
        if (tell) record_status(MI_STATUS_BAD_INDEX);
        live = false;
      }
    }
  }
  int h = pair / ng, g = pair - h * ng;
  const char* k_src = a.k_src + row * a.k_sb[0] + p * a.k_sb[2] + w * 8 * (int)sizeof(T);
  const char* v_src = a.v_src + row * a.v_sb[0] + p * a.v_sb[2] + w * 8 * (int)sizeof(T);
  auto load = [&](int h, int g, Raw8<T> (&k)[2], Raw8<T> (&v)[2]) {
    const int at = g * kKv4Group * (int)sizeof(T);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      k[n] = kv4_load8<T, VEC>(k_src + h * a.k_sb[1] + at + n * 16 * (int)sizeof(T));
      v[n] = kv4_load8<T, VEC>(v_src + h * a.v_sb[1] + at + n * 16 * (int)sizeof(T));
    }
  };
  Raw8<T> k[2] = {}, v[2] = {};
  if (live) load(h, g, k, v);
  int64_t block = 0;
  unsigned offset = 0;
  if (live) {
    if constexpr (CHUNKS) {
      if (pos < 0 || pos >= a.table_width * a.block_size) {
        if (tell) record_status(MI_STATUS_BAD_LENGTH);
        live = false;
      } else {
        const unsigned logical = (unsigned)pos / (unsigned)a.block_size;  // pos < 2^31
        offset = (unsigned)pos - logical * (unsigned)a.block_size;
        block = a.block_tables[row * a.table_stride + logical];
        if (block < 0 || block >= a.num_blocks) {
          if (tell) record_status(MI_STATUS_BAD_BLOCK);
          live = false;
        }
      }
    } else {
      const int64_t slot = a.slots[token];
      if (slot < 0 || slot >= a.num_blocks * a.block_size) {
        if (tell) record_status(MI_STATUS_BAD_SLOT);
        live = false;
      } else {
        block = (unsigned)slot / (unsigned)a.block_size;  // slots < 2^31
        offset = (unsigned)slot - (unsigned)block * (unsigned)a.block_size;
      }
    }
  }
  if (!__any_sync(0xffffffffu, live)) return;
  char* k_page = a.k_pool + block * a.heads * a.page_bytes;
  char* v_page = a.v_pool + block * a.heads * a.page_bytes;
  const int par0 = a.block_size * (a.head_dim >> 1) + (int)offset * ng * 4;
  while (true) {
    Raw8<T> k_next[2] = {}, v_next[2] = {};
    const bool more = pair + step < pairs;
    const int h_next = NG ? h + step / (NG ? NG : 1) : (pair + step) / ng;
    const int g_next = NG ? g : pair + step - h_next * ng;
    if (more && live) load(h_next, g_next, k_next, v_next);
    uint32_t word, kc[2], vc[2];
    kv4_quantise<T>(k, v, w, kc, vc, word);
    if (live) {
      const int64_t page = h * a.page_bytes;
      const int64_t code_at = page + ((int64_t)g * a.block_size + offset) * 16 + w * 4;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        *reinterpret_cast<uint32_t*>(k_page + code_at + n * 8) = kc[n];
        *reinterpret_cast<uint32_t*>(v_page + code_at + n * 8) = vc[n];
      }
      *reinterpret_cast<uint32_t*>((w ? v_page : k_page) + page + par0 + g * 4) = word;
    }
    if (!more) return;
    pair += step;
    h = h_next;
    g = g_next;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      k[n] = k_next[n];
      v[n] = v_next[n];
    }
  }
}

// One CTA per gathered block of K (blockIdx.y 0) or V (1): flat over (token, head, 8-value unit), a lane
// reading four bytes of codes and writing eight values, so that a warp's stores are contiguous.  PH: units
// of a head (head_dim / 8), 0 for one not known at compile time.
template <typename T, int PH>
__global__ void __launch_bounds__(kKv4Threads) kv4_gather_kernel(const Kv4GatherArgs a) {
  constexpr int N = 16 / (int)sizeof(T);
  constexpr int MLP = 4;  // units in flight a lane
  const unsigned item = blockIdx.x;  // b * blocks_per_row + j
  const unsigned b = item / (unsigned)a.blocks_per_row;
  const int64_t j = item - b * (unsigned)a.blocks_per_row;
  const int per_head = PH ? PH : a.head_dim >> 3;
  const int rows = a.block_size * a.heads;  // (token, head)
  const int total = rows * per_head;
  int64_t valid = a.block_size;  // tokens of this block that are read
  if (a.lengths) valid = min((int64_t)a.block_size, max((int64_t)0, a.lengths[b] - j * a.block_size));
  if (valid == 0 && !a.fill_past) return;
  int64_t block = 0;
  if (valid > 0) {
    block = a.block_ids[b * a.id_stride + j];
    if (block < 0 || block >= a.num_blocks) {
      if (threadIdx.x == 0 && blockIdx.y == 0) record_status(MI_STATUS_BAD_BLOCK);
      valid = 0;
    }
  }
  const int ng = a.head_dim / kKv4Group;
  const char* pool = (blockIdx.y ? a.v_pool : a.k_pool) + block * a.heads * a.page_bytes;
  const int par_off = a.block_size * (a.head_dim >> 1);
  uint4* out = reinterpret_cast<uint4*>((blockIdx.y ? a.v_out : a.k_out) + (int64_t)item * total * 8 * (int)sizeof(T));
  // Unit i is 8-value unit w of (token t, head h); stepping by a CTA's width moves the three by fixed amounts.
  const int row0 = threadIdx.x / per_head;
  int w = threadIdx.x - row0 * per_head;
  int t = row0 / a.heads;
  int h = row0 - t * a.heads;
  const int step_row = kKv4Threads / per_head, step_w = kKv4Threads - step_row * per_head;
  const int step_t = step_row / a.heads, step_h = step_row - step_t * a.heads;
  for (int i0 = threadIdx.x; i0 < total; i0 += MLP * kKv4Threads) {
    uint32_t code[MLP], par[MLP];
#pragma unroll
    for (int n = 0; n < MLP; ++n) {
      code[n] = par[n] = 0u;  // stands for zeros
      if (t < valid) {
        const char* page = pool + h * a.page_bytes;
        code[n] = __ldg(reinterpret_cast<const uint32_t*>(page + ((w >> 2) * a.block_size + t) * 16) + (w & 3));
        par[n] = __ldg(reinterpret_cast<const uint32_t*>(page + par_off) + t * ng + (w >> 2));
      }
      t += step_t;
      h += step_h;
      if (PH == 0 || kKv4Threads % (PH ? PH : 1) != 0) {
        w += step_w;
        if (w >= per_head) w -= per_head, ++h;
      }
      if (h >= a.heads) h -= a.heads, ++t;
    }
#pragma unroll
    for (int n = 0; n < MLP; ++n) {
      const int i = i0 + n * kKv4Threads;
      if (i >= total) break;
      const Raw8<T> v = kv4_values<T>(code[n], par[n]);
#pragma unroll
      for (int c = 0; c < 8 / N; ++c) out[(int64_t)i * (8 / N) + c] = reinterpret_cast<const uint4*>(v.w)[c];
    }
  }
}

template <typename T>
cudaError_t launch_kv4_store_t(const Kv4StoreArgs& a, bool chunks, bool vec, cudaStream_t s) {
  const int64_t tokens = chunks ? a.batch * a.padded_len : a.num_tokens;
  const int64_t tiles = (tokens + kKv4Tile - 1) / kKv4Tile;
  const int pair_tiles = (a.heads * (a.head_dim / kKv4Group) + kKv4StoreThreads / 32 - 1) / (kKv4StoreThreads / 32);
  // every pair of a token in one CTA where the tokens fill the SMs, else the pairs spread over CTAs
  const dim3 grid((unsigned)tiles, (unsigned)(tiles >= 148 * 4 ? 1 : pair_tiles));
  auto launch = [&](auto kernel) { kernel<<<grid, kKv4StoreThreads, 0, s>>>(a); };
  const int ng = a.head_dim / kKv4Group;
  if (chunks) {
    if (vec && ng == 4) launch(kv4_store_kernel<T, true, true, 4>);
    else if (vec) launch(kv4_store_kernel<T, true, true, 0>);
    else launch(kv4_store_kernel<T, false, true, 0>);
  } else {
    if (vec && ng == 4) launch(kv4_store_kernel<T, true, false, 4>);
    else if (vec) launch(kv4_store_kernel<T, true, false, 0>);
    else launch(kv4_store_kernel<T, false, false, 0>);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_kv4_gather_t(const Kv4GatherArgs& a, cudaStream_t s) {
  const dim3 grid((unsigned)(a.batch * a.blocks_per_row), 2);
  if (a.head_dim == 128) kv4_gather_kernel<T, 16><<<grid, kKv4Threads, 0, s>>>(a);
  else if (a.head_dim == 64) kv4_gather_kernel<T, 8><<<grid, kKv4Threads, 0, s>>>(a);
  else kv4_gather_kernel<T, 0><<<grid, kKv4Threads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_store(const Kv4StoreArgs& a, bool chunks, bool vec, int dtype, cudaStream_t s) {
  if (dtype == MI_BF16) return launch_kv4_store_t<__nv_bfloat16>(a, chunks, vec, s);
  if (dtype == MI_F16) return launch_kv4_store_t<__half>(a, chunks, vec, s);
  return launch_kv4_store_t<float>(a, chunks, vec, s);
}

cudaError_t launch_kv4_gather(const Kv4GatherArgs& a, int dtype, cudaStream_t s) {
  if (dtype == MI_BF16) return launch_kv4_gather_t<__nv_bfloat16>(a, s);
  if (dtype == MI_F16) return launch_kv4_gather_t<__half>(a, s);
  return launch_kv4_gather_t<float>(a, s);
}

}  // namespace mi

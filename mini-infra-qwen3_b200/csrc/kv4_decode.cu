// Paged decode attention over the 4-bit cache (format: kv4_format.cuh), one query token per sequence.
//
// A row's output is sum_t p_t v_t / sum_t p_t, p_t = exp(scale * q.k_t), k_t and v_t the values their
// codes stand for.
//
// Tensor-core kernel (16-bit types, head_dim 64/128, block size 16/32, at most 8 query heads per KV
// head).  With k = m + s c per group g of 32 values,
//     q.k_t = sum_g s_tg (q_g . c_tg) + m_tg sum(q_g),     o = sum_t (p_t s_tg) (c_tg - 8) + p_t (m_tg + 8 s_tg),
// so the codes themselves are the MMA operands and the steps and minima enter once per token and group:
// there is no pass that dequantises.  A code is masked out of its word straight into a half: c in bits
// 0-3 of a half is the subnormal c * 2^-24, in bits 4-7 it is 16 c * 2^-24, both exact, so one AND makes
// two operands and one shift serves eight codes.  The 16s go into q (K) and into the epilogue (V).
//   * Tokens are the M rows of S^T = K Q^T (m16n8k16, N = up to 8 query heads), head_dim values those of
//     O^T = V^T P^T; the transposed orientation fills all 16 rows where the query heads would fill at
//     most 8.  P^T gets from accumulator to operand layout by movmatrix, once per group of 32 values
//     because p s differs by group.
//   * q is scaled by a power of two to a largest value in [2^14, 2^15) and held in fp16: exact for the
//     16-bit types except far below the row's largest value (absolute error 2^-24 of it).
//   * p s is held in fp16.  The softmax's running reference is one of p * s, not of p: it keeps the largest
//     product in fp16's upper range, so rounding costs at most 2^-11 of a weight (a group whose step is below
//     2^-25 of its token's widest loses more of its own); an fp16 model, whose output has as many bits,
//     carries the rounding's remainder in a second fp16 operand.
//   * Scores, sums, the minimum terms and O are fp32.  An output of a long row is small beside sum p s c (hundreds of
//     times over 32,768 tokens of like weights), and an MMA rounds towards zero at every step, at the place of its
//     largest term: hence the codes count from 8, their middle, and hence O stands outside the accumulators, which
//     hold the sum of 16 or 32 tokens and are added to it with a rounding to nearest.  For bf16 the middle goes in by
//     an MMA with -8 in place of the codes; that starts the sum at 128 p s, whose last place takes up to 1e-4 of a long
//     row's output, so an fp16 model's operands are c - 8 themselves (one subtraction for two).  Relative
//     errors, 900 rows of 32,768 tokens of like weights: with whole codes summed in the accumulators 2.3e-2 (fp16) and
//     1.6e-2 (bf16), now 2.2e-4 and 1.7e-3, the outputs' rounding.  It takes 5 to 23 % of the time (64 rows of
//     16,384, bf16: 217 -> 228 us at 32/8 heads, 241 -> 287 at 64/8; fp16: 250 -> 299, 286 -> 353).
// Persistent CTAs, three a SM: a producer warp brings whole pages (all heads of a block in one bulk copy for
// K and one for V) into a ring of steps of 32 tokens x 4 KV heads (or 64 x 2, 128 x 1), 4 consumer warps each
// take a (KV head, 32 tokens) of a step.  The sequences' steps form one stream that the CTAs share in equal
// ranges; pieces of a sequence cut by a border are merged by the combine kernel.
// Bound by HBM: 64 rows of 32,768 tokens, 32/8 heads, bf16, 2.68 GB of pages in 454 us, 5.9 TB/s, where a copy
// reaches 6.55; run for seconds the power limit lowers the clocks and the ALU work of cutting codes shows (64 rows of
// up to 32,768: 234 us -> 270).  One CTA per (row, 1,024 tokens) took 260 us where equal ranges took 236: its waves
// ended raggedly.
//
// Generic kernel (any type, head_dim, block size and group count): one CTA per (sequence, query head);
// its warps take the pages in turn, a lane holding value lane of every group, with an online softmax in
// fp32, and merge in shared memory.
#include <algorithm>
#include <type_traits>

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
      // fmaxf passes a NaN score by, its weight does not: the row becomes NaN wherever the token stands
      const float alpha = m_new == -INFINITY ? 1.f : exp2f(m_run - m_new);
      const float pr = x == -INFINITY ? 0.f : exp2f(x - m_new);
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
    const float f = m_all == -INFINITY ? 1.f : exp2f(sm[w] - m_all);  // a warp of no tokens: 0, of sums 0
    l += f * sl[w];
    o += f * so[w][d];
  }
  T* dst = reinterpret_cast<T*>(a.out + b * a.out_sb) + (int64_t)hq * a.head_dim;
  dst[d] = Elem<T>::from_f(ctx == 0 ? 0.f : o / l);
}

constexpr int kKv4Consumers = 4;  // consumer warps of the tensor-core kernel's CTA
constexpr int kKv4SplitThreads = (kKv4Consumers + 1) * 32;
constexpr int kKv4CtasPerSm = 3;
constexpr int kKv4Smem = 74 * 1024;  // of a CTA
constexpr int kKv4MinSteps = 2;    // steps of a CTA, at least
constexpr int kKv4WholeSteps = 8;  // sequences of at most this many are not cut
constexpr int kKv4Unit = 32;  // tokens a consumer warp takes at a time: two 16-row tiles

template <int D, int BS, int HB, int SH>
struct Kv4Shape {
  static constexpr int kGroups = D / kKv4Group;
  static constexpr int kCols = 8 / SH;                  // query heads of a KV head, rounded up
  static constexpr int kUnits = kKv4Consumers / HB;     // units of a step: one (KV head, unit) per warp
  static constexpr int kTokens = kUnits * kKv4Unit;     // tokens of a step
  static constexpr int kPages = kTokens / BS;           // and its pages
  static constexpr int kPageBytes = BS * D / 2 + BS * kGroups * 4;
  static constexpr int kStageBytes = kPages * HB * 2 * kPageBytes;
  static constexpr int kMergeBytes = kUnits > 1 ? kKv4Consumers * kCols * (D + 2) * 4 : 0;
  static constexpr int kStages = std::min(6, (kKv4Smem - kMergeBytes - 128) / (kStageBytes + 16));
  static constexpr int kSmemBytes = kMergeBytes + kStages * (kStageBytes + 16) + 128;
};

constexpr float kKv4TopLog2 = 11.f;   // p * s of a new reference: at most 2^11
constexpr float kKv4Limit = 32768.f;  // p * s above this moves the reference (fp16 ends at 65504)
constexpr float kKv4Narrow = 0x1p-53f;  // steps below this count as this: p stays below 2^68 whatever the steps

__device__ __forceinline__ float pow2(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }  // -126 <= n <= 128

// Four operands out of eight codes: codes (0, 4), (1, 5) times 16, (2, 6), (3, 7) times 16, as halves
// in units of 2^-24.
__device__ __forceinline__ void kv4_operands(uint32_t w, uint32_t (&o)[4]) {
  o[0] = w & 0x000f000fu;
  o[1] = w & 0x00f000f0u;
  const uint32_t w8 = w >> 8;
  o[2] = w8 & 0x000f000fu;
  o[3] = w8 & 0x00f000f0u;
}

// Two halves base + c, c a code, as c - 8 (exact).
__device__ __forceinline__ uint32_t kv4_centred(uint32_t w, float base_and_8) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(base_and_8));
  return *reinterpret_cast<const uint32_t*>(&d);
}

template <int NG>
__device__ __forceinline__ void kv4_params(const uint8_t* p, uint32_t (&w)[NG]) {
  if constexpr (NG == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  }
}

// Where a CTA's share of the work lies.  The sequences (row b, block of HB KV heads), one after the other,
// are a stream of steps; CTA c takes steps [c * quota, (c + 1) * quota).  A sequence of no tokens has one
// step, which writes its zeros.
struct Kv4Walk {
  int64_t b;
  int64_t rest;  // steps left to this CTA, the current sequence's included
  int hb;
  int pos;       // first step of the current sequence that is this CTA's
  int steps;     // of the current sequence
  int ctx;       // tokens of the current sequence
  __device__ __forceinline__ int take() const { return (int)min(rest, (int64_t)(steps - pos)); }
};

template <int TOKENS>
__device__ __forceinline__ int kv4_steps(int ctx) {
  return max(1, (ctx + TOKENS - 1) / TOKENS);
}

// Tokens of row b, at most what its block table covers.
__device__ __forceinline__ int kv4_ctx(const Kv4DecodeArgs& a, int64_t b) {
  return (int)max((int64_t)0, min(a.context_lens[b], a.max_blocks * a.block_size));
}

template <int TOKENS>
__device__ __forceinline__ void kv4_advance(const Kv4DecodeArgs& a, Kv4Walk& w, int heads_per_cta, int next_ctx) {
  w.rest -= w.take();
  w.pos = 0;
  if (++w.hb * heads_per_cta == a.hkv) {
    w.hb = 0;
    ++w.b;
    w.ctx = next_ctx;
    w.steps = kv4_steps<TOKENS>(next_ctx);
  }
}

// This CTA's start, by every thread: a block-wide scan over the rows' steps.  False where it has none.
template <int TOKENS>
__device__ bool kv4_start(const Kv4DecodeArgs& a, int heads_per_cta, Kv4Walk& w, int64_t& quota) {
  __shared__ int64_t s_sum[kKv4SplitThreads / 32];
  __shared__ Kv4Walk s_walk;
  const int nhb = a.hkv / heads_per_cta;
  if (a.whole) {  // whole sequences: no scan
    const int64_t n = a.batch * nhb;
    const int64_t first = blockIdx.x * n / gridDim.x, last = (blockIdx.x + 1) * n / gridDim.x;
    if (first >= last) return false;
    w.b = first / nhb;
    w.hb = (int)(first - w.b * nhb);
    w.pos = 0;
    w.ctx = kv4_ctx(a, w.b);
    w.steps = kv4_steps<TOKENS>(w.ctx);
    w.rest = 0;  // counted in steps: filled in below
    for (int64_t q = first; q < last; ++q) w.rest += kv4_steps<TOKENS>(q / nhb == w.b ? w.ctx : kv4_ctx(a, q / nhb));
    quota = 0;
    return true;
  }
  const int64_t per = (a.batch + kKv4SplitThreads - 1) / kKv4SplitThreads;
  const int64_t b0 = min(a.batch, per * threadIdx.x), b1 = min(a.batch, b0 + per);
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += (int64_t)nhb * kv4_steps<TOKENS>(kv4_ctx(a, b));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t scan = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan += up;
  }
  if (lane == 31) s_sum[warp] = scan;
  __syncthreads();
  int64_t total = 0, before = scan - mine;
  for (int i = 0; i < kKv4SplitThreads / 32; ++i) {
    if (i < warp) before += s_sum[i];
    total += s_sum[i];
  }
  quota = max((int64_t)a.min_steps, (total + gridDim.x - 1) / gridDim.x);
  const int64_t first = quota * blockIdx.x;
  if (first >= total) return false;
  if (first >= before && first < before + mine) {  // one thread's rows hold the start
    int64_t at = before;
    for (int64_t b = b0; b < b1; ++b) {
      const int ctx = kv4_ctx(a, b);
      const int steps = kv4_steps<TOKENS>(ctx);
      if (first < at + (int64_t)nhb * steps) {
        const int64_t in = first - at;
        s_walk.b = b;
        s_walk.rest = min(quota, total - first);
        s_walk.hb = (int)(in / steps);
        s_walk.pos = (int)(in - (int64_t)s_walk.hb * steps);
        s_walk.steps = steps;
        s_walk.ctx = ctx;
        break;
      }
      at += (int64_t)nhb * steps;
    }
  }
  __syncthreads();
  w = s_walk;
  return true;
}

// Four values of a row's sum, relative to ref, with the sum l of its weights: the output where this CTA had
// the whole sequence (slot < 0), else one of the CTA's two partials.
template <typename T, int D>
__device__ __forceinline__ void kv4_emit(const Kv4DecodeArgs& a, int64_t b, int hq, int slot, int row, int d,
                                         const float (&v)[4], float ref, float l, bool first) {
  if (slot < 0) {
    T* dst = reinterpret_cast<T*>(a.out + b * a.out_sb) + (int64_t)hq * D + d;
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = Elem<T>::from_f(v[i] * inv);
    return;
  }
  const int64_t idx = ((int64_t)blockIdx.x * 2 + slot) * a.part_rows + row;
  *reinterpret_cast<float4*>(a.ws_o + idx * D + d) = make_float4(v[0], v[1], v[2], v[3]);
  if (first) *reinterpret_cast<float2*>(a.ws_ml + idx * 2) = make_float2(ref, l);
}

template <typename T, int D, int BS, int HB, int SH>
__global__ void __launch_bounds__(kKv4SplitThreads, kKv4CtasPerSm) kv4_decode_split_kernel(const Kv4DecodeArgs a) {
  using S = Kv4Shape<D, BS, HB, SH>;
  constexpr int NG = S::kGroups;
  constexpr int NST = S::kStages;
  constexpr int PG = S::kPages;
  constexpr int UN = S::kUnits;
  constexpr int kCols = S::kCols;
  constexpr bool kTwo = std::is_same<T, __half>::value;  // p * s as two fp16 operands
  static_assert(NST >= 2, "a ring");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // programmatic dependent of the append
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  float* merge = reinterpret_cast<float*>(smem + NST * S::kStageBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + NST * S::kStageBytes + S::kMergeBytes);
  uint64_t* empty_bar = full_bar + NST;

  if (blockIdx.x == 0)
    for (int64_t b = threadIdx.x; b < a.batch; b += kKv4SplitThreads)
      if (a.context_lens[b] > a.max_blocks * a.block_size) record_status(MI_STATUS_BAD_LENGTH);
  Kv4Walk w;
  int64_t quota;
  if (threadIdx.x == 0) {
    if (a.cuts) a.cuts[blockIdx.x].pieces = 0;
    for (int i = 0; i < NST; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], kKv4Consumers);
    }
    fence_mbar_init();
  }
  if (!kv4_start<S::kTokens>(a, HB, w, quota)) return;  // uniform for the CTA
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int nhb = a.hkv / HB;
  bool aborted = false;
  int st = 0, phase = 0;  // of the ring

  if (warp == kKv4Consumers) {
    // ---------------- producer: lane 2p + kv copies K or V of page p of a step ----------------
    constexpr uint32_t kBytes = HB * S::kPageBytes;
    const int my_page = lane >> 1;
    const char* pool = (lane & 1) ? a.v_pool : a.k_pool;
    const int64_t block_bytes = (int64_t)a.hkv * S::kPageBytes;
    // Block ids come 32 pages at a time, one a lane, the next 32 (of the next sequence at the end of one)
    // loaded while these are used.
    static_assert(32 % PG == 0, "a step's pages lie in one window");
    auto ids_from = [&](int64_t b, int page) {
      return page + lane < a.max_blocks ? a.block_tables[b * a.table_stride + page + lane] : 0;
    };
    int64_t ids_next = ids_from(w.b, w.pos * PG);
    while (true) {
      const int n = w.take();
      const bool more = w.rest > n;
      const int64_t next_b = w.b + (w.hb + 1 == nhb);
      const int next_ctx = more ? (next_b != w.b ? kv4_ctx(a, next_b) : w.ctx) : 0;
      const int n_pages = (w.ctx + BS - 1) / BS;
      const int64_t head_off = (int64_t)w.hb * kBytes;
      int64_t ids = 0;
      for (int s = 0; s < n; ++s) {
        const int first = (w.pos + s) * PG;
        const int npg = min(PG, n_pages - first);
        const int in = s * PG % 32;
        if (in == 0) {
          ids = ids_next;
          if (s * PG + 32 < n * PG) ids_next = ids_from(w.b, first + 32);
          else if (more) ids_next = ids_from(next_b, 0);
        }
        int64_t blk = __shfl_sync(0xffffffffu, ids, in + (my_page < PG ? my_page : 0));
        if (npg <= 0) continue;  // a sequence of no tokens
        mbar_wait(&empty_bar[st], phase ^ 1, aborted);
        aborted = __any_sync(0xffffffffu, aborted);
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], (uint32_t)npg * 2 * kBytes);
        __syncwarp();
        if (my_page < npg) {
          if (blk < 0 || blk >= a.num_blocks) {
            record_status(MI_STATUS_BAD_BLOCK);
            blk = 0;  // the null block
          }
          bulk_load(smem + st * S::kStageBytes + lane * kBytes, pool + blk * block_bytes + head_off, kBytes,
                    &full_bar[st]);
        }
        if (++st == NST) st = 0, phase ^= 1;
      }
      if (!more) return;
      kv4_advance<S::kTokens>(a, w, HB, next_ctx);
    }
  }

  // ---------------- consumers: one warp per (KV head, unit of 32 tokens) ----------------
  const int hl = warp / UN;
  const int un = warp % UN;
  const int r = lane >> 2;  // MMA row (token or value) and, of a B operand, its column
  const int t = lane & 3;
  // rows of the 8x8 matrices: (token octet, 16 bytes of a group) x two groups
  const uint32_t mat_row = (uint32_t)(((lane >> 3) & 1) * 8 + (lane & 7) + (lane >> 4) * BS) * 16;
  constexpr uint32_t kPar = BS * D / 2;  // of a page
  const uint32_t k_off = (un * (kKv4Unit / BS) * 2 * HB + hl) * S::kPageBytes;
  // The unit's two tiles: tile i's K page and the token offset in it (V pages lie HB pages further); and
  // the tile of this lane's weights, which are one set of four for both tiles (SH = 2) or one for each.
  constexpr int kSets = 2 / SH;
  constexpr int kTilePage = BS == 16 ? 2 * HB * S::kPageBytes : 0;
  constexpr int kTileTok = BS == 16 ? 0 : 16;
  constexpr int kTileStep = kTilePage + kTileTok * 16;  // from a tile's codes to the next one's
  const int my_tile = SH == 2 ? t >> 1 : 0;
  const uint32_t my_par = my_tile * (kTilePage + kTileTok * NG * 4) + kPar + r * NG * 4;
  // SH = 2: ones in the columns of the first tile, and of the second.  Products rather than masks: the
  // ALU pipe, where the codes are cut, is the busiest.
  const __half2 ones[2] = {__float2half2_rn(r < 4 ? 1.f : 0.f), __float2half2_rn(r < 4 ? 0.f : 1.f)};
  auto masked = [&](uint32_t w, int i) {
    if constexpr (SH == 1) return w;
    const __half2 m = __hmul2(*reinterpret_cast<const __half2*>(&w), ones[i]);
    return *reinterpret_cast<const uint32_t*>(&m);
  };
  // -8 in place of the codes, in their units: 2^-24 for rows r, 2^-20 for rows r + 8
  constexpr uint32_t kEights[4] = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};

  // What a warp knows of its place is kept in shared memory: the loop over the tokens needs the registers.
  struct Place {
    Kv4Walk w;
    int64_t quota, done;  // done: steps of this CTA before the current sequence
    int next_ctx;
  };
  __shared__ Place s_place[kKv4Consumers];
  volatile Place& pl = s_place[warp];
  if (lane == 0) {
    Place first;
    first.w = w;
    first.quota = quota;
    first.done = 0;
    first.next_ctx = 0;
    s_place[warp] = first;
  }
  __syncwarp();

  while (true) {  // one sequence's share at a time
    const int n_steps = (int)min(pl.w.rest, (int64_t)(pl.w.steps - pl.w.pos));
    const int ctx = pl.w.ctx;
    if (lane == 0 && pl.w.rest > n_steps) pl.next_ctx = pl.w.hb + 1 == nhb ? kv4_ctx(a, pl.w.b + 1) : ctx;
    int left = min(ctx - pl.w.pos * S::kTokens, n_steps * S::kTokens) - un * kKv4Unit;  // tokens from this unit on

    // q as the B operand of S^T: this lane holds column r's values d = 32 g + 8 t + 0..7 of every group.
    // Column c is query head c % kCols; with SH = 2 the first four columns are for the first tile's
    // tokens, the last four for the second's.
    uint32_t qb[NG][4];
    uint32_t mb[3];  // B operands of the minimum term, see below
    float unit[2];   // what one unit of q * (code operand) stands for, times the softmax scale: columns 2t, 2t + 1
    {
      float qv[NG][8], qsum[NG];
      const bool valid = r % kCols < a.groups;
      const T* qp =
          reinterpret_cast<const T*>(a.q + pl.w.b * a.q_sb +
                                     (int64_t)((pl.w.hb * HB + hl) * a.groups + (valid ? r % kCols : 0)) * a.q_sh);
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        qsum[g] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          qv[g][i] = valid ? Elem<T>::to_f(qp[g * kKv4Group + t * 8 + i]) : 0.f;
          top = fmaxf(top, fabsf(qv[g][i]));
          qsum[g] += qv[g][i];
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);  // 2^e <= top < 2^(e+1)
      const float up = pow2(14 - e);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 1);
        qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 2);
        qsum[g] *= a.scale_log2;
        float u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = qv[g][i] * up * ((i & 1) ? 0.0625f : 1.f);
        qb[g][0] = pack2<__half>(u[0], u[4]);
        qb[g][1] = pack2<__half>(u[1], u[5]);
        qb[g][2] = pack2<__half>(u[2], u[6]);
        qb[g][3] = pack2<__half>(u[3], u[7]);
      }
      // The minimum term sum_g m_g sum(q_g) as a bf16 MMA on the parameter words themselves: columns 2t
      // and 2t + 1 of a token's row are (s, m) of group t % NG.  The steps meet zeros; sum(q_g) enters
      // as three bfloat16s, 24 bits of it: in k 2t + 1, in k 2t + 9 and in a second MMA (NG = 4), or in
      // k 2t + 1 of both pairs of lanes and in k 2t + 9 (NG = 2).
      float mine = qsum[0];
#pragma unroll
      for (int g = 1; g < NG; ++g) mine = (t % NG) == g ? qsum[g] : mine;
      uint32_t part[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        part[i] = bf16_bits(mine);
        mine -= __uint_as_float(part[i] << 16);
      }
      if constexpr (NG == 4) {
        mb[0] = part[0] << 16, mb[1] = part[1] << 16, mb[2] = part[2] << 16;
      } else {
        mb[0] = (t < 2 ? part[0] : part[1]) << 16, mb[1] = t < 2 ? part[2] << 16 : 0u, mb[2] = 0u;
      }
      const float mine_unit = a.scale_log2 * pow2(e) * 1024.f;  // 2^(e - 14) of q, 2^24 of the codes
      unit[0] = __shfl_sync(0xffffffffu, mine_unit, 8 * t);  // accumulator columns 2t, 2t + 1
      unit[1] = __shfl_sync(0xffffffffu, mine_unit, 8 * t + 4);
    }

    float o[D / 16][4];  // O^T less z: rows are values, columns 2t, 2t + 1
    float z[NG][2];      // sum p (m + 8 s) of this lane's tokens
    float l[2] = {0.f, 0.f};
    float ref[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) z[g][0] = z[g][1] = 0.f;

    for (int it = ctx > 0 ? n_steps : 0; it > 0; --it, left -= S::kTokens) {
      mbar_wait(&full_bar[st], phase, aborted);
      if (left > 0) {
        const uint8_t* k_unit = smem + st * S::kStageBytes + k_off;
        const uint32_t k_mat = smem_u32(k_unit) + mat_row;
        // V's matrices: as K's, or (SH = 2) the token octets of one group in both tiles
        const uint32_t v_mat = k_mat + HB * S::kPageBytes + (SH == 1 ? 0 : (lane >> 4) * (kTileStep - BS * 16));
        const bool tail = left < kKv4Unit;  // nothing past the sequence's end counts, whatever the pages hold there
#pragma unroll 1  // unrolled, the second set's loads come forward and spill 200 bytes
        for (int n = 0; n < kSets; ++n) {
          // ---- scores: x[0..1] token r, x[2..3] token r + 8 of the set's tile; columns 2t, 2t + 1 ----
          float x[4], wide[2];
          const uint8_t* k_par = k_unit + my_par + n * (kTilePage + kTileTok * NG * 4);
          uint32_t kw[2][NG];
          kv4_params<NG>(k_par, kw[0]);
          kv4_params<NG>(k_par + 8 * NG * 4, kw[1]);
          float y[4], s[4];
#pragma unroll
          for (int i = 0; i < SH; ++i) {  // the minimum term
            const uint8_t* par = k_unit + (n + i) * (kTilePage + kTileTok * NG * 4) + kPar + (r * NG + t % NG) * 4;
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(par);
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(par + 8 * NG * 4);
            const uint32_t both[4] = {w0, w1, w0, w1}, once[4] = {w0, w1, 0u, 0u};
            float u[4];
            Mma16816<__nv_bfloat16>::zero(u, both, mb[0], mb[1]);
            if constexpr (NG == 4) Mma16816<__nv_bfloat16>::run(u, once, mb[2], 0u);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = i && my_tile == 0 ? y[j] : u[j];
          }
#pragma unroll
          for (int gp = 0; gp < NG / 2; ++gp) {
            float acc[2][4];
#pragma unroll
            for (int i = 0; i < SH; ++i) {
              uint32_t c[4];
              ldmatrix_x4(k_mat + (n + i) * (kTilePage + kTileTok * 16) + gp * 2 * BS * 16, c[0], c[1], c[2], c[3]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t lo[4], hi[4];
                kv4_operands(c[2 * j], lo);
                kv4_operands(c[2 * j + 1], hi);
                const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]};
                const uint32_t a1[4] = {lo[2], hi[2], lo[3], hi[3]};
                float u[4];
                Mma16816<__half>::zero(u, a0, qb[gp * 2 + j][0], qb[gp * 2 + j][1]);
                Mma16816<__half>::run(u, a1, qb[gp * 2 + j][2], qb[gp * 2 + j][3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][e] = i && my_tile == 0 ? acc[j][e] : u[e];
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int g = gp * 2 + j;
              const float s0 = kv4_step(kw[0][g]), s1 = kv4_step(kw[1][g]);
              s[0] = g ? fmaf(acc[j][0], s0, s[0]) : acc[j][0] * s0;
              s[1] = g ? fmaf(acc[j][1], s0, s[1]) : acc[j][1] * s0;
              s[2] = g ? fmaf(acc[j][2], s1, s[2]) : acc[j][2] * s1;
              s[3] = g ? fmaf(acc[j][3], s1, s[3]) : acc[j][3] * s1;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = fmaf(s[j], unit[j & 1], y[j]);
          // widest step of each token (positive bfloat16s order as integers)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t vw[NG];
            kv4_params<NG>(k_par + HB * S::kPageBytes + j * 8 * NG * 4, vw);
            uint32_t w = vw[0];
#pragma unroll
            for (int g = 1; g < NG; ++g) w = __vmaxu2(w, vw[g]);
            wide[j] = fmaxf(kv4_step(w), kKv4Narrow);
          }
          if (tail) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if ((n + my_tile) * 16 + j * 8 + r >= left) {
                x[2 * j] = x[2 * j + 1] = -INFINITY;
                wide[j] = kKv4Narrow;
              }
          }
          // ---- weights p = 2^(x - ref).  A reference moves only when some p * s would leave fp16's range:
          // then to where the largest p * s of these tokens is 2^11 ----
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = ex2_approx(x[j] - ref[j & 1]);
          const float most = fmaxf(fmaxf(p[0], p[1]) * wide[0], fmaxf(p[2], p[3]) * wide[1]);
          if (__any_sync(0xffffffffu, most > kKv4Limit)) {
            const float wl[2] = {log2f(wide[0]) - kKv4TopLog2, log2f(wide[1]) - kKv4TopLog2};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float want = fmaxf(x[c] + wl[0], x[c + 2] + wl[1]);
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) want = fmaxf(want, __shfl_xor_sync(0xffffffffu, want, off));
              want = fmaxf(want, ref[c]);
              const float base = want == -INFINITY ? 0.f : want;
              const float alpha = ex2_approx(ref[c] - base);  // 0 from the initial -inf
              l[c] *= alpha;
#pragma unroll
              for (int g = 0; g < NG; ++g) z[g][c] *= alpha;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                o[i][c] *= alpha;
                o[i][c + 2] *= alpha;
              }
              p[c] = ex2_approx(x[c] - base);
              p[c + 2] = ex2_approx(x[c + 2] - base);
              ref[c] = want;
            }
          }
          // ---- O^T += (V^T - 8) (p s)^T, z += p (m + 8 s) ----
          l[0] += p[0] + p[2];
          l[1] += p[1] + p[3];
          const uint8_t* v_par = k_unit + my_par + n * (kTilePage + kTileTok * NG * 4) + HB * S::kPageBytes;
          uint32_t vw[2][NG];
          kv4_params<NG>(v_par, vw[0]);
          kv4_params<NG>(v_par + 8 * NG * 4, vw[1]);
          if (tail) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if ((n + my_tile) * 16 + j * 8 + r >= left) {
#pragma unroll
                for (int g = 0; g < NG; ++g) vw[j][g] = 0u;
              }
          }
#pragma unroll
          for (int gp = 0; gp < NG / 2; ++gp) {
            uint32_t c[4];  // codes: SH = 1 of both groups, SH = 2 of one group of both tiles
            if constexpr (SH == 1) ldmatrix_x4_trans(v_mat + n * kTileStep + gp * 2 * BS * 16, c[0], c[1], c[2], c[3]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int g = gp * 2 + j;
              const float s0 = kv4_step(vw[0][g]), s1 = kv4_step(vw[1][g]);
              // the value of code 8, the codes' middle
              const float m0 = fmaf(8.f, s0, kv4_min(vw[0][g])), m1 = fmaf(8.f, s1, kv4_min(vw[1][g]));
              z[g][0] = fmaf(p[2], m1, fmaf(p[0], m0, z[g][0]));
              z[g][1] = fmaf(p[3], m1, fmaf(p[1], m0, z[g][1]));
              const float f[4] = {p[0] * s0, p[1] * s0, p[2] * s1, p[3] * s1};
              const uint32_t h0 = pack2<__half>(f[0], f[1]), h1 = pack2<__half>(f[2], f[3]);
              uint32_t pb[2], rest[2];  // p s as a B operand, and what fp16 left of it
              pb[0] = movmatrix_trans(h0);
              pb[1] = movmatrix_trans(h1);
              if constexpr (kTwo) {
                const float2 g0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                const float2 g1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                rest[0] = movmatrix_trans(pack2<__half>(f[0] - g0.x, f[1] - g0.y));
                rest[1] = movmatrix_trans(pack2<__half>(f[2] - g1.x, f[3] - g1.y));
              }
              if constexpr (SH == 2) ldmatrix_x4_trans(v_mat + g * BS * 16, c[0], c[1], c[2], c[3]);
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                // sum (c - 8) p s of these tokens, the remainders first; added to O with a rounding
                float u[4];
                uint32_t cd[SH][4];
#pragma unroll
                for (int i = 0; i < SH; ++i) {
                  const int w = SH == 1 ? 2 * j : 2 * i;
                  const uint32_t lo = half ? c[w] >> 8 : c[w], hi = half ? c[w + 1] >> 8 : c[w + 1];
                  if constexpr (kTwo) {
                    cd[i][0] = kv4_centred((lo & 0x000f000fu) | 0x64006400u, 1032.f);
                    cd[i][1] = kv4_centred((lo & 0x00f000f0u) | 0x54005400u, 72.f);
                    cd[i][2] = kv4_centred((hi & 0x000f000fu) | 0x64006400u, 1032.f);
                    cd[i][3] = kv4_centred((hi & 0x00f000f0u) | 0x54005400u, 72.f);
                  } else {
                    cd[i][0] = lo & 0x000f000fu, cd[i][1] = lo & 0x00f000f0u;
                    cd[i][2] = hi & 0x000f000fu, cd[i][3] = hi & 0x00f000f0u;
                  }
                }
                if constexpr (kTwo) {
                  Mma16816<__half>::zero(u, cd[0], masked(rest[0], 0), masked(rest[1], 0));
                  if constexpr (SH == 2) Mma16816<__half>::run(u, cd[SH - 1], masked(rest[0], 1), masked(rest[1], 1));
                } else {
                  Mma16816<__half>::zero(u, kEights, pb[0], pb[1]);
                }
#pragma unroll
                for (int i = 0; i < SH; ++i) Mma16816<__half>::run(u, cd[i], masked(pb[0], i), masked(pb[1], i));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[2 * g + half][e] += u[e];
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[st]);
      if (++st == NST) st = 0, phase ^= 1;
    }

    if constexpr (SH == 2) {
      // a head's sums over the first and the second tiles meet: columns 2t and 2t + 4
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float other = __shfl_xor_sync(0xffffffffu, ref[c], 2);
        const float both = fmaxf(ref[c], other);
        const float alpha = both == -INFINITY ? 1.f : ex2_approx(ref[c] - both);
        ref[c] = both;
        l[c] *= alpha;
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 2);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          z[g][c] *= alpha;
          z[g][c] += __shfl_xor_sync(0xffffffffu, z[g][c], 2);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          o[i][c] *= alpha;
          o[i][c] += __shfl_xor_sync(0xffffffffu, o[i][c], 2);
          o[i][c + 2] *= alpha;
          o[i][c + 2] += __shfl_xor_sync(0xffffffffu, o[i][c + 2], 2);
        }
      }
    }
    // ---- this warp's sums over the lanes that share columns, then its rows: heads 2t, 2t + 1, values
    // d = 32 g + 4 r + 0..3 (rows r of tile 2g, r + 8 of it, times 16, and of tile 2g + 1) ----
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], off);
#pragma unroll
        for (int g = 0; g < NG; ++g) z[g][c] += __shfl_xor_sync(0xffffffffu, z[g][c], off);
      }
    }
    auto value = [&](int g, int c, int i) {
      return fmaf(o[2 * g + (i >> 1)][c + (i & 1) * 2], kTwo ? 1.f : i & 1 ? 0x1p20f : 0x1p24f, z[g][c]);
    };
    // The rows' outputs where all of the sequence was here, else a partial: slot 0 the CTA's first, 1 its last.
    const int64_t b = pl.w.b;
    const int hb = pl.w.hb, pos = pl.w.pos, steps = pl.w.steps;
    const int taken = (int)min(pl.w.rest, (int64_t)(steps - pos));
    const int head0 = hb * HB;
    const int slot = pos == 0 && taken == steps ? -1 : pl.done > 0;
    if (slot >= 0 && pos == 0 && threadIdx.x == 0) {  // the sequence starts here and is cut: say how often
      Kv4Cut cut;
      cut.b = b;
      cut.hb = hb;
      cut.slot = slot;
      const int64_t at = blockIdx.x * pl.quota + pl.done;
      cut.pieces = (int)((at + steps - 1) / pl.quota - blockIdx.x) + 1;
      a.cuts[blockIdx.x] = cut;
    }
    if (pl.w.ctx == 0) {  // a row of no tokens
      for (int i = threadIdx.x; i < HB * a.groups * D; i += kKv4Consumers * 32)
        reinterpret_cast<T*>(a.out + b * a.out_sb)[(int64_t)head0 * a.groups * D + i] = Elem<T>::from_f(0.f);
    } else if constexpr (UN > 1) {
      // the warps of a KV head merge in shared memory
      float* so = merge;                             // [warp][column][D]
      float* sml = so + kKv4Consumers * kCols * D;   // [warp][column](ref, l)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = warp * kCols + 2 * t + c;
        if (2 * t + c >= kCols) continue;
#pragma unroll
        for (int g = 0; g < NG; ++g)
          *reinterpret_cast<float4*>(so + col * D + g * kKv4Group + r * 4) =
              make_float4(value(g, c, 0), value(g, c, 1), value(g, c, 2), value(g, c, 3));
        if (r == 0) *reinterpret_cast<float2*>(sml + 2 * col) = make_float2(ref[c], l[c]);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kKv4Consumers * 32) : "memory");
      // four values of one (KV head, query head) at a time
      constexpr int kVec = D / 4;
      for (int i = threadIdx.x; i < HB * a.groups * kVec; i += kKv4Consumers * 32) {
        const int row = i / kVec, d = (i - row * kVec) * 4;
        const int hm = row / a.groups, head = row - hm * a.groups;
        float m_all = -INFINITY;
#pragma unroll
        for (int u = 0; u < UN; ++u) m_all = fmaxf(m_all, sml[2 * ((hm * UN + u) * kCols + head)]);
        float l_all = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int col = (hm * UN + u) * kCols + head;
          const float f = m_all == -INFINITY ? 1.f : ex2_approx(sml[2 * col] - m_all);
          l_all = fmaf(f, sml[2 * col + 1], l_all);
          const float4 x = *reinterpret_cast<const float4*>(so + col * D + d);
          v[0] = fmaf(f, x.x, v[0]), v[1] = fmaf(f, x.y, v[1]), v[2] = fmaf(f, x.z, v[2]), v[3] = fmaf(f, x.w, v[3]);
        }
        kv4_emit<T, D>(a, b, (head0 + hm) * a.groups + head, slot, row, d, v, m_all, l_all, d == 0);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kKv4Consumers * 32) : "memory");  // before the next sequence's sums
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int head = 2 * t + c;
        if (head >= kCols || head >= a.groups) continue;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float v[4] = {value(g, c, 0), value(g, c, 1), value(g, c, 2), value(g, c, 3)};
          kv4_emit<T, D>(a, b, (head0 + hl) * a.groups + head, slot, hl * a.groups + head, g * kKv4Group + r * 4, v, ref[c], l[c],
                         g == 0 && r == 0);
        }
      }
    }
    if (pl.w.rest <= taken) return;
    __syncwarp();
    if (lane == 0) {
      pl.done = pl.done + taken;
      pl.w.rest = pl.w.rest - taken;
      pl.w.pos = 0;
      const bool row_done = hb + 1 == nhb;
      pl.w.hb = row_done ? 0 : hb + 1;
      if (row_done) {
        pl.w.b = b + 1;
        pl.w.ctx = pl.next_ctx;
        pl.w.steps = kv4_steps<S::kTokens>(pl.next_ctx);
      }
    }
    __syncwarp();
  }
}

// Merges the partials of the sequence that CTA blockIdx.x of the split kernel started and did not finish:
// WPR warps a row, each over every WPR-th piece, lanes over values.  One warp a row where sequences are
// cut a few times (the chain of dependent loads is what costs: 3 us), eight where they are cut often.
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(256) kv4_combine_kernel(const Kv4DecodeArgs a) {
  constexpr int PER = D / 32;
  using Vec = typename std::conditional<PER == 4, float4, float2>::type;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // programmatic dependent of the split kernel
  const Kv4Cut cut = a.cuts[blockIdx.x];
  if (cut.pieces == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % WPR;
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml);
  __shared__ float sa[8][D + 2];
  for (int row = blockIdx.y * (8 / WPR) + warp / WPR; row < a.part_rows; row += gridDim.y * (8 / WPR)) {
    // piece i: CTA blockIdx.x + i, in its first slot but for the first piece
    const int64_t first = ((int64_t)blockIdx.x * 2 + cut.slot) * a.part_rows + row;
    const int64_t second = ((int64_t)blockIdx.x * 2 + 2) * a.part_rows + row;
    auto at = [&](int i) { return i == 0 ? first : second + (int64_t)(i - 1) * 2 * a.part_rows; };
    float m_all = -INFINITY, acc[PER], l = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (int i0 = part; i0 < cut.pieces; i0 += 4 * WPR) {  // four pieces' loads at once, then their sums
      float2 x[4];
      Vec v[4];
      float m_new = m_all;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * WPR;
        x[k] = i < cut.pieces ? ml[at(i)] : make_float2(-INFINITY, 0.f);
        v[k] = i < cut.pieces ? *reinterpret_cast<const Vec*>(a.ws_o + at(i) * D + lane * PER) : Vec{};
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) m_new = fmaxf(m_new, x[k].x);
      const float keep = m_new == -INFINITY ? 1.f : ex2_approx(m_all - m_new);
      m_all = m_new;
      l *= keep;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] *= keep;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = m_new == -INFINITY ? 1.f : ex2_approx(x[k].x - m_new);
        l = fmaf(f, x[k].y, l);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = fmaf(f, reinterpret_cast<const float*>(&v[k])[e], acc[e]);
      }
    }
    if constexpr (WPR > 1) {  // one row a CTA: the loop runs once
#pragma unroll
      for (int e = 0; e < PER; ++e) sa[warp][lane * PER + e] = acc[e];
      if (lane == 0) {
        sa[warp][D] = l;
        sa[warp][D + 1] = m_all;
      }
      __syncthreads();
      if (part != 0) return;
      m_all = sa[0][D + 1];
#pragma unroll
      for (int i = 1; i < WPR; ++i) m_all = fmaxf(m_all, sa[i][D + 1]);
      l = 0.f;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        const float f = m_all == -INFINITY ? 1.f : ex2_approx(sa[i][D + 1] - m_all);
        l = fmaf(f, sa[i][D], l);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = fmaf(f, sa[i][lane * PER + e], acc[e]);
      }
    }
    T* dst = reinterpret_cast<T*>(a.out + cut.b * a.out_sb) + ((int64_t)cut.hb * a.part_rows + row) * D + lane * PER;
    const float inv = 1.f / l;
#pragma unroll
    for (int e = 0; e < PER; ++e) dst[e] = Elem<T>::from_f(acc[e] * inv);
  }
}

template <typename T, int D, int BS, int HB, int SH>
cudaError_t launch_kv4_split(const Kv4DecodeArgs& a, cudaStream_t s) {
  using S = Kv4Shape<D, BS, HB, SH>;
  auto kern = kv4_decode_split_kernel<T, D, BS, HB, SH>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.ctas);
  cfg.blockDim = dim3(kKv4SplitThreads);
  cfg.dynamicSmemBytes = S::kSmemBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess || a.whole) return e;
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  if (a.ctas > 16 * a.batch * (a.hkv / HB)) {
    cfg.gridDim = dim3((unsigned)a.ctas, (unsigned)a.part_rows);
    return cudaLaunchKernelEx(&cfg, kv4_combine_kernel<T, D, 8>, a);
  }
  cfg.gridDim = dim3((unsigned)a.ctas, (unsigned)((a.part_rows + 7) / 8));
  return cudaLaunchKernelEx(&cfg, kv4_combine_kernel<T, D, 1>, a);
}

template <typename T, int D, int BS>
cudaError_t launch_kv4_split_hb(const Kv4DecodeArgs& a, int hb, cudaStream_t s) {
  switch (hb) {
    case 4: return a.groups <= 4 ? launch_kv4_split<T, D, BS, 4, 2>(a, s) : launch_kv4_split<T, D, BS, 4, 1>(a, s);
    case 2: return a.groups <= 4 ? launch_kv4_split<T, D, BS, 2, 2>(a, s) : launch_kv4_split<T, D, BS, 2, 1>(a, s);
    default: return a.groups <= 4 ? launch_kv4_split<T, D, BS, 1, 2>(a, s) : launch_kv4_split<T, D, BS, 1, 1>(a, s);
  }
}

template <typename T>
cudaError_t launch_kv4_split_t(const Kv4DecodeArgs& a, int hb, cudaStream_t s) {
  if (a.head_dim == 128)
    return a.block_size == 16 ? launch_kv4_split_hb<T, 128, 16>(a, hb, s) : launch_kv4_split_hb<T, 128, 32>(a, hb, s);
  return a.block_size == 16 ? launch_kv4_split_hb<T, 64, 16>(a, hb, s) : launch_kv4_split_hb<T, 64, 32>(a, hb, s);
}

}  // namespace

Kv4DecodePlan plan_kv4_decode(int64_t batch, int hq, int hkv, int head_dim, int64_t max_blocks, int block_size,
                              int dtype) {
  Kv4DecodePlan p{};
  const int groups = hq / hkv;
  p.use_mma = (dtype == MI_BF16 || dtype == MI_F16) && (head_dim == 64 || head_dim == 128) &&
              (block_size == 16 || block_size == 32) && groups >= 1 && groups <= 8;
  if (!p.use_mma) return p;
  p.heads_per_cta = (hkv % 4 == 0) ? 4 : (hkv % 2 == 0) ? 2 : 1;
  const int64_t step_tokens = kKv4Consumers / p.heads_per_cta * kKv4Unit;
  const int64_t sequences = batch * (hkv / p.heads_per_cta);
  const int64_t steps = (max_blocks * block_size + step_tokens - 1) / step_tokens;  // of the longest sequence, at most
  const int64_t ctas = 148 * kKv4CtasPerSm;
  p.part_rows = p.heads_per_cta * groups;
  p.min_steps = kKv4MinSteps;
  p.whole = steps <= kKv4WholeSteps;
  p.ctas = (int)std::min<int64_t>(ctas, p.whole ? sequences : (sequences * steps + p.min_steps - 1) / p.min_steps);
  if (p.whole) return p;
  const size_t rows = (size_t)p.ctas * 2 * p.part_rows;
  p.o_bytes = (rows * head_dim * sizeof(float) + 255) & ~size_t(255);
  p.ml_bytes = (rows * 2 * sizeof(float) + 255) & ~size_t(255);
  p.ws_bytes = p.o_bytes + p.ml_bytes + (((size_t)p.ctas * sizeof(Kv4Cut) + 255) & ~size_t(255));
  return p;
}

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, const Kv4DecodePlan& plan, int dtype, cudaStream_t s) {
  if (plan.use_mma) {
    if (dtype == MI_BF16) return launch_kv4_split_t<__nv_bfloat16>(a, plan.heads_per_cta, s);
    return launch_kv4_split_t<__half>(a, plan.heads_per_cta, s);
  }
  const unsigned grid = (unsigned)(a.batch * a.hq);
  if (dtype == MI_BF16) kv4_decode_generic_kernel<__nv_bfloat16><<<grid, kKv4Warps * 32, 0, s>>>(a);
  else if (dtype == MI_F16) kv4_decode_generic_kernel<__half><<<grid, kKv4Warps * 32, 0, s>>>(a);
  else kv4_decode_generic_kernel<float><<<grid, kKv4Warps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mi

// Attention over a packed row of documents (gfx950): forward, and the two
// kernels of its backward.
//
// Rows are tokens; documents [ds, de) follow one another, each with a prefix
// end pe in [ds, de].  Key j is seen by query i of the same document when
// (j <= i or j < pe) and i - j < window.  For a fixed query these keys are one
// range [lo, hi), for a fixed key these queries are one range, and both ends
// grow with the row, so a tile's masks are two comparisons per element, needed
// only in blocks that a range's end crosses.
//
//   z_ij = scale q_i . k_j, then cap tanh(z_ij / cap) with a softcap
//   p_ij = exp(z_ij - lse_i),  o_i = sum_j p_ij v_j
//   delta_i = sum_d do_id o_id,  ds_ij = p_ij (do_i . v_j - delta_i) z'_ij
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// where z' = scale, times 1 - (z / cap)^2 with a softcap.
//
// A workgroup owns kAttnRows rows of one document and one head (backward of
// keys: one key head and its query heads one after the other), so that no value
// of another document, and none behind the last one, enters its products.
//
// Every product is a 32 x 32 MFMA arranged so that its left operand comes from
// an LDS tile and the softmax stays in registers: with the scores transposed
// (keys down, the wave's 32 queries across) a lane holds 16 keys of one query,
// which is the layout the next product wants its right operand in -- the order
// of the summed index differs, and the left operand is read from LDS in the
// same order.  Sums are fp32.  P and dS are rounded to the inputs' type before
// their products, since only then these run on the bf16 matrix instructions (at
// most 2^-8 of each term; the fp32 ones have a sixteenth of their rate); the row sums of P
// are taken before that rounding, and delta from O before its own (attn_store_out).
#pragma once

#include <type_traits>

#include "flce_device.h"

namespace mtf {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kAttnRows = 128;    // rows of a workgroup: 4 waves of 32
constexpr int kAttnThreads = 256;
constexpr float kAttnLowest = -3.402823466e38f;  // a maximum before any score: no finite one lies below
constexpr int kPlanHeader = 16;   // int32 words before the plan's tiles
constexpr int kPlanTile = 8;
constexpr int kPlanBuckets = 1024;

// One tile of the plan.  For a query tile [beg, end) are the keys its rows see,
// for a key tile the queries that see its rows.  tail: rows behind the last
// document, whose results are zeros.
struct AttnTile {
  int32_t row0, rows, ds, de, pe, beg, end, tail;
};

__device__ __forceinline__ int32_t attn_row_lo(int32_t i, int32_t ds, int32_t w) {
  return max(ds, i - w + 1);
}
__device__ __forceinline__ int32_t attn_row_hi(int32_t i, int32_t pe) { return max(i + 1, pe); }
__device__ __forceinline__ int32_t attn_col_lo(int32_t j, int32_t ds, int32_t pe) {
  return j < pe ? ds : j;
}
__device__ __forceinline__ int32_t attn_col_hi(int32_t j, int32_t de, int32_t w) {
  return j > de - w ? de : j + w;
}

// Blocks of 64 rows that a tile visits.
__device__ __forceinline__ int32_t attn_cost(const AttnTile& t) { return (t.end - t.beg + 63) >> 6; }

// The plan: tiles of every document and of the rows behind the last one, the
// costliest first (counting sort by the blocks a tile visits), so that the
// workgroups dispatched last are the short ones.  One workgroup, bound by the chain
// of its steps: 6.3 us for 4096 tokens in 12 documents, 7.2 for 32768 in 64 (with the
// sum and the maximum of the costs by LDS atomics on one word 8.5 and 11.4).
//   plan: kPlanHeader words ([0] = tiles, [1] = the key tiles'
//   cost, [2] = the costliest one's), tiles_max query tiles, tiles_max key
//   tiles, S + 2 words of scratch.  status: 0, or 1 for cu_seqlens that are not
//   0 = cu[0] <= ... <= cu[S] <= T, or 2 for a prefix outside its document; the
//   plan of such a call is one tail over all T rows (status 1) or clamps the
//   prefix (status 2), so that no kernel reads out of range.
__global__ __launch_bounds__(1024) void attn_plan_kernel(const int32_t* cu, const int32_t* prefix,
                                                         int32_t S, int32_t T, int32_t window,
                                                         int32_t tiles_max, int32_t* plan,
                                                         int32_t* status) {
  __shared__ int32_t hist[2][kPlanBuckets];
  __shared__ int32_t wave_sum[16];
  __shared__ int32_t bad, bad_prefix, most;
  __shared__ unsigned long long total;
  const int32_t tid = threadIdx.x;
  AttnTile* qt = reinterpret_cast<AttnTile*>(plan + kPlanHeader);
  AttnTile* kt = qt + tiles_max;
  int32_t* off = reinterpret_cast<int32_t*>(kt + tiles_max);
  if (tid == 0) bad = cu[0] != 0 || cu[S] > T || cu[S] < 0, bad_prefix = most = 0, total = 0;
  hist[0][tid] = hist[1][tid] = 0;
  __syncthreads();
  for (int32_t s = tid; s < S; s += 1024) {
    const int32_t a = cu[s], b = cu[s + 1];
    if (b < a) atomicOr(&bad, 1);
    if (prefix && (prefix[s] < 0 || prefix[s] > b - a)) atomicOr(&bad_prefix, 1);
  }
  __syncthreads();
  const bool broken = bad != 0;
  const int32_t end = broken ? 0 : cu[S];
  if (tid == 0) *status = broken ? 1 : (bad_prefix ? 2 : 0);
  // off[s] = first tile of document s (s == S: of the tail), off[S + 1] = tiles
  int32_t base = 0;
  for (int64_t s0 = 0; s0 <= S; s0 += 1024) {
    const int64_t s = s0 + tid;
    int32_t n = 0;
    if (s < S && !broken) n = (cu[s + 1] - cu[s] + kAttnRows - 1) / kAttnRows;
    if (s == S) n = (T - end + kAttnRows - 1) / kAttnRows;
    int32_t x = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t y = __shfl_up(x, d);
      if ((tid & 63) >= d) x += y;
    }
    if ((tid & 63) == 63) wave_sum[tid >> 6] = x;
    __syncthreads();
    int32_t before = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < (tid >> 6)) before += wave_sum[w];
      all += wave_sum[w];
    }
    if (s <= S) off[s] = before + x - n;
    base += all;
    __syncthreads();
  }
  const int32_t tiles = base;
  if (tid == 0) plan[0] = tiles;
  __threadfence_block();
  __syncthreads();
  // twice over the tiles: their costs' histogram, then their places
  unsigned long long my_total = 0;
  int32_t my_most = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int32_t t = tid; t < tiles; t += 1024) {
      int32_t a = 0, b = S;  // the last document whose first tile is <= t
      while (a < b) {
        const int32_t m = a + (b - a + 1) / 2;
        if (off[m] <= t) a = m; else b = m - 1;
      }
      AttnTile q;
      q.tail = a == S;
      q.ds = q.tail ? end : cu[a];
      q.de = q.tail ? T : cu[a + 1];
      q.row0 = q.ds + (t - off[a]) * kAttnRows;
      q.rows = min(kAttnRows, q.de - q.row0);
      q.pe = q.ds;
      if (prefix && !q.tail) q.pe = q.ds + min(max(prefix[a], 0), q.de - q.ds);
      AttnTile k = q;
      const int32_t last = q.row0 + q.rows - 1;
      q.beg = q.tail ? 0 : attn_row_lo(q.row0, q.ds, window);
      q.end = q.tail ? 0 : attn_row_hi(last, q.pe);
      k.beg = k.tail ? 0 : attn_col_lo(k.row0, k.ds, k.pe);
      k.end = k.tail ? 0 : attn_col_hi(last, k.de, window);
      const int32_t cq = min(kPlanBuckets - 1, attn_cost(q));
      const int32_t ck = min(kPlanBuckets - 1, attn_cost(k));
      if (pass == 0) {
        my_total += (unsigned long long)attn_cost(k);
        my_most = max(my_most, attn_cost(k));
        atomicAdd(&hist[0][cq], 1);
        atomicAdd(&hist[1][ck], 1);
      } else {  // (the order within a bucket changes no result)
        qt[atomicAdd(&hist[0][cq], 1)] = q;
        kt[atomicAdd(&hist[1][ck], 1)] = k;
      }
    }
    if (pass == 0 && (tid & ~63) < tiles) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        my_total += __shfl_xor(my_total, d);
        my_most = max(my_most, __shfl_xor(my_most, d));
      }
      if ((tid & 63) == 0) {
        atomicAdd(&total, my_total);
        atomicMax(&most, my_most);
      }
    }
    __syncthreads();
    if (pass == 0) {  // hist[b] -> tiles in the costlier buckets
      if (tid == 0) plan[1] = (int32_t)min(total, 0x7fffffffull), plan[2] = most;
      for (int which = 0; which < 2; ++which) {
        const int32_t bucket = kPlanBuckets - 1 - tid;
        const int32_t n = hist[which][bucket];
        int32_t x = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int32_t y = __shfl_up(x, d);
          if ((tid & 63) >= d) x += y;
        }
        if ((tid & 63) == 63) wave_sum[tid >> 6] = x;
        __syncthreads();
        for (int w = 0; w < (tid >> 6); ++w) x += wave_sum[w];
        hist[which][bucket] = x - n;
        __syncthreads();
      }
    }
  }
}

// --- tiles, fragments, products -------------------------------------------

// An LDS tile of rows of DP elements in 16-byte chunks, the chunk index XORed
// with a permutation of the row's low bits: 16 consecutive rows of one chunk
// (the row fragments) lie in distinct 16-byte slots of a 256-byte window, and
// so do the pieces that four consecutive rows (bf16: a transposing read of a
// half wave) or rows four apart (fp32: a wave's column read) contribute.
template <class T, int DP>
struct AttnLds {
  static constexpr uint32_t kRowB = DP * sizeof(T);
  static constexpr uint32_t kCh = kRowB / 16;
  __device__ __forceinline__ static uint32_t swz(uint32_t row) {
    if constexpr (sizeof(T) == 4)
      return (((row >> 2) & 1u) << 3) | (((row >> 3) & 1u) << 2) | (row & 3u);
    else if constexpr (DP == 64)
      return (((row >> 1) & 1u) << 2) | ((row >> 2) & 3u);
    else
      return ((row & 3u) << 2) | ((row >> 2) & 3u);
  }
  __device__ __forceinline__ static uint32_t off(uint32_t row, uint32_t chunk) {
    return row * kRowB + ((chunk ^ swz(row)) << 4);
  }
};

typedef __amdgpu_buffer_rsrc_t attn_rsrc_t;

__device__ __forceinline__ attn_rsrc_t attn_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4_t attn_load16(attn_rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}
__device__ __forceinline__ void attn_store16(u32x4_t v, attn_rsrc_t r, uint32_t off) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0);
}

constexpr uint32_t kAttnOut = 0xfffffff0u;  // an offset past every resource: loads give 0, stores are dropped

// The rows that a lane keeps in registers as the right operand of a product
// over d: row (l & 31) of the wave, half of d by l >> 5.
template <class T, int DP>
struct AttnFrag {
  static constexpr int kN = (int)(DP * sizeof(T) / 32);
  u32x4_t v[kN];
  __device__ __forceinline__ static uint32_t chunk(int t) {
    const uint32_t h = lane_id() >> 5;
    return sizeof(T) == 4 ? h * (uint32_t)kN + (uint32_t)t : 2u * (uint32_t)t + h;
  }
  // base (uniform): the first of the wave's rows, `stride` bytes apart; rows at or
  // beyond `rows` and chunks at or beyond d_bytes are zeros.
  __device__ __forceinline__ void load(const char* base, uint32_t stride, int32_t rows, uint32_t d_bytes) {
    const uint32_t row = lane_id() & 31u;
    const attn_rsrc_t r = attn_rsrc(base, rows > 0 ? (uint32_t)(min(rows, 32) - 1) * stride + d_bytes : 0u);
#pragma unroll
    for (int t = 0; t < kN; ++t)
      v[t] = attn_load16(r, (int32_t)row < rows && chunk(t) * 16u < d_bytes ? row * stride + chunk(t) * 16u
                                                                           : kAttnOut);
  }
};

// acc[r] += sum_d tile[row0 + R(r)][d] * frag row (l & 31), R(r) = 8 (r / 4) +
// 4 (l >> 5) + r % 4.
template <class T, int DP>
__device__ __forceinline__ void attn_row_product(f32x16_t& acc, const char* tile, uint32_t row0,
                                                 const AttnFrag<T, DP>& frag) {
  const uint32_t row = row0 + (lane_id() & 31u);
#pragma unroll
  for (int t = 0; t < AttnFrag<T, DP>::kN; ++t) {
    const u32x4_t a = lds_read16(tile, AttnLds<T, DP>::off(row, AttnFrag<T, DP>::chunk(t)));
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                    __builtin_bit_cast(bf16x8_t, frag.v[t]), acc, 0,
                                                    0, 0);
    } else {
      const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, frag.v[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], acc, 0, 0, 0);
    }
  }
}

// The same with the right operand in an LDS tile too (row col0 + (l & 31)).
template <class T, int DP>
__device__ __forceinline__ void attn_row_product(f32x16_t& acc, const char* tile, uint32_t row0,
                                                 const char* right, uint32_t col0) {
  const uint32_t row = row0 + (lane_id() & 31u), col = col0 + (lane_id() & 31u);
#pragma unroll
  for (int t = 0; t < AttnFrag<T, DP>::kN; ++t) {
    const u32x4_t a = lds_read16(tile, AttnLds<T, DP>::off(row, AttnFrag<T, DP>::chunk(t)));
    const u32x4_t b = lds_read16(right, AttnLds<T, DP>::off(col, AttnFrag<T, DP>::chunk(t)));
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                    __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
    } else {
      const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], acc, 0, 0, 0);
    }
  }
}

typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;

// acc[db][r] += sum over the 32 rows of tile[row0 + row][32 db + R(r)] * w[row],
// w held as attn_row_product leaves it (w[r] belongs to row R(r)).
template <class T, int DP>
__device__ __forceinline__ void attn_col_product(f32x16_t (&acc)[DP / 32], const char* tile,
                                                 uint32_t row0, const f32x16_t& w) {
  typedef AttnLds<T, DP> L;
  const uint32_t l = lane_id(), h = l >> 5;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {  // rows 16 t .. + 15, slot j: row 16 t + 8 (j / 4) + 4 h + j % 4
      u32x4_t b;
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = pack_bf16x2(w[8 * t + 2 * e], w[8 * t + 2 * e + 1]);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        // a 16-lane group's lane g * 16 + i reads row (i >> 2), columns 4 (i & 3) .. + 3 of the
        // group's 4 x 16 block and receives column i of its four rows
        bf16x4_t a[2];
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
          const uint32_t row = row0 + 16u * t + 8u * u + 4u * h + ((l & 15u) >> 2);
          const uint32_t ch = 4u * db + 2u * ((l >> 4) & 1u) + ((l & 3u) >> 1);
          a[u] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (lds_bf16x4_t*)(tile + L::off(row, ch) + (l & 1u) * 8u));
        }
        const bf16x8_t av = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7);
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av, __builtin_bit_cast(bf16x8_t, b),
                                                          acc[db], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t row = row0 + 8u * (r / 4) + 4u * h + r % 4;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        const uint32_t d = 32u * db + (l & 31u);
        const float x = *reinterpret_cast<const float*>(tile + L::off(row, d / 4) + (d % 4) * 4u);
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, w[r], acc[db], 0, 0, 0);
      }
    }
  }
}

// LDS DMA: LDS[dst + size lane] = mem[r + off], `size` bytes per lane.
__device__ __forceinline__ void attn_dma16(attn_rsrc_t r, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)dst, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void attn_dma4(attn_rsrc_t r, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)dst, 4, off, 0, 0, 0);
}

// ROWS rows of a [rows, head, d] tensor from memory to an LDS tile by LDS DMA: an
// instruction writes 1 KiB of the tile in order, so the lane that writes a slot
// loads the chunk that the swizzle puts there.  Rows at or beyond `rows` and
// chunks at or beyond d_bytes arrive as zeros (an offset past the resource
// touches no memory).  The resource starts at the tile's first row, so 32-bit
// offsets reach it wherever it lies.
template <class T, int DP, int ROWS>
struct AttnDma {
  static constexpr int kN = (int)(ROWS * AttnLds<T, DP>::kCh / kAttnThreads);
  uint32_t off[kN];
  uint32_t stride, d_bytes;
  __device__ __forceinline__ void init(uint32_t stride_b, uint32_t d_bytes_) {
    stride = stride_b;
    d_bytes = d_bytes_;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t idx = (wave_id() * kN + (uint32_t)i) * 64u + lane_id();
      const uint32_t row = idx / AttnLds<T, DP>::kCh;
      const uint32_t ch = (idx % AttnLds<T, DP>::kCh) ^ AttnLds<T, DP>::swz(row);
      off[i] = ch * 16u < d_bytes ? row * stride + ch * 16u : kAttnOut;
    }
  }
  __device__ __forceinline__ void issue(const char* base, int32_t rows, char* tile) const {
    const uint32_t bytes = rows > 0 ? (uint32_t)(min(rows, ROWS) - 1) * stride + d_bytes : 0u;
    const attn_rsrc_t r = attn_rsrc(base, bytes);
#pragma unroll
    for (int i = 0; i < kN; ++i)
      attn_dma16(r, tile + (wave_id() * kN + (uint32_t)i) * 1024u, off[i]);
  }
};

// Which of two LDS buffers a block uses, known to the compiler: the buffer's
// place then is part of an LDS instruction's own offset.
template <uint32_t N>
using AttnBuf = std::integral_constant<uint32_t, N>;

// This wave's LDS DMA has landed and every wave's LDS reads are done.
__device__ __forceinline__ void attn_sync() {
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
  __syncthreads();
}

// Sums of the two halves of the wave (a row's two lanes), in both.
__device__ __forceinline__ float attn_pair_add(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                                  __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float attn_pair_max(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                                  __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// Order of a run of N matrix instructions and their LDS reads (READS for each):
// the reads of AHEAD of them first, then one instruction and the reads of a later
// one in turn.  Left to itself the compiler, short of registers, reads each
// operand right before its use and every instruction waits for the LDS.
template <int N, int READS, int AHEAD>
__device__ __forceinline__ void attn_sched_reads() {
  constexpr int kMfma = 0x8, kDsRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kDsRead, READS * AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kDsRead, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, AHEAD, 0);
}

// Keeps a rarely entered branch a branch: turned into selects, the masks of the
// few blocks that a range's end crosses would be evaluated in all of them.
__device__ __forceinline__ void attn_no_if_conversion() { asm volatile("" ::: "memory"); }

// The kernels' CAP: 0 no softcap; 1 a softcap up to kAttnCapFast, 2 one above it (fp32:
// any).  With bf16 inputs tanh is 1 - 2 / (exp(2x) + 1), whose absolute error of some
// 1.5 2^-23 is softcap times that in a score: up to 256 at most 5e-5 of a probability, a
// 40th of the rounding of P; at 1e6 it would be 0.2, where the cap should change
// nothing.  Above 256 a small x takes the series (x^9 on: 2^-30 of it), so that the
// error is 2^-19 of the score at most, less than that of its sum.  16384 tokens, 32
// heads of 128, forward and backward: 10.8 ms, 12.4 above 256.  fp32 takes the
// library's tanh.
constexpr float kAttnCapFast = 256.0f;

template <class T, int CAP>
__device__ __forceinline__ float attn_tanh(float x) {
  if constexpr (sizeof(T) == 4) return tanhf(x);
  const float t = fmaf(-2.0f, __builtin_amdgcn_rcpf(fast_exp2(x * (2.0f * kLog2e)) + 1.0f), 1.0f);
  if constexpr (CAP == 1) return t;
  const float y = x * x;
  const float p = fmaf(fmaf(fmaf(-17.0f / 315.0f, y, 2.0f / 15.0f), y, -1.0f / 3.0f), y * x, x);
  return y < 0.015625f ? p : t;  // (a NaN in both)
}

// acc^T [DP x 32 rows] * s (one per row) to the wave's rows of D elements, `pitch`
// elements apart from base (uniform) on; rows at or beyond `rows` are not written.
// The two lanes of a row hold four elements in turn; bf16 pairs of fours are
// exchanged so that each lane writes 16 bytes.
template <int DP, class Out>
__device__ __forceinline__ void attn_store(const f32x16_t (&acc)[DP / 32], float s, Out* base, int64_t pitch,
                                           int32_t rows, int32_t D) {
  const uint32_t h = lane_id() >> 5, row = lane_id() & 31u;
  const uint32_t stride = (uint32_t)(pitch * (int64_t)sizeof(Out));
  const attn_rsrc_t r =
      attn_rsrc(base, rows > 0 ? (uint32_t)(min(rows, 32) - 1) * stride + (uint32_t)D * sizeof(Out) : 0u);
  const uint32_t at = (int32_t)row < rows ? row * stride : kAttnOut;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) {
    if constexpr (sizeof(Out) == 2) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4_t v;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x = pack_bf16x2(acc[db][8 * g + 2 * e] * s, acc[db][8 * g + 2 * e + 1] * s);
          const uint32_t y = pack_bf16x2(acc[db][8 * g + 4 + 2 * e] * s, acc[db][8 * g + 5 + 2 * e] * s);
          const auto z = __builtin_amdgcn_permlane32_swap(x, y, false, false);
          v[e] = z[0];
          v[2 + e] = z[1];
        }
        const uint32_t d = 32u * db + 16u * g + 8u * h;
        attn_store16(v, r, (int32_t)d < D && at != kAttnOut ? at + d * 2u : kAttnOut);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t d = 32u * db + 8u * g + 4u * h;
        const f32x4_t v = {acc[db][4 * g] * s, acc[db][4 * g + 1] * s, acc[db][4 * g + 2] * s,
                           acc[db][4 * g + 3] * s};
        attn_store16(__builtin_bit_cast(u32x4_t, v), r,
                     (int32_t)d < D && at != kAttnOut ? at + d * 4u : kAttnOut);
      }
    }
  }
}

// acc * s as attn_store writes it in bf16, rounded to nearest with ties away from
// zero, and, if `low` is not null, the byte beneath each value's two: with it the
// backward has the value to 16 bits (attn_unround), for delta.  Where a few keys hold
// all of a row's probability, dO . V - delta cancels, and delta from the rounded
// rows alone leaves dQ and dK off by 0.0057 of their norm (rows of two keys; with
// these bytes 0.0025, of which 0.0017 is the outputs' own rounding), in long documents
// by 0.0027 against 0.0024.  It costs a byte per element, written and read: nothing in
// long documents, 41 -> 43 us of the forward and 59 -> 61 of dQ for 4096 tokens in
// 12.  The bytes lie as a wave's lanes hold and want them,
// attn_low_bytes(D) for each row and head: chunks of 8 elements, the even ones, then
// the odd ones.  low_pitch: bytes from row to row.
__device__ __host__ __forceinline__ int32_t attn_low_bytes(int32_t D) { return (D + 31) & ~31; }

template <int DP>
__device__ __forceinline__ void attn_store_out(const f32x16_t (&acc)[DP / 32], float s, __bf16* base,
                                               int64_t pitch, int32_t rows, int32_t D, char* low,
                                               int64_t low_pitch) {
  const uint32_t h = lane_id() >> 5, row = lane_id() & 31u;
  const uint32_t stride = (uint32_t)pitch * 2u, low_stride = (uint32_t)low_pitch;
  const uint32_t n = (uint32_t)attn_low_bytes(D) / 2, last = (uint32_t)(min(rows, 32) - 1);
  const attn_rsrc_t r = attn_rsrc(base, rows > 0 ? last * stride + (uint32_t)D * 2u : 0u);
  const attn_rsrc_t r_low = attn_rsrc(low, rows > 0 && low ? last * low_stride + 2 * n : 0u);
  const bool mine = (int32_t)row < rows;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) {
    uint32_t bytes[4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t top[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // pairs of the eight elements that a half wave holds
        const uint32_t x = __float_as_uint(acc[db][8 * g + 2 * e] * s);
        const uint32_t y = __float_as_uint(acc[db][8 * g + 2 * e + 1] * s);
        top[e] = __builtin_amdgcn_perm(y + 0x8000u, x + 0x8000u, 0x07060302u);
        const uint32_t b = __builtin_amdgcn_perm(y, x, 0x0c0c0501u);
        bytes[2 * g + e / 2] = e & 1 ? __builtin_amdgcn_perm(b, bytes[2 * g + e / 2], 0x05040100u) : b;
      }
      u32x4_t v;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto z = __builtin_amdgcn_permlane32_swap(top[e], top[2 + e], false, false);
        v[e] = z[0];
        v[2 + e] = z[1];
      }
      const uint32_t d = 32u * db + 16u * g + 8u * h;
      attn_store16(v, r, mine && (int32_t)d < D ? row * stride + d * 2u : kAttnOut);
    }
    if (low) {
      const auto x = __builtin_amdgcn_permlane32_swap(bytes[0], bytes[1], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(bytes[2], bytes[3], false, false);
      attn_store16(u32x4_t{x[0], x[1], y[0], y[1]}, r_low,
                   mine && 16u * db < n ? row * low_stride + h * n + 16u * db : kAttnOut);
    }
  }
}

// The value that attn_store_out rounded to `top` (its bits, the lower half zero), from
// byte `i` of `low`: rounded up where that byte is 128 or more, so that it counts
// from -128 on; the middle of what lies beneath it.
__device__ __forceinline__ float attn_unround(uint32_t top, uint32_t low, int i) {
  return __uint_as_float((top | 0x80u) + ((uint32_t)__builtin_amdgcn_sbfe((int32_t)low, 8 * i, 8) << 8));
}

// The two waves of a pair (SPLIT = 2): the odd one leaves its accumulators, m and
// sum in LDS and is done (false); the even one gets the other's m and sum, and its
// accumulators from attn_add_pair.
template <int DP>
__device__ __forceinline__ bool attn_join_pair(const f32x16_t (&acc)[DP / 32], float& m, float& sum,
                                               char* lds) {
  float* at = reinterpret_cast<float*>(lds) + (wave_id() >> 1) * (64 * (DP / 2 + 2)) + lane_id();
  __syncthreads();  // the tiles have been read
  if (wave_id() & 1u) {
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) at[64 * i] = acc[i / 16][i % 16];
    at[64 * (DP / 2)] = m;
    at[64 * (DP / 2 + 1)] = sum;
  }
  __syncthreads();
  if (wave_id() & 1u) return false;
  m = at[64 * (DP / 2)];
  sum = at[64 * (DP / 2 + 1)];
  return true;
}
template <int DP>
__device__ __forceinline__ void attn_add_pair(f32x16_t (&acc)[DP / 32], float f, float f2, const char* lds) {
  const float* at = reinterpret_cast<const float*>(lds) + (wave_id() >> 1) * (64 * (DP / 2 + 2)) + lane_id();
#pragma unroll
  for (int i = 0; i < DP / 2; ++i)
    acc[i / 16][i % 16] = fmaf(at[64 * i], f2, acc[i / 16][i % 16] * f);
}

// rows x D zeros, rows `pitch` elements apart (D: whole 16-byte chunks).
template <class Out>
__device__ __forceinline__ void attn_zero_rows(Out* base, int32_t rows, int64_t pitch, int32_t D) {
  const int32_t per = D * (int32_t)sizeof(Out) / 16;
  for (int32_t i = threadIdx.x; i < rows * per; i += kAttnThreads)
    *reinterpret_cast<u32x4_t*>(reinterpret_cast<char*>(base + (int64_t)(i / per) * pitch) +
                                (i % per) * 16) = u32x4_t{0u, 0u, 0u, 0u};
}

// Tile `at` of a plan, or tail < 0 where the plan has fewer.  Read through the
// scalar cache (the plan was written by an earlier launch), the count beside it.
__device__ __forceinline__ AttnTile attn_tile(const int32_t* plan, int64_t at, int32_t ti) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_t;
  const scalar_t c = (scalar_t)(uintptr_t)(plan);
  const scalar_t p = (scalar_t)(uintptr_t)(plan + kPlanHeader + at * kPlanTile);
  const int32_t tiles = c[0];
  AttnTile t = {p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
  if (ti >= tiles) t.tail = -1;
  return t;
}

// Workgroups among which the query heads of a key tile's group are divided, each
// writing fp32 parts of dK and dV for attn_join_kernel; with one, a workgroup
// writes the results themselves.  (cost of this tile, most of the costliest, total
// of all `tiles`, in blocks of 64 queries of one head.)
//   The costliest tile more than 1.25 times what each of 512 resident workgroups
//   gets of all the work, few long documents among short ones: as many as keep a
//   workgroup below three quarters of that.  64 documents in 32768 tokens, 6 heads
//   a group, dK/dV and join: 295 us; every tile in 6 parts 422, in 3 479 us.
//   Otherwise, where a tile has 128 blocks on average: 2048 workgroups, so that
//   they end together; one document of 16384 tokens 4.15 ms, undivided 4.4.
//   Otherwise one: 256 documents of 128 tokens take 76 us so, 148 divided, since
//   the parts are most of the bytes.
__device__ __forceinline__ int32_t attn_parts(int32_t cost, int32_t most, int32_t total, int32_t tiles,
                                              int32_t Hq, int32_t G, int32_t parts_max) {
  const int64_t work = (int64_t)total * Hq;
  int32_t n = 1;
  if ((int64_t)most * G * 410 > work)
    while (n < parts_max && (int64_t)cost * G * 700 > n * work) ++n;
  else if ((int64_t)total * G >= (int64_t)tiles * 128)
    while (n < parts_max && (int64_t)n * tiles * (Hq / G) < 2048) ++n;
  const int32_t per = (G + n - 1) / n;
  return (G + per - 1) / per;
}

// Half `which` of a query tile, the later rows first; false if it has none.
__device__ __forceinline__ bool attn_half(AttnTile& t, int32_t which, int32_t window) {
  constexpr int32_t kHalf = kAttnRows / 2;
  if (which == 1) {
    t.rows = min(t.rows, kHalf);
  } else {
    t.row0 += kHalf;
    t.rows -= kHalf;
    if (t.rows <= 0) return false;
  }
  if (!t.tail) {
    t.beg = attn_row_lo(t.row0, t.ds, window);
    t.end = attn_row_hi(t.row0 + t.rows - 1, t.pe);
  }
  return true;
}

struct AttnArgs {
  const char *q, *k, *v, *o, *dout;            // element (t, h, d) at t * *_t + h * *_h + d * size
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, do_t, do_h;  // bytes
  char *out, *dq, *dk, *dv;                    // [T, heads, D], contiguous
  char* out_lo;                                // attn_store_out's bytes, rows [T, Hq]; or null
  float *lse, *delta;                          // [Hq, T]; lse in units of log2
  float *lse_lo, *factor;                      // [Hq, T]: what its rounding took from lse (or null); kAttnFar
  int32_t* items;                              // attn_items
  float* part;                                 // [Hk][slots][2][kAttnRows][D]: dK, dV of one part
  const int32_t* plan;
  int32_t T, Hq, Hk, G, D, tiles_max, window, parts_max, slots;
  float scale;     // of the scores
  float z_mul;     // log2 units: scale log2(e), or cap log2(e) with a softcap
  float cap_mul;   // scale / cap
};

__device__ __forceinline__ int32_t attn_parts(const AttnTile& t, const AttnArgs& a) {
  const auto* head = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)a.plan;
  return attn_parts(attn_cost(t), head[2], head[1], head[0], a.Hq, a.G, a.parts_max);
}

// What attn_dkdv_kernel's workgroups of one key head take: (tile, part) pairs, the
// costliest first (counting sort), and none without work among them: those would
// be dealt out in turn with the others and leave the shader engines that get them
// idle (9.4 instead of 4.4 ms).  Tiles with several parts get places for them in
// a.part, as long as there are any (attn_slots of the host has enough for what
// attn_parts divides).  One workgroup.
//   a.items: [0] pairs; from 4 on the pairs; from 4 + 2 tiles_max parts_max on for
//   each tile its parts and the first one's place
__device__ __forceinline__ int32_t attn_tile_info(const AttnArgs& a, int32_t ti) {
  return 4 + 2 * a.tiles_max * a.parts_max + 2 * ti;
}
__device__ __forceinline__ void attn_items(const AttnArgs& a, int32_t* scratch) {
  int32_t* hist = scratch;                  // kPlanBuckets
  int32_t* sums = scratch + kPlanBuckets;   // one per thread
  int32_t* used = sums + kAttnThreads;      // places given out
  const int32_t tid = (int32_t)threadIdx.x, tiles = a.plan[0];
  constexpr int32_t kPer = kPlanBuckets / kAttnThreads;
  const AttnTile* kt = reinterpret_cast<const AttnTile*>(a.plan + kPlanHeader) + a.tiles_max;
  // costs of an item are at most G times that of the first tile (the costliest)
  const int64_t most = tiles > 0 ? max((int64_t)1, (int64_t)attn_cost(kt[0]) * a.G) : 1;
  for (int32_t i = tid; i < kPlanBuckets; i += kAttnThreads) hist[i] = 0;
  if (tid == 0) *used = 0;
  __syncthreads();
  for (int pass = 0; pass < 2; ++pass) {
    for (int32_t t = tid; t < tiles; t += kAttnThreads) {
      const int32_t cost = attn_cost(kt[t]);
      int32_t* info = a.items + attn_tile_info(a, t);
      if (pass == 0) {
        int32_t n = attn_parts(kt[t], a), slot = 0;
        if (n > 1) {
          slot = atomicAdd(used, n);
          if (slot + n > a.slots) n = 1;
        }
        info[0] = n;
        info[1] = slot;
      }
      const int32_t parts = info[0];  // (this thread's own of the first pass)
      const int32_t per = (a.G + parts - 1) / parts;
      for (int32_t p = 0; p < parts; ++p) {
        const int64_t c = (int64_t)cost * min(per, a.G - p * per);
        const int32_t b = (int32_t)(min(c, most) * (kPlanBuckets - 1) / most);
        const int32_t at = atomicAdd(&hist[kPlanBuckets - 1 - b], 1);
        if (pass == 1) {
          a.items[4 + 2 * at] = t;
          a.items[5 + 2 * at] = p;
        }
      }
    }
    __syncthreads();
    if (pass == 0) {  // counts -> first places
      int32_t n = 0;
      for (int32_t i = 0; i < kPer; ++i) n += hist[tid * kPer + i];
      sums[tid] = n;
      __syncthreads();
      int32_t at = 0;
      for (int32_t i = 0; i < tid; ++i) at += sums[i];
      if (tid == kAttnThreads - 1) a.items[0] = at + n;
      for (int32_t i = 0; i < kPer; ++i) {
        const int32_t m = hist[tid * kPer + i];
        hist[tid * kPer + i] = at;
        at += m;
      }
      __syncthreads();
    }
  }
}

// A row's probabilities are 2^(z - lse) times a factor 2^-lse_lo, which is far from 1
// where the scores are so large that lse has no room for the logarithm of the sum
// beside the maximum (beyond some 2^20: of two equal scores of 1e9 each would count
// whole).  Below kAttnFar it is within 2^-12 ln 2 of 1, and so are the probabilities
// by the rounding of scores of that size; dK and dV leave it out there.
constexpr float kAttnFar = 8192.0f;

// --- forward ----------------------------------------------------------------

constexpr int kAttnKeys = 64;  // keys per block of the forward and of dQ

// SPLIT = 2: a workgroup takes half a tile, its waves in pairs that share 32 rows,
// each over half of every block's keys, and join at the end: twice the workgroups,
// each with half the way, where there are few of them (attn_split of the host).
//
// Long rows are bound by the matrix instructions at the clock that the power limit
// leaves, and by the LDS behind them (an instruction's left operand is 1 KiB, four
// SIMDs ask for 128 bytes a cycle, all the LDS has): one document of 32768 tokens,
// 32 heads of 128, 7.5 to 8.4 ms from box to box, 1050 to 1170 TFLOP/s, 0.88 of what a
// large matrix product reaches there.  A softcap adds two transcendentals per score to
// the exponential (16384 tokens: 2.1 -> 2.7 ms, MFMA busy 43%).  Short documents are
// bound by each workgroup's first tile, masks and last partial tile: 4096 tokens of 12
// documents 45 us.  Row tiles of 128 with two workgroups on a CU: a wave alone on its SIMD
// with twice the rows hides neither the LDS nor the softmax (dK and dV below).
template <class T, int DP, int CAP, int SPLIT>
__global__ __launch_bounds__(kAttnThreads, (sizeof(T) == 2 ? 2 : 1)) void attn_fwd_kernel(AttnArgs a) {
  typedef AttnLds<T, DP> L;
  constexpr uint32_t kTile = kAttnKeys * L::kRowB;
  __shared__ __attribute__((aligned(1024))) char smem[4 * kTile];  // 2 x (K, V)
  const uint32_t id = blockIdx.x;
  // consecutive workgroups lie on different XCDs: with 8 key heads an XCD's L2 holds one of them
  const uint32_t kvh = id % (uint32_t)a.Hk, rest = id / (uint32_t)a.Hk;
  const uint32_t head = kvh * (uint32_t)a.G + rest % (uint32_t)a.G;
  const int32_t ti = (int32_t)(rest / (uint32_t)a.G) / SPLIT;
  AttnTile t = attn_tile(a.plan, ti, ti);
  if (t.tail < 0) return;
  if constexpr (SPLIT == 2)
    if (!attn_half(t, (int32_t)(rest / (uint32_t)a.G) & 1, a.window)) return;
  const int64_t o_t = (int64_t)a.Hq * a.D;
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)t.row0 * o_t + (int64_t)head * a.D;
  float* lse = a.lse + (int64_t)head * a.T;
  if (t.tail) {
    attn_zero_rows(out, t.rows, o_t, a.D);
    for (int32_t i = threadIdx.x; i < t.rows; i += kAttnThreads) lse[t.row0 + i] = 0.f;
    return;
  }
  const uint32_t w = wave_id(), l = lane_id(), h = l >> 5;
  const uint32_t d_bytes = (uint32_t)a.D * sizeof(T);
  const int32_t r0 = t.row0 + 32 * (int32_t)(w / SPLIT), row = r0 + (int32_t)(l & 31u);
  // the wave's keys of a block: kOwn from `first` on
  constexpr int32_t kOwn = kAttnKeys / SPLIT;
  const int32_t first = SPLIT == 2 ? 32 * (int32_t)(w & 1u) : 0;
  const int32_t r_end = t.row0 + t.rows;
  const bool active = r0 < r_end, valid = row < r_end;
  const int32_t r_last = min(r0 + 31, r_end - 1);
  // the wave's keys [w_lo, w_hi), of which every row sees [f_lo, f_hi)
  const int32_t w_lo = attn_row_lo(r0, t.ds, a.window), w_hi = attn_row_hi(r_last, t.pe);
  const int32_t f_lo = attn_row_lo(r_last, t.ds, a.window), f_hi = attn_row_hi(r0, t.pe);
  const int32_t lo = attn_row_lo(row, t.ds, a.window), hi = valid ? attn_row_hi(row, t.pe) : lo;

  f32x16_t acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16_t{};
  float m = kAttnLowest, sum = 0.f;

  const char* kbase = a.k + (int64_t)kvh * a.k_h;
  const char* vbase = a.v + (int64_t)kvh * a.v_h;
  AttnDma<T, DP, kAttnKeys> sk, sv;
  sk.init((uint32_t)a.k_t, d_bytes);
  sv.init((uint32_t)a.v_t, d_bytes);
  auto fetch = [&](int32_t k0, uint32_t buf) {
    sk.issue(kbase + (int64_t)k0 * a.k_t, t.end - k0, smem + buf * 2 * kTile);
    sv.issue(vbase + (int64_t)k0 * a.v_t, t.end - k0, smem + buf * 2 * kTile + kTile);
  };
  fetch(t.beg, 0);
  AttnFrag<T, DP> qf;
  qf.load(a.q + (int64_t)r0 * a.q_t + (int64_t)head * a.q_h, (uint32_t)a.q_t, r_end - r0, d_bytes);
  auto block = [&](int32_t k0, auto buf) {
    attn_sync();
    // into the buffer that every wave has left at the barrier
    if (k0 + kAttnKeys < t.end) fetch(k0 + kAttnKeys, buf.value ^ 1u);
    k0 += first;
    if (!active || k0 >= w_hi || k0 + kOwn <= w_lo) return;
    const char* kt = smem + buf.value * 2 * kTile;
    f32x16_t s[2 / SPLIT];
#pragma unroll
    for (uint32_t b = 0; b < 2 / SPLIT; ++b) {
      s[b] = f32x16_t{};
      attn_row_product<T, DP>(s[b], kt, (uint32_t)first + 32u * b, qf);
    }
    if constexpr (sizeof(T) == 2) attn_sched_reads<DP / 8 / SPLIT, 1, 4>();
    if constexpr (CAP) {
#pragma unroll
      for (int b = 0; b < 2 / SPLIT; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = attn_tanh<T, CAP>(s[b][r] * a.cap_mul);
    }
    if (k0 < f_lo || k0 + kOwn > f_hi) {
      attn_no_if_conversion();
      const uint32_t from = (uint32_t)(k0 + 4 * (int32_t)h - lo), n = (uint32_t)(hi - lo);
#pragma unroll
      for (int b = 0; b < 2 / SPLIT; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (from + (uint32_t)(32 * b + 8 * (r / 4) + r % 4) >= n) s[b][r] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 32 / SPLIT; ++i) mx = fmaxf(mx, s[i / 16][i % 16]);
    mx = attn_pair_max(mx) * a.z_mul;
    // the running maximum moves when it has to: up to 2^8 of slack costs no
    // precision in a floating format and saves rescaling the sums.  Each row goes
    // by its own scores, so that no other row of the wave changes its rounding.
    const bool grown = mx > m + 8.f;
    if (__any(grown)) {
      const float mn = grown ? mx : m, f = fast_exp2(m - mn);
      m = mn;
      sum *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
    }
#pragma unroll
    for (int b = 0; b < 2 / SPLIT; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = fast_exp2(fmaf(s[b][r], a.z_mul, -m));
        sum += s[b][r];
      }
#pragma unroll
    for (uint32_t b = 0; b < 2 / SPLIT; ++b)
      attn_col_product<T, DP>(acc, kt + kTile, (uint32_t)first + 32u * b, s[b]);
    if constexpr (sizeof(T) == 2) attn_sched_reads<DP / 8 / SPLIT, 2, 4>();
  };
  for (int32_t k0 = t.beg; k0 < t.end; k0 += 2 * kAttnKeys) {
    block(k0, AttnBuf<0>());
    if (k0 + kAttnKeys < t.end) block(k0 + kAttnKeys, AttnBuf<1>());
  }
  sum = attn_pair_add(sum);
  if constexpr (SPLIT == 2) {
    float m2 = m, sum2 = sum;
    if (!attn_join_pair<DP>(acc, m2, sum2, smem)) return;
    const float mn = fmaxf(m, m2), f = fast_exp2(m - mn), f2 = fast_exp2(m2 - mn);
    m = mn;
    sum = sum * f + sum2 * f2;
    attn_add_pair<DP>(acc, f, f2, smem);
  }
  if (valid && h == 0) {
    const float rest = fast_log2(sum), both = m + rest;
    lse[row] = both;
    if (a.lse_lo) {  // (the error of a sum, exactly)
      const float part = both - m;
      a.lse_lo[(int64_t)head * a.T + row] = (m - (both - part)) + (rest - part);
    }
  }
  const int64_t at = (int64_t)r0 * o_t + (int64_t)head * a.D;
  if constexpr (sizeof(T) == 2) {
    const int64_t n = attn_low_bytes(a.D);
    attn_store_out<DP>(acc, 1.0f / sum, reinterpret_cast<T*>(a.out) + at, o_t, r_end - r0, a.D,
                       a.out_lo ? a.out_lo + ((int64_t)r0 * a.Hq + head) * n : nullptr, a.Hq * n);
  } else {
    attn_store<DP>(acc, 1.0f / sum, reinterpret_cast<T*>(a.out) + at, o_t, r_end - r0, a.D);
  }
}

// --- backward: delta and dQ ---------------------------------------------------

// Three products per block (scores, dP, dQ) with Q, dO and dQ in registers; delta
// comes from the rows' own dO and O, once.  dQ has a kernel of its own, and the
// scores and dP are formed again for dK and dV: adding dQ from a kernel of the keys
// would take atomics, whose order changes results, or a copy of dQ per key tile.
// 16384 tokens, 32 heads of 128: 2.8 to 2.9 ms from box to box, 1140 to 1190 TFLOP/s;
// with a softcap 3.6.
template <class T, int DP, int CAP, int SPLIT>
__global__ __launch_bounds__(kAttnThreads, (sizeof(T) == 2 ? 2 : 1)) void attn_dq_kernel(AttnArgs a) {
  typedef AttnLds<T, DP> L;
  constexpr uint32_t kTile = kAttnKeys * L::kRowB;
  __shared__ __attribute__((aligned(1024))) char smem[4 * kTile];  // 2 x (K, V)
  static_assert(sizeof(smem) >= 4 * (kPlanBuckets + kAttnThreads + 1), "attn_items");
  if (blockIdx.x == 0) {  // beside the others, for the launch that follows
    attn_items(a, reinterpret_cast<int32_t*>(smem));
    return;
  }
  const uint32_t id = blockIdx.x - 1;
  const uint32_t kvh = id % (uint32_t)a.Hk, rest = id / (uint32_t)a.Hk;
  const uint32_t head = kvh * (uint32_t)a.G + rest % (uint32_t)a.G;
  const int32_t ti = (int32_t)(rest / (uint32_t)a.G) / SPLIT;
  AttnTile t = attn_tile(a.plan, ti, ti);
  if (t.tail < 0) return;
  if constexpr (SPLIT == 2)
    if (!attn_half(t, (int32_t)(rest / (uint32_t)a.G) & 1, a.window)) return;
  const int64_t o_t = (int64_t)a.Hq * a.D;
  T* dq = reinterpret_cast<T*>(a.dq) + (int64_t)head * a.D;
  if (t.tail) {
    attn_zero_rows(dq + (int64_t)t.row0 * o_t, t.rows, o_t, a.D);
    return;
  }
  const uint32_t w = wave_id(), l = lane_id(), h = l >> 5;
  const uint32_t d_bytes = (uint32_t)a.D * sizeof(T);
  const int32_t r0 = t.row0 + 32 * (int32_t)(w / SPLIT), row = r0 + (int32_t)(l & 31u);
  // the wave's keys of a block: kOwn from `first` on
  constexpr int32_t kOwn = kAttnKeys / SPLIT;
  const int32_t first = SPLIT == 2 ? 32 * (int32_t)(w & 1u) : 0;
  const int32_t r_end = t.row0 + t.rows;
  const bool active = r0 < r_end, valid = row < r_end;
  const int32_t r_last = min(r0 + 31, r_end - 1);
  const int32_t w_lo = attn_row_lo(r0, t.ds, a.window), w_hi = attn_row_hi(r_last, t.pe);
  const int32_t f_lo = attn_row_lo(r_last, t.ds, a.window), f_hi = attn_row_hi(r0, t.pe);
  const int32_t lo = attn_row_lo(row, t.ds, a.window);
  // a row that sees one key has p = 1 and ds = 0 exactly, which do . v - delta, two
  // sums in different orders, would miss by their rounding: it counts as seeing none
  const int32_t hi = valid && attn_row_hi(row, t.pe) - lo > 1 ? attn_row_hi(row, t.pe) : lo;

  const char* kbase = a.k + (int64_t)kvh * a.k_h;
  const char* vbase = a.v + (int64_t)kvh * a.v_h;
  AttnDma<T, DP, kAttnKeys> sk, sv;
  sk.init((uint32_t)a.k_t, d_bytes);
  sv.init((uint32_t)a.v_t, d_bytes);
  auto fetch = [&](int32_t k0, uint32_t buf) {
    sk.issue(kbase + (int64_t)k0 * a.k_t, t.end - k0, smem + buf * 2 * kTile);
    sv.issue(vbase + (int64_t)k0 * a.v_t, t.end - k0, smem + buf * 2 * kTile + kTile);
  };
  fetch(t.beg, 0);
  AttnFrag<T, DP> qf, dof, of;
  dof.load(a.dout + (int64_t)r0 * a.do_t + (int64_t)head * a.do_h, (uint32_t)a.do_t, r_end - r0, d_bytes);
  of.load(a.o + ((int64_t)r0 * o_t + (int64_t)head * a.D) * (int64_t)sizeof(T), (uint32_t)o_t * sizeof(T),
          r_end - r0, d_bytes);
  u32x4_t low[sizeof(T) == 2 ? DP / 32 : 1];
  if constexpr (sizeof(T) == 2) {  // (without out_lo: zeros)
    const uint32_t n = (uint32_t)attn_low_bytes(a.D) / 2, stride = 2 * n * (uint32_t)a.Hq;
    const int32_t rows = a.out_lo ? min(r_end - r0, 32) : 0;
    const attn_rsrc_t r = attn_rsrc(a.out_lo + ((int64_t)r0 * a.Hq + head) * (2 * n),
                                    rows > 0 ? (uint32_t)(rows - 1) * stride + 2 * n : 0u);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      low[i] = attn_load16(r, (int32_t)(l & 31u) < rows && 16u * i < n ? (l & 31u) * stride + h * n + 16u * i
                                                                       : kAttnOut);
  }
  qf.load(a.q + (int64_t)r0 * a.q_t + (int64_t)head * a.q_h, (uint32_t)a.q_t, r_end - r0, d_bytes);
  const float lse = valid ? a.lse[(int64_t)head * a.T + row] : 0.f;
  const float factor = valid && a.lse_lo ? fast_exp2(-a.lse_lo[(int64_t)head * a.T + row]) : 1.0f;
  float delta = 0.f;
#pragma unroll
  for (int i = 0; i < AttnFrag<T, DP>::kN; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = of.v[i][e], y = dof.v[i][e];
      if constexpr (sizeof(T) == 2) {
        const uint32_t lw = low[i / 2][2 * (i % 2) + e / 2];
        delta = fmaf(attn_unround(x << 16, lw, 2 * (e % 2)), __uint_as_float(y << 16), delta);
        delta = fmaf(attn_unround(x & 0xffff0000u, lw, 2 * (e % 2) + 1), __uint_as_float(y & 0xffff0000u),
                     delta);
      } else {
        delta = fmaf(__uint_as_float(x), __uint_as_float(y), delta);
      }
    }
  delta = attn_pair_add(delta);
  if (valid && h == 0) {
    a.delta[(int64_t)head * a.T + row] = delta;
    a.factor[(int64_t)head * a.T + row] = factor;
  }
  f32x16_t acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16_t{};
  auto block = [&](int32_t k0, auto buf) {
    attn_sync();
    if (k0 + kAttnKeys < t.end) fetch(k0 + kAttnKeys, buf.value ^ 1u);
    k0 += first;
    if (!active || k0 >= w_hi || k0 + kOwn <= w_lo) return;
    const char* kt = smem + buf.value * 2 * kTile;
    const bool edge = k0 < f_lo || k0 + kOwn > f_hi;
#pragma unroll
    for (uint32_t b = 0; b < 2 / SPLIT; ++b) {
      f32x16_t s = f32x16_t{}, dp = f32x16_t{};
      attn_row_product<T, DP>(s, kt, (uint32_t)first + 32u * b, qf);
      attn_row_product<T, DP>(dp, kt + kTile, (uint32_t)first + 32u * b, dof);
      if constexpr (sizeof(T) == 2) attn_sched_reads<DP / 8, 1, 4>();
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = s[r];
        if constexpr (CAP) x = attn_tanh<T, CAP>(x * a.cap_mul);
        s[r] = fast_exp2(fmaf(x, a.z_mul, -lse)) * (dp[r] - delta);
        if constexpr (CAP) s[r] *= fmaf(-x, x, 1.0f);
      }
      if (edge) {
        attn_no_if_conversion();
        const uint32_t from = (uint32_t)(k0 + 32 * (int32_t)b + 4 * (int32_t)h - lo);
        const uint32_t n = (uint32_t)(hi - lo);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (from + (uint32_t)(8 * (r / 4) + r % 4) >= n) s[r] = 0.f;
      }
      attn_col_product<T, DP>(acc, kt, (uint32_t)first + 32u * b, s);
      if constexpr (sizeof(T) == 2) attn_sched_reads<DP / 16, 2, 4>();
    }
  };
  for (int32_t k0 = t.beg; k0 < t.end; k0 += 2 * kAttnKeys) {
    block(k0, AttnBuf<0>());
    if (k0 + kAttnKeys < t.end) block(k0 + kAttnKeys, AttnBuf<1>());
  }
  if constexpr (SPLIT == 2) {
    float none = 0.f, none2 = 0.f;
    if (!attn_join_pair<DP>(acc, none, none2, smem)) return;
    attn_add_pair<DP>(acc, 1.0f, 1.0f, smem);
  }
  // (linear in the row's probabilities)
  attn_store<DP>(acc, a.scale * factor, dq + (int64_t)r0 * o_t, o_t, r_end - r0, a.D);
}

// --- backward: dK and dV --------------------------------------------------------

// Rows of Q and dO per block: 32 where a row of an LDS tile takes 256 bytes or
// more (two workgroups per CU then fit its LDS), 64 else.
template <class T, int DP>
constexpr int attn_q_rows() {
  return sizeof(T) * DP >= 256 ? 32 : 64;
}

// Both accumulators of a wave's 32 keys take 128 registers at DP = 128 and the
// keys' K rows 32; their V rows stay in LDS, because with them in registers too a
// wave needs more than the 256 that let two share a SIMD, and a wave alone hides
// neither the LDS reads nor the softmax.  One document of 16384 tokens, 32 heads
// of 128 (8 key heads): 4.2 to 4.3 ms from box to box, 1020 to 1050 TFLOP/s; where it
// took 4.1, 7.4 with V in registers and 5.5 as two kinds of workgroup, dK and dV each
// with their own scores.
template <class T, int DP, int CAP>
__global__ __launch_bounds__(kAttnThreads, (sizeof(T) == 2 ? 2 : 1)) void attn_dkdv_kernel(AttnArgs a) {
  typedef AttnLds<T, DP> L;
  constexpr int kQ = attn_q_rows<T, DP>();
  constexpr bool kVLds = sizeof(T) == 2 && DP == 128;
  constexpr uint32_t kTile = kQ * L::kRowB;
  constexpr uint32_t kBuf = 2 * kTile + 3 * 256;
  __shared__ __attribute__((aligned(1024))) char smem[2 * kBuf];  // 2 x (Q, dO, lse, delta, factor)
  __shared__ __attribute__((aligned(1024))) char vt[kVLds ? kAttnRows * L::kRowB : 16];
  typedef const __attribute__((address_space(4))) int32_t* scalar_t;
  const scalar_t items = (scalar_t)(uintptr_t)a.items;
  const uint32_t kvh = blockIdx.x % (uint32_t)a.Hk;
  const int32_t item = (int32_t)(blockIdx.x / (uint32_t)a.Hk);
  if (item >= items[0]) return;
  const int32_t ti = items[4 + 2 * item], hs = items[5 + 2 * item];
  const AttnTile t = attn_tile(a.plan, (int64_t)a.tiles_max + ti, ti);
  const int32_t info = attn_tile_info(a, ti), parts = items[info], slot = items[info + 1] + hs;
  const int64_t o_t = (int64_t)a.Hk * a.D;
  const int64_t o_at = (int64_t)t.row0 * o_t + (int64_t)kvh * a.D;
  T* dk = reinterpret_cast<T*>(a.dk) + o_at;
  T* dv = reinterpret_cast<T*>(a.dv) + o_at;
  if (t.tail) {
    attn_zero_rows(dk, t.rows, o_t, a.D);
    attn_zero_rows(dv, t.rows, o_t, a.D);
    return;
  }
  const uint32_t w = wave_id(), l = lane_id(), h = l >> 5;
  const uint32_t d_bytes = (uint32_t)a.D * sizeof(T);
  const int32_t j0 = t.row0 + 32 * (int32_t)w, key = j0 + (int32_t)(l & 31u);
  const int32_t j_end = t.row0 + t.rows;
  const bool active = j0 < j_end, valid = key < j_end;
  const int32_t j_last = min(j0 + 31, j_end - 1);
  // the queries [w_lo, w_hi) that see some key of the wave; [f_lo, f_hi) see all of them
  const int32_t w_lo = attn_col_lo(j0, t.ds, t.pe), w_hi = attn_col_hi(j_last, t.de, a.window);
  const int32_t f_lo = attn_col_lo(j_last, t.ds, t.pe), f_hi = attn_col_hi(j0, t.de, a.window);
  const int32_t lo = attn_col_lo(key, t.ds, t.pe);
  const int32_t hi = valid ? attn_col_hi(key, t.de, a.window) : lo;
  // the queries [s_lo, s_hi) that see one key: ds = 0 exactly (attn_dq_kernel); no
  // block with one of them is seen whole
  int32_t s_lo = t.ds, s_hi = t.pe <= t.ds + 1 ? t.ds + 1 : t.ds;
  if (a.window == 1) s_lo = max(t.ds, t.pe - 1), s_hi = t.de;  // (s_lo <= s_hi)

  AttnFrag<T, DP> kf, vf;
  kf.load(a.k + (int64_t)j0 * a.k_t + (int64_t)kvh * a.k_h, (uint32_t)a.k_t, j_end - j0, d_bytes);
  if constexpr (kVLds) {
    AttnDma<T, DP, kAttnRows> sv;
    sv.init((uint32_t)a.v_t, d_bytes);
    sv.issue(a.v + (int64_t)t.row0 * a.v_t + (int64_t)kvh * a.v_h, t.rows, vt);
  } else {
    vf.load(a.v + (int64_t)j0 * a.v_t + (int64_t)kvh * a.v_h, (uint32_t)a.v_t, j_end - j0, d_bytes);
  }
  f32x16_t ak[DP / 32], av[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) ak[i] = av[i] = f32x16_t{};

  // the group's heads one after the other, each over the query blocks of [beg, end)
  const int32_t per = (a.G + parts - 1) / parts;
  const int32_t g0 = hs * per, g1 = min(a.G, g0 + per);
  AttnDma<T, DP, kQ> sq, sdo;
  sq.init((uint32_t)a.q_t, d_bytes);
  sdo.init((uint32_t)a.do_t, d_bytes);
  // from the last block to the first: workgroups of one document then pass the
  // same blocks at the same time, whichever keys they own, and find them in L2
  const int32_t i_last = t.beg + (t.end - t.beg - 1) / kQ * kQ;
  int32_t fg = g0, fi = i_last;  // the block to fetch next
  auto fetch = [&](uint32_t buf) {
    const int64_t head = (int64_t)kvh * a.G + fg;
    const int32_t n = min(kQ, t.end - fi);
    char* at = smem + buf * kBuf;
    sq.issue(a.q + (int64_t)fi * a.q_t + head * a.q_h, n, at);
    sdo.issue(a.dout + (int64_t)fi * a.do_t + head * a.do_h, n, at + kTile);
    if (w < 3) {  // the rows' lse by the first wave, their delta and factor by the next two
      const float* from = (w == 0 ? a.lse : w == 1 ? a.delta : a.factor) + head * a.T + fi;
      attn_dma4(attn_rsrc(from, 4u * (uint32_t)n), at + 2 * kTile + w * 256u, l * 4u);
    }
    fi -= kQ;
    if (fi < t.beg) fi = i_last, ++fg;
  };
  const int32_t blocks = g1 > g0 ? (g1 - g0) * ((t.end - t.beg + kQ - 1) / kQ) : 0;
  if (blocks > 0) fetch(0);
  const uint32_t range = (uint32_t)(hi - lo), ones = (uint32_t)(s_hi - s_lo);
  int32_t i0 = i_last;
  auto block = [&](int32_t n, auto buf) {
    attn_sync();
    if (n + 1 < blocks) fetch(buf.value ^ 1u);
    if (active && i0 < w_hi && i0 + kQ > w_lo) {
      const char* qt = smem + buf.value * kBuf;
      const float* rows = reinterpret_cast<const float*>(qt + 2 * kTile);
      // (in one branch with the masks: with a branch of its own the registers spill)
      const bool far = __any(fabsf(rows[l & (uint32_t)(kQ - 1)]) >= kAttnFar);
      const bool edge = i0 < f_lo || i0 + kQ > f_hi || far;
#pragma unroll
      for (int b = 0; b < kQ / 32; ++b) {
        f32x16_t s = f32x16_t{}, dp = f32x16_t{};
        attn_row_product<T, DP>(s, qt, 32u * b, kf);
        if constexpr (kVLds)
          attn_row_product<T, DP>(dp, qt + kTile, 32u * b, vt, 32u * w);
        else
          attn_row_product<T, DP>(dp, qt + kTile, 32u * b, vf);
        if constexpr (sizeof(T) == 2 && !kVLds) attn_sched_reads<DP / 8, 1, 4>();
        if constexpr (kVLds) {
          attn_sched_reads<DP / 16, 1, 3>();
          attn_sched_reads<DP / 16, 2, 2>();
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(rows + 32 * b + 8 * g + 4 * h);
          const f32x4_t delta = *reinterpret_cast<const f32x4_t*>(rows + 64 + 32 * b + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float x = s[r];
            if constexpr (CAP) x = attn_tanh<T, CAP>(x * a.cap_mul);
            s[r] = fast_exp2(fmaf(x, a.z_mul, -lse[e]));
            dp[r] = s[r] * (dp[r] - delta[e]);
            if constexpr (CAP) dp[r] *= fmaf(-x, x, 1.0f);
          }
        }
        if (edge) {
          attn_no_if_conversion();
          const uint32_t from = (uint32_t)(i0 + 32 * b + 4 * (int32_t)h - lo);
          const uint32_t one = (uint32_t)(i0 + 32 * b + 4 * (int32_t)h - s_lo);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint32_t at = (uint32_t)(8 * (r / 4) + r % 4);
            if (from + at >= range) s[r] = dp[r] = 0.f;
            if (one + at < ones) dp[r] = 0.f;
          }
          if (far) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const f32x4_t f = *reinterpret_cast<const f32x4_t*>(rows + 128 + 32 * b + 8 * g + 4 * h);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                s[4 * g + e] *= f[e];
                dp[4 * g + e] *= f[e];
              }
            }
          }
        }
        attn_col_product<T, DP>(av, qt + kTile, 32u * b, s);
        attn_col_product<T, DP>(ak, qt, 32u * b, dp);
        if constexpr (sizeof(T) == 2) attn_sched_reads<DP / 8, 2, (kVLds ? 3 : 4)>();
      }
    }
    i0 -= kQ;
    if (i0 < t.beg) i0 = i_last;
  };
  for (int32_t n = 0; n < blocks; n += 2) {
    block(n, AttnBuf<0>());
    if (n + 1 < blocks) block(n + 1, AttnBuf<1>());
  }
  if (parts > 1) {
    float* part = a.part + (((int64_t)kvh * a.slots + slot) * 2 * kAttnRows + (j0 - t.row0)) * a.D;
    attn_store<DP>(ak, a.scale, part, a.D, j_end - j0, a.D);
    attn_store<DP>(av, 1.0f, part + (int64_t)kAttnRows * a.D, a.D, j_end - j0, a.D);
  } else {
    const int64_t at = (int64_t)(j0 - t.row0) * o_t;
    attn_store<DP>(ak, a.scale, dk + at, o_t, j_end - j0, a.D);
    attn_store<DP>(av, 1.0f, dv + at, o_t, j_end - j0, a.D);
  }
}

// dK and dV of the tiles whose heads were divided, as the sums of their parts in
// order; four workgroups per tile and key head.
template <class T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(AttnArgs a) {
  const int32_t rest = (int32_t)(blockIdx.x >> 2);
  const int32_t kvh = rest % a.Hk, ti = rest / a.Hk;
  const AttnTile t = attn_tile(a.plan, (int64_t)a.tiles_max + ti, ti);
  if (t.tail != 0) return;
  const int32_t* info = a.items + attn_tile_info(a, ti);
  const int32_t parts = info[0], n = kAttnRows * a.D;
  if (parts == 1) return;
  const float* slot = a.part + ((int64_t)kvh * a.slots + info[1]) * 2 * n;
  const int32_t per = a.D / 4;
  for (int32_t i = (int32_t)((blockIdx.x & 3u) * kAttnThreads + threadIdx.x); i < 2 * t.rows * per;
       i += 4 * kAttnThreads) {
    const int32_t which = i >= t.rows * per, j = i - which * t.rows * per;
    const int64_t at = ((int64_t)(t.row0 + j / per) * a.Hk + kvh) * a.D + (j % per) * 4;
    const float* from = slot + which * n + (j / per) * a.D + (j % per) * 4;
    f32x4_t x = f32x4_t{};
    for (int32_t s0 = 0; s0 < parts; s0 += 4) {  // four loads in flight, added in order
      f32x4_t y[4];
#pragma unroll
      for (int32_t s = 0; s < 4; ++s)
        y[s] = s0 + s < parts
                   ? *reinterpret_cast<const f32x4_t*>(from + (int64_t)(s0 + s) * 2 * n)
                   : f32x4_t{};
#pragma unroll
      for (int32_t s = 0; s < 4; ++s) x += y[s];
    }
    T* to = reinterpret_cast<T*>(which ? a.dv : a.dk) + at;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    else
      *reinterpret_cast<f32x4_t*>(to) = x;
  }
}

}  // namespace mtf

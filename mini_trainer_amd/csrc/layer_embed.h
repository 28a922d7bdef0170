// Token embedding and its gradient (gfx950).
//
//   out[t] = scale W[id_t]                       (fp32, rounded once)
//   dW[v]  = scale sum over t with id_t = v of dout[t]
//
// Both are bound by memory.  The gradient sums rows of dout that lie anywhere; fp32
// atomics would repeat nothing and collide on the frequent tokens, so the tokens are
// sorted by id first (embed_sort_kernel) and each row of dW has one owner that adds its
// tokens in their order and writes the row once (embed_rows_kernel).  A row of more
// than kEmbedPiece tokens is summed in pieces by as many workgroups beforehand
// (embed_pieces_kernel), since a tokenizer's most frequent ids each own some per cent
// of all tokens; its owner adds the pieces in their order.  So results repeat.
//
// The sort is one launch without a word between workgroups: workgroup b of kBuckets
// takes the ids equal to b modulo kBuckets (the frequent ids, which lie side by side,
// come apart), reads all ids, counts the tokens of smaller buckets, which is where its
// own begin, and the tokens of each of its ids per wave; a scan over (id, wave) then
// gives each wave its places, and a second reading of the ids fills them in.  It reads
// every id kBuckets times, out of L2.
#pragma once

#include "step_norm.h"

namespace mtf {

constexpr int kEmbedSlots = 1024;    // ids of a bucket at most (64 KiB of counters)
constexpr int32_t kEmbedPiece = 32;  // tokens of a piece

struct EmbedArgs {
  const void* ids;
  const char *w, *dout;
  char *out, *dw;          // dw: rows of the type, or the fp32 accumulator
  int32_t* status;         // null: ids are not reported
  int32_t *starts, *order; // [buckets * per + 1], [T]
  float* part;             // [2 * pieces][part_t]
  int64_t w_t, dout_t, dw_t, part_t;
  int64_t padding;         // an id whose row gets no gradient, or -1
  int32_t T, V, H;
  int32_t log_buckets, per;
  float scale;
};

template <class I>
__device__ __forceinline__ int64_t embed_id(const EmbedArgs& a, int32_t t) {
  return (int64_t)reinterpret_cast<const I*>(a.ids)[t];
}
// Place of a valid id among all ids as they are sorted.
__device__ __forceinline__ int32_t embed_place(const EmbedArgs& a, int32_t id) {
  return (id & ((1 << a.log_buckets) - 1)) * a.per + (id >> a.log_buckets);
}

// A row is read by 2^log_lanes lanes of a wave, K vectors of V elements each; rows
// wider than a wave's 64 K vectors are cut into column chunks, narrower ones share a
// wave.  Returns this lane's row, its first vector, and the number of vectors.
struct EmbedSpan {
  int64_t row;
  int32_t first, step, nv;
};
template <int V, int K>
__device__ __forceinline__ EmbedSpan embed_span(int32_t H, int32_t log_lanes) {
  EmbedSpan s;
  s.nv = H / V;
  s.step = 1 << log_lanes;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave_id();
  const int32_t lane = lane_id() & (s.step - 1);
  const int32_t chunks = log_lanes == 6 ? (s.nv + 64 * K - 1) / (64 * K) : 1;
  const int64_t rows = unit / chunks;
  s.first = (int32_t)(unit - rows * chunks) * 64 * K + lane;
  s.row = rows * (64 >> log_lanes) + (lane_id() >> log_lanes);
  return s;
}

template <class T, class I, int V, int K>
__global__ __launch_bounds__(256) void embed_forward_kernel(EmbedArgs a, int32_t log_lanes) {
  typedef NormVec<T, V> Vec;
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  if (s.row >= a.T) return;
  const int64_t id = embed_id<I>(a, (int32_t)s.row);
  const bool good = id >= 0 && id < a.V;
  if (!good && a.status && s.first == 0) *a.status = 1;
  const T* w = reinterpret_cast<const T*>(a.w) + (good ? id : 0) * a.w_t;
  T* out = reinterpret_cast<T*>(a.out) + s.row * (int64_t)a.H;
  // (a row that an id out of range asks for is NaN, which no loss hides)
  const float scale = good ? a.scale : __builtin_nanf("");
  typename Vec::Raw raw[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (s.first + k * s.step < s.nv) raw[k] = Vec::raw(w + (int64_t)(s.first + k * s.step) * V);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = s.first + k * s.step;
    if (v >= s.nv) continue;
    float x[V];
    Vec::open(raw[k], x);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] *= scale;
    Vec::store(out + (int64_t)v * V, x);
  }
}

// The sum of v over the 1024 threads of the workgroup and over those before this one.
__device__ __forceinline__ int32_t embed_scan(int32_t v, int32_t* sums, int32_t& before) {
  int32_t in = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t up = __shfl_up(in, d);
    if ((int)lane_id() >= d) in += up;
  }
  __syncthreads();  // (sums may still be read from the call before)
  if (lane_id() == 63) sums[wave_id()] = in;
  __syncthreads();
  int32_t all = 0;
  before = in - v;
  for (int w = 0; w < 16; ++w) {
    if (w < (int)wave_id()) before += sums[w];
    all += sums[w];
  }
  return all;
}

template <class I>
__global__ __launch_bounds__(1024) void embed_sort_kernel(EmbedArgs a) {
  __shared__ int32_t counts[16 * kEmbedSlots];  // [wave][slot]
  __shared__ int32_t sums[16];
  const int32_t bucket = blockIdx.x, mask = (1 << a.log_buckets) - 1, per = a.per;
  int32_t* own = counts + wave_id() * per;
  for (int32_t i = threadIdx.x; i < 16 * per; i += 1024) counts[i] = 0;
  __syncthreads();
  // this wave's tokens: a run of whole groups of 64
  const int64_t run = ((int64_t)a.T + 1023) / 1024 * 64;
  const int64_t begin = run * wave_id(), end = begin + run < a.T ? begin + run : a.T;
  int32_t less = 0;
#pragma unroll 4
  for (int64_t t = begin + lane_id(); t < end; t += 64) {
    const int64_t id = embed_id<I>(a, (int32_t)t);
    if (id < 0 || id >= a.V || id == a.padding) continue;
    const int32_t b = (int32_t)id & mask;
    less += b < bucket;
    if (b == bucket) atomicAdd(&own[(int32_t)id >> a.log_buckets], 1);
  }
  int32_t before;
  const int32_t base = embed_scan(less, sums, before);  // (its barriers end the counting)
  const int32_t slot = threadIdx.x;
  int32_t n = 0;
  if (slot < per)
    for (int w = 0; w < 16; ++w) n += counts[w * per + slot];
  const int32_t all = embed_scan(n, sums, before);
  if (slot < per) {
    int32_t at = base + before;
    a.starts[bucket * per + slot] = at;
    for (int w = 0; w < 16; ++w) {
      const int32_t c = counts[w * per + slot];
      counts[w * per + slot] = at;
      at += c;
    }
  }
  if (bucket == mask && threadIdx.x == 0) a.starts[(bucket + 1) * per] = base + all;
  __syncthreads();
  for (int64_t t0 = begin; t0 < end; t0 += 64) {
    const int64_t t = t0 + lane_id();
    const int64_t id = t < end ? embed_id<I>(a, (int32_t)t) : -1;
    const bool mine = id >= 0 && id < a.V && id != a.padding && ((int32_t)id & mask) == bucket;
    const int32_t s = (int32_t)id >> a.log_buckets;
    uint64_t left = __ballot(mine);
    while (left) {  // each distinct id among these 64 tokens
      const int leader = __builtin_ctzll(left);
      const int32_t which = __builtin_amdgcn_readlane(s, leader);
      const uint64_t same = __ballot(mine && s == which);
      int32_t at = 0;
      if ((int)lane_id() == leader) at = atomicAdd(&own[which], __popcll(same));
      at = __builtin_amdgcn_readlane(at, leader);
      if (mine && s == which) a.order[at + __popcll(same & ((1ull << lane_id()) - 1))] = (int32_t)t;
      left &= ~same;
    }
  }
}

// sum[k] += the rows of dout of the tokens order[p0 .. p1), in their order.
template <class T, int V, int K>
__device__ __forceinline__ void embed_add_rows(const EmbedArgs& a, const EmbedSpan& s, int32_t p0,
                                               int32_t p1, float (&sum)[K][V]) {
  typedef NormVec<T, V> Vec;
  constexpr int U = 4;  // rows in flight
  const T* dout = reinterpret_cast<const T*>(a.dout);
  for (int32_t p = p0; p < p1; p += U) {
    typename Vec::Raw raw[U][K];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u >= p1) continue;
      const T* row = dout + (int64_t)a.order[p + u] * a.dout_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s.first + k * s.step < s.nv) raw[u][k] = Vec::raw(row + (int64_t)(s.first + k * s.step) * V);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u >= p1) continue;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (s.first + k * s.step >= s.nv) continue;
        float x[V];
        Vec::open(raw[u][k], x);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[k][i] += x[i];
      }
    }
  }
}

// Piece r of the sorted tokens: what of it belongs to rows of more than kEmbedPiece
// tokens.  Such a row is here from the start of the piece on (partial row 2 r), or
// begins inside and goes on behind it (2 r + 1): at most one of each.
template <class T, class I, int V, int K>
__global__ __launch_bounds__(256) void embed_pieces_kernel(EmbedArgs a, int32_t log_lanes) {
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  const int64_t total = a.starts[(int64_t)a.per << a.log_buckets];
  const int64_t p0 = s.row * kEmbedPiece;
  if (p0 >= total) return;
  const int32_t end = (int32_t)(p0 + kEmbedPiece < total ? p0 + kEmbedPiece : total);
  for (int32_t p = (int32_t)p0; p < end;) {
    const int32_t place = embed_place(a, (int32_t)embed_id<I>(a, a.order[p]));
    const int32_t s0 = a.starts[place], s1 = a.starts[place + 1];
    if (s1 - s0 > kEmbedPiece) {
      float sum[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) sum[k][i] = 0.f;
      embed_add_rows<T, V, K>(a, s, p, s1 < end ? s1 : end, sum);
      float* to = a.part + (2 * s.row + (s0 > (int32_t)p0)) * a.part_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s.first + k * s.step < s.nv)
#pragma unroll
          for (int i = 0; i < V; ++i) to[(int64_t)(s.first + k * s.step) * V + i] = sum[k][i];
    }
    p = s1;
  }
}

// Every row of dW (ADD false), or of each id that occurs, added to the accumulator:
// then row r stands for the r-th sorted token, where that is the first of its id.
template <class T, class I, int V, int K, bool ADD>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs a, int32_t log_lanes) {
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  int64_t id = s.row;
  if (ADD) {
    if (s.row >= a.starts[(int64_t)a.per << a.log_buckets]) return;
    id = embed_id<I>(a, a.order[s.row]);
  } else if (id >= a.V) {
    return;
  }
  const int32_t place = embed_place(a, (int32_t)id);
  const int32_t s0 = a.starts[place], s1 = a.starts[place + 1];
  if (ADD && s0 != s.row) return;
  float sum[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[k][i] = 0.f;
  if (s1 - s0 <= kEmbedPiece) {
    embed_add_rows<T, V, K>(a, s, s0, s1, sum);
  } else {
    const int32_t c0 = s0 / kEmbedPiece, c1 = (s1 - 1) / kEmbedPiece;
#pragma unroll 4
    for (int32_t c = c0; c <= c1; ++c) {
      const float* from = a.part + (2 * (int64_t)c + (c == c0 && s0 % kEmbedPiece != 0)) * a.part_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s.first + k * s.step < s.nv)
#pragma unroll
          for (int i = 0; i < V; ++i) sum[k][i] += from[(int64_t)(s.first + k * s.step) * V + i];
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = s.first + k * s.step;
    if (v >= s.nv) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[k][i] *= a.scale;
    if constexpr (ADD) {
      float* to = reinterpret_cast<float*>(a.dw) + id * a.dw_t + (int64_t)v * V;
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] += sum[k][i];
    } else {
      NormVec<T, V>::store(reinterpret_cast<T*>(a.dw) + id * a.dw_t + (int64_t)v * V, sum[k]);
    }
  }
}

}  // namespace mtf

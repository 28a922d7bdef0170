// Token embedding and its gradient (gfx950).
//
//   out[t] = scale W[id_t]                       (fp32, rounded once)
//   dW[v]  = scale sum over t with id_t = v of dout[t]
//
// Both are bound by memory: 65536 tokens into 128256 x 4096 in bf16, the lookup 160 us (5.8
// TB/s of rows read and written), the gradient 22 + 84 + 235 us, of which 1.05 GB of dW are
// the most.  The gradient sums rows of dout that lie anywhere; fp32
// atomics would repeat nothing and collide on the frequent tokens, so the tokens are
// sorted by id first (embed_sort_kernel) and each row of dW has one owner that adds its
// tokens in their order and writes the row once (embed_rows_kernel).  A row of more
// than kEmbedPiece tokens is summed in pieces by as many workgroups beforehand
// (embed_pieces_kernel), since a tokenizer's most frequent ids each own some per cent
// of all tokens; its owner adds the pieces in their order.  So results repeat.
//
// The sort is one launch without a word between workgroups: workgroup b of the buckets
// takes the ids equal to b modulo their number (the frequent ids, which lie side by side,
// come apart), reads all ids, counts the tokens of smaller buckets, which is where its
// own begin, and the tokens of each of its ids per wave; a scan over (id, wave) then
// gives each wave its places, which the tokens kept in LDS from the first pass fill in
// (or, where they were too many, a second reading of the ids).  It reads every id once
// per bucket, out of L2, 512 ids of a wave in flight.
// Up to kEmbedDirect tokens nothing is sorted: each row of dW looks through all ids by
// itself (embed_direct_kernel), one launch for three.
#pragma once

#include "flce_device.h"

namespace mtf {

constexpr int kEmbedSlots = 1024;    // ids of a bucket at most (64 KiB of counters)
constexpr int32_t kEmbedPiece = 32;  // tokens of a piece
constexpr int kEmbedFlight = 2;       // rows of dout, or partial rows, that a row of dW has in flight
constexpr int32_t kEmbedList = 512;  // tokens of a bucket and wave that are kept between its passes
constexpr int32_t kEmbedDirect = 256;  // tokens that are not sorted, at most

// V elements of T, 16 bytes or one element, aligned as one: rows of an odd width begin
// anywhere, and the memory instructions take any address of an element (gradient of 447
// tokens into 67988 x 4415 in bf16 by single elements 317 us, so 147; of 65536 into 32000 x
// 4095 314 and 215, the lookup 427 and 192).
template <class T, int V>
struct EmbedVec {
  typedef T Whole __attribute__((ext_vector_type(V)));
  typedef Whole Raw __attribute__((aligned(sizeof(T))));
  __device__ __forceinline__ static Raw raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ static void open(const Raw& v, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)v[i];
  }
  __device__ __forceinline__ static void store(T* p, const float (&x)[V]) {
    Whole v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)x[i];
    *reinterpret_cast<Raw*>(p) = v;
  }
};

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
  int32_t log_buckets, per, wide;  // wide: ids of 64 bits
  float scale;
};

__device__ __forceinline__ int64_t embed_id(const EmbedArgs& a, int32_t t) {
  return a.wide ? reinterpret_cast<const int64_t*>(a.ids)[t] : reinterpret_cast<const int32_t*>(a.ids)[t];
}
// Place of a valid id among all ids as they are sorted.
__device__ __forceinline__ int32_t embed_place(const EmbedArgs& a, int32_t id) {
  return (id & ((1 << a.log_buckets) - 1)) * a.per + (id >> a.log_buckets);
}

// A row is read by 2^log_lanes lanes of a wave, K vectors of V elements each; rows
// wider than a wave's 64 K vectors are cut into column chunks, narrower ones share a
// wave.  The last vector ends with the row: where V does not divide H it begins within
// the one before, with equal values (H is at least V).
struct EmbedSpan {
  int64_t row;                 // this lane's
  int32_t first, step, nv, H;  // its first vector, the distance to its next, a row's vectors
  template <int V>
  __device__ __forceinline__ int32_t at(int32_t v) const {  // the first element of vector v
    return v * V < H - V ? v * V : H - V;
  }
};
template <int V, int K>
__device__ __forceinline__ EmbedSpan embed_span(int32_t H, int32_t log_lanes) {
  EmbedSpan s;
  s.H = H;
  s.nv = (H + V - 1) / V;
  s.step = 1 << log_lanes;
  const uint32_t unit = blockIdx.x * 4u + wave_id();  // (below 2^26: 2^32 threads)
  const uint32_t lane = lane_id() & (uint32_t)(s.step - 1);
  const uint32_t chunks = log_lanes == 6 ? (uint32_t)(s.nv + 64 * K - 1) / (64u * K) : 1u;
  const uint32_t rows = chunks == 1 ? unit : unit / chunks;
  s.first = (int32_t)((unit - rows * chunks) * 64u * K + lane);
  s.row = (int64_t)rows * (64 >> log_lanes) + (lane_id() >> log_lanes);
  return s;
}

template <class T, int V, int K>
__global__ __launch_bounds__(256) void embed_forward_kernel(EmbedArgs a, int32_t log_lanes) {
  typedef EmbedVec<T, V> Vec;
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  if (s.row >= a.T) return;
  const int64_t id = embed_id(a, (int32_t)s.row);
  const bool good = id >= 0 && id < a.V;
  if (!good && a.status && s.first == 0) *a.status = 1;
  const T* w = reinterpret_cast<const T*>(a.w) + (good ? id : 0) * a.w_t;
  T* out = reinterpret_cast<T*>(a.out) + s.row * (int64_t)a.H;
  // (a row that an id out of range asks for is NaN, which no loss hides)
  const float scale = good ? a.scale : __builtin_nanf("");
  typename Vec::Raw raw[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (s.first + k * s.step < s.nv) raw[k] = Vec::raw(w + s.template at<V>(s.first + k * s.step));
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = s.first + k * s.step;
    if (v >= s.nv) continue;
    float x[V];
    Vec::open(raw[k], x);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] *= scale;
    Vec::store(out + s.template at<V>(v), x);
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

// An id as an unsigned number that is V or more where it does not count.
__device__ __forceinline__ uint32_t embed_key(int32_t id, uint32_t padding) {
  return (uint32_t)id == padding ? 0xffffffffu : (uint32_t)id;
}
__device__ __forceinline__ uint32_t embed_key(int64_t id, uint32_t padding) {
  return (uint64_t)id >> 32 ? 0xffffffffu : embed_key((int32_t)id, padding);
}

template <class I>
__global__ __launch_bounds__(1024) void embed_sort_kernel(EmbedArgs a) {
  __shared__ int32_t counts[16 * kEmbedSlots];  // [wave][slot]
  // the bucket's tokens among a wave's, as they come: place in the run << 10 | slot
  __shared__ uint32_t list[16][kEmbedList];
  __shared__ int32_t sums[16];
  static_assert(kEmbedSlots == 1 << 10, "slots of 10 bits");
  constexpr int U = 8;  // groups of 64 ids in flight
  const int32_t per = a.per;
  const uint32_t bucket = blockIdx.x, mask = (1u << a.log_buckets) - 1, padding = (uint32_t)a.padding;
  int32_t* own = counts + wave_id() * per;
  uint32_t* mine = list[wave_id()];
  for (int32_t i = threadIdx.x; i < 16 * per; i += 1024) counts[i] = 0;
  __syncthreads();
  // this wave's tokens: a run of whole groups of 64
  const int64_t run = ((int64_t)a.T + 1023) / 1024 * 64;
  const int64_t begin = run * wave_id(), end = begin + run < a.T ? begin + run : a.T;
  auto fetch = [&](int64_t t0, uint32_t (&key)[U]) {
    const I* ids = reinterpret_cast<const I*>(a.ids) + t0 + lane_id();
    I id[U];
    if (t0 + 64 * U <= end) {
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = ids[u * 64];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = t0 + u * 64 + lane_id() < end ? ids[u * 64] : (I)-1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) key[u] = embed_key(id[u], padding);
  };
  int32_t less = 0, found = 0;
  for (int64_t t0 = begin; t0 < end; t0 += 64 * U) {
    uint32_t key[U];
    fetch(t0, key);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool counts_here = key[u] < (uint32_t)a.V;
      const uint32_t b = key[u] & mask, slot = key[u] >> a.log_buckets;
      less += counts_here && b < bucket;
      const bool here = counts_here && b == bucket;
      const uint64_t m = __ballot(here);
      if (!m) continue;
      if (here) {
        atomicAdd(&own[slot], 1);
        const int32_t at = found + __popcll(m & ((1ull << lane_id()) - 1));
        if (at < kEmbedList) mine[at] = (uint32_t)(t0 - begin + u * 64 + lane_id()) << 10 | slot;
      }
      found += __popcll(m);
    }
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
  // places for up to 64 tokens of this wave, in their order
  auto place = [&](bool here, uint32_t s, int64_t t) {
    uint64_t left = __ballot(here);
    while (left) {  // each distinct id among them
      const int leader = __builtin_ctzll(left);
      const uint32_t which = __builtin_amdgcn_readlane(s, leader);
      const uint64_t same = __ballot(here && s == which);
      int32_t at = 0;
      if ((int)lane_id() == leader) at = atomicAdd(&own[which], __popcll(same));
      at = __builtin_amdgcn_readlane(at, leader);
      if (here && s == which) a.order[at + __popcll(same & ((1ull << lane_id()) - 1))] = (int32_t)t;
      left &= ~same;
    }
  };
  if (found <= kEmbedList && run <= 1 << 22) {  // (places in the run of 22 bits)
    for (int32_t i = 0; i < found; i += 64) {
      const bool here = i + (int32_t)lane_id() < found;
      const uint32_t e = here ? mine[i + lane_id()] : 0;
      place(here, e & 1023u, begin + (e >> 10));
    }
    return;
  }
  for (int64_t t0 = begin; t0 < end; t0 += 64 * U) {  // too many for the list: the ids again
    uint32_t key[U];
    fetch(t0, key);
#pragma unroll
    for (int u = 0; u < U; ++u)
      place(key[u] < (uint32_t)a.V && (key[u] & mask) == bucket, key[u] >> a.log_buckets,
            t0 + u * 64 + lane_id());
  }
}

// sum[k] += the rows of dout of U tokens from order[p] on, all on their way before the
// first is added.  WAVE: lane i holds the token of p0 + i, for the whole wave.  (Vectors
// past the row's end are read from its last one and never stored.)
template <class T, int V, int K, int U, bool WAVE>
__device__ __forceinline__ void embed_add(const EmbedArgs& a, const EmbedSpan& s, int32_t p, int32_t p0,
                                          int32_t token, float (&sum)[K][V]) {
  typedef EmbedVec<T, V> Vec;
  typename Vec::Raw raw[U][K];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int32_t t = WAVE ? __builtin_amdgcn_readlane(token, p + u - p0) : a.order[p + u];
    const T* row = reinterpret_cast<const T*>(a.dout) + (int64_t)t * a.dout_t;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = s.first + k * s.step;
      raw[u][k] = Vec::raw(row + s.template at<V>(v));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float x[V];
      Vec::open(raw[u][k], x);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[k][i] += x[i];
    }
}

// The same for the tokens order[p0 .. p1), in their order, U at a time (WAVE: at most 64).
template <class T, int V, int K, int U, bool WAVE>
__device__ __forceinline__ void embed_add_rows(const EmbedArgs& a, const EmbedSpan& s, int32_t p0,
                                               int32_t p1, int32_t token, float (&sum)[K][V]) {
  int32_t p = p0;
  for (; p + U <= p1; p += U) embed_add<T, V, K, U, WAVE>(a, s, p, p0, token, sum);
  if constexpr (U > 4) {
    if (p + 4 <= p1) embed_add<T, V, K, 4, WAVE>(a, s, p, p0, token, sum), p += 4;
  }
  if constexpr (U > 2) {
    if (p + 2 <= p1) embed_add<T, V, K, 2, WAVE>(a, s, p, p0, token, sum), p += 2;
  }
  if (p < p1) embed_add<T, V, K, 1, WAVE>(a, s, p, p0, token, sum);
}

// Piece r of the sorted tokens: what of it belongs to rows of more than kEmbedPiece
// tokens.  Such a row is here from the start of the piece on (partial row 2 r), or
// begins inside and goes on behind it (2 r + 1): at most one of each.  Each lane looks
// one token's row up (one after the other they took 14 of the 22 us of 16384 tokens of
// width 1536).  What bounds it is rows of dout in no order: 209 MB of them in 82 us with 2 to
// 8 in flight, half the rate of rows in their order.
template <class T, int V, int K>
__global__ __launch_bounds__(256) void embed_pieces_kernel(EmbedArgs a) {
  static_assert(kEmbedPiece <= 64, "a token of a piece for each lane");
  EmbedSpan s = embed_span<V, K>(a.H, 6);
  const int32_t total = a.starts[(int64_t)a.per << a.log_buckets];
  const int32_t p0 = (int32_t)__builtin_amdgcn_readfirstlane((int32_t)s.row) * kEmbedPiece;
  if (p0 >= total) return;
  const int32_t end = p0 + kEmbedPiece < total ? p0 + kEmbedPiece : total;
  int32_t s0 = 0, s1 = 0, token = 0;
  const int32_t p = p0 + (int32_t)lane_id();
  if (p < end) {
    token = a.order[p];
    const int32_t place = embed_place(a, (int32_t)embed_id(a, token));
    s0 = a.starts[place], s1 = a.starts[place + 1];
  }
  uint64_t left = __ballot(s1 - s0 > kEmbedPiece);
  while (left) {
    const int at = __builtin_ctzll(left);
    const int32_t begin = __builtin_amdgcn_readlane(s0, at), stop = __builtin_amdgcn_readlane(s1, at);
    const int32_t q0 = p0 + at, q1 = stop < end ? stop : end;
    left &= q1 - p0 < 64 ? ~0ull << (q1 - p0) : 0;
    float sum[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[k][i] = 0.f;
    embed_add_rows<T, V, K, 8, true>(a, s, q0, q1, __shfl(token, (int)lane_id() + at), sum);
    float* to = a.part + (2 * s.row + (begin > p0)) * a.part_t;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (s.first + k * s.step < s.nv)
#pragma unroll
        for (int i = 0; i < V; ++i) to[s.template at<V>(s.first + k * s.step) + i] = sum[k][i];
  }
}

// sum scaled into row id of dW, or added to it.
template <class T, int V, int K, bool ADD>
__device__ __forceinline__ void embed_put_row(const EmbedArgs& a, const EmbedSpan& s, int64_t id,
                                              float (&sum)[K][V]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = s.first + k * s.step;
    if (v >= s.nv) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[k][i] *= a.scale;
    if constexpr (ADD) {
      float* to = reinterpret_cast<float*>(a.dw) + id * a.dw_t + s.template at<V>(v);
      const int32_t twice = v * V - s.template at<V>(v);  // elements that are the vector's before
      if (twice == 0) {
        const typename EmbedVec<float, V>::Raw old = EmbedVec<float, V>::raw(to);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[k][i] += old[i];
        EmbedVec<float, V>::store(to, sum[k]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i >= twice) to[i] += sum[k][i];
      }
    } else {
      EmbedVec<T, V>::store(reinterpret_cast<T*>(a.dw) + id * a.dw_t + s.template at<V>(v), sum[k]);
    }
  }
}

// A word that no thread of the launch writes, read for the whole wave by a scalar load.
__device__ __forceinline__ int32_t embed_word(const int32_t* p, int64_t i) {
  typedef const __attribute__((address_space(4))) int32_t* const_ptr;
  return ((const_ptr)(uintptr_t)p)[i];
}

// sum[k] += U partial rows, every second one from `at` on, all on their way before the first
// is added.
template <int V, int K, int U>
__device__ __forceinline__ void embed_add_parts(const EmbedArgs& a, const EmbedSpan& s, int64_t at,
                                                float (&sum)[K][V]) {
  typedef EmbedVec<float, V> Vec;
  typename Vec::Raw raw[U][K];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = s.first + k * s.step;
      raw[u][k] = Vec::raw(a.part + (at + 2 * u) * a.part_t + s.template at<V>(v));
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[k][i] += raw[u][k][i];
}

// sum[k] = the sum of the sorted tokens [s0, s1), which are one row's.
template <class T, int V, int K, bool WAVE>
__device__ __forceinline__ void embed_sum_row(const EmbedArgs& a, const EmbedSpan& s, int32_t s0, int32_t s1,
                                              float (&sum)[K][V]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[k][i] = 0.f;
  if (s1 - s0 <= kEmbedPiece) {
    int32_t token = 0;
    if (WAVE && s0 + (int32_t)lane_id() < s1) token = a.order[s0 + lane_id()];
    embed_add_rows<T, V, K, kEmbedFlight, WAVE>(a, s, s0, s1, token, sum);
    return;
  }
  int32_t c = s0 / kEmbedPiece;
  const int32_t end = (s1 - 1) / kEmbedPiece + 1;
  embed_add_parts<V, K, 1>(a, s, 2 * (int64_t)c + (s0 % kEmbedPiece != 0), sum);
  for (++c; c + kEmbedFlight <= end; c += kEmbedFlight)
    embed_add_parts<V, K, kEmbedFlight>(a, s, 2 * (int64_t)c, sum);
  for (; c < end; ++c) embed_add_parts<V, K, 1>(a, s, 2 * (int64_t)c, sum);
}

// Every row of dW (ADD false), or of each id that occurs, added to the accumulator:
// then row r stands for the r-th sorted token, where that is the first of its id.
// Most rows have no token and wait for one lookup.  Scalar loads make it shorter (65536
// tokens into 128256 x 4096: 243 instead of 270 us), and few registers, with them many
// waves, hide it (4 rows of dout and 4 partial rows in flight instead of 2 and 2: 281;
// 4 or 8 rows to a wave: 283 and 286).
template <class T, int V, int K, bool ADD>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs a, int32_t log_lanes) {
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  const int32_t total = ADD ? embed_word(a.starts, (int64_t)a.per << a.log_buckets) : a.V;
  float sum[K][V];
  if (log_lanes == 6) {  // (one row for the wave)
    const int32_t row = __builtin_amdgcn_readfirstlane((int32_t)s.row);
    if (row >= total) return;
    const int32_t id = ADD ? (int32_t)embed_id(a, embed_word(a.order, row)) : row;
    const int32_t place = embed_place(a, __builtin_amdgcn_readfirstlane(id));
    const int32_t s0 = embed_word(a.starts, place), s1 = embed_word(a.starts, place + 1);
    if (ADD && s0 != row) return;
    embed_sum_row<T, V, K, true>(a, s, s0, s1, sum);
    embed_put_row<T, V, K, ADD>(a, s, id, sum);
    return;
  }
  if (s.row >= total) return;
  const int64_t id = ADD ? embed_id(a, a.order[s.row]) : s.row;
  const int32_t place = embed_place(a, (int32_t)id);
  const int32_t s0 = a.starts[place], s1 = a.starts[place + 1];
  if (ADD && s0 != s.row) return;
  embed_sum_row<T, V, K, false>(a, s, s0, s1, sum);
  embed_put_row<T, V, K, ADD>(a, s, id, sum);
}

// The same for at most kEmbedDirect tokens: the lanes of a wave hold 64 ids at a time,
// and each row takes those that are its own.  With ADD row r stands for token r, where no
// token before it has its id.
template <class T, int V, int K, bool ADD>
__global__ __launch_bounds__(256) void embed_direct_kernel(EmbedArgs a, int32_t log_lanes) {
  const EmbedSpan s = embed_span<V, K>(a.H, log_lanes);
  const int32_t group = lane_id() >> log_lanes;
  int64_t id = -1;  // (a row that is not there takes no token)
  if (s.row < (ADD ? a.T : a.V)) id = ADD ? embed_id(a, (int32_t)s.row) : s.row;
  const bool there = id >= 0 && id < a.V;
  if (id == a.padding || !there) id = -1;
  const int32_t wanted = (int32_t)id;
  const T* dout = reinterpret_cast<const T*>(a.dout);
  bool first = true;  // no token of the row has come yet
  bool owner = there && (!ADD || id >= 0);
  float sum[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[k][i] = 0.f;
  for (int32_t t0 = 0; t0 < a.T; t0 += 64) {
    const int32_t t = t0 + (int32_t)lane_id();
    const int64_t here = t < a.T ? embed_id(a, t) : -2;
    uint64_t mine = 0;
    for (int g = 0; g < 64 >> log_lanes; ++g) {
      const int32_t asks = __builtin_amdgcn_readlane(wanted, g << log_lanes);
      const uint64_t m = __ballot(here == (int64_t)asks && asks >= 0);
      if (g == group) mine = m;
    }
    if (ADD && mine && first) {
      first = false;
      owner = t0 + __builtin_ctzll(mine) == (int32_t)s.row;
    }
    if (!owner) mine = 0;
    while (mine) {
      const T* row = dout + (int64_t)(t0 + __builtin_ctzll(mine)) * a.dout_t;
      mine &= mine - 1;
      const bool two = mine != 0;
      const T* next = two ? dout + (int64_t)(t0 + __builtin_ctzll(mine)) * a.dout_t : row;
      mine &= mine - 1;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int32_t v = s.first + k * s.step;
        if (v >= s.nv) continue;
        const typename EmbedVec<T, V>::Raw r0 = EmbedVec<T, V>::raw(row + s.template at<V>(v));
        const typename EmbedVec<T, V>::Raw r1 = EmbedVec<T, V>::raw(next + s.template at<V>(v));
        float x[V], y[V];
        EmbedVec<T, V>::open(r0, x);
        EmbedVec<T, V>::open(r1, y);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sum[k][i] += x[i];
          if (two) sum[k][i] += y[i];
        }
      }
    }
  }
  if (owner) embed_put_row<T, V, K, ADD>(a, s, ADD ? id : s.row, sum);
}

}  // namespace mtf

// Orthogonalised updates by Newton-Schulz steps (gfx950).
//
//   X0 = G / (|G| + eps),   X <- a X + (b A + c A^2) X,   A = X X^T
//
// over the shorter side r of G [m, n] (X is G's transpose in the products where m > n).
// Each step is three products: A and A^2 are symmetric, so that only the tiles on and
// below the diagonal are computed and written twice.
//
// Number formats.  The products run on fp16 MFMA with fp32 sums; X itself is carried in
// fp32 from step to step and enters a X unrounded, since that term alone lifts the small
// singular values (by a^steps, 485 for the usual coefficients): a rounding there would be
// lifted with them.  A is rounded as E = A - mu I with mu its mean eigenvalue tr(A) / r:
//
//   b A + c A^2 = p(mu) I + (b + 2 c mu) E + c E^2,   p(t) = b t + c t^2
//   X <- (a + p(mu)) X + D X,   D = (b + 2 c mu) E + c E^2
//
// Around mu the terms no longer cancel (a + b + c = 0.7 out of 3.4, -4.8 and 2.0), and E
// is small where A is near a multiple of one.  fp32 updates take three products for each, of
// the values rounded to fp16 and of what that rounding left (1.1e-6 of the norm; fp32 products
// 2.9e-6).  bf16 updates take one, whose operand X~ is X rounded: D (X~ - X) is small where all
// eigenvalues of A lie near mu, but D is -p(mu) along singular vectors of small singular
// values, and what gets in there is lifted by the later steps as those are (half of the singular
// values strong, the others 0.05 of them: 0.004 of the norm after 5 steps, 0.04 after 12).  So
//
//   X <- (a + f p(mu)) X + (1 - f) p(mu) X~ + D X~,   f = max(0, 1 - |E|^2 / (r mu^2))
//
// with the error (M - f p(mu) I) (X~ - X), M = b A + c A^2.  Its sum over the eigenvalues, each
// lifted to about 1 in the end, is least where f mu is their harmonic mean: that ratio to mu is
// 1 - variance / mu^2 for large random matrices, and 0 where the eigenvalues spread further.  The
// last two steps, after which little is lifted, take f = 1.  |E|^2 is the trace of E^2, from
// the diagonal tiles of that product.  Five steps of the usual coefficients are then off by
// 0.0003 to 0.0016 of their norm before the last rounding to bf16, which itself is 0.0017, over
// nine kinds of spectra of 33 rows and more (products of bf16 operands: 0.018 at 4096 x 4096),
// by 0.002 where a few eigenvalues, which the variance does not show, lie far below many equal ones.
// Those coefficients do not settle, so that more steps carry errors on (12: 0.001 to 0.003,
// more where a singular value comes to lie where their map is steep); with ones that do it
// stays below the rounding.  fp16 copies are scaled by powers of two that keep them below 2^15.
//
// Copies of X in fp16: L [r, c], whose rows are contiguous along the long side (A), and
// S [c, r] (D X); a product writes both of the X it forms, out of one image in LDS.
// All rows end in zeros up to whole stages of 64.
//
// 4096 x 4096 in bf16: A 76 us, D 75 (1810 TFLOP/s if they were whole), D X 148 (141 in the
// last two steps), of which some 45 move X (4 bytes read, 8 written an element) with no product
// beside them: one tile of 256 x 256 fills a CU.  The products are bound by LDS (192 x 192 tiles) and the power limit
// (1.9 to 2.2 GHz).  28 of 256 x 1536: D X 31 us, 4.9 TB/s (much of it out of the cache behind L2):
// with four stages of K a tile's product, its reads of X and its writes follow one another.
#pragma once

#include "step_norm.h"
#include "update_gemm.h"

namespace mtf {

constexpr int kUpdParts = 1024;  // partial sums of squares of G, at most

// Per matrix, in fp32: the factor of X0 over its fp16 copy, mu, the two factors of X0
// over G, 2^k and 1 / (|G| + eps) / 2^k (their product leaves fp32's range where |G| does), and
// the power of two of G's fp16 copy.
enum { kUpdFactor = 0, kUpdInverse = 1, kUpdMu = 2, kUpdShift = 3, kUpdExponent = 4, kUpdState = 5 };

// f of a matrix with the trace `square` of E^2.  (Any f is right: where these numbers leave
// fp32's range it is one of 0 .. 1.)
__device__ __forceinline__ float upd_share(float square, float mu, int32_t r) {
  return fminf(fmaxf(1.f - square / ((float)r * mu * mu), 0.f), 1.f);
}

// 1 / (|G| + eps) in 64 bits; for a zero matrix, where it matters to nothing, one that fp32
// holds, so that X0 is zero and not its product with infinity.
__device__ __forceinline__ double upd_inverse(double norm, double eps) {
  return norm == 0.0 && eps > 0.0 ? 1.0 : 1.0 / (norm + eps);
}

struct UpdArgs {
  const char* in;
  char* out;
  char* ws;               // of the first matrix; the others follow ws_stride bytes apart
  int64_t ws_stride, in_row, in_batch;
  int64_t l, s0, s1, e, d, fragments, carrier, partial, spread, norm, state, parts;  // byte offsets
  double eps;
  int32_t m, n, r, c, ld_r, ld_c;        // ld_r, ld_c: r and c up to whole stages
  int32_t norm_parts, partials, spreads; // partial sums of |G|^2, of |X|^2, and of E^2's trace
  int32_t batch, tiles_m, tiles_n, tiles;
  int32_t split;                         // workgroups of a tile of A
  int32_t first, last;                   // of the steps
  int32_t lifted;                        // not of the last two steps: f counts (above)
  int32_t x_exponent;                    // X's fp16 copy is X 2^x_exponent, but for the first step's
  float a, b, cc;                        // the step's coefficients
  float x_unscale, e_scale, e_unscale, d_scale, d_unscale, x_scale;
  int32_t vec;                           // rows of G and of the result are whole 16-byte vectors
};

// Sums of squares of G, in 64 bits: workgroup p of norm_parts takes every
// norm_parts-th run of 256 vectors.
template <class T, int V>
__global__ __launch_bounds__(256) void upd_norm_kernel(UpdArgs a) {
  __shared__ double sums[4];
  const T* in = reinterpret_cast<const T*>(a.in) + (int64_t)blockIdx.y * a.in_batch;
  const int32_t per_row = (a.n + 256 * V - 1) / (256 * V);
  const int64_t runs = (int64_t)a.m * per_row;
  double s = 0.0;
  constexpr int U = 4;  // runs in flight
  for (int64_t u0 = blockIdx.x; u0 < runs; u0 += (int64_t)U * a.norm_parts) {
    T raw[U][V];
    bool there[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t u = u0 + (int64_t)k * a.norm_parts;
      const uint32_t row = (uint32_t)(u < runs ? u : 0) / (uint32_t)per_row;  // (runs: below 2^31)
      const int32_t col = (int32_t)((uint32_t)(u < runs ? u : 0) - row * per_row) * 256 * V + (int32_t)threadIdx.x * V;
      there[k] = u < runs && col < a.n;
      typedef T vec_t __attribute__((ext_vector_type(V)));
      const vec_t v = *reinterpret_cast<const vec_t*>(in + (there[k] ? row * a.in_row + col : 0));
#pragma unroll
      for (int i = 0; i < V; ++i) raw[k][i] = v[i];
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double x = there[k] ? (double)(float)raw[k][i] : 0.0;
        s = fma(x, x, s);
      }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
  if (lane_id() == 0) sums[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<double*>(a.ws + (int64_t)blockIdx.y * a.ws_stride + a.norm)[blockIdx.x] =
        sums[0] + sums[1] + sums[2] + sums[3];
}

__device__ __forceinline__ uint16_t upd_half(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ float upd_float(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }

// G as fp16, scaled by the power of two that brings its norm to 2^13 .. 2^14: a 64 x 64
// tile, as it lies and transposed, zeros up to whole stages.
template <class T, int V, int TERMS>
__global__ __launch_bounds__(256) void upd_convert_kernel(UpdArgs a) {
  __shared__ uint16_t tile[TERMS == 3 ? 2 : 1][64][66];
  __shared__ double sums[4];
  char* ws = a.ws + (int64_t)blockIdx.y * a.ws_stride;
  double s = 0.0;
  for (int i = threadIdx.x; i < a.norm_parts; i += 256) s += reinterpret_cast<const double*>(ws + a.norm)[i];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
  if (lane_id() == 0) sums[wave_id()] = s;
  __syncthreads();
  const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
  const double inverse = upd_inverse(norm, a.eps);
  const int exponent = norm > 0.0 && norm < INFINITY ? 13 - ilogb(norm) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    float* state = reinterpret_cast<float*>(ws + a.state);
    state[kUpdFactor] = (float)ldexp(inverse, -exponent);
    state[kUpdShift] = (float)ldexp(1.0, exponent / 2);
    state[kUpdInverse] = (float)ldexp(inverse, -(exponent / 2));
    state[kUpdMu] = (float)(norm * inverse * (norm * inverse) / a.r);
    state[kUpdExponent] = (float)exponent;
  }
  const int32_t across = (a.n + 63) / 64;
  const int32_t row0 = (int32_t)(blockIdx.x / across) * 64, col0 = (int32_t)(blockIdx.x % across) * 64;
  const int32_t i = threadIdx.x >> 2, j = (threadIdx.x & 3) * 16;
  const bool tall = a.m > a.n;
  const T* in = reinterpret_cast<const T*>(a.in) + (int64_t)blockIdx.y * a.in_batch;
  uint16_t* natural = reinterpret_cast<uint16_t*>(ws + (tall ? a.s0 : a.l));
  uint16_t* transposed = reinterpret_cast<uint16_t*>(ws + (tall ? a.l : a.s0));
  constexpr int64_t P = TERMS == 3 ? 2 : 1;
  const int64_t ld_nat = P * (tall ? a.ld_r : a.ld_c), ld_tr = P * (tall ? a.ld_c : a.ld_r);
  uint16_t part[TERMS == 3 ? 2 : 1][16];
  if constexpr (V == 1) {  // a wave reads 64 columns of 16 rows, and each thread its part out of LDS
    const int32_t col = col0 + (int32_t)lane_id(), w = (int32_t)wave_id() * 16;
    const T* from = in + (col < a.n ? col : a.n - 1);
    T x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = from[(int64_t)(row0 + w + k < a.m ? row0 + w + k : a.m - 1) * a.in_row];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float v = col < a.n && row0 + w + k < a.m ? ldexpf((float)x[k], exponent) : 0.f;
      const uint16_t h = upd_half(v);
      tile[0][w + k][lane_id()] = h;
      if constexpr (TERMS == 3) tile[1][w + k][lane_id()] = upd_half(v - upd_float(h));
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t)
#pragma unroll
      for (int k = 0; k < 16; ++k) part[t][k] = tile[t][i][j + k];
  } else {
#pragma unroll
    for (int k = 0; k < 16; k += V) {
      float x[V];
#pragma unroll
      for (int q = 0; q < V; ++q) x[q] = 0.f;
      if (row0 + i < a.m && col0 + j + k < a.n)  // (whole vectors)
        NormVec<T, V>::load(in + (int64_t)(row0 + i) * a.in_row + col0 + j + k, x);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const float v = ldexpf(x[q], exponent);
        part[0][k + q] = upd_half(v);
        if constexpr (TERMS == 3) part[1][k + q] = upd_half(v - upd_float(part[0][k + q]));
      }
    }
#pragma unroll
    for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t)
#pragma unroll
      for (int k = 0; k < 16; ++k) tile[t][i][j + k] = part[t][k];
  }
  if (row0 + i < a.m) {
#pragma unroll
    for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t) {
      u32x4_t* to = reinterpret_cast<u32x4_t*>(natural + (row0 + i) * ld_nat + upd_column<TERMS>(col0 + j, t));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t v;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[k] = (uint32_t)part[t][8 * h + 2 * k] | (uint32_t)part[t][8 * h + 2 * k + 1] << 16;
        to[h] = v;
      }
    }
  }
  __syncthreads();
  if (col0 + i >= a.n) return;
#pragma unroll
  for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t) {
    u32x4_t* to = reinterpret_cast<u32x4_t*>(transposed + (col0 + i) * ld_tr + upd_column<TERMS>(row0 + j, t));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_t v;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = (uint32_t)tile[t][j + 8 * h + 2 * k][i] | (uint32_t)tile[t][j + 8 * h + 2 * k + 1][i] << 16;
      to[h] = v;
    }
  }
}

// --- tiles -----------------------------------------------------------------------

template <int TERMS>
__device__ __forceinline__ UpdMatrix upd_matrix(const char* at, int32_t rows, int32_t ld) {
  const uint32_t wide = (uint32_t)ld * (TERMS == 3 ? 2u : 1u);
  return {at, (uint32_t)rows * wide * 2u, wide, (uint32_t)rows};
}

// A lane's place in the tile: fragment (fm, fn) holds four columns of one row.
template <int F>
struct UpdPlace {
  uint32_t row, col;
  __device__ __forceinline__ UpdPlace() {
    row = (wave_id() >> 1) * 16 * F + (lane_id() & 15u);
    col = (wave_id() & 1u) * 16 * F + 4 * (lane_id() >> 4);
  }
};

// Four values of the tile as fp16 into the image (plane 0), or what their rounding left.
template <int F>
__device__ __forceinline__ void upd_put(char* image, uint32_t row, uint32_t col, const float (&x)[4], bool rest) {
  f16x4_t h;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = (_Float16)x[i];
    if (rest) h[i] = (_Float16)(x[i] - (float)h[i]);
  }
  *reinterpret_cast<f16x4_t*>(image + row * upd_pitch(F) + col * 2) = h;
}

// The image's rows to rows row0.. (below `rows`) of a matrix, columns col0.. (below ld); t: to
// which of its terms.
template <int F, int TERMS>
__device__ __forceinline__ void upd_write_rows(const char* image, char* to, int t, int32_t row0, int32_t col0,
                                               int32_t rows, int32_t ld) {
  constexpr int64_t P = TERMS == 3 ? 2 : 1;
  constexpr int kChunks = upd_tile(F) / 8;
  for (int q = threadIdx.x; q < upd_tile(F) * kChunks; q += 256) {
    const int32_t i = q / kChunks, j = (q % kChunks) * 8;
    if (row0 + i < rows && col0 + j < ld)
      *reinterpret_cast<u32x4_t*>(to + ((row0 + i) * (P * ld) + upd_column<TERMS>(col0 + j, t)) * 2) =
          *reinterpret_cast<const u32x4_t*>(image + i * upd_pitch(F) + j * 2);
  }
}

typedef short i16x4_t __attribute__((ext_vector_type(4)));

// The image's columns to rows row0.. of a matrix: column i of the image is row row0 + i,
// image row j column col0 + j.  A transposing read hands lane i of 16 the column c0 + i
// of four rows (its lane 4 e + q reads columns c0 + 4 q .. of row e).
template <int F, int TERMS>
__device__ __forceinline__ void upd_write_columns(const char* image, char* to, int t, int32_t row0, int32_t col0,
                                                  int32_t rows, int32_t ld) {
  constexpr int64_t P = TERMS == 3 ? 2 : 1;
  constexpr int kTile = upd_tile(F);
  const uint32_t l = lane_id(), in = l & 15u;
  // a wave's unit: 16 columns of 32 rows, 8 rows to each 16 lanes
  for (int u = wave_id(); u < (kTile / 16) * (kTile / 32); u += 4) {
    const uint32_t c0 = (u % (kTile / 16)) * 16, j0 = (u / (kTile / 16)) * 32 + (l >> 4) * 8;
    const char* from = image + (j0 + (in >> 2)) * upd_pitch(F) + (c0 + 4 * (in & 3u)) * 2;
    typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)from);
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(from + 4 * upd_pitch(F)));
    const int32_t i = row0 + (int32_t)(c0 + in), j = col0 + (int32_t)j0;
    if (i < rows && j < ld) {
      struct { i16x4_t lo, hi; } both{lo, hi};
      *reinterpret_cast<u32x4_t*>(to + (i * (P * ld) + upd_column<TERMS>(j, t)) * 2) = __builtin_bit_cast(u32x4_t, both);
    }
  }
}

// Tile `at` of the lower triangle, in bands of 8 tile rows walked column by column.
__device__ __forceinline__ void upd_triangle(uint32_t at, uint32_t tiles, uint32_t& ti, uint32_t& tj) {
  uint32_t first = 0, rows = tiles < 8 ? tiles : 8;
  for (;;) {  // tiles of a band: the columns before it, full, and its own triangle
    const uint32_t n = rows * first + rows * (rows + 1) / 2;
    if (at < n) break;
    at -= n;
    first += rows;
    rows = tiles - first < 8 ? tiles - first : 8;
  }
  if (at < rows * first) {
    tj = at / rows;
    ti = first + at % rows;
  } else {
    at -= rows * first;
    uint32_t j = 0;
    while (at >= rows - j) at -= rows - j, ++j;
    tj = first + j;
    ti = first + j + at;
  }
  ti = __builtin_amdgcn_readfirstlane(ti);
  tj = __builtin_amdgcn_readfirstlane(tj);
}

// Both writes of a symmetric matrix's tile, whose fragment (fm, fn) value(fm, fn, x) gives.
template <int F, int TERMS, class Value>
__device__ __forceinline__ void upd_write_symmetric(char* lds, char* to, int32_t row0, int32_t col0, int32_t r,
                                                    int32_t ld, Value value) {
  const UpdPlace<F> p;
#pragma unroll
  for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int fm = 0; fm < F; ++fm) {
#pragma unroll
      for (int fn = 0; fn < F; ++fn) {
        float x[4];
        value(fm, fn, t, x);
        upd_put<F>(lds, p.row + 16 * fm, p.col + 16 * fn, x, t);
      }
      sched_fence();  // (a row of fragments at a time: all at once would spill)
    }
    __syncthreads();
    upd_write_rows<F, TERMS>(lds, to, t, row0, col0, r, ld);
    if (row0 != col0) upd_write_columns<F, TERMS>(lds, to, t, col0, row0, r, ld);
  }
}

// Where a lane's four values of a 16 x 16 fragment lie in a matrix kept by fragments, in
// elements: 64 lanes side by side.
__device__ __forceinline__ int64_t upd_fragment(int32_t row, int32_t col, int32_t across) {
  return ((int64_t)(row >> 4) * across + (col >> 4)) * 256 + 4 * (int32_t)lane_id();
}

// What upd_symmetric_kernel computes: E = A - mu I from L, whole tiles of it, its parts where
// a.split workgroups share a tile's long axis (few tiles), or the sum of these parts, in
// their order; or D = (b + 2 c mu) E + c E^2 from E.
enum { kUpdWhole, kUpdPart, kUpdJoin, kUpdSquare };

template <int F, int TERMS, int WHAT>
__global__ __launch_bounds__(256) void upd_symmetric_kernel(UpdArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[upd_lds(F)];
  float* sums = reinterpret_cast<float*>(lds);  // (before and after the tile)
  constexpr bool SQUARE = WHAT == kUpdSquare;
  const uint32_t group = xcd_remap(blockIdx.x, gridDim.x);
  const uint32_t id = WHAT == kUpdPart ? group / (uint32_t)a.split : group;
  const uint32_t matrix = id / (uint32_t)a.tiles, tile = id - matrix * (uint32_t)a.tiles;
  uint32_t ti, tj;
  upd_triangle(tile, (uint32_t)a.tiles_m, ti, tj);
  char* ws = a.ws + (int64_t)__builtin_amdgcn_readfirstlane(matrix) * a.ws_stride;
  const int32_t row0 = (int32_t)ti * upd_tile(F), col0 = (int32_t)tj * upd_tile(F);
  const UpdMatrix x = SQUARE ? upd_matrix<TERMS>(ws + a.e, a.r, a.ld_r) : upd_matrix<TERMS>(ws + a.l, a.r, a.ld_c);
  float* state = reinterpret_cast<float*>(ws + a.state);
  float mu = 0.f;
  if constexpr (WHAT == kUpdPart) {
  } else if constexpr (!SQUARE) {
    if (a.first) {
      mu = state[kUpdMu];
    } else {  // |X|^2 / r from the tiles of the product before: the same in every workgroup
      const float* partial = reinterpret_cast<const float*>(ws + a.partial);
      float s = 0.f;
      for (int k = threadIdx.x; k < a.partials; k += 256) s += partial[k];
      s = norm_wave_sum(s);
      if (lane_id() == 0) sums[wave_id()] = s;
      __syncthreads();
      mu = (sums[0] + sums[1] + sums[2] + sums[3]) / (float)a.r;
      __syncthreads();
      if (ti == 0 && threadIdx.x == 0) state[kUpdMu] = mu;
    }
  } else {
    mu = state[kUpdMu];
  }
  f32x4_t acc[F][F];
  // the parts of this tile, by fragments
  f32x4_t* parts = reinterpret_cast<f32x4_t*>(ws + a.parts) + (int64_t)tile * a.split * F * F * 256 + threadIdx.x;
  if constexpr (WHAT == kUpdJoin) {
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
      for (int n = 0; n < F; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int q = 0; q < a.split; ++q)
#pragma unroll
      for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) acc[m][n] += parts[(q * F * F + m * F + n) * 256];
  } else {
    UpdOperand<F> oa, ob;
    oa.init(x, (uint32_t)row0, (wave_id() >> 1) * 16 * F);
    ob.init(x, (uint32_t)col0, (wave_id() & 1u) * 16 * F);
    const int stages = (int)x.ld / kUpdStage;
    if constexpr (WHAT == kUpdPart) {
      const int part = (int)(group - id * (uint32_t)a.split);
      const int begin = stages * part / a.split, end = stages * (part + 1) / a.split;
      upd_mainloop<F, TERMS>(lds, oa, ob, begin, end - begin, acc);
#pragma unroll
      for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) parts[(part * F * F + m * F + n) * 256] = acc[m][n];
      return;
    } else {
      upd_mainloop<F, TERMS>(lds, oa, ob, 0, stages, acc);
    }
  }
  const UpdPlace<F> p;
  // E is also kept by fragments, for the product that squares it: the same lanes of the
  // same tile read it there
  const int32_t across = a.ld_r / 16;
  f16x4_t* kept = reinterpret_cast<f16x4_t*>(ws + a.fragments);
  const int64_t kept_plane = (int64_t)a.ld_r * a.ld_r / 4;
  // a wave's fragment that lies within whole stages of the matrix
  auto within = [&](int fm, int fn) {
    return row0 + (int32_t)(wave_id() >> 1) * 16 * F + 16 * fm < a.ld_r &&
           col0 + (int32_t)(wave_id() & 1u) * 16 * F + 16 * fn < a.ld_r;
  };
  if constexpr (!SQUARE) {
    const float f = (a.first ? state[kUpdFactor] * state[kUpdFactor] : a.x_unscale * a.x_unscale) * a.e_scale;
    const float centre = mu * a.e_scale;
    upd_write_symmetric<F, TERMS>(
        lds, ws + a.e, row0, col0, a.r, a.ld_r, [&](int fm, int fn, int t, float (&x)[4]) {
          const int32_t row = row0 + (int32_t)p.row + 16 * fm, col = col0 + (int32_t)p.col + 16 * fn;
          f16x4_t h;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = acc[fm][fn][i] * f;
            if (row == col + i && row < a.r) x[i] -= centre;
            h[i] = (_Float16)x[i];
            if (t) h[i] = (_Float16)(x[i] - (float)h[i]);
          }
          if (within(fm, fn)) kept[t * kept_plane + upd_fragment(row, col, across) / 4] = h;
        });
  } else {
    if constexpr (TERMS == 1) {
      if (a.lifted && ti == tj) {  // this tile's part of the trace of E^2
        float s = 0.f;
#pragma unroll
        for (int fm = 0; fm < F; ++fm)
#pragma unroll
          for (int fn = 0; fn < F; ++fn)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s += p.row + 16 * fm == p.col + 16 * fn + i ? acc[fm][fn][i] : 0.f;
        s = norm_wave_sum(s);
        if (lane_id() == 0) sums[wave_id()] = s;
        __syncthreads();
        if (threadIdx.x == 0)
          reinterpret_cast<float*>(ws + a.spread)[ti] =
              (sums[0] + sums[1] + sums[2] + sums[3]) * a.e_unscale * a.e_unscale;
        __syncthreads();
      }
    }
    const float linear = (a.b + 2.f * a.cc * mu) * a.e_unscale * a.d_scale;
    const float square = a.cc * a.e_unscale * a.e_unscale * a.d_scale;
    f16x4_t held[TERMS == 3 ? 2 : 1][F][F];  // (in the registers of the loop's fragments)
#pragma unroll
    for (int fm = 0; fm < F; ++fm)
#pragma unroll
      for (int fn = 0; fn < F; ++fn) {
        const int32_t row = row0 + (int32_t)p.row + 16 * fm, col = col0 + (int32_t)p.col + 16 * fn;
        const f16x4_t* at = kept + upd_fragment(row, col, across) / 4;
        held[0][fm][fn] = f16x4_t{0, 0, 0, 0};
        if constexpr (TERMS == 3) held[1][fm][fn] = f16x4_t{0, 0, 0, 0};
        if (!within(fm, fn)) continue;
        held[0][fm][fn] = at[0];
        if constexpr (TERMS == 3) held[1][fm][fn] = at[kept_plane];
      }
    upd_write_symmetric<F, TERMS>(
        lds, ws + a.d, row0, col0, a.r, a.ld_r, [&](int fm, int fn, int t, float (&x)[4]) {
          if (TERMS == 1 || t == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float e = (float)held[0][fm][fn][i];
              if constexpr (TERMS == 3) e += (float)held[1][fm][fn][i];
              x[i] = fmaf(linear, e, square * acc[fm][fn][i]);
            }
            if constexpr (TERMS == 3) acc[fm][fn] = f32x4_t{x[0], x[1], x[2], x[3]};
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = acc[fm][fn][i];
          }
        });
  }
}

typedef f32x4_t any_f32x4_t __attribute__((aligned(4)));

// X <- (a + f p(mu)) X + (1 - f) p(mu) X~ + D X~, as it lies in memory [m, n]: D S^T, or S D
// where m > n.  Writes the carried X, both fp16 copies and the tile's sum of squares, or at
// the last step the result.
// LIFTED: f counts (one kernel with a branch for it would spill).
template <class T, int F, int TERMS, bool LIFTED>
__global__ __launch_bounds__(256) void upd_apply_kernel(UpdArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[upd_lds(F)];
  float* sums = reinterpret_cast<float*>(lds);  // (before and after the tile)
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  const uint32_t matrix = __builtin_amdgcn_readfirstlane(id / (uint32_t)a.tiles);
  uint32_t tm, tn;
  grouped_tile(id - matrix * (uint32_t)a.tiles, (uint32_t)a.tiles_m, (uint32_t)a.tiles_n, 8, tm, tn);
  char* ws = a.ws + (int64_t)matrix * a.ws_stride;
  const int32_t row0 = (int32_t)tm * upd_tile(F), col0 = (int32_t)tn * upd_tile(F);
  const bool tall = a.m > a.n;
  const UpdMatrix d = upd_matrix<TERMS>(ws + a.d, a.r, a.ld_r), s = upd_matrix<TERMS>(ws + a.s0, a.c, a.ld_r);
  UpdOperand<F> oa, ob;
  oa.init(tall ? s : d, (uint32_t)row0, (wave_id() >> 1) * 16 * F);
  ob.init(tall ? d : s, (uint32_t)col0, (wave_id() & 1u) * 16 * F);
  f32x4_t acc[F][F];
  upd_mainloop<F, TERMS>(lds, oa, ob, 0, (int)d.ld / kUpdStage, acc);
  const float* state = reinterpret_cast<const float*>(ws + a.state);
  const float mu = state[kUpdMu];
  const float product = a.d_unscale * (a.first ? state[kUpdFactor] : a.x_unscale);
  const float around = mu * (a.b + a.cc * mu);
  float share = 1.f;
  if constexpr (LIFTED) {
    const float* spread = reinterpret_cast<const float*>(ws + a.spread);
    float s = 0.f;
    for (int32_t k = (int32_t)lane_id(); k < a.spreads; k += 64) s += spread[k];
    share = upd_share(norm_wave_sum(s), mu, a.r);
  }
  const float copied = (1.f - share) * around * (a.first ? state[kUpdFactor] : a.x_unscale);
  const int exponent = a.first ? (int)state[kUpdExponent] : a.x_exponent;
  const float linear = (a.a + share * around) * (a.first ? state[kUpdInverse] : 1.f);
  const float shift = a.first ? state[kUpdShift] : 1.f;
  const T* in = reinterpret_cast<const T*>(a.in) + (int64_t)matrix * a.in_batch;
  float* carrier = reinterpret_cast<float*>(ws + a.carrier);
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)matrix * a.m * a.n;
  const UpdPlace<F> p;
  const int32_t across = (a.n + 15) / 16;
  // a wave's fragment that lies at least partly within the matrix
  auto within = [&](int fm, int fn) {
    return row0 + (int32_t)(wave_id() >> 1) * 16 * F + 16 * fm < a.m &&
           col0 + (int32_t)(wave_id() & 1u) * 16 * F + 16 * fn < a.n;
  };
  // Whether four elements of G and of the result from `col` on go one by one: in fp32 where
  // the row ends within them (vectors lie at any element's address: 3 of 1001 x 1537 479 -> 470
  // us), in bf16 where not all rows are whole vectors (asked per fragment it costs the 256 x
  // 256 tiles of 14336 x 4096 2%)
  auto singly = [&](int32_t col) { return sizeof(T) == 4 ? col + 4 > a.n : !a.vec; };
  // X before the step: G, or what the last step left, which is zero past the matrix's ends
  auto fetch = [&](int fm, f32x4_t (&x)[F]) __attribute__((always_inline)) {
#pragma unroll
    for (int fn = 0; fn < F; ++fn) {
      x[fn] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (!within(fm, fn)) continue;
      const int32_t row = row0 + (int32_t)p.row + 16 * fm, col = col0 + (int32_t)p.col + 16 * fn;
      if (!a.first) {
        x[fn] = *reinterpret_cast<const f32x4_t*>(carrier + upd_fragment(row, col, across));
        continue;
      }
      const T* from = in + (int64_t)row * a.in_row + col;
      if (row >= a.m) continue;
      if (singly(col)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < a.n) x[fn][i] = (float)from[i];
      } else if (col < a.n) {
        if constexpr (sizeof(T) == 4) {
          x[fn] = *reinterpret_cast<const any_f32x4_t*>(from);
        } else {
          const u32x2_t v = *reinterpret_cast<const u32x2_t*>(from);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[fn][i] = __uint_as_float((i & 1) ? (v[i / 2] & 0xffff0000u) : (v[i / 2] << 16));
        }
      }
    }
  };
  // bf16 results of whole vectors leave through the image, the fp16 copies always
  const bool by_image = sizeof(T) == 2 && a.vec;
  float ss = 0.f;
  f32x4_t held[3][F];  // this row of fragments, and two on their way
  fetch(0, held[0]);
  if (F > 1) fetch(1, held[1]);
#pragma unroll
  for (int fm = 0; fm < F; ++fm) {
    if (fm + 2 < F) fetch(fm + 2, held[(fm + 2) % 3]);
#pragma unroll
    for (int fn = 0; fn < F; ++fn) {
      const int32_t row = row0 + (int32_t)p.row + 16 * fm, col = col0 + (int32_t)p.col + 16 * fn;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = fmaf(linear, held[fm % 3][fn][i] * shift, product * acc[fm][fn][i]);
        if constexpr (LIFTED)
          x[i] = fmaf(copied, upd_float(upd_half(ldexpf(held[fm % 3][fn][i], exponent))), x[i]);
        ss = fmaf(x[i], x[i], ss);
      }
      if (!a.last) {
        if (within(fm, fn))
          *reinterpret_cast<f32x4_t*>(carrier + upd_fragment(row, col, across)) = f32x4_t{x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= a.x_scale;
        upd_put<F>(lds, p.row + 16 * fm, p.col + 16 * fn, x, false);
        if constexpr (TERMS == 3) acc[fm][fn] = f32x4_t{x[0], x[1], x[2], x[3]};
      } else if (by_image) {
        *reinterpret_cast<u32x2_t*>(lds + (p.row + 16 * fm) * upd_pitch(F) + (p.col + 16 * fn) * 2) =
            u32x2_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
      } else if (row < a.m) {
        T* to = out + (int64_t)row * a.n + col;
        if (sizeof(T) == 2 || singly(col)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (col + i < a.n) to[i] = (T)x[i];
        } else if (col < a.n) {
          *reinterpret_cast<any_f32x4_t*>(to) = f32x4_t{x[0], x[1], x[2], x[3]};
        }
      }
    }
    sched_fence();
  }
  if (a.last) {
    if (!by_image) return;
    __syncthreads();
    upd_write_rows<F, 1>(lds, reinterpret_cast<char*>(out), 0, row0, col0, a.m, a.n);
    return;
  }
#pragma unroll
  for (int t = 0; t < (TERMS == 3 ? 2 : 1); ++t) {
    if (t) {
      __syncthreads();
#pragma unroll
      for (int fm = 0; fm < F; ++fm) {
#pragma unroll
        for (int fn = 0; fn < F; ++fn) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = acc[fm][fn][i];
          upd_put<F>(lds, p.row + 16 * fm, p.col + 16 * fn, x, true);
        }
        sched_fence();
      }
    }
    __syncthreads();
    char *l = ws + a.l, *next = ws + a.s1;
    if (tall) {
      upd_write_rows<F, TERMS>(lds, next, t, row0, col0, a.c, a.ld_r);
      upd_write_columns<F, TERMS>(lds, l, t, col0, row0, a.r, a.ld_c);
    } else {
      upd_write_rows<F, TERMS>(lds, l, t, row0, col0, a.r, a.ld_c);
      upd_write_columns<F, TERMS>(lds, next, t, col0, row0, a.c, a.ld_r);
    }
  }
  ss = norm_wave_sum(ss);
  __syncthreads();
  if (lane_id() == 0) sums[wave_id()] = ss;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<float*>(ws + a.partial)[id - matrix * (uint32_t)a.tiles] = sums[0] + sums[1] + sums[2] + sums[3];
}

}  // namespace mtf

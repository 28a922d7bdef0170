// Orthogonalised updates of small matrices (gfx950): all steps of one matrix in one
// workgroup and one launch, where the tiles of update_kernels.h would take three launches a
// step that mostly wait (128 x 352: 56 us here; 128 x 360 in 17 launches there 89).
//
// The mathematics and the number formats are those of update_kernels.h; bf16 matrices of at
// most 32 rows take three products to a term, too, where LDS holds both terms of X.  X [r, c]
// (r at most 128) lies in LDS in fp16, as do E and D; X in fp32 stays in the registers of the
// wave that owns its columns (16 at a time: fragment columns w, w + 8, ...).  Of the
// 8 waves each forms a block of up to 2 x 4 fragments of X X^T; where there are fewer blocks
// than waves the long axis is split between them and their parts are added in LDS one wave
// after the other, in a fixed order.  D X reads X's columns as operands through
// transposing LDS reads, and the wave that owns them writes them back.
// It is bound by LDS and by the barriers between its products: 128 x 352 in bf16 keeps the
// LDS of its CU busy for 58% of the 56 us (half of that conflicts), each SIMD's matrix
// instructions for 24%.  Its largest matrices are the last that profit: 64 x 416 in fp32 takes 58
// us here, 64 x 424 94 by the tiles.
#pragma once

#include "update_kernels.h"

namespace mtf {

constexpr int kUpdSmallSteps = 16;
constexpr int kUpdSmallLds = 160 * 1024;

struct UpdStep {
  float a, b, c, x_unscale, e_scale, e_unscale, d_scale, d_unscale, x_scale;
};
struct UpdSmallArgs {
  const char* in;
  char* out;
  int64_t in_row, in_batch;
  double eps;
  int32_t m, n, r, c, steps, vec;  // vec: as in UpdArgs
  UpdStep step[kUpdSmallSteps];
};

// Fragment columns of X that a wave owns at most, with R fragment rows: 128 or fewer
// registers hold them, and LDS the rest of what as many columns need.
constexpr int upd_small_columns(int R, int terms) {
  return terms == 3 ? (R == 1 ? 24 : R == 2 ? 12 : 4) : (R == 1 ? 32 : R == 2 ? 16 : R == 4 ? 8 : 3);
}
// Of these, how many go through a product together: they share its reads of D and hide each
// other's latencies.
constexpr int upd_small_group(int R) { return R == 1 ? 8 : R == 2 ? 4 : R == 4 ? 2 : 1; }
constexpr int upd_small_k(int R) { return R == 1 ? 32 : 16 * R; }              // K of E and D
constexpr int upd_small_pitch(int halves) { return halves * 2 + 16; }            // an odd number of 16 bytes
constexpr int upd_small_split(int R) { return R <= 2 ? 8 : R == 4 ? 4 : 1; }     // parts of the long axis
// Bytes of LDS for a matrix whose long side is c.
constexpr int64_t upd_small_lds(int R, int64_t c, int terms) {
  const int64_t planes = terms == 3 ? 2 : 1;
  return planes * 16 * R * (((c + 31) / 32 * 32) * 2 + 16) + 2 * planes * 16 * R * upd_small_pitch(upd_small_k(R)) +
         (upd_small_split(R) > 1 ? 16 * R * 16 * R * 4 : 0) + 128;
}

template <class T, int R, int TERMS>
__global__ __launch_bounds__(512) void upd_small_kernel(UpdSmallArgs a) {
  constexpr int P = TERMS == 3 ? 2 : 1, COLS = upd_small_columns(R, TERMS), K = upd_small_k(R), PE = upd_small_pitch(K);
  constexpr int GROUP = upd_small_group(R);
  static_assert(COLS % GROUP == 0, "whole groups");
  constexpr int BR = R < 2 ? R : 2, BC = R < 4 ? R : 4, BLOCKS = (R / BR) * (R / BC), SPLIT = upd_small_split(R);
  static_assert(BLOCKS * SPLIT == 8, "eight waves");
  __shared__ __attribute__((aligned(16))) char lds[kUpdSmallLds];
  const int32_t ld = (a.c + 31) / 32 * 32, PL = upd_small_pitch(ld);
  const int32_t plane_l = 16 * R * PL, plane_e = 16 * R * PE;
  char* const L = lds;
  char* const E = L + P * plane_l;
  char* const D = E + P * plane_e;
  float* const sum = reinterpret_cast<float*>(D + P * plane_e);  // [16 R][16 R] where SPLIT > 1
  double* const sums = reinterpret_cast<double*>(reinterpret_cast<char*>(sum) + (SPLIT > 1 ? 16 * R * 16 * R * 4 : 0));
  float* const spread = reinterpret_cast<float*>(sums + 8);  // [BLOCKS]
  const uint32_t l = lane_id(), w = wave_id(), l16 = l & 15u, g = l >> 4;
  const bool tall = a.m > a.n;
  const int64_t matrix = blockIdx.x;
  const T* in = reinterpret_cast<const T*>(a.in) + matrix * a.in_batch;
  T* out = reinterpret_cast<T*>(a.out) + matrix * a.m * a.n;
  typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

  // A fragment's operand: 16 rows of an LDS matrix, 8 halves from k on for each 16 lanes.
  auto operand = [&](const char* m, int32_t pitch, int f, int32_t kk) {
    return *reinterpret_cast<const u32x4_t*>(m + (16 * f + l16) * pitch + (32 * kk + 8 * g) * 2);
  };
  // products of fragments with both planes: value x rest, rest x value, value x value
  auto multiply = [&](const u32x4_t (&y)[P], const u32x4_t (&x)[P], f32x4_t c) {
    if constexpr (TERMS == 3) {
      c = upd_mma(y[1], x[0], c);
      c = upd_mma(y[0], x[1], c);
    }
    return upd_mma(y[0], x[0], c);
  };
  auto put = [&](char* m, int32_t plane, int32_t pitch, int32_t row, int32_t col, const float (&x)[4]) {
#pragma unroll
    for (int t = 0; t < P; ++t) {
      f16x4_t h;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = (_Float16)x[i];
        if (t) h[i] = (_Float16)(x[i] - (float)h[i]);
      }
      *reinterpret_cast<f16x4_t*>(m + t * plane + row * pitch + col * 2) = h;
    }
  };

  // G, as it is, by rows of its own into L's place as rows of X (from there, and not from
  // memory, each lane takes its elements: 16 x 4096 64 -> 20 us for the first step)
  const int32_t PT = P * PL;  // bytes of a row there
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  auto staged = [&](int32_t i, int32_t j) { return reinterpret_cast<T*>(L + i * PT) + j; };
  if (a.vec) {
    const uint32_t per = (uint32_t)a.n / V, all = (uint32_t)a.m * per;
#pragma unroll 4
    for (uint32_t q = threadIdx.x; q < all; q += 512) {
      const int32_t i = (int32_t)(q / per), j = (int32_t)(q % per) * V;
      const vec_t v = *reinterpret_cast<const vec_t*>(in + i * a.in_row + j);
      if (!tall) {
        *reinterpret_cast<vec_t*>(staged(i, j)) = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) *staged(j + e, i) = v[e];
      }
    }
  } else {
#pragma unroll 4
    for (uint32_t q = threadIdx.x; q < (uint32_t)a.m * (uint32_t)a.n; q += 512) {
      const int32_t i = (int32_t)(q / (uint32_t)a.n), j = (int32_t)(q % (uint32_t)a.n);
      *(tall ? staged(j, i) : staged(i, j)) = in[i * a.in_row + j];
    }
  }
  __syncthreads();
  typedef T four_t __attribute__((ext_vector_type(4)));
  f32x4_t x[COLS][R];
  double square = 0.0;
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    const int32_t col = 16 * (int32_t)(w + 8 * j) + 4 * (int32_t)g;
#pragma unroll
    for (int f = 0; f < R; ++f) x[j][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (16 * (int32_t)(w + 8 * j) >= a.c) continue;
#pragma unroll
    for (int f = 0; f < R; ++f) {
      const int32_t row = 16 * f + (int32_t)l16;
      const four_t v = *reinterpret_cast<const four_t*>(staged(row, col));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[j][f][i] = row < a.r && col + i < a.c ? (float)v[i] : 0.f;
        square = fma((double)x[j][f][i], (double)x[j][f][i], square);
      }
    }
    sched_fence();  // (here and below: what these columns need is gone before the next)
  }
  for (int32_t i = threadIdx.x; i < 2 * P * plane_e / 16; i += 512)
    reinterpret_cast<u32x4_t*>(E)[i] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) square += __shfl_down(square, d);
  if (l == 0) sums[w] = square;
  __syncthreads();
  square = 0.0;
  for (int i = 0; i < 8; ++i) square += sums[i];
  const double norm = sqrt(square), inverse = upd_inverse(norm, a.eps);
  const int exponent = norm > 0.0 && norm < INFINITY ? 13 - ilogb(norm) : 0;
  float unscale = (float)ldexp(inverse, -exponent);
  float mu = (float)(norm * inverse * (norm * inverse) / a.r);
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    const int32_t at = 16 * (int32_t)(w + 8 * j);
    if (at >= ld) continue;
#pragma unroll
    for (int f = 0; f < R; ++f) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = ldexpf(x[j][f][i], exponent);
        x[j][f][i] = v[i] * unscale;
      }
      put(L, plane_l, PL, 16 * f + l16, at + 4 * g, v);
    }
    sched_fence();
  }
  __syncthreads();

  const int block = w % BLOCKS, part = w / BLOCKS;
  const int fr = block / (R / BC) * BR, fc = block % (R / BC) * BC;  // the block's first fragments
  for (int step = 0; step < a.steps; ++step) {
    const UpdStep k = a.step[step];
    // E = A - mu I
    f32x4_t acc[BR][BC];
#pragma unroll
    for (int i = 0; i < BR; ++i)
#pragma unroll
      for (int j = 0; j < BC; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int32_t kk = part; kk < ld / 32; kk += SPLIT) {
      u32x4_t p[BR][P], q[BC][P];
#pragma unroll
      for (int t = 0; t < P; ++t) {
#pragma unroll
        for (int i = 0; i < BR; ++i) p[i][t] = operand(L + t * plane_l, PL, fr + i, kk);
#pragma unroll
        for (int j = 0; j < BC; ++j) q[j][t] = operand(L + t * plane_l, PL, fc + j, kk);
      }
#pragma unroll
      for (int i = 0; i < BR; ++i)
#pragma unroll
        for (int j = 0; j < BC; ++j) acc[i][j] = multiply(q[j], p[i], acc[i][j]);
    }
    const float f = unscale * unscale * k.e_scale, centre = mu * k.e_scale;
    if constexpr (SPLIT > 1) {
      for (int s = 0; s < SPLIT; ++s) {
        if (part == s) {
#pragma unroll
          for (int i = 0; i < BR; ++i)
#pragma unroll
            for (int j = 0; j < BC; ++j) {
              f32x4_t* to = reinterpret_cast<f32x4_t*>(sum + (16 * (fr + i) + l16) * 16 * R + 16 * (fc + j) + 4 * g);
              *to = s ? *to + acc[i][j] : acc[i][j];
            }
        }
        __syncthreads();
      }
      for (int32_t q = threadIdx.x; q < 16 * R * 4 * R; q += 512) {
        const int32_t row = q / (4 * R), col = q % (4 * R) * 4;
        const f32x4_t s = *reinterpret_cast<const f32x4_t*>(sum + row * 16 * R + col);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = s[i] * f - (row == col + i && row < a.r ? centre : 0.f);
        put(E, plane_e, PE, row, col, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < BR; ++i)
#pragma unroll
        for (int j = 0; j < BC; ++j) {
          const int32_t row = 16 * (fr + i) + (int32_t)l16, col = 16 * (fc + j) + 4 * (int32_t)g;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * f - (row == col + e && row < a.r ? centre : 0.f);
          put(E, plane_e, PE, row, col, v);
        }
    }
    __syncthreads();
    // D = (b + 2 c mu) E + c E^2
    if (part == 0) {
      const float linear = (k.b + 2.f * k.c * mu) * k.e_unscale * k.d_scale;
      const float squared = k.c * k.e_unscale * k.e_unscale * k.d_scale;
#pragma unroll
      for (int i = 0; i < BR; ++i)
#pragma unroll
        for (int j = 0; j < BC; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < K / 32; ++kk) {
        u32x4_t p[BR][P], q[BC][P];
#pragma unroll
        for (int t = 0; t < P; ++t) {
#pragma unroll
          for (int i = 0; i < BR; ++i) p[i][t] = operand(E + t * plane_e, PE, fr + i, kk);
#pragma unroll
          for (int j = 0; j < BC; ++j) q[j][t] = operand(E + t * plane_e, PE, fc + j, kk);
        }
#pragma unroll
        for (int i = 0; i < BR; ++i)
#pragma unroll
          for (int j = 0; j < BC; ++j) acc[i][j] = multiply(q[j], p[i], acc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < BR; ++i)
#pragma unroll
        for (int j = 0; j < BC; ++j) {
          const int32_t row = 16 * (fr + i) + (int32_t)l16, col = 16 * (fc + j) + 4 * (int32_t)g;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = 0.f;
#pragma unroll
          for (int t = 0; t < P; ++t) {
            const f16x4_t h = *reinterpret_cast<const f16x4_t*>(E + t * plane_e + row * PE + col * 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += (float)h[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(linear, v[e], squared * acc[i][j][e]);
          put(D, plane_e, PE, row, col, v);
        }
      if (TERMS == 1 && step + 2 < a.steps) {  // this block's part of the trace of E^2
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < BR; ++i)
#pragma unroll
          for (int j = 0; j < BC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s += 16 * (fr + i) + (int32_t)l16 == 16 * (fc + j) + 4 * (int32_t)g + e ? acc[i][j][e] : 0.f;
        s = norm_wave_sum(s);
        if (l == 0) spread[w] = s;
      }
    }
    __syncthreads();
    // X <- (a + f p(mu)) X + (1 - f) p(mu) X~ + D X~, each wave its columns
    const float around = mu * (k.b + k.c * mu);
    const bool lifted = TERMS == 1 && step + 2 < a.steps;
    float share = 1.f;
    if (lifted) {
      float s = 0.f;
      for (int i = 0; i < BLOCKS; ++i) s += spread[i];
      share = upd_share(s * k.e_unscale * k.e_unscale, mu, a.r);
    }
    const float product = k.d_unscale * unscale, linear = k.a + share * around;
    const float copied = (1.f - share) * around * unscale;
    float ss = 0.f;
#pragma unroll
    for (int j0 = 0; j0 < COLS; j0 += GROUP) {
      if (16 * (int32_t)(w + 8 * j0) >= ld) continue;
      f32x4_t y[GROUP][R];
#pragma unroll
      for (int j = 0; j < GROUP; ++j)
#pragma unroll
        for (int f = 0; f < R; ++f) y[j][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      // X~ of the group, on its way beside the products (where each element waited for its own,
      // 128 x 352 took 59 us)
      f16x4_t h[GROUP][TERMS == 1 ? R : 1];
      if constexpr (TERMS == 1) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
          const int32_t at = 16 * (int32_t)(w + 8 * (j0 + j));
#pragma unroll
          for (int f = 0; f < R; ++f)
            h[j][f] = *reinterpret_cast<const f16x4_t*>(L + (16 * f + l16) * PL + ((at < ld ? at : 0) + 4 * g) * 2);
        }
      }
#pragma unroll
      for (int kk = 0; kk < K / 32; ++kk) {
        // rows 32 kk + 8 g .. of a column's halves; a single fragment row has no more than 16
        // of these 32
        const int32_t k0 = 32 * kk + 8 * (int32_t)g;
        const char* from = L + ((k0 < 16 * R ? k0 : 0) + (int32_t)(l16 >> 2)) * PL + 8 * (int32_t)(l16 & 3u);
        u32x4_t q[GROUP][P];
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
#pragma unroll
          for (int t = 0; t < P; ++t) {
            const int32_t at = 16 * (int32_t)(w + 8 * (j0 + j));
            const char* p = from + t * plane_l + (at < ld ? at : 0) * 2;
            struct { i16x4_t lo, hi; } both;
            both.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)p);
            both.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 4 * PL));
            q[j][t] = __builtin_bit_cast(u32x4_t, both);
            if (R == 1 && k0 >= 16) q[j][t] = u32x4_t{0u, 0u, 0u, 0u};
          }
#pragma unroll
        for (int f = 0; f < R; ++f) {
          u32x4_t p[P];
#pragma unroll
          for (int t = 0; t < P; ++t) p[t] = operand(D + t * plane_e, PE, f, kk);
#pragma unroll
          for (int j = 0; j < GROUP; ++j) y[j][f] = multiply(q[j], p, y[j][f]);
        }
      }
#pragma unroll
      for (int j = 0; j < GROUP; ++j) {
        const int32_t at = 16 * (int32_t)(w + 8 * (j0 + j));
        if (at >= ld) continue;
#pragma unroll
        for (int f = 0; f < R; ++f) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = fmaf(linear, x[j0 + j][f][i], product * y[j][f][i]);
            if constexpr (TERMS == 1) v[i] = fmaf(copied, (float)h[j][f][i], v[i]);
            x[j0 + j][f][i] = v[i];
            ss = fmaf(v[i], v[i], ss);
            v[i] *= k.x_scale;  // (the last step's go nowhere)
          }
          put(L, plane_l, PL, 16 * f + l16, at + 4 * g, v);
        }
      }
      sched_fence();
    }
    if (step + 1 == a.steps) break;
    ss = norm_wave_sum(ss);
    if (l == 0) reinterpret_cast<float*>(sums)[w] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < 8; ++i) ss += reinterpret_cast<const float*>(sums)[i];
    mu = ss / (float)a.r;
    unscale = a.step[step + 1].x_unscale;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    const int32_t col = 16 * (int32_t)(w + 8 * j) + 4 * (int32_t)g;
    if (16 * (int32_t)(w + 8 * j) >= ld) continue;
#pragma unroll
    for (int f = 0; f < R; ++f) {
      four_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (T)x[j][f][i];
      *reinterpret_cast<four_t*>(staged(16 * f + l16, col)) = v;
    }
    sched_fence();
  }
  __syncthreads();
  if (a.vec) {
    const uint32_t per = (uint32_t)a.n / V, all = (uint32_t)a.m * per;
    for (uint32_t q = threadIdx.x; q < all; q += 512) {
      const int32_t i = (int32_t)(q / per), j = (int32_t)(q % per) * V;
      vec_t v;
      if (!tall) {
        v = *reinterpret_cast<const vec_t*>(staged(i, j));
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = *staged(j + e, i);
      }
      *reinterpret_cast<vec_t*>(out + (int64_t)i * a.n + j) = v;
    }
  } else {
    for (uint32_t q = threadIdx.x; q < (uint32_t)a.m * (uint32_t)a.n; q += 512) {
      const int32_t i = (int32_t)(q / (uint32_t)a.n), j = (int32_t)(q % (uint32_t)a.n);
      out[q] = *(tall ? staged(j, i) : staged(i, j));
    }
  }
}

}  // namespace mtf

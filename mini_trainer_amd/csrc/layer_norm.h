// Layer norm, with the residual addition before it or without (gfx950).
//
//   h = x, or residual_scale residual + block_scale x      (the new residual)
//   m = mean(h),  r = 1 / sqrt(mean((h - m)^2) + eps),  hn = (h - m) r
//   y = hn w + b
//
// and its gradient, with d = dy w:
//   g  = dh + r (d - mean(d) - hn mean(d hn))
//   dresidual = residual_scale g,  dx = block_scale g
//   dw = sum_t dy hn,  db = sum_t dy
//
// Rows live in registers as in step_norm.h, whose vectors, sums and column sums
// these kernels use.  The variance is the mean square of the centred row, formed from
// the registers in a second sum: E[h^2] - m^2 would cancel for rows whose mean is large
// against their deviation.
// In bf16 the forward keeps 8 bits of h beyond the rounded residual (lo), a byte per
// element against 16 of all else: with the rounded h alone dw is off by 0.0024 of its
// norm, its own rounding by 0.0017, and rows with a large mean lose more.
//
// Bound by HBM: 32768 x 4096 in bf16 with a residual, forward 206 us (5.9 TB/s of 1.21 GB),
// backward 235 us (5.2 TB/s of 1.23 GB).  Rows that are no whole vectors go by single
// elements (2999 x 1601 in fp32: 13 and 24 us, 2.9 and 2.4 TB/s).
#pragma once

#include "step_norm.h"

namespace mtf {

struct LayerNormArgs {
  const char *x, *residual, *w, *b;  // residual, w, b: null where absent
  const char *dy, *dh, *h;           // backward; h: the new residual, or x
  char *y, *h_out, *dx, *dresidual;
  uint8_t* lo;                       // [T, H], bf16 with a residual; null: not kept
  float *stat;                       // [2][T]: r, m
  float *part;                       // [2][parts][H]: dw, db
  int64_t x_t, r_t, dy_t, dh_t, h_t; // row pitches in elements
  int64_t T;
  int32_t H, parts;
  float eps, block_scale, residual_scale;
};

// The low byte of fp32 h beside hi, h rounded to bf16: the signed distance of h, rounded
// to 24 bits, from hi.  (0 for NaN; half a step up, 128, is taken as 127.)
__device__ __forceinline__ uint32_t low_byte(float h, float hi) {
  const int32_t d = (int32_t)((__float_as_uint(h) + 0x80u) >> 8) - (int32_t)(__float_as_uint(hi) >> 8);
  return h == h ? (uint32_t)(d > 127 ? 127 : d) & 0xffu : 0u;
}
__device__ __forceinline__ float with_low_byte(float hi, uint32_t byte) {
  return __uint_as_float(__float_as_uint(hi) + (uint32_t)((int32_t)(int8_t)byte * 256));
}

// V bytes of a row from element v V on.
template <int V>
struct LowBytes {
  typedef typename std::conditional<V == 1, uint8_t, u32x2_t>::type Raw;
  __device__ __forceinline__ static uint32_t at(const Raw& r, int i) {
    if constexpr (V == 1) return r;
    else return (r[i / 4] >> (8 * (i % 4))) & 0xffu;
  }
  __device__ __forceinline__ static void store(uint8_t* p, const float (&h)[V]) {
    Raw r;
    if constexpr (V == 1) {
      r = (uint8_t)low_byte(h[0], (float)(__bf16)h[0]);
    } else {
      r = Raw{0u, 0u};
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        float lo = h[i], hi = h[i + 1];
        round_pair(lo, hi);
        r[i / 4] |= (low_byte(h[i], lo) | low_byte(h[i + 1], hi) << 8) << (8 * (i % 4));
      }
    }
    *reinterpret_cast<Raw*>(p) = r;
  }
};

template <class T, int V, int K, int TPR, bool RES>
__global__ __launch_bounds__(norm_threads(TPR)) void layer_norm_fwd_kernel(LayerNormArgs a) {
  constexpr int kRows = norm_threads(TPR) / TPR;
  typedef NormVec<T, V> Vec;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (row >= a.T) return;  // (whole waves; with TPR > 64 the workgroup)
  const int32_t lane = threadIdx.x % TPR, nv = a.H / V;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_t;
  const float inv_h = 1.0f / (float)a.H;
  float h[K][V];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
#pragma unroll
    for (int i = 0; i < V; ++i) h[k][i] = 0.f;
    if (v < nv) {
      Vec::load(x + (int64_t)v * V, h[k]);
      if constexpr (RES) {
        float r[V];
        Vec::load(reinterpret_cast<const T*>(a.residual) + row * a.r_t + (int64_t)v * V, r);
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = fmaf(a.block_scale, h[k][i], a.residual_scale * r[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) s += h[k][i];
    }
  }
  if constexpr (RES) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      Vec::store(reinterpret_cast<T*>(a.h_out) + row * a.H + (int64_t)v * V, h[k]);
      if constexpr (sizeof(T) == 2) {
        if (a.lo) LowBytes<V>::store(a.lo + row * a.H + (int64_t)v * V, h[k]);
      }
    }
  }
  const float mean = norm_row_sum<TPR>(s, scratch, turn) * inv_h;
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (lane + k * TPR >= nv) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      h[k][i] -= mean;
      ss = fmaf(h[k][i], h[k][i], ss);
    }
  }
  const float rstd = 1.0f / sqrtf(norm_row_sum<TPR>(ss, scratch, turn) * inv_h + a.eps);
  if (lane == 0 && a.stat) {
    a.stat[row] = rstd;
    a.stat[a.T + row] = mean;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
    if (v >= nv) continue;
    float w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 1.f, b[i] = 0.f;
    if (a.w) Vec::load(reinterpret_cast<const T*>(a.w) + (int64_t)v * V, w);
    if (a.b) Vec::load(reinterpret_cast<const T*>(a.b) + (int64_t)v * V, b);
#pragma unroll
    for (int i = 0; i < V; ++i) h[k][i] = fmaf(h[k][i] * rstd, w[i], b[i]);
    Vec::store(reinterpret_cast<T*>(a.y) + row * a.H + (int64_t)v * V, h[k]);
  }
}

template <class T, int V, int K, int TPR, bool RES>
__global__ __launch_bounds__(norm_threads(TPR)) void layer_norm_bwd_kernel(LayerNormArgs a) {
  constexpr int kRows = norm_threads(TPR) / TPR;
  constexpr bool kLow = RES && sizeof(T) == 2;
  typedef NormVec<T, V> Vec;
  typedef LowBytes<V == 1 ? 1 : 8> Low;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int32_t lane = threadIdx.x % TPR, nv = a.H / V;
  const int32_t part = (int32_t)blockIdx.x * kRows + (int32_t)(threadIdx.x / TPR);
  const float inv_h = 1.0f / (float)a.H;
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  // the weight stays in registers over the rows, and the next row's tensors are on
  // their way while this one is worked on (single elements are read as they are used)
  constexpr bool kHold = V > 1;
  typename Vec::Raw w_raw[kHold ? K : 1];
  typename Vec::Raw r_h[kHold ? K : 1], r_dy[kHold ? K : 1], r_dh[kHold && RES ? K : 1];
  typename Low::Raw r_lo[kHold && kLow ? K : 1];
  if (kHold && a.w) {
#pragma unroll
    for (int k = 0; k < (kHold ? K : 0); ++k)
      if (lane + k * TPR < nv)
        w_raw[k] = Vec::raw(reinterpret_cast<const T*>(a.w) + (int64_t)(lane + k * TPR) * V);
  }
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < (kHold ? K : 0); ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      r_h[k] = Vec::raw(reinterpret_cast<const T*>(a.h) + row * a.h_t + (int64_t)v * V);
      r_dy[k] = Vec::raw(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + (int64_t)v * V);
      if constexpr (RES) {
        if (a.dh) r_dh[k] = Vec::raw(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + (int64_t)v * V);
      }
      if constexpr (kLow)
        r_lo[k] = *reinterpret_cast<const typename Low::Raw*>(a.lo + row * a.H + (int64_t)v * V);
    }
  };
  if (part < a.T) fetch(part);
  for (int64_t row = part; row < a.T; row += a.parts) {
    const float rstd = a.stat[row], mean = a.stat[a.T + row];
    float hn[K][V], g[K][V], d[RES ? K : 1][V];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hn[k][i] = g[k][i] = 0.f;
        if constexpr (RES) d[k][i] = 0.f;
      }
      if (v >= nv) continue;
      float w[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = 1.f;
      if constexpr (kHold) {
        if (a.w) Vec::open(w_raw[k], w);
        Vec::open(r_h[k], hn[k]);
        Vec::open(r_dy[k], g[k]);
        if constexpr (RES) {
          if (a.dh) Vec::open(r_dh[k], d[k]);
        }
        if constexpr (kLow) {
#pragma unroll
          for (int i = 0; i < V; ++i) hn[k][i] = with_low_byte(hn[k][i], Low::at(r_lo[k], i));
        }
      } else {
        if (a.w) Vec::load(reinterpret_cast<const T*>(a.w) + v, w);
        Vec::load(reinterpret_cast<const T*>(a.h) + row * a.h_t + v, hn[k]);
        Vec::load(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + v, g[k]);
        if constexpr (RES) {
          if (a.dh) Vec::load(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + v, d[k]);
        }
        if constexpr (kLow) hn[k][0] = with_low_byte(hn[k][0], a.lo[row * a.H + v]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hn[k][i] = (hn[k][i] - mean) * rstd;
        dw[k][i] = fmaf(g[k][i], hn[k][i], dw[k][i]);
        db[k][i] += g[k][i];
        g[k][i] *= w[i];
        s0 += g[k][i];
        s1 = fmaf(g[k][i], hn[k][i], s1);
      }
    }
    if (kHold && row + a.parts < a.T) fetch(row + a.parts);
    s0 = norm_row_sum<TPR>(s0, scratch, turn) * inv_h;
    s1 = norm_row_sum<TPR>(s1, scratch, turn) * inv_h;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        g[k][i] = rstd * (fmaf(-hn[k][i], s1, g[k][i]) - s0);
        if constexpr (RES) {
          g[k][i] += d[k][i];
          d[k][i] = a.residual_scale * g[k][i];
          g[k][i] *= a.block_scale;
        }
      }
      if constexpr (RES) {
        if (a.dresidual)
          Vec::store(reinterpret_cast<T*>(a.dresidual) + row * a.H + (int64_t)v * V, d[k]);
      }
      if (a.dx) Vec::store(reinterpret_cast<T*>(a.dx) + row * a.H + (int64_t)v * V, g[k]);
    }
  }
  if (part < a.parts) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t c = (int64_t)part * a.H + (int64_t)v * V + i;
        a.part[c] = dw[k][i];
        a.part[(int64_t)a.parts * a.H + c] = db[k][i];
      }
    }
  }
}

}  // namespace mtf

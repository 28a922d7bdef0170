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
// norm, its own rounding by 0.0017, and rows with a large mean lose more.  These 16 bits leave
// hn off by up to 2^-16 |m| r: nothing beside the gradients' own rounding up to means of
// 200 deviations, but dw is off by 0.0026 of its norm at 500, 0.0053 at 1000 and 0.019 at 4000,
// where 24 bits, at another byte an element each way, would give 0.0016.  (dx stays at 0.0017
// to 0.0019; y comes from the unrounded h, and without a residual, and in fp32, all of h is kept.)
// dw and db add each workgroup's rows one after the other and then up to 2048 partial rows
// in 16 runs: many short rows in fp32 are off by 2.4e-7 of their norm (1800 and 65536 x 64; sums
// in halves 1.6e-7 and 1.3e-7), 16384 x 4096 by 1.8e-7 (1.9e-7).
//
// Bound by HBM: 32768 x 4096 in bf16 with a residual, forward 206 us (5.9 TB/s of 1.21 GB),
// backward 235 us (5.2 TB/s of 1.23 GB); without one 105 (5.1 TB/s) and 162 (5.0); 16384 x
// 4096 in fp32 with one 184 (5.8) and 215 (5.0), without 104 (5.2) and 159 (5.1).  Rows of any width go by 16-byte vectors at the
// address of any element, the last one ending with the row: where it begins within the one
// before, both hold equal values, and the sums over a row take them once (16384 x 4095 in bf16 by
// single elements 259 and 426 us, so 136 and 174; 4096 wide 111 and 124).
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

// NormVec's vectors at the address of any element.
template <class T, int V>
struct LayerVec : NormVec<T, V> {
  typedef typename NormVec<T, V>::Raw Whole;
  typedef Whole Raw __attribute__((aligned(sizeof(T))));
  __device__ __forceinline__ static Raw raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ static void load(const T* p, float (&out)[V]) {
    const Whole v = *reinterpret_cast<const Raw*>(p);
    NormVec<T, V>::open(v, out);
  }
  __device__ __forceinline__ static void store(T* p, const float (&in)[V]) {
    Whole v;
    NormVec<T, V>::store(reinterpret_cast<T*>(&v), in);
    *reinterpret_cast<Raw*>(p) = v;
  }
};

// The first element of vector v of a row of H, and how many of it are the vector's before.
template <int V>
__device__ __forceinline__ int32_t layer_at(int32_t v, int32_t H) { return v * V < H - V ? v * V : H - V; }
template <int V>
__device__ __forceinline__ int32_t layer_twice(int32_t v, int32_t H) { return v * V - layer_at<V>(v, H); }

// V bytes of a row.
template <int V>
struct LowBytes {
  typedef typename std::conditional<V == 1, uint8_t, u32x2_t>::type Whole;
  typedef Whole Raw __attribute__((aligned(1)));
  __device__ __forceinline__ static uint32_t at(const Whole& r, int i) {
    if constexpr (V == 1) return r;
    else return (r[i / 4] >> (8 * (i % 4))) & 0xffu;
  }
  __device__ __forceinline__ static void store(uint8_t* p, const float (&h)[V]) {
    Whole r;
    if constexpr (V == 1) {
      r = (uint8_t)low_byte(h[0], (float)(__bf16)h[0]);
    } else {
      r = Whole{0u, 0u};
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
  typedef LayerVec<T, V> Vec;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (row >= a.T) return;  // (whole waves; with TPR > 64 the workgroup)
  const int32_t lane = threadIdx.x % TPR, nv = (a.H + V - 1) / V;
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
      const int32_t at = layer_at<V>(v, a.H);
      Vec::load(x + at, h[k]);
      if constexpr (RES) {
        float r[V];
        Vec::load(reinterpret_cast<const T*>(a.residual) + row * a.r_t + at, r);
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = fmaf(a.block_scale, h[k][i], a.residual_scale * r[i]);
      }
      const int32_t twice = v * V - at;
      if (twice == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) s += h[k][i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) s += i < twice ? 0.f : h[k][i];
      }
    }
  }
  if constexpr (RES) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      const int64_t at = row * a.H + layer_at<V>(v, a.H);
      Vec::store(reinterpret_cast<T*>(a.h_out) + at, h[k]);
      if constexpr (sizeof(T) == 2) {
        if (a.lo) LowBytes<V>::store(a.lo + at, h[k]);
      }
    }
  }
  const float mean = norm_row_sum<TPR>(s, scratch, turn) * inv_h;
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
    if (v >= nv) continue;
    const int32_t twice = layer_twice<V>(v, a.H);
#pragma unroll
    for (int i = 0; i < V; ++i) h[k][i] -= mean;
    if (twice == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(h[k][i], h[k][i], ss);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) ss = i < twice ? ss : fmaf(h[k][i], h[k][i], ss);
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
    const int32_t at = layer_at<V>(v, a.H);
    if (a.w) Vec::load(reinterpret_cast<const T*>(a.w) + at, w);
    if (a.b) Vec::load(reinterpret_cast<const T*>(a.b) + at, b);
#pragma unroll
    for (int i = 0; i < V; ++i) h[k][i] = fmaf(h[k][i] * rstd, w[i], b[i]);
    Vec::store(reinterpret_cast<T*>(a.y) + row * a.H + at, h[k]);
  }
}

template <class T, int V, int K, int TPR, bool RES>
__global__ __launch_bounds__(norm_threads(TPR)) void layer_norm_bwd_kernel(LayerNormArgs a) {
  constexpr int kRows = norm_threads(TPR) / TPR;
  constexpr bool kLow = RES && sizeof(T) == 2;
  typedef LayerVec<T, V> Vec;
  typedef LowBytes<V == 1 ? 1 : 8> Low;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int32_t lane = threadIdx.x % TPR, nv = (a.H + V - 1) / V;
  const int32_t part = (int32_t)blockIdx.x * kRows + (int32_t)(threadIdx.x / TPR);
  const float inv_h = 1.0f / (float)a.H;
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  // the weight stays in registers over the rows, and the next row's tensors are on
  // their way while this one is worked on (wider rows leave no registers for it:
  // 16384 x 12288 in bf16 391 us, held 1555)
  constexpr bool kHold = K * V * TPR <= 8192;
  typename Vec::Raw w_raw[kHold ? K : 1];
  typename Vec::Raw r_h[kHold ? K : 1], r_dy[kHold ? K : 1], r_dh[kHold && RES ? K : 1];
  typename Low::Raw r_lo[kHold && kLow ? K : 1];
  if (kHold && a.w) {
#pragma unroll
    for (int k = 0; k < (kHold ? K : 0); ++k)
      if (lane + k * TPR < nv)
        w_raw[k] = Vec::raw(reinterpret_cast<const T*>(a.w) + layer_at<V>(lane + k * TPR, a.H));
  }
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < (kHold ? K : 0); ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      const int32_t at = layer_at<V>(v, a.H);
      r_h[k] = Vec::raw(reinterpret_cast<const T*>(a.h) + row * a.h_t + at);
      r_dy[k] = Vec::raw(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + at);
      if constexpr (RES) {
        if (a.dh) r_dh[k] = Vec::raw(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + at);
      }
      if constexpr (kLow)
        r_lo[k] = *reinterpret_cast<const typename Low::Raw*>(a.lo + row * a.H + at);
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
        const int32_t at = layer_at<V>(v, a.H);
        if (a.w) Vec::load(reinterpret_cast<const T*>(a.w) + at, w);
        Vec::load(reinterpret_cast<const T*>(a.h) + row * a.h_t + at, hn[k]);
        Vec::load(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + at, g[k]);
        if constexpr (RES) {
          if (a.dh) Vec::load(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + at, d[k]);
        }
        if constexpr (kLow) {
          const typename Low::Whole lo = *reinterpret_cast<const typename Low::Raw*>(a.lo + row * a.H + at);
#pragma unroll
          for (int i = 0; i < V; ++i) hn[k][i] = with_low_byte(hn[k][i], Low::at(lo, i));
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hn[k][i] = (hn[k][i] - mean) * rstd;
        dw[k][i] = fmaf(g[k][i], hn[k][i], dw[k][i]);
        db[k][i] += g[k][i];
        g[k][i] *= w[i];
      }
      const int32_t twice = layer_twice<V>(v, a.H);
      if (twice == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          s0 += g[k][i];
          s1 = fmaf(g[k][i], hn[k][i], s1);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          s0 += i < twice ? 0.f : g[k][i];
          s1 = i < twice ? s1 : fmaf(g[k][i], hn[k][i], s1);
        }
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
      const int64_t at = row * a.H + layer_at<V>(v, a.H);
      if constexpr (RES) {
        if (a.dresidual) Vec::store(reinterpret_cast<T*>(a.dresidual) + at, d[k]);
      }
      if (a.dx) Vec::store(reinterpret_cast<T*>(a.dx) + at, g[k]);
    }
  }
  if (part < a.parts) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t c = (int64_t)part * a.H + layer_at<V>(v, a.H) + i;
        a.part[c] = dw[k][i];
        a.part[(int64_t)a.parts * a.H + c] = db[k][i];
      }
    }
  }
}

}  // namespace mtf

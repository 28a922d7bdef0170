// Residual and norms between two blocks of a decoder (gfx950).
//
//   u = x, or with a norm after the block  u = x / rms(x) (offset + pw)
//   h = residual_scale residual + block_scale gate u        (the new residual)
//   y = h / rms(h) (offset + w),   rms(t) = sqrt(mean(t^2) + eps)
//
// and its gradient, with hn = h / rms(h), xn = x / rms(x), dn = dy (offset + w):
//   gh = dh + (dn - hn mean(dn hn)) / rms(h)
//   dresidual = residual_scale gh,  du = block_scale gate gh
//   dx = du, or (du (offset + pw) - xn mean(du (offset + pw) xn)) / rms(x)
//   dw = sum_t dy hn,  dpw = sum_t du xn,  dgate = sums of block_scale gh u
//
// Both passes are bound by memory: each tensor is read once and written once
// (65536 x 4096 bf16, no norm or gate on x: forward 355 us, 6.0 TB/s, backward 385
// us, 5.6 TB/s; 16384 x 3584 with both: 86 us, 5.5 TB/s, and 147 us, 4.8 TB/s; a
// large copy reaches 5.2).  The backward fetches the next row while it reduces the
// present one: without that 506 and 233 us.
// The backward takes h as it was stored, rounded to the type, which saves an fp32
// copy of it (4 T H bytes written and read, against 8 T H of all else in bf16): its
// bf16 gradients are off by 0.0022 to 0.0025 of their norm, their own rounding alone
// by 0.0017.
// A row lives in the registers of its TPR threads (K vectors of V elements
// each) between its loads and its stores; everything is computed in fp32 and
// rounded once.  The weight gradients are summed in registers over the rows a
// workgroup walks, written as one partial row per group of TPR threads and
// added in a fixed order by norm_columns_kernel, so that results repeat.
#pragma once

#include <type_traits>

#include "flce_device.h"

namespace mtf {

struct NormArgs {
  const char *x, *residual, *w, *pw, *gate;  // pw, gate: null where absent
  const char *dy, *dh, *h;                   // backward: upstream gradients, new residual
  char *y, *h_out, *dx, *dresidual, *dgate;  // dgate: one per row or element (gate modes 2, 3)
  float *rstd;                               // [2][T]: 1 / rms(h), 1 / rms(x)
  float *part;                               // [3][parts][H]: dw, dpw, dgate (mode 1)
  int64_t x_t, r_t, gate_t, dy_t, dh_t, h_t; // row pitches in elements
  int64_t T;
  int32_t H, gate_mode, parts;               // gate: 0 none, 1 [H], 2 [T], 3 [T, H]
  float eps, block_scale, residual_scale, offset;
};

template <class T, int V>
struct NormVec {
  typedef typename std::conditional<V == 1, T, u32x4_t>::type Raw;  // V elements as they lie in memory
  __device__ __forceinline__ static Raw raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ static void open(const Raw& v, float (&out)[V]) {
    if constexpr (V == 1) {
      out[0] = (float)v;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(T) == 2)
          out[i] = __uint_as_float((i & 1) ? (v[i / 2] & 0xffff0000u) : (v[i / 2] << 16));
        else
          out[i] = __uint_as_float(v[i]);
      }
    }
  }
  // V elements at p as fp32
  __device__ __forceinline__ static void load(const T* p, float (&out)[V]) { open(raw(p), out); }
  __device__ __forceinline__ static void store(T* p, const float (&in)[V]) {
    if constexpr (V == 1) {
      p[0] = (T)in[0];
    } else {
      u32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2)
          v[i] = pack_bf16x2(in[2 * i], in[2 * i + 1]);
        else
          v[i] = __float_as_uint(in[i]);
      }
      *reinterpret_cast<u32x4_t*>(p) = v;
    }
  }
};

// The sum of v over a wave, in each lane, without LDS: pairs, quads, halves of
// 8 and 16 lanes by DPP, then rows and halves by swaps.
__device__ __forceinline__ float norm_wave_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, true));   // quad_perm 2 3 0 1
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, true));  // half row mirrored
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xf, 0xf, true));  // row mirrored
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// The sum of v over the TPR threads of a row, in each of them.  TPR = 64 is one
// wave; otherwise the workgroup's waves meet in one of the two halves of `scratch`
// (16 floats each), which takes turns: a half is written again only after the
// barrier of the sum between, which every reader of it has reached.
template <int TPR>
__device__ __forceinline__ float norm_row_sum(float v, float* scratch, uint32_t& turn) {
  v = norm_wave_sum(v);
  if constexpr (TPR > 64) {
    float* at = scratch + turn * 16u;
    turn ^= 1u;
    if (lane_id() == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += at[i];
  }
  return v;
}

constexpr int norm_threads(int tpr) { return tpr > 256 ? tpr : 256; }

template <class T, int V, int K, int TPR>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_fwd_kernel(NormArgs a) {
  constexpr int kRows = norm_threads(TPR) / TPR;
  typedef NormVec<T, V> Vec;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (row >= a.T) return;  // (whole waves; with TPR > 64 the workgroup)
  const int32_t lane = threadIdx.x % TPR, nv = a.H / V;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_t;
  const T* r = reinterpret_cast<const T*>(a.residual) + row * a.r_t;
  const float inv_h = 1.0f / (float)a.H;
  float u[K][V], h[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
#pragma unroll
    for (int i = 0; i < V; ++i) u[k][i] = h[k][i] = 0.f;
    if (v < nv) {
      Vec::load(x + (int64_t)v * V, u[k]);
      Vec::load(r + (int64_t)v * V, h[k]);
    }
  }
  if (a.pw) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(u[k][i], u[k][i], ss);
    const float rstd = 1.0f / sqrtf(norm_row_sum<TPR>(ss, scratch, turn) * inv_h + a.eps);
    if (lane == 0) a.rstd[a.T + row] = rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      float w[V];
      if (v < nv) {
        Vec::load(reinterpret_cast<const T*>(a.pw) + (int64_t)v * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) u[k][i] *= rstd * (a.offset + w[i]);
      }
    }
  }
  float bs = a.block_scale;
  if (a.gate_mode == 2) bs *= (float)reinterpret_cast<const T*>(a.gate)[row * a.gate_t];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
    if (v < nv) {
      if (a.gate_mode == 1 || a.gate_mode == 3) {
        float g[V];
        Vec::load(reinterpret_cast<const T*>(a.gate) + (a.gate_mode == 3 ? row * a.gate_t : 0) +
                      (int64_t)v * V, g);
#pragma unroll
        for (int i = 0; i < V; ++i) u[k][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[k][i] = fmaf(bs, u[k][i], a.residual_scale * h[k][i]);
        ss = fmaf(h[k][i], h[k][i], ss);
      }
      Vec::store(reinterpret_cast<T*>(a.h_out) + row * a.H + (int64_t)v * V, h[k]);
    }
  }
  const float rstd = 1.0f / sqrtf(norm_row_sum<TPR>(ss, scratch, turn) * inv_h + a.eps);
  if (lane == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t v = lane + k * TPR;
    if (v < nv) {
      float w[V];
      Vec::load(reinterpret_cast<const T*>(a.w) + (int64_t)v * V, w);
#pragma unroll
      for (int i = 0; i < V; ++i) h[k][i] *= rstd * (a.offset + w[i]);
      Vec::store(reinterpret_cast<T*>(a.y) + row * a.H + (int64_t)v * V, h[k]);
    }
  }
}

// EXTRA: a norm after the block or a gate, for which x is read again.
template <class T, int V, int K, int TPR, bool EXTRA>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_bwd_kernel(NormArgs a) {
  constexpr int kRows = norm_threads(TPR) / TPR;
  typedef NormVec<T, V> Vec;
  __shared__ float scratch[32];
  uint32_t turn = 0;
  const int32_t lane = threadIdx.x % TPR, nv = a.H / V;
  const int32_t part = (int32_t)blockIdx.x * kRows + (int32_t)(threadIdx.x / TPR);
  const float inv_h = 1.0f / (float)a.H;
  float dw[K][V], dpw[EXTRA ? K : 1][V], dg[EXTRA ? K : 1][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[k][i] = 0.f;
      if constexpr (EXTRA) dpw[k][i] = dg[k][i] = 0.f;
    }
  // the weights stay in registers over the rows (single elements are read again)
  constexpr bool kHold = V > 1;
  typename Vec::Raw w_raw[kHold ? K : 1], pw_raw[kHold && EXTRA ? K : 1], g_raw[kHold && EXTRA ? K : 1];
  if constexpr (kHold) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      w_raw[k] = Vec::raw(reinterpret_cast<const T*>(a.w) + (int64_t)v * V);
      if constexpr (EXTRA) {
        if (a.pw) pw_raw[k] = Vec::raw(reinterpret_cast<const T*>(a.pw) + (int64_t)v * V);
        if (a.gate_mode == 1) g_raw[k] = Vec::raw(reinterpret_cast<const T*>(a.gate) + (int64_t)v * V);
      }
    }
  }
  // The next row's tensors are on their way while this one is worked on (vectors
  // only: as single elements they would take too many registers).
  typename Vec::Raw r_h[kHold ? K : 1], r_dy[kHold ? K : 1], r_dh[kHold ? K : 1], r_x[kHold && EXTRA ? K : 1];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < (kHold ? K : 0); ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
      r_h[k] = Vec::raw(reinterpret_cast<const T*>(a.h) + row * a.h_t + (int64_t)v * V);
      r_dy[k] = Vec::raw(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + (int64_t)v * V);
      if (a.dh) r_dh[k] = Vec::raw(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + (int64_t)v * V);
      if constexpr (EXTRA)
        r_x[k] = Vec::raw(reinterpret_cast<const T*>(a.x) + row * a.x_t + (int64_t)v * V);
    }
  };
  if (part < a.T) fetch(part);
  for (int64_t row = part; row < a.T; row += a.parts) {
    const float rstd = a.rstd[row];
    float hn[K][V], g[K][V], d[K][V], u[EXTRA ? K : 1][V];
    float s1 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
#pragma unroll
      for (int i = 0; i < V; ++i) hn[k][i] = g[k][i] = d[k][i] = 0.f;
      if (v < nv) {
        float w[V];
        if constexpr (kHold) {
          Vec::open(w_raw[k], w);
          Vec::open(r_h[k], hn[k]);
          Vec::open(r_dy[k], g[k]);
          if (a.dh) Vec::open(r_dh[k], d[k]);
          if constexpr (EXTRA) Vec::open(r_x[k], u[k]);
        } else {
          Vec::load(reinterpret_cast<const T*>(a.w) + v, w);
          Vec::load(reinterpret_cast<const T*>(a.h) + row * a.h_t + v, hn[k]);
          Vec::load(reinterpret_cast<const T*>(a.dy) + row * a.dy_t + v, g[k]);
          if (a.dh) Vec::load(reinterpret_cast<const T*>(a.dh) + row * a.dh_t + v, d[k]);
          if constexpr (EXTRA) Vec::load(reinterpret_cast<const T*>(a.x) + row * a.x_t + v, u[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          hn[k][i] *= rstd;
          dw[k][i] = fmaf(g[k][i], hn[k][i], dw[k][i]);
          g[k][i] *= a.offset + w[i];
          s1 = fmaf(g[k][i], hn[k][i], s1);
        }
      }
    }
    if (kHold && row + a.parts < a.T) fetch(row + a.parts);
    s1 = norm_row_sum<TPR>(s1, scratch, turn) * inv_h;
    float s2 = 0.f, s3 = 0.f, bs = a.block_scale, rstd_x = 0.f;
    if constexpr (EXTRA) {
      if (a.gate_mode == 2) bs *= (float)reinterpret_cast<const T*>(a.gate)[row * a.gate_t];
      if (a.pw) rstd_x = a.rstd[a.T + row];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        g[k][i] = fmaf(rstd, fmaf(-hn[k][i], s1, g[k][i]), d[k][i]);  // gh
        d[k][i] = a.residual_scale * g[k][i];
      }
      if (a.dresidual) Vec::store(reinterpret_cast<T*>(a.dresidual) + row * a.H + (int64_t)v * V, d[k]);
      if constexpr (EXTRA) {
        float gate[V], pw[V];
#pragma unroll
        for (int i = 0; i < V; ++i) gate[i] = pw[i] = 1.f;
        if (a.gate_mode == 3)
          Vec::load(reinterpret_cast<const T*>(a.gate) + row * a.gate_t + (int64_t)v * V, gate);
        if (a.gate_mode == 1) {
          if constexpr (kHold)
            Vec::open(g_raw[k], gate);
          else
            Vec::load(reinterpret_cast<const T*>(a.gate) + v, gate);
        }
        if (a.pw) {
          if constexpr (kHold)
            Vec::open(pw_raw[k], pw);
          else
            Vec::load(reinterpret_cast<const T*>(a.pw) + v, pw);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            u[k][i] *= rstd_x;  // xn
            pw[i] += a.offset;
          }
        }
        float dgate[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dgate[i] = a.block_scale * g[k][i] * (u[k][i] * pw[i]);
          if (a.gate_mode == 1) dg[k][i] += dgate[i];
          s3 += dgate[i];
          g[k][i] *= bs * gate[i];  // du
          dpw[k][i] = fmaf(g[k][i], u[k][i], dpw[k][i]);
          g[k][i] *= pw[i];
          s2 = fmaf(g[k][i], u[k][i], s2);
        }
        if (a.gate_mode == 3 && a.dgate)
          Vec::store(reinterpret_cast<T*>(a.dgate) + row * a.H + (int64_t)v * V, dgate);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) g[k][i] *= bs;
      }
    }
    if constexpr (EXTRA) {
      if (a.pw) s2 = norm_row_sum<TPR>(s2, scratch, turn) * inv_h;
      if (a.gate_mode == 2) {
        s3 = norm_row_sum<TPR>(s3, scratch, turn);
        if (lane == 0 && a.dgate) reinterpret_cast<T*>(a.dgate)[row] = (T)s3;
      }
    }
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int32_t v = lane + k * TPR;
        if (v >= nv) continue;
        if constexpr (EXTRA) {
          if (a.pw) {
#pragma unroll
            for (int i = 0; i < V; ++i) g[k][i] = rstd_x * fmaf(-u[k][i], s2, g[k][i]);
          }
        }
        Vec::store(reinterpret_cast<T*>(a.dx) + row * a.H + (int64_t)v * V, g[k]);
      }
    }
  }
  if (part < a.parts) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t v = lane + k * TPR;
      if (v >= nv) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t c = (int64_t)part * a.H + (int64_t)v * V + i, n = (int64_t)a.parts * a.H;
        a.part[c] = dw[k][i];
        if constexpr (EXTRA) {
          if (a.pw) a.part[n + c] = dpw[k][i];
          if (a.gate_mode == 1) a.part[2 * n + c] = dg[k][i];
        }
      }
    }
  }
}

// Column sums of part[which][parts][H] in order: 64 columns per workgroup, 16
// groups of rows.  out[which] null: not wanted.
template <class T>
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* part, int32_t parts,
                                                            int32_t H, T* dw, T* dpw, T* dgate) {
  __shared__ float sums[16][64];
  const int32_t c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  T* out = blockIdx.y == 0 ? dw : blockIdx.y == 1 ? dpw : dgate;
  if (!out) return;
  const float* p = part + (int64_t)blockIdx.y * parts * H;
  float s = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int32_t r = g; r < parts; r += 16) s += p[(int64_t)r * H + c];
  }
  sums[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g == 0 && c < H) {
    for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
    out[c] = (T)s;
  }
}

}  // namespace mtf

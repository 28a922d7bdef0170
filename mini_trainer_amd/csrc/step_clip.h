// The global norm of many gradients and their scaling in place (gfx950).
//
//   norm = sqrt(sum over all elements of g^2)   (or the largest |g|)
//   coef = min(1, max_norm / (norm + 1e-6)),  g *= coef
//
// Bound by memory: one read for the norm, and one read and write only where
// the gradients have to be scaled.  Gradients come in as a table in the kernel
// arguments (up to kClipTensors per launch: nothing is copied to the device, and
// a captured launch keeps its table); chunks of one size are dealt to workgroups
// over all of a launch's tensors.  Each workgroup writes the sum of its chunks to a
// place of its own and one workgroup adds these in order, so that results repeat.
// 1.5e9 elements in bf16 and 2.3e8 in fp32, 4.0 GB: norm 730 us (5.5 TB/s), scaling
// 1430 us (5.6 TB/s; a large copy reaches 5.2).
// Squares are formed and added in 64 bits: exact for every input (a square
// leaves fp32's range from 2^64 on), and the fp64 rate still covers the memory's.
#pragma once

#include "flce_device.h"

namespace mtf {

constexpr int kClipTensors = 80;

struct ClipTable {
  char* ptr[kClipTensors];
  int64_t numel[kClipTensors];
  int64_t cols[kClipTensors];       // elements per row; 0: all elements lie in one run
  int64_t pitch[kClipTensors];      // elements from row to row
  uint32_t first[kClipTensors + 1]; // first chunk of each tensor, within the launch
  uint8_t bf16[kClipTensors];
  int32_t n;
  int32_t chunk;                    // elements, a multiple of 2048
};

__device__ __forceinline__ int32_t clip_find(const ClipTable& t, uint32_t chunk) {
  int32_t a = 0, b = t.n - 1;
  while (a < b) {
    const int32_t m = (a + b + 1) / 2;
    if (t.first[m] <= chunk) a = m; else b = m - 1;
  }
  return a;
}

// f(pointer, lanes) over the elements [e0, e1) of tensor i: whole 16-byte
// vectors where the run allows it (f.vec), single elements otherwise (f.one).
template <class T, class F>
__device__ __forceinline__ void clip_walk(const ClipTable& t, int32_t i, int64_t e0, int64_t e1, F& f) {
  constexpr int V = 16 / (int)sizeof(T);
  T* p = reinterpret_cast<T*>(t.ptr[i]);
  const int32_t tid = threadIdx.x;
  if (t.cols[i] == 0) {
    const int64_t skew = (int64_t)((reinterpret_cast<uintptr_t>(p + e0) & 15u) / sizeof(T));
    const int64_t v0 = min(e1, e0 + (skew ? V - skew : 0)), nv = (e1 - v0) / V;
    if (tid < v0 - e0) f.one(p + e0 + tid);
    for (int64_t v = tid; v < nv; v += 256 * 4) {
      u32x4_t x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v + 256 * u < nv) x[u] = *reinterpret_cast<const u32x4_t*>(p + v0 + (v + 256 * u) * V);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v + 256 * u < nv) f.vec(p + v0 + (v + 256 * u) * V, x[u]);
    }
    const int64_t tail = v0 + nv * V;
    if (tid < e1 - tail) f.one(p + tail + tid);
  } else {
    for (int64_t e = e0 + tid; e < e1; e += 256) f.one(p + (e / t.cols[i]) * t.pitch[i] + e % t.cols[i]);
  }
}

template <class T>
__device__ __forceinline__ float clip_el(const u32x4_t& x, int i) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float((i & 1) ? (x[i / 2] & 0xffff0000u) : (x[i / 2] << 16));
  return __uint_as_float(x[i]);
}

template <class T, bool INF>
struct ClipSum {
  double s[2] = {0.0, 0.0};
  float m = 0.f;
  __device__ __forceinline__ void add(float v, int k) {
    if constexpr (INF) {
      const float av = fabsf(v);
      m = (av > m || av != av) ? av : m;  // (a NaN stays: no later value is greater)
    } else {
      s[k] = fma((double)v, (double)v, s[k]);
    }
  }
  __device__ __forceinline__ void one(T* p) { add((float)*p, 0); }
  __device__ __forceinline__ void vec(T*, const u32x4_t& x) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) add(clip_el<T>(x, i), i & 1);
  }
};

// One combined value of two partial ones: the sum, or the larger with NaN kept.
template <bool INF>
__device__ __forceinline__ double clip_join(double a, double b) {
  if constexpr (INF) return (a != a) ? a : ((b > a || b != b) ? b : a);
  return a + b;
}

template <bool INF>
__device__ __forceinline__ double clip_block(double v, double* scratch, int waves) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = clip_join<INF>(v, __shfl_xor(v, d));
  if (lane_id() == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < waves; ++i) v = clip_join<INF>(v, scratch[i]);
  return v;
}

template <bool INF>
__global__ __launch_bounds__(256) void clip_norm_kernel(ClipTable t, double* parts) {
  __shared__ double scratch[4];
  double v = 0.0;
  for (uint32_t c = blockIdx.x; c < t.first[t.n]; c += gridDim.x) {
    const int32_t i = clip_find(t, c);
    const int64_t e0 = (int64_t)(c - t.first[i]) * t.chunk, e1 = min(t.numel[i], e0 + t.chunk);
    if (t.bf16[i]) {
      ClipSum<__bf16, INF> f;
      clip_walk<__bf16>(t, i, e0, e1, f);
      v = clip_join<INF>(v, INF ? (double)f.m : f.s[0] + f.s[1]);
    } else {
      ClipSum<float, INF> f;
      clip_walk<float>(t, i, e0, e1, f);
      v = clip_join<INF>(v, INF ? (double)f.m : f.s[0] + f.s[1]);
    }
  }
  v = clip_block<INF>(v, scratch, 4);
  if (threadIdx.x == 0) parts[blockIdx.x] = v;
}

// out[0] = norm, out[1] = coef (NaN and infinite norms as torch has them: a
// NaN scales everything to NaN, an infinity to 0 or NaN).
template <bool INF>
__global__ __launch_bounds__(1024) void clip_join_kernel(const double* parts, int64_t n,
                                                         double max_norm, float* out) {
  __shared__ double scratch[16];
  double v = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) v = clip_join<INF>(v, parts[i]);
  v = clip_block<INF>(v, scratch, 16);
  if (threadIdx.x == 0) {
    const double norm = INF ? v : sqrt(v);
    const double c = max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = (float)(c > 1.0 ? 1.0 : c);
  }
}

template <class T>
struct ClipScale {
  float c;
  __device__ __forceinline__ void one(T* p) { *p = (T)((float)*p * c); }
  __device__ __forceinline__ void vec(T* p, const u32x4_t& x) {
    u32x4_t y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2)
        y[i] = pack_bf16x2(clip_el<T>(x, 2 * i) * c, clip_el<T>(x, 2 * i + 1) * c);
      else
        y[i] = __float_as_uint(clip_el<T>(x, i) * c);
    }
    *reinterpret_cast<u32x4_t*>(p) = y;
  }
};

__global__ __launch_bounds__(256) void clip_scale_kernel(ClipTable t, const float* out) {
  const float c = out[1];
  if (c == 1.0f) return;  // nothing to scale: every product would be its factor
  const int32_t i = clip_find(t, blockIdx.x);
  // from the tensor's last chunk on: what the norm read last may still lie in a cache
  const int64_t e0 = (int64_t)(t.first[i + 1] - 1 - blockIdx.x) * t.chunk;
  const int64_t e1 = min(t.numel[i], e0 + t.chunk);
  if (t.bf16[i]) {
    ClipScale<__bf16> f{c};
    clip_walk<__bf16>(t, i, e0, e1, f);
  } else {
    ClipScale<float> f{c};
    clip_walk<float>(t, i, e0, e1, f);
  }
}

}  // namespace mtf

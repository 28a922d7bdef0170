// C ABI of libmt_flce.so, the operators of a packed training step around the
// loss: residual and norms, gradient norm and clipping.
// Declarations and contracts: include/mt_flce.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "../../include/mt_flce.h"
#include "capi_common.h"
#include "step_clip.h"
#include "step_norm.h"

using namespace mtf;

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// --- residual and norms --------------------------------------------------------

// Calls f with the kernels' template arguments for a row of H elements: the
// fewest threads and registers that hold it (vec: rows of whole aligned 16-byte
// vectors).
template <class T, class F>
int norm_pick(int64_t H, bool vec, F f) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) {
    if (H <= 64 * 2 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 2>(),
                                  std::integral_constant<int, 64>());
    if (H <= 256 * 1 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 1>(),
                                   std::integral_constant<int, 256>());
    if (H <= 256 * 2 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 2>(),
                                   std::integral_constant<int, 256>());
    if (H <= 256 * 4 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 4>(),
                                   std::integral_constant<int, 256>());
    if (H <= 1024 * 4 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 4>(),
                                    std::integral_constant<int, 1024>());
  }
  if (H <= 256 * 8) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(),
                             std::integral_constant<int, 256>());
  if (H <= 1024 * 8) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(),
                              std::integral_constant<int, 1024>());
  return f(std::integral_constant<int, 1>(), std::integral_constant<int, 32>(),
           std::integral_constant<int, 1024>());
}

constexpr int64_t kNormMaxH = 1024 * 32;
// Workgroups of the backward, each walking its rows and summing their weight
// gradients: two per CU.  Its 198 to 232 registers (norm before the block and
// gate) let no more reside: 147 us for 16384 x 3584, with 768 182, with 1024 157;
// the plain form, 65536 x 4096: 382, 387, 453 us.
constexpr int64_t kNormGroups = 512;

// Rows at a time of the backward, and so partial rows of the weight gradients, at
// most: kNormGroups workgroups, of four rows up to the width that a wave holds
// (norm_pick, bf16) and of one above it.
int64_t norm_parts(int64_t T, int64_t H) {
  return H <= 64 * 2 * 8 ? std::max<int64_t>(4, std::min<int64_t>(cdiv(T, 4), kNormGroups) * 4)
                         : std::min<int64_t>(T, kNormGroups);
}

int norm_check(const mt_norm_args* p, bool backward) {
  if (!p) return fail(MT_ERR_INVALID_ARGUMENT, "null arguments");
  const mt_norm_args& a = *p;
  const int es = esize(a.dtype);
  if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16", a.dtype);
  if (a.T < 0 || a.T > kMaxRows) return fail(MT_ERR_INVALID_ARGUMENT, "T=%lld out of range", (long long)a.T);
  if (a.H <= 0) return fail(MT_ERR_INVALID_ARGUMENT, "H=%lld out of range", (long long)a.H);
  if (a.H > kNormMaxH)
    return fail(MT_ERR_UNSUPPORTED, "H=%lld is above %lld", (long long)a.H, (long long)kNormMaxH);
  if (a.gate_mode < 0 || a.gate_mode > 3 || (a.gate_mode != 0) != (a.gate != nullptr))
    return fail(MT_ERR_INVALID_ARGUMENT, "gate_mode=%d does not fit the gate pointer", a.gate_mode);
  if (!(a.eps >= 0.f) || !std::isfinite(a.eps) || !std::isfinite(a.block_scale) ||
      !std::isfinite(a.residual_scale) || !std::isfinite(a.weight_offset))
    return fail(MT_ERR_INVALID_ARGUMENT, "eps must be >= 0 and the scales finite");
  if (a.x_t < a.H || a.residual_t < a.H || (a.gate_mode == 3 && a.gate_t < a.H) ||
      (a.gate_mode == 2 && a.gate_t < 1) ||
      (backward && ((a.dnormed && a.dnormed_t < a.H) || (a.dresidual_out && a.dresidual_out_t < a.H))))
    return fail(MT_ERR_INVALID_ARGUMENT, "row pitches must be >= H");
  if (a.T == 0) return MT_OK;
  if (!a.weight || !a.rstd || !a.new_residual || (!backward && (!a.x || !a.residual || !a.normed)) ||
      (backward && (!a.dnormed || ((a.post_weight || a.gate) && !a.x))))
    return fail(MT_ERR_INVALID_ARGUMENT, "null tensor pointer");
  const void* all[] = {a.x, a.residual, a.weight, a.post_weight, a.gate, a.normed, a.new_residual,
                       a.dnormed, a.dresidual_out, a.dx, a.dresidual, a.dgate};
  for (const void* x : all)
    if (reinterpret_cast<uintptr_t>(x) % es != 0)
      return fail(MT_ERR_INVALID_ARGUMENT, "tensors must be aligned to their element size");
  return MT_OK;
}

// Whether every row of every tensor is whole aligned 16-byte vectors.
bool norm_vectors(const mt_norm_args& a) {
  const int64_t V = 16 / esize(a.dtype);
  const void* all[] = {a.x, a.residual, a.weight, a.post_weight, a.gate_mode == 2 ? nullptr : a.gate,
                       a.normed, a.new_residual, a.dnormed, a.dresidual_out, a.dx, a.dresidual,
                       a.gate_mode == 2 ? nullptr : a.dgate};
  for (const void* x : all)
    if (!aligned16(x)) return false;
  return a.H % V == 0 && a.x_t % V == 0 && a.residual_t % V == 0 &&
         (a.gate_mode != 3 || a.gate_t % V == 0) && a.dnormed_t % V == 0 && a.dresidual_out_t % V == 0;
}

NormArgs norm_args(const mt_norm_args& a) {
  NormArgs k{};
  k.x = static_cast<const char*>(a.x);
  k.residual = static_cast<const char*>(a.residual);
  k.w = static_cast<const char*>(a.weight);
  k.pw = static_cast<const char*>(a.post_weight);
  k.gate = static_cast<const char*>(a.gate);
  k.dy = static_cast<const char*>(a.dnormed);
  k.dh = static_cast<const char*>(a.dresidual_out);
  k.h = static_cast<const char*>(a.new_residual);
  k.y = static_cast<char*>(a.normed);
  k.h_out = static_cast<char*>(a.new_residual);
  k.dx = static_cast<char*>(a.dx);
  k.dresidual = static_cast<char*>(a.dresidual);
  k.dgate = static_cast<char*>(a.dgate);
  k.rstd = a.rstd;
  k.x_t = a.x_t, k.r_t = a.residual_t, k.gate_t = a.gate_t;
  k.dy_t = a.dnormed_t, k.dh_t = a.dresidual_out_t, k.h_t = a.H;
  k.T = a.T;
  k.H = (int32_t)a.H;
  k.gate_mode = a.gate_mode;
  k.eps = a.eps;
  k.block_scale = a.block_scale;
  k.residual_scale = a.residual_scale;
  k.offset = a.weight_offset;
  return k;
}

template <class T>
int launch_norm_fwd(const NormArgs& k, bool vec, hipStream_t stream) {
  return norm_pick<T>(k.H, vec, [&](auto V, auto K, auto TPR) {
    constexpr int threads = norm_threads(decltype(TPR)::value);
    constexpr int rows = threads / decltype(TPR)::value;
    if (cdiv(k.T, rows) * threads >= (int64_t)1 << 32)  // threads of a launch
      return fail(MT_ERR_UNSUPPORTED, "%lld rows of %d exceed one launch", (long long)k.T, k.H);
    hipLaunchKernelGGL((norm_fwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value>),
                       dim3((uint32_t)cdiv(k.T, rows)), dim3(threads), 0, stream, k);
    return check_launch("norm_fwd_kernel");
  });
}

template <class T>
int launch_norm_bwd(NormArgs k, const mt_norm_args& a, bool vec, hipStream_t stream) {
  const int rc = norm_pick<T>(k.H, vec, [&](auto V, auto K, auto TPR) {
    constexpr int threads = norm_threads(decltype(TPR)::value);
    constexpr int rows = threads / decltype(TPR)::value;
    const int64_t groups = std::min<int64_t>(cdiv(k.T, rows), kNormGroups);
    k.parts = (int32_t)(groups * rows);
    if (k.parts > norm_parts(k.T, k.H))  // (the workspace's partial rows)
      return fail(MT_ERR_UNSUPPORTED, "%d partial rows", (int)k.parts);
    auto kern = (k.pw || k.gate)
                    ? norm_bwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, true>
                    : norm_bwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, false>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)groups), dim3(threads), 0, stream, k);
    return check_launch("norm_bwd_kernel");
  });
  if (rc != MT_OK) return rc;
  T* dgate = k.gate_mode == 1 ? static_cast<T*>(a.dgate) : nullptr;
  T* dpw = k.pw ? static_cast<T*>(a.dpost_weight) : nullptr;
  if (!a.dweight && !dpw && !dgate) return MT_OK;
  hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((uint32_t)cdiv(k.H, 64), dgate ? 3 : dpw ? 2 : 1),
                     dim3(1024), 0, stream, k.part, k.parts, k.H, static_cast<T*>(a.dweight), dpw, dgate);
  return check_launch("norm_columns_kernel");
}

// --- gradient norm and clipping --------------------------------------------------

int64_t clip_chunks(const int64_t* numel, int64_t n, int64_t chunk) {
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) chunks += cdiv(numel[i], chunk);
  return chunks;
}
// Elements of a chunk: 8192, a step of the four 16-byte loads that each of a
// workgroup's threads keeps in flight (bf16), or as many more as keep a launch's
// chunks below 2^24.  Scaling 4.0 GB: 1430 us; chunks of 32768 1510, of 131072,
// which end unevenly, 1575.
int64_t clip_chunk(const int64_t* numel, int64_t n) {
  int64_t chunk = 8192;
  while (clip_chunks(numel, n, chunk) > (1 << 23) + n) chunk *= 2;
  return chunk;
}

constexpr int64_t kClipMost = (int64_t)1 << 40;  // elements of one tensor

int clip_check(void* const* ptrs, const int64_t* numel, const int64_t* cols, const int64_t* pitch,
               const int32_t* dtypes, int64_t n) {
  if (n < 0 || n > (1 << 24)) return fail(MT_ERR_INVALID_ARGUMENT, "n=%lld out of range", (long long)n);
  if (n > 0 && (!ptrs || !numel || !cols || !pitch || !dtypes))
    return fail(MT_ERR_INVALID_ARGUMENT, "null table");
  for (int64_t i = 0; i < n; ++i) {
    const int es = esize(dtypes[i]);
    if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "tensor %lld: dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16",
                         (long long)i, dtypes[i]);
    if (numel[i] < 0 || numel[i] > kClipMost || (numel[i] > 0 && !ptrs[i]) ||
        reinterpret_cast<uintptr_t>(ptrs[i]) % es != 0)
      return fail(MT_ERR_INVALID_ARGUMENT, "tensor %lld: bad size or pointer", (long long)i);
    if (cols[i] < 0 || (cols[i] > 0 && (pitch[i] < cols[i] || numel[i] % cols[i] != 0)))
      return fail(MT_ERR_INVALID_ARGUMENT, "tensor %lld: rows of %lld elements, %lld apart", (long long)i,
                  (long long)cols[i], (long long)pitch[i]);
  }
  return MT_OK;
}

// Workgroups of a launch of clip_norm_kernel, each with one sum.  4.0 GB, norm and
// the sums' addition: 742 us; 4096 of them 735, one for each chunk 730, whose sums
// are 4 MB.
constexpr int64_t kClipGroups = 2048;

// Calls launch(table, chunks) for the tensors in
// groups of up to kClipTensors, from the last tensor on with `reverse`.
template <class F>
int clip_groups(void* const* ptrs, const int64_t* numel, const int64_t* cols, const int64_t* pitch,
                const int32_t* dtypes, int64_t n, bool reverse, F launch) {
  const int64_t chunk = clip_chunk(numel, n);
  for (int64_t done = 0; done < n;) {
    ClipTable t;
    t.n = 0;
    t.chunk = (int32_t)std::min<int64_t>(chunk, 1 << 30);
    uint32_t chunks = 0;
    for (; done < n && t.n < kClipTensors; ++done) {
      const int64_t at = reverse ? n - 1 - done : done;
      if (numel[at] > 0) {
        t.ptr[t.n] = static_cast<char*>(ptrs[at]);
        t.numel[t.n] = numel[at];
        t.cols[t.n] = cols[at] == numel[at] ? 0 : cols[at];
        t.pitch[t.n] = pitch[at];
        t.bf16[t.n] = dtypes[at] == MT_DTYPE_BF16;
        t.first[t.n] = chunks;
        chunks += (uint32_t)cdiv(numel[at], t.chunk);
        ++t.n;
      }
    }
    t.first[t.n] = chunks;
    if (chunks) MT_TRY(launch(t, chunks));
  }
  return MT_OK;
}

}  // namespace

extern "C" {

int mt_norm_forward(const mt_norm_args* args, mt_stream_t stream) {
  MT_TRY(norm_check(args, false));
  const mt_norm_args& a = *args;
  if (a.T == 0) return MT_OK;
  const NormArgs k = norm_args(a);
  return a.dtype == MT_DTYPE_BF16 ? launch_norm_fwd<__bf16>(k, norm_vectors(a), (hipStream_t)stream)
                                  : launch_norm_fwd<float>(k, norm_vectors(a), (hipStream_t)stream);
}

size_t mt_norm_backward_workspace_bytes(int64_t T, int64_t H) {
  return T <= 0 || T > kMaxRows || H <= 0 || H > kNormMaxH ? 0 : (size_t)3 * norm_parts(T, H) * (size_t)H * 4;
}

int mt_norm_backward(const mt_norm_args* args, void* workspace, size_t workspace_bytes,
                     mt_stream_t stream) {
  MT_TRY(norm_check(args, true));
  const mt_norm_args& a = *args;
  if (a.T == 0) return MT_OK;
  const size_t need = mt_norm_backward_workspace_bytes(a.T, a.H);
  if (!workspace || !aligned16(workspace))
    return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned workspace");
  if (workspace_bytes < need)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, need);
  NormArgs k = norm_args(a);
  k.part = static_cast<float*>(workspace);
  return a.dtype == MT_DTYPE_BF16 ? launch_norm_bwd<__bf16>(k, a, norm_vectors(a), (hipStream_t)stream)
                                  : launch_norm_bwd<float>(k, a, norm_vectors(a), (hipStream_t)stream);
}

size_t mt_grad_norm_workspace_bytes(const int64_t* numel, int64_t n) {
  if (!numel || n <= 0) return 8;
  if (n > (1 << 24)) return 0;  // (clip_check refuses these)
  for (int64_t i = 0; i < n; ++i)
    if (numel[i] < 0 || numel[i] > kClipMost) return 0;
  const int64_t chunks = clip_chunks(numel, n, clip_chunk(numel, n));
  return 8 * (size_t)std::max<int64_t>(1, std::min(chunks, cdiv(n, kClipTensors) * kClipGroups));
}

int mt_grad_norm(void* const* ptrs, const int64_t* numel, const int64_t* cols, const int64_t* pitch,
                 const int32_t* dtypes, int64_t n, int inf_norm, double max_norm, void* workspace,
                 size_t workspace_bytes, float* out, mt_stream_t stream) {
  MT_TRY(clip_check(ptrs, numel, cols, pitch, dtypes, n));
  if (!(max_norm >= 0.0)) return fail(MT_ERR_INVALID_ARGUMENT, "max_norm must be >= 0");
  if (!workspace || !out || !aligned16(workspace))
    return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned workspace or result");
  const size_t need = mt_grad_norm_workspace_bytes(numel, n);
  if (workspace_bytes < need)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, need);
  hipStream_t s = (hipStream_t)stream;
  double* parts = static_cast<double*>(workspace);
  int64_t total = 0;
  MT_TRY(clip_groups(ptrs, numel, cols, pitch, dtypes, n, false, [&](const ClipTable& t, uint32_t chunks) {
    const uint32_t groups = (uint32_t)std::min<int64_t>(chunks, kClipGroups);
    if (inf_norm)
      hipLaunchKernelGGL(clip_norm_kernel<true>, dim3(groups), dim3(256), 0, s, t, parts + total);
    else
      hipLaunchKernelGGL(clip_norm_kernel<false>, dim3(groups), dim3(256), 0, s, t, parts + total);
    total += groups;
    return check_launch("clip_norm_kernel");
  }));
  if (inf_norm)
    hipLaunchKernelGGL(clip_join_kernel<true>, dim3(1), dim3(1024), 0, s, parts, total, max_norm, out);
  else
    hipLaunchKernelGGL(clip_join_kernel<false>, dim3(1), dim3(1024), 0, s, parts, total, max_norm, out);
  return check_launch("clip_join_kernel");
}

int mt_grad_scale(void* const* ptrs, const int64_t* numel, const int64_t* cols, const int64_t* pitch,
                  const int32_t* dtypes, int64_t n, const float* norm_and_coef, mt_stream_t stream) {
  MT_TRY(clip_check(ptrs, numel, cols, pitch, dtypes, n));
  if (!norm_and_coef) return fail(MT_ERR_INVALID_ARGUMENT, "null pointer argument");
  return clip_groups(ptrs, numel, cols, pitch, dtypes, n, true,
                     [&](const ClipTable& t, uint32_t chunks) {
                       hipLaunchKernelGGL(clip_scale_kernel, dim3(chunks), dim3(256), 0,
                                          (hipStream_t)stream, t, norm_and_coef);
                       return check_launch("clip_scale_kernel");
                     });
}

}  // extern "C"

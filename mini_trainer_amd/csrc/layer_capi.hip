// C ABI of libmt_flce.so, the operators at the ends of a decoder's layers: token
// embedding and layer norm.  Declarations and contracts: include/mt_flce.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mt_flce.h"
#include "capi_common.h"
#include "layer_embed.h"
#include "layer_norm.h"
#include "norm_pick.h"

using namespace mtf;

namespace {

// --- token embedding -------------------------------------------------------------

constexpr int64_t kEmbedMostH = (int64_t)1 << 24;
constexpr int64_t kEmbedMostPitch = (int64_t)1 << 32;

// 256 buckets, a workgroup for each CU, or as many more as keep a bucket's ids in LDS.
int embed_log_buckets(int64_t V) {
  int log = 8;
  while (cdiv(V, (int64_t)1 << log) > kEmbedSlots) ++log;
  return log;
}

struct EmbedLayout {
  int log_buckets;
  int64_t per, part_t;
  size_t order, part, bytes;  // offsets of the parts behind starts, and the whole
};
EmbedLayout embed_layout(int64_t T, int64_t V, int64_t H) {
  EmbedLayout l{};
  if (T <= kEmbedDirect) return l;  // (nothing is sorted)
  l.log_buckets = embed_log_buckets(V);
  l.per = cdiv(V, (int64_t)1 << l.log_buckets);
  l.part_t = cdiv(H, 4) * 4;
  const auto up = [](size_t n) { return (n + 63) / 64 * 64; };
  l.order = up(4 * (((size_t)l.per << l.log_buckets) + 1));
  l.part = l.order + up(4 * (size_t)T);
  l.bytes = l.part + 2 * (size_t)cdiv(T, kEmbedPiece) * (size_t)l.part_t * 4;
  return l;
}

int embed_check(const mt_embed_args* p, bool backward) {
  if (!p) return fail(MT_ERR_INVALID_ARGUMENT, "null arguments");
  const mt_embed_args& a = *p;
  const int es = esize(a.dtype);
  if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16", a.dtype);
  if (a.ids_bytes != 4 && a.ids_bytes != 8)
    return fail(MT_ERR_INVALID_ARGUMENT, "ids of %d bytes: 4 and 8 are supported", a.ids_bytes);
  if (a.T < 0 || a.T > kMaxRows) return fail(MT_ERR_INVALID_ARGUMENT, "T=%lld out of range", (long long)a.T);
  if (a.V < 1 || a.V > kMaxRows) return fail(MT_ERR_INVALID_ARGUMENT, "V=%lld out of range", (long long)a.V);
  if (a.H < 1) return fail(MT_ERR_INVALID_ARGUMENT, "H=%lld out of range", (long long)a.H);
  if (a.H > kEmbedMostH)
    return fail(MT_ERR_UNSUPPORTED, "H=%lld is above %lld", (long long)a.H, (long long)kEmbedMostH);
  if (!std::isfinite(a.scale)) return fail(MT_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (a.padding_idx < -1 || a.padding_idx >= a.V)
    return fail(MT_ERR_INVALID_ARGUMENT, "padding_idx=%lld out of range", (long long)a.padding_idx);
  if ((!backward && a.weight_t < a.H) || (backward && ((a.T > 0 && a.dout_t < a.H) || a.dweight_t < a.H)))
    return fail(MT_ERR_INVALID_ARGUMENT, "row pitches must be >= H");
  if ((!backward && a.weight_t > kEmbedMostPitch) ||
      (backward && ((a.T > 0 && a.dout_t > kEmbedMostPitch) || a.dweight_t > kEmbedMostPitch)))
    return fail(MT_ERR_UNSUPPORTED, "rows more than 2^32 elements apart");
  if ((a.T > 0 && !a.ids) || (!backward && a.T > 0 && (!a.weight || !a.out)) ||
      (backward && ((a.T > 0 && !a.dout) || !a.dweight)))
    return fail(MT_ERR_INVALID_ARGUMENT, "null tensor pointer");
  const int des = a.accumulate ? 4 : es;
  if (reinterpret_cast<uintptr_t>(a.ids) % a.ids_bytes || reinterpret_cast<uintptr_t>(a.weight) % es ||
      reinterpret_cast<uintptr_t>(a.out) % es || reinterpret_cast<uintptr_t>(a.dout) % es ||
      reinterpret_cast<uintptr_t>(a.dweight) % des || reinterpret_cast<uintptr_t>(a.status) % 4)
    return fail(MT_ERR_INVALID_ARGUMENT, "tensors must be aligned to their element size");
  return MT_OK;
}

EmbedArgs embed_args(const mt_embed_args& a) {
  EmbedArgs k{};
  k.ids = a.ids;
  k.w = static_cast<const char*>(a.weight);
  k.dout = static_cast<const char*>(a.dout);
  k.out = static_cast<char*>(a.out);
  k.dw = static_cast<char*>(a.dweight);
  k.status = a.status;
  k.w_t = a.weight_t, k.dout_t = a.dout_t, k.dw_t = a.dweight_t;
  k.padding = a.padding_idx;
  k.T = (int32_t)a.T, k.V = (int32_t)a.V, k.H = (int32_t)a.H;
  k.wide = a.ids_bytes == 8;
  k.scale = a.scale;
  return k;
}

// Calls f(V, K, log2 of the lanes of a row, workgroups) with the variant for `rows`
// rows of H elements: 16-byte vectors (one element where a row is shorter), as many of them in
// flight per lane (up to kMost) as a row fills; rows of few vectors share a wave unless share
// is false.
template <class T, int kMost, class F>
int embed_pick(int64_t rows, int64_t H, F f, bool share = true) {
  constexpr int W = 16 / (int)sizeof(T);
  const int64_t nv = H < W ? H : cdiv(H, W);
  int log_lanes = 6;
  while (share && log_lanes > 0 && nv <= (int64_t)1 << (log_lanes - 1)) --log_lanes;
  const auto with = [&](auto V, auto K) {
    const int64_t chunks = log_lanes == 6 ? cdiv(nv, 64 * decltype(K)::value) : 1;
    const int64_t units = cdiv(rows, 64 >> log_lanes) * chunks;
    if (cdiv(units, 4) * 256 >= (int64_t)1 << 32)  // threads of a launch
      return fail(MT_ERR_UNSUPPORTED, "%lld rows of %lld exceed one launch", (long long)rows, (long long)H);
    return f(V, K, log_lanes, (uint32_t)cdiv(units, 4));
  };
  constexpr std::integral_constant<int, W> whole{};
  if (H < W) return with(std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
  if constexpr (kMost >= 4) {
    if (nv > 128) return with(whole, std::integral_constant<int, 4>());
  }
  if (nv > 64) return with(whole, std::integral_constant<int, 2>());
  return with(whole, std::integral_constant<int, 1>());
}

template <class T>
int launch_embed_forward(const EmbedArgs& k, hipStream_t stream) {
  return embed_pick<T, 4>(k.T, k.H, [&](auto V, auto K, int log_lanes, uint32_t groups) {
    hipLaunchKernelGGL((embed_forward_kernel<T, decltype(V)::value, decltype(K)::value>), dim3(groups), dim3(256), 0,
                       stream, k, log_lanes);
    return check_launch("embed_forward_kernel");
  });
}

template <class T>
int launch_embed_backward(const EmbedArgs& k, bool accumulate, hipStream_t stream) {
  const bool direct = k.T <= kEmbedDirect;
  if (!direct) {
    if (k.wide) hipLaunchKernelGGL(embed_sort_kernel<int64_t>, dim3(1u << k.log_buckets), dim3(1024), 0, stream, k);
    else hipLaunchKernelGGL(embed_sort_kernel<int32_t>, dim3(1u << k.log_buckets), dim3(1024), 0, stream, k);
    MT_TRY(check_launch("embed_sort_kernel"));
    MT_TRY((embed_pick<T, 2>(cdiv(k.T, kEmbedPiece), k.H, [&](auto V, auto K, int, uint32_t groups) {
      hipLaunchKernelGGL((embed_pieces_kernel<T, decltype(V)::value, decltype(K)::value>), dim3(groups), dim3(256), 0,
                         stream, k);
      return check_launch("embed_pieces_kernel");
    }, false)));
  }
  if (accumulate && k.T == 0) return MT_OK;
  return embed_pick<T, 2>(accumulate ? k.T : k.V, k.H, [&](auto V, auto K, int log_lanes, uint32_t groups) {
    constexpr int v = decltype(V)::value, n = decltype(K)::value;
    auto kern = direct ? (accumulate ? embed_direct_kernel<T, v, n, true> : embed_direct_kernel<T, v, n, false>)
                       : (accumulate ? embed_rows_kernel<T, v, n, true> : embed_rows_kernel<T, v, n, false>);
    hipLaunchKernelGGL(kern, dim3(groups), dim3(256), 0, stream, k, log_lanes);
    return check_launch(direct ? "embed_direct_kernel" : "embed_rows_kernel");
  });
}

// --- layer norm --------------------------------------------------------------------

int layer_norm_check(const mt_layer_norm_args* p, bool backward) {
  if (!p) return fail(MT_ERR_INVALID_ARGUMENT, "null arguments");
  const mt_layer_norm_args& a = *p;
  const int es = esize(a.dtype);
  if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16", a.dtype);
  if (a.T < 0 || a.T > kMaxRows) return fail(MT_ERR_INVALID_ARGUMENT, "T=%lld out of range", (long long)a.T);
  if (a.H <= 0) return fail(MT_ERR_INVALID_ARGUMENT, "H=%lld out of range", (long long)a.H);
  if (a.H > kNormMaxH)
    return fail(MT_ERR_UNSUPPORTED, "H=%lld is above %lld", (long long)a.H, (long long)kNormMaxH);
  if (!(a.eps >= 0.f) || !std::isfinite(a.eps) || !std::isfinite(a.block_scale) ||
      !std::isfinite(a.residual_scale))
    return fail(MT_ERR_INVALID_ARGUMENT, "eps must be >= 0 and the scales finite");
  const bool res = a.has_residual != 0;
  if ((!(backward && res) && a.x_t < a.H) || (!backward && res && a.residual_t < a.H) ||
      (backward && (a.dnormed_t < a.H || (a.dresidual_out && a.dresidual_out_t < a.H))))
    return fail(MT_ERR_INVALID_ARGUMENT, "row pitches must be >= H");
  if (a.T == 0) return MT_OK;
  if ((!backward && (!a.x || !a.normed || (res && (!a.residual || !a.new_residual)))) ||
      (backward && (!a.dnormed || !a.stat || (res ? !a.new_residual : !a.x) ||
                    (res && a.dtype == MT_DTYPE_BF16 && !a.residual_lo))))
    return fail(MT_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!res && (a.dresidual || a.dresidual_out))
    return fail(MT_ERR_INVALID_ARGUMENT, "gradients of a residual that there is not");
  const void* all[] = {a.x, a.residual, a.weight, a.bias, a.normed, a.new_residual,
                       a.dnormed, a.dresidual_out, a.dx, a.dresidual, a.dweight, a.dbias};
  for (const void* x : all)
    if (reinterpret_cast<uintptr_t>(x) % es != 0)
      return fail(MT_ERR_INVALID_ARGUMENT, "tensors must be aligned to their element size");
  if (reinterpret_cast<uintptr_t>(a.stat) % 4)
    return fail(MT_ERR_INVALID_ARGUMENT, "stat must be aligned to 4 bytes");
  return MT_OK;
}

LayerNormArgs layer_norm_args(const mt_layer_norm_args& a, bool backward) {
  const bool res = a.has_residual != 0;
  LayerNormArgs k{};
  k.x = static_cast<const char*>(a.x);
  k.residual = static_cast<const char*>(a.residual);
  k.w = static_cast<const char*>(a.weight);
  k.b = static_cast<const char*>(a.bias);
  k.dy = static_cast<const char*>(a.dnormed);
  k.dh = static_cast<const char*>(a.dresidual_out);
  k.h = res ? static_cast<const char*>(a.new_residual) : k.x;
  k.y = static_cast<char*>(a.normed);
  k.h_out = backward ? nullptr : static_cast<char*>(a.new_residual);
  k.dx = static_cast<char*>(a.dx);
  k.dresidual = static_cast<char*>(a.dresidual);
  k.lo = a.residual_lo;
  k.stat = a.stat;
  k.x_t = a.x_t, k.r_t = a.residual_t, k.dy_t = a.dnormed_t, k.dh_t = a.dresidual_out_t;
  k.h_t = res ? a.H : a.x_t;
  k.T = a.T;
  k.H = (int32_t)a.H;
  k.eps = a.eps;
  k.block_scale = a.block_scale;
  k.residual_scale = a.residual_scale;
  return k;
}

// Calls f with the kernels' template arguments for a row of H elements: the fewest threads and
// registers that hold it (norm_pick's, but for rows of any width and alignment).
template <class T, class F>
int layer_norm_pick(int64_t H, F f) {
  constexpr int W = 16 / (int)sizeof(T);
  constexpr std::integral_constant<int, W> V{};
  const auto with = [&](auto K, auto TPR) { return f(V, K, TPR); };
  constexpr std::integral_constant<int, 1> k1{};
  constexpr std::integral_constant<int, 2> k2{};
  constexpr std::integral_constant<int, 4> k4{};
  constexpr std::integral_constant<int, 64> wave{};
  constexpr std::integral_constant<int, 256> four{};
  constexpr std::integral_constant<int, 1024> all{};
  if (H < W) return f(k1, k1, wave);
  if (H <= 64 * 2 * W) return with(k2, wave);
  if (H <= 256 * 1 * W) return with(k1, four);
  if (H <= 256 * 2 * W) return with(k2, four);
  if (H <= 256 * 4 * W) return with(k4, four);
  if (H <= 1024 * 2 * W) return with(k2, all);
  if constexpr (W == 8) return with(k4, all);
  else return H <= 1024 * 4 * W ? with(k4, all) : with(std::integral_constant<int, 8>(), all);
}

template <class T>
int launch_layer_norm_fwd(const LayerNormArgs& k, bool res, hipStream_t stream) {
  return layer_norm_pick<T>(k.H, [&](auto V, auto K, auto TPR) {
    constexpr int threads = norm_threads(decltype(TPR)::value);
    constexpr int rows = threads / decltype(TPR)::value;
    if (cdiv(k.T, rows) * threads >= (int64_t)1 << 32)  // threads of a launch
      return fail(MT_ERR_UNSUPPORTED, "%lld rows of %d exceed one launch", (long long)k.T, k.H);
    auto kern = res ? layer_norm_fwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, true>
                    : layer_norm_fwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, false>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)cdiv(k.T, rows)), dim3(threads), 0, stream, k);
    return check_launch("layer_norm_fwd_kernel");
  });
}

template <class T>
int launch_layer_norm_bwd(LayerNormArgs k, const mt_layer_norm_args& a, bool res, hipStream_t stream) {
  MT_TRY(layer_norm_pick<T>(k.H, [&](auto V, auto K, auto TPR) {
    constexpr int threads = norm_threads(decltype(TPR)::value);
    constexpr int rows = threads / decltype(TPR)::value;
    const int64_t groups = std::min<int64_t>(cdiv(k.T, rows), kNormGroups);
    k.parts = (int32_t)(groups * rows);
    if (k.parts > norm_parts(k.T, k.H))  // (the workspace's partial rows)
      return fail(MT_ERR_UNSUPPORTED, "%d partial rows", (int)k.parts);
    auto kern = res ? layer_norm_bwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, true>
                    : layer_norm_bwd_kernel<T, decltype(V)::value, decltype(K)::value, decltype(TPR)::value, false>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)groups), dim3(threads), 0, stream, k);
    return check_launch("layer_norm_bwd_kernel");
  }));
  if (!a.dweight && !a.dbias) return MT_OK;
  hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((uint32_t)cdiv(k.H, 64), a.dbias ? 2 : 1), dim3(1024), 0,
                     stream, k.part, k.parts, k.H, static_cast<T*>(a.dweight), static_cast<T*>(a.dbias),
                     static_cast<T*>(nullptr));
  return check_launch("norm_columns_kernel");
}

}  // namespace

extern "C" {

int mt_embed_forward(const mt_embed_args* args, mt_stream_t stream) {
  MT_TRY(embed_check(args, false));
  const mt_embed_args& a = *args;
  if (a.T == 0) return MT_OK;
  const EmbedArgs k = embed_args(a);
  hipStream_t s = (hipStream_t)stream;
  return a.dtype == MT_DTYPE_BF16 ? launch_embed_forward<__bf16>(k, s) : launch_embed_forward<float>(k, s);
}

size_t mt_embed_backward_workspace_bytes(int64_t T, int64_t V, int64_t H) {
  return T < 0 || T > kMaxRows || V < 1 || V > kMaxRows || H < 1 || H > kEmbedMostH ? 0
                                                                                   : embed_layout(T, V, H).bytes;
}

int mt_embed_backward(const mt_embed_args* args, void* workspace, size_t workspace_bytes, mt_stream_t stream) {
  MT_TRY(embed_check(args, true));
  const mt_embed_args& a = *args;
  const EmbedLayout l = embed_layout(a.T, a.V, a.H);
  if (l.bytes && (!workspace || !aligned16(workspace)))
    return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned workspace");
  if (workspace_bytes < l.bytes)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, l.bytes);
  EmbedArgs k = embed_args(a);
  char* ws = static_cast<char*>(workspace);
  k.starts = reinterpret_cast<int32_t*>(ws);
  k.order = reinterpret_cast<int32_t*>(ws + l.order);
  k.part = reinterpret_cast<float*>(ws + l.part);
  k.part_t = l.part_t;
  k.log_buckets = l.log_buckets;
  k.per = (int32_t)l.per;
  hipStream_t s = (hipStream_t)stream;
  const bool acc = a.accumulate != 0;
  return a.dtype == MT_DTYPE_BF16 ? launch_embed_backward<__bf16>(k, acc, s)
                                  : launch_embed_backward<float>(k, acc, s);
}

int mt_layer_norm_forward(const mt_layer_norm_args* args, mt_stream_t stream) {
  MT_TRY(layer_norm_check(args, false));
  const mt_layer_norm_args& a = *args;
  if (a.T == 0) return MT_OK;
  const LayerNormArgs k = layer_norm_args(a, false);
  const bool res = a.has_residual != 0;
  return a.dtype == MT_DTYPE_BF16 ? launch_layer_norm_fwd<__bf16>(k, res, (hipStream_t)stream)
                                  : launch_layer_norm_fwd<float>(k, res, (hipStream_t)stream);
}

size_t mt_layer_norm_backward_workspace_bytes(int64_t T, int64_t H) {
  return T <= 0 || T > kMaxRows || H <= 0 || H > kNormMaxH ? 0 : (size_t)2 * norm_parts(T, H) * (size_t)H * 4;
}

int mt_layer_norm_backward(const mt_layer_norm_args* args, void* workspace, size_t workspace_bytes,
                           mt_stream_t stream) {
  MT_TRY(layer_norm_check(args, true));
  const mt_layer_norm_args& a = *args;
  if (a.T == 0) return MT_OK;
  const size_t need = mt_layer_norm_backward_workspace_bytes(a.T, a.H);
  if (!workspace || !aligned16(workspace))
    return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned workspace");
  if (workspace_bytes < need)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, need);
  LayerNormArgs k = layer_norm_args(a, true);
  k.part = static_cast<float*>(workspace);
  const bool res = a.has_residual != 0;
  return a.dtype == MT_DTYPE_BF16 ? launch_layer_norm_bwd<__bf16>(k, a, res, (hipStream_t)stream)
                                  : launch_layer_norm_bwd<float>(k, a, res, (hipStream_t)stream);
}

}  // extern "C"

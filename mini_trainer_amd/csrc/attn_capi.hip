// C ABI of libmt_flce.so, attention over a packed row.  Declarations and
// contracts: include/mt_flce.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mt_flce.h"
#include "capi_common.h"
#include "attn_kernels.h"

using namespace mtf;

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of a plan at most: every document and the tail end in a partial one.
inline int64_t attn_tiles(int64_t T, int64_t S) { return cdiv(T, kAttnRows) + S + 1; }

inline size_t plan_bytes(int64_t T, int64_t S) {
  return 4 * ((size_t)kPlanHeader + 2 * (size_t)kPlanTile * attn_tiles(T, S) + (size_t)S + 2);
}

// Workgroups at most that share the query heads of a key tile's group
// (attn_parts): one where no workgroup can have more than some ten blocks to visit,
// so that the parts need no launch of their own.
int32_t attn_parts_max(const mt_attn_args& a) {
  const int64_t G = a.heads / a.kv_heads;
  return cdiv(a.T, 64) * G <= 12 ? 1 : (int32_t)G;
}

inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Places for the parts of one key head.  Where attn_parts goes by the costliest
// tile, a tile of cost c gets fewer than 700 c / (total kv_heads) + 1 parts and more
// than one only if that quotient is above 1: below 1400 / kv_heads together.  Where
// it goes by the number of tiles, n tiles kv_heads < 2048 + tiles kv_heads, and it
// divides below 2048 tiles x kv_heads: below 4096 / kv_heads.  (A whole copy of dK
// and dV for each of four heads of a group takes 4.3 GB at 131072 tokens with 8
// heads of 128; this 0.2 GB, in the same time.)
int64_t attn_slots(const mt_attn_args& a) {
  const int64_t parts = attn_parts_max(a);
  if (parts == 1) return 0;
  const int64_t most = cdiv(a.T, kAttnRows) * a.kv_heads < 2048 ? 4096 : 1400;
  return std::min(parts * attn_tiles(a.T, a.S), cdiv(most, a.kv_heads) + parts);
}

// One fp32 number for each row and query head: delta, and the factor of its
// probabilities.
size_t attn_row_bytes(const mt_attn_args& a) { return round256((size_t)a.heads * (size_t)a.T * 4); }

size_t attn_part_bytes(const mt_attn_args& a) {
  return (size_t)attn_slots(a) * (size_t)a.kv_heads * 2 * kAttnRows * (size_t)a.head_dim * 4;
}

size_t attn_item_bytes(const mt_attn_args& a) {
  return round256(16 + 8 * (size_t)attn_tiles(a.T, a.S) * ((size_t)attn_parts_max(a) + 1));
}

constexpr int64_t kMaxHeads = 65536;

int attn_check(const mt_attn_args* p, bool backward) {
  if (!p) return fail(MT_ERR_INVALID_ARGUMENT, "null arguments");
  const mt_attn_args& a = *p;
  const int es = esize(a.dtype);
  if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16", a.dtype);
  if (a.T < 0 || a.T > kMaxRows || a.S < 0 || a.S > kMaxRows)
    return fail(MT_ERR_INVALID_ARGUMENT, "T=%lld or S=%lld out of range", (long long)a.T, (long long)a.S);
  if (a.heads <= 0 || a.kv_heads <= 0 || a.heads > kMaxHeads || a.heads % a.kv_heads != 0)
    return fail(MT_ERR_INVALID_ARGUMENT, "heads=%lld must be a positive multiple of kv_heads=%lld",
                (long long)a.heads, (long long)a.kv_heads);
  if (a.head_dim <= 0 || a.head_dim % (16 / es) != 0)
    return fail(MT_ERR_UNSUPPORTED, "head_dim=%lld must be whole 16-byte chunks (pad the rows)",
                (long long)a.head_dim);
  if (a.head_dim > 128)
    return fail(MT_ERR_UNSUPPORTED, "head_dim=%lld is above 128", (long long)a.head_dim);
  if (a.window < 1 || a.window > INT32_MAX)
    return fail(MT_ERR_INVALID_ARGUMENT, "window=%lld out of range", (long long)a.window);
  if (!(a.scale > 0.f) || !std::isfinite(a.scale) || !(a.softcap >= 0.f) || !std::isfinite(a.softcap))
    return fail(MT_ERR_INVALID_ARGUMENT, "scale must be positive and softcap >= 0 (0 = off), both finite");
  if (a.softcap > 0.f && !(std::isnormal(a.scale / a.softcap) && std::isfinite(a.softcap * kLog2e)))
    return fail(MT_ERR_INVALID_ARGUMENT, "scale / softcap and softcap log2(e) must be normal fp32 numbers");
  // workgroups of kAttnThreads, of which a launch takes fewer than 2^32 threads
  if ((attn_tiles(a.T, a.S) + 1) * std::max(a.heads, 4 * a.kv_heads) >= ((int64_t)1 << 32) / kAttnThreads)
    return fail(MT_ERR_UNSUPPORTED, "%lld tiles (of %d rows, and one for each document) x %lld heads "
                "exceed one launch", (long long)attn_tiles(a.T, a.S), kAttnRows, (long long)a.heads);
  const int64_t strides[] = {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, backward ? a.dout_t : 0,
                             backward ? a.dout_h : 0};
  for (int64_t s : strides)
    if (s < 0 || s % (16 / es) != 0)
      return fail(MT_ERR_INVALID_ARGUMENT, "strides must be whole 16-byte chunks, not negative");
  for (int i = 0; i < 8; i += 2)
    if (strides[i] > (int64_t)1 << 24)
      return fail(MT_ERR_UNSUPPORTED, "rows %lld elements apart: at most 2^24", (long long)strides[i]);
  for (int i = 1; i < 8; i += 2)  // (all heads' addresses in 64 bits)
    if (strides[i] > (int64_t)1 << 40)
      return fail(MT_ERR_UNSUPPORTED, "heads %lld elements apart: at most 2^40", (long long)strides[i]);
  if (a.T == 0) return MT_OK;
  const void* need[] = {a.q, a.k, a.v, a.out, a.lse, a.plan};
  for (const void* x : need)
    if (!x || !aligned16(x))
      return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned (16 bytes) tensor pointer");
  if (!aligned16(a.out_lo)) return fail(MT_ERR_INVALID_ARGUMENT, "misaligned (16 bytes) out_lo");
  if (backward) {
    const void* more[] = {a.dout, a.dq, a.dk, a.dv};
    for (const void* x : more)
      if (!x || !aligned16(x))
        return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned (16 bytes) gradient pointer");
  }
  return MT_OK;
}

AttnArgs attn_args(const mt_attn_args& a) {
  const int64_t es = esize(a.dtype);
  AttnArgs k{};
  k.q = static_cast<const char*>(a.q);
  k.k = static_cast<const char*>(a.k);
  k.v = static_cast<const char*>(a.v);
  k.o = static_cast<const char*>(a.out);
  k.dout = static_cast<const char*>(a.dout);
  k.q_t = a.q_t * es, k.q_h = a.q_h * es, k.k_t = a.k_t * es, k.k_h = a.k_h * es;
  k.v_t = a.v_t * es, k.v_h = a.v_h * es, k.do_t = a.dout_t * es, k.do_h = a.dout_h * es;
  k.out = static_cast<char*>(a.out);
  k.dq = static_cast<char*>(a.dq);
  k.dk = static_cast<char*>(a.dk);
  k.dv = static_cast<char*>(a.dv);
  k.lse = a.lse;
  k.lse_lo = a.lse_lo;
  k.out_lo = a.dtype == MT_DTYPE_BF16 ? static_cast<char*>(a.out_lo) : nullptr;
  k.plan = a.plan;
  k.T = (int32_t)a.T;
  k.Hq = (int32_t)a.heads;
  k.Hk = (int32_t)a.kv_heads;
  k.G = k.Hq / k.Hk;
  k.D = (int32_t)a.head_dim;
  k.tiles_max = (int32_t)attn_tiles(a.T, a.S);
  k.window = (int32_t)a.window;
  k.parts_max = 1;
  k.scale = a.scale;
  k.z_mul = (a.softcap > 0.f ? a.softcap : a.scale) * kLog2e;
  k.cap_mul = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  return k;
}

// The kernels' CAP for a call.
int attn_cap(const mt_attn_args& a) {
  return !(a.softcap > 0.f) ? 0 : a.dtype == MT_DTYPE_BF16 && a.softcap <= kAttnCapFast ? 1 : 2;
}

// kernel<T, DP, CAP, more> for a type, head width and CAP.
#define MT_ATTN_PICK(kernel, dtype, D, cap, ...)                                              \
  ((dtype) == MT_DTYPE_BF16                                                                   \
       ? ((D) <= 64 ? MT_ATTN_PICK_CAP(kernel, __bf16, 64, cap, __VA_ARGS__)                  \
                    : MT_ATTN_PICK_CAP(kernel, __bf16, 128, cap, __VA_ARGS__))                \
       : ((D) <= 64 ? ((cap) ? kernel<float, 64, 2 __VA_ARGS__> : kernel<float, 64, 0 __VA_ARGS__>)          \
                    : ((cap) ? kernel<float, 128, 2 __VA_ARGS__> : kernel<float, 128, 0 __VA_ARGS__>)))
#define MT_ATTN_PICK_CAP(kernel, T, DP, cap, ...)                                             \
  ((cap) == 0 ? kernel<T, DP, 0 __VA_ARGS__>                                                  \
              : (cap) == 1 ? kernel<T, DP, 1 __VA_ARGS__> : kernel<T, DP, 2 __VA_ARGS__>)
#define MT_COMMA ,

// Half tiles (SPLIT = 2 of the kernels) where the rows give fewer workgroups than
// 512 places, two on each CU: 2048 tokens of 8 documents, 14 heads of 64 in fp32,
// forward 46 -> 32 us, dQ 64 -> 46; with more of them the smaller tiles cost more
// than they balance (4096 tokens, 32 heads of 128: 43 -> 55 and 62 -> 74 us).
int attn_split(const mt_attn_args& a) { return cdiv(a.T, kAttnRows) * a.heads <= 512 ? 2 : 1; }

}  // namespace

extern "C" {

size_t mt_attn_plan_bytes(int64_t T, int64_t S) {
  return T < 0 || T > kMaxRows || S < 0 || S > kMaxRows ? 0 : plan_bytes(T, S);
}

int mt_attn_plan(const int32_t* cu_seqlens, const int32_t* prefix_lens, int64_t S, int64_t T,
                 int64_t window, int32_t* plan, size_t plan_size, int32_t* status, mt_stream_t stream) {
  if (T < 0 || T > kMaxRows || S < 0 || S > kMaxRows || attn_tiles(T, S) > INT32_MAX)
    return fail(MT_ERR_INVALID_ARGUMENT, "bad sizes T=%lld S=%lld", (long long)T, (long long)S);
  if (window < 1 || window > INT32_MAX)
    return fail(MT_ERR_INVALID_ARGUMENT, "window=%lld out of range", (long long)window);
  if (!cu_seqlens || !plan || !status) return fail(MT_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!aligned16(plan)) return fail(MT_ERR_INVALID_ARGUMENT, "plan must be 16-byte aligned");
  if (plan_size < plan_bytes(T, S))
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "plan: %zu bytes, %zu needed", plan_size, plan_bytes(T, S));
  hipLaunchKernelGGL(attn_plan_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, cu_seqlens,
                     prefix_lens, (int32_t)S, (int32_t)T, (int32_t)window, (int32_t)attn_tiles(T, S),
                     plan, status);
  return check_launch("attn_plan_kernel");
}

int mt_attn_forward(const mt_attn_args* args, mt_stream_t stream) {
  MT_TRY(attn_check(args, false));
  const mt_attn_args& a = *args;
  if (a.T == 0) return MT_OK;
  const AttnArgs k = attn_args(a);
  const int split = attn_split(a);
  auto kern = split == 2 ? MT_ATTN_PICK(attn_fwd_kernel, a.dtype, a.head_dim, attn_cap(a), MT_COMMA 2)
                         : MT_ATTN_PICK(attn_fwd_kernel, a.dtype, a.head_dim, attn_cap(a), MT_COMMA 1);
  hipLaunchKernelGGL(kern, dim3((uint32_t)(split * k.tiles_max * k.Hq)), dim3(kAttnThreads), 0,
                     (hipStream_t)stream, k);
  return check_launch("attn_fwd_kernel");
}

size_t mt_attn_backward_workspace_bytes(const mt_attn_args* args) {
  if (!args || args->T <= 0 || args->T > kMaxRows || args->S < 0 || args->S > kMaxRows ||
      args->kv_heads <= 0 || args->heads < args->kv_heads || args->heads > kMaxHeads ||
      args->head_dim <= 0 || args->head_dim > 128)
    return 0;  // (attn_check refuses these)
  return 2 * attn_row_bytes(*args) + attn_item_bytes(*args) + attn_part_bytes(*args);
}

int mt_attn_backward(const mt_attn_args* args, void* workspace, size_t workspace_bytes,
                     mt_stream_t stream) {
  MT_TRY(attn_check(args, true));
  const mt_attn_args& a = *args;
  if (a.T == 0) return MT_OK;
  const size_t need = mt_attn_backward_workspace_bytes(args);
  if (!workspace || !aligned16(workspace))
    return fail(MT_ERR_INVALID_ARGUMENT, "null or misaligned workspace");
  if (workspace_bytes < need)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, need);
  AttnArgs k = attn_args(a);
  k.delta = static_cast<float*>(workspace);
  k.factor = reinterpret_cast<float*>(static_cast<char*>(workspace) + attn_row_bytes(a));
  char* items = static_cast<char*>(workspace) + 2 * attn_row_bytes(a);
  k.items = reinterpret_cast<int32_t*>(items);
  k.part = reinterpret_cast<float*>(items + attn_item_bytes(a));
  k.parts_max = attn_parts_max(a);
  k.slots = (int32_t)attn_slots(a);
  const int cap = attn_cap(a);
  hipStream_t s = (hipStream_t)stream;
  const int split = attn_split(a);
  auto dq = split == 2 ? MT_ATTN_PICK(attn_dq_kernel, a.dtype, a.head_dim, cap, MT_COMMA 2)
                       : MT_ATTN_PICK(attn_dq_kernel, a.dtype, a.head_dim, cap, MT_COMMA 1);
  hipLaunchKernelGGL(dq, dim3((uint32_t)(split * k.tiles_max * k.Hq + 1)), dim3(kAttnThreads), 0, s, k);
  MT_TRY(check_launch("attn_dq_kernel"));
  auto dkdv = MT_ATTN_PICK(attn_dkdv_kernel, a.dtype, a.head_dim, cap, );
  hipLaunchKernelGGL(dkdv, dim3((uint32_t)(k.tiles_max * k.Hk * k.parts_max)), dim3(kAttnThreads), 0, s, k);
  MT_TRY(check_launch("attn_dkdv_kernel"));
  if (k.parts_max == 1) return MT_OK;
  auto join = a.dtype == MT_DTYPE_BF16 ? attn_join_kernel<__bf16> : attn_join_kernel<float>;
  hipLaunchKernelGGL(join, dim3((uint32_t)(4 * k.tiles_max * k.Hk)), dim3(kAttnThreads), 0, s, k);
  return check_launch("attn_join_kernel");
}

}  // extern "C"

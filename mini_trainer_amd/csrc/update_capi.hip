// C ABI of libmt_flce.so, the update behind a step's clipped gradients: its
// orthogonalisation.  Declarations and contracts: include/mt_flce.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/mt_flce.h"
#include "capi_common.h"
#include "update_kernels.h"
#include "update_small.h"

using namespace mtf;

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kUpdMost = (int64_t)1 << 31;  // bytes of a copy in fp16
constexpr int64_t kUpdReach = 0xf0000000;      // and of both its terms: offsets of 32 bits
constexpr int64_t kUpdGroup = (int64_t)2 << 30; // bytes of the workspace that a stack of matrices asks for
constexpr int kUpdMostSteps = 64;
constexpr int kUpdCus = 256;

// Workgroups that share the long axis, `stages` of K, of each of `tiles` tiles of 64 of A: as
// many as fill the CUs twice, at most 16, where that saves more than the launch that adds
// their parts costs (a stage of a lone tile 0.22 us, the launch 6).  One 256 x 16384 (10
// tiles of 256 stages): 424 -> 190 us.
int64_t upd_split(int64_t tiles, int64_t stages) {
  if (tiles >= kUpdCus) return 1;
  const int64_t n = std::min<int64_t>({16, 2 * kUpdCus / tiles, stages / 4});
  return n > 1 && 0.22 * (double)(stages - cdiv(stages, n)) > 6.0 ? n : 1;
}

struct UpdLayout {
  int64_t r, c, ld_r, ld_c;
  int64_t l, s0, s1, e, d, fragments, carrier, partial, spread, norm, state, parts, bytes;  // of one matrix
};
bool upd_layout(int64_t m, int64_t n, int dtype, UpdLayout& x) {
  const auto up = [](int64_t v) { return cdiv(v, 64) * 64; };
  if (m < 1 || n < 1 || m > (1 << 30) || n > (1 << 30)) return false;
  x.r = std::min(m, n), x.c = std::max(m, n);
  x.ld_r = up(x.r), x.ld_c = up(x.c);
  const int64_t planes = dtype == MT_DTYPE_F32 ? 2 : 1;
  for (int64_t one : {x.r * x.ld_c * 2, x.c * x.ld_r * 2, x.r * x.ld_r * 2})
    if (one >= kUpdMost || planes * one > kUpdReach) return false;
  int64_t at = 0;
  const auto take = [&](int64_t& where, int64_t bytes) { where = at, at += cdiv(bytes, 256) * 256; };
  take(x.l, x.r * x.ld_c * 2 * planes);
  take(x.s0, x.c * x.ld_r * 2 * planes);
  take(x.s1, x.c * x.ld_r * 2 * planes);
  take(x.e, x.r * x.ld_r * 2 * planes);
  take(x.d, x.r * x.ld_r * 2 * planes);
  take(x.fragments, x.ld_r * x.ld_r * 2 * planes);
  take(x.carrier, cdiv(m, 16) * cdiv(n, 16) * 1024);
  take(x.partial, cdiv(m, 64) * cdiv(n, 64) * 4);  // (of the smallest tiles)
  take(x.spread, cdiv(x.r, 64) * 4);
  take(x.norm, kUpdParts * 8);
  take(x.state, kUpdState * 4);
  const int64_t tiles = cdiv(x.r, 64) * (cdiv(x.r, 64) + 1) / 2, split = upd_split(tiles, x.ld_c / 64);  // (a stack splits less)
  take(x.parts, split > 1 ? tiles * split * 64 * 64 * 4 : 0);
  x.bytes = at;
  return true;
}

int upd_check(const mt_orthogonalize_args* p, UpdLayout& l) {
  if (!p) return fail(MT_ERR_INVALID_ARGUMENT, "null arguments");
  const mt_orthogonalize_args& a = *p;
  const int es = esize(a.dtype);
  if (!es) return fail(MT_ERR_INVALID_ARGUMENT, "dtype %d is not MT_DTYPE_F32 or MT_DTYPE_BF16", a.dtype);
  if (a.batch < 0 || a.m < 0 || a.n < 0)
    return fail(MT_ERR_INVALID_ARGUMENT, "batch=%lld m=%lld n=%lld out of range", (long long)a.batch,
                (long long)a.m, (long long)a.n);
  if (a.steps < 1 || a.steps > kUpdMostSteps)
    return fail(MT_ERR_INVALID_ARGUMENT, "steps=%d: 1 to %d are supported", a.steps, kUpdMostSteps);
  if (!(a.eps >= 0.0) || !std::isfinite(a.eps)) return fail(MT_ERR_INVALID_ARGUMENT, "eps must be >= 0 and finite");
  if (!a.coefficients) return fail(MT_ERR_INVALID_ARGUMENT, "null coefficients");
  if (a.batch == 0 || a.m == 0 || a.n == 0) return MT_OK;
  if (a.batch > (1 << 24) || !upd_layout(a.m, a.n, a.dtype, l))
    return fail(MT_ERR_UNSUPPORTED, "%lld matrices of %lld x %lld: a matrix in fp16 must stay below 2 GiB (of fp32 ones below 1.875)",
                (long long)a.batch, (long long)a.m, (long long)a.n);
  const int64_t most = (int64_t)1 << 40;
  if (a.in_row < a.n || a.in_row > most || a.in_batch < 0 || a.in_batch > most)
    return fail(MT_ERR_INVALID_ARGUMENT, "rows %lld, matrices %lld elements apart", (long long)a.in_row,
                (long long)a.in_batch);
  if (!a.in || !a.out) return fail(MT_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (reinterpret_cast<uintptr_t>(a.in) % es || reinterpret_cast<uintptr_t>(a.out) % es)
    return fail(MT_ERR_INVALID_ARGUMENT, "tensors must be aligned to their element size");
  return MT_OK;
}

// The scales of a step's fp16 copies: powers of two that keep what they hold below 2^14,
// from what the coefficients can make of singular values in [0, most].
struct UpdScales {
  int x, e, d;
  double next;  // the largest singular value after the step
};
bool upd_scales(const double* k, double most, UpdScales& s) {
  const auto scale = [](double bound) {
    return bound > 0.0 ? std::max(-100, std::min(14 - std::ilogb(bound) - 1, 60)) : 0;
  };
  double top = 0.0, lo = 0.0, hi = 0.0;
  for (int i = 0; i <= 4096; ++i) {  // (the grid's gaps and the roundings below it: 1%)
    const double v = most * i / 4096, t = v * v;
    top = std::max(top, std::fabs(v * (k[0] + t * (k[1] + t * k[2]))));
    const double p = t * (k[1] + t * k[2]);
    lo = std::min(lo, p), hi = std::max(hi, p);
  }
  s.x = scale(most), s.e = scale(most * most * 1.01), s.d = scale((hi - lo) * 1.01);
  s.next = top * 1.01;
  return std::isfinite(top) && top < 1e6 && hi - lo < 1e12;
}

// The tile of a product of tiles(t) output tiles of t x t, `stages` stages of K each, that
// move `bytes` an element beside it: the one that costs least, in us.  A CU takes one
// after the other its share of them; tiles of 64 share it and hide most of what they move behind
// each other's products, the larger ones do not.  A lone tile is as slow as its
// stages' latency.  The constants are fitted to 24 sizes in bf16 and 12 in fp32 (three terms
// to a stage) from 128 x 352 to 14336 x 4096 and 1 to 200 matrices, timed with every tile: the
// choice is within 7% of the best at each (4096 x 4096, all of its symmetric products in
// tiles of 64, 128, 192 and 256: 2022, 1831, 1567 and 1807 us; 28 of 256 x 1536: 305, 324,
// 401, 482; 3 of 1001 x 1537 in fp32, all products: 455, 680, 981).
template <class Tiles>
int upd_pick(Tiles tiles, double stages, double bytes, bool split) {
  struct Kind { int F; double stage, alone, exposed; };
  static const Kind one[] = {{8, 1.6, 0.75, 1.0}, {6, 1.07, 0.72, 1.0}, {4, 0.54, 0.3, 1.0}, {2, 0.25, 0.22, 0.36}};
  // (F = 8 would spill in its two writes of an image)
  static const Kind three[] = {{6, 2.2, 1.6, 1.0}, {4, 1.1, 0.75, 1.0}, {2, 0.5, 0.5, 0.36}};
  const Kind* kinds = split ? three : one;
  const int count = split ? 3 : 4;
  constexpr double kRate = 21e3;  // bytes a us of a CU, when all of them ask
  int best = 2;
  double least = INFINITY;
  for (int i = 0; i < count; ++i) {
    const Kind& k = kinds[i];
    const int64_t n = tiles(upd_tile(k.F));
    const double busy = std::min(1.0, std::max((double)n / kUpdCus, 0.15));
    const double moved = bytes * upd_tile(k.F) * upd_tile(k.F) / kRate * busy, product = stages * k.stage;
    const double many = (double)cdiv(n, kUpdCus) *
                        (std::max(moved, product) + k.exposed * std::min(moved, product));
    const double cost = std::max(many, 2.0 + 0.145 * k.F * k.F + stages * k.alone + moved);
    if (cost < least) least = cost, best = k.F;
  }
  return best;
}

template <int MOST, class F>
int upd_with(int kind, F f) {
  switch (kind) {
    case 8: return f(std::integral_constant<int, MOST>());
    case 6: return f(std::integral_constant<int, 6>());
    case 4: return f(std::integral_constant<int, 4>());
    default: return f(std::integral_constant<int, 2>());
  }
}

// The fragment rows of the small matrices' kernel that a matrix goes to (0: none), and the
// products to a term there.  bf16 matrices of at most 32 rows take three as fp32 ones do,
// where LDS holds them: a rounding of one of their few elements reaches the whole result
// (4 x 4 off by up to 0.015 of the norm, 16 x 64 of rank 1 by 0.008, so by 1e-6 before the
// last rounding).
struct UpdSmall {
  int rows, terms;
};
UpdSmall upd_small(const UpdLayout& l, int steps, int dtype) {
  if (steps > kUpdSmallSteps) return {0, 0};
  const auto rows = [&](int terms, int most) {
    for (int R = 1; R <= most; R *= 2)
      if (l.r <= 16 * R)
        return l.c <= 128 * upd_small_columns(R, terms) && upd_small_lds(R, l.c, terms) <= kUpdSmallLds ? R : 0;
    return 0;
  };
  const int split = rows(3, dtype == MT_DTYPE_F32 ? 4 : 2);
  if (split || dtype == MT_DTYPE_F32) return {split, 3};
  return {rows(1, 8), 1};
}

template <class T>
int launch_small(UpdSmall way, const UpdSmallArgs& k, int64_t batch, hipStream_t stream) {
  const auto with = [&](auto rows, auto terms) {
    hipLaunchKernelGGL((upd_small_kernel<T, decltype(rows)::value, decltype(terms)::value>), dim3((uint32_t)batch),
                       dim3(512), 0, stream, k);
    return check_launch("upd_small_kernel");
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  constexpr std::integral_constant<int, 3> three{};
  constexpr std::integral_constant<int, 4> four{};
  if (way.terms == 3) {
    if (way.rows == 1) return with(one, three);
    if (way.rows == 2) return with(two, three);
    if constexpr (sizeof(T) == 4) return with(four, three);
  } else if constexpr (sizeof(T) == 2) {
    if (way.rows == 1) return with(one, one);
    if (way.rows == 2) return with(two, one);
    if (way.rows == 4) return with(four, one);
    return with(std::integral_constant<int, 8>(), one);
  }
  return fail(MT_ERR_UNSUPPORTED, "%d rows of fragments, %d terms", way.rows, way.terms);
}

template <class T>
int launch_orthogonalize(UpdArgs k, const mt_orthogonalize_args& p, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T), TERMS = sizeof(T) == 4 ? 3 : 1;
  const int64_t small_tiles = cdiv(k.r, 64) * (cdiv(k.r, 64) + 1) / 2;
  k.split = (int32_t)upd_split(k.batch * small_tiles, k.ld_c / 64);
  const int64_t runs = (int64_t)k.m * cdiv(k.n, 256 * (k.vec ? V : 1));
  k.norm_parts = (int32_t)std::min<int64_t>(cdiv(runs, 4), kUpdParts);
  const dim3 norm_grid((uint32_t)k.norm_parts, (uint32_t)k.batch);
  if (k.vec) hipLaunchKernelGGL((upd_norm_kernel<T, V>), norm_grid, dim3(256), 0, stream, k);
  else hipLaunchKernelGGL((upd_norm_kernel<T, 1>), norm_grid, dim3(256), 0, stream, k);
  MT_TRY(check_launch("upd_norm_kernel"));
  const dim3 convert_grid((uint32_t)(cdiv(k.m, 64) * cdiv(k.n, 64)), (uint32_t)k.batch);
  if (k.vec) hipLaunchKernelGGL((upd_convert_kernel<T, V, TERMS>), convert_grid, dim3(256), 0, stream, k);
  else hipLaunchKernelGGL((upd_convert_kernel<T, 1, TERMS>), convert_grid, dim3(256), 0, stream, k);
  MT_TRY(check_launch("upd_convert_kernel"));

  const auto triangle = [&](int64_t t) { return k.batch * (cdiv(k.r, t) * (cdiv(k.r, t) + 1) / 2); };
  const auto all = [&](int64_t t) { return k.batch * cdiv(k.m, t) * cdiv(k.n, t); };
  // both symmetric products go by one tile (fragments of E pass between them): by their mean
  constexpr int planes = TERMS == 3 ? 2 : 1;
  const int symmetric = upd_pick(triangle, (cdiv(k.c, 64) + cdiv(k.r, 64)) / 2.0, 6.0 * planes, TERMS == 3);
  const int apply = upd_pick(all, (double)cdiv(k.r, 64), 8.0 + 4.0 * planes, TERMS == 3);
  constexpr int kMost = TERMS == 3 ? 6 : 8;
  double most = 1.0;
  UpdScales now, next;
  if (!upd_scales(p.coefficients, most, now)) return fail(MT_ERR_UNSUPPORTED, "these coefficients diverge");
  for (int step = 0; step < p.steps; ++step, now = next) {
    const double* q = p.coefficients + 3 * step;
    next = now;
    if (step + 1 < p.steps && !upd_scales(q + 3, now.next, next))
      return fail(MT_ERR_UNSUPPORTED, "these coefficients diverge");
    k.first = step == 0, k.last = step + 1 == p.steps, k.lifted = step + 2 < p.steps;
    k.x_exponent = now.x;
    k.a = (float)q[0], k.b = (float)q[1], k.cc = (float)q[2];
    k.x_unscale = std::ldexp(1.f, -now.x), k.x_scale = std::ldexp(1.f, next.x);
    k.e_scale = std::ldexp(1.f, now.e), k.e_unscale = std::ldexp(1.f, -now.e);
    k.d_scale = std::ldexp(1.f, now.d), k.d_unscale = std::ldexp(1.f, -now.d);
    MT_TRY(upd_with<kMost>(symmetric, [&](auto F) {
      constexpr int f = decltype(F)::value;
      k.tiles_m = k.tiles_n = (int32_t)cdiv(k.r, upd_tile(f));
      k.tiles = k.tiles_m * (k.tiles_m + 1) / 2, k.spreads = k.tiles_m;
      const dim3 grid((uint32_t)(k.tiles * k.batch));
      if (f == 2 && k.split > 1) {
        hipLaunchKernelGGL((upd_symmetric_kernel<2, TERMS, kUpdPart>), dim3(grid.x * (uint32_t)k.split), dim3(256), 0,
                           stream, k);
        MT_TRY(check_launch("upd_symmetric_kernel"));
        hipLaunchKernelGGL((upd_symmetric_kernel<2, TERMS, kUpdJoin>), grid, dim3(256), 0, stream, k);
      } else {
        hipLaunchKernelGGL((upd_symmetric_kernel<f, TERMS, kUpdWhole>), grid, dim3(256), 0, stream, k);
      }
      MT_TRY(check_launch("upd_symmetric_kernel"));
      hipLaunchKernelGGL((upd_symmetric_kernel<f, TERMS, kUpdSquare>), grid, dim3(256), 0, stream, k);
      return check_launch("upd_symmetric_kernel");
    }));
    MT_TRY(upd_with<kMost>(apply, [&](auto F) {
      constexpr int f = decltype(F)::value;
      k.tiles_m = (int32_t)cdiv(k.m, upd_tile(f)), k.tiles_n = (int32_t)cdiv(k.n, upd_tile(f));
      k.tiles = k.partials = k.tiles_m * k.tiles_n;
      const auto kern = TERMS == 1 && k.lifted ? upd_apply_kernel<T, f, TERMS, TERMS == 1>
                                               : upd_apply_kernel<T, f, TERMS, false>;
      hipLaunchKernelGGL(kern, dim3((uint32_t)(k.tiles * k.batch)), dim3(256), 0, stream, k);
      return check_launch("upd_apply_kernel");
    }));
    std::swap(k.s0, k.s1);
  }
  return MT_OK;
}

}  // namespace

extern "C" {

size_t mt_orthogonalize_workspace_bytes(const mt_orthogonalize_args* args) {
  UpdLayout l;
  if (!args || args->batch < 1 || args->batch > (1 << 24) || !esize(args->dtype) ||
      !upd_layout(args->m, args->n, args->dtype, l) || upd_small(l, args->steps, args->dtype).rows)
    return 0;
  return (size_t)(l.bytes * std::max<int64_t>(1, std::min(args->batch, kUpdGroup / l.bytes)));
}

int mt_orthogonalize(const mt_orthogonalize_args* args, void* workspace, size_t workspace_bytes,
                     mt_stream_t stream) {
  UpdLayout l;
  MT_TRY(upd_check(args, l));
  const mt_orthogonalize_args& a = *args;
  if (a.batch == 0 || a.m == 0 || a.n == 0) return MT_OK;
  const int es = esize(a.dtype);
  const int64_t V = 16 / es;
  const bool vec = aligned16(a.in) && aligned16(a.out) && a.n % V == 0 && (a.m == 1 || a.in_row % V == 0) &&
                   (a.batch == 1 || a.in_batch % V == 0);
  const UpdSmall small = upd_small(l, a.steps, a.dtype);
  UpdSmallArgs sm{};
  double most = 1.0;
  for (int step = 0; step < a.steps; ++step) {  // before anything is launched
    UpdScales s;
    const double* q = a.coefficients + 3 * step;
    if (!std::isfinite(q[0]) || !std::isfinite(q[1]) || !std::isfinite(q[2]))
      return fail(MT_ERR_INVALID_ARGUMENT, "coefficients must be finite");
    if (!upd_scales(q, most, s))
      return fail(MT_ERR_UNSUPPORTED, "coefficients that carry singular values beyond 10^6");
    most = s.next;
    if (small.rows) {
      if (step) sm.step[step - 1].x_scale = std::ldexp(1.f, s.x);
      sm.step[step] = {(float)q[0], (float)q[1], (float)q[2], std::ldexp(1.f, -s.x), std::ldexp(1.f, s.e),
                       std::ldexp(1.f, -s.e), std::ldexp(1.f, s.d), std::ldexp(1.f, -s.d), 1.f};
    }
  }
  if (small.rows) {
    sm.in_row = a.in_row, sm.in_batch = a.in_batch;
    sm.eps = a.eps;
    sm.m = (int32_t)a.m, sm.n = (int32_t)a.n, sm.r = (int32_t)l.r, sm.c = (int32_t)l.c;
    sm.steps = a.steps, sm.vec = vec;
    constexpr int64_t most_at_once = (int64_t)1 << 22;  // workgroups of a launch
    for (int64_t at = 0; at < a.batch; at += most_at_once) {
      const int64_t n = std::min(most_at_once, a.batch - at);
      sm.in = static_cast<const char*>(a.in) + at * a.in_batch * es;
      sm.out = static_cast<char*>(a.out) + at * a.m * a.n * es;
      MT_TRY(a.dtype == MT_DTYPE_BF16 ? launch_small<__bf16>(small, sm, n, (hipStream_t)stream)
                                      : launch_small<float>(small, sm, n, (hipStream_t)stream));
    }
    return MT_OK;
  }
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(MT_ERR_INVALID_ARGUMENT, "null workspace, or one that is not aligned to 256 bytes");
  if (workspace_bytes < (size_t)l.bytes)
    return fail(MT_ERR_WORKSPACE_TOO_SMALL, "workspace: %zu bytes, %zu needed", workspace_bytes, (size_t)l.bytes);
  // matrices at a time: what the workspace holds, within one launch's workgroups
  const int64_t tiles = cdiv(a.m, 64) * cdiv(a.n, 64);
  const int64_t group = std::min<int64_t>({a.batch, (int64_t)(workspace_bytes / (size_t)l.bytes), 32768,
                                           std::max<int64_t>(1, (1 << 23) / tiles)});
  if (tiles > (1 << 23)) return fail(MT_ERR_UNSUPPORTED, "%lld x %lld exceeds one launch", (long long)a.m, (long long)a.n);
  UpdArgs k{};
  k.ws = static_cast<char*>(workspace);
  k.ws_stride = l.bytes;
  k.in_row = a.in_row, k.in_batch = a.in_batch;
  k.l = l.l, k.s0 = l.s0, k.s1 = l.s1, k.e = l.e, k.d = l.d;
  k.fragments = l.fragments, k.carrier = l.carrier, k.partial = l.partial, k.spread = l.spread;
  k.norm = l.norm, k.state = l.state, k.parts = l.parts;
  k.eps = a.eps;
  k.m = (int32_t)a.m, k.n = (int32_t)a.n, k.r = (int32_t)l.r, k.c = (int32_t)l.c;
  k.ld_r = (int32_t)l.ld_r, k.ld_c = (int32_t)l.ld_c;
  k.vec = vec;
  for (int64_t at = 0; at < a.batch; at += group) {
    k.batch = (int32_t)std::min(group, a.batch - at);
    k.in = static_cast<const char*>(a.in) + at * a.in_batch * es;
    k.out = static_cast<char*>(a.out) + at * a.m * a.n * es;
    MT_TRY(a.dtype == MT_DTYPE_BF16 ? launch_orthogonalize<__bf16>(k, a, (hipStream_t)stream)
                                    : launch_orthogonalize<float>(k, a, (hipStream_t)stream));
  }
  return MT_OK;
}

}  // extern "C"

// The matrix products of an orthogonalised update (gfx950): C = A B^T in fp16 with fp32
// sums, both operands' rows contiguous along K.
//
// Workgroup = 4 waves, output tile 32 F x 32 F; wave (wm, wn) = (w >> 1, w & 1) owns a
// block of 16 F x 16 F = F x F fragments of v_mfma_f32_16x16x32_f16.  F = 8 keeps 256
// accumulators a lane (the AGPR file), reads the fewest LDS bytes per flop and leaves one
// wave per SIMD; smaller F share a CU between workgroups.
//
// K advances in stages of 64 (128 bytes of each operand row), in two halves of 32, out of
// a ring of LDS slots that LDS DMA fills: three for A, N = two (F = 8) or three for B, so
// that one operand's DMA is issued beside each half.  With F0, F1 the fragments of the
// halves of stage g:
//
//   phase 1   F^2 MFMAs on F0(g)  | 2 F LDS reads of F1(g), F DMA: A of stage g + 2
//   sync      own reads retired, own DMA of stage g + 1 landed, barrier
//   phase 2   F^2 MFMAs on F1(g)  | 2 F LDS reads of F0(g + 1), F DMA: B of stage g + N
//
// The barrier lies between two blocks of MFMAs whose operands are in registers.  Memory
// instructions are spread thinly between the MFMAs by scheduling fences, as in
// flce_gemm_bf16.h, whose tile layout (tile_off) and waits these loops use.
//
// Rows past the operand's end and K past its last stage need no masks: a buffer's bound
// turns reads beyond its last row into zeros, and operands are stored with zeros up to
// whole stages.
#pragma once

#include "flce_gemm_bf16.h"

namespace mtf {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

constexpr int kUpdStage = 64;  // K elements of a stage

constexpr int upd_tile(int F) { return 32 * F; }
constexpr int upd_slot(int F) { return upd_tile(F) * 128; }   // bytes: one operand, one stage
constexpr int upd_pitch(int F) { return upd_tile(F) * 2 + 16; }  // bytes of an image row, see below
// Stages of A and of B that the ring holds.  More would cost tiles of 64 their neighbours on
// the CU (4 instead of 3: one 256 x 16384 370 instead of 424 us, 28 of 256 x 1536 289 instead
// of 261).
constexpr int upd_slots_a(int) { return 3; }
constexpr int upd_slots_b(int F) { return F == 8 ? 2 : 3; }
constexpr int upd_lds(int F) { return (upd_slots_a(F) + upd_slots_b(F)) * upd_slot(F); }

__device__ __forceinline__ f32x4_t upd_mma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b),
                                                c, 0, 0, 0);
}

// An operand: `rows` rows of ld halves (whole stages).  fp32 updates keep the value rounded
// to fp16 and what the rounding left (hi, lo), 32 of each in turn: a stage is 32 columns of
// the matrix, hi in its first half and lo in its second.
struct UpdMatrix {
  const char* at;
  uint32_t bytes;  // 2 rows ld, below 0xf0000000
  uint32_t ld;     // halves of a row
  uint32_t rows;
};
// Place in a row of 2 ld halves of column `col`, t = 1 for lo; with one term a row is the
// matrix's.
template <int TERMS>
__device__ __forceinline__ int32_t upd_column(int32_t col, int t) {
  return TERMS == 1 ? col : (col & ~31) * 2 + 32 * t + (col & 31);
}

template <int F>
struct UpdOperand {
  rsrc_t rsrc;
  uint32_t off[F];
  uint32_t frag[2];

  __device__ __forceinline__ void init(const UpdMatrix& m, uint32_t row0, uint32_t wave_row0) {
    rsrc = make_rsrc(m.at, m.bytes);
    const uint32_t l = lane_id();
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)F; ++i) {
      // DMA instruction q fills 1 KiB: 8 rows of a 16-row group, in tile_off's order
      const uint32_t q = wave_id() * F + i;
      const uint32_t row = (q >> 1) * 16 + ((l >> 3) & 1u) * 8 + (q & 1u) * 4 + (l >> 4);
      const uint32_t chunk = (l & 7u) ^ ((q & 1u) * 4 + (l >> 4));
      off[i] = row0 + row < m.rows ? (row0 + row) * m.ld * 2u + chunk * 16u : 0xf0000000u;
    }
#pragma unroll
    for (uint32_t kk = 0; kk < 2; ++kk) frag[kk] = tile_off(wave_row0 + (l & 15u), kk * 4 + (l >> 4));
  }
  __device__ __forceinline__ void issue(char* slot, int kt, int i) const {
    dma16(rsrc, slot + (wave_id() * F + (uint32_t)i) * 1024u, off[i], (uint32_t)kt * 128u);
  }
  __device__ __forceinline__ u32x4_t read(const char* slot, int kk, int f) const {
    return lds_read16(slot, frag[kk] + (uint32_t)f * 2048u);
  }
};

template <int N>
__device__ __forceinline__ void upd_wait_vm() {  // every DMA but the last N issued has landed
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// acc = sum over the KT stages from `first` on of A B^T; with TERMS = 3 of hi hi, hi lo and lo hi.
template <int F, int TERMS>
__device__ __forceinline__ void upd_mainloop(char* lds, const UpdOperand<F>& a, const UpdOperand<F>& b, int first,
                                             int KT, f32x4_t (&acc)[F][F]) {
  constexpr int kSlot = upd_slot(F), NA = upd_slots_a(F), NB = upd_slots_b(F);
  static_assert(NA == NB || NA == NB + 1, "what the waits count on");
  static_assert(upd_lds(F) >= upd_tile(F) * upd_pitch(F), "an image of the tile");
  // MFMAs before each LDS read; the others follow the last one and hide its latency
  constexpr int kPer = F >= 8 ? 3 : F >= 6 ? 2 : 1;
  char* const slots_b = lds;
  char* const slots_a = lds + NB * kSlot;
  // Past the end the DMA loads the last stage again, into slots that are not read any more,
  // so that every stage issues as much.
  auto at = [&](int s) __attribute__((always_inline)) { return first + (s < KT ? s : KT - 1); };
#pragma unroll
  for (int m = 0; m < F; ++m)
#pragma unroll
    for (int n = 0; n < F; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // the stages that the phases are ahead
#pragma unroll
  for (int s = 0; s < (NA - 1 > NB ? NA - 1 : NB); ++s) {
    const int kt = at(s);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (s < NA - 1) a.issue(slots_a + s * kSlot, kt, i);
      if (s < NB) b.issue(slots_b + s * kSlot, kt, i);
    }
  }
  upd_wait_vm<F * (NA + NB - 3)>();  // stage 0: of A NA - 2 stages follow it, of B NB - 1
  __builtin_amdgcn_s_barrier();
  u32x4_t fa0[F], fb0[F], fa1[F], fb1[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    fa0[f] = a.read(slots_a, 0, f);
    fb0[f] = b.read(slots_b, 0, f);
  }
  lgkm_wait0();
  int ga = 0, gb = 0;  // slots of stage g
  for (int g = 0; g < KT; ++g) {
    sched_fence();
    const int ga1 = ga == NA - 1 ? 0 : ga + 1, gap = ga == 0 ? NA - 1 : ga - 1;  // of stages g + 1 and g - 1
    const int gb1 = gb == NB - 1 ? 0 : gb + 1;
    const char* ra = slots_a + ga * kSlot;
    const char* rb = slots_b + gb * kSlot;
    int kt = at(g + NA - 1);
    if constexpr (TERMS == 3) {
      // hi hi beside the reads of lo, hi lo beside the DMA of A, and behind the barrier lo hi
      // beside the next stage's reads of hi, each of B into the registers that its column of
      // products has just left (a third fewer LDS reads and DMA than three products of one
      // term)
#pragma unroll
      for (int n = 0; n < F; ++n) {
#pragma unroll
        for (int m = 0; m < F; ++m) acc[m][n] = upd_mma(fb0[n], fa0[m], acc[m][n]);
        fa1[n] = a.read(ra, 1, n);
        fb1[n] = b.read(rb, 1, n);
        sched_fence();
      }
#pragma unroll
      for (int n = 0; n < F; ++n) {
#pragma unroll
        for (int m = 0; m < F; ++m) acc[m][n] = upd_mma(fb1[n], fa0[m], acc[m][n]);
        a.issue(slots_a + gap * kSlot, kt, n);
        sched_fence();
      }
      lgkm_wait0();
      upd_wait_vm<F * (NA + NB - 4)>();  // as below
      __builtin_amdgcn_s_barrier();
      sched_fence();
      kt = at(g + NB);
#pragma unroll
      for (int n = 0; n < F; ++n) {
        fa0[n] = a.read(slots_a + ga1 * kSlot, 0, n);
#pragma unroll
        for (int m = 0; m < F; ++m) acc[m][n] = upd_mma(fb0[n], fa1[m], acc[m][n]);
        b.issue(slots_b + gb * kSlot, kt, n);
        fb0[n] = b.read(slots_b + gb1 * kSlot, 0, n);
        sched_fence();
      }
      ga = ga1, gb = gb1;
      continue;
    }
#pragma unroll
    for (int i = 0; i < 2 * F; ++i) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int k = i * kPer + j;
        acc[k / F][k % F] = upd_mma(fb0[k % F], fa0[k / F], acc[k / F][k % F]);
      }
      if (i & 1) fb1[i >> 1] = b.read(rb, 1, i >> 1);
      else fa1[i >> 1] = a.read(ra, 1, i >> 1);
      if (i & 1) a.issue(slots_a + gap * kSlot, kt, i >> 1);
      sched_fence();
    }
#pragma unroll
    for (int k = 2 * F * kPer; k < F * F; ++k)
      acc[k / F][k % F] = upd_mma(fb0[k % F], fa0[k / F], acc[k / F][k % F]);
    sched_fence();
    // stage g + 1 has landed: the stages g + 2 .. g + NA - 1 of A and .. g + NB - 1 of B follow it
    lgkm_wait0();
    upd_wait_vm<F * (NA + NB - 4)>();
    __builtin_amdgcn_s_barrier();
    sched_fence();
    const char* ra1 = slots_a + ga1 * kSlot;
    const char* rb1 = slots_b + gb1 * kSlot;
    kt = at(g + NB);
#pragma unroll
    for (int i = 0; i < 2 * F; ++i) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int k = i * kPer + j;
        acc[k / F][k % F] = upd_mma(fb1[k % F], fa1[k / F], acc[k / F][k % F]);
      }
      if (i & 1) b.issue(slots_b + gb * kSlot, kt, i >> 1);
      if (i & 1) fb0[i >> 1] = b.read(rb1, 0, i >> 1);
      else fa0[i >> 1] = a.read(ra1, 0, i >> 1);
      sched_fence();
    }
#pragma unroll
    for (int k = 2 * F * kPer; k < F * F; ++k)
      acc[k / F][k % F] = upd_mma(fb1[k % F], fa1[k / F], acc[k / F][k % F]);
    sched_fence();
    lgkm_wait0();
    ga = ga1, gb = gb1;
  }
  wait_vm0();
  __syncthreads();  // the ring is free
}

}  // namespace mtf

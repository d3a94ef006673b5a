// The MFMA stages and the copy rings of the 256x256 core's dense operands (plz_gemm2.cuh): shared by
// the GEMM kernels of plz_gemm2.hip and the vocabulary losses of plz_vocab.hip.
#pragma once
#include "plz_gemm2.cuh"

namespace plz {
namespace g2 {

// Row stride in bytes of a 256x256 bf16 tile staged in LDS by an epilogue: padded so that the two
// 64-byte row segments a wave writes per instruction fall in different banks.
constexpr int EPI_RS = 528;

// Masked register-path copies for a partial reduction stage (r >= rend reads as zero) and for
// the rank-r second segment.
__device__ __forceinline__ void copy_row_tile_masked(uint4* lds, const uint16_t* p, int64_t ld,
                                                     int64_t row0, int64_t nrows, int64_t r0,
                                                     int64_t rend, int64_t half = 0) {
#pragma unroll
  for (int it = 0; it < COPY_INSTS; ++it) {
    const int ch = it * NTHR + threadIdx.x;
    const int row = ch >> 3, c = ch & 7;
    const int64_t gr = row0 + row, gk = r0 + 8 * c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (gr < nrows && gk < rend)
      v = *reinterpret_cast<const uint4*>(p + half_row(gr, half) * ld + gk);
    lds[row_chunk(row, c)] = v;
  }
}
__device__ __forceinline__ void copy_col_tile_masked(uint4* lds, const uint16_t* p, int64_t ld,
                                                     int64_t row0, int64_t nrows, int64_t r0,
                                                     int64_t rend) {
#pragma unroll
  for (int it = 0; it < COPY_INSTS; ++it) {
    const int ch = it * NTHR + threadIdx.x;
    const int kr = ch >> 5, c = ch & 31;
    const int64_t gr = row0 + 8 * c, gk = r0 + kr;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (gr < nrows && gk < rend) v = *reinterpret_cast<const uint4*>(p + gk * ld + gr);
    lds[col_chunk(kr, c)] = v;
  }
}

// One reduction stage of MFMAs on LDS tiles: 4 k-steps of 16, 4x4 blocks of 32x32 per wave.
// Fragments are double-buffered in registers: the LDS reads of k-step ks+1 are issued before
// the 16 MFMAs of k-step ks, so one wave per SIMD keeps the matrix core busy. The scheduling
// barriers pin that order (left alone, the compiler sinks each A read next to its first
// MFMA and exposes the LDS latency every 4 MFMAs). fill(part), part = 0..1, runs between
// the MFMA groups: VALU work for the next stage (the palette dequantisation) that then
// overlaps with the matrix core.
template <bool A_COL, bool B_COL>
__device__ __forceinline__ void load_frags(const lds_u8* a_s, const lds_u8* b_s, int ks, int wi,
                                           int wj, int lane, bf16x8 (&a)[WT_I], bf16x8 (&b)[WT_J]) {
#pragma unroll
  for (int i = 0; i < WT_I; ++i)
    a[i] = A_COL ? frag_col(a_s, wi * (32 * WT_I) + 32 * i, ks, lane)
                 : frag_row((const uint4*)a_s, wi * (32 * WT_I) + 32 * i, ks, lane);
#pragma unroll
  for (int j = 0; j < WT_J; ++j)
    b[j] = B_COL ? frag_col(b_s, wj * (32 * WT_J) + 32 * j, ks, lane)
                 : frag_row((const uint4*)b_s, wj * (32 * WT_J) + 32 * j, ks, lane);
}
constexpr int MFMA_PER_KSTEP = WT_I * WT_J;  // 8
__device__ __forceinline__ void mma_kstep(f32x16 (&acc)[WT_I][WT_J], const bf16x8 (&a)[WT_I],
                                          const bf16x8 (&b)[WT_J]) {
#pragma unroll
  for (int i = 0; i < WT_I; ++i)
#pragma unroll
    for (int j = 0; j < WT_J; ++j)
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
}
// Instruction interleave of one k-step (MFMA_PER_KSTEP MFMAs): the LDS reads of the next
// k-step, the next stage's global->LDS copies (first k-step only) and the palette
// dequantisation (VALU and LDS stores) are spread between the MFMAs, so that no burst of one
// kind stalls the issue of MFMAs (sched_group_barrier masks: 0x008 MFMA, 0x100 LDS read,
// 0x200 LDS write, 0x020 VMEM, 0x002 VALU).
template <int NREAD, int NVMEM, int NVALU, int NWRITE>
__device__ __forceinline__ void interleave_kstep() {
  constexpr int M = MFMA_PER_KSTEP;
  constexpr int R = (NREAD + M - 1) / M, V = (NVMEM + M - 1) / M;
  constexpr int A = (NVALU + M - 1) / M, W = (NWRITE + M - 1) / M;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (R > 0 && i * R < NREAD) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    if (V > 0 && i * V < NVMEM) __builtin_amdgcn_sched_group_barrier(0x020, V, 0);
    if (A > 0) __builtin_amdgcn_sched_group_barrier(0x002, A, 0);
    if (W > 0 && i * W < NWRITE) __builtin_amdgcn_sched_group_barrier(0x200, W, 0);
  }
}

// A whole stage without overlap (the partial and LoRA stages). Only the first nks k-steps
// hold data (the rest of the stage is zero fill), so only those run.
template <bool A_COL, bool B_COL>
__device__ __forceinline__ void mma_stage_sync(const lds_u8* a_s, const lds_u8* b_s,
                                               f32x16 (&acc)[WT_I][WT_J], int wi, int wj,
                                               int lane, int nks) {
#pragma unroll
  for (int ks = 0; ks < BK / 16; ++ks) {
    if (ks >= nks) break;
    bf16x8 a[WT_I], b[WT_J];
    load_frags<A_COL, B_COL>(a_s, b_s, ks, wi, wj, lane, a, b);
    mma_kstep(acc, a, b);
  }
}

// a_s, b_s: this stage's tiles; na_s, nb_s: the LDS slots that dma(na_s, nb_s) and
// fill(part, nb_s) write for a later stage. All four are distinct slots, and saying so
// (__restrict__) lets the compiler see that the fragment reads cannot alias the copies in
// flight: without it, it waits for every outstanding copy before the first LDS read that
// follows them, one k-step after issuing the next stage's copies.
template <bool A_COL, bool B_COL, bool FILL, typename Dma, typename Fill>
__device__ __forceinline__ void mma_stage(const lds_u8* __restrict__ a_s,
                                          const lds_u8* __restrict__ b_s,
                                          lds_u8* __restrict__ na_s, lds_u8* __restrict__ nb_s,
                                          f32x16 (&acc)[WT_I][WT_J], int wi, int wj, int lane,
                                          Dma&& dma, Fill&& fill) {
  // LDS read instructions per k-step: a row fragment is one ds_read_b128, a col fragment two
  // ds_read_b64_tr_b16
  constexpr int NREAD = WT_I * (A_COL ? 2 : 1) + WT_J * (B_COL ? 2 : 1);
  // palette dequantisation of one word: ~31 VALU and two 16-byte LDS stores (k-steps 0, 1)
  constexpr int NV = FILL ? 32 : 0;
  constexpr int NW = FILL ? 2 : 0;
  // global->LDS copies of the next stage issued by dma(): COPY_INSTS per dense operand
  constexpr int NDMA = COPY_INSTS * (FILL ? 1 : 2);
  ColBases<WT_I> ca;
  ColBases<WT_J> cb;
  if constexpr (A_COL) col_bases(a_s, wi * (32 * WT_I), lane, ca);
  if constexpr (A_COL && B_COL) col_bases(b_s, wj * (32 * WT_J), lane, cb);
  auto frags = [&](int ks, bf16x8 (&a)[WT_I], bf16x8 (&b)[WT_J]) {
    if constexpr (!A_COL) {  // one Col operand at most: the compiler's own addressing is as good
      load_frags<false, B_COL>(a_s, b_s, ks, wi, wj, lane, a, b);
      return;
    }
#pragma unroll
    for (int i = 0; i < WT_I; ++i)
      a[i] = A_COL ? frag_col_at(ca.p1[i], ca.p2[i], ks)
                   : frag_row((const uint4*)a_s, wi * (32 * WT_I) + 32 * i, ks, lane);
#pragma unroll
    for (int j = 0; j < WT_J; ++j)
      b[j] = B_COL ? frag_col_at(cb.p1[j], cb.p2[j], ks)
                   : frag_row((const uint4*)b_s, wj * (32 * WT_J) + 32 * j, ks, lane);
  };
  bf16x8 a0[WT_I], b0[WT_J], a1[WT_I], b1[WT_J];
  frags(0, a0, b0);
  __builtin_amdgcn_sched_barrier(0);
  frags(1, a1, b1);
  dma(na_s, nb_s);
  mma_kstep(acc, a0, b0);
  fill(0, nb_s);
  interleave_kstep<NREAD, NDMA, NV, NW>();
  __builtin_amdgcn_sched_barrier(0);
  frags(2, a0, b0);
  mma_kstep(acc, a1, b1);
  fill(1, nb_s);
  interleave_kstep<NREAD, 0, NV, NW>();
  __builtin_amdgcn_sched_barrier(0);
  frags(3, a1, b1);
  mma_kstep(acc, a0, b0);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  mma_kstep(acc, a1, b1);
  interleave_kstep<0, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
}

// One stage of the dense kernels' two-slot ring whose last k-step overlaps the boundary with
// the next stage. A barrier between stages stalls every SIMD: the workgroup's waves reach it
// together, and behind it each wave must read the next stage's first fragments before its
// next MFMA. Here the barrier runs before the last k-step instead: k-steps 0..2 issue their
// MFMAs and the fragment reads of the following k-step; bar() waits for this wave's copies of
// the next stage and its own fragment reads and passes the barrier, after which no wave reads
// this stage's slot any more and the next stage's tiles are complete; dma() then copies the
// stage after next into this stage's slot (d_a, d_b: the same LDS as a_s, b_s, written only
// after the barrier), and the last k-step's MFMAs cover the reads of the next stage's first
// fragments into a0/b0.
template <bool A_COL, bool B_COL, typename Bar, typename Dma>
__device__ __forceinline__ void mma_stage_pipe(const lds_u8* __restrict__ a_s,
                                               const lds_u8* __restrict__ b_s,
                                               const lds_u8* __restrict__ na_s,
                                               const lds_u8* __restrict__ nb_s,
                                               lds_u8* __restrict__ d_a, lds_u8* __restrict__ d_b,
                                               f32x16 (&acc)[WT_I][WT_J], int wi, int wj,
                                               int lane, bf16x8 (&a0)[WT_I], bf16x8 (&b0)[WT_J],
                                               Bar&& bar, Dma&& dma) {
  constexpr int NREAD = WT_I * (A_COL ? 2 : 1) + WT_J * (B_COL ? 2 : 1);
  bf16x8 a1[WT_I], b1[WT_J];
  load_frags<A_COL, B_COL>(a_s, b_s, 1, wi, wj, lane, a1, b1);
  mma_kstep(acc, a0, b0);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  load_frags<A_COL, B_COL>(a_s, b_s, 2, wi, wj, lane, a0, b0);
  mma_kstep(acc, a1, b1);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  load_frags<A_COL, B_COL>(a_s, b_s, 3, wi, wj, lane, a1, b1);
  mma_kstep(acc, a0, b0);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  bar();
  __builtin_amdgcn_sched_barrier(0);
  dma(d_a, d_b);
  load_frags<A_COL, B_COL>(na_s, nb_s, 0, wi, wj, lane, a0, b0);
  mma_kstep(acc, a1, b1);
  interleave_kstep<NREAD, 2 * COPY_INSTS, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
}

// mma_stage_pipe for two Col tiles (the dW kernels' ring): fragment reads through per-stage
// opaque addresses (ColBases, see col_bases), those of the next stage formed after the barrier
// from its slots na_s / nb_s and carried into the next call through ca / cb.
template <typename Bar, typename Dma>
__device__ __forceinline__ void mma_stage_pipe_col(ColBases<WT_I>& ca, ColBases<WT_J>& cb,
                                                   const lds_u8* __restrict__ na_s,
                                                   const lds_u8* __restrict__ nb_s,
                                                   lds_u8* __restrict__ d1, lds_u8* __restrict__ d2,
                                                   f32x16 (&acc)[WT_I][WT_J], int wi, int wj,
                                                   int lane, bf16x8 (&a0)[WT_I],
                                                   bf16x8 (&b0)[WT_J], Bar&& bar, Dma&& dma) {
  constexpr int NREAD = 2 * (WT_I + WT_J);
  auto frags = [&](int ks, bf16x8 (&a)[WT_I], bf16x8 (&b)[WT_J]) {
#pragma unroll
    for (int i = 0; i < WT_I; ++i) a[i] = frag_col_at(ca.p1[i], ca.p2[i], ks);
#pragma unroll
    for (int j = 0; j < WT_J; ++j) b[j] = frag_col_at(cb.p1[j], cb.p2[j], ks);
  };
  bf16x8 a1[WT_I], b1[WT_J];
  frags(1, a1, b1);
  mma_kstep(acc, a0, b0);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  frags(2, a0, b0);
  mma_kstep(acc, a1, b1);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  frags(3, a1, b1);
  mma_kstep(acc, a0, b0);
  interleave_kstep<NREAD, 0, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
  bar();
  __builtin_amdgcn_sched_barrier(0);
  dma(d1, d2);
  col_bases(na_s, wi * (32 * WT_I), lane, ca);
  col_bases(nb_s, wj * (32 * WT_J), lane, cb);
  frags(0, a0, b0);
  mma_kstep(acc, a1, b1);
  interleave_kstep<NREAD, 2 * COPY_INSTS, 0, 0>();
  __builtin_amdgcn_sched_barrier(0);
}

// Full stages 0 .. nfull-1 of two dense operands through two stage slots of 64 KB, the barrier between
// stages moved before each stage's last k-step (mma_stage_pipe): right after it the copies of stage
// kt+2 go into stage kt's slot, a full stage ahead of the barrier that completes them. Past the last
// stage the copies repeat stage nfull-1 into the idle slot, so every stage issues the same
// instructions. copy(kt, slot) issues the copies of stage kt; on return the LDS is free.
template <bool A_COL, bool B_COL, typename Copy>
__device__ __forceinline__ void dense_stages(lds_u8* lbase, int nfull, f32x16 (&acc)[WT_I][WT_J],
                                             int wi, int wj, int lane, Copy&& copy_stage) {
  auto slot = [&](int kt) { return lbase + (kt & 1) * 2 * TILE_BYTES; };
  auto copy = [&](int kt, lds_u8* as) {
    const int ks = kt < nfull ? kt : nfull - 1;
    copy_stage(ks, as, as + TILE_BYTES);
  };
  bf16x8 a0[WT_I], b0[WT_J];
  if (nfull > 0) {
    copy(0, slot(0));
    copy(1, slot(1));
    wait_vmcnt<2 * COPY_INSTS>();  // stage 0 has landed; stage 1 may be in flight
    stage_barrier();
    load_frags<A_COL, B_COL>(slot(0), slot(0) + TILE_BYTES, 0, wi, wj, lane, a0, b0);
  }
  for (int kt = 0; kt < nfull; ++kt) {
    lds_u8* const cs = slot(kt);
    const lds_u8* const ns = slot(kt + 1);
    mma_stage_pipe<A_COL, B_COL>(
        cs, cs + TILE_BYTES, ns, ns + TILE_BYTES, cs, cs + TILE_BYTES, acc, wi, wj, lane, a0, b0,
        [&] {
          wait_vmcnt<0>();  // this wave's copies of stage kt+1
          stage_barrier();
        },
        [&](lds_u8* da, lds_u8*) { copy(kt + 2, da); });
  }
  __builtin_amdgcn_s_waitcnt(0);  // the repeated copies past the last stage
  __syncthreads();
}

// Full stages of two Col operands (32 KB each per stage) through a ring of 5 operand slots. The
// operand that changes between consecutive tiles of the walk misses L2 more often and leads: it is
// copied two stages ahead, the other one stage ahead. Copy c of the sequence lead_0, other_0, lead_1,
// other_1, ... goes to slot c % 5. Stages run as mma_stage_pipe_col: the barrier before stage s's
// last k-step frees the slots of lead_s and other_s, and the two copies issued right after it,
// other_s+2 then lead_s+3, go to exactly those slots (c = 2s+5 and 2s+6); the slots of lead_s+1,
// other_s+1 and lead_s+2 stay live. Past the last stage the copies repeat stage nfull-1 into the
// free slots, so every stage issues the same instructions. copy(a, kt, dst) issues the copies of
// operand A (else B) of stage kt. The caller waits for the repeated copies.
template <bool A_LEADS, typename Copy>
__device__ __forceinline__ void col_stages(lds_u8* lbase, int nfull, f32x16 (&acc)[WT_I][WT_J],
                                           int wi, int wj, int lane, Copy&& copy_stage) {
  auto slot = [&](bool is_a, int kt) -> lds_u8* {
    return lbase + ((2 * kt + (is_a == A_LEADS ? 0 : 1)) % RING_SLOTS) * TILE_BYTES;
  };
  auto copy = [&](bool a, int kt, lds_u8* dst) {
    const int ks = kt < nfull ? kt : nfull - 1;
    copy_stage(a, ks, dst);
  };
  ColBases<WT_I> ca;
  ColBases<WT_J> cb;
  bf16x8 a0[WT_I], b0[WT_J];
  if (nfull > 0) {
    copy(A_LEADS, 0, slot(A_LEADS, 0));
    copy(!A_LEADS, 0, slot(!A_LEADS, 0));
    __builtin_amdgcn_sched_barrier(0);
    copy(A_LEADS, 1, slot(A_LEADS, 1));
    copy(!A_LEADS, 1, slot(!A_LEADS, 1));
    copy(A_LEADS, 2, slot(A_LEADS, 2));
    wait_vmcnt<3 * COPY_INSTS>();  // stage 0 has landed; lead_1, other_1, lead_2 may not
    stage_barrier();
    col_bases(slot(true, 0), wi * (32 * WT_I), lane, ca);
    col_bases(slot(false, 0), wj * (32 * WT_J), lane, cb);
#pragma unroll
    for (int i = 0; i < WT_I; ++i) a0[i] = frag_col_at(ca.p1[i], ca.p2[i], 0);
#pragma unroll
    for (int j = 0; j < WT_J; ++j) b0[j] = frag_col_at(cb.p1[j], cb.p2[j], 0);
  }
  for (int kt = 0; kt < nfull; ++kt) {
    mma_stage_pipe_col(
        ca, cb, slot(true, kt + 1), slot(false, kt + 1), slot(A_LEADS, kt), slot(!A_LEADS, kt), acc,
        wi, wj, lane, a0, b0,
        [&] {
          wait_vmcnt<COPY_INSTS>();  // stage kt+1 has landed; lead_kt+2 may not
          stage_barrier();
        },
        [&](lds_u8* other_next2, lds_u8* lead_next3) {
          copy(!A_LEADS, kt + 2, other_next2);
          __builtin_amdgcn_sched_barrier(0);  // other_kt+2 is issued before lead_kt+3
          copy(A_LEADS, kt + 3, lead_next3);
        });
  }
}

}  // namespace g2
}  // namespace plz

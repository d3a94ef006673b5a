// Losses over a large vocabulary from hidden states and head weights, no logits kept beyond a call:
//
//   z = x W^T                               x bf16 [N, H], W bf16 [V, H], fp32 sums
//   cross entropy   loss_n = log sum_v exp z_nv - z_n,label
//                   dz_nv  = softmax(z_n)_v - [v = label_n]
//   distillation    p = softmax(z_teacher / T), q = softmax(z / T)
//                   loss_n = sum_v p_v (log p_v - log q_v),   dz_nv = (q_v - p_v) / T
//   dx = dz W,  dW = dz^T x
//
// The rows that take part (a label other than ignore_index; a mask that is set) are packed first, so
// the others cost nothing and nothing of them, a NaN neither, reaches a sum. Every tile of logits is
// 256 words x 256 rows of the 256x256 core with the words along the accumulator registers: a lane
// holds 64 words of a row, so a row's maximum and sum of exponentials are register work, one exchange
// with the other half wave and one through LDS. The forward keeps those statistics of each tile
// (8 bytes a row and 256 words) and joins them in a second kernel, in 64 bits. The backward computes
// the logits of a piece of the vocabulary again, now with the rows' normalisers at hand, rounds dz to
// bf16 into a workspace dz^T [words, rows] of at most kPieceBytes, and multiplies it with x (dW of the
// piece) and with W (dx, its fp32 parts summed over pieces and splits in a fixed order). What rounding
// the greatest dz of each row leaves, of few rows every dz, is added to both products. The scale of a
// mean and of its gradient is applied to the fp32 sums, not to dz: it would be rounded with it.
//
// A sum or mean whose logits are few enough has its gradients with the forward (step): the tiles keep
// what dz is made of and a memory-bound pass makes dz of it once the normalisers are known, instead of
// computing the logits again. A cross entropy keeps its exponentials relative to the tile's maximum, in
// fp16; a distillation keeps both sides' logits in fp32, since dz is the difference of probabilities
// that may be close. Other distillations do the same with a piece of the vocabulary at a time.
#include <algorithm>

#include "plz_gemm2_dense.cuh"
#include "palettize_hip.h"

namespace plz {
namespace voc {

using namespace g2;

constexpr float kLog2e = 1.4426950408889634f;
constexpr size_t kPieceBytes = (size_t)1 << 30;  // of dz, and of the logits of a piece
constexpr size_t kKeepBytes = (size_t)8 << 30;   // of what a step keeps
// Exponentials relative to the tile's maximum are kept in fp16 times this: the greatest is then 2^15, and
// those from 2^-29 on are normal, off by 2^-11 of their own value, an eighth of what rounding dz, or the
// gradient, to bf16 may be off (as they are, from 2^-14 on: beside a word of probability 1 those of 10^-6
// were off by 3%). Below, by 2^-40 of the tile's maximum. (The label's dz comes from its logit in fp32.)
constexpr float kKeptScale = 32768.f;
constexpr size_t kLdsLogits = 2 * 2 * TILE_BYTES + 8192;  // two stages and the statistics' exchange
constexpr size_t kLdsRing = RING_SLOTS * TILE_BYTES;
constexpr int kPackMost = 64;  // rows of a packing workgroup, at most
// Where no more rows than these take part, dz is two bf16, the second the first's rounding: row n's lies kTwo
// rows behind it, in the half of the 256-row tile that would be empty. The products' fp32 sums add both, so
// that rounding dz does not show: in one bf16 it is off by as much as the gradient's own rounding, more or
// less by the rows' chance where few are summed (a distillation's gradients of 16 rows 1.3 to 1.9 times the
// error of those from dz in fp32, of 900 rows 1.4 to 1.5). dx's products are the same, dW's stages twice as
// many, each reading the rows of x once more.
constexpr int kTwo = 128;
__host__ __device__ constexpr bool two_parts(int64_t rows) { return rows <= kTwo; }

enum { KEY_NONE = 0, KEY_INT64 = 1, KEY_INT32 = 2, KEY_MASK = 3 };
// What a launch over tiles of logits leaves: their statistics, the gradients of the logits, the
// statistics and the exponentials in fp16, or the statistics and the logits in fp32 (of both sides)
enum { CE_STATS, CE_GRAD, CE_KEEP, Z_KEEP };

// ---- rows that take part --------------------------------------------------------------------------
struct Meta {
  int rows;     // how many take part
  int done;     // workgroups that have written their rows' losses
  float alpha;  // backward: the scale of the gradients that every row shares
  int z;        // backward: splits of dx's reduction over the words of a piece
};
struct PackArgs {
  const void* key;  // labels or mask
  int kind;
  int per;  // rows of a workgroup, a divisor of TILE
  int64_t ignore, V, N;
  const uint16_t* x[2];  // student, teacher
  uint16_t* xp[2];
  int64_t H[2];
  Meta* meta;
  int32_t* src;    // [Np] the row of a packed row
  int32_t* lab;    // [Np] labels, -1: no word
  float* zero[5];  // forward: outputs that are 0 for rows that take no part (or NULL)
  uint16_t* grad_x;  // gradients of x, which are 0 for them (or NULL)
  // backward
  const float *lse_in[2], *rest_in[2];
  float *lse[2], *rest[2];  // [Np]
  const float* grad;
  int reduction;  // PLZ_REDUCE_*
  float* g;       // [Np], reduction none
  float inv_t;
  int64_t words, z_floats;  // of a piece, and of dx's parts: 0 without dx
  int cus;
};

// Modelled time of dx over the words of a piece for `rows` rows in z splits: whole waves of workgroups
// at 1.9 us a stage and 4 stages of prologue and epilogue, the fp32 parts (8 bytes an element and split
// written and read) at half of 5 TB/s; infinite for splits of less than 3 stages or parts of more than
// `floats`.
__host__ __device__ inline float dx_us(int z, int64_t rows, int64_t words, int64_t H, int C, int64_t floats) {
  const int tiles = (int)((rows + TILE - 1) / TILE * ((H + TILE - 1) / TILE));
  const int len = (int)((words + z * BK - 1) / (z * BK));
  if (z > 1 && (len < 3 || z * ((rows + 3) / 4 * 4) * H > floats)) return INFINITY;
  const float part = 16.f * (float)rows * (float)H / 5.0e6f;
  return (float)(((int64_t)tiles * z + C - 1) / C) * ((float)len + 4.f) * 1.9f + (float)z * part;
}
constexpr int kMaxSplits = 64;
inline int dx_splits(int64_t rows, int64_t words, int64_t H, int C) {
  int best = 1;
  for (int z = 2; z <= kMaxSplits; ++z)
    if (dx_us(z, rows, words, H, C, INT64_MAX) < dx_us(best, rows, words, H, C, INT64_MAX)) best = z;
  return best;
}

__device__ __forceinline__ bool takes_part(const PackArgs& a, int64_t r) {
  switch (a.kind) {
    case KEY_INT64: return reinterpret_cast<const int64_t*>(a.key)[r] != a.ignore;
    case KEY_INT32: return reinterpret_cast<const int32_t*>(a.key)[r] != a.ignore;
    case KEY_MASK: return reinterpret_cast<const uint8_t*>(a.key)[r] != 0;
    default: return true;
  }
}

__device__ __forceinline__ int label_of(const PackArgs& a, int64_t r) {
  if (a.kind != KEY_INT64 && a.kind != KEY_INT32) return -1;
  const int64_t l = a.kind == KEY_INT64 ? reinterpret_cast<const int64_t*>(a.key)[r]
                                        : reinterpret_cast<const int32_t*>(a.key)[r];
  return l >= 0 && l < a.V ? (int)l : -1;
}

// By one wave: a split of dx a lane, the fastest of the model
__device__ __forceinline__ void write_meta(const PackArgs& a, int rows) {
  const int lane = threadIdx.x & 63;
  int z = lane + 1;
  float us = a.z_floats ? dx_us(z, rows, a.words, a.H[0], a.cus, a.z_floats) : 0.f;
#pragma unroll
  for (int o = 1; o < kMaxSplits; o <<= 1) {
    const float u = __shfl_xor(us, o);
    const int v = __shfl_xor(z, o);
    if (u < us || (u == us && v < z)) {
      us = u;
      z = v;
    }
  }
  if (lane == 0) {
    float alpha = a.inv_t;
    if (a.grad && a.reduction != PLZ_REDUCE_NONE) alpha *= a.grad[0];
    if (a.reduction == PLZ_REDUCE_MEAN && rows > 0) alpha /= (float)rows;
    *a.meta = Meta{rows, 0, alpha, z};
  }
}

// A workgroup packs a.per rows behind all that take part before them, which it counts itself (the keys
// of 16384 rows are 128 KB in the L2s). Behind the rows' workgroups come TILE / a.per that clear the
// packed rows up to the next whole tile: dW's reduction runs over those of the last stage, and
// multiplying zeros takes less power than what was there. The first of them writes meta.
__global__ __launch_bounds__(256) void pack_kernel(const PackArgs a) {
  __shared__ int red[4];
  __shared__ int at[kPackMost];
  const int64_t r0 = min((int64_t)blockIdx.x * a.per, a.N);
  const int pad = (int)(blockIdx.x - (a.N + a.per - 1) / a.per);  // < 0: rows
  int before = (int)r0;
  if (a.kind != KEY_NONE) {
    int c = 0;
#pragma unroll 4
    for (int64_t r = threadIdx.x; r < r0; r += 256) c += takes_part(a, r) ? 1 : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    before = red[0] + red[1] + red[2] + red[3];
  }
  if (pad >= 0) {
    const int rows = before, first = rows + pad * a.per;
    const int end = min(first + a.per, (rows + TILE - 1) / TILE * TILE);
    for (int k = 0; k < 2; ++k) {
      if (!a.x[k] || first >= end) continue;
      const int64_t c8 = a.H[k] / 8;
      uint4* d = reinterpret_cast<uint4*>(a.xp[k]) + first * c8;
      for (int64_t c = threadIdx.x; c < (end - first) * c8; c += 256) d[c] = make_uint4(0, 0, 0, 0);
    }
    if (pad == 0 && threadIdx.x < 64) write_meta(a, rows);
    return;
  }
  const int n = (int)min((int64_t)a.per, a.N - r0);
  if (threadIdx.x < 64) {
    const int i = threadIdx.x;
    const bool on = i < n && takes_part(a, r0 + i);
    const uint64_t all = __ballot(on);
    if (i < a.per) at[i] = on ? before + __popcll(all & ((1ull << i) - 1)) : -1;
    if (i < n) {
      const int64_t r = r0 + i;
      const int p = at[i];
      if (on) {
        a.src[p] = (int)r;
        if (a.kind == KEY_INT64 || a.kind == KEY_INT32) a.lab[p] = label_of(a, r);
        for (int k = 0; k < 2; ++k)
          if (a.lse_in[k]) {
            a.lse[k][p] = a.lse_in[k][r];
            a.rest[k][p] = a.rest_in[k][r];
          }
        if (a.g) a.g[p] = a.grad[r];
      } else {
        for (int k = 0; k < 5; ++k)
          if (a.zero[k]) a.zero[k][r] = 0.f;
      }
    }
  }
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    if (!a.x[k]) continue;
    const int64_t H = a.H[k];
    const int c8 = (int)(H / 8);
    const uint4* from = reinterpret_cast<const uint4*>(a.x[k] + r0 * H);
    uint4* to = reinterpret_cast<uint4*>(a.xp[k]);
#pragma unroll 4
    for (int j = threadIdx.x; j < n * c8; j += 256) {
      const int i = j / c8, p = at[i];
      if (p >= 0) to[(int64_t)p * c8 + (j - i * c8)] = from[j];
      else if (k == 0 && a.grad_x) reinterpret_cast<uint4*>(a.grad_x + r0 * H)[j] = make_uint4(0, 0, 0, 0);
    }
  }
}

// ---- tiles of logits ------------------------------------------------------------------------------
struct LogitArgs {
  const uint16_t* w[2];  // student, teacher
  const uint16_t* x[2];  // packed rows [Np, H]
  int64_t H[2];
  int sides;
  int64_t v0, v1;  // the words of this launch
  int64_t Np;
  const Meta* meta;
  const int32_t* lab;
  const float *lse, *rest;  // [Np]
  const float* g;    // [Np] or NULL
  float inv_t;
  float* stats;  // [tile of words][planes][Np]: maximum and sum of the student, of the teacher
  int planes, tile0;  // tile0: the first of this launch
  float* zlab;        // [Np]
  // [tile of rows][word of the piece, whole tiles][256 rows]: dz, or the exponentials kept for it
  uint16_t* dzt;
  int64_t words;  // of a piece, whole tiles
  float* low;     // CE_GRAD: [Np] what rounding the labels' dz left (or NULL)
  float* kept;    // logits over T, [side][tile of the launch][256 * 256] in the accumulators' order
  int64_t kept_side;  // floats of a side
};

// exp(d) as 2^(d log2 e): d is formed first, so its rounding and the product's are relative to the
// distance from the maximum (or the normaliser), which is small wherever the exponential counts
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// What rounding d to bf16 (high) leaves, and that in bf16
__device__ __forceinline__ float left_of(float d, uint16_t high) {
  const float l = d - bf2f(high);
  return fabsf(l) < INFINITY ? l : 0.f;  // else the first part is infinite or NaN
}
__device__ __forceinline__ uint16_t low_part(float d, uint16_t high) { return (uint16_t)f2bf(left_of(d, high)); }

// two exponentials as a step keeps them
__device__ __forceinline__ uint32_t kept2(float a, float b) {
  return f2h(a * kKeptScale) | (f2h(b * kKeptScale) << 16);
}

// The statistics of a set of words: the maximum and the sum of exponentials relative to it.
struct Stat {
  float m, s;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  const float M = fmaxf(a.m, b.m);
  // no word above -inf on either side: nothing to scale (inf - inf is not 0)
  if (M == -INFINITY) return Stat{M, a.s + b.s};
  return Stat{M, a.s * exp_of(a.m - M) + b.s * exp_of(b.m - M)};
}
// A set of words' sum of the teacher's exponentials times ((teacher - its maximum) - (student - its
// maximum)), relative to the maxima Mt and Ms of more words. (Without weight there it is nothing, also
// where the student's logits were -inf and it was infinite.)
__device__ __forceinline__ float cross_of(float c, const Stat& student, const Stat& teacher, float Ms, float Mt) {
  const float f = teacher.m == -INFINITY ? 0.f : exp_of(teacher.m - Mt);
  if (f == 0.f) return 0.f;
  const float moved = student.m == -INFINITY ? 0.f : student.m - Ms;
  return f * (c + teacher.s * ((teacher.m - Mt) - moved));
}
// over lanes l and l ^ 32
__device__ __forceinline__ float swap32_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap32_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16 bytes to a uniform address and a lane's 32-bit offset. Not a buffer store: behind one whose scalar
// offset is a register, gfx950 still reads the data while the next instruction may write it again, and
// the compiler leaves no gap (values of the last lanes of every 16 were those of the next block). The
// empty asm statement keeps the address in scalar registers: folded with the lanes' offsets, 32 stores
// would take 32 pairs of vector registers.
__device__ __forceinline__ void store16(void* base, uint32_t off, u32x4 v) {
  typedef __attribute__((address_space(1))) char gchar;
  typedef __attribute__((address_space(1))) u32x4 gu32x4;
  uint64_t p = reinterpret_cast<uint64_t>(base);
  asm volatile("" : "+s"(p));
  __builtin_nontemporal_store(v, reinterpret_cast<gu32x4*>(reinterpret_cast<gchar*>(p) + off));
}

typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) uint16_t lds_u16t;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

// acc[word, row] of words i0 .. and rows j0 ..; words from v1 on repeat the last one
__device__ __forceinline__ void logits_tile(lds_u8* lbase, const uint16_t* w, const uint16_t* x,
                                            int64_t H, int64_t i0, int64_t v1, int64_t j0,
                                            f32x16 (&acc)[WT_I][WT_J], int wi, int wj, int lane) {
#pragma unroll
  for (int i = 0; i < WT_I; ++i)
#pragma unroll
    for (int j = 0; j < WT_J; ++j) acc[i][j] = f32x16{};
  const int64_t nw = min((int64_t)TILE, v1 - i0);
  const uint16_t* wt = w + i0 * H;
  const uint16_t* xt = x + j0 * H;
  const TileDma dA = row_tile_dma(wt, H, 0, nw), dB = row_tile_dma(xt, H, 0, TILE);
  const int nfull = (int)(H / BK);
  dense_stages<false, false>(lbase, nfull, acc, wi, wj, lane, [&](int kt, lds_u8* As, lds_u8* Bs) {
    tile_copy(As, dA, (uint32_t)(kt * BK * 2));
    tile_copy(Bs, dB, (uint32_t)(kt * BK * 2));
  });
  if (H % BK) {
    copy_row_tile_masked((uint4*)lbase, wt, H, 0, nw, (int64_t)nfull * BK, H);
    copy_row_tile_masked((uint4*)(lbase + TILE_BYTES), xt, H, 0, TILE, (int64_t)nfull * BK, H);
    __syncthreads();
    mma_stage_sync<false, false>(lbase, lbase + TILE_BYTES, acc, wi, wj, lane,
                                 (int)((H % BK + 15) / 16));
    __syncthreads();
  }
}

// The two operands of a tile of logits: a lane's offsets of the copies of a stage, 64 rows apart, and the
// bit that takes its chunk of a last stage that is not whole out of the buffer. What is out of the
// buffer, rows past the last too, is zero in LDS: the hardware checks the range.
struct Operands {
  BufRsrc w, x;
  uint32_t off[COPY_INSTS], past;
  int stages;
};
__device__ __forceinline__ Operands operands_of(const uint16_t* w, const uint16_t* x, int64_t H, int64_t nw) {
  Operands o;
  o.w = make_rsrc(w, (uint32_t)(nw * H * 2));
  o.x = make_rsrc(x, (uint32_t)(TILE * H * 2));
  const int row = threadIdx.x >> 3, c = (threadIdx.x & 7) ^ row_swz(row);  // of every 64 rows the same
#pragma unroll
  for (int it = 0; it < COPY_INSTS; ++it) o.off[it] = (uint32_t)(((64 * it + row) * H + c * 8) * 2);
  o.stages = (int)((H + BK - 1) / BK);
  o.past = H % BK && c * 8 >= H % BK ? kBufOob : 0;
  return o;
}
__device__ __forceinline__ void copy_operands(const Operands& o, int kt, lds_u8* as) {
  const uint32_t past = kt == o.stages - 1 ? o.past : 0;
  TileDma d;
#pragma unroll
  for (int it = 0; it < COPY_INSTS; ++it) d.off[it] = o.off[it] | past;
  d.r = o.w;
  tile_copy(as, d, (uint32_t)(kt * BK * 2));
  d.r = o.x;
  tile_copy(as + TILE_BYTES, d, (uint32_t)(kt * BK * 2));
}

// STREAM: the stages of all the workgroup's tiles follow each other through the two slots without a
// break: the last two stages of a tile copy the first two of the next one, which are on their way
// during the epilogue. For two stages at least.
template <int MODE, bool STREAM>
__global__ __launch_bounds__(NTHR) void logits_kernel(const LogitArgs a) {
  extern __shared__ uint4 smem[];
  lds_u8* lbase = (lds_u8*)smem;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave / WAVES_J, wj = wave % WAVES_J;
  const int rows = a.meta->rows;
  const bool two = two_parts(rows);
  const int tiles_i = (int)((a.v1 - a.v0 + TILE - 1) / TILE), tiles_j = (rows + TILE - 1) / TILE;
  const int64_t total = (int64_t)tiles_i * tiles_j;
  // Every XCD walks a run of its own, four tiles of words at a time over the rows, of one side after the
  // other. Both sides' logits are stored: with 4, 8 or 16 tiles of rows its 32 workgroups would then start
  // and store their tiles in step, so there it is six. With four and with six, ms of both sides' logits and
  // the pass over them:  151936 x 2560  151936 x 1024  50257 x 1600  32000 x 2560  128256 x 4096
  //   1024 rows           1.80  1.75     1.04  0.97     0.440  0.438  0.360  0.357   2.12   2.13
  //   2048                3.53  3.36     2.08  1.91     0.846  0.814  0.721  0.710   4.07   4.08
  //   4096                6.69  6.63     3.90  3.78     1.61   1.56   1.41   1.39    7.91   7.88
  //   1280                2.12  2.13     1.24  1.25     0.533  0.532  0.448  0.453   2.59   2.60
  //   1792                2.88  2.94     1.64  1.70     0.711  0.725  0.619  0.624   3.52   3.63
  // (2560 rows would be 0 to 4% faster with six, and a cross entropy's 4096 are not: 2.62 and 2.63.)
  const int group = MODE == Z_KEEP && tiles_j % 4 == 0 ? 6 : 4;
  const int xcd = blockIdx.x % 8, step = gridDim.x / 8;
  const int64_t begin = total * xcd / 8, run = total * (xcd + 1) / 8 - begin;
  struct Tile {
    int side, tile_i, tile_j;
    int64_t i0, j0;
  };
  auto tile_at = [&](int64_t at) {
    Tile t;
    t.side = MODE == Z_KEEP && at >= run ? 1 : 0;
    tile_coords(group, tiles_i, tiles_j, (int)(begin + at - t.side * run), t.tile_i, t.tile_j);
    t.i0 = a.v0 + (int64_t)t.tile_i * TILE;
    t.j0 = (int64_t)t.tile_j * TILE;
    return t;
  };
  const int64_t ends = run * a.sides;
  int64_t at = blockIdx.x / 8;
  if (at >= ends) return;
  Tile t = tile_at(at);
  Operands o;
  auto operands = [&](const Tile& t) {
    const int64_t H = a.H[t.side];
    o = operands_of(a.w[t.side] + t.i0 * H, a.x[t.side] + t.j0 * H, H, min((int64_t)TILE, a.v1 - t.i0));
  };
  int slot = 0;  // of the next stage
  bf16x8 fa[WT_I], fb[WT_J];
  auto slot_at = [&](int k) { return lbase + (k & 1) * 2 * TILE_BYTES; };
  if constexpr (STREAM) {
    operands(t);
    copy_operands(o, 0, slot_at(0));
    copy_operands(o, 1, slot_at(1));
    wait_vmcnt<2 * COPY_INSTS>();  // stage 0 has landed; stage 1 may be in flight
    stage_barrier();
    load_frags<false, false>(slot_at(0), slot_at(0) + TILE_BYTES, 0, wi, wj, lane, fa, fb);
  }
  for (;;) {
    const int side = t.side, tile_i = t.tile_i, tile_j = t.tile_j;
    const int64_t i0 = t.i0, j0 = t.j0;
    f32x16 acc[WT_I][WT_J];
    const int64_t next = at + step;
    if constexpr (STREAM) {
#pragma unroll
      for (int i = 0; i < WT_I; ++i)
#pragma unroll
        for (int j = 0; j < WT_J; ++j) acc[i][j] = f32x16{};
      const int n = o.stages;
      auto stages = [&](int from, int to, int skip) {
        for (int kt = from; kt < to; ++kt, ++slot) {
          lds_u8* const cs = slot_at(slot);
          const lds_u8* const ns = slot_at(slot + 1);
          mma_stage_pipe<false, false>(
              cs, cs + TILE_BYTES, ns, ns + TILE_BYTES, cs, cs + TILE_BYTES, acc, wi, wj, lane, fa, fb,
              [&] {
                wait_vmcnt<0>();  // this wave's copies of the next stage
                stage_barrier();
              },
              [&](lds_u8* da, lds_u8*) { copy_operands(o, kt + 2 - skip, da); });
        }
      };
      stages(0, n - 2, 0);
      // behind the last tile its first stages are copied once more, and not used
      if (next < ends) t = tile_at(next);
      operands(t);
      stages(n - 2, n, n);
    } else {
      logits_tile(lbase, a.w[side], a.x[side], a.H[side], i0, a.v1, j0, acc, wi, wj, lane);
      if (next < ends) t = tile_at(next);
    }

    // This lane's word of block ti and register e is vl + 32 ti + 8 (e / 4) + e % 4, from the tile's
    // first one; of the tile's words, nw exist.
    const int vl = wi * (32 * WT_I) + 4 * (lane >> 5);
    const int nw = (int)min((int64_t)TILE, a.v1 - i0);
#pragma unroll
    for (int tj = 0; tj < WT_J; ++tj) {
      const int nl = wj * (32 * WT_J) + 32 * tj + (lane & 31);
      const int64_t n = j0 + nl;
      const bool live = n < rows;
      // the label's logit, in the one lane that holds it: false elsewhere. lv: the label from vl
      float zl = 0.f;
      auto holds = [&](int l) {
        const int lv = l - vl;
        // its registers are those of words 0..3 of every 8
        const bool mine = lv >= 0 && lv < 32 * WT_I && (lv & 4) == 0;
        if (__ballot(mine) == 0) return false;
#pragma unroll
        for (int ti = 0; ti < WT_I; ++ti) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            zl = lv == 32 * ti + 8 * (e >> 2) + (e & 3) ? acc[ti][tj][e] : zl;
          __builtin_amdgcn_sched_barrier(0);
        }
        return mine;
      };
      if constexpr (MODE != CE_GRAD) {
        if constexpr (MODE == Z_KEEP) {
          float* const kept = a.kept + side * a.kept_side +
                              ((int64_t)tile_j * tiles_i + tile_i) * (TILE * TILE);
#pragma unroll
          for (int ti = 0; ti < WT_I; ++ti) {
            acc[ti][tj] *= a.inv_t;
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
              const f32x4 v = {acc[ti][tj][4 * e4], acc[ti][tj][4 * e4 + 1], acc[ti][tj][4 * e4 + 2],
                               acc[ti][tj][4 * e4 + 3]};
              store16(kept + ((ti * WT_J + tj) * 4 + e4) * NTHR * 4, threadIdx.x * 16,
                      __builtin_bit_cast(u32x4, v));
            }
          }
        } else {
          if (live && holds(a.lab[n] - (int)i0)) a.zlab[n] = zl;
        }
        if (nw < TILE) {  // words that do not exist
#pragma unroll
          for (int ti = 0; ti < WT_I; ++ti) {
            const int left = nw - vl - 32 * ti;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              acc[ti][tj][e] = 8 * (e >> 2) + (e & 3) < left ? acc[ti][tj][e] : -INFINITY;
          }
        }
        // the tile's maximum: of the lane, of both halves, of both waves of the column, which meet in
        // LDS behind the stages' slots
        float m = -INFINITY;
#pragma unroll
        for (int ti = 0; ti < WT_I; ++ti)
#pragma unroll
          for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[ti][tj][e]);
        m = swap32_max(m);
        lds_f32* ex = reinterpret_cast<lds_f32*>(lbase + 4 * TILE_BYTES) + wj * 256;
        ex[wi * 32 + (lane & 31)] = m;
        __syncthreads();
        m = fmaxf(ex[lane & 31], ex[32 + (lane & 31)]);
        const float m0 = m == -INFINITY ? 0.f : m;
        uint16_t* const exps =
            MODE == CE_KEEP ? a.dzt + ((int64_t)tile_j * a.words + (i0 - a.v0)) * TILE : nullptr;
        float sum = 0.f;
#pragma unroll
        for (int ti = 0; ti < WT_I; ++ti) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              p[e] = exp_of(acc[ti][tj][8 * h + e] - m0);
              sum += p[e];
            }
            if constexpr (MODE == CE_KEEP) {
              u32x4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = kept2(p[2 * e], p[2 * e + 1]);
              store16(exps + ti * 8192 + tj * 1024 + h * 512, wi * 65536 + wj * 4096 + lane * 16, v);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        sum = swap32_sum(sum);
        if (wi == 1 && lane < 32) ex[64 + lane] = sum;
        __syncthreads();
        if (wi == 0 && lane < 32 && live) {
          float* out = a.stats + ((int64_t)(a.tile0 + tile_i) * a.planes + 2 * side) * a.Np + n;
          out[0] = m;
          out[a.Np] = sum + ex[64 + lane];
        }
        __syncthreads();
      } else {
        // dz of this row's words, bf16, into the tile staged in LDS [word][row]
        const float lse = live ? a.lse[n] : 0.f, rest = live ? a.rest[n] : 0.f;
        float g = live && a.g ? a.g[n] : 1.f;
        int l = live ? a.lab[n] : 0;
        if (l < 0) g = __builtin_nanf("");  // no such word: nothing to learn from
        l -= (int)i0;
#pragma unroll
        for (int ti = 0; ti < WT_I; ++ti) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float d = live ? exp_of((acc[ti][tj][e] - lse) - rest) * g : 0.f;
            const uint16_t high = (uint16_t)f2bf(d);
            lds_u8* const at = lbase + (vl + 32 * ti + 8 * (e >> 2) + (e & 3)) * EPI_RS + nl * 2;
            if (!two) {
              *reinterpret_cast<lds_u16t*>(at) = high;
            } else if (nl < kTwo) {
              *reinterpret_cast<lds_u16t*>(at) = high;
              *reinterpret_cast<lds_u16t*>(at + kTwo * 2) = low_part(d, high);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (live && holds(l)) {
          const float d = expm1f((zl - lse) - rest) * g;
          const uint16_t high = (uint16_t)f2bf(d);
          *reinterpret_cast<lds_u16t*>(lbase + l * EPI_RS + nl * 2) = high;
          if (two) *reinterpret_cast<lds_u16t*>(lbase + l * EPI_RS + (nl + kTwo) * 2) = low_part(d, high);
          if (a.low) a.low[n] = left_of(d, high);
        }
      }
    }
    if constexpr (MODE == CE_GRAD) {
      __syncthreads();
      uint16_t* out = a.dzt + ((int64_t)tile_j * a.words + (i0 - a.v0)) * TILE;
#pragma unroll 4
      for (int it = 0; it < TILE * TILE / 8 / NTHR; ++it) {
        const int ch = it * NTHR + threadIdx.x;
        const int row = ch >> 5, c8 = (ch & 31) * 8;
        u32x4 v = *reinterpret_cast<const lds_u32x4*>(lbase + row * EPI_RS + c8 * 2);
        if (row >= nw) v = u32x4{0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(out + row * TILE + c8) = v;
      }
      __syncthreads();
    }
    at = next;
    if (at >= ends) break;
  }
  __builtin_amdgcn_s_waitcnt(0);  // the copies past the last tile
}

// ---- tiles of logits of few rows ------------------------------------------------------------------------
// 128 words x 32 NB rows by four waves of 32 words each, reduction stages of 64 through a ring of
// kFewSlots of the words' 16 KB and the rows' 4 NB KB: two workgroups a CU, each with several stages on
// their way, where the 256x256 tiles would leave CUs without work or multiply rows that do not exist.
// HBM-bound for up to 32 rows (W is read once, ~100 KB a CU in flight), by the LDS reads of five
// fragments for four MFMAs at 128. The statistics are those of 128 words.
constexpr int kFewWords = 128;
constexpr int kFewThreads = 256;
template <int NB>
constexpr int few_slots() { return NB == 1 ? 4 : NB == 2 ? 3 : 2; }
template <int NB>
constexpr int few_stage() { return (kFewWords + 32 * NB) * BK * 2; }

// acc[word, row] of the wave's 32 words and 32 NB rows of x, the copies' row i of 32 NB being
// row_of(i) (none, < 0: zeros); of the tile's 128 words, nw exist, of x's rows nx
template <int NB, typename Row>
__device__ __forceinline__ void few_tile(lds_u8* lbase, const uint16_t* w, const uint16_t* x, int64_t H,
                                         int nw, int nx, Row&& row_of, f32x16 (&acc)[NB], int wave,
                                         int lane) {
  constexpr int SLOTS = few_slots<NB>(), STAGE = few_stage<NB>(), COPIES = 4 + NB;
  // copies: a lane's chunk of 16 bytes of every 32 rows, swizzled as the core's row tiles
  const BufRsrc rw = make_rsrc(w, (uint32_t)(nw * H * 2)), rx = make_rsrc(x, (uint32_t)(nx * H * 2));
  uint32_t ow[4], ox[NB];
  const int row = threadIdx.x >> 3, ch = (threadIdx.x & 7) ^ row_swz(row);
#pragma unroll
  for (int i = 0; i < 4; ++i) ow[i] = (uint32_t)(((32 * i + row) * H + ch * 8) * 2);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int r = row_of(32 * i + row);
    ox[i] = r < 0 ? kBufOob : (uint32_t)((r * H + ch * 8) * 2);
  }
  // a last stage that is not whole: chunks past the width are out of the buffer and zero (Operands)
  const int nst = (int)((H + BK - 1) / BK);
  const uint32_t out = H % BK && ch * 8 >= H % BK ? kBufOob : 0;
  const int wbase = __builtin_amdgcn_readfirstlane(wave * 1024);
  auto copy = [&](int kt, int slot) {
    lds_u8* d = lbase + slot * STAGE + wbase;
    const uint32_t past = kt == nst - 1 ? out : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, d + i * 4096, 16, ow[i] | past, kt * (BK * 2), 0, 0);
#pragma unroll
    for (int i = 0; i < NB; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, d + (4 + i) * 4096, 16, ox[i] | past, kt * (BK * 2), 0, 0);
  };
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = f32x16{};
  // Stage kt is waited for with the SLOTS - 2 stages behind it still on their way; the barrier also
  // frees the slot of stage kt - 1, which stage kt + SLOTS - 1 goes to. Past the last stage the copies
  // repeat it, so that every stage waits for as many.
#pragma unroll
  for (int k = 0; k < SLOTS - 1; ++k) copy(min(k, nst - 1), k);
  int slot = 0;
  for (int kt = 0; kt < nst; ++kt) {
    wait_vmcnt<(SLOTS - 2) * COPIES>();
    stage_barrier();
    copy(min(kt + SLOTS - 1, nst - 1), slot == 0 ? SLOTS - 1 : slot - 1);
    __builtin_amdgcn_sched_barrier(0);
    const lds_u8* s = lbase + slot * STAGE;
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      const bf16x8 fa = frag_row((const uint4*)s, 32 * wave, ks, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            fa, frag_row((const uint4*)(s + 16384), 32 * i, ks, lane), acc[i], 0, 0, 0);
    }
    slot = slot == SLOTS - 1 ? 0 : slot + 1;
  }
  __builtin_amdgcn_s_waitcnt(0);  // the repeated copies past the last stage
  __syncthreads();
}

// The row of x that is the k-th of those that take part: bit k of the set ones of two masks of 64 rows
__device__ __forceinline__ int kth_row(uint64_t m0, uint64_t m1, int k) {
  const int c0 = __popcll(m0);
  uint64_t m = k < c0 ? m0 : m1;
  int at = k < c0 ? 0 : 64;
  k -= k < c0 ? 0 : c0;
  if (k >= __popcll(m)) return -1;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    const int c = __popcll(m & ((1ull << s) - 1));
    if (k >= c) {
      k -= c;
      m >>= s;
      at += s;
    }
  }
  return at;
}

// GATHER (up to 128 rows, x as it came, no dW): every wave finds the rows that take part from the
// keys itself and the copies pick them out, instead of a launch that packs them (losses alone of 17 rows of
// 32000 x 1024 23.2 -> 20.9 us a call, of 16 of 151936 x 2560 149 -> 142); one workgroup more leaves what
// the other kernels need.
template <int MODE, int NB, bool GATHER>
__global__ __launch_bounds__(kFewThreads) void few_kernel(const LogitArgs a, const PackArgs k) {
  extern __shared__ uint4 smem[];
  lds_u8* lbase = (lds_u8*)smem;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t m0 = 0, m1 = 0;
  if constexpr (GATHER) {
    m0 = __ballot(lane < k.N && takes_part(k, lane));
    m1 = __ballot(64 + lane < k.N && takes_part(k, 64 + lane));
  }
  const int rows = GATHER ? __popcll(m0) + __popcll(m1) : a.meta->rows;
  if (GATHER && blockIdx.x == 0) {
    const int r = threadIdx.x;
    if (r < 64) write_meta(k, rows);
    if (r < k.N) {
      const uint64_t m = r < 64 ? m0 : m1;
      if (m >> (r & 63) & 1) {
        const int p = __popcll(m & ((1ull << (r & 63)) - 1)) + (r < 64 ? 0 : __popcll(m0));
        k.src[p] = r;
        k.lab[p] = label_of(k, r);
      } else {
#pragma unroll
        for (int z = 0; z < 5; ++z)
          if (k.zero[z]) k.zero[z][r] = 0.f;
      }
    }
    if (k.grad_x && rows < k.N) {
      const int c8 = (int)(k.H[0] / 8);
      for (int i = 0; i < (int)k.N; ++i) {
        if ((i < 64 ? m0 >> i : m1 >> (i - 64)) & 1) continue;
        uint4* d = reinterpret_cast<uint4*>(k.grad_x) + (int64_t)i * c8;
        for (int c = threadIdx.x; c < c8; c += kFewThreads) d[c] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  const int tiles_i = (int)((a.v1 - a.v0 + kFewWords - 1) / kFewWords);
  const int tiles_j = (rows + 32 * NB - 1) / (32 * NB);
  const int total = tiles_i * tiles_j;
  int at = (int)blockIdx.x - (GATHER ? 1 : 0), side = 0;
  if (MODE == Z_KEEP && at >= total) {
    at -= total;
    side = 1;
  }
  if (at >= total || (side == 1 && a.sides < 2)) return;
  // the rows' tiles of a tile of words on one XCD, after each other
  const int xcd = at % 8, q8 = total / 8, r8 = total % 8;
  const int item = xcd * q8 + (xcd < r8 ? xcd : r8) + at / 8;
  const int tile_i = item / tiles_j, tile_j = item % tiles_j;
  const int64_t i0 = a.v0 + (int64_t)tile_i * kFewWords, j0 = (int64_t)tile_j * (32 * NB), H = a.H[side];
  const int nw = (int)min((int64_t)kFewWords, a.v1 - i0);
  f32x16 acc[NB];
  int lab[NB];  // labels of the lane's rows
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int n = 32 * i + (lane & 31);
    lab[i] = -1;
    if (MODE != Z_KEEP && j0 + n < rows)
      lab[i] = GATHER ? label_of(k, kth_row(m0, m1, n)) : a.lab[j0 + n];
  }
  if constexpr (GATHER)
    few_tile<NB>(lbase, a.w[side] + i0 * H, a.x[side], H, nw, (int)k.N,
                 [&](int i) { return kth_row(m0, m1, i); }, acc, wave, lane);
  else
    few_tile<NB>(lbase, a.w[side] + i0 * H, a.x[side] + j0 * H, H, nw, 32 * NB,
                 [](int i) { return i; }, acc, wave, lane);

  // The wave's 32 words of the panel's block, 16 a lane: word vl + 8 (e / 4) + e % 4 of the tile.
  const int vl = 32 * wave + 4 * (lane >> 5);
  const int64_t rel = i0 - a.v0;  // within the launch
  const int block = (int)(rel % TILE) / 32 + wave, wi = block >> 2, ti = block & 3;
  lds_f32* ex = reinterpret_cast<lds_f32*>(lbase);
  float m[NB], sum[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int64_t n = j0 + 32 * i + (lane & 31);
    const int nb = (int)(n % TILE) / 32;
    if constexpr (MODE == Z_KEEP) {
      const int tiles256 = (int)((a.v1 - a.v0 + TILE - 1) / TILE);
      float* const kept = a.kept + side * a.kept_side +
                          ((j0 + 32 * i) / TILE * tiles256 + rel / TILE) * (TILE * TILE);
      acc[i] *= a.inv_t;
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const f32x4 v = {acc[i][4 * e4], acc[i][4 * e4 + 1], acc[i][4 * e4 + 2], acc[i][4 * e4 + 3]};
        *reinterpret_cast<f32x4*>(kept + ((ti * WT_J + (nb & 1)) * 4 + e4) * NTHR * 4 +
                                  ((wi * WAVES_J + (nb >> 1)) * 64 + lane) * 4) = v;
      }
    } else if (n < rows) {
      const int lv = lab[i] - (int)i0 - vl;
      if (lv >= 0 && lv < 32 && (lv & 4) == 0) {
        float zl = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) zl = lv == 8 * (e >> 2) + (e & 3) ? acc[i][e] : zl;
        a.zlab[n] = zl;
      }
    }
    m[i] = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (8 * (e >> 2) + (e & 3) >= nw - vl) acc[i][e] = -INFINITY;
      m[i] = fmaxf(m[i], acc[i][e]);
    }
    m[i] = swap32_max(m[i]);
    if (lane < 32) ex[wave * (32 * NB) + 32 * i + lane] = m[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NB; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) m[i] = fmaxf(m[i], ex[k * (32 * NB) + 32 * i + (lane & 31)]);
    const float m0 = m[i] == -INFINITY ? 0.f : m[i];
    const int64_t n0 = j0 + 32 * i;
    uint16_t* const exps =
        MODE == CE_KEEP ? a.dzt + (n0 / TILE * a.words + rel / TILE * TILE) * TILE + block * 8192 +
                              (n0 % TILE) / 32 * 1024
                        : nullptr;
    sum[i] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp_of(acc[i][8 * h + e] - m0);
        sum[i] += p[e];
      }
      if constexpr (MODE == CE_KEEP) {
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = kept2(p[2 * e], p[2 * e + 1]);
        *reinterpret_cast<u32x4*>(exps + h * 512 + lane * 8) = v;
      }
    }
    sum[i] = swap32_sum(sum[i]);
    if (lane < 32) ex[(4 + wave) * (32 * NB) + 32 * i + lane] = sum[i];
  }
  __syncthreads();
  const int64_t n = j0 + threadIdx.x;
  if (threadIdx.x < 32 * NB && n < rows) {
    float t = -INFINITY, u = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      t = fmaxf(t, ex[k * (32 * NB) + threadIdx.x]);
      u += ex[(4 + k) * (32 * NB) + threadIdx.x];
    }
    float* out = a.stats + ((int64_t)(a.tile0 + tile_i) * a.planes + 2 * side) * a.Np + n;
    out[0] = t;
    out[a.Np] = u;
  }
}

// Sum of p ((t - max t) - (s - max s)) over the words of each tile of a launch that kept both sides'
// logits, with the maxima and the weights relative to the teacher's of the tile: the fifth plane of the
// statistics. What all logits of a row have in common is no part of the loss, and is none of the sum's
// rounding either. HBM-bound, 8 bytes a logit. A workgroup takes a tile's column of 64 rows, wave w its
// words 64 w .. 64 w + 63.
struct CrossArgs {
  const float* kept;
  int64_t kept_side;
  const Meta* meta;
  float* stats;
  int64_t Np, v0, v1;
  int halves;  // statistics of 128 words
};
__global__ __launch_bounds__(256) void cross_kernel(const CrossArgs a) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wj = (int)blockIdx.x & 3;
  const int tiles_i = (int)((a.v1 - a.v0 + TILE - 1) / TILE);
  const int64_t tile = (int64_t)blockIdx.x >> 2;
  const int tile_j = (int)(tile / tiles_i), tile_i = (int)(tile % tiles_i);
  const int rows = a.meta->rows;
  if (tile_j * TILE + wj * 64 >= rows) return;
  const int nw = (int)min((int64_t)TILE, a.v1 - a.v0 - (int64_t)tile_i * TILE);
  // the statistics of this wave's words
  const int wi = w >> 1;
  float* const st0 = a.stats + tile_j * TILE + wj * 64;
  const int64_t tile_v = a.v0 / TILE + tile_i;
  const float* st = st0 + (a.halves ? 2 * tile_v + wi : tile_v) * 5 * a.Np;
#pragma unroll
  for (int tj = 0; tj < WT_J; ++tj) {
    const int n = 32 * tj + (lane & 31);
    const bool any = (!a.halves || nw > 128 * wi) && tile_j * TILE + wj * 64 + n < rows;
    const float ms = any ? st[n] : 0.f, mt = any ? st[2 * a.Np + n] : 0.f;
    const float ms0 = ms == -INFINITY ? 0.f : ms, mt0 = mt == -INFINITY ? 0.f : mt;
    float c = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int ti = 2 * (w & 1) + t;
      const int left = nw - 128 * wi - 32 * ti - 4 * (lane >> 5);
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int64_t o = tile * (TILE * TILE / 4) + ((ti * WT_J + tj) * 4 + e4) * NTHR +
                          (wi * WAVES_J + wj) * 64 + lane;
        const float4 z = reinterpret_cast<const float4*>(a.kept)[o];
        const float4 t = reinterpret_cast<const float4*>(a.kept + a.kept_side)[o];
        const float zs[4] = {z.x, z.y, z.z, z.w}, zt[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp_of(zt[e] - mt0);
          // a word without weight counts for nothing, however far the two sides are
          if (8 * e4 + e < left && p != 0.f) c += p * ((zt[e] - mt0) - (zs[e] - ms0));
        }
      }
    }
    c = swap32_sum(c);
    if (lane < 32) sh[w][n] = c;
  }
  __syncthreads();
  if (lane + tile_j * TILE + wj * 64 >= rows || w > (a.halves && nw > 128 ? 1 : 0)) return;
  if (a.halves) st0[((2 * tile_v + w) * 5 + 4) * a.Np + lane] = sh[2 * w][lane] + sh[2 * w + 1][lane];
  else st0[(tile_v * 5 + 4) * a.Np + lane] = sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane];
}

// ---- the losses' total --------------------------------------------------------------------------------
struct Total {
  const float* loss;  // [N]
  int64_t N;
  float* out;  // {sum, mean over the rows that take part (0 without one), their number}, or NULL
};
// A row's loss goes past the XCD's L2 (agent scope), and the barrier in add_up waits until it has: no
// fence, which would write the L2 back once a workgroup (5 us of a launch of 256).
__device__ __forceinline__ void put_loss(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// By the last workgroup of 256 threads that has written its rows' losses: which one it is does not
// change the order of the sum.
__device__ __forceinline__ void add_up(const Total& t, Meta* meta) {
  __shared__ int last;
  __shared__ double red[4];
  if (!t.out) return;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();  // the workgroup's losses are written
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(&meta->done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  double s = 0;
#pragma unroll 16
  for (int64_t r = threadIdx.x; r < t.N; r += 256)
    s += __hip_atomic_load(t.loss + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = red[0] + red[1] + red[2] + red[3];
    const int rows = meta->rows;
    t.out[0] = (float)s;
    t.out[1] = rows > 0 ? (float)(s / rows) : 0.f;
    t.out[2] = (float)rows;
  }
}
__global__ void no_total_kernel(float* out) {  // of no rows
  if (threadIdx.x < 3) out[threadIdx.x] = 0.f;
}

// ---- joining the tiles' statistics ------------------------------------------------------------------
// 256 threads: 1 << rb_log rows, the rest of the threads along the tiles; each joins its tiles in order,
// then pairs of threads join theirs, so the order is fixed.
struct JoinArgs {
  const float* stats;
  const float* zlab;
  Meta* meta;
  const int32_t* src;
  const int32_t* lab;
  int64_t Np;
  int tiles, rb_log;
  Total total;
  float* loss;     // [N]
  float* lse[2];   // [N], and what rounding them leaves
  float* rest_out[2];
  float* lsep[2];  // [Np], of the packed rows (or NULL), and what rounding them leaves
  float* rest[2];
  float* apart;    // [Np] the teacher's normaliser less the student's (or NULL)
  int32_t* best[2];  // [Np] the tile of each side's maximum (or NULL)
  float* low;        // cross entropy: [Np] what rounding the labels' dz will leave (or NULL)
};
// JOIN_LSE: both sides' normalisers, the loss comes later; JOIN_BEST: the tiles of the maxima alone
enum { JOIN_CE, JOIN_KL, JOIN_LSE, JOIN_BEST };
template <int WHAT>
__device__ __forceinline__ void write_row(const JoinArgs& a, int64_t p, const Stat& s0, const Stat& s1, float c) {
  const int64_t r = a.src[p];
  const double exact = (double)s0.m + log((double)s0.s);
  const float lse = (float)exact;
  a.lse[0][r] = lse;
  a.rest_out[0][r] = (float)(exact - lse);
  if (a.lsep[0]) {
    a.lsep[0][p] = lse;
    a.rest[0][p] = (float)(exact - lse);
  }
  if constexpr (WHAT != JOIN_CE) {
    const double exact_t = (double)s1.m + log((double)s1.s);
    const float lt = (float)exact_t;
    a.lse[1][r] = lt;
    a.rest_out[1][r] = (float)(exact_t - lt);
    if (a.lsep[1]) {
      a.lsep[1][p] = lt;
      a.rest[1][p] = (float)(exact_t - lt);
    }
    // from the sums' quotient (and the maxima's difference): as a difference of two rounded normalisers it
    // would lose their common part
    const double quotient = log((double)s1.s / s0.s);
    if constexpr (WHAT == JOIN_KL) put_loss(a.loss + r, (float)((double)c / s1.s - quotient));
    else a.apart[p] = (float)(((double)s1.m - s0.m) + quotient);
  } else {
    put_loss(a.loss + r, a.lab[p] < 0 ? __builtin_nanf("")
                                      : (float)((double)s0.m - a.zlab[p] + log((double)s0.s)));
    if (a.low && a.lab[p] >= 0) {  // as finish_kernel forms it
      const float d = expm1f((a.zlab[p] - lse) - (float)(exact - lse));
      a.low[p] = left_of(d, (uint16_t)f2bf(d));
    }
  }
}

template <int WHAT>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
  constexpr int PLANES = WHAT == JOIN_CE ? 2 : WHAT == JOIN_KL ? 5 : 4;
  constexpr bool BEST = WHAT == JOIN_LSE || WHAT == JOIN_BEST;
  __shared__ float sh[PLANES][256];
  __shared__ int sh_best[BEST ? 2 : 1][256];
  int best0 = 0, best1 = 0;
  const int RB = 1 << a.rb_log, slices = 256 >> a.rb_log;
  const int rl = threadIdx.x & (RB - 1), sl = threadIdx.x >> a.rb_log;
  const int64_t p = (int64_t)blockIdx.x * RB + rl;
  const bool live = p < a.meta->rows;
  Stat s0{-INFINITY, 0.f}, s1{-INFINITY, 0.f};
  float c = 0.f;
  // both sides' words, and with the fifth plane theirs in common
  auto add = [&](const Stat& t0, const Stat& t1, float tc) {
    const Stat m0 = join(s0, t0);
    if constexpr (PLANES > 2) {
      const Stat m1 = join(s1, t1);
      if constexpr (PLANES > 4)
        c = cross_of(c, s0, s1, m0.m, m1.m) + cross_of(tc, t0, t1, m0.m, m1.m);
      s1 = m1;
    }
    s0 = m0;
  };
  if (live) {
#pragma unroll 4
    for (int t = sl; t < a.tiles; t += slices) {
      const float* v = a.stats + (int64_t)t * PLANES * a.Np + p;
      if constexpr (BEST) {
        if (v[0] > s0.m) best0 = t;
        if (v[2 * a.Np] > s1.m) best1 = t;
      }
      add(Stat{v[0], v[a.Np]}, PLANES > 2 ? Stat{v[2 * a.Np], v[3 * a.Np]} : Stat{},
          PLANES > 4 ? v[4 * a.Np] : 0.f);
    }
  }
  for (int half = slices / 2; half >= 1; half >>= 1) {
    if (sl >= half && sl < 2 * half) {
      sh[0][threadIdx.x] = s0.m;
      sh[1][threadIdx.x] = s0.s;
      if constexpr (PLANES > 2) {
        sh[2][threadIdx.x] = s1.m;
        sh[3][threadIdx.x] = s1.s;
        if constexpr (PLANES > 4) sh[4][threadIdx.x] = c;
      }
      if constexpr (BEST) {
        sh_best[0][threadIdx.x] = best0;
        sh_best[1][threadIdx.x] = best1;
      }
    }
    __syncthreads();
    if (sl < half) {
      const int i = threadIdx.x + half * RB;
      if constexpr (BEST) {
        if (sh[0][i] > s0.m) best0 = sh_best[0][i];
        if (sh[2][i] > s1.m) best1 = sh_best[1][i];
      }
      if constexpr (PLANES == 2) add(Stat{sh[0][i], sh[1][i]}, Stat{}, 0.f);
      else add(Stat{sh[0][i], sh[1][i]}, Stat{sh[2][i], sh[3][i]}, PLANES > 4 ? sh[PLANES - 1][i] : 0.f);
    }
    // (the next round writes the lower half of what this one read)
  }
  if (live && sl == 0) {
    if constexpr (WHAT != JOIN_BEST) write_row<WHAT>(a, p, s0, s1, c);
    if (BEST && a.best[0]) {
      a.best[0][p] = best0;
      a.best[1][p] = best1;
    }
  }
  if constexpr (!BEST) add_up(a.total, a.meta);
}

// The loss of every row that takes part from its parts [parts][Np], in order
__global__ __launch_bounds__(256) void rows_kernel(const float* __restrict__ part, int parts, Meta* meta,
                                                   const int32_t* __restrict__ src, int64_t Np,
                                                   float* loss, Total total) {
  __shared__ double sh[256];
  const int rl = threadIdx.x & 7, sl = threadIdx.x >> 3;  // 8 rows
  const int64_t p = (int64_t)blockIdx.x * 8 + rl;
  const bool live = p < meta->rows;
  double s = 0;
  if (live) {
#pragma unroll 4
    for (int k = sl; k < parts; k += 32) s += part[k * Np + p];
  }
  sh[threadIdx.x] = s;
  __syncthreads();
  if (live && sl == 0) {
    for (int k = 1; k < 32; ++k) s += sh[k * 8 + rl];
    put_loss(loss + src[p], (float)s);
  }
  add_up(total, meta);
}

// ---- the word whose gradient is the greatest -----------------------------------------------------------
// One word often holds nearly all of a row's dz (97% of its squares where teacher and student lean to other
// words), and rounding that one to bf16 is then what the gradients are off by, as much as by their own
// rounding. So what the rounding leaves of it is added to the products' sums. Of a cross entropy it is the
// label's word: 1 - q is the sum of all others' q. Of a distillation it is looked for in the tiles of both
// sides' maxima, a row a wave, 4 words a lane, with dz as finish_kernel forms it. Of a vocabulary in pieces
// every piece has its own, which its dW adds; dx adds the greatest of all pieces.
struct TopArgs {
  const float* kept;
  int64_t kept_side;
  int64_t n, v0;  // words, and the first of them
  int best_shift;  // best counts tiles of 256 words >> best_shift
  const Meta* meta;
  const int32_t* best[2];
  const float *lse[2], *rest[2];
  const float* g;  // [Np] or NULL
  int32_t* word;   // [Np], -1: none
  float* low;      // [Np]
  int32_t* x_word;  // of the pieces so far (or NULL)
  float *x_low, *x_most;
};
__global__ __launch_bounds__(256) void top_kernel(const TopArgs a) {
  const int lane = threadIdx.x & 63, p = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (p >= a.meta->rows) return;
  const int tiles_i = (int)((a.n + TILE - 1) / TILE);
  const int half = lane & 1, e4 = (lane >> 1) & 3, ti = (lane >> 3) & 3, wi = lane >> 5;
  const int nl = p % TILE, wj = nl / 64, tj = nl / 32 % 2;
  const float lse = a.lse[0][p], lt = a.lse[1][p], rest = a.rest[0][p], rest_t = a.rest[1][p];
  const float g = a.g ? a.g[p] : 1.f;
  float most = 0.f;
  int word = -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int t = a.best[side][p] >> a.best_shift;
    const int64_t o = ((int64_t)(p / TILE) * tiles_i + t) * (TILE * TILE / 4) +
                      ((ti * WT_J + tj) * 4 + e4) * NTHR + (wi * WAVES_J + wj) * 64 + nl % 32 + 32 * half;
    const f32x4 zs = reinterpret_cast<const f32x4*>(a.kept)[o];
    const f32x4 zt = reinterpret_cast<const f32x4*>(a.kept + a.kept_side)[o];
    const int v = t * TILE + (wi * 4 + ti) * 32 + 8 * e4 + 4 * half;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = (exp_of((zs[e] - lse) - rest) - exp_of((zt[e] - lt) - rest_t)) * g;
      if (v + e < a.n && fabsf(d) > fabsf(most)) {
        most = d;
        word = v + e;
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float d = __shfl_xor(most, o);
    const int w = __shfl_xor(word, o);
    if (fabsf(d) > fabsf(most) || (fabsf(d) == fabsf(most) && w > word)) {
      most = d;
      word = w;
    }
  }
  if (lane == 0) {
    const float low = left_of(most, (uint16_t)f2bf(most));
    word = word < 0 ? -1 : (int)a.v0 + word;
    a.word[p] = word;
    a.low[p] = low;
    if (a.x_word && (a.v0 == 0 || fabsf(most) > a.x_most[p])) {
      a.x_word[p] = word;
      a.x_low[p] = low;
      a.x_most[p] = fabsf(most);
    }
  }
}

// ---- dz of tiles that were kept ----------------------------------------------------------------------
// A workgroup takes blocks of 32 words x 256 rows (wave column wj the rows 64 wj ..): HBM-bound, 4
// (cross entropy, in place) or 10 bytes a logit. The cross entropy's block of exponentials lies where
// its dz goes, and is in registers before any of that is written. A distillation's blocks also add up
// their words' share of the loss.
// (Blocks of a workgroup: a distillation's parts of the loss are read again, 2 of 1, 2, 4 and 8 measured;
// 4 or 8 cost the cross entropy a tenth.)
constexpr int kFinishKl = 2;
struct FinishArgs {
  uint16_t* dzt;
  int64_t words, n, Np;  // of the panels, of the piece
  int per;               // blocks of a workgroup, of one tile
  int stat_log;          // words of a statistic: 7 or 8
  const Meta* meta;
  const int32_t* lab;
  const float* stats;
  const float* zlab;
  // [Np] normalisers, and what rounding them left: where a word holds nearly all, its gradient
  // is a small difference, and the rounding of a normaliser of 16 (10^-6) would be 1% of 10^-4
  const float *lse[2], *rest[2];
  const float* apart;   // [Np]
  const float* g;       // [Np] or NULL
  const float* kept;
  int64_t kept_side;
  float* loss;  // [words / 32 / per][Np], or NULL
};
template <bool KL>
__global__ __launch_bounds__(256) void finish_kernel(const FinishArgs a) {
  __shared__ __align__(16) uint8_t st[32 * EPI_RS];
  const int lane = threadIdx.x & 63, wj = threadIdx.x >> 6;
  const int tiles_i = (int)((a.n + TILE - 1) / TILE), of = 8 / a.per;
  const int64_t tile = (int64_t)blockIdx.x / of;
  const int tile_j = (int)(tile / tiles_i), tile_i = (int)(tile % tiles_i);
  const int rows = a.meta->rows;
  const bool two = two_parts(rows);
  if (tile_j * TILE >= rows) return;
  const int part = (int)blockIdx.x % of;
  float kl[WT_J] = {0.f, 0.f};
  for (int block = part * a.per; block < (part + 1) * a.per; ++block) {
    const int wi = block >> 2, ti = block & 3;
    uint8_t* at = reinterpret_cast<uint8_t*>(a.dzt + ((int64_t)tile_j * a.words + tile_i * TILE) * TILE) +
                  block * 16384;
    const int v0 = tile_i * TILE + block * 32;  // the block's first word
    uint4 raw[KL ? 1 : WT_J][2];
    if constexpr (!KL) {
#pragma unroll
      for (int tj = 0; tj < WT_J; ++tj)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          raw[tj][h] = *reinterpret_cast<const uint4*>(at + wj * 4096 + tj * 2048 + h * 1024 + lane * 16);
    }
#pragma unroll
    for (int tj = 0; tj < WT_J; ++tj) {
      const int nl = wj * 64 + 32 * tj + (lane & 31), n = tile_j * TILE + nl;
      const bool live = n < rows;
      const float lse = live ? a.lse[0][n] : 0.f, rest = live ? a.rest[0][n] : 0.f;
      const int left = (int)(a.n - v0) - 4 * (lane >> 5);  // words from the lane's first one
      float d[16];
      if constexpr (KL) {
        const float lt = live ? a.lse[1][n] : 0.f, rest_t = live ? a.rest[1][n] : 0.f;
        const float apart = live && a.loss ? a.apart[n] : 0.f;
        const float g = live && a.g ? a.g[n] : 1.f;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int64_t o = tile * (TILE * TILE / 4) + ((ti * WT_J + tj) * 4 + e4) * NTHR +
                            (wi * WAVES_J + wj) * 64 + lane;
          const f32x4 zs = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.kept) + o);
          const f32x4 zt =
              __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.kept + a.kept_side) + o);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float q = exp_of((zs[e] - lse) - rest), p = exp_of((zt[e] - lt) - rest_t);
            d[4 * e4 + e] = (q - p) * g;
            // a word without weight counts for nothing, however far the two sides are
            if (8 * e4 + e < left && p != 0.f) kl[tj] += p * ((zt[e] - zs[e]) - apart);
          }
        }
      } else {
        const int l = live ? a.lab[n] : 0;
        float f = 0.f;
        if (live && v0 < a.n)
          f = exp_of((a.stats[(int64_t)(v0 >> a.stat_log) * 2 * a.Np + n] - lse) - rest) * (1.f / kKeptScale);
        if (l < 0) f = __builtin_nanf("");  // no such word: nothing to learn from
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w[4] = {raw[tj][h].x, raw[tj][h].y, raw[tj][h].z, raw[tj][h].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[8 * h + 2 * e] = h2f(w[e] & 0xffffu) * f;
            d[8 * h + 2 * e + 1] = h2f(w[e] >> 16) * f;
          }
        }
        // the label's word from the logit itself
        const int lv = l - v0 - 4 * (lane >> 5);
        if (live && lv >= 0 && lv < 32 && (lv & 4) == 0) {
          const float dl = expm1f((a.zlab[n] - lse) - rest);
#pragma unroll
          for (int e = 0; e < 16; ++e) d[e] = lv == 8 * (e >> 2) + (e & 3) ? dl : d[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = 8 * (e >> 2) + (e & 3);
        const float v = live && row < left ? d[e] : 0.f;
        const uint16_t high = (uint16_t)f2bf(v);
        uint16_t* const to = reinterpret_cast<uint16_t*>(st + (row + 4 * (lane >> 5)) * EPI_RS) + nl;
        if (!two) {
          *to = high;
        } else if (nl < kTwo) {
          *to = high;
          to[kTwo] = low_part(v, high);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int c = it * 256 + threadIdx.x;
      *reinterpret_cast<uint4*>(at + c * 16) =
          *reinterpret_cast<const uint4*>(st + (c >> 5) * EPI_RS + (c & 31) * 16);
    }
    __syncthreads();
  }
  if constexpr (KL) {
    if (!a.loss) return;
#pragma unroll
    for (int tj = 0; tj < WT_J; ++tj) {
      const int n = tile_j * TILE + wj * 64 + 32 * tj + (lane & 31);
      const float s = swap32_sum(kl[tj]);
      if (lane < 32 && n < rows) a.loss[((int64_t)tile_i * of + part) * a.Np + n] = s;
    }
  }
}

// A Col tile's copies of p[r][H] whose columns past H are out of the buffer, and so zero, as the rows
// past rtotal. p may be of up to 4 GiB (less 16 bytes: rows are of whole 16), which kBufOob lies within.
// (Only the power goes by it: what the columns past H give is stored nowhere.)
constexpr uint32_t kPastAll = 0xfffffff0u;
__device__ __forceinline__ TileDma col_tile_zero(const uint16_t* p, int64_t H, int64_t col0, int64_t rtotal) {
  TileDma d = col_tile_dma(p, H, col0, H, rtotal);
#pragma unroll
  for (int it = 0; it < COPY_INSTS; ++it) {
    const int pch = it * NTHR + threadIdx.x;
    if (col0 + (((pch & 31) ^ col_swz(pch >> 5)) * 8) >= H) d.off[it] = kPastAll;
  }
  return d;
}

// ---- dW of a piece: dz^T [words, rows] x [rows, H] ----------------------------------------------------
struct DwArgs {
  const uint16_t* dzt;
  int64_t panel;  // words of dz's panels, whole tiles
  const uint16_t* x;
  int64_t Np, H, words;
  const Meta* meta;
  int64_t v0;     // the piece's first word
  uint16_t* out;  // [words][H]
  const int32_t* top;  // [Np] words, or NULL
  const float* low;    // [Np] what rounding their dz left
};
// acc += the remainders of dz of the tile's words i0 .. times their rows of x, 64 rows a stage. The rows are
// looked through 4096 at a time, their words loaded together (512 at a time cost a dW of 4096 rows of 151936
// words 5% instead of 3%).
__device__ __forceinline__ void dw_remainders(lds_u8* lbase, const DwArgs& a, int64_t i0, int64_t j0,
                                              f32x16 (&acc)[WT_I][WT_J], int wi, int wj, int lane) {
  typedef __attribute__((address_space(3))) int lds_int;
  constexpr int LOOKS = 8;
  static_assert(LOOKS * (NTHR / 64) == 64, "a count a lane");
  // behind the tiles of a stage, the list: row (below 2^22) | word of the tile << 22, up to 63 + 4096
  lds_int* const list = reinterpret_cast<lds_int*>(lbase + 2 * TILE_BYTES);
  lds_int* const counts = reinterpret_cast<lds_int*>(lbase + 4 * TILE_BYTES);
  const int rows = a.meta->rows, wave = threadIdx.x >> 6;
  const int64_t first = a.v0 + i0;
  int have = 0;
  for (int base = 0; base < rows; base += LOOKS * NTHR) {
    int word[LOOKS];
    uint64_t mine[LOOKS];
#pragma unroll
    for (int k = 0; k < LOOKS; ++k) {
      const int r = base + k * NTHR + (int)threadIdx.x;
      word[k] = r < rows ? a.top[r] : -1;
    }
#pragma unroll
    for (int k = 0; k < LOOKS; ++k) {
      const bool in = word[k] >= first && word[k] < first + TILE;
      word[k] = in ? (int)(word[k] - first) : -1;
      mine[k] = __ballot(in);
      if (lane == 0) counts[k * (NTHR / 64) + wave] = __popcll(mine[k]);
    }
    __syncthreads();
    // in the rows' order: 64 of them a count, summed over the counts before
    const int count = counts[lane];
    int upto = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      upto += lane >= o ? v : 0;
    }
#pragma unroll
    for (int k = 0; k < LOOKS; ++k) {
      const int at = __shfl(upto - count, k * (NTHR / 64) + wave);
      if (word[k] >= 0)
        list[have + at + __popcll(mine[k] & ((1ull << lane) - 1))] =
            (base + k * NTHR + (int)threadIdx.x) | word[k] << 22;
    }
    have += __shfl(upto, 63);
    __syncthreads();
    int from = 0;
    while (have - from >= BK || (have > from && base + LOOKS * NTHR >= rows)) {
      const int n = min(have - from, BK);
      // A: zeros but for a remainder a column; B: the rows' x
      uint4* const as = (uint4*)lbase;
      uint4* const bs = (uint4*)(lbase + TILE_BYTES);
      const int e = (int)threadIdx.x < n ? list[from + threadIdx.x] : 0;
      const float low = (int)threadIdx.x < n ? a.low[e & 0x3fffff] : 0.f;
#pragma unroll
      for (int it = 0; it < COPY_INSTS; ++it) {
        const int ch = it * NTHR + threadIdx.x;
        as[ch] = make_uint4(0, 0, 0, 0);
        const int kr = ch >> 5, c = ch & 31;
        const int64_t h = j0 + 8 * c;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (kr < n && h < a.H)
          v = *reinterpret_cast<const uint4*>(a.x + (int64_t)(list[from + kr] & 0x3fffff) * a.H + h);
        bs[col_chunk(kr, c)] = v;
      }
      __syncthreads();
      if ((int)threadIdx.x < n) {
        const int k = (int)threadIdx.x;
        *reinterpret_cast<lds_u16t*>(lbase + row_chunk((int)((uint32_t)e >> 22), k >> 3) * 16 + (k & 7) * 2) =
            (uint16_t)f2bf(low);
      }
      __syncthreads();
      mma_stage_sync<false, true>(lbase, lbase + TILE_BYTES, acc, wi, wj, lane, (n + 15) / 16);
      __syncthreads();
      from += n;
    }
    have -= from;
    if (from > 0) {  // what is left, fewer than 64, to the front
      const int moved = (int)threadIdx.x < have ? list[from + threadIdx.x] : 0;
      __syncthreads();
      if ((int)threadIdx.x < have) list[threadIdx.x] = moved;
    }
  }
}
__global__ __launch_bounds__(NTHR) void dw_kernel(const DwArgs a) {
  extern __shared__ uint4 smem[];
  lds_u8* lbase = (lds_u8*)smem;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave / WAVES_J, wj = wave % WAVES_J;
  const int tiles_i = (int)((a.words + TILE - 1) / TILE), tiles_j = (int)((a.H + TILE - 1) / TILE);
  const Item item = map_item(tiles_i * tiles_j, false, 0, 1, (int)blockIdx.x, 0, 1);
  int tile_i, tile_j;
  tile_coords(4, tiles_i, tiles_j, item.bid, tile_i, tile_j);
  const int64_t i0 = (int64_t)tile_i * TILE, j0 = (int64_t)tile_j * TILE;
  f32x16 acc[WT_I][WT_J];
#pragma unroll
  for (int i = 0; i < WT_I; ++i)
#pragma unroll
    for (int j = 0; j < WT_J; ++j) acc[i][j] = f32x16{};
  // whole stages: the packed rows past the last one are cleared, and so is dz there
  const bool two = two_parts(a.meta->rows);
  const int part = (a.meta->rows + BK - 1) / BK, nst = two ? 2 * part : part;
  // (row_tile_dma bounds the copies by its rows: here by all panels)
  TileDma dA = row_tile_dma(a.dzt + i0 * TILE, TILE, 0, TILE);
  dA.r = make_rsrc(a.dzt + i0 * TILE, (uint32_t)((a.Np / TILE * a.panel - i0) * TILE * 2));
  const TileDma dB = col_tile_zero(a.x, a.H, j0, a.Np);
  const uint32_t panel = (uint32_t)(a.panel * TILE * 2);
  dense_stages<false, true>(lbase, nst, acc, wi, wj, lane, [&](int kt, lds_u8* As, lds_u8* Bs) {
    const bool second = two && kt >= part;  // the second parts, times the same rows of x
    const int ka = second ? kt + kTwo / BK - part : kt, kb = second ? kt - part : kt;
    tile_copy(As, dA, (uint32_t)(ka / (TILE / BK)) * panel + (uint32_t)(ka % (TILE / BK)) * (BK * 2));
    tile_copy(Bs, dB, (uint32_t)((int64_t)kb * BK * a.H * 2));
  });
  if (a.top && !two) dw_remainders(lbase, a, i0, j0, acc, wi, wj, lane);
  const float alpha = a.meta->alpha;
#pragma unroll
  for (int ti = 0; ti < WT_I; ++ti)
#pragma unroll
    for (int tj = 0; tj < WT_J; ++tj)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = wi * (32 * WT_I) + 32 * ti + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        const int col = wj * (32 * WT_J) + 32 * tj + (lane & 31);
        *reinterpret_cast<lds_u16t*>(lbase + row * EPI_RS + col * 2) =
            (uint16_t)f2bf(alpha * acc[ti][tj][e]);
      }
  __syncthreads();
#pragma unroll 4
  for (int it = 0; it < TILE * TILE / 8 / NTHR; ++it) {
    const int ch = it * NTHR + threadIdx.x;
    const int row = ch >> 5, c8 = (ch & 31) * 8;
    if (i0 + row < a.words && j0 + c8 < a.H)
      __builtin_nontemporal_store(
          *reinterpret_cast<const lds_u32x4*>(lbase + row * EPI_RS + c8 * 2),
          reinterpret_cast<u32x4*>(a.out + (i0 + row) * a.H + j0 + c8));
  }
}

// ---- dx of a piece: dz [rows, words] W [words, H], in splits of the words --------------------------------
struct DxArgs {
  const uint16_t* dzt;
  int64_t panel;  // words of dz's panels, whole tiles
  const uint16_t* w;
  int64_t H, words;
  const Meta* meta;
  float* part;  // [z][rows / 4][H][4]
  int add;      // to what earlier pieces left
};
__global__ __launch_bounds__(NTHR) void dx_kernel(const DxArgs a) {
  extern __shared__ uint4 smem[];
  lds_u8* lbase = (lds_u8*)smem;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave / WAVES_J, wj = wave % WAVES_J;
  const int rows = a.meta->rows, z = a.meta->z;
  const int tiles_i = (rows + TILE - 1) / TILE, tiles_j = (int)((a.H + TILE - 1) / TILE);
  const int T = tiles_i * tiles_j;
  if ((int64_t)blockIdx.x >= (int64_t)T * z) return;  // the launch is for as many as there may be
  const int64_t split = ((a.words + z - 1) / z + BK - 1) / BK * BK;
  const Item item = map_item(T, false, 0, 1, (int)blockIdx.x % T, (int)blockIdx.x / T, z);
  const int zsl = item.zsl;
  int tile_i, tile_j;
  // (two tiles of rows at a time; 1, 2 and 4 are within 1% of each other at six shapes of 1000 to 3890 rows
  // and 32000 x 1024 to 128256 x 4096)
  tile_coords(2, tiles_i, tiles_j, item.bid, tile_i, tile_j);
  const int64_t i0 = (int64_t)tile_i * TILE, j0 = (int64_t)tile_j * TILE;
  const int64_t rbeg = (int64_t)zsl * split, rend = min(a.words, rbeg + split);
  f32x16 acc[WT_I][WT_J];
#pragma unroll
  for (int i = 0; i < WT_I; ++i)
#pragma unroll
    for (int j = 0; j < WT_J; ++j) acc[i][j] = f32x16{};
  // whole stages: words past the last are past both buffers and zero (Operands)
  const int nst = rend > rbeg ? (int)((rend - rbeg + BK - 1) / BK) : 0;
  const TileDma dA = col_tile_dma(a.dzt + tile_i * a.panel * TILE, TILE, 0, TILE, rend);
  const TileDma dB = col_tile_zero(a.w, a.H, j0, rend);
  col_stages<true>(lbase, nst, acc, wi, wj, lane, [&](bool is_a, int kt, lds_u8* dst) {
    const int64_t r0 = rbeg + (int64_t)kt * BK;
    if (is_a) tile_copy(dst, dA, (uint32_t)(r0 * TILE * 2));
    else tile_copy(dst, dB, (uint32_t)(r0 * a.H * 2));
  });
  __builtin_amdgcn_s_waitcnt(0);  // the repeated copies past the last stage
  if (two_parts(rows)) {
    // the waves of rows kTwo .. hand the second parts' sums to those of the same columns
    __syncthreads();
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    lds_f32x4* ex = reinterpret_cast<lds_f32x4*>(lbase) + (threadIdx.x & (NTHR / 2 - 1));
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (wi == 1 - half) {
#pragma unroll
        for (int i = 0; i < WT_I * WT_J * 4; ++i) {
          f32x16& t = acc[i / (WT_J * 4)][i / 4 % WT_J];
          const int e = i % 4 * 4;
          if (half == 0) {
            ex[i * (NTHR / 2)] = f32x4{t[e], t[e + 1], t[e + 2], t[e + 3]};
          } else {
            const f32x4 v = ex[i * (NTHR / 2)];
            // Of an infinite weight the second part, 0 or of the other sign, would make NaN of the first's
            // infinity; there the first has it all.
#pragma unroll
            for (int k = 0; k < 4; ++k) t[e + k] += fabsf(v[k]) < INFINITY ? v[k] : 0.f;
          }
        }
      }
      __syncthreads();
    }
  }
  // Four rows of a column are four registers: their sums lie together. From the tile's first four rows a
  // lane's offset and a uniform one of its registers.
  const int64_t quads = (rows + 3) / 4;
  float* const part = a.part + ((int64_t)item.zsl * quads + i0 / 4) * a.H * 4;
  const int q0 = wi * (8 * WT_I) + (lane >> 5), nq = (int)(quads - i0 / 4);
#pragma unroll
  for (int tj = 0; tj < WT_J; ++tj) {
    const int64_t h = j0 + wj * (32 * WT_J) + 32 * tj + (lane & 31);
    if (h >= a.H) continue;
    const uint32_t off = (uint32_t)((q0 * a.H + h) * 16);
#pragma unroll
    for (int ti = 0; ti < WT_I; ++ti)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int q = 8 * ti + 2 * e4;
        if (q0 + q >= nq) continue;
        float* const base = part + q * a.H * 4;
        f32x4 v = {acc[ti][tj][4 * e4], acc[ti][tj][4 * e4 + 1], acc[ti][tj][4 * e4 + 2],
                   acc[ti][tj][4 * e4 + 3]};
        if (a.add) v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(base) + off);
        store16(base, off, __builtin_bit_cast(u32x4, v));
      }
  }
}

// The gradients of four packed rows: alpha times the sums of their parts, in order, a column a thread
// (two a thread: 11 and 13 us at 1640 rows of 1600, but 9.7 and 7.3 at 90 of 512)
__global__ __launch_bounds__(256) void dx_sum_kernel(const float* __restrict__ part,
                                                     const int32_t* __restrict__ src,
                                                     const Meta* __restrict__ meta, int H,
                                                     uint16_t* __restrict__ out,
                                                     const int32_t* __restrict__ top,
                                                     const float* __restrict__ low,
                                                     const uint16_t* __restrict__ w) {
  const int hb = (H + 255) / 256;  // workgroups of four rows
  const int64_t q = (int)blockIdx.x / hb;
  const int h = (int)blockIdx.x % hb * 256 + threadIdx.x;
  const int rows = meta->rows, z = meta->z;
  const int64_t quads = (rows + 3) / 4;
  if (q >= quads || h >= H) return;
  int64_t at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = 4 * q + i < rows ? (int64_t)src[4 * q + i] * H + h : -1;
  f32x4 left = {};  // (loaded beside the parts)
  if (top && !two_parts(rows)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = at[i] >= 0 ? top[4 * q + i] : -1;
      const float l = t >= 0 ? low[4 * q + i] * bf2f(w[(int64_t)t * H + h]) : 0.f;
      left[i] = fabsf(l) < INFINITY ? l : 0.f;  // (as dx_kernel's second parts)
    }
  }
  f32x4 a = {};
  const f32x4* v = reinterpret_cast<const f32x4*>(part) + q * H + h;
#pragma unroll 8
  for (int k = 0; k < z; ++k, v += quads * H) a += *v;
  a += left;
  const float alpha = meta->alpha;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at[i] >= 0) out[at[i]] = (uint16_t)f2bf(alpha * a[i]);
}

// ---- host ---------------------------------------------------------------------------------------------
static int cu_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0)
      v = 256;
    cache[dev] = v;
  }
  return cache[dev];
}
static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Words of a piece: `bytes` a logit of all rows in kPieceBytes and W's rows of it within the 4 GiB that
// the copies of dx address, the pieces of one size but for the last tiles.
static int64_t piece_words(int64_t N, int64_t V, int64_t H, int bytes) {
  const int64_t tiles = up(V, TILE) / TILE;
  const int64_t held = (int64_t)(kPieceBytes / bytes) / std::max(up(N, TILE), (int64_t)1);
  const int64_t addressed = (((int64_t)1 << 31) - 1) / H;
  const int64_t most = std::max(std::min(held, addressed) / TILE, (int64_t)1);
  const int64_t pieces = (tiles + most - 1) / most;
  return (tiles + pieces - 1) / pieces * TILE;
}
// The workspace, carved in order; p = NULL: sizes only.
struct Carve {
  char* p;
  size_t used = 0;
  template <typename T>
  T* take(size_t n) {
    T* r = p ? reinterpret_cast<T*>(p + used) : nullptr;
    used += (n * sizeof(T) + 255) / 256 * 256;
    return r;
  }
};
struct Ws {
  Meta* meta;
  int32_t *src, *lab;
  uint16_t* xp[2];
  float* zlab;
  float* stats;
  float* kept;
  float *lse[2], *rest[2];
  float* apart;
  // of more than kTwo rows: each row's word whose dz is the greatest and what rounding that left; of a
  // distillation the tiles that it is looked for in, and of its backward that of all pieces so far
  int32_t *best[2], *top, *x_top;
  float *low, *x_low, *x_most;
  float* kl;
  float* g;
  uint16_t* dzt;
  float* part;
  int64_t words, part_floats;  // of a piece
};
enum { WS_FWD, WS_BWD, WS_STEP };
// Whether the tiles are those of few rows: one row of them (where half of a 256x256 tile's rows do not
// exist: 128 rows of 151936 x 2560 215 us, 129 by the other tiles 241), or two workgroups a CU for all of
// them (us here and by the other tiles: 256 rows of 32000 x 1024 / 2560 31.6 / 55.7 and 38.3 / 63.6, 768 of
// 8000 x 2560 51 and 65; 384 of 32000 x 1024 43.9 and 41.1, 256 of 151936 x 2560 299 and 249).
static bool few(int64_t N, int64_t V, int64_t Ht) {
  const int64_t tiles = up(V, kFewWords) / kFewWords * (up(N, 128) / 128) * (Ht ? 2 : 1);
  return N <= 128 || tiles <= 2 * cu_count();
}
static int stat_words(int64_t N, int64_t V, int64_t Ht) { return few(N, V, Ht) ? kFewWords : TILE; }
static Ws carve(Carve& c, int use, int64_t N, int64_t V, int64_t H, int64_t Ht, bool grad_x) {
  Ws w = {};
  const int64_t Np = up(N, TILE), Vp = up(V, TILE);
  w.words = use == WS_STEP ? Vp : piece_words(N, V, H, !Ht ? 2 : use == WS_FWD ? 8 : 10);
  w.meta = c.take<Meta>(1);
  w.src = c.take<int32_t>(Np);
  w.lab = c.take<int32_t>(Np);
  w.xp[0] = c.take<uint16_t>(Np * H);
  if (Ht) {
    w.xp[1] = c.take<uint16_t>(Np * Ht);
    w.kept = c.take<float>((size_t)(2 * Np * w.words));
  } else {
    w.zlab = c.take<float>(Np);
  }
  if (Ht || use != WS_BWD)
    w.stats = c.take<float>((size_t)((use == WS_BWD ? w.words : Vp) / stat_words(N, V, Ht)) * (Ht ? 5 : 2) * Np);
  if (use == WS_FWD) return w;
  for (int k = 0; k < (Ht ? 2 : 1); ++k) {
    w.lse[k] = c.take<float>(Np);
    w.rest[k] = c.take<float>(Np);
  }
  if (use == WS_BWD) w.g = c.take<float>(Np);
  if (!two_parts(N)) {
    for (int k = 0; k < (Ht ? 2 : 0); ++k) w.best[k] = c.take<int32_t>(Np);
    w.top = w.x_top = Ht ? c.take<int32_t>(Np) : w.lab;
    w.low = w.x_low = c.take<float>(Np);
    if (Ht && use == WS_BWD) {
      w.x_top = c.take<int32_t>(Np);
      w.x_low = c.take<float>(Np);
      w.x_most = c.take<float>(Np);
    }
  }
  if (use == WS_STEP && Ht) {
    w.apart = c.take<float>(Np);
    w.kl = c.take<float>((size_t)(Vp / 32 / kFinishKl) * Np);
  }
  w.dzt = c.take<uint16_t>((size_t)w.words * Np);
  if (grad_x) {
    // dx's parts: the splits that all rows would take
    w.part_floats = (int64_t)dx_splits(N, w.words, H, cu_count()) * up(N, 4) * H;
    w.part = c.take<float>((size_t)w.part_floats);
  }
  return w;
}
// Whether the forward of so many rows may keep what the gradients are made of
static bool step_fits(int64_t N, int64_t V, int64_t H, int64_t Ht) {
  const int64_t logits = up(N, TILE) * up(V, TILE);
  return N > 0 && V < ((int64_t)1 << 31) - TILE && logits <= (int64_t)(kKeepBytes / (Ht ? 10 : 2)) &&
         logits * 2 < ((int64_t)1 << 32) && V * H < ((int64_t)1 << 31);
}

static bool a16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// What the two losses share: the sides of a call and its checks.
struct Sides {
  const uint16_t *x, *w, *tx, *tw;
  const void* key;
  int kind;
  int64_t ignore;
  float inv_t;
  int64_t N, V, H, Ht;
};
static int check(const Sides& s, bool kl, const char* what) {
  PLZ_REQUIRE(s.N >= 0 && s.V >= 1 && s.H >= 8 && (!kl || s.Ht >= 8), "%s: bad shape", what);
  PLZ_REQUIRE(s.H % 8 == 0 && s.Ht % 8 == 0, "%s: hidden widths must be multiples of 8", what);
  const int64_t lim = (int64_t)1 << 31;
  if (up(s.N, TILE) * s.H >= lim || up(s.N, TILE) * s.Ht >= lim || s.V >= lim - TILE ||
      s.N >= ((int64_t)1 << 22) || std::max(s.H, s.Ht) >= ((int64_t)1 << 22) ||
      up(s.N, TILE) / TILE * (up(s.V, TILE) / TILE) >= lim) {
    set_error("%s: 2^31 values of x, words or tiles, 2^22 rows or a width of 2^22, or more", what);
    return PLZ_EUNSUPPORTED;
  }
  PLZ_REQUIRE(s.w && (s.x || s.N == 0) && (!kl || (s.tw && (s.tx || s.N == 0))),
              "%s: null pointer", what);
  PLZ_REQUIRE(a16(s.x) && a16(s.w) && a16(s.tx) && a16(s.tw),
              "%s: x and weights must be 16-byte aligned", what);
  if (kl) PLZ_REQUIRE(s.inv_t > 0.f && s.inv_t < INFINITY, "%s: bad temperature", what);
  return PLZ_OK;
}
static int check_ws(const void* ws, size_t have, size_t need, const char* what) {
  if (!ws || have < need) {
    set_error("%s: workspace of %zu bytes needed, %zu given", what, need, ws ? have : 0);
    return PLZ_EWORKSPACE;
  }
  PLZ_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace must be 16-byte aligned", what);
  return PLZ_OK;
}

static PackArgs pack_args(const Sides& s, const Ws& w) {
  PackArgs a = {};
  a.key = s.key; a.kind = s.kind; a.ignore = s.ignore; a.V = s.V; a.N = s.N;
  a.x[0] = s.x; a.xp[0] = w.xp[0]; a.H[0] = s.H;
  if (s.Ht) {
    a.x[1] = s.tx; a.xp[1] = w.xp[1]; a.H[1] = s.Ht;
  }
  a.meta = w.meta; a.src = w.src; a.lab = w.lab;
  // (every workgroup counts: with 4 rows each, 2^20 keys would be read 2^17 times)
  a.per = s.N <= 2048 ? 4 : s.N <= 16384 ? 8 : kPackMost;
  a.words = w.words; a.z_floats = w.part_floats; a.cus = cu_count();
  a.inv_t = s.inv_t;
  a.reduction = PLZ_REDUCE_NONE;
  return a;
}
static int pack(const PackArgs& a, hipStream_t st, const char* what) {
  hipLaunchKernelGGL(pack_kernel, dim3((unsigned)((a.N + a.per - 1) / a.per + TILE / a.per)), dim3(256), 0,
                     st, a);
  return check_launch(what);
}
static LogitArgs logit_args(const Sides& s, const Ws& w) {
  LogitArgs a = {};
  a.w[0] = s.w; a.x[0] = w.xp[0]; a.H[0] = s.H;
  a.w[1] = s.tw; a.x[1] = w.xp[1]; a.H[1] = s.Ht;
  a.sides = s.Ht ? 2 : 1;
  a.Np = up(s.N, TILE);
  a.meta = w.meta; a.lab = w.lab; a.inv_t = s.inv_t;
  a.stats = w.stats; a.zlab = w.zlab;
  a.lse = w.lse[0];
  a.rest = w.rest[0];
  a.dzt = w.dzt; a.words = w.words; a.low = w.low;
  a.kept = w.kept; a.kept_side = up(s.N, TILE) * w.words;
  return a;
}
template <int MODE, int NB, bool GATHER>
static int few_logits(const LogitArgs& a, const PackArgs& k, hipStream_t st, const char* what) {
  static uint64_t done = 0;
  const int64_t N = k.N;
  auto kern = few_kernel<MODE, NB, GATHER>;
  constexpr size_t lds = (size_t)few_slots<NB>() * few_stage<NB>();
  if (int rc = reserve_lds((const void*)kern, lds, done, what)) return rc;
  const int64_t items = up(a.v1 - a.v0, kFewWords) / kFewWords * (up(N, 32 * NB) / (32 * NB)) * a.sides;
  hipLaunchKernelGGL(kern, dim3((unsigned)(items + GATHER)), dim3(kFewThreads), lds, st, a, k);
  return check_launch(what);
}
template <int MODE, bool GATHER>
static int few_logits(const LogitArgs& a, const PackArgs& k, hipStream_t st, const char* what) {
  return k.N <= 32   ? few_logits<MODE, 1, GATHER>(a, k, st, what)
         : k.N <= 64 ? few_logits<MODE, 2, GATHER>(a, k, st, what)
                     : few_logits<MODE, 4, GATHER>(a, k, st, what);
}
template <int MODE>
static int logits(const LogitArgs& a, const PackArgs& k, const Sides& s, hipStream_t st, const char* what) {
  if constexpr (MODE != CE_GRAD) {
    if (few(s.N, s.V, s.Ht)) {
      // (a forward of up to 128 rows gathers them)
      if constexpr (MODE == CE_STATS) return few_logits<MODE, 4, false>(a, k, st, what);
      else return few_logits<MODE, false>(a, k, st, what);
    }
  }
  const bool stream = MODE != CE_GRAD && a.H[0] > BK && (a.sides < 2 || a.H[1] > BK);
  static uint64_t done[2] = {0, 0};
  // (a gradient's epilogue stages the tile where the next one's stages would go)
  auto kern = stream ? logits_kernel<MODE, MODE != CE_GRAD> : logits_kernel<MODE, false>;
  if (int rc = reserve_lds((const void*)kern, kLdsLogits, done[stream], what)) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)(cu_count() / 8 * 8)), dim3(NTHR), kLdsLogits, st, a);
  return check_launch(what);
}

// dW and dx of a piece of n words from its dz
struct Products {
  const Sides& s;
  const Ws& w;
  uint16_t *grad_x, *grad_w;
  int64_t panel;  // words of dz's panels
  hipStream_t st;
  const char* what;
  int piece(int64_t v0, int64_t n, bool add) const {
    static uint64_t done_w = 0, done_x = 0;
    if (int rc = reserve_lds((const void*)dw_kernel, kLdsLogits, done_w, what)) return rc;
    if (int rc = reserve_lds((const void*)dx_kernel, kLdsRing, done_x, what)) return rc;
    const int64_t tiles_h = up(s.H, TILE) / TILE;
    if (grad_w) {
      const DwArgs d = {w.dzt, panel, w.xp[0], up(s.N, TILE), s.H, n, w.meta, v0, grad_w + v0 * s.H,
                        w.top, w.low};
      hipLaunchKernelGGL(dw_kernel, dim3((unsigned)(up(n, TILE) / TILE * tiles_h)), dim3(NTHR),
                         kLdsLogits, st, d);
      if (int rc = check_launch(what)) return rc;
    }
    if (grad_x) {
      const DxArgs d = {w.dzt, panel, s.w + v0 * s.H, s.H, n, w.meta, w.part, add};
      // z tiles of rows: z rows H <= the parts' floats, and a split each of a tile that is not full
      const int64_t items = (w.part_floats / s.H / TILE + kMaxSplits) * tiles_h;
      hipLaunchKernelGGL(dx_kernel, dim3((unsigned)items), dim3(NTHR), kLdsRing, st, d);
      if (int rc = check_launch(what)) return rc;
    }
    return PLZ_OK;
  }
  int sum() const {
    if (!grad_x) return PLZ_OK;
    hipLaunchKernelGGL(dx_sum_kernel, dim3((unsigned)(up(s.N, 4) / 4 * (up(s.H, 256) / 256))),
                       dim3(256), 0, st, w.part, w.src, w.meta, (int)s.H, grad_x, w.x_top, w.x_low,
                       s.w);
    return check_launch(what);
  }
};

static FinishArgs finish_args(const Sides& s, const Ws& w, int64_t n) {
  FinishArgs f = {};
  f.dzt = w.dzt; f.words = w.words; f.n = n; f.Np = up(s.N, TILE);
  f.per = s.Ht ? kFinishKl : 1;
  f.stat_log = few(s.N, s.V, s.Ht) ? 7 : 8;
  f.meta = w.meta; f.lab = w.lab; f.stats = w.stats; f.zlab = w.zlab;
  f.lse[0] = w.lse[0]; f.lse[1] = w.lse[1]; f.apart = w.apart;
  f.rest[0] = w.rest[0]; f.rest[1] = w.rest[1];
  f.kept = w.kept; f.kept_side = f.Np * w.words;
  return f;
}
template <bool KL>
static int finish(const FinishArgs& f, hipStream_t st, const char* what) {
  hipLaunchKernelGGL(finish_kernel<KL>, dim3((unsigned)(f.Np / TILE * (up(f.n, TILE) / TILE) * (8 / f.per))),
                     dim3(256), 0, st, f);
  return check_launch(what);
}

// Workgroups of a join and the rows of each
static unsigned join_grid(int64_t N, int& rb_log) {
  rb_log = N >= 4096 ? 4 : N >= 512 ? 2 : 0;
  return (unsigned)((N + (1 << rb_log) - 1) >> rb_log);
}
// Each row's word whose dz is the greatest of the n words from v0 on, whose logits are kept
static int top(const Sides& s, const Ws& w, int64_t n, int64_t v0, const float* g, hipStream_t st,
               const char* what) {
  const bool halves = stat_words(s.N, s.V, s.Ht) < TILE;
  TopArgs t = {w.kept, up(s.N, TILE) * w.words, n, v0, halves, w.meta, {w.best[0], w.best[1]},
               {w.lse[0], w.lse[1]}, {w.rest[0], w.rest[1]}, g, w.top, w.low};
  if (w.x_most) {
    t.x_word = w.x_top; t.x_low = w.x_low; t.x_most = w.x_most;
  }
  hipLaunchKernelGGL(top_kernel, dim3((unsigned)((s.N + 3) / 4)), dim3(256), 0, st, t);
  return check_launch(what);
}

// The forward, and with grad_x or grad_w the gradients of its sum or mean (step)
template <bool KL, bool STEP>
static int forward(const Sides& s, int reduction, float* loss, float* lse, float* total,
                   uint16_t* grad_x, uint16_t* grad_w, void* ws, size_t ws_bytes, hipStream_t st,
                   const char* what) {
  if (int rc = check(s, KL, what)) return rc;
  PLZ_REQUIRE(s.N == 0 || (loss && lse), "%s: null pointer", what);
  const int use = STEP ? WS_STEP : WS_FWD;
  if (STEP) {
    PLZ_REQUIRE(reduction == PLZ_REDUCE_SUM || reduction == PLZ_REDUCE_MEAN, "%s: bad reduction %d",
                what, reduction);
    PLZ_REQUIRE(a16(grad_x) && a16(grad_w), "%s: gradients must be 16-byte aligned", what);
    if (!step_fits(s.N, s.V, s.H, s.Ht)) {
      set_error("%s: no rows, or more logits than a forward keeps", what);
      return PLZ_EUNSUPPORTED;
    }
  }
  Carve c{reinterpret_cast<char*>(ws)};
  const Ws w = carve(c, use, s.N, s.V, s.H, s.Ht, grad_x != nullptr);
  if (int rc = check_ws(ws, ws_bytes, c.used, what)) return rc;
  const int64_t Np = up(s.N, TILE), Vp = up(s.V, TILE);
  const int stat = stat_words(s.N, s.V, s.Ht);
  const Total sums = {loss, s.N, total};
  if (s.N == 0 && total) {
    hipLaunchKernelGGL(no_total_kernel, dim3(1), dim3(64), 0, st, total);
    return check_launch(what);
  }
  if (s.N > 0) {
    PackArgs p = pack_args(s, w);
    p.zero[0] = loss;
    p.zero[1] = lse;
    p.zero[2] = lse + s.N;
    if (KL) {
      p.zero[3] = lse + 2 * s.N;
      p.zero[4] = lse + 3 * s.N;
    }
    if (STEP) {
      p.reduction = reduction;
      p.grad_x = grad_x;
    }
    LogitArgs l = logit_args(s, w);
    l.planes = !KL ? 2 : STEP ? 4 : 5;
    // (dW reads the packed rows; few() holds for up to 128)
    const bool gather = s.N <= 128 && !grad_w;
    if (gather) {
      l.x[0] = s.x;
      l.x[1] = s.tx;
    } else if (int rc = pack(p, st, what)) {
      return rc;
    }
    for (int64_t v0 = 0; v0 < s.V; v0 += KL ? w.words : s.V) {
      l.v0 = v0;
      l.v1 = KL ? std::min(s.V, v0 + w.words) : s.V;
      l.tile0 = (int)(v0 / stat);
      constexpr int MODE = KL ? Z_KEEP : STEP ? CE_KEEP : CE_STATS;
      const int rc = gather ? few_logits<MODE, true>(l, p, st, what) : logits<MODE>(l, p, s, st, what);
      if (rc) return rc;
      if (KL && !STEP) {
        const CrossArgs x = {l.kept, l.kept_side, w.meta, w.stats, Np, l.v0, l.v1, stat < TILE};
        hipLaunchKernelGGL(cross_kernel, dim3((unsigned)(Np / TILE * (up(l.v1 - l.v0, TILE) / TILE) * 4)),
                           dim3(256), 0, st, x);
        if (int rc = check_launch(what)) return rc;
      }
    }
    JoinArgs j = {};
    j.stats = w.stats; j.zlab = w.zlab; j.meta = w.meta; j.src = w.src; j.lab = w.lab;
    j.Np = Np;
    j.tiles = (int)(up(s.V, stat) / stat);
    const unsigned joins = join_grid(s.N, j.rb_log);
    j.loss = loss;
    j.lse[0] = lse;
    j.lse[1] = lse + s.N;
    j.rest_out[0] = lse + (KL ? 2 : 1) * s.N;
    j.rest_out[1] = lse + 3 * s.N;
    j.lsep[0] = w.lse[0];
    j.lsep[1] = w.lse[1];
    j.rest[0] = w.rest[0];
    j.rest[1] = w.rest[1];
    j.apart = w.apart;
    j.best[0] = w.best[0];
    j.best[1] = w.best[1];
    j.low = KL ? nullptr : w.low;
    j.total = sums;
    hipLaunchKernelGGL(join_kernel<!KL ? JOIN_CE : STEP ? JOIN_LSE : JOIN_KL>,
                       dim3(joins), dim3(256), 0, st, j);
    if (int rc = check_launch(what)) return rc;
  }
  if (STEP && (KL || grad_x || grad_w)) {
    FinishArgs f = finish_args(s, w, s.V);
    f.loss = w.kl;
    if (KL && w.top)
      if (int rc = top(s, w, s.V, 0, nullptr, st, what)) return rc;
    if (int rc = finish<KL>(f, st, what)) return rc;
    if (KL) {
      hipLaunchKernelGGL(rows_kernel, dim3((unsigned)((s.N + 7) / 8)), dim3(256), 0, st, w.kl,
                         (int)(Vp / 32 / f.per), w.meta, w.src, Np, loss, sums);
      if (int rc = check_launch(what)) return rc;
    }
  }
  if (!STEP || (!grad_x && !grad_w)) return PLZ_OK;
  const Products prod = {s, w, grad_x, grad_w, Vp, st, what};
  if (int rc = prod.piece(0, s.V, false)) return rc;
  return prod.sum();
}

template <bool KL>
static int backward(const Sides& s, const float* lse, const float* grad, int reduction,
                    uint16_t* grad_x, uint16_t* grad_w, void* ws, size_t ws_bytes, hipStream_t st,
                    const char* what) {
  if (int rc = check(s, KL, what)) return rc;
  PLZ_REQUIRE(reduction == PLZ_REDUCE_NONE || reduction == PLZ_REDUCE_SUM || reduction == PLZ_REDUCE_MEAN,
              "%s: bad reduction %d", what, reduction);
  PLZ_REQUIRE(s.N == 0 || (lse && grad), "%s: null pointer", what);
  PLZ_REQUIRE(a16(grad_x) && a16(grad_w), "%s: gradients must be 16-byte aligned", what);
  if (!grad_x && !grad_w) return PLZ_OK;
  if (s.N == 0) {
    if (grad_w) zero_async(grad_w, (size_t)s.V * s.H * 2, st);
    return check_launch(what);
  }
  Carve c{reinterpret_cast<char*>(ws)};
  const Ws w = carve(c, WS_BWD, s.N, s.V, s.H, s.Ht, grad_x != nullptr);
  if (int rc = check_ws(ws, ws_bytes, c.used, what)) return rc;
  const int64_t words = w.words;
  PackArgs p = pack_args(s, w);
  p.grad = grad;
  p.reduction = reduction;
  if (reduction == PLZ_REDUCE_NONE) p.g = w.g;
  p.grad_x = grad_x;
  for (int k = 0; k < (KL ? 2 : 1); ++k) {
    p.lse_in[k] = lse + k * s.N;
    p.rest_in[k] = lse + ((KL ? 2 : 1) + k) * s.N;
    p.lse[k] = w.lse[k];
    p.rest[k] = w.rest[k];
  }
  if (int rc = pack(p, st, what)) return rc;
  LogitArgs l = logit_args(s, w);
  l.g = p.g;
  l.planes = KL ? 4 : 2;
  const Products prod = {s, w, grad_x, grad_w, words, st, what};
  for (int64_t v0 = 0; v0 < s.V; v0 += words) {
    l.v0 = v0;
    l.v1 = std::min(s.V, v0 + words);
    if (int rc = logits<KL ? Z_KEEP : CE_GRAD>(l, p, s, st, what)) return rc;
    if (KL) {
      if (w.top) {
        const int stat = stat_words(s.N, s.V, s.Ht);
        JoinArgs j = {};
        j.stats = w.stats; j.meta = w.meta; j.Np = l.Np;
        j.tiles = (int)(up(l.v1 - l.v0, stat) / stat);
        j.best[0] = w.best[0]; j.best[1] = w.best[1];
        const unsigned joins = join_grid(s.N, j.rb_log);
        hipLaunchKernelGGL(join_kernel<JOIN_BEST>, dim3(joins), dim3(256), 0, st, j);
        if (int rc = check_launch(what)) return rc;
        if (int rc = top(s, w, l.v1 - l.v0, l.v0, p.g, st, what)) return rc;
      }
      FinishArgs f = finish_args(s, w, l.v1 - l.v0);
      f.g = p.g;
      if (int rc = finish<true>(f, st, what)) return rc;
    }
    if (int rc = prod.piece(v0, l.v1 - v0, v0 > 0)) return rc;
  }
  return prod.sum();
}

static Sides ce_sides(const uint16_t* x, const uint16_t* w, const void* labels, int bytes,
                      int64_t ignore, int64_t N, int64_t V, int64_t H) {
  return Sides{x, w, nullptr, nullptr, labels, bytes == 8 ? KEY_INT64 : KEY_INT32, ignore, 1.f, N, V, H, 0};
}
static Sides kl_sides(const uint16_t* x, const uint16_t* w, const uint16_t* tx, const uint16_t* tw,
                      const uint8_t* mask, float inv_t, int64_t N, int64_t V, int64_t H, int64_t Ht) {
  return Sides{x, w, tx, tw, mask, mask ? KEY_MASK : KEY_NONE, 0, inv_t, N, V, H, Ht};
}

}  // namespace voc
}  // namespace plz

using namespace plz;
using namespace plz::voc;

extern "C" {

size_t plz_vocab_loss_workspace(int64_t N, int64_t V, int64_t H, int64_t H_teacher) {
  if (N < 0 || V < 1 || H < 8 || H_teacher < 0) return 0;
  Carve c{nullptr};
  carve(c, WS_FWD, N, V, H, H_teacher, false);
  return c.used;
}
size_t plz_vocab_loss_bwd_workspace(int64_t N, int64_t V, int64_t H, int64_t H_teacher, int grad_x) {
  if (N < 1 || V < 1 || H < 8 || H_teacher < 0) return 0;
  Carve c{nullptr};
  carve(c, WS_BWD, N, V, H, H_teacher, grad_x != 0);
  return c.used;
}
size_t plz_vocab_loss_step_workspace(int64_t N, int64_t V, int64_t H, int64_t H_teacher, int grad_x) {
  if (N < 1 || V < 1 || H < 8 || H_teacher < 0 || !step_fits(N, V, H, H_teacher)) return 0;
  Carve c{nullptr};
  carve(c, WS_STEP, N, V, H, H_teacher, grad_x != 0);
  return c.used;
}

int plz_linear_ce_fwd(const uint16_t* x, const uint16_t* w, const void* labels, int label_bytes,
                      int64_t ignore_index, float* loss, float* lse, float* total, void* workspace,
                      size_t workspace_bytes, int64_t N, int64_t V, int64_t H, void* stream) {
  PLZ_REQUIRE(label_bytes == 8 || label_bytes == 4, "plz_linear_ce_fwd: labels of 4 or 8 bytes expected");
  PLZ_REQUIRE(labels || N == 0, "plz_linear_ce_fwd: null pointer");
  return forward<false, false>(ce_sides(x, w, labels, label_bytes, ignore_index, N, V, H),
                               PLZ_REDUCE_NONE, loss, lse, total, nullptr, nullptr, workspace,
                               workspace_bytes, (hipStream_t)stream, "plz_linear_ce_fwd");
}
int plz_linear_ce_step(const uint16_t* x, const uint16_t* w, const void* labels, int label_bytes,
                       int64_t ignore_index, int reduction, float* loss, float* lse, float* total,
                       uint16_t* grad_x, uint16_t* grad_w, void* workspace, size_t workspace_bytes,
                       int64_t N, int64_t V, int64_t H, void* stream) {
  PLZ_REQUIRE(label_bytes == 8 || label_bytes == 4, "plz_linear_ce_step: labels of 4 or 8 bytes expected");
  PLZ_REQUIRE(labels || N == 0, "plz_linear_ce_step: null pointer");
  return forward<false, true>(ce_sides(x, w, labels, label_bytes, ignore_index, N, V, H), reduction,
                              loss, lse, total, grad_x, grad_w, workspace, workspace_bytes,
                              (hipStream_t)stream, "plz_linear_ce_step");
}
int plz_linear_ce_bwd(const uint16_t* x, const uint16_t* w, const void* labels, int label_bytes,
                      int64_t ignore_index, const float* lse, const float* grad, int reduction,
                      uint16_t* grad_x, uint16_t* grad_w, void* workspace, size_t workspace_bytes,
                      int64_t N, int64_t V, int64_t H, void* stream) {
  PLZ_REQUIRE(label_bytes == 8 || label_bytes == 4, "plz_linear_ce_bwd: labels of 4 or 8 bytes expected");
  PLZ_REQUIRE(labels || N == 0, "plz_linear_ce_bwd: null pointer");
  return backward<false>(ce_sides(x, w, labels, label_bytes, ignore_index, N, V, H), lse, grad,
                         reduction, grad_x, grad_w, workspace, workspace_bytes, (hipStream_t)stream,
                         "plz_linear_ce_bwd");
}
int plz_linear_kl_fwd(const uint16_t* x, const uint16_t* w, const uint16_t* teacher_x,
                      const uint16_t* teacher_w, const uint8_t* mask, float inv_temperature,
                      float* loss, float* lse, float* total, void* workspace, size_t workspace_bytes,
                      int64_t N, int64_t V, int64_t H, int64_t H_teacher, void* stream) {
  return forward<true, false>(
      kl_sides(x, w, teacher_x, teacher_w, mask, inv_temperature, N, V, H, H_teacher), PLZ_REDUCE_NONE,
      loss, lse, total, nullptr, nullptr, workspace, workspace_bytes, (hipStream_t)stream,
      "plz_linear_kl_fwd");
}
int plz_linear_kl_step(const uint16_t* x, const uint16_t* w, const uint16_t* teacher_x,
                       const uint16_t* teacher_w, const uint8_t* mask, float inv_temperature,
                       int reduction, float* loss, float* lse, float* total, uint16_t* grad_x,
                       uint16_t* grad_w, void* workspace, size_t workspace_bytes, int64_t N, int64_t V,
                       int64_t H, int64_t H_teacher, void* stream) {
  return forward<true, true>(
      kl_sides(x, w, teacher_x, teacher_w, mask, inv_temperature, N, V, H, H_teacher), reduction, loss,
      lse, total, grad_x, grad_w, workspace, workspace_bytes, (hipStream_t)stream, "plz_linear_kl_step");
}
int plz_linear_kl_bwd(const uint16_t* x, const uint16_t* w, const uint16_t* teacher_x,
                      const uint16_t* teacher_w, const uint8_t* mask, float inv_temperature,
                      const float* lse, const float* grad, int reduction, uint16_t* grad_x,
                      uint16_t* grad_w, void* workspace, size_t workspace_bytes, int64_t N, int64_t V,
                      int64_t H, int64_t H_teacher, void* stream) {
  return backward<true>(kl_sides(x, w, teacher_x, teacher_w, mask, inv_temperature, N, V, H, H_teacher),
                        lse, grad, reduction, grad_x, grad_w, workspace, workspace_bytes,
                        (hipStream_t)stream, "plz_linear_kl_bwd");
}

}  // extern "C"

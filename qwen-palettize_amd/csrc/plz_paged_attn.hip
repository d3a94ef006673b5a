// Attention of one new token a request over a paged key-value cache.
//
//   s_t = scale q[b, h] . K[t, h / G],  o[b, h] = sum_t softmax(s)_t V[t, h / G],
//   lse[b, h] = log sum_t exp(s_t),     t = 0 .. lens[b] - 1,  G = Hq / Hkv
// over the pages of request b (layouts: plz_paged.hip). A request without tokens gives o = 0 and
// lse = -inf; one whose length passes its block table, or that has a page number outside the
// cache among those it needs, gives NaN.
//
// Every cached value is needed once, for G heads: 2 G operations a byte, so the cache's bytes bound
// it, and the work is to keep enough of them in flight. A wave takes a tile of 32 tokens of one kv
// head straight from memory into the registers that feed the matrix instructions, no LDS between:
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, A = 16 tokens x 32 values of K, B = 16 heads. The K cache
//                 is stored in 8-value pieces, [D / 8][P][8], so that the 16 lanes of a piece read 256
//                 consecutive bytes (row-major K would give each of them 16 bytes of its own row, which
//                 takes the memory pipeline four times as long).
//   O^T += V^T P^T  the scores that a lane holds (head l % 16; tokens 4 g .. 4 g + 3 of both halves of
//                 the tile, g = l / 16) are already the B operand, if tokens are numbered that way. A
//                 lane loads the same 8 tokens of D / 16 consecutive values of V (16 lanes a row, row
//                 after row) and turns its 8 x D / 16 block in registers, one byte permute a word.
// The weights enter as two bf16 pieces (p = hi + lo, together 16 bits): one piece would be as large an
// error as the output's own rounding, and the matrix pipe has the room. The running maximum of a head
// moves only when a tile exceeds it by more than 2^8.
//
// The four waves of a workgroup share a run of tiles (plz_paged.h) and join through LDS; runs that
// share a request leave their maximum, sum and unscaled output in the workspace, and a second kernel
// joins those in the order of the runs.
#include "plz_paged.h"
#include "palettize_hip.h"

namespace plz {
namespace paged {

constexpr int NW = 4, NT = 64 * NW;  // waves, threads
constexpr int PARTS = 512;           // workgroups: two for each of 256 CUs
constexpr int HT = 16;               // heads a workgroup (columns of the matrix instruction)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct AttnArgs {
  const uint16_t *q, *kc, *vc;
  const int32_t *table, *lens;
  uint16_t* o;
  float *lse, *part;
  int2* shared;  // [parts]: of run w, {the request that it begins and does not finish or -1, its last run}
  int64_t ldq;
  int B, W, Hq, Hkv, G, tiles_h, parts, num_pages, shift;  // tiles_h = head tiles a kv head
  float scale_log2;
};

// one partial result: heads x D values, then the heads' maxima (log2 units) and sums
__host__ __device__ __forceinline__ int64_t part_floats(int heads, int D) {
  return ((int64_t)heads * (D + 2) + 3) / 4 * 4;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Tiles of the requests before request `b0` of this thread's share (k consecutive requests from
// threadIdx.x * k), and of all: inclusive sums over the workgroup.
__device__ __forceinline__ int scan_tiles(int v, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int u = __shfl_up(s, off);
    if (lane >= off) s += u;
  }
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + s - v;
}

template <int D>
__global__ __launch_bounds__(NT, D == 256 ? 1 : 2) void paged_attn_kernel(AttnArgs g) {
  constexpr int KS = D / 32, VEC = D / 16, VDW = VEC / 2;
  __shared__ int s_part[NW], s_empty[NW], s_at[2];
  __shared__ float s_m[NW][HT], s_l[NW][HT];
  __shared__ float s_o[NW][HT][D];
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = 1 << g.shift, cap = g.W << g.shift;

  // this workgroup's run of tiles, kv head and head tile; the head tiles of one run (the same K and
  // V) sit side by side on one XCD (id % 8)
  int w, hk, ht;
  {
    const int id = (int)blockIdx.x, per = 8 * g.tiles_h, pair = id / per * 8 + id % 8;
    ht = id % per / 8;
    w = pair / g.Hkv;
    hk = pair - w * g.Hkv;
  }
  if (w >= g.parts) return;  // the last eighth's padding
  const int h0 = ht * HT, nh = min(g.G - h0, HT);  // heads hk G + h0 .. + nh - 1
  const int per_thread = (g.B + NT - 1) / NT, b0 = threadIdx.x * per_thread;
  int mine = 0;
  bool none = false;
  for (int b = b0; b < min(b0 + per_thread, g.B); ++b) {
    const int n = tiles_of(g.lens[b], cap);
    mine += n;
    none |= n == 0;
  }
  if (lane == 0) s_empty[wave] = 0;
  if (__builtin_amdgcn_ballot_w64(none) != 0 && lane == 0) s_empty[wave] = 1;
  int total;
  int pre = scan_tiles(mine, s_part, total);
  const int runs = run_count(total, g.parts, NW);
  int open = -1, open_last = 0;  // the request that this run begins and does not finish, its last run
  if (w < runs) {
  const int r0 = run_begin(total, runs, w), r1 = run_begin(total, runs, w + 1);
  if (pre <= r0 && r0 < pre + mine) {
    int b = b0;
    for (;; ++b) {
      const int n = tiles_of(g.lens[b], cap);
      if (r0 < pre + n) break;
      pre += n;
    }
    s_at[0] = b;
    s_at[1] = pre;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(s_at[0]);
  int first = __builtin_amdgcn_readfirstlane(s_at[1]);  // request b's first tile among all
  const uint32_t koff = (uint32_t)(grp * P + col) * 16;
  const uint32_t voff = (uint32_t)(4 * grp * D + col * VEC) * 2;
  const int64_t page_bytes = (int64_t)D * 2 << g.shift;  // of one kv head

  for (;; ++b) {
    const int len = g.lens[b], n = tiles_of(len, cap);
    if (n == 0) continue;
    const int t0 = max(r0 - first, 0), t1 = min(r1 - first, n);
    const int32_t* row = g.table + (int64_t)b * g.W;

    // the heads' queries (columns past nh: zeros)
    bf16x8 qf[KS];
    {
      const uint16_t* qp = g.q + b * g.ldq + (int64_t)(hk * g.G + h0 + min(col, nh - 1)) * D + 8 * grp;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 x = *reinterpret_cast<const uint4*>(qp + 32 * s);
        if (col >= nh) x = make_uint4(0, 0, 0, 0);
        qf[s] = __builtin_bit_cast(bf16x8, x);
      }
    }
    f32x4 acc[VEC];
    float mrun, neg, lrun;  // maximum (log2 units), -maximum (0 for -inf), this lane's sum
    bool bad = false;

    u32x4 kr[2][KS];
    uint32_t vr[8][VDW];
    int pages = 0;  // lane 2 j + half: the page of half of this wave's j-th tile from jbase
    int jbase = 0;
    auto fetch_pages = [&](int j0) {
      jbase = j0;
      const int tile = t0 + wave + NW * (j0 + (lane >> 1));
      int tok = tile * TILE + (lane & 1) * 16;
      if (tok >= len) tok -= 16;  // a second half without tokens: the first one's page
      pages = 0;
      if (tile < t1) {
        pages = row[tok >> g.shift];
        if ((uint32_t)pages >= (uint32_t)g.num_pages) {
          bad = true;
          pages = 0;
        }
      }
      bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    };
    auto load_k = [&](int j) {
      const int tok = (t0 + wave + NW * j) * TILE;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int page = __builtin_amdgcn_readlane(pages, 2 * (j - jbase) + half);
        const int at = (tok + 16 * half) & (P - 1);
        const char* base = reinterpret_cast<const char*>(g.kc) +
                           ((int64_t)page * g.Hkv + hk) * page_bytes + (int64_t)at * 16;
#pragma unroll
        for (int s = 0; s < KS; ++s)
          kr[half][s] = *reinterpret_cast<const u32x4*>(base + (int64_t)s * 64 * P + koff);
      }
    };
    auto load_v = [&](int j) {
      const int tok = (t0 + wave + NW * j) * TILE;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int page = __builtin_amdgcn_readlane(pages, 2 * (j - jbase) + half);
        const int at = (tok + 16 * half) & (P - 1);
        const char* base = reinterpret_cast<const char*>(g.vc) +
                           ((int64_t)page * g.Hkv + hk) * page_bytes + (int64_t)at * D * 2;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t(&d)[VDW] = vr[4 * half + t];
          if constexpr (VDW == 2) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(base + t * D * 2 + voff);
            d[0] = x[0], d[1] = x[1];
          } else {
#pragma unroll
            for (int c = 0; c < VDW / 4; ++c) {
              const u32x4 x = *reinterpret_cast<const u32x4*>(base + t * D * 2 + voff + 16 * c);
#pragma unroll
              for (int i = 0; i < 4; ++i) d[4 * c + i] = x[i];
            }
          }
        }
      }
    };

    const int nj = (t1 - t0 - wave + NW - 1) / NW;  // this wave's tiles (<= 0: none)
    // once; where that leaves NaN (an infinite value times the two pieces of its weight, of which the
    // second may be 0 or of the other sign) again with the first pieces alone, for those outputs
    for (bool coarse = false;; coarse = true) {
    mrun = -INFINITY;
    neg = lrun = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = f32x4{};
    if (nj > 0) {
      fetch_pages(0);
      load_k(0);
      load_v(0);
    }
    for (int j = 0; j < nj; ++j) {
      const int left = len - (t0 + wave + NW * j) * TILE;  // tokens from the tile's first on
      f32x4 st[2] = {f32x4{}, f32x4{}};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          st[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[half][s]),
                                                             qf[s], st[half], 0, 0, 0);
      const bool more = j + 1 < nj;
      // V of this tile is still on its way: its pages are not needed again
      if (more) {
        if (j + 1 - jbase == 32) fetch_pages(j + 1);
        load_k(j + 1);
      }
      if (left < TILE) {  // the last tile of the request
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (16 * (e >> 2) + 4 * grp + (e & 3) >= left) {
            st[e >> 2][e & 3] = -INFINITY;
#pragma unroll
            for (int i = 0; i < VDW; ++i) vr[e][i] = 0;  // weight 0, but 0 x NaN is not
          }
      }
      float x[8], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = st[e >> 2][e & 3] * g.scale_log2;
        mx = fmaxf(mx, x[e]);
      }
      if (__builtin_amdgcn_ballot_w64(mx > mrun + 8.f) != 0) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mnew = mx > mrun + 8.f ? mx : mrun;
        const float alpha = mnew == mrun ? 1.f : exp2_fast(mrun - mnew);
        mrun = mnew;
        neg = mnew == -INFINITY ? 0.f : -mnew;
        lrun *= alpha;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= alpha;
      }
      u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = exp2_fast(x[e] + neg), p1 = exp2_fast(x[e + 1] + neg);
        lrun += p0 + p1;
        const uint32_t h = f2bf2(p0, p1);
        hi[e / 2] = h;
        lo[e / 2] = f2bf2(p0 - __builtin_bit_cast(float, h << 16),
                          p1 - __builtin_bit_cast(float, h & 0xffff0000u));
      }
      const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, lo);
#pragma unroll
      for (int i = 0; i < VDW; ++i) {
        u32x4 even, odd;  // values 2 i and 2 i + 1 of the 8 tokens
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          even[t] = perm(vr[2 * t + 1][i], vr[2 * t][i], 0x05040100u);
          odd[t] = perm(vr[2 * t + 1][i], vr[2 * t][i], 0x07060302u);
        }
        const bf16x8 ve = __builtin_bit_cast(bf16x8, even), vo = __builtin_bit_cast(bf16x8, odd);
        acc[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, ph, acc[2 * i], 0, 0, 0);
        acc[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, ph, acc[2 * i + 1], 0, 0, 0);
        if (!coarse) {
          acc[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, pl, acc[2 * i], 0, 0, 0);
          acc[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, pl, acc[2 * i + 1], 0, 0, 0);
        }
      }
      if (more) load_v(j + 1);
    }

    // the wave's results: value (4 grp + r) VEC + i of head col is acc[i][r]
    lrun += __shfl_xor(lrun, 16);
    lrun += __shfl_xor(lrun, 32);
    bool nan = false;
    if (col < nh) {
      if (grp == 0) {
        s_m[wave][col] = mrun;
        s_l[wave][col] = bad ? __builtin_nanf("") : lrun;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          f32x4* to = reinterpret_cast<f32x4*>(&s_o[wave][col][(4 * grp + r) * VEC + i]);
          f32x4 x = {acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
          if (coarse) {
            const f32x4 fine = *to;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = fine[c] == fine[c] ? fine[c] : x[c];
          }
          *to = x;
          const float any = x[0] + x[1] + x[2] + x[3];
          nan |= any != any;
        }
    }
    if (coarse || __builtin_amdgcn_ballot_w64(nan) == 0) break;
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == n;
    if (t0 == 0 && !whole) {
      open = b;
      open_last = run_of(total, runs, first + n - 1);
    }
    float* part = g.part + (((int64_t)(hk * g.tiles_h + ht) * g.parts + w) * 2 + (t0 == 0)) *
                               part_floats(min(g.G, HT), D);
    for (int e = threadIdx.x; e < nh * (D / 4); e += NT) {
      const int h = e / (D / 4), d = e % (D / 4) * 4;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) m = fmaxf(m, s_m[i][h]);
      const float ref = m == -INFINITY ? 0.f : m;
      f32x4 sum = {};
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float wt = exp2_fast(s_m[i][h] - ref);
        l += wt * s_l[i][h];
        sum += wt * *reinterpret_cast<const f32x4*>(&s_o[i][h][d]);
      }
      if (whole) {
        const float inv = 1.f / l;
        const int64_t at = (int64_t)b * g.Hq + hk * g.G + h0 + h;
        *reinterpret_cast<u32x2*>(g.o + at * D + d) =
            u32x2{f2bf2(sum[0] * inv, sum[1] * inv), f2bf2(sum[2] * inv, sum[3] * inv)};
        if (d == 0) g.lse[at] = (ref + log2f(l)) * kLn2;
      } else {
        if (d == 0) {
          part[nh * D + h] = m;
          part[nh * D + nh + h] = l;
        }
        *reinterpret_cast<f32x4*>(part + h * D + d) = sum;
      }
    }
    first += n;
    if (first >= r1) break;
    __syncthreads();  // the waves' results have been read
  }
  }
  if (hk == 0 && ht == 0 && threadIdx.x == 0) g.shared[w] = make_int2(open, open_last);

  // requests without tiles, spread over the runs
  int empty = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) empty |= s_empty[i];
  const int every = max(runs, 1);
  if (empty && w < every)
    for (int b = w + every * wave; b < g.B; b += every * NW) {
      const int len = g.lens[b];
      if (tiles_of(len, cap) != 0) continue;
      const float x = len <= 0 ? 0.f : __builtin_nanf("");
      const int64_t at = (int64_t)b * g.Hq + hk * g.G + h0;
      for (int e = lane; e < nh * (D / 4); e += 64)
        *reinterpret_cast<u32x2*>(g.o + at * D + 4 * e) = u32x2{f2bf2(x, x), f2bf2(x, x)};
      if (lane < nh) g.lse[at + lane] = len <= 0 ? -INFINITY : x;
    }
}

// A workgroup a (run, query head): the parts of the request that the run begins and does not finish
// (`shared`), in the order of their runs.
constexpr int JT = 256;
template <int D>
__global__ __launch_bounds__(JT) void paged_join_kernel(AttnArgs g) {
  constexpr int SETS = JT / (D / 4);  // threads a value: every SETS-th part each
  __shared__ float s_w[PARTS], s_l[PARTS], s_max[JT / 64];
  __shared__ f32x4 s_o[SETS][D / 4];
  const int w0 = blockIdx.x, h = blockIdx.y;
  const int2 open = g.shared[w0];
  const int b = open.x, count = open.y - w0 + 1;
  if (b < 0) return;
  const int hk = h / g.G, ht = (h - hk * g.G) / HT, hh = (h - hk * g.G) % HT;
  const int nh = min(g.G - ht * HT, HT);
  const int64_t size = part_floats(min(g.G, HT), D);
  const float* base = g.part + ((int64_t)(hk * g.tiles_h + ht) * g.parts + w0) * 2 * size;
  auto part = [&](int i) { return base + (2 * (int64_t)i + (i == 0)) * size; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < count; i += JT) {
    const float* p = part(i) + nh * D + hh;
    const float x = p[0];
    s_w[i] = x;
    s_l[i] = p[nh];
    m = fmaxf(m, x);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < JT / 64; ++i) m = fmaxf(m, s_max[i]);
  const float ref = m == -INFINITY ? 0.f : m;
  const int set = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
  f32x4 sum = {};
#pragma unroll 4
  for (int i = set; i < count; i += SETS)
    sum += exp2_fast(s_w[i] - ref) * *reinterpret_cast<const f32x4*>(part(i) + hh * D + 4 * c);
  s_o[set][c] = sum;
  __syncthreads();
  if (set != 0) return;
  float l = 0.f;
  for (int i = 0; i < count; ++i) l += exp2_fast(s_w[i] - ref) * s_l[i];
#pragma unroll
  for (int i = 1; i < SETS; ++i) sum += s_o[i][c];
  const float inv = 1.f / l;
  const int64_t at = (int64_t)b * g.Hq + h;
  *reinterpret_cast<u32x2*>(g.o + at * D + 4 * c) =
      u32x2{f2bf2(sum[0] * inv, sum[1] * inv), f2bf2(sum[2] * inv, sum[3] * inv)};
  if (c == 0) g.lse[at] = (ref + log2f(l)) * kLn2;
}

// workgroups a (kv head, head tile)
static int parts_of(int kv_heads, int head_tiles) {
  const int n = PARTS / (kv_heads * head_tiles);
  return n > 1 ? n : 1;
}

}  // namespace paged
}  // namespace plz

using namespace plz;
using namespace plz::paged;

extern "C" {

size_t plz_paged_attn_workspace(int64_t batch, int heads, int kv_heads, int head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || heads % kv_heads) return 0;
  const int G = heads / kv_heads, ht = (G + HT - 1) / HT;
  const size_t parts = (size_t)parts_of(kv_heads, ht);
  return parts * kv_heads * ht * 2 * part_floats(G < HT ? G : HT, head_dim) * sizeof(float) +
         parts * sizeof(int2);
}

int plz_paged_attn(const uint16_t* q, int64_t ld_q, const uint16_t* k_cache,
                   const uint16_t* v_cache, const int32_t* block_table, const int32_t* lens,
                   uint16_t* o, float* lse, void* workspace, size_t workspace_bytes, int64_t batch,
                   int64_t width, int heads, int kv_heads, int head_dim, int64_t num_pages,
                   int page_size, float scale, void* stream) {
  const char* const what = "plz_paged_attn";
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("%s: head_dim %d is not supported (64, 128 or 256)", what, head_dim);
    return PLZ_EUNSUPPORTED;
  }
  PLZ_REQUIRE(batch >= 0 && width >= 0 && heads > 0 && kv_heads > 0 && num_pages > 0,
              "%s: need batch, width >= 0 and heads, kv_heads and pages", what);
  PLZ_REQUIRE(heads % kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", what,
              heads, kv_heads);
  PLZ_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
              "%s: page_size must be a power of two of 16 to 1024, got %d", what, page_size);
  const int64_t lim = (int64_t)1 << 30;
  PLZ_REQUIRE(batch <= 65536 && width <= lim && num_pages <= lim && width * page_size <= lim &&
                  num_pages * page_size <= lim && heads <= 16384 &&
                  batch * width * page_size <= lim * TILE,
              "%s: batch goes up to 65536, heads to 16384, width x page_size and num_pages x "
              "page_size to 2^30, batch x width x page_size to 2^35", what);
  PLZ_REQUIRE(scale > 0.f, "%s: scale must be positive", what);
  if (batch == 0) return PLZ_OK;
  PLZ_REQUIRE(ld_q >= (int64_t)heads * head_dim && ld_q % 8 == 0,
              "%s: the row pitch of q is a multiple of 8 and at least the heads' width", what);
  PLZ_REQUIRE(q && k_cache && v_cache && (width == 0 || block_table) && lens && o && lse,
              "%s: null pointer", what);
  for (const void* p : {(const void*)q, (const void*)k_cache, (const void*)v_cache, (const void*)o})
    PLZ_REQUIRE(((uintptr_t)p & 15) == 0, "%s: q, the caches and o must be 16-byte aligned", what);
  const size_t need = plz_paged_attn_workspace(batch, heads, kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("%s: workspace of %zu bytes (16-byte aligned) required", what, need);
    return PLZ_EWORKSPACE;
  }
  AttnArgs g{q, k_cache, v_cache, block_table, lens, o, lse, (float*)workspace, nullptr, ld_q,
             (int)batch, (int)width, heads, kv_heads, heads / kv_heads, 0, 0, (int)num_pages, 0,
             scale * kLog2e};
  g.tiles_h = (g.G + HT - 1) / HT;
  g.parts = parts_of(kv_heads, g.tiles_h);
  g.shared = reinterpret_cast<int2*>(g.part + (int64_t)g.parts * kv_heads * g.tiles_h * 2 *
                                                  part_floats(g.G < HT ? g.G : HT, head_dim));
  while ((1 << g.shift) < page_size) ++g.shift;
  const int pairs = (g.parts * kv_heads + 7) / 8 * 8;
  const dim3 grid((unsigned)(pairs * g.tiles_h)), join((unsigned)g.parts, (unsigned)heads);
  auto launch = [&](auto kernel, dim3 blocks, int threads) {
    hipLaunchKernelGGL(kernel, blocks, dim3(threads), 0, (hipStream_t)stream, g);
    return check_launch(what);
  };
  int rc = head_dim == 64    ? launch(paged_attn_kernel<64>, grid, NT)
           : head_dim == 128 ? launch(paged_attn_kernel<128>, grid, NT)
                             : launch(paged_attn_kernel<256>, grid, NT);
  if (rc != PLZ_OK || g.parts == 1) return rc;
  return head_dim == 64    ? launch(paged_join_kernel<64>, join, JT)
         : head_dim == 128 ? launch(paged_join_kernel<128>, join, JT)
                           : launch(paged_join_kernel<256>, join, JT);
}

}  // extern "C"

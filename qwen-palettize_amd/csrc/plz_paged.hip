// The paged key-value cache of a decoding batch: who holds which page, and what goes into it.
//
// A cache is a pool of pages of P tokens (P a power of two, 16..1024). One layer's pages are
//   k_cache bf16 [num_pages, kv_heads, D / 8, P, 8]   value d of a token at [d / 8][token][d % 8]
//   v_cache bf16 [num_pages, kv_heads, P, D]
// (the order of K: plz_paged_attn.hip). Page w of request b, block_table[b, w], holds its tokens
// w P .. w P + P - 1; a token's slot is page * P + its offset. The pages that no request holds are
// a stack: free_pages[0 .. free_count).
//
//   paged_step        one scheduler step: pages handed back and taken, block table, slots and
//                     positions of the step's token rows, all from the requests' lengths
//   paged_rope_write  per-head RMSNorm and rotation of the rows' q and k, q written out, k and v
//                     written into their slots
#include "plz_paged.h"
#include "palettize_hip.h"

namespace plz {
namespace paged {

// ---- one scheduler step -------------------------------------------------------------------
// With L = lens[b], k = min(keep[b], L) tokens kept, a = new_tokens[b], pages(n) = ceil(n / P):
//   request b hands back its pages pages(k) .. pages(L) - 1 (pushed in order of b), then takes
//   want_b = pages(min(k + a, W P)) - pages(k) pages off the top, in order of b, while they last:
//   given_b = clamp(pool - sum_{b' < b} want_b', 0, want_b)
//   lens_out[b] = min(k + a, (pages(k) + given_b) P): what has room; token i of b, row starts[b] + i,
//   has position k + i and the slot of that position, -1 where there is no room.
// starts is the running sum of a, or b `each` where every request owns `each` rows (a at most that).
// Everything is a prefix sum over the requests, then independent work a page and a token, which find
// their request by binary search in the sums. One workgroup does it, a thread a request (in chunks of
// its threads, twice, for larger batches: the pages handed back have to be on the stack before any is
// taken): a step of 8 requests takes 3.0 us (5.1 with two passes for every batch, 1024 threads and sums
// by shuffles), of which 1 is the launch and the rest dependent memory accesses. More than 4096 token
// rows go to a second launch over the whole card (ONE_LAUNCH_ROWS).
struct StepArgs {
  const int32_t *lens, *keep, *add;
  int32_t *table, *stack;
  const int32_t* count;
  int32_t *slots, *pos, *starts, *lens_out, *count_out;
  int B, W, F, rows, shift;  // shift = log2 P
  int each;                  // rows a request owns, 0: as many as it has tokens
};

// The last i in [0, n) with start[i] <= j (start ascending, start[0] <= j)
__device__ __forceinline__ int find_row(const int* start, int n, int j) {
  int lo = 0;
  for (int len = n; len > 1;) {
    const int half = len >> 1;
    if (start[lo + half] <= j) {
      lo += half;
      len -= half;
    } else {
      len = half;
    }
  }
  return lo;
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Inclusive sums over the workgroup's threads of v and of u, u's at most cap (0 <= u <= cap <= 2^30, so
// that no sum overflows; v's do not by the entry point's limits). part: two words a wave.
template <int ST>
__device__ __forceinline__ void block_scan(int& v, int& u, int cap, int2* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  u = wave_scan(u, cap);
  __syncthreads();  // part's last readers are done
  if (lane == 63) part[wave] = make_int2(v, u);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w)
    if (w < wave) {
      v += part[w].x;
      u = min(u + part[w].y, cap);
    }
}

// TOKENS: the token rows too; else only the position of each request's first one (rows_kernel)
template <int ST, bool TOKENS>
__global__ __launch_bounds__(ST) void step_kernel(StepArgs g) {
  __shared__ int2 part[ST / 64];
  __shared__ int s_tok[ST], s_page[ST], s_keep[ST], s_hold[ST], s_len[ST], s_new[ST], s_last[2];
  const int tid = threadIdx.x, P1 = (1 << g.shift) - 1, cap = g.W << g.shift;
  const int count = clampi(*g.count, 0, g.F);
  const bool one = g.B <= ST;  // all requests at once
  int L = 0, k = 0, a = 0;
  auto load = [&](int b) {
    L = k = a = 0;
    if (b < g.B) {
      L = clampi(g.lens[b], 0, cap);
      k = g.keep ? clampi(g.keep[b], 0, L) : L;
      a = clampi(g.add[b], 0, g.each ? g.each : g.rows);
    }
  };
  // a request's rows: as many as its tokens, or those that it owns (rows = B each then)
  auto owned = [&](int b) { return g.each ? (b < g.B ? g.each : 0) : a; };
  // pages handed back
  int back = 0;  // by the chunks before
  int ends = 0;  // of a single chunk: the token rows up to this request's last
  for (int b0 = 0; b0 < g.B; b0 += ST) {
    const int nb = min(ST, g.B - b0);
    load(b0 + tid);
    const int hold = (k + P1) >> g.shift, n = ((L + P1) >> g.shift) - hold;
    int end = n;
    ends = owned(b0 + tid);
    block_scan<ST>(end, ends, g.rows, part);
    s_hold[tid] = hold;
    s_page[tid] = end - n;
    if (tid == ST - 1) s_last[0] = end;
    __syncthreads();
    const int total = s_last[0];
    for (int j = tid; j < total; j += ST) {
      const int r = find_row(s_page, nb, j), at = count + back + j;
      if (at < g.F) g.stack[at] = g.table[(int64_t)(b0 + r) * g.W + s_hold[r] + j - s_page[r]];
    }
    back += total;
    if (total > 0 || !one) __syncthreads();
  }
  const int pool = min(count + back, g.F);
  // pages taken, lengths, rows
  int tok0 = 0, want0 = 0;  // rows used and pages asked for by the chunks before
  for (int b0 = 0; b0 < g.B; b0 += ST) {
    const int b = b0 + tid, nb = min(ST, g.B - b0);
    int none = 0;
    if (!one) {
      load(b);
      ends = owned(b);
      block_scan<ST>(none, ends, g.rows, part);
      ends = min(tok0 + ends, g.rows);
    }
    // the row before: the previous thread's end
    s_tok[tid] = ends;
    __syncthreads();
    const int tok = tid ? s_tok[tid - 1] : tok0;
    a = min(a, ends - tok);
    const int hold = (k + P1) >> g.shift;
    const int full = (int)min((int64_t)k + a, (int64_t)cap);
    const int want = ((full + P1) >> g.shift) - hold;
    int want_end = want;
    none = 0;
    block_scan<ST>(want_end, none, 0, part);
    want_end += want0;
    const int before = want_end - want;
    const int given = clampi(pool - before, 0, want);
    const int len = min(full, (hold + given) << g.shift);
    s_tok[tid] = tok;  // block_scan's barriers: the ends have been read
    s_page[tid] = before;
    s_keep[tid] = k;
    s_hold[tid] = hold;
    s_len[tid] = len;
    s_new[tid] = a;
    if (tid == ST - 1) {
      s_last[0] = ends;
      s_last[1] = want_end;
    }
    if (b < g.B) {
      g.lens_out[b] = len;
      g.starts[b + 1] = ends;
      if (!TOKENS && ends > tok) g.pos[tok] = a > 0 ? k : -1;
    }
    __syncthreads();
    const int tok1 = s_last[0], want1 = s_last[1];
    for (int j = want0 + tid; j < min(want1, pool); j += ST) {
      const int r = find_row(s_page, nb, j);
      g.table[(int64_t)(b0 + r) * g.W + s_hold[r] + j - s_page[r]] = g.stack[pool - 1 - j];
    }
    if constexpr (TOKENS)
      for (int t = tok0 + tid; t < tok1; t += ST) {
        const int r = find_row(s_tok, nb, t), i = t - s_tok[r];
        const int pos = i < s_new[r] ? s_keep[r] + i : 0;
        int slot = -1;
        if (i < s_new[r] && pos < s_len[r]) {
          const int w = pos >> g.shift;
          const int page = w < s_hold[r] ? g.table[(int64_t)(b0 + r) * g.W + w]
                                         : g.stack[pool - 1 - (s_page[r] + w - s_hold[r])];
          if (page >= 0 && page < g.F) slot = (page << g.shift) + (pos & P1);
        }
        g.slots[t] = slot;
        g.pos[t] = pos;
      }
    tok0 = tok1;
    want0 = want1;
    if (!one) __syncthreads();
  }
  if constexpr (TOKENS)
    for (int t = tok0 + tid; t < g.rows; t += ST) {
      g.slots[t] = -1;
      g.pos[t] = 0;
    }
  if (tid == 0) {
    g.starts[0] = 0;
    *g.count_out = pool - min(pool, want0);
  }
}

// The token rows of a step whose table, lengths and starts step_kernel<TOKENS = false> has left, with
// the position of each request's first token in its row of pos.
constexpr int RT = 256, STAGED = 4096;
// 3300 rows 7.1 us in one launch and 7.6 in two, 5500 10.4 and 8.8, 7300 9.7 and 7.6, 27000 27 and 8.6: the
// one workgroup is bound by the instructions of its searches (four rows a thread side by side: no gain)
constexpr int64_t ONE_LAUNCH_ROWS = 4096;
__global__ __launch_bounds__(RT) void rows_kernel(StepArgs g) {
  __shared__ int s_starts[STAGED];
  const int P1 = (1 << g.shift) - 1, total = g.starts[g.B];
  const int* starts = g.starts;
  if (g.B <= STAGED) {
    for (int i = threadIdx.x; i < g.B; i += RT) s_starts[i] = g.starts[i];
    starts = s_starts;
  }
  __syncthreads();
  for (int t = blockIdx.x * RT + threadIdx.x; t < g.rows; t += gridDim.x * RT) {
    int slot = -1, pos = 0;
    if (t < total) {
      const int b = find_row(starts, g.B, t), i = t - starts[b];
      const int k = g.pos[t - i];  // -1: the request owns rows and has no token
      const bool live = k >= 0 && (!g.each || i < g.add[b]);
      pos = live ? k + i : 0;
      if (live && pos < g.lens_out[b]) {
        const int page = g.table[(int64_t)b * g.W + (pos >> g.shift)];
        if (page >= 0 && page < g.F) slot = (page << g.shift) + (pos & P1);
      }
      if (i == 0 && k >= 0) {
        g.slots[t] = slot;
        continue;
      }
    }
    g.slots[t] = slot;
    g.pos[t] = pos;
  }
}

// ---- norm, rotation, write --------------------------------------------------------------------
// A row (token t, head) of D values: n = x rsqrt(mean(x^2) + eps) w (w NULL: n = x), then
//   y_j = n_j cos[p, j] - n_{j + D/2} sin[p, j]  (j < D/2),   n_j cos[p, j] + n_{j - D/2} sin[p, j]
// at the token's position p, all in fp32 and rounded once to bf16 (the training layers' norm and
// rotation round the normalised and the weighted value too, as the modules that they stand for do:
// here there is no such module to match). D / 8 lanes a row, 8 values a lane; the partner of value
// j is in lane l ^ (D / 16). Bound by its bytes: 16384 tokens of 32/8 heads of 128 (407 MB read and
// written) take 77.2 us, 5.3 TB/s; a plain copy reaches 5.1. Up to 8 heads a workgroup share their tokens'
// sines (109 us with one), and the workgroups of one block of tokens run side by side on one XCD (86 with
// the blocks side by side: 58 MB of sines fetched again). 4 rows of a lane are in flight. K in its 8-value
// pieces is stored as fast as in rows would be. One token takes the 3 us of its memory latencies.
struct WriteArgs {
  const uint16_t *q, *k, *v, *qw, *kw;
  const float *cosv, *sinv;
  const int32_t *pos, *slots;
  uint16_t *q_out, *kc, *vc;
  int64_t T, ldq, ldk, ldv;
  int H, Hkv, max_pos, shift;
  int64_t slots_end;  // num_pages * P
  float eps;
  int each, groups;  // heads a workgroup, workgroups a block of tokens
};

// 16 bytes at base + 16 at, past the L2s' replacement order: whole rows that this kernel is done with
// (16384 tokens 80.1 -> 77.2 us; the 64-byte pieces of K are left to the L2 to put together)
__device__ __forceinline__ void store_nt(uint16_t* base, int64_t at, uint4 v) {
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(base) + at);
}

template <int LPR, int U>  // U rows of a lane in flight
__global__ __launch_bounds__(256) void rope_write_kernel(WriteArgs g) {
  constexpr int D = 8 * LPR, RPW = 64 / LPR, TB = 4 * RPW;  // tokens a workgroup
  const int lane = threadIdx.x & 63, l = lane % LPR;
  // the groups of heads of one block of tokens side by side on one XCD (id % 8), whose L2 then has the
  // tokens' sines and cosines for all of them
  const int seq = (int)(blockIdx.x >> 3), group = seq % g.groups;
  const int64_t t = ((int64_t)(seq / g.groups) * 8 + (blockIdx.x & 7)) * TB +
                    (threadIdx.x >> 6) * RPW + lane / LPR;
  if (t - (threadIdx.x >> 6) * RPW - lane / LPR >= g.T) return;  // the last eight blocks' padding
  const bool valid = t < g.T;
  const int64_t tt = valid ? t : 0;
  const int slot = g.slots[tt], p = g.pos[tt];
  const bool placed = p >= 0 && p < g.max_pos;  // else nothing is stored, and q is NaN
  const bool stored = valid && placed && slot >= 0 && slot < g.slots_end;
  const int64_t page = stored ? slot >> g.shift : 0;
  const int64_t at = stored ? slot & ((1 << g.shift) - 1) : 0;
  const int all = g.H + 2 * g.Hkv;  // heads: q's, k's, v's
  const int head0 = group * g.each, head1 = min(head0 + g.each, all);
  // the heads' sources and the row's sines are on their way together
  float c[8], s[8], w[8];
  const bool turns = head0 < g.H + g.Hkv;
  if (turns) {
    const int64_t row = (int64_t)(placed ? p : 0) * D + 8 * l;
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(g.cosv + row + j);
      const f32x4 b = *reinterpret_cast<const f32x4*>(g.sinv + row + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[j + e] = a[e];
        s[j + e] = l < LPR / 2 ? -b[e] : b[e];
      }
    }
  }
  const uint16_t* weight = head0 < g.H ? g.qw : g.kw;  // the one that w holds
  if (turns && weight) unpack8(reinterpret_cast<const uint4*>(weight)[l], w);
  for (int first = head0; first < head1; first += U) {
    uint4 xv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int head = min(first + i, head1 - 1);
      const uint16_t* src = head < g.H           ? g.q + tt * g.ldq + (int64_t)head * D
                            : head < g.H + g.Hkv ? g.k + tt * g.ldk + (int64_t)(head - g.H) * D
                                                 : g.v + tt * g.ldv + (int64_t)(head - g.H - g.Hkv) * D;
      xv[i] = reinterpret_cast<const uint4*>(src)[l];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int head = first + i;
      if (head >= head1) break;
      const int kind = head < g.H ? 0 : head < g.H + g.Hkv ? 1 : 2;
      const int h = kind == 0 ? head : kind == 1 ? head - g.H : head - g.H - g.Hkv;
      const int64_t block = page * g.Hkv + h;  // of D * P values
      if (kind == 2) {
        if (stored) store_nt(g.vc, ((block << g.shift) + at) * LPR + l, xv[i]);
        continue;
      }
      float f[8], o[8];
      unpack8(xv[i], f);
      const uint16_t* wt = kind == 0 ? g.qw : g.kw;
      if (wt) {
        if (wt != weight) {
          unpack8(reinterpret_cast<const uint4*>(wt)[l], w);
          weight = wt;
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off);
        const float r = rsqrtf(ss * (1.f / D) + g.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j] = f[j] * c[j] + __shfl_xor(f[j], LPR / 2) * s[j];
        if (!placed) o[j] = __builtin_nanf("");
      }
      const uint4 out = pack8(o);
      if (kind == 0) {
        if (valid) store_nt(g.q_out, (tt * g.H + h) * LPR + l, out);
      } else if (stored) {
        reinterpret_cast<uint4*>(g.kc)[((block * LPR + l) << g.shift) + at] = out;
      }
    }
  }
}

static bool a16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace paged
}  // namespace plz

using namespace plz;
using namespace plz::paged;

extern "C" {

int plz_paged_step(const int32_t* lens, const int32_t* keep, const int32_t* new_tokens,
                   int32_t* block_table, int32_t* free_pages, const int32_t* free_count,
                   int32_t* slots, int32_t* positions, int32_t* starts, int32_t* lens_out,
                   int32_t* free_count_out, int64_t batch, int64_t width, int64_t num_pages,
                   int64_t rows, int64_t rows_each, int page_size, void* stream) {
  PLZ_REQUIRE(batch >= 0 && width >= 0 && num_pages >= 0 && rows >= 0,
              "plz_paged_step: negative shape");
  PLZ_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
              "plz_paged_step: page_size must be a power of two of 16 to 1024, got %d", page_size);
  const int64_t lim = (int64_t)1 << 30;
  PLZ_REQUIRE(batch <= lim && width <= lim && num_pages <= lim && rows <= lim &&
                  batch * width <= lim && width * page_size <= lim &&
                  num_pages * page_size <= lim,
              "plz_paged_step: batch x width, width x page_size, num_pages x page_size and rows "
              "go up to 2^30");
  PLZ_REQUIRE(rows_each >= 0 && rows_each <= lim && (rows_each == 0 || rows == batch * rows_each),
              "plz_paged_step: with rows_each (%lld) there are batch x rows_each rows, got %lld",
              (long long)rows_each, (long long)rows);
  PLZ_REQUIRE(free_count && free_count_out && starts && (num_pages == 0 || free_pages) &&
                  (batch == 0 || (lens && new_tokens && lens_out)) &&
                  (batch * width == 0 || block_table) && (rows == 0 || (slots && positions)),
              "plz_paged_step: null pointer");
  PLZ_REQUIRE(batch == 0 || (lens_out != new_tokens && lens_out != keep),
              "plz_paged_step: lens_out may be lens, not new_tokens or keep");
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const StepArgs g{lens,  keep,   new_tokens, block_table,    free_pages, free_count, slots,
                   positions, starts, lens_out,   free_count_out, (int)batch, (int)width,
                   (int)num_pages, (int)rows, shift, (int)rows_each};
  auto launch = [&](auto kernel, int blocks, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 0, (hipStream_t)stream,
                       g);
    return check_launch("plz_paged_step");
  };
  if (rows <= ONE_LAUNCH_ROWS)
    return batch <= 256 && rows <= 256 ? launch(step_kernel<256, true>, 1, 256)
                                       : launch(step_kernel<1024, true>, 1, 1024);
  const int rc = launch(step_kernel<1024, false>, 1, 1024);
  const int64_t blocks = (rows + RT - 1) / RT;
  return rc != PLZ_OK ? rc : launch(rows_kernel, (int)(blocks < 2048 ? blocks : 2048), RT);
}

int plz_paged_rope_write(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t ld_q,
                         int64_t ld_k, int64_t ld_v, const uint16_t* q_weight,
                         const uint16_t* k_weight, const float* cos_table, const float* sin_table,
                         const int32_t* positions, const int32_t* slots, uint16_t* q_out,
                         uint16_t* k_cache, uint16_t* v_cache, int64_t tokens, int heads,
                         int kv_heads, int head_dim, int64_t max_positions, int64_t num_pages,
                         int page_size, float eps, void* stream) {
  const char* const what = "plz_paged_rope_write";
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("%s: head_dim %d is not supported (64, 128 or 256)", what, head_dim);
    return PLZ_EUNSUPPORTED;
  }
  PLZ_REQUIRE(tokens >= 0 && heads > 0 && kv_heads > 0 && max_positions > 0 && num_pages > 0,
              "%s: need tokens >= 0 and heads, kv_heads, positions and pages", what);
  PLZ_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
              "%s: page_size must be a power of two of 16 to 1024, got %d", what, page_size);
  const int64_t lim = (int64_t)1 << 30;
  PLZ_REQUIRE(tokens <= lim && heads <= 16384 && kv_heads <= 16384 && max_positions <= lim &&
                  num_pages <= lim && num_pages * page_size <= lim,
              "%s: tokens, positions and num_pages x page_size go up to 2^30, heads to 16384", what);
  if (tokens == 0) return PLZ_OK;
  PLZ_REQUIRE(ld_q >= (int64_t)heads * head_dim && ld_k >= (int64_t)kv_heads * head_dim &&
                  ld_v >= (int64_t)kv_heads * head_dim && ld_q % 8 == 0 && ld_k % 8 == 0 &&
                  ld_v % 8 == 0,
              "%s: a row pitch is a multiple of 8 and at least the heads' width", what);
  PLZ_REQUIRE((q_weight == nullptr) == (k_weight == nullptr),
              "%s: q_weight and k_weight go together", what);
  PLZ_REQUIRE(q && k && v && cos_table && sin_table && positions && slots && q_out && k_cache &&
                  v_cache,
              "%s: null pointer", what);
  PLZ_REQUIRE(a16(q) && a16(k) && a16(v) && a16(q_weight) && a16(k_weight) && a16(cos_table) &&
                  a16(sin_table) && a16(q_out) && a16(k_cache) && a16(v_cache),
              "%s: operands must be 16-byte aligned", what);
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  // Heads a workgroup: as many as leave it 1024 workgroups, up to 8 (its tokens' sines are read once)
  const int lpr = head_dim / 8, tb = 4 * (64 / lpr), all = heads + 2 * kv_heads;
  const int64_t blocks = (tokens + tb - 1) / tb;
  int each = 1;
  while (each < 8 && blocks * all >= 2048 * (int64_t)each) each *= 2;
  const int groups = (all + each - 1) / each;
  const WriteArgs g{q,     k,      v,   q_weight, k_weight, cos_table, sin_table, positions,
                    slots, q_out, k_cache, v_cache, tokens, ld_q, ld_k, ld_v,
                    heads, kv_heads, (int)max_positions, shift, num_pages * page_size, eps, each, groups};
  // a launch takes fewer than 2^32 threads
  PLZ_REQUIRE((blocks + 7) / 8 * 8 * groups < ((int64_t)1 << 24), "%s: too many tokens x heads", what);
  const dim3 grid((unsigned)((blocks + 7) / 8 * 8 * groups));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, g);
  };
  if (each < 4)
    lpr == 8    ? launch(rope_write_kernel<8, 1>)
    : lpr == 16 ? launch(rope_write_kernel<16, 1>)
                : launch(rope_write_kernel<32, 1>);
  else
    lpr == 8    ? launch(rope_write_kernel<8, 4>)
    : lpr == 16 ? launch(rope_write_kernel<16, 4>)
                : launch(rope_write_kernel<32, 4>);
  return check_launch(what);
}

}  // extern "C"

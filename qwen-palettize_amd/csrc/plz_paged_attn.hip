// Attention of one new token a request over a paged key-value cache.
//
//   s_t = scale q[b, h] . K[t, h / G],  o[b, h] = sum_t softmax(s)_t V[t, h / G],
//   lse[b, h] = log sum_t exp(s_t),     t = 0 .. lens[b] - 1,  G = Hq / Hkv
// over the pages of request b (layouts: plz_paged.hip). A request without tokens gives o = 0 and
// lse = -inf; one whose length passes its block table, or that has a page number outside the
// cache among those it needs, gives NaN.
//
// Every cached value is needed once, for G heads: 2 G operations a byte, so the cache's bytes bound
// it, and the work is to keep enough of them in flight: 64 requests of 8192 tokens (2.15 GB, 32/8 heads
// of 128) take 320 us, 6.7 TB/s (times here are of calls replayed from a graph, the second kernel among
// them); shorter batches add the 3-4 us before the first bytes arrive (lengths, block table, the first
// tiles of all waves at once) and the second launch. A wave takes a tile of 32 tokens of one kv head
// straight from memory into the registers that feed the matrix instructions, no LDS between:
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, A = 16 tokens x 32 values of K, B = 16 heads. The K cache
//                 is stored in 8-value pieces, [D / 8][P][8], so that the 16 lanes of a piece read 256
//                 consecutive bytes (row-major K would give each of them 16 bytes of its own row, which
//                 takes the memory pipeline four times as long).
//   O^T += V^T P^T  the scores that a lane holds (head l % 16; tokens 4 g .. 4 g + 3 of both halves of
//                 the tile, g = l / 16) are already the B operand, if tokens are numbered that way. A
//                 lane loads the same 8 tokens of D / 16 consecutive values of V (16 lanes a row, row
//                 after row) and turns its 8 x D / 16 block in registers, one byte permute a word.
// The weights enter as two bf16 pieces (p = hi + lo, together 16 bits): one piece would be as large an
// error as the output's own rounding, and the matrix pipe has the room (no difference in time). The
// running maximum of a head moves only when a tile exceeds it by more than 2^8. K and V are loaded past
// the L2s' replacement order, since with up to 16 heads a kv head nobody reads them again (359 -> 320 us;
// a batch of 74 MB that the last-level cache could hold from call to call 21.6 -> 21.7). With more heads
// the head tiles beside a workgroup on its XCD read them too, and may fetch them once more: 16 x 4096
// tokens, 4 kv heads with 20 heads each (134 MB), take 36 us, as many bytes of one request of 32768 with
// one head tile 28. Two tiles of V in flight a wave: no gain (28.0 -> 28.8); three waves a SIMD instead of
// two: 361 -> 385.
//
// Each wave has a run of tiles (plz_paged.h) and goes through its requests without a word to the
// others; the next requests' lengths, pages and queries are on their way while it is at this one. Only
// what a run has of a request that it does not have whole is joined: through LDS among the waves of a
// workgroup, through the workspace among workgroups, by a second kernel, both in the order of the runs.
// (256 ragged requests up to 1024 tokens: 59 us with one run a workgroup and a join after each request,
// 33.4 so.) The runs are dealt from the lengths by every wave for itself, a lane a request, in DPP sums.
#include "plz_paged.h"
#include "palettize_hip.h"

namespace plz {
namespace paged {

constexpr int NW = 4, NT = 64 * NW;  // waves, threads
constexpr int PARTS = 512;           // most workgroups: two for each of 256 CUs (parts_of)
constexpr int HT = 16;               // heads a workgroup (columns of the matrix instruction)
constexpr int ALONE = 512;           // tokens up to which a table's requests get waves of their own (own_waves)
constexpr int64_t ALONE_MOST = (int64_t)1 << 22;  // and how many of these at most: a launch has 2^32 threads
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct AttnArgs {
  const uint16_t *q, *kc, *vc;
  const int32_t *table, *lens;
  uint16_t* o;
  float *lse, *part;
  float2* part_ml;  // [Hq][place][parts]: a part's maximum (log2 units) and sum
  // What the second kernel joins: of workgroup w, {the request that it begins and does not finish or
  // -1, the workgroup that does}; or, where there are fewer requests than that (by_request), of request
  // b {the workgroup that begins it or -1, the one that ends it}.
  int2* open;
  int by_request;
  int alone;  // waves a request, when each has its own ones in one workgroup (no workspace, no second
              // kernel); 0: equal runs
  int64_t ldq;
  int B, W, Hq, Hkv, G, tiles_h, parts, num_pages, shift;  // tiles_h = head tiles a kv head
  float scale_log2;
};

// A wave's partial result: heads x D values, then the heads' maxima (log2 units) and sums
__host__ __device__ __forceinline__ int part_floats(int heads, int D) {
  return (heads * (D + 2) + 3) / 4 * 4;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// a value that is the same in every lane, where the compiler does not see it
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
constexpr int kNt = 2;  // buffer loads: nontemporal

// op over the four lanes of a column (l, l ^ 16, l ^ 32, l ^ 48), by swaps of rows and halves between two
// registers: no LDS, where shuffles go through it (32 ragged requests 20.3 -> 20.1 us, 48 with heads of 64
// 9.5 -> 9.3). The swapped pair goes through plain integers: a bit cast of a vector's element compiles into
// one of element 0.
template <class Op>
__device__ __forceinline__ float across(float v, Op op) {
  const auto pair = [&](auto both) {
    const uint32_t a = both[0], c = both[1];
    return op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, c));
  };
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  const uint32_t y = __builtin_bit_cast(uint32_t, pair(__builtin_amdgcn_permlane16_swap(x, x, false, false)));
  return pair(__builtin_amdgcn_permlane32_swap(y, y, false, false));
}

enum { HAS_CARRIED = 1, CARRIED_ENDS = 2, HAS_OPEN = 4 };  // a wave's parts

template <int D>
__global__ __launch_bounds__(NT, D == 256 ? 1 : 2) void paged_attn_kernel(AttnArgs g) {
  constexpr int KS = D / 32, VEC = D / 16, VDW = VEC / 2;
  extern __shared__ f32x4 s_res[];  // partial results, [wave][place]
  __shared__ int s_has[NW], s_req[NW][2], s_last[NW];
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = 1 << g.shift, cap = g.W << g.shift;

  // the head tiles of one workgroup number (the same K and V) sit side by side on one XCD (id % 8)
  int pair = (int)blockIdx.x, ht = 0;
  if (g.tiles_h > 1) {
    const int per = 8 * g.tiles_h, r = pair % per;
    ht = r >> 3;
    pair = pair / per * 8 + (r & 7);
  }
  const int w = pair / g.Hkv, hk = pair - w * g.Hkv;
  if (w >= g.parts) return;  // the last eighth's padding
  const int h0 = ht * HT, nh = min(g.G - h0, HT);  // heads hk G + h0 .. + nh - 1
  const int slot = part_floats(min(g.G, HT), D);
  float* const res = reinterpret_cast<float*>(s_res) + wave * 2 * slot;
  if (lane == 0) s_has[wave] = 0;

  // The requests that this wave shares with others (all of them, or its own one), its number among these
  // and how many they are: every request's tiles (a lane takes `each` consecutive ones) and their sums
  const int number = w * NW + wave, from = g.alone ? number / g.alone : 0;
  const int to = g.alone ? min(from + 1, g.B) : g.B;
  const int me = g.alone ? number % g.alone : number, waves = g.alone ? g.alone : g.parts * NW;
  const int each = (to - from + 63) >> 6;
  // Loads of lengths and pages have no branch around them: where paths of a divergent one meet, the
  // compiler takes the uniform values that meet there for divergent too, and with them all loops and
  // branches below (219 -> 203 registers, 256 ragged requests 34.1 -> 33.4 us).
  auto length = [&](int b) {
    const int n = g.lens[min(b, g.B - 1)];
    return b < to ? n : 0;
  };
  int win_at = from, win = 0;  // lane l: the length of request win_at + l
  int mine = 0;
  bool none = false;  // some request has no tiles
  for (int i = 0; i < each; ++i) {
    const int b = from + lane * each + i;
    win = length(b);
    const int n = tiles_of(win, cap);
    mine += n;
    none |= n == 0 && b < to;
  }
  none = __builtin_amdgcn_ballot_w64(none) != 0;
  int sum = wave_scan(mine);
  const int total = __builtin_amdgcn_readlane(sum, 63);
  const Deal runs = deal(total, waves);

  if (me < runs.runs) {
    const int r0 = run_begin(runs, me), r1 = run_begin(runs, me + 1);
    // the request that holds tile r0, and its first tile among all: the lane, then its requests
    auto holder = [&]() { return __builtin_ctzll(__builtin_amdgcn_ballot_w64(r0 < sum)); };
    int at = holder();
    int first = __builtin_amdgcn_readlane(sum - mine, at);
    if (each > 1) {
      for (win_at = from + at * each;; win_at += 64) {
        win = length(win_at + lane);
        mine = tiles_of(win, cap);
        sum = first + wave_scan(mine);
        const int end = __builtin_amdgcn_readlane(sum, 63);
        if (r0 < end || win_at + 64 >= to) break;
        first = end;
      }
      at = __builtin_amdgcn_ballot_w64(r0 < sum) ? holder() : 63;
      first = __builtin_amdgcn_readlane(sum - mine, at);
    }
    int b = win_at + at, len = __builtin_amdgcn_readlane(win, at), n = tiles_of(len, cap);
    const uint32_t koff = (uint32_t)(grp * P + col) * 16;
    const uint32_t voff = (uint32_t)(4 * grp * D + col * VEC) * 2;
    const int64_t page_bytes = (int64_t)D * 2 << g.shift;  // of one kv head

    // lane 2 j + half: the page of that half of tile t + j of request `req`, or of its last one
    auto fetch_pages = [&](int req, int t, int tokens, int tiles) {
      int tok = min(t + (lane >> 1), tiles - 1) * TILE + (lane & 1) * 16;
      if (tok >= tokens) tok -= 16;  // a second half without tokens: the first one's page
      return g.table[(int64_t)req * g.W + (max(tok, 0) >> g.shift)];
    };
    // pages outside the cache become page 0, which exists; whether there were any
    auto check_pages = [&](int& pages) {
      const bool out = (uint32_t)pages >= (uint32_t)g.num_pages;
      if (out) pages = 0;
      return __builtin_amdgcn_ballot_w64(out) != 0;
    };
    u32x4 kr[2][KS], qf[KS], qn[KS];
    uint32_t vr[8][VDW];
    auto load_q = [&](int req, u32x4(&to)[KS]) {  // columns past nh: the last head again
      const uint16_t* qp =
          g.q + req * g.ldq + (int64_t)(hk * g.G + h0 + min(col, nh - 1)) * D + 8 * grp;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        to[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s);
      }
    };
    // Buffer loads: a lane whose token does not exist (`tokens` in the request) gets an offset out of
    // range, reads zeros and moves nothing, so that what lies behind a request's last token costs nothing
    // and cannot reach the products (256 ragged requests up to 1024 36.2 -> 34.4 us; a branch around a
    // second half without tokens does that too, but a branch that may have issued loads makes the compiler
    // wait for all of them).
    auto page_rsrc = [&](const uint16_t* cache, int page) {
      const char* base = reinterpret_cast<const char*>(cache) + ((int64_t)page * g.Hkv + hk) * page_bytes;
      return make_rsrc(base, (uint32_t)page_bytes);
    };
    auto load_k = [&](int page0, int page1, int tile, int tokens) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const BufRsrc rsrc = page_rsrc(g.kc, uniform(half ? page1 : page0));
        const int first_tok = uniform(tile) * TILE + 16 * half;
        const uint32_t off = first_tok + col < tokens ? koff : kBufOob;
#pragma unroll
        for (int s = 0; s < KS; ++s)
          kr[half][s] = __builtin_amdgcn_raw_buffer_load_b128(
              rsrc, (int)off, s * 64 * P + (first_tok & (P - 1)) * 16, kNt);
      }
    };
    auto load_v = [&](int page0, int page1, int tile, int tokens) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const BufRsrc rsrc = page_rsrc(g.vc, uniform(half ? page1 : page0));
        const int first_tok = uniform(tile) * TILE + 16 * half, at = (first_tok & (P - 1)) * D * 2;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t(&d)[VDW] = vr[4 * half + t];
          const uint32_t off = first_tok + 4 * grp + t < tokens ? voff + t * D * 2 : kBufOob;
          if constexpr (VDW == 2) {
            const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)off, at, kNt);
            d[0] = x[0], d[1] = x[1];
          } else {
#pragma unroll
            for (int c = 0; c < VDW / 4; ++c) {
              const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off + 16 * c, at, kNt);
#pragma unroll
              for (int i = 0; i < 4; ++i) d[4 * c + i] = x[i];
            }
          }
        }
      }
    };
    f32x4 acc[VEC];
    // the tile's scores (log2 units) of this lane's 8 tokens; `left` tokens remain in the request
    auto scores = [&](float(&x)[8]) {
      f32x4 st[2] = {f32x4{}, f32x4{}};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) st[half] = mfma16(kr[half][s], qf[s], st[half]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = st[e >> 2][e & 3] * g.scale_log2;
    };
    auto mask = [&](float(&x)[8], int left) {
      if (left >= TILE) return;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (16 * (e >> 2) + 4 * grp + (e & 3) >= left) x[e] = -INFINITY;
    };
    // acc += V^T p for one or two pieces of p
    auto weigh = [&](u32x4 hi, u32x4 lo, bool both) {
#pragma unroll
      for (int i = 0; i < VDW; ++i) {
        u32x4 even, odd;  // values 2 i and 2 i + 1 of the 8 tokens
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          even[t] = perm(vr[2 * t + 1][i], vr[2 * t][i], 0x05040100u);
          odd[t] = perm(vr[2 * t + 1][i], vr[2 * t][i], 0x07060302u);
        }
        acc[2 * i] = mfma16(even, hi, acc[2 * i]);
        acc[2 * i + 1] = mfma16(odd, hi, acc[2 * i + 1]);
        if (both) {
          acc[2 * i] = mfma16(even, lo, acc[2 * i]);
          acc[2 * i + 1] = mfma16(odd, lo, acc[2 * i + 1]);
        }
      }
    };
    // value (4 grp + r) VEC + i of head col is acc[i][r]
    auto put = [&](float* to) {
      if (col < nh) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<f32x4*>(to + col * D + (4 * grp + r) * VEC + i) =
                f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
      }
    };

    int t = r0 - first, t0 = t, pos = r0;  // tile of the request, its first one here; tile among all
    int page_t = t, pages = fetch_pages(b, t, len, n);
    load_q(b, qf);
    bool bad_next = false;
    // The requests that the run goes on to: the next one, whose queries are loaded while this one is
    // worked on, and the one after it, whose pages are: loads come back in order, so pages asked for
    // behind a tile's K and V would hold up the tile that needs them until those are here.
    int b1 = 0, len1 = 0, n1 = 0, pages1 = 0, b2 = 0, len2 = 0, n2 = 0, pages2 = 0;
    auto find_after = [&](int req, int& at_req, int& tokens, int& tiles) {
      for (at_req = min(req + 1, to - 1);; ++at_req) {
        if (at_req >= win_at + 64) {
          win_at = at_req;
          win = length(win_at + lane);
        }
        tokens = __builtin_amdgcn_readlane(win, at_req - win_at);
        tiles = tiles_of(tokens, cap);
        if (tiles > 0 || at_req == to - 1) break;
      }
    };
    auto look_ahead = [&]() {
      if (first + n >= r1) return;
      load_q(b1, qn);
      if (first + n + n1 >= r1) return;
      find_after(b1, b2, len2, n2);
      pages2 = fetch_pages(b2, 0, len2, n2);
    };
    if (first + n < r1) {
      find_after(b, b1, len1, n1);
      pages1 = fetch_pages(b1, 0, len1, n1);
    }
    bool bad = check_pages(pages);
    {
      const int page0 = __builtin_amdgcn_readlane(pages, 0), page1 = __builtin_amdgcn_readlane(pages, 1);
      load_k(page0, page1, t, len);
      load_v(page0, page1, t, len);
    }
    look_ahead();
    float mrun = -INFINITY, neg = 0.f, lrun = 0.f;  // maximum (log2 units), -maximum or 0, own sum
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = f32x4{};

    for (;;) {
      float x[8];
      scores(x);
      // K of the next tile into the registers that are free now
      const bool more = pos + 1 < r1, same = t + 1 < n;
      int page0 = 0, page1 = 0, t_next = 0, l_next = len;
      if (more) {
        if (same) {
          t_next = t + 1;
          if (t_next - page_t == 32) {
            page_t = t_next;
            pages = fetch_pages(b, t_next, len, n);
            bad |= check_pages(pages);
          }
          page0 = __builtin_amdgcn_readlane(pages, 2 * (t_next - page_t));
          page1 = __builtin_amdgcn_readlane(pages, 2 * (t_next - page_t) + 1);
        } else {
          l_next = len1;
          bad_next = check_pages(pages1);
          page0 = __builtin_amdgcn_readlane(pages1, 0);
          page1 = __builtin_amdgcn_readlane(pages1, 1);
        }
        load_k(page0, page1, t_next, l_next);
      }
      mask(x, len - t * TILE);
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[e]);
      if (__builtin_amdgcn_ballot_w64(mx > mrun + 8.f) != 0) {
        mx = across(mx, [](float a, float b) { return fmaxf(a, b); });
        const float mnew = mx > mrun + 8.f ? mx : mrun;
        const float alpha = mnew == mrun ? 1.f : exp2_fast(mrun - mnew);
        mrun = mnew;
        neg = mnew == -INFINITY ? 0.f : -mnew;
        lrun *= alpha;
        if (t != t0) {  // nothing is in acc before the first tile
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] *= alpha;
        }
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
      weigh(hi, lo, true);
      if (more) load_v(page0, page1, t_next, l_next);
      ++pos;
      if (more && same) {
        t = t_next;
        continue;
      }

      // the request ends, here or for this run
      const bool carried = t0 > 0, whole = !carried && !same;
      lrun = across(lrun, [](float a, float b) { return a + b; });
      float any = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) any += acc[i][0] + acc[i][1] + acc[i][2] + acc[i][3];
      float* const left = res + place_of(carried) * slot;
      if (__builtin_amdgcn_ballot_w64(any != any && col < nh) != 0) {
        // An infinite value times the two pieces of its weight is NaN where the second is 0 or of the
        // other sign. For the outputs that are NaN, once more with the first pieces alone.
        put(left);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = f32x4{};
        for (int tt = t0; tt <= t; ++tt) {
          int again = fetch_pages(b, tt, len, n);
          check_pages(again);
          const int p0 = __builtin_amdgcn_readlane(again, 0), p1 = __builtin_amdgcn_readlane(again, 1);
          load_k(p0, p1, tt, len);
          load_v(p0, p1, tt, len);
          scores(x);
          mask(x, len - tt * TILE);
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            hi[e / 2] = f2bf2(exp2_fast(x[e] + neg), exp2_fast(x[e + 1] + neg));
          weigh(hi, hi, false);
        }
        if (col < nh) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float fine = left[col * D + (4 * grp + r) * VEC + i];
              if (fine == fine) acc[i][r] = fine;
            }
        }
        if (more) {
          load_k(page0, page1, t_next, l_next);
          load_v(page0, page1, t_next, l_next);
        }
      }
      if (bad) lrun = __builtin_nanf("");
      if (whole) {
        if (col < nh) {
          const float inv = 1.f / lrun;
          const int64_t at = (int64_t)b * g.Hq + hk * g.G + h0 + col;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint32_t out[VDW];
#pragma unroll
            for (int i = 0; i < VDW; ++i) out[i] = f2bf2(acc[2 * i][r] * inv, acc[2 * i + 1][r] * inv);
            uint16_t* const to = g.o + at * D + (4 * grp + r) * VEC;
            if constexpr (VDW == 2) {
              *reinterpret_cast<u32x2*>(to) = u32x2{out[0], out[1]};
            } else {
#pragma unroll
              for (int i = 0; i < VDW; i += 4)
                *reinterpret_cast<u32x4*>(to + 2 * i) = u32x4{out[i], out[i + 1], out[i + 2], out[i + 3]};
            }
          }
          if (grp == 0) g.lse[at] = ((mrun == -INFINITY ? 0.f : mrun) + log2f(lrun)) * kLn2;
        }
        if (g.by_request && lane == 0 && hk + ht == 0) g.open[b] = make_int2(-1, 0);
      } else {
        put(left);
        if (grp == 0 && col < nh) {
          left[nh * D + col] = mrun;
          left[nh * D + nh + col] = lrun;
        }
        if (lane == 0) {
          s_has[wave] |= carried ? HAS_CARRIED | (same ? 0 : CARRIED_ENDS) : HAS_OPEN;
          s_req[wave][place_of(carried)] = b;
          if (!carried) s_last[wave] = run_of(runs, first + n - 1) / NW;
        }
      }
      if (!more) break;
      first += n;
      b = b1, len = len1, n = n1, pages = pages1, bad = bad_next;
      b1 = b2, len1 = len2, n1 = n2, pages1 = pages2;
      page_t = t = t0 = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = qn[s];
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = f32x4{};
      mrun = -INFINITY;
      neg = lrun = 0.f;
      look_ahead();
    }
  }
  __syncthreads();

  // join the waves' parts of one request: a carried one (start -1), and what each wave begins
  int open = -1, open_last = 0;
  const int heads_max = min(g.G, HT);
  for (int start = -1; start < NW; ++start) {
    const int w0 = max(start, 0), place = start < 0 ? 0 : 1;
    if (!(s_has[w0] & (start < 0 ? HAS_CARRIED : HAS_OPEN))) continue;
    int count = 1;  // parts, of waves w0 .. w0 + count - 1
    bool ended = start < 0 && (s_has[0] & CARRIED_ENDS);
    while (!ended && w0 + count < NW && (s_has[w0 + count] & HAS_CARRIED))
      ended = s_has[w0 + count++] & CARRIED_ENDS;
    const bool whole = start >= 0 && ended;
    const int b = s_req[w0][place];
    if (start >= 0 && !ended) {
      open = b;
      open_last = s_last[w0];
    }
    if (g.by_request && threadIdx.x == 0 && hk + ht == 0 && start >= 0)
      g.open[b] = ended ? make_int2(-1, 0) : make_int2(w, s_last[w0]);
    // [kv head][head tile][workgroup][place][heads][D]
    float* part_out =
        g.part + (((int64_t)(hk * g.tiles_h + ht) * g.parts + w) * 2 + place) * (heads_max * D);
    for (int e = threadIdx.x; e < nh * (D / 4); e += NT) {
      const int h = e / (D / 4), d = e % (D / 4) * 4;
      const float* from = reinterpret_cast<const float*>(s_res) + (w0 * 2 + place) * slot;
      auto part = [&](int i) {  // the first one in its place, the others carried
        return i ? from + (2 * i - place) * slot : from;
      };
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < count; ++i) m = fmaxf(m, part(i)[nh * D + h]);
      const float ref = m == -INFINITY ? 0.f : m;
      f32x4 sum = {};
      for (int i = 0; i < count; ++i) {
        const float* p = part(i);
        const float wt = exp2_fast(p[nh * D + h] - ref);
        l += wt * p[nh * D + nh + h];
        sum += wt * *reinterpret_cast<const f32x4*>(p + h * D + d);
      }
      if (whole) {
        const float inv = 1.f / l;
        const int64_t at = (int64_t)b * g.Hq + hk * g.G + h0 + h;
        *reinterpret_cast<u32x2*>(g.o + at * D + d) =
            u32x2{f2bf2(sum[0] * inv, sum[1] * inv), f2bf2(sum[2] * inv, sum[3] * inv)};
        if (d == 0) g.lse[at] = (ref + log2f(l)) * kLn2;
      } else {
        *reinterpret_cast<f32x4*>(part_out + h * D + d) = sum;
        if (d == 0)
          g.part_ml[((int64_t)(hk * g.G + h0 + h) * 2 + place) * g.parts + w] = make_float2(m, l);
      }
    }
  }
  if (g.open && !g.by_request && threadIdx.x == 0 && hk + ht == 0)
    g.open[w] = make_int2(open, open_last);

  // requests without tiles, spread over all waves
  if (none)
    for (int b = from + me; b < to; b += waves) {
      const int len = g.lens[b];
      if (tiles_of(len, cap) != 0) continue;
      const float x = len <= 0 ? 0.f : __builtin_nanf("");
      const int64_t at = (int64_t)b * g.Hq + hk * g.G + h0;
      for (int e = lane; e < nh * (D / 4); e += 64)
        *reinterpret_cast<u32x2*>(g.o + at * D + 4 * e) = u32x2{f2bf2(x, x), f2bf2(x, x)};
      if (lane < nh) g.lse[at + lane] = len <= 0 ? -INFINITY : x;
      if (g.by_request && lane == 0 && hk + ht == 0) g.open[b] = make_int2(-1, 0);
    }
}

// A workgroup an entry of `open` and a query head: the parts of a request in the order of their runs.
constexpr int JT = 128;
template <int D>
__global__ __launch_bounds__(JT) void paged_join_kernel(AttnArgs g) {
  constexpr int SETS = JT / (D / 4);  // threads a value: every SETS-th part each
  constexpr int EACH = (PARTS + JT - 1) / JT, AHEAD = 8;
  __shared__ float2 s_ml[EACH * JT];
  __shared__ float s_max[JT / 64], s_l[SETS];
  __shared__ f32x4 s_o[SETS][D / 4];
  const int h = blockIdx.y;
  const int2 open = g.open[blockIdx.x];
  const int b = g.by_request ? blockIdx.x : open.x, w0 = g.by_request ? open.x : blockIdx.x;
  if (open.x < 0) return;
  const int count = open.y - w0 + 1;
  const float2* ml = g.part_ml + (int64_t)h * 2 * g.parts;
  float2 x[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int w = min(w0 + (int)threadIdx.x + k * JT, g.parts - 1);
    x[k] = ml[w == w0 ? g.parts + w : w];
  }
  const int hk = h / g.G, ht = (h - hk * g.G) / HT, hh = (h - hk * g.G) % HT;
  const int size = min(g.G, HT) * D, set = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
  const float* base =
      g.part + ((int64_t)(hk * g.tiles_h + ht) * g.parts + w0) * 2 * size + hh * D + 4 * c;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int i = threadIdx.x + k * JT;
    s_ml[i] = x[k];
    if (i < count) m = fmaxf(m, x[k].x);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  f32x4 sum = {};
  float l = 0.f, ref = 0.f;
  for (int i0 = 0; i0 < count; i0 += SETS * AHEAD) {
    f32x4 v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = min(i0 + k * SETS + set, count - 1);
      v[k] = *reinterpret_cast<const f32x4*>(base + (int64_t)(2 * i + (i == 0)) * size);
    }
    if (i0 == 0) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < JT / 64; ++k) m = fmaxf(m, s_max[k]);
      ref = m == -INFINITY ? 0.f : m;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * SETS + set;
      if (i < count) {
        const float2 p = s_ml[i];
        const float wt = exp2_fast(p.x - ref);
        l += wt * p.y;
        sum += wt * v[k];
      }
    }
  }
  s_o[set][c] = sum;
  if (c == 0) s_l[set] = l;
  __syncthreads();
  if (set != 0) return;
#pragma unroll
  for (int i = 1; i < SETS; ++i) {
    sum += s_o[i][c];
    l += s_l[i];
  }
  const float inv = 1.f / l;
  const int64_t at = (int64_t)b * g.Hq + h;
  *reinterpret_cast<u32x2*>(g.o + at * D + 4 * c) =
      u32x2{f2bf2(sum[0] * inv, sum[1] * inv), f2bf2(sum[2] * inv, sum[3] * inv)};
  if (c == 0) g.lse[at] = (ref + log2f(l)) * kLn2;
}

// Waves of its own for every request (and kv head, head tile) instead of equal runs, by the most tokens
// that its table can hold: one launch and no workspace, and a call that the host bounds saves another 4 us
// by the launch. Four, two or one, so that all workgroups have their place at once if they can;
// short ones get one wave rather than two, whose start and join cost more than their tiles; what takes
// several rounds even so pays up to 320 tokens. 0: equal runs. 32/8 heads of 128, in us, equal runs / 1 / 2 / 4:
//    50 tokens: B 16 7.1 5.2 5.7 5.1, B 96 9.8 6.7 8.0 9.8, B 256 14.4 12.3 16.4 21.0, ragged 13.4 7.9 11.4 16.6
//   200 tokens: B 16 9.5 12.7 10.1 7.3, B 96 23.4 17.1 18.1 19.0, ragged 11.8 11.6 10.0 11.3,
//               B 256 38 36 39 40, ragged 18.2 14.7 16.9 21.5
//   500 tokens: B 16 12.5 25.3 16.4 10.8, B 64 26.0 29.4 25.1 24.3, B 192 ragged 21.3 26.2 22.0 22.6,
//               B 256 ragged 26.0 27.1 27.1 28.2;   1000 tokens: B 1 8.7, 14.4 with four, B 256 168 and 165
// 1024 of 20 to 200 tokens: one 3 to 14% faster than equal runs. Heads of 64 and 256 are alike, with more
// and fewer workgroups in place: 128 requests of 200 tokens 18.0 13.3 12.9 15.4, 64 27.6 27.8 21.6 25.4.
static int own_waves(int64_t batch, int64_t width, int64_t page_size, int64_t kv_heads, int64_t tiles,
                     int D) {
  const int64_t longest = width * page_size;
  if (longest > ALONE || batch > ALONE_MOST || batch * kv_heads * tiles > ALONE_MOST) return 0;
  const int64_t all = batch * kv_heads * tiles, resident = D == 64 ? 768 : D == 128 ? 512 : 256;
  if (all <= resident) return 4;
  if (all <= 2 * resident) return longest * D <= 128 * 128 ? 1 : 2;
  return longest <= 320 ? 1 : 0;
}
// Workgroups a (kv head, head tile): two a CU in all, one where a part is large (more than 1024 values:
// writing and joining them costs more than the second workgroup's loads bring) or a workgroup takes the
// whole CU's registers (heads of 256). Two and one: 16 x 4096 tokens, 4 kv heads of 128 with 20 heads
// each 37.0 and 36.1 us (ragged, 32 up to 4096 and 8 heads each, so parts of 1024: 15.7 and 15.4); 8 kv
// heads of 256 with 4 heads each, 32 x 2048, 92.4 and 85.6; small parts, 32 ragged up to 4096 20.1 and 21.6.
static int parts_of(int kv_heads, int G, int D) {
  const int heads = G < HT ? G : HT, tiles = (G + HT - 1) / HT;
  const int n = (D == 256 || heads * D > 1024 ? PARTS / 2 : PARTS) / (kv_heads * tiles);
  return n > 1 ? n : 1;
}
template <int D>
static int launch_paged_attn(const AttnArgs& g, hipStream_t stream, const char* what) {
  // LDS: two places a wave; past 64 KB (16 heads of 128 values) the kernel asks for the most it can use
  const size_t lds = (size_t)NW * 2 * part_floats(g.G < HT ? g.G : HT, D) * sizeof(float);
  static uint64_t lds_done = 0;
  if (lds > 48 * 1024) {
    const int rc = reserve_lds((const void*)paged_attn_kernel<D>,
                               (size_t)NW * 2 * part_floats(HT, D) * sizeof(float), lds_done, what);
    if (rc != PLZ_OK) return rc;
  }
  hipLaunchKernelGGL(paged_attn_kernel<D>,
                     dim3((unsigned)(((int64_t)g.parts * g.Hkv + 7) / 8 * 8 * g.tiles_h)), dim3(NT), lds,
                     stream, g);
  const int rc = check_launch(what);
  if (rc != PLZ_OK || g.alone || g.parts == 1) return rc;
  hipLaunchKernelGGL(paged_join_kernel<D>,
                     dim3((unsigned)(g.by_request ? g.B : g.parts), (unsigned)g.Hq), dim3(JT), 0, stream,
                     g);
  return check_launch(what);
}

}  // namespace paged
}  // namespace plz

using namespace plz;
using namespace plz::paged;

extern "C" {

size_t plz_paged_attn_workspace(int64_t batch, int64_t width, int page_size, int heads, int kv_heads,
                                int head_dim) {
  if (batch <= 0 || width < 0 || page_size <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
      heads % kv_heads)
    return 0;
  const int G = heads / kv_heads, ht = (G + HT - 1) / HT;
  if (own_waves(batch, width, page_size, kv_heads, ht, head_dim)) return 0;
  const size_t parts = (size_t)parts_of(kv_heads, G, head_dim);
  return parts * kv_heads * ht * 2 * (G < HT ? G : HT) * head_dim * sizeof(float) +
         parts * heads * 2 * sizeof(float2) + parts * sizeof(int2);
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
  const size_t need =
      plz_paged_attn_workspace(batch, width, page_size, heads, kv_heads, head_dim);
  if (need == 0) workspace = nullptr;
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("%s: workspace of %zu bytes (16-byte aligned) required", what, need);
    return PLZ_EWORKSPACE;
  }
  AttnArgs g{q, k_cache, v_cache, block_table, lens, o, lse, (float*)workspace, nullptr, nullptr, 0, 0, ld_q,
             (int)batch, (int)width, heads, kv_heads, heads / kv_heads, 0, 0, (int)num_pages, 0,
             scale * kLog2e};
  g.tiles_h = (g.G + HT - 1) / HT;
  g.parts = parts_of(kv_heads, g.G, head_dim);
  if (need == 0) {
    g.alone = own_waves(batch, width, page_size, kv_heads, g.tiles_h, head_dim);
    g.parts = (g.B * g.alone + NW - 1) / NW;
  } else {
    g.part_ml = reinterpret_cast<float2*>(
        g.part + (int64_t)g.parts * kv_heads * g.tiles_h * 2 * (g.G < HT ? g.G : HT) * head_dim);
    g.open = reinterpret_cast<int2*>(g.part_ml + (int64_t)g.parts * heads * 2);
    g.by_request = batch < g.parts;
  }
  while ((1 << g.shift) < page_size) ++g.shift;
  return head_dim == 64    ? launch_paged_attn<64>(g, (hipStream_t)stream, what)
         : head_dim == 128 ? launch_paged_attn<128>(g, (hipStream_t)stream, what)
                           : launch_paged_attn<256>(g, (hipStream_t)stream, what);
}

}  // extern "C"

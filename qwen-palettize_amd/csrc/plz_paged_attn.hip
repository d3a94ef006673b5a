// Attention of one new token a request over a paged key-value cache.
//
//   s_t = scale q[b, h] . K[t, h / G],  o[b, h] = sum_t softmax(s)_t V[t, h / G],
//   lse[b, h] = log sum_t exp(s_t),     t = 0 .. lens[b] - 1,  G = Hq / Hkv
// over the pages of request b (layouts: plz_paged.hip). A request without tokens gives o = 0 and
// lse = -inf; one whose length passes its block table, or that has a page number outside the
// cache among those it needs, gives NaN.
//
// A workgroup a (request, query head); a wave takes every fourth token, its lanes D / 64 values
// each, with the running max and sum of the softmax; the four waves are joined through LDS.
#include "plz_common.h"
#include "palettize_hip.h"

namespace plz {
namespace paged {

template <int D>
__global__ __launch_bounds__(256) void paged_attn_kernel(
    const uint16_t* __restrict__ q, int64_t ldq, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, const int32_t* __restrict__ table,
    const int32_t* __restrict__ lens, uint16_t* __restrict__ o, float* __restrict__ lse, int W,
    int Hq, int Hkv, int num_pages, int shift, float scale) {
  constexpr int E = D / 64;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  __shared__ int s_bad;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x, h = blockIdx.y, hk = h / (Hq / Hkv), P = 1 << shift;
  const int n = max(lens[b], 0), cap = W << shift;
  if (threadIdx.x == 0) s_bad = n > cap;
  __syncthreads();
  float qv[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = bf2f(q[b * ldq + (int64_t)h * D + E * lane + e]) * scale;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = wave; t < min(n, cap); t += 4) {
    const int page = table[(int64_t)b * W + (t >> shift)], at = t & (P - 1);
    if (page < 0 || page >= num_pages) {
      s_bad = 1;
      break;
    }
    const int64_t base = ((int64_t)page * Hkv + hk) * D * P;
    float s = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = E * lane + e;
      s += qv[e] * bf2f(kc[base + ((int64_t)(d >> 3) * P + at) * 8 + (d & 7)]);
      v[e] = bf2f(vc[base + (int64_t)at * D + d]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __expf(m - ref), p = __expf(s - ref);
    l = l * alpha + p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * alpha + p * v[e];
    m = mn;
  }
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[wave][E * lane + e] = acc[e];
  __syncthreads();
  const float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float w[4], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = __expf(s_m[i] - ref);
    sum += w[i] * s_l[i];
  }
  for (int d = threadIdx.x; d < D; d += 256) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x += w[i] * s_o[i][d];
    x = s_bad ? __builtin_nanf("") : n == 0 ? 0.f : x / sum;
    o[((int64_t)b * Hq + h) * D + d] = (uint16_t)f2bf(x);
  }
  if (threadIdx.x == 0)
    lse[(int64_t)b * Hq + h] = s_bad ? __builtin_nanf("") : n == 0 ? -INFINITY : ref + logf(sum);
}

}  // namespace paged
}  // namespace plz

using namespace plz;
using namespace plz::paged;

extern "C" {

size_t plz_paged_attn_workspace(int64_t batch, int heads, int kv_heads, int head_dim) {
  (void)batch, (void)heads, (void)kv_heads, (void)head_dim;
  return 0;
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
                  num_pages * page_size <= lim && heads <= 16384,
              "%s: batch goes up to 65536, heads to 16384, width x page_size and num_pages x "
              "page_size to 2^30", what);
  PLZ_REQUIRE(scale > 0.f, "%s: scale must be positive", what);
  if (batch == 0) return PLZ_OK;
  PLZ_REQUIRE(ld_q >= (int64_t)heads * head_dim && ld_q % 8 == 0,
              "%s: the row pitch of q is a multiple of 8 and at least the heads' width", what);
  PLZ_REQUIRE(q && k_cache && v_cache && (width == 0 || block_table) && lens && o && lse,
              "%s: null pointer", what);
  for (const void* p : {(const void*)q, (const void*)k_cache, (const void*)v_cache, (const void*)o})
    PLZ_REQUIRE(((uintptr_t)p & 15) == 0, "%s: q, the caches and o must be 16-byte aligned", what);
  (void)workspace, (void)workspace_bytes;
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const dim3 grid((unsigned)batch, (unsigned)heads);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, q, ld_q, k_cache, v_cache,
                       block_table, lens, o, lse, (int)width, heads, kv_heads, (int)num_pages,
                       shift, scale);
  };
  if (head_dim == 64)
    launch(paged_attn_kernel<64>);
  else if (head_dim == 128)
    launch(paged_attn_kernel<128>);
  else
    launch(paged_attn_kernel<256>);
  return check_launch(what);
}

}  // extern "C"

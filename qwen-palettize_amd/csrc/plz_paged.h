// How a batch's cached tokens are dealt to the waves of plz_paged_attn.hip (plain integer rules, checked
// on the host), and the sums over a wave's lanes that the paged kernels share.
#pragma once
#include <stdint.h>

#include "plz_common.h"

namespace plz {
namespace paged {

constexpr int TILE = 32;  // tokens a wave takes at a time

// Tiles of a request: its tokens in TILEs; none for an empty one and for one whose length passes its
// block table (cap tokens), which is answered with NaN.
__host__ __device__ __forceinline__ int tiles_of(int len, int cap) {
  return len <= 0 || len > cap ? 0 : (len + TILE - 1) / TILE;
}

// The tiles of all requests, one behind the other (`total` of them), are cut into runs of equal length
// (the first `rem` one tile longer), one a wave: a long request is shared by many waves, a wave takes
// several short ones. Runs are numbered through the workgroups, `waves` in each.
struct Deal {
  int runs, q, rem;
};
__host__ __device__ __forceinline__ Deal deal(int total, int most) {
  const int runs = total < most ? total : most;
  const int q = runs > 0 ? total / runs : 0;
  return Deal{runs, q, total - q * runs};
}
__host__ __device__ __forceinline__ int run_begin(Deal d, int i) {
  return i * d.q + (i < d.rem ? i : d.rem);
}
// the run that holds tile p
__host__ __device__ __forceinline__ int run_of(Deal d, int p) {
  const int longer = d.rem * (d.q + 1);
  return p < longer ? p / (d.q + 1) : d.rem + (p - longer) / d.q;
}

// What a run has of a request: from tile 0 or from later on (CARRIED, then it is the run's first), to
// its last tile or not. Parts that are not whole are left for others to join: the part of a carried
// request in place 0, that of one which begins here and ends elsewhere in place 1.
__host__ __device__ __forceinline__ int place_of(bool carried) { return carried ? 0 : 1; }


// Inclusive sum of v over the wave's lanes, in DPP moves (rows of 16, then rows 0 and 2 into 1 and 3,
// then the lower half's sum into the upper): no LDS, where shuffles go through it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_0(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_or_0<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += dpp_or_0<0x112, 0xF>(v);
  v += dpp_or_0<0x114, 0xF>(v);
  v += dpp_or_0<0x118, 0xF>(v);
  v += dpp_or_0<0x142, 0xA>(v);  // row_bcast 15 and 31
  v += dpp_or_0<0x143, 0xC>(v);
  return v;
}
// the same with every sum held at cap, for 0 <= v <= cap <= 2^30
__device__ __forceinline__ int wave_scan(int v, int cap) {
  v = min(v + dpp_or_0<0x111, 0xF>(v), cap);
  v = min(v + dpp_or_0<0x112, 0xF>(v), cap);
  v = min(v + dpp_or_0<0x114, 0xF>(v), cap);
  v = min(v + dpp_or_0<0x118, 0xF>(v), cap);
  v = min(v + dpp_or_0<0x142, 0xA>(v), cap);
  v = min(v + dpp_or_0<0x143, 0xC>(v), cap);
  return v;
}

}  // namespace paged
}  // namespace plz

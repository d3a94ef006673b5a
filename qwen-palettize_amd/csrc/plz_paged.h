// How a batch's cached tokens are dealt to workgroups (plz_paged_attn.hip); plain integer rules, so
// that they are checked on the host.
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

}  // namespace paged
}  // namespace plz

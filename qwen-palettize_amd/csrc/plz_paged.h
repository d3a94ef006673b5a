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

// The tiles of all requests, one behind the other (`total` of them), are cut into `parts` runs of equal
// length, one a workgroup: a long request is shared by many, a workgroup takes several short ones.
// No run is shorter than one tile a wave (`waves`).
__host__ __device__ __forceinline__ int run_count(int total, int parts, int waves) {
  const int n = (total + waves - 1) / waves;
  return n < parts ? n : parts;
}
__host__ __device__ __forceinline__ int run_begin(int total, int runs, int w) {
  return (int)((int64_t)total * w / runs);
}
// the run that holds tile p: the largest w with run_begin(w) <= p
__host__ __device__ __forceinline__ int run_of(int total, int runs, int p) {
  return (int)((((int64_t)p + 1) * runs + total - 1) / total) - 1;
}

}  // namespace paged
}  // namespace plz

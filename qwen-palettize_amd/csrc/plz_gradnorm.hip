// The global norm of many gradients, and gradients clipped by it (torch.nn.utils.clip_grad_norm_, which
// train_qwen.py:1303-1319 calls for each of its two tiers):
//
//   norm = sqrt(sum of the squares of every value of every tensor)
//   out_i = grad_i * min(1, max_norm / (norm + 1e-6))
//
// Values are bf16, fp16 or fp32 and are squared and summed in 64 bits: no square of an fp32 value
// overflows or vanishes, and the sum's order, which is fixed, hardly matters. HBM-bound: the norm reads
// every value once; what clips reads them again, from the last to the first, since the Infinity Cache
// still holds the end of what the norm read, and writes them. The tensors' addresses travel as kernel
// arguments, kTensors a launch: no table is copied to the GPU, and a captured graph holds them.
#include "plz_common.h"
#include "palettize_hip.h"

namespace plz {
namespace gn {

constexpr int kThreads = 256;
constexpr int kVec = 8;                        // values a thread takes at a time
constexpr int kChunk = kThreads * kVec * 16;  // values of a workgroup
constexpr int kTensors = 128;                  // of a launch: 3.9 KB of arguments

struct Tensors {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t n[kTensors];
  int32_t begin[kTensors + 1];  // first workgroup of each in this launch
  uint8_t in_type[kTensors], out_type[kTensors];
  uint8_t aligned[kTensors];    // both on 16 bytes
  int count;
};

__device__ __forceinline__ int tensor_of(const Tensors& t, int b) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.begin[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float value(const void* p, int type, int64_t i) {
  if (type == PLZ_DT_FP32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t b = reinterpret_cast<const uint16_t*>(p)[i];
  return type == PLZ_DT_BF16 ? bf2f(b) : h2f(b);
}
__device__ __forceinline__ void put(void* p, int type, int64_t i, float v) {
  if (type == PLZ_DT_FP32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(type == PLZ_DT_BF16 ? f2bf(v) : f2h(v));
}

// 8 values from i on
template <int TYPE>
struct Raw {
  uint4 a, b;
};
template <int TYPE>
__device__ __forceinline__ Raw<TYPE> load8(const void* p, int64_t i) {
  Raw<TYPE> r;
  if (TYPE == PLZ_DT_FP32) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
    r.a = q[0];
    r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ void values(const Raw<TYPE>& r, float (&f)[kVec]) {
  const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  if (TYPE == PLZ_DT_FP32) {
    const uint32_t b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = __uint_as_float(a[j]);
      f[4 + j] = __uint_as_float(b[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = TYPE == PLZ_DT_BF16 ? bf2f(a[j] & 0xffffu) : h2f(a[j] & 0xffffu);
      f[2 * j + 1] = TYPE == PLZ_DT_BF16 ? bf2f(a[j] >> 16) : h2f(a[j] >> 16);
    }
  }
}

template <int TYPE>
__device__ __forceinline__ double squares(const void* p, int64_t i0, int64_t end) {
  double s0 = 0, s1 = 0;
  const int64_t whole = end - (end - i0) % kVec;
#pragma unroll 4
  for (int64_t i = i0 + (int64_t)threadIdx.x * kVec; i < whole; i += kThreads * kVec) {
    float f[kVec];
    values<TYPE>(load8<TYPE>(p, i), f);
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
      s0 = __builtin_fma((double)f[j], (double)f[j], s0);
      s1 = __builtin_fma((double)f[j + 1], (double)f[j + 1], s1);
    }
  }
  if (threadIdx.x < end - whole) {
    const double v = value(p, TYPE, whole + threadIdx.x);
    s0 += v * v;
  }
  return s0 + s1;
}

__device__ __forceinline__ double block_sum(double v, double* red, int waves) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
  for (int w = 0; w < waves; ++w) s += red[w];
  return s;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(const Tensors t, double* __restrict__ part) {
  __shared__ double red[kThreads / 64];
  const int k = tensor_of(t, (int)blockIdx.x), type = t.in_type[k];
  const int64_t i0 = (int64_t)((int)blockIdx.x - t.begin[k]) * kChunk;
  const int64_t end = min(t.n[k], i0 + kChunk);
  const void* p = t.in[k];
  double s = 0;
  if (!t.aligned[k]) {
    for (int64_t i = i0 + threadIdx.x; i < end; i += kThreads) {
      const double v = value(p, type, i);
      s += v * v;
    }
  } else if (type == PLZ_DT_BF16) {
    s = squares<PLZ_DT_BF16>(p, i0, end);
  } else if (type == PLZ_DT_FP16) {
    s = squares<PLZ_DT_FP16>(p, i0, end);
  } else {
    s = squares<PLZ_DT_FP32>(p, i0, end);
  }
  s = block_sum(s, red, kThreads / 64);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// out = norm; *factor = min(1, max_norm / (norm + 1e-6)), NaN for a norm of NaN
__global__ __launch_bounds__(1024) void norm_kernel(const double* __restrict__ part, int64_t n,
                                                    float max_norm, float* __restrict__ out,
                                                    float* __restrict__ factor) {
  __shared__ double red[16];
  double s = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = block_sum(s, red, 16);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s);
    *out = (float)norm;
    if (factor) {
      const double c = max_norm / (norm + 1e-6);
      *factor = c > 1.0 ? 1.f : (float)c;
    }
  }
}

template <int IN, int OUT>
__device__ __forceinline__ void scale(const void* p, void* o, int64_t i0, int64_t end, float c) {
  const int64_t whole = end - (end - i0) % kVec;
#pragma unroll 4
  for (int64_t i = i0 + (int64_t)threadIdx.x * kVec; i < whole; i += kThreads * kVec) {
    float f[kVec];
    values<IN>(load8<IN>(p, i), f);
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[j] *= c;
    if (OUT == PLZ_DT_FP32) {
      float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(o) + i);
      d[0] = make_float4(f[0], f[1], f[2], f[3]);
      d[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = OUT == PLZ_DT_BF16 ? f2bf2(f[2 * j], f[2 * j + 1])
                                  : f2h(f[2 * j]) | (f2h(f[2 * j + 1]) << 16);
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(o) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (threadIdx.x < end - whole)
    put(o, OUT, whole + threadIdx.x, value(p, IN, whole + threadIdx.x) * c);
}
template <int IN>
__device__ __forceinline__ void scale_to(int out_type, const void* p, void* o, int64_t i0, int64_t end,
                                         float c) {
  if (out_type == PLZ_DT_BF16) scale<IN, PLZ_DT_BF16>(p, o, i0, end, c);
  else if (out_type == PLZ_DT_FP16) scale<IN, PLZ_DT_FP16>(p, o, i0, end, c);
  else scale<IN, PLZ_DT_FP32>(p, o, i0, end, c);
}

__global__ __launch_bounds__(kThreads) void clip_kernel(const Tensors t,
                                                        const float* __restrict__ factor) {
  const int b = t.begin[t.count] - 1 - (int)blockIdx.x;
  const int k = tensor_of(t, b), in = t.in_type[k], out = t.out_type[k];
  const float c = *factor;
  const void* p = t.in[k];
  void* o = t.out[k];
  if (p == o && c == 1.f) return;  // in place, and nothing changes
  const int64_t i0 = (int64_t)(b - t.begin[k]) * kChunk, end = min(t.n[k], i0 + kChunk);
  if (!t.aligned[k]) {
    for (int64_t i = i0 + threadIdx.x; i < end; i += kThreads) put(o, out, i, value(p, in, i) * c);
  } else if (in == PLZ_DT_BF16) {
    scale_to<PLZ_DT_BF16>(out, p, o, i0, end, c);
  } else if (in == PLZ_DT_FP16) {
    scale_to<PLZ_DT_FP16>(out, p, o, i0, end, c);
  } else {
    scale_to<PLZ_DT_FP32>(out, p, o, i0, end, c);
  }
}

constexpr int64_t kMaxBlocks = 0x7fffff;  // of a launch: 2^31 threads
static int64_t chunks(int64_t n) { return (n + kChunk - 1) / kChunk; }
static size_t part_bytes(int64_t blocks) { return ((size_t)blocks * sizeof(double) + 255) / 256 * 256; }

// Tensors first .. count - 1 into a launch, as many as it holds: how many were taken
static int fill(Tensors& t, const void* const* in, void* const* out, const int64_t* n,
                const int32_t* in_type, const int32_t* out_type, int first, int count) {
  t.count = 0;
  t.begin[0] = 0;
  int i = first;
  for (; i < count && t.count < kTensors; ++i) {
    if (n[i] == 0) continue;
    const int64_t end = t.begin[t.count] + chunks(n[i]);
    if (end > kMaxBlocks) break;  // one tensor always fits
    const int k = t.count++;
    t.in[k] = in[i];
    t.out[k] = out ? out[i] : nullptr;
    t.n[k] = n[i];
    t.in_type[k] = (uint8_t)in_type[i];
    t.out_type[k] = (uint8_t)(out ? out_type[i] : 0);
    t.aligned[k] = (((uintptr_t)in[i] | (out ? (uintptr_t)out[i] : 0)) & 15) == 0;
    t.begin[t.count] = (int32_t)end;
  }
  return i - first;
}

static int check(const void* const* in, const int64_t* n, const int32_t* type, int count,
                 const char* what) {
  PLZ_REQUIRE(count >= 0 && (count == 0 || (in && n && type)), "%s: null pointer or bad count", what);
  for (int i = 0; i < count; ++i) {
    PLZ_REQUIRE(n[i] >= 0 && chunks(n[i]) <= kMaxBlocks && (n[i] == 0 || in[i]),
                "%s: tensor %d is null or too large", what, i);
    PLZ_REQUIRE(type[i] == PLZ_DT_BF16 || type[i] == PLZ_DT_FP16 || type[i] == PLZ_DT_FP32,
                "%s: tensor %d has type %d", what, i, type[i]);
    PLZ_REQUIRE(((uintptr_t)in[i] & (type[i] == PLZ_DT_FP32 ? 3 : 1)) == 0,
                "%s: tensor %d is not aligned to its values", what, i);
  }
  return PLZ_OK;
}

static int norm(const void* const* in, const int64_t* n, const int32_t* type, int count, float max_norm,
                float* out, bool clip, void* ws, size_t ws_bytes, hipStream_t st, const char* what) {
  if (int rc = check(in, n, type, count, what)) return rc;
  PLZ_REQUIRE(out, "%s: null pointer", what);
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) blocks += chunks(n[i]);
  const size_t need = part_bytes(blocks) + 256;
  if (!ws || ws_bytes < need) {
    set_error("%s: workspace of %zu bytes needed, %zu given", what, need, ws ? ws_bytes : 0);
    return PLZ_EWORKSPACE;
  }
  PLZ_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace must be 16-byte aligned", what);
  float* factor = reinterpret_cast<float*>(ws);
  double* part = reinterpret_cast<double*>(reinterpret_cast<char*>(ws) + 256);
  Tensors t;
  int64_t b = 0;
  for (int i = 0; i < count;) {
    i += fill(t, in, nullptr, n, type, nullptr, i, count);
    if (t.count == 0) continue;
    hipLaunchKernelGGL(squares_kernel, dim3((unsigned)t.begin[t.count]), dim3(kThreads), 0, st, t,
                       part + b);
    if (int rc = check_launch(what)) return rc;
    b += t.begin[t.count];
  }
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, st, part, blocks, max_norm, out,
                     clip ? factor : nullptr);
  return check_launch(what);
}

// out[i] = in[i] * *factor: launches from the last tensors to the first, as the workgroups within each
static int scale_all(const void* const* in, void* const* out, const int64_t* sizes,
                     const int32_t* in_type, const int32_t* out_type, int count, const float* factor,
                     hipStream_t st, const char* what) {
  Tensors t;
  for (int hi = count; hi > 0;) {
    int lo = hi, taken = 0;
    int64_t blocks = 0;
    while (lo > 0 && taken < kTensors && blocks + chunks(sizes[lo - 1]) <= kMaxBlocks) {
      blocks += chunks(sizes[--lo]);
      taken += sizes[lo] > 0;
    }
    fill(t, in, out, sizes, in_type, out_type, lo, hi);
    hi = lo;
    if (t.count == 0) continue;
    hipLaunchKernelGGL(clip_kernel, dim3((unsigned)t.begin[t.count]), dim3(kThreads), 0,
                       st, t, factor);
    if (int rc = check_launch(what)) return rc;
  }
  return PLZ_OK;
}

}  // namespace gn
}  // namespace plz

using namespace plz;
using namespace plz::gn;

extern "C" {

size_t plz_grad_norm_workspace(const int64_t* sizes, int count) {
  if (count < 0 || (count > 0 && !sizes)) return 0;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) blocks += sizes[i] > 0 ? chunks(sizes[i]) : 0;
  return part_bytes(blocks) + 256;
}

int plz_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int count,
                  float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  return norm(grads, sizes, dtypes, count, 0.f, norm_out, false, workspace, workspace_bytes,
              (hipStream_t)stream, "plz_grad_norm");
}

int plz_clip_grads(const void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                   void* const* out, const int32_t* out_dtypes, int count, float max_norm,
                   float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "plz_clip_grads";
  PLZ_REQUIRE(max_norm >= 0.f, "%s: max_norm must not be negative", what);
  if (int rc = check(reinterpret_cast<const void* const*>(out), sizes, out_dtypes, count, what)) return rc;
  if (int rc = check(grads, sizes, dtypes, count, what)) return rc;
  for (int i = 0; i < count; ++i)
    PLZ_REQUIRE(sizes[i] == 0 || grads[i] != out[i] || dtypes[i] == out_dtypes[i],
                "%s: tensor %d would change its type in place", what, i);
  if (int rc = norm(grads, sizes, dtypes, count, max_norm, norm_out, true, workspace, workspace_bytes,
                    (hipStream_t)stream, what))
    return rc;
  return scale_all(grads, out, sizes, dtypes, out_dtypes, count, reinterpret_cast<const float*>(workspace),
                   (hipStream_t)stream, what);
}

int plz_scale_grads(void* const* grads, const int64_t* sizes, const int32_t* dtypes, int count,
                    const float* factor, void* stream) {
  const char* what = "plz_scale_grads";
  const void* const* in = reinterpret_cast<const void* const*>(grads);
  if (int rc = check(in, sizes, dtypes, count, what)) return rc;
  PLZ_REQUIRE(factor, "%s: null pointer", what);
  return scale_all(in, grads, sizes, dtypes, dtypes, count, factor, (hipStream_t)stream, what);
}

}  // extern "C"

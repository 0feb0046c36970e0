// What the kernels of the selective scan share (selective.cu, selective_heads.cu).
#pragma once

#include "common.cuh"

namespace b200 {
namespace selective {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// SiLU; with 16-bit rows through the fast exponential and division (relative errors near 1e-6)
template <typename T>
__device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 2) return __fdividef(x, 1.0f + __expf(-x));
  else return x / (1.0f + expf(-x));
}
// log(1 + e^z) = max(z, 0) + log(1 + e), e = e^-|z|.  With 16-bit rows log(1 + e) = 2 artanh(s), s = e / (2 + e) <=
// 1/3, by seven terms of its series (the next one is below 2^-26), and e by the fast power of two of a
// product in two parts: a step size enters every later state, so it keeps 2^-21 where logarithms of
// sums near 1 would leave 2^-15 of small ones.
template <typename T>
__device__ __forceinline__ float softplus(float z) {
  const float over = z < 0.0f ? 0.0f : z;
  if constexpr (sizeof(T) == 2) {
    const float q = fmaxf(-fabsf(z), -120.0f), p = q * kLog2e;
    const float low = fmaf(q, 1.925963033e-8f, fmaf(q, kLog2e, -p));
    float e = exp2_fast(p);
    e = fmaf(e, 0.69314718f * low, e);
    const float s = __fdividef(e, 2.0f + e), t = s * s;
    float f = fmaf(t, 1.0f / 13.0f, 1.0f / 11.0f);
    f = fmaf(t, f, 1.0f / 9.0f);
    f = fmaf(t, f, 1.0f / 7.0f);
    f = fmaf(t, f, 1.0f / 5.0f);
    f = fmaf(t, f, 1.0f / 3.0f);
    f = fmaf(t, f, 1.0f);
    return fmaf(2.0f * s, f, over);
  } else {
    return over + log1pf(expf(-fabsf(z)));
  }
}

// Rows of the step that belong to a request.
struct Portion {
  int first, end;
};
__device__ __forceinline__ Portion portion_of(int r, int nd, const int* cu_q, int T) {
  if (r < nd) return {r, r + 1};
  return {nd + cu_q[r - nd], min(nd + cu_q[r - nd + 1], T)};
}

struct ScanArgs {
  const void* x;             // [T, heads * width]
  const void* dt;            // [T, heads] or [T, heads * width], the rows' type or fp32
  const void *b, *c;         // [T, groups * N]
  const void* z;             // [T, heads * width] or null
  void* out;                 // [T, heads * width]
  const float* a_log;        // [heads] or [heads * width, N]
  const float* d;            // like the step sizes' row, or null
  const float* dt_bias;      // likewise
  float* state;              // [slots, heads * width, N] or null
  const long long* positions;
  const int *slots, *wslots;
  const int* cu_q;
  long long ldx, lddt, ldb, ldc, ldz, ldo;
  float dt_min, dt_max;
  int T, heads, width, N, groups, num_slots, nd, np, dt_f32, softplus, wide;
};

// The step size that comes of a row's number (NaN stays NaN).
template <typename T>
__device__ __forceinline__ float step_from(const ScanArgs& a, float z, float bias) {
  z += bias;
  if (a.softplus) z = softplus<T>(z);
  return z < a.dt_min ? a.dt_min : z > a.dt_max ? a.dt_max : z;
}
template <typename T>
__device__ __forceinline__ float step_size(const ScanArgs& a, long long row, int i) {
  const long long at = row * a.lddt + i;
  const float z = a.dt_f32 ? static_cast<const float*>(a.dt)[at] : to_f32<T>(static_cast<const T*>(a.dt)[at]);
  return step_from<T>(a, z, a.dt_bias != nullptr ? a.dt_bias[i] : 0.0f);
}

// Portions of prompts by products of tiles (selective_heads.cu): rates per head, bf16 rows on 16-byte boundaries.
bool heads_by_tiles(const ScanArgs& a);
int launch_heads_by_tiles(const ScanArgs& a, cudaStream_t s);

}  // namespace selective
}  // namespace b200

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
// SiLU and softplus: with 16-bit rows through the fast exponential, division and logarithm (relative errors
// near 1e-6; the logarithm of 1 + e switches to its series where e would be rounded away)
template <typename T>
__device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 2) return __fdividef(x, 1.0f + __expf(-x));
  else return x / (1.0f + expf(-x));
}
__device__ __forceinline__ float softplus(float z) {
  return fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z)));
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

template <typename T>
__device__ __forceinline__ float step_size(const ScanArgs& a, long long row, int i) {
  const long long at = row * a.lddt + i;
  float z = a.dt_f32 ? static_cast<const float*>(a.dt)[at] : to_f32<T>(static_cast<const T*>(a.dt)[at]);
  if (a.dt_bias != nullptr) z += a.dt_bias[i];
  if (a.softplus) z = softplus(z);
  return fminf(fmaxf(z, a.dt_min), a.dt_max);
}

// Portions of prompts by products of tiles (selective_heads.cu): rates per head, bf16 rows on 16-byte boundaries.
bool heads_by_tiles(const ScanArgs& a);
int launch_heads_by_tiles(const ScanArgs& a, cudaStream_t s);

}  // namespace selective
}  // namespace b200

// What the kernels of the selective scan share (selective.cu,
// selective_step.cu, selective_heads.cu) and the causal convolution (causal_conv.cu).
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
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Decays of a token from its step size and two rates (base 2).  The special function unit's powers of two come out
// low, by 2e-8 on average where they are near 1, and a state that lasts a thousand tokens would add that up; with 2e-8 on
// the exponent, which the product's addition gives for nothing, the mean error is below 1.3e-8 from 2^-14 to 1, like
// the one of the slow exponential.  A step of 0 still gives 1.
__device__ __forceinline__ float2 decays(float2 step, float2 rate) {
  const float2 p = __ffma2_rn(step, rate, make_float2(2e-8f, 2e-8f));
  return make_float2(exp2_fast(p.x), exp2_fast(p.y));
}
// The decay of an exponent where a token has one per head, or few.  Near 1 the exponential is high by 1.5e-8 on average, which
// a state that lasts thousands of tokens adds up (2.9e-5 after 4000); there the power series to p^5, off by less than p^6 /
// 720 = 8.3e-11, whose last addition alone rounds.
__device__ __forceinline__ float decay_of(float p) {
  float s = fmaf(p, 1.0f / 120.0f, 1.0f / 24.0f);
  s = fmaf(p, s, 1.0f / 6.0f);
  s = fmaf(p, s, 0.5f);
  s = fmaf(p, s, 1.0f);
  const float e = expf(p);
  return fabsf(p) < 0.0625f ? fmaf(p, s, 1.0f) : e;
}
// SiLU; with 16-bit rows through the fast exponential and division (relative errors near 1e-6)
template <typename T>
__device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 2) return x * rcp_fast(1.0f + exp2_fast(-kLog2e * x));
  else return x / (1.0f + expf(-x));
}
// log(1 + e^z) = max(z, 0) + log(1 + e), e = e^-|z|.  With 16-bit rows log(1 + e) = e P(e), P of degree 9
// interpolated at the Chebyshev points of [0, 1] (off by 8.2e-9, as a part of it 1.2e-8, in fp32 1.3e-7), and e by the fast power of two
// of a product in two parts: a step size enters every later state, so it keeps 2^-22 where the fast logarithm of a
// sum near 1 would leave 2^-15 of small ones.  Two numbers at a time.
__device__ __forceinline__ float2 softplus_pair(float2 z) {
  const float2 q = make_float2(fmaxf(-fabsf(z.x), -120.0f), fmaxf(-fabsf(z.y), -120.0f));
  const float2 p = __fmul2_rn(q, make_float2(kLog2e, kLog2e));
  const float2 low = __ffma2_rn(q, make_float2(1.925963033e-8f, 1.925963033e-8f),
                                __ffma2_rn(q, make_float2(kLog2e, kLog2e), make_float2(-p.x, -p.y)));
  float2 e = make_float2(exp2_fast(p.x), exp2_fast(p.y));
  e = __ffma2_rn(e, __fmul2_rn(low, make_float2(0.69314718f, 0.69314718f)), e);
  constexpr float k[10] = {1.0f,          -0.4999989271f, 0.3332971036f,  -0.2495161593f, 0.1966327429f,
                           -0.1526966691f, 0.1054362357f, -0.0563736148f, 0.0195425283f,  -0.0031760570f};
  float2 f = make_float2(k[9], k[9]);
#pragma unroll
  for (int i = 8; i >= 0; --i) f = __ffma2_rn(f, e, make_float2(k[i], k[i]));
  // (NaN: not below 0)
  return __ffma2_rn(f, e, make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y));
}
template <typename T>
__device__ __forceinline__ float softplus(float z) {
  if constexpr (sizeof(T) == 2) return softplus_pair(make_float2(z, z)).x;
  else return (z < 0.0f ? 0.0f : z) + log1pf(expf(-fabsf(z)));
}

// Rows of the step that belong to a request.
struct Portion {
  int first, end;
};
__device__ __forceinline__ Portion portion_of(int r, int nd, const int* cu_q, int T) {
  if (r < nd) return {r, r + 1};
  return {nd + max(cu_q[r - nd], 0), min(nd + cu_q[r - nd + 1], T)};
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
  int T, heads, width, N, groups, num_slots, nd, np, dt_f32, softplus, limits, wide;
};

// Step sizes that come of rows' numbers (NaN stays NaN).
__device__ __forceinline__ float limited(const ScanArgs& a, float z) {
  return z < a.dt_min ? a.dt_min : z > a.dt_max ? a.dt_max : z;
}
template <typename T>
__device__ __forceinline__ float step_from(const ScanArgs& a, float z, float bias) {
  z += bias;
  if (a.softplus) z = softplus<T>(z);
  return a.limits ? limited(a, z) : z;
}
template <typename T>
__device__ __forceinline__ float step_size(const ScanArgs& a, long long row, int i) {
  const long long at = row * a.lddt + i;
  const float z = a.dt_f32 ? static_cast<const float*>(a.dt)[at] : to_f32<T>(static_cast<const T*>(a.dt)[at]);
  return step_from<T>(a, z, a.dt_bias != nullptr ? a.dt_bias[i] : 0.0f);
}

// V neighbouring elements, in one access where V is 4
template <typename T, int V>
struct Raw {
  T e[V];
};
template <>
struct __align__(8) Raw<__nv_bfloat16, 4> {
  __nv_bfloat16 e[4];
};
template <>
struct __align__(8) Raw<__half, 4> {
  __half e[4];
};
template <>
struct __align__(16) Raw<float, 4> {
  float e[4];
};

// One token per request (selective_step.cu).  dtype: 0 bf16, 1 fp16, 2 fp32.
int launch_single_tokens(const ScanArgs& a, bool per_channel, int dtype, cudaStream_t s);
// The whole step where its portions are short and rates are per head; false where it does not apply.
bool launch_short_portions(const ScanArgs& a, int dtype, cudaStream_t s, int* rc);
// Portions of prompts by products of tiles (selective_heads.cu): rates per head, bf16 rows on 16-byte boundaries.
bool heads_by_tiles(const ScanArgs& a);
int launch_heads_by_tiles(const ScanArgs& a, cudaStream_t s);

}  // namespace selective
}  // namespace b200

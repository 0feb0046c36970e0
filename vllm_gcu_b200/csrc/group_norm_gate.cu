// Group norm of rows with a gate (sm_100a): each of `groups` consecutive parts of a row is divided by its root mean
// square or, centred, freed of its mean first, times a weight, plus a bias.  The gate's activation
// multiplies the row in front of the norm or the result behind it; without a gate the activation may be
// that of the result.
//
// A part of a row is a problem of its own: rows * groups of them.  A team of threads (one warp up to 1024
// elements, a CTA above) holds its part in registers, NI vectors of V elements per thread, so that mean and
// variance are two passes over registers and memory is read once; wider parts are read again.  Bytes bound it
// (8192 rows of 8 x 1024, bf16: 75 us, 5.3 TB/s, among other calls, 68 in a captured graph): weights come from L1
// in 16 bytes, and nothing branches per element (140 us without either; teams that walked rows of one group, to keep
// its weights and have a row under way, had registers for too few of them: 297 us).
#include "common.cuh"

namespace b200 {
namespace gated_norm {

enum Act : int { kNone = 0, kSilu = 1, kSigmoid = 2 };

struct Args {
  const void *x, *z;         // [T, C]; z may be null
  void* out;                 // [T, C]
  const float *w, *bias;     // [C]; bias may be null
  long long ldx, ldz, ldo;
  float eps;
  int T, C, groups, width;   // width: C / groups
  int act, center, after;
  int parts;                 // T * groups
};

// fp32 forms for 16-bit rows: the fast exponential and division, relative errors near 1e-6.  (Selects, no
// branches: `act` is the same for all.)
template <typename T>
__device__ __forceinline__ float activate(float v, int act) {
  float s;
  if constexpr (sizeof(T) == 2) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
  } else s = 1.0f / (1.0f + expf(-v));
  return (act == kSigmoid ? 1.0f : v) * (act == kNone ? 1.0f : s);
}
enum Gate : int { kNoGate = 0, kBefore = 1, kAfter = 2 };

// V floats of a weight or bias
template <int V>
__device__ __forceinline__ void floats(const float* from, float (&to)[V]) {
  if constexpr (V == 1) {
    to[0] = from[0];
  } else {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const float4 f = *reinterpret_cast<const float4*>(from + v);
      to[v] = f.x; to[v + 1] = f.y; to[v + 2] = f.z; to[v + 3] = f.w;
    }
  }
}

template <typename T, int V>
struct Raw {
  T e[V];
};
template <>
struct __align__(16) Raw<__nv_bfloat16, 8> {
  __nv_bfloat16 e[8];
};
template <>
struct __align__(16) Raw<__half, 8> {
  __half e[8];
};
template <>
struct __align__(16) Raw<float, 4> {
  float e[4];
};

// Sum over the team of a thread: a warp or the whole CTA.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* red) {
  if constexpr (TEAM == 32) return warp_sum(v);
  else return block_sum(v, red);
}

template <typename T, int V, int NI, int TEAM, int GATE>
__global__ void __launch_bounds__(TEAM == 32 ? 128 : TEAM) group_norm_gate_kernel(const Args a) {
  __shared__ float red[32];
  using R = Raw<T, V>;
  grid_release_small();
  grid_wait();
  const int lane = TEAM == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int part = TEAM == 32 ? static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (part >= a.parts) return;                   // (a whole team)
  const long long t = part / a.groups;
  const int c0 = part % a.groups * a.width;
  const T* x = static_cast<const T*>(a.x) + t * a.ldx + c0;
  const T* z = static_cast<const T*>(a.z) + t * a.ldz + c0;
  T* out = static_cast<T*>(a.out) + t * a.ldo + c0;
  const float inv_n = 1.0f / static_cast<float>(a.width);

  R rx[NI], rz[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = (i * TEAM + lane) * V;
    if (c < a.width) {
      rx[i] = *reinterpret_cast<const R*>(x + c);
      if (GATE != kNoGate) rz[i] = *reinterpret_cast<const R*>(z + c);
    }
  }
  float f[NI][V];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if ((i * TEAM + lane) * V < a.width) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[i][v] = to_f32<T>(rx[i].e[v]);
        if (GATE == kBefore) f[i][v] *= activate<T>(to_f32<T>(rz[i].e[v]), a.act);
        sum += f[i][v];
      }
    }
  }
  const float mean = a.center ? team_sum<TEAM>(sum, red) * inv_n : 0.0f;
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if ((i * TEAM + lane) * V < a.width) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[i][v] -= mean;
        ss = fmaf(f[i][v], f[i][v], ss);
      }
    }
  }
  const float inv = 1.0f / sqrtf(team_sum<TEAM>(ss, red) * inv_n + a.eps);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = (i * TEAM + lane) * V;
    if (c < a.width) {
      float w[V], b[V];
      floats<V>(a.w + c0 + c, w);
      if (a.bias != nullptr) {
        floats<V>(a.bias + c0 + c, b);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) b[v] = 0.0f;
      }
      R y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float q = fmaf(f[i][v] * inv, w[v], b[v]);
        if (GATE == kAfter) q *= activate<T>(to_f32<T>(rz[i].e[v]), a.act);
        else if (GATE == kNoGate) q = activate<T>(q, a.act);
        y.e[v] = from_f32<T>(q);
      }
      *reinterpret_cast<R*>(out + c) = y;
    }
  }
}

// Parts that do not fit a CTA's registers: read once for the mean, once for the variance, once for the result.
template <typename T>
__global__ void __launch_bounds__(1024) group_norm_gate_wide_kernel(const Args a) {
  __shared__ float red[32];
  grid_release_small();
  grid_wait();
  const long long part = blockIdx.x;
  const long long t = part / a.groups;
  const int c0 = static_cast<int>(part % a.groups) * a.width;
  const T* x = static_cast<const T*>(a.x) + t * a.ldx + c0;
  const T* z = a.z != nullptr ? static_cast<const T*>(a.z) + t * a.ldz + c0 : nullptr;
  T* out = static_cast<T*>(a.out) + t * a.ldo + c0;
  const float n = static_cast<float>(a.width);
  auto value = [&](int c) {
    float f = to_f32<T>(x[c]);
    if (z != nullptr && !a.after) f *= activate<T>(to_f32<T>(z[c]), a.act);
    return f;
  };
  float mean = 0.0f;
  if (a.center) {
    float sum = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) sum += value(c);
    mean = block_sum(sum, red) / n;
  }
  float ss = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
    const float f = value(c) - mean;
    ss = fmaf(f, f, ss);
  }
  const float inv = 1.0f / sqrtf(block_sum(ss, red) / n + a.eps);
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
    float q = (value(c) - mean) * inv * a.w[c0 + c];
    if (a.bias != nullptr) q += a.bias[c0 + c];
    if (z != nullptr && a.after) q *= activate<T>(to_f32<T>(z[c]), a.act);
    else if (z == nullptr) q = activate<T>(q, a.act);
    out[c] = from_f32<T>(q);
  }
}

template <typename T, int V, int NI, int TEAM>
int launch(const Args& a, cudaStream_t s) {
  constexpr int kPer = TEAM == 32 ? 4 : 1;
  const dim3 grid((a.parts + kPer - 1) / kPer), cta(TEAM * kPer);
  if (a.z == nullptr) return launch_overlapped(group_norm_gate_kernel<T, V, NI, TEAM, kNoGate>, grid, cta, 0, s, a);
  if (a.after) return launch_overlapped(group_norm_gate_kernel<T, V, NI, TEAM, kAfter>, grid, cta, 0, s, a);
  return launch_overlapped(group_norm_gate_kernel<T, V, NI, TEAM, kBefore>, grid, cta, 0, s, a);
}
template <typename T, int V>
int launch(const Args& a, cudaStream_t s) {
  const int vecs = (a.width + V - 1) / V;
  if (vecs <= 32) return launch<T, V, 1, 32>(a, s);
  if (vecs <= 64) return launch<T, V, 2, 32>(a, s);
  if (vecs <= 128) return launch<T, V, 4, 32>(a, s);
  if (vecs <= 256) return launch<T, V, 2, 128>(a, s);
  if (vecs <= 512) return launch<T, V, 2, 256>(a, s);
  if (vecs <= 1024) return launch<T, V, 2, 512>(a, s);
  if (vecs <= 2048) return launch<T, V, 4, 512>(a, s);
  return launch_overlapped(group_norm_gate_wide_kernel<T>, dim3(a.parts), dim3(1024), 0, s, a);
}
template <typename T>
int launch_any(const Args& a, bool wide, cudaStream_t s) {
  return wide ? launch<T, 16 / sizeof(T)>(a, s) : launch<T, 1>(a, s);
}

}  // namespace gated_norm
}  // namespace b200

// The arguments of a call, packed by the launcher (ops/cuda.py).  dtype: 0 bf16, 1 fp16, 2 fp32 rows; act: 0 none,
// 1 SiLU, 2 sigmoid; wide: parts of rows may be read 16 bytes at a time.
namespace {
struct NormCall {
  const void *x, *z;
  void* out;
  const float *w, *bias;
  long long ldx, ldz, ldo;
  float eps;
  int T, C, groups, act, center, after, wide, dtype;
};
}  // namespace

B200_API int b200_group_norm_gate(const void* call, void* stream) {
  using namespace b200::gated_norm;
  const NormCall& k = *static_cast<const NormCall*>(call);
  if (k.T <= 0 || k.C <= 0) return 0;
  const long long parts = static_cast<long long>(k.T) * k.groups;
  if (k.groups <= 0 || k.C % k.groups != 0 || parts > 0x7ffffff0ll) return -8;
  const Args a{k.x, k.z, k.out, k.w, k.bias, k.ldx, k.ldz, k.ldo, k.eps, k.T, k.C, k.groups, k.C / k.groups, k.act,
               k.center, k.after, static_cast<int>(parts)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (k.dtype) {
    case 0: return launch_any<__nv_bfloat16>(a, k.wide, s);
    case 1: return launch_any<__half>(a, k.wide, s);
    case 2: return launch_any<float>(a, k.wide, s);
  }
  return -8;
}

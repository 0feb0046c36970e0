// Short causal convolution of a state-space mixer (sm_100a), over the rows of a step: nd single tokens, one per
// request, then the portions of np prompts (offsets behind row nd in cu_q):
//   c_t = act(bias + sum_j w[j] x of (taps - 1 - j) tokens ago), per channel
// A request's last inputs lie in ring [slot, taps - 1, channels], position p in row p % (taps - 1), read in one slot
// and left in another (usually the same).  A portion that starts at position 0 starts from zeros whatever the slot holds.  A
// request whose slot is outside the ring (padding of a captured batch) gives rows of zeros; one whose write slot is
// outside leaves its inputs nowhere.
#include "selective.cuh"

namespace b200 {
namespace selective {

struct ConvArgs {
  const void* x;             // [T, C], row pitch ldx
  const float* w;            // [taps, C], last row: current token
  const float* bias;         // [C] or null
  void* ring;                // [slots, taps - 1, C] or null
  void* out;                 // [T, C], row pitch ldo
  const long long* positions;
  const int *slots, *wslots; // [requests], may be null without a ring
  const int* cu_q;
  long long ldx, ldo;
  int T, C, num_slots, nd, np, silu, strip;
};

constexpr int kMaxTaps = 8;
constexpr int kStrip = 16;                       // rows of prompts that a CTA walks, at least
static_assert(kStrip >= kMaxTaps, "a row that reads the ring lies in the strip of its portion's first row");

// A CTA: a strip of rows, V channels per thread.  A single token is a strip of its own; strips of
// prompts are a.strip rows long, but that the first taps - 1 rows of a portion stay in one strip: they
// are the only ones that read the ring, and the threads that read a channel of it then write it, so
// reading and writing need no second launch.
// Bytes bound it: rows are read once (those in front of a strip a second time, from L2) and written once.  8192 rows of
// 10240 channels, bf16, 4 taps: 81 us, 4.2 TB/s, half of it the two special functions of SiLU per element.  Four channels
// per thread and kBatch rows under way: with eight channels the registers of the window leave 12 warps an SM (107 us);
// strips of 64 rows make the search for a row's request and the window in front of the strip seldom (16 rows: 8 us more).
template <typename T, int NT, int V>
__global__ void __launch_bounds__(128) causal_conv_kernel(const ConvArgs a) {
  constexpr int kBack = NT - 1;
  using R = Raw<T, V>;
  grid_release_small();
  grid_wait();
  const int c = (blockIdx.y * 128 + threadIdx.x) * V;
  const int strip = blockIdx.x;
  int lo, hi, req;
  if (strip < a.nd) {
    lo = req = strip;
    hi = lo + 1;
  } else {
    lo = a.nd + (strip - a.nd) * a.strip;
    hi = min(lo + a.strip, a.T);
    TokenPlace pl = token_place(lo, a.nd, a.np, a.cu_q);
    if (pl.req < 0) return;                      // behind the last portion
    req = pl.req;
    Portion po = portion_of(req, a.nd, a.cu_q, a.T);
    if (lo > po.first && lo - po.first < kBack) lo = min(po.first + kBack, po.end);
    if (hi < a.T) {
      pl = token_place(hi, a.nd, a.np, a.cu_q);
      if (pl.req >= 0) {
        po = portion_of(pl.req, a.nd, a.cu_q, a.T);
        if (hi > po.first && hi - po.first < kBack) hi = min(po.first + kBack, po.end);
      }
    }
  }
  if (c >= a.C) return;
  const T* x = static_cast<const T*>(a.x) + c;
  T* out = static_cast<T*>(a.out) + c;
  auto ring_row = [&](int slot, long long pos) {
    return reinterpret_cast<R*>(static_cast<T*>(a.ring) +
                                (static_cast<long long>(slot) * kBack + pos % (kBack > 0 ? kBack : 1)) * a.C + c);
  };
  float w[NT][V], b[V];
  auto floats = [&](const float* from, float (&to)[V]) {
    if constexpr (V == 1) {
      to[0] = from[0];
    } else {
#pragma unroll
      for (int v = 0; v < V; v += 4) {
        const float4 f = *reinterpret_cast<const float4*>(from + v);
        to[v] = f.x; to[v + 1] = f.y; to[v + 2] = f.z; to[v + 3] = f.w;
      }
    }
  };
#pragma unroll
  for (int j = 0; j < NT; ++j) floats(a.w + static_cast<long long>(j) * a.C + c, w[j]);
  if (a.bias != nullptr) {
    floats(a.bias + c, b);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = 0.0f;
  }

  int t = lo;
  while (t < hi) {
    // rows [t, end) of one request
    Portion po = portion_of(req, a.nd, a.cu_q, a.T);
    while (po.end <= t) {                        // portions without rows
      if (++req >= a.nd + a.np) return;
      po = portion_of(req, a.nd, a.cu_q, a.T);
    }
    const int end = min(hi, po.end);
    R old[kBack > 0 ? kBack : 1];
#pragma unroll
    for (int j = 0; j < kBack; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) old[j].e[v] = from_f32<T>(0.0f);
    const int slot = a.ring != nullptr ? a.slots[req] : 0;
    const bool padding = a.ring != nullptr && (slot < 0 || slot >= a.num_slots);
    const bool kept = a.ring != nullptr && !padding;
    const long long pos = kept ? a.positions[po.first] : 0;     // of the portion's first row
#pragma unroll
    for (int j = 0; j < kBack; ++j) {
      const int row = t - kBack + j;
      if (row >= po.first)
        old[j] = *reinterpret_cast<const R*>(x + row * a.ldx);
      else if (kept && pos + (row - po.first) >= 0)
        old[j] = *ring_row(slot, pos + (row - po.first));
    }
    if (kept && t == po.first) {
      const int ws = a.wslots[req];
      if (ws >= 0 && ws < a.num_slots) {
#pragma unroll
        for (int j = 0; j < kBack; ++j) {        // the last kBack positions behind this portion
          const int row = po.end - kBack + j;
          const long long p = pos + (row - po.first);
          if (row >= po.first && p >= 0) {
            *ring_row(ws, p) = *reinterpret_cast<const R*>(x + row * a.ldx);
          } else if (p >= 0 && ws != slot) {     // row - po.first in [-kBack, -1]
#pragma unroll
            for (int i = 0; i < kBack; ++i)
              if (i == row - po.first + kBack) *ring_row(ws, p) = old[i];
          }
        }
      }
    }
    if (padding) {
      R none;
#pragma unroll
      for (int v = 0; v < V; ++v) none.e[v] = from_f32<T>(0.0f);
      for (; t < end; ++t) *reinterpret_cast<R*>(out + t * a.ldo) = none;
      continue;
    }
    float f[NT][V];                              // rows of the window, the last one is the token's
#pragma unroll
    for (int j = 0; j < kBack; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) f[j][v] = to_f32<T>(old[j].e[v]);
    auto row = [&](const R& now) {
      R y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[kBack][v] = to_f32<T>(now.e[v]);
        float s = b[v];
#pragma unroll
        for (int j = 0; j < NT; ++j) s = fmaf(w[j][v], f[j][v], s);
        y.e[v] = from_f32<T>(a.silu ? silu<T>(s) : s);
#pragma unroll
        for (int j = 0; j < kBack; ++j) f[j][v] = f[j + 1][v];
      }
      *reinterpret_cast<R*>(out + t * a.ldo) = y;
    };
    constexpr int kBatch = 8;
    while (t + kBatch <= end) {
      R now[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) now[i] = *reinterpret_cast<const R*>(x + (t + i) * a.ldx);
#pragma unroll
      for (int i = 0; i < kBatch; ++i, ++t) row(now[i]);
    }
    for (; t < end; ++t) row(*reinterpret_cast<const R*>(x + t * a.ldx));
  }
}

template <typename T, int V>
int launch_conv(ConvArgs a, int taps, cudaStream_t s) {
  const int blocks = (a.C + 128 * V - 1) / (128 * V), rows = a.np > 0 ? a.T - a.nd : 0;
  // longer strips while there are four of them per SM
  a.strip = kStrip;
  while (a.strip < 64 && static_cast<long long>(rows) * blocks >= 8ll * a.strip * sm_count()) a.strip *= 2;
  const dim3 grid(a.nd + (rows + a.strip - 1) / a.strip, blocks);
  if (grid.x == 0) return 0;
  switch (taps) {
#define CONV(n) case n: return launch_overlapped(causal_conv_kernel<T, n, V>, grid, dim3(128), 0, s, a)
    CONV(1); CONV(2); CONV(3); CONV(4); CONV(5); CONV(6); CONV(7); CONV(8);
#undef CONV
  }
  return -8;
}
template <typename T>
int conv_any(const ConvArgs& a, int taps, bool wide, cudaStream_t s) {
  return wide ? launch_conv<T, 4>(a, taps, s) : launch_conv<T, 1>(a, taps, s);
}

}  // namespace selective
}  // namespace b200

// The arguments of a call come packed, as the launchers pack them (ops/cuda.py): converting each of them one by one took
// longer than the kernels of small steps.
namespace {
struct ConvCall {
  const void* x;
  const float *w, *bias;
  void *ring, *out;
  const long long* positions;
  const int *slots, *wslots, *cu_q;
  long long ldx, ldo;
  int taps, num_slots, T, C, nd, np, silu, wide, dtype;
};
}  // namespace

// Short causal convolution of a step's rows.  dtype: 0 bf16, 1 fp16, 2 fp32; taps 1 .. 8; wide: rows, ring, weights, bias
// and out may be read four elements at a time.  ring may be null (every portion starts from zeros).
B200_API int b200_causal_conv(const void* call, void* stream) {
  using namespace b200::selective;
  const ConvCall& k = *static_cast<const ConvCall*>(call);
  if (k.T <= 0 || k.C <= 0 || k.nd + k.np <= 0) return 0;
  ConvArgs a;
  a.x = k.x; a.w = k.w; a.bias = k.bias; a.ring = k.taps > 1 ? k.ring : nullptr; a.out = k.out;
  a.positions = k.positions; a.slots = k.slots; a.wslots = k.wslots; a.cu_q = k.cu_q; a.ldx = k.ldx; a.ldo = k.ldo;
  a.T = k.T; a.C = k.C; a.num_slots = k.num_slots; a.nd = k.nd; a.np = k.np; a.silu = k.silu; a.strip = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (k.dtype) {
    case 0: return conv_any<__nv_bfloat16>(a, k.taps, k.wide, s);
    case 1: return conv_any<__half>(a, k.taps, k.wide, s);
    case 2: return conv_any<float>(a, k.taps, k.wide, s);
  }
  return -8;
}


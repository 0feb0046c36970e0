// Operators of a state-space mixer between its projections (sm_100a), over the rows of a step: nd
// single tokens, one per request, then the portions of np prompts (offsets behind row nd in cu_q).
//
//   causal_conv      c_t = act(bias + sum_j w[j] x of (taps - 1 - j) tokens ago), per channel
//   selective_step   one token of every request through the scan
//   selective_scan   h_t = exp(dt_t A) h_(t-1) + dt_t x_t B_t,  y_t = C_t . h_t + d x_t, over portions
//
// State of a request, read in one slot and left in another (usually the same):
//   ring   [slot, taps - 1, channels] in the model's type: row p % (taps - 1) holds the input of position p
//   state  [slot, columns, N] fp32
// A portion that starts at position 0 starts from zeros whatever the slot holds, so slots need no
// clearing.  A request whose slot is outside the state (padding of a captured batch) gives rows of
// zeros and touches no state; one whose write slot is outside leaves its state nowhere.
//
// Columns: a head holds `width` columns of x, each with N numbers of state.  Rates per head (a_log
// [heads]): one step size and one decay per head and token.  Rates per channel (a_log [columns, N]): a
// step size per column, a decay per column and number; the heads are then the groups that share B
// and C.
#include "selective.cuh"

namespace b200 {
namespace selective {

// V neighbouring elements: 16 bytes where V > 1
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
template <typename T>
constexpr int kWide = 16 / sizeof(T);

// ---------------------------------------------------------------------------
// short causal convolution
// ---------------------------------------------------------------------------
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
  int T, C, num_slots, nd, np, silu;
};

constexpr int kMaxTaps = 8;
constexpr int kStrip = 16;                       // rows of prompts that a CTA walks
static_assert(kStrip >= kMaxTaps, "a row that reads the ring lies in the strip of its portion's first row");

// A CTA: a strip of rows, V channels per thread.  A single token is a strip of its own; strips of
// prompts are kStrip rows long, but that the first taps - 1 rows of a portion stay in one strip: they
// are the only ones that read the ring, and the threads that read a channel of it then write it, so
// reading and writing need no second launch.
// Bytes bound it: rows are read once (those in front of a strip a second time, from L2) and written once.
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
    lo = a.nd + (strip - a.nd) * kStrip;
    hi = min(lo + kStrip, a.T);
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
  const R* ring = nullptr;
  auto ring_row = [&](int slot, long long pos) {
    return reinterpret_cast<R*>(static_cast<T*>(a.ring) +
                                (static_cast<long long>(slot) * kBack + pos % kBack) * a.C + c);
  };
  float w[NT][V], b[V];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) w[j][v] = a.w[static_cast<long long>(j) * a.C + c + v];
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = a.bias ? a.bias[c + v] : 0.0f;

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
          if (row >= po.first) {
            *ring_row(ws, p) = *reinterpret_cast<const R*>(x + row * a.ldx);
          } else if (p >= 0 && ws != slot) {     // row - po.first in [-kBack, -1]
#pragma unroll
            for (int i = 0; i < kBack; ++i)
              if (i == row - po.first + kBack) *ring_row(ws, p) = old[i];
          }
        }
      }
    }
    for (; t < end; ++t) {
      const R now = *reinterpret_cast<const R*>(x + t * a.ldx);
      R y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s = b[v];
#pragma unroll
        for (int j = 0; j < kBack; ++j) s = fmaf(w[j][v], to_f32<T>(old[j].e[v]), s);
        s = fmaf(w[kBack][v], to_f32<T>(now.e[v]), s);
        if (a.silu) s = silu<T>(s);
        y.e[v] = from_f32<T>(padding ? 0.0f : s);
      }
      *reinterpret_cast<R*>(out + t * a.ldo) = y;
#pragma unroll
      for (int j = 0; j + 1 < kBack; ++j) old[j] = old[j + 1];
      if (kBack > 0) old[kBack > 0 ? kBack - 1 : 0] = now;
    }
  }
}

// ---------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------
// One token per request.  A row of N numbers of state is spread over LPR lanes, four numbers (one
// where V is 1) at a time; a warp takes kRows rows per lane group at once, so that their loads are under
// way together.  The state's bytes bound it: read once, written once.
template <typename T, bool CH, int LPR, int NC, int V>
__global__ void __launch_bounds__(128) selective_step_kernel(const ScanArgs a) {
  constexpr int kRows = NC > 1 ? 4 : 8, kGroups = 32 / LPR;
  grid_release_small();
  grid_wait();
  const int r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = lane & (LPR - 1), grp = lane / LPR;
  const int cols = a.heads * a.width;
  const int c0 = (blockIdx.x * 4 + warp) * kRows * kGroups + grp;    // column of row i: c0 + i * kGroups
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  const bool padding = a.state != nullptr && (slot < 0 || slot >= a.num_slots);
  T* out = static_cast<T*>(a.out) + r * a.ldo;
  if (padding) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (l == 0 && c0 + i * kGroups < cols) out[c0 + i * kGroups] = from_f32<T>(0.0f);
    return;
  }
  const bool old = a.state != nullptr && a.positions[r] != 0;
  const int ws = a.state != nullptr ? a.wslots[r] : -1;
  const bool keep = ws >= 0 && ws < a.num_slots;
  const long long pitch = static_cast<long long>(cols) * a.N;
  float h[kRows][NC][V];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int col = c0 + i * kGroups;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int n = (l + LPR * k) * V;
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][k][v] = 0.0f;
      if (old && col < cols && n < a.N) {
        const float* src = a.state + slot * pitch + static_cast<long long>(col) * a.N + n;
        if constexpr (V == 4) {
          const float4 q = *reinterpret_cast<const float4*>(src);
          h[i][k][0] = q.x; h[i][k][1] = q.y; h[i][k][2] = q.z; h[i][k][3] = q.w;
        } else {
          h[i][k][0] = *src;
        }
      }
    }
  }
  float bb[NC][V], cc[NC][V];
  int group = -1, head = -1;
  float dt = 0.0f, decay = 0.0f;
  float y[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int col = min(c0 + i * kGroups, cols - 1);
    const int hd = col / a.width;
    const int g = hd / (a.heads / a.groups);
    if (g != group) {
      group = g;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int n = (l + LPR * k) * V + v;
          const bool in = n < a.N;
          bb[k][v] = in ? to_f32<T>(static_cast<const T*>(a.b)[r * a.ldb + g * a.N + n]) : 0.0f;
          cc[k][v] = in ? to_f32<T>(static_cast<const T*>(a.c)[r * a.ldc + g * a.N + n]) : 0.0f;
        }
    }
    if (CH || hd != head) {
      head = hd;
      dt = step_size<T>(a, r, CH ? col : hd);
      if (!CH) decay = expf(-dt * expf(a.a_log[hd]));
    }
    const float x = to_f32<T>(static_cast<const T*>(a.x)[r * a.ldx + col]);
    const float dx = dt * x;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int n = (l + LPR * k) * V + v;
        float e = decay;
        if (CH) e = n < a.N ? expf(-dt * expf(a.a_log[static_cast<long long>(col) * a.N + n])) : 0.0f;
        h[i][k][v] = fmaf(e, h[i][k][v], dx * bb[k][v]);
        s = fmaf(h[i][k][v], cc[k][v], s);
      }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (a.d != nullptr) s = fmaf(a.d[CH ? col : hd], x, s);
    if (a.z != nullptr) s *= silu<T>(to_f32<T>(static_cast<const T*>(a.z)[r * a.ldz + col]));
    y[i] = s;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int col = c0 + i * kGroups;
    if (col >= cols) continue;
    if (l == 0) out[col] = from_f32<T>(y[i]);
    if (!keep) continue;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int n = (l + LPR * k) * V;
      if (n >= a.N) continue;
      float* dst = a.state + ws * pitch + static_cast<long long>(col) * a.N + n;
      if constexpr (V == 4)
        *reinterpret_cast<float4*>(dst) = make_float4(h[i][k][0], h[i][k][1], h[i][k][2], h[i][k][3]);
      else
        *dst = h[i][k][0];
    }
  }
}

// Portions of prompts, token after token.  A CTA holds kCols columns of one head of one request; LPC
// lanes share a column, RPL numbers of its state each, in registers.  Inputs are staged through shared memory
// kChunk tokens at a time.
constexpr int kChunk = 16;

template <typename T, bool CH, int LPC, int RPL>
__global__ void __launch_bounds__(128) selective_scan_kernel(const ScanArgs a) {
  constexpr int NP = LPC * RPL, kCols = 128 / LPC;
  __shared__ __align__(16) float sb[kChunk][NP], sc[kChunk][NP];
  __shared__ float sdt[kChunk][kCols], sx[kChunk][kCols], sy[kChunk][kCols];
  __shared__ float sdecay[kChunk];
  grid_release_small();
  grid_wait();
  const int r = a.nd + blockIdx.x, hd = blockIdx.y, p0 = blockIdx.z * kCols;
  const int l = threadIdx.x & (LPC - 1), col = threadIdx.x / LPC;
  const int cols = min(kCols, a.width - p0);
  const int c0 = hd * a.width + p0;                          // first column of the CTA
  const int g = hd / (a.heads / a.groups);
  const Portion po = portion_of(r, a.nd, a.cu_q, a.T);
  if (po.first >= po.end) return;
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  T* out = static_cast<T*>(a.out) + c0;
  if (a.state != nullptr && (slot < 0 || slot >= a.num_slots)) {
    for (int t = po.first; t < po.end; ++t)
      if (threadIdx.x < cols) out[t * a.ldo + threadIdx.x] = from_f32<T>(0.0f);
    return;
  }
  const bool old = a.state != nullptr && a.positions[po.first] != 0;
  const int ws = a.state != nullptr ? a.wslots[r] : -1;
  const bool keep = ws >= 0 && ws < a.num_slots;
  const long long pitch = static_cast<long long>(a.heads) * a.width * a.N;
  const long long at = static_cast<long long>(c0 + col) * a.N;
  float h[RPL], rate[RPL];
#pragma unroll
  for (int i = 0; i < RPL; ++i) {
    const int n = (i / 4 * LPC + l) * 4 + i % 4;
    const bool in = n < a.N && col < cols;
    h[i] = old && in ? a.state[slot * pitch + at + n] : 0.0f;
    rate[i] = CH && in ? -expf(a.a_log[at + n]) * kLog2e : 0.0f;
  }
  const float head_rate = CH ? 0.0f : -expf(a.a_log[hd]);

  for (int t0 = po.first; t0 < po.end; t0 += kChunk) {
    const int n = min(kChunk, po.end - t0);
    for (int e = threadIdx.x; e < n * NP; e += 128) {
      const int i = e / NP, k = e % NP;
      const long long t = t0 + i;
      sb[i][k] = k < a.N ? to_f32<T>(static_cast<const T*>(a.b)[t * a.ldb + g * a.N + k]) : 0.0f;
      sc[i][k] = k < a.N ? to_f32<T>(static_cast<const T*>(a.c)[t * a.ldc + g * a.N + k]) : 0.0f;
    }
    for (int e = threadIdx.x; e < n * cols; e += 128) {
      const int i = e / cols, k = e % cols;
      const long long t = t0 + i;
      sx[i][k] = to_f32<T>(static_cast<const T*>(a.x)[t * a.ldx + c0 + k]);
      if (CH) sdt[i][k] = step_size<T>(a, t, c0 + k);
    }
    if (!CH && threadIdx.x < n) {
      const float dt = step_size<T>(a, t0 + threadIdx.x, hd);
      sdt[threadIdx.x][0] = dt;
      sdecay[threadIdx.x] = expf(dt * head_rate);
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const float dt = CH ? sdt[i][col < cols ? col : 0] : sdt[i][0];
      const float dx = dt * sx[i][col < cols ? col : 0];
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < RPL; k += 4) {
        const float4 bq = *reinterpret_cast<const float4*>(&sb[i][(k / 4 * LPC + l) * 4]);
        const float4 cq = *reinterpret_cast<const float4*>(&sc[i][(k / 4 * LPC + l) * 4]);
        const float be[4] = {bq.x, bq.y, bq.z, bq.w}, ce[4] = {cq.x, cq.y, cq.z, cq.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = CH ? exp2f(dt * rate[k + j]) : sdecay[i];
          h[k + j] = fmaf(e, h[k + j], dx * be[j]);
          s = fmaf(h[k + j], ce[j], s);
        }
      }
#pragma unroll
      for (int o = 1; o < LPC; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (l == 0) sy[i][col] = s;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n * cols; e += 128) {
      const int i = e / cols, k = e % cols;
      const long long t = t0 + i;
      float y = sy[i][k];
      if (a.d != nullptr) y = fmaf(a.d[CH ? c0 + k : hd], sx[i][k], y);
      if (a.z != nullptr) y *= silu<T>(to_f32<T>(static_cast<const T*>(a.z)[t * a.ldz + c0 + k]));
      out[t * a.ldo + k] = from_f32<T>(y);
    }
    __syncthreads();
  }
  if (keep && col < cols) {
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      const int n = (i / 4 * LPC + l) * 4 + i % 4;
      if (n < a.N) a.state[ws * pitch + at + n] = h[i];
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T, int V>
int launch_conv(const ConvArgs& a, int taps, cudaStream_t s) {
  const int prompt = a.np > 0 ? (a.T - a.nd + kStrip - 1) / kStrip : 0;
  const dim3 grid(a.nd + prompt, (a.C + 128 * V - 1) / (128 * V));
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
  return wide ? launch_conv<T, kWide<T>>(a, taps, s) : launch_conv<T, 1>(a, taps, s);
}

template <typename T, bool CH>
int launch_step(const ScanArgs& a, cudaStream_t s) {
  const int cols = a.heads * a.width;
#define STEP(LPR, NC, V)                                                              \
  launch_overlapped(selective_step_kernel<T, CH, LPR, NC, V>,                         \
                    dim3((cols + 4 * (NC > 1 ? 4 : 8) * (32 / LPR) - 1) /             \
                             (4 * (NC > 1 ? 4 : 8) * (32 / LPR)), a.nd),              \
                    dim3(128), 0, s, a)
  if (a.N % 4 == 0) {
    if (a.N <= 16) return STEP(4, 1, 4);
    if (a.N <= 32) return STEP(8, 1, 4);
    if (a.N <= 64) return STEP(16, 1, 4);
    if (a.N <= 128) return STEP(32, 1, 4);
    return STEP(32, 2, 4);
  }
  if (a.N <= 32) return STEP(32, 1, 1);
  if (a.N <= 128) return STEP(32, 4, 1);
  return STEP(32, 8, 1);
#undef STEP
}

template <typename T, bool CH>
int launch_scan(const ScanArgs& a, cudaStream_t s) {
#define SCAN(LPC, RPL)                                                                                        \
  launch_overlapped(selective_scan_kernel<T, CH, LPC, RPL>,                                                   \
                    dim3(a.np, a.heads, (a.width + 128 / LPC - 1) / (128 / LPC)), dim3(128), 0, s, a)
  if (a.N <= 16) return SCAN(4, 4);
  if (a.N <= 32) return SCAN(4, 8);
  if (a.N <= 64) return SCAN(8, 8);
  if (a.N <= 128) return SCAN(8, 16);
  return SCAN(16, 16);
#undef SCAN
}

template <typename T, bool CH>
int scan_any(const ScanArgs& a, cudaStream_t s) {
  if (a.nd > 0) {
    const int rc = launch_step<T, CH>(a, s);
    if (rc != 0) return rc;
  }
  if (a.np == 0) return 0;
  if constexpr (!CH && std::is_same<T, __nv_bfloat16>::value)
    if (heads_by_tiles(a)) return launch_heads_by_tiles(a, s);
  return launch_scan<T, CH>(a, s);
}

}  // namespace selective
}  // namespace b200

// Short causal convolution of a step's rows.  dtype: 0 bf16, 1 fp16, 2 fp32; taps 1 .. 8; wide: rows, ring and
// out may be read 16 bytes at a time.  ring may be null (every portion starts from zeros).
B200_API int b200_causal_conv(const void* x, long long ldx, const float* w, int taps, const float* bias, void* ring,
                              int num_slots, const long long* positions, const int* slots, const int* wslots,
                              const int* cu_q, void* out, long long ldo, int T, int C, int nd, int np, int silu,
                              int wide, int dtype, void* stream) {
  using namespace b200::selective;
  if (T <= 0 || C <= 0 || nd + np <= 0) return 0;
  ConvArgs a;
  a.x = x; a.w = w; a.bias = bias; a.ring = taps > 1 ? ring : nullptr; a.out = out; a.positions = positions;
  a.slots = slots; a.wslots = wslots; a.cu_q = cu_q; a.ldx = ldx; a.ldo = ldo; a.T = T; a.C = C;
  a.num_slots = num_slots; a.nd = nd; a.np = np; a.silu = silu;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return conv_any<__nv_bfloat16>(a, taps, wide, s);
    case 1: return conv_any<__half>(a, taps, wide, s);
    case 2: return conv_any<float>(a, taps, wide, s);
  }
  return -8;
}

// Selective scan of a step's rows; per_channel: a_log [heads * width, N] and a step size per column, else
// a_log [heads] and a step size per head.  state may be null (every portion starts from zeros).
B200_API int b200_selective_scan(const void* x, long long ldx, const void* dt, long long lddt, int dt_f32,
                                 const void* b, long long ldb, const void* c, long long ldc, const void* z,
                                 long long ldz, const float* a_log, int per_channel, const float* d,
                                 const float* dt_bias, int softplus, float dt_min, float dt_max, float* state,
                                 int num_slots, const long long* positions, const int* slots, const int* wslots,
                                 const int* cu_q, void* out, long long ldo, int T, int heads, int width, int N,
                                 int groups, int nd, int np, int wide, int dtype, void* stream) {
  using namespace b200::selective;
  if (T <= 0 || heads <= 0 || width <= 0 || nd + np <= 0) return 0;
  if (N < 1 || N > 256) return -8;
  ScanArgs a;
  a.x = x; a.dt = dt; a.b = b; a.c = c; a.z = z; a.out = out; a.a_log = a_log; a.d = d; a.dt_bias = dt_bias;
  a.state = state; a.positions = positions; a.slots = slots; a.wslots = wslots; a.cu_q = cu_q;
  a.ldx = ldx; a.lddt = lddt; a.ldb = ldb; a.ldc = ldc; a.ldz = ldz; a.ldo = ldo;
  a.dt_min = dt_min; a.dt_max = dt_max; a.T = T; a.heads = heads; a.width = width; a.N = N; a.groups = groups;
  a.num_slots = num_slots; a.nd = nd; a.np = np; a.dt_f32 = dt_f32; a.softplus = softplus;
  a.wide = wide;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return per_channel ? scan_any<__nv_bfloat16, true>(a, s) : scan_any<__nv_bfloat16, false>(a, s);
    case 1: return per_channel ? scan_any<__half, true>(a, s) : scan_any<__half, false>(a, s);
    case 2: return per_channel ? scan_any<float, true>(a, s) : scan_any<float, false>(a, s);
  }
  return -8;
}

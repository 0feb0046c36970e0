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
  int T, C, num_slots, nd, np, silu, strip;
};

constexpr int kMaxTaps = 8;
constexpr int kStrip = 16;                       // rows of prompts that a CTA walks, at least
static_assert(kStrip >= kMaxTaps, "a row that reads the ring lies in the strip of its portion's first row");

// A CTA: a strip of rows, V channels per thread.  A single token is a strip of its own; strips of
// prompts are a.strip rows long, but that the first taps - 1 rows of a portion stay in one strip: they
// are the only ones that read the ring, and the threads that read a channel of it then write it, so
// reading and writing need no second launch.
// Bytes bound it: rows are read once (those in front of a strip a second time, from L2) and written once.  Four
// channels per thread and kBatch rows under way: with eight channels the registers of the window leave 12 warps an
// SM (8192 rows of 10240 channels 107 us, so 87); strips of 64 rows make the search for a row's request and
// the window in front of the strip seldom (16 rows: 8 us more).
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

// ---------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------
// Sums of ROWS values over LPR neighbouring lanes, lane by lane fewer rows: while there are rows to part, two halves of
// the lanes take a half of the rows each.  Leaves kLeft sums per lane, of rows from `first` on.
template <int ROWS, int LPR>
struct RowSums {
  static constexpr int kParted = ROWS < LPR ? ROWS : LPR, kLeft = ROWS / kParted;
  float v[kLeft];
  int first;
  __device__ __forceinline__ RowSums(float (&s)[ROWS], int l) {
    first = 0;
#pragma unroll
    for (int half = ROWS / 2, o = LPR / 2; half >= kLeft && o > 0; half >>= 1, o >>= 1) {
      const bool up = l & o;
      if (up) first += half;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float mine = up ? s[i + half] : s[i], theirs = up ? s[i] : s[i + half];
        s[i] = mine + __shfl_xor_sync(0xffffffffu, theirs, o);
      }
    }
#pragma unroll
    for (int o = LPR / kParted / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < kLeft; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
#pragma unroll
    for (int i = 0; i < kLeft; ++i) v[i] = s[i];
  }
  __device__ __forceinline__ static bool keeps(int l) { return l % (LPR / kParted) == 0; }
};

// Four neighbours of a row of B or C.
template <typename T, bool WIDE>
__device__ __forceinline__ float4 load_four(const T* p, bool in) {
  Raw<T, 4> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.e[i] = from_f32<T>(0.0f);
  if (in) {
    if (WIDE) {
      v = *reinterpret_cast<const Raw<T, 4>*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.e[i] = p[i];
    }
  }
  return make_float4(to_f32<T>(v.e[0]), to_f32<T>(v.e[1]), to_f32<T>(v.e[2]), to_f32<T>(v.e[3]));
}
// a state's four numbers after a token, and their part of the read-out
__device__ __forceinline__ float update(float4& h, float2 e0, float2 e1, float2 dx, const float4& b, const float4& c) {
  const float2 h0 = __ffma2_rn(e0, make_float2(h.x, h.y), __fmul2_rn(dx, make_float2(b.x, b.y)));
  const float2 h1 = __ffma2_rn(e1, make_float2(h.z, h.w), __fmul2_rn(dx, make_float2(b.z, b.w)));
  const float2 s = __ffma2_rn(h1, make_float2(c.z, c.w), __fmul2_rn(h0, make_float2(c.x, c.y)));
  h = make_float4(h0.x, h0.y, h1.x, h1.y);
  return s.x + s.y;
}

// One token per request, rates per head, where a warp's columns belong to one head (width a multiple of their number)
// and N is one of 4: a row of N numbers is spread over LPR lanes, NC times four each.  The state's bytes bound it: a warp
// has 4 KB of it under way at once, and what a head's columns share is worked out once per warp (by row, 70 per cent of the
// issue slots went into that: 96 requests of 80 heads of 64 x 128 in 113 us, 4.4 TB/s).
template <typename T, int LPR, int NC, bool WIDE>
__global__ void __launch_bounds__(128) heads_step_kernel(const ScanArgs a) {
  constexpr int kRows = NC > 1 ? 4 : 8, kGroups = 32 / LPR, kWarpCols = kRows * kGroups;
  grid_release_small();
  grid_wait();
  const int r = blockIdx.y, lane = threadIdx.x & 31, l = lane & (LPR - 1), grp = lane / LPR;
  const int cols = a.heads * a.width;
  const int c0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kWarpCols;
  if (c0 >= cols) return;
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  const int ws = a.state != nullptr ? a.wslots[r] : -1;
  const bool old = a.state != nullptr && a.positions[r] != 0;
  T* out = static_cast<T*>(a.out) + r * a.ldo + c0;
  if (a.state != nullptr && (slot < 0 || slot >= a.num_slots)) {
    for (int i = lane; i < kWarpCols; i += 32) out[i] = from_f32<T>(0.0f);
    return;
  }
  const long long pitch = static_cast<long long>(cols) * a.N;
  const long long at = static_cast<long long>(c0 + grp) * a.N + l * 4;
  float4 h[kRows][NC];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      h[i][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (old && (l + LPR * k) * 4 < a.N)
        h[i][k] = *reinterpret_cast<const float4*>(a.state + slot * pitch + at + i * kGroups * a.N + LPR * k * 4);
    }
  const int hd = c0 / a.width, g = hd / (a.heads / a.groups);
  // x of the warp's columns: column j in lane j % 32
  float x[kWarpCols / 32 + 1];
#pragma unroll
  for (int j = 0; j <= (kWarpCols - 1) / 32; ++j)
    x[j] = j * 32 + lane < kWarpCols ? to_f32<T>(static_cast<const T*>(a.x)[r * a.ldx + c0 + j * 32 + lane]) : 0.0f;
  float4 b[NC], c[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int n = (l + LPR * k) * 4;
    b[k] = load_four<T, WIDE>(static_cast<const T*>(a.b) + r * a.ldb + g * a.N + n, n < a.N);
    c[k] = load_four<T, WIDE>(static_cast<const T*>(a.c) + r * a.ldc + g * a.N + n, n < a.N);
  }
  const float dt = step_size<T>(a, r, hd);
  const float decay = expf(-dt * expf(a.a_log[hd]));
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float dx = dt * __shfl_sync(0xffffffffu, x[i * kGroups / 32], (i * kGroups + grp) & 31);
    s[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      s[i] += update(h[i][k], make_float2(decay, decay), make_float2(decay, decay), make_float2(dx, dx), b[k], c[k]);
  }
  if (ws >= 0 && ws < a.num_slots) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if ((l + LPR * k) * 4 < a.N)
          *reinterpret_cast<float4*>(a.state + ws * pitch + at + i * kGroups * a.N + LPR * k * 4) = h[i][k];
  }
  const RowSums<kRows, LPR> sums(s, l);
  const float skip = a.d != nullptr ? a.d[hd] : 0.0f;
#pragma unroll
  for (int i = 0; i < sums.kLeft; ++i) {
    const int j = (sums.first + i) * kGroups + grp;      // column of the warp
    float xv = 0.0f;
#pragma unroll
    for (int m = 0; m <= (kWarpCols - 1) / 32; ++m) {
      const float v = __shfl_sync(0xffffffffu, x[m], j & 31);
      if (j / 32 == m) xv = v;
    }
    float y = fmaf(skip, xv, sums.v[i]);
    if (a.z != nullptr) y *= silu<T>(to_f32<T>(static_cast<const T*>(a.z)[r * a.ldz + c0 + j]));
    if (sums.keeps(l)) out[j] = from_f32<T>(y);
  }
}

// One token per request, rates per channel, N a multiple of 4 up to 128: a warp holds 32 / LPR columns of RQ requests, so
// that rates and skips are fetched and worked out once for them.
template <typename T, int LPR, int RQ, bool WIDE>
__global__ void __launch_bounds__(128) channels_step_kernel(const ScanArgs a) {
  constexpr int kGroups = 32 / LPR;
  grid_release_small();
  grid_wait();
  const int lane = threadIdx.x & 31, l = lane & (LPR - 1), grp = lane / LPR;
  const int cols = a.heads * a.width;
  const int c0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kGroups;
  if (c0 >= cols) return;
  const bool in = c0 + grp < cols && l * 4 < a.N, mine = c0 + grp < cols;
  const int col = min(c0 + grp, cols - 1), n = l * 4;
  const int g = col / (cols / a.groups);
  const int r0 = blockIdx.y * RQ;
  const long long pitch = static_cast<long long>(cols) * a.N, at = static_cast<long long>(col) * a.N + n;
  float4 h[RQ], b[RQ], c[RQ];
  float x[RQ], dt[RQ], z[RQ];
  int ws[RQ];
  bool padding[RQ];
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const int r = min(r0 + i, a.nd - 1);
    const int slot = a.state != nullptr ? a.slots[r] : 0;
    ws[i] = a.state != nullptr && r0 + i < a.nd ? a.wslots[r] : -1;
    padding[i] = a.state != nullptr && (slot < 0 || slot >= a.num_slots);
    if (padding[i]) ws[i] = -1;
    h[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.state != nullptr && !padding[i] && in && a.positions[r] != 0)
      h[i] = *reinterpret_cast<const float4*>(a.state + slot * pitch + at);
  }
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const int r = min(r0 + i, a.nd - 1);
    x[i] = to_f32<T>(static_cast<const T*>(a.x)[r * a.ldx + col]);
    dt[i] = a.dt_f32 ? static_cast<const float*>(a.dt)[r * a.lddt + col]
                     : to_f32<T>(static_cast<const T*>(a.dt)[r * a.lddt + col]);
    z[i] = a.z != nullptr ? to_f32<T>(static_cast<const T*>(a.z)[r * a.ldz + col]) : 0.0f;
    b[i] = load_four<T, WIDE>(static_cast<const T*>(a.b) + r * a.ldb + g * a.N + n, in);
    c[i] = load_four<T, WIDE>(static_cast<const T*>(a.c) + r * a.ldc + g * a.N + n, in);
  }
  float4 rate = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (in) rate = *reinterpret_cast<const float4*>(a.a_log + at);
  rate = make_float4(-expf(rate.x) * kLog2e, -expf(rate.y) * kLog2e, -expf(rate.z) * kLog2e, -expf(rate.w) * kLog2e);
  const float bias = a.dt_bias != nullptr ? a.dt_bias[col] : 0.0f, skip = a.d != nullptr ? a.d[col] : 0.0f;
  float s[RQ];
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const float step = step_from<T>(a, dt[i], bias), dx = step * x[i];
    const float2 p0 = __fmul2_rn(make_float2(step, step), make_float2(rate.x, rate.y));
    const float2 p1 = __fmul2_rn(make_float2(step, step), make_float2(rate.z, rate.w));
    const float2 e0 = make_float2(exp2_fast(p0.x), exp2_fast(p0.y)), e1 = make_float2(exp2_fast(p1.x), exp2_fast(p1.y));
    s[i] = update(h[i], e0, e1, make_float2(dx, dx), b[i], c[i]);
    s[i] = in ? s[i] : 0.0f;
    if (in && ws[i] >= 0 && ws[i] < a.num_slots) *reinterpret_cast<float4*>(a.state + ws[i] * pitch + at) = h[i];
  }
  const RowSums<RQ, LPR> sums(s, l);
#pragma unroll
  for (int i = 0; i < sums.kLeft; ++i) {
    const int k = sums.first + i, r = r0 + k;
    if (!mine || !sums.keeps(l) || r >= a.nd) continue;
    float xv = 0.0f, zv = 0.0f;
    bool none = false;
#pragma unroll
    for (int m = 0; m < RQ; ++m)
      if (m == k) {
        xv = x[m];
        zv = z[m];
        none = padding[m];
      }
    float y = fmaf(skip, xv, sums.v[i]);
    if (a.z != nullptr) y *= silu<T>(zv);
    static_cast<T*>(a.out)[r * a.ldo + col] = from_f32<T>(none ? 0.0f : y);
  }
}

// One token per request, in general.  A row of N numbers of state is spread over LPR lanes, four numbers (one
// where V is 1) at a time; a warp takes kRows rows per lane group at once, so that their loads are under
// way together.
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

// Portions of prompts, token after token.  A CTA holds the columns of one request that kCore / LPC lane groups
// make: a column's numbers of state lie in the registers of LPC lanes, NPL each, and a token costs a number one
// decay (rates per channel: a power of two, which the special function unit does 16 of per clock and SM: it bounds
// them), two multiply-adds and a product.  Inputs pass through shared memory kTok tokens at a time.  While the core
// warps walk tile i, four warps of helpers turn tile i + 1 into step sizes and factors, finish tile i - 1 (skip,
// gate, store) and copy tile i + 3, each helper the eight neighbouring elements that it copied itself; one
// barrier per tile.  (Without helpers, all warps doing both in turn, 235 us for 2048 tokens of 8192 channels: what is
// done per element is half of the instructions, and the chain along the tokens leaves the scheduler idle.)
// The sum over the lanes of a column is the helpers': up to four lanes leave a part of it each; where there are
// more, pairs of lanes trade the parts of two tokens first, so that each ends up with those of its own token.  With
// few numbers per lane, decays and inputs of eight tokens are made before their chain is walked.
template <int LPC>
constexpr int kCore = LPC >= 8 ? 256 : 128;
constexpr int kHelp = 128;
template <int LPC, int NPL>
constexpr int kTok = LPC == 2 || LPC * NPL >= 128 ? 16 : 32;

template <typename T>
struct __align__(16) Eight {
  T e[8];
};
// Eight neighbours of a row, `n` of them there, into shared memory, zeros behind them.
template <typename T, bool WIDE>
__device__ __forceinline__ void copy_eight(Eight<T>* to, const T* from, int n) {
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to) + 16 * i),
                   "l"(reinterpret_cast<const char*>(from) + 16 * i), "r"(n > 0 ? 16 : 0)
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) to->e[i] = i < n ? from[i] : from_f32<T>(0.0f);
  }
}

template <typename T, bool CH, int LPC, int NPL>
struct ScanTile {
  static constexpr int kTokens = kTok<LPC, NPL>, kCols = kCore<LPC> / LPC, kVecs = kTokens * kCols / 8;
  // as they are in memory, by the helper that copied them: rows for four tiles, the rest for two
  Eight<T> x[4][kVecs], z[4][kVecs], bc_raw[2][2 * kTokens * LPC * NPL / 8];
  Eight<float> dt[2][CH ? kVecs : 1];                        // (rows of 16 bits: the first half)
  // by tile parity
  float bc[2][2][kTokens][LPC * NPL];                        // B, C
  float2 d[2][kTokens][kCols];                               // step size (rates per head: decay), step size times x
  static constexpr int kParts = LPC < 4 ? LPC : 4;
  // Parts of C . h.  A helper reads the parts of eight columns in a row, 128 bytes, and its neighbours those of the next
  // ones: column c of token t lies in place c ^ key, so that they start in different banks.
  float y[2][kTokens][kCols][kParts];
  static __device__ __forceinline__ int key(int t, int c) { return (t * (kCols / 8) + c / 8) & 7; }
};

template <typename T, bool CH, int LPC, int NPL, bool WIDE>
__global__ void __launch_bounds__(kCore<LPC> + kHelp) selective_scan_kernel(const ScanArgs a) {
  using Tile = ScanTile<T, CH, LPC, NPL>;
  constexpr int NP = LPC * NPL, kCols = Tile::kCols, TOK = Tile::kTokens;
  constexpr int kHalf = NPL / 2;
  static_assert(Tile::kVecs <= kHelp, "one vector of eight per helper");
  extern __shared__ float4 raw[];
  Tile& sm = *reinterpret_cast<Tile*>(raw);
  // The next kernel is let go by the ends of the CTAs: CTAs of a next scan that came early would be placed
  // beside the running ones, several on an SM and none on others (two such passes 427 us each, so 253).
  grid_wait();
  const int r = a.nd + blockIdx.x, g = blockIdx.y, per = a.heads / a.groups * a.width;
  const int p0 = blockIdx.z * kCols, cols = min(kCols, per - p0);
  const int c0 = g * per + p0;                               // first column of the CTA
  const Portion po = portion_of(r, a.nd, a.cu_q, a.T);
  if (po.first >= po.end) return;
  const int tiles = (po.end - po.first + TOK - 1) / TOK;
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  T* out = static_cast<T*>(a.out) + c0;
  if (a.state != nullptr && (slot < 0 || slot >= a.num_slots)) {
    for (int t = po.first; t < po.end; ++t)
      if (threadIdx.x < cols) out[t * a.ldo + threadIdx.x] = from_f32<T>(0.0f);
    return;
  }

  if (threadIdx.x >= kCore<LPC>) {
    // ---------------- helpers ----------------
    const int me = threadIdx.x - kCore<LPC>;
    // eight elements of a tile: token vt, columns vc and on; what belongs to a column stays
    const int vt = me / (kCols / 8), vc = me % (kCols / 8) * 8;
    const int vn = me < Tile::kVecs ? max(0, min(8, cols - vc)) : 0;
    const bool one_head = !CH && a.width % 8 == 0;           // eight columns share a step size
    const T* bsrc = static_cast<const T*>(a.b) + g * a.N;
    const T* csrc = static_cast<const T*>(a.c) + g * a.N;
    uint32_t head_dt[2] = {0u, 0u};                          // rates per head: raw step sizes of two tiles under way
    auto bring = [&](int tile) {
      if (tile < tiles) {
        const int t0 = po.first + tile * TOK, n = po.end - t0;
        if (one_head && vt < n && vn > 0) {
          const long long k = static_cast<long long>(t0 + vt) * a.lddt + (c0 + vc) / a.width;
          uint32_t v;
          if (a.dt_f32 || sizeof(T) == 4) v = static_cast<const uint32_t*>(a.dt)[k];
          else v = static_cast<const unsigned short*>(a.dt)[k];
          if (tile & 1) head_dt[1] = v;
          else head_dt[0] = v;
        }
        if (me < Tile::kVecs) {
          const int here = vt < n ? vn : 0;
          const long long t = t0 + (here > 0 ? vt : 0);
          const int c = c0 + (here > 0 ? vc : 0);
          copy_eight<T, WIDE>(&sm.x[tile & 3][me], static_cast<const T*>(a.x) + t * a.ldx + c, here);
          if (a.z != nullptr) copy_eight<T, WIDE>(&sm.z[tile & 3][me], static_cast<const T*>(a.z) + t * a.ldz + c, here);
          if (CH) {
            Eight<float>* to = &sm.dt[tile & 1][me];
            if (a.dt_f32) copy_eight<float, WIDE>(to, static_cast<const float*>(a.dt) + t * a.lddt + c, here);
            else copy_eight<T, WIDE>(reinterpret_cast<Eight<T>*>(to), static_cast<const T*>(a.dt) + t * a.lddt + c, here);
          }
        }
        for (int e = me; e < 2 * TOK * NP / 8; e += kHelp) {
          const int m = e / (TOK * NP / 8), k = e / (NP / 8) % TOK, c = e % (NP / 8) * 8;
          const int here = k < n ? max(0, min(8, a.N - c)) : 0;
          copy_eight<T, WIDE>(&sm.bc_raw[tile & 1][e], (m == 0 ? bsrc : csrc) + (t0 + (here > 0 ? k : 0)) *
                              (m == 0 ? a.ldb : a.ldc) + (here > 0 ? c : 0), here);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    bring(0);
    bring(1);
    float2 bias[4], skip[4];
    float hrate[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int which = CH ? c0 + vc + i : (c0 + vc + i) / a.width;
      const bool in = i < vn;
      (i & 1 ? bias[i / 2].y : bias[i / 2].x) = in && a.dt_bias != nullptr ? a.dt_bias[which] : 0.0f;
      (i & 1 ? skip[i / 2].y : skip[i / 2].x) = in && a.d != nullptr ? a.d[which] : 0.0f;
      hrate[i] = !CH && in ? -expf(a.a_log[which]) : 0.0f;
    }
    // step sizes and factors; a token behind the portion has a step of 0, which leaves a state as it is
    auto convert = [&](int tile) {
      const int t0 = po.first + tile * TOK, here = vt < po.end - t0 ? vn : 0;
      if (me < Tile::kVecs) {
        const Eight<T> x = sm.x[tile & 3][me];
        float2 dt[4], decay[4];
        if (CH) {
          const Eight<float>* from = &sm.dt[tile & 1][me];
          float f[8];
          if (a.dt_f32) {
            const Eight<float> v = *from;
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v.e[i];
          } else {
            const Eight<T> v = *reinterpret_cast<const Eight<T>*>(from);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(v.e[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) dt[i] = make_float2(f[2 * i] + bias[i].x, f[2 * i + 1] + bias[i].y);
          if (a.softplus) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (sizeof(T) == 2) dt[i] = softplus_pair(dt[i]);
              else dt[i] = make_float2(softplus<T>(dt[i].x), softplus<T>(dt[i].y));
            }
          }
          if (a.limits) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dt[i] = make_float2(limited(a, dt[i].x), limited(a, dt[i].y));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) decay[i] = dt[i];
        } else {
          float step = 0.0f, e = 1.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i < here && (i == 0 || !one_head)) {
              if (one_head) {
                const uint32_t v = tile & 1 ? head_dt[1] : head_dt[0];
                float z = __uint_as_float(v);
                if (sizeof(T) == 2 && !a.dt_f32) {
                  const unsigned short u = static_cast<unsigned short>(v);
                  z = to_f32<T>(*reinterpret_cast<const T*>(&u));
                }
                step = step_from<T>(a, z, bias[0].x);
              } else {
                step = step_size<T>(a, t0 + vt, (c0 + vc + i) / a.width);
              }
              e = expf(step * hrate[i]);
            }
            (i & 1 ? dt[i / 2].y : dt[i / 2].x) = step;
            (i & 1 ? decay[i / 2].y : decay[i / 2].x) = e;
          }
        }
        float2* to = &sm.d[tile & 1][vt][vc];
        float2 dx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          dx[i] = __fmul2_rn(dt[i], make_float2(to_f32<T>(x.e[2 * i]), to_f32<T>(x.e[2 * i + 1])));
        if (here < 8) {
          const float none = CH ? 0.0f : 1.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i >= here) {
              (i & 1 ? decay[i / 2].y : decay[i / 2].x) = none;
              (i & 1 ? dx[i / 2].y : dx[i / 2].x) = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(to + 2 * i) = make_float4(decay[i].x, dx[i].x, decay[i].y, dx[i].y);
      }
      for (int e = me; e < 2 * TOK * NP / 8; e += kHelp) {
        const Eight<T> v = sm.bc_raw[tile & 1][e];
        float* to = &sm.bc[tile & 1][0][0][0] + e * 8;
#pragma unroll
        for (int k = 0; k < 8; k += 4)
          *reinterpret_cast<float4*>(to + k) =
              make_float4(to_f32<T>(v.e[k]), to_f32<T>(v.e[k + 1]), to_f32<T>(v.e[k + 2]), to_f32<T>(v.e[k + 3]));
      }
    };
    auto finish = [&](int tile) {
      const int t0 = po.first + tile * TOK, here = vt < po.end - t0 ? vn : 0;
      if (here <= 0) return;
      const Eight<T> x = sm.x[tile & 3][me];
      Eight<T> z, y;
      if (a.z != nullptr) z = sm.z[tile & 3][me];
      const float* from = sm.y[tile & 1][vt][vc];
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (Tile::kParts == 4) {
          const float4 v = *reinterpret_cast<const float4*>(from + 4 * (i ^ (me & 7)));
          q[i] = (v.x + v.y) + (v.z + v.w);
        } else {
          const float2 v = *reinterpret_cast<const float2*>(from + 2 * (i ^ (me & 7)));
          q[i] = v.x + v.y;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = fmaf(i & 1 ? skip[i / 2].y : skip[i / 2].x, to_f32<T>(x.e[i]), q[i]);
      if (a.z != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] *= silu<T>(to_f32<T>(z.e[i]));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y.e[i] = from_f32<T>(q[i]);
      T* to = out + static_cast<long long>(t0 + vt) * a.ldo + vc;
      if (WIDE) {
        *reinterpret_cast<Eight<T>*>(to) = y;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < here) to[i] = y.e[i];
      }
    };
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    convert(0);
    bring(2);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (i + 1 < tiles) convert(i + 1);
      if (i > 0) finish(i - 1);
      bring(i + 3);
      __syncthreads();
    }
    finish(tiles - 1);
    return;
  }

  // ---------------- core ----------------
  const int l = threadIdx.x & (LPC - 1), col = threadIdx.x / LPC;
  const bool old = a.state != nullptr && a.positions[po.first] != 0;
  const int ws = a.state != nullptr ? a.wslots[r] : -1;
  const bool keep = ws >= 0 && ws < a.num_slots;
  const long long pitch = static_cast<long long>(a.heads) * a.width * a.N;
  const long long at = static_cast<long long>(c0 + col) * a.N;
  float2 h[kHalf], rate[kHalf];
  constexpr int kVec = NPL < 4 ? NPL : 4;                    // neighbouring numbers of a lane
  auto number = [&](int i) { return (i / kVec * LPC + l) * kVec + i % kVec; };
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int n = number(i);
    const bool in = n < a.N && col < cols;
    const float v = old && in ? a.state[slot * pitch + at + n] : 0.0f;
    const float q = CH && in ? -expf(a.a_log[at + n]) * kLog2e : 0.0f;
    (i & 1 ? h[i / 2].y : h[i / 2].x) = v;
    (i & 1 ? rate[i / 2].y : rate[i / 2].x) = q;
  }
  constexpr int kE = CH ? kHalf : 1;
  struct Ahead {                                             // decays and inputs of four tokens
    float2 e[4][kE], u[4][kHalf];
  };
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
    const float2* sd = &sm.d[tile & 1][0][col];
    const float* sb = &sm.bc[tile & 1][0][0][kVec * l];
    const float* sc = &sm.bc[tile & 1][1][0][kVec * l];
    // numbers 2 k and 2 k + 1 of this lane and, where it has four neighbours, the next two
    auto load = [&](const float* from, int t, int k, float2& p, float2& q) {
      from += t * NP + k / 2 * LPC * 4;
      if constexpr (kVec == 4) {
        const float4 v = *reinterpret_cast<const float4*>(from);
        p = make_float2(v.x, v.y);
        q = make_float2(v.z, v.w);
      } else {
        p = *reinterpret_cast<const float2*>(from);
      }
    };
    auto token_ahead = [&](int t, float2 (&e)[kE], float2 (&u)[kHalf]) {
      const float2 dd = sd[t * kCols];
      const float2 dx = make_float2(dd.y, dd.y), step = make_float2(dd.x, dd.x);
      if (!CH) e[0] = step;
#pragma unroll
      for (int k = 0; k < kHalf; k += 2) {
        float2 b[2];
        load(sb, t, k, b[0], b[1]);
#pragma unroll
        for (int j = k; j < k + kVec / 2; ++j) {
          u[j] = __fmul2_rn(dx, b[j - k]);
          if (CH) {
            const float2 p = __fmul2_rn(step, rate[j]);
            e[CH ? j : 0] = make_float2(exp2_fast(p.x), exp2_fast(p.y));
          }
        }
      }
    };
    auto token = [&](int t, const float2 (&e)[kE], const float2 (&u)[kHalf]) {
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kHalf; k += 2) {
        float2 c[2];
        load(sc, t, k, c[0], c[1]);
#pragma unroll
        for (int j = k; j < k + kVec / 2; ++j) {
          h[j] = __ffma2_rn(e[CH ? j : 0], h[j], u[j]);
          s = j == 0 ? __fmul2_rn(h[j], c[0]) : __ffma2_rn(h[j], c[j - k], s);
        }
      }
      return s.x + s.y;
    };
    auto leave = [&](int i, float (&part)[4]) {              // (i is a multiple of 4: no part of a key)
      float(*sy)[kCols][Tile::kParts] = sm.y[tile & 1] + i;
      if constexpr (LPC <= 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) sy[u][col ^ Tile::key(u, col)][l] = part[u];
      } else {
        // round by round, the lanes of a column part by one bit of l, and the tokens with them
#pragma unroll
        for (int o = LPC / 2; o >= 4; o >>= 1) {
          const bool up = l & o;
#pragma unroll
          for (int u = 0; u < 16 / LPC * (o / 4); ++u) {
            const int half = 16 / LPC * (o / 4);
            const float mine = up ? part[u + half] : part[u], theirs = up ? part[u] : part[u + half];
            part[u] = mine + __shfl_xor_sync(0xffffffffu, theirs, o);
          }
        }
        // 16 lanes: token l / 4; 8 lanes: tokens 2 (l / 4) and the next
#pragma unroll
        for (int u = 0; u < 16 / LPC; ++u) {
          const int t = l / 4 * (16 / LPC) + u;
          sy[t][col ^ Tile::key(t, col)][l & 3] = part[u];
        }
      }
    };
    auto make = [&](int i, Ahead& to) {
#pragma unroll
      for (int u = 0; u < 4; ++u) token_ahead(i + u, to.e[u], to.u[u]);
    };
    auto walk = [&](int i, const Ahead& from) {
      float part[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) part[u] = token(i + u, from.e[u], from.u[u]);
      leave(i, part);
    };
    if constexpr (NPL <= 4) {
      Ahead even, odd;
#pragma unroll 1
      for (int i = 0; i < TOK; i += 8) {
        make(i, even);
        make(i + 4, odd);
        walk(i, even);
        walk(i + 4, odd);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < TOK; i += 4) {
        float part[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float2 e[kE], v[kHalf];
          token_ahead(i + u, e, v);
          part[u] = token(i + u, e, v);
        }
        leave(i, part);
      }
    }
    __syncthreads();
  }
  if (keep && col < cols) {
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (number(i) < a.N) a.state[ws * pitch + at + number(i)] = i & 1 ? h[i / 2].y : h[i / 2].x;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
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

template <typename T, int LPR, int NC>
int launch_heads_step(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCtaCols = 4 * (NC > 1 ? 4 : 8) * (32 / LPR);
  const dim3 grid((a.heads * a.width + kCtaCols - 1) / kCtaCols, a.nd);
  return a.wide ? launch_overlapped(heads_step_kernel<T, LPR, NC, true>, grid, dim3(128), 0, s, a)
                : launch_overlapped(heads_step_kernel<T, LPR, NC, false>, grid, dim3(128), 0, s, a);
}
template <typename T, int LPR, int RQ>
int launch_channels_step(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCtaCols = 4 * (32 / LPR);
  const dim3 grid((a.heads * a.width + kCtaCols - 1) / kCtaCols, (a.nd + RQ - 1) / RQ);
  return a.wide ? launch_overlapped(channels_step_kernel<T, LPR, RQ, true>, grid, dim3(128), 0, s, a)
                : launch_overlapped(channels_step_kernel<T, LPR, RQ, false>, grid, dim3(128), 0, s, a);
}
// Requests that share a warp: four where that leaves eight warps to an SM (64 requests of 8192 channels of 16: two and
// four 24 us, eight, whose registers leave 12 warps an SM, 34).
template <typename T, int LPR>
int launch_channels_step(const ScanArgs& a, cudaStream_t s) {
  const long long warps = (static_cast<long long>(a.heads) * a.width + 32 / LPR - 1) / (32 / LPR);
  auto enough = [&](int rq) { return warps * ((a.nd + rq - 1) / rq) >= 8ll * sm_count(); };
  if (enough(4)) return launch_channels_step<T, LPR, 4>(a, s);
  return launch_channels_step<T, LPR, 1>(a, s);
}

template <typename T, bool CH>
int launch_step(const ScanArgs& a, cudaStream_t s) {
  const int cols = a.heads * a.width;
  if (a.N % 4 == 0 && reinterpret_cast<uintptr_t>(a.a_log) % (CH ? 16 : 4) == 0) {
    if constexpr (CH) {
      if (a.N <= 8) return launch_channels_step<T, 2>(a, s);
      if (a.N <= 16) return launch_channels_step<T, 4>(a, s);
      if (a.N <= 32) return launch_channels_step<T, 8>(a, s);
      if (a.N <= 64) return launch_channels_step<T, 16>(a, s);
      if (a.N <= 128) return launch_channels_step<T, 32>(a, s);
    } else {
      if (a.N > 64 && a.N <= 128 && a.width % 8 == 0) return launch_heads_step<T, 32, 1>(a, s);
      if (a.N > 128 && a.width % 4 == 0) return launch_heads_step<T, 32, 2>(a, s);
      if (a.N > 32 && a.N <= 64 && a.width % 16 == 0) return launch_heads_step<T, 16, 1>(a, s);
      if (a.N > 16 && a.N <= 32 && a.width % 32 == 0) return launch_heads_step<T, 8, 1>(a, s);
      if (a.N <= 16 && a.width % 64 == 0) return launch_heads_step<T, 4, 1>(a, s);
    }
  }
#define STEP(LPR, NC, V)                                                              \
  launch_overlapped(selective_step_kernel<T, CH, LPR, NC, V>,                         \
                    dim3((cols + 4 * (NC > 1 ? 4 : 8) * (32 / LPR) - 1) /             \
                             (4 * (NC > 1 ? 4 : 8) * (32 / LPR)), a.nd),              \
                    dim3(128), 0, s, a)
  if (a.N % 4 == 0) {
    if constexpr (!CH) {
      if (a.N <= 16) return STEP(4, 1, 4);
      if (a.N <= 32) return STEP(8, 1, 4);
      if (a.N <= 64) return STEP(16, 1, 4);
      if (a.N <= 128) return STEP(32, 1, 4);
    }
    return STEP(32, 2, 4);
  }
  if (a.N <= 32) return STEP(32, 1, 1);
  if (a.N <= 128) return STEP(32, 4, 1);
  return STEP(32, 8, 1);
#undef STEP
}

template <typename T, bool CH, int LPC, int NPL, bool WIDE>
int launch_scan(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCols = kCore<LPC> / LPC, kSmem = sizeof(ScanTile<T, CH, LPC, NPL>);
  const auto kernel = selective_scan_kernel<T, CH, LPC, NPL, WIDE>;
  if (kSmem > 48 * 1024) {
    const int rc = launch_code(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (rc != 0) return rc;
  }
  const int per = a.heads / a.groups * a.width;
  return launch_overlapped(kernel, dim3(a.np, a.groups, (per + kCols - 1) / kCols), dim3(kCore<LPC> + kHelp), kSmem,
                           s, a);
}
template <typename T, bool CH, bool WIDE>
int launch_scan(const ScanArgs& a, cudaStream_t s) {
  if (a.N <= 8) return launch_scan<T, CH, 4, 2, WIDE>(a, s);
  if (a.N <= 16) return launch_scan<T, CH, 4, 4, WIDE>(a, s);
  if (a.N <= 32) return launch_scan<T, CH, 8, 4, WIDE>(a, s);
  if (a.N <= 64) return launch_scan<T, CH, 16, 4, WIDE>(a, s);
  if (a.N <= 128) return launch_scan<T, CH, 16, 8, WIDE>(a, s);
  return launch_scan<T, CH, 16, 16, WIDE>(a, s);
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
  // eight elements at a time: rows on 16-byte boundaries, and no group or row of B and C ends inside one
  const bool wide = a.wide && a.N % 8 == 0 && a.heads / a.groups * a.width % 8 == 0 &&
                    (!CH || (a.lddt % 8 == 0 && reinterpret_cast<uintptr_t>(a.dt) % 16 == 0));
  return wide ? launch_scan<T, CH, true>(a, s) : launch_scan<T, CH, false>(a, s);
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
struct ScanCall {
  const void *x, *dt, *b, *c, *z;
  void* out;
  const float *a_log, *d, *dt_bias;
  float* state;
  const long long* positions;
  const int *slots, *wslots, *cu_q;
  long long ldx, lddt, ldb, ldc, ldz, ldo;
  float dt_min, dt_max;
  int dt_f32, per_channel, softplus, num_slots, T, heads, width, N, groups, nd, np, wide, dtype;
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

// Selective scan of a step's rows; per_channel: a_log [heads * width, N] and a step size per column, else
// a_log [heads] and a step size per head.  state may be null (every portion starts from zeros).  wide: rows of x, b,
// c, z and out start on 16-byte boundaries.
B200_API int b200_selective_scan(const void* call, void* stream) {
  using namespace b200::selective;
  const ScanCall& k = *static_cast<const ScanCall*>(call);
  if (k.T <= 0 || k.heads <= 0 || k.width <= 0 || k.nd + k.np <= 0) return 0;
  if (k.N < 1 || k.N > 256) return -8;
  ScanArgs a;
  a.x = k.x; a.dt = k.dt; a.b = k.b; a.c = k.c; a.z = k.z; a.out = k.out; a.a_log = k.a_log; a.d = k.d;
  a.dt_bias = k.dt_bias; a.state = k.state; a.positions = k.positions; a.slots = k.slots; a.wslots = k.wslots;
  a.cu_q = k.cu_q; a.ldx = k.ldx; a.lddt = k.lddt; a.ldb = k.ldb; a.ldc = k.ldc; a.ldz = k.ldz; a.ldo = k.ldo;
  a.dt_min = k.dt_min; a.dt_max = k.dt_max; a.T = k.T; a.heads = k.heads; a.width = k.width; a.N = k.N;
  a.groups = k.groups; a.num_slots = k.num_slots; a.nd = k.nd; a.np = k.np; a.dt_f32 = k.dt_f32;
  a.softplus = k.softplus; a.wide = k.wide;
  a.limits = k.dt_max < INFINITY || k.dt_min > 0.0f || !k.softplus;    // (a softplus is not below 0)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool channels = k.per_channel != 0;
  switch (k.dtype) {
    case 0: return channels ? scan_any<__nv_bfloat16, true>(a, s) : scan_any<__nv_bfloat16, false>(a, s);
    case 1: return channels ? scan_any<__half, true>(a, s) : scan_any<__half, false>(a, s);
    case 2: return channels ? scan_any<float, true>(a, s) : scan_any<float, false>(a, s);
  }
  return -8;
}

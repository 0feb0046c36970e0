// Selective scan of single tokens (sm_100a), one per request: see selective.cu for the formulas and the state's layout.
#include <algorithm>

#include "selective.cuh"

namespace b200 {
namespace selective {

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
  // row i's number, where each lane has those of the rows whose sums it is left with
  template <typename V>
  __device__ __forceinline__ static V of(const V (&own)[kLeft], int i) {
    if constexpr (kParted == 1) return own[i];
    else return __shfl_sync(0xffffffffu, own[i % kLeft], i / kLeft * (LPR / kParted), LPR);
  }
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

// Single tokens and short portions, rates per head, where a warp's columns belong to one head (width a multiple of
// their number) and N is one of 4: a row of N numbers is spread over LPR lanes, NC times four each, and stays in
// registers while the warp walks the request's tokens, the next one under way.  The state's bytes bound it: a warp
// has 4 KB of it under way at once, and what a head's columns share is worked out once per warp.  96 requests of
// 80 heads of 64 x 128: 77 us, 6.5 TB/s, the copy's rate (row by row, 70 per cent of the issue slots went into
// what they share: 113; with the next token's registers, which MANY is for, 91).
template <typename T, int LPR, int NC, bool MANY, bool WIDE>
__global__ void __launch_bounds__(128) heads_step_kernel(const ScanArgs a) {
  constexpr int kRows = NC > 1 ? 4 : 8, kGroups = 32 / LPR, kWarpCols = kRows * kGroups, kX = (kWarpCols + 31) / 32;
  grid_release_small();
  grid_wait();
  const int r = blockIdx.y, lane = threadIdx.x & 31, l = lane & (LPR - 1), grp = lane / LPR;
  const int cols = a.heads * a.width;
  const int c0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kWarpCols;
  if (c0 >= cols) return;
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  const int ws = a.state != nullptr ? a.wslots[r] : -1;
  Portion po = {r, r + 1};
  if constexpr (MANY) {
    po = portion_of(r, a.nd, a.cu_q, a.T);
    if (po.first >= po.end) return;
  }
  const bool old = a.state != nullptr && a.positions[po.first] != 0;
  T* out = static_cast<T*>(a.out) + c0;
  if (a.state != nullptr && (slot < 0 || slot >= a.num_slots)) {
    for (int t = po.first; t < po.end; ++t)
      for (int i = lane; i < kWarpCols; i += 32) out[t * a.ldo + i] = from_f32<T>(0.0f);
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
  const T* bsrc = static_cast<const T*>(a.b) + g * a.N + l * 4;
  const T* csrc = static_cast<const T*>(a.c) + g * a.N + l * 4;
  const float rate = expf(a.a_log[hd]), skip = a.d != nullptr ? a.d[hd] : 0.0f;
  const float bias = a.dt_bias != nullptr ? a.dt_bias[hd] : 0.0f;
  struct Token {
    float x[kX];                                 // x of the warp's columns: column j in lane j % 32
    float4 b[NC], c[NC];
    float dt;
  };
  auto bring = [&](long long t, Token& to) {
#pragma unroll
    for (int j = 0; j < kX; ++j) {
      const int c = min(j * 32 + lane, kWarpCols - 1);
      to.x[j] = to_f32<T>(static_cast<const T*>(a.x)[t * a.ldx + c0 + c]);
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      to.b[k] = load_four<T, WIDE>(bsrc + t * a.ldb + LPR * k * 4, (l + LPR * k) * 4 < a.N);
      to.c[k] = load_four<T, WIDE>(csrc + t * a.ldc + LPR * k * 4, (l + LPR * k) * 4 < a.N);
    }
    to.dt = a.dt_f32 ? static_cast<const float*>(a.dt)[t * a.lddt + hd]
                     : to_f32<T>(static_cast<const T*>(a.dt)[t * a.lddt + hd]);
  };
  Token now, next;
  bring(po.first, now);
  int t = po.first;
  do {
    const bool more = MANY && t + 1 < po.end;
    if (more) bring(t + 1, next);
    const float dt = step_from<T>(a, now.dt, bias);
    const float decay = decay_of(-dt * rate);
    float s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float dx = dt * __shfl_sync(0xffffffffu, now.x[i * kGroups / 32], (i * kGroups + grp) & 31);
      s[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < NC; ++k)
        s[i] += update(h[i][k], make_float2(decay, decay), make_float2(decay, decay), make_float2(dx, dx), now.b[k],
                       now.c[k]);
    }
    if (!more && ws >= 0 && ws < a.num_slots) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if ((l + LPR * k) * 4 < a.N)
            *reinterpret_cast<float4*>(a.state + ws * pitch + at + i * kGroups * a.N + LPR * k * 4) = h[i][k];
    }
    const RowSums<kRows, LPR> sums(s, l);
#pragma unroll
    for (int i = 0; i < sums.kLeft; ++i) {
      const int j = (sums.first + i) * kGroups + grp;    // column of the warp
      float xv = 0.0f;
#pragma unroll
      for (int m = 0; m < kX; ++m) {
        const float v = __shfl_sync(0xffffffffu, now.x[m], j & 31);
        if (j / 32 == m) xv = v;
      }
      float y = fmaf(skip, xv, sums.v[i]);
      if (a.z != nullptr) y *= silu<T>(to_f32<T>(static_cast<const T*>(a.z)[t * a.ldz + c0 + j]));
      if (sums.keeps(l)) out[t * a.ldo + j] = from_f32<T>(y);
    }
    if constexpr (MANY) now = next;
  } while (MANY && ++t < po.end);
}

// One token per request, rates per channel, N a multiple of 4 up to 128: a warp holds 32 / LPR columns of RQ
// requests, so that rates and skips are fetched and worked out once for them; what is one number per column and request
// (slots, step sizes, x, gates) is one lane's, the one that RowSums leaves that request's sum in, and goes round from there.
// 64 requests of 8192 channels of 16, bf16: 16.5 us, 4.3 TB/s (23.4 with all of them in every lane: issue slots);
// the chain slot - state - sum - row of a warp that lives for a few microseconds bounds it.
template <typename T, int LPR, int RQ, bool WIDE>
__global__ void __launch_bounds__(128) channels_step_kernel(const ScanArgs a) {
  constexpr int kGroups = 32 / LPR;
  using Sums = RowSums<RQ, LPR>;
  constexpr int kOwn = Sums::kLeft, kApart = LPR / Sums::kParted;    // requests of a lane, lanes of the same ones
  grid_release_small();
  grid_wait();
  const int lane = threadIdx.x & 31, l = lane & (LPR - 1), grp = lane / LPR;
  const int cols = a.heads * a.width;
  const int c0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kGroups;
  if (c0 >= cols) return;
  const bool in = c0 + grp < cols && l * 4 < a.N, mine = c0 + grp < cols;
  const int col = min(c0 + grp, cols - 1), n = l * 4;
  const int g = col / (cols / a.groups);
  const int r0 = blockIdx.y * RQ, own = r0 + l / kApart * kOwn;
  constexpr int kPadding = -2, kNone = -1;
  const long long pitch = static_cast<long long>(cols) * a.N, at = static_cast<long long>(col) * a.N + n;
  float4 h[RQ], b[RQ], c[RQ];
  int from[kOwn], to[kOwn];                      // slots
#pragma unroll
  for (int m = 0; m < kOwn; ++m) {
    const int r = min(own + m, a.nd - 1);        // (behind the last request: its row again, and nothing is kept)
    from[m] = to[m] = kNone;
    if (a.state != nullptr) {
      const int slot = a.slots[r], ws = a.wslots[r];
      const long long pos = a.positions[r];
      const bool there = slot >= 0 && slot < a.num_slots;
      from[m] = !there ? kPadding : pos != 0 ? slot : kNone;
      if (there && ws >= 0 && ws < a.num_slots && own + m < a.nd) to[m] = ws;
    }
  }
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const int slot = Sums::of(from, i);
    h[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (slot >= 0 && in) h[i] = *reinterpret_cast<const float4*>(a.state + slot * pitch + at);
  }
  float x[kOwn], dt[kOwn], z[kOwn], dx[kOwn];
#pragma unroll
  for (int m = 0; m < kOwn; ++m) {
    const int r = min(own + m, a.nd - 1);
    x[m] = to_f32<T>(static_cast<const T*>(a.x)[r * a.ldx + col]);
    dt[m] = a.dt_f32 ? static_cast<const float*>(a.dt)[r * a.lddt + col]
                     : to_f32<T>(static_cast<const T*>(a.dt)[r * a.lddt + col]);
    z[m] = a.z != nullptr ? to_f32<T>(static_cast<const T*>(a.z)[r * a.ldz + col]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const int r = min(r0 + i, a.nd - 1);
    b[i] = load_four<T, WIDE>(static_cast<const T*>(a.b) + r * a.ldb + g * a.N + n, in);
    c[i] = load_four<T, WIDE>(static_cast<const T*>(a.c) + r * a.ldc + g * a.N + n, in);
  }
  float4 rate = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (in) rate = *reinterpret_cast<const float4*>(a.a_log + at);
  rate = make_float4(-expf(rate.x) * kLog2e, -expf(rate.y) * kLog2e, -expf(rate.z) * kLog2e, -expf(rate.w) * kLog2e);
  const float bias = a.dt_bias != nullptr ? a.dt_bias[col] : 0.0f, skip = a.d != nullptr ? a.d[col] : 0.0f;
#pragma unroll
  for (int m = 0; m < kOwn; ++m) {
    dt[m] = step_from<T>(a, dt[m], bias);
    dx[m] = dt[m] * x[m];
  }
  float s[RQ];
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const float step = Sums::of(dt, i), add = Sums::of(dx, i);
    const int ws = Sums::of(to, i);
    const float2 e0 = decays(make_float2(step, step), make_float2(rate.x, rate.y));
    const float2 e1 = decays(make_float2(step, step), make_float2(rate.z, rate.w));
    s[i] = update(h[i], e0, e1, make_float2(add, add), b[i], c[i]);
    s[i] = in ? s[i] : 0.0f;
    if (in && ws >= 0) *reinterpret_cast<float4*>(a.state + ws * pitch + at) = h[i];
  }
  const Sums sums(s, l);
#pragma unroll
  for (int m = 0; m < kOwn; ++m) {
    const int r = own + m;
    if (!mine || !sums.keeps(l) || r >= a.nd) continue;
    float y = fmaf(skip, x[m], sums.v[m]);
    if (a.z != nullptr) y *= silu<T>(z[m]);
    static_cast<T*>(a.out)[r * a.ldo + col] = from_f32<T>(from[m] == kPadding ? 0.0f : y);
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
      if (!CH) decay = decay_of(-dt * expf(a.a_log[hd]));
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
        if (CH) e = n < a.N ? decay_of(-dt * expf(a.a_log[static_cast<long long>(col) * a.N + n])) : 0.0f;
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

template <typename T, int LPR, int NC, bool MANY>
int launch_heads_step(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCtaCols = 4 * (NC > 1 ? 4 : 8) * (32 / LPR);
  const dim3 grid((a.heads * a.width + kCtaCols - 1) / kCtaCols, MANY ? a.nd + a.np : a.nd);
  return a.wide ? launch_overlapped(heads_step_kernel<T, LPR, NC, MANY, true>, grid, dim3(128), 0, s, a)
                : launch_overlapped(heads_step_kernel<T, LPR, NC, MANY, false>, grid, dim3(128), 0, s, a);
}
template <typename T, int LPR, int RQ>
int launch_channels_step(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCtaCols = 4 * (32 / LPR);
  const dim3 grid((a.heads * a.width + kCtaCols - 1) / kCtaCols, (a.nd + RQ - 1) / RQ);
  return a.wide ? launch_overlapped(channels_step_kernel<T, LPR, RQ, true>, grid, dim3(128), 0, s, a)
                : launch_overlapped(channels_step_kernel<T, LPR, RQ, false>, grid, dim3(128), 0, s, a);
}
// Requests that share a warp: four where that leaves eight warps to an SM (calls of 64 requests of 8192 channels of 16 in
// a row, us: two 19.5, four 19, eight, whose registers leave few warps an SM, 22).
template <typename T, int LPR>
int launch_channels_step(const ScanArgs& a, cudaStream_t s) {
  const long long warps = (static_cast<long long>(a.heads) * a.width + 32 / LPR - 1) / (32 / LPR);
  auto enough = [&](int rq) { return warps * ((a.nd + rq - 1) / rq) >= 8ll * sm_count(); };
  if (enough(4)) return launch_channels_step<T, LPR, 4>(a, s);
  return launch_channels_step<T, LPR, 1>(a, s);
}

constexpr int kNotTaken = -1000;
// The single tokens of a step (MANY: all of its requests) by heads_step_kernel, where the sizes allow it.
template <typename T, bool MANY>
int launch_heads(const ScanArgs& a, cudaStream_t s) {
  if (a.N % 4 != 0) return kNotTaken;
  if (a.N > 64 && a.N <= 128 && a.width % 8 == 0) return launch_heads_step<T, 32, 1, MANY>(a, s);
  if (a.N > 128 && a.width % 4 == 0) return launch_heads_step<T, 32, 2, MANY>(a, s);
  if (a.N > 32 && a.N <= 64 && a.width % 16 == 0) return launch_heads_step<T, 16, 1, MANY>(a, s);
  if (a.N > 16 && a.N <= 32 && a.width % 32 == 0) return launch_heads_step<T, 8, 1, MANY>(a, s);
  if (a.N <= 16 && a.width % 64 == 0) return launch_heads_step<T, 4, 1, MANY>(a, s);
  return kNotTaken;
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
      const int rc = launch_heads<T, false>(a, s);
      if (rc != kNotTaken) return rc;
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

// Steps whose portions are short, whose state's way in and out is most of the work.  Only the mean length is known here,
// and one portion may hold nearly all of the rows.
//
// Where the others would go by tiles: us by this kernel and by tiles, 96 requests of 80 heads of 64 x 128: 74 and 392 for
// 1 token each, 147 and 392 for 4, 247 and 393 for 8, 449 and 395 for 16.  A token of a portion takes 0.55 us, so the rows of a step are kept
// to what the tiles would take twice as long for were they all one portion's (8 us for a CTA per SM).
//
// Where they would go token after token (selective.cu), us by this kernel and by that one, 16 heads of 64 x 128 in 16 bits:
// even portions, 48 of 8 tokens 25 and 90, 12 of 32 31 and 38, 1 of 16 11 and 5; one long portion beside others of one
// token, 300 and nine 184 and 57, 30 and one 20 and 7.  Both are estimated, for an even step and for one whose rows are
// all one portion's, from times of 2 to 80 heads of 32 to 128 columns with 16 to 256 numbers: this kernel 0.55 us a token (32
// bits: 0.45) and no faster than the states' arithmetic, the other one its start per CTA and SM and then its tokens.
// An even step (drafted tokens that are verified) counts double.  What the rule costs at the most: 12 portions of 4
// tokens, 16 heads of 64 x 16, 8 us where a walk takes 4; 300 and nine, 32 heads of 64 x 64, 184 where the other takes 66.
bool worth_a_walk(const ScanArgs& a, int dtype, long long rows) {
  const int per = a.heads / a.groups * a.width, cta_cols = a.N <= 32 ? 32 : 16;
  const double ctas = static_cast<double>(a.groups) * ((per + cta_cols - 1) / cta_cols), sms = sm_count();
  const double rounds = ctas * a.np / sms;
  const double start = std::max(rounds, 1.0) * (a.N <= 16 ? 2.1 : a.N <= 128 ? 4.2 : 6.5);
  const double alone = a.N <= 16 ? 0.05 : 0.12;
  const double shared = ctas * (a.N <= 64 ? 0.0008 : a.N <= 128 ? 0.0011 : 0.0018);
  const double arithmetic = 5.2e-7 * rows * a.heads * a.width * a.N;
  auto walk = [&](double n) { return std::max(2 + (dtype == 2 ? 0.45 : 0.55) * n, arithmetic); };
  auto other = [&](double n) { return start + std::max(alone, shared) * n; };
  const double mean = static_cast<double>(rows) / a.np;
  return walk(mean) * walk(rows) <= 2 * other(mean) * other(rows);
}

bool launch_short_portions(const ScanArgs& a, int dtype, cudaStream_t s, int* rc) {
  const long long rows = a.T - a.nd;
  if (a.np == 0) return false;
  if (dtype == 0 && heads_by_tiles(a)) {
    const long long ctas = static_cast<long long>(a.np) * a.heads * (a.width / 64), sms = sm_count();
    if (rows > 12ll * a.np || rows > 28 * ((ctas + sms - 1) / sms)) return false;
  } else if (rows > 32ll * a.np || rows > 512 || !worth_a_walk(a, dtype, rows)) {
    return false;
  }
  *rc = dtype == 0   ? launch_heads<__nv_bfloat16, true>(a, s)
        : dtype == 1 ? launch_heads<__half, true>(a, s)
                     : launch_heads<float, true>(a, s);
  return *rc != kNotTaken;
}

int launch_single_tokens(const ScanArgs& a, bool per_channel, int dtype, cudaStream_t s) {
  switch (dtype) {
    case 0: return per_channel ? launch_step<__nv_bfloat16, true>(a, s) : launch_step<__nv_bfloat16, false>(a, s);
    case 1: return per_channel ? launch_step<__half, true>(a, s) : launch_step<__half, false>(a, s);
    case 2: return per_channel ? launch_step<float, true>(a, s) : launch_step<float, false>(a, s);
  }
  return -8;
}

}  // namespace selective
}  // namespace b200

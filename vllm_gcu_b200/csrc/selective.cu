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

// Portions of prompts, token after token.  A CTA holds the columns of one request that kThreads / LPC lane groups
// make: a column's numbers of state lie in the registers of LPC lanes, NPL each, and a token costs a number one
// decay (rates per channel: a power of two, which the special function unit does 16 of per clock and SM: it bounds
// them), two multiply-adds and a product.  Inputs pass through shared memory kTok tokens at a time: while a
// tile is worked on, the next one is on its way to registers, eight neighbouring elements per thread, and a
// thread finishes the elements that it brought (skip, gate, store).  Each token's sum over the lanes of a column
// is left for kSum tokens, then lanes trade partial sums so that each ends up with the sums of its own
// tokens: 3 exchanges for 4 tokens of 4 lanes instead of 8.
template <int LPC>
constexpr int kScanThreads = LPC == 16 ? 256 : 128;

template <typename T>
struct __align__(16) Eight {
  T e[8];
};
// eight neighbours of a row; `n` of them are there
template <typename T, bool WIDE>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int n) {
  Eight<T> v;
  if (WIDE) {
    if (n > 0) v = *reinterpret_cast<const Eight<T>*>(p);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) v.e[i] = from_f32<T>(0.0f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.e[i] = i < n ? p[i] : from_f32<T>(0.0f);
  }
  return v;
}

template <typename T, bool CH, int LPC, int NPL, bool WIDE>
__global__ void __launch_bounds__(kScanThreads<LPC>) selective_scan_kernel(const ScanArgs a) {
  constexpr int kThreads = kScanThreads<LPC>, NP = LPC * NPL, kCols = kThreads / LPC, kTok = LPC == 2 || NP > 128 ? 16 : 32;
  constexpr int kSum = LPC < 8 ? LPC : 8;
  constexpr int kVecs = kTok * kCols / 8;                    // threads that bring and finish elements
  constexpr int kParts = (2 * kTok * NP / 8 + kThreads - 1) / kThreads;
  static_assert(kVecs <= kThreads, "one vector of eight per thread");
  __shared__ __align__(16) float sbc[2][kTok][NP];           // B, C
  __shared__ __align__(16) float2 sd[kTok][kCols];           // step size (rates per head: decay), step size times x
  __shared__ __align__(16) float sy[kTok][kCols + 4];
  grid_release_small();
  grid_wait();
  const int r = a.nd + blockIdx.x, g = blockIdx.y, per = a.heads / a.groups * a.width;
  const int l = threadIdx.x & (LPC - 1), col = threadIdx.x / LPC;
  const int p0 = blockIdx.z * kCols, cols = min(kCols, per - p0);
  const int c0 = g * per + p0;                               // first column of the CTA
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
  float2 h[NPL / 2], rate[NPL / 2];
  auto number = [&](int i) { return (i / 4 * LPC + l) * 4 + i % 4; };
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int n = number(i);
    const bool in = n < a.N && col < cols;
    const float v = old && in ? a.state[slot * pitch + at + n] : 0.0f;
    const float q = CH && in ? -expf(a.a_log[at + n]) * kLog2e : 0.0f;
    (i & 1 ? h[i / 2].y : h[i / 2].x) = v;
    (i & 1 ? rate[i / 2].y : rate[i / 2].x) = q;
  }

  // this thread's eight elements of a tile: token vt, columns vc and on; what belongs to a column stays
  const int vt = threadIdx.x / (kCols / 8), vc = threadIdx.x % (kCols / 8) * 8;
  const int vn = threadIdx.x < kVecs ? max(0, min(8, cols - vc)) : 0;
  const bool one_head = !CH && a.width % 8 == 0;             // eight columns share a step size
  float bias[8], skip[8], hrate[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int which = CH ? c0 + vc + i : (c0 + vc + i) / a.width;
    const bool in = i < vn;
    bias[i] = in && a.dt_bias != nullptr ? a.dt_bias[which] : 0.0f;
    skip[i] = in && a.d != nullptr ? a.d[which] : 0.0f;
    hrate[i] = !CH && in ? -expf(a.a_log[which]) : 0.0f;
  }
  Eight<T> x, z, dth, bc[kParts];
  Eight<float> dtf;
  auto bring = [&](int t0) {
    const int n = po.end - t0;
    const int here = vt < n ? vn : 0;
    const long long t = t0 + vt;
    const int which = CH ? c0 + vc : (c0 + vc) / a.width;
    x = load_eight<T, WIDE>(static_cast<const T*>(a.x) + t * a.ldx + c0 + vc, here);
    if (a.z != nullptr) z = load_eight<T, WIDE>(static_cast<const T*>(a.z) + t * a.ldz + c0 + vc, here);
    if (CH) {
      if (a.dt_f32) dtf = load_eight<float, false>(static_cast<const float*>(a.dt) + t * a.lddt + which, here);
      else dth = load_eight<T, WIDE>(static_cast<const T*>(a.dt) + t * a.lddt + which, here);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i > 0 && one_head) break;
        if (i >= here) break;
        const long long k = t * a.lddt + (c0 + vc + i) / a.width;
        if (a.dt_f32) dtf.e[i] = static_cast<const float*>(a.dt)[k];
        else dth.e[i] = static_cast<const T*>(a.dt)[k];
      }
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int e = threadIdx.x + i * kThreads;
      const int m = e / (kTok * NP / 8), k = e / (NP / 8) % kTok, c = e % (NP / 8) * 8;
      const T* row = m == 0 ? static_cast<const T*>(a.b) + (t0 + k) * a.ldb : static_cast<const T*>(a.c) + (t0 + k) * a.ldc;
      bc[i] = load_eight<T, WIDE>(row + g * a.N + c, m < 2 && k < n ? max(0, min(8, a.N - c)) : 0);
    }
  };
  bring(po.first);

  for (int t0 = po.first; t0 < po.end; t0 += kTok) {
    // registers -> shared memory; a token behind the portion has a step of 0, which leaves a state as it is
    const bool here = vt < po.end - t0 && threadIdx.x < kVecs;
    if (threadIdx.x < kVecs) {
      float dt = 0.0f, decay = 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (here && i < vn && (i == 0 || !one_head)) {
          dt = step_from<T>(a, a.dt_f32 ? dtf.e[i] : to_f32<T>(dth.e[i]), bias[i]);
          if (!CH) decay = expf(dt * hrate[i]);
        }
        const bool in = here && i < vn;
        sd[vt][vc + i] = in ? make_float2(CH ? dt : decay, dt * to_f32<T>(x.e[i])) : make_float2(CH ? 0.0f : 1.0f, 0.0f);
      }
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int e = threadIdx.x + i * kThreads;
      if (e < 2 * kTok * NP / 8) {
        float* to = &sbc[0][0][0] + e * 8;
#pragma unroll
        for (int k = 0; k < 8; k += 4)
          *reinterpret_cast<float4*>(to + k) = make_float4(to_f32<T>(bc[i].e[k]), to_f32<T>(bc[i].e[k + 1]),
                                                           to_f32<T>(bc[i].e[k + 2]), to_f32<T>(bc[i].e[k + 3]));
      }
    }
    __syncthreads();
    const Eight<T> xs = x, zs = z;
    if (t0 + kTok < po.end) bring(t0 + kTok);
#pragma unroll 1
    for (int i = 0; i < kTok; i += kSum) {
      float part[kSum];
#pragma unroll
      for (int u = 0; u < kSum; ++u) {
        const float2 dd = sd[i + u][col];
        const float2 dx = make_float2(dd.y, dd.y);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < NPL / 4; ++k) {
          const float4 bq = *reinterpret_cast<const float4*>(&sbc[0][i + u][(k * LPC + l) * 4]);
          const float4 cq = *reinterpret_cast<const float4*>(&sbc[1][i + u][(k * LPC + l) * 4]);
          const float2 be[2] = {make_float2(bq.x, bq.y), make_float2(bq.z, bq.w)};
          const float2 ce[2] = {make_float2(cq.x, cq.y), make_float2(cq.z, cq.w)};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float2 e = make_float2(dd.x, dd.x);
            if (CH) {
              e = __fmul2_rn(e, rate[2 * k + j]);
              e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
            }
            h[2 * k + j] = __ffma2_rn(e, h[2 * k + j], __fmul2_rn(dx, be[j]));
            s = __ffma2_rn(h[2 * k + j], ce[j], s);
          }
        }
        part[u] = s.x + s.y;
      }
      // lane l of a column gets the sums of token i + l % kSum
#pragma unroll
      for (int o = kSum / 2; o > 0; o >>= 1) {
        const bool up = l & o;
#pragma unroll
        for (int u = 0; u < o; ++u) {
          const float mine = up ? part[u + o] : part[u], theirs = up ? part[u] : part[u + o];
          part[u] = mine + __shfl_xor_sync(0xffffffffu, theirs, o);
        }
      }
#pragma unroll
      for (int o = kSum; o < LPC; o <<= 1) part[0] += __shfl_xor_sync(0xffffffffu, part[0], o);
      if (l < kSum) sy[i + l][col] = part[0];
    }
    __syncthreads();
    if (here && vn > 0) {
      Eight<T> y;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f = fmaf(skip[i], to_f32<T>(xs.e[i]), sy[vt][vc + i]);
        if (a.z != nullptr) f *= silu<T>(to_f32<T>(zs.e[i]));
        y.e[i] = from_f32<T>(f);
      }
      T* to = out + static_cast<long long>(t0 + vt) * a.ldo + vc;
      if (WIDE) {
        *reinterpret_cast<Eight<T>*>(to) = y;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < vn) to[i] = y.e[i];
      }
    }
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

template <typename T, bool CH, bool WIDE>
int launch_scan(const ScanArgs& a, cudaStream_t s) {
  const int per = a.heads / a.groups * a.width;
#define SCAN(LPC, NPL)                                                                                     \
  launch_overlapped(selective_scan_kernel<T, CH, LPC, NPL, WIDE>,                                          \
                    dim3(a.np, a.groups, (per + kScanThreads<LPC> / LPC - 1) / (kScanThreads<LPC> / LPC)), \
                    dim3(kScanThreads<LPC>), 0, s, a)
  if (a.N <= 8) return SCAN(2, 4);
  if (a.N <= 16) return SCAN(4, 4);
  if (a.N <= 32) return SCAN(8, 4);
  if (a.N <= 64) return SCAN(16, 4);
  if (a.N <= 128) return SCAN(16, 8);
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
  // eight elements at a time: rows on 16-byte boundaries, and no group or row of B and C ends inside one
  const bool wide = a.wide && a.N % 8 == 0 && a.heads / a.groups * a.width % 8 == 0 &&
                    (!CH || a.dt_f32 || (a.lddt % 8 == 0 && reinterpret_cast<uintptr_t>(a.dt) % 16 == 0));
  return wide ? launch_scan<T, CH, true>(a, s) : launch_scan<T, CH, false>(a, s);
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

// Selective scan of prompts with rates per head, by products of tiles (sm_100a, tcgen05).
//
// A chunk of 128 tokens of a head, with L_i the sum of dt A (base 2) up to and with token i and H the state in
// front of it, is
//   y_i  = sum_{j <= i} 2^(L_i - L_j) dt_j (C_i . B_j) x_j  +  2^(L_i) C_i . H
//   H'   = 2^(L_end) H + sum_j 2^(L_end - L_j) dt_j x_j B_j
// Four products per chunk, operands bf16, sums fp32 in tensor memory:
//   G  [i x j]      = C B^T                            both tiles as they are in memory
//   Y2 [i x (p, 2)] = C (H_hi | H_lo)                  the state in two parts of bf16
//   S  [n x (p, 3)] = B^T (W_hi | W_mid | W_lo)        W_j = 2^(L_end - L_j) dt_j x_j in three parts: all 24 bits,
//                                                      since the state is kept in 32
//   Y1 [i x p]      = (M_hi + M_lo) X                  M_ij = G_ij 2^(L_i - L_j) dt_j in place of G, two parts
// H lives in registers (lane n, 16 columns p per warp) and goes on as fp32.  Two parts leave 2^-17 of a
// factor, which does not show beside the rows' own rounding to bf16; one part alone would make a result's error
// 1.4 times as large.
//
// Decays (none above 1: step sizes are not below 0): a difference L_i - L_j is taken of sums in two floats or, in the
// 32 x 32 blocks on the diagonal, of 32-bit numbers whose rounding the two sides' factors make good, so that a
// strong decay in front does not cost those behind it their bits.  Outside the diagonal 2^(L_i - L_j) is a product of two
// factors below 1, with L at the row block's start between them: 32 exponentials a row instead of 128.
//
// A CTA walks the chunks of 64 columns of one head of one request; 16 warps do the arithmetic between the
// products, one warp moves tiles (TMA), one issues the products, two compute step sizes and decays, a chunk
// each, ahead of the rest.  W of a chunk is made a chunk ahead, M while the tensor cores do Y2 and S, state and result
// while they do Y1 and the next chunk's G.  Lanes 96 and up have four blocks of M that are not zero where lanes below 32
// have one, so their warps make less of W.
//
// 4096 tokens of 128 heads, 8 groups, N = 128, in one prompt: 114 us in a captured graph, up to 125 among other calls, 32
// chunks of 3.35 us and 5 us of start (156 MB: 24 us at the copy's rate; the products' 78 GFLOP, splits included: 47 us); as
// long with 8 heads, one chain of chunks per 64 columns.  The arithmetic between the products bounds it: 60 per cent of the issue slots and half of the integer pipe, most of that for splits into parts of bf16;
// tensor pipe 36 per cent.  On the way: 8 warps 213 us; decays from sums in 64 bits, by one warp, 131; with
// more of it unrolled the instruction caches miss (no wait, no loop over products or groups is copied: 137 so, 119).
#include "selective.cuh"

namespace b200 {
namespace selective {
namespace tiles {

constexpr unsigned int kKernelId = 75;
constexpr int kRows = 128, kP = 64;                    // tokens of a chunk, columns of a CTA
constexpr int kSub = kRows * 128;                      // bytes of 128 rows of 64 bf16
constexpr int kOffC = 0, kOffB = 2 * kSub, kOffX = 4 * kSub, kOffW = 6 * kSub, kOffH = 9 * kSub;
constexpr int kOffScal = 11 * kSub;

// Per chunk, by token: written by one warp, read by all.
struct Scalars {
  float row[kRows];       // 2^(L_i - L at the start of i's block of 32)
  float diag[kRows];      // that exponent, rounded
  float row_low[kRows];   // 2^(what the rounding left off)
  float col_low[kRows];   // dt_j / 2^(the same)
  float off[192];         // dt_j 2^(L at the start of block I - L_j): I = 1 (32), 2 (64), 3 (96 of them)
  float w[kRows];         // dt_j 2^(L_end - L_j)
  float e[kRows];         // 2^(L_i)
  float end[4];           // 2^(L_end)
  int bad[kP];            // by column: the first token whose x is infinite or no number (kRows: none)
  int any_bad[4];
};
constexpr int kOffBars = kOffScal + 4 * static_cast<int>(sizeof(Scalars));
constexpr int kSmem = kOffBars + 256 + 1024;
static_assert(kSmem <= 232448, "shared memory of a CTA");

enum Bar {
  kCFull, kBFull, kCFree, kBFree, kXFull0, kXFull1, kYReady0, kYReady1, kSFree0, kSFree1, kSFree2, kSFree3, kGDone,
  kMReady, kWReady, kSDone, kHReady, kYDone, kYFree, kBars
};
// columns of tensor memory
constexpr uint32_t kColG = 0, kColY2 = 128, kColY1 = 256, kColS = 320, kTmem = 512;
constexpr uint32_t kIdescAMajorMN = 1u << 15;
constexpr int kWarps = 16;                             // of arithmetic: four per 32 lanes of tensor memory
constexpr int kScal = 2;                               // of step sizes and decays, a chunk each in turn
constexpr int kThreads = (kWarps + 2 + kScal) * 32;

// fp32 pairs: two operations per instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 bits2(uint32_t x, uint32_t y) {
  return make_float2(__uint_as_float(x), __uint_as_float(y));
}
__device__ __forceinline__ uint32_t pack(float2 v) { return pack_bf16x2(v.x, v.y); }
// a pair in bf16, and what that left off (times -1 twice: a subtraction of pairs is a multiply-add)
__device__ __forceinline__ uint32_t split(float2& v) {
  const uint32_t hi = pack(v);
  v = fma2(unpack_bf16x2(hi), both(-1.0f), v);
  return hi;
}
// 16 bytes of column chunk u (of 8) of row r in a tile of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t tile_at(int r, int u) { return r * 128 + ((u ^ (r & 7)) << 4); }

// A sum in two floats: 48 bits, by Knuth's exact sum of two numbers.  (In 64 bits it took a chunk's warp twice as
// long, for the conversions of 28 differences a lane.)
struct Two {
  float hi, lo;
};
__device__ __forceinline__ Two add(Two a, Two b) {
  const float s = a.hi + b.hi, v = s - a.hi;
  const float e = (a.hi - (s - v)) + (b.hi - v) + (a.lo + b.lo);
  const float hi = s + e;
  return {hi, e - (hi - s)};
}
__device__ __forceinline__ float less(Two a, Two b) { return (a.hi - b.hi) + (a.lo - b.lo); }
__device__ __forceinline__ Two shfl(Two v, int from) {
  return {__shfl_sync(0xffffffffu, v.hi, from), __shfl_sync(0xffffffffu, v.lo, from)};
}

// What a lane needs of the step sizes of tokens 4 lane .. + 3 of a chunk, as it lies in memory: nothing waits for it here.
__device__ __forceinline__ void load_steps(const ScanArgs& a, int hd, long long t0, int n, uint32_t (&z)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long long at = (t0 + min(4 * lane + k, n - 1)) * a.lddt + hd;    // (behind the last token: it again)
    if (a.dt_f32) z[k] = static_cast<const uint32_t*>(a.dt)[at];
    else z[k] = static_cast<const unsigned short*>(a.dt)[at];
  }
}
// Step sizes and decays of n tokens, four per lane.  rate: -exp(a_log) log2(e).
__device__ __forceinline__ void chunk_scalars(const ScanArgs& a, int n, float bias, Two rate, const uint32_t (&z)[4],
                                              Scalars* s) {
  const int lane = threadIdx.x & 31;
  float dt[4];
  Two L[4], run = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    dt[k] = step_from<__nv_bfloat16>(a, __uint_as_float(a.dt_f32 ? z[k] : z[k] << 16), bias);
    Two la = {dt[k] * rate.hi, 0.0f};
    la.lo = fmaf(dt[k], rate.hi, -la.hi) + dt[k] * rate.lo;
    if (la.hi < -160.0f) la = {-160.0f, 0.0f};          // 2^-160 is 0 in fp32; sums stay exact to 2^-33
    if (4 * lane + k >= n) {
      dt[k] = 0.0f;
      la = {0.0f, 0.0f};
    }
    run = add(run, la);
    L[k] = run;
  }
  Two before = run;                                     // over the lanes: inclusive, then what lies in front of one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Two v = {__shfl_up_sync(0xffffffffu, before.hi, o), __shfl_up_sync(0xffffffffu, before.lo, o)};
    if (lane >= o) before = add(v, before);
  }
  before = {__shfl_up_sync(0xffffffffu, before.hi, 1), __shfl_up_sync(0xffffffffu, before.lo, 1)};
  if (lane == 0) before = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 4; ++k) L[k] = add(before, L[k]);
  const Two ref1 = shfl(L[3], 7), ref2 = shfl(L[3], 15), ref3 = shfl(L[3], 23), end = shfl(L[3], 31);
  const int block = lane >> 3;
  const Two none = {0.0f, 0.0f}, ref = block == 0 ? none : block == 1 ? ref1 : block == 2 ? ref2 : ref3;
  const Two minus = {-ref.hi, -ref.lo};
  float row[4], diag[4], rl[4], cl[4], w[4], e[4], o1[4], o2[4], o3[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const Two l = add(L[k], minus);
    diag[k] = l.hi;
    row[k] = exp2_fast(l.hi);
    rl[k] = exp2_fast(l.lo);
    cl[k] = dt[k] * exp2_fast(-l.lo);
    w[k] = dt[k] * exp2_fast(less(end, L[k]));
    e[k] = exp2_fast(L[k].hi);
    o1[k] = dt[k] * exp2_fast(less(ref1, L[k]));        // (lanes behind the reference: not kept)
    o2[k] = dt[k] * exp2_fast(less(ref2, L[k]));
    o3[k] = dt[k] * exp2_fast(less(ref3, L[k]));
  }
  auto put = [&](float* to, const float (&v)[4]) {
    *reinterpret_cast<float4*>(to + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
  };
  put(s->row, row);
  put(s->diag, diag);
  put(s->row_low, rl);
  put(s->col_low, cl);
  put(s->w, w);
  put(s->e, e);
  if (lane < 8) put(s->off, o1);
  if (lane < 16) put(s->off + 32, o2);
  if (lane < 24) put(s->off + 96, o3);
  if (lane == 0) s->end[0] = exp2_fast(end.hi);
  s->bad[lane] = s->bad[lane + 32] = kRows;
  if (lane == 0) s->any_bad[0] = 0;
}

// Numbers of x that are infinite or none, eight at `x` (columns col and on of a token): in the product M X they would
// show in the tokens in front, whose weights are 0.  Zeros take their place there (W keeps them), and the
// results of their column from their token on are no numbers.
__device__ __noinline__ void hide_bad(Scalars* s, unsigned char* x, int token, int col) {
  unsigned short* v = reinterpret_cast<unsigned short*>(x);
  for (int i = 0; i < 8; ++i) {
    if ((v[i] & 0x7f80) != 0x7f80) continue;
    v[i] = 0;
    atomicMin(&s->bad[col + i], token);
    s->any_bad[0] = 1;
  }
}

__device__ __noinline__ uint4 show_bad(const Scalars* s, uint4 y, int token, int col) {
  uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (token >= s->bad[col + i]) v[i / 2] |= 0x7fffu << (i % 2 * 16);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A wait of a warp that computes.  No lane leaves: when the budget runs out the warp goes on over numbers without
// meaning to the end of its chunk; the flag ends it there, and the warps that load and multiply at once.  (All lanes ask:
// by the first lane alone, and the others behind a barrier of the warp, a chunk took 400 cycles more.)
__device__ __noinline__ bool wait_for(uint64_t* bar, uint32_t parity, unsigned int* st, unsigned int detail,
                                      volatile uint32_t* abort_flag) {
  return mbar_wait(bar, parity, st, kKernelId, detail, abort_flag);
}
__device__ __forceinline__ void pass_warp(uint64_t* bar, uint32_t parity, unsigned int* st, unsigned int detail,
                                          volatile uint32_t* abort_flag) {
  if (!mbar_test(bar, parity)) wait_for(bar, parity, st, detail, abort_flag);
  __syncwarp();
}
__device__ __forceinline__ bool given_up(volatile uint32_t* abort_flag) {
  return __any_sync(0xffffffffu, *abort_flag != 0u) != 0;
}

template <int N>
__global__ void __launch_bounds__(kThreads, 1)
heads_kernel(const ScanArgs a, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
             const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ CUtensorMap tm_y, unsigned int* status) {
  constexpr int kU = N / 64;                            // sub-tiles of B and C
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  Scalars* scal = reinterpret_cast<Scalars*>(smem + kOffScal);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kBars);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBars; ++i) {
      const bool by_warps = i == kYReady0 || i == kYReady1 || (i >= kSFree0 && i <= kSFree3) || i == kMReady ||
                            i == kWReady || i == kHReady || i == kYFree;
      mbar_init(&bar[i], by_warps ? kWarps : i == kXFull0 || i == kXFull1 ? 2 : 1);   // x, and its scalars
    }
    *abort_flag = 0u;
    mbar_fence_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_b);
    tma_prefetch_desc(&tm_c);
  }
  if (warp == kWarps + 1) {
    tmem_alloc(tmem_slot, kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_release();
  grid_wait();

  const int r = a.nd + blockIdx.y, p_blocks = a.width / kP;
  const int hd = blockIdx.x / p_blocks, p0 = blockIdx.x % p_blocks * kP;
  const int col0 = hd * a.width + p0, group = hd / (a.heads / a.groups);
  const Portion po = portion_of(r, a.nd, a.cu_q, a.T);
  const int chunks = max(0, po.end - po.first + kRows - 1) / kRows;
  const int slot = a.state != nullptr ? a.slots[r] : 0;
  const bool padding = a.state != nullptr && (slot < 0 || slot >= a.num_slots);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + col0;

  if (padding) {
    for (int e = threadIdx.x; e < (po.end - po.first) * 8; e += kThreads)
      *reinterpret_cast<uint4*>(out + (po.first + (e >> 3)) * a.ldo + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
  } else if (warp < kWarps) {
    // ---------------- arithmetic between the products ----------------
    const int q = warp & 3, part = warp >> 2;           // lanes of tensor memory; 16 of 64 columns
    const int i = q * 32 + lane;                        // lane of tensor memory: token, or number of the state
    const uint32_t mine = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const bool old = a.state != nullptr && chunks > 0 && a.positions[po.first] != 0;
    const int ws = a.state != nullptr ? a.wslots[r] : -1;
    const long long head_at = (static_cast<long long>(a.heads) * a.width * N);
    const long long at = (static_cast<long long>(col0) + part * 16) * N + i;
    float2 h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      h[k] = both(0.0f);
      const float* from = a.state + slot * head_at + at + 2 * k * N;
      if (old && i < N) h[k] = make_float2(from[0], from[N]);
    }
    auto put_state = [&]() {
      if (i < N) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float2 f = h[u * 4 + k];
            hi[k] = split(f);
            lo[k] = pack(f);
          }
          unsigned char* to = smem + kOffH + tile_at(i, part * 2 + u);
          *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(to + kSub) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kHReady]);
    };
    const float skip = a.d != nullptr ? a.d[hd] : 0.0f;
    // 4 rows of W at a time, in groups of 12, 8, 8 and 4 rows for the warps of the four quarters
    const int w_rows = q == 0 ? 12 : q == 3 ? 4 : 8;
    const int w_first = part * 32 + (q == 0 ? 0 : q == 1 ? 12 : q == 2 ? 20 : 28);
    // W of chunk c = x times its weight, in three parts
    auto make_w = [&](int c) {
      const int n = min(kRows, po.end - po.first - c * kRows);
      Scalars* s = scal + (c & 3);
      unsigned char* x = smem + kOffX + (c & 1) * kSub;
      pass_warp(&bar[kXFull0 + (c & 1)], (c >> 1) & 1, status, 0x101u, abort_flag);
      // rows of other requests: zeros, they may hold anything
      if (n < kRows) pass_warp(&bar[kBFull], c & 1, status, 0x102u, abort_flag);
#pragma unroll 1
      for (int k = 0; k < w_rows; k += 4) {
        const int row = w_first + k + (lane >> 3);
        const uint32_t to = tile_at(row, lane & 7);
        uint4 v = *reinterpret_cast<const uint4*>(x + to);
        if (row >= n) {
          v = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(x + to) = v;
#pragma unroll
          for (int b = 0; b < kU; ++b) *reinterpret_cast<uint4*>(smem + kOffB + b * kSub + to) = v;
        }
        const float2 w = both(s->w[row]);
        const uint32_t in[4] = {v.x, v.y, v.z, v.w};
        uint32_t p[3][4];
        float2 none = both(0.0f);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float2 f = unpack_bf16x2(in[m]);
          none = fma2(f, both(0.0f), none);
          f = mul2(w, f);
          p[0][m] = split(f);
          p[1][m] = split(f);
          p[2][m] = pack(f);
        }
#pragma unroll
        for (int m = 0; m < 3; ++m)
          *reinterpret_cast<uint4*>(smem + kOffW + m * kSub + to) = make_uint4(p[m][0], p[m][1], p[m][2], p[m][3]);
        if (none.x + none.y != 0.0f) hide_bad(s, x + to, row, (lane & 7) * 8);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kWReady]);
    };

    // (turn -1: the state in front and W of the first chunk; one copy of the code for both: the kernel's instructions
    // are more than their caches hold, and what does not fit costs every warp)
#pragma unroll 1
    for (int c = -1; c < chunks; ++c) {
      if (given_up(abort_flag)) break;
      const int stage = c & 1, four = c & 3, n = min(kRows, po.end - po.first - c * kRows);
      const Scalars* s = scal + four;
      unsigned char* x = smem + kOffX + stage * kSub;
      if (c >= 0) {
      // M in place of G, every fourth group of 16 columns
      pass_warp(&bar[kGDone], c & 1, status, 0x103u, abort_flag);
      tc_fence_after();
      {
        const float row = s->row[i], di = s->diag[i], low = s->row_low[i];
        const float* off = s->off + (q == 2 ? 32 : q == 3 ? 96 : 0);
#pragma unroll 1
        for (int j = part; j < 8; j += 4) {
          uint32_t m[16];
          if (j > 2 * q + 1) {
#pragma unroll
            for (int k = 0; k < 16; ++k) m[k] = 0u;
          } else {
            uint32_t g[16];
            tmem_ld_32x16(mine + kColG + 16 * j, g);
            float2 f[8];                                // what G is multiplied by
            if (j < 2 * q) {
#pragma unroll
              for (int k = 0; k < 8; k += 2) {
                const float4 o = *reinterpret_cast<const float4*>(off + 16 * j + 2 * k);
                f[k] = mul2(make_float2(o.x, o.y), both(row));
                f[k + 1] = mul2(make_float2(o.z, o.w), both(row));
              }
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 8; ++k) f[k] = mul2(f[k], bits2(g[2 * k], g[2 * k + 1]));
            } else {
#pragma unroll
              for (int k = 0; k < 8; k += 2) {
                const float4 d = *reinterpret_cast<const float4*>(s->diag + 16 * j + 2 * k);
                const float4 o = *reinterpret_cast<const float4*>(s->col_low + 16 * j + 2 * k);
                f[k] = mul2(make_float2(exp2_fast(di - d.x), exp2_fast(di - d.y)), mul2(make_float2(o.x, o.y), both(low)));
                f[k + 1] = mul2(make_float2(exp2_fast(di - d.z), exp2_fast(di - d.w)),
                                mul2(make_float2(o.z, o.w), both(low)));
              }
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                f[k] = mul2(f[k], bits2(g[2 * k], g[2 * k + 1]));
                if (16 * j + 2 * k > i) f[k].x = 0.0f;
                if (16 * j + 2 * k + 1 > i) f[k].y = 0.0f;
              }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              m[k] = split(f[k]);
              m[8 + k] = pack(f[k]);
            }
          }
          tmem_st_32x16(mine + kColG + 16 * j, m);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kMReady]);

      // the state behind the chunk
      pass_warp(&bar[kSDone], c & 1, status, 0x104u, abort_flag);
      tc_fence_after();
      {
        const float keep = s->end[0];
        uint32_t v[3][16];
#pragma unroll
        for (int m = 0; m < 3; ++m) tmem_ld_32x16(mine + kColS + m * 64 + part * 16, v[m]);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          h[k] = fma2(both(keep), h[k],
                      add2(bits2(v[0][2 * k], v[0][2 * k + 1]),
                           add2(bits2(v[1][2 * k], v[1][2 * k + 1]), bits2(v[2][2 * k], v[2][2 * k + 1]))));
      }
      tc_fence_before();
      }
      put_state();
      if (c + 1 < chunks) make_w(c + 1);                 // (the products with W of this chunk are through)
      if (c < 0) continue;

      // the result's rows
      pass_warp(&bar[kYDone], c & 1, status, 0x105u, abort_flag);
      tc_fence_after();
      {
        uint32_t y1[16], y2[16], y3[16];
        tmem_ld_32x16(mine + kColY1 + part * 16, y1);
        tmem_ld_32x16(mine + kColY2 + part * 16, y2);
        tmem_ld_32x16(mine + kColY2 + 64 + part * 16, y3);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kYFree]);
        const float2 e = both(s->e[i]);
        const bool bad = s->any_bad[0] != 0;
        const long long t = po.first + c * kRows + i;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          unsigned char* at_x = x + tile_at(i, part * 2 + u);
          const uint4 xv = *reinterpret_cast<const uint4*>(at_x);
          const uint32_t xi[4] = {xv.x, xv.y, xv.z, xv.w};
          float2 f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int k2 = u * 8 + 2 * k;
            f[k] = fma2(e, add2(bits2(y2[k2], y2[k2 + 1]), bits2(y3[k2], y3[k2 + 1])),
                        fma2(both(skip), unpack_bf16x2(xi[k]), bits2(y1[k2], y1[k2 + 1])));
          }
          if (a.z != nullptr && i < n) {
            float z[8];
            vec8_load(static_cast<const __nv_bfloat16*>(a.z) + t * a.ldz + col0 + part * 16 + u * 8, z);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              f[k] = mul2(f[k], make_float2(silu<__nv_bfloat16>(z[2 * k]), silu<__nv_bfloat16>(z[2 * k + 1])));
          }
          uint4 y = make_uint4(pack(f[0]), pack(f[1]), pack(f[2]), pack(f[3]));
          if (bad) y = show_bad(s, y, i, part * 16 + u * 8);
          // a whole chunk leaves as a tile, in place of its x; the last rows of a portion one by one
          if (n == kRows) *reinterpret_cast<uint4*>(at_x) = y;
          else if (i < n) *reinterpret_cast<uint4*>(out + t * a.ldo + part * 16 + u * 8) = y;
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane < 2) mbar_arrive(&bar[lane == 0 ? kYReady0 + stage : kSFree0 + four]);
    }
    if (!given_up(abort_flag) && chunks > 0 && ws >= 0 && ws < a.num_slots && i < N) {
#pragma unroll
      for (int k = 0; k < 16; ++k) a.state[ws * head_at + at + k * N] = k & 1 ? h[k / 2].y : h[k / 2].x;
    }
  } else if (warp == kWarps) {
    // ---------------- tiles ----------------
    if (elect_one()) {
      int issued = 0;
      // the result of chunk c, which lies in place of its x, to memory
      auto send = [&](int c) {
        if (!wait_for(&bar[kYReady0 + (c & 1)], (c >> 1) & 1, status, 0x200u, abort_flag)) return false;
        if (po.end - po.first - c * kRows >= kRows) {
          tma_store_2d(&tm_y, smem + kOffX + (c & 1) * kSub, col0, po.first + c * kRows);
          tma_store_commit();
        }
        return true;
      };
      bool ok = true;
      for (int c = 0; c < chunks; ++c) {
        const int y = po.first + c * kRows, stage = c & 1;
        if (c >= 2) {
          ok = send(c - 2);
          if (!ok) break;
          tma_store_wait_read<0>();
        }
        mbar_expect_tx(&bar[kXFull0 + stage], kSub);
        tma_load_2d(smem + kOffX + stage * kSub, &tm_x, &bar[kXFull0 + stage], col0, y);
        issued = 4 * c + 1;
        ok = c < 1 || wait_for(&bar[kCFree], (c - 1) & 1, status, 0x201u, abort_flag);
        if (!ok) break;
        mbar_expect_tx(&bar[kCFull], kU * kSub);
        for (int u = 0; u < kU; ++u) tma_load_2d(smem + kOffC + u * kSub, &tm_c, &bar[kCFull], group * N + u * 64, y);
        issued = 4 * c + 2;
        ok = c < 1 || wait_for(&bar[kBFree], (c - 1) & 1, status, 0x202u, abort_flag);
        if (!ok) break;
        mbar_expect_tx(&bar[kBFull], kU * kSub);
        for (int u = 0; u < kU; ++u) tma_load_2d(smem + kOffB + u * kSub, &tm_b, &bar[kBFull], group * N + u * 64, y);
        issued = 4 * c + 3;
        // the next chunk's tiles of B and C to L2: their buffers are free only when this chunk's products are through;
        // x of the chunk behind it
        if (c + 2 < chunks) tma_prefetch_2d(&tm_x, col0, y + 2 * kRows);
        if (c + 1 < chunks)
          for (int u = 0; u < kU; ++u) {
            tma_prefetch_2d(&tm_c, group * N + u * 64, y + kRows);
            tma_prefetch_2d(&tm_b, group * N + u * 64, y + kRows);
          }
      }
      for (int c = max(0, chunks - 2); c < chunks && ok; ++c) ok = send(c);
      tma_store_wait<0>();
      // copies in flight end before the CTA does, also when a wait ran out
      if (*abort_flag != 0u && issued > 0) {
        const int c = issued >> 2, what = issued & 3;
        wait_for(&bar[kXFull0 + (c & 1)], (c >> 1) & 1, status, 0x210u, nullptr);
        if (c >= 1) wait_for(&bar[kXFull0 + ((c - 1) & 1)], ((c - 1) >> 1) & 1, status, 0x211u, nullptr);
        if (what >= 2 || c >= 1) wait_for(&bar[kCFull], (what >= 2 ? c : c - 1) & 1, status, 0x212u, nullptr);
        if (what >= 3 || c >= 1) wait_for(&bar[kBFull], (what >= 3 ? c : c - 1) & 1, status, 0x213u, nullptr);
      }
    }
  } else if (warp == kWarps + 1) {
    // ---------------- products ----------------
    if (elect_one()) {
      constexpr uint32_t kIdG = make_idesc(kRows, 128, 1, 1);
      constexpr uint32_t kIdY2 = make_idesc(kRows, 128, 1, 1) | kIdescBMajorMN;
      constexpr uint32_t kIdS = make_idesc(kRows, 192, 1, 1) | kIdescAMajorMN | kIdescBMajorMN;
      constexpr uint32_t kIdY1 = make_idesc(kRows, kP, 1, 1) | kIdescBMajorMN;
      constexpr uint32_t kStep = 2048 >> 4;              // 16 rows of a tile
      const uint32_t base = smem_u32(smem);
      const uint64_t c_k = make_desc_k_sw128(base + kOffC), b_k = make_desc_k_sw128(base + kOffB);
      // (64 numbers of state: lanes 64 and up of S come from memory that holds nothing, and nobody reads them)
      const uint64_t b_mn = make_desc_mn_sw128(base + kOffB, kSub);
      const uint64_t w_mn = make_desc_mn_sw128(base + kOffW, kSub), h_mn = make_desc_mn_sw128(base + kOffH, kSub);
      const uint64_t x_mn = make_desc_mn_sw128(base + kOffX, kSub);
      auto wait = [&](int b, int parity, uint32_t what) {
        const bool there = wait_for(&bar[b], parity, status, 0x300u + what, abort_flag);
        tc_fence_after();
        return there;
      };
      for (int c = 0; c < chunks; ++c) {
        const int ph = c & 1;
        if (!wait(kCFull, ph, 0) || !wait(kBFull, ph, 1)) break;
#pragma unroll 1
        for (int k = 0; k < N / 16; ++k) {
          const uint32_t step = (k >> 2) * (kSub >> 4) + (k & 3) * 2;
          umma_f16(tmem + kColG, c_k + step, b_k + step, kIdG, k > 0);
        }
        umma_commit(&bar[kGDone]);
        if (!wait(kHReady, ph, 2) || (c > 0 && !wait(kYFree, ph ^ 1, 3))) break;
#pragma unroll 1
        for (int k = 0; k < N / 16; ++k)
          umma_f16(tmem + kColY2, c_k + (k >> 2) * (kSub >> 4) + (k & 3) * 2, h_mn + k * kStep, kIdY2, k > 0);
        umma_commit(&bar[kCFree]);
        if (!wait(kWReady, ph, 4)) break;
#pragma unroll 1
        for (int k = 0; k < 8; ++k) umma_f16(tmem + kColS, b_mn + k * kStep, w_mn + k * kStep, kIdS, k > 0);
        umma_commit(&bar[kBFree]);
        umma_commit(&bar[kSDone]);                       // (and Y2: the state may be replaced)
        if (!wait(kMReady, ph, 5)) break;
        const uint64_t x = x_mn + (c & 1) * (kSub >> 4);
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
          umma_f16_ts(tmem + kColY1, tmem + kColG + 16 * k, x + k * kStep, kIdY1, k > 0);
          umma_f16_ts(tmem + kColY1, tmem + kColG + 16 * k + 8, x + k * kStep, kIdY1, 1);
        }
        umma_commit(&bar[kYDone]);
      }
    }
  } else {
    // ---------------- step sizes and decays ----------------
    auto rows = [&](int c) { return min(kRows, po.end - po.first - c * kRows); };
    uint32_t z[4], next[4];
    const int first = warp - kWarps - 2;
    if (first < chunks) load_steps(a, hd, po.first + first * kRows, rows(first), z);
    const float bias = a.dt_bias != nullptr ? a.dt_bias[hd] : 0.0f;
    const float per = -expf(a.a_log[hd]);
    const Two rate = {per * kLog2e, fmaf(per, kLog2e, -(per * kLog2e)) + per * 1.925963033e-8f};
    for (int c = first; c < chunks; c += kScal) {
      if (c + kScal < chunks) load_steps(a, hd, po.first + (c + kScal) * kRows, rows(c + kScal), next);
      if (c >= 4) pass_warp(&bar[kSFree0 + (c & 3)], ((c >> 2) & 1) ^ 1, status, 0x400u, abort_flag);
      if (given_up(abort_flag)) break;
      chunk_scalars(a, rows(c), bias, rate, z, scal + (c & 3));
      __syncwarp();
      // (the barrier's turn before, two chunks ago, is over)
      if (c >= 2) pass_warp(&bar[kXFull0 + (c & 1)], ((c >> 1) & 1) ^ 1, status, 0x401u, abort_flag);
      if (lane == 0) mbar_arrive(&bar[kXFull0 + (c & 1)]);
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] = next[k];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarps + 1) tmem_dealloc(tmem, kTmem);
}

template <int N>
int launch(const ScanArgs& a, cudaStream_t s) {
  CUtensorMap x, b, c, y;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t gn = static_cast<uint64_t>(a.groups) * N;
  const uint64_t cols = static_cast<uint64_t>(a.heads) * a.width;
  auto pitch = [&](long long ld, uint64_t width) { return a.T > 1 ? 2 * static_cast<uint64_t>(ld) : 2 * width; };
  int rc = encode_tmap_2d(&x, bf, 2, a.x, a.T, cols, pitch(a.ldx, cols), kRows, 64, sw);
  if (rc == 0) rc = encode_tmap_2d(&b, bf, 2, a.b, a.T, gn, pitch(a.ldb, gn), kRows, 64, sw);
  if (rc == 0) rc = encode_tmap_2d(&c, bf, 2, a.c, a.T, gn, pitch(a.ldc, gn), kRows, 64, sw);
  if (rc == 0) rc = encode_tmap_2d(&y, bf, 2, a.out, a.T, cols, pitch(a.ldo, cols), kRows, 64, sw);
  if (rc != 0) return rc;
  unsigned int* status = status_ptr();
  if (status == nullptr) return -9;
  static bool ready[64] = {};                            // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -9;
  if (dev >= 64 || !ready[dev]) {
    const int e = launch_code(cudaFuncSetAttribute(heads_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (e != 0) return e;
    if (dev < 64) ready[dev] = true;
  }
  return launch_overlapped(heads_kernel<N>, dim3(a.heads * (a.width / kP), a.np), dim3(kThreads), kSmem, s, a, x, b, c, y,
                           status);
}

}  // namespace tiles

bool heads_by_tiles(const ScanArgs& a) {
  // (rows that share elements, as those of an expanded tensor, have no tensor map)
  const long long cols = static_cast<long long>(a.heads) * a.width, gn = static_cast<long long>(a.groups) * a.N;
  const bool apart = a.T == 1 || (a.ldx >= cols && a.ldb >= gn && a.ldc >= gn);
  return a.wide && apart && a.width % tiles::kP == 0 && (a.N == 64 || a.N == 128) && a.dt_min >= 0.0f;
}
int launch_heads_by_tiles(const ScanArgs& a, cudaStream_t s) {
  return a.N == 128 ? tiles::launch<128>(a, s) : tiles::launch<64>(a, s);
}

}  // namespace selective
}  // namespace b200

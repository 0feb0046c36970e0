// Selective state space scan (sm_100a), over the rows of a step: nd single tokens, one per request
// (selective_step.cu), then the portions of np prompts (offsets behind row nd in cu_q):
//   h_t = exp(dt_t A) h_(t-1) + dt_t x_t B_t,   y_t = C_t . h_t + d x_t   (times SiLU(z_t))
//
// state [slot, columns, N] fp32 of a request, read in one slot and left in another (usually the same).  A portion that
// starts at position 0 starts from zeros whatever the slot holds, so slots need no clearing.  A request whose
// slot is outside the state (padding of a captured batch) gives rows of zeros and touches no state; one whose
// write slot is outside leaves its state nowhere.
//
// Columns: a head holds `width` columns of x, each with N numbers of state.  Rates per head (a_log
// [heads]): one step size and one decay per head and token.  Rates per channel (a_log [columns, N]): a
// step size per column, a decay per column and number; the heads are then the groups that share B
// and C.  Portions with rates per head go by products of tiles where they can (selective_heads.cu), the others
// token after token.
#include "selective.cuh"

namespace b200 {
namespace selective {

// Portions of prompts, token after token.  A CTA holds the columns of one request that kCore / LPC lane groups
// make: a column's numbers of state lie in the registers of LPC lanes, NPL each, and a token costs a number one
// decay (rates per channel: a power of two, of which the special function unit does 16 per clock and SM), two
// multiply-adds and a product.  Inputs pass through shared memory kTok tokens at a time.  While the core warps
// walk tile i, four warps copy tile i + 2 and turn tile i + 1 into step sizes and factors, eight neighbouring
// elements a thread, and four others finish tile i - 1 (skip, gate, store); one barrier per tile.  What is done
// per element is half of the instructions and the chain along the tokens leaves the scheduler idle: 2048 tokens of
// 8192 channels took 235 us with all warps doing both in turn and 145 with four warps for the elements. The sum
// over the lanes of a column is the helpers': four lanes leave a part of it each; where there are more, pairs of
// lanes trade the parts of two tokens first, so that each ends up with those of its own token.  With few numbers
// per lane, decays and inputs of eight tokens are made before their chain is walked. Shared memory's bandwidth
// bounds rates per channel: 11 turns of 128 bytes a warp and token, about 100 of 120 cycles a token on the SMs
// that hold two CTAs: 2048 tokens of 8192 channels in 132 us, 73 per cent of all SMs' turns.  (Two columns per
// lane group, whose B and C would be read once, leave one core warp a scheduler: 143 us.  B and C in 16 bits until
// a lane has them save 4 of the turns and cost 8 instructions: 139.)
template <int LPC>
constexpr int kCore = LPC >= 8 ? 256 : 128;
constexpr int kHelp = 128;                       // threads that bring elements, and threads that finish them
template <int LPC, int NPL>
constexpr int kTok = LPC * NPL >= 128 ? 16 : 32;

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
  // as they are in memory: rows for four tiles, the rest for two
  Eight<T> x[4][kVecs], z[4][kVecs], bc_raw[2][2 * kTokens * LPC * NPL / 8];
  Eight<float> dt[2][CH ? kVecs : 1];                        // (rows of 16 bits: the first half)
  // by tile parity
  float bc[2][2][kTokens][LPC * NPL];                        // B, C
  // Step size (rates per head: decay) and step size times x, two columns in a place: column c of token t lies in
  // place c / 2 ^ pair_key, so that helpers, who write four places in a row each, start in different banks.
  float4 d[2][kTokens][kCols / 2];
  static __device__ __forceinline__ int pair_key(int t, int c) { return (t * (kCols / 8) + c / 8) >> 1 & 3; }
  static constexpr int kParts = 4;
  // Parts of C . h.  A helper reads the parts of eight columns in a row, 128 bytes, and its neighbours those of the next
  // ones: column c of token t lies in place c ^ key, so that they start in different banks.
  float y[2][kTokens][kCols][kParts];
  static __device__ __forceinline__ int key(int t, int c) { return (t * (kCols / 8) + c / 8) & 7; }
};

template <typename T, bool CH, int LPC, int NPL, bool WIDE>
__global__ void __launch_bounds__(kCore<LPC> + 2 * kHelp) selective_scan_kernel(const ScanArgs a) {
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
    const bool front = threadIdx.x < kCore<LPC> + kHelp;     // copies and factors; else: finishes
    const int me = (threadIdx.x - kCore<LPC>) % kHelp;
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
    if (front) bring(0);
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
              e = decay_of(step * hrate[i]);
            }
            (i & 1 ? dt[i / 2].y : dt[i / 2].x) = step;
            (i & 1 ? decay[i / 2].y : decay[i / 2].x) = e;
          }
        }
        float4* to = &sm.d[tile & 1][vt][vc / 2];
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
          to[i ^ Tile::pair_key(vt, vc)] = make_float4(decay[i].x, dx[i].x, decay[i].y, dx[i].y);
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
      const float* from = sm.y[tile & 1][vt][0];
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(from + 4 * ((vc + i) ^ (me & 7)));
        q[i] = (v.x + v.y) + (v.z + v.w);
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
    if (front) {
      bring(1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      convert(0);
    }
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      if (front) {
        bring(i + 2);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (i + 1 < tiles) convert(i + 1);
      } else if (i > 0) {
        finish(i - 1);
      }
      __syncthreads();
    }
    if (!front) finish(tiles - 1);
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
    const float w = CH && in ? -expf(a.a_log[at + n]) * kLog2e : 0.0f;
    (i & 1 ? h[i / 2].y : h[i / 2].x) = v;
    (i & 1 ? rate[i / 2].y : rate[i / 2].x) = w;
  }
  constexpr int kE = CH ? kHalf : 1;
  struct Ahead {                                             // decays and inputs of a token
    float2 e[kE], u[kHalf];
  };
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
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
    auto token_ahead = [&](int i, int u, Ahead& to) {        // token i + u, i a multiple of 4: no part of a key
      const float4* place = &sm.d[tile & 1][i + u][col / 2 ^ Tile::pair_key(u, col)];
      const float2 dd = reinterpret_cast<const float2*>(place)[col & 1];
      const float2 dx = make_float2(dd.y, dd.y), step = make_float2(dd.x, dd.x);
      if (!CH) to.e[0] = step;
#pragma unroll
      for (int k = 0; k < kHalf; k += 2) {
        float2 b[2];
        load(sb, i + u, k, b[0], b[1]);
#pragma unroll
        for (int j = k; j < k + kVec / 2; ++j) {
          to.u[j] = __fmul2_rn(dx, b[j - k]);
          if (CH) to.e[CH ? j : 0] = decays(step, rate[j]);
        }
      }
    };
    auto token = [&](int t, const Ahead& from) {
      float2 s;
#pragma unroll
      for (int k = 0; k < kHalf; k += 2) {
        float2 c[2];
        load(sc, t, k, c[0], c[1]);
#pragma unroll
        for (int j = k; j < k + kVec / 2; ++j) {
          h[j] = __ffma2_rn(from.e[CH ? j : 0], h[j], from.u[j]);
          s = j == 0 ? __fmul2_rn(h[j], c[0]) : __ffma2_rn(h[j], c[j - k], s);
        }
      }
      return s.x + s.y;
    };
    auto leave = [&](int i, float (&part)[4]) {              // (i is a multiple of 4: no part of a key)
      float(*sy)[kCols][Tile::kParts] = sm.y[tile & 1] + i;
      if constexpr (LPC == 4) {
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
    constexpr int kAhead = NPL <= 4 ? 8 : 4;
#pragma unroll 1
    for (int i = 0; i < TOK; i += kAhead) {
      Ahead x[kAhead];
      if constexpr (NPL <= 4) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) token_ahead(i + u / 4 * 4, u % 4, x[u]);
      }
#pragma unroll
      for (int g4 = 0; g4 < kAhead; g4 += 4) {
        float part[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if constexpr (NPL > 4) token_ahead(i, u, x[u]);
          part[u] = token(i + g4 + u, x[g4 + u]);
        }
        leave(i + g4, part);
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

template <typename T, bool CH, int LPC, int NPL, bool WIDE>
int launch_scan(const ScanArgs& a, cudaStream_t s) {
  constexpr int kCols = ScanTile<T, CH, LPC, NPL>::kCols, kSmem = sizeof(ScanTile<T, CH, LPC, NPL>);
  const auto kernel = selective_scan_kernel<T, CH, LPC, NPL, WIDE>;
  if (kSmem > 48 * 1024) {
    const int rc = launch_code(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (rc != 0) return rc;
  }
  const int per = a.heads / a.groups * a.width;
  return launch_overlapped(kernel, dim3(a.np, a.groups, (per + kCols - 1) / kCols), dim3(kCore<LPC> + 2 * kHelp), kSmem,
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
  int rc = 0;
  if (!channels && launch_short_portions(a, k.dtype, s, &rc)) return rc;
  if (a.nd > 0) {
    rc = launch_single_tokens(a, channels, k.dtype, s);
    if (rc != 0) return rc;
  }
  if (a.np == 0) return 0;
  switch (k.dtype) {
    case 0: return channels ? scan_any<__nv_bfloat16, true>(a, s) : scan_any<__nv_bfloat16, false>(a, s);
    case 1: return channels ? scan_any<__half, true>(a, s) : scan_any<__half, false>(a, s);
    case 2: return channels ? scan_any<float, true>(a, s) : scan_any<float, false>(a, s);
  }
  return -8;
}

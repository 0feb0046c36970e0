// Attention of few query rows per request over a cache in 8 bits with scales, head dimension 128, on tcgen05 (included by
// attention_block_scaled.cu, whose Args, Place and Call it uses).
//
// The codes go to the tensor cores as they are, K and V tiles straight from TMA, and what they meet is brought to 8 bits
// without loss instead: a query and a probability are sums of 8-bit numbers ("parts") of falling weight, which are as
// many columns of the small operand.
//   S^T = K Q^T    M = 128 tokens (K-major rows of 128 bytes), N = 3 kR columns: part x query row
//   O^T = V^T P^T  M = 128 columns of the values (MN-major, as they lie), N = 3 or 4 kR columns, K = 128 tokens
// e4m3: parts of 4 bits each, every one 16 times the rest of the one before, 12 bits together (probabilities are rounded
// to fp16 before); int8: digits to the base 128 of a number of 21 bits, 28 for probabilities, whose small ones lose
// bits where numbers of one size for all do not; the products' sums are exact.  A lane of the softmax warps owns a token: block scales are
// factors of its scores and of its probabilities, and there is no conversion of codes at all, which is what bounds a kernel
// that feeds 16-bit matrix instructions from 8-bit codes (attention_block_scaled.cu, head dimensions 64 and 256: there a
// chunk of 16 tokens takes a warp 490 instructions, here 80 of them for four query rows).
//
// Warps: 0..3 queries and softmax (lane = token of a tile; at the end column of the output), 4 TMA, 5 tcgen05.mma and
// tensor memory.  Scores and probabilities are double-buffered: K Q^T of a tile runs while the one before is at its softmax.
// The running maximum is raised when a score exceeds it by 2 (log2), which all four warps vote on; then the sums in
// tensor memory are taken to registers, rescaled, and start anew (rare behind the first tiles, and the only form for sums
// of whole numbers).
#pragma once

namespace b200 {
namespace rows8 {

constexpr int kTcTile = 128;                 // tokens of a stage
constexpr int kTcThreads = 192;
constexpr int kTcStageBytes = 2 * kTcTile * 128;
constexpr float kRaise = 2.0f;               // log2, by which a score may exceed the running maximum
constexpr int kMostTiles = 512;              // int8: whose sums of whole numbers one accumulator takes, 2^16 * 127 * 128 < 2^31

template <bool kInt8, int kR>
struct Tc {
  static constexpr int kParts = kInt8 ? 4 : 3;                 // of a probability
  static constexpr int kN = (kParts * kR + 15) / 16 * 16;      // columns of scores, and of outputs
  static constexpr int kAlloc = 3 * kN <= 64 ? 64 : 3 * kN <= 128 ? 128 : 3 * kN <= 256 ? 256 : 512;
  static constexpr int kStages = kR == 32 ? 5 : 3;             // (one CTA an SM with 512 columns, else two)
  static constexpr int kOffQ = kStages * kTcStageBytes;
  static constexpr int kOffP = kOffQ + kN * 128;
  static constexpr int kOffBar = kOffP + 2 * kN * 128;
  static constexpr int kOffRow = kOffBar + 256;                // factor and position of every row
  static constexpr int kOffMax = kOffRow + 2 * kR * 4;         // of every warp and row
  static constexpr int kBytes = kOffMax + 5 * kR * 4 + 1024;
};

template <int kColumns>
__device__ __forceinline__ void tmem_ld_columns(uint32_t addr, uint32_t* r) {
  static_assert(kColumns == 16 || kColumns == 32, "loads of this kernel");
  if constexpr (kColumns == 16) tmem_ld_32x16(addr, *reinterpret_cast<uint32_t(*)[16]>(r));
  else tmem_ld_32x32(addr, *reinterpret_cast<uint32_t(*)[32]>(r));
}

// A pair of fp16 numbers as three pairs of e4m3 parts: x = p0 + p1 / 16 + p2 / 256, each pair in 16 bits.
__device__ __forceinline__ void parts_e4m3(uint32_t x, uint32_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(x));
    p[i] = c;
    if (i < 2) {
      uint32_t back;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(c));
      const __half2 rest = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&back)),
                                   __floats2half2_rn(16.0f, 16.0f));
      x = *reinterpret_cast<const uint32_t*>(&rest);
    }
  }
}

template <bool kInt8>
__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kInt8) umma_i8(d, a, b, idesc, accumulate);
  else umma_f8(d, a, b, idesc, accumulate);
}

// Numbers of a lane's columns, parts put together: [part * kR + row] -> [row].
template <bool kInt8, int kR, int kParts>
__device__ __forceinline__ void sum_parts(uint32_t tmem, float (&s)[kR]) {
  constexpr int kLoad = kR <= 16 ? 16 : 32;
  // weights of the parts: 128^-p (the last digit's is 1) or 16^-p
  auto weight = [](int p) {
    return kInt8 ? static_cast<float>(1 << 7 * (kParts - 1 - p)) : 1.0f / static_cast<float>(1 << 4 * p);
  };
  const float last = weight(kParts - 1);
  if constexpr (kR <= 8) {
    constexpr int kN = Tc<kInt8, kR>::kN;
    uint32_t v[kN];
#pragma unroll
    for (int c = 0; c < kN; c += kLoad) tmem_ld_columns<kLoad>(tmem + c, v + c);
    tmem_ld_wait();
#pragma unroll
    for (int r = 0; r < kR; ++r) {
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) {
        const uint32_t u = v[p * kR + r];
        const float x = kInt8 ? static_cast<float>(static_cast<int>(u)) : __uint_as_float(u);
        s[r] = p == kParts - 1 ? x * last : fmaf(x, weight(p), s[r]);
      }
    }
  } else {
    // part after part: fewer registers
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p) {
      uint32_t v[kR];
      tmem_ld_columns<kLoad>(tmem + p * kR, v);
      tmem_ld_wait();
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const float x = kInt8 ? static_cast<float>(static_cast<int>(v[r])) : __uint_as_float(v[r]);
        s[r] = p == kParts - 1 ? x * last : fmaf(x, weight(p), s[r]);
      }
    }
  }
}

// Vote of the softmax warps (named barrier 1).
__device__ __forceinline__ bool any_of_128(bool mine) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return r != 0u;
}
__device__ __forceinline__ void sync_128() {
  __syncwarp();
  asm volatile("bar.sync 1, 128;" ::: "memory");
}

template <typename T, bool kInt8, int kR, bool kCluster>
__global__ void __launch_bounds__(kTcThreads, kR == 32 ? 1 : 2)
    rows_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  using S = Tc<kInt8, kR>;
  constexpr int kN = S::kN, kStages = S::kStages, kParts = S::kParts;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);      // [kStages]
  uint64_t* empty = full + kStages;                                     // [kStages]
  uint64_t* q_full = empty + kStages;
  uint64_t* s_full = q_full + 1;            // [2]
  uint64_t* s_free = s_full + 2;            // [2]
  uint64_t* p_full = s_free + 2;            // [2]
  uint64_t* o_done = p_full + 2;            // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* adds = tmem_slot + 2;  // [2]: whether P V of the buffer's tile adds to what is there
  static_assert((2 * kStages + 9) * 8 + 16 <= 256, "barrier area");
  float* row_factor = reinterpret_cast<float*>(smem + S::kOffRow);
  int* row_pos = reinterpret_cast<int*>(row_factor + kR);
  float* warp_top = reinterpret_cast<float*>(smem + S::kOffMax);        // [4][kR]
  float* part_lse = warp_top + 4 * kR;                                  // [kR]
  float* part_o = reinterpret_cast<float*>(smem);                       // [kR][128], where the stages were

  grid_wait();
  const Place p = place_of<kR>(a);
  if (p.row0 >= p.rows) return;             // surplus rows (of a whole cluster)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.z;
  const int live = min(kR, p.rows - p.row0);
  const int tiles_all = (p.chunks + 7) / 8;
  const int per_split = (tiles_all + a.splits - 1) / a.splits * 8;
  const int c0 = split * per_split, c1 = min(p.chunks, c0 + per_split);
  const int ntiles = c1 > c0 ? (c1 - c0 + 7) / 8 : 0;
  auto first_token = [&](int chunk) { return (chunk < p.firsts ? chunk : p.lo_chunk + chunk - p.firsts) * kChunk; };
  const int* bt = a.block_tables + static_cast<long long>(p.b) * a.max_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 4);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], 4);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_done[b], 1);
    }
    *abort_flag = 0u;
    mbar_fence_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_release();                           // (behind the allocation, see common.cuh)

  if (warp == 4) {
    // ---------------- TMA: lane = chunk of a tile, keys or values ----------------
    const int chunk = (lane >> 1) & 7, kv = lane & 1;
    auto row_of = [&](int it) {
      const int c = c0 + it * 8 + chunk;
      if (c >= c1) return 0;
      const int tok = first_token(c);
      return bt[tok / a.block_size] * a.block_size + tok % a.block_size;
    };
    int row = row_of(0);
    for (int it = 0; it < ntiles; ++it) {
      const int next = row_of(it + 1);
      const int st = it % kStages;
      if (!mbar_wait_warp(&empty[st], ((it / kStages) & 1) ^ 1, a.status, kKernelId, 0x300u + st, abort_flag)) break;
      const int n = min(8, c1 - c0 - it * 8);
      if (lane == 0) mbar_expect_tx(&full[st], static_cast<uint32_t>(n) * 2u * kChunk * 128u);
      __syncwarp();
      if (lane < 2 * n)
        tma_load_2d(smem + st * kTcStageBytes + kv * (kTcStageBytes / 2) + chunk * (kChunk * 128), kv == 0 ? &tmK : &tmV,
                    &full[st], p.kvh * 128, row);
      row = next;
    }
  } else if (warp == 5) {
    // ---------------- tcgen05.mma ----------------
    if (elect_one()) {
      constexpr uint32_t kA = kInt8 ? 1 : 0, kC = kInt8 ? 2 : 1;          // s8 or e4m3, s32 or f32
      constexpr uint32_t kIdescS = make_idesc(kTcTile, kN, kA, kA, kC);
      constexpr uint32_t kIdescO = make_idesc(128, kN, kA, kA, kC) | 1u << 15;      // A is MN-major
      const uint64_t q_desc = make_desc_k_sw128(smem_u32(smem + S::kOffQ));
      const uint64_t p_desc = make_desc_k_sw128(smem_u32(smem + S::kOffP));
      const uint64_t k_desc = make_desc_k_sw128(smem_u32(smem));
      const uint64_t v_desc = make_desc_mn_sw128(smem_u32(smem) + kTcStageBytes / 2, kTcTile * 128);
      auto pv = [&](int j) -> bool {
        const int b = j & 1, st = j % kStages;
        if (!mbar_wait(&p_full[b], (j >> 1) & 1, a.status, kKernelId, 0x320u + b, abort_flag)) return false;
        tc_fence_after();
        const uint32_t add = adds[b];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8<kInt8>(tmem + 2 * kN, v_desc + static_cast<uint32_t>((st * kTcStageBytes + ks * 4096) >> 4),
                      p_desc + static_cast<uint32_t>((b * kN * 128 + ks * 32) >> 4), kIdescO, add | (ks > 0 ? 1u : 0u));
        umma_commit(&o_done[b]);
        umma_commit(&empty[st]);
        return true;
      };
      bool ok = ntiles == 0 || mbar_wait(q_full, 0, a.status, kKernelId, 0x322u, abort_flag);
      for (int it = 0; ok && it < ntiles; ++it) {
        const int b = it & 1, st = it % kStages;
        ok = mbar_wait(&full[st], (it / kStages) & 1, a.status, kKernelId, 0x330u + st, abort_flag) &&
             mbar_wait(&s_free[b], ((it >> 1) & 1) ^ 1, a.status, kKernelId, 0x340u + b, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8<kInt8>(tmem + b * kN, k_desc + static_cast<uint32_t>((st * kTcStageBytes + ks * 32) >> 4),
                      q_desc + static_cast<uint32_t>(ks * 2), kIdescS, ks > 0 ? 1u : 0u);
        umma_commit(&s_full[b]);
        if (it > 0) ok = pv(it - 1);
      }
      if (ok && ntiles > 0) pv(ntiles - 1);
    }
    __syncwarp();
  } else {
    // ---------------- queries ----------------
    for (int r = warp; r < kR; r += 4) {
      const int row = p.row0 + r;
      const bool valid = r < live;
      const int token = row / p.G, head = p.kvh * p.G + row % p.G;
      uint2 raw = make_uint2(0u, 0u);
      if (valid)
        raw = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) +
                                              static_cast<long long>(p.q_start + token) * a.ldq + head * 128 + lane * 4);
      const T* e = reinterpret_cast<const T*>(&raw);
      float x[4], top = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = to_f32<T>(e[i]);
        top = fmaxf(top, finite_size(x[i]));
      }
      const int e2 = max(-100, min(126, static_cast<int>(__float_as_uint(warp_max(top)) >> 23) - 127));
      uint32_t w[3] = {0u, 0u, 0u};
      float unit;                           // of the parts, times 2^e2
      if constexpr (kInt8) {
        // |x| 2^-e2 < 2 as whole numbers below 2^20 in magnitude, digits -64 .. 63 (the first up to 64)
        const float down = power_of_two(-e2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = __float2int_rn(fminf(fmaxf(x[i] * down, -2.0f), 2.0f) * 524287.0f);
          const int d2 = ((f + 64) & 127) - 64, f1 = (f - d2) >> 7;
          const int d1 = ((f1 + 64) & 127) - 64, d0 = (f1 - d1) >> 7;
          w[0] |= static_cast<uint32_t>(d0 & 255) << (8 * i);
          w[1] |= static_cast<uint32_t>(d1 & 255) << (8 * i);
          w[2] |= static_cast<uint32_t>(d2 & 255) << (8 * i);
        }
        unit = 1.0f / 524287.0f;
      } else {
        // the largest in [128, 256), in 32 bits: a bf16 number's 8 bits are two parts, an fp16 number's 11 are three
        const float down = power_of_two(-e2);
        unit = 1.0f / 128.0f;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float y0 = x[i] * down * 128.0f, y1 = x[i + 1] * down * 128.0f;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
            w[k] |= c << (8 * i);
            y0 = (y0 - e4m3_to_f32(static_cast<uint8_t>(c & 255u))) * 16.0f;
            y1 = (y1 - e4m3_to_f32(static_cast<uint8_t>(c >> 8))) * 16.0f;
          }
        }
      }
      const bool wrong = __any_sync(0xffffffffu, !(fabsf(x[0]) < INFINITY) || !(fabsf(x[1]) < INFINITY) ||
                                                     !(fabsf(x[2]) < INFINITY) || !(fabsf(x[3]) < INFINITY));
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int n = k * kR + r;
        *reinterpret_cast<uint32_t*>(smem + S::kOffQ + (n >> 3) * 1024 + (n & 7) * 128 + (((lane >> 2) ^ (n & 7)) << 4) +
                                     (lane & 3) * 4) = w[k];
      }
      if (lane == 0) {
        // (a row that holds infinities or NaN gives NaN, as its products do)
        row_factor[r] = wrong ? __int_as_float(0x7fffffff) : power_of_two(e2) * unit * a.scale * kLog2e;
        row_pos[r] = p.pos0 + min(token, (p.rows - 1) / p.G);
      }
    }
    // columns of no row, of queries and of both buffers of probabilities
    for (int i = threadIdx.x; i < (kN - 3 * kR) * 32; i += 128) {
      const int n = 3 * kR + (i >> 5);
      const int at = (n >> 3) * 1024 + (n & 7) * 128 + (i & 31) * 4;
      *reinterpret_cast<uint32_t*>(smem + S::kOffQ + at) = 0u;
      if (n < kParts * kR) continue;
      *reinterpret_cast<uint32_t*>(smem + S::kOffP + at) = 0u;
      *reinterpret_cast<uint32_t*>(smem + S::kOffP + kN * 128 + at) = 0u;
    }
    fence_async_smem();
    sync_128();                             // (factors and positions)
    if (lane == 0) mbar_arrive(q_full);

    // ---------------- softmax: lane = token of the tile ----------------
    const int i_tok = warp * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    float m[kR], l[kR], o[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      m[r] = -INFINITY;
      l[r] = o[r] = 0.0f;
    }
    // what P V of earlier tiles left in tensor memory
    constexpr float kUnit = kInt8 ? 67108864.0f : 64.0f;       // of a probability: 4 of them fill the parts
    constexpr float kBack = 1.0f / kUnit;
    auto drain = [&]() {
      float v[kR];
      sum_parts<kInt8, kR, kParts>(lane_addr + 2 * kN, v);
#pragma unroll
      for (int r = 0; r < kR; ++r) o[r] = fmaf(v[r], kBack, o[r]);
    };
    auto block_of = [&](int it) {           // of this lane's token, -1: none
      const int c = c0 + it * 8 + (i_tok >> 4);
      return it < ntiles && c < c1 ? bt[first_token(c) / a.block_size] : -1;
    };
    auto scales_of = [&](int it, int block, float& ks, float& vs) {
      ks = 0.0f;
      vs = power_of_two(kLowExponent);      // (a block that was never written has no scale: its keys count all the same)
      if (block >= 0 && block < a.num_blocks) {
        const long long at = static_cast<long long>(block) * a.Hkv + p.kvh;
        ks = a.ks[at];
        vs = fmaxf(a.vs[at], vs);
      } else if (it < ntiles && c0 + it * 8 + (i_tok >> 4) < c1) {
        report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(p.b));
      }
    };
    float ks, vs;
    scales_of(0, block_of(0), ks, vs);
    int block_next = block_of(1);
    bool drained = true;                    // nothing of this epoch in tensor memory
    for (int it = 0; it < ntiles; ++it) {
      const int b = it & 1;
      float ks_next, vs_next;
      scales_of(it + 1, block_next, ks_next, vs_next);
      block_next = block_of(it + 2);
      const int c = c0 + it * 8 + (i_tok >> 4);
      const int tok = first_token(c) + (i_tok & 15);
      const bool there = c < c1;
      const bool whole = there && tok <= p.lo_pos && (a.window <= 0 || tok > p.hi_pos - a.window || tok < a.first);
      const bool all_whole = __all_sync(0xffffffffu, whole);
      mbar_pass_warp(&s_full[b], (it >> 1) & 1, a.status, kKernelId, 0x350u + b, abort_flag);
      tc_fence_after();
      float x[kR];
      sum_parts<kInt8, kR, 3>(lane_addr + b * kN, x);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[b]);
      const float l2vs = __log2f(vs), unit = __fdividef(1.0f, vs);
      bool over = kInt8 && it % kMostTiles == kMostTiles - 1;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        x[r] = fmaf(x[r], row_factor[r] * ks, l2vs);
        if (!all_whole) {
          const int pos = row_pos[r];
          if (!there || tok > pos || (a.window > 0 && tok <= pos - a.window && tok >= a.first)) x[r] = -INFINITY;
        }
        over = over || x[r] > m[r] + kRaise;
      }
      if (any_of_128(over)) {
        // new maxima of all rows; the sums in tensor memory belong to the old ones
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float top = warp_max(x[r]);
          if (lane == 0) warp_top[warp * kR + r] = top;
        }
        sync_128();
        if (!drained) {
          mbar_pass_warp(&o_done[b ^ 1], ((it - 1) >> 1) & 1, a.status, kKernelId, 0x360u, abort_flag);
          tc_fence_after();
          drain();
          tc_fence_before();
        }
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float top = fmaxf(fmaxf(warp_top[r], warp_top[kR + r]), fmaxf(warp_top[2 * kR + r], warp_top[3 * kR + r]));
          const float m_new = fmaxf(m[r], top);
          const float corr = m[r] == -INFINITY ? 0.0f : ex2(m[r] - m_new);
          m[r] = m_new;
          l[r] *= corr;
          o[r] *= corr;
        }
        sync_128();                         // (warp_top is free again)
        drained = true;
      }
      if (threadIdx.x == 0) adds[b] = drained ? 0u : 1u;
      drained = false;
      // P V two tiles ago has read this buffer
      if (it >= 2) mbar_pass_warp(&o_done[b], ((it - 2) >> 1) & 1, a.status, kKernelId, 0x370u + b, abort_flag);
      uint8_t* sp = smem + S::kOffP + b * kN * 128 + (i_tok & 15);
      const int c16 = i_tok >> 4;
      auto put = [&](int n, uint32_t byte) {
        sp[(n >> 3) * 1024 + (n & 7) * 128 + ((c16 ^ (n & 7)) << 4)] = static_cast<uint8_t>(byte);
      };
#pragma unroll
      for (int r = 0; r < kR; r += 2) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mr = m[r + e] == -INFINITY ? 0.0f : m[r + e];
          v[e] = ex2(x[r + e] - mr);        // up to 4
          l[r + e] = fmaf(v[e], unit, l[r + e]);
        }
        if constexpr (kInt8) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t f = min(__float2uint_rn(v[e] * kUnit), (1u << 28) - 1u);
#pragma unroll
            for (int k = 0; k < kParts; ++k) put(k * kR + r + e, f >> 7 * (kParts - 1 - k) & 127u);
          }
        } else {
          uint32_t q[3];
          parts_e4m3(pack_half(v[0] * kUnit, v[1] * kUnit), q);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            put(k * kR + r, q[k]);
            put(k * kR + r + 1, q[k] >> 8);
          }
        }
      }
      if (!all_whole) {
        // what lies behind the last key, in a gap that no row sees, or was not loaded may be anything
        if (!there || tok > p.hi_pos || (a.window > 0 && tok <= p.lo_pos - a.window && tok >= a.first)) {
          uint4* v = reinterpret_cast<uint4*>(smem + it % kStages * kTcStageBytes + kTcStageBytes / 2 + i_tok * 128);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k ^ (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[b]);
      ks = ks_next;
      vs = vs_next;
    }
    if (ntiles > 0) {
      mbar_pass_warp(&o_done[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1, a.status, kKernelId, 0x380u, abort_flag);
      tc_fence_after();
      drain();
      tc_fence_before();
    }
    // sums over the tokens
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const float sum = warp_sum(l[r]);
      if (lane == 0) warp_top[warp * kR + r] = *abort_flag != 0u ? 0.0f : sum;
    }
    sync_128();
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (r >= live) break;
      const float L = (warp_top[r] + warp_top[kR + r]) + (warp_top[2 * kR + r] + warp_top[3 * kR + r]);
      const float val = L == 0.0f ? 0.0f : o[r] / L;
      const float mr = m[r] == -INFINITY ? 0.0f : m[r];
      const float lse = L == 0.0f ? -INFINITY : mr + log2f(L);
      const int d = i_tok;
      if constexpr (kCluster) {
        part_o[r * 128 + d] = val;
        if (d == 0) part_lse[r] = lse;
        continue;
      }
      const int row = p.row0 + r, token = p.q_start + row / p.G, head = p.kvh * p.G + row % p.G;
      if (a.splits > 1) {
        const long long base = (static_cast<long long>(token) * a.Hq + head) * a.splits + split;
        a.tmp_out[base * 128 + d] = val;
        if (d == 0) a.tmp_lse[base] = lse;
      } else {
        static_cast<T*>(a.out)[static_cast<long long>(token) * a.ldo + head * 128 + d] = from_f32<T>(val);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, S::kAlloc);
  if constexpr (kCluster) merge_cluster<T, 128>(a, p, live, part_lse, part_o);
}

template <typename T, bool kInt8, int kR, bool kCluster>
int launch_tc(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, cudaStream_t s) {
  static_assert(Tc<kInt8, kR>::kBytes <= 232448, "exceeds the shared memory of one CTA");
  static_assert(kR * 128 * 4 <= Tc<kInt8, kR>::kOffQ, "merge buffers must fit");
  static bool done[64] = {};
  return launch_splits(rows_tc_kernel<T, kInt8, kR, kCluster>, done, kTcThreads, Tc<kInt8, kR>::kBytes, kCluster, a, tmK, tmV, s);
}

}  // namespace rows8
}  // namespace b200

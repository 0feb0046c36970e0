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
// Warps: 0..3 (32 rows: 0..7) queries and softmax, lane = token of a tile and at the end column of the output; then one
// for TMA, block tables and scales and one for tcgen05.mma and tensor memory.  K Q^T of a tile runs while the one before is
// at its softmax; keys and values have places of their own, given back when their product is done.
// The running maximum is raised when a score exceeds it by 4 (log2), which all softmax warps vote on; then the sums in
// tensor memory are taken to registers, rescaled, and start anew (rare behind the first tiles, and the only form for sums
// of whole numbers).
#pragma once

namespace b200 {
namespace rows8 {

constexpr int kTcTile = 128;                 // tokens of a tile
constexpr int kTcBytes = kTcTile * 128;      // of its keys, or values
constexpr int kGroup = 4;                    // tiles whose block-table entries and scales a lane each of the TMA warp reads
constexpr int kGroups = 4;                   // places for their scales
constexpr float kRaise = 4.0f;               // log2, by which a score may exceed the running maximum
constexpr int kMostTiles = 512;              // int8: whose sums of whole numbers one accumulator takes, 2^16 * 127 * 128 < 2^31

template <bool kInt8, int kR>
struct Tc {
  static constexpr int kParts = kInt8 ? 4 : 3;                 // of a probability
  static constexpr int kNS = (3 * kR + 15) / 16 * 16;          // columns of scores
  static constexpr int kN = (kParts * kR + 15) / 16 * 16;      // and of outputs
  static constexpr int kWarps = kR == 32 ? 8 : 4;              // of the softmax
  static constexpr int kRW = kR * 4 / kWarps;                  // rows of one of them
  static constexpr int kThreads = kWarps * 32 + 64;
  // CTAs of an SM, which hide each other's starts and ends, and places for keys and values of each
  static constexpr int kCtas = kR == 4 ? 3 : 2;
  static constexpr int kStages = kR == 8 ? 3 : 2;
  static constexpr int kScores = kR == 32 ? 1 : 2;             // score buffers (32 rows: else one CTA had all of tensor memory)
  static constexpr int kColumns = kScores * kNS + kN;
  static constexpr int kAlloc = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : 256;
  static_assert(kColumns <= 256, "tensor memory of two CTAs");
  static constexpr int kOffQ = 2 * kStages * kTcBytes;         // (keys, then values in front)
  static constexpr int kOffP = kOffQ + kNS * 128;
  static constexpr int kOffScale = kOffP + 2 * kN * 128;       // [kGroups][32] scales of keys, log2 and inverse of values', flag
  static constexpr int kOffBar = kOffScale + kGroups * 32 * 16;
  static constexpr int kOffRow = kOffBar + 256;                // factor and position of every row
  static constexpr int kOffMax = kOffRow + 2 * kR * 4;         // of four warps and every row; log2 sums of the rows
  static constexpr int kBytes = kOffMax + 5 * kR * 4 + 1024;
};

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

// Numbers of a lane's columns, parts put together: column part * kStride + row -> [row].
template <bool kInt8, int kRW, int kStride, int kParts>
__device__ __forceinline__ void sum_parts(uint32_t tmem, float (&s)[kRW]) {
  // weights of the parts: 128^-p (the last digit's is 1) or 16^-p
  auto weight = [](int p) {
    return kInt8 ? static_cast<float>(1 << 7 * (kParts - 1 - p)) : 1.0f / static_cast<float>(1 << 4 * p);
  };
  const float last = weight(kParts - 1);
  auto number = [](uint32_t u) { return kInt8 ? static_cast<float>(static_cast<int>(u)) : __uint_as_float(u); };
  if constexpr (kStride <= 8) {
    constexpr int kLoads = (kParts * kStride + 15) / 16;
    uint32_t v[kLoads * 16];
#pragma unroll
    for (int c = 0; c < kLoads; ++c) tmem_ld_32x16(tmem + c * 16, *reinterpret_cast<uint32_t(*)[16]>(v + c * 16));
    tmem_ld_wait();
#pragma unroll
    for (int r = 0; r < kRW; ++r) {
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) {
        const float x = number(v[p * kStride + r]);
        s[r] = p == kParts - 1 ? x * last : fmaf(x, weight(p), s[r]);
      }
    }
  } else {
    static_assert(kStride <= 8 || kRW == 16, "one load a part");
    // (part after part: registers)
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p) {
      uint32_t v[16];
      tmem_ld_32x16(tmem + p * kStride, v);
      tmem_ld_wait();
#pragma unroll
      for (int r = 0; r < kRW; ++r) s[r] = p == kParts - 1 ? number(v[r]) * last : fmaf(number(v[r]), weight(p), s[r]);
    }
  }
}

// Vote of the softmax warps (named barrier 1).
template <int kThreads>
__device__ __forceinline__ bool any_of(bool mine) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(mine)), "n"(kThreads)
      : "memory");
  return r != 0u;
}
template <int kThreads>
__device__ __forceinline__ void sync_softmax() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
}
// Largest number of a warp (NaN aside), by the order of whole numbers.
__device__ __forceinline__ float warp_top_of(float x) {
  int i = __float_as_int(x == x ? x : -INFINITY);
  i = i < 0 ? i ^ 0x7fffffff : i;
  i = __reduce_max_sync(0xffffffffu, i);
  return __int_as_float(i < 0 ? i ^ 0x7fffffff : i);
}

template <typename T, bool kInt8, int kR, bool kCluster>
__global__ void __launch_bounds__(Tc<kInt8, kR>::kThreads, Tc<kInt8, kR>::kCtas)
    rows_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  using S = Tc<kInt8, kR>;
  constexpr int kN = S::kN, kNS = S::kNS, kStages = S::kStages, kParts = S::kParts, kWarps = S::kWarps, kRW = S::kRW, kScores = S::kScores;
  constexpr int kSoft = kWarps * 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);    // [kStages]
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* q_full = v_empty + kStages;
  uint64_t* c_full = q_full + 1;            // [kGroups] scales of a group of tiles
  uint64_t* s_full = c_full + kGroups;      // [kScores]
  uint64_t* s_free = s_full + kScores;      // [kScores]
  uint64_t* p_full = s_free + kScores;      // [2]
  uint64_t* o_done = p_full + 2;            // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* adds = tmem_slot + 2;  // [2]: whether P V of the buffer's tile adds to what is there
  static_assert((4 * kStages + 5 + kGroups + 2 * kScores) * 8 + 16 <= 256, "barrier area");
  float4* chunk_scale = reinterpret_cast<float4*>(smem + S::kOffScale);
  float* row_factor = reinterpret_cast<float*>(smem + S::kOffRow);
  int* row_pos = reinterpret_cast<int*>(row_factor + kR);
  float* warp_top = reinterpret_cast<float*>(smem + S::kOffMax);        // [4][kR]
  float* part_lse = warp_top + 4 * kR;                                  // [kR]
  float* part_o = reinterpret_cast<float*>(smem);                       // [kR][128], where keys were

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

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(q_full, kWarps);
    for (int g = 0; g < kGroups; ++g) mbar_init(&c_full[g], 1);
    for (int b = 0; b < kScores; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], kWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&p_full[b], kWarps);
      mbar_init(&o_done[b], 1);
    }
    *abort_flag = 0u;
    mbar_fence_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == kWarps + 1) {
    tmem_alloc(tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_release();                           // (behind the allocation, see common.cuh)

  if (warp == kWarps) {
    // ---------------- TMA, block tables, scales ----------------
    // lane = (tile of a group of four, chunk of it); a group's blocks are read two groups ahead, its scales one
    const int* bt = a.block_tables + static_cast<long long>(p.b) * a.max_blocks;
    auto chunk_of = [&](int g) { return c0 + g * (8 * kGroup) + lane; };
    auto block_of = [&](int g) {
      const int c = chunk_of(g);
      return c < c1 ? bt[first_token(c) / a.block_size] : 0;
    };
    auto row_of = [&](int g, int block) { return block * a.block_size + first_token(chunk_of(g)) % a.block_size; };
    auto scales_of = [&](int g, int block) {
      float4 s = make_float4(0.0f, power_of_two(kLowExponent), 0.0f, 0.0f);
      const int c = chunk_of(g);
      if (c >= c1) return s;
      if (block >= 0 && block < a.num_blocks) {
        const long long at = static_cast<long long>(block) * a.Hkv + p.kvh;
        s.x = a.ks[at];
        s.y = a.vs[at];
      } else {
        report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(p.b));
      }
      return s;
    };
    auto publish = [&](int g, float4 s) {
      const int c = chunk_of(g), tok = first_token(c);
      // (a block that was never written has no scale: its keys count all the same)
      const float vs = fmaxf(s.y, power_of_two(kLowExponent));
      s.y = __log2f(vs);
      s.z = __fdividef(1.0f, vs);
      // whether all rows see all of the chunk
      s.w = c < c1 && tok + kChunk - 1 <= p.lo_pos && (a.window <= 0 || tok > p.hi_pos - a.window || tok + kChunk <= a.first)
                ? 1.0f : 0.0f;
      chunk_scale[g % kGroups * 32 + lane] = s;
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_full[g % kGroups]);
    };
    int block = block_of(0), block_next = block_of(1);
    float4 scales = scales_of(0, block);
    int row = row_of(0, block), row_next = row_of(1, block_next);
    bool ok = true;
    // copies of tile `it`, whose rows lie in `rows`
    auto copy = [&](int it, int rows, bool values) {
      const int st = it % kStages, n = min(8, c1 - c0 - it * 8);
      ok = mbar_wait_warp(values ? &v_empty[st] : &k_empty[st], ((it / kStages) & 1) ^ 1, a.status, kKernelId,
                          0x300u + st, abort_flag);
      if (!ok) return;
      const int y = __shfl_sync(0xffffffffu, rows, it % kGroup * 8 + (lane & 7));
      uint64_t* bar = values ? &v_full[st] : &k_full[st];
      if (lane == 0) mbar_expect_tx(bar, static_cast<uint32_t>(n) * kChunk * 128u);
      __syncwarp();
      if (lane < n)
        tma_load_2d(smem + ((values ? kStages : 0) + st) * kTcBytes + lane * (kChunk * 128), values ? &tmV : &tmK, bar,
                    p.kvh * 128, y);
    };
    if (ntiles > 0) copy(0, row, false);
    for (int it = 0; it < ntiles && ok; ++it) {
      const int g = it / kGroup;
      const bool first = it % kGroup == 0;
      int block_after = 0;
      float4 scales_next = scales;
      if (first) {
        block_after = block_of(g + 2);
        scales_next = scales_of(g + 1, block_next);
      }
      if (it + 1 < ntiles) copy(it + 1, (it + 1) % kGroup == 0 ? row_next : row, false);
      if (ok) copy(it, row, true);
      // (behind the copies: nothing in front waits for this tile's softmax)
      if (first) {
        publish(g, scales);
        scales = scales_next;
        block_next = block_after;
      }
      if (it % kGroup == kGroup - 1) {
        row = row_next;
        row_next = row_of(g + 2, block_next);
      }
    }
  } else if (warp == kWarps + 1) {
    // ---------------- tcgen05.mma ----------------
    if (elect_one()) {
      constexpr uint32_t kA = kInt8 ? 1 : 0, kC = kInt8 ? 2 : 1;          // s8 or e4m3, s32 or f32
      constexpr uint32_t kIdescS = make_idesc(kTcTile, kNS, kA, kA, kC);
      constexpr uint32_t kIdescO = make_idesc(128, kN, kA, kA, kC) | 1u << 15;      // A is MN-major
      const uint64_t q_desc = make_desc_k_sw128(smem_u32(smem + S::kOffQ));
      const uint64_t p_desc = make_desc_k_sw128(smem_u32(smem + S::kOffP));
      const uint64_t k_desc = make_desc_k_sw128(smem_u32(smem));
      const uint64_t v_desc = make_desc_mn_sw128(smem_u32(smem + kStages * kTcBytes), kTcBytes);
      auto pv = [&](int j) -> bool {
        const int b = j & 1, st = j % kStages;
        if (!mbar_wait(&v_full[st], (j / kStages) & 1, a.status, kKernelId, 0x310u + st, abort_flag) ||
            !mbar_wait(&p_full[b], (j >> 1) & 1, a.status, kKernelId, 0x320u + b, abort_flag))
          return false;
        tc_fence_after();
        const uint32_t add = adds[b];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8<kInt8>(tmem + kScores * kNS, v_desc + static_cast<uint32_t>((st * kTcBytes + ks * 4096) >> 4),
                      p_desc + static_cast<uint32_t>((b * kN * 128 + ks * 32) >> 4), kIdescO, add | (ks > 0 ? 1u : 0u));
        umma_commit(&o_done[b]);
        umma_commit(&v_empty[st]);
        return true;
      };
      bool ok = ntiles == 0 || mbar_wait(q_full, 0, a.status, kKernelId, 0x322u, abort_flag);
      for (int it = 0; ok && it < ntiles; ++it) {
        const int b = it % kScores, st = it % kStages;
        ok = mbar_wait(&k_full[st], (it / kStages) & 1, a.status, kKernelId, 0x330u + st, abort_flag) &&
             mbar_wait(&s_free[b], ((it / kScores) & 1) ^ 1, a.status, kKernelId, 0x340u + b, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8<kInt8>(tmem + b * kNS, k_desc + static_cast<uint32_t>((st * kTcBytes + ks * 32) >> 4),
                      q_desc + static_cast<uint32_t>(ks * 2), kIdescS, ks > 0 ? 1u : 0u);
        umma_commit(&s_full[b]);
        umma_commit(&k_empty[st]);
        if (it > 0) ok = pv(it - 1);
      }
      if (ok && ntiles > 0) pv(ntiles - 1);
    }
    __syncwarp();
  } else {
    // ---------------- queries ----------------
    for (int r = warp; r < kR; r += kWarps) {
      const int row = p.row0 + r;
      const int token = row / p.G, head = p.kvh * p.G + row % p.G;
      uint2 raw = make_uint2(0u, 0u);
      if (r < live)
        raw = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) +
                                              static_cast<long long>(p.q_start + token) * a.ldq + head * 128 + lane * 4);
      const T* e = reinterpret_cast<const T*>(&raw);
      float x[4], top = 0.0f;
      bool number = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = to_f32<T>(e[i]);
        number = number && fabsf(x[i]) < INFINITY;
        top = fmaxf(top, finite_size(x[i]));
      }
      const int e2 = max(-100, min(126, static_cast<int>(__float_as_uint(warp_top_of(top)) >> 23) - 127));
      const float down = power_of_two(-e2);
      uint32_t w[3] = {0u, 0u, 0u};
      float unit;                           // of the parts, times 2^e2
      if constexpr (kInt8) {
        // |x| 2^-e2 < 2 as whole numbers of 21 bits, digits -64 .. 63 (the first one up to 64)
        unit = 1.0f / 524287.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = __float2int_rn(fminf(fmaxf(x[i] * down, -2.0f), 2.0f) * 524287.0f);
          const int d2 = ((f + 64) & 127) - 64, f1 = (f - d2) >> 7;
          const int d1 = ((f1 + 64) & 127) - 64, d0 = (f1 - d1) >> 7;
          w[0] |= static_cast<uint32_t>(d0 & 255) << (8 * i);
          w[1] |= static_cast<uint32_t>(d1 & 255) << (8 * i);
          w[2] |= static_cast<uint32_t>(d2 & 255) << (8 * i);
        }
      } else {
        // the largest in [128, 256), in 32 bits: a bf16 number's 8 bits are two parts, an fp16 number's 11 are three
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
      number = __all_sync(0xffffffffu, number);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int n = k * kR + r;
        *reinterpret_cast<uint32_t*>(smem + S::kOffQ + (n >> 3) * 1024 + (n & 7) * 128 + (((lane >> 2) ^ (n & 7)) << 4) +
                                     (lane & 3) * 4) = w[k];
      }
      if (lane == 0) {
        // (a row that holds infinities or NaN gives NaN, as its products do)
        row_factor[r] = number ? power_of_two(e2) * unit * a.scale * kLog2e : __int_as_float(0x7fffffff);
        row_pos[r] = p.pos0 + min(token, (p.rows - 1) / p.G);
      }
    }
    // columns of no row, of queries and of both buffers of probabilities
    auto clear = [&](int from, int to, int off) {
      for (int i = threadIdx.x; i < (to - from) * 32; i += kSoft) {
        const int n = from + (i >> 5);
        *reinterpret_cast<uint32_t*>(smem + off + (n >> 3) * 1024 + (n & 7) * 128 + (i & 31) * 4) = 0u;
      }
    };
    clear(3 * kR, kNS, S::kOffQ);
    clear(kParts * kR, kN, S::kOffP);
    clear(kParts * kR, kN, S::kOffP + kN * 128);
    fence_async_smem();
    sync_softmax<kSoft>();                  // (factors and positions)
    if (lane == 0) mbar_arrive(q_full);

    // ---------------- softmax: lane = token of the tile ----------------
    const int row0 = warp / 4 * kRW;        // first row of the warp
    const int i_tok = (warp & 3) * 32 + lane, c16 = i_tok >> 4;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + row0;
    float m[kRW], l[kRW], o[kRW];
#pragma unroll
    for (int r = 0; r < kRW; ++r) {
      m[r] = -INFINITY;
      l[r] = o[r] = 0.0f;
    }
    constexpr float kUnit = kInt8 ? 16777216.0f : 16.0f;       // of a probability: 16 of them fill the parts
    // what P V of earlier tiles left in tensor memory
    auto drain = [&]() {
      float v[kRW];
      sum_parts<kInt8, kRW, kR, kParts>(lane_addr + kScores * kNS, v);
#pragma unroll
      for (int r = 0; r < kRW; ++r) o[r] = fmaf(v[r], 1.0f / kUnit, o[r]);
    };
    bool drained = true;                    // nothing of these maxima in tensor memory
    for (int it = 0; it < ntiles; ++it) {
      const int g = it / kGroup;
      if (it % kGroup == 0)
        mbar_pass_warp(&c_full[g % kGroups], (g / kGroups) & 1, a.status, kKernelId, 0x390u, abort_flag);
      const float4 scale = chunk_scale[g % kGroups * 32 + it % kGroup * 8 + c16];
      const bool all_whole = __all_sync(0xffffffffu, scale.w != 0.0f);
      // (the scores of a tile are there when P V two tiles ago is done, which was issued before: its probabilities may
      // be overwritten)
      mbar_pass_warp(&s_full[it % kScores], (it / kScores) & 1, a.status, kKernelId, 0x350u, abort_flag);
      tc_fence_after();
      float x[kRW];
      sum_parts<kInt8, kRW, kR, 3>(lane_addr + it % kScores * kNS, x);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[it % kScores]);
#pragma unroll
      for (int r = 0; r < kRW; ++r) x[r] *= row_factor[row0 + r] * scale.x;
      int tok = 0;
      bool lost = false;                    // no row sees the token
      if (!all_whole) {
        const int c = c0 + it * 8 + c16;
        const bool there = c < c1;
        tok = first_token(c) + (i_tok & 15);
        lost = !there || tok > p.hi_pos || (a.window > 0 && tok <= p.lo_pos - a.window && tok >= a.first);
#pragma unroll
        for (int r = 0; r < kRW; ++r) {
          const int pos = row_pos[row0 + r];
          if (!there || tok > pos || (a.window > 0 && tok <= pos - a.window && tok >= a.first)) x[r] = -INFINITY;
        }
      }
      // exponents, relative to the running maximum (in place: a new maximum moves them on)
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < kRW; ++r) {
        x[r] += scale.y - (m[r] == -INFINITY ? 0.0f : m[r]);
        top = fmaxf(top, m[r] == -INFINITY && x[r] > -INFINITY ? INFINITY : x[r]);
      }
      if (any_of<kSoft>(top > kRaise || (kInt8 && it % kMostTiles == kMostTiles - 1))) {
        // new maxima of all rows; the sums in tensor memory belong to the old ones
#pragma unroll
        for (int r = 0; r < kRW; ++r) {
          const float t = warp_top_of(x[r]);
          if (lane == 0) warp_top[(warp & 3) * kR + row0 + r] = t;
        }
        sync_softmax<kSoft>();
        if (!drained) {
          mbar_pass_warp(&o_done[(it - 1) & 1], ((it - 1) >> 1) & 1, a.status, kKernelId, 0x360u, abort_flag);
          tc_fence_after();
          drain();
          tc_fence_before();
        }
#pragma unroll
        for (int r = 0; r < kRW; ++r) {
          const float* t = warp_top + row0 + r;
          const float over = fmaxf(fmaxf(t[0], t[kR]), fmaxf(t[2 * kR], t[3 * kR]));       // the old maximum
          if (over > 0.0f || m[r] == -INFINITY) {
            const float up = over == -INFINITY ? 0.0f : over;
            const float corr = m[r] == -INFINITY ? 0.0f : ex2(-up);
            m[r] = over == -INFINITY ? m[r] : m[r] == -INFINITY ? over : m[r] + over;
            l[r] *= corr;
            o[r] *= corr;
            x[r] -= up;
          }
        }
        sync_softmax<kSoft>();              // (warp_top is free again)
        drained = true;
      }
      if (threadIdx.x == 0) adds[it & 1] = drained ? 0u : 1u;
      drained = false;
      uint8_t* sp = smem + S::kOffP + (it & 1) * kN * 128 + (i_tok & 15);
      auto put = [&](int n, uint32_t byte) {
        sp[(n >> 3) * 1024 + (n & 7) * 128 + ((c16 ^ (n & 7)) << 4)] = static_cast<uint8_t>(byte);
      };
#pragma unroll
      for (int r = 0; r < kRW; r += 2) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[e] = ex2(x[r + e]);             // up to 16
          l[r + e] = fmaf(v[e], scale.z, l[r + e]);
        }
        if constexpr (kInt8) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t f = min(__float2uint_rn(v[e] * kUnit), (1u << 28) - 1u);
#pragma unroll
            for (int k = 0; k < kParts; ++k) put(k * kR + row0 + r + e, f >> 7 * (kParts - 1 - k) & 127u);
          }
        } else {
          uint32_t q[3];
          parts_e4m3(pack_half(v[0] * kUnit, v[1] * kUnit), q);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            put(k * kR + row0 + r, q[k]);
            put(k * kR + row0 + r + 1, q[k] >> 8);
          }
        }
      }
      if (lost && warp < 4) {
        // what lies behind the last key, in a gap that no row sees, or was not loaded may be anything
        mbar_wait(&v_full[it % kStages], (it / kStages) & 1, a.status, kKernelId, 0x3a0u, abort_flag);
        uint4* v = reinterpret_cast<uint4*>(smem + (kStages + it % kStages) * kTcBytes + i_tok * 128);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k ^ (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[it & 1]);
    }
    if (ntiles > 0) {
      mbar_pass_warp(&o_done[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1, a.status, kKernelId, 0x380u, abort_flag);
      tc_fence_after();
      drain();
      tc_fence_before();
    }
    // sums over the tokens
#pragma unroll
    for (int r = 0; r < kRW; ++r) {
      const float sum = warp_sum(l[r]);
      if (lane == 0) warp_top[(warp & 3) * kR + row0 + r] = *abort_flag != 0u ? 0.0f : sum;
    }
    sync_softmax<kSoft>();
#pragma unroll
    for (int r = 0; r < kRW; ++r) {
      if (row0 + r >= live) break;
      const float* t = warp_top + row0 + r;
      const float L = (t[0] + t[kR]) + (t[2 * kR] + t[3 * kR]);
      const float val = L == 0.0f ? 0.0f : o[r] / L;
      const float lse = L == 0.0f ? -INFINITY : (m[r] == -INFINITY ? 0.0f : m[r]) + log2f(L);
      const int d = i_tok;
      if constexpr (kCluster) {
        part_o[(row0 + r) * 128 + d] = val;
        if (d == 0) part_lse[row0 + r] = lse;
        continue;
      }
      const int row = p.row0 + row0 + r, token = p.q_start + row / p.G, head = p.kvh * p.G + row % p.G;
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
  if (warp == kWarps + 1) tmem_dealloc(tmem, S::kAlloc);
  if constexpr (kCluster) merge_cluster<T, 128>(a, p, live, part_lse, part_o);
}

template <typename T, bool kInt8, int kR, bool kCluster>
int launch_tc(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, cudaStream_t s) {
  using S = Tc<kInt8, kR>;
  static_assert(S::kBytes * S::kCtas + 1024 * S::kCtas <= 233472, "shared memory of the CTAs of an SM");
  static_assert(kR * 128 * 4 <= S::kOffQ, "merge buffers must fit");
  static bool done[64] = {};
  return launch_splits(rows_tc_kernel<T, kInt8, kR, kCluster>, done, S::kThreads, S::kBytes, kCluster, a, tmK, tmV, s);
}

}  // namespace rows8
}  // namespace b200

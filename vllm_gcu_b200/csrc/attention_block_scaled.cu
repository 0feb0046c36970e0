// Attention of few query rows per request over a key / value cache held in 8 bits with a scale for each block of tokens
// and head (block_scaled.cuh): single tokens of running requests, drafts that are checked, short portions; bf16 and fp16
// queries, head dimensions 64 and 256 (128: attention_block_scaled_tc.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - m)
//
// over the keys j at or in front of the query that lie in its window or among the request's first tokens.
//
// Bound by memory: a key and its value are 2 D bytes for which every query row of the key head computes 4 D operations.
// Products run on mma.sync (16 rows at most a key head's queries fill of a tcgen05 tile's 128).  A CTA takes one request
// and key head, or a split of its keys; one warp walks the block table and issues a TMA copy per 16 tokens of a tile of
// 64, the others take 16 tokens each.  Codes become fp16, which holds both kinds exactly, with two conversions a word:
//   * the contraction over D takes the columns in any order, so that a lane reads 16 neighbouring codes of a key at
//     once: columns 32 t .. 32 t + 31 for lane t of four; queries are put into the same order;
//   * the columns of a value go to the accumulators in any order as well, lane g of eight holds 16 g .. 16 g + 15.  Pairs
//     of tokens for the contraction come from byte permutations of two tokens' words, where 16-bit values take a
//     transposing load.
// Both reads are free of bank conflicts in the 128-byte swizzle.
// Queries are scaled to a largest number in [1, 2) by a power of two, so that fp16 holds bf16 ones; what falls below its
// range is 2^-24 of the row's largest.  The scale of a block's keys is a factor of its scores.  That of its values
// joins the exponent: p'_j = p_j * scale, so that codes are all that the second product sees; the running maximum is that
// of the exponents with it, and the sum of p takes p' / scale.  The maximum is raised only when it is exceeded by 4 (log2), to
// which p' reaches 2^4, and fp16 holds 2^11 p': to 2^-11 of itself down to 2^-25 of the largest contribution and in steps
// of 2^-35 of it below, so that the many keys behind one that takes nearly all of a row (18 nats are 2^-26) keep their sum.
#include "block_scaled.cuh"

namespace b200 {
namespace rows8 {

using namespace block_scaled;

constexpr unsigned int kKernelId = 77;
constexpr int kChunk = 16;         // tokens of a TMA box, and of a warp at a time
constexpr int kTile = 64;          // tokens of a stage
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 4.0f;     // log2, by which a score may exceed the running maximum
constexpr float kUp = 11.0f;       // log2 of what a probability is held with
constexpr float kDown = 1.0f / 2048.0f;
// Scales of values (log2) below which a key's p' may vanish beside those of blocks of larger values while its p counts in the
// sum (a block of zeros has the least scale of all): there the sum takes p by itself.
constexpr float kSmallScale = -40.0f;

struct Args {
  const void* q;               // [T, Hq * D], row pitch ldq
  void* out;                   // [T, Hq * D], row pitch ldo
  float *tmp_out, *tmp_lse;    // splits without a cluster: [T, Hq, splits, D], [T, Hq, splits]; D 128: two parts a CTA
  int4* units;                 // D 128: what the CTA's share starts inside of
  const float *ks, *vs;        // [num_blocks, Hkv]
  const int *cu_q;             // [B + 1], null: one token per request
  const int *seq_lens, *block_tables;
  long long ldq, ldo;
  int B, Hq, Hkv, splits, row_blocks, max_blocks, block_size, num_blocks, window, first;
  float scale;
  unsigned int* status;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ld_peer(const float* p, uint32_t rank) {
  uint32_t addr;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Row r of a CTA's request and key head: token r / G of the step's tokens, query head r % G of the key head's.
struct Place {
  int b, kvh, G, rows, row0, q_start, pos0;
  int lo_pos, hi_pos;            // positions of the CTA's rows
  int firsts, lo_chunk, chunks;  // chunks of first tokens, first chunk of the window, chunks in all
};

template <int kRows>
__device__ __forceinline__ Place place_of(const Args& a) {
  Place p;
  // (the key heads of a request, whose rows lie side by side, run at the same time)
  p.b = blockIdx.y;
  p.kvh = blockIdx.x / a.row_blocks;
  p.G = a.Hq / a.Hkv;
  p.row0 = blockIdx.x % a.row_blocks * kRows;
  const int q_len = a.cu_q != nullptr ? a.cu_q[p.b + 1] - a.cu_q[p.b] : 1;
  p.q_start = a.cu_q != nullptr ? a.cu_q[p.b] : p.b;
  p.rows = q_len * p.G;
  const int len = min(a.seq_lens[p.b], a.max_blocks * a.block_size);
  p.pos0 = len - q_len;
  p.lo_pos = p.pos0 + p.row0 / p.G;
  p.hi_pos = p.pos0 + (min(p.row0 + kRows, p.rows) - 1) / p.G;
  const int lo = a.window > 0 ? max(0, p.lo_pos - a.window + 1) : 0;
  p.lo_chunk = lo / kChunk;
  p.firsts = a.window > 0 ? min(p.lo_chunk, (a.first + kChunk - 1) / kChunk) : 0;
  p.chunks = p.row0 < p.rows && p.hi_pos >= 0 ? p.firsts + p.hi_pos / kChunk + 1 - p.lo_chunk : 0;
  return p;
}

// The splits of a cluster, each with its rows' log2 sums and outputs in shared memory: every CTA adds up a share of the
// numbers.  All threads of the cluster call it.
template <typename T, int HD>
__device__ __forceinline__ void merge_cluster(const Args& a, const Place& p, int live, const float* part_lse,
                                              const float* part_o) {
  cluster_sync();
  uint32_t rank;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  for (int idx = static_cast<int>(rank) * blockDim.x + threadIdx.x; idx < live * HD; idx += a.splits * blockDim.x) {
    const int r = idx / HD, d = idx % HD;
    float pl[8], po[8], M = -INFINITY, o = 0.0f, sum = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      pl[s] = -INFINITY;
      if (s >= a.splits) continue;
      pl[s] = ld_peer(part_lse + r, s);
      po[s] = ld_peer(part_o + idx, s);
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) M = fmaxf(M, pl[s]);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (pl[s] == -INFINITY) continue;
      const float w = exp2f(pl[s] - M);
      sum += w;
      o = fmaf(w, po[s], o);
    }
    const int row = p.row0 + r, token = p.q_start + row / p.G, head = p.kvh * p.G + row % p.G;
    static_cast<T*>(a.out)[static_cast<long long>(token) * a.ldo + head * HD + d] =
        from_f32<T>(sum == 0.0f ? 0.0f : o / sum);
  }
  cluster_sync();                   // nobody leaves while another CTA may still read its numbers
}

// (`done`: per device, whether the kernel has its shared memory)
using Kernel = void (*)(CUtensorMap, CUtensorMap, Args);
inline int set_shared(Kernel kernel, bool (&done)[64], int smem) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || done[dev]) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return launch_code(e);
  done[dev] = true;
  return 0;
}
// Launch with the splits of a request and key head as a cluster, or as CTAs on their own.
inline int launch_splits(Kernel kernel, bool (&done)[64], int threads, int smem, bool cluster, const Args& a,
                         const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t s) {
  const int set = set_shared(kernel, done, smem);
  if (set != 0) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.Hkv * a.row_blocks, a.B, a.splits);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = a.splits;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return launch_code(cudaLaunchKernelEx(&cfg, kernel, tmK, tmV, a));
}

// Columns of a head's row that accumulator `nt` of lane column c (0 .. 7) holds
template <int HD>
__device__ __forceinline__ int column_of(int nt, int c) {
  constexpr int kPer = HD == 64 ? 8 : 16;            // neighbouring columns of a lane
  return nt / kPer * 128 + c * kPer + nt % kPer;
}

// kGroups: row groups of 16 (four warps each).  kCluster: the splits of a request and key head are a cluster and merge in
// shared memory.
template <typename T, bool kInt8, int HD, int kGroups, bool kCluster>
__global__ void __launch_bounds__(kGroups * 128 + 32)
    rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  constexpr int kRows = 16 * kGroups, kConsumers = 128 * kGroups;
  constexpr int kCols = HD < 128 ? HD : 128, kBoxes = HD / kCols, kBoxBytes = kChunk * kCols;
  constexpr int kStageBytes = 2 * kTile * HD;
  constexpr int kStages = HD == 256 ? 3 : 8;
  constexpr int kNT = HD / 8;
  extern __shared__ uint8_t smem_raw[];
  // (an offset, so that the compiler knows the accesses to be of shared memory)
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* empty_bar = full_bar + kStages;
  volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(empty_bar + kStages);
  // merges (in the stages' memory): maxima and sums of every warp, its outputs; a cluster's CTAs: sums, outputs
  float* sm_m = reinterpret_cast<float*>(smem);
  float* sm_l = sm_m + 4 * kRows;
  float* sm_o = sm_l + 4 * kRows;
  float* part_lse = sm_o + 4 * kRows * HD;
  float* part_o = part_lse + kRows;

  grid_release();
  grid_wait();
  const Place p = place_of<kRows>(a);
  if (p.row0 >= p.rows) return;                      // surplus rows (of a whole cluster)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.z;
  const int live = min(kRows, p.rows - p.row0);
  const int tiles_all = (p.chunks + 3) / 4;
  const int per_split = (tiles_all + a.splits - 1) / a.splits * 4;
  const int c0 = split * per_split, c1 = min(p.chunks, c0 + per_split);
  const int ntiles = c1 > c0 ? (c1 - c0 + 3) / 4 : 0;
  auto first_token = [&](int chunk) { return (chunk < p.firsts ? chunk : p.lo_chunk + chunk - p.firsts) * kChunk; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 4 * kGroups);
    }
    *abort_flag = 0u;
    mbar_fence_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  const int* bt = a.block_tables + static_cast<long long>(p.b) * a.max_blocks;

  if (warp == 4 * kGroups) {
    // ---------------- producer: lane = chunk of a tile and of eight tiles' block-table entries ----------------
    auto row_of = [&](int it) {                      // cache row of chunk `lane` behind tile it
      const int c = c0 + it * 4 + lane;
      if (c >= c1) return 0;
      const int tok = first_token(c);
      return bt[tok / a.block_size] * a.block_size + tok % a.block_size;
    };
    int stage = 0;
    uint32_t phase = 0;
    int row = row_of(0);
    bool ok = true;
    for (int it0 = 0; it0 < ntiles && ok; it0 += 8) {
      const int next = it0 + 8 < ntiles ? row_of(it0 + 8) : 0;
      for (int i = 0; i < 8 && it0 + i < ntiles; ++i) {
        ok = mbar_wait_warp(&empty_bar[stage], phase ^ 1u, a.status, kKernelId, 0x100u + stage, abort_flag);
        if (!ok) break;
        const int n = min(4, c1 - c0 - (it0 + i) * 4);
        if (lane == 0) mbar_expect_tx(&full_bar[stage], static_cast<uint32_t>(n) * 2u * kChunk * HD);
        __syncwarp();
        // lane = (chunk, keys or values, box of 128 columns)
        const int c = lane / (2 * kBoxes), kv = lane / kBoxes % 2, box = lane % kBoxes;
        const int y = __shfl_sync(0xffffffffu, row, (i * 4 + c) & 31);
        if (c < n)
          tma_load_2d(smem + stage * kStageBytes + kv * (kStageBytes / 2) + (c * kBoxes + box) * kBoxBytes,
                      kv == 0 ? &tmK : &tmV, &full_bar[stage], p.kvh * HD + box * kCols, y);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
      row = next;
    }
  } else {
    // ---------------- consumers ----------------
    const int g = lane >> 2, tig = lane & 3;
    const int part = warp & 3;                       // chunk of a tile
    const int group = kGroups == 1 ? 0 : warp >> 2;  // rows
    // scales of this warp's chunk of 32 tiles, one a lane
    // (a block that was never written has no scale: its values are zeros, its keys count all the same)
    auto scales_of = [&](int it, float& ks, float& vs) {
      const int c = c0 + (it + lane) * 4 + part;
      ks = 0.0f;
      vs = power_of_two(kLowExponent);
      if (c < c1) {
        const int block = bt[first_token(c) / a.block_size];
        if (block >= 0 && block < a.num_blocks) {
          const long long at = static_cast<long long>(block) * a.Hkv + p.kvh;
          ks = a.ks[at];
          vs = fmaxf(a.vs[at], vs);
        } else {
          report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(p.b));
        }
      }
    };
    float ks_now, vs_now, ks_next = 0.0f, vs_next = 0.0f;
    scales_of(0, ks_now, vs_now);

    // queries: [step][fragment]; step s of half h contracts columns 128 h + 32 tig + 4 s .. + 3 (HD 64: 16 tig + 4 s ..)
    constexpr int kSteps = HD / 16, kPerLane = HD == 64 ? 16 : 32, kStepsHalf = kPerLane / 4;
    uint32_t qf[kSteps][4];
    float row_scale[2];
    int pos[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = p.row0 + group * 16 + g + 8 * r;
      const bool valid = row < p.rows;
      const int token = row / p.G, head = p.kvh * p.G + row % p.G;
      pos[r] = p.pos0 + token;
      const T* src = static_cast<const T*>(a.q) + static_cast<long long>(p.q_start + token) * a.ldq + head * HD;
      uint4 raw4[HD / 32];
      const uint32_t* raw = reinterpret_cast<const uint32_t*>(raw4);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int col = i / (kPerLane / 8) * 128 + tig * kPerLane + i % (kPerLane / 8) * 8;
        raw4[i] = valid ? *reinterpret_cast<const uint4*>(src + col) : make_uint4(0u, 0u, 0u, 0u);
      }
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const T* e = reinterpret_cast<const T*>(&raw[i]);
        top = fmaxf(top, fmaxf(finite_size(to_f32<T>(e[0])), finite_size(to_f32<T>(e[1]))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e2 = max(-100, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
      const float down = power_of_two(-e2);
      row_scale[r] = power_of_two(e2) * a.scale * kLog2e;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const T* e = reinterpret_cast<const T*>(&raw[i]);
        qf[i >> 1][(i & 1) * 2 + r] = pack_half(to_f32<T>(e[0]) * down, to_f32<T>(e[1]) * down);
      }
    }
    float o_acc[kNT][4];
#pragma unroll
    for (int i = 0; i < kNT; ++i) o_acc[i][0] = o_acc[i][1] = o_acc[i][2] = o_acc[i][3] = 0.0f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    const uint32_t smem_base = smem_u32(smem);

    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int it = 0; it < ntiles; ++it) {
      if ((it & 31) == 0) {
        if (it > 0) { ks_now = ks_next; vs_now = vs_next; }
        if (it + 32 < ntiles) scales_of(it + 32, ks_next, vs_next);
      }
      const float ks = __shfl_sync(0xffffffffu, ks_now, it & 31);
      const float vs = __shfl_sync(0xffffffffu, vs_now, it & 31);
      ok = mbar_wait_warp(&full_bar[stage], phase, a.status, kKernelId, 0x200u + stage, abort_flag);
      if (!ok) break;
      const int chunk = c0 + it * 4 + part;
      if (chunk < c1) {
        const uint32_t sk = smem_base + stage * kStageBytes + part * kBoxes * kBoxBytes;
        const uint32_t sv = sk + kStageBytes / 2;
        const int tok0 = first_token(chunk);
        const float l2vs = __log2f(vs);
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
          const int row = j * 8 + g;
#pragma unroll
          for (int half = 0; half < kBoxes; ++half) {
            const uint32_t base = sk + half * kBoxBytes + row * kCols;
#pragma unroll
            for (int u = 0; u < kPerLane / 16; ++u) {
              const int c = HD == 64 ? tig ^ ((row >> 1) & 3) : (2 * tig + u) ^ g;
              const uint4 w = lds128(base + c * 16);
              const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t b0, b1;
                unpack4<kInt8>(words[i], b0, b1);
                mma16816(s[j], qf[half * kStepsHalf + u * 4 + i], b0, b1);
              }
            }
          }
        }
        // (the CTA's rows all see all keys of most chunks)
        const bool whole = tok0 + kChunk - 1 <= p.lo_pos &&
                           (a.window <= 0 || tok0 > p.hi_pos - a.window || tok0 + kChunk <= a.first);
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float f = row_scale[r] * ks;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaf(s[j][2 * r + e], f, l2vs);
              if (!whole) {
                const int tok = tok0 + j * 8 + 2 * tig + e;
                if (tok > pos[r] || (a.window > 0 && tok <= pos[r] - a.window && tok >= a.first)) x = -INFINITY;
              }
              s[j][2 * r + e] = x;
              top[r] = fmaxf(top[r], x);
            }
          }
        }
        if (__any_sync(0xffffffffu, top[0] > m_run[0] + kRaise || top[1] > m_run[1] + kRaise)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            const float m_new = fmaxf(m_run[r], top[r]);
            // (the sum, which may be as large as the inverse of a small scale, in two steps)
            const float root = m_run[r] == -INFINITY ? 0.0f : ex2(0.5f * (m_run[r] - m_new)), corr = root * root;
            m_run[r] = m_new;
            l_run[r] = l_run[r] * root * root;
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              o_acc[nt][2 * r] *= corr;
              o_acc[nt][2 * r + 1] *= corr;
            }
          }
        }
        const float unit = __fdividef(1.0f, vs);
        const bool small = l2vs < kSmallScale;       // (the same for the warp)
        if (small) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float m = m_run[r] == -INFINITY ? 0.0f : m_run[r] + l2vs;
            l_run[r] += (ex2(s[0][2 * r] - m) + ex2(s[0][2 * r + 1] - m)) + (ex2(s[1][2 * r] - m) + ex2(s[1][2 * r + 1] - m));
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float m = m_run[r] == -INFINITY ? 0.0f : m_run[r] - kUp;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v = ex2(s[j][2 * r + e] - m);
              s[j][2 * r + e] = v;
              sum += v;
            }
          }
          if (!small) l_run[r] = fmaf(sum * kDown, unit, l_run[r]);
        }
        uint32_t pf[4];
        pf[0] = pack_half(s[0][0], s[0][1]);
        pf[1] = pack_half(s[0][2], s[0][3]);
        pf[2] = pack_half(s[1][0], s[1][1]);
        pf[3] = pack_half(s[1][2], s[1][3]);
        // values of tokens 2 tig, 2 tig + 1 and those 8 behind them
        constexpr int kWords = HD == 64 ? 2 : 4;     // of a lane's columns in a box
#pragma unroll
        for (int half = 0; half < kBoxes; ++half) {
          uint32_t v[4][kWords];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int row = 2 * tig + (t & 1) + (t >> 1) * 8;
            if constexpr (HD == 64) {
              const uint2 w = lds64(sv + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
              v[t][0] = w.x; v[t][1] = w.y;
            } else {
              const uint4 w = lds128(sv + half * kBoxBytes + row * 128 + ((g ^ (row & 7)) << 4));
              v[t][0] = w.x; v[t][1] = w.y; v[t][2] = w.z; v[t][3] = w.w;
            }
          }
          if (!whole) {
            // what lies behind the last key, or in a gap that no row sees, may be anything
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int tok = tok0 + 2 * tig + (t & 1) + (t >> 1) * 8;
              if (tok > p.hi_pos || (a.window > 0 && tok <= p.lo_pos - a.window && tok >= a.first)) {
#pragma unroll
                for (int w = 0; w < kWords; ++w) v[t][w] = 0u;
              }
            }
          }
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
#pragma unroll
            for (int lohi = 0; lohi < 2; ++lohi) {
              const uint32_t sel = lohi == 0 ? 0x5140u : 0x7362u;
              uint32_t a0, a1, b0, b1;
              unpack4<kInt8>(__byte_perm(v[0][w], v[1][w], sel), a0, a1);
              unpack4<kInt8>(__byte_perm(v[2][w], v[3][w], sel), b0, b1);
              const int nt = half * 16 + w * 4 + lohi * 2;
              mma16816(o_acc[nt], pf, a0, b0);
              mma16816(o_acc[nt + 1], pf, a1, b1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[stage]);
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      if (!ok) l_run[r] = 0.0f;
    }
    // the four warps of a row group: the stages' memory is free once all consumers are here
    asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory");
    if (tig == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sm_m[part * kRows + group * 16 + g + 8 * r] = m_run[r];
        sm_l[part * kRows + group * 16 + g + 8 * r] = l_run[r];
      }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sm_o[(part * kRows + group * 16 + g + (e >> 1) * 8) * HD + column_of<HD>(nt, 2 * tig + (e & 1))] =
            o_acc[nt][e] * kDown;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory");
    for (int idx = threadIdx.x; idx < live * HD; idx += kConsumers) {
      const int r = idx / HD, d = idx % HD;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w * kRows + r]);
      float L = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = sm_m[w * kRows + r];
        // (a warp without keys has no sum; one whose scores are all NaN has no maximum)
        const float root = mw == -INFINITY ? (sm_l[w * kRows + r] == 0.0f ? 0.0f : 1.0f) : exp2f(0.5f * (mw - M));
        if (root == 0.0f) continue;
        L = fmaf(sm_l[w * kRows + r] * root, root, L);
        o = fmaf(sm_o[(w * kRows + r) * HD + d], root * root, o);
      }
      const float val = L == 0.0f ? 0.0f : o / L;
      const float lse = L == 0.0f ? -INFINITY : M + log2f(L);
      if constexpr (kCluster) {
        part_o[idx] = val;
        if (d == 0) part_lse[r] = lse;
        continue;
      }
      const int row = p.row0 + r, token = p.q_start + row / p.G, head = p.kvh * p.G + row % p.G;
      if (a.splits > 1) {
        const long long base = (static_cast<long long>(token) * a.Hq + head) * a.splits + split;
        a.tmp_out[base * HD + d] = val;
        if (d == 0) a.tmp_lse[base] = lse;
      } else {
        static_cast<T*>(a.out)[static_cast<long long>(token) * a.ldo + head * HD + d] = from_f32<T>(val);
      }
    }
  }
  if constexpr (kCluster) merge_cluster<T, HD>(a, p, live, part_lse, part_o);
}

// Splits that are no cluster: a warp a row.
template <typename T, int HD>
__global__ void __launch_bounds__(128) merge_rows_kernel(const Args a, int total) {
  grid_release_small();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= total) return;
  const int token = row / a.Hq, head = row % a.Hq;
  const long long base = static_cast<long long>(row) * a.splits;
  // (up to 32 splits: one a lane)
  const float mine = lane < a.splits ? a.tmp_lse[base + lane] : -INFINITY;
  const float M = warp_max(mine);
  const float weight = mine == -INFINITY ? 0.0f : exp2f(mine - M);
  const float sum = warp_sum(weight);
  float o[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) o[i] = 0.0f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float w = __shfl_sync(0xffffffffu, weight, s);
    if (w == 0.0f) continue;        // nothing seen: its output is zeros
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] = fmaf(w, a.tmp_out[(base + s) * HD + i * 32 + lane], o[i]);
  }
  T* out = static_cast<T*>(a.out) + static_cast<long long>(token) * a.ldo + head * HD;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) out[i * 32 + lane] = from_f32<T>(sum == 0.0f ? 0.0f : o[i] / sum);
}

// The arguments of a call come packed, as ops/cuda.py packs them.
struct Call {
  const void* q;
  void* out;
  const void *kc, *vc;
  const float *ks, *vs;
  const int *cu_q, *seq_lens, *block_tables;
  float *tmp_out, *tmp_lse;
  int* units;
  long long ldq, ldo, slot_bytes;
  float scale;
  int T, B, max_q, Hq, Hkv, D, splits, max_blocks, block_size, num_blocks, window, first, int8, dtype;
  int pad;
};

template <typename T, bool kInt8, int HD, int kGroups, bool kCluster>
int launch_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, cudaStream_t s) {
  constexpr int kStages = HD == 256 ? 3 : 8;
  constexpr int kMerge = (8 * 16 * kGroups + 4 * 16 * kGroups * HD + (kCluster ? 16 * kGroups * (HD + 1) : 0)) * 4;
  constexpr int kRing = kStages * 2 * kTile * HD;
  // (the merge's numbers lie where the stages were; the barriers behind the stages are not used any more by then)
  constexpr int kSmem = (kMerge > kRing ? kMerge : kRing) + 256 + 1024;
  static_assert(kSmem <= 232448, "exceeds the shared memory of one CTA");
  static bool done[64] = {};
  return launch_splits(rows_kernel<T, kInt8, HD, kGroups, kCluster>, done, kGroups * 128 + 32, kSmem, kCluster, a, tmK, tmV, s);
}

template <typename T, bool kInt8, int HD>
int launch_any(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, int T_rows, bool two, cudaStream_t s) {
  constexpr int kTwo = HD == 256 ? 1 : 2;           // (the accumulators of 256 columns leave no registers for eight warps)
  if (a.splits > 1 && a.splits <= 8)
    return two ? launch_rows<T, kInt8, HD, kTwo, true>(tmK, tmV, a, s) : launch_rows<T, kInt8, HD, 1, true>(tmK, tmV, a, s);
  const int e = two ? launch_rows<T, kInt8, HD, kTwo, false>(tmK, tmV, a, s)
                    : launch_rows<T, kInt8, HD, 1, false>(tmK, tmV, a, s);
  if (e != 0 || a.splits <= 1) return e;
  const int total = T_rows * a.Hq;
  return launch_overlapped(merge_rows_kernel<T, HD>, dim3((total + 3) / 4), dim3(128), 0, s, a, total);
}

}  // namespace rows8
}  // namespace b200

#include "attention_block_scaled_tc.cuh"

namespace b200 {
namespace rows8 {

// Rows that a CTA takes, of `all` of a request and key head.  (D 128: 28 rows in two blocks, which read the keys one behind
// the other and so the second time from L2, 53 us where a CTA of 32 took 60: 32 requests of 2450 keys, 4 heads.)
inline int rows_of_cta(int D, long long all) {
  if (D == 128) return all <= 4 ? 4 : all <= 8 ? 8 : 16;
  return D == 64 && all > 16 ? 32 : 16;
}

template <typename T, bool kInt8>
int launch_width(int D, const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, int T_rows, int rows, cudaStream_t s) {
  switch (D) {
    case 64: return launch_any<T, kInt8, 64>(tmK, tmV, a, T_rows, rows > 16, s);
    case 256: return launch_any<T, kInt8, 256>(tmK, tmV, a, T_rows, false, s);
    case 128:
      switch (rows) {
        case 4: return launch_tc<T, kInt8, 4>(tmK, tmV, a, a.splits, s);
        case 8: return launch_tc<T, kInt8, 8>(tmK, tmV, a, a.splits, s);
        case 16: return launch_tc<T, kInt8, 16>(tmK, tmV, a, a.splits, s);
      }
  }
  return -8;
}

}  // namespace rows8
}  // namespace b200

// Rows of a CTA and CTAs that run at the same time for head dimension 128 and so many query rows a request and key head:
// rows << 16 | CTAs.
B200_API int b200_block_scaled_slots(int rows, int int8) {
  using namespace b200::rows8;
  const int per = rows_of_cta(128, rows);
  return per << 16 | (int8 ? tc_slots<true>(per) : tc_slots<false>(per));
}

// Attention over blocks with scales.  dtype 0 bf16, 1 fp16; D 64, 128 or 256; max_q: most tokens of a request;
// block_size a multiple of 16.  D 64 and 256: up to 32 splits, more than 8 need tmp_out and tmp_lse (fp32 [T, Hq, splits, D]
// and [T, Hq, splits]).  D 128: `splits` CTAs, tmp_out [2 * splits, rows of a CTA, 128], tmp_lse [2 * splits, rows of a CTA],
// units int32 [splits, 4]; a multiple of Hkv.
B200_API int b200_block_scaled_rows(const void* call, void* stream) {
  using namespace b200;
  using namespace b200::rows8;
  const Call& k = *static_cast<const Call*>(call);
  if (k.B <= 0 || k.T <= 0 || k.Hkv <= 0) return 0;
  if (k.splits < 1 || k.Hq % k.Hkv != 0 || k.block_size % kChunk != 0) return -2;
  if (k.D == 128 ? k.tmp_out == nullptr || k.tmp_lse == nullptr || k.units == nullptr
                 : k.splits > 32 || (k.splits > 8 && (k.tmp_out == nullptr || k.tmp_lse == nullptr)))
    return -5;
  const int cols = k.D < 128 ? k.D : 128;
  const CUtensorMapSwizzle swizzle = k.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap tmK, tmV;
  const uint64_t rows = static_cast<uint64_t>(k.num_blocks) * k.block_size, width = static_cast<uint64_t>(k.Hkv) * k.D;
  int r = encode_tmap_2d(&tmK, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k.kc, rows, width, k.slot_bytes, kChunk, cols, swizzle);
  if (r == 0) r = encode_tmap_2d(&tmV, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k.vc, rows, width, k.slot_bytes, kChunk, cols, swizzle);
  if (r != 0) return r < 0 ? -6 : r;
  const int group = k.Hq / k.Hkv;
  const long long all = static_cast<long long>(k.max_q) * group;
  // rows of a CTA
  const int per = rows_of_cta(k.D, all);
  Args a;
  a.q = k.q; a.out = k.out; a.tmp_out = k.tmp_out; a.tmp_lse = k.tmp_lse;
  a.units = reinterpret_cast<int4*>(k.units); a.ks = k.ks; a.vs = k.vs; a.cu_q = k.cu_q;
  a.seq_lens = k.seq_lens; a.block_tables = k.block_tables; a.ldq = k.ldq; a.ldo = k.ldo; a.B = k.B; a.Hq = k.Hq;
  a.Hkv = k.Hkv; a.splits = k.splits; a.max_blocks = k.max_blocks; a.block_size = k.block_size;
  a.num_blocks = k.num_blocks; a.window = k.window; a.first = k.first; a.scale = k.scale;
  const long long row_blocks = (all + per - 1) / per;
  if (k.D != 128 && k.B > 65535) return -2;          // (a dimension of the grid)
  a.row_blocks = static_cast<int>(row_blocks);
  a.status = status_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k.dtype == 0)
    return k.int8 ? launch_width<__nv_bfloat16, true>(k.D, tmK, tmV, a, k.T, per, s)
                  : launch_width<__nv_bfloat16, false>(k.D, tmK, tmV, a, k.T, per, s);
  if (k.dtype == 1)
    return k.int8 ? launch_width<__half, true>(k.D, tmK, tmV, a, k.T, per, s)
                  : launch_width<__half, false>(k.D, tmK, tmV, a, k.T, per, s);
  return -8;
}

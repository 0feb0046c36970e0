// Attention of few query rows per request over a cache in 8 bits with scales, head dimension 128, on tcgen05 (included by
// attention_block_scaled.cu, whose Args, Place and Call it uses).
//
// The codes go to the tensor cores as they are, K and V tiles straight from TMA, and what they meet is brought to 8 bits
// without loss instead: a query and a probability are sums of 8-bit numbers ("parts") of falling weight, which are as
// many columns of the small operand.
//   S^T = K Q^T    M = 128 tokens (K-major rows of 128 bytes), N = 3 kR columns: part x query row
//   O^T = V^T P^T  M = 128 columns of the values (MN-major, as they lie), N = 4 kR columns, K = 128 tokens
// e4m3: parts of 4 bits each of a query, every one 16 times the rest of the one before, 12 bits together.  Probabilities are
// floating-point numbers there as well, since many keys may lie far below one that takes nearly all of a row: 2^11 times
// the probability as fp16, which is the sum of four e5m2 numbers (its upper byte, and 8 times the rest, three times) without
// rounding, so 11 bits down to 2^-25 of the largest and steps of 2^-35 of it below (parts in e4m3, which has one exponent
// bit less, would end at 2^-21, four of them at 2^-25; 16 nats are 2^-23).  int8: a query of 21 bits as digits to the base
// 128, a probability as a multiple of 2^-31, whose four bytes are unsigned digits to the base 256; the products' sums are
// exact.  What lies 16 nats below the largest is off by up to 2^-9 of itself there, 18 nats 2^-6: whole numbers have no
// exponent, and a fifth digit would leave room for two CTAs an SM in place of three.  A lane of the softmax warps owns a
// token: block scales are factors of its scores and of its probabilities, and there is no conversion of codes at all, which
// is what bounds a kernel that feeds 16-bit matrix instructions from 8-bit codes (attention_block_scaled.cu, head dimensions
// 64 and 256).
//
// Bound by memory: 256 requests of 1024 to 1279 keys, 8 key heads, 4 query rows each: 110 us and 613 MB, 85 per cent of the
// measured copy rate, tensor pipe 4.6 per cent, issue slots 35 per cent; 4 requests of 31007 to 120001 keys, 4 key heads, 7
// query rows: 63 us and 324 MB, 78 per cent.  What the rate does not explain is some 5 us of start (lengths, block table,
// first tile).  16 rows a CTA: by the softmax, 32 x 4 tokens of 7 query heads behind 1500 to 3391 keys 46 us, issue slots 53
// per cent, their warps most often waiting for scores from tensor memory.
//
// A CTA stays on its SM and takes an even share of the tiles of all requests for one key head, one behind the other (as
// many CTAs as run at the same time, or one per tile where there are fewer; those of a share's key heads are neighbours,
// since the heads' rows of a token lie side by side and memory is read in pieces of two: 613 against 904 MB where a CTA
// took the key heads one after the other): the shares depend on the lengths that the step holds, not on a bound that a
// captured graph was made with, no CTA has more than a tile more than another one, and a request's start (block table,
// queries) overlaps with the end of the one before.  Where a share begins or ends inside a request's keys, its part of the
// result goes to memory, and merge_units_kernel puts the parts together in their order.
//
// Warps: four for every eight rows queries and softmax, lane = token of a tile and at the end column of the output; then one
// for TMA, block tables and scales and one for tcgen05.mma and tensor memory.  K Q^T of a tile runs while the one before is
// at its softmax; keys and values have places of their own, given back when their product is done.
// The running maximum is raised when a score exceeds it by 4 (log2; int8, whose numbers end where they start higher, by 1: 32 x
// 4 tokens of 28 rows 50.5 us, with 4 48.5, single tokens the same), which all softmax warps vote on; then the sums in
// tensor memory are taken to registers, rescaled, and start anew (rare behind the first tiles, and the only form for sums
// of whole numbers).
#pragma once

namespace b200 {
namespace rows8 {

constexpr int kTcTile = 128;                 // tokens of a tile
constexpr int kTcBytes = kTcTile * 128;      // of its keys, or values
constexpr int kGroup = 4;                    // tiles whose block-table entries and scales a lane each of the TMA warp reads
constexpr int kGroups = 4;                   // places for their scales
constexpr int kMostTiles = 512;              // int8: whose sums of whole numbers one accumulator takes, 2^16 * 128 * 255 < 2^31

template <bool kInt8, int kR>
struct Tc {
  static constexpr int kParts = 4;                             // of a probability
  static constexpr int kNS = (3 * kR + 15) / 16 * 16;          // columns of scores
  static constexpr int kN = (kParts * kR + 15) / 16 * 16;      // and of outputs
  static constexpr int kRW = kR < 8 ? kR : 8;                  // rows of a softmax warp
  static constexpr int kWarps = 4 * kR / kRW;
  static constexpr int kThreads = kWarps * 32 + 64;
  // CTAs of an SM, which hide each other's starts and ends, and places for keys and values of each
  static constexpr int kCtas = kR == 4 ? 3 : 2;
  static constexpr int kStages = kR == 8 ? 3 : 2;
  static constexpr int kScores = 2;                            // score buffers
  static constexpr int kColumns = kScores * kNS + kN;
  static constexpr int kAlloc = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : 256;
  static_assert(kAlloc * kCtas <= 512, "tensor memory of an SM");
  static constexpr int kOffQ = 2 * kStages * kTcBytes;         // (keys, then values in front)
  static constexpr int kOffP = kOffQ + kNS * 128;
  // [kGroups][32] scales of keys, log2 and inverse of values' (below 0: a small one), flag
  static constexpr int kOffScale = kOffP + 2 * kN * 128;
  static constexpr int kOffBar = kOffScale + kGroups * 32 * 16;
  static constexpr int kOffWork = kOffBar + 384;               // [2]
  static constexpr int kOffRow = kOffWork + 128;               // (16-byte places) factor and position of every row; [2] token and head
  static constexpr int kOffMax = kOffRow + 6 * kR * 4;         // of four warps and every row; inverse sum and log2 of them
  static constexpr int kBytes = kOffMax + 6 * kR * 4 + 1024;
};

// A pair of fp16 numbers as four pairs of e5m2 parts, each in the upper bytes of the pair's halves: x = p0 + p1 / 8 + p2 / 64 +
// p3 / 512.  e5m2 is the upper byte of fp16: a part takes the three leading bits of what is left (or what reaches 2^-16).
// The rest of a number below 2^16 is below 2^13, so that 8 times it is one as well.
__device__ __forceinline__ void parts_e5m2(uint32_t x, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = x & 0xff00ff00u;
    if (i < 3) {
      const __half2 rest = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&p[i])),
                                   __floats2half2_rn(8.0f, 8.0f));
      x = *reinterpret_cast<const uint32_t*>(&rest);
    }
  }
}

template <bool kInt8>
__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kInt8) umma_i8(d, a, b, idesc, accumulate);
  else umma_f8(d, a, b, idesc, accumulate);
}

__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}

// Numbers of a lane's columns, parts put together: column part * kStride + row -> [row].
template <bool kInt8, int kRW, int kStride, int kParts, int kBits>
__device__ __forceinline__ void sum_parts(uint32_t tmem, float (&s)[kRW]) {
  // weights of the parts: of digits to the base 2^kBits (the last one's is 1), or 2^(-kBits p)
  auto weight = [](int p) {
    return kInt8 ? static_cast<float>(1 << kBits * (kParts - 1 - p)) : 1.0f / static_cast<float>(1 << kBits * p);
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
    uint32_t v[kParts][kRW];
    static_assert(kRW == 8, "loads of eight columns");
#pragma unroll
    for (int p = 0; p < kParts; ++p) tmem_ld_32x8(tmem + p * kStride, v[p]);
    tmem_ld_wait();
#pragma unroll
    for (int r = 0; r < kRW; ++r) {
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) {
        const float x = number(v[p][r]);
        s[r] = p == kParts - 1 ? x * last : fmaf(x, weight(p), s[r]);
      }
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

// Waits whose code is small: some thirty of them lie in the kernel, whose first pass is as long as its instructions take
// to arrive (mbar_wait's loop is unrolled: 150 KB in all, and 6 us until the first tile was done).
__device__ __noinline__ void wait_failed(unsigned int* status, unsigned int detail, volatile uint32_t* abort_flag) {
  report_status(status, kStatusMbarTimeout, kKernelId, detail);
  *abort_flag = 1u;
}
__device__ __noinline__ void bad_block(unsigned int* status, unsigned int detail) {
  report_status(status, kStatusBounds, kKernelId, detail);
}
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, unsigned int* status, unsigned int detail,
                                         volatile uint32_t* abort_flag) {
#pragma unroll 1
  for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
    if (mbar_test(bar, parity)) return true;
    if ((i & 1023u) == 1023u && *abort_flag != 0u) return false;
  }
  wait_failed(status, detail, abort_flag);
  return false;
}
// By all lanes of a warp: with one answer; or going on whatever it is.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, unsigned int* status, unsigned int detail,
                                          volatile uint32_t* abort_flag) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, status, detail, abort_flag)) != 0;
}
__device__ __forceinline__ void pass_warp(uint64_t* bar, uint32_t parity, unsigned int* status, unsigned int detail,
                                          volatile uint32_t* abort_flag) {
  wait_one(bar, parity, status, detail, abort_flag);
  __syncwarp();
}

// An even share of `total` tiles for each of n: where share j starts, and the share that tile x lies in.
struct Shares {
  int each, more;            // the first `more` shares have one tile more
  __device__ __forceinline__ Shares(int total, int n) : each(total / n), more(total - total / n * n) {}
  __device__ __forceinline__ int start(int j) const { return j * each + min(j, more); }
  __device__ __forceinline__ int of(int x) const {
    const int front = more * (each + 1);
    return x < front ? x / (each + 1) : more + (x - front) / each;
  }
};

// Sums, or largest, of kRW numbers over the lanes of a warp, in kRW - 1 and a few exchanges: this lane has that of row
// `row`.  (NaN is passed over by the largest.)
template <int kRW, bool kMax>
__device__ __forceinline__ float over_lanes(float (&v)[kRW], int lane, int& row) {
  auto join = [](float x, float y) { return kMax ? fmaxf(x, y) : x + y; };
  row = 0;
  int d = 16;
#pragma unroll
  for (int n = kRW / 2; n > 0; n >>= 1, d >>= 1) {
    const bool upper = (lane & d) != 0;
    row = upper ? row + n : row;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
      v[i] = join(keep, __shfl_xor_sync(0xffffffffu, give, d));
    }
  }
#pragma unroll
  for (; d > 0; d >>= 1) v[0] = join(v[0], __shfl_xor_sync(0xffffffffu, v[0], d));
  return v[0];
}

// What the TMA warp tells the others about the part of a request's and key head's tiles that the CTA takes.
struct Work {
  int q_start;             // -1: no more work
  int pos0, kvh, row0, rows;
  int lo_pos, hi_pos;      // positions of the CTA's rows
  int firsts, lo_chunk;
  int c0, c1;              // chunks
  int ntiles;
  int part;                // -1: all of the tiles; place of the part's numbers
  int pad[3];
};

// Tiles of rows kR * block .. of request b (1 where the rows see no key: they give zeros), 0 where there are no such rows.
template <int kR>
__device__ __noinline__ Place tc_place(const Args& a, int b, int block, int* tiles) {
  Place p;
  p.b = b;
  p.kvh = 0;
  p.G = a.Hq / a.Hkv;
  p.row0 = block * kR;
  p.q_start = a.cu_q != nullptr ? a.cu_q[b] : b;
  const int q_len = a.cu_q != nullptr ? a.cu_q[b + 1] - p.q_start : 1;
  p.rows = q_len * p.G;
  const int len = min(a.seq_lens[b], a.max_blocks * a.block_size);
  p.pos0 = len - q_len;
  p.lo_pos = p.pos0;
  p.hi_pos = len - 1;
  if (a.row_blocks > 1) {
    p.lo_pos += p.row0 / p.G;
    p.hi_pos = p.pos0 + (min(p.row0 + kR, p.rows) - 1) / p.G;
  }
  const int lo = a.window > 0 ? max(0, p.lo_pos - a.window + 1) : 0;
  p.lo_chunk = lo / kChunk;
  p.firsts = a.window > 0 ? min(p.lo_chunk, (a.first + kChunk - 1) / kChunk) : 0;
  p.chunks = p.hi_pos >= 0 ? p.firsts + p.hi_pos / kChunk + 1 - p.lo_chunk : 0;
  *tiles = p.row0 < p.rows ? max(1, (p.chunks + 7) / 8) : 0;
  return p;
}

template <typename T, bool kInt8, int kR>
__global__ void __launch_bounds__(Tc<kInt8, kR>::kThreads, Tc<kInt8, kR>::kCtas)
    rows_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ Args a) {
  using S = Tc<kInt8, kR>;
  constexpr int kN = S::kN, kNS = S::kNS, kStages = S::kStages, kParts = S::kParts, kWarps = S::kWarps, kRW = S::kRW, kScores = S::kScores;
  constexpr int kSoft = kWarps * 32;
  extern __shared__ uint8_t smem_raw[];
  // (an offset, so that the compiler knows the accesses to be of shared memory)
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
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
  uint64_t* w_full = o_done + 2;            // [2] a Work is there
  uint64_t* w_empty = w_full + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(w_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* adds = tmem_slot + 2;  // [2]: whether P V of the buffer's tile adds to what is there
  static_assert((4 * kStages + 9 + kGroups + 2 * kScores) * 8 + 16 <= 384, "barrier area");
  static_assert(sizeof(Work) == 64, "place of the works");
  float4* chunk_scale = reinterpret_cast<float4*>(smem + S::kOffScale);
  Work* works = reinterpret_cast<Work*>(smem + S::kOffWork);
  float* row_factor = reinterpret_cast<float*>(smem + S::kOffRow);
  int* row_pos = reinterpret_cast<int*>(row_factor + kR);
  int2* row_place = reinterpret_cast<int2*>(row_pos + kR);              // [2][kR]
  float* warp_top = reinterpret_cast<float*>(smem + S::kOffMax);        // [4][kR]
  float* row_inv = warp_top + 4 * kR;                                   // [kR]
  float* row_lse = row_inv + kR;                                        // [kR]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
      mbar_init(&w_full[b], 1);
      mbar_init(&w_empty[b], kWarps + 1);
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
  grid_wait();

  if (warp == kWarps) {
    // ---------------- work, TMA, block tables, scales ----------------
    // tiles of the requests (those of the first 512 stay where scales will lie)
    int* kept = reinterpret_cast<int*>(smem + S::kOffScale);
    static_assert(kGroups * 32 * 16 >= 512 * 4, "room for the requests' tiles");
    int total = 0;
#pragma unroll 1
    for (int b = lane; b < a.B; b += 32) {
      int n = 0;
#pragma unroll 1
      for (int rb = 0; rb < a.row_blocks; ++rb) {
        int t;
        tc_place<kR>(a, b, rb, &t);
        if (t == 0) break;
        n += t;
      }
      if (b < 512) kept[b] = n;
      total += n;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    // this CTA's key head and tiles; every share has one at least, those behind the last tile have none
    const int kvh = static_cast<int>(blockIdx.x) % a.Hkv, cta = static_cast<int>(blockIdx.x) / a.Hkv;
    const int ctas = min(total, static_cast<int>(gridDim.x) / a.Hkv);
    const Shares shares(total, max(ctas, 1));
    int at = cta < ctas ? shares.start(cta) : 0;
    const int end = cta < ctas ? shares.start(cta + 1) : 0;
    // request of the first one, and the tile in it
    int b = 0, in_b = 0;
    if (at < end) {
      int base = 0;
#pragma unroll 1
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        int n = 0;
        if (b0 + lane < a.B) {
          if (b0 + lane < 512) {
            n = kept[b0 + lane];
          } else {
#pragma unroll 1
            for (int rb = 0; rb < a.row_blocks; ++rb) {
              int t;
              tc_place<kR>(a, b0 + lane, rb, &t);
              n += t;
            }
          }
        }
        int inc = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += x;
        }
        const uint32_t vote = __ballot_sync(0xffffffffu, at < base + inc);
        if (vote != 0u) {
          const int src = __ffs(vote) - 1;
          b = b0 + src;
          in_b = at - base - __shfl_sync(0xffffffffu, inc - n, src);
          break;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    __syncwarp();
    int rb = 0, tile = 0, tiles = 0;                        // row block, its next tile, its tiles
    Place p = {};
    if (at < end) {
#pragma unroll 1
      for (;; ++rb) {
        p = tc_place<kR>(a, b, rb, &tiles);
        if (in_b < tiles) break;
        in_b -= tiles;
      }
      tile = in_b;
    }
    // a share that starts inside a request's tiles tells the shares that they lie in
    if (lane == 0)
      a.units[blockIdx.x] = tile == 0 ? make_int4(-1, 0, 0, 0)
                                      : make_int4(b, rb, shares.of(at - tile), shares.of(at - tile + tiles - 1));
    bool ok = true;
    int t = 0, groups = 0;                                  // tiles and groups of tiles so far
    for (int w = 0; ok; ++w) {
      Work k = {};
      k.q_start = -1;
      if (at < end) {
        const int n = min(tiles - tile, end - at);
        k.q_start = p.q_start;
        k.pos0 = p.pos0; k.kvh = kvh; k.row0 = p.row0; k.rows = p.rows; k.lo_pos = p.lo_pos; k.hi_pos = p.hi_pos;
        k.firsts = p.firsts; k.lo_chunk = p.lo_chunk;
        k.c0 = tile * 8;
        k.c1 = min(p.chunks, (tile + n) * 8);
        k.ntiles = n;
        // a part that starts inside a request's tiles is the CTA's first one
        k.part = n == tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (tile == 0 ? 1 : 0);
      }
      ok = wait_warp(&w_empty[w & 1], ((w >> 1) & 1) ^ 1, a.status, 0x3b0u, abort_flag);
      if (!ok) break;
      if (lane == 0) {
        works[w & 1] = k;
        mbar_arrive(&w_full[w & 1]);
      }
      __syncwarp();
      if (k.q_start < 0) break;

      // lane = (tile of a group of four, chunk of it); a group's blocks are read two groups ahead, its scales one
      const int* bt = a.block_tables + static_cast<long long>(p.b) * a.max_blocks;
      auto first_token = [&](int chunk) { return (chunk < p.firsts ? chunk : p.lo_chunk + chunk - p.firsts) * kChunk; };
      auto chunk_of = [&](int g) { return k.c0 + g * (8 * kGroup) + lane; };
      auto block_of = [&](int g) {
        const int c = chunk_of(g);
        return c < k.c1 ? bt[first_token(c) / a.block_size] : 0;
      };
      auto row_of = [&](int g, int block) { return block * a.block_size + first_token(chunk_of(g)) % a.block_size; };
      auto scales_of = [&](int g, int block) {
        float4 s = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
        if (chunk_of(g) >= k.c1) return s;
        if (block >= 0 && block < a.num_blocks) {
          const long long i = static_cast<long long>(block) * a.Hkv + kvh;
          s.x = a.ks[i];
          s.y = a.vs[i];
        } else {
          bad_block(a.status, static_cast<unsigned>(p.b));
        }
        return s;
      };
      auto publish = [&](int g, float4 s) {
        const int c = chunk_of(g), tok = first_token(c), slot = (groups + g) % kGroups;
        // (a block that was never written has no scale: its keys count all the same)
        const float vs = fmaxf(s.y, power_of_two(kLowExponent));
        s.y = __log2f(vs);
        s.z = __fdividef(1.0f, vs);
        if (s.y < kSmallScale) s.z = -s.z;
        // whether all rows see all of the chunk
        s.w = c < k.c1 && tok + kChunk - 1 <= p.lo_pos &&
                      (a.window <= 0 || tok > p.hi_pos - a.window || tok + kChunk <= a.first) ? 1.0f : 0.0f;
        chunk_scale[slot * 32 + lane] = s;
        __syncwarp();
        if (lane == 0) mbar_arrive(&c_full[slot]);
      };
      // rows of groups g and g + 1, block of g + 1, scales of g
      int row = 0, row_next = 0, block_next = 0;
      float4 scales = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      // copies of tiles: a tile's keys, then the values of the one before
#pragma unroll 1
      for (int it = -1; it < k.ntiles && ok; ++it) {
        const int g = it >= 0 ? it / kGroup : -1;
        const bool first = it < 0 || it % kGroup == 0;
        float4 scales_next = scales;
        int block_after = 0;
        if (first) {
          // (of group 0 before anything, its scales with the first tile)
          if (it < 0) {
            block_next = block_of(0);
            row_next = row_of(0, block_next);
          }
          block_after = block_of(g + 2);
          scales_next = scales_of(g + 1, block_next);
        }
#pragma unroll 1
        for (int values = 0; values < 2; ++values) {
          const int i = values ? it : it + 1;
          if (i < 0 || i >= k.ntiles) continue;
          const int st = (t + i) % kStages, n = max(0, min(8, k.c1 - k.c0 - i * 8));
          ok = wait_warp((values ? v_empty : k_empty) + st, (((t + i) / kStages) & 1) ^ 1, a.status, 0x300u + st, abort_flag);
          if (!ok) break;
          const int y = __shfl_sync(0xffffffffu, !values && i % kGroup == 0 ? row_next : row, i % kGroup * 8 + (lane & 7));
          uint64_t* bar = (values ? v_full : k_full) + st;
          if (lane == 0) mbar_expect_tx(bar, static_cast<uint32_t>(n) * kChunk * 128u);
          __syncwarp();
          if (lane < n)
            tma_load_2d(smem + ((values ? kStages : 0) + st) * kTcBytes + lane * (kChunk * 128), values ? &tmV : &tmK, bar,
                        kvh * 128, y);
        }
        // (behind the copies: nothing in front waits for this tile's softmax)
        if (it >= 0 && first) publish(g, scales);
        if (first) {
          scales = scales_next;
          block_next = block_after;
        }
        if (it < 0 || it % kGroup == kGroup - 1) {
          row = row_next;
          row_next = row_of(g + 2, block_next);
        }
      }
      t += k.ntiles;
      groups += (k.ntiles + kGroup - 1) / kGroup;
      // the next row block or request
      at += k.ntiles;
      tile = 0;
      if (at < end) {
        ++rb;
        tiles = 0;
        if (rb < a.row_blocks) p = tc_place<kR>(a, b, rb, &tiles);
        while (tiles == 0) {
          rb = 0;
          p = tc_place<kR>(a, ++b, 0, &tiles);
        }
      }
    }
    // The next kernel may start now, not before: its CTAs would take registers of this one's that are still to come, whose
    // tiles would then wait for a first CTA's end (steps one behind the other 160 us a pass, alone 120).
    grid_release();
  } else if (warp == kWarps + 1) {
    // ---------------- tcgen05.mma ----------------
    if (elect_one()) {
      constexpr uint32_t kA = kInt8 ? 1 : 0, kC = kInt8 ? 2 : 1;          // s8 or e4m3, s32 or f32
      constexpr uint32_t kIdescS = make_idesc(kTcTile, kNS, kA, kA, kC);
      constexpr uint32_t kIdescO = make_idesc(128, kN, kA, kInt8 ? 0 : 1, kC) | 1u << 15;    // B u8 or e5m2; A is MN-major
      const uint64_t q_desc = make_desc_k_sw128(smem_u32(smem + S::kOffQ));
      const uint64_t p_desc = make_desc_k_sw128(smem_u32(smem + S::kOffP));
      const uint64_t k_desc = make_desc_k_sw128(smem_u32(smem));
      const uint64_t v_desc = make_desc_mn_sw128(smem_u32(smem + kStages * kTcBytes), kTcBytes);
      auto pv = [&](int j) -> bool {
        const int b = j & 1, st = j % kStages;
        if (!wait_one(&v_full[st], (j / kStages) & 1, a.status, 0x310u + st, abort_flag) ||
            !wait_one(&p_full[b], (j >> 1) & 1, a.status, 0x320u + b, abort_flag))
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
      bool ok = true;
      int t = 0;
      for (int w = 0; ok; ++w) {
        ok = wait_one(&w_full[w & 1], (w >> 1) & 1, a.status, 0x3c0u, abort_flag);
        if (!ok) break;
        const bool over = static_cast<volatile Work*>(works)[w & 1].q_start < 0;
        const int ntiles = static_cast<volatile Work*>(works)[w & 1].ntiles;
        mbar_arrive(&w_empty[w & 1]);
        if (over) break;
        ok = wait_one(q_full, w & 1, a.status, 0x322u, abort_flag);
        for (int it = 0; ok && it < ntiles; ++it, ++t) {
          const int b = t % kScores, st = t % kStages;
          ok = wait_one(&k_full[st], (t / kStages) & 1, a.status, 0x330u + st, abort_flag) &&
               wait_one(&s_free[b], ((t / kScores) & 1) ^ 1, a.status, 0x340u + b, abort_flag);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma8<kInt8>(tmem + b * kNS, k_desc + static_cast<uint32_t>((st * kTcBytes + ks * 32) >> 4),
                        q_desc + static_cast<uint32_t>(ks * 2), kIdescS, ks > 0 ? 1u : 0u);
          umma_commit(&s_full[b]);
          umma_commit(&k_empty[st]);
          if (it > 0) ok = pv(t - 1);
        }
        if (ok) ok = pv(t - 1);
      }
    }
    __syncwarp();
  } else {
    const int row0 = kWarps == 4 ? 0 : warp / 4 * kRW;       // first row of the warp
    static_assert(kWarps == 4 || kRW % 8 == 0, "places of rows in groups of eight");
    const int i_tok = (warp & 3) * 32 + lane, c16 = i_tok >> 4;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + row0;
    const int G = a.Hq / a.Hkv;
    const float inv_g = 1.0f / static_cast<float>(G);
    // ---------------- queries of a part ----------------
    auto queries = [&](const Work& k, int w) {
      const int live = min(kR, k.rows - k.row0);
      constexpr int kMine = kR / kWarps;
      uint2 raws[kMine];
      // row / G: half a G off the next whole number, and 2^-23 of itself wrong
      auto token_of = [&](int r) { return __float2int_rd((static_cast<float>(k.row0 + r) + 0.5f) * inv_g); };
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r = warp + i * kWarps, token = token_of(r), head = k.kvh * G + k.row0 + r - token * G;
        raws[i] = make_uint2(0u, 0u);
        if (r < live)
          raws[i] = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) +
                                                    static_cast<long long>(k.q_start + token) * a.ldq + head * 128 + lane * 4);
      }
#pragma unroll
      for (int mine = 0; mine < kMine; ++mine) {
        const int r = warp + mine * kWarps;
        const int token = token_of(r), head = k.kvh * G + k.row0 + r - token * G;
        const T* e = reinterpret_cast<const T*>(&raws[mine]);
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
        uint32_t part[3] = {0u, 0u, 0u};
        float unit;                         // of the parts, times 2^e2
        if constexpr (kInt8) {
          // |x| 2^-e2 < 2 as whole numbers of 21 bits, digits -64 .. 63 (the first one up to 64)
          unit = 1.0f / 524287.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int f = __float2int_rn(fminf(fmaxf(x[i] * down, -2.0f), 2.0f) * 524287.0f);
            const int d2 = ((f + 64) & 127) - 64, f1 = (f - d2) >> 7;
            const int d1 = ((f1 + 64) & 127) - 64, d0 = (f1 - d1) >> 7;
            part[0] |= static_cast<uint32_t>(d0 & 255) << (8 * i);
            part[1] |= static_cast<uint32_t>(d1 & 255) << (8 * i);
            part[2] |= static_cast<uint32_t>(d2 & 255) << (8 * i);
          }
        } else {
          // the largest in [128, 256), in 32 bits: a bf16 number's 8 bits are two parts, an fp16 number's 11 are three
          unit = 1.0f / 128.0f;
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            float y0 = x[i] * down * 128.0f, y1 = x[i + 1] * down * 128.0f;
#pragma unroll
            for (int j = 0; j < 3; ++j) {
              const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
              part[j] |= c << (8 * i);
              y0 = (y0 - e4m3_to_f32(static_cast<uint8_t>(c & 255u))) * 16.0f;
              y1 = (y1 - e4m3_to_f32(static_cast<uint8_t>(c >> 8))) * 16.0f;
            }
          }
        }
        number = __all_sync(0xffffffffu, number);
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const int n = j * kR + r;
          *reinterpret_cast<uint32_t*>(smem + S::kOffQ + (n >> 3) * 1024 + (n & 7) * 128 +
                                       (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4) = part[j];
        }
        if (lane == 0) {
          // (a row that holds infinities or NaN gives NaN, as its products do)
          row_factor[r] = number ? power_of_two(e2) * unit * a.scale * kLog2e : __int_as_float(0x7fffffff);
          // (rows of no query see what the last one sees)
          row_pos[r] = min(k.pos0 + token, k.hi_pos);
          row_place[(w & 1) * kR + r] = make_int2(k.q_start + token, head);
        }
      }
      fence_async_smem();
      sync_softmax<kSoft>();                // (factors and positions)
      if (lane == 0) mbar_arrive(q_full);
    };
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

    // ---------------- softmax: lane = token of the tile ----------------
    // (2 or 16 of them fill the parts)
    constexpr float kUnit = kInt8 ? 2147483648.0f : 2048.0f, kMost = kInt8 ? 1.0f : kRaise;
    int t = 0, groups = 0;
    Work k = {};
    float m[kRW], l[kRW], o[kRW];
#pragma unroll
    for (int r = 0; r < kRW; ++r) m[r] = l[r] = o[r] = 0.0f;
    // what P V of earlier tiles left in tensor memory
    auto drain = [&]() {
      float v[kRW];
      sum_parts<kInt8, kRW, kR, kParts, kInt8 ? 8 : 3>(lane_addr + kScores * kNS, v);
#pragma unroll
      for (int r = 0; r < kRW; ++r) o[r] = fmaf(v[r], 1.0f / kUnit, o[r]);
    };
#pragma unroll 1
    for (int w = 0;; ++w) {
      // the next part's queries first: its scores are computed while the results of the one before are written
      pass_warp(&w_full[w & 1], (w >> 1) & 1, a.status, 0x3d0u, abort_flag);
      Work next = works[w & 1];
      // (a wait that ran out ends all warps at the same place: what they would read is not there; and all warps are done
      // with the rows' factors)
      if (any_of<kSoft>(*abort_flag != 0u)) next.q_start = -1;
      if (next.q_start >= 0) queries(next, w);
      if (w > 0) {
        pass_warp(&o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, a.status, 0x380u, abort_flag);
        tc_fence_after();
        drain();
        tc_fence_before();
        // sums over the tokens
        int mine;
        const float sum = over_lanes<kRW, false>(l, lane, mine);
        warp_top[(warp & 3) * kR + row0 + mine] = *abort_flag != 0u ? 0.0f : sum;
        if (k.part >= 0 && (warp & 3) == 0 && lane == 0) {
#pragma unroll
          for (int r = 0; r < kRW; ++r) row_lse[row0 + r] = m[r];
        }
        sync_softmax<kSoft>();
        const int i = threadIdx.x;
        if (i < kR) {
          const float L = (warp_top[i] + warp_top[kR + i]) + (warp_top[2 * kR + i] + warp_top[3 * kR + i]);
          row_inv[i] = L == 0.0f ? 0.0f : __fdividef(1.0f, L);
          if (k.part >= 0 && k.row0 + i < k.rows)
            a.tmp_lse[static_cast<long long>(k.part) * kR + i] = L == 0.0f ? -INFINITY : row_lse[i] + log2f(L);
        }
        sync_softmax<kSoft>();
        const int live = min(kR, k.rows - k.row0), d = i_tok;
        const int2* place = row_place + ((w - 1) & 1) * kR + row0;
#pragma unroll
        for (int r = 0; r < kRW; ++r) {
          const float inv = row_inv[row0 + r];
          const float val = inv == 0.0f ? 0.0f : o[r] * inv;
          if (row0 + r >= live) {
          } else if (k.part >= 0) {
            a.tmp_out[(static_cast<long long>(k.part) * kR + row0 + r) * 128 + d] = val;
          } else {
            static_cast<T*>(a.out)[place[r].x * a.ldo + place[r].y * 128 + d] = from_f32<T>(val);
          }
          m[r] = l[r] = o[r] = 0.0f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_empty[(w - 1) & 1]);
      }
      if (next.q_start < 0) break;
      k = next;
      uint32_t unseen = (1u << kRW) - 1u;   // rows of which no key was seen (the same in all warps): their maximum is 0
      bool drained = true;                  // nothing of these maxima in tensor memory
#pragma unroll 1
      for (int it = 0; it < k.ntiles; ++it, ++t) {
        const int g = groups + it / kGroup;
        if (it % kGroup == 0)
          pass_warp(&c_full[g % kGroups], (g / kGroups) & 1, a.status, 0x390u, abort_flag);
        const float4 scale = chunk_scale[g % kGroups * 32 + it % kGroup * 8 + c16];
        const bool all_whole = __all_sync(0xffffffffu, scale.w != 0.0f);
        // (the scores of a tile are there when P V two tiles ago is done, which was issued before: its probabilities may
        // be overwritten)
        pass_warp(&s_full[t % kScores], (t / kScores) & 1, a.status, 0x350u, abort_flag);
        tc_fence_after();
        float x[kRW];
        sum_parts<kInt8, kRW, kR, 3, kInt8 ? 7 : 4>(lane_addr + t % kScores * kNS, x);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t % kScores]);
        // exponents, relative to the running maximum
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < kRW; r += 4) {
          const float4 f = *reinterpret_cast<const float4*>(row_factor + row0 + r);
          x[r] = fmaf(x[r], f.x * scale.x, scale.y - m[r]);
          x[r + 1] = fmaf(x[r + 1], f.y * scale.x, scale.y - m[r + 1]);
          x[r + 2] = fmaf(x[r + 2], f.z * scale.x, scale.y - m[r + 2]);
          x[r + 3] = fmaf(x[r + 3], f.w * scale.x, scale.y - m[r + 3]);
        }
        bool lost = false;                  // no row sees the token
        if (!all_whole) {
          const int c = k.c0 + it * 8 + c16;
          const bool there = c < k.c1;
          const int tok = (c < k.firsts ? c : k.lo_chunk + c - k.firsts) * kChunk + (i_tok & 15);
          lost = !there || tok > k.hi_pos || (a.window > 0 && tok <= k.lo_pos - a.window && tok >= a.first);
#pragma unroll
          for (int r = 0; r < kRW; ++r) {
            const int pos = row_pos[row0 + r];
            if (!there || tok > pos || (a.window > 0 && tok <= pos - a.window && tok >= a.first)) x[r] = -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < kRW; ++r) top = fmaxf(top, x[r]);
        if (unseen != 0u) {
#pragma unroll
          for (int r = 0; r < kRW; ++r)
            if ((unseen >> r & 1u) != 0u && x[r] > -INFINITY) top = INFINITY;
        }
        if (any_of<kSoft>(top > kMost || (kInt8 && it % kMostTiles == kMostTiles - 1))) {
          // new maxima of all rows; the sums in tensor memory belong to the old ones
          float tops[kRW];
#pragma unroll
          for (int r = 0; r < kRW; ++r) tops[r] = x[r];
          int mine;
          const float largest = over_lanes<kRW, true>(tops, lane, mine);
          warp_top[(warp & 3) * kR + row0 + mine] = largest == largest ? largest : -INFINITY;
          sync_softmax<kSoft>();
          if (!drained) {
            pass_warp(&o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, a.status, 0x360u, abort_flag);
            tc_fence_after();
            drain();
            tc_fence_before();
          }
          // lane r has row r's
          const float* w4 = warp_top + row0 + lane % kRW;
          float up = fmaxf(fmaxf(w4[0], w4[kR]), fmaxf(w4[2 * kR], w4[3 * kR]));         // over the old maximum
          const bool seen = (unseen >> lane % kRW & 1u) == 0u;
          const bool moves = seen ? up > 0.0f : up > -INFINITY;
          if (!moves) up = 0.0f;
          // (the sum, which may be as large as the inverse of a small scale, in two steps)
          const float root = moves ? (seen ? ex2(-0.5f * up) : 0.0f) : 1.0f;
          unseen &= ~__ballot_sync(0xffffffffu, moves && lane < kRW);
#pragma unroll
          for (int r = 0; r < kRW; ++r) {
            const float d = __shfl_sync(0xffffffffu, up, r), c = __shfl_sync(0xffffffffu, root, r);
            m[r] += d;
            l[r] = l[r] * c * c;
            o[r] *= c * c;
            x[r] -= d;
          }
          sync_softmax<kSoft>();            // (warp_top is free again)
          drained = true;
        }
        if (__any_sync(0xffffffffu, scale.z < 0.0f)) {
          const float up = scale.z < 0.0f ? __log2f(-scale.z) : -INFINITY;
#pragma unroll
          for (int r = 0; r < kRW; ++r) l[r] += ex2(x[r] + up);
        }
        const float unit = fmaxf(scale.z, 0.0f);            // of a probability in the sum
        if (threadIdx.x == 0) adds[t & 1] = drained ? 0u : 1u;
        drained = false;
        // (rows of a warp start at a multiple of 8 columns: their places in a group of eight are constants; bits 4 .. 6 of an
        // address are those of c16 alone)
        const uint32_t sp = smem_u32(smem) + S::kOffP + (t & 1) * kN * 128 + row0 * 128 + (i_tok & 15) + (c16 << 4);
        auto put = [&](int n, uint32_t byte) {
          asm volatile("st.shared.u8 [%0], %1;" ::"r"((sp ^ ((n & 7) << 4)) + (n >> 3) * 1024 + (n & 7) * 128), "r"(byte)
                       : "memory");
        };
#pragma unroll
        for (int r = 0; r < kRW; r += 2) {
          float v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            v[e] = ex2(x[r + e]);           // up to 16 (int8: 2)
            l[r + e] = fmaf(v[e], unit, l[r + e]);
          }
          if constexpr (kInt8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t f = __float2uint_rn(v[e] * kUnit);       // (2 of them: the largest number)
#pragma unroll
              for (int j = 0; j < kParts; ++j) put(j * kR + r + e, f >> 8 * (kParts - 1 - j));
            }
          } else {
            uint32_t q[4];
            parts_e5m2(pack_half(v[0] * kUnit, v[1] * kUnit), q);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              put(j * kR + r, q[j] >> 8);
              put(j * kR + r + 1, q[j] >> 24);
            }
          }
        }
        if (lost && warp < 4) {
          // what lies behind the last key, in a gap that no row sees, or was not loaded may be anything
          wait_one(&v_full[t % kStages], (t / kStages) & 1, a.status, 0x3a0u, abort_flag);
          uint4* v = reinterpret_cast<uint4*>(smem + (kStages + t % kStages) * kTcBytes + i_tok * 128);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j ^ (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t & 1]);
      }
      groups += (k.ntiles + kGroup - 1) / kGroup;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarps + 1) tmem_dealloc(tmem, S::kAlloc);
}

// Parts of a request's rows that several CTAs computed: by the CTAs whose numbers are those of all parts but the first, a
// row at a time for each warp, or, of many parts, for each CTA, whose warps take every fourth part.  Bound by latency (unit,
// sums, outputs one behind the other): with all rows merged by the second part's CTA one request of 32000 keys, a key head and 8
// query rows, 250 parts, took 91 us in all, now 24; 256 requests of two or three parts each 128 and 121 (the merge itself 6 us with a cold L2).
constexpr int kFewParts = 8;                 // that a warp takes by itself
template <typename T>
__global__ void __launch_bounds__(128) merge_units_kernel(const Args a, int kR) {
  grid_release_small();
  grid_wait();
  __shared__ float4 sm_o[4][32];
  __shared__ float sm_sum[4];
  const int4 unit = a.units[blockIdx.x];           // request, row block, first and last share
  if (unit.x < 0) return;
  const int kvh = static_cast<int>(blockIdx.x) % a.Hkv, share = static_cast<int>(blockIdx.x) / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_start = a.cu_q != nullptr ? a.cu_q[unit.x] : unit.x;
  const int G = a.Hq / a.Hkv, rows = (a.cu_q != nullptr ? a.cu_q[unit.x + 1] - q_start : 1) * G;
  const int parts = unit.w - unit.z + 1, number = share - unit.z - 1, n = min(kR, rows - unit.y * kR);
  const bool many = parts > kFewParts;
  // the first share's part is its last one, the others' is their first
  auto place = [&](int i) { return static_cast<long long>(2 * ((unit.z + i) * a.Hkv + kvh) + (i == 0 ? 1 : 0)) * kR; };
  const int on = many ? parts - 1 : 4 * (parts - 1), every = many ? 4 : 1;
  for (int r = many ? number : 4 * number + warp; r < n; r += on) {
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, a.tmp_lse[place(i) + r]);
    M = warp_max(M);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    for (int i0 = many ? warp : 0; i0 < parts; i0 += 32 * every) {
      const int i_lane = i0 + lane * every;
      const float lse = i_lane < parts ? a.tmp_lse[place(i_lane) + r] : -INFINITY;
      const float mine = lse == -INFINITY ? 0.0f : exp2f(lse - M);
      const int count = min(32, (parts - i0 + every - 1) / every);
#pragma unroll 8
      for (int j = 0; j < count; ++j) {
        const float w = __shfl_sync(0xffffffffu, mine, j);
        const float4 x = reinterpret_cast<const float4*>(a.tmp_out + (place(i0 + j * every) + r) * 128)[lane];
        sum += w;
        o.x = fmaf(w, x.x, o.x);
        o.y = fmaf(w, x.y, o.y);
        o.z = fmaf(w, x.z, o.z);
        o.w = fmaf(w, x.w, o.w);
      }
    }
    if (many) {                                    // (the same for all threads)
      sm_o[warp][lane] = o;
      if (lane == 0) sm_sum[warp] = sum;
      __syncthreads();
      o = sm_o[0][lane];
      sum = sm_sum[0];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 x = sm_o[w][lane];
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        sum += sm_sum[w];
      }
      __syncthreads();
      if (warp != 0) continue;
    }
    const int row = unit.y * kR + r, token = q_start + row / G, head = kvh * G + row % G;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out) + static_cast<long long>(token) * a.ldo + head * 128 + lane * 4;
    T v[4] = {from_f32<T>(o.x * inv), from_f32<T>(o.y * inv), from_f32<T>(o.z * inv), from_f32<T>(o.w * inv)};
    *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
  }
}

// CTAs that run at the same time.
template <bool kInt8>
int tc_slots(int rows) {
  const int ctas = rows == 4 ? Tc<kInt8, 4>::kCtas : rows == 8 ? Tc<kInt8, 8>::kCtas : Tc<kInt8, 16>::kCtas;
  return ctas * sm_count();
}

template <typename T, bool kInt8, int kR>
int launch_tc(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, int ctas, cudaStream_t s) {
  using S = Tc<kInt8, kR>;
  static_assert(S::kBytes * S::kCtas + 1024 * S::kCtas <= 233472, "shared memory of the CTAs of an SM");
  static bool done[64] = {};
  const int e = set_shared(rows_tc_kernel<T, kInt8, kR>, done, S::kBytes);
  if (e != 0) return e;
  const int r = launch_overlapped(rows_tc_kernel<T, kInt8, kR>, dim3(ctas), dim3(S::kThreads), S::kBytes, s, tmK, tmV, a);
  if (r != 0) return r;
  return launch_overlapped(merge_units_kernel<T>, dim3(ctas), dim3(128), 0, s, a, kR);
}

}  // namespace rows8
}  // namespace b200

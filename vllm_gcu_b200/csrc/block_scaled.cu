// A key / value cache held in 8 bits with a scale for each block of tokens and head: writes of a step's keys and
// values, expansion of a request's blocks for prefill attention, copies and forks of blocks.
//
// Cache: codes [blocks, block_size, heads, D], scales fp32 [blocks, heads], both for keys and for values.
#include "block_scaled.cuh"

namespace b200 {
namespace block_scaled {

constexpr unsigned int kKernelId = 76;

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------
struct WriteArgs {
  const void *k, *v;           // [T, H * D], row pitches ldk, ldv (elements)
  uint8_t *kc, *vc;
  float *ks, *vs;
  const long long* slots;      // [T], -1: none
  long long ldk, ldv, slot_bytes, num_slots;
  int T, H, block_size, window;
  unsigned int* status;
};

// Eight neighbours of a row as floats.
template <typename T, bool kWide>
struct Eight {
  uint4 raw[sizeof(T) == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(raw) / 16); ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T* e = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(raw)[i >> 1];
      return __uint_as_float((i & 1) != 0 ? w & 0xffff0000u : w << 16);
    } else {
      return to_f32<T>(reinterpret_cast<const T*>(raw)[i]);
    }
  }
  // largest magnitude of the finite ones
  __device__ __forceinline__ float top() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_size(at(i)));
    return m;
  }
  // largest bits behind the sign, of 16-bit types in pairs: the order of magnitudes, infinities and NaN above all others
  __device__ __forceinline__ uint32_t top_bits(uint32_t m) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(raw) / 4); ++i) {
      if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7fffffffu);
      else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    return m;
  }
};

// Bound by the chain slot - scale - row - maximum - code: 8192 rows of 8 heads of 128, 50 MB, 14.4 us, 53 per cent of the
// measured copy rate and 56 per cent of the issue slots.
// A warp takes one head of the keys or the values for every run of rows that starts in its window of `window` rows: a run
// is the rows of one block, which follow each other in rising order of slots, and lies in no other warp.  The rows of a run
// stay in registers (the first kHold pieces of a lane; blocks of 32 tokens and more are read again from L1) between their
// maximum and their codes.  A run that does not start its block raises the block's scale where a number does not fit, and
// rounds the codes in front of it anew.
template <typename T, bool kInt8, bool kWide, int D>
__global__ void __launch_bounds__(256, sizeof(T) == 4 || D == 256 ? 2 : 4) write_kernel(const WriteArgs a) {
  grid_release_small();
  grid_wait();
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;      // lanes of a row, rows of a pass
  constexpr int kHold = D == 256 || sizeof(T) == 4 ? 8 : 16 / kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int plane = blockIdx.y * 8 + warp;
  if (plane >= 2 * a.H) return;
  const bool values = plane >= a.H;
  const int h = values ? plane - a.H : plane;
  const int row0 = blockIdx.x * a.window;
  auto page_of = [&](int t) -> int {                      // -1: the row goes nowhere
    if (t < 0 || t >= a.T) return -1;
    const long long s = a.slots[t];
    if (s >= a.num_slots) {
      report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(t));
      return -1;
    }
    return s < 0 ? -1 : static_cast<int>(s / a.block_size);
  };
  const int mine = lane < a.window ? page_of(row0 + lane) : -1;
  int before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) before = page_of(row0 - 1);
  uint32_t starts = __ballot_sync(0xffffffffu, mine >= 0 && mine != before);
  const T* src = static_cast<const T*>(values ? a.v : a.k) + h * D + (lane % kLanes) * 8;
  const long long ld = values ? a.ldv : a.ldk;
  uint8_t* cache = (values ? a.vc : a.kc) + h * D + (lane % kLanes) * 8;
  float* scales = values ? a.vs : a.ks;
  while (starts != 0u) {
    const int first = row0 + __ffs(starts) - 1;
    starts &= starts - 1u;
    const int page = __shfl_sync(0xffffffffu, mine, first - row0);
    const long long slot0 = static_cast<long long>(page) * a.block_size;
    const long long at = static_cast<long long>(page) * a.H + h;
    float old = scales[at];
    // places of the run's first 32 rows, a lane each, and its rows
    int place = -1, n = 0;
#pragma unroll 1
    for (int base = 0; base < a.block_size; base += 32) {
      const int t = first + base + lane;
      const long long in = t < a.T && base + lane < a.block_size ? a.slots[t] - slot0 : -1;
      const bool ours = in >= 0 && in < a.block_size;
      if (base == 0) place = static_cast<int>(in);
      const uint32_t out = __ballot_sync(0xffffffffu, !ours);
      n = base + (out != 0u ? __ffs(out) - 1 : 32);
      if (out != 0u) break;
    }
    const int off = __shfl_sync(0xffffffffu, place, 0);
    if (off == 0) old = 0.0f;
    Eight<T, kWide> held[kHold];
    uint32_t bits = 0u;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int r = i * kRows + lane / kLanes;
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(held[0].raw) / 16); ++j) held[i].raw[j] = make_uint4(0u, 0u, 0u, 0u);
      if (r < n) held[i].load(src + (first + r) * ld);
    }
#pragma unroll
    for (int i = 0; i < kHold; ++i) bits = held[i].top_bits(bits);
#pragma unroll 1
    for (int r = kHold * kRows + lane / kLanes; r < n; r += kRows) {
      Eight<T, kWide> e;
      e.load(src + (first + r) * ld);
      bits = e.top_bits(bits);
    }
    if constexpr (sizeof(T) == 2) bits = max(bits & 0xffffu, bits >> 16);
    bits = __reduce_max_sync(0xffffffffu, bits);
    // (rare: numbers that are none, which do not count, and sizes above what the largest scale holds)
    constexpr uint32_t kInfinity = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    float top;
    if (bits < kInfinity) {
      if constexpr (sizeof(T) == 4) {
        top = __uint_as_float(bits);
      } else {
        const uint16_t half = static_cast<uint16_t>(bits);
        top = to_f32<T>(*reinterpret_cast<const T*>(&half));
      }
    } else {
      top = 0.0f;
      for (int r = lane / kLanes; r < n; r += kRows) {
        Eight<T, kWide> e;
        e.load(src + (first + r) * ld);
        top = fmaxf(top, e.top());
      }
      top = warp_max(top);
    }
    const float need = power_of_two(scale_exponent<kInt8>(top));
    const bool plain = bits < kInfinity && need < power_of_two(kHighExponent);
    const float scale = old > need ? old : need;          // (old may be anything where nothing was written yet)
    const float unit = 1.0f / scale;
    if (off > 0 && scale != old) {
      const float ratio = old > 0.0f ? old * unit : 0.0f;
      for (int r = lane / kLanes; r < off; r += kRows) {
        uint2* p = reinterpret_cast<uint2*>(cache + (slot0 + r) * a.slot_bytes);
        uint2 w = *p;
        uint32_t* half = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t lo, hi;
          unpack4<kInt8>(half[i], lo, hi);
          const float2 x = half_pair(lo), y = half_pair(hi);
          half[i] = codes4<kInt8>(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
        }
        *p = w;
      }
    }
    uint8_t* block = cache + slot0 * a.slot_bytes;
    const int pitch = static_cast<int>(a.slot_bytes);
    auto store = [&](const Eight<T, kWide>& e, int r, int in) {
      if (in < 0) in = static_cast<int>(a.slots[first + r] - slot0);
      uint2 w;
      if (plain) {
        const float lo[4] = {e.at(0), e.at(1), e.at(2), e.at(3)}, hi[4] = {e.at(4), e.at(5), e.at(6), e.at(7)};
        w.x = codes4_of<kInt8>(lo, unit);
        w.y = codes4_of<kInt8>(hi, unit);
      } else {
        w.x = codes4<kInt8>(e.at(0) * unit, e.at(1) * unit, e.at(2) * unit, e.at(3) * unit);
        w.y = codes4<kInt8>(e.at(4) * unit, e.at(5) * unit, e.at(6) * unit, e.at(7) * unit);
      }
      *reinterpret_cast<uint2*>(block + static_cast<long long>(in) * pitch) = w;
    };
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int r = i * kRows + lane / kLanes;
      const int in = __shfl_sync(0xffffffffu, place, r);
      if (r < n) store(held[i], r, in);
    }
#pragma unroll 1
    for (int r = kHold * kRows + lane / kLanes; r < n; r += kRows) {
      Eight<T, kWide> e;
      e.load(src + (first + r) * ld);
      store(e, r, -1);
    }
    if (lane == 0 && (scale != old || off == 0)) scales[at] = scale;
  }
}

template <typename T, bool kInt8, bool kWide>
int launch_write(const WriteArgs& a, int D, cudaStream_t s) {
  const dim3 grid((a.T + a.window - 1) / a.window, (2 * a.H + 7) / 8);
  switch (D) {
    case 64: return launch_overlapped(write_kernel<T, kInt8, kWide, 64>, grid, dim3(256), 0, s, a);
    case 128: return launch_overlapped(write_kernel<T, kInt8, kWide, 128>, grid, dim3(256), 0, s, a);
    case 256: return launch_overlapped(write_kernel<T, kInt8, kWide, 256>, grid, dim3(256), 0, s, a);
  }
  return -8;
}

// ---------------------------------------------------------------------------
// expansion
// ---------------------------------------------------------------------------
// Keys of a request that a step's tokens can see, in 16 bits, in tiles of 128 that follow each other request after
// request: the tiles with the first tokens that stay visible, then those from the first token's window on.
struct ExpandArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  void *ko, *vo;               // [tiles * 128, H * D]
  int* table;                  // [B, table_width]: expanded tile of each tile of keys
  const int *cu_q, *seq_lens, *block_tables;
  long long slot_bytes;
  int B, H, D, block_size, max_blocks, num_blocks, table_width, tiles, window, first;
  unsigned int* status;
};

constexpr int kTileKeys = 128;

// (fp16: what lies beyond 65504 is held there, also the largest number of the type, whose code stands for 65536, and
// what lies below 2^-25 is lost; every code times its scale is a bf16 number.)
// 16 keys of a tile and their values by a CTA: a thread 8 codes at a time (one store of 16 bytes beside its neighbours'),
// four of the keys and four of the values under way.  Bound by memory: one byte read and two written, and most of what is
// written stays in L2 for the attention behind it (12.3 us for 7048 keys of 8 heads of 128, 43 MB: 53 per cent of
// the measured copy rate, with the latency of lengths, table entry, code and store one behind the other).
template <typename T, bool kInt8>
__global__ void __launch_bounds__(256) expand_kernel(const ExpandArgs a) {
  grid_release_small();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int tile = blockIdx.x / (kTileKeys / 16), part = blockIdx.x % (kTileKeys / 16);
  int base = 0, seq = -1, key_tile = 0, keys = 0, gap = 0;     // keys from `first` to `gap`: in no token's window
  for (int b0 = 0; b0 < a.B && seq < 0; b0 += 32) {
    const int b = b0 + lane;
    int count = 0, lo = 0, firsts = 0, len = 0, hidden = 0;
    if (b < a.B) {
      len = min(min(a.seq_lens[b], a.max_blocks * a.block_size), a.table_width * kTileKeys);
      const int q = a.cu_q[b + 1] - a.cu_q[b];
      if (q > 0 && len > 0) {
        if (a.window > 0) {
          hidden = max(0, len - q - a.window + 1);
          lo = hidden / kTileKeys;
          firsts = min(lo, (a.first + kTileKeys - 1) / kTileKeys);
        }
        count = firsts + (len + kTileKeys - 1) / kTileKeys - lo;
      }
    }
    int inc = count;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += n;
    }
    const int start = base + inc - count;
    const uint32_t vote = __ballot_sync(0xffffffffu, tile >= start && tile < start + count);
    if (vote != 0u) {
      const int from = __ffs(vote) - 1;
      const int j = tile - __shfl_sync(0xffffffffu, start, from), nf = __shfl_sync(0xffffffffu, firsts, from);
      const int l = __shfl_sync(0xffffffffu, lo, from);
      seq = b0 + from;
      key_tile = j < nf ? j : l + j - nf;
      keys = __shfl_sync(0xffffffffu, len, from);
      gap = __shfl_sync(0xffffffffu, hidden, from);
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (seq < 0) return;
  if (threadIdx.x == 0 && part == 0) a.table[static_cast<long long>(seq) * a.table_width + key_tile] = tile;
  const int key0 = key_tile * kTileKeys + part * 16;
  const int vecs = a.H * a.D / 8;                         // of a key
  const long long to = (static_cast<long long>(tile) * kTileKeys + part * 16) * a.H * a.D;
  int block = 0;
  if (key0 < keys) {
    block = a.block_tables[static_cast<long long>(seq) * a.max_blocks + key0 / a.block_size];
    if (block < 0 || block >= a.num_blocks) {
      if (threadIdx.x == 0) report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(block));
      keys = 0;
    }
  }
  const long long from = (static_cast<long long>(block) * a.block_size + key0 % a.block_size) * a.slot_bytes;
  const uint8_t* cache[2] = {a.kc + from, a.vc + from};
  const float* scales[2] = {a.ks + static_cast<long long>(block) * a.H, a.vs + static_cast<long long>(block) * a.H};
  T* out[2] = {static_cast<T*>(a.ko) + to, static_cast<T*>(a.vo) + to};
  constexpr int kAtOnce = 4;
  const int rows_on = 256 / vecs, on = 256 - rows_on * vecs, head_shift = a.D == 64 ? 3 : a.D == 128 ? 4 : 5;
  int r = static_cast<int>(threadIdx.x) / vecs, c = static_cast<int>(threadIdx.x) - r * vecs;
  for (int i0 = threadIdx.x; i0 < 16 * vecs; i0 += 256 * kAtOnce) {
    uint2 w[2][kAtOnce];
    float scale[2][kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      // what no token sees is zeros
      const bool seen = r < 16 && key0 + r < keys && (key0 + r >= gap || key0 + r < a.first);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        w[kv][u] = make_uint2(0u, 0u);
        scale[kv][u] = 0.0f;
        if (seen) {
          w[kv][u] = *reinterpret_cast<const uint2*>(cache[kv] + r * a.slot_bytes + c * 8);
          scale[kv][u] = scales[kv][c >> head_shift];
        }
      }
      r += rows_on;
      c += on;
      if (c >= vecs) {
        c -= vecs;
        ++r;
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * 256;
      if (i >= 16 * vecs) break;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t in[2] = {w[kv][u].x, w[kv][u].y};
        float f[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t lo, hi;
          unpack4<kInt8>(in[j], lo, hi);
          const float2 x = half_pair(lo), y = half_pair(hi);
          f[4 * j] = x.x * scale[kv][u]; f[4 * j + 1] = x.y * scale[kv][u];
          f[4 * j + 2] = y.x * scale[kv][u]; f[4 * j + 3] = y.y * scale[kv][u];
        }
        if constexpr (std::is_same<T, __half>::value) {
          // (an infinity times a probability of 0 would reach the rows that do not see the key)
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = fminf(fmaxf(f[j], -65504.0f), 65504.0f);
        }
        vec8_store<T>(out[kv] + static_cast<long long>(i) * 8, f);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// copies and forks
// ---------------------------------------------------------------------------
// A cache's tensors, as ops/cuda.py lays them out in device memory: where the blocks of a tensor start, the bytes of a
// block, and those of a token (0: a block's entry has no tokens, like a scale's).
struct Plane {
  unsigned long long base;
  long long block_bytes, token_bytes;
};

struct CopyArgs {
  const Plane* planes;
  int num_planes, num_blocks;
  // copies
  const long long* pairs;      // [n, 2], -1 in either place: none
  // forks
  const int *tables, *seq_lens, *parents, *fresh;
  int* out;
  int n, width, num_requests, block_size, pieces;
  unsigned int* status;
};

// blockIdx.x: pair or answer, .y: tensors (strided), .z: piece of a block.  16 bytes a thread at a time, four under way;
// entries of scales by words, others by bytes.
__device__ __forceinline__ void copy_bytes(const uint8_t* src, uint8_t* dst, long long bytes, int t, int step) {
  const unsigned long long low = reinterpret_cast<unsigned long long>(src) | reinterpret_cast<unsigned long long>(dst) |
                                 static_cast<unsigned long long>(bytes);
  if ((low & 15u) == 0u) {
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(dst);
    const long long n = bytes / 16;
    constexpr int kAtOnce = 4;
    for (long long i = t; i < n; i += static_cast<long long>(step) * kAtOnce) {
      uint4 v[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i + static_cast<long long>(u) * step < n) v[u] = s[i + static_cast<long long>(u) * step];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i + static_cast<long long>(u) * step < n) d[i + static_cast<long long>(u) * step] = v[u];
    }
  } else if ((low & 3u) == 0u) {
    for (long long i = t; i < bytes / 4; i += step)
      reinterpret_cast<uint32_t*>(dst)[i] = reinterpret_cast<const uint32_t*>(src)[i];
  } else {
    for (long long i = t; i < bytes; i += step) dst[i] = src[i];
  }
}

// Bound by latency (table or pair, then plane, then bytes): 64 forks of 32 layers, 24 MB read and written, 8.8 us in a
// captured graph, 2.4 times the bytes' time.  kWarp: a warp a tensor (blocks of up to 16 KB; with a CTA for each piece 12.3
// us).
template <bool kFork, bool kWarp>
__global__ void __launch_bounds__(128) copy_kernel(const CopyArgs a) {
  grid_release_small();
  grid_wait();
  const int n = blockIdx.x;
  long long src = -1, dst = -1;
  int used = a.block_size;
  if constexpr (kFork) {
    const int parent = a.parents[n];
    const bool known = parent >= 0 && parent < a.num_requests;
    const int* row = a.tables + static_cast<long long>(known ? parent : 0) * a.width;
    const int len = known ? a.seq_lens[parent] : 0, fresh = known ? a.fresh[n] : -1;
    const int last = len >= 0 ? len / a.block_size : a.width;   // block that takes the next token
    if (blockIdx.y == 0 && blockIdx.z == 0)
      for (int i = threadIdx.x; i < a.width; i += blockDim.x)
        a.out[static_cast<long long>(n) * a.width + i] = !known ? 0 : i == last && fresh >= 0 ? fresh : row[i];
    used = len >= 0 ? len % a.block_size : 0;
    if (fresh < 0 || used == 0 || last >= a.width) return;
    src = row[last];
    dst = fresh;
  } else {
    src = a.pairs[2 * n];
    dst = a.pairs[2 * n + 1];
    if (src < 0 || dst < 0) return;
  }
  if (src < 0 || dst < 0 || src >= a.num_blocks || dst >= a.num_blocks) {
    if (threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
      report_status(a.status, kStatusBounds, kKernelId, static_cast<unsigned>(n));
    return;
  }
  if (src == dst) return;
  const int first = kWarp ? blockIdx.y * 4 + (threadIdx.x >> 5) : blockIdx.y, on = kWarp ? 4 * gridDim.y : gridDim.y;
  const int t = kWarp ? threadIdx.x & 31 : blockIdx.z * 128 + threadIdx.x, step = kWarp ? 32 : a.pieces * 128;
  for (int p = first; p < a.num_planes; p += on) {
    const Plane plane = a.planes[p];
    const long long bytes = kFork && plane.token_bytes > 0 ? used * plane.token_bytes : plane.block_bytes;
    uint8_t* base = reinterpret_cast<uint8_t*>(plane.base);
    copy_bytes(base + src * plane.block_bytes, base + dst * plane.block_bytes, bytes, t, step);
  }
}

// The arguments of a call come packed, as ops/cuda.py packs them.
struct WriteCall {
  const void *k, *v;
  void *kc, *vc;
  float *ks, *vs;
  const long long* slots;
  long long ldk, ldv, slot_bytes, num_slots;
  int T, H, D, block_size, wide, int8, dtype, pad;
};
struct ExpandCall {
  const void *kc, *vc;
  const float *ks, *vs;
  void *ko, *vo;
  int* table;
  const int *cu_q, *seq_lens, *block_tables;
  long long slot_bytes;
  int B, H, D, block_size, max_blocks, num_blocks, table_width, tiles, window, first, int8, dtype;
};
struct CopyCall {
  const Plane* planes;
  const long long* pairs;
  const int *tables, *seq_lens, *parents, *fresh;
  int* out;
  long long largest;
  int num_planes, num_blocks, n, width, num_requests, block_size;
};

template <typename T>
int write_any(const WriteArgs& a, const WriteCall& k, cudaStream_t s) {
  if (k.int8) return k.wide ? launch_write<T, true, true>(a, k.D, s) : launch_write<T, true, false>(a, k.D, s);
  return k.wide ? launch_write<T, false, true>(a, k.D, s) : launch_write<T, false, false>(a, k.D, s);
}

}  // namespace block_scaled
}  // namespace b200

// Keys and values of a step into their blocks.  dtype: 0 bf16, 1 fp16, 2 fp32; D 64, 128 or 256; wide: rows may be
// read 16 bytes at a time.
B200_API int b200_block_scaled_cache(const void* call, void* stream) {
  using namespace b200;
  using namespace b200::block_scaled;
  const WriteCall& k = *static_cast<const WriteCall*>(call);
  if (k.T <= 0 || k.H <= 0) return 0;
  if (k.block_size <= 0 || k.num_slots > 0x7fffffffll * k.block_size) return -2;
  WriteArgs a;
  a.k = k.k; a.v = k.v; a.kc = static_cast<uint8_t*>(k.kc); a.vc = static_cast<uint8_t*>(k.vc);
  a.ks = k.ks; a.vs = k.vs; a.slots = k.slots; a.ldk = k.ldk; a.ldv = k.ldv; a.slot_bytes = k.slot_bytes;
  a.num_slots = k.num_slots; a.T = k.T; a.H = k.H; a.block_size = k.block_size;
  a.window = k.T <= 512 ? 1 : 16;
  a.status = status_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (k.dtype) {
    case 0: return write_any<__nv_bfloat16>(a, k, s);
    case 1: return write_any<__half>(a, k, s);
    case 2: return write_any<float>(a, k, s);
  }
  return -8;
}

// Blocks of a step's requests in 16 bits (dtype 0 bf16, 1 fp16), `tiles` tiles of 128 keys.
B200_API int b200_block_scaled_expand(const void* call, void* stream) {
  using namespace b200;
  using namespace b200::block_scaled;
  const ExpandCall& k = *static_cast<const ExpandCall*>(call);
  if (k.B <= 0 || k.tiles <= 0) return 0;
  ExpandArgs a;
  a.kc = static_cast<const uint8_t*>(k.kc); a.vc = static_cast<const uint8_t*>(k.vc); a.ks = k.ks; a.vs = k.vs;
  a.ko = k.ko; a.vo = k.vo; a.table = k.table; a.cu_q = k.cu_q; a.seq_lens = k.seq_lens;
  a.block_tables = k.block_tables; a.slot_bytes = k.slot_bytes; a.B = k.B; a.H = k.H; a.D = k.D;
  a.block_size = k.block_size; a.max_blocks = k.max_blocks; a.num_blocks = k.num_blocks;
  a.table_width = k.table_width; a.tiles = k.tiles; a.window = k.window; a.first = k.first;
  a.status = status_ptr();
  const dim3 grid(k.tiles * (kTileKeys / 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k.dtype == 0)
    return k.int8 ? launch_overlapped(expand_kernel<__nv_bfloat16, true>, grid, dim3(256), 0, s, a)
                  : launch_overlapped(expand_kernel<__nv_bfloat16, false>, grid, dim3(256), 0, s, a);
  if (k.dtype == 1)
    return k.int8 ? launch_overlapped(expand_kernel<__half, true>, grid, dim3(256), 0, s, a)
                  : launch_overlapped(expand_kernel<__half, false>, grid, dim3(256), 0, s, a);
  return -8;
}

// Copies of blocks (`pairs`) or forks of requests (`parents`) in all tensors of a cache.  `largest`: bytes of the largest
// block of a tensor.
B200_API int b200_cache_pages(const void* call, void* stream) {
  using namespace b200;
  using namespace b200::block_scaled;
  const CopyCall& k = *static_cast<const CopyCall*>(call);
  if (k.n <= 0) return 0;
  CopyArgs a;
  a.planes = k.planes; a.num_planes = k.num_planes; a.num_blocks = k.num_blocks; a.pairs = k.pairs; a.tables = k.tables;
  a.seq_lens = k.seq_lens; a.parents = k.parents; a.fresh = k.fresh; a.out = k.out; a.n = k.n; a.width = k.width;
  a.num_requests = k.num_requests; a.block_size = k.block_size;
  a.status = status_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.pieces = 1;
  if (k.largest <= 16384) {
    const int rows = (k.num_planes + 3) / 4;
    const dim3 grid(k.n, rows < 1 ? 1 : rows < 65535 ? rows : 65535);
    if (k.pairs != nullptr) return launch_overlapped(copy_kernel<false, true>, grid, dim3(128), 0, s, a);
    return launch_overlapped(copy_kernel<true, true>, grid, dim3(128), 0, s, a);
  }
  // 8 KB a CTA: four 16-byte pieces of a thread
  const long long pieces = (k.largest + 8191) / 8192;
  a.pieces = static_cast<int>(pieces > 64 ? 64 : pieces);
  const dim3 grid(k.n, k.num_planes < 1 ? 1 : k.num_planes < 65535 ? k.num_planes : 65535, a.pieces);
  if (k.pairs != nullptr) return launch_overlapped(copy_kernel<false, false>, grid, dim3(128), 0, s, a);
  return launch_overlapped(copy_kernel<true, false>, grid, dim3(128), 0, s, a);
}

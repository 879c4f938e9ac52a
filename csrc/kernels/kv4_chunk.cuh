// SPDX-License-Identifier: Apache-2.0
// Attention of long runs of query rows over the 4-bit cache on the 5th
// generation tensor cores (included by kv4_attention.cu).
//
// A unit is 256 query rows (two tiles of 128) of one request and key head
// against a range of keys, 128 at a time.  Roles of a block of 13 warps:
//   warps 0-3, 4-7  softmax of the first and the second row tile, a thread a
//                   row: scores from TMEM, weights back to TMEM as f16, in
//                   the place of the scores;
//   warps 8-11      a thread a token: codes from global memory (one tile
//                   ahead in registers) to f16 in shared memory, in the
//                   128-byte swizzle that the products read;
//   warp 12         one thread issues S = Q K^T (N = 128) and O += P V (P
//                   from TMEM, V with channels as the major axis).
// While one row tile's products run the other's softmax does; the order PV0,
// S0, PV1, S1 of the products keeps both busy, and the products of one thread
// run in order, so the scores of the next keys may take the place of weights
// just used.
//
// Numbers.  f16 holds 11 bits, and a scale of 8 bits times a code between -8
// and 7 (3 bits and a power of two) is exact in them.  So a key is the product
// s (code - 8), and what is the same for 64 channels, o = mid + s / 2, meets
// the sum of the query's channels in a few more columns of the product (both
// as two f16 each, 22 bits): scores are exact to f32.  Values are o + s (code -
// 8), o and the sum rounded to f16.  f16's range is handled by powers of two:
// a query row is scaled to 2^8, 32 neighbouring tokens (what a warp turns, and
// what a softmax thread takes at once) share a power of two for keys and one
// for values, which the softmax puts into its scale and into the weights.
// Scores, maxima, sums and outputs are f32.  The maximum is followed loosely (by 8 in
// the base-2 logarithm), so the output is rescaled rarely.
#pragma once

#include "kernels/kv4.cuh"
#include "kernels/sm100.cuh"

namespace vccl {
namespace model {
namespace {

constexpr int kChunkRows = 256;
constexpr int kChunkKeys = 128;
constexpr int kChunkThreads = 13 * 32;
constexpr int kNoExponent = -1000;  // of 32 tokens that are all zero

// 32 lanes x 32 bit, 32 consecutive columns per thread.
__device__ __forceinline__ void tmemLoad32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmemStore16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmemStore32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// f16 products: A in shared memory or TMEM, B in shared memory.  Shared-memory
// descriptors come as two words, of which only the first moves from product to
// product: the one thread that issues them would else be what the tensor cores
// wait for (a product of 128 x 128 x 16 takes 64 clocks; with 64-bit
// descriptors made anew the thread took 100 for each).
template <bool ACCUMULATE>
__device__ __forceinline__ void mmaF16(uint32_t d, uint32_t aLo, uint32_t aHi, uint32_t bLo, uint32_t bHi, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %6, 0;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n}\n" ::"r"(d),
      "r"(aLo), "r"(aHi), "r"(bLo), "r"(bHi), "r"(idesc), "n"(ACCUMULATE ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mmaF16Tmem(uint32_t d, uint32_t a, uint32_t bLo, uint32_t bHi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(bLo), "r"(bHi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D f32, A = B = f16, A K-major; transposeB: B's major axis is N.
__host__ __device__ constexpr uint32_t idescF16(int m, int n, bool transposeB) {
  return (1u << 4) | (transposeB ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// N-major operand in the 128-byte swizzle: atoms of 64 channels by 8 tokens;
// the next 64 channels 16 KiB on (leading), the next 8 tokens 1 KiB on (stride).
__device__ __forceinline__ uint64_t smemDescMn(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
  d |= static_cast<uint64_t>(16384u >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// K-major operand of 16 columns without a swizzle: 8 rows of 16 bytes to an
// atom, the next 8 columns 128 bytes on, the next 8 rows 256.
__device__ __forceinline__ uint64_t smemDescPlain(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
  d |= static_cast<uint64_t>(128u >> 4) << 16;
  d |= static_cast<uint64_t>(256u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  return d;
}
constexpr int kPlainBytes = 128 * 32;
__device__ __forceinline__ int plainRow(int row) { return (row >> 3) * 256 + (row & 7) * 16; }

__device__ __forceinline__ float halfOf(float x) { return __half2float(__float2half_rn(x)); }

// Columns that carry sum over groups of a_g b_g, a and b as two f16 each; a
// side's columns of one group are (high, high, low) or (high, low, high).
template <int G, bool QUERY>
__device__ __forceinline__ void storeSums(uint8_t* block, int row, const float (&x)[G]) {
  float y[8] = {};
#pragma unroll
  for (int g = 0; g < G; g++) {
    const float high = halfOf(x[g]), low = x[g] - high;
    y[3 * g] = high;
    y[3 * g + 1] = QUERY ? high : low;
    y[3 * g + 2] = QUERY ? low : high;
  }
  *reinterpret_cast<uint4*>(block + plainRow(row)) = pack8<__half>(y);
  *reinterpret_cast<uint4*>(block + plainRow(row) + 128) = make_uint4(0, 0, 0, 0);
}

// 2^e for -126 <= e <= 127 (clamped).
__device__ __forceinline__ float powerOfTwo(int e) {
  return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23);
}
__device__ __forceinline__ int exponentOf(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127; }

template <int G>
struct ChunkSmem {
  static constexpr int kBlock = 16384;  // 128 rows of 64 f16
  static constexpr int kQ = 0;          // [2 row tiles][G]
  static constexpr int kK = kQ + 2 * G * kBlock;  // [2 stages][G]
  static constexpr int kV = kK + 2 * G * kBlock;
  static constexpr int kQSums = kV + 2 * G * kBlock;  // [2 row tiles]
  static constexpr int kKSums = kQSums + 2 * kPlainBytes;  // [2 stages]
  static constexpr int kInfo = kKSums + 2 * kPlainBytes;
  static constexpr int kStarts = kInfo + 1024;  // units before each request
};

// What the tokens of a tile bring, by 32 (one warp's).
struct ChunkInfo {
  uint32_t valid[4];   // the token is there
  uint32_t bad[2][4];  // its values of a group are not finite (and zero in the product)
  int keyExp[4], valueExp[4];
};

struct ChunkControl {
  ChunkInfo info[4];
  uint64_t qFull[2], kFull[2], kEmpty[2], vFull[2], vEmpty[2], sFull[2], pFull[2], oFull[2], drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(ChunkControl) <= 1024, "the control block's place");

struct ChunkUnit {
  Request r;
  int b, head, row0;  // first of the unit's rows in the request's (token, head of the group) order
  int tiles;          // row tiles with rows
  int from, upto;     // tiles of keys
};

__device__ __forceinline__ int chunkUnitsOf(const AttnArgs& p, const Request& r) {
  const long long rows = static_cast<long long>(r.rows) * p.group;
  return isLong(p, r) ? static_cast<int>((rows + kChunkRows - 1) / kChunkRows) * p.kvHeads * p.splits : 0;
}

// Unit u: the heads of a request, the last rows of a head first (they see
// most keys), the shares of its keys.
__device__ __forceinline__ ChunkUnit chunkUnit(const AttnArgs& p, const int* starts, int u) {
  ChunkUnit c;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (starts[m + 1] > u) hi = m;
    else lo = m + 1;
  }
  c.b = lo;
  c.r = requestOf(p, lo);
  const long long rows = static_cast<long long>(c.r.rows) * p.group;
  const int perHead = static_cast<int>((rows + kChunkRows - 1) / kChunkRows);
  int i = u - starts[lo];
  const int share = i % p.splits;
  i /= p.splits;
  c.head = i / perHead;
  c.row0 = (perHead - 1 - i % perHead) * kChunkRows;
  const int left = static_cast<int>(min(rows - c.row0, static_cast<long long>(kChunkRows)));
  c.tiles = left > 128 ? 2 : 1;
  const int last = (c.row0 + left - 1) / p.group;  // the unit's last token
  const int seen = min(max(c.r.kv - c.r.rows + last + 1, 0), c.r.kv);
  const int all = (seen + kChunkKeys - 1) / kChunkKeys, each = (all + p.splits - 1) / p.splits;
  c.from = min(share * each, all);
  c.upto = min(c.from + each, all);
  return c;
}

// One token's row of codes -> f16 in shared memory: 8 channels a store.
// scale, offset: of its groups, already divided by the power of two.  KEYS:
// the order of the words, and products alone (the offsets go to storeSums).
template <int G, bool KEYS>
__device__ __forceinline__ void widen(const uint32_t (&w)[8 * G], const float (&scale)[G], const float (&offset)[G], uint8_t* block,
                                      int t) {
  __half2 s[G], o[G];
#pragma unroll
  for (int g = 0; g < G; g++) {
    s[g] = __float2half2_rn(scale[g]);
    o[g] = __float2half2_rn(offset[g]);
  }
  const __half2 minus8 = __float2half2_rn(-1032.0f), sixteenth = __float2half2_rn(0.0625f), minus72 = __float2half2_rn(-72.0f);
#pragma unroll
  for (int i = 0; i < 8 * G; i++) {
    const int b = KEYS ? (i / (2 * G)) * 2 + (i & 1) : i / G, g = KEYS ? (i / 2) % G : i % G;
    const uint32_t lo = w[i], hi = __byte_perm(w[i], 0u, 0x4341);
    uint32_t h[4] = {(lo & 0x000F000Fu) | 0x64006400u, (lo & 0x00F000F0u) | 0x64006400u, (hi & 0x000F000Fu) | 0x64006400u,
                     (hi & 0x00F000F0u) | 0x64006400u};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const __half2 c = *reinterpret_cast<const __half2*>(&h[k]);  // 1024 + code, or 1024 + 16 code: both exact
      const __half2 d = (k & 1) ? __hfma2(c, sixteenth, minus72) : __hadd2(c, minus8);
      const __half2 v = KEYS ? __hmul2(d, s[g]) : __hfma2(d, s[g], o[g]);
      h[k] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(block + g * ChunkSmem<G>::kBlock + t * 128 + ((b ^ (t & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
  }
}

// A wait of a whole warp: every lane goes on, or none does.
__device__ __forceinline__ bool warpWait(uint64_t* bar, uint32_t parity, volatile int* abortFlag) {
  return __all_sync(~0u, sm100::mbarWait(bar, parity, abortFlag));
}

// Keys of 32 that a row sees, of which `left` are in its range.
__device__ __forceinline__ uint32_t seenOf(uint32_t valid, int left) {
  return valid & (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1);
}

// First look at a row's scores: the maximum over the keys that it sees, in
// the base-2 logarithm.  EDGE: some row of the warp does not see some key.
// Scores come 32 at a time, the next under way.
template <bool EDGE>
__device__ __forceinline__ float tileMaximum(uint32_t scores, const ChunkInfo& info, float unit, int left) {
  uint32_t s[2][32];
  float top = kNone;
  tmemLoad32(scores, s[0]);
#pragma unroll
  for (int k = 0; k < 4; k++) {
    sm100::tmemLoadWait();
    if (k < 3) tmemLoad32(scores + 32 * (k + 1), s[(k + 1) & 1]);
    const uint32_t seen = EDGE ? seenOf(info.valid[k], left - 32 * k) : ~0u;
    float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; i++) {
      const float v = __uint_as_float(s[k & 1][i]);
      x[i & 1] = fmaxf(x[i & 1], !EDGE || ((seen >> i) & 1u) ? v : -INFINITY);
    }
    const float most = fmaxf(x[0], x[1]);
    if (most > -INFINITY) top = fmaxf(top, most * unit * powerOfTwo(info.keyExp[k]));
  }
  return top;
}

// Second look: the weights, to TMEM in the place of the scores; returns their
// sum.  off: minus the maximum; ref: the power of two that the outputs have.
template <bool EDGE>
__device__ __forceinline__ float tileWeights(uint32_t scores, const ChunkInfo& info, float unit, int left, float m, int ref) {
  uint32_t s[2][32];
  float sum = 0.0f;
  tmemLoad32(scores, s[0]);
#pragma unroll
  for (int k = 0; k < 4; k++) {
    sm100::tmemLoadWait();
    if (k < 3) tmemLoad32(scores + 32 * (k + 1), s[(k + 1) & 1]);
    const uint32_t seen = EDGE ? seenOf(info.valid[k], left - 32 * k) : ~0u;
    const int ve = info.valueExp[k], shift = ve == kNoExponent ? 0 : max(ve - ref, -100);
    const float scale = unit * powerOfTwo(info.keyExp[k]), off = static_cast<float>(shift) - m;
    float part[2] = {0.0f, 0.0f};
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float a = exp2Fast(fmaf(__uint_as_float(s[k & 1][2 * i]), scale, off));
      float b = exp2Fast(fmaf(__uint_as_float(s[k & 1][2 * i + 1]), scale, off));
      if (EDGE) {
        if (!((seen >> (2 * i)) & 1u)) a = 0.0f;
        if (!((seen >> (2 * i + 1)) & 1u)) b = 0.0f;
      }
      part[0] += a;
      part[1] += b;
      w[i] = packHalf(a, b);
    }
    sum = fmaf(part[0] + part[1], powerOfTwo(-shift), sum);
    // Scores 32 (k + 1) on are under way or to come: the weights end before them.
    tmemStore16(scores + 16 * k, w);
  }
  return sum;
}

template <int G>
struct RawToken {
  uint32_t k[8 * G], v[8 * G], kp[G], vp[G];
  bool there;
};

template <int G>
__global__ void __launch_bounds__(kChunkThreads, 1) chunkKernel(const __grid_constant__ AttnArgs p) {
  extern __shared__ uint8_t smemRaw[];
  constexpr int D = 64 * G;
  using L = ChunkSmem<G>;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~static_cast<uintptr_t>(1023));
  ChunkControl& ctl = *reinterpret_cast<ChunkControl*>(smem + L::kInfo);
  int* starts = reinterpret_cast<int*>(smem + L::kStarts);
  volatile int* abortFlag = &ctl.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      sm100::mbarInit(&ctl.qFull[i], 128);
      sm100::mbarInit(&ctl.kFull[i], 128);
      sm100::mbarInit(&ctl.kEmpty[i], 1);
      sm100::mbarInit(&ctl.vFull[i], 128);
      sm100::mbarInit(&ctl.vEmpty[i], 1);
      sm100::mbarInit(&ctl.sFull[i], 1);
      sm100::mbarInit(&ctl.pFull[i], 128);
      sm100::mbarInit(&ctl.oFull[i], 1);
    }
    sm100::mbarInit(&ctl.drain, 1);
    ctl.abort = 0;
    sm100::fenceBarrierInit();
  }
  if (warp == 12) {
    sm100::tmemAlloc(&ctl.tmem, 512);
    sm100::tmemRelinquish();
  }
  // Units before each request: one warp, 32 requests a step.
  if (warp == 0) {
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int b = base + lane;
      int v = b < p.batch ? chunkUnitsOf(p, requestOf(p, b)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += x;
      }
      if (b < p.batch) starts[b + 1] = before + v;
      before += __shfl_sync(~0u, v, 31);
    }
    if (lane == 0) starts[0] = 0;
  }
  sm100::tcFenceBefore();
  __syncthreads();
  sm100::tcFenceAfter();
  const uint32_t tmem = ctl.tmem;
  const int units = starts[p.batch];
  constexpr uint32_t kOut = 256;  // columns of the outputs, behind two times 128 of scores

  if (warp < 8) {
    // ---------------- softmax ----------------
    const int t = warp >> 2, row = threadIdx.x & 127;
    const uint32_t scores = tmem + t * 128 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t output = tmem + kOut + t * D + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint32_t seq = 0;               // tiles of keys of the block so far: the place of their info
    uint32_t sCount = 0, oCount = 0;  // scores and outputs of this row tile so far
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const ChunkUnit c = chunkUnit(p, starts, u);
      if (t >= c.tiles) {
        seq += c.upto - c.from;  // the info ring moves on
        continue;
      }
      const long long mine = static_cast<long long>(c.row0) + t * 128 + row;
      const bool live = mine < static_cast<long long>(c.r.rows) * p.group;
      const int token = live ? static_cast<int>(mine / p.group) : 0, h = c.head * p.group + (live ? static_cast<int>(mine % p.group) : 0);
      const int limit = live ? min(max(c.r.kv - c.r.rows + token + 1, 0), c.r.kv) : c.r.kv;
      float m = kNone, l = 0.0f, unit = 1.0f;
      int ref = kNoExponent;  // the outputs are in units of 2^ref
      uint32_t poison = 0;
      if (c.from < c.upto) {
        // The row's channels, scaled to 2^8, and their sums as the left operand.
        float amax = 0.0f, sums[G] = {};
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + static_cast<long long>(c.r.start + token) * p.qTok + static_cast<long long>(h) * p.qHead;
        uint4 raw[8 * G];
#pragma unroll
        for (int i = 0; i < 8 * G; i++) {
          raw[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
          float x[8];
          if (p.half16) unpack8<__half>(raw[i], x);
          else unpack8<__nv_bfloat16>(raw[i], x);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            amax = fmaxf(amax, fabsf(x[e]));
            sums[i / 8] += x[e];
          }
        }
        const int e = exponentOf(amax);
        const bool plain = amax == 0.0f || e > 120 || e < -100;
        const float f = (plain ? 1.0f : powerOfTwo(8 - e)) * (p.scaleLog2 < 0.0f ? -1.0f : 1.0f);
        unit = (plain ? 1.0f : powerOfTwo(e - 8)) * fabsf(p.scaleLog2);
#pragma unroll
        for (int i = 0; i < 8 * G; i++) {
          float x[8];
          if (p.half16) unpack8<__half>(raw[i], x);
          else unpack8<__nv_bfloat16>(raw[i], x);
#pragma unroll
          for (int k = 0; k < 8; k++) x[k] *= f;
          *reinterpret_cast<uint4*>(smem + L::kQ + (t * G + i / 8) * L::kBlock + row * 128 + (((i & 7) ^ (row & 7)) << 4)) = pack8<__half>(x);
        }
#pragma unroll
        for (int g = 0; g < G; g++) sums[g] *= f;
        storeSums<G, true>(smem + L::kQSums + t * kPlainBytes, row, sums);
        sm100::fenceProxyAsyncShared();
        sm100::mbarArrive(&ctl.qFull[t]);
        for (int j = c.from; j < c.upto; j++, seq++) {
          if (!warpWait(&ctl.sFull[t], sCount & 1u, abortFlag)) {
            ok = false;
            break;
          }
          sCount++;
          sm100::tcFenceAfter();
          const ChunkInfo& info = ctl.info[seq & 3];
          const int left = limit - j * kChunkKeys;  // keys of the tile in the row's range
          const uint32_t valid = info.valid[0] & info.valid[1] & info.valid[2] & info.valid[3];
          const bool edge = __any_sync(~0u, left < kChunkKeys || valid != ~0u);
          int newRef = ref;
#pragma unroll
          for (int k = 0; k < 4; k++) newRef = max(newRef, info.valueExp[k]);
          const float top = edge ? tileMaximum<true>(scores, info, unit, left) : tileMaximum<false>(scores, info, unit, left);
          if (__any_sync(~0u, top > m + 8.0f || newRef > ref)) {
            const float next = fmaxf(m, top), shrink = exp2Fast(m - next);
            if (j > c.from) {
              const float factor = shrink * (ref == kNoExponent ? 1.0f : powerOfTwo(max(ref - newRef, -126)));
#pragma unroll 1
              for (int k = 0; k < D / 32; k++) {
                uint32_t o[32];
                tmemLoad32(output + 32 * k, o);
                sm100::tmemLoadWait();
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                tmemStore32(output + 32 * k, o);
              }
              tmemStoreWait();
            }
            l *= shrink;
            m = next;
            ref = newRef;
          }
          l += edge ? tileWeights<true>(scores, info, unit, left, m, ref) : tileWeights<false>(scores, info, unit, left, m, ref);
#pragma unroll
          for (int g = 0; g < G; g++)
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (info.bad[g][k] & seenOf(info.valid[k], left - 32 * k)) poison |= 1u << g;
          tmemStoreWait();
          sm100::tcFenceBefore();
          sm100::mbarArrive(&ctl.pFull[t]);
        }
      }
      // The result, or this share of it.
      const bool any = c.from < c.upto;
      if (!ok || (!any && p.splits > 1)) continue;  // an empty share counts as absent
      if (any) {
        if (!warpWait(&ctl.oFull[t], oCount & 1u, abortFlag)) {
          ok = false;
          continue;
        }
        oCount++;
        sm100::tcFenceAfter();
      }
      const bool whole = p.splits == 1, none = l == 0.0f;
      const float factor = (whole ? (none ? 0.0f : 1.0f / l) : 1.0f) * (ref == kNoExponent ? 1.0f : powerOfTwo(ref));
      const long long slot = static_cast<long long>(u) * kChunkRows + t * 128 + row;
#pragma unroll 1
      for (int k = 0; k < D / 32; k++) {
        uint32_t o[32];
        float y[32];
        if (any) {  // the whole warp or none of it
          tmemLoad32(output + 32 * k, o);
          sm100::tmemLoadWait();
        }
        const bool spoilt = (poison >> (k / 2)) & 1u;
#pragma unroll
        for (int i = 0; i < 32; i++) y[i] = none ? 0.0f : spoilt ? NAN : __uint_as_float(o[i]) * factor;
        if (live) {
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const float z[8] = {y[8 * v], y[8 * v + 1], y[8 * v + 2], y[8 * v + 3], y[8 * v + 4], y[8 * v + 5], y[8 * v + 6], y[8 * v + 7]};
            if (whole) {
              const long long at = static_cast<long long>(c.r.start + token) * p.oTok + static_cast<long long>(h) * p.oHead + 32 * k + 8 * v;
              if (p.half16) *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + at) = pack8<__half>(z);
              else *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + at) = pack8<__nv_bfloat16>(z);
            } else {
              float* dst = p.chunkPartial + slot * D + 32 * k + 8 * v;
              *reinterpret_cast<float4*>(dst) = make_float4(z[0], z[1], z[2], z[3]);
              *reinterpret_cast<float4*>(dst + 4) = make_float4(z[4], z[5], z[6], z[7]);
            }
          }
        }
      }
      if (live) {
        if (!whole) p.chunkStats[slot] = make_float2(m, l);
        else if (p.lse != nullptr) p.lse[static_cast<long long>(c.r.start + token) * p.qHeads + h] = none ? -INFINITY : (m + log2f(l)) * kLn2;
      }
      sm100::tcFenceBefore();  // the next unit's products come behind these loads
    }
  } else if (warp < 12) {
    // ---------------- codes to f16 ----------------
    const int tid = threadIdx.x - 256, w = warp - 8;
    // The tile whose page number is under way: two tiles ahead of the one that is turned.
    int u = blockIdx.x, j = 0, upto = 0, head = 0, kv = 0;
    const int* pages = nullptr;
    bool exists = false;
    int token = 0, page = -1;
    auto advance = [&]() {
      j++;
      while (j >= upto) {
        if (u >= units) {
          exists = false;
          return;
        }
        const ChunkUnit c = chunkUnit(p, starts, u);
        u += gridDim.x;
        j = c.from;
        upto = c.upto;
        head = c.head;
        kv = c.r.kv;
        pages = p.table + static_cast<long long>(c.b) * p.width;
      }
      exists = true;
      token = j * kChunkKeys + tid;
      page = token < kv ? pages[token / (p.blocksPerPage * 16)] : -1;
    };
    auto fetch = [&](RawToken<G>& r) {
      r.there = exists && page >= 0 && page < p.pages;
      if (r.there) {
        const int place = token % (p.blocksPerPage * 16);
        const uint8_t* block = p.cache + ((static_cast<long long>(page) * p.kvHeads + head) * p.blocksPerPage + (place >> 4)) * (18 * D);
        const int at = place & 15;
        const uint4* k = reinterpret_cast<const uint4*>(block + at * (D / 2));
        const uint4* v = reinterpret_cast<const uint4*>(block + 8 * D + kv4::valueRow(at) * (D / 2));
#pragma unroll
        for (int i = 0; i < 2 * G; i++) {
          const uint4 a = __ldg(k + i), b = __ldg(v + i);
          r.k[4 * i] = a.x;
          r.k[4 * i + 1] = a.y;
          r.k[4 * i + 2] = a.z;
          r.k[4 * i + 3] = a.w;
          r.v[4 * i] = b.x;
          r.v[4 * i + 1] = b.y;
          r.v[4 * i + 2] = b.z;
          r.v[4 * i + 3] = b.w;
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
          r.kp[g] = __ldg(reinterpret_cast<const uint32_t*>(block + 16 * D + at * (4 * G)) + g);
          r.vp[g] = __ldg(reinterpret_cast<const uint32_t*>(block + 17 * D + at * (4 * G)) + g);
        }
      } else {  // zeros: codes of 0 with nothing to scale
#pragma unroll
        for (int i = 0; i < 8 * G; i++) r.k[i] = r.v[i] = 0;
#pragma unroll
        for (int g = 0; g < G; g++) r.kp[g] = r.vp[g] = 0;
      }
    };
    RawToken<G> raw, next;
    advance();
    fetch(raw);
    bool here = exists;
    if (exists) advance();
    for (uint32_t seq = 0; here; seq++) {
      const bool follows = exists;
      fetch(next);
      if (exists) advance();
      // Parameters of the 32 tokens of this warp, and their powers of two.
      float ks[G], km[G], vs[G], vm[G], kTop = 0.0f, vTop = 0.0f;
      ChunkInfo& info = ctl.info[seq & 3];
#pragma unroll
      for (int g = 0; g < G; g++) {
        ks[g] = kv4::bf16Lo(raw.kp[g]);
        km[g] = kv4::bf16Hi(raw.kp[g]);
        vs[g] = kv4::bf16Lo(raw.vp[g]);
        vm[g] = kv4::bf16Hi(raw.vp[g]);
        const bool bad = !(isfinite(vs[g]) && isfinite(vm[g]));
        if (bad) vs[g] = vm[g] = 0.0f;
        const uint32_t whose = __ballot_sync(~0u, bad);
        if (lane == 0) info.bad[g][w] = whose;
        kTop = fmaxf(kTop, fmaf(8.5f, fabsf(ks[g]), fabsf(km[g])));
        vTop = fmaxf(vTop, fmaf(8.5f, fabsf(vs[g]), fabsf(vm[g])));
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        kTop = fmaxf(kTop, __shfl_xor_sync(~0u, kTop, o));
        vTop = fmaxf(vTop, __shfl_xor_sync(~0u, vTop, o));
      }
      const int ke = kTop == 0.0f || !(kTop < INFINITY) ? 0 : max(exponentOf(kTop), -100) - 12;
      const int ve = vTop == 0.0f ? kNoExponent : max(exponentOf(vTop), -100) - 12;
      const uint32_t there = __ballot_sync(~0u, raw.there);
      if (lane == 0) {
        info.valid[w] = there;
        info.keyExp[w] = ke;
        info.valueExp[w] = ve;
      }
      const float kf = powerOfTwo(-ke), vf = ve == kNoExponent ? 1.0f : powerOfTwo(-ve);
#pragma unroll
      for (int g = 0; g < G; g++) {
        ks[g] *= kf;
        km[g] = fmaf(0.5f, ks[g], km[g] * kf);  // value = m + s (code - 8) from here on
        vs[g] *= vf;
        vm[g] = fmaf(0.5f, vs[g], vm[g] * vf);
      }
      const int st = seq & 1;
      const uint32_t parity = ((seq >> 1) & 1u) ^ 1u;
      if (!warpWait(&ctl.kEmpty[st], parity, abortFlag)) break;
      widen<G, true>(raw.k, ks, km, smem + L::kK + st * G * L::kBlock, tid);
      storeSums<G, false>(smem + L::kKSums + st * kPlainBytes, tid, km);
      sm100::fenceProxyAsyncShared();
      sm100::mbarArrive(&ctl.kFull[st]);
      if (!warpWait(&ctl.vEmpty[st], parity, abortFlag)) break;
      widen<G, false>(raw.v, vs, vm, smem + L::kV + st * G * L::kBlock, tid);
      sm100::fenceProxyAsyncShared();
      sm100::mbarArrive(&ctl.vFull[st]);
      raw = next;
      here = follows;
    }
  } else if (lane == 0) {
    // ---------------- products ----------------
    constexpr uint32_t kScores = idescF16(128, 128, false), kOutputs = idescF16(128, D, true);
    const uint32_t qSums = sm100::smemAddr(smem + L::kQSums), kSums = sm100::smemAddr(smem + L::kKSums);
    const uint32_t qBase = sm100::smemAddr(smem + L::kQ), kBase = sm100::smemAddr(smem + L::kK), vBase = sm100::smemAddr(smem + L::kV);
    uint32_t seq = 0, qCount[2] = {0, 0}, pCount[2] = {0, 0};
    bool ok = true;
    // Words of the descriptors: addresses count 16 bytes.
    const uint64_t rows = sm100::smemDescSw128(0), plain = smemDescPlain(0), major = smemDescMn(0);
    const uint32_t rowsLo = static_cast<uint32_t>(rows), rowsHi = static_cast<uint32_t>(rows >> 32);
    const uint32_t plainLo = static_cast<uint32_t>(plain), plainHi = static_cast<uint32_t>(plain >> 32);
    const uint32_t majorLo = static_cast<uint32_t>(major), majorHi = static_cast<uint32_t>(major >> 32);
    constexpr uint32_t kStep = L::kBlock >> 4;
    auto issueScores = [&](int t, uint32_t s) {
      const uint32_t d = tmem + t * 128, q = rowsLo + (qBase >> 4) + t * (G * kStep), k = rowsLo + (kBase >> 4) + (s & 1) * (G * kStep);
      mmaF16<false>(d, q, rowsHi, k, rowsHi, kScores);
#pragma unroll
      for (int i = 1; i < 4 * G; i++)
        mmaF16<true>(d, q + (i >> 2) * kStep + 2 * (i & 3), rowsHi, k + (i >> 2) * kStep + 2 * (i & 3), rowsHi, kScores);
      mmaF16<true>(d, plainLo + (qSums >> 4) + t * (kPlainBytes >> 4), plainHi, plainLo + (kSums >> 4) + (s & 1) * (kPlainBytes >> 4),
                   plainHi, kScores);
      sm100::mmaCommit(&ctl.sFull[t]);
    };
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const ChunkUnit c = chunkUnit(p, starts, u);
      const int n = c.upto - c.from;
      if (n <= 0) continue;
      for (int t = 0; t < c.tiles && ok; t++) ok = sm100::mbarWait(&ctl.qFull[t], qCount[t]++ & 1u, abortFlag);
      ok = ok && sm100::mbarWait(&ctl.kFull[seq & 1], (seq >> 1) & 1u, abortFlag);
      if (!ok) break;
      sm100::tcFenceAfter();
      for (int t = 0; t < c.tiles; t++) issueScores(t, seq);
      sm100::mmaCommit(&ctl.kEmpty[seq & 1]);
      for (int j = 0; j < n && ok; j++, seq++) {
        for (int t = 0; t < c.tiles; t++) {
          ok = sm100::mbarWait(&ctl.pFull[t], pCount[t]++ & 1u, abortFlag);
          if (ok && t == 0) ok = sm100::mbarWait(&ctl.vFull[seq & 1], (seq >> 1) & 1u, abortFlag);
          if (!ok) break;
          sm100::tcFenceAfter();
#pragma unroll
          for (int k = 0; k < 8; k++)
            mmaF16Tmem(tmem + kOut + t * D, tmem + t * 128 + 8 * k, majorLo + (vBase >> 4) + (seq & 1) * (G * kStep) + 128 * k, majorHi,
                       kOutputs, k > 0 ? 1u : static_cast<uint32_t>(j));
          if (j + 1 == n) sm100::mmaCommit(&ctl.oFull[t]);
          if (t + 1 == c.tiles) sm100::mmaCommit(&ctl.vEmpty[seq & 1]);
          if (j + 1 < n) {
            if (t == 0) {
              ok = sm100::mbarWait(&ctl.kFull[(seq + 1) & 1], ((seq + 1) >> 1) & 1u, abortFlag);
              if (!ok) break;
              sm100::tcFenceAfter();
            }
            issueScores(t, seq + 1);
            if (t + 1 == c.tiles) sm100::mmaCommit(&ctl.kEmpty[(seq + 1) & 1]);
          }
        }
      }
    }
    if (!ok) {  // let the products that were issued end before the block does
      sm100::mmaCommit(&ctl.drain);
      volatile int never = 0;
      sm100::mbarWait(&ctl.drain, 0, &never, 200000000ull);
    }
  }
  __syncwarp();
  sm100::tcFenceBefore();
  __syncthreads();
  sm100::tcFenceAfter();
  if (warp == 12) sm100::tmemDealloc(tmem, 512);
  if (threadIdx.x == 0) {
    if (*abortFlag && p.errorFlag != nullptr) *reinterpret_cast<volatile int*>(p.errorFlag) = 1;
    if (blockIdx.x == 0)
      for (int b = 0; b <= p.batch; b++) p.chunkStarts[b] = starts[b];
  }
}

// Joins the shares of every row of a long request (splits > 1), a warp a row.
template <int G>
__global__ void __launch_bounds__(128) chunkJoinKernel(const __grid_constant__ AttnArgs p) {
  constexpr int D = 64 * G;
  const int lane = threadIdx.x & 31;
  const long long id = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (id >= static_cast<long long>(p.tokens) * p.qHeads) return;
  const int t = static_cast<int>(id / p.qHeads), h = static_cast<int>(id - static_cast<long long>(t) * p.qHeads);
  const int b = requestOfRow(p, t, lane);
  if (b >= p.batch) return;
  const Request r = requestOf(p, b);
  if (t < r.start || t >= r.start + r.rows || !isLong(p, r)) return;
  const int row = (t - r.start) * p.group + h % p.group;
  const int perHead = static_cast<int>((static_cast<long long>(r.rows) * p.group + kChunkRows - 1) / kChunkRows);
  const int first = p.chunkStarts[b] + ((h / p.group) * perHead + perHead - 1 - row / kChunkRows) * p.splits;
  float y[2 * G] = {};
  float m = kNone, l = 0.0f;
  for (int s = 0; s < p.splits; s++) {
    // the same split as the kernel's (uniform over the unit's rows)
    const int last = min((row / kChunkRows + 1) * kChunkRows, r.rows * p.group) - 1;
    const int seen = min(max(r.kv - r.rows + last / p.group + 1, 0), r.kv);
    const int all = (seen + kChunkKeys - 1) / kChunkKeys, each = (all + p.splits - 1) / p.splits;
    if (s * each >= all) break;
    const long long slot = static_cast<long long>(first + s) * kChunkRows + row % kChunkRows;
    const float2 st = p.chunkStats[slot];
    const float top = fmaxf(m, st.x), old = exp2Fast(m - top), add = exp2Fast(st.x - top);
    m = top;
    l = l * old + st.y * add;
    const float2* src = reinterpret_cast<const float2*>(p.chunkPartial + slot * D) + lane;
#pragma unroll
    for (int g = 0; g < G; g++) {
      const float2 v = src[32 * g];
      y[2 * g] = fmaf(v.x, add, y[2 * g] * old);
      y[2 * g + 1] = fmaf(v.y, add, y[2 * g + 1] * old);
    }
  }
  storeRow<G>(p, t, h, lane, y, m, l);
}

}  // namespace
}  // namespace model
}  // namespace vccl

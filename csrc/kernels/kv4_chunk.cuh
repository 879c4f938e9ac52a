// SPDX-License-Identifier: Apache-2.0
// Attention of long runs of query rows over the 4-bit cache on the 5th
// generation tensor cores (included by kv4_attention.cu).
//
// A unit is 256 query rows (two tiles of 128) of one request and key head
// against a range of keys, 64 at a time.  Roles of a block of 16 warps
// (registers go by fours of warps; the last two only hand theirs over):
//   warps 0-3, 4-7  softmax of the first and the second row tile, a thread a
//                   row: scores from TMEM, weights back to TMEM as f16, in
//                   the place of the scores;
//   warps 8-9       a thread a token: key codes from global memory (one tile
//   10-11           ahead in registers) to f16 in shared memory, in the
//                   128-byte swizzle that the products read; value codes;
//   warps 12, 13    issue S = Q K^T (N = 64) and O += P V (P from TMEM, V with
//                   channels as the major axis) of a row tile each: one thread
//                   for both took 80 to 100 clocks a product, more than the
//                   tensor cores do.
// A row tile has two places for scores, so the products of the keys after next
// go on beside the softmax of these (with 128 keys and one place the softmax
// waited 1700 of 7800 clocks for its scores, and read them twice for want of
// registers).  The products of one thread run in order, so scores may take the
// place of weights just used.
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
// Where some of the 32 are far below the largest (2^8 for values, 2^14 for
// keys) each is divided by a power of its own, and the softmax puts that back
// token by token.  A row's outputs are in units of the largest weight times
// value that it met, so what it does not see or gives no weight costs the rest
// no bits.  Both groups of 64 channels share a row's weights, so where one's
// values are more than 2^16 above the other's the other loses bits.  Scores,
// maxima, sums and outputs are f32.  The maximum is followed loosely (by 8 in
// the base-2 logarithm), so the output is rescaled rarely.
//
// Measured: 842 us, 715 TFLOP/s, for 4 requests of 1024 rows against 2000 to
// 9000 tokens, 64 heads on 8 (the single-token kernel takes 3.4 ms); 1.8 ms where
// every 32 tokens hold values 2^10 apart.  The softmax bounds it: 2230 of
// 3070 clocks when a tile took as many.
#pragma once

#include "kernels/kv4.cuh"
#include "kernels/sm100.cuh"

namespace vccl {
namespace model {
namespace {

constexpr int kChunkRows = 256;
constexpr int kChunkKeys = 64;
constexpr int kChunkStages = 4;     // tiles of keys, and of values, in shared memory
constexpr int kChunkThreads = 16 * 32;
constexpr int kLeastExponent = -112;  // of 32 tokens that are all zero, or next to it
// Binary orders that 32 tokens may lie apart and share a power of two: keys and
// their sums then keep all bits; a row whose weight is on the smallest value
// loses 2^-21 of it for each other token.
constexpr int kKeysApart = 14, kValuesApart = 8;
// The largest weight times value of a row becomes 2^6 in f16, times up to 2^13
// of the value, when its unit moves, and may grow to 2^15 until it moves again.
constexpr float kTopWeight = 6.0f, kMostWeight = 15.0f;

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
// the next 64 channels 8 KiB on (leading), the next 8 tokens 1 KiB on (stride).
__device__ __forceinline__ uint64_t smemDescMn(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
  d |= static_cast<uint64_t>(8192u >> 4) << 16;
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
  static constexpr int kQBlock = 16384;  // 128 rows of 64 f16
  static constexpr int kBlock = 8192;    // 64 tokens of 64 f16
  static constexpr int kQ = 0;           // [2 row tiles][G]
  static constexpr int kK = kQ + 2 * G * kQBlock;  // [stages][G]
  static constexpr int kV = kK + kChunkStages * G * kBlock;
  static constexpr int kQSums = kV + kChunkStages * G * kBlock;  // [2 row tiles]
  static constexpr int kKSums = kQSums + 2 * 128 * 32;           // [stages]
  static constexpr int kInfo = kKSums + kChunkStages * 64 * 32;
  static constexpr int kStarts = kInfo + 1680;  // units before each request
};

// Of a tile, by 32 tokens: some are not there or not finite; keys, values with
// powers of two of their own.
constexpr uint32_t kUneven = 1, kOwnKeys = 2, kOwnValues = 4;

// What the tokens of a tile bring, by 32.
struct alignas(16) ChunkInfo {
  uint32_t valid[2];               // the token is there
  float keyUnit[2];                // the power of two that its keys are divided by
  float valueExp[2];               // the logarithm of that of its values
  uint32_t kind[2];
  uint32_t bad[2][2];              // its values of a group are not finite (and zero in the product)
  // Where they have powers of their own: 127 + the orders that the token's is
  // below the largest, which the two above are then of.
  uint8_t keyOrder[64], valueOrder[64];
};

struct ChunkControl {
  ChunkInfo info[2 * kChunkStages];  // written with the keys, read until the weights are there
  uint64_t kFull[kChunkStages], kEmpty[kChunkStages], vFull[kChunkStages], vEmpty[kChunkStages];
  // A wait tells a phase of a barrier from the one before it alone, so what
  // can be two tiles ahead has a barrier for each place.
  uint64_t qFull[2], sFull[2][2], pFull[2][2], pvDone[2][2], drain[2];
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(ChunkControl) <= ChunkSmem<2>::kStarts - ChunkSmem<2>::kInfo, "the control block's place");

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
  const int rows = c.r.rows * p.group;  // at most tokens * q heads
  const int perHead = (rows + kChunkRows - 1) / kChunkRows;
  int i = u - starts[lo];
  const int share = i % p.splits;
  i /= p.splits;
  c.head = i / perHead;
  c.row0 = (perHead - 1 - i % perHead) * kChunkRows;
  const int left = min(rows - c.row0, kChunkRows);
  c.tiles = left > 128 ? 2 : 1;
  const int last = (c.row0 + left - 1) / p.group;  // the unit's last token
  const int seen = min(max(c.r.kv - c.r.rows + last + 1, 0), c.r.kv);
  const int all = (seen + kChunkKeys - 1) / kChunkKeys, each = (all + p.splits - 1) / p.splits;
  c.from = min(share * each, all);
  c.upto = min(c.from + each, all);
  return c;
}

// The unit that this block takes in a round: rounds go to and fro, since the
// units of a head come heaviest first.
__device__ __forceinline__ int unitOfRound(int round) {
  const int n = gridDim.x, b = blockIdx.x;
  return round * n + ((round & 1) ? n - 1 - b : b);
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
  if (__all_sync(~0u, sm100::mbarTryWait(bar, parity))) return true;
  return __all_sync(~0u, sm100::mbarWait(bar, parity, abortFlag));
}

// Keys of 32 that a row sees, of which `left` are in its range.
__device__ __forceinline__ uint32_t seenOf(uint32_t valid, int left) {
  return valid & (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1);
}

// 32 scores of a row; those of keys that it does not see become -inf.
template <bool EDGE>
__device__ __forceinline__ void loadScores(uint32_t at, uint32_t (&s)[32], uint32_t seen) {
  tmemLoad32(at, s);
  sm100::tmemLoadWait();
  if (EDGE) {
#pragma unroll
    for (int i = 0; i < 32; i++)
      if (!((seen >> i) & 1u)) s[i] = 0xFF800000u;
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^-n and -n from the byte 127 - n that i is of four.
__device__ __forceinline__ float powerOfOrder(uint32_t four, int i) {
  return __uint_as_float(__byte_perm(four, 0u, 0x0444 | (i << 12)) >> 1);
}
__device__ __forceinline__ float logOfOrder(uint32_t four, int i) {
  return __uint_as_float(__byte_perm(four, 0x4B000000u, 0x7650 | i)) - 8388735.0f;  // 2^23 + 127
}

// Scores of keys with powers of their own, in units of the largest one's.
__device__ __forceinline__ void levelScores(uint32_t (&s)[32], const uint8_t* orders) {
  const uint32_t* four = reinterpret_cast<const uint32_t*>(orders);
#pragma unroll
  for (int i = 0; i < 32; i++) s[i] = __float_as_uint(__uint_as_float(s[i]) * powerOfOrder(four[i >> 2], i & 3));
}

// The weights of 32 scores, to TMEM in their place; returns their sum.  orders:
// of the values, where they have powers of their own.
template <bool OWN>
__device__ __forceinline__ float halfWeights(const uint32_t (&s)[32], uint32_t at, float scale, float off, const uint8_t* orders) {
  const uint32_t* four = reinterpret_cast<const uint32_t*>(orders);
  uint64_t part[2] = {0, 0};
  const uint64_t by = pair(scale), plus = pair(off);
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float2 x = unpair(fma2(pair(s[2 * i], s[2 * i + 1]), by, plus));
    float a = exp2Fast(x.x), b = exp2Fast(x.y);
    part[i & 1] = add2(part[i & 1], pair(__float_as_uint(a), __float_as_uint(b)));
    if (OWN) {
      a *= powerOfOrder(four[i >> 1], (2 * i) & 3);
      b *= powerOfOrder(four[i >> 1], (2 * i + 1) & 3);
    }
    w[i] = packHalf(a, b);
  }
  tmemStore16(at, w);
  const float2 sum = unpair(add2(part[0], part[1]));
  return sum.x + sum.y;
}

// What a softmax thread keeps of its row.
struct RowState {
  float m, l;      // maximum followed loosely (base-2 logarithm), sum
  float ref;       // the outputs are in units of 2^ref
  uint32_t poison; // groups whose values are not finite
};

// Not zero (a softmax scale of zero, or one next to it): unseen scores are
// -inf, and scores times the smallest number count nothing.
__device__ __forceinline__ float notZero(float x) { return x < FLT_MIN ? FLT_MIN : x; }

// Moves the maximum and the unit of the outputs where a row of the warp needs
// it.  top: the largest score; high: the largest score plus logarithm of the
// value.  Returns false if a wait ran out.
template <int D>
__device__ __forceinline__ bool follow(RowState& r, float top, float high, uint32_t output, bool first, uint64_t* before,
                                       uint32_t beforeParity, volatile int* abortFlag) {
  if (!__any_sync(~0u, top > r.m + 8.0f || high > r.m + r.ref + kMostWeight)) return true;
  // What was the largest weight times value shrinks with the other weights.
  const float next = fmaxf(r.m, top), old = r.ref + (r.m - next), ref = fmaxf(old, high - next - kTopWeight);
  if (!first) {
    // the products with the weights before these have ended
    if (!warpWait(before, beforeParity, abortFlag)) return false;
    sm100::tcFenceAfter();
    const float factor = exp2Fast(old - ref);
#pragma unroll 1
    for (int k = 0; k < D / 16; k++) {
      uint32_t o[16];
      sm100::tmemLoad16(output + 16 * k, o);
      sm100::tmemLoadWait();
#pragma unroll
      for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
      tmemStore16(output + 16 * k, o);
    }
  }
  r.l *= exp2Fast(r.m - next);
  r.m = next;
  r.ref = ref;
  return true;
}

// Weights of values in much smaller units than the outputs': 2^40 apart they
// are nothing in f16, and all of them still count in the sum.
__device__ __forceinline__ float shiftOf(float valueExp, float ref) { return fmaxf(valueExp - ref, -40.0f); }

__device__ __forceinline__ uint32_t poisoned(const ChunkInfo& info, uint32_t seen0, uint32_t seen1) {
  const uint4 bad = *reinterpret_cast<const uint4*>(info.bad);
  return (((bad.x & seen0) | (bad.y & seen1)) ? 1u : 0u) | (((bad.z & seen0) | (bad.w & seen1)) ? 2u : 0u);
}

// One tile's scores to weights.  EDGE: tokens are missing or not finite, or some
// row of the warp does not see some; OWN: some have powers of two of their own.
// Returns false if a wait ran out.
template <int G, bool EDGE, bool OWN>
__device__ __forceinline__ bool tileSoftmax(RowState& r, uint32_t scores, uint32_t output, const ChunkInfo& info, float unit,
                                            int left, bool first, uint64_t* before, uint32_t beforeParity, volatile int* abortFlag) {
  const float2 keyUnit = *reinterpret_cast<const float2*>(info.keyUnit), valueExp = *reinterpret_cast<const float2*>(info.valueExp);
  const float scale0 = notZero(unit * keyUnit.x), scale1 = notZero(unit * keyUnit.y);
  const uint32_t seen0 = EDGE ? seenOf(info.valid[0], left) : ~0u, seen1 = EDGE ? seenOf(info.valid[1], left - 32) : ~0u;
  float top = kNone, high = kNone;
#pragma unroll 1
  for (int k = 0; k < 2; k++) {
    uint32_t s[32];
    loadScores<EDGE>(scores + 32 * k, s, k ? seen1 : seen0);
    if (OWN && (info.kind[k] & kOwnKeys)) levelScores(s, info.keyOrder + 32 * k);
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = __uint_as_float(s[i]);
#pragma unroll
    for (int i = 4; i < 32; i += 2) x[(i >> 1) & 3] = max3(x[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    const float most = max3(x[0], x[1], fmaxf(x[2], x[3])), scale = k ? scale1 : scale0;
    if (!EDGE || most > -INFINITY) {
      top = fmaxf(top, most * scale);
      float weighed = most * scale;  // with the values' orders
      if (OWN && (info.kind[k] & kOwnValues)) {
        const uint32_t* four = reinterpret_cast<const uint32_t*>(info.valueOrder + 32 * k);
        weighed = kNone;
#pragma unroll
        for (int i = 0; i < 32; i++) weighed = fmaxf(weighed, fmaf(__uint_as_float(s[i]), scale, logOfOrder(four[i >> 2], i & 3)));
      }
      high = fmaxf(high, weighed + (k ? valueExp.y : valueExp.x));
    }
  }
  if (!follow<64 * G>(r, top, high, output, first, before, beforeParity, abortFlag)) return false;
  const float shift0 = shiftOf(valueExp.x, r.ref), shift1 = shiftOf(valueExp.y, r.ref);
#pragma unroll 1
  for (int k = 0; k < 2; k++) {
    uint32_t s[32];
    loadScores<EDGE>(scores + 32 * k, s, k ? seen1 : seen0);
    const float shift = k ? shift1 : shift0, scale = k ? scale1 : scale0;
    float sum;
    if (OWN && (info.kind[k] & kOwnKeys)) levelScores(s, info.keyOrder + 32 * k);
    if (OWN && (info.kind[k] & kOwnValues)) sum = halfWeights<true>(s, scores + 16 * k, scale, shift - r.m, info.valueOrder + 32 * k);
    else sum = halfWeights<false>(s, scores + 16 * k, scale, shift - r.m, nullptr);
    r.l = fmaf(sum, exp2Fast(-shift), r.l);
  }
  if (EDGE) r.poison |= poisoned(info, seen0, seen1);
  return true;
}

// Rare code stands out of the way of the other: in line it cost the whole
// kernel 2 %, and short requests, whose tiles all are at an edge, 8 %.
struct Followed {
  RowState row;
  bool ok;
};
template <int G>
__device__ __noinline__ Followed ownSoftmax(RowState r, uint32_t scores, uint32_t output, const ChunkInfo* info, float unit, int left,
                                            bool first, uint64_t* before, uint32_t beforeParity, volatile int* abortFlag) {
  const bool ok = tileSoftmax<G, true, true>(r, scores, output, *info, unit, left, first, before, beforeParity, abortFlag);
  return {r, ok};
}

// Logarithm of the power of two of a token's keys or values: divided by it,
// the largest is below 2^13.  That of the largest of 32, most, or the token's
// own where some lie more than `apart` orders below (at most kMostOrders then:
// a weight times 2^kMostOrders is an f32).  scale, mid: of the lane's token.
constexpr int kMostOrders = 100;
struct Exponent {
  int most, mine;
  bool own;
};
template <int G>
__device__ __forceinline__ Exponent exponentOf32(const float (&scale)[G], const float (&mid)[G], int apart) {
  float top = 0.0f;
#pragma unroll
  for (int g = 0; g < G; g++) top = fmaxf(top, fmaf(8.5f, fabsf(scale[g]), fabsf(mid[g])));
  // positive floats are ordered like their bits
  const int most = exponentOf(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top)))), mine = exponentOf(top);
  const bool own = __any_sync(~0u, top > 0.0f && mine < most - apart);
  const int e = max(most - 12, kLeastExponent);
  return {e, own ? max(max(mine - 12, kLeastExponent), e - kMostOrders) : e, own};
}

// A token's row of codes with its parameters; a key thread has those of the
// values too (it writes down what the softmax needs of both, before the scores
// can be there).
template <int G>
struct RawToken {
  uint32_t w[8 * G], keyParams[G], valueParams[G];
  bool there;
};

// Registers a thread, of the 128 that each of the four warpgroups starts with.
constexpr int kSoftmaxRegisters = 160, kWidenRegisters = 112, kIssueRegisters = 80;
static_assert(2 * kSoftmaxRegisters + kWidenRegisters + kIssueRegisters == 4 * 128, "what one gives the others take");
template <int N>
__device__ __forceinline__ void moreRegisters() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewerRegisters() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// The products of row tile T, by one warp: all of it waits, one thread issues.
// The block has all 512 columns of TMEM, from column 0 on, so places in it are
// constants.
template <int G, int T>
__device__ __forceinline__ void issueProducts(const AttnArgs& p, const int* starts, int units, const uint8_t* smem, ChunkControl& ctl) {
  constexpr int D = 64 * G;
  using L = ChunkSmem<G>;
  constexpr uint32_t kScores = idescF16(128, kChunkKeys, false), kOutputs = idescF16(128, D, true);
  constexpr uint32_t kQStep = L::kQBlock >> 4, kStep = L::kBlock >> 4;
  volatile int* abortFlag = &ctl.abort;
  // Words of the descriptors: addresses count 16 bytes.
  const uint64_t rows = sm100::smemDescSw128(0), plain = smemDescPlain(0), major = smemDescMn(0);
  const uint32_t rowsHi = static_cast<uint32_t>(rows >> 32), plainHi = static_cast<uint32_t>(plain >> 32), majorHi = static_cast<uint32_t>(major >> 32);
  const uint32_t base = sm100::smemAddr(smem) >> 4;
  const uint32_t q = static_cast<uint32_t>(rows) + base + (L::kQ >> 4) + T * G * kQStep;
  const uint32_t qSums = static_cast<uint32_t>(plain) + base + (L::kQSums >> 4) + T * (128 * 32 >> 4);
  uint32_t seq = 0, qCount = 0, sCount = 0, pCount = 0;
  // Scores of the keys in a stage, to the place that is free.
  auto issueScores = [&](uint32_t st) {
    const uint32_t d = T * 128 + (sCount & 1) * 64;
    const uint32_t k = static_cast<uint32_t>(rows) + base + (L::kK >> 4) + st * (G * kStep);
    const uint32_t kSums = static_cast<uint32_t>(plain) + base + (L::kKSums >> 4) + st * (64 * 32 >> 4);
    if (sm100::electOne()) {
      mmaF16<false>(d, q, rowsHi, k, rowsHi, kScores);
#pragma unroll
      for (int i = 1; i < 4 * G; i++)
        mmaF16<true>(d, q + (i >> 2) * kQStep + 2 * (i & 3), rowsHi, k + (i >> 2) * kStep + 2 * (i & 3), rowsHi, kScores);
      mmaF16<true>(d, qSums, plainHi, kSums, plainHi, kScores);
      sm100::mmaCommit(&ctl.sFull[T][sCount & 1]);
      sm100::mmaCommit(&ctl.kEmpty[st]);
    }
    __syncwarp();
    sCount++;
  };
  bool ok = true;
  for (int round = 0, u = unitOfRound(0); u < units && ok; u = unitOfRound(++round)) {
    const ChunkUnit c = chunkUnit(p, starts, u);
    const int n = c.upto - c.from;
    if (T >= c.tiles) {  // nothing of this row tile: its share of every stage is let go once it is there
      for (int j = 0; j < n && ok; j++, seq++) {
        const uint32_t st = seq & 3, parity = (seq >> 2) & 1u;
        ok = warpWait(&ctl.kFull[st], parity, abortFlag) && warpWait(&ctl.vFull[st], parity, abortFlag);
        if (ok && sm100::electOne()) {
          sm100::mbarArrive(&ctl.kEmpty[st]);
          sm100::mbarArrive(&ctl.vEmpty[st]);
        }
        __syncwarp();
      }
      continue;
    }
    if (n <= 0) continue;
    ok = warpWait(&ctl.qFull[T], qCount++ & 1u, abortFlag);
    for (int i = 0; i < 2 && i < n && ok; i++) {
      const uint32_t s = seq + i;
      ok = warpWait(&ctl.kFull[s & 3], (s >> 2) & 1u, abortFlag);
      if (!ok) break;
      sm100::tcFenceAfter();
      issueScores(s & 3);
    }
    for (int j = 0; j < n && ok; j++, seq++) {
      const uint32_t st = seq & 3, place = pCount & 1, weights = T * 128 + place * 64;
      ok = warpWait(&ctl.pFull[T][place], (pCount >> 1) & 1u, abortFlag) && warpWait(&ctl.vFull[st], (seq >> 2) & 1u, abortFlag);
      if (!ok) break;
      pCount++;
      sm100::tcFenceAfter();
      const uint32_t v = static_cast<uint32_t>(major) + base + (L::kV >> 4) + st * (G * kStep);
      if (sm100::electOne()) {
#pragma unroll
        for (int k = 0; k < kChunkKeys / 16; k++)
          mmaF16Tmem(256 + T * D, weights + 8 * k, v + 128 * k, majorHi, kOutputs, k > 0 ? 1u : static_cast<uint32_t>(j));
        sm100::mmaCommit(&ctl.pvDone[T][place]);
        sm100::mmaCommit(&ctl.vEmpty[st]);
      }
      __syncwarp();
      if (j + 2 < n) {
        const uint32_t far = (seq + 2) & 3;
        ok = warpWait(&ctl.kFull[far], ((seq + 2) >> 2) & 1u, abortFlag);
        if (!ok) break;
        sm100::tcFenceAfter();
        issueScores(far);
      }
    }
  }
  // Every product and arrival that was issued ends before the block does: the
  // barriers' memory is the next block's.
  if (sm100::electOne()) sm100::mmaCommit(&ctl.drain[T]);
  __syncwarp();
  volatile int never = 0;
  sm100::mbarWait(&ctl.drain[T], 0, &never, 200000000ull);
}

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
    for (int i = 0; i < kChunkStages; i++) {
      sm100::mbarInit(&ctl.kFull[i], 64);
      sm100::mbarInit(&ctl.kEmpty[i], 2);
      sm100::mbarInit(&ctl.vFull[i], 64);
      sm100::mbarInit(&ctl.vEmpty[i], 2);
    }
    for (int i = 0; i < 2; i++) {
      sm100::mbarInit(&ctl.qFull[i], 128);
      sm100::mbarInit(&ctl.sFull[i][0], 1);
      sm100::mbarInit(&ctl.sFull[i][1], 1);
      sm100::mbarInit(&ctl.pFull[i][0], 128);
      sm100::mbarInit(&ctl.pFull[i][1], 128);
      sm100::mbarInit(&ctl.pvDone[i][0], 1);
      sm100::mbarInit(&ctl.pvDone[i][1], 1);
    }
    sm100::mbarInit(&ctl.drain[0], 1);
    sm100::mbarInit(&ctl.drain[1], 1);
    ctl.abort = 0;
    sm100::fenceBarrierInit();
  }
  if (warp == 12) {
    sm100::tmemAlloc(&ctl.tmem, 512);
    sm100::tmemRelinquish();
  }
  // Units before each request: one warp, 32 requests a step.  Starts that fall
  // back give the same rows to several requests; units past those that the
  // scratch was made for are left out.
  if (warp == 0) {
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int b = base + lane;
      long long v = b < p.batch ? chunkUnitsOf(p, requestOf(p, b)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += x;
      }
      const int upto = static_cast<int>(min(before + v, static_cast<long long>(p.unitsMost)));
      if (b < p.batch) starts[b + 1] = upto;
      before = __shfl_sync(~0u, upto, 31);
    }
    if (lane == 0) starts[0] = 0;
  }
  sm100::tcFenceBefore();
  __syncthreads();
  sm100::tcFenceAfter();
  const uint32_t tmem = ctl.tmem;
  if (threadIdx.x == 0 && tmem != 0) ctl.abort = 1;  // all columns start at the first
  const int units = starts[p.batch];
  constexpr uint32_t kOut = 256;  // columns of the outputs, behind two times 128 of scores

  if (warp < 8) {
    // ---------------- softmax ----------------
    moreRegisters<kSoftmaxRegisters>();
    const int t = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t output = tmem + kOut + t * D + lanes;
    uint32_t seq = 0;    // tiles of keys of the block so far: the place of their info
    uint32_t count = 0;  // of those, the ones with this row tile
    float unit = 1.0f;   // what a score counts in the base-2 logarithm
    int limit = 0;       // keys that the row sees
    // A unit's queries: the row's channels, scaled to 2^8, and their sums as
    // the left operand.
    auto loadQuery = [&](const ChunkUnit& c) {
      const int mine = c.row0 + t * 128 + row;
      const bool live = mine < c.r.rows * p.group;
      const int token = live ? mine / p.group : 0, h = c.head * p.group + (live ? mine - token * p.group : 0);
      limit = live ? min(max(c.r.kv - c.r.rows + token + 1, 0), c.r.kv) : c.r.kv;
      float amax = 0.0f, sums[G] = {};
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + static_cast<long long>(c.r.start + token) * p.qTok + static_cast<long long>(h) * p.qHead;
      uint4 raw[8 * G];
#pragma unroll
      for (int i = 0; i < 8 * G; i++) raw[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 8 * G; i++) {
        float x[8];
        if (p.half16) unpack8<__half>(raw[i], x);
        else unpack8<__nv_bfloat16>(raw[i], x);
#pragma unroll
        for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
      }
      const int e = exponentOf(amax);
      const bool plain = e > 127 || e < -118;  // not finite; counts as zero
      const float f = (plain ? 1.0f : powerOfTwo(8 - e)) * (p.scaleLog2 < 0.0f ? -1.0f : 1.0f);
      unit = (plain ? 1.0f : powerOfTwo(e - 8)) * fabsf(p.scaleLog2);
#pragma unroll
      for (int i = 0; i < 8 * G; i++) {
        float x[8];
        if (p.half16) unpack8<__half>(raw[i], x);
        else unpack8<__nv_bfloat16>(raw[i], x);
#pragma unroll
        for (int k = 0; k < 8; k++) {
          x[k] *= f;
          sums[i / 8] += x[k];
        }
        *reinterpret_cast<uint4*>(smem + L::kQ + (t * G + i / 8) * L::kQBlock + row * 128 + (((i & 7) ^ (row & 7)) << 4)) = pack8<__half>(x);
      }
      storeSums<G, true>(smem + L::kQSums + t * (128 * 32), row, sums);
      sm100::fenceProxyAsyncShared();
      sm100::mbarArrive(&ctl.qFull[t]);
    };
    // The next unit with keys for this row tile, from unit u on; its queries
    // are loaded as soon as the last scores of the unit before are there.
    bool ok = true;
    int round = 0, u = unitOfRound(0);
    if (u < units) {
      const ChunkUnit c = chunkUnit(p, starts, u);
      if (t < c.tiles && c.from < c.upto) loadQuery(c);
    }
    for (; u < units && ok; u = unitOfRound(++round)) {
      const ChunkUnit c = chunkUnit(p, starts, u);
      const bool any = t < c.tiles && c.from < c.upto;
      const int mineLimit = limit;
      const float mineUnit = unit;
      RowState state = {kNone, 0.0f, static_cast<float>(kLeastExponent), 0};
      if (!any) {
        seq += c.upto - c.from;
      } else {
        for (int j = c.from; j < c.upto; j++, seq++, count++) {
          const uint32_t scores = tmem + t * 128 + (count & 1) * 64 + lanes;
          ok = warpWait(&ctl.sFull[t][count & 1], (count >> 1) & 1u, abortFlag);
          if (!ok) break;
          sm100::tcFenceAfter();
          const ChunkInfo& info = ctl.info[seq & 7];
          const int left = mineLimit - j * kChunkKeys;  // keys of the tile in the row's range
          uint64_t* before = &ctl.pvDone[t][(count - 1) & 1];
          const uint32_t parity = ((count - 1) >> 1) & 1u;
          const uint32_t kind = info.kind[0] | info.kind[1];
          if (!__any_sync(~0u, left < kChunkKeys || kind != 0)) {
            ok = tileSoftmax<G, false, false>(state, scores, output, info, mineUnit, left, j == c.from, before, parity, abortFlag);
          } else if (kind <= kUneven) {
            ok = tileSoftmax<G, true, false>(state, scores, output, info, mineUnit, left, j == c.from, before, parity, abortFlag);
          } else {
            const Followed f = ownSoftmax<G>(state, scores, output, &info, mineUnit, left, j == c.from, before, parity, abortFlag);
            state = f.row;
            ok = f.ok;
          }
          if (!ok) break;
          tmemStoreWait();
          sm100::tcFenceBefore();
          sm100::mbarArrive(&ctl.pFull[t][count & 1]);
        }
      }
      if (!ok) break;
      if (unitOfRound(round + 1) < units) {
        const ChunkUnit next = chunkUnit(p, starts, unitOfRound(round + 1));
        if (t < next.tiles && next.from < next.upto) loadQuery(next);
      }
      // The result, or this share of it.
      if (t >= c.tiles || (!any && p.splits > 1)) continue;  // an empty share counts as absent
      if (any) {
        ok = warpWait(&ctl.pvDone[t][(count - 1) & 1], ((count - 1) >> 1) & 1u, abortFlag);
        if (!ok) break;
        sm100::tcFenceAfter();
      }
      const int mine = c.row0 + t * 128 + row;
      const bool live = mine < c.r.rows * p.group;
      const int token = live ? mine / p.group : 0, h = c.head * p.group + (live ? mine - token * p.group : 0);
      const float m = state.m, l = state.l;
      const bool whole = p.splits == 1, none = l == 0.0f;
      const float factor = (whole ? (none ? 0.0f : 1.0f / l) : 1.0f) * exp2Fast(state.ref);
      const long long slot = static_cast<long long>(u) * kChunkRows + t * 128 + row;
#pragma unroll 1
      for (int k = 0; k < D / 32; k++) {
        uint32_t o[32];
        float y[32];
        if (any) {  // the whole warp or none of it
          tmemLoad32(output + 32 * k, o);
          sm100::tmemLoadWait();
        }
        const bool spoilt = (state.poison >> (k / 2)) & 1u;
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
    fewerRegisters<kWidenRegisters>();
    const bool keys = warp < 10;
    const int tid = threadIdx.x & 63, w = warp & 1;
    // The tile after next: its token's page number is under way.
    int round = 0, u = unitOfRound(0), j = 0, upto = 0, head = 0, kv = 0;
    const int* pages = nullptr;
    bool exists = false;
    int token = 0, page = -1;
    const int pageTokens = p.blocksPerPage * 16;
    auto pageOfToken = [&](int x) { return p.pageShift >= 0 ? x >> p.pageShift : x / pageTokens; };
    auto advance = [&]() {
      j++;
      while (j >= upto) {
        if (u >= units) {
          exists = false;
          return;
        }
        const ChunkUnit c = chunkUnit(p, starts, u);
        u = unitOfRound(++round);
        j = c.from;
        upto = c.upto;
        head = c.head;
        kv = c.r.kv;
        pages = p.table + static_cast<long long>(c.b) * p.width;
      }
      exists = true;
      token = j * kChunkKeys + tid;
      page = token < kv ? pages[pageOfToken(token)] : -1;
    };
    auto fetch = [&](RawToken<G>& r) {
      r.there = exists && page >= 0 && page < p.pages;
      const int place = token - pageOfToken(token) * pageTokens, at = place & 15;
      const uint8_t* block = p.cache + ((static_cast<long long>(r.there ? page : 0) * p.kvHeads + head) * p.blocksPerPage + (place >> 4)) * (18 * D);
      const uint4* codes = reinterpret_cast<const uint4*>(block + (keys ? at : 16 + kv4::valueRow(at)) * (D / 2));
#pragma unroll
      for (int i = 0; i < 2 * G; i++) {
        uint4 a = make_uint4(0, 0, 0, 0);  // codes of 0 with nothing to scale
        if (r.there) a = __ldg(codes + i);
        r.w[4 * i] = a.x;
        r.w[4 * i + 1] = a.y;
        r.w[4 * i + 2] = a.z;
        r.w[4 * i + 3] = a.w;
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        r.keyParams[g] = r.there && keys ? __ldg(reinterpret_cast<const uint32_t*>(block + 16 * D + at * (4 * G)) + g) : 0;
        r.valueParams[g] = r.there ? __ldg(reinterpret_cast<const uint32_t*>(block + 17 * D + at * (4 * G)) + g) : 0;
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
      const int st = seq & 3;
      const uint32_t parity = ((seq >> 2) & 1u) ^ 1u;
      float s[G], m[G];
      uint32_t bad[G];
#pragma unroll
      for (int g = 0; g < G; g++) {
        s[g] = kv4::bf16Lo(raw.valueParams[g]);
        m[g] = kv4::bf16Hi(raw.valueParams[g]);
        const bool odd = !(isfinite(s[g]) && isfinite(m[g]));
        if (odd) s[g] = m[g] = 0.0f;
        bad[g] = __ballot_sync(~0u, odd);
      }
      const Exponent ve = exponentOf32<G>(s, m, kValuesApart);
      if (keys) {
#pragma unroll
        for (int g = 0; g < G; g++) {
          s[g] = kv4::bf16Lo(raw.keyParams[g]);
          m[g] = kv4::bf16Hi(raw.keyParams[g]);
        }
        const Exponent ke = exponentOf32<G>(s, m, kKeysApart);
        const float f = powerOfTwo(-ke.mine);
#pragma unroll
        for (int g = 0; g < G; g++) {
          s[g] *= f;
          m[g] = fmaf(0.5f, s[g], m[g] * f);  // value = m + s (code - 8) from here on
        }
        const uint32_t present = __ballot_sync(~0u, raw.there);
        if (!warpWait(&ctl.kEmpty[st], parity, abortFlag)) break;
        ChunkInfo& info = ctl.info[seq & 7];
        if (ke.own) info.keyOrder[tid] = static_cast<uint8_t>(127 + ke.mine - ke.most);
        if (ve.own) info.valueOrder[tid] = static_cast<uint8_t>(127 + ve.mine - ve.most);
        if (lane == 0) {
          info.valid[w] = present;
          info.keyUnit[w] = powerOfTwo(ke.most);
          info.valueExp[w] = static_cast<float>(ve.most);
          info.kind[w] = (present != ~0u || bad[0] != 0 || bad[G - 1] != 0 ? kUneven : 0) | (ke.own ? kOwnKeys : 0) | (ve.own ? kOwnValues : 0);
#pragma unroll
          for (int g = 0; g < 2; g++) info.bad[g][w] = g < G ? bad[g < G ? g : 0] : 0;
        }
        widen<G, true>(raw.w, s, m, smem + L::kK + st * G * L::kBlock, tid);
        storeSums<G, false>(smem + L::kKSums + st * (64 * 32), tid, m);
        sm100::fenceProxyAsyncShared();
        sm100::mbarArrive(&ctl.kFull[st]);
      } else {
        const float f = powerOfTwo(-ve.mine);
#pragma unroll
        for (int g = 0; g < G; g++) {
          s[g] *= f;
          m[g] = fmaf(0.5f, s[g], m[g] * f);
        }
        if (!warpWait(&ctl.vEmpty[st], parity, abortFlag)) break;
        widen<G, false>(raw.w, s, m, smem + L::kV + st * G * L::kBlock, tid);
        sm100::fenceProxyAsyncShared();
        sm100::mbarArrive(&ctl.vFull[st]);
      }
      raw = next;
      here = follows;
    }
  } else {
    fewerRegisters<kIssueRegisters>();
    if (warp == 12) issueProducts<G, 0>(p, starts, units, smem, ctl);
    if (warp == 13) issueProducts<G, 1>(p, starts, units, smem, ctl);
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
    if (s * each >= all || first + s >= p.chunkStarts[b + 1]) break;
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

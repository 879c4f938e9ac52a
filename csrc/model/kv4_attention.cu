// SPDX-License-Identifier: Apache-2.0
// Attention of ragged query rows over the 4-bit paged cache.
//
// Mathematics.  With value = mid + scale (code - 7.5) for each token and group
// of 64 channels,
//   q . k_t = sum_g [ scale_tg (q_g . c_tg) + (mid_tg - 7.5 scale_tg) sum(q_g) ]
//   sum_t p_t v_t = sum_t (p_t scale_tg) (c_tg - 7.5) + sum_t p_t mid_tg
// so the tensor cores multiply the codes themselves, and scale and midpoint
// act on accumulators and on the softmax weights.  A code c read as an f16
// bit pattern is the subnormal c * 2^-24 (its neighbour in bits 4-7 is
// 16 c * 2^-24), exact in the tensor cores' products; one AND makes a pair
// of operands.  Query rows are scaled by a power of two and held in f16,
// which is exact for bf16 and f16 inputs but for channels below 2^-26 of the
// row's largest.  The weights p_t scale_tg are rounded to f16 (11 bits) in
// units of the largest one that the row has met, so a large value that a row
// does not see, or gives no weight, costs the others nothing (with a unit for
// all rows from the scales alone, one value 2^20 above the rest left a tenth
// of error); the sum of the rounded ones, which the 7.5 multiplies, is a
// product with ones on the tensor cores.  Everything else is f32.
//
// Shape.  S^T = K Q^T: rows of the m16n8k16 products are 16 tokens, columns 8
// query rows (a query row is one head of one token; the heads that share a key
// head stand together), so a group of 8 heads fills the tile.  O^T = V^T P^T
// the same way; movmatrix turns the accumulator of S^T into the operand P^T.
//
// Work.  A unit is a request, a key head and R = 8 * NT query rows; its
// length is the request's tokens in tiles of 32.  The tiles of all units in a
// row are cut into equal ranges, one for each warp of the grid, whatever the
// lengths are; a warp that gets a whole unit writes the result, the others
// write partial sums (unnormalised output, maximum, sum) that a second kernel
// joins in order.
//
// Measured: 140 us, 4.3 TB/s of cache, for 64 requests of 500 to 16000 tokens,
// 64 heads on 8; the widening of codes bounds it (280 instructions a block of
// 16 tokens, almost half of them on the ALU pipe).  One request of 900 tokens takes
// 12 us, which is the latency of two launches and eight dependent loads.
#include <cfloat>
#include <climits>
#include <mutex>

#include "kernels/kv4.cuh"
#include "model/common.cuh"
#include "vccl_x.h"

namespace vccl {
namespace model {
namespace {

constexpr int kTile = 32;          // tokens that a warp takes in one step
constexpr int kWarps = 12;         // per block, one block per SM
constexpr int kStages = 3;         // tiles that a warp has in shared memory
constexpr int kBlocks = kTile / kv4::kBlockTokens;  // blocks in a tile
constexpr int kMaxBatch = 4096;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNone = -1e30f;    // a maximum over nothing
// Weights in f16: the largest p * scale that a look finds becomes 4; until the
// next look p grows by 2^8 at most, and scales by what keeps p * scale below
// 2^15.  The factor that makes it so stays where f32 holds all products.
constexpr float kWeightTop = 4.0f, kScaleRoom = 128.0f, kFactorMost = 0x1p118f, kFactorLeast = 0x1p-120f;

struct AttnArgs {
  const void* q;
  long long qTok, qHead;
  const uint8_t* cache;
  const int* table;
  const int* kvLens;
  const int* qStarts;
  void* out;
  long long oTok, oHead;
  float* lse;
  long long* prefix;  // [batch + 1] tiles before each request (written by block 0)
  float2* stats;      // [2 * workers][R] maximum (log2), sum
  float* partial;     // [2 * workers][R][D]
  int width, batch, tokens, qHeads, kvHeads, group, pages, blocksPerPage;
  int pageShift;  // tokens of a page = 1 << pageShift, or -1
  int workers, half16, zeroTail;
  float scaleLog2;
  // Requests of at least longRows query rows a key head go to chunkKernel (0: none do).
  int longRows, splits;
  int unitsMost;        // that the scratch has room for; requests that do not overlap have no more
  int* chunkStarts;     // [batch + 1] units before each request
  float2* chunkStats;   // [units][256] maximum (log2), sum, with splits > 1
  float* chunkPartial;  // [units][256][D]
  int* errorFlag;       // mapped host word, set when a wait ran out
};

// What a request brings: its first row, its rows, its tokens.
struct Request {
  int start, rows, kv;
};

__device__ __forceinline__ Request requestOf(const AttnArgs& p, int b) {
  const int s = min(max(p.qStarts[b], 0), p.tokens), e = min(max(p.qStarts[b + 1], s), p.tokens);
  const long long most = static_cast<long long>(p.width) * p.blocksPerPage * kv4::kBlockTokens;
  return {s, e - s, static_cast<int>(min(static_cast<long long>(max(p.kvLens[b], 0)), most))};
}

__device__ __forceinline__ bool isLong(const AttnArgs& p, const Request& r) {
  return p.longRows > 0 && static_cast<long long>(r.rows) * p.group >= p.longRows;
}

__device__ __forceinline__ int unitsOf(const AttnArgs& p, const Request& r, int R) {
  if (isLong(p, r)) return 0;
  const long long rows = static_cast<long long>(r.rows) * p.group;
  return static_cast<int>((rows + R - 1) / R);
}

__device__ __forceinline__ int tilesOf(const Request& r) { return (r.kv + kTile - 1) / kTile; }

// A quotient that is mostly one of 32-bit numbers (a 64-bit division takes
// over a hundred instructions).
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// Tiles to warps: every warp that takes part has `each` tiles, the first
// `more` of them one more.
struct Split {
  int workers;
  long long each, more;
  __device__ __forceinline__ Split(long long total, int most) {
    workers = static_cast<int>(min(static_cast<long long>(most), total));
    each = quotient(total, workers);
    more = total - each * workers;
  }
  __device__ __forceinline__ long long start(int w) const { return w * each + min(static_cast<long long>(w), more); }
  __device__ __forceinline__ int owner(long long tile) const {
    const long long ahead = more * (each + 1);
    return static_cast<int>(tile < ahead ? quotient(tile, each + 1) : more + quotient(tile - ahead, each));
  }
};

// prefix[b] = tiles of the requests before b (all heads and row tiles).
template <int THREADS>
__device__ void scanTiles(const AttnArgs& p, int R, long long* prefix) {
  __shared__ long long warpSums[THREADS / 32];
  __shared__ long long carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    carry = 0;
    prefix[0] = 0;
  }
  __syncthreads();
  for (int base = 0; base < p.batch; base += THREADS) {
    const int b = base + threadIdx.x;
    long long v = 0;
    if (b < p.batch) {
      const Request r = requestOf(p, b);
      v = static_cast<long long>(unitsOf(p, r, R)) * p.kvHeads * tilesOf(r);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warpSums[warp] = v;
    __syncthreads();
    long long before = carry;
    for (int i = 0; i < warp; i++) before += warpSums[i];
    if (b < p.batch) prefix[b + 1] = before + v;
    __syncthreads();
    if (threadIdx.x == THREADS - 1) carry = before + v;
    __syncthreads();
  }
}

__device__ __forceinline__ int findRequest(const long long* prefix, int batch, long long tile) {
  int lo = 0, hi = batch - 1;  // the last b with prefix[b] <= tile whose tiles are not all before
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (prefix[m + 1] > tile) hi = m;
    else lo = m + 1;
  }
  return lo;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void mmaFirst(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t packHalf(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float exp2Fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Shared memory by its 32-bit address: one register and an immediate.
template <int WORDS>
__device__ __forceinline__ void loadWords(uint32_t at, uint32_t* w) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

// A block in shared memory is as in global memory, but that for D = 128 the
// 16-byte chunks of value rows 4i + 2 and 4i + 3 change places in twos: lanes
// of four rows then read from different banks.
__device__ __forceinline__ int swapTwos(int chunk) { return chunk ^ ((chunk & 8) >> 2); }

// to: of the block, plus 16 * lane; from: likewise.
template <int G>
__device__ __forceinline__ void copyBlock(uint32_t to, const uint8_t* from, int lane) {
  constexpr int D = 64 * G, kChunks = 18 * D / 16;
  const uint32_t swapped = to + 16 * (swapTwos(lane) - lane);
#pragma unroll
  for (int j = 0; j < (kChunks + 31) / 32; j++) {
    const bool values = G == 2 && j >= D / 64 && j < D / 32;  // chunks D / 2 to D
    if (32 * (j + 1) <= kChunks || 32 * j + lane < kChunks)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((values ? swapped : to) + 512 * j), "l"(from + 512 * j) : "memory");
  }
}

// What a lane reads of a block: of keys, tokens g and g + 8, words (group,
// half); of values, tokens 2q, 2q + 1, 8 + 2q, 9 + 2q, the word of each group;
// scales and midpoints of tokens g and g + 8.
struct LaneOffsets {
  uint32_t keys, params, values;
};

template <int G>
__device__ __forceinline__ LaneOffsets offsetsOf(int lane) {
  constexpr int D = 64 * G;
  const int g = lane >> 2, q = lane & 3;
  return {static_cast<uint32_t>(g * (D / 2) + q * (8 * G)), static_cast<uint32_t>(g * (4 * G)),
          static_cast<uint32_t>(q * (D / 2) + (G == 2 ? (g * 8) ^ ((q & 2) << 4) : g * 4))};
}

template <int G>
__device__ __forceinline__ void readKeys(uint32_t (&k)[2][2 * G], uint32_t (&kp)[2][G], uint32_t block, const LaneOffsets& at) {
  constexpr int D = 64 * G;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    loadWords<2 * G>(block + at.keys + 4 * i * D, k[i]);
    loadWords<G>(block + at.params + 16 * D + 32 * G * i, kp[i]);
  }
}

template <int G>
__device__ __forceinline__ void readValueParams(uint32_t (&vp)[2][G], uint32_t block, const LaneOffsets& at) {
#pragma unroll
  for (int i = 0; i < 2; i++) loadWords<G>(block + at.params + 17 * 64 * G + 32 * G * i, vp[i]);
}

template <int G>
__device__ __forceinline__ void readValues(uint32_t (&v)[4][G], uint32_t block, const LaneOffsets& at) {
  constexpr int D = 64 * G;
#pragma unroll
  for (int i = 0; i < 4; i++) loadWords<G>(block + at.values + 8 * D + 2 * i * D, v[i]);
}

// A warp's state for one unit.
template <int G, int NT>
struct Unit {
  uint32_t qb[NT][G][4][2];  // Q^T operands: word half h, code pair u -> [2h + u]
  float qs[NT][2];           // log2(e) * scale * 2^24 / (power of two of the row), rows 2q and 2q + 1
  float sq[NT][G][2];        // sum of the row's group, in units of qs
  int limit[NT][2];          // tokens that the row sees
  int most, least;           // of all rows of the unit
  float m[NT][2], l[NT][2];
  float o[NT][G][4][4];      // 2^-24 * by * sum p' c; odd j: of c + 16 c', c that of j - 1
  float ones[NT][G][4];      // by * sum p', of the tokens whose codes have their middle in o
  float mid[NT][G][2];       // sum p mid
  float by[NT][G][2];        // p' = p scale is held as by * p' in f16
  float lim[G];              // the scale above which by is looked at
};

template <int G, int NT>
__device__ __forceinline__ void loadQuery(Unit<G, NT>& u, const AttnArgs& p, const Request& r, int head, int row0,
                                          int lane) {
  const int g = lane >> 2, q = lane & 3;
  int most = 0, least = INT_MAX;
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const long long row = static_cast<long long>(row0) + 8 * n + g;
    const bool live = row < static_cast<long long>(r.rows) * p.group;
    const int i = live ? static_cast<int>(row / p.group) : 0, h = head * p.group + (live ? static_cast<int>(row % p.group) : 0);
    float x[G][16];
    float amax = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
      uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (live) {
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + (r.start + i) * p.qTok + h * p.qHead + 64 * gr + 16 * q;
        v[0] = *reinterpret_cast<const uint4*>(src);
        v[1] = *reinterpret_cast<const uint4*>(src + 8);
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float y[8];
        if (p.half16) unpack8<__half>(v[j], y);
        else unpack8<__nv_bfloat16>(v[j], y);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x[gr][8 * j + e] = y[e];
          amax = fmaxf(amax, fabsf(y[e]));
        }
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
    // f = 2^(12 - exponent of the largest), 1 / f beside it; a row below 2^-114
    // counts as zero, one that is not finite stays so.
    const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    const bool plain = e > 127 || e < -114;
    const float f = plain ? 1.0f : __uint_as_float(static_cast<uint32_t>(127 + 12 - e) << 23);
    const float back = plain ? 1.0f : __uint_as_float(static_cast<uint32_t>(127 - 12 + e) << 23);
    float qs = back * p.scaleLog2 * 16777216.0f;
    float sq[G];
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j++) s = fmaf(x[gr][j], f, s);
      s += __shfl_xor_sync(~0u, s, 1);
      s += __shfl_xor_sync(~0u, s, 2);
      sq[gr] = s * 5.9604644775390625e-8f;
#pragma unroll
      for (int w = 0; w < 4; w++) {  // word half w / 2, code pair w % 2: channels 4w .. 4w + 3 of the lane's 16
        const float* y = &x[gr][4 * w];
        u.qb[n][gr][w][0] = packHalf(y[0] * f, y[1] * f);
        u.qb[n][gr][w][1] = packHalf(y[2] * f * 0.0625f, y[3] * f * 0.0625f);
      }
    }
    // A row behind the last one is computed like the last one, and not stored.
    const int lim = live ? max(r.kv - r.rows + i + 1, 0) : r.kv;
    // Columns 2q and 2q + 1 of the accumulators belong to the rows of lanes 8q and 8q + 4.
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int src = 4 * (2 * q + c);
      u.qs[n][c] = __shfl_sync(~0u, qs, src);
      u.limit[n][c] = min(__shfl_sync(~0u, lim, src), r.kv);
#pragma unroll
      for (int gr = 0; gr < G; gr++) u.sq[n][gr][c] = __shfl_sync(~0u, sq[gr], src);
      u.m[n][c] = kNone;
      u.l[n][c] = 0.0f;
      most = max(most, u.limit[n][c]);
      least = min(least, u.limit[n][c]);
#pragma unroll
      for (int gr = 0; gr < G; gr++) {
        u.mid[n][gr][c] = 0.0f;
        u.by[n][gr][c] = kFactorMost;
      }
    }
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        u.ones[n][gr][j] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) u.o[n][gr][j][k] = 0.0f;
      }
    }
  }
#pragma unroll
  for (int gr = 0; gr < G; gr++) u.lim[gr] = kScaleRoom / kFactorMost;
  most = max(most, __shfl_xor_sync(~0u, most, 1));
  u.most = max(most, __shfl_xor_sync(~0u, most, 2));
  least = min(least, __shfl_xor_sync(~0u, least, 1));
  u.least = min(least, __shfl_xor_sync(~0u, least, 2));
}

// The two bytes of a word's upper halves, each in the low byte of 16 bits.
__device__ __forceinline__ uint32_t upperBytes(uint32_t w) { return __byte_perm(w, 0u, 0x4341); }

// The second half of a tile: weights of the scores x, and their products with
// the values.  EDGE: some row does not see some token.
template <int G, int NT, bool EDGE>
__device__ __forceinline__ void weighValues(Unit<G, NT>& u, float (&x)[kBlocks][NT][4], const float (&s)[kBlocks][2][G],
                                            const float (&mid)[kBlocks][2][G], uint32_t tile, const LaneOffsets& at) {
  constexpr int D = 64 * G, B = kBlocks;
#pragma unroll
  for (int b = 0; b < B; b++) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const float w = exp2Fast(x[b][n][2 * i + c]);
          x[b][n][2 * i + c] = w;
          u.l[n][c] += w;
          if (!EDGE || w != 0.0f) {  // a row must not meet a NaN of a token that it does not see
#pragma unroll
            for (int gr = 0; gr < G; gr++) u.mid[n][gr][c] = fmaf(w, mid[b][i][gr], u.mid[n][gr][c]);
          }
        }
    // O^T: rows are channels 8g + 2j (from the low halves of the words) and
    // 8g + 2j + 1.  Odd j take a byte's two codes together, c + 16 c': the end
    // takes c back out.
    uint32_t v[4][G];
    readValues<G>(v, tile + b * 18 * D, at);
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        // p * by first: it is finite, and nothing where p is, whatever the scale
        const uint64_t by = pair(u.by[n][gr][0], u.by[n][gr][1]);
        const float2 w01 = unpair(mul2(mul2(pair(x[b][n][0], x[b][n][1]), by), pair(s[b][0][gr])));
        const float2 w23 = unpair(mul2(mul2(pair(x[b][n][2], x[b][n][3]), by), pair(s[b][1][gr])));
        float w[4] = {w01.x, w01.y, w23.x, w23.y};
        if (EDGE) {
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = x[b][n][k] == 0.0f ? 0.0f : w[k];
        }
        b0[n] = transpose8x8(packHalf(w[0], w[1]));
        b1[n] = transpose8x8(packHalf(w[2], w[3]));
        mma(u.ones[n][gr], 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, b0[n], b1[n]);
      }
      const uint32_t x0 = __byte_perm(v[0][gr], v[1][gr], 0x5410), y0 = __byte_perm(v[0][gr], v[1][gr], 0x7632);
      const uint32_t x1 = __byte_perm(v[2][gr], v[3][gr], 0x5410), y1 = __byte_perm(v[2][gr], v[3][gr], 0x7632);
      const uint32_t xs0 = upperBytes(x0), ys0 = upperBytes(y0), xs1 = upperBytes(x1), ys1 = upperBytes(y1);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        mma(u.o[n][gr][0], x0 & 0x000F000Fu, y0 & 0x000F000Fu, x1 & 0x000F000Fu, y1 & 0x000F000Fu, b0[n], b1[n]);
        mma(u.o[n][gr][1], x0 & 0x00FF00FFu, y0 & 0x00FF00FFu, x1 & 0x00FF00FFu, y1 & 0x00FF00FFu, b0[n], b1[n]);
        mma(u.o[n][gr][2], xs0 & 0x000F000Fu, ys0 & 0x000F000Fu, xs1 & 0x000F000Fu, ys1 & 0x000F000Fu, b0[n], b1[n]);
        mma(u.o[n][gr][3], xs0, ys0, xs1, ys1, b0[n], b1[n]);
      }
    }
  }
}

// Of two pairs of bf16, a without signs: the larger sizes.  Two instructions a
// word, where scales already in f32 took three microseconds of 140 more.
__device__ __forceinline__ uint32_t maxSizes(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{ .reg .b32 s; abs.bf16x2 s, %2; max.bf16x2 %0, %1, s; }" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Takes the middle of the codes out of the sums.  The tensor cores drop what is
// below the last bit of an f32 sum, every step in the same direction, and the
// sums of codes are up to a thousand times what is left without their mean:
// after 60000 tokens in a row the result was 9 % off.  So it goes every
// kMiddleTiles tiles, 8 steps (every 8 tiles cost the same).
constexpr int kMiddleTiles = 4;
template <int G, int NT>
__device__ __forceinline__ void takeMiddle(Unit<G, NT>& u) {
  // 2^-24 * 7.5 of a code, 2^-24 * 127.5 of c + 16 c'
  const uint64_t one = pair(-7.5f * 5.9604644775390625e-8f), two = pair(-127.5f * 5.9604644775390625e-8f);
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
      const uint64_t ones = pair(u.ones[n][gr][0], u.ones[n][gr][1]);  // rows are alike
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const float2 o = unpair(fma2(ones, (j & 1) ? two : one, pair(u.o[n][gr][j][k], u.o[n][gr][j][k + 1])));
          u.o[n][gr][j][k] = o.x;
          u.o[n][gr][j][k + 1] = o.y;
        }
#pragma unroll
      for (int k = 0; k < 4; k++) u.ones[n][gr][k] = 0.0f;
    }
}

// A tile of 32 tokens that starts at token t0 of the request.  Two blocks at a
// time give the scheduler twice the independent work of one, and share the
// looks at the maximum (one block at a time: 166 us where this took 146 then, 64
// requests of 500 to 16000 tokens, 8 key heads).  there: bit b, block b exists.
// middle: the sums so far give up theirs, while the scores are on their way.
template <int G, int NT>
__device__ __forceinline__ void tileStep(Unit<G, NT>& u, uint32_t tile, const LaneOffsets& at, int t0, uint32_t there, int lane, bool middle) {
  constexpr int D = 64 * G, B = kBlocks;
  const int g = lane >> 2;
  // S^T, group by group: the scale of a token and group acts on the group's
  // sum.  z is the score in units of qs; x what it passes the maximum by.
  float z[B][NT][4], x[B][NT][4];
#pragma unroll
  for (int b = 0; b < B; b++) {
    uint32_t k[2][2 * G], kp[2][G];
    readKeys<G>(k, kp, tile + b * 18 * D, at);
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
      float acc[NT][4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t w0 = k[0][2 * gr + h], w1 = k[1][2 * gr + h];
        const uint32_t s0 = upperBytes(w0), s1 = upperBytes(w1);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          if (h == 0)
            mmaFirst(acc[n], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, u.qb[n][gr][0][0],
                     u.qb[n][gr][0][1]);
          else
            mma(acc[n], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, u.qb[n][gr][2][0],
                u.qb[n][gr][2][1]);
          mma(acc[n], s0 & 0x000F000Fu, s1 & 0x000F000Fu, s0 & 0x00F000F0u, s1 & 0x00F000F0u, u.qb[n][gr][2 * h + 1][0],
              u.qb[n][gr][2 * h + 1][1]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {  // tokens g, g + 8
        const float s = kv4::bf16Lo(kp[i][gr]), off = fmaf(-7.5f, s, kv4::bf16Hi(kp[i][gr]));
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float y = gr == 0 ? off * u.sq[n][gr][c] : fmaf(off, u.sq[n][gr][c], z[b][n][2 * i + c]);
            z[b][n][2 * i + c] = fmaf(acc[n][2 * i + c], s, y);
          }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) x[b][n][e] = fmaf(z[b][n][e], u.qs[n][e & 1], -u.m[n][e & 1]);
  }
  float s[B][2][G], mid[B][2][G];
  uint32_t widest[G] = {};  // the largest |scale| (low half); of tokens that no row sees, too
#pragma unroll
  for (int b = 0; b < B; b++) {
    uint32_t vp[2][G];
    readValueParams<G>(vp, tile + b * 18 * D, at);
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int gr = 0; gr < G; gr++) {
        s[b][i][gr] = kv4::bf16Lo(vp[i][gr]);
        mid[b][i][gr] = kv4::bf16Hi(vp[i][gr]);
        widest[gr] = maxSizes(widest[gr], vp[i][gr]);
      }
  }
  if (middle) takeMiddle(u);
  // Tokens behind some row's last one, or on no page: their scores are none,
  // and the parameters of those that no row sees may be anything.
  const bool edge = t0 + kTile > u.least || there != (1u << B) - 1;
  if (edge) {
#pragma unroll
    for (int b = 0; b < B; b++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int t = ((there >> b) & 1u) ? t0 + 16 * b + g + 8 * i : INT_MAX;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++)
            if (t >= u.limit[n][c]) x[b][n][2 * i + c] = -INFINITY;
        if (t >= u.most) {
#pragma unroll
          for (int gr = 0; gr < G; gr++) s[b][i][gr] = mid[b][i][gr] = 0.0f;
        }
      }
  }
  // The maximum is followed loosely: it moves when a score passes it by 8
  // (weights reach 2^8), and the factor of the weights when a scale might take
  // them out of f16, so most tiles take neither a reduction nor a rescaling.
  float high = x[0][0][0], wide[G];
#pragma unroll
  for (int b = 0; b < B; b++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) high = fmaxf(high, x[b][n][e]);
  bool grow = high > 8.0f;
#pragma unroll
  for (int gr = 0; gr < G; gr++) {
    wide[gr] = kv4::bf16Lo(widest[gr]);
    grow = grow || wide[gr] > u.lim[gr];
  }
  if (__any_sync(~0u, grow)) {
    float most[G];  // of the factors
#pragma unroll
    for (int gr = 0; gr < G; gr++) most[gr] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float f[G][2];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float top = kNone;
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
          for (int i = 0; i < 2; i++)
            if (x[b][n][2 * i + c] != -INFINITY) top = fmaxf(top, z[b][n][2 * i + c] * u.qs[n][c]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float m = fmaxf(u.m[n][c], top), alpha = exp2Fast(u.m[n][c] - m);
        u.m[n][c] = m;
        u.l[n][c] *= alpha;
        float largest[G] = {};  // p |scale| of the tokens that the row sees
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
          for (int i = 0; i < 2; i++)
            if (x[b][n][2 * i + c] != -INFINITY) {
              x[b][n][2 * i + c] = fmaf(z[b][n][2 * i + c], u.qs[n][c], -m);
              const float w = exp2Fast(x[b][n][2 * i + c]);
#pragma unroll
              for (int gr = 0; gr < G; gr++) largest[gr] = fmaxf(largest[gr], w * fabsf(s[b][i][gr]));
            }
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
          u.mid[n][gr][c] *= alpha;
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) largest[gr] = fmaxf(largest[gr], __shfl_xor_sync(~0u, largest[gr], o));
          // What was the largest so far has shrunk with the other weights.
          const float old = u.by[n][gr][c], want = fminf(__fdividef(old, alpha), __fdividef(kWeightTop, largest[gr]));
          const float by = fmaxf(fminf(want, kFactorMost), kFactorLeast), moved = alpha * by;
          f[gr][c] = moved == old ? 1.0f : __fdividef(moved, old);
          u.by[n][gr][c] = by;
          most[gr] = fmaxf(most[gr], by);
        }
      }
#pragma unroll
      for (int gr = 0; gr < G; gr++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          u.ones[n][gr][k] *= f[gr][k & 1];
#pragma unroll
          for (int j = 0; j < 4; j++) u.o[n][gr][j][k] *= f[gr][k & 1];
        }
    }
#pragma unroll
    for (int gr = 0; gr < G; gr++) u.lim[gr] = __fdividef(kScaleRoom, most[gr]);
  }
  if (edge) weighValues<G, NT, true>(u, x, s, mid, tile, at);
  else weighValues<G, NT, false>(u, x, s, mid, tile, at);
}

template <typename T>
__device__ __forceinline__ void storeOut(void* out, long long at, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(static_cast<T*>(out) + at) = pack8<T>(y);
}

// slot < 0: the unit is whole, write the result; else the partial sums.
template <int G, int NT>
__device__ __forceinline__ void finish(Unit<G, NT>& u, const AttnArgs& p, const Request& r, int head, int row0, int lane,
                                       int slot) {
  constexpr int D = 64 * G, R = 8 * NT;
  const int g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      float l = u.l[n][c], mid[G];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
      for (int gr = 0; gr < G; gr++) {
        mid[gr] = u.mid[n][gr][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mid[gr] += __shfl_xor_sync(~0u, mid[gr], o);
      }
      const int local = 8 * n + 2 * q + c;
      const long long row = static_cast<long long>(row0) + local;
      if (row >= static_cast<long long>(r.rows) * p.group) continue;
      const int i = static_cast<int>(row / p.group), h = head * p.group + static_cast<int>(row % p.group);
      const bool none = l == 0.0f;
      const float norm = slot < 0 ? (none ? 0.0f : 1.0f / l) : 1.0f;
#pragma unroll
      for (int gr = 0; gr < G; gr++) {
        const float back = __fdividef(1.0f, u.by[n][gr][c]);
        const float base = fmaf(-7.5f * u.ones[n][gr][c], back, mid[gr]);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          // channel 8g + j: the sum of its code, times 2^-24
          const float* o = u.o[n][gr][j >> 1];
          const float* low = u.o[n][gr][(j >> 1) & ~1];
          const int at = 2 * (j & 1) + c;
          const float sum = (j & 2) ? (o[at] - low[at]) * 1048576.0f : o[at] * 16777216.0f;
          y[j] = fmaf(sum, back, base) * norm;
        }
        if (slot < 0) {
          const long long at = (r.start + i) * p.oTok + h * p.oHead + 64 * gr + 8 * g;
          if (p.half16) storeOut<__half>(p.out, at, y);
          else storeOut<__nv_bfloat16>(p.out, at, y);
        } else {
          float* dst = p.partial + (static_cast<long long>(slot) * R + local) * D + 64 * gr + 8 * g;
          *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
      if (g == 0) {
        if (slot >= 0) p.stats[static_cast<long long>(slot) * R + local] = make_float2(u.m[n][c], l);
        else if (p.lse != nullptr)
          p.lse[static_cast<long long>(r.start + i) * p.qHeads + h] = none ? -INFINITY : (u.m[n][c] + log2f(l)) * kLn2;
      }
    }
}

// Two row tiles need the registers of three warps for two.
constexpr int warpsFor(int nt) { return nt == 1 ? kWarps : 8; }

template <int G>
constexpr int tileBytes() {
  return kBlocks * 18 * 64 * G;
}

template <int G, int NT>
__global__ void __launch_bounds__(warpsFor(NT) * 32, 1) attnKernel(const __grid_constant__ AttnArgs p) {
  extern __shared__ uint4 shared[];  // the warps' rings, then the prefix sums
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be set up beside this
  constexpr int R = 8 * NT, D = 64 * G, kThreads = warpsFor(NT) * 32;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) + (threadIdx.x >> 5) * (kStages * tileBytes<G>());
  long long* prefix = reinterpret_cast<long long*>(reinterpret_cast<uint8_t*>(shared) + warpsFor(NT) * kStages * tileBytes<G>());
  scanTiles<kThreads>(p, R, prefix);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= p.batch; b += kThreads) p.prefix[b] = prefix[b];
  const long long total = prefix[p.batch];
  if (total == 0) return;
  const int lane = threadIdx.x & 31;
  const LaneOffsets offsets = offsetsOf<G>(lane);
  const uint8_t* mine = p.cache + 16 * lane;
  // Neighbouring ranges go to different blocks, so that few tiles spread over the SMs.
  const int w = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
  const Split split(total, p.workers);
  if (w >= split.workers) return;
  const long long first = split.start(w), last = split.start(w + 1);
  long long tile = first;
  while (tile < last) {
    const int b = findRequest(prefix, p.batch, tile);
    const Request r = requestOf(p, b);
    const int nt = tilesOf(r), units = unitsOf(p, r, R);
    const long long off = tile - prefix[b];
    const int unit = static_cast<int>(quotient(off, nt)), from = static_cast<int>(off - static_cast<long long>(unit) * nt);
    const int head = unit / units, row0 = (unit - head * units) * R;
    const int upto = static_cast<int>(min(static_cast<long long>(nt), from + (last - tile)));
    const int* pages = p.table + static_cast<long long>(b) * p.width;

    // Lane i looks up block 32 j + i of the range: its page, then its address.
    // The pages of the next 32 are under way while these are copied.
    const int known = (r.kv + kv4::kBlockTokens - 1) / kv4::kBlockTokens;
    auto pageOf = [&](int block) { return block < known ? pages[block / p.blocksPerPage] : -1; };
    int pageAhead = pageOf(from * kBlocks + lane);
    Unit<G, NT> u;
    loadQuery<G, NT>(u, p, r, head, row0, lane);
    // Tiles of this range that some row sees.
    const int count = min(upto, (u.most + kTile - 1) / kTile) - from;
    long long address = 0;
    uint32_t there = 0, thereBefore = 0;  // blocks of this look-up, and the last, whose page exists
    int in = 0, out = 0;                  // places in the ring
    auto issue = [&](int i) {             // i-th tile of the range
      if (i < count) {
        const int at = (i * kBlocks) & 31;
        if (at == 0) {
          const int block = (from + i) * kBlocks + lane, page = pageAhead;
          const bool ok = page >= 0 && page < p.pages;
          address = ((static_cast<long long>(page) * p.kvHeads + head) * p.blocksPerPage + block % p.blocksPerPage) * (18 * D);
          thereBefore = there;
          there = __ballot_sync(~0u, ok);
          pageAhead = pageOf(block + 32);
        }
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
          const long long from = __shfl_sync(~0u, address, at + b);
          if ((there >> (at + b)) & 1u) copyBlock<G>(ring + in * tileBytes<G>() + b * 18 * D + 16 * lane, mine + from, lane);
        }
      }
      in = in + 1 == kStages ? 0 : in + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) issue(i);
    for (int i = 0; i < count; i++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();  // the tile is there for every lane, and the one before has been read by all
      const int next = i + kStages - 1;
      issue(next);
      // the look-up may have moved on to the next 32 blocks
      const bool moved = ((i ^ next) & (32 / kBlocks)) && (next & ~(32 / kBlocks - 1)) < count;
      const uint32_t mask = ((moved ? thereBefore : there) >> ((i * kBlocks) & 31)) & ((1u << kBlocks) - 1);
      if (mask != 0) tileStep<G, NT>(u, ring + out * tileBytes<G>(), offsets, (from + i) * kTile, mask, lane, (i & (kMiddleTiles - 1)) == kMiddleTiles - 1);
      out = out + 1 == kStages ? 0 : out + 1;
    }
    __syncwarp();  // the ring is read by all before the next unit's copies
    const bool whole = from == 0 && upto == nt;
    // A range has at most two partial units: the one it starts in, and the one it ends in.
    finish<G, NT>(u, p, r, head, row0, lane, whole ? -1 : tile == first ? 2 * w : 2 * w + 1);
    tile += upto - from;
  }
}

// The request whose rows hold t (batch if none), by a whole warp: 32 starts
// are looked at together, so 1024 requests take two looks.
__device__ __forceinline__ int requestOfRow(const AttnArgs& p, int t, int lane) {
  int lo = 0, n = p.batch;  // it is one of lo .. lo + n - 1, or none of them
  while (n > 32) {
    const int step = (n + 31) >> 5, at = lo + min(lane * step, n - 1);
    const uint32_t before = __ballot_sync(~0u, lane * step < n && p.qStarts[at] <= t);
    if (before == 0) return p.batch;
    const int piece = 31 - __clz(before);
    n = min(step, n - piece * step);
    lo += piece * step;
  }
  const uint32_t ahead = __ballot_sync(~0u, lane < n && p.qStarts[lo + lane + 1] > t);
  return ahead == 0 ? p.batch : lo + __ffs(ahead) - 1;
}

// A joined row: a lane has channels 2 lane and 2 lane + 1 of every group.
template <int G>
__device__ __forceinline__ void storeRow(const AttnArgs& p, int t, int h, int lane, const float (&y)[2 * G], float m, float l) {
  const bool none = l == 0.0f;
  const float norm = none ? 0.0f : 1.0f / l;
  const long long at = t * p.oTok + h * p.oHead + 2 * lane;
#pragma unroll
  for (int gr = 0; gr < G; gr++) {
    if (p.half16) *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + at + 64 * gr) = __floats2half2_rn(y[2 * gr] * norm, y[2 * gr + 1] * norm);
    else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + at + 64 * gr) = __floats2bfloat162_rn(y[2 * gr] * norm, y[2 * gr + 1] * norm);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[static_cast<long long>(t) * p.qHeads + h] = none ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Joins the partial sums of every row whose unit was cut, and clears the rows
// that see nothing or stand behind the last request.  A block of four warps
// takes one row where parts are many (WIDE: few rows in all), else each warp
// takes one.  The loads of a row depend on one another three deep: starts and
// lengths, maxima and sums, outputs.
template <int G, bool WIDE>
__global__ void __launch_bounds__(128) joinKernel(const __grid_constant__ AttnArgs p, int R) {
  constexpr int D = 64 * G;
  __shared__ float sums[WIDE ? 4 : 1][WIDE ? D : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long id = WIDE ? blockIdx.x : blockIdx.x * 4LL + warp;
  int t = 0, h = 0, b = p.batch;
  Request r{0, 0, 0};
  bool inside = false, mine = false;
  if (id < static_cast<long long>(p.tokens) * p.qHeads) {
    t = static_cast<int>(id / p.qHeads);
    h = static_cast<int>(id - static_cast<long long>(t) * p.qHeads);
    b = requestOfRow(p, t, lane);
    if (b < p.batch) r = requestOf(p, b);
    inside = t >= r.start && t < r.start + r.rows;
    mine = inside ? !isLong(p, r) : p.zeroTail != 0;
  }
  const int nt = inside ? tilesOf(r) : 0;
  float y[2 * G] = {};
  float m = kNone, l = 0.0f;
  // The partial sums are there.  Every thread waits, those without a row too:
  // this grid may end only behind the one before it, whose scratch the next
  // kernel on the stream may take.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!mine) return;
  if (nt > 0) {
    const int row = (t - r.start) * p.group + h % p.group, units = unitsOf(p, r, R);
    const long long total = p.prefix[p.batch];
    const long long a = p.prefix[b] + (static_cast<long long>(h / p.group) * units + row / R) * nt;
    const Split split(total, p.workers);
    const int w0 = split.owner(a), w1 = split.owner(a + nt - 1);
    if (w0 == w1) return;  // written by its warp
    // 32 parts at a time: a lane reads the maximum and the sum of one.
    for (int base = w0; base <= w1; base += 32) {
      const int w = base + lane, n = min(32, w1 - base + 1);
      long long slot = 0;
      float2 st = make_float2(kNone, 0.0f);
      if (lane < n) {
        slot = (2LL * w + (split.start(w) < a ? 1 : 0)) * R + row % R;
        st = p.stats[slot];
      }
      float top = st.x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      top = fmaxf(m, top);
      const float old = exp2Fast(m - top), add = exp2Fast(st.x - top);
      m = top;
      float sum = st.y * add;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(~0u, sum, o);
      l = l * old + sum;
#pragma unroll
      for (int k = 0; k < 2 * G; k++) y[k] *= old;
#pragma unroll 8
      for (int k = WIDE ? warp : 0; k < n; k += WIDE ? 4 : 1) {
        const float f = __shfl_sync(~0u, add, k);
        const float2* src = reinterpret_cast<const float2*>(p.partial + __shfl_sync(~0u, slot, k) * D) + lane;
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
          const float2 v = src[32 * gr];
          y[2 * gr] = fmaf(v.x, f, y[2 * gr]);
          y[2 * gr + 1] = fmaf(v.y, f, y[2 * gr + 1]);
        }
      }
    }
    if (WIDE) {  // the warps' shares, in order
#pragma unroll
      for (int k = 0; k < 2 * G; k++) sums[warp][64 * (k >> 1) + 2 * lane + (k & 1)] = y[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2 * G; k++) {
        const int d = 64 * (k >> 1) + 2 * lane + (k & 1);
        y[k] = (sums[0][d] + sums[WIDE ? 1 : 0][d]) + (sums[WIDE ? 2 : 0][d] + sums[WIDE ? 3 : 0][d]);
      }
    }
  }
  if (WIDE && warp > 0) return;
  storeRow<G>(p, t, h, lane, y, m, l);
}

}  // namespace
}  // namespace model
}  // namespace vccl

#include "kernels/kv4_chunk.cuh"

namespace vccl {
namespace model {
namespace {

int smsOfDevice() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Requests with this many query rows a key head go to the tensor-core kernel
// (a quarter of its 256-row units), and it is launched where the requests
// bring kLongMean rows on average (a launch that finds none costs 3 us).
constexpr int kLongRows = 64, kLongMean = 24;

struct ChunkPlan {
  bool use;
  int splits;
  long long units;  // at most, shares included: below 2^31 as the rows of all heads are
};

ChunkPlan chunkPlan(int batch, int tokens, int qHeads, int kvHeads) {
  const long long rows = static_cast<long long>(tokens) * (qHeads / kvHeads);
  if (rows < kLongRows || rows < static_cast<long long>(kLongMean) * batch) return {false, 1, 0};
  const long long most = rows / kLongRows;
  const long long units = kvHeads * (rows / kChunkRows + (batch < most ? batch : most));
  // Fewer units than twice the SMs: the keys are shared out as well.
  const long long s = 2LL * smsOfDevice() / units;
  const int splits = static_cast<int>(s < 1 ? 1 : s > 16 ? 16 : s);
  return {true, splits, units * splits};
}

// One abort word per device in mapped host memory: a launch that gave up a
// wait sets it, and the next call on that device, or the next look by
// vcclKv4AttentionStatus, reads it.  Made at the first
// launch, which may be a captured one: an allocation of host memory puts
// nothing on a stream, so captures (this thread's and others') allow it in
// relaxed mode.
std::mutex gFlagMu;
int* gHostFlags[64] = {};
int* gDevFlags[64] = {};

int* chunkErrorFlag() {
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  std::lock_guard<std::mutex> lock(gFlagMu);
  if (gDevFlags[dev] == nullptr) {
    int* h = nullptr;
    int* d = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    cudaError_t e = cudaHostAlloc(reinterpret_cast<void**>(&h), 64, cudaHostAllocMapped | cudaHostAllocPortable);
    if (e == cudaSuccess) {
      *h = 0;
      e = cudaHostGetDevicePointer(reinterpret_cast<void**>(&d), h, 0);
      if (e != cudaSuccess) cudaFreeHost(h);
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    gHostFlags[dev] = h;
    gDevFlags[dev] = d;
  }
  return gDevFlags[dev];
}

bool takeChunkError() {
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  std::lock_guard<std::mutex> lock(gFlagMu);
  volatile int* h = gHostFlags[dev];
  if (h == nullptr || *h == 0) return false;
  *h = 0;
  return true;
}

template <int G>
cudaError_t launchChunk(const AttnArgs& p, long long units, cudaStream_t st) {
  const int fixed = ChunkSmem<G>::kStarts + 1024;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allowShared(chunkKernel<G>, fixed + (kMaxBatch + 1) * static_cast<int>(sizeof(int)), done);
  if (e != cudaSuccess) return e;
  const int sms = smsOfDevice();
  chunkKernel<G><<<static_cast<int>(units < sms ? units : sms), kChunkThreads, fixed + (p.batch + 1) * sizeof(int), st>>>(p);
  return cudaGetLastError();
}

// Two tiles of 8 query rows where a request brings more than 8 rows of a key
// head on average (a warp then reads the cache once for 16 rows).
int rowTiles(int batch, int tokens, int group) {
  return group > 8 || static_cast<long long>(tokens) * group > 8LL * batch ? 2 : 1;
}

template <int G, int NT>
cudaError_t launchAttn(const AttnArgs& p, int grid, cudaStream_t st) {
  constexpr int kRings = warpsFor(NT) * kStages * tileBytes<G>();
  const size_t smem = kRings + static_cast<size_t>(p.batch + 1) * sizeof(long long);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allowShared(attnKernel<G, NT>, kRings + (kMaxBatch + 1) * static_cast<int>(sizeof(long long)), done);
  if (e != cudaSuccess) return e;
  attnKernel<G, NT><<<grid, warpsFor(NT) * 32, smem, st>>>(p);
  return cudaGetLastError();
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

}  // namespace
}  // namespace model
}  // namespace vccl

using namespace vccl;
using namespace vccl::model;

extern "C" {

size_t vcclKv4AttentionWorkspace(int batch, int tokens, int qHeads, int kvHeads, int D) {
  if (batch <= 0 || tokens < 0 || kvHeads <= 0 || qHeads < kvHeads || D <= 0) return 0;
  const int nt = rowTiles(batch, tokens, qHeads / kvHeads);
  const size_t slots = static_cast<size_t>(smsOfDevice()) * warpsFor(nt) * 2 * 8 * nt;
  const ChunkPlan cp = chunkPlan(batch, tokens, qHeads, kvHeads);
  const size_t chunkSlots = cp.use && cp.splits > 1 ? static_cast<size_t>(cp.units) * kChunkRows : 0;
  return align256((batch + 1) * sizeof(long long)) + align256(slots * sizeof(float2)) + align256(slots * D * sizeof(float)) +
         align256((batch + 1) * sizeof(int)) + align256(chunkSlots * sizeof(float2)) + chunkSlots * D * sizeof(float);
}

vcclResult_t vcclKv4AttentionStatus(void) {
  if (!takeChunkError()) return vcclSuccess;
  VERR("vcclKv4Attention: an earlier call on this device gave up (a pipeline wait ran out); its output is invalid");
  return vcclInternalError;
}

vcclResult_t vcclxKv4AttentionInjectAbort(void) {
  if (chunkErrorFlag() == nullptr) return vcclSystemError;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(gFlagMu);
  *gHostFlags[dev & 63] = 1;
  return vcclSuccess;
}

vcclResult_t vcclKv4Attention(const vcclHeads_t* q, const vcclKv4_t* cache, const int* table, int width,
                              const int* kvLens, const int* qStarts, int batch, int tokens, float scale,
                              const vcclHeads_t* out, float* lse, int zeroTail, void* workspace,
                              vcclDataType_t datatype, vcclStream_t stream) {
  if (!cacheOk(cache) || !tokensOk(tokens) || batch <= 0 || batch > kMaxBatch || width <= 0 ||
      static_cast<long long>(width) * cache->pageSize > (1 << 30) ||  // token numbers and a tile more fit an int
      (datatype != vcclBfloat16 && datatype != vcclFloat16))
    return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  if (!headsOk(q, 2) || !headsOk(out, 2) || q->heads != out->heads || q->heads % cache->kvHeads != 0 || !table ||
      !kvLens || !qStarts || !workspace || static_cast<long long>(tokens) * q->heads > INT_MAX)
    return vcclInvalidArgument;
  const vcclResult_t before = vcclKv4AttentionStatus();
  if (before != vcclSuccess) return before;
  TraceRange trace("vccl Kv4Attention");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int group = q->heads / cache->kvHeads, nt = rowTiles(batch, tokens, group), R = 8 * nt;
  const int grid = smsOfDevice();
  AttnArgs p{};
  p.q = q->data;
  p.qTok = q->tokenStride;
  p.qHead = q->headStride;
  p.cache = static_cast<const uint8_t*>(cache->data);
  p.table = table;
  p.kvLens = kvLens;
  p.qStarts = qStarts;
  p.out = out->data;
  p.oTok = out->tokenStride;
  p.oHead = out->headStride;
  p.lse = lse;
  p.width = width;
  p.batch = batch;
  p.tokens = tokens;
  p.qHeads = q->heads;
  p.kvHeads = cache->kvHeads;
  p.group = group;
  p.pages = cache->pages;
  p.blocksPerPage = cache->pageSize / kv4::kBlockTokens;
  p.pageShift = (cache->pageSize & (cache->pageSize - 1)) == 0 ? __builtin_ctz(cache->pageSize) : -1;
  p.workers = grid * warpsFor(nt);
  p.half16 = datatype == vcclFloat16;
  p.zeroTail = zeroTail;
  p.scaleLog2 = scale * 1.44269504088896340736f;
  char* ws = static_cast<char*>(workspace);
  p.prefix = reinterpret_cast<long long*>(ws);
  ws += align256((batch + 1) * sizeof(long long));
  p.stats = reinterpret_cast<float2*>(ws);
  ws += align256(static_cast<size_t>(p.workers) * 2 * R * sizeof(float2));
  p.partial = reinterpret_cast<float*>(ws);
  ws += align256(static_cast<size_t>(p.workers) * 2 * R * cache->D * sizeof(float));
  const ChunkPlan cp = chunkPlan(batch, tokens, q->heads, cache->kvHeads);
  if (cp.use) {
    p.longRows = kLongRows;
    p.splits = cp.splits;
    p.unitsMost = static_cast<int>(cp.units);
    p.chunkStarts = reinterpret_cast<int*>(ws);
    ws += align256((batch + 1) * sizeof(int));
    const size_t chunkSlots = cp.splits > 1 ? static_cast<size_t>(cp.units) * kChunkRows : 0;
    p.chunkStats = reinterpret_cast<float2*>(ws);
    ws += align256(chunkSlots * sizeof(float2));
    p.chunkPartial = reinterpret_cast<float*>(ws);
    p.errorFlag = chunkErrorFlag();
    if (p.errorFlag == nullptr) {
      VERR("vcclKv4Attention: no host memory for the word that reports a launch that gave up");
      return vcclSystemError;
    }
    const cudaError_t c = cache->D == 128 ? launchChunk<2>(p, cp.units, st) : launchChunk<1>(p, cp.units, st);
    if (c != cudaSuccess) {
      VERR("vcclKv4Attention: %s", cudaGetErrorString(c));
      return vcclSystemError;
    }
  }
  cudaError_t e;
  if (cache->D == 128) e = nt == 1 ? launchAttn<2, 1>(p, grid, st) : launchAttn<2, 2>(p, grid, st);
  else e = nt == 1 ? launchAttn<1, 1>(p, grid, st) : launchAttn<1, 2>(p, grid, st);
  if (e != cudaSuccess) {
    VERR("vcclKv4Attention: %s", cudaGetErrorString(e));
    return vcclSystemError;
  }
  // Launched beside the kernel before it: its blocks find their requests
  // while that one ends, and wait for its results.
  cudaLaunchConfig_t cfg{};
  // A block a row while every SM gets no more than four (8 rows of 29 parts:
  // 7 us with a warp a row, 4 with a block).
  const long long rows = static_cast<long long>(tokens) * q->heads;
  const bool wide = rows <= 4LL * smsOfDevice();
  cfg.gridDim = dim3(static_cast<unsigned>(wide ? rows : (rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cache->D == 128) e = wide ? cudaLaunchKernelEx(&cfg, joinKernel<2, true>, p, R) : cudaLaunchKernelEx(&cfg, joinKernel<2, false>, p, R);
  else e = wide ? cudaLaunchKernelEx(&cfg, joinKernel<1, true>, p, R) : cudaLaunchKernelEx(&cfg, joinKernel<1, false>, p, R);
  if (e != cudaSuccess) {
    VERR("vcclKv4Attention: %s", cudaGetErrorString(e));
    return vcclSystemError;
  }
  if (cp.use && cp.splits > 1) {
    const unsigned blocks = static_cast<unsigned>((rows + 3) / 4);
    if (cache->D == 128) chunkJoinKernel<2><<<blocks, 128, 0, st>>>(p);
    else chunkJoinKernel<1><<<blocks, 128, 0, st>>>(p);
    return launched("vcclKv4Attention");
  }
  return vcclSuccess;
}

}  // extern "C"

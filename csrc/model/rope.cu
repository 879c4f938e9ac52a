// SPDX-License-Identifier: Apache-2.0
// Norm and rotation of query and key heads, its gradients, and the write and
// read of the 4-bit cache (the write runs after norm and rotation in the same
// pass, or alone).
//
// A row (one head of one token) is held by LANES neighbouring lanes with 8
// channels each.  In norm and rotation by themselves, and their gradients, a
// lane has 4 channels of the row's first half and the same 4 of its second (two
// 8-byte loads): the two channels of a pair then meet in a lane, and a row of
// 128 takes 4 shuffles instead of 13, which shared the shared-memory pipe with
// the cosines (8192 tokens of 72 heads: 88 us before, 73 now).  In the kernel
// that writes the cache a lane has 8 neighbouring channels of every row, as a
// word of codes does.  The cosines and sines of a block's tokens are taken
// once, into shared memory: the angle position * invFreq is a product in 64
// bits, reduced to [-pi, pi] there, since positions reach millions.
//
// All of it should be bound by memory, every operand being read or written
// once, and was bound by instructions at first (309 for each warp's step of
// two rows of 128 channels).  So a warp's step takes rows of one kind
// (queries, keys or values), whose strides and weights are then uniform, the
// token and head come from a product with a reciprocal, and the next step's
// row is loaded before this one is worked on.
#include <type_traits>

#include "kernels/kv4.cuh"
#include "model/common.cuh"

namespace vccl {
namespace model {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void put2(float* x, uint64_t v) {
  const float2 f = unpair(v);
  x[0] = f.x;
  x[1] = f.y;
}

struct Rope {
  const int* positions;
  const float* invFreq;
  const void* weight[2];  // of queries, of keys
  int half;               // 0: no rotation
  int interleaved;
  float eps;
};

struct Cache {
  uint8_t* data;
  long long tokens;  // pages * pageSize
  int heads;
  int blocksPerPage;
  int shift;  // blocksPerPage = 1 << shift, or -1
  int D;
};

__device__ __forceinline__ uint8_t* cacheBlock(const Cache& c, int slot, int head) {
  const int block = slot >> 4, page = c.shift >= 0 ? block >> c.shift : block / c.blocksPerPage;
  return c.data + ((static_cast<long long>(page) * c.heads + head) * c.blocksPerPage + (block - page * c.blocksPerPage)) *
                      kv4::blockBytes(c.D);
}

// One kind of rows: heads of every token, read or written with strides in
// elements.
struct Side {
  const void* in;
  void* out;
  int inTok, inHead, outTok, outHead;
  int heads;
  uint32_t recip;  // ceil(2^32 / heads); 0 for one head
};

// Where a lane's row stands in a block of tokens.
struct Row {
  int t, h;
  bool live;
};

template <int LANES>
__device__ __forceinline__ Row rowOf(const Side& d, int step, int n, bool active) {
  const int row = step * (32 / LANES) + (threadIdx.x & 31) / LANES;
  Row r;
  r.t = d.recip ? static_cast<int>(__umulhi(static_cast<uint32_t>(row), d.recip)) : row;
  r.h = row - r.t * d.heads;
  r.live = active && r.t < n;
  return r;
}

template <int LANES>
__device__ __forceinline__ int stepsOf(const Side& d, int n) {
  return (n * d.heads + 32 / LANES - 1) / (32 / LANES);
}

// A warp's steps of one kind after `before` steps of the kinds ahead, which
// the block's warps took in turn.  load(row) fetches, work(row) uses what was
// fetched one step before.  A kind is a constant of the code: its strides and
// weights are operands, not look-ups (14 a step of 205 instructions).
template <int LANES, typename Load, typename Work>
__device__ __forceinline__ void eachRow(const Side& d, int before, int n, bool active, Load&& load, Work&& work) {
  constexpr int kWarps = kThreads / 32;
  const int end = stepsOf<LANES>(d, n);
  int step = ((threadIdx.x >> 5) - before) & (kWarps - 1);
  if (step >= end) return;
  Row ahead = rowOf<LANES>(d, step, n, active);
  load(ahead);
  while (step < end) {
    const Row row = ahead;
    step += kWarps;
    work(row, [&]() {
      if (step < end) {
        ahead = rowOf<LANES>(d, step, n, active);
        load(ahead);
      }
    });
  }
}

template <typename T>
__device__ __forceinline__ const T* inOf(const Side& d, int token, int h) {
  return static_cast<const T*>(d.in) + static_cast<long long>(token) * d.inTok + static_cast<long long>(h) * d.inHead;
}
template <typename T>
__device__ __forceinline__ T* outOf(const Side& d, int token, int h) {
  return static_cast<T*>(d.out) + static_cast<long long>(token) * d.outTok + static_cast<long long>(h) * d.outHead;
}

// cos and sin of position * f, in 64 bits: k turns of 2 pi are taken off
// first (positions reach millions, and a large argument would cost more).
__device__ __forceinline__ void cosSin(int position, float f, float* c, float* s) {
  const double a = static_cast<double>(position) * static_cast<double>(f);
  const double turns = rint(a * 0.15915494309189533577);
  double sd, cd;
  sincos(fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586477, a)), &sd, &cd);
  *c = static_cast<float>(cd);
  *s = static_cast<float>(sd);
}

// Of tokens [t0, t0 + n): cosines, sines, negative sines, half each.
__device__ __forceinline__ void fillAngles(const Rope& r, int t0, int n, float* smem) {
  for (int i = threadIdx.x; i < n * r.half; i += blockDim.x) {
    const int t = i / r.half, j = i - t * r.half;
    float c, s;
    cosSin(r.positions[t0 + t], r.invFreq[j], &c, &s);
    float* at = smem + t * 3 * r.half + j;
    at[0] = c;
    at[r.half] = s;
    at[2 * r.half] = -s;
  }
}

// The weights as f32, D of queries and D of keys.
template <typename T>
__device__ __forceinline__ void fillWeights(const Rope& r, int D, float* smem) {
  for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
    const T* w = static_cast<const T*>(r.weight[i >= D]);
    if (w != nullptr) smem[i] = static_cast<float>(w[i >= D ? i - D : i]);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = a.z;
  x[3] = a.w;
  x[4] = b.x;
  x[5] = b.y;
  x[6] = b.z;
  x[7] = b.w;
}

// Rotates the channels of a row in place.  angles: of the row's token.  Every
// operation rounds by itself.
template <int LANES>
__device__ __forceinline__ void rotate(float (&x)[8], int lane, const Rope& r, const float* angles) {
  const float* up = angles + r.half;        // what the second channel of a pair takes
  const float* down = angles + 2 * r.half;  // what the first one takes
  if (r.interleaved) {
    if (8 * lane < 2 * r.half) {
      const float4 c = *reinterpret_cast<const float4*>(angles + 4 * lane);
      const float4 u = *reinterpret_cast<const float4*>(up + 4 * lane);
      const float4 d = *reinterpret_cast<const float4*>(down + 4 * lane);
      const float cc[4] = {c.x, c.y, c.z, c.w}, uu[4] = {u.x, u.y, u.z, u.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __fadd_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, dd[i]));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, uu[i]));
      }
    }
    return;
  }
  const int h = r.half >> 3;  // lanes that hold the first channels of the pairs
  const int src = lane < h ? lane + h : lane < 2 * h ? lane - h : lane;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = __shfl_sync(~0u, x[i], src, LANES);
  if (lane < 2 * h) {
    const int j = 8 * (lane < h ? lane : lane - h);
    float c[8], s[8];
    load8(angles + j, c);
    load8((lane < h ? down : up) + j, s);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
  }
}

// Sum of a row's squares, in the order in which torch's mean over a row of
// 64 or 128 adds them on this GPU, so that a program that comes from
// elementary torch operations keeps its bits, and with them its 4-bit codes
// (a last bit of the norm moves one bf16 key in 10^5 and one code in 10^6):
// fours in order (rows of 128; one by one for 64), then the sums of the upper
// half of the row onto those of the lower half, and so on.  Lanes trade what
// they do not keep, so a row of 128 takes 5 shuffles, one of 64 takes 10.
// Rows of the cache are of these two sizes.
__device__ __forceinline__ float four(const float* x) {
  float s = __fmul_rn(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 4; i++) s = __fadd_rn(s, __fmul_rn(x[i], x[i]));
  return s;
}

template <int LANES>
__device__ __forceinline__ float squaresOfRow(const float (&x)[8], int lane) {
  static_assert(LANES == 8 || LANES == 16, "rows of 64 or 128");
  if constexpr (LANES == 16) {
    const float a = four(x), b = four(x + 4);
    const bool up = lane & 8;  // keeps the sums of the second fours
    float v = up ? b : a;
    v = __fadd_rn(v, __shfl_xor_sync(~0u, up ? a : b, 8));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(~0u, v, o));
    return __fadd_rn(v, __shfl_xor_sync(~0u, v, 8));
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __fmul_rn(x[i], x[i]);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {  // keeps the upper half of what it has where its bit o is set
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; i++) {
        const float got = __shfl_xor_sync(~0u, up ? v[i] : v[i + o], o);
        v[i] = __fadd_rn(up ? v[i + o] : v[i], got);
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v[0] = __fadd_rn(v[0], __shfl_xor_sync(~0u, v[0], o));
    return v[0];
  }
}

// ---- rows in halves: channels 4 lane .. + 3 and D / 2 + 4 lane .. + 3 --------

template <typename T>
__device__ __forceinline__ uint4 loadHalves(const T* row, int lane, int D) {
  const uint2 a = *reinterpret_cast<const uint2*>(row + 4 * lane), b = *reinterpret_cast<const uint2*>(row + D / 2 + 4 * lane);
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <typename T>
__device__ __forceinline__ void storeHalves(T* row, int lane, int D, const uint4& v) {
  *reinterpret_cast<uint2*>(row + 4 * lane) = make_uint2(v.x, v.y);
  *reinterpret_cast<uint2*>(row + D / 2 + 4 * lane) = make_uint2(v.z, v.w);
}
__device__ __forceinline__ void loadHalves(const float* row, int lane, int D, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(row + 4 * lane), b = *reinterpret_cast<const float4*>(row + D / 2 + 4 * lane);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = a.z;
  x[3] = a.w;
  x[4] = b.x;
  x[5] = b.y;
  x[6] = b.z;
  x[7] = b.w;
}

// The same sums in the same order as squaresOfRow; rows of other sizes: fours
// in order, then a tree over the lanes.
template <int LANES>
__device__ __forceinline__ float squaresOfHalves(const float (&x)[8], int lane, int D) {
  if (LANES == 8 && D == 64) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __fadd_rn(__fmul_rn(x[i], x[i]), __fmul_rn(x[4 + i], x[4 + i]));
#pragma unroll
    for (int o = 4; o > 1; o >>= 1) {  // keeps the upper half of what it has where its bit o is set
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o / 2; i++) {
        const float got = __shfl_xor_sync(~0u, up ? v[i] : v[i + o / 2], o);
        v[i] = __fadd_rn(up ? v[i + o / 2] : v[i], got);
      }
    }
    v[0] = __fadd_rn(v[0], __shfl_xor_sync(~0u, v[0], 1));
    v[0] = __fadd_rn(v[0], __shfl_xor_sync(~0u, v[0], 4));
    return __fadd_rn(v[0], __shfl_xor_sync(~0u, v[0], 2));
  }
  float s = __fadd_rn(four(x), four(x + 4));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(~0u, s, o));
  return s;
}

// rotate() for rows in halves.
template <int LANES, bool BACK>
__device__ __forceinline__ void rotateHalves(float (&x)[8], int lane, int D, const Rope& r, const float* angles) {
  const float* up = angles + (BACK ? 2 : 1) * r.half;    // what the second channel of a pair takes
  const float* down = angles + (BACK ? 1 : 2) * r.half;  // what the first one takes
  if (r.interleaved) {
#pragma unroll
    for (int v = 0; v < 2; v++) {
      const int first = (v ? D / 2 : 0) + 4 * lane;
      if (first < 2 * r.half && 8 * lane < D) {
        const float2 c = *reinterpret_cast<const float2*>(angles + first / 2);
        const float2 u = *reinterpret_cast<const float2*>(up + first / 2), d = *reinterpret_cast<const float2*>(down + first / 2);
        const float cc[2] = {c.x, c.y}, uu[2] = {u.x, u.y}, dd[2] = {d.x, d.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float a = x[4 * v + 2 * i], b = x[4 * v + 2 * i + 1];
          x[4 * v + 2 * i] = __fadd_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, dd[i]));
          x[4 * v + 2 * i + 1] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, uu[i]));
        }
      }
    }
    return;
  }
  if (2 * r.half == D) {
    if (8 * lane < D) {
      const float4 c = *reinterpret_cast<const float4*>(angles + 4 * lane), s = *reinterpret_cast<const float4*>(up + 4 * lane);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = x[i], b = x[4 + i];
        x[i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
        x[4 + i] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, ss[i]));
      }
    }
    return;
  }
  // Some channels rotate: the partners of a lane's channels are in other lanes.
  float y[8];
#pragma unroll
  for (int v = 0; v < 2; v++) {
    const int first = (v ? D / 2 : 0) + 4 * lane;
    const int partner = first < r.half ? first + r.half : first < 2 * r.half ? first - r.half : first;
    const int at = min(partner >= D / 2 ? partner - D / 2 : partner, D / 2 - 4) / 4;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = __shfl_sync(~0u, x[i], at, LANES), b = __shfl_sync(~0u, x[4 + i], at, LANES);
      y[4 * v + i] = partner >= D / 2 ? b : a;
    }
  }
#pragma unroll
  for (int v = 0; v < 2; v++) {
    const int first = (v ? D / 2 : 0) + 4 * lane;
    if (first < 2 * r.half && 8 * lane < D) {
      const bool low = first < r.half;
      const int j = low ? first : first - r.half;
      const float4 c = *reinterpret_cast<const float4*>(angles + j), s = *reinterpret_cast<const float4*>((low ? down : up) + j);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; i++) x[4 * v + i] = __fadd_rn(__fmul_rn(x[4 * v + i], cc[i]), __fmul_rn(y[4 * v + i], ss[i]));
    }
  }
}

struct NormRopeArgs {
  Side side[2];  // queries, keys
  Rope rope;
  int tokens, D, tpb;
};

// Block: tpb tokens, all their heads.  Norm and rotation round after every
// f32 operation (no contraction): the bits of elementary operations, and of
// the write to the cache.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 4) normRopeKernel(const __grid_constant__ NormRopeArgs p) {
  extern __shared__ float4 shared[];
  float* weights = reinterpret_cast<float*>(shared);
  float* angles = weights + 2 * p.D;
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % LANES;
  const bool active = 8 * lane < p.D;
  fillWeights<T>(p.rope, p.D, weights);
  fillAngles(p.rope, t0, n, angles);
  __syncthreads();
  const float share = 1.0f / p.D;
  auto rows = [&](const Side& d, const void* weight, const float* w0, int before) {
    uint4 ahead;
    eachRow<LANES>(
        d, before, n, active,
        [&](const Row& r) { ahead = r.live ? loadHalves(inOf<T>(d, t0 + r.t, r.h), lane, p.D) : make_uint4(0, 0, 0, 0); },
        [&](const Row& row, auto&& next) {
          float x[8];
          unpack8<T>(ahead, x);
          next();
          if (weight != nullptr) {
            const float r = rsqrtf(__fadd_rn(__fmul_rn(squaresOfHalves<LANES>(x, lane, p.D), share), p.rope.eps));
            if (active) {
              float w[8];
              loadHalves(w0, lane, p.D, w);
#pragma unroll
              for (int i = 0; i < 8; i++) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
            }
          }
          rotateHalves<LANES, false>(x, lane, p.D, p.rope, angles + min(row.t, n - 1) * 3 * p.rope.half);
          if (row.live) storeHalves(outOf<T>(d, t0 + row.t, row.h), lane, p.D, pack8<T>(x));
        });
  };
  rows(p.side[0], p.rope.weight[0], weights, 0);
  rows(p.side[1], p.rope.weight[1], weights + p.D, stepsOf<LANES>(p.side[0], n));
}

struct AppendArgs {
  Side side[3];  // queries, keys, values (of which queries alone are written as they are)
  Rope rope;
  Cache cache;
  const int* slots;
  int tokens, D, tpb;
};

// Block: tpb tokens, all their heads; without a rotation keys and values go to
// the cache as they are.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 4) appendKernel(const __grid_constant__ AppendArgs p) {
  extern __shared__ float4 shared[];
  float* weights = reinterpret_cast<float*>(shared);
  float* angles = weights + 2 * p.D;
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % LANES;
  const int G = p.D / kv4::kGroup, g = lane >> 3, b = lane & 7;
  const bool turned = p.rope.half > 0;
  if (turned) {
    fillWeights<T>(p.rope, p.D, weights);
    fillAngles(p.rope, t0, n, angles);
    __syncthreads();
  }
  const float share = 1.0f / p.D;
  // Norm and rotation of a row of queries or keys.
  auto turn = [&](uint4& raw, const Row& row, const void* weight, const float* w0) {
    float x[8];
    unpack8<T>(raw, x);
    if (weight != nullptr) {
      const float r = rsqrtf(__fadd_rn(__fmul_rn(squaresOfRow<LANES>(x, lane), share), p.rope.eps));
      float w[8];
      load8(w0 + 8 * lane, w);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
    }
    rotate<LANES>(x, lane, p.rope, angles + min(row.t, n - 1) * 3 * p.rope.half);
    raw = pack8<T>(x);
  };
  uint4 ahead;
  int slotAhead = -1;
  int before = 0;
  if (turned) {
    const Side& d = p.side[0];
    eachRow<LANES>(
        d, before, n, true,
        [&](const Row& r) { ahead = r.live ? *reinterpret_cast<const uint4*>(inOf<T>(d, t0 + r.t, r.h) + 8 * lane) : make_uint4(0, 0, 0, 0); },
        [&](const Row& row, auto&& next) {
          uint4 raw = ahead;
          next();
          turn(raw, row, p.rope.weight[0], weights);
          if (row.live) *reinterpret_cast<uint4*>(outOf<T>(d, t0 + row.t, row.h) + 8 * lane) = raw;
        });
    before = stepsOf<LANES>(d, n);
  }
  auto store = [&](const Side& d, auto keys) {
    // the row and the word of a lane's codes in a block, but for the token
    const int wordAt = 4 * (keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G));
    eachRow<LANES>(
        d, before, n, true,
        [&](const Row& r) {
          ahead = make_uint4(0, 0, 0, 0);
          slotAhead = -1;
          if (r.live) {
            ahead = *reinterpret_cast<const uint4*>(inOf<T>(d, t0 + r.t, r.h) + 8 * lane);
            slotAhead = p.slots[t0 + r.t];
          }
        },
        [&](const Row& row, auto&& next) {
          uint4 raw = ahead;
          const int slot = slotAhead;
          next();
          if (keys && turned) turn(raw, row, p.rope.weight[1], weights + p.D);
          uint32_t params;
          const uint32_t word = kv4::quantise8<T>(raw, &params);
          if (slot >= 0 && slot < p.cache.tokens) {
            uint8_t* blk = cacheBlock(p.cache, slot, row.h);
            const int place = slot & 15, rowAt = keys ? place : 16 + kv4::valueRow(place);
            *reinterpret_cast<uint32_t*>(blk + rowAt * (p.D / 2) + wordAt) = word;
            if (b == 0) *reinterpret_cast<uint32_t*>(blk + (keys ? 16 : 17) * p.D + place * (4 * G) + 4 * g) = params;
          }
        });
    before += stepsOf<LANES>(d, n);
  };
  store(p.side[1], std::true_type{});
  store(p.side[2], std::false_type{});
}

struct ReadArgs {
  Side side[2];  // keys, values: out
  Cache cache;
  const int* slots;
  int tokens, tpb;
};

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(dst) = pack8<T>(x);
}
template <>
__device__ __forceinline__ void store8<float>(float* dst, const float (&x)[8]) {
  *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// Block: tpb tokens, their keys and then their values.  27 us for 16384 tokens
// of 8 heads (3.2 TB/s): the latency of codes, then the ALU.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) readKernel(const __grid_constant__ ReadArgs p) {
  constexpr int D = 8 * LANES, G = D / kv4::kGroup;
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % LANES, g = lane >> 3, b = lane & 7;
  // The slots first, so that a row's codes are one load away.
  __shared__ int slots[16];
  if (threadIdx.x < n) slots[threadIdx.x] = p.slots[t0 + threadIdx.x];
  __syncthreads();
  auto rows = [&](const Side& d, auto keys, int before) {
    const int wordAt = 4 * (keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G));
    uint32_t wordAhead = 0, paramsAhead = 0;
    eachRow<LANES>(
        d, before, n, true,
        [&](const Row& row) {
          wordAhead = paramsAhead = 0;  // reads as 0
          const int slot = row.live ? slots[row.t] : -1;
          if (slot >= 0 && slot < p.cache.tokens) {
            const uint8_t* blk = cacheBlock(p.cache, slot, row.h);
            const int place = slot & 15, rowAt = keys ? place : 16 + kv4::valueRow(place);
            wordAhead = *reinterpret_cast<const uint32_t*>(blk + rowAt * (D / 2) + wordAt);
            paramsAhead = *reinterpret_cast<const uint32_t*>(blk + (keys ? 16 : 17) * D + place * (4 * G) + 4 * g);
          }
        },
        [&](const Row& row, auto&& next) {
          float x[8];
          kv4::dequantise8(wordAhead, paramsAhead, x);
          next();
          if (row.live) store8<T>(outOf<T>(d, t0 + row.t, row.h) + 8 * lane, x);
        });
  };
  rows(p.side[0], std::true_type{}, 0);
  rows(p.side[1], std::false_type{}, stepsOf<LANES>(p.side[0], n));
}

struct BackwardArgs {
  Side side[2];    // gradients of the outputs in, of the inputs out
  Side forward[2];  // the inputs
  Rope rope;
  float* partial;  // [grid][2][D] sums of dy * x^ (where a weight is given)
  int tokens, D, tpb;
};

// Blocks of the backward kernel: each adds up its rows' weight gradients, so
// their number bounds the workspace.
constexpr int kBackwardBlocks = 148 * 4;

// dx = r (w g - x^ mean(w g x^)), dw = sum g x^ with g = R^-1 dy, x^ = x r,
// r = 1 / sqrt(mean x^2 + eps).  Sums and products of neighbouring channels go
// in pairs of f32, one instruction for both: 72 us for 8192 tokens of 40 heads
// of 128 (3.5 TB/s), 76 without; with rows of neighbouring channels and no
// pairs it was 72 too.  The forward pass gains nothing from pairs (73
// us for 72 heads, 4.1 TB/s): its products may not merge with its sums, which
// the compiler does with pairs.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 3) backwardKernel(const __grid_constant__ BackwardArgs p) {
  extern __shared__ float4 shared[];
  float* weights = reinterpret_cast<float*>(shared);
  float* angles = weights + 2 * p.D;
  const int lane = threadIdx.x % LANES;
  const bool active = 8 * lane < p.D;
  const float share = 1.0f / p.D;
  fillWeights<T>(p.rope, p.D, weights);
  uint64_t dw[2][4] = {};  // pairs of f32
  for (int t0 = blockIdx.x * p.tpb; t0 < p.tokens; t0 += gridDim.x * p.tpb) {
    const int n = min(p.tpb, p.tokens - t0);
    __syncthreads();  // the angles of the tokens before are read
    fillAngles(p.rope, t0, n, angles);
    __syncthreads();
    auto rows = [&](const Side& d, const Side& forward, const void* weight, const float* w0, uint64_t (&dw)[4], int before) {
      uint4 dyAhead, xAhead;
      eachRow<LANES>(
          d, before, n, active,
          [&](const Row& r) {
            dyAhead = xAhead = make_uint4(0, 0, 0, 0);
            if (r.live) {
              dyAhead = loadHalves(inOf<T>(d, t0 + r.t, r.h), lane, p.D);
              if (weight != nullptr) xAhead = loadHalves(inOf<T>(forward, t0 + r.t, r.h), lane, p.D);
            }
          },
          [&](const Row& row, auto&& next) {
            float g[8], x[8];
            unpack8<T>(dyAhead, g);
            unpack8<T>(xAhead, x);
            next();
            rotateHalves<LANES, true>(g, lane, p.D, p.rope, angles + min(row.t, n - 1) * 3 * p.rope.half);
            if (weight != nullptr) {
              float w[8] = {};
              if (active) loadHalves(w0, lane, p.D, w);
              uint64_t g2[4], x2[4], w2[4], sq2 = 0, gx2 = 0;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                g2[i] = pair(g[2 * i], g[2 * i + 1]);
                x2[i] = pair(x[2 * i], x[2 * i + 1]);
                w2[i] = mul2(pair(w[2 * i], w[2 * i + 1]), g2[i]);
                sq2 = fma2(x2[i], x2[i], sq2);
                gx2 = fma2(w2[i], x2[i], gx2);
              }
              const float2 sqs = unpair(sq2), gxs = unpair(gx2);
              float sq = sqs.x + sqs.y, gx = gxs.x + gxs.y;
#pragma unroll
              for (int o = 1; o < LANES; o <<= 1) {
                sq += __shfl_xor_sync(~0u, sq, o);
                gx += __shfl_xor_sync(~0u, gx, o);
              }
              const float r = rsqrtf(fmaf(sq, share, p.rope.eps));
              // A row behind the last one counts as zero (its r may be infinite).
              const float on = row.live ? r : 0.0f;
              const float m = gx * on * on * share;  // r mean(w g x^): dx = r w g - x r m
              const uint64_t minus = pair(-m * on), on2 = pair(on), r2 = pair(r);
#pragma unroll
              for (int i = 0; i < 4; i++) {
                dw[i] = fma2(mul2(g2[i], on2), x2[i], dw[i]);
                put2(g + 2 * i, fma2(x2[i], minus, mul2(r2, w2[i])));
              }
            }
            if (row.live) storeHalves(outOf<T>(d, t0 + row.t, row.h), lane, p.D, pack8<T>(g));
          });
    };
    rows(p.side[0], p.forward[0], p.rope.weight[0], weights, dw[0], 0);
    rows(p.side[1], p.forward[1], p.rope.weight[1], weights + p.D, dw[1], stepsOf<LANES>(p.side[0], n));
  }
  if (p.partial == nullptr) return;
  // Rows of the block, then the block's sums to its own place.
  constexpr int kRows = kThreads / LANES;
  const int row0 = threadIdx.x / LANES;
  __shared__ float sums[kThreads * 8];
#pragma unroll
  for (int which = 0; which < 2; which++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (active) put2(sums + row0 * (LANES * 8) + (i < 2 ? 0 : p.D / 2) + 4 * lane + 2 * (i & 1), dw[which][i]);
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
      float s = 0.0f;
      for (int r = 0; r < kRows; r++) s += sums[r * (LANES * 8) + d];
      p.partial[(static_cast<long long>(blockIdx.x) * 2 + which) * p.D + d] = s;
    }
  }
}

// The blocks' sums in a fixed order: the same bits on every run.  32 channels
// a block, its 32 warps a share of the sums each.
template <typename T>
__global__ void __launch_bounds__(1024) weightGradKernel(const float* partial, int blocks, int D, T* dqw, T* dkw) {
  const int which = blockIdx.y, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane, part = threadIdx.x >> 5;
  T* out = which ? dkw : dqw;
  if (out == nullptr) return;
  __shared__ double sums[32][33];
  double s = 0.0;
  if (d < D) {
#pragma unroll 8
    for (int b = part; b < blocks; b += 32) s += partial[(static_cast<long long>(b) * 2 + which) * D + d];
  }
  sums[part][lane] = s;
  __syncthreads();
  // Warp w adds up channel w.
  s = sums[lane][part];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (lane == 0 && blockIdx.x * 32 + part < D) out[blockIdx.x * 32 + part] = static_cast<T>(static_cast<float>(s));
}

int lanesFor(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Tokens a block takes: enough rows for a dozen steps, so that the angles are
// shared and loads overlap, but no fewer blocks than twice the SMs.
int tokensPerBlock(int tokens, int heads, int D) {
  const int rows = kThreads / lanesFor(D);
  int tpb = 1;
  while (tpb < 16 && tpb * heads < 12 * rows && tokens / (2 * tpb) >= 2 * 148) tpb *= 2;
  return tpb;
}

size_t sharedBytes(const Rope& r, int tpb, int D) { return (static_cast<size_t>(3) * tpb * r.half + 2 * D) * sizeof(float); }

// Kinds of rows from the descriptions; an absent one has no heads.
Side sideOf(const vcclHeads_t* in, const vcclHeads_t* out) {
  Side s{};
  if (in != nullptr) {
    s.in = in->data;
    s.inTok = static_cast<int>(in->tokenStride);
    s.inHead = static_cast<int>(in->headStride);
    s.heads = in->heads;
  }
  if (out != nullptr) {
    s.out = out->data;
    s.outTok = static_cast<int>(out->tokenStride);
    s.outHead = static_cast<int>(out->headStride);
    s.heads = out->heads;
  }
  s.recip = s.heads > 1 ? static_cast<uint32_t>(((1ull << 32) + s.heads - 1) / s.heads) : 0;
  return s;
}

bool ropeOk(const vcclRope_t* r, int D, int tokens) {
  if (r == nullptr || (tokens > 0 && (r->positions == nullptr)) || r->invFreq == nullptr) return false;
  if (r->half < 8 || r->half % 8 != 0 || 2 * r->half > D || !(r->eps >= 0.0f)) return false;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  return aligned(r->qWeight) && aligned(r->kWeight);
}

Rope ropeOf(const vcclRope_t* r) {
  if (r == nullptr) return {nullptr, nullptr, {nullptr, nullptr}, 0, 0, 0.0f};
  return {r->positions, r->invFreq, {r->qWeight, r->kWeight}, r->half, r->interleaved, r->eps};
}

template <typename T>
void launchNormRope(const NormRopeArgs& p, cudaStream_t st) {
  const int grid = (p.tokens + p.tpb - 1) / p.tpb;
  const size_t smem = sharedBytes(p.rope, p.tpb, p.D);
  switch (lanesFor(p.D)) {
    case 8: normRopeKernel<T, 8><<<grid, kThreads, smem, st>>>(p); break;
    case 16: normRopeKernel<T, 16><<<grid, kThreads, smem, st>>>(p); break;
    default: normRopeKernel<T, 32><<<grid, kThreads, smem, st>>>(p); break;
  }
}

template <typename T>
void launchAppend(const AppendArgs& p, cudaStream_t st) {
  const int grid = (p.tokens + p.tpb - 1) / p.tpb;
  const size_t smem = sharedBytes(p.rope, p.tpb, p.D);
  if (p.D == 64) appendKernel<T, 8><<<grid, kThreads, smem, st>>>(p);
  else appendKernel<T, 16><<<grid, kThreads, smem, st>>>(p);
}

template <typename T>
void launchBackward(const BackwardArgs& p, int grid, cudaStream_t st) {
  const size_t smem = sharedBytes(p.rope, p.tpb, p.D);
  switch (lanesFor(p.D)) {
    case 8: backwardKernel<T, 8><<<grid, kThreads, smem, st>>>(p); break;
    case 16: backwardKernel<T, 16><<<grid, kThreads, smem, st>>>(p); break;
    default: backwardKernel<T, 32><<<grid, kThreads, smem, st>>>(p); break;
  }
}

template <typename T>
void launchRead(const ReadArgs& p, int grid, cudaStream_t st) {
  if (p.cache.D == 64) readKernel<T, 8><<<grid, kThreads, 0, st>>>(p);
  else readKernel<T, 16><<<grid, kThreads, 0, st>>>(p);
}

bool sixteenBit(vcclDataType_t t) { return t == vcclBfloat16 || t == vcclFloat16; }

Cache cacheOf(const vcclKv4_t* c) {
  const int per = c->pageSize / kv4::kBlockTokens;
  int shift = 0;
  while ((1 << shift) < per) shift++;
  return {static_cast<uint8_t*>(c->data), static_cast<long long>(c->pages) * c->pageSize, c->kvHeads, per,
          (1 << shift) == per ? shift : -1, c->D};
}

}  // namespace
}  // namespace model
}  // namespace vccl

using namespace vccl;
using namespace vccl::model;

extern "C" {

vcclResult_t vcclQkNormRope(const vcclHeads_t* q, const vcclHeads_t* k, const vcclRope_t* rope,
                            const vcclHeads_t* qOut, const vcclHeads_t* kOut, int tokens, int D,
                            vcclDataType_t datatype, vcclStream_t stream) {
  if (!tokensOk(tokens) || D <= 0 || D % 8 != 0 || D > 256 || !sixteenBit(datatype) || !ropeOk(rope, D, tokens))
    return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  if (!headsOk(q, 2) || !headsOk(k, 2) || !headsOk(qOut, 2) || !headsOk(kOut, 2) || q->heads != qOut->heads ||
      k->heads != kOut->heads)
    return vcclInvalidArgument;
  TraceRange trace("vccl QkNormRope");
  NormRopeArgs p{};
  p.side[0] = sideOf(q, qOut);
  p.side[1] = sideOf(k, kOut);
  p.rope = ropeOf(rope);
  p.tokens = tokens;
  p.D = D;
  p.tpb = tokensPerBlock(tokens, q->heads + k->heads, D);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchNormRope<__nv_bfloat16>(p, st);
  else launchNormRope<__half>(p, st);
  return launched("vcclQkNormRope");
}

size_t vcclQkNormRopeBackwardWorkspace(int D) {
  return D > 0 ? static_cast<size_t>(kBackwardBlocks) * 2 * D * sizeof(float) : 0;
}

vcclResult_t vcclQkNormRopeBackward(const vcclHeads_t* dq, const vcclHeads_t* dk, const vcclHeads_t* q,
                                    const vcclHeads_t* k, const vcclRope_t* rope, const vcclHeads_t* dqIn,
                                    const vcclHeads_t* dkIn, void* dqWeight, void* dkWeight, void* workspace,
                                    int tokens, int D, vcclDataType_t datatype, vcclStream_t stream) {
  if (!tokensOk(tokens) || D <= 0 || D % 8 != 0 || D > 256 || !sixteenBit(datatype) || !ropeOk(rope, D, tokens))
    return vcclInvalidArgument;
  const bool weights = rope->qWeight != nullptr || rope->kWeight != nullptr;
  if ((rope->qWeight != nullptr) != (dqWeight != nullptr) || (rope->kWeight != nullptr) != (dkWeight != nullptr) ||
      (weights && workspace == nullptr))
    return vcclInvalidArgument;
  if (tokens > 0 && (!headsOk(dq, 2) || !headsOk(dk, 2) || !headsOk(q, 2) || !headsOk(k, 2) || !headsOk(dqIn, 2) ||
                     !headsOk(dkIn, 2) || q->heads != dq->heads || k->heads != dk->heads ||
                     q->heads != dqIn->heads || k->heads != dkIn->heads))
    return vcclInvalidArgument;
  TraceRange trace("vccl QkNormRopeBackward");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int grid = 0;
  if (tokens > 0) {
    BackwardArgs p{};
    p.side[0] = sideOf(dq, dqIn);
    p.side[1] = sideOf(dk, dkIn);
    p.forward[0] = sideOf(q, nullptr);
    p.forward[1] = sideOf(k, nullptr);
    p.rope = ropeOf(rope);
    p.partial = weights ? static_cast<float*>(workspace) : nullptr;
    p.tokens = tokens;
    p.D = D;
    p.tpb = tokensPerBlock(tokens, q->heads + k->heads, D);
    grid = (tokens + p.tpb - 1) / p.tpb;
    if (grid > kBackwardBlocks) grid = kBackwardBlocks;
    if (datatype == vcclBfloat16) launchBackward<__nv_bfloat16>(p, grid, st);
    else launchBackward<__half>(p, grid, st);
  }
  if (weights) {  // without tokens the sums are zero
    const dim3 g((D + 31) / 32, 2);
    const float* part = static_cast<const float*>(workspace);
    if (datatype == vcclBfloat16)
      weightGradKernel<<<g, 1024, 0, st>>>(part, grid, D, static_cast<__nv_bfloat16*>(dqWeight),
                                          static_cast<__nv_bfloat16*>(dkWeight));
    else
      weightGradKernel<<<g, 1024, 0, st>>>(part, grid, D, static_cast<__half*>(dqWeight), static_cast<__half*>(dkWeight));
  }
  return launched("vcclQkNormRopeBackward");
}

vcclResult_t vcclKv4Append(const vcclKv4_t* cache, const vcclHeads_t* k, const vcclHeads_t* v, const int* slots,
                           const vcclRope_t* rope, const vcclHeads_t* q, const vcclHeads_t* qOut, int tokens,
                           vcclDataType_t datatype, vcclStream_t stream) {
  if (!tokensOk(tokens) || !cacheOk(cache) || !sixteenBit(datatype)) return vcclInvalidArgument;
  if (rope != nullptr && !ropeOk(rope, cache->D, tokens)) return vcclInvalidArgument;
  if ((rope == nullptr) != (q == nullptr) || (q == nullptr) != (qOut == nullptr)) return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  if (slots == nullptr || !headsOk(k, 2) || !headsOk(v, 2) || k->heads != cache->kvHeads || v->heads != cache->kvHeads)
    return vcclInvalidArgument;
  if (q != nullptr && (!headsOk(q, 2) || !headsOk(qOut, 2) || q->heads != qOut->heads)) return vcclInvalidArgument;
  TraceRange trace("vccl Kv4Append");
  AppendArgs p{};
  p.side[0] = sideOf(q, qOut);
  p.side[1] = sideOf(k, nullptr);
  p.side[2] = sideOf(v, nullptr);
  p.rope = ropeOf(rope);
  p.cache = cacheOf(cache);
  p.slots = slots;
  p.tokens = tokens;
  p.D = cache->D;
  p.tpb = tokensPerBlock(tokens, p.side[0].heads + 2 * cache->kvHeads, cache->D);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchAppend<__nv_bfloat16>(p, st);
  else launchAppend<__half>(p, st);
  return launched("vcclKv4Append");
}

vcclResult_t vcclKv4Read(const vcclKv4_t* cache, const int* slots, const vcclHeads_t* k, const vcclHeads_t* v,
                         int tokens, vcclDataType_t datatype, vcclStream_t stream) {
  if (!tokensOk(tokens) || !cacheOk(cache) || !(sixteenBit(datatype) || datatype == vcclFloat32)) return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  const int elem = datatype == vcclFloat32 ? 4 : 2;
  if (slots == nullptr || !headsOk(k, elem) || !headsOk(v, elem) || k->heads != cache->kvHeads ||
      v->heads != cache->kvHeads)
    return vcclInvalidArgument;
  TraceRange trace("vccl Kv4Read");
  const int tpb = tokensPerBlock(tokens, 2 * cache->kvHeads, cache->D);
  const ReadArgs p{{sideOf(nullptr, k), sideOf(nullptr, v)}, cacheOf(cache), slots, tokens, tpb};
  const int grid = (tokens + tpb - 1) / tpb;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchRead<__nv_bfloat16>(p, grid, st);
  else if (datatype == vcclFloat16) launchRead<__half>(p, grid, st);
  else launchRead<float>(p, grid, st);
  return launched("vcclKv4Read");
}

}  // extern "C"

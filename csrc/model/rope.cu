// SPDX-License-Identifier: Apache-2.0
// Norm and rotation of query and key heads, its gradients, and the write and
// read of the 4-bit cache (the write runs after norm and rotation in the same
// pass, or alone).
//
// A row (one head of one token) is held by LANES neighbouring lanes with 8
// channels each (16-byte loads and stores); the mean square, the partner
// channels of the rotation and the group extremes of the 4-bit rounding are
// shuffles among them.  The cosines and sines of a block's tokens are taken
// once, into shared memory: the angle position * invFreq is a product in 64
// bits, reduced to [-pi, pi] there, since positions reach millions.
// All of it is bound by memory: every operand is read or written once.
#include "kernels/kv4.cuh"
#include "model/common.cuh"

namespace vccl {
namespace model {
namespace {

constexpr int kThreads = 256;

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
  int D;
};

__device__ __forceinline__ uint8_t* cacheBlock(const Cache& c, int slot, int head) {
  const int block = slot >> 4, page = block / c.blocksPerPage;
  return c.data + ((static_cast<long long>(page) * c.heads + head) * c.blocksPerPage + block % c.blocksPerPage) *
                      kv4::blockBytes(c.D);
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

// cos and sin of tokens [t0, t0 + n) into smem: cos at [i * half + j], sin at
// tpb * half further on.
__device__ __forceinline__ void fillAngles(const Rope& r, int t0, int n, int tpb, float* smem) {
  for (int i = threadIdx.x; i < n * r.half; i += blockDim.x) {
    float c, s;
    cosSin(r.positions[t0 + i / r.half], r.invFreq[i % r.half], &c, &s);
    smem[i] = c;
    smem[tpb * r.half + i] = s;
  }
}

// Rotates the channels of a row in place; back: by the negative angle.
// cosv, sinv: of the row's token.
template <int LANES>
__device__ __forceinline__ void rotate(float (&x)[8], int lane, const Rope& r, const float* cosv, const float* sinv,
                                       float sign) {
  if (r.interleaved) {
    if (8 * lane < 2 * r.half) {
      const float4 c = *reinterpret_cast<const float4*>(cosv + 4 * lane);
      const float4 s = *reinterpret_cast<const float4*>(sinv + 4 * lane);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sign * s.x, sign * s.y, sign * s.z, sign * s.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, ss[i]));
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
    const float sg = lane < h ? -sign : sign;
#pragma unroll
    for (int v = 0; v < 2; v++) {
      const float4 c = *reinterpret_cast<const float4*>(cosv + j + 4 * v);
      const float4 s = *reinterpret_cast<const float4*>(sinv + j + 4 * v);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; i++) x[4 * v + i] = __fadd_rn(__fmul_rn(x[4 * v + i], cc[i]), __fmul_rn(sg * y[4 * v + i], ss[i]));
    }
  }
}

// Sum of a row's squares, in the order in which torch's mean over a row of
// 64 or 128 adds them on this GPU, so that a program that comes from
// elementary torch operations keeps its bits, and with them its 4-bit codes
// (a last bit of the norm moves one bf16 key in 10^5 and one code in 10^6):
// fours in order (rows of 128; one by one for 64), then the sums of the upper
// half of the row onto those of the lower half, and so on.  Lanes trade what
// they do not keep, so a row of 128 takes 5 shuffles, one of 64 takes 10.
// Other rows: fours in order, then a tree over the lanes.
__device__ __forceinline__ float four(const float* x) {
  float s = __fmul_rn(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 4; i++) s = __fadd_rn(s, __fmul_rn(x[i], x[i]));
  return s;
}

template <int LANES>
__device__ __forceinline__ float squaresOfRow(const float (&x)[8], int lane, int D) {
  if (LANES == 16 && D == 128) {
    const float a = four(x), b = four(x + 4);
    const bool up = lane & 8;  // keeps the sums of the second fours
    float v = up ? b : a;
    v = __fadd_rn(v, __shfl_xor_sync(~0u, up ? a : b, 8));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(~0u, v, o));
    return __fadd_rn(v, __shfl_xor_sync(~0u, v, 8));
  }
  if (LANES == 8 && D == 64) {
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
  float s = __fadd_rn(four(x), four(x + 4));
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) s = __fadd_rn(s, __shfl_xor_sync(~0u, s, o));
  return s;
}

struct ForwardArgs {
  Heads in[3];   // queries, keys, values (values, and queries, may be absent)
  Heads out[2];  // queries, keys (keys absent where they go to the cache)
  Rope rope;
  Cache cache;  // data == nullptr: no cache
  const int* slots;
  int tokens, D, tpb;
};

// The rows of a block in steps: token and head without a division.
struct RowWalk {
  int t, h, dt, dh, heads;
  __device__ __forceinline__ RowWalk(int row, int step, int heads_)
      : t(row / heads_), h(row % heads_), dt(step / heads_), dh(step % heads_), heads(heads_) {}
  __device__ __forceinline__ void next() {
    t += dt;
    h += dh;
    if (h >= heads) {
      h -= heads;
      t++;
    }
  }
};

// Block: tpb tokens, all their heads (queries, keys, values in that order).
// Norm and rotation round after every f32 operation (no contraction), so that
// the fused write gives the bits of the two calls it stands for.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 4) forwardKernel(ForwardArgs p) {
  extern __shared__ float angles[];
  constexpr int kRows = kThreads / LANES;
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % LANES;
  const bool active = 8 * lane < p.D;
  const int nq = p.in[0].heads, nk = p.in[1].heads;
  const int rows = n * (nq + nk + p.in[2].heads);
  RowWalk at(threadIdx.x / LANES, kRows, nq + nk + p.in[2].heads);

  // The next row is under way while one is worked on.
  auto load = [&]() {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (at.t < n && active) {
      const int which = (at.h >= nq) + (at.h >= nq + nk), h = at.h - (which > 0 ? nq : 0) - (which > 1 ? nk : 0);
      const Heads& in = p.in[which];
      v = *reinterpret_cast<const uint4*>(static_cast<const T*>(in.data) + (t0 + at.t) * in.tok + h * in.head + 8 * lane);
    }
    return v;
  };
  uint4 ahead = load();
  uint4 weight[2] = {};
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (p.rope.weight[i] != nullptr && active)
      weight[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.rope.weight[i]) + 8 * lane);
  const bool normed = p.rope.weight[0] != nullptr || p.rope.weight[1] != nullptr;
  if (p.rope.half > 0) {
    fillAngles(p.rope, t0, n, p.tpb, angles);
    __syncthreads();
  }
  const float share = 1.0f / p.D;
  // Whole warps step together: a row behind the last one is masked.
  for (int base = 0; base < rows; base += kRows) {
    const int t = at.t, which = (at.h >= nq) + (at.h >= nq + nk);
    const int h = at.h - (which > 0 ? nq : 0) - (which > 1 ? nk : 0);
    const bool live = t < n && active;
    uint4 raw = ahead;
    at.next();
    if (base + kRows < rows) ahead = load();
    if (__any_sync(~0u, which < 2)) {
      float x[8];
      unpack8<T>(raw, x);
      if (normed) {
        const float r = rsqrtf(__fadd_rn(__fmul_rn(squaresOfRow<LANES>(x, lane, p.D), share), p.rope.eps));
        if (which < 2 && p.rope.weight[which] != nullptr) {
          float w[8];
          unpack8<T>(which ? weight[1] : weight[0], w);
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
        }
      }
      if (p.rope.half > 0) {
        const float* c = angles + min(t, n - 1) * p.rope.half;
        rotate<LANES>(x, lane, p.rope, c, c + p.tpb * p.rope.half, 1.0f);
        // a row of values shares the warp, and keeps its bits
        if (which < 2) raw = pack8<T>(x);
      }
      if (which < 2 && live && p.out[which].data != nullptr) {
        const Heads& out = p.out[which];
        *reinterpret_cast<uint4*>(static_cast<T*>(out.data) + (t0 + t) * out.tok + h * out.head + 8 * lane) = raw;
      }
    }
    if (p.cache.data != nullptr && __any_sync(~0u, which > 0)) {
      uint32_t params;
      const uint32_t word = kv4::quantise8<T>(raw, &params);
      const int slot = which > 0 && live ? p.slots[t0 + t] : -1;
      if (slot >= 0 && slot < p.cache.tokens) {
        uint8_t* blk = cacheBlock(p.cache, slot, h);
        const int place = slot & 15, G = p.D / kv4::kGroup, g = lane >> 3, b = lane & 7;
        const bool keys = which == 1;
        const int rowAt = keys ? place : 16 + kv4::valueRow(place);
        const int wordAt = keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G);
        *reinterpret_cast<uint32_t*>(blk + rowAt * (p.D / 2) + 4 * wordAt) = word;
        if (b == 0) *reinterpret_cast<uint32_t*>(blk + (keys ? 16 : 17) * p.D + place * (4 * G) + 4 * g) = params;
      }
    }
  }
}

struct ReadArgs {
  Cache cache;
  const int* slots;
  Heads out[2];
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

// Block: tpb tokens, their keys and then their values.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) readKernel(ReadArgs p) {
  constexpr int kRows = kThreads / LANES, D = 8 * LANES, G = D / kv4::kGroup;
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % LANES, g = lane >> 3, b = lane & 7, heads = p.cache.heads;
  RowWalk at(threadIdx.x / LANES, kRows, 2 * heads);
  for (; at.t < n; at.next()) {
    const bool keys = at.h < heads;
    const int h = keys ? at.h : at.h - heads;
    const int slot = p.slots[t0 + at.t];
    float x[8] = {};
    if (slot >= 0 && slot < p.cache.tokens) {
      const uint8_t* blk = cacheBlock(p.cache, slot, h);
      const int place = slot & 15;
      const int rowAt = keys ? place : 16 + kv4::valueRow(place);
      const int wordAt = keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + rowAt * (D / 2) + 4 * wordAt);
      const uint32_t params = *reinterpret_cast<const uint32_t*>(blk + (keys ? 16 : 17) * D + place * (4 * G) + 4 * g);
      kv4::dequantise8(word, params, x);
    }
    const Heads& out = keys ? p.out[0] : p.out[1];
    store8<T>(static_cast<T*>(out.data) + (t0 + at.t) * out.tok + h * out.head + 8 * lane, x);
  }
}

struct BackwardArgs {
  Heads dy[2], x[2], dx[2];
  Rope rope;
  float* partial;  // [grid][2][D] sums of dy * x^ (where a weight is given)
  int tokens, D, tpb;
};

// Blocks of the backward kernel: each adds up its rows' weight gradients, so
// their number bounds the workspace.
constexpr int kBackwardBlocks = 148 * 4;

// dx = r (w g - x^ mean(w g x^)), dw = sum g x^ with g = R^-1 dy, x^ = x r,
// r = 1 / sqrt(mean x^2 + eps).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 3) backwardKernel(BackwardArgs p) {
  extern __shared__ float angles[];
  constexpr int kRows = kThreads / LANES;
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
  const bool active = 8 * lane < p.D;
  const int nq = p.x[0].heads, heads = nq + p.x[1].heads;
  const float share = 1.0f / p.D;
  const bool normed = p.rope.weight[0] != nullptr || p.rope.weight[1] != nullptr;
  uint4 weight[2] = {};
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (p.rope.weight[i] != nullptr && active)
      weight[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.rope.weight[i]) + 8 * lane);
  float dw[2][8] = {};
  for (int t0 = blockIdx.x * p.tpb; t0 < p.tokens; t0 += gridDim.x * p.tpb) {
    const int n = min(p.tpb, p.tokens - t0), rows = n * heads;
    RowWalk at(row0, kRows, heads);
    // The next row is under way while one is worked on.
    auto load = [&](uint4& dy, uint4& x) {
      dy = x = make_uint4(0, 0, 0, 0);
      if (at.t < n && active) {
        const int which = at.h >= nq, h = at.h - (which ? nq : 0);
        const Heads& a = p.dy[which];
        dy = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.data) + (t0 + at.t) * a.tok + h * a.head + 8 * lane);
        if (p.rope.weight[which] != nullptr) {
          const Heads& b = p.x[which];
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(b.data) + (t0 + at.t) * b.tok + h * b.head + 8 * lane);
        }
      }
    };
    uint4 dyAhead, xAhead;
    load(dyAhead, xAhead);
    __syncthreads();  // the angles of the tokens before are read
    fillAngles(p.rope, t0, n, p.tpb, angles);
    __syncthreads();
    for (int base = 0; base < rows; base += kRows) {
      const int t = at.t, which = at.h >= nq, h = at.h - (which ? nq : 0);
      const bool live = t < n && active;
      float g[8], x[8];
      unpack8<T>(dyAhead, g);
      unpack8<T>(xAhead, x);
      at.next();
      if (base + kRows < rows) load(dyAhead, xAhead);
      const float* c = angles + min(t, n - 1) * p.rope.half;
      rotate<LANES>(g, lane, p.rope, c, c + p.tpb * p.rope.half, -1.0f);
      if (normed) {
        float w[8], wg[8];
        unpack8<T>(which ? weight[1] : weight[0], w);
        float gx = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          wg[i] = g[i] * w[i];
          gx += wg[i] * x[i];
        }
        float sq = four(x) + four(x + 4);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) {
          sq += __shfl_xor_sync(~0u, sq, o);
          gx += __shfl_xor_sync(~0u, gx, o);
        }
        if (p.rope.weight[which] != nullptr) {
          const float r = rsqrtf(sq * share + p.rope.eps);
          const float m = gx * r * share;  // mean(w g x^)
          const float on = live ? r : 0.0f;
          // A row behind the last one counts as zero (its r may be infinite).
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float xh = x[i] * on;
            if (which) dw[1][i] += g[i] * xh;
            else dw[0][i] += g[i] * xh;
            g[i] = r * (wg[i] - xh * m);
          }
        }
      }
      if (live) {
        const Heads& o = p.dx[which];
        *reinterpret_cast<uint4*>(static_cast<T*>(o.data) + (t0 + t) * o.tok + h * o.head + 8 * lane) = pack8<T>(g);
      }
    }
  }
  if (p.partial == nullptr) return;
  // Rows of the block, then the block's sums to its own place.
  __shared__ float sums[kThreads * 8];
#pragma unroll
  for (int which = 0; which < 2; which++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) sums[row0 * (LANES * 8) + 8 * lane + i] = dw[which][i];
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

size_t angleBytes(const Rope& r, int tpb) { return static_cast<size_t>(2) * tpb * r.half * sizeof(float); }

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
void launchForward(const ForwardArgs& p, cudaStream_t st) {
  const int grid = (p.tokens + p.tpb - 1) / p.tpb;
  const size_t smem = angleBytes(p.rope, p.tpb);
  switch (lanesFor(p.D)) {
    case 8: forwardKernel<T, 8><<<grid, kThreads, smem, st>>>(p); break;
    case 16: forwardKernel<T, 16><<<grid, kThreads, smem, st>>>(p); break;
    default: forwardKernel<T, 32><<<grid, kThreads, smem, st>>>(p); break;
  }
}

template <typename T>
void launchBackward(const BackwardArgs& p, int grid, cudaStream_t st) {
  const size_t smem = angleBytes(p.rope, p.tpb);
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

bool cacheOk(const vcclKv4_t* c) {
  return c != nullptr && c->data != nullptr && (reinterpret_cast<uintptr_t>(c->data) & 15u) == 0 && c->pages > 0 &&
         c->pageSize > 0 && c->pageSize % kv4::kBlockTokens == 0 && c->kvHeads > 0 && (c->D == 64 || c->D == 128) &&
         static_cast<long long>(c->pages) * c->pageSize <= INT32_MAX;
}

Cache cacheOf(const vcclKv4_t* c) {
  return {static_cast<uint8_t*>(c->data), static_cast<long long>(c->pages) * c->pageSize, c->kvHeads,
          c->pageSize / kv4::kBlockTokens, c->D};
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
  if (tokens < 0 || D <= 0 || D % 8 != 0 || D > 256 || !sixteenBit(datatype) || !ropeOk(rope, D, tokens))
    return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  if (!headsOk(q, 2) || !headsOk(k, 2) || !headsOk(qOut, 2) || !headsOk(kOut, 2) || q->heads != qOut->heads ||
      k->heads != kOut->heads)
    return vcclInvalidArgument;
  TraceRange trace("vccl QkNormRope");
  ForwardArgs p{};
  p.in[0] = headsOf(q);
  p.in[1] = headsOf(k);
  p.out[0] = headsOf(qOut);
  p.out[1] = headsOf(kOut);
  p.rope = ropeOf(rope);
  p.tokens = tokens;
  p.D = D;
  p.tpb = tokensPerBlock(tokens, q->heads + k->heads, D);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchForward<__nv_bfloat16>(p, st);
  else launchForward<__half>(p, st);
  return launched("vcclQkNormRope");
}

size_t vcclQkNormRopeBackwardWorkspace(int D) {
  return D > 0 ? static_cast<size_t>(kBackwardBlocks) * 2 * D * sizeof(float) : 0;
}

vcclResult_t vcclQkNormRopeBackward(const vcclHeads_t* dq, const vcclHeads_t* dk, const vcclHeads_t* q,
                                    const vcclHeads_t* k, const vcclRope_t* rope, const vcclHeads_t* dqIn,
                                    const vcclHeads_t* dkIn, void* dqWeight, void* dkWeight, void* workspace,
                                    int tokens, int D, vcclDataType_t datatype, vcclStream_t stream) {
  if (tokens < 0 || D <= 0 || D % 8 != 0 || D > 256 || !sixteenBit(datatype) || !ropeOk(rope, D, tokens))
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
    p.dy[0] = headsOf(dq);
    p.dy[1] = headsOf(dk);
    p.x[0] = headsOf(q);
    p.x[1] = headsOf(k);
    p.dx[0] = headsOf(dqIn);
    p.dx[1] = headsOf(dkIn);
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
  if (tokens < 0 || !cacheOk(cache) || !sixteenBit(datatype)) return vcclInvalidArgument;
  if (rope != nullptr && !ropeOk(rope, cache->D, tokens)) return vcclInvalidArgument;
  if ((rope == nullptr) != (q == nullptr) || (q == nullptr) != (qOut == nullptr)) return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  if (slots == nullptr || !headsOk(k, 2) || !headsOk(v, 2) || k->heads != cache->kvHeads || v->heads != cache->kvHeads)
    return vcclInvalidArgument;
  if (q != nullptr && (!headsOk(q, 2) || !headsOk(qOut, 2) || q->heads != qOut->heads)) return vcclInvalidArgument;
  TraceRange trace("vccl Kv4Append");
  ForwardArgs p{};
  p.in[0] = headsOf(q);
  p.in[1] = headsOf(k);
  p.in[2] = headsOf(v);
  p.out[0] = headsOf(qOut);
  p.rope = ropeOf(rope);
  p.cache = cacheOf(cache);
  p.slots = slots;
  p.tokens = tokens;
  p.D = cache->D;
  p.tpb = tokensPerBlock(tokens, p.in[0].heads + 2 * cache->kvHeads, cache->D);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchForward<__nv_bfloat16>(p, st);
  else launchForward<__half>(p, st);
  return launched("vcclKv4Append");
}

vcclResult_t vcclKv4Read(const vcclKv4_t* cache, const int* slots, const vcclHeads_t* k, const vcclHeads_t* v,
                         int tokens, vcclDataType_t datatype, vcclStream_t stream) {
  if (tokens < 0 || !cacheOk(cache) || !(sixteenBit(datatype) || datatype == vcclFloat32)) return vcclInvalidArgument;
  if (tokens == 0) return vcclSuccess;
  const int elem = datatype == vcclFloat32 ? 4 : 2;
  if (slots == nullptr || !headsOk(k, elem) || !headsOk(v, elem) || k->heads != cache->kvHeads ||
      v->heads != cache->kvHeads)
    return vcclInvalidArgument;
  TraceRange trace("vccl Kv4Read");
  const int tpb = tokensPerBlock(tokens, 2 * cache->kvHeads, cache->D);
  const ReadArgs p{cacheOf(cache), slots, {headsOf(k), headsOf(v)}, tokens, tpb};
  const int grid = (tokens + tpb - 1) / tpb;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) launchRead<__nv_bfloat16>(p, grid, st);
  else if (datatype == vcclFloat16) launchRead<__half>(p, grid, st);
  else launchRead<float>(p, grid, st);
  return launched("vcclKv4Read");
}

}  // extern "C"

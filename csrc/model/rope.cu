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

// cos and sin of position * f: k turns of 2 pi are taken off in 64 bits.
__device__ __forceinline__ void cosSin(int position, float f, float* c, float* s) {
  const double a = static_cast<double>(position) * static_cast<double>(f);
  const double turns = rint(a * 0.15915494309189533577);
  const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586477, a));
  sincosf(static_cast<float>(r), s, c);
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
        x[2 * i] = a * cc[i] - b * ss[i];
        x[2 * i + 1] = b * cc[i] + a * ss[i];
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
      for (int i = 0; i < 4; i++) x[4 * v + i] = x[4 * v + i] * cc[i] + sg * y[4 * v + i] * ss[i];
    }
  }
}

template <int LANES>
__device__ __forceinline__ float rowSum(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

struct ForwardArgs {
  Heads in[3];   // queries, keys, values (values, and queries, may be absent)
  Heads out[2];  // queries, keys (keys absent where they go to the cache)
  Rope rope;
  Cache cache;  // data == nullptr: no cache
  const int* slots;
  int tokens, D, tpb;
};

// Block: tpb tokens, all their heads (queries, keys, values in that order).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) forwardKernel(ForwardArgs p) {
  extern __shared__ float angles[];
  const int t0 = blockIdx.x * p.tpb, n = min(p.tpb, p.tokens - t0);
  if (p.rope.half > 0) {
    fillAngles(p.rope, t0, n, p.tpb, angles);
    __syncthreads();
  }
  constexpr int kRows = kThreads / LANES;
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
  const bool active = 8 * lane < p.D;
  const int heads = p.in[0].heads + p.in[1].heads + p.in[2].heads;
  const int rows = n * heads;
  // Whole warps step together: a row behind the last one is masked.
  for (int base = 0; base < rows; base += kRows) {
    const int row = base + row0;
    const bool live = row < rows && active;
    const int t = row < rows ? row / heads : 0;
    int h = row < rows ? row % heads : 0, which = 0;
    if (h >= p.in[0].heads) {
      h -= p.in[0].heads;
      which = 1;
      if (h >= p.in[1].heads) {
        h -= p.in[1].heads;
        which = 2;
      }
    }
    float x[8] = {};
    if (live) {
      const Heads& in = p.in[which];
      const T* src = static_cast<const T*>(in.data) + (t0 + t) * in.tok + h * in.head + 8 * lane;
      unpack8<T>(*reinterpret_cast<const uint4*>(src), x);
    }
    // Every lane of the warp takes part in the shuffles; rows of values (and
    // rows without a weight or an angle) keep their channels.
    const void* wp = which < 2 ? p.rope.weight[which] : nullptr;
    if (p.rope.weight[0] != nullptr || p.rope.weight[1] != nullptr) {
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) sq += x[i] * x[i];
      sq = rowSum<LANES>(sq);
      if (wp != nullptr && active) {
        const float r = rsqrtf(sq / p.D + p.rope.eps);
        float w[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(wp) + 8 * lane), w);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = x[i] * r * w[i];
      }
    }
    if (p.rope.half > 0) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = x[i];
      rotate<LANES>(y, lane, p.rope, angles + t * p.rope.half, angles + (p.tpb + t) * p.rope.half, 1.0f);
      if (which < 2) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = y[i];
      }
    }
    if (which < 2 && p.out[which].data != nullptr) {
      if (live) {
        const Heads& out = p.out[which];
        *reinterpret_cast<uint4*>(static_cast<T*>(out.data) + (t0 + t) * out.tok + h * out.head + 8 * lane) = pack8<T>(x);
      }
    }
    if (p.cache.data != nullptr) {
      // The keys as the model's type holds them (values are read in it).
      const uint4 v = pack8<T>(x);
      unpack8<T>(v, x);
      uint32_t params;
      const uint32_t word = kv4::quantise8(x, ~0u, &params);
      const int slot = which > 0 && live ? p.slots[t0 + t] : -1;
      if (slot >= 0 && slot < p.cache.tokens) {
        uint8_t* blk = cacheBlock(p.cache, slot, h);
        const int at = slot & 15, G = p.D / kv4::kGroup, g = lane >> 3, b = lane & 7;
        const bool keys = which == 1;
        const int rowAt = keys ? at : 16 + kv4::valueRow(at);
        const int wordAt = keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G);
        *reinterpret_cast<uint32_t*>(blk + rowAt * (p.D / 2) + 4 * wordAt) = word;
        if (b == 0)
          *reinterpret_cast<uint32_t*>(blk + (keys ? 16 : 17) * p.D + at * (4 * G) + 4 * g) = params;
      }
    }
  }
}

struct ReadArgs {
  Cache cache;
  const int* slots;
  Heads out[2];
  int tokens;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) readKernel(ReadArgs p) {
  const int lanes = p.cache.D / 8, heads = p.cache.heads;
  const long long total = static_cast<long long>(p.tokens) * 2 * heads * lanes;
  for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * kThreads) {
    const int lane = static_cast<int>(i % lanes);
    const long long row = i / lanes;
    const int hh = static_cast<int>(row % (2 * heads)), t = static_cast<int>(row / (2 * heads));
    const bool keys = hh < heads;
    const int h = keys ? hh : hh - heads;
    const int slot = p.slots[t];
    float x[8] = {};
    if (slot >= 0 && slot < p.cache.tokens) {
      const uint8_t* blk = cacheBlock(p.cache, slot, h);
      const int D = p.cache.D, at = slot & 15, G = D / kv4::kGroup, g = lane >> 3, b = lane & 7;
      const int rowAt = keys ? at : 16 + kv4::valueRow(at);
      const int wordAt = keys ? kv4::keyWord(b, g, G) : kv4::valueWord(b, g, G);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + rowAt * (D / 2) + 4 * wordAt);
      const uint32_t params = *reinterpret_cast<const uint32_t*>(blk + (keys ? 16 : 17) * D + at * (4 * G) + 4 * g);
      kv4::dequantise8(word, params, x);
    }
    const Heads& out = p.out[keys ? 0 : 1];
    store8<T>(static_cast<T*>(out.data) + t * out.tok + h * out.head + 8 * lane, x);
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
__global__ void __launch_bounds__(kThreads) backwardKernel(BackwardArgs p) {
  extern __shared__ float angles[];
  constexpr int kRows = kThreads / LANES;
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
  const bool active = 8 * lane < p.D;
  const int heads = p.x[0].heads + p.x[1].heads;
  float dw[2][8] = {};
  for (int t0 = blockIdx.x * p.tpb; t0 < p.tokens; t0 += gridDim.x * p.tpb) {
    const int n = min(p.tpb, p.tokens - t0);
    __syncthreads();  // the angles of the tokens before are read
    fillAngles(p.rope, t0, n, p.tpb, angles);
    __syncthreads();
    const int rows = n * heads;
    for (int base = 0; base < rows; base += kRows) {
      const int row = base + row0;
      const bool live = row < rows && active;
      const int t = row < rows ? row / heads : 0;
      int h = row < rows ? row % heads : 0;
      const int which = h >= p.x[0].heads;
      if (which) h -= p.x[0].heads;
      float g[8] = {}, x[8] = {};
      const void* wp = p.rope.weight[which];
      if (live) {
        const Heads& a = p.dy[which];
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.data) + (t0 + t) * a.tok + h * a.head + 8 * lane), g);
        if (wp != nullptr) {
          const Heads& b = p.x[which];
          unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(b.data) + (t0 + t) * b.tok + h * b.head + 8 * lane), x);
        }
      }
      rotate<LANES>(g, lane, p.rope, angles + t * p.rope.half, angles + (p.tpb + t) * p.rope.half, -1.0f);
      if (p.rope.weight[0] != nullptr || p.rope.weight[1] != nullptr) {
        float w[8] = {};
        if (wp != nullptr && active)
          unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(wp) + 8 * lane), w);
        float sq = 0.0f, gx = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          sq += x[i] * x[i];
          gx += g[i] * w[i] * x[i];
        }
        sq = rowSum<LANES>(sq);
        gx = rowSum<LANES>(gx);
        if (wp != nullptr) {
          const float r = rsqrtf(sq / p.D + p.rope.eps);
          const float m = gx * r / p.D;  // mean(w g x^)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float xh = x[i] * r;
            if (live) {  // a row behind the last one may hold 0 * inf
              if (which) dw[1][i] += g[i] * xh;
              else dw[0][i] += g[i] * xh;
            }
            g[i] = r * (g[i] * w[i] - xh * m);
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

// The blocks' sums in a fixed order: the same bits on every run.
template <typename T>
__global__ void weightGradKernel(const float* partial, int blocks, int D, T* dqw, T* dkw) {
  const int which = blockIdx.y, d = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  T* out = which ? dkw : dqw;
  if (out == nullptr) return;
  __shared__ double sums[8][32];
  double s = 0.0;
  if (d < D)
    for (int b = part; b < blocks; b += 8) s += partial[(static_cast<long long>(b) * 2 + which) * D + d];
  sums[part][threadIdx.x & 31] = s;
  __syncthreads();
  if (part == 0 && d < D) {
    for (int i = 1; i < 8; i++) s += sums[i][threadIdx.x & 31];
    out[d] = static_cast<T>(static_cast<float>(s));
  }
}

int lanesFor(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Tokens a block takes: about four rows for every group of lanes, so that
// the angles are shared and loads overlap, but no fewer blocks than SMs.
int tokensPerBlock(int tokens, int heads, int D) {
  const int rows = kThreads / lanesFor(D);
  int tpb = 1;
  while (tpb < 16 && tpb * heads < 4 * rows && tokens / (2 * tpb) >= 148) tpb *= 2;
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
      weightGradKernel<<<g, 256, 0, st>>>(part, grid, D, static_cast<__nv_bfloat16*>(dqWeight),
                                          static_cast<__nv_bfloat16*>(dkWeight));
    else
      weightGradKernel<<<g, 256, 0, st>>>(part, grid, D, static_cast<__half*>(dqWeight), static_cast<__half*>(dkWeight));
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
  const ReadArgs p{cacheOf(cache), slots, {headsOf(k), headsOf(v)}, tokens};
  const long long work = static_cast<long long>(tokens) * 2 * cache->kvHeads * (cache->D / 8);
  const long long blocks = (work + kThreads - 1) / kThreads;
  const int grid = static_cast<int>(blocks < 148 * 16 ? blocks : 148 * 16);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (datatype == vcclBfloat16) readKernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
  else if (datatype == vcclFloat16) readKernel<__half><<<grid, kThreads, 0, st>>>(p);
  else readKernel<float><<<grid, kThreads, 0, st>>>(p);
  return launched("vcclKv4Read");
}

}  // extern "C"

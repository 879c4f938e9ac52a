// SPDX-License-Identifier: Apache-2.0
// Block tables and slots of a serving step, built on the GPU from request
// lengths (vcclPagePlan).
//
// Pages live on a stack in global memory.  With L_i, n_i as in the header,
// need_i = ceil((L_i + n_i) / P) - ceil(L_i / P) and U_i its prefix sums
// (inclusive), request i is granted iff U_i <= |stack| or need_i = 0; U is
// monotone, so the pages taken are G = max U_i over the granted ones, and
// request i's j-th page is stack[|stack| - G + U_i - need_i + j].  Taking
// from the top in ascending order makes a step that releases what an equal
// step took give the same pages back.
#include <climits>

#include "model/common.cuh"

namespace vccl {
namespace model {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxBatch = 8192;

struct PlanArgs {
  const int* lens;
  const int* newLens;
  const unsigned char* finished;
  int* table;
  int* pool;
  const int* freeCount;
  int batch, width, poolSize, page, tokens;
  int* positions;
  int* slots;
  int* requests;
  int* qStarts;
  int* kvLens;
  int* lensOut;
  int* countOut;
  // [2 * batch + 1] place on the stack of the first page that a request takes;
  // lengths and count after the step.  lensOut may be lens and countOut
  // freeCount, which every block of the first kernel reads: the second writes.
  int* scratch;
};

struct Pair {
  long long a, b;
};

// Inclusive prefix sums over the block, added to *carry, which moves on.
__device__ __forceinline__ Pair blockScan(Pair v, Pair* warpSums, Pair* carry) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(~0u, v.a, o), b = __shfl_up_sync(~0u, v.b, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
    }
  }
  if (lane == 31) warpSums[warp] = v;
  __syncthreads();
  Pair w = warpSums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(~0u, w.a, o), b = __shfl_up_sync(~0u, w.b, o);
    if (lane >= o) {
      w.a += a;
      w.b += b;
    }
  }
  const int before = warp > 0 ? warp - 1 : 0;
  const long long a = __shfl_sync(~0u, w.a, before), b = __shfl_sync(~0u, w.b, before);
  const Pair total = {__shfl_sync(~0u, w.a, 31), __shfl_sync(~0u, w.b, 31)};
  v.a += carry->a + (warp > 0 ? a : 0);
  v.b += carry->b + (warp > 0 ? b : 0);
  carry->a += total.a;
  carry->b += total.b;
  __syncthreads();  // warpSums may be written again
  return v;
}

__device__ __forceinline__ long long pagesOf(long long tokens, int page) { return (tokens + page - 1) / page; }

// The last i of n whose start is at most x (starts rise; starts[0] <= x).
__device__ __forceinline__ int findStart(const int* starts, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (starts[m] <= x) lo = m;
    else hi = m - 1;
  }
  return lo;
}

// Block 0: lengths and grants.  The other blocks move the released pages onto
// the stack, one a thread, whoever's they are (a warp for each request left
// most warps idle behind a few long ones); every block takes the prefix sums
// of the released pages for itself, so none waits for another.  Latency bounds
// the plan: 7 us for both kernels with 256 requests, 14 with 2000 requests of
// 107777 rows that release 28 thousand pages (38 with a warp a request).
__global__ void __launch_bounds__(kPlanThreads) planStateKernel(PlanArgs p) {
  extern __shared__ int scratch[];  // released pages before each request, rows up to and including it
  int* sReleased = scratch;
  int* sEnd = sReleased + p.batch;
  __shared__ Pair warpSums[32];
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;  // read behind several barriers

  const int count = min(max(*p.freeCount, 0), p.poolSize);
  Pair sums = {0, 0};
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    Pair v = {0, 0};
    if (i < p.batch) {
      if (p.finished != nullptr && p.finished[i])
        v.a = min(pagesOf(max(p.lens[i], 0), p.page), static_cast<long long>(p.width));
      v.b = max(p.newLens[i], 0);
    }
    const Pair s = blockScan(v, warpSums, &sums);
    if (i < p.batch) {
      sReleased[i] = static_cast<int>(min(s.a - v.a, static_cast<long long>(INT_MAX)));
      sEnd[i] = static_cast<int>(min(s.b, static_cast<long long>(INT_MAX)));
    }
  }
  __syncthreads();
  const int room = p.poolSize - count;
  const int released = static_cast<int>(min(sums.a, static_cast<long long>(room)));
  const int stack = count + released;
  if (blockIdx.x > 0) {
    for (int e = (blockIdx.x - 1) * kPlanThreads + threadIdx.x; e < released; e += (gridDim.x - 1) * kPlanThreads) {
      const int i = findStart(sReleased, p.batch, e);
      p.pool[count + e] = p.table[static_cast<long long>(i) * p.width + e - sReleased[i]];
    }
    return;
  }

  Pair asked = {0, 0};
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    long long left = 0, n = 0, need = 0;
    bool fits = false;
    if (i < p.batch) {
      left = p.finished != nullptr && p.finished[i] ? 0 : max(p.lens[i], 0);
      n = max(p.newLens[i], 0);
      const long long want = pagesOf(left + n, p.page);
      fits = want <= p.width && sEnd[i] <= p.tokens;
      need = fits ? want - pagesOf(left, p.page) : 0;
    }
    const long long upto = blockScan({need, 0}, warpSums, &asked).a;
    if (i < p.batch) {
      const bool granted = fits && (need == 0 || upto <= stack);
      if (granted && need > 0) atomicMax(&taken, static_cast<int>(upto));
      sReleased[i] = granted ? static_cast<int>(min(upto - need, static_cast<long long>(INT_MAX))) : 0;
      p.qStarts[i + 1] = sEnd[i];
      if (i == 0) p.qStarts[0] = 0;
      p.kvLens[i] = granted ? static_cast<int>(left + n) : 0;
      p.scratch[p.batch + i] = static_cast<int>(left + (granted ? n : 0));
    }
  }
  __syncthreads();
  const int bottom = stack - taken;
  for (int i = threadIdx.x; i < p.batch; i += kPlanThreads) p.scratch[i] = bottom + sReleased[i];
  if (threadIdx.x == 0) p.scratch[2 * p.batch] = bottom;
}

// Each row's request, position and slot; the first row of a page that its
// request takes puts the page into the table.  What the table held before is
// read only for pages that the request had, so no block waits for another.
__global__ void __launch_bounds__(256) planRowsKernel(PlanArgs p) {
  extern __shared__ int starts[];  // [batch + 1]
  for (int i = threadIdx.x; i <= p.batch; i += blockDim.x) starts[i] = p.qStarts[i];
  __syncthreads();
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  for (int i = t; i < p.batch; i += gridDim.x * blockDim.x) p.lensOut[i] = p.scratch[p.batch + i];
  if (t == 0) *p.countOut = p.scratch[2 * p.batch];
  if (t >= p.tokens) return;
  int position = 0, slot = -1, who = -1;
  if (t < starts[p.batch]) {
    who = findStart(starts, p.batch, t);
    const int start = starts[who], n = starts[who + 1] - start, kv = p.kvLens[who];
    if (kv > 0) {  // granted
      const int left = kv - n, have = static_cast<int>(pagesOf(left, p.page));
      position = left + t - start;
      const int j = position / p.page;
      int* entry = p.table + static_cast<long long>(who) * p.width + j;
      int page;
      if (j < have) {
        page = *entry;
      } else {
        page = p.pool[p.scratch[who] + j - have];
        if (t == start || position == j * p.page) *entry = page;
      }
      slot = page * p.page + position - j * p.page;
    }
  }
  p.positions[t] = position;
  p.slots[t] = slot;
  p.requests[t] = who;
}

}  // namespace
}  // namespace model
}  // namespace vccl

using namespace vccl;

extern "C" vcclResult_t vcclPagePlan(const int* lens, const int* newLens, const unsigned char* finished, int* table,
                                     int* freePages, const int* freeCount, int batch, int width, int poolSize,
                                     int pageSize, int tokens, int* positions, int* slots, int* requests,
                                     int* qStarts, int* kvLens, int* lensOut, int* countOut, int* scratch, vcclStream_t stream) {
  if (!lens || !newLens || !table || !freePages || !freeCount || !qStarts || !kvLens || !lensOut || !countOut || !scratch ||
      batch <= 0 || batch > model::kPlanMaxBatch || width <= 0 || poolSize <= 0 || pageSize <= 0 || !model::tokensOk(tokens) ||
      static_cast<long long>(poolSize) * pageSize > INT_MAX || static_cast<long long>(width) * pageSize > INT_MAX ||
      (tokens > 0 && (!positions || !slots || !requests)))
    return vcclInvalidArgument;
  TraceRange trace("vccl PagePlan");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const model::PlanArgs p{lens,     newLens, finished,  table, freePages, freeCount, batch,  width,   poolSize, pageSize,
                          tokens,   positions, slots, requests, qStarts, kvLens, lensOut, countOut, scratch};
  const size_t smem = static_cast<size_t>(batch) * 2 * sizeof(int);
  // For every batch: what a kernel has without asking, 48 KiB, holds its static shared memory too.
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = model::allowShared(model::planStateKernel, model::kPlanMaxBatch * 2 * static_cast<int>(sizeof(int)), done);
  if (e != cudaSuccess) {
    VERR("vcclPagePlan: %s", cudaGetErrorString(e));
    return vcclSystemError;
  }
  // A thread for each page that the finished requests may hold, 148 blocks at most.
  const long long held = finished ? (static_cast<long long>(batch) * width + model::kPlanThreads - 1) / model::kPlanThreads : 0;
  model::planStateKernel<<<1 + static_cast<int>(held < 147 ? held : 147), model::kPlanThreads, smem, st>>>(p);
  // The rows are made from what the first kernel writes: without it they are not launched.
  const vcclResult_t state = model::launched("vcclPagePlan");
  if (state != vcclSuccess) return state;
  model::planRowsKernel<<<tokens > 0 ? (tokens + 255) / 256 : 1, 256, (batch + 1) * sizeof(int), st>>>(p);
  return model::launched("vcclPagePlan");
}

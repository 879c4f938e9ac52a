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
};

struct Sums {
  long long a, b, c;
};

// Inclusive prefix sums over the block; *total is the block's sum.
__device__ __forceinline__ Sums blockScan(Sums v, Sums* warpSums, Sums* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(~0u, v.a, o), b = __shfl_up_sync(~0u, v.b, o), c = __shfl_up_sync(~0u, v.c, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
      v.c += c;
    }
  }
  __syncthreads();  // warpSums of an earlier call are read
  if (lane == 31) warpSums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < static_cast<int>(blockDim.x >> 5) ? warpSums[lane] : Sums{0, 0, 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(~0u, w.a, o), b = __shfl_up_sync(~0u, w.b, o), c = __shfl_up_sync(~0u, w.c, o);
      if (lane >= o) {
        w.a += a;
        w.b += b;
        w.c += c;
      }
    }
    warpSums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) {
    const Sums w = warpSums[warp - 1];
    v.a += w.a;
    v.b += w.b;
    v.c += w.c;
  }
  *total = warpSums[(blockDim.x >> 5) - 1];
  return v;
}

__device__ __forceinline__ long long pagesOf(long long tokens, int page) { return (tokens + page - 1) / page; }

// One block: lengths, grants, the stack and the table.
__global__ void __launch_bounds__(kPlanThreads) planStateKernel(PlanArgs p) {
  extern __shared__ int scratch[];  // have, first page (of the taken ones), pages to take: batch each
  int* sHave = scratch;
  int* sFirst = sHave + p.batch;
  int* sNeed = sFirst + p.batch;
  __shared__ Sums warpSums[32];
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;

  const int count = min(max(*p.freeCount, 0), p.poolSize);
  // Pages released, per request (in sNeed for the moment) and in all.
  long long released = 0;
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int r = 0;
    if (i < p.batch && p.finished != nullptr && p.finished[i])
      r = static_cast<int>(min(pagesOf(max(p.lens[i], 0), p.page), static_cast<long long>(p.width)));
    Sums total;
    const Sums s = blockScan({r, 0, 0}, warpSums, &total);
    if (i < p.batch) {
      sNeed[i] = r;
      sFirst[i] = static_cast<int>(released + s.a - r);
    }
    released += total.a;
  }
  __syncthreads();
  // Onto the stack, a warp a request.
  for (int i = threadIdx.x >> 5; i < p.batch; i += kPlanThreads / 32)
    for (int j = threadIdx.x & 31; j < sNeed[i]; j += 32) {
      const long long at = static_cast<long long>(count) + sFirst[i] + j;
      if (at < p.poolSize) p.pool[at] = p.table[static_cast<long long>(i) * p.width + j];
    }
  const long long stack = min(count + released, static_cast<long long>(p.poolSize));
  __syncthreads();

  long long rows = 0, asked = 0;
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    long long left = 0, n = 0;
    if (i < p.batch) {
      left = p.finished != nullptr && p.finished[i] ? 0 : max(p.lens[i], 0);
      n = max(p.newLens[i], 0);
    }
    Sums total;
    const long long end = rows + blockScan({n, 0, 0}, warpSums, &total).a;
    rows += total.a;
    const long long have = pagesOf(left, p.page), want = pagesOf(left + n, p.page);
    const bool fits = want <= p.width && end <= p.tokens;
    const long long need = fits ? want - have : 0;
    const long long upto = asked + blockScan({need, 0, 0}, warpSums, &total).a;
    asked += total.a;
    if (i < p.batch) {
      const bool granted = fits && (need == 0 || upto <= stack);
      if (granted && need > 0) atomicMax(&taken, static_cast<int>(upto));
      sHave[i] = static_cast<int>(min(have, static_cast<long long>(p.width)));
      sFirst[i] = static_cast<int>(upto - need);
      sNeed[i] = granted ? static_cast<int>(need) : 0;
      p.qStarts[i + 1] = static_cast<int>(min(end, static_cast<long long>(INT_MAX)));
      if (i == 0) p.qStarts[0] = 0;
      p.kvLens[i] = granted ? static_cast<int>(left + n) : 0;
      p.lensOut[i] = static_cast<int>(left + (granted ? n : 0));
    }
  }
  __syncthreads();
  const long long bottom = stack - taken;
  for (int i = threadIdx.x >> 5; i < p.batch; i += kPlanThreads / 32)
    for (int j = threadIdx.x & 31; j < sNeed[i]; j += 32)
      p.table[static_cast<long long>(i) * p.width + sHave[i] + j] = p.pool[bottom + sFirst[i] + j];
  if (threadIdx.x == 0) *p.countOut = static_cast<int>(bottom);
}

// Each row's request, position and slot.
__global__ void planRowsKernel(PlanArgs p) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= p.tokens) return;
  int lo = 0, hi = p.batch;  // the first request that ends behind t
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (p.qStarts[m + 1] > t) hi = m;
    else lo = m + 1;
  }
  int position = 0, slot = -1;
  if (lo < p.batch) {
    const int start = p.qStarts[lo], n = p.qStarts[lo + 1] - start, kv = p.kvLens[lo];
    if (kv >= n && kv > 0) {
      position = kv - n + t - start;
      slot = p.table[static_cast<long long>(lo) * p.width + position / p.page] * p.page + position % p.page;
    }
  }
  p.positions[t] = position;
  p.slots[t] = slot;
  p.requests[t] = lo < p.batch ? lo : -1;
}

}  // namespace
}  // namespace model
}  // namespace vccl

using namespace vccl;

extern "C" vcclResult_t vcclPagePlan(const int* lens, const int* newLens, const unsigned char* finished, int* table,
                                     int* freePages, const int* freeCount, int batch, int width, int poolSize,
                                     int pageSize, int tokens, int* positions, int* slots, int* requests,
                                     int* qStarts, int* kvLens, int* lensOut, int* countOut, vcclStream_t stream) {
  if (!lens || !newLens || !table || !freePages || !freeCount || !qStarts || !kvLens || !lensOut || !countOut ||
      batch <= 0 || batch > model::kPlanMaxBatch || width <= 0 || poolSize <= 0 || pageSize <= 0 || tokens < 0 ||
      static_cast<long long>(poolSize) * pageSize > INT_MAX || static_cast<long long>(width) * pageSize > INT_MAX ||
      (tokens > 0 && (!positions || !slots || !requests)))
    return vcclInvalidArgument;
  TraceRange trace("vccl PagePlan");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const model::PlanArgs p{lens,   newLens,  finished, table,     freePages, freeCount, batch,  width,   poolSize,
                          pageSize, tokens, positions, slots,    requests,  qStarts,   kvLens, lensOut, countOut};
  const size_t smem = static_cast<size_t>(batch) * 3 * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(model::planStateKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               model::kPlanMaxBatch * 3 * static_cast<int>(sizeof(int)));
    if (e != cudaSuccess) {
      VERR("vcclPagePlan: %s", cudaGetErrorString(e));
      return vcclSystemError;
    }
  }
  model::planStateKernel<<<1, model::kPlanThreads, smem, st>>>(p);
  if (tokens > 0) model::planRowsKernel<<<(tokens + 255) / 256, 256, 0, st>>>(p);
  return model::launched("vcclPagePlan");
}

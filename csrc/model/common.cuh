// SPDX-License-Identifier: Apache-2.0
// Shared by the model operators: 8-element vectors of 16-bit types, checks
// of tensor descriptions, launch results.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common/log.h"
#include "common/trace.h"
#include "vccl_model.h"

namespace vccl {
namespace model {

// Rows of a call: row numbers rounded up to whole blocks stay in an int.
constexpr int kMaxTokens = 1 << 30;
inline bool tokensOk(int tokens) { return tokens >= 0 && tokens <= kMaxTokens; }

// 16-byte vectors: base and strides in whole vectors, and strides and head
// counts that the kernels' index arithmetic holds (products are 64 bits).
inline bool headsOk(const vcclHeads_t* h, int elemBytes) {
  if (h == nullptr || h->data == nullptr || h->heads <= 0 || h->heads > 32768) return false;
  const long long vec = 16 / elemBytes, most = 1ll << 31;
  return (reinterpret_cast<uintptr_t>(h->data) & 15u) == 0 && h->tokenStride % vec == 0 && h->headStride % vec == 0 &&
         h->tokenStride >= 0 && h->tokenStride < most && h->headStride >= 0 && h->headStride < most;
}

inline bool cacheOk(const vcclKv4_t* c) {
  return c != nullptr && c->data != nullptr && (reinterpret_cast<uintptr_t>(c->data) & 15u) == 0 && c->pages > 0 &&
         c->pageSize > 0 && c->pageSize % 16 == 0 && c->kvHeads > 0 && (c->D == 64 || c->D == 128) &&
         static_cast<long long>(c->pages) * c->pageSize <= INT32_MAX;
}

inline vcclResult_t launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return vcclSuccess;
  VERR("%s: %s", what, cudaGetErrorString(e));
  return vcclSystemError;
}

// Raises a kernel's shared-memory limit, once for each device.
template <typename Kernel>
inline cudaError_t allowShared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// T is __nv_bfloat16 or __half.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]);

template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]);

template <>
__device__ __forceinline__ uint4 pack8<__nv_bfloat16>(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <>
__device__ __forceinline__ uint4 pack8<__half>(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two f32 in one register pair, worked on by one instruction.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pair(float x) { return pair(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ float2 unpair(uint64_t v) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }

}  // namespace model
}  // namespace vccl

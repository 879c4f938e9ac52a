// SPDX-License-Identifier: Apache-2.0
// The 4-bit key/value block: where everything stands, and how a value is
// rounded to 4 bits.
//
// A block of 16 tokens of one head (18 * D bytes, D = 64 * G):
//   [0, 8D)      key codes, one row of D / 2 bytes a token, tokens in order
//   [8D, 16D)    value codes, likewise; of each eight tokens the even ones first
//   [16D, 17D)   keys: per token and group of 64 channels bf16 scale, bf16 midpoint
//   [17D, 18D)   values: the same
//
// The order of channels inside a row is the order in which the lanes of a
// warp hold the fragments of mma.m16n8k16, so that attention loads codes from
// global memory straight into the registers the tensor cores read:
//   * a 32-bit word holds 8 neighbouring channels; nibble n < 4 is channel 2n,
//     nibble n >= 4 channel 2(n - 4) + 1, so `word & 0x000F000F` is a pair of
//     neighbouring channels in the two 16-bit halves;
//   * keys (rows of the A operand are tokens, its columns channels): lane
//     quarter q of a row of lanes owns channels 16q .. 16q + 15 of every
//     group, stored together: word ((b / 2) * G + group) * 2 + b % 2 for
//     block b of 8 channels;
//   * values (rows of A are channels, columns tokens): lane row g owns
//     channels 8g .. 8g + 7 of every group: word b * G + group.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace vccl {
namespace kv4 {

constexpr int kBlockTokens = 16;
constexpr int kGroup = 64;

__host__ __device__ __forceinline__ int blockBytes(int D) { return 18 * D; }

// Row of value codes that token t of a block has.
__device__ __forceinline__ int valueRow(int t) { return (t & 8) + ((t & 1) << 2) + ((t & 7) >> 1); }

// Word of a row for block b (0..7) of 8 channels in a group.
__device__ __forceinline__ int keyWord(int b, int group, int G) { return ((b >> 1) * G + group) * 2 + (b & 1); }
__device__ __forceinline__ int valueWord(int b, int group, int G) { return b * G + group; }

__device__ __forceinline__ float minNan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float maxNan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight channels of a group held by one of eight neighbouring lanes (mask:
// the lanes that run) -> the word of codes; scale and midpoint (equal in the
// eight lanes) packed as two bf16.  Every step is one IEEE operation in f32,
// so the bytes are the same on every machine:
//   scale = bf16((max - min) / 15), mid = bf16((max + min) / 2),
//   code = clamp(rint((x - mid) / scale + 7.5), 0, 15).
// A group whose scale or midpoint is not finite is stored as NaN.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], unsigned mask, uint32_t* params) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; i++) {
    lo = minNan(lo, x[i]);
    hi = maxNan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = minNan(lo, __shfl_xor_sync(mask, lo, o));
    hi = maxNan(hi, __shfl_xor_sync(mask, hi, o));
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
  const __nv_bfloat16 mb = __float2bfloat16_rn(__fmul_rn(__fadd_rn(hi, lo), 0.5f));
  const float s = __bfloat162float(sb), m = __bfloat162float(mb);
  if (!(isfinite(s) && isfinite(m))) {
    *params = 0x7FC07FC0u;
    return 0;
  }
  *params = static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | (static_cast<uint32_t>(__bfloat16_as_ushort(mb)) << 16);
  const float d = s > 0.0f ? s : 1.0f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float r = rintf(__fadd_rn(__fdiv_rn(__fsub_rn(x[i], m), d), 7.5f));
    const uint32_t c = static_cast<uint32_t>(fminf(fmaxf(r, 0.0f), 15.0f));
    w |= c << (4 * ((i >> 1) + 4 * (i & 1)));
  }
  return w;
}

__device__ __forceinline__ float bf16Lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16Hi(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

__device__ __forceinline__ void dequantise8(uint32_t w, uint32_t params, float (&x)[8]) {
  const float s = bf16Lo(params), m = bf16Hi(params);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float c = static_cast<float>((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u);
    x[i] = __fmaf_rn(c - 7.5f, s, m);
  }
}

}  // namespace kv4
}  // namespace vccl

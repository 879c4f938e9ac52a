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

// NaN-propagating extremes of pairs in the 16-bit type (exact).
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
#define VCCL_KV4_EXTREME(name, intrinsic, T, T2)                                                     \
  template <>                                                                                        \
  __device__ __forceinline__ uint32_t name<T>(uint32_t a, uint32_t b) {                              \
    const T2 r = intrinsic(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));      \
    return *reinterpret_cast<const uint32_t*>(&r);                                                   \
  }
VCCL_KV4_EXTREME(min2, __hmin2_nan, __nv_bfloat16, __nv_bfloat162)
VCCL_KV4_EXTREME(max2, __hmax2_nan, __nv_bfloat16, __nv_bfloat162)
VCCL_KV4_EXTREME(min2, __hmin2_nan, __half, __half2)
VCCL_KV4_EXTREME(max2, __hmax2_nan, __half, __half2)
#undef VCCL_KV4_EXTREME

__device__ __forceinline__ float maxNan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float minNan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ void pairToFloat(uint32_t v, float* lo, float* hi);
template <>
__device__ __forceinline__ void pairToFloat<__nv_bfloat16>(uint32_t v, float* lo, float* hi) {
  *lo = __uint_as_float(v << 16);
  *hi = __uint_as_float(v & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void pairToFloat<__half>(uint32_t v, float* lo, float* hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  *lo = f.x;
  *hi = f.y;
}

// Eight channels of a group, held by one of eight neighbouring lanes of a
// warp that runs as a whole -> the word of codes; scale and midpoint (equal
// in the eight lanes) packed as two bf16.  What is stored is defined by one
// IEEE operation in f32 after the other, so the bytes are the same on every
// machine:
//   scale = bf16((max - min) / 15), mid = bf16((max + min) / 2),
//   code = clamp(rint((x - mid) / scale + 7.5), 0, 15).
// A group whose scale or midpoint is not finite is stored as NaN.
//
// Eight divisions a lane made the write of a prompt bound by instructions
// (64 us for 16384 tokens of 8 heads, 46 now; the bytes take 13).  So
// code / 15 = (x - mid) / (15 scale) + 1/2 is a product with 1 / (15 scale),
// held to [0, 1] by the instruction's saturation; 15 times that plus 96 rounds
// to a multiple of 2^-17, which is more than it is off by: where the code is
// on the border of two it comes out as k + 1/2 exactly, and the next addition
// rounds it to even as rint does.  What comes out as k + 1/2 without being it
// (x - mid is then not a whole number of scales; one group in millions) and
// scales next to the smallest take the division.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const uint4& raw, uint32_t* params) {
  uint32_t lo2 = min2<T>(min2<T>(raw.x, raw.y), min2<T>(raw.z, raw.w));
  uint32_t hi2 = max2<T>(max2<T>(raw.x, raw.y), max2<T>(raw.z, raw.w));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo2 = min2<T>(lo2, __shfl_xor_sync(~0u, lo2, o));
    hi2 = max2<T>(hi2, __shfl_xor_sync(~0u, hi2, o));
  }
  float l0, l1, h0, h1;
  pairToFloat<T>(lo2, &l0, &l1);
  pairToFloat<T>(hi2, &h0, &h1);
  const float lo = minNan(l0, l1), hi = maxNan(h0, h1);
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
  const __nv_bfloat16 mb = __float2bfloat16_rn(__fmul_rn(__fadd_rn(hi, lo), 0.5f));
  const float s = __bfloat162float(sb), m = __bfloat162float(mb);
  if (!(isfinite(s) && isfinite(m))) {
    *params = 0x7FC07FC0u;
    return 0;
  }
  *params = static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | (static_cast<uint32_t>(__bfloat16_as_ushort(mb)) << 16);
  const float d = s > 0.0f ? s : 1.0f;
  const float share = __frcp_rn(15.0f * d);
  const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
  // 1.5 * 2^23 - 96: 96 + code becomes a whole number in the low bits.
  constexpr float kWhole = 12582816.0f;
  float a[8], t[8], u[8], worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float x[2];
    pairToFloat<T>(in[i >> 1], &x[0], &x[1]);
    a[i] = __fsub_rn(x[i & 1], m);
    t[i] = __fmaf_rn(__saturatef(__fmaf_rn(a[i], share, 0.5f)), 15.0f, 96.0f);
    u[i] = __fadd_rn(t[i], kWhole);
    worst = fmaxf(worst, fabsf(__fsub_rn(t[i], __fsub_rn(u[i], kWhole))));
  }
  if (worst == 0.5f || d < 1e-30f) {
    bool exact = d >= 1e-30f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const bool border = fabsf(__fsub_rn(t[i], __fsub_rn(u[i], kWhole))) == 0.5f;
      exact = exact && !(border && __fmaf_rn(__fsub_rn(103.5f, t[i]), d, a[i]) != 0.0f);
    }
    if (!exact) {
#pragma unroll 1
      for (int k = 0; k < 8; k++) {
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) q = i == k ? a[i] : q;
        q = __fadd_rn(fminf(fmaxf(rintf(__fadd_rn(__fdiv_rn(q, d), 7.5f)), 0.0f), 15.0f), kWhole + 96.0f);
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = i == k ? q : u[i];
      }
    }
  }
  uint32_t w = 0u - 0x4B400000u * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 8; i++) w += __float_as_uint(u[i]) << (4 * ((i >> 1) + 4 * (i & 1)));
  return w;
}

__device__ __forceinline__ float bf16Lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16Hi(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

__device__ __forceinline__ void dequantise8(uint32_t w, uint32_t params, float (&x)[8]) {
  const float s = bf16Lo(params), m = bf16Hi(params);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int at = 4 * ((i >> 1) + 4 * (i & 1));
    // code at bit 1 of 2^22, whose last bit is worth 1/2: 2^22 + code
    const uint32_t c = (at > 0 ? w >> (at - 1) : w << 1) & 0x1Eu;
    x[i] = __fmaf_rn(__uint_as_float(0x4A800000u | c) - 4194311.5f, s, m);
  }
}

}  // namespace kv4
}  // namespace vccl

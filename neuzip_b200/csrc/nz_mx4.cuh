// Microscaled 4-bit floating point: the format and its conversions.
//
// A row is cut into blocks of 32 consecutive elements (the last one is filled up with zeros).
// For a block with the largest magnitude a,
//     s = 2^max(floor(log2 a) - 2, -127)          one byte, exponent + 127 (e8m0)
//     code = v / s rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign, ties to the
//            even code, magnitudes above 6 to 6   four bits (e2m1)
// so that a / s lies in [4, 8).  A block that holds an infinity or a NaN has the scale byte 255
// and stands for NaN throughout.  Element 2j of a row is the low half of byte j.
//
// Codes lie row by row, 16 bytes a block.  Scales lie as the tensor cores take them: for a tile of
// 128 rows and 128 columns 512 bytes, of which row r, block b of the four has byte
// (r % 32) * 16 + (r / 32) * 4 + b; the two halves of 256 columns (a "step" of the product) follow
// each other, then the steps of a row tile, then the row tiles.  The blocks that fill the last step
// have the scale byte 0.  Every matrix of a stack begins a row tile of its own.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "nz_common.cuh"

namespace nz {

constexpr uint32_t kMxBlock = 32;            // elements that share a scale
constexpr uint32_t kMxStep = 256;            // columns of a step: 128 bytes of codes a row
constexpr uint32_t kMxTileRows = 128;
constexpr uint32_t kMxChunk = 512;           // scales of 128 rows x 128 columns

struct MxShape {
  uint64_t matrices, rows, cols;
  __host__ __device__ uint64_t code_pitch() const { return (cols + kMxBlock - 1) / kMxBlock * 16; }
  __host__ __device__ uint64_t steps() const { return (cols + kMxStep - 1) / kMxStep; }
  __host__ __device__ uint64_t row_tiles() const { return (rows + kMxTileRows - 1) / kMxTileRows; }
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// The scale byte of a block whose largest magnitude has these bits (a NaN's are above infinity's).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t largest_bits) {
  const uint32_t e = largest_bits >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// 1 / s, which is a normal number for every s = 2^-127 .. 2^125; 0 for the NaN scale.
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FFFFFFFu : byte ? byte << 23 : 0x00400000u);
}
// Two magnitudes to codes, the first in the low half; the instruction saturates at 6 and rounds
// ties to even.
__device__ __forceinline__ uint32_t mx_encode2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\t"
      "cvt.u32.u8 %0, b;\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}
// The two numbers of a byte, the low half first.
__device__ __forceinline__ float2 mx_decode2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.u8.u32 b, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
      : "=r"(h)
      : "r"(byte));
  __half2 v;
  memcpy(&v, &h, 4);
  return __half22float2(v);
}

// Checks that the entry points share (they set the error text).
bool mx_shape(const char *who, uint64_t matrices, uint64_t rows, uint64_t cols);
bool mx_dtype(const char *who, int dtype);

// Offset of the scale of row r (in a tile whose scales take `chunks` chunks of 128 rows), block b of
// the step.
__host__ __device__ __forceinline__ uint32_t mx_scale_offset(uint32_t r, uint32_t b, uint32_t chunks) {
  return ((b >> 2) * chunks + (r >> 7)) * kMxChunk + (r & 31u) * 16u + ((r >> 5) & 3u) * 4u + (b & 3u);
}

// Eight consecutive elements of a row, of which `left` exist, as fp32 (the others 0).
template <typename T, bool VEC>
__device__ __forceinline__ void mx_load8(const T *src, int64_t left, float (&v)[8]) {
  if (VEC) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (left > 0) raw = *reinterpret_cast<const uint4 *>(src);
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_float<T>(src[i]) : 0.f;
  }
}

// A warp quantises a step of a row: lane l holds elements 8 l .. 8 l + 7, four lanes a block.
// Gives the lane's eight codes and the scale byte of its block.
__device__ __forceinline__ void mx_quantize8(const float (&v)[8], uint32_t &codes, uint32_t &byte) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
  a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
  byte = mx_scale_byte(a);
  const float inv = mx_inverse_scale(byte);
  codes = 0;
  if (byte != 255u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) codes |= mx_encode2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
  }
}
// The scale bytes of the half step that the lane's half warp holds, as the word at its address.
__device__ __forceinline__ uint32_t mx_pack_scales(uint32_t byte, uint32_t lane) {
  uint32_t word = byte << (8 * ((lane >> 2) & 3u));
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
  return word;
}

}  // namespace nz

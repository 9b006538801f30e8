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
// Storage is the order in which the tensor cores take operands from shared memory, so that a
// product fetches whole runs of it.  A matrix is cut into tiles of 128 rows (the last one is filled
// up with zeros), a tile into steps of 256 columns.  A step lies in one piece: its blocks, one
// after the other, each with 16 bytes for every row of the tile, then its scales.  These are two
// chunks, one for each 128 columns, of 512 bytes in which row r, block b of four has byte
// (r % 32) * 16 + (r / 32) * 4 + b.  The last step has as many blocks as there are; scales of
// blocks that do not exist are 0.  Inputs of a product lie the same way in tiles of another number
// of rows, with all eight blocks in every step and a pair of chunks for every 128 rows.
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
  __host__ __device__ uint64_t blocks() const { return (cols + kMxBlock - 1) / kMxBlock; }
  __host__ __device__ uint64_t steps() const { return (cols + kMxStep - 1) / kMxStep; }
  __host__ __device__ uint64_t row_tiles() const { return (rows + kMxTileRows - 1) / kMxTileRows; }
  // bytes of a row tile of one matrix, of all of them
  __host__ __device__ uint64_t tile_bytes() const {
    return blocks() * (kMxTileRows * 16) + steps() * (2 * kMxChunk);
  }
  __host__ __device__ uint64_t bytes() const { return matrices * row_tiles() * tile_bytes(); }
};
constexpr uint32_t kMxBlockBytes = kMxTileRows * 16;                    // a block of a tile
constexpr uint32_t kMxStepBytes = 8 * kMxBlockBytes + 2 * kMxChunk;     // a full step of a tile

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
// Eight numbers to a word of codes, the first in the lowest bits; the instruction saturates at 6 and
// rounds ties to even.
__device__ __forceinline__ uint32_t mx_encode8(const float2 (&f)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(f[0].x), "f"(f[0].y), "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y));
  return r;
}
// The eight numbers of a word of codes as four pairs of fp16, which holds them exactly.
__device__ __forceinline__ void mx_decode8(uint32_t word, uint32_t (&pair)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(pair[0]), "=r"(pair[1]), "=r"(pair[2]), "=r"(pair[3])
      : "r"(word));
}

// Checks that the entry points share (they set the error text).
bool mx_shape(const char *who, uint64_t matrices, uint64_t rows, uint64_t cols);
bool mx_dtype(const char *who, int dtype);

// How wide rows of 16-bit elements can be read (see mx_load_block).
inline int mx_wide_rows(const void *p, uint64_t stride, uint64_t cols) {
  const uint64_t apart = (uint64_t)(uintptr_t)p | stride * 2 | cols * 2;
  return apart % 32 == 0 ? 2 : apart % 16 == 0 ? 1 : 0;
}

// The product for few rows (nz_mx4_few.cu): whether it takes a call, and the call.
bool mx_few_rows(const MxShape &w, uint64_t n_rows, bool grouped);
int mx_few(const MxShape &w, int dtype, const void *packed, const void *x, uint64_t x_stride, uint64_t n_rows,
           uint64_t per_input, const void *experts, const void *bias, void *y, void *status, cudaStream_t st);

// Offset of the scale of row r (in a tile of up to 128 * chunks rows), block b of the step.
__host__ __device__ __forceinline__ uint32_t mx_scale_offset(uint32_t r, uint32_t b, uint32_t chunks) {
  return ((b >> 2) * chunks + (r >> 7)) * kMxChunk + (r & 31u) * 16u + ((r >> 5) & 3u) * 4u + (b & 3u);
}

// The items w, w + stride, ... of groups of `per` pieces each, without a 64-bit division for every one
// (4096 x 11008 is quantised in 25.0 us so and in 26.6 with divisions, 28672 x 8192 in 105 and 110).
struct MxWalk {
  uint64_t group, far;
  uint32_t piece, near, per;
  __device__ __forceinline__ MxWalk(uint64_t w, uint64_t stride, uint32_t per_)
      : group(w / per_), far(stride / per_), piece((uint32_t)(w % per_)), near((uint32_t)(stride % per_)), per(per_) {}
  __device__ __forceinline__ void next() {
    group += far;
    piece += near;
    if (piece >= per) {
      piece -= per;
      ++group;
    }
  }
};

// Rows that are not even 16-byte aligned go through shared memory, eight rows of 128 columns a warp:
// loads and stores of a warp are then runs of a row, and a thread still has a block.
struct MxTurn {
  uint16_t e[8][136];         // 272 bytes a row: the rows' blocks fall on different banks
};
// Lane l's block (l / 8) of row l % 8.  `src` is column 0 of the lane's row, `cols` how many there are.
__device__ __forceinline__ void mx_load_turned(const void *src, uint32_t cols, MxTurn &t, uint32_t (&w)[16]) {
  const uint32_t lane = threadIdx.x & 31;
  uint16_t v[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint16_t *row = (const uint16_t *)__shfl_sync(0xFFFFFFFFu, (unsigned long long)src, j);
    const uint32_t n = __shfl_sync(0xFFFFFFFFu, cols, j);
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) v[j][c] = 32 * c + lane < n ? __ldg(row + 32 * c + lane) : 0;
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) t.e[j][32 * c + lane] = v[j][c];
  __syncwarp();
  const uint4 *from = reinterpret_cast<const uint4 *>(&t.e[lane & 7u][(lane >> 3) * 32]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 q = from[i];
    w[4 * i] = q.x;
    w[4 * i + 1] = q.y;
    w[4 * i + 2] = q.z;
    w[4 * i + 3] = q.w;
  }
}
// Runs of n <= 128 16-bit elements in shared memory to global memory, ROWS of them by a warp: two elements
// a store, and one where a run begins or ends in the middle of a word.  All are read before any is
// written (one by one, each waits for the one before: 250 cycles a run).  dst[k] is null for no run.
template <int ROWS>
__device__ __forceinline__ void mx_store_runs(uint16_t *const (&dst)[ROWS], const uint16_t *e, uint32_t apart,
                                              uint32_t n) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t word[ROWS][2], ends[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const uint16_t *from = e + k * apart;
    const uint32_t odd = (uint32_t)((uintptr_t)dst[k] >> 1) & 1u, at = 2 * lane + odd;
    word[k][0] = (uint32_t)from[at] | (uint32_t)from[at + 1] << 16;
    word[k][1] = (uint32_t)from[at + 64] | (uint32_t)from[at + 65 < 128 ? at + 65 : 127] << 16;
    ends[k] = (uint32_t)from[0] | (uint32_t)from[n ? n - 1 : 0] << 16;
  }
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (!dst[k]) continue;
    const uint32_t odd = (uint32_t)((uintptr_t)dst[k] >> 1) & 1u, at = 2 * lane + odd;
    if (at + 1 < n) *reinterpret_cast<uint32_t *>(dst[k] + at) = word[k][0];
    if (at + 65 < n) *reinterpret_cast<uint32_t *>(dst[k] + at + 64) = word[k][1];
    if (lane == 0 && odd && n) dst[k][0] = (uint16_t)ends[k];
    if (lane == 31 && n > odd && ((n - odd) & 1u)) dst[k][n - 1] = (uint16_t)(ends[k] >> 16);
  }
}

// The 32 elements of a block, of which `left` exist (the others are 0), as 16 words of two.
// WIDE: 2 = the row is 32-byte aligned, 1 = 16-byte aligned, 0 = neither; left is a multiple of
// 16, of 8, anything.
template <int WIDE>
__device__ __forceinline__ void mx_load_block(const void *src, int64_t left, uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = 0;
  if (WIDE == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (left > 16 * h)
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[8 * h]), "=r"(w[8 * h + 1]), "=r"(w[8 * h + 2]), "=r"(w[8 * h + 3]),
                       "=r"(w[8 * h + 4]), "=r"(w[8 * h + 5]), "=r"(w[8 * h + 6]), "=r"(w[8 * h + 7])
                     : "l"((const uint8_t *)src + 32 * h));
  } else if (WIDE == 1) {
#pragma unroll
    for (int h = 0; h < 4; ++h)
      if (left > 8 * h) {
        const uint4 v = __ldg((const uint4 *)src + h);
        w[4 * h] = v.x;
        w[4 * h + 1] = v.y;
        w[4 * h + 2] = v.z;
        w[4 * h + 3] = v.w;
      }
  } else {
    const uint16_t *e = (const uint16_t *)src;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < left) w[i / 2] |= (uint32_t)__ldg(e + i) << (16 * (i & 1));
  }
}
template <typename T>
__device__ __forceinline__ float2 mx_unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 mx_unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 mx_unpack2<__half>(uint32_t w) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
// The fp32 bits of the largest of two 16-bit magnitudes (which are ordered like whole numbers).
template <typename T> __device__ __forceinline__ uint32_t mx_largest_bits(uint32_t pair);
template <> __device__ __forceinline__ uint32_t mx_largest_bits<__nv_bfloat16>(uint32_t pair) {
  return max(pair & 0xFFFF0000u, pair << 16);
}
template <> __device__ __forceinline__ uint32_t mx_largest_bits<__half>(uint32_t pair) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(pair >> 16, pair & 0xFFFFu)))) & 0x7FFFFFFFu;
}
// Codes and scale byte of a block.
template <typename T>
__device__ __forceinline__ void mx_quantize_block(const uint32_t (&w)[16], uint32_t (&code)[4], uint32_t &byte) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(a) : "r"(w[i] & 0x7FFF7FFFu));
  byte = mx_scale_byte(mx_largest_bits<T>(a));
  const float inv = mx_inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = mx_unpack2<T>(w[4 * i + j]);
      f[j].x *= inv;
      f[j].y *= inv;
    }
    code[i] = byte == 255u ? 0u : mx_encode8(f);
  }
}
// The scale bytes of the four blocks of 128 columns, which lanes l, l + 8, l + 16, l + 24 hold, as
// the word at their address.
__device__ __forceinline__ uint32_t mx_pack_scales(uint32_t byte, uint32_t lane) {
  uint32_t word = byte << (8 * (lane >> 3));
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 16);
  return word;
}

}  // namespace nz

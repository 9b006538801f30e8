// Weights in microscaled 4-bit floating point: quantisation, the way back, row lookup.
// The format is described in nz_mx4.cuh.
#include "nz_mx4.cuh"

namespace nz {

constexpr int kMxThreads = 256;

// One warp per (row, step) of the stack, in a grid-stride loop.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx4_quantize_kernel(const T *__restrict__ in, MxShape s, uint8_t *__restrict__ codes,
                    uint8_t *__restrict__ scales) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t warps = (uint64_t)gridDim.x * (kMxThreads / 32);
  const uint64_t steps = s.steps(), pitch = s.code_pitch(), total = s.matrices * s.rows * steps;
  for (uint64_t w = (uint64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); w < total;
       w += warps) {
    const uint64_t row = w / steps, step = w - row * steps;
    const uint64_t col = step * kMxStep + lane * 8;
    float v[8];
    mx_load8<T, VEC>(in + row * s.cols + col, (int64_t)s.cols - (int64_t)col, v);
    uint32_t code, byte;
    mx_quantize8(v, code, byte);
    if (col / 2 < pitch) *reinterpret_cast<uint32_t *>(codes + row * pitch + col / 2) = code;
    const uint32_t word = mx_pack_scales(byte, lane);
    if ((lane & 15u) == 0) {
      const uint64_t matrix = row / s.rows, r = row - matrix * s.rows;
      const uint64_t tile = matrix * s.row_tiles() + r / kMxTileRows;
      *reinterpret_cast<uint32_t *>(scales + (tile * steps + step) * (2 * kMxChunk) +
                                    mx_scale_offset((uint32_t)(r % kMxTileRows), lane >> 2, 1)) = word;
    }
  }
}

// The way back: one warp per (row, step).  With a list, output row i is row list[i] of the stack
// (zeros and a status bit where there is no such row).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx4_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, MxShape s,
                      const int64_t *__restrict__ list, uint64_t out_rows, T *__restrict__ out,
                      uint32_t *status) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t warps = (uint64_t)gridDim.x * (kMxThreads / 32);
  const uint64_t steps = s.steps(), pitch = s.code_pitch(), total = out_rows * steps;
  for (uint64_t w = (uint64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); w < total;
       w += warps) {
    const uint64_t to = w / steps, step = w - to * steps;
    const uint64_t col = step * kMxStep + lane * 8;
    if (col >= s.cols) continue;
    uint64_t row = to;
    uint32_t code = 0, byte = 0;
    bool there = true;
    if (list) {
      const int64_t want = list[to];
      there = want >= 0 && (uint64_t)want < s.matrices * s.rows;
      row = there ? (uint64_t)want : 0;
      if (!there && lane == 0 && step == 0 && status) atomicOr(status, NZ_STATUS_BAD_INDEX);
    }
    if (there) {
      const uint64_t matrix = row / s.rows, r = row - matrix * s.rows;
      const uint64_t tile = matrix * s.row_tiles() + r / kMxTileRows;
      code = *reinterpret_cast<const uint32_t *>(codes + row * pitch + col / 2);
      byte = scales[(tile * steps + step) * (2 * kMxChunk) +
                    mx_scale_offset((uint32_t)(r % kMxTileRows), lane >> 2, 1)];
    }
    const float scale = mx_scale(byte);
    T e[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = mx_decode2((code >> (8 * i)) & 255u);
      e[2 * i] = from_float<T>(f.x * scale);
      e[2 * i + 1] = from_float<T>(f.y * scale);
    }
    T *dst = out + to * s.cols + col;
    if (VEC) {
      uint4 raw;
      memcpy(&raw, e, 16);
      *reinterpret_cast<uint4 *>(dst) = raw;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < s.cols) dst[i] = e[i];
    }
  }
}

bool mx_shape(const char *who, uint64_t matrices, uint64_t rows, uint64_t cols) {
  // 32-bit row numbers in the product, byte offsets in 64 bits
  if (cols >= (1ull << 31) || rows >= (1ull << 31) || matrices >= (1ull << 31) ||
      matrices * rows >= (1ull << 31)) {
    set_error("%s: a stack of %llu matrices [%llu, %llu] has 2^31 or more rows or columns", who,
              (unsigned long long)matrices, (unsigned long long)rows, (unsigned long long)cols);
    return false;
  }
  return true;
}
bool mx_dtype(const char *who, int dtype) {
  if (dtype == NZ_DTYPE_BF16 || dtype == NZ_DTYPE_FP16) return true;
  set_error("%s: dtype must be NZ_DTYPE_BF16 or NZ_DTYPE_FP16 (got %d)", who, dtype);
  return false;
}
static unsigned mx_grid(uint64_t warps) {
  const uint64_t blocks = (warps + kMxThreads / 32 - 1) / (kMxThreads / 32);
  const uint64_t most = (uint64_t)sm_count() * 8;            // 2048 threads an SM, twice over
  return (unsigned)(blocks < most ? blocks : most);
}

}  // namespace nz

extern "C" uint64_t nz_mx4_code_bytes(uint64_t matrices, uint64_t rows, uint64_t cols) {
  return matrices * rows * nz::MxShape{matrices, rows, cols}.code_pitch();
}

extern "C" uint64_t nz_mx4_scale_bytes(uint64_t matrices, uint64_t rows, uint64_t cols) {
  const nz::MxShape s{matrices, rows, cols};
  return matrices * s.row_tiles() * s.steps() * 2 * nz::kMxChunk;
}

extern "C" int nz_mx4_quantize(const void *in, int dtype, uint64_t matrices, uint64_t rows,
                               uint64_t cols, void *codes, void *scales, void *stream) {
  using namespace nz;
  if (!mx_dtype("nz_mx4_quantize", dtype) || !mx_shape("nz_mx4_quantize", matrices, rows, cols))
    return NZ_E_ARG;
  const MxShape s{matrices, rows, cols};
  const uint64_t warps = matrices * rows * s.steps();
  if (warps == 0) return NZ_OK;
  if (!in || !codes || !scales || ((uintptr_t)in & 1) || ((uintptr_t)codes & 15) ||
      ((uintptr_t)scales & 15)) {
    set_error("nz_mx4_quantize: null or misaligned pointer (codes and scales 16-byte aligned)");
    return NZ_E_ARG;
  }
  const bool vec = cols % 8 == 0 && ((uintptr_t)in & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
#define NZ_MX_GO(T, VEC)                                                                          \
  mx4_quantize_kernel<T, VEC><<<mx_grid(warps), kMxThreads, 0, st>>>((const T *)in, s,            \
                                                                     (uint8_t *)codes, (uint8_t *)scales)
  if (dtype == NZ_DTYPE_BF16) {
    if (vec) NZ_MX_GO(__nv_bfloat16, true); else NZ_MX_GO(__nv_bfloat16, false);
  } else {
    if (vec) NZ_MX_GO(__half, true); else NZ_MX_GO(__half, false);
  }
#undef NZ_MX_GO
  NZ_LAUNCH_CHECK("mx4_quantize_kernel");
  return NZ_OK;
}

static int mx4_dequantize(const char *who, const void *codes, const void *scales, uint64_t matrices,
                          uint64_t rows, uint64_t cols, int dtype, const int64_t *list,
                          uint64_t out_rows, void *out, void *status, void *stream) {
  using namespace nz;
  if (!mx_dtype(who, dtype) || !mx_shape(who, matrices, rows, cols)) return NZ_E_ARG;
  const MxShape s{matrices, rows, cols};
  const uint64_t warps = out_rows * s.steps();
  if (warps == 0) return NZ_OK;
  if (out_rows >= (1ull << 40)) {
    set_error("%s: too many rows", who);
    return NZ_E_ARG;
  }
  const bool held = matrices * rows > 0;       // a list may name rows of an empty table: all are bad
  if ((held && (!codes || !scales)) || !out || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15) ||
      ((uintptr_t)out & 1) || ((uintptr_t)list & 7)) {
    set_error("%s: null or misaligned pointer (codes and scales 16-byte aligned)", who);
    return NZ_E_ARG;
  }
  const bool vec = cols % 8 == 0 && ((uintptr_t)out & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
#define NZ_MX_GO(T, VEC)                                                                     \
  mx4_dequantize_kernel<T, VEC><<<mx_grid(warps), kMxThreads, 0, st>>>(                      \
      (const uint8_t *)codes, (const uint8_t *)scales, s, list, out_rows, (T *)out, (uint32_t *)status)
  if (dtype == NZ_DTYPE_BF16) {
    if (vec) NZ_MX_GO(__nv_bfloat16, true); else NZ_MX_GO(__nv_bfloat16, false);
  } else {
    if (vec) NZ_MX_GO(__half, true); else NZ_MX_GO(__half, false);
  }
#undef NZ_MX_GO
  NZ_LAUNCH_CHECK("mx4_dequantize_kernel");
  return NZ_OK;
}

extern "C" int nz_mx4_dequantize(const void *codes, const void *scales, uint64_t matrices,
                                 uint64_t rows, uint64_t cols, int dtype, void *out, void *stream) {
  return mx4_dequantize("nz_mx4_dequantize", codes, scales, matrices, rows, cols, dtype, nullptr,
                        matrices * rows, out, nullptr, stream);
}

extern "C" int nz_mx4_gather_rows(const void *codes, const void *scales, uint64_t matrices,
                                  uint64_t rows, uint64_t cols, int dtype, const void *row_list,
                                  uint64_t n_list, void *out, void *status, void *stream) {
  if (n_list && !row_list) {
    nz::set_error("nz_mx4_gather_rows: null row list");
    return NZ_E_ARG;
  }
  return mx4_dequantize("nz_mx4_gather_rows", codes, scales, matrices, rows, cols, dtype,
                        (const int64_t *)row_list, n_list, out, status, stream);
}

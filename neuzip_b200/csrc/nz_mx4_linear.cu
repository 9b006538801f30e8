// y = q(x) q(W)^T (+ bias) with both operands in microscaled 4-bit floating point, W one matrix or
// a stack of which every row of the result names one (a mixture-of-experts layer).
#include "nz_mx4.cuh"

namespace nz {

struct MxLinearArgs {
  MxShape w;
  const uint8_t *codes, *scales;
  const void *x;
  uint64_t x_stride;          // elements between rows of x
  uint64_t n_rows;            // rows of y
  uint32_t per_input;         // rows of y that share a row of x
  const int64_t *experts;     // matrix of every row of y, or null
  const void *bias;           // [matrices, rows] or null
  void *y;
  uint32_t *status;
};

// One warp per element of y; a lane takes every 32nd block of the row.
template <typename T>
__global__ void mx4_linear_simple_kernel(const MxLinearArgs p) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t at = (uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (at >= p.n_rows * p.w.rows) return;
  const uint64_t row = at / p.w.rows, n = at - row * p.w.rows;
  T *y = (T *)p.y + at;
  uint64_t e = 0;
  if (p.experts) {
    const int64_t want = p.experts[row];
    if (want < 0 || (uint64_t)want >= p.w.matrices) {
      if (lane == 0) {
        *y = from_float<T>(0.f);
        if (want != -1 && p.status) atomicOr(p.status, NZ_STATUS_BAD_INDEX);
      }
      return;
    }
    e = (uint64_t)want;
  }
  const T *x = (const T *)p.x + row / p.per_input * p.x_stride;
  const uint64_t steps = p.w.steps(), pitch = p.w.code_pitch();
  const uint8_t *code = p.codes + (e * p.w.rows + n) * pitch;
  const uint8_t *scale = p.scales + (e * p.w.row_tiles() + n / kMxTileRows) * steps * (2 * kMxChunk);
  float sum = 0.f;
  for (uint64_t b = lane; b < pitch / 16; b += 32) {
    float v[32];
    uint32_t a = 0;
    for (uint32_t i = 0; i < 32; ++i) {
      v[i] = b * 32 + i < p.w.cols ? to_float<T>(x[b * 32 + i]) : 0.f;
      a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = mx_scale_byte(a);
    const float inv = mx_inverse_scale(byte);
    float part = 0.f;
    for (uint32_t i = 0; i < 16; ++i) {
      const float2 f = mx_decode2(byte == 255u ? 0u : mx_encode2(v[2 * i] * inv, v[2 * i + 1] * inv));
      const float2 g = mx_decode2(code[b * 16 + i]);
      part += f.x * g.x + f.y * g.y;
    }
    const uint32_t sw = scale[b / 8 * (2 * kMxChunk) +
                              mx_scale_offset((uint32_t)(n % kMxTileRows), (uint32_t)(b & 7), 1)];
    sum += part * mx_scale(byte) * mx_scale(sw);
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) {
    if (p.bias) sum += to_float<T>(((const T *)p.bias)[e * p.w.rows + n]);
    *y = from_float<T>(sum);
  }
}

}  // namespace nz

extern "C" uint64_t nz_mx4_linear_workspace_bytes(uint64_t, uint64_t, uint64_t, uint64_t) { return 16; }

extern "C" int nz_mx4_linear(const void *codes, const void *scales, uint64_t matrices, uint64_t rows,
                             uint64_t cols, int dtype, const void *x, uint64_t x_stride,
                             uint64_t n_rows, uint64_t per_input, const void *experts,
                             const void *bias, void *y, void *workspace, uint64_t workspace_bytes,
                             void *status, void *stream) {
  using namespace nz;
  if (!mx_dtype("nz_mx4_linear", dtype) || !mx_shape("nz_mx4_linear", matrices, rows, cols))
    return NZ_E_ARG;
  if (n_rows == 0 || rows == 0) return NZ_OK;
  if (cols == 0 || matrices == 0 || (!experts && matrices != 1)) {
    set_error("nz_mx4_linear: %llu matrices of %llu columns (one matrix, or experts' numbers)",
              (unsigned long long)matrices, (unsigned long long)cols);
    return NZ_E_ARG;
  }
  if (n_rows >= (1ull << 31) || per_input == 0 || n_rows % per_input) {
    set_error("nz_mx4_linear: %llu rows, %llu to an input row", (unsigned long long)n_rows,
              (unsigned long long)per_input);
    return NZ_E_ARG;
  }
  if (n_rows > per_input && x_stride < cols) {
    set_error("nz_mx4_linear: rows of %llu elements cannot be %llu apart", (unsigned long long)cols,
              (unsigned long long)x_stride);
    return NZ_E_ARG;
  }
  if (!codes || !scales || !x || !y || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15) ||
      ((uintptr_t)x & 1) || ((uintptr_t)y & 1) || ((uintptr_t)bias & 1) || ((uintptr_t)experts & 7) ||
      !workspace || ((uintptr_t)workspace & 255)) {
    set_error("nz_mx4_linear: null or misaligned pointer (codes and scales 16-byte, experts 8-byte, "
              "workspace 256-byte aligned)");
    return NZ_E_ARG;
  }
  if (workspace_bytes < nz_mx4_linear_workspace_bytes(matrices, rows, cols, n_rows)) {
    set_error("nz_mx4_linear: workspace of %llu bytes is too small", (unsigned long long)workspace_bytes);
    return NZ_E_CAPACITY;
  }
  const MxLinearArgs p{{matrices, rows, cols}, (const uint8_t *)codes, (const uint8_t *)scales, x,
                       x_stride, n_rows, (uint32_t)per_input, (const int64_t *)experts, bias, y,
                       (uint32_t *)status};
  const uint64_t blocks = (n_rows * rows + 7) / 8;
  if (!blocks) return NZ_OK;
  if (dtype == NZ_DTYPE_BF16)
    mx4_linear_simple_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
  else
    mx4_linear_simple_kernel<__half><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
  NZ_LAUNCH_CHECK("mx4_linear_simple_kernel");
  return NZ_OK;
}

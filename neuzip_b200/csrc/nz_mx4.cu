// Weights in microscaled 4-bit floating point: quantisation, the way back, row lookup.
// Format and storage are described in nz_mx4.cuh.
#include "nz_mx4.cuh"

namespace nz {

constexpr int kMxThreads = 256;

// A thread takes a block, a warp eight rows of four blocks: its loads are whole sectors, its stores
// 128 bytes in a piece.  Warps take items (eight rows, 128 columns) in a grid-stride loop; the rows
// that fill up the last tile are items too.
template <typename T, int WIDE>
__global__ void __launch_bounds__(kMxThreads)
mx4_quantize_kernel(const T *__restrict__ in, MxShape s, uint8_t *__restrict__ packed) {
  __shared__ __align__(16) MxTurn turn[WIDE ? 1 : kMxThreads / 32];
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t warps = (uint64_t)gridDim.x * (kMxThreads / 32);
  const uint32_t halves = 2 * (uint32_t)s.steps(), blocks = (uint32_t)s.blocks();
  const uint32_t tile_groups = (uint32_t)s.row_tiles() * (kMxTileRows / 8);
  const uint64_t tile_bytes = s.tile_bytes(), groups = s.matrices * tile_groups;
  for (MxWalk w((uint64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5), warps, halves); w.group < groups;
       w.next()) {
    const uint64_t group = w.group;
    const uint32_t half = w.piece, block = half * 4 + (lane >> 3);
    const uint64_t matrix = s.matrices == 1 ? 0 : group >> 32 ? group / tile_groups : (uint32_t)group / tile_groups;
    const uint32_t row = (uint32_t)(group - matrix * tile_groups) * 8 + (lane & 7u);
    uint32_t v[16], code[4], byte;
    const T *src = in + (matrix * s.rows + row) * s.cols;
    if (WIDE) {
      const int64_t left = row < s.rows ? (int64_t)s.cols - (int64_t)block * kMxBlock : 0;
      mx_load_block<WIDE>(src + (uint64_t)block * kMxBlock, left, v);
    } else {
      const uint64_t first = (uint64_t)half * 128, left = s.cols > first ? s.cols - first : 0;
      mx_load_turned(src + first, row < s.rows ? (uint32_t)(left < 128 ? left : 128) : 0, turn[threadIdx.x >> 5], v);
    }
    mx_quantize_block<T>(v, code, byte);
    uint8_t *step = packed + (matrix * s.row_tiles() + row / kMxTileRows) * tile_bytes +
                    (uint64_t)(half >> 1) * kMxStepBytes;
    const uint32_t r = row % kMxTileRows, first = (half >> 1) * 8;
    if (block < blocks)
      *reinterpret_cast<uint4 *>(step + (block - first) * kMxBlockBytes + r * 16) =
          make_uint4(code[0], code[1], code[2], code[3]);
    const uint32_t word = mx_pack_scales(byte, lane);
    if (lane < 8) {
      const uint32_t held = blocks - first < 8 ? blocks - first : 8;
      *reinterpret_cast<uint32_t *>(step + held * kMxBlockBytes + mx_scale_offset(r, (half & 1) * 4, 1)) = word;
    }
  }
}

// Where the codes and the scale of a block of a row lie.
struct MxPlace {
  const uint8_t *codes, *scale;
};
__device__ __forceinline__ MxPlace mx_place(const uint8_t *packed, const MxShape &s, uint64_t row, uint32_t block) {
  const uint32_t matrix = s.matrices == 1 ? 0 : (uint32_t)row / (uint32_t)s.rows;    // the stack has < 2^31 rows
  const uint32_t r = (uint32_t)(row - (uint64_t)matrix * s.rows), blocks = (uint32_t)s.blocks(), first = block & ~7u;
  const uint8_t *step = packed + (matrix * s.row_tiles() + r / kMxTileRows) * s.tile_bytes() +
                        (uint64_t)(block >> 3) * kMxStepBytes;
  const uint32_t held = blocks - first < 8 ? blocks - first : 8;
  return {step + (block - first) * kMxBlockBytes + (r % kMxTileRows) * 16,
          step + held * kMxBlockBytes + mx_scale_offset(r % kMxTileRows, block & 7u, 1)};
}
// The row of the stack that is row `to` of the output; false (and a status bit) where the list names
// none.
__device__ __forceinline__ bool mx_listed(const int64_t *list, const MxShape &s, uint64_t to, uint64_t &row,
                                          uint32_t *status) {
  row = to;
  if (!list) return true;
  const int64_t want = __ldg(list + to);
  if (want >= 0 && (uint64_t)want < s.matrices * s.rows) {
    row = (uint64_t)want;
    return true;
  }
  if (status) atomicOr(status, NZ_STATUS_BAD_INDEX);
  return false;
}

// The way back, the same items.  With a list, output row i is row list[i] of the stack (zeros and a
// status bit where there is no such row).
template <typename T, int WIDE>
__global__ void __launch_bounds__(kMxThreads)
mx4_dequantize_kernel(const uint8_t *__restrict__ packed, MxShape s, const int64_t *__restrict__ list,
                      uint64_t out_rows, T *__restrict__ out, uint32_t *status) {
  __shared__ __align__(16) MxTurn turns[WIDE ? 1 : kMxThreads / 32];
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t warps = (uint64_t)gridDim.x * (kMxThreads / 32);
  const uint32_t blocks = (uint32_t)s.blocks(), quads = (blocks + 3) / 4;
  const uint64_t groups = (out_rows + 7) / 8;
  for (MxWalk w((uint64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5), warps, quads); w.group < groups;
       w.next()) {
    const uint64_t group = w.group, to = group * 8 + (lane & 7u);
    const uint32_t quad = w.piece, block = quad * 4 + (lane >> 3);
    uint64_t row;
    uint4 code = make_uint4(0, 0, 0, 0);
    uint32_t byte = 0;
    if (block < blocks && to < out_rows && mx_listed(list, s, to, row, status)) {
      const MxPlace at = mx_place(packed, s, row, block);
      code = __ldg(reinterpret_cast<const uint4 *>(at.codes));
      byte = __ldg(at.scale);
    }
    const float scale = mx_scale(byte);
    const uint32_t c[4] = {code.x, code.y, code.z, code.w};
    uint32_t v[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t pair[4];
      mx_decode8(c[k], pair);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = mx_unpack2<__half>(pair[i]);
        T e[2] = {from_float<T>(f.x * scale), from_float<T>(f.y * scale)};
        memcpy(&v[4 * k + i], e, 4);
      }
    }
    if (WIDE == 0) {
      MxTurn &turn = turns[threadIdx.x >> 5];
      __syncwarp();
      uint4 *own = reinterpret_cast<uint4 *>(&turn.e[lane & 7u][(lane >> 3) * 32]);
#pragma unroll
      for (int i = 0; i < 4; ++i) own[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      __syncwarp();
      const uint64_t first = (uint64_t)quad * 128;
      const uint32_t n = (uint32_t)(s.cols - first < 128 ? s.cols - first : 128);
      for (uint32_t j = 0; j < 8; j += 4) {
        uint16_t *dst[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          dst[k] = group * 8 + j + k < out_rows
                       ? reinterpret_cast<uint16_t *>(out + (group * 8 + j + k) * s.cols + first) : nullptr;
        mx_store_runs<4>(dst, turn.e[j], 136, n);
      }
      continue;
    }
    if (block >= blocks || to >= out_rows) continue;
    T *dst = out + to * s.cols + (uint64_t)block * kMxBlock;
    const uint64_t left = s.cols - (uint64_t)block * kMxBlock;
    if (WIDE == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (left > 16 * h)
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 16 * h),
                       "r"(v[8 * h]), "r"(v[8 * h + 1]), "r"(v[8 * h + 2]), "r"(v[8 * h + 3]),
                       "r"(v[8 * h + 4]), "r"(v[8 * h + 5]), "r"(v[8 * h + 6]), "r"(v[8 * h + 7])
                       : "memory");
    } else {
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (left > 8 * h)
          *reinterpret_cast<uint4 *>(dst + 8 * h) = make_uint4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
    }
  }
}

bool mx_shape(const char *who, uint64_t matrices, uint64_t rows, uint64_t cols) {
  // 32-bit row and block numbers, byte offsets in 64 bits
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
  // what is resident at a time: 5 blocks an SM (4096 x 11008: 25.0 us; 4 an SM 27.6, 6 29.6)
  const uint64_t most = (uint64_t)sm_count() * 5;
  return (unsigned)(blocks < most ? blocks : most);
}
}  // namespace nz

extern "C" uint64_t nz_mx4_bytes(uint64_t matrices, uint64_t rows, uint64_t cols) {
  return nz::MxShape{matrices, rows, cols}.bytes();
}

template <typename T>
static int quantize(const void *in, const nz::MxShape &s, void *packed, cudaStream_t st) {
  using namespace nz;
  const uint64_t warps = s.matrices * s.row_tiles() * (kMxTileRows / 8) * 2 * s.steps();
  const int wide = mx_wide_rows(in, s.cols, s.cols);
  auto kern = wide == 2 ? mx4_quantize_kernel<T, 2> : wide == 1 ? mx4_quantize_kernel<T, 1>
                                                                : mx4_quantize_kernel<T, 0>;
  kern<<<mx_grid(warps), kMxThreads, 0, st>>>((const T *)in, s, (uint8_t *)packed);
  NZ_LAUNCH_CHECK("mx4_quantize_kernel");
  return NZ_OK;
}

extern "C" int nz_mx4_quantize(const void *in, int dtype, uint64_t matrices, uint64_t rows,
                               uint64_t cols, void *packed, void *stream) {
  using namespace nz;
  if (!mx_dtype("nz_mx4_quantize", dtype) || !mx_shape("nz_mx4_quantize", matrices, rows, cols))
    return NZ_E_ARG;
  const MxShape s{matrices, rows, cols};
  if (s.bytes() == 0) return NZ_OK;
  if (!in || !packed || ((uintptr_t)in & 1) || ((uintptr_t)packed & 15)) {
    set_error("nz_mx4_quantize: null or misaligned pointer (stored bytes 16-byte aligned)");
    return NZ_E_ARG;
  }
  return dtype == NZ_DTYPE_BF16 ? quantize<__nv_bfloat16>(in, s, packed, (cudaStream_t)stream)
                                : quantize<__half>(in, s, packed, (cudaStream_t)stream);
}

template <typename T>
static int dequantize(const void *packed, const nz::MxShape &s, const void *list, uint64_t out_rows,
                      void *out, void *status, cudaStream_t st) {
  using namespace nz;
  const int wide = mx_wide_rows(out, s.cols, s.cols);
  const uint64_t warps = (out_rows + 7) / 8 * ((s.blocks() + 3) / 4);
  auto kern = wide == 2 ? mx4_dequantize_kernel<T, 2> : wide == 1 ? mx4_dequantize_kernel<T, 1>
                                                                  : mx4_dequantize_kernel<T, 0>;
  kern<<<mx_grid(warps), kMxThreads, 0, st>>>((const uint8_t *)packed, s, (const int64_t *)list, out_rows,
                                              (T *)out, (uint32_t *)status);
  NZ_LAUNCH_CHECK("mx4_dequantize_kernel");
  return NZ_OK;
}

static int dequantize_checked(const char *who, const void *packed, uint64_t matrices, uint64_t rows,
                              uint64_t cols, int dtype, const void *list, uint64_t out_rows, void *out,
                              void *status, void *stream) {
  using namespace nz;
  if (!mx_dtype(who, dtype) || !mx_shape(who, matrices, rows, cols)) return NZ_E_ARG;
  const MxShape s{matrices, rows, cols};
  if (out_rows == 0 || cols == 0) return NZ_OK;
  if (out_rows >= (1ull << 40)) {
    set_error("%s: too many rows", who);
    return NZ_E_ARG;
  }
  // a list may name rows of an empty table: none of them exists
  if ((s.bytes() && !packed) || !out || ((uintptr_t)packed & 15) || ((uintptr_t)out & 1) ||
      ((uintptr_t)list & 7)) {
    set_error("%s: null or misaligned pointer (stored bytes 16-byte aligned)", who);
    return NZ_E_ARG;
  }
  return dtype == NZ_DTYPE_BF16
             ? dequantize<__nv_bfloat16>(packed, s, list, out_rows, out, status, (cudaStream_t)stream)
             : dequantize<__half>(packed, s, list, out_rows, out, status, (cudaStream_t)stream);
}

extern "C" int nz_mx4_dequantize(const void *packed, uint64_t matrices, uint64_t rows, uint64_t cols,
                                 int dtype, void *out, void *stream) {
  return dequantize_checked("nz_mx4_dequantize", packed, matrices, rows, cols, dtype, nullptr,
                            matrices * rows, out, nullptr, stream);
}

extern "C" int nz_mx4_gather_rows(const void *packed, uint64_t matrices, uint64_t rows, uint64_t cols,
                                  int dtype, const void *row_list, uint64_t n_list, void *out,
                                  void *status, void *stream) {
  if (n_list && !row_list) {
    nz::set_error("nz_mx4_gather_rows: null row list");
    return NZ_E_ARG;
  }
  return dequantize_checked("nz_mx4_gather_rows", packed, matrices, rows, cols, dtype, row_list, n_list,
                            out, status, stream);
}

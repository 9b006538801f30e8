// The 4-bit product for few rows of x (the single tokens of generation), one launch: y = q(x) q(W)^T
// where W's bytes are what has to be moved and the tensor cores have nothing to gain.
//
// A lane is a row of W (a feature): storage holds 16 bytes of a block for 32 consecutive rows in
// 512 consecutive bytes, one wide load of a warp.  The warps of a CTA share out the steps of 32
// features; every one requests a whole step (eight blocks) before it needs it, the first one
// before the rows of x are quantised, which every CTA does for itself.  Twice an e2m1 number is a
// whole number of at most 12: codes become bytes by a byte permutation that looks up a table of
// eight (a set sign bit gives 0, so that one permutation gives the positive numbers and one, with
// the sign bits turned over, the negative ones), and dp4a adds products of four.  A block's sum is
// exact; it is scaled by a power of two and added in fp32.  What bounds it is those instructions,
// 44 for 32 weights, as much as memory.
#include <atomic>

#include "nz_mx4.cuh"

namespace nz {

constexpr int kMxFewWarps = 16;
constexpr uint32_t kMxFewSmem = 96 * 1024;

struct MxFewArgs {
  MxShape w;
  const uint8_t *packed;
  uint64_t tile_bytes;
  uint32_t blocks, steps;
  const void *x;
  uint64_t x_stride;
  int wide;                   // how x can be loaded, see mx_load_block
  uint32_t n_rows, per_input;
  const int64_t *experts;
  const void *bias;
  void *y;
  uint32_t *status;
};

// 2^(a + b - 256), a and b scale bytes: the scales of two blocks of doubled codes; exact down to
// 2^-149, the largest finite power where it would overflow (no finite sum needs that one).
__device__ __forceinline__ float mx_few_scale(uint32_t a, uint32_t b) {
  if (a == 255u || b == 255u) return __uint_as_float(0x7FFFFFFFu);
  const int e = (int)(a + b) - 256 + 127;
  if (e > 0) return __uint_as_float((uint32_t)(e < 254 ? e : 254) << 23);
  return e > -23 ? __uint_as_float(0x00800000u >> (1 - e)) : 0.f;
}

// The bytes of four codes (the low half of `word`): positive numbers, and magnitudes of negative
// ones with the sign bits turned over.
__device__ __forceinline__ uint32_t mx_few_bytes(uint32_t word) {
  // in PTX the fourth bit of a selector stands for the chosen byte's sign, which is 0 for all eight
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(0x03020100u), "r"(0x0C080604u), "r"(word));
  return r;
}

template <typename T, int NT>
__global__ void __launch_bounds__(kMxFewWarps * 32) mx4_few_kernel(const MxFewArgs p) {
  extern __shared__ uint4 few_smem[];
  __shared__ float sums[kMxFewWarps][NT][32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t feature = blockIdx.x * 32 + lane;
  // dense: NT rows of x; a stack: one row of y
  uint32_t row0 = blockIdx.y * NT;
  uint64_t matrix = 0;
  if (p.experts) {
    const int64_t e = __ldg(p.experts + row0);
    if (e < 0 || (uint64_t)e >= p.w.matrices) {
      if (threadIdx.x < 32 && feature < p.w.rows)
        ((T *)p.y)[(uint64_t)row0 * p.w.rows + feature] = from_float<T>(0.f);
      if (e != -1 && threadIdx.x == 0 && p.status) atomicOr(p.status, NZ_STATUS_BAD_INDEX);
      return;
    }
    matrix = (uint64_t)e;
  }
  const uint32_t tile = feature / kMxTileRows, in_tile = feature % kMxTileRows;
  const uint8_t *w = p.packed + (matrix * p.w.row_tiles() + tile) * p.tile_bytes;

  uint4 code[8];
  uint32_t scale[2];
  auto request = [&](uint32_t step) {
    const uint8_t *at = w + (uint64_t)step * kMxStepBytes;
    const uint32_t held = min(8u, p.blocks - 8 * step);
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b) {
      code[b] = make_uint4(0, 0, 0, 0);
      if (b < held)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(code[b].x), "=r"(code[b].y), "=r"(code[b].z), "=r"(code[b].w)
                     : "l"(at + b * kMxBlockBytes + in_tile * 16));
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      asm volatile("ld.global.nc.u32 %0, [%1];"
                   : "=r"(scale[h])
                   : "l"(at + held * kMxBlockBytes + mx_scale_offset(in_tile, 4 * h, 1)));
  };
  if (warp < p.steps) request(warp);

  // x: for every row 8 words of doubled numbers a block, then the scale bytes
  uint4 *xq = few_smem;
  uint8_t *xs = reinterpret_cast<uint8_t *>(few_smem + (size_t)NT * p.blocks * 2);
  for (uint32_t i = threadIdx.x; i < NT * p.blocks; i += blockDim.x) {
    const uint32_t t = i / p.blocks, block = i - t * p.blocks;
    const uint32_t row = row0 + t;
    uint32_t v[16], c[4], byte;
    const T *src = (const T *)p.x + row / p.per_input * p.x_stride + (uint64_t)block * kMxBlock;
    const int64_t left = row < p.n_rows ? (int64_t)p.w.cols - (int64_t)block * kMxBlock : 0;
    if (p.wide == 2) mx_load_block<2>(src, left, v);
    else if (p.wide == 1) mx_load_block<1>(src, left, v);
    else mx_load_block<0>(src, left, v);
    mx_quantize_block<T>(v, c, byte);
    uint32_t q[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // positive numbers minus the magnitudes of negative ones, byte by byte
      q[2 * k] = __vsub4(mx_few_bytes(c[k]), mx_few_bytes(c[k] ^ 0x88888888u));
      q[2 * k + 1] = __vsub4(mx_few_bytes(c[k] >> 16), mx_few_bytes((c[k] ^ 0x88888888u) >> 16));
    }
    xq[2 * i] = make_uint4(q[0], q[1], q[2], q[3]);
    xq[2 * i + 1] = make_uint4(q[4], q[5], q[6], q[7]);
    xs[i] = (uint8_t)byte;
  }
  __syncthreads();

  float sum[NT] = {};
  for (uint32_t step = warp; step < p.steps; step += warps) {
    const uint32_t held = min(8u, p.blocks - 8 * step);
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b) {
      if (b >= held) break;
      const uint32_t word[4] = {code[b].x, code[b].y, code[b].z, code[b].w};
      const uint32_t ws = (scale[b >> 2] >> (8 * (b & 3u))) & 255u;
      int dot[NT] = {}, neg[NT] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t plus[4], minus[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t c = word[2 * h + k], d = c ^ 0x88888888u;
          plus[2 * k] = mx_few_bytes(c);
          plus[2 * k + 1] = mx_few_bytes(c >> 16);
          minus[2 * k] = mx_few_bytes(d);
          minus[2 * k + 1] = mx_few_bytes(d >> 16);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint4 x = xq[2 * (t * p.blocks + 8 * step + b) + h];
          const uint32_t xv[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            dot[t] = __dp4a((int)plus[k], (int)xv[k], dot[t]);
            neg[t] = __dp4a((int)minus[k], (int)xv[k], neg[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
        sum[t] = fmaf((float)(dot[t] - neg[t]), mx_few_scale(ws, xs[t * p.blocks + 8 * step + b]), sum[t]);
    }
    if (step + warps < p.steps) request(step + warps);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) sums[warp][t][lane] = sum[t];
  __syncthreads();
  if (warp < NT && row0 + warp < p.n_rows && feature < p.w.rows) {
    float total = 0.f;
    for (uint32_t k = 0; k < warps; ++k) total += sums[k][warp][lane];
    if (p.bias) total += to_float<T>(((const T *)p.bias)[matrix * p.w.rows + feature]);
    ((T *)p.y)[(uint64_t)(row0 + warp) * p.w.rows + feature] = from_float<T>(total);
  }
}

// Whether a product goes this way.  A dense one: up to 4 rows.  With a stack every row reads its
// matrix by itself: that pays as long as rows that share a matrix add little to read (about what
// the sorting and the larger kernel's set-up cost, 12 us or 40 MB).
bool mx_few_rows(const MxShape &w, uint64_t n_rows, bool grouped) {
  if ((grouped ? 1 : n_rows) * (w.blocks() * 33) > kMxFewSmem) return false;
  if (!grouped) return n_rows <= 4;
  if (n_rows > 64) return false;
  double miss = 1;
  for (uint64_t i = 0; i < n_rows; ++i) miss *= 1 - 1.0 / (double)w.matrices;
  const double again = (double)n_rows - (double)w.matrices * (1 - miss);
  return again * (double)(w.row_tiles() * w.tile_bytes()) <= 40e6;
}

template <typename T, int NT>
static int few_launch(const MxFewArgs &p, cudaStream_t st) {
  static std::atomic<bool> done[kMaxDeviceOrdinals];
  int dev = 0;
  NZ_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDeviceOrdinals || !done[dev].load(std::memory_order_acquire)) {
    NZ_CUDA_TRY(cudaFuncSetAttribute(mx4_few_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)kMxFewSmem + 256));
    if (dev >= 0 && dev < kMaxDeviceOrdinals) done[dev].store(true, std::memory_order_release);
  }
  const uint32_t groups = (uint32_t)((p.w.rows + 31) / 32), rows = p.experts ? p.n_rows : 1;
  // 16 warps where the features alone do not fill the SMs
  uint32_t warps = (uint64_t)groups * rows > 2ull * sm_count() ? 8 : kMxFewWarps;
  if (warps > p.steps) warps = p.steps;
  if (warps < NT) warps = NT;                  // a warp adds up and stores a row
  const size_t smem = (size_t)NT * p.blocks * 33;
  mx4_few_kernel<T, NT><<<dim3(groups, rows), warps * 32, (smem + 15) & ~(size_t)15, st>>>(p);
  NZ_LAUNCH_CHECK("mx4_few_kernel");
  return NZ_OK;
}

int mx_few(const MxShape &w, int dtype, const void *packed, const void *x, uint64_t x_stride, uint64_t n_rows,
           uint64_t per_input, const void *experts, const void *bias, void *y, void *status, cudaStream_t st) {
  MxFewArgs p;
  p.w = w;
  p.packed = (const uint8_t *)packed;
  p.tile_bytes = w.tile_bytes();
  p.blocks = (uint32_t)w.blocks();
  p.steps = (uint32_t)w.steps();
  p.x = x;
  p.x_stride = x_stride;
  p.wide = mx_wide_rows(x, x_stride, w.cols);
  p.n_rows = (uint32_t)n_rows;
  p.per_input = (uint32_t)per_input;
  p.experts = (const int64_t *)experts;
  p.bias = bias;
  p.y = y;
  p.status = (uint32_t *)status;
  const bool one = experts || n_rows == 1, two = n_rows == 2;
  if (dtype == NZ_DTYPE_BF16)
    return one ? few_launch<__nv_bfloat16, 1>(p, st) : two ? few_launch<__nv_bfloat16, 2>(p, st)
                                                           : few_launch<__nv_bfloat16, 4>(p, st);
  return one ? few_launch<__half, 1>(p, st) : two ? few_launch<__half, 2>(p, st) : few_launch<__half, 4>(p, st);
}

}  // namespace nz

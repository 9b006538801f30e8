// The 4-bit product for few rows of x (the single tokens of generation), one launch: y = q(x) q(W)^T
// where W's bytes are what has to be moved and the tensor cores have nothing to gain.
//
// A lane is a row of W (a feature): storage holds 16 bytes of a block for 32 consecutive rows in
// 512 consecutive bytes, one wide load of a warp.  One CTA an SM; its 16 warps share out the steps
// of 32 features, or of more where there are few steps, and then go on to the next features.
// Every warp keeps a step or two (4 KB each) on the way, across features too: what a CTA has in
// flight covers the latency of memory, and nothing is waited for between items but the other
// warps' sums.  (A CTA of 8 warps for every 32 features, gone after them, was bound by the
// latencies of its start: 18.5 us for one row through two 4096 x 11008 matrices.)
// Codes become fp16, which holds them and sums of eight products (at most 288, in quarters)
// exactly, two to an instruction; a block's four sums are added in fp32, scaled by a power of two
// and added up.
#include <atomic>

#include "nz_mx4.cuh"

namespace nz {

constexpr int kMxFewWarps = 16;
constexpr int kMxFewRows = 64;               // rows of y with a stack
constexpr uint32_t kMxFewSmem = 128 * 1024;

struct MxFewArgs {
  MxShape w;
  const uint8_t *packed;
  uint64_t tile_bytes;
  uint32_t blocks, steps;
  uint32_t split;             // warps that share out the steps of the same features
  const void *x;
  uint64_t x_stride;
  int wide;                   // how x can be loaded, see mx_load_block
  uint32_t n_rows, per_input;
  const int64_t *experts;
  const void *bias;
  void *y;
  uint32_t *status;
};

// The sum of a block's products times 2^(a + b - 254), the scales of the two blocks, added to `to`; NaN where
// either scale is.  The power may lie far outside fp32 while the product does not (a sum of 1/4 times 2^128, or of
// a thousand times 2^-150): it is multiplied by halves, and only the sum with `to` rounds.
__device__ __forceinline__ float mx_few_add(float sum, uint32_t a, uint32_t b, float to) {
  const int e = (int)(a + b) - 254, h = e >> 1;
  const float first = __uint_as_float((uint32_t)(h + 127) << 23), second = __uint_as_float((uint32_t)(e - h + 127) << 23);
  return fmaf(sum * first, a == 255u || b == 255u ? __uint_as_float(0x7FFFFFFFu) : second, to);
}

__device__ __forceinline__ void mx_few_fma(uint32_t &acc, uint32_t a, uint32_t b) {
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(a), "r"(b));
}
__device__ __forceinline__ float2 mx_few_floats(uint32_t pair) {
  __half2 h;
  memcpy(&h, &pair, 4);
  return __half22float2(h);
}

// A step of 32 rows of W, one a lane.
struct MxFewStep {
  uint4 code[8];
  uint32_t scale[2];
};

template <typename T, int NT>
__global__ void __launch_bounds__(kMxFewWarps * 32, 1) mx4_few_kernel(const MxFewArgs p) {
  extern __shared__ uint4 few_smem[];
  __shared__ float sums[2][kMxFewWarps][NT][32];
  __shared__ int64_t experts[kMxFewRows];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // warps of the same features, first step and stride of each of them
  const uint32_t part = warp & (p.split - 1), sub = warp / p.split;
  const uint32_t wide = kMxFewWarps / p.split * 32;          // features of an item
  const uint32_t strips = ((uint32_t)p.w.rows + wide - 1) / wide;
  const uint32_t items = p.experts ? p.n_rows * strips : strips;
  if (p.experts) {
    if (threadIdx.x < p.n_rows) experts[threadIdx.x] = __ldg(p.experts + threadIdx.x);
    __syncthreads();
  }
  // matrix of an item, or -1
  auto matrix_of = [&](uint32_t item) -> int64_t {
    if (!p.experts) return 0;
    const int64_t e = experts[item / strips];
    return e >= 0 && (uint64_t)e < p.w.matrices ? e : -1;
  };
  // The next step to request, an item or more ahead of the one at work.
  uint32_t next_item = blockIdx.x, next_step = part;
  auto request = [&](MxFewStep &s) {
    while (next_item < items && (next_step >= p.steps || matrix_of(next_item) < 0 ||
                                 next_item % strips * wide + sub * 32 >= p.w.rows)) {
      next_item += gridDim.x;
      next_step = part;
      if (part >= p.steps) return;             // this warp never has a step
    }
    if (next_item >= items) return;
    const uint32_t feature = next_item % strips * wide + sub * 32 + lane, in_tile = feature % kMxTileRows;
    const uint8_t *at = p.packed +
                        ((uint64_t)matrix_of(next_item) * p.w.row_tiles() + feature / kMxTileRows) * p.tile_bytes +
                        (uint64_t)next_step * kMxStepBytes;
    const uint32_t held = min(8u, p.blocks - 8 * next_step);
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b)
      if (b < held)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(s.code[b].x), "=r"(s.code[b].y), "=r"(s.code[b].z), "=r"(s.code[b].w)
                     : "l"(at + b * kMxBlockBytes + in_tile * 16));
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      asm volatile("ld.global.nc.u32 %0, [%1];"
                   : "=r"(s.scale[h])
                   : "l"(at + held * kMxBlockBytes + mx_scale_offset(in_tile, 4 * h, 1)));
    next_step += p.split;
  };
  // x: for every row 16 pairs of numbers a block, then the scale bytes
  uint4 *xq = few_smem;
  uint8_t *xs = reinterpret_cast<uint8_t *>(few_smem + (size_t)NT * p.blocks * 4);
  float sum[NT];
  auto consume = [&](const MxFewStep &s, uint32_t step) {
    const uint32_t held = min(8u, p.blocks - 8 * step);
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b) {
      if (b >= held) break;
      const uint32_t word[4] = {s.code[b].x, s.code[b].y, s.code[b].z, s.code[b].w};
      const uint32_t ws = (s.scale[b >> 2] >> (8 * (b & 3u))) & 255u;
      uint32_t acc[NT][2] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t pair[4];
        mx_decode8(word[k], pair);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint4 x = xq[4 * (t * p.blocks + 8 * step + b) + k];
          mx_few_fma(acc[t][k >> 1], pair[0], x.x);
          mx_few_fma(acc[t][k >> 1], pair[1], x.y);
          mx_few_fma(acc[t][k >> 1], pair[2], x.z);
          mx_few_fma(acc[t][k >> 1], pair[3], x.w);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 f = mx_few_floats(acc[t][0]), g = mx_few_floats(acc[t][1]);
        sum[t] = mx_few_add((f.x + f.y) + (g.x + g.y), ws, xs[t * p.blocks + 8 * step + b], sum[t]);
      }
    }
  };

  MxFewStep even, odd;
  request(even);
  request(odd);
  uint32_t turn = 0, half = 0;
  int64_t have = -1;                           // the row of x (the first of NT) in shared memory
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t row = p.experts ? item / strips : 0, strip = item % strips;
    const int64_t matrix = matrix_of(item);
    const uint32_t feature = strip * wide + sub * 32 + lane;
    if (matrix < 0) {
      if (part == 0 && feature < p.w.rows)
        ((T *)p.y)[(uint64_t)row * p.w.rows + feature] = from_float<T>(0.f);
      if (threadIdx.x == 0 && strip == 0 && experts[row] != -1 && p.status)
        atomicOr(p.status, NZ_STATUS_BAD_INDEX);
      continue;
    }
    if (have != (int64_t)(row / p.per_input)) {
      have = row / p.per_input;
      __syncthreads();                         // the row before has been used
      for (uint32_t i = threadIdx.x; i < NT * p.blocks; i += kMxFewWarps * 32) {
        const uint32_t t = i / p.blocks, block = i - t * p.blocks;
        uint32_t v[16], c[4], byte;
        const T *src = (const T *)p.x + (row + t) / p.per_input * p.x_stride + (uint64_t)block * kMxBlock;
        const int64_t left = row + t < p.n_rows ? (int64_t)p.w.cols - (int64_t)block * kMxBlock : 0;
        if (p.wide == 2) mx_load_block<2>(src, left, v);
        else if (p.wide == 1) mx_load_block<1>(src, left, v);
        else mx_load_block<0>(src, left, v);
        mx_quantize_block<T>(v, c, byte);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t q[4];
          mx_decode8(c[k], q);
          xq[4 * i + k] = make_uint4(q[0], q[1], q[2], q[3]);
        }
        xs[i] = (uint8_t)byte;
      }
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[t] = 0.f;
    if (strip * wide + sub * 32 < p.w.rows)
      for (uint32_t step = part; step < p.steps; step += p.split) {
        if (turn & 1u) {
          consume(odd, step);
          request(odd);
        } else {
          consume(even, step);
          request(even);
        }
        ++turn;
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[half][warp][t][lane] = sum[t];
    // One barrier for an item with a matrix: these sums are written again two such items on, behind the barrier
    // of the one between.  Items without a matrix pass no barrier and take no turn.
    __syncthreads();
    for (int t = part; t < NT; t += p.split)
      if (row + t < p.n_rows && feature < p.w.rows) {
        float total = 0.f;
        for (uint32_t k = 0; k < p.split; ++k) total += sums[half][sub * p.split + k][t][lane];
        if (p.bias) total += to_float<T>(((const T *)p.bias)[(uint64_t)matrix * p.w.rows + feature]);
        ((T *)p.y)[(uint64_t)(row + t) * p.w.rows + feature] = from_float<T>(total);
      }
    half ^= 1u;
  }
}

// Whether a product goes this way: what the CUDA cores have to do, rows of y times elements of a
// matrix, decides.  Measured against the tensor cores' way, in us: one row 4096 x 4096 (16.8 M) 5.6 : 8.2,
// 8192 x 8192 13.8 : 12.8; 1024 x 1024 one row 4.6 : 5.8, two 5.4 : 5.8, four 7.9 : 5.8; one token to 8
// experts 1408 x 2048 (23 M) 8.5 : 8.9, where a step more of columns begins to turn it (1408 x 2080 9.3 : 8.9).
bool mx_few_rows(const MxShape &w, uint64_t n_rows, bool grouped) {
  if ((grouped ? 1 : n_rows) * (w.blocks() * 65) > kMxFewSmem) return false;
  if (n_rows > (grouped ? kMxFewRows : 2)) return false;
  return (double)n_rows * (double)w.rows * (double)w.cols <= 24e6;
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
  const uint32_t wide = kMxFewWarps / p.split * 32;
  const uint64_t items = (p.w.rows + wide - 1) / wide * (p.experts ? p.n_rows : 1);
  const unsigned grid = items < (uint64_t)sm_count() ? (unsigned)items : (unsigned)sm_count();
  const size_t smem = (size_t)NT * p.blocks * 65;
  mx4_few_kernel<T, NT><<<grid, kMxFewWarps * 32, (smem + 15) & ~(size_t)15, st>>>(p);
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
  p.split = 1;
  while (p.split < kMxFewWarps && p.split < p.steps) p.split *= 2;
  p.x = x;
  p.x_stride = x_stride;
  p.wide = mx_wide_rows(x, x_stride, w.cols);
  p.n_rows = (uint32_t)n_rows;
  p.per_input = (uint32_t)per_input;
  p.experts = (const int64_t *)experts;
  p.bias = bias;
  p.y = y;
  p.status = (uint32_t *)status;
  const bool one = experts || n_rows == 1;
  if (dtype == NZ_DTYPE_BF16) return one ? few_launch<__nv_bfloat16, 1>(p, st) : few_launch<__nv_bfloat16, 2>(p, st);
  return one ? few_launch<__half, 1>(p, st) : few_launch<__half, 2>(p, st);
}

}  // namespace nz

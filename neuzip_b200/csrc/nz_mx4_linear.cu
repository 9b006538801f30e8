// y = q(x) q(W)^T (+ bias) with both operands in microscaled 4-bit floating point, W one matrix or
// a stack of which every row of the result names one (a mixture-of-experts layer).
//
// The tensor cores take the stored form as it is: tcgen05.mma kind::mxf4 multiplies 4-bit operands
// from shared memory, scales from tensor memory, and adds in fp32.  Kernels of a call:
//   route      (stack only) puts the rows of y in order of their matrix, in "slots" of p.tok rows
//              of which all have the same matrix; the last slot of a matrix is not full
//   quantise   turns the rows of x into codes and scales, in slot order, in the workspace
//   product    one work item = (slot, tile of 128 rows of W, range of steps of 256 columns)
// A tile of W is the M side of the MMA (128 tensor-memory lanes), a slot the N side (its columns).
#include <cuda.h>
#include <string.h>

#include <mutex>

#include "nz_mx4.cuh"

#include "nz_decode_core.cuh"

namespace nz {

constexpr uint32_t kMxMaxTok = 240;          // rows of x in a slot: what two accumulators leave room for
constexpr uint32_t kMxMaxStages = 12;
constexpr uint32_t kMxABytes = kMxTileRows * 128;            // codes of a tile's step
constexpr uint32_t kMxSfABytes = 2 * kMxChunk;               // and its scales
constexpr int kMxLinThreads = 192;           // TMA, MMA, 4 warps that store
constexpr uint32_t kMxMaxExperts = 8192;
constexpr uint32_t kMxNone = 0xFFFFFFFFu;
// Tensor memory, 512 columns: two accumulators, between and behind them the scales of one step.
constexpr uint32_t kMxAcc1 = 256, kMxSfB = 240, kMxSfA = 496;

struct MxLinearArgs {
  MxShape w;
  const uint8_t *codes, *scales;
  const void *x;
  uint64_t x_stride;          // elements between rows of x
  uint32_t n_rows;            // rows of y
  uint32_t per_input;         // rows of y that share a row of x
  const int64_t *experts;     // matrix of every row of y, or null
  const void *bias;           // [matrices, rows] or null
  void *y;
  uint32_t *status;
  // plan
  uint32_t tok, chunks;       // rows of a slot, 128-row chunks of its scales
  uint32_t slots;             // slots there can be
  uint32_t row_tiles, steps;
  uint32_t split;             // 1: the steps of a tile may be shared between CTAs
  uint32_t stages, stage_bytes;
  // workspace
  uint32_t *n_slots;          // stack: slots that there are
  uint32_t *counters;         // split: arrivals at every tile
  uint32_t *slot_expert, *slot_rows;       // stack: matrix of a slot, rows in it
  uint32_t *row_of;           // stack: row of y at every place of the slots
  uint32_t *place_of;         // stack: place of every row of y, kMxNone without a matrix
  uint8_t *x_codes, *x_scales;
  float *partial;             // split: two [tok][128] pieces a CTA
};

// ------------------------------------------------------------------ PTX
__device__ __forceinline__ void mx_mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mx_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void mx_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void mx_tma_2d(uint32_t dst, const CUtensorMap *map, int32_t c0, int32_t c1,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// Shared-memory matrix descriptors: bits 0-13 address >> 4, 16-29 leading and 32-45 stride byte
// offset >> 4, 46-47 version 1, 61-63 layout.  Codes: K-major, 128-byte swizzle (layout 2), groups
// of 8 rows 1024 bytes apart.  Scales: no swizzle, groups of 8 rows of 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t mx_desc_codes(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t mx_desc_scales(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (8ull << 32) | (1ull << 46);
}
// One chunk of scales (32 rows of 16 bytes) to four tensor-memory columns, the same in all four
// groups of 32 lanes.
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// D (+)= A B^T over 64 columns, a scale per 32 columns of either operand.
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mx_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void mx_tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void mx_tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Bounded wait that also watches the CTA's abort flag; false when it was given up.
__device__ __forceinline__ bool mx_wait(uint32_t bar, uint32_t parity, const volatile uint32_t *abort_flag) {
  for (uint32_t it = 0; it < kMaxWaitIters; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u && *abort_flag) return false;
  }
  return false;
}
// Barrier of the four warps that store, and a vote over them: the same verdict for all, so that none
// waits here for one that has left.
__device__ __forceinline__ void mx_store_barrier() {
  asm volatile("bar.sync 1, 128;" ::: "memory");
}
__device__ __forceinline__ bool mx_store_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// ------------------------------------------------------------------ rows in order of their matrix
// One block.  Counts the rows of every matrix, gives each matrix as many slots as it fills, then
// gives every row a place.  Which rows of a matrix come first is open; no result depends on it.
constexpr int kMxRouteThreads = 1024;
constexpr int kMxRouteBatch = 8;             // numbers a thread reads at a time

__global__ void __launch_bounds__(kMxRouteThreads) mx4_route_kernel(const MxLinearArgs p) {
  extern __shared__ uint32_t route_smem[];
  uint32_t *count = route_smem, *next = route_smem + p.w.matrices;
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t carry;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t experts = (uint32_t)p.w.matrices;
  for (uint32_t e = tid; e < experts; e += kMxRouteThreads) count[e] = 0;
  if (tid == 0) carry = 0;
  if (p.split)
    for (uint32_t i = tid; i < p.slots * p.row_tiles; i += kMxRouteThreads) p.counters[i] = 0;
  __syncthreads();
  for (uint64_t r0 = tid; r0 < p.n_rows; r0 += kMxRouteThreads * kMxRouteBatch) {
    int64_t e[kMxRouteBatch];
#pragma unroll
    for (int i = 0; i < kMxRouteBatch; ++i)
      e[i] = r0 + i * kMxRouteThreads < p.n_rows ? p.experts[r0 + i * kMxRouteThreads] : -1;
#pragma unroll
    for (int i = 0; i < kMxRouteBatch; ++i) {
      if (e[i] >= 0 && e[i] < (int64_t)experts) atomicAdd(&count[e[i]], 1u);
      else if (e[i] != -1 && p.status) atomicOr(p.status, NZ_STATUS_BAD_INDEX);
    }
  }
  __syncthreads();
  for (uint32_t e0 = 0; e0 < experts; e0 += kMxRouteThreads) {
    const uint32_t e = e0 + tid;
    const uint32_t rows = e < experts ? count[e] : 0;
    const uint32_t mine = (rows + p.tok - 1) / p.tok;
    uint32_t sum = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= (uint32_t)o) sum += v;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    uint32_t before = carry;
    for (uint32_t k = 0; k < warp; ++k) before += warp_sum[k];
    const uint32_t first = before + sum - mine;
    if (e < experts) {
      next[e] = first * p.tok;
      for (uint32_t k = 0; k < mine; ++k) {
        p.slot_expert[first + k] = e;
        p.slot_rows[first + k] = rows - k * p.tok < p.tok ? rows - k * p.tok : p.tok;
      }
    }
    __syncthreads();
    if (tid == kMxRouteThreads - 1) carry = before + sum;
    __syncthreads();
  }
  if (tid == 0) *p.n_slots = carry;
  for (uint64_t r0 = tid; r0 < p.n_rows; r0 += kMxRouteThreads * kMxRouteBatch) {
    int64_t e[kMxRouteBatch];
#pragma unroll
    for (int i = 0; i < kMxRouteBatch; ++i)
      e[i] = r0 + i * kMxRouteThreads < p.n_rows ? p.experts[r0 + i * kMxRouteThreads] : -1;
#pragma unroll
    for (int i = 0; i < kMxRouteBatch; ++i) {
      const uint64_t r = r0 + i * kMxRouteThreads;
      if (r >= p.n_rows) continue;
      uint32_t place = kMxNone;
      if (e[i] >= 0 && e[i] < (int64_t)experts) {
        place = atomicAdd(&next[e[i]], 1u);
        p.row_of[place] = (uint32_t)r;
      }
      p.place_of[r] = place;
    }
  }
}

// ------------------------------------------------------------------ the rows of x
// One warp per (row of x, step): quantised once, written to the place of every row of y it serves.
// Rows of y without a matrix are set to zero here.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_quantize_rows_kernel(const MxLinearArgs p) {
  if (p.experts) dependent_wait();
  dependent_trigger();
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t pitch = (uint32_t)p.w.code_pitch(), cols = (uint32_t)p.w.cols;
  if (p.split && !p.experts)
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < p.slots * p.row_tiles; i += gridDim.x * 256)
      p.counters[i] = 0;
  const uint64_t total = (uint64_t)(p.n_rows / p.per_input) * p.steps;
  for (uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (uint64_t)gridDim.x * 8) {
    const uint32_t row = (uint32_t)(w / p.steps), step = (uint32_t)(w - (uint64_t)row * p.steps);
    const uint32_t col = step * kMxStep + lane * 8;
    float v[8];
    mx_load8<T, VEC>((const T *)p.x + row * p.x_stride + col, (int64_t)cols - col, v);
    uint32_t code, byte;
    mx_quantize8(v, code, byte);
    const uint32_t word = mx_pack_scales(byte, lane);
    for (uint32_t j = 0; j < p.per_input; ++j) {
      const uint32_t r = row * p.per_input + j;
      const uint32_t place = p.experts ? p.place_of[r] : r;
      if (place == kMxNone) {
        const uint64_t n = p.w.rows, a = n * step / p.steps, b = n * (step + 1) / p.steps;
        for (uint64_t i = a + lane; i < b; i += 32) ((T *)p.y)[r * n + i] = from_float<T>(0.f);
        continue;
      }
      if (col < 2 * pitch) *reinterpret_cast<uint32_t *>(p.x_codes + (uint64_t)place * pitch + col / 2) = code;
      if ((lane & 15u) == 0) {
        const uint32_t slot = place / p.tok, i = place - slot * p.tok;
        *reinterpret_cast<uint32_t *>(p.x_scales +
                                      ((uint64_t)slot * p.steps + step) * (2 * kMxChunk * p.chunks) +
                                      mx_scale_offset(i, lane >> 2, p.chunks)) = word;
      }
    }
  }
}

// ------------------------------------------------------------------ the product
// The items of a CTA, in the same order for every role of it.  Without splitting a CTA takes every
// gridDim.x-th tile; with it, an equal share of all steps of all tiles, one after the other, so
// that at most its first and its last tile are shared with its neighbours.
struct MxItems {
  uint32_t tiles, steps, split, row_tiles, n_slots;
  uint32_t tile;              // next tile
  uint64_t unit, end;         // split: next and last step
  uint32_t slot, row_tile, k0, k1;     // current item

  __device__ __forceinline__ MxItems(const MxLinearArgs &p, uint32_t n_slots_)
      : tiles(n_slots_ * p.row_tiles), steps(p.steps), split(p.split), row_tiles(p.row_tiles),
        n_slots(n_slots_), tile(blockIdx.x), unit(0), end(0), slot(0), row_tile(0), k0(0), k1(0) {
    if (split) {
      const uint64_t units = (uint64_t)tiles * steps, ctas = sharers(units);
      if (blockIdx.x < ctas) {
        unit = units * blockIdx.x / ctas;
        end = units * (blockIdx.x + 1) / ctas;
      }
    }
  }
  // CTAs with a share: every share has a step at least
  __device__ __forceinline__ uint64_t sharers(uint64_t units) const {
    return units < gridDim.x ? units : gridDim.x;
  }
  // the CTA whose share has this step
  __device__ __forceinline__ uint32_t owner(uint64_t at) const {
    const uint64_t units = (uint64_t)tiles * steps;
    return (uint32_t)(((at + 1) * sharers(units) - 1) / units);
  }
  // Neighbouring tiles share a tile of W with up to 8 slots, and those slots with the next tiles
  // of W, so that what runs at a time reads little from outside L2.
  __device__ __forceinline__ void place(uint32_t t) {
    const uint32_t band = t / (8 * row_tiles), rest = t - band * 8 * row_tiles;
    const uint32_t wide = n_slots - band * 8 < 8 ? n_slots - band * 8 : 8;
    row_tile = rest / wide;
    slot = band * 8 + rest - row_tile * wide;
  }
  __device__ __forceinline__ bool next() {
    if (split) {
      if (unit >= end) return false;
      tile = (uint32_t)(unit / steps);
      k0 = (uint32_t)(unit - (uint64_t)tile * steps);
      const uint64_t left = end - unit;
      k1 = left < steps - k0 ? k0 + (uint32_t)left : steps;
      unit += k1 - k0;
      place(tile);
      return true;
    }
    if (tile >= tiles) return false;
    k0 = 0;
    k1 = steps;
    place(tile);
    tile += gridDim.x;
    return true;
  }
};

// Shared-memory map: stages (1024-aligned; codes of W, codes of x, scales of W, scales of x), then
constexpr uint32_t kMxBarFull = 0, kMxBarEmpty = 8 * kMxMaxStages, kMxBarAccFull = 16 * kMxMaxStages,
                   kMxBarAccEmpty = kMxBarAccFull + 16, kMxBarDrain = kMxBarAccEmpty + 16,
                   kMxTmemSlot = kMxBarDrain + 8,
                   kMxAbortSlot = kMxTmemSlot + 4, kMxLastSlot = kMxAbortSlot + 4, kMxMiscBytes = 256;
static_assert(kMxLastSlot + 4 <= kMxMiscBytes, "barriers");

template <typename T>
__global__ void __launch_bounds__(kMxLinThreads, 1)
mx4_product_kernel(const MxLinearArgs p, const __grid_constant__ CUtensorMap w_map,
                   const __grid_constant__ CUtensorMap x_map) {
  extern __shared__ uint8_t mx_smem[];
  const uint32_t base = (smem_u32(mx_smem) + 1023u) & ~1023u;
  const uint32_t misc_a = base + p.stages * p.stage_bytes;
  uint8_t *misc = mx_smem + (misc_a - smem_u32(mx_smem));
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(misc + kMxAbortSlot);
  volatile uint32_t *last_flag = reinterpret_cast<volatile uint32_t *>(misc + kMxLastSlot);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t x_bytes = p.tok * 128, sfb_bytes = p.chunks * 2 * kMxChunk;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (uint32_t s = 0; s < p.stages; ++s) {
      mbar_init(misc_a + kMxBarFull + 8 * s, 1);
      mbar_init(misc_a + kMxBarEmpty + 8 * s, 1);
    }
    for (uint32_t a = 0; a < 2; ++a) {
      mbar_init(misc_a + kMxBarAccFull + 8 * a, 1);
      mbar_init(misc_a + kMxBarAccEmpty + 8 * a, 4);
    }
    mbar_init(misc_a + kMxBarDrain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  dependent_wait();
  // after the wait: a CTA that holds tensor memory never waits for another kernel
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     misc_a + kMxTmemSlot)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  mx_fence_before();
  __syncthreads();
  mx_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(misc + kMxTmemSlot);
  const uint32_t n_slots = p.experts ? *p.n_slots : p.slots;
  MxItems items(p, n_slots);

  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      uint64_t done = 0;
      bool ok = true;
      while (ok && items.next()) {
        const uint32_t e = p.experts ? p.slot_expert[items.slot] : 0;
        const int32_t w_row = (int32_t)((uint64_t)e * p.w.rows + items.row_tile * kMxTileRows);
        const uint8_t *sfa = p.scales + ((uint64_t)e * p.row_tiles + items.row_tile) * p.steps * kMxSfABytes;
        const uint8_t *sfb = p.x_scales + (uint64_t)items.slot * p.steps * sfb_bytes;
        for (uint32_t k = items.k0; k < items.k1; ++k, ++done) {
          if (done >= p.stages && !mx_wait(misc_a + kMxBarEmpty + 8 * stage, phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t at = base + stage * p.stage_bytes, bar = misc_a + kMxBarFull + 8 * stage;
          mbar_expect_tx(bar, p.stage_bytes);
          mx_tma_2d(at, &w_map, (int32_t)(k * 128), w_row, bar);
          mx_tma_2d(at + kMxABytes, &x_map, (int32_t)(k * 128), (int32_t)(items.slot * p.tok), bar);
          bulk_g2s(at + kMxABytes + x_bytes, sfa + (uint64_t)k * kMxSfABytes, kMxSfABytes, bar);
          bulk_g2s(at + kMxABytes + x_bytes + kMxSfABytes, sfb + (uint64_t)k * sfb_bytes, sfb_bytes, bar);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        if (p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
      }
      // copies still in flight land before the CTA's shared memory is given away: after an abort
      // nobody else waits for them
      if (!ok) {
        const uint64_t from = done > p.stages ? done - p.stages : 0;
        for (uint64_t i = from; i < done; ++i) {
          const uint32_t s = (uint32_t)(i % p.stages), ph = (uint32_t)(i / p.stages) & 1u;
          for (uint32_t it = 0; it < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarFull + 8 * s, ph); ++it) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- tensor cores
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, item = 0;
      bool ok = true;
      const uint32_t k64 = (uint32_t)((p.w.cols + 63) / 64);
      while (ok && items.next()) {
        const uint32_t rows = p.experts ? p.slot_rows[items.slot]
                                        : min(p.tok, p.n_rows - items.slot * p.tok);
        const uint32_t n = (rows + 15u) & ~15u;
        // 4-bit operands (type 1), e8m0 scales, M = 128
        const uint32_t idesc0 = (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | (1u << 27);
        const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u);
        if (item >= 2 && !mx_wait(misc_a + kMxBarAccEmpty + 8 * acc, ((item >> 1) & 1u) ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        mx_fence_after();
        for (uint32_t k = items.k0; k < items.k1; ++k) {
          if (!mx_wait(misc_a + kMxBarFull + 8 * stage, phase, abort_flag)) {
            ok = false;
            break;
          }
          mx_fence_after();
          const uint32_t at = base + stage * p.stage_bytes;
          const uint64_t ad = mx_desc_codes(at), bd = mx_desc_codes(at + kMxABytes);
          const uint32_t sfa = at + kMxABytes + x_bytes, sfb = sfa + kMxSfABytes;
          // copies and products of one thread run in order: the scales of the step before have
          // been used when these replace them
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            mx_copy_scales(tmem + kMxSfA + 4 * h, mx_desc_scales(sfa + h * kMxChunk));
            for (uint32_t c = 0; c < p.chunks; ++c)
              mx_copy_scales(tmem + kMxSfB + 8 * h + 4 * c, mx_desc_scales(sfb + (h * p.chunks + c) * kMxChunk));
          }
          const uint32_t last = min(4u, k64 - 4 * k);
          for (uint32_t j = 0; j < last; ++j) {
            // 64 columns are 32 bytes; the scales of two of them share a tensor-memory column, the
            // second starts at byte 2
            const uint32_t id = (j & 1u) * 2u;
            mx_mma(d, ad + 2 * j, bd + 2 * j, idesc0 | (id << 4) | (id << 29), tmem + kMxSfA + 4 * (j >> 1),
                   tmem + kMxSfB + 8 * (j >> 1), (k > items.k0) | (j > 0));
          }
          mx_commit(misc_a + kMxBarEmpty + 8 * stage);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) mx_commit(misc_a + kMxBarAccFull + 8 * acc);
        ++item;
      }
      if (!ok) {
        if (p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        // what has been issued still uses shared and tensor memory
        mx_commit(misc_a + kMxBarDrain);
        for (uint32_t it = 0; it < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarDrain, 0); ++it) {
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- results
    const uint32_t sub = warp & 3u;                   // tensor-memory lanes 32 sub .. + 31
    uint32_t item = 0;
    while (items.next()) {
      const uint32_t rows = p.experts ? p.slot_rows[items.slot]
                                      : min(p.tok, p.n_rows - items.slot * p.tok);
      const uint32_t e = p.experts ? p.slot_expert[items.slot] : 0;
      const uint32_t feature = items.row_tile * kMxTileRows + 32 * sub + lane;
      const bool real = feature < p.w.rows;
      const float bias = p.bias && real ? to_float<T>(((const T *)p.bias)[e * p.w.rows + feature]) : 0.f;
      const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u) + ((32u * sub) << 16);
      if (!mx_store_all(mx_wait(misc_a + kMxBarAccFull + 8 * acc, (item >> 1) & 1u, abort_flag))) {
        if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      mx_fence_after();
      const uint32_t whole = items.k0 == 0 && items.k1 == items.steps;
      const uint32_t place0 = items.slot * p.tok;
      float *piece = whole ? nullptr
                           : p.partial + ((uint64_t)blockIdx.x * 2 + (items.k0 == 0)) * p.tok * kMxTileRows +
                                 32 * sub + lane;
      for (uint32_t c0 = 0; c0 < rows; c0 += 16) {
        uint32_t v[16];
        mx_tmem_ld16(d + c0, v);
        mx_tmem_ld_wait();
        if (c0 + 16 >= rows) {
          // the last columns are out: the tensor cores may have this accumulator again
          mx_fence_before();
          __syncwarp();
          if (lane == 0) mx_mbar_arrive(misc_a + kMxBarAccEmpty + 8 * acc);
        }
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
          if (c0 + i >= rows) break;
          if (!whole) {
            piece[(uint64_t)(c0 + i) * kMxTileRows] = __uint_as_float(v[i]);
          } else if (real) {
            const uint64_t r = p.experts ? p.row_of[place0 + c0 + i] : place0 + c0 + i;
            ((T *)p.y)[r * p.w.rows + feature] = from_float<T>(__uint_as_float(v[i]) + bias);
          }
        }
      }
      if (!whole) {
        // The CTA that brings the last piece of a tile adds all of them, in the order of the steps.
        const uint32_t t = (uint32_t)((items.unit - 1) / items.steps);
        const uint32_t first = items.owner((uint64_t)t * items.steps);
        const uint32_t last = items.owner((uint64_t)(t + 1) * items.steps - 1);
        __threadfence();
        mx_store_barrier();
        if (threadIdx.x == 64) {
          const uint32_t seen = atomicAdd(p.counters + t, 1u);
          __threadfence();
          *last_flag = seen == last - first;
        }
        mx_store_barrier();
        const bool mine = *last_flag != 0;
        mx_store_barrier();                           // the flag may be written again
        if (mine && real) {
          __threadfence();
          constexpr uint32_t kBatch = 8;
          for (uint32_t t0 = 0; t0 < rows; t0 += kBatch) {
            float sum[kBatch] = {};
            for (uint32_t c = first; c <= last; ++c) {
              const float *from = p.partial + ((uint64_t)c * 2 + (c == first)) * p.tok * kMxTileRows +
                                  32 * sub + lane;
              float add[kBatch];
#pragma unroll
              for (uint32_t i = 0; i < kBatch; ++i)
                add[i] = t0 + i < rows ? __ldcg(from + (uint64_t)(t0 + i) * kMxTileRows) : 0.f;
#pragma unroll
              for (uint32_t i = 0; i < kBatch; ++i) sum[i] += add[i];
            }
#pragma unroll
            for (uint32_t i = 0; i < kBatch; ++i) {
              if (t0 + i >= rows) break;
              const uint64_t r = p.experts ? p.row_of[place0 + t0 + i] : place0 + t0 + i;
              ((T *)p.y)[r * p.w.rows + feature] = from_float<T>(sum[i] + bias);
            }
          }
        }
      }
      ++item;
    }
  }

  // ---- common exit: everybody is done with tensor memory, then it is freed
  __syncwarp();
  mx_fence_before();
  __syncthreads();
  if (warp == 1) {
    mx_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// --------------------------------------------------------------------- host
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn mx_encode_tiled() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)ptr;
  });
  return fn;
}
// Codes as a matrix of bytes [rows, pitch], fetched 128 columns of bytes by `box` rows at a time.
static bool mx_map(CUtensorMap *map, const void *codes, uint64_t rows, uint64_t pitch, uint32_t box) {
  const cuuint64_t dim[2] = {pitch, rows};
  const cuuint64_t stride[1] = {pitch};
  const cuuint32_t size[2] = {128, box}, step[2] = {1, 1};
  return mx_encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dim, stride,
                           size, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct MxPlan {
  uint32_t tok, chunks, row_tiles, steps, split, grid, stages, stage_bytes;
  uint64_t slots;
  uint64_t counters, slot_expert, slot_rows, row_of, place_of, x_codes, x_scales, partial, bytes;
};

static bool mx_plan(const MxShape &w, uint64_t n_rows, bool grouped, MxPlan &g) {
  const uint32_t sms = (uint32_t)sm_count();
  g.row_tiles = (uint32_t)w.row_tiles();
  g.steps = (uint32_t)w.steps();
  const uint64_t groups = grouped ? (w.matrices < n_rows ? w.matrices : n_rows) : 1;
  const uint64_t average = (n_rows + groups - 1) / groups;
  uint64_t tok = (average + 15) / 16 * 16;
  if (tok > kMxMaxTok) tok = kMxMaxTok;
  g.tok = (uint32_t)tok;
  g.chunks = g.tok > 128 ? 2 : 1;
  // every matrix's last slot may be short
  g.slots = grouped ? (n_rows - groups) / tok + groups : (n_rows + tok - 1) / tok;
  const uint64_t tiles = g.slots * g.row_tiles;
  if (g.slots * tok >= (1ull << 31) || tiles >= (1ull << 31)) return false;
  g.split = tiles < 4ull * sms;
  const uint64_t units = g.split ? tiles * g.steps : tiles;
  g.grid = (uint32_t)(units < sms ? units : sms);
  g.stage_bytes = kMxABytes + g.tok * 128 + kMxSfABytes + g.chunks * 2 * kMxChunk;
  g.stages = (kMaxDynamicSmem - 1024 - kMxMiscBytes) / g.stage_bytes;
  if (g.stages > kMxMaxStages) g.stages = kMxMaxStages;
  uint64_t at = 256;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~255ull;
    return here;
  };
  g.counters = take(g.split ? tiles * 4 : 0);
  g.slot_expert = take(grouped ? g.slots * 4 : 0);
  g.slot_rows = take(grouped ? g.slots * 4 : 0);
  g.row_of = take(grouped ? g.slots * tok * 4 : 0);
  g.place_of = take(grouped ? n_rows * 4 : 0);
  g.x_codes = take(g.slots * tok * w.code_pitch());
  g.x_scales = take(g.slots * g.steps * g.chunks * 2 * kMxChunk);
  g.partial = take(g.split ? (uint64_t)g.grid * 2 * tok * kMxTileRows * 4 : 0);
  g.bytes = at;
  return true;
}

// The kernel's shared memory above 48 KB has to be asked for once per device.
template <typename K>
static cudaError_t mx_opt_in(K kern, int bytes, bool (&done)[kMaxDeviceOrdinals]) {
  static std::mutex mu;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && dev < kMaxDeviceOrdinals && done[dev]) return cudaSuccess;
  err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && dev >= 0 && dev < kMaxDeviceOrdinals) done[dev] = true;
  return err;
}

template <typename T>
static int mx_launch(const MxLinearArgs &p, const MxPlan &g, const CUtensorMap &w_map,
                     const CUtensorMap &x_map, cudaStream_t st) {
  static bool product_done[kMaxDeviceOrdinals] = {}, route_done[kMaxDeviceOrdinals] = {};
  NZ_CUDA_TRY(mx_opt_in(mx4_product_kernel<T>, (int)kMaxDynamicSmem, product_done));
  const bool vec = p.w.cols % 8 == 0 && p.x_stride % 8 == 0 && ((uintptr_t)p.x & 15) == 0;
  const uint64_t warps = (uint64_t)(p.n_rows / p.per_input) * p.steps, blocks = (warps + 7) / 8;
  const unsigned most = (unsigned)sm_count() * 8;
  const unsigned grid = blocks < most ? (unsigned)blocks : most;
  auto rows_kernel = vec ? mx4_quantize_rows_kernel<T, true> : mx4_quantize_rows_kernel<T, false>;
  if (p.experts) {
    NZ_CUDA_TRY(mx_opt_in(mx4_route_kernel, (int)(kMxMaxExperts * 8), route_done));
    mx4_route_kernel<<<1, kMxRouteThreads, p.w.matrices * 8, st>>>(p);
    NZ_LAUNCH_CHECK("mx4_route_kernel");
    NZ_CUDA_TRY(launch_dependent(rows_kernel, grid, 256, 0, st, p));
  } else {
    rows_kernel<<<grid, 256, 0, st>>>(p);
    NZ_LAUNCH_CHECK("mx4_quantize_rows_kernel");
  }
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + kMxMiscBytes;
  NZ_CUDA_TRY(launch_dependent(mx4_product_kernel<T>, g.grid, kMxLinThreads, smem, st, p, w_map, x_map));
  return NZ_OK;
}

}  // namespace nz

extern "C" uint64_t nz_mx4_linear_workspace_bytes(uint64_t matrices, uint64_t rows, uint64_t cols,
                                                  uint64_t n_rows) {
  using namespace nz;
  if (matrices == 0 || rows == 0 || cols == 0 || n_rows == 0) return 256;
  MxPlan one, many;
  const MxShape w{matrices, rows, cols};
  uint64_t bytes = 256;
  if (matrices == 1 && mx_plan(w, n_rows, false, one)) bytes = one.bytes;
  if (mx_plan(w, n_rows, true, many) && many.bytes > bytes) bytes = many.bytes;
  return bytes;
}

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
  if (experts && matrices > kMxMaxExperts) {
    set_error("nz_mx4_linear: a stack of %llu matrices, at most %u can be chosen from",
              (unsigned long long)matrices, kMxMaxExperts);
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
  const MxShape w{matrices, rows, cols};
  MxPlan g;
  if (!mx_plan(w, n_rows, experts != nullptr, g)) {
    set_error("nz_mx4_linear: the product of %llu rows is too large for one call", (unsigned long long)n_rows);
    return NZ_E_ARG;
  }
  if (workspace_bytes < g.bytes) {
    set_error("nz_mx4_linear: workspace of %llu bytes is smaller than the %llu required",
              (unsigned long long)workspace_bytes, (unsigned long long)g.bytes);
    return NZ_E_CAPACITY;
  }
  if (!mx_encode_tiled()) {
    set_error("nz_mx4_linear: the driver does not provide cuTensorMapEncodeTiled");
    return NZ_E_CUDA;
  }
  uint8_t *ws = (uint8_t *)workspace;
  CUtensorMap w_map, x_map;
  if (!mx_map(&w_map, codes, matrices * rows, w.code_pitch(), kMxTileRows) ||
      !mx_map(&x_map, ws + g.x_codes, g.slots * g.tok, w.code_pitch(), g.tok)) {
    set_error("nz_mx4_linear: cuTensorMapEncodeTiled failed");
    return NZ_E_CUDA;
  }
  MxLinearArgs p;
  memset(&p, 0, sizeof(p));
  p.w = w;
  p.codes = (const uint8_t *)codes;
  p.scales = (const uint8_t *)scales;
  p.x = x;
  p.x_stride = x_stride;
  p.n_rows = (uint32_t)n_rows;
  p.per_input = (uint32_t)per_input;
  p.experts = (const int64_t *)experts;
  p.bias = bias;
  p.y = y;
  p.status = (uint32_t *)status;
  p.tok = g.tok;
  p.chunks = g.chunks;
  p.slots = (uint32_t)g.slots;
  p.row_tiles = g.row_tiles;
  p.steps = g.steps;
  p.split = g.split;
  p.stages = g.stages;
  p.stage_bytes = g.stage_bytes;
  p.n_slots = (uint32_t *)ws;
  p.counters = (uint32_t *)(ws + g.counters);
  p.slot_expert = (uint32_t *)(ws + g.slot_expert);
  p.slot_rows = (uint32_t *)(ws + g.slot_rows);
  p.row_of = (uint32_t *)(ws + g.row_of);
  p.place_of = (uint32_t *)(ws + g.place_of);
  p.x_codes = ws + g.x_codes;
  p.x_scales = ws + g.x_scales;
  p.partial = (float *)(ws + g.partial);
  return dtype == NZ_DTYPE_BF16 ? mx_launch<__nv_bfloat16>(p, g, w_map, x_map, (cudaStream_t)stream)
                                : mx_launch<__half>(p, g, w_map, x_map, (cudaStream_t)stream);
}

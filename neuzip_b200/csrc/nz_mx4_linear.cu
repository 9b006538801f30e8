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
#include <math.h>
#include <string.h>

#include <mutex>

#include "nz_mx4.cuh"

#include "nz_decode_core.cuh"

namespace nz {

constexpr uint32_t kMxMaxTok = 240;          // rows of x in a slot: what two accumulators leave room for
constexpr uint32_t kMxMaxStages = 12;
constexpr int kMxLinThreads = 192;           // TMA, MMA, 4 warps that store
constexpr uint32_t kMxMaxExperts = 8192;
constexpr uint32_t kMxNone = 0xFFFFFFFFu;
// Tensor memory, 512 columns: two accumulators, between and behind them the scales of one step.
constexpr uint32_t kMxAcc1 = 256, kMxSfB = 240, kMxSfA = 496;

struct MxLinearArgs {
  MxShape w;
  const uint8_t *packed;
  uint64_t tile_bytes;
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
  uint32_t row_tiles, steps, blocks;
  uint32_t x_step_bytes;      // a step of a slot: codes, scales
  uint32_t split;             // 1: the steps of a tile may be shared between CTAs
  uint32_t stages, stage_bytes;
  uint32_t wide_y;            // 1: rows of y are whole 16-byte pieces
  // workspace
  uint32_t *n_slots;          // stack: slots that there are
  uint32_t *counters;         // split: arrivals at every tile
  uint32_t *slot_expert, *slot_rows;       // stack: matrix of a slot, rows in it
  uint32_t *row_of;           // stack: row of y at every place of the slots
  uint32_t *place_of;         // stack: place of every row of y, kMxNone without a matrix
  uint8_t *x_packed;
  float *partial;             // split: a piece [tok][128] of every CTA
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
// Shared-memory matrix descriptors, no swizzle: bits 0-13 address >> 4, 16-29 leading and 32-45
// stride byte offset >> 4, 46-47 version 1.  Codes of a tile of `rows` rows, K-major: groups of 8
// rows of 16 bytes are 128 bytes apart (stride), the next 16 bytes of a row 16 * rows (leading).
// Scales: groups of 8 rows of 16 bytes 128 bytes apart, one column of 16 bytes.
__device__ __forceinline__ uint64_t mx_desc_codes(uint32_t addr, uint32_t rows) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)rows << 16) | (8ull << 32) | (1ull << 46);
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
// The same for a converged warp: one verdict for all lanes.
__device__ __forceinline__ bool mx_wait_warp(uint32_t bar, uint32_t parity, const volatile uint32_t *abort_flag) {
  return __all_sync(0xFFFFFFFFu, mx_wait(bar, parity, abort_flag));
}
// One lane of a converged warp.  The instructions below take their operands from the registers that
// a warp shares; a branch that the compiler knows to be one lane's leaves the operands there, while
// under `lane == 0` every one is moved across first (a step of four products took 1000 cycles to
// issue that way).
__device__ __forceinline__ bool mx_elect() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
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
// As in mx4_quantize_kernel a thread takes a block, a warp eight rows of x of four blocks.  A row is
// quantised once and written to the place of every row of y it serves.  Rows of y without a matrix
// are set to zero here.
template <typename T, int WIDE>
__global__ void __launch_bounds__(256) mx4_quantize_rows_kernel(const MxLinearArgs p) {
  if (p.experts) dependent_wait();
  dependent_trigger();
  const uint32_t lane = threadIdx.x & 31;
  if (p.split && !p.experts)
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < p.slots * p.row_tiles; i += gridDim.x * 256)
      p.counters[i] = 0;
  const uint32_t halves = 2 * p.steps, inputs = p.n_rows / p.per_input;
  const uint64_t total = (uint64_t)((inputs + 7) / 8) * halves;
  for (uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (uint64_t)gridDim.x * 8) {
    const uint32_t group = (uint32_t)(w / halves), half = (uint32_t)(w - (uint64_t)group * halves);
    const uint32_t row = group * 8 + (lane & 7u), block = half * 4 + (lane >> 3);
    uint32_t v[16], code[4], byte;
    const int64_t left = row < inputs ? (int64_t)p.w.cols - (int64_t)block * kMxBlock : 0;
    mx_load_block<WIDE>((const T *)p.x + row * p.x_stride + (uint64_t)block * kMxBlock, left, v);
    mx_quantize_block<T>(v, code, byte);
    const uint32_t word = mx_pack_scales(byte, lane);
    if (row >= inputs) continue;
    for (uint32_t j = 0; j < p.per_input; ++j) {
      const uint32_t r = row * p.per_input + j;
      const uint32_t place = p.experts ? p.place_of[r] : r;
      if (place == kMxNone) {
        // the row's lanes of all its warps share it out
        const uint64_t n = p.w.rows;
        for (uint64_t i = block; i < n; i += 4 * halves) ((T *)p.y)[r * n + i] = from_float<T>(0.f);
        continue;
      }
      const uint32_t slot = place / p.tok, i = place - slot * p.tok;
      uint8_t *step = p.x_packed + ((uint64_t)slot * p.steps + (half >> 1)) * p.x_step_bytes;
      *reinterpret_cast<uint4 *>(step + ((block & 7u) * p.tok + i) * 16) =
          make_uint4(code[0], code[1], code[2], code[3]);
      if (lane < 8)
        *reinterpret_cast<uint32_t *>(step + 128 * p.tok + mx_scale_offset(i, (half & 1) * 4, p.chunks)) = word;
    }
  }
}

// ------------------------------------------------------------------ the product
// The items of a CTA, in the same order for every role of it.  Where there are at least two CTAs
// for every tile, its steps are divided among `pieces` of them; else a CTA takes every
// gridDim.x-th tile.  What an item needs from the slot tables is fetched an item ahead.
struct MxItem {
  uint32_t slot, row_tile, tile, piece, k0, k1, expert, rows;
};
struct MxItems {
  const MxLinearArgs &p;
  uint32_t n_slots, tiles, pieces;
  uint32_t at;                // number of the item that is fetched
  MxItem ahead;

  __device__ __forceinline__ MxItems(const MxLinearArgs &p_, uint32_t n_slots_)
      : p(p_), n_slots(n_slots_), tiles(n_slots_ * p_.row_tiles), pieces(1), at(blockIdx.x) {
    if (p.split && tiles) {
      const uint32_t most = gridDim.x / tiles;
      pieces = most < 1 ? 1 : most < p.steps ? most : p.steps;
    }
    fetch();
  }
  // Neighbouring tiles share a tile of W with up to 8 slots, and those slots with the next tiles
  // of W, so that what runs at a time reads little from outside L2.
  __device__ __forceinline__ void fetch() {
    if (at >= tiles * pieces) return;
    const uint32_t t = at / pieces;
    ahead.tile = t;
    ahead.piece = at - t * pieces;
    ahead.k0 = p.steps * ahead.piece / pieces;
    ahead.k1 = p.steps * (ahead.piece + 1) / pieces;
    const uint32_t band = t / (8 * p.row_tiles), rest = t - band * 8 * p.row_tiles;
    const uint32_t wide = n_slots - band * 8 < 8 ? n_slots - band * 8 : 8;
    ahead.row_tile = rest / wide;
    ahead.slot = band * 8 + rest - ahead.row_tile * wide;
    if (p.experts) {
      ahead.expert = __ldcg(p.slot_expert + ahead.slot);
      ahead.rows = __ldcg(p.slot_rows + ahead.slot);
    } else {
      ahead.expert = 0;
      ahead.rows = min(p.tok, p.n_rows - ahead.slot * p.tok);
    }
  }
  __device__ __forceinline__ bool next(MxItem &item) {
    if (at >= tiles * pieces) return false;
    item = ahead;
    // the same in all lanes; the shuffle lets the compiler know
    item.expert = __shfl_sync(0xFFFFFFFFu, item.expert, 0);
    item.rows = __shfl_sync(0xFFFFFFFFu, item.rows, 0);
    at += gridDim.x;
    fetch();
    return true;
  }
};

// Shared-memory map: stages (a step of a tile of W, a step of a slot), then
constexpr uint32_t kMxBarFull = 0, kMxBarEmpty = 8 * kMxMaxStages, kMxBarAccFull = 16 * kMxMaxStages,
                   kMxBarAccEmpty = kMxBarAccFull + 16, kMxBarDrain = kMxBarAccEmpty + 16,
                   kMxTmemSlot = kMxBarDrain + 8,
                   kMxAbortSlot = kMxTmemSlot + 4, kMxLastSlot = kMxAbortSlot + 4, kMxTurn = 256,
                   kMxMiscBytes = kMxTurn + 4 * 1024;      // 16 rows x 32 features of y for each storing warp
static_assert(kMxLastSlot + 4 <= kMxTurn, "barriers");

template <typename T>
__global__ void __launch_bounds__(kMxLinThreads, 1)
mx4_product_kernel(const MxLinearArgs p) {
  extern __shared__ uint8_t mx_smem[];
  const uint32_t base = (smem_u32(mx_smem) + 127u) & ~127u;
  const uint32_t misc_a = base + p.stages * p.stage_bytes;
  uint8_t *misc = mx_smem + (misc_a - smem_u32(mx_smem));
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(misc + kMxAbortSlot);
  volatile uint32_t *last_flag = reinterpret_cast<volatile uint32_t *>(misc + kMxLastSlot);
  const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

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
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t *>(misc + kMxTmemSlot), 0);
  const uint32_t n_slots = p.experts ? __shfl_sync(0xFFFFFFFFu, __ldcg(p.n_slots), 0) : p.slots;
  MxItems items(p, n_slots);

  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    uint32_t stage = 0, phase = 0;
    uint64_t done = 0;
    bool ok = true;
    MxItem it;
    while (ok && items.next(it)) {
      const uint8_t *w = p.packed + ((uint64_t)it.expert * p.row_tiles + it.row_tile) * p.tile_bytes;
      const uint8_t *x = p.x_packed + (uint64_t)it.slot * p.steps * p.x_step_bytes;
      for (uint32_t k = it.k0; k < it.k1; ++k, ++done) {
        if (done >= p.stages && !mx_wait_warp(misc_a + kMxBarEmpty + 8 * stage, phase ^ 1, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t at = base + stage * p.stage_bytes, bar = misc_a + kMxBarFull + 8 * stage;
        const uint32_t w_bytes = min(8u, p.blocks - 8 * k) * kMxBlockBytes + 2 * kMxChunk;
        if (mx_elect()) {
          mbar_expect_tx(bar, w_bytes + p.x_step_bytes);
          bulk_g2s(at, w + (uint64_t)k * kMxStepBytes, w_bytes, bar);
          bulk_g2s(at + kMxStepBytes, x + (uint64_t)k * p.x_step_bytes, p.x_step_bytes, bar);
        }
        __syncwarp();
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {
      if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
      *abort_flag = 1;
      // copies still in flight land before the CTA's shared memory is given away: after an abort
      // nobody else waits for them
      for (uint64_t i = done > p.stages ? done - p.stages : 0; i < done; ++i) {
        const uint32_t s = (uint32_t)(i % p.stages), ph = (uint32_t)(i / p.stages) & 1u;
        for (uint32_t n = 0; n < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarFull + 8 * s, ph); ++n) {
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- tensor cores
    uint32_t stage = 0, phase = 0, item = 0;
    bool ok = true;
    const uint32_t k64 = (p.blocks + 1) / 2;
    MxItem it;
    while (ok && items.next(it)) {
      const uint32_t n = (it.rows + 15u) & ~15u;
      // 4-bit operands (type 1), e8m0 scales, M = 128
      const uint32_t idesc0 = (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | (1u << 27);
      const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u);
      if (item >= 2 && !mx_wait_warp(misc_a + kMxBarAccEmpty + 8 * acc, ((item >> 1) & 1u) ^ 1u, abort_flag)) {
        ok = false;
        break;
      }
      mx_fence_after();
      for (uint32_t k = it.k0; k < it.k1; ++k) {
        if (!mx_wait_warp(misc_a + kMxBarFull + 8 * stage, phase, abort_flag)) {
          ok = false;
          break;
        }
        mx_fence_after();
        const uint32_t at = base + stage * p.stage_bytes;
        const uint64_t ad = mx_desc_codes(at, kMxTileRows), bd = mx_desc_codes(at + kMxStepBytes, p.tok);
        const uint64_t sfa = mx_desc_scales(at + min(8u, p.blocks - 8 * k) * kMxBlockBytes);
        const uint64_t sfb = mx_desc_scales(at + kMxStepBytes + 128 * p.tok);
        const uint32_t last = min(4u, k64 - 4 * k);
        if (mx_elect()) {
          // copies and products of one thread run in order: the scales of the step before have
          // been used when these replace them
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            mx_copy_scales(tmem + kMxSfA + 4 * h, sfa + h * (kMxChunk >> 4));
            mx_copy_scales(tmem + kMxSfB + 8 * h, sfb + h * p.chunks * (kMxChunk >> 4));
            if (p.chunks == 2) mx_copy_scales(tmem + kMxSfB + 8 * h + 4, sfb + (2 * h + 1) * (kMxChunk >> 4));
          }
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) {
            // 64 columns are two blocks; the scales of four share a tensor-memory column, the second
            // product's start at byte 2
            constexpr uint32_t kSecond = (2u << 4) | (2u << 29);
            if (j < last)
              mx_mma(d, ad + 2 * j * kMxTileRows, bd + 2 * j * p.tok, idesc0 | ((j & 1u) ? kSecond : 0u),
                     tmem + kMxSfA + 4 * (j >> 1), tmem + kMxSfB + 8 * (j >> 1), (k > it.k0) | (j > 0));
          }
          mx_commit(misc_a + kMxBarEmpty + 8 * stage);
          if (k + 1 == it.k1) mx_commit(misc_a + kMxBarAccFull + 8 * acc);
        }
        __syncwarp();
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      ++item;
    }
    if (!ok) {
      if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
      *abort_flag = 1;
      // what has been issued still uses shared and tensor memory
      if (mx_elect()) mx_commit(misc_a + kMxBarDrain);
      __syncwarp();
      for (uint32_t n = 0; n < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarDrain, 0); ++n) {
      }
    }
  } else {
    // ---------------------------------------------------------------- results
    const uint32_t sub = warp & 3u;                   // tensor-memory lanes 32 sub .. + 31
    T *turn = reinterpret_cast<T *>(misc + kMxTurn) + sub * 512;
    uint32_t item = 0;
    MxItem it;
    while (items.next(it)) {
      const uint32_t rows = it.rows, place0 = it.slot * p.tok;
      const uint32_t feature = it.row_tile * kMxTileRows + 32 * sub + lane;
      const bool real = feature < p.w.rows;
      const float bias = p.bias && real ? to_float<T>(((const T *)p.bias)[it.expert * p.w.rows + feature]) : 0.f;
      // 16 rows of y of this warp's 32 features, from a value for every row in each lane
      T *y = (T *)p.y + it.row_tile * kMxTileRows + 32 * sub;
      auto store16 = [&](const float (&f)[16], uint32_t row_here, uint32_t count) {
        if (p.wide_y) {
          // turned in shared memory: four lanes take a row's 64 bytes
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) turn[i * 32 + lane] = from_float<T>(f[i] + bias);
          __syncwarp();
          const bool in = it.row_tile * kMxTileRows + 32 * sub + 8 * (lane & 3u) < p.w.rows;
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t i = 8 * h + (lane >> 2);
            const uint64_t r = __shfl_sync(0xFFFFFFFFu, row_here, i);
            const uint4 piece = *reinterpret_cast<const uint4 *>(turn + i * 32 + 8 * (lane & 3u));
            if (i < count && in) *reinterpret_cast<uint4 *>(y + r * p.w.rows + 8 * (lane & 3u)) = piece;
          }
          __syncwarp();
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            const uint64_t r = __shfl_sync(0xFFFFFFFFu, row_here, i);
            if (i < count && real) y[r * p.w.rows + lane] = from_float<T>(f[i] + bias);
          }
        }
      };
      // lane i of 16 knows the row of y of column c0 + i; fetched 16 columns ahead
      auto row_at = [&](uint32_t c) -> uint32_t {
        if (!p.experts) return place0 + c + (lane & 15u);
        return c + (lane & 15u) < rows ? p.row_of[place0 + c + (lane & 15u)] : 0u;
      };
      uint32_t row_next = row_at(0);
      const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u) + ((32u * sub) << 16);
      if (!mx_store_all(mx_wait(misc_a + kMxBarAccFull + 8 * acc, (item >> 1) & 1u, abort_flag))) {
        if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      mx_fence_after();
      const bool whole = items.pieces == 1;
      float *piece = whole ? nullptr : p.partial + (uint64_t)blockIdx.x * p.tok * kMxTileRows + 32 * sub + lane;
      for (uint32_t c0 = 0; c0 < rows; c0 += 16) {
        uint32_t v[16];
        mx_tmem_ld16(d + c0, v);
        const uint32_t row_here = row_next;
        row_next = row_at(c0 + 16);
        mx_tmem_ld_wait();
        if (c0 + 16 >= rows) {
          // the last columns are out: the tensor cores may have this accumulator again
          mx_fence_before();
          __syncwarp();
          if (lane == 0) mx_mbar_arrive(misc_a + kMxBarAccEmpty + 8 * acc);
        }
        if (!whole) {
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i)
            if (c0 + i < rows) piece[(uint64_t)(c0 + i) * kMxTileRows] = __uint_as_float(v[i]);
        } else {
          float f[16];
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
          store16(f, row_here, rows - c0);
        }
      }
      if (!whole) {
        // The CTA that brings the last piece of a tile adds all of them, in the order of the steps.
        __threadfence();
        mx_store_barrier();
        if (threadIdx.x == 64) {
          const uint32_t seen = atomicAdd(p.counters + it.tile, 1u);
          __threadfence();
          *last_flag = seen == items.pieces - 1;
        }
        mx_store_barrier();
        if (*last_flag) {
          const float *from = p.partial + (uint64_t)it.tile * items.pieces * p.tok * kMxTileRows + 32 * sub + lane;
          for (uint32_t c0 = 0; c0 < rows; c0 += 16) {
            float sum[16] = {};
            const uint32_t row_here = row_at(c0);
            for (uint32_t q0 = 0; q0 < items.pieces; q0 += 4) {
              float add[4][16];                       // loads in flight
#pragma unroll
              for (uint32_t q = 0; q < 4; ++q)
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i)
                  add[q][i] = q0 + q < items.pieces && c0 + i < rows
                                  ? __ldcg(from + ((uint64_t)(q0 + q) * p.tok + c0 + i) * kMxTileRows) : 0.f;
#pragma unroll
              for (uint32_t q = 0; q < 4; ++q)
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) sum[i] += add[q][i];
            }
            store16(sum, row_here, rows - c0);
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
struct MxPlan {
  uint32_t tok, chunks, row_tiles, steps, split, grid, stages, stage_bytes, x_step_bytes;
  uint64_t slots;
  uint64_t counters, slot_expert, slot_rows, row_of, place_of, x_packed, partial, bytes;
};

// The rows of a slot, by an estimate of the time (in cycles) that the product takes with them: an
// SM takes in about 40 bytes a cycle, the tensor cores need 2 cycles a row and step, and what
// an item costs beside its steps grows with its rows.
static double mx_cost(uint64_t tok, double slots, uint64_t row_tiles, uint64_t steps, uint32_t sms) {
  const double tiles = slots * (double)row_tiles;
  double pieces = 1, waves = ceil(tiles / sms);
  if (tiles * 2 <= sms) {
    pieces = floor(sms / tiles);
    if (pieces > (double)steps) pieces = (double)steps;
    waves = 1;
  }
  const double load = (kMxStepBytes + tok * 128.0 + (tok > 128 ? 2 : 1) * 2.0 * kMxChunk) / 40.0;
  const double mma = 2.0 * tok;
  const double step = load > mma ? load : mma;
  return waves * (ceil(steps / pieces) * step + 1000 + 8.0 * tok) +
         (pieces > 1 ? 2000 + 4.0 * tok * pieces : 0);
}

static bool mx_plan(const MxShape &w, uint64_t n_rows, bool grouped, MxPlan &g) {
  const uint32_t sms = (uint32_t)sm_count();
  g.row_tiles = (uint32_t)w.row_tiles();
  g.steps = (uint32_t)w.steps();
  const uint64_t groups = grouped ? (w.matrices < n_rows ? w.matrices : n_rows) : 1;
  // matrices that are likely to be named, and half a slot of each that stays empty
  const double hit = grouped ? (double)w.matrices * (1 - pow(1 - 1.0 / (double)w.matrices, (double)n_rows)) : 1;
  uint64_t tok = 16;
  double best = 0;
  for (uint64_t t = 16; t <= kMxMaxTok; t += 16) {
    double slots = grouped ? (double)n_rows / t + hit / 2 : ceil((double)n_rows / t);
    if (slots < hit) slots = hit;
    const double cost = mx_cost(t, slots, g.row_tiles, g.steps, sms);
    if (t == 16 || cost < best) {
      best = cost;
      tok = t;
    }
  }
  g.tok = (uint32_t)tok;
  g.chunks = g.tok > 128 ? 2 : 1;
  // every matrix's last slot may be short
  g.slots = grouped ? (n_rows - groups) / tok + groups : (n_rows + tok - 1) / tok;
  const uint64_t tiles = g.slots * g.row_tiles;
  if (g.slots * tok >= (1ull << 31) || tiles >= (1ull << 31)) return false;
  // a stack may turn out to need fewer tiles than there can be
  g.split = g.steps > 1 && (grouped ? tiles < 2ull * sms : 2 * tiles <= sms);
  const uint64_t units = g.split ? tiles * g.steps : tiles;
  g.grid = (uint32_t)(units < sms ? units : sms);
  g.x_step_bytes = g.tok * 128 + g.chunks * 2 * kMxChunk;
  g.stage_bytes = kMxStepBytes + g.x_step_bytes;
  g.stages = (kMaxDynamicSmem - 128 - kMxMiscBytes) / g.stage_bytes;
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
  g.x_packed = take(g.slots * g.steps * g.x_step_bytes);
  g.partial = take(g.split ? (uint64_t)g.grid * tok * kMxTileRows * 4 : 0);
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
static int mx_launch(const MxLinearArgs &p, const MxPlan &g, cudaStream_t st) {
  static bool product_done[kMaxDeviceOrdinals] = {}, route_done[kMaxDeviceOrdinals] = {};
  NZ_CUDA_TRY(mx_opt_in(mx4_product_kernel<T>, (int)kMaxDynamicSmem, product_done));
  const int wide = mx_wide_rows(p.x, p.x_stride, p.w.cols);
  const uint64_t warps = (uint64_t)((p.n_rows / p.per_input + 7) / 8) * 2 * p.steps, blocks = (warps + 7) / 8;
  const unsigned most = (unsigned)sm_count() * 8;
  const unsigned grid = blocks < most ? (unsigned)blocks : most;
  auto rows_kernel = wide == 2   ? mx4_quantize_rows_kernel<T, 2>
                     : wide == 1 ? mx4_quantize_rows_kernel<T, 1>
                                 : mx4_quantize_rows_kernel<T, 0>;
  if (p.experts) {
    NZ_CUDA_TRY(mx_opt_in(mx4_route_kernel, (int)(kMxMaxExperts * 8), route_done));
    mx4_route_kernel<<<1, kMxRouteThreads, p.w.matrices * 8, st>>>(p);
    NZ_LAUNCH_CHECK("mx4_route_kernel");
    NZ_CUDA_TRY(launch_dependent(rows_kernel, grid, 256, 0, st, p));
  } else {
    rows_kernel<<<grid, 256, 0, st>>>(p);
    NZ_LAUNCH_CHECK("mx4_quantize_rows_kernel");
  }
  const size_t smem = 128 + (size_t)p.stages * p.stage_bytes + kMxMiscBytes;
  NZ_CUDA_TRY(launch_dependent(mx4_product_kernel<T>, g.grid, kMxLinThreads, smem, st, p));
  return NZ_OK;
}

}  // namespace nz

extern "C" uint64_t nz_mx4_linear_workspace_bytes(uint64_t matrices, uint64_t rows, uint64_t cols,
                                                  uint64_t n_rows, int grouped) {
  using namespace nz;
  const MxShape w{matrices, rows, cols};
  MxPlan g;
  if (matrices == 0 || rows == 0 || cols == 0 || n_rows == 0 || mx_few_rows(w, n_rows, grouped != 0) ||
      !mx_plan(w, n_rows, grouped != 0, g))
    return 0;
  return g.bytes;
}

extern "C" int nz_mx4_linear(const void *packed, uint64_t matrices, uint64_t rows, uint64_t cols, int dtype,
                             const void *x, uint64_t x_stride, uint64_t n_rows, uint64_t per_input,
                             const void *experts, const void *bias, void *y, void *workspace,
                             uint64_t workspace_bytes, void *status, void *stream) {
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
  if (!packed || !x || !y || ((uintptr_t)packed & 15) ||
      ((uintptr_t)x & 1) || ((uintptr_t)y & 1) || ((uintptr_t)bias & 1) || ((uintptr_t)experts & 7) ||
      ((uintptr_t)workspace & 255)) {
    set_error("nz_mx4_linear: null or misaligned pointer (stored bytes 16-byte, experts 8-byte, "
              "workspace 256-byte aligned)");
    return NZ_E_ARG;
  }
  const MxShape w{matrices, rows, cols};
  if (mx_few_rows(w, n_rows, experts != nullptr))
    return mx_few(w, dtype, packed, x, x_stride, n_rows, per_input, experts, bias, y, status,
                  (cudaStream_t)stream);
  MxPlan g;
  if (!mx_plan(w, n_rows, experts != nullptr, g)) {
    set_error("nz_mx4_linear: the product of %llu rows is too large for one call", (unsigned long long)n_rows);
    return NZ_E_ARG;
  }
  if (!workspace || workspace_bytes < g.bytes) {
    set_error("nz_mx4_linear: workspace of %llu bytes is smaller than the %llu required",
              (unsigned long long)workspace_bytes, (unsigned long long)g.bytes);
    return NZ_E_CAPACITY;
  }
  uint8_t *ws = (uint8_t *)workspace;
  MxLinearArgs p;
  memset(&p, 0, sizeof(p));
  p.w = w;
  p.packed = (const uint8_t *)packed;
  p.tile_bytes = w.tile_bytes();
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
  p.blocks = (uint32_t)w.blocks();
  p.x_step_bytes = g.x_step_bytes;
  p.split = g.split;
  p.stages = g.stages;
  p.stage_bytes = g.stage_bytes;
  p.wide_y = rows % 8 == 0 && ((uintptr_t)y & 15) == 0;
  p.n_slots = (uint32_t *)ws;
  p.counters = (uint32_t *)(ws + g.counters);
  p.slot_expert = (uint32_t *)(ws + g.slot_expert);
  p.slot_rows = (uint32_t *)(ws + g.slot_rows);
  p.row_of = (uint32_t *)(ws + g.row_of);
  p.place_of = (uint32_t *)(ws + g.place_of);
  p.x_packed = ws + g.x_packed;
  p.partial = (float *)(ws + g.partial);
  return dtype == NZ_DTYPE_BF16 ? mx_launch<__nv_bfloat16>(p, g, (cudaStream_t)stream)
                                : mx_launch<__half>(p, g, (cudaStream_t)stream);
}

// y = q(x) q(W)^T (+ bias) with both operands in microscaled 4-bit floating point, W one matrix or
// a stack of which every row of the result names one (a mixture-of-experts layer).
//
// The tensor cores take the stored form as it is: tcgen05.mma kind::mxf4 multiplies 4-bit operands from
// shared memory with their scales from tensor memory and adds in fp32 there.  Rows of x that share a
// matrix are brought together in "slots" of up to p.tok (a dense product has slots too).  A tile of
// 128 rows of W is the M side of the products (tensor-memory lanes), a slot the N side (columns), a step
// 256 columns of both.  A step of a tile of W lies in one piece (nz_mx4.cuh): a bulk copy fetches it, no
// tensor map is needed, and memory is read in runs of 17 KB.
//
// One persistent CTA an SM: a thread that copies, a thread that issues, four warps that store.  Steps go
// through a ring of stages (full[s]: bytes have arrived, empty[s]: tcgen05.commit); two accumulators
// let the products of a tile run while the one before is stored.  Each of the two loops is one thread's,
// taken by elect.sync: under `lane == 0` the compiler moves every operand of an instruction across
// the warp first, and a step took 1000 cycles to issue instead of 300.
//
// Ways of running, chosen by an estimate of their times (mx_cost) from sizes alone:
//   few     (nz_mx4_few.cu) one or two rows, or some rows of a stack, on the CUDA cores
//   fused   one launch; every CTA quantises the rows of its slots itself, into shared memory, by 12 warps.
//           The less host time (one launch, no workspace); up to about 4 rows it takes 1 us more on the device
//   alone   a kernel quantises x into the workspace, and the product reads W meanwhile (a programmatic
//           dependent launch): its ring is full of W when the inputs come
//   shared  the same, and the steps of all tiles are divided evenly over the SMs, not tiles; the CTA that
//           finishes a tile last adds its pieces in the order of the steps, so that bits do not depend on
//           who is last
//   pair    two CTAs with cta_group::2: 256 rows of W, half of a slot's step each.  A step then brings 34
//           instead of 51 KB into an SM.  Large products are bound by that traffic and the power it
//           takes: 8192 rows x 8192 x 28672 took 1293 us alone and takes 730 to 790 in pairs under sustained
//           load, and 580 if nothing but scales were copied
// Rows find their slots in every block (up to 1024 rows and 256 matrices) or by a kernel of one block.
//
// Measured on a B200, cold weights, in a graph (the bytes at 6.54 TB/s in brackets, in us; rows x inner x
// outer size): 16 x 4096 x 11008 9.7 (3.7), 16 x 8192 x 8192 12.5 (5.4), 16 x 8192 x 28672 24.7 (19.1);
// 64 experts 2048 x 1408, 32 tokens to 8 each 22.3 (14.8).  What is over the bytes is 6 to 7.5 us.  6 of them
// are the same for all: two launches (2), the first bytes' latency (2), the last step's products and
// stores (1), the end of the grid (1).  The rest grows with what is left uneven in the last wave of tiles
// and, for experts, with finding the rows' slots in every block (1).
#include <cuda.h>
#include <math.h>
#include <string.h>

#include <mutex>

#include "nz_mx4.cuh"

#include "nz_decode_core.cuh"

namespace nz {

constexpr uint32_t kMxMaxTok = 240;          // rows of x in a slot: what two accumulators leave room for
constexpr uint32_t kMxMaxStages = 12;
constexpr int kMxLinThreads = 192;           // a warp that copies, one that issues, 4 that store
constexpr uint32_t kMxHelpers = 8;           // fused: more warps that quantise
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
  uint32_t split;             // > 0: the steps of a tile may be shared, where there are two CTAs or more for
                              // every tile between this many
  uint32_t in_block;          // stack: few rows of y, which every block groups by itself
  uint32_t pair;              // 1: two CTAs share a slot's step and take two tiles of W
  uint32_t x_resident;        // bytes of a slot's steps in shared memory, quantised there; else 0
  int wide;                   // how rows of x can be read, see mx_load_block
  uint32_t stages, stage_bytes;
  uint32_t wide_y;            // 1: rows of y are whole 16-byte pieces
  // workspace
  uint32_t *n_slots;          // stack: slots that there are
  uint32_t *counters;         // split: arrivals at every tile
  uint32_t *slot_expert, *slot_rows;       // stack: matrix of a slot, rows in it
  uint32_t *row_of;           // stack: row of y at every place of the slots
  uint2 *place_of;            // stack: see MxWhere, of every row of y
  uint8_t *x_packed;
  float *partial;             // split: two pieces [tok][128] of every CTA
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
// The instructions of a CTA alone and of a pair of CTAs (PAIR: issued by the pair's first CTA, they
// use both CTAs' shared and tensor memory at the same addresses).
// One chunk of scales (32 rows of 16 bytes) to four tensor-memory columns, the same in all four
// groups of 32 lanes.
template <bool PAIR>
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint64_t desc) {
  if (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// D (+)= A B^T over 64 columns, a scale per 32 columns of either operand.
template <bool PAIR>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// Arrives at the barrier (of both CTAs of a pair) when what this thread has issued is done.
template <bool PAIR>
__device__ __forceinline__ void mx_commit(uint32_t bar) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mx_tmem_alloc(uint32_t slot) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void mx_tmem_free(uint32_t tmem) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}
// This CTA's number in its pair; an arrival at the first CTA's barrier; a barrier of both CTAs.
__device__ __forceinline__ uint32_t mx_pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t mx_of_first(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void mx_arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mx_of_first(bar)) : "memory");
}
// A run of 256-byte rows to this CTA's shared memory; its bytes count at a barrier of either CTA of the
// pair, which only the tensor form of the copy can do.
__device__ __forceinline__ void mx_pair_copy(uint32_t dst, const CUtensorMap *map, int32_t row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(0), "r"(row)
      : "memory");
}
__device__ __forceinline__ void mx_pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mx_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// The same on a barrier at which the other CTA of a pair arrives.
__device__ __forceinline__ bool mx_wait_pair(uint32_t bar, uint32_t parity, const volatile uint32_t *abort_flag) {
  for (uint32_t it = 0; it < kMaxWaitIters; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kWaitHintNs)
        : "memory");
    if (ok) return true;
    if ((it & 63u) == 63u && *abort_flag) return false;
  }
  return false;
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

// Columns of a product for so many rows of x.
__device__ __forceinline__ uint32_t mx_columns(uint32_t rows) { return (rows + 15u) & ~15u; }

// Where a row of x goes: its slot (kMxNone: nowhere); in its low half the row's number in the slot, in its
// high half its place among the codes of a step's first block.  For a pair of CTAs the first half of
// the product's columns lies by itself before the second one.
struct MxWhere {
  uint32_t slot, at;
  __device__ __forceinline__ uint32_t row() const { return at & 0xFFFFu; }
  __device__ __forceinline__ uint32_t code() const { return at >> 16; }
};
__device__ __forceinline__ uint2 mx_where(const MxLinearArgs &p, uint32_t slot, uint32_t i, uint32_t rows) {
  uint32_t code = i;
  if (p.pair) {
    const uint32_t split = mx_columns(rows) / 2;
    if (i >= split) code = 8 * (p.tok / 2) + i - split;
  }
  return make_uint2(slot, code << 16 | i);
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
      count[e] = rows + first * p.tok;             // one past its last place, were its slots without gaps
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
      uint2 where = make_uint2(kMxNone, 0);
      if (e[i] >= 0 && e[i] < (int64_t)experts) {
        const uint32_t place = atomicAdd(&next[e[i]], 1u), slot = place / p.tok;
        p.row_of[place] = (uint32_t)r;
        where = mx_where(p, slot, place - slot * p.tok, min(p.tok, count[e[i]] - slot * p.tok));
      }
      p.place_of[r] = where;
    }
  }
}

// ------------------------------------------------------------------ few rows, in every block
// Up to 1024 rows of y and 256 matrices: the blocks of both kernels work the order out for
// themselves, so that no kernel has to run before them and the product's first copies wait for
// nothing.  Slots follow the matrices' numbers, places within a matrix the rows' numbers.
constexpr uint32_t kMxBlockRows = 1024, kMxBlockExperts = 256;
constexpr uint32_t kMxBlockSlots = kMxBlockExperts + kMxBlockRows / 16;

__device__ __forceinline__ uint32_t mx_expert(const MxLinearArgs &p, uint32_t r) {
  const int64_t e = r < p.n_rows ? __ldg(p.experts + r) : -1;
  return e >= 0 && e < (int64_t)p.w.matrices ? (uint32_t)e : kMxNone;
}
// The first slot of matrix e = the lane's, of 32 consecutive ones, and the slots up to here.
__device__ __forceinline__ uint32_t mx_first_slot(uint32_t mine, uint32_t &before) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= (uint32_t)o) sum += v;
  }
  const uint32_t first = before + sum - mine;
  before += __shfl_sync(0xFFFFFFFFu, sum, 31);
  return first;
}

// Places of all rows (256 threads).
struct MxPlaces {
  uint16_t count[kMxBlockRows / 32][kMxBlockExperts];      // of 32 rows; then, of the rows before them
  uint32_t first[kMxBlockExperts];                         // first place of a matrix
  uint32_t place[kMxBlockRows];
};
__device__ __forceinline__ void mx_find_places(const MxLinearArgs &p, MxPlaces &s) {
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t chunks = (p.n_rows + 31) / 32, experts = (uint32_t)p.w.matrices;
  uint32_t e[4], rank[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) e[i] = mx_expert(p, (warp + 8 * i) * 32 + lane);
  for (uint32_t i = tid; i < chunks * kMxBlockExperts / 2; i += 256) reinterpret_cast<uint32_t *>(s.count)[i] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e[i]);
    rank[i] = __popc(same & ((1u << lane) - 1u));
    if (rank[i] == 0 && e[i] != kMxNone) s.count[warp + 8 * i][e[i]] = (uint16_t)__popc(same);
  }
  __syncthreads();
  if (tid < experts) {
    uint32_t rows = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
      const uint32_t here = s.count[c][tid];
      s.count[c][tid] = (uint16_t)rows;
      rows += here;
    }
    s.first[tid] = (rows + p.tok - 1) / p.tok;
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
      const uint32_t first = mx_first_slot(e0 + lane < experts ? s.first[e0 + lane] : 0, before);
      if (e0 + lane < experts) s.first[e0 + lane] = first * p.tok;
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t r = (warp + 8 * i) * 32 + lane;
    if (r >= p.n_rows) continue;
    uint32_t place = kMxNone;
    if (e[i] != kMxNone) {
      place = s.first[e[i]] + s.count[warp + 8 * i][e[i]] + rank[i];
      if (blockIdx.x == 0) p.row_of[place] = r;
    } else if (blockIdx.x == 0 && p.status && __ldg(p.experts + r) != -1) {
      atomicOr(p.status, NZ_STATUS_BAD_INDEX);
    }
    s.place[r] = place;
  }
  __syncthreads();
}
// The slots alone (all threads of the block): matrix << 18 | number among the matrix's slots << 9 |
// rows of each, their number, and the matrix of every row.
constexpr uint16_t kMxNoMatrix = 0xFFFF;
template <uint32_t THREADS>
__device__ __forceinline__ void mx_find_slots(const MxLinearArgs &p, uint32_t *table, uint32_t *count,
                                              uint16_t *ids, uint32_t *n) {
  const uint32_t lane = threadIdx.x & 31, experts = (uint32_t)p.w.matrices;
  uint32_t e[(kMxBlockRows + THREADS - 1) / THREADS];
#pragma unroll
  for (uint32_t i = 0; i < sizeof(e) / 4; ++i) e[i] = mx_expert(p, threadIdx.x + i * THREADS);
  for (uint32_t i = threadIdx.x; i < experts; i += THREADS) count[i] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < sizeof(e) / 4; ++i) {
    const uint32_t r = threadIdx.x + i * THREADS;
    if (r < kMxBlockRows) ids[r] = (uint16_t)e[i];                 // kMxNone becomes kMxNoMatrix
    if (e[i] != kMxNone) atomicAdd(count + e[i], 1u);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
      const uint32_t rows = e0 + lane < experts ? count[e0 + lane] : 0, mine = (rows + p.tok - 1) / p.tok;
      const uint32_t first = mx_first_slot(mine, before);
      for (uint32_t k = 0; k < mine; ++k)
        table[first + k] = (e0 + lane) << 18 | k << 9 | min(p.tok, rows - k * p.tok);
    }
    if (lane == 0) *n = before;
  }
  __syncthreads();
}
// The rows of the k-th slot of a matrix, in order (a warp).
__device__ __forceinline__ void mx_list_rows(const MxLinearArgs &p, const uint16_t *ids, uint32_t matrix, uint32_t k,
                                             uint16_t *list) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t before = 0;
  for (uint32_t r0 = 0; r0 < p.n_rows; r0 += 32) {
    const bool mine = ids[r0 + lane] == matrix;
    const uint32_t same = __ballot_sync(0xFFFFFFFFu, mine), at = before + __popc(same & ((1u << lane) - 1u)) - k * p.tok;
    if (mine && at < p.tok) list[at] = (uint16_t)(r0 + lane);
    before += __popc(same);
  }
  __syncwarp();
}

// ------------------------------------------------------------------ the rows of x
// As in mx4_quantize_kernel a thread takes a block, a warp eight rows of x of four blocks.  A row is
// quantised once and written to the place of every row of y it serves.  Rows of y without a matrix
// are set to zero here.
template <typename T, int WIDE>
__global__ void __launch_bounds__(256) mx4_quantize_rows_kernel(const MxLinearArgs p) {
  extern __shared__ uint32_t rows_smem[];
  __shared__ __align__(16) MxTurn turn[WIDE ? 1 : 8];
  MxPlaces &places = *reinterpret_cast<MxPlaces *>(rows_smem);       // in_block
  // The product may come in now.  All that was launched before this kernel is complete (its own launch is
  // an ordinary one), W among it, which the product begins to read while this kernel runs.
  dependent_trigger();
  const uint32_t lane = threadIdx.x & 31;
  if (p.in_block) mx_find_places(p, places);
  if (p.split && (!p.experts || p.in_block))
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < p.slots * p.row_tiles; i += gridDim.x * 256)
      p.counters[i] = 0;
  // Items are rows of x, or where there are few of them rows of y: then a row of x that serves several
  // is quantised for each, by warps of their own.
  const uint32_t serves = p.in_block ? 1 : p.per_input, shared = p.per_input / serves;
  constexpr uint32_t kAhead = 4;
  const uint32_t apart = p.pair ? p.tok / 2 : p.tok;            // rows of a block of codes
  const uint32_t halves = 2 * p.steps, inputs = p.n_rows / serves;
  const uint32_t groups = (inputs + 7) / 8;
  for (MxWalk w((uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (uint64_t)gridDim.x * 8, halves); w.group < groups;
       w.next()) {
    const uint32_t group = (uint32_t)w.group, half = w.piece;
    const uint32_t row = group * 8 + (lane & 7u), block = half * 4 + (lane >> 3);
    uint32_t v[16], code[4], byte;
    // where the row goes, known before the row is there
    uint2 where[kAhead];
    auto find = [&](uint32_t j0) {
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        const uint32_t r = row * serves + j0 + j;
        if (row >= inputs || j0 + j >= serves) continue;
        if (p.in_block || !p.experts) {
          const uint32_t place = p.in_block ? places.place[r] : r, slot = place / p.tok;
          where[j] = place == kMxNone ? make_uint2(kMxNone, 0)
                                      : mx_where(p, slot, place - slot * p.tok, min(p.tok, p.n_rows - slot * p.tok));
        } else {
          where[j] = __ldcg(p.place_of + r);
        }
      }
    };
    find(0);
    const T *src = (const T *)p.x + row / shared * p.x_stride;
    if (WIDE) {
      const int64_t left = row < inputs ? (int64_t)p.w.cols - (int64_t)block * kMxBlock : 0;
      mx_load_block<WIDE>(src + (uint64_t)block * kMxBlock, left, v);
    } else {
      const uint64_t first = (uint64_t)half * 128, left = p.w.cols > first ? p.w.cols - first : 0;
      mx_load_turned(src + first, row < inputs ? (uint32_t)(left < 128 ? left : 128) : 0, turn[threadIdx.x >> 5], v);
    }
    mx_quantize_block<T>(v, code, byte);
    const uint32_t word = mx_pack_scales(byte, lane);
    if (row >= inputs) continue;
    for (uint32_t j0 = 0; j0 < serves; j0 += kAhead) {
      if (j0) find(j0);
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        if (j0 + j >= serves) break;
        const MxWhere to{where[j].x, where[j].y};
        if (to.slot == kMxNone) {
          // the row's lanes of all its warps share it out
          const uint64_t n = p.w.rows;
          T *y = (T *)p.y + (uint64_t)(row * serves + j0 + j) * n;
          for (uint64_t i = block; i < n; i += 4 * halves) y[i] = from_float<T>(0.f);
          continue;
        }
        uint8_t *step = p.x_packed + ((uint64_t)to.slot * p.steps + (half >> 1)) * p.x_step_bytes;
        *reinterpret_cast<uint4 *>(step + ((block & 7u) * apart + to.code()) * 16) =
            make_uint4(code[0], code[1], code[2], code[3]);
        if (lane < 8)
          *reinterpret_cast<uint32_t *>(step + 128 * p.tok + mx_scale_offset(to.row(), (half & 1) * 4, p.chunks)) =
              word;
      }
    }
  }
}

// ------------------------------------------------------------------ the product
// The items of a CTA, in the same order for every role of it.  A CTA takes every gridDim.x-th tile;
// or, with p.split, an equal share of all steps of all tiles, one after the other, so that only its
// first and its last tile are shared with its neighbours (where there are two CTAs or more for a
// tile, the shares are equal parts of tiles).  For a pair of CTAs (p.pair, never with p.split) a tile is
// two tiles of W, one for each.  What an item needs from the slot tables is fetched an
// item ahead.
struct MxItem {
  uint32_t slot, row_tile, tile, k0, k1, expert, rows, number;
};
struct MxItems {
  const MxLinearArgs &p;
  const uint32_t *table;      // slots that the block has worked out
  uint32_t n_slots, tiles, across;     // across: tiles that a slot has
  uint32_t shares;            // split: CTAs that have one
  uint32_t at, end;           // next tile, or next and last step
  MxItem ahead;

  __device__ __forceinline__ MxItems(const MxLinearArgs &p_, const uint32_t *table_, uint32_t n_slots_)
      : p(p_), table(table_), n_slots(n_slots_), across(p_.pair ? (p_.row_tiles + 1) / 2 : p_.row_tiles),
        shares(0), at(p_.pair ? blockIdx.x / 2 : blockIdx.x) {
    tiles = end = n_slots * across;
    if (p.split) {
      const uint32_t units = tiles * p.steps;
      shares = gridDim.x;
      if (tiles && 2 * tiles <= gridDim.x) shares = tiles * min(min(gridDim.x / tiles, p.steps), p.split);
      if (shares > units) shares = units;
      at = end = 0;
      if (blockIdx.x < shares) {
        at = units * blockIdx.x / shares;          // the plan keeps these products below 2^32
        end = units * (blockIdx.x + 1) / shares;
      }
    }
    fetch();
  }
  // the CTA whose share has this step: every share has one at least
  __device__ __forceinline__ uint32_t owner(uint32_t step) const {
    return ((step + 1) * shares - 1) / (tiles * p.steps);
  }
  // Neighbouring tiles share a tile of W with up to 8 slots, and those slots with the next tiles
  // of W, so that what runs at a time reads little from outside L2.
  __device__ __forceinline__ void fetch() {
    if (at >= end) return;
    const uint32_t t = p.split ? at / p.steps : at;
    ahead.tile = t;
    ahead.k0 = p.split ? at - t * p.steps : 0;
    ahead.k1 = p.split ? min(p.steps, ahead.k0 + (end - at)) : p.steps;
    const uint32_t band = t / (8 * across), rest = t - band * 8 * across;
    const uint32_t wide = n_slots - band * 8 < 8 ? n_slots - band * 8 : 8;
    ahead.row_tile = rest / wide;
    ahead.slot = band * 8 + rest - ahead.row_tile * wide;
    if (p.in_block) {
      ahead.expert = table[ahead.slot] >> 18;
      ahead.number = (table[ahead.slot] >> 9) & 511u;
      ahead.rows = table[ahead.slot] & 511u;
    } else if (p.experts) {
      ahead.expert = __ldcg(p.slot_expert + ahead.slot);
      ahead.rows = __ldcg(p.slot_rows + ahead.slot);
    } else {
      ahead.expert = 0;
      ahead.rows = min(p.tok, p.n_rows - ahead.slot * p.tok);
    }
  }
  __device__ __forceinline__ bool next(MxItem &item) {
    if (at >= end) return false;
    item = ahead;
    at += p.split ? item.k1 - item.k0 : p.pair ? gridDim.x / 2 : gridDim.x;
    fetch();
    return true;
  }
};

// Pair: W, the codes of a pair's half of a slot's step, and its scales, as rows of 256 bytes.
struct MxPairMaps {
  CUtensorMap w, x_codes, x_scales;
};

// The rows of a slot into shared memory, by all warps that store or help (this one is number `sub`), a
// block a thread: a warp takes up to 8 rows at a time (as many as a power of two of them that there
// are) and the blocks of them that fill it, and requests four such pieces before it works on them.
template <typename T>
__device__ __forceinline__ void mx_quantize_slot(const MxLinearArgs &p, const MxItem &it, const uint16_t *row_list,
                                                 uint32_t sub, uint32_t x_at, uint32_t x_codes) {
  constexpr uint32_t kWarps = 4 + kMxHelpers, kAhead = 4;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t shift = it.rows > 4 ? 3 : it.rows > 2 ? 2 : it.rows - 1;
  const uint32_t each = 32u >> shift;                         // blocks of a piece
  const uint32_t padded = (p.blocks + 1) & ~1u;               // the products take blocks in pairs
  const uint32_t across = (padded + each - 1) / each, total = ((it.rows - 1) >> shift) + 1;
  const uint32_t pieces = total * across;
  for (uint32_t w0 = sub; w0 < pieces; w0 += kWarps * kAhead) {
    uint32_t v[kAhead][16], to[kAhead], block[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const uint32_t w = w0 + k * kWarps, group = w / across;
      const uint32_t i = (group << shift) + (lane & ((1u << shift) - 1u));
      block[k] = (w - group * across) * each + (lane >> shift);
      const bool there = w < pieces && i < it.rows && block[k] < padded;
      to[k] = there ? i : kMxNone;
      const uint32_t row = there ? (p.experts ? row_list[i] : it.slot * p.tok + i) / p.per_input : 0;
      const T *src = (const T *)p.x + row * p.x_stride + (uint64_t)block[k] * kMxBlock;
      const int64_t left = there ? (int64_t)p.w.cols - (int64_t)block[k] * kMxBlock : 0;
      if (p.wide == 2) mx_load_block<2>(src, left, v[k]);
      else if (p.wide == 1) mx_load_block<1>(src, left, v[k]);
      else mx_load_block<0>(src, left, v[k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      if (to[k] == kMxNone) continue;
      uint32_t code[4], byte;
      mx_quantize_block<T>(v[k], code, byte);
      const uint32_t step = x_at + (block[k] >> 3) * p.x_step_bytes;
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(step + ((block[k] & 7u) * p.tok + to[k]) * 16),
                   "r"(code[0]), "r"(code[1]), "r"(code[2]), "r"(code[3])
                   : "memory");
      asm volatile("st.shared.u8 [%0], %1;" ::"r"(step + x_codes + mx_scale_offset(to[k], block[k] & 7u, p.chunks)),
                   "r"(byte)
                   : "memory");
    }
  }
  // visible to the tensor cores' reads
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// How a product runs: in CTAs by themselves behind the kernel that quantises x, in pairs of CTAs
// behind it, or in CTAs that quantise the rows of their slot themselves, in one launch.
enum MxMode { kMxAlone, kMxPair, kMxFused };
__host__ __device__ constexpr int mx_threads(MxMode mode) { return kMxLinThreads + (mode == kMxFused ? (int)kMxHelpers * 32 : 0); }

// Shared-memory map: a slot's steps (fused), stages (a step of a tile of W and, unless fused, of a
// slot), then
constexpr uint32_t kMxBarFull = 0, kMxBarEmpty = 8 * kMxMaxStages, kMxBarAccFull = 16 * kMxMaxStages,
                   kMxBarAccEmpty = kMxBarAccFull + 16, kMxBarDrain = kMxBarAccEmpty + 16,
                   kMxBarX = kMxBarDrain + 8, kMxTmemSlot = kMxBarX + 8, kMxAbortSlot = kMxTmemSlot + 4,
                   kMxLastSlot = kMxAbortSlot + 4, kMxSlotCount = kMxLastSlot + 4,
                   kMxTurn = 512,               // 16 rows x 32 features of y for each storing warp
                   kMxTable = kMxTurn + 4 * 1024, kMxIds = kMxTable + 4 * kMxBlockSlots,
                   kMxRowList = kMxIds + 2 * kMxBlockRows,      // fused: a slot's rows, for each warp
                   kMxMiscBytes = kMxRowList + (4 + kMxHelpers) * 512;
static_assert(kMxSlotCount + 4 <= kMxTurn && 4 * kMxBlockExperts <= 4 * 1024, "barriers");

template <typename T, MxMode MODE>
__global__ void __launch_bounds__(mx_threads(MODE), 1)
mx4_product_kernel(const MxLinearArgs p, const __grid_constant__ MxPairMaps maps) {
  constexpr bool PAIR = MODE == kMxPair, FUSED = MODE == kMxFused;
  extern __shared__ uint8_t mx_smem[];
  const uint32_t x_at = (smem_u32(mx_smem) + 127u) & ~127u, base = x_at + (FUSED ? p.x_resident : 0);
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
      mbar_init(misc_a + kMxBarAccEmpty + 8 * a, PAIR ? 8 : 4);      // storing warps
    }
    mbar_init(misc_a + kMxBarDrain, 1);
    mbar_init(misc_a + kMxBarX, 4 + kMxHelpers);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // The allocation may wait for a CTA of another kernel on this SM to free its columns; that CTA never
  // waits for this one, nor does the kernel that this one waits for below, which uses none.
  if (warp == 1) {
    mx_tmem_alloc<PAIR>(misc_a + kMxTmemSlot);
  }
  uint32_t *table = reinterpret_cast<uint32_t *>(misc + kMxTable);
  uint16_t *ids = reinterpret_cast<uint16_t *>(misc + kMxIds);
  if (p.in_block)
    mx_find_slots<mx_threads(MODE)>(p, table, reinterpret_cast<uint32_t *>(misc + kMxTurn), ids,
                  reinterpret_cast<uint32_t *>(misc + kMxSlotCount));
  mx_fence_before();
  __syncthreads();
  if (PAIR) mx_pair_sync();                    // both CTAs' barriers are there
  mx_fence_after();
  const uint32_t rank = PAIR ? mx_pair_rank() : 0;
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t *>(misc + kMxTmemSlot), 0);
  // W does not come from the kernel before, which is this call's own: the first stages' are on their
  // way while that kernel runs, unless the items depend on its tables.
  const bool known = !p.experts || p.in_block;
  auto slots_now = [&]() {
    return !p.experts ? p.slots
           : p.in_block ? *reinterpret_cast<uint32_t *>(misc + kMxSlotCount) : __ldcg(p.n_slots);
  };
  // the CTA's tile of W; where a pair has one tile left, the second CTA reads it too and stores nothing
  auto my_tile = [&](const MxItem &it) { return PAIR ? 2 * it.row_tile + rank : it.row_tile; };
  auto w_tile = [&](const MxItem &it) {
    return p.packed + ((uint64_t)it.expert * p.row_tiles + min(my_tile(it), p.row_tiles - 1)) * p.tile_bytes;
  };
  const uint32_t x_rows = PAIR ? p.tok / 2 : p.tok;                 // rows of a slot that this CTA holds
  const uint32_t x_codes = x_rows * 128, x_scales = p.chunks * 2 * kMxChunk, x_bytes = x_codes + x_scales;
  // fused: a warp's part of an item's rows, unless the item before had the same slot
  auto prepare_rows = [&](const MxItem &it, uint16_t *row_list, uint32_t sub, uint32_t &have) {
    if (have != it.slot) {
      have = it.slot;
      if (p.in_block) mx_list_rows(p, ids, it.expert, it.number, row_list);
      mx_quantize_slot<T>(p, it, row_list, sub, x_at, x_codes);
    }
    __syncwarp();
    if (lane == 0) mx_mbar_arrive(misc_a + kMxBarX);
  };
  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (mx_elect()) {
      // the bytes of a stage count at this CTA's barrier; a pair's at the first CTA's, which expects
      // the second one's too.  A pair copies whole steps (behind a tile's short last step lies the next
      // tile, or zeros).
      auto load_w = [&](const uint8_t *w, uint32_t k, uint32_t stage) {
        const uint32_t at = base + stage * p.stage_bytes, bar = misc_a + kMxBarFull + 8 * stage;
        if (PAIR) {
          if (rank == 0) mbar_expect_tx(bar, 2 * (kMxStepBytes + x_bytes));
          mx_pair_copy(at, &maps.w, (int32_t)((w - p.packed) / 256), mx_of_first(bar));
        } else {
          const uint32_t bytes = min(8u, p.blocks - 8 * k) * kMxBlockBytes + 2 * kMxChunk;
          mbar_expect_tx(bar, FUSED ? bytes : bytes + x_bytes);
          bulk_g2s(at, w, bytes, bar);
        }
      };
      auto load_x = [&](const uint8_t *x, uint32_t stage) {
        const uint32_t at = base + stage * p.stage_bytes + kMxStepBytes, bar = misc_a + kMxBarFull + 8 * stage;
        if (PAIR) {
          const int32_t row = (int32_t)((x - p.x_packed) / 256), half = (int32_t)(x_codes / 256);
          mx_pair_copy(at, &maps.x_codes, row + (int32_t)rank * half, mx_of_first(bar));
          mx_pair_copy(at + x_codes, &maps.x_scales, row + 2 * half, mx_of_first(bar));
        } else {
          bulk_g2s(at, x, x_bytes, bar);
        }
      };
      uint32_t early = 0;
      if (known) {
        MxItems items(p, table, slots_now());
        MxItem it;
        while (early < p.stages && items.next(it)) {
          const uint8_t *w = w_tile(it) + (uint64_t)it.k0 * kMxStepBytes;
          for (uint32_t k = it.k0; k < it.k1 && early < p.stages; ++k, ++early, w += kMxStepBytes)
            load_w(w, k, early);
        }
      }
      dependent_wait();
      uint32_t stage = 0, phase = 0;
      uint64_t done = 0;
      bool ok = true;
      MxItems items(p, table, slots_now());
      MxItem it;
      while (ok && items.next(it)) {
        const uint8_t *x = p.x_packed + ((uint64_t)it.slot * p.steps + it.k0) * p.x_step_bytes;
        const uint8_t *w = w_tile(it) + (uint64_t)it.k0 * kMxStepBytes;
        for (uint32_t k = it.k0; k < it.k1; ++k, ++done, w += kMxStepBytes, x += p.x_step_bytes) {
          if (done >= p.stages && !mx_wait(misc_a + kMxBarEmpty + 8 * stage, phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          if (done >= early) load_w(w, k, stage);
          if (!FUSED) load_x(x, stage);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        if (p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        // copies still in flight land before the CTA's shared memory is given away: after an abort
        // nobody else waits for them (a pair's first CTA does so for both)
        for (uint64_t i = done > p.stages ? done - p.stages : 0; i < done && rank == 0; ++i) {
          const uint32_t s = (uint32_t)(i % p.stages), ph = (uint32_t)(i / p.stages) & 1u;
          for (uint32_t n = 0; n < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarFull + 8 * s, ph); ++n) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- tensor cores
    dependent_wait();
    if (rank == 0 && mx_elect()) {
      uint32_t stage = 0, phase = 0, item = 0;
      bool ok = true;
      const uint32_t k64 = (p.blocks + 1) / 2;
      // in units of descriptors: two blocks, a stage, the chunks of a step's half
      const uint64_t a_step = 2 * kMxTileRows, b_step = 2 * x_rows, stage_step = p.stage_bytes >> 4;
      const uint64_t a_chunk = kMxChunk >> 4, b_chunk = p.chunks * a_chunk;
      const uint64_t a0 = mx_desc_codes(base, kMxTileRows), sfa0 = mx_desc_scales(base);
      const uint64_t b0 = mx_desc_codes(FUSED ? x_at : base + kMxStepBytes, x_rows);
      const uint64_t sfb0 = mx_desc_scales((FUSED ? x_at : base + kMxStepBytes) + x_codes);
      const bool two = p.chunks == 2;
      // whether a stage has arrived is asked a step ahead: the answer takes a hundred cycles, which the
      // issuing of the step before covers
      bool there = mx_test(misc_a + kMxBarFull, 0);
      MxItems items(p, table, slots_now());
      MxItem it;
      while (ok && items.next(it)) {
        // 4-bit operands (type 1), e8m0 scales, N, M = 128 or 256
        const uint32_t idesc0 = (1u << 7) | (1u << 10) | ((mx_columns(it.rows) >> 3) << 17) | (1u << 23) |
                                ((PAIR ? 2u : 1u) << 27);
        const uint32_t idesc1 = idesc0 | (2u << 4) | (2u << 29);       // the scales at byte 2
        const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u);
        if (item >= 2 && !mx_wait_pair(misc_a + kMxBarAccEmpty + 8 * acc, ((item >> 1) & 1u) ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        if (FUSED && !mx_wait(misc_a + kMxBarX, item & 1u, abort_flag)) {
          ok = false;
          break;
        }
        for (uint32_t k = it.k0; k < it.k1; ++k) {
          if (!there && !mx_wait(misc_a + kMxBarFull + 8 * stage, phase, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t done = misc_a + kMxBarEmpty + 8 * stage;
          const uint64_t at = stage * stage_step, x_step = FUSED ? k * (uint64_t)(p.x_step_bytes >> 4) : at;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
          there = mx_test(misc_a + kMxBarFull + 8 * stage, phase);
          mx_fence_after();
          const uint64_t ad = a0 + at, bd = b0 + x_step, sfb = sfb0 + x_step;
          const uint64_t sfa = sfa0 + at + min(8u, p.blocks - 8 * k) * (kMxBlockBytes >> 4);
          const uint32_t last = k64 - 4 * k, more = k > it.k0;
          // Copies and products of one thread run in order: the scales of the step before have been
          // used when these replace them.  64 columns are two blocks; the scales of four share a
          // tensor-memory column.
          mx_copy_scales<PAIR>(tmem + kMxSfA, sfa);
          mx_copy_scales<PAIR>(tmem + kMxSfB, sfb);
          if (two) mx_copy_scales<PAIR>(tmem + kMxSfB + 4, sfb + a_chunk);
          mx_mma<PAIR>(d, ad, bd, idesc0, tmem + kMxSfA, tmem + kMxSfB, more);
          if (last > 1) mx_mma<PAIR>(d, ad + a_step, bd + b_step, idesc1, tmem + kMxSfA, tmem + kMxSfB, 1);
          if (last > 2) {
            mx_copy_scales<PAIR>(tmem + kMxSfA + 4, sfa + a_chunk);
            mx_copy_scales<PAIR>(tmem + kMxSfB + 8, sfb + b_chunk);
            if (two) mx_copy_scales<PAIR>(tmem + kMxSfB + 12, sfb + b_chunk + a_chunk);
            mx_mma<PAIR>(d, ad + 2 * a_step, bd + 2 * b_step, idesc0, tmem + kMxSfA + 4, tmem + kMxSfB + 8, 1);
            if (last > 3)
              mx_mma<PAIR>(d, ad + 3 * a_step, bd + 3 * b_step, idesc1, tmem + kMxSfA + 4, tmem + kMxSfB + 8, 1);
          }
          mx_commit<PAIR>(done);
        }
        if (ok) mx_commit<PAIR>(misc_a + kMxBarAccFull + 8 * acc);
        ++item;
      }
      if (!ok) {
        if (p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        // what has been issued still uses shared and tensor memory
        mx_commit<PAIR>(misc_a + kMxBarDrain);
        for (uint32_t n = 0; n < kMaxWaitIters && !mbar_try_wait(misc_a + kMxBarDrain, 0); ++n) {
        }
      }
    }
  } else if (FUSED && warp >= 6) {
    // ---------------------------------------------------------------- rows of x, with the storing warps
    MxItems items(p, table, slots_now());
    uint16_t *row_list = reinterpret_cast<uint16_t *>(misc + kMxRowList) + (warp - 2) * 256;
    uint32_t item = 0, have = kMxNone;
    MxItem it;
    while (items.next(it)) {
      // the slot before has been used when its products are done
      const uint32_t b = item - 1;
      if (item && !__all_sync(0xFFFFFFFFu, mx_wait(misc_a + kMxBarAccFull + 8 * (b & 1u), (b >> 1) & 1u, abort_flag))) {
        if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      prepare_rows(it, row_list, warp - 2, have);
      ++item;
    }
  } else {
    // ---------------------------------------------------------------- results
    dependent_wait();
    MxItems items(p, table, slots_now());
    const uint32_t sub = warp & 3u;                   // tensor-memory lanes 32 sub .. + 31
    T *const turns = reinterpret_cast<T *>(misc + kMxTurn), *const turn = turns + sub * 512;
    uint16_t *row_list = reinterpret_cast<uint16_t *>(misc + kMxRowList) + sub * 256;
    if (FUSED && p.in_block) {
      // rows of y without a matrix
      for (uint32_t r = blockIdx.x; r < p.n_rows; r += gridDim.x)
        if (ids[r] == kMxNoMatrix) {
          for (uint64_t i = 32 * sub + lane; i < p.w.rows; i += 128) ((T *)p.y)[r * p.w.rows + i] = from_float<T>(0.f);
          if (threadIdx.x == 64 && p.status && __ldg(p.experts + r) != -1) atomicOr(p.status, NZ_STATUS_BAD_INDEX);
        }
    }
    uint32_t item = 0, have = kMxNone;
    MxItem it;
    while (items.next(it)) {
      if (FUSED) {
        // the products of the item before are done, or its sums would not have been read
        prepare_rows(it, row_list, sub, have);
      }
      const uint32_t rows = it.rows, place0 = it.slot * p.tok;
      const uint32_t feature = my_tile(it) * kMxTileRows + 32 * sub + lane;
      const bool real = feature < p.w.rows;
      const float bias = p.bias && real ? to_float<T>(((const T *)p.bias)[it.expert * p.w.rows + feature]) : 0.f;
      // 16 rows of y of this warp's 32 features, from a value for every row in each lane
      T *y = (T *)p.y + my_tile(it) * kMxTileRows + 32 * sub;
      auto store16 = [&](const float (&f)[16], uint32_t row_here, uint32_t count) {
        if (p.wide_y) {
          // turned in shared memory: four lanes take a row's 64 bytes
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) turn[i * 32 + lane] = from_float<T>(f[i] + bias);
          __syncwarp();
          const bool in = my_tile(it) * kMxTileRows + 32 * sub + 8 * (lane & 3u) < p.w.rows;
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t i = 8 * h + (lane >> 2);
            const uint64_t r = __shfl_sync(0xFFFFFFFFu, row_here, i);
            const uint4 piece = *reinterpret_cast<const uint4 *>(turn + i * 32 + 8 * (lane & 3u));
            if (i < count && in) *reinterpret_cast<uint4 *>(y + r * p.w.rows + 8 * (lane & 3u)) = piece;
          }
          __syncwarp();
        } else {
          // Rows begin anywhere.  The four warps put their 32 features together, then each stores four
          // rows of all 128: a sector that is written in parts costs a read as well, and so a row has two
          // of them instead of eight.
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) turns[i * 128 + 32 * sub + lane] = from_float<T>(f[i] + bias);
          mx_store_barrier();
          const uint32_t first = my_tile(it) * kMxTileRows;
          const uint32_t n = first < p.w.rows ? min(kMxTileRows, (uint32_t)p.w.rows - first) : 0;
          uint16_t *dst[4];
#pragma unroll
          for (uint32_t h = 0; h < 4; ++h) {
            const uint32_t i = 4 * sub + h;
            const uint64_t r = __shfl_sync(0xFFFFFFFFu, row_here, i);
            dst[h] = i < count ? reinterpret_cast<uint16_t *>(y - 32 * sub + r * p.w.rows) : nullptr;
          }
          mx_store_runs<4>(dst, reinterpret_cast<uint16_t *>(turns + 4 * sub * 128), 128, n);
          mx_store_barrier();
        }
      };
      // lane i of 16 knows the row of y of column c0 + i; fetched 16 columns ahead
      auto row_at = [&](uint32_t c) -> uint32_t {
        if (!p.experts) return place0 + c + (lane & 15u);
        if (c + (lane & 15u) >= rows) return 0u;
        return FUSED ? row_list[c + (lane & 15u)] : p.row_of[place0 + c + (lane & 15u)];
      };
      uint32_t row_next = row_at(0);
      const uint32_t acc = item & 1u, d = tmem + (acc ? kMxAcc1 : 0u) + ((32u * sub) << 16);
      if (!mx_store_all(mx_wait(misc_a + kMxBarAccFull + 8 * acc, (item >> 1) & 1u, abort_flag))) {
        if (lane == 0 && p.status) atomicOr(p.status, NZ_STATUS_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      mx_fence_after();
      const bool whole = it.k0 == 0 && it.k1 == p.steps;
      // pieces of a CTA: its first tile's where it does not begin it, and its last one's
      auto piece_of = [&](uint32_t cta, bool begins) {
        return p.partial + ((uint64_t)cta * 2 + begins) * p.tok * kMxTileRows + 32 * sub + lane;
      };
      float *piece = whole ? nullptr : piece_of(blockIdx.x, it.k0 == 0);
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
          if (lane == 0) {
            if (PAIR) mx_arrive_first(misc_a + kMxBarAccEmpty + 8 * acc);
            else mx_mbar_arrive(misc_a + kMxBarAccEmpty + 8 * acc);
          }
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
        const uint32_t first = items.owner(it.tile * p.steps);
        const uint32_t pieces = items.owner(it.tile * p.steps + p.steps - 1) - first + 1;
        mx_store_barrier();
        if (threadIdx.x == 64) {
          __threadfence();                            // cumulative: the warps' stores, then the arrival
          const uint32_t seen = atomicAdd(p.counters + it.tile, 1u);
          __threadfence();
          *last_flag = seen == pieces - 1;
        }
        mx_store_barrier();
        if (*last_flag) {
          for (uint32_t c0 = 0; c0 < rows; c0 += 16) {
            float sum[16] = {};
            const uint32_t row_here = row_at(c0);
            for (uint32_t q0 = 0; q0 < pieces; q0 += 4) {
              float add[4][16];                       // loads in flight
#pragma unroll
              for (uint32_t q = 0; q < 4; ++q)
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i)
                  add[q][i] = q0 + q < pieces && c0 + i < rows
                                  ? __ldcg(piece_of(first + q0 + q, q0 + q == 0) + (uint64_t)(c0 + i) * kMxTileRows)
                                  : 0.f;
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

  // ---- common exit: everybody is done with tensor memory (and with the other CTA's barriers), then
  // it is freed
  __syncwarp();
  mx_fence_before();
  __syncthreads();
  if (PAIR) mx_pair_sync();
  if (warp == 1) {
    mx_fence_after();
    mx_tmem_free<PAIR>(tmem);
  }
}

// --------------------------------------------------------------------- host
struct MxPlan {
  uint32_t tok, chunks, row_tiles, steps, split, in_block, pair, fused, pieces, x_resident, grid, stages, stage_bytes, x_step_bytes;
  uint64_t slots;
  uint64_t counters, slot_expert, slot_rows, row_of, place_of, x_packed, partial, bytes;
};

// The rows of a slot and the way of running, by an estimate of the time (in cycles) that a call takes.
// `kind`: whole tiles, shared tiles, tiles of a pair of CTAs, of which `sms` then counts the pairs, or whole
// tiles whose CTAs quantise their rows themselves (for each slot they take, before its products) instead of a
// kernel of its own.
// A step takes the longest of: its products (2 cycles a row), their issuing (420), its bytes into an SM (80
// a cycle) and into all of them (7400 from L2; 3400 of W from memory).  A launch before the product costs
// 5000 (its device time is hidden in part, its host time is not), a pair's start 2000 more, an item beside
// its steps 300 and 8 a row.  The pieces of a shared tile are joined four at a time, 16 columns in 1800.
// Measured in us on the device, what it chooses first (rows x inner x outer size, every way forced in turn):
//   16 x 4096 x 11008 alone 9.7, pairs 10.7, fused 14.0, shared 14.2; 64 x 4096 x 11008 alone 10.2, pairs 11.1
//   4 x 4096 x 11008 fused 10.7, alone 9.6 and 4 more of host time; 4 x 8192 x 512 shared 9.5, alone 11.5
//   4 x 16384 x 2048 shared 12.2, alone 18.5; 16 x 16384 x 2048 shared 12.7, alone 18.5
//   2048 x 4096 x 11008 pairs 45.4, alone 48.4; 2048 x 8192 x 28672 pairs 175, alone 223
// Where it is off: 256 x 16384 x 2048 shared 23.8, alone 21.3; 256 x 2048 x 16384 pairs 14.2, alone 12.3;
// 256 x 4096 x 11008 pairs 16.4, alone 15.8.
enum MxKind { kMxWhole, kMxShared, kMxPaired, kMxOneLaunch };
static double mx_cost(uint64_t tok, double slots, const MxShape &w, double n_rows, double hit, uint32_t sms,
                      MxKind kind, uint32_t &pieces) {
  const double pair = kind == kMxPaired ? 2 : 1;
  const double tiles = slots * ceil((double)w.row_tiles() / pair), steps = (double)w.steps();
  const double bytes = kMxStepBytes + tok * 128.0 / pair + (tok > 128 ? 2 : 1) * 2.0 * kMxChunk;
  // with so many tiles at work; slots of a matrix share what comes from memory
  auto step = [&](double active) {
    double longest = fmax(fmax(2.0 * tok, 420), bytes / 80);
    longest = fmax(longest, bytes * pair * active / 7400);
    return fmax(longest, pair * kMxStepBytes * (hit / slots) * active / 3400);
  };
  const double item = 300 + 8.0 * tok, join = ceil(tok / 16.0) * 1800;
  pieces = 1;
  if (kind == kMxShared) {
    if (2 * tiles > sms)           // equal shares: a CTA joins pieces at both of its ends
      return 5000 + ceil(tiles * steps / sms) * step(sms) + 2 * (3000 + join);
    double best = 0;
    for (uint32_t p = 2; p <= 16 && p <= steps && p * tiles <= sms; ++p) {
      const double cost = 5000 + ceil(steps / p) * step(p * tiles) + 3000 + ceil(p / 4.0) * join;
      if (pieces == 1 || cost < best) {
        best = cost;
        pieces = p;
      }
    }
    return pieces == 1 ? 1e30 : best;
  }
  const double waves = floor(tiles / sms), rest = tiles - waves * sms;
  const double product = waves * (steps * step(sms) + 300) + (rest > 0 ? steps * step(rest) + 300 : 0) + item;
  if (kind == kMxOneLaunch) {
    const double rows = tok < n_rows / slots ? tok : n_rows / slots;
    const double at_once = rows > 4 ? 8 : rows > 2 ? 4 : rows > 1 ? 2 : 1;
    const double parts = ceil(rows / at_once) * ceil((double)w.blocks() * at_once / 32);
    return ceil(tiles / sms) * (800 + ceil(parts / (4 + kMxHelpers)) * 1200) + product;
  }
  return 5000 + (kind == kMxPaired ? 2000 : 0) + product;
}

// Pairs of CTAs that the device runs at a time.
static uint32_t mx_pairs();

static bool mx_make_plan(const MxShape &w, uint64_t n_rows, bool grouped, MxPlan &g) {
  const uint32_t sms = (uint32_t)sm_count(), n_pairs = mx_pairs();
  g.row_tiles = (uint32_t)w.row_tiles();
  g.steps = (uint32_t)w.steps();
  g.in_block = grouped && n_rows <= kMxBlockRows && w.matrices <= kMxBlockExperts;
  const uint64_t groups = grouped ? (w.matrices < n_rows ? w.matrices : n_rows) : 1;
  // matrices that are likely to be named, and half a slot of each that stays empty
  const double hit = grouped ? (double)w.matrices * (1 - pow(1 - 1.0 / (double)w.matrices, (double)n_rows)) : 1;
  uint64_t tok = 16;
  double best = -1;
  g.split = g.pair = g.fused = 0;
  for (uint64_t t = 16; t <= kMxMaxTok; t += 16) {
    double slots = grouped ? (double)n_rows / t + hit / 2 : ceil((double)n_rows / t);
    if (slots < hit) slots = hit;
    for (MxKind kind : {kMxWhole, kMxShared, kMxPaired, kMxOneLaunch}) {
      // steps times CTAs in 32 bits, and no more than a few tiles a CTA, or nothing is gained
      if (kind == kMxShared && (g.steps == 1 || slots * (double)w.row_tiles() * g.steps > 4e6)) continue;
      // the places of a pair's inputs depend on the slots' rows, which tables tell
      if (kind == kMxPaired && (g.in_block || n_pairs == 0)) continue;
      // a slot's rows beside four stages of W
      if (kind == kMxOneLaunch && ((grouped && !g.in_block) ||
                                   g.steps * (t * 128 + (t > 128 ? 2 : 1) * 2ull * kMxChunk) + 4 * kMxStepBytes >
                                       kMaxDynamicSmem - 128 - kMxMiscBytes))
        continue;
      uint32_t pieces;
      const double cost = mx_cost(t, slots, w, (double)n_rows, hit, kind == kMxPaired ? n_pairs : sms, kind, pieces);
      if (best < 0 || cost < best) {
        best = cost;
        tok = t;
        g.split = kind == kMxShared;
        g.pair = kind == kMxPaired;
        g.fused = kind == kMxOneLaunch;
        g.pieces = pieces;
      }
    }
    if (t >= n_rows) break;
  }
  g.tok = (uint32_t)tok;
  g.chunks = g.tok > 128 ? 2 : 1;
  // every matrix's last slot may be short
  g.slots = grouped ? (n_rows - groups) / tok + groups : (n_rows + tok - 1) / tok;
  const uint64_t tiles = g.slots * g.row_tiles;
  if (g.slots * tok >= (1ull << 31) || tiles >= (1ull << 31)) return false;
  if (g.split && tiles * g.steps >= (1ull << 32) / (sms + 1)) g.split = 0;
  const uint64_t units = g.split ? tiles * g.steps : tiles;
  g.grid = (uint32_t)(units < sms ? units : sms);
  if (g.pair) {
    const uint64_t pairs = g.slots * ((g.row_tiles + 1) / 2);
    g.grid = 2 * (uint32_t)(pairs < n_pairs ? pairs : n_pairs);
  }
  g.x_step_bytes = g.tok * 128 + g.chunks * 2 * kMxChunk;
  g.x_resident = g.fused ? g.steps * g.x_step_bytes : 0;
  g.stage_bytes = kMxStepBytes + (g.fused  ? 0
                                  : g.pair ? g.tok * 64 + g.chunks * 2 * kMxChunk
                                           : g.x_step_bytes);
  g.stages = (kMaxDynamicSmem - 128 - kMxMiscBytes - g.x_resident) / g.stage_bytes;
  if (g.stages > kMxMaxStages) g.stages = kMxMaxStages;
  g.bytes = 0;
  if (g.fused) return true;                    // no workspace
  uint64_t at = 256;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~255ull;
    return here;
  };
  const bool tables = grouped && !g.in_block;
  g.counters = take(g.split ? tiles * 4 : 0);
  g.slot_expert = take(tables ? g.slots * 4 : 0);
  g.slot_rows = take(tables ? g.slots * 4 : 0);
  g.row_of = take(grouped ? g.slots * tok * 4 : 0);
  g.place_of = take(tables ? n_rows * 8 : 0);
  g.x_packed = take(g.slots * g.steps * g.x_step_bytes);
  g.partial = take(g.split ? (uint64_t)g.grid * 2 * tok * kMxTileRows * 4 : 0);
  g.bytes = at;
  return true;
}

// Plans of recent calls: a program makes the same few over and over.
static bool mx_plan(const MxShape &w, uint64_t n_rows, bool grouped, MxPlan &g) {
  struct Kept {
    MxShape w = {0, 0, 0};
    uint64_t n_rows = 0;
    int dev = -1;
    bool grouped = false, fits = false;
    MxPlan g;
  };
  static thread_local Kept kept[64];
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return mx_make_plan(w, n_rows, grouped, g);
  }
  Kept &k = kept[(w.rows * 7 + w.cols * 13 + n_rows * 31 + w.matrices * 3 + grouped) % 64];
  if (k.dev != dev || k.w.matrices != w.matrices || k.w.rows != w.rows || k.w.cols != w.cols ||
      k.n_rows != n_rows || k.grouped != grouped) {
    k.fits = mx_make_plan(w, n_rows, grouped, k.g);
    k.w = w;
    k.n_rows = n_rows;
    k.grouped = grouped;
    k.dev = dev;
  }
  g = k.g;
  return k.fits;
}

// The kernels' shared memory above 48 KB has to be asked for, and the pairs counted, once per device.
struct MxDevice {
  std::mutex mu;
  bool ready = false;
  uint32_t pairs = 0;
};
static cudaLaunchConfig_t mx_config(unsigned grid, size_t smem, bool pair, cudaStream_t st,
                                    cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kMxLinThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pair ? 2 : 1;
  return cfg;
}
static cudaError_t mx_device(uint32_t *pairs) {
  static MxDevice devices[kMaxDeviceOrdinals];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= kMaxDeviceOrdinals) return cudaErrorInvalidDevice;
  MxDevice &d = devices[dev];
  std::lock_guard<std::mutex> lock(d.mu);
  if (!d.ready) {
    const int most = (int)kMaxDynamicSmem;
    const auto larger = cudaFuncAttributeMaxDynamicSharedMemorySize;
    if ((err = cudaFuncSetAttribute(mx4_product_kernel<__nv_bfloat16, kMxFused>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_product_kernel<__half, kMxFused>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_product_kernel<__nv_bfloat16, kMxAlone>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_product_kernel<__half, kMxAlone>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_product_kernel<__nv_bfloat16, kMxPair>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_product_kernel<__half, kMxPair>, larger, most)) != cudaSuccess ||
        (err = cudaFuncSetAttribute(mx4_route_kernel, larger, (int)(kMxMaxExperts * 8))) != cudaSuccess)
      return err;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = mx_config(2 * 1024, kMaxDynamicSmem, true, 0, attr);
    int clusters = 0;
    if ((err = cudaOccupancyMaxActiveClusters(&clusters, mx4_product_kernel<__nv_bfloat16, kMxPair>, &cfg)) !=
        cudaSuccess)
      return err;
    d.pairs = (uint32_t)clusters;
    d.ready = true;
  }
  *pairs = d.pairs;
  return cudaSuccess;
}
static uint32_t mx_pairs() {
  uint32_t pairs = 0;
  if (mx_device(&pairs) != cudaSuccess) {
    cudaGetLastError();
    return 0;                                  // without a device the size helpers still answer
  }
  return pairs;
}

typedef CUresult (*MxEncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                    const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                    CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                    CUtensorMapFloatOOBfill);
static bool mx_map(CUtensorMap *map, const void *bytes, uint64_t rows, uint32_t box) {
  static std::once_flag once;
  static MxEncodeTiledFn encode = nullptr;
  std::call_once(once, [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      encode = (MxEncodeTiledFn)fn;
  });
  const cuuint64_t dim[2] = {256, rows}, stride[1] = {256};
  const cuuint32_t size[2] = {256, box}, step[2] = {1, 1};
  return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(bytes), dim, stride, size, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
static int mx_launch(const MxLinearArgs &p, const MxPlan &g, cudaStream_t st) {
  MxPairMaps maps;
  memset(&maps, 0, sizeof(maps));
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = mx_config(
      g.grid, 128 + g.x_resident + (size_t)p.stages * p.stage_bytes + kMxMiscBytes, p.pair != 0, st, attr);
  if (g.fused) {
    cfg.numAttrs = 0;
    cfg.blockDim = dim3(mx_threads(kMxFused));
    NZ_CUDA_TRY(cudaLaunchKernelEx(&cfg, mx4_product_kernel<T, kMxFused>, p, maps));
    return NZ_OK;
  }
  if (p.pair) {
    const uint64_t x_rows = (uint64_t)p.slots * p.steps * p.x_step_bytes / 256;
    if (!mx_map(&maps.w, p.packed, p.w.bytes() / 256, kMxStepBytes / 256) ||
        !mx_map(&maps.x_codes, p.x_packed, x_rows, p.tok / 4) ||
        !mx_map(&maps.x_scales, p.x_packed, x_rows, p.chunks * 2 * kMxChunk / 256)) {
      set_error("nz_mx4_linear: cuTensorMapEncodeTiled failed");
      return NZ_E_CUDA;
    }
  }
  uint32_t pairs = 0;
  NZ_CUDA_TRY(mx_device(&pairs));
  const uint64_t rows = p.in_block ? p.n_rows : p.n_rows / p.per_input;
  const uint64_t warps = (rows + 7) / 8 * 2 * p.steps, blocks = (warps + 7) / 8;
  const unsigned most = (unsigned)sm_count() * 8;
  const unsigned grid = blocks < most ? (unsigned)blocks : most;
  auto rows_kernel = p.wide == 2   ? mx4_quantize_rows_kernel<T, 2>
                     : p.wide == 1 ? mx4_quantize_rows_kernel<T, 1>
                                 : mx4_quantize_rows_kernel<T, 0>;
  if (p.experts && !p.in_block) {
    mx4_route_kernel<<<1, kMxRouteThreads, p.w.matrices * 8, st>>>(p);
    NZ_LAUNCH_CHECK("mx4_route_kernel");
  }
  rows_kernel<<<grid, 256, p.in_block ? sizeof(MxPlaces) : 0, st>>>(p);
  NZ_LAUNCH_CHECK("mx4_quantize_rows_kernel");
  NZ_CUDA_TRY(p.pair ? cudaLaunchKernelEx(&cfg, mx4_product_kernel<T, kMxPair>, p, maps)
                     : cudaLaunchKernelEx(&cfg, mx4_product_kernel<T, kMxAlone>, p, maps));
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

extern "C" int nz_mx4_linear_way(uint64_t matrices, uint64_t rows, uint64_t cols, uint64_t n_rows, int grouped) {
  using namespace nz;
  const MxShape w{matrices, rows, cols};
  MxPlan g;
  if (!mx_shape("nz_mx4_linear_way", matrices, rows, cols) || matrices == 0 || rows == 0 || cols == 0 ||
      n_rows == 0 || n_rows >= (1ull << 31) || matrices > (grouped ? kMxMaxExperts : 1))
    return -1;
  if (mx_few_rows(w, n_rows, grouped != 0)) return NZ_MX4_FEW_ROWS;
  if (!mx_plan(w, n_rows, grouped != 0, g)) return -1;
  return g.fused ? NZ_MX4_ONE_LAUNCH : g.pair ? NZ_MX4_PAIRS : g.split ? NZ_MX4_SHARED_TILES : NZ_MX4_WHOLE_TILES;
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
  if (workspace_bytes < g.bytes || (g.bytes && !workspace)) {
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
  p.split = g.split ? (g.pieces > 1 ? g.pieces : 4) : 0;
  p.in_block = g.in_block;
  p.pair = g.pair;
  p.x_resident = g.x_resident;
  p.wide = mx_wide_rows(x, x_stride, cols);
  p.stages = g.stages;
  p.stage_bytes = g.stage_bytes;
  p.wide_y = rows % 8 == 0 && ((uintptr_t)y & 15) == 0;
  p.n_slots = (uint32_t *)ws;
  p.counters = (uint32_t *)(ws + g.counters);
  p.slot_expert = (uint32_t *)(ws + g.slot_expert);
  p.slot_rows = (uint32_t *)(ws + g.slot_rows);
  p.row_of = (uint32_t *)(ws + g.row_of);
  p.place_of = (uint2 *)(ws + g.place_of);
  p.x_packed = ws + g.x_packed;
  p.partial = (float *)(ws + g.partial);
  return dtype == NZ_DTYPE_BF16 ? mx_launch<__nv_bfloat16>(p, g, (cudaStream_t)stream)
                                : mx_launch<__half>(p, g, (cudaStream_t)stream);
}

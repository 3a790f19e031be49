// Tile product of the dense layers around a forest (ht_gated_linear.cu, ht_class_loss.cu) on the tensor cores:
//
//     out[m, n] = sum_k A(m, k) B(n, k)        16-bit operands (bf16 or fp16), fp32 accumulation in tensor memory
//
// handed to an epilogue 32 columns at a time, so that what a layer does with its products (softmax sums, the loss's gradient,
// activation and gate, a scaled store) happens before they leave the registers.  Either operand is stored with k
// contiguous ([rows][k]) or with m / n contiguous ([k][rows], "MN"), which is what the three products of a layer need of
// one stored matrix: y = x w^T, dx = dy w, dw = dy^T x, without a transposed copy.
//
// fp32 operands come as three bf16 planes (x = x0 + x1 + x2, each the rounding of what is left: 24 bits): the products x0 y0 in one
// accumulator, and x0 y1, x1 y0, x1 y1, x0 y2, x2 y0 in a second; what is left out is below 2^-24 of a term.  The tensor core truncates
// when it adds to an accumulator, always towards zero (measured: 32 instructions in a row lose about 9e-7 of the sum, which is more than an fp32
// sum loses to rounding).  So the large products leave for registers every 16 instructions (256 values of k) and are added there in
// fp32; the small ones are 2^-8 of those and stay to the end.  (Every 8 instructions would lose half of that, 2e-7 instead of 4e-7, but leave the
// epilogue of a tile no time beside the next one's products.)
// The gradients of an fp16 layer and what they are multiplied by come as two planes: x0 y0, and x0 y1, x1 y0.
//
// A persistent kernel of 320 threads a CTA, one CTA per SM, alone (CTAS = 1, tiles of 128 rows) or in clusters of two that share a
// tile of 256 rows (CTAS = 2): tcgen05.mma.cta_group::2 reads each CTA's 128 rows of A and half of B's rows from that CTA's shared
// memory, which halves what a product moves of B into and out of shared memory, the resource that bounds the single form
// (16384 x 16384 x 1024, bf16: 1110 TFLOP/s alone, 1280 in pairs; 8192 cubed 1200 and 1520).
//   warp 0      one lane issues the TMA loads (cp.async.bulk.tensor, 128-byte swizzle, no multicast) into a ring of stages of 64 values of
//               k; in a pair both CTAs load their part and their bytes arrive at the first CTA's barrier;
//   warp 1      allocates tensor memory, and one lane (of the first CTA) issues tcgen05.mma.kind::f16 (M 128 or 256, N up to 256,
//               K 16) and commits each stage back to the loads and each finished accumulator to the epilogue, of both CTAs;
//   warps 2-9   the epilogue, under the main loop of the next tile: two warps per quarter of the CTA's 128 lanes, each with one half
//               of the columns.
// Tensor memory: two accumulators of 256 columns, used in turn; with two or three planes one for the large and one for the small products,
// and the small ones of a block are issued first, so that the large ones' accumulator is read out meanwhile.
// Tiles are walked in groups of 16 row blocks, rows fastest, so that what the SMs read at one time is shared in L2.
// Every wait is bounded: when one runs out the kernel flags HT_FLAG_PIPELINE_TIMEOUT, every role stops at its own next wait, the
// loads wait for their copies in flight, the tensor memory is freed and the kernel returns.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "ht_common.cuh"
#include "ht_tile_common.cuh"
#include "ht_tma.cuh"

namespace ht {
namespace dense {

using namespace tile;

constexpr int kTileM = 128, kTileK = 64;
constexpr int kTileThreads = 320;
constexpr int kEpilogueWarps = 8;
// Blocks of 64 values of k between two visits of the registers: with three planes, for fp32 results; with two, for fp16 ones, 64 instructions lose
// 2e-6 of a sum.
template <int PLANES>
constexpr int kChunkBlocks = PLANES == 3 ? 4 : 16;
constexpr int kMostStages = 12;
constexpr uint32_t kStageBudget = 192 * 1024;
constexpr uint32_t kBoxBytes = 4096;  // of an epilogue warp: 32 rows of 32 columns on their way to or from memory
constexpr size_t kTileSmem = 1024 + kStageBudget + kEpilogueWarps * kBoxBytes + 512;

#define HT_TRY(expr)                    \
  do {                                  \
    const int rc_ = (expr);             \
    if (rc_ != HT_OK) return rc_;       \
  } while (0)

// The kernels of these layers follow one another closely: each lets the next one's blocks start as SMs become free, and waits for the one before
// to have ended, with its results in memory, before it touches memory that others touch (2 to 4 us less a kernel than one after the
// other).
__device__ __forceinline__ void after_previous_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// What these kernels read may have been written while they were resident already, by the kernel before: all of it, a call's inputs too, by plain
// loads.  (__ldg, and pointers that are const and __restrict__, are for what nothing writes as long as the kernel lives.)
template <typename V>
__device__ __forceinline__ V load_plain(const V *p) {
  return *p;
}

template <typename... Parameters, typename... Arguments>
cudaError_t launch_with(const cudaLaunchConfig_t &config, void (*kernel)(Parameters...), const Arguments &...arguments) {
  return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

// Launches a kernel that begins with after_previous_kernel(), in clusters of `ctas`.  `most`: of shared memory in any of the kernel's launches,
// asked for once on a device.
template <auto KERNEL, typename... Arguments>
int launch_next(dim3 grid, int threads, size_t shared, size_t most, cudaStream_t stream, int ctas, const Arguments &...arguments) {
  if (shared > 48 * 1024) {
    static std::atomic<uint64_t> granted{0};  // devices, by number
    int device = 0;
    HT_CUDA_TRY(cudaGetDevice(&device));
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if ((granted.load(std::memory_order_relaxed) & bit) == 0) {
      HT_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
      granted.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = (unsigned)ctas;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = ctas > 1 ? 2 : 1;
  HT_CUDA_TRY(launch_with(config, KERNEL, arguments...));
  HT_CHECK_LAUNCH();
  return HT_OK;
}

// A 16-bit matrix in device memory, row-major, `pitch` elements from row to row (a multiple of 8, base on 16 bytes); with
// several planes, `plane` elements apart.
struct Matrix {
  const void *data = nullptr;
  int64_t rows = 0, cols = 0, pitch = 0;
  int planes = 1;
  int64_t plane = 0;
};

struct alignas(64) TileArgs {
  CUtensorMap a[2], b[2];
  uint32_t *status_word;
  uint32_t instruction;
  int m_blocks, n_blocks, tiles;
  int bn;                  // columns of a tile: both halves of a pair together
  int k, k_blocks;         // of one segment
  int segments;            // 2: the sum over k goes on in a[1], b[1]
  int part_blocks;         // blocks of 64 values of k, of both segments together, in a part; tiles are counted part by part
  int b_n0, b_k0;          // where B's rows / values of k begin
  int stages;
  uint32_t a_bytes, stage_bytes;  // of one CTA
};

// How a product is cut: CTAs that share a tile of 128 rows each, its columns, parts of k.
struct TileShape {
  int ctas, bn;
  int split = 1;  // parts of k, each with sums of its own
  int rows() const { return 128 * ctas; }
};

// What an epilogue thread is at: one row of the tile, and one half of its columns.
struct Where {
  int row;       // of the output
  bool inside;   // row < rows of the output
  uint32_t box;  // shared memory of the warp
  int col;       // the first of this half's columns
  int units;     // of 32 columns in this half
  int next_row, next_col;  // the same of this warp's next tile; beyond the matrix where there is none
  int m_block, n_block, part, half, quarter, lane;
};

__device__ __forceinline__ uint64_t k_major_descriptor(uint32_t address) {
  uint64_t desc = (uint64_t)((address >> 4) & 0x3fffu);
  desc |= (uint64_t)1u << 16;              // leading byte offset: not used with k contiguous
  desc |= (uint64_t)(1024u >> 4) << 32;    // stride byte offset: from 8 rows to the next 8
  desc |= (uint64_t)1u << 46;              // descriptor version of this architecture
  desc |= (uint64_t)2u << 61;              // 128-byte swizzle
  return desc;
}
// m (n) contiguous: boxes of 64 of them by 64 values of k; `group`: bytes from one box to the next 64.
__device__ __forceinline__ uint64_t mn_major_descriptor(uint32_t address, uint32_t group) {
  uint64_t desc = (uint64_t)((address >> 4) & 0x3fffu);
  desc |= (uint64_t)(group >> 4) << 16;    // leading byte offset: to the next 64 of m
  desc |= (uint64_t)(1024u >> 4) << 32;    // stride byte offset: from 8 values of k to the next 8
  desc |= (uint64_t)1u << 46;
  desc |= (uint64_t)2u << 61;
  return desc;
}

// The warps that issue loads and products run as a whole, and `one` (set in one lane, by elect.sync) predicates the instruction itself:
// descriptors, addresses and coordinates are then the same in every lane.  In a branch that one lane takes a product of 16 values of k took 240
// cycles, whatever its columns, where 256 columns need 128; that they were moved to uniform registers for every instruction is inferred from that.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}

template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t one, uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t instruction, uint32_t accumulate) {
  if constexpr (CTAS == 2) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instruction), "r"(accumulate), "r"(one)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instruction), "r"(accumulate), "r"(one)
        : "memory");
  }
}

// Arrives on the barrier (in a pair: on both CTAs') once every tcgen05 operation this thread issued before has completed.
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t one, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)3), "r"(one)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one)
        : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of the first CTA's counterpart of a barrier.
__device__ __forceinline__ uint32_t of_first_cta(const uint64_t *bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(bar)));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 32 columns of this warp's lanes: issued and waited for in one statement, so that nothing reads a register before it arrives.
__device__ __forceinline__ void tmem_load_32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// global -> this CTA's shared memory, issued by the lane that has `one`; `bar`: the barrier that counts the bytes, in a pair the first
// CTA's.
template <int CTAS>
__device__ __forceinline__ void load_3d(uint32_t one, uint32_t dst, const CUtensorMap *map, int col, int row, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];\n\t}" ::"r"(dst),
        "l"(map), "r"(col), "r"(row), "r"(0), "r"(bar), "r"(one)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
        "l"(map), "r"(col), "r"(row), "r"(0), "r"(bar), "r"(one)
        : "memory");
}

template <int CTAS, int PLANES, bool A_MN, bool B_MN, class Epilogue>
__global__ void __launch_bounds__(kTileThreads, 1) dense_tile_kernel(const __grid_constant__ TileArgs a, const __grid_constant__ Epilogue epilogue) {
  constexpr bool kPair = Epilogue::kPair;  // the tile's columns are those of two matrices, half and half
  static_assert(!kPair || !B_MN, "a pair's weights have k contiguous");
  constexpr bool kSplit = PLANES > 1;
  constexpr int kBuffers = kSplit ? 1 : 2;  // accumulators that are used in turn
  extern __shared__ __align__(1024) unsigned char tile_smem[];
  unsigned char *base = tile_smem + ((1024u - (smem_addr(tile_smem) & 1023u)) & 1023u);
  const uint32_t stages = smem_addr(base);
  uint64_t *full = reinterpret_cast<uint64_t *>(base + kStageBudget + kEpilogueWarps * kBoxBytes);  // [stages]
  uint64_t *empty = full + kMostStages;                                // [stages]
  uint64_t *accumulated = empty + kMostStages;                         // [2] an accumulator is complete
  uint64_t *drained = accumulated + 2;                                 // [2] ... and has been read out
  uint64_t *drained_small = drained + 2;                               // the small products' accumulator
  uint64_t *settled = drained_small + 1;                               // every product issued has ended
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(settled + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)cluster_rank() : 0;
  const int first_tile = (int)blockIdx.x / CTAS, tile_step = (int)gridDim.x / CTAS;
  constexpr uint32_t kColumns = 512;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accumulated[b], 1);
      mbar_init(&drained[b], kEpilogueWarps * CTAS);
    }
    mbar_init(drained_small, kEpilogueWarps * CTAS);
    mbar_init(settled, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  auto everybody = [&]() {  // the CTA's threads, or the pair's
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if constexpr (CTAS == 2)
      cluster_sync();
    else
      __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  everybody();
  const uint32_t tmem = *tmem_slot;
  after_previous_kernel();

  auto give_up = [&]() {
    if (a.status_word != nullptr) atomicOr(a.status_word, HT_FLAG_PIPELINE_TIMEOUT);
  };
  // What one turn of the loops is: a tile, and a part of k.  Groups of 16 row blocks, the rows of a group fastest.
  struct Turn {
    int mb, nb, part, first, last;  // blocks of k: first .. last - 1
  };
  const int all_blocks = a.segments * a.k_blocks, per_part = a.m_blocks * a.n_blocks;
  auto place = [&](int index) {
    constexpr int kGroup = 16;
    Turn t;
    t.part = index / per_part;
    const int tile = index - t.part * per_part;
    const int per_group = kGroup * a.n_blocks, g = tile / per_group, in = tile - g * per_group;
    const int rows = min(kGroup, a.m_blocks - g * kGroup);
    t.nb = in / rows;
    t.mb = g * kGroup + (in - t.nb * rows);
    t.first = t.part * a.part_blocks;
    t.last = min(all_blocks, t.first + a.part_blocks);
    return t;
  };
  // A wait of the whole warp.
  auto arrived = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };

  if (warp == 0) {
    {
      const uint32_t one = elect_one();
      uint32_t it = 0, s = 0, phase = 1;
      bool ok = true;
      for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
        const Turn turn = place(tile);
        const int m0 = (turn.mb * CTAS + rank) * kTileM;
        const int half = a.bn / 2;
        // a pair of matrices: one each to the CTAs of a pair, both to one alone
        const int n0 = a.b_n0 + turn.nb * (kPair ? half : a.bn) + (CTAS == 2 && !kPair ? rank * half : 0);
        for (int kb = turn.first; kb < turn.last; ++kb, ++it) {
          if (!arrived(&empty[s], phase)) {
            give_up();
            ok = false;
            break;
          }
          const int segment = kb >= a.k_blocks ? 1 : 0;
          const int k0 = (kb - segment * a.k_blocks) * kTileK;
          const uint32_t at = stages + s * a.stage_bytes, bt = at + a.a_bytes;
          const uint32_t bar = CTAS == 2 ? of_first_cta(&full[s]) : smem_addr(&full[s]);
          if (rank == 0 && one) mbar_expect_tx(&full[s], a.stage_bytes * CTAS);
          const CUtensorMap *am = &a.a[segment], *bm = &a.b[segment];
          if (A_MN) {
            for (int g = 0; g < kTileM / 64; ++g) load_3d<CTAS>(one, at + (uint32_t)g * (8192u * PLANES), am, m0 + 64 * g, k0, bar);
          } else {
            load_3d<CTAS>(one, at, am, k0, m0, bar);
          }
          if (B_MN) {
            for (int g = 0; g < (a.bn / CTAS + 63) / 64; ++g) load_3d<CTAS>(one, bt + (uint32_t)g * (8192u * PLANES), bm, n0 + 64 * g, a.b_k0 + k0, bar);
          } else if (kPair) {
            load_3d<CTAS>(one, bt, &a.b[rank], k0, n0, bar);
            if (CTAS == 1) load_3d<CTAS>(one, bt + (uint32_t)half * 128u * PLANES, &a.b[1], k0, n0, bar);
          } else {
            load_3d<CTAS>(one, bt, bm, a.b_k0 + k0, n0, bar);
          }
          if (++s == (uint32_t)a.stages) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      // The last use of every stage ends before the CTA leaves: the commits that arrive here (in a pair, from the other CTA), or, where a
      // wait ran out, the copies still in flight.
      const uint32_t issued = min(it, (uint32_t)a.stages);
      for (uint32_t j = 1; j <= issued; ++j) {
        const uint32_t i = it - j, s = i % (uint32_t)a.stages;
        mbar_wait(ok ? &empty[s] : &full[s], (i / (uint32_t)a.stages) & 1u, ok ? kMaxSpins : 4096);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t one = elect_one();
      const uint32_t tmem_d = __reduce_or_sync(0xffffffffu, tmem);  // the same in a uniform register
      uint32_t s = 0, phase = 0, chunk = 0, t = 0;
      // A lane whose wait ran out waits no more, and the warp goes on: the products of what the stages hold are thrown away, and no branch
      // depends on a wait.
      bool ok = true;
      auto wait_here = [&](uint64_t *bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity)) {
          ok = false;
          give_up();
        }
      };
      // rows of B in a CTA; two matrices in one CTA lie one after the other, plane by plane
      const uint32_t b_rows = (uint32_t)(CTAS == 2 || kPair ? a.bn / 2 : a.bn);
      const uint64_t a_plane = (A_MN ? 8192u : (uint32_t)kTileM * 128u) >> 4, b_plane = (B_MN ? 8192u : b_rows * 128u) >> 4;
      constexpr uint32_t step_a = A_MN ? 128u : 2u, step_b = B_MN ? 128u : 2u;  // 16 values of k, in units of 16 bytes
      for (int tile = first_tile; tile < a.tiles; tile += tile_step, ++t) {
        uint32_t d = tmem_d;
        const Turn at_work = place(tile);
        for (int kb = at_work.first; kb < at_work.last; ++kb) {
          const int since = kb - at_work.first;
          const bool first = kSplit ? since % kChunkBlocks<PLANES> == 0 : since == 0;
          if (kSplit && since == 0) wait_here(drained_small, (t & 1u) ^ 1u);
          const uint32_t buffer = chunk % kBuffers;
          auto turn = [&]() {  // the accumulator's previous sum has been read
            if (!first) return;
            d = tmem_d + buffer * 256u;
            wait_here(&drained[buffer], ((chunk / kBuffers) & 1u) ^ 1u);
          };
          if (!kSplit) turn();
          wait_here(&full[s], phase);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int left = a.k - (kb >= a.k_blocks ? kb - a.k_blocks : kb) * kTileK;
          const int steps = left >= kTileK ? 4 : (left + 15) / 16;
          const uint32_t at = stages + s * a.stage_bytes, bt = at + a.a_bytes;
          const uint64_t da = A_MN ? mn_major_descriptor(at, 8192u * PLANES) : k_major_descriptor(at);
          const uint64_t db = B_MN ? mn_major_descriptor(bt, 8192u * PLANES) : k_major_descriptor(bt);
          constexpr int kParts = kSplit && kPair && CTAS == 1 ? 2 : 1;  // two matrices in one CTA, several planes: an instruction each
          auto large = [&](int kk) {
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              mma_f16<CTAS>(one, d + (uint32_t)part * b_rows, da + (uint64_t)(step_a * (uint32_t)kk),
                            db + (uint64_t)part * (PLANES * b_plane) + (uint64_t)(step_b * (uint32_t)kk), a.instruction, kk > 0 || !first);
          };
          auto small = [&](int kk) {
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint64_t ak = da + (uint64_t)(step_a * (uint32_t)kk);
              const uint64_t bk = db + (uint64_t)part * (PLANES * b_plane) + (uint64_t)(step_b * (uint32_t)kk);
              const uint32_t to = tmem_d + 256u + (uint32_t)part * b_rows;
              if constexpr (PLANES == 3) {
                mma_f16<CTAS>(one, to, ak + 2 * a_plane, bk, a.instruction, kk > 0 || since > 0);
                mma_f16<CTAS>(one, to, ak, bk + 2 * b_plane, a.instruction, 1u);
                mma_f16<CTAS>(one, to, ak + a_plane, bk + b_plane, a.instruction, 1u);
              }
              mma_f16<CTAS>(one, to, ak + a_plane, bk, a.instruction, PLANES == 3 || kk > 0 || since > 0);
              mma_f16<CTAS>(one, to, ak, bk + b_plane, a.instruction, 1u);
            }
          };
          if (kSplit) {
            for (int kk = 0; kk < steps; ++kk) small(kk);
            turn();
            if (first) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          if (steps == 4) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) large(kk);
          } else {
            for (int kk = 0; kk < steps; ++kk) large(kk);
          }
          mma_commit<CTAS>(one, smem_addr(&empty[s]));
          if (++s == (uint32_t)a.stages) {
            s = 0;
            phase ^= 1u;
          }
          if (kb == at_work.last - 1 || (kSplit && since % kChunkBlocks<PLANES> == kChunkBlocks<PLANES> - 1)) {
            mma_commit<CTAS>(one, smem_addr(&accumulated[buffer]));
            ++chunk;
          }
        }
      }
      // whatever became of the waits: tensor memory is not freed under a product
      mma_commit<CTAS>(one, smem_addr(settled));
      mbar_wait(settled, 0u);
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;  // a warp may only touch the lanes 32 (warp % 4) ...
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t chunk = 0;
    // of 32 columns (a pair: 32 of each), the first half of them, rounded up, for one of the two warps
    const int all_units = kPair ? a.bn / 64 : a.bn / 32, unit0 = half * ((all_units + 1) / 2), units = (all_units + 1 - half) / 2;
    Where w;
    w.half = half, w.quarter = quarter, w.lane = lane, w.units = units;
    w.box = stages + kStageBudget + (uint32_t)(warp - 2) * kBoxBytes;
    auto wait_for = [&](uint32_t c) {
      bool there = mbar_wait(&accumulated[c % kBuffers], (c / kBuffers) & 1u);
      if (!there) give_up();
      there = __all_sync(0xffffffffu, there);  // a warp reads tensor memory together or not at all
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return there;
    };
    auto release = [&](uint64_t *bar) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if constexpr (CTAS == 2)
          // (relaxed: what is handed back is tensor memory that has been read; a release would wait for the stores of the tile before)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(of_first_cta(bar)) : "memory");
        else
          mbar_arrive(bar);
      }
    };
    for (int tile = first_tile; tile < a.tiles; tile += tile_step) {
      const Turn turn = place(tile);
      w.n_block = turn.nb, w.part = turn.part;
      w.m_block = turn.mb * CTAS + rank;
      w.row = w.m_block * kTileM + quarter * 32 + lane;
      w.inside = w.row < epilogue.rows;
      typename Epilogue::State state;
      const int col0 = w.n_block * (kPair ? a.bn / 2 : a.bn);
      w.col = col0 + unit0 * 32;
      w.next_row = 0x7fffffff, w.next_col = 0;
      if (tile + tile_step < a.tiles) {
        const Turn next = place(tile + tile_step);
        w.next_row = (next.mb * CTAS + rank) * kTileM + quarter * 32 + lane;
        w.next_col = next.nb * (kPair ? a.bn / 2 : a.bn) + unit0 * 32;
      }
      epilogue.begin(state, w, tile == first_tile);  // under the tile's products
      if constexpr (!kSplit) {
        if (!wait_for(chunk)) break;
        const uint32_t acc = lanes + (chunk & 1u) * 256u;
#pragma unroll 1
        for (int u = 0; u < units; ++u) {
          const int c = (unit0 + u) * 32;
          float v[32];
          tmem_load_32(acc + (uint32_t)c, v);
          if constexpr (kPair) {
            float v2[32];
            tmem_load_32(acc + (uint32_t)(a.bn / 2 + c), v2);
            if (u == units - 1) release(&drained[chunk & 1u]);
            epilogue.unit(state, w, col0 + c, v, v2);
          } else {
            if (u == units - 1) release(&drained[chunk & 1u]);
            epilogue.unit(state, w, col0 + c, v);
          }
        }
        ++chunk;
      } else {
        // sums over the chunks of k in registers: up to 4 x 32 columns (a pair: 2 x 32 of each matrix, the gate's first)
        constexpr int kMostUnits = CTAS == 2 ? 4 : 2;
        float sum[kMostUnits][32];
        const int parts = kPair ? 2 * units : units;
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[u][i] = 0.0f;
        auto column = [&](int u) { return kPair ? (u & 1) * (a.bn / 2) + (unit0 + (u >> 1)) * 32 : (unit0 + u) * 32; };
        bool there = true;
        const int chunks = (turn.last - turn.first + kChunkBlocks<PLANES> - 1) / kChunkBlocks<PLANES>;
        for (int c = 0; c <= chunks; ++c) {
          if (c < chunks && !(there = wait_for(chunk))) break;
          const uint32_t acc = lanes + (c < chunks ? 0u : 256u);
#pragma unroll
          for (int u = 0; u < kMostUnits; ++u) {
            if (u >= parts) break;
            float v[32];
            tmem_load_32(acc + (uint32_t)column(u), v);
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[u][i] += v[i];
          }
          if (c < chunks) ++chunk;
          release(c < chunks ? &drained[0] : drained_small);
        }
        if (!there) break;
        // one copy of the epilogue's code, and the columns pass by: four copies did not stay in the instruction cache
        constexpr int kAtOnce = kPair ? 2 : 1;
#pragma unroll 1
        for (int u = 0; u < parts; u += kAtOnce) {
          if constexpr (kPair)
            epilogue.unit(state, w, col0 + column(u), sum[0], sum[1]);
          else
            epilogue.unit(state, w, col0 + column(u), sum[0]);
#pragma unroll
          for (int q = 0; q + kAtOnce < kMostUnits; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[q][i] = sum[q + kAtOnce][i];
        }
      }
      epilogue.end(state, w);
    }
  }
  everybody();
  if (warp == 1) {
    if constexpr (CTAS == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
  if constexpr (CTAS == 2) cluster_sync();
}

// ---- host side -------------------------------------------------------------------------------------------------------

// Boxes of 64 columns (128 bytes) by `box_rows` rows of every plane.
inline bool encode_matrix_16(CUtensorMap *map, const Matrix &m, int box_rows) {
  tma::EncodeTiledFn fn = tma::encode_tiled_fn();
  if (fn == nullptr) return false;
  if ((reinterpret_cast<uintptr_t>(m.data) & 15u) != 0 || (m.pitch & 7) != 0 || (m.plane & 7) != 0) return false;
  if (m.rows < 1 || m.cols < 1 || m.rows > 0x7fffffff || m.cols > 0x7fffffff || box_rows < 1 || box_rows > 256) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)m.planes};
  const cuuint64_t strides[2] = {(cuuint64_t)m.pitch * 2u, (cuuint64_t)(m.planes > 1 ? m.plane : m.pitch) * 2u};
  const cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, (cuuint32_t)m.planes};
  const cuuint32_t elem[3] = {1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(m.data), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct TileProblem {
  Matrix a[2], b[2];       // a pair: b[0] and b[1] side by side; two segments: a[0] b[0] + a[1] b[1]
  int segments = 1;
  int64_t rows = 0, cols = 0, k = 0;  // cols: of the output (a pair: of each matrix)
  int64_t b_n0 = 0, b_k0 = 0;
  bool f16 = false;        // operands in fp16, else bf16
  uint32_t *status_word = nullptr;
};

inline int sm_count(int *sms) {
  int device = 0;
  HT_CUDA_TRY(cudaGetDevice(&device));
  HT_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
  return HT_OK;
}

// How to cut a product: the shape with which the SMs are done first.  Cycles of a step of 16 values of k, measured: a pair of CTAs with 256
// columns 160, with 128 columns 118, in steps of 32 between; one CTA with 256 columns 170, with 192 150, with 128 125, with 64 120
// (three planes: 6 of those, two: 3, of 128 columns at the most alone).  A tile costs about 1300 cycles besides, a launch in pairs 1200.  Against
// that, the operands have to come from memory once, 23 bytes a cycle and SM where all read, twice that where few do.  Where `most_parts`
// allows it, k is cut as well: each part writes its sums in fp32, and a kernel adds them (8 bytes a value and part, about 6000 cycles).
// Measured against the other shapes, us: 1555 x 336 to 2 x 1008, bf16: 7.5 with what is taken, alone and 256, 8.1 to 8.9 with others; 1003 x
// 776 x 10008: 24.5 in pairs, 30.8 and 33.6 alone; 600 x 2048 to 2 x 300, fp32: 39 with 128 columns, 67 with 256.
inline TileShape tile_shape(int64_t rows, int64_t cols, int64_t k, int planes, bool pair, int most_parts = 1) {
  constexpr int kPlanSMs = 148;
  constexpr double kBytesPerCycle = 23.0;
  TileShape best = {1, 128};
  double least = 0.0;
  for (int split = 1; split <= most_parts && (split == 1 || k / split >= 4 * kTileK); ++split)
    for (int ctas = 2; ctas >= 1; --ctas)
      for (int bn = ctas == 1 && planes > 1 ? 128 : 256; bn >= (ctas == 2 || pair ? 128 : 64); bn -= 32) {
        if (bn % (ctas == 2 ? (pair ? 64 : 32) : pair ? 128 : 64) != 0) continue;
        const int64_t n = pair ? bn / 2 : bn;
        const int64_t tiles = ((rows + 128 * ctas - 1) / (128 * ctas)) * ((cols + n - 1) / n) * ctas * split, last = tiles % kPlanSMs;
        const double rounds = (double)((tiles + kPlanSMs - 1) / kPlanSMs);
        const double step = ctas == 2 ? 75.0 + 0.335 * bn : bn == 256 ? 170.0 : bn == 192 ? 150.0 : bn == 128 ? 125.0 : 120.0;
        const double products = rounds * ((planes == 3 ? 6.0 : planes == 2 ? 3.0 : 1.0) * (double)((k / split + 15) / 16) * step + 1300.0) + (ctas == 2 ? 1200.0 : 0.0);
        const double bytes = 2.0 * planes * (double)k * (double)(rows + cols * (pair ? 2 : 1)) / (double)tiles;
        const double memory = bytes / kBytesPerCycle * ((double)(tiles / kPlanSMs) + (last > 0 ? std::max(0.5, (double)last / kPlanSMs) : 0.0));
        const double sums = split > 1 ? 6000.0 + 8.0 * split * (double)rows * (double)cols / (kBytesPerCycle * kPlanSMs) : 0.0;
        const double cycles = std::max(products, memory) + sums;
        if (least == 0.0 || cycles < least * 0.999) {
          best = {ctas, bn, split};
          least = cycles;
        }
      }
  return best;
}

constexpr int round_up_to(int v, int to) { return (v + to - 1) / to * to; }

// Blocks of k in a part, and the parts that have any.
inline int part_blocks_of(const TileProblem &p, const TileShape &shape) {
  return (int)((p.segments * ((p.k + kTileK - 1) / kTileK) + shape.split - 1) / shape.split);
}
inline int parts_of(const TileProblem &p, const TileShape &shape) {
  const int per = part_blocks_of(p, shape);
  return (int)((p.segments * ((p.k + kTileK - 1) / kTileK) + per - 1) / per);
}

template <int PLANES, bool A_MN, bool B_MN, class Epilogue>
int launch_tiles(const TileProblem &p, const Epilogue &epilogue, const TileShape &shape, int sms, cudaStream_t stream) {
  constexpr bool kPair = Epilogue::kPair;
  if (p.rows < 1 || p.cols < 1 || p.k < 1) return HT_ERR_INVALID_ARGUMENT;
  TileArgs a = {};
  const int bn = shape.bn, columns = kPair ? bn / 2 : bn;  // of the output
  const int b_rows = kPair || shape.ctas == 2 ? bn / 2 : bn;   // of one load
  for (int s = 0; s < p.segments || (kPair && s < 2); ++s) {
    if (s < p.segments && !encode_matrix_16(&a.a[s], p.a[s], A_MN ? kTileK : kTileM)) return HT_ERR_UNSUPPORTED;
    if (!encode_matrix_16(&a.b[s], p.b[s], B_MN ? kTileK : b_rows)) return HT_ERR_UNSUPPORTED;
  }
  const int64_t m_blocks = (p.rows + shape.rows() - 1) / shape.rows(), n_blocks = (p.cols + columns - 1) / columns;
  if (m_blocks * n_blocks * shape.split > 0x3fffffff || p.k > 0x3fffffff) return HT_ERR_UNSUPPORTED;
  a.status_word = p.status_word;
  const int n = PLANES > 1 && kPair && shape.ctas == 1 ? bn / 2 : bn;  // columns of one instruction
  a.instruction = (1u << 4) | ((p.f16 ? 0u : 1u) << 7) | ((p.f16 ? 0u : 1u) << 10) | ((A_MN ? 1u : 0u) << 15) |
                  ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(shape.rows() >> 4) << 24);
  a.m_blocks = (int)m_blocks;
  a.n_blocks = (int)n_blocks;
  a.tiles = (int)(m_blocks * n_blocks * parts_of(p, shape));
  a.bn = bn;
  a.k = (int)p.k;
  a.k_blocks = (int)((p.k + kTileK - 1) / kTileK);
  a.segments = p.segments;
  a.part_blocks = part_blocks_of(p, shape);
  a.b_n0 = (int)p.b_n0;
  a.b_k0 = (int)p.b_k0;
  a.a_bytes = (uint32_t)kTileM * 128u * PLANES;
  a.stage_bytes = a.a_bytes + (uint32_t)(B_MN ? round_up_to(bn / shape.ctas, 64) : bn / shape.ctas) * 128u * PLANES;
  a.stages = (int)std::min<uint32_t>(kStageBudget / a.stage_bytes, kMostStages);
  const dim3 grid((unsigned)(shape.ctas * std::min(a.tiles, std::max(sms / shape.ctas, 1))));
  return shape.ctas == 2 ? launch_next<dense_tile_kernel<2, PLANES, A_MN, B_MN, Epilogue>>(grid, kTileThreads, kTileSmem, kTileSmem, stream, 2, a, epilogue)
                         : launch_next<dense_tile_kernel<1, PLANES, A_MN, B_MN, Epilogue>>(grid, kTileThreads, kTileSmem, kTileSmem, stream, 1, a, epilogue);
}

}  // namespace dense
}  // namespace ht

// Tile product under weights held as microscaled 4-bit numbers (ht_mx4.cuh), on the tensor cores:
//
//     y[n, o] = sum_k x[n, k] W[o, k]       x as 1, 2 or 3 bf16 numbers a value, W exact in bf16, fp32 accumulation in tensor memory
//
// The 128 outputs of a tile are the rows of tcgen05.mma and x's rows its columns.  Weights are never written as bf16 but to tensor memory, where the
// instruction takes its first operand from: a thread has an output, which is a lane, reads 32 bytes of its codes from shared memory, multiplies them with
// their scales and stores 64 values of k as 32 columns.  What is left in shared memory is x alone, read once by the tensor core, and a weight costs
// 17 bytes of traffic for 32.
//
// A persistent kernel of 480 threads a CTA, one CTA an SM:
//   warp 0       one lane issues the TMA loads of x into a ring of 4 stages of 64 values of k;
//   warp 1       allocates tensor memory; one lane issues tcgen05.mma.kind::f16 (M 128, N up to 192, K 16, the first operand in tensor memory) and
//                commits each stage to those who fill it, and each finished accumulator to the epilogue;
//   warps 2-5    the epilogue, a quarter of the lanes each, under the next tile's products;
//   warps 6-13   the weights: two sets of four warps, a quarter of the lanes each, take every other stage of a box;
//   warp 14      one lane issues the TMA loads of codes into a ring of 4 boxes of 256 values of k, ahead of x.
// Tensor memory: two accumulators in turn (three numbers: of two parts each), and 4 stages of 32 columns of weights.
// With three numbers the products of the first one have an accumulator, those of the others, 2^-8 of them, a second; both leave for
// registers every 256 values of k and are added there in fp32 (the tensor core truncates when it adds; ht_dense_tile.cuh).
// What bounds it: power and the tensor pipe with many rows (8192 x 1024 to 50000 of bf16: 680 to 690 us in a burst, 1220 TFLOP/s, and 790 in a
// long loop; ht_linear_mx4.cu decodes once there);
// with few the decoding, 280 cycles for a stage (64 rows 17 us, 17 rows 16.7).  The product with both operands in shared memory needs 48 cycles for 16
// values of k and 64 columns, this one 32, and 96 with 192, the tensor core's own rate.
// A tile starts with the first stage of the ring: the last box of a tile may leave stages out.  Every wait is bounded, as in ht_dense_tile.cuh.
#pragma once

#include "ht_mx4.cuh"

namespace ht {
namespace mx4 {

using namespace tile;
using dense::load_plain;

constexpr int kTileM = 128, kTileK = 64;
constexpr int kTileThreads = 480;
constexpr int kStages = 4, kBoxes = 4, kBoxStages = 4;
constexpr uint32_t kBoxBytes = kTileM * 128;
constexpr int kWeightWarps = 8, kSetWarps = 4, kEpilogueWarps = 4;
constexpr uint32_t kWeightColumn = 384;
// Rows of x in a tile at the most, and the columns of an accumulator.
template <int P>
constexpr int kMostRows = P == 1 ? 192 : P == 2 ? 128 : 96;
template <int P>
constexpr size_t kTileBytes = 1024 + (size_t)kStages * P * kMostRows<P> * 128 + (size_t)kBoxes * kBoxBytes + 512;

struct alignas(64) TileArgs {
  CUtensorMap x, codes;
  const uint8_t *scales;
  uint32_t *status_word;
  uint32_t instruction;
  int rows, outputs, blocks, k;
  int bn;  // rows of x in a tile
  int m_blocks, n_blocks, tiles, k_blocks;
};

// The instructions of the warp that issues the products are few and follow one another closely: with a wait for x, one for weights and calls
// of general helpers a stage of 64 columns took 730 cycles of it, twice what 192 columns need of the tensor core.
__device__ __forceinline__ void mma_weights(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t instruction, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(instruction), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Whether a barrier's phase has passed, without waiting.
__device__ __forceinline__ bool passed(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for it, `tries` times at the most; 0 is left when they ran out, and no wait after that tries more than once.
__device__ __forceinline__ void wait_for_phase(uint64_t *bar, uint32_t parity, uint32_t &tries) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, %0;\n\t"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.gt.s32 q, n, 0;\n\t"
      "@q bra AGAIN;\n\t"
      "mov.u32 %0, 0;\n\t"
      "DONE:\n\t}"
      : "+r"(tries)
      : "r"(smem_addr(bar)), "r"(parity), "n"(kTryNanoseconds)
      : "memory");
}
__device__ __forceinline__ void load_2d(uint32_t one, uint32_t dst, const CUtensorMap *map, int col, int row, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
      "l"(map), "r"(col), "r"(row), "r"(bar), "r"(one)
      : "memory");
}
// 32 columns of this warp's lanes, and the wait until they are there.
__device__ __forceinline__ void tmem_store_32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n\t"
      "tcgen05.wait::st.sync.aligned;"
      :
      : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

template <typename T, int P>
__global__ void __launch_bounds__(kTileThreads, 1) mx4_tile_kernel(const __grid_constant__ TileArgs a, const T *bias, T *y) {
  extern __shared__ __align__(1024) unsigned char mx4_smem[];
  unsigned char *base = mx4_smem + ((1024u - (smem_addr(mx4_smem) & 1023u)) & 1023u);
  const uint32_t stage_bytes = (uint32_t)(P * a.bn) * 128u;
  const uint32_t boxes = smem_addr(base), stages = boxes + kBoxes * kBoxBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(base + kBoxes * kBoxBytes + (size_t)kStages * P * kMostRows<P> * 128);  // x and weights are there
  uint64_t *empty = full + kStages;           // of both
  uint64_t *box_full = empty + kStages;       // codes
  uint64_t *box_empty = box_full + kBoxes;
  uint64_t *accumulated = box_empty + kBoxes; // [2] an accumulator is complete
  uint64_t *drained = accumulated + 2;        // [2] ... and has been read out
  uint64_t *settled = drained + 2;            // every product issued has ended
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(settled + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kColumns = 512;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1 + kSetWarps);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBoxes; ++b) {
      mbar_init(&box_full[b], 1);
      mbar_init(&box_empty[b], kWeightWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accumulated[b], 1);
      mbar_init(&drained[b], kEpilogueWarps);
    }
    mbar_init(settled, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  auto everybody = [&]() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  everybody();
  const uint32_t tmem = *tmem_slot;
  dense::after_previous_kernel();

  auto give_up = [&]() {
    if (a.status_word != nullptr) atomicOr(a.status_word, HT_FLAG_PIPELINE_TIMEOUT);
  };
  // Tiles go in groups of 16 blocks of outputs, those of a group fastest.
  struct Turn {
    int mb, nb;
  };
  auto place = [&](int tile) {
    constexpr int kGroup = 16;
    const int per_group = kGroup * a.n_blocks, g = tile / per_group, in = tile - g * per_group;
    const int blocks = min(kGroup, a.m_blocks - g * kGroup);
    Turn t;
    t.nb = in / blocks;
    t.mb = g * kGroup + (in - t.nb * blocks);
    return t;
  };
  auto arrived = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
  const int tile_boxes = (a.k_blocks + kBoxStages - 1) / kBoxStages;

  if (warp == 0) {
    const uint32_t one = dense::elect_one();
    uint32_t phases = 0xfu, used = 0;  // a bit for each stage
    bool ok = true;
    for (int tile = (int)blockIdx.x; tile < a.tiles && ok; tile += (int)gridDim.x) {
      const Turn turn = place(tile);
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        const uint32_t s = (uint32_t)kb % kStages;  // (a tile starts with the first stage)
        if (!(ok = arrived(&empty[s], (phases >> s) & 1u))) break;
        phases ^= 1u << s;
        used |= 1u << s;
        if (one) mbar_expect_tx(&full[s], stage_bytes);
        dense::load_3d<1>(one, stages + s * stage_bytes, &a.x, kb * kTileK, turn.nb * a.bn, smem_addr(&full[s]));
      }
    }
    if (!ok) give_up();
    // The last use of every stage ends before the CTA leaves, or, where a wait ran out, the copies still in flight.
    for (uint32_t s = 0; s < kStages; ++s)
      if ((used >> s) & 1u) mbar_wait(ok ? &empty[s] : &full[s], (phases >> s) & 1u, ok ? kMaxSpins : 4096);
  } else if (warp == 1) {
    const uint32_t tmem_d = __reduce_or_sync(0xffffffffu, tmem);  // the same in a uniform register
    uint32_t chunk = 0, tries = kMaxSpins, phases = 0;  // phases: of each stage's barrier, a bit
    const uint32_t plane = (uint32_t)a.bn * 128u >> 4;
    const int last_steps = (a.k - (a.k_blocks - 1) * kTileK + 15) / 16;
    bool there[2] = {false, false};
    for (int tile = (int)blockIdx.x; tile < a.tiles; tile += (int)gridDim.x) {
      for (int q = 0; q < tile_boxes; ++q) {
        const uint32_t buffer = chunk & 1u, d = tmem_d + buffer * (kWeightColumn / 2);
        const int here = min(kBoxStages, a.k_blocks - q * kBoxStages);
        const bool last = q == tile_boxes - 1, fresh = P == 3 || q == 0, ends = P == 3 || last;
        if (fresh) wait_for_phase(&drained[buffer], ((chunk >> 1) & 1u) ^ 1u, tries);
#pragma unroll
        for (int s = 0; s < kStages; s += 2) {  // two stages at a time; the barriers of the next two are looked at under their products
          if (s >= here) break;
          const bool both = s + 1 < here;
          if (!there[0]) wait_for_phase(&full[s], (phases >> s) & 1u, tries);
          if (both && !there[1]) wait_for_phase(&full[s + 1], (phases >> (s + 1)) & 1u, tries);
          phases ^= both ? 3u << s : 1u << s;
          const int next = s + 2 < here ? s + 2 : 0;
          there[0] = passed(&full[next], (phases >> next) & 1u);
          there[1] = passed(&full[next + 1], (phases >> (next + 1)) & 1u);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (dense::elect_one()) {
            auto products = [&](int stage, int kk) {
              const uint32_t more = s > 0 || stage > 0 || kk > 0 || !fresh;
              const uint64_t db = dense::k_major_descriptor(stages + (uint32_t)(s + stage) * stage_bytes) + 2u * (uint32_t)kk;
              const uint32_t wa = tmem_d + kWeightColumn + (uint32_t)(s + stage) * 32u + 8u * (uint32_t)kk;
              if constexpr (P == 3) {
                const uint32_t small = d + kMostRows<3>;
                mma_weights(small, wa, db + 2 * plane, a.instruction, more);
                mma_weights(small, wa, db + plane, a.instruction, 1u);
              } else if constexpr (P == 2) {
                mma_weights(d, wa, db + plane, a.instruction, more);
              }
              mma_weights(d, wa, db, a.instruction, P == 2 ? 1u : more);
            };
            const bool ends_here = last && s + 2 >= here;  // the tile's last stage is one of these
#pragma unroll
            for (int stage = 0; stage < 2; ++stage) {
              if (stage == 1 && !both) break;
              if (ends_here && s + stage == here - 1) {
                for (int kk = 0; kk < last_steps; ++kk) products(stage, kk);
              } else {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) products(stage, kk);
              }
              commit(&empty[s + stage]);
            }
            if (ends && s + 2 >= here) commit(&accumulated[buffer]);
          }
          __syncwarp();
        }
        if (ends) ++chunk;
      }
    }
    if (tries == 0) give_up();
    // whatever became of the waits: tensor memory is not freed under a product
    if (dense::elect_one()) commit(settled);
    __syncwarp();
    mbar_wait(settled, 0u);
  } else if (warp < 2 + kEpilogueWarps) {
    const int quarter = warp & 3;  // a warp may only touch the lanes 32 (warp % 4) ...
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t chunk = 0;
    const int units = a.bn / 32;
    auto wait_for = [&](uint32_t c) {
      const bool there = arrived(&accumulated[c & 1u], (c >> 1) & 1u);
      if (!there) give_up();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return there;
    };
    auto release = [&](uint32_t c) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[c & 1u]);
    };
    for (int tile = (int)blockIdx.x; tile < a.tiles; tile += (int)gridDim.x) {
      const Turn turn = place(tile);
      const int o = turn.mb * kTileM + quarter * 32 + lane;
      const float add = bias != nullptr && o < a.outputs ? dense::to_float(bias[o]) : 0.0f;
      auto store = [&](int unit, const float (&v)[32]) {
        const int row = turn.nb * a.bn + 32 * unit, count = a.rows - row;
        if (o >= a.outputs) return;
        T *const to = y + (int64_t)row * a.outputs + o;
        if (count >= 32) {
#pragma unroll
          for (int c = 0; c < 32; ++c) to[(uint64_t)(uint32_t)a.outputs * (uint32_t)c] = dense::from_float<T>(fmaf(v[c], kHeld, add));
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c < count) to[(uint64_t)(uint32_t)a.outputs * (uint32_t)c] = dense::from_float<T>(fmaf(v[c], kHeld, add));
        }
      };
      if constexpr (P < 3) {
        if (!wait_for(chunk)) break;
        const uint32_t acc = lanes + (chunk & 1u) * (kWeightColumn / 2);
#pragma unroll 1
        for (int u = 0; u < units; ++u) {
          float v[32];
          dense::tmem_load_32(acc + 32u * (uint32_t)u, v);
          if (u == units - 1) release(chunk);
          store(u, v);
        }
        ++chunk;
      } else {
        constexpr int kUnits = kMostRows<3> / 32;
        float sum[kUnits][32];
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[u][i] = 0.0f;
        const int chunks = tile_boxes;
        bool there = true;
        for (int c = 0; c < chunks && (there = wait_for(chunk)); ++c, ++chunk) {
          const uint32_t acc = lanes + (chunk & 1u) * (kWeightColumn / 2);
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            if (u >= units) break;
            float v[32];
#pragma unroll
            for (int part = 1; part >= 0; --part) {
              dense::tmem_load_32(acc + 32u * (uint32_t)u + (uint32_t)(part * kMostRows<3>), v);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[u][i] += v[i];
            }
          }
          release(chunk);
        }
        if (!there) break;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (u < units) store(u, sum[u]);
      }
    }
  } else if (warp == kTileThreads / 32 - 1) {
    const uint32_t one = dense::elect_one();
    uint32_t box = 0;
    bool ok = true;
    for (int tile = (int)blockIdx.x; tile < a.tiles && ok; tile += (int)gridDim.x) {
      const Turn turn = place(tile);
      for (int q = 0; q < tile_boxes; ++q, ++box) {
        const uint32_t b = box % kBoxes;
        if (!(ok = arrived(&box_empty[b], ((box / kBoxes) & 1u) ^ 1u))) break;
        if (one) mbar_expect_tx(&box_full[b], kBoxBytes);
        load_2d(one, boxes + b * kBoxBytes, &a.codes, q * 128, turn.mb * kTileM, smem_addr(&box_full[b]));
      }
    }
    if (!ok) give_up();
    const uint32_t issued = min(box, (uint32_t)kBoxes);
    for (uint32_t j = 1; j <= issued; ++j) {
      const uint32_t i = box - j, b = i % kBoxes;
      mbar_wait(ok ? &box_empty[b] : &box_full[b], (i / kBoxes) & 1u, ok ? kMaxSpins : 4096);
    }
  } else {
    const int quarter = warp & 3, set = (warp - 2 - kEpilogueWarps) / kSetWarps;
    const int at = quarter * 32 + lane;  // this thread's output in a tile
    const uint32_t number = opaque_one();
    const uint32_t weights = tmem + ((uint32_t)(quarter * 32) << 16) + kWeightColumn;
    // The scales of this thread's stages of a box: two stages of two blocks.  Loaded a box ahead, and not touched before they are used.
    struct Scales {
      uint8_t b[4];
    };
    auto scales_of = [&](int tile) { return a.scales + (int64_t)min(place(min(tile, a.tiles - 1)).mb * kTileM + at, a.outputs - 1) * a.blocks; };
    auto fetch_scales = [&](const uint8_t *from, int q) {
      Scales r;
      const int first = 2 * (q * kBoxStages + set);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int block = first + 4 * (j >> 1) + (j & 1);
        r.b[j] = 127;
        if (block < a.blocks) r.b[j] = load_plain(from + block);
      }
      return r;
    };
    uint32_t box = 0, phases = 0xfu;
    const uint8_t *from = scales_of((int)blockIdx.x);
    Scales next = fetch_scales(from, 0);
    bool ok = true;
    for (int tile = (int)blockIdx.x; tile < a.tiles && ok; tile += (int)gridDim.x) {
      for (int q = 0; q < tile_boxes; ++q, ++box) {
        const Scales scales = next;
        const int stages_here = min(kBoxStages, a.k_blocks - q * kBoxStages);
        if (q + 1 == tile_boxes) from = scales_of(tile + (int)gridDim.x);
        next = fetch_scales(from, q + 1 < tile_boxes ? q + 1 : 0);
        const uint32_t b = box % kBoxes;
        if (!(ok = arrived(&box_full[b], (box / kBoxes) & 1u))) break;
        const uint32_t row = boxes + b * kBoxBytes + (uint32_t)at * 128u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int in_box = set + 2 * j;
          if (in_box >= stages_here) break;
          const uint4 c0 = lds_b128(row + 16u * ((uint32_t)(2 * in_box) ^ ((uint32_t)at & 7u)));
          const uint4 c1 = lds_b128(row + 16u * ((uint32_t)(2 * in_box + 1) ^ ((uint32_t)at & 7u)));
          const Scale s0 = scale_of(scales.b[2 * j]), s1 = scale_of(scales.b[2 * j + 1]);
          uint32_t v[32];
          weights_of(c0.x, s0, number, v), weights_of(c0.y, s0, number, v + 4), weights_of(c0.z, s0, number, v + 8), weights_of(c0.w, s0, number, v + 12);
          weights_of(c1.x, s1, number, v + 16), weights_of(c1.y, s1, number, v + 20), weights_of(c1.z, s1, number, v + 24), weights_of(c1.w, s1, number, v + 28);
          const uint32_t s = (uint32_t)in_box;
          if (!(ok = arrived(&empty[s], (phases >> s) & 1u))) break;
          phases ^= 1u << s;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          tmem_store_32(weights + s * 32u, v);
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&box_empty[b]);
      }
    }
    if (!ok) give_up();
  }
  everybody();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
}

// Boxes of 128 bytes of 128 rows of the codes.
inline bool encode_codes(CUtensorMap *map, const void *codes, int64_t outputs, int64_t blocks) {
  tma::EncodeTiledFn fn = tma::encode_tiled_fn();
  if (fn == nullptr || (reinterpret_cast<uintptr_t>(codes) & 15u) != 0) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)blocks * 16u, (cuuint64_t)outputs};
  const cuuint64_t strides[1] = {(cuuint64_t)blocks * 16u};
  const cuuint32_t box[2] = {128u, (cuuint32_t)kTileM};
  const cuuint32_t elem[2] = {1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of x in a tile: those with which the SMs are done first.  A stage costs 2.5 cycles a row and number of x (the loads of
// x; its products 2), 280 at the least (the weights' decoding), a tile 1000 besides.  2048 x 1024 to 1000 of fp32 takes 21.2 us with 64 rows, two
// rounds of 148 tiles, and 24.9 with 96, two as well; 17 rows of bf16, 1024 to 50000, 16.7 with 32 and 38 with 128.
template <int P>
int rows_of_tile(int64_t rows, int64_t outputs, int64_t k_blocks, int sms) {
  const int64_t m_blocks = (outputs + kTileM - 1) / kTileM;
  int best = 32;
  int64_t least = 0;
  for (int bn = 32; bn <= kMostRows<P>; bn += 32) {  // (of equal ones the smallest: rows that are not there are read as zeros)
    const int64_t tiles = m_blocks * ((rows + bn - 1) / bn), rounds = (tiles + sms - 1) / sms;
    const int64_t cycles = rounds * (k_blocks * std::max<int64_t>(280, 5 * P * bn / 2) + 1000);
    if (least == 0 || cycles < least) best = bn, least = cycles;
  }
  return best;
}

template <typename T, int P>
int launch_tiles(const dense::Matrix &x, const void *codes, const uint8_t *scales, const T *bias, T *y, int64_t rows, int64_t features, int64_t outputs,
                 uint32_t *status_word, int sms, cudaStream_t stream) {
  TileArgs a = {};
  a.bn = rows_of_tile<P>(rows, outputs, (features + kTileK - 1) / kTileK, sms);
  if (!dense::encode_matrix_16(&a.x, x, a.bn) || !encode_codes(&a.codes, codes, outputs, blocks_of(features))) return HT_ERR_UNSUPPORTED;
  a.scales = scales;
  a.status_word = status_word;
  a.rows = (int)rows, a.outputs = (int)outputs, a.blocks = (int)blocks_of(features), a.k = (int)features;
  const int64_t m_blocks = (outputs + kTileM - 1) / kTileM, n_blocks = (rows + a.bn - 1) / a.bn;
  if (m_blocks * n_blocks > 0x3fffffff) return HT_ERR_UNSUPPORTED;
  a.m_blocks = (int)m_blocks, a.n_blocks = (int)n_blocks, a.tiles = (int)(m_blocks * n_blocks);
  a.k_blocks = (int)((features + kTileK - 1) / kTileK);
  a.instruction = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(a.bn >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
  return dense::launch_next<mx4_tile_kernel<T, P>>(dim3((unsigned)std::min(a.tiles, sms)), kTileThreads, kTileBytes<P>, kTileBytes<P>, stream, 1, a, bias, y);
}

}  // namespace mx4
}  // namespace ht

// A class drawn from each row of scores with a given random number, under bounds on the classes that count.
//
//     m = max s      w_i = exp((s_i - m) / T)                     (T = 0: the first class of the largest score)
//     order: larger scores first, of equal ones the lower class.  What counts is a prefix of that order, the shortest of
//       top_k classes;  the least that holds top_p of the weight of the first top_k;  the classes with w_i >= min_p;  never none
//     W = sum of w over what counts;  the class is the first i, in the order of classes, whose sum of w up to it is above u W
//     log_prob = (s_i - m) / T - log W
//
// A border that moves by 1e-8 of W picks another class once in some thousand rows of many classes, so the decisions are those of 64-bit weights
// and sums.  Where many classes are summed that is done in fp32 first, with a bound on what it is off by; where a border is nearer than that, once
// more in 64 bits (EXACT).  That exponential is table-driven (P. T. P. Tang, Table-driven implementation of the exponential function, ACM TOMS 15,
// 1989): 2^(k / 64) from a table and a polynomial of degree 4, 4e-14.
//
// A row belongs to a CTA, or, where there are few rows, to a cluster of up to 8 that have a part each; it stays in shared memory where it fits.  A
// prefix of the order is held as its last class, (score, class).  To find it nothing is sorted but a list of up to 1024 classes around the place:
//   top_k   up to 200: every thread has the maxima of 4 parts of what it has read; the one of about place k among those, found by halving the
//           range, bounds the k-th largest score from below, and not many more classes than k are above it
//   top_p   the same with the first 192 classes, where those hold enough
//   else    classes are counted, or their weights summed, by 2048 ranges of the score or of its bits; the ranges that the place may be in are listed, or
//           divided again, or are one score
// What counts of a list is drawn from there; otherwise the row is summed in order, warp by warp, and one warp walks its part.
// CTAs of a cluster exchange sums, counts, ranges and lists through each other's shared memory and all come to the same decisions.  No sum depends on
// the order of atomic additions: the same call gives the same bits.
#include "ht_dense.cuh"

#include <math_constants.h>

#include <cstddef>

namespace ht {
namespace sample {
namespace {

using dense::after_previous_kernel;
using dense::load_plain;
using dense::to_float;
using tile::smem_addr;

constexpr int kMostWarps = 32, kMostCtas = 8, kList = 1024, kBins = 2048, kParts = 4, kCounted = 256;
constexpr uint32_t kFirst = 192;     // classes that are listed first for top_p
constexpr uint32_t kListed = 200;   // top_k up to which the classes are listed: what is sorted by counting, a little more at the most
constexpr double kTail = -80.0;      // whatever the classes below exp() of this are, they do not weigh 2^-53 of the row together
constexpr int kPassed = 0x7fffffff;  // no limit on the class among equal scores

struct Args {
  const void *scores;
  int64_t rows, stride;
  int classes;
  const float *uniform;
  double temperature, factor, top_p, min_p;  // factor: 64 / (T ln 2)
  int64_t top_k;
  const float *row_temperature, *row_top_p, *row_min_p;
  const int64_t *row_top_k;
  int64_t *drawn;
  float *log_probs;
  uint32_t row_bytes;  // of shared memory for a row, or a CTA's part of it
};

// 2^(k / 64), rounded to nearest; copied 16 bytes at a time.
struct alignas(16) Powers {
  double of[64];
};
__device__ const Powers kPowers = {{
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
}};

// Larger for larger scores; both zeros are one score.
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s + 0.0f);
  return (b & 0x80000000u) != 0u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0u ? key & 0x7fffffffu : ~key); }

struct alignas(16) Shared {
  double table[64];
  double sums[2][kMostWarps][2];
  uint32_t words[2][kMostWarps], lows[2][kMostWarps];
  double cta_sums[2][kMostCtas][2];
  uint32_t cta_words[2][kMostCtas], cta_lows[2][kMostCtas];
  uint32_t count, bin[2];
  uint32_t ranks[kCounted];
  union {
    uint64_t list[kList];
    uint32_t bins[kBins];
  };
};
constexpr size_t kRowAt = (sizeof(Shared) + 127) / 128 * 128;
constexpr size_t kMergedBytes = sizeof(uint64_t) * kList;  // of a cluster's list in each of its CTAs, behind that

constexpr double kStepOf = 0.69314718055994531 / 64.0;  // ln 2 / 64

// w = exp((s - m) / T) as 2^(a / 64) with a = (s - m) 64 / (T ln 2).
struct Weight {
  double m, c;
  const double *table;
  float m_, c_;  // of the rough one
  __device__ __forceinline__ double operator()(float s) const {
    const double a = ((double)s - m) * c;
    constexpr double kStep = kStepOf;
    if (!(a > -746.0 / kStep)) return 0.0;
    constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52: what is added to it is rounded to a whole number, in the low bits
    const double t = a + kWhole, r = a - (t - kWhole);
    const int k = __double2loint(t), power = k >> 6;
    const double f = r * kStep;
    const double p = f * fma(f, fma(f, fma(f, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0);
    const double e = table[k & 63];
    const double v = fma(e, p, e);
    if (power < -1000) return __hiloint2double(__double2hiint(v) + ((power + 100) << 20), __double2loint(v)) * 0x1p-100;  // perhaps subnormal
    return __hiloint2double(__double2hiint(v) + (power << 20), __double2loint(v));
  }
  // 2^y with y = (s - m) / (T ln 2) in fp32, off by kOff + |y| kOffPower of itself: the hardware's exponential 2^-22, the sum of a vector of them 3 2^-24;
  // difference, factor and product 2^-24 of y each.
  static constexpr double kOff = 4.3e-7, kOffPower = 1.25e-7;
  __device__ __forceinline__ float rough(float s, float &y) const {
    y = fmaxf((s - m_) * c_, -200.0f);  // (2^-200 is 0)
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
  }
};

// The logarithm of what counts: fp32's, and a step of Newton's method with the exponential above, log x = y + (x exp(-y) - 1), which leaves the
// square of its error.  (The 64-bit function took longer than the sums of a row.)
__device__ __forceinline__ double log_of(double x, const double *table) {
  const float y = logf((float)x);
  const Weight w = {0.0, 64.0 * 1.4426950408889634, table, 0.0f, 0.0f};
  return (double)y + fma(x, w(-y), -1.0);
}

// The last class of a prefix of the order.
struct Last {
  float score;
  int at;
  __device__ __forceinline__ bool holds(float s, int i) const { return s > score || (s == score && i <= at); }
};

// A sum and what it may be off by.
struct Sum {
  double value, off;
};

template <typename T>
struct Row {
  static constexpr int kPer = 16 / (int)sizeof(T);
  const T *base;         // where the row's first 16 bytes start in memory
  unsigned char *shared; // vector `first` in shared memory, or null
  int head, classes, vectors, first;
  // Class j kPer - head + i is number i of vector j.
  __device__ __forceinline__ uint4 from_memory(int j) const {
    const int c = j * kPer - head;
    if (c >= 0 && c + kPer <= classes) return load_plain(reinterpret_cast<const uint4 *>(base) + j);
    T t[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) t[i] = c + i >= 0 && c + i < classes ? base[j * (int64_t)kPer + i] : dense::from_float<T>(-CUDART_INF_F);
    return *reinterpret_cast<const uint4 *>(t);
  }
  __device__ __forceinline__ uint4 words(int j) const { return shared != nullptr ? reinterpret_cast<const uint4 *>(shared)[j - first] : from_memory(j); }
  __device__ __forceinline__ void values(int j, float (&v)[kPer]) const {
    T t[kPer];
    *reinterpret_cast<uint4 *>(t) = words(j);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = to_float(t[i]);
  }
};

// The largest scores of 4 parts of what a thread reads, no number where there is one among them, and the least of all, word by word.
template <typename T>
struct Extremes {
  uint32_t top[kParts], low;
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (sizeof(T) == 4)
      asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (std::is_same<T, __half>::value)
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static uint32_t smaller(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (sizeof(T) == 4)
      asm("min.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (std::is_same<T, __half>::value)
      asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static constexpr uint32_t kInfinity = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  static constexpr uint32_t kSigns = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
  __device__ __forceinline__ Extremes() : top{kInfinity | kSigns, kInfinity | kSigns, kInfinity | kSigns, kInfinity | kSigns}, low(kInfinity) {}
  // (an end of the row holds what is no class of it: of those the least are no matter)
  __device__ __forceinline__ void add(const uint4 &q, bool end) {
    top[0] = larger(top[0], q.x), top[1] = larger(top[1], q.y), top[2] = larger(top[2], q.z), top[3] = larger(top[3], q.w);
    if (!end) low = smaller(smaller(low, smaller(q.x, q.y)), smaller(q.z, q.w));
  }
  __device__ __forceinline__ float least(float (&part_max)[kParts]) const {
    constexpr int kIn = 4 / (int)sizeof(T);
    T t[kIn];
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      *reinterpret_cast<uint32_t *>(t) = top[i];
      part_max[i] = to_float(t[0]);
      if (kIn == 2) asm("max.NaN.f32 %0, %1, %2;" : "=f"(part_max[i]) : "f"(part_max[i]), "f"(to_float(t[kIn - 1])));
    }
    *reinterpret_cast<uint32_t *>(t) = low;
    return fminf(to_float(t[0]), to_float(t[kIn - 1]));
  }
};

template <typename T, int C>
struct Team {  // C CTAs at work on a row
  static constexpr int kPer = Row<T>::kPer;
  Shared &sh;
  uint64_t *merged;  // the list of all CTAs
  Row<T> row;
  int lane, warp, warps, rank, first, last;  // of this warp: vectors first .. last - 1
  uint32_t turn = 0, far_turn = 0;  // of the buffers that reductions use one after the other, in a CTA and between them

  // What follows has seen what all threads of the team did before.
  __device__ __forceinline__ void meet() const {
    if constexpr (C > 1) {
      __syncwarp();
      dense::cluster_sync();
    } else
      __syncthreads();
  }
  template <typename V>
  __device__ __forceinline__ V *of_cta(V *p, int r) const {
    if constexpr (C == 1) return p;
    uint64_t to;
    asm("mapa.u64 %0, %1, %2;" : "=l"(to) : "l"(p), "r"(r));
    return reinterpret_cast<V *>(to);
  }

  // f(values, class of the first) for every vector of this warp's part of the row.
  template <typename F>
  __device__ __forceinline__ void each_vector(F &&f) const {
#pragma unroll 1
    for (int j = first + lane; j < last; j += 32) {
      float v[kPer];
      row.values(j, v);
      f(v, j * kPer - row.head);
    }
  }
  // The same for vectors with a score from `least` on among them.
  template <typename F>
  __device__ __forceinline__ void each_vector_from(float least, F &&f) const {
    if (least == -CUDART_INF_F) {
      each_vector(f);
      return;
    }
#pragma unroll 2
    for (int j = first + lane; j < last; j += 32) {
      const uint4 q = row.words(j);
      const uint32_t top = Extremes<T>::larger(Extremes<T>::larger(q.x, q.y), Extremes<T>::larger(q.z, q.w));
      T t[kPer];
      *reinterpret_cast<uint32_t *>(t) = top;
      if (!(fmaxf(to_float(t[0]), to_float(t[4 / (int)sizeof(T) - 1])) >= least)) continue;
      *reinterpret_cast<uint4 *>(t) = q;
      float v[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = to_float(t[i]);
      f(v, j * kPer - row.head);
    }
  }
  // f(score, class) for every class, or for those of such vectors.
  template <typename F>
  __device__ __forceinline__ void each_from(float least, F &&f) const {
    each_vector_from(least, [&](const float (&v)[kPer], int c) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) f(v[i], c + i);
    });
  }
  template <typename F>
  __device__ __forceinline__ void each(F &&f) const {
    each_vector([&](const float (&v)[kPer], int c) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) f(v[i], c + i);
    });
  }
  // Both numbers of all threads, summed, to all of them.
  __device__ __forceinline__ void reduce(double &a, double &b) {
    auto in_warp = [&](double &v) {
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    };
    in_warp(a), in_warp(b);
    if (lane == 0) sh.sums[turn][warp][0] = a, sh.sums[turn][warp][1] = b;
    __syncthreads();
    a = lane < warps ? sh.sums[turn][lane][0] : 0.0;
    b = lane < warps ? sh.sums[turn][lane][1] : 0.0;
    in_warp(a), in_warp(b);
    if constexpr (C > 1) {
      if (warp == 0 && lane < C) {
        double *to = of_cta(&sh.cta_sums[far_turn][rank][0], lane);
        to[0] = a, to[1] = b;
      }
      meet();
      a = sh.cta_sums[far_turn][0][0], b = sh.cta_sums[far_turn][0][1];
#pragma unroll
      for (int r = 1; r < C; ++r) a += sh.cta_sums[far_turn][r][0], b += sh.cta_sums[far_turn][r][1];
      far_turn ^= 1u;
    }
    turn ^= 1u;
  }
  // The largest and the least of all threads' numbers.
  __device__ __forceinline__ void range(uint32_t &top, uint32_t &low) {
    auto in_warp = [&]() { top = __reduce_max_sync(0xffffffffu, top), low = __reduce_min_sync(0xffffffffu, low); };
    in_warp();
    if (lane == 0) sh.words[turn][warp] = top, sh.lows[turn][warp] = low;
    __syncthreads();
    top = lane < warps ? sh.words[turn][lane] : 0u;
    low = lane < warps ? sh.lows[turn][lane] : 0xffffffffu;
    in_warp();
    if constexpr (C > 1) {
      if (warp == 0 && lane < C) *of_cta(&sh.cta_words[far_turn][rank], lane) = top, *of_cta(&sh.cta_lows[far_turn][rank], lane) = low;
      meet();
      top = lane < C ? sh.cta_words[far_turn][lane] : 0u;
      low = lane < C ? sh.cta_lows[far_turn][lane] : 0xffffffffu;
      in_warp();
      far_turn ^= 1u;
    }
    turn ^= 1u;
  }
  __device__ __forceinline__ double sum(double v) {
    double none = 0.0;
    reduce(v, none);
    return v;
  }
  // The least, or the sum, of all threads' numbers; of the CTA's alone with `alone`.
  template <bool LEAST>
  __device__ __forceinline__ uint32_t words(uint32_t v, bool alone = false) {
    auto in_warp = [](uint32_t x) { return LEAST ? __reduce_min_sync(0xffffffffu, x) : __reduce_add_sync(0xffffffffu, x); };
    v = in_warp(v);
    if (lane == 0) sh.words[turn][warp] = v;
    __syncthreads();
    v = in_warp(lane < warps ? sh.words[turn][lane] : LEAST ? 0xffffffffu : 0u);
    if (C > 1 && !alone) {
      if (warp == 0 && lane < C) *of_cta(&sh.cta_words[far_turn][rank], lane) = v;
      meet();
      v = in_warp(lane < C ? sh.cta_words[far_turn][lane] : LEAST ? 0xffffffffu : 0u);
      far_turn ^= 1u;
    }
    turn ^= 1u;
    return v;
  }

  // Both numbers of the CTA's threads, summed.
  __device__ __forceinline__ void counts(uint32_t &a, uint32_t &b) {
    a = __reduce_add_sync(0xffffffffu, a), b = __reduce_add_sync(0xffffffffu, b);
    if (lane == 0) sh.words[turn][warp] = a, sh.lows[turn][warp] = b;
    __syncthreads();
    a = __reduce_add_sync(0xffffffffu, lane < warps ? sh.words[turn][lane] : 0u);
    b = __reduce_add_sync(0xffffffffu, lane < warps ? sh.lows[turn][lane] : 0u);
    turn ^= 1u;
  }

  // What a prefix weighs.
  __device__ __forceinline__ Sum weigh(const Weight &w, const Last &end, bool exact) {
    double value = 0.0, powers = 0.0;
    if (exact) {
      each_from(end.score, [&](float s, int i) {
        if (end.holds(s, i)) value += w(s);
      });
      return {sum(value), 0.0};
    }
    value = rough_sum(w, end, powers);
    reduce(value, powers);
    return {value, 1.01 * (Weight::kOff * value + Weight::kOffPower * powers)};
  }
  // This thread's part of that; powers: the sum of w |y|.
  __device__ __forceinline__ double rough_sum(const Weight &w, const Last &end, double &powers) const {
    double value = 0.0;
    float of_powers = 0.0f;
    auto vector = [&](const float (&v)[kPer]) {
      float e[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float y;
        e[i] = w.rough(v[i], y);
        of_powers = fmaf(e[i], -y, of_powers);
      }
#pragma unroll
      for (int d = kPer / 2; d >= 1; d /= 2)
#pragma unroll
        for (int i = 0; i < d; ++i) e[i] += e[i + d];
      value += (double)e[0];
    };
    if (end.score == -CUDART_INF_F) {
      each_vector([&](const float (&v)[kPer], int) { vector(v); });
    } else {
      each_vector_from(end.score, [&](const float (&v)[kPer], int c) {
        float held[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) held[i] = end.holds(v[i], c + i) ? v[i] : -CUDART_INF_F;
        vector(held);
      });
    }
    powers = (double)of_powers;
    return value;
  }

  // Lists the classes that `visit` adds, as many as fit, and gives their number; in `merged` for all CTAs.
  template <typename F>
  __device__ __forceinline__ uint32_t list(F &&visit) {
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    visit([&](float s, int i) {
      const uint32_t at = atomicAdd(&sh.count, 1u);
      if (at < (uint32_t)kList) sh.list[at] = (uint64_t)key_of(s) << 32 | (0xffffffffu - (uint32_t)i);
    });
    __syncthreads();
    uint32_t n = sh.count;
    if constexpr (C > 1) {
      if (warp == 0 && lane < C) *of_cta(&sh.cta_words[far_turn][rank], lane) = n;
      meet();
      n = 0;
      for (int r = 0; r < C; ++r) n += sh.cta_words[far_turn][r];
      if (n <= (uint32_t)kList) {
        uint32_t at = 0;
        for (int r = 0; r < C; ++r) {
          const uint32_t of_r = sh.cta_words[far_turn][r];
          const uint64_t *from = of_cta(sh.list, r);
          for (uint32_t i = threadIdx.x; i < of_r; i += blockDim.x) merged[at + i] = from[i];
          at += of_r;
        }
      }
      far_turn ^= 1u;
      meet();
    }
    return n;
  }
  // Sorts the list, the largest first: by counting what is larger, or bitonic with as many places as the next power of two.
  __device__ __forceinline__ void sort(int n) {
    int places = 32;
    while (places < n) places *= 2;
    if (places <= kCounted && places <= (int)blockDim.x) {
      const int e = (int)threadIdx.x & (places - 1), part = (int)threadIdx.x / places, parts = (int)blockDim.x / places;
      if ((int)threadIdx.x < places) sh.ranks[threadIdx.x] = 0;
      __syncthreads();
      const uint64_t own = e < n ? merged[e] : 0;
      uint32_t larger = 0;
      if (part < parts)
        for (int i = part; i < n; i += parts) larger += merged[i] > own ? 1u : 0u;
      if (e < n && larger > 0u) atomicAdd(&sh.ranks[e], larger);
      __syncthreads();
      if (part == 0 && e < n) merged[sh.ranks[e]] = own;
      __syncthreads();
      return;
    }
    for (int i = n + (int)threadIdx.x; i < places; i += (int)blockDim.x) merged[i] = 0;
    __syncthreads();
    for (int size = 2; size <= places; size *= 2)
      for (int d = size / 2; d >= 1; d /= 2) {
        for (int i = (int)threadIdx.x; i < places / 2; i += (int)blockDim.x) {
          const int a = 2 * i - (i & (d - 1)), b = a + d;
          const uint64_t x = merged[a], y = merged[b];
          if ((x < y) == ((a & size) == 0)) merged[a] = y, merged[b] = x;
        }
        __syncthreads();
      }
  }
  __device__ __forceinline__ Last listed(int i) const {
    const uint64_t e = merged[i];
    return {score_of((uint32_t)(e >> 32)), (int)(0xffffffffu - (uint32_t)e)};
  }
  // weight(i) for the list's first n, summed in order: this thread's neighbours from .. to - 1 and what is ahead of them; gives the whole.
  template <typename F>
  __device__ __forceinline__ double scan(int n, F &&weight, int &from, int &to, double &ahead, double *mine = nullptr) {
    const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;  // kList / threads at the most
    from = min((int)threadIdx.x * per, n), to = min(from + per, n);
    double own = 0.0;
    for (int i = from; i < to; ++i) own += weight(i);
    double upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += t;
    }
    if (lane == 31) sh.sums[turn][warp][0] = upto;
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int i = 0; i < warps; ++i) {
      if (i == warp) before = all;
      all += sh.sums[turn][i][0];
    }
    turn ^= 1u;
    ahead = before + (upto - own);
    if (mine != nullptr) *mine = own;
    return all;
  }
  // Of the sorted list's first n, with `before` of weight ahead of them: how many start below `target`, whose own error is `off`: -1 where that
  // makes a difference.
  __device__ __forceinline__ int places_below(int n, const Weight &w, double before, double target, double off, double *whole = nullptr) {
    int from, to;
    double at;
    const double all = scan(n, [&](int i) { return w(listed(i).score); }, from, to, at);
    if (whole != nullptr) *whole = all;
    at += before;
    uint32_t count = 0;
    for (int i = from; i < to; ++i) {
      count += (at < target - off ? 1u : 0u) + (at < target + off ? 0x10000u : 0u);
      at += w(listed(i).score);
    }
    count = words<false>(count, true);
    return (count & 0xffffu) == count >> 16 ? (int)(count >> 16) : -1;
  }

  // The class of the n-th (from 1) of those with this score, in the order of classes.
  __device__ __forceinline__ int nth_of(float score, uint32_t n) {
    uint32_t own = 0;
    each_from(score, [&](float s, int) { own += s == score ? 1u : 0u; });
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) sh.words[turn][warp] = own;
    __syncthreads();
    uint32_t ahead = 0, of_cta_all = 0;
    for (int i = 0; i < warps; ++i) {
      if (i == warp) ahead = of_cta_all;
      of_cta_all += sh.words[turn][i];
    }
    if constexpr (C > 1) {
      if (warp == 0 && lane < C) *of_cta(&sh.cta_words[far_turn][rank], lane) = of_cta_all;
      meet();
      for (int r = 0; r < rank; ++r) ahead += sh.cta_words[far_turn][r];
      far_turn ^= 1u;
    }
    turn ^= 1u;
    uint32_t found = 0xffffffffu;
    if (ahead < n && n <= ahead + own) {
      for (int j0 = first; j0 < last; j0 += 32) {
        const int j = j0 + lane;
        float v[kPer];
        uint32_t here = 0;
        if (j < last) {
          row.values(j, v);
#pragma unroll
          for (int i = 0; i < kPer; ++i) here += v[i] == score ? 1u : 0u;
        }
        uint32_t upto = here;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t t = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += t;
        }
        uint32_t at = ahead + upto - here;
        if (at < n && n <= at + here) {
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (v[i] == score && ++at == n) found = (uint32_t)(j * kPer - row.head + i);
        }
        ahead += __shfl_sync(0xffffffffu, upto, 31);
        if (ahead >= n) break;
      }
    }
    return (int)words<true>(found);
  }

  // The last class of the shortest prefix that reaches `target`, counted (WEIGHTS false) or weighed, among the classes that `base` holds and
  // whose keys are in [low, high]; all others of base are above, or weigh too little to matter.  For weights `all` is what base weighs; `off` is
  // target's error, and *sure is false, whatever comes back, where that or what is summed roughly makes a difference (never with EXACT: then all
  // that is weighed or counted in units is, in 64 bits); a target is `share` of what base weighs.  Two pieces of code, so that rows of rough weights carry
  // none of the other's (4096 rows of 21841 with wide nuclei 781 us; 917 with the choice at each weight, 793 with the 64-bit one as a call).
  template <bool WEIGHTS, bool EXACT>
  __device__ __forceinline__ Last narrow(const Weight &w, const Last &base, uint32_t low, uint32_t high, double target, double off, double all, double share, bool *sure) {
    double above = 0.0;
    uint32_t classes = (uint32_t)row.classes;  // in [low, high], at the most
    bool by_score = true, split_by_score = true, more_below = false;
    for (;;) {
      // By ranges, highest first: of the score at first, over which scores are spread more evenly, then of its key, and so on in turn.  Weights
      // are counted in units of 2^-31 of what is in [low, high], so that a count is below 2^32 with half a unit more for each of 2^30 classes.
      const uint32_t width = high - low;
      const int shift = max(0, 21 - (int)__clz((int)width));
      const float low_score = score_of(low), high_score = score_of(high);
      const float slope = by_score ? ((float)kBins - 1.0f) / (high_score - low_score) : 0.0f;
      const uint32_t last_bin = by_score ? (uint32_t)kBins - 1u : width >> shift;
      auto inside = [&](float s, int i) { return s >= low_score && s <= high_score && (s != base.score || i <= base.at); };
      auto range_of = [&](float s) { return by_score ? min((uint32_t)((high_score - s) * slope), last_bin) : (high - key_of(s)) >> shift; };
      const double scale = fmin(2147483648.0 / all, 1e30);  // (as fp32 as well)
      const float scale_ = (float)scale;
      meet();
      for (int i = (int)threadIdx.x; i < kBins; i += (int)blockDim.x) sh.bins[i] = 0;
      __syncthreads();
      each_from(low_score, [&](float s, int i) {
        if (inside(s, i)) {
          float y;
          atomicAdd(&sh.bins[range_of(s)], !WEIGHTS ? 1u : EXACT ? (uint32_t)fma(w(s), scale, 0.5) : (uint32_t)fmaf(w.rough(s, y), scale_, 0.5f));
        }
      });
      meet();
      const uint32_t *bins = sh.bins;
      if constexpr (C > 1) {  // of all CTAs together
        uint32_t *const together = reinterpret_cast<uint32_t *>(merged);
        for (int i = (int)threadIdx.x; i < kBins; i += (int)blockDim.x) {
          uint32_t v = 0;
#pragma unroll
          for (int r = 0; r < C; ++r) v += of_cta(sh.bins, r)[i];
          together[i] = v;
        }
        bins = together;
        meet();  // (the CTAs' own have been read: their place is the list's)
      }
      // The ranges between which the sum reaches the target.  Counts are bounds of weights and not weights: each class is off by half a unit, and rough
      // weights by 2^-16 of themselves (|y| is below 116 here).  A sum that is in reach of nothing at all starts with the first range, whose
      // classes may all count 0, and one that is not reached ends with the last.
      uint32_t wanted_low, wanted_high;
      if constexpr (WEIGHTS) {
        const double slack = (EXACT ? 0.0 : 32768.0) + 0.5 * (double)classes + 2.0;
        wanted_low = (uint32_t)fmin(fmax((target - off - above) * scale - slack, 0.0), 4294967295.0);
        wanted_high = (uint32_t)fmin(fmax((target + off - above) * scale + slack, 1.0), 4294967295.0);
      } else {
        wanted_low = wanted_high = (uint32_t)(target - above);
      }
      const int per = kBins / (int)blockDim.x;  // of a thread
      uint32_t own = 0;
      for (int i = 0; i < per; ++i) own += bins[(int)threadIdx.x * per + i];
      uint32_t upto = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += t;
      }
      if (lane == 31) sh.words[turn][warp] = upto;
      if (threadIdx.x == 0) sh.bin[0] = 0, sh.bin[1] = last_bin;
      __syncthreads();
      uint32_t at = upto - own;
      for (int i = 0; i < warp; ++i) at += sh.words[turn][i];
      turn ^= 1u;
      for (int i = 0; i < per; ++i) {
        const uint32_t one = bins[(int)threadIdx.x * per + i];
        if (at < wanted_low && wanted_low <= at + one) sh.bin[0] = (uint32_t)((int)threadIdx.x * per + i);
        if (at < wanted_high && wanted_high <= at + one) sh.bin[1] = (uint32_t)((int)threadIdx.x * per + i);
        at += one;
      }
      __syncthreads();
      const uint32_t end_bin = sh.bin[1], first_bin = min(sh.bin[0], end_bin);
      // The window's ends as scores: the lowest key whose range is below `bin` (a search by 32 places at a time).
      auto key_below = [&](uint32_t bin) {
        uint32_t from = low, to = high + 1u;  // (high is below every key that is not a score's)
        while (from < to) {
          const uint32_t step = (to - from + 31u) / 32u, place = from + (uint32_t)lane * step;
          const uint32_t below = __ballot_sync(0xffffffffu, place < to && range_of(score_of(place)) < bin);  // from some lane on
          const uint32_t first_below = below != 0u ? (uint32_t)__ffs((int)below) - 1u : (to - from + step - 1u) / step;
          if (first_below == 0u) return from;
          const uint32_t next = from + first_below * step;
          from += (first_below - 1u) * step + 1u;
          if (below != 0u) to = next;
        }
        return to;
      };
      const uint32_t key_above = key_below(first_bin), key_inside = key_below(end_bin + 1u);
      const float inside_score = score_of(key_inside);
      const bool some_above = key_above <= high;
      const float above_score = some_above ? score_of(key_above) : CUDART_INF_F;  // from here on: above the window
      double over = 0.0, powers = 0.0, within = 0.0;  // what is above the window weighs, and the window
      uint32_t least_key = 0xffffffffu, least_gap = 0xffffffffu;  // of the window: its keys reach from `lowest` to `highest`
      float of_powers = 0.0f;
      const bool limited = base.score > -CUDART_INF_F;
      const uint32_t n = list([&](auto &&add) {
        each_vector_from(inside_score, [&](const float (&v)[kPer], int c) {
          float e[kPer];
          bool some = false;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const bool up = v[i] >= above_score && v[i] <= high_score && (!limited || v[i] != base.score || c + i <= base.at);
            if (!WEIGHTS) {
              e[i] = up ? 1.0f : 0.0f;
            } else if (EXACT) {
              e[i] = 0.0f;
              if (up) over += w(v[i]);
            } else {
              float y;
              e[i] = w.rough(up ? v[i] : -CUDART_INF_F, y);
              of_powers = fmaf(e[i], -y, of_powers);
            }
            some |= v[i] >= inside_score && v[i] < above_score;
          }
#pragma unroll
          for (int d = kPer / 2; d >= 1; d /= 2)
#pragma unroll
            for (int i = 0; i < d; ++i) e[i] += e[i + d];
          over += (double)e[0];
          if (some) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
              if (v[i] >= inside_score && v[i] < above_score && inside(v[i], c + i)) {
                const uint32_t key = key_of(v[i]);
                least_key = min(least_key, key), least_gap = min(least_gap, 0xffffffffu - key);
                if (WEIGHTS) {
                  float y;
                  within += EXACT ? w(v[i]) : (double)w.rough(v[i], y);
                }
                add(v[i], c + i);
              }
          }
        });
      });
      powers = (double)of_powers;
      reduce(over, powers);
      if (WEIGHTS && !EXACT) off += 1.01 * (Weight::kOff * over + Weight::kOffPower * powers);
      over += above;
      if (WEIGHTS && over >= target - off) *sure = false;
      more_below |= key_inside > low;
      if (n == 0u) return {low_score, low_score == base.score ? base.at : kPassed};
      if (n <= (uint32_t)kList) {
        sort((int)n);
        int places;
        if (WEIGHTS) {
          double weight;
          places = places_below((int)n, w, over, target, off, &weight);
          if (!EXACT && (places < 0 || !*sure || (over + weight < target + off && more_below))) {  // once more, what is above and what there is in 64 bits
            double whole = 0.0;
            over = 0.0;
            each_from(base.score, [&](float s, int i) {
              if (!base.holds(s, i)) return;
              const double one = w(s);
              whole += one;
              over += s > high_score || (s >= above_score && s <= high_score) ? one : 0.0;
            });
            reduce(whole, over);
            target = share * whole;
            *sure = over < target && (over + weight >= target || !more_below);
            places = places_below((int)n, w, over, target, 0.0);
          }
        } else {
          places = (int)(target - over);
        }
        return listed(max(min(places, (int)n), 1) - 1);
      }
      const uint32_t lowest = words<true>(least_key), highest = 0xffffffffu - words<true>(least_gap);
      if (lowest == highest) {  // more of one score than the list holds
        const float s = score_of(lowest);
        const double one = WEIGHTS ? w(s) : 1.0, missing = target - over;
        auto places = [&](double left) { return one * n <= left ? n : (uint32_t)fmax(ceil(left / one), 1.0); };
        if (WEIGHTS && (places(missing - off) != places(missing + off) || (over + one * n < target + off && more_below))) *sure = false;
        // (among those that base holds the first ones are the first ones of all)
        return {s, nth_of(s, places(missing))};
      }
      low = lowest, high = highest;
      above = over;
      classes = n;
      if constexpr (WEIGHTS) {
        const bool wide = first_bin == 0u && end_bin == last_bin;  // the counts tell nothing
        if (!EXACT && (wide || !*sure)) {
          *sure = false;
          return {low_score, kPassed};
        }
        all = sum(within) * (EXACT ? 1.0 : 1.0 + 0x1p-15);
        if (EXACT && wide) {  // one class may weigh all of the units: half of the scores, or of their keys in turn, by what they weigh
          uint32_t middle = low + (high - low) / 2u;
          if (split_by_score) middle = min(max(key_of(0.5f * score_of(low) + 0.5f * score_of(high)), low), high - 1u);
          split_by_score = !split_by_score;
          const float middle_score = score_of(middle), lowest_score = score_of(low);
          double upper = 0.0, lower = 0.0;
          uint32_t uppers = 0, above_middle = 0xffffffffu, below_middle = 0xffffffffu;
          each_from(lowest_score, [&](float s, int i) {
            if (!(s >= lowest_score) || !inside(s, i) || key_of(s) > high) return;
            const uint32_t key = key_of(s);
            if (s > middle_score)
              upper += w(s), ++uppers, above_middle = min(above_middle, key);
            else
              lower += w(s), below_middle = min(below_middle, 0xffffffffu - key);
          });
          reduce(upper, lower);
          uppers = words<false>(uppers), above_middle = words<true>(above_middle), below_middle = 0xffffffffu - words<true>(below_middle);
          if (above + upper < target) {
            above += upper, high = below_middle, all = lower, classes -= uppers;
          } else {
            low = above_middle, all = upper, classes = uppers, more_below = true;
          }
          by_score = true;
          continue;
        }
      }
      by_score = !by_score;
    }
  }
};

template <typename T, int C>
__global__ void __launch_bounds__(32 * kMostWarps) sample_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char sample_smem[];
  Shared &sh = *reinterpret_cast<Shared *>(sample_smem);
  constexpr int kPer = Row<T>::kPer;
  after_previous_kernel();
  const int64_t r = blockIdx.x / C;
  const T *from = static_cast<const T *>(a.scores) + r * a.stride;
  Row<T> row;
  row.head = (int)((reinterpret_cast<uintptr_t>(from) & 15u) / sizeof(T));
  row.base = from - row.head;
  row.classes = a.classes;
  row.vectors = (int)(((int64_t)row.head + a.classes + kPer - 1) / kPer);
  row.shared = nullptr;
  const int warps = (int)blockDim.x / 32, warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int rank = C > 1 ? (int)(blockIdx.x % C) : 0;
  const int part = (row.vectors + C * warps - 1) / (C * warps), ordinal = rank * warps + warp;
  row.first = min(rank * warps * part, row.vectors);
  Team<T, C> team = {sh, C > 1 ? reinterpret_cast<uint64_t *>(sample_smem + kRowAt) : sh.list, row, lane, warp, warps, rank, min(ordinal * part, row.vectors),
                     min((ordinal + 1) * part, row.vectors)};

  // the row into shared memory, and its largest and least score
  if (a.row_bytes > 0) {
    unsigned char *const to = sample_smem + kRowAt + (C > 1 ? kMergedBytes : 0);
    for (int j = team.first + lane; j < team.last; j += 32) {
      const int first = j * kPer - row.head;
      if (first >= 0 && first + kPer <= a.classes)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to) + 16u * (uint32_t)(j - row.first)),
                     "l"(reinterpret_cast<const uint4 *>(row.base) + j)
                     : "memory");
      else
        reinterpret_cast<uint4 *>(to)[j - row.first] = row.from_memory(j);
    }
    team.row.shared = to;
  }
  static_assert(alignof(Powers) >= 16 && alignof(Shared) >= 16 && offsetof(Shared, table) % 16 == 0, "16 bytes are copied from and to here");
  if (threadIdx.x < 32)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_addr(sh.table) + 16u * threadIdx.x), "l"(kPowers.of + 2 * threadIdx.x) : "memory");
  const double temperature = a.row_temperature != nullptr ? (double)load_plain(a.row_temperature + r) : a.temperature;
  const double top_p = a.row_top_p != nullptr ? (double)load_plain(a.row_top_p + r) : a.top_p;
  const double min_p = a.row_min_p != nullptr ? (double)load_plain(a.row_min_p + r) : a.min_p;
  const int64_t asked = a.row_top_k != nullptr ? load_plain(a.row_top_k + r) : a.top_k;
  const double u = (double)load_plain(a.uniform + r);
  const int top_k = asked > 0 && asked < a.classes ? (int)asked : a.classes;
  asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (C > 1) team.meet();  // every CTA is there before another one writes to it

  // (no lane reads another's part of the row; the table comes before the first barrier)
  float part_max[kParts];
  Extremes<T> extremes;
#pragma unroll 1
  for (int j = team.first + lane; j < team.last; j += 32) extremes.add(team.row.words(j), j == 0 || j == row.vectors - 1);
  float low_ = extremes.least(part_max);
  for (int j = 0; j < row.vectors; j = j == 0 && row.vectors > 1 ? row.vectors - 1 : row.vectors) {  // the ends
    if (j < team.first || j >= team.last || (j - team.first) % 32 != lane) continue;
    float v[kPer];
    team.row.values(j, v);
#pragma unroll
    for (int i = 0; i < kPer; ++i) low_ = fminf(low_, v[i] > -CUDART_INF_F ? v[i] : CUDART_INF_F);
  }
  // (no number where one of them is none)
  const float own_top = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
  const bool number = part_max[0] == part_max[0] && part_max[1] == part_max[1] && part_max[2] == part_max[2] && part_max[3] == part_max[3];
  uint32_t top_key = number ? key_of(own_top) : 0xffffffffu, low_key_ = key_of(low_);
  team.range(top_key, low_key_);
  const float m = top_key == 0xffffffffu ? CUDART_INF_F : score_of(top_key);
  const bool bounds = temperature >= 0.0 && temperature < CUDART_INF && top_p == top_p && min_p == min_p && u >= 0.0 && u <= 1.0;
  auto answer = [&](int64_t drawn, float log_prob) { a.drawn[r] = drawn, a.log_probs[r] = log_prob; };
  // (a CTA of a cluster leaves when no other one reads from it any more)
  if (!bounds || !(m > -CUDART_INF_F && m < CUDART_INF_F)) {
    if (rank == 0 && threadIdx.x == 0) answer(-1, CUDART_NAN_F);
    if constexpr (C > 1) team.meet();
    return;
  }
  if (temperature == 0.0 || top_k == 1 || top_p <= 0.0 || min_p > 1.0) {
    uint32_t at = 0xffffffffu;
    team.each_from(m, [&](float s, int i) {
      if (s == m) at = min(at, (uint32_t)i);
    });
    at = team.template words<true>(at);
    if (rank == 0 && threadIdx.x == 0) answer((int64_t)at, 0.0f);
    if constexpr (C > 1) team.meet();
    return;
  }
  float low = score_of(low_key_);  // the least finite score
  if (low == -CUDART_INF_F && (top_k < a.classes || top_p < 1.0)) {
    float least = CUDART_INF_F;
    team.each([&](float s, int) { least = fminf(least, s > -CUDART_INF_F ? s : CUDART_INF_F); });
    low = score_of(team.template words<true>(key_of(least)));
  }
  const double factor = a.row_temperature == nullptr ? a.factor : fmin(64.0 * 1.4426950408889634 / temperature, 1e300);
  const Weight w = {(double)m, factor, sh.table, m, (float)fmin(factor / 64.0, 3e38)};

  const bool rough_fails = w.c_ < 1e-37f || w.c_ >= 3e38f;  // a factor that fp32 does not hold

  // what counts: up to `end`, the first `held` of the sorted list where that is above 0
  const double tail = fmax((double)low, (double)m + kTail * temperature);
  const uint32_t high_key = key_of(m), low_key = min(key_of(tail > (double)low ? (float)tail : low), high_key);
  Last end = {-CUDART_INF_F, kPassed};
  int held = 0;
  if (top_k < a.classes || top_p < 1.0) {
    const bool by_count = top_k < a.classes;
    // A lower bound for the score of place `wanted`: at least so many of the parts' maxima are not below it.  Of a cluster each CTA has its share
    // of them and a little more, and what is listed is counted.
    const uint32_t wanted = by_count ? (uint32_t)top_k : kFirst, share = C == 1 ? wanted : wanted / C + wanted / (4 * C) + 8u;
    uint32_t bound = 0;
    if (share <= blockDim.x * kParts) {
      uint32_t keys[kParts], from_key = key_of(low), to_key = high_key;
#pragma unroll
      for (int i = 0; i < kParts; ++i) keys[i] = key_of(part_max[i]);
      // by fifths: the counts of four places at a time, two to a word
      while (from_key < to_key) {
        const uint32_t step = (to_key - from_key) / 5u + 1u;
        uint32_t place[4], n[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          place[q] = min(from_key + (uint32_t)(q + 1) * step, to_key);
#pragma unroll
          for (int i = 0; i < kParts; ++i) n[q / 2] += keys[i] >= place[q] ? 1u << (16 * (q % 2)) : 0u;
        }
        team.counts(n[0], n[1]);
        bool near = false;
        uint32_t to = to_key;
#pragma unroll
        for (int q = 3; q >= 0; --q) {  // the highest place that has enough
          const uint32_t count = (n[q / 2] >> (16 * (q % 2))) & 0xffffu;
          if (count < share) {
            to = place[q] - 1u;
          } else {
            from_key = place[q];
            near = count <= share + share / 8u;
            break;
          }
        }
        to_key = to;
        if (near) break;
      }
      bound = from_key;
      if constexpr (C > 1) bound = 0xffffffffu - team.template words<true>(0xffffffffu - bound);
    }
    const float bound_score = score_of(bound);
    uint32_t n = 0xffffffffu;
    if (bound > 0u && wanted <= kListed)
      n = team.list([&](auto &&add) {
        team.each_from(bound_score, [&](float s, int i) {
          if (s >= bound_score) add(s, i);
        });
      });
    // (whether all is listed that there is, or the list goes as far as place `wanted`)
    const bool whole = bound == key_of(low);
    if (by_count && (n < wanted || (C > 1 && n == 0xffffffffu)) && !whole) n = 0xffffffffu, bound = 0;
    if (n <= (uint32_t)kList) {
      team.sort((int)n);
      held = by_count ? min(top_k, (int)n) : (int)n;
    }
    Sum all = {0.0, 0.0};
    if (by_count && held == 0) {
      const uint32_t from_key = max(bound, key_of(low));
      double inside = 0.0;
      const float from_score = score_of(from_key);
      team.each_from(from_score, [&](float s, int) { inside += s >= from_score ? 1.0 : 0.0; });
      inside = team.sum(inside);
      bool sure = true;
      if (inside >= (double)top_k) end = team.template narrow<false, true>(w, end, from_key, high_key, (double)top_k, 0.0, 1.0, 0.0, &sure);
    }
    if (top_p < 1.0) {
      if (by_count && held > 0) {
        team.places_below(held, w, 0.0, 0.0, 0.0, &all.value);
        held = max(team.places_below(held, w, 0.0, top_p * all.value, 0.0), 1);
      } else {
        bool exact = rough_fails;
        int places = -1;
        for (;;) {
          all = team.weigh(w, end, exact);
          double weight = 0.0;
          if (held > 0) places = team.places_below(held, w, 0.0, top_p * all.value, top_p * all.off, &weight);
          if (held > 0 && weight < top_p * (all.value + all.off) && !whole) held = 0;  // not enough of them, or perhaps not
          if (held > 0 && places >= 0) {
            held = max(places, 1);
            break;
          }
          if (held == 0) {
            bool sure = true;
            // what weighs less than its part of half of 1 - top_p is not held: all of it together is below that half
            const double slight = (double)m + temperature * log(fmax(0.49 * (1.0 - top_p) * all.value / (double)a.classes, 1e-35));
            const uint32_t slight_key = slight > (double)low ? min(key_of(__double2float_rd(slight)), high_key) : low_key;
            const uint32_t from_key = max(max(low_key, slight_key), key_of(end.score));
            const Last last = exact ? team.template narrow<true, true>(w, end, from_key, high_key, top_p * all.value, 0.0, all.value, top_p, &sure)
                                    : team.template narrow<true, false>(w, end, from_key, high_key, top_p * all.value, top_p * all.off, all.value, top_p, &sure);
            if (sure || exact) {
              end = last;
              break;
            }
          }
          exact = true;
        }
      }
    }
  }
  if (min_p > 0.0) {
    const float least = __double2float_ru(fmax((double)m + temperature * log(min_p), -3.4028234663852886e38));  // the lowest score that weighs so much
    if (least > end.score) end = {least, kPassed};
    if (held > 0) {
      uint32_t n = 0;
      for (int i = (int)threadIdx.x; i < held; i += (int)blockDim.x) n += team.listed(i).score >= least ? 1u : 0u;
      held = (int)max(team.template words<false>(n, true), 1u);
    }
  }

  if (held > 0) {  // drawn from the list: in the order of classes
    for (int i = (int)threadIdx.x; i < held; i += (int)blockDim.x) team.merged[i] = team.merged[i] << 32 | team.merged[i] >> 32;
    __syncthreads();
    team.sort(held);
    auto score = [&](int i) { return score_of((uint32_t)team.merged[i]); };
    int first, last;
    double at;
    const double all = team.scan(held, [&](int i) { return w(score(i)); }, first, last, at), target = u * all;
    // the first that passes the target, or the last that weighs anything
    uint32_t passing = 0xffffffffu, some = 0;
    for (int i = first; i < last; ++i) {
      const double one = w(score(i));
      at += one;
      if (one > 0.0) {
        some = (uint32_t)i + 1u;
        if (at > target) passing = min(passing, (uint32_t)i);
      }
    }
    passing = team.template words<true>(passing, true);
    if (passing == 0xffffffffu) passing = 0xffffffffu - team.template words<true>(0xffffffffu - some, true) - 1u;
    if (rank == 0 && threadIdx.x == 0)
      answer((int64_t)(0xffffffffu - (uint32_t)(team.merged[passing] >> 32)), (float)(((double)score((int)passing) - (double)m) * factor * kStepOf - log_of(all, sh.table)));
    if constexpr (C > 1) team.meet();
    return;
  }

  // the sums of the warps' parts, then along one part
  for (bool exact = rough_fails;; exact = true) {
    double own = 0.0, powers = 0.0;
    if (exact)
      team.each_from(end.score, [&](float s, int i) {
        if (end.holds(s, i)) own += w(s);
      });
    else
      own = team.rough_sum(w, end, powers);
    // the warps' parts, one after the other
    const uint32_t turn = team.turn;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) own += __shfl_xor_sync(0xffffffffu, own, d), powers += __shfl_xor_sync(0xffffffffu, powers, d);
    if (lane == 0) sh.sums[turn][warp][0] = own, sh.sums[turn][warp][1] = powers;
    __syncthreads();
    own = lane < warps ? sh.sums[turn][lane][0] : 0.0;
    powers = lane < warps ? sh.sums[turn][lane][1] : 0.0;
    double upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += t;
      powers += __shfl_xor_sync(0xffffffffu, powers, d);
    }
    double all = __shfl_sync(0xffffffffu, upto, 31), ahead = 0.0;
    int at_cta = 0;
    if constexpr (C > 1) {
      if (warp == 0 && lane < C) {
        double *to = team.of_cta(&sh.cta_sums[team.far_turn][rank][0], lane);
        to[0] = all, to[1] = powers;
      }
      team.meet();
      all = powers = 0.0;
#pragma unroll
      for (int i = 0; i < C; ++i) all += sh.cta_sums[team.far_turn][i][0], powers += sh.cta_sums[team.far_turn][i][1];
      at_cta = -1;
      for (int i = 0; i < C; ++i) {  // the first CTA whose part ends above the target, or (u = 1, rounding) the last that weighs anything
        const double s = sh.cta_sums[team.far_turn][i][0];
        if (s > 0.0) {
          if (at_cta >= 0) ahead += sh.cta_sums[team.far_turn][at_cta][0];
          at_cta = i;
          if (ahead + s > u * all) break;
        }
      }
      team.far_turn ^= 1u;
    }
    const double target = u * all;
    team.turn ^= 1u;
    const double off = exact ? 0.0 : 2.02 * (Weight::kOff * all + Weight::kOffPower * powers);  // of a sum and of the target together
    // the place of the first of ascending sums that passes the target, among those that weigh anything, or of the last that does
    auto place_of = [&](bool passes, bool weighs) {
      const uint32_t some = __ballot_sync(0xffffffffu, weighs), passing = __ballot_sync(0xffffffffu, passes) & some;
      return passing != 0u ? __ffs((int)passing) - 1 : 31 - __clz((int)some);
    };
    bool sure = true;
    if (rank == at_cta) {
      const int place = place_of(ahead + upto > target, own > 0.0);
      ahead += __shfl_sync(0xffffffffu, upto - own, place);
      // that part's vectors, the CTA's threads in order
      const int part_first = min((rank * warps + place) * part, row.vectors), part_last = min(part_first + part, row.vectors);
      auto weights_of = [&](int i, float (&v)[kPer], double (&e)[kPer]) {
        team.row.values(part_first + i, v);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          float y;
          const bool held = end.holds(v[q], (part_first + i) * kPer - row.head + q);
          e[q] = !held ? 0.0 : exact ? w(v[q]) : (double)w.rough(v[q], y);
        }
      };
      auto of_vector = [&](int i) {
        float v[kPer];
        if (exact) {
          double e[kPer], sum = 0.0;
          weights_of(i, v, e);
#pragma unroll
          for (int q = 0; q < kPer; ++q) sum += e[q];
          return sum;
        }
        float e[kPer];
        team.row.values(part_first + i, v);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          float y;
          e[q] = w.rough(end.holds(v[q], (part_first + i) * kPer - row.head + q) ? v[q] : -CUDART_INF_F, y);
        }
#pragma unroll
        for (int d = kPer / 2; d >= 1; d /= 2)
#pragma unroll
          for (int q = 0; q < d; ++q) e[q] += e[q + d];
        return (double)e[0];
      };
      int first, last;
      double at, whole;
      team.scan(part_last - part_first, of_vector, first, last, at, &whole);
      at += ahead;
      // the first thread whose sum passes the target, or the last that has any
      const bool passes = whole > 0.0 && at + whole > target;
      uint32_t who = team.template words<true>(passes ? threadIdx.x : 0xffffffffu, true);
      if (who == 0xffffffffu) who = 0xffffffffu - team.template words<true>(0xffffffffu - (whole > 0.0 ? threadIdx.x + 1u : 0u), true) - 1u;
      if (threadIdx.x == who) {
        int found = -1;
        float found_score = 0.0f;
        bool passed = false, near = true;
        for (int i = first; i < last && !passed; ++i) {
          float v[kPer];
          double e[kPer];
          weights_of(i, v, e);
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const double before = at;
            at += e[q];
            if (e[q] > 0.0 && !passed) {
              found = (part_first + i) * kPer - row.head + q, found_score = v[q];
              passed = at > target;
              near = target - before <= off || at - target <= off;
            }
          }
        }
        sure = exact || !near;
        if (sure) answer((int64_t)found, (float)(((double)found_score - (double)m) * factor * kStepOf - log_of(all, sh.table)));
      }
    }
    if (exact) break;
    if (team.template words<true>(sure ? 1u : 0u) != 0u) break;
  }
  if constexpr (C > 1) team.meet();
}

constexpr size_t kMostBytes = 227 * 1024;

int screen(const ht_sample_problem *p) {
  if (p == nullptr || p->rows < 0 || p->classes < 1 || p->stride < p->classes) return HT_ERR_INVALID_ARGUMENT;
  if (p->dtype != HT_DTYPE_F32 && p->dtype != HT_DTYPE_BF16 && p->dtype != HT_DTYPE_F16) return HT_ERR_INVALID_ARGUMENT;
  if (p->row_temperature == nullptr && !(p->temperature >= 0.0 && p->temperature < HUGE_VAL)) return HT_ERR_INVALID_ARGUMENT;
  if ((p->row_top_p == nullptr && !(p->top_p >= 0.0 && p->top_p <= 1.0)) || (p->row_min_p == nullptr && !(p->min_p >= 0.0 && p->min_p <= 1.0)))
    return HT_ERR_INVALID_ARGUMENT;
  if (p->row_top_k == nullptr && p->top_k < 0) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows > 0x7fffff00 || p->classes > 0x3fffff00) return HT_ERR_UNSUPPORTED;
  return HT_OK;
}

template <typename T, int C>
int launch_of(Args a, int64_t vectors, cudaStream_t stream) {
  const int64_t of_cta = (vectors + C - 1) / C;
  // 1024 threads an SM, between the CTAs that it holds: as many as shared memory and the rows admit; two vectors a thread at the least
  const size_t room = kMostBytes / (kRowAt + kMergedBytes + 16 * (size_t)of_cta + 1024);
  const int64_t resident = std::max<int64_t>(1, std::min<int64_t>((int64_t)room, (a.rows * C + 147) / 148));
  int threads = 1024;
  while (threads > 128 && (threads * resident > 1024 || threads * 2 > of_cta)) threads /= 2;
  const int warps = threads / 32;
  const size_t row = 16 * (size_t)((vectors + C * warps - 1) / (C * warps) * warps), before = kRowAt + (C > 1 ? kMergedBytes : 0);
  if (before + row <= kMostBytes) a.row_bytes = (uint32_t)row;
  return dense::launch_next<sample_kernel<T, C>>(dim3((unsigned)(a.rows * C)), threads, before + a.row_bytes, kMostBytes, stream, C, a);
}

template <typename T>
int launch(const ht_sample_problem &p, const void *scores, const float *uniform, int64_t *drawn, float *log_probs, cudaStream_t stream) {
  constexpr int kPer = Row<T>::kPer;
  const double factor = std::min(64.0 * 1.4426950408889634 / p.temperature, 1e300);
  const Args a = {scores, p.rows, p.stride, (int)p.classes, uniform, p.temperature, factor, p.top_p, p.min_p, p.top_k, p.row_temperature, p.row_top_p, p.row_min_p,
                  p.row_top_k, drawn, log_probs, 0};
  const int64_t vectors = (p.classes + 2 * kPer - 2) / kPer;
  // a cluster where the rows leave SMs idle and a CTA's part is still some vectors a thread
  int ctas = p.rows <= 18 ? 8 : p.rows <= 37 ? 4 : p.rows <= 74 ? 2 : 1;
  while (ctas > 1 && vectors < 256 * ctas) ctas /= 2;
  return ctas == 8   ? launch_of<T, 8>(a, vectors, stream)
         : ctas == 4 ? launch_of<T, 4>(a, vectors, stream)
         : ctas == 2 ? launch_of<T, 2>(a, vectors, stream)
                     : launch_of<T, 1>(a, vectors, stream);
}

}  // namespace
}  // namespace sample
}  // namespace ht

using namespace ht;

extern "C" int ht_sample_classes(const ht_sample_problem *p, const void *scores, const float *uniform, int64_t *drawn, float *log_probs, ht_stream_t stream) {
  const int rc = sample::screen(p);
  if (rc != HT_OK) return rc;
  if (p->rows == 0) return HT_OK;
  if (scores == nullptr || uniform == nullptr || drawn == nullptr || log_probs == nullptr) return HT_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return p->dtype == HT_DTYPE_F32    ? sample::launch<float>(*p, scores, uniform, drawn, log_probs, s)
         : p->dtype == HT_DTYPE_BF16 ? sample::launch<__nv_bfloat16>(*p, scores, uniform, drawn, log_probs, s)
                                     : sample::launch<__half>(*p, scores, uniform, drawn, log_probs, s);
}

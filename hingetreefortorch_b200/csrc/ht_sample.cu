// A class drawn from each row of scores with a given random number, under bounds on the classes that count.
//
//     m = max s      w_i = exp((s_i - m) / T)                     (T = 0: the first class of the largest score)
//     order: larger scores first, of equal ones the lower class.  What counts is a prefix of that order, the shortest of
//       top_k classes;  the least that holds top_p of the weight of the first top_k;  the classes with w_i >= min_p;  never none
//     W = sum of w over what counts;  the class is the first i, in the order of classes, whose sum of w up to it is above u W
//     log_prob = (s_i - m) / T - log W
//
// A border that moves by 1e-8 of W picks another class once in some thousand rows of many classes, so weights and sums are 64-bit numbers: the
// decisions are those of the formulas.  The exponential is table-driven (P. T. P. Tang, Table-driven implementation of the exponential
// function, ACM TOMS 15, 1989): 2^(k / 64) from a table and a polynomial of degree 4, 4e-14.
//
// A CTA takes a row, which stays in shared memory where it fits.  A prefix of the order is held as its last class, (score, class).  To find it nothing
// is sorted but a list of up to 1024 classes around the place:
//   top_k   every thread has the maxima of up to 4 parts of what it has read; the k-th largest of those, found by halving the range,
//           bounds the k-th largest score from below, and not many more classes than k are above it
//   top_p   the same with the first 512 classes, where those hold enough
//   else    classes are counted, or their weights summed roughly, by 2048 ranges of the score's bits; the range with the place in it is listed, or
//           divided again, or is one score
// No sum depends on the order of atomic additions: the same call gives the same bits.
#include "ht_dense.cuh"

#include <math_constants.h>

namespace ht {
namespace sample {
namespace {

using dense::after_previous_kernel;
using dense::load_plain;
using dense::to_float;
using tile::smem_addr;

constexpr int kMostWarps = 32, kList = 1024, kBins = 2048, kParts = 4;
constexpr int kFirst = 512;          // classes that are listed first for top_p
constexpr double kTail = -80.0;      // whatever the classes below exp() of this are, they do not weigh 2^-53 of the row together
constexpr int kPassed = 0x7fffffff;  // no limit on the class among equal scores

struct Args {
  const void *scores;
  int64_t rows, stride;
  int classes;
  const float *uniform;
  double temperature, top_p, min_p;
  int64_t top_k;
  const float *row_temperature, *row_top_p, *row_min_p;
  const int64_t *row_top_k;
  int64_t *drawn;
  float *log_probs;
  uint32_t row_bytes;  // of shared memory for a row
};

// Larger for larger scores; both zeros are one score.
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s + 0.0f);
  return (b & 0x80000000u) != 0u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0u ? key & 0x7fffffffu : ~key); }

struct Shared {
  double table[64];
  double sums[kMostWarps];
  float floats[kMostWarps];
  uint32_t words[kMostWarps];
  uint32_t count, low, high, bin;
  double above;
  int drawn;
  float drawn_score;
  union {
    uint64_t list[kList];
    uint32_t bins[kBins];
  };
};

constexpr size_t kRowAt = (sizeof(Shared) + 127) / 128 * 128;

// w = exp((s - m) / T) as 2^(a / 64) with a = (s - m) 64 / (T ln 2).
struct Weight {
  double m, c;
  const double *table;
  __device__ __forceinline__ double operator()(float s) const {
    const double a = ((double)s - m) * c;
    constexpr double kStep = 0.69314718055994531 / 64.0;
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
};

// The last class of a prefix of the order.
struct Last {
  float score;
  int at;
  __device__ __forceinline__ bool holds(float s, int i) const { return s > score || (s == score && i <= at); }
};

template <typename T>
struct Row {
  static constexpr int kPer = 16 / (int)sizeof(T);
  const T *base;         // where the row's first 16 bytes start in memory
  unsigned char *shared; // the same in shared memory, or null
  int head, classes, vectors;
  // Class j kPer - head + i is number i of vector j.
  __device__ __forceinline__ uint4 from_memory(int j) const {
    const int first = j * kPer - head;
    if (first >= 0 && first + kPer <= classes) return load_plain(reinterpret_cast<const uint4 *>(base) + j);
    T t[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) t[i] = first + i >= 0 && first + i < classes ? base[j * (int64_t)kPer + i] : dense::from_float<T>(-CUDART_INF_F);
    return *reinterpret_cast<const uint4 *>(t);
  }
  __device__ __forceinline__ void values(int j, float (&v)[kPer]) const {
    T t[kPer];
    *reinterpret_cast<uint4 *>(t) = shared != nullptr ? reinterpret_cast<const uint4 *>(shared)[j] : from_memory(j);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = to_float(t[i]);
  }
};

template <typename T>
struct Team {  // a CTA at work on a row
  static constexpr int kPer = Row<T>::kPer;
  Shared &sh;
  Row<T> row;
  int lane, warp, warps, first, last;  // of this warp: vectors first .. last - 1

  // f(score, class) for every class of this warp's part of the row.
  template <typename F>
  __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 1
    for (int j = first + lane; j < last; j += 32) {
      float v[kPer];
      row.values(j, v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) f(v[i], j * kPer - row.head + i);
    }
  }
  __device__ __forceinline__ double warp_sum(double v) const {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
  }
  // Of all threads, to all of them; two barriers.
  __device__ __forceinline__ double sum(double v) const {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.sums[warp] = v;
    __syncthreads();
    return warp_sum(lane < warps ? sh.sums[lane] : 0.0);
  }
  __device__ __forceinline__ float largest(float v) const {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    __syncthreads();
    if (lane == 0) sh.floats[warp] = v;
    __syncthreads();
    v = lane < warps ? sh.floats[lane] : -CUDART_INF_F;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
  }
  __device__ __forceinline__ uint32_t least(uint32_t v) const {
    v = __reduce_min_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sh.words[warp] = v;
    __syncthreads();
    return __reduce_min_sync(0xffffffffu, lane < warps ? sh.words[lane] : 0xffffffffu);
  }
  __device__ __forceinline__ uint32_t total(uint32_t v) const {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sh.words[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, lane < warps ? sh.words[lane] : 0u);
  }

  // Lists the classes that `takes` says, as many as fit, and gives their number; a barrier follows the list.
  template <typename F>
  __device__ __forceinline__ uint32_t list(F &&takes) const {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each([&](float s, int i) {
      if (takes(s, i)) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < (uint32_t)kList) sh.list[at] = (uint64_t)key_of(s) << 32 | (0xffffffffu - (uint32_t)i);
      }
    });
    __syncthreads();
    return sh.count;
  }
  // Sorts the list, the largest first: bitonic, as many places as the next power of two.
  __device__ __forceinline__ void sort(int n) const {
    int places = 2;
    while (places < n) places *= 2;
    for (int i = n + (int)threadIdx.x; i < places; i += (int)blockDim.x) sh.list[i] = 0;
    __syncthreads();
    for (int size = 2; size <= places; size *= 2)
      for (int d = size / 2; d >= 1; d /= 2) {
        for (int i = (int)threadIdx.x; i < places / 2; i += (int)blockDim.x) {
          const int a = 2 * i - (i & (d - 1)), b = a + d;
          const uint64_t x = sh.list[a], y = sh.list[b];
          if ((x < y) == ((a & size) == 0)) sh.list[a] = y, sh.list[b] = x;
        }
        __syncthreads();
      }
  }
  __device__ __forceinline__ Last listed(int i) const {
    const uint64_t e = sh.list[i];
    return {score_of((uint32_t)(e >> 32)), (int)(0xffffffffu - (uint32_t)e)};
  }
  // Of the sorted list's first n, with `before` of weight ahead of them: how many start below `target`, and the weight of all n in *weight.
  __device__ __forceinline__ int places_below(int n, const Weight &w, double before, double target, double *weight) const {
    // every thread has neighbours: kList / threads of them at the most
    const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x, from = (int)threadIdx.x * per, to = min(from + per, n);
    double own = 0.0;
    for (int i = from; i < to; ++i) own += w(listed(i).score);
    double upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += t;
    }
    __syncthreads();
    if (lane == 31) sh.sums[warp] = upto;
    __syncthreads();
    double ahead = 0.0, all = 0.0;
    for (int i = 0; i < warps; ++i) {
      if (i < warp) ahead += sh.sums[i];
      all += sh.sums[i];
    }
    *weight = all;
    double at = before + ahead + (upto - own);
    uint32_t count = 0;
    for (int i = from; i < to; ++i) {
      count += at < target ? 1u : 0u;
      at += w(listed(i).score);
    }
    return (int)total(count);
  }

  // The class of the n-th (from 1) of those with this score, in the order of classes.
  __device__ __forceinline__ int nth_of(float score, uint32_t n) const {
    uint32_t own = 0;
    each([&](float s, int) { own += s == score ? 1u : 0u; });
    own = __reduce_add_sync(0xffffffffu, own);
    __syncthreads();
    if (lane == 0) sh.words[warp] = own;
    if (threadIdx.x == 0) sh.drawn = kPassed;
    __syncthreads();
    uint32_t ahead = 0;
    for (int i = 0; i < warp; ++i) ahead += sh.words[i];
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
            if (v[i] == score && ++at == n) sh.drawn = j * kPer - row.head + i;
        }
        ahead += __shfl_sync(0xffffffffu, upto, 31);
        if (ahead >= n) break;
      }
    }
    __syncthreads();
    return sh.drawn;
  }

  // The last class of the shortest prefix that reaches `target`, counted (WEIGHTS false) or weighed, among the classes that `base` holds and
  // whose keys are in [low, high]; all others of base are above and are `above` together.  For weights `all` is about what base weighs.
  template <bool WEIGHTS>
  __device__ __forceinline__ Last narrow(const Weight &w, const Last &base, uint32_t low, uint32_t high, double above, double target, double all) const {
    for (;;) {
      // by ranges of the key, highest first
      const uint32_t width = high - low;
      int shift = 0;
      while ((width >> shift) >= (uint32_t)kBins) ++shift;
      const double scale = 2147483648.0 / all;
      __syncthreads();
      for (int i = (int)threadIdx.x; i < kBins; i += (int)blockDim.x) sh.bins[i] = 0;
      __syncthreads();
      each([&](float s, int i) {
        const uint32_t key = key_of(s);
        if (key >= low && key <= high && base.holds(s, i)) atomicAdd(&sh.bins[(high - key) >> shift], WEIGHTS ? (uint32_t)(w(s) * scale + 0.5) : 1u);
      });
      __syncthreads();
      // the range in which the sum reaches the target: warps take neighbouring ranges
      const uint32_t wanted = WEIGHTS ? (uint32_t)fmin(fmax((target - above) * scale, 1.0), 2147483647.0) : (uint32_t)(target - above);
      if (warp == 0) {
        uint32_t own = 0;
        for (int i = 0; i < kBins / 32; ++i) own += sh.bins[lane * (kBins / 32) + i];
        uint32_t upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t t = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += t;
        }
        uint32_t at = upto - own;
        if (at < wanted && wanted <= upto) {
          int b = lane * (kBins / 32);
          while (at + sh.bins[b] < wanted) at += sh.bins[b++];
          sh.bin = (uint32_t)b;
        }
        if (lane == 31 && upto < wanted) sh.bin = width >> shift;  // (rounding: the last)
      }
      __syncthreads();
      uint32_t bin = sh.bin;
      const uint32_t last_bin = width >> shift;
      int moved = 0;  // the way that the range has moved since: it does not come back
      double over;
      uint32_t n;
      Last end;
      for (;;) {  // (a rough sum may be one range off)
        const uint32_t top = high - (bin << shift), bottom = top - low < (1u << shift) ? low : top - (1u << shift) + 1u;
        double mine = 0.0;
        uint32_t least_key = 0xffffffffu, least_gap = 0xffffffffu;  // of the range: its keys reach from `lowest` to `highest`
        n = list([&](float s, int i) {
          const uint32_t key = key_of(s);
          if (key < bottom || key > high || !base.holds(s, i)) return false;
          if (key > top) {
            mine += WEIGHTS ? w(s) : 1.0;
            return false;
          }
          least_key = min(least_key, key), least_gap = min(least_gap, 0xffffffffu - key);
          return true;
        });
        over = above + sum(mine);
        if (bin > 0u && moved <= 0 && ((WEIGHTS && over >= target) || (n == 0u && moved < 0))) {
          --bin;
          moved = -1;
          continue;
        }
        const bool may_rise = bin < last_bin && moved >= 0;
        if (n == 0u && may_rise) {
          ++bin;
          moved = 1;
          continue;
        }
        if (n == 0u) return {score_of(bottom), kPassed};
        const uint32_t lowest = least(least_key), highest = 0xffffffffu - least(least_gap);
        if (n <= (uint32_t)kList) {
          sort((int)n);
          double weight;
          int places;
          if (WEIGHTS) {
            places = places_below((int)n, w, over, target, &weight);
            if (over + weight < target && may_rise) {
              ++bin;
              moved = 1;
              continue;
            }
          } else {
            places = (int)(target - over);
          }
          end = listed(max(min(places, (int)n), 1) - 1);
          __syncthreads();
          return end;
        }
        if (lowest == highest) {  // more of one score than the list holds
          const float s = score_of(lowest);
          const double one = WEIGHTS ? w(s) : 1.0, missing = target - over;
          if (WEIGHTS && over + one * n < target && may_rise) {
            ++bin;
            moved = 1;
            continue;
          }
          const uint32_t places = one * n <= missing ? n : (uint32_t)fmax(ceil(missing / one), 1.0);
          // (among those that base holds the first ones are the first ones of all)
          return {s, nth_of(s, places)};
        }
        low = lowest, high = highest;
        above = over;
        break;
      }
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(32 * kMostWarps) sample_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char sample_smem[];
  Shared &sh = *reinterpret_cast<Shared *>(sample_smem);
  constexpr int kPer = Row<T>::kPer;
  after_previous_kernel();
  const int64_t r = blockIdx.x;
  const T *from = static_cast<const T *>(a.scores) + r * a.stride;
  Row<T> row;
  row.head = (int)((reinterpret_cast<uintptr_t>(from) & 15u) / sizeof(T));
  row.base = from - row.head;
  row.classes = a.classes;
  row.vectors = (int)(((int64_t)row.head + a.classes + kPer - 1) / kPer);
  row.shared = nullptr;
  const int warps = (int)blockDim.x / 32, warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int part = (row.vectors + warps - 1) / warps;
  Team<T> team = {sh, row, lane, warp, warps, min(warp * part, row.vectors), min((warp + 1) * part, row.vectors)};

  // the row into shared memory, and its largest and least score
  if (a.row_bytes > 0) {
    unsigned char *const to = sample_smem + kRowAt;
    for (int j = team.first + lane; j < team.last; j += 32) {
      const int first = j * kPer - row.head;
      if (first >= 0 && first + kPer <= a.classes)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to) + 16u * (uint32_t)j), "l"(reinterpret_cast<const uint4 *>(row.base) + j) : "memory");
      else
        reinterpret_cast<uint4 *>(to)[j] = row.from_memory(j);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    team.row.shared = to;
  }
  if (threadIdx.x < 64) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
  const double temperature = a.row_temperature != nullptr ? (double)load_plain(a.row_temperature + r) : a.temperature;
  const double top_p = a.row_top_p != nullptr ? (double)load_plain(a.row_top_p + r) : a.top_p;
  const double min_p = a.row_min_p != nullptr ? (double)load_plain(a.row_min_p + r) : a.min_p;
  const int64_t asked = a.row_top_k != nullptr ? load_plain(a.row_top_k + r) : a.top_k;
  const double u = (double)load_plain(a.uniform + r);
  const int top_k = asked > 0 && asked < a.classes ? (int)asked : a.classes;

  __syncthreads();  // (all of the row: no warp reads another's part, but the table)
  float part_max[kParts], low = CUDART_INF_F;
  bool number = true;
#pragma unroll
  for (int i = 0; i < kParts; ++i) part_max[i] = -CUDART_INF_F;
#pragma unroll 1
  for (int j = team.first + lane; j < team.last; j += 32) {
    float v[kPer];
    team.row.values(j, v);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float &top = part_max[i * kParts / kPer];
      top = fmaxf(top, v[i]);
      number &= v[i] == v[i];
      if (v[i] > -CUDART_INF_F) low = fminf(low, v[i]);
    }
  }
  const float m = team.largest(fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3])));
  low = -team.largest(-low);
  const bool bounds = temperature >= 0.0 && temperature < CUDART_INF && top_p == top_p && min_p == min_p && u >= 0.0 && u <= 1.0;
  if (__syncthreads_or(!number) || !bounds || !(m > -CUDART_INF_F && m < CUDART_INF_F)) {
    if (threadIdx.x == 0) a.drawn[r] = -1, a.log_probs[r] = CUDART_NAN_F;
    return;
  }
  if (temperature == 0.0 || top_k == 1 || top_p <= 0.0 || min_p > 1.0) {
    uint32_t at = 0xffffffffu;
    team.each([&](float s, int i) {
      if (s == m) at = min(at, (uint32_t)i);
    });
    at = team.least(at);
    if (threadIdx.x == 0) a.drawn[r] = (int64_t)at, a.log_probs[r] = 0.0f;
    return;
  }
  const Weight w = {(double)m, fmin(64.0 * 1.4426950408889634 / temperature, 1e300), sh.table};

  // what counts: up to `end`
  const double lowest = fmax((double)low, (double)m + kTail * temperature);
  Last end = {-CUDART_INF_F, kPassed};
  const uint32_t high_key = key_of(m);
  const uint32_t low_key = min(key_of(lowest > (double)low ? (float)lowest : low), high_key);
  if (top_k < a.classes || top_p < 1.0) {
    const bool by_count = top_k < a.classes;
    const uint32_t wanted = (uint32_t)(by_count ? top_k : kFirst);
    // a lower bound for the score of place `wanted`: at least so many of the parts' maxima are not below it
    uint32_t bound = 0;
    if (wanted <= blockDim.x * kParts) {
      uint32_t keys[kParts], from_key = key_of(low), to_key = high_key;
#pragma unroll
      for (int i = 0; i < kParts; ++i) keys[i] = key_of(part_max[i]);
      while (from_key < to_key) {
        const uint32_t middle = from_key + (to_key - from_key) / 2u + 1u;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < kParts; ++i) n += keys[i] >= middle ? 1u : 0u;
        n = team.total(n);
        if (n >= wanted) {
          from_key = middle;
          if (n <= wanted + wanted / 16u) break;
        } else {
          to_key = middle - 1u;
        }
      }
      bound = from_key;
    }
    const uint32_t n = bound > 0u ? team.list([&](float s, int) { return key_of(s) >= bound; }) : 0xffffffffu;
    if (n <= (uint32_t)kList) team.sort((int)n);
    double all = 0.0;
    bool done = false;
    if (by_count) {
      if (n <= (uint32_t)kList) {
        end = team.listed(min(top_k, (int)n) - 1);
        if (top_p < 1.0) {
          const int held = min(top_k, (int)n);
          team.places_below(held, w, 0.0, 0.0, &all);
          double ignored;
          end = team.listed(max(team.places_below(held, w, 0.0, top_p * all, &ignored), 1) - 1);
        }
        done = true;
        __syncthreads();
      } else {
        const uint32_t from_key = max(bound, key_of(low));
        double inside = 0.0;
        team.each([&](float s, int) { inside += key_of(s) >= from_key ? 1.0 : 0.0; });
        inside = team.sum(inside);
        if (inside >= (double)top_k) end = team.template narrow<false>(w, end, from_key, high_key, 0.0, (double)top_k, 1.0);
      }
    }
    if (!done && top_p < 1.0) {
      double own = 0.0;
      team.each([&](float s, int i) {
        if (end.holds(s, i)) own += w(s);
      });
      all = team.sum(own);
      if (!by_count && n <= (uint32_t)kList) {
        double weight;
        const int places = team.places_below((int)n, w, 0.0, top_p * all, &weight);
        if (weight >= top_p * all) {
          end = team.listed(max(places, 1) - 1);
          done = true;
        }
        __syncthreads();
      }
      if (!done) end = team.template narrow<true>(w, end, max(low_key, key_of(end.score)), high_key, 0.0, top_p * all, all);
    }
  }

  // the draw: the sums of the warps' parts, then along one part
  auto weight = [&](float s, int i) {
    if (!end.holds(s, i)) return 0.0;
    const double v = w(s);
    return v >= min_p ? v : 0.0;
  };
  double own = 0.0;
  team.each([&](float s, int i) { own += weight(s, i); });
  own = team.warp_sum(own);
  __syncthreads();
  if (lane == 0) sh.sums[warp] = own;
  __syncthreads();
  double all = 0.0, ahead = 0.0;
  int place = -1;
  for (int i = 0; i < warps; ++i) all += sh.sums[i];
  const double target = u * all;
  for (int i = 0; i < warps; ++i) {  // the first part that ends above the target, or (u = 1, rounding) the last that weighs anything
    const double s = sh.sums[i];
    if (s > 0.0) {
      if (place >= 0) ahead += sh.sums[place];
      place = i;
      if (ahead + s > target) break;
    }
  }
  if (warp == place) {
    int found = -1;
    float found_score = 0.0f;
    for (int j0 = team.first; j0 < team.last; j0 += 32) {
      const int j = j0 + lane;
      float v[kPer];
      double here = 0.0;
      if (j < team.last) {
        team.row.values(j, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) here += weight(v[i], j * kPer - row.head + i);
      }
      double upto = here;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += t;
      }
      const uint32_t reached = __ballot_sync(0xffffffffu, ahead + upto > target), some = __ballot_sync(0xffffffffu, here > 0.0);
      // the lane in which the sum passes the target, or (lanes' sums may differ in their last bit) the last one so far that weighs anything
      const uint32_t passing = reached & some;
      const int at = passing != 0u ? __ffs((int)passing) - 1 : some != 0u ? 31 - __clz((int)some) : -1;
      if (lane == at) {
        double sum = ahead + (upto - here);
        bool passed = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int c = j * kPer - row.head + i;
          const double one = weight(v[i], c);
          sum += one;
          if (one > 0.0 && !passed) {
            found = c;
            found_score = v[i];
            passed = sum > target;
          }
        }
      }
      if (at >= 0) {
        found = __shfl_sync(0xffffffffu, found, at);
        found_score = __shfl_sync(0xffffffffu, found_score, at);
      }
      if (reached != 0u && found >= 0) break;
      ahead += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      a.drawn[r] = found;
      a.log_probs[r] = (float)(((double)found_score - (double)m) / temperature - log(all));
    }
  }
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

template <typename T>
int launch(const ht_sample_problem &p, const void *scores, const float *uniform, int64_t *drawn, float *log_probs, cudaStream_t stream) {
  constexpr int kPer = Row<T>::kPer;
  Args a = {scores, p.rows, p.stride, (int)p.classes, uniform, p.temperature, p.top_p, p.min_p, p.top_k, p.row_temperature, p.row_top_p, p.row_min_p,
            p.row_top_k, drawn, log_probs, 0};
  const int64_t vectors = (p.classes + 2 * kPer - 2) / kPer;
  if (kRowAt + 16 * (size_t)vectors <= kMostBytes) a.row_bytes = 16u * (uint32_t)vectors;
  const int threads = vectors >= 4096 ? 1024 : vectors >= 2048 ? 512 : vectors >= 512 ? 256 : 128;
  return dense::launch_next<sample_kernel<T>>(dim3((unsigned)p.rows), threads, kRowAt + a.row_bytes, kMostBytes, stream, 1, a);
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

// Drawing a token of each row of logits by a given random number (pg_sample in
// include/ptxgen_b200.h).
//
// With m the row's largest logit and weights w = exp((x - m) / T), the kept tokens are a prefix of
// the tokens ordered by logit, the largest first and ties by the lowest column: the shortest of the
// first top_k; the fewest whose weights reach top_p of the top_k ones' sum; and those with w >=
// min_p. The token drawn is the lowest kept column c with
//   sum of w over the kept columns up to c  >  u * (sum of w over all kept columns).
//
// Which token that is hangs on sums of up to 100000s of weights next to a border, so sums in 32 bits
// would give another token about once in a hundred rows of a flat distribution. Weights and sums are
// 64-bit numbers here, weights to 2^-38: any order of the sum gives the same token but for one draw in 10^9.
//
// A cluster of blocks takes a row, each a part of it, which stays in shared memory while it is gone
// through: the largest logit; the sum of weights, where top_p is of all; then the last kept token is
// searched as a value and a column, by histograms over ever narrower intervals of values until an
// interval holds one value or few tokens, which are ranked; and last the warps' sums of kept
// weights, which lie one after another in the row, say in which of them the drawn token is, and that
// warp goes through its part once more.
#include "common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kPerSm = 2;             // blocks an SM holds
constexpr int kParts = 8;             // blocks a row is cut in at most (a portable cluster)
constexpr int kBins = 1024;           // two a thread
constexpr int kFew = 512;             // tokens that are ranked one against another
constexpr int kTable = 16;            // 2^(i / 16): one bank of shared memory each
constexpr int kResident = 88 * 1024;  // bytes of a part that stay in shared memory
// Each interval is one of 1024 of the last one and never all of it. Values that lie evenly take two or
// three; ones of ever smaller size, ten binades at a time, 28.
constexpr int kLevels = 64;
// From so many rows on, those without limits take a block each and one pass over a row. With and without,
// in microseconds, bf16: 32 rows of 32001 14 and 13, 64 of 128256 both 38, 128 of 128256 42 and 66, 128 of
// 32001 11 and 22, 300 of 32001 22 and 49.
constexpr int kDrawRows = 128;
constexpr float kLargest = 3.402823466e38f;
constexpr double kSteep = 200.0 * (1 << 24);
constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

struct Arguments {
  const void *logits;
  const float *uniform, *temperature, *top_p, *min_p;
  const int *top_k;
  int64_t *tokens;
  float *logp;
  int64_t row_stride;
  int vocab, resident;  // whether parts stay in shared memory
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <class T> struct Vec;  // 16 bytes of T as f32
template <> struct Vec<float> {
  static constexpr int n = 4;
  __device__ static void get(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static void get(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  __device__ static void get(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
};
template <class T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest() { return -INFINITY; }
template <> __device__ __forceinline__ __nv_bfloat16 lowest() { return __float2bfloat16(-INFINITY); }
template <> __device__ __forceinline__ __half lowest() { return __float2half(-INFINITY); }

// A key whose order as a whole number is the logits' order, -0 equal to 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Weights below about 2^-500 of that of `top` stay there.
__device__ __forceinline__ float floor_of(float top, double scale) {
  return fmaxf(-kLargest, __double2float_rd(top - 500.0 / scale));
}

// What a warp, and then a block, knows of its tokens.
struct Extent {
  float top, low;  // the largest and the lowest that is more than -inf
};
struct Mass {  // of the tokens above a bin and within it
  double above, within;
  float top, low;  // of the bin
  int count;       // of the bin
};

struct Shared {
  double power[kTable];
  double warp_sum[kWarps];           // the warps' sums of kept weights
  double all_sums[kParts * kWarps];
  Mass warp_mass[kWarps], mass;
  Extent warp_extent[kWarps], extent;
  double warp_total[kWarps], total;
  unsigned bins[kBins], upto[kBins];
  unsigned warp_bins[kWarps];
  uint64_t few[kFew];                // block 0's: tokens to rank
  double few_weight[kFew];
  uint64_t border;                   // block 0's: the last kept token
  int few_n;
  int bin;
};

// 2^t to about 2^-38, for t = d scale of -1000 to 1000 (whose product is not rounded): 2^(i/16) from a
// table, and e^x with |x| <= a = ln 2 / 32 by the series up to x^4 and, in place of x^5 / 120, the cubic
// that is nearest to it there (Chebyshev's: it leaves a^5 / 1920). 2^0 is 1.
__device__ __forceinline__ double power_of_two(const double *power, double d, double scale) {
  constexpr double kShift = 6755399441055744.0 / kTable;  // 1.5 * 2^52 in steps of 1/16
  constexpr double k2 = kLn2 * kLn2, kA2 = k2 / (4 * kTable * kTable);
  const double z = fma(d, scale, kShift);
  const int n = __double2loint(z);  // t in 16ths, rounded
  const double r = fma(d, scale, kShift - z);
  double p = fma(r, k2 * k2 / 24, k2 * kLn2 * (1.0 / 6 + 1.25 * kA2 / 120));
  p = fma(r, p, k2 / 2);
  p = fma(r, p, kLn2 * (1.0 - 0.3125 * kA2 * kA2 / 120)) * r;
  const double f = power[n & (kTable - 1)];
  const double y = fma(f, p, f);
  return __hiloint2double(__double2hiint(y) + (n >> 4 << 20), __double2loint(y));
}

// A block's part of a row: columns [first, last). Warp w takes a run of its 16-byte vectors, so
// that the warps' parts lie in the row's order; columns outside read as -inf, which has no weight.
template <class T>
struct Part {
  const T *row;
  const uint4 *held;  // its vectors in shared memory
  int first, last, base, vectors, begin, end;  // the warp's run of vectors

  __device__ Part(const T *r, int a, int b, const uint4 *shared) : row(r), held(shared), first(a),
                                                                  last(b) {
    const int over = static_cast<int>((reinterpret_cast<uintptr_t>(r + a) & 15) / sizeof(T));
    base = a - over;
    vectors = b > a ? (b - base + Vec<T>::n - 1) / Vec<T>::n : 0;
    const int each = (vectors + kThreads - 1) / kThreads * 32, warp = threadIdx.x >> 5;
    begin = min(warp * each, vectors);
    end = min(begin + each, vectors);
  }
  __device__ uint4 fetch(int v) const {
    const int at = base + v * Vec<T>::n;
    if (at >= first && at + Vec<T>::n <= last) return pg::load16(row + at);
    union {
      uint4 raw;
      T x[Vec<T>::n];
    } u;
#pragma unroll
    for (int i = 0; i < Vec<T>::n; ++i)
      u.x[i] = at + i >= first && at + i < last ? row[at + i] : lowest<T>();
    return u.raw;
  }
  __device__ void load(int v, float *x) const {
    Vec<T>::get(held ? held[v] : fetch(v), x);
  }
  // f(x, column) of each token of this thread
  template <class F>
  __device__ void each(F f) const {
    for (int v = begin + (threadIdx.x & 31); v < end; v += 32) {
      float x[Vec<T>::n];
      load(v, x);
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i) f(x[i], base + v * Vec<T>::n + i);
    }
  }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int off = 16; off; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// The tokens that are kept: those above a value, and of those at it the ones up to a column; and
// all at least as large as `least`.
struct Kept {
  float value, least;
  int column;
  __device__ bool has(float x, int at) const {
    return x >= least && (x > value || (x == value && at <= column));
  }
};

// An interval of values in kBins equal bins, the largest values first.
struct Bins {
  float hi, lo, up, per;  // up: so that a difference of numbers near the smallest has its inverse
  __device__ Bins(float h, float l) : hi(h), lo(l), up(h - l < 0x1p-100f ? 0x1p100f : 1.0f) {
    per = kBins / fminf((hi - lo) * up, kLargest);
  }
  __device__ bool has(float x) const { return x >= lo && x <= hi; }
  __device__ int of(float x) const {
    return min(kBins - 1, max(0, __float2int_rz((hi - x) * up * per)));
  }
};

template <class T>
struct Row {
  const Part<T> &part;
  Shared &sh;
  cg::cluster_group cluster;
  int blocks, rank;
  float top, low;   // the row's largest and lowest finite logits
  float mine;       // the thread's largest
  double scale;     // log2 e / T
  float floor;      // what is below weighs as much, 2^-500 or less

  __device__ double weight(float x) const {
    return power_of_two(sh.power, static_cast<double>(fmaxf(x, floor)) - static_cast<double>(top), scale);
  }

  // f(x, column)'s sum over the row, in an order of its own for each size of a row
  template <class F>
  __device__ double total(F f) {
    double sum = 0.0;
    part.each([&](float x, int at) { sum += f(x, at); });
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) sh.warp_total[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) sum += sh.warp_total[w];
      sh.total = sum;
    }
    cluster.sync();
    sum = 0.0;
    for (int b = 0; b < blocks; ++b) sum += cluster.map_shared_rank(&sh, b)->total;
    return sum;
  }

  // The lowest column at which f's sums along the row exceed `share` of their total (or `goal` where
  // that is not negative), and f there; the warp that has it calls found(column, f, total). Where
  // rounding leaves no such column it is the last one that has any.
  template <class F, class G>
  __device__ void locate(F f, double share, double goal, G found) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double sum = 0.0;
    part.each([&](float x, int at) { sum += f(x, at); });
    sum = warp_sum(sum);
    if (lane == 0) sh.warp_sum[warp] = sum;
    cluster.sync();
    const int n = blocks * kWarps;
    for (int i = tid; i < n; i += kThreads)
      sh.all_sums[i] = cluster.map_shared_rank(&sh, i / kWarps)->warp_sum[i % kWarps];
    __syncthreads();
    // every warp adds all sums up in the same order, so that one warp's end is the next one's start
    constexpr int kEach = kParts * kWarps / 32;
    double s[kEach], mine = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = lane * kEach + i;
      s[i] = at < n ? sh.all_sums[at] : 0.0;
      mine += s[i];
    }
    double upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    const double all = __shfl_sync(0xffffffffu, upto, 31);
    const double before = __shfl_up_sync(0xffffffffu, upto, 1);
    double at = lane ? before : 0.0;
    const double target = goal >= 0.0 ? goal : share * all;
    int hit = -1, last = -1;  // the first warp whose end is past the target; the last with any weight
    double hit_at = 0.0, last_at = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const double next = at + s[i];
      if (s[i] > 0.0) {
        last = lane * kEach + i, last_at = at;
        if (hit < 0 && next > target) hit = last, hit_at = at;
      }
      at = next;
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0);
    const unsigned lasts = __ballot_sync(0xffffffffu, last >= 0);
    const int from = hits ? __ffs(hits) - 1 : 31 - __clz(lasts | 1);
    const int owner = __shfl_sync(0xffffffffu, hits ? hit : last, from);
    double start = __shfl_sync(0xffffffffu, hits ? hit_at : last_at, from);
    if (owner != rank * kWarps + warp) return;
    // this warp's part once more, 32 vectors at a time
    int best = -1;
    double best_f = 0.0;
    for (int v0 = part.begin; v0 < part.end; v0 += 32) {
      const int v = v0 + lane;
      double y[Vec<T>::n], here = 0.0;
      float x[Vec<T>::n];
      if (v < part.end) part.load(v, x);
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i) {
        y[i] = v < part.end ? f(x[i], part.base + v * Vec<T>::n + i) : 0.0;
        here += y[i];
      }
      double sums = here;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, sums, off);
        if (lane >= off) sums += o;
      }
      double c = start + (sums - here);
      bool past = false;
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i) {
        c += y[i];
        if (y[i] > 0.0 && !past) {  // the first past the target, or else the last with any
          best = part.base + v * Vec<T>::n + i, best_f = y[i];
          past = c > target;
        }
      }
      const unsigned pasts = __ballot_sync(0xffffffffu, past);
      if (pasts) {
        const int src = __ffs(pasts) - 1;
        best = __shfl_sync(0xffffffffu, best, src);
        best_f = __shfl_sync(0xffffffffu, best_f, src);
        break;
      }
      start += __shfl_sync(0xffffffffu, sums, 31);
      // no lane is past it: the last one with any weight stands until a later one is
      int b = best;
#pragma unroll
      for (int off = 16; off; off >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, off));
      const unsigned who = __ballot_sync(0xffffffffu, best == b);
      best_f = __shfl_sync(0xffffffffu, best_f, __ffs(who) - 1);
      best = b;
    }
    if (lane == 0) found(best, best_f, all);
  }


  // Blocks' histograms, added up: sh.upto[b] is the sum of bins 0 to b.
  __device__ void scan_bins() {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cluster.sync();
    uint2 n = make_uint2(0, 0);
    for (int b = 0; b < blocks; ++b) {
      const uint2 o = reinterpret_cast<const uint2 *>(cluster.map_shared_rank(&sh, b)->bins)[tid];
      n.x += o.x, n.y += o.y;
    }
    unsigned upto = n.x + n.y;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 31) sh.warp_bins[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += sh.warp_bins[w];
    reinterpret_cast<uint2 *>(sh.upto)[tid] = make_uint2(upto - n.y, upto);
  }

  // The first bin up to which there are `goal` or more; kBins if there is none.
  __device__ int first_bin(unsigned goal) {
    if (threadIdx.x == 0) sh.bin = kBins;
    __syncthreads();
    const uint2 upto = reinterpret_cast<const uint2 *>(sh.upto)[threadIdx.x];
    const unsigned before = threadIdx.x ? sh.upto[2 * threadIdx.x - 1] : 0;
    if (before < goal && upto.y >= goal) sh.bin = 2 * threadIdx.x + (upto.x < goal);
    __syncthreads();
    return sh.bin;
  }

  // Masses of the tokens of `kept` above a bin and within it.
  __device__ Mass mass_of(const Kept &kept, const Bins &bins, int bin, bool weights) {
    Mass m{0.0, 0.0, -INFINITY, INFINITY, 0};
    part.each([&](float x, int at) {
      if (!(x >= bins.lo) || !kept.has(x, at)) return;
      const int b = x > bins.hi ? -1 : bins.of(x);
      if (b > bin) return;
      const double w = weights ? weight(x) : 0.0;
      if (b < bin) {
        m.above += w;
      } else {
        m.within += w;
        m.top = fmaxf(m.top, x), m.low = fminf(m.low, x);
        ++m.count;
      }
    });
    const auto join = [](Mass a, const Mass &b) {
      a.above += b.above, a.within += b.within;
      a.top = fmaxf(a.top, b.top), a.low = fminf(a.low, b.low);
      a.count += b.count;
      return a;
    };
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      Mass o;
      o.above = __shfl_xor_sync(0xffffffffu, m.above, off);
      o.within = __shfl_xor_sync(0xffffffffu, m.within, off);
      o.top = __shfl_xor_sync(0xffffffffu, m.top, off);
      o.low = __shfl_xor_sync(0xffffffffu, m.low, off);
      o.count = __shfl_xor_sync(0xffffffffu, m.count, off);
      m = join(m, o);
    }
    if ((threadIdx.x & 31) == 0) sh.warp_mass[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) m = join(m, sh.warp_mass[w]);
      sh.mass = m;
    }
    cluster.sync();
    m = cluster.map_shared_rank(&sh, 0)->mass;
    for (int b = 1; b < blocks; ++b) m = join(m, cluster.map_shared_rank(&sh, b)->mass);
    cluster.sync();  // it may be made anew at once
    return m;
  }

  // The tokens of `kept` with values in [low, top], no more than kFew, ranked by block 0; the last
  // kept one is the `count`-th of them, or the first up to which `above` and their weights reach
  // `goal`. Where they are more than kFew after all, nothing is ranked and the result is 0.
  __device__ uint64_t rank_few(const Kept &kept, float hi_value, float lo_value, int count,
                               double above, double goal) {
    Shared &first = *cluster.map_shared_rank(&sh, 0);
    if (rank == 0 && threadIdx.x == 0) sh.few_n = 0;
    cluster.sync();
    part.each([&](float x, int at) {
      if (x >= lo_value && x <= hi_value && kept.has(x, at)) {
        const int i = atomicAdd(&first.few_n, 1);
        if (i < kFew)
          first.few[i] = static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~at);
      }
    });
    cluster.sync();
    if (first.few_n > kFew) return 0;
    if (rank == 0) {
      const int n = sh.few_n, tid = threadIdx.x, lane = tid & 31;
      uint64_t e = 0;
      int place = 0;
      if (tid < n) {
        e = sh.few[tid];
        for (int j = 0; j < n; ++j) place += sh.few[j] > e;
      }
      __syncthreads();
      if (tid < n) {
        sh.few[place] = e;
        sh.few_weight[place] = goal < 0.0 ? 0.0 : weight(logit_of(static_cast<uint32_t>(e >> 32)));
      }
      __syncthreads();
      if (goal < 0.0) {
        if (tid == 0) sh.border = sh.few[min(max(count, 1), n) - 1];
      } else if (tid < 32) {
        int at = n - 1;
        for (int i0 = 0; i0 < n; i0 += 32) {
          const double w = i0 + lane < n ? sh.few_weight[i0 + lane] : 0.0;
          double upto = w;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += o;
          }
          const unsigned reached = __ballot_sync(0xffffffffu, i0 + lane < n && above + upto >= goal);
          if (reached) {
            at = i0 + __ffs(reached) - 1;
            break;
          }
          above += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) sh.border = sh.few[at];
      }
    }
    cluster.sync();
    return first.border;
  }

  // The `count`-th of the tokens that have the value x, by columns.
  __device__ uint64_t tie(const Kept &kept, float x, double count) {
    Shared &first = *cluster.map_shared_rank(&sh, 0);
    locate([&](float y, int at) { return y == x && kept.has(y, at) ? 1.0 : 0.0; }, 0.0, count - 0.5,
           [&](int column, double, double) {
             first.border = static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~column);
           });
    cluster.sync();
    return first.border;
  }

  __device__ void clear_bins() {
    reinterpret_cast<uint2 *>(sh.bins)[threadIdx.x] = make_uint2(0, 0);
    __syncthreads();
  }

  static __device__ void limit(Kept &kept, uint64_t border) {
    kept.value = logit_of(static_cast<uint32_t>(border >> 32));
    kept.column = static_cast<int>(~static_cast<uint32_t>(border));
  }

  // Keeps the first k.
  __device__ void keep_count(Kept &kept, unsigned k) {
    float hi = top, lo = low;
    const unsigned threads = blocks * kThreads;
    if (hi > lo && k <= threads / 4 * 3 && part.vectors >= 2 * kThreads) {
      // No fewer than k tokens are as large as the k-th of the threads' largest, and few more: those
      // below (by two bins, for the rounding) need not be counted.
      const Bins bins(hi, lo);
      clear_bins();
      if (bins.has(mine)) atomicAdd(&sh.bins[bins.of(mine)], 1u);
      scan_bins();
      const int bin = first_bin(k);
      if (bin < kBins) lo = fmaxf(lo, hi - (bin + 2) / (bins.up * bins.per));
      cluster.sync();
      if (k <= kFew / 2) {
        const uint64_t border = rank_few(kept, hi, lo, k, 0.0, -1.0);
        if (border) {
          limit(kept, border);
          return;
        }
      }
    }
    for (int level = 0; hi > lo && level < kLevels; ++level) {
      const Bins bins(hi, lo);
      clear_bins();
      part.each([&](float x, int) {
        if (bins.has(x)) atomicAdd(&sh.bins[bins.of(x)], 1u);
      });
      scan_bins();
      const int bin = first_bin(k);
      if (bin == kBins) return;  // fewer than k
      const unsigned before = bin ? sh.upto[bin - 1] : 0, count = sh.upto[bin] - before;
      k -= before;
      const Mass m = mass_of(kept, bins, bin, false);
      hi = m.top, lo = m.low;
      if (hi > lo && count <= kFew) {
        limit(kept, rank_few(kept, hi, lo, k, 0.0, -1.0));
        return;
      }
    }
    limit(kept, tie(kept, hi, k));
  }

  // Keeps the fewest whose weights reach `goal`; `sum` is that of all kept ones, no more than `count`.
  __device__ void keep_mass(Kept &kept, double goal, double sum, int count) {
    // Tokens that all together weigh less than what may be left out are: those below this.
    const double spare = (sum - goal) / count * 0.999;
    const float some = spare > 0.0
                           ? __double2float_rd(static_cast<double>(top) + log2(spare) / scale)
                           : -INFINITY;
    float hi = top, lo = fmaxf(low, some);
    double above = 0.0;
    const float per_weight = static_cast<float>(2147483648.0 / sum);
    const float scale_f = static_cast<float>(fmin(scale, static_cast<double>(kLargest)));
    for (int level = 0; hi > lo && level < kLevels; ++level) {
      const Bins bins(hi, lo);
      clear_bins();
      part.each([&](float x, int at) {
        if (bins.has(x) && kept.has(x, at))
          atomicAdd(&sh.bins[bins.of(x)],
                    __float2uint_rn(exp2_fast((x - top) * scale_f) * per_weight));
      });
      scan_bins();
      // about where the goal is reached; the sums in 64 bits say whether it is here or next to it
      int bin = first_bin(max(1u, static_cast<unsigned>((goal - above) / sum * 2147483648.0)));
      bin = min(bin, kBins - 1);
      Mass m = mass_of(kept, bins, bin, true);
      // `above` counts all above hi as well: the sums are of the kept ones from the top. A turn back
      // would be rounding's doing.
      for (int turn = 0;;) {
        const int step = m.above >= goal && bin > 0                              ? -1
                         : m.above + m.within < goal && bin < kBins - 1 ? 1
                                                                        : 0;
        if (!step || step == -turn) break;
        turn = step;
        bin += step;
        m = mass_of(kept, bins, bin, true);
      }
      above = m.above;
      if (!m.count) return;
      hi = m.top, lo = m.low;
      if (hi > lo && m.count <= kFew) {
        limit(kept, rank_few(kept, hi, lo, 0, above, goal));
        return;
      }
    }
    limit(kept, tie(kept, hi, fmax(1.0, ceil((goal - above) / weight(hi)))));
  }
};

// A row by the definition, taken by a cluster.
template <class T>
__device__ __forceinline__ void sample_row(const Arguments &a, Shared &sh, int row, uint4 *held) {
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *x_row = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int64_t v64 = a.vocab;
  const Part<T> part(x_row, static_cast<int>(v64 * rank / blocks),
                     static_cast<int>(v64 * (rank + 1) / blocks), held);
  const float u = a.uniform[row];
  const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  if (tid < kTable) sh.power[tid] = exp2(tid / static_cast<double>(kTable));

  Extent e{-INFINITY, INFINITY};
  for (int v = part.begin + lane; v < part.end; v += 32) {
    const uint4 raw = part.fetch(v);
    if (held) held[v] = raw;
    float x[Vec<T>::n];
    Vec<T>::get(raw, x);
#pragma unroll
    for (int i = 0; i < Vec<T>::n; ++i) {
      e.top = max_nan(e.top, x[i]);
      if (x[i] > -INFINITY) e.low = fminf(e.low, x[i]);
    }
  }
  const float mine = e.top;
  const auto join = [](Extent p, const Extent &q) {
    return Extent{max_nan(p.top, q.top), fminf(p.low, q.low)};
  };
#pragma unroll
  for (int off = 16; off; off >>= 1)
    e = join(e, Extent{__shfl_xor_sync(0xffffffffu, e.top, off),
                       __shfl_xor_sync(0xffffffffu, e.low, off)});
  if (lane == 0) sh.warp_extent[warp] = e;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) e = join(e, sh.warp_extent[w]);
    sh.extent = e;
  }
  cluster.sync();
  e = cluster.map_shared_rank(&sh, 0)->extent;
  for (int b = 1; b < blocks; ++b) e = join(e, cluster.map_shared_rank(&sh, b)->extent);

  const bool good = fabsf(e.top) < INFINITY && u == u && temperature >= 0.0f && top_p == top_p &&
                    min_p <= 1.0f;
  if (!good) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      a.logp[row] = NAN;
    }
    cluster.sync();  // a block's extent is read until here
    return;
  }
  // No larger than gives the logit next below the largest 2^-200 of its weight, so that as an f32 number
  // the floor, too, is above 2^-1000.
  const double scale = fmin(kLog2e / temperature, kSteep / fabs(static_cast<double>(e.top)));
  const float floor = floor_of(e.top, scale);
  Row<T> r{part, sh, cluster, blocks, rank, e.top, e.low, mine, scale, floor};
  Kept kept{-INFINITY, -kLargest, 0};
  const auto write = [&](int column, double w, double all) {
    a.tokens[row] = column;
    a.logp[row] = static_cast<float>(log(w / all));
  };
  if (temperature == 0.0f) {
    r.locate([&](float x, int) { return x == e.top ? 1.0 : 0.0; }, 0.0, 0.0,
             [&](int column, double, double) { write(column, 1.0, 1.0); });
  } else {
    if (top_k > 0 && top_k < a.vocab) r.keep_count(kept, top_k);
    if (top_p < 1.0f) {
      const bool all = kept.value == -INFINITY;
      const double sum = r.total([&](float x, int at) {
        return x > -INFINITY && (all || kept.has(x, at)) ? r.weight(x) : 0.0;
      });
      r.keep_mass(kept, fmax(static_cast<double>(top_p) * sum, 1e-300), sum,
                  all ? a.vocab : min(top_k, a.vocab));
    }
    // most are below min_p by their value already; the weight itself decides near it
    if (min_p > 0.0f)
      kept.least = fmaxf(-kLargest, __double2float_rd(static_cast<double>(e.top) +
                                                      log2(min_p * 0.999999) / r.scale));
    const double least = min_p;
    r.locate([&](float x, int at) {
               if (!kept.has(x, at)) return 0.0;
               const double w = r.weight(x);
               return w >= least ? w : 0.0;
             },
             fmaxf(u, 0.0f), -1.0, write);
  }
  cluster.sync();  // the blocks' sums are read until here
}

template <class T>
__global__ void __launch_bounds__(kThreads, kPerSm) sample_kernel(const __grid_constant__ Arguments a) {
  __shared__ Shared sh;
  extern __shared__ uint4 held[];
  pg::wait_for_earlier_kernels();
  sample_row<T>(a, sh, blockIdx.x / cg::this_cluster().num_blocks(), a.resident ? held : nullptr);
}

// ... by a block, for a row that a kernel hardly ever has.
template <class T>
__device__ __noinline__ void sample_rare_row(const Arguments &a, Shared &sh, int row) {
  sample_row<T>(a, sh, row, nullptr);
}

// Rows without limits. A block takes a row and goes over it once, a run of it a warp, with each warp's weights
// by the largest logit of the first that it has met (and by a larger one, its sum scaled, where later ones'
// weights pass 2^400). Then all of the block goes over the run of the warp that has the token.
//
// Ten 64-bit instructions a token bound it, 20 cycles of a quarter of an SM for 32 tokens, and one in eight
// of those for its conversion: 2000 rows of 50257 bf16 logits take 131 us, where these alone take 56 and
// HBM 31. (By sample_kernel, which keeps a row in shared memory and waits for all of it twice, 315 us; with
// the series in place of the table of 16 up to 2^-51, two instructions more, 166.) Tables of 256 numbers
// lie in the same banks for eight of 32 lanes: with one both kernels wait for shared memory.
constexpr int kBatch = 4;  // vectors a thread has in flight
template <class T>
__global__ void __launch_bounds__(kThreads, kPerSm) draw_kernel(const __grid_constant__ Arguments a) {
  __shared__ Shared sh;
  __shared__ float refs[kWarps];
  __shared__ int odd, hit;
  pg::wait_for_earlier_kernels();
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int N = Vec<T>::n;
  const T *x_row = static_cast<const T *>(a.logits) + row * a.row_stride;
  const Part<T> part(x_row, 0, a.vocab, nullptr);
  const float u = a.uniform[row];
  const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  const double scale = kLog2e / temperature;
  // What is none of an ordinary row goes by the definition: also u = 0, for which weights must be 0 that
  // are 2^-500 here, and any that is not finite.
  if (!(u > 0.0f && u < 1.0f && scale > 1e-30 && scale < 1e30)) {
    sample_rare_row<T>(a, sh, row);
    return;
  }
  if (tid < kTable) sh.power[tid] = exp2(tid / static_cast<double>(kTable));
  if (tid == 0) odd = 0, hit = -1;
  __syncthreads();

  const float scale_f = static_cast<float>(scale);
  float ref = -INFINITY, floor = -INFINITY;  // of the warp
  double sum = 0.0, ref_d = 0.0;
  const auto weigh = [&](float x) {
    return power_of_two(sh.power, static_cast<double>(fmaxf(x, floor)) - ref_d, scale);
  };
  const auto take = [&](const uint4 *raw, auto number) {
    constexpr int n = decltype(number)::value;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      float x[N];
      Vec<T>::get(raw[k], x);
#pragma unroll
      for (int i = 0; i < N; ++i) top = max_nan(top, x[i]);
    }
    if (__any_sync(kAll, !((top - ref) * scale_f <= 400.0f))) {
#pragma unroll
      for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(kAll, top, o));
      if (!(top < INFINITY && fabsf(top) * scale_f < static_cast<float>(kSteep)) && top != -INFINITY) odd = 1;
      if (top == -INFINITY || odd) return;  // all of them are
      sum = ref == -INFINITY ? 0.0 : sum * exp2(fmax((static_cast<double>(ref) - top) * scale, -2000.0));
      ref = top;
      ref_d = ref;
      floor = floor_of(ref, scale);
    }
#pragma unroll
    for (int k = 0; k < n; ++k) {
      float x[N];
      Vec<T>::get(raw[k], x);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += weigh(x[i]);
    }
  };
  const uint4 none = [] {
    union {
      uint4 raw;
      T x[N];
    } u;
    for (int i = 0; i < N; ++i) u.x[i] = lowest<T>();
    return u.raw;
  }();
  // the row's first and last vector may hold others' numbers: they come one number at a time
  const int inner = max(part.begin, 1), outer = min(part.end, part.vectors - 1);
  int v0 = inner;
  for (; v0 + 32 * kBatch <= outer; v0 += 32 * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) raw[k] = pg::load16(x_row + part.base + (v0 + 32 * k + lane) * N);
    take(raw, std::integral_constant<int, kBatch>());
  }
  for (; v0 < outer; v0 += 32) {
    const uint4 raw = v0 + lane < outer ? pg::load16(x_row + part.base + (v0 + lane) * N) : none;
    take(&raw, std::integral_constant<int, 1>());
  }
  if (part.begin == 0 || part.end == part.vectors) {
    uint4 raw = none;
    const int last = part.vectors - 1;
    const int v = lane == 0 && part.begin == 0 ? 0 : lane == 1 && last > 0 && part.begin <= last ? last : -1;
    if (v >= 0 && v < part.end) raw = part.fetch(v);
    take(&raw, std::integral_constant<int, 1>());
  }
  sum = warp_sum(sum);
  if (lane == 0) sh.warp_total[warp] = sum, refs[warp] = ref;
  __syncthreads();
  // all warps' sums by the largest reference, added up along the row
  float top = lane < kWarps ? refs[lane] : -INFINITY;
  const float mine = top;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
  if (odd || top == -INFINITY) {
    __syncthreads();
    sample_rare_row<T>(a, sh, row);
    return;
  }
  const double by =
      mine == -INFINITY ? 0.0 : exp2(fmax((static_cast<double>(mine) - top) * scale, -2000.0));
  double upto = lane < kWarps ? sh.warp_total[lane] * by : 0.0;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const double other = __shfl_up_sync(kAll, upto, o);
    if (lane >= o) upto += other;
  }
  const double all = __shfl_sync(kAll, upto, kWarps - 1), target = u * all;
  const unsigned past = __ballot_sync(kAll, lane < kWarps && upto > target);
  const int owner = past ? __ffs(past) - 1 : kWarps - 1;
  double start = owner ? __shfl_sync(kAll, upto, owner - 1) : 0.0;
  const double owner_by = __shfl_sync(kAll, by, owner);
  ref = __shfl_sync(kAll, mine, owner);
  ref_d = ref;
  floor = floor_of(ref, scale);
  const int each = (part.vectors + kThreads - 1) / kThreads * 32;
  const int begin = min(owner * each, part.vectors), end = min(begin + each, part.vectors);
  for (int v0 = begin; v0 < end; v0 += kThreads) {
    const int v = v0 + tid;
    float x[N];
    double y[N], here = 0.0;
    if (v < end) part.load(v, x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      y[i] = v < end && x[i] > -INFINITY ? weigh(x[i]) * owner_by : 0.0;
      here += y[i];
    }
    double sums = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double other = __shfl_up_sync(kAll, sums, o);
      if (lane >= o) sums += other;
    }
    if (lane == 31) sh.warp_sum[warp] = sums;
    __syncthreads();
    double before = start;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    for (int w = 0; w < kWarps; ++w) start += sh.warp_sum[w];
    // one thread's start is the end of the one before it, so that one at most has the target
    const double left = __shfl_up_sync(kAll, sums, 1);
    double c = lane ? before + left : before;
    if (c <= target && before + sums > target) {
      int best = 0;
      double best_y = 0.0;
      bool past = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        c += y[i];
        if (y[i] > 0.0 && !past) {
          best = part.base + v * N + i, best_y = y[i];
          past = c > target;
        }
      }
      hit = best;
      a.tokens[row] = best;
      a.logp[row] = static_cast<float>(log(best_y / all));
    }
    __syncthreads();
    if (hit >= 0) return;
  }
  sample_rare_row<T>(a, sh, row);  // rounding has left no column
}

template <class T>
int launch_sample(Arguments a, int rows, int sms, cudaStream_t stream) {
  if (!a.top_k && !a.top_p && !a.min_p && (a.top_k_all == 0 || a.top_k_all >= a.vocab) &&
      a.top_p_all >= 1.0f && a.min_p_all == 0.0f && rows >= kDrawRows)
    return pg::launch<draw_kernel<T>>("draw_kernel", dim3(rows), kThreads, 0, stream, a);
  // Blocks a row: as many as let a part stay in shared memory, and more where that leaves SMs
  // without any, but no part shorter than one vector a thread.
  const auto part_bytes = [&](int blocks) {
    return (static_cast<int64_t>(a.vocab) + blocks - 1) / blocks * sizeof(T) + 48;
  };
  int blocks = 1;
  while (blocks < kParts && (part_bytes(blocks) > kResident ||
                             (rows * 2ll * blocks <= kPerSm * sms &&
                              a.vocab / (2 * blocks) >= kThreads * Vec<T>::n)))
    blocks *= 2;
  const int64_t bytes = part_bytes(blocks);
  a.resident = bytes <= kResident;
  static std::atomic<uint64_t> done{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return pg::runtime_fail(e, "sample_kernel");
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(reinterpret_cast<const void *>(sample_kernel<T>),
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kResident);
    if (e != cudaSuccess) return pg::runtime_fail(e, "sample_kernel");
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = a.resident ? static_cast<size_t>((bytes + 15) / 16 * 16) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {static_cast<unsigned>(blocks), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
  return e == cudaSuccess ? PG_OK : pg::runtime_fail(e, "sample_kernel");
}

}  // namespace

extern "C" int pg_sample(const pg_sample_args *p, uint64_t stream) {
  if (!p) return pg::argument_fail("pg_sample: null arguments");
  const unsigned size = p->dtype == PG_DT_F32 ? 4 : 2;
  if (p->dtype != PG_DT_F32 && p->dtype != PG_DT_BF16 && p->dtype != PG_DT_F16)
    return pg::argument_fail("pg_sample: dtype %d, want f32, bf16 or f16", p->dtype);
  if (p->rows < 0 || p->rows > INT32_MAX / kParts || p->vocab < 1 || p->vocab > INT32_MAX / 2 ||
      (p->rows > 1 && p->row_stride < p->vocab))
    return pg::argument_fail("pg_sample: %d rows of %d logits, %lld apart", p->rows, p->vocab,
                             static_cast<long long>(p->row_stride));
  if ((!p->temperature && !(p->temperature_all >= 0.0f)) ||
      (!p->top_p && !(p->top_p_all > 0.0f && p->top_p_all <= 1.0f)) ||
      (!p->min_p && !(p->min_p_all >= 0.0f && p->min_p_all <= 1.0f)) ||
      (!p->top_k && p->top_k_all < 0))
    return pg::argument_fail("pg_sample: temperature %g, top_k %d, top_p %g, min_p %g: want at "
                             "least 0, at least 0, 0 to 1 without 0, 0 to 1", p->temperature_all,
                             p->top_k_all, p->top_p_all, p->min_p_all);
  if (!p->rows) return PG_OK;
  if (!p->logits || !p->uniform || !p->tokens || !p->logp || p->logits % size ||
      ((p->uniform | p->temperature | p->top_k | p->top_p | p->min_p | p->logp) & 3) ||
      (p->tokens & 7))
    return pg::argument_fail("pg_sample: an argument is null or misaligned");
  int sms;
  const int rc = pg::sm_count(&sms);
  if (rc) return rc;
  Arguments a = {};
  a.logits = reinterpret_cast<const void *>(p->logits);
  a.uniform = reinterpret_cast<const float *>(p->uniform);
  a.temperature = reinterpret_cast<const float *>(p->temperature);
  a.top_k = reinterpret_cast<const int *>(p->top_k);
  a.top_p = reinterpret_cast<const float *>(p->top_p);
  a.min_p = reinterpret_cast<const float *>(p->min_p);
  a.tokens = reinterpret_cast<int64_t *>(p->tokens);
  a.logp = reinterpret_cast<float *>(p->logp);
  a.row_stride = p->row_stride;
  a.vocab = p->vocab;
  a.temperature_all = p->temperature_all, a.top_k_all = p->top_k_all;
  a.top_p_all = p->top_p_all, a.min_p_all = p->min_p_all;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(stream));
  return p->dtype == PG_DT_F32    ? launch_sample<float>(a, p->rows, sms, s)
         : p->dtype == PG_DT_BF16 ? launch_sample<__nv_bfloat16>(a, p->rows, sms, s)
                                  : launch_sample<__half>(a, p->rows, sms, s);
}

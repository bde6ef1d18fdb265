// Log probabilities of given tokens, the distribution's entropy and its top alternatives, and
// the gradient of the first two (pg_logprobs, pg_logprobs_grad in include/ptxgen_b200.h).
//
// With m the row's largest logit, s = sum exp(x - m) and t = sum (x - m) exp(x - m):
//   log p_j = (x_j - m) - log s,  entropy H = log s - t / s,
//   d x_j = a ([j = token] - p_j) - b p_j (log p_j + H)   for gradients a of log p_token, b of H.
// One pass keeps m, s and t in 32 bits a thread (t in powers of two), rescaling s and t when m
// grows:
//   s' = s f,  t' = (t + (m - m') s) f,  f = exp(m - m').
// x - m is cut off where exp is 0 long since, so a logit of -inf adds 0 to t and not 0 * inf; m
// starts at the lowest finite number, so a row of lowest numbers is an even distribution and only
// a row of nothing but -inf (s = 0) has none: it gives NaN, as does a row with a NaN or +inf. The
// gradient goes by the pair (m, log s), not by their sum, which would lose log s beside a large m.
#include "common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

// Small blocks, not a few large ones: one's sums and selection meet the others' loads (four of 256
// threads an SM against two of 512, 4096 x 50257 in bf16: 85 us against 110).
constexpr int kOnSm = 1024;          // threads of the forward kernel that an SM holds
// Threads of the gradient's blocks: short rows leave less of a small one idle (forward and gradient
// of 3682 x 1718 in f16: 20.5 us with 128, 25.7 with 256; 4096 x 50257 in bf16: 207 and 209).
constexpr int kThreads = 128;
constexpr int kBatch = 4;            // 16-byte loads a thread has in flight
constexpr int kTopMax = PG_LOGPROB_TOP;
constexpr int kParts = 8;            // blocks a row is cut in at most (a portable cluster)
constexpr int kCandidates = 1024;    // elements the selection of the top ones may look at
constexpr float kLowest = -3.402823466e38f;
constexpr float kCut = -1e4f;        // of x - m in powers of two, below which exp is 0
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

// ... with results below 2^-126 kept
__device__ __forceinline__ float exp2_small(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <class T> struct Vec;  // 16 bytes of T as f32
template <> struct Vec<float> {
  static constexpr int n = 4;
  static constexpr bool small = true;  // holds numbers near 2^-126
  __device__ static void get(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 put(const float *x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr bool small = true;
  __device__ static void get(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 put(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static constexpr bool small = false;
  __device__ static void get(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  __device__ static uint4 put(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, float *to) { *to = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16 *to) {
  *to = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void from_float(float x, __half *to) { *to = __float2half_rn(x); }

// Row sums: the largest logit m, and with d = (x - m) log2 e the sums of 2^d and of d 2^d.
struct Sums {
  float m, s, t;
};

__device__ __forceinline__ void rescale(Sums &a, float m) {
  const float d = max_nan((a.m - m) * kLog2e, kCut), f = exp2_fast(d);
  a.t = (a.t + d * a.s) * f;
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = max_nan(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  a.s += b.s;
  a.t += b.t;
  return a;
}

// One vector more. The subtraction comes before the scaling, so that it is exact for the large
// numbers of a mask; two at a time otherwise, since instructions bound this, not memory.
template <int N>
__device__ __forceinline__ void add(Sums &a, const float *x) {
  float top = a.m;
#pragma unroll
  for (int i = 0; i < N; i += 2) top = pg::max3(top, x[i], x[i + 1]);
  if (top != a.m) rescale(a, top);
  const pg::Two m(-a.m, -a.m), scale(kLog2e, kLog2e);
  pg::Two s(a.s, 0.0f), t(a.t, 0.0f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float d, e;
    mul(add(pg::Two(x[i], x[i + 1]), m), scale).get(d, e);
    d = max_nan(d, kCut);
    e = max_nan(e, kCut);
    const pg::Two p(exp2_fast(d), exp2_fast(e));
    s = add(s, p);
    t = fma(pg::Two(d, e), p, t);
  }
  float u, v;
  s.get(u, v);
  a.s = u + v;
  t.get(u, v);
  a.t = u + v;
}

// A key whose order as a whole number is the logits' order, NaN above all, -0 equal to 0; 0 is
// no logit's key.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// ... and of a logit at a column, ties to the lowest column.
__device__ __forceinline__ uint64_t entry_of(float x, int column) {
  return static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~column);
}

// One block's part of a row, columns [first, last): thread i takes the 16-byte vectors i, i +
// THREADS, ... of the part that are aligned, counted from the aligned address at or below its
// start; columns outside the part read as -inf.
template <class T>
struct Part {
  const T *row;
  int first, last, base, vectors;  // base: the column of vector 0 (it may lie below first)

  __device__ Part(const T *r, int a, int b) : row(r), first(a), last(b) {
    const int over = static_cast<int>(
        (reinterpret_cast<uintptr_t>(r + a) & 15) / sizeof(T));
    base = a - over;
    vectors = b > a ? (b - base + Vec<T>::n - 1) / Vec<T>::n : 0;
  }
  __device__ bool whole(int v) const {
    return base + v * Vec<T>::n >= first && base + (v + 1) * Vec<T>::n <= last;
  }
  __device__ void load(int v, float *x) const {
    const int at = base + v * Vec<T>::n;
    if (whole(v)) {
      Vec<T>::get(pg::load16(row + at), x);
      return;
    }
#pragma unroll
    for (int i = 0; i < Vec<T>::n; ++i)
      x[i] = at + i >= first && at + i < last ? to_float(row[at + i]) : -INFINITY;
  }
};

template <int THREADS>
struct Shared {
  Sums warp[THREADS / 32];
  Sums row;                          // the part's sums
  Sums part[kParts];                 // the parts' sums
  uint32_t chosen[THREADS];         // the threads whose strips are looked at again
  uint64_t found[kCandidates];
  uint64_t top[kTopMax];             // the part's top entries, best first; 0 where there is none
  uint64_t best;
  uint64_t warp_best[THREADS / 32];
  int chosen_n, found_n;
};

// The part's `k` largest entries into sh.top. Each thread's largest logit is known from the sums;
// with T at most the k-th largest of those, at least k elements are T or above, and every one of them
// lies in the strip of a thread whose largest is. So only those few strips are read again (from
// L2, a warp to a strip, one load a lane where a strip is short), and what reaches T is ranked by
// counting. Where more than kCandidates reach it (many equal logits), the entries are taken one
// at a time instead, each the largest below the last.
template <class T, int THREADS>
__device__ void select_top(const Part<T> &part, float mine, bool any, int k,
                           Shared<THREADS> &sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t key = any ? key_of(mine) : 0;
  if (tid == 0) sh.chosen_n = sh.found_n = 0;
  if (tid < kTopMax) sh.top[tid] = 0;
  // A t with at least k threads at t or above, near the largest such: 2^13 of a key is 2^-10 of a
  // logit, so it lets few more in. Mostly all k are within four binades of the largest one.
  __syncthreads();
  const uint32_t top = key_of(sh.row.m), near = top > 1u << 25 ? top - (1u << 25) : 0;
  uint32_t t = 0;
  int bit = 31;
  if (__syncthreads_count(key >= near) >= k) t = near, bit = 24;
  for (; bit >= 13; --bit)
    if (__syncthreads_count(key >= t + (1u << bit)) >= k) t += 1u << bit;
  if (any && key >= t) sh.chosen[atomicAdd(&sh.chosen_n, 1)] = tid;
  __syncthreads();
  const int strips = sh.chosen_n;
  for (int c = warp; c < strips; c += THREADS / 32)
    for (int v = sh.chosen[c] + lane * THREADS; v < part.vectors; v += 32 * THREADS) {
      float x[Vec<T>::n];
      part.load(v, x);
      const int at = part.base + v * Vec<T>::n;
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i)
        if (key_of(x[i]) >= t && at + i >= part.first && at + i < part.last) {
          const int slot = atomicAdd(&sh.found_n, 1);
          if (slot < kCandidates) sh.found[slot] = entry_of(x[i], at + i);
        }
    }
  __syncthreads();
  const int n = sh.found_n;
  if (n <= kCandidates) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t e = sh.found[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.found[j] > e;
      if (rank < k) sh.top[rank] = e;
    }
    __syncthreads();
    return;
  }
  uint64_t below = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int v = tid; v < part.vectors; v += THREADS) {
      float x[Vec<T>::n];
      part.load(v, x);
      const int at = part.base + v * Vec<T>::n;
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i) {
        const uint64_t e = entry_of(x[i], at + i);
        if (e < below && e > best && at + i >= part.first && at + i < part.last) best = e;
      }
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    if (lane == 0) sh.warp_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < THREADS / 32; ++w) best = sh.warp_best[w] > best ? sh.warp_best[w] : best;
      sh.best = sh.top[r] = best;
    }
    __syncthreads();
    below = sh.best;
    if (!below) break;  // the part has no more
  }
  __syncthreads();
}

// One cluster of blocks a row; block r of it takes the r-th part. 4096 x 50257 in bf16 take 78 us (5.3
// TB/s); 1000 x 128256 with the top 20 68 us (3.8 TB/s), with issue at 56 %, special functions at 47 %
// and DRAM at 53 % of what they can: 1000 blocks are 1.7 waves of what the SMs hold, and rows that have
// left L2 are read again for their top entries. At few rows the parts keep all SMs
// reading and latency bounds it: 4 x 32001 in f32 with the top 5 take 8 us.
template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS, kOnSm / THREADS)
    logprobs_kernel(const T *logits, int64_t row_stride, const void *tokens, int token_bytes,
                    int vocab, int top, float *logp, float *entropy, float2 *norm,
                    float *top_logp, int32_t *top_ids) {
  __shared__ Shared<THREADS> sh;
  pg::wait_for_earlier_kernels();
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *x_row = logits + row * row_stride;
  const int64_t v64 = vocab;
  const Part<T> part(x_row, static_cast<int>(v64 * rank / parts),
                     static_cast<int>(v64 * (rank + 1) / parts));
  Sums mine{kLowest, 0.0f, 0.0f};
  int v = tid;
  // whole batches, the next one's loads on their way while one is added up
  const auto batch_here = [&](int at) {
    return at + (kBatch - 1) * THREADS < part.vectors && part.whole(at) &&
           part.whole(at + (kBatch - 1) * THREADS);
  };
  const T *const vectors = part.row + part.base;
  if (v < part.vectors && !part.whole(v)) {  // the first vector may start before the part
    float x[Vec<T>::n];
    part.load(v, x);
    add<Vec<T>::n>(mine, x);
    v += THREADS;
  }
  if (batch_here(v)) {
    uint4 raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      raw[u] = pg::load16(vectors + static_cast<int64_t>(v + u * THREADS) * Vec<T>::n);
    for (bool more = true; more;) {
      v += kBatch * THREADS;
      more = batch_here(v);
      uint4 next[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (more) next[u] = pg::load16(vectors + static_cast<int64_t>(v + u * THREADS) * Vec<T>::n);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        float x[Vec<T>::n];
        Vec<T>::get(raw[u], x);
        add<Vec<T>::n>(mine, x);
        raw[u] = next[u];
      }
    }
  }
  for (; v < part.vectors; v += THREADS) {
    float x[Vec<T>::n];
    part.load(v, x);
    add<Vec<T>::n>(mine, x);
  }
  // a thread that met nothing but -inf has added nothing
  const float largest = mine.s == 0.0f ? -INFINITY : mine.m;
  const bool any = tid < part.vectors;
  Sums all = mine;
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    Sums o;
    o.m = __shfl_xor_sync(0xffffffffu, all.m, off);
    o.s = __shfl_xor_sync(0xffffffffu, all.s, off);
    o.t = __shfl_xor_sync(0xffffffffu, all.t, off);
    all = join(all, o);
  }
  if (lane == 0) sh.warp[warp] = all;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < THREADS / 32; ++w) all = join(all, sh.warp[w]);
    sh.row = all;
  }
  if (top) select_top(part, largest, any, top, sh);
  if (parts > 1) {
    // the first block copies the others' sums and lists, and only then do those end
    cluster.sync();
    if (rank == 0) {
      if (tid < parts) sh.part[tid] = cluster.map_shared_rank(&sh, tid)->row;
      for (int i = tid; i < parts * top; i += THREADS)
        sh.found[i] = cluster.map_shared_rank(&sh, i / top)->top[i % top];
    }
    cluster.sync();
    if (rank) return;
  } else {
    if (tid < top) sh.found[tid] = sh.top[tid];
    if (tid == 0) sh.part[0] = all;
    __syncthreads();
  }
  // every thread joins the parts' sums in the same order
  Sums r = sh.part[0];
  for (int p = 1; p < parts; ++p) r = join(r, sh.part[p]);
  const float log_s = logf(r.s);
  const bool none = r.s == 0.0f;
  if (tid == 0) {
    const int64_t token = token_bytes == 8 ? static_cast<const int64_t *>(tokens)[row]
                                           : static_cast<const int32_t *>(tokens)[row];
    float lp = 0.0f;
    if (token != -1)
      lp = token < 0 || token >= vocab || none ? NAN : (to_float(x_row[token]) - r.m) - log_s;
    logp[row] = lp;
    entropy[row] = none ? NAN : log_s - kLn2 * (r.t / r.s);
    norm[row] = make_float2(r.m, log_s);
  }
  for (int i = tid; i < parts * top; i += THREADS) {
    const uint64_t e = sh.found[i];
    int place = 0;
    for (int j = 0; j < parts * top; ++j) place += sh.found[j] > e;
    if (e && place < top) {
      const int64_t at = static_cast<int64_t>(row) * top + place;
      top_ids[at] = static_cast<int32_t>(~static_cast<uint32_t>(e));
      top_logp[at] = none ? NAN : (logit_of(static_cast<uint32_t>(e >> 32)) - r.m) - log_s;
    }
  }
}

// Reads each logit once and writes its gradient; HBM bounds it: 4096 x 50257 in bf16 take 127 us
// (6.5 TB/s). Rows go last to first, so that those a forward pass over the same logits read last
// are still in L2.
template <class T>
__global__ void __launch_bounds__(kThreads)
    logprobs_grad_kernel(const T *logits, int64_t row_stride, const void *tokens, int token_bytes,
                         int rows, int vocab, const float2 *norm, const float *entropy,
                         const float *d_logp, const float *d_entropy, T *out, int64_t out_stride,
                         int per_row) {
  constexpr int n = Vec<T>::n, span = n * kThreads * kBatch;
  pg::wait_for_earlier_kernels();
  const int row = rows - 1 - blockIdx.x / per_row;
  const int piece = blockIdx.x % per_row;
  const T *x_row = logits + row * row_stride;
  T *y_row = out + row * out_stride;
  const int64_t token = token_bytes == 8 ? static_cast<const int64_t *>(tokens)[row]
                                         : static_cast<const int32_t *>(tokens)[row];
  const float2 l = norm[row];
  const float h = entropy[row];
  float a = d_logp && token != -1 ? d_logp[row] : 0.0f;
  if (token < -1 || token >= vocab) a = NAN;
  const float b = d_entropy ? d_entropy[row] : 0.0f;
  const float c = fmaf(b, h, a);
  // -p (a + b (log p + H)) of two columns; the token's a is added after. Probabilities below
  // 2^-126 become 0 but for f32 and bf16 results, which can hold such numbers times a large factor.
  const pg::Two m(-l.x, -l.x), log_s(-l.y, -l.y), scale(kLog2e, kLog2e), b2(-b, -b), c2(-c, -c);
  const auto grad = [&](float &x, float &y) {
    add(add(pg::Two(x, y), m), log_s).get(x, y);
    const pg::Two lp(max_nan(x, kCut), max_nan(y, kCut));
    mul(lp, scale).get(x, y);
    const pg::Two p = Vec<T>::small ? pg::Two(exp2_small(x), exp2_small(y))
                                    : pg::Two(exp2_fast(x), exp2_fast(y));
    mul(p, fma(b2, lp, c2)).get(x, y);
  };
  const auto grad_one = [&](int column) {
    float x = to_float(x_row[column]), y = x;
    grad(x, y);
    from_float(column == token ? x + a : x, y_row + column);
  };
  const int over_x = static_cast<int>((reinterpret_cast<uintptr_t>(x_row) & 15) / sizeof(T));
  const int over_y = static_cast<int>((reinterpret_cast<uintptr_t>(y_row) & 15) / sizeof(T));
  const int first = piece * span - over_x;  // a vector boundary of the logits
  if (over_x == over_y) {
    uint4 raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = first + (u * kThreads + static_cast<int>(threadIdx.x)) * n;
      if (at >= 0 && at + n <= vocab) raw[u] = pg::load16(x_row + at);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = first + (u * kThreads + static_cast<int>(threadIdx.x)) * n;
      if (at >= 0 && at + n <= vocab) {
        float x[n];
        Vec<T>::get(raw[u], x);
#pragma unroll
        for (int i = 0; i < n; i += 2) grad(x[i], x[i + 1]);
        const int64_t here = token - at;
        if (here >= 0 && here < n) {
#pragma unroll
          for (int i = 0; i < n; ++i)
            if (i == here) x[i] += a;
        }
        *reinterpret_cast<uint4 *>(y_row + at) = Vec<T>::put(x);
      } else {
        for (int i = 0; i < n; ++i)
          if (at + i >= 0 && at + i < vocab)
            grad_one(at + i);
      }
    }
    return;
  }
  // logits and gradients lie differently on 16-byte boundaries: one element at a time
  for (int at = first + static_cast<int>(threadIdx.x); at < first + span; at += kThreads)
    if (at >= 0 && at < vocab) grad_one(at);
}

template <class T, int THREADS>
int launch_logprobs(uint64_t logits, int64_t row_stride, uint64_t tokens, int token_bytes,
                    int rows, int vocab, int top, int sms, uint64_t logp, uint64_t entropy,
                    uint64_t norm, uint64_t top_logp, uint64_t top_ids, cudaStream_t stream) {
  // blocks a row: as many as the SMs hold at once, up to a portable cluster, and no part
  // shorter than one load of each thread
  int parts = 1;
  const int least = THREADS * Vec<T>::n, most = kOnSm / THREADS * sms;
  while (parts < kParts && rows * 2ll * parts <= most && vocab / (2 * parts) >= least) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * parts);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(
      &cfg, logprobs_kernel<T, THREADS>, reinterpret_cast<const T *>(logits), row_stride,
      reinterpret_cast<const void *>(tokens), token_bytes, vocab, top,
      reinterpret_cast<float *>(logp), reinterpret_cast<float *>(entropy),
      reinterpret_cast<float2 *>(norm), reinterpret_cast<float *>(top_logp),
      reinterpret_cast<int32_t *>(top_ids));
  return e == cudaSuccess ? PG_OK : pg::runtime_fail(e, "logprobs_kernel");
}

template <class T>
int run_logprobs(uint64_t logits, int64_t row_stride, uint64_t tokens, int token_bytes, int rows,
                 int vocab, int top, uint64_t logp, uint64_t entropy, uint64_t norm,
                 uint64_t top_logp, uint64_t top_ids, cudaStream_t stream) {
  int sms;
  int rc = pg::sm_count(&sms);
  if (rc) return rc;
  // Blocks of 128 threads where they fill the GPU, since a row's sums are joined sooner, but not
  // where the top entries of long rows are asked for: a thread's strip is read again for each it
  // may hold. 128 against 256, in microseconds: 3682 x 1718 with the gradient 26 and 32, 4096 x 50257
  // 207 and 213, 600 x 2000 9.2 and 8.8; with top entries 4000 x 25000 56 and 70, 3000 x 32000 62 and
  // 72, 1500 x 64000 67 and 57, 300 x 8000 11.6 and 9.1.
  const auto launch = rows > 8 * sms && (!top || vocab <= 32768) ? launch_logprobs<T, 128>
                                                                 : launch_logprobs<T, 256>;
  return launch(logits, row_stride, tokens, token_bytes, rows, vocab, top, sms, logp, entropy, norm,
                top_logp, top_ids, stream);
}

template <class T>
int run_grad(uint64_t logits, int64_t row_stride, uint64_t tokens, int token_bytes, int rows,
             int vocab, uint64_t norm, uint64_t entropy, uint64_t d_logp, uint64_t d_entropy,
             uint64_t out, int64_t out_stride, cudaStream_t stream) {
  constexpr int span = Vec<T>::n * kThreads * kBatch;
  // a row may start in the middle of its first vector
  const int per_row = (vocab + Vec<T>::n - 2) / span + 1;
  return pg::launch<logprobs_grad_kernel<T>>(
      "logprobs_grad_kernel", dim3(static_cast<unsigned>(rows) * per_row), kThreads, 0, stream,
                    reinterpret_cast<const T *>(logits), row_stride,
                    reinterpret_cast<const void *>(tokens), token_bytes, rows, vocab,
                    reinterpret_cast<const float2 *>(norm), reinterpret_cast<const float *>(entropy),
                    reinterpret_cast<const float *>(d_logp),
                    reinterpret_cast<const float *>(d_entropy), reinterpret_cast<T *>(out),
                    out_stride, per_row);
}

int check(const char *what, uint64_t logits, int64_t row_stride, int dtype, uint64_t tokens,
          int token_bytes, int32_t rows, int32_t vocab) {
  const unsigned size = dtype == PG_DT_F32 ? 4 : 2;
  if (dtype != PG_DT_F32 && dtype != PG_DT_BF16 && dtype != PG_DT_F16)
    return pg::argument_fail("%s: dtype %d, want f32, bf16 or f16", what, dtype);
  if (rows < 0 || vocab < 1 || vocab > INT32_MAX / 2 || (rows > 1 && row_stride < vocab))
    return pg::argument_fail("%s: %d rows of %d logits, %lld apart", what, rows, vocab,
                             static_cast<long long>(row_stride));
  if (token_bytes != 4 && token_bytes != 8)
    return pg::argument_fail("%s: tokens of %d bytes, want 4 or 8", what, token_bytes);
  if (rows && (!logits || !tokens || logits % size || tokens % token_bytes))
    return pg::argument_fail("%s: logits or tokens null or misaligned", what);
  return PG_OK;
}

inline cudaStream_t stream_of(uint64_t s) {
  return reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(s));
}

}  // namespace

extern "C" int pg_logprobs(uint64_t logits, int64_t row_stride, int32_t dtype, uint64_t tokens,
                           int32_t token_bytes, int32_t rows, int32_t vocab, int32_t top,
                           uint64_t logp, uint64_t entropy, uint64_t norm, uint64_t top_logp,
                           uint64_t top_ids, uint64_t stream) {
  int rc = check("pg_logprobs", logits, row_stride, dtype, tokens, token_bytes, rows, vocab);
  if (rc) return rc;
  if (top < 0 || top > kTopMax || top > vocab)
    return pg::argument_fail("pg_logprobs: top %d of %d logits, want 0..%d", top, vocab, kTopMax);
  if (rows > INT32_MAX / 8) return pg::argument_fail("pg_logprobs: %d rows", rows);
  if (!rows) return PG_OK;
  if (!logp || !entropy || !norm || (top && (!top_logp || !top_ids)) ||
      ((logp | entropy | top_logp | top_ids) & 3) || (norm & 7))
    return pg::argument_fail("pg_logprobs: an output is null or misaligned");
  const auto run = dtype == PG_DT_F32    ? run_logprobs<float>
                   : dtype == PG_DT_BF16 ? run_logprobs<__nv_bfloat16>
                                         : run_logprobs<__half>;
  return run(logits, row_stride, tokens, token_bytes, rows, vocab, top, logp, entropy, norm,
             top_logp, top_ids, stream_of(stream));
}

extern "C" int pg_logprobs_grad(uint64_t logits, int64_t row_stride, int32_t dtype,
                                uint64_t tokens, int32_t token_bytes, int32_t rows, int32_t vocab,
                                uint64_t norm, uint64_t entropy, uint64_t d_logp,
                                uint64_t d_entropy, uint64_t out, int64_t out_stride,
                                uint64_t stream) {
  int rc = check("pg_logprobs_grad", logits, row_stride, dtype, tokens, token_bytes, rows, vocab);
  if (rc) return rc;
  const unsigned size = dtype == PG_DT_F32 ? 4 : 2;
  if (rows > 1 && out_stride < vocab)
    return pg::argument_fail("pg_logprobs_grad: output rows %lld apart, %d long",
                             static_cast<long long>(out_stride), vocab);
  if (static_cast<int64_t>(rows) * (vocab / (kThreads * kBatch * 4) + 2) > INT32_MAX)
    return pg::argument_fail("pg_logprobs_grad: %d rows of %d logits", rows, vocab);
  if (!rows) return PG_OK;
  if (!norm || !entropy || !out || ((entropy | d_logp | d_entropy) & 3) || (norm & 7) || out % size)
    return pg::argument_fail("pg_logprobs_grad: an argument is null or misaligned");
  const auto run = dtype == PG_DT_F32    ? run_grad<float>
                   : dtype == PG_DT_BF16 ? run_grad<__nv_bfloat16>
                                         : run_grad<__half>;
  return run(logits, row_stride, tokens, token_bytes, rows, vocab, norm, entropy, d_logp,
             d_entropy, out, out_stride, stream_of(stream));
}

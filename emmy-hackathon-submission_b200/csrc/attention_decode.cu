// Attention of one new token a sequence, or a few, at head sizes of up to 128 (pg_attention).
//
// HBM bounds it: every key and value is read once and used for the query heads of its group
// only. So the work is cut evenly by keys, not by sequences: the blocks of 64 keys of all
// (sequence, kv head) pairs form one line, each pair with a few more for what it costs by itself,
// and block c takes the c-th of as many equal pieces of it as there are blocks. A pair whose keys
// lie in several pieces is joined by the last block that finishes one, in the pieces' order. 48
// sequences of up to 32768 keys, 64 heads on 8 of 128 in bf16, take 355 us (6.0 TB/s).
//
// Within a block each of four warps takes every fourth 16 keys by itself: it copies their rows
// into its own ring in shared memory (cp.async, 16 bytes a lane, rows of whole heads, swizzled so
// that the matrix loads meet no bank twice), and multiplies on the tensor cores (mma.sync
// m16n8k16: with at most 16 rows of queries a larger tile would be empty, and at one use of each
// key the memory is slower by far). A weight goes into the second product as the sum of two
// numbers of the values' type, the rounded weight and what the rounding left, so that the result
// is rounded once; that doubles the second product, which the memory hides. In f16, which has
// nothing below 2^-24, weights and their sum are 2^15 of what they are.
//
// f32 goes the same way by eights of keys (m16n8k8, TF32). A factor x of either product is taken as
// hi, 11 bits of it, and lo, 11 bits of the rest, and hi hi' + hi lo' + lo hi' is summed. Left out
// are lo lo' and the roundings of lo: up to 2^-22 and 2^-23 of a product, of either sign, since lo is
// rounded and one factor's hi too. A step's weighted values are summed apart and then added in f32:
// the tensor cores do not round their sums to nearest, and over 1000s of steps that alone put
// results 5e-6 off (24 sequences of up to 40000 keys; 3.3e-7 so, 4.2e-7 by f32 FMA). A factor that
// is not finite has no two parts: scores that come out as NaN are made anew by plain products, and
// values are looked through at every step. 32 sequences of up to 8000 keys, 64 heads on 8 of 128,
// take 265 us (3.4 TB/s), bound by the instructions' latency at two warps a scheduler; 32-bit FMA
// from shared memory took 735.
//
// Several queries' heads make more rows, 16 to a pair of their own, so each of their groups of 16
// reads the keys again, from L2. What some row of a step must not see has weight 0 there; values
// that are not finite are zeroed in such steps, and added again at the end for rows that see them. In
// the other steps they meet both parts of a weight, the second of which may be 0 or negative: a result
// that is not finite has the visible values looked through and is made of those that are not.
#include "attention.cuh"

namespace {

using pg::Attention;
using pg::Blocks;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRows = 16;
constexpr int kPerSm = 2;             // blocks an SM holds
// What a pair costs by itself, in blocks of keys (64 sequences of up to 8000 keys on 8 kv heads:
// 126 us with 8 or 4, 159 with 0).
constexpr int kPair = 8;
constexpr float kCut = 2.0f;

template <class T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static constexpr float shift = 0.0f;  // weights go in as 2^shift of what they are
  __device__ static void run(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t exponent = 0x7f80;
  __device__ static float low(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ static float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  // two weights rounded, and the two that rounding left
  __device__ static void split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 l =
        __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  }
  __device__ static uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};
template <> struct Mma<__half> {
  static constexpr float shift = 15.0f;  // at most 2^15 of 65504
  static constexpr uint32_t exponent = 0x7c00;
  __device__ static float low(uint32_t w) {
    return __low2float(*reinterpret_cast<const __half2 *>(&w));
  }
  __device__ static float high(uint32_t w) {
    return __high2float(*reinterpret_cast<const __half2 *>(&w));
  }
  __device__ static void run(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static void split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  }
  __device__ static uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};

template <> struct Mma<float> {
  static constexpr float shift = 0.0f;
  __device__ static void run(float *d, const uint32_t *a, const uint32_t *b) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
  __device__ static uint32_t nearest(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
  }
  // a key or value: the 11 leading bits, which the largest number has too, and what is left
  __device__ static void split(float x, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = nearest(x - __uint_as_float(hi));
  }
  // a query's number or a weight: rounded, so that what is left has either sign
  __device__ static void split_near(float x, uint32_t &hi, uint32_t &lo) {
    hi = nearest(x);
    lo = nearest(x - __uint_as_float(hi));
  }
};

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool real) {
  const int bytes = real ? 16 : 0;  // 0: the 16 bytes are zeroed and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t at, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <class T, int DIM>
struct Ring {
  static constexpr int size = sizeof(T);
  static constexpr int row = DIM * size, chunks = row / 16;
  static constexpr int step = 32 / size;          // keys a warp takes at a time
  static constexpr int keys = step * kWarps;      // keys of a block's step
  static constexpr int tile = step * row;         // a warp's keys, or values
  static constexpr int stage = 2 * tile;
  static constexpr int stages = (size == 4 ? 256 : 384) / DIM;
  static constexpr int warp = stages * stage;
  // f32: the queries' fragments in their two parts, of which registers have no room for one
  static constexpr int q = kWarps * warp, q_part = size == 4 ? 16 * row : 0;
  static constexpr int bytes = q + 2 * q_part;
  static_assert(warp >= kRows * (DIM + 2) * 4, "a warp's result takes its ring's place");
  __device__ static int at(int r, int chunk) { return r * row + ((chunk ^ (r & 7)) << 4); }
};

// A sequence as the kernel takes it: `count` queries from row `query` on, the last of `length`
// tokens, which makes `pairs` of a head and 16 rows.
struct Sequence {
  int slot, length, query, count, row_groups;
  Blocks blocks;
  uint32_t pairs;
};

template <bool MANY, int KEYS>
__device__ __forceinline__ Sequence sequence_of(const Attention &a, int b) {
  Sequence s;
  s.slot = a.slots ? a.slots[b] : b;
  s.query = MANY ? a.starts[b] : b;
  s.count = MANY ? max(0, a.starts[b + 1] - s.query) : 1;
  s.length = 0;
  if (MANY && (s.query < 0 || s.count > a.queries - s.query)) {
    atomicOr(a.status, PG_CACHE_TOO_LONG);
    s.count = 0;
  }
  if (s.slot < 0 || s.slot >= a.slot_rows) {
    atomicOr(a.status, PG_CACHE_BAD_SLOT);
  } else {
    const int most = a.width * a.page_size;
    s.length = a.lens[s.slot];
    if (s.length < 0 || s.length > most) {
      atomicOr(a.status, PG_CACHE_TOO_LONG);
      s.length = s.length < 0 ? 0 : most;
    }
  }
  s.row_groups = (s.count * a.group + kRows - 1) / kRows;
  s.blocks = pg::blocks_of(a, s.length - s.count, s.length - 1, KEYS);
  s.pairs = s.blocks.count ? a.heads * s.row_groups : 0;
  return s;
}

// A pair of a kv head and 16 rows, as far as a block has a piece of it.
struct Pair {
  int query, row0, rows, head, lo, hi;  // lo..hi: the positions of the sequence's queries
  int block0, block1;                   // of its blocks of keys
  uint32_t first, c0, c1;               // its place on the line, the pieces that it lies in
  Blocks blocks;
  const int *pages;
  unsigned last;
  // whether all rows see all of a step's keys
  template <int STEP>
  __device__ bool all_see(const Attention &a, int key) const {
    return key + STEP - 1 <= lo &&
           (!a.window || key > hi - a.window || key + STEP <= a.sinks);
  }
};

// Four numbers of T at an address, or to it.
template <class T>
__device__ __forceinline__ float4 load4(const char *at) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4 *>(at);
  } else {
    const uint2 w = *reinterpret_cast<const uint2 *>(at);
    return make_float4(Mma<T>::low(w.x), Mma<T>::high(w.x), Mma<T>::low(w.y), Mma<T>::high(w.y));
  }
}
template <class T>
__device__ __forceinline__ void store4(char *at, float4 x) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4 *>(at) = x;
  else
    *reinterpret_cast<uint2 *>(at) = make_uint2(Mma<T>::pack(x.x, x.y), Mma<T>::pack(x.z, x.w));
}

// q . k with k a row of a stage, one product after another.
template <class R>
__device__ __noinline__ float plain_product(const char *q, const char *stage, int row, int dim) {
  float sum = 0.0f;
  for (int c = 0; c < dim / 4; ++c) {
    const float4 x = *reinterpret_cast<const float4 *>(q + 16 * c);
    const float4 y = *reinterpret_cast<const float4 *>(stage + R::at(row, c));
    sum = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, sum))));
  }
  return sum;
}

// What the warps of a block have of a pair, from their rings' places: joined, and written as the
// result, or left for the block that finishes the pair last, which joins all. A function of its own
// for the registers: what is needed here only would otherwise be held through the loop over the
// keys, whose loads of operands then wait for one another (a tenth of the whole).
template <class T, int DIM, bool MANY>
__device__ __noinline__ void finish_pair(const Attention &a, Pair &sh, uint32_t per, int odd) {
  using R = Ring<T, DIM>;
  extern __shared__ float4 smem4[];
  const Pair p = sh;
  const int tid = threadIdx.x;
  const auto query_of = [&](int r) { return MANY ? (p.row0 + r) / a.group : 0; };
  const auto head_of = [&](int r) {
    return p.head * a.group + (MANY ? (p.row0 + r) % a.group : p.row0 + r);
  };
  const bool alone = p.c0 == p.c1;
  constexpr int kPartial = kRows * (DIM + 2);
  // a block has at most two pairs that others share: one that its piece starts with, and one
  // it leaves in the middle of
  const auto slot_of = [&](uint32_t piece) {
    return a.partial + (2ll * piece + (p.first > piece * per)) * kPartial;
  };
  const auto write = [&](int r, int col, float4 x, float sum) {
    if (r >= p.rows || col >= a.dim) return;
    // a query before the sequence's start sees no key: zeros. Any other sees itself, so a sum of 0
    // means that all its scores are -inf: 0 / 0.
    const float inv = sum == 0.0f ? NAN : 1.0f / sum;
    const bool none = p.lo + query_of(r) < 0;
    store4<T>(a.out + (p.query + query_of(r)) * a.out_token + head_of(r) * a.out_head +
                  col * R::size,
              none ? make_float4(0, 0, 0, 0)
                   : make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
  };
  // thread's columns: four of row `warp`, `warp + 4`, ...
  constexpr int lanes = DIM / 4;
  for (int i = tid; i < p.rows * lanes; i += kThreads) {
    const int r = i / lanes, col = 4 * (i % lanes);
    float top = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      top = fmaxf(top, reinterpret_cast<float *>(smem4)[w * (R::warp / 4) + kRows * DIM + r]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float *from = reinterpret_cast<float *>(smem4) + w * (R::warp / 4);
      const float f = pg::factor(from[kRows * DIM + r], base);
      const float4 x = *reinterpret_cast<const float4 *>(from + r * DIM + col);
      sum += f * from[kRows * DIM + kRows + r];
      acc.x = fmaf(f, x.x, acc.x), acc.y = fmaf(f, x.y, acc.y);
      acc.z = fmaf(f, x.z, acc.z), acc.w = fmaf(f, x.w, acc.w);
    }
    // a score that is NaN or +inf makes the sum NaN, and with it all the row's results
    const bool lost = sum < INFINITY && !(fabsf(acc.x) < INFINITY && fabsf(acc.y) < INFINITY &&
                                          fabsf(acc.z) < INFINITY && fabsf(acc.w) < INFINITY);
    if ((odd || lost) && col < a.dim) {
      bool first[4] = {true, true, true, true};
      const auto add = [&](int k, float value, float &to) {
        if (fabsf(value) < INFINITY) return;
        pg::add_odd(value, to, first[k]);
        first[k] = false;
      };
      for (int i = 0; i < p.block1 - p.block0; ++i)
        for (int j = 0; j < R::keys; ++j) {
          const int key = p.blocks.key_block(p.block0 + i) * R::keys + j;
          if (!pg::sees(a, p.lo + query_of(r), key) ||
              (sizeof(T) != 4 && !lost && p.all_see<R::step>(a, key / R::step * R::step)))
            continue;
          const int page = p.pages[key / a.page_size];
          if (page < 0 || page >= a.pages) continue;
          const float4 x = load4<T>(a.v + page * a.v_page + p.head * a.v_head +
                                    static_cast<int64_t>(key % a.page_size) * a.dim * R::size +
                                    col * R::size);
          add(0, x.x, acc.x);
          add(1, x.y, acc.y);
          add(2, x.z, acc.z);
          add(3, x.w, acc.w);
        }
    }
    if (alone) {
      write(r, col, acc, sum);
    } else {
      float *to = slot_of(blockIdx.x);
      *reinterpret_cast<float4 *>(to + r * DIM + col) = acc;
      if (col == 0) {
        to[kRows * DIM + r] = top;
        to[kRows * DIM + kRows + r] = sum;
      }
    }
  }
  if (!alone) {
    __threadfence();
    __syncthreads();
    // the counter of the piece that the pair starts in: no other pair's
    if (tid == 0) sh.last = atomicInc(a.arrived + p.c0, p.c1 - p.c0) == p.c1 - p.c0;
    __syncthreads();
    if (sh.last) {
      __threadfence();
      // as many pieces as the rings have room for at a time, all their loads in flight together
      constexpr int kBatch = R::bytes / (kPartial * 4), kPieces16 = kPartial / 4;
      constexpr int kEach = kThreads / lanes, kMine = kRows / kEach;
      const int col = 4 * (tid % lanes), first_r = tid / lanes;
      const int used = p.rows * lanes;  // 16-byte pieces of the rows there are
      float *const stage = reinterpret_cast<float *>(smem4);
      const uint32_t stage_at = static_cast<uint32_t>(__cvta_generic_to_shared(stage));
      float top[kMine], sum[kMine];
      float4 acc[kMine];
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        top[k] = -INFINITY, sum[k] = 0.0f;
        acc[k] = make_float4(0, 0, 0, 0);
      }
      for (uint32_t at = p.c0; at <= p.c1; at += kBatch) {
        const int here = min(static_cast<uint32_t>(kBatch), p.c1 - at + 1);
        __syncthreads();
        for (int i = 0; i < here; ++i) {
          const float *from = slot_of(at + i);
          for (int j = tid; j < used + kRows / 2; j += kThreads) {
            const int piece = j < used ? j : j - used + kRows * lanes;  // rows, then m and l
            copy16(stage_at + (i * kPieces16 + piece) * 16, from + 4 * piece, true);
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        for (int i = 0; i < here; ++i) {
          const float *from = stage + i * kPartial;
#pragma unroll
          for (int k = 0; k < kMine; ++k) {
            const int r = first_r + k * kEach;
            if (r >= p.rows) continue;
            const float m_here = from[kRows * DIM + r], most = fmaxf(top[k], m_here);
            const float base = most == -INFINITY ? 0.0f : most;
            const float f = pg::factor(m_here, base), old = pg::factor(top[k], base);
            const float4 x = *reinterpret_cast<const float4 *>(from + r * DIM + col);
            top[k] = most;
            sum[k] = fmaf(f, from[kRows * DIM + kRows + r], old * sum[k]);
            acc[k].x = fmaf(f, x.x, old * acc[k].x), acc[k].y = fmaf(f, x.y, old * acc[k].y);
            acc[k].z = fmaf(f, x.z, old * acc[k].z), acc[k].w = fmaf(f, x.w, old * acc[k].w);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kMine; ++k) write(first_r + k * kEach, col, acc[k], sum[k]);
    }
  }
}

// A block's piece of the line: up to which place it goes and how long a piece is; and the pair it is
// at: its sequence, and the sequence's place on the line.
struct Plan {
  uint32_t end, per, before;
  int sequence, turn;
};

// MANY: sequences have any number of queries, not one each.
template <class T, int DIM, bool MANY>
__global__ void __launch_bounds__(kThreads, kPerSm)
    decode_kernel(const __grid_constant__ Attention a) {
  using R = Ring<T, DIM>;
  extern __shared__ float4 smem4[];
  __shared__ uint3 warp_sum[kWarps];
  __shared__ Pair sh;
  __shared__ Plan plan_here;
  // read each time: held in registers, it would crowd the loop over the keys
  volatile Plan &plan = plan_here;
  __shared__ int odds[2];  // whether a value that is not finite was zeroed, by turns of pairs
  pg::wait_for_earlier_kernels();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const uint32_t c = blockIdx.x;
  if (tid < 2) odds[tid] = 0;

  // Every block works the line out for itself: thread i counts the pairs and their blocks of keys
  // of a run of sequences.
  const int run = (a.batch + kThreads - 1) / kThreads;
  const int first_b = min(tid * run, a.batch), end_b = min(first_b + run, a.batch);
  uint32_t pairs = 0, keys = 0, longest = 0;
  for (int b = first_b; b < end_b; ++b) {
    const Sequence s = sequence_of<MANY, R::keys>(a, b);
    pairs += s.pairs;
    keys += s.pairs * s.blocks.count;
    longest = max(longest, static_cast<uint32_t>(s.blocks.count));
    if (!s.length && b % gridDim.x == c)  // no key: zeros
      for (int i = 0; i < s.count * a.heads * a.group; ++i)
        for (int j = 0; j < a.dim * R::size / 16; ++j)
          *reinterpret_cast<uint4 *>(a.out + (s.query + i / (a.heads * a.group)) * a.out_token +
                                     i % (a.heads * a.group) * a.out_head + j * 16) =
              make_uint4(0, 0, 0, 0);
  }
  uint32_t pairs_upto = pairs, keys_upto = keys;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, pairs_upto, off);
    const uint32_t k = __shfl_up_sync(0xffffffffu, keys_upto, off);
    if (lane >= off) pairs_upto += o, keys_upto += k;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) warp_sum[warp] = make_uint3(pairs_upto, keys_upto, longest);
  __syncthreads();
  uint32_t all_pairs = 0, all_keys = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint3 s = warp_sum[w];
    if (w < warp) pairs_upto += s.x, keys_upto += s.y;
    all_pairs += s.x;
    all_keys += s.y;
    longest = max(longest, s.z);
  }
  if (!all_keys) return;
  const uint32_t total = all_keys + kPair * all_pairs;
  // The length of a piece; piece c is [c per, (c + 1) per). As few as give every block one, but the
  // last block to finish a pair reads all its pieces, so the longest is not cut in more than about
  // kCut times the root of its blocks: one sequence of 60000 keys on one kv head takes 45 us so,
  // 53 with twice as many pieces at most and 55 with half as many.
  const uint32_t least = static_cast<uint32_t>(sqrtf(static_cast<float>(longest)) / kCut);
  const uint32_t per = max((total + gridDim.x - 1) / gridDim.x, least);
  if (static_cast<uint64_t>(c) * per >= total) return;
  uint32_t u = c * per;
  const uint32_t upto = keys_upto + kPair * pairs_upto;
  const uint32_t before = upto - keys - kPair * pairs;
  if (u >= before && u < upto) {
    uint32_t at = before;
    for (int b = first_b; b < end_b; ++b) {
      const Sequence s = sequence_of<MANY, R::keys>(a, b);
      const uint32_t next = at + s.pairs * (s.blocks.count + kPair);
      if (u < next) {
        plan.sequence = b;
        plan.before = at;
        plan.end = min(total, u + per);
        plan.per = per;
        plan.turn = 0;
        break;
      }
      at = next;
    }
  }
  __syncthreads();

  char *ring = reinterpret_cast<char *>(smem4) + warp * R::warp;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  while (u < plan.end) {
    int b = plan.sequence;
    Sequence seq = sequence_of<MANY, R::keys>(a, b);
    while (!seq.pairs) seq = sequence_of<MANY, R::keys>(a, ++b);
    const Blocks &blocks = seq.blocks;
    const uint32_t before = plan.before, per = plan.per;
    const uint32_t units = blocks.count + kPair, pair = (u - before) / units;
    const int head = pair / seq.row_groups, row0 = (pair % seq.row_groups) * kRows;
    const int rows = min(kRows, seq.count * a.group - row0);
    const uint32_t pair_first = before + pair * units;
    const uint32_t stop = min(plan.end, pair_first + units);
    const int block0 = max(0, static_cast<int>(u - pair_first) - kPair);
    const int block1 = static_cast<int>(stop - pair_first) - kPair;
    if (block1 <= 0) break;  // the piece ends before the pair's first block
    __syncthreads();
    if (tid == 0) {
      const bool ends = stop == before + seq.pairs * units;  // the sequence's last pair
      plan.sequence = b + ends;
      if (ends) plan.before = stop;
    }
    u = stop;
    const int *pages = a.table + seq.slot * a.table_row;
    // the positions of the queries: of all, and of this thread's rows g and g + 8
    const int lo = seq.length - seq.count, hi = seq.length - 1;
    if (tid == 0)
      sh = Pair{seq.query, row0, rows, head, lo, hi, block0, block1, pair_first,
                (pair_first + kPair) / per, (pair_first + units - 1) / per, blocks, pages, 0};
    const auto query_of = [&](int r) { return MANY ? (row0 + r) / a.group : 0; };
    const auto head_of = [&](int r) {
      return head * a.group + (MANY ? (row0 + r) % a.group : row0 + r);
    };
    const int pos[2] = {lo + query_of(g), lo + query_of(g + 8)};
    int *const odd = odds + plan.turn;

    // the queries' fragments: rows g and g + 8, columns 2 t and 2 t + 8 of each 16 (f32: t and t + 4
    // of each 8)
    uint32_t q[sizeof(T) == 4 ? 1 : DIM / 16][4];
    const auto q_word = [&](int k, int h, int i) {
      const int r = g + 8 * h;
      return r < rows && 32 * k + 16 * i < a.dim * R::size
                 ? *reinterpret_cast<const uint32_t *>(a.q + (seq.query + query_of(r)) * a.q_token +
                                                       head_of(r) * a.q_head + 32 * k + 16 * i +
                                                       4 * t4)
                 : 0u;
    };
    uint4 *const q_hi = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(smem4) + R::q) + lane;
    uint4 *const q_lo = q_hi + R::q_part / 16;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = warp; k < DIM / 8; k += kWarps) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          Mma<T>::split_near(__uint_as_float(q_word(k, e & 1, e >> 1)), hi[e], lo[e]);
        q_hi[32 * k] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        q_lo[32 * k] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < DIM / 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) q[k][e] = q_word(k, e & 1, e >> 1);
    }
    float o[DIM / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

    // The warp's steps are the blocks' 16 keys at 16 warp (f32: 8 at 8 warp). A step whose keys all
    // are seen and lie in one page, as they do where pages are whole groups of so many, needs one
    // look at the table and one address; else lane r knows key r's page and row.
    const int steps = block1 - block0;
    const bool whole_pages = a.page_size % R::step == 0;
    const auto first_key = [&](int i) {
      return blocks.key_block(block0 + i) * R::keys + R::step * warp;
    };
    const auto all_seen = [&](int key) {
      return key + R::step - 1 <= lo &&
             (!a.window || key > hi - a.window || key + R::step <= a.sinks);
    };
    const auto some_see = [&](int key) {
      return key <= hi && (!a.window || key > lo - a.window || key < a.sinks);
    };
    const auto page_for = [&](int i) {  // as the table names it; -1: not seen
      if (i >= steps) return -1;
      const int key = first_key(i);
      if (whole_pages && all_seen(key)) return pages[key / a.page_size];
      return some_see(key + (lane & (R::step - 1))) ? pages[(key + (lane & (R::step - 1))) / a.page_size] : -1;
    };
    const int sub = lane / R::chunks, chunk = lane % R::chunks;
    const bool column = chunk * 16 < a.dim * R::size;
    const int64_t row_bytes = static_cast<int64_t>(R::size) * a.dim;
    const char *const k_head = a.k + head * a.k_head + chunk * 16;
    const char *const v_head = a.v + head * a.v_head + chunk * 16;
    constexpr int kCopies = R::step * R::chunks / 32, kRowsEach = 32 / R::chunks;
    const auto issue = [&](int i, int page) {
      if (i < steps) {
        const uint32_t to = ring_at + (i % R::stages) * R::stage;
        const int key = first_key(i);
        if (whole_pages && all_seen(key)) {
          bool real = column;
          if (page < 0 || page >= a.pages) {
            atomicOr(a.status, PG_CACHE_BAD_PAGE);
            real = false, page = 0;
          }
          const int64_t in = (key % a.page_size + sub) * row_bytes;
          const char *k = k_head + page * a.k_page + in, *v = v_head + page * a.v_page + in;
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            const uint32_t at = to + R::at(j * kRowsEach + sub, chunk);
            copy16(at, k, real);
            copy16(at + R::tile, v, real);
            k += kRowsEach * row_bytes;
            v += kRowsEach * row_bytes;
          }
        } else {
          const int mine_key = key + (lane & (R::step - 1));
          if (some_see(mine_key) && (page < 0 || page >= a.pages)) {
            atomicOr(a.status, PG_CACHE_BAD_PAGE);
            page = -1;
          }
          const int mine_row = mine_key % a.page_size;
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            const int r = j * kRowsEach + sub;
            const int at_page = __shfl_sync(0xffffffffu, page, r);
            const int row = __shfl_sync(0xffffffffu, mine_row, r);
            const bool real = at_page >= 0 && column;
            const int64_t in = real ? row * row_bytes : 0, pg = real ? at_page : 0;
            copy16(to + R::at(r, chunk), k_head + pg * a.k_page + in, real);
            copy16(to + R::tile + R::at(r, chunk), v_head + pg * a.v_page + in, real);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // pages are asked for two steps before their rows are
    int next = page_for(0), after = page_for(1);
#pragma unroll
    for (int i = 0; i < R::stages - 1; ++i) {
      const int page = next;
      next = after;
      after = page_for(i + 2);
      issue(i, page);
    }
    for (int i = 0; i < steps; ++i) {
      const int page = next;
      next = after;
      after = page_for(i + R::stages + 1);
      issue(i + R::stages - 1, page);
      asm volatile("cp.async.wait_group %0;" ::"n"(R::stages - 1) : "memory");
      __syncwarp();
      const uint32_t ks = ring_at + (i % R::stages) * R::stage, vs = ks + R::tile;
      constexpr int kN = R::step / 8;
      float s[kN][4] = {};
      if constexpr (sizeof(T) == 4) {
        // even and odd columns, and hi by hi and the rest, by themselves: four short chains of sums
        float part[4][4] = {};
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          uint32_t x[4];  // 8 keys by columns 16 k.., four 8 x 4 matrices along the columns
          load_matrices(ks + R::at(lane & 7, 4 * k + (lane >> 3)), x);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 a_hi = q_hi[32 * (2 * k + j)], a_lo = q_lo[32 * (2 * k + j)];
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) Mma<T>::split(__uint_as_float(x[2 * j + e]), hi[e], lo[e]);
            Mma<T>::run(part[j], &a_hi.x, hi);
            Mma<T>::run(part[2 + j], &a_hi.x, lo);
            Mma<T>::run(part[2 + j], &a_lo.x, hi);
          }
        }
        bool none = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[0][e] = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
          none |= s[0][e] != s[0][e];
        }
        // a factor that is not finite has no two parts: such products are made anew, as they stand
        if (__any_sync(0xffffffffu, none))
          for (int e = 0; e < 4; ++e) {
            const int r = g + 8 * (e >> 1);
            if (r < rows)
              s[0][e] = plain_product<R>(
                  a.q + (seq.query + query_of(r)) * a.q_token + head_of(r) * a.q_head,
                  ring + (i % R::stages) * R::stage, 2 * t4 + (e & 1), a.dim);
          }
      } else {
#pragma unroll
        for (int k = 0; k < DIM / 32; ++k)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t x[4];  // keys 8 n.. by columns 32 k.., four 8 x 8 matrices along the columns
            load_matrices(ks + R::at(8 * n + (lane & 7), 4 * k + (lane >> 3)), x);
            Mma<T>::run(s[n], q[2 * k], x[0], x[1]);
            Mma<T>::run(s[n], q[2 * k + 1], x[2], x[3]);
          }
      }
      const int key = first_key(i);
      const bool masked = !all_seen(key);
      bool look = MANY && masked;
      if constexpr (sizeof(T) == 4) {
        // 0 times a number that is not finite is NaN
        pg::Two none(0.0f, 0.0f);
        const pg::Two zero(0.0f, 0.0f);
#pragma unroll
        for (int j = lane; j < R::step * R::chunks; j += 32) {
          const float4 x = *reinterpret_cast<const float4 *>(
              ring + (i % R::stages) * R::stage + R::tile + j * 16);
          none = fma(pg::Two(x.x, x.y), zero, none);
          none = fma(pg::Two(x.z, x.w), zero, none);
        }
        float x, y;
        none.get(x, y);
        look = __any_sync(0xffffffffu, x + y != 0.0f);
      }
      if (look) {
        bool any = false;
        for (int j = lane; j < R::step * R::chunks; j += 32) {
          uint4 *const at =
              reinterpret_cast<uint4 *>(ring + (i % R::stages) * R::stage + R::tile + j * 16);
          if constexpr (sizeof(T) == 4) any |= pg::clean32(at);
          else any |= pg::clean<Mma<T>::exponent>(at);
        }
        if (any) *const_cast<volatile int *>(odd) = 1;
        __syncwarp();
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= a.scale_log2;
          if (masked && !pg::sees(a, pos[e >> 1], key + 2 * t4 + 8 * n + (e & 1)))
            s[n][e] = -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float f = pg::factor(m[h], top[h] == -INFINITY ? 0.0f : top[h]);
          m[h] = top[h];
          l[h] *= f;
#pragma unroll
          for (int n = 0; n < DIM / 8; ++n) {
            o[n][2 * h] *= f;
            o[n][2 * h + 1] *= f;
          }
        }
      }
      const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = s[n][2 * h] - base[h], y = s[n][2 * h + 1] - base[h];
          if constexpr (Mma<T>::shift != 0.0f) x += Mma<T>::shift, y += Mma<T>::shift;
          x = pg::exp2_fast(x);
          y = pg::exp2_fast(y);
          l[h] += x + y;
          if constexpr (sizeof(T) == 4) {
            Mma<T>::split_near(x, hi[h], lo[h]);  // the product's keys are 0, 2, 4, 6, 1, 3, 5, 7
            Mma<T>::split_near(y, hi[2 + h], lo[2 + h]);
          } else {
            Mma<T>::split(x, y, hi[2 * n + h], lo[2 * n + h]);
          }
        }
      if constexpr (sizeof(T) == 4) {
        const char *const v = ring + (i % R::stages) * R::stage + R::tile + 4 * (g & 3);
#pragma unroll
        for (int n = 0; n < DIM / 8; ++n) {
          uint32_t v_hi[2], v_lo[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            Mma<T>::split(
                *reinterpret_cast<const float *>(v + R::at(2 * t4 + e, 2 * n + (g >> 2))),
                v_hi[e], v_lo[e]);
          // a step's products by themselves: the tensor cores do not round their sums to nearest, and
          // thousands of steps would add those errors up
          float sum[4] = {};
          Mma<T>::run(sum, hi, v_lo);
          Mma<T>::run(sum, lo, v_hi);
          Mma<T>::run(sum, hi, v_hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] += sum[e];
        }
      } else {
#pragma unroll
        for (int n = 0; n < DIM / 16; ++n) {
          uint32_t x[4];  // keys 0.. and 8.. by columns 16 n.. and 16 n + 8.., transposed
          load_matrices_t(vs + R::at(lane & 15, 2 * n + (lane >> 4)), x);
          Mma<T>::run(o[2 * n], hi, x[0], x[1]);
          Mma<T>::run(o[2 * n], lo, x[0], x[1]);
          Mma<T>::run(o[2 * n + 1], hi, x[2], x[3]);
          Mma<T>::run(o[2 * n + 1], lo, x[2], x[3]);
        }
      }
      __syncwarp();  // the stage may be filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // the warps' results, in their rings' places: rows of DIM numbers, then m and l of each row
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    float *res = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h;
#pragma unroll
      for (int n = 0; n < DIM / 8; ++n)
        *reinterpret_cast<float2 *>(res + r * DIM + 8 * n + 2 * t4) =
            make_float2(o[n][2 * h], o[n][2 * h + 1]);
      if (t4 == 0) {
        res[kRows * DIM + r] = m[h];
        res[kRows * DIM + kRows + r] = l[h];
      }
    }
    __syncthreads();

    finish_pair<T, DIM, MANY>(a, sh, plan.per, odds[plan.turn]);
    __syncthreads();  // the rings are free again
    if (tid == 0) {
      odds[plan.turn] = 0;  // for the turn after the next
      plan.turn = plan.turn ^ 1;
    }
    __syncthreads();
  }
}

template <class T, int DIM>
int launch_decode(const Attention &a, int sms, cudaStream_t stream) {
  const dim3 grid(kPerSm * sms);
  if (a.starts)
    return pg::launch<decode_kernel<T, DIM, true>>("decode_kernel", grid, kThreads,
                                                   Ring<T, DIM>::bytes, stream, a);
  return pg::launch<decode_kernel<T, DIM, false>>("decode_kernel", grid, kThreads,
                                                  Ring<T, DIM>::bytes, stream, a);
}

}  // namespace

namespace pg {

// Whether this kernel takes a batch and not the large tiles of attention_prompt.cu: at up to 48
// rows a sequence on average, which those fill badly. The average says little of an uneven batch:
// 100 single tokens and one chunk of 1024, 4000 keys each and 4 heads on each of 8, come here and
// take 997 us, where the chunk alone takes 126 there and the tokens 289 here; 63 and one of 2048
// go there and take 387, alone 176 and 195. Even batches, by rows a sequence, this against those,
// in microseconds at head size 128: 7 sequences of up to 20000 keys on 4 kv heads, 16 rows 43 and
// 83, 32 rows 56 and 84, 48 rows 60 and 84, 64 rows 70 and 96; 32 of up to 8000 on 8, 16 rows 74
// and 157, 32 rows 119 and 158, 48 rows 155 and 160, 64 rows 191 and 160; 100 of up to 500 on 4,
// 48 rows 51 and 49, 64 rows 63 and 50.
// f32 has no such tiles, so it is taken at up to 256 rows, and at up to 1024 where most keys are
// seen by all of a sequence's queries, since a group of 16 rows goes through all that any sees. This
// against attention.cu: 8 sequences on 4 kv heads of 128, up to 4056 keys, 64 rows 86 and 164, 256
// rows 253 and 390, 1024 rows 947 and 1270; of no other keys than the queries, 256 rows 13 and 17,
// 512 rows 25 and 17; with a window of 100 and heads of 64, 256 rows 28 and 32, 512 rows 45 and 34.
bool decode_takes(const Attention &a, bool f32, int most, int max_len) {
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  const bool early = !a.window && max_len / 8ll * a.batch >= a.queries;
  if (a.starts && rows > (f32 ? early ? 1024ll : 256ll : 48ll) * a.batch) return false;
  // its blocks of 32 keys or more count in 31 bits
  return (rows / kRows + a.batch) * a.heads * (most / 32 + 2ll + kPair) < INT32_MAX;
}

int decode(const Attention &a, int dtype, int sms, cudaStream_t stream) {
  if (dtype == PG_DT_F32)
    return a.dim <= 64 ? launch_decode<float, 64>(a, sms, stream)
                       : launch_decode<float, 128>(a, sms, stream);
  if (dtype == PG_DT_BF16)
    return a.dim <= 64 ? launch_decode<__nv_bfloat16, 64>(a, sms, stream)
                       : launch_decode<__nv_bfloat16, 128>(a, sms, stream);
  return a.dim <= 64 ? launch_decode<__half, 64>(a, sms, stream)
                     : launch_decode<__half, 128>(a, sms, stream);
}

}  // namespace pg

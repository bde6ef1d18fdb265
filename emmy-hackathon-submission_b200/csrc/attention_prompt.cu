// Attention of several new tokens a sequence for the 16-bit types at head sizes of up to 128, on
// the fifth-generation tensor cores (pg_attention with starts).
//
// A block takes 256 rows (queries times the heads of one kv head's group, so the heads that read
// the same keys share every load of them) as two tiles of 128, and a part of the blocks of 128
// keys that they see. Per block of keys and tile, S = Q K^T (128 x 128 x DIM) goes to tensor
// memory, 128 threads, one a row, turn S into weights P there, and O += P V accumulates in tensor
// memory with P read from it. The two tiles take turns: while one's weights are computed the
// tensor cores work for the other.
//
//   warps 0-3, 4-7  the rows' threads of tile 0 and tile 1
//   warp 8          issues the products, the two tiles' strictly in turn: issued as they come,
//                   they mix, and both tiles then wait for both
//   warps 9, 10     bring keys and values, page by page, into a ring in shared memory
//
// Where pages are whole groups of eight keys, two warps bring them with TMA, a box eight keys by
// 64 columns, 128-byte swizzled as the products read it. Pages of other sizes come in 16-byte
// pieces through cp.async, whose arithmetic then bounds the kernel: two sequences of 4096 new
// tokens and up to 8192 keys, 32 heads on 8 of 128 in bf16, take 1814 us that way, 498 with TMA
// (885 TFLOP/s of the products that count).
//
// The rows' threads bound it beside the products: 128 x 128 exponentials take the 16 lanes an SM
// has for them 1024 cycles, the two products of DIM = 128 the same, and where a tile's weights
// wait for its scores neither is at work. O is rescaled only when a row's running maximum has
// grown by more than 2^8 since the last time, so that a weight is at most 2^8 and rescaling is
// rare; the sum l goes by the same maximum, so the result is the same.
//
// Rounding: weights go into the second product in the values' type (up to 2^-8 or 2^-11 of each, at
// random), as the tensor cores take both operands in one type; S, m, l and O are in 32 bits. In f16,
// which rounds coarsely below 2^-14, weights and their sum are 2^7 of what they are.
//
// A masked place has weight 0, and 0 times a value that is not finite would be NaN. So the values
// of each block that some row must not see in full are looked through before they are used: what
// is not finite is zeroed and a flag raised, and at the end a row adds the ones it does see again.
// Rows past the sequence's length are zeroed. In the other blocks a weight that was rounded to 0 may
// have met an infinite value: a result that is not finite is made of the visible values that are not.
//
// Every wait is bounded: one that takes over two seconds sets PG_ATTENTION_WAIT in the status
// word, and all roles leave their loops; the block then frees its tensor memory and returns.
#include "attention.cuh"

#include <cuda.h>

#include <numeric>

// Encodes a tensor map of 2-byte elements, 128-byte swizzled (launcher.cpp).
int pg_detail_tensormap(void *map, int rank, uint64_t base, const uint64_t *dims,
                        const uint64_t *strides_bytes, const uint32_t *box);

namespace {

using pg::Attention;
using pg::Blocks;
using pg::max3;
using pg::Tile;
using pg::Two;

constexpr int kKeys = 128, kRows = 256, kHalf = 128;
constexpr int kThreads = 384;
constexpr int kCopyWarps = 2, kCopyThreads = 32 * kCopyWarps;  // without TMA
constexpr int kLag = 2;  // tiles whose cp.async copies are in flight before the oldest is waited for
constexpr float kGrow = 8.0f;
constexpr unsigned long long kWaitNs = 2000000000ull;

template <int DIM>
struct Plan {
  // 128 queries, keys or values: by eight rows, then by 64 columns, each such 1024 bytes swizzled
  static constexpr int atom = 1024, chunks = DIM / 64, group = chunks * atom;
  static constexpr int tile = 16 * group;
  static constexpr int stages = DIM == 128 ? 5 : 8;
  static constexpr int q = 0, ring = 2 * tile, bars = ring + stages * tile;
  // over half an SM's shared memory, so that no other block that takes all its tensor memory
  // is resident beside this one
  static constexpr int bytes = 1024 + bars + 256;
  static_assert(bytes > 116 * 1024 && bytes <= 232448 && stages > kLag + 1, "shared memory");
  __device__ static int at(int r, int piece) {    // 16-byte piece of a row
    return (r >> 3) * group + (piece >> 3) * atom + (r & 7) * 128 + (((piece & 7) ^ (r & 7)) << 4);
  }
};

__device__ __forceinline__ uint32_t shared_at(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// One box of a tensor map into shared memory; its bytes count at the barrier.
__device__ __forceinline__ void tma_load_4d(uint32_t to, const CUtensorMap *map, int x, int y,
                                            int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
               "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z),
               "r"(w), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\n"
               "mbarrier.try_wait.parity.shared.b64 p, [%1], %2, 0x989680;\n"
               "selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// Waits for a phase of a barrier; false once a wait of this block has run out of time.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *failed,
                                         unsigned *status) {
  if (bar_try(bar, parity)) return true;
  const unsigned long long begin = now_ns();
  while (!bar_try(bar, parity)) {
    if (*failed) return false;
    if (now_ns() - begin > kWaitNs) {
      *failed = 1;
      atomicOr(status, PG_ATTENTION_WAIT);
      return false;
    }
  }
  return true;
}
// ... for what this thread has in flight, also after a wait has run out of time.
__device__ void bar_drain(uint32_t bar, uint32_t parity, unsigned *status) {
  int failed = 0;
  bar_wait(bar, parity, &failed, status);
}

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// The products are issued by one lane of a warp that runs as a whole, so that operands stay in
// uniform registers: issued from a branch of one thread's, each took longer than its work.
__device__ __forceinline__ void commit(uint32_t bar, uint32_t elected) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\n@q tcgen05.commit.cta_group::1."
               "mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar), "r"(elected)
               : "memory");
}
// D (tensor memory) = A B (+ D): both from shared memory, or A from tensor memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add,
                                       uint32_t elected) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add)), "r"(elected)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add,
                                       uint32_t elected) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
               "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add)), "r"(elected)
               : "memory");
}

#define PG_R8(x, i) x(i), x(i + 1), x(i + 2), x(i + 3), x(i + 4), x(i + 5), x(i + 6), x(i + 7)
#define PG_R32(x) PG_R8(x, 0), PG_R8(x, 8), PG_R8(x, 16), PG_R8(x, 24)

// 32 columns of this thread's row of tensor memory
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t *v) {
#define PG_OUT(i) "=r"(v[i])
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PG_R32(PG_OUT)
      : "r"(at));
#undef PG_OUT
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t *v) {
#define PG_IN(i) "r"(v[i])
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PG_R32(
          PG_IN),
      "r"(at)
      : "memory");
#undef PG_IN
}
__device__ __forceinline__ void wait_loads() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// What was loaded is used after this point only.
__device__ __forceinline__ void tie(uint32_t *v) {
#define PG_TIE(i) "+r"(v[i])
  asm volatile("" : PG_R32(PG_TIE));
#undef PG_TIE
}
__device__ __forceinline__ void wait_stores() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// The largest score of a row of a block, and m.
__device__ __forceinline__ float largest(const float *s, float m) {
  float top[4] = {m, s[0], s[1], s[2]};
#pragma unroll
  for (int k = 3; k < kKeys - 1; k += 2) top[k / 2 & 3] = max3(top[k / 2 & 3], s[k], s[k + 1]);
  return max3(max3(top[0], top[1], top[2]), top[3], s[kKeys - 1]);
}

template <class T> struct Type;
template <> struct Type<__nv_bfloat16> {
  static constexpr float shift = 0.0f;  // weights go in as 2^shift of what they are
  static constexpr uint32_t format = 1, exponent = 0x7f80;
  __device__ static uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  __device__ static float low(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ static float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <> struct Type<__half> {
  static constexpr float shift = 15.0f - kGrow;  // at most 2^15 of 65504
  static constexpr uint32_t format = 0, exponent = 0x7c00;
  __device__ static uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  __device__ static float low(uint32_t w) {
    return __low2float(*reinterpret_cast<const __half2 *>(&w));
  }
  __device__ static float high(uint32_t w) {
    return __high2float(*reinterpret_cast<const __half2 *>(&w));
  }
};

// A shared-memory operand of 128-byte swizzled rows: `rows` is the distance of its groups of
// eight, `columns` that of its 64-column chunks where columns are the product's N.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t rows, uint32_t columns) {
  const uint32_t lo = ((at >> 4) & 0x3fff) | ((columns >> 4) << 16);
  const uint32_t hi = (rows >> 4) | (1u << 14) | (2u << 29);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// 32-bit sums, M = 128, N columns; B with its N side contiguous or its K side
template <class T>
__device__ constexpr uint32_t product(int n, bool n_contiguous) {
  return (1u << 4) | (Type<T>::format << 7) | (Type<T>::format << 10) |
         (static_cast<uint32_t>(n_contiguous) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (128u >> 4 << 24);
}

// Which blocks of keys every row of a tile, with queries at positions lo..hi, sees in full.
struct Seen {
  int low, high, sinks;  // those that start in low..high, or end within the sinks
  __device__ Seen(const Attention &a, int lo, int hi, int length)
      : low(a.window ? hi - a.window + 1 : 0), high(min(lo + 1, length) - kKeys), sinks(a.sinks) {}
  __device__ bool all(int key0) const {
    return key0 <= high && (key0 >= low || key0 + kKeys <= sinks);
  }
};

struct Head {  // what the roles share
  uint32_t tmem;
  int failed, odd;
  unsigned last;
};

// Adds the values that are not finite and that the query at `pos` sees to 32 columns of its result: of
// all blocks of keys, or of those that some row must not see in full. A function of its own for the
// registers, as it is hardly ever called: in the kernel it made every step slower (508 us for 498).
template <class T>
__device__ __noinline__ void add_values(const Attention &a, const int *pages, int length, Blocks blocks,
                                        Seen both, int b0, int steps, int head, int pos, int k,
                                        bool all, float *x) {
  uint32_t met = 0;
  for (int j = 0; j < steps; ++j) {
    const int key0 = blocks.key_block(b0 + j) * kKeys;
    if (!all && both.all(key0)) continue;
    for (int key = key0; key < min(key0 + kKeys, length); ++key) {
      if (!pg::sees(a, pos, key)) continue;
      const int page = pages[key / a.page_size];
      if (page < 0 || page >= a.pages) continue;
      const char *v = a.v + page * a.v_page + head * a.v_head +
                      static_cast<int64_t>(key % a.page_size) * a.dim * 2 + 64 * k;
      for (int c = 0; c < 32; c += 2) {
        if (32 * k + c >= a.dim) break;
        const uint32_t w = *reinterpret_cast<const uint32_t *>(v + 2 * c);
        const float value[2] = {Type<T>::low(w), Type<T>::high(w)};
        for (int e = 0; e < 2; ++e)
          if (!(fabsf(value[e]) < INFINITY)) {
            pg::add_odd(value[e], x[c + e], !(met >> (c + e) & 1));
            met |= 1u << (c + e);
          }
      }
    }
  }
}

// Without TMA the maps and `boxes` are empty.
template <class T, int DIM, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ Attention a, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map, int run) {
  using P = Plan<DIM>;
  extern __shared__ char smem_raw[];
  __shared__ Head sh;
  char *smem = reinterpret_cast<char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  pg::wait_for_earlier_kernels();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.x, tile_id = gridDim.y - 1 - blockIdx.y, part = blockIdx.z;
  const Tile t = pg::find_tile(a, tile_id);
  if (!t.rows) return;
  const int first_pos = t.length - t.count;
  const int tiles = t.rows > kHalf ? 2 : 1;
  const int lo = first_pos + t.row / a.group, hi = first_pos + (t.row + t.rows - 1) / a.group;
  const Blocks blocks = pg::blocks_of(a, lo, hi, kKeys);
  const Seen both(a, lo, hi, t.length);
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks.count) * part / a.parts);
  const int steps =
      static_cast<int>(static_cast<int64_t>(blocks.count) * (part + 1) / a.parts) - b0;

  const uint32_t smem_at = shared_at(smem), bars = smem_at + P::bars;
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (P::stages + s); };
  const uint32_t q_full = bars + 16 * P::stages;
  const auto s_full = [&](int i) { return q_full + 8 + 8 * i; };
  const auto p_full = [&](int i) { return q_full + 24 + 8 * i; };
  const uint32_t o_full = q_full + 40;
  if (tid == 0) {
    for (int s = 0; s < P::stages; ++s) {
      bar_init(full(s), TMA ? 1 : kCopyThreads);
      bar_init(empty(s), 1);
    }
    bar_init(q_full, 2 * kHalf);
    for (int i = 0; i < 2; ++i) {
      bar_init(s_full(i), 1);
      bar_init(p_full(i), kHalf);
    }
    bar_init(o_full, 1);
    sh.failed = sh.odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     shared_at(&sh.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;  // S and P of tile i at 128 i, O at 256 + 128 i
  volatile int *failed = &sh.failed;

  // Registers: three groups of 128 threads start with 168 each; the rows' threads, which hold a
  // row of S and what is made of it, take what the third group can do without (2 x 232 + 40 or
  // 2 x 200 + 104 = 3 x 168).
  if (warp >= 8) {
    if (TMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (TMA && (warp == 9 || warp == 10)) {
      // --- copies: one warp the keys of each block, one the values; lane i the i-th page run ----
      const int half = warp - 9, runs = kKeys / run;
      const CUtensorMap *map = half ? &v_map : &k_map;
      const auto key_of = [&](int j) { return blocks.key_block(b0 + j) * kKeys + lane * run; };
      const auto page_for = [&](int j) {  // -1: the run lies past the length
        if (j >= steps || lane >= runs || key_of(j) >= t.length) return -1;
        return t.pages[key_of(j) / a.page_size];
      };
      int next = page_for(0), j = 0;
      bool ok = true;
      for (; j < steps; ++j) {
        const bool real = lane < runs && key_of(j) < t.length;
        int page = next;
        next = page_for(j + 1);
        if (real && (page < 0 || page >= a.pages)) {
          atomicOr(a.status, PG_CACHE_BAD_PAGE);
          page = a.pages;  // past the last page: the copy fills in zeros
        }
        const int row = key_of(j) % a.page_size, n = 2 * j + half, s = n % P::stages;
        const int held = __popc(__ballot_sync(0xffffffffu, real));
        if (n >= P::stages) ok = bar_wait(empty(s), (n / P::stages - 1) & 1, failed, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) bar_expect(full(s), held * run * 128 * P::chunks);
        __syncwarp();
        if (real) {
          const uint32_t to = smem_at + P::ring + s * P::tile + lane * (run / 8) * P::group;
          // a box is eight rows of 64 columns
          for (int g = 0; g < run / 8; ++g)
#pragma unroll
            for (int k = 0; k < P::chunks; ++k)
              tma_load_4d(to + g * P::group + k * P::atom, map, 64 * k, row + 8 * g, head, page,
                          full(s));
        }
      }
      // no copy is in flight when the block's shared memory goes
      for (int k = max(0, j - P::stages); k < j; ++k) {
        const int n = 2 * k + half;
        if (n + P::stages >= 2 * j + half) bar_drain(full(n % P::stages), n / P::stages & 1, a.status);
      }
    } else if (!TMA && (warp == 9 || warp == 10)) {
      // --- copies: K and V of each block in turn ----------------------------------------------
      const int w = warp - 9;
      constexpr int kPieces = DIM / 8, kPer = 32 / kPieces;  // rows a warp copies at once
      const int sub = lane / kPieces, piece = lane % kPieces;
      const auto pages_of = [&](int j, int2 *p) {  // keys lane, lane + 32, ... of step j
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = make_int2(-1, 0);
          const int key = blocks.key_block(b0 + j) * kKeys + lane + 32 * i;
          if (j < steps && key < t.length) {
            const int entry = key / a.page_size;
            p[i] = make_int2(t.pages[entry], key - entry * a.page_size);
            if (p[i].x < 0 || p[i].x >= a.pages) {
              atomicOr(a.status, PG_CACHE_BAD_PAGE);
              p[i].x = -1;
            }
          }
        }
      };
      const auto finish = [&](int n) {  // tile n has landed: look it over and hand it on
        const int s = n % P::stages;
        if (n & 1) {
          const int key0 = blocks.key_block(b0 + (n >> 1)) * kKeys;
          if (!both.all(key0)) {
            bool odd = false;
            for (int i = w; i < kKeys / kPer; i += kCopyWarps) {  // the pieces it has copied
              odd |= pg::clean<Type<T>::exponent>(reinterpret_cast<uint4 *>(smem + P::ring + s * P::tile +
                                                        P::at(i * kPer + sub, piece)));
            }
            if (odd) *const_cast<volatile int *>(&sh.odd) = 1;
          }
        }
        fence_async();
        bar_arrive(full(s));
      };
      int2 p[4], next[4];
      pages_of(0, p);
      int n = 0, done = 0;
      bool ok = true;
      for (int j = 0; j < steps && ok; ++j) {
        pages_of(j + 1, next);
        for (int half = 0; half < 2; ++half, ++n) {
          const int s = n % P::stages;
          if (n >= P::stages) ok = bar_wait(empty(s), (n / P::stages - 1) & 1, failed, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const char *from = (half ? a.v : a.k) + head * (half ? a.v_head : a.k_head);
          const int64_t page_bytes = half ? a.v_page : a.k_page;
          const uint32_t to = smem_at + P::ring + s * P::tile;
#pragma unroll 4
          for (int i = w; i < kKeys / kPer; i += kCopyWarps) {
            const int r = i * kPer + sub, run = (i * kPer) >> 5;
            const int2 mine = run == 0 ? p[0] : run == 1 ? p[1] : run == 2 ? p[2] : p[3];
            const int page = __shfl_sync(0xffffffffu, mine.x, r & 31);
            const int row = __shfl_sync(0xffffffffu, mine.y, r & 31);
            const bool real = page >= 0 && piece * 8 < a.dim;
            const char *src = real ? from + page * page_bytes +
                                         static_cast<int64_t>(row) * a.dim * 2 + piece * 16
                                   : from;
            const int bytes = real ? 16 : 0;  // 0: zeroed, nothing read
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             to + P::at(r, piece)),
                         "l"(src), "r"(bytes)
                         : "memory");
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          if (n >= kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
            finish(done++);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = next[i];
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (ok && done < n) finish(done++);
    } else if (warp == 8 && steps) {
      // --- products --------------------------------------------------------------------------
      const uint32_t elected = lane == 0;
      constexpr uint32_t s_desc = product<T>(kKeys, false), o_desc = product<T>(DIM, true);
      const auto scores = [&](int i, int s) {  // S_i = Q_i K^T
        const uint32_t q_at = smem_at + P::q + i * P::tile, k_at = smem_at + P::ring + s * P::tile;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          const uint32_t off = (k >> 2) * P::atom + (k & 3) * 32;
          mma_ss(tmem + 128 * i, operand(q_at + off, P::group, 16),
                 operand(k_at + off, P::group, 16), s_desc, k > 0, elected);
        }
        commit(s_full(i), elected);
      };
      const auto values = [&](int i, int s, bool add) {  // O_i (+)= P_i V
        const uint32_t v_at = smem_at + P::ring + s * P::tile;
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * k,
                 operand(v_at + k * 2 * P::group, P::group, P::atom), o_desc, add || k > 0,
                 elected);
      };
      const auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, bar_wait(bar, parity, failed, a.status));
      };
      bool ok = wait(q_full, 0) && wait(full(0), 0);
      if (ok) {
        fence_after();
        for (int i = 0; i < tiles; ++i) scores(i, 0);
        commit(empty(0), elected);
      }
      for (int j = 0; j < steps && ok; ++j) {
        const int nv = 2 * j + 1, nk = 2 * j + 2, sv = nv % P::stages, sk = nk % P::stages;
        const bool more = j + 1 < steps;
        ok = wait(full(sv), nv / P::stages & 1) && (!more || wait(full(sk), nk / P::stages & 1));
        for (int i = 0; i < tiles && ok; ++i) {
          ok = wait(p_full(i), j & 1);
          if (!ok) break;
          fence_after();
          values(i, sv, j > 0);
          if (more) scores(i, sk);
        }
        if (!ok) break;
        commit(empty(sv), elected);
        if (more) commit(empty(sk), elected);
      }
      commit(o_full, elected);
      // whatever was issued ends before the block's shared and tensor memory go
      bar_drain(o_full, 0, a.status);
    }
    __syncwarp();
  } else {
    // --- a row's thread --------------------------------------------------------------------------
    if (TMA) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int i = warp >> 2, r = tid & 127, row = i * kHalf + r;
    const bool real = row < t.rows;
    const int at = t.row + row, token = at / a.group, h = head * a.group + at - token * a.group;
    const int pos = real ? first_pos + token : -1;
    const float c = fabsf(a.scale_log2);  // a negative scale turns the queries' signs instead
    {
      const char *from = a.q + (t.query + token) * a.q_token + h * a.q_head;
      const uint32_t flip = a.scale_log2 < 0 ? 0x80008000u : 0u;
#pragma unroll
      for (int piece = 0; piece < DIM / 8; ++piece) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real && piece * 8 < a.dim) {
          x = pg::load16(from + piece * 16);
          x.x ^= flip, x.y ^= flip, x.z ^= flip, x.w ^= flip;
        }
        *reinterpret_cast<uint4 *>(smem + P::q + i * P::tile + P::at(r, piece)) = x;
      }
      fence_async();
      bar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp, lane at 16
    const uint32_t s_at = tmem + lanes + 128 * i, o_at = tmem + lanes + 256 + 128 * i;
    const int row_last = min(t.rows - 1, i * kHalf + kHalf - 1);
    const Seen mine(a, first_pos + (t.row + i * kHalf) / a.group,
                    first_pos + (t.row + row_last) / a.group, t.length);
    // Steps whole.. (as many as wholes) are blocks of the window that every row sees in full. What
    // the others need is worked out only there: two numbers are what the registers have room for.
    const int at_first = blocks.first - blocks.sink + b0;  // the key block at step 0
    const int whole =
        max(max(0, blocks.sink - b0), (max(both.low, 0) + kKeys - 1) / kKeys - at_first);
    const int whole_end = both.high < 0 ? 0 : min(steps, both.high / kKeys + 1 - at_first);
    const unsigned wholes = max(0, whole_end - whole);
    float m = -INFINITY, l = 0.0f;
    const bool active = i < tiles;
    bool ok = true;
    for (int j = 0; j < steps && active; ++j) {
      ok = __all_sync(0xffffffffu, bar_wait(s_full(i), j & 1, failed, a.status));
      if (!ok) break;
      fence_after();
      float s[kKeys];
      uint32_t *const s_bits = reinterpret_cast<uint32_t *>(s);
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_load(s_at + 32 * k, s_bits + 32 * k);
      wait_loads();
#pragma unroll
      for (int k = 0; k < 4; ++k) tie(s_bits + 32 * k);
      const int key0 = blocks.key_block(b0 + j) * kKeys;
      if (static_cast<unsigned>(j - whole) >= wholes) {
        asm volatile("" ::: "memory");  // a branch, not predicated instructions in every block
        if (TMA && i == 0 && !both.all(key0)) {
          // The values of a block that some row must not see in full, before this step's weights
          // are handed on: tile 0's are used first. A thread takes row r.
          const int n = 2 * j + 1, slot = n % P::stages;
          ok = bar_wait(full(slot), n / P::stages & 1, failed, a.status);
          bool odd = false;
          char *const values = smem + P::ring + slot * P::tile;
#pragma unroll 4
          for (int piece = 0; piece < DIM / 8; ++piece) {
            uint4 *at16 = reinterpret_cast<uint4 *>(values + P::at(r, piece));
            if (key0 + r >= t.length) *at16 = make_uint4(0, 0, 0, 0);
            else odd |= pg::clean<Type<T>::exponent>(at16);
          }
          if (odd) *const_cast<volatile int *>(&sh.odd) = 1;
          fence_async();
        }
        if (!mine.all(key0)) {
          const int to = pos - key0, from = a.window ? to - a.window : -1, sink = a.sinks - key0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // bit e: key 32 k + e is seen
            const auto below = [&](int n) {  // the bits of keys below n
              n -= 32 * k;
              return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
            };
            const uint32_t seen = below(to + 1) & (~below(from + 1) | below(sink));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen >> e & 1)) s[32 * k + e] = -INFINITY;
          }
        }
      }
      const float most = largest(s, m);
      // the first block's maximum stands until a row's has grown by 2^8 (or is NaN)
      if (j == 0) {
        m = most;
      } else if (__any_sync(0xffffffffu, !((most - m) * c <= kGrow))) {
        const float f = m == -INFINITY ? 0.0f : pg::exp2_fast((m - most) * c);
        m = most;
        l *= f;
#pragma unroll
        for (int k = 0; k < DIM / 32; ++k) {
          uint32_t x[32];
          tmem_load(o_at + 32 * k, x);
          wait_loads();
          tie(x);
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
          tmem_store(o_at + 32 * k, x);
        }
      }
      // an infinite maximum gives NaN, as the formula does, in every weight
      const float base =
          m == -INFINITY ? 0.0f : m == INFINITY ? NAN : Type<T>::shift - m * c;
      Two sum[2] = {Two(l, 0.0f), Two(0.0f, 0.0f)};
      const Two c2(c, c), base2(base, base);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float y, z;
          fma(Two(s[64 * k + 2 * e], s[64 * k + 2 * e + 1]), c2, base2).get(y, z);
          y = pg::exp2_fast(y);
          z = pg::exp2_fast(z);
          sum[e & 1] = add(sum[e & 1], Two(y, z));
          x[e] = Type<T>::pack(y, z);
        }
        tmem_store(s_at + 32 * k, x);
      }
      {
        float y, z;
        add(sum[0], sum[1]).get(y, z);
        l = y + z;
      }
      wait_stores();
      fence_before();
      bar_arrive(p_full(i));
    }
    if (steps && active && ok) ok = bar_wait(o_full, 0, failed, a.status);
    ok = __all_sync(0xffffffffu, ok);
    fence_after();
    const bool have = steps > 0 && active && ok;  // O holds something

    // 32 columns of the row's result, before it is divided by l
    const auto result = [&](int k, float *x) {
      if (!have) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0.0f;
        return;
      }
      tmem_load(o_at + 32 * k, reinterpret_cast<uint32_t *>(x));
      wait_loads();
      tie(reinterpret_cast<uint32_t *>(x));
      bool lost = false;
#pragma unroll
      for (int e = 0; e < 32; ++e) lost |= !(fabsf(x[e]) < INFINITY);
      // a score that is NaN or +inf makes l NaN, and with it all the row's results
      if (pos < 0 || !(l < INFINITY) || !(lost || *const_cast<volatile int *>(&sh.odd))) return;
      float y[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) y[e] = x[e];
      add_values<T>(a, t.pages, t.length, blocks, both, b0, steps, head, pos, k, lost, y);
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = y[e];
    };
    const auto write = [&](int k, const float *x, float inv) {
      char *to = a.out + (t.query + token) * a.out_token + h * a.out_head + 64 * k;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * k + 8 * q < a.dim) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pos < 0 ? 0u : Type<T>::pack(x[8 * q + 2 * e] * inv, x[8 * q + 2 * e + 1] * inv);
          *reinterpret_cast<uint4 *>(to + 16 * q) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    if (a.parts == 1) {
      const float inv = l == 0.0f ? NAN : 1.0f / l;  // 0: all its scores are -inf, 0 / 0
#pragma unroll 1
      for (int k = 0; k < DIM / 32; ++k) {
        float x[32];
        result(k, x);
        if (real) write(k, x, inv);
      }
    } else {
      // Every part leaves its rows, four columns of all rows together; the last one to arrive
      // joins them, in the parts' order.
      const int64_t pair = static_cast<int64_t>(tile_id) * a.heads + head;
      constexpr int64_t size = static_cast<int64_t>(kRows) * (DIM + 2);
      float *all = a.partial + pair * a.parts * size;
      float *to = all + part * size;
      const auto o_of = [&](float *base, int c4) {
        return reinterpret_cast<float4 *>(base) + c4 * kRows + row;
      };
      const auto ml_of = [&](float *base) {
        return reinterpret_cast<float2 *>(base + kRows * DIM) + row;
      };
#pragma unroll 1
      for (int k = 0; k < DIM / 32; ++k) {
        float x[32];
        result(k, x);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *o_of(to, 8 * k + q) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
      }
      *ml_of(to) = make_float2(m, l);
      __threadfence();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (tid == 0) sh.last = atomicInc(a.arrived + pair, a.parts - 1) == a.parts - 1u;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (sh.last) {
        __threadfence();
        float top = -INFINITY, total = 0.0f;
        for (int p = 0; p < a.parts; ++p) top = fmaxf(top, __ldcg(ml_of(all + p * size)).x);
        for (int p = 0; p < a.parts; ++p) {
          const float2 ml = __ldcg(ml_of(all + p * size));
          total += ml.x == -INFINITY ? 0.0f : ml.y * pg::exp2_fast((ml.x - top) * c);
        }
        const float inv = total == 0.0f ? NAN : 1.0f / total;
#pragma unroll 1
        for (int k = 0; k < DIM / 32; ++k) {
          float x[32] = {};
          for (int p = 0; p < a.parts; ++p) {
            const float pm = __ldcg(ml_of(all + p * size)).x;
            const float f = pm == -INFINITY ? 0.0f : pg::exp2_fast((pm - top) * c);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 y = __ldcg(o_of(all + p * size, 8 * k + q));
              x[4 * q] = fmaf(f, y.x, x[4 * q]);
              x[4 * q + 1] = fmaf(f, y.y, x[4 * q + 1]);
              x[4 * q + 2] = fmaf(f, y.z, x[4 * q + 2]);
              x[4 * q + 3] = fmaf(f, y.w, x[4 * q + 3]);
            }
          }
          if (real) write(k, x, inv);
        }
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// The tensor map of the keys or values: columns, a page's rows, heads and pages. (Heads and pages
// as one coordinate leave a fifth for the groups of eight rows and so one box for a whole run of
// keys, but the many small boxes cost nothing: 500 us each for 4096 new tokens of up to 8192.)
int encode(CUtensorMap *map, const Attention &a, const char *base, int64_t head, int64_t page) {
  const uint64_t dims[4] = {static_cast<uint64_t>(a.dim), static_cast<uint64_t>(a.page_size),
                            static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.pages)};
  const uint64_t strides[3] = {2ull * a.dim, static_cast<uint64_t>(head),
                               static_cast<uint64_t>(page)};
  const uint32_t box[4] = {64, 8, 1, 1};
  return pg_detail_tensormap(map, 4, reinterpret_cast<uintptr_t>(base), dims, strides, box);
}

template <class T, int DIM>
int launch_prompt(Attention a, int max_len, int64_t partial_bytes, int sms, cudaStream_t stream) {
  a.rows_per_tile = kRows;
  const int tiles = pg::tile_bound(a, kRows);
  if (tiles > 65535)
    return pg::argument_fail("pg_attention: %d queries of %d heads: too many tiles", a.queries,
                             a.group);
  a.parts = pg::choose_parts(a, tiles, kRows, DIM, kKeys, max_len, sms, partial_bytes);
  CUtensorMap k_map = {}, v_map = {};
  // a kv head's tiles of the latest queries, which see the most keys, go first
  const dim3 grid(a.heads, tiles, a.parts);
  const int run = std::gcd(a.page_size, kKeys);  // the keys that a page and a block always share
  if (run < 8)
    return pg::launch<prompt_kernel<T, DIM, false>>("prompt_kernel", grid, kThreads,
                      Plan<DIM>::bytes, stream, a, k_map, v_map, run);
  int rc = encode(&k_map, a, a.k, a.k_head, a.k_page);
  if (!rc) rc = encode(&v_map, a, a.v, a.v_head, a.v_page);
  if (rc) return rc;
  return pg::launch<prompt_kernel<T, DIM, true>>("prompt_kernel", grid, kThreads,
                    Plan<DIM>::bytes, stream, a, k_map, v_map, run);
}

}  // namespace

namespace pg {

int prompt_16bit(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                 cudaStream_t stream) {
  if (bf16)
    return a.dim <= 64
               ? launch_prompt<__nv_bfloat16, 64>(a, max_len, partial_bytes, sms, stream)
               : launch_prompt<__nv_bfloat16, 128>(a, max_len, partial_bytes, sms, stream);
  return a.dim <= 64 ? launch_prompt<__half, 64>(a, max_len, partial_bytes, sms, stream)
                     : launch_prompt<__half, 128>(a, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

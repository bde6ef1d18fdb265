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
// Over a cache in 8 bits seven warps (9 to 15) widen what they have copied to f16, for both types, or the
// keys and values were widened before (attention_prompt_8bit.cu, which says when).
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
#pragma once

#include "attention.cuh"

#include <cuda.h>

#include <numeric>
#include <type_traits>

// Encodes a tensor map of 2-byte elements, 128-byte swizzled (launcher.cpp).
int pg_detail_tensormap(void *map, int rank, uint64_t base, const uint64_t *dims,
                        const uint64_t *strides_bytes, const uint32_t *box);

namespace {

using pg::Attention;
using pg::Blocks;
using pg::max3;
using pg::Sight;
using pg::Tile;
using pg::Two;

constexpr int kKeys = 128, kRows = 256, kHalf = 128;
constexpr int kThreads = 384;
constexpr int kThreads8 = 512, kConvertWarps = 7;  // of a cache in 8 bits
constexpr int kCopyWarps = 2, kCopyThreads = 32 * kCopyWarps;  // without TMA
constexpr int kLag = 2;  // tiles whose cp.async copies are in flight before the oldest is waited for
constexpr float kGrow = 8.0f;
constexpr unsigned long long kWaitNs = 2000000000ull;

// What a cache holds: numbers of the type T; f16 ones whatever T is, as 2^-k (keys) and 2^-v (values) of
// what they are, with the ints k and v for each page, of kKeys keys, at k_scale; the whole numbers of 8
// bits as f16 ones, with Scales for each page there; or the 8 bits.
enum Held { kOfType, kShifted, kWhole, kBytes };

struct Scales {
  int shift, unused[3];
  float k[128], v[128];  // v's as 2^-shift of what they are, 1 at most
};

template <int DIM, Held HELD>
struct Plan {
  // 128 queries, keys or values: by eight rows, then by 64 columns, each such 1024 bytes swizzled
  static constexpr int atom = 1024, chunks = DIM / 64, group = chunks * atom;
  static constexpr int tile = 16 * group;
  static constexpr int raw = HELD == kBytes ? kKeys * DIM : 0;  // keys or values in 8 bits, on their way
  static constexpr int stages = DIM == 128 ? HELD >= kWhole ? 4 : 5 : 8;
  static constexpr int scales = HELD == kWhole ? 8 * 1024 : 0;  // a step's, for each warp of rows
  static constexpr int q = 0, ring = 2 * tile, raws = ring + stages * tile, ks = raws + 2 * raw,
                       bars = ks + scales;
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

// 16 numbers of 8 bits times their scale, rounded to f16.
__device__ __forceinline__ void widen(const uint4 &raw, float scale, uint4 *to) {
  const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u,
                         raw.w ^ 0x80808080u};
  const Two off(-8388736.0f, -8388736.0f), by(scale, scale);  // 2^23 + 128
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t of = w[i / 2];
    const Two x(__uint_as_float(__byte_perm(of, 0x4b000000u, i & 1 ? 0x7442 : 0x7440)),
                __uint_as_float(__byte_perm(of, 0x4b000000u, i & 1 ? 0x7443 : 0x7441)));
    float y, z;
    mul(add(x, off), by).get(y, z);
    out[i] = Type<__half>::pack(y, z);
  }
  to[0] = make_uint4(out[0], out[1], out[2], out[3]);
  to[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

// e, so that 2^-e brings scales of at most `top`, as bits, to 2^7..2^8, and numbers to 2^15. What falls below
// f16's 2^-14 so is under 2^-28 of the largest. A row's weights are held times 2^e of its values, so for
// those e is at least -60: the weights of values that are all 0 must not be lost beside others.
__device__ __forceinline__ int shift_of(unsigned top, bool values) {
  return max(static_cast<int>(top >> 23) - 134, values ? -60 : -126);
}
// A scale's magnitude as bits, 0 if it is not finite.
__device__ __forceinline__ unsigned magnitude(const char *scale) {
  const unsigned x = *reinterpret_cast<const unsigned *>(scale) & 0x7fffffffu;
  return x < 0x7f800000u ? x : 0;
}

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
  unsigned k_top[kThreads8 / 32], v_top[kThreads8 / 32];  // kBytes: the largest scales a warp has seen
};

// Adds the values that are not finite and that the query at `pos` sees to 32 columns of its result: of
// all blocks of keys, or of those that some row must not see in full. A function of its own for the
// registers, as it is hardly ever called: in the kernel it made every step slower (508 us for 498).
template <class T, bool TREE, bool K8>
__device__ __noinline__ void add_values(const Attention &a, const int *pages, int length, Blocks blocks,
                                        Seen both, int b0, int steps, int head, Sight<TREE> sight,
                                        int k, bool all, float *x) {
  uint32_t met = 0;
  for (int j = 0; j < steps; ++j) {
    const int key0 = blocks.key_block(b0 + j) * kKeys;
    if (!all && both.all(key0)) continue;
    for (int key = key0; key < min(key0 + kKeys, length); ++key) {
      if (!sight.sees(a, key)) continue;
      const int page = pages[key / a.page_size];
      if (page < 0 || page >= a.pages) continue;
      constexpr int size = K8 ? 1 : 2;
      const int row = key % a.page_size;
      const char *v = a.v + page * a.v_page + head * a.v_head +
                      static_cast<int64_t>(row) * a.dim * size + 32 * size * k;
      float scale = 0.0f;
      if constexpr (K8) {
        scale = *reinterpret_cast<const float *>(a.v_scale + page * a.vs_page + head * a.vs_head +
                                                 row * 4ll);
        if (fabsf(scale) < INFINITY) continue;
      }
      for (int c = 0; c < 32; c += 2) {
        if (32 * k + c >= a.dim) break;
        float value[2];
        if constexpr (K8) {
          value[0] = scale * static_cast<int8_t>(v[c]), value[1] = scale * static_cast<int8_t>(v[c + 1]);
        } else {
          const uint32_t w = *reinterpret_cast<const uint32_t *>(v + 2 * c);
          value[0] = Type<T>::low(w), value[1] = Type<T>::high(w);
        }
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
// TREE: a sequence's new tokens are a tree. Where numbers are SHIFTED, queries are brought into f16 too, by
// row; a row's scores are in powers of 2, with v added to them, so that its weights are what they are times
// 2^v as its maximum is, and l takes them times 2^-v. Where they are WHOLE, scores are multiplied by their
// keys' scales, and weights by their values', which makes two f16 numbers: the rounded one and the rest.
template <class T, int DIM, bool TMA, bool TREE, Held HELD>
__global__ void __launch_bounds__(HELD == kBytes ? kThreads8 : kThreads, 1)
    prompt_kernel(const __grid_constant__ Attention a, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map, int run) {
  constexpr bool SHIFTED = HELD != kOfType, K8 = HELD == kBytes, WHOLE = HELD == kWhole;
  using P = Plan<DIM, HELD>;
  using C = std::conditional_t<SHIFTED, __half, T>;  // what products are of
  static_assert(!(TMA && K8), "keys in 8 bits come by cp.async");
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
  // a tree's: they see what is before it, and some may see all of it
  const int lo = TREE ? first_pos - 1 : first_pos + t.row / a.group;
  const int hi = TREE ? t.length - 1 : first_pos + (t.row + t.rows - 1) / a.group;
  const Blocks blocks = pg::blocks_of(a, lo, hi, kKeys);
  const Seen both(a, lo, hi, t.length);
  const int parts =
      TREE ? max(1, min(a.parts, (blocks.count + a.part_blocks - 1) / a.part_blocks)) : a.parts;
  if (TREE && part >= parts) return;
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks.count) * part / parts);
  const int steps =
      static_cast<int>(static_cast<int64_t>(blocks.count) * (part + 1) / parts) - b0;

  const uint32_t smem_at = shared_at(smem), bars = smem_at + P::bars;
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (P::stages + s); };
  const uint32_t q_full = bars + 16 * P::stages;
  const auto s_full = [&](int i) { return q_full + 8 + 8 * i; };
  const auto p_full = [&](int i) { return q_full + 24 + 8 * i; };
  const uint32_t o_full = q_full + 40;
  if (tid == 0) {
    for (int s = 0; s < P::stages; ++s) {
      bar_init(full(s), TMA ? 1 : K8 ? 32 * kConvertWarps : kCopyThreads);
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
  if constexpr (K8) {  // one shift for all keys of the part, and one for its values
    unsigned k_top = 0, v_top = 0;
#pragma unroll 4
    for (int n = tid; n < steps * kKeys; n += kThreads8) {
      const int key = blocks.key_block(b0 + n / kKeys) * kKeys + n % kKeys;
      if (key >= t.length) continue;
      const int entry = pg::page_index(a, key), page = t.pages[entry];
      if (page < 0 || page >= a.pages) continue;
      const int64_t row = (key - entry * a.page_size) * 4ll;
      k_top = max(k_top, magnitude(a.k_scale + page * a.ks_page + head * a.ks_head + row));
      v_top = max(v_top, magnitude(a.v_scale + page * a.vs_page + head * a.vs_head + row));
    }
    sh.k_top[warp] = __reduce_max_sync(0xffffffffu, k_top);
    sh.v_top[warp] = __reduce_max_sync(0xffffffffu, v_top);
  }
  fence_before();
  __syncthreads();
  fence_after();
  int2 shift = make_int2(0, 0);
  if constexpr (K8) {
    unsigned k_top = 0, v_top = 0;
#pragma unroll
    for (int w = 0; w < kThreads8 / 32; ++w) k_top = max(k_top, sh.k_top[w]), v_top = max(v_top, sh.v_top[w]);
    shift = make_int2(shift_of(k_top, false), shift_of(v_top, true));
  }
  const uint32_t tmem = sh.tmem;  // S and P of tile i at 128 i, O at 256 + 128 i
  volatile int *failed = &sh.failed;

  // Registers: three groups of 128 threads start with 168 each; the rows' threads, which hold a
  // row of S and what is made of it, take what the third group can do without (2 x 232 + 40 or
  // 2 x 200 + 104 = 3 x 168). With keys in 8 bits there are four groups of 128 each: 2 x 200 + 2 x 56.
  if (warp >= 8) {
    if (TMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    else if (K8) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
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
    } else if (K8 && warp >= 9) {
      // --- keys and values in 8 bits: copied 16 bytes at a time to where the same thread takes them up a
      // step later, widens them to f16, and hands them on in the products' layout --
      const int w = warp - 9;
      constexpr int kPieces = DIM / 16, kPer = 32 / kPieces;  // 16 bytes of a row; rows a warp takes at once
      constexpr int kMine = (kKeys / kPer + kConvertWarps - 1) / kConvertWarps;
      const int sub = lane / kPieces, piece = lane % kPieces;
      const bool column = piece * 16 < a.dim;
      // where a thread's m-th row of step j is, among the pages
      const auto row_key = [&](int j, int m) {
        return blocks.key_block(b0 + j) * kKeys + (m * kConvertWarps + w) * kPer + sub;
      };
      const auto page_for = [&](int j, int m) {  // as the table names it; -1: there is no such key
        if (j >= steps || (m * kConvertWarps + w) * kPer >= kKeys) return -1;
        const int key = row_key(j, m);
        if (key >= t.length) return -1;
        const int page = t.pages[pg::page_index(a, key)];
        return page < 0 ? a.pages : page;
      };
      const auto place = [&](int half, int m) {  // a thread's m-th row's 16 bytes
        return smem_at + P::raws + half * P::raw +
               ((m * kConvertWarps + w) * kPer * kPieces + lane) * 16;
      };
      const float by[2] = {pg::power_of_2(-shift.x), pg::power_of_2(-shift.y)};
      float scales[2][kMine];
      int pages[kMine];
      const auto issue = [&](int half, int j) {
        const char *from = (half ? a.v : a.k) + head * (half ? a.v_head : a.k_head) + piece * 16;
        const char *of = (half ? a.v_scale : a.k_scale) + head * (half ? a.vs_head : a.ks_head);
        const int64_t page_bytes = half ? a.v_page : a.k_page;
        const int64_t of_bytes = half ? a.vs_page : a.ks_page;
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
          const bool real = pages[m] >= 0;
          const int key = row_key(j, m), row = key - pg::page_index(a, key) * a.page_size;
          scales[half][m] =
              real ? *reinterpret_cast<const float *>(of + pages[m] * of_bytes + row * 4ll) : 0.0f;
          const char *src = real && column ? from + pages[m] * page_bytes +
                                                 static_cast<int64_t>(row) * a.dim
                                           : from;
          const int bytes = real && column ? 16 : 0;  // 0: zeroed, nothing read
          if ((m * kConvertWarps + w) * kPer < kKeys)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place(half, m)),
                         "l"(src), "r"(bytes)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const auto checked = [&](int page) {
        if (page >= a.pages) {
          atomicOr(a.status, PG_CACHE_BAD_PAGE);
          return -1;
        }
        return page;
      };
      int next[kMine];
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        pages[m] = checked(page_for(0, m));
        next[m] = page_for(1, m);
      }
      issue(0, 0);
      issue(1, 0);
      bool ok = true;
      for (int j = 0; j < steps && ok; ++j) {
        const int key0 = blocks.key_block(b0 + j) * kKeys;
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
          pages[m] = checked(next[m]);
          next[m] = page_for(j + 2, m);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int n = 2 * j + half, s = n % P::stages;
          if (n >= P::stages) ok = bar_wait(empty(s), (n / P::stages - 1) & 1, failed, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          char *const to = smem + P::ring + s * P::tile;
          // values that some row must not see are looked over: what is not finite is zeroed here
          const bool look = half && !both.all(key0);
#pragma unroll
          for (int m = 0; m < kMine; ++m) {
            const int r = (m * kConvertWarps + w) * kPer + sub;
            if (r - sub >= kKeys) break;
            const float scale = scales[half][m];
            uint4 out[2];
            widen(*reinterpret_cast<const uint4 *>(smem + (place(half, m) - smem_at)), scale * by[half], out);
            if (look && !(fabsf(scale) < INFINITY)) {
              bool odd = pg::clean<Type<C>::exponent>(out);
              odd |= pg::clean<Type<C>::exponent>(out + 1);
              if (odd) *const_cast<volatile int *>(&sh.odd) = 1;
            }
            *reinterpret_cast<uint4 *>(to + P::at(r, 2 * piece)) = out[0];
            *reinterpret_cast<uint4 *>(to + P::at(r, 2 * piece + 1)) = out[1];
          }
          fence_async();
          bar_arrive(full(s));
          issue(half, j + 1);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (!TMA && !K8 && (warp == 9 || warp == 10)) {
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
              odd |= pg::clean<Type<C>::exponent>(reinterpret_cast<uint4 *>(smem + P::ring + s * P::tile +
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
      constexpr uint32_t s_desc = product<C>(kKeys, false), o_desc = product<C>(DIM, true);
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
        if constexpr (WHOLE) {
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 64 + 8 * k,
                   operand(v_at + k * 2 * P::group, P::group, P::atom), o_desc, true, elected);
        }
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
    const Sight<TREE> sight = real ? Sight<TREE>::of(a, first_pos, t.count, t.query, token)
                                   : Sight<TREE>{-1, 0, 0};
    const int pos = sight.pos;
    const float c = fabsf(a.scale_log2);  // a negative scale turns the queries' signs instead
    int q_shift = 0;                      // queries are 2^-q_shift of what they are
    {
      const char *from = a.q + (t.query + token) * a.q_token + h * a.q_head;
      const uint32_t flip = a.scale_log2 < 0 ? 0x80008000u : 0u;
      constexpr bool to_f16 = !std::is_same_v<T, C>;
      if (to_f16 && real) {  // the largest that is finite comes to 2^14..2^15
        uint32_t top = 0;
#pragma unroll 4
        for (int piece = 0; piece < a.dim / 8; ++piece) {
          const uint4 x = pg::load16(from + piece * 16);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t y = w[e / 2] >> 16 * (e & 1) & 0x7fff;
            if (y < Type<T>::exponent) top = max(top, y);
          }
        }
        q_shift = max(static_cast<int>(top >> 7) - 141, -126);
      }
      const float by = pg::power_of_2(-q_shift);
#pragma unroll
      for (int piece = 0; piece < DIM / 8; ++piece) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real && piece * 8 < a.dim) {
          x = pg::load16(from + piece * 16);
          x.x ^= flip, x.y ^= flip, x.z ^= flip, x.w ^= flip;
          if constexpr (to_f16) {
            uint32_t *const w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = Type<C>::pack(Type<T>::low(w[e]) * by, Type<T>::high(w[e]) * by);
          }
        }
        *reinterpret_cast<uint4 *>(smem + P::q + i * P::tile + P::at(r, piece)) = x;
      }
      fence_async();
      bar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp, lane at 16
    const uint32_t s_at = tmem + lanes + 128 * i, o_at = tmem + lanes + 256 + 128 * i;
    const int row_last = min(t.rows - 1, i * kHalf + kHalf - 1);
    const Seen mine(a, TREE ? lo : first_pos + (t.row + i * kHalf) / a.group,
                    TREE ? hi : first_pos + (t.row + row_last) / a.group, t.length);
    // Steps whole.. (as many as wholes) are blocks of the window that every row sees in full. What
    // the others need is worked out only there: two numbers are what the registers have room for.
    const int at_first = blocks.first - blocks.sink + b0;  // the key block at step 0
    const int whole =
        max(max(0, blocks.sink - b0), (max(both.low, 0) + kKeys - 1) / kKeys - at_first);
    const int whole_end = both.high < 0 ? 0 : min(steps, both.high / kKeys + 1 - at_first);
    const unsigned wholes = max(0, whole_end - whole);
    float m = -INFINITY, l = 0.0f;
    const auto shifts_of = [&](int j) {  // asked for a step before
      if (HELD != kShifted || j >= steps) return shift;
      return *reinterpret_cast<const int2 *>(a.k_scale + t.pages[blocks.key_block(b0 + j)] * a.ks_page +
                                             head * a.ks_head);
    };
    int2 next = shifts_of(0);
    float4 *const ks = reinterpret_cast<float4 *>(smem + P::ks) + warp * 64;
    float4 next_k = {}, next_v = {};
    const auto scales_of = [&](int j) {
      if (!WHOLE || j >= steps) return;
      const Scales &x = *reinterpret_cast<const Scales *>(
          a.k_scale + t.pages[blocks.key_block(b0 + j)] * a.ks_page + head * a.ks_head);
      next.y = x.shift;
      next_k = reinterpret_cast<const float4 *>(x.k)[lane];
      next_v = reinterpret_cast<const float4 *>(x.v)[lane];
    };
    scales_of(0);
    const float m_to_2 = SHIFTED ? 1.0f : c;  // brings m into powers of 2
    const bool active = i < tiles;
    bool ok = true;
    for (int j = 0; j < steps && active; ++j) {
      ok = __all_sync(0xffffffffu, bar_wait(s_full(i), j & 1, failed, a.status));
      if (!ok) break;
      fence_after();
      if constexpr (HELD == kShifted) {
        shift = next;
        next = shifts_of(j + 1);
      }
      if constexpr (WHOLE) {
        __syncwarp();  // the last step's have been read
        ks[lane] = make_float4(next_k.x * c, next_k.y * c, next_k.z * c, next_k.w * c);
        ks[32 + lane] = next_v;
        shift = next;
        scales_of(j + 1);
        __syncwarp();
      }
      const float to_2 = WHOLE     ? 1.0f
                         : SHIFTED ? c * pg::power_of_2(min(max(q_shift + shift.x, -126), 127))
                                   : c;
      const float plus = static_cast<float>(shift.y);
      float s[kKeys];
      uint32_t *const s_bits = reinterpret_cast<uint32_t *>(s);
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_load(s_at + 32 * k, s_bits + 32 * k);
      wait_loads();
#pragma unroll
      for (int k = 0; k < 4; ++k) tie(s_bits + 32 * k);
      if constexpr (WHOLE) {
#pragma unroll
        for (int k = 0; k < kKeys / 4; ++k) {
          const float4 x = ks[k];
          mul(Two(s[4 * k], s[4 * k + 1]), Two(x.x, x.y)).get(s[4 * k], s[4 * k + 1]);
          mul(Two(s[4 * k + 2], s[4 * k + 3]), Two(x.z, x.w)).get(s[4 * k + 2], s[4 * k + 3]);
        }
      }
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
            else odd |= pg::clean<Type<C>::exponent>(at16);
          }
          if (odd) *const_cast<volatile int *>(&sh.odd) = 1;
          fence_async();
        }
        if (!mine.all(key0)) {
          const int from = a.window ? pos - key0 - a.window : -1, sink = a.sinks - key0;
          const int to = TREE ? sight.base - 1 - key0 : pos - key0;  // the last key of a row
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // bit e: key 32 k + e is seen
            const auto below = [&](int n) {  // the bits of keys below n
              n -= 32 * k;
              return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
            };
            uint32_t seen = below(to + 1) & (~below(from + 1) | below(sink));
            if constexpr (TREE) {  // and the tree's keys, the first of them at to + 1
              const int at = to + 1 - 32 * k;
              if (at > -64 && at < 32)
                seen |= static_cast<uint32_t>(at >= 0 ? sight.mask << at : sight.mask >> -at);
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen >> e & 1)) s[32 * k + e] = -INFINITY;
          }
        }
      }
      const float most = SHIFTED ? fmaxf(m, fmaf(largest(s, -INFINITY), to_2, plus)) : largest(s, m);
      // the first block's maximum stands until a row's has grown by 2^8 (or is NaN)
      if (j == 0) {
        m = most;
      } else if (__any_sync(0xffffffffu, !((most - m) * m_to_2 <= kGrow))) {
        const float f = m == -INFINITY ? 0.0f : pg::exp2_fast((m - most) * m_to_2);
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
      const float base = m == -INFINITY ? 0.0f
                         : m == INFINITY ? NAN
                         : SHIFTED            ? plus + Type<C>::shift - m
                                         : Type<C>::shift - m * c;
      Two sum[2] = {Two(SHIFTED ? 0.0f : l, 0.0f), Two(0.0f, 0.0f)};
      const Two c2(to_2, to_2), base2(base, base);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t x[32], rest[WHOLE ? 32 : 1];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float y, z;
          fma(Two(s[64 * k + 2 * e], s[64 * k + 2 * e + 1]), c2, base2).get(y, z);
          y = pg::exp2_fast(y);
          z = pg::exp2_fast(z);
          sum[e & 1] = add(sum[e & 1], Two(y, z));
          if constexpr (WHOLE) {
            const float2 by = reinterpret_cast<const float2 *>(ks + 32)[32 * k + e];
            mul(Two(y, z), Two(by.x, by.y)).get(y, z);
          }
          x[e] = Type<C>::pack(y, z);
          if constexpr (WHOLE) rest[e] = Type<C>::pack(y - Type<C>::low(x[e]), z - Type<C>::high(x[e]));
        }
        tmem_store(s_at + 32 * k, x);
        if constexpr (WHOLE) tmem_store(s_at + 64 + 32 * k, rest);  // the scores there have been read
      }
      {
        float y, z;
        add(sum[0], sum[1]).get(y, z);
        l = SHIFTED ? fmaf(y + z, pg::power_of_2(-shift.y), l) : y + z;
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
      if (sight.none() || !(l < INFINITY) || !(lost || *const_cast<volatile int *>(&sh.odd))) return;
      float y[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) y[e] = x[e];
      add_values<C, TREE, HELD == kBytes>(a, t.pages, t.length, blocks, both, b0, steps, head, sight, k, lost, y);
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
            w[e] = sight.none() ? 0u : Type<T>::pack(x[8 * q + 2 * e] * inv, x[8 * q + 2 * e + 1] * inv);
          *reinterpret_cast<uint4 *>(to + 16 * q) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    if (parts == 1) {
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
      if (tid == 0) sh.last = atomicInc(a.arrived + pair, parts - 1) == parts - 1u;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (sh.last) {
        __threadfence();
        float top = -INFINITY, total = 0.0f;
        for (int p = 0; p < parts; ++p) top = fmaxf(top, __ldcg(ml_of(all + p * size)).x);
        for (int p = 0; p < parts; ++p) {
          const float2 ml = __ldcg(ml_of(all + p * size));
          total += ml.x == -INFINITY ? 0.0f : ml.y * pg::exp2_fast((ml.x - top) * m_to_2);
        }
        const float inv = total == 0.0f ? NAN : 1.0f / total;
#pragma unroll 1
        for (int k = 0; k < DIM / 32; ++k) {
          float x[32] = {};
          for (int p = 0; p < parts; ++p) {
            const float pm = __ldcg(ml_of(all + p * size)).x;
            const float f = pm == -INFINITY ? 0.0f : pg::exp2_fast((pm - top) * m_to_2);
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

template <class T, int DIM, bool TREE, Held HELD>
int launch_prompt(Attention a, int max_len, int64_t partial_bytes, int sms, cudaStream_t stream) {
  a.rows_per_tile = kRows;
  int tiles = pg::tile_bound(a, kRows);
  if (TREE) {
    const int64_t most = a.batch * ((static_cast<int64_t>(PG_ATTENTION_TREE) * a.group + kRows - 1) / kRows);
    tiles = static_cast<int>(most < tiles ? most : tiles);
  }
  if (tiles > 65535)
    return pg::argument_fail("pg_attention: %d queries of %d heads: too many tiles", a.queries,
                             a.group);
  a.parts = pg::choose_parts(a, tiles, kRows, DIM, kKeys, max_len, sms, partial_bytes);
  if (TREE) {
    // A tree's few rows go over all of a context, so lengths of unlike size leave most SMs idle at the
    // end: long ones are cut, in parts as long as a third or a fourth of the longest (16 trees of 64
    // tokens on up to 16384 keys, 32 heads on 8 of 128: 277 us in one part, 149 so).
    const int64_t pairs = static_cast<int64_t>(tiles) * a.heads, longest = max_len / kKeys + 1;
    const int64_t each = pairs * kRows * (DIM + 2) * 4ll;
    int64_t parts = a.parts;
    if (parts == 1 && pairs <= pg::kCounters) {
      parts = 4ll * sms / pairs;
      parts = partial_bytes / each < parts ? partial_bytes / each : parts;
      parts = longest / 4 < parts ? longest / 4 : parts;
      a.parts = static_cast<int>(parts < 1 ? 1 : parts);
    }
    a.part_blocks = static_cast<int>((longest + a.parts - 1) / a.parts);
  }
  CUtensorMap k_map = {}, v_map = {};
  // a kv head's tiles of the latest queries, which see the most keys, go first
  const dim3 grid(a.heads, tiles, a.parts);
  const int run = std::gcd(a.page_size, kKeys);  // the keys that a page and a block always share
  if constexpr (HELD == kBytes) {
    return pg::launch<prompt_kernel<T, DIM, false, TREE, HELD>>("prompt_kernel", grid, kThreads8,
                      Plan<DIM, HELD>::bytes, stream, a, k_map, v_map, run);
  } else {
    if constexpr (HELD == kOfType)
      if (run < 8)
        return pg::launch<prompt_kernel<T, DIM, false, TREE, HELD>>("prompt_kernel", grid, kThreads,
                          Plan<DIM, HELD>::bytes, stream, a, k_map, v_map, run);
    int rc = encode(&k_map, a, a.k, a.k_head, a.k_page);
    if (!rc) rc = encode(&v_map, a, a.v, a.v_head, a.v_page);
    if (rc) return rc;
    return pg::launch<prompt_kernel<T, DIM, true, TREE, HELD>>("prompt_kernel", grid, kThreads,
                      Plan<DIM, HELD>::bytes, stream, a, k_map, v_map, run);
  }
}

template <class T, bool TREE, Held HELD>
int run_prompt_of(const Attention &a, int max_len, int64_t partial_bytes, int sms, cudaStream_t stream) {
  return a.dim <= 64 ? launch_prompt<T, 64, TREE, HELD>(a, max_len, partial_bytes, sms, stream)
                     : launch_prompt<T, 128, TREE, HELD>(a, max_len, partial_bytes, sms, stream);
}

template <bool TREE, Held HELD>
int run_prompt(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
               cudaStream_t stream) {
  return bf16 ? run_prompt_of<__nv_bfloat16, TREE, HELD>(a, max_len, partial_bytes, sms, stream)
              : run_prompt_of<__half, TREE, HELD>(a, max_len, partial_bytes, sms, stream);
}

}  // namespace

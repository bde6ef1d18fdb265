// Attention of one new token a sequence for the 16-bit types at head sizes of up to 128
// (pg_attention without starts).
//
// HBM bounds it: every key and value is read once and used for the query heads of its group
// only. So the work is cut evenly by keys, not by sequences: the blocks of 64 keys of all
// (sequence, kv head) pairs form one line, and block c takes the c-th of as many equal pieces of
// it as there are blocks. A pair whose keys lie in several pieces is joined by the last block that finishes one, in
// the pieces' order.
//
// Within a block each of four warps takes every fourth 16 keys by itself: it copies their rows
// into its own ring in shared memory (cp.async, 16 bytes a lane, rows of whole heads, swizzled so
// that the matrix loads meet no bank twice), and multiplies on the tensor cores (mma.sync
// m16n8k16: with at most 16 rows of queries a larger tile would be empty, and at one use of
// each key the memory is slower by far). A weight goes into the second product as the sum of two
// numbers of the values' type, the rounded weight and what the rounding left, so that the
// result is rounded once; that doubles the second product, which the memory hides.
#include "attention.cuh"

namespace {

using pg::Attention;
using pg::Blocks;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 16;             // keys a warp takes at a time
constexpr int kKeys = kStep * kWarps; // keys of a block's step
constexpr int kRows = 16;
constexpr int kPerSm = 2;             // blocks an SM holds

template <class T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  __device__ static void run(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
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

template <int DIM>
struct Ring {
  static constexpr int row = DIM * 2, chunks = DIM / 8;
  static constexpr int tile = kStep * row;        // 16 keys, or 16 values
  static constexpr int stage = 2 * tile;
  static constexpr int stages = 384 / DIM;
  static constexpr int warp = stages * stage;
  static constexpr int bytes = kWarps * warp;
  static_assert(warp >= kRows * (DIM + 2) * 4, "a warp's result takes its ring's place");
  __device__ static int at(int r, int chunk) { return r * row + ((chunk ^ (r & 7)) << 4); }
};

__device__ __forceinline__ int length_of(const Attention &a, int b, int *slot) {
  const int s = a.slots ? a.slots[b] : b;
  *slot = s;
  if (s < 0 || s >= a.slot_rows) {
    atomicOr(a.status, PG_CACHE_BAD_SLOT);
    return 0;
  }
  const int n = a.lens[s], most = a.width * a.page_size;
  if (n < 0 || n > most) {
    atomicOr(a.status, PG_CACHE_TOO_LONG);
    return n < 0 ? 0 : most;
  }
  return n;
}

__device__ __forceinline__ int blocks_in(const Attention &a, int length) {
  return pg::blocks_of(a, length - 1, length - 1, kKeys).count;
}

template <class T, int DIM>
__global__ void __launch_bounds__(kThreads, kPerSm) decode_kernel(Attention a) {
  using R = Ring<DIM>;
  extern __shared__ float4 smem4[];
  __shared__ uint32_t warp_sum[kWarps];
  __shared__ int found_b;
  __shared__ uint32_t found_before;
  __shared__ unsigned last;
  pg::wait_for_earlier_kernels();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const uint32_t row_groups = (a.group + kRows - 1) / kRows, per_block = a.heads * row_groups;
  const uint32_t c = blockIdx.x;

  // Every block works the line out for itself: thread i counts the units (blocks of keys of a
  // head and row group) of a run of sequences.
  const int run = (a.batch + kThreads - 1) / kThreads;
  const int first_b = min(tid * run, a.batch), end_b = min(first_b + run, a.batch);
  uint32_t mine = 0;
  for (int b = first_b; b < end_b; ++b) {
    int slot;
    const int n = length_of(a, b, &slot);
    mine += blocks_in(a, n);
    if (!n && b % gridDim.x == c)  // no key: zeros
      for (int h = 0; h < a.heads * a.group; ++h)
        for (int j = 0; j < a.dim / 8; ++j)
          *reinterpret_cast<uint4 *>(a.out + b * a.out_token + h * a.out_head + j * 16) =
              make_uint4(0, 0, 0, 0);
  }
  mine *= per_block;
  uint32_t upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += o;
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += warp_sum[w];
    total += warp_sum[w];
  }
  // The units of a piece; piece c is [c per, (c + 1) per). One is not too few: four sequences of
  // up to 777 keys take 12 us, with at least two 16.5, with four 19.5.
  const uint32_t per = (total + gridDim.x - 1) / gridDim.x;
  if (static_cast<uint64_t>(c) * per >= total) return;
  uint32_t u = c * per;
  const uint32_t u_end = min(total, u + per), before = upto - mine;
  if (u >= before && u < upto) {
    uint32_t at = before;
    for (int b = first_b; b < end_b; ++b) {
      int slot;
      const uint32_t units = blocks_in(a, length_of(a, b, &slot)) * per_block;
      if (u < at + units) {
        found_b = b;
        found_before = at;
        break;
      }
      at += units;
    }
  }
  __syncthreads();
  int b = found_b;
  uint32_t seq_before = found_before;

  char *ring = reinterpret_cast<char *>(smem4) + warp * R::warp;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  while (u < u_end) {
    int slot;
    const int length = length_of(a, b, &slot);
    const Blocks blocks = pg::blocks_of(a, length - 1, length - 1, kKeys);
    if (!blocks.count) {
      ++b;
      continue;
    }
    const uint32_t pair = (u - seq_before) / blocks.count;
    const int head = pair / row_groups, row0 = (pair % row_groups) * kRows;
    const int rows = min(kRows, a.group - row0);
    const uint32_t pair_first = seq_before + pair * blocks.count;
    const int block0 = u - pair_first;
    const uint32_t stop = min(u_end, pair_first + blocks.count);
    const int block1 = stop - pair_first;
    const int *pages = a.table + slot * a.table_row;
    const int pos = length - 1;

    // the queries' fragments: rows g and g + 8, columns 2 t and 2 t + 8 of each 16
    uint32_t q[DIM / 16][4];
#pragma unroll
    for (int k = 0; k < DIM / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = g + 8 * (i & 1), col = 16 * k + 2 * t4 + 8 * (i >> 1);
        q[k][i] = r < rows && col < a.dim
                      ? *reinterpret_cast<const uint32_t *>(
                            a.q + b * a.q_token + (head * a.group + row0 + r) * a.q_head + col * 2)
                      : 0u;
      }
    float o[DIM / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

    // The warp's steps are the blocks' 16 keys at 16 warp. A step whose keys all are seen and lie
    // in one page, as they do where pages are whole groups of 16, needs one look at the table and
    // one address; else lane r < 16 knows key r's page and row.
    const int steps = block1 - block0;
    const bool whole_pages = a.page_size % kStep == 0;
    const auto first_key = [&](int i) {
      return blocks.key_block(block0 + i) * kKeys + kStep * warp;
    };
    const auto all_seen = [&](int key) {
      return key + kStep - 1 <= pos &&
             (!a.window || key > pos - a.window || key + kStep <= a.sinks);
    };
    const auto page_for = [&](int i) {  // as the table names it; -1: not seen
      if (i >= steps) return -1;
      const int key = first_key(i);
      if (whole_pages && all_seen(key)) return pages[key / a.page_size];
      return pg::sees(a, pos, key + (lane & 15)) ? pages[(key + (lane & 15)) / a.page_size] : -1;
    };
    const int sub = lane / R::chunks, chunk = lane % R::chunks;
    const bool column = chunk * 8 < a.dim;
    const int64_t row_bytes = 2ll * a.dim;
    const char *const k_head = a.k + head * a.k_head + chunk * 16;
    const char *const v_head = a.v + head * a.v_head + chunk * 16;
    constexpr int kCopies = kStep * R::chunks / 32, kRowsEach = 32 / R::chunks;
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
          const int mine_key = key + (lane & 15);
          if (pg::sees(a, pos, mine_key) && (page < 0 || page >= a.pages)) {
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
    int next = page_for(0);
#pragma unroll
    for (int i = 0; i < R::stages - 1; ++i) {
      const int page = next;
      next = page_for(i + 1);
      issue(i, page);
    }
    for (int i = 0; i < steps; ++i) {
      const int page = next;
      next = page_for(i + R::stages);
      issue(i + R::stages - 1, page);
      asm volatile("cp.async.wait_group %0;" ::"n"(R::stages - 1) : "memory");
      __syncwarp();
      const uint32_t ks = ring_at + (i % R::stages) * R::stage, vs = ks + R::tile;
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < DIM / 32; ++k)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t x[4];  // keys 8 n.. by columns 32 k.., four 8 x 8 matrices along the columns
          load_matrices(ks + R::at(8 * n + (lane & 7), 4 * k + (lane >> 3)), x);
          Mma<T>::run(s[n], q[2 * k], x[0], x[1]);
          Mma<T>::run(s[n], q[2 * k + 1], x[2], x[3]);
        }
      const int key = first_key(i);
      const bool masked = !all_seen(key);
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= a.scale_log2;
          if (masked && !pg::sees(a, pos, key + 2 * t4 + 8 * n + (e & 1))) s[n][e] = -INFINITY;
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
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = pg::exp2_fast(s[n][2 * h] - base[h]);
          const float y = pg::exp2_fast(s[n][2 * h + 1] - base[h]);
          l[h] += x + y;
          Mma<T>::split(x, y, hi[2 * n + h], lo[2 * n + h]);
        }
#pragma unroll
      for (int n = 0; n < DIM / 16; ++n) {
        uint32_t x[4];  // keys 0.. and 8.. by columns 16 n.. and 16 n + 8.., transposed
        load_matrices_t(vs + R::at(lane & 15, 2 * n + (lane >> 4)), x);
        Mma<T>::run(o[2 * n], hi, x[0], x[1]);
        Mma<T>::run(o[2 * n], lo, x[0], x[1]);
        Mma<T>::run(o[2 * n + 1], hi, x[2], x[3]);
        Mma<T>::run(o[2 * n + 1], lo, x[2], x[3]);
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

    const uint32_t c0 = pair_first / per, c1 = (pair_first + blocks.count - 1) / per;
    const bool alone = c0 == c1;
    constexpr int kPartial = kRows * (DIM + 2);
    // a block has at most two pairs that others share: one that its piece starts with, and one
    // it leaves in the middle of
    const auto slot_of = [&](uint32_t piece) {
      return a.partial + (2ll * piece + (pair_first > piece * per)) * kPartial;
    };
    // thread's columns: four of row `warp`, `warp + 4`, ...
    const int lanes = DIM / 4;
    for (int i = tid; i < kRows * lanes; i += kThreads) {
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
      if (alone) {
        if (r < rows && col < a.dim) {
          const float inv = 1.0f / sum;
          *reinterpret_cast<uint2 *>(a.out + b * a.out_token +
                                     (head * a.group + row0 + r) * a.out_head + col * 2) =
              make_uint2(Mma<T>::pack(acc.x * inv, acc.y * inv),
                         Mma<T>::pack(acc.z * inv, acc.w * inv));
        }
      } else {
        float *to = slot_of(c);
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
      if (tid == 0) last = atomicInc(a.arrived + c0, c1 - c0) == c1 - c0;
      __syncthreads();
      if (last) {
        __threadfence();
        for (int i = tid; i < rows * lanes; i += kThreads) {
          const int r = i / lanes, col = 4 * (i % lanes);
          float top = -INFINITY, sum = 0.0f;
          float4 acc = make_float4(0, 0, 0, 0);
          for (uint32_t p = c0; p <= c1; ++p) top = fmaxf(top, __ldcg(slot_of(p) + kRows * DIM + r));
          const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
          for (uint32_t p = c0; p <= c1; ++p) {
            const float *from = slot_of(p);
            const float f = pg::factor(__ldcg(from + kRows * DIM + r), base);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + r * DIM + col));
            sum += f * __ldcg(from + kRows * DIM + kRows + r);
            acc.x = fmaf(f, x.x, acc.x), acc.y = fmaf(f, x.y, acc.y);
            acc.z = fmaf(f, x.z, acc.z), acc.w = fmaf(f, x.w, acc.w);
          }
          if (col < a.dim) {
            const float inv = 1.0f / sum;
            *reinterpret_cast<uint2 *>(a.out + b * a.out_token +
                                       (head * a.group + row0 + r) * a.out_head + col * 2) =
                make_uint2(Mma<T>::pack(acc.x * inv, acc.y * inv),
                           Mma<T>::pack(acc.z * inv, acc.w * inv));
          }
        }
      }
    }
    __syncthreads();  // the rings are free again
    u = stop;
    if (u == seq_before + blocks.count * per_block) {
      seq_before = u;
      ++b;
    }
  }
}

template <class T, int DIM>
int launch_decode(const Attention &a, int sms, cudaStream_t stream) {
  return pg::launch<decode_kernel<T, DIM>>("decode_kernel", dim3(kPerSm * sms), kThreads,
                                           Ring<DIM>::bytes, stream, a);
}

}  // namespace

namespace pg {

bool decode_fits(const Attention &a, int max_len) {
  const int64_t pairs = static_cast<int64_t>(a.batch) * a.heads * ((a.group + kRows - 1) / kRows);
  return pairs * (max_len / kKeys + 2ll) < INT32_MAX;
}

int decode_16bit(const Attention &a, bool bf16, int sms, cudaStream_t stream) {
  if (bf16)
    return a.dim <= 64 ? launch_decode<__nv_bfloat16, 64>(a, sms, stream)
                       : launch_decode<__nv_bfloat16, 128>(a, sms, stream);
  return a.dim <= 64 ? launch_decode<__half, 64>(a, sms, stream)
                     : launch_decode<__half, 128>(a, sms, stream);
}

}  // namespace pg

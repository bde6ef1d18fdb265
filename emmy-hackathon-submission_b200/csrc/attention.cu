// Attention over a paged cache in 32-bit arithmetic, for every type and head size
// (pg_attention in include/ptxgen_b200.h).
#include "attention.cuh"

namespace {

using pg::Attention;
using pg::Blocks;
using pg::Tile;
using pg::Two;

constexpr int kThreads = 256;
constexpr int kKeys = 64;  // keys a step takes

template <class T> struct Load;  // 16 bytes of T as f32
template <> struct Load<float> {
  static constexpr int n = 4;
  __device__ static void get(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <> struct Load<__nv_bfloat16> {
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
template <> struct Load<__half> {
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

__device__ __forceinline__ void store(float x, float *to) { *to = x; }
__device__ __forceinline__ void store(float x, __nv_bfloat16 *to) { *to = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store(float x, __half *to) { *to = __float2half_rn(x); }

template <int ROWS, int DIM>
struct Layout {
  static constexpr int stride = DIM + 4;  // floats: eight rows' 16-byte pieces on all banks
  static constexpr int p_stride = kKeys + 4;
  static constexpr int q = 0, k = q + ROWS * stride, v = k + kKeys * stride,
                       p = v + kKeys * stride, floats = p + ROWS * p_stride;
  static constexpr int bytes = floats * 4 + kKeys * 16;
};

// A block takes ROWS rows (queries times heads of one kv head's group) and a part of the blocks
// of 64 keys they see. 16 threads share a row group: each has R rows and J of the keys of a step,
// then R rows and DIM / 16 of the columns of o. The products run two at a time in FMA (f32x2) from
// shared memory, whose reads and the barriers of a step bound it: 1024 f32 queries of 16 heads on
// up to 4096 keys take 1.14 ms, 26 TFLOP/s. The 16-bit types have kernels on the tensor cores at
// head sizes of up to 128.
// A value in a masked place may be anything: its weight is 0 and, where a step holds a value
// that is not finite, the masked places are skipped one by one.
template <class T, int ROWS, int DIM>
__global__ void __launch_bounds__(kThreads) attention_kernel(Attention a) {
  using L = Layout<ROWS, DIM>;
  constexpr int R = ROWS / 16, C = DIM / 64, J = kKeys / 16;
  extern __shared__ float4 smem4[];
  float *smem = reinterpret_cast<float *>(smem4);
  float *qs = smem + L::q, *ks = smem + L::k, *vs = smem + L::v, *ps = smem + L::p;
  int64_t *key_at = reinterpret_cast<int64_t *>(smem + L::floats);  // k's and v's byte offsets
  __shared__ unsigned last;
  pg::wait_for_earlier_kernels();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, row0 = ty * R;
  const int head = blockIdx.y, part = blockIdx.z;
  const Tile t = pg::find_tile(a, gridDim.x - 1 - blockIdx.x);
  if (!t.rows) return;
  const int first_pos = t.length - t.count;
  const int lo = first_pos + t.row / a.group, hi = first_pos + (t.row + t.rows - 1) / a.group;
  const Blocks blocks = pg::blocks_of(a, lo, hi, kKeys);
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks.count) * part / a.parts);
  const int b1 = static_cast<int>(static_cast<int64_t>(blocks.count) * (part + 1) / a.parts);
  const int pieces = a.dim / Load<T>::n;

  for (int i = tid; i < ROWS * (DIM / Load<T>::n); i += kThreads) {
    const int r = i / (DIM / Load<T>::n), c = i % (DIM / Load<T>::n);
    float x[Load<T>::n] = {};
    if (r < t.rows && c < pieces) {
      const int at = t.row + r, h = head * a.group + at % a.group;
      Load<T>::get(pg::load16(a.q + (t.query + at / a.group) * a.q_token + h * a.q_head + c * 16),
                   x);
    }
#pragma unroll
    for (int j = 0; j < Load<T>::n; ++j) qs[r * L::stride + c * Load<T>::n + j] = x[j];
  }

  float m[R], l[R], o[R][4 * C];
  int pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
    pos[r] = row0 + r < t.rows ? first_pos + (t.row + row0 + r) / a.group : -1;
#pragma unroll
    for (int c = 0; c < 4 * C; ++c) o[r][c] = 0.0f;
  }

  for (int b = b0; b < b1; ++b) {
    const int key0 = blocks.key_block(b) * kKeys;
    __syncthreads();
    if (tid < kKeys) {
      const int key = key0 + tid;
      int64_t ka = -1, va = -1;
      if (key < t.length) {
        const int page = pg::page_of(a, t, key);
        const int64_t in_page = static_cast<int64_t>(key % a.page_size) * a.dim * sizeof(T);
        if (page >= 0) {
          ka = page * a.k_page + head * a.k_head + in_page;
          va = page * a.v_page + head * a.v_head + in_page;
        }
      }
      key_at[tid] = ka;
      key_at[kKeys + tid] = va;
    }
    __syncthreads();
    bool odd = false;
    // loads in batches, so that they are in flight together
    constexpr int kAll = kKeys * (DIM / Load<T>::n), kBatch = 4;
    for (int i0 = tid; i0 < kAll; i0 += kBatch * kThreads) {
      uint4 kk[kBatch], vv[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kThreads, r = i / (DIM / Load<T>::n), c = i % (DIM / Load<T>::n);
        kk[u] = vv[u] = make_uint4(0, 0, 0, 0);
        if (i < kAll && key_at[r] >= 0 && c < pieces) {
          kk[u] = pg::load16(a.k + key_at[r] + c * 16);
          vv[u] = pg::load16(a.v + key_at[kKeys + r] + c * 16);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kThreads, r = i / (DIM / Load<T>::n), c = i % (DIM / Load<T>::n);
        if (i >= kAll) break;
        float x[Load<T>::n], y[Load<T>::n];
        Load<T>::get(kk[u], x);
        Load<T>::get(vv[u], y);
        float *const k_to = ks + r * L::stride + c * Load<T>::n;
        float *const v_to = vs + r * L::stride + c * Load<T>::n;
#pragma unroll
        for (int j = 0; j < Load<T>::n; j += 4) {
          *reinterpret_cast<float4 *>(k_to + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          *reinterpret_cast<float4 *>(v_to + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
        }
#pragma unroll
        for (int j = 0; j < Load<T>::n; ++j) odd |= !(fabsf(y[j]) < INFINITY);
      }
    }
    odd = __syncthreads_or(odd);

    // two products an instruction: of the even and of the odd columns
    Two s2[R][J];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j) s2[r][j] = Two(0.0f, 0.0f);
#pragma unroll 4
    for (int d = 0; d < DIM; d += 4) {
      float4 q[R], k[J];
#pragma unroll
      for (int r = 0; r < R; ++r)
        q[r] = *reinterpret_cast<const float4 *>(qs + (row0 + r) * L::stride + d);
#pragma unroll
      for (int j = 0; j < J; ++j)
        k[j] = *reinterpret_cast<const float4 *>(ks + (tx + 16 * j) * L::stride + d);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          s2[r][j] = fma(Two(q[r].x, q[r].y), Two(k[j].x, k[j].y), s2[r][j]);
          s2[r][j] = fma(Two(q[r].z, q[r].w), Two(k[j].z, k[j].w), s2[r][j]);
        }
    }
    float s[R][J];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float x, y;
        s2[r][j].get(x, y);
        s[r][j] = x + y;
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int key = key0 + tx + 16 * j;
        const bool seen = pg::sees(a, pos[r], key) && key_at[tx + 16 * j] >= 0;
        s[r][j] = seen ? s[r][j] * a.scale_log2 : -INFINITY;
        top = fmaxf(top, s[r][j]);
      }
#pragma unroll
      for (int off = 8; off; off >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float base = top == -INFINITY ? 0.0f : top;
      const float f = pg::factor(m[r], base);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float p = pg::exp2_fast(s[r][j] - base);
        ps[(row0 + r) * L::p_stride + tx + 16 * j] = p;
        sum += p;
      }
#pragma unroll
      for (int off = 8; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      l[r] = l[r] * f + sum;
      m[r] = top;
#pragma unroll
      for (int c = 0; c < 4 * C; ++c) o[r][c] *= f;
    }
    __syncwarp();  // a row's weights come from its own half-warp
    if (!odd) {
#pragma unroll 4
      for (int j = 0; j < kKeys; ++j) {
        float4 v[C];
#pragma unroll
        for (int c = 0; c < C; ++c)
          v[c] = *reinterpret_cast<const float4 *>(vs + j * L::stride + 64 * c + 4 * tx);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float p = ps[(row0 + r) * L::p_stride + j];
#pragma unroll
          for (int c = 0; c < C; ++c) {
            float *const to = o[r] + 4 * c;
            fma(Two(p, p), Two(v[c].x, v[c].y), Two(to[0], to[1])).get(to[0], to[1]);
            fma(Two(p, p), Two(v[c].z, v[c].w), Two(to[2], to[3])).get(to[2], to[3]);
          }
        }
      }
    } else {
      for (int j = 0; j < kKeys; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (!pg::sees(a, pos[r], key0 + j)) continue;
          const float p = ps[(row0 + r) * L::p_stride + j];
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[r][4 * c + e] = fmaf(p, vs[j * L::stride + 64 * c + 4 * tx + e], o[r][4 * c + e]);
        }
    }
  }

  if (a.parts > 1) {
    // every part leaves its rows; the last one to arrive joins them, in the parts' order
    const int64_t pair = static_cast<int64_t>(gridDim.x - 1 - blockIdx.x) * a.heads + head;
    const int64_t size = static_cast<int64_t>(ROWS) * (a.dim + 2);
    float *all = a.partial + pair * a.parts * size;
    float *mine = all + part * size;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float *to = mine + (row0 + r) * (a.dim + 2);
      if (tx == 0) {
        to[0] = m[r];
        to[1] = l[r];
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (64 * c + 4 * tx + e < a.dim) to[2 + 64 * c + 4 * tx + e] = o[r][4 * c + e];
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicInc(a.arrived + pair, a.parts - 1) == a.parts - 1u;
    __syncthreads();
    if (!last) return;
    __threadfence();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll 8
      for (int i = 0; i < a.parts; ++i)
        top = fmaxf(top, __ldcg(all + i * size + (row0 + r) * (a.dim + 2)));
      const float base = top == -INFINITY ? 0.0f : top;
      l[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < 4 * C; ++c) o[r][c] = 0.0f;
#pragma unroll 4
      for (int i = 0; i < a.parts; ++i) {
        const float *from = all + i * size + (row0 + r) * (a.dim + 2);
        const float f = pg::factor(__ldcg(from), base);
        l[r] += f * __ldcg(from + 1);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (64 * c + 4 * tx + e < a.dim)
              o[r][4 * c + e] += f * __ldcg(from + 2 + 64 * c + 4 * tx + e);
      }
    }
  }

#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row0 + r >= t.rows) continue;
    const int at = t.row + row0 + r, h = head * a.group + at % a.group;
    T *to = reinterpret_cast<T *>(a.out + (t.query + at / a.group) * a.out_token + h * a.out_head);
    // a query before the sequence's start sees no key: zeros. Any other sees itself, so l = 0
    // means that all its scores are -inf, and 0 / 0 is what the formula gives.
    const float inv = 1.0f / l[r];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (64 * c + 4 * tx + e < a.dim)
          store(pos[r] < 0 ? 0.0f : o[r][4 * c + e] * inv, to + 64 * c + 4 * tx + e);
  }
}

template <class T, int ROWS, int DIM>
int launch_tiles(Attention a, int tiles, cudaStream_t stream) {
  a.rows_per_tile = ROWS;
  return pg::launch<attention_kernel<T, ROWS, DIM>>(
      "attention_kernel", dim3(tiles, a.heads, a.parts), kThreads, Layout<ROWS, DIM>::bytes, stream,
      a);
}

template <class T, int ROWS>
int launch_dim(const Attention &a, int tiles, cudaStream_t stream) {
  if (a.dim <= 64) return launch_tiles<T, ROWS, 64>(a, tiles, stream);
  if (a.dim <= 128) return launch_tiles<T, ROWS, 128>(a, tiles, stream);
  return launch_tiles<T, ROWS, 256>(a, tiles, stream);
}

template <class T>
int run(Attention a, int max_len, int64_t partial_bytes, int sms, cudaStream_t stream) {
  // 16 rows where a sequence has no more on average (single tokens), 64 where it does: a step
  // costs the same whether its rows are in use or not
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  const int size = rows <= 16ll * a.batch ? 16 : 64;
  const int tiles = pg::tile_bound(a, size);
  // few rows read the keys at the memory's speed at best, and eight parts a block that an SM holds
  // even out ragged lengths: 32 sequences of up to 8000 keys with f32 heads of 256 take 1540 us so,
  // 1665 with four and 2470 in one part
  a.parts = pg::choose_parts(a, tiles, size, a.dim, kKeys, max_len, (size == 16 ? 16 : 2) * sms,
                             partial_bytes);
  return size == 16 ? launch_dim<T, 16>(a, tiles, stream) : launch_dim<T, 64>(a, tiles, stream);
}

int check(const pg_attention_args *p, int size) {
  const char *what = "pg_attention";
  if (p->batch < 0 || p->queries < 0 || p->heads < 1 || p->group < 1 || p->dim < 1 ||
      p->page_size < 1 || p->pages < 1 || p->width < 1 || p->slot_rows < (p->batch > 0))
    return pg::argument_fail("%s: batch %d, queries %d, heads %d, group %d, dim %d, page_size %d, "
                             "pages %d, width %d, slot_rows %d: out of range", what, p->batch,
                             p->queries, p->heads, p->group, p->dim, p->page_size, p->pages,
                             p->width, p->slot_rows);
  if (p->dim > PG_ATTENTION_DIM || p->dim * size % 16)
    return pg::argument_fail("%s: head size %d of %d-byte elements: want a multiple of 16 bytes "
                             "and at most %d", what, p->dim, size, PG_ATTENTION_DIM);
  if (static_cast<int64_t>(p->page_size) * p->width > INT32_MAX / 2 || p->heads > 65535 ||
      static_cast<int64_t>(p->queries) * p->group > INT32_MAX / 2)
    return pg::argument_fail("%s: %d pages of %d keys, %d kv heads or %d queries of %d heads: too "
                             "many", what, p->width, p->page_size, p->heads, p->queries, p->group);
  if (p->window < 0 || p->sinks < 0 || p->max_len < 0 || !(p->scale == p->scale))
    return pg::argument_fail("%s: window %d, sinks %d, max_len %d, scale %g", what, p->window,
                             p->sinks, p->max_len, p->scale);
  if (!p->starts && p->queries != p->batch)
    return pg::argument_fail("%s: %d queries for %d sequences and no starts", what, p->queries,
                             p->batch);
  if (!p->batch || !p->queries) return PG_OK;
  if (!p->q || !p->k || !p->v || !p->out || !p->table || !p->lens || !p->workspace)
    return pg::argument_fail("%s: null pointer", what);
  if ((p->q | p->k | p->v |
       static_cast<uint64_t>(p->q_token | p->q_head | p->k_page | p->k_head | p->v_page |
                             p->v_head)) & 15)
    return pg::argument_fail("%s: q, k, v and their strides must be multiples of 16 bytes", what);
  if ((p->out | static_cast<uint64_t>(p->out_token | p->out_head)) & 15)
    return pg::argument_fail("%s: out and its strides must be multiples of 16 bytes", what);
  if ((p->starts | p->slots | p->table | p->lens) & 3 || p->workspace & 255)
    return pg::argument_fail("%s: starts, slots, table and lens must be 4-byte aligned and the "
                             "workspace 256-byte aligned", what);
  if (p->workspace_bytes < PG_ATTENTION_WORKSPACE)
    return pg::argument_fail("%s: a workspace of %lld bytes, want %d", what,
                             static_cast<long long>(p->workspace_bytes), PG_ATTENTION_WORKSPACE);
  return PG_OK;
}

}  // namespace

extern "C" int pg_attention(const pg_attention_args *p, uint64_t stream) {
  if (!p) return pg::argument_fail("pg_attention: null arguments");
  const int dtype = p->dtype;
  if (dtype != PG_DT_F32 && dtype != PG_DT_BF16 && dtype != PG_DT_F16)
    return pg::argument_fail("pg_attention: dtype %d, want f32, bf16 or f16", dtype);
  int rc = check(p, dtype == PG_DT_F32 ? 4 : 2);
  if (rc || !p->batch || !p->queries) return rc;
  int sms;
  if ((rc = pg::sm_count(&sms))) return rc;
  const auto ptr = [](uint64_t x) { return reinterpret_cast<char *>(static_cast<uintptr_t>(x)); };
  Attention a = {};
  a.q = ptr(p->q), a.k = ptr(p->k), a.v = ptr(p->v), a.out = ptr(p->out);
  a.starts = reinterpret_cast<int *>(ptr(p->starts));
  a.slots = reinterpret_cast<int *>(ptr(p->slots));
  a.table = reinterpret_cast<int *>(ptr(p->table));
  a.lens = reinterpret_cast<int *>(ptr(p->lens));
  a.status = reinterpret_cast<unsigned *>(ptr(p->workspace));
  a.arrived = a.status + 64;
  a.partial = reinterpret_cast<float *>(a.arrived + pg::kCounters);
  a.q_token = p->q_token, a.q_head = p->q_head;
  a.out_token = p->out_token, a.out_head = p->out_head;
  a.k_page = p->k_page, a.k_head = p->k_head, a.v_page = p->v_page, a.v_head = p->v_head;
  a.table_row = p->table_stride;
  a.batch = p->batch, a.queries = p->queries, a.heads = p->heads, a.group = p->group;
  a.dim = p->dim, a.page_size = p->page_size, a.pages = p->pages, a.width = p->width;
  a.slot_rows = p->slot_rows, a.sinks = p->sinks;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  const int64_t most = static_cast<int64_t>(p->width) * p->page_size;
  // A window that the longest sequence fits in hides nothing. Positions less a smaller one stay in 32
  // bits, those of queries before a sequence's start too.
  a.window = p->window >= most ? 0 : p->window;
  const int max_len = static_cast<int>(p->max_len && p->max_len < most ? p->max_len : most);
  const int64_t partial_bytes = p->workspace_bytes - 256 - pg::kCounters * 4ll;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(stream));
  if (a.dim <= 128) {
    if (pg::decode_takes(a, dtype == PG_DT_F32, static_cast<int>(most), max_len))
      return pg::decode(a, dtype, sms, s);
    // which masks a score before it is scaled, and 0 times a masked one's -inf is NaN
    if (a.starts && dtype != PG_DT_F32 && a.scale_log2 != 0.0f)
      return pg::prompt_16bit(a, dtype == PG_DT_BF16, max_len, partial_bytes, sms, s);
  }
  if (dtype == PG_DT_F32) return run<float>(a, max_len, partial_bytes, sms, s);
  if (dtype == PG_DT_BF16) return run<__nv_bfloat16>(a, max_len, partial_bytes, sms, s);
  return run<__half>(a, max_len, partial_bytes, sms, s);
}

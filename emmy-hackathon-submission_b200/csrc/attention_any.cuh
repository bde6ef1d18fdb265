// Attention over a paged cache in 32-bit arithmetic, for every type and head size
// (pg_attention in include/ptxgen_b200.h).
#pragma once

#include "attention.cuh"

namespace {

using pg::Attention;
using pg::Blocks;
using pg::Sight;
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

template <> struct Load<int8_t> {  // times the row's scale
  static constexpr int n = 16;
  __device__ static void get(const uint4 &v, float *x, float scale) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      x[i] = scale * static_cast<float>(static_cast<int8_t>(w[i / 4] >> 8 * (i % 4)));
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
  static constexpr int bytes = floats * 4 + kKeys * 24;
};

// A block takes ROWS rows (queries times heads of one kv head's group) and a part of the blocks
// of 64 keys they see. 16 threads share a row group: each has R rows and J of the keys of a step,
// then R rows and DIM / 16 of the columns of o. The products run two at a time in FMA (f32x2) from
// shared memory, whose reads and the barriers of a step bound it: 1024 f32 queries of 16 heads on
// up to 4096 keys take 1.14 ms, 26 TFLOP/s. The 16-bit types have kernels on the tensor cores at
// head sizes of up to 128.
// A value in a masked place may be anything: its weight is 0 and, where a step holds a value
// that is not finite, the masked places are skipped one by one.
// K: the keys' and values' type, T or int8_t
template <class T, class K, int ROWS, int DIM, bool TREE>
__global__ void __launch_bounds__(kThreads) attention_kernel(Attention a) {
  using L = Layout<ROWS, DIM>;
  constexpr bool k8 = sizeof(K) == 1;
  constexpr int R = ROWS / 16, C = DIM / 64, J = kKeys / 16;
  extern __shared__ float4 smem4[];
  float *smem = reinterpret_cast<float *>(smem4);
  float *qs = smem + L::q, *ks = smem + L::k, *vs = smem + L::v, *ps = smem + L::p;
  int64_t *key_at = reinterpret_cast<int64_t *>(smem + L::floats);  // k's and v's byte offsets
  float *scale_at = reinterpret_cast<float *>(key_at + 2 * kKeys);  // k's and v's scales
  __shared__ unsigned last;
  pg::wait_for_earlier_kernels();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, row0 = ty * R;
  const int head = blockIdx.y, part = blockIdx.z;
  const Tile t = pg::find_tile(a, gridDim.x - 1 - blockIdx.x);
  if (!t.rows) return;
  const int first_pos = t.length - t.count;
  // a tree's: they see what is before it, and some may see all of it
  const int lo = TREE ? first_pos - 1 : first_pos + t.row / a.group;
  const int hi = TREE ? t.length - 1 : first_pos + (t.row + t.rows - 1) / a.group;
  const Blocks blocks = pg::blocks_of(a, lo, hi, kKeys);
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks.count) * part / a.parts);
  const int b1 = static_cast<int>(static_cast<int64_t>(blocks.count) * (part + 1) / a.parts);
  const int pieces = a.dim / Load<T>::n, kv_pieces = a.dim / Load<K>::n;

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
  Sight<TREE> sight[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
    sight[r] = row0 + r < t.rows ? Sight<TREE>::of(a, first_pos, t.count, t.query,
                                                  (t.row + row0 + r) / a.group)
                                 : Sight<TREE>{-1, 0, 0};
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
        const int row = key % a.page_size;
        const int64_t in_page = static_cast<int64_t>(row) * a.dim * sizeof(K);
        if (page >= 0) {
          ka = page * a.k_page + head * a.k_head + in_page;
          va = page * a.v_page + head * a.v_head + in_page;
          if (k8) {
            scale_at[tid] = *reinterpret_cast<const float *>(
                a.k_scale + page * a.ks_page + head * a.ks_head + row * 4ll);
            scale_at[kKeys + tid] = *reinterpret_cast<const float *>(
                a.v_scale + page * a.vs_page + head * a.vs_head + row * 4ll);
          }
        }
      }
      key_at[tid] = ka;
      key_at[kKeys + tid] = va;
    }
    __syncthreads();
    bool odd = false;
    // loads in batches, so that they are in flight together
    constexpr int kAll = kKeys * (DIM / Load<K>::n), kBatch = 4;
    for (int i0 = tid; i0 < kAll; i0 += kBatch * kThreads) {
      uint4 kk[kBatch], vv[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kThreads, r = i / (DIM / Load<K>::n), c = i % (DIM / Load<K>::n);
        kk[u] = vv[u] = make_uint4(0, 0, 0, 0);
        if (i < kAll && key_at[r] >= 0 && c < kv_pieces) {
          kk[u] = pg::load16(a.k + key_at[r] + c * 16);
          vv[u] = pg::load16(a.v + key_at[kKeys + r] + c * 16);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kThreads, r = i / (DIM / Load<K>::n), c = i % (DIM / Load<K>::n);
        if (i >= kAll) break;
        float x[Load<K>::n], y[Load<K>::n];
        if constexpr (k8) {
          const bool real = key_at[r] >= 0;
          Load<K>::get(kk[u], x, real ? scale_at[r] : 0.0f);
          Load<K>::get(vv[u], y, real ? scale_at[kKeys + r] : 0.0f);
        } else {
          Load<K>::get(kk[u], x);
          Load<K>::get(vv[u], y);
        }
        float *const k_to = ks + r * L::stride + c * Load<K>::n;
        float *const v_to = vs + r * L::stride + c * Load<K>::n;
#pragma unroll
        for (int j = 0; j < Load<K>::n; j += 4) {
          *reinterpret_cast<float4 *>(k_to + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          *reinterpret_cast<float4 *>(v_to + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
        }
#pragma unroll
        for (int j = 0; j < Load<K>::n; ++j) odd |= !(fabsf(y[j]) < INFINITY);
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
        const bool seen = sight[r].sees(a, key) && key_at[tx + 16 * j] >= 0;
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
          if (!sight[r].sees(a, key0 + j)) continue;
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
          store(sight[r].none() ? 0.0f : o[r][4 * c + e] * inv, to + 64 * c + 4 * tx + e);
  }
}

template <class T, class K, int ROWS, int DIM, bool TREE>
int launch_tiles(Attention a, int tiles, cudaStream_t stream) {
  a.rows_per_tile = ROWS;
  return pg::launch<attention_kernel<T, K, ROWS, DIM, TREE>>(
      "attention_kernel", dim3(tiles, a.heads, a.parts), kThreads, Layout<ROWS, DIM>::bytes, stream,
      a);
}

// LEAST: the smallest size of head that has a kernel of its own
template <class T, class K, int ROWS, int LEAST, bool TREE>
int launch_dim(const Attention &a, int tiles, cudaStream_t stream) {
  if constexpr (LEAST <= 64)
    if (a.dim <= 64) return launch_tiles<T, K, ROWS, 64, TREE>(a, tiles, stream);
  if constexpr (LEAST <= 128)
    if (a.dim <= 128) return launch_tiles<T, K, ROWS, 128, TREE>(a, tiles, stream);
  return launch_tiles<T, K, ROWS, 256, TREE>(a, tiles, stream);
}

template <class T, class K, int LEAST, bool TREE>
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
  return size == 16 ? launch_dim<T, K, 16, LEAST, TREE>(a, tiles, stream)
                    : launch_dim<T, K, 64, LEAST, TREE>(a, tiles, stream);
}

}  // namespace

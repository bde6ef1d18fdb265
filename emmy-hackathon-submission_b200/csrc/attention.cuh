// What the attention kernels share: the arguments, which keys a query sees, the tiles of a
// ragged batch and the joining of partial results.
//
// Query i of a sequence of `len` tokens whose last `count` tokens are the queries stands at
// position pos = len - count + i, and sees key j when j <= pos and (window == 0 or j > pos -
// window or j < sinks). With scores s_j = scale q . k_j over the keys it sees,
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j,
// held as a running m, l (the sum) and o in 32 bits while the keys pass, o and l scaled by
// exp(m - m') when m grows to m'. Two disjoint sets of keys join the same way:
//   m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise.
// A query that sees no key (l = 0) gives zeros. The kernels work in powers of two: the scale is
// multiplied by log2 e and exp becomes exp2.
#pragma once

#include "common.cuh"

#include <cmath>

namespace pg {

struct Attention {
  const char *q, *k, *v;
  char *out;
  const int *starts, *slots, *table, *lens;
  float *partial;       // per (tile, kv head, part): rows * (dim + 2) floats
  unsigned *arrived;    // per (tile, kv head): parts that have finished; 0 between calls
  unsigned *status;
  int64_t q_token, q_head, out_token, out_head;       // bytes
  int64_t k_page, k_head, v_page, v_head, table_row;  // bytes, bytes, bytes, bytes, words
  int batch, queries, heads, group, dim, page_size, pages, width, slot_rows;
  int window, sinks, parts, rows_per_tile;
  float scale_log2;
};

// The keys that the queries of a tile see among them, in blocks of `size` keys: the blocks of
// the sinks, then those of the window, each block once.
struct Blocks {
  int sink, first, count;  // blocks [0, sink) and [first, first + count - sink)
  __device__ int key_block(int i) const { return i < sink ? i : first + i - sink; }
};

__device__ __forceinline__ Blocks blocks_of(const Attention &a, int lo_pos, int hi_pos, int size) {
  // queries at positions lo_pos..hi_pos; none where hi_pos < 0
  Blocks b{0, 0, 0};
  if (hi_pos < 0) return b;
  const int last = hi_pos / size;
  const int low = a.window ? max(0, max(lo_pos, 0) - a.window + 1) : 0;
  b.first = low / size;
  if (a.window && a.sinks > 0)
    b.sink = min(b.first, (min(a.sinks, hi_pos + 1) + size - 1) / size);
  b.count = b.sink + last - b.first + 1;
  return b;
}

__device__ __forceinline__ bool sees(const Attention &a, int pos, int key) {
  return key <= pos && (!a.window || key > pos - a.window || key < a.sinks);
}

// A tile: rows [row, row + rows) of the (query, head in group) rows of one sequence.
struct Tile {
  int sequence, row, rows, query, count, length;  // query: the sequence's first query
  const int *pages;
};

// The tile-th tile of the batch, or one with no rows past the last. A warp calls it together.
__device__ __forceinline__ Tile find_tile(const Attention &a, int tile) {
  const int lane = threadIdx.x & 31;
  Tile t{0, 0, 0, 0, 0, 0, nullptr};
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    int start = 0, count = 0;
    if (b < a.batch) {
      start = a.starts ? a.starts[b] : b;
      count = a.starts ? max(0, a.starts[b + 1] - start) : 1;
      if (start < 0 || count > a.queries - start) {
        atomicOr(a.status, PG_CACHE_TOO_LONG);
        count = 0;
      }
    }
    const int tiles = static_cast<int>(
        (static_cast<int64_t>(count) * a.group + a.rows_per_tile - 1) / a.rows_per_tile);
    int upto = tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    const int mine = tile - base - (upto - tiles);
    const unsigned hit = __ballot_sync(0xffffffffu, mine >= 0 && mine < tiles);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int slot_in = __shfl_sync(0xffffffffu, b, src);
      t.sequence = slot_in;
      t.row = __shfl_sync(0xffffffffu, mine, src) * a.rows_per_tile;
      t.query = __shfl_sync(0xffffffffu, start, src);
      t.count = __shfl_sync(0xffffffffu, count, src);
      t.rows = min(a.rows_per_tile, t.count * a.group - t.row);
      const int slot = a.slots ? a.slots[slot_in] : slot_in;
      if (slot < 0 || slot >= a.slot_rows) {
        if (lane == 0) atomicOr(a.status, PG_CACHE_BAD_SLOT);
        t.length = 0;
        return t;
      }
      t.pages = a.table + slot * a.table_row;
      t.length = a.lens[slot];
      if (t.length < 0 || t.length > static_cast<int64_t>(a.width) * a.page_size) {
        if (lane == 0) atomicOr(a.status, PG_CACHE_TOO_LONG);
        t.length = t.length < 0 ? 0 : a.width * a.page_size;
      }
      return t;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return t;
}

// The page of a key, or -1 (with a status bit) where the table names none that exists.
__device__ __forceinline__ int page_of(const Attention &a, const Tile &t, int key) {
  const int page = t.pages[key / a.page_size];
  if (page >= 0 && page < a.pages) return page;
  atomicOr(a.status, PG_CACHE_BAD_PAGE);
  return -1;
}

// Zeroes the 16-bit numbers at `at` that are not finite (their exponent's bits are EXPONENT);
// whether there were any.
template <uint32_t EXPONENT>
__device__ __forceinline__ bool clean(uint4 *at) {
  const uint4 x = *at;
  uint32_t u[4] = {x.x, x.y, x.z, x.w};
  bool any = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((u[k] & EXPONENT) == EXPONENT) u[k] &= 0xffff0000u, any = true;
    if ((u[k] >> 16 & EXPONENT) == EXPONENT) u[k] &= 0x0000ffffu, any = true;
  }
  if (any) *at = make_uint4(u[0], u[1], u[2], u[3]);
  return any;
}

// ... the f32 numbers.
__device__ __forceinline__ bool clean32(uint4 *at) {
  const uint4 x = *at;
  uint32_t u[4] = {x.x, x.y, x.z, x.w};
  bool any = false;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if ((u[k] & 0x7f800000u) == 0x7f800000u) u[k] = 0, any = true;
  if (any) *at = make_uint4(u[0], u[1], u[2], u[3]);
  return any;
}

// Adds a visible value that is not finite to its column's sum. Its products with the weights as they
// were rounded may be NaN (0 times infinity), so the first such value takes the place of a sum that is
// not finite, and only the others add to it.
__device__ __forceinline__ void add_odd(float value, float &sum, bool first) {
  sum = first && !(fabsf(sum) < INFINITY) ? value : sum + value;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp2(a - b) for running maxima: 0 for a = -inf, whatever b
__device__ __forceinline__ float factor(float a, float b) {
  return a == -INFINITY ? 0.0f : exp2_fast(a - b);
}

// Kernels for head sizes of up to 128: few rows a sequence (attention_decode.cu), and many in the
// 16-bit types (attention_prompt.cu).
bool decode_takes(const Attention &a, bool f32, int most, int max_len);
int decode(const Attention &a, int dtype, int sms, cudaStream_t stream);
int prompt_16bit(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                 cudaStream_t stream);

// --- host side -------------------------------------------------------------------------------

constexpr int kCounters = 4096;  // (tile, kv head) pairs that may be cut in parts

// The most tiles a batch can have: whole ones and one part-full one a sequence.
inline int tile_bound(const Attention &a, int rows_per_tile) {
  if (!a.starts) return a.batch * ((a.group + rows_per_tile - 1) / rows_per_tile);
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  return static_cast<int>(rows / rows_per_tile) + (a.batch < a.queries ? a.batch : a.queries);
}

// Parts that each tile's keys are cut in: enough to give `blocks` blocks work, each part at
// least four steps of `keys` keys at the longest length, no more than the workspace holds.
inline int choose_parts(const Attention &a, int tiles, int rows_per_tile, int columns, int keys,
                        int max_len, int blocks, int64_t partial_bytes) {
  const int64_t pairs = static_cast<int64_t>(tiles) * a.heads;
  if (pairs * 2 > blocks || pairs > kCounters) return 1;
  int64_t seen = max_len;
  if (a.window) {
    const int64_t near = static_cast<int64_t>(a.window) + a.sinks + 2 * keys;
    seen = near < seen ? near : seen;
  }
  int64_t parts = blocks / pairs;
  const int64_t steps = (seen + 4ll * keys - 1) / (4ll * keys);
  parts = steps < parts ? steps : parts;
  // the last part to finish reads all: no more than about twice the root of the steps
  const int64_t most = 2 * static_cast<int64_t>(std::sqrt(static_cast<double>(seen / keys + 1)));
  parts = most < parts ? most : parts;
  const int64_t each = pairs * rows_per_tile * (columns + 2) * 4ll;
  parts = partial_bytes / each < parts ? partial_bytes / each : parts;
  return static_cast<int>(parts < 1 ? 1 : parts);
}

}  // namespace pg

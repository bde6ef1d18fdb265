// The paged key-value cache's page operations (pg_cache_* in include/ptxgen_b200.h).
//
// A sequence (a slot) holds lens[slot] tokens in the pages its table row names; refs[p] counts
// the rows that name page p, and a page is free when its count is 0. An operation that takes
// pages takes the lowest free ones, in the order of its slots, so results never depend on
// timing. Everything happens on the device in stream order: no operation waits for the host.
//
// extend and fork are planned by one block (of cache_extend, cache_fork_plan): it checks every
// request before it changes anything, so a request that cannot be met (no pages, a bad or
// repeated slot) sets a bit of the status word and leaves the cache as it was. Its write is queued
// all the same, and would go to the slots' older tokens: so extend marks each of its slots as
// refused or not, and write leaves out the marked ones. The bulk of the
// work (rows of keys and values, table rows, counts) is done by a second kernel over the whole
// GPU that the plan's scratch array drives.
#include "common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr int kPlan = 1024;   // threads of a planning block
// Blocks that look through the parents' table rows before a fork is planned (250 children of parents
// of up to 700 tokens in 24 layers: 120 us with 8, 125 with 1; of up to 30000 in one layer: 39, 49).
constexpr int kLook = 8;
constexpr int kCopy = 256;    // threads of a copying block
// Copying blocks an SM gets at most, eight times what it holds: a block that ends makes room for
// the next, which spreads the copies better than blocks that stay and loop in step. With 8, 64 and
// 512: half the pages of 96 sequences of up to 900 tokens moved in 16 layers 210, 193, 207 us; 250
// children of 24 layers forked 127, 120, 122; 48 sequences of up to 4096 tokens written 143, 131,
// 130 (with their extend and free).
constexpr int kCopyPerSm = 64;
constexpr int kUnroll = 4;    // 16-byte loads a copying thread has in flight

// Scratch words (int32): [0] whether the plan went through, [1] its number of pages, then
// three arrays of `pages` words each.
constexpr int kHeader = 4;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Exclusive prefix sum of v over the block's threads; *total gets the sum. All threads call it.
__device__ int block_scan(int v, int *slots, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += up;
  }
  if (lane == 31) slots[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = slots[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += up;
    }
    slots[lane] = w;
  }
  __syncthreads();
  const int base = warp ? slots[warp - 1] : 0;
  *total = slots[kPlan / 32 - 1];
  __syncthreads();
  return base + inc - v;
}

// Writes the ids of the lowest `need` pages p in [first, pages) whose count is zero (or, with
// `live`, is not) to out, ascending; returns how many there were. All threads call it.
__device__ int find_pages(const int *refs, int first, int pages, int need, bool live, int *out,
                          int *slots) {
  int found = 0;
  for (int base = first; base < pages && found < need; base += 4 * kPlan) {
    const int p = base + 4 * static_cast<int>(threadIdx.x);
    int mask = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (p + j < pages && (refs[p + j] > 0) == live) mask |= 1 << j;
    int total;
    int at = found + block_scan(__popc(mask), slots, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (mask >> j & 1) {
        if (at < need) out[at] = p + j;
        ++at;
      }
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

__device__ void set_status(const pg_cache &c, unsigned bits) {
  atomicOr(reinterpret_cast<unsigned *>(c.status), bits);
}

__device__ __forceinline__ int *refs_of(const pg_cache &c) {
  return reinterpret_cast<int *>(c.refs);
}
__device__ __forceinline__ int *lens_of(const pg_cache &c) {
  return reinterpret_cast<int *>(c.lens);
}
__device__ __forceinline__ int *refused_of(const pg_cache &c) {
  return reinterpret_cast<int *>(c.refused);
}
__device__ __forceinline__ int *row_of(const pg_cache &c, int slot) {
  return reinterpret_cast<int *>(c.table) + slot * c.table_stride;
}

// Claims a slot for one operation by storing the complement of its length, so that a second
// claim of the same slot sees a negative number. Returns the length, or -1 on a second claim.
__device__ int claim(int *len) {
  const int old = atomicMin(len, -1);
  if (old < 0) return -1;
  atomicExch(len, ~old);
  return old;
}

// --- extend: room for the new tokens of each slot ----------------------------------------------
// One block: the pages it hands out are found by a scan of the counts that stops at the last one
// needed, and 4096 counts are 16 KB, so the latency of a few dependent loads bounds it: 5 us for a
// few slots, 13 us for 48 slots and 6000 pages. 64 slots that take a page each: 5 us where the free
// pages begin at 2600, 28 at 98600, since every scan begins at page 0.

__global__ void __launch_bounds__(kPlan) cache_extend(pg_cache c, const int *slots_in,
                                                      const int *starts, int n) {
  __shared__ int warp_slots[32];
  __shared__ unsigned bad;
  pg::wait_for_earlier_kernels();
  if (threadIdx.x == 0) bad = 0;
  int *lens = lens_of(c), *refs = refs_of(c);
  int *scratch = reinterpret_cast<int *>(c.scratch);
  int *fresh = scratch + kHeader, *offset = fresh + c.pages, *length = offset + c.slots + 1;
  __syncthreads();
  // every request's old length (-1: not claimed here) and its first page among the fresh ones
  int need = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    int want = 0, len = -1;
    if (i < n) {
      const int slot = slots_in[i], count = starts[i + 1] - starts[i];
      if (slot < 0 || slot >= c.slots) {
        atomicOr(&bad, PG_CACHE_BAD_SLOT);
      } else if ((len = claim(lens + slot)) < 0) {
        atomicOr(&bad, PG_CACHE_BAD_SLOT);
      } else if (count < 0 || count > c.width * static_cast<int64_t>(c.page_size) - len) {
        atomicOr(&bad, PG_CACHE_TOO_LONG);
      } else {
        want = ceil_div(len + count, c.page_size) - ceil_div(len, c.page_size);
      }
      length[i] = len;
    }
    int total;
    const int at = need + block_scan(want, warp_slots, &total);
    if (i < n) offset[i] = at;
    need += total;
  }
  if (need > c.pages) need = c.pages + 1;  // more than there are: the search below falls short
  if (threadIdx.x == 0) offset[n] = need;
  __syncthreads();
  if (!bad) {
    const int got = find_pages(refs, 0, c.pages, min(need, c.pages), false, fresh, warp_slots);
    if (got < need && threadIdx.x == 0) bad = PG_CACHE_NO_PAGES;
    __syncthreads();
  }
  if (bad) {
    for (int i = threadIdx.x; i < n; i += kPlan) {
      const int slot = slots_in[i];
      if (length[i] >= 0) lens[slot] = length[i];
      if (slot >= 0 && slot < c.slots) refused_of(c)[slot] = 1;
    }
    if (threadIdx.x == 0) set_status(c, bad);
    return;
  }
  for (int r = threadIdx.x; r < need; r += kPlan) {
    int lo = 0, hi = n;  // the last request whose first page is at or before r and has any
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offset[mid] <= r) lo = mid; else hi = mid;
    }
    row_of(c, slots_in[lo])[ceil_div(length[lo], c.page_size) + r - offset[lo]] = fresh[r];
    refs[fresh[r]] = 1;
  }
  for (int i = threadIdx.x; i < n; i += kPlan) {
    lens[slots_in[i]] = length[i] + starts[i + 1] - starts[i];
    refused_of(c)[slots_in[i]] = 0;
  }
}

// --- write: new rows of one layer into the slots' pages ----------------------------------------
// A warp takes one token: its slot and page are the same for all lanes, and its heads' rows of
// keys and values are 16-byte pieces that the lanes load together before they store any. HBM
// bounds it, each piece read and written once: 5.9 TB/s with 48 sequences of up to 4096 tokens of
// 8 heads of 128 in bf16, their extend counted in.

__device__ __forceinline__ int find_sequence(const int *starts, int n, int token) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= token) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kCopy) cache_write(pg_cache c, int layer, const int *slots_in,
                                                     const int *starts, int n, int tokens,
                                                     pg_rows k, pg_rows v) {
  pg::wait_for_earlier_kernels();
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (kCopy / 32);
  const int pieces = c.row_bytes / 16, all = c.heads * pieces;
  if (blockIdx.x == 0 && threadIdx.x == 0 && (starts[0] < 0 || starts[n] > tokens))
    set_status(c, PG_CACHE_TOO_LONG);  // tokens that have no rows
  for (int t = (blockIdx.x * kCopy + threadIdx.x) >> 5; t < tokens; t += warps) {
    if (t < starts[0] || t >= starts[n]) continue;
    const int i = find_sequence(starts, n, t);
    const int slot = slots_in[i];
    if (slot < 0 || slot >= c.slots) {
      if (lane == 0) set_status(c, PG_CACHE_BAD_SLOT);
      continue;
    }
    if (refused_of(c)[slot]) {
      if (lane == 0) set_status(c, PG_CACHE_REFUSED);
      continue;
    }
    const int pos = lens_of(c)[slot] - (starts[i + 1] - t);
    const int64_t entry = pos / c.page_size;
    const int page = pos >= 0 && entry < c.width ? row_of(c, slot)[entry] : -1;
    if (page < 0 || page >= c.pages) {
      if (lane == 0) set_status(c, PG_CACHE_BAD_PAGE);
      continue;
    }
    const int64_t to = layer * c.layer_stride + page * c.page_stride +
                       static_cast<int64_t>(pos % c.page_size) * c.row_bytes;
    for (int base = lane; base < all; base += 32 * kUnroll) {
      uint4 kk[kUnroll], vv[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = base + 32 * u, head = j / pieces, piece = j - head * pieces;
        if (j < all) {
          kk[u] = pg::load16(reinterpret_cast<const char *>(k.data) + t * k.token_stride +
                             head * k.head_stride + piece * 16);
          vv[u] = pg::load16(reinterpret_cast<const char *>(v.data) + t * v.token_stride +
                             head * v.head_stride + piece * 16);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = base + 32 * u, head = j / pieces, piece = j - head * pieces;
        if (j < all) {
          const int64_t at = to + head * c.head_stride + piece * 16;
          *reinterpret_cast<uint4 *>(c.k + at) = kk[u];
          *reinterpret_cast<uint4 *>(c.v + at) = vv[u];
        }
      }
    }
  }
}

// --- free: a slot lets go of its pages ---------------------------------------------------------

__global__ void __launch_bounds__(kCopy) cache_free(pg_cache c, const int *slots_in, int n) {
  __shared__ int held;
  pg::wait_for_earlier_kernels();
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int slot = slots_in[i];
    if (slot < 0 || slot >= c.slots) {
      if (threadIdx.x == 0) set_status(c, PG_CACHE_BAD_SLOT);
      continue;
    }
    // the exchange gives a slot listed twice to one block only
    if (threadIdx.x == 0) {
      held = atomicExch(lens_of(c) + slot, 0);
      refused_of(c)[slot] = 0;
    }
    __syncthreads();
    const int count = min(ceil_div(held, c.page_size), c.width);
    int *row = row_of(c, slot);
    for (int j = threadIdx.x; j < count; j += kCopy) {
      const int page = row[j];
      row[j] = -1;
      if (page < 0 || page >= c.pages || atomicSub(refs_of(c) + page, 1) <= 0)
        set_status(c, PG_CACHE_BAD_PAGE);
    }
    __syncthreads();
  }
}

// --- copying rows of pages ---------------------------------------------------------------------
// Copies the first `rows` rows of every head of page `from` to page `to` in one layer's keys or
// values. HBM bounds it: each piece is read and written once, 16 bytes a lane, and 6.2 TB/s to 6.8
// are reached by the forks and moves named above.

// A cache in 8 bits has its rows' scales copied, too.

__device__ void copy_rows(const pg_cache &c, const pg_cache_scales &s, bool values, int layer,
                          int from, int to, int rows) {
  char *const base = reinterpret_cast<char *>(values ? c.v : c.k);
  if (const uint64_t scales = values ? s.v : s.k) {
    char *const at = reinterpret_cast<char *>(scales) + layer * s.layer_stride;
    for (int i = threadIdx.x; i < c.heads * rows; i += kCopy) {
      const int head = i / rows;
      const int64_t in = head * s.head_stride + (i - head * rows) * 4ll;
      *reinterpret_cast<float *>(at + to * s.page_stride + in) =
          *reinterpret_cast<const float *>(at + from * s.page_stride + in);
    }
  }
  const int per_head = rows * (c.row_bytes / 16), all = c.heads * per_head;
  const char *src = base + layer * c.layer_stride + from * c.page_stride;
  char *dst = base + layer * c.layer_stride + to * c.page_stride;
  for (int at = threadIdx.x; at < all; at += kCopy * kUnroll) {
    uint4 x[kUnroll];
    int64_t off[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = at + kCopy * u, head = j / per_head;
      off[u] = head * c.head_stride + static_cast<int64_t>(j - head * per_head) * 16;
      if (j < all) x[u] = pg::load16(src + off[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (at + kCopy * u < all) *reinterpret_cast<uint4 *>(dst + off[u]) = x[u];
  }
}

// Pair i's pages, whole, in every layer's keys and values.
__global__ void __launch_bounds__(kCopy) cache_copy(pg_cache c, pg_cache_scales s,
                                                    const int *from, const int *to, int n) {
  pg::wait_for_earlier_kernels();
  const int64_t tasks = static_cast<int64_t>(n) * c.layers * 2;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int i = static_cast<int>(task / (2 * c.layers));
    const int plane = static_cast<int>(task - static_cast<int64_t>(i) * 2 * c.layers);
    const int a = from[i], b = to[i];
    if (a < 0 || a >= c.pages || b < 0 || b >= c.pages) {
      if (threadIdx.x == 0) set_status(c, PG_CACHE_BAD_PAGE);
      continue;
    }
    copy_rows(c, s, plane & 1, plane >> 1, a, b, c.page_size);
  }
}

// --- fork: children that share their parents' full pages ---------------------------------------

// Whether a page id that a parent's row holds within its length is out of range; a warp takes a row.
__device__ bool bad_rows(const pg_cache &c, const int *parents, int n, int warp, int warps) {
  constexpr int kAhead = 4;  // entries a lane has in flight
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (int i = warp; i < n; i += warps) {
    const int parent = parents[i];
    if (parent < 0 || parent >= c.slots) continue;
    const int *row = row_of(c, parent);
    const int count = min(ceil_div(lens_of(c)[parent], c.page_size), c.width);
    for (int j = lane; j < count; j += 32 * kAhead) {
      int page[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) page[u] = j + 32 * u < count ? row[j + 32 * u] : 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) bad |= page[u] < 0 || page[u] >= c.pages;
    }
  }
  return bad;
}

// The cluster's blocks look through the rows, then the first one plans by itself.
__global__ void __cluster_dims__(kLook, 1, 1) __launch_bounds__(kPlan)
    cache_fork_plan(pg_cache c, const int *parents, const int *children, int n) {
  __shared__ int warp_slots[32];
  __shared__ unsigned bad;
  pg::wait_for_earlier_kernels();
  cg::cluster_group cluster = cg::this_cluster();
  if (threadIdx.x == 0) bad = 0;
  cluster.sync();
  const int rank = cluster.block_rank();
  if (bad_rows(c, parents, n, (rank * kPlan + threadIdx.x) >> 5, kLook * kPlan / 32))
    atomicOr(cluster.map_shared_rank(&bad, 0), PG_CACHE_BAD_PAGE);
  cluster.sync();
  if (rank) return;
  int *lens = lens_of(c), *refs = refs_of(c);
  int *scratch = reinterpret_cast<int *>(c.scratch);
  int *fresh = scratch + kHeader, *offset = fresh + c.pages, *claimed = offset + c.slots + 1;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int child = children[i];
    claimed[i] = -1;
    if (child < 0 || child >= c.slots) {
      atomicOr(&bad, PG_CACHE_BAD_SLOT);
      continue;
    }
    claimed[i] = claim(lens + child);
    if (claimed[i] != 0) atomicOr(&bad, PG_CACHE_BAD_SLOT);  // taken, or listed twice
  }
  __syncthreads();
  int need = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    int want = 0;
    if (i < n) {
      const int parent = parents[i];
      const int len = parent >= 0 && parent < c.slots ? lens[parent] : -1;
      // a parent that is a child of this call is claimed: its length reads negative
      if (len < 0 || ceil_div(len, c.page_size) > c.width) atomicOr(&bad, PG_CACHE_BAD_SLOT);
      else want = len % c.page_size != 0;
    }
    int total;
    const int at = need + block_scan(want, warp_slots, &total);
    if (i < n) offset[i] = at;
    need += total;
  }
  __syncthreads();
  if (!bad) {
    const int got = find_pages(refs, 0, c.pages, need, false, fresh, warp_slots);
    if (got < need && threadIdx.x == 0) bad = PG_CACHE_NO_PAGES;
    __syncthreads();
  }
  if (threadIdx.x == 0) scratch[0] = !bad;
  if (bad) {
    for (int i = threadIdx.x; i < n; i += kPlan)
      if (claimed[i] >= 0) lens[children[i]] = claimed[i];
    if (threadIdx.x == 0) set_status(c, bad);
    return;
  }
  for (int r = threadIdx.x; r < need; r += kPlan) refs[fresh[r]] = 1;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    lens[children[i]] = lens[parents[i]];
    refused_of(c)[children[i]] = 0;
  }
}

// Task i * (2 layers + 1) + j: child i's table row and counts (j = 0), or the rows in use of its
// open page in one layer's keys or values.
__global__ void __launch_bounds__(kCopy) cache_fork_copy(pg_cache c, pg_cache_scales s,
                                                         const int *parents, const int *children,
                                                         int n) {
  pg::wait_for_earlier_kernels();
  const int *scratch = reinterpret_cast<const int *>(c.scratch);
  if (!scratch[0]) return;
  const int *fresh = scratch + kHeader, *offset = fresh + c.pages;
  const int parts = 2 * c.layers + 1;
  const int64_t tasks = static_cast<int64_t>(n) * parts;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int i = static_cast<int>(task / parts);
    const int part = static_cast<int>(task - static_cast<int64_t>(i) * parts);
    const int len = lens_of(c)[parents[i]], full = len / c.page_size, open = len % c.page_size;
    const int *from = row_of(c, parents[i]);
    if (part) {
      if (open)
        copy_rows(c, s, !(part & 1), (part - 1) >> 1, from[full], fresh[offset[i]], open);
      continue;
    }
    int *row = row_of(c, children[i]);
    for (int j = threadIdx.x; j < full; j += kCopy) {
      row[j] = from[j];
      atomicAdd(refs_of(c) + from[j], 1);
    }
    if (open && threadIdx.x == 0) row[full] = fresh[offset[i]];
  }
}

// --- compact: the live pages move to the front -------------------------------------------------
// With L live pages, the k-th free page below L takes the k-th live page at or above L, both
// ascending: the fewest moves, and no page is both read and written.

__global__ void __launch_bounds__(kPlan) cache_compact_plan(pg_cache c) {
  __shared__ int warp_slots[32];
  pg::wait_for_earlier_kernels();
  int *refs = refs_of(c);
  int *scratch = reinterpret_cast<int *>(c.scratch);
  int *holes = scratch + kHeader, *movers = holes + c.pages, *place = movers + c.pages;
  int mine = 0;
  for (int p = threadIdx.x; p < c.pages; p += kPlan) mine += refs[p] > 0;
  int live;
  block_scan(mine, warp_slots, &live);
  const int moves = find_pages(refs, 0, live, live, false, holes, warp_slots);
  find_pages(refs, live, c.pages, moves, true, movers, warp_slots);
  for (int i = threadIdx.x; i < moves; i += kPlan) {
    place[movers[i]] = holes[i];
    refs[holes[i]] = refs[movers[i]];
    refs[movers[i]] = 0;
  }
  if (threadIdx.x == 0) {
    scratch[0] = live;
    scratch[1] = moves;
  }
}

// Tasks below `slots` rewrite one slot's table row; the others move one page in one layer's
// keys or values.
__global__ void __launch_bounds__(kCopy) cache_compact_move(pg_cache c, pg_cache_scales s) {
  pg::wait_for_earlier_kernels();
  const int *scratch = reinterpret_cast<const int *>(c.scratch);
  const int live = scratch[0], moves = scratch[1];
  const int *holes = scratch + kHeader, *movers = holes + c.pages, *place = movers + c.pages;
  if (!moves) return;
  const int64_t tasks = c.slots + static_cast<int64_t>(moves) * 2 * c.layers;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    if (task < c.slots) {
      const int slot = static_cast<int>(task);
      int *row = row_of(c, slot);
      const int count = min(ceil_div(lens_of(c)[slot], c.page_size), c.width);
      for (int j = threadIdx.x; j < count; j += kCopy) {
        const int page = row[j];
        if (page >= c.pages) set_status(c, PG_CACHE_BAD_PAGE);
        else if (page >= live) row[j] = place[page];
      }
      continue;
    }
    const int64_t move = task - c.slots;
    const int i = static_cast<int>(move / (2 * c.layers));
    const int plane = static_cast<int>(move - static_cast<int64_t>(i) * 2 * c.layers);
    copy_rows(c, s, plane & 1, plane >> 1, movers[i], holes[i], c.page_size);
  }
}

// --- rows in 8 bits ----------------------------------------------------------------------------
// A row (one token's numbers of one head) is held as q = round(x / s), halves to even, with s = max |x| /
// 127 in f32: at 16 bits of it that is 8, and an error of at most s / 2. As few lanes as have 16 numbers
// each take a row. 40 sequences of up to 4096 tokens of 8 heads of 128 in bf16 are written and read back in
// 248 us, where HBM alone takes 140: the quotients are as much work as the bytes.

// 16 numbers of T at an address as f32, and to it.
template <class T> struct Sixteen;
template <> struct Sixteen<float> {
  static constexpr int words = 4;
  __device__ static void get(const uint4 *raw, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[4 * i] = __uint_as_float(raw[i].x), x[4 * i + 1] = __uint_as_float(raw[i].y);
      x[4 * i + 2] = __uint_as_float(raw[i].z), x[4 * i + 3] = __uint_as_float(raw[i].w);
    }
  }
  __device__ static void put(const float *x, uint4 *raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      raw[i] = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]),
                          __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
  }
};
template <class T, class T2> struct Sixteen16 {
  static constexpr int words = 2;
  __device__ static void get(const uint4 *raw, float *x) {
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w,
                           raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T2 h = *reinterpret_cast<const T2 *>(&w[i]);
      x[2 * i] = __low2float(h), x[2 * i + 1] = __high2float(h);
    }
  }
};
template <> struct Sixteen<__nv_bfloat16> : Sixteen16<__nv_bfloat16, __nv_bfloat162> {
  __device__ static void put(const float *x, uint4 *raw) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    raw[0] = make_uint4(w[0], w[1], w[2], w[3]), raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
};
template <> struct Sixteen<__half> : Sixteen16<__half, __half2> {
  __device__ static void put(const float *x, uint4 *raw) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    raw[0] = make_uint4(w[0], w[1], w[2], w[3]), raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
};

// x / s for 16 numbers, rounded, halves to even. x times 1 / s is off by up to 2^-16 at 127, so what it
// rounds to, q, may be one off where the quotient is next to a half. The remainder x - q s is exact in
// f32 (a multiple of half the scale's last bit, no larger than about s / 2), and against s / 2 it tells.
// bf16 rows have exact halves often: a number and the largest are whole numbers below 256 by powers of two.
// For scales of 2^-100 and more.
__device__ __forceinline__ uint4 quantise(const float *x, float s) {
  const float inverse = 1.0f / s;
  // from where on a remainder is too large: s / 2 for an odd q, the number after it for an even one
  const uint32_t even = __float_as_uint(0.5f * s) + 1;
  constexpr float kShift = 12582912.0f;  // 1.5 * 2^23: its last bits are a whole number's
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    y[i] = fmaf(x[i], inverse, kShift);
    const float r = fmaf(kShift - y[i], s, x[i]);
    if (fabsf(r) >= __uint_as_float(even - (__float_as_uint(y[i]) & 1))) y[i] += copysignf(1.0f, r);
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __byte_perm(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]), 0x0040);
    const uint32_t b =
        __byte_perm(__float_as_uint(y[4 * i + 2]), __float_as_uint(y[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(a, b, 0x5410);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ... of any other scale, whose inverse may be no f32 number, and which may have lost bits itself: by 64-bit
// division, where the quotient of two f32 numbers is a half only if it is one.
__device__ __noinline__ uint4 quantise_small(const uint4 *raw, int words, float s) {
  uint32_t w[4] = {};
  if (s > 0.0f)
    for (int i = 0; i < 16; ++i) {
      const uint32_t bits = reinterpret_cast<const uint32_t *>(raw)[words == 4 ? i : i / 2];
      // 16-bit rows with such scales are bf16: f16 has no numbers as small
      const float x = __uint_as_float(words == 4 ? bits : i & 1 ? bits & 0xffff0000u : bits << 16);
      const double q = rint(static_cast<double>(x) / static_cast<double>(s));
      const int b = static_cast<int>(fmin(fmax(q, -127.0), 127.0)) & 255;
      w[i / 4] |= b << 8 * (i % 4);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Where a token's rows are in a layer: its place among the pages, or -1 where there is none.
struct Place {
  int page, row;
};
__device__ __forceinline__ Place place_of(const pg_cache &c, const int *slots_in, const int *starts,
                                          int n, int t, bool marks) {
  const bool first = (threadIdx.x & 31) == 0;
  const Place none{-1, 0};
  if (t < starts[0] || t >= starts[n]) return none;
  const int i = find_sequence(starts, n, t);
  const int slot = slots_in[i];
  if (slot < 0 || slot >= c.slots) {
    if (first) set_status(c, PG_CACHE_BAD_SLOT);
    return none;
  }
  if (marks && refused_of(c)[slot]) {
    if (first) set_status(c, PG_CACHE_REFUSED);
    return none;
  }
  const int pos = lens_of(c)[slot] - (starts[i + 1] - t);
  const int64_t entry = pos / c.page_size;
  const int page = pos >= 0 && entry < c.width ? row_of(c, slot)[entry] : -1;
  if (page < 0 || page >= c.pages) {
    if (first) set_status(c, PG_CACHE_BAD_PAGE);
    return none;
  }
  return Place{page, pos % c.page_size};
}


// WRITE: rows are quantised into the cache, else read back from it. A warp takes one token.
template <class T, bool WRITE>
__global__ void __launch_bounds__(kCopy, 4) cache8_rows(pg_cache c, pg_cache_scales s, int layer,
                                                     const int *slots_in, const int *starts, int n,
                                                     int tokens, pg_rows k, pg_rows v) {
  using X = Sixteen<T>;
  constexpr int kRowsAhead = WRITE ? 2 : 4;  // rows that a lane has in flight
  pg::wait_for_earlier_kernels();
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kCopy / 32);
  const int pieces = c.row_bytes / 16;
  int lanes = 1;  // that take a row
  while (lanes < pieces) lanes *= 2;
  const int sub = lane & (lanes - 1), step = 32 / lanes, rows = 2 * c.heads;
  if (blockIdx.x == 0 && threadIdx.x == 0 && (starts[0] < 0 || starts[n] > tokens))
    set_status(c, PG_CACHE_TOO_LONG);  // tokens that have no rows
  for (int t = (blockIdx.x * kCopy + threadIdx.x) >> 5; t < tokens; t += warps) {
    const Place at = place_of(c, slots_in, starts, n, t, WRITE);
    if (at.page < 0) continue;
    const int64_t in_cache = layer * c.layer_stride + at.page * c.page_stride +
                             static_cast<int64_t>(at.row) * c.row_bytes + sub * 16;
    const int64_t in_scales = layer * s.layer_stride + at.page * s.page_stride + at.row * 4ll;
    // row r of this lane's: the plane's first, then the other's
    const auto head_of = [&](int r) { return r < c.heads ? r : r - c.heads; };
    const auto cache_at = [&](int r) {
      return reinterpret_cast<uint4 *>((r < c.heads ? c.k : c.v) + in_cache +
                                       head_of(r) * c.head_stride);
    };
    const auto scale_at = [&](int r) {
      return reinterpret_cast<float *>((r < c.heads ? s.k : s.v) + in_scales +
                                       head_of(r) * s.head_stride);
    };
    const auto user_at = [&](int r) {
      const pg_rows &u = r < c.heads ? k : v;
      return reinterpret_cast<uint4 *>(u.data + t * u.token_stride + head_of(r) * u.head_stride) +
             sub * X::words;
    };
    for (int base = lane / lanes; base < rows + lane / lanes; base += kRowsAhead * step) {
      if constexpr (WRITE) {
        uint4 raw[kRowsAhead][X::words] = {};
#pragma unroll
        for (int j = 0; j < kRowsAhead; ++j) {
          const int r = base + j * step;
          if (r < rows && sub < pieces)
#pragma unroll
            for (int i = 0; i < X::words; ++i) raw[j][i] = user_at(r)[i];
        }
#pragma unroll
        for (int j = 0; j < kRowsAhead; ++j) {
          const int r = base + j * step;
          float x[16];
          X::get(raw[j], x);
          float most = 0.0f;  // NaN if one is
#pragma unroll
          for (int i = 0; i < 16; i += 2) most = pg::max3(most, fabsf(x[i]), fabsf(x[i + 1]));
          for (int off = lanes / 2; off; off /= 2) {
            const float o = __shfl_xor_sync(0xffffffffu, most, off);
            most = pg::max3(most, o, o);
          }
          const bool finite = most < INFINITY;
          const float scale = finite ? __fdiv_rn(most, 127.0f) : NAN;
          if (r < rows && sub < pieces) {
            // of a row that is not finite nothing is kept but that
            *cache_at(r) = !finite            ? make_uint4(0, 0, 0, 0)
                           : scale < 0x1p-100f ? quantise_small(raw[j], X::words, scale)
                                               : quantise(x, scale);
            if (sub == 0) *scale_at(r) = scale;
          }
        }
      } else {
        uint4 raw[kRowsAhead];
        float scale[kRowsAhead];
#pragma unroll
        for (int j = 0; j < kRowsAhead; ++j) {
          const int r = base + j * step;
          if (r < rows && sub < pieces) raw[j] = *cache_at(r), scale[j] = *scale_at(r);
        }
#pragma unroll
        for (int j = 0; j < kRowsAhead; ++j) {
          const int r = base + j * step;
          if (!(r < rows && sub < pieces)) continue;
          const uint32_t w[4] = {raw[j].x ^ 0x80808080u, raw[j].y ^ 0x80808080u,
                                 raw[j].z ^ 0x80808080u, raw[j].w ^ 0x80808080u};
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)  // 2^23 + 128 + q, less the former
            x[i] = (__uint_as_float(__byte_perm(w[i / 4], 0x4b000000u, 0x7440 + i % 4)) -
                    8388736.0f) * scale[j];
          uint4 out[X::words];
          X::put(x, out);
#pragma unroll
          for (int i = 0; i < X::words; ++i) user_at(r)[i] = out[i];
        }
      }
    }
  }
}

// The rows of a cache that is not in 8 bits, as they are.
__global__ void __launch_bounds__(kCopy) cache_read(pg_cache c, int layer, const int *slots_in,
                                                    const int *starts, int n, int tokens, pg_rows k,
                                                    pg_rows v) {
  pg::wait_for_earlier_kernels();
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kCopy / 32);
  const int pieces = c.row_bytes / 16, all = 2 * c.heads * pieces;
  if (blockIdx.x == 0 && threadIdx.x == 0 && (starts[0] < 0 || starts[n] > tokens))
    set_status(c, PG_CACHE_TOO_LONG);
  for (int t = (blockIdx.x * kCopy + threadIdx.x) >> 5; t < tokens; t += warps) {
    const Place at = place_of(c, slots_in, starts, n, t, false);
    if (at.page < 0) continue;
    const int64_t in = layer * c.layer_stride + at.page * c.page_stride +
                       static_cast<int64_t>(at.row) * c.row_bytes;
    for (int base = lane; base < all; base += 32 * kUnroll) {
      uint4 x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = base + 32 * u, r = j / pieces, head = r < c.heads ? r : r - c.heads;
        if (j < all)
          x[u] = pg::load16(reinterpret_cast<const char *>(r < c.heads ? c.k : c.v) + in +
                            head * c.head_stride + (j - r * pieces) * 16);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = base + 32 * u, r = j / pieces, head = r < c.heads ? r : r - c.heads;
        const pg_rows &to = r < c.heads ? k : v;
        if (j < all)
          *reinterpret_cast<uint4 *>(to.data + t * to.token_stride + head * to.head_stride +
                                     (j - r * pieces) * 16) = x[u];
      }
    }
  }
}

// --- keep: an accepted branch stays, the rest of the drafted tokens goes ---------------------------
// Of a slot's last tokens (its drafts) those in a set stay and move together, behind what was there
// before. A block takes a slot's rows of one layer, and a thread 16 bytes of all of them from the first
// to the last: a token never moves up, so what a move writes over has been moved before or goes. The
// blocks all look whether a slot's request can be met, in the same way and before anything changes; the
// pages and lengths follow in a second kernel.

constexpr int kDrafts = 64;  // bits of a set

struct Drafts {
  bool good;
  int slot, length, base, moves;  // base: the position of the first of them
  uint64_t kept;
};

// A warp's: the request of entry i, and where its moves come from and go to (byte offsets of rows in a
// layer's keys; page and row are what the scales need).
__device__ Drafts drafts_of(const pg_cache &c, const int *slots_in, const int *starts,
                            const uint64_t *kept, int n, int i, int2 *from, int2 *to) {
  const int lane = threadIdx.x & 31;
  Drafts d{};
  d.slot = slots_in[i];
  const int count = starts[i + 1] - starts[i];
  unsigned bad = 0;
  bool twice = false;
  for (int j = lane; j < n; j += 32) twice |= j != i && slots_in[j] == d.slot;
  if (__any_sync(0xffffffffu, twice) || d.slot < 0 || d.slot >= c.slots) {
    bad = PG_CACHE_BAD_SLOT;
  } else if (refused_of(c)[d.slot]) {
    bad = PG_CACHE_REFUSED;
  } else {
    d.length = lens_of(c)[d.slot];
    d.base = d.length - count;
    if (count < 0 || count > kDrafts || d.base < 0 || d.length > c.width * static_cast<int64_t>(c.page_size))
      bad = PG_CACHE_TOO_LONG;
  }
  if (!bad) {
    d.kept = count < 64 ? kept[i] & ((1ull << count) - 1) : kept[i];
    const int *row = row_of(c, d.slot);
    bool wrong = false;
    for (int b = lane; b < kDrafts; b += 32) {
      if (b >= count) continue;
      const int pos = d.base + b, page = row[pos / c.page_size];
      if (page < 0 || page >= c.pages) wrong = true;
      const int rank = __popcll(d.kept & ((1ull << b) - 1));
      if (!(d.kept >> b & 1) || wrong) continue;
      const int target = d.base + rank, target_page = row[target / c.page_size];
      if (target_page < 0 || target_page >= c.pages) {
        wrong = true;
        continue;
      }
      // other slots may read what is shared
      if (rank != b && refs_of(c)[target_page] != 1) wrong = true;
      from[rank] = make_int2(page, pos % c.page_size);
      to[rank] = make_int2(target_page, target % c.page_size);
    }
    if (__any_sync(0xffffffffu, wrong)) bad = PG_CACHE_BAD_PAGE;
  }
  d.good = !bad;
  d.moves = __popcll(d.kept);
  if (bad && lane == 0) set_status(c, bad);
  __syncwarp();
  return d;
}

__global__ void __launch_bounds__(kCopy) cache_keep_move(pg_cache c, pg_cache_scales s,
                                                         const int *slots_in, const int *starts,
                                                         const uint64_t *kept, int n) {
  __shared__ int2 from[kDrafts], to[kDrafts];
  __shared__ int first, moves;
  pg::wait_for_earlier_kernels();
  int *verdict = reinterpret_cast<int *>(c.scratch) + kHeader;
  const int pieces = c.row_bytes / 16, plane = c.heads * pieces;
  const int64_t tasks = static_cast<int64_t>(n) * c.layers;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int i = static_cast<int>(task / c.layers), layer = static_cast<int>(task % c.layers);
    __syncthreads();
    if (threadIdx.x < 32) {
      const Drafts d = drafts_of(c, slots_in, starts, kept, n, i, from, to);
      if (threadIdx.x == 0) {
        // those that stay in front stay where they are
        first = __ffsll(~d.kept) ? __ffsll(~d.kept) - 1 : kDrafts;
        moves = d.good ? d.moves : 0;
        if (layer == 0) verdict[i] = d.good;
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * plane; j += kCopy) {
      const int r = j < plane ? j : j - plane, head = r / pieces;
      char *const at = reinterpret_cast<char *>(j < plane ? c.k : c.v) + layer * c.layer_stride +
                       head * c.head_stride + (r - head * pieces) * 16;
      for (int m0 = first; m0 < moves; m0 += kUnroll) {
        uint4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (m0 + u < moves)
            x[u] = pg::load16(at + from[m0 + u].x * c.page_stride +
                              static_cast<int64_t>(from[m0 + u].y) * c.row_bytes);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (m0 + u < moves)
            *reinterpret_cast<uint4 *>(at + to[m0 + u].x * c.page_stride +
                                       static_cast<int64_t>(to[m0 + u].y) * c.row_bytes) = x[u];
      }
    }
    if (s.k)
      for (int j = threadIdx.x; j < 2 * c.heads; j += kCopy) {
        char *const at = reinterpret_cast<char *>(j < c.heads ? s.k : s.v) + layer * s.layer_stride +
                         (j < c.heads ? j : j - c.heads) * s.head_stride;
        for (int m = first; m < moves; ++m)
          *reinterpret_cast<float *>(at + to[m].x * s.page_stride + to[m].y * 4ll) =
              *reinterpret_cast<const float *>(at + from[m].x * s.page_stride + from[m].y * 4ll);
      }
  }
}

// A warp a slot: its new length, and the pages past it go.
__global__ void __launch_bounds__(kCopy) cache_keep_drop(pg_cache c, const int *slots_in,
                                                         const int *starts, const uint64_t *kept,
                                                         int n) {
  pg::wait_for_earlier_kernels();
  const int lane = threadIdx.x & 31, i = (blockIdx.x * kCopy + threadIdx.x) >> 5;
  const int *verdict = reinterpret_cast<const int *>(c.scratch) + kHeader;
  if (i >= n || !verdict[i]) return;
  const int slot = slots_in[i], count = starts[i + 1] - starts[i];
  const uint64_t set = count < 64 ? kept[i] & ((1ull << count) - 1) : kept[i];
  const int old = lens_of(c)[slot], length = old - count + __popcll(set);
  int *row = row_of(c, slot);
  for (int j = ceil_div(length, c.page_size) + lane; j < ceil_div(old, c.page_size); j += 32) {
    const int page = row[j];
    row[j] = -1;
    if (atomicSub(refs_of(c) + page, 1) <= 0) set_status(c, PG_CACHE_BAD_PAGE);
  }
  __syncwarp();
  if (lane == 0) lens_of(c)[slot] = length;
}

// --- host side ---------------------------------------------------------------------------------

int check(const char *what, const pg_cache *c) {
  if (!c) return pg::argument_fail("%s: null cache", what);
  if (!c->k || !c->v || !c->refs || !c->table || !c->lens || !c->status || !c->scratch)
    return pg::argument_fail("%s: the cache has a null pointer", what);
  if (c->layers < 1 || c->pages < 1 || c->heads < 1 || c->page_size < 1 || c->row_bytes < 16 ||
      c->slots < 1 || c->width < 1)
    return pg::argument_fail("%s: layers %d, pages %d, heads %d, page_size %d, row_bytes %d, "
                             "slots %d, width %d: all must be positive", what, c->layers,
                             c->pages, c->heads, c->page_size, c->row_bytes, c->slots, c->width);
  if (static_cast<int64_t>(c->page_size) * c->width > INT32_MAX / 2 ||
      static_cast<int64_t>(c->heads) * c->page_size * c->row_bytes > INT32_MAX)
    return pg::argument_fail("%s: a slot holds %d pages of %d rows of %d heads: too many", what,
                             c->width, c->page_size, c->heads);
  if ((c->k | c->v | static_cast<uint64_t>(c->layer_stride | c->page_stride | c->head_stride |
                                           c->row_bytes)) & 15)
    return pg::argument_fail("%s: keys, values, their strides and rows must be multiples of 16 "
                             "bytes (rows are %d)", what, c->row_bytes);
  if ((c->refs | c->table | c->lens | c->status | c->scratch) & 3)
    return pg::argument_fail("%s: counts, table, lengths, status and scratch must be 4-byte "
                             "aligned", what);
  if (c->table_stride < c->width || c->scratch_words < PG_CACHE_SCRATCH(c->pages, c->slots))
    return pg::argument_fail("%s: table_stride %lld below the width %d, or %lld scratch words "
                             "below the %lld needed", what,
                             static_cast<long long>(c->table_stride), c->width,
                             static_cast<long long>(c->scratch_words),
                             static_cast<long long>(PG_CACHE_SCRATCH(c->pages, c->slots)));
  return PG_OK;
}

int check_list(const char *what, const pg_cache *c, uint64_t a, uint64_t b, int n, int most) {
  int rc = check(what, c);
  if (rc) return rc;
  if (n < 0 || n > most) return pg::argument_fail("%s: %d entries, want 0..%d", what, n, most);
  if (n && (!a || !b || ((a | b) & 3)))
    return pg::argument_fail("%s: a list is null or not 4-byte aligned", what);
  return PG_OK;
}

// ... of slots, by the calls that set, read or clear their marks.
int check_slots(const char *what, const pg_cache *c, uint64_t a, uint64_t b, int n) {
  int rc = check_list(what, c, a, b, n, c ? c->slots : 0);
  if (rc) return rc;
  if (n && (!c->refused || c->refused & 3))
    return pg::argument_fail("%s: the slots' marks are null or not 4-byte aligned", what);
  return PG_OK;
}

int check_rows(const char *what, const pg_rows *r) {
  if (!r || !r->data) return pg::argument_fail("%s: null rows", what);
  if ((r->data | static_cast<uint64_t>(r->token_stride | r->head_stride)) & 15)
    return pg::argument_fail("%s: rows and their strides must be multiples of 16 bytes", what);
  return PG_OK;
}

int check_scales(const char *what, const pg_cache *c, const pg_cache_scales *s) {
  if (!s || !s->k || !s->v) return pg::argument_fail("%s: null scales", what);
  if ((s->k | s->v | static_cast<uint64_t>(s->layer_stride | s->page_stride | s->head_stride)) & 3)
    return pg::argument_fail("%s: scales and their strides must be multiples of 4 bytes", what);
  if (c->row_bytes > 512)
    return pg::argument_fail("%s: heads of %d in 8 bits, want 512 at most", what, c->row_bytes);
  return PG_OK;
}

const pg_cache_scales kNoScales = {};

// Blocks for `tasks` tasks: one each, up to the most, which loop.
int copy_grid(int64_t tasks, int *grid) {
  int sms;
  int rc = pg::sm_count(&sms);
  if (rc) return rc;
  const int64_t most = static_cast<int64_t>(sms) * kCopyPerSm;
  *grid = static_cast<int>(tasks < most ? (tasks < 1 ? 1 : tasks) : most);
  return PG_OK;
}

inline cudaStream_t stream_of(uint64_t s) {
  return reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(s));
}
inline const int *ints(uint64_t p) {
  return reinterpret_cast<const int *>(static_cast<uintptr_t>(p));
}

}  // namespace

extern "C" int pg_cache_extend(const pg_cache *c, uint64_t slots, uint64_t starts, int32_t n,
                               uint64_t stream) {
  int rc = check_slots("pg_cache_extend", c, slots, starts, n);
  if (rc || !n) return rc;
  return pg::launch<cache_extend>("cache_extend", dim3(1), kPlan, 0, stream_of(stream), *c,
                    ints(slots), ints(starts), n);
}

extern "C" int pg_cache_write(const pg_cache *c, int32_t layer, uint64_t slots, uint64_t starts,
                              int32_t n, int32_t tokens, const pg_rows *k, const pg_rows *v,
                              uint64_t stream) {
  int rc = check_slots("pg_cache_write", c, slots, starts, n);
  if (rc) return rc;
  if (layer < 0 || layer >= c->layers || tokens < 0)
    return pg::argument_fail("pg_cache_write: layer %d of %d, %d tokens", layer, c->layers,
                             tokens);
  if (!n || !tokens) return PG_OK;
  if ((rc = check_rows("pg_cache_write", k)) || (rc = check_rows("pg_cache_write", v))) return rc;
  int grid;
  if ((rc = copy_grid((tokens + kCopy / 32 - 1) / (kCopy / 32), &grid))) return rc;
  return pg::launch<cache_write>("cache_write", dim3(grid), kCopy, 0, stream_of(stream), *c,
                    layer, ints(slots), ints(starts), n, tokens, *k, *v);
}

extern "C" int pg_cache_free(const pg_cache *c, uint64_t slots, int32_t n, uint64_t stream) {
  int rc = check_slots("pg_cache_free", c, slots, slots, n);
  if (rc || !n) return rc;
  int grid;
  if ((rc = copy_grid(n, &grid))) return rc;
  return pg::launch<cache_free>("cache_free", dim3(grid), kCopy, 0, stream_of(stream), *c,
                    ints(slots), n);
}

static int copy_pages(const char *what, const pg_cache *c, const pg_cache_scales &s, uint64_t from,
                      uint64_t to, int32_t n, uint64_t stream) {
  int rc = check_list(what, c, from, to, n, c ? c->pages : 0);
  if (rc || !n) return rc;
  int grid;
  if ((rc = copy_grid(static_cast<int64_t>(n) * c->layers * 2, &grid))) return rc;
  return pg::launch<cache_copy>("cache_copy", dim3(grid), kCopy, 0, stream_of(stream), *c, s,
                    ints(from), ints(to), n);
}

static int fork(const char *what, const pg_cache *c, const pg_cache_scales &s, uint64_t parents,
                uint64_t children, int32_t n, uint64_t stream) {
  int rc = check_slots(what, c, parents, children, n);
  if (rc || !n) return rc;
  int grid;
  if ((rc = copy_grid(static_cast<int64_t>(n) * (2 * c->layers + 1), &grid))) return rc;
  rc = pg::launch<cache_fork_plan>("cache_fork_plan", dim3(kLook), kPlan, 0, stream_of(stream), *c,
                  ints(parents), ints(children), n);
  if (rc) return rc;
  return pg::launch<cache_fork_copy>("cache_fork_copy", dim3(grid), kCopy, 0, stream_of(stream),
                    *c, s, ints(parents), ints(children), n);
}

static int compact(const char *what, const pg_cache *c, const pg_cache_scales &s, uint64_t stream) {
  int rc = check(what, c);
  if (rc) return rc;
  int grid;
  if ((rc = copy_grid(c->slots + static_cast<int64_t>(c->pages) * c->layers, &grid))) return rc;
  rc = pg::launch<cache_compact_plan>("cache_compact_plan", dim3(1), kPlan, 0, stream_of(stream),
                  *c);
  if (rc) return rc;
  return pg::launch<cache_compact_move>("cache_compact_move", dim3(grid), kCopy, 0,
                    stream_of(stream), *c, s);
}

extern "C" int pg_cache_copy(const pg_cache *c, uint64_t from, uint64_t to, int32_t n,
                             uint64_t stream) {
  return copy_pages("pg_cache_copy", c, kNoScales, from, to, n, stream);
}

extern "C" int pg_cache_fork(const pg_cache *c, uint64_t parents, uint64_t children, int32_t n,
                             uint64_t stream) {
  return fork("pg_cache_fork", c, kNoScales, parents, children, n, stream);
}

extern "C" int pg_cache_compact(const pg_cache *c, uint64_t stream) {
  return compact("pg_cache_compact", c, kNoScales, stream);
}

// Of a cache in 8 bits: the arguments' checks that all of these share.
static int check8(const char *what, const pg_cache *c, const pg_cache_scales *s) {
  const int rc = check(what, c);
  return rc ? rc : check_scales(what, c, s);
}

extern "C" int pg_cache8_copy(const pg_cache *c, const pg_cache_scales *s, uint64_t from, uint64_t to,
                              int32_t n, uint64_t stream) {
  const int rc = check8("pg_cache8_copy", c, s);
  return rc ? rc : copy_pages("pg_cache8_copy", c, *s, from, to, n, stream);
}

extern "C" int pg_cache8_fork(const pg_cache *c, const pg_cache_scales *s, uint64_t parents,
                              uint64_t children, int32_t n, uint64_t stream) {
  const int rc = check8("pg_cache8_fork", c, s);
  return rc ? rc : fork("pg_cache8_fork", c, *s, parents, children, n, stream);
}

extern "C" int pg_cache8_compact(const pg_cache *c, const pg_cache_scales *s, uint64_t stream) {
  const int rc = check8("pg_cache8_compact", c, s);
  return rc ? rc : compact("pg_cache8_compact", c, *s, stream);
}

// Rows in and out of a layer, the arguments of both.
static int check_layer(const char *what, const pg_cache *c, int32_t layer, uint64_t slots,
                       uint64_t starts, int32_t n, int32_t tokens, const pg_rows *k,
                       const pg_rows *v) {
  int rc = check_slots(what, c, slots, starts, n);
  if (rc) return rc;
  if (layer < 0 || layer >= c->layers || tokens < 0)
    return pg::argument_fail("%s: layer %d of %d, %d tokens", what, layer, c->layers, tokens);
  if (!n || !tokens) return PG_OK;
  if ((rc = check_rows(what, k))) return rc;
  return check_rows(what, v);
}

template <class T, bool WRITE>
static int launch_rows(const pg_cache *c, const pg_cache_scales *s, int32_t layer, uint64_t slots,
                       uint64_t starts, int32_t n, int32_t tokens, const pg_rows *k,
                       const pg_rows *v, uint64_t stream) {
  int grid;
  const int rc = copy_grid((tokens + kCopy / 32 - 1) / (kCopy / 32), &grid);
  if (rc) return rc;
  return pg::launch<cache8_rows<T, WRITE>>("cache8_rows", dim3(grid), kCopy, 0, stream_of(stream),
                                           *c, *s, layer, ints(slots), ints(starts), n, tokens, *k,
                                           *v);
}

extern "C" int pg_cache8_write(const pg_cache *c, const pg_cache_scales *s, int32_t layer,
                               uint64_t slots, uint64_t starts, int32_t n, int32_t tokens,
                               int32_t dtype, const pg_rows *k, const pg_rows *v, uint64_t stream) {
  const char *what = "pg_cache8_write";
  int rc = check8(what, c, s);
  if (!rc) rc = check_layer(what, c, layer, slots, starts, n, tokens, k, v);
  if (rc) return rc;
  if (dtype != PG_DT_F32 && dtype != PG_DT_BF16 && dtype != PG_DT_F16)
    return pg::argument_fail("%s: dtype %d, want f32, bf16 or f16", what, dtype);
  if (!n || !tokens) return PG_OK;
  const auto run = dtype == PG_DT_F32    ? launch_rows<float, true>
                   : dtype == PG_DT_BF16 ? launch_rows<__nv_bfloat16, true>
                                         : launch_rows<__half, true>;
  return run(c, s, layer, slots, starts, n, tokens, k, v, stream);
}

extern "C" int pg_cache_read(const pg_cache *c, const pg_cache_scales *s, int32_t layer,
                             uint64_t slots, uint64_t starts, int32_t n, int32_t tokens,
                             int32_t dtype, const pg_rows *k, const pg_rows *v, uint64_t stream) {
  const char *what = "pg_cache_read";
  int rc = s ? check8(what, c, s) : PG_OK;
  if (!rc) rc = check_layer(what, c, layer, slots, starts, n, tokens, k, v);
  if (rc) return rc;
  if (s && dtype != PG_DT_F32 && dtype != PG_DT_BF16 && dtype != PG_DT_F16)
    return pg::argument_fail("%s: dtype %d, want f32, bf16 or f16", what, dtype);
  if (!n || !tokens) return PG_OK;
  if (!s) {
    int grid;
    if ((rc = copy_grid((tokens + kCopy / 32 - 1) / (kCopy / 32), &grid))) return rc;
    return pg::launch<cache_read>("cache_read", dim3(grid), kCopy, 0, stream_of(stream), *c, layer,
                                  ints(slots), ints(starts), n, tokens, *k, *v);
  }
  const auto run = dtype == PG_DT_F32    ? launch_rows<float, false>
                   : dtype == PG_DT_BF16 ? launch_rows<__nv_bfloat16, false>
                                         : launch_rows<__half, false>;
  return run(c, s, layer, slots, starts, n, tokens, k, v, stream);
}

extern "C" int pg_cache_keep(const pg_cache *c, const pg_cache_scales *s, uint64_t slots,
                             uint64_t starts, uint64_t kept, int32_t n, uint64_t stream) {
  const char *what = "pg_cache_keep";
  int rc = s ? check8(what, c, s) : PG_OK;
  if (!rc) rc = check_slots(what, c, slots, starts, n);
  if (rc || !n) return rc;
  if (!kept || kept & 7) return pg::argument_fail("%s: kept is null or not 8-byte aligned", what);
  int grid;
  if ((rc = copy_grid(static_cast<int64_t>(n) * c->layers, &grid))) return rc;
  const uint64_t *sets = reinterpret_cast<const uint64_t *>(static_cast<uintptr_t>(kept));
  rc = pg::launch<cache_keep_move>("cache_keep_move", dim3(grid), kCopy, 0, stream_of(stream), *c,
                                   s ? *s : kNoScales, ints(slots), ints(starts), sets, n);
  if (rc) return rc;
  return pg::launch<cache_keep_drop>("cache_keep_drop", dim3((n + kCopy / 32 - 1) / (kCopy / 32)),
                                     kCopy, 0, stream_of(stream), *c, ints(slots), ints(starts),
                                     sets, n);
}

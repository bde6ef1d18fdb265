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

__device__ void copy_rows(const pg_cache &c, char *base, int layer, int from, int to, int rows) {
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
__global__ void __launch_bounds__(kCopy) cache_copy(pg_cache c, const int *from, const int *to,
                                                    int n) {
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
    copy_rows(c, reinterpret_cast<char *>(plane & 1 ? c.v : c.k), plane >> 1, a, b, c.page_size);
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
__global__ void __launch_bounds__(kCopy) cache_fork_copy(pg_cache c, const int *parents,
                                                         const int *children, int n) {
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
        copy_rows(c, reinterpret_cast<char *>(part & 1 ? c.k : c.v), (part - 1) >> 1, from[full],
                  fresh[offset[i]], open);
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
__global__ void __launch_bounds__(kCopy) cache_compact_move(pg_cache c) {
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
    copy_rows(c, reinterpret_cast<char *>(plane & 1 ? c.v : c.k), plane >> 1, movers[i],
              holes[i], c.page_size);
  }
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

extern "C" int pg_cache_copy(const pg_cache *c, uint64_t from, uint64_t to, int32_t n,
                             uint64_t stream) {
  int rc = check_list("pg_cache_copy", c, from, to, n, c ? c->pages : 0);
  if (rc || !n) return rc;
  int grid;
  if ((rc = copy_grid(static_cast<int64_t>(n) * c->layers * 2, &grid))) return rc;
  return pg::launch<cache_copy>("cache_copy", dim3(grid), kCopy, 0, stream_of(stream), *c,
                    ints(from), ints(to), n);
}

extern "C" int pg_cache_fork(const pg_cache *c, uint64_t parents, uint64_t children, int32_t n,
                             uint64_t stream) {
  int rc = check_slots("pg_cache_fork", c, parents, children, n);
  if (rc || !n) return rc;
  int grid;
  if ((rc = copy_grid(static_cast<int64_t>(n) * (2 * c->layers + 1), &grid))) return rc;
  rc = pg::launch<cache_fork_plan>("cache_fork_plan", dim3(kLook), kPlan, 0, stream_of(stream), *c,
                  ints(parents), ints(children), n);
  if (rc) return rc;
  return pg::launch<cache_fork_copy>("cache_fork_copy", dim3(grid), kCopy, 0, stream_of(stream),
                    *c, ints(parents), ints(children), n);
}

extern "C" int pg_cache_compact(const pg_cache *c, uint64_t stream) {
  int rc = check("pg_cache_compact", c);
  if (rc) return rc;
  int grid;
  if ((rc = copy_grid(c->slots + static_cast<int64_t>(c->pages) * c->layers, &grid))) return rc;
  rc = pg::launch<cache_compact_plan>("cache_compact_plan", dim3(1), kPlan, 0, stream_of(stream),
                  *c);
  if (rc) return rc;
  return pg::launch<cache_compact_move>("cache_compact_move", dim3(grid), kCopy, 0,
                    stream_of(stream), *c);
}

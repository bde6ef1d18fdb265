// The kernel of many new tokens (attention_prompt.cuh) over a cache in 8 bits.
//
// Its blocks take 256 rows each, and those of one kv head widen the same keys over and over: seven warps
// beside the products need 7000 cycles for what a step's exponentials and products need 4000 for. So
// where a sequence has rows for several blocks, its keys and values are widened once, into the
// workspace as a 16-bit cache with pages of 128 tokens, as many kv heads at a time as there is room for,
// and the kernel runs over that. Both ways round a key or value to the type once, so the results are
// the same.
#include "attention_prompt.cuh"

namespace {

constexpr int kWiden = 256;  // threads of a widening block
// Bytes of the workspace that stay the parts' (of a long sequence's result).
constexpr int64_t kPartsBytes = 16 << 20;
// Widening comes first from so many rows a sequence on, if it takes few rounds or each of them has tiles
// for all SMs. With and without, bf16, 32 heads on 8 of 128, up to 8192 keys, in microseconds: 2 sequences
// with 2048 new tokens (8192 rows) 477 and 898, 512 213 and 384, 256 170 and 212, 128 132 and 149, 64 127
// and 93; 8 sequences with 256, in eight rounds of one kv head, 581 and 448, with 64 475 and 415.
constexpr int64_t kWidenRows = 768;
constexpr int kFewRounds = 3;

// Block (i, h): keys 128 i.. of the batch's sequences, each with `blocks` such blocks, of kv head first + h;
// block (i, heads + h) the values. HBM bounds it: a byte read and two written.
template <class T>
__global__ void __launch_bounds__(kWiden)
    widen_kernel(Attention a, int blocks, int first, int heads, char *k_to, char *v_to, int *table,
                 int *lens) {
  pg::wait_for_earlier_kernels();
  const int b = blockIdx.x / blocks, block = blockIdx.x - b * blocks;
  const int head = blockIdx.y < heads ? blockIdx.y : blockIdx.y - heads;
  const bool values = static_cast<int>(blockIdx.y) >= heads, main = !blockIdx.y && !threadIdx.x;
  const int slot = a.slots ? a.slots[b] : b;
  int length = 0;
  if (slot < 0 || slot >= a.slot_rows) {
    if (main) atomicOr(a.status, PG_CACHE_BAD_SLOT);
  } else {
    const int most = min(blocks * kKeys, a.width * a.page_size);
    length = a.lens[slot];
    if (length < 0 || length > most) {
      if (main) atomicOr(a.status, PG_CACHE_TOO_LONG);
      length = length < 0 ? 0 : most;
    }
  }
  if (main) {
    table[blockIdx.x] = blockIdx.x;
    if (block == 0) lens[b] = length;
  }
  const int key0 = block * kKeys;
  if (key0 >= length) return;
  if (a.window) {  // what no query sees is not needed
    const int start = a.starts[b], count = max(0, a.starts[b + 1] - start);
    if (key0 + kKeys <= length - count - a.window && key0 >= a.sinks) return;
  }
  const int *pages = a.table + slot * a.table_row;
  const int pieces = a.dim / 16;
  const char *from = (values ? a.v : a.k) + (first + head) * (values ? a.v_head : a.k_head);
  const char *of = (values ? a.v_scale : a.k_scale) + (first + head) * (values ? a.vs_head : a.ks_head);
  const int64_t page_bytes = values ? a.v_page : a.k_page, of_bytes = values ? a.vs_page : a.ks_page;
  uint4 *const to = reinterpret_cast<uint4 *>(
      (values ? v_to : k_to) + (static_cast<int64_t>(blockIdx.x) * heads + head) * kKeys * a.dim * 2);
  constexpr int kAhead = 4;  // loads a thread has in flight
  for (int i0 = threadIdx.x; i0 < kKeys * pieces; i0 += kWiden * kAhead) {
    uint4 raw[kAhead];
    float scale[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kWiden, r = i / pieces, key = key0 + r;
      raw[u] = make_uint4(0, 0, 0, 0);
      scale[u] = 0.0f;
      if (i >= kKeys * pieces || key >= length) continue;
      const int entry = pg::page_index(a, key), row = key - entry * a.page_size, page = pages[entry];
      if (page < 0 || page >= a.pages) {
        atomicOr(a.status, PG_CACHE_BAD_PAGE);
        continue;
      }
      raw[u] = pg::load16(from + page * page_bytes + static_cast<int64_t>(row) * a.dim +
                          (i - r * pieces) * 16);
      scale[u] = *reinterpret_cast<const float *>(of + page * of_bytes + row * 4ll);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kWiden;
      if (i >= kKeys * pieces) continue;
      uint4 out[2];
      widen<T>(raw[u], scale[u], out);
      to[2 * i] = out[0], to[2 * i + 1] = out[1];
    }
  }
}

template <class T>
int widen_first(Attention a, bool bf16, int max_len, int heads, int blocks, int64_t head_bytes, int sms,
                cudaStream_t stream) {
  const int64_t meta = (4ll * a.batch * (blocks + 1) + 255) / 256 * 256;
  char *const scratch = reinterpret_cast<char *>(a.partial) + kPartsBytes;
  int *const table = reinterpret_cast<int *>(scratch);
  int *const lens = table + static_cast<int64_t>(a.batch) * blocks;
  const int rounds = (a.heads + heads - 1) / heads;
  for (int i = 0; i < rounds; ++i) {
    // as even as they come
    const int first = static_cast<int>(static_cast<int64_t>(a.heads) * i / rounds);
    const int n = static_cast<int>(static_cast<int64_t>(a.heads) * (i + 1) / rounds) - first;
    char *const k = scratch + meta, *const v = k + n * head_bytes;
    int rc = pg::launch<widen_kernel<T>>("widen_kernel", dim3(a.batch * blocks, 2 * n), kWiden, 0,
                                         stream, a, blocks, first, n, k, v, table, lens);
    if (rc) return rc;
    Attention b = a;
    b.q += first * a.group * a.q_head, b.out += first * a.group * a.out_head;
    b.k = k, b.v = v, b.k_scale = b.v_scale = nullptr;
    b.k_head = b.v_head = static_cast<int64_t>(kKeys) * a.dim * 2;
    b.k_page = b.v_page = n * b.k_head;
    b.table = table, b.table_row = blocks, b.lens = lens, b.slots = nullptr;
    b.slot_rows = a.batch, b.heads = n, b.page_size = kKeys, b.width = blocks;
    b.pages = a.batch * blocks;
    b.page_mul = 1, b.page_shift = 7;
    rc = a.mask ? pg::prompt_tree(b, bf16, max_len, kPartsBytes, sms, stream)
                : pg::prompt_16bit(b, bf16, max_len, kPartsBytes, sms, stream);
    if (rc) return rc;
  }
  return PG_OK;
}

}  // namespace

namespace pg {

int prompt_8bit(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                cudaStream_t stream) {
  const int64_t blocks = (max_len + kKeys - 1ll) / kKeys;
  const int64_t head_bytes = a.batch * blocks * kKeys * a.dim * 2;  // of its keys
  const int64_t room = partial_bytes - kPartsBytes - 4 * a.batch * (blocks + 1) - 256;
  const int64_t heads = room > 0 ? room / (2 * head_bytes) : 0;
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  if (heads >= 1 && a.batch * blocks <= INT32_MAX / 2 && rows >= kWidenRows * a.batch &&
      (heads * kFewRounds >= a.heads || heads * rows >= static_cast<int64_t>(kRows) * sms))
    return (bf16 ? widen_first<__nv_bfloat16> : widen_first<__half>)(
        a, bf16, max_len, static_cast<int>(heads < a.heads ? heads : a.heads), static_cast<int>(blocks),
        head_bytes, sms, stream);
  return a.mask ? run_prompt<true, true>(a, bf16, max_len, partial_bytes, sms, stream)
                : run_prompt<false, true>(a, bf16, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

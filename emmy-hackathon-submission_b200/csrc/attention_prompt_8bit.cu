// The kernel of many new tokens (attention_prompt.cuh) over a cache in 8 bits.
//
// Its blocks take 256 rows each, and those of one kv head widen the same keys over and over: seven warps
// beside the products need 7000 cycles for what a step's exponentials and products need 4000 for. So
// where a sequence has rows for several blocks, its keys and values are widened once, into the workspace as
// a 16-bit cache with pages of 128 tokens, as many kv heads at a time as there is room for, and the kernel
// runs over that.
//
// For f16 results the whole numbers are what is widened, scores are multiplied by each key's scale and
// weights by each value's, which go in as two f16 numbers, so that nothing but the result is rounded.
// Elsewhere, for bf16 results or
// without room in the workspace, numbers go to f16 as 2^-e of what they are, with one e for
// the keys, and one for the values, of a page of a head or of a block's part. bf16 would lose too much:
// keys rounded to it change a score of 8 by a hundredth, and results by three times as much as all other
// roundings together. In f16 they add little to bf16 results (1.8e-3 off with their own rounding of 1.6e-3)
// but would make f16 ones 4.9e-4 off, where theirs is 2.1e-4. The rows' threads bound it, so whole numbers
// cost: two sequences of 2048 new tokens and up to 8192 keys, 32 heads on 8 of 128, take 490 us in bf16 and
// 892 us in f16 (675 with one number a weight, and results up to 1.5 times as far off).
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
template <bool WHOLE>
__global__ void __launch_bounds__(kWiden)
    widen_kernel(Attention a, int blocks, int first, int heads, char *k_to, char *v_to, char *scales,
                 int *table, int *lens) {
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
  __shared__ unsigned top;  // the largest scale that is finite
  if (!threadIdx.x) top = 0;
  __syncthreads();
  if (threadIdx.x < kKeys && key0 + static_cast<int>(threadIdx.x) < length) {
    const int key = key0 + threadIdx.x, entry = pg::page_index(a, key), page = pages[entry];
    if (page >= 0 && page < a.pages) {
      atomicMax(&top, magnitude(of + page * of_bytes + (key - entry * a.page_size) * 4ll));
    }
  }
  __syncthreads();
  const int shift = shift_of(top, values);
  const float by = pg::power_of_2(-shift);
  const int64_t at_scales = static_cast<int64_t>(blockIdx.x) * heads + head;
  Scales *const whole = reinterpret_cast<Scales *>(scales) + at_scales;
  if (!threadIdx.x) {
    int2 *const to = reinterpret_cast<int2 *>(scales) + at_scales;
    if (!WHOLE) (values ? to->y : to->x) = shift;
    else if (values) whole->shift = shift + 8;
  }
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
      if constexpr (WHOLE) {  // a scale that is not finite goes into the numbers
        const bool finite = fabsf(scale[u]) < INFINITY;
        widen(raw[u], finite ? 1.0f : scale[u], out);
        if (i % pieces == 0)
          (values ? whole->v : whole->k)[i / pieces] =
              values ? finite ? scale[u] * by * 0x1p-8f : 0.0f : finite ? scale[u] : 1.0f;
      } else {
        widen(raw[u], scale[u] * by, out);
      }
      to[2 * i] = out[0], to[2 * i + 1] = out[1];
    }
  }
}

int widen_first(Attention a, bool bf16, int max_len, int heads, int blocks, int sms, cudaStream_t stream) {
  const int pages = a.batch * blocks;
  char *const scratch = reinterpret_cast<char *>(a.partial) + kPartsBytes;
  int *const table = reinterpret_cast<int *>(scratch), *const lens = table + pages;
  char *const k = scratch + (4ll * (pages + a.batch) + 255) / 256 * 256;
  for (int first = 0; first < a.heads; first += heads) {
    const int n = a.heads - first < heads ? a.heads - first : heads;
    Attention b = a;
    const int64_t head_bytes = static_cast<int64_t>(kKeys) * a.dim * 2;
    char *const v = k + pages * n * head_bytes;
    char *const scales = v + pages * n * head_bytes;
    const auto widen_all = [&](auto whole) {
      return pg::launch<widen_kernel<decltype(whole)::value>>("widen_kernel", dim3(pages, 2 * n), kWiden, 0,
                                                              stream, a, blocks, first, n, k, v, scales, table,
                                                              lens);
    };
    int rc = bf16 ? widen_all(std::false_type()) : widen_all(std::true_type());
    if (rc) return rc;
    b.q += first * a.group * a.q_head, b.out += first * a.group * a.out_head;
    b.k = k, b.v = v, b.k_scale = scales;
    b.k_head = b.v_head = head_bytes, b.k_page = b.v_page = n * head_bytes;
    b.ks_head = bf16 ? sizeof(int2) : sizeof(Scales), b.ks_page = n * b.ks_head;
    b.table = table, b.table_row = blocks, b.lens = lens, b.slots = nullptr;
    b.slot_rows = a.batch, b.heads = n, b.page_size = kKeys, b.width = blocks, b.pages = pages;
    if (bf16)
      rc = a.mask ? run_prompt_of<__nv_bfloat16, true, kShifted>(b, max_len, kPartsBytes, sms, stream)
                  : run_prompt_of<__nv_bfloat16, false, kShifted>(b, max_len, kPartsBytes, sms, stream);
    else
      rc = a.mask ? run_prompt_of<__half, true, kWhole>(b, max_len, kPartsBytes, sms, stream)
                  : run_prompt_of<__half, false, kWhole>(b, max_len, kPartsBytes, sms, stream);
    if (rc) return rc;
  }
  return PG_OK;
}

}  // namespace

namespace pg {

int prompt_8bit(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                cudaStream_t stream) {
  const int64_t blocks = (max_len + kKeys - 1ll) / kKeys, pages = a.batch * blocks;
  const int64_t room = partial_bytes - kPartsBytes - 4 * (pages + a.batch) - 256;
  // of a kv head: keys, values and scales
  const int64_t each = pages * (kKeys * a.dim * 4ll + (bf16 ? sizeof(int2) : sizeof(Scales)));
  int64_t heads = room > 0 ? room / each : 0;
  heads = heads < a.heads ? heads : a.heads;
  heads = heads < 32767 ? heads : 32767;  // twice as many rows of blocks
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  if (heads >= 1 && pages <= INT32_MAX / 2 &&
      (!bf16 || (rows >= kWidenRows * a.batch &&
                 (heads * kFewRounds >= a.heads || heads * rows >= static_cast<int64_t>(kRows) * sms)))) {
    const int64_t rounds = (a.heads + heads - 1) / heads;  // as even as they come
    return widen_first(a, bf16, max_len, static_cast<int>((a.heads + rounds - 1) / rounds),
                       static_cast<int>(blocks), sms, stream);
  }
  return a.mask ? run_prompt<true, kBytes>(a, bf16, max_len, partial_bytes, sms, stream)
                : run_prompt<false, kBytes>(a, bf16, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

// The single-token kernel (attention_decode.cuh) for caches in f32, bf16 and f16.
#include "attention_decode.cuh"

namespace pg {

// Whether this kernel takes a batch and not the large tiles of attention_prompt.cu: at up to 48
// rows a sequence on average, which those fill badly. The average says little of an uneven batch:
// 100 single tokens and one chunk of 1024, 4000 keys each and 4 heads on each of 8, come here and
// take 997 us, where the chunk alone takes 126 there and the tokens 289 here; 63 and one of 2048
// go there and take 387, alone 176 and 195. Even batches, by rows a sequence, this against those,
// in microseconds at head size 128: 7 sequences of up to 20000 keys on 4 kv heads, 16 rows 43 and
// 83, 32 rows 56 and 84, 48 rows 60 and 84, 64 rows 70 and 96; 32 of up to 8000 on 8, 16 rows 74
// and 157, 32 rows 119 and 158, 48 rows 155 and 160, 64 rows 191 and 160; 100 of up to 500 on 4,
// 48 rows 51 and 49, 64 rows 63 and 50.
// f32 has no such tiles, so it is taken at up to 256 rows, and at up to 1024 where most keys are
// seen by all of a sequence's queries, since a group of 16 rows goes through all that any sees. This
// against attention.cu: 8 sequences on 4 kv heads of 128, up to 4056 keys, 64 rows 86 and 164, 256
// rows 253 and 390, 1024 rows 947 and 1270; of no other keys than the queries, 256 rows 13 and 17,
// 512 rows 25 and 17; with a window of 100 and heads of 64, 256 rows 28 and 32, 512 rows 45 and 34.
bool decode_takes(const Attention &a, bool f32, int most, int max_len) {
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  const bool early = !a.window && max_len / 8ll * a.batch >= a.queries;
  if (a.starts && rows > (f32 ? early ? 1024ll : 256ll : 48ll) * a.batch) return false;
  return decode_counts(a, most);
}

bool decode_counts(const Attention &a, int most) {
  const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
  // blocks of 32 keys or more
  return (rows / kRows + a.batch) * a.heads * (most / 32 + 2ll + kPair) < INT32_MAX;
}

int decode(const Attention &a, int dtype, int sms, cudaStream_t stream) {
  return dtype == PG_DT_F32    ? launch_decode<float, float>(a, sms, stream)
         : dtype == PG_DT_BF16 ? launch_decode<__nv_bfloat16, __nv_bfloat16>(a, sms, stream)
                               : launch_decode<__half, __half>(a, sms, stream);
}

}  // namespace pg

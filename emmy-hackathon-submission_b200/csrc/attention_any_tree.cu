// The kernel of every head size (attention_any.cuh) for trees of drafted tokens.
#include "attention_any.cuh"

namespace pg {

int any_rows_tree(const Attention &a, int dtype, int max_len, int64_t partial_bytes, int sms,
                  cudaStream_t stream) {
  if (a.k_scale)
    return dtype == PG_DT_F32
               ? run<float, int8_t, 256, true>(a, max_len, partial_bytes, sms, stream)
           : dtype == PG_DT_BF16
               ? run<__nv_bfloat16, int8_t, 256, true>(a, max_len, partial_bytes, sms, stream)
               : run<__half, int8_t, 256, true>(a, max_len, partial_bytes, sms, stream);
  return dtype == PG_DT_F32 ? run<float, float, 256, true>(a, max_len, partial_bytes, sms, stream)
         : dtype == PG_DT_BF16
             ? run<__nv_bfloat16, __nv_bfloat16, 256, true>(a, max_len, partial_bytes, sms, stream)
             : run<__half, __half, 256, true>(a, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

// The single-token kernel (attention_decode.cuh) for trees of drafted tokens.
#include "attention_decode.cuh"

namespace pg {

int decode_tree(const Attention &a, int dtype, int sms, cudaStream_t stream) {
  if (a.k_scale)
    return dtype == PG_DT_F32    ? launch_dim<float, int8_t, kTree>(a, sms, stream)
           : dtype == PG_DT_BF16 ? launch_dim<__nv_bfloat16, int8_t, kTree>(a, sms, stream)
                                 : launch_dim<__half, int8_t, kTree>(a, sms, stream);
  return dtype == PG_DT_F32    ? launch_dim<float, float, kTree>(a, sms, stream)
         : dtype == PG_DT_BF16 ? launch_dim<__nv_bfloat16, __nv_bfloat16, kTree>(a, sms, stream)
                               : launch_dim<__half, __half, kTree>(a, sms, stream);
}

}  // namespace pg

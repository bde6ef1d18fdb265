// The single-token kernel (attention_decode.cuh) over a cache in 8 bits.
#include "attention_decode.cuh"

namespace pg {

int decode_8bit(const Attention &a, int dtype, int sms, cudaStream_t stream) {
  return dtype == PG_DT_F32    ? launch_decode<float, int8_t>(a, sms, stream)
         : dtype == PG_DT_BF16 ? launch_decode<__nv_bfloat16, int8_t>(a, sms, stream)
                               : launch_decode<__half, int8_t>(a, sms, stream);
}

}  // namespace pg

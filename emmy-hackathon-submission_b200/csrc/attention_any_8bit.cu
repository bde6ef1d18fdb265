// The kernel of every head size (attention_any.cuh) over a cache in 8 bits.
// Heads of up to 128 have kernels on the tensor cores, so one size of tile serves these.
#include "attention_any.cuh"

namespace pg {

int any_rows_8bit(const Attention &a, int dtype, int max_len, int64_t partial_bytes, int sms,
                  cudaStream_t stream) {
  return dtype == PG_DT_F32
             ? run<float, int8_t, 256, false>(a, max_len, partial_bytes, sms, stream)
         : dtype == PG_DT_BF16
             ? run<__nv_bfloat16, int8_t, 256, false>(a, max_len, partial_bytes, sms, stream)
             : run<__half, int8_t, 256, false>(a, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

// The kernel of many new tokens (attention_prompt.cuh) over a cache in 8 bits.
#include "attention_prompt.cuh"

namespace pg {

int prompt_8bit(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                cudaStream_t stream) {
  return a.mask ? run_prompt<true, true>(a, bf16, max_len, partial_bytes, sms, stream)
                : run_prompt<false, true>(a, bf16, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

// The kernel of many new tokens (attention_prompt.cuh) for trees of drafted tokens.
#include "attention_prompt.cuh"

namespace pg {

int prompt_tree(const Attention &a, bool bf16, int max_len, int64_t partial_bytes, int sms,
                cudaStream_t stream) {
  return run_prompt<true, kOfType>(a, bf16, max_len, partial_bytes, sms, stream);
}

}  // namespace pg

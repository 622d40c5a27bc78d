// gated_ffn on bf16 operands (policy_ffn.cuh)
#include "policy_ffn.cuh"

int inb::pol::ffn_bf16(const InbFfnArgs& a, bool bwd, cudaStream_t s) {
  return bwd ? ffn_backward<bf16>(a, s) : ffn_forward<bf16>(a, s);
}

// gated_ffn on fp16 operands (policy_ffn.cuh)
#include "policy_ffn.cuh"

int inb::pol::ffn_f16(const InbFfnArgs& a, bool bwd, cudaStream_t s) {
  return bwd ? ffn_backward<f16>(a, s) : ffn_forward<f16>(a, s);
}

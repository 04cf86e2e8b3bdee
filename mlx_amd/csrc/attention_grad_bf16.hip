// attention_grad_bf16.hip -- the kernels of attention_grad.h for bfloat16
#include "attention_grad.h"

namespace mlxrocm {

int launch_attention_grad_bf16(const AttentionGradArgs& g, hipStream_t s) {
  return launch_grad_typed<bf16_t>(g, s);
}

} // namespace mlxrocm

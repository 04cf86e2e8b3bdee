// attention_grad_f16.hip -- the kernels of attention_grad.h for float16
#include "attention_grad.h"

namespace mlxrocm {

int launch_attention_grad_f16(const AttentionGradArgs& g, hipStream_t s) {
  return launch_grad_typed<f16_t>(g, s);
}

} // namespace mlxrocm

// attention_grad_f32.hip -- the kernels of attention_grad.h for float32
#include "attention_grad.h"

namespace mlxrocm {

int launch_attention_grad_f32(const AttentionGradArgs& g, hipStream_t s) {
  return launch_grad_typed<float>(g, s);
}

} // namespace mlxrocm

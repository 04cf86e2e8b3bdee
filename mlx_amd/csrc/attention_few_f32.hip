// attention_few_f32.hip -- the kernels of attention_few.h for float32
#include "attention_few.h"

namespace mlxrocm {

int launch_attention_few_f32(const AttentionArgs& a, hipStream_t s) {
  return launch_few_typed<float>(a, s);
}

} // namespace mlxrocm

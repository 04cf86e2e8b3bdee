// attention_few_f16.hip -- the kernels of attention_few.h for float16
#include "attention_few.h"

namespace mlxrocm {

int launch_attention_few_f16(const AttentionArgs& a, hipStream_t s) {
  return launch_few_typed<f16_t>(a, s);
}

} // namespace mlxrocm

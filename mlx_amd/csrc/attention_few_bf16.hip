// attention_few_bf16.hip -- the kernels of attention_few.h for bfloat16
#include "attention_few.h"

namespace mlxrocm {

int launch_attention_few_bf16(const AttentionArgs& a, hipStream_t s) {
  return launch_few_typed<bf16_t>(a, s);
}

} // namespace mlxrocm

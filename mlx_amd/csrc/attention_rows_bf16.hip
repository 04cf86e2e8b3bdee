// attention_rows_bf16.hip -- the kernels of attention_rows.h for bfloat16
#include "attention_rows.h"

namespace mlxrocm {

int launch_attention_rows_bf16(const AttentionArgs& a, hipStream_t s) {
  return launch_rows_typed<bf16_t>(a, s);
}

} // namespace mlxrocm

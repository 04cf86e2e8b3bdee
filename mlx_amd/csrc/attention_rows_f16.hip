// attention_rows_f16.hip -- the kernels of attention_rows.h for float16
#include "attention_rows.h"

namespace mlxrocm {

int launch_attention_rows_f16(const AttentionArgs& a, hipStream_t s) {
  return launch_rows_typed<f16_t>(a, s);
}

} // namespace mlxrocm

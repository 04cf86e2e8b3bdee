// attention_rows_f32.hip -- the kernels of attention_rows.h for float32
#include "attention_rows.h"

namespace mlxrocm {

int launch_attention_rows_f32(const AttentionArgs& a, hipStream_t s) {
  return launch_rows_typed<float>(a, s);
}

} // namespace mlxrocm

// attention_join.hip -- joins what several workgroups have of the same rows, each over a run of
// the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, m = max_s m_s.
#include "attention.h"

namespace mlxrocm {

namespace {

// A row has `width` threads (a power of two), four columns each.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionArgs a, int width) {
  const int R = a.G * a.Lq;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * R;
  const int64_t n =
      static_cast<int64_t>(blockIdx.x) * (256 / width) + static_cast<int>(threadIdx.x) / width;
  if (n >= rows) {
    return;
  }
  const int d = 4 * (static_cast<int>(threadIdx.x) % width);
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) {
    top = fmaxf(top, a.part_ml[s * rows + n].x);
  }
  const float less = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  floatx4 sum = {};
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.part_ml[s * rows + n];
    const float by = ml.x == less ? 1.0f : __builtin_amdgcn_exp2f(ml.x - less);
    if (by != 0.0f || ml.y != ml.y) { // a run that saw nothing has nothing
      total = fmaf(by, ml.y, total);
      if (d < a.D) {
        const float4 v = *reinterpret_cast<const float4*>(a.part_out + (s * rows + n) * a.D + d);
        sum += by * floatx4{v.x, v.y, v.z, v.w};
      }
    }
  }
  const int head = static_cast<int>(n / R);
  const int row = static_cast<int>(n - static_cast<int64_t>(head) * R);
  const int b = head / a.Hkv;
  const int hk = head - b * a.Hkv;
  const int i = row / a.G;
  const bool seeing = length_of(a, b) - a.Lq + i >= 0;
  const float over = total == 0.0f || !seeing ? 0.0f : 1.0f / total;
  if (d < a.D) {
    T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.G, row) + d;
    store4<T>(out, seeing ? sum * over : floatx4{});
  }
  if (a.lse != nullptr && d == 0) {
    a.lse[(static_cast<int64_t>(b) * a.Hq + hk * a.G + row - i * a.G) * a.Lq + i] =
        seeing ? top + log2f(total) : 0.0f;
  }
}

} // namespace

int launch_attention_join(const AttentionArgs& a, int dtype, hipStream_t s) {
  MLXROCM_REHEARSE("attention_join");
  const int width = a.D <= 64 ? 16 : a.D <= 128 ? 32 : 64;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Lq;
  const unsigned grid = static_cast<unsigned>((rows + 256 / width - 1) / (256 / width));
  return dispatch_dtype(dtype, [&](auto t) {
    attention_join_kernel<decltype(t)><<<grid, 256, 0, s>>>(a, width);
    MLXROCM_HIP_TRY(hipGetLastError());
    return static_cast<int>(MLXROCM_OK);
  });
}

} // namespace mlxrocm

// attention_join.hip -- joins what several workgroups have of the same rows, each over a run of
// the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, m = max_s m_s.
//
// A row is joined by WAVES waves.  A lane has the maximum and sum of one run (there are at most
// 64), so the weights of all runs are there after one load; lanes add up the runs, four
// columns each and 64 WAVES / WIDTH runs at a time, whose loads do not wait for the weights.
// Few rows of many runs take a workgroup each, many rows a wave each.  (28 rows of 64 runs:
// one run behind the other 45 us, a wave for a row 13.7, a workgroup for a row 5.8, its loads
// ahead of the weights 3.8.)
#include "attention.h"

#include <algorithm>

namespace mlxrocm {

namespace {

// 2^(m_s - m): not zero, so that an infinite o_s stays infinite
__device__ __forceinline__ float weight_of(float part, float top) {
  return part == top ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(part - top), 0x1p-126f);
}

// WIDTH lanes have the columns of a run
template <typename T, int WIDTH, int WAVES>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionArgs a) {
  constexpr int kAtOnce = 64 / WIDTH * WAVES;
  __shared__ floatx4 sums[WAVES > 1 ? WAVES : 1][WIDTH];
  const int R = a.G * a.Lq;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * R; // (less than 2^26)
  const int wave = threadIdx.x >> 6;
  const int n = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  if (n >= rows) {
    return; // (whole waves; with WAVES > 1 none)
  }
  const int lane = threadIdx.x & 63;
  const float2 ml =
      lane < a.splits ? a.part_ml[lane * rows + n] : make_float2(-INFINITY, 0.0f);
  // the columns of 64 runs, or as many as eight loads have, are on their way with the weights
  constexpr int kFirst = 64 / kAtOnce < 8 ? 64 / kAtOnce : 8;
  const int d = 4 * (lane % WIDTH);
  const float* part = a.part_out + static_cast<int64_t>(n) * a.D + (d < a.D ? d : 0);
  const int own = (WAVES > 1 ? wave * (64 / WIDTH) : 0) + lane / WIDTH;
  const auto load = [&](int s) {
    return *reinterpret_cast<const float4*>(part + min(s, a.splits - 1) * rows * a.D);
  };
  float4 first[kFirst] = {};
#pragma unroll
  for (int x = 0; x < kFirst; ++x) {
    if (x * kAtOnce < a.splits) {
      first[x] = load(x * kAtOnce + own);
    }
  }
  const int head = n / R;
  const int row = n - head * R;
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
  const int i = a.of_G.divide(row);
  const bool seeing = length_of(a, b) - a.Lq + i >= 0;
  const float top = max_lanes(ml.x);
  const float less = top == -INFINITY ? 0.0f : top;
  // a run that saw nothing has nothing
  const bool has = !(ml.y == 0.0f);
  const float by = has ? weight_of(ml.x, less) : 0.0f;
  const float total = sum_lanes(by * ml.y);
  floatx4 sum = {};
  const auto add = [&](int s, const float4& v) {
    const float w = __shfl(by, s & 63, 64);
    if (s < a.splits && w != 0.0f) {
      sum += w * floatx4{v.x, v.y, v.z, v.w};
    }
  };
#pragma unroll
  for (int x = 0; x < kFirst; ++x) {
    add(x * kAtOnce + own, first[x]);
  }
#pragma unroll 8
  for (int s0 = kFirst * kAtOnce; s0 < a.splits; s0 += kAtOnce) {
    add(s0 + own, load(s0 + own));
  }
  if constexpr (WIDTH <= 32) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      sum[x] = WIDTH == 16 ? sum_quarters(sum[x]) : sum_halves(sum[x]);
    }
  }
  if constexpr (WAVES > 1) {
    if (lane < WIDTH) {
      sums[wave][lane] = sum;
    }
    __syncthreads();
    if (wave != 0) {
      return;
    }
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      sum += sums[w][lane % WIDTH];
    }
  }
  const float over = total == 0.0f ? 0.0f : 1.0f / total;
  if (lane < WIDTH && d < a.D) {
    T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, row) + d;
    T* low = low_of<T>(a, lse_at(a, b, hk, row));
    store_result<T>(out, low == nullptr ? nullptr : low + d, seeing ? sum * over : floatx4{});
  }
  if (a.lse != nullptr && lane == 0) {
    a.lse[lse_at(a, b, hk, row)] = seeing ? top + log2f(total) : 0.0f;
  }
}

// The same for two to four runs of many rows: a thread has four columns.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_few_kernel(const AttentionArgs a) {
  const int R = a.G * a.Lq;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * R;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = at / (a.D / 4);
  const int d = static_cast<int>(at - n * (a.D / 4)) * 4;
  if (n >= rows) {
    return;
  }
  float2 ml[4];
  floatx4 x[4];
  float top = -INFINITY;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t from = min(s, a.splits - 1) * rows + n;
    const float4 v = *reinterpret_cast<const float4*>(a.part_out + from * a.D + d);
    x[s] = floatx4{v.x, v.y, v.z, v.w};
    ml[s] = s < a.splits ? a.part_ml[from] : make_float2(-INFINITY, 0.0f);
    top = fmaxf(top, ml[s].x);
  }
  const float less = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  floatx4 sum = {};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if (!(ml[s].y == 0.0f)) {
      const float by = weight_of(ml[s].x, less);
      total = fmaf(by, ml[s].y, total);
      sum += by * x[s];
    }
  }
  const int head = static_cast<int>(n / R);
  const int row = static_cast<int>(n - static_cast<int64_t>(head) * R);
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
  const int i = a.of_G.divide(row);
  const bool seeing = length_of(a, b) - a.Lq + i >= 0;
  const float over = total == 0.0f ? 0.0f : 1.0f / total;
  T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, row) + d;
  T* low = low_of<T>(a, lse_at(a, b, hk, row));
  store_result<T>(out, low == nullptr ? nullptr : low + d, seeing ? sum * over : floatx4{});
  if (a.lse != nullptr && d == 0) {
    a.lse[lse_at(a, b, hk, row)] = seeing ? top + log2f(total) : 0.0f;
  }
}

// Sums of partial gradients: a thread has four columns of a row of dq, or of a key's dk or dv.
template <typename T>
__global__ __launch_bounds__(256) void attention_sum_dq_kernel(const AttentionGradArgs g) {
  const AttentionArgs& a = g.a;
  const int R = a.G * a.Lq;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * R;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = at / (a.D / 4);
  const int d = static_cast<int>(at - n * (a.D / 4)) * 4;
  if (n >= rows) {
    return;
  }
  floatx4 sum = {};
#pragma unroll 4
  for (int s = 0; s < g.plan.dq_splits.d; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(g.part_dq + (s * rows + n) * a.D + d);
    sum += floatx4{v.x, v.y, v.z, v.w};
  }
  const int head = static_cast<int>(n / R);
  const int row = static_cast<int>(n - static_cast<int64_t>(head) * R);
  const int b = head / a.Hkv;
  T* to = static_cast<T*>(g.dq) + row_offset(g.dq_strides, b, head - b * a.Hkv, a.of_G, row) + d;
  store4<T>(to, sum * g.scale);
}

template <typename T>
__global__ __launch_bounds__(256) void attention_sum_dkv_kernel(const AttentionGradArgs g, int keys) {
  const AttentionArgs& a = g.a;
  const GradPlan& plan = g.plan;
  const int each = 2 * a.D / 4; // of a key
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = at / each;
  if (n >= static_cast<int64_t>(a.B) * a.Hkv * keys) {
    return;
  }
  const int c = static_cast<int>(at - n * each) * 4; // column of dk, then of dv
  const int head = static_cast<int>(n / keys);
  const int key = static_cast<int>(n - static_cast<int64_t>(head) * keys);
  const int block = key / kGradBlock;
  const bool wide = block < plan.wide_blocks;
  const int splits = wide ? plan.wide_splits.d : plan.splits.d;
  if (splits == 1) {
    return; // (whole already)
  }
  const int piece = wide ? block * splits
                         : plan.wide_blocks * plan.wide_splits.d + (block - plan.wide_blocks) * splits;
  const float* part = g.part_dkv +
      (static_cast<int64_t>(head) * plan.part_pieces() + piece) * (kGradBlock * 2 * a.D) +
      (key - block * kGradBlock) * 2 * a.D + c;
  floatx4 sum = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(
        part + static_cast<int64_t>(s) * (kGradBlock * 2 * a.D));
    sum += floatx4{v.x, v.y, v.z, v.w};
  }
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
  const bool of_k = c < a.D;
  const int64_t* strides = of_k ? g.dk_strides : g.dv_strides;
  T* to = static_cast<T*>(of_k ? g.dk : g.dv) + b * strides[0] + hk * strides[1] +
      key * strides[2] + (of_k ? c : c - a.D);
  store4<T>(to, of_k ? sum * g.scale : sum);
}

} // namespace

int launch_attention_grad_join(const AttentionGradArgs& g, int dtype, hipStream_t s) {
  const AttentionArgs& a = g.a;
  MLXROCM_REHEARSE("attention_sum");
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (g.plan.dq_splits.d > 1) {
      const int64_t n = static_cast<int64_t>(a.B) * a.Hq * a.Lq * (a.D / 4);
      attention_sum_dq_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(g);
      MLXROCM_HIP_TRY(hipGetLastError());
    }
    if (g.plan.dkv_split()) {
      // (only the blocks of kept keys, if the others are not cut)
      const int keys =
          g.plan.splits.d > 1 ? a.keys : std::min(a.keys, g.plan.wide_blocks * kGradBlock);
      const int64_t n = static_cast<int64_t>(a.B) * a.Hkv * keys * (a.D / 2);
      attention_sum_dkv_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(g, keys);
      MLXROCM_HIP_TRY(hipGetLastError());
    }
    return static_cast<int>(MLXROCM_OK);
  });
}

namespace {

template <typename T, int WIDTH>
void launch_join_of(const AttentionArgs& a, int64_t rows, hipStream_t s) {
  if (rows <= 2048) {
    attention_join_kernel<T, WIDTH, 4><<<static_cast<unsigned>(rows), 256, 0, s>>>(a);
  } else {
    attention_join_kernel<T, WIDTH, 1><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, s>>>(a);
  }
}

} // namespace

int launch_attention_join(const AttentionArgs& a, int dtype, hipStream_t s) {
  MLXROCM_REHEARSE("attention_join");
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Lq;
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.splits <= 4) {
      const int64_t n = rows * (a.D / 4);
      attention_join_few_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(a);
    } else if (a.D <= 64) {
      launch_join_of<T, 16>(a, rows, s);
    } else if (a.D <= 128) {
      launch_join_of<T, 32>(a, rows, s);
    } else {
      launch_join_of<T, 64>(a, rows, s);
    }
    MLXROCM_HIP_TRY(hipGetLastError());
    return static_cast<int>(MLXROCM_OK);
  });
}

} // namespace mlxrocm

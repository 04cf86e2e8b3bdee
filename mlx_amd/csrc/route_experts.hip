// route_experts.hip -- the experts of each token and their weights, and the gradient of the logits.
//
// Of a row's logits l: scores s = softmax(l) or sigmoid(l); choice c = s + bias; the experts lie in
// groups of equal size, of which those with the largest sum of their `group_best` largest
// choices stay; of the experts there the k with the largest choices are chosen, in that order, the
// lowest index first where they are equal.  Weights w = scale s, or scale s / (sum of the chosen s).
//
// Choices decide what is computed, so their order is taken exactly: of the logits themselves where
// they have the scores' order (no bias, no sums), else of choices formed in 64 bits.  Compared are
// integers of the floats' order, with room below the lowest for what is taken already.
//
// What bounds it: the instructions of k searches for the largest.  Sixteen lanes have a row, one of
// the rows of lanes that DPP instructions rotate within: the largest of sixteen lanes is four
// instructions, for four rows of a wavefront at once.  A lane holds neighbouring experts of one
// group, so that the lowest lane that has the largest value has the lowest index.
#include "common.h"

namespace mlxrocm {

namespace {

constexpr int kLanes = 16; // of a row
constexpr int kRows = 16;  // of a workgroup: 256 threads
constexpr int kMostChosen = 32;
constexpr int kMostExperts = 1024;

struct RouteArgs {
  const void* logits;
  const float* bias; // or null
  int32_t* indices;
  void* weights;
  // gradients
  const void* grad;
  void* out;
  int64_t rows, stride, grad_stride;
  int experts, k, groups, top_groups, group_best;
  int group_size;
  int group_lanes; // lanes of a group, a power of two
  int sigmoid, normalize, vector;
  float scale;
};

// ---- sixteen lanes ----
template <int Rotate>
__device__ __forceinline__ int rotated(int v) {
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + Rotate, 0xf, 0xf, false); // row_ror
}
template <int Rotate>
__device__ __forceinline__ int64_t rotated(int64_t v) {
  const uint32_t lo = rotated<Rotate>(static_cast<int>(v));
  const uint32_t hi = rotated<Rotate>(static_cast<int>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
template <int Rotate>
__device__ __forceinline__ float rotated(float v) {
  return __int_as_float(rotated<Rotate>(__float_as_int(v)));
}
template <typename K>
__device__ __forceinline__ K largest16(K v) {
  v = max(v, rotated<8>(v));
  v = max(v, rotated<4>(v));
  v = max(v, rotated<2>(v));
  return max(v, rotated<1>(v));
}
__device__ __forceinline__ float largest16(float v) {
  v = fmaxf(v, rotated<8>(v));
  v = fmaxf(v, rotated<4>(v));
  v = fmaxf(v, rotated<2>(v));
  return fmaxf(v, rotated<1>(v));
}
// (the same in every lane: the order of the sum is a lane's own, rotated, but every step adds
// two sums of which each has the other's other half)
__device__ __forceinline__ float sum16(float v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  return v + rotated<1>(v);
}
// The lowest of the sixteen lanes where `is`
__device__ __forceinline__ int first16(bool is) {
  const uint64_t lanes = __ballot(is);
  const uint32_t mine = static_cast<uint32_t>(lanes >> (threadIdx.x & 48)) & 0xffffu;
  return __ffs(static_cast<int>(mine)) - 1;
}

// ---- integers in the order of floats; NaN is the lowest, as -inf is ----
__device__ __forceinline__ int key_of(float v) {
  const int bits = __float_as_int(v + 0.0f); // (-0 becomes 0)
  const int key = bits ^ ((bits >> 31) & 0x7fffffff);
  return v != v ? static_cast<int>(0x807fffff) : key;
}
__device__ __forceinline__ int64_t key_of(double v) {
  const int64_t bits = __double_as_longlong(v + 0.0);
  const int64_t key = bits ^ ((bits >> 63) & 0x7fffffffffffffffLL);
  return v != v ? static_cast<int64_t>(0x800fffffffffffffULL) : key;
}
__device__ __forceinline__ float value_of(int key) {
  return __int_as_float(key ^ ((key >> 31) & 0x7fffffff));
}
__device__ __forceinline__ double value_of(int64_t key) {
  return __longlong_as_double(key ^ ((key >> 63) & 0x7fffffffffffffffLL));
}
template <typename K>
struct Lowest;
template <>
struct Lowest<int> {
  using Value = float;
  static constexpr int taken = static_cast<int>(0x80000000u);
};
template <>
struct Lowest<int64_t> {
  using Value = double;
  static constexpr int64_t taken = static_cast<int64_t>(0x8000000000000000ULL);
};

// e^(l - m) of the largest logit m: 1 where they are equal (both may be infinite), and nothing
// where there is no logit at all
__device__ __forceinline__ float above(float l, float m) {
  return m == -INFINITY ? (l != l ? l : 0.0f) : l == m ? 1.0f : expf(l - m);
}

// Of the logits of a lane, V of a group's neighbours, those that exist: 0 .. n - 1
template <typename T, int V>
__device__ __forceinline__ void read_logits(const T* p, int n, int vector, float (&l)[V]) {
  constexpr int kWide = 16 / sizeof(T);
  if (V % kWide == 0 && vector && n == V) {
    if constexpr (V % kWide == 0) {
#pragma unroll
      for (int j = 0; j < V; j += kWide) {
        union {
          uint4 u;
          T e[kWide];
        } raw;
        raw.u = *reinterpret_cast<const uint4*>(p + j);
#pragma unroll
        for (int i = 0; i < kWide; ++i) {
          l[j + i] = to_f32(raw.e[i]);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    l[j] = j < n ? to_f32(p[j]) : -INFINITY;
  }
}

struct Place { // of a lane in its row
  int lane, group, first, n; // experts first .. first + n - 1 of the row
};
template <int V>
__device__ __forceinline__ Place place_of(const RouteArgs& a) {
  Place p;
  p.lane = threadIdx.x & 15;
  p.group = p.lane / a.group_lanes;
  const int at = (p.lane & (a.group_lanes - 1)) * V;
  p.first = p.group * a.group_size + at;
  p.n = p.group < a.groups ? min(V, max(0, a.group_size - at)) : 0;
  return p;
}

// Takes the largest of the row out of `keys` and says where it was: its key, and in the lane that
// had it (the others -1) which of its values.
template <int V, typename K>
__device__ __forceinline__ K take(K (&keys)[V], int* which) {
  K best = keys[0];
#pragma unroll
  for (int j = 1; j < V; ++j) {
    best = max(best, keys[j]);
  }
  const K all = largest16(best);
  const bool mine = first16(best == all) == (threadIdx.x & 15);
  int at = -1;
#pragma unroll
  for (int j = V - 1; j >= 0; --j) {
    at = mine && keys[j] == all ? j : at;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    keys[j] = at == j ? Lowest<K>::taken : keys[j];
  }
  *which = at;
  return all;
}

// Leaves the groups that count
template <int V, typename K>
__device__ __forceinline__ void keep_groups(const RouteArgs& a, const Place& p, K (&keys)[V]) {
  using F = typename Lowest<K>::Value;
  // the largest, and the second largest, of the lane's; then of the group's lanes
  K one = Lowest<K>::taken;
  K two = Lowest<K>::taken;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    two = max(two, min(one, keys[j]));
    one = max(one, keys[j]);
  }
  for (int d = 1; d < a.group_lanes; d *= 2) {
    const K other = __shfl_xor(one, d, 64);
    const K other_two = __shfl_xor(two, d, 64);
    two = max(max(two, other_two), min(one, other));
    one = max(one, other);
  }
  K mark = one;
  if (a.group_best == 2) {
    mark = key_of(value_of(one) + value_of(two));
  }
  mark = p.group < a.groups ? mark : Lowest<K>::taken;
  bool stays = false;
  for (int n = 0; n < a.top_groups; ++n) {
    const K best = largest16(mark);
    const int lane = first16(mark == best);
    const bool mine = lane / a.group_lanes == p.group;
    stays |= mine;
    mark = mine ? Lowest<K>::taken : mark;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    keys[j] = stays ? keys[j] : Lowest<K>::taken;
  }
}

struct Chosen {
  int index;
  float logit;
};

template <typename T, int V, bool kSums>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  using K = std::conditional_t<kSums, int64_t, int>;
  __shared__ Chosen chosen[kRows][kMostChosen];
  const int slot = threadIdx.x / kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
  const int64_t at = min(row, a.rows - 1); // (sixteen lanes work or not together; all vote)
  const T* logits = static_cast<const T*>(a.logits) + at * a.stride;
  const Place p = place_of<V>(a);
  float l[V];
  read_logits<T, V>(logits + p.first, p.n, a.vector, l);

  // softmax: the largest logit and the sum above it
  float most = -INFINITY;
  float total = 0.0f;
  if (!a.sigmoid && (kSums || !a.normalize)) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      most = fmaxf(most, l[j]);
    }
    most = largest16(most);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      total += j < p.n ? above(l[j], most) : 0.0f;
    }
    total = sum16(total);
  }

  K keys[V];
  if constexpr (kSums) {
    double sum = 0.0;
    double s[V];
    if (!a.sigmoid) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] = l[j] == -INFINITY ? 0.0
            : l[j] == most       ? 1.0
                                 : exp(static_cast<double>(l[j]) - static_cast<double>(most));
        sum += s[j];
      }
      for (int d = 1; d < kLanes; d *= 2) {
        sum += __shfl_xor(sum, d, 64);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      double c = a.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l[j]))) : s[j] / sum;
      if (a.bias != nullptr && j < p.n) {
        c += static_cast<double>(a.bias[p.first + j]);
      }
      c = l[j] == -INFINITY ? -static_cast<double>(INFINITY) : c;
      keys[j] = j < p.n ? key_of(c) : Lowest<K>::taken;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      keys[j] = j < p.n ? key_of(l[j]) : Lowest<K>::taken;
    }
  }
  if (a.top_groups < a.groups) {
    keep_groups<V, K>(a, p, keys);
  }
  for (int n = 0; n < a.k; ++n) {
    int which;
    take<V, K>(keys, &which);
    if (which >= 0) {
      float logit = l[0];
#pragma unroll
      for (int j = 1; j < V; ++j) {
        logit = which == j ? l[j] : logit;
      }
      chosen[slot][n] = {p.first + which, logit};
    }
  }
  __syncthreads();
  if (row >= a.rows) {
    return;
  }

  // each of the sixteen lanes has two of the chosen at most
  float s[2];
  float low = 0.0f; // sigmoid: all counted up, where all are tiny
  Chosen c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool is = p.lane + 16 * i < a.k;
    c[i] = chosen[slot][is ? p.lane + 16 * i : 0];
    if (!is) {
      c[i].logit = -INFINITY;
    }
  }
  if (a.normalize) {
    if (a.sigmoid) {
      low = largest16(fmaxf(fminf(c[0].logit, 0.0f), fminf(c[1].logit, 0.0f)));
      low = low == -INFINITY ? 0.0f : low;
    } else {
      most = largest16(fmaxf(c[0].logit, c[1].logit));
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = a.sigmoid
        ? expf(fminf(c[i].logit, 0.0f) - low) / (1.0f + expf(-fabsf(c[i].logit)))
        : above(c[i].logit, most);
    s[i] = c[i].logit != c[i].logit ? c[i].logit : s[i];
    s[i] = p.lane + 16 * i < a.k ? s[i] : 0.0f;
  }
  if (a.normalize) {
    total = sum16(s[0] + s[1]);
  } else if (a.sigmoid) {
    total = 1.0f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (p.lane + 16 * i < a.k) {
      const int64_t to = row * a.k + p.lane + 16 * i;
      a.indices[to] = c[i].index;
      const float w = total == 0.0f ? 0.0f : s[i] / total * a.scale;
      static_cast<T*>(a.weights)[to] = from_f32<T>(w);
    }
  }
}

// The gradient of the logits from that of the weights.  With r = s / (sum of the chosen s) and g =
// scale grad: normalised, g' = g - sum(g r) for the chosen, times r (softmax) or r (1 - s)
// (sigmoid); else s (g - sum(g s)) for all experts (softmax; g is 0 for those not chosen) or
// g s (1 - s) for the chosen (sigmoid).
template <typename T, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(const RouteArgs a) {
  extern __shared__ float by_expert[]; // [kRows][experts]: of the chosen g s; then the gradients
  const int slot = threadIdx.x / kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
  const int64_t at = min(row, a.rows - 1);
  const T* logits = static_cast<const T*>(a.logits) + at * a.stride;
  const T* grad = static_cast<const T*>(a.grad) + at * a.grad_stride;
  float* mine = by_expert + slot * a.experts;
  const Place p = place_of<V>(a);
  const bool dense = !a.sigmoid && !a.normalize;
  float l[V];
  float most = -INFINITY;
  float total = 1.0f;
  if (dense) {
    read_logits<T, V>(logits + p.first, p.n, a.vector, l);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      most = fmaxf(most, l[j]);
    }
    most = largest16(most);
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      l[j] = j < p.n ? above(l[j], most) : 0.0f;
      total += l[j];
    }
    total = sum16(total);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j < p.n) {
      mine[p.first + j] = 0.0f;
    }
  }
  int index[2];
  bool has[2];
  float g[2];
  float x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool is = p.lane + 16 * i < a.k;
    index[i] = is ? a.indices[at * a.k + p.lane + 16 * i] : -1;
    has[i] = static_cast<uint32_t>(index[i]) < static_cast<uint32_t>(a.experts);
    g[i] = has[i] ? to_f32(grad[p.lane + 16 * i]) * a.scale : 0.0f;
    x[i] = has[i] ? to_f32(logits[index[i]]) : -INFINITY;
  }
  float low = 0.0f;
  if (a.normalize) {
    if (a.sigmoid) {
      low = largest16(fmaxf(fminf(x[0], 0.0f), fminf(x[1], 0.0f)));
      low = low == -INFINITY ? 0.0f : low;
    } else {
      most = largest16(fmaxf(x[0], x[1]));
    }
  }
  float s[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = a.sigmoid ? expf(fminf(x[i], 0.0f) - low) / (1.0f + expf(-fabsf(x[i])))
                     : above(x[i], most);
    s[i] = x[i] != x[i] ? x[i] : s[i];
    s[i] = has[i] ? s[i] : 0.0f;
  }
  if (a.normalize) {
    total = sum16(s[0] + s[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = total == 0.0f ? 0.0f : s[i] / total;
  }
  const float dot = a.sigmoid && !a.normalize ? 0.0f : sum16(g[0] * s[0] + g[1] * s[1]);
  __syncthreads(); // (the zeros are other lanes')
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (has[i]) {
      // 1 - sigmoid(x) without cancellation
      const float rest = !a.sigmoid ? 1.0f : 1.0f / (1.0f + expf(x[i]));
      mine[index[i]] = dense ? g[i] * s[i] : (g[i] - dot) * s[i] * rest;
    }
  }
  __syncthreads();
  if (row >= a.rows) {
    return;
  }
  T* out = static_cast<T*>(a.out) + row * a.experts + p.first;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j < p.n) {
      float v = mine[p.first + j];
      if (dense) {
        v -= total == 0.0f ? 0.0f : l[j] / total * dot;
      }
      out[j] = from_f32<T>(v);
    }
  }
}

int check(
    const char* tag, RouteArgs& a, int64_t rows, int experts, int k, int groups, int top_groups,
    int group_best, int dtype) {
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] unknown dtype %d", tag, dtype);
  }
  if (rows < 0 || experts < 1 || experts > kMostExperts) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %lld rows of %d experts", tag,
        static_cast<long long>(rows), experts);
  }
  if (groups < 1 || groups > kLanes || experts % groups != 0 || top_groups < 1 ||
      top_groups > groups || group_best < 1 || group_best > 2) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d of %d groups of %d experts by their best %d", tag,
        top_groups, groups, experts, group_best);
  }
  a.group_size = experts / groups;
  if (k < 1 || k > kMostChosen || k > top_groups * a.group_size || group_best > a.group_size) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d of %d experts", tag, k, top_groups * a.group_size);
  }
  if (rows > (int64_t{1} << 24) * kRows - kRows) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", tag); // 2^32 threads
  }
  a.rows = rows;
  a.experts = experts;
  a.k = k;
  a.groups = groups;
  a.top_groups = top_groups;
  a.group_best = group_best;
  a.group_lanes = kLanes;
  while (a.group_lanes * groups > kLanes) {
    a.group_lanes /= 2;
  }
  return MLXROCM_OK;
}

// The smallest power of two of values for a lane
template <typename F>
int by_values(const RouteArgs& a, F&& go) {
  const int v = (a.group_size + a.group_lanes - 1) / a.group_lanes;
  v <= 1 ? go(IntC<1>{})
      : v <= 2  ? go(IntC<2>{})
      : v <= 4  ? go(IntC<4>{})
      : v <= 8  ? go(IntC<8>{})
      : v <= 16 ? go(IntC<16>{})
      : v <= 32 ? go(IntC<32>{})
                : go(IntC<64>{});
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

bool wide_rows(const void* p, int64_t stride, int group_size, size_t size) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride * size) |
          static_cast<uintptr_t>(group_size * size)) % 16 == 0;
}

} // namespace

} // namespace mlxrocm

extern "C" int mlxrocm_route_experts(
    const void* logits,
    const float* bias,
    int32_t* indices,
    void* weights,
    int64_t rows,
    int64_t stride,
    int experts,
    int k,
    int sigmoid,
    int groups,
    int top_groups,
    int group_best,
    int normalize,
    float scale,
    int dtype,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_route_experts");
  using namespace mlxrocm;
  RouteArgs a{};
  const int rc =
      check("route_experts", a, rows, experts, k, groups, top_groups, group_best, dtype);
  if (rc != MLXROCM_OK || rows == 0) {
    return rc;
  }
  if (logits == nullptr || indices == nullptr || weights == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[route_experts] null pointer");
  }
  a.logits = logits;
  a.bias = bias;
  a.indices = indices;
  a.weights = weights;
  a.stride = stride;
  a.sigmoid = sigmoid;
  a.normalize = normalize;
  a.scale = scale;
  a.vector = wide_rows(logits, stride, a.group_size, dtype_size(dtype));
  const bool sums = bias != nullptr || (group_best > 1 && top_groups < groups);
  const unsigned grid = static_cast<unsigned>((rows + kRows - 1) / kRows);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_values(a, [&](auto v) {
      if (sums) {
        route_kernel<T, decltype(v)::value, true>
            <<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
      } else {
        route_kernel<T, decltype(v)::value, false>
            <<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
      }
    });
  });
}

extern "C" int mlxrocm_route_experts_vjp(
    const void* logits,
    const int32_t* indices,
    const void* grad,
    void* out,
    int64_t rows,
    int64_t stride,
    int64_t grad_stride,
    int experts,
    int k,
    int sigmoid,
    int normalize,
    float scale,
    int dtype,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_route_experts_vjp");
  using namespace mlxrocm;
  RouteArgs a{};
  const int rc = check("route_experts_vjp", a, rows, experts, k, 1, 1, 1, dtype);
  if (rc != MLXROCM_OK || rows == 0) {
    return rc;
  }
  if (logits == nullptr || indices == nullptr || grad == nullptr || out == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[route_experts_vjp] null pointer");
  }
  a.logits = logits;
  a.indices = const_cast<int32_t*>(indices);
  a.grad = grad;
  a.out = out;
  a.stride = stride;
  a.grad_stride = grad_stride;
  a.sigmoid = sigmoid;
  a.normalize = normalize;
  a.scale = scale;
  a.vector = wide_rows(logits, stride, a.group_size, dtype_size(dtype));
  const unsigned grid = static_cast<unsigned>((rows + kRows - 1) / kRows);
  const size_t lds = sizeof(float) * kRows * experts;
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_values(a, [&](auto v) {
      route_grad_kernel<T, decltype(v)::value>
          <<<grid, 256, lds, static_cast<hipStream_t>(stream)>>>(a);
    });
  });
}

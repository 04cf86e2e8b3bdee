// route_experts.hip -- the experts of each token and their weights, and the gradient of the logits.
//
// Of a row's logits l: scores s = softmax(l) or sigmoid(l); choice c = s + bias; the experts lie in
// groups of equal size, of which those with the largest sum of their `group_best` largest
// choices stay; of the experts there the k with the largest choices are chosen, in that order, the
// lowest index first where they are equal.  Weights w = scale s, or scale s / (sum of the chosen s).
//
// Choices decide what is computed, so their order is taken exactly: of the logits themselves where
// they have the scores' order (no bias, no sums), else of choices in 64 bits.  Those are formed in 32
// bits first; where all that are chosen, and the first that is not, are further apart than 32 bits can be
// off, the order is known, and only a wavefront with a row where they are not forms them in 64.  Compared
// are integers of the floats' order, with room below the lowest for what is taken already.
//
// What bounds it: the instructions of k searches for the largest.  Sixteen lanes have a row, one of
// the rows of lanes that DPP instructions rotate within: the largest of sixteen lanes is four
// instructions, for four rows of a wavefront at once.  A lane holds neighbouring experts of one
// group, so that the lowest lane that has the largest value has the lowest index.
#include <type_traits>

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
  int sigmoid, normalize;
  int full; // whether every lane has V experts
  int vector, wide_out, wide_bias; // whether rows of logits, their gradient, bias are aligned (kWide)
  float scale;
};

// ---- sixteen lanes ----
template <int Rotate>
__device__ __forceinline__ int rotated(int v) {
  return __builtin_amdgcn_mov_dpp(v, 0x120 + Rotate, 0xf, 0xf, true); // row_ror
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
// below every value's: what has been taken (in 32 steps), what does not exist
template <>
struct Lowest<int> {
  static constexpr int taken = static_cast<int>(0x80000000u);
  static constexpr int none = taken + 64;
  static constexpr int least = static_cast<int>(0x807fffffu); // -inf
};
template <>
struct Lowest<int64_t> {
  static constexpr int64_t taken = static_cast<int64_t>(0x8000000000000000ULL);
  static constexpr int64_t none = taken + 64;
};

// e^(l - m) of the largest logit m: 1 where they are equal (both may be infinite).  Where there is no
// logit at all (-inf) m is 0, so that nothing is above it.
__device__ __forceinline__ float base_of(float most) {
  return most == -INFINITY ? 0.0f : most;
}
__device__ __forceinline__ float above(float l, float m) {
  return expf(l == m ? 0.0f : l - m);
}

// V of a group's neighbours in a lane are read and written W at a time where all rows allow it
template <typename T, int V>
constexpr int kWide = V * sizeof(T) <= 16 ? V : 16 / sizeof(T);
template <typename T, int W>
struct alignas(W * sizeof(T)) Wide {
  T e[W];
};

// Those that exist: 0 .. n - 1
template <typename T, int V>
__device__ __forceinline__ void read_logits(const T* p, int n, int vector, float (&l)[V]) {
  constexpr int W = kWide<T, V>;
  if (vector && n == V) {
#pragma unroll
    for (int j = 0; j < V; j += W) {
      const Wide<T, W> raw = *reinterpret_cast<const Wide<T, W>*>(p + j);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        l[j + i] = to_f32(raw.e[i]);
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

// In which step it was taken, kMostChosen: in none
template <typename K>
__device__ __forceinline__ int step_of(K key) {
  return key < Lowest<K>::none ? static_cast<int>(key - Lowest<K>::taken) : kMostChosen;
}

// Takes the k largest of a row out of `keys`, lowest index first of equal ones, and leaves
// Lowest::taken + n in the place of the n-th
template <int V, typename K>
__device__ __forceinline__ void take_in_order(int k, K (&keys)[V]) {
  for (int n = 0; n < k; ++n) {
    K best = keys[0];
#pragma unroll
    for (int j = 1; j < V; ++j) {
      best = max(best, keys[j]);
    }
    const K all = largest16(best);
    bool mine = first16(best == all) == (threadIdx.x & 15);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool is = mine && keys[j] == all;
      keys[j] = is ? Lowest<K>::taken + n : keys[j];
      mine = mine && !is;
    }
  }
}

// The same where no two are equal or, if `margin` is not negative, nearer to each other than
// margin (1 + the larger's size): false where two are, whose order this does not tell.  (Without
// the search for the lowest index: 44 instructions a choice of 16 values a lane instead of 100.)
template <int V>
__device__ __forceinline__ bool take(int k, float margin, int (&keys)[V]) {
  // (equal ones are taken in one step: they show in how many were)
  const auto taken = [&] {
    int count = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      count += keys[j] < Lowest<int>::none;
    }
    count += rotated<8>(count);
    count += rotated<4>(count);
    count += rotated<2>(count);
    return count + rotated<1>(count);
  };
  bool apart = true;
  float last = 0.0f;
  for (int n = 0;; ++n) {
    int best = keys[0];
#pragma unroll
    for (int j = 1; j < V; ++j) {
      best = max(best, keys[j]);
    }
    best = largest16(best);
    if (margin >= 0.0f) {
      const float v = value_of(best);
      // (none left: as far as can be.  Infinities and NaN are not apart.)
      apart = apart && (n == 0 || best < Lowest<int>::least || last - v > margin * (1.0f + fabsf(last)));
      last = v;
    }
    if (n == k) {
      return apart && taken() == k;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      keys[j] = keys[j] == best ? Lowest<int>::taken + n : keys[j];
    }
    if (margin < 0.0f && n + 1 == k) {
      return true;
    }
  }
}

// Leaves the groups that count; says whether the last that does and the first that does not are
// further than margin apart (if that is not negative)
template <int V, typename K>
__device__ __forceinline__ bool keep_groups(
    const RouteArgs& a, const Place& p, float margin, K (&keys)[V]) {
  // the largest, and the second largest, of the lane's; then of the group's lanes
  K one = Lowest<K>::none;
  K two = Lowest<K>::none;
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
  mark = p.group < a.groups ? mark : Lowest<K>::none;
  bool stays = false;
  K last = 0;
  for (int n = 0; n < a.top_groups; ++n) {
    last = largest16(mark);
    const bool mine = first16(mark == last) / a.group_lanes == p.group;
    stays |= mine;
    mark = mine ? Lowest<K>::none : mark;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    keys[j] = stays ? keys[j] : Lowest<K>::none;
  }
  if (margin < 0.0f) {
    return true;
  }
  const auto v = value_of(last);
  return v - value_of(largest16(mark)) > margin * (1 + fabs(v));
}

struct Chosen {
  int index;
  float logit;
};

template <typename T, int V, bool kSums>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
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
    most = base_of(largest16(most));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      total += above(l[j], most); // (what does not exist is -inf)
    }
    total = sum16(total);
  }
  float b[V];
  if (kSums && a.bias != nullptr) {
    read_logits<float, V>(a.bias + p.first, p.n, a.wide_bias, b);
  }

  int place[V]; // which choice a value is
  // Unique keys: a 16-bit logit leaves the lower 13 bits free, which tell the index, the lowest
  // the largest.  Else margins: logits need not be apart by more than nothing; choices in 32 bits are
  // off by 2^-21 and their rounding (sigmoid), by (V + 32) 2^-24 (softmax: sums of V values a lane,
  // of e^x with x off by its rounding): what is further apart than twice that has the order of 64 bits.
  constexpr bool kUnique = !kSums && sizeof(T) == 2;
  const float margin = kUnique ? -1.0f : !kSums ? 0.0f : a.sigmoid ? 0x1p-19f : (V + 32) * 0x1p-22f;
  const bool grouped = a.top_groups < a.groups;
  bool known = true;
  {
    int keys[V];
    if constexpr (kSums) {
      float c[V];
      if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -1.44269504f));
        }
      } else {
        const float by = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = above(l[j], most) * by;
        }
      }
      if (a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] += b[j];
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // (neither masked nor NaN; -0 is no sum)
        const int bits = __float_as_int(fmaxf(l[j] > -INFINITY ? c[j] : -INFINITY, -INFINITY));
        keys[j] = bits ^ ((bits >> 31) & 0x7fffffff);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        keys[j] = key_of(l[j]);
        if constexpr (kUnique) {
          keys[j] = (keys[j] & ~0x1fff) + 0x1000 + (kMostExperts - 1 - p.first - j);
        }
      }
    }
    if (!a.full) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        keys[j] = j < p.n ? keys[j] : Lowest<int>::none;
      }
    }
    if (grouped) {
      // (a group's mark may be a sum of two)
      known = keep_groups<V, int>(a, p, kSums ? 2.0f * margin : margin, keys);
    }
    known = take<V>(a.k, margin, keys) && known;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      place[j] = step_of(keys[j]);
    }
  }
  // (the sixteen lanes of a row agree)
  if (!kUnique && __any(!known)) {
    if constexpr (kSums) {
      int64_t keys[V];
      double c[V];
      if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = 1.0 / (1.0 + exp(-static_cast<double>(l[j])));
        }
      } else {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = exp(l[j] == most ? 0.0 : static_cast<double>(l[j]) - static_cast<double>(most));
          sum += c[j];
        }
        for (int d = 1; d < kLanes; d *= 2) {
          sum += __shfl_xor(sum, d, 64);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] /= sum;
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (a.bias != nullptr) {
          c[j] += static_cast<double>(b[j]);
        }
        keys[j] = key_of(l[j] == -INFINITY ? -static_cast<double>(INFINITY) : c[j]);
        keys[j] = j < p.n ? keys[j] : Lowest<int64_t>::none;
      }
      if (grouped) {
        keep_groups<V, int64_t>(a, p, -1.0f, keys);
      }
      take_in_order<V, int64_t>(a.k, keys);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        place[j] = step_of(keys[j]);
      }
    } else {
      int keys[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        keys[j] = j < p.n ? key_of(l[j]) : Lowest<int>::none;
      }
      if (grouped) {
        keep_groups<V, int>(a, p, -1.0f, keys);
      }
      take_in_order<V, int>(a.k, keys);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        place[j] = step_of(keys[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (place[j] < a.k) {
      chosen[slot][place[j]] = {p.first + j, l[j]};
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
      most = base_of(largest16(fmaxf(c[0].logit, c[1].logit)));
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float x = c[i].logit;
    s[i] = a.sigmoid ? expf(fminf(x, 0.0f) - low) / (1.0f + expf(-fabsf(x))) : above(x, most);
    s[i] = x != x ? x : s[i];
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
    most = base_of(largest16(most));
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      l[j] = above(l[j], most);
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
      most = base_of(largest16(fmaxf(x[0], x[1])));
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
  constexpr int W = kWide<T, V>;
  const float by = total == 0.0f ? 0.0f : dot / total;
#pragma unroll
  for (int j = 0; j < V; j += W) {
    Wide<T, W> v;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float g = j + i < p.n ? mine[p.first + j + i] : 0.0f;
      v.e[i] = from_f32<T>(dense ? g - l[j + i] * by : g);
    }
    if (a.wide_out && p.n == V) {
      *reinterpret_cast<Wide<T, W>*>(out + j) = v;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (j + i < p.n) {
          out[j + i] = v.e[i];
        }
      }
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

// Whether every run of the values that a lane reads at once is aligned
template <typename T, int V>
bool wide_rows(const RouteArgs& a, const void* p, int64_t stride) {
  constexpr uintptr_t bytes = kWide<T, V> * sizeof(T);
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride * sizeof(T)) |
          (a.groups > 1 ? a.group_size * sizeof(T) : 0)) % bytes == 0;
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
  const bool sums = bias != nullptr || (group_best > 1 && top_groups < groups);
  const unsigned grid = static_cast<unsigned>((rows + kRows - 1) / kRows);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_values(a, [&](auto v) {
      a.full = a.group_size == decltype(v)::value * a.group_lanes && a.groups * a.group_lanes == kLanes;
      a.vector = wide_rows<T, decltype(v)::value>(a, logits, stride);
      a.wide_bias = wide_rows<float, decltype(v)::value>(a, bias, 0);
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
  const unsigned grid = static_cast<unsigned>((rows + kRows - 1) / kRows);
  const size_t lds = sizeof(float) * kRows * experts;
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_values(a, [&](auto v) {
      a.vector = wide_rows<T, decltype(v)::value>(a, logits, stride);
      a.wide_out = wide_rows<T, decltype(v)::value>(a, out, experts);
      route_grad_kernel<T, decltype(v)::value>
          <<<grid, 256, lds, static_cast<hipStream_t>(stream)>>>(a);
    });
  });
}

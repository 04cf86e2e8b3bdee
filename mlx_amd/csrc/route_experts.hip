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
// off, the order is known.  Where they are not, the few that can be meant are formed in 64 (sigmoids: a
// lane each), and only where that does not tell either, the whole row is: softmaxes, equal choices,
// and choices of 2^21 and more, of which 32 bits say nothing.
//
// What bounds it: the instructions of k searches for the largest.  Sixteen lanes have a row, one of
// the rows of lanes that DPP instructions rotate within: the largest of sixteen lanes is four
// instructions, for four rows of a wavefront at once.  A lane holds neighbouring experts of one
// group, so that the lowest lane that has the largest value has the lowest index.  16384 tokens, 8 of
// 256 experts in 4 of 8 groups by sigmoid and bias in float32 (17.8 MB): 15 us, with every choice in 64
// bits 25.7; 8 of 192 in 2 of 3 groups by their best two 13.6, by softmax 24; 32749 tokens, 4 of 60 by
// logits in float16: 6.9 (0.7 of it reading), gradient 7.2; one token 2.1, the launch.
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
__device__ __forceinline__ uint32_t rotated(uint32_t v) {
  return static_cast<uint32_t>(rotated<Rotate>(static_cast<int>(v)));
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
  static __device__ int sum(int one, int two) { return key_of(value_of(one) + value_of(two)); }
};
template <>
struct Lowest<int64_t> {
  static constexpr int64_t taken = static_cast<int64_t>(0x8000000000000000ULL);
  static constexpr int64_t none = taken + 64;
  static __device__ int64_t sum(int64_t one, int64_t two) {
    return key_of(value_of(one) + value_of(two));
  }
};
template <>
struct Lowest<float> {
  static constexpr float none = -INFINITY;
  static __device__ float sum(float one, float two) { return one + two; }
};
template <>
struct Lowest<uint32_t> {
  static constexpr uint32_t none = 0;
  static __device__ uint32_t sum(uint32_t one, uint32_t) { return one; } // (not called for)
};

template <typename K>
__device__ __forceinline__ K larger(K a, K b) {
  if constexpr (std::is_same_v<K, float>) {
    return fmaxf(a, b);
  } else {
    return max(a, b);
  }
}
template <typename K>
__device__ __forceinline__ K smaller(K a, K b) {
  if constexpr (std::is_same_v<K, float>) {
    return fminf(a, b);
  } else {
    return min(a, b);
  }
}

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

// The largest and the second largest of a group
template <int V, typename K>
__device__ __forceinline__ void best_two(const RouteArgs& a, const K (&keys)[V], K* best, K* second) {
  // of the lane's; then of the group's lanes
  K one = keys[0];
  K two = Lowest<K>::none;
#pragma unroll
  for (int j = 1; j < V; ++j) {
    two = larger(two, smaller(one, keys[j]));
    one = larger(one, keys[j]);
  }
  for (int d = 1; d < a.group_lanes; d *= 2) {
    const K other = __shfl_xor(one, d, 64);
    const K other_two = __shfl_xor(two, d, 64);
    two = larger(larger(two, other_two), smaller(one, other));
    one = larger(one, other);
  }
  *best = one;
  *second = two;
}

// The groups with the largest marks: whether the lane's is one of them
template <typename K>
__device__ __forceinline__ bool largest_groups(const RouteArgs& a, const Place& p, K mark, float* gap) {
  mark = p.group < a.groups ? mark : Lowest<K>::none;
  bool stays = false;
  K last = mark;
  for (int n = 0; n < a.top_groups; ++n) {
    last = largest16(mark);
    const bool mine = first16(mark == last) / a.group_lanes == p.group;
    stays |= mine;
    mark = mine ? Lowest<K>::none : mark;
  }
  if constexpr (std::is_same_v<K, float>) { // how far the first that does not is from the last that does
    *gap = last - largest16(mark);
  }
  return stays;
}

// By the sum of the group_best largest `keys` of each
template <int V, typename K>
__device__ __forceinline__ bool group_counts(
    const RouteArgs& a, const Place& p, const K (&keys)[V], float* gap) {
  K one, two;
  best_two<V, K>(a, keys, &one, &two);
  return largest_groups<K>(a, p, a.group_best == 2 ? Lowest<K>::sum(one, two) : one, gap);
}

// A choice of sigmoids (or a logit) in 64 bits
__device__ __forceinline__ double exact_choice(bool sums, float l, float b) {
  if (!sums) {
    return static_cast<double>(l);
  }
  return l == -INFINITY ? -static_cast<double>(INFINITY)
                        : 1.0 / (1.0 + exp(-static_cast<double>(l))) + static_cast<double>(b);
}

// The groups that count by the choices in 64 bits of those that are their best two (or one) of `c`,
// which are off by less than a quarter of `apart`; *exact is false where it is not known which those are.
template <int V>
__device__ __forceinline__ bool exact_groups(
    const RouteArgs& a, const Place& p, const float (&c)[V], const float (&l)[V], const float (&b)[V],
    float apart, bool* exact) {
  float one, two;
  best_two<V, float>(a, c, &one, &two);
  float third = -INFINITY;
  float l_of[2] = {-INFINITY, -INFINITY};
  float b_of[2] = {0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    third = c[j] < two ? fmaxf(third, c[j]) : third;
    if (c[j] == one) {
      l_of[0] = l[j];
      b_of[0] = a.bias == nullptr ? 0.0f : b[j];
    } else if (c[j] == two) {
      l_of[1] = l[j];
      b_of[1] = a.bias == nullptr ? 0.0f : b[j];
    }
  }
  for (int d = 1; d < a.group_lanes; d *= 2) {
    third = fmaxf(third, __shfl_xor(third, d, 64));
  }
  bool known = one - two > apart;
  // each lane the choices of those that it has; of a group's lanes one has the best, one the second
  // (equal ones cannot be told apart here)
  double sum = l_of[0] == -INFINITY ? 0.0 : exact_choice(true, l_of[0], b_of[0]);
  // how many have the best, and the second: a lane may have more than one of them
  constexpr int kSecond = 1 << 16;
  int has = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    has += c[j] == one ? 1 : c[j] == two ? kSecond : 0;
  }
  if (a.group_best == 2) {
    known = known && two - third > apart;
    sum += l_of[1] == -INFINITY ? 0.0 : exact_choice(true, l_of[1], b_of[1]);
  }
  for (int d = 1; d < a.group_lanes; d *= 2) {
    sum += __shfl_xor(sum, d, 64);
    has += __shfl_xor(has, d, 64);
  }
  known = known && has % kSecond == 1 && (a.group_best == 1 || has / kSecond == 1);
  // (a group whose two are not known: nor are the row's)
  const uint32_t not_known = static_cast<uint32_t>(
      __ballot(!known && p.group < a.groups) >> (threadIdx.x & 48));
  *exact = (not_known & 0xffff) == 0;
  return largest_groups<int64_t>(a, p, key_of(sum), nullptr);
}

// The n-th largest of sixteen lanes' distinct unsigned `keys` is the largest u with u - (the one
// before) nearest to 2^32: what is below the one before wraps round to the top, in order, what is
// not stays at the bottom.  So a step is a subtraction and half a three-way maximum a value.  Lane n
// gets the n-th in `mine`; false if two of them, or the last and the first that is not taken, are
// nearer than `apart`.
template <int V>
__device__ __forceinline__ bool take(
    int k, uint32_t apart, const uint32_t (&keys)[V], uint32_t (&mine)[2]) {
  const int lane = threadIdx.x & 15;
  bool known = true;
  uint32_t last = 0;
  for (int n = 0; n <= k; ++n) {
    uint32_t best = keys[0] - last;
#pragma unroll
    for (int j = 1; j < V; ++j) {
      best = max(best, keys[j] - last);
    }
    best = largest16(best);
    known = known && (n == 0 || 0u - best > apart);
    last += best;
    mine[0] = lane == n ? last : mine[0];
    if (k > 16) {
      mine[1] = lane + 16 == n ? last : mine[1];
    }
  }
  return known;
}

// The expert of a key that tells the distance from the largest, and the place
template <int V>
__device__ __forceinline__ int expert_of(const RouteArgs& a, uint32_t key) {
  const int place = 16 * V - 1 - static_cast<int>(key & (16 * V - 1));
  const int lane = place / V;
  return lane / a.group_lanes * a.group_size + (lane & (a.group_lanes - 1)) * V + place % V;
}

template <typename T, int V, bool kSums>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  __shared__ int chosen[kRows][kMostChosen];
  const int slot = threadIdx.x / kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
  const int64_t at = min(row, a.rows - 1); // (sixteen lanes work or not together; all vote)
  const T* logits = static_cast<const T*>(a.logits) + at * a.stride;
  const Place p = place_of<V>(a);
  float l[V];
  read_logits<T, V>(logits + p.first, p.n, a.vector, l);

  // softmax: the largest logit and the sum above it
  float most = 0.0f;
  float total = 0.0f;
  if (!a.sigmoid && (kSums || !a.normalize)) {
    most = l[0];
#pragma unroll
    for (int j = 1; j < V; ++j) {
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
  const bool grouped = a.top_groups < a.groups;
  int index[2];
  float logit[2];

  // 16-bit logits leave 13 bits of a float free: those tell the index, the lowest the largest, and
  // every key is another.  Else a key is the distance from the row's largest choice in fixed point,
  // and the place; two are told apart if they are further from each other than the choices can be off:
  // logits by their rounding; sigmoids by 2^-21, softmaxes by (V + 32) 2^-24 (sums of V values a
  // lane, of e^x with x off by its rounding), with their rounding 2^-23 of their size.
  constexpr bool kUnique = !kSums && sizeof(T) == 2;
  constexpr uint32_t kPlaces = 16 * V;
  bool known = true;
  int refined = -1; // the lane's choice, if it was found so
  uint32_t mine[2] = {0, 0};
  {
    uint32_t keys[V];
    if constexpr (kUnique) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const uint32_t key = static_cast<uint32_t>(key_of(l[j])) ^ 0x80000000u;
        keys[j] = (key & ~0x1fffu) + 0x1000 + (kMostExperts - 1 - p.first - j);
        keys[j] = j < p.n ? keys[j] : 0;
      }
      if (grouped) {
        float gap;
        const bool counts = group_counts<V, uint32_t>(a, p, keys, &gap);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          keys[j] = counts ? keys[j] : 0;
        }
      }
      take<V>(a.k, 0, keys, mine);
    } else {
      float c[V];
      float off; // of a choice
      float scale = kSums ? 0x1p32f / kPlaces / 4 : 0x1p32f / kPlaces / 32;
      if constexpr (kSums) {
        if (a.sigmoid) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            c[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -1.44269504f));
          }
        } else {
          const float by = 1.0f / total; // (NaN, or nothing at all: no choice is known below)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            c[j] = above(l[j], most) * by;
          }
        }
        off = a.sigmoid ? 0x1p-20f : (V + 32) * 0x1p-23f;
        if (a.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            c[j] += b[j];
          }
        }
      } else {
        off = 0x1p-20f; // (of a distance of 32 at most)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = l[j];
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) { // neither masked nor NaN
        c[j] = fmaxf(l[j] > -INFINITY ? c[j] : -INFINITY, -INFINITY);
      }
      bool counts = p.n > 0;
      if (grouped) {
        float gap;
        const bool stays = group_counts<V, float>(a, p, c, &gap);
        counts = stays && counts;
        if constexpr (kSums) {
          float size = 1.0f; // (of what the choices are off by; lanes may have none)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            size = c[j] > -INFINITY ? fmaxf(size, fabsf(c[j])) : size;
          }
          const float apart = 4.0f * off * (1.0f + largest16(size));
          known = gap > apart;
          if (a.sigmoid && __any(!known)) {
            bool exact;
            const bool also = exact_groups<V>(a, p, c, l, b, apart, &exact);
            counts = !known && exact ? also && p.n > 0 : counts;
            known = known || exact;
          }
        } else {
          known = gap >= 0.0f; // (logits are what they are; equal ones by index)
        }
      }
      float top = c[0];
#pragma unroll
      for (int j = 1; j < V; ++j) {
        top = fmaxf(top, c[j]);
      }
      top = largest16(counts ? top : -INFINITY);
      off *= kSums ? 1.0f + fabsf(top) : 1.0f;
      constexpr float kEnd = 0x1p32f / kPlaces - 256.0f; // (below the last in 24 bits)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float far = fminf((top - c[j]) * scale, kEnd);
        keys[j] = (0xffffffffu - static_cast<uint32_t>(far) * kPlaces) -
            (static_cast<uint32_t>(p.lane) * V + j);
        keys[j] = counts ? keys[j] : 0;
      }
      if (!a.full) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          keys[j] = j < p.n ? keys[j] : 0;
        }
      }
      // both of them off, and both cut to whole numbers; choices as large as a bias of 2^21 are off by
      // more than the keys reach, and no order is known
      const float most_off = 2.0f * off * scale;
      constexpr float kReach = 0x1p32f / kPlaces - 4.0f;
      const uint32_t apart = (static_cast<uint32_t>(fminf(most_off, kReach)) + 3) * kPlaces;
      known = known && most_off < kReach && fabsf(top) < INFINITY;
      bool in_order = take<V>(a.k, apart, keys, mine);
      // Where they are too near each other, but the first n >= k of sixteen are known to be the
      // largest: a lane each, their choices in 64 bits, and a place for each.
      if (__any(known && !in_order) && a.k < 16 && !(kSums && !a.sigmoid)) {
        uint32_t one[2] = {0, 0};
        take<V>(15, 0, keys, one);
        const uint32_t next = __shfl_down(one[0], 1, kLanes);
        const uint32_t ends = static_cast<uint32_t>(
            __ballot(one[0] - next > apart && p.lane >= a.k - 1 && p.lane < 15) >>
            (threadIdx.x & 48)) & 0xffffu;
        const bool is = p.lane < __ffs(static_cast<int>(ends)); // (none: 0)
        const int mine_of = expert_of<V>(a, one[0]);
        const int e = is && mine_of < a.experts ? mine_of : 0;
        const int64_t key = is ? key_of(exact_choice(
                                     kSums, to_f32(logits[e]), a.bias == nullptr ? 0.0f : a.bias[e]))
                               : Lowest<int64_t>::none;
        int place = 0;
        const auto behind = [&](auto r) {
          const int64_t other = rotated<decltype(r)::value>(key);
          const int index_of = rotated<decltype(r)::value>(e);
          place += other > key || (other == key && index_of < e);
        };
        behind(IntC<1>{}); behind(IntC<2>{}); behind(IntC<3>{}); behind(IntC<4>{}); behind(IntC<5>{});
        behind(IntC<6>{}); behind(IntC<7>{}); behind(IntC<8>{}); behind(IntC<9>{}); behind(IntC<10>{});
        behind(IntC<11>{}); behind(IntC<12>{}); behind(IntC<13>{}); behind(IntC<14>{}); behind(IntC<15>{});
        // (what is at the end of the range is only known to be there or beyond)
        const uint32_t low = static_cast<uint32_t>(
            __ballot(is && one[0] <= apart) >> (threadIdx.x & 48)) & 0xffffu;
        const bool found = known && !in_order && ends != 0 && low == 0;
        if (found && is && place < a.k) {
          chosen[slot][place] = e;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (found) {
          refined = p.lane < a.k ? chosen[slot][p.lane] : 0;
          in_order = true;
        }
      }
      known = known && in_order;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (kUnique) {
      index[i] = kMostExperts - 1 - static_cast<int>(mine[i] & 0xfff);
    } else {
      index[i] = expert_of<V>(a, mine[i]);
    }
  }
  index[0] = refined >= 0 ? refined : index[0];
  // (the sixteen lanes of a row agree)
  if (!kUnique && __any(!known)) {
    int place[V]; // which choice a value is
    const auto order = [&](auto&& keys) {
      using K = std::remove_reference_t<decltype(keys[0])>;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        keys[j] = j < p.n ? keys[j] : Lowest<K>::none;
      }
      if (grouped) {
        const bool counts = group_counts<V, K>(a, p, keys, nullptr);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          keys[j] = counts ? keys[j] : Lowest<K>::none;
        }
      }
      take_in_order<V, K>(a.k, keys);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        place[j] = step_of(keys[j]);
      }
    };
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
      }
      order(keys);
    } else {
      int keys[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        keys[j] = key_of(l[j]);
      }
      order(keys);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (place[j] < a.k) {
        chosen[slot][place[j]] = p.first + j;
      }
    }
    // (the wavefront's own rows)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      index[i] = p.lane + 16 * i < a.k ? chosen[slot][p.lane + 16 * i] : 0;
    }
  }
  if (row >= a.rows) {
    return;
  }

  // each of the sixteen lanes has two of the chosen at most
  float s[2];
  float low = 0.0f; // sigmoid: all counted up, where all are tiny
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    logit[i] = -INFINITY;
    if (p.lane + 16 * i < a.k) {
      if constexpr (kUnique) { // (its lower 13 bits are none again)
        const float v = value_of(static_cast<int>((mine[i] & ~0x1fffu) ^ 0x80000000u));
        logit[i] = __int_as_float(__float_as_int(v) & ~0x1fff);
        if (logit[i] == -INFINITY) { // (or NaN)
          logit[i] = to_f32(logits[index[i]]);
        }
      } else {
        logit[i] = to_f32(logits[index[i]]);
      }
    }
  }
  if (a.normalize) {
    if (a.sigmoid) {
      low = largest16(fmaxf(fminf(logit[0], 0.0f), fminf(logit[1], 0.0f)));
      low = low == -INFINITY ? 0.0f : low;
    } else {
      most = base_of(largest16(fmaxf(logit[0], logit[1])));
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float x = logit[i];
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
      a.indices[to] = index[i];
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

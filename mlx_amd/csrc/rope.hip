// rope.hip -- rotary positions, alone and on the way into a paged cache.
//
// Pair i of a head's first `dims` columns turns by the angle scale * position / freqs[i], with
// freqs[i] = base^(2 i / dims) unless they are given: (a, b) -> (a cos - b sin, b cos + a sin).
// The pair is (i, i + dims / 2), or (2 i, 2 i + 1) if traditional.  With several axes the pairs
// are dealt out in sections, each with the position along its axis.  The gradient turns back.
//
// Angles are formed in turns and in 64 bits, and only what is left of a whole turn is rounded to
// 32: a position of 2^20 would lose 0.06 radians in 32.  The products are 32 bits, rounded once.
//
// What bounds it: reading and writing the heads.  Cosines and sines of a token are the same for all
// of its heads, so a workgroup takes whole tokens (or a run of the heads of one, where tokens
// are few), makes a table of them in LDS, and its threads go through the heads' columns: 2 V
// columns a thread and turn, V of each half, so that lanes read and write 16 bytes at a time
// where strides and alignment allow it.  4 x 2500 tokens, 28 heads of 128 in bfloat16, 143 MB: 27 us,
// 5.2 TB/s, which is what a copy of that size reaches; 1021 tokens, 16 heads of 80 in float32, 32 columns
// turned, 10 MB: 5, launch and one round of workgroups.
//
// The cache update is the same pass over the query heads (to a new tensor), the key heads (to the
// pages) and the value heads (a copy to the pages).  16 prompts padded to 1531 tokens, 28 and 4 heads
// of 128 in bfloat16: 72 us, 254 MB for tokens and 77 of zeros for padding, 4.6 TB/s; one token each of 48
// sequences, 64 and 8 heads: 4.
#include <cmath>

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kMostPairs = 128;
constexpr int kMostAxes = 4;
constexpr int kThreads = 256;

struct RopeArgs {
  const char* from[3]; // x, or q, k, v
  char* to[3];
  int64_t from_strides[3][3], to_strides[3][3]; // elements: [sequence, head, token]; pages: [page, head, row]
  int ends[3];  // heads of x or q; with those of k; with those of v
  int B, L, D;
  int pairs;    // dims / 2
  int step;     // columns between the two of a pair: 1 (traditional) or pairs
  int rotated;  // items of a head that are rotated, of 2 V columns each
  Divisor items; // D / (2 V)
  Divisor slots; // heads of a workgroup
  int tokens;    // of a workgroup (1 if its heads are not all)
  int token_groups;
  float sign;
  // positions: [axes][B][L], int32 or int64; null: the place in the cache
  const void* positions;
  int64_t position_strides[3];
  int wide_positions;
  int axis_ends[kMostAxes]; // pairs up to each axis' last
  int axes;
  const float* freqs; // or null
  double scale_turns; // scale / (2 pi)
  // the cache
  const int32_t* table;
  const int32_t* lengths; // or null
  int64_t table_stride;
  int pages, table_width;
  Divisor page; // rows of a page
  double turns[kMostPairs]; // per position, without freqs
};

template <typename T, int V>
struct alignas((V * sizeof(T) > 16) ? 16 : V * sizeof(T)) Columns {
  T v[V];
};

template <typename T, int V, bool kCache>
__global__ __launch_bounds__(kThreads) void rope_kernel(const RopeArgs a) {
  extern __shared__ float2 table[]; // [tokens][pairs]: cosine, sine
  const int b = blockIdx.x / a.token_groups;
  const int first = (blockIdx.x - b * a.token_groups) * a.tokens;
  const int count = min(a.tokens, a.L - first);
  const int64_t before = kCache ? static_cast<int64_t>(a.lengths[b]) - a.L : 0; // (of token 0)

  for (int n = threadIdx.x; n < count * a.pairs; n += kThreads) {
    const int t = n / a.pairs;
    const int pair = n - t * a.pairs;
    int64_t position = before + first + t;
    if (a.positions != nullptr) {
      int axis = 0;
      while (axis + 1 < a.axes && pair >= a.axis_ends[axis]) {
        ++axis;
      }
      const int64_t at = axis * a.position_strides[0] + b * a.position_strides[1] +
          (first + t) * a.position_strides[2];
      position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[at]
                                  : static_cast<const int32_t*>(a.positions)[at];
    }
    const double rate =
        a.freqs != nullptr ? a.scale_turns / static_cast<double>(a.freqs[pair]) : a.turns[pair];
    double turns = static_cast<double>(position) * rate;
    // to the nearest quarter: an eighth of a turn is left, whose rounding is off by 0.4 2^-24 radians
    const double quarters = rint(4.0 * turns);
    float sine, cosine;
    sincospif(2.0f * static_cast<float>(turns - 0.25 * quarters), &sine, &cosine);
    const int quarter = static_cast<int>(quarters - 4.0 * floor(0.25 * quarters)); // 0 .. 3
    const float across = quarter & 1 ? -sine : cosine;
    const float up = quarter & 1 ? cosine : sine;
    table[n] = make_float2(quarter & 2 ? -across : across, a.sign * (quarter & 2 ? -up : up));
  }
  __syncthreads();

  const int slot0 = blockIdx.y * a.slots.d;
  const int slots = min(a.slots.d, a.ends[2] - slot0);
  const int all = count * slots * a.items.d;
  for (int n = threadIdx.x; n < all; n += kThreads) {
    int item, slot;
    int t = a.items.divide(n, &item);
    if (slots == a.slots.d) {
      t = a.slots.divide(t, &slot);
    } else { // the last run of heads, of one token
      slot = t;
      t = 0;
    }
    slot += slot0;
    const int which = kCache ? (slot >= a.ends[0]) + (slot >= a.ends[1]) : 0;
    const int head = slot - (which == 0 ? 0 : a.ends[which - 1]);
    const int64_t token = first + t;
    const int64_t(&fs)[3] = a.from_strides[which];
    const int64_t(&ts)[3] = a.to_strides[which];
    const T* src = reinterpret_cast<const T*>(a.from[which]) + b * fs[0] + head * fs[1] + token * fs[2];
    T* dst = reinterpret_cast<T*>(a.to[which]);
    const int64_t place = before + token;
    if (!kCache || which == 0) {
      dst += b * ts[0] + head * ts[1] + token * ts[2];
    } else {
      if (place < 0 || place >= static_cast<int64_t>(a.table_width) * a.page.d) {
        continue;
      }
      int row_of_page;
      const int at = a.page.divide(static_cast<int>(place), &row_of_page);
      const int page = a.table[b * a.table_stride + at];
      if (page < 0 || page >= a.pages) {
        continue;
      }
      dst += page * ts[0] + head * ts[1] + row_of_page * ts[2];
    }
    const bool turn = item < a.rotated && which < 2;
    const int one = !turn || a.step == 1 ? item * 2 * V : item * V;
    const int two = turn && a.step != 1 ? one + a.step : one + V;
    Columns<T, V> x;
    Columns<T, V> y;
    if (kCache && place < 0) { // padding in front: zeros
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x.v[i] = y.v[i] = from_f32<T>(0.0f);
      }
      *reinterpret_cast<Columns<T, V>*>(dst + one) = x;
      *reinterpret_cast<Columns<T, V>*>(dst + two) = y;
      continue;
    }
    x = *reinterpret_cast<const Columns<T, V>*>(src + one);
    y = *reinterpret_cast<const Columns<T, V>*>(src + two);
    if (turn) {
      const float2* angles = table + t * a.pairs + item * V;
      if (a.step != 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 r = angles[i];
          const float p = to_f32(x.v[i]);
          const float q = to_f32(y.v[i]);
          x.v[i] = from_f32<T>(fmaf(p, r.x, -(q * r.y)));
          y.v[i] = from_f32<T>(fmaf(q, r.x, p * r.y));
        }
      } else if constexpr (V == 1) {
        const float2 r = angles[0];
        const float p = to_f32(x.v[0]);
        const float q = to_f32(y.v[0]);
        x.v[0] = from_f32<T>(fmaf(p, r.x, -(q * r.y)));
        y.v[0] = from_f32<T>(fmaf(q, r.x, p * r.y));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          Columns<T, V>& z = i < V / 2 ? x : y;
          const int j = 2 * (i % (V / 2));
          const float2 r = angles[i];
          const float p = to_f32(z.v[j]);
          const float q = to_f32(z.v[j + 1]);
          z.v[j] = from_f32<T>(fmaf(p, r.x, -(q * r.y)));
          z.v[j + 1] = from_f32<T>(fmaf(q, r.x, p * r.y));
        }
      }
    }
    *reinterpret_cast<Columns<T, V>*>(dst + one) = x;
    *reinterpret_cast<Columns<T, V>*>(dst + two) = y;
  }
}

// What both entry points check and set of the rotation: positions, pairs, rates.
int set_rotation(
    const char* tag,
    RopeArgs& a,
    int D,
    int dims,
    int traditional,
    double base,
    double scale,
    const float* freqs,
    const void* positions,
    const int64_t* position_strides,
    int wide_positions,
    int axes,
    const int* sections,
    int inverse) {
  if (D % 2 != 0 || dims <= 0 || dims % 2 != 0 || dims > D || dims > 2 * kMostPairs) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d columns cannot be rotated of %d", tag, dims, D);
  }
  if (axes < 1 || axes > kMostAxes) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] %d axes", tag, axes);
  }
  if (!(base > 0.0) || !std::isfinite(base) || !std::isfinite(scale)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] base must be positive, base and scale finite", tag);
  }
  a.D = D;
  a.pairs = dims / 2;
  a.step = traditional ? 1 : a.pairs;
  a.sign = inverse ? -1.0f : 1.0f;
  a.axes = axes;
  int end = 0;
  for (int i = 0; i < axes; ++i) {
    const int pairs = axes == 1 ? a.pairs : sections[i];
    if (pairs < 0 || pairs > a.pairs) {
      return fail(MLXROCM_INVALID_ARGUMENT, "[%s] section of %d pairs", tag, pairs);
    }
    end += pairs;
    a.axis_ends[i] = end;
  }
  if (end != a.pairs) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] sections of %d pairs for %d columns", tag, end, dims);
  }
  a.positions = positions;
  a.wide_positions = wide_positions;
  if (positions != nullptr && position_strides != nullptr) {
    for (int i = 0; i < 3; ++i) {
      a.position_strides[i] = position_strides[i];
    }
  }
  a.freqs = freqs;
  a.scale_turns = scale / (2.0 * M_PI);
  if (freqs == nullptr) {
    for (int i = 0; i < a.pairs; ++i) {
      a.turns[i] = a.scale_turns * std::pow(base, -static_cast<double>(i) / a.pairs);
    }
  }
  return MLXROCM_OK;
}

// Columns of a half that a thread takes: as many as divide both parts of a head and keep every
// access aligned, 16 bytes at most.
int columns_of(const RopeArgs& a, int tensors, size_t size) {
  int v = static_cast<int>(16 / size);
  const auto fits = [&](int c) {
    if (a.pairs % c != 0 || (a.D - 2 * a.pairs) % (2 * c) != 0) {
      return false;
    }
    const int64_t bytes = static_cast<int64_t>(c * size);
    for (int w = 0; w < tensors; ++w) {
      int64_t bits = reinterpret_cast<intptr_t>(a.from[w]) | reinterpret_cast<intptr_t>(a.to[w]);
      for (int i = 0; i < 3; ++i) {
        bits |= a.from_strides[w][i] * static_cast<int64_t>(size);
        bits |= a.to_strides[w][i] * static_cast<int64_t>(size);
      }
      if ((bits & (bytes - 1)) != 0) {
        return false;
      }
    }
    return true;
  };
  while (v > 1 && !fits(v)) {
    v /= 2;
  }
  return v;
}

template <typename T, bool kCache>
int launch(const char* tag, RopeArgs& a, hipStream_t stream) {
  const int v = columns_of(a, kCache ? 3 : 1, sizeof(T));
  a.items = Divisor(a.D / (2 * v));
  a.rotated = a.pairs / v;
  // Two tokens a workgroup where there are four workgroups a CU of them; else one token, and its
  // heads are cut until there are two workgroups a CU or a thread has one item.  us with one, two, four
  // (bfloat16): into the cache 16 ragged prompts of up to 1531 tokens, 36 heads of 128 77, 72, 75, as many
  // of 1531 89, 88, 93, 8 of 2000, 10 heads of 256 30, 27, 28; alone 4 x 2500, 28 of 128 25, 24, 25, 12000,
  // 12 of 96 16.3, 12.6, 12.8, 4096, 8 of 256 9.1, 8.9, 8.9, 11200, 32 of 64 18.2, 17.2, 15.8, 4096, 64 of 128
  // 22.2, 22.6, 22.8.
  const int heads = a.ends[2];
  const int64_t tokens = static_cast<int64_t>(a.B) * a.L;
  a.tokens = tokens >= 4 * 512 ? 2 : 1;
  int slots = heads;
  if (a.tokens == 1) {
    while (slots > 1 && slots * a.items.d > kThreads &&
           tokens * ((heads + slots - 1) / slots) < 512) {
      slots = (slots + 1) / 2;
    }
  }
  a.slots = Divisor(slots);
  a.token_groups = (a.L + a.tokens - 1) / a.tokens;
  const int64_t blocks = static_cast<int64_t>(a.B) * a.token_groups;
  const int64_t runs = (heads + slots - 1) / slots;
  if (blocks >= int64_t{1} << 24 || runs > 65535 || // (2^32 threads)
      static_cast<int64_t>(a.tokens) * slots * a.items.d > INT32_MAX) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", tag);
  }
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(runs));
  const size_t lds = sizeof(float2) * a.tokens * a.pairs;
  const auto go = [&](auto kernel) {
    kernel<<<grid, kThreads, lds, stream>>>(a);
    return MLXROCM_OK;
  };
  if constexpr (sizeof(T) == 2) {
    if (v == 8) {
      go(rope_kernel<T, 8, kCache>);
    }
  }
  if (v == 4) {
    go(rope_kernel<T, 4, kCache>);
  } else if (v == 2) {
    go(rope_kernel<T, 2, kCache>);
  } else if (v == 1) {
    go(rope_kernel<T, 1, kCache>);
  }
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

} // namespace

} // namespace mlxrocm

extern "C" int mlxrocm_rope(
    const void* x,
    void* out,
    int B,
    int H,
    int L,
    int D,
    const int64_t* strides,
    const void* positions,
    const int64_t* position_strides,
    int wide_positions,
    int axes,
    const int* sections,
    int dims,
    int traditional,
    double base,
    double scale,
    const float* freqs,
    int inverse,
    int dtype,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_rope");
  using namespace mlxrocm;
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[rope] unknown dtype %d", dtype);
  }
  if (B < 0 || H < 0 || L < 0 || D < 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[rope] negative dimension");
  }
  if (axes > 1 && sections == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[rope] null sections");
  }
  RopeArgs a{};
  const int rc = set_rotation(
      "rope", a, D, dims, traditional, base, scale, freqs, positions, position_strides,
      wide_positions, axes, sections, inverse);
  if (rc != MLXROCM_OK) {
    return rc;
  }
  if (B == 0 || H == 0 || L == 0) {
    return MLXROCM_OK;
  }
  if (x == nullptr || out == nullptr || strides == nullptr || positions == nullptr ||
      position_strides == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[rope] null pointer");
  }
  a.from[0] = static_cast<const char*>(x);
  a.to[0] = static_cast<char*>(out);
  for (int i = 0; i < 3; ++i) {
    a.from_strides[0][i] = strides[i];
    a.to_strides[0][i] = strides[3 + i];
    a.ends[i] = H;
  }
  a.B = B;
  a.L = L;
  return dispatch_dtype(dtype, [&](auto t) {
    return launch<decltype(t), false>("rope", a, static_cast<hipStream_t>(stream));
  });
}

extern "C" int mlxrocm_rope_cache_update(
    const void* q,
    const void* k,
    const void* v,
    void* q_out,
    void* k_pages,
    void* v_pages,
    const int32_t* table,
    const int32_t* lengths,
    int B,
    int Hq,
    int Hkv,
    int L,
    int D,
    int pages,
    int page_size,
    int table_width,
    const int64_t* strides,
    const void* positions,
    const int64_t* position_strides,
    int wide_positions,
    int axes,
    const int* sections,
    int dims,
    int traditional,
    double base,
    double scale,
    const float* freqs,
    int dtype,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_rope_cache_update");
  using namespace mlxrocm;
  const char* tag = "rope_cache_update";
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] unknown dtype %d", tag, dtype);
  }
  if (B < 0 || Hq < 0 || Hkv < 0 || L < 0 || D < 0 || pages < 0 || table_width < 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] negative dimension", tag);
  }
  if (page_size <= 0 || page_size % 16 != 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] page size %d is not a multiple of 16", tag, page_size);
  }
  if (axes > 1 && (sections == nullptr || positions == nullptr)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] several axes without sections or positions", tag);
  }
  RopeArgs a{};
  const int rc = set_rotation(
      tag, a, D, dims, traditional, base, scale, freqs, positions, position_strides,
      wide_positions, axes, sections, 0);
  if (rc != MLXROCM_OK) {
    return rc;
  }
  const int64_t heads = static_cast<int64_t>(Hq) + 2 * static_cast<int64_t>(Hkv);
  if (B == 0 || L == 0 || heads == 0) {
    return MLXROCM_OK;
  }
  if ((Hq > 0 && (q == nullptr || q_out == nullptr)) ||
      (Hkv > 0 && (k == nullptr || v == nullptr)) || lengths == nullptr || strides == nullptr ||
      (Hkv > 0 && pages > 0 && table_width > 0 &&
       (k_pages == nullptr || v_pages == nullptr || table == nullptr)) ||
      (positions != nullptr && position_strides == nullptr)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer", tag);
  }
  if (static_cast<int64_t>(table_width) * page_size > INT32_MAX || heads > INT32_MAX) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", tag);
  }
  const void* from[3] = {q, k, v};
  void* to[3] = {q_out, k_pages, v_pages};
  for (int w = 0; w < 3; ++w) {
    a.from[w] = static_cast<const char*>(from[w]);
    a.to[w] = static_cast<char*>(to[w]);
    for (int i = 0; i < 3; ++i) {
      a.from_strides[w][i] = strides[3 * w + i];
      a.to_strides[w][i] = strides[9 + 3 * w + i];
    }
    a.ends[w] = Hq + w * Hkv;
  }
  a.B = B;
  a.L = L;
  a.table = table;
  a.table_stride = strides[18];
  a.lengths = lengths;
  a.pages = pages;
  a.page = Divisor(page_size);
  a.table_width = pages == 0 ? 0 : table_width; // (no place is in a cache without pages)
  return dispatch_dtype(dtype, [&](auto t) {
    return launch<decltype(t), true>(tag, a, static_cast<hipStream_t>(stream));
  });
}

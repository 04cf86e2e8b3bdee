// adapter.hip -- what low-rank adapters of many requests add to a shared projection, and the
// gradients.
//
//   h[t] = scale x[t] A[i]^T       (r numbers; i the adapter of token t)
//   out[t] = y[t] + h[t] B[i]^T
//   g[t] = scale dout[t] B[i],  dx[t] = g[t] A[i]
//   dA[i] = sum over its tokens of g[t]^T x[t],  dB[i] = sum of dout[t]^T h[t]
//
// What bounds it: HBM.  The products are some r operations a byte; x, y and the result are read and
// written once, and so are the adapters in use.  A workgroup has tokens of one adapter (so each
// adapter is read once for all of its tokens), as the columns of the matrix instruction's result; what
// is read goes from memory into the instruction's operands without LDS, 16 bytes a lane.
//
//   group    the tokens by adapter, and the tiles of them (one workgroup).  Up to 64 indices need
//            none: every workgroup finds its tile by itself, an index a lane (13 prompts: 6 us less).
//   shrink   h or g, in 32 bits.  The four wavefronts of a workgroup and, for few tokens, several
//            workgroups share a token's sum; the parts are added in one order by who reads them.
//   expand   out or dx.  16-bit types: h as the sum of numbers of the type, against the same operand
//            of B: three in bfloat16, all of float32's 24 bits; two in float16, 23 bits of the token's
//            largest, which h is counted by a power of two to bring to 2^13 (a smaller rank keeps 23 of
//            its own down to 2^-16 of that, then 2^-38 of it).  So sums that cancel keep what 32 bits
//            have of them (with two numbers, 17 bits, in bfloat16 8192 tokens of 4096 to 14336 by rank 16
//            take as long, 16384 of 8192 to 1024 by rank 32 with gradients 284 us instead of 288).
//   turn     A and B with their two dimensions swapped, for the gradients: then g and dx are the
//            same two products.
//   tokens   dB and dA in one launch: sums over tokens, cut so that workgroups fill the card; dB
//            first, whose dout the products before have just read (47 us of 235 MB then, 66 behind dx).
//            h and g as three bfloat16 numbers, float16 activations as two.
//   join     their parts, in order; zeros for adapters without tokens.
//
// Measured, bfloat16: 8192 tokens of 4096 values to 14336 by rank 16: shrink 19 us, expand 113 (470 MB,
// 4.2 TB/s); backward group 5, turn 5, shrink 64 (235 MB, while the 235 MB before are still written back;
// alone 48), tokens 64 (302 MB), join 6, expand 21.  13 x 601 tokens of 14336 to 4096 by rank 32, float16:
// shrink 65 (224 MB, and as many bytes of A from L2), expand 42 (128 MB).  48 requests of 64 adapters of
// rank 64, 4096 to 14336: 8 and 20, where their 86 MB take 17.
//
// No atomics: the same inputs give the same bits.
#include <cmath>

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kFew = 64;           // indices, or rows of a tile, that a wavefront has in its lanes
constexpr int kMostAdapters = 1024;
constexpr int kMostRank = 256;

// Rows of an adapter: sorted rows first .. first + rows - 1
struct Tile {
  int adapter; // -1: none
  int first, rows;
  int slot; // of the partial sums; -1: the only ones
};

// Where the rows of a call lie and which adapters they have
struct Rows {
  const int32_t* indices; // [n], each for `span` rows; null: all rows have adapter 0
  int n, adapters;
  Divisor span;
  const int32_t* order; // [n] by adapter; null: no grouping (few indices)
  const Tile* tiles;
  const int32_t* n_tiles;

  __device__ __forceinline__ int adapter_of(int entry) const {
    const int i = indices == nullptr ? 0 : indices[entry];
    return static_cast<uint32_t>(i) < static_cast<uint32_t>(adapters) ? i : -1;
  }
  __device__ __forceinline__ int row(int sorted) const {
    int rest;
    const int entry = span.divide(sorted, &rest);
    return (order == nullptr ? entry : order[entry]) * span.d + rest;
  }
};

// The rows of a workgroup's tile to LDS (64 at most) and their adapter; how many there are, none
// if the workgroup has nothing to do.  All threads call it.
__device__ __forceinline__ int find_rows(const Rows& r, int block, int tile, int* to, int* adapter) {
  __shared__ int found[2];
  __shared__ int entries[kFew];
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int rows = 0;
    int of = -1;
    if (r.tiles != nullptr) {
      if (block < *r.n_tiles) {
        const Tile t = r.tiles[block];
        rows = t.rows;
        of = t.adapter;
        if (lane < rows) {
          to[lane] = r.row(t.first + lane);
        }
      }
    } else if (r.n == 1) {
      const int first = block * tile;
      rows = min(tile, r.span.d - first);
      of = r.adapter_of(0);
      if (lane < rows) {
        to[lane] = first + lane;
      }
    } else if (r.span.d == 1) {
      // Single tokens: the first of its kind has them all (a vote; by tiles: 34 us instead of 29, 48
      // requests of rank 64)
      const int mine = lane < r.n ? r.adapter_of(lane) : -2;
      of = __shfl(mine, block, 64);
      const uint64_t like = __ballot(mine == of);
      if (__ffsll(static_cast<unsigned long long>(like)) - 1 == block) {
        rows = __popcll(like);
        if (mine == of) {
          to[__popcll(like & ((uint64_t{1} << lane) - 1))] = lane;
        }
      }
    } else {
      // Each lane an index: how many are like it, and how many of those before it.  The first of
      // its kind has the kind's tiles.
      of = lane < r.n ? r.adapter_of(lane) : -2;
      int like = 0;
      int before = 0;
      for (int i = 0; i < r.n; ++i) {
        const bool same = __builtin_amdgcn_readlane(of, i) == of;
        like += same;
        before += same && i < lane;
      }
      const int all = like * r.span.d;
      const int tiles = of != -2 && before == 0 ? (all + tile - 1) / tile : 0;
      int up = tiles;
      for (int d = 1; d < 64; d *= 2) {
        const int other = __shfl_up(up, d, 64);
        up += lane >= d ? other : 0;
      }
      const uint64_t mine = __ballot(block >= up - tiles && block < up);
      if (mine != 0) {
        const int first = __ffsll(static_cast<unsigned long long>(mine)) - 1;
        const int from = (block - __shfl(up - tiles, first, 64)) * tile;
        rows = min(tile, __shfl(all, first, 64) - from);
        const int kind = __shfl(of, first, 64);
        if (of == kind) {
          entries[before] = lane;
        }
        of = kind;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (lane < rows) {
          int rest;
          const int entry = r.span.divide(from + lane, &rest);
          to[lane] = entries[entry] * r.span.d + rest;
        }
      }
    }
    if (lane == 0) {
      found[0] = rows;
      found[1] = of;
    }
  }
  __syncthreads();
  *adapter = __builtin_amdgcn_readfirstlane(found[1]);
  return __builtin_amdgcn_readfirstlane(found[0]);
}

// ---------------------------------------------------------------- operands
template <typename T>
constexpr int kPer = 16 / sizeof(T); // values of an operand in a lane
template <typename T>
constexpr int kStep = 4 * kPer<T>; // of an instruction (float32: of four)

template <typename T>
__device__ __forceinline__ void multiply(const uint4& a, const uint4& b, floatx4& c) {
  if constexpr (sizeof(T) == 4) {
    const float4 x = __builtin_bit_cast(float4, a);
    const float4 y = __builtin_bit_cast(float4, b);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, c, 0, 0, 0);
  } else {
    c = mfma16<T>(a, b, c);
  }
}

// Elements k .. k + 15 / sizeof(T) of a row of n; what lies past its end is zero (kWhole: nothing
// does).  Sixteen bytes at once also where they are not aligned, as in store_part (4110 tokens of 1024
// values to 1001 by rank 128, float16 with gradients: 182 us; both element by element 339).
template <typename T, bool kAligned, bool kWhole = false>
__device__ __forceinline__ uint4 operand(const T* row, int k, int n) {
  union {
    uint4 u;
    T e[kPer<T>];
  } raw;
  if constexpr (kAligned) { // (n is a multiple)
    if constexpr (kWhole) {
      return *reinterpret_cast<const uint4*>(row + k);
    }
    return k < n ? *reinterpret_cast<const uint4*>(row + k) : uint4{0, 0, 0, 0};
  } else if (kWhole || k + kPer<T> <= n) {
    __builtin_memcpy(&raw.u, row + k, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kPer<T>; ++i) {
      raw.e[i] = k + i < n ? row[k + i] : static_cast<T>(0.0f);
    }
  }
  return raw.u;
}

struct ShrinkArgs {
  Rows rows;
  const void* x; // [T, K]
  int64_t x_stride;
  const void* a; // [adapters, r, K]
  int64_t a_stride, a_row;
  const float* scales; // [adapters], or null
  float scale;
  float* h; // [splits, T, padded]
  int64_t split_stride;
  int K, r, padded; // padded: r up to a multiple of 16
  int per_split;    // of K, a multiple of 4 steps
  int tile;
};

// kGroups groups of 16 tokens, kChunks of 16 ranks; the four wavefronts have parts of the sums.
// (The same part for different tokens, so that A comes from memory once for 128 tokens: 86 us
// instead of 66, 7813 tokens of 14336 values to rank 32, float16.)
template <typename T, int kGroups, int kChunks, bool kAligned>
__global__ __launch_bounds__(256) void shrink_kernel(const ShrinkArgs a) {
  __shared__ int rows[kFew];
  __shared__ floatx4 parts[3][kGroups * kChunks][64];
  int adapter;
  const int count = find_rows(a.rows, blockIdx.x, a.tile, rows, &adapter);
  if (count == 0 || adapter < 0) {
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15;
  const int quarter = lane >> 4;
  const int rank0 = blockIdx.z * kChunks * 16;
  const T* w = static_cast<const T*>(a.a) + adapter * a.a_stride;
  const T* w_row[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    w_row[c] = w + min(rank0 + 16 * c + column, a.r - 1) * a.a_row; // (past r: not stored)
  }
  const float scale = a.scale * (a.scales == nullptr ? 1.0f : a.scales[adapter]);
  const int begin = blockIdx.y * a.per_split;
  const int end = min(a.K, begin + a.per_split);
  for (int base = 0; base < count; base += 16 * kGroups) {
    const T* x_row[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      x_row[i] = static_cast<const T*>(a.x) +
          rows[min(base + 16 * i + column, count - 1)] * a.x_stride;
    }
    floatx4 sum[kGroups][kChunks] = {};
    // A wavefront's two steps are neighbours, so that it reads whole lines.  What others on the CU
    // ask for meanwhile is enough: with the next turn's operands on their way, and with four steps
    // in a turn, a call takes 64 us instead of 52 (8192 tokens of 14336 values to rank 16: 4.5 TB/s).
    constexpr int kAhead = 2;
    constexpr int kTurn = kAhead * kStep<T>;
    const auto turn = [&](int k0, auto whole) {
      uint4 xs[kAhead][kGroups];
      uint4 ws[kAhead][kChunks];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const int k = k0 + s * kStep<T> + quarter * kPer<T>;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          xs[s][i] = operand<T, kAligned, whole.value>(x_row[i], k, end);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          ws[s][c] = operand<T, kAligned, whole.value>(w_row[c], k, end);
        }
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
            multiply<T>(ws[s][c], xs[s][i], sum[i][c]);
          }
        }
      }
    };
    int k = begin + wave * kTurn;
    for (; k + kTurn <= end; k += 4 * kTurn) {
      turn(k, std::true_type{});
    }
    if (k < end) {
      turn(k, std::false_type{});
    }
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          parts[wave - 1][i * kChunks + c][lane] = sum[i][c];
        }
      }
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const int slot = base + 16 * i + column;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          floatx4 s = sum[i][c];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            s += parts[p][i * kChunks + c][lane];
          }
          const int rank = rank0 + 16 * c + 4 * quarter;
          if (slot < count && rank < a.padded) {
            floatx4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[k] = rank + k < a.r ? s[k] * scale : 0.0f;
            }
            *reinterpret_cast<floatx4*>(
                a.h + blockIdx.y * a.split_stride + static_cast<int64_t>(rows[slot]) * a.padded +
                rank) = v;
          }
        }
      }
    }
    __syncthreads();
  }
}

struct ExpandArgs {
  Rows rows;
  const float* h; // [splits, T, padded]
  float* h_sum;   // null, or where its sum stays: [T, padded]
  int64_t split_stride;
  int splits, padded;
  const void* b; // [adapters, N, r]
  int64_t b_stride, b_row;
  int N, r;
  const void* y; // [T, N], or null
  int64_t y_stride;
  void* out; // [T, N]
  int columns; // of a workgroup: a multiple of 256
  int tile;
};

// Four ranks of the sum of a token's parts, in order
__device__ __forceinline__ floatx4 sum_of_parts(const float* p, int splits, int64_t split_stride) {
  floatx4 v = *reinterpret_cast<const floatx4*>(p);
  for (int s = 1; s < splits; s += 5) { // (five asked for at once; 16 parts at most)
    floatx4 part[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      part[i] = *reinterpret_cast<const floatx4*>(p + min(s + i, splits - 1) * split_stride);
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      if (s + i < splits) {
        v += part[i];
      }
    }
  }
  return v;
}

// Eight ranks of a token's h times `by`: the first, second or third of the numbers of the type whose
// sum it is; float32: four, as they are
template <typename T>
__device__ __forceinline__ uint4 rank_operand(const float (&v)[kPer<T>], int part, float by) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(uint4, make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float of[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = v[2 * i + j] * by;
        const float upper = round_to<T>(x);
        const float rest = fabsf(upper) < INFINITY ? x - upper : 0.0f; // (of what is finite)
        const float lower = round_to<T>(rest);
        of[j] = part == 0 ? upper : part == 1 ? lower : rest - lower;
      }
      w[i] = pack2<T>(of[0], of[1]);
    }
    return uint4{w[0], w[1], w[2], w[3]};
  }
}

template <typename T>
union Part { // 16 bytes of a row
  uint4 u;
  T e[kPer<T>];
};
template <typename T, bool kAligned>
__device__ __forceinline__ void store_part(T* row, int n, int end, const Part<T>& v) {
  if constexpr (kAligned) {
    if (n < end) {
      *reinterpret_cast<uint4*>(row + n) = v.u;
    }
  } else if (n + kPer<T> <= end) {
    __builtin_memcpy(row + n, &v.u, 16);
  } else {
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) {
      if (n + k < end) {
        row[n + k] = v.e[k];
      }
    }
  }
}

// (128 ranks: within the registers of two workgroups a CU.  With one, 4110 tokens to 1001 columns in bfloat16
// take 42 us instead of 31)
template <typename T, int kGroups, int kChunks, bool kAligned, bool kAdd>
__global__ __launch_bounds__(256, kChunks == 8 ? 2 : 1) void expand_kernel(const ExpandArgs a) {
  constexpr int kPitch = 16 * kChunks + 4; // (rows of neighbouring tokens four banks apart)
  constexpr int kParts = 16 / kPer<T>;     // of a lane's results
  __shared__ int rows[kFew];
  __shared__ alignas(16) float held[16 * kGroups][kPitch];
  int adapter;
  const int count = find_rows(a.rows, blockIdx.x, a.tile, rows, &adapter);
  if (count == 0) {
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15;
  const int quarter = lane >> 4;
  const T* y = static_cast<const T*>(a.y);
  T* out = static_cast<T*>(a.out);
  const int n_block = blockIdx.y * a.columns;
  const int n_end = min(a.N, n_block + a.columns);
  if (adapter < 0) { // y as it is
    const int units = (n_end - n_block + kPer<T> - 1) / kPer<T>;
    for (int n = threadIdx.x; n < count * units; n += 256) {
      const int t = n / units;
      const int at = n_block + (n - t * units) * kPer<T>;
      const int64_t row = rows[t];
      Part<T> v;
      v.u = kAdd ? operand<T, kAligned>(y + row * a.y_stride, at, a.N) : uint4{0, 0, 0, 0};
      store_part<T, kAligned>(out + row * a.N, at, n_end, v);
    }
    return;
  }
  // An instruction has 16 ranks (float32), 32, or 16 of the first parts and the same of the second
  // (bfloat16: then of the third, and nothing); of those the lane has kPer from rank_of on
  constexpr bool kWhole = sizeof(T) == 2 && kChunks > 1;
  constexpr int kParted = sizeof(T) == 4 ? 1 : std::is_same_v<T, bf16_t> ? 3 : 2;
  constexpr int kTerms = sizeof(T) == 4 || kWhole ? kParted : kParted - 1;
  constexpr int kSteps = kWhole ? kChunks / 2 : kChunks;
  constexpr int kRanks = kWhole ? 32 : 16;
  const int rank_of = sizeof(T) == 4 ? 4 * quarter : kWhole ? 8 * quarter : 8 * (quarter & 1);
  const T* b = static_cast<const T*>(a.b) + adapter * a.b_stride;
  const int n_begin = n_block + 64 * wave;
  // Of 64 columns a lane's results are 16 bytes of neighbours, the four quarters' side by side: row
  // 4 q + i of tile j is column 4 V (j / t) + V q + 4 (j % t) + i, V values in 16 bytes, t = V / 4
  constexpr int kTiles = kPer<T> / 4;
  uint4 weights[4][kSteps];
  const auto ask_b = [&](int n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 4 * kPer<T> * (j / kTiles) + kPer<T> * (column >> 2) + 4 * (j % kTiles) +
          (column & 3);
      const T* b_row = b + min(n, a.N - 1) * a.b_row;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        if constexpr (kAligned) { // (r is a multiple of what is read)
          const int k = kRanks * c + rank_of;
          const uint4 v = operand<T, true, true>(b_row, min(k, a.r - kPer<T>), a.r);
          weights[j][c] = k < a.r ? v : uint4{0, 0, 0, 0};
        } else {
          weights[j][c] = operand<T, false>(b_row, kRanks * c + rank_of, a.r);
        }
      }
    }
  };
  for (int base = 0; base < count; base += 16 * kGroups) {
    const int mine = min(16 * kGroups, count - base);
    const bool works = n_begin < n_end;
    if (works) {
      ask_b(n_begin);
    }
    int64_t row[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      row[i] = rows[base + min(16 * i + column, mine - 1)];
    }
    Part<T> next[kGroups][kParts];
    const auto ask_y = [&](int n0) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const int n = n0 + kPer<T> * (quarter + 4 * p);
          if constexpr (kAligned) { // (what is past the end is not stored)
            next[i][p].u =
                operand<T, true, true>(y + row[i] * a.y_stride, min(n, a.N - kPer<T>), a.N);
          } else {
            next[i][p].u = operand<T, false>(y + row[i] * a.y_stride, n, a.N);
          }
        }
      }
    };
    if (kAdd && works) {
      ask_y(n_begin);
    }
    // the tokens' h, the sum of its parts, for all four wavefronts
    const int quads = a.padded / 4;
    for (int n = threadIdx.x; n < mine * quads; n += 256) {
      const int t = n / quads;
      const int k = 4 * (n - t * quads);
      const int64_t at = static_cast<int64_t>(rows[base + t]) * a.padded + k;
      const floatx4 v = sum_of_parts(a.h + at, a.splits, a.split_stride);
      *reinterpret_cast<floatx4*>(&held[t][k]) = v;
      if (a.h_sum != nullptr && blockIdx.y == 0) {
        *reinterpret_cast<floatx4*>(a.h_sum + at) = v;
      }
    }
    __syncthreads();
    uint4 h[kGroups][kSteps][kTerms];
    float back[kGroups]; // float16: what h was divided by
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int t = min(16 * i + column, mine - 1);
      float v[kSteps][kPer<T>];
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
#pragma unroll
        for (int j = 0; j < kPer<T>; j += 4) {
          floatx4 q = {0.0f, 0.0f, 0.0f, 0.0f};
          if (kRanks * c + rank_of < a.padded) {
            q = *reinterpret_cast<const floatx4*>(&held[t][kRanks * c + rank_of + j]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[c][j + k] = q[k];
            const float m = fabsf(q[k]);
            most = m < INFINITY ? fmaxf(most, m) : most;
          }
        }
      }
      float by = 1.0f;
      back[i] = 1.0f;
      if constexpr (std::is_same_v<T, f16_t>) {
        most = fmaxf(most, __shfl_xor(most, 16, 64)); // (the other ranks' lanes)
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        // 2^13 over the power of two below the largest: exponents 13 - e and e - 13
        const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
        const int up = min(max(13 - e, -100), 100);
        by = most > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 + up) << 23) : 1.0f;
        back[i] = most > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 - up) << 23) : 1.0f;
      }
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
#pragma unroll
        for (int t = 0; t < kTerms; ++t) {
          h[i][c][t] = rank_operand<T>(v[c], kTerms == kParted ? t : t == 1 ? 2 : quarter >= 2, by);
          if (kTerms < kParted && t == 1 && quarter >= 2) {
            h[i][c][t] = uint4{0, 0, 0, 0};
          }
        }
      }
    }
    const auto columns = [&](int n0, auto more) {
      floatx4 sum[kGroups][4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
#pragma unroll
            for (int t = 0; t < kTerms; ++t) {
              multiply<T>(weights[j][c], h[i][c][t], sum[i][j]);
            }
          }
        }
      }
      Part<T> v[kGroups][kParts];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          v[i][p] = next[i][p];
        }
      }
      if constexpr (more.value) {
        ask_b(n0 + 256);
        if constexpr (kAdd) {
          ask_y(n0 + 256);
        }
      }
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
#pragma unroll
          for (int k = 0; k < kPer<T>; ++k) {
            const float s = sum[i][kTiles * p + k / 4][k % 4] * back[i];
            v[i][p].e[k] = from_f32<T>(kAdd ? to_f32(v[i][p].e[k]) + s : s);
          }
          if (16 * i + column < mine) {
            store_part<T, kAligned>(
                out + row[i] * a.N, n0 + kPer<T> * (quarter + 4 * p), a.N, v[i][p]);
          }
        }
      }
    };
    if (works) {
      int n0 = n_begin;
      for (; n0 + 256 < n_end; n0 += 256) {
        columns(n0, std::true_type{});
      }
      columns(n0, std::false_type{});
    }
    __syncthreads(); // (the next tokens' h)
  }
}

// ---------------------------------------------------------------- grouping
struct GroupArgs {
  const int32_t* indices;
  int n, adapters, span;
  int tile, segment; // rows of a tile; of a run of tokens of the adapters' gradients (0: none)
  int32_t* order;
  Tile* tiles;
  Tile* segments;
  int32_t* counts; // number of tiles, of segments
  int32_t* slots;  // [adapters][2]: first partial sum, how many; -1: nothing to join
};

constexpr int kGroupWaves = 8;

// One workgroup; wavefront w has entries [w, w + 1) * run.  LDS: (wavefronts + 5) (adapters + 1)
// numbers.
__global__ __launch_bounds__(64 * kGroupWaves) void group_kernel(const GroupArgs a) {
  extern __shared__ int32_t before[]; // [wave][adapter], the last "adapter" is none
  // of each: first entry, tile, segment and partial sum; entries
  int32_t* places = before + kGroupWaves * (a.adapters + 1);
  int32_t* totals = places + 4 * (a.adapters + 1);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int buckets = a.adapters + 1;
  for (int i = threadIdx.x; i < kGroupWaves * buckets; i += 64 * kGroupWaves) {
    before[i] = 0;
  }
  __syncthreads();
  const int run = (a.n + kGroupWaves * 64 - 1) / (kGroupWaves * 64) * 64;
  volatile int32_t* mine = before + wave * buckets; // (lane 0 writes what all read)
  const auto bucket = [&](int i) {
    const int of = i < a.n ? (a.indices == nullptr ? 0 : a.indices[i]) : -1;
    return static_cast<uint32_t>(of) < static_cast<uint32_t>(a.adapters) ? of : a.adapters;
  };
  const int last = min(a.n, (wave + 1) * run);
  // Of 64 entries those that are alike take their places at once: how many are before each
  const auto each = [&](auto&& place) {
    for (int first = wave * run; first < last; first += 64) {
      const int i = first + lane;
      const int of = bucket(i);
      uint64_t left = __ballot(i < last);
      while (left != 0) {
        const int leader = __ffsll(static_cast<unsigned long long>(left)) - 1;
        const int which = __builtin_amdgcn_readlane(of, leader);
        const uint64_t same = __ballot(of == which) & left;
        place(i, which, same);
        left &= ~same;
      }
    }
  };
  each([&](int, int which, uint64_t same) {
    if (lane == 0) {
      mine[which] = mine[which] + __popcll(same);
    }
  });
  __syncthreads();
  // Sums over wavefronts, then over buckets, by the first wavefront: of entries, tiles, segments
  // and partial sums
  if (wave == 0) {
    int entry = 0;
    int tile = 0;
    int segment = 0;
    int slot = 0;
    for (int first = 0; first < buckets; first += 64) {
      const int of = first + lane;
      int sum = 0;
      if (of < buckets) {
        for (int w = 0; w < kGroupWaves; ++w) {
          const int c = before[w * buckets + of];
          before[w * buckets + of] = sum;
          sum += c;
        }
      }
      const int rows = sum * a.span;
      const int tiles = (rows + a.tile - 1) / a.tile;
      const int segments =
          a.segment == 0 || of >= a.adapters ? 0 : (rows + a.segment - 1) / a.segment;
      const int slots = segments > 1 ? segments : 0;
      int up[4] = {sum, tiles, segments, slots};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        for (int d = 1; d < 64; d *= 2) {
          const int other = __shfl_up(up[i], d, 64);
          up[i] += lane >= d ? other : 0;
        }
      }
      const int at = entry + up[0] - sum;
      if (of < buckets) {
        for (int w = 0; w < kGroupWaves; ++w) {
          before[w * buckets + of] += at;
        }
        places[4 * of] = at;
        places[4 * of + 1] = tile + up[1] - tiles;
        places[4 * of + 2] = segment + up[2] - segments;
        places[4 * of + 3] = slots > 0 ? slot + up[3] - slots : -1;
        totals[of] = sum;
        if (a.segment != 0 && of < a.adapters) {
          a.slots[2 * of] = segments == 1 ? -1 : slot + up[3] - slots;
          a.slots[2 * of + 1] = slots;
        }
      }
      entry += __shfl(up[0], 63, 64);
      tile += __shfl(up[1], 63, 64);
      segment += __shfl(up[2], 63, 64);
      slot += __shfl(up[3], 63, 64);
    }
    if (lane == 0) {
      a.counts[0] = tile;
      a.counts[1] = segment;
    }
  }
  __syncthreads();
  // the tiles and segments of a bucket by a wavefront
  for (int of = wave; of < buckets; of += kGroupWaves) {
    const int rows = totals[of] * a.span;
    const int from = places[4 * of] * a.span;
    const int adapter = of < a.adapters ? of : -1;
    for (int i = lane; i * a.tile < rows; i += 64) {
      a.tiles[places[4 * of + 1] + i] =
          Tile{adapter, from + i * a.tile, min(a.tile, rows - i * a.tile), -1};
    }
    if (a.segment != 0 && adapter >= 0) {
      const int slot = places[4 * of + 3];
      for (int i = lane; i * a.segment < rows; i += 64) {
        a.segments[places[4 * of + 2] + i] =
            Tile{adapter, from + i * a.segment, min(a.segment, rows - i * a.segment),
                 slot < 0 ? -1 : slot + i};
      }
    }
  }
  each([&](int i, int which, uint64_t same) {
    const int at = mine[which]; // (read by all before one writes: they are one wavefront)
    if (same >> lane & 1) {
      a.order[at + __popcll(same & ((uint64_t{1} << lane) - 1))] = i;
    }
    if (lane == 0) {
      mine[which] = at + __popcll(same);
    }
  });
}

// ---------------------------------------------------------------- turned weights
struct TurnArgs {
  struct {
    const void* from; // [adapters, R, C]
    void* to;         // [adapters, C, padded]: padded >= R, zeros behind
    int R, C, padded, across; // blocks of 64 columns
    int64_t blocks;
  } of[2]; // B, and A (no blocks where it is not wanted)
  const int32_t* slots; // of adapters that are not in use: {0 or more, 0}
};
template <typename T>
__global__ __launch_bounds__(256) void turn_kernel(const TurnArgs a) {
  __shared__ T tile[64][65 + (sizeof(T) == 2 ? 1 : 0)];
  const int adapter = blockIdx.y;
  if (a.slots[2 * adapter] >= 0 && a.slots[2 * adapter + 1] == 0) {
    return;
  }
  const bool second = blockIdx.x >= a.of[0].blocks;
  const auto& m = a.of[second];
  const int block = blockIdx.x - (second ? static_cast<int>(a.of[0].blocks) : 0);
  const int c0 = block % m.across * 64;
  const int r0 = block / m.across * 64;
  const T* from = static_cast<const T*>(m.from) + static_cast<int64_t>(adapter) * m.R * m.C;
  T* to = static_cast<T*>(m.to) + static_cast<int64_t>(adapter) * m.C * m.padded;
  // (a matrix of few columns or rows has few here, too)
  const int columns = min(64, m.C - c0);
  const int rows = min(64, m.padded - r0);
  for (int n = threadIdx.x; n < rows * columns; n += 256) {
    const int y = n / columns;
    const int x = n - y * columns;
    tile[y][x] =
        r0 + y < m.R ? from[static_cast<int64_t>(r0 + y) * m.C + c0 + x] : static_cast<T>(0.0f);
  }
  __syncthreads();
  for (int n = threadIdx.x; n < rows * columns; n += 256) {
    const int y = n / rows;
    const int x = n - y * rows;
    to[static_cast<int64_t>(c0 + y) * m.padded + r0 + x] = tile[x][y];
  }
}

// ---------------------------------------------------------------- sums over tokens
// bfloat16 numbers whose sum n values are, of which the first of a pair is in the lower half: each is
// what is left without its last 16 bits.  (Rounded ones take half as many instructions again.)
template <int kParts, int n>
__device__ __forceinline__ void cut(const float (&v)[n], uint32_t (&w)[kParts][n / 2]) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    most = fmaxf(most, fabsf(v[i]));
  }
  const bool infinite = __any(most == INFINITY); // (of infinity nothing is left; NaN stays NaN)
#pragma unroll
  for (int i = 0; i < n / 2; ++i) {
    float x = v[2 * i];
    float y = v[2 * i + 1];
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const uint32_t x_bits = __float_as_uint(x);
      const uint32_t y_bits = __float_as_uint(y);
      w[k][i] = __builtin_amdgcn_perm(y_bits, x_bits, 0x07060302);
      x -= __uint_as_float(x_bits & 0xffff0000u);
      y -= __uint_as_float(y_bits & 0xffff0000u);
      if (k == 0 && infinite) {
        x = fabsf(v[2 * i]) == INFINITY ? 0.0f : x;
        y = fabsf(v[2 * i + 1]) == INFINITY ? 0.0f : y;
      }
    }
  }
}

struct TokenSum {
  const float* p; // [splits, T, padded]: h or g
  int splits;
  const void* q; // [T, W]: dout or x
  int64_t q_stride;
  int W;
  int across;   // blocks of columns; 0: this sum is not wanted
  float* parts; // [slots, r, W]
  void* out;    // [adapters, r, W], or [adapters, W, r] (turned)
  int turned;
};
struct TokenArgs {
  Rows rows; // tiles: the segments
  int64_t split_stride;
  int padded, r;
  TokenSum of[2]; // dB, dA
};

constexpr int kTokens = 32;  // of a tile in LDS
constexpr int kColumns = 256;
constexpr int kMostSegment = 2048;

// The result's rows are columns of q, its columns are ranks: kChunks of 16.  A wavefront has 64
// columns of q, in the order of expand_kernel.  Two tiles of 32 tokens in LDS: one is read while
// the other's loads are in flight.
template <typename T, int kChunks, bool kAligned>
__global__ __launch_bounds__(256) void token_kernel(const TokenArgs a) {
  // (rows a quarter of the banks apart, so that the four rows of a transposed read do not meet)
  constexpr int kPitch = kColumns + 32 / sizeof(T);
  __shared__ alignas(16) T q_tile[2][kTokens][kPitch];
  __shared__ alignas(16) float p_tile[2][kTokens][16 * kChunks + 4];
  __shared__ int rows[kMostSegment];
  if (static_cast<int>(blockIdx.x) >= *a.rows.n_tiles) {
    return;
  }
  const Tile tile = a.rows.tiles[blockIdx.x];
  const bool second = static_cast<int>(blockIdx.y) >= a.of[0].across;
  const TokenSum& m = a.of[second];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15;
  const int quarter = lane >> 4;
  const int c0 = (blockIdx.y - (second ? a.of[0].across : 0)) * kColumns;
  const int rank0 = blockIdx.z * kChunks * 16;
  for (int n = threadIdx.x; n < tile.rows; n += 256) {
    rows[n] = a.rows.row(tile.first + n);
  }
  __syncthreads();
  floatx4 sum[4][kChunks] = {};
  constexpr int kUnits = kColumns / kPer<T>;
  constexpr int kLoads = kTokens * kUnits / 256;
  constexpr int kQuads = kTokens * 4 * kChunks; // of p
  constexpr int kPLoads = (kQuads + 255) / 256;
  uint4 got[kLoads];
  floatx4 p_got[kPLoads];
  const auto ask = [&](int first) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = i * 256 + threadIdx.x;
      const int t = first + n / kUnits;
      const int c = c0 + (n % kUnits) * kPer<T>;
      got[i] = uint4{0, 0, 0, 0};
      if (t < tile.rows && c < m.W) {
        got[i] = operand<T, kAligned>(
            static_cast<const T*>(m.q) + rows[t] * m.q_stride, c, m.W);
      }
    }
#pragma unroll
    for (int i = 0; i < kPLoads; ++i) {
      const int n = i * 256 + threadIdx.x;
      const int t = first + n / (4 * kChunks);
      const int k = rank0 + n % (4 * kChunks) * 4;
      p_got[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      if (n < kQuads && t < tile.rows && k < a.padded) {
        p_got[i] = sum_of_parts(
            m.p + static_cast<int64_t>(rows[t]) * a.padded + k, m.splits, a.split_stride);
      }
    }
  };
  ask(0);
  int which = 0;
  for (int first = 0; first < tile.rows; first += kTokens, which ^= 1) {
    // (the other of the two tiles may still be read)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = i * 256 + threadIdx.x;
      *reinterpret_cast<uint4*>(&q_tile[which][n / kUnits][(n % kUnits) * kPer<T>]) = got[i];
    }
#pragma unroll
    for (int i = 0; i < kPLoads; ++i) {
      const int n = i * 256 + threadIdx.x;
      if (n < kQuads) {
        *reinterpret_cast<floatx4*>(
            &p_tile[which][n / (4 * kChunks)][n % (4 * kChunks) * 4]) = p_got[i];
      }
    }
    __syncthreads();
    if (first + kTokens < tile.rows) {
      ask(first + kTokens);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int t0 = 0; t0 < kTokens; t0 += 4) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[j] = q_tile[which][t0 + quarter]
                      [64 * wave + 16 * j + column];
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const float p = p_tile[which][t0 + quarter][16 * c + column];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j], p, sum[j][c], 0, 0, 0);
          }
        }
      }
    } else {
      // In bfloat16, whose range is float32's: p as three numbers, a float16 q as two, both exactly
      uint4 q[4][std::is_same_v<T, bf16_t> ? 1 : 2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // A lane of sixteen gives the place of 4 columns of a token and gets 4 tokens of a column
        uint32_t w[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int t = 8 * quarter + 4 * half + (column >> 2);
          const uint32_t at =
              lds_address(
              &q_tile[which][t][64 * wave + 32 * (j / 2) + 8 * (column & 3) + 4 * (j % 2)]);
          const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) shortx4*)(LdsBytes)(uintptr_t)at);
          const uint2 u = __builtin_bit_cast(uint2, x);
          w[2 * half] = u.x;
          w[2 * half + 1] = u.y;
        }
        if constexpr (std::is_same_v<T, bf16_t>) {
          q[j][0] = uint4{w[0], w[1], w[2], w[3]};
        } else {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = half_of<f16_t>(w[i / 2], i % 2);
          }
          uint32_t part[2][4];
          cut(v, part);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            q[j][k] = uint4{part[k][0], part[k][1], part[k][2], part[k][3]};
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = p_tile[which][8 * quarter + i][16 * c + column];
        }
        uint32_t w[3][4];
        cut(v, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const uint4 p = uint4{w[k][0], w[k][1], w[k][2], w[k][3]};
            sum[j][c] = mfma16<bf16_t>(q[j][0], p, sum[j][c]);
            if constexpr (std::is_same_v<T, f16_t>) {
              sum[j][c] = mfma16<bf16_t>(q[j][1], p, sum[j][c]);
            }
          }
        }
      }
    }
  }
  // A lane has 16 bytes of neighbouring columns of q (float32: 4, else 8) for rank 16 c + column
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int rank = rank0 + 16 * c + column;
    if (rank >= a.r) {
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int kTiles = kPer<T> / 4;
      const int n = c0 + 64 * wave + 4 * kPer<T> * (j / kTiles) + kPer<T> * quarter + 4 * (j % kTiles);
      const floatx4 v = sum[j][c];
      if (tile.slot >= 0) {
        float* to = m.parts + (static_cast<int64_t>(tile.slot) * a.r + rank) * m.W + n;
        if (kAligned && n < m.W) { // (W is a multiple of 4 at least, the parts are aligned)
          *reinterpret_cast<floatx4*>(to) = v;
          continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n + i < m.W) {
            to[i] = v[i];
          }
        }
        continue;
      }
      T* out = static_cast<T*>(m.out) + static_cast<int64_t>(tile.adapter) * a.r * m.W;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n + i < m.W) {
          out[m.turned ? static_cast<int64_t>(n + i) * a.r + rank
                       : static_cast<int64_t>(rank) * m.W + n + i] = from_f32<T>(v[i]);
        }
      }
    }
  }
}

struct JoinArgs {
  const int32_t* slots;
  int r;
  TokenSum of[2];
};
// Of an adapter's sum 16 ranks of 64 columns a workgroup, through LDS where the result is turned, so
// that a row's ranks are written side by side; zeros as they lie, 16 bytes a thread
constexpr int kJoined = 64;
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
  __shared__ float held[kJoined][17];
  const int adapter = blockIdx.z;
  const int first = a.slots[2 * adapter];
  const int count = a.slots[2 * adapter + 1];
  if (first < 0) {
    return;
  }
  const int blocks = a.of[0].across * (kColumns / kJoined);
  const bool second = static_cast<int>(blockIdx.x) >= blocks;
  const TokenSum& m = a.of[second];
  const int block = blockIdx.x - (second ? blocks : 0);
  T* out = static_cast<T*>(m.out) + static_cast<int64_t>(adapter) * a.r * m.W;
  if (count == 0) {
    const int all = a.r * m.W; // (2^29 at most)
    const int across = m.across * (kColumns / kJoined);
    const int from = (blockIdx.y * across + block) * 16 * kJoined;
    const int end = min(all, from + 16 * kJoined);
    for (int n = from + kPer<T> * threadIdx.x; n < end; n += 256 * kPer<T>) {
      Part<T> zero;
      zero.u = uint4{0, 0, 0, 0};
      store_part<T, false>(out, n, end, zero);
    }
    return;
  }
  const int c0 = block * kJoined;
  const int rank0 = blockIdx.y * 16;
  const int column = threadIdx.x & 63;
  const int ranks = min(16, a.r - rank0);
  const int wave = threadIdx.x >> 6;
  if (c0 + column < m.W) {
    // (four ranks a thread, of two parts at once)
    const int64_t part = static_cast<int64_t>(a.r) * m.W;
    const float* p = m.parts + first * part + static_cast<int64_t>(rank0) * m.W + c0 + column;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < count; s += 2) {
      float one[4];
      float two[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = static_cast<int64_t>(min(wave + 4 * j, ranks - 1)) * m.W;
        one[j] = p[s * part + at];
        two[j] = p[min(s + 1, count - 1) * part + at];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += one[j];
        v[j] += s + 1 < count ? two[j] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = wave + 4 * j;
      if (i >= ranks) {
        break;
      }
      if (m.turned) {
        held[column][i] = v[j];
      } else {
        out[static_cast<int64_t>(rank0 + i) * m.W + c0 + column] = from_f32<T>(v[j]);
      }
    }
  }
  if (m.turned) {
    __syncthreads();
    for (int n = threadIdx.x; n < 16 * kJoined; n += 256) {
      const int c = n / 16;
      const int i = n % 16;
      if (c0 + c < m.W && i < ranks) {
        out[static_cast<int64_t>(c0 + c) * a.r + rank0 + i] = from_f32<T>(held[c][i]);
      }
    }
  }
}
static_assert(kColumns % kJoined == 0);

// ---------------------------------------------------------------- plans
// Sizes of a call and where things lie in its workspace, in bytes
struct Plan {
  bool grouped;
  int tile; // rows of a tile
  int chunks;      // of 16 ranks in a workgroup of sums over tokens
  int rank_blocks; // workgroups side by side for more
  int shrink_chunks, shrink_blocks; // the same of shrink
  int padded;
  int most_tiles;
  int splits, per_split; // of K (forward) or N (gradients)
  int columns;           // of a workgroup of expand
  int segment, most_segments, most_slots;
  size_t order, tiles, counts, segments, slots, h, turned_a, turned_b, parts_a, parts_b, bytes;
  int padded_n;
};

struct Sizes {
  int64_t T;
  int n, adapters, r, K, N, dtype;
};

size_t claim(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) / 256 * 256;
  return here;
}

int round_up(int v, int to) {
  return (v + to - 1) / to * to;
}

Plan plan_of(const Sizes& s, bool gradients) {
  Plan p{};
  const size_t size = dtype_size(s.dtype);
  const int step = s.dtype == MLXROCM_FLOAT32 ? 16 : 32;
  p.grouped = gradients || s.n > kFew;
  p.padded = round_up(s.r, 16);
  const int chunks = p.padded / 16;
  p.chunks = chunks <= 1 ? 1 : chunks <= 2 ? 2 : chunks <= 4 ? 4 : 8;
  p.rank_blocks = (chunks + p.chunks - 1) / p.chunks;
  const bool few = s.T <= kFew;
  p.tile = few || p.chunks == 8 ? 16 : 32;
  const int64_t kinds = s.n < s.adapters + 1 ? s.n : s.adapters + 1;
  const int64_t tiles = p.grouped       ? s.T / p.tile + kinds
      : s.n == 1    ? (s.T + p.tile - 1) / p.tile
      : s.T == s.n ? s.n
                    : s.T / p.tile + kinds;
  p.most_tiles = static_cast<int>(tiles);
  // Parts of a sum until there are about two workgroups a CU.  us of a call with 16 outputs, with 1, 2,
  // 4, 8 parts: 8192 tokens of 14336 values to rank 16 (257 tiles) 60, 52, 57, 60, 4096 tokens of 4096
  // to rank 64 (132) 31, 32, 27, 24, 2000 tokens to rank 16 (63) 16, 11, 10, 10, 48 requests to rank 64
  // 21, 14, 10, 10.
  // Where 16 parts are not enough, fewer ranks a workgroup: 3 tokens of 14336 values to rank 128 of
  // three adapters, float32, 17 us instead of 29, one token of 4096 in bfloat16 9.4 instead of 12.1.
  p.shrink_chunks = p.chunks;
  p.shrink_blocks = p.rank_blocks;
  while (p.shrink_chunks > 1 && tiles * p.shrink_blocks * 16 < 480) {
    p.shrink_chunks /= 2;
    p.shrink_blocks = (chunks + p.shrink_chunks - 1) / p.shrink_chunks;
  }
  const int sum_over = gradients ? s.N : s.K;
  int splits = 1;
  while (splits < 16 && tiles * p.shrink_blocks * splits < 480 &&
         sum_over >= 2 * splits * 4 * step * 2) {
    splits *= 2;
  }
  p.per_split = round_up((sum_over + splits - 1) / splits, 8 * step);
  p.splits = (sum_over + p.per_split - 1) / p.per_split;
  const int out_columns = gradients ? s.K : s.N;
  p.columns = 256;
  while (p.columns < 1024 && tiles * ((out_columns + 2 * p.columns - 1) / (2 * p.columns)) >= 512) {
    p.columns *= 2;
  }
  size_t at = 0;
  if (p.grouped) {
    p.order = claim(at, sizeof(int32_t) * s.n);
    p.tiles = claim(at, sizeof(Tile) * p.most_tiles);
    p.counts = claim(at, sizeof(int32_t) * 2);
  }
  p.h = claim(at, sizeof(float) * p.splits * s.T * p.padded); // (gradients: g)
  if (gradients) {
    const int64_t blocks = (s.K + kColumns - 1) / kColumns + (s.N + kColumns - 1) / kColumns;
    // 640 workgroups, by tokens: 8192 tokens of 4096 values to 14336 by rank 16 290 us (320: 320, 1024: 302),
    // 16384 of 8192 to 1024 by rank 32 292 (320: 306).  At least 64 tokens, as parts are written and read
    // again; of rank 128 96 (64, 96, 128: 4110 tokens of 1024 to 1001, float16 204, 182, 185, to 1024 149,
    // 144, 141; 1400 of 2048 to 2048 by rank 256 192, 184, 185; 2048 of 2048 to 512 111, 101, 104).
    const int64_t segment = s.T * blocks * p.rank_blocks / 640 / kTokens * kTokens;
    const int least = p.chunks == 8 ? 96 : 64;
    p.segment =
        static_cast<int>(segment < least ? least : segment > kMostSegment ? kMostSegment : segment);
    p.most_segments = static_cast<int>(s.T / p.segment + kinds);
    p.most_slots = static_cast<int>(2 * (s.T / p.segment) + 1);
    p.segments = claim(at, sizeof(Tile) * p.most_segments);
    p.slots = claim(at, sizeof(int32_t) * 2 * s.adapters);
    p.padded_n = round_up(s.N, 16);
    p.turned_a = claim(at, size * s.adapters * s.K * p.padded);
    p.turned_b = claim(at, size * s.adapters * s.r * p.padded_n);
    p.parts_a = claim(at, sizeof(float) * p.most_slots * s.r * s.K);
    p.parts_b = claim(at, sizeof(float) * p.most_slots * s.r * s.N);
  }
  p.bytes = at;
  return p;
}

int check_sizes(const char* tag, const Sizes& s) {
  if (!valid_dtype(s.dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] unknown dtype %d", tag, s.dtype);
  }
  if (s.T < 0 || s.n < 0 || s.K < 1 || s.N < 1 || (s.n == 0 ? s.T != 0 : s.T % s.n != 0)) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d indices for %lld rows of %d and %d", tag, s.n,
        static_cast<long long>(s.T), s.K, s.N);
  }
  if (s.adapters < 1 || s.adapters > kMostAdapters || s.r < 1 || s.r > kMostRank) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d adapters of rank %d", tag, s.adapters, s.r);
  }
  if (s.T >= int64_t{1} << 24 || s.K >= 1 << 21 || s.N >= 1 << 21) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", tag);
  }
  return MLXROCM_OK;
}

bool aligned16(const void* p, int64_t stride, size_t size) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride) * size) % 16 == 0;
}

// fn(chunks, aligned) with both known to the compiler
template <typename F>
int by_chunks(int chunks, bool aligned, F&& fn) {
  const auto with = [&](auto is) {
    chunks == 1 ? fn(IntC<1>{}, is)
        : chunks == 2 ? fn(IntC<2>{}, is)
        : chunks == 4 ? fn(IntC<4>{}, is)
                      : fn(IntC<8>{}, is);
  };
  aligned ? with(std::true_type{}) : with(std::false_type{});
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

template <typename T>
int shrink(const ShrinkArgs& a, const Plan& p, bool aligned, hipStream_t stream) {
  const dim3 grid(p.most_tiles, p.splits, p.shrink_blocks);
  return by_chunks(p.shrink_chunks, aligned, [&](auto chunks, auto is) {
    constexpr int c = decltype(chunks)::value;
    constexpr bool al = decltype(is)::value;
    if constexpr (al && c <= 4) {
      if (p.tile == 32) {
        shrink_kernel<T, 2, c, al><<<grid, 256, 0, stream>>>(a);
        return;
      }
    }
    shrink_kernel<T, 1, c, al><<<grid, 256, 0, stream>>>(a); // (in several turns)
  });
}

template <typename T>
int expand(const ExpandArgs& a, const Plan& p, bool aligned, hipStream_t stream) {
  const dim3 grid(p.most_tiles, (a.N + p.columns - 1) / p.columns);
  const auto launch = [&](auto groups, auto chunks, auto is) {
    constexpr int g = decltype(groups)::value;
    constexpr int c = decltype(chunks)::value;
    constexpr bool al = decltype(is)::value;
    if (a.y != nullptr) {
      expand_kernel<T, g, c, al, true><<<grid, 256, 0, stream>>>(a);
    } else {
      expand_kernel<T, g, c, al, false><<<grid, 256, 0, stream>>>(a);
    }
  };
  const auto go = [&](auto chunks, auto is) {
    if constexpr (decltype(is)::value && decltype(chunks)::value <= 4) {
      if (p.tile == 32) {
        launch(IntC<2>{}, chunks, is);
        return;
      }
    }
    launch(IntC<1>{}, chunks, is);
  };
  if (p.padded > 128) {
    if (aligned) {
      go(IntC<16>{}, std::true_type{});
    } else {
      go(IntC<16>{}, std::false_type{});
    }
    MLXROCM_HIP_TRY(hipGetLastError());
    return MLXROCM_OK;
  }
  return by_chunks(p.chunks, aligned, go);
}

// Both sums in one launch if either can have 16 bytes at a time or neither, and their joins in one
template <typename T>
int token_sums(TokenArgs a, const Plan& p, const int32_t* slots, int adapters, hipStream_t stream) {
  const auto aligned = [](const TokenSum& m) {
    return aligned16(m.q, m.q_stride, sizeof(T)) && aligned16(nullptr, m.W, sizeof(T));
  };
  const auto launch = [&](const TokenArgs& k, bool is) {
    const dim3 grid(p.most_segments, k.of[0].across + k.of[1].across, p.rank_blocks);
    return by_chunks(p.chunks, is, [&](auto chunks, auto al) {
      token_kernel<T, decltype(chunks)::value, decltype(al)::value><<<grid, 256, 0, stream>>>(k);
    });
  };
  const bool is = aligned(a.of[a.of[0].across == 0]);
  const bool together = a.of[1].across == 0 || aligned(a.of[1]) == is;
  TokenArgs first = a;
  TokenArgs second = a;
  if (!together) {
    first.of[1].across = second.of[0].across = 0;
  }
  int status = launch(first, is);
  if (status == MLXROCM_OK && !together) {
    status = launch(second, !is);
  }
  if (status != MLXROCM_OK) {
    return status;
  }
  const JoinArgs j{slots, a.r, {a.of[0], a.of[1]}};
  const dim3 grid((a.of[0].across + a.of[1].across) * (kColumns / kJoined), (a.r + 15) / 16, adapters);
  join_kernel<T><<<grid, 256, 0, stream>>>(j);
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

int group(const GroupArgs& a, hipStream_t stream) {
  const size_t lds = sizeof(int32_t) * (kGroupWaves + 5) * (a.adapters + 1);
  group_kernel<<<1, 64 * kGroupWaves, lds, stream>>>(a);
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

Rows rows_of(const Sizes& s, const Plan& p, const int32_t* indices, char* ws) {
  Rows r{};
  r.indices = indices;
  r.n = s.n;
  r.adapters = s.adapters;
  r.span = Divisor(s.T / s.n);
  if (p.grouped) {
    r.order = reinterpret_cast<const int32_t*>(ws + p.order);
    r.tiles = reinterpret_cast<const Tile*>(ws + p.tiles);
    r.n_tiles = reinterpret_cast<const int32_t*>(ws + p.counts);
  }
  return r;
}

GroupArgs grouping(const Sizes& s, const Plan& p, const int32_t* indices, char* ws) {
  GroupArgs g{};
  g.indices = indices;
  g.n = s.n;
  g.adapters = s.adapters;
  g.span = static_cast<int>(s.T / s.n);
  g.tile = p.tile;
  g.segment = p.segment;
  g.order = reinterpret_cast<int32_t*>(ws + p.order);
  g.tiles = reinterpret_cast<Tile*>(ws + p.tiles);
  g.segments = reinterpret_cast<Tile*>(ws + p.segments);
  g.counts = reinterpret_cast<int32_t*>(ws + p.counts);
  g.slots = reinterpret_cast<int32_t*>(ws + p.slots);
  return g;
}

} // namespace

} // namespace mlxrocm

// The products of both directions: sums over `K` of rows of x and of weights [adapters, r, K],
// then of those and weights [adapters, N, ranks] (and y)
namespace mlxrocm {
namespace {

ShrinkArgs shrinking(const Sizes& s, const Plan& p, const Rows& rows, float* h) {
  ShrinkArgs a{};
  a.rows = rows;
  a.h = h;
  a.split_stride = s.T * p.padded;
  a.r = s.r;
  a.padded = p.padded;
  a.per_split = p.per_split;
  a.tile = p.tile;
  return a;
}

ExpandArgs expanding(const Sizes& s, const Plan& p, const Rows& rows, const float* h) {
  ExpandArgs a{};
  a.rows = rows;
  a.h = h;
  a.split_stride = s.T * p.padded;
  a.splits = p.splits;
  a.padded = p.padded;
  a.columns = p.columns;
  a.tile = p.tile;
  return a;
}

} // namespace
} // namespace mlxrocm

extern "C" size_t mlxrocm_adapter_matmul_workspace_size(
    int64_t rows, int n_indices, int adapters, int rank, int K, int N, int dtype) {
  using namespace mlxrocm;
  const Sizes s{rows, n_indices, adapters, rank, K, N, dtype};
  return check_sizes("adapter_matmul", s) != MLXROCM_OK || rows == 0 ? 0 : plan_of(s, false).bytes;
}

extern "C" size_t mlxrocm_adapter_matmul_h_size(
    int64_t rows, int n_indices, int adapters, int rank, int K, int N, int dtype) {
  using namespace mlxrocm;
  const Sizes s{rows, n_indices, adapters, rank, K, N, dtype};
  return check_sizes("adapter_matmul", s) != MLXROCM_OK
      ? 0
      : sizeof(float) * static_cast<size_t>(rows) * round_up(rank, 16);
}

extern "C" int mlxrocm_adapter_matmul(
    const void* x,
    const void* a,
    const void* b,
    const int32_t* indices,
    const float* scales,
    const void* y,
    void* out,
    float* h,
    int64_t rows,
    int n_indices,
    int adapters,
    int rank,
    int K,
    int N,
    int64_t x_stride,
    int64_t y_stride,
    float scale,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_adapter_matmul");
  using namespace mlxrocm;
  const char* tag = "adapter_matmul";
  const Sizes s{rows, n_indices, adapters, rank, K, N, dtype};
  const int rc = check_sizes(tag, s);
  if (rc != MLXROCM_OK || rows == 0) {
    return rc;
  }
  const Plan p = plan_of(s, false);
  if (out == nullptr || b == nullptr || x == nullptr || a == nullptr ||
      (indices == nullptr && n_indices != 1) || (p.bytes > 0 && workspace == nullptr)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer", tag);
  }
  if (workspace_bytes < p.bytes) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] workspace of %zu bytes, %zu needed", tag, workspace_bytes,
        p.bytes);
  }
  char* ws = static_cast<char*>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t size = dtype_size(dtype);
  if (p.grouped) {
    const int status = group(grouping(s, p, indices, ws), st);
    if (status != MLXROCM_OK) {
      return status;
    }
  }
  const Rows r = rows_of(s, p, indices, ws);
  float* parts = reinterpret_cast<float*>(ws + p.h);
  ShrinkArgs sa = shrinking(s, p, r, parts);
  sa.x = x;
  sa.x_stride = x_stride;
  sa.a = a;
  sa.a_stride = static_cast<int64_t>(rank) * K;
  sa.a_row = K;
  sa.scales = scales;
  sa.scale = scale;
  sa.K = K;
  ExpandArgs ea = expanding(s, p, r, parts);
  ea.h_sum = h;
  ea.b = b;
  ea.b_stride = static_cast<int64_t>(N) * rank;
  ea.b_row = rank;
  ea.N = N;
  ea.r = rank;
  ea.y = y;
  ea.y_stride = y_stride;
  ea.out = out;
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int status = shrink<T>(sa, p, aligned16(x, x_stride, size) && aligned16(a, K, size), st);
    if (status != MLXROCM_OK) {
      return status;
    }
    return expand<T>(
        ea, p,
        aligned16(b, rank, size) && aligned16(out, N, size) &&
            (y == nullptr || aligned16(y, y_stride, size)),
        st);
  });
}

extern "C" size_t mlxrocm_adapter_matmul_vjp_workspace_size(
    int64_t rows, int n_indices, int adapters, int rank, int K, int N, int dtype) {
  using namespace mlxrocm;
  const Sizes s{rows, n_indices, adapters, rank, K, N, dtype};
  return check_sizes("adapter_matmul_vjp", s) != MLXROCM_OK || rows == 0 ? 0
                                                                        : plan_of(s, true).bytes;
}

extern "C" int mlxrocm_adapter_matmul_vjp(
    const void* x,
    const void* a,
    const void* b,
    const int32_t* indices,
    const float* scales,
    const float* h,
    const void* dout,
    void* dx,
    void* da,
    void* db,
    int64_t rows,
    int n_indices,
    int adapters,
    int rank,
    int K,
    int N,
    int64_t x_stride,
    int64_t dout_stride,
    float scale,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_adapter_matmul_vjp");
  using namespace mlxrocm;
  const char* tag = "adapter_matmul_vjp";
  const Sizes s{rows, n_indices, adapters, rank, K, N, dtype};
  const int rc = check_sizes(tag, s);
  if (rc != MLXROCM_OK || rows == 0) {
    return rc;
  }
  const Plan p = plan_of(s, true);
  if (x == nullptr || a == nullptr || b == nullptr || dout == nullptr ||
      (indices == nullptr && n_indices != 1) || (db != nullptr && h == nullptr) ||
      workspace == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer", tag);
  }
  if (workspace_bytes < p.bytes) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] workspace of %zu bytes, %zu needed", tag, workspace_bytes,
        p.bytes);
  }
  char* ws = static_cast<char*>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t size = dtype_size(dtype);
  const GroupArgs grouped = grouping(s, p, indices, ws);
  const int status = group(grouped, st);
  if (status != MLXROCM_OK) {
    return status;
  }
  const Rows r = rows_of(s, p, indices, ws);
  Rows runs = r;
  runs.tiles = grouped.segments;
  runs.n_tiles = grouped.counts + 1;
  float* g = reinterpret_cast<float*>(ws + p.h);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const auto turn = [&](bool both) {
      const auto tiles = [](int n) { return (n + 63) / 64; };
      TurnArgs ta{};
      ta.of[0] = {b, ws + p.turned_b, N, rank, p.padded_n, tiles(rank),
                  static_cast<int64_t>(tiles(rank)) * tiles(p.padded_n)};
      if (both) {
        ta.of[1] = {a, ws + p.turned_a, rank, K, p.padded, tiles(K),
                    static_cast<int64_t>(tiles(K)) * tiles(p.padded)};
      }
      ta.slots = grouped.slots;
      const dim3 grid(static_cast<unsigned>(ta.of[0].blocks + ta.of[1].blocks), adapters);
      turn_kernel<T><<<grid, 256, 0, st>>>(ta);
      return hipGetLastError();
    };
    const bool needs_g = dx != nullptr || da != nullptr;
    if (needs_g) {
      MLXROCM_HIP_TRY(turn(dx != nullptr));
      ShrinkArgs sa = shrinking(s, p, r, g);
      sa.x = dout;
      sa.x_stride = dout_stride;
      sa.a = ws + p.turned_b;
      sa.a_stride = static_cast<int64_t>(rank) * p.padded_n;
      sa.a_row = p.padded_n;
      sa.scales = scales;
      sa.scale = scale;
      sa.K = N;
      const int done = shrink<T>(
          sa, p, aligned16(dout, dout_stride, size) && static_cast<size_t>(N) * size % 16 == 0, st);
      if (done != MLXROCM_OK) {
        return done;
      }
    }
    // (right behind what has read dout already)
    if (da != nullptr || db != nullptr) {
      const auto across = [](const void* to, int W) {
        return to == nullptr ? 0 : (W + kColumns - 1) / kColumns;
      };
      TokenArgs k{};
      k.rows = runs;
      k.split_stride = rows * p.padded;
      k.padded = p.padded;
      k.r = rank;
      k.of[0] = {h, 1, dout, dout_stride, N, across(db, N), reinterpret_cast<float*>(ws + p.parts_b),
                 db, 1};
      k.of[1] = {g, p.splits, x, x_stride, K, across(da, K), reinterpret_cast<float*>(ws + p.parts_a),
                 da, 0};
      const int done = token_sums<T>(k, p, grouped.slots, adapters, st);
      if (done != MLXROCM_OK) {
        return done;
      }
    }
    if (dx != nullptr) {
      ExpandArgs ea = expanding(s, p, r, g);
      ea.b = ws + p.turned_a;
      ea.b_stride = static_cast<int64_t>(K) * p.padded;
      ea.b_row = p.padded;
      ea.N = K;
      ea.r = p.padded;
      ea.out = dx;
      const int done = expand<T>(ea, p, aligned16(dx, K, size), st);
      if (done != MLXROCM_OK) {
        return done;
      }
    }
    return static_cast<int>(MLXROCM_OK);
  });
}

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
//   group    the tokens by adapter, and the tiles of them (one workgroup).  Up to 64 single tokens
//            need none: the first token of an adapter finds the others by a vote.
//   shrink   h or g, in 32 bits.  The four wavefronts of a workgroup and, for few tokens, several
//            workgroups share a token's sum; the parts are added in one order by who reads them.
//   expand   out or dx.  16-bit types: h as the sum of two numbers of the type, in one instruction
//            of 32: sixteen ranks of the upper parts, then of the lower ones, against the same
//            sixteen columns of B twice.  So h keeps 16 bits (bfloat16) or 22, and the result's own
//            rounding is all that is seen.  float16: h counts a power of two that brings the
//            token's largest to 2^13.
//   turn     A and B with their two dimensions swapped, for the gradients: then g and dx are the
//            same two products.
//   tokens   dA and dB: sums over tokens, cut so that workgroups fill the card.
//   join     their parts, in order; zeros for adapters without tokens.
//
// No atomics: the same inputs give the same bits.
#include <cmath>

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kDecode = 64;        // single tokens that need no grouping
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
  const int32_t* order; // [n] by adapter; null: no grouping (decode, or one index)
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
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    if (r.tiles != nullptr) {
      const bool is = block < *r.n_tiles;
      const Tile t = r.tiles[is ? block : 0];
      if (is && lane < t.rows) {
        to[lane] = r.row(t.first + lane);
      }
      if (lane == 0) {
        found[0] = is ? t.rows : 0;
        found[1] = t.adapter;
      }
    } else if (r.n == 1) {
      const int first = block * tile;
      const int rows = min(tile, r.span.d - first);
      if (lane < rows) {
        to[lane] = first + lane;
      }
      if (lane == 0) {
        found[0] = rows;
        found[1] = r.adapter_of(0);
      }
    } else {
      const int of = lane < r.n ? r.adapter_of(lane) : -2;
      const int mine = __shfl(of, block, 64);
      const uint64_t same = __ballot(of == mine);
      if (of == mine) {
        to[__popcll(same & ((uint64_t{1} << lane) - 1))] = lane;
      }
      if (lane == 0) {
        found[0] = __ffsll(static_cast<unsigned long long>(same)) - 1 == block ? __popcll(same) : 0;
        found[1] = mine;
      }
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

// Elements k .. k + 15 / sizeof(T) of a row of n; what lies past its end is zero
template <typename T, bool kAligned>
__device__ __forceinline__ uint4 operand(const T* row, int k, int n) {
  if constexpr (kAligned) { // (n is a multiple)
    return k < n ? *reinterpret_cast<const uint4*>(row + k) : uint4{0, 0, 0, 0};
  } else {
    union {
      uint4 u;
      T e[kPer<T>];
    } raw;
#pragma unroll
    for (int i = 0; i < kPer<T>; ++i) {
      raw.e[i] = k + i < n ? row[k + i] : static_cast<T>(0.0f);
    }
    return raw.u;
  }
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

// kGroups groups of 16 tokens, kChunks of 16 ranks
template <typename T, int kGroups, int kChunks, bool kAligned>
__global__ __launch_bounds__(256) void shrink_kernel(const ShrinkArgs a) {
  __shared__ int rows[kDecode];
  __shared__ floatx4 parts[3][kGroups * kChunks][64];
  int adapter;
  const int count = find_rows(a.rows, blockIdx.x, a.tile, rows, &adapter);
  if (count == 0 || adapter < 0) {
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
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
    constexpr int kAhead = kChunks <= 2 ? 4 : 2; // steps whose operands are asked for at once
    for (int k0 = begin + wave * kStep<T>; k0 < end; k0 += kAhead * 4 * kStep<T>) {
      uint4 x[kAhead][kGroups];
      uint4 v[kAhead][kChunks];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const int k = k0 + s * 4 * kStep<T> + quarter * kPer<T>;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          x[s][i] = operand<T, kAligned>(x_row[i], k, end);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          v[s][c] = operand<T, kAligned>(w_row[c], k, end);
        }
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
            multiply<T>(v[s][c], x[s][i], sum[i][c]);
          }
        }
      }
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
            float4 v;
            v.x = rank < a.r ? s[0] * scale : 0.0f;
            v.y = rank + 1 < a.r ? s[1] * scale : 0.0f;
            v.z = rank + 2 < a.r ? s[2] * scale : 0.0f;
            v.w = rank + 3 < a.r ? s[3] * scale : 0.0f;
            *reinterpret_cast<float4*>(
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

// Eight (float32: four) ranks of a token's h: the sum of its parts, times `by`
template <typename T>
__device__ __forceinline__ uint4 rank_operand(const float (&v)[kPer<T>], int quarter, float by) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(uint4, make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float part[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = v[2 * i + j] * by;
        const float upper = round_to<T>(x);
        // (of what is not finite there is no lower part)
        part[j] = quarter < 2 ? upper : fabsf(upper) < INFINITY ? x - upper : 0.0f;
      }
      w[i] = pack2<T>(part[0], part[1]);
    }
    return uint4{w[0], w[1], w[2], w[3]};
  }
}

template <typename T, int kGroups, int kChunks, bool kAligned>
__global__ __launch_bounds__(256) void expand_kernel(const ExpandArgs a) {
  __shared__ int rows[kDecode];
  int adapter;
  const int count = find_rows(a.rows, blockIdx.x, a.tile, rows, &adapter);
  if (count == 0) {
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int column = lane & 15;
  const int quarter = lane >> 4;
  // first of the ranks of a chunk that the lane has
  const int rank_of = sizeof(T) == 4 ? 4 * quarter : 8 * (quarter & 1);
  const T* b = static_cast<const T*>(a.b) + adapter * a.b_stride;
  const int n_end = min(a.N, static_cast<int>(blockIdx.y + 1) * a.columns);
  for (int base = 0; base < count; base += 16 * kGroups) {
    int64_t row[kGroups];
    uint4 h[kGroups][kChunks];
    float back[kGroups]; // float16: what h was divided by
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      row[i] = rows[min(base + 16 * i + column, count - 1)];
      back[i] = 1.0f;
      if (adapter < 0) {
        continue;
      }
      float v[kChunks][kPer<T>];
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int j = 0; j < kPer<T>; ++j) {
          v[c][j] = 0.0f;
        }
        if (16 * c < a.padded) {
          const float* p = a.h + row[i] * a.padded + 16 * c + rank_of;
          for (int s = 0; s < a.splits; ++s, p += a.split_stride) {
#pragma unroll
            for (int j = 0; j < kPer<T>; j += 4) {
              const float4 q = *reinterpret_cast<const float4*>(p + j);
              v[c][j] += q.x;
              v[c][j + 1] += q.y;
              v[c][j + 2] += q.z;
              v[c][j + 3] += q.w;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kPer<T>; ++j) {
          const float m = fabsf(v[c][j]);
          most = m < INFINITY ? fmaxf(most, m) : most;
        }
      }
      float by = 1.0f;
      if constexpr (std::is_same_v<T, f16_t>) {
        most = fmaxf(most, __shfl_xor(most, 16, 64)); // (the other ranks' lanes)
        // 2^13 over the power of two below the largest: exponents 13 - e and e - 13
        const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
        const int up = min(max(13 - e, -100), 100);
        by = most > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 + up) << 23) : 1.0f;
        back[i] = most > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 - up) << 23) : 1.0f;
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        h[i][c] = rank_operand<T>(v[c], quarter, by);
      }
    }
    for (int n0 = blockIdx.y * a.columns + 64 * wave; n0 < n_end; n0 += 256) {
      // Columns 16 q + 4 j + i of the 64 are row 4 q + i of the j-th tile, so that a lane's
      // results are 16 neighbours
      floatx4 sum[kGroups][4] = {};
      if (adapter >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = min(n0 + 16 * (column >> 2) + 4 * j + (column & 3), a.N - 1);
          const T* b_row = b + n * a.b_row;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint4 v = operand<T, kAligned>(b_row, 16 * c + rank_of, a.r);
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
              multiply<T>(v, h[i][c], sum[i][j]);
            }
          }
        }
      }
      const int n = n0 + 16 * quarter;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (base + 16 * i + column >= count) {
          continue;
        }
        const T* y = a.y == nullptr ? nullptr : static_cast<const T*>(a.y) + row[i] * a.y_stride + n;
        T* out = static_cast<T*>(a.out) + row[i] * a.N + n;
#pragma unroll
        for (int part = 0; part < 16; part += kPer<T>) {
          union {
            uint4 u;
            T e[kPer<T>];
          } raw;
          raw.u = uint4{0, 0, 0, 0};
          if (y != nullptr) {
            raw.u = operand<T, kAligned>(y + part, 0, a.N - n - part);
          }
          if (adapter >= 0) {
#pragma unroll
            for (int k = 0; k < kPer<T>; ++k) {
              const float s = sum[i][(part + k) / 4][k % 4] * back[i];
              raw.e[k] = from_f32<T>(y == nullptr ? s : to_f32(raw.e[k]) + s);
            }
          }
          if constexpr (kAligned) {
            if (n + part < a.N) {
              *reinterpret_cast<uint4*>(out + part) = raw.u;
            }
          } else {
#pragma unroll
            for (int k = 0; k < kPer<T>; ++k) {
              if (n + part + k < a.N) {
                out[part + k] = raw.e[k];
              }
            }
          }
        }
      }
    }
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

// One workgroup; wavefront w has entries [w, w + 1) * run.  LDS: counts[wavefronts][adapters + 1].
__global__ __launch_bounds__(64 * kGroupWaves) void group_kernel(const GroupArgs a) {
  extern __shared__ int32_t before[]; // [wave][adapter], the last "adapter" is none
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
        const int adapter = of < a.adapters ? of : -1;
        for (int i = 0; i < tiles; ++i) {
          a.tiles[tile + up[1] - tiles + i] =
              Tile{adapter, at * a.span + i * a.tile, min(a.tile, rows - i * a.tile), -1};
        }
        for (int i = 0; i < segments; ++i) {
          a.segments[segment + up[2] - segments + i] =
              Tile{adapter, at * a.span + i * a.segment, min(a.segment, rows - i * a.segment),
                   slots > 0 ? slot + up[3] - slots + i : -1};
        }
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
  const void* from; // [adapters, R, C]
  void* to;         // [adapters, C, padded]: padded >= R, zeros behind
  int R, C, padded;
  const int32_t* slots; // of adapters that are not in use: {0 or more, 0}
};
template <typename T>
__global__ __launch_bounds__(256) void turn_kernel(const TurnArgs a) {
  __shared__ T tile[64][65 + (sizeof(T) == 2 ? 1 : 0)];
  const int adapter = blockIdx.z;
  if (a.slots[2 * adapter] >= 0 && a.slots[2 * adapter + 1] == 0) {
    return;
  }
  const int c0 = blockIdx.x * 64;
  const int r0 = blockIdx.y * 64;
  const T* from = static_cast<const T*>(a.from) + static_cast<int64_t>(adapter) * a.R * a.C;
  T* to = static_cast<T*>(a.to) + static_cast<int64_t>(adapter) * a.C * a.padded;
  const int x = threadIdx.x & 63;
  for (int i = threadIdx.x >> 6; i < 64; i += 4) {
    const bool is = r0 + i < a.R && c0 + x < a.C;
    tile[i][x] = is ? from[static_cast<int64_t>(r0 + i) * a.C + c0 + x] : static_cast<T>(0.0f);
  }
  __syncthreads();
  for (int i = threadIdx.x >> 6; i < 64; i += 4) {
    if (c0 + i < a.C && r0 + x < a.padded) {
      to[static_cast<int64_t>(c0 + i) * a.padded + r0 + x] = tile[x][i];
    }
  }
}

// ---------------------------------------------------------------- sums over tokens
struct TokenArgs {
  Rows rows; // tiles: the segments
  const float* p; // [splits, T, padded]: g or h
  int64_t split_stride;
  int splits, padded, r;
  const void* q; // [T, W]: x or dout
  int64_t q_stride;
  int W;
  float* parts; // [slots, r, W]
  void* out;    // [adapters, r, W], or [adapters, W, r] (turned)
  int turned;
};

constexpr int kTokens = 32;  // of a tile in LDS
constexpr int kColumns = 256;

// The result's rows are columns of q, its columns are ranks: kChunks of 16.  A wavefront has 64
// columns of q, in the order of expand_kernel.
template <typename T, int kChunks, bool kAligned>
__global__ __launch_bounds__(256) void token_kernel(const TokenArgs a) {
  // (rows a quarter of the banks apart, so that the four rows of a transposed read do not meet)
  constexpr int kPitch = kColumns + 32 / sizeof(T);
  __shared__ alignas(16) T q_tile[kTokens][kPitch];
  __shared__ float p_tile[kTokens][16 * kChunks + 4];
  if (static_cast<int>(blockIdx.x) >= *a.rows.n_tiles) {
    return;
  }
  const Tile tile = a.rows.tiles[blockIdx.x];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int column = lane & 15;
  const int quarter = lane >> 4;
  const int c0 = blockIdx.y * kColumns;
  const int rank0 = blockIdx.z * kChunks * 16;
  floatx4 sum[4][kChunks] = {};
  for (int first = 0; first < tile.rows; first += kTokens) {
    const int count = min(kTokens, tile.rows - first);
    constexpr int kUnits = kColumns / kPer<T>;
    uint4 got[kTokens * kUnits / 256];
#pragma unroll
    for (int i = 0; i < kTokens * kUnits / 256; ++i) {
      const int n = i * 256 + threadIdx.x;
      const int t = n / kUnits;
      const int c = c0 + (n % kUnits) * kPer<T>;
      got[i] = uint4{0, 0, 0, 0};
      if (t < count && c < a.W) {
        const int64_t row = a.rows.row(tile.first + first + t);
        got[i] = operand<T, kAligned>(static_cast<const T*>(a.q) + row * a.q_stride, c, a.W);
      }
    }
    __syncthreads(); // (the last tile has been read)
#pragma unroll
    for (int i = 0; i < kTokens * kUnits / 256; ++i) {
      const int n = i * 256 + threadIdx.x;
      *reinterpret_cast<uint4*>(&q_tile[n / kUnits][(n % kUnits) * kPer<T>]) = got[i];
    }
    for (int n = threadIdx.x; n < kTokens * 16 * kChunks; n += 256) {
      const int t = n / (16 * kChunks);
      const int k = n % (16 * kChunks);
      float v = 0.0f;
      if (t < count && rank0 + k < a.r) {
        const float* p =
            a.p + static_cast<int64_t>(a.rows.row(tile.first + first + t)) * a.padded + rank0 + k;
        for (int i = 0; i < a.splits; ++i) {
          v += p[i * a.split_stride];
        }
      }
      p_tile[t][k] = v;
    }
    __syncthreads();
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int t0 = 0; t0 < kTokens; t0 += 4) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[j] = q_tile[t0 + quarter][64 * wave + 16 * (column >> 2) + 4 * j + (column & 3)];
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const float p = p_tile[t0 + quarter][16 * c + column];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j], p, sum[j][c], 0, 0, 0);
          }
        }
      }
    } else {
      // In bfloat16, whose range is float32's: p as two numbers, a float16 q as two as well (exactly)
      uint4 p[2][kChunks];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        uint32_t w[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = p_tile[8 * quarter + 2 * i][16 * c + column];
          const float y = p_tile[8 * quarter + 2 * i + 1][16 * c + column];
          const float x_upper = round_to<bf16_t>(x);
          const float y_upper = round_to<bf16_t>(y);
          w[0][i] = pack2<bf16_t>(x_upper, y_upper);
          w[1][i] = pack2<bf16_t>(
              fabsf(x_upper) < INFINITY ? x - x_upper : 0.0f,
              fabsf(y_upper) < INFINITY ? y - y_upper : 0.0f);
        }
        p[0][c] = uint4{w[0][0], w[0][1], w[0][2], w[0][3]};
        p[1][c] = uint4{w[1][0], w[1][1], w[1][2], w[1][3]};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // A lane of sixteen gives the place of 4 columns of a token and gets 4 tokens of a column
        uint32_t w[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int t = 8 * quarter + 4 * half + (column >> 2);
          const uint32_t at =
              lds_address(&q_tile[t][64 * wave + 16 * (column & 3) + 4 * j]);
          const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) shortx4*)(LdsBytes)(uintptr_t)at);
          const uint2 u = __builtin_bit_cast(uint2, x);
          w[2 * half] = u.x;
          w[2 * half + 1] = u.y;
        }
        if constexpr (std::is_same_v<T, bf16_t>) {
          const uint4 q = uint4{w[0], w[1], w[2], w[3]};
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            sum[j][c] = mfma16<bf16_t>(q, p[0][c], sum[j][c]);
            sum[j][c] = mfma16<bf16_t>(q, p[1][c], sum[j][c]);
          }
        } else {
          uint32_t upper[4];
          uint32_t lower[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = half_of<f16_t>(w[i], 0);
            const float y = half_of<f16_t>(w[i], 1);
            const float x_upper = round_to<bf16_t>(x);
            const float y_upper = round_to<bf16_t>(y);
            upper[i] = pack2<bf16_t>(x_upper, y_upper);
            lower[i] = pack2<bf16_t>(
                fabsf(x_upper) < INFINITY ? x - x_upper : 0.0f,
                fabsf(y_upper) < INFINITY ? y - y_upper : 0.0f);
          }
          const uint4 q = uint4{upper[0], upper[1], upper[2], upper[3]};
          const uint4 rest = uint4{lower[0], lower[1], lower[2], lower[3]};
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            sum[j][c] = mfma16<bf16_t>(q, p[0][c], sum[j][c]);
            sum[j][c] = mfma16<bf16_t>(q, p[1][c], sum[j][c]);
            sum[j][c] = mfma16<bf16_t>(rest, p[0][c], sum[j][c]);
          }
        }
      }
    }
  }
  // A lane has 16 neighbouring columns of q for rank 16 c + column
  const int n = c0 + 64 * wave + 16 * quarter;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int rank = rank0 + 16 * c + column;
    if (rank >= a.r) {
      continue;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (n + i >= a.W) {
        continue;
      }
      const float v = sum[i / 4][c][i % 4];
      if (tile.slot >= 0) {
        a.parts[(static_cast<int64_t>(tile.slot) * a.r + rank) * a.W + n + i] = v;
      } else {
        T* out = static_cast<T*>(a.out) + static_cast<int64_t>(tile.adapter) * a.r * a.W;
        out[a.turned ? static_cast<int64_t>(n + i) * a.r + rank
                     : static_cast<int64_t>(rank) * a.W + n + i] = from_f32<T>(v);
      }
    }
  }
}

struct JoinArgs {
  const float* parts;
  const int32_t* slots;
  void* out;
  int r, W, turned;
};
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
  const int adapter = blockIdx.z;
  const int first = a.slots[2 * adapter];
  const int count = a.slots[2 * adapter + 1];
  const int n = blockIdx.x * 256 + threadIdx.x;
  const int rank = blockIdx.y;
  if (first < 0 || n >= a.W) {
    return;
  }
  float v = 0.0f;
  for (int s = 0; s < count; ++s) {
    v += a.parts[(static_cast<int64_t>(first + s) * a.r + rank) * a.W + n];
  }
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(adapter) * a.r * a.W;
  out[a.turned ? static_cast<int64_t>(n) * a.r + rank : static_cast<int64_t>(rank) * a.W + n] =
      from_f32<T>(v);
}

// ---------------------------------------------------------------- plans
// Sizes of a call and where things lie in its workspace, in bytes
struct Plan {
  bool grouped;
  int tile, groups;  // rows of a tile: 16 groups
  int chunks;        // of 16 ranks in a workgroup of shrink and of sums over tokens
  int rank_blocks;
  int padded;
  int most_tiles;
  int splits, per_split; // of K (forward) or N (gradients)
  int columns;           // of a workgroup of expand
  int segment, most_segments, most_slots;
  size_t order, tiles, counts, segments, slots, h, h_bytes, turned_a, turned_b, parts, bytes;
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
  const int64_t span = s.n == 0 ? 0 : s.T / s.n;
  const size_t size = dtype_size(s.dtype);
  const int step = s.dtype == MLXROCM_FLOAT32 ? 16 : 32;
  p.grouped = gradients || !(s.n == 1 || (span == 1 && s.n <= kDecode));
  p.padded = round_up(s.r, 16);
  const int chunks = p.padded / 16;
  p.chunks = chunks <= 1 ? 1 : chunks <= 2 ? 2 : chunks <= 4 ? 4 : 8;
  p.rank_blocks = (chunks + p.chunks - 1) / p.chunks;
  const bool few = s.T <= kDecode;
  p.groups = few || p.chunks == 8 ? 1 : 2;
  p.tile = 16 * p.groups;
  const int64_t kinds = s.n < s.adapters + 1 ? s.n : s.adapters + 1;
  const int64_t tiles = p.grouped ? s.T / p.tile + kinds
      : s.n == 1                  ? (s.T + p.tile - 1) / p.tile
                                  : s.n;
  p.most_tiles = static_cast<int>(tiles);
  // parts of a sum until there are two workgroups a CU, each with two steps of its wavefronts
  const int sum_over = gradients ? s.N : s.K;
  int splits = 1;
  while (splits < 16 && tiles * p.rank_blocks * splits < 512 &&
         sum_over >= 2 * splits * 4 * step * 2) {
    splits *= 2;
  }
  p.per_split = round_up((sum_over + splits - 1) / splits, 4 * step);
  p.splits = (sum_over + p.per_split - 1) / p.per_split;
  const int out_columns = gradients ? s.K : s.N;
  p.columns = 256;
  while (p.columns < 2048 && tiles * ((out_columns + 2 * p.columns - 1) / (2 * p.columns)) >= 2048) {
    p.columns *= 2;
  }
  size_t at = 0;
  if (p.grouped) {
    p.order = claim(at, sizeof(int32_t) * s.n);
    p.tiles = claim(at, sizeof(Tile) * p.most_tiles);
    p.counts = claim(at, sizeof(int32_t) * 2);
  }
  p.h_bytes = sizeof(float) * p.splits * s.T * p.padded;
  p.h = claim(at, p.h_bytes); // (gradients: g)
  if (gradients) {
    const int wide = s.K > s.N ? s.K : s.N;
    const int64_t blocks = (wide + kColumns - 1) / kColumns;
    int64_t segment = s.T * blocks * p.rank_blocks / 1024 / kTokens * kTokens;
    p.segment = static_cast<int>(segment < 64 ? 64 : segment > 4096 ? 4096 : segment);
    p.most_segments = static_cast<int>(s.T / p.segment + kinds);
    p.most_slots = static_cast<int>(2 * (s.T / p.segment) + 1);
    p.segments = claim(at, sizeof(Tile) * p.most_segments);
    p.slots = claim(at, sizeof(int32_t) * 2 * s.adapters);
    p.padded_n = round_up(s.N, 16);
    p.turned_a = claim(at, size * s.adapters * s.K * p.padded);
    p.turned_b = claim(at, size * s.adapters * s.r * p.padded_n);
    p.parts = claim(at, sizeof(float) * p.most_slots * s.r * wide);
  }
  p.bytes = at;
  return p;
}

int check_sizes(const char* tag, const Sizes& s) {
  if (!valid_dtype(s.dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] unknown dtype %d", tag, s.dtype);
  }
  if (s.T < 0 || s.n < 0 || s.K < 0 || s.N < 0 || (s.n == 0 ? s.T != 0 : s.T % s.n != 0)) {
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
  const dim3 grid(p.most_tiles, p.splits, p.rank_blocks);
  return by_chunks(p.chunks, aligned, [&](auto chunks, auto is) {
    constexpr int c = decltype(chunks)::value;
    constexpr bool al = decltype(is)::value;
    if (p.groups == 1) {
      shrink_kernel<T, 1, c, al><<<grid, 256, 0, stream>>>(a);
    } else if constexpr (c < 8) {
      shrink_kernel<T, 2, c, al><<<grid, 256, 0, stream>>>(a);
    }
  });
}

template <typename T>
int expand(const ExpandArgs& a, const Plan& p, bool aligned, hipStream_t stream) {
  const dim3 grid(p.most_tiles, (a.N + p.columns - 1) / p.columns);
  const auto go = [&](auto chunks, auto is) {
    constexpr int c = decltype(chunks)::value;
    constexpr bool al = decltype(is)::value;
    if (p.groups == 1) {
      expand_kernel<T, 1, c, al><<<grid, 256, 0, stream>>>(a);
    } else if constexpr (c < 8) {
      expand_kernel<T, 2, c, al><<<grid, 256, 0, stream>>>(a);
    }
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

template <typename T>
int token_sums(const TokenArgs& a, const Plan& p, bool aligned, hipStream_t stream) {
  const dim3 grid(p.most_segments, (a.W + kColumns - 1) / kColumns, p.rank_blocks);
  return by_chunks(p.chunks, aligned, [&](auto chunks, auto is) {
    token_kernel<T, decltype(chunks)::value, decltype(is)::value><<<grid, 256, 0, stream>>>(a);
  });
}

int group(const GroupArgs& a, hipStream_t stream) {
  const size_t lds = sizeof(int32_t) * kGroupWaves * (a.adapters + 1);
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
  return check_sizes("adapter_matmul", s) != MLXROCM_OK || rows == 0 ? 0 : plan_of(s, false).h_bytes;
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
  if ((N > 0 && (out == nullptr || b == nullptr)) || (K > 0 && (x == nullptr || a == nullptr)) ||
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
  if (h == nullptr) {
    h = reinterpret_cast<float*>(ws + p.h);
  }
  ShrinkArgs sa = shrinking(s, p, r, h);
  sa.x = x;
  sa.x_stride = x_stride;
  sa.a = a;
  sa.a_stride = static_cast<int64_t>(rank) * K;
  sa.a_row = K;
  sa.scales = scales;
  sa.scale = scale;
  sa.K = K;
  ExpandArgs ea = expanding(s, p, r, h);
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
    if (p.splits > 0) {
      const int status =
          shrink<T>(sa, p, aligned16(x, x_stride, size) && aligned16(a, K, size), st);
      if (status != MLXROCM_OK) {
        return status;
      }
    }
    if (N == 0) {
      return static_cast<int>(MLXROCM_OK);
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
  const Plan forward = plan_of(s, false);
  if ((K > 0 && (x == nullptr || a == nullptr)) || (N > 0 && (b == nullptr || dout == nullptr)) ||
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
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const auto turn = [&](const void* from, size_t to, int R, int C, int padded) {
      const TurnArgs ta{from, ws + to, R, C, padded, grouped.slots};
      const dim3 grid((C + 63) / 64, (padded + 63) / 64, adapters);
      turn_kernel<T><<<grid, 256, 0, st>>>(ta);
      return hipGetLastError();
    };
    const auto sums = [&](const float* from, int splits, const void* q, int64_t stride, int W,
                          void* to, int turned) {
      TokenArgs k{};
      k.rows = runs;
      k.p = from;
      k.split_stride = rows * p.padded;
      k.splits = splits;
      k.padded = p.padded;
      k.r = rank;
      k.q = q;
      k.q_stride = stride;
      k.W = W;
      k.parts = parts;
      k.out = to;
      k.turned = turned;
      const int done = token_sums<T>(
          k, p, aligned16(q, stride, size) && static_cast<size_t>(W) * size % 16 == 0, st);
      if (done != MLXROCM_OK) {
        return done;
      }
      const JoinArgs j{parts, grouped.slots, to, rank, W, turned};
      join_kernel<T><<<dim3((W + 255) / 256, rank, adapters), 256, 0, st>>>(j);
      MLXROCM_HIP_TRY(hipGetLastError());
      return static_cast<int>(MLXROCM_OK);
    };
    if (K > 0 && (dx != nullptr || da != nullptr)) {
      if (N > 0) {
        MLXROCM_HIP_TRY(turn(b, p.turned_b, N, rank, p.padded_n));
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
            sa, p,
            aligned16(dout, dout_stride, size) && static_cast<size_t>(N) * size % 16 == 0, st);
        if (done != MLXROCM_OK) {
          return done;
        }
      }
      if (dx != nullptr) {
        MLXROCM_HIP_TRY(turn(a, p.turned_a, rank, K, p.padded));
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
      if (da != nullptr) {
        const int done = sums(g, p.splits, x, x_stride, K, da, 0);
        if (done != MLXROCM_OK) {
          return done;
        }
      }
    }
    if (N > 0 && db != nullptr) {
      return sums(h, forward.splits, dout, dout_stride, N, db, 1);
    }
    return static_cast<int>(MLXROCM_OK);
  });
}

// attention_rows.h -- attention of many rows: workgroups of 128 rows, four waves of 32,
// over tiles of keys and values in LDS.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   s_ij = scale q_i . k_j
//
// in one pass over the keys: a running maximum m and sum, which rescale what has been
// summed when the maximum grows.  It is let grow by less than 2^kSlack unnoticed (the sums
// are floats and the probabilities are rounded relatively), so rescaling is rare.
//
// S^T = K Q^T and O^T = V^T P^T, columns are rows of the tile (attention.h): q stays in
// registers, K is read from LDS by rows and V by columns.  The tiles are fetched by
// direct-to-LDS loads a tile ahead into the other of two buffers.
#pragma once

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kRowsBlock = 128; // rows of a workgroup
constexpr float kSlack = 8.0f;  // log2

template <typename T, int DT>
struct RowsShape {
  // keys of a tile: 16 KB of K and as much of V, 32 keys at least
  static constexpr int kKeys = DT * sizeof(T) <= 256 ? 64 : 32;
  static constexpr int kTileBytes = kKeys * DT * sizeof(T);
  static constexpr int kPasses = kTileBytes / (256 * 16); // loads of a thread per tile
};

// Fetches the rows of keys [begin, end) of k and v to LDS; rows past them repeat the last one,
// so that nothing is read that no row sees.
template <typename T, int DT, bool PAGED>
__device__ __forceinline__ void fetch_keys(
    const AttentionArgs& a, int b, int hk, int begin, int end, T* k_tile, T* v_tile) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  const T* k = static_cast<const T*>(a.k);
  const T* v = static_cast<const T*>(a.v);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int n = 0; n < S::kPasses; ++n) {
    const int u = n * 256 + threadIdx.x;
    const int row = u / L::kUnits;
    const int d = ((u % L::kUnits) ^ L::swizzle(row)) * L::kUnit;
    const KeyRow r = key_row<PAGED>(a, b, hk, min(begin + row, end - 1));
    const bool in = d < a.D;
    const uint32_t to = (n * 256 + wave * 64) * 16;
    dma16_from(lds_address(k_tile) + to, in ? static_cast<const void*>(k + r.k + d) : &kNoData);
    dma16_from(lds_address(v_tile) + to, in ? static_cast<const void*>(v + r.v + d) : &kNoData);
  }
}

template <typename T, int DT, bool PAGED>
__global__ __launch_bounds__(256) void attention_rows_kernel(const AttentionArgs a, int blocks) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int KT = S::kKeys;
  constexpr int kBoth = 2 * S::kTileBytes / sizeof(T); // K and V
  __shared__ __align__(16) T lds[2 * kBoth];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  int head, piece;
  piece_of(a.B * a.Hkv, blocks * a.splits, &head, &piece);
  // the last rows see most keys: they come first
  const int block = blocks - 1 - piece / a.splits;
  const int split = piece % a.splits;
  const int b = head / a.Hkv;
  const int hk = head - b * a.Hkv;
  const int R = a.G * a.Lq;
  const int length = length_of(a, b);
  const int first_row = max(0, a.Lq - length) * a.G; // rows before it see nothing
  const int lo = max(block * kRowsBlock, first_row);
  const int hi = min(block * kRowsBlock + kRowsBlock, R) - 1;
  const int r0 = block * kRowsBlock + 32 * wave;
  const int row = r0 + (lane & 31);
  const bool stored = row < R;
  const bool seeing = stored && row >= first_row && length > 0;

  int t0 = 0, t1 = 0;
  KeyRange range = {};
  if (lo <= hi && length > 0) {
    range = keys_of(a, length, lo, hi, KT);
    t0 = static_cast<int>(static_cast<int64_t>(range.tiles) * split / a.splits);
    t1 = static_cast<int>(static_cast<int64_t>(range.tiles) * (split + 1) / a.splits);
  }
  // what this wave's own rows see
  const int w_lo = max(r0, first_row);
  const int w_hi = min(r0 + 31, R - 1);
  const bool works = w_lo <= w_hi && length > 0;
  const int p0 = length - a.Lq;
  const int p_lo = p0 + w_lo / a.G;
  const int p_hi = p0 + w_hi / a.G;
  const int from = min(max(row, lo), hi); // a row that sees something, in any lane
  const int p = p0 + from / a.G;
  const int seen_from = p - a.window + 1;

  Frag<T> q[DT / 16];
  if (t0 < t1) {
    const T* src = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.G, from);
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
      const int d = 16 * c + 8 * h;
      q[c] = d < a.D ? load_frag<T>(src + d) : zero_frag<T>();
      flip<T>(q[c], a.q_sign);
    }
  }

  floatx16 o[DT / 32];
  float m, l; // of this lane's half of the keys: the maximum is common, the sum is its own
  // A masked value that is not finite would reach rows that do not see it, as 0 * inf: where a
  // result is not finite the rows are done again, those values apart from the products.
  for (int careful = 0;; careful = 1) {
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
      o[d] = floatx16{};
    }
    m = -INFINITY;
    l = 0.0f;
    int begin, end;
    if (t0 < t1) {
      tile_of(range, t0, KT, &begin, &end);
      fetch_keys<T, DT, PAGED>(a, b, hk, begin, end, lds, lds + kBoth / 2);
    }
    for (int t = t0; t < t1; ++t) {
      wait_loads();
      __syncthreads();
      const T* k_tile = lds + ((t - t0) & 1) * kBoth;
      const T* v_tile = k_tile + kBoth / 2;
      tile_of(range, t, KT, &begin, &end);
      if (t + 1 < t1) {
        int b1, e1;
        tile_of(range, t + 1, KT, &b1, &e1);
        T* next = lds + ((t + 1 - t0) & 1) * kBoth;
        fetch_keys<T, DT, PAGED>(a, b, hk, b1, e1, next, next + kBoth / 2);
      }
      if (!works || none_seen(begin, end, p_lo, p_hi, a.window, a.keep)) {
        continue;
      }
      floatx16 s[KT / 32];
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
        s[g] = floatx16{};
#pragma unroll
        for (int c = 0; c < DT / 16; ++c) {
          s[g] = mma32<T>(L::load_rows(k_tile, 32 * g + (lane & 31), 2 * c + h), q[c], s[g]);
        }
      }
      const bool whole =
          end - begin == KT && all_seen(begin, end, p_lo, p_hi, a.window, a.keep);
      if (!whole) {
        const int last = min(p, end - 1);
#pragma unroll
        for (int g = 0; g < KT / 32; ++g) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = begin + 32 * g + 8 * (i / 4) + 4 * h + i % 4;
            s[g][i] = j <= last && (j >= seen_from || j < a.keep) ? s[g][i] : -INFINITY;
          }
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          top = fmaxf(top, s[g][i]);
        }
      }
      top = max_halves(top) * a.scale_log2;
      if (__any(top > m + kSlack)) {
        const float now = fmaxf(m, top);
        const float by = now == m ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= by;
#pragma unroll
        for (int d = 0; d < DT / 32; ++d) {
          o[d] *= by;
        }
      }
      const float less = m == -INFINITY ? 0.0f : m;
      float sum = 0.0f;
      Frag<T> w[KT / 16];
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(s[g][i], a.scale_log2, -less));
          sum += e[i];
        }
        w[2 * g] = frag_of<T>(e);
        w[2 * g + 1] = frag_of<T>(e + 8);
      }
      l += sum;
      const bool apart = careful != 0 && !whole;
#pragma unroll
      for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
        for (int g = 0; g < KT / 16; ++g) {
          Frag<T> f = L::load_cols(v_tile, 16 * g, 32 * d, lane);
          if (apart) {
            drop_not_finite<T>(f);
          }
          o[d] = mma32<T>(f, w[g], o[d]);
        }
      }
      if (apart) {
        for (int n = 0; n < end - begin; ++n) {
          const int j = begin + n;
          const bool sees = j <= p && (j >= seen_from || j < a.keep);
#pragma unroll
          for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = L::value(v_tile, n, 32 * d + 8 * (i / 4) + 4 * h + i % 4);
              o[d][i] += sees && not_finite(x) ? x : 0.0f;
            }
          }
        }
      }
    }
    bool odd = false;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        odd = odd || not_finite(o[d][i]);
      }
    }
    if (!__syncthreads_or(odd && careful == 0)) {
      break;
    }
  }

  l = sum_halves(l);
  if (!stored) {
    return;
  }
  if (a.splits > 1) {
    const int64_t at = (static_cast<int64_t>(split) * a.B * a.Hkv + head) * R + row;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * d + 8 * i + 4 * h;
        if (c < a.D) {
          *reinterpret_cast<float4*>(a.part_out + at * a.D + c) =
              make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        }
      }
    }
    if (h == 0) {
      a.part_ml[at] = make_float2(m, seeing ? l : 0.0f);
    }
    return;
  }
  const float by = l == 0.0f ? 0.0f : 1.0f / l; // nothing but scores of -inf
  T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.G, row);
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * d + 8 * i + 4 * h;
      if (c < a.D) {
        store4<T>(out + c, seeing ? floatx4{o[d][4 * i] * by, o[d][4 * i + 1] * by,
                                            o[d][4 * i + 2] * by, o[d][4 * i + 3] * by}
                                  : floatx4{});
      }
    }
  }
  if (a.lse != nullptr && h == 0) {
    const int i = row / a.G;
    a.lse[(static_cast<int64_t>(b) * a.Hq + hk * a.G + row - i * a.G) * a.Lq + i] =
        seeing ? m + log2f(l) : 0.0f;
  }
}

template <typename T, int DT>
int launch_rows_of(const AttentionArgs& a, hipStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.G) * a.Lq + kRowsBlock - 1) / kRowsBlock;
  MLXROCM_REHEARSE("attention_rows(dim=%d,splits=%d)", DT, a.splits);
  const dim3 grid(static_cast<unsigned>(blocks * a.B * a.Hkv * a.splits));
  if (a.table != nullptr) {
    attention_rows_kernel<T, DT, true><<<grid, 256, 0, s>>>(a, static_cast<int>(blocks));
  } else {
    attention_rows_kernel<T, DT, false><<<grid, 256, 0, s>>>(a, static_cast<int>(blocks));
  }
  MLXROCM_HIP_TRY(hipGetLastError());
  return static_cast<int>(MLXROCM_OK);
}

template <typename T>
int launch_rows_typed(const AttentionArgs& a, hipStream_t s) {
  if (a.D <= 64) {
    return launch_rows_of<T, 64>(a, s);
  } else if (a.D <= 96) {
    return launch_rows_of<T, 96>(a, s);
  } else if (a.D <= 128) {
    return launch_rows_of<T, 128>(a, s);
  }
  return launch_rows_of<T, 256>(a, s);
}

} // namespace

} // namespace mlxrocm

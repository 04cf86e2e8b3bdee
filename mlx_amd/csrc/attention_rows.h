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
//
// Bound by its instructions: 8192 tokens, 32 heads of 128 on 8, bfloat16 0.55 ms, 1.0 PFLOP/s, where a
// library's product of 8192^3 reaches 1.1; matrix and vector instructions are each busy for half of
// the cycles, at the clock that the power cap leaves.  2048 tokens over 32768 in pages 1.14 ms.
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
  static constexpr int kTile = kKeys * Tile<T, DT>::kPitch; // elements
  static constexpr int kPasses = kKeys / Tile<T, DT>::kRowsOfPass;
};

// Columns past D are not loaded: they are zero from the start.
template <typename T>
__device__ __forceinline__ void clear_lds(T* lds, int elements) {
  for (int i = threadIdx.x * (16 / sizeof(T)); i < elements; i += 256 * (16 / sizeof(T))) {
    *reinterpret_cast<uint4*>(lds + i) = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
}

// Fetches tiles of keys and values to LDS, 16 bytes a lane, four waves beside each other.  What
// differs between lanes is kept as 32-bit offsets, what differs between tiles is the same for all
// lanes (the 16 keys from a multiple of 16 on are in one page): a load takes no vector arithmetic.
template <typename T, int DT, bool PAGED>
struct KeyStream {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  const AttentionArgs& a;
  int b, hk, length, wave;
  int d[L::kTurns];                            // this lane's column
  uint32_t k_off[L::kTurns], v_off[L::kTurns]; // bytes from the first row of a load
  const T *k, *v;                              // of the head; contiguous: of the sequence's head
  // PAGED: lane i has where the rows of keys 16 i .. 16 i + 15 of a tile begin, or their pages
  int ids = 0;
  int in_page = 0;

  __device__ __forceinline__ KeyStream(
      const AttentionArgs& args, int b_, int hk_, int length_, int wave_, int lane)
      : a(args),
        b(b_),
        hk(hk_),
        length(length_),
        wave(wave_),
        k(static_cast<const T*>(args.k) + hk_ * args.k_strides[1] +
          (PAGED ? 0 : b_ * args.k_strides[0])),
        v(static_cast<const T*>(args.v) + hk_ * args.v_strides[1] +
          (PAGED ? 0 : b_ * args.v_strides[0])) {
    const int row = lane / L::kPlaces;
#pragma unroll
    for (int x = 0; x < L::kTurns; ++x) {
      d[x] = ((lane % L::kPlaces) ^
              L::swizzle(x * L::kRowsOfPass + wave * L::kRowsOfLoad + row)) *
          L::kUnit;
      k_off[x] = static_cast<uint32_t>((row * a.k_strides[2] + d[x]) * sizeof(T));
      v_off[x] = static_cast<uint32_t>((row * a.v_strides[2] + d[x]) * sizeof(T));
    }
  }
  // The pages of the tile from `begin` on, before the loads of the one before it
  __device__ __forceinline__ void look_up(int begin) {
    if constexpr (PAGED) {
      const int lane = threadIdx.x & 63;
      const int j = min(begin + 16 * (lane & (S::kKeys / 16 - 1)), a.keys - 1);
      ids = a.table[b * a.table_stride + a.page.divide(j, &in_page)];
    }
  }
  __device__ __forceinline__ void fetch(int begin, T* k_tile, T* v_tile) const {
    const bool inside = begin + S::kKeys <= length && (a.near & 1) != 0;
    if (inside) {
      // (a multiplication for all lanes, where the scalar unit would take one for each load)
      int64_t k_at, v_at;
      if constexpr (PAGED) {
        const int64_t id = min(max(ids, 0), a.pages - 1);
        k_at = id * a.k_strides[0] + in_page * a.k_strides[2];
        v_at = id * a.v_strides[0] + in_page * a.v_strides[2];
      } else {
        k_at = begin * a.k_strides[2];
        v_at = begin * a.v_strides[2];
      }
      const auto from = [](const T* p, int64_t at, int lane) {
        if constexpr (PAGED) {
          at = static_cast<int64_t>(
              static_cast<uint64_t>(static_cast<uint32_t>(
                  __builtin_amdgcn_readlane(static_cast<int>(at >> 32), lane)))
                  << 32 |
              static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at), lane)));
        }
        return p + at;
      };
#pragma unroll
      for (int n = 0; n < S::kPasses; ++n) {
        const int row = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
        // rows from the first of the tile, or of the 16 in one page
        const int64_t rest = PAGED ? row % 16 : row;
        const T* kp = from(k, k_at, row / 16) + rest * a.k_strides[2];
        const T* vp = from(v, v_at, row / 16) + rest * a.v_strides[2];
        const uint32_t to = row * L::kPitch * sizeof(T);
        if (d[n % L::kTurns] < a.D) {
          dma16_at(lds_address(k_tile) + to, k_off[n % L::kTurns], kp);
          dma16_at(lds_address(v_tile) + to, v_off[n % L::kTurns], vp);
        }
      }
    } else { // keys past the end repeat the last one
#pragma unroll
      for (int n = 0; n < S::kPasses; ++n) {
        const int row = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
        const int j = begin + row + static_cast<int>(threadIdx.x & 63) / L::kPlaces;
        const KeyRow r = key_row<PAGED>(a, PAGED ? b : 0, 0, min(j, length - 1));
        const uint32_t to = row * L::kPitch * sizeof(T);
        if (d[n % L::kTurns] < a.D) {
          dma16_from(lds_address(k_tile) + to, k + r.k + d[n % L::kTurns]);
          dma16_from(lds_address(v_tile) + to, v + r.v + d[n % L::kTurns]);
        }
      }
    }
  }
};

template <typename T, int DT, bool PAGED>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(DT * sizeof(T) <= 256 ? 2 : 1, DT * sizeof(T) <= 256 ? 2 : 1)))
void attention_rows_kernel(const AttentionArgs a, const Grid grid, int blocks) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int KT = S::kKeys;
  constexpr int kBoth = 2 * S::kTile; // K and V
  __shared__ __align__(1024) T lds[2 * kBoth];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  int head, piece;
  grid.find(&head, &piece);
  // the last rows see most keys: they come first
  int split;
  const int block = blocks - 1 - a.of_splits.divide(piece, &split);
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
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
    run_of(range.tiles, split, a.of_splits, &t0, &t1);
  }
  // what this wave's own rows see
  const int w_lo = max(r0, first_row);
  const int w_hi = min(r0 + 31, R - 1);
  const bool works = w_lo <= w_hi && length > 0;
  const int p0 = length - a.Lq;
  const int b_lo = p0 + a.of_G.divide(lo); // the workgroup's, and the wave's
  const int b_hi = p0 + a.of_G.divide(hi);
  const int p_lo = p0 + a.of_G.divide(w_lo);
  const int p_hi = p0 + a.of_G.divide(w_hi);
  const int from = min(max(row, lo), hi); // a row that sees something, in any lane
  const int p = p0 + a.of_G.divide(from);

  Frag<T> q[DT / 16];
  if (t0 < t1) {
    const T* src = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.of_G, from);
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
      const int d = 16 * c + 8 * h;
      q[c] = d < a.D ? load_frag<T>(src + d) : zero_frag<T>();
      flip<T>(q[c], a.q_sign);
    }
  }

  floatx16 o[DT / 32];
  float m, l; // of this lane's half of the keys: the maximum is common, the sum is its own
  if (a.D < L::kPitch) {
    clear_lds<T>(lds, 2 * kBoth);
  }
  KeyStream<T, DT, PAGED> keys(a, b, hk, length, wave, lane);
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
    o[d] = floatx16{};
  }
  m = -INFINITY;
  l = 0.0f;
  bool odd = false; // some value is not finite
  if (t0 < t1) {
    const int begin = tile_of(range, t0, KT).begin;
    keys.look_up(begin);
    keys.fetch(begin, lds, lds + kBoth / 2);
    keys.look_up(tile_of(range, t0 + 1, KT).begin);
  }
  for (int t = t0; t < t1; ++t) {
    wait_loads();
    __syncthreads();
    T* k_tile = lds + ((t - t0) & 1) * kBoth;
    T* v_tile = k_tile + kBoth / 2;
    const KeyTile tile = tile_of(range, t, KT);
    if (t + 1 < t1) {
      T* next = lds + ((t + 1 - t0) & 1) * kBoth;
      keys.fetch(tile_of(range, t + 1, KT).begin, next, next + kBoth / 2);
      keys.look_up(tile_of(range, t + 2, KT).begin);
    }
    const int begin = tile.begin;
    if (!whole_tile(a, tile, KT, b_lo, b_hi) &&
        any_of_block(odd_values<T, S::kTile>(v_tile))) {
      odd = true;
      copy_finite<T, S::kTile>(v_tile, v_tile);
      __syncthreads();
    }
    if (!works || none_seen(begin, tile.end, p_lo, p_hi, a.window, a.keep)) {
      continue;
    }
    floatx16 s[KT / 32];
#pragma unroll
    for (int g = 0; g < KT / 32; ++g) {
      s[g] = floatx16{};
    }
    read_ahead<T, (KT / 32) * (DT / 16)>(
        [&](int n) { return L::load_rows(k_tile, 32 * (n % (KT / 32)), n / (KT / 32), lane); },
        [&](int n, const Frag<T>& f) {
          s[n % (KT / 32)] = mma32<T>(f, q[n / (KT / 32)], s[n % (KT / 32)]);
        });
    const bool whole = whole_tile(a, tile, KT, p_lo, p_hi);
    if (!whole) {
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
        const uint32_t sees = seen_bits(a, tile, p, 32 * g) >> 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[g][i] = (sees >> (8 * (i / 4) + i % 4) & 1) != 0 ? s[g][i] : -INFINITY;
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
    // 16 keys at a time: their products run beside the exponentials of the next 16
    constexpr int kSteps = DT / 32; // products of 16 keys
    float sum = 0.0f;
    float e[8];
    const auto weigh = [&](int g, int i) {
      e[i] = __builtin_amdgcn_exp2f(fmaf(s[g / 2][8 * (g % 2) + i], a.scale_log2, -less));
      sum += e[i];
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      weigh(0, i);
    }
    Frag<T> w = frag_of<T>(e);
    read_ahead<T, (KT / 16) * kSteps>(
        [&](int n) { return L::load_cols(v_tile, 16 * (n / kSteps), 32 * (n % kSteps), lane); },
        [&](int n, const Frag<T>& f) {
          o[n % kSteps] = mma32<T>(f, w, o[n % kSteps]);
          const int g = n / kSteps + 1;
          if (g < KT / 16) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (i * kSteps / 8 == n % kSteps) {
                weigh(g, i);
              }
            }
            if (n % kSteps == kSteps - 1) {
              w = frag_of<T>(e);
            }
          }
        });
    l += sum;
  }
  l = sum_halves(l);
  // In float16 a probability below 2^-25 is zero: what is not finite in a tile that all rows see may
  // have made NaN of a sum
  constexpr bool kProbe = std::is_same<T, f16_t>::value;
  if constexpr (kProbe) {
    floatx4 probe = {};
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        probe[i % 4] = fmaf(o[d][i], 0.0f, probe[i % 4]);
      }
    }
    // (a row without a sum is NaN as it is)
    odd = odd || (l == l && !(probe[0] + probe[1] + probe[2] + probe[3] == 0.0f));
  }
  const int64_t part = (static_cast<int64_t>(split) * a.B * a.Hkv + head) * R;
  if (stored && a.splits > 1) {
    float* to = a.part_out + (part + row) * a.D;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * d + 8 * i + 4 * h;
        if (c < a.D) {
          *reinterpret_cast<float4*>(to + c) =
              make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        }
      }
    }
    if (h == 0) {
      a.part_ml[part + row] = make_float2(m, seeing ? l : 0.0f);
    }
  } else if (stored) {
    const float by = l == 0.0f ? 0.0f : 1.0f / l; // nothing but scores of -inf
    const int64_t n = lse_at(a, b, hk, row);
    T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, row);
    T* low = low_of<T>(a, n);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * d + 8 * i + 4 * h;
        if (c < a.D) {
          const floatx4 x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
          store_result<T>(
              out + c, low == nullptr ? nullptr : low + c, seeing ? x * by : floatx4{});
        }
      }
    }
    if (a.lse != nullptr && h == 0) {
      a.lse[n] = seeing ? m + log2f(l) : 0.0f;
    }
  }
  if (kProbe ? any_of_block(odd) : odd) { // the same for all
    float* totals = reinterpret_cast<float*>(lds); // of the rows
    __syncthreads(); // (no tile is read any more)
    if (h == 0) {
      totals[32 * wave + lane] = l;
    }
    after_stores();
    const int d = threadIdx.x;
    store_infinite(
        a, d, t0, t1, [&](int t) { return tile_of(range, t, KT); },
        [&](int j) {
          return to_f32(static_cast<const T*>(a.v)[key_row<PAGED>(a, b, hk, j).v + d]);
        },
        lo, hi, p0, [&](int r) { return totals[r - block * kRowsBlock]; },
        [&](int r, auto store) {
          if (a.splits > 1) {
            store(a.part_out + (part + r) * a.D + d);
          } else {
            store(static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, r) + d);
          }
        });
  }
}

template <typename T, int DT>
int launch_rows_of(const AttentionArgs& a, hipStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.G) * a.Lq + kRowsBlock - 1) / kRowsBlock;
  MLXROCM_REHEARSE("attention_rows(dim=%d,splits=%d)", DT, a.splits);
  const Grid grid(
      static_cast<int64_t>(a.B) * a.Hkv, blocks * a.splits, DT * sizeof(T) <= kPairBytes);
  if (a.table != nullptr) {
    attention_rows_kernel<T, DT, true>
        <<<grid.blocks(), 256, 0, s>>>(a, grid, static_cast<int>(blocks));
  } else {
    attention_rows_kernel<T, DT, false>
        <<<grid.blocks(), 256, 0, s>>>(a, grid, static_cast<int>(blocks));
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

// attention_few.h -- attention of few rows, up to 32 for a workgroup (a token, or a few, for all
// heads that share a key head; small problems in several workgroups): bound by reading the keys and
// values once, or where those are few by the latency of some dependent reads.
//
// The keys of a (sequence, key head) are cut into `splits` runs of tiles of 32, a workgroup
// each, and within a workgroup its four waves take tiles in turn, each with a running maximum
// and sum of its own; nothing waits for another wave until all keys are read.  The waves'
// results are joined in LDS, those of the runs by the join kernel.  One token over 65000, 28 heads of
// 128 on 4, float16 24 us, 5.5 TB/s; 32 sequences of 1024 to 8192 126 us, 4.8 TB/s; one of 515 6.6 us.
//
// Keys and values go from memory straight into the operands of the 16x16 matrix instruction:
//   S^T = K Q^T    a lane has 16 bytes of key l % 16
//   O^T = V^T P^T  a lane has E consecutive columns (E (l % 16) on) of the 8 values whose
//                  probabilities it holds; two keys' dwords are interleaved by v_perm, and the
//                  e-th instruction makes the columns E m + e.  So a load covers whole rows of v.
#pragma once

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kFewKeys = 32; // keys of a tile

template <typename T, int DT>
struct FewShape {
  static constexpr int kE = DT == 64 ? 4 : DT == 96 ? 6 : 8; // columns of a lane
  static constexpr int kGroups = DT == 256 ? 2 : 1;          // of 16 kE columns
  static constexpr int kDwords = kE * sizeof(T) / 4;
  static constexpr bool kNext = DT * sizeof(T) <= 256;
};

// The keys of one tile as this lane's operands need them.
template <typename T, int DT>
struct FewTile {
  using S = FewShape<T, DT>;
  Frag<T> k[2][DT / 32];
  uint32_t v[S::kGroups][8][S::kDwords];
};

template <int N>
__device__ __forceinline__ void load_dwords(const void* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = *(reinterpret_cast<const uint4*>(p) + i / 4);
      w[i] = x.x;
      w[i + 1] = x.y;
      w[i + 2] = x.z;
      w[i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 x = *(reinterpret_cast<const uint2*>(p) + i / 2);
      w[i] = x.x;
      w[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = *(reinterpret_cast<const uint32_t*>(p) + i);
    }
  }
}

// Loads keys [begin, end) of which the first is a multiple of 16; keys before `low` or from `end`
// on are replaced by the nearest that is read anyway.
template <typename T, int DT, bool PAGED>
__device__ __forceinline__ void load_tile(
    const AttentionArgs& a, int b, int hk, int begin, int low, int end, int lane,
    FewTile<T, DT>& tile) {
  using S = FewShape<T, DT>;
  const T* kp = static_cast<const T*>(a.k);
  const T* vp = static_cast<const T*>(a.v);
  const int m = lane & 15;
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    // the 16 keys of one operand lie in one page
    const int first = min(begin + 16 * t, (end - 1) & ~15);
    const KeyRow r = key_row<PAGED>(a, b, hk, first);
    const int least = max(low - first, 0);
    const int most = end - 1 - first;
    const T* k = kp + r.k + min(max(m, least), most) * a.k_strides[2];
#pragma unroll
    for (int c = 0; c < DT / 32; ++c) {
      const int d = 32 * c + 8 * g;
      tile.k[t][c] = d < a.D ? load_frag<T>(k + d) : zero_frag<T>();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* v = vp + r.v + min(max(4 * g + i, least), most) * a.v_strides[2];
#pragma unroll
      for (int n = 0; n < S::kGroups; ++n) {
        const int d = (16 * n + m) * S::kE;
        if (d < a.D) {
          load_dwords<S::kDwords>(v + d, tile.v[n][4 * t + i]);
        } else {
#pragma unroll
          for (int e = 0; e < S::kDwords; ++e) {
            tile.v[n][4 * t + i][e] = 0;
          }
        }
      }
    }
  }
}

// Column e of the lane's columns over its 8 keys
template <typename T, int DT>
__device__ __forceinline__ Frag<T> column(
    const uint32_t (&v)[8][FewShape<T, DT>::kDwords], int e) {
  Frag<T> f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f.w[j] = __uint_as_float(v[j][e]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f.w[j] = __builtin_amdgcn_perm(
          v[2 * j + 1][e / 2], v[2 * j][e / 2], e % 2 != 0 ? 0x07060302u : 0x05040100u);
    }
  }
  return f;
}

// NT: tiles of 16 rows
template <typename T, int DT, int NT, bool PAGED>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(DT * NT * sizeof(T) <= 256 ? 2 : 1)))
void attention_few_kernel(const AttentionArgs a, const Grid grid, int blocks) {
  using S = FewShape<T, DT>;
  constexpr int KT = kFewKeys;
  __shared__ struct { // the waves' results of 16 rows, while they are joined
    float o[4][16][DT + 4];
    float m[4][16], l[4][16];
    float total[16 * NT];
    int4 odd; // of each wave
  } join;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4;
  int head, split;
  grid.find(&head, &split);
  int r0 = 0;
  if (blocks > 1) { // (the last see most keys)
    r0 = (blocks - 1 - a.of_splits.divide(split, &split)) * 16 * NT;
  }
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
  const int R = a.G * a.Lq;
  const int length = length_of(a, b);
  // rows that see something: lo .. hi, or none (an empty sequence: lo >= R)
  const int lo = max(r0, max(0, a.Lq - length) * a.G);
  const int hi = min(r0 + 16 * NT, R) - 1;

  KeyRange range = {};
  int t0 = 0, t1 = 0;
  if (lo <= hi) {
    range = keys_of(a, length, lo, hi, KT);
    run_of(range.tiles, split, a.of_splits, &t0, &t1);
  }
  const int p0 = length - a.Lq;
  const int p_lo = p0 + a.of_G.divide(lo);
  const int p_hi = p0 + a.of_G.divide(hi);

  Frag<T> q[NT][DT / 32];
  int p[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = min(max(r0 + 16 * n + (lane & 15), lo), hi);
    p[n] = p0 + a.of_G.divide(row);
    const T* src = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.of_G, row);
#pragma unroll
    for (int c = 0; c < DT / 32; ++c) {
      const int d = 32 * c + 8 * g;
      q[n][c] = d < a.D && lo <= hi ? load_frag<T>(src + d) : zero_frag<T>();
      flip<T>(q[n][c], a.q_sign);
    }
  }

  floatx4 o[NT][S::kGroups][S::kE];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int x = 0; x < S::kGroups; ++x) {
#pragma unroll
      for (int e = 0; e < S::kE; ++e) {
        o[n][x][e] = floatx4{};
      }
    }
  }
  bool odd = false; // some value is not finite
  // the next tile is on its way while one is worked on, where registers are left for it
  FewTile<T, DT> tile, next;
  const auto load = [&](int t, FewTile<T, DT>& to) {
    const KeyTile at = tile_of(range, t, KT);
    load_tile<T, DT, PAGED>(a, b, hk, at.begin, at.low, at.end, lane, to);
  };
  if (S::kNext && t0 + wave < t1) {
    load(t0 + wave, next);
  }
  for (int t = t0 + wave; t < t1; t += 4) {
    const KeyTile at = tile_of(range, t, KT);
    if constexpr (S::kNext) {
      tile = next;
      if (t + 4 < t1) {
        load(t + 4, next);
      }
    } else {
      load(t, tile);
    }
    const bool whole = whole_tile(a, at, KT, p_lo, p_hi);
    // In 16 bits a probability is the sum of two numbers: little here waits for the products (8
    // sequences of 5 tokens over a window of 4096 22.4 us, 21.6 with one, a token over 65000 27.8 and
    // 27.7), and the result is as near as its own rounding lets it be (with one, 1.4 times as far off)
    constexpr int kTerms = sizeof(T) == 2 ? 2 : 1;
    Frag<T> w[NT][kTerms];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      floatx4 s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x] = floatx4{};
#pragma unroll
        for (int c = 0; c < DT / 32; ++c) {
          s[x] = mma16<T>(tile.k[x][c], q[n][c], s[x]);
        }
      }
      if (!whole) {
        const Seen sees(a, at, p[n], 4 * g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i / 4][i % 4] = sees(16 * (i / 4) + i % 4) ? s[i / 4][i % 4] : -INFINITY;
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        top = fmaxf(top, s[i / 4][i % 4]);
      }
      top *= a.scale_log2;
      if (__any(top > m[n])) {
        const float now = fmaxf(m[n], max_quarters(top));
        const float by = now == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - now);
        m[n] = now;
        l[n] *= by;
#pragma unroll
        for (int x = 0; x < S::kGroups; ++x) {
#pragma unroll
          for (int e = 0; e < S::kE; ++e) {
            o[n][x][e] *= by;
          }
        }
      }
      const float less = m[n] == -INFINITY ? 0.0f : m[n];
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], a.scale_log2, -less));
        l[n] += e[i];
      }
      w[n][0] = frag_of<T>(e);
      if constexpr (kTerms == 2) {
        w[n][1] = rest_of<T>(e, w[n][0]);
      }
    }
    // (rows of one position see the same keys, and those alone are loaded, as are those of whole
    // tiles: a value that is not finite reaches all rows, if as NaN where a probability or its second
    // term is zero or of the other sign.  That is seen of the sums.)
    if (a.Lq > 1 && !whole) {
      uint32_t bits = 0;
#pragma unroll
      for (int x = 0; x < S::kGroups * 8; ++x) {
#pragma unroll
        for (int e = 0; e < S::kDwords; ++e) {
          bits |= odd_bits<T>(tile.v[x / 8][x % 8][e]);
        }
      }
      if (__any(is_odd<T>(bits))) {
        odd = true;
#pragma unroll
        for (int x = 0; x < S::kGroups * 8; ++x) {
#pragma unroll
          for (int e = 0; e < S::kDwords; ++e) {
            tile.v[x / 8][x % 8][e] = finite_part<T>(tile.v[x / 8][x % 8][e]);
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < S::kGroups; ++x) {
#pragma unroll
      for (int e = 0; e < S::kE; ++e) {
        const Frag<T> f = column<T, DT>(tile.v[x], e);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (const Frag<T>& term : w[n]) {
            o[n][x][e] = mma16<T>(f, term, o[n][x][e]);
          }
        }
      }
    }
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = sum_quarters(l[n]);
    floatx4 probe = {}; // NaN if some sum is not finite
#pragma unroll
    for (int x = 0; x < S::kGroups * S::kE; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        probe[i] = fmaf(o[n][x / S::kE][x % S::kE][i], 0.0f, probe[i]);
      }
    }
    // (a row without a sum of probabilities is NaN as it is)
    odd = odd || (l[n] == l[n] && !(probe[0] + probe[1] + probe[2] + probe[3] == 0.0f));
  }

  const int any_odd = __any(odd);
  int4 all_odd = {};
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads(); // the tile of rows before has been joined
    if (g == 0) {
      join.m[wave][lane] = m[n];
      join.l[wave][lane] = l[n];
    }
    if (n == 0 && lane == 0) {
      reinterpret_cast<int*>(&join.odd)[wave] = any_odd;
    }
#pragma unroll
    for (int x = 0; x < S::kGroups; ++x) {
#pragma unroll
      for (int e = 0; e < S::kE; ++e) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          join.o[wave][lane & 15][(16 * x + 4 * g + i) * S::kE + e] = o[n][x][e][i];
        }
      }
    }
    __syncthreads();
    if (n == 0) {
      all_odd = join.odd;
    }
    // 16 threads for a row
    const int at = threadIdx.x >> 4;
    const int row = r0 + 16 * n + at;
    if (row <= hi) {
      float top = join.m[0][at];
#pragma unroll
      for (int x = 1; x < 4; ++x) {
        top = fmaxf(top, join.m[x][at]);
      }
      const float less = top == -INFINITY ? 0.0f : top;
      float by[4], total = 0.0f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        by[x] = join.m[x][at] == less ? 1.0f : __builtin_amdgcn_exp2f(join.m[x][at] - less);
        total += by[x] * join.l[x][at];
      }
      const bool seeing = row >= lo;
      const float over = total == 0.0f ? 0.0f : 1.0f / total;
      const int64_t part = (static_cast<int64_t>(split) * a.B * a.Hkv + head) * R + row;
      T* out = static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, row);
      T* low = low_of<T>(a, lse_at(a, b, hk, row));
      for (int d = 4 * (threadIdx.x & 15); d < a.D; d += 64) {
        floatx4 sum4 = {};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 v = *reinterpret_cast<const float4*>(&join.o[x][at][d]);
          sum4 += by[x] * floatx4{v.x, v.y, v.z, v.w};
        }
        if (a.splits > 1) {
          *reinterpret_cast<float4*>(a.part_out + part * a.D + d) =
              make_float4(sum4[0], sum4[1], sum4[2], sum4[3]);
        } else {
          store_result<T>(
              out + d, low == nullptr ? nullptr : low + d, seeing ? sum4 * over : floatx4{});
        }
      }
      if ((threadIdx.x & 15) == 0) {
        join.total[16 * n + at] = total;
        if (a.splits > 1) {
          a.part_ml[part] = make_float2(top, seeing ? total : 0.0f);
        } else if (a.lse != nullptr) {
          a.lse[lse_at(a, b, hk, row)] = seeing ? top + log2f(total) : 0.0f;
        }
      }
    }
  }
  if ((all_odd.x | all_odd.y | all_odd.z | all_odd.w) != 0) { // the same for all
    after_stores();
    const int64_t part = (static_cast<int64_t>(split) * a.B * a.Hkv + head) * R;
    const int d = threadIdx.x;
    store_infinite(
        a, d, t0, t1, [&](int t) { return tile_of(range, t, KT); },
        [&](int j) {
          return to_f32(static_cast<const T*>(a.v)[key_row<PAGED>(a, b, hk, j).v + d]);
        },
        lo, hi, p0, [&](int r) { return join.total[r - r0]; },
        [&](int r, auto store) {
          if (a.splits > 1) {
            store(a.part_out + (part + r) * a.D + d);
          } else {
            store(static_cast<T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, r) + d);
          }
        });
  }
}

template <typename T, int DT, int NT>
int launch_few_rows(const AttentionArgs& a, hipStream_t s) {
  MLXROCM_REHEARSE("attention_few(dim=%d,rows=%d,splits=%d)", DT, 16 * NT, a.splits);
  const int blocks = (a.G * a.Lq + 16 * NT - 1) / (16 * NT);
  const Grid grid(static_cast<int64_t>(a.B) * a.Hkv, blocks * a.splits, false);
  if (a.table != nullptr) {
    attention_few_kernel<T, DT, NT, true><<<grid.blocks(), 256, 0, s>>>(a, grid, blocks);
  } else {
    attention_few_kernel<T, DT, NT, false><<<grid.blocks(), 256, 0, s>>>(a, grid, blocks);
  }
  MLXROCM_HIP_TRY(hipGetLastError());
  return static_cast<int>(MLXROCM_OK);
}

template <typename T, int DT>
int launch_few_of(const AttentionArgs& a, hipStream_t s) {
  if constexpr (DT <= 64 || (sizeof(T) == 4 && DT <= 128)) {
    if (a.G * a.Lq > 16) {
      return launch_few_rows<T, DT, 2>(a, s);
    }
  }
  return launch_few_rows<T, DT, 1>(a, s);
}

template <typename T>
int launch_few_typed(const AttentionArgs& a, hipStream_t s) {
  if (a.D <= 64) {
    return launch_few_of<T, 64>(a, s);
  } else if (a.D == 96) { // six columns of a lane end at 96 only
    return launch_few_of<T, 96>(a, s);
  } else if (a.D <= 128) {
    return launch_few_of<T, 128>(a, s);
  }
  return launch_few_of<T, 256>(a, s);
}

} // namespace

} // namespace mlxrocm

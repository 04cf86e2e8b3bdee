// attention_grad.h -- the gradients of attention from that of its result (attention.h has the
// names and layouts):
//
//   P_ij  = exp(s_ij - lse_i)             delta_i = do_i . o_i
//   dS_ij = P_ij (do_i . v_j - delta_i)
//   dq_i  = scale sum_j dS_ij k_j         dk_j = scale sum_i dS_ij q_i      dv_j = sum_i P_ij do_i
//
// The probabilities are formed again from the sums that the forward kept.  Two kernels, each with
// its result in registers and the other side in LDS tiles: dq over keys, dk and dv over rows (of
// all heads that share the key head, so their sum needs no second pass).  Seven products where one
// kernel with atomic sums of dq would take five: no result depends on the order of arrival.
#pragma once

#include "attention_rows.h"

namespace mlxrocm {

namespace {

// ---- dq: workgroups of 128 rows, as the forward -----------------------------------------
template <typename T, int DT>
__global__ __launch_bounds__(256, DT * sizeof(T) <= 256 ? 2 : 1) void attention_dq_kernel(const AttentionGradArgs ga, int blocks) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int KT = S::kKeys;
  constexpr int kBoth = 2 * S::kTile;
  __shared__ __align__(16) T lds[2 * kBoth];
  const AttentionArgs& a = ga.a;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  int head, piece;
  piece_of(a.B * a.Hkv, blocks, &head, &piece);
  const int block = blocks - 1 - piece;
  const int b = head / a.Hkv;
  const int hk = head - b * a.Hkv;
  const int R = a.G * a.Lq;
  const int length = length_of(a, b);
  const int first_row = max(0, a.Lq - length) * a.G;
  const int lo = max(block * kRowsBlock, first_row);
  const int hi = min(block * kRowsBlock + kRowsBlock, R) - 1;
  const int r0 = block * kRowsBlock + 32 * wave;
  const int row = r0 + (lane & 31);
  const bool stored = row < R;
  const bool seeing = stored && row >= first_row && length > 0;

  const bool any = lo <= hi && length > 0;
  const KeyRange range = any ? keys_of(a, length, lo, hi, KT) : KeyRange{};
  const int w_lo = max(r0, first_row);
  const int w_hi = min(r0 + 31, R - 1);
  const bool works = w_lo <= w_hi && length > 0;
  const int p0 = length - a.Lq;
  const int p_lo = p0 + w_lo / a.G;
  const int p_hi = p0 + w_hi / a.G;
  const int from = min(max(row, lo), hi);
  const int i_from = from / a.G;
  const int p = p0 + i_from;
  const int seen_from = p - a.window + 1;

  Frag<T> q[DT / 16], dout[DT / 16];
  float lse = 0.0f, delta = 0.0f;
  if (any) {
    const T* src = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.G, from);
    const T* dsrc = static_cast<const T*>(ga.dout) + row_offset(ga.dout_strides, b, hk, a.G, from);
    const T* osrc = static_cast<const T*>(a.out) + row_offset(a.out_strides, b, hk, a.G, from);
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
      const int d = 16 * c + 8 * h;
      q[c] = d < a.D ? load_frag<T>(src + d) : zero_frag<T>();
      flip<T>(q[c], a.q_sign);
      dout[c] = d < a.D ? load_frag<T>(dsrc + d) : zero_frag<T>();
      if (d < a.D) {
        float x[8], y[8];
        load8<T>(dsrc + d, x);
        load8<T>(osrc + d, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          delta = fmaf(x[e], y[e], delta);
        }
      }
    }
    delta = sum_halves(delta);
    const int64_t at =
        (static_cast<int64_t>(b) * a.Hq + hk * a.G + from - i_from * a.G) * a.Lq + i_from;
    lse = a.lse[at];
    if (seeing && h == 0) {
      ga.delta[at] = delta;
    }
  }

  if (a.D < L::kPitch) {
    clear_lds<T>(lds, 2 * kBoth);
  }
  KeyStream<T, DT, false> keys(a, b, hk, length, wave, lane);
  floatx16 dq[DT / 32];
  // (a masked key that is not finite: see attention_rows_kernel)
  for (int careful = 0;; careful = 1) {
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
      dq[d] = floatx16{};
    }
    if (range.tiles > 0) {
      keys.fetch(tile_of(range, 0, KT).begin, lds, lds + kBoth / 2);
    }
    for (int t = 0; t < range.tiles; ++t) {
      wait_loads();
      __syncthreads();
      const T* k_tile = lds + (t & 1) * kBoth;
      const T* v_tile = k_tile + kBoth / 2;
      const KeyTile tile = tile_of(range, t, KT);
      if (t + 1 < range.tiles) {
        T* next = lds + ((t + 1) & 1) * kBoth;
        keys.fetch(tile_of(range, t + 1, KT).begin, next, next + kBoth / 2);
      }
      const int begin = tile.begin;
      if (!works || none_seen(begin, tile.end, p_lo, p_hi, a.window, a.keep)) {
        continue;
      }
      const bool whole = whole_tile(a, tile, KT, p_lo, p_hi);
      const int last = min(p, tile.end - 1);
      const bool apart = careful != 0 && !whole;
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
        floatx16 s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < DT / 16; ++c) {
          s = mma32<T>(L::load_rows(k_tile, 32 * g + (lane & 31), 2 * c + h), q[c], s);
          dp = mma32<T>(L::load_rows(v_tile, 32 * g + (lane & 31), 2 * c + h), dout[c], dp);
        }
        float ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -lse));
          ds[i] = e * (dp[i] - delta);
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = begin + 32 * g + 8 * (i / 4) + 4 * h + i % 4;
            const bool sees = j >= tile.low && j <= last && (j >= seen_from || j < a.keep);
            ds[i] = sees ? ds[i] : 0.0f;
          }
        }
        const Frag<T> w[2] = {frag_of<T>(ds), frag_of<T>(ds + 8)};
#pragma unroll
        for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            Frag<T> f = L::load_cols(k_tile, 32 * g + 16 * n, 32 * d, lane);
            if (apart) {
              drop_not_finite<T>(f);
            }
            dq[d] = mma32<T>(f, w[n], dq[d]);
          }
        }
      }
      if (apart) {
        for (int n = max(tile.low - begin, 0); n < tile.end - begin; ++n) {
          const int j = begin + n;
          const bool sees = j <= p && (j >= seen_from || j < a.keep);
#pragma unroll
          for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = L::value(k_tile, n, 32 * d + 8 * (i / 4) + 4 * h + i % 4);
              dq[d][i] += sees && not_finite(x) ? x : 0.0f;
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
        odd = odd || not_finite(dq[d][i]);
      }
    }
    if (!__syncthreads_or(odd && careful == 0)) {
      break;
    }
  }
  if (!stored) {
    return;
  }
  T* to = static_cast<T*>(ga.dq) + row_offset(ga.dq_strides, b, hk, a.G, row);
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * d + 8 * i + 4 * h;
      if (c < a.D) {
        store4<T>(to + c, seeing ? floatx4{dq[d][4 * i], dq[d][4 * i + 1], dq[d][4 * i + 2],
                                           dq[d][4 * i + 3]} *
                               ga.scale
                                 : floatx4{});
      }
    }
  }
}

// ---- dk, dv: workgroups of 128 keys ------------------------------------------------------
constexpr int kKeysBlock = 128;

// What a row's probabilities need beside q: its sum, its delta and its position.
struct RowStats {
  float lse, delta;
  int p;
};
template <int N>
struct StatsTile {
  float lse[N], delta[N];
  int p[N];
};

// Fetches tiles of rows of q and dout to LDS (see KeyStream).  Where a power of two of heads
// share a key head, a lane's rows lie at the same offsets from the first of each load.
template <typename T, int DT>
struct RowStream {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  const AttentionGradArgs& ga;
  int b, hk, end, wave;
  int d;
  uint32_t q_off, d_off;

  __device__ __forceinline__ RowStream(
      const AttentionGradArgs& args, int b_, int hk_, int end_, int wave_, int lane)
      : ga(args), b(b_), hk(hk_), end(end_), wave(wave_) {
    const int row = lane / L::kPlaces;
    const int i = row / ga.a.G;
    const int g = row - i * ga.a.G;
    d = ((lane % L::kPlaces) ^ L::swizzle(wave * L::kRowsOfLoad + row)) * L::kUnit;
    q_off = static_cast<uint32_t>(
        (g * ga.a.q_strides[1] + i * ga.a.q_strides[2] + d) * sizeof(T));
    d_off = static_cast<uint32_t>(
        (g * ga.dout_strides[1] + i * ga.dout_strides[2] + d) * sizeof(T));
  }
  // Rows from `begin` on (a multiple of G); rows past the end repeat the last one
  __device__ __forceinline__ void fetch(int begin, T* q_tile, T* d_tile) const {
    const AttentionArgs& a = ga.a;
    const T* q = static_cast<const T*>(a.q);
    const T* dout = static_cast<const T*>(ga.dout);
    const bool inside = begin + S::kKeys <= end && (a.near & 2) != 0;
#pragma unroll
    for (int n = 0; n < S::kPasses; ++n) {
      const int row = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
      const uint32_t to = row * L::kPitch * sizeof(T);
      if (inside) {
        const T* qp = q + row_offset(a.q_strides, b, hk, a.G, begin + row);
        const T* dp = dout + row_offset(ga.dout_strides, b, hk, a.G, begin + row);
        if (d < a.D) {
          dma16(lds_address(q_tile) + to, q_off, qp);
          dma16(lds_address(d_tile) + to, d_off, dp);
        }
      } else {
        const int r =
            min(begin + row + static_cast<int>(threadIdx.x & 63) / L::kPlaces, end - 1);
        if (d < a.D) {
          dma16_from(
              lds_address(q_tile) + to, q + row_offset(a.q_strides, b, hk, a.G, r) + d);
          dma16_from(
              lds_address(d_tile) + to, dout + row_offset(ga.dout_strides, b, hk, a.G, r) + d);
        }
      }
    }
  }
};

template <typename T, int DT>
__global__ __launch_bounds__(256, DT * sizeof(T) <= 128 ? 2 : 1) void attention_dkv_kernel(const AttentionGradArgs ga, int blocks) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int RT = S::kKeys; // rows of a tile
  constexpr int kBoth = 2 * S::kTile;
  // this lane's key and value: in registers, but for 256 floats, which are read again for
  // each tile (with both results they would need all 512 registers)
  constexpr bool kHeld = DT * sizeof(T) <= 512;
  __shared__ __align__(16) T lds[2 * kBoth];
  __shared__ __align__(16) StatsTile<RT> stats[2];
  const AttentionArgs& a = ga.a;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  int head, block;
  piece_of(a.B * a.Hkv, blocks, &head, &block);
  const int b = head / a.Hkv;
  const int hk = head - b * a.Hkv;
  const int length = length_of(a, b);
  const int k0 = block * kKeysBlock;
  const int k1 = min(k0 + kKeysBlock, length); // keys of this workgroup that are seen
  const int p0 = length - a.Lq;
  // the tokens that see one of them
  const int i0 = max(max(0, -p0), k0 - p0);
  const int i1 = k0 < a.keep ? a.Lq : min(a.Lq, k1 - 1 + a.window - p0);
  const bool any = k0 < k1 && i0 < i1;
  const int begin_row = i0 * a.G;
  const int end_row = i1 * a.G;
  const int tiles = any ? (end_row - begin_row + RT - 1) / RT : 0;

  const int w0 = k0 + 32 * wave;
  const int w1 = min(w0 + 32, k1); // the wave's keys [w0, w1)
  const bool works = w0 < w1;
  const int key = w0 + (lane & 31);
  const KeyRow at = key_row<false>(a, b, hk, min(key, max(length, 1) - 1));
  const T* k_src = static_cast<const T*>(a.k) + at.k;
  const T* v_src = static_cast<const T*>(a.v) + at.v;
  const auto key_frag = [&](int c) {
    const int d = 16 * c + 8 * h;
    Frag<T> f = d < a.D ? load_frag<T>(k_src + d) : zero_frag<T>();
    flip<T>(f, a.q_sign);
    return f;
  };
  const auto value_frag = [&](int c) {
    const int d = 16 * c + 8 * h;
    return d < a.D ? load_frag<T>(v_src + d) : zero_frag<T>();
  };
  Frag<T> k[kHeld ? DT / 16 : 1], v[kHeld ? DT / 16 : 1];
  if constexpr (kHeld) {
    if (any) {
#pragma unroll
      for (int c = 0; c < DT / 16; ++c) {
        k[c] = key_frag(c);
        v[c] = value_frag(c);
      }
    }
  }
  const auto stats_of = [&](int t) {
    const int r = min(begin_row + t * RT + static_cast<int>(threadIdx.x), end_row - 1);
    const int i = r / a.G;
    const int64_t n = (static_cast<int64_t>(b) * a.Hq + hk * a.G + r - i * a.G) * a.Lq + i;
    return RowStats{a.lse[n], ga.delta[n], p0 + i};
  };

  if (a.D < L::kPitch) {
    clear_lds<T>(lds, 2 * kBoth);
  }
  const RowStream<T, DT> rows(ga, b, hk, end_row, wave, lane);
  floatx16 dk[DT / 32], dv[DT / 32];
  // (a masked row that is not finite: see attention_rows_kernel)
  for (int careful = 0;; careful = 1) {
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
      dk[d] = floatx16{};
      dv[d] = floatx16{};
    }
    RowStats mine = {};
    if (tiles > 0) {
      if (threadIdx.x < RT) {
        mine = stats_of(0);
      }
      rows.fetch(begin_row, lds, lds + kBoth / 2);
    }
    for (int t = 0; t < tiles; ++t) {
      StatsTile<RT>& st = stats[t & 1];
      wait_loads();
      if (threadIdx.x < RT) {
        st.lse[threadIdx.x] = mine.lse;
        st.delta[threadIdx.x] = mine.delta;
        st.p[threadIdx.x] = mine.p;
      }
      __syncthreads();
      const T* q_tile = lds + (t & 1) * kBoth;
      const T* d_tile = q_tile + kBoth / 2;
      const int begin = begin_row + t * RT;
      const int count = min(RT, end_row - begin);
      if (t + 1 < tiles) {
        if (threadIdx.x < RT) {
          mine = stats_of(t + 1);
        }
        T* next = lds + ((t + 1) & 1) * kBoth;
        rows.fetch(begin + RT, next, next + kBoth / 2);
      }
      const int p_lo = st.p[0];
      const int p_hi = st.p[count - 1];
      if (!works || none_seen(w0, w1, p_lo, p_hi, a.window, a.keep)) {
        continue;
      }
      const bool whole = count == RT && w1 - w0 == 32 &&
          all_seen(w0, w1, p_lo, p_hi, a.window, a.keep);
      const bool apart = careful != 0 && !whole;
#pragma unroll
      for (int g = 0; g < RT / 32; ++g) {
        floatx16 s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < DT / 16; ++c) {
          const Frag<T> kc = kHeld ? k[kHeld ? c : 0] : key_frag(c);
          const Frag<T> vc = kHeld ? v[kHeld ? c : 0] : value_frag(c);
          s = mma32<T>(L::load_rows(q_tile, 32 * g + (lane & 31), 2 * c + h), kc, s);
          dp = mma32<T>(L::load_rows(d_tile, 32 * g + (lane & 31), 2 * c + h), vc, dp);
        }
        float e[16], ds[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int n = 32 * g + 2 * i + 4 * h;
          const float4 lse = *reinterpret_cast<const float4*>(st.lse + n);
          const float4 delta = *reinterpret_cast<const float4*>(st.delta + n);
          const float ls[4] = {lse.x, lse.y, lse.z, lse.w};
          const float de[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            e[i + x] = __builtin_amdgcn_exp2f(fmaf(s[i + x], a.scale_log2, -ls[x]));
            ds[i + x] = e[i + x] * (dp[i + x] - de[x]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int n = 32 * g + 8 * (i / 4) + 4 * h + i % 4;
            const int p = st.p[n];
            const bool sees = n < count && key < k1 && key <= p &&
                (p - key < a.window || key < a.keep);
            e[i] = sees ? e[i] : 0.0f;
            ds[i] = sees ? ds[i] : 0.0f;
          }
        }
        const Frag<T> we[2] = {frag_of<T>(e), frag_of<T>(e + 8)};
        const Frag<T> ws[2] = {frag_of<T>(ds), frag_of<T>(ds + 8)};
#pragma unroll
        for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            Frag<T> fd = L::load_cols(d_tile, 32 * g + 16 * n, 32 * d, lane);
            Frag<T> fq = L::load_cols(q_tile, 32 * g + 16 * n, 32 * d, lane);
            if (apart) {
              drop_not_finite<T>(fd);
              drop_not_finite<T>(fq);
            }
            dv[d] = mma32<T>(fd, we[n], dv[d]);
            dk[d] = mma32<T>(fq, ws[n], dk[d]);
          }
        }
      }
      if (apart) {
        for (int n = 0; n < count; ++n) {
          const int p = st.p[n];
          const bool sees = key < k1 && key <= p && (p - key < a.window || key < a.keep);
#pragma unroll
          for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int c = 32 * d + 8 * (i / 4) + 4 * h + i % 4;
              const float x = L::value(q_tile, n, c);
              const float y = L::value(d_tile, n, c);
              dk[d][i] += sees && not_finite(x) ? x : 0.0f;
              dv[d][i] += sees && not_finite(y) ? y : 0.0f;
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
        odd = odd || not_finite(dk[d][i]) || not_finite(dv[d][i]);
      }
    }
    if (!__syncthreads_or(odd && careful == 0)) {
      break;
    }
  }
  if (key >= a.keys || key >= k0 + kKeysBlock) {
    return;
  }
  const bool seen = key < k1;
  const int64_t k_to = b * ga.dk_strides[0] + hk * ga.dk_strides[1] + key * ga.dk_strides[2];
  const int64_t v_to = b * ga.dv_strides[0] + hk * ga.dv_strides[1] + key * ga.dv_strides[2];
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * d + 8 * i + 4 * h;
      if (c < a.D) {
        const floatx4 x = {dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]};
        const floatx4 y = {dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]};
        store4<T>(static_cast<T*>(ga.dk) + k_to + c, seen ? x * ga.scale : floatx4{});
        store4<T>(static_cast<T*>(ga.dv) + v_to + c, seen ? y : floatx4{});
      }
    }
  }
}

template <typename T, int DT>
int launch_grad_of(const AttentionGradArgs& g, hipStream_t s) {
  const AttentionArgs& a = g.a;
  const int rows = static_cast<int>(
      (static_cast<int64_t>(a.G) * a.Lq + kRowsBlock - 1) / kRowsBlock);
  const int keys = (a.keys + kKeysBlock - 1) / kKeysBlock;
  if (rows > 0) {
    attention_dq_kernel<T, DT><<<rows * a.B * a.Hkv, 256, 0, s>>>(g, rows);
    MLXROCM_HIP_TRY(hipGetLastError());
  }
  if (keys > 0) {
    attention_dkv_kernel<T, DT><<<keys * a.B * a.Hkv, 256, 0, s>>>(g, keys);
    MLXROCM_HIP_TRY(hipGetLastError());
  }
  return static_cast<int>(MLXROCM_OK);
}

template <typename T>
int launch_grad_typed(const AttentionGradArgs& g, hipStream_t s) {
  if (g.a.D <= 64) {
    return launch_grad_of<T, 64>(g, s);
  } else if (g.a.D <= 96) {
    return launch_grad_of<T, 96>(g, s);
  } else if (g.a.D <= 128) {
    return launch_grad_of<T, 128>(g, s);
  }
  return launch_grad_of<T, 256>(g, s);
}

} // namespace

} // namespace mlxrocm

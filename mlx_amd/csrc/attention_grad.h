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
// Bound as the forward: 8192 tokens, 32 heads of 128 on 8, bfloat16 dq 0.73 ms, dk and dv 1.21, 1.1 and
// 0.91 PFLOP/s.
#pragma once

#include "attention_rows.h"

namespace mlxrocm {

namespace {

// A lane's column of a partial sum
template <int DT>
__device__ __forceinline__ void store_part(
    float* to, const floatx16 (&x)[DT / 32], bool any, int D, int h) {
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * d + 8 * i + 4 * h;
      if (c < D) {
        *reinterpret_cast<float4*>(to + c) = any
            ? make_float4(x[d][4 * i], x[d][4 * i + 1], x[d][4 * i + 2], x[d][4 * i + 3])
            : make_float4(0, 0, 0, 0);
      }
    }
  }
}

// Float16 has five bits of exponent: as an operand the probabilities of many keys, and more so their
// gradients beside a small dout, would lose bits or be zero, those beside a large one infinite (2048
// tokens, 128 columns, dout of 1e-4: dq three times as far off as its own rounding, now as far).  So
// probabilities count 2^kProbabilityUp times.  Their gradients, and so the sums, count 2^up times: of
// dq for each row, a number that only falls, to where the largest is some 2^kRangeFirst once one is
// above 2^kRangeMost; of dk for all of a workgroup, by the largest ones of its rows, which dq's kernel
// leaves behind.  (The sums of dk and dv take all registers: to multiply them on the way, 256 columns,
// took 530 us instead of 240.)
template <typename T>
constexpr bool kRanged = std::is_same<T, f16_t>::value;
constexpr int kProbabilityUp = 14;
constexpr int kRangeStart = 64; // (a gradient below 2^-49 is nothing in the results)
constexpr int kRangeFirst = 9;
constexpr int kRangeMost = 15;

__device__ __forceinline__ int exponent_of(float x) { // of x > 0
  return static_cast<int>(__float_as_uint(x) >> 23) - 127;
}

// A row's 16 gradients, which count 2^up times, as do the largest so far and the sums that have them
template <int STEPS>
__device__ __forceinline__ void
fit_range(float (&ds)[16], int& up, float& largest, floatx16 (&sums)[STEPS]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    top = fmaxf(top, fabsf(ds[i]));
  }
  top = max_halves(top);
  largest = fmaxf(largest, top);
  constexpr float kMost = 1 << kRangeMost;
  if (__any(top > kMost)) {
    const int by = top > kMost ? kRangeFirst - exponent_of(top) : 0;
    up += by;
    const float times = ldexpf(1.0f, by);
    largest *= times;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      ds[i] *= times;
    }
#pragma unroll
    for (int d = 0; d < STEPS; ++d) {
      sums[d] *= times;
    }
  }
}

// ---- dq: workgroups of 128 rows, as the forward -----------------------------------------
template <typename T, int DT>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(DT * sizeof(T) <= 256 ? 2 : 1, DT * sizeof(T) <= 256 ? 2 : 1)))
void attention_dq_kernel(const AttentionGradArgs ga, const Grid grid, int blocks) {
  using S = RowsShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int KT = S::kKeys;
  constexpr int kBoth = 2 * S::kTile;
  __shared__ __align__(1024) T lds[2 * kBoth];
  const AttentionArgs& a = ga.a;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  const Divisor& splits = ga.plan.dq_splits;
  int head, piece, split;
  grid.find(&head, &piece);
  const int block = blocks - 1 - splits.divide(piece, &split);
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
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
  int t0, t1;
  run_of(range.tiles, split, splits, &t0, &t1);
  const int w_lo = max(r0, first_row);
  const int w_hi = min(r0 + 31, R - 1);
  const bool works = w_lo <= w_hi && length > 0;
  const int p0 = length - a.Lq;
  const int b_lo = p0 + a.of_G.divide(lo); // the workgroup's, and the wave's
  const int b_hi = p0 + a.of_G.divide(hi);
  const int p_lo = p0 + a.of_G.divide(w_lo);
  const int p_hi = p0 + a.of_G.divide(w_hi);
  const int from = min(max(row, lo), hi);
  const int i_from = a.of_G.divide(from);
  const int p = p0 + i_from;

  Frag<T> q[DT / 16], dout[DT / 16];
  float lse = 0.0f, delta = 0.0f;
  int up = kRanged<T> ? kRangeStart : 0;
  float largest = 0.0f;
  if (any) {
    const T* src = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.of_G, from);
    const T* dsrc = static_cast<const T*>(ga.dout) + row_offset(ga.dout_strides, b, hk, a.of_G, from);
    const T* osrc = static_cast<const T*>(a.out) + row_offset(a.out_strides, b, hk, a.of_G, from);
    const int64_t at = lse_at(a, b, hk, from);
    const T* low = low_of<T>(a, at);
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
        if (sizeof(T) == 2 && low != nullptr) {
          load8<T>(low + d, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            delta = fmaf(x[e], y[e], delta);
          }
        }
      }
    }
    delta = sum_halves(delta);
    lse = a.lse[at];
    if (seeing && h == 0 && split == 0) {
      ga.delta[at] = delta;
    }
  }

  if (a.D < L::kPitch) {
    clear_lds<T>(lds, 2 * kBoth);
  }
  KeyStream<T, DT, false> keys(a, b, hk, length, wave, lane);
  floatx16 dq[DT / 32];
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
    dq[d] = zero_sum();
  }
  if (t0 < t1) {
    keys.fetch(tile_of(range, t0, KT).begin, lds, lds + kBoth / 2);
  }
  bool odd = false; // some key was left out of the products
  for (int t = t0; t < t1; ++t) {
    wait_loads();
    __syncthreads();
    const T* k_tile = lds + ((t - t0) & 1) * kBoth;
    const T* v_tile = k_tile + kBoth / 2;
    T* next = lds + ((t + 1 - t0) & 1) * kBoth;
    const KeyTile tile = tile_of(range, t, KT);
    // The scores need the keys as they are: those without what is not finite lie where the
    // next tile will, which is fetched after them.
    const bool apart = !whole_tile(a, tile, KT, b_lo, b_hi) &&
        any_of_block(odd_values<T, S::kTile>(k_tile));
    if (apart) {
      odd = true;
      copy_finite<T, S::kTile>(k_tile, next);
      __syncthreads();
    } else if (t + 1 < t1) {
      keys.fetch(tile_of(range, t + 1, KT).begin, next, next + kBoth / 2);
    }
    const T* cols = apart ? next : k_tile;
    if (works && !none_seen(tile.begin, tile.end, p_lo, p_hi, a.window, a.keep)) {
      const bool whole = whole_tile(a, tile, KT, p_lo, p_hi);
#pragma unroll
      for (int g = 0; g < KT / 32; ++g) {
        floatx16 s = {}, dp = {};
        read_ahead<T, DT / 8>(
            [&](int n) { return L::load_rows(n % 2 == 0 ? k_tile : v_tile, 32 * g, n / 2, lane); },
            [&](int n, const Frag<T>& f) {
              if (n % 2 == 0) {
                s = mma32<T>(f, q[n / 2], s);
              } else {
                dp = mma32<T>(f, dout[n / 2], dp);
              }
            });
        float ds[16];
        const float less = kRanged<T> ? lse - up : lse;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -less));
          ds[i] = e * (dp[i] - delta);
        }
        if (!whole) {
          asm volatile(""); // a branch, not 16 selections for every tile
          const uint32_t sees = seen_bits(a, tile, p, 32 * g) >> 4 * h;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            ds[i] = (sees >> (8 * (i / 4) + i % 4) & 1) != 0 ? ds[i] : 0.0f;
          }
        }
        if constexpr (kRanged<T>) {
          fit_range(ds, up, largest, dq);
        }
        const Frag<T> w[2] = {frag_of<T>(ds), frag_of<T>(ds + 8)};
        read_ahead<T, DT / 16>(
            [&](int n) { return L::load_cols(cols, 32 * g + 16 * (n % 2), 32 * (n / 2), lane); },
            [&](int n, const Frag<T>& f) { dq[n / 2] = mma32<T>(f, w[n % 2], dq[n / 2]); });
      }
    }
    if (apart && t + 1 < t1) {
      __syncthreads();
      keys.fetch(tile_of(range, t + 1, KT).begin, next, next + kBoth / 2);
    }
  }
  if constexpr (kRanged<T>) {
    const float down = ldexpf(1.0f, -up);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
      dq[d] *= down;
    }
    // (a row that has an infinite one has no others)
    largest = max_lanes(not_finite(largest) ? 0.0f : largest * down);
    if (lane == 0) {
      ga.largest[((static_cast<int64_t>(head) * splits.d + split) * blocks + block) * 4 + wave] =
          largest;
    }
  }
  const int64_t part = (static_cast<int64_t>(split) * a.B * a.Hkv + head) * R;
  if (stored && splits.d > 1) {
    store_part<DT>(ga.part_dq + (part + row) * a.D, dq, seeing, a.D, h);
  } else if (stored) {
    T* to = static_cast<T*>(ga.dq) + row_offset(ga.dq_strides, b, hk, a.of_G, row);
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
  if (odd) { // the same for all
    after_stores();
    const int d = threadIdx.x;
    for (int t = t0; t < t1 && d < a.D; ++t) {
      const KeyTile tile = tile_of(range, t, KT);
      for (int j = max(tile.begin, tile.low); j < tile.end; ++j) {
        const float x = to_f32(static_cast<const T*>(a.k)[key_row<false>(a, b, hk, j).k + d]);
        for (int r = lo; not_finite(x) && r <= hi; ++r) {
          if (!sees_key(a, p0 + a.of_G.divide(r), j)) {
            continue;
          }
          if (splits.d > 1) {
            add_to(ga.part_dq + (part + r) * a.D + d, x);
          } else {
            add_to(static_cast<T*>(ga.dq) + row_offset(ga.dq_strides, b, hk, a.of_G, r) + d, x);
          }
        }
      }
    }
  }
}

// ---- dk, dv: workgroups of 128 keys ------------------------------------------------------
constexpr int kKeysBlock = kGradBlock;

// What a row's probabilities need beside q: its sum, its delta and its position.
struct RowStats {
  float lse, delta;
};
template <int N>
struct StatsTile {
  float lse[N], delta[N];
};

// Fetches tiles of rows of q and dout to LDS (see KeyStream).  Where a power of two of heads
// share a key head, a lane's rows lie at the same offsets from the first of each load.
template <typename T, int DT, int ROWS>
struct RowStream {
  using L = Tile<T, DT>;
  static constexpr int kPasses = ROWS / L::kRowsOfPass;
  const AttentionGradArgs& ga;
  int b, hk, end, wave;
  int d[L::kTurns];
  uint32_t q_off[L::kTurns], d_off[L::kTurns];
  bool near;
  const T *q, *dout;                       // the first row of the next tile
  int64_t q_pass[kPasses], d_pass[kPasses]; // from there, of each load

  __device__ __forceinline__ RowStream(
      const AttentionGradArgs& args, int b_, int hk_, int begin, int end_, int wave_, int lane)
      : ga(args), b(b_), hk(hk_), end(end_), wave(wave_), near((args.a.near & 2) != 0) {
    const AttentionArgs& a = ga.a;
    const int row = lane / L::kPlaces;
    const int i = row >> a.g_log2;
    const int g = row & (a.G - 1);
#pragma unroll
    for (int x = 0; x < L::kTurns; ++x) {
      d[x] = ((lane % L::kPlaces) ^
              L::swizzle(x * L::kRowsOfPass + wave * L::kRowsOfLoad + row)) *
          L::kUnit;
      q_off[x] = static_cast<uint32_t>(
          (g * a.q_strides[1] + i * a.q_strides[2] + d[x]) * sizeof(T));
      d_off[x] = static_cast<uint32_t>(
          (g * ga.dout_strides[1] + i * ga.dout_strides[2] + d[x]) * sizeof(T));
    }
    q = static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.of_G, begin);
    dout = static_cast<const T*>(ga.dout) + row_offset(ga.dout_strides, b, hk, a.of_G, begin);
#pragma unroll
    for (int n = 0; n < kPasses; ++n) {
      const int first = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
      const int fi = first >> a.g_log2;
      const int fg = first & (a.G - 1);
      q_pass[n] = fg * a.q_strides[1] + fi * a.q_strides[2];
      d_pass[n] = fg * ga.dout_strides[1] + fi * ga.dout_strides[2];
    }
  }
  // Rows from `begin` on, one tile after the other; rows past the end repeat the last one
  __device__ __forceinline__ void fetch(int begin, T* q_tile, T* d_tile) {
    const AttentionArgs& a = ga.a;
    const bool inside = near && begin + ROWS <= end;
    if (inside) {
#pragma unroll
      for (int n = 0; n < kPasses; ++n) {
        const int row = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
        const uint32_t to = row * L::kPitch * sizeof(T);
        if (d[n % L::kTurns] < a.D) {
          dma16_at(lds_address(q_tile) + to, q_off[n % L::kTurns], q + q_pass[n]);
          dma16_at(lds_address(d_tile) + to, d_off[n % L::kTurns], dout + d_pass[n]);
        }
      }
      // (a tile is whole tokens: a power of two of heads up to its rows share a key head)
      q += (ROWS >> a.g_log2) * a.q_strides[2];
      dout += (ROWS >> a.g_log2) * ga.dout_strides[2];
    } else {
#pragma unroll
      for (int n = 0; n < kPasses; ++n) {
        const int row = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
        const uint32_t to = row * L::kPitch * sizeof(T);
        const int r =
            min(begin + row + static_cast<int>(threadIdx.x & 63) / L::kPlaces, end - 1);
        if (d[n % L::kTurns] < a.D) {
          dma16_from(
              lds_address(q_tile) + to,
              static_cast<const T*>(a.q) + row_offset(a.q_strides, b, hk, a.of_G, r) +
                  d[n % L::kTurns]);
          dma16_from(
              lds_address(d_tile) + to,
              static_cast<const T*>(ga.dout) + row_offset(ga.dout_strides, b, hk, a.of_G, r) +
                  d[n % L::kTurns]);
        }
      }
    }
  }
};

// Two waves a SIMD leave 256 registers.  Both results of 128 columns take 128 of them, and keys
// and values 64: the values stay in LDS then (read again for each tile, a quarter more
// than is read anyway), and a tile is 32 rows, so that two workgroups fit, of whose sums and deltas
// four are in registers at a time.  8192 tokens, 32 heads of 128, both gradients 2.05 ms; with two
// fragments read ahead instead of four a hundredth more.  Of 256 columns one wave a SIMD has 512 registers:
// 4096 tokens, 8 heads of 256 on 2 0.45 ms; a kernel for dk and one for dv, which make the scores
// twice, 0.55 ms.
template <typename T, int DT>
struct DkvShape {
  static constexpr bool kTwo = DT * sizeof(T) <= 256; // waves a SIMD
  static constexpr bool kValuesInLds = sizeof(T) == 2 && DT >= 96;
  static constexpr int kRows = kValuesInLds || sizeof(T) == 4 ? 32 : 64; // of a tile
  static constexpr int kTile = kRows * Tile<T, DT>::kPitch;
};

template <typename T, int DT>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(DkvShape<T, DT>::kTwo ? 2 : 1, DkvShape<T, DT>::kTwo ? 2 : 1)))
void attention_dkv_kernel(const AttentionGradArgs ga, const Grid grid) {
  using S = DkvShape<T, DT>;
  using L = Tile<T, DT>;
  constexpr int RT = S::kRows;
  constexpr int kBoth = 2 * S::kTile;
  // this lane's key and value: in registers, but for 256 floats, which are read again for
  // each tile (with both results they would need all 512 registers)
  constexpr bool kKeyHeld = DT * sizeof(T) <= 512;
  constexpr bool kValueHeld = kKeyHeld && !S::kValuesInLds;
  __shared__ __align__(1024) T lds[2 * kBoth];
  __shared__ __align__(1024) T values[S::kValuesInLds ? kKeysBlock * L::kPitch : 16];
  __shared__ __align__(16) StatsTile<RT> stats[2];
  const AttentionArgs& a = ga.a;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  const GradPlan& plan = ga.plan;
  int head, piece;
  grid.find(&head, &piece);
  // the first keys are seen by most rows: they come first
  const int wide = plan.wide_blocks * plan.wide_splits.d;
  const Divisor& splits = piece < wide ? plan.wide_splits : plan.splits;
  int split;
  const int block = piece < wide ? splits.divide(piece, &split)
                                 : plan.wide_blocks + splits.divide(piece - wide, &split);
  int hk;
  const int b = a.of_Hkv.divide(head, &hk);
  const int length = length_of(a, b);
  const int k0 = block * kKeysBlock;
  const int k1 = min(k0 + kKeysBlock, length); // keys of this workgroup that are seen
  const int p0 = length - a.Lq;
  // the tokens that see one of them
  const int i0 = max(max(0, -p0), k0 - p0);
  const int i1 = k0 < a.keep ? a.Lq : min(a.Lq, k1 - 1 + a.window - p0);
  const int all = k0 < k1 && i0 < i1 ? ((i1 - i0) * a.G + RT - 1) / RT : 0; // tiles of rows
  int s0, s1;
  run_of(all, split, splits, &s0, &s1);
  const int tiles = s1 - s0; // of this run
  const bool any = tiles > 0;
  const int begin_row = i0 * a.G + s0 * RT;
  const int end_row = min(i1 * a.G, i0 * a.G + s1 * RT);

  const int w0 = k0 + 32 * wave;
  const int w1 = min(w0 + 32, k1); // the wave's keys [w0, w1)
  const bool works = w0 < w1;
  const int key = w0 + (lane & 31);
  // The rows that see this lane's key are [see_from, see_to): the tokens from its own on, as long as
  // it is in their windows
  const int64_t left = static_cast<int64_t>(key) + a.window - p0;
  const int see_from = min(max(key - p0, 0), a.Lq) * a.G;
  const int see_to = key >= k1      ? 0
      : key < a.keep || left > a.Lq ? a.Lq * a.G
                                    : max(static_cast<int>(left), 0) * a.G;
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
  Frag<T> k[kKeyHeld ? DT / 16 : 1], v[kValueHeld ? DT / 16 : 1];
  if (any) {
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
      if constexpr (kKeyHeld) {
        k[c] = key_frag(c);
      }
      if constexpr (kValueHeld) {
        v[c] = value_frag(c);
      }
    }
  }
  if (a.D < L::kPitch) {
    clear_lds<T>(lds, 2 * kBoth);
    if constexpr (S::kValuesInLds) {
      clear_lds<T>(values, kKeysBlock * L::kPitch);
    }
  }
  if constexpr (S::kValuesInLds) {
    if (any) { // keys past the end repeat the last one
#pragma unroll
      for (int n = 0; n < kKeysBlock / L::kRowsOfPass; ++n) {
        const int first = n * L::kRowsOfPass + wave * L::kRowsOfLoad;
        const int r = first + lane / L::kPlaces;
        const int d = ((lane % L::kPlaces) ^ L::swizzle(r)) * L::kUnit;
        if (d < a.D) {
          dma16_from(
              lds_address(values) + first * L::kPitch * sizeof(T),
              static_cast<const T*>(a.v) +
                  key_row<false>(a, b, hk, min(k0 + r, length - 1)).v + d);
        }
      }
    }
  }
  // 2^(up - kProbabilityUp), for gradients of at most 2^kRangeMost
  float times = 1.0f;
  if constexpr (kRanged<T>) {
    __shared__ float tops[4];
    if (any) {
      const int waves = (a.G * a.Lq + kRowsBlock - 1) / kRowsBlock * 4; // of dq's kernel, 32 rows each
      const int first = begin_row / 32, count = (end_row + 31) / 32 - first;
      float top = 0.0f;
      for (int x = 0; x < plan.dq_splits.d; ++x) {
        const float* of = ga.largest + (static_cast<int64_t>(head) * plan.dq_splits.d + x) * waves;
        for (int i = threadIdx.x; i < count; i += 256) {
          top = fmaxf(top, of[first + i]);
        }
      }
      top = max_lanes(top);
      if (lane == 0) {
        tops[wave] = top;
      }
      __syncthreads();
      top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      const int up = min(kRangeStart, kRangeMost - 1 - exponent_of(top));
      times = __int_as_float(__builtin_amdgcn_readfirstlane(
          __float_as_int(ldexpf(1.0f, up - kProbabilityUp))));
    }
  }
  const auto stats_of = [&](int t) {
    const int r = min(begin_row + t * RT + static_cast<int>(threadIdx.x), end_row - 1);
    const int i = a.of_G.divide(r);
    const int64_t n = (static_cast<int64_t>(b) * a.Hq + hk * a.G + r - i * a.G) * a.Lq + i;
    return kRanged<T> ? RowStats{a.lse[n] - kProbabilityUp, ga.delta[n] * times}
                      : RowStats{a.lse[n], ga.delta[n]};
  };

  RowStream<T, DT, RT> rows(ga, b, hk, begin_row, end_row, wave, lane);
  floatx16 dk[DT / 32], dv[DT / 32];
#pragma unroll
  for (int d = 0; d < DT / 32; ++d) {
    dk[d] = zero_sum();
    dv[d] = zero_sum();
  }
  RowStats mine = {};
  if (tiles > 0) {
    if (threadIdx.x < RT) {
      mine = stats_of(0);
    }
    rows.fetch(begin_row, lds, lds + kBoth / 2);
  }
  bool odd = false; // some row was left out of the products
  for (int t = 0; t < tiles; ++t) {
    StatsTile<RT>& st = stats[t & 1];
    wait_loads();
    if (threadIdx.x < RT) {
      st.lse[threadIdx.x] = mine.lse;
      st.delta[threadIdx.x] = mine.delta;
    }
    __syncthreads();
    const T* q_tile = lds + (t & 1) * kBoth;
    const T* d_tile = q_tile + kBoth / 2;
    T* next = lds + ((t + 1) & 1) * kBoth;
    const int begin = begin_row + t * RT;
    const int count = min(RT, end_row - begin);
    if (t + 1 < tiles && threadIdx.x < RT) {
      mine = stats_of(t + 1);
    }
    const int p_lo = p0 + a.of_G.divide(begin);
    const int p_hi = p0 + a.of_G.divide(begin + count - 1);
    // (as in attention_dq_kernel)
    const bool apart =
        !(count == RT && all_seen(k0, k1, p_lo, p_hi, a.window, a.keep)) &&
        any_of_block(odd_values<T, 2 * S::kTile>(q_tile));
    if (apart) {
      odd = true;
      copy_finite<T, 2 * S::kTile>(q_tile, next);
      __syncthreads();
    } else if (t + 1 < tiles) {
      rows.fetch(begin + RT, next, next + kBoth / 2);
    }
    const T* q_cols = apart ? next : q_tile;
    const T* d_cols = q_cols + kBoth / 2;
    if (works && !none_seen(w0, w1, p_lo, p_hi, a.window, a.keep)) {
      const bool whole = count == RT && w1 - w0 == 32 &&
          all_seen(w0, w1, p_lo, p_hi, a.window, a.keep);
      // Products of the two halves of the tile in turn, the exponentials of one half beside
      // the products of the other.
      constexpr int kHalves = RT / 32;
      constexpr int kSteps = DT / 16; // matrix instructions of a product
      floatx16 e[kHalves], dp[kHalves]; // scores, probabilities, and their gradients at last
      uint32_t sees[kHalves];           // of 32 rows, this lane's from 4 h on
      const auto product = [&](const auto& read, const auto& use, const auto& beside) {
        read_ahead<T, kSteps>(read, [&](int n, const Frag<T>& f) {
          use(n, f);
          beside(n);
        });
      };
      const auto nothing = [](int) {};
      const auto scores = [&](int g, const auto& beside) {
        e[g] = floatx16{};
        product(
            [&](int n) { return L::load_rows(q_tile, 32 * g, n, lane); },
            [&](int n, const Frag<T>& f) {
              e[g] = mma32<T>(f, kKeyHeld ? k[kKeyHeld ? n : 0] : key_frag(n), e[g]);
            },
            beside);
      };
      const auto d_weights = [&](int g, const auto& beside) {
        dp[g] = floatx16{};
        if constexpr (S::kValuesInLds) {
          Frag<T> d_rows;
          read_ahead<T, 2 * kSteps>(
              [&](int n) {
                return n % 2 == 0 ? L::load_rows(d_tile, 32 * g, n / 2, lane)
                                  : L::load_rows(values, 32 * wave, n / 2, lane);
              },
              [&](int n, const Frag<T>& f) {
                if (n % 2 == 0) {
                  d_rows = f;
                } else {
                  dp[g] = mma32<T>(d_rows, f, dp[g]);
                  beside(n / 2);
                }
              });
        } else {
          product(
              [&](int n) { return L::load_rows(d_tile, 32 * g, n, lane); },
              [&](int n, const Frag<T>& f) {
                dp[g] = mma32<T>(f, kValueHeld ? v[kValueHeld ? n : 0] : value_frag(n), dp[g]);
              },
              beside);
        }
      };
      struct Weights {
        Frag<T> of[2]; // 16 rows each
      };
      const auto packed = [&](int g) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] = e[g][i];
        }
        return Weights{{frag_of<T>(x), frag_of<T>(x + 8)}};
      };
      const auto add_packed = [&](const T* cols, int g, const Weights& w, floatx16(&to)[DT / 32],
                                  const auto& beside) {
        product(
            [&](int n) { return L::load_cols(cols, 32 * g + 16 * (n % 2), 32 * (n / 2), lane); },
            [&](int n, const Frag<T>& f) { to[n / 2] = mma32<T>(f, w.of[n % 2], to[n / 2]); },
            beside);
      };
      const auto add = [&](const T* cols, int g, floatx16(&to)[DT / 32], const auto& beside) {
        add_packed(cols, g, packed(g), to, beside);
      };
      // the n-th of kSteps parts of a half's exponentials, and of what becomes of them
      const auto exponentials = [&](int g) {
        return [&, g](int n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i * kSteps / 16 == n) {
              e[g][i] = __builtin_amdgcn_exp2f(fmaf(
                  e[g][i], a.scale_log2, -st.lse[32 * g + 8 * (i / 4) + 4 * h + i % 4]));
            }
          }
        };
      };
      const auto d_scores = [&](int g) {
        return [&, g](int n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i * kSteps / 16 == n) {
              const float delta = st.delta[32 * g + 8 * (i / 4) + 4 * h + i % 4];
              e[g][i] *= kRanged<T> ? fmaf(dp[g][i], times, -delta) : dp[g][i] - delta;
            }
          }
        };
      };
      const auto hide = [&](int g) {
        if (!whole) {
          asm volatile(""); // a branch, not 16 selections for every tile
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            e[g][i] = (sees[g] >> (8 * (i / 4) + i % 4) & 1) != 0 ? e[g][i] : 0.0f;
          }
        }
      };
      if (!whole) {
#pragma unroll
        for (int g = 0; g < kHalves; ++g) {
          sees[g] = (bits_below(min(see_to, end_row) - begin - 32 * g) &
                     ~bits_below(see_from - begin - 32 * g)) >>
              4 * h;
        }
      }
      if constexpr (kHalves == 2) {
        scores(0, nothing);
        scores(1, exponentials(0));
        hide(0);
        d_weights(0, exponentials(1));
        hide(1);
        add(d_cols, 0, dv, d_scores(0));
        hide(0); // (again: what is not finite in a row that is not seen)
        d_weights(1, nothing);
        add(q_cols, 0, dk, nothing);
        add(d_cols, 1, dv, d_scores(1));
        hide(1);
        add(q_cols, 1, dk, nothing);
      } else { // (in the order that holds the fewest registers)
        d_weights(0, nothing);
        scores(0, nothing);
        // (four rows' numbers in registers at a time, not all sixteen)
        const auto by_fours = [&](const float* of, const auto& use) {
          float4 next = *reinterpret_cast<const float4*>(of + 4 * h);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4 now = next;
            if (x < 3) {
              next = *reinterpret_cast<const float4*>(of + 8 * (x + 1) + 4 * h);
            }
            use(4 * x, now.x);
            use(4 * x + 1, now.y);
            use(4 * x + 2, now.z);
            use(4 * x + 3, now.w);
            __builtin_amdgcn_sched_barrier(0);
          }
        };
        by_fours(st.lse, [&](int i, float lse) {
          e[0][i] = __builtin_amdgcn_exp2f(fmaf(e[0][i], a.scale_log2, -lse));
        });
        hide(0);
        const auto probabilities = packed(0);
        by_fours(st.delta, [&](int i, float delta) {
          e[0][i] *= kRanged<T> ? fmaf(dp[0][i], times, -delta) : dp[0][i] - delta;
        });
        hide(0);
        const auto d_probabilities = packed(0);
        add_packed(d_cols, 0, probabilities, dv, nothing);
        add_packed(q_cols, 0, d_probabilities, dk, nothing);
      }
    }
    if (apart && t + 1 < tiles) {
      __syncthreads();
      rows.fetch(begin + RT, next, next + kBoth / 2);
    }
  }
  if constexpr (kRanged<T>) {
    constexpr float kDown = 1.0f / (1 << kProbabilityUp);
    const float down = kDown / times;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d) {
      dk[d] *= down;
      dv[d] *= kDown;
    }
  }
  const bool parts = splits.d > 1;
  float* part = ga.part_dkv +
      (static_cast<int64_t>(head) * plan.part_pieces() + piece) * (kKeysBlock * 2 * a.D);
  if (parts) {
    float* to = part + (key - k0) * 2 * a.D;
    store_part<DT>(to, dk, key < k1, a.D, h);
    store_part<DT>(to + a.D, dv, key < k1, a.D, h);
  } else if (key < a.keys) {
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
  if (odd) { // the same for all
    after_stores();
    const int d = threadIdx.x;
    for (int r = begin_row; r < end_row && d < a.D; ++r) {
      const float x = to_f32(
          static_cast<const T*>(a.q)[row_offset(a.q_strides, b, hk, a.of_G, r) + d]);
      const float y = to_f32(
          static_cast<const T*>(ga.dout)[row_offset(ga.dout_strides, b, hk, a.of_G, r) + d]);
      for (int j = k0; (not_finite(x) || not_finite(y)) && j < k1; ++j) {
        if (!sees_key(a, p0 + a.of_G.divide(r), j)) {
          continue;
        }
        if (parts) {
          add_to(part + (j - k0) * 2 * a.D + d, not_finite(x) ? x : 0.0f);
          add_to(part + (j - k0) * 2 * a.D + a.D + d, not_finite(y) ? y : 0.0f);
          continue;
        }
        if (not_finite(x)) {
          add_to(
              static_cast<T*>(ga.dk) + b * ga.dk_strides[0] + hk * ga.dk_strides[1] +
                  j * ga.dk_strides[2] + d,
              x);
        }
        if (not_finite(y)) {
          add_to(
              static_cast<T*>(ga.dv) + b * ga.dv_strides[0] + hk * ga.dv_strides[1] +
                  j * ga.dv_strides[2] + d,
              y);
        }
      }
    }
  }
}

template <typename T, int DT>
int launch_grad_of(const AttentionGradArgs& g, hipStream_t s) {
  const AttentionArgs& a = g.a;
  MLXROCM_REHEARSE(
      "attention_dq(dim=%d,splits=%d)+attention_dkv(dim=%d,splits=%d,kept=%dx%d)", DT,
      g.plan.dq_splits.d, DT, g.plan.splits.d, g.plan.wide_blocks, g.plan.wide_splits.d);
  const int rows = static_cast<int>(
      (static_cast<int64_t>(a.G) * a.Lq + kRowsBlock - 1) / kRowsBlock);
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
  if (rows > 0) {
    const Grid grid(
        heads, static_cast<int64_t>(rows) * g.plan.dq_splits.d, DT * sizeof(T) <= kPairBytes);
    attention_dq_kernel<T, DT><<<grid.blocks(), 256, 0, s>>>(g, grid, rows);
    MLXROCM_HIP_TRY(hipGetLastError());
  }
  if (g.plan.blocks > 0) {
    const Grid grid(heads, g.plan.pieces(), DT * sizeof(T) <= kPairBytes);
    attention_dkv_kernel<T, DT><<<grid.blocks(), 256, 0, s>>>(g, grid);
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

// attention.h -- what the attention kernels share: their arguments, which keys a
// query sees, where the rows of keys, values and queries lie, fragments of the
// matrix instructions and tiles in LDS.
//
// For one sequence and one key head the G query heads that share it and the Lq new
// tokens are taken together as R = G Lq rows: row r is token i = r / G of query head
// hk G + r % G, at position p = length - Lq + i of the sequence.  It sees key j where
//   0 <= j <= p  and  (p - j < window or j < keep),
// nothing if p < 0 (padding in front of a short sequence).  Every key that is read is
// so read once for all heads that share it, and the sums over those heads that the
// gradients of keys and values need are sums over rows.
//
// Every product is formed with the queries (forward, dq) or the keys (dk, dv) as the
// columns of the matrix instruction's result: a lane then holds one column, so running
// maxima, sums and rescaling are plain per-lane arithmetic, and the probabilities are
// where the next product wants its second operand: a result has in register i of lane l
// (32x32) row 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32, and an operand has 8
// values along the contraction.  The order in which a sum over keys is taken is free, so
// registers 8 q .. 8 q + 7 of a lane serve as those 8 values without moving: they stand
// for keys 16 q + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3}, h = l / 32, and the other
// operand is read from LDS in that order.
#pragma once

#include "mfma_dequant.h"
#include "mfma_loads.h"

namespace mlxrocm {

// n / d for n below 2^31 in a multiplication: with m = 2^32 / d the quotient is short by one at
// most.  (The compiler's own division takes some forty instructions, and a workgroup has several
// before its first load.)
struct Divisor {
  int d = 1;
  uint32_t m = 0xffffffffu;
  Divisor() = default;
  explicit Divisor(int64_t by)
      : d(by < 1 ? 1 : static_cast<int>(by)),
        m(by <= 1 ? 0xffffffffu : static_cast<uint32_t>((uint64_t{1} << 32) / by)) {}
#ifdef __HIPCC__
  __device__ __forceinline__ int divide(int n, int* rest) const {
    int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), m));
    int r = n - q * d;
    if (r >= d) {
      ++q;
      r -= d;
    }
    *rest = r;
    return q;
  }
  __device__ __forceinline__ int divide(int n) const {
    int rest;
    return divide(n, &rest);
  }
#endif
};

struct AttentionArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse; // [B, Hq, Lq]: log2 of the sum of exp(score), for the gradients; may be null
  void* low;  // [B, Hq, Lq, D]: what rounding took from out, for the gradients; may be null
  const int* lengths; // [B], or null: every sequence has `keys`
  const int* table;   // [B, table_stride], or null: contiguous keys
  int64_t table_stride;
  int B, Hq, Hkv, G, Lq, D;
  int keys;      // most keys a sequence can have
  Divisor page;  // rows of a page (table)
  int pages;
  Divisor of_G, of_Hkv, of_splits;
  // strides in elements; of k and v: [sequence or page, head, row]
  int64_t q_strides[3], k_strides[3], v_strides[3], out_strides[3]; // [sequence, head, token]
  float scale_log2; // |scale| log2(e)
  uint32_t q_sign;  // 0x80008000 (16-bit types), 0x80000000 (float32) where scale < 0
  int window, keep;
  int g_log2; // of a power of two of heads (near & 2)
  int near; // the rows of one load lie within 32-bit offsets: of keys (1), of queries (2)
  int splits;
  float* part_out; // [splits, B Hkv, R, D], not yet divided by the sums
  float2* part_ml; // [splits, B Hkv, R]: maximum (log2 units) and sum
};

// How the gradients' sums are cut, for work enough at once: those of dq over keys, those of dk and
// dv over rows.  The blocks of the keys that every later row sees (under a window) have many more
// rows than the others.
struct GradPlan {
  Divisor dq_splits;
  int wide_blocks; // blocks of kept keys, with wide_splits runs each; the others have splits
  Divisor wide_splits, splits;
  int blocks; // of keys
  __host__ __device__ int pieces() const {
    return wide_blocks * wide_splits.d + (blocks - wide_blocks) * splits.d;
  }
  __host__ __device__ bool dkv_split() const { return wide_splits.d > 1 || splits.d > 1; }
  // Those of which partial sums are kept: the first ones, the wide blocks'
  __host__ __device__ int part_pieces() const {
    return splits.d > 1 ? pieces() : wide_blocks * wide_splits.d;
  }
};

// The gradients' further operands.
struct AttentionGradArgs {
  AttentionArgs a; // out: the forward's result, lse: its sums
  const void* dout;
  void* dq;
  void* dk;
  void* dv;
  float* delta; // [B, Hq, Lq]: sum over D of dout * out
  float* largest; // float16: [B Hkv, splits of dq, 32 rows] of the probabilities' gradients
  int64_t dout_strides[3], dq_strides[3], dk_strides[3], dv_strides[3];
  float scale;
  GradPlan plan;
  float* part_dq;  // [splits, B Hkv, R, D] where dq is split
  float* part_dkv; // [piece, key of the block, 2, D] where dk and dv are
};

constexpr int kGradBlock = 128; // rows or keys of a workgroup

// One unit for each type: by the dtype of a call
int launch_attention_few_f32(const AttentionArgs& a, hipStream_t s);
int launch_attention_few_f16(const AttentionArgs& a, hipStream_t s);
int launch_attention_few_bf16(const AttentionArgs& a, hipStream_t s);
int launch_attention_rows_f32(const AttentionArgs& a, hipStream_t s);
int launch_attention_rows_f16(const AttentionArgs& a, hipStream_t s);
int launch_attention_rows_bf16(const AttentionArgs& a, hipStream_t s);
int launch_attention_join(const AttentionArgs& a, int dtype, hipStream_t s);
int launch_attention_grad_join(const AttentionGradArgs& g, int dtype, hipStream_t s);
int launch_attention_grad_f32(const AttentionGradArgs& g, hipStream_t s);
int launch_attention_grad_f16(const AttentionGradArgs& g, hipStream_t s);
int launch_attention_grad_bf16(const AttentionGradArgs& g, hipStream_t s);

#ifdef __HIPCC__

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// 8 consecutive values along a contraction, as one lane of an operand holds them.
template <typename T>
struct Frag {
  uint32_t w[4];
};
template <>
struct Frag<float> {
  float w[8];
};

template <typename T>
__device__ __forceinline__ uint4 frag_bits(const Frag<T>& f) {
  return make_uint4(f.w[0], f.w[1], f.w[2], f.w[3]);
}

// A sum that starts at zero, as the compiler is not to know: it splits vectors that it sees begin
// with constants into scalars where paths meet, and then moves all of them between the two files
// of registers around the products (16 times 16 of them in a tile of 256 columns).
__device__ __forceinline__ floatx16 zero_sum() {
  floatx16 x = {};
  asm("" : "+v"(x));
  return x;
}

// c + a b over 16 values of the contraction (8 in each half of the wave): one
// instruction for the 16-bit types; float32 takes eight of two values each.
template <typename T>
__device__ __forceinline__ floatx16 mma32(const Frag<T>& a, const Frag<T>& b, floatx16 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w[j], b.w[j], c, 0, 0, 0);
    }
    return c;
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// The same for 16 x 16 results over 32 values of the contraction.
template <typename T>
__device__ __forceinline__ floatx4 mma16(const Frag<T>& a, const Frag<T>& b, floatx4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.w[j], b.w[j], c, 0, 0, 0);
    }
    return c;
  } else {
    return mfma16<T>(frag_bits<T>(a), frag_bits<T>(b), c);
  }
}

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
  Frag<T> f;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(f.w) / 4); ++i) {
    f.w[i] = 0;
  }
  return f;
}

// 8 consecutive elements of memory (16-byte aligned)
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* p) {
  Frag<T> f;
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  if constexpr (sizeof(T) == 4) {
    const uint4 b = *reinterpret_cast<const uint4*>(p + 4);
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f.w[i] = __uint_as_float(u[i]);
    }
  } else {
    f.w[0] = a.x;
    f.w[1] = a.y;
    f.w[2] = a.z;
    f.w[3] = a.w;
  }
  return f;
}

// Negated where scale < 0 (exact), so that maxima are taken of what is exponentiated.
template <typename T>
__device__ __forceinline__ void flip(Frag<T>& f, uint32_t sign) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(f.w) / 4); ++i) {
    if constexpr (sizeof(T) == 4) {
      f.w[i] = __uint_as_float(__float_as_uint(f.w[i]) ^ sign);
    } else {
      f.w[i] ^= sign;
    }
  }
}

// Probabilities (or their gradients) as an operand.  For the 16-bit types this is where
// they are rounded to the type of the values they multiply: the matrix instruction takes
// both operands in one type, and a probability's relative error of 2^-9 (2^-12) is that of
// the value beside it.  Sums of probabilities are taken before it, in 32 bits.  Results are 1.4 times as
// far off as their own rounding for it (2048 tokens over 32768, bfloat16, against 64 bits 0.0023 of the
// norm instead of 0.0017).  A second term (rest_of) is taken where it costs nothing, of few rows; of many
// it would cost a quarter to a third: 1.02 ms would be 1.35, 4096 tokens under a window of 1024 86 us 107.
template <typename T>
__device__ __forceinline__ Frag<T> frag_of(const float* p) {
  Frag<T> f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f.w[i] = p[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.w[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
    }
  }
  return f;
}

// What rounding to frag_of's 16-bit operand took from 8 values
template <typename T>
__device__ __forceinline__ Frag<T> rest_of(const float* p, const Frag<T>& rounded) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t bits = static_cast<uint16_t>(rounded.w[i / 2] >> 16 * (i % 2));
    rest[i] = p[i] - to_f32(__builtin_bit_cast(T, bits));
  }
  return frag_of<T>(rest);
}

// 4 values to consecutive elements (aligned to all of them)
template <typename T>
__device__ __forceinline__ void store4(T* p, const floatx4& v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}

__device__ __forceinline__ bool not_finite(float v) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
}

// The values of a dword with zeros for infinities and NaN.
template <typename T>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return not_finite(__uint_as_float(w)) ? 0 : w;
  } else {
    constexpr uint32_t kExp = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
    w = (w & kExp) == kExp ? w & 0xffff0000u : w;
    return (w & (kExp << 16)) == (kExp << 16) ? w & 0xffffu : w;
  }
}

// This lane's value and that of lane ^ 32, in either order.
__device__ __forceinline__ float2 both_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_halves(float v) {
  const float2 r = both_halves(v);
  return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float sum_halves(float v) {
  const float2 r = both_halves(v);
  return r.x + r.y;
}
// ... over the lanes l % 16 + 0, 16, 32, 48
__device__ __forceinline__ float max_quarters(float v) {
  const uint32_t u = __float_as_uint(max_halves(v));
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_quarters(float v) {
  const uint32_t u = __float_as_uint(sum_halves(v));
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// ... and over all 64
template <int N>
__device__ __forceinline__ float rotated(float v) { // by N within 16 lanes
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max_lanes(float v) {
  v = fmaxf(v, rotated<8>(v));
  v = fmaxf(v, rotated<4>(v));
  v = fmaxf(v, rotated<2>(v));
  v = fmaxf(v, rotated<1>(v));
  return max_quarters(v);
}
__device__ __forceinline__ float sum_lanes(float v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  v += rotated<1>(v);
  return sum_quarters(v);
}

// N products whose LDS operands are read AHEAD products ahead: use(i, operand) and what it does
// beside the product stay in their order.  Left alone, the compiler reads an operand, waits for
// it, multiplies and reads the next: that takes the fewest registers.
template <typename T, int N, int AHEAD = 4, typename Read, typename Use>
__device__ __forceinline__ void read_ahead(const Read& read, const Use& use) {
  constexpr int kAhead = sizeof(T) == 4 ? 1 : N < AHEAD ? N : AHEAD;
  Frag<T> ring[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    ring[i] = read(i);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, ring[i % kAhead]);
    if (i + kAhead < N) {
      ring[i % kAhead] = read(i + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- which keys ----------------------------------------------------------------
// The rows of one tile of rows that see anything are first .. last; the keys they see lie
// in [0, a_end) (the ones that are kept) and [w_low, w_end), cut into tiles of KT keys.  Tiles
// begin at multiples of 16, whose keys lie in one page: the first of the second range with some
// keys that nobody sees.
struct KeyRange {
  int a_end, w_low, w_end;
  int a_tiles, tiles;
};

__device__ __forceinline__ KeyRange
keys_of(const AttentionArgs& a, int length, int first_row, int last_row, int kt) {
  const int p_lo = length - a.Lq + a.of_G.divide(first_row);
  const int p_hi = length - a.Lq + a.of_G.divide(last_row);
  KeyRange r;
  r.w_end = p_hi + 1;
  r.w_low = max(0, p_lo - a.window + 1);
  r.a_end = min(a.keep, p_hi + 1);
  if (r.a_end >= r.w_low) { // one range
    r.a_end = 0;
    r.w_low = 0;
  }
  r.a_tiles = (r.a_end + kt - 1) / kt;
  r.tiles = r.a_tiles + (r.w_end - (r.w_low & ~15) + kt - 1) / kt;
  return r;
}

// Keys of tile t: kt from `begin` on, of which [low, end) belong to it
struct KeyTile {
  int begin, low, end;
};
__device__ __forceinline__ KeyTile tile_of(const KeyRange& r, int t, int kt) {
  const bool a = t < r.a_tiles;
  KeyTile k;
  k.begin = a ? t * kt : (r.w_low & ~15) + (t - r.a_tiles) * kt;
  k.low = a ? 0 : r.w_low;
  k.end = min(k.begin + kt, a ? r.a_end : r.w_end);
  return k;
}
// Tiles [*first, *last) of run `split`: as equal as they come
__device__ __forceinline__ void
run_of(int tiles, int split, const Divisor& splits, int* first, int* last) {
  int rest;
  const int each = splits.divide(tiles, &rest);
  *first = split * each + min(split, rest);
  *last = *first + each + (split < rest ? 1 : 0);
}

// Whether positions lo .. hi see all of a tile
__device__ __forceinline__ bool
whole_tile(const AttentionArgs& a, const KeyTile& k, int kt, int lo, int hi) {
  return k.begin >= k.low && k.end - k.begin == kt && k.end - 1 <= lo &&
      (hi - k.begin < a.window || k.end <= a.keep);
}

// Whether a tile's keys [begin, end) are all seen by, or all hidden from, positions lo .. hi
__device__ __forceinline__ bool all_seen(
    int begin, int end, int lo, int hi, int window, int keep) {
  return end - 1 <= lo && (hi - begin < window || end <= keep);
}
__device__ __forceinline__ bool none_seen(
    int begin, int end, int lo, int hi, int window, int keep) {
  return begin > hi || (lo - (end - 1) >= window && begin >= keep);
}

// Which of its keys a lane sees, n = key - begin - (its own first): counted from there, each
// comparison is with a constant and no key's number takes a register.
struct Seen {
  int low, last, from, keep;
  __device__ __forceinline__ Seen(const AttentionArgs& a, const KeyTile& t, int p, int own)
      : low(t.low - t.begin - own),
        last(min(p, t.end - 1) - t.begin - own),
        from(p - a.window + 1 - t.begin - own),
        keep(a.keep - t.begin - own) {}
  __device__ __forceinline__ bool operator()(int n) const {
    return n >= low && n <= last && (n >= from || n < keep);
  }
};

// The bits below x
__device__ __forceinline__ uint32_t bits_below(int x) {
  return x >= 32 ? ~0u : (1u << max(x, 0)) - 1;
}

// The same of keys first .. first + 31 of a tile, a bit each
__device__ __forceinline__ uint32_t seen_bits(
    const AttentionArgs& a, const KeyTile& t, int p, int first) {
  const int begin = t.begin + first;
  const int low = t.low - begin, to = min(p + 1, t.end) - begin;
  return (bits_below(to) & ~bits_below(max(low, p - a.window + 1 - begin))) |
      (bits_below(min(a.keep - begin, to)) & ~bits_below(low));
}

// Offsets of key j's row in k and in v: through the page table, whose entries are clamped to
// pages that exist, or along contiguous keys.
struct KeyRow {
  int64_t k, v;
};
template <bool PAGED>
__device__ __forceinline__ KeyRow key_row(const AttentionArgs& a, int b, int hk, int j) {
  int64_t first = b;
  int at = j;
  if constexpr (PAGED) {
    int in_page;
    const int page = a.page.divide(j, &in_page);
    const int id = a.table[b * a.table_stride + page];
    first = min(max(id, 0), a.pages - 1);
    at = in_page;
  }
  KeyRow r;
  r.k = first * a.k_strides[0] + hk * a.k_strides[1] + at * a.k_strides[2];
  r.v = first * a.v_strides[0] + hk * a.v_strides[1] + at * a.v_strides[2];
  return r;
}

// Length of a sequence, within the keys that it can have
__device__ __forceinline__ int length_of(const AttentionArgs& a, int b) {
  return a.lengths == nullptr ? a.keys : min(max(a.lengths[b], 0), a.keys);
}

// Offset of row r's token in a [sequence, head, token] tensor
__device__ __forceinline__ int64_t row_offset(
    const int64_t (&strides)[3], int b, int hk, const Divisor& G, int r) {
  int g;
  const int i = G.divide(r, &g);
  return b * strides[0] + (hk * G.d + g) * strides[1] + i * strides[2];
}

// Which (sequence, key head) and which of its pieces a workgroup has.  Workgroups go to the 8 dies
// in turn, and each die has an L2 of its own: eight heads side by side, one on each die, so that
// all that read a head's keys find them in one L2.  A head's pieces come with the most work first.
//
// Where two workgroups fit a CU (`pairs`) and all do at once, workgroup n shares one with n + 256:
// of a die's workgroups by work the first 32 are followed by the others from the last on, so that
// much work is beside little.  Causal, 2048 tokens, 16 heads of 64, float32 103 us instead of 152,
// twice 1000, 32 of 64 on 8, bfloat16 22.7 instead of 28.0; the gradients of 4 times 900 tokens, 16
// heads of 80, float32 539 instead of 735.
constexpr int kPairBytes = 384; // of a row: two workgroups fit a CU up to there

struct Grid {
  int heads, pieces;
  int last; // number of a die's last workgroup, if they are paired, else 0
  Divisor of_eight, of_last; // 8 pieces; the heads of the last, smaller group, or the groups if paired
  Grid(int64_t heads_, int64_t pieces_, bool pairs)
      : heads(static_cast<int>(heads_)),
        pieces(static_cast<int>(pieces_)),
        last(pairs && heads_ % 8 == 0 && heads_ * pieces_ > 256 && heads_ * pieces_ <= 512
                 ? static_cast<int>(heads_ * pieces_ / 8 - 1)
                 : 0),
        of_eight(8 * pieces_),
        of_last(last > 0 ? heads_ / 8 : heads_ % 8) {}
  unsigned blocks() const { return static_cast<unsigned>(heads) * pieces; }
  __device__ __forceinline__ void find(int* head, int* piece) const {
    int rest, at;
    if (last > 0) {
      int n = static_cast<int>(blockIdx.x >> 3), group;
      n = n < 32 ? n : 32 + last - n;
      *piece = of_last.divide(n, &group);
      *head = group * 8 + static_cast<int>(blockIdx.x & 7);
      return;
    }
    const int group = of_eight.divide(blockIdx.x, &rest);
    if (group * 8 + 8 <= heads) {
      at = rest & 7;
      *piece = rest >> 3;
    } else {
      *piece = of_last.divide(rest, &at);
    }
    *head = group * 8 + at;
  }
};

// ---- tiles in LDS -----------------------------------------------------------------
typedef __attribute__((address_space(3))) const char* LdsBytes;

// Rows of DT elements in 16-byte units, a power of two of places for them, unit u of row r at
// place u ^ swizzle(r).  LDS has 64 banks: sixteen rows read at one unit (load_rows) and four rows
// read 64 bytes wide (load_cols) lie in all of them once.
template <typename T, int DT>
struct Tile {
  static constexpr int kUnit = 16 / sizeof(T);
  static constexpr int kPitch = DT == 96 ? 128 : DT;
  static constexpr int kPlaces = kPitch / kUnit;
  static constexpr int kRowsOfLoad = 64 / kPlaces; // that the 64 lanes of one load cover
  static constexpr int kRowsOfPass = 4 * kRowsOfLoad; // ... and those of a workgroup's four waves
  // Loads after which a lane's columns repeat (the swizzle has the low bits of a row's number)
  static constexpr int kTurns = kRowsOfPass >= 16 ? 1 : 16 / kRowsOfPass;

  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (kPlaces == 8) { // two rows to the banks' width
      return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    } else {
      return (row & 3) << 2 | (row >> 2 & 3);
    }
  }
  static __device__ __forceinline__ int at(int row, int unit) {
    return row * kPitch + (unit ^ swizzle(row)) * kUnit;
  }
  // Elements 16 c + 8 h .. 16 c + 8 h + 7 of row `row` + lane % 32, h = lane / 32; row: a multiple of
  // 32.  Tiles are aligned to 1024 bytes, the longest row: the unit's number is exclusive ored into
  // the address.
  static __device__ __forceinline__ Frag<T> load_rows(const T* tile, int row, int c, int lane) {
    constexpr int kOf8 = 8 / kUnit; // units of 8 elements
    const int r = lane & 31;
    const uint32_t own =
        (r * kPlaces + ((kOf8 * (lane >> 5)) ^ swizzle(r))) * 16 + lds_address(tile);
    const uint32_t p = own ^ (2 * kOf8 * c * 16);
    Frag<T> f;
    const auto a = *(__attribute__((address_space(3))) const raw_u32x4*)(
        (LdsBytes)(uintptr_t)p + row * kPitch * sizeof(T));
    if constexpr (sizeof(T) == 4) {
      const auto b = *(__attribute__((address_space(3))) const raw_u32x4*)(
          (LdsBytes)(uintptr_t)(p ^ 16) + row * kPitch * sizeof(T));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.w[i] = __uint_as_float(a[i]);
        f.w[4 + i] = __uint_as_float(b[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.w[i] = a[i];
      }
    }
    return f;
  }
  // element d + lane % 32 of rows row + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3}; row: a multiple of
  // 16, d of 32.  The transposing read takes four rows of 16 columns from 16 lanes' addresses and
  // gives each lane a column.
  static __device__ __forceinline__ Frag<T> load_cols(const T* tile, int row, int d, int lane) {
    Frag<T> f;
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      const int c = d + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = row + 8 * (j / 4) + 4 * h + j % 4;
        f.w[j] = tile[at(r, c / 4) + c % 4];
      }
    } else {
      const int y = 4 * h + (lane >> 2 & 3); // row of the first four
      const int u = (lane >> 4 & 1) << 1 | (lane >> 1 & 1);
      const uint32_t own =
          (y * kPlaces + (u ^ swizzle(y))) * 16 + 8 * (lane & 1) + lds_address(tile);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t p = own ^ ((d / 8) ^ (swizzle(8 * half))) * 16;
        const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) shortx4*)(
                (LdsBytes)(uintptr_t)p + (row + 8 * half) * kPitch * sizeof(T)));
        const uint2 w = __builtin_bit_cast(uint2, x);
        f.w[2 * half] = w.x;
        f.w[2 * half + 1] = w.y;
      }
    }
    return f;
  }
};

// 64 lanes x 16 bytes from each lane's own address to LDS, lane by lane from `at` (uniform);
// vmcnt counts them (the wait state behind the write of M0: see dma16).
__device__ __forceinline__ void dma16_from(uint32_t at, const void* p) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(p), "s"(at)
               : "memory");
}
// dma16 from an address that is the same in all lanes, wherever the compiler keeps it: if a vector
// instruction writes the scalar registers right before, the load has to keep five wait states
// behind it, which the compiler does not do for inline assembly.
__device__ __forceinline__ void dma16_at(uint32_t at, uint32_t voff, const void* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u)); // (an int)
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
  const uint64_t base = static_cast<uint64_t>(hi) << 32 | lo;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(voff), "s"(base), "s"(at)
               : "memory");
}
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- what is not finite ------------------------------------------------------------
// A masked value that is not finite would reach rows that do not see it: 0 * inf.  Tiles that not
// all rows see are looked through for such values (the exponent's bits, plus one, carry into the
// sign's place).  Where there are any, the product takes zeros for them, and when the result
// is stored the rows that do see them get them (store_infinite; of keys and of the gradients' rows
// they are added; added twice they change nothing).
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  constexpr uint32_t kOne = sizeof(T) == 4           ? 0x00800000u
      : std::is_same<T, bf16_t>::value ? 0x00800080u
                                       : 0x04000400u;
  constexpr uint32_t kMagnitude = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  return (w & kMagnitude) + kOne;
}
template <typename T>
__device__ __forceinline__ bool is_odd(uint32_t bits) {
  return (bits & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u)) != 0;
}

// Whether this thread's 256th of a tile in LDS has one
template <typename T, int ELEMENTS>
__device__ __forceinline__ bool odd_values(const T* tile) {
  constexpr int kUnit = 16 / sizeof(T);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < ELEMENTS / (256 * kUnit); ++i) {
    const uint4 w =
        *reinterpret_cast<const uint4*>(tile + (i * 256 + static_cast<int>(threadIdx.x)) * kUnit);
    bits |= odd_bits<T>(w.x) | odd_bits<T>(w.y) | odd_bits<T>(w.z) | odd_bits<T>(w.w);
  }
  return is_odd<T>(bits);
}

// Whether any thread of the workgroup says so, as a scalar: what follows from it does too
__device__ __forceinline__ bool any_of_block(bool v) {
  return __builtin_amdgcn_readfirstlane(__syncthreads_or(v)) != 0;
}

// This thread's 256th of a tile, with zeros for what is not finite
template <typename T, int ELEMENTS>
__device__ __forceinline__ void copy_finite(const T* from, T* to) {
  constexpr int kUnit = 16 / sizeof(T);
  for (int i = threadIdx.x * kUnit; i < ELEMENTS; i += 256 * kUnit) {
    const uint4 w = *reinterpret_cast<const uint4*>(from + i);
    *reinterpret_cast<uint4*>(to + i) = make_uint4(
        finite_part<T>(w.x), finite_part<T>(w.y), finite_part<T>(w.z), finite_part<T>(w.w));
  }
}

// p[at] += x in the type of p
template <typename T>
__device__ __forceinline__ void add_to(T* p, float x) {
  *p = from_f32<T>(to_f32(*p) + x);
}

// Row r among the sums that the gradients need
__device__ __forceinline__ int64_t lse_at(const AttentionArgs& a, int b, int hk, int r) {
  int g;
  const int i = a.of_G.divide(r, &g);
  return (static_cast<int64_t>(b) * a.Hq + hk * a.G + g) * a.Lq + i;
}

// Four columns of a result, and what rounding takes from them: delta would be as far off as the
// gradients' own rounding (of tokens that see few), were it formed from the rounded result alone
template <typename T>
__device__ __forceinline__ T* low_of(const AttentionArgs& a, int64_t row) { // (row: lse_at)
  return a.low == nullptr ? nullptr : static_cast<T*>(a.low) + row * a.D;
}
template <typename T>
__device__ __forceinline__ void store_result(T* out, T* low, floatx4 x) {
  store4<T>(out, x);
  if constexpr (sizeof(T) == 2) {
    if (low != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float rounded = to_f32(from_f32<T>(x[i]));
        x[i] = not_finite(rounded) ? 0.0f : x[i] - rounded;
      }
      store4<T>(low, x);
    }
  }
}

// Stores of this workgroup are behind, its threads may add to them
__device__ __forceinline__ void after_stores() {
  __threadfence_block();
  __syncthreads();
}

__device__ __forceinline__ bool sees_key(const AttentionArgs& a, int p, int j) {
  return j <= p && (p - j < a.window || j < a.keep);
}

// Column d of the rows lo .. hi that see a value of v which is not finite: the sum of all such values
// that they see, whatever the products made of it (NaN, where a probability was rounded to zero).  A
// row whose sum of probabilities is NaN stays NaN.  tile(t): a tile's keys, value(j): that of key j,
// total(r): a row's sum, with(r, store): calls store with the place of row r's result.
template <typename Tile, typename Value, typename Total, typename With>
__device__ __forceinline__ void store_infinite(
    const AttentionArgs& a, int d, int t0, int t1, const Tile& tile, const Value& value, int lo,
    int hi, int p0, const Total& total, const With& with) {
  for (int turn = 0; turn < 2; ++turn) { // zeros, then the sums
    for (int t = t0; t < t1 && d < a.D; ++t) {
      const KeyTile k = tile(t);
      for (int j = max(k.begin, k.low); j < k.end; ++j) {
        const float x = value(j);
        for (int r = lo; not_finite(x) && r <= hi; ++r) {
          if (sees_key(a, p0 + a.of_G.divide(r), j) && total(r) == total(r)) {
            with(r, [&](auto* p) {
              using T = std::remove_reference_t<decltype(*p)>;
              *p = turn == 0 ? from_f32<T>(0.0f) : from_f32<T>(to_f32(*p) + x);
            });
          }
        }
      }
    }
  }
}

#endif // __HIPCC__

} // namespace mlxrocm

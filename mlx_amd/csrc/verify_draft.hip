// verify_draft.hip -- drafted tokens against the probabilities of the model that they were
// drafted for, so that what is kept is distributed as that model's own samples.
//
// Draft x_i is taken while u_i q_i(x_i) < p_i(x_i) (u: given numbers in [0, 1); without q,
// drafts are certain: q_i(x_i) = 1).  At the first that is not, n, a token is drawn from
// max(p_n - q_n, 0) (from p_n if that is zero throughout); if all were taken, from p_n.
//
// The draw has to be the same whatever the order in which weights are summed: a weight w
// counts as the whole number floor(min(w, 1) 2^40), sums of up to 2^22 of them are exact in
// 64 bits, and the token is the first whose running sum exceeds t = min(floor(u N), N - 1),
// N their total.  Probabilities below 2^-40 are not drawn.
//
// Two kernels: sums of parts of the one row that is drawn from (bound by reading it), then one
// workgroup for each sequence finds the part and the token in it (bound by the latency of a few
// dependent reads, for which the first kernel leaves n behind).  32 sequences, 128256 tokens, f32:
// 6.9 us and 3.9 us; one sequence, 32000 tokens: 3.8 us and 2.4 us.
#include "common.h"

namespace mlxrocm {

namespace {

constexpr int kPart = 1024; // values of a row that a wave sums
constexpr int kChunk = 4 * kPart; // that a workgroup sums
constexpr int kMostVocab = 1 << 22;

struct VerifyArgs {
  const int32_t* draft; // [B, K]
  const void* target;   // [B, K + 1, V]
  const void* probs;    // [B, K, V], or null
  const float* accept;  // [B, K]
  const float* sample;  // [B]
  const int32_t* lengths; // [B], or null: K drafts each
  int32_t* tokens;      // [B, K + 1]
  int32_t* accepted;    // [B]
  int B, K, V, parts;
  int64_t target_strides[2], probs_strides[2]; // [sequence, draft]
  uint64_t* sums; // [B, parts, 2]: of the weights; of p, where that of the weights is zero
  int32_t* taken; // [B]
};

__device__ __forceinline__ uint64_t whole(float w) {
  // (NaN counts nothing)
  return w > 0.0f ? static_cast<uint64_t>(fminf(w, 1.0f) * 0x1p40f) : 0;
}

// How many drafts of sequence b are taken: the whole wave asks, 64 drafts at a time.  (What does
// not depend on what is read comes first: each read is a wait.)
template <typename T>
__device__ __forceinline__ int taken(const VerifyArgs& a, int b, int drafted) {
  const T* target = static_cast<const T*>(a.target) + b * a.target_strides[0];
  const T* probs = static_cast<const T*>(a.probs) + b * a.probs_strides[0];
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < drafted; i0 += 64) {
    const int i = i0 + lane;
    const int64_t at = static_cast<int64_t>(b) * a.K + min(i, a.K - 1); // (drafted > 0: K > 0)
    const int x = a.draft[at];
    const double u = a.accept[at];
    bool out = i < drafted;
    if (out && x >= 0 && x < a.V) {
      const double p = to_f32(target[i * a.target_strides[1] + x]);
      const double q = a.probs == nullptr ? 1.0 : to_f32(probs[i * a.probs_strides[1] + x]);
      out = !(u * q < p); // a product of two 32-bit values is exact in 64
    }
    const uint64_t mask = __ballot(out);
    if (mask != 0) {
      return i0 + __ffsll(static_cast<unsigned long long>(mask)) - 1;
    }
  }
  return drafted;
}

__device__ __forceinline__ int drafted_of(const VerifyArgs& a, int b) {
  return a.lengths == nullptr ? a.K : min(max(a.lengths[b], 0), a.K);
}

// The row that sequence b draws from
template <typename T>
struct Row {
  const T* p;
  const T* q;  // null: none to take away
  int without; // the token that counts nothing, or -1

  __device__ __forceinline__ Row(const VerifyArgs& a, int b, int n, int drafted) {
    p = static_cast<const T*>(a.target) + b * a.target_strides[0] + n * a.target_strides[1];
    q = nullptr;
    without = -1;
    if (n < drafted) {
      if (a.probs != nullptr) {
        q = static_cast<const T*>(a.probs) + b * a.probs_strides[0] + n * a.probs_strides[1];
      } else {
        without = a.draft[static_cast<int64_t>(b) * a.K + n];
      }
    }
  }
  // Values j .. j + 3 of p and the weights of the draw; nothing past V
  __device__ __forceinline__ void load(int j, int V, float (&pj)[4], float (&w)[4]) const {
    float qj[4];
    four(p, j, V, pj);
    if (q != nullptr) {
      four(q, j, V, qj);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = q != nullptr ? pj[i] - qj[i] : j + i == without ? 0.0f : pj[i];
    }
  }

  // (one load where the row begins at a multiple of four values: the same for all)
  static __device__ __forceinline__ void four(const T* of, int j, int V, float (&v)[4]) {
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    };
    if (reinterpret_cast<uintptr_t>(of) % sizeof(Four) == 0 && j + 3 < V) {
      const Four x = *reinterpret_cast<const Four*>(of + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = to_f32(x.v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = j + i < V ? to_f32(of[j + i]) : 0.0f;
      }
    }
  }
};

// v of another lane of the wave, 0 where there is none or ROWS (of 16 lanes) leaves this one out
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(
      0, static_cast<int>(static_cast<uint32_t>(v)), CONTROL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(
      0, static_cast<int>(static_cast<uint32_t>(v >> 32)), CONTROL, ROWS, 0xf, false);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// Sums of lanes 0 .. this one
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += moved<0x111, 0xf>(v); // from 1, 2, 4 and 8 lanes below
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v); // the last lane of a row for the next row, of rows 0 and 2
  v += moved<0x143, 0xc>(v); // lane 31 for the upper half
  return v;
}

// Workspace of a sequence: two sums for each part, and how many drafts are taken
inline int parts_of(int V) {
  return (V + kPart - 1) / kPart;
}

template <typename T>
__global__ __launch_bounds__(256) void verify_sums_kernel(const VerifyArgs a) {
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int part = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int drafted = drafted_of(a, b);
  const int n = taken<T>(a, b, drafted);
  const Row<T> row(a, b, n, drafted);
  constexpr int kTurns = kPart / 256;
  float p[kTurns][4], w[kTurns][4];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    row.load(part * kPart + 256 * i + 4 * lane, a.V, p[i], w[i]);
  }
  const auto sum = [](const float (&of)[kTurns][4]) {
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s += whole(of[i][j]);
      }
    }
    const uint64_t all = wave_scan(s); // of the wave in lane 63
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(all), 63);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(all >> 32), 63);
    return static_cast<uint64_t>(hi) << 32 | lo;
  };
  const uint64_t of_w = sum(w);
  // where a weight is not zero anywhere, nothing is drawn from p itself
  const uint64_t of_p = of_w == 0 ? sum(p) : 0;
  if (part < a.parts && lane < 2) {
    a.sums[(static_cast<int64_t>(b) * a.parts + part) * 2 + lane] = lane == 0 ? of_w : of_p;
  }
  if (blockIdx.x == 0) { // all but the token that is drawn
    for (int i = threadIdx.x; i <= a.K; i += 256) {
      if (i != n) {
        a.tokens[static_cast<int64_t>(b) * (a.K + 1) + i] =
            i < n ? a.draft[static_cast<int64_t>(b) * a.K + i] : -1;
      }
    }
    if (threadIdx.x == 0) {
      a.accepted[b] = n;
      a.taken[b] = n;
    }
  }
}

// Sums of the values of threads 0 .. this one
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* wave_totals) {
  const int lane = threadIdx.x & 63;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) {
    wave_totals[threadIdx.x >> 6] = v;
  }
  __syncthreads();
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) {
    v += wave_totals[w];
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void verify_pick_kernel(const VerifyArgs a) {
  __shared__ uint64_t totals[4];
  __shared__ uint64_t before; // sum of the parts before the one that is drawn from
  __shared__ int found;
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int n = a.taken[b];
  const float u = a.sample[b];
  const Row<T> row(a, b, n, drafted_of(a, b));
  const uint64_t* sums = a.sums + static_cast<int64_t>(b) * a.parts * 2;
  const int each = (a.parts + 255) / 256;
  const int begin = min(tid * each, a.parts), end = min(begin + each, a.parts);
  uint64_t w_sum = 0, p_sum = 0;
  for (int c = begin; c < end; ++c) {
    w_sum += sums[2 * c];
    p_sum += sums[2 * c + 1];
  }
  if (tid == 0) {
    found = -1;
  }
  uint64_t mine = w_sum;
  uint64_t up_to = block_scan(mine, totals);
  uint64_t N = totals[0] + totals[1] + totals[2] + totals[3];
  const bool of_p = N == 0;
  if (of_p) { // the same for all
    mine = p_sum;
    up_to = block_scan(mine, totals);
    N = totals[0] + totals[1] + totals[2] + totals[3];
  }
  uint64_t t = 0;
  if (N > 0) {
    const double at = floor(static_cast<double>(u) * static_cast<double>(N));
    t = at >= 0.0 ? (at < static_cast<double>(N) ? static_cast<uint64_t>(at) : N - 1) : 0;
    t = t < N ? t : N - 1;
    uint64_t sum = up_to - mine;
    if (sum <= t && t < up_to) { // (one thread)
      int c = begin;
      for (; c < end - 1; ++c) {
        const uint64_t next = sum + sums[2 * c + (of_p ? 1 : 0)];
        if (t < next) {
          break;
        }
        sum = next;
      }
      found = c;
      before = sum;
    }
  }
  __syncthreads();
  const int64_t to = static_cast<int64_t>(b) * (a.K + 1) + n;
  if (found < 0) { // nothing to draw from; the same for all
    if (tid == 0) {
      a.tokens[to] = -1;
    }
    return;
  }
  float p[4], w[4];
  const int j0 = found * kPart + 4 * tid;
  row.load(j0, a.V, p, w);
  uint64_t weight[4], of_four = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    weight[i] = whole(of_p ? p[i] : w[i]);
    of_four += weight[i];
  }
  uint64_t sum = before + block_scan(of_four, totals) - of_four;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sum <= t && t < sum + weight[i]) { // (one of them)
      a.tokens[to] = j0 + i;
    }
    sum += weight[i];
  }
}

} // namespace

} // namespace mlxrocm

extern "C" size_t mlxrocm_verify_draft_workspace_size(int B, int V) {
  if (B <= 0 || V <= 0) {
    return 0;
  }
  return static_cast<size_t>(B) *
      (mlxrocm::parts_of(V) * 2 * sizeof(uint64_t) + sizeof(int32_t));
}

extern "C" int mlxrocm_verify_draft(
    const int32_t* draft,
    const void* target,
    const void* probs,
    const float* accept,
    const float* sample,
    const int32_t* lengths,
    int32_t* tokens,
    int32_t* accepted,
    int B,
    int K,
    int V,
    const int64_t* strides,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_verify_draft");
  using namespace mlxrocm;
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[verify_draft] unknown dtype %d", dtype);
  }
  if (B < 0 || K < 0 || V <= 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[verify_draft] negative dimension or no vocabulary");
  }
  if (V > kMostVocab || B > 65535) {
    return fail(
        MLXROCM_UNSUPPORTED, "[verify_draft] %d sequences of %d probabilities exceed the grid", B, V);
  }
  if (B == 0) {
    return MLXROCM_OK;
  }
  if (target == nullptr || sample == nullptr || tokens == nullptr || accepted == nullptr ||
      strides == nullptr || (K > 0 && (draft == nullptr || accept == nullptr))) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[verify_draft] null pointer");
  }
  const size_t need = mlxrocm_verify_draft_workspace_size(B, V);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[verify_draft] workspace of %zu bytes, %zu needed",
        workspace_bytes, need);
  }
  VerifyArgs a{};
  a.draft = draft;
  a.target = target;
  a.probs = K > 0 ? probs : nullptr;
  a.accept = accept;
  a.sample = sample;
  a.lengths = lengths;
  a.tokens = tokens;
  a.accepted = accepted;
  a.B = B;
  a.K = K;
  a.V = V;
  a.parts = parts_of(V);
  a.target_strides[0] = strides[0];
  a.target_strides[1] = strides[1];
  a.probs_strides[0] = strides[2];
  a.probs_strides[1] = strides[3];
  a.sums = static_cast<uint64_t*>(workspace);
  a.taken = reinterpret_cast<int32_t*>(a.sums + static_cast<int64_t>(B) * a.parts * 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    verify_sums_kernel<T><<<dim3((V + kChunk - 1) / kChunk, B), 256, 0, s>>>(a);
    MLXROCM_HIP_TRY(hipGetLastError());
    verify_pick_kernel<T><<<B, 256, 0, s>>>(a);
    MLXROCM_HIP_TRY(hipGetLastError());
    return static_cast<int>(MLXROCM_OK);
  });
}

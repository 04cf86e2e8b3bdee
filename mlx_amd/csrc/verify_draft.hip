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
// Two kernels: sums of chunks of the one row that is drawn from (bound by reading it), then one
// workgroup for each sequence finds the chunk and the token in it.
#include "common.h"

namespace mlxrocm {

namespace {

constexpr int kChunk = 4096; // values of a row that a workgroup sums
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
  int B, K, V, chunks;
  int64_t target_strides[2], probs_strides[2]; // [sequence, draft]
  uint64_t* sums; // [B, chunks, 2]: of the weights, of p
};

__device__ __forceinline__ uint64_t whole(float w) {
  // (NaN counts nothing)
  return w > 0.0f ? static_cast<uint64_t>(fminf(w, 1.0f) * 0x1p40f) : 0;
}

// How many drafts of sequence b are taken: the whole wave asks, 64 drafts at a time
template <typename T>
__device__ __forceinline__ int taken(const VerifyArgs& a, int b, int drafted) {
  const T* target = static_cast<const T*>(a.target) + b * a.target_strides[0];
  const T* probs = static_cast<const T*>(a.probs) + b * a.probs_strides[0];
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < drafted; i0 += 64) {
    const int i = i0 + lane;
    bool out = i < drafted;
    if (out) {
      const int x = a.draft[static_cast<int64_t>(b) * a.K + i];
      if (x >= 0 && x < a.V) {
        const double p = to_f32(target[i * a.target_strides[1] + x]);
        const double q = a.probs == nullptr ? 1.0 : to_f32(probs[i * a.probs_strides[1] + x]);
        // a product of two 32-bit values is exact in 64
        out = !(static_cast<double>(a.accept[static_cast<int64_t>(b) * a.K + i]) * q < p);
      }
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
  __device__ __forceinline__ float weight(int j, float pj) const {
    return q != nullptr ? pj - to_f32(q[j]) : j == without ? 0.0f : pj;
  }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    v += __shfl_xor(static_cast<unsigned long long>(v), off, 64);
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void verify_sums_kernel(const VerifyArgs a) {
  __shared__ uint64_t part[4][2];
  const int b = blockIdx.y;
  const int drafted = drafted_of(a, b);
  const Row<T> row(a, b, taken<T>(a, b, drafted), drafted);
  uint64_t w = 0, p = 0;
  const int begin = blockIdx.x * kChunk;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int j = begin + i * 256 + static_cast<int>(threadIdx.x);
    if (j < a.V) {
      const float pj = to_f32(row.p[j]);
      w += whole(row.weight(j, pj));
      p += whole(pj);
    }
  }
  w = wave_sum64(w);
  p = wave_sum64(p);
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6][0] = w;
    part[threadIdx.x >> 6][1] = p;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const int x = threadIdx.x;
    a.sums[(static_cast<int64_t>(b) * a.chunks + blockIdx.x) * 2 + x] =
        part[0][x] + part[1][x] + part[2][x] + part[3][x];
  }
}

// Sums of the values of threads 0 .. this one
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* wave_totals) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t below = __shfl_up(static_cast<unsigned long long>(v), off, 64);
    v += lane >= off ? below : 0;
  }
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
  __shared__ uint64_t before; // sum of the chunks before the one that is drawn from
  __shared__ int chunk, token;
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int drafted = drafted_of(a, b);
  const int n = taken<T>(a, b, drafted);
  const Row<T> row(a, b, n, drafted);
  const uint64_t* sums = a.sums + static_cast<int64_t>(b) * a.chunks * 2;
  // (chunks: at most 1024, four to a thread)
  const int c0 = 4 * tid;
  uint64_t w[4], p[4], w_sum = 0, p_sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = c0 + i < a.chunks;
    w[i] = in ? sums[2 * (c0 + i)] : 0;
    p[i] = in ? sums[2 * (c0 + i) + 1] : 0;
    w_sum += w[i];
    p_sum += p[i];
  }
  if (tid == 0) {
    chunk = -1;
    token = -1;
  }
  uint64_t end = block_scan(w_sum, totals);
  uint64_t N = totals[0] + totals[1] + totals[2] + totals[3];
  const bool of_p = N == 0;
  if (of_p) { // the same for all
    end = block_scan(p_sum, totals);
    N = totals[0] + totals[1] + totals[2] + totals[3];
  }
  const float u = a.sample[b];
  uint64_t t = 0;
  if (N > 0) {
    const double at = floor(static_cast<double>(u) * static_cast<double>(N));
    t = at >= 0.0 ? (at < static_cast<double>(N) ? static_cast<uint64_t>(at) : N - 1) : 0;
    t = t < N ? t : N - 1;
    uint64_t sum = end - (of_p ? p_sum : w_sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t next = sum + (of_p ? p[i] : w[i]);
      if (sum <= t && t < next) {
        chunk = c0 + i;
        before = sum;
      }
      sum = next;
    }
  }
  __syncthreads();
  const int c = chunk;
  if (c >= 0) { // the same for all
    constexpr int kEach = kChunk / 256;
    const int j0 = c * kChunk + tid * kEach;
    uint64_t each[kEach], mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int j = j0 + i;
      const float pj = j < a.V ? to_f32(row.p[j]) : 0.0f;
      each[i] = j < a.V ? whole(of_p ? pj : row.weight(j, pj)) : 0;
      mine += each[i];
    }
    uint64_t sum = before + block_scan(mine, totals) - mine;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (sum <= t && t < sum + each[i]) {
        token = j0 + i;
      }
      sum += each[i];
    }
    __syncthreads();
  }
  const int drawn = token;
  for (int i = tid; i <= a.K; i += 256) {
    a.tokens[static_cast<int64_t>(b) * (a.K + 1) + i] =
        i < n ? a.draft[static_cast<int64_t>(b) * a.K + i] : i == n ? drawn : -1;
  }
  if (tid == 0) {
    a.accepted[b] = n;
  }
}

} // namespace

} // namespace mlxrocm

extern "C" size_t mlxrocm_verify_draft_workspace_size(int B, int V) {
  if (B <= 0 || V <= 0) {
    return 0;
  }
  return static_cast<size_t>(B) * ((V + mlxrocm::kChunk - 1) / mlxrocm::kChunk) * 2 *
      sizeof(uint64_t);
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
  a.chunks = (V + kChunk - 1) / kChunk;
  a.target_strides[0] = strides[0];
  a.target_strides[1] = strides[1];
  a.probs_strides[0] = strides[2];
  a.probs_strides[1] = strides[3];
  a.sums = static_cast<uint64_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    verify_sums_kernel<T><<<dim3(a.chunks, B), 256, 0, s>>>(a);
    MLXROCM_HIP_TRY(hipGetLastError());
    verify_pick_kernel<T><<<B, 256, 0, s>>>(a);
    MLXROCM_HIP_TRY(hipGetLastError());
    return static_cast<int>(MLXROCM_OK);
  });
}

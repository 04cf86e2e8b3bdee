// paged_cache.hip -- new keys and values into the pages of a cache.
//
// Token i of sequence b goes to position p = lengths[b] - L + i: row p % page of page
// table[b][p / page], for each head.  Positions before 0 are padding.  A copy, 16 bytes a
// thread; what bounds it is reading and writing them: 16 prompts of up to 1531 tokens, 4 heads of 128,
// 56 MB, 13.4 us; one token 2.5 us, a launch.
#include "common.h"

namespace mlxrocm {

namespace {

struct UpdateArgs {
  const char* from[2]; // k, v
  char* to[2];
  const int32_t* table;
  const int32_t* lengths;
  int H, L, units; // units of 16 bytes of a head's row
  int pages, page, table_width;
  int64_t table_stride;
  int64_t from_strides[2][3], to_strides[2][3]; // bytes: [sequence, head, token], [page, head, row]
  int64_t n;                                    // B L H units
};

__global__ __launch_bounds__(256) void paged_update_kernel(const UpdateArgs a) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (n >= a.n) {
    return;
  }
  const int64_t row = n / a.units;
  const int unit = static_cast<int>(n - row * a.units);
  const int64_t token = row / a.H;
  const int head = static_cast<int>(row - token * a.H);
  const int b = static_cast<int>(token / a.L);
  const int i = static_cast<int>(token - static_cast<int64_t>(b) * a.L);
  const int64_t p = static_cast<int64_t>(a.lengths[b]) - a.L + i;
  if (p < 0 || p >= static_cast<int64_t>(a.table_width) * a.page) {
    return;
  }
  const int at = static_cast<int>(p) / a.page;
  const int slot = static_cast<int>(p) - at * a.page;
  const int page = a.table[b * a.table_stride + at];
  if (page < 0 || page >= a.pages) {
    return;
  }
  const int w = blockIdx.y;
  const int64_t (&fs)[3] = a.from_strides[w];
  const int64_t (&ts)[3] = a.to_strides[w];
  const char* src = a.from[w] + b * fs[0] + head * fs[1] + i * fs[2] + unit * 16;
  char* dst = a.to[w] + page * ts[0] + head * ts[1] + slot * ts[2] + unit * 16;
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
}

} // namespace

} // namespace mlxrocm

extern "C" int mlxrocm_paged_cache_update(
    const void* k,
    const void* v,
    void* k_pages,
    void* v_pages,
    const int32_t* table,
    const int32_t* lengths,
    int B,
    int Hkv,
    int L,
    int D,
    int pages,
    int page_size,
    int table_width,
    const int64_t* strides,
    int dtype,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_paged_cache_update");
  using namespace mlxrocm;
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[paged_cache_update] unknown dtype %d", dtype);
  }
  if (B < 0 || Hkv < 0 || L < 0 || D < 0 || pages < 0 || table_width < 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[paged_cache_update] negative dimension");
  }
  if (page_size <= 0 || page_size % 16 != 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[paged_cache_update] page size %d is not a multiple of 16",
        page_size);
  }
  const int64_t size = static_cast<int64_t>(dtype_size(dtype));
  if (D * size % 16 != 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[paged_cache_update] rows of %d elements are not a multiple of 16 bytes",
        D);
  }
  UpdateArgs a{};
  a.units = static_cast<int>(D * size / 16);
  a.n = static_cast<int64_t>(B) * L * Hkv * a.units;
  if (a.n == 0 || pages == 0 || table_width == 0) {
    return MLXROCM_OK;
  }
  if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr ||
      table == nullptr || lengths == nullptr || strides == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[paged_cache_update] null pointer");
  }
  uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
      reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages);
  for (int i = 0; i < 12; ++i) {
    bits |= static_cast<uintptr_t>(strides[i] * size);
  }
  if (bits % 16 != 0) {
    return fail(MLXROCM_UNSUPPORTED, "[paged_cache_update] operands are not aligned to 16 bytes");
  }
  if (static_cast<int64_t>(table_width) * page_size > INT32_MAX || a.n > int64_t{1} << 38) {
    return fail(MLXROCM_UNSUPPORTED, "[paged_cache_update] the problem exceeds the grid");
  }
  a.from[0] = static_cast<const char*>(k);
  a.from[1] = static_cast<const char*>(v);
  a.to[0] = static_cast<char*>(k_pages);
  a.to[1] = static_cast<char*>(v_pages);
  a.table = table;
  a.lengths = lengths;
  a.H = Hkv;
  a.L = L;
  a.pages = pages;
  a.page = page_size;
  a.table_width = table_width;
  a.table_stride = strides[12];
  for (int w = 0; w < 2; ++w) {
    for (int i = 0; i < 3; ++i) {
      a.from_strides[w][i] = strides[3 * w + i] * size;
      a.to_strides[w][i] = strides[6 + 3 * w + i] * size;
    }
  }
  const dim3 grid(static_cast<unsigned>((a.n + 255) / 256), 2);
  paged_update_kernel<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  MLXROCM_HIP_TRY(hipGetLastError());
  return MLXROCM_OK;
}

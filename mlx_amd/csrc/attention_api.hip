// attention_api.hip -- the entry points of attention: checks, the choice of kernel and of the
// number of runs that the keys are cut into.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace mlxrocm {

namespace {

constexpr int kMostKeys = 1 << 30; // positions and their differences stay in 32 bits
constexpr int kMostSplits = 64;

int64_t heads_of(const AttentionArgs& a) {
  return static_cast<int64_t>(a.B) * a.Hkv;
}

// Rows of a workgroup of the kernel for few rows
int64_t few_block(const AttentionArgs& a, int dtype) {
  const int wide = dtype == MLXROCM_FLOAT32 ? 128 : 64; // columns of which 32 rows are few
  return static_cast<int64_t>(a.G) * a.Lq > 16 && a.D <= wide ? 32 : 16;
}

// Workgroups of the kernel for few rows, and the keys that one of them is over
struct FewWork {
  int64_t rows, each, blocks, keys;
  FewWork(const AttentionArgs& a, int dtype)
      : rows(static_cast<int64_t>(a.G) * a.Lq),
        each(few_block(a, dtype)),
        blocks((rows + each - 1) / each * heads_of(a)),
        keys(std::min<int64_t>(
            a.keys - std::min(a.Lq, a.keys) / 2,
            static_cast<int64_t>(a.window) + a.keep + (each + a.G - 1) / a.G)) {}
};

// Whether the kernel for few rows takes a call, else the one of 128-row tiles, which reads keys and
// values less often but has its waves wait for each other.  us, few / tiles, each with its best
// number of runs.  One workgroup for all rows, 4096 keys: 8 sequences of 32 rows of 64 columns
// 22.0 / 24.5; 4 of 16 rows of 256 17.6 / 20.1.  More, bfloat16 (workgroups x keys): 16 heads of 128,
// 512 tokens (512 x 256) 15.5 / 21.5; 8 key heads of 128 for 32, 128 tokens (256 x 64) 6.9 / 10.0;
// 64 rows each over 4096 keys (32 x 4096) 15.7 / 16.9; 36 rows for 32 key heads over 8192
// (96 x 8192) 51 / 32; 16 heads of 64, 2048 tokens (1024 x 1024) 54 / 37; 16 heads of 64, 8 times
// 512 tokens under a window of 64 (2048 x 96) 26 / 14.  Of 96 columns, whose lines the tiles pad to
// 128, more: 12 heads on 4, twice 400 tokens (608 x 200) 11.8 / 18.6, 16 heads, twice 330 (672 x 165)
// 12.9 / 18.1; but 16 heads of 64, 4 times 330 (704 x 165) 15.9 / 12.8, of 128, 4 times 160 (640 x 80)
// 14.5 / 10.7.  Of 96 above 768: 800 x 200 14.0 / 18.7, 832 x 100 12.6 / 11.8, 912 x 150 16.4 / 11.9,
// 1088 x 90 15.5 / 10.1, 1200 x 200 18.6 / 14.4.
// float32, 80 columns: 64 x 64 13.2 / 17.9, 32 x 1580 23.1 / 25.9, 26 x 2150 23.6 / 25.7, 512 x 96
// 25.2 / 28.2, 512 x 128 29.5 / 30.7, 256 x 256 31.4 / 32.0, 304 x 132 30.3 / 27.3; above 2^16 512 x 160
// 37.3 / 32.9, 256 x 500 53.7 / 46.5, 768 x 160 54.9 / 42.5, 1024 x 64 48 / 31.  256 columns, of which the
// tiles hold a workgroup of 128 rows to a CU: 64 x 64 16.4 / 43.2, 304 x 80 29.2 / 62.0.
bool few(const AttentionArgs& a, int dtype) {
  const FewWork w(a, dtype);
  const int64_t most = a.D == 96 && dtype != MLXROCM_FLOAT32 ? 768 : 512;
  const int64_t work = dtype == MLXROCM_FLOAT32 && a.D <= 128 ? 1 << 16 : 1 << 17;
  return w.rows <= w.each || (w.blocks <= most && w.blocks * w.keys <= work);
}

// Runs that the keys of a row are cut into.  Few rows, by runs, us (16-bit, 8 or 64 key heads of
// 128, 256 workgroups marked): one sequence of 515 tokens 4 9.3, 8 8.4, 16 8.7; of 2048 8 10.1,
// 16 9.1, 32* 9.7; of 8192 16 15.1, 32* 12.9, 64 14.4; 8 of 1024 2 14.2, 4* 11.5, 8 11.8; 8 of 20011
// under a window of 4096 4* 23.4, 8 21.8, 16 26.7; 32 of 8192 1* 190, 2 187, 4 188.  Tiles: 64 rows over
// 4096 8 22.6, 16 17.4, 32* 17.5, 64 22.9; 8 times 64 rows over 500 2 17.3, 4* 16.7, 8 22.2; 512 rows
// over 32768 2* 480, 4 306, 8 317.
int splits_of(const AttentionArgs& a, int dtype) {
  const int64_t span =
      std::min<int64_t>(a.keys, static_cast<int64_t>(a.window) + a.keep + a.Lq);
  const int64_t heads = heads_of(a);
  int64_t splits;
  if (few(a, dtype)) {
    const FewWork w(a, dtype);
    // a workgroup for each CU; not one more of float32, of which a CU holds one (26 workgroups of 80 columns
    // over 2150 keys 9 runs 23.6, 10 37.2; one token, 3 sequences of 4600, 8 key heads of 128 32 / 42)
    const int64_t once = dtype == MLXROCM_FLOAT32 ? std::max<int64_t>(256 / w.blocks, 1)
                                                  : (256 + w.blocks - 1) / w.blocks;
    const int64_t reach = w.rows <= w.each ? span : w.keys;
    splits = std::min<int64_t>(
        std::max<int64_t>(once, std::min<int64_t>(2 * once, reach / 512)), reach / 72);
  } else {
    const int64_t blocks = (static_cast<int64_t>(a.G) * a.Lq + 127) / 128 * heads;
    // float32's matrix instruction takes 16 times as long: fewer keys are a run's worth, and it is
    // busy with the one workgroup that a CU holds of more than 64 columns.  (3 times 16 heads of 80,
    // 509 tokens, window 128: 1 52, 2 63; 16 heads of 256, 512 tokens: 1 230, 4* 90, 8 95.)
    splits = dtype == MLXROCM_FLOAT32
        ? std::min<int64_t>((a.D <= 64 ? 512 : 256) / blocks, span / 64)
        : std::min<int64_t>(
              512 / blocks,
              std::max<int64_t>(span / 256, std::min<int64_t>(span / 128, 256 / blocks)));
  }
  return static_cast<int>(std::min<int64_t>(std::max<int64_t>(splits, 1), kMostSplits));
}

size_t round256(size_t n) {
  return (n + 255) / 256 * 256;
}

size_t workspace_of(const AttentionArgs& a, int dtype) {
  const int splits = splits_of(a, dtype);
  if (splits == 1) {
    return 0;
  }
  const size_t rows = static_cast<size_t>(splits) * a.B * a.Hq * a.Lq;
  return round256(rows * a.D * sizeof(float)) + rows * sizeof(float2);
}

// The cuts of the gradients' sums: parts of some tiles each, and a thousand workgroups if there
// are as many, half as many where a CU holds one (8 heads of 256 on 2, 4096 tokens 614 instead of
// 743 us).  us of the gradients' kernels, bfloat16, parts of at least 256, 512, 768 and 1024 keys or
// rows: 64 heads of 128 on 8, 500 tokens 73, 83, 100, 113; 28 on 4, 2 times 1000 tokens 188, 140, 141,
// 149; 32 on 8, 4096 tokens under a window of 256 with 4 kept 266, 247, 255, 256, with none 217, 221,
// 197, 198.
// Up to a workgroup for each CU parts of 64 are enough: 16 heads of 128 on 4, 300 tokens 48 (128: 50,
// 256: 53, 512: 73), 8 of 256 on one, 500 75 (75, 93, 116), 12 of 96 on 4, 1500 under a window of 128 56 (56,
// 49, 58), float32, 32 of 128 on 8, 150 79 (103).
GradPlan grad_plan_of(const AttentionArgs& a, int dtype) {
  GradPlan p{};
  const int64_t rows = static_cast<int64_t>(a.G) * a.Lq;
  const int64_t row_blocks = (rows + kGradBlock - 1) / kGradBlock;
  p.blocks = (a.keys + kGradBlock - 1) / kGradBlock;
  // float32's matrix instruction takes 16 times as long: less is enough for a part
  const int64_t least = dtype == MLXROCM_FLOAT32 ? 128 : 512;
  const int64_t fill = a.D * dtype_size(dtype) <= 256 ? 1024 : 512;
  const int64_t reach = static_cast<int64_t>(a.window) + kGradBlock; // tokens
  const int64_t span = std::min<int64_t>(a.keys, reach + a.keep);
  const auto parts = [&](int64_t blocks, int64_t of_least, int64_t of_64) {
    const int64_t whole = std::max<int64_t>(blocks * heads_of(a), 1);
    const int64_t wanted = std::max<int64_t>(
        std::min<int64_t>((fill + whole - 1) / whole, of_least),
        std::min<int64_t>((256 + whole - 1) / whole, of_64));
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(wanted, kMostSplits)));
  };
  p.dq_splits = Divisor(row_blocks > 0 ? parts(row_blocks, span / least, span / 64) : 1);
  const int64_t seen_by = std::min<int64_t>(a.Lq, reach) * a.G;
  if (a.window < a.keys && seen_by < rows) {
    p.wide_blocks = static_cast<int>(std::min<int64_t>(
        p.blocks, (static_cast<int64_t>(a.keep) + kGradBlock - 1) / kGradBlock));
  }
  const int splits =
      p.blocks > 0 ? parts(p.blocks, (seen_by + least / 2) / least, (seen_by + 63) / 64) : 1;
  p.splits = Divisor(splits);
  // Runs no longer than the others', but no more workgroups than fill the card: each keeps 128 keys' sums
  // in float32.  us of both gradients, bfloat16, 8192 tokens, with as many as fill it / as would be no
  // longer: 32 heads on 8 under a window of 64, all kept 2080 / 3530 (4.3 GB), 8 times that with 4096 kept
  // 13350 / 16540 (11.3 GB); 8 heads of 256 on 2, 4096 tokens, 1000 kept 333 / 390.
  int64_t wide = splits;
  if (p.wide_blocks > 0) {
    const int64_t whole = p.wide_blocks * heads_of(a);
    wide = std::min<int64_t>(rows * splits / std::max<int64_t>(seen_by, 1), (fill + whole - 1) / whole);
    wide = std::max<int64_t>(1, std::min<int64_t>({wide, (rows + 63) / 64, kMostSplits}));
  }
  p.wide_splits = Divisor(wide);
  return p;
}

// delta, in float16 the largest gradients of probabilities, then the partial sums of dq, then those of
// dk and dv
struct GradWorkspace {
  size_t largest, part_dq, part_dkv, total;
  GradWorkspace(const AttentionArgs& a, const GradPlan& p, int dtype) {
    const size_t rows = static_cast<size_t>(a.B) * a.Hq * a.Lq;
    const size_t blocks = (static_cast<size_t>(a.G) * a.Lq + kGradBlock - 1) / kGradBlock;
    largest = round256(rows * sizeof(float));
    part_dq = largest +
        (dtype == MLXROCM_FLOAT16
             ? round256(heads_of(a) * p.dq_splits.d * blocks * (kGradBlock / 32) * sizeof(float))
             : 0);
    part_dkv = part_dq +
        (p.dq_splits.d > 1 ? round256(rows * a.D * p.dq_splits.d * sizeof(float)) : 0);
    total = part_dkv +
        (p.dkv_split() ? static_cast<size_t>(heads_of(a)) * p.part_pieces() * kGradBlock * 2 * a.D *
                 sizeof(float)
                       : 0);
  }
};

// Shapes alone; `name` for messages
int check_shape(const char* name, const AttentionArgs& a, int dtype) {
  if (!valid_dtype(dtype)) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] unknown dtype %d", name, dtype);
  }
  if (a.B < 0 || a.Hq < 0 || a.Hkv < 0 || a.Lq < 0 || a.keys < 0 || a.D <= 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] negative dimension", name);
  }
  if (a.D % 8 != 0 || a.D > 256) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] head dimension %d is not a multiple of 8 up to 256", name,
        a.D);
  }
  if (a.Hkv == 0 ? a.Hq != 0 : a.Hq % a.Hkv != 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] %d query heads cannot share %d key heads", name, a.Hq,
        a.Hkv);
  }
  if (a.window < 1 || a.keep < 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] window %d must be positive and keep %d not negative", name,
        a.window, a.keep);
  }
  // what indexes the launch and the rows in 32 bits
  const int64_t rows = static_cast<int64_t>(a.G) * a.Lq;
  if (a.keys > kMostKeys || rows > kMostKeys ||
      ((rows + 15) / 16 * kMostSplits + a.keys / 128 + 1) * a.B * a.Hkv > INT32_MAX / 8) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", name);
  }
  return MLXROCM_OK;
}

int check_operand(
    const char* name, const char* what, const void* p, const int64_t (&strides)[3], int dtype) {
  if (p == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer: %s", name, what);
  }
  const int64_t unit = 16 / static_cast<int64_t>(dtype_size(dtype));
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || strides[0] % unit != 0 ||
      strides[1] % unit != 0 || strides[2] % unit != 0) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] %s is not aligned to 16 bytes", name, what);
  }
  return MLXROCM_OK;
}

#define TRY(expr)          \
  do {                     \
    const int rc_ = expr;  \
    if (rc_ != MLXROCM_OK) \
      return rc_;          \
  } while (0)

void take(int64_t (&to)[3], const int64_t* from) {
  to[0] = from[0];
  to[1] = from[1];
  to[2] = from[2];
}

// Whether the rows that one load covers (eight at most) lie within 31 bits of bytes of the first
bool near(const int64_t (&strides)[3], int dtype, int G) {
  const int64_t most = INT32_MAX / static_cast<int64_t>(dtype_size(dtype));
  const auto within = [&](int64_t n) { return n > -most / 16 && n < most / 16; };
  return within(strides[2]) && (G == 1 || within(strides[1])) && strides[1] >= 0 &&
      strides[2] >= 0;
}

void set_near(AttentionArgs& a, int dtype) {
  a.near = near(a.k_strides, dtype, 1) && near(a.v_strides, dtype, 1) ? 1 : 0;
}

void set_scale(AttentionArgs& a, float scale, int dtype) {
  // (no score is worth less than 1e-30 log2 units: a scale of zero would make NaN of the -inf of
  // masked scores)
  a.scale_log2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);
  a.q_sign = std::signbit(scale) ? (dtype == MLXROCM_FLOAT32 ? 0x80000000u : 0x80008000u) : 0u;
}

AttentionArgs shape_of(
    int B, int Hq, int Hkv, int Lq, int keys, int D, int window, int keep) {
  AttentionArgs a{};
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hkv > 0 ? Hq / Hkv : 0;
  a.Lq = Lq;
  a.keys = keys;
  a.D = D;
  a.of_G = Divisor(a.G);
  a.of_Hkv = Divisor(Hkv);
  a.window = std::min(window, kMostKeys);
  a.keep = std::min(keep, kMostKeys);
  return a;
}

// Whether the gradients get what rounding took from a 16-bit result: its share in delta is that of a
// mean over the keys that a token sees, and matters where those are few.  Errors of dq in their own
// rounding's, with / without it (1.42 with delta exact): 23 tokens 1.43 / 1.58, 235 1.42 / 1.51, 1500
// without it 1.46.  8192 tokens, 32 heads of 128, forward and gradients 2.62 / 2.60 ms.
bool keeps_low(const AttentionArgs& a, int dtype) {
  return dtype != MLXROCM_FLOAT32 &&
      std::min<int64_t>(a.keys, static_cast<int64_t>(a.window) + a.keep) <= 2048;
}

size_t lse_bytes(const AttentionArgs& a) {
  return round256(static_cast<size_t>(a.B) * a.Hq * a.Lq * sizeof(float));
}

int take_lse(const char* name, AttentionArgs& a, float* lse, int dtype) {
  if (reinterpret_cast<uintptr_t>(lse) % 16 != 0) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] lse is not aligned to 16 bytes", name);
  }
  a.lse = lse;
  if (lse != nullptr && keeps_low(a, dtype)) {
    a.low = reinterpret_cast<char*>(lse) + lse_bytes(a);
  }
  return MLXROCM_OK;
}

bool empty(const AttentionArgs& a) {
  return a.B == 0 || a.Hq == 0 || a.Lq == 0;
}

// (keys and values that no query reads have gradients of zero)
bool no_gradients(const AttentionArgs& a) {
  return empty(a) && (a.B == 0 || a.Hkv == 0 || a.keys == 0);
}

int run(const char* name, AttentionArgs& a, int dtype, void* workspace, size_t bytes,
        hipStream_t s) {
  a.splits = splits_of(a, dtype);
  a.of_splits = Divisor(a.splits);
  set_near(a, dtype);
  if (a.splits > 1 && !rehearsing()) {
    const size_t need = workspace_of(a, dtype);
    if (workspace == nullptr || bytes < need) {
      return fail(
          MLXROCM_INVALID_ARGUMENT, "[%s] workspace of %zu bytes, %zu needed", name, bytes, need);
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
      return fail(MLXROCM_INVALID_ARGUMENT, "[%s] workspace is not aligned to 16 bytes", name);
    }
    const size_t rows = static_cast<size_t>(a.splits) * a.B * a.Hq * a.Lq;
    a.part_out = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(
        static_cast<char*>(workspace) + round256(rows * a.D * sizeof(float)));
  }
  if (few(a, dtype)) {
    TRY(dtype == MLXROCM_FLOAT32       ? launch_attention_few_f32(a, s)
            : dtype == MLXROCM_FLOAT16 ? launch_attention_few_f16(a, s)
                                       : launch_attention_few_bf16(a, s));
  } else {
    TRY(dtype == MLXROCM_FLOAT32       ? launch_attention_rows_f32(a, s)
            : dtype == MLXROCM_FLOAT16 ? launch_attention_rows_f16(a, s)
                                       : launch_attention_rows_bf16(a, s));
  }
  return a.splits > 1 ? launch_attention_join(a, dtype, s) : static_cast<int>(MLXROCM_OK);
}

int run_grad(const AttentionGradArgs& g, int dtype, hipStream_t s) {
  TRY(dtype == MLXROCM_FLOAT32       ? launch_attention_grad_f32(g, s)
          : dtype == MLXROCM_FLOAT16 ? launch_attention_grad_f16(g, s)
                                     : launch_attention_grad_bf16(g, s));
  return g.plan.dq_splits.d > 1 || g.plan.dkv_split() ? launch_attention_grad_join(g, dtype, s)
                                                    : static_cast<int>(MLXROCM_OK);
}

} // namespace

} // namespace mlxrocm

extern "C" size_t mlxrocm_window_attention_workspace_size(
    int B, int Hq, int Hkv, int Lq, int Lk, int D, int window, int keep, int dtype) {
  using namespace mlxrocm;
  const AttentionArgs a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  return check_shape("window_attention", a, dtype) != MLXROCM_OK || empty(a) ? 0
                                                                             : workspace_of(a, dtype);
}

extern "C" size_t mlxrocm_window_attention_lse_size(
    int B, int Hq, int Hkv, int Lq, int Lk, int D, int window, int keep, int dtype) {
  using namespace mlxrocm;
  const AttentionArgs a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  if (check_shape("window_attention", a, dtype) != MLXROCM_OK || empty(a)) {
    return 0;
  }
  return lse_bytes(a) + (keeps_low(a, dtype) ? static_cast<size_t>(B) * Hq * Lq * D * 2 : 0);
}

extern "C" int mlxrocm_window_attention(
    const void* q,
    const void* k,
    const void* v,
    void* out,
    float* lse,
    const int32_t* lengths,
    int B,
    int Hq,
    int Hkv,
    int Lq,
    int Lk,
    int D,
    const int64_t* strides,
    float scale,
    int window,
    int keep,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_window_attention");
  using namespace mlxrocm;
  const char* name = "window_attention";
  AttentionArgs a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  TRY(check_shape(name, a, dtype));
  if (empty(a)) {
    return MLXROCM_OK;
  }
  if (!std::isfinite(scale) || strides == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] scale is not finite or strides are null", name);
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  TRY(take_lse(name, a, lse, dtype));
  a.lengths = lengths;
  take(a.q_strides, strides);
  take(a.k_strides, strides + 3);
  take(a.v_strides, strides + 6);
  take(a.out_strides, strides + 9);
  TRY(check_operand(name, "q", q, a.q_strides, dtype));
  TRY(check_operand(name, "out", out, a.out_strides, dtype));
  if (Lk > 0) {
    TRY(check_operand(name, "k", k, a.k_strides, dtype));
    TRY(check_operand(name, "v", v, a.v_strides, dtype));
  }
  set_scale(a, scale, dtype);
  return run(name, a, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" size_t mlxrocm_window_attention_vjp_workspace_size(
    int B, int Hq, int Hkv, int Lq, int Lk, int D, int window, int keep, int dtype) {
  using namespace mlxrocm;
  const AttentionArgs a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  return check_shape("window_attention_vjp", a, dtype) != MLXROCM_OK
      ? 0
      : GradWorkspace(a, grad_plan_of(a, dtype), dtype).total;
}

extern "C" int mlxrocm_window_attention_vjp(
    const void* q,
    const void* k,
    const void* v,
    const void* out,
    const float* lse,
    const void* dout,
    void* dq,
    void* dk,
    void* dv,
    const int32_t* lengths,
    int B,
    int Hq,
    int Hkv,
    int Lq,
    int Lk,
    int D,
    const int64_t* strides,
    float scale,
    int window,
    int keep,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_window_attention_vjp");
  using namespace mlxrocm;
  const char* name = "window_attention_vjp";
  AttentionGradArgs g{};
  AttentionArgs& a = g.a;
  a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  TRY(check_shape(name, a, dtype));
  if (no_gradients(a)) {
    return MLXROCM_OK;
  }
  if (!std::isfinite(scale) || strides == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] scale is not finite or strides are null", name);
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = const_cast<void*>(out);
  TRY(take_lse(name, a, const_cast<float*>(lse), dtype));
  a.lengths = lengths;
  a.splits = 1;
  g.dout = dout;
  g.dq = dq;
  g.dk = dk;
  g.dv = dv;
  g.scale = scale;
  take(a.q_strides, strides);
  take(a.k_strides, strides + 3);
  take(a.v_strides, strides + 6);
  take(a.out_strides, strides + 9);
  take(g.dout_strides, strides + 12);
  take(g.dq_strides, strides + 15);
  take(g.dk_strides, strides + 18);
  take(g.dv_strides, strides + 21);
  if (!empty(a)) {
    TRY(check_operand(name, "q", q, a.q_strides, dtype));
    TRY(check_operand(name, "out", out, a.out_strides, dtype));
    TRY(check_operand(name, "dout", dout, g.dout_strides, dtype));
    TRY(check_operand(name, "dq", dq, g.dq_strides, dtype));
    if (lse == nullptr) {
      return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer: lse", name);
    }
  }
  g.plan = grad_plan_of(a, dtype);
  const GradWorkspace parts(a, g.plan, dtype);
  if (parts.total > 0) {
    if (workspace == nullptr || workspace_bytes < parts.total) {
      return fail(
          MLXROCM_INVALID_ARGUMENT, "[%s] workspace of %zu bytes, %zu needed", name,
          workspace_bytes, parts.total);
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
      return fail(MLXROCM_INVALID_ARGUMENT, "[%s] workspace is not aligned to 16 bytes", name);
    }
    char* at = static_cast<char*>(workspace);
    g.delta = static_cast<float*>(workspace);
    g.largest = reinterpret_cast<float*>(at + parts.largest);
    g.part_dq = reinterpret_cast<float*>(at + parts.part_dq);
    g.part_dkv = reinterpret_cast<float*>(at + parts.part_dkv);
  }
  if (Lk > 0) {
    TRY(check_operand(name, "k", k, a.k_strides, dtype));
    TRY(check_operand(name, "v", v, a.v_strides, dtype));
    TRY(check_operand(name, "dk", dk, g.dk_strides, dtype));
    TRY(check_operand(name, "dv", dv, g.dv_strides, dtype));
  }
  set_scale(a, scale, dtype);
  set_near(a, dtype);
  if (a.G > 0 && (a.G & (a.G - 1)) == 0 && a.G <= 32 && near(a.q_strides, dtype, a.G) &&
      near(g.dout_strides, dtype, a.G)) {
    a.near |= 2;
    a.g_log2 = __builtin_ctz(a.G);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  TRY(run_grad(g, dtype, s));
  return MLXROCM_OK;
}

extern "C" size_t mlxrocm_paged_attention_workspace_size(
    int B, int Hq, int Hkv, int Lq, int D, int max_keys, int window, int keep, int dtype) {
  using namespace mlxrocm;
  const AttentionArgs a = shape_of(B, Hq, Hkv, Lq, max_keys, D, window, keep);
  return check_shape("paged_attention", a, dtype) != MLXROCM_OK || empty(a) ? 0 : workspace_of(a, dtype);
}

extern "C" int mlxrocm_paged_attention(
    const void* q,
    const void* k_pages,
    const void* v_pages,
    const int32_t* table,
    const int32_t* lengths,
    void* out,
    int B,
    int Hq,
    int Hkv,
    int Lq,
    int D,
    int pages,
    int page_size,
    int table_width,
    const int64_t* strides,
    float scale,
    int window,
    int keep,
    int dtype,
    void* workspace,
    size_t workspace_bytes,
    mlxrocm_stream_t stream) {
  mlxrocm::ApiRange api_range("mlxrocm_paged_attention");
  using namespace mlxrocm;
  const char* name = "paged_attention";
  if (page_size <= 0 || page_size % 16 != 0) {
    return fail(
        MLXROCM_INVALID_ARGUMENT, "[%s] page size %d is not a multiple of 16", name, page_size);
  }
  if (pages < 0 || table_width < 0) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] negative dimension", name);
  }
  const int64_t keys = static_cast<int64_t>(table_width) * page_size;
  if (keys > kMostKeys) {
    return fail(MLXROCM_UNSUPPORTED, "[%s] the problem exceeds the grid", name);
  }
  AttentionArgs a =
      shape_of(B, Hq, Hkv, Lq, pages == 0 ? 0 : static_cast<int>(keys), D, window, keep);
  TRY(check_shape(name, a, dtype));
  if (empty(a)) {
    return MLXROCM_OK;
  }
  if (!std::isfinite(scale) || strides == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] scale is not finite or strides are null", name);
  }
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.out = out;
  a.lengths = lengths;
  a.table = table;
  a.page = Divisor(page_size);
  a.pages = pages;
  take(a.q_strides, strides);
  take(a.k_strides, strides + 3);
  take(a.v_strides, strides + 6);
  take(a.out_strides, strides + 9);
  a.table_stride = strides[12];
  TRY(check_operand(name, "q", q, a.q_strides, dtype));
  TRY(check_operand(name, "out", out, a.out_strides, dtype));
  if (lengths == nullptr) {
    return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer: lengths", name);
  }
  if (a.keys > 0) {
    TRY(check_operand(name, "k_pages", k_pages, a.k_strides, dtype));
    TRY(check_operand(name, "v_pages", v_pages, a.v_strides, dtype));
    if (table == nullptr) {
      return fail(MLXROCM_INVALID_ARGUMENT, "[%s] null pointer: table", name);
    }
  }
  set_scale(a, scale, dtype);
  return run(name, a, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int mlxrocm_attention_plan(
    int B,
    int Hq,
    int Hkv,
    int Lq,
    int keys,
    int D,
    int window,
    int keep,
    int dtype,
    char* plan,
    size_t plan_bytes) {
  using namespace mlxrocm;
  RehearsalScope rehearsal(plan, plan_bytes);
  AttentionArgs a = shape_of(B, Hq, Hkv, Lq, keys, D, window, keep);
  TRY(check_shape("attention_plan", a, dtype));
  return empty(a) ? static_cast<int>(MLXROCM_OK)
                  : run("attention_plan", a, dtype, nullptr, 0, nullptr);
}

extern "C" int mlxrocm_window_attention_vjp_plan(
    int B,
    int Hq,
    int Hkv,
    int Lq,
    int Lk,
    int D,
    int window,
    int keep,
    int dtype,
    char* plan,
    size_t plan_bytes) {
  using namespace mlxrocm;
  RehearsalScope rehearsal(plan, plan_bytes);
  AttentionGradArgs g{};
  g.a = shape_of(B, Hq, Hkv, Lq, Lk, D, window, keep);
  TRY(check_shape("window_attention_vjp_plan", g.a, dtype));
  g.plan = grad_plan_of(g.a, dtype);
  return no_gradients(g.a) ? static_cast<int>(MLXROCM_OK) : run_grad(g, dtype, nullptr);
}

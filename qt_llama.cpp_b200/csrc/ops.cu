// ops.cu — C ABI entry points of the permutation and MXFP4 operators
// (declared in include/mrml_moe.h): argument checks, workspace layouts and
// the order of kernel launches on the caller's stream.
#include <algorithm>

#include "../../include/mrml_moe.h"
#include "checks.h"
#include "kernels.h"
#include "mx4.cuh"

namespace {

using mrml::align256;
using mrml::aligned16;
using mrml::kMaxExperts;
using mrml::kMaxTopK;

bool is_float(int type) { return type == MRML_F32 || type == MRML_F16 || type == MRML_BF16; }
bool is_gguf(int type) { return type == MRML_Q4_0 || type == MRML_Q8_0; }
bool elem_aligned(const void* p, int type) { return ((uintptr_t)p & (mrml::elem_bytes(type) - 1)) == 0; }

// The most (token, slot) pairs of a call: every chunk of a large sort sums the
// counts of all chunks, which beyond this would take longer than the rest.
constexpr long long kMaxPairs = 1ll << 26;
// The widest row, and the most sorted rows: the kernels' column and row indices are ints.
constexpr int kMaxCols = 1 << 24, kMaxRows = 0x7fffff00;

// Rows of the sorted order, padding included; -1 when the arguments are
// invalid.
long long rows_bound(int E, int K, int T, int align) {
  if (E <= 0 || K <= 0 || T < 0 || align <= 0 || align > 128) return -1;
  const long long pairs = (long long)T * K;
  if (pairs > kMaxPairs) return -1;
  const long long rows = pairs + std::min<long long>(E, pairs) * (align - 1);
  return rows > kMaxRows ? -1 : rows;
}

// Shapes of the permutation entry points.
int check_tokens(int type, int H, int K, int T) {
  if (!is_float(type)) return MRML_ERR_UNSUPPORTED;
  if (H <= 0 || K <= 0 || T < 0) return MRML_ERR_INVALID_ARGUMENT;
  if (H > kMaxCols || K > kMaxTopK || (long long)T * K > kMaxPairs) return MRML_ERR_UNSUPPORTED;
  // the gather takes a warp per 1024 values of a token
  if ((long long)T * ((H + 1023) / 1024) > 0x7fffffffll) return MRML_ERR_UNSUPPORTED;
  return MRML_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (!ws || ((uintptr_t)ws & 255u) != 0) return MRML_ERR_INVALID_ARGUMENT;
  return have < need ? MRML_ERR_WORKSPACE_TOO_SMALL : MRML_OK;
}

// MXFP4 matrix shapes; one CTA takes 8 rows x 1024 columns (quantiser), 16 x
// 128 (dequantiser), 64 x 128 (both directions).
int check_matrix(int rows, int cols, int matrices) {
  if (rows < 0 || cols <= 0 || matrices < 0) return MRML_ERR_INVALID_ARGUMENT;
  if (matrices > 65535 || rows > kMaxRows || cols > kMaxRows) return MRML_ERR_UNSUPPORTED;
  if (((long long)rows + 127) / 16 * (((long long)cols + 127) / 128) > 0x7fffffffll) return MRML_ERR_UNSUPPORTED;
  return MRML_OK;
}

struct SortWs {
  int* status;
  int32_t* chunk_cnt;
  size_t bytes;
};
SortWs carve_sort(void* base, int E, int K, int T) {
  uint8_t* p = static_cast<uint8_t*>(base);
  SortWs w;
  w.status = static_cast<int*>(base);
  w.chunk_cnt = reinterpret_cast<int32_t*>(p ? p + 256 : nullptr);
  w.bytes = 256 + align256(mrml::sort_chunk_ints((long long)T * K, E) * 4);
  return w;
}

struct ExpertsWs {
  SortWs sort;
  int32_t *offsets, *counts, *pos, *pair;
  uint8_t *x, *act;  // MXFP4 rows in expert order: tokens [H], activations [I]
  uint8_t* flat;     // the tokens quantised row by row (large batches)
  float* y;          // down products [row][H]
  int n_rows;
  size_t bytes;
};
ExpertsWs carve_experts(void* base, int H, int I, int E, int K, int T) {
  ExpertsWs w;
  uint8_t* p = static_cast<uint8_t*>(base);
  w.sort = carve_sort(base, E, K, T);
  size_t off = w.sort.bytes;
  auto take = [&](size_t n) {
    uint8_t* r = p ? p + off : nullptr;
    off += align256(n);
    return r;
  };
  w.n_rows = (int)rows_bound(E, K, T, mrml::kMxRows);
  w.offsets = reinterpret_cast<int32_t*>(take((size_t)(E + 1) * 4));
  w.counts = reinterpret_cast<int32_t*>(take((size_t)E * 4));
  w.pos = reinterpret_cast<int32_t*>(take((size_t)T * K * 4));
  w.pair = reinterpret_cast<int32_t*>(take((size_t)w.n_rows * 4));
  w.x = take(mrml::mx_matrix_bytes(w.n_rows, H));
  w.act = take(mrml::mx_matrix_bytes(w.n_rows, I));
  w.flat = take(mrml::mx4_flat_bytes(H, K, T));
  w.y = reinterpret_cast<float*>(take((size_t)w.n_rows * H * 4));
  w.bytes = off;
  return w;
}

// Shapes of a product: the grid's units have to fit an int.
int check_product(int type, int M, int N, int K) {
  if (!is_float(type)) return MRML_ERR_UNSUPPORTED;
  if (M < 0 || N <= 0 || K <= 0) return MRML_ERR_INVALID_ARGUMENT;
  if (M > kMaxRows || N > kMaxRows || K > kMaxCols) return MRML_ERR_UNSUPPORTED;  // offsets in a tile fit an int
  if (((long long)M + 127) / 128 * (((long long)N + 127) / 128) > (1ll << 30)) return MRML_ERR_UNSUPPORTED;
  return MRML_OK;
}

// Shapes of the expert layer.
int check_experts(int type, int H, int I, int E, int K, int T) {
  MRML_TRY(check_tokens(type, H, K, T));
  if (I <= 0 || E <= 0) return MRML_ERR_INVALID_ARGUMENT;
  if (E > kMaxExperts || I > kMaxCols) return MRML_ERR_UNSUPPORTED;
  const long long n_rows = rows_bound(E, K, T, mrml::kMxRows);
  if (n_rows < 0) return MRML_ERR_UNSUPPORTED;
  return check_product(type, (int)n_rows, std::max(2 * I, H), std::max(H, I));
}

// `early`: a was written by the launch right before, b not (launch_mx4_gemm).
int matmul(int type, const uint8_t* a, const uint8_t* b, void* out, int64_t ldo, int M, int N, int K, void* workspace,
           size_t workspace_bytes, bool early, mrml_stream_t stream) {
  MRML_TRY(check_product(type, M, N, K));
  if (ldo < N) return MRML_ERR_INVALID_ARGUMENT;
  if (M == 0) return MRML_OK;
  if (!a || !b || !out || !aligned16(a) || !aligned16(b) || !elem_aligned(out, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(check_workspace(workspace, workspace_bytes, mrml_moe_mx4_matmul_workspace_bytes(M, N, K)));
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_mx4_gemm(type, b, a, nullptr, nullptr, 1, M, N, K, false, out, ldo, nullptr, M, early,
                                    static_cast<int*>(workspace), s));
  return MRML_OK;
}

}  // namespace

extern "C" {

int mrml_moe_sorted_rows(int E, int K, int T, int align) {
  const long long n = rows_bound(E, K, T, align);
  return n < 0 ? MRML_ERR_INVALID_ARGUMENT : (int)n;
}

size_t mrml_moe_sort_workspace_bytes(int E, int K, int T) {
  if (rows_bound(E, K, T, 1) < 0 || E > kMaxExperts) return 0;
  return carve_sort(nullptr, E, K, T).bytes;
}

int mrml_moe_sort(const int32_t* ids, int32_t* offsets, int32_t* counts, int32_t* pos, int32_t* pair, int E, int K,
                  int T, int align, void* workspace, size_t workspace_bytes, mrml_stream_t stream) {
  if (E <= 0 || K <= 0 || T < 0 || align <= 0) return MRML_ERR_INVALID_ARGUMENT;
  if (E > kMaxExperts || K > kMaxTopK || align > 128) return MRML_ERR_UNSUPPORTED;
  const long long n_rows = rows_bound(E, K, T, align);
  if (n_rows < 0) return MRML_ERR_UNSUPPORTED;
  if (!offsets || !counts || (T > 0 && (!ids || !pos || !pair))) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(check_workspace(workspace, workspace_bytes, carve_sort(nullptr, E, K, T).bytes));
  MRML_TRY(mrml::check_device());
  const SortWs w = carve_sort(workspace, E, K, T);
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_sort(ids, offsets, counts, pos, pair, E, T * K, align, (int)n_rows, w.chunk_cnt, w.status, s));
  return MRML_OK;
}

int mrml_moe_permute(int type, const void* x, int64_t ldx, const int32_t* pair, void* rows, int H, int K, int n_rows,
                     mrml_stream_t stream) {
  MRML_TRY(check_tokens(type, H, K, 0));
  if (n_rows < 0 || ldx < H) return MRML_ERR_INVALID_ARGUMENT;
  if (n_rows > kMaxRows) return MRML_ERR_UNSUPPORTED;
  if (n_rows == 0) return MRML_OK;
  if (!x || !pair || !rows || !elem_aligned(x, type) || !elem_aligned(rows, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_permute(type, x, ldx, pair, rows, H, K, n_rows, s));
  return MRML_OK;
}

int mrml_moe_permute_grad(int type, const void* drows, const int32_t* pos, void* dx, int64_t lddx, int H, int K, int T,
                          mrml_stream_t stream) {
  return mrml_moe_unpermute(type, drows, pos, nullptr, dx, lddx, H, K, T, stream);
}

int mrml_moe_unpermute(int type, const void* rows, const int32_t* pos, const float* probs, void* out, int64_t ldo,
                       int H, int K, int T, mrml_stream_t stream) {
  MRML_TRY(check_tokens(type, H, K, T));
  if (ldo < H) return MRML_ERR_INVALID_ARGUMENT;
  if (T == 0) return MRML_OK;
  if (!rows || !pos || !out || !elem_aligned(rows, type) || !elem_aligned(out, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_unpermute(type, rows, pos, probs, out, ldo, H, K, T, s));
  return MRML_OK;
}

int mrml_moe_unpermute_grad(int type, const void* dout, int64_t lddout, const void* rows, const int32_t* pos,
                            const int32_t* pair, const float* probs, void* drows, float* dprobs, int H, int K, int T,
                            int n_rows, mrml_stream_t stream) {
  MRML_TRY(check_tokens(type, H, K, T));
  if (lddout < H || n_rows < 0) return MRML_ERR_INVALID_ARGUMENT;
  if (n_rows > kMaxRows) return MRML_ERR_UNSUPPORTED;
  if (T == 0) {  // no pairs: every row is one without
    if (!drows || n_rows == 0) return MRML_OK;
    if (!elem_aligned(drows, type)) return MRML_ERR_INVALID_ARGUMENT;
    MRML_TRY(mrml::check_device());
    return mrml::cuda_status(
        cudaMemsetAsync(drows, 0, (size_t)n_rows * H * mrml::elem_bytes(type), (cudaStream_t)stream));
  }
  if (!drows && !dprobs) return MRML_OK;
  if (n_rows < T * K && drows) return MRML_ERR_INVALID_ARGUMENT;
  if (!dout || !pos || (drows && !pair) || (dprobs && !rows)) return MRML_ERR_INVALID_ARGUMENT;
  if (!elem_aligned(dout, type) || !elem_aligned(rows, type) || !elem_aligned(drows, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_unpermute_grad(type, dout, lddout, rows, pos, pair, probs, drows, dprobs, H, K, T, n_rows, s));
  return MRML_OK;
}

size_t mrml_moe_mx4_bytes(int rows, int cols, int matrices) {
  if (check_matrix(rows, cols, matrices) != MRML_OK) return 0;
  return mrml::mx_matrix_bytes(rows, cols) * (size_t)matrices;
}

int mrml_moe_mx4_quantize(int type, const void* x, int64_t ldx, int64_t matrix_stride, uint8_t* dst, int rows,
                          int cols, int matrices, int gated, mrml_stream_t stream) {
  if (!is_float(type) && !is_gguf(type)) return MRML_ERR_UNSUPPORTED;
  MRML_TRY(check_matrix(rows, cols, matrices));
  if (gated && rows % 2 != 0) return MRML_ERR_INVALID_ARGUMENT;
  if (is_gguf(type)) {  // contiguous block rows
    if (cols % 32 != 0 || ldx != cols || (matrices > 1 && matrix_stride != (int64_t)rows * cols))
      return MRML_ERR_INVALID_ARGUMENT;
  } else if (ldx < cols || (matrices > 1 && matrix_stride < 0)) {
    return MRML_ERR_INVALID_ARGUMENT;
  }
  if (rows == 0 || matrices == 0) return MRML_OK;
  if (!x || !dst || !aligned16(dst) || !elem_aligned(x, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_mx4_quantize(type, x, ldx, matrices > 1 ? matrix_stride : 0, dst, rows, cols, matrices,
                                        gated != 0, s));
  return MRML_OK;
}

int mrml_moe_mx4_quantize_both(int type, const void* x, int64_t ldx, uint8_t* dst, uint8_t* dst_t, int rows, int cols,
                               mrml_stream_t stream) {
  if (!is_float(type)) return MRML_ERR_UNSUPPORTED;
  MRML_TRY(check_matrix(rows, cols, 1));
  MRML_TRY(check_matrix(cols, std::max(rows, 1), 1));
  if (ldx < cols) return MRML_ERR_INVALID_ARGUMENT;
  if (rows == 0) return MRML_OK;
  if (!x || !dst || !dst_t || !aligned16(dst) || !aligned16(dst_t) || !elem_aligned(x, type))
    return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_mx4_quantize_both(type, x, ldx, dst, dst_t, rows, cols, s));
  return MRML_OK;
}

int mrml_moe_mx4_dequantize(int type, const uint8_t* src, void* out, int64_t ldo, int64_t matrix_stride, int rows,
                            int cols, int matrices, int gated, mrml_stream_t stream) {
  if (!is_float(type)) return MRML_ERR_UNSUPPORTED;
  MRML_TRY(check_matrix(rows, cols, matrices));
  if ((gated && rows % 2 != 0) || ldo < cols) return MRML_ERR_INVALID_ARGUMENT;
  if (matrices > 1 && matrix_stride < 0) return MRML_ERR_INVALID_ARGUMENT;
  if (rows == 0 || matrices == 0) return MRML_OK;
  if (!src || !out || !aligned16(src) || !elem_aligned(out, type)) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(mrml::check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  MRML_LAUNCH(mrml::launch_mx4_dequantize(type, src, out, ldo, matrices > 1 ? matrix_stride : 0, rows, cols, matrices,
                                          gated != 0, s));
  return MRML_OK;
}

size_t mrml_moe_mx4_matmul_workspace_bytes(int M, int N, int K) {
  return check_product(MRML_F32, M, N, K) == MRML_OK ? 256 : 0;
}

int mrml_moe_mx4_matmul(int type, const uint8_t* a, const uint8_t* b, void* out, int64_t ldo, int M, int N, int K,
                        void* workspace, size_t workspace_bytes, mrml_stream_t stream) {
  return matmul(type, a, b, out, ldo, M, N, K, workspace, workspace_bytes, false, stream);
}

size_t mrml_moe_mx4_linear_workspace_bytes(int T, int N, int K) {
  const size_t mm = mrml_moe_mx4_matmul_workspace_bytes(T, N, K);
  if (mm == 0 || check_matrix(T, K, 1) != MRML_OK) return 0;
  return mm + align256(mrml::mx_matrix_bytes(T, K));
}

int mrml_moe_mx4_linear(int type, const void* x, int64_t ldx, const uint8_t* w, void* out, int64_t ldo, int T, int N,
                        int K, void* workspace, size_t workspace_bytes, mrml_stream_t stream) {
  MRML_TRY(check_product(type, T, N, K));
  MRML_TRY(check_matrix(T, K, 1));
  if (ldx < K || ldo < N) return MRML_ERR_INVALID_ARGUMENT;
  if (T == 0) return MRML_OK;
  if (!x || !w || !out) return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(check_workspace(workspace, workspace_bytes, mrml_moe_mx4_linear_workspace_bytes(T, N, K)));
  const size_t mm = mrml_moe_mx4_matmul_workspace_bytes(T, N, K);
  uint8_t* xq = static_cast<uint8_t*>(workspace) + mm;
  if (!aligned16(w) || !elem_aligned(x, type) || !elem_aligned(out, type)) return MRML_ERR_INVALID_ARGUMENT;
  if (mrml::mx4_few_tokens(T, K)) {
    MRML_TRY(mrml::check_device());
    const cudaStream_t s = (cudaStream_t)stream;
    MRML_LAUNCH(mrml::launch_mx4_few(type, w, x, ldx, T, N, K, out, ldo, static_cast<int*>(workspace), s));
    return MRML_OK;
  }
  MRML_TRY(mrml_moe_mx4_quantize(type, x, ldx, 0, xq, T, K, 1, 0, stream));
  return matmul(type, xq, w, out, ldo, T, N, K, workspace, mm, true, stream);
}

size_t mrml_moe_mx4_experts_workspace_bytes(int H, int I, int E, int K, int T) {
  return check_experts(MRML_F32, H, I, E, K, T) == MRML_OK ? carve_experts(nullptr, H, I, E, K, T).bytes : 0;
}

int mrml_moe_mx4_experts(int type, const uint8_t* gate_up, const uint8_t* down, const int32_t* ids, const float* probs,
                         const float* down_scale, const void* x, int64_t ldx, void* out, int64_t ldo, int H, int I,
                         int E, int K, int T, void* workspace, size_t workspace_bytes, mrml_stream_t stream) {
  MRML_TRY(check_experts(type, H, I, E, K, T));
  if (ldx < H || ldo < H) return MRML_ERR_INVALID_ARGUMENT;
  if (T == 0) return MRML_OK;
  if (!gate_up || !down || !ids || !probs || !x || !out) return MRML_ERR_INVALID_ARGUMENT;
  if (!aligned16(gate_up) || !aligned16(down) || !elem_aligned(x, type) || !elem_aligned(out, type))
    return MRML_ERR_INVALID_ARGUMENT;
  MRML_TRY(check_workspace(workspace, workspace_bytes, carve_experts(nullptr, H, I, E, K, T).bytes));
  MRML_TRY(mrml::check_device());
  const ExpertsWs w = carve_experts(workspace, H, I, E, K, T);
  const cudaStream_t s = (cudaStream_t)stream;
  const long long pairs = (long long)T * K;
  if (mrml::mx4_few_pairs(T, K, H)) {  // three launches: no sort, no gather
    MRML_LAUNCH(mrml::launch_mx4_few_gate_up(type, gate_up, x, ldx, ids, w.pos, T, K, E, H, I, w.act, w.sort.status, s));
    MRML_LAUNCH(mrml::launch_mx4_few_down(down, w.act, ids, T, K, E, H, I, w.y, w.sort.status, s));
    MRML_LAUNCH(mrml::launch_combine_rows(type, w.y, w.pos, probs, ids, down_scale, out, ldo, H, K, T, s));
    return MRML_OK;
  }
  MRML_LAUNCH(mrml::launch_sort(ids, w.offsets, w.counts, w.pos, mrml::mx4_flat_bytes(H, K, T) ? w.pair : nullptr,
                                E, T * K, mrml::kMxRows, w.n_rows, w.sort.chunk_cnt, w.sort.status, s));
  MRML_LAUNCH(mrml::launch_mx4_gather(type, x, ldx, w.pos, w.pair, w.offsets + E, w.x, w.flat, T, H, K, w.n_rows, s));
  MRML_LAUNCH(mrml::launch_mx4_gemm(MRML_F32, gate_up, w.x, w.offsets, w.counts, E, 0, 2 * I, H, true, nullptr, 0,
                                    w.act, pairs, true, w.sort.status, s));
  MRML_LAUNCH(mrml::launch_mx4_gemm(MRML_F32, down, w.act, w.offsets, w.counts, E, 0, H, I, false, w.y, H,
                                    nullptr, pairs, true, w.sort.status, s));
  MRML_LAUNCH(mrml::launch_combine_rows(type, w.y, w.pos, probs, ids, down_scale, out, ldo, H, K, T, s));
  return MRML_OK;
}

}  // extern "C"

// Entry points of the products with bias, activation and residual in their epilogue: checks, then
// the tensor-core tiles (linear_nt_sm100.cu), or the SIMT tiles for what those do not take.
#include "linear_epi.cuh"

namespace tob {
namespace sm100 {
int linear_nt_launch(int kind, bool block_scaled, const LinOps& o, const LinEpi& ep,
                     cudaStream_t st);
// TO_EUNSUPPORTED (nothing launched) where the tiles do not apply.
int linear_pair_launch(int kind, const LinOps& o, const LinEpi& ep, cudaStream_t st);
int linear_bs_launch(int kind, const LinOps& o, const LinEpi& ep, cudaStream_t st);
}
int64_t linear_relay_bytes(int kind, const LinOps& o);
int linear_relay(int kind, LinOps* o, void* ws, cudaStream_t st);
int linear_dense_simt_launch(const void* a, int64_t lda, const void* b, int64_t M, int64_t N,
                             int64_t K, const LinEpi& ep, cudaStream_t st);
int linear_w8a8_simt_launch(bool fp8, const void* a, const void* b, int64_t M, int64_t N, int64_t K,
                            int64_t bn, int64_t bk, const LinEpi& ep, cudaStream_t st);

namespace {

// Products of int8 codes that an int32 sum holds whatever they are: (-128)^2 x 131072 is 2^31.
constexpr int64_t kInt32Terms = 131071;

LinOps make_ops(const void* a, int64_t lda, const void* b, int64_t M, int64_t N, int64_t K,
                bool b_mn) {
  return LinOps{a, b, lda, b_mn ? N : K, K, b_mn ? N : K, M, N, K};
}

// Many tokens: CTA-pair tiles, or folding tiles with block scales; few tokens or a small grid: weights
// as rows. All of them over aligned copies of the operands that TMA cannot read.
int tensor_core_launch(const char* op, int kind, bool block_scaled, LinOps o, const LinEpi& ep,
                       void* ws, size_t ws_bytes, cudaStream_t st) {
  const int64_t need = linear_relay_bytes(kind, o);
  if (need > 0) {
    if (!ws || (int64_t)ws_bytes < need)
      return fail(TO_ENOSPACE, "%s: workspace of %zu bytes is too small (%lld)", op, ws_bytes,
                  (long long)need);
    if (!aligned16(ws)) return fail(TO_EINVAL, "%s: workspace is not 16-byte aligned", op);
    const int rc = linear_relay(kind, &o, ws, st);
    if (rc) return rc;
  }
  const int rc = block_scaled ? sm100::linear_bs_launch(kind, o, ep, st)
                              : sm100::linear_pair_launch(kind, o, ep, st);
  if (rc != TO_EUNSUPPORTED) return rc;
  return sm100::linear_nt_launch(kind, block_scaled, o, ep, st);
}

// Fills the epilogue common to both products; TO_OK or a recorded failure.
int make_epi(LinEpi* ep, const char* op, const void* bias, int act, const void* res, int64_t ldr,
             void* c, int64_t ldc, int dtype, int64_t M, int64_t N) {
  if (dtype != TO_F32 && dtype != TO_F16 && dtype != TO_BF16)
    return fail(TO_EUNSUPPORTED, "%s: output dtype %s (float32, float16 and bfloat16)", op,
                dtype_name(dtype));
  if (act < kActNone || act > kActGelu)
    return fail(TO_EINVAL, "%s: unknown activation %d", op, act);
  if (M > 1 && (ldc < N || (res != nullptr && ldr < N)))
    return fail(TO_EINVAL, "%s: row strides (%lld, %lld) shorter than N=%lld", op, (long long)ldr,
                (long long)ldc, (long long)N);
  if (!c) return fail(TO_EINVAL, "%s: null output", op);
  ep->bias = bias;
  ep->res = res;
  ep->ldr = ldr;
  ep->c = c;
  ep->ldc = ldc;
  ep->dtype = dtype;
  ep->act = act;
  ep->form = act_form(act);
  return TO_OK;
}

int w8a8_epi_entry(bool fp8, const void* a, const void* b, const float* a_s, const float* b_s,
                   const void* bias, int act, const void* res, int64_t ldr, void* c, int64_t ldc,
                   int c_dtype, int64_t M, int64_t N, int64_t K, int64_t bn, int64_t bk,
                   void* ws, size_t ws_bytes, void* stream) {
  const char* op = fp8 ? "w8a8_block_fp8_matmul_bias_act" : "w8a8_block_int8_matmul_bias_act";
  if (M < 0 || N < 0 || K <= 0 || bn <= 0 || bk <= 0 || M > kDimMax || N > kDimMax ||
      K > kDimMax)
    return fail(TO_EINVAL, "%s: invalid M=%lld N=%lld K=%lld block=[%lld,%lld]", op, (long long)M,
                (long long)N, (long long)K, (long long)bn, (long long)bk);
  LinEpi ep;
  if (M == 0 || N == 0) return TO_OK;
  if (!a || !b || !a_s || !b_s) return fail(TO_EINVAL, "%s: null pointer", op);
  const int rc = make_epi(&ep, op, bias, act, res, ldr, c, ldc, c_dtype, M, N);
  if (rc) return rc;
  const int64_t kt = ceil_div(K, bk);
  ep.a_s = a_s;
  ep.b_s = b_s;
  ep.a_s_ld = ep.b_s_ld = kt;
  ep.bn = bn >= N ? N : bn;
  cudaStream_t st = (cudaStream_t)stream;
  // The tensor-core tiles change scales on whole 128-byte K slices; one K block needs none.
  if (kt > 1 && bk % 128 != 0) {
    if (!fp8 && bk > kInt32Terms)
      return fail(TO_EUNSUPPORTED, "%s: block_k=%lld, an int32 block sum holds %lld products (or a "
                  "multiple of 128)", op, (long long)bk, (long long)kInt32Terms);
    return linear_w8a8_simt_launch(fp8, a, b, M, N, K, ep.bn, bk, ep, st);
  }
  // One block of more products than int32 holds: its 128-product slices are added up in fp32, as if
  // each were a block of its own with the same scales.
  const bool fold = kt > 1 || (!fp8 && K > kInt32Terms);
  ep.kb_per_scale = (int)(kt > 1 ? bk / 128 : ceil_div(K, 128));
  return tensor_core_launch(op, fp8 ? TO_E4M3 : TO_I8, fold, make_ops(a, K, b, M, N, K, false), ep,
                            ws, ws_bytes, st);
}

}  // namespace
}  // namespace tob

extern "C" {

size_t to_gemm_bias_act_workspace_size(const void* a, int64_t lda, const void* b, int dtype,
                                       int64_t M, int64_t N, int64_t K) {
  if ((dtype != TO_F16 && dtype != TO_BF16) || M <= 0 || N <= 0 || K <= 0) return 0;
  return (size_t)tob::linear_relay_bytes(dtype, tob::make_ops(a, lda, b, M, N, K, true));
}

size_t to_w8a8_gemm_bias_act_workspace_size(const void* a, const void* b, int64_t M, int64_t N,
                                            int64_t K, int64_t block_k) {
  if (M <= 0 || N <= 0 || K <= 0 || block_k <= 0 || (block_k < K && block_k % 128 != 0)) return 0;
  return (size_t)tob::linear_relay_bytes(TO_I8, tob::make_ops(a, K, b, M, N, K, false));
}

int to_gemm_bias_act(const void* a, int64_t lda, const void* b, const void* bias, int act,
                     const void* residual, int64_t ldr, void* c, int64_t ldc, int dtype, int64_t M,
                     int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tob;
  const char* op = "gemm_bias_act";
  if (M < 0 || N < 0 || K < 0 || M > kDimMax || N > kDimMax || K > kDimMax)
    return fail(TO_EINVAL, "%s: invalid shape M=%lld N=%lld K=%lld", op, (long long)M,
                (long long)N, (long long)K);
  if (M > 1 && lda < K)
    return fail(TO_EINVAL, "%s: row stride %lld shorter than K=%lld", op, (long long)lda,
                (long long)K);
  if (M == 0 || N == 0) return TO_OK;
  if (K > 0 && (!a || !b)) return fail(TO_EINVAL, "%s: null pointer", op);
  LinEpi ep;
  const int rc = make_epi(&ep, op, bias, act, residual, ldr, c, ldc, dtype, M, N);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TO_F32 || K == 0)
    return linear_dense_simt_launch(a, lda, b, M, N, K, ep, st);
  return tensor_core_launch(op, dtype, false, make_ops(a, lda, b, M, N, K, true), ep, workspace,
                            workspace_bytes, st);
}

int to_w8a8_i8_gemm_bias_act(const int8_t* a, const int8_t* b, const float* a_s, const float* b_s,
                             const void* bias, int act, const void* residual, int64_t ldr, void* c,
                             int64_t ldc, int c_dtype, int64_t M, int64_t N, int64_t K,
                             int64_t block_n, int64_t block_k, void* workspace,
                             size_t workspace_bytes, void* stream) {
  return tob::w8a8_epi_entry(false, a, b, a_s, b_s, bias, act, residual, ldr, c, ldc, c_dtype, M, N,
                             K, block_n, block_k, workspace, workspace_bytes, stream);
}

int to_w8a8_fp8_gemm_bias_act(const void* a, const void* b, const float* a_s, const float* b_s,
                              const void* bias, int act, const void* residual, int64_t ldr, void* c,
                              int64_t ldc, int c_dtype, int64_t M, int64_t N, int64_t K,
                              int64_t block_n, int64_t block_k, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return tob::w8a8_epi_entry(true, a, b, a_s, b_s, bias, act, residual, ldr, c, ldc, c_dtype, M, N,
                             K, block_n, block_k, workspace, workspace_bytes, stream);
}

}  // extern "C"

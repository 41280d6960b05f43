// Entry point of the products of 8-bit rows (fp8.cuh) and the choice between their kernels.
#include "fp8_gemm.cuh"

extern "C" int stu_linear_fp8(const void* x, const void* x_scales, const void* W, const void* W_scales, const void* W2, const void* W2_scales,
                              const void* resid, long long resid_row_stride, void* y, long long y_row_stride, void* y_scales, int M, int N, int K,
                              int flags, void* stream) {
  if (!x || !x_scales || !W || !W_scales || !y) return STU_ERR_NULL;
  if (W2 && (!W2_scales || !y_scales)) return STU_ERR_NULL;
  if (M < 0 || N <= 0 || K <= 0 || N > INT32_MAX - fp8::PIECE || K > INT32_MAX - fp8::PIECE || M > INT32_MAX - fp8::PIECE) return STU_ERR_SHAPE;
  if (W2 && resid) return STU_ERR_UNSUPPORTED;
  if (flags & ~STU_FLAG_OVERLAP) return STU_ERR_UNSUPPORTED;
  const void* rows[] = {x, x_scales, W, W_scales, W2, W2_scales, W2 ? y : nullptr, y_scales};
  for (const void* p : rows)
    if (!aligned16(p)) return STU_ERR_ALIGN;
  if (((uintptr_t)y | (uintptr_t)resid) & 1u) return STU_ERR_ALIGN;
  if (M == 0) return STU_OK;
  const unsigned char *w2 = (const unsigned char*)W2, *w2s = (const unsigned char*)W2_scales;
  const Fp8Product p{(const unsigned char*)x, (const unsigned char*)x_scales, (const unsigned char*)W, (const unsigned char*)W_scales, w2, w2s,
                     (const bf16*)resid, resid_row_stride, W2 ? nullptr : (bf16*)y, y_row_stride, W2 ? (unsigned char*)y : nullptr,
                     (unsigned char*)y_scales, M, N, K, (flags & STU_FLAG_OVERLAP) != 0};
  return fp8_narrow_takes(p) ? fp8_narrow(p, (cudaStream_t)stream) : fp8_gemm(p, (cudaStream_t)stream);
}

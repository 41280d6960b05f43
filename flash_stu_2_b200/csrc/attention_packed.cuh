// What the kernels for packed prompts share: which keys a row sees, and the launch of the tensor-core kernel.
#pragma once
#include "common.cuh"

namespace packed {

constexpr int NOBODY = 0x7fffffff;

// First visible key of row i, which lies in one of the sequences lo .. hi - 1 (cu ascending): at most i, whatever cu holds.
__device__ __forceinline__ int first_key_in(const int* __restrict__ cu, int lo, int hi, int i, int window) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return min(max(max(cu[lo], 0), window < 0 ? 0 : i - window), i);
}
// The same for any row: NOBODY where it belongs to no sequence (before the first or behind the last).
__device__ __forceinline__ int first_key(const int* __restrict__ cu, int S, int i, int rows, int window) {
  return i >= rows || i < cu[0] || i >= cu[S] ? NOBODY : first_key_in(cu, 0, S, i, window);
}

}  // namespace packed

// bf16, hd a multiple of 8 up to 128, rows on the 16-byte grid (attention_packed_umma.cu)
int launch_packed_umma(const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows, int H,
                       int Hk, int hd, int window, float softcap, int* status, cudaStream_t st);
// fp32, hd up to 128 (attention_packed_f32.cu)
int launch_packed_f32(const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows, int H,
                      int Hk, int hd, int window, float softcap, cudaStream_t st);

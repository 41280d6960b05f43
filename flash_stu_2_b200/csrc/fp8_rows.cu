// Rows to 8 bits (fp8.cuh): quantisation of any rows, and RMSNorm, with or without a branch that is added first, whose result never exists
// in more bits outside of registers.
#include "fp8.cuh"

namespace {

constexpr int PER_LANE = 16;   // consecutive values of a lane: 16 bytes of output; 8 lanes share a block, a warp covers a piece

// 16 values from p on, of which `valid` exist (the rest: 0).
template <typename T>
__device__ __forceinline__ void load16(const T* p, int valid, bool vec, float* v) {
  if (vec && valid >= PER_LANE) {
#pragma unroll
    for (int i = 0; i < PER_LANE; i += Elem<T>::VEC) load_vec(p + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) v[i] = i < valid ? Elem<T>::to_f(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, int valid, bool vec, const float* v) {
  if (vec && valid >= PER_LANE) {
#pragma unroll
    for (int i = 0; i < PER_LANE; i += Elem<T>::VEC) store_vec(p + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < PER_LANE; i++)
      if (i < valid) p[i] = Elem<T>::from_f(v[i]);
  }
}

__device__ __forceinline__ uint32_t block_max(uint32_t a) {   // over the 8 lanes of a block
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// A warp: the 512 values (16 per lane) of `row` in group g, columns behind `cols` zero.
__device__ __forceinline__ void emit(float* v, int row, int g, int groups, int padded, unsigned char* q, unsigned char* scales) {
  const int lane = threadIdx.x & 31, col = g * fp8::PIECE + lane * PER_LANE;
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < PER_LANE; i++) a = max(a, fp8::magnitude(v[i]));
  a = block_max(a);
  if (__any_sync(0xffffffffu, a >= fp8::INF_BITS)) {   // infinities or NaN: the scale is that of the others
    a = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
      v[i] = fp8::nan_unless_finite(v[i]);
      a = max(a, v[i] == v[i] ? fp8::magnitude(v[i]) : 0u);
    }
    a = block_max(a);
  }
  const uint32_t b = fp8::scale_byte(a);
  const float inv = fp8::inverse_scale(b);
#pragma unroll
  for (int i = 0; i < PER_LANE; i++) v[i] *= inv;
  if (col < padded)
    *reinterpret_cast<uint4*>(q + (size_t)row * padded + col) =
        make_uint4(fp8::pack4(v[0], v[1], v[2], v[3]), fp8::pack4(v[4], v[5], v[6], v[7]), fp8::pack4(v[8], v[9], v[10], v[11]),
                   fp8::pack4(v[12], v[13], v[14], v[15]));
  uint32_t word = b << (8 * (lane >> 3));   // blocks behind the last: all zeros, byte 0
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  word |= __shfl_xor_sync(0xffffffffu, word, 16);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scales + fp8::scale_word(row, g, groups)) = word;
}

// Byte 0 for the rows that fill up the last 128, by one CTA.
__device__ __forceinline__ void clear_padding(int rows, int groups, unsigned char* scales) {
  const int pad = ((rows + 127) & ~127) - rows;
  for (int i = threadIdx.x; i < pad * groups; i += blockDim.x)
    *reinterpret_cast<uint32_t*>(scales + fp8::scale_word(rows + i % pad, i / pad, groups)) = 0;
}

constexpr int Q_WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(Q_WARPS * 32) quantize_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                                                                unsigned char* __restrict__ scales, int rows, int cols, long long xs, int vec) {
  pdl_trigger();
  pdl_wait();
  const int groups = fp8::groups_of(cols), padded = fp8::blocks_of(cols) * fp8::BLOCK;
  if (blockIdx.x == gridDim.x - 1) return clear_padding(rows, groups, scales);
  const long long item = (long long)blockIdx.x * Q_WARPS + (threadIdx.x >> 5);
  const int row = (int)(item / groups), g = (int)(item - (long long)row * groups);
  if (row >= rows) return;
  const int col = g * fp8::PIECE + (threadIdx.x & 31) * PER_LANE;
  float v[PER_LANE];
  load16(x + (size_t)row * xs + col, cols - col, vec != 0, v);
  emit(v, row, g, groups, padded, q, scales);
}

// s = round(x + add), stored where add is given; q = s * rsqrt(mean(s^2) + eps) * w to 8 bits.  wpr warps share a row, each of which holds NCH
// pieces of it in registers between the statistics and the scaling: x and add are read once, sum and q written once (HBM-bound where rows are
// many).  Statistics in fp32: 16 values in order, then lanes, then warps.
template <typename T, int NCH>
__global__ void __launch_bounds__(512) rmsnorm_fp8_kernel(const T* x, const T* add, const T* __restrict__ w, T* sum,
                                                          unsigned char* __restrict__ q, unsigned char* __restrict__ scales, int rows, int cols,
                                                          long long xs, long long as, long long ss, float eps, int vec, int wpr) {
  __shared__ float part[16];
  pdl_trigger();
  pdl_wait();
  const int groups = fp8::groups_of(cols), padded = fp8::blocks_of(cols) * fp8::BLOCK;
  if (blockIdx.x == gridDim.x - 1) return clear_padding(rows, groups, scales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_cta = (blockDim.x >> 5) / wpr;
  const int row = blockIdx.x * per_cta + warp / wpr, sub = warp % wpr;
  const bool live = row < rows;
  float v[NCH][PER_LANE], sq = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int col = (sub + i * wpr) * fp8::PIECE + lane * PER_LANE, valid = live ? cols - col : 0;
    load16(x + (size_t)row * xs + col, valid, vec != 0, v[i]);
  }
  if (add) {
#pragma unroll
    for (int i = 0; i < NCH; i++) {
      const int col = (sub + i * wpr) * fp8::PIECE + lane * PER_LANE, valid = live ? cols - col : 0;
      float a[PER_LANE];
      load16(add + (size_t)row * as + col, valid, vec != 0, a);
#pragma unroll
      for (int j = 0; j < PER_LANE; j++) v[i][j] = round_to<T>(v[i][j] + a[j]);
      store16(sum + (size_t)row * ss + col, valid, vec != 0, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; i++)
#pragma unroll
    for (int j = 0; j < PER_LANE; j++) sq = fmaf(v[i][j], v[i][j], sq);
  sq = warp_sum(sq);
  if (wpr > 1) {
    if (lane == 0) part[warp] = sq;
    __syncthreads();
    sq = 0.f;
    for (int i = 0; i < wpr; i++) sq += part[warp - sub + i];
  }
  if (!live) return;
  const float r = rsqrtf(sq / (float)cols + eps);
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int g = sub + i * wpr, col = g * fp8::PIECE + lane * PER_LANE;
    if (g < groups) {   // (of the whole warp)
      float g16[PER_LANE];
      load16(w + col, cols - col, vec != 0, g16);
#pragma unroll
      for (int j = 0; j < PER_LANE; j++) v[i][j] = col + j < cols ? v[i][j] * r * g16[j] : 0.f;
      emit(v[i], row, g, groups, padded, q, scales);
    }
  }
}

template <typename T>
bool on_grid(const void* p, long long stride) { return aligned16(p) && stride % Elem<T>::VEC == 0; }

template <typename T>
int launch_quantize(const void* x, void* q, void* scales, int rows, int cols, long long xs, cudaStream_t st) {
  const long long items = (long long)rows * fp8::groups_of(cols), ctas = (items + Q_WARPS - 1) / Q_WARPS + 1;
  if (ctas > INT32_MAX) return STU_ERR_SHAPE;
  const cudaError_t e = launch_maybe_overlapped(quantize_kernel<T>, dim3((unsigned)ctas), dim3(Q_WARPS * 32), 0, st, true, (const T*)x,
                                                (unsigned char*)q, (unsigned char*)scales, rows, cols, xs, (int)on_grid<T>(x, xs));
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}

template <typename T>
int launch_rmsnorm(const void* x, const void* add, const void* w, void* sum, void* q, void* scales, int rows, int cols, long long xs, long long as,
                   long long ss, float eps, cudaStream_t st) {
  const int groups = fp8::groups_of(cols);
  int wpr = 1;
  while (wpr * 4 < groups) wpr *= 2;
  while (wpr < groups && wpr < 16 && (long long)rows * wpr < 148 * 8) wpr *= 2;   // few rows: a shorter chain each
  const int nch = (groups + wpr - 1) / wpr, warps = wpr > 8 ? wpr : 8, per_cta = warps / wpr;
  const int vec = on_grid<T>(x, xs) && aligned16(w) && (!add || (on_grid<T>(add, as) && on_grid<T>(sum, ss)));
  const dim3 grid((rows + per_cta - 1) / per_cta + 1), block(warps * 32);
  cudaError_t e;
#define STU_NORM(N_)                                                                                                              \
  e = launch_maybe_overlapped(rmsnorm_fp8_kernel<T, N_>, grid, block, 0, st, true, (const T*)x, (const T*)add, (const T*)w, (T*)sum, \
                              (unsigned char*)q, (unsigned char*)scales, rows, cols, xs, as, ss, eps, vec, wpr)
  if (nch == 1) STU_NORM(1);
  else if (nch == 2) STU_NORM(2);
  else if (nch == 3) STU_NORM(3);
  else STU_NORM(4);
#undef STU_NORM
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

extern "C" int stu_quantize_fp8(const void* x, void* q, void* scales, int rows, int cols, long long x_row_stride, int dtype, void* stream) {
  if (!x || !q || !scales) return STU_ERR_NULL;
  if (rows < 0 || cols <= 0 || cols > INT32_MAX - fp8::PIECE) return STU_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(scales)) return STU_ERR_ALIGN;
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (rows == 0) return STU_OK;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == STU_F32 ? launch_quantize<float>(x, q, scales, rows, cols, x_row_stride, st)
                          : launch_quantize<bf16>(x, q, scales, rows, cols, x_row_stride, st);
}

extern "C" int stu_rmsnorm_fp8(const void* x, const void* add, const void* w, void* sum, void* q, void* scales, int rows, int cols,
                               long long x_row_stride, long long add_row_stride, long long sum_row_stride, float eps, int dtype, void* stream) {
  if (!x || !w || !q || !scales || (add && !sum)) return STU_ERR_NULL;
  if (rows < 0 || cols <= 0 || cols > 32768) return STU_ERR_SHAPE;   // 16 warps x 4 pieces
  if (!aligned16(q) || !aligned16(scales)) return STU_ERR_ALIGN;
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (rows == 0) return STU_OK;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == STU_F32 ? launch_rmsnorm<float>(x, add, w, sum, q, scales, rows, cols, x_row_stride, add_row_stride, sum_row_stride, eps, st)
                          : launch_rmsnorm<bf16>(x, add, w, sum, q, scales, rows, cols, x_row_stride, add_row_stride, sum_row_stride, eps, st);
}

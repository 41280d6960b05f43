// Rows to 8 bits (fp8.cuh): quantisation of any rows, and RMSNorm, with or without a branch that is added first, whose result never exists
// in more bits outside of registers.  HBM-bound where rows are many (bf16: 100000 x 1024 quantised in 47 us, 6.5 TB/s; 65536 x 1024 normalised in 45, 4.5 TB/s, with a
// branch in 84, 5.6 TB/s; fp32 with a branch 142, 6.2 TB/s); a launch's latency where they are few (1 x 1536 1.9 us).
#include <algorithm>

#include "fp8.cuh"

int device_sm_count();   // gemm_tc.cu

namespace {

// A warp has a piece of a row: 512 columns, four blocks.  A lane has V groups of 32 bytes, 32 groups apart, P values each: whole sectors, and 8 or 16 lanes
// per block.  (Vectors of 16 bytes, 32 apart, take half the lines per load but a shuffle more per block and vector: 65536 x 1024 bf16 with a branch 98 us, so 85;
// fp32 in groups of 64 bytes 1999 x 1000 10.9 us, so 7.0.)
enum Grid { ANY, BY16, BY32 };   // what the addresses of all rows are multiples of
template <typename T> struct Lane {
  static constexpr int P = 32 / sizeof(T), V = 512 / (32 * P);
  uint32_t w[V][8];
  static __device__ __forceinline__ int column(int g, int i) { return g * fp8::PIECE + (i * 32 + (int)(threadIdx.x & 31)) * P; }
  __device__ __forceinline__ float get(int i, int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i][e]);
    else return __uint_as_float(e & 1 ? w[i][e >> 1] & 0xffff0000u : w[i][e >> 1] << 16);
  }
  __device__ __forceinline__ void set2(int i, int e, float a, float b) {   // values e and e + 1, rounded
    if constexpr (sizeof(T) == 4) {
      w[i][e] = __float_as_uint(a);
      w[i][e + 1] = __float_as_uint(b);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[i][e >> 1] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
// The words from byte `shift` on (uniform in the warp, a multiple of 2, 0 < shift < 16), of which there are 8 + 4.
__device__ __forceinline__ void move_down(uint32_t (&r)[12], int shift) {
#pragma unroll
  for (int j = 0; j < 10; j++) r[j] = shift & 8 ? r[j + 2] : r[j];
#pragma unroll
  for (int j = 0; j < 9; j++) r[j] = shift & 4 ? r[j + 1] : r[j];
  if (shift & 2) {
#pragma unroll
    for (int j = 0; j < 8; j++) r[j] = __funnelshift_r(r[j], r[j + 1], 16);
  }
}
__device__ __forceinline__ void take(uint32_t* r, const char* at, bool ok) {
  const uint4 u = ok ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
  r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
}
// A row's piece g, columns from `cols` on zero (cols = 0: nothing is read), whole warps.  Rows off the 16-byte grid are read in aligned vectors that
// hold a byte of the row at least, three for two, and moved (7996 x 1111 bf16, value by value 12.2, now 8.6 us).
template <Grid GRID, typename T> __device__ __forceinline__ Lane<T> load(const T* row, int g, int cols) {
  constexpr int P = Lane<T>::P;
  const int off = GRID != ANY ? 0 : (int)(reinterpret_cast<uintptr_t>(row) & 15);
  const char* end = reinterpret_cast<const char*>(row + cols);
  Lane<T> v;
#pragma unroll
  for (int i = 0; i < Lane<T>::V; i++) {
    const int col = Lane<T>::column(g, i);
    const char* at = reinterpret_cast<const char*>(row + col) - off;
    uint32_t(&w)[8] = v.w[i];
    if (GRID == BY32 && col + P <= cols) {
      asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(at));
      continue;
    }
    if (!off) {
      take(w, at, col < cols);
      take(w + 4, at + 16, col < cols && at + 16 < end);
    } else {
      uint32_t r[12];
      take(r, at, col < cols);
      take(r + 4, at + 16, col < cols && at + 16 < end);
      take(r + 8, at + 32, col < cols && at + 32 < end);
      move_down(r, off);
#pragma unroll
      for (int j = 0; j < 8; j++) w[j] = r[j];
    }
    if (col + P > cols) {   // (what lies behind the row is not the row's)
#pragma unroll
      for (int e = 0; e < P; e++)
        if (col + e >= cols) {
          if constexpr (sizeof(T) == 4) w[e] = 0;
          else w[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
        }
    }
  }
  return v;
}
// The same to memory: no byte beside the row or of another warp's piece is touched.
template <Grid GRID, typename T> __device__ __forceinline__ void store(T* row, int g, int cols, const Lane<T>& v) {
  constexpr int P = Lane<T>::P, V = Lane<T>::V, A = P / 2;   // A: values of an aligned vector
  const int off = GRID != ANY ? 0 : (int)(reinterpret_cast<uintptr_t>(row) & 15), lane = threadIdx.x & 31, ahead = off / (int)sizeof(T);
  const int last = cols - (cols + ahead) % A;   // behind the row's last whole aligned vector
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int col = Lane<T>::column(g, i);
    if (GRID == BY32 && col + P <= cols) {
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + col), "r"(v.w[i][0]), "r"(v.w[i][1]), "r"(v.w[i][2]), "r"(v.w[i][3]),
                   "r"(v.w[i][4]), "r"(v.w[i][5]), "r"(v.w[i][6]), "r"(v.w[i][7]) : "memory");
      continue;
    }
    uint32_t r[12] = {};
    if (off) {   // the aligned vectors from `ahead` values before the lane's on: those are the neighbour's, lane 0's the last lane's of the groups before
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, v.w[i][4 + j], 1), m = i ? __shfl_sync(0xffffffffu, v.w[i ? i - 1 : 0][4 + j], 31) : 0u;
        r[j] = lane ? n : m;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) r[4 + j] = v.w[i][j];
      move_down(r, 16 - off);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) r[j] = v.w[i][j];
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int c = col - ahead + k * A;
      if (c >= g * fp8::PIECE && c + A <= cols) *reinterpret_cast<uint4*>(row + c) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
    }
    // single values: the piece's first ones up to an aligned vector, its last ones and the row's last ones behind one
    const bool head = off && lane == 0 && i == 0, tail = off && lane == 31 && i == V - 1;
#pragma unroll
    for (int e = 0; e < P; e++)
      if (col + e < cols && ((head && e < A - ahead) || (tail && e >= P - ahead) || col + e >= last)) {
        if constexpr (sizeof(T) == 4) row[col + e] = __uint_as_float(v.w[i][e]);
        else reinterpret_cast<uint16_t*>(row)[col + e] = (uint16_t)(e & 1 ? v.w[i][e >> 1] >> 16 : v.w[i][e >> 1]);
      }
  }
}

// max(a, |b|, |c|), NaN if one of them is
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
// The 512 values of `row` in group g, columns behind `cols` zero, to 8 bits.  A block: 8 lanes (bf16), or a group of 16 (fp32).
template <typename T> __device__ __forceinline__ void emit(float (&v)[Lane<T>::V][Lane<T>::P], int row, int g, int groups, int padded, unsigned char* q,
                                                           unsigned char* scales) {
  constexpr int P = Lane<T>::P, V = Lane<T>::V, MATES = 128 / P;
  const int lane = threadIdx.x & 31;
  float a[V], most = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++) {
    a[i] = 0.f;
#pragma unroll
    for (int e = 0; e < P; e += 2) a[i] = max_magnitude(a[i], v[i][e], v[i][e + 1]);
    most = max_magnitude(most, a[i], 0.f);
  }
  if (__any_sync(0xffffffffu, !(most < INFINITY))) {   // infinities or NaN: the scale is that of the others
#pragma unroll
    for (int i = 0; i < V; i++) {
      a[i] = 0.f;
#pragma unroll
      for (int e = 0; e < P; e++) {
        v[i][e] = fp8::nan_unless_finite(v[i][e]);
        a[i] = fmaxf(a[i], fabsf(v[i][e]));   // (of numbers alone)
      }
    }
  }
#pragma unroll
  for (int o = 1; o < MATES; o <<= 1)
#pragma unroll
    for (int i = 0; i < V; i++) a[i] = fmaxf(a[i], __shfl_xor_sync(0xffffffffu, a[i], o));
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const uint32_t b = fp8::scale_byte(__float_as_uint(a[i]));
    const float inv = fp8::inverse_scale(b);
    const int col = Lane<T>::column(g, i);
    uint32_t o[P / 4];
#pragma unroll
    for (int j = 0; j < P / 4; j++) o[j] = fp8::pack4(v[i][4 * j] * inv, v[i][4 * j + 1] * inv, v[i][4 * j + 2] * inv, v[i][4 * j + 3] * inv);
    if (col < padded) {
      unsigned char* to = q + (size_t)row * padded + col;
      if constexpr (P == 8) *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
      else *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    word |= b << (8 * ((i * 32 + lane) / MATES));   // blocks behind the last: all zeros, byte 0
  }
#pragma unroll
  for (int o = MATES; o < 32; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scales + fp8::scale_word(row, g, groups)) = word;
}

// Byte 0 for the rows that fill up the last 128, by one CTA.
__device__ __forceinline__ void clear_padding(int rows, int groups, unsigned char* scales) {
  const int pad = ((rows + 127) & ~127) - rows;
  for (int i = threadIdx.x; i < pad * groups; i += blockDim.x)
    *reinterpret_cast<uint32_t*>(scales + fp8::scale_word(rows + i % pad, i / pad, groups)) = 0;
}

constexpr int WARPS = 8;

template <typename T, Grid GRID>
__global__ void __launch_bounds__(WARPS * 32) quantize_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                                                              unsigned char* __restrict__ scales, int rows, int cols, long long xs) {
  pdl_trigger();
  pdl_wait();
  const int groups = fp8::groups_of(cols), padded = fp8::blocks_of(cols) * fp8::BLOCK;
  if (blockIdx.x == gridDim.x - 1) return clear_padding(rows, groups, scales);
  const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int row = (int)(item / groups), g = (int)(item - (long long)row * groups);
  if (row >= rows) return;
  const Lane<T> raw = load<GRID>(x + (size_t)row * xs, g, cols);
  float v[Lane<T>::V][Lane<T>::P];
#pragma unroll
  for (int i = 0; i < Lane<T>::V; i++)
#pragma unroll
    for (int e = 0; e < Lane<T>::P; e++) v[i][e] = raw.get(i, e);
  emit<T>(v, row, g, groups, padded, q, scales);
}

// 1 / sqrt(a): the hardware's, which is off by up to two units in the last place, and a step of Newton's method with the product's rounding error in it: every
// such unit moves one in a million of the 8-bit values to its neighbour.
__device__ __forceinline__ float inverse_sqrt(float a) {
  const float y = rsqrtf(a), h = a * y, l = fmaf(a, y, -h), e = fmaf(-l, y, fmaf(-h, y, 1.f));
  const float r = fmaf(0.5f * y, e, y);
  return isfinite(r) ? r : y;   // (a = 0 or infinite)
}

// Of a piece: a lane's 16 values in order, then the lanes.
template <typename T> __device__ __forceinline__ float sum_squares(const Lane<T>& v) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < Lane<T>::V; j++)
#pragma unroll
    for (int e = 0; e < Lane<T>::P; e++) s = fmaf(v.get(j, e), v.get(j, e), s);
  return warp_sum(s);
}
template <typename T> __device__ __forceinline__ void scale_and_emit(const Lane<T>& v, const Lane<T>& w, float r, int row, int g, int groups, int cols, int padded,
                                                                     unsigned char* q, unsigned char* scales) {
  constexpr int P = Lane<T>::P, V = Lane<T>::V;
  float f[V][P];
#pragma unroll
  for (int j = 0; j < V; j++)
#pragma unroll
    for (int e = 0; e < P; e++) f[j][e] = v.get(j, e) * r * w.get(j, e);
  if (g == groups - 1) {   // (an infinite r times the zeros behind the row)
#pragma unroll
    for (int j = 0; j < V; j++)
#pragma unroll
      for (int e = 0; e < P; e++)
        if (Lane<T>::column(g, j) + e >= cols) f[j][e] = 0.f;
  }
  emit<T>(f, row, g, groups, padded, q, scales);
}

// s = round(x + add), stored where add is given; q = s * rsqrt(mean(s^2) + eps) * w to 8 bits.  wpr warps share a row, each of which holds NCH
// pieces of it between the statistics and the scaling, in the type that they came in: x and add are read once, sum and q written once.  Statistics in
// fp32: a lane's 16 values in order, then the lanes of a piece, then the pieces in order, whoever has them: a row's result does not depend on how many rows there are.
template <typename T, int NCH, Grid GRID>
__global__ void __launch_bounds__(512) rmsnorm_fp8_kernel(const T* x, const T* add, const T* __restrict__ w, T* sum, unsigned char* __restrict__ q,
                                                          unsigned char* __restrict__ scales, int rows, int cols, long long xs, long long as,
                                                          long long ss, float eps, int wpr) {
  __shared__ float part[16 * NCH];
  pdl_trigger();
  pdl_wait();
  const int groups = fp8::groups_of(cols), padded = fp8::blocks_of(cols) * fp8::BLOCK;
  if (blockIdx.x == gridDim.x - 1) return clear_padding(rows, groups, scales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_cta = (blockDim.x >> 5) / wpr;
  const int row = blockIdx.x * per_cta + warp / wpr, sub = warp % wpr, live = row < rows ? cols : 0;
  constexpr int P = Lane<T>::P, V = Lane<T>::V;
  Lane<T> v[NCH];
  float sq[NCH];
#pragma unroll
  for (int i = 0; i < NCH; i++) v[i] = load<GRID>(x + (size_t)row * xs, sub + i * wpr, live);
  if (add) {
#pragma unroll
    for (int i = 0; i < NCH; i++) {
      const Lane<T> a = load<GRID>(add + (size_t)row * as, sub + i * wpr, live);
#pragma unroll
      for (int j = 0; j < V; j++)
#pragma unroll
        for (int e = 0; e < P; e += 2) v[i].set2(j, e, v[i].get(j, e) + a.get(j, e), v[i].get(j, e + 1) + a.get(j, e + 1));
      store<GRID>(sum + (size_t)row * ss, sub + i * wpr, live, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; i++) sq[i] = sum_squares(v[i]);
  float total = 0.f;
  if (wpr > 1) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NCH; i++) part[(warp - sub) * NCH + sub + i * wpr] = sq[i];
    }
    __syncthreads();
    for (int i = 0; i < groups; i++) total += part[(warp - sub) * NCH + i];
  } else {
#pragma unroll
    for (int i = 0; i < NCH; i++) total += sq[i];   // (pieces that do not exist add 0)
  }
  if (row >= rows) return;
  const float r = inverse_sqrt(total / (float)cols + eps);
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int g = sub + i * wpr;
    if (g < groups) {   // (of the whole warp)
      scale_and_emit<T>(v[i], load<GRID>(w, g, cols), r, row, g, groups, cols, padded, q, scales);
    }
  }
}

// The same without a branch for the many bf16 rows of a prefill: a warp takes row after row and asks for the next one before it works on this one, so that loads
// are under way all the time.  us, a CTA per 8 rows, which has loaded when it begins to compute, and so: 65536 x 1024 47.4 and 45.3, 16384 x 1536 23.8 and
// 18.8, 8192 x 1536 13.5 and 11.8.  Where there are more bytes to load the registers that hold them ahead cost more than they gain: with a branch 84.1 and
// 85.4, fp32 60.5 and 72.8, with a branch 142 and 159.
template <typename T, int NCH, Grid GRID>
__global__ void __launch_bounds__(WARPS * 32, NCH <= 2 ? 3 : 2) rmsnorm_fp8_rows_kernel(const T* __restrict__ x, const T* __restrict__ w, unsigned char* __restrict__ q,
                                                                                         unsigned char* __restrict__ scales, int rows, int cols, long long xs,
                                                                                         float eps) {
  pdl_trigger();
  pdl_wait();
  const int groups = fp8::groups_of(cols), padded = fp8::blocks_of(cols) * fp8::BLOCK;
  if (blockIdx.x == gridDim.x - 1) return clear_padding(rows, groups, scales);
  const int stride = (gridDim.x - 1) * WARPS;
  int row = blockIdx.x * WARPS + (threadIdx.x >> 5);
  Lane<T> v[NCH], next[NCH], wv[NCH];
#pragma unroll
  for (int i = 0; i < NCH; i++) next[i] = load<GRID>(x + (size_t)row * xs, i, row < rows ? cols : 0);
  if constexpr (NCH <= 2) {
#pragma unroll
    for (int i = 0; i < NCH; i++) wv[i] = load<GRID>(w, i, cols);
  }
  for (; row < rows; row += stride) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; i++) {
      v[i] = next[i];
      next[i] = load<GRID>(x + (size_t)(row + stride) * xs, i, row + stride < rows ? cols : 0);
    }
#pragma unroll
    for (int i = 0; i < NCH; i++) total += sum_squares(v[i]);
    const float r = inverse_sqrt(total / (float)cols + eps);
#pragma unroll
    for (int i = 0; i < NCH; i++)
      if (i < groups) scale_and_emit<T>(v[i], NCH <= 2 ? wv[i] : load<GRID>(w, i, cols), r, row, i, groups, cols, padded, q, scales);
  }
}

// What the addresses of all rows are multiples of.
template <typename T> Grid grid_of(const void* p, long long stride) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * (long long)sizeof(T));
  return a & 15 ? ANY : a & 31 ? BY16 : BY32;
}

template <typename T>
int launch_quantize(const void* x, void* q, void* scales, int rows, int cols, long long xs, cudaStream_t st) {
  const long long items = (long long)rows * fp8::groups_of(cols), ctas = (items + WARPS - 1) / WARPS + 1;
  if (ctas > INT32_MAX) return STU_ERR_SHAPE;
  const Grid grid = grid_of<T>(x, xs);
  const cudaError_t e = launch_maybe_overlapped(grid == ANY ? quantize_kernel<T, ANY> : grid == BY16 ? quantize_kernel<T, BY16> : quantize_kernel<T, BY32>,
                                                dim3((unsigned)ctas), dim3(WARPS * 32), 0, st, true, (const T*)x, (unsigned char*)q,
                                                (unsigned char*)scales, rows, cols, xs);
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}

template <typename T, Grid GRID>
int launch_rmsnorm_on(const T* x, const T* add, const T* w, T* sum, unsigned char* q, unsigned char* scales, int rows, int cols, long long xs, long long as,
                      long long ss, float eps, cudaStream_t st) {
  const int groups = fp8::groups_of(cols);
  int wpr = 1;
  while (wpr * 4 < groups) wpr *= 2;
  while (wpr < groups && wpr < 16 && (long long)rows * wpr < device_sm_count() * WARPS) wpr *= 2;   // few rows: a shorter chain each
  const int nch = (groups + wpr - 1) / wpr, warps = wpr > WARPS ? wpr : WARPS, per_cta = warps / wpr;
  const dim3 grid((rows + per_cta - 1) / per_cta + 1), block(warps * 32);
  if constexpr (GRID != ANY && sizeof(T) == 2) {
    const int ctas = (nch <= 2 ? 3 : 2) * device_sm_count();
    if (!add && wpr == 1 && rows >= ctas * WARPS) {
      const auto many = nch == 1 ? rmsnorm_fp8_rows_kernel<T, 1, GRID> : nch == 2 ? rmsnorm_fp8_rows_kernel<T, 2, GRID>
                        : nch == 3 ? rmsnorm_fp8_rows_kernel<T, 3, GRID> : rmsnorm_fp8_rows_kernel<T, 4, GRID>;
      const cudaError_t e = launch_maybe_overlapped(many, dim3(ctas + 1), dim3(WARPS * 32), 0, st, true, x, w, q, scales, rows, cols, xs, eps);
      if (e != cudaSuccess) return (int)e;
      STU_CHECK_LAUNCH();
      return STU_OK;
    }
  }
  const auto kernel = nch == 1 ? rmsnorm_fp8_kernel<T, 1, GRID> : nch == 2 ? rmsnorm_fp8_kernel<T, 2, GRID>
                      : nch == 3 ? rmsnorm_fp8_kernel<T, 3, GRID> : rmsnorm_fp8_kernel<T, 4, GRID>;
  const cudaError_t e = launch_maybe_overlapped(kernel, grid, block, 0, st, true, x, add, w, sum, q, scales, rows, cols, xs, as, ss, eps, wpr);
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}
template <typename T>
int launch_rmsnorm(const void* x, const void* add, const void* w, void* sum, void* q, void* scales, int rows, int cols, long long xs, long long as,
                   long long ss, float eps, cudaStream_t st) {
  Grid grid = std::min(grid_of<T>(x, xs), grid_of<T>(w, 0));
  if (add) grid = std::min(grid, std::min(grid_of<T>(add, as), grid_of<T>(sum, ss)));
  const auto launch = grid == ANY ? launch_rmsnorm_on<T, ANY> : grid == BY16 ? launch_rmsnorm_on<T, BY16> : launch_rmsnorm_on<T, BY32>;
  return launch((const T*)x, (const T*)add, (const T*)w, (T*)sum, (unsigned char*)q, (unsigned char*)scales, rows, cols, xs, as, ss, eps, st);
}

// Whether an address is one of a whole element.
bool whole(const void* p, int dtype) { return !(reinterpret_cast<uintptr_t>(p) & (dtype == STU_F32 ? 3u : 1u)); }

}  // namespace

extern "C" int stu_quantize_fp8(const void* x, void* q, void* scales, int rows, int cols, long long x_row_stride, int dtype, void* stream) {
  if (!x || !q || !scales) return STU_ERR_NULL;
  if (rows < 0 || cols <= 0 || cols > INT32_MAX - fp8::PIECE) return STU_ERR_SHAPE;
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (!aligned16(q) || !aligned16(scales) || !whole(x, dtype)) return STU_ERR_ALIGN;
  if (rows == 0) return STU_OK;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == STU_F32 ? launch_quantize<float>(x, q, scales, rows, cols, x_row_stride, st)
                          : launch_quantize<bf16>(x, q, scales, rows, cols, x_row_stride, st);
}

extern "C" int stu_rmsnorm_fp8(const void* x, const void* add, const void* w, void* sum, void* q, void* scales, int rows, int cols,
                               long long x_row_stride, long long add_row_stride, long long sum_row_stride, float eps, int dtype, void* stream) {
  if (!x || !w || !q || !scales || (add && !sum)) return STU_ERR_NULL;
  if (rows < 0 || cols <= 0 || cols > 32768) return STU_ERR_SHAPE;   // 16 warps x 4 pieces
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (!aligned16(q) || !aligned16(scales) || !whole(x, dtype) || !whole(add, dtype) || !whole(w, dtype) || !whole(sum, dtype)) return STU_ERR_ALIGN;
  if (rows == 0) return STU_OK;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == STU_F32 ? launch_rmsnorm<float>(x, add, w, sum, q, scales, rows, cols, x_row_stride, add_row_stride, sum_row_stride, eps, st)
                          : launch_rmsnorm<bf16>(x, add, w, sum, q, scales, rows, cols, x_row_stride, add_row_stride, sum_row_stride, eps, st);
}

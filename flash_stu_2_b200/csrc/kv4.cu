// Keys and values into a ring cache of 4 bits (kv4.cuh), and back.
#include "kv4.cuh"

int device_sm_count();   // gemm_tc.cu

namespace {

// The keys and values of qkv's rows into the rings: eight lanes per piece of a row.  Rows are `cu`'s packed sequences (sequence b: rows cu[b] ..
// cu[b + 1] - 1), or `per_seq` each.  Of each sequence the last `slots` are written, at positions pos[2 b] and up; the last CTA moves pos on.
// Bound by HBM: 4 (fp32: 8) bytes of a key and a value are read where 1.1 are written.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_write_kernel(const T* __restrict__ qkv, long long row_stride, unsigned char* __restrict__ k4,
                                                        unsigned char* __restrict__ v4, int* __restrict__ pos, const int* __restrict__ cu, int B,
                                                        long long rows, int per_seq, int H, int Hk, int hd, int slots) {
  const int pieces = kv4::pieces_of(hd), width = kv4::width_of(hd);
  const int units = 2 * Hk * pieces;                 // of a row: keys' heads, then values'
  const long long total = rows * units, head_bytes = kv4::head_bytes(hd, slots);
  const int i = threadIdx.x & 7;
  for (long long u0 = ((long long)blockIdx.x * 256 + (threadIdx.x & ~31)) >> 3; u0 < total; u0 += (long long)gridDim.x * 32) {   // warp-uniform
    const long long u = u0 + ((threadIdx.x & 31) >> 3);
    const long long row = u < total ? u / units : rows - 1;
    const int unit = (int)(u - row * units);
    int b, first, end;
    if (cu) {   // the sequence of the row: the last one that begins at or before it and is not empty
      int lo = 0, hi = B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= row) lo = mid;
        else hi = mid;
      }
      b = lo;
      first = cu[b];
      end = cu[b + 1];
    } else {
      b = (int)(row / per_seq);
      first = 0;
      end = per_seq;
    }
    const long long t = cu ? row - first : row - (long long)b * per_seq;
    const int count = end - first;
    const bool keep = u < total && t >= 0 && t < count && t >= (long long)count - slots;
    const int piece = unit % pieces, head = unit / pieces % Hk, which = unit / (pieces * Hk) & 1;
    const bool there = keep && piece * 64 + i * 8 < hd;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there) kv4::load8<VEC>(qkv + row * row_stride + (long long)(H + which * Hk + head) * hd + piece * 64 + i * 8, x);
    uint32_t word, scale;
    kv4::quantize(x, there, word, scale);
    if (keep) {
      const int slot = kv4::slot_of(pos[2 * b] + (int)t, slots);
      unsigned char* ring = (which ? v4 : k4) + ((long long)b * Hk + head) * head_bytes;
      if (i * 8 < width / pieces) reinterpret_cast<uint32_t*>(ring)[(long long)slot * (width / 8) + kv4::word_at(i, piece, pieces)] = word;
      if (i == 0) reinterpret_cast<uint32_t*>(ring + (long long)slots * (width / 2))[(long long)slot * pieces + piece] = scale;
    }
  }
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&pos[1], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (last) {
    for (int b = threadIdx.x; b < B; b += 256) pos[2 * b] += cu ? max(cu[b + 1] - cu[b], 0) : per_seq;
    if (threadIdx.x == 0) pos[1] = 0;
  }
}

__device__ __forceinline__ void store8(float* p, const float* x) {
  store_vec(p, x);
  store_vec(p + 4, x + 4);
}
__device__ __forceinline__ void store8(bf16* p, const float* x) { store_vec(p, x); }

// Rings as values [B][slots][Hk hd]: a thread per word.
template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const unsigned char* __restrict__ k4, const unsigned char* __restrict__ v4, T* __restrict__ k,
                                                       T* __restrict__ v, int B, int Hk, int hd, int slots) {
  const int pieces = kv4::pieces_of(hd), width = kv4::width_of(hd), words = hd / 8;
  const long long total = (long long)B * slots * Hk * words, head_bytes = kv4::head_bytes(hd, slots);
  const unsigned char* from = blockIdx.y ? v4 : k4;
  T* to = blockIdx.y ? v : k;
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < total; u += (long long)gridDim.x * 256) {
    const long long at = u / words;
    const int w = (int)(u - at * words);
    const long long bs = at / Hk;
    const int head = (int)(at - bs * Hk);
    const long long b = bs / slots;
    const int slot = (int)(bs - b * slots), piece = w >> 3;
    const unsigned char* ring = from + (b * Hk + head) * head_bytes;
    const uint32_t word = reinterpret_cast<const uint32_t*>(ring)[(long long)slot * (width / 8) + kv4::word_at(w & 7, piece, pieces)];
    const uint32_t scale = reinterpret_cast<const uint32_t*>(ring + (long long)slots * (width / 2))[(long long)slot * pieces + piece];
    const float low = __uint_as_float(scale << 16), step = __uint_as_float(scale & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = fmaf((float)(word >> 4 * e & 15u), step, low);
    store8(to + u * 8, x);
  }
}

template <typename T>
int launch_write(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const int* cu, int B, long long rows, int per_seq, int H, int Hk,
                 int hd, int slots, cudaStream_t st) {
  const long long warps = (rows * 2 * Hk * kv4::pieces_of(hd) + 3) / 4;
  const int grid = (int)(warps < 8 ? 1 : (warps + 7) / 8 < 8ll * device_sm_count() ? (warps + 7) / 8 : 8ll * device_sm_count());
  const bool vec = aligned16(qkv) && row_stride % (16 / (int)sizeof(T)) == 0;
  if (vec)
    kv4_write_kernel<T, true><<<grid, 256, 0, st>>>((const T*)qkv, row_stride, (unsigned char*)k4, (unsigned char*)v4, pos, cu, B, rows, per_seq, H, Hk,
                                                    hd, slots);
  else
    kv4_write_kernel<T, false><<<grid, 256, 0, st>>>((const T*)qkv, row_stride, (unsigned char*)k4, (unsigned char*)v4, pos, cu, B, rows, per_seq, H, Hk,
                                                     hd, slots);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

extern "C" int stu_kv4_write(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const int* cu_seqlens, int B, long long rows, int H,
                             int Hk, int hd, int slots, int dtype, void* stream) {
  if (!qkv || !k4 || !v4 || !pos) return STU_ERR_NULL;
  const int rc = kv4::geometry(B, H, Hk, hd, slots, dtype);
  if (rc != STU_OK) return rc;
  if (rows <= 0 || rows > 0x7fffffffll || row_stride < (long long)(H + 2 * Hk) * hd || (!cu_seqlens && rows % B)) return STU_ERR_SHAPE;
  if (!aligned16(k4) || !aligned16(v4)) return STU_ERR_ALIGN;
  const int per_seq = cu_seqlens ? 0 : (int)(rows / B);
  return dtype == STU_F32 ? launch_write<float>(qkv, row_stride, k4, v4, pos, cu_seqlens, B, rows, per_seq, H, Hk, hd, slots, (cudaStream_t)stream)
                          : launch_write<bf16>(qkv, row_stride, k4, v4, pos, cu_seqlens, B, rows, per_seq, H, Hk, hd, slots, (cudaStream_t)stream);
}

extern "C" int stu_kv4_read(const void* k4, const void* v4, void* k, void* v, int B, int Hk, int hd, int slots, int dtype, void* stream) {
  if (!k4 || !v4 || !k || !v) return STU_ERR_NULL;
  const int rc = kv4::geometry(B, Hk, Hk, hd, slots, dtype);
  if (rc != STU_OK) return rc;
  if (!aligned16(k4) || !aligned16(v4) || !aligned16(k) || !aligned16(v)) return STU_ERR_ALIGN;
  const long long blocks = ((long long)B * slots * Hk * (hd / 8) + 255) / 256;
  const dim3 grid((unsigned)(blocks < 0x3fffffff ? blocks : 0x3fffffff), 2);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == STU_F32)
    kv4_read_kernel<float><<<grid, 256, 0, st>>>((const unsigned char*)k4, (const unsigned char*)v4, (float*)k, (float*)v, B, Hk, hd, slots);
  else
    kv4_read_kernel<bf16><<<grid, 256, 0, st>>>((const unsigned char*)k4, (const unsigned char*)v4, (bf16*)k, (bf16*)v, B, Hk, hd, slots);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

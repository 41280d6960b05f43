// Attention of whole prompts, packed behind one another: causal, sliding window, ALiBi, soft cap, several query heads to a key head.
//
// Every position of a packed row is relative (i - j is the same counted from the sequence's start or from the first row), so the sequences are one
// long one in which query i sees keys from max(its sequence's first row, i - window) on.  A tile of queries may span sequences; nothing but the
// first visible key of each row tells them apart, and that grows with i.
//   score = cap tanh(q.k / sqrt(hd) / cap) - slope_h (i - j);  out = softmax(score) . V     (flash_stu/modules/attention.py:72-101)
#include "attention_packed.cuh"

int* device_status_word();   // gemm_tc.cu

namespace {

constexpr int QT = 32, KT = 32;

// bf16 whose rows the tensor copies cannot take (off the 16-byte grid, heads of no multiple of 8), in fp32 on the CUDA cores: a CTA per 32 queries of one head, eight warps of four queries; keys and values of 32
// positions in shared memory as fp32 (keys transposed), lane = key for the scores, lane = dimension for the weighted values.
// Bound by shared memory: both operands of every multiply-add come from there.  16 prompts of 14140 tokens, 12 heads of 128, window 1024: 6.5 ms (8 TFLOP/s).
__global__ void __launch_bounds__(256) packed_attend_kernel(const bf16* __restrict__ qkv, long long row_stride, const int* __restrict__ cu, int S,
                                                            const float* __restrict__ slopes, bf16* __restrict__ out, long long out_stride, int rows, int H,
                                                            int Hk, int hd, int window, float scale, float softcap) {
  extern __shared__ __align__(16) float smem[];
  __shared__ int first[QT];
  const int hdp = (hd + 31) & ~31, dpl = hdp >> 5;
  float (*Qs)[QT] = reinterpret_cast<float (*)[QT]>(smem);                              // [dim][query]
  float (*Kt)[KT + 1] = reinterpret_cast<float (*)[KT + 1]>(smem + hdp * QT);           // [dim][key]
  float* Vs = smem + hdp * QT + hdp * (KT + 1);                                         // [key][hdp]
  const int h = blockIdx.y, g = h / (H / Hk), q0 = blockIdx.x * QT, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < QT * hdp; e += 256) {
    const int qi = e / hdp, c = e % hdp, i = q0 + qi;
    Qs[c][qi] = i < rows && c < hd ? Elem<bf16>::to_f(qkv[i * row_stride + (long long)h * hd + c]) * scale : 0.f;
  }
  if (threadIdx.x < QT) first[threadIdx.x] = packed::first_key(cu, S, q0 + threadIdx.x, rows, window);
  __syncthreads();
  float m[4], l[4], acc[4][4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[u][e] = 0.f;
  }
  const float slope = slopes ? slopes[h] : 0.f;
  int j_lo = packed::NOBODY, j_hi = -1;   // keys that any row of the tile sees
  for (int qi = 0; qi < QT; qi++) {
    j_lo = min(j_lo, first[qi]);
    if (first[qi] != packed::NOBODY) j_hi = q0 + qi;
  }
  for (int jt = j_lo; jt <= j_hi; jt += KT) {
    __syncthreads();
    for (int e = threadIdx.x; e < KT * hdp; e += 256) {
      const int kj = e / hdp, c = e % hdp, j = jt + kj;
      const bool ok = j <= j_hi && c < hd;
      const bf16* at = qkv + j * row_stride + (long long)(H + g) * hd + c;
      Kt[c][kj] = ok ? Elem<bf16>::to_f(*at) : 0.f;
      Vs[kj * hdp + c] = ok ? Elem<bf16>::to_f(at[(long long)Hk * hd]) : 0.f;
    }
    __syncthreads();
    const int j = jt + lane;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < hd; c++) {
      const float kv = Kt[c][lane];
      const float4 q4 = *reinterpret_cast<const float4*>(&Qs[c][warp * 4]);
      s[0] = fmaf(q4.x, kv, s[0]);
      s[1] = fmaf(q4.y, kv, s[1]);
      s[2] = fmaf(q4.z, kv, s[2]);
      s[3] = fmaf(q4.w, kv, s[3]);
    }
    float pr[4];
    bool seen[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = q0 + warp * 4 + u;
      seen[u] = j >= first[warp * 4 + u] && j <= i;
      float sc = s[u];
      if (softcap > 0.f) sc = softcap * tanhf(sc / softcap);
      sc = seen[u] ? sc - slope * (float)(i - j) : -INFINITY;
      const float top = fmaxf(m[u], warp_max(sc)), corr = top == -INFINITY ? 1.f : __expf(m[u] - top);
      pr[u] = sc == -INFINITY ? 0.f : __expf(sc - top);   // (what is not seen, and what is, with no weight: there may be no maximum yet)
      l[u] = l[u] * corr + warp_sum(pr[u]);
      m[u] = top;
#pragma unroll
      for (int e = 0; e < 4; e++) acc[u][e] *= corr;
    }
    for (int kj = 0; kj < KT; kj++) {
      float pv[4];
#pragma unroll
      for (int u = 0; u < 4; u++) pv[u] = __shfl_sync(0xffffffffu, pr[u], kj);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (!__shfl_sync(0xffffffffu, (int)seen[u], kj)) continue;   // (a masked value may be NaN)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (e < dpl) acc[u][e] = fmaf(pv[u], Vs[kj * hdp + lane + 32 * e], acc[u][e]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int i = q0 + warp * 4 + u;
    if (first[warp * 4 + u] == packed::NOBODY) continue;
    const float inv = 1.f / l[u];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int c = lane + 32 * e;
      if (e < dpl && c < hd) out[i * out_stride + (long long)h * hd + c] = Elem<bf16>::from_f(acc[u][e] * inv);
    }
  }
}

}  // namespace

extern "C" int stu_swa_packed(const void* qkv, long long row_stride, const int* cu_seqlens, int S, const float* slopes, void* out, long long out_stride,
                              long long rows, int H, int Hk, int hd, int window, float softcap, int* status, int dtype, void* stream) {
  if (!qkv || !cu_seqlens || !out) return STU_ERR_NULL;
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (S <= 0 || rows <= 0 || rows > 0x7fffff00ll || Hk <= 0 || H < Hk || H % Hk || H > 65535 || hd <= 0 ||
      row_stride < (long long)(H + 2 * Hk) * hd || out_stride < (long long)H * hd)
    return STU_ERR_SHAPE;
  if (hd > 128) return STU_ERR_UNSUPPORTED;
  if (!status) status = device_status_word();
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == STU_BF16 && hd % 8 == 0 && aligned16(qkv) && row_stride % 8 == 0 && aligned16(out) && out_stride % 8 == 0)
    return launch_packed_umma(qkv, row_stride, cu_seqlens, S, slopes, out, out_stride, (int)rows, H, Hk, hd, window, softcap, status, st);
  if (dtype == STU_F32) return launch_packed_f32(qkv, row_stride, cu_seqlens, S, slopes, out, out_stride, (int)rows, H, Hk, hd, window, softcap, st);
  const float scale = 1.0f / sqrtf((float)hd);
  const dim3 grid((unsigned)((rows + QT - 1) / QT), H);
  const int hdp = (hd + 31) & ~31;
  const size_t smem = (size_t)(hdp * QT + hdp * (KT + 1) + KT * hdp) * sizeof(float);
  static SmemLimit limit;
  const cudaError_t e = allow_smem((const void*)packed_attend_kernel, 64 * 1024, limit);
  if (e != cudaSuccess) return (int)e;
  packed_attend_kernel<<<grid, 256, smem, st>>>((const bf16*)qkv, row_stride, cu_seqlens, S, slopes, (bf16*)out, out_stride, (int)rows, H, Hk, hd, window,
                                                scale, softcap);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

// Products of two e4m3 operands with a scale for each 128 of a row (fp8.cuh): y = x W^T for few rows of x, the weights streamed once; and
// the entry point of all of them.
//
// A warp multiplies 16 features by 8 NG tokens with mma.sync (m16n8k32, fp32 sums): a block of 128 columns at a time, whose sum it scales by
// the two powers of two and adds up, so a block's sum is a chain of 4.  A lane takes 32 consecutive bytes of its rows of a block: the order of
// the columns inside a block is free as long as both operands have it, so whole lines are loaded and no fragment is shuffled.
// 16 warps are groups of 16 features x slices of K; slices meet in shared memory.  Weights come through a ring of asynchronous
// copies in which every lane reads what it copied itself (no barrier).  What bounds it: HBM, the weights once; before, latency.
#include <cooperative_groups.h>

#include "fp8.cuh"
#include "fp8_gemm.cuh"

namespace cg = cooperative_groups;

int device_sm_count();   // gemm_tc.cu

namespace {

constexpr int WARPS = 16, STAGES = 4;
constexpr int RING_BYTES = WARPS * 32 * 64 * STAGES;   // a lane: 2 rows x 32 bytes per stage

struct Operand {   // 8-bit rows
  const unsigned char *q, *scales;
};

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// gt groups of 16 features per CTA (DUAL: the first half of the gate's, the second of the up's), WARPS / gt slices of K.  DUAL: the CTAs of a
// cluster have the 128 features of one block of h and settle its scale.
template <int NG, bool DUAL>
__global__ void __launch_bounds__(WARPS * 32, 1)
    fp8_stream_kernel(Operand x, Operand w, Operand w2, const bf16* resid, long long ldr, bf16* y, long long ldy, unsigned char* hq,
                      unsigned char* hs, int M, int N, int K, int gt, int overlap) {
  constexpr int MT = 8 * NG, PITCH = 20;   // (16 features and 4 of padding: rows of tokens start in other banks)
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ uint32_t s_amax[MT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int slices = WARPS / gt, group = warp % gt, slice = warp / gt;
  const int F = (DUAL ? gt / 2 : gt) * 16, f0 = blockIdx.x * F, m0 = blockIdx.y * MT;
  const int nkb = fp8::blocks_of(K), groups = fp8::groups_of(K), pitch = nkb * fp8::BLOCK;
  // (when the next kernel may start: epilogue.cuh, PdlTrigger)
  if (overlap && !DUAL) pdl_trigger();
  if (!overlap) {
    pdl_wait();
    pdl_trigger();
  }

  const bool up = DUAL && group >= gt / 2;
  const Operand& wm = up ? w2 : w;
  const int n = f0 + (up ? group - gt / 2 : group) * 16 + g;
  const int n_lo = min(n, N - 1), n_hi = min(n + 8, N - 1);   // (rows past the last are computed from it and left out)
  const unsigned char *w_lo = wm.q + (size_t)n_lo * pitch + q * 32, *w_hi = wm.q + (size_t)n_hi * pitch + q * 32;
  const unsigned char *ws_lo = wm.scales + fp8::scale_word(n_lo, 0, groups), *ws_hi = wm.scales + fp8::scale_word(n_hi, 0, groups);
  const int iters = slice < nkb ? (nkb - slice + slices - 1) / slices : 0;
  uint4* mine = reinterpret_cast<uint4*>(ring) + threadIdx.x;   // [stage][4][threads]
  auto issue = [&](int it) {
    if (it < iters) {
      const size_t off = (size_t)(slice + it * slices) * fp8::BLOCK;
      uint4* to = mine + (it % STAGES) * 4 * WARPS * 32;
      copy16(to, w_lo + off);
      copy16(to + WARPS * 32, w_lo + off + 16);
      copy16(to + 2 * WARPS * 32, w_hi + off);
      copy16(to + 3 * WARPS * 32, w_hi + off + 16);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) issue(i);
  if (overlap) pdl_wait();   // the weights alone were asked for ahead of it
  if (overlap && DUAL) pdl_trigger();

  const unsigned char* xr[NG];
  const unsigned char *xs0[NG], *xs1[NG];
#pragma unroll
  for (int i = 0; i < NG; i++) {
    xr[i] = x.q + (size_t)min(m0 + 8 * i + g, M - 1) * pitch + q * 32;
    xs0[i] = x.scales + fp8::scale_word(min(m0 + 8 * i + 2 * q, M - 1), 0, groups);
    xs1[i] = x.scales + fp8::scale_word(min(m0 + 8 * i + 2 * q + 1, M - 1), 0, groups);
  }
  float acc[NG][4];
#pragma unroll
  for (int i = 0; i < NG; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
  for (int it = 0; it < iters; it++) {
    const int kb = slice + it * slices;
    const size_t so = (size_t)(kb >> 2) * fp8::PIECE + (kb & 3);
    uint4 xv[NG][2];
    float sx0[NG], sx1[NG];
#pragma unroll
    for (int i = 0; i < NG; i++) {
      xv[i][0] = *reinterpret_cast<const uint4*>(xr[i] + (size_t)kb * fp8::BLOCK);
      xv[i][1] = *reinterpret_cast<const uint4*>(xr[i] + (size_t)kb * fp8::BLOCK + 16);
      sx0[i] = fp8::scale_of(xs0[i][so]);
      sx1[i] = fp8::scale_of(xs1[i][so]);
    }
    const float sw_lo = fp8::scale_of(ws_lo[so]), sw_hi = fp8::scale_of(ws_hi[so]);
    issue(it + STAGES - 1);   // into the stage that the turn before has read
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    const uint4* from = mine + (it % STAGES) * 4 * WARPS * 32;
    const uint4 a = from[0], b = from[WARPS * 32], c = from[2 * WARPS * 32], d = from[3 * WARPS * 32];
#pragma unroll
    for (int i = 0; i < NG; i++) {
      float t[4] = {0.f, 0.f, 0.f, 0.f};
      mma_e4m3(t, a.x, c.x, a.y, c.y, xv[i][0].x, xv[i][0].y);
      mma_e4m3(t, a.z, c.z, a.w, c.w, xv[i][0].z, xv[i][0].w);
      mma_e4m3(t, b.x, d.x, b.y, d.y, xv[i][1].x, xv[i][1].y);
      mma_e4m3(t, b.z, d.z, b.w, d.w, xv[i][1].z, xv[i][1].w);
      acc[i][0] = fmaf(t[0], sw_lo * sx0[i], acc[i][0]);
      acc[i][1] = fmaf(t[1], sw_lo * sx1[i], acc[i][1]);
      acc[i][2] = fmaf(t[2], sw_hi * sx0[i], acc[i][2]);
      acc[i][3] = fmaf(t[3], sw_hi * sx1[i], acc[i][3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the ring is read: the slices' sums take its place, [warp][token][feature]
  float* red = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int i = 0; i < NG; i++) {
    float* to = red + (warp * MT + 8 * i + 2 * q) * PITCH + g;
    to[0] = acc[i][0];
    to[PITCH] = acc[i][1];
    to[8] = acc[i][2];
    to[PITCH + 8] = acc[i][3];
  }
  if (threadIdx.x < MT) s_amax[threadIdx.x] = 0;
  __syncthreads();
  auto total = [&](int grp, int t, int f) {
    float v = 0.f;
    for (int s = 0; s < slices; s++) v += red[((s * gt + grp) * MT + t) * PITCH + f];
    return v;
  };
  if constexpr (!DUAL) {
    for (int i = threadIdx.x; i < F * MT; i += WARPS * 32) {
      const int t = i / F, f = i - t * F, m = m0 + t;
      if (m < M && f0 + f < N) {
        float v = total(f >> 4, t, f & 15);
        if (resid) v = __bfloat162float(resid[(size_t)m * ldr + f0 + f]) + round_to<bf16>(v);
        y[(size_t)m * ldy + f0 + f] = __float2bfloat16_rn(v);
      }
    }
  } else {
    float* h = red + WARPS * MT * PITCH;   // [token][F]
    for (int i = threadIdx.x; i < F * MT; i += WARPS * 32) {
      const int t = i / F, f = i - t * F;
      float v = 0.f;
      if (f0 + f < N) v = fp8::gelu(total(f >> 4, t, f & 15)) * total((f >> 4) + gt / 2, t, f & 15);
      v = fp8::nan_unless_finite(v);
      h[i] = v;
      atomicMax(&s_amax[t], v == v ? fp8::magnitude(v) : 0u);   // (a maximum: the order does not tell)
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int parts = cluster.num_blocks();
    const int hb = f0 / fp8::BLOCK, hblocks = fp8::blocks_of(N), hgroups = fp8::groups_of(N);
    const int words = F / 4;
    for (int i = threadIdx.x; i < words * MT; i += WARPS * 32) {
      const int t = i / words, f = (i - t * words) * 4, m = m0 + t;
      if (m >= M) continue;
      uint32_t a = 0;
      for (int r = 0; r < parts; r++) a = max(a, *cluster.map_shared_rank(&s_amax[t], r));
      const uint32_t b = fp8::scale_byte(a);
      const float inv = fp8::inverse_scale(b);
      const float* v = h + t * F + f;
      *reinterpret_cast<uint32_t*>(hq + (size_t)m * hblocks * fp8::BLOCK + f0 + f) = fp8::pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      if (f == 0 && f0 % fp8::BLOCK == 0) hs[fp8::scale_word(m, hb >> 2, hgroups) + (hb & 3)] = (unsigned char)b;
    }
    // byte 0 for the rows that fill up the last 128 and for the blocks that fill up the last four
    if (f0 % fp8::BLOCK == 0) {
      const int last = hb == hblocks - 1 ? hgroups * 4 : hb + 1;
      const bool bottom = blockIdx.y == gridDim.y - 1;
      const int end = bottom ? (M + 127) & ~127 : m0 + MT;
      for (int m = m0 + threadIdx.x; m < end; m += WARPS * 32)
        for (int kb = m < M ? hb + 1 : hb; kb < last; kb++) hs[fp8::scale_word(m, kb >> 2, hgroups) + (kb & 3)] = 0;
    }
    cluster.sync();   // the others have read s_amax
  }
}

template <int NG, bool DUAL>
int launch_stream(const Operand& x, const Operand& w, const Operand& w2, const bf16* resid, long long ldr, bf16* y, long long ldy,
                  unsigned char* hq, unsigned char* hs, int M, int N, int K, int overlap, cudaStream_t st) {
  static SmemLimit limit;
  constexpr int MT = 8 * NG;
  const size_t sums = (size_t)WARPS * MT * 20 * sizeof(float) + (DUAL ? 128 * MT * sizeof(float) : 0);
  const size_t smem = sums > (size_t)RING_BYTES ? sums : (size_t)RING_BYTES;
  cudaError_t e = allow_smem((const void*)fp8_stream_kernel<NG, DUAL>, smem, limit);
  if (e != cudaSuccess) return (int)e;
  // features per CTA: the most that still give every SM a CTA
  const int sms = device_sm_count(), tiles_m = (M + MT - 1) / MT;
  int F = 128;
  const auto ctas = [&](int f) { return DUAL ? (long long)fp8::blocks_of(N) * (128 / f) : (N + f - 1) / f; };
  while (F > 16 && ctas(F) * tiles_m < sms) F /= 2;
  const int gt = (DUAL ? 2 : 1) * F / 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas(F), (unsigned)tiles_m);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (DUAL && F < 128) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = 128 / F;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  if (pdl_enabled()) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  e = cudaLaunchKernelEx(&cfg, fp8_stream_kernel<NG, DUAL>, x, w, w2, resid, ldr, y, ldy, hq, hs, M, N, K, gt, overlap);
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

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
  if (M == 0) return STU_OK;
  cudaStream_t st = (cudaStream_t)stream;
  const Operand a{(const unsigned char*)x, (const unsigned char*)x_scales}, w{(const unsigned char*)W, (const unsigned char*)W_scales},
      w2{(const unsigned char*)W2, (const unsigned char*)W2_scales};
  const int overlap = (flags & STU_FLAG_OVERLAP) != 0;
#define STU_STREAM(NG_, DUAL_)                                                                                                       \
  launch_stream<NG_, DUAL_>(a, w, w2, (const bf16*)resid, resid_row_stride, DUAL_ ? nullptr : (bf16*)y, y_row_stride,                \
                            DUAL_ ? (unsigned char*)y : nullptr, (unsigned char*)y_scales, M, N, K, overlap, st)
  if (M > 32)
    return fp8_gemm({a.q, a.scales, w.q, w.scales, w2.q, w2.scales, (const bf16*)resid, resid_row_stride, W2 ? nullptr : (bf16*)y, y_row_stride,
                     W2 ? (unsigned char*)y : nullptr, (unsigned char*)y_scales, M, N, K}, st);
  if (M <= 8) return W2 ? STU_STREAM(1, true) : STU_STREAM(1, false);
  if (M <= 16) return W2 ? STU_STREAM(2, true) : STU_STREAM(2, false);
  return W2 ? STU_STREAM(4, true) : STU_STREAM(4, false);
#undef STU_STREAM
}

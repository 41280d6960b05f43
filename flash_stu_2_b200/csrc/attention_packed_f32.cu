// Attention of packed prompts in fp32 on mma.sync (attention_packed.cu says what is computed): heads of up to 128 dimensions, padded with zeros to 64 or 128.
//
// A value is the sum of three bf16 (its leading bits, what these leave, and what is left then: 24 bits), and a product of two values six of theirs (all but the
// three smallest, 2^-24 of it), summed in fp32: as exact as fp32 products.  A CTA is 64 queries of one head in four warps of 16; per tile of 32 keys
//   S = Q K^T   the queries' three parts stay in shared memory, as do the keys' and values' of a tile, which are cut up as they come in
//   softmax     in registers, against the running maximum (exp2 domain, tanh of the library for the cap)
//   O += P V    the weights' three parts are made from the accumulators where they lie
// A product takes all values of a tile, masked ones with a weight of 0: those whose leading part would not be finite (infinities, NaN, and what bf16 rounds to infinity,
// from 2^128 - 2^119 on) are zeros there, and are added for the rows that see them, where a tile has any.  Queries and keys as large have their scores from fp32
// products on the CUDA cores, as their parts' products would be NaN.  (NaN itself is NaN in its parts' products too.)
// The keys' first tile is the first that any row sees.  Six products instead of one on the older tensor path (1024 multiply-adds a clock and SM) leave 90 TFLOP/s; the CUDA cores'
// 74 need both operands of every product from shared memory or registers.  Shared memory: 120 KB for heads of 128 (one CTA per SM), 60 for heads of 64.
// Measured: 128 + 700 tokens, 8 heads of 64, 53 us where there are only 104 CTAs: a warp per scheduler, whose products (24 % of the pipe), cutting up and softmax follow one another.  On the CUDA
// cores the same took 379 us.
#include "attention_packed.cuh"

namespace {

constexpr int BM = 64, BN = 32;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float MOST = 0x1.ffp127f;   // what is smaller rounds to a finite bf16

template <int HD> struct Smem {
  static constexpr int PITCH = HD + 8;                          // bf16 values between rows: eight rows' 16 bytes lie in different banks
  static constexpr int Q_PART = BM * PITCH, KV_PART = BN * PITCH;
  static constexpr int BYTES = 3 * (Q_PART + 2 * KV_PART) * 2;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The three parts of two values, each pair in one register.  (Not finite: the leading part alone.)
__device__ __forceinline__ void parts_of(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    p[i] = *reinterpret_cast<const uint32_t*>(&h);
    x -= __uint_as_float(p[i] << 16);
    y -= __uint_as_float(p[i] & 0xffff0000u);
    if (i == 0) {   // infinity less itself is none
      x = x == x ? x : 0.f;
      y = y == y ? y : 0.f;
    }
  }
}
__device__ __forceinline__ float exp2_fast(float x) {   // relative error 2^-22; 0 for -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int HD, bool VEC>
__global__ void __launch_bounds__(128) packed_f32_kernel(const float* __restrict__ qkv, long long row_stride, const int* __restrict__ cu, int S,
                                                         const float* __restrict__ slopes, float* __restrict__ out, long long out_stride, int rows, int H,
                                                         int Hk, int hd, int window, float scale, float softcap) {
  typedef Smem<HD> L;
  constexpr int P = L::PITCH;
  extern __shared__ __align__(16) bf16 smem[];
  bf16 *Qs = smem, *Ks = Qs + 3 * L::Q_PART, *Vs = Ks + 3 * L::KV_PART;   // [part][row][PITCH]
  __shared__ int s_first[BM], s_odd[2];   // whether a tile has values past MOST (this and the next tile's)
  const int h = blockIdx.y, g = h / (H / Hk), q0 = (int)(gridDim.x - 1 - blockIdx.x) * BM;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gr = lane >> 2, c = lane & 3;
  // 4 values of a row of qkv, zeros past the head and past the rows
  auto four = [&](int row, int end, const float* column, int d, float (&x)[4]) {
    if (VEC && row < end && d + 4 <= hd) {
      load_vec(column + row * row_stride + d, x);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = row < end && d + e < hd ? column[row * row_stride + d + e] : 0.f;
    }
  };
  auto put = [&](bf16* at, int part, const float (&x)[4]) {
    uint32_t a[3], b[3];
    parts_of(x[0], x[1], a);
    parts_of(x[2], x[3], b);
#pragma unroll
    for (int i = 0; i < 3; i++) *reinterpret_cast<uint2*>(at + i * part) = make_uint2(a[i], b[i]);
  };
  if (threadIdx.x < BM) s_first[threadIdx.x] = packed::first_key(cu, S, q0 + threadIdx.x, rows, window);
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  bool big = false;
  for (int e = threadIdx.x; e < BM * (HD / 4); e += 128) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
    float x[4];
    four(q0 + r, rows, qkv + (long long)h * hd, d, x);
#pragma unroll
    for (int u = 0; u < 4; u++) big |= fabsf(x[u]) >= MOST;
    put(Qs + r * P + d, L::Q_PART, x);
  }
  const bool big_queries = __syncthreads_or(big);
  int j_lo = packed::NOBODY, j_hi = -1;   // keys that any row of the tile sees
  for (int r = 0; r < BM; r++) {
    j_lo = min(j_lo, s_first[r]);
    if (s_first[r] != packed::NOBODY) j_hi = q0 + r;
  }
  const int r0 = warp * 16 + gr;         // this lane's rows: r0 and r0 + 8
  const int first[2] = {s_first[r0], s_first[r0 + 8]};
  int w_lo = packed::NOBODY, w_hi = -1;  // the same of the warp's rows
  for (int r = warp * 16; r < warp * 16 + 16; r++) {
    w_lo = min(w_lo, s_first[r]);
    if (s_first[r] != packed::NOBODY) w_hi = q0 + r;
  }
  const float c2 = slopes ? slopes[h] * LOG2E : 0.f, k0 = softcap > 0.f ? scale / softcap : scale * LOG2E, k1 = softcap * LOG2E;
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < HD / 8; n++)
#pragma unroll
    for (int e = 0; e < 4; e++) o[n][e] = 0.f;

  constexpr int MINE = 2 * BN * (HD / 4) / 128;   // fours of a tile that this thread brings: the next tile's are under way while this one is multiplied
  float coming[MINE][4];
  auto fetch = [&](int jt) {
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      const int e = threadIdx.x + 128 * i, which = e / (BN * (HD / 4)), r = e / (HD / 4) % BN, d = e % (HD / 4) * 4;
      four(jt + r, j_hi + 1, qkv + (long long)(H + which * Hk + g) * hd, d, coming[i]);
    }
  };
  if (j_lo <= j_hi) fetch(j_lo);
  for (int jt = j_lo, turn = 0; jt <= j_hi; jt += BN, turn ^= 1) {
    __syncthreads();   // the tile before has been read
    big = false;
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      const int e = threadIdx.x + 128 * i, which = e / (BN * (HD / 4)), r = e / (HD / 4) % BN, d = e % (HD / 4) * 4;
      if (which) {
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (!(fabsf(coming[i][u]) < MOST)) {
            coming[i][u] = 0.f;
            s_odd[turn] = 1;
          }
      } else {
#pragma unroll
        for (int u = 0; u < 4; u++) big |= fabsf(coming[i][u]) >= MOST;
      }
      put((which ? Vs : Ks) + r * P + d, L::KV_PART, coming[i]);
    }
    const bool big_scores = __syncthreads_or(big) || big_queries;   // (the same for the whole CTA)
    if (threadIdx.x == 0) s_odd[turn ^ 1] = 0;   // (written again behind the next barrier)
    if (jt + BN <= j_hi) fetch(jt + BN);
    if (jt > w_hi || jt + BN <= w_lo) continue;   // (nothing here for this warp's rows)
    float s[BN / 8][4];
#pragma unroll
    for (int n = 0; n < BN / 8; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[n][e] = 0.f;
#pragma unroll 1
    for (int ks = 0; ks < HD / 16; ks++) {
      uint32_t q[3][4];
#pragma unroll
      for (int i = 0; i < 3; i++)
        ldmatrix_x4(q[i], Qs + i * L::Q_PART + (warp * 16 + (lane & 15)) * P + ks * 16 + (lane >> 4) * 8);
      uint32_t k[BN / 16][3][4];   // 16 keys: two tiles of 8
#pragma unroll
      for (int np = 0; np < BN / 16; np++)
#pragma unroll
        for (int i = 0; i < 3; i++)
          ldmatrix_x4(k[np][i], Ks + i * L::KV_PART + (np * 16 + (lane & 7) + 8 * (lane >> 4)) * P + ks * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll
      for (int t = 0; t < 6; t++) {   // the small products first; a product's sum is there 20 clocks later: four of them take turns
        constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int np = 0; np < BN / 16; np++) {
          mma(s[2 * np], q[A[t]], k[np][B[t]][0], k[np][B[t]][1]);
          mma(s[2 * np + 1], q[A[t]], k[np][B[t]][2], k[np][B[t]][3]);
        }
      }
    }
    if (big_scores) {
#pragma unroll
      for (int n = 0; n < BN / 8; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = jt + n * 8 + 2 * c + (e & 1), i = q0 + r0 + 8 * (e >> 1);
          if (j < first[e >> 1] || j > i) continue;
          const float *q = qkv + i * row_stride + (long long)h * hd, *k = qkv + j * row_stride + (long long)(H + g) * hd;
          float x = 0.f;
#pragma unroll 1
          for (int d = 0; d < hd; d++) x = fmaf(q[d], k[d], x);
          s[n][e] = x;
        }
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < BN / 8; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int j = jt + n * 8 + 2 * c + (e & 1), i = q0 + r0 + 8 * (e >> 1);
        float x = s[n][e] * k0;
        if (softcap > 0.f) x = tanhf(x) * k1;
        x = fmaf(-c2, (float)(i - j), x);
        s[n][e] = j >= first[e >> 1] && j <= i ? x : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; r++) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float ref = top[r] == -INFINITY ? 0.f : top[r], corr = exp2_fast(m[r] - ref);   // (a row without a key yet: all of it stays 0)
      m[r] = top[r];
      l[r] *= corr;
#pragma unroll
      for (int n = 0; n < HD / 8; n++) {
        o[n][2 * r] *= corr;
        o[n][2 * r + 1] *= corr;
      }
#pragma unroll
      for (int n = 0; n < BN / 8; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) l[r] += s[n][2 * r + e] = exp2_fast(s[n][2 * r + e] - ref);
    }
#pragma unroll
    for (int kk = 0; kk < BN / 16; kk++) {
      uint32_t w[3][4];   // the weights' parts: the accumulators of two tiles of keys are an operand of 16
#pragma unroll
      for (int e = 0; e < 4; e++) {
        uint32_t p[3];
        parts_of(s[2 * kk + (e >> 1)][2 * (e & 1)], s[2 * kk + (e >> 1)][2 * (e & 1) + 1], p);
#pragma unroll
        for (int i = 0; i < 3; i++) w[i][e] = p[i];
      }
#pragma unroll
      for (int np = 0; np < HD / 16; np += 2) {
        uint32_t v[2][3][4];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int i = 0; i < 3; i++)
            ldmatrix_x4_trans(v[u][i], Vs + i * L::KV_PART + (kk * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * P + (np + u) * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int t = 0; t < 6; t++) {
          constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
          for (int u = 0; u < 2; u++) {
            mma(o[2 * (np + u)], w[A[t]], v[u][B[t]][0], v[u][B[t]][1]);
            mma(o[2 * (np + u) + 1], w[A[t]], v[u][B[t]][2], v[u][B[t]][3]);
          }
        }
      }
    }
    if (s_odd[turn]) {   // (the same for the whole CTA)
#pragma unroll
      for (int n = 0; n < BN / 8; n++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int j = jt + n * 8 + k;
          const float w0 = __shfl_sync(0xffffffffu, s[n][k & 1], (lane & ~3) + (k >> 1)), w1 = __shfl_sync(0xffffffffu, s[n][2 + (k & 1)], (lane & ~3) + (k >> 1));
          if (j > j_hi) continue;
          const float* v = qkv + j * row_stride + (long long)(H + Hk + g) * hd;
#pragma unroll
          for (int d8 = 0; d8 < HD / 8; d8++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int d = d8 * 8 + 2 * c + e;
              const float x = d < hd ? v[d] : 0.f;
              if (!(fabsf(x) < MOST)) {
                if (j >= first[0] && j <= q0 + r0) o[d8][e] = fmaf(w0, x, o[d8][e]);
                if (j >= first[1] && j <= q0 + r0 + 8) o[d8][2 + e] = fmaf(w1, x, o[d8][2 + e]);
              }
            }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; r++) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int i = q0 + r0 + 8 * r;
    if (first[r] == packed::NOBODY) continue;
    const float inv = 1.f / l[r];
    float* dst = out + i * out_stride + (long long)h * hd;
#pragma unroll
    for (int n = 0; n < HD / 8; n++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (n * 8 + 2 * c + e < hd) dst[n * 8 + 2 * c + e] = o[n][2 * r + e] * inv;
  }
}

template <int HD, bool VEC>
int launch(const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows, int H, int Hk, int hd,
           int window, float softcap, cudaStream_t st) {
  static SmemLimit limit;
  const cudaError_t e = allow_smem((const void*)packed_f32_kernel<HD, VEC>, Smem<HD>::BYTES, limit);
  if (e != cudaSuccess) return (int)e;
  packed_f32_kernel<HD, VEC><<<dim3((unsigned)((rows + BM - 1) / BM), H), 128, Smem<HD>::BYTES, st>>>(
      (const float*)qkv, row_stride, cu, S, slopes, (float*)out, out_stride, rows, H, Hk, hd, window, 1.0f / sqrtf((float)hd), softcap);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

int launch_packed_f32(const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows, int H,
                      int Hk, int hd, int window, float softcap, cudaStream_t st) {
  const bool vec = aligned16(qkv) && row_stride % 4 == 0 && hd % 4 == 0;
  auto go = [&](auto f) { return f(qkv, row_stride, cu, S, slopes, out, out_stride, rows, H, Hk, hd, window, softcap, st); };
  if (hd <= 64) return vec ? go(launch<64, true>) : go(launch<64, false>);
  return vec ? go(launch<128, true>) : go(launch<128, false>);
}

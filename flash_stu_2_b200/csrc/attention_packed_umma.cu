// Attention of packed prompts on the 5th-generation tensor cores: bf16, heads of a multiple of 8 dimensions up to 128 (attention_packed.cu says what
// is computed, and how one tile of queries may span sequences).
//
// One CTA = 256 rows of one head as two tiles of 128 queries, which take turns: while the softmax of one runs, the tensor core works for the other.  Key tiles of
// 128 rows, on multiples of 128, from the first key that any row sees to the diagonal; each tile of queries skips those that none of its rows sees.
//   S = Q K^T   tcgen05.mma, M = 128 queries, N = 128 keys; Q, K and V come by cp.async.bulk.tensor from qkv itself, seen as [rows][heads][hd] (what a
//               box has past hd is filled with zeros: a head of 96 is one of 128 with zeros behind it); S lands in tensor memory
//   softmax     four warps per tile, a row per thread: soft cap, ALiBi, mask, exponentials in the exp2 domain against a maximum that moves only
//               when the row's outgrows it by 2^8 (then the row of O in tensor memory is rescaled); P in bf16 goes back over S
//   O += P V    tcgen05.mma, P from tensor memory, V as it lies (rows of keys: the operand whose rows are the sum's index), accumulating in tensor memory
// The two tiles' S and O are the 512 columns that there are, so P has to take S's place; the next S of a tile is issued behind the product
// that reads its P, and a CTA's products run in the order of issue.
// Rounded weights against a maximum that lags: the largest are off by up to 2^-9, which against the row's own maximum would be exactly 1.  Heads of 64 are divided by the sum of the
// rounded ones, so that a row of one large weight is not off by that; it takes 5 % of the time, and heads of 128 are not (error against 64 bits of 16 prompts 2.2e-3, of which 1.6e-3
// is the output's rounding).
// With ALiBi the maximum is taken for what it will be at the row's end if the scores stay as they are.  Where they do not, all of a row's weights may be too small for fp32:
// the row is computed again, as below.
// Measured: 16384 tokens, 16 heads of 128 on 2, 1120 to 1150 us (0.96 to 0.98 PFLOP/s, the tensor pipe 58 % busy at 1.45 GHz, where the library's products keep it 87 % busy at 1.3); 16 prompts of
// 14140 tokens, 12 heads of 128, window 1024, cap and ALiBi, 141 us (380 TFLOP/s); 9311 tokens, 12 heads of 64, window 512, 73 us.  Bound by the softmax where there is a cap or a short window (2900
// clocks of a warp for a tile whose products take 1024), else by the chain from scores to the next scores.  Instead: key tiles of 64 1115 to 1240 us for the 16384 tokens, an issuer per tile of queries 1258.
// The tensor core adds 0 times what a masked key's value holds: where that is NaN or infinite, a row with a finite sum of weights has a result that is not, and is
// computed again on the CUDA cores over the keys that it sees.  (One key after the other by a warp, and a warp's rows in turn, which is slow where many rows of many keys meet one: an infinite value in the
// first row of 16384, 16 heads, no window, 0.98 s instead of 1.1 ms.  32 keys at a time, a lane per key, took 0.40 s, and the 16 prompts above 146 us instead of 141 by the registers that it holds.)
#include <cuda.h>

#include "attention_packed.cuh"
#include "tma.cuh"

namespace {

constexpr int BM = 128, BN = 128, STAGES = 4;
// Eight warps of softmax, the issuer, the producer, and two without work that make these a warpgroup, whose registers go to the softmax: 256 threads of
// 208 and 128 of 80 are less than the launch's 384 of 168.  (216 of them: more is spilled elsewhere, the 16 prompts take 148 us instead of 141.)
constexpr int THREADS = 384, REGS_SOFTMAX = 208, REGS_OTHERS = 80;
constexpr int STATUS_PACKED = 13;
constexpr float LOG2E = 1.4426950408889634f;
// tanh(y) = y (T0 + T1 y^2 + T2 y^4) for |y| <= 1/2: relative error 2.3e-5 (Chebyshev interpolation on [0, 1/4] in y^2)
constexpr float T0 = 0.999977239f, T1 = -0.331685329f, T2 = 0.115185198f;
// ... = y (T0_TINY + T1_TINY y^2) for |y| <= 1/5: 2.6e-5 (the least there is)
constexpr float T0_TINY = 0.999973796f, T1_TINY = -0.328076375f;
// How far a score may outgrow what scores are counted from (heads of 64, 9311 tokens, with 2 instead of 8: error against 64 bits 2.02e-3 instead of 2.05e-3, 75 us instead of 73); the least sum of weights (what it leaves out is below 2^-126 a key)
constexpr float LAG = 8.f, LEAST = 0x1p-90f;

// Of 8 pairs of weights those that the FMA pipe makes (16384 tokens: 1140 us with 1 of them, 1070 to 1115 with 2, 1144 with 3, 1236 with 4); pairs whose arithmetic is interleaved
constexpr int POLY_OF_8 = 2, ILP = 8;

template <int HD> struct Smem {
  static constexpr int KB = HD / 64;                   // blocks of 64 dimensions
  static constexpr int TILE = KB * 16384;              // 128 rows
  static constexpr int KV = 2 * TILE;                  // behind the two tiles of queries
  static constexpr int BYTES = KV + STAGES * TILE + 1024;
};

struct Ctl {
  uint64_t q_full[2], s_full[2], p_full[2][2], pv_done[2], kv_full[STAGES], kv_empty[STAGES];
  uint32_t tmem_slot;
  int abort_flag, first[2 * BM];
};

// K-major rows of 64 values (128-byte swizzle), groups of 8 rows 1 KB apart
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// rows are the sum's index: 64 columns a row, the next 64 columns a whole block of 128 rows further
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(16384 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__host__ __device__ constexpr uint32_t idesc(int n, bool b_rows_k) {   // D fp32, A and B bf16, M = 128
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_rows_k ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tma::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// Loads have landed: nothing that reads r may move ahead of this.
template <int N> __device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// pairs of fp32 values in 64-bit registers
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float lo, float hi) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ f32x2 pair_of(uint32_t lo, uint32_t hi) { return (f32x2)hi << 32 | lo; }
__device__ __forceinline__ void split(f32x2 v, uint32_t& lo, uint32_t& hi) { asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v)); }
__device__ __forceinline__ void split(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float exp2_hw(float x) {   // 0 for -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where one is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x on the FMA pipe, beside the special-function unit, which takes 8 clocks of a warp for every exponential: x = k + f with f in [-1/2, 1/2] (adding 1.5 2^23
// rounds to whole numbers), a polynomial of degree 3 in f (minimax among those that are 1 at 0, relative error 1.02e-4 against 2^-9 of the weights' rounding), k added
// to the exponent.  x is raised to -127, where f is 0, the polynomial 1 and the sum 0: what is masked has no weight at all (a small one in its place would be seen in the
// products: 2^-125 of the largest finite value is 8).  Between -127 and -126 the sum is below 2^-126, whatever it is.  NaN leaves as a number that bf16 rounds to
// infinity: its row's result is not finite, is computed again, and is NaN.
template <int N> __device__ __forceinline__ void exp2_poly(const uint32_t* x, f32x2* y) {
  f32x2 f[N], t[N], p[N];
  const f32x2 big = pair_of(12582912.f, 12582912.f), unbig = pair_of(-12582912.f, -12582912.f), minus = pair_of(-1.f, -1.f);
#pragma unroll
  for (int u = 0; u < N; u++) f[u] = pair_of(max_nan(__uint_as_float(x[2 * u]), -127.f), max_nan(__uint_as_float(x[2 * u + 1]), -127.f));
#pragma unroll
  for (int u = 0; u < N; u++) t[u] = add2(f[u], big);
#pragma unroll
  for (int u = 0; u < N; u++) p[u] = add2(t[u], unbig);
#pragma unroll
  for (int u = 0; u < N; u++) f[u] = fma2(p[u], minus, f[u]);
#pragma unroll
  for (int u = 0; u < N; u++) p[u] = fma2(f[u], pair_of(0.0550089329f, 0.0550089329f), pair_of(0.242210969f, 0.242210969f));
#pragma unroll
  for (int u = 0; u < N; u++) p[u] = fma2(f[u], p[u], pair_of(0.693282902f, 0.693282902f));
#pragma unroll
  for (int u = 0; u < N; u++) p[u] = fma2(f[u], p[u], pair_of(1.f, 1.f));
#pragma unroll
  for (int u = 0; u < N; u++) {
    uint32_t p0, p1, t0, t1;
    split(p[u], p0, p1);
    split(t[u], t0, t1);
    y[u] = pair_of(p0 + (t0 << 23), p1 + (t1 << 23));
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS)); }

// A bounded wait whose first look costs little: most of these barriers have completed by the time they are asked for (tma::warp_wait_bounded takes 115 clocks
// then, of the 1024 that a tile's two products take).
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, tma::mbar_try_wait(bar, parity))) return true;
  return tma::warp_wait_bounded(bar, parity, abort_flag);
}

// 128 scores s -> cap(s) + c2 (column) + bt, by the polynomial of degree 2 or 1 in s^2, eight pairs at a time
template <bool SMALL, bool ALIBI>
__device__ __forceinline__ void capped(uint32_t (&sr)[128], f32x2 cap0, f32x2 cap1, f32x2 cap2, f32x2 tiny0, f32x2 tiny1, f32x2 cc, f32x2 bt) {
  f32x2 add[ILP];
#pragma unroll
  for (int u = 0; u < ILP; u++) add[u] = ALIBI ? fma2(cc, pair_of((float)(2 * u), (float)(2 * u + 1)), bt) : bt;
  const f32x2 further = mul2(cc, pair_of(2.f * ILP, 2.f * ILP));
#pragma unroll
  for (int c0 = 0; c0 < 128; c0 += 2 * ILP) {
    f32x2 sv[ILP], sq[ILP], p[ILP];
#pragma unroll
    for (int u = 0; u < ILP; u++) sv[u] = pair_of(sr[c0 + 2 * u], sr[c0 + 2 * u + 1]);
#pragma unroll
    for (int u = 0; u < ILP; u++) sq[u] = mul2(sv[u], sv[u]);
#pragma unroll
    for (int u = 0; u < ILP; u++) p[u] = SMALL ? fma2(sq[u], cap2, cap1) : fma2(sq[u], tiny1, tiny0);
    if (SMALL) {
#pragma unroll
      for (int u = 0; u < ILP; u++) p[u] = fma2(sq[u], p[u], cap0);
    }
#pragma unroll
    for (int u = 0; u < ILP; u++) split(fma2(sv[u], p[u], add[u]), sr[c0 + 2 * u], sr[c0 + 2 * u + 1]);
    if (ALIBI && c0 + 2 * ILP < 128) {
#pragma unroll
      for (int u = 0; u < ILP; u++) add[u] = add2(add[u], further);
    }
  }
}

// Row i once more, by a warp, over the keys that it sees and no other.
__device__ void row_again(const bf16* __restrict__ qkv, long long row_stride, bf16* __restrict__ dst, int i, int first, int h, int g, int H, int Hk, int hd,
                          float slope, float scale, float softcap, int lane) {
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; e++) q[e] = lane + 32 * e < hd ? __bfloat162float(qkv[i * row_stride + (long long)h * hd + lane + 32 * e]) * scale : 0.f;
  for (int j = first; j <= i; j++) {
    const bf16 *k = qkv + j * row_stride + (long long)(H + g) * hd, *v = k + (long long)Hk * hd;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (lane + 32 * e < hd) s = fmaf(q[e], __bfloat162float(k[lane + 32 * e]), s);
    s = warp_sum(s);
    if (softcap > 0.f) s = softcap * tanhf(s / softcap);
    s -= slope * (float)(i - j);
    // (a score of minus infinity weighs nothing, the first ones too, behind which there is no maximum yet)
    const float top = fmaxf(m, s), corr = top == -INFINITY ? 1.f : __expf(m - top), p = s == -INFINITY ? 0.f : __expf(s - top);
    m = top;
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (lane + 32 * e < hd) o[e] = fmaf(p, __bfloat162float(v[lane + 32 * e]), o[e] * corr);
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (lane + 32 * e < hd) dst[lane + 32 * e] = __float2bfloat16_rn(o[e] / l);
}

template <int HD, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(THREADS, 1) packed_umma_kernel(const __grid_constant__ CUtensorMap map, const bf16* __restrict__ qkv, long long row_stride,
                                                             const int* __restrict__ cu, int S, const float* __restrict__ slopes, bf16* __restrict__ out,
                                                             long long out_stride, int rows, int H, int Hk, int hd, int window, float scale,
                                                             float softcap, int* status) {
  typedef Smem<HD> L;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Ctl ctl;
  volatile int* abort_flag = &ctl.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, g = h / (H / Hk);
  const int q0 = (int)(gridDim.x - 1 - blockIdx.x) * 2 * BM;   // (without a window the last rows see most: they go first)
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      tma::mbar_init(&ctl.q_full[i], 1);
      tma::mbar_init(&ctl.s_full[i], 1);
      tma::mbar_init(&ctl.p_full[i][0], 4);
      tma::mbar_init(&ctl.p_full[i][1], 4);
      tma::mbar_init(&ctl.pv_done[i], 1);
    }
    for (int s = 0; s < STAGES; s++) {
      tma::mbar_init(&ctl.kv_full[s], 1);
      tma::mbar_init(&ctl.kv_empty[s], 1);
    }
    ctl.abort_flag = 0;
    tma::fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tma::smem_u32(&ctl.tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // The sequences of the first and of the last row of the CTA (counted by all threads: one reading of cu, however many there are), and every row's first key
  const int row_lo = max(q0, cu[0]), row_hi = min(min(q0 + 2 * BM, rows), cu[S]) - 1;   // rows of sequences
  int below = 0, upto = 0;
  for (int s0 = 0; s0 < S; s0 += THREADS) {   // (block-uniform)
    const int at = s0 + threadIdx.x < S ? cu[s0 + threadIdx.x] : 0x7fffffff;
    below += __syncthreads_count(at <= row_lo);
    upto += __syncthreads_count(at <= row_hi);
  }
  if (warp == 9 && elect_one()) {   // the queries, while their keys are looked for
#pragma unroll
    for (int i = 0; i < 2; i++)
      if (max(row_lo, q0 + i * BM) <= min(row_hi, q0 + i * BM + BM - 1)) {   // (a tile that has rows of a sequence, and whose products wait for it)
        tma::mbar_expect_tx(&ctl.q_full[i], L::TILE);
#pragma unroll
        for (int kb = 0; kb < L::KB; kb++) tma::load_3d(smem + i * L::TILE + kb * 16384, &map, &ctl.q_full[i], kb * 64, h, q0 + i * BM);
      }
  }
  __syncwarp();
  const int seq_lo = max(below - 1, 0), seq_hi = max(upto, seq_lo + 1);
  if (threadIdx.x < 2 * BM) {
    const int i = q0 + threadIdx.x;
    ctl.first[threadIdx.x] = i >= row_lo && i <= row_hi ? packed::first_key_in(cu, seq_lo, seq_hi, i, window) : packed::NOBODY;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ctl.tmem_slot;
  // key tiles of the two tiles of queries: begin .. end - 1
  int begin[2], end[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int lo = max(row_lo, q0 + i * BM), hi = min(row_hi, q0 + i * BM + BM - 1);
    begin[i] = lo <= hi ? ctl.first[lo - q0] / BN : 0;
    end[i] = lo <= hi ? hi / BN + 1 : 0;
    begin[i] = min(begin[i], end[i]);
  }
  const int t_lo = end[0] == 0 ? begin[1] : end[1] == 0 ? begin[0] : min(begin[0], begin[1]), t_hi = max(end[0], end[1]);
  auto active = [&](int i, int t) { return t >= begin[i] && t < end[i]; };

  if (warp == 9) {
    // ------------------------------------------------------------------ producer
    give_registers();
    const bool leader = elect_one();
    auto load = [&](unsigned char* dst, uint64_t* bar, int head, int row) {
      if (leader) {
        tma::mbar_expect_tx(bar, L::TILE);
#pragma unroll
        for (int kb = 0; kb < L::KB; kb++) tma::load_3d(dst + kb * 16384, &map, bar, kb * 64, head, row);
      }
      __syncwarp();
    };
    bool ok = true;
    int n = 0;
    auto load_kv = [&](int head, int t) {
      const int s = n % STAGES;
      ok = ok && tma::warp_wait_bounded(&ctl.kv_empty[s], ((uint32_t)(n / STAGES) & 1u) ^ 1u, abort_flag);
      if (ok) load(smem + L::KV + s * L::TILE, &ctl.kv_full[s], head, t * BN);
      n++;
    };
    for (int t = t_lo; ok && t < t_hi; t++) {
      load_kv(H + g, t);
      load_kv(H + Hk + g, t);
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ MMA issuer
    give_registers();
    const bool leader = elect_one();
    const uint32_t base = tma::smem_u32(smem);
    bool ok = true;
    auto stage_of = [&](int n) { return base + L::KV + (uint32_t)(n % STAGES) * L::TILE; };
    int landed = 0;   // stages that have been waited for
    auto wait_kv = [&](int n) {
      for (; ok && landed <= n; landed++) ok = wait_for(&ctl.kv_full[landed % STAGES], (uint32_t)(landed / STAGES) & 1u, abort_flag);
      return ok;
    };
    for (int t = t_lo; ok && t <= t_hi; t++) {
      const int nk = 2 * (t - t_lo), nv = nk - 1;   // the stages of K of t and V of t - 1
      const uint64_t k = desc_k(stage_of(nk)), v = desc_mn(stage_of(nv + STAGES));
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const bool product = active(i, t - 1), scores = active(i, t);
        if (!wait_kv(scores ? nk : nv)) break;
        if (product) {
          const uint32_t n = (uint32_t)(t - 1 - begin[i]);
#pragma unroll
          for (int half = 0; half < 2; half++) {   // (the first 64 keys' weights come while the others' are made)
            ok = ok && wait_for(&ctl.p_full[i][half], n & 1u, abort_flag);
            if (!ok) break;
            fence_after();
            if (leader) {
#pragma unroll
              for (int kk = half * 4; kk < half * 4 + 4; kk++)
                umma_ts(tmem + 256 + i * HD, tmem + i * 128 + kk * 8, v + (uint64_t)(kk * (2048 >> 4)), idesc(HD, true), (n | kk) ? 1u : 0u);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (leader && !scores) umma_commit(&ctl.pv_done[i]);   // the tile's last
        }
        if (scores) {
          if (t == begin[i]) {
            ok = wait_for(&ctl.q_full[i], 0, abort_flag);
            if (!ok) break;
          }
          fence_after();
          if (leader) {
            const uint64_t q = desc_k(base + i * L::TILE);
#pragma unroll
            for (int kb = 0; kb < L::KB; kb++)
#pragma unroll
              for (int kk = 0; kk < 4; kk++)
                umma_ss(tmem + i * 128, q + kb * (16384 >> 4) + 2 * kk, k + kb * (16384 >> 4) + 2 * kk, idesc(BN, false), (kb | kk) ? 1u : 0u);
            umma_commit(&ctl.s_full[i]);   // (the products before are complete then, too)
          }
        }
        if (leader) {
          if (product && (i == 1 || !active(1, t - 1))) umma_commit(&ctl.kv_empty[(nv + STAGES) % STAGES]);
          if (scores && (i == 1 || !active(1, t))) umma_commit(&ctl.kv_empty[nk % STAGES]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 8) {
    // -------------------------------------------------------------------- softmax warps (a quarter of the lanes of tensor memory each)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int tile = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int i = q0 + tile * BM + row, first = ctl.first[tile * BM + row];
    const int last_first = max(row_lo, q0 + tile * BM) <= min(row_hi, q0 + tile * BM + BM - 1) ? ctl.first[min(row_hi, q0 + tile * BM + BM - 1) - q0] : 0;
    const bool whole = row_lo <= q0 + tile * BM && row_hi >= q0 + tile * BM + BM - 1;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tm_s = tmem + tile * 128 + lanes, tm_o = tmem + 256 + tile * HD + lanes;
    const float c2 = ALIBI ? slopes[h] * LOG2E : 0.f;
    const float k0 = CAP ? scale / softcap : 0.f, k1 = CAP ? softcap * LOG2E : scale * LOG2E;
    const float kk0 = k0 * k0;
    // tanh(s k0) k1 = s times a polynomial in s^2, while |s| is below most_tiny (degree 1) or most_small (degree 2)
    const f32x2 cap0 = pair_of(k0 * k1 * T0, k0 * k1 * T0), cap1 = pair_of(k0 * k1 * kk0 * T1, k0 * k1 * kk0 * T1),
                cap2 = pair_of(k0 * k1 * kk0 * kk0 * T2, k0 * k1 * kk0 * kk0 * T2), kp = pair_of(k1, k1), cc = pair_of(c2, c2);
    const f32x2 cap_tiny0 = pair_of(k0 * k1 * T0_TINY, k0 * k1 * T0_TINY), cap_tiny1 = pair_of(k0 * k1 * kk0 * T1_TINY, k0 * k1 * kk0 * T1_TINY);
    const float most_tiny = CAP ? 0.2f / k0 : 0.f, most_small = CAP ? 0.5f / k0 : 0.f;
    float ref = 0.f, l = 0.f;   // what scores are counted from: the row's maximum, or one that it has outgrown by less than LAG
    bool any_key = false, ok = true;
    const int nt = end[tile] - begin[tile];
    for (int n = 0; n < nt; n++) {
      const int jt = (begin[tile] + n) * BN;
      ok = wait_for(&ctl.s_full[tile], (uint32_t)n & 1u, abort_flag);
      if (!ok) break;
      fence_after();
      uint32_t sr[128];
#pragma unroll
      for (int c = 0; c < 4; c++) tmem_ld32(tm_s + c * 32, sr + c * 32);
      tmem_wait_ld(sr);
      const bool interior = whole && jt >= last_first && jt + BN - 1 <= q0 + tile * BM;   // all rows of the tile see all keys of this one
      uint32_t seen[4];
      uint32_t dead = 0, partly = 0;   // blocks of 32 keys that no row of the warp sees, and that some do not see all of
      if (!interior) {
        const int lo = max(first - jt, 0), hi = first == packed::NOBODY ? -1 : min(i - jt, BN - 1);
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const int a = max(lo - 32 * w, 0), b = min(hi - 32 * w, 31);
          seen[w] = a > b ? 0u : (0xffffffffu >> (31 - (b - a))) << a;
          dead |= __any_sync(0xffffffffu, seen[w] != 0u) ? 0u : 1u << w;
          partly |= __all_sync(0xffffffffu, seen[w] == 0xffffffffu) ? 0u : 1u << w;
        }
      }
      // scores in the exp2 domain, counted from ref: s k1 (or its cap) + c2 (j - i) - ref
      const float base_t = ALIBI ? fmaf(c2, (float)(jt - i), -ref) : -ref;
      const f32x2 bt = pair_of(base_t, base_t);
      if (CAP) {
        float most[4] = {0.f, 0.f, 0.f, 0.f};   // (a NaN score is not in it: every form carries it on)
#pragma unroll
        for (int c = 0; c < 128; c += 2) most[c >> 1 & 3] = max3(most[c >> 1 & 3], fabsf(__uint_as_float(sr[c])), fabsf(__uint_as_float(sr[c + 1])));
        const float biggest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        if (__all_sync(0xffffffffu, biggest < most_tiny)) capped<false, ALIBI>(sr, cap0, cap1, cap2, cap_tiny0, cap_tiny1, cc, bt);
        else capped<true, ALIBI>(sr, cap0, cap1, cap2, cap_tiny0, cap_tiny1, cc, bt);
        const bool large = !(biggest < most_small);
        if (__any_sync(0xffffffffu, large)) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint32_t raw[32];
            tmem_ld32(tm_s + q * 32, raw);
            tmem_wait_ld(raw);
#pragma unroll
            for (int c = 0; c < 32; c++) {
              float th;   // the hardware's: relative error 2^-11
              asm("tanh.approx.f32 %0, %1;" : "=f"(th) : "f"(__uint_as_float(raw[c]) * k0));
              if (large) sr[q * 32 + c] = __float_as_uint(fmaf(th, k1, ALIBI ? fmaf(c2, (float)(q * 32 + c), base_t) : base_t));
            }
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 128; c += 2)
          split(fma2(pair_of(sr[c], sr[c + 1]), kp, ALIBI ? fma2(cc, pair_of((float)c, (float)(c + 1)), bt) : bt), sr[c], sr[c + 1]);
      }
#pragma unroll
      for (int w = 0; w < 4; w++)
        if (partly >> w & 1u) {
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (!(seen[w] >> c & 1u)) sr[w * 32 + c] = 0xff800000u;   // -infinity
        }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; c += 2) mx[c >> 1 & 3] = max3(mx[c >> 1 & 3], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = top > (any_key ? LAG : -INFINITY);   // the row has outgrown ref, or has its first key: ref moves, and what has been summed up shrinks
      if (__any_sync(0xffffffffu, grow)) {
        // (ALiBi alone lifts what is to come by up to c2 (i - the last key here): ref is set as high, or heads with steep slopes would move it in every tile)
        const float rise = ALIBI ? fmaxf(c2, 0.f) * (float)max(i - jt - (BN - 1), 0) : 0.f;
        const float shift = grow ? top + rise : 0.f, corr = grow && any_key ? exp2_hw(-shift) : 1.f;
        const f32x2 neg = pair_of(-shift, -shift);
        ref += shift;
        l *= corr;
#pragma unroll
        for (int c = 0; c < 128; c += 2) split(add2(pair_of(sr[c], sr[c + 1]), neg), sr[c], sr[c + 1]);
        if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < HD / 16; c++) {   // (the product of the tile before is complete: these scores were issued behind it)
            uint32_t o[16];
            tmem_ld16(tm_o + c * 16, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st16(tm_o + c * 16, o);
          }
          tmem_wait_st();
        }
        any_key |= grow;
      }
      f32x2 sum[2] = {0, 0};
#pragma unroll
      for (int half = 0; half < 2; half++) {
#pragma unroll
        for (int w = 2 * half; w < 2 * half + 2; w++) {
          if (dead >> w & 1u) {
#pragma unroll
            for (int u = 0; u < 16; u++) sr[w * 16 + u] = 0;
          } else {
#pragma unroll
            for (int c0 = w * 32; c0 < w * 32 + 32; c0 += 16) {   // 8 pairs: the first of them on the FMA pipe
              f32x2 p[8];
              exp2_poly<POLY_OF_8>(sr + c0, p);
#pragma unroll
              for (int u = POLY_OF_8; u < 8; u++) p[u] = pair_of(exp2_hw(__uint_as_float(sr[c0 + 2 * u])), exp2_hw(__uint_as_float(sr[c0 + 2 * u + 1])));
              uint32_t rounded[8];
#pragma unroll
              for (int u = 0; u < 8; u++) {
                float p0, p1;
                split(p[u], p0, p1);
                rounded[u] = pack_bf16(p0, p1);
              }
#pragma unroll
              for (int u = 0; u < 8; u++) sum[u & 1] = add2(sum[u & 1], HD == 64 ? pair_of(rounded[u] << 16, rounded[u] & 0xffff0000u) : p[u]);
#pragma unroll
              for (int u = 0; u < 8; u++) sr[(c0 >> 1) + u] = rounded[u];
            }
          }
        }
        tmem_st32(tm_s + half * 32, sr + half * 32);
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) tma::mbar_arrive(&ctl.p_full[tile][half]);
      }
      float s0, s1;
      split(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
    }
    if (ok && nt > 0) ok = wait_for(&ctl.pv_done[tile], 0, abort_flag);
    if (ok && nt > 0) {
      fence_after();
      const float inv_l = 1.f / l;
      bf16* dst = out + i * out_stride + (long long)h * hd;
      bool finite = true;
#pragma unroll 1
      for (int c = 0; c < HD / 32; c++) {
        uint32_t o[32];
        tmem_ld32(tm_o + c * 32, o);
        tmem_wait_ld(o);
        if (first != packed::NOBODY) {
#pragma unroll
          for (int v = 0; v < 4; v++) {
            if (c * 32 + v * 8 < hd) {
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; e++) {
                f[e] = __uint_as_float(o[v * 8 + e]) * inv_l;
                finite &= fabsf(f[e]) < INFINITY;
              }
              store_vec(dst + c * 32 + v * 8, f);
            }
          }
        }
      }
      __syncwarp();   // a row that is computed again has been stored by its thread, and is stored by all of them below: in this order
      uint32_t again = __ballot_sync(0xffffffffu, first != packed::NOBODY && (l < LEAST || (!finite && fabsf(l) < INFINITY)));
      for (; again; again &= again - 1) {
        const int r = tile * BM + quarter * 32 + __ffs(again) - 1;
        row_again(qkv, row_stride, out + (long long)(q0 + r) * out_stride + (long long)h * hd, q0 + r, ctl.first[r], h, g, H, Hk, hd, ALIBI ? slopes[h] : 0.f,
                  scale, CAP ? softcap : 0.f, lane);
      }
    }
    fence_before();
  } else {
    give_registers();
  }
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) {
      if (status) atomicExch(status, STATUS_PACKED);
      const uint64_t start = tma::global_ns();   // copies under way still land in this CTA's shared memory: it keeps it for longer than any copy takes
      while (tma::global_ns() - start < 200000ull) {}
    }
    __syncthreads();
  }
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int HD, bool CAP, bool ALIBI>
int launch(const CUtensorMap& map, const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows,
           int H, int Hk, int hd, int window, float softcap, int* status, cudaStream_t st) {
  static SmemLimit limit;
  const cudaError_t e = allow_smem((const void*)packed_umma_kernel<HD, CAP, ALIBI>, Smem<HD>::BYTES, limit);
  if (e != cudaSuccess) return (int)e;
  packed_umma_kernel<HD, CAP, ALIBI><<<dim3((unsigned)((rows + 2 * BM - 1) / (2 * BM)), H), THREADS, Smem<HD>::BYTES, st>>>(
      map, (const bf16*)qkv, row_stride, cu, S, slopes, (bf16*)out, out_stride, rows, H, Hk, hd, window, 1.0f / sqrtf((float)hd), softcap, status);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

int launch_packed_umma(const void* qkv, long long row_stride, const int* cu, int S, const float* slopes, void* out, long long out_stride, int rows, int H,
                       int Hk, int hd, int window, float softcap, int* status, cudaStream_t st) {
  CUtensorMap map;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)(H + 2 * Hk), (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, 1, BM};
  const int rc = tma::encode_bf16(&map, qkv, 3, dims, strides, box, true);
  if (rc != STU_OK) return rc;
  auto go = [&](auto kernel) { return kernel(map, qkv, row_stride, cu, S, slopes, out, out_stride, rows, H, Hk, hd, window, softcap, status, st); };
  if (hd <= 64)
    return softcap > 0.f ? slopes ? go(launch<64, true, true>) : go(launch<64, true, false>) : slopes ? go(launch<64, false, true>) : go(launch<64, false, false>);
  return softcap > 0.f ? slopes ? go(launch<128, true, true>) : go(launch<128, true, false>) : slopes ? go(launch<128, false, true>) : go(launch<128, false, false>);
}

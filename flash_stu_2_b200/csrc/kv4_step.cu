// Attention of one new token per sequence over its ring of 4 bits (kv4.cuh), which takes the token's key and value in.
//
// A CTA (or a cluster of up to 8 that share the keys) works for one key head of one sequence and up to 8 of its query heads; a warp takes 32 slots at a time.
//   scores   mma.sync, the numbers of 16 keys as rows, 8 queries as columns: a number n becomes bf16 by putting its bits under those of 128 (128 + n is exact), so
//            that two of them cost a shift and a logical operation.  A piece's scale is the same for all of a row's products:
//              q.k = sum over pieces of  step (q.(128 + n)) + (lowest - 128 step) sum(q)
//   softmax  a lane per key, the scores handed over through shared memory, a key's queries side by side (one access of 16 bytes for four scores or eight weights): cap, ALiBi,
//            window, exponentials in the exp2 domain against a maximum that moves only when a score outgrows it by 2^8, one vote of the warp for all rows
//   values   mma.sync, weights times the values' steps as rows; a number enters as n - 8 (the tensor core's sums are cut off, not rounded: with 128 + n the error of
//            16384 of them was four times the output's rounding); what lowest and the 8s add is summed up beside, one number per piece.  The weights' rows are 8 of 16: a
//            weight is two bf16, its leading bits and what these left, in rows r and r + 8 (error 2^-16)
// fp32: queries and weights are three bf16 each (the third in a product of its own), and scores are made of n - 8, too.
// Slots come by bulk copies, 128 at a time for the CTA's four warps, into three stages (18 KB each for heads of 128).
// Warps are merged through shared memory, CTAs of a cluster through distributed shared memory, in a fixed order; the new token's own key and value join there, as
// they are.  The ring's slot of the new token holds one that is out of everyone's window; it is written by one warp.
// Bound by instructions and a warp's chain of scores, softmax and values where the grid is large (32 sequences, 12 heads of 128, 1024 keys: 23.4 us, 2.4 TB/s of HBM's 6.5), by latency where it is small.
#include <cooperative_groups.h>

#include "kv4.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

int device_sm_count();   // gemm_tc.cu
int* device_status_word();

namespace {

constexpr int WARPS = 4, TILE = 32;      // warps of a CTA; slots that a warp takes at a time
constexpr int BLOCK = WARPS * TILE, STAGES = 3;
constexpr float NOTHING = -3.0e38f;      // the maximum of no scores
constexpr float LAG = 8.f;               // exp2 domain
constexpr int STATUS_KV4 = 14;

template <typename T, int W> struct Geometry {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NP = W / 64 ? W / 64 : 1;          // pieces
  static constexpr int WPL = W == 32 ? 1 : 2;             // words of a key's piece per lane
  static constexpr int KS = 2 * WPL;                      // steps of 16 dimensions per piece
  static constexpr int NT = W == 32 ? 4 : 8;              // tiles of 8 dimensions per piece
  static constexpr int PARTS = F32 ? 3 : 2;               // bf16 that a weight is
  static constexpr int ROWS_BYTES = BLOCK * W / 2, SCALE_BYTES = BLOCK * 4 * NP, STAGE = 2 * (ROWS_BYTES + SCALE_BYTES);   // keys, values, their scales
  static constexpr int P_BYTES = NP * PARTS * TILE * 16;
  __host__ __device__ static constexpr int warp_bytes(int rows) { return NP * rows * TILE * 4 + P_BYTES; }
  __host__ __device__ static constexpr int bytes(int rows) { return STAGES * STAGE + WARPS * warp_bytes(rows); }
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first of a sum
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t (&r)[2], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}
// numbers s of the two halves of w, as bf16: 128 + n, or n - 8 (CENTRED).  (mask, base and off: 0x000f000f, 0x43004300 and 0x43084308 from registers, which an
// instruction takes two of, where it takes one constant)
struct Bits { uint32_t mask, base, off; };
template <bool CENTRED> __device__ __forceinline__ uint32_t numbers(uint32_t w, int s, const Bits& k) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w >> 4 * s), "r"(k.mask), "r"(k.base));   // (w & mask) | base
  if (CENTRED) asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(k.off));
  return v;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float rounded(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
__device__ __forceinline__ float exp2_fast(float x) {   // relative error 2^-22; 0 for -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int N> __device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char* p) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  if constexpr (N == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
}
template <int N> __device__ __forceinline__ void load_rows(uint32_t (&w)[N], const float* p) {
  if constexpr (N == 8) {
    load_words(*reinterpret_cast<uint32_t(*)[4]>(w), reinterpret_cast<const unsigned char*>(p));
    load_words(*reinterpret_cast<uint32_t(*)[4]>(w + 4), reinterpret_cast<const unsigned char*>(p + 4));
  } else {
    load_words(w, reinterpret_cast<const unsigned char*>(p));
  }
}
// bf16 v[0], v[1], ... from p on
template <int N> __device__ __forceinline__ void store_halves(unsigned char* p, const uint32_t* v) {
  if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
  if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = make_uint2(v[0], v[1]);
  if constexpr (N == 2) *reinterpret_cast<uint32_t*>(p) = v[0];
  if constexpr (N == 1) *reinterpret_cast<unsigned short*>(p) = (unsigned short)v[0];
}

// NR: rows of queries that there is room for
template <typename T, int W, int NR>
__global__ void __launch_bounds__(WARPS * 32, W == 128 ? 3 : 4) kv4_step_kernel(
    const T* __restrict__ qkv, long long row_stride, unsigned char* k4, unsigned char* v4, int* __restrict__ pos, const float* __restrict__ slopes,
    T* __restrict__ out, int B, int H, int Hk, int hd, int slots, int window, float scale, float softcap, int update_cache, int splits, int* status) {
  typedef Geometry<T, W> G;
  constexpr bool F32 = G::F32;
  constexpr int NP = G::NP, KS = G::KS, NT = G::NT;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) float s_qsum[2][8], s_slope[8];
  __shared__ float s_own[8], s_m[WARPS][8], s_l[WARPS][8], c_m[8], c_l[8];
  const int g = blockIdx.x / splits, part = blockIdx.x - g * splits, b = blockIdx.y;
  const int R = H / Hk, r0 = blockIdx.z * 8, rows = min(8, R - r0), h0 = g * R + r0;   // the query heads h0 .. h0 + rows - 1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gr = lane >> 2, c = lane & 3;
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ int abort_flag;
  unsigned char* mine = smem + STAGES * G::STAGE + warp * G::warp_bytes(NR);
  float* sS = reinterpret_cast<float*>(mine);             // [piece][32 keys][row]; of 8 rows the halves change places with every fourth key (banks)
  unsigned char* sP = mine + NP * NR * TILE * 4;          // [piece][hi, mid (, lo)][32 keys][8 rows] bf16
  for (int e = lane; e < G::P_BYTES / 4; e += 32) reinterpret_cast<uint32_t*>(sP)[e] = 0;   // (rows that there is no room for stay as they are)
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) {
      tma::mbar_init(&full[i], 1);
      tma::mbar_init(&empty[i], WARPS);
    }
    abort_flag = 0;
    tma::fence_barrier_init();
  }
  Bits bits = {0x000f000fu, 0x43004300u, 0x43084308u};
  asm volatile("" : "+r"(bits.mask), "+r"(bits.base), "+r"(bits.off));
  pdl_trigger();   // launched with the programmatic attribute: resident while the projection in front of it drains
  pdl_wait();
  const int t = pos[2 * b];
  if (update_cache) {   // every CTA has read its position before it arrives here; the last one to arrive moves all of them on
    __syncthreads();
    // (The first warp has the copies to ask for.  Ordered arrivals take a step of 32 sequences 0.7 us of 23.4; by the first warp 0.3, and one of one sequence 0.6 of 9.2.)
    if (threadIdx.x == 32 && kv4::last_to_arrive(&pos[1], gridDim.x * gridDim.y * gridDim.z)) {
      pos[1] = 0;
      for (int i = 0; i < B; i++) pos[2 * i] += 1;
    }
  }
  const int newest = kv4::slot_of(t, slots), live = min(max(t, 0), window);   // the `live` slots before slot `newest`, around the ring's end
  const int first = newest >= live ? newest - live : newest - live + slots, tiles_all = (slots + BLOCK - 1) / BLOCK, tile0 = first / BLOCK;   // tiles of the CTA: 128 slots
  int tiles = 0;
  if (live > 0) {
    const int last = newest > 0 ? newest - 1 : slots - 1;
    tiles = first <= last ? last / BLOCK - tile0 + 1 : min(tiles_all, tiles_all - tile0 + last / BLOCK + 1);
  }
  const int parts = min(splits, max(1, tiles));   // CTAs that have something to do (a barrier of the cluster waits for none that has left)
  if (part >= parts) return;
  const long long head_bytes = kv4::head_bytes(W, slots);
  unsigned char *kb = k4 + ((long long)b * Hk + g) * head_bytes, *vb = v4 + ((long long)b * Hk + g) * head_bytes;
  const long long scales_at = (long long)slots * (W / 2);
  const T* row = qkv + (long long)b * row_stride;

  const unsigned char *kscales = kb + (long long)slots * (W / 2), *vscales = vb + (long long)slots * (W / 2);
  bool ok = true;
  auto fetch = [&](int turn) {   // the CTA's turn-th tile (of the ring's last, what there is), by the first warp
    const int n = part + turn * parts;
    if (warp != 0 || n >= tiles || !ok) return;
    const int stage = turn % STAGES;
    ok = tma::warp_wait_bounded(&empty[stage], ((uint32_t)(turn / STAGES) & 1u) ^ 1u, &abort_flag);
    if (ok && lane == 0) {
      const int tile = tile0 + n < tiles_all ? tile0 + n : tile0 + n - tiles_all, here = min(BLOCK, slots - tile * BLOCK);
      unsigned char* to = smem + stage * G::STAGE;
      uint64_t* bar = &full[stage];
      const uint32_t row_at = (uint32_t)tile * G::ROWS_BYTES, scale_at = (uint32_t)tile * G::SCALE_BYTES;
      const uint32_t row_bytes = here * (W / 2), scale_bytes = here * 4 * NP;
      tma::mbar_expect_tx(bar, 2 * (row_bytes + scale_bytes));
      tma::bulk_load(to, kb + row_at, row_bytes, bar);
      tma::bulk_load(to + 2 * G::ROWS_BYTES, kscales + scale_at, scale_bytes, bar);
      tma::bulk_load(to + G::ROWS_BYTES, vb + row_at, row_bytes, bar);
      tma::bulk_load(to + 2 * G::ROWS_BYTES + G::SCALE_BYTES, vscales + scale_at, scale_bytes, bar);
    }
    __syncwarp();
  };
  __syncwarp();   // (the first warp's first lane has made the barriers)
  for (int turn = 0; turn < STAGES - 1; turn++) fetch(turn);

  // queries in the order of the numbers: step u of piece p holds, of word i = 2 c + u / 2 (or c), dimensions s, s + 4 (columns 2 c, 2 c + 1) and s + 1, s + 5
  uint32_t qa[NP][KS][F32 ? 6 : 2];
  {
    const T* q = row + (long long)(h0 + gr) * hd;
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
      for (int u = 0; u < KS; u++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const int d = 64 * p + 8 * (G::WPL * c + (u >> 1)) + 2 * (u & 1) + half;
          const float x0 = gr < rows && d < hd ? Elem<T>::to_f(q[d]) : 0.f, x1 = gr < rows && d + 4 < hd ? Elem<T>::to_f(q[d + 4]) : 0.f;
          if (F32) {
            const float h0_ = rounded(x0), h1_ = rounded(x1), m0_ = rounded(x0 - h0_), m1_ = rounded(x1 - h1_);
            qa[p][u][half] = bf16_pair(h0_, h1_);
            qa[p][u][2 + half] = bf16_pair(m0_, m1_);
            qa[p][u][4 + half] = bf16_pair(x0 - h0_ - m0_, x1 - h1_ - m1_);
          } else {
            qa[p][u][half] = bf16_pair(x0, x1);
          }
        }
  }
  if (threadIdx.x < 8) s_qsum[0][threadIdx.x] = s_qsum[1][threadIdx.x] = s_slope[threadIdx.x] = 0.f;   // rows without a query are computed beside the others
  __syncthreads();
  for (int r = warp; r < rows; r += WARPS) {   // each query's sums, and its score with the new token's own key
    const T *q = row + (long long)(h0 + r) * hd, *k = row + (long long)(H + g) * hd;
    float sum0 = 0.f, sum1 = 0.f, dot = 0.f;
    for (int d = lane; d < hd; d += 32) {
      const float x = Elem<T>::to_f(q[d]);
      (d < 64 ? sum0 : sum1) += x;
      dot = fmaf(x, Elem<T>::to_f(k[d]), dot);
    }
    sum0 = warp_sum(sum0);
    sum1 = warp_sum(sum1);
    dot = warp_sum(dot) * scale;
    if (softcap > 0.f) dot = softcap * tanhf(dot / softcap);
    if (lane == 0) {
      s_qsum[0][r] = sum0;
      s_qsum[1][r] = sum1;
      s_own[r] = dot * LOG2E;
      s_slope[r] = slopes ? slopes[h0 + r] * LOG2E : 0.f;
    }
  }
  __syncthreads();
  if (update_cache && part == 0 && blockIdx.z == 0 && warp == WARPS - 1) {   // the new key and value: eight lanes per piece
    const int unit = lane >> 3, which = unit / NP, piece = unit % NP, i = lane & 7;
    const bool on = unit < 2 * NP, there = on && piece * 64 + i * 8 < hd;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there) kv4::load8<false>(row + (long long)(H + which * Hk + g) * hd + piece * 64 + i * 8, x);
    uint32_t word, sc;
    kv4::quantize(x, there, word, sc);
    unsigned char* ring = which ? vb : kb;
    if (on && i * 8 < W / NP) reinterpret_cast<uint32_t*>(ring)[(long long)newest * (W / 8) + kv4::word_at(i, piece, NP)] = word;
    if (on && i == 0) reinterpret_cast<uint32_t*>(ring + scales_at)[(long long)newest * NP + piece] = sc;
  }

  float m[NR], bar[NR], l[NR], low[NR][NP], o[NP][NT][4];   // bar: what a score has to pass for the maximum to move
  // a score is what is summed up times k_in, or, capped, tanh of that times k_out
  const float k_in = softcap > 0.f ? scale / softcap : scale * LOG2E, k_out = softcap * LOG2E;
#pragma unroll
  for (int r = 0; r < NR; r++) {
    m[r] = bar[r] = NOTHING;
    l[r] = 0.f;
#pragma unroll
    for (int p = 0; p < NP; p++) low[r][p] = 0.f;
  }
#pragma unroll
  for (int p = 0; p < NP; p++)
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[p][d][e] = 0.f;

  // the column of this lane's key among 16: the keys whose words a lane of the second product takes together, c, c + 4, c + 8 and c + 12, are in rows that lie in
  // more banks than neighbours
  const int column = (lane & 16) + 2 * (lane & 3) + ((lane >> 2) & 1) + (lane & 8);
  for (int turn = 0, n = part; n < tiles; n += parts, turn++) {   // (the same for the whole CTA)
    const int tile = tile0 + n < tiles_all ? tile0 + n : tile0 + n - tiles_all, stage = turn % STAGES;
    const unsigned char *rows_k = smem + stage * G::STAGE + warp * TILE * (W / 2), *rows_v = rows_k + G::ROWS_BYTES;
    const unsigned char *scale_k = smem + stage * G::STAGE + 2 * G::ROWS_BYTES + (warp * TILE + lane) * 4 * NP, *scale_v = scale_k + G::SCALE_BYTES;
    const uint32_t phase = (uint32_t)(turn / STAGES) & 1u;
    fetch(turn + STAGES - 1);
    ok = ok && (__all_sync(0xffffffffu, tma::mbar_try_wait(&full[stage], phase)) || tma::warp_wait_bounded(&full[stage], phase, &abort_flag));
    if (!ok) break;
    // ---- scores of 2 x 16 keys with 8 queries (a product's sum is there for the next 20 clocks later: four of them take turns)
    {
      uint32_t k[4][NP * G::WPL];
#pragma unroll
      for (int j = 0; j < 4; j++) load_words(k[j], rows_k + (8 * j + gr) * (W / 2) + c * (W / 8));
      float s[NP][2][4];
#pragma unroll
      for (int u = 0; u < KS; u++)
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t w0 = k[2 * j][(u >> 1) * NP + p], w1 = k[2 * j + 1][(u >> 1) * NP + p];
            const uint32_t a0 = numbers<F32>(w0, 2 * (u & 1), bits), a1 = numbers<F32>(w1, 2 * (u & 1), bits);
            const uint32_t a2 = numbers<F32>(w0, 2 * (u & 1) + 1, bits), a3 = numbers<F32>(w1, 2 * (u & 1) + 1, bits);
            if (u == 0) mma_first(s[p][j], a0, a1, a2, a3, qa[p][u][0], qa[p][u][1]);
            else mma(s[p][j], a0, a1, a2, a3, qa[p][u][0], qa[p][u][1]);
            if (F32) {
              mma(s[p][j], a0, a1, a2, a3, qa[p][u][2], qa[p][u][3]);
              mma(s[p][j], a0, a1, a2, a3, qa[p][u][4], qa[p][u][5]);
            }
          }
#pragma unroll
      for (int p = 0; p < NP; p++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 2; e++)   // key 16 j + gr + 8 e, queries 2 c and 2 c + 1
            if (2 * c < NR) {
              float* at = sS + (p * TILE + 16 * j + gr + 8 * e) * NR + (NR == 8 ? (2 * c) ^ (gr & 4) : 2 * c);
              if (NR == 1) *at = s[p][j][2 * e];
              else *reinterpret_cast<float2*>(at) = make_float2(s[p][j][2 * e], s[p][j][2 * e + 1]);
            }
    }
    __syncwarp();
    // ---- a lane per key
    const int slot = tile * BLOCK + warp * TILE + lane, behind = newest > slot ? newest - slot : newest - slot + slots;   // 1 .. slots
    const bool seen = slot < slots && behind <= live;
    const float far = (float)behind;
    float kstep[NP], klow[NP], vstep[NP], vlow[NP];
    uint32_t ks[NP], vs[NP];
    load_words(ks, scale_k);
    load_words(vs, scale_v);
#pragma unroll
    for (int p = 0; p < NP; p++) {
      kstep[p] = __uint_as_float(ks[p] & 0xffff0000u);
      klow[p] = fmaf(F32 ? 8.f : -128.f, kstep[p], __uint_as_float(ks[p] << 16)) * k_in;
      kstep[p] *= k_in;
      vstep[p] = seen ? __uint_as_float(vs[p] & 0xffff0000u) : 0.f;
      vlow[p] = seen ? fmaf(8.f, vstep[p], __uint_as_float(vs[p] << 16)) : 0.f;
    }
    float x[NR];   // scores, then weights
#pragma unroll
    for (int r = 0; r < NR; r++) x[r] = 0.f;
#pragma unroll
    for (int p = 0; p < NP; p++) {
      uint32_t raw[NR], qsum[NR];
      load_rows(qsum, s_qsum[p]);
      const float* at = sS + (p * TILE + lane) * NR;
      if constexpr (NR == 8) {
        load_words(*reinterpret_cast<uint32_t(*)[4]>(raw), reinterpret_cast<const unsigned char*>(at + (lane & 4)));
        load_words(*reinterpret_cast<uint32_t(*)[4]>(raw + 4), reinterpret_cast<const unsigned char*>(at + (4 ^ (lane & 4))));
      } else {
        load_words(raw, reinterpret_cast<const unsigned char*>(at));
      }
#pragma unroll
      for (int r = 0; r < NR; r++) x[r] = fmaf(kstep[p], __uint_as_float(raw[r]), fmaf(klow[p], __uint_as_float(qsum[r]), x[r]));
    }
    bool over = false;
    uint32_t slope[NR];
    load_rows(slope, s_slope);
#pragma unroll
    for (int r = 0; r < NR; r++) {
      if (softcap > 0.f) {
        if (F32) x[r] = tanhf(x[r]);
        else asm("tanh.approx.f32 %0, %0;" : "+f"(x[r]));   // relative error 2^-11
        x[r] *= k_out;
      }
      x[r] = seen ? fmaf(-__uint_as_float(slope[r]), far, x[r]) : -INFINITY;
      over = over || x[r] > bar[r];
    }
    const bool moved = __any_sync(0xffffffffu, over);   // seldom: one vote for all rows
    float shrink = 1.f;   // of row gr
    if (moved) {
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const float top = fmaxf(m[r], warp_max(x[r])), corr = exp2_fast(m[r] - top);   // (0 where there was no key yet)
        m[r] = top;
        bar[r] = top + LAG;
        l[r] *= corr;
#pragma unroll
        for (int p = 0; p < NP; p++) low[r][p] *= corr;
        if (gr == r) shrink = corr;
      }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
      x[r] = exp2_fast(x[r] - m[r]);
      l[r] += x[r];
    }
#pragma unroll
    for (int p = 0; p < NP; p++) {
      unsigned char* at = sP + (p * G::PARTS * TILE + column) * 16;
      uint32_t hi[(NR + 1) / 2], mid[(NR + 1) / 2], lo[(NR + 1) / 2];
#pragma unroll
      for (int r = 0; r < NR; r += 2) {   // what is left of a weight that is cut off is exact
        const float a0 = x[r] * vstep[p], a1 = r + 1 < NR ? x[r + 1 < NR ? r + 1 : r] * vstep[p] : 0.f;
        const float b0 = a0 - __uint_as_float(__float_as_uint(a0) & 0xffff0000u), b1 = a1 - __uint_as_float(__float_as_uint(a1) & 0xffff0000u);
        hi[r / 2] = __byte_perm(__float_as_uint(a0), __float_as_uint(a1), 0x7632);
        if (F32) {
          mid[r / 2] = __byte_perm(__float_as_uint(b0), __float_as_uint(b1), 0x7632);
          lo[r / 2] = bf16_pair(b0 - __uint_as_float(__float_as_uint(b0) & 0xffff0000u), b1 - __uint_as_float(__float_as_uint(b1) & 0xffff0000u));
        } else {
          mid[r / 2] = bf16_pair(b0, b1);
        }
      }
      store_halves<NR>(at, hi);
      store_halves<NR>(at + TILE * 16, mid);
      if (F32) store_halves<NR>(at + 2 * TILE * 16, lo);
#pragma unroll
      for (int r = 0; r < NR; r++) low[r][p] = fmaf(x[r], vlow[p], low[r][p]);
    }
    if (moved) {   // (for the whole warp)
#pragma unroll
      for (int p = 0; p < NP; p++)
#pragma unroll
        for (int d = 0; d < NT; d++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[p][d][e] *= shrink;
    }
    __syncwarp();
    // ---- weighted values: 2 x 16 keys
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      uint32_t v[4][NP];   // (of a head of 32 a lane's word holds its four numbers and those of the next row's lane)
#pragma unroll
      for (int e = 0; e < 4; e++) load_words(v[e], rows_v + (16 * kk + c + 4 * e) * (W / 2) + (W == 32 ? gr >> 1 : gr * NP) * 4);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        uint32_t a[4], a3[2] = {0u, 0u};
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(sP + (p * G::PARTS * TILE + 16 * kk + (lane & 7)) * 16);
        // rows 0 - 7 (leading bits) and 8 - 15 (what they left) of keys 0 - 7, then of keys 8 - 15
        ldmatrix_x4_trans(a, at + ((lane & 8) ? TILE * 16 : 0) + (lane >> 4) * 128);
        if (F32) ldmatrix_x2_trans(a3, at + 2 * TILE * 16 + ((lane & 8) ? 128 : 0));
        uint32_t lo[2], hi[2];   // numbers 0 - 3 and 4 - 7 of two keys
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t x = v[2 * e][p], y = v[2 * e + 1][p];
          lo[e] = __byte_perm(x, y, W == 32 && (gr & 1) ? 0x7632 : 0x5410);
          hi[e] = __byte_perm(x, y, 0x7632);
        }
#pragma unroll
        for (int d = 0; d < NT; d++) {
          const uint32_t b0 = numbers<true>(d < 4 ? lo[0] : hi[0], d & 3, bits), b1 = numbers<true>(d < 4 ? lo[1] : hi[1], d & 3, bits);
          mma(o[p][d], a[0], a[1], a[2], a[3], b0, b1);
          if (F32) mma(o[p][d], a3[0], 0u, a3[1], 0u, b0, b1);
        }
      }
    }
    __syncwarp();
    if (lane == 0) tma::mbar_arrive(&empty[stage]);
  }
  // ---- this warp's rows; then the CTA's
  __syncthreads();   // (what they are written to is other warps' scratch)
  if (abort_flag) {   // a copy that did not land in time: none is under way any more when the CTA ends
    if (threadIdx.x == 0) {
      if (status) atomicExch(status, STATUS_KV4);
      const uint64_t start = tma::global_ns();
      while (tma::global_ns() - start < 200000ull) {}
    }
    __syncthreads();
  }
  float* sO = reinterpret_cast<float*>(smem);   // [warp][row][W]
#pragma unroll
  for (int r = 0; r < NR; r++) {
    if (r < rows) {
      const float sum = warp_sum(l[r]);
#pragma unroll
      for (int p = 0; p < NP; p++) low[r][p] = warp_sum(low[r][p]);
      if (lane == 0) {
        s_m[warp][r] = m[r];
        s_l[warp][r] = sum;
      }
      if (gr == r) {
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
          for (int d = 0; d < NT; d++)
#pragma unroll
            for (int e = 0; e < 2; e++) sO[(warp * NR + r) * W + 64 * p + (2 * c + e) * NT + d] = o[p][d][e] + o[p][d][2 + e] + low[r][p];
      }
    }
  }
  __syncthreads();
  const bool one = parts == 1;
  for (int e = threadIdx.x; e < rows * W; e += WARPS * 32) {
    const int r = e / W, d = e % W;
    float top = one ? s_own[r] : NOTHING, num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = exp2_fast(s_m[w][r] - top);
      num = fmaf(sO[(w * NR + r) * W + d], f, num);
      den = fmaf(s_l[w][r], f, den);
    }
    if (one) {
      const float f = exp2_fast(s_own[r] - top);
      if (d < hd) out[((long long)b * H + h0 + r) * hd + d] = Elem<T>::from_f(fmaf(f, Elem<T>::to_f(row[(long long)(H + Hk + g) * hd + d]), num) / (den + f));
    } else {
      sO[r * W + d] = num;   // (each thread reads its own column of all warps before)
      if (d == 0) {
        c_m[r] = top;
        c_l[r] = den;
      }
    }
  }
  if (one) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (part == 0) {
    for (int e = threadIdx.x; e < rows * W; e += WARPS * 32) {
      const int r = e / W, d = e % W;
      float top = s_own[r], num = 0.f, den = 0.f;
      for (int i = 0; i < parts; i++) top = fmaxf(top, *cluster.map_shared_rank(&c_m[r], i));
      for (int i = 0; i < parts; i++) {
        const float f = exp2_fast(*cluster.map_shared_rank(&c_m[r], i) - top);
        num = fmaf(*cluster.map_shared_rank(&sO[r * W + d], i), f, num);
        den = fmaf(*cluster.map_shared_rank(&c_l[r], i), f, den);
      }
      const float f = exp2_fast(s_own[r] - top);
      if (d < hd) out[((long long)b * H + h0 + r) * hd + d] = Elem<T>::from_f(fmaf(f, Elem<T>::to_f(row[(long long)(H + Hk + g) * hd + d]), num) / (den + f));
    }
  }
  cluster.sync();   // the other CTAs' results stay alive until they are read
}

template <typename T, int W, int NR>
int launch(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const float* slopes, void* out, int B, int H, int Hk, int hd, int slots,
           int window, float softcap, int update_cache, int* status, cudaStream_t st) {
  typedef Geometry<T, W> G;
  const size_t smem = G::bytes(NR);
  static_assert(G::bytes(NR) >= WARPS * NR * W * 4, "the warps' rows are merged there");
  static SmemLimit limit;
  cudaError_t e = allow_smem((const void*)kv4_step_kernel<T, W, NR>, smem, limit);
  if (e != cudaSuccess) return (int)e;
  const int groups = (H / Hk + 7) / 8;
  // CTAs that share the keys: as many as take least by rounds of what the SMs hold at a time, times a CTA's tiles with its beginning and end (3 tiles, with a cluster 5), three tenths more for
  // each further CTA on an SM.  Of 37 measured sizes (12 to 1536 sequences' heads, 500 to 16384 keys, heads of 64 and 128) the time is 2 % above the best number's on average, at most 28 %;
  // with the fullest SM's work alone, as if clusters began as places become free, it was 8 % (all without ordered arrivals).  Heads of 128, us with 1, 2, 3, 4, 8 CTAs: 12 heads of 1025 keys 14.3, 11.9, 10.2, 10.0, 8.6; 384
  // of them 22.7, 31.4, 36.1, 45.3, 78.4; 128 of 16385 keys, 8 queries each, 309, 170, 119, 154, 158.
  const long long pairs = (long long)Hk * B * groups, sms = device_sm_count();
  const int tiles = window / BLOCK + 1, per_sm = W == 128 ? 3 : 4;
  int splits = 1;
  double least = 1e30;
  for (int s = 1; s <= 8 && s <= tiles; s++) {
    const long long at_a_time = sms * per_sm / s, rounds = (pairs + at_a_time - 1) / at_a_time, on_one = (pairs * s + sms - 1) / sms;
    const double cost = (double)rounds * ((double)tiles / s + (s > 1 ? 5 : 3)) * (0.7 + 0.3 * (double)(on_one < per_sm ? on_one : per_sm));
    if (cost < least) {
      least = cost;
      splits = s;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(Hk * splits, B, groups);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (splits > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = splits;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  if (pdl_enabled()) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  e = cudaLaunchKernelEx(&cfg, kv4_step_kernel<T, W, NR>, (const T*)qkv, row_stride, (unsigned char*)k4, (unsigned char*)v4, pos, slopes, (T*)out, B, H, Hk, hd,
                         slots, window, 1.0f / sqrtf((float)hd), softcap, update_cache, splits, status);
  return (int)e;
}

}  // namespace

extern "C" int stu_kv4_step(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const float* slopes, void* out, int B, int H, int Hk,
                            int hd, int slots, int window, float softcap, int update_cache, int* status, int dtype, void* stream) {
  if (!qkv || !k4 || !v4 || !pos || !out) return STU_ERR_NULL;
  const int rc = kv4::geometry(B, H, Hk, hd, slots, dtype);
  if (rc != STU_OK) return rc;
  if (window < 0 || window >= slots || B > 65535 || row_stride < (long long)(H + 2 * Hk) * hd) return STU_ERR_SHAPE;
  if (!aligned16(k4) || !aligned16(v4)) return STU_ERR_ALIGN;
  if (!status) status = device_status_word();
  const int R = H / Hk < 8 ? H / Hk : 8;
  auto go = [&](auto f) { return f(qkv, row_stride, k4, v4, pos, slopes, out, B, H, Hk, hd, slots, window, softcap, update_cache, status, (cudaStream_t)stream); };
  auto by_rows = [&](auto one, auto two, auto four, auto eight) { return R == 1 ? go(one) : R == 2 ? go(two) : R <= 4 ? go(four) : go(eight); };
  if (dtype == STU_F32) {
    if (hd <= 32) return by_rows(launch<float, 32, 1>, launch<float, 32, 2>, launch<float, 32, 4>, launch<float, 32, 8>);
    if (hd <= 64) return by_rows(launch<float, 64, 1>, launch<float, 64, 2>, launch<float, 64, 4>, launch<float, 64, 8>);
    return by_rows(launch<float, 128, 1>, launch<float, 128, 2>, launch<float, 128, 4>, launch<float, 128, 8>);
  }
  if (hd <= 32) return by_rows(launch<bf16, 32, 1>, launch<bf16, 32, 2>, launch<bf16, 32, 4>, launch<bf16, 32, 8>);
  if (hd <= 64) return by_rows(launch<bf16, 64, 1>, launch<bf16, 64, 2>, launch<bf16, 64, 4>, launch<bf16, 64, 8>);
  return by_rows(launch<bf16, 128, 1>, launch<bf16, 128, 2>, launch<bf16, 128, 4>, launch<bf16, 128, 8>);
}

// Products of two e4m3 operands with a scale for each 128 of a row (fp8.cuh) on the 5th-generation tensor cores: D[M,N] = x[M,K] . W[N,K]^T,
// fp32 sums in tensor memory.
//
// kind::mxf8f6f4 multiplies every 32 columns of a row by a power of two that it finds in tensor memory.  The scales of 128 rows and four blocks of
// 128 columns are one 32-bit word per row, 512 bytes in the order that tcgen05.cp takes: they come by TMA with every fourth k-block, one thread
// copies them over, and the four instructions of a k-block take the byte that their descriptor names.  So no sum ever passes a register
// before its epilogue.
//
// A pair of CTAs on neighbouring SMs computes tiles of 256 x 256 (gate/up: 256 x 128 of both) with cta_group::2, or a CTA alone tiles of 128
// rows where those would leave SMs idle.  Warp 0 of a CTA is its TMA producer, warp 1 of the first CTA issues scale copies and instructions, warps 2..9 drain
// the accumulators.  The kernel is persistent; two accumulators of 256 columns and the scales do not fit 512 columns, so the accumulators
// share 32 columns: the epilogue reads those first and hands them back ahead of the rest.
//
// gate/up: a thread has 64 of the 128 features of a block of its row, two warps settle the block's scale through shared memory, and the row
// leaves in 8 bits.
//
// Every wait is bounded, as in gemm_tc.cu: on expiry the waiter tells the others, raises the status word, and the CTAs drain their copies, free
// their tensor memory and return.
#include <cuda.h>

#include <new>

#include "fp8.cuh"
#include "fp8_gemm.cuh"
#include "tma.cuh"

int device_sm_count();      // gemm_tc.cu
int* device_status_word();  // gemm_tc.cu

namespace {

constexpr int BM = 128, BK = 128;   // rows of x per CTA; bytes of a k-block: a block of 128 columns, one row of the 128-byte swizzle
constexpr int A_BYTES = BM * BK;
constexpr int EPI_WARPS = 8, BLOCK_BYTES = 32 * 64 * 2;   // an epilogue warp's block of 32 rows x 64 bf16 columns
constexpr uint32_t WAIT_LIMIT = 1u << 22;

__device__ __forceinline__ void load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(tma::smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(tma::smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(tma::smem_u32(dst)), "l"(map), "r"(tma::smem_u32(bar)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ bool mbar_ready(uint64_t* bar, uint32_t parity) {   // without waiting
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(tma::smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// shared::cluster address of the pair's first CTA's copy of a shared-memory object
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tma::smem_u32(p)));
  return a;
}
__device__ __forceinline__ uint32_t load_from_cta(const volatile int* p, uint32_t cta) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tma::smem_u32((const void*)p)), "r"(cta));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void store_to_cta(const volatile int* p, uint32_t cta, int v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tma::smem_u32((const void*)p)), "r"(cta));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void pair_sync() {   // both CTAs, all threads; orders no stores
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Shared-memory descriptors: an operand tile, rows of 128 bytes in the 128-byte swizzle, 8-row groups 1024 bytes apart; a piece of scales, 32 rows of
// 16 bytes without a swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t scales_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

template <int CTAS> __device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (CTAS == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// One instruction: 32 columns of K.  sf: which byte of the scale words.
template <int CTAS, int N>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t sfa, uint32_t sfb, uint32_t sf, uint32_t accumulate) {
  // D fp32, A and B e4m3, both K-major, scales E8M0
  const uint32_t idesc = (1u << 23) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(CTAS * BM >> 4) << 24) | (sf << 29) | (sf << 4);
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// Arrives (at the barrier of both CTAs of a pair) when what was issued so far is done.
template <int CTAS> __device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tma::smem_u32(bar)),
                 "h"((uint16_t)3) : "memory");
  else
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

// Bands of group_m row tiles, rows first inside a band.
__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
  const int band = tile / (group_m * tiles_n), r = tile - band * group_m * tiles_n, rows = min(group_m, tiles_m - band * group_m);
  tn = r / rows;
  tm = band * group_m + (r - tn * rows);
}

struct Out {
  bf16* y;             // plain: rows of ldy elements
  long long ldy;
  const bf16* resid;   // may be NULL, may be y
  long long ldr;
  unsigned char *hq, *hs;   // gate/up
};

template <bool DUAL, int CTAS, int TN> struct Form {
  static constexpr int MMA_N = DUAL ? 2 * TN : TN;                     // accumulator columns
  static constexpr int B_ROWS = MMA_N / CTAS;                          // rows of B in a CTA's shared memory
  static constexpr int TILE_BYTES = A_BYTES + B_ROWS * BK;             // of one CTA
  static constexpr int SCALE_BYTES = fp8::PIECE * (1 + (MMA_N + 127) / 128);
  static constexpr int STAGES = DUAL ? (CTAS == 2 ? 6 : 4) : 5;
  // accumulators at columns 0 and SECOND, scales behind them, twice 16 columns (x at 0, W from 4 on)
  static constexpr int SHARED = MMA_N == 256 ? 32 : 0, SECOND = MMA_N - SHARED, SCALES = SECOND + MMA_N;
  static constexpr uint32_t TMEM_COLS = MMA_N == 256 ? 512 : 2 * MMA_N + 32 <= 256 ? 256 : 512;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * (TILE_BYTES + SCALE_BYTES) + (DUAL ? 2048 : EPI_WARPS * BLOCK_BYTES) + 1024;
  static_assert(SMEM <= 227 * 1024 && SMEM > 114 * 1024, "one CTA per SM");
  static_assert(SCALES + 32 <= (int)TMEM_COLS, "tensor memory");
};

template <bool DUAL, int CTAS, int TN>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(64 + 32 * EPI_WARPS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmB2,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmSB2, int M, int N,
                    int K, int tiles_m, int tiles_n, int group_m, Out out, int* status, int drop_first_copy, unsigned long long wait_ns) {
  using F = Form<DUAL, CTAS, TN>;
  constexpr bool PAIR = CTAS == 2;
  constexpr int MMA_N = F::MMA_N, STAGES = F::STAGES, SHARED = F::SHARED;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* scales = smem + STAGES * F::TILE_BYTES;            // [stage]: of x, then of W
  unsigned char* blocks = scales + STAGES * F::SCALE_BYTES;         // plain: one per epilogue warp; gate/up: maxima [2][4][2][32] and marks
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(blocks + (DUAL ? 2048 : EPI_WARPS * BLOCK_BYTES));   // used in the first CTA alone
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;    // [2]
  uint64_t* tmem_empty = tmem_full + 2;        // [2], first CTA alone
  uint64_t* shared_read = tmem_empty + 2;      // [2], first CTA alone: the columns that this accumulator shares have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(shared_read + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [2]: this CTA gave up, the other one did
  int* issued_ctr = reinterpret_cast<int*>(tmem_slot + 3);
  int* consumed_ctr = issued_ctr + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? blockIdx.x & 1 : 0, pair = blockIdx.x / CTAS, pairs = gridDim.x / CTAS;
  const int num_tiles = tiles_m * tiles_n, num_kb = fp8::blocks_of(K);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      tma::mbar_init(&full_bar[s], 1);
      tma::mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      tma::mbar_init(&tmem_full[i], 1);
      tma::mbar_init(&tmem_empty[i], CTAS * EPI_WARPS);
      tma::mbar_init(&shared_read[i], CTAS * EPI_WARPS / 2);
    }
    abort_flag[0] = abort_flag[1] = 0;
    *issued_ctr = 0;
    *consumed_ctr = 0;
    tma::fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_u32(tmem_slot)), "r"(F::TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_u32(tmem_slot)), "r"(F::TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();      // everything so far ran beside the end of the kernel in front
  pdl_trigger();

  if (warp == 0) {
    // ---------------- TMA producer (of either CTA: its 128 rows of x, its part of the rows of W, the scales of both)
    const bool leader = elect_one();
    const CUtensorMap* mapB = DUAL && rank ? &tmB2 : &tmB;   // gate/up in a pair: the first CTA brings the gate rows, the second the up rows
    const uint32_t full0 = in_first_cta(full_bar);
    int g = 0, s = 0;
    uint32_t ph = 1;
    bool ok = true, ready = false;
    for (int tile = pair; ok && tile < num_tiles; tile += pairs) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, group_m, tm, tn);
      const int m0 = (CTAS * tm + rank) * BM, n0 = tn * TN + (DUAL ? 0 : rank * F::B_ROWS), nb = tn * TN / 128;
      for (int kb = 0; kb < num_kb; kb++, g++) {
        if (!ready) ok = tma::warp_wait_bounded(&empty_bar[s], ph, abort_flag, wait_ns);
        if (!ok) break;
        const int s1 = s + 1 == STAGES ? 0 : s + 1;
        const uint32_t ph1 = s1 ? ph : ph ^ 1u;
        const bool ready1 = mbar_ready(&empty_bar[s1], ph1);   // asked for here, looked at behind the copies
        if (leader) {
          const bool with_scales = (kb & 3) == 0;
          unsigned char *sa = smem + s * F::TILE_BYTES, *ss = scales + s * F::SCALE_BYTES;
          if (rank == 0) tma::mbar_expect_tx(&full_bar[s], CTAS * (F::TILE_BYTES + (with_scales ? F::SCALE_BYTES : 0)));   // of both CTAs
          if (!(drop_first_copy && g == 0)) {   // (failure-detection test: the first stage never fills)
            const uint32_t bar = full0 + s * (uint32_t)sizeof(uint64_t);
            if constexpr (PAIR) {
              load_2d_pair(sa, &tmA, bar, kb * BK, m0);
              load_2d_pair(sa + A_BYTES, mapB, bar, kb * BK, n0);
              if (with_scales) {
                load_3d_pair(ss, &tmSA, bar, 0, kb >> 2, m0 / BM);
                load_3d_pair(ss + fp8::PIECE, &tmSB, bar, 0, kb >> 2, nb);
                if (DUAL) load_3d_pair(ss + 2 * fp8::PIECE, &tmSB2, bar, 0, kb >> 2, nb);
              }
            } else {
              load_2d(sa, &tmA, &full_bar[s], kb * BK, m0);
              load_2d(sa + A_BYTES, &tmB, &full_bar[s], kb * BK, n0);
              if (DUAL) load_2d(sa + A_BYTES + TN * BK, &tmB2, &full_bar[s], kb * BK, n0);
              if (with_scales) {
                tma::load_3d(ss, &tmSA, &full_bar[s], 0, kb >> 2, m0 / BM);
                tma::load_3d(ss + fp8::PIECE, &tmSB, &full_bar[s], 0, kb >> 2, nb);
                if (DUAL) tma::load_3d(ss + 2 * fp8::PIECE, &tmSB2, &full_bar[s], 0, kb >> 2, nb);
              }
            }
          }
        }
        ready = __all_sync(0xffffffffu, ready1);
        s = s1, ph = ph1;
      }
    }
    if (leader) *issued_ctr = g;
    // the last stages' releases arrive in both CTAs: wait for them here, so that none is under way to a CTA that has left
    for (int h = max(g - STAGES, 0); ok && h < g; h++)
      ok = tma::warp_wait_bounded(&empty_bar[h % STAGES], (uint32_t)(h / STAGES) & 1u, abort_flag, wait_ns);
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- issuer of the pair
      const bool leader = elect_one();
      const uint64_t da0 = operand_desc(tma::smem_u32(smem)), db0 = operand_desc(tma::smem_u32(smem) + A_BYTES);
      const uint64_t ds0 = scales_desc(tma::smem_u32(scales));
      int g = 0, s = 0, it = 0, pieces = 0;
      uint32_t ph = 0, sf_cols = tmem_base + F::SCALES;
      bool ok = true, ready = false;
      for (int tile = pair; ok && tile < num_tiles; tile += pairs, it++) {
        const int buf = it & 1;
        const uint32_t acc = tmem_base + (uint32_t)buf * F::SECOND;
        ok = tma::warp_wait_bounded(&tmem_empty[buf], (((uint32_t)it >> 1) & 1u) ^ 1u, abort_flag, wait_ns);
        if (SHARED && ok && it > 0) ok = tma::warp_wait_bounded(&shared_read[buf ^ 1], ((uint32_t)(it - 1) >> 1) & 1u, abort_flag, wait_ns);
        if (!ok) break;
        for (int kb = 0; kb < num_kb; kb++, g++) {
          if (!ready) ok = tma::warp_wait_bounded(&full_bar[s], ph, abort_flag, wait_ns);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int s1 = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t ph1 = s1 ? ph : ph ^ 1u;
          const bool ready1 = mbar_ready(&full_bar[s1], ph1);
          if ((kb & 3) == 0) sf_cols = tmem_base + F::SCALES + 16 * (pieces++ & 1);
          if (leader) {
            if ((kb & 3) == 0) {   // in order with the instructions around it
              const uint64_t ds = ds0 + (uint64_t)(s * (F::SCALE_BYTES >> 4));
#pragma unroll
              for (int i = 0; i < F::SCALE_BYTES / fp8::PIECE; i++) copy_scales<CTAS>(sf_cols + 4 * i, ds + i * (fp8::PIECE >> 4));
            }
            const uint64_t da = da0 + (uint64_t)(s * (F::TILE_BYTES >> 4)), db = db0 + (uint64_t)(s * (F::TILE_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < BK / 32; kk++)   // 32 bytes along K inside the swizzled row: +2
              multiply<CTAS, MMA_N>(acc, da + 2 * kk, db + 2 * kk, sf_cols, sf_cols + 4, kb & 3, (kb | kk) ? 1u : 0u);
            commit<CTAS>(&empty_bar[s]);
          }
          ready = __all_sync(0xffffffffu, ready1);
          s = s1, ph = ph1;
        }
        if (ok && leader) commit<CTAS>(&tmem_full[buf]);
        __syncwarp();
      }
      if (leader) *consumed_ctr = g;
    }
  } else {
    // ---------------- epilogue warps: TMEM lane quarter = warp % 4 (32 rows), half of the columns
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t hand_back = in_first_cta(tmem_empty), hand_shared = in_first_cta(shared_read);
    int it = 0;
    for (int tile = pair; tile < num_tiles; tile += pairs, it++) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, group_m, tm, tn);
      const int m0 = (CTAS * tm + rank) * BM, first = m0 + quarter * 32, buf = it & 1;
      bool ok = tma::warp_wait_bounded(&tmem_full[buf], ((uint32_t)it >> 1) & 1u, abort_flag, wait_ns);
      const uint32_t acc = tmem_base + (uint32_t)buf * F::SECOND + ((uint32_t)(quarter * 32) << 16);
      const bool shares = SHARED && half == (buf ^ 1);   // the first accumulator's last columns, the second one's first
      auto shared_done = [&](int i) {
        if (SHARED && i == 0 && shares) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(hand_shared + buf * (uint32_t)sizeof(uint64_t));
        }
      };
      auto all_done = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(hand_back + buf * (uint32_t)sizeof(uint64_t));
      };
      if constexpr (DUAL) {
        float h[64];
        uint32_t a = 0;
        if (ok) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int sub = 64 * half + 32 * (buf ? i : 1 - i);
            uint32_t r[32], r2[32];
            tmem_ld32(acc + sub, r);
            tmem_ld32(acc + TN + sub, r2);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            shared_done(i);
            if (i == 1) all_done();
#pragma unroll
            for (int j = 0; j < 32; j++) h[32 * i + j] = fp8::gelu(__uint_as_float(r[j])) * __uint_as_float(r2[j]);
            const int left = N - (tn * TN + sub);
            if (left < 32) {
#pragma unroll
              for (int j = 0; j < 32; j++) h[32 * i + j] = j < left ? h[32 * i + j] : 0.f;
            }
          }
#pragma unroll
          for (int j = 0; j < 64; j++) a = max(a, fp8::magnitude(h[j]));
          if (a >= fp8::INF_BITS) {   // infinities or NaN: the scale is that of the others
            a = 0;
#pragma unroll
            for (int j = 0; j < 64; j++) {
              h[j] = fp8::nan_unless_finite(h[j]);
              a = max(a, h[j] == h[j] ? fp8::magnitude(h[j]) : 0u);
            }
          }
        }
        // the other half's maximum; a warp that gave up still comes here, and then both leave
        uint32_t* maxima = reinterpret_cast<uint32_t*>(blocks) + buf * 256 + quarter * 64;
        maxima[half * 32 + lane] = ok ? a : 0xffffffffu;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        const uint32_t other = maxima[(half ^ 1) * 32 + lane];
        if (!ok || other == 0xffffffffu) break;
        const uint32_t b = fp8::scale_byte(max(a, other));
        const float inv = fp8::inverse_scale(b);
        const int row = first + lane, hblocks = fp8::blocks_of(N), hgroups = fp8::groups_of(N);
        if (row < M) {
          unsigned char* to = out.hq + (size_t)row * hblocks * fp8::BLOCK + tn * TN + 64 * half;
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int sub = 32 * (buf ? i : 1 - i);
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
              w[j] = fp8::pack4(h[32 * i + 4 * j] * inv, h[32 * i + 4 * j + 1] * inv, h[32 * i + 4 * j + 2] * inv, h[32 * i + 4 * j + 3] * inv);
            *reinterpret_cast<uint4*>(to + sub) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(to + sub + 16) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
        if (half == 0 && row < ((M + 127) & ~127)) {   // byte 0 for rows and blocks that do not exist
          unsigned char* to = out.hs + fp8::scale_word(row, tn >> 2, hgroups);
          to[tn & 3] = row < M ? (unsigned char)b : 0;
          if (tn == hblocks - 1)
            for (int j = (tn & 3) + 1; j < 4; j++) to[j] = 0;
        }
      } else {
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bf16* st = reinterpret_cast<bf16*>(blocks + (warp - 2) * BLOCK_BYTES);
        auto at = [&](int row, int piece) { return st + row * 64 + ((piece ^ (row & 7)) << 3); };   // 8 values, 16 bytes
        const bool on_grid = !((out.ldy & 7) || (reinterpret_cast<uintptr_t>(out.y) & 15)) &&
                             !(out.resid && ((out.ldr & 7) || (reinterpret_cast<uintptr_t>(out.resid) & 15)));
        const int rows = min(32, M - first);   // this warp's
#pragma unroll 1
        for (int i = 0; i < TN / 128; i++) {
          const int c = 128 * (buf ? i : TN / 128 - 1 - i) + 64 * half, n = tn * TN + c;   // 64 columns
          uint32_t r[2][32];
          tmem_ld32(acc + c, r[0]);
          tmem_ld32(acc + c + 32, r[1]);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          shared_done(i);
          if (i == TN / 128 - 1) all_done();
          if (n >= N || rows <= 0) continue;
#pragma unroll
          for (int p = 0; p < 8; p++) {
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = __uint_as_float(r[p >> 2][(p & 3) * 8 + j]);
            store_vec(at(lane, p), o);
          }
          __syncwarp();
          // whole lines: 8 lanes per row, 4 rows at a time
          const int piece = lane & 7, r0 = lane >> 3, np = n + piece * 8;
          if (on_grid && n + 64 <= N) {
            bf16* yc = out.y + (size_t)(first + r0) * out.ldy + np;
            uint4 v[8];
            if (out.resid) {
              const bf16* rc = out.resid + (size_t)(first + r0) * out.ldr + np;
#pragma unroll
              for (int j = 0; j < 8; j++)
                v[j] = r0 + 4 * j < rows ? *reinterpret_cast<const uint4*>(rc + (size_t)(4 * j) * out.ldr) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (r0 + 4 * j < rows) {
                const uint4 mine = *reinterpret_cast<const uint4*>(at(r0 + 4 * j, piece));
                if (out.resid) {
                  float o[8], s[8];
                  load_vec(reinterpret_cast<const bf16*>(&mine), o);
                  load_vec(reinterpret_cast<const bf16*>(&v[j]), s);
#pragma unroll
                  for (int e = 0; e < 8; e++) o[e] += s[e];
                  store_vec(yc + (size_t)(4 * j) * out.ldy, o);
                } else {
                  *reinterpret_cast<uint4*>(yc + (size_t)(4 * j) * out.ldy) = mine;
                }
              }
          } else {   // off the 16-byte grid, or the last columns: single values, 32 columns side by side
#pragma unroll 1
            for (int e = lane; e < min(64, N - n); e += 32)
#pragma unroll 4
              for (int j = 0; j < rows; j++) {
                float v = __bfloat162float(at(j, e >> 3)[e & 7]);
                if (out.resid) v += __bfloat162float(out.resid[(size_t)(first + j) * out.ldr + n + e]);
                out.y[(size_t)(first + j) * out.ldy + n + e] = __float2bfloat16_rn(v);
              }
          }
          __syncwarp();   // the block has been read
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncwarp();
  __syncthreads();
  if constexpr (PAIR) {
    if (threadIdx.x == 0 && *abort_flag) {   // tell the other CTA
      store_to_cta(abort_flag + 1, rank ^ 1, 1);
      asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
    __syncwarp();
    pair_sync();   // neither CTA leaves while the other's instructions, copies' barriers or arrivals still use its memory
  }
  if (abort_flag[0] || abort_flag[1]) {
    // A wait ran out: report it, and let copies that were issued but never consumed land (bounded) before shared memory is released.
    if (rank == 0 && threadIdx.x == 0) {
      if (status) atomicExch(status, 3);
      const int issued = PAIR ? max(*issued_ctr, (int)load_from_cta(issued_ctr, 1)) : *issued_ctr, consumed = *consumed_ctr;
      const uint64_t start = tma::global_ns();
      for (int g = consumed; g < issued; g++) {
        for (uint32_t w = 0; w < WAIT_LIMIT; ++w) {
          if (tma::mbar_try_wait(&full_bar[g % STAGES], (uint32_t)(g / STAGES) & 1u)) break;
          if ((w & 255u) == 255u && tma::global_ns() - start > wait_ns) break;
        }
      }
    }
    __syncwarp();
    if constexpr (PAIR) pair_sync();
    else __syncthreads();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(F::TMEM_COLS));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(F::TMEM_COLS));
  }
}

// ---------------------------------------------------------------------------------------------- host
// Tensor maps are an address and a shape: kept per thread (encoding one takes a microsecond, a launch needs up to six).
struct MapKey {
  const void* base;
  long long rows, cols;
  int box;   // rows of a box; scales: -1 or -2, pieces of a box
  bool operator==(const MapKey& o) const { return base == o.base && rows == o.rows && cols == o.cols && box == o.box; }
};
struct MapSlot {
  MapKey key;
  CUtensorMap map;
  bool used;
};
constexpr int MAP_SLOTS = 1024;

int encode(CUtensorMap* map, const MapKey& k) {
  const tma::EncodeTiledFn fn = tma::encode_fn();
  if (!fn) return STU_ERR_UNSUPPORTED;
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r;
  if (k.box > 0) {   // values: boxes of a k-block
    const cuuint64_t dims[2] = {(cuuint64_t)fp8::blocks_of((int)k.cols) * fp8::BLOCK, (cuuint64_t)k.rows}, strides[1] = {dims[0]};
    const cuuint32_t box[2] = {BK, (cuuint32_t)k.box};
    r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(k.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {           // scales: [128 rows][512 columns][512 bytes]
    const cuuint64_t groups = (cuuint64_t)fp8::groups_of((int)k.cols);
    const cuuint64_t dims[3] = {fp8::PIECE / 4, groups, (cuuint64_t)(k.rows + 127) / 128}, strides[2] = {fp8::PIECE, fp8::PIECE * groups};
    const cuuint32_t box[3] = {fp8::PIECE / 4, 1, (cuuint32_t)-k.box};
    r = fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<void*>(k.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  return r == CUDA_SUCCESS ? STU_OK : STU_ERR_UNSUPPORTED;
}
int map_of(CUtensorMap* map, const void* base, long long rows, long long cols, int box) {
  static thread_local MapSlot* table = nullptr;
  if (!table) table = new (std::nothrow) MapSlot[MAP_SLOTS]();
  const MapKey key{base, rows, cols, box};
  if (!table) return encode(map, key);
  const unsigned long long h = (unsigned long long)(uintptr_t)base * 0x9E3779B97F4A7C15ull + (unsigned long long)rows * 0xC2B2AE3D27D4EB4Full +
                               (unsigned long long)cols * 0x165667B19E3779F9ull + (unsigned long long)(long long)box * 0x27D4EB2F165667C5ull;
  MapSlot& slot = table[(h >> 20) % MAP_SLOTS];
  if (!(slot.used && slot.key == key)) {
    const int rc = encode(&slot.map, key);
    slot.used = rc == STU_OK;
    if (rc != STU_OK) return rc;
    slot.key = key;
  }
  *map = slot.map;
  return STU_OK;
}

// Pairs of CTAs that the current device runs at a time.
template <bool DUAL, int CTAS, int TN> int device_clusters() {
  static std::atomic<int> found[STU_MAX_DEVICES] = {};
  int dev = 0;
  if (CTAS == 1 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= STU_MAX_DEVICES) return device_sm_count() / CTAS;
  int n = found[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS * device_sm_count());
    cfg.blockDim = dim3(64 + 32 * EPI_WARPS);
    cfg.dynamicSmemBytes = Form<DUAL, CTAS, TN>::SMEM;
    if (cudaOccupancyMaxActiveClusters(&n, fp8_gemm_kernel<DUAL, CTAS, TN>, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = device_sm_count() / CTAS;
    }
    found[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <bool DUAL, int CTAS, int TN>
int launch(const Fp8Product& p, cudaStream_t st) {
  using F = Form<DUAL, CTAS, TN>;
  static SmemLimit limit;
  cudaError_t e = allow_smem((const void*)fp8_gemm_kernel<DUAL, CTAS, TN>, F::SMEM, limit);
  if (e != cudaSuccess) return (int)e;
  const int b_box = DUAL ? TN : F::B_ROWS, s_box = DUAL ? -1 : -((TN + 127) / 128);
  CUtensorMap a, b, b2, sa, sb, sb2;
  int rc = map_of(&a, p.x, p.M, p.K, BM);
  if (!rc) rc = map_of(&b, p.w, p.N, p.K, b_box);
  if (!rc) rc = map_of(&sa, p.xs, p.M, p.K, -1);
  if (!rc) rc = map_of(&sb, p.ws, p.N, p.K, s_box);
  b2 = b, sb2 = sb;
  if (DUAL) {
    if (!rc) rc = map_of(&b2, p.w2, p.N, p.K, b_box);
    if (!rc) rc = map_of(&sb2, p.w2s, p.N, p.K, s_box);
  }
  if (rc) return rc;
  const int tiles_m = (p.M + CTAS * BM - 1) / (CTAS * BM), tiles_n = (p.N + TN - 1) / TN, most = device_clusters<DUAL, CTAS, TN>();
  const long long tiles = (long long)tiles_m * tiles_n;
  if (tiles > INT32_MAX / 2) return STU_ERR_SHAPE;
  const Out out{p.y, p.ldy, p.resid, p.ldr, p.hq, p.hs};
  e = launch_maybe_overlapped(fp8_gemm_kernel<DUAL, CTAS, TN>, dim3(CTAS * (unsigned)(tiles < most ? tiles : most)), dim3(64 + 32 * EPI_WARPS), F::SMEM, st, true,
                              a, b, b2, sa, sb, sb2, p.M, p.N, p.K, tiles_m, tiles_n, tiles_m < 8 ? tiles_m : 8, out, device_status_word(),
                              (int)take_dropped_stage(), wait_bound_ns());
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

int fp8_gemm(const Fp8Product& p, cudaStream_t st) {
  if (p.w2) return p.M > BM ? launch<true, 2, 128>(p, st) : launch<true, 1, 128>(p, st);
  if (p.M <= BM) return launch<false, 1, 128>(p, st);
  return p.N > 128 ? launch<false, 2, 256>(p, st) : launch<false, 2, 128>(p, st);
}

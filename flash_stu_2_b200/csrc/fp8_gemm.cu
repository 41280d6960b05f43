// Products of two e4m3 operands with a scale for each 128 of a row (fp8.cuh) on the 5th-generation tensor cores: D[M,N] = x[M,K] . W[N,K]^T,
// fp32 sums in tensor memory.
//
// kind::mxf8f6f4 multiplies every 32 columns of a row by a power of two that it finds in tensor memory.  The scales of 128 rows and four blocks of
// 128 columns are one 32-bit word per row, 512 bytes in the order that tcgen05.cp takes: they come by TMA with every fourth k-block, one thread
// copies them over, and the four instructions of a k-block take the byte that their descriptor names.  So no sum ever passes a register
// before its epilogue.
//
// A pair of CTAs on neighbouring SMs computes tiles of 256 x 256 (gate/up: 256 x 128 of both) with cta_group::2, or a CTA alone tiles of 128
// rows where those would leave SMs idle.  A thread of warp 0 of a CTA is its TMA producer, one of warp 1 of the first CTA issues scale copies and instructions,
// warps 2..9 drain the accumulators.  (The tensor core takes few instructions ahead: what the issuer does between two stages is time that it may stand still, and the
// arithmetic of the other warps draws it out.  Whole warps that agree on every wait and issue by a lane: 16384 x 6144 x 1536 gate/up 250 us, so 230; 2048 x 4096 x
// 1024 20.5, so 18.4.)  The kernel is persistent; two accumulators of 256 columns and the scales do not fit 512 columns, so the accumulators
// share 32 columns: the epilogue reads those first and hands them back ahead of the rest.
//
// gate/up: a thread has 64 of the 128 features of a block of its row, two warps settle the block's scale through shared memory, and the row
// leaves in 8 bits.
//
// Sums: the tensor core cuts what it adds off towards zero, so that they are short by a few 2^-24 (K = 18432: some 10^-6) of the magnitudes in them where rounded fp32 sums
// would be off to either side.  Of a gate/up product's 8-bit results (16384 x 6144 x 1536) 5 in a million are the neighbour of the right one for it, 20 with fp32 sums and
// the tanh form; where a block's largest value is that close to a scale's border, the block can have the other scale (one of 5.5 million).  bf16 results that are not the
// nearest, here and with rounded fp32 sums: K = 1536 6 and 5 in 100,000, 6144 31 and 8, 18432 109 and 18.
//
// Every wait is bounded, as in gemm_tc.cu: on expiry the waiter tells the others, raises the status word, and the CTAs drain their copies, free
// their tensor memory and return.
#include <memory>
#include <new>

#include "fp8_gemm.cuh"

int device_sm_count();      // gemm_tc.cu
int* device_status_word();  // gemm_tc.cu

using namespace fp8;

namespace {

constexpr int EPI_WARPS = 8, BLOCK_BYTES = 32 * 32 * 2;   // an epilogue warp's block of 32 rows x 32 bf16 columns

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
  // A stage is one k-block.  (Of two, which the producer and the issuer are done with in less time, a pair has room for three, and one of those is on its
  // way: 8192 x 8192 x 8192 369 us, so 358; 4096 x 6144 x 1536 gate/up 67, so 61.)
  static constexpr int TILE_BYTES = A_BYTES + B_ROWS * BK;             // of one CTA
  static constexpr int SCALE_BYTES = fp8::PIECE * (1 + (MMA_N + 127) / 128);
  static constexpr int STAGES = (227 * 1024 - 2048 - (DUAL ? 2048 : EPI_WARPS * BLOCK_BYTES)) / (TILE_BYTES + SCALE_BYTES);
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
    if (elect_one()) {
      // ---------------- TMA producer, one thread (of either CTA: its 128 rows of x, its part of the rows of W, the scales of both)
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
          if (!ready) ok = tma::mbar_wait_bounded(&empty_bar[s], ph, abort_flag, wait_ns);
          if (!ok) break;
          const int s1 = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t ph1 = s1 ? ph : ph ^ 1u;
          const bool ready1 = mbar_ready(&empty_bar[s1], ph1);   // asked for here, looked at behind the copies
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
          ready = ready1;
          s = s1, ph = ph1;
        }
      }
      *issued_ctr = g;
      // the last stages' releases arrive in both CTAs: wait for them here, so that none is under way to a CTA that has left
      for (int h = max(g - STAGES, 0); ok && h < g; h++)
        ok = tma::mbar_wait_bounded(&empty_bar[h % STAGES], (uint32_t)(h / STAGES) & 1u, abort_flag, wait_ns);
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      // ---------------- issuer of the pair: one thread
      const uint64_t da0 = operand_desc(tma::smem_u32(smem)), db0 = operand_desc(tma::smem_u32(smem) + A_BYTES);
      const uint64_t ds0 = scales_desc(tma::smem_u32(scales));
      int g = 0, s = 0, it = 0, pieces = 0;
      uint32_t ph = 0, sf_cols = tmem_base + F::SCALES;
      bool ok = true, ready = false;
      for (int tile = pair; ok && tile < num_tiles; tile += pairs, it++) {
        const int buf = it & 1;
        const uint32_t acc = tmem_base + (uint32_t)buf * F::SECOND;
        ok = tma::mbar_wait_bounded(&tmem_empty[buf], (((uint32_t)it >> 1) & 1u) ^ 1u, abort_flag, wait_ns);
        if (SHARED && ok && it > 0) ok = tma::mbar_wait_bounded(&shared_read[buf ^ 1], ((uint32_t)(it - 1) >> 1) & 1u, abort_flag, wait_ns);
        if (!ok) break;
        for (int kb = 0; kb < num_kb; kb++, g++) {
          if (!ready) ok = tma::mbar_wait_bounded(&full_bar[s], ph, abort_flag, wait_ns);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int s1 = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t ph1 = s1 ? ph : ph ^ 1u;
          const bool ready1 = mbar_ready(&full_bar[s1], ph1);
          if ((kb & 3) == 0) sf_cols = tmem_base + F::SCALES + 16 * (pieces++ & 1);
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
          ready = ready1;
          s = s1, ph = ph1;
        }
        if (ok) commit<CTAS>(&tmem_full[buf]);
      }
      *consumed_ctr = g;
    }
  } else {
    // ---------------- epilogue warps: TMEM lane quarter = warp % 4 (32 rows), half of the columns
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t hand_back = in_first_cta(tmem_empty), hand_shared = in_first_cta(shared_read);
    const bool on_grid = !((out.ldy & 7) || (reinterpret_cast<uintptr_t>(out.y) & 15)) &&
                         !(out.resid && ((out.ldr & 7) || (reinterpret_cast<uintptr_t>(out.resid) & 15)));
    int it = 0;
    for (int tile = pair; tile < num_tiles; tile += pairs, it++) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, group_m, tm, tn);
      const int m0 = (CTAS * tm + rank) * BM, first = m0 + quarter * 32, buf = it & 1;
      // plain: a half's columns, 64 of every 128, in SUBS blocks of 32; a block's residuals (four vectors, or 32 rows' values of a column), asked for ahead of its
      // sums (3000 x 1111 x 1000 off the 16-byte grid, behind them and with loads and stores in turn 25.3 us, so 17.2; on it 700 rows 10.1, so 9.2)
      constexpr int SUBS = TN / 64;
      const int rows = min(32, M - first);   // this warp's
      const int piece = lane & 3, r0 = lane >> 2;   // 64 bytes of a row by 4 lanes, 8 rows at a time
      const auto column = [&](int i) {
        const int sub = buf ? i : SUBS - 1 - i;
        return 128 * (sub >> 1) + 64 * half + 32 * (sub & 1);
      };
      uint32_t v[32];
      const auto ask = [&](int i) {
        const int n = tn * TN + column(i);
        if (on_grid && n + 32 <= N) {
          const bf16* rc = out.resid + (size_t)(first + r0) * out.ldr + n + piece * 8;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint4 u = r0 + 8 * j < rows ? *reinterpret_cast<const uint4*>(rc + (size_t)(8 * j) * out.ldr) : make_uint4(0, 0, 0, 0);
            v[4 * j] = u.x, v[4 * j + 1] = u.y, v[4 * j + 2] = u.z, v[4 * j + 3] = u.w;
          }
        } else {
          const uint16_t* rc = reinterpret_cast<const uint16_t*>(out.resid) + (size_t)first * out.ldr + n + lane;
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = n + lane < N && j < rows ? rc[(size_t)j * out.ldr] : 0u;
        }
      };
      if (!DUAL && out.resid) ask(0);
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
            // The arithmetic behind the arrivals, not between loads and arrivals, where the compiler would put it and the issuer would wait for it at every tile
            // (16384 x 6144 x 1536 in a loop 287 us, so 254; in bursts 244, so 227).
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; j++) asm volatile("" : "+r"(r[j]), "+r"(r2[j]));
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
        auto at = [&](int row, int p) { return st + row * 32 + ((p ^ ((row >> 1) & 3)) << 3); };   // 8 values, 16 bytes
#pragma unroll 1
        for (int i = 0; i < SUBS; i++) {
          const int c = column(i), n = tn * TN + c;
          uint32_t r[32];
          tmem_ld32(acc + c, r);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          shared_done(i);
          if (i == SUBS - 1) all_done();
          if (n < N && rows > 0) {
#pragma unroll
            for (int p = 0; p < 4; p++) {
              float o[8];
#pragma unroll
              for (int j = 0; j < 8; j++) o[j] = __uint_as_float(r[p * 8 + j]);
              store_vec(at(lane, p), o);
            }
            __syncwarp();
            // (what is read of the block is read ahead of the first store: that might be to it, for all that the compiler knows)
            if (on_grid && n + 32 <= N) {
              bf16* yc = out.y + (size_t)(first + r0) * out.ldy + n + piece * 8;
              uint4 mine[4];
#pragma unroll
              for (int j = 0; j < 4; j++) mine[j] = *reinterpret_cast<const uint4*>(at(r0 + 8 * j, piece));
              if (out.resid) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  float o[8], s[8];
                  load_vec(reinterpret_cast<const bf16*>(&mine[j]), o);
                  load_vec(reinterpret_cast<const bf16*>(&v[4 * j]), s);
#pragma unroll
                  for (int e = 0; e < 8; e++) o[e] += s[e];
                  store_vec(reinterpret_cast<bf16*>(&mine[j]), o);
                }
              }
#pragma unroll
              for (int j = 0; j < 4; j++)
                if (r0 + 8 * j < rows) *reinterpret_cast<uint4*>(yc + (size_t)(8 * j) * out.ldy) = mine[j];
            } else {   // off the 16-byte grid, or the last columns: single values, side by side
              uint16_t* yc = reinterpret_cast<uint16_t*>(out.y) + (size_t)first * out.ldy + n + lane;
              uint16_t mine[32];
#pragma unroll
              for (int j = 0; j < 32; j++) mine[j] = reinterpret_cast<const uint16_t*>(at(j, lane >> 3))[lane & 7];
              if (out.resid) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                  mine[j] = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float((uint32_t)mine[j] << 16) + __uint_as_float(v[j] << 16)));
              }
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (n + lane < N && j < rows) yc[(size_t)j * out.ldy] = mine[j];
            }
          }
          if (out.resid && i + 1 < SUBS) ask(i + 1);
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
// Tensor maps are an address and a shape, whatever lies there: kept per thread (encoding one takes a microsecond, a launch needs up to six).
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
}  // namespace

int fp8_tensor_map(CUtensorMap* map, const void* base, long long rows, long long cols, int box) {
  static thread_local std::unique_ptr<MapSlot[]> table;
  if (!table) table.reset(new (std::nothrow) MapSlot[MAP_SLOTS]());
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

namespace {

template <bool DUAL, int CTAS, int TN> cudaError_t allow_shared() {
  static SmemLimit limit;
  return allow_smem((const void*)fp8_gemm_kernel<DUAL, CTAS, TN>, Form<DUAL, CTAS, TN>::SMEM, limit);
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
    if (allow_shared<DUAL, CTAS, TN>() != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, fp8_gemm_kernel<DUAL, CTAS, TN>, &cfg) != cudaSuccess || n < 1) {
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
  cudaError_t e = allow_shared<DUAL, CTAS, TN>();
  if (e != cudaSuccess) return (int)e;
  const int b_box = DUAL ? TN : F::B_ROWS, s_box = DUAL ? -1 : -((TN + 127) / 128);
  CUtensorMap a, b, b2, sa, sb, sb2;
  int rc = fp8_tensor_map(&a, p.x, p.M, p.K, BM);
  if (!rc) rc = fp8_tensor_map(&b, p.w, p.N, p.K, b_box);
  if (!rc) rc = fp8_tensor_map(&sa, p.xs, p.M, p.K, -1);
  if (!rc) rc = fp8_tensor_map(&sb, p.ws, p.N, p.K, s_box);
  b2 = b, sb2 = sb;
  if (DUAL) {
    if (!rc) rc = fp8_tensor_map(&b2, p.w2, p.N, p.K, b_box);
    if (!rc) rc = fp8_tensor_map(&sb2, p.w2s, p.N, p.K, s_box);
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
  const auto waves = [&](int rows, int cols, int room) {
    return ((long long)((p.M + rows - 1) / rows) * ((p.N + cols - 1) / cols) + room - 1) / room;
  };
  // Gate/up: a CTA alone on 128 rows where that is fewer rounds than pairs on 256 (us, alone and in pairs: 128 x 18432 x 1536 14.1 and 15.7, 333 x 6144 x 1536
  // 11.0 and 14.5, 700 16.1 and 14.9, 1024 21.3 and 19.1, 2048 37.6 and 33.3).
  if (p.w2)
    return waves(128, 128, device_sm_count()) < waves(256, 128, device_clusters<true, 2, 128>()) ? launch<true, 1, 128>(p, st) : launch<true, 2, 128>(p, st);
  // Plain: tiles of 128 columns where a round of them, about 3/4 of the time of one of 256, makes up for their number (us, 128 and 256 columns:
  // 1024 x 1536 x 18432 34.7 and 47.3, 1024 x 1536 x 6144 15.2 and 20.2, 2048 x 1536 x 6144 24.4 and 21.9, 1024 x 8192 x 2048 20.2 and 17.9).
  return 3 * waves(256, 128, device_clusters<false, 2, 128>()) < 4 * waves(256, 256, device_clusters<false, 2, 256>()) ? launch<false, 2, 128>(p, st)
                                                                                                                     : launch<false, 2, 256>(p, st);
}

// Products of 8-bit rows (fp8.cuh) for few tokens: the weights are the 128-row operand of the tensor core, the tokens its columns, and K is cut over a
// thread-block cluster so that a few thousand features occupy all SMs.  What bounds it: HBM, the weights once; for small weights the time
// from a launch over the first bytes and the cluster's meeting to the last store.
//
// A thread of warp 0 of a CTA brings 128 features (gate/up: 128 of both), NT tokens and their scales by TMA into a ring, one of warp 1 copies the scales into tensor
// memory and issues kind::mxf8f6f4 (see fp8_gemm.cu), the others drain the sums and send each to the CTA of the cluster whose share its token is in, where it
// counts towards a barrier.  A warp there adds up a token's 128 features over the cluster, in the order of K, and stores them; gate/up: one warp has the whole
// block of h and settles its scale by a reduction.  The cluster meets once, behind the set-up and unnoticed (Mode: or behind the products); a CTA alone passes its sums on in shared memory.  (Sums left in shared memory and fetched between two meetings of the cluster
// took 700 and 600 ns for those and 1000 for the rest: 1 x 1024 x 4096 4.7 us, so 3.8; gate/up 1 x 4096 x 1024 5.8, so 5.1; 128 x 1536 x 6144 9.2, so 8.6; but 333 tokens, whose
// sends are many, 12.1, so 12.3.  Sent by bulk copies of staged rows 5.2.)  On mma.sync the conversions to halves and the fragments of tokens took 370 instructions for 2 KB of
// weights, more than an SM issues in the time that they take to arrive: 18432 x 1536 gate/up of 8 tokens 25.5 us.
#include <cooperative_groups.h>

#include "fp8_gemm.cuh"

namespace cg = cooperative_groups;
using namespace fp8;

int device_sm_count();      // gemm_tc.cu
int* device_status_word();  // gemm_tc.cu

namespace {

constexpr int MAX_STAGES = 12, MAX_KS = 8;

// Where sums go.  ALONE (K is not cut): where the CTA's ring was, so that two CTAs fit an SM.  EARLY: they come while the ring may still be in use, to memory of their own; the
// cluster has met ahead of the products.  LATE, for 128 tokens, whose sums would leave a ring of four k-blocks instead of three stages of two: where the ring was, behind a meeting of CTAs that are
// done with theirs.  (us, early with stages of one, and late, by k-blocks of a CTA: 6 of 128 x 1536 x 6144 8.7 and 9.15, 8 of 512 x 1024 x 4096 9.85 and 10.2, 16 of 333 x 1536 x 6144 12.25 and
// 12.15, 24 of 512 x 1536 x 6144 15.3 and 14.8, 72 of 512 x 1536 x 18432 29.4 and 26.9.)
enum Mode { ALONE, EARLY, LATE };

template <bool DUAL, int NT, Mode MODE> struct Narrow {
  static constexpr int WS = DUAL ? 2 : 1;                           // matrices
  static constexpr int DRAIN = NT >= 64 ? 8 : 4, THREADS = 64 + 32 * DRAIN;   // warps that read the sums
  // k-blocks of a stage: waiting for one, announcing its bytes and sending off its copies takes the producer 360 cycles and 27 more per copy, whatever
  // their size, so that single blocks of 16 KB came at 45 bytes a cycle at most (8 x 1536 x 18432 13.7 us, 66 with K whole);
  // where blocks are of 32 KB and the sums that come from elsewhere leave room for few, stages of one (32 x 6144 x 1536 gate/up 10.0 us, so 9.75)
  static constexpr int KBS = DUAL ? (NT <= 16 ? 2 : 1) : NT <= 32 ? 4 : NT <= 64 || MODE == LATE ? 2 : 1;
  static constexpr int W_BYTES = WS * A_BYTES, X_BYTES = NT * BK, KB_BYTES = W_BYTES + X_BYTES;
  static constexpr int SCALE_BYTES = PIECE * (WS + 1);
  static constexpr int STAGE = KBS * KB_BYTES + SCALE_BYTES;        // (the scales of all stages lie behind the tiles)
  static constexpr int ROWS = WS * 128;                             // sums of a token
  static constexpr int SUM_BYTES = (NT + MAX_KS) * ROWS * 4;        // room for a CTA's share of the tokens, from each of the cluster
  static constexpr int SF_COLS = 4 * (WS + 1), SCALES = WS * NT;    // tensor memory: sums, then twice the scales
  static constexpr uint32_t TMEM_COLS = SCALES + 2 * SF_COLS <= 64 ? 64 : SCALES + 2 * SF_COLS <= 128 ? 128 : SCALES + 2 * SF_COLS <= 256 ? 256 : 512;
};
constexpr int TAIL = (2 * MAX_STAGES + 2) * 8 + 32;                 // barriers, tensor memory's address, marks
template <bool DUAL, int NT, Mode MODE> __host__ __device__ constexpr int before_tail(int stages) {
  const int ring = stages * Narrow<DUAL, NT, MODE>::STAGE, sums = Narrow<DUAL, NT, MODE>::SUM_BYTES;
  return MODE == EARLY ? ring + sums : ring > sums ? ring : sums;
}
template <bool DUAL, int NT, Mode MODE> constexpr size_t smem_bytes(int stages) { return 1024 + (size_t)before_tail<DUAL, NT, MODE>(stages) + TAIL; }

// A value to CTA `to` of the cluster, where it counts towards what the barrier expects.
__device__ __forceinline__ void send(uint32_t addr, uint32_t bar, int to, uint32_t v) {
  asm volatile("{\n\t.reg .b32 a, b;\n\tmapa.shared::cluster.u32 a, %0, %2;\n\tmapa.shared::cluster.u32 b, %1, %2;\n\t"
               "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [a], %3, [b];\n\t}"
               ::"r"(addr), "r"(bar), "r"(to), "r"(v) : "memory");
}
__device__ __forceinline__ void meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Behind a wait for the barrier: what other CTAs stored before they arrived is seen.
__device__ __forceinline__ void acquire_cluster(uint64_t* bar) {
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%0], 0;\n\t}" ::"r"(tma::smem_u32(bar)) : "memory");
}

template <bool DUAL, int NT, Mode MODE>
__global__ void __launch_bounds__(Narrow<DUAL, NT, MODE>::THREADS, 1)
    fp8_narrow_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW2, const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ CUtensorMap tmSW, const __grid_constant__ CUtensorMap tmSW2, const __grid_constant__ CUtensorMap tmSX,
                      const bf16* resid, long long ldr, bf16* y, long long ldy, unsigned char* hq, unsigned char* hs, int M, int N, int K, int stages,
                      int overlap, int* status, int drop_first_copy, unsigned long long wait_ns) {
  using C = Narrow<DUAL, NT, MODE>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int TILES = C::KBS * C::KB_BYTES, KBS = C::KBS, THREADS = C::THREADS;
  unsigned char* scales = smem + stages * TILES;
  cg::cluster_group cluster = cg::this_cluster();
  const int ks = MODE == ALONE ? 1 : cluster.num_blocks(), rank = MODE == ALONE ? 0 : cluster.block_rank();
  float* sums = reinterpret_cast<float*>(smem + (MODE == EARLY ? stages * C::STAGE : 0));   // [this CTA's tokens][CTA that they come from][feature], gate/up: 128 gate, 128 up
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + before_tail<DUAL, NT, MODE>(stages));
  uint64_t* empty_bar = full_bar + MAX_STAGES;
  uint64_t* tmem_full = empty_bar + MAX_STAGES;
  uint64_t* received = tmem_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* issued_ctr = reinterpret_cast<int*>(tmem_slot + 2);
  int* consumed_ctr = issued_ctr + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nb = blockIdx.x, t0 = blockIdx.z * NT, num_kb = blocks_of(K), last = min(NT, M - t0);   // tokens of this tile
  const int owned = max(last - rank + ks - 1, 0) / ks;   // of these tokens, every ks-th is this CTA's to add up
  // this CTA's k-blocks, in stages that begin at multiples of KBS: none reaches over a group of four, whose scales are a piece
  const int kb0 = (int)((long long)num_kb * rank / ks), kb_end = (int)((long long)num_kb * (rank + 1) / ks), st0 = kb0 / KBS;
  const int nst = kb_end > kb0 ? (kb_end - 1) / KBS - st0 + 1 : 0;
  const auto first_kb = [&](int g) { return max(kb0, (st0 + g) * KBS); };
  const auto blocks_in = [&](int g) { return min(kb_end, (st0 + g + 1) * KBS) - first_kb(g); };
  const auto with_scales = [&](int g) { return g == 0 || (first_kb(g) & 3) == 0; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      tma::mbar_init(&full_bar[s], 1);
      tma::mbar_init(&empty_bar[s], 1);
    }
    tma::mbar_init(tmem_full, 1);
    tma::mbar_init(received, 1);
    *abort_flag = 0;
    *issued_ctr = *consumed_ctr = 0;
    tma::fence_barrier_init();
    tma::mbar_expect_tx(received, MODE == ALONE ? 0 : owned * ks * C::ROWS * 4);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_u32(tmem_slot)), "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  if (MODE == EARLY) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // sums may come
  // (when the next kernel may start: epilogue.cuh, PdlTrigger)
  if (overlap && !DUAL) pdl_trigger();

  if (warp == 0) {
    // ---------------- TMA producer: one thread (the whole warp waits for the kernel in front)
    const bool leader = elect_one();
    const auto load_w = [&](int g, int s) {
      const int kb = first_kb(g), n = blocks_in(g);
      unsigned char *tile = smem + s * TILES, *sc = scales + s * C::SCALE_BYTES;
#pragma unroll
      for (int j = 0; j < KBS; j++)
        if (j < n) {
          load_2d(tile + j * C::KB_BYTES, &tmW, &full_bar[s], (kb + j) * BK, nb * 128);
          if (DUAL) load_2d(tile + j * C::KB_BYTES + A_BYTES, &tmW2, &full_bar[s], (kb + j) * BK, nb * 128);
        }
      if (with_scales(g)) {
        tma::load_3d(sc, &tmSW, &full_bar[s], 0, kb >> 2, nb);
        if (DUAL) tma::load_3d(sc + PIECE, &tmSW2, &full_bar[s], 0, kb >> 2, nb);
      }
    };
    const auto load_x = [&](int g, int s) {
      const int kb = first_kb(g), n = blocks_in(g);
#pragma unroll
      for (int j = 0; j < KBS; j++)
        if (j < n) load_2d(smem + s * TILES + j * C::KB_BYTES + C::W_BYTES, &tmX, &full_bar[s], (kb + j) * BK, t0);
      if (with_scales(g)) tma::load_3d(scales + s * C::SCALE_BYTES + C::WS * PIECE, &tmSX, &full_bar[s], 0, kb >> 2, t0 / 128);
    };
    const auto expect = [&](int g, int s) { tma::mbar_expect_tx(&full_bar[s], blocks_in(g) * C::KB_BYTES + (with_scales(g) ? C::SCALE_BYTES : 0)); };
    // the first round's weights, ahead of the wait where that is allowed
    const int pre = min(stages, nst);
    if (!overlap) pdl_wait();
    const int first = drop_first_copy ? 1 : 0;   // (failure-detection test: the first stage never fills)
    if (leader) {
      for (int g = 0; g < pre; g++) {
        expect(g, g);
        if (g >= first) load_w(g, g);
      }
    }
    __syncwarp();
    if (overlap) pdl_wait();
    if (!overlap || DUAL) pdl_trigger();
    if (leader) {
      for (int g = first; g < pre; g++) load_x(g, g);
      int g = pre, s = pre == stages ? 0 : pre;
      uint32_t ph = 0;   // of the stage's first release
      for (; g < nst; g++) {
        if (!tma::mbar_wait_bounded(&empty_bar[s], ph, abort_flag, wait_ns)) break;
        expect(g, s);
        load_w(g, s);
        load_x(g, s);
        if (++s == stages) s = 0, ph ^= 1u;
      }
      *issued_ctr = g;
    }
  } else if (warp == 1) {
    if (elect_one()) {
      // ---------------- issuer: one thread
      const uint64_t dw0 = operand_desc(tma::smem_u32(smem)), dx0 = operand_desc(tma::smem_u32(smem) + C::W_BYTES), ds0 = scales_desc(tma::smem_u32(scales));
      int g = 0, s = 0, pieces = 0;
      uint32_t ph = 0, sf = tmem_base + C::SCALES;
      for (; g < nst; g++) {
        if (!tma::mbar_wait_bounded(&full_bar[s], ph, abort_flag, wait_ns)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int kb = first_kb(g), n = blocks_in(g);
        const bool copy = with_scales(g);
        if (copy) sf = tmem_base + C::SCALES + C::SF_COLS * (pieces++ & 1);
        if (copy) {   // in order with the instructions around it
#pragma unroll
          for (int i = 0; i <= C::WS; i++) copy_scales<1>(sf + 4 * i, ds0 + (uint64_t)((s * C::SCALE_BYTES + i * PIECE) >> 4));
        }
        const uint64_t dw = dw0 + (uint64_t)(s * (TILES >> 4)), dx = dx0 + (uint64_t)(s * (TILES >> 4));
#pragma unroll
        for (int j = 0; j < KBS; j++)
          if (j < n) {
#pragma unroll
            for (int kk = 0; kk < BK / 32; kk++)
#pragma unroll
              for (int i = 0; i < C::WS; i++)
                multiply<1, NT>(tmem_base + i * NT, dw + ((j * C::KB_BYTES + i * A_BYTES) >> 4) + 2 * kk, dx + ((j * C::KB_BYTES) >> 4) + 2 * kk, sf + 4 * i,
                                sf + 4 * C::WS, (kb + j) & 3, (g | j | kk) ? 1u : 0u);
          }
        if (g + stages < nst) commit<1>(&empty_bar[s]);   // (nobody waits for the last round's)
        if (g + 1 == nst) commit<1>(tmem_full);
        if (++s == stages) s = 0, ph ^= 1u;
      }
      *consumed_ctr = g;
    }
  } else {
    // ---------------- drain: TMEM lane quarter = warp % 4, a feature per thread
    const int quarter = warp & 3, half = (warp - 2) >> 2;   // (eight warps: either half of the tokens)
    if (MODE == EARLY) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const bool ok = nst > 0 && tma::warp_wait_bounded(tmem_full, 0, abort_flag, wait_ns);   // (else zeros: the others count on them)
    if (MODE == LATE) meet();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float* mine = sums + rank * C::ROWS + quarter * 32 + lane;
    const uint32_t to = tma::smem_u32(mine), bar = tma::smem_u32(received);
#pragma unroll 1
    for (int i = 0; i < C::WS; i++)
#pragma unroll 1
      for (int c0 = half * (NT / 2); c0 < min(last, C::DRAIN == 8 ? (half + 1) * (NT / 2) : NT); c0 += 32) {
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < 32; c++) r[c] = 0u;
        if (ok) {   // (16 tokens: the columns behind them are other sums or scales, unread)
          tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(i * NT + c0), r);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        if constexpr (MODE == ALONE) {
#pragma unroll
          for (int c = 0; c < (NT < 32 ? NT : 32); c++)
            if (c0 + c < last) mine[(c0 + c) * C::ROWS + i * 128] = __uint_as_float(r[c]);
        } else {
          int owner = c0 % ks, at = c0 / ks;
#pragma unroll
          for (int c = 0; c < (NT < 32 ? NT : 32); c++)
            if (c0 + c < last) {
              send(to + (uint32_t)(at * ks * C::ROWS + i * 128) * 4, bar, owner, r[c]);
              if (++owner == ks) owner = 0, at++;
            }
        }
      }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncwarp();
  if (warp < 2) {
    if (MODE == LATE) meet();
    else if (MODE == EARLY) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  pdl_wait();   // (returns at once: the producer has waited; outputs and residual rows are touched behind it)
  const int hblocks = blocks_of(N), hgroups = groups_of(N);
  if (DUAL && rank == 0) {   // byte 0 for the rows that fill up the last 128 and for the blocks that fill up the last four
    const int end = nb == hblocks - 1 ? hgroups * 4 : nb + 1, bottom = min(t0 + NT, M) == M ? (M + 127) & ~127 : t0 + NT;
    for (int m = t0 + threadIdx.x; m < bottom; m += THREADS)
      for (int kb = m < M ? nb + 1 : nb; kb < end; kb++) hs[scale_word(m, kb >> 2, hgroups) + (kb & 3)] = 0;
  }
  // ---------------- this CTA's share of the cluster's sums: a warp per token, four features per lane
  bool all = true;
  if constexpr (MODE != ALONE) {
    all = tma::warp_wait_bounded(received, 0, abort_flag, 4 * wait_ns);   // (the others send by the end of their own waits)
    acquire_cluster(received);
  } else {
    __syncthreads();
  }
  for (int own = warp; all && own < owned; own += THREADS / 32) {
    const int t = rank + ks * own;
    float v[C::WS][4];
#pragma unroll
    for (int i = 0; i < C::WS; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) v[i][j] = 0.f;
#pragma unroll 4
    for (int r = 0; r < ks; r++) {
      const float* from = sums + (own * ks + r) * C::ROWS + 4 * lane;
#pragma unroll
      for (int i = 0; i < C::WS; i++) {
        const float4 a = *reinterpret_cast<const float4*>(from + i * 128);
        v[i][0] += a.x, v[i][1] += a.y, v[i][2] += a.z, v[i][3] += a.w;
      }
    }
    const int m = t0 + t, n = nb * 128 + 4 * lane;
    if constexpr (DUAL) {
      float h[4];
      uint32_t a = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        h[j] = nan_unless_finite(n + j < N ? gelu(v[0][j]) * v[1][j] : 0.f);
        a = max(a, h[j] == h[j] ? magnitude(h[j]) : 0u);
      }
      a = __reduce_max_sync(0xffffffffu, a);
      const uint32_t b = scale_byte(a);
      const float inv = inverse_scale(b);
      *reinterpret_cast<uint32_t*>(hq + (size_t)m * hblocks * BLOCK + n) = pack4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
      if (lane == 0) hs[scale_word(m, nb >> 2, hgroups) + (nb & 3)] = (unsigned char)b;
    } else {
      const size_t ry = (size_t)m * ldy + n, rr = (size_t)m * ldr + n;
#pragma unroll
      for (int j = 0; j < 4; j++) v[0][j] = round_to<bf16>(v[0][j]);
      if (n + 4 <= N && !(reinterpret_cast<uintptr_t>(y + ry) & 7) && !(resid && (reinterpret_cast<uintptr_t>(resid + rr) & 7))) {
        if (resid) {
          const uint2 s = *reinterpret_cast<const uint2*>(resid + rr);
          v[0][0] += __uint_as_float(s.x << 16), v[0][1] += __uint_as_float(s.x & 0xffff0000u);
          v[0][2] += __uint_as_float(s.y << 16), v[0][3] += __uint_as_float(s.y & 0xffff0000u);
        }
        const __nv_bfloat162 p0 = __floats2bfloat162_rn(v[0][0], v[0][1]), p1 = __floats2bfloat162_rn(v[0][2], v[0][3]);
        *reinterpret_cast<uint2*>(y + ry) = make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (n + j < N) y[ry + j] = __float2bfloat16_rn(resid ? __bfloat162float(resid[rr + j]) + v[0][j] : v[0][j]);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {
    // A wait ran out: report it, and let copies that were issued but never consumed, and the others' sums, land (bounded) before shared memory is released.
    if (MODE != ALONE) cluster.sync();   // (with those that gave up; who has left counts as here)
    if (threadIdx.x == 0) {
      if (status) atomicExch(status, 3);
      const uint64_t start = tma::global_ns();
      const auto land = [&](uint64_t* bar, uint32_t parity) {
        for (uint32_t w = 0; w < WAIT_LIMIT; ++w) {
          if (tma::mbar_try_wait(bar, parity)) break;
          if ((w & 255u) == 255u && tma::global_ns() - start > wait_ns) break;
        }
      };
      land(received, 0);
      for (int g = *consumed_ctr; g < *issued_ctr; g++) land(&full_bar[g % stages], (uint32_t)(g / stages) & 1u);
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS));
  }
}

template <bool DUAL, int NT, Mode MODE>
cudaError_t configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* at, dim3 grid, size_t smem) {
  cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(Narrow<DUAL, NT, MODE>::THREADS);
  cfg.dynamicSmemBytes = smem;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = at[0].val.clusterDim.z = 1;
  at[0].val.clusterDim.y = grid.y;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  static SmemLimit limit;
  return allow_smem((const void*)fp8_narrow_kernel<DUAL, NT, MODE>, smem, limit);
}
template <bool DUAL, int NT, Mode MODE> constexpr int deepest() {
  int stages = MAX_STAGES;
  while (stages > 2 && smem_bytes<DUAL, NT, MODE>(stages) > 227 * 1024) stages--;
  return stages;
}

// Clusters of ks CTAs with the deepest ring that the current device runs at a time (a cluster lies in one of its groups of SMs).
template <bool DUAL, int NT> int cluster_room(int ks) {
  static std::atomic<int> found[STU_MAX_DEVICES][MAX_KS + 1] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= STU_MAX_DEVICES) return 0;
  if ((n = found[dev][ks].load(std::memory_order_relaxed)) != 0) return n;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at[1];
  if (configure<DUAL, NT, EARLY>(cfg, at, dim3(1024, ks), smem_bytes<DUAL, NT, EARLY>(deepest<DUAL, NT, EARLY>())) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, fp8_narrow_kernel<DUAL, NT, EARLY>, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = -1;   // (none: K is not cut that way)
  }
  found[dev][ks].store(n, std::memory_order_relaxed);
  return n;
}
// CTAs that share a tile's K: the most whose clusters run at a time (74, 45, 33, 26, 22, 15, 15 of 2 to 8), up to 6 for plain products of up to 32 tokens whose K has fewer than 16 blocks.  us, ks = 1 / 2 /
// 4 / 6 / 8, weights from HBM: gate/up of 1 token, 4096 x 1024 (32 tiles) 5.9 / 5.3 / 5.2 / 9.4 (two rounds) / 12.8, 6144 x 1536 (48) 7.8 / 7.5 / 11.3, 18432 x 1536 (144) 13.5 / 17.6, 1000 x 1000 (8) 5.6 / 4.4 / 3.9 /
// 4.0 / 3.9; plain of 1 token, 8 k-blocks, x 1024 3.5 / 3.2 / 2.9 / 2.8 / 3.1; 12, x 1536 4.2 / 3.6 / 3.3 / 3.3 / 3.6; 20, x 1001 5.4 / 4.7 / 3.5 / 3.4 / 3.5; of 32, 32 k-blocks, x 1024 9.4 / 7.3 / 5.3 / 4.9 / 4.7; 144, x 1536
// 32.5 / 19.8 / 13.1 / 10.9 / 10.1; of 64, 8 k-blocks, x 1000 5.8 / 5.5 / 4.6 / 4.6 / 4.3.  (3, 5 and 7 lie between their neighbours.  16 tiles of 8 and 16 blocks take 5 to 13 % less with 4 than with 6.)
template <bool DUAL, int NT> int cluster_size(const Fp8Product& p) {
  const long long tiles = (long long)blocks_of(p.N) * ((p.M + NT - 1) / NT);
  const int num_kb = blocks_of(p.K), sms = device_sm_count();
  const int most = !DUAL && NT <= 32 && num_kb < 16 ? 6 : MAX_KS;
  for (int ks = num_kb < most ? num_kb : most; ks > 1; ks--)
    if (tiles * ks <= sms && tiles <= cluster_room<DUAL, NT>(ks)) return ks;
  return 1;
}

template <bool DUAL, int NT, Mode MODE>
int launch(const Fp8Product& p, int ks, cudaStream_t st) {
  using C = Narrow<DUAL, NT, MODE>;
  const int tiles_m = (p.M + NT - 1) / NT, blocks = blocks_of(p.N), num_kb = blocks_of(p.K);
  if (tiles_m > 65535) return STU_ERR_SHAPE;
  // one deep ring per SM, or two CTAs per SM where there are that many
  constexpr size_t two = 233472 / 2 - 1024;
  int stages = deepest<DUAL, NT, MODE>();
  if ((long long)blocks * ks * tiles_m > device_sm_count() && smem_bytes<DUAL, NT, MODE>(2) <= two)
    while (stages > 2 && smem_bytes<DUAL, NT, MODE>(stages) > two) stages--;
  const int most = ((num_kb + ks - 1) / ks + C::KBS - 1) / C::KBS + 1;   // (a range may begin inside a stage)
  if (stages > most) stages = most;
  CUtensorMap w, w2, x, sw, sw2, sx;
  int rc = fp8_tensor_map(&w, p.w, p.N, p.K, 128);
  if (!rc) rc = fp8_tensor_map(&x, p.x, p.M, p.K, NT);
  if (!rc) rc = fp8_tensor_map(&sw, p.ws, p.N, p.K, -1);
  if (!rc) rc = fp8_tensor_map(&sx, p.xs, p.M, p.K, -1);
  w2 = w, sw2 = sw;
  if (DUAL) {
    if (!rc) rc = fp8_tensor_map(&w2, p.w2, p.N, p.K, 128);
    if (!rc) rc = fp8_tensor_map(&sw2, p.w2s, p.N, p.K, -1);
  }
  if (rc) return rc;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at[2];
  cudaError_t e = configure<DUAL, NT, MODE>(cfg, at, dim3(blocks, ks, tiles_m), smem_bytes<DUAL, NT, MODE>(stages));
  if (e != cudaSuccess) return (int)e;
  cfg.stream = st;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, fp8_narrow_kernel<DUAL, NT, MODE>, w, w2, x, sw, sw2, sx, p.resid, p.ldr, p.y, p.ldy, p.hq, p.hs, p.M, p.N, p.K, stages,
                         p.overlap, device_status_word(), (int)take_dropped_stage(), wait_bound_ns());
  if (e != cudaSuccess) return (int)e;
  STU_CHECK_LAUNCH();
  return STU_OK;
}
template <bool DUAL, int NT> int launch(const Fp8Product& p, cudaStream_t st) {
  const int ks = cluster_size<DUAL, NT>(p);
  constexpr Mode OTHER = NT < 128 ? ALONE : LATE;   // (128 tokens come here where K is cut: fp8_narrow_takes)
  const bool early = NT < 128 ? ks > 1 : blocks_of(p.K) < 16 * ks;
  return early ? launch<DUAL, NT, EARLY>(p, ks, st) : launch<DUAL, NT, OTHER>(p, ks, st);
}

}  // namespace

// Whether a product takes less time here than on the tiles of fp8_gemm.cu (us, here and there, weights from HBM).  Plain: up to 64 tokens (64: 1024 x 4096 5.1 and 10.1, 18432 x 1536 9.2 and
// 10.8, 4096 x 1024 5.4 and 5.5; of 48 such products 64 x 8192 x 2048 alone is slower, 8.2 and 7.9).  More: 128 of them take 6.05 + 0.32 per k-block of a CTA here, one round of tiles
// there 4.1 + 0.2 per k-block, 1.4 more where the last columns are not 32 and 4.5 more for rows off the 16-byte grid, which leave in single values (K over 8 CTAs: 128 x 1024 x 4096 7.1 and 10.4;
// 128 x 1024 x 1024 5.9 and 5.7; over 6: 128 x 2048 x 2048 7.1 and 7.4, 200 x 520 x 700 5.8 and 6.7; over 4: 512 x 1024 x 4096 8.9 and 10.4, 256 x 2048 x 2048 8.0 and 7.5, 128 x 4096 x 1024 7.1 and 5.9; over 3:
// 384 x 1536 x 6144 11.1 and 13.8; over 2: 700 x 1536 x 18432 25.1 and 33.3, 700 x 1024 x 4096 11.3 and 10.4, 700 x 1111 x 1000 8.3 and 10.3).
// Gate/up, whose sums are twice as many to bring together: up to 24 tokens (24: 18432 x 1536 15.1 and 16.0, 12288 x 1024 10.1 and 10.6), up to 32 where K is shared (4096 x 1024 7.5 and 7.9, 6144 x 1536
// 10.1 and 11.7; not: 18432 x 1536 16.0 and 16.0, 12288 x 1024 11.0 and 10.6).
bool fp8_narrow_takes(const Fp8Product& p) {
  if (p.w2) return p.M <= 24 || (p.M <= 32 && cluster_size<true, 32>(p) > 1);
  if (p.M <= 64) return true;
  const long long ks = cluster_size<false, 128>(p), num_kb = blocks_of(p.K);
  const bool on_grid = !((p.ldy | (p.resid ? p.ldr : 0)) & 7) && aligned16(p.y) && aligned16(p.resid);
  return ks > 1 && (4100 + 200 * num_kb + (!on_grid ? 4500 : p.N & 31 ? 1400 : 0)) * ks > 6050 * ks + 320 * num_kb;
}

int fp8_narrow(const Fp8Product& p, cudaStream_t st) {
  if (p.w2) return p.M <= 16 ? launch<true, 16>(p, st) : launch<true, 32>(p, st);
  return p.M <= 16 ? launch<false, 16>(p, st) : p.M <= 32 ? launch<false, 32>(p, st) : p.M <= 64 ? launch<false, 64>(p, st) : launch<false, 128>(p, st);
}

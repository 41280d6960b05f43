// Products of 8-bit rows on tcgen05: what is between their entry point and the kernels that take them, and the instructions of both kernels.
#pragma once
#include <cuda.h>

#include "fp8.cuh"
#include "tma.cuh"

struct Fp8Product {
  const unsigned char *x, *xs, *w, *ws, *w2, *w2s;   // values and scales (fp8.cuh); w2 = NULL: plain
  const bf16* resid;                                 // plain: may be NULL, may be y
  long long ldr;
  bf16* y;
  long long ldy;
  unsigned char *hq, *hs;                            // gate/up: 8-bit rows of N columns
  int M, N, K;
  int overlap;                                       // the weights may be fetched ahead of the kernel before this one's end
};

int fp8_gemm(const Fp8Product& p, cudaStream_t st);     // fp8_gemm.cu
int fp8_narrow(const Fp8Product& p, cudaStream_t st);   // fp8_narrow.cu
bool fp8_narrow_takes(const Fp8Product& p);
// Tensor map of 8-bit rows' values (box > 0: rows of a box of one k-block) or of their scales (box < 0: pieces of a box), kept per thread.
int fp8_tensor_map(CUtensorMap* map, const void* base, long long rows, long long cols, int box);

namespace fp8 {

constexpr int BM = 128, BK = 128;   // rows of the first operand per CTA; bytes of a k-block: a block of 128 columns, one row of the 128-byte swizzle
constexpr int A_BYTES = BM * BK;
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

}  // namespace fp8

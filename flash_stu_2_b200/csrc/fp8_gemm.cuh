// A product of 8-bit rows, between its entry point and the kernels that take it.
#pragma once
#include "common.cuh"

struct Fp8Product {
  const unsigned char *x, *xs, *w, *ws, *w2, *w2s;   // values and scales (fp8.cuh); w2 = NULL: plain
  const bf16* resid;                                 // plain: may be NULL, may be y
  long long ldr;
  bf16* y;
  long long ldy;
  unsigned char *hq, *hs;                            // gate/up: 8-bit rows of N columns
  int M, N, K;
};

int fp8_gemm(const Fp8Product& p, cudaStream_t st);   // fp8_gemm.cu

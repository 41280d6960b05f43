// Keys and values into a ring cache of 4 bits (kv4.cuh), and back.
#include "kv4.cuh"

int device_sm_count();   // gemm_tc.cu

namespace {

// The keys and values of qkv's rows into the rings: a warp per row, eight lanes per piece.  Rows are `cu`'s packed sequences (sequence b: rows cu[b] ..
// cu[b + 1] - 1), or `per_seq` each.  Of each sequence the last `slots` are written, at positions pos[2 b] and up; the last CTA moves pos on.
// HBM reads 4 (fp32: 8) bytes of a key and a value where it writes 1.1; the arithmetic, 75 instructions for a lane's 8 numbers, takes longer.
// Write and read of 16 prompts of 14140 tokens, 12 heads of 128: 72 us; with a grid of one round, and four units at a time, 75.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_write_kernel(const T* __restrict__ qkv, long long row_stride, unsigned char* __restrict__ k4,
                                                        unsigned char* __restrict__ v4, int* __restrict__ pos, const int* __restrict__ cu, int B, int rows,
                                                        int per_seq, int H, int Hk, int hd, int slots, int most) {
  const int two = hd > 64, width = kv4::width_of(hd);   // two pieces
  const int units = 2 * Hk << two;                      // of a row: keys' heads, then values'
  const long long head_bytes = kv4::head_bytes(hd, slots);
  const int i = threadIdx.x & 7, mine = threadIdx.x >> 3 & 3;
  // few rows: several warps share one
  const int warps = gridDim.x * 8, share = max(1, min((units + 3) / 4, min(warps, most) / rows)), warp = blockIdx.x * 8 + (threadIdx.x >> 5);
  for (int at = warp; at < rows * share; at += warps) {   // (rows * share: at most the warps, or rows)
    const int row = at / share, part = at - row * share;
    int b, t, count;
    if (cu) {   // the sequence of the row: the last one that begins at or before it and is not empty
      int lo = 0, hi = B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= row) lo = mid;
        else hi = mid;
      }
      b = lo;
      t = row - cu[b];
      count = cu[b + 1] - cu[b];
    } else {
      b = row / per_seq;
      t = row - b * per_seq;
      count = per_seq;
    }
    if (t < 0 || t >= count || t < count - slots) continue;   // (the same for the whole warp)
    const long long slot = kv4::slot_of(pos[2 * b] + t, slots);
    const T* from = qkv + row * row_stride + (long long)H * hd + i * 8;
    for (int u0 = 4 * part; u0 < units; u0 += 8 * share) {   // eight units at a time: the second four's values are under way with the first's
      float x[2][8];
      bool on[2], there[2];
      int head[2], piece[2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int unit = u0 + 4 * share * k + mine;
        piece[k] = unit & two;   // heads of keys, then of values: as they lie in the row
        head[k] = unit >> two;
        on[k] = unit < units;
        there[k] = on[k] && piece[k] * 64 + i * 8 < hd;
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = 0.f;
        if (there[k]) kv4::load8<VEC>(from + head[k] * hd + piece[k] * 64, x[k]);
      }
#pragma unroll
      for (int k = 0; k < 2; k++) {
        if (u0 + 4 * share * k >= units) break;   // (the same for the whole warp)
        uint32_t word, scale;
        kv4::quantize(x[k], there[k], word, scale);
        if (on[k]) {
          const bool value = head[k] >= Hk;
          unsigned char* ring = (value ? v4 : k4) + ((long long)b * Hk + (value ? head[k] - Hk : head[k])) * head_bytes;
          if (i * 8 < width >> two) reinterpret_cast<uint32_t*>(ring)[slot * (width / 8) + kv4::word_at(i, piece[k], 1 + two)] = word;
          if (i == 0) reinterpret_cast<uint32_t*>(ring + (long long)slots * (width / 2))[(slot << two) + piece[k]] = scale;
        }
      }
    }
  }
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) last = kv4::last_to_arrive(&pos[1], (int)gridDim.x);
  __syncthreads();
  if (last) {
    for (int b = threadIdx.x; b < B; b += 256) pos[2 * b] += cu ? max(cu[b + 1] - cu[b], 0) : per_seq;
    if (threadIdx.x == 0) pos[1] = 0;
  }
}

// Rings as values [B][slots][Hk hd]: a warp takes 8 slots of a head at a time, four lanes a row, as the bytes lie.  Bound by HBM: 32 rings of 1040 slots, 12
// heads of 128, 68 to 70 us (3.8 TB/s, four fifths of it written in runs of 256 bytes per row and head).
// bf16: a number enters as a bf16 (exact), and one multiply-add of pairs, rounded once, makes the value.
template <typename T, int W>
__global__ void __launch_bounds__(256) kv4_read_kernel(const unsigned char* __restrict__ k4, const unsigned char* __restrict__ v4, T* __restrict__ k,
                                                       T* __restrict__ v, int Hk, int hd, int slots, int runs) {
  constexpr int NP = W > 64 ? 2 : 1, WORDS = W / 32;    // pieces; words of a lane: NP of them hold dimensions 8 i .. 8 i + 7 of each piece
  const int run = blockIdx.x / runs, first = (blockIdx.x - run * runs) * 64 + (threadIdx.x >> 5) * 8;   // a CTA: 64 slots of one sequence's head
  const int slot = first + ((threadIdx.x & 31) >> 2), c = threadIdx.x & 3;
  if (slot >= slots) return;
  const long long head_bytes = kv4::head_bytes(W, slots);
  const unsigned char* ring = (blockIdx.y ? v4 : k4) + run * head_bytes;
  const int b = run / Hk, head = run - b * Hk;
  T* to = (blockIdx.y ? v : k) + ((long long)b * slots + slot) * Hk * hd + (long long)head * hd;
  uint32_t w[WORDS], sc[NP];
  if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(ring + slot * (W / 2ll) + c * 16);
  if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(ring + slot * (W / 2ll) + c * 8);
  if constexpr (WORDS == 1) w[0] = *reinterpret_cast<const uint32_t*>(ring + slot * (W / 2ll) + c * 4);
#pragma unroll
  for (int p = 0; p < NP; p++) sc[p] = reinterpret_cast<const uint32_t*>(ring + slots * (W / 2ll))[slot * NP + p];
#pragma unroll
  for (int e = 0; e < WORDS; e++) {
    const int p = e % NP, d = 64 * p + 8 * (WORDS / NP * c + e / NP);
    if (d >= hd) continue;
    if constexpr (sizeof(T) == 2) {
      const uint32_t step = __byte_perm(sc[p], 0, 0x3232), low = __byte_perm(sc[p], 0, 0x1010);
      uint32_t y[4], o[4];
#pragma unroll
      for (int s = 0; s < 4; s++) {   // numbers s and s + 4
        uint32_t n = ((w[e] >> 4 * s) & 0x000f000fu) | 0x43004300u;
        asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(n) : "r"(0x43004300u));
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y[s]) : "r"(n), "r"(step), "r"(low));
      }
      o[0] = __byte_perm(y[0], y[1], 0x5410);
      o[1] = __byte_perm(y[2], y[3], 0x5410);
      o[2] = __byte_perm(y[0], y[1], 0x7632);
      o[3] = __byte_perm(y[2], y[3], 0x7632);
      *reinterpret_cast<uint4*>(to + d) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      const float low = __uint_as_float(sc[p] << 16), step = __uint_as_float(sc[p] & 0xffff0000u);
      float x[8];
#pragma unroll
      for (int s = 0; s < 8; s++) x[s] = fmaf(__uint_as_float(((w[e] >> 4 * s) & 15u) | 0x4b000000u) - 8388608.f, step, low);
      store_vec(reinterpret_cast<float*>(to) + d, x);
      store_vec(reinterpret_cast<float*>(to) + d + 4, x + 4);
    }
  }
}

template <typename T>
int launch_write(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const int* cu, int B, long long rows, int per_seq, int H, int Hk,
                 int hd, int slots, cudaStream_t st) {
  // a warp per row; where there are fewer rows than fit on the SMs at once (8 CTAs each), several for one; where there are more, up to 8 rounds of CTAs, which leave no SM
  // waiting for the slowest warp's last row.  No CTA waits for another; each counts itself once.
  const long long warps = rows * ((2 * Hk * kv4::pieces_of(hd) + 3) / 4), most = 8ll * device_sm_count();
  const int grid = (int)((warps + 7) / 8 < most ? (warps + 7) / 8 : (rows + 7) / 8 < most ? most : (rows + 7) / 8 < 8 * most ? (rows + 7) / 8 : 8 * most);
  const bool vec = aligned16(qkv) && row_stride % (16 / (int)sizeof(T)) == 0;
  if (vec)
    kv4_write_kernel<T, true><<<grid, 256, 0, st>>>((const T*)qkv, row_stride, (unsigned char*)k4, (unsigned char*)v4, pos, cu, B, (int)rows, per_seq, H, Hk,
                                                    hd, slots, (int)most * 8);
  else
    kv4_write_kernel<T, false><<<grid, 256, 0, st>>>((const T*)qkv, row_stride, (unsigned char*)k4, (unsigned char*)v4, pos, cu, B, (int)rows, per_seq, H, Hk,
                                                     hd, slots, (int)most * 8);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

}  // namespace

extern "C" int stu_kv4_write(const void* qkv, long long row_stride, void* k4, void* v4, int* pos, const int* cu_seqlens, int B, long long rows, int H,
                             int Hk, int hd, int slots, int dtype, void* stream) {
  if (!qkv || !k4 || !v4 || !pos) return STU_ERR_NULL;
  const int rc = kv4::geometry(B, H, Hk, hd, slots, dtype);
  if (rc != STU_OK) return rc;
  // (above the last row there is room for a grid's warps, 512 per SM: the rows' count passes no 32 bits)
  if (rows <= 0 || rows > 0x7ff00000ll || row_stride < (long long)(H + 2 * Hk) * hd || (!cu_seqlens && rows % B)) return STU_ERR_SHAPE;
  if (!aligned16(k4) || !aligned16(v4)) return STU_ERR_ALIGN;
  const int per_seq = cu_seqlens ? 0 : (int)(rows / B);
  return dtype == STU_F32 ? launch_write<float>(qkv, row_stride, k4, v4, pos, cu_seqlens, B, rows, per_seq, H, Hk, hd, slots, (cudaStream_t)stream)
                          : launch_write<bf16>(qkv, row_stride, k4, v4, pos, cu_seqlens, B, rows, per_seq, H, Hk, hd, slots, (cudaStream_t)stream);
}

extern "C" int stu_kv4_read(const void* k4, const void* v4, void* k, void* v, int B, int Hk, int hd, int slots, int dtype, void* stream) {
  if (!k4 || !v4 || !k || !v) return STU_ERR_NULL;
  const int rc = kv4::geometry(B, Hk, Hk, hd, slots, dtype);
  if (rc != STU_OK) return rc;
  if (!aligned16(k4) || !aligned16(v4) || !aligned16(k) || !aligned16(v)) return STU_ERR_ALIGN;
  const long long runs = (slots + 63) / 64;
  if (runs * B * Hk > 0x7fffffffll) return STU_ERR_SHAPE;
  const dim3 grid((unsigned)(runs * B * Hk), 2);
  auto go = [&](auto kernel, auto* one) {
    kernel<<<grid, 256, 0, (cudaStream_t)stream>>>((const unsigned char*)k4, (const unsigned char*)v4, (decltype(one))k, (decltype(one))v, Hk, hd, slots, (int)runs);
  };
  if (dtype == STU_F32)
    hd <= 32 ? go(kv4_read_kernel<float, 32>, (float*)nullptr) : hd <= 64 ? go(kv4_read_kernel<float, 64>, (float*)nullptr) : go(kv4_read_kernel<float, 128>, (float*)nullptr);
  else
    hd <= 32 ? go(kv4_read_kernel<bf16, 32>, (bf16*)nullptr) : hd <= 64 ? go(kv4_read_kernel<bf16, 64>, (bf16*)nullptr) : go(kv4_read_kernel<bf16, 128>, (bf16*)nullptr);
  STU_CHECK_LAUNCH();
  return STU_OK;
}

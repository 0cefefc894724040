// C[M, N] (bf16) = A B^T + bias of e4m3 operands with a power-of-two scale for each block of 128 (fp8_block.h): A [M, Kp] with 1 x 128 scales
// (activations, output gradients), B [N, Kp] with 128 x 128 scales (weights; for the input gradient their transposed copy).
//   C[m][n] = bias[n] + sum over k-blocks b of 2^(ea[m][b] + eb[n / 128][b]) sum_{k in b} a[m][k] b[n][k]
// The scales are powers of two, so v_mfma_scale_f32_16x16x128_f8f6f4 applies both inside the matrix instruction (one k-block of 128 per
// instruction): no second accumulator, no multiply per block; sums are fp32 throughout and rounded to bf16 once.
// Measured: 66560 x 4096 x 1024 282 us at the least and 321 as the median of 23 in a row, under which the clock falls (1.98, 1.74 PF/s in the persistent kernel,
// eight k-tiles a tile; 8192^3 2.7 PF/s); medians: 9984 x 2304 x 768 31 us, 9984 x 768 x 2304 30 us, 1237 x 777 x 1000 8.5 us, 8 x 4096 x 1024 3.4 us, 1 x 1024 x 4096
// 4.9 us (latency: every wave four blocks, one after the other).
#include "../../include/uc2_hip.h"
#include "common.h"
#include "fp8_block.h"
#include "gemm_tile.h"
#include "gemm_pp8_kernel.h"

bool uc2_gemm_pp8_supported(const GemmArgs& p);                   // gemm_pp8.hip: whole 256 x 256 tiles, an even number of blocks

typedef __attribute__((ext_vector_type(8))) int blk_i32x8;
typedef __attribute__((ext_vector_type(4))) int blk_i32x4;

struct BlkGemm {
  int M, N, Kb, lda, ldb, ldc, lds_a, vec;                         // Kb = Kp / 128; lds_a: rows of A's scale words; vec: C takes 8-byte stores
  const unsigned char *A, *B; const unsigned* sa; const unsigned char* sb;
  const float* bias; bf16* C;
};

// the matrix instruction with A and B swapped: the accumulator block is [n][m], a lane holds row m = lane & 15 and columns 4 (lane >> 4) + 0..3
__device__ __forceinline__ f32x4 blk_mfma(blk_i32x8 b, blk_i32x8 a, f32x4 c, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, sb, 0, sa);
}
__device__ __forceinline__ blk_i32x8 blk_cat(blk_i32x4 lo, blk_i32x4 hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ void blk_put(const BlkGemm& p, int m, int n, const f32x4& v) {
  if (m >= p.M || n >= p.N) return;
  bf16* c = p.C + (size_t)m * p.ldc + n;
  if (n + 4 <= p.N) {
    f32x4 x = v;
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += p.bias[n + e];
    }
    if (p.vec) { *reinterpret_cast<bf16x4*>(c) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]}; return; }
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = (bf16)x[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (n + e < p.N) c[e] = (bf16)(v[e] + (p.bias ? p.bias[n + e] : 0.f));
  }
}

// ---- few rows: the weight's bytes are the work.  A workgroup owns 16 columns and 16 MB rows, its 8 waves take the k-blocks in turn -- both
// operands straight from memory into the matrix instruction's registers, 32 bytes per lane and block -- and are added in wave order.
template <int MB>
__global__ __launch_bounds__(512) void gemm_fp8_block_rows_kernel(BlkGemm p) {
  __shared__ f32x4 red[8][MB][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
  const unsigned char* b = p.B + (size_t)min(n0 + i, p.N - 1) * p.ldb + 32 * g;
  const unsigned char* sb = p.sb + (size_t)(n0 >> 7) * p.Kb;
  const unsigned char* a[MB];
  int row[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) { row[j] = min(m0 + 16 * j + i, p.M - 1); a[j] = p.A + (size_t)row[j] * p.lda + 32 * g; }
  f32x4 acc[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int kt = w; kt < p.Kb; kt += 8) {
    const blk_i32x4* bp = reinterpret_cast<const blk_i32x4*>(b + (size_t)kt * 128);
    const blk_i32x8 bv = blk_cat(bp[0], bp[1]);
    const int es = sb[kt];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const blk_i32x4* ap = reinterpret_cast<const blk_i32x4*>(a[j] + (size_t)kt * 128);
      const int ea = p.sa[(size_t)(kt >> 2) * p.lds_a + row[j]] >> (8 * (kt & 3));
      acc[j] = blk_mfma(bv, blk_cat(ap[0], ap[1]), acc[j], es, ea);
    }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) red[w][j][lane] = acc[j];
  __syncthreads();
  for (int j = w; j < MB; j += 8) {
    f32x4 s = red[0][j][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][j][lane];
    blk_put(p, m0 + 16 * j + i, n0 + 4 * g, s);
  }
}

// ---- any size: WB x WB blocks of 16 per wave, 2 x 2 waves; k-tiles of one block (128 bytes) double-buffered in LDS through registers
template <int WB>
__global__ __launch_bounds__(256) void gemm_fp8_block_tile_kernel(BlkGemm p) {
  constexpr int T = 32 * WB, NL = T * 8 / 256;                     // tile edge; 16-byte pieces per thread and operand
  __shared__ __attribute__((aligned(16))) unsigned char la[2][T * 128], lb[2][T * 128];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, i = lane & 15, wm = w >> 1, wn = w & 1;
  const int m0 = blockIdx.x * T, n0 = blockIdx.y * T;
  const unsigned char *as[NL], *bs[NL];
  int off[NL];
#pragma unroll
  for (int n = 0; n < NL; ++n) {
    const int r = (t + n * 256) >> 3, c = t & 7;
    as[n] = p.A + (size_t)min(m0 + r, p.M - 1) * p.lda + c * 16;
    bs[n] = p.B + (size_t)min(n0 + r, p.N - 1) * p.ldb + c * 16;
    off[n] = r * 128 + ((c ^ ((r >> 1) & 7)) << 4);
  }
  int row[WB];
#pragma unroll
  for (int j = 0; j < WB; ++j) row[j] = min(m0 + wm * 16 * WB + 16 * j + i, p.M - 1);
  const unsigned char* sb = p.sb + (size_t)(n0 >> 7) * p.Kb;
  f32x4 acc[WB][WB];
#pragma unroll
  for (int x = 0; x < WB; ++x)
#pragma unroll
    for (int y = 0; y < WB; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
  blk_i32x4 ra[NL], rb[NL];
  auto fetch = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NL; ++n) { ra[n] = *reinterpret_cast<const blk_i32x4*>(as[n] + (size_t)kt * 128); rb[n] = *reinterpret_cast<const blk_i32x4*>(bs[n] + (size_t)kt * 128); }
  };
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NL; ++n) { *reinterpret_cast<blk_i32x4*>(la[buf] + off[n]) = ra[n]; *reinterpret_cast<blk_i32x4*>(lb[buf] + off[n]) = rb[n]; }
  };
  unsigned sw[WB];
  fetch(0); put(0);
  __syncthreads();
  const int sz = (i >> 1) & 7;                                    // (16 rows of one chunk column: 16 places of the 256 bytes that the banks hold)
  for (int kt = 0; kt < p.Kb; ++kt) {
    const int buf = kt & 1;
    if (kt + 1 < p.Kb) fetch(kt + 1);
    if ((kt & 3) == 0) {
#pragma unroll
      for (int j = 0; j < WB; ++j) sw[j] = p.sa[(size_t)(kt >> 2) * p.lds_a + row[j]];
    }
    const int es = sb[kt];
    blk_i32x8 bv[WB];
#pragma unroll
    for (int y = 0; y < WB; ++y) {
      const unsigned char* q = lb[buf] + (wn * 16 * WB + 16 * y + i) * 128;
      bv[y] = blk_cat(*reinterpret_cast<const blk_i32x4*>(q + (((2 * g) ^ sz) << 4)), *reinterpret_cast<const blk_i32x4*>(q + (((2 * g + 1) ^ sz) << 4)));
    }
#pragma unroll
    for (int x = 0; x < WB; ++x) {
      const unsigned char* q = la[buf] + (wm * 16 * WB + 16 * x + i) * 128;
      const blk_i32x8 av = blk_cat(*reinterpret_cast<const blk_i32x4*>(q + (((2 * g) ^ sz) << 4)), *reinterpret_cast<const blk_i32x4*>(q + (((2 * g + 1) ^ sz) << 4)));
#pragma unroll
      for (int y = 0; y < WB; ++y) acc[x][y] = blk_mfma(bv[y], av, acc[x][y], es, (int)sw[x]);
      sw[x] >>= 8;
    }
    if (kt + 1 < p.Kb) put(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < WB; ++x)
#pragma unroll
    for (int y = 0; y < WB; ++y) blk_put(p, m0 + wm * 16 * WB + 16 * x + i, n0 + wn * 16 * WB + 16 * y + 4 * g, acc[x][y]);
}

static void blk_launch_tiles(const BlkGemm& p, hipStream_t st) {
  // the rows kernel while it is one workgroup per CU at most: its waves share the blocks of K, where a tile takes them one after the other (measured,
  // us: 256 x 1024 x 4096 11.3 against 14.3 in 64 x 64 tiles, 64 x 4096 x 1024 4.7 / 5.3; beyond, 512 x 768 x 768 5.8 / 4.8, 128 x 4096 x 1024 7.0 / 5.5)
  if ((long long)((p.N + 15) / 16) * ((p.M + 63) / 64) <= 256) {
    const dim3 grid((p.N + 15) / 16, (p.M + 63) / 64);
    if (p.M <= 16) hipLaunchKernelGGL(gemm_fp8_block_rows_kernel<1>, grid, dim3(512), 0, st, p);
    else if (p.M <= 32) hipLaunchKernelGGL(gemm_fp8_block_rows_kernel<2>, grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL(gemm_fp8_block_rows_kernel<4>, grid, dim3(512), 0, st, p);
    return;
  }
  // 128 x 128 tiles once there is one for each CU, 64 x 64 ones below (4096 x 1024 x 4096: 34 us against 37; 4096 x 768 x 768, 192 tiles: 10.0 / 8.3)
  const long long t128 = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
  const int T = t128 >= 256 ? 128 : 64;
  const dim3 grid((p.M + T - 1) / T, (p.N + T - 1) / T);
  if (T == 128) hipLaunchKernelGGL(gemm_fp8_block_tile_kernel<4>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(gemm_fp8_block_tile_kernel<2>, grid, dim3(256), 0, st, p);
}
static void blk_launch(BlkGemm p, hipStream_t st) {
  // whole 256 x 256 tiles go to the persistent kernel from 128 of them on, where the two meet (8192 x 1024 x 4096: 44 us both; 192 tiles of K = 768: 16.5
  // against 21.7; 96: 13.9 / 13.0); what is left of the rows and of the columns to the kernels above
  const int M0 = p.M / 256 * 256, N0 = p.N / 256 * 256;
  if ((long long)(M0 / 256) * (N0 / 256) >= 128 && ((uintptr_t)p.sb & 1) == 0) {
    GemmArgs g{};                                                  // (the "bf16 view" of bytes: K and leading dimensions halved)
    g.A = p.A; g.B = p.B; g.C = p.C; g.bias = p.bias; g.M = M0; g.N = N0; g.K = p.Kb * 64; g.lda = p.lda / 2; g.ldb = p.ldb / 2; g.ldc = g.ldaux = p.ldc;
    g.epi = EPI_NONE; g.split_k = 1; g.a_vec = g.b_vec = 1; g.alpha = 1.0f;
    g.blk_sa = p.sa; g.blk_sa_ld = p.lds_a; g.blk_sb = p.sb; g.blk_sb_ld = p.Kb;
    if (uc2_gemm_pp8_supported(g)) {
      g.col_group = pp8_col_group(N0);
      pp8_launch0<EPI_NONE, false, true>(g, st);
      if (N0 < p.N) {
        BlkGemm c = p;
        c.M = M0; c.N = p.N - N0; c.B += (size_t)N0 * p.ldb; c.sb += (size_t)(N0 / 128) * p.Kb; c.C += N0;
        if (c.bias) c.bias += N0;
        blk_launch_tiles(c, st);
      }
      if (M0 < p.M) {
        BlkGemm r = p;
        r.M = p.M - M0; r.A += (size_t)M0 * p.lda; r.sa += M0; r.C += (size_t)M0 * p.ldc;
        blk_launch_tiles(r, st);
      }
      return;
    }
  }
  blk_launch_tiles(p, st);
}

extern "C" int uc2_gemm_fp8_block(int M, int N, int K, const void* A8, int lda, const void* scale_a, int rows_a, const void* B8, int ldb,
                                  const void* scale_b, const float* bias, void* C, int ldc, void* stream) {
  UC2_CHECK_ARG(M >= 0 && M < 0x7FFFFF00 && N >= 0 && K >= 1 && K <= (1 << 30));
  if (M == 0 || N == 0) return 0;
  const int Kp = (K + 127) / 128 * 128;
  UC2_CHECK_ARG((N + 63) / 64 < 65536);                            // (a launch's second grid dimension)
  UC2_CHECK_ARG(A8 && scale_a && B8 && scale_b && C);
  UC2_CHECK_ARG(lda >= Kp && ldb >= Kp && ldc >= N && rows_a >= M && (lda % 16) == 0 && (ldb % 16) == 0);
  UC2_CHECK_ARG((((uintptr_t)A8 | (uintptr_t)B8) & 15) == 0 && ((uintptr_t)scale_a & 3) == 0 && ((uintptr_t)C & 1) == 0 && ((uintptr_t)bias & 3) == 0);
  BlkGemm p{};
  p.M = M; p.N = N; p.Kb = Kp / 128; p.lda = lda; p.ldb = ldb; p.ldc = ldc; p.lds_a = rows_a;
  p.vec = (ldc % 4) == 0 && ((uintptr_t)C & 7) == 0;
  p.A = (const unsigned char*)A8; p.B = (const unsigned char*)B8; p.sa = (const unsigned*)scale_a; p.sb = (const unsigned char*)scale_b;
  p.bias = bias; p.C = (bf16*)C;
  blk_launch(p, (hipStream_t)stream);
  UC2_LAUNCH_CHECK();
  return 0;
}

// Quantisation to e4m3 under power-of-two block scales (fp8_block.h): rows in blocks of 1 x 128 (activations, output gradients), weights in
// blocks of 128 x 128, in both orientations from one read -- a square block has the same scale in W and in W^T, so the input gradient's
// operand holds the very bytes of the forward's.  HBM-bound: x once in, one byte per element (two for a weight) out.
// Measured (medians): rows 66560 x 1024 bf16 37 us (5.6 TB/s), 9984 x 2304 15 us (4.6); a 2304 x 768 fp32 weight in both orientations 6 us: one round of memory
// latency and a reduction on 108 workgroups, one per block, which is what a block's maximum needs (its bytes at a copy's rate: 2.2).
#include "../../include/uc2_hip.h"
#include "common.h"
#include "fp8_block.h"

// a wave takes 512 columns of R rows: R loads in flight, then R reductions over 16 lanes
template <typename T, int R, bool WHOLE>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(int M, int K, int Kp, const T* __restrict__ x, long long ldx, unsigned char* __restrict__ q,
                                                             unsigned* __restrict__ scale, int lds, int groups, long long items) {
  const int lane = threadIdx.x & 63;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= items) return;
  const int rb = (int)(item / groups), g = (int)(item - (long long)rb * groups), c = g * 512 + lane * 8;
  Blk8<T> x8[R];
#pragma unroll
  for (int r = 0; r < R; ++r) x8[r].template load<WHOLE>(x + (size_t)min(rb * R + r, M - 1) * ldx, c, K);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = rb * R + r;
    float v[8];
    x8[r].template get<WHOLE>(v, c, K);
    if (row < M) blk_quant_row(v, c, Kp, q + (size_t)row * Kp, scale + (size_t)g * lds + row, lane);
  }
}
extern "C" int uc2_fp8_quant_rows(int dtype, int M, int K, const void* x, long long ldx, void* out, void* scale, void* stream) {
  UC2_CHECK_ARG(dtype == 0 || dtype == 1);
  UC2_CHECK_ARG(M >= 0 && K >= 1 && K <= (1 << 30) && ldx >= K);
  if (M == 0) return 0;
  UC2_CHECK_ARG(x && out && scale && ((uintptr_t)out & 7) == 0 && ((uintptr_t)scale & 3) == 0);
  const int Kp = (K + 127) / 128 * 128, groups = (Kp + 511) / 512;
  // four rows per wave once that leaves two waves for every SIMD (2048), one row below
  const int R = (long long)M * groups >= 8192 ? 4 : 1;
  const int most = (int)(UC2_MOST_BLOCKS(256) * 4ll / groups) * R, el = dtype == 1 ? 2 : 4;      // rows of a launch: 2^28 of 512 columns
  hipStream_t st = (hipStream_t)stream;
#define QROWS_(T_, R_, W_) hipLaunchKernelGGL((fp8_quant_rows_kernel<T_, R_, W_>), dim3((unsigned)blocks), dim3(256), 0, st, n, K, Kp, (const T_*)xp, ldx, (unsigned char*)out + (size_t)m0 * Kp, (unsigned*)scale + m0, M, groups, items)
#define QROWS(T_, R_) do { if (K % 8 == 0) QROWS_(T_, R_, true); else QROWS_(T_, R_, false); } while (0)
  for (long long m0 = 0; m0 < M; m0 += most) {
    const int n = (int)(M - m0 < most ? M - m0 : most);
    const char* xp = (const char*)x + (size_t)m0 * ldx * el;
    const long long items = (long long)((n + R - 1) / R) * groups, blocks = (items + 3) / 4;
    if (dtype == 1) { if (R == 4) QROWS(bf16, 4); else QROWS(bf16, 1); } else { if (R == 4) QROWS(float, 4); else QROWS(float, 1); }
    UC2_LAUNCH_CHECK();
  }
  return 0;
}

// one workgroup per 128 x 128 block; a thread holds 8 x 8 elements, so its 8-byte pieces of W^T are made in registers
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void fp8_quant_square_kernel(int N, int K, int Np, int Kp, const T* __restrict__ w, long long ldw, unsigned char* __restrict__ q,
                                                               unsigned char* __restrict__ scale, unsigned char* __restrict__ qt, unsigned char* __restrict__ scale_t) {
  __shared__ float wm[4];
  const int kb = blockIdx.x, nb = blockIdx.y, t = threadIdx.x, r0 = nb * 128 + (t >> 4) * 8, c0 = kb * 128 + (t & 15) * 8;
  float v[8][8], m = 0.f;
  Blk8<T> w8[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    w8[r].template load<WHOLE>(w + (size_t)min(r0 + r, N - 1) * ldw, c0, K);
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    w8[r].template get<WHOLE>(v[r], c0, K);
    if (r0 + r >= N) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[r][e] = 0.f;
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) m = fmaxf(m, blk_amax8(v[r]));
  m = wave_max(m);
  if ((t & 63) == 0) wm[t >> 6] = m;
  __syncthreads();
  const unsigned e = blk_exponent(fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3])));
  const float s = blk_inverse(e);
  if (t == 0) {
    scale[(size_t)nb * (Kp / 128) + kb] = (unsigned char)e;
    if (qt) scale_t[(size_t)kb * (Np / 128) + nb] = (unsigned char)e;
  }
  unsigned lo[8], hi[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    lo[r] = blk_pack4(v[r][0] * s, v[r][1] * s, v[r][2] * s, v[r][3] * s);
    hi[r] = blk_pack4(v[r][4] * s, v[r][5] * s, v[r][6] * s, v[r][7] * s);
    if (r0 + r < N) *reinterpret_cast<uint2*>(q + (size_t)(r0 + r) * Kp + c0) = uint2{lo[r], hi[r]};
  }
  if (!qt) return;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    unsigned a = 0, b = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a |= (((c < 4 ? lo[r] : hi[r]) >> (8 * (c & 3))) & 255u) << (8 * r);
      b |= (((c < 4 ? lo[4 + r] : hi[4 + r]) >> (8 * (c & 3))) & 255u) << (8 * r);
    }
    if (c0 + c < K) *reinterpret_cast<uint2*>(qt + (size_t)(c0 + c) * Np + r0) = uint2{a, b};
  }
}
extern "C" int uc2_fp8_quant_square(int dtype, int N, int K, const void* w, long long ldw, void* out, void* scale, void* out_t, void* scale_t, void* stream) {
  UC2_CHECK_ARG(dtype == 0 || dtype == 1);
  UC2_CHECK_ARG(N >= 0 && K >= 1 && N <= 65535 * 128 && K <= (1 << 23) && ldw >= K);      // (65535: a launch's second grid dimension)
  if (N == 0) return 0;
  UC2_CHECK_ARG(w && out && scale && (out_t == nullptr) == (scale_t == nullptr) && (((uintptr_t)out | (uintptr_t)out_t) & 7) == 0);
  const int Kp = (K + 127) / 128 * 128, Np = (N + 127) / 128 * 128;
  hipStream_t st = (hipStream_t)stream;
#define QSQ(T_, W_) hipLaunchKernelGGL((fp8_quant_square_kernel<T_, W_>), dim3(Kp / 128, Np / 128), dim3(256), 0, st, N, K, Np, Kp, (const T_*)w, ldw, (unsigned char*)out, (unsigned char*)scale, (unsigned char*)out_t, (unsigned char*)scale_t)
  if (dtype == 1) { if (K % 8 == 0) QSQ(bf16, true); else QSQ(bf16, false); } else { if (K % 8 == 0) QSQ(float, true); else QSQ(float, false); }
  UC2_LAUNCH_CHECK();
  return 0;
}

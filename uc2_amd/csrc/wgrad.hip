// Weight and bias gradient of a linear layer on bf16 rows of any size, stride and alignment, in one pass over them:
//   dW[n][k] = sum over rows m of dY[m][n] X[m][k]   (fp32),   db[n] = sum over m of dY[m][n]
// Both operands are contracted over their ROWS: 64-row slabs go row-major into LDS (through registers: unaligned and partial columns become
// whole zero-padded chunks on the way) and are read transposed (ds_read_b64_tr_b16) into v_mfma_f32_32x32x16_bf16, both in the same row
// order, which is all that a contraction asks for.  128 x 128 tiles, 2 x 2 waves: 64 KiB of LDS, two workgroups per CU.  The rows are split over workgroups until the chip is full; the parts
// (fp32) are added in split order by a second kernel: no atomics, the same bits every run.  The workgroups of the first column of tiles also
// add up the dY values they stage anyway.
// Bound by the matrix instructions and the parts: measured with db, 20000 x 1100 x 900 93 us (0.43 PF/s), 33280 x 4000 x 1000 480 us (0.55 PF/s); whole tiles
// (below) 9984 x 2304 x 768 38 us and 9 for db and 14 for the sum of the parts.
#include "../../include/uc2_hip.h"
#include "common.h"
#include "fp8_block.h"

struct WgradArgs {
  int M, N, K, tn, tk, splits, per;                     // tiles along n and k, row splits, slabs per split
  const bf16 *dy, *x; long long lddy, ldx;
  float* dw; long long lddw; float* db;
  float* part; float* pdb; int dsplits;                 // [splits][N][K], [dsplits][N]
};

// chunk swizzle: the 8 rows x 4 chunks of a transposing read meet each of the 16 chunk columns twice, its least
__device__ __forceinline__ int wg_swz(int row) { return ((row & 1) << 3) | ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3); }
// 8 columns of a row from the clamped column cc = min(c, n - 8) and row (no branch around the load: hipcc waits for a load at the end of a branch that
// uses it); wg_fix moves them into place and clears what is behind the row or the matrix.  Rows of less than 8 columns (TINY): one by one.
template <bool TINY> __device__ __forceinline__ bf16x8 wg_load(const bf16* x, long long ld, int m, int M, int cc, int n) {
  const bf16* row = x + (size_t)min(m, M - 1) * ld;
  if (!TINY) return *reinterpret_cast<const blk_bf16x8_u*>(row + cc);
  bf16x8 v = {};
#pragma unroll
  for (int e = 0; e < 8; ++e) if (cc + e < n) v[e] = row[cc + e];
  return v;
}
__device__ __forceinline__ bf16x8 wg_fix(bf16x8 v, int shift, bool keep) {         // shift: 16-bit places, 0 .. 8
  typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
  u64x2 u = __builtin_bit_cast(u64x2, v);
  const int b = shift * 16;
  unsigned long long lo = b < 64 ? u[0] >> b : b < 128 ? u[1] >> (b - 64) : 0ull, hi = b < 64 ? u[1] >> b : 0ull;
  if (b > 0 && b < 64) lo |= u[1] << (64 - b);
  return keep ? __builtin_bit_cast(bf16x8, u64x2{lo, hi}) : bf16x8{};
}
// fragment: columns cb .. cb + 31 (lane & 31), rows 16 ks + {4 h .. + 3, 8 + 4 h .. + 3} of the slab
__device__ __forceinline__ bf16x8 wg_frag(const char* lds, int cb, int ks, int lane) {
  typedef __attribute__((address_space(3))) short4v* lp;
  const int h = lane >> 5, i = lane & 15, dh = (lane >> 4) & 1;
  const int r0 = 16 * ks + 4 * h + (i >> 2), r1 = r0 + 8, c = (cb >> 3) + 2 * dh + ((i >> 1) & 1), sub = (i & 1) * 8;
  const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + r0 * 256 + ((c ^ wg_swz(r0)) << 4) + sub));
  const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + r1 * 256 + ((c ^ wg_swz(r1)) << 4) + sub));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <bool TINY>
__global__ __launch_bounds__(256, 2) void wgrad_kernel(WgradArgs a) {
  __shared__ __attribute__((aligned(16))) char ly[2][64 * 256], lx[2][64 * 256];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, wn = w >> 1, wk = w & 1;
  // blocks go to the 8 XCDs in turn: each gets a contiguous share of the split-major list, so that the tiles which read the same rows share an L2
  const int items = a.tn * a.tk * a.splits, share = (items + 7) >> 3, local = blockIdx.x >> 3, item = (blockIdx.x & 7) * share + local;
  if (item >= items || local >= share) return;
  const int split = item / (a.tn * a.tk), tile = item - split * a.tn * a.tk, n0 = (tile / a.tk) * 128, k0 = (tile % a.tk) * 128;
  const int slabs = (a.M + 63) / 64, s0 = split * a.per, s1 = min(slabs, s0 + a.per);
  const int c = t & 15, rt = t >> 4;
  const bool sums = a.db != nullptr && k0 == 0;
  const int ny = n0 + 8 * c, nx = k0 + 8 * c;
  const int cy = TINY ? ny : min(ny, a.N - 8), cx = TINY ? nx : min(nx, a.K - 8), fy = TINY ? 0 : min(ny - cy, 8), fx = TINY ? 0 : min(nx - cx, 8);
  const bool edge = n0 + 128 > a.N || k0 + 128 > a.K;              // (uniform)
  f32x16 acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  float cs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  // two sets of staging registers: a slab's loads have two slabs' matrix instructions to land in (with one set a slab took as long as its loads)
  struct Slab { bf16x8 y[4], x[4]; } va, vb;
  auto fetch = [&](Slab& v, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = s * 64 + rt + 16 * i;
      v.y[i] = wg_load<TINY>(a.dy, a.lddy, m, a.M, cy, a.N);
      v.x[i] = wg_load<TINY>(a.x, a.ldx, m, a.M, cx, a.K);
    }
  };
  auto put = [&](Slab& v, int s, int buf) __attribute__((always_inline)) {
    if (edge || (s + 1) * 64 > a.M) {                               // (uniform)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool keep = s * 64 + rt + 16 * i < a.M;
        v.y[i] = wg_fix(v.y[i], fy, keep);
        v.x[i] = wg_fix(v.x[i], fx, keep);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = rt + 16 * i, off = r * 256 + ((c ^ wg_swz(r)) << 4);
      *reinterpret_cast<bf16x8*>(ly[buf] + off) = v.y[i];
      *reinterpret_cast<bf16x8*>(lx[buf] + off) = v.x[i];
      if (sums) {
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] += (float)v.y[i][e];
      }
    }
  };
  auto step = [&](int s, int buf, Slab& next, Slab& far) __attribute__((always_inline)) {       // next: slab s + 1, landed or landing
    if (s + 2 < s1) fetch(far, s + 2);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const bf16x8 y0 = wg_frag(ly[buf], wn * 64, ks, lane), y1 = wg_frag(ly[buf], wn * 64 + 32, ks, lane);
      const bf16x8 x0 = wg_frag(lx[buf], wk * 64, ks, lane), x1 = wg_frag(lx[buf], wk * 64 + 32, ks, lane);
      // accumulator block [k][n]: a lane holds one n (lane & 31) and, four at a time, neighbouring k
      acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x0, y0, acc[0][0], 0, 0, 0);
      acc[0][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x1, y0, acc[0][1], 0, 0, 0);
      acc[1][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x0, y1, acc[1][0], 0, 0, 0);
      acc[1][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x1, y1, acc[1][1], 0, 0, 0);
    }
    if (s + 1 < s1) put(next, s + 1, buf ^ 1);
    __syncthreads();
  };
  if (s0 < s1) {
    fetch(va, s0);
    if (s0 + 1 < s1) fetch(vb, s0 + 1);
    put(va, s0, 0);
  }
  __syncthreads();
  for (int s = s0; s < s1; s += 2) {
    step(s, 0, vb, va);
    if (s + 1 < s1) step(s + 1, 1, va, vb);
  }
  float* out = a.splits == 1 ? a.dw : a.part + (size_t)split * a.N * a.K;
  const long long ld = a.splits == 1 ? a.lddw : a.K;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int n = n0 + wn * 64 + 32 * x + (lane & 31);
    if (n < a.N) {
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int k = k0 + wk * 64 + 32 * y + 8 * q + 4 * (lane >> 5);
          float* p = out + (size_t)n * ld + k;
          if (k + 4 <= a.K) *reinterpret_cast<blk_f32x4_u*>(p) = blk_f32x4_u{acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2], acc[x][y][4 * q + 3]};
          else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (k + e < a.K) p[e] = acc[x][y][4 * q + e];
          }
        }
    }
  }
  if (sums) {                                           // (uniform; the last loop iteration ended with a barrier)
    float* red = reinterpret_cast<float*>(ly[0]);       // [16 row groups][128 columns]
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rt * 128 + 8 * c + e] = cs[e];
    __syncthreads();
    if (t < 128 && n0 + t < a.N) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += red[i * 128 + t];
      (a.splits == 1 ? a.db : a.pdb + (size_t)split * a.N)[n0 + t] = s;
    }
  }
}
// column sums of dY alone (beside a weight gradient that another kernel makes): 256 columns and a share of the rows per workgroup
__global__ __launch_bounds__(256) void wgrad_cols_kernel(WgradArgs a) {
  __shared__ float red[8][256];
  const int t = threadIdx.x, n = blockIdx.x * 256 + (t & 31) * 8, rt = t >> 5;
  const int per = (a.M + a.dsplits - 1) / a.dsplits, m0 = blockIdx.y * per, m1 = min(a.M, m0 + per);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int m = m0 + rt; m < m1; m += 8) {
    const bf16x8 v = wg_load<false>(a.dy, a.lddy, m, a.M, n, a.N);      // (N is a multiple of 256 here)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += (float)v[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rt][(t & 31) * 8 + e] = s[e];
  __syncthreads();
  if (blockIdx.x * 256 + t < a.N) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += red[i][t];
    a.pdb[(size_t)blockIdx.y * a.N + blockIdx.x * 256 + t] = x;
  }
}
// sum of the splits in order; the last workgroups take db
__global__ __launch_bounds__(256) void wgrad_sum_kernel(WgradArgs a) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4, nk = (long long)a.N * a.K;
  if (i < nk) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = i + 4 <= nk;
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      const float* p = a.part + (size_t)k * nk + i;
      if (whole) {
        const blk_f32x4_u v = *reinterpret_cast<const blk_f32x4_u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (i + e < nk) s[e] += p[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e >= nk) break;
      if (a.lddw == a.K) a.dw[i + e] = s[e];
      else { const long long n = (i + e) / a.K; a.dw[n * a.lddw + (i + e - n * a.K)] = s[e]; }
    }
  } else if (a.db) {                                    // a column per thread
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x - (nk + 3) / 4;
    if (n >= a.N) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.dsplits; ++k) s += a.pdb[(size_t)k * a.N + n];
    a.db[n] = s;
  }
}

extern "C" int uc2_gemm(int dtype, int trans_a, int trans_b, int M, int N, int K, const void* A, int lda, const void* B, int ldb, void* C, int ldc, int c_is_f32,
                        const float* bias, int epilogue, const void* aux_in, void* aux_out, int ldaux, int accumulate, int split_k, int variant, void* workspace,
                        size_t workspace_bytes, int flags, void* stream);

static void wgrad_plan(int M, int N, int K, WgradArgs& a) {
  a.tn = (N + 127) / 128; a.tk = (K + 127) / 128;
  const long long tiles = (long long)a.tn * a.tk;
  const int slabs = (M + 63) / 64;
  // two workgroups per CU (512), each split four slabs (256 rows) at least
  long long s = 512 / tiles, most = (slabs + 3) / 4;
  if (s > most) s = most;
  if (s < 1) s = 1;
  a.per = (int)((slabs + s - 1) / s);
  a.splits = a.per ? (slabs + a.per - 1) / a.per : 1;
  a.dsplits = a.splits;
}
// Whole 256 x 256 tiles of aligned rows go to uc2_gemm's persistent kernel (variant 12), its partial tiles to the sum kernel here: 9984 x 2304 x 768
// 51 us against 84 of the kernel above, 33280 x 4096 x 1024 236 against 478.  Splits: one round of items over the 256 CUs; from two splits on (the path that
// leaves its parts).
static int wgrad_whole_splits(int M, int N, int K) {
  if ((N & 255) || (K & 255) || (M & 127) || M < 1024) return 0;
  const long long tiles = (long long)(N / 256) * (K / 256);
  long long s = 256 / tiles, most = M / 512;
  if (s > most) s = most;
  if (s < 2) s = 2;
  // that kernel gives every split the same even number of 64-row slabs: as many splits as have any
  const int slabs = M / 64, per = (int)(((slabs + s - 1) / s + 1) & ~1ll);
  const int n = (slabs + per - 1) / per;
  return n < 2 ? 0 : n;
}
static int wgrad_cols_splits(int M, int N) {
  const int want = 1024 / ((N + 255) / 256), most = (M + 63) / 64;
  const int s = want < most ? want : most;
  return s < 1 ? 1 : s > 32 ? 32 : s;
}
static bool wgrad_sizes_ok(int M, int N, int K) { return M >= 1 && M < 0x7FFFFF00 && N >= 1 && K >= 1 && N <= (1 << 23) && K <= (1 << 23) && (long long)((N + 127) / 128) * ((K + 127) / 128) < (1ll << 30); }
static size_t wgrad_up(size_t n) { return (n + 255) & ~(size_t)255; }
extern "C" size_t uc2_linear_wgrad_workspace(int M, int N, int K) {
  if (!wgrad_sizes_ok(M, N, K)) return 0;
  WgradArgs a{};
  wgrad_plan(M, N, K, a);
  size_t need = a.splits > 1 ? wgrad_up((size_t)a.splits * N * K * 4) + (size_t)a.splits * N * 4 : 0;
  if (const int s = wgrad_whole_splits(M, N, K)) {
    const size_t whole = wgrad_up((size_t)s * N * K * 4) + (size_t)wgrad_cols_splits(M, N) * N * 4;
    if (whole > need) need = whole;
  }
  return need;
}
static void wgrad_sum(const WgradArgs& a, hipStream_t st) {
  const long long n4 = ((long long)a.N * a.K + 3) / 4 + (a.db ? a.N : 0);
  hipLaunchKernelGGL(wgrad_sum_kernel, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, st, a);
}
extern "C" int uc2_linear_wgrad(int M, int N, int K, const void* dy, long long lddy, const void* x, long long ldx, float* dw, long long lddw, float* dbias,
                                void* ws, size_t ws_bytes, void* stream) {
  UC2_CHECK_ARG(wgrad_sizes_ok(M, N, K));
  UC2_CHECK_ARG(dy && x && dw && lddy >= N && ldx >= K && lddw >= K);
  UC2_CHECK_ARG((((uintptr_t)dy | (uintptr_t)x) & 1) == 0 && (((uintptr_t)dw | (uintptr_t)dbias) & 3) == 0);
  const size_t need = uc2_linear_wgrad_workspace(M, N, K);
  UC2_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0));
  WgradArgs a{};
  wgrad_plan(M, N, K, a);
  a.M = M; a.N = N; a.K = K; a.dy = (const bf16*)dy; a.x = (const bf16*)x; a.lddy = lddy; a.ldx = ldx; a.dw = dw; a.lddw = lddw; a.db = dbias;
  a.part = (float*)ws;
  hipStream_t st = (hipStream_t)stream;
  const int whole = wgrad_whole_splits(M, N, K);
  if (whole && (lddy & 7) == 0 && (ldx & 7) == 0 && (((uintptr_t)dy | (uintptr_t)x | (uintptr_t)dw) & 15) == 0 && 2ull * M * lddy < (1ull << 32) && 2ull * M * ldx < (1ull << 32)) {
    const int e = uc2_gemm(1, 1, 1, N, K, M, dy, (int)lddy, x, (int)ldx, dw, K, 1, nullptr, 0, nullptr, nullptr, 0, 1, whole, 12, ws, (size_t)whole * N * K * 4,
                           1 /* UC2_GEMM_DEFER_REDUCE */, stream);
    if (e != 0) return e;
    a.splits = whole;
    a.dsplits = wgrad_cols_splits(M, N);
    a.pdb = (float*)((char*)ws + wgrad_up((size_t)whole * N * K * 4));
    if (dbias) hipLaunchKernelGGL(wgrad_cols_kernel, dim3((N + 255) / 256, a.dsplits), dim3(256), 0, st, a);
    wgrad_sum(a, st);
    UC2_LAUNCH_CHECK();
    return 0;
  }
  if (a.splits > 1) a.pdb = (float*)((char*)ws + wgrad_up((size_t)a.splits * N * K * 4));
  const dim3 grid((unsigned)((a.tn * a.tk * a.splits + 7) / 8 * 8));
  if (N < 8 || K < 8) hipLaunchKernelGGL(wgrad_kernel<true>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(wgrad_kernel<false>, grid, dim3(256), 0, st, a);
  if (a.splits > 1) wgrad_sum(a, st);
  UC2_LAUNCH_CHECK();
  return 0;
}

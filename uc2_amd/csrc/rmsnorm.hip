// Root-mean-square norm of a residual stream, forward and backward, and the e4m3 form of its output that a block-scaled product reads.
//   s = T(x + residual)              the stream that is carried on, rounded to the tensors' type: the norm and its backward read what is kept
//   y = s rstd w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   dx = rstd (g - h mean(g h)) + ds,  g = dy w,  h = s rstd;    dw = sum over rows of dy h
// Everything between one read and one write of each element is fp32.  HBM-bound: forward 4 M H elements (x, residual in; s, y out), backward
// 4 M H (s, dy, ds in; dx out).  A row stays in registers between its reduction and its use: NW waves per row, NV chunks of 8 elements
// per lane (rows up to 64 * 8 * NV * NW wide).  Rows need no alignment: the vector loads are unaligned ones (legal for global memory on
// gfx950), a row's last partial chunk goes element by element.
// Measured (medians): 66560 x 1024 bf16 with a residual: forward 84 us (6.5 TB/s), backward 112 and 5 for dw's sum over the 512 workgroups (4.9 TB/s: it lives on
// three streams in and one out, as a copy does); 33280 x 1024 to e4m3 37 us (6.5 TB/s); 4099 x 1000 fp32 12 + 14 + 4 us (5.4, 4.7 TB/s).
#include "../../include/uc2_hip.h"
#include "common.h"
#include "fp8_block.h"

struct RmsArgs {
  int M, H; float eps;
  const void *x, *res, *s, *dy, *ds; const float* w; const float* rstd_in;
  void *y, *s_out, *dx; float* rstd; float* part;
  unsigned char* q; unsigned* qs; int Kp, ldqs;       // ldqs: the operand's rows
};

// sum over the NW waves of a row (the workgroup holds whole rows: NW = 1 needs no LDS)
template <int NW> __device__ __forceinline__ float row_sum(float v, float* red, int w) {
  v = wave_sum(v);
  if (NW == 1) return v;
  __syncthreads();                                    // (the previous row's sums have been read)
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) t += red[i];
  return t;
}

template <typename T, int NW, int NV, bool Q, bool WHOLE>
__global__ __launch_bounds__(NW == 16 ? 1024 : 256) void rms_fwd_kernel(RmsArgs a) {
  constexpr int RPB = NW == 1 ? 4 : 1;                // rows per workgroup
  __shared__ float red[NW > 1 ? NW : 1];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, w = NW == 1 ? 0 : wv;
  const int row = blockIdx.x * RPB + (NW == 1 ? wv : 0);
  if (row >= a.M) return;                             // (NW > 1: uniform over the workgroup)
  const T* x = (const T*)a.x + (size_t)row * a.H;
  const T* res = a.res ? (const T*)a.res + (size_t)row * a.H : nullptr;
  float v[NV][8];
  float ss = 0.f;
  Blk8<T> x8[NV], r8[NV];
  Blk8<float> w8[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) x8[i].template load<WHOLE>(x, ((i * NW + w) * 64 + lane) * 8, a.H);
  if (res) {
#pragma unroll
    for (int i = 0; i < NV; ++i) r8[i].template load<WHOLE>(res, ((i * NW + w) * 64 + lane) * 8, a.H);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) w8[i].template load<WHOLE>(a.w, ((i * NW + w) * 64 + lane) * 8, a.H);
#pragma unroll
  for (int i = 0; i < NV; ++i) x8[i].template get<WHOLE>(v[i], ((i * NW + w) * 64 + lane) * 8, a.H);
  if (res) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * NW + w) * 64 + lane) * 8;
      float r[8];
      r8[i].template get<WHOLE>(r, c, a.H);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = to_f<T>(from_f<T>(v[i][e] + r[e]));
      blk_store8((T*)a.s_out + (size_t)row * a.H, c, a.H, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  ss = row_sum<NW>(ss, red, w);
  const float r = 1.0f / sqrtf(ss / (float)a.H + a.eps);
  if (a.rstd && w == 0 && lane == 0) a.rstd[row] = r;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = ((i * NW + w) * 64 + lane) * 8;
    float g[8];
    w8[i].template get<WHOLE>(g, c, a.H);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * r * g[e];
    if (a.y) blk_store8((T*)a.y + (size_t)row * a.H, c, a.H, v[i]);
    if (Q) blk_quant_row(v[i], c, a.Kp, a.q + (size_t)row * a.Kp, a.qs + (size_t)(i * NW + w) * a.ldqs + row, lane);
  }
}

// dx and the workgroup's share of dw: rows are dealt to the waves (NW = 1) or workgroups in turn, each lane keeps the sums of its own columns
template <typename T, int NW, int NV, bool WHOLE>
__global__ __launch_bounds__(NW == 16 ? 1024 : 256) void rms_bwd_kernel(RmsArgs a) {
  constexpr int RPB = NW == 1 ? 4 : 1;
  __shared__ float red[NW > 1 ? NW : 1];
  __shared__ float cols[NW == 1 ? 64 * 8 * NV : 1];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, w = NW == 1 ? 0 : wv;
  float dw[NV][8], g[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    blk_load8<WHOLE>(a.w, ((i * NW + w) * 64 + lane) * 8, a.H, g[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  }
  for (int row = blockIdx.x * RPB + (NW == 1 ? wv : 0); row < a.M; row += gridDim.x * RPB) {
    const size_t at = (size_t)row * a.H;
    float h[NV][8], d[NV][8];
    Blk8<T> s8[NV], y8[NV], z8[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) s8[i].template load<WHOLE>((const T*)a.s + at, ((i * NW + w) * 64 + lane) * 8, a.H);
#pragma unroll
    for (int i = 0; i < NV; ++i) y8[i].template load<WHOLE>((const T*)a.dy + at, ((i * NW + w) * 64 + lane) * 8, a.H);
    if (a.ds) {
#pragma unroll
      for (int i = 0; i < NV; ++i) z8[i].template load<WHOLE>((const T*)a.ds + at, ((i * NW + w) * 64 + lane) * 8, a.H);
    }
    const float r = a.rstd_in[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      s8[i].template get<WHOLE>(h[i], ((i * NW + w) * 64 + lane) * 8, a.H);
      y8[i].template get<WHOLE>(d[i], ((i * NW + w) * 64 + lane) * 8, a.H);
    }
    float c = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] *= r;
        dw[i][e] = fmaf(d[i][e], h[i][e], dw[i][e]);
        d[i][e] *= g[i][e];
        c = fmaf(d[i][e], h[i][e], c);
      }
    c = row_sum<NW>(c, red, w) / (float)a.H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = ((i * NW + w) * 64 + lane) * 8;
      float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (a.ds) z8[i].template get<WHOLE>(z, col, a.H);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = fmaf(r, fmaf(-h[i][e], c, d[i][e]), z[e]);
      blk_store8((T*)a.dx + at, col, a.H, z);
    }
  }
  if (!a.part) return;
  float* out = a.part + (size_t)blockIdx.x * a.H;
  if (NW == 1) {                                      // the four waves hold the same columns: added in wave order
    for (int k = 0; k < 4; ++k) {
      if (wv == k)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* p = &cols[(i * 8 + e) * 64 + lane];
            *p = (k ? *p : 0.f) + dw[i][e];
          }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 64 * 8 * NV; i += 256) {
      const int c = ((i >> 9) * 64 + (i & 63)) * 8 + ((i >> 6) & 7);
      if (c < a.H) out[c] = cols[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) blk_store8(out, ((i * NW + w) * 64 + lane) * 8, a.H, dw[i]);
  }
}
// dw[c] = sum of the n workgroups' shares, in a fixed order: 16 columns per workgroup, 64 rows at a time
__global__ __launch_bounds__(1024) void rms_dw_kernel(int n, int H, const float* __restrict__ part, float* __restrict__ dw) {
  __shared__ float red[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  float s = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int i = y; i < n; i += 64) s += part[(size_t)i * H + c];
  }
  red[y][x] = s;
  __syncthreads();
  if (threadIdx.x < 16 && c < H) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) t += red[i][x];
    dw[c] = t;
  }
}

// waves per row and chunks per lane: the fewest registers that hold the row
static void rms_shape(int H, int& nw, int& nv) {
  nw = H <= 2048 ? 1 : H <= 8192 ? 4 : 16;
  const int per = (H + 512 * nw - 1) / (512 * nw);
  nv = per <= 1 && nw == 1 ? 1 : per <= 2 ? 2 : 4;     // (nw = 16: per <= 2)
}
static int rms_bwd_blocks(int M, int H) {
  int nw, nv;
  rms_shape(H, nw, nv);
  const int rows = nw == 1 ? (M + 3) / 4 : M;
  // two workgroups per CU: 66560 x 1024 in 104 us, 110 with twice or four times as many; a single one for two rounds of rows at most: it writes dw itself
  // and saves the second launch (forward and backward of 8 x 1024 in a graph 7.3 us against 8.5; four rounds: 9.4 against 8.7)
  return rows <= 2 ? 1 : rows < 512 ? rows : 512;
}
#define RMS_GO(KERN, T_, ...)                                                                                                       \
  do {                                                                                                                              \
    if (nw == 1) { if (nv == 1) KERN(T_, 1, 1, __VA_ARGS__); else if (nv == 2) KERN(T_, 1, 2, __VA_ARGS__); else KERN(T_, 1, 4, __VA_ARGS__); } \
    else if (nw == 4) { if (nv == 2) KERN(T_, 4, 2, __VA_ARGS__); else KERN(T_, 4, 4, __VA_ARGS__); }                                 \
    else KERN(T_, 16, 2, __VA_ARGS__);                                                                                                \
  } while (0)

extern "C" int uc2_rms_fwd(int dtype, int M, int H, const void* x, const void* residual, const float* gamma, float eps, void* sum, void* y,
                           float* rstd, void* q_out, void* q_scale, void* stream) {
  UC2_CHECK_ARG(dtype == 0 || dtype == 1);
  UC2_CHECK_ARG(M >= 0 && M <= (1 << 30) && H >= 1 && H <= 16384 && eps >= 0.f);
  if (M == 0) return 0;
  UC2_CHECK_ARG(x && gamma && (y || q_out) && (residual == nullptr) == (sum == nullptr) && (q_out == nullptr) == (q_scale == nullptr));
  UC2_CHECK_ARG(((uintptr_t)q_out & 7) == 0 && ((uintptr_t)q_scale & 3) == 0);
  RmsArgs a{};
  a.M = M; a.H = H; a.eps = eps; a.x = x; a.res = residual; a.w = gamma; a.s_out = sum; a.y = y; a.rstd = rstd;
  a.q = (unsigned char*)q_out; a.qs = (unsigned*)q_scale; a.Kp = (H + 127) / 128 * 128; a.ldqs = M;
  int nw, nv;
  rms_shape(H, nw, nv);
  const int rpb = nw == 1 ? 4 : 1, threads = nw == 16 ? 1024 : 256, most = UC2_MOST_BLOCKS(threads) * rpb, el = dtype == 1 ? 2 : 4;
  hipStream_t st = (hipStream_t)stream;
  const bool whole = H % 8 == 0;
#define RMS_F(T_, NW_, NV_, Q_)                                                                                                     \
  do {                                                                                                                              \
    if (whole) hipLaunchKernelGGL((rms_fwd_kernel<T_, NW_, NV_, Q_, true>), dim3(blocks), dim3(threads), 0, st, a);                  \
    else hipLaunchKernelGGL((rms_fwd_kernel<T_, NW_, NV_, Q_, false>), dim3(blocks), dim3(threads), 0, st, a);                       \
  } while (0)
  for (int m0 = 0; m0 < M; m0 += most) {                           // (one launch below 2^26 rows of 2048)
    a.M = M - m0 < most ? M - m0 : most;
    const int blocks = (a.M + rpb - 1) / rpb;
    const size_t at = (size_t)m0 * H * el;
    a.x = (const char*)x + at;
    if (residual) { a.res = (const char*)residual + at; a.s_out = (char*)sum + at; }
    if (y) a.y = (char*)y + at;
    if (rstd) a.rstd = rstd + m0;
    if (q_out) { a.q = (unsigned char*)q_out + (size_t)m0 * a.Kp; a.qs = (unsigned*)q_scale + m0; }
    if (dtype == 1) { if (q_out) RMS_GO(RMS_F, bf16, true); else RMS_GO(RMS_F, bf16, false); }
    else { if (q_out) RMS_GO(RMS_F, float, true); else RMS_GO(RMS_F, float, false); }
    UC2_LAUNCH_CHECK();
  }
  return 0;
}
extern "C" size_t uc2_rms_bwd_workspace(int M, int H) {
  const int n = M > 0 && H > 0 && H <= 16384 ? rms_bwd_blocks(M, H) : 0;
  return n > 1 ? (size_t)n * H * 4 : 0;
}
extern "C" int uc2_rms_bwd(int dtype, int M, int H, const void* dy, const void* dsum, const void* sum, const float* gamma, const float* rstd,
                           void* dx, float* dgamma, void* ws, size_t ws_bytes, void* stream) {
  UC2_CHECK_ARG(dtype == 0 || dtype == 1);
  UC2_CHECK_ARG(M >= 0 && M <= (1 << 30) && H >= 1 && H <= 16384);
  hipStream_t st = (hipStream_t)stream;
  if (M == 0) {
    if (dgamma) hipLaunchKernelGGL(rms_dw_kernel, dim3((H + 15) / 16), dim3(1024), 0, st, 0, H, (const float*)nullptr, dgamma);
    UC2_LAUNCH_CHECK();
    return 0;
  }
  UC2_CHECK_ARG(dy && sum && gamma && rstd && dx);
  const size_t need = uc2_rms_bwd_workspace(M, H);
  UC2_CHECK_ARG(((uintptr_t)dgamma & 3) == 0 && (!dgamma || need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 3) == 0)));
  RmsArgs a{};
  a.M = M; a.H = H; a.s = sum; a.dy = dy; a.ds = dsum; a.w = gamma; a.rstd_in = rstd; a.dx = dx; a.part = !dgamma ? nullptr : need ? (float*)ws : dgamma;
  int nw, nv;
  rms_shape(H, nw, nv);
  const int blocks = rms_bwd_blocks(M, H), threads = nw == 16 ? 1024 : 256;
  const bool whole = H % 8 == 0;
#define RMS_B(T_, NW_, NV_, ...)                                                                                                    \
  do {                                                                                                                              \
    if (whole) hipLaunchKernelGGL((rms_bwd_kernel<T_, NW_, NV_, true>), dim3(blocks), dim3(threads), 0, st, a);                      \
    else hipLaunchKernelGGL((rms_bwd_kernel<T_, NW_, NV_, false>), dim3(blocks), dim3(threads), 0, st, a);                           \
  } while (0)
  if (dtype == 1) RMS_GO(RMS_B, bf16, 0); else RMS_GO(RMS_B, float, 0);
  if (dgamma && need) hipLaunchKernelGGL(rms_dw_kernel, dim3((H + 15) / 16), dim3(1024), 0, st, blocks, H, (const float*)ws, dgamma);
  UC2_LAUNCH_CHECK();
  return 0;
}

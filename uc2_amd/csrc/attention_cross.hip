// Attention from one sequence to the states of another (cross attention): queries [B, Lq, nh, D], keys / values [B, Lk, nkv, D], every
// tensor with its own batch / row / head strides (a fused projection's slices are read in place), nkv dividing nh.
//   x = scale q k^T + key_mask[b, key];  p = softmax_key(x) over the keys that take part;  out = p v
// A key takes no part behind its sequence's length k_lens[b] or where key_mask <= UC2_XATTN_REMOVED (-1e30, -inf included): whatever
// its k / v rows hold (NaN of a padded buffer too) reaches nothing, its gradients are zero.  A row without any key gives zeros and
// passes no gradient.  The softmax runs online in one pass over the keys; scores never reach memory, only one fp32 log2-sum-exp per row.
//
// One skeleton for the three kernels, on the 32 x 32 matrix instructions.  A wave OWNS 32 columns -- packed query rows
// r = i G + g of the G = nh / nkv heads that share a key head (forward, dQ), or keys (dK / dV) -- whose vectors stay in registers as the
// second operand.  The other side STREAMS through LDS in tiles of TT rows, double-buffered, staged through registers so that rows that take no
// part become zeros on the way.  The product (streamed rows x owned columns) leaves a lane with ONE owned column (lane & 31) and 16
// streamed rows per block: the softmax's maximum, sum and rescaling are lane-local but for one exchange between the wave's halves, and
// the weights feed the second product (contraction over streamed rows) straight from the accumulator registers: the order in which that
// product sums its rows is free, so the streamed tile is read transposed (ds_read_b64_tr_b16) in the accumulator's own row order.
// dK / dV of a shared head sum over its G heads by streaming all their rows.  Sums are made in a fixed order: no atomics, same bits every run.
//
// When the owned tiles alone do not fill the chip (single tokens, short batches), the streamed axis is split over workgroups into fp32
// partials (outputs with maximum and sum; gradients), joined by a second small kernel.
// Roundings below fp32: the weights (forward, dV) and the score gradients (dQ, dK) to bf16 where they enter the second product, results to T; each at most half
// a step of its value, so they leave the results off by 2.2e-3 to 2.5e-3 of their norm where one rounding of the result makes 1.7e-3.
// Measured, bf16 (the least and the median of 23 launches in a row, under which the clock falls): 2 x 2048 x 4096, 16 heads of 64: forward 103 - 115 us (0.60 - 0.67
// PF/s), backward 271 - 296 (0.58 - 0.63, 0.81 - 0.89 with the products that it makes twice); the vector pipe is busy 50 % (forward) and 44 % of that, the
// matrix pipe 28 % and 40 %, and two waves per SIMD, all that the registers hold, overlap them little (products between the vector instructions of one
// wave, raised priorities: no gain).  With dropout, which draws a hash per weight and loads no fragment ahead: 147 - 154 and 379 - 402.  104 x 60 x 100, 12
// heads of 64: 17 + 42 us (its bytes at a copy's rate: 14 + 23).  16 x 1 x 16384, 16 heads over 4 key heads: 26 us and 5 for the join (4.8 TB/s).  fp32, 8 x 77 x 211: 13 + 5
// and 35 + 6 us.
#include "../../include/uc2_hip.h"
#include "common.h"

typedef __attribute__((ext_vector_type(4))) __bf16 xa_bf16x4;

#define XA_LOG2E 1.4426950408889634f
#define XA_REMOVED (-1e30f)

struct XaView { const char* p; long long sb, sl, sh; };          // byte strides of batch, row, head
struct XaOut { char* p; long long sb, sl, sh; };

// a kernel's work: owned tiles per (batch, key head), splits of the streamed axis, blocks; partials [splits][B nkv][rows][..] (dkv: dK, then dV, per split)
struct XaSide { int tiles, splits, blocks; float* part; };

struct XaArgs {
  int B, Lq, Lk, nkv, G, R;                                       // R = Lq G packed rows per (batch, key head)
  int BH;                                                         // B nkv
  XaSide fwd, dq, dkv;
  XaView q, k, v, o, dout;
  float* o32;                                                     // bf16: the output before its rounding, [B nkv][R][D], for delta
  float* delta;                                                   // [B nkv][R], where a kernel of its own forms them
  XaOut out, gq, gk, gv;
  const float* kmask; long long kmask_sb; const int* klens;
  float scale, scale2;                                            // scale2 = scale log2 e
  float* lse;                                                     // [B nkv][R], base 2
  float* pml;                                                     // the forward's maxima and sums [splits][B nkv][R][2]
  uint32_t thresh; float keep_scale; const uint64_t* seed_ptr; uint64_t seed_imm; int nh;
};

template <typename T, int D> struct XaCfg {
  static constexpr int RB = D * (int)sizeof(T);                   // bytes of a row
  static constexpr int CPR = RB / 16;                             // 16-byte chunks of a row
  // streamed rows per tile: 64 rows of 128 bytes or less, 32 longer ones: 32 KiB of LDS for two double-buffered tensors (64 KiB for fp32
  // at D = 128), and at most 128 staging registers in a workgroup of one wave
  static constexpr int TT = RB <= 128 ? 64 : 32;
  static constexpr int NB = TT / 32;                              // 32-row blocks per tile
  static constexpr int KS = sizeof(T) == 2 ? D / 16 : D / 8;      // chunks a lane holds of an owned vector
  static constexpr int DB = D / 32;                               // 32-wide blocks of the head dimension
};

// chunk swizzle of a row.  256 bytes (64 banks) hold 16 chunks: the 16 rows that a quarter wave reads one chunk column of fall on 16 of them, and so do
// the 4 rows x 2 chunks x 2 halves of a transposing read twice over, which is its least (the first choice, by the row's low three bits, cost a third of
// the LDS cycles in conflicts)
template <int CPR> __device__ __forceinline__ int xa_swz(int row) {
  if (CPR == 4) return (row >> 2) & 3;
  if (CPR == 8) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);
  return ((row & 1) << 3) | ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);
}

__device__ __forceinline__ f32x16 xa_all(float x) { return f32x16{x, x, x, x, x, x, x, x, x, x, x, x, x, x, x, x}; }
__device__ __forceinline__ f32x16 xa_zero() { return xa_all(0.f); }
template <typename T, int D> struct XaMma;
template <int D> struct XaMma<bf16, D> {
  typedef XaCfg<bf16, D> C;
  typedef bf16x8 Frag;
  // acc[16] += rows blk*32.. of the tile (lane's row: lane & 31) against the owned vectors
  static __device__ __forceinline__ f32x16 rows(const char* lds, int blk, const Frag (&own)[C::KS], int lane, f32x16 acc = xa_zero()) {
    const int row = blk * 32 + (lane & 31), h = lane >> 5, sw = xa_swz<C::CPR>(row);
#pragma unroll
    for (int s = 0; s < C::KS; ++s) {
      const bf16x8 a = *reinterpret_cast<const bf16x8*>(lds + row * C::RB + (((2 * s + h) ^ sw) << 4));
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, own[s], acc, 0, 0, 0);
    }
    return acc;
  }
  // out[db] (head dimension x owned columns) += tile rows^T x w[16] (the accumulator order of rows())
  typedef bf16x8 Turned[C::DB];                                   // 16 rows of the tile, transposed
  static __device__ __forceinline__ void turn(const char* lds, int blk, int ks, Turned& a, int lane) {
    const int h = lane >> 5, i = lane & 15, dh = (lane >> 4) & 1;
    const int row0 = blk * 32 + 16 * ks + 4 * h + (i >> 2), row1 = row0 + 8;
#pragma unroll
    for (int db = 0; db < C::DB; ++db) {
      const int c = 4 * db + 2 * dh + ((i >> 1) & 1), sub = (i & 1) * 8;
      typedef __attribute__((address_space(3))) short4v* lp;
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + row0 * C::RB + ((c ^ xa_swz<C::CPR>(row0)) << 4) + sub));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + row1 * C::RB + ((c ^ xa_swz<C::CPR>(row1)) << 4) + sub));
      a[db] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  static __device__ __forceinline__ void cols(const Turned& a, int ks, const float (&w)[16], f32x16 (&out)[C::DB]) {
    bf16x8 b;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = (bf16)w[8 * ks + j];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) out[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[db], b, out[db], 0, 0, 0);
  }
  static __device__ __forceinline__ void cols(const char* lds, int blk, const float (&w)[16], f32x16 (&out)[C::DB], int lane) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      Turned a;
      turn(lds, blk, ks, a, lane);
      cols(a, ks, w, out);
    }
  }
};
template <int D> struct XaMma<float, D> {
  typedef XaCfg<float, D> C;
  typedef f32x4 Frag;
  struct Turned {};                                               // (read value by value)
  static __device__ __forceinline__ f32x16 rows(const char* lds, int blk, const Frag (&own)[C::KS], int lane, f32x16 acc = xa_zero()) {
    const int row = blk * 32 + (lane & 31), h = lane >> 5, sw = xa_swz<C::CPR>(row);
#pragma unroll
    for (int s = 0; s < C::KS; ++s) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + row * C::RB + (((2 * s + h) ^ sw) << 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], own[s][j], acc, 0, 0, 0);
    }
    return acc;
  }
  static __device__ __forceinline__ void cols(const char* lds, int blk, const float (&w)[16], f32x16 (&out)[C::DB], int lane) {
    const int h = lane >> 5, l31 = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = blk * 32 + 8 * (r >> 2) + 4 * h + (r & 3), sw = xa_swz<C::CPR>(row);
#pragma unroll
      for (int db = 0; db < C::DB; ++db) {
        const float a = *reinterpret_cast<const float*>(lds + row * C::RB + (((8 * db + (l31 >> 2)) ^ sw) << 4) + (l31 & 3) * 4);
        out[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[r], out[db], 0, 0, 0);
      }
    }
  }
};

template <typename T, int D> __device__ __forceinline__ void xa_turn(const char* lds, int blk, typename XaMma<T, D>::Turned (&a)[2], int lane) {
  XaMma<T, D>::turn(lds, blk, 0, a[0], lane);
  XaMma<T, D>::turn(lds, blk, 1, a[1], lane);
}
// the order of a block's start: READS reads of LDS, then PRODUCTS matrix instructions with MORE reads (for the second products) between them
template <int READS, int PRODUCTS, int MORE> __device__ __forceinline__ void xa_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, (MORE + PRODUCTS - 1) / PRODUCTS, 0);
  }
}

// position of packed row r: (query i, head g of the group)
__device__ __forceinline__ void xa_split(const XaArgs& a, int r, int& i, int& g) {
  if (a.G == 1) { i = r; g = 0; } else { i = (int)((unsigned)r / (unsigned)a.G); g = r - i * a.G; }
}
// rows of a key-like tensor (PACKED false) or of a query-like one (packed rows)
template <bool PACKED> __device__ __forceinline__ const char* xa_row(const XaArgs& a, const XaView& x, int b, int kvh, int r) {
  if (!PACKED) return x.p + b * x.sb + (long long)r * x.sl + kvh * x.sh;
  int i, g;
  xa_split(a, r, i, g);
  return x.p + b * x.sb + (long long)i * x.sl + (long long)(kvh * a.G + g) * x.sh;
}
// base-2 additive mask of a key from the mask's entry (read apart: a tile's loads are issued together and nothing waits for one of them before put()
// does); -inf: no part
__device__ __forceinline__ float xa_key_raw(const XaArgs& a, int b, int key, int len) { return a.kmask ? a.kmask[b * a.kmask_sb + min(key, len - 1)] : 0.f; }
__device__ __forceinline__ float xa_key_bias(const XaArgs& a, float raw, int key, int len) {
  return key >= len || (a.kmask && raw <= XA_REMOVED) ? -INFINITY : raw * XA_LOG2E;
}
// A fragment read from memory in front of a loop that has loads in flight: waited for here, or the compiler, which cannot tell the first round from the others,
// waits for every load of the loop in front of the fragment's first use (2048 x 4096, 16 heads of 128, forward: 138 us, so 123)
template <typename F, int N> __device__ __forceinline__ void xa_arrived(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Staging of TT rows x D of two tensors by NT threads, through registers.  A thread's chunks lie at the same 32-bit offsets from the tile's first row in every
// tile (packed rows: where G divides TT), so a tile's loads cost no vector arithmetic; no branch around them: rows behind the last one load that
// one's, and keep() clears what takes no part on the way into LDS.
template <typename T, int D, int NT, bool PACKED> struct XaStage {
  typedef XaCfg<T, D> C;
  static constexpr int N = C::TT * C::CPR / NT;                  // chunks per thread and tensor
  static_assert(N >= 1 && C::TT * C::CPR % NT == 0, "");
  typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
  u32x4 x[N], y[N];
  const char *px, *py;                                            // row 0 of the two tensors (wave-uniform)
  unsigned ox[N], oy[N];
  int limit, t;
  __device__ __forceinline__ unsigned off(const XaArgs& a, const XaView& X, int r, int c) const {
    if (!PACKED || a.G == 1) return (unsigned)(r * (int)X.sl) + c * 16;
    const int i = (int)((unsigned)r / (unsigned)a.G);
    return (unsigned)(i * (int)X.sl + (r - i * a.G) * (int)X.sh) + c * 16;
  }
  __device__ __forceinline__ void init(const XaArgs& a, const XaView& X, const XaView& Y, int b, int kvh, int limit_, int t_) {
    limit = limit_; t = t_;
    px = X.p + b * X.sb + (PACKED ? kvh * a.G : kvh) * X.sh;
    py = Y.p + b * Y.sb + (PACKED ? kvh * a.G : kvh) * Y.sh;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = t + n * NT;
      ox[n] = off(a, X, idx / C::CPR, idx % C::CPR);
      oy[n] = off(a, Y, idx / C::CPR, idx % C::CPR);
    }
  }
  // every chunk of tile tt (tt * TT < limit)
  __device__ __forceinline__ void load(const XaArgs& a, const XaView& X, const XaView& Y, int tt) {
    const int row0 = tt * C::TT;
    const bool even = !PACKED || a.G == 1 || C::TT % a.G == 0;    // (uniform)
    if (even && row0 + C::TT <= limit) {
      const int i0 = PACKED ? row0 / a.G : row0;
      const char *qx = px + (long long)i0 * X.sl, *qy = py + (long long)i0 * Y.sl;
#pragma unroll
      for (int n = 0; n < N; ++n) { x[n] = *reinterpret_cast<const u32x4*>(qx + ox[n]); y[n] = *reinterpret_cast<const u32x4*>(qy + oy[n]); }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int idx = t + n * NT, r = min(row0 + idx / C::CPR, limit - 1), c = idx % C::CPR;
        int i = r, g = 0;
        if (PACKED) xa_split(a, r, i, g);
        x[n] = *reinterpret_cast<const u32x4*>(px + (long long)i * X.sl + (long long)g * X.sh + c * 16);
        y[n] = *reinterpret_cast<const u32x4*>(py + (long long)i * Y.sl + (long long)g * Y.sh + c * 16);
      }
    }
  }
  // fix (uniform): some row of the tile takes no part; bit r of part: row r does
  __device__ __forceinline__ void store(char* lx, char* ly, bool fix, unsigned long long part) {
    if (fix) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const bool keep = (part >> ((t + n * NT) / C::CPR)) & 1;
        if (!keep) { x[n] = u32x4{0, 0, 0, 0}; y[n] = u32x4{0, 0, 0, 0}; }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = t + n * NT, row = idx / C::CPR, c = idx % C::CPR;
      const int o = row * C::RB + ((c ^ xa_swz<C::CPR>(row)) << 4);
      *reinterpret_cast<u32x4*>(lx + o) = x[n];
      *reinterpret_cast<u32x4*>(ly + o) = y[n];
    }
  }
};

// -delta of a staged tile of packed rows: the values of `out` (bf16: before their rounding, see xa_delta_row) beside XaStage's chunks of dout, multiplied
// on the way into LDS and summed over a row's CPR neighbouring threads
template <typename T, int D, int NT> struct XaDelta {
  typedef XaCfg<T, D> C;
  static constexpr int N = C::TT * C::CPR / NT, E = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
  f32x4 z[N][E / 4];
  const char* p; int t;
  __device__ __forceinline__ void init(const XaArgs& a, int bh, int b, int kvh, int t_) {
    t = t_;
    p = sizeof(T) == 2 ? reinterpret_cast<const char*>(a.o32 + (size_t)bh * a.R * D) : a.o.p + b * a.o.sb + (long long)(kvh * a.G) * a.o.sh;
  }
  __device__ __forceinline__ void load(const XaArgs& a, int tt) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = t + n * NT, r = min(tt * C::TT + idx / C::CPR, a.R - 1), c = idx % C::CPR;
      const char* at = p;
      if (sizeof(T) == 2) {
        at += ((long long)r * D + c * 8) * 4;
      } else {
        int i, g;
        xa_split(a, r, i, g);
        at += (long long)i * a.o.sl + (long long)g * a.o.sh + c * 16;
      }
#pragma unroll
      for (int j = 0; j < E / 4; ++j) z[n][j] = reinterpret_cast<const f32x4*>(at)[j];
    }
  }
  __device__ __forceinline__ void store(const XaArgs& a, const u32x4 (&y)[N], float* d, int tt) {
    typedef T V __attribute__((ext_vector_type(E)));
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = t + n * NT, row = idx / C::CPR;
      const V g = __builtin_bit_cast(V, y[n]);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(z[n][e / 4][e % 4], (float)g[e], s);
#pragma unroll
      for (int k = 1; k < C::CPR; k <<= 1) s += __shfl_xor(s, k);
      if (idx % C::CPR == 0) d[row] = tt * C::TT + row < a.R ? -s : 0.f;
    }
  }
};

// owned vectors of the lane: column r (query row or key), zeros where it takes no part
template <typename T, int D, bool PACKED>
__device__ __forceinline__ void xa_own(const XaArgs& a, const XaView& X, int b, int kvh, int r, bool take, int lane, typename XaMma<T, D>::Frag (&f)[XaCfg<T, D>::KS]) {
  typedef typename XaMma<T, D>::Frag Frag;
  const int h = lane >> 5;
  if (take) {
    const char* p = xa_row<PACKED>(a, X, b, kvh, r);
#pragma unroll
    for (int s = 0; s < XaCfg<T, D>::KS; ++s) f[s] = *reinterpret_cast<const Frag*>(p + (2 * s + h) * 16);
  } else {
#pragma unroll
    for (int s = 0; s < XaCfg<T, D>::KS; ++s) f[s] = __builtin_bit_cast(Frag, uint4{0, 0, 0, 0});
  }
}
// delta[r] = dout . out of an owned row, with the output as it was before its rounding to bf16: a row's gradients of the scores, p (dp - delta), nearly
// cancel where it has few keys or one that outweighs the others, and an output off by 2^-9 there left dq and dk off by 4e-3 to 8e-3 of their norm
// (2 to 40 keys; with this 2.5e-3, what the roundings of the score gradients and of the result make)
template <typename T, int D>
__device__ __forceinline__ float xa_delta_row(const XaArgs& a, int bh, int b, int kvh, int r, bool take, int lane, const typename XaMma<T, D>::Frag (&go)[XaCfg<T, D>::KS]) {
  constexpr int E = 16 / sizeof(T);
  float s = 0.f;
  if (take) {
    const char* p = sizeof(T) == 2 ? reinterpret_cast<const char*>(a.o32 + ((size_t)bh * a.R + r) * D) : xa_row<true>(a, a.o, b, kvh, r);
#pragma unroll
    for (int k = 0; k < XaCfg<T, D>::KS; ++k)
#pragma unroll
      for (int j = 0; j < E / 4; ++j) {
        const f32x4 o = reinterpret_cast<const f32x4*>(p + (2 * k + (lane >> 5)) * E * 4)[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(o[e], (float)go[k][4 * j + e], s);
      }
  }
  return s + __shfl_xor(s, 32);
}
// 4 consecutive values of the head dimension
__device__ __forceinline__ void xa_put4(bf16* p, float a, float b, float c, float d) {
  *reinterpret_cast<xa_bf16x4*>(p) = xa_bf16x4{(bf16)a, (bf16)b, (bf16)c, (bf16)d};
}
__device__ __forceinline__ void xa_put4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
template <typename T, int DB> __device__ __forceinline__ void xa_put_row(char* row, const f32x16 (&o)[DB], float mul, int lane) {
  T* p = reinterpret_cast<T*>(row) + 4 * (lane >> 5);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int k = 0; k < 4; ++k) xa_put4(p + 32 * db + 8 * k, o[db][4 * k] * mul, o[db][4 * k + 1] * mul, o[db][4 * k + 2] * mul, o[db][4 * k + 3] * mul);
}

// block -> (batch and key head, owned tile, split): blocks go to the 8 XCDs in turn, the tiles and splits of one (batch, key head) share its
// streamed rows, so they are put on one XCD and its L2 (worth nothing below 8 heads: plain order there)
__device__ __forceinline__ bool xa_block(const XaArgs& a, const XaSide& side, int blk, int& bh, int& tile, int& split) {
  const int per = side.tiles * side.splits;
  if (a.BH >= 8) {
    const int x = blk & 7, n = blk >> 3, grp = n / per;
    bh = grp * 8 + x;
    blk = n - grp * per;
  } else {
    bh = blk / per;
    blk -= bh * per;
  }
  tile = blk / side.splits;
  split = blk - tile * side.splits;
  return bh < a.BH;
}
// over the wave's two halves
__device__ __forceinline__ float xa_max2(float x) {
  typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
  const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ int xa_len(const XaArgs& a, int b) { return a.klens ? max(0, min(a.klens[b], a.Lk)) : a.Lk; }
// Whether just one key of the sequence takes part.  The softmax over one key is constant, so dq and dk are zero; p (dp - delta) would leave fp32's rounding
// noise there, dp and delta being sums of the same products in two orders.  Their last factor, the scale, is zero then (NaN stays NaN).  seen: keys that take part
// among those that the wave has met, `all`: it has met every one; the mask is read, up to its second key, by a wave that met one of them only (one that met
// none has zeros to scale).
__device__ __forceinline__ bool xa_alone(const XaArgs& a, int b, int len, int lane, int seen, bool all) {
  if (!a.kmask) return len == 1;
  if (seen != 1 || all) return seen == 1;
  int n = 0;
  for (int j0 = 0; n < 2 && j0 < len; j0 += 256) {
    float raw[4];                                                 // (four loads in flight)
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = xa_key_raw(a, b, j0 + 64 * u + lane, len);
#pragma unroll
    for (int u = 0; u < 4; ++u) n += __popcll(__ballot(j0 + 64 * u + lane < len && !(raw[u] <= XA_REMOVED)));
  }
  return n == 1;
}

template <typename T, int D, int NS, bool DROP>
__global__ __launch_bounds__(NS * 64) void xattn_fwd_kernel(XaArgs a) {
  typedef XaCfg<T, D> C;
  typedef XaMma<T, D> M;
  __shared__ __attribute__((aligned(16))) char lk[2][C::TT * C::RB], lv[2][C::TT * C::RB];
  __shared__ __attribute__((aligned(16))) float lb[2][C::TT];
  __shared__ __attribute__((aligned(16))) uint32_t lh[2][DROP ? C::TT : 4];
  int bh, tile, split;
  if (!xa_block(a, a.fwd, blockIdx.x, bh, tile, split)) return;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, b = bh / a.nkv, kvh = bh - b * a.nkv;
  const int r = (tile * NS + w) * 32 + (lane & 31);
  const bool mine = r < a.R, live = (tile * NS + w) * 32 < a.R;      // live: the wave has a row (the others only stage)
  const int len = xa_len(a, b), nt = (len + C::TT - 1) / C::TT, per = (nt + a.fwd.splits - 1) / a.fwd.splits;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  const uint64_t seed = DROP ? a.seed_imm + (a.seed_ptr ? *a.seed_ptr : 0ull) : 0ull;
  uint32_t hq = 0;
  if (DROP && mine) { int i, g; xa_split(a, r, i, g); hq = attn_line_hash(seed, b * a.nh + kvh * a.G + g, i, UC2_ATTN_SALT_Q); }

  typename M::Frag q[C::KS];
  xa_own<T, D, true>(a, a.q, b, kvh, r, mine, lane, q);
  f32x16 o[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  XaStage<T, D, NS * 64, false> st;
  st.init(a, a.k, a.v, b, kvh, len, t);
  float raw = 0.f;                                                // (in every wave: it clears its own rows by it)
  auto fetch = [&](int tt) __attribute__((always_inline)) {
    st.load(a, a.k, a.v, tt);
    raw = xa_key_raw(a, b, tt * C::TT + (lane & (C::TT - 1)), len);
  };
  auto put = [&](int tt, int buf) __attribute__((always_inline)) {
    const float bias = xa_key_bias(a, raw, tt * C::TT + (lane & (C::TT - 1)), len);
    st.store(lk[buf], lv[buf], a.kmask != nullptr || (tt + 1) * C::TT > len, __ballot(bias != -INFINITY));
    if (t < C::TT) { lb[buf][t] = bias; if (DROP) lh[buf][t] = attn_line_hash(seed, bh, tt * C::TT + t, UC2_ATTN_SALT_K); }
  };
  if (t0 < t1) { fetch(t0); put(t0, 0); }
  xa_arrived(q);
  __syncthreads();
  int buf = 0;
  for (int tt = t0; tt < t1; ++tt) {
    if (tt + 1 < t1) fetch(tt + 1);
    const bool masked = a.kmask != nullptr || (tt + 1) * C::TT > len || a.scale2 < 0.f;      // (uniform)
    // m is the maximum the weights are taken against: brought up only once a row's has grown by 2^8 (weights up to 256 lose nothing in fp32 or bf16,
    // and the output and sum are rescaled in the first tiles only)
    auto raise = [&](float mx) __attribute__((always_inline)) {
      mx = xa_max2(mx);
      if (!__any(mx > m + 8.f)) return;
      const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= al;
      m = mn;
    };
    auto weigh = [&](int n, const f32x16& s, float sc, float mu, float (&p)[16]) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint4 hk = {0, 0, 0, 0};
        if (DROP) hk = *reinterpret_cast<const uint4*>(&lh[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
        const uint32_t hh[4] = {hk.x, hk.y, hk.z, hk.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = __builtin_amdgcn_exp2f(fmaf(s[4 * k + e], sc, -mu));
          l += v;
          p[4 * k + e] = DROP ? (attn_keep(hq, hh[e], a.thresh) ? v * a.keep_scale : 0.f) : v;
        }
      }
    };
    if (live && !masked && sizeof(T) == 2) {
      if constexpr (sizeof(T) == 2) {
        // a whole tile: its LDS reads issued in front of what waits for them, the values' during the first product (2 x 2048 x 4096, 16 heads: 112 -> 106 us)
        f32x16 s[C::NB];
        typename M::Turned v[C::NB][2];
#pragma unroll
        for (int n = 0; n < C::NB; ++n) s[n] = M::rows(lk[buf], n, q, lane);
#pragma unroll
        for (int n = 0; n < C::NB; ++n) xa_turn<T, D>(lv[buf], n, v[n], lane);
        xa_ahead<C::NB * C::KS, C::NB * C::KS, C::NB * C::DB * 4>();
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < C::NB; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[n][e]);
        raise(mx * a.scale2);
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int n = 0; n < C::NB; ++n) {
          float p[16];
          weigh(n, s[n], a.scale2, mu, p);
          M::cols(v[n][0], 0, p, o);
          M::cols(v[n][1], 1, p, o);
        }
      }
    } else if (live) {
      f32x16 s[C::NB];
      const int left = len - tt * C::TT;                          // keys from this tile on: a block of 32 behind them is not computed
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < C::NB; ++n) {
        if (n > 0 && n * 32 >= left) break;
        s[n] = M::rows(lk[buf], n, q, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                             // x = scale2 s + mask, in base 2
          f32x4 bv = {0.f, 0.f, 0.f, 0.f};
          if (masked) bv = *reinterpret_cast<const f32x4*>(&lb[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
#pragma unroll
          for (int e = 0; e < 4; ++e) { s[n][4 * k + e] = fmaf(s[n][4 * k + e], a.scale2, bv[e]); mx = fmaxf(mx, s[n][4 * k + e]); }
        }
      }
      raise(mx);
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int n = 0; n < C::NB; ++n) {
        if (n > 0 && n * 32 >= left) break;
        float p[16];
        weigh(n, s[n], 1.f, mu, p);
        M::cols(lv[buf], n, p, o, lane);
      }
    }
    if (tt + 1 < t1) put(tt + 1, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  l += __shfl_xor(l, 32);
  if (!mine) return;
  if (a.fwd.splits == 1) {
    int i, g;
    xa_split(a, r, i, g);
    const float inv = l > 0.f ? 1.0f / l : (l == l ? 0.f : l);     // no key: zeros; NaN stays NaN
    xa_put_row<T, C::DB>(a.out.p + b * a.out.sb + (long long)i * a.out.sl + (long long)(kvh * a.G + g) * a.out.sh, o, inv, lane);
    if (a.lse && lane < 32) a.lse[(size_t)bh * a.R + r] = m + __log2f(l);
    if (sizeof(T) == 2 && a.o32) xa_put_row<float, C::DB>(reinterpret_cast<char*>(a.o32 + ((size_t)bh * a.R + r) * D), o, inv, lane);
  } else {
    const size_t row = ((size_t)split * a.BH + bh) * a.R + r;
    xa_put_row<float, C::DB>(reinterpret_cast<char*>(a.fwd.part + row * D), o, 1.0f, lane);
    if (lane < 32) { a.pml[2 * row] = m; a.pml[2 * row + 1] = l; }
  }
}

// joins the splits of the forward (64 at most): W waves per row; lane s of each first holds split s's factor, then the waves share the splits, a lane
// summing its elements, and are added in wave order (one wave for 32 splits of 256 rows took 11 us: four trips to memory one after the other)
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void xattn_join_kernel(XaArgs a) {
  constexpr int E = D / 64 > 0 ? D / 64 : 1;
  __shared__ float red[W > 1 ? W * 64 * E : 1];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, w = W > 1 ? wv : 0;
  const long long row = W > 1 ? (long long)blockIdx.x : (long long)blockIdx.x * 4 + wv, rows = (long long)a.BH * a.R;
  if (row >= rows) return;                                        // (W > 1: uniform)
  const int bh = (int)(row / a.R), r = (int)(row - (long long)bh * a.R);
  float m = -INFINITY, l = 0.f;
  if (lane < a.fwd.splits) { const float2 v = *reinterpret_cast<const float2*>(a.pml + 2 * (lane * rows + row)); m = v.x; l = v.y; }
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  const float top = wave_max(m), mu = top == -INFINITY ? 0.f : top;
  const float f = __builtin_amdgcn_exp2f(m - mu);
  l = wave_sum(f * l);
  const float* p = a.fwd.part + row * D + (D >= 64 ? lane : lane % D);
#pragma unroll 8
  for (int s = w; s < a.fwd.splits; s += W) {
    const float x = __shfl(f, s);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(x, p[s * rows * D + 64 * e], o[e]);
  }
  if (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) red[(w * E + e) * 64 + lane] = o[e];
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < W; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += red[(k * E + e) * 64 + lane];
  }
  const float inv = l > 0.f ? 1.0f / l : (l == l ? 0.f : l);
  const int b = bh / a.nkv, kvh = bh - b * a.nkv;
  int i, g;
  xa_split(a, r, i, g);
  T* out = reinterpret_cast<T*>(a.out.p + b * a.out.sb + (long long)i * a.out.sl + (long long)(kvh * a.G + g) * a.out.sh);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (D >= 64 || lane < D) {
      out[lane + 64 * e] = from_f<T>(o[e] * inv);
      if (sizeof(T) == 2 && a.o32) a.o32[row * D + lane + 64 * e] = o[e] * inv;
    }
  if (a.lse && lane == 0) a.lse[row] = top + __log2f(l);
}

// The backward is one launch of two kinds of workgroups, dK / dV and dQ: neither needs the other (each forms delta[r] = dout . out itself, but for long
// key axes), so a short problem pays one launch and one latency instead of two.
template <typename T, int D, bool DROP> struct XaLds {
  typedef XaCfg<T, D> C;
  __attribute__((aligned(16))) char x[2][C::TT * C::RB], y[2][C::TT * C::RB];
  __attribute__((aligned(16))) float s[2][C::TT], d[2][C::TT];
  __attribute__((aligned(16))) uint32_t h[2][DROP ? C::TT : 4];
};

// dQ (owned query rows, streamed keys)
//   dx = p (dp - delta),  dp = dout v^T (dropped as the forward's weights were),  dq = scale dx k  (zero where one key takes part: xa_alone)
template <typename T, int D, int NS, bool DROP, bool PRE>
__device__ __forceinline__ void xa_dq(const XaArgs& a, int blk, XaLds<T, D, DROP>& sh) {
  typedef XaCfg<T, D> C;
  typedef XaMma<T, D> M;
  int bh, tile, split;
  if (!xa_block(a, a.dq, blk, bh, tile, split)) return;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, b = bh / a.nkv, kvh = bh - b * a.nkv;
  const int r = (tile * NS + w) * 32 + (lane & 31);
  const bool mine = r < a.R, live = (tile * NS + w) * 32 < a.R;      // live: the wave has a row (the others only stage)
  const int len = xa_len(a, b), nt = (len + C::TT - 1) / C::TT, per = (nt + a.dq.splits - 1) / a.dq.splits;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  const uint64_t seed = DROP ? a.seed_imm + (a.seed_ptr ? *a.seed_ptr : 0ull) : 0ull;
  uint32_t hq = 0;
  if (DROP && mine) { int i, g; xa_split(a, r, i, g); hq = attn_line_hash(seed, b * a.nh + kvh * a.G + g, i, UC2_ATTN_SALT_Q); }

  typename M::Frag q[C::KS], go[C::KS];
  xa_own<T, D, true>(a, a.q, b, kvh, r, mine, lane, q);
  xa_own<T, D, true>(a, a.dout, b, kvh, r, mine, lane, go);
  float lse = INFINITY;
  const float delta = !PRE ? xa_delta_row<T, D>(a, bh, b, kvh, r, mine, lane, go) : mine ? a.delta[(size_t)bh * a.R + r] : 0.f;
  if (mine) {
    lse = a.lse[(size_t)bh * a.R + r];
    if (lse == -INFINITY) lse = INFINITY;                          // a row without any key: p = 0
  }
  const float nlse = -lse;
  const f32x16 ndelta = xa_all(DROP ? 0.f : -delta);              // dp's sums start at -delta (dropout scales dp first)
  constexpr bool AHEAD = sizeof(T) == 2 && !DROP;
  f32x16 dq[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[db][e] = 0.f;
  XaStage<T, D, NS * 64, false> st;
  st.init(a, a.k, a.v, b, kvh, len, t);
  float raw = 0.f;                                                // (in every wave: it clears its own rows by it)
  int seen = 0;                                                   // keys of the split that take part
  auto fetch = [&](int tt) __attribute__((always_inline)) {
    st.load(a, a.k, a.v, tt);
    raw = xa_key_raw(a, b, tt * C::TT + (lane & (C::TT - 1)), len);
  };
  auto put = [&](int tt, int buf) __attribute__((always_inline)) {
    const float bias = xa_key_bias(a, raw, tt * C::TT + (lane & (C::TT - 1)), len);
    const unsigned long long take = __ballot(bias != -INFINITY);
    seen += __popcll(take << (64 - C::TT));
    st.store(sh.x[buf], sh.y[buf], a.kmask != nullptr || (tt + 1) * C::TT > len, take);
    if (t < C::TT) { sh.s[buf][t] = bias; if (DROP) sh.h[buf][t] = attn_line_hash(seed, bh, tt * C::TT + t, UC2_ATTN_SALT_K); }
  };
  if (t0 < t1) { fetch(t0); put(t0, 0); }
  xa_arrived(q);
  xa_arrived(go);
  __syncthreads();
  int buf = 0;
  for (int tt = t0; tt < t1; ++tt) {
    if (tt + 1 < t1) fetch(tt + 1);
    const bool masked = a.kmask != nullptr || (tt + 1) * C::TT > len;
#pragma unroll
    for (int n = 0; n < C::NB; ++n) {
      if (!live || tt * C::TT + n * 32 >= len) break;
      const f32x16 s = M::rows(sh.x[buf], n, q, lane);
      const f32x16 dp = M::rows(sh.y[buf], n, go, lane, ndelta);
      typename M::Turned tx[2];
      if constexpr (AHEAD) {
        xa_turn<T, D>(sh.x[buf], n, tx, lane);
        xa_ahead<2 * C::KS, 2 * C::KS, 8 * C::DB>();
      }
      float ds[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 bv = {nlse, nlse, nlse, nlse};
        uint4 hk = {0, 0, 0, 0};
        if (masked) bv += *reinterpret_cast<const f32x4*>(&sh.s[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
        if (DROP) hk = *reinterpret_cast<const uint4*>(&sh.h[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
        const uint32_t hh[4] = {hk.x, hk.y, hk.z, hk.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * k + e], a.scale2, bv[e]));
          ds[4 * k + e] = p * (DROP ? (attn_keep(hq, hh[e], a.thresh) ? dp[4 * k + e] * a.keep_scale : 0.f) - delta : dp[4 * k + e]);
        }
      }
      if constexpr (AHEAD) { M::cols(tx[0], 0, ds, dq); M::cols(tx[1], 1, ds, dq); }
      else M::cols(sh.x[buf], n, ds, dq, lane);
    }
    if (tt + 1 < t1) put(tt + 1, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  const float scale = xa_alone(a, b, len, lane, seen, a.dq.splits == 1) ? 0.f : a.scale;
  if (!mine) return;
  if (a.dq.splits == 1) {
    int i, g;
    xa_split(a, r, i, g);
    xa_put_row<T, C::DB>(a.gq.p + b * a.gq.sb + (long long)i * a.gq.sl + (long long)(kvh * a.G + g) * a.gq.sh, dq, scale, lane);
  } else {
    xa_put_row<float, C::DB>(reinterpret_cast<char*>(a.dq.part + (((size_t)split * a.BH + bh) * a.R + r) * D), dq, scale, lane);
  }
}

// dK, dV (owned keys, streamed packed query rows):  dv = p^T dout,  dk = scale dx^T q
template <typename T, int D, int NS, bool DROP, bool PRE>
__device__ __forceinline__ void xa_dkv(const XaArgs& a, int blk, XaLds<T, D, DROP>& sh) {
  typedef XaCfg<T, D> C;
  typedef XaMma<T, D> M;
  int bh, tile, split;
  if (!xa_block(a, a.dkv, blk, bh, tile, split)) return;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, b = bh / a.nkv, kvh = bh - b * a.nkv;
  const int key = (tile * NS + w) * 32 + (lane & 31);
  const int len = xa_len(a, b);
  const float bias = len > 0 ? xa_key_bias(a, xa_key_raw(a, b, key, len), key, len) : -INFINITY;
  const bool part = bias != -INFINITY, live = (tile * NS + w) * 32 < len;      // live: the wave has a key
  const int nt = tile * NS * 32 < len ? (a.R + C::TT - 1) / C::TT : 0;          // a tile behind the length: zeros
  const int per = (nt + a.dkv.splits - 1) / a.dkv.splits;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  const uint64_t seed = DROP ? a.seed_imm + (a.seed_ptr ? *a.seed_ptr : 0ull) : 0ull;
  const uint32_t hk = DROP ? attn_line_hash(seed, bh, key, UC2_ATTN_SALT_K) : 0u;

  typename M::Frag kf[C::KS], vf[C::KS];
  xa_own<T, D, false>(a, a.k, b, kvh, key, part, lane, kf);
  xa_own<T, D, false>(a, a.v, b, kvh, key, part, lane, vf);
  f32x16 dk[C::DB], dv[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) { dk[db][e] = 0.f; dv[db][e] = 0.f; }
  XaStage<T, D, NS * 64, true> st;
  st.init(a, a.q, a.dout, b, kvh, a.R, t);
  XaDelta<T, D, NS * 64> dl8;
  if (!PRE) dl8.init(a, bh, b, kvh, t);
  float lse = 0.f, delta = 0.f;
  auto fetch = [&](int tt) __attribute__((always_inline)) {
    st.load(a, a.q, a.dout, tt);
    if (!PRE) dl8.load(a, tt);
    const size_t at = (size_t)bh * a.R + min(tt * C::TT + (lane & (C::TT - 1)), a.R - 1);
    lse = a.lse[at];
    if (PRE) delta = a.delta[at];
  };
  auto put = [&](int tt, int buf) __attribute__((always_inline)) {
    st.store(sh.x[buf], sh.y[buf], (tt + 1) * C::TT > a.R, (1ull << min(63, a.R - tt * C::TT)) - 1);      // (fewer rows than a tile's 32 or 64)
    if (!PRE) dl8.store(a, st.y, sh.d[buf], tt);
    const int r = tt * C::TT + t;
    if (t < C::TT) {
      sh.s[buf][t] = r >= a.R || lse == -INFINITY ? -INFINITY : -lse;      // behind the last row, and rows without any key: p = 0
      if (PRE) sh.d[buf][t] = r < a.R ? -delta : 0.f;
      if (DROP && r < a.R) { int i, g; xa_split(a, r, i, g); sh.h[buf][t] = attn_line_hash(seed, b * a.nh + kvh * a.G + g, i, UC2_ATTN_SALT_Q); }
    }
  };
  if (t0 < t1) { fetch(t0); put(t0, 0); }
  xa_arrived(kf);
  xa_arrived(vf);
  __syncthreads();
  int buf = 0;
  for (int tt = t0; tt < t1; ++tt) {
    if (tt + 1 < t1) fetch(tt + 1);
#pragma unroll
    for (int n = 0; n < C::NB; ++n) {
      if (!live || tt * C::TT + n * 32 >= a.R) break;
      const f32x16 s = M::rows(sh.x[buf], n, kf, lane);
      // the rows' -log-sum-exp and -delta; without dropout dp's sums start at -delta (dropout scales dp first, and loads both late, for the registers)
      f32x4 lv[4], dl[4];
      f32x16 nd = xa_zero();
      auto line = [&](int k) __attribute__((always_inline)) {
        lv[k] = *reinterpret_cast<const f32x4*>(&sh.s[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
        dl[k] = *reinterpret_cast<const f32x4*>(&sh.d[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
      };
      if (!DROP) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          line(k);
#pragma unroll
          for (int e = 0; e < 4; ++e) nd[4 * k + e] = dl[k][e];
        }
      }
      const f32x16 dp = M::rows(sh.y[buf], n, vf, lane, nd);
      if (!DROP && a.kmask) {
#pragma unroll
        for (int k = 0; k < 4; ++k) lv[k] += f32x4{bias, bias, bias, bias};
      }
      float p[16], ds[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint4 hv = {0, 0, 0, 0};
        if (DROP) {
          line(k);
          if (a.kmask) lv[k] += f32x4{bias, bias, bias, bias};
          hv = *reinterpret_cast<const uint4*>(&sh.h[buf][n * 32 + 8 * k + 4 * (lane >> 5)]);
        }
        const uint32_t hh[4] = {hv.x, hv.y, hv.z, hv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[4 * k + e], a.scale2, lv[k][e]));
          float d = dp[4 * k + e], y = x;
          if (DROP) { const bool keep = attn_keep(hh[e], hk, a.thresh); d = (keep ? d * a.keep_scale : 0.f) + dl[k][e]; y = keep ? x * a.keep_scale : 0.f; }
          p[4 * k + e] = y;
          ds[4 * k + e] = x * d;
        }
      }
      M::cols(sh.y[buf], n, p, dv, lane);
      M::cols(sh.x[buf], n, ds, dk, lane);
    }
    if (tt + 1 < t1) put(tt + 1, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  const float scale = xa_alone(a, b, len, lane, __popcll(__ballot(part && lane < 32)), false) ? 0.f : a.scale;
  if (key >= a.Lk) return;
  if (!part) {                                                     // (without a mask its column was computed: on zero vectors, into this lane alone)
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) { dk[db][e] = 0.f; dv[db][e] = 0.f; }
  }
  if (a.dkv.splits == 1) {
    xa_put_row<T, C::DB>(a.gk.p + b * a.gk.sb + (long long)key * a.gk.sl + kvh * a.gk.sh, dk, scale, lane);
    xa_put_row<T, C::DB>(a.gv.p + b * a.gv.sb + (long long)key * a.gv.sl + kvh * a.gv.sh, dv, 1.0f, lane);
  } else {
    const size_t n = (size_t)a.BH * a.Lk, row = (size_t)bh * a.Lk + key;
    xa_put_row<float, C::DB>(reinterpret_cast<char*>(a.dkv.part + (split * 2 * n + row) * D), dk, scale, lane);
    xa_put_row<float, C::DB>(reinterpret_cast<char*>(a.dkv.part + ((split * 2 + 1) * n + row) * D), dv, 1.0f, lane);
  }
}

template <typename T, int D, int NS, bool DROP, bool PRE = false>
__global__ __launch_bounds__(NS * 64) void xattn_bwd_kernel(XaArgs a) {
  __shared__ XaLds<T, D, DROP> sh;
  if ((int)blockIdx.x < a.dkv.blocks) xa_dkv<T, D, NS, DROP, PRE>(a, blockIdx.x, sh);
  else xa_dq<T, D, NS, DROP, PRE>(a, blockIdx.x - a.dkv.blocks, sh);
}

// delta of every row, where many workgroups would form it again: CPR lanes per row
template <typename T, int D>
__global__ __launch_bounds__(256) void xattn_delta_kernel(XaArgs a) {
  typedef XaCfg<T, D> C;
  constexpr int E = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(E)));
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x, row = idx / C::CPR, rows = (long long)a.BH * a.R;
  const int c = (int)(idx % C::CPR);
  float s = 0.f;
  if (row < rows) {
    const int bh = (int)(row / a.R), r = (int)(row - (long long)bh * a.R), b = bh / a.nkv, kvh = bh - b * a.nkv;
    const char* p = sizeof(T) == 2 ? reinterpret_cast<const char*>(a.o32 + row * D) : xa_row<true>(a, a.o, b, kvh, r);
    const V g = *reinterpret_cast<const V*>(xa_row<true>(a, a.dout, b, kvh, r) + c * 16);
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      const f32x4 o = reinterpret_cast<const f32x4*>(p + c * E * 4)[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(o[e], (float)g[4 * j + e], s);
    }
  }
#pragma unroll
  for (int k = 1; k < C::CPR; k <<= 1) s += __shfl_xor(s, k);
  if (row < rows && c == 0) a.delta[row] = s;
}

// sums of the splits' gradients in split order: dK and dV, then dQ, where they were split
template <typename T, int D>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XaArgs a) {
  const long long rk = a.dkv.splits > 1 ? (long long)a.BH * a.Lk : 0, rq = a.dq.splits > 1 ? (long long)a.BH * a.R : 0;
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  long long row = idx / (D / 4);
  if (row >= 2 * rk + rq) return;
  const int c = (int)(idx - row * (D / 4)) * 4;
  const bool isq = row >= 2 * rk;
  if (isq) row -= 2 * rk;
  const XaSide& side = isq ? a.dq : a.dkv;
  const long long all = isq ? rq : 2 * rk;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < side.splits; ++k) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(side.part + ((size_t)k * all + row) * D + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  const int len = isq ? a.R : a.Lk;
  const long long lr = !isq && row >= rk ? row - rk : row;
  const int bh = (int)(lr / len), r = (int)(lr - (long long)bh * len), b = bh / a.nkv, kvh = bh - b * a.nkv;
  char* p;
  if (isq) {
    int i, g;
    xa_split(a, r, i, g);
    p = a.gq.p + b * a.gq.sb + (long long)i * a.gq.sl + (long long)(kvh * a.G + g) * a.gq.sh;
  } else {
    const XaOut& x = row >= rk ? a.gv : a.gk;
    p = x.p + b * x.sb + (long long)r * x.sl + kvh * x.sh;
  }
  xa_put4(reinterpret_cast<T*>(p) + c, s[0], s[1], s[2], s[3]);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------
static int xa_tt(int dtype, int D) { return D * (dtype ? 2 : 4) <= 128 ? 64 : 32; }
// waves of a workgroup: as many 32-column waves as there are columns, up to 4 (they share the streamed tile); two at least for fp32
// vectors of 128, whose staging by one wave alone spills
static int xa_ns(int dtype, int D, int cols) { return cols <= 32 && !(dtype == 0 && D == 128) ? 1 : cols <= 64 ? 2 : 4; }
// splits of the streamed axis, each two tiles at least: until the launch has 1024 waves, one per SIMD (4 x 512 x 512, 12 heads, forward and backward 40 us;
// up to 2048: 63 us, for the partials and their sum); workgroups of one wave, whose tiles wait for memory alone, to 2048 (16 x 1 x 16384: 32 us
// against 35)
static int xa_splits(const Uc2CrossAttn* p, int ns, int cols, int streamed) {
  const int tt = xa_tt(p->dtype, p->D);
  const long long bh = (long long)p->B * p->nkv;
  const long long waves = bh * ((cols + 32 * ns - 1) / (32 * ns)) * ns, nt = (streamed + tt - 1) / tt;
  long long s = waves > 0 ? (ns > 1 ? 1024 : 2048) / waves : 1;
  const long long most = p->dtype == 0 ? nt : nt / 2;             // (a tile of fp32 products is work enough: 8 x 77 x 211, 12 heads, 65 -> 59 us)
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
static size_t xa_up(size_t n) { return (n + 255) & ~(size_t)255; }
struct XaPlan { int ns_bwd, s_fwd, s_dq, s_dkv; bool pre; size_t fwd, delta, part_dkv, bwd; };
static XaPlan xa_plan(const Uc2CrossAttn* p) {
  XaPlan r{};
  const long long bh = (long long)p->B * p->nkv, R = (long long)p->Lq * (p->nh / p->nkv);
  r.s_fwd = xa_splits(p, xa_ns(p->dtype, p->D, (int)R), (int)R, p->Lk);
  if (r.s_fwd > 1) r.fwd = xa_up((size_t)r.s_fwd * bh * R * p->D * 4) + xa_up((size_t)r.s_fwd * bh * R * 8);
  const int nq = xa_ns(p->dtype, p->D, (int)R), nk = xa_ns(p->dtype, p->D, p->Lk);
  r.ns_bwd = nq > nk ? nq : nk;                                   // one launch: one size of workgroup
  if (p->dtype == 0 && p->D == 128) r.ns_bwd = 4;                 // (staging of three tensors by two waves spills)
  r.s_dq = xa_splits(p, r.ns_bwd, (int)R, p->Lk);
  r.s_dkv = xa_splits(p, r.ns_bwd, p->Lk, (int)R);
  r.part_dkv = r.s_dkv > 1 ? xa_up((size_t)r.s_dkv * 2 * bh * p->Lk * p->D * 4) : 0;
  // delta by a kernel of its own where five workgroups or more stream the same rows and there is work to hide a launch in: from 2^22 scores on.  Forward and
  // backward with it / without, us: 2^20 scores (128 x 2000, 4 heads) 24.7 / 23.2 for bf16 heads of 64, 41.0 / 39.5 for heads of 128, fp32 53.4 / 51.8; 2^22 (512 x 2048, 4
  // heads) 37.3 / 36.0, 59.6 / 61.8, 78.0 / 78.4; 2^24 (2 x 1024 x 1024, 8 heads) 56.2 / 55.5, 103.8 / 110.3, 210 / 215; 2^27 (2 x 2048 x 2048, 16 heads) 186 / 192, 446 / 503, 1370 / 1428
  r.pre = r.ns_bwd == 4 && p->Lk > 512 && bh * R * p->Lk >= (1 << 22);
  r.delta = r.pre ? xa_up((size_t)bh * R * 4) : 0;
  r.bwd = r.delta + r.part_dkv + (r.s_dq > 1 ? (size_t)r.s_dq * bh * R * p->D * 4 : 0);
  return r;
}
static bool xa_str_ok(long long sb, long long sl, long long sh, int el) {      // 16-byte rows
  return ((sb | sl | sh) & (16 / el - 1)) == 0 && sb >= 0 && sl >= 0 && sh >= 0 && sl < (1 << 22) && sh < (1 << 22);      // (64 rows within 2^31 bytes)
}
// a dimension of one element has no stride
static void xa_one(int n, long long& a, long long& b) { if (n <= 1) a = b = 0; }
static Uc2CrossAttn xa_norm(const Uc2CrossAttn* p) {
  Uc2CrossAttn d = *p;
  xa_one(d.B, d.q_sb, d.o_sb); xa_one(d.Lq, d.q_sl, d.o_sl); xa_one(d.nh, d.q_sh, d.o_sh);
  xa_one(d.B, d.k_sb, d.v_sb); xa_one(d.Lk, d.k_sl, d.v_sl); xa_one(d.nkv, d.k_sh, d.v_sh);
  if (d.B <= 1) d.key_mask_sb = 0;
  return d;
}
static int xa_check(const Uc2CrossAttn* p) {
  UC2_CHECK_ARG(p != nullptr);
  UC2_CHECK_ARG(p->dtype == 0 || p->dtype == 1);
  UC2_CHECK_ARG(p->D == 32 || p->D == 64 || p->D == 128);
  UC2_CHECK_ARG(p->B >= 0 && p->Lq >= 0 && p->Lk >= 0 && p->nkv >= 1 && p->nh >= 1 && p->nh % p->nkv == 0);
  UC2_CHECK_ARG((long long)p->Lq * (p->nh / p->nkv) < (1ll << 30) && p->Lk < (1 << 30));
  UC2_CHECK_ARG((long long)p->B * p->nkv < (1ll << 24));
  UC2_CHECK_ARG(p->drop_p >= 0.f && p->drop_p < 1.f);
  return 0;
}
static int xa_keys(const Uc2CrossAttn* p) {
  const int el = p->dtype ? 2 : 4;
  UC2_CHECK_ARG(p->Lk == 0 || (p->k && p->v));
  UC2_CHECK_ARG(xa_str_ok(p->k_sb, p->k_sl, p->k_sh, el) && xa_str_ok(p->v_sb, p->v_sl, p->v_sh, el));
  UC2_CHECK_ARG((((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0);
  return 0;
}
static int xa_ptrs(const Uc2CrossAttn* p, bool backward) {
  const int el = p->dtype ? 2 : 4;
  UC2_CHECK_ARG(p->q && (p->out || (backward && p->dtype == 1 && p->out_f32)));
  UC2_CHECK_ARG(!backward || p->dtype == 0 || p->out_f32);
  UC2_CHECK_ARG(xa_str_ok(p->q_sb, p->q_sl, p->q_sh, el) && xa_str_ok(p->o_sb, p->o_sl, p->o_sh, el));
  UC2_CHECK_ARG((((uintptr_t)p->q | (uintptr_t)p->out | (uintptr_t)p->out_f32) & 15) == 0);
  return xa_keys(p);
}
static XaArgs xa_args(const Uc2CrossAttn* p) {
  const int el = p->dtype ? 2 : 4;
  XaArgs a{};
  a.B = p->B; a.Lq = p->Lq; a.Lk = p->Lk; a.nkv = p->nkv; a.nh = p->nh; a.G = p->nh / p->nkv; a.R = p->Lq * a.G; a.BH = p->B * p->nkv;
  a.q = {(const char*)p->q, p->q_sb * el, p->q_sl * el, p->q_sh * el};
  a.k = {(const char*)p->k, p->k_sb * el, p->k_sl * el, p->k_sh * el};
  a.v = {(const char*)p->v, p->v_sb * el, p->v_sl * el, p->v_sh * el};
  a.out = {(char*)p->out, p->o_sb * el, p->o_sl * el, p->o_sh * el};
  a.o = {(const char*)p->out, p->o_sb * el, p->o_sl * el, p->o_sh * el};
  a.kmask = p->key_mask; a.kmask_sb = p->key_mask_sb; a.klens = p->k_lens;
  a.scale = p->scale; a.scale2 = p->scale * XA_LOG2E;
  a.lse = p->lse; a.o32 = p->out_f32;
  a.thresh = drop_thresh(p->drop_p); a.keep_scale = 1.0f / (1.0f - p->drop_p); a.seed_ptr = p->seed; a.seed_imm = p->site;
  return a;
}
static bool xa_side(const XaArgs& a, XaSide& side, int cols, int ns, int splits) {      // false: more blocks than a launch takes
  side.tiles = (cols + 32 * ns - 1) / (32 * ns);
  side.splits = splits;
  const long long n = (long long)(a.BH >= 8 ? (a.BH + 7) / 8 * 8 : a.BH) * side.tiles * splits;
  side.blocks = (int)n;
  return n <= UC2_MOST_BLOCKS(64 * ns);
}
#define XA_LAUNCH(KERN, TT_, DD_, NN_, grid)                                                                                        \
  do {                                                                                                                              \
    if (a.thresh) hipLaunchKernelGGL((KERN<TT_, DD_, NN_, true>), dim3(grid), dim3(NN_ * 64), 0, st, a);                             \
    else hipLaunchKernelGGL((KERN<TT_, DD_, NN_, false>), dim3(grid), dim3(NN_ * 64), 0, st, a);                                     \
  } while (0)
#define XA_NS(KERN, TT_, DD_, MOST)      /* MOST: bytes of the rows that two waves may stage */                                       \
  do {                                                                                                                              \
    if constexpr (DD_ * sizeof(TT_) <= 256) { if (ns == 1) { XA_LAUNCH(KERN, TT_, DD_, 1, grid); break; } }                          \
    if constexpr (DD_ * sizeof(TT_) <= MOST) { if (ns == 2) { XA_LAUNCH(KERN, TT_, DD_, 2, grid); break; } }                         \
    XA_LAUNCH(KERN, TT_, DD_, 4, grid);                                                                                             \
  } while (0)
#define XA_TD(WHAT)                                                                                                                 \
  do {                                                                                                                              \
    if (p->dtype == 1) { if (p->D == 32) { WHAT(bf16, 32); } else if (p->D == 64) { WHAT(bf16, 64); } else { WHAT(bf16, 128); } }     \
    else { if (p->D == 32) { WHAT(float, 32); } else if (p->D == 64) { WHAT(float, 64); } else { WHAT(float, 128); } }                \
  } while (0)

extern "C" size_t uc2_xattn_workspace(const Uc2CrossAttn* p, int backward) {
  if (xa_check(p) != 0) return 0;
  const XaPlan pl = xa_plan(p);
  return backward ? pl.bwd : pl.fwd;
}

extern "C" int uc2_xattn_fwd(const Uc2CrossAttn* attn, void* ws, size_t ws_bytes, void* stream) {
  if (int e = xa_check(attn)) return e;
  const Uc2CrossAttn norm = xa_norm(attn), *p = &norm;
  if (p->B == 0 || p->Lq == 0) return 0;
  if (int e = xa_ptrs(p, false)) return e;
  const XaPlan pl = xa_plan(p);
  UC2_CHECK_ARG(pl.fwd == 0 || (ws && ws_bytes >= pl.fwd && ((uintptr_t)ws & 15) == 0));
  hipStream_t st = (hipStream_t)stream;
  XaArgs a = xa_args(p);
  const int ns = xa_ns(p->dtype, p->D, a.R);
  UC2_CHECK_ARG(xa_side(a, a.fwd, a.R, ns, pl.s_fwd));
  if (pl.s_fwd > 1) {
    a.fwd.part = (float*)ws;
    a.pml = (float*)((char*)ws + xa_up((size_t)pl.s_fwd * a.BH * a.R * p->D * 4));
  }
  const int grid = a.fwd.blocks;
#define XA_GO(T_, D_) XA_NS(xattn_fwd_kernel, T_, D_, 512)
  XA_TD(XA_GO);
#undef XA_GO
  UC2_LAUNCH_CHECK();
  if (pl.s_fwd > 1) {
    // four waves per row from 8 splits on
    const bool wide = pl.s_fwd >= 8;
    const long long rows = (long long)a.BH * a.R, blocks = wide ? rows : (rows + 3) / 4;
    UC2_CHECK_ARG(blocks <= UC2_MOST_BLOCKS(256));
#define XA_GO(T_, D_)                                                                                                               \
  if (wide) hipLaunchKernelGGL((xattn_join_kernel<T_, D_, 4>), dim3((unsigned)blocks), dim3(256), 0, st, a);                         \
  else hipLaunchKernelGGL((xattn_join_kernel<T_, D_, 1>), dim3((unsigned)blocks), dim3(256), 0, st, a)
    XA_TD(XA_GO);
#undef XA_GO
    UC2_LAUNCH_CHECK();
  }
  return 0;
}

extern "C" int uc2_xattn_bwd(const Uc2CrossAttn* attn, const Uc2CrossAttnGrad* grad, void* ws, size_t ws_bytes, void* stream) {
  if (int e = xa_check(attn)) return e;
  UC2_CHECK_ARG(grad != nullptr);
  const Uc2CrossAttn norm = xa_norm(attn), *p = &norm;
  Uc2CrossAttnGrad gnorm = *grad, *g = &gnorm;
  xa_one(p->B, g->dout_sb, g->dq_sb); xa_one(p->Lq, g->dout_sl, g->dq_sl); xa_one(p->nh, g->dout_sh, g->dq_sh);
  xa_one(p->B, g->dk_sb, g->dv_sb); xa_one(p->Lk, g->dk_sl, g->dv_sl); xa_one(p->nkv, g->dk_sh, g->dv_sh);
  if (p->B == 0) return 0;
  const int el = p->dtype ? 2 : 4;
  UC2_CHECK_ARG(p->Lq == 0 || (g->dout && g->dq && p->lse));
  UC2_CHECK_ARG(p->Lk == 0 || (g->dk && g->dv));
  UC2_CHECK_ARG(xa_str_ok(g->dout_sb, g->dout_sl, g->dout_sh, el) && xa_str_ok(g->dq_sb, g->dq_sl, g->dq_sh, el));
  UC2_CHECK_ARG(xa_str_ok(g->dk_sb, g->dk_sl, g->dk_sh, el) && xa_str_ok(g->dv_sb, g->dv_sl, g->dv_sh, el));
  UC2_CHECK_ARG((((uintptr_t)g->dout | (uintptr_t)g->dq | (uintptr_t)g->dk | (uintptr_t)g->dv) & 15) == 0);
  if (int e = p->Lq > 0 ? xa_ptrs(p, true) : xa_keys(p)) return e;      // (without queries the keys are read all the same)
  const XaPlan pl = xa_plan(p);
  UC2_CHECK_ARG(pl.bwd == 0 || (ws && ws_bytes >= pl.bwd && ((uintptr_t)ws & 15) == 0));
  hipStream_t st = (hipStream_t)stream;
  XaArgs a = xa_args(p);
  a.dout = {(const char*)g->dout, g->dout_sb * el, g->dout_sl * el, g->dout_sh * el};
  a.gq = {(char*)g->dq, g->dq_sb * el, g->dq_sl * el, g->dq_sh * el};
  a.gk = {(char*)g->dk, g->dk_sb * el, g->dk_sl * el, g->dk_sh * el};
  a.gv = {(char*)g->dv, g->dv_sb * el, g->dv_sl * el, g->dv_sh * el};
  const int ns = pl.ns_bwd;
  UC2_CHECK_ARG(xa_side(a, a.dkv, a.Lk, ns, pl.s_dkv) && xa_side(a, a.dq, a.R, ns, pl.s_dq));
  a.delta = (float*)ws;
  a.dkv.part = (float*)((char*)ws + pl.delta);
  a.dq.part = (float*)((char*)ws + pl.delta + pl.part_dkv);
  UC2_CHECK_ARG((long long)a.dkv.blocks + a.dq.blocks <= UC2_MOST_BLOCKS(64 * ns));
  const int grid = a.dkv.blocks + a.dq.blocks;
  if (grid == 0) return 0;                                        // (neither queries nor keys)
  if (pl.pre && a.R > 0) {
    const long long lanes = (long long)a.BH * a.R * (p->D * el / 16), n = (lanes + 255) / 256;
    UC2_CHECK_ARG(n <= UC2_MOST_BLOCKS(256));
#define XA_GO(T_, D_) hipLaunchKernelGGL((xattn_delta_kernel<T_, D_>), dim3((unsigned)n), dim3(256), 0, st, a);                    \
    if (a.thresh) hipLaunchKernelGGL((xattn_bwd_kernel<T_, D_, 4, true, true>), dim3(grid), dim3(256), 0, st, a);                   \
    else hipLaunchKernelGGL((xattn_bwd_kernel<T_, D_, 4, false, true>), dim3(grid), dim3(256), 0, st, a)
    XA_TD(XA_GO);
#undef XA_GO
  } else {
#define XA_GO(T_, D_) XA_NS(xattn_bwd_kernel, T_, D_, 256)
    XA_TD(XA_GO);
#undef XA_GO
  }
  UC2_LAUNCH_CHECK();
  const long long rows = (pl.s_dkv > 1 ? 2ll * a.BH * a.Lk : 0) + (pl.s_dq > 1 ? (long long)a.BH * a.R : 0), blocks = (rows * (p->D / 4) + 255) / 256;
  UC2_CHECK_ARG(blocks <= UC2_MOST_BLOCKS(256));
  if (blocks > 0) {
#define XA_GO(T_, D_) hipLaunchKernelGGL((xattn_sum_kernel<T_, D_>), dim3((unsigned)blocks), dim3(256), 0, st, a)
    XA_TD(XA_GO);
#undef XA_GO
    UC2_LAUNCH_CHECK();
  }
  return 0;
}

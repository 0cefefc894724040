// e4m3 values under one power of two for each block of 128: the format of the block-scaled products (gemm_fp8_block.hip), written by
// fp8_block.hip and rmsnorm.hip.
//   block value = e4m3(x 2^-e) 2^e,  e the smallest integer with max |x| <= 448 2^e, kept as the byte e + 127 (E8M0, what the scaled
//   matrix instruction reads); 1 at least, an all-zero block included.  An infinity or NaN becomes the e4m3 NaN.
//   activations [M, K]: bytes [M, Kp], Kp = K rounded up to 128, zeros behind K; scales of 1 x 128 blocks as 32-bit words [ceil(Kp / 512)][M]: the
//   bytes of four neighbouring blocks of a row, the rows of one word adjacent (a product's lanes read 16 rows as one 64-byte segment)
//   weights [N, K]: bytes [N, Kp], scales of 128 x 128 blocks as bytes [ceil(N / 128)][Kp / 128]
#pragma once
#include "common.h"

typedef bf16 blk_bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef float blk_f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

// elements c .. c + 7 (c < n) of a row of n that ends inside them, zeros behind its end: the row's last eight, shifted down (eight guarded loads
// in their place made the workgroups of a matrix's last columns several times slower than the others)
__device__ __forceinline__ bf16x8 blk_tail8(const bf16* row, int c, int n) {
  if (n < 8) {
    bf16x8 v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) if (c + e < n) v[e] = row[c + e];
    return v;
  }
  typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
  u64x2 u = __builtin_bit_cast(u64x2, (bf16x8)*reinterpret_cast<const blk_bf16x8_u*>(row + n - 8));
  const int sh = (c + 8 - n) * 16;                     // 16 .. 112 bits
  const unsigned long long lo = sh < 64 ? (u[0] >> sh) | (u[1] << (64 - sh)) : u[1] >> (sh - 64), hi = sh < 64 ? u[1] >> sh : 0ull;
  return __builtin_bit_cast(bf16x8, u64x2{lo, hi});
}
// Eight neighbouring elements of a row, loaded (no alignment needed) and converted in two steps: every load of a row is issued before the first is used.
// WHOLE (rows of a multiple of 8): no branch -- hipcc waits for a load at the end of the branch that uses it, and a chunk behind the row's end loads
// the row's last one and counts as zeros.  Otherwise the last chunk goes element by element.
template <typename T> struct Blk8;
template <> struct Blk8<bf16> {
  bf16x8 v;
  template <bool WHOLE> __device__ __forceinline__ void load(const bf16* row, int c, int n) {
    if (WHOLE) v = *reinterpret_cast<const blk_bf16x8_u*>(row + min(c, n - 8));
    else if (c + 8 <= n) v = *reinterpret_cast<const blk_bf16x8_u*>(row + c);
    else if (c < n) v = blk_tail8(row, c, n);
    else v = bf16x8{};
  }
  template <bool WHOLE> __device__ __forceinline__ void get(float (&o)[8], int c, int n) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (WHOLE && c >= n) ? 0.f : (float)v[e];
  }
};
template <> struct Blk8<float> {
  f32x4 v[2];
  template <bool WHOLE> __device__ __forceinline__ void load(const float* row, int c, int n) {
    if (WHOLE) {
      const float* p = row + min(c, n - 8);
      v[0] = *reinterpret_cast<const blk_f32x4_u*>(p); v[1] = *reinterpret_cast<const blk_f32x4_u*>(p + 4);
    } else if (c + 8 <= n) {
      v[0] = *reinterpret_cast<const blk_f32x4_u*>(row + c); v[1] = *reinterpret_cast<const blk_f32x4_u*>(row + c + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e >> 2][e & 3] = c + e < n ? row[c + e] : 0.f;
    }
  }
  template <bool WHOLE> __device__ __forceinline__ void get(float (&o)[8], int c, int n) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (WHOLE && c >= n) ? 0.f : v[e >> 2][e & 3];
  }
};
template <bool WHOLE, typename T> __device__ __forceinline__ void blk_load8(const T* row, int c, int n, float (&v)[8]) {
  Blk8<T> r;
  r.template load<WHOLE>(row, c, n);
  r.template get<WHOLE>(v, c, n);
}
__device__ __forceinline__ void blk_store8(bf16* row, int c, int n, const float (&v)[8]) {
  if (c + 8 <= n) {
    blk_bf16x8_u x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (bf16)v[e];
    *reinterpret_cast<blk_bf16x8_u*>(row + c) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) if (c + e < n) row[c + e] = (bf16)v[e];
  }
}
__device__ __forceinline__ void blk_store8(float* row, int c, int n, const float (&v)[8]) {
  if (c + 8 <= n) {
    *reinterpret_cast<blk_f32x4_u*>(row + c) = blk_f32x4_u{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<blk_f32x4_u*>(row + c + 4) = blk_f32x4_u{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) if (c + e < n) row[c + e] = v[e];
  }
}

// biased exponent of a block with maximum `amax`: 448 = 1.75 * 2^8, so e = exponent(amax) - 8, one more where its significand is over 1.75
__device__ __forceinline__ unsigned blk_exponent(float amax) {
  const int b = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8;
  return (unsigned)(b < 1 ? 1 : b);                   // (at most 248: an infinity's)
}
__device__ __forceinline__ float blk_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }      // 2^-e: 6 .. 253, a normal number
// no clamp: |x 2^-e| <= 448 by the choice of e, and the conversion turns infinities and NaN into the e4m3 NaN
__device__ __forceinline__ unsigned blk_pack4(float a, float b, float c, float d) {
  unsigned r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ float blk_amax8(const float (&v)[8]) {
  return fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), fmaxf(fmaxf(fabsf(v[4]), fabsf(v[5])), fmaxf(fabsf(v[6]), fabsf(v[7]))));
}
// a wave's 512 consecutive elements of a row (lane: c .. c + 7): bytes, and the word of its four blocks' scales
__device__ __forceinline__ void blk_quant_row(const float (&v)[8], int c, int Kp, unsigned char* q, unsigned* word, int lane) {
  float m = blk_amax8(v);
  m = fmaxf(m, __shfl_xor(m, 1)); m = fmaxf(m, __shfl_xor(m, 2)); m = fmaxf(m, __shfl_xor(m, 4)); m = fmaxf(m, __shfl_xor(m, 8));
  const unsigned e = blk_exponent(m);
  const float s = blk_inverse(e);
  if (c < Kp)
    *reinterpret_cast<uint2*>(q + c) = uint2{blk_pack4(v[0] * s, v[1] * s, v[2] * s, v[3] * s), blk_pack4(v[4] * s, v[5] * s, v[6] * s, v[7] * s)};
  const unsigned p = e << ((lane >> 4) * 8);
  unsigned pk = p | __shfl_xor(p, 16);
  pk |= __shfl_xor(pk, 32);
  if (lane == 0 && (c & ~511) < Kp) *word = pk;
}

#include "gemm_tile.h"

// ------------------------------------------------------------------------------------------------------
// The ping-pong kernel of gemm_pp16.hip on OCP fp8 (e4m3) operands: v_mfma_scale_f32_16x16x128_f8f6f4 with unit block scales
// ("fp8 MFMA GEMMs").  Both operands k-contiguous e4m3 bytes, handed over as "bf16" matrices of half the
// width (same bytes: a k-tile of 64 "bf16" = 128 e4m3 values = the same 128-byte LDS rows, units, swizzles, LDS-DMA pieces and
// counted vmcnt as the bf16 kernel).  A phase is 8 MFMAs of 32 cycles on the same 64 x 32 quadrant where the bf16 kernel runs 16 of
// 16: the same phase time for twice the contraction depth, i.e. half the main loop per flop; the epilogue is the bf16 kernel's plus
// the de-scaling multiply (alpha = 1 / (scale_a scale_b), a power of two: the accumulators start at bias / alpha, exactly).
// bf16 output, whole 256 x 256 tiles, an even number of k-tiles; epilogues none / GELU + gelu' / x gelu' (+ column sums) / + residual.
// ------------------------------------------------------------------------------------------------------
#include "gemm_pp8_kernel.h"

// p is the "bf16 view" of the e4m3 problem (K, lda, ldb halved; gemm_fast.hip uc2_gemm_fp8_launch): whole 256 x 256 tiles, an even
// number (>= 2) of 128-byte k-tiles, 32-bit staging offsets, 16-byte aligned bf16 output / aux tensors
bool uc2_gemm_pp8_supported(const GemmArgs& p) {
  const int ktiles = p.K / 64;
  if ((p.M % 256) || (p.N & 255) || (p.K % 64) || (ktiles & 1) || ktiles < 2) return false;
  if (2ull * p.M * p.lda >= (1ull << 32) || 2ull * p.N * p.ldb >= (1ull << 32)) return false;
  if (p.c_f32 || p.accumulate || (p.ldc & 7) || (p.ldaux & 7) || ((uintptr_t)p.C & 15) || ((uintptr_t)p.aux_in & 15) ||
      ((uintptr_t)p.aux_out & 15) || ((uintptr_t)p.bias & 15)) return false;
  if (p.epi == EPI_GELU) return p.aux_deriv && p.aux_out != nullptr;
  if (p.epi == EPI_DGELU) return p.aux_deriv != 0;
  return p.epi == EPI_NONE || p.epi == EPI_ADD || p.epi == EPI_DROPADD;
}

void uc2_gemm_pp8_launch(const GemmArgs& p0, hipStream_t st) {
  GemmArgs p = p0;
  p.split_k = 1; p.partial = nullptr; p.queue = nullptr; p.skew = 0;
  p.col_group = pp8_col_group(p.N);
  if (p.q_out) {                                       // (uc2_gemm_fp8_q has checked: GELU + gelu' or x gelu' kinds only)
    if (p.epi == EPI_GELU) pp8_launch0<EPI_GELU_D, true>(p, st);
    else pp8_launch0<EPI_MUL, true>(p, st);
    return;
  }
  if (p.epi == EPI_GELU) pp8_launch0<EPI_GELU_D>(p, st);
  else if (p.epi == EPI_DGELU) pp8_launch0<EPI_MUL>(p, st);
  else if (p.epi == EPI_ADD) pp8_launch0<EPI_ADD>(p, st);
  else if (p.epi == EPI_DROPADD) pp8_launch0<EPI_DROPADD>(p, st);
  else pp8_launch0<EPI_NONE>(p, st);
}

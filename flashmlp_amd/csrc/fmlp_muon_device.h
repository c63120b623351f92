// Device-side parts of the orthogonalised updates that more than one translation unit uses.
#pragma once
#include "fmlp_muon.h"
#include "fmlp_vec.h"

namespace fmlp {

// hi and lo fp16 terms of 8 values times s (a power of two: a s is exact)
__device__ __forceinline__ void split8(const float* f, float s, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    hi[j] = pack2<false>(f[2 * j] * s, f[2 * j + 1] * s);
    lo[j] = pack2<false>(__builtin_fmaf(f[2 * j], s, -lo_f32<false>(hi[j])), __builtin_fmaf(f[2 * j + 1], s, -hi_f32<false>(hi[j])));
  }
}

// Where P, and what leads to it, has the 8 values of row r, inner indices 16 k + 4 g + {0..3, 8..11} (unit g of 16, in
// the order that the matrix instruction's results have rows in): a wave's operand of 32 rows is one run of 1 KB.
template <int NP>
__device__ __forceinline__ size_t muon_chunk(int r, int k, int g) {
  return ((size_t)(r >> 5) * (NP / 16) + k) * 512 + g * 256 + (r & 31) * 8;
}

__device__ __forceinline__ MuonInfo info_of(float trace, const MuonSteps& s, float p_scale, float* inv) {
  const float norm = __builtin_sqrtf(trace);
  *inv = s.normalise ? 1.f / (norm + s.eps) : 1.f;
  // |u| <= norm: as fp16 up to 2^14. (Sums of squares below fp32 leave a norm of 0 and values below 2^-74.)
  int e = 0;
  (void)frexpf(fmaxf(norm, 0x1p-74f), &e);
  const float us = ldexpf(1.f, min(max(14 - e, -100), 100));
  return MuonInfo{us, *inv / us / p_scale};
}

}  // namespace fmlp

// Runs of elements of any io type as floats, 16 bytes at a time, from and to addresses aligned to the elements only.
#pragma once
#include "fmlp_device.h"
#include "fmlp_launch.h"

namespace fmlp {

template <int IO>
constexpr int kPiece = IO == IO_F32 ? 4 : 8;  // elements of 16 bytes

template <int IO>
__device__ __forceinline__ float elem_f32(const void* base, long long i) {
  if constexpr (IO == IO_F32) return ((const float*)base)[i];
  else return to_f32<IO == IO_BF16>(((const u16*)base)[i]);
}

// 16 bytes at element i as bits; elements n .. of them are zeros and not read
template <int IO>
__device__ __forceinline__ u32x4 load_piece(const void* base, long long i, int n) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (IO == IO_F32) {
    const unsigned* p = (const unsigned*)base + i;
    if (n >= 4) __builtin_memcpy(&v, p, 16);
    else
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < n) v[j] = p[j];
  } else {
    const u16* p = (const u16*)base + i;
    if (n >= 8) __builtin_memcpy(&v, p, 16);
    else
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < n) v[j >> 1] |= (unsigned)p[j] << (16 * (j & 1));
  }
  return v;
}
template <int IO>
__device__ __forceinline__ void store_piece(void* base, long long i, int n, const u32x4& v) {
  if constexpr (IO == IO_F32) {
    unsigned* p = (unsigned*)base + i;
    if (n >= 4) __builtin_memcpy(p, &v, 16);
    else
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < n) p[j] = v[j];
  } else {
    u16* p = (u16*)base + i;
    if (n >= 8) __builtin_memcpy(p, &v, 16);
    else
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < n) p[j] = (u16)(v[j >> 1] >> (16 * (j & 1)));
  }
}
template <int IO>
__device__ __forceinline__ void unpack_piece(const u32x4& v, float (&f)[kPiece<IO>]) {
  if constexpr (IO == IO_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = lo_f32<IO == IO_BF16>(v[j]);
      f[2 * j + 1] = hi_f32<IO == IO_BF16>(v[j]);
    }
  }
}
template <int IO>
__device__ __forceinline__ u32x4 pack_piece(const float (&f)[kPiece<IO>]) {
  if constexpr (IO == IO_F32) {
    return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
  } else {
    constexpr bool BF = IO == IO_BF16;
    return u32x4{pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7])};
  }
}

}  // namespace fmlp

// Helpers of the gated MLP's calls on gfx950: its projections' rows padded to whole 16-byte vectors, and the sum over
// heads of fp32 outputs. Both move a few MB beside the products' work; their launches are most of their time.
#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

// One 16-byte piece of a padded row a thread: H=16 D=64 E=683 both matrices 4.9 us, one launch each 9.6.
template <typename T>
__global__ void __launch_bounds__(256) pad_pair_kernel(const T* __restrict__ wg, const T* __restrict__ wu,
                                                       T* __restrict__ dst, long long pieces, int E, int ppr) {
  constexpr int N = 16 / sizeof(T);
  const long long p = (long long)blockIdx.x * 256 + threadIdx.x;
  if (p >= 2 * pieces) return;
  const bool second = p >= pieces;
  const long long i = second ? p - pieces : p, row = i / ppr;
  const int c = (int)(i - row * ppr) * N;
  const T* s = (second ? wu : wg) + row * E + c;
  T v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = c + j < E ? s[j] : (T)0;
  u32x4 w;
  __builtin_memcpy(&w, v, 16);
  *(u32x4*)(dst + p * N) = w;
}

// dst[i] = scale * sum over the heads of src[head][i], in head order, four values a thread.
template <int IO>
__global__ void __launch_bounds__(256) head_sum_kernel(const float* __restrict__ src, void* __restrict__ dst, long long n,
                                                       int H, float scale) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 v = *(const float4*)(src + i);
  int h = 1;
  for (; h + 4 <= H; h += 4) {
    float4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = *(const float4*)(src + (size_t)(h + k) * n + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v.x += u[k].x;
      v.y += u[k].y;
      v.z += u[k].z;
      v.w += u[k].w;
    }
  }
  for (; h < H; ++h) {
    const float4 u = *(const float4*)(src + (size_t)h * n + i);
    v.x += u.x;
    v.y += u.y;
    v.z += u.z;
    v.w += u.w;
  }
  v = float4{v.x * scale, v.y * scale, v.z * scale, v.w * scale};
  if constexpr (IO == IO_F32) *(float4*)((float*)dst + i) = v;
  else *(u32x2*)((u16*)dst + i) = u32x2{pack2<IO == IO_BF16>(v.x, v.y), pack2<IO == IO_BF16>(v.z, v.w)};
}

}  // namespace

hipError_t launch_head_sum(const float* src, void* dst, int64_t n, int64_t H, float scale, int io, hipStream_t st) {
  const long long blocks = (n / 4 + 255) / 256;
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 g((unsigned)blocks), b(256);
  if (io == IO_F32) hipLaunchKernelGGL(head_sum_kernel<IO_F32>, g, b, 0, st, src, dst, (long long)n, (int)H, scale);
  else if (io == IO_BF16) hipLaunchKernelGGL(head_sum_kernel<IO_BF16>, g, b, 0, st, src, dst, (long long)n, (int)H, scale);
  else hipLaunchKernelGGL(head_sum_kernel<IO_F16>, g, b, 0, st, src, dst, (long long)n, (int)H, scale);
  return hipGetLastError();
}

hipError_t launch_gated_pad(const void* wg, const void* wu, void* dst, int64_t rows, int64_t E, int64_t ldw, int es,
                            hipStream_t st) {
  const int ppr = (int)(ldw * es / 16);
  const long long pieces = rows * ppr, blocks = (2 * pieces + 255) / 256;
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (es == 4)
    hipLaunchKernelGGL(pad_pair_kernel<unsigned>, dim3((unsigned)blocks), dim3(256), 0, st, (const unsigned*)wg,
                       (const unsigned*)wu, (unsigned*)dst, pieces, (int)E, ppr);
  else
    hipLaunchKernelGGL(pad_pair_kernel<u16>, dim3((unsigned)blocks), dim3(256), 0, st, (const u16*)wg, (const u16*)wu,
                       (u16*)dst, pieces, (int)E, ppr);
  return hipGetLastError();
}

}  // namespace fmlp

// Global norm of many gradients and their clipping on gfx950.
//
//   norm = sqrt(sum over all elements of all tensors of g^2)
//   out  = g min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM bytes: every gradient is read once for the norm and once, with its result written, for the
// scaling. The tensors are cut into chunks of equal size, a workgroup each, whatever their number and sizes; a
// launch takes as many tensors as its arguments hold (kMaxTensors). Squares are summed in 64 bits: bf16
// and fp32 gradients reach 1e38, whose squares 32 bits do not hold, and the 64-bit additions hide
// behind the loads (32-bit squares measured the same). 302 M bf16 gradients into fp32: norm 114 us (5.3 TB/s), scaling
// 355 (1.8 GB, 5.1 TB/s); non-temporal stores 490, the second pass in reverse order no gain. Partial sums go through the
// workspace and are added in a fixed order. The coefficient is an fp32 number unless the norm is beyond fp32.
#include <algorithm>
#include <cfloat>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

// Elements of a workgroup of the scaling: 302 M bf16 gradients into fp32 in 390 us with 64 K, 361 with 16 K, 354 with 8 K.
constexpr long long kScaleChunk = 8192;
constexpr int kMaxTensors = 112;  // per launch: the table below stays within 4 KB of kernel arguments

struct ClipTable {
  const void* grad[kMaxTensors];
  void* out[kMaxTensors];
  unsigned long long numel[kMaxTensors];
  unsigned first[kMaxTensors];  // the tensor's first workgroup
  unsigned char io[kMaxTensors], out_io[kMaxTensors];
  int n;
};
static_assert(sizeof(ClipTable) <= 3840, "kernel arguments");

// tensor of workgroup b: the last one whose first workgroup is at most b (empty tensors own none)
__device__ __forceinline__ int tensor_of(const ClipTable& t, unsigned b) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// 8 elements at p, which is aligned to its elements only
template <int IO>
__device__ __forceinline__ void load8f(const void* base, long long i, float (&f)[8]) {
  if constexpr (IO == IO_F32) {
    __builtin_memcpy(f, (const float*)base + i, 32);
  } else {
    u32x4 v;
    __builtin_memcpy(&v, (const u16*)base + i, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = lo_f32<IO == IO_BF16>(v[j]);
      f[2 * j + 1] = hi_f32<IO == IO_BF16>(v[j]);
    }
  }
}
template <int IO>
__device__ __forceinline__ float load1f(const void* base, long long i) {
  if constexpr (IO == IO_F32) return ((const float*)base)[i];
  else return to_f32<IO == IO_BF16>(((const u16*)base)[i]);
}
template <int IO>
__device__ __forceinline__ void store8f(void* base, long long i, const float (&f)[8]) {
  if constexpr (IO == IO_F32) {
    __builtin_memcpy((float*)base + i, f, 32);
  } else {
    constexpr bool BF = IO == IO_BF16;
    const u32x4 v = {pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7])};
    __builtin_memcpy((u16*)base + i, &v, 16);
  }
}
template <int IO>
__device__ __forceinline__ void store1f(void* base, long long i, float v) {
  if constexpr (IO == IO_F32) ((float*)base)[i] = v;
  else ((u16*)base)[i] = from_f32<IO == IO_BF16>(v);
}

template <int IO>
__device__ __forceinline__ double chunk_sum(const void* g, long long i0, long long i1) {
  double s[4] = {0, 0, 0, 0};
  long long i = i0 + threadIdx.x * 8;
  for (; i + 3 * 2048 + 8 <= i1; i += 4 * 2048) {
    float f[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) load8f<IO>(g, i + u * 2048, f[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[u] = __builtin_fma((double)f[u][j], (double)f[u][j], s[u]);
  }
  for (; i < i1; i += 2048)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < i1) {
        const double v = load1f<IO>(g, i + j);
        s[j & 3] = __builtin_fma(v, v, s[j & 3]);
      }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__global__ void __launch_bounds__(256) norm_kernel(ClipTable t, long long chunk, double* part) {
  __shared__ double w[4];
  const int k = tensor_of(t, blockIdx.x);
  const long long i0 = (long long)(blockIdx.x - t.first[k]) * chunk;
  const long long i1 = min((long long)t.numel[k], i0 + chunk);
  double s;
  if (t.io[k] == IO_F32) s = chunk_sum<IO_F32>(t.grad[k], i0, i1);
  else if (t.io[k] == IO_BF16) s = chunk_sum<IO_BF16>(t.grad[k], i0, i1);
  else s = chunk_sum<IO_F16>(t.grad[k], i0, i1);
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}

// The norm, and the coefficient torch's clipping uses (a NaN norm stays one: min would drop it): an fp32 number, but
// where a finite norm is beyond fp32, which is then kept in 64 bits.
__global__ void __launch_bounds__(1024) norm_finish_kernel(const double* part, long long n, float max_norm, float* norm,
                                                           double* coef) {
  __shared__ double w[16];
  double s = 0;
  for (long long i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double v = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += w[i];
  v = __builtin_sqrt(v);
  const float r = (float)v;
  *norm = r;
  if (coef) {
    const bool beyond = r > FLT_MAX && v <= DBL_MAX;
    const double c = beyond ? (double)max_norm / v : (double)(max_norm / (r + 1e-6f));
    *coef = c > 1. ? 1. : c;
  }
}

template <int IO, int OIO>
__device__ __forceinline__ void chunk_scale(const void* g, void* out, long long i0, long long i1, float c) {
  long long i = i0 + threadIdx.x * 8;
  for (; i + 3 * 2048 + 8 <= i1; i += 4 * 2048) {
    float f[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) load8f<IO>(g, i + u * 2048, f[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[u][j] *= c;
      store8f<OIO>(out, i + u * 2048, f[u]);
    }
  }
  for (; i < i1; i += 2048)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < i1) store1f<OIO>(out, i + j, load1f<IO>(g, i + j) * c);
}

// The same with a coefficient of 64 bits, for norms beyond fp32: rare, so element by element.
__device__ __forceinline__ void chunk_scale64(int io, int out_io, const void* g, void* out, long long i0, long long i1, double c) {
  for (long long i = i0 + threadIdx.x; i < i1; i += 256) {
    const float f = io == IO_F32 ? load1f<IO_F32>(g, i) : io == IO_BF16 ? load1f<IO_BF16>(g, i) : load1f<IO_F16>(g, i);
    const float v = (float)((double)f * c);
    if (out_io == IO_F32) store1f<IO_F32>(out, i, v);
    else if (out_io == IO_BF16) store1f<IO_BF16>(out, i, v);
    else store1f<IO_F16>(out, i, v);
  }
}

template <int IO>
__device__ __forceinline__ void chunk_scale_to(int out_io, const void* g, void* out, long long i0, long long i1, float c) {
  if (out_io == IO_F32) chunk_scale<IO, IO_F32>(g, out, i0, i1, c);
  else if (out_io == IO_BF16) chunk_scale<IO, IO_BF16>(g, out, i0, i1, c);
  else chunk_scale<IO, IO_F16>(g, out, i0, i1, c);
}

__global__ void __launch_bounds__(256) scale_kernel(ClipTable t, long long chunk, const double* coef) {
  const double c64 = *coef;
  const float c = (float)c64;
  const int k = tensor_of(t, blockIdx.x);
  if (c == 1.f && t.grad[k] == t.out[k]) return;  // in place and within the limit: the values stay
  const long long i0 = (long long)(blockIdx.x - t.first[k]) * chunk;
  const long long i1 = min((long long)t.numel[k], i0 + chunk);
  if (c64 == c64 && (double)c != c64) chunk_scale64(t.io[k], t.out_io[k], t.grad[k], t.out[k], i0, i1, c64);
  else if (t.io[k] == IO_F32) chunk_scale_to<IO_F32>(t.out_io[k], t.grad[k], t.out[k], i0, i1, c);
  else if (t.io[k] == IO_BF16) chunk_scale_to<IO_BF16>(t.out_io[k], t.grad[k], t.out[k], i0, i1, c);
  else chunk_scale_to<IO_F16>(t.out_io[k], t.grad[k], t.out[k], i0, i1, c);
}

}  // namespace

ClipPlan clip_plan(int n, const int64_t* numel, int num_cus) {
  ClipPlan p{};
  long long total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  // eight workgroups a CU where the tensors are large enough, of 8 K to 64 K elements each
  p.chunk = 8192;
  while (p.chunk < 65536 && total / p.chunk > 8LL * num_cus) p.chunk *= 2;
  for (int i = 0; i < n; ++i) p.blocks += (numel[i] + p.chunk - 1) / p.chunk;
  p.ws_bytes = (size_t)(p.blocks + 1) * sizeof(double);
  return p;
}

// f(table, workgroups, workgroups before it) for as many tables as the tensors take, in chunks of `chunk` elements
template <typename F>
static hipError_t for_tables(int n, const ClipTensor* t, long long chunk, F f) {
  long long done = 0;
  for (int i = 0; i < n;) {
    ClipTable tab{};
    long long blocks = 0;
    for (; i < n && tab.n < kMaxTensors; ++i) {
      const long long b = (t[i].numel + chunk - 1) / chunk;
      if (b == 0) continue;
      if (b > 0x7fffffffLL) return hipErrorInvalidValue;
      if (blocks + b > 0x7fffffffLL) break;
      const int k = tab.n++;
      tab.grad[k] = t[i].grad;
      tab.out[k] = t[i].out;
      tab.numel[k] = (unsigned long long)t[i].numel;
      tab.first[k] = (unsigned)blocks;
      tab.io[k] = (unsigned char)t[i].io;
      tab.out_io[k] = (unsigned char)t[i].out_io;
      blocks += b;
    }
    if (blocks == 0) continue;
    f(tab, blocks, done);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    done += blocks;
  }
  return hipSuccess;
}

hipError_t launch_clip(int n, const ClipTensor* t, const ClipPlan& p, bool clip, float max_norm, float* norm, void* ws,
                       hipStream_t st) {
  double* part = (double*)ws;
  double* coef = clip ? part + p.blocks : nullptr;
  hipError_t e = for_tables(n, t, p.chunk, [&](const ClipTable& tab, long long blocks, long long done) {
    hipLaunchKernelGGL(norm_kernel, dim3((unsigned)blocks), dim3(256), 0, st, tab, p.chunk, part + done);
  });
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(1024), 0, st, part, p.blocks, max_norm, norm, coef);
  if ((e = hipGetLastError()) != hipSuccess || !clip) return e;
  return for_tables(n, t, kScaleChunk, [&](const ClipTable& tab, long long blocks, long long) {
    hipLaunchKernelGGL(scale_kernel, dim3((unsigned)blocks), dim3(256), 0, st, tab, (long long)kScaleChunk, coef);
  });
}

}  // namespace fmlp

// Routing for gfx950: each token's k experts of N and their weights, and the logits' gradient.
//
//   p = softmax(l);  the k largest l, ties to the lowest index;  w = p of them, or p over their sum (normalize)
//   normalize: dl = w (dw - sum w dw) at the chosen ones, 0 elsewhere
//   else:      dl = p ([chosen] dw - sum over the chosen of p dw)
//
// A row has a group of 1 to 64 lanes with 8 (16) consecutive logits each; a round of the choice is each lane's largest
// key that is left, compared over the group. Keys are the logits' bits in an order that integers compare, NaN
// largest; key 0 is what no choice takes: a masked logit (-infinity) and one that is taken. A
// token with fewer than k unmasked logits has -1 and the weight 0 in place of the rest.
#include "fmlp_experts.h"
#include "fmlp_vec.h"

namespace fmlp {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ unsigned key_of(float f) {
  if (f != f) return 0xffffffffu;
  const unsigned u = __float_as_uint(f + 0.f);  // -0 is 0
  if (u == 0xff800000u) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// VPL logits of a row from element i0 of it; -infinity past the row's end
template <int IO, int VPL>
__device__ __forceinline__ void load_logits(const void* logits, long long row, int i0, int N, bool there, float (&v)[VPL]) {
  constexpr int E = kPiece<IO>;
#pragma unroll
  for (int q = 0; q < VPL / E; ++q) {
    const int n = there ? N - i0 - q * E : 0;
    float f[E];
    unpack_piece<IO>(load_piece<IO>(logits, row + i0 + q * E, n), f);
#pragma unroll
    for (int j = 0; j < E; ++j) v[q * E + j] = j < n ? f[j] : -__builtin_inff();
  }
}

template <int IO, int VPL>
__global__ void __launch_bounds__(kThreads) route_fwd_kernel(RouteArgs a, int lg) {
  extern __shared__ float route_lds[];
  const int G = 1 << lg, rows = kThreads >> lg, k = a.k;
  float* ew = route_lds;             // [rows][k] exponentials of the chosen
  int* ei = (int*)(ew + rows * k);   // [rows][k] their experts
  float* inv = (float*)(ei + rows * k);  // [rows] factor of the row's weights
  const int r = (int)threadIdx.x >> lg, g = (int)threadIdx.x & (G - 1);
  const long long t0 = (long long)blockIdx.x * rows, t = t0 + r;
  float v[VPL];
  load_logits<IO, VPL>(a.logits, t * a.stride, g * VPL, a.N, t < a.T, v);
  unsigned key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) key[i] = key_of(v[i]);
  float top = 0.f, sum = 0.f;
  for (int j = 0; j < k; ++j) {
    unsigned bk = key[0];
    int bi = 0;
#pragma unroll
    for (int i = 1; i < VPL; ++i)
      if (key[i] > bk) {
        bk = key[i];
        bi = i;
      }
    bi += g * VPL;
    for (int d = 1; d < G; d <<= 1) {
      const unsigned ok = (unsigned)__shfl_xor((int)bk, d, 64);
      const int oi = __shfl_xor(bi, d, 64);
      if (ok > bk || (ok == bk && oi < bi)) {
        bk = ok;
        bi = oi;
      }
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (bi == g * VPL + i) key[i] = 0u;
    const float l = of_key(bk);
    if (j == 0) top = l;
    const float e = bk == 0u ? 0.f : exp_of(l - top);
    sum += e;
    if (g == 0) {
      ew[r * k + j] = e;
      ei[r * k + j] = bk == 0u ? -1 : bi;
    }
  }
  if (!a.normalize) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += v[i] == -__builtin_inff() ? 0.f : exp_of(v[i] - top);
    for (int d = 1; d < G; d <<= 1) sum += __shfl_xor(sum, d, 64);
  }
  if (g == 0) inv[r] = sum == 0.f ? 0.f : 1.f / sum;
  __syncthreads();
  for (int i = threadIdx.x; i < rows * k; i += kThreads) {
    const int row = i / k;
    if (t0 + row >= a.T) break;
    const int e = ei[i];
    a.experts[t0 * k + i] = e;
    a.weights[t0 * k + i] = e < 0 ? 0.f : ew[i] * inv[row];
  }
}

template <int IO, int VPL>
__global__ void __launch_bounds__(kThreads) route_bwd_kernel(RouteArgs a, int lg) {
  const int G = 1 << lg, k = a.k;
  const int r = (int)threadIdx.x >> lg, g = (int)threadIdx.x & (G - 1);
  const long long t = (long long)blockIdx.x * (kThreads >> lg) + r;
  const bool there = t < a.T;
  const float* w = a.weights + t * k;
  const float* dw = a.dweights + t * k;
  const int32_t* ex = a.experts + t * k;
  float inner = 0.f;
  if (there)
    for (int j = 0; j < k; ++j)
      if (ex[j] >= 0) inner += w[j] * dw[j];
  float d[VPL];
  if (a.normalize) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] = 0.f;
  } else {
    float v[VPL], top = -__builtin_inff(), sum = 0.f;
    load_logits<IO, VPL>(a.logits, t * a.stride, g * VPL, a.N, there, v);
    bool nan = false;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      nan = nan || v[i] != v[i];
      top = fmaxf(top, v[i]);
    }
    if (nan) top = __uint_as_float(0x7fc00000u);
    for (int s = 1; s < G; s <<= 1) {
      const float o = __shfl_xor(top, s, 64);
      top = o != o || top != top ? __uint_as_float(0x7fc00000u) : fmaxf(top, o);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      d[i] = v[i] == -__builtin_inff() ? 0.f : exp_of(v[i] - top);
      sum += d[i];
    }
    for (int s = 1; s < G; s <<= 1) sum += __shfl_xor(sum, s, 64);
    const float f = sum == 0.f ? 0.f : -inner / sum;
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] *= f;
  }
  if (!there) return;
  for (int j = 0; j < k; ++j) {
    const int at = ex[j] - g * VPL;
    const float add = a.normalize ? w[j] * (dw[j] - inner) : w[j] * dw[j];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (at == i) d[i] += add;
  }
  constexpr int E = kPiece<IO>;
#pragma unroll
  for (int q = 0; q < VPL / E; ++q) {
    const int i0 = g * VPL + q * E;
    float f[E];
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = d[q * E + j];
    store_piece<IO>(a.dlogits, t * a.N + i0, a.N - i0, pack_piece<IO>(f));
  }
}

template <typename F>
hipError_t by_form(const RouteArgs& a, F f) {
  // 8 logits a lane, 16 where 64 lanes would not do
  const int vpl = a.N <= 512 ? 8 : 16;
  int lg = 0;
  while ((vpl << lg) < a.N) ++lg;
  const long long rows = kThreads >> lg, blocks = (a.T + rows - 1) / rows;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks);
  const auto io = [&](auto VPL) {
    if (a.io == IO_F32) f(std::integral_constant<int, IO_F32>{}, VPL, grid, lg);
    else if (a.io == IO_BF16) f(std::integral_constant<int, IO_BF16>{}, VPL, grid, lg);
    else f(std::integral_constant<int, IO_F16>{}, VPL, grid, lg);
  };
  if (vpl == 8) io(std::integral_constant<int, 8>{});
  else io(std::integral_constant<int, 16>{});
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route_fwd(const RouteArgs& a, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  return by_form(a, [&](auto IO, auto VPL, dim3 grid, int lg) {
    const size_t rows = (size_t)kThreads >> lg, lds = rows * (2 * (size_t)a.k + 1) * 4;
    hipLaunchKernelGGL((route_fwd_kernel<decltype(IO)::value, decltype(VPL)::value>), grid, dim3(kThreads), lds, st, a, lg);
  });
}

hipError_t launch_route_bwd(const RouteArgs& a, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  return by_form(a, [&](auto IO, auto VPL, dim3 grid, int lg) {
    hipLaunchKernelGGL((route_bwd_kernel<decltype(IO)::value, decltype(VPL)::value>), grid, dim3(kThreads), 0, st, a, lg);
  });
}

}  // namespace fmlp

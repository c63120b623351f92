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
//
// Bound by vector issue, about 60 instructions a round and wave of 8 rows at 64 experts: 65536 x 64 bf16, 8 a token, 11.7 us (12 MB),
// the gradient 7.3 (15 MB). Maxima over the group through the LDS crossbar and every lane's scan of the chosen index: 16.4; the choices
// of a row read by each of its lanes: 10.4.
#include <algorithm>

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

// The largest v, and the sum, over a group of 1 << LG lanes: within 16 lanes by DPP (lanes swapped in pairs, pairs in quads, quads and
// halves mirrored), beyond by the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <int LG, typename OP>
__device__ __forceinline__ int group_reduce(int v, OP op) {
  if constexpr (LG > 0) v = op(v, dpp<0xB1>(v));
  if constexpr (LG > 1) v = op(v, dpp<0x4E>(v));
  if constexpr (LG > 2) v = op(v, dpp<0x141>(v));
  if constexpr (LG > 3) v = op(v, dpp<0x140>(v));
  if constexpr (LG > 4) v = op(v, __shfl_xor(v, 16, 64));
  if constexpr (LG > 5) v = op(v, __shfl_xor(v, 32, 64));
  return v;
}
template <int LG>
__device__ __forceinline__ unsigned group_max(unsigned v) {
  return (unsigned)group_reduce<LG>((int)v, [](int a, int b) { return (int)max((unsigned)a, (unsigned)b); });
}
template <int LG>
__device__ __forceinline__ float group_sum(float v) {
  return __int_as_float(group_reduce<LG>(__float_as_int(v), [](int a, int b) { return __float_as_int(__int_as_float(a) + __int_as_float(b)); }));
}

template <int IO, int VPL, int LG>
__global__ void __launch_bounds__(kThreads) route_fwd_kernel(RouteArgs a) {
  extern __shared__ float route_lds[];
  constexpr int G = 1 << LG, ROWS = kThreads >> LG;
  const int k = a.k;
  float* ew = route_lds;                 // [ROWS][k] exponentials of the chosen
  int* ei = (int*)(ew + ROWS * k);       // [ROWS][k] their experts
  float* inv = (float*)(ei + ROWS * k);  // [ROWS] factor of the row's weights
  const int r = (int)threadIdx.x >> LG, g = (int)threadIdx.x & (G - 1), first = (int)threadIdx.x & 63 & ~(G - 1);
  const long long t0 = (long long)blockIdx.x * ROWS, t = t0 + r;
  float v[VPL];
  load_logits<IO, VPL>(a.logits, t * a.stride, g * VPL, a.N, t < a.T, v);
  unsigned key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) key[i] = key_of(v[i]);
  float top = 0.f, sum = 0.f;
  for (int j = 0; j < k; ++j) {
    unsigned mk = key[0];
    int mi = 0;
#pragma unroll
    for (int i = 1; i < VPL; ++i)
      if (key[i] > mk) {
        mk = key[i];
        mi = i;
      }
    const unsigned bk = group_max<LG>(mk);
    // the first lane that has it: lanes' logits follow one another
    const unsigned long long has = (__ballot(mk == bk) >> first) & (G == 64 ? ~0ull : (1ull << (G & 63)) - 1);
    const bool mine = __ffsll((long long)has) - 1 == g;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (mine && i == mi) key[i] = 0u;
    const float l = of_key(bk);
    if (j == 0) top = l;
    const float e = bk == 0u ? 0.f : exp_of(l - top);
    sum += e;
    if (mine) {
      ew[r * k + j] = e;
      ei[r * k + j] = bk == 0u ? -1 : g * VPL + mi;
    }
  }
  if (!a.normalize) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += v[i] == -__builtin_inff() ? 0.f : exp_of(v[i] - top);
    sum = group_sum<LG>(sum);
  }
  if (g == 0) inv[r] = sum == 0.f ? 0.f : 1.f / sum;
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * k; i += kThreads) {
    const int row = i / k;
    if (t0 + row >= a.T) break;
    const int e = ei[i];
    a.experts[t0 * k + i] = e;
    a.weights[t0 * k + i] = e < 0 ? 0.f : ew[i] * inv[row];
  }
}

template <int IO, int VPL, int LG>
__global__ void __launch_bounds__(kThreads) route_bwd_kernel(RouteArgs a) {
  extern __shared__ float route_lds[];
  constexpr int G = 1 << LG, ROWS = kThreads >> LG;
  const int k = a.k;
  float* lw = route_lds;             // [ROWS][k] w dw of the chosen
  float* lv = lw + ROWS * k;         // [ROWS][k] w
  int* le = (int*)(lv + ROWS * k);   // [ROWS][k] experts
  const int r = (int)threadIdx.x >> LG, g = (int)threadIdx.x & (G - 1);
  const long long t0 = (long long)blockIdx.x * ROWS, t = t0 + r;
  const bool there = t < a.T;
  float d[VPL];
  if (!a.normalize) load_logits<IO, VPL>(a.logits, t * a.stride, g * VPL, a.N, there, d);
  for (int i = threadIdx.x; i < ROWS * k; i += kThreads) {
    const bool in = i < (a.T - t0) * k;
    const int e = in ? a.experts[t0 * k + i] : -1;
    const float w = in ? a.weights[t0 * k + i] : 0.f, dw = in ? a.dweights[t0 * k + i] : 0.f;
    lw[i] = e < 0 ? 0.f : w * dw;
    lv[i] = w;
    le[i] = e;
  }
  __syncthreads();
  float inner = 0.f;
  for (int j = 0; j < k; ++j) inner += lw[r * k + j];
  if (a.normalize) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] = 0.f;
  } else {
    unsigned tk = 0u;
#pragma unroll
    for (int i = 0; i < VPL; ++i) tk = max(tk, key_of(d[i]));
    const float top = of_key(group_max<LG>(tk));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      d[i] = d[i] == -__builtin_inff() ? 0.f : exp_of(d[i] - top);
      sum += d[i];
    }
    sum = group_sum<LG>(sum);
    const float f = sum == 0.f ? 0.f : -inner / sum;
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] *= f;
  }
  if (!there) return;
  for (int j = 0; j < k; ++j) {
    const int e = le[r * k + j], at = e < 0 ? -1 : e - g * VPL;
    const float add = a.normalize ? __builtin_fmaf(-lv[r * k + j], inner, lw[r * k + j]) : lw[r * k + j];
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

// f(io, logits of a lane, log2 of a row's lanes, workgroups, arguments): 8 logits a lane, 16 where 64 lanes would not do. Rows beyond
// kLaunchThreads' (2^25 of more than 256 experts) take another launch.
template <typename F>
hipError_t by_form(const RouteArgs& all, F f) {
  int lg = 0;
  while (lg < 6 && (8 << lg) < all.N) ++lg;
  const long long rows = kThreads >> lg, most = kLaunchThreads / kThreads * rows, es = all.io == IO_F32 ? 4 : 2;
  RouteArgs a = all;
  dim3 grid;
  const auto io = [&](auto VPL, auto LG) {
    if (a.io == IO_F32) f(std::integral_constant<int, IO_F32>{}, VPL, LG, grid, a);
    else if (a.io == IO_BF16) f(std::integral_constant<int, IO_BF16>{}, VPL, LG, grid, a);
    else f(std::integral_constant<int, IO_F16>{}, VPL, LG, grid, a);
  };
  const auto eight = std::integral_constant<int, 8>{};
  for (long long t0 = 0; t0 < all.T; t0 += most) {
    a.T = std::min(most, all.T - t0);
    a.logits = all.logits == nullptr ? nullptr : (const char*)all.logits + t0 * all.stride * es;
    a.weights = all.weights + t0 * all.k;
    a.experts = all.experts + t0 * all.k;
    if (all.dweights != nullptr) {
      a.dweights = all.dweights + t0 * all.k;
      a.dlogits = (char*)all.dlogits + t0 * all.N * es;
    }
    grid = dim3((unsigned)((a.T + rows - 1) / rows));
    switch (lg) {
      case 0: io(eight, std::integral_constant<int, 0>{}); break;
      case 1: io(eight, std::integral_constant<int, 1>{}); break;
      case 2: io(eight, std::integral_constant<int, 2>{}); break;
      case 3: io(eight, std::integral_constant<int, 3>{}); break;
      case 4: io(eight, std::integral_constant<int, 4>{}); break;
      case 5: io(eight, std::integral_constant<int, 5>{}); break;
      default:
        if (a.N <= 512) io(eight, std::integral_constant<int, 6>{});
        else io(std::integral_constant<int, 16>{}, std::integral_constant<int, 6>{});
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_route_fwd(const RouteArgs& all, hipStream_t st) {
  return by_form(all, [&](auto IO, auto VPL, auto LG, dim3 grid, const RouteArgs& a) {
    constexpr int L = decltype(LG)::value;
    const size_t lds = (size_t)(kThreads >> L) * (2 * (size_t)a.k + 1) * 4;
    hipLaunchKernelGGL((route_fwd_kernel<decltype(IO)::value, decltype(VPL)::value, L>), grid, dim3(kThreads), lds, st, a);
  });
}

hipError_t launch_route_bwd(const RouteArgs& all, hipStream_t st) {
  return by_form(all, [&](auto IO, auto VPL, auto LG, dim3 grid, const RouteArgs& a) {
    constexpr int L = decltype(LG)::value;
    const size_t lds = (size_t)(kThreads >> L) * 3 * (size_t)a.k * 4;
    hipLaunchKernelGGL((route_bwd_kernel<decltype(IO)::value, decltype(VPL)::value, L>), grid, dim3(kThreads), lds, st, a);
  });
}

}  // namespace fmlp

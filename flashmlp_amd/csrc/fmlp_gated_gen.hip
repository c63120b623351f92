// Gated multi-head MLP on gfx950, kernels that read every operand from global memory.
//
//   forward   G = X Wg, U = X Wu, h = act(G) U, O = h W2                       per head
//   backward  dH = dO W2^T, dG = dH U act'(G), dU = dH act(G),
//             dX = dG Wg^T + dU Wu^T, dWg = X^T dG, dWu = X^T dU, dW2 = h^T dO
//
// All contractions on 32x32 MFMA tiles with fp32 sums; h, dG and dU are rounded to the io type
// where they become MFMA operands (16-bit io; fp32 io rounds nothing), as the ungated kernels do.
// The (H, B, E) planes never leave registers. One operand layout serves both MFMA shapes: a lane
// holds 8 k-slots 8 (l / 32) + j; 16-bit io contracts the 16 slots in one v_mfma_f32_32x32x16, fp32
// in eight v_mfma_f32_32x32x2 that pair slot j of both lane halves.
#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

template <int IO>
struct GenIo {
  typedef u16 T;
  typedef u32x4 Frag;
};
template <>
struct GenIo<IO_F32> {
  typedef float T;
  struct Frag {
    float v[8];
  };
};

template <int IO>
__device__ __forceinline__ f32x16 mma(const typename GenIo<IO>::Frag& a, const typename GenIo<IO>::Frag& b, f32x16 c) {
  if constexpr (IO == IO_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
  } else {
    return mfma<IO == IO_BF16>(a, b, c);
  }
}

template <int IO>
__device__ __forceinline__ typename GenIo<IO>::Frag frag_of(const typename GenIo<IO>::T (&v)[8]) {
  typename GenIo<IO>::Frag f;
  if constexpr (IO == IO_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (unsigned)v[2 * j] | ((unsigned)v[2 * j + 1] << 16);
  }
  return f;
}

// fp32 values i0 .. i0 + 7 of a C tile as an operand (its rows become the k-slots)
template <int IO>
__device__ __forceinline__ typename GenIo<IO>::Frag frag_c(const float (&v)[16], int i0) {
  typename GenIo<IO>::Frag f;
  if constexpr (IO == IO_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = v[i0 + j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pack2<IO == IO_BF16>(v[i0 + 2 * j], v[i0 + 2 * j + 1]);
  }
  return f;
}

// 8 elements p[j * step] as an operand; element j is zero where !ok(j)
template <int IO, typename F>
__device__ __forceinline__ typename GenIo<IO>::Frag gather(const typename GenIo<IO>::T* p, F off, bool any) {
  typename GenIo<IO>::T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const long long o = any ? off(j) : -1;
    v[j] = o >= 0 ? p[o] : (typename GenIo<IO>::T)0;
  }
  return frag_of<IO>(v);
}

template <int IO>
__device__ __forceinline__ void put(void* out, size_t i, float v) {
  if constexpr (IO == IO_F32) ((float*)out)[i] = v;
  else ((u16*)out)[i] = from_f32<IO == IO_BF16>(v);
}

// act(z) and act'(z), the activation chosen at run time
__device__ __forceinline__ void act_any(int act, float z, float& h, float& f) {
  if (act == ACT_SILU) act_hf<ACT_SILU>(z, h, f);
  else if (act == ACT_LEAKY) act_hf<ACT_LEAKY>(z, h, f);
  else if (act == ACT_SIGMOID) act_hf<ACT_SIGMOID>(z, h, f);
  else act_hf<ACT_NONE>(z, h, f);
}

// row of element i of a C tile held by lane half g; as a k-slot order: i = 8 s + j is slot j of step s
__device__ __forceinline__ int crow(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// Forward: a wave owns 32 rows (lane = row), walks E in tiles of 32 columns.
template <int IO, int D>
__global__ void __launch_bounds__(256) gated_gen_fwd(GatedArgs a, int tiles) {
  typedef typename GenIo<IO>::T T;
  typedef typename GenIo<IO>::Frag Frag;
  constexpr int KS = D / 16, NT = (D + 31) / 32;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int h = blockIdx.x / tiles, b0 = (blockIdx.x % tiles) * 128 + (threadIdx.x >> 6) * 32;
  const int b = b0 + l32, E = (int)a.E, B = (int)a.B;
  const T* X = (const T*)a.x + (size_t)h * a.sx + (size_t)b * D;
  const T* Wg = (const T*)a.wg + (size_t)h * D * a.ldw;
  const T* Wu = (const T*)a.wu + (size_t)h * D * a.ldw;
  const T* W2 = (const T*)a.w2 + (size_t)h * E * D;
  f32x16 o[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) o[n] = zero16();
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + l32;
    f32x16 zg = zero16(), zu = zero16();
#pragma unroll 1
    for (int k = 0; k < KS; ++k) {
      const int d = k * 16 + 8 * g;
      const Frag x = gather<IO>(X, [&](int j) { return (long long)(d + j); }, b < B);
      const auto w = [&](int j) { return (long long)(d + j) * a.ldw + e; };
      zg = mma<IO>(gather<IO>(Wg, w, e < E), x, zg);
      zu = mma<IO>(gather<IO>(Wu, w, e < E), x, zu);
    }
    float hv[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s, f;
      act_any(a.act, zg[i], s, f);
      hv[i] = e0 + crow(i, g) < E ? s * zu[i] : 0.f;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int d = n * 32 + l32;
        const auto w = [&](int j) {
          const int ee = e0 + crow(8 * s + j, g);
          return ee < E ? (long long)ee * D + d : -1LL;
        };
        o[n] = mma<IO>(frag_c<IO>(hv, 8 * s), gather<IO>(W2, w, d < D), o[n]);
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = b0 + crow(i, g), d = n * 32 + l32;
      if (r < B && d < D) put<IO>(a.o, ((size_t)h * B + r) * D + d, o[n][i]);
    }
}

// dX: the same walk; Z and dH transposed (lane = row), dX += dG Wg^T + dU Wu^T.
template <int IO, int D>
__global__ void __launch_bounds__(256) gated_gen_dx(GatedArgs a, int tiles) {
  typedef typename GenIo<IO>::T T;
  typedef typename GenIo<IO>::Frag Frag;
  constexpr int KS = D / 16, NT = (D + 31) / 32;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int h = blockIdx.x / tiles, b0 = (blockIdx.x % tiles) * 128 + (threadIdx.x >> 6) * 32;
  const int b = b0 + l32, E = (int)a.E, B = (int)a.B;
  const T* X = (const T*)a.x + (size_t)h * a.sx + (size_t)b * D;
  const T* dO = (const T*)a.dout + (size_t)h * a.sdo + (size_t)b * D;
  const T* Wg = (const T*)a.wg + (size_t)h * D * a.ldw;
  const T* Wu = (const T*)a.wu + (size_t)h * D * a.ldw;
  const T* W2 = (const T*)a.w2 + (size_t)h * E * D;
  f32x16 o[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) o[n] = zero16();
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + l32;
    f32x16 zg = zero16(), zu = zero16(), dh = zero16();
#pragma unroll 1
    for (int k = 0; k < KS; ++k) {
      const int d = k * 16 + 8 * g;
      const auto row = [&](int j) { return (long long)(d + j); };
      const auto w = [&](int j) { return (long long)(d + j) * a.ldw + e; };
      const Frag x = gather<IO>(X, row, b < B);
      zg = mma<IO>(gather<IO>(Wg, w, e < E), x, zg);
      zu = mma<IO>(gather<IO>(Wu, w, e < E), x, zu);
      dh = mma<IO>(gather<IO>(W2, [&](int j) { return (long long)e * D + d + j; }, e < E), gather<IO>(dO, row, b < B), dh);
    }
    float dg[16], du[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s, f;
      act_any(a.act, zg[i], s, f);
      const bool in = e0 + crow(i, g) < E;
      dg[i] = in ? dh[i] * zu[i] * f : 0.f;
      du[i] = in ? dh[i] * s : 0.f;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int d = n * 32 + l32;
        const auto w = [&](int j) {
          const int ee = e0 + crow(8 * s + j, g);
          return ee < E ? (long long)d * a.ldw + ee : -1LL;
        };
        o[n] = mma<IO>(frag_c<IO>(dg, 8 * s), gather<IO>(Wg, w, d < D), o[n]);
        o[n] = mma<IO>(frag_c<IO>(du, 8 * s), gather<IO>(Wu, w, d < D), o[n]);
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = b0 + crow(i, g), d = n * 32 + l32;
      if (r < B && d < D) put<IO>(a.dx, ((size_t)h * B + r) * D + d, o[n][i]);
    }
}

// dW: a wave owns 32 columns of E and at most 128 columns of D of all three gradients and walks the
// rows 32 at a time; Z and dH with lane = column of E, so that h, dG and dU are operands as they come.
template <int IO, int D>
__global__ void __launch_bounds__(64) gated_gen_dw(GatedArgs a, int etiles) {
  typedef typename GenIo<IO>::T T;
  typedef typename GenIo<IO>::Frag Frag;
  constexpr int KS = D / 16, DS = D > 128 ? D / 128 : 1, NT = (D / DS + 31) / 32;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int part = blockIdx.x % DS, t = blockIdx.x / DS;
  const int h = t / etiles, e0 = (t % etiles) * 32, e = e0 + l32, E = (int)a.E, B = (int)a.B, d0 = part * 128;
  const T* X = (const T*)a.x + (size_t)h * a.sx;
  const T* dO = (const T*)a.dout + (size_t)h * a.sdo;
  const T* Wg = (const T*)a.wg + (size_t)h * D * a.ldw;
  const T* Wu = (const T*)a.wu + (size_t)h * D * a.ldw;
  const T* W2 = (const T*)a.w2 + (size_t)h * E * D;
  f32x16 sg[NT], su[NT], s2[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) sg[n] = su[n] = s2[n] = zero16();
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + l32;
    f32x16 zg = zero16(), zu = zero16(), dh = zero16();
#pragma unroll 1
    for (int k = 0; k < KS; ++k) {
      const int d = k * 16 + 8 * g;
      const auto row = [&](int j) { return (long long)b * D + d + j; };
      const auto w = [&](int j) { return (long long)(d + j) * a.ldw + e; };
      const Frag x = gather<IO>(X, row, b < B);
      zg = mma<IO>(x, gather<IO>(Wg, w, e < E), zg);
      zu = mma<IO>(x, gather<IO>(Wu, w, e < E), zu);
      dh = mma<IO>(gather<IO>(dO, row, b < B), gather<IO>(W2, [&](int j) { return (long long)e * D + d + j; }, e < E), dh);
    }
    float hv[16], dg[16], du[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s, f;
      act_any(a.act, zg[i], s, f);
      hv[i] = s * zu[i];
      dg[i] = dh[i] * zu[i] * f;
      du[i] = dh[i] * s;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int d = d0 + n * 32 + l32;
        const auto row = [&](int j) {
          const int r = b0 + crow(8 * s + j, g);
          return r < B ? (long long)r * D + d : -1LL;
        };
        const Frag x = gather<IO>(X, row, d < D);
        s2[n] = mma<IO>(frag_c<IO>(hv, 8 * s), gather<IO>(dO, row, d < D), s2[n]);  // rows e, columns d
        sg[n] = mma<IO>(x, frag_c<IO>(dg, 8 * s), sg[n]);                            // rows d, columns e
        su[n] = mma<IO>(x, frag_c<IO>(du, 8 * s), su[n]);
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = crow(i, g), d = d0 + n * 32;
      if (e0 + r < E && d + l32 < D) put<IO>(a.dw2, ((size_t)h * E + e0 + r) * D + d + l32, s2[n][i] * a.dw_scale);
      if (d + r < D && e < E) {
        put<IO>(a.dwg, ((size_t)h * D + d + r) * E + e, sg[n][i] * a.dw_scale);
        put<IO>(a.dwu, ((size_t)h * D + d + r) * E + e, su[n][i] * a.dw_scale);
      }
    }
}

enum { GEN_FWD, GEN_DX, GEN_DW };

template <int IO, int D>
hipError_t launch_d(const GatedArgs& a, int what, hipStream_t st) {
  const long long rows = (a.B + 127) / 128, ets = (a.E + 31) / 32;
  const long long n = what == GEN_DW ? a.H * ets * (D > 128 ? D / 128 : 1) : a.H * rows;
  if (n <= 0) return hipSuccess;
  if (n > 0x7fffffffLL) return hipErrorInvalidValue;
  if (what == GEN_FWD) hipLaunchKernelGGL((gated_gen_fwd<IO, D>), dim3((unsigned)n), dim3(256), 0, st, a, (int)rows);
  else if (what == GEN_DX) hipLaunchKernelGGL((gated_gen_dx<IO, D>), dim3((unsigned)n), dim3(256), 0, st, a, (int)rows);
  else hipLaunchKernelGGL((gated_gen_dw<IO, D>), dim3((unsigned)n), dim3(64), 0, st, a, (int)ets);
  return hipGetLastError();
}

template <int IO>
hipError_t launch_io(const GatedArgs& a, int what, hipStream_t st) {
  switch (a.D) {
    case 16: return launch_d<IO, 16>(a, what, st);
    case 32: return launch_d<IO, 32>(a, what, st);
    case 64: return launch_d<IO, 64>(a, what, st);
    case 128: return launch_d<IO, 128>(a, what, st);
    case 256: return launch_d<IO, 256>(a, what, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_gen(const GatedArgs& a, int what, hipStream_t st) {
  if (a.io == IO_F32) return launch_io<IO_F32>(a, what, st);
  return a.io == IO_BF16 ? launch_io<IO_BF16>(a, what, st) : launch_io<IO_F16>(a, what, st);
}

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

hipError_t launch_gated_gen_fwd(const GatedArgs& a, hipStream_t st) { return launch_gen(a, GEN_FWD, st); }
hipError_t launch_gated_gen_dx(const GatedArgs& a, hipStream_t st) { return launch_gen(a, GEN_DX, st); }
hipError_t launch_gated_gen_dw(const GatedArgs& a, hipStream_t st) { return launch_gen(a, GEN_DW, st); }

}  // namespace fmlp

// Newton-Schulz steps on Gram matrices for gfx950.
//
//   X <- q(X X^T) X,  q(l) = a + b l + c l^2,  is on G = X X^T alone:  Q = a + b G + c G^2,  P <- Q P,  G <- Q G Q
//
// All of these are polynomials of one symmetric matrix: symmetric, and they commute. So a matrix's row is its column, and
// what a wave holds as columns of a product (the result layout of the matrix instruction: lane = column, 16 rows of a
// tile) is, as rows, what it writes to LDS for the next product's left operand, 16 bytes at a time, and as columns the
// right operand straight from its registers. Each wave owns 32 columns of G, P and the product. So a left operand L is L^T, and
// rounding leaves none quite symmetric: products are ordered as Q^T G^T Q, whose antisymmetric part
// shrinks with q^2. (Q^T Q^T G lets it grow 7-fold a step where l is near 1: 2e-4 instead of 3e-6 after five steps at n = 16.)
//
// 32-bit values go through the matrix units as two fp16 terms, hi + lo, of the value times a power of two (22 bits; the
// host's bounds of the eigenvalues keep them in range), three products with fp32 sums: 3/16 of the time of fp32
// products at an error of the size of fp32 rounding.
#include "fmlp_device.h"
#include "fmlp_muon.h"

namespace fmlp {
namespace {

// hi and lo fp16 terms of 8 values times s
__device__ __forceinline__ void split8(const float* f, float s, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = f[2 * j] * s, b = f[2 * j + 1] * s;
    hi[j] = pack2<false>(a, b);
    lo[j] = pack2<false>(a - lo_f32<false>(hi[j]), b - hi_f32<false>(hi[j]));
  }
}

// ---------------------------------------------------------------------------------------------
// NP <= 128: a workgroup a matrix, NP / 32 waves
// ---------------------------------------------------------------------------------------------
// byte offset of 16-byte unit u of row r of a [NP][NP] fp16 matrix: units are swapped within a row so that 16
// consecutive rows' units lie on all banks
template <int NP>
__device__ __forceinline__ int unit_off(int r, int u) {
  constexpr int UR = NP / 8;  // units of a row
  const int f = UR >= 16 ? r & 15 : UR == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  return r * (NP * 2) + ((u ^ f) << 4);
}

// The wave's columns as rows of the left operand: unit (tile t, half s, g) of row n holds the 8 values that the lane of
// column n and half g has in acc[t][8 s ..].
template <int NP>
__device__ __forceinline__ void put_left(const f32x16 (&v)[NP / 32], float s, int n, int g) {
#pragma unroll
  for (int t = 0; t < NP / 32; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[t][8 * h + j];
      u32x4 hi, lo;
      split8(f, s, hi, lo);
      const int at = unit_off<NP>(n, t * 4 + h * 2 + g);
      lds_write16(at, hi);
      lds_write16(NP * NP * 2 + at, lo);
    }
}

// out = (left operand in LDS, times its scale) * b, times `back`
template <int NP>
__device__ __forceinline__ void product(f32x16 (&out)[NP / 32], const f32x16 (&b)[NP / 32], float sb, float back, int g,
                                        int l32) {
  constexpr int RB = NP / 32;
#pragma unroll
  for (int t = 0; t < RB; ++t) out[t] = zero16();
#pragma unroll
  for (int kt = 0; kt < RB; ++kt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = b[kt][8 * h + j];
      u32x4 bh, bl;
      split8(f, sb, bh, bl);
#pragma unroll
      for (int t = 0; t < RB; ++t) {
        const int at = unit_off<NP>(32 * t + l32, kt * 4 + h * 2 + g);
        const u32x4 ah = lds_read16(at), al = lds_read16(NP * NP * 2 + at);
        out[t] = mfma<false>(al, bh, out[t]);
        out[t] = mfma<false>(ah, bl, out[t]);
        out[t] = mfma<false>(ah, bh, out[t]);
      }
    }
#pragma unroll
  for (int t = 0; t < RB; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) out[t][i] *= back;
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

template <int NP>
__global__ void __launch_bounds__(NP * 2, 2) iter_kernel(const float* __restrict__ G0, int parts, u16* __restrict__ P0,
                                                         MuonInfo* __restrict__ info, MuonSteps s) {
  constexpr int RB = NP / 32, SCR = NP * NP * 4;  // LDS: the left operand, then the waves' sums
  const int lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = wave * 32 + l32;
  const long long m = blockIdx.x;

  f32x16 G[RB], P[RB], T[RB];
  const float* src = G0 + m * parts * (NP * NP) + (size_t)n * NP + 4 * g;
#pragma unroll
  for (int t = 0; t < RB; ++t) G[t] = zero16();
  for (int p = 0; p < parts; ++p)
#pragma unroll
    for (int t = 0; t < RB; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = *(const float4*)(src + (size_t)p * (NP * NP) + 32 * t + 8 * q);
        G[t][4 * q] += v.x;
        G[t][4 * q + 1] += v.y;
        G[t][4 * q + 2] += v.z;
        G[t][4 * q + 3] += v.w;
      }
  // the lane that has element (n, n) of the trace: row 8 (i / 4) + 4 g + i % 4 of tile `wave` is l32
  float d = 0.f;
#pragma unroll
  for (int t = 0; t < RB; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (t == wave && 8 * (i >> 2) + 4 * g + (i & 3) == l32) d = G[t][i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  float* scr = (float*)(fmlp_lds + SCR);
  if (lane == 0) scr[wave] = d;
  __syncthreads();
  float trace = 0.f;
#pragma unroll
  for (int w = 0; w < RB; ++w) trace += scr[w];
  float inv;
  const MuonInfo fo = info_of(trace, s, s.p_scale[s.steps - 1], &inv);
  if (threadIdx.x == 0) info[m] = fo;
#pragma unroll
  for (int t = 0; t < RB; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) G[t][i] = G[t][i] * inv * inv;

  for (int k = 0; k < s.steps; ++k) {
    const float sg = s.g_scale[k], sq = s.q_scale[k];
    put_left<NP>(G, sg, n, g);
    __syncthreads();
    product<NP>(T, G, sg, 1.f / sg / sg, g, l32);
#pragma unroll
    for (int t = 0; t < RB; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float one = t == wave && 8 * (i >> 2) + 4 * g + (i & 3) == l32 ? s.a[k] : 0.f;
        T[t][i] = __builtin_fmaf(s.c[k], T[t][i], __builtin_fmaf(s.b[k], G[t][i], one));
      }
    if (k + 1 < s.steps) product<NP>(G, T, sq, 1.f / sg / sq, g, l32);  // G Q, in G's place
    __syncthreads();
    put_left<NP>(T, sq, n, g);
    __syncthreads();
    if (k == 0) {
#pragma unroll
      for (int t = 0; t < RB; ++t) P[t] = T[t];
    } else {
      const float sp = s.p_scale[k - 1];
      product<NP>(T, P, sp, 1.f / sq / sp, g, l32);
#pragma unroll
      for (int t = 0; t < RB; ++t) P[t] = T[t];
    }
    if (k + 1 < s.steps) {
      const float st = sg * sq * 0x1p-14f;  // G Q has G's bound times Q's
      product<NP>(T, G, st, 1.f / sq / st, g, l32);
#pragma unroll
      for (int t = 0; t < RB; ++t) G[t] = T[t];
    }
    __syncthreads();
  }
  const float sp = s.p_scale[s.steps - 1];
  u16* dst = P0 + m * (2 * NP * NP) + (size_t)n * NP + 4 * g;
#pragma unroll
  for (int t = 0; t < RB; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = P[t][8 * h + j];
      u32x4 hi, lo;
      split8(f, sp, hi, lo);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        *(u32x2*)(dst + 32 * t + 16 * h + 8 * q) = u32x2{hi[2 * q], hi[2 * q + 1]};
        *(u32x2*)(dst + NP * NP + 32 * t + 16 * h + 8 * q) = u32x2{lo[2 * q], lo[2 * q + 1]};
      }
    }
}

template <int NP>
hipError_t launch_one(long long matrices, const float* G, int parts, u16* P, MuonInfo* info, const MuonSteps& s, hipStream_t st) {
  constexpr int lds = NP * NP * 4 + 64;
  auto k = iter_kernel<NP>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3((unsigned)matrices), dim3(NP * 2), lds, st, G, parts, P, info, s);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// NP = 256: neither LDS nor a wave's registers hold a matrix; each product is a launch of 32 x 32 tiles, its operands from L2
// ---------------------------------------------------------------------------------------------
constexpr int N2 = 256, kMat = 2 * N2 * N2;  // fp16 values of a matrix, first terms, then second ones

__device__ __forceinline__ void put4(u16* dst, float s, const float* f) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = f[j];
    v[4 + j] = 0.f;
  }
  u32x4 hi, lo;
  split8(v, s, hi, lo);
  *(u32x2*)dst = u32x2{hi[0], hi[1]};
  *(u32x2*)(dst + N2 * N2) = u32x2{lo[0], lo[1]};
}

// G as fp16 terms from its partial sums; block b: 16 rows of matrix b / 16
__global__ void __launch_bounds__(256) sum256_kernel(const float* __restrict__ G0, int parts, u16* __restrict__ G,
                                                     MuonInfo* __restrict__ info, MuonSteps s) {
  __shared__ float scr[4];
  const long long m = blockIdx.x >> 4;
  const float* src = G0 + m * parts * (N2 * N2);
  float d = 0.f;
  for (int p = 0; p < parts; ++p) d += src[(size_t)p * (N2 * N2) + (size_t)threadIdx.x * (N2 + 1)];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  if ((threadIdx.x & 63) == 0) scr[threadIdx.x >> 6] = d;
  __syncthreads();
  float inv;
  const MuonInfo fo = info_of((scr[0] + scr[1]) + (scr[2] + scr[3]), s, s.p_scale[s.steps - 1], &inv);
  if (threadIdx.x == 0 && (blockIdx.x & 15) == 0) info[m] = fo;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const size_t at = (size_t)(blockIdx.x & 15) * (16 * N2) + (size_t)(u * 256 + threadIdx.x) * 4;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p) {
      const float4 v = *(const float4*)(src + (size_t)p * (N2 * N2) + at);
      f[0] += v.x;
      f[1] += v.y;
      f[2] += v.z;
      f[3] += v.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = f[j] * inv * inv;
    put4(G + m * kMat + at, s.g_scale[0], f);
  }
}

struct Prod256 {
  const u16* a;  // matrices
  const u16* b;
  u16* out;
  float back, scale;  // 1 / (the operands' scales), the result's scale
  float ca, cb, cc, cg;  // where one of the first three is not 0: ca 1 + cb cg A + cc A B
};

// 64 x 64 tiles of out, a wave 32 x 32; blockIdx.y picks one of two independent products
__global__ void __launch_bounds__(256) prod256_kernel(Prod256 p0, Prod256 p1) {
  const Prod256 p = blockIdx.y == 0 ? p0 : p1;
  const int lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, wave = (int)threadIdx.x >> 6;
  const long long m = blockIdx.x >> 4;
  const int tile = blockIdx.x & 15;
  const int r0 = (tile >> 2) * 64 + (wave >> 1) * 32, c0 = (tile & 3) * 64 + (wave & 1) * 32;
  const u16* A = p.a + m * kMat + (size_t)(r0 + l32) * N2 + 8 * g;
  const u16* B = p.b + m * kMat + (size_t)(c0 + l32) * N2 + 8 * g;
  f32x16 acc = zero16();
#pragma unroll 4
  for (int k = 0; k < N2; k += 16) {
    const u32x4 ah = *(const u32x4*)(A + k), al = *(const u32x4*)(A + N2 * N2 + k);
    const u32x4 bh = *(const u32x4*)(B + k), bl = *(const u32x4*)(B + N2 * N2 + k);
    acc = mfma<false>(al, bh, acc);
    acc = mfma<false>(ah, bl, acc);
    acc = mfma<false>(ah, bh, acc);
  }
  // lane: column c0 + l32, rows r0 + 8 q + 4 g ..; stored as row c0 + l32 (the matrices are symmetric)
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = r0 + 8 * q + 4 * g;
    const size_t at = (size_t)(c0 + l32) * N2 + r;
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = acc[4 * q + j] * p.back;
    if (p.cc != 0.f || p.ca != 0.f || p.cb != 0.f) {
      const u16* a = p.a + m * kMat + at;
      const u32x2 h = *(const u32x2*)a, l = *(const u32x2*)(a + N2 * N2);
      const float v[4] = {lo_f32<false>(h[0]) + lo_f32<false>(l[0]), hi_f32<false>(h[0]) + hi_f32<false>(l[0]),
                          lo_f32<false>(h[1]) + lo_f32<false>(l[1]), hi_f32<false>(h[1]) + hi_f32<false>(l[1])};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = __builtin_fmaf(p.cc, f[j], __builtin_fmaf(p.cb, v[j] * p.cg, r + j == c0 + l32 ? p.ca : 0.f));
    }
    put4(p.out + m * kMat + at, p.scale, f);
  }
}

hipError_t launch_256(long long matrices, const float* G0, int parts, u16* P, MuonInfo* info, const MuonSteps& s, void* ws,
                      hipStream_t st) {
  const size_t one = (size_t)matrices * kMat;
  u16* G = (u16*)ws;
  u16 *Q = G + one, *T = Q + one, *R = T + one;
  hipLaunchKernelGGL(sum256_kernel, dim3((unsigned)(matrices * 16)), dim3(256), 0, st, G0, parts, G, info, s);
  hipError_t e = hipGetLastError();
  const auto run = [&](const Prod256& a, const Prod256* b) {
    if (e != hipSuccess) return;
    hipLaunchKernelGGL(prod256_kernel, dim3((unsigned)(matrices * 16), b ? 2 : 1), dim3(256), 0, st, a, b ? *b : a);
    e = hipGetLastError();
  };
  // P_k, the product of the steps' polynomials so far, takes turns in R and P, the last one in P; the first step's Q is P_0
  const auto pk = [&](int k) { return (s.steps - 1 - k) % 2 == 0 ? P : R; };
  for (int k = 0; k < s.steps; ++k) {
    const float sg = s.g_scale[k], sq = s.q_scale[k];
    u16* q = k == 0 ? pk(0) : Q;
    run(Prod256{G, G, q, 1.f / sg / sg, sq, s.a[k], s.b[k], s.c[k], 1.f / sg}, nullptr);
    Prod256 next{};
    if (k > 0) next = Prod256{q, pk(k - 1), pk(k), 1.f / sq / s.p_scale[k - 1], s.p_scale[k], 0.f, 0.f, 0.f, 0.f};
    if (k + 1 == s.steps) {
      if (k > 0) run(next, nullptr);
      break;
    }
    const float stt = sg * sq * 0x1p-14f;  // G Q has G's bound times Q's
    run(Prod256{G, q, T, 1.f / sg / sq, stt, 0.f, 0.f, 0.f, 0.f}, k > 0 ? &next : nullptr);
    run(Prod256{q, T, G, 1.f / sq / stt, s.g_scale[k + 1], 0.f, 0.f, 0.f, 0.f}, nullptr);
  }
  return e;
}

}  // namespace

size_t muon_iter_ws_bytes(int NP, long long matrices) {
  return NP == 256 ? (size_t)matrices * kMat * 4 * sizeof(u16) : 0;
}

hipError_t launch_muon_iter(int NP, long long matrices, const float* G, int parts, unsigned short* P, MuonInfo* info,
                            const MuonSteps& s, void* ws, hipStream_t st) {
  if (matrices == 0) return hipSuccess;
  if (NP == 32) return launch_one<32>(matrices, G, parts, P, info, s, st);
  if (NP == 64) return launch_one<64>(matrices, G, parts, P, info, s, st);
  if (NP == 128) return launch_one<128>(matrices, G, parts, P, info, s, st);
  return launch_256(matrices, G, parts, P, info, s, ws, st);
}

}  // namespace fmlp

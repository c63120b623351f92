// Gated MLP for gfx950, fp32 io: forward, dX and weight gradients on v_mfma_f32_32x32x2_f32, whose
// 64 clocks per product (16 times a 16-bit one's) are what bounds all three; nothing is rounded before the
// results. The same shapes as the 16-bit kernels: chunks of E or subtiles of rows in a double buffer in LDS filled
// by buffer loads, everything else in registers. One LDS read of four bytes a lane feeds a product, so the
// reads, the activations and the barriers fit beside the products without a schedule written down.
//
// H=12 B=1024 D=64 E=768 SiLU: forward 48 us, dX 71, weight gradients 93 (products 48-52 % of the cycles: 96 tiles and
// 72 column tiles split to fill 256 CUs leave rounds uneven); D = 128 H=8 B=1024 E=512: 49, 71, 95 (the weight
// gradients spill 45 registers, 96 bytes a lane); D = 256, the same: 82, 211, 149 (dX holds X, dO and its sums in
// registers and spills 224, 480 bytes a lane; chunks are single-buffered, as two do not fit the LDS).
//
// Product q of a contraction over d takes d = 2 q + g from lane half g; a contraction over the rows of a C tile
// takes element i of it as it lies (row 8 (i / 4) + 4 g + i % 4).
// LDS rows are swizzled in 16-byte pieces so that reads along rows and down rows meet at most two lanes a bank.
#include <algorithm>
#include <type_traits>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

__device__ __forceinline__ float lds_f32(int off) {
  return *(const FMLP_LDS float*)((FMLP_LDS char*)fmlp_lds + off);
}
__device__ __forceinline__ f32x16 mma(float a, float b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int crow(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// Tile [rows][32 columns], 8 pieces a row: piece p of row r at place p ^ (r / 2 % 8).
__device__ __forceinline__ int off32(int r, int c) { return r * 128 + ((((c >> 2) ^ (r >> 1)) & 7) << 4) + (c & 3) * 4; }
// Tile [rows][D columns], D / 4 pieces a row: piece p of row r at place p ^ (r % 16) (D = 32: r / 2 % 8)
template <int D>
__device__ __forceinline__ int offD(int r, int c) {
  if constexpr (D == 32) return off32(r, c);
  else return r * (4 * D) + (((c >> 2) ^ (r & 15)) << 4) + (c & 3) * 4;
}
// the piece that belongs at 16-byte place p of such a tile
__device__ __forceinline__ void place32(int p, int& r, int& q) {
  r = p >> 3;
  q = (p & 7) ^ ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ void placeD(int p, int& r, int& q) {
  if constexpr (D == 32) {
    place32(p, r, q);
  } else {
    r = p / (D / 4);
    q = (p % (D / 4)) ^ (r & 15);
  }
}

__device__ __forceinline__ void barrier_all() {
  wait_vmcnt<0>();
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Chunk loads of the forward and dX: Wg, Wu [D][32], W2 [32][D] of chunk cg into LDS at `at`.
template <int D, int DG>
struct Chunk {
  static constexpr int NP = 8 * D / 256;  // 16-byte pieces a thread and matrix
  const float *wg, *wu, *w2;
  int E, e_end, ldw;
  unsigned o1[NP], o2[NP];
  int col[NP];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      int r, q;
      place32(k * 256 + (int)threadIdx.x, r, q);
      col[k] = q * 4;
      o1[k] = r < DG ? (unsigned)r * (unsigned)ldw * 4u + (unsigned)q * 16u : BUF_OOB;
      placeD<D>(k * 256 + (int)threadIdx.x, r, q);
      o2[k] = q * 4 < DG ? (unsigned)(r * DG * 4 + q * 16) : BUF_OOB;
    }
  }
  __device__ __forceinline__ void load(int cg, int at) const {
    const int lim = e_end - cg * 32, rem = clamp0(DG * ldw * 4 - 128 * cg, 0x7fffffff);
    const i32x4 rg = make_rsrc_words(wg + (size_t)cg * 32, rem), ru = make_rsrc_words(wu + (size_t)cg * 32, rem);
    const i32x4 r2 = make_rsrc_words(w2 + (size_t)cg * 32 * DG, clamp0(lim, 32) * DG * 4);
    const int a = at + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const unsigned o = col[k] < lim ? o1[k] : BUF_OOB;
      buf_load16_lds(rg, o, a + k * 4096);
      buf_load16_lds(ru, o, a + 128 * D + k * 4096);
      buf_load16_lds(r2, o2[k], a + 256 * D + k * 4096);
    }
  }
};

// Forward (BWD = false) and dX: four waves of 32 rows; chunks cb .. ce - 1 of E.
template <int D, int DG, int ACT, bool BWD>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 64 ? 1 : 2)))
gated32_rows_kernel(const float* __restrict__ X, const float* __restrict__ Wg, const float* __restrict__ Wu,
                    const float* __restrict__ W2, const float* __restrict__ dO, float* __restrict__ out, int B, int E,
                    int ldw, long long sx, long long sdo, int H, int T, int xs, int nct, float* __restrict__ ws) {
  constexpr int KQ = DG / 2, NTN = D / 32, SLOT = 384 * D;
  constexpr bool TWO = D <= 128;  // two chunks fit the LDS
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  int h, bt, cb = 0, ce = (E + 31) >> 5;
  if (xs == 1) {
    const unsigned t = (unsigned)xcd_remap(blockIdx.x, gridDim.x);
    h = (int)(t / (unsigned)T);
    bt = (int)(t % (unsigned)T);
  } else {
    const unsigned s = blockIdx.x / (unsigned)xs, p = blockIdx.x - s * xs;
    h = (int)(s % (unsigned)H);
    bt = (int)(s / (unsigned)H);
    cb = (int)p * nct;
    ce = min(ce, cb + nct);
  }
  Chunk<D, DG> ch;
  ch.wg = Wg + (size_t)h * DG * ldw;
  ch.wu = Wu + (size_t)h * DG * ldw;
  ch.w2 = W2 + (size_t)h * E * DG;
  ch.E = E;
  ch.e_end = min(E, ce * 32);
  ch.ldw = ldw;
  ch.init();
  ch.load(cb, 0);
  const int b_wave = (bt * 4 + wave) * 32, b = b_wave + l32;
  float x[KQ], d[BWD ? KQ : 1];
#pragma unroll
  for (int q = 0; q < KQ; ++q) {
    x[q] = b < B ? X[(size_t)h * sx + (size_t)b * DG + 2 * q + g] : 0.f;
    if constexpr (BWD) d[q] = b < B ? dO[(size_t)h * sdo + (size_t)b * DG + 2 * q + g] : 0.f;
  }
  f32x16 o[NTN];
#pragma unroll
  for (int n = 0; n < NTN; ++n) o[n] = zero16();
  int row8[8];  // row reads of [D][32]: row 2 q + g, column l32 (the swizzle depends on q % 8)
#pragma unroll
  for (int k = 0; k < 8; ++k) row8[k] = off32(2 * k + g, l32);
  for (int c = cb; c < ce; ++c) {
    const int at = TWO ? ((c - cb) & 1) * SLOT : 0;
    if (!TWO && c > cb) {
      barrier_all();
      ch.load(c, 0);
    }
    barrier_all();  // chunk c has landed, and chunk c - 1 is read
    if (TWO && c + 1 < ce) ch.load(c + 1, SLOT - at);
    f32x16 zg = zero16(), zu = zero16(), dh = zero16();
#pragma unroll
    for (int q = 0; q < KQ; ++q) {
      const int a = at + row8[q & 7] + (q >> 3) * 2048;
      zg = mma(lds_f32(a), x[q], zg);
      zu = mma(lds_f32(a + 128 * D), x[q], zu);
      if constexpr (BWD) dh = mma(lds_f32(at + 256 * D + offD<D>(l32, 2 * q + g)), d[q], dh);
      if (D == 256 && (q & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // (reads moved further ahead spill registers)
    }
    if constexpr (!BWD) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = act_f<ACT>(zg[i]) * zu[i];
#pragma unroll
        for (int n = 0; n < NTN; ++n) o[n] = mma(v, lds_f32(at + 256 * D + offD<D>(crow(i, g), n * 32 + l32)), o[n]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s, f;
        act_hf<ACT>(zg[i], s, f);
        const float dg = dh[i] * f * zu[i], du = dh[i] * s;
#pragma unroll
        for (int n = 0; n < NTN; ++n) {
          const int a = at + off32(n * 32 + l32, crow(i, g));
          o[n] = mma(dg, lds_f32(a), o[n]);
          o[n] = mma(du, lds_f32(a + 128 * D), o[n]);
        }
        if (D == 256) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const bool split = xs > 1;
  float* dst = split ? ws + (size_t)blockIdx.x * 128 * DG : out + (size_t)h * B * DG;
  const int r0 = split ? wave * 32 : b_wave, rows = split ? B - bt * 128 : B;
#pragma unroll
  for (int n = 0; n < NTN; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + crow(i, g), c = n * 32 + l32;
      if (r < rows && c < DG) dst[(size_t)r * DG + c] = o[n][i];
    }
}

// Weight gradients: four waves of 32 columns of E; X and dO subtiles of 32 rows. W2's columns stay in LDS at
// D = 128, where three matrices and three gradient tiles do not fit the registers. At D = 256 the four waves share
// 32 columns of E and own a quarter of D each: of the weights, of the contractions over d, whose partial G, U and
// dH go through LDS and are added in wave order by all, and of the gradients.
template <int D, int DG, int ACT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
gated32_dw_kernel(const float* __restrict__ X, const float* __restrict__ Wg, const float* __restrict__ Wu,
                  const float* __restrict__ W2, const float* __restrict__ dO, float* __restrict__ dWg,
                  float* __restrict__ dWu, float* __restrict__ dW2, int H, int B, int E, int ldw, long long sx,
                  long long sdo, int nE, int nS, int rows_per_split, float scale, float* __restrict__ ws) {
  constexpr bool QUARTER = D == 256;
  constexpr int DW = QUARTER ? 64 : D;  // columns of D of a wave
  constexpr int KQ = (QUARTER ? DW : DG) / 2, NTN = DW / 32, SLOT = 256 * D, NP = 8 * D / 256;
  constexpr bool W2LDS = D == 128, TWO = !QUARTER;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  const unsigned t = (unsigned)xcd_remap(blockIdx.x, gridDim.x);
  const int et = (int)(t % (unsigned)nE);
  const unsigned hs = t / (unsigned)nE;
  const int s = (int)(hs % (unsigned)nS), h = (int)(hs / (unsigned)nS);
  const int e0 = (QUARTER ? et : et * 4 + wave) * 32, e = e0 + l32, d0 = QUARTER ? wave * DW : 0;
  const int r0 = s * rows_per_split, r1 = min(B, r0 + rows_per_split), NSUB = max(0, (r1 - r0 + 31) >> 5);
  const float* Xh = X + (size_t)h * sx;
  const float* dOh = dO + (size_t)h * sdo;
  unsigned so[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    int r, q;
    placeD<D>(k * 256 + (int)threadIdx.x, r, q);
    so[k] = q * 4 < DG ? (unsigned)(r * DG * 4 + q * 16) : BUF_OOB;
  }
  auto load_sub = [&](int i, int at) {
    const int b = r0 + 32 * i, n = clamp0(r1 - b, 32) * DG * 4;
    const i32x4 rx = make_rsrc_words(Xh + (size_t)b * DG, n), rd = make_rsrc_words(dOh + (size_t)b * DG, n);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      buf_load16_lds(rx, so[k], at + wave * 1024 + k * 4096);
      buf_load16_lds(rd, so[k], at + 128 * D + wave * 1024 + k * 4096);
    }
  };
  load_sub(0, 0);
  if constexpr (W2LDS) {  // rows e of the E-tile behind the two subtiles
    const int eb = et * 128;
    const i32x4 r2 = make_rsrc_words(W2 + (size_t)h * E * DG + (size_t)eb * DG, clamp0(E - eb, 128) * DG * 4);
#pragma unroll
    for (int k = 0; k < 4 * NP; ++k) {
      int r, q;
      placeD<D>(k * 256 + (int)threadIdx.x, r, q);
      buf_load16_lds(r2, (unsigned)(r * DG * 4 + q * 16), 2 * SLOT + wave * 1024 + k * 4096);
    }
  }
  float wg[KQ], wu[KQ], w2[W2LDS ? 1 : KQ];
#pragma unroll
  for (int q = 0; q < KQ; ++q) {
    const int d = d0 + 2 * q + g;
    const size_t at = ((size_t)h * DG + d) * ldw + e;
    wg[q] = e < E ? Wg[at] : 0.f;
    wu[q] = e < E ? Wu[at] : 0.f;
    if constexpr (!W2LDS) w2[q] = e < E ? W2[((size_t)h * E + e) * DG + d] : 0.f;
  }
  f32x16 ag[NTN], au[NTN], a2[NTN];
#pragma unroll
  for (int n = 0; n < NTN; ++n) ag[n] = au[n] = a2[n] = zero16();
  for (int i = 0; i < NSUB; ++i) {
    const int at = TWO ? (i & 1) * SLOT : 0;
    if (!TWO && i > 0) {
      barrier_all();
      load_sub(i, 0);
    }
    barrier_all();
    if (TWO && i + 1 < NSUB) load_sub(i + 1, SLOT - at);
    f32x16 zg = zero16(), zu = zero16(), dh = zero16();
#pragma unroll
    for (int q = 0; q < KQ; ++q) {
      const int a = offD<D>(l32, d0 + 2 * q + g);
      const float x = lds_f32(at + a);
      zg = mma(x, wg[q], zg);
      zu = mma(x, wu[q], zu);
      dh = mma(lds_f32(at + 128 * D + a), W2LDS ? lds_f32(2 * SLOT + wave * 128 * D + a) : w2[W2LDS ? 0 : q], dh);
      if (W2LDS && (q & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // (reads moved further ahead spill registers)
    }
    if constexpr (QUARTER) {  // the waves' partial sums, [wave][12][lane] of four values behind the subtile
#pragma unroll
      for (int k = 0; k < 12; ++k) {
        const f32x16& v = k < 4 ? zg : k < 8 ? zu : dh;
        const int j = 4 * (k & 3);
        lds_write16(SLOT + ((wave * 12 + k) * 64 + lane) * 16, u32x4{__float_as_uint(v[j]), __float_as_uint(v[j + 1]),
                                                                     __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3])});
      }
      barrier_all();
      zg = zu = dh = zero16();
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int k = 0; k < 12; ++k) {
          const u32x4 u = lds_read16(SLOT + ((w * 12 + k) * 64 + lane) * 16);
          f32x16& v = k < 4 ? zg : k < 8 ? zu : dh;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * (k & 3) + j] += __uint_as_float(u[j]);
        }
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float sv, f;
      act_hf<ACT>(zg[k], sv, f);
      const float hv = sv * zu[k], dg = dh[k] * f * zu[k], du = dh[k] * sv;
#pragma unroll
      for (int n = 0; n < NTN; ++n) {
        const int a = at + offD<D>(crow(k, g), d0 + n * 32 + l32);
        const float x = lds_f32(a);
        ag[n] = mma(x, dg, ag[n]);
        au[n] = mma(x, du, au[n]);
        a2[n] = mma(hv, lds_f32(a + 128 * D), a2[n]);
      }
      if (W2LDS) __builtin_amdgcn_sched_barrier(0);
    }
  }
  wait_vmcnt<0>();  // (loads that no subtile waited for)
  const size_t n1 = (size_t)H * E * DG;
  if (nS > 1) {
    scale = 1.f;  // the sum applies it
    dWg = ws + (size_t)s * 3 * n1;
    dWu = dWg + n1;
    dW2 = dWu + n1;
  }
#pragma unroll
  for (int n = 0; n < NTN; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = crow(i, g), c = d0 + n * 32;
      if (e0 + r < E && c + l32 < DG) dW2[((size_t)h * E + e0 + r) * DG + c + l32] = a2[n][i] * scale;
      if (e < E && c + r < DG) {
        const size_t at = ((size_t)h * DG + c + r) * E + e;
        dWg[at] = ag[n][i] * scale;
        dWu[at] = au[n][i] * scale;
      }
    }
}

__global__ void __launch_bounds__(256) gated32_dw_reduce(const float* __restrict__ ws, float* dWg, float* dWu, float* dW2,
                                                         long long quads, int nS, float scale) {
  const long long q = (long long)blockIdx.x * 256 + threadIdx.x;
  if (q >= 3 * quads) return;
  const int m = q >= 2 * quads ? 2 : q >= quads ? 1 : 0;
  const float4* src = (const float4*)ws + q;
  float4 v = src[0];
  for (int s = 1; s < nS; ++s) {
    const float4 u = src[(size_t)s * 3 * quads];
    v.x += u.x;
    v.y += u.y;
    v.z += u.z;
    v.w += u.w;
  }
  v.x *= scale;
  v.y *= scale;
  v.z *= scale;
  v.w *= scale;
  *(float4*)((m == 0 ? dWg : m == 1 ? dWu : dW2) + 4 * (q - m * quads)) = v;
}

template <int D, int DG, int ACT, bool BWD>
hipError_t launch_rows(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st) {
  auto k = gated32_rows_kernel<D, DG, ACT, BWD>;
  constexpr int lds = (D <= 128 ? 2 : 1) * 384 * D;
  static std::atomic<unsigned long long> done{0};
  hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  void* out = BWD ? a.dx : a.o;
  const int T = (int)(p.tiles / a.H);
  hipLaunchKernelGGL(k, dim3((unsigned)(p.tiles * p.xs)), dim3(256), lds, st, (const float*)a.x, (const float*)a.wg,
                     (const float*)a.wu, (const float*)a.w2, (const float*)a.dout, (float*)out, (int)a.B, (int)a.E,
                     (int)a.ldw, (long long)a.sx, (long long)a.sdo, (int)a.H, T, p.xs, p.nct, (float*)a.ws);
  if ((e = hipGetLastError()) != hipSuccess || p.xs == 1) return e;
  return launch_tile_reduce((const float*)a.ws, out, false, (int)a.B, DG, 128, (int)a.H, T, p.xs, (int)p.tiles, 1, st);
}

template <int D, int DG, int ACT>
hipError_t launch_dw(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st) {
  auto k = gated32_dw_kernel<D, DG, ACT>;
  constexpr int lds = D == 256 ? 256 * D + 48 * 1024 : 512 * D + (D == 128 ? 512 * D : 0);
  static std::atomic<unsigned long long> done{0};
  hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3((unsigned)p.programs), dim3(256), lds, st, (const float*)a.x, (const float*)a.wg,
                     (const float*)a.wu, (const float*)a.w2, (const float*)a.dout, (float*)a.dwg, (float*)a.dwu,
                     (float*)a.dw2, (int)a.H, (int)a.B, (int)a.E, (int)a.ldw, (long long)a.sx, (long long)a.sdo, p.nE,
                     p.nS, p.rows_per_split, a.dw_scale, (float*)a.ws);
  if ((e = hipGetLastError()) != hipSuccess || p.nS == 1) return e;
  const long long quads = (long long)a.H * a.E * a.D / 4, blocks = (3 * quads + 255) / 256;
  hipLaunchKernelGGL(gated32_dw_reduce, dim3((unsigned)blocks), dim3(256), 0, st, (const float*)a.ws, (float*)a.dwg,
                     (float*)a.dwu, (float*)a.dw2, quads, p.nS, a.dw_scale);
  return hipGetLastError();
}

template <int D, int DG, typename F>
hipError_t by_act(int act, F f) {
  switch (act) {
    case ACT_SILU: return f(std::integral_constant<int, D>{}, std::integral_constant<int, DG>{}, std::integral_constant<int, ACT_SILU>{});
    case ACT_LEAKY: return f(std::integral_constant<int, D>{}, std::integral_constant<int, DG>{}, std::integral_constant<int, ACT_LEAKY>{});
    case ACT_SIGMOID: return f(std::integral_constant<int, D>{}, std::integral_constant<int, DG>{}, std::integral_constant<int, ACT_SIGMOID>{});
    default: return f(std::integral_constant<int, D>{}, std::integral_constant<int, DG>{}, std::integral_constant<int, ACT_NONE>{});
  }
}
template <typename F>
hipError_t by_d(const GatedArgs& a, F f) {
  switch (a.D) {
    case 16: return by_act<32, 16>(a.act, f);
    case 32: return by_act<32, 32>(a.act, f);
    case 64: return by_act<64, 64>(a.act, f);
    case 128: return by_act<128, 128>(a.act, f);
    default: return by_act<256, 256>(a.act, f);
  }
}

}  // namespace

// Tiles of 128 rows, split over E where whole tiles leave CUs idle or cut a last round short: the products of
// the workgroups of a CU share its matrix units, so a round costs its chunks whether one or three run there.
GatedFwdPlan gated32_rows_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole) {
  const long long N = std::max(num_cus, 1), nch = (E + 31) / 32;
  GatedFwdPlan p{};
  p.xs = 1;
  p.nct = (int)nch;
  p.tiles = H * ((B + 127) / 128);
  if (p.tiles <= 0) return p;
  const double chunk_us = 3.4 * (double)std::max<long long>(D, 32) / 64.0;
  double best = 0;
  for (long long want = 1; want <= (whole ? 1 : 16) && want <= nch; ++want) {
    const long long nct = (nch + want - 1) / want, xs = (nch + nct - 1) / nct;
    if (xs != want) continue;
    double t = (double)((p.tiles * xs + N - 1) / N) * (double)nct * chunk_us;
    if (xs > 1) t += 3.0 + (double)(H * B * D * xs) * 8.0 / 4.2e6;
    if (best == 0 || t < best) {
      best = t;
      p.xs = (int)xs;
      p.nct = (int)nct;
    }
  }
  p.ws_bytes = p.xs > 1 ? (size_t)p.tiles * p.xs * 128 * D * sizeof(float) : 0;
  return p;
}

GatedDwPlan gated32_dw_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole) {
  GatedDwPlan p{};
  const long long N = std::max(num_cus, 1), subs = (B + 31) / 32;
  p.nE = (int)(D == 256 ? (E + 31) / 32 : (E + 127) / 128);
  const long long base = H * p.nE;
  const double sub_us = D == 256 ? 8.0 : 5.8 * (double)std::max<long long>(D, 32) / 64.0;
  double best = 0;
  p.nS = 1;
  p.rows_per_split = (int)std::max<long long>(subs * 32, 32);
  for (long long n = 1; n <= (whole ? 1 : 32) && (n == 1 || n <= subs); ++n) {
    const long long per = std::max<long long>((subs + n - 1) / n, 1);
    if (n > 1 && (subs + per - 1) / per != n) continue;
    double t = (double)((base * n + N - 1) / N) * (4.0 + sub_us * (double)per);
    if (n > 1) t += 4.0 + (double)(3 * H * D * E * n) * 8.0 / 3.0e6;
    if (best == 0 || t < best) {
      best = t;
      p.nS = (int)n;
      p.rows_per_split = (int)per * 32;
    }
  }
  p.programs = base * p.nS;
  p.ws_bytes = p.nS > 1 ? (size_t)p.nS * 3 * H * D * E * sizeof(float) : 0;
  return p;
}

hipError_t launch_gated32_fwd(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st) {
  if (p.tiles <= 0) return hipSuccess;
  return by_d(a, [&](auto D, auto DG, auto A) { return launch_rows<decltype(D)::value, decltype(DG)::value, decltype(A)::value, false>(a, p, st); });
}
hipError_t launch_gated32_dx(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st) {
  if (p.tiles <= 0) return hipSuccess;
  return by_d(a, [&](auto D, auto DG, auto A) { return launch_rows<decltype(D)::value, decltype(DG)::value, decltype(A)::value, true>(a, p, st); });
}
hipError_t launch_gated32_dw(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st) {
  if (p.programs <= 0) return hipSuccess;
  return by_d(a, [&](auto D, auto DG, auto A) { return launch_dw<decltype(D)::value, decltype(DG)::value, decltype(A)::value>(a, p, st); });
}

}  // namespace fmlp

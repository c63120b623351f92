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
// Measured, a step (four products): 0.7 us at NP = 32, 2.4 at 64, 8.6 at 128 (matrix instructions alone 0.2, 0.7 and 5.4: the
// rest is the chain of LDS reads, conversions and three barriers, as few matrices leave one workgroup a CU); at 256, whose
// products are launches, 15 for 8 matrices and 120 for 192. 32 columns a wave instead of 16: 64 x 683 24 us instead of 18.
//
// 32-bit values go through the matrix units as two fp16 terms, hi + lo, of the value times a power of two (22 bits; the
// host's bounds of the eigenvalues keep them in range), three products with fp32 sums: 3/16 of the time of fp32
// products at an error of the size of fp32 rounding.
#include "fmlp_muon_device.h"

namespace fmlp {
namespace {

// ---------------------------------------------------------------------------------------------
// NP <= 128: a workgroup a matrix, NP / 16 waves of 16 columns each
// ---------------------------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 16 x 16 x 32: A lane l row l % 16, B lane l column l % 16, inner slots 8 (l / 16) ..; result column l % 16, rows
// 4 (l / 16) ..
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// byte offset of 16-byte unit u of row r of a [NP][NP] fp16 matrix: units are swapped within a row so that 16
// consecutive rows' units lie on all banks
template <int NP>
__device__ __forceinline__ int unit_off(int r, int u) {
  constexpr int UR = NP / 8;  // units of a row
  const int f = UR >= 16 ? r & 15 : UR == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  return r * (NP * 2) + ((u ^ f) << 4);
}

// A wave's 16 columns of a matrix as both fp16 terms: unit k of the lane of column n and quarter q holds rows
// 32 k + 4 q + {0..3, 16..19}, the order that two tiles of a result have them in
template <int NP>
struct Cols {
  u32x4 hi[NP / 32], lo[NP / 32];
};
template <int NP>
__device__ __forceinline__ void pack_cols(const f32x4 (&v)[NP / 16], float s, Cols<NP>& c) {
#pragma unroll
  for (int k = 0; k < NP / 32; ++k) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v[2 * k + (j >> 2)][j & 3];
    split8(f, s, c.hi[k], c.lo[k]);
  }
}
// the columns as rows of the left operand
template <int NP>
__device__ __forceinline__ void put_left(const Cols<NP>& c, int n, int q) {
#pragma unroll
  for (int k = 0; k < NP / 32; ++k) {
    const int at = unit_off<NP>(n, 4 * k + q);
    lds_write16(at, c.hi[k]);
    lds_write16(NP * NP * 2 + at, c.lo[k]);
  }
}

// out = (left operand in LDS) * b, in the terms' scales. A step has 32 of the inner dimension for TP tiles of rows.
template <int NP>
__device__ __forceinline__ void product(f32x4 (&out)[NP / 16], const Cols<NP>& b, int q, int l16) {
  constexpr int TP = 2, GROUPS = NP / 16 / TP, STEPS = NP / 32 * GROUPS, AHEAD = 1;
  u32x4 ah[AHEAD + 1][TP], al[AHEAD + 1][TP];
  const auto fetch = [&](int j) {
    const int k = j / GROUPS, p = j % GROUPS;
#pragma unroll
    for (int t = 0; t < TP; ++t) {
      const int at = unit_off<NP>(l16, 4 * k + q) + (p * TP + t) * (16 * NP * 2);
      ah[j % (AHEAD + 1)][t] = lds_read16(at);
      al[j % (AHEAD + 1)][t] = lds_read16(NP * NP * 2 + at);
    }
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) fetch(j);
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    const int k = j / GROUPS, p = j % GROUPS, e = j % (AHEAD + 1);
    if (j + AHEAD < STEPS) fetch(j + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma16(al[e][t], b.hi[k], k == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : out[p * TP + t]);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma16(ah[e][t], b.lo[k], out[p * TP + t]);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma16(ah[e][t], b.hi[k], out[p * TP + t]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int NP>
__global__ void __launch_bounds__(NP * 4) __attribute__((amdgpu_waves_per_eu(2, 2)))
iter_kernel(const float* __restrict__ G0, int parts, u16* __restrict__ P0, MuonInfo* __restrict__ info, MuonSteps s) {
  constexpr int TN = NP / 16, SCR = NP * NP * 4;  // LDS: the left operand, then the waves' sums
  const int lane = (int)threadIdx.x & 63, q = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = wave * 16 + l16;
  const long long m = xcd_remap((int)blockIdx.x, (int)gridDim.x);

  f32x4 v[TN];
  const float* src = G0 + m * parts * (NP * NP) + (size_t)n * NP + 4 * q;
#pragma unroll
  for (int t = 0; t < TN; ++t) v[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int UP = NP == 128 ? 2 : 1;  // partial sums in flight at once
  for (int p = 0; p < parts; p += UP) {
    f32x4 w[UP][TN];
#pragma unroll
    for (int u = 0; u < UP; ++u)
#pragma unroll
      for (int t = 0; t < TN; ++t) w[u][t] = *(const f32x4*)(src + (size_t)min(p + u, parts - 1) * (NP * NP) + 16 * t);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < UP; ++u)
      if (p + u < parts)
#pragma unroll
        for (int t = 0; t < TN; ++t) v[t] += w[u][t];
  }
  // the lane that has element (n, n): row 4 q + i of tile `wave` is l16
  const auto diagonal = [&](int t, int i) { return t == wave && 4 * q + i == l16; };
  float d = 0.f;
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (diagonal(t, i)) d = v[t][i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  float* scr = (float*)(fmlp_lds + SCR);
  if (lane == 0) scr[wave] = d;
  __syncthreads();
  float trace = 0.f;
#pragma unroll
  for (int w = 0; w < TN; ++w) trace += scr[w];
  float inv;
  const MuonInfo fo = info_of(trace, s, s.p_scale[s.steps - 1], &inv);
  if (threadIdx.x == 0) info[m] = fo;
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[t][i] = v[t][i] * inv * inv;

  Cols<NP> G, P;
  pack_cols<NP>(v, s.g_scale[0], G);
  for (int k = 0; k < s.steps; ++k) {
    const float sg = s.g_scale[k], sq = s.q_scale[k];
    const bool last = k + 1 == s.steps;
    put_left<NP>(G, n, q);
    __syncthreads();
    product<NP>(v, G, q, l16);
    // Q = a + b G + c G^2, in G's place
    const float cc = s.c[k] / sg / sg, cb = s.b[k] / sg, ca = s.a[k];
#pragma unroll
    for (int u = 0; u < NP / 32; ++u) {
      float f[8];
      const u32x4 gh = G.hi[u], gl = G.lo[u];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = j & 1 ? hi_f32<false>(gh[j >> 1]) + hi_f32<false>(gl[j >> 1])
                              : lo_f32<false>(gh[j >> 1]) + lo_f32<false>(gl[j >> 1]);
        f[j] = __builtin_fmaf(cc, v[2 * u + (j >> 2)][j & 3], __builtin_fmaf(cb, x, diagonal(2 * u + (j >> 2), j & 3) ? ca : 0.f));
      }
      split8(f, sq, G.hi[u], G.lo[u]);
    }
    if (!last) product<NP>(v, G, q, l16);  // G Q
    __syncthreads();
    put_left<NP>(G, n, q);
    __syncthreads();
    // G Q has G's bound times Q's
    const float st = sg * sq * 0x1p-14f;
    if (k == 0) P = G;
    if (!last) pack_cols<NP>(v, st / sg / sq, G);
    if (k > 0) {
      product<NP>(v, P, q, l16);
      pack_cols<NP>(v, s.p_scale[k] / sq / s.p_scale[k - 1], P);
    }
    if (!last) {
      product<NP>(v, G, q, l16);
      pack_cols<NP>(v, s.g_scale[k + 1] / sq / st, G);
      __syncthreads();
    }
  }
  // rows 32 k + 16 h + 4 q ..: half q / 2 of unit q % 2 of 16 inner indices
  u16* dst = P0 + m * (2 * NP * NP) + muon_chunk<NP>(n, 0, q & 1) + 4 * (q >> 1);
#pragma unroll
  for (int k = 0; k < NP / 32; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *(u32x2*)(dst + (2 * k + h) * 512) = u32x2{P.hi[k][2 * h], P.hi[k][2 * h + 1]};
      *(u32x2*)(dst + NP * NP + (2 * k + h) * 512) = u32x2{P.lo[k][2 * h], P.lo[k][2 * h + 1]};
    }
}

template <int NP>
hipError_t launch_one(long long matrices, const float* G, int parts, u16* P, MuonInfo* info, const MuonSteps& s, hipStream_t st) {
  constexpr int lds = NP * NP * 4 + 64;  // (the waves' sums behind the operand)
  auto k = iter_kernel<NP>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3((unsigned)matrices), dim3(NP * 4), lds, st, G, parts, P, info, s);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// NP = 256: neither LDS nor a wave's registers hold a matrix; each product is a launch of 32 x 32 tiles, its operands from L2
// ---------------------------------------------------------------------------------------------
constexpr int N2 = 256, kMat = 2 * N2 * N2;  // fp16 values of a matrix, first terms, then second ones (muon_chunk's order)

// Workgroup b of tiles of many matrices: matrix and tile. Workgroups go to the eight XCDs in turn; a matrix stays on
// one, whose L2 then holds what the launches before wrote of it.
template <int TILES>
__device__ __forceinline__ bool place(long long matrices, long long* m, int* tile) {
  const unsigned b = blockIdx.x >> 3;
  const long long each = (matrices + 7) / 8;
  *m = (blockIdx.x & 7) * each + b / TILES;
  *tile = b % TILES;
  return *m < matrices;
}
template <int TILES>
unsigned place_blocks(long long matrices) {
  return (unsigned)((matrices + 7) / 8 * 8 * TILES);
}

// G as fp16 terms from its partial sums; a tile is 16 rows
__global__ void __launch_bounds__(256) sum256_kernel(const float* __restrict__ G0, int parts, u16* __restrict__ G,
                                                     MuonInfo* __restrict__ info, MuonSteps s, long long matrices) {
  __shared__ float scr[4];
  long long m;
  int tile;
  if (!place<16>(matrices, &m, &tile)) return;
  const float* src = G0 + m * parts * (N2 * N2);
  float d = 0.f;
  f32x4 f[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) f[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* mine = src + tile * (16 * N2) + threadIdx.x * 4;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    d += src[(size_t)p * (N2 * N2) + (size_t)threadIdx.x * (N2 + 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u) f[u] += *(const f32x4*)(mine + (size_t)p * (N2 * N2) + u * 1024);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  if ((threadIdx.x & 63) == 0) scr[threadIdx.x >> 6] = d;
  __syncthreads();
  float inv;
  const MuonInfo fo = info_of((scr[0] + scr[1]) + (scr[2] + scr[3]), s, s.p_scale[s.steps - 1], &inv);
  if (threadIdx.x == 0 && tile == 0) info[m] = fo;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    // row and inner indices k .. k + 3: half of a unit
    const int row = tile * 16 + u * 4 + ((int)threadIdx.x >> 6), k = ((int)threadIdx.x & 63) * 4;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < 4 ? f[u][j] * inv * inv : 0.f;
    u32x4 hi, lo;
    split8(v, s.g_scale[0], hi, lo);
    u16* dst = G + m * kMat + muon_chunk<N2>(row, k >> 4, (k >> 2) & 1) + (k & 8) / 2;
    *(u32x2*)dst = u32x2{hi[0], hi[1]};
    *(u32x2*)(dst + N2 * N2) = u32x2{lo[0], lo[1]};
  }
}

struct Prod256 {
  const u16* a;  // matrices
  const u16* b;
  u16* out;
  float back, scale;  // 1 / (the operands' scales), the result's scale
  float ca, cb, cc, cg;  // with POLY: ca 1 + cb cg A + cc A B
};

// A's own values where a lane has a 32 x 32 tile of a product at row r, column c: column c + l32, rows r + 16 h + 4 g + {0..3, 8..11},
// which are a unit of row c + l32 (the matrices are symmetric); and what becomes of the tile. POLY: ca 1 + cb cg A + cc A B
struct Own {
  u32x4 hi[2], lo[2];
};
__device__ __forceinline__ void own256(Own& o, const Prod256& p, long long m, int r, int c, int g, int l32) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const u16* at = p.a + m * kMat + muon_chunk<N2>(c + l32, r / 16 + h, g);
    o.hi[h] = *(const u32x4*)at;
    o.lo[h] = *(const u32x4*)(at + N2 * N2);
  }
}
template <bool POLY>
__device__ __forceinline__ void finish256(const Prod256& p, const f32x16& acc, const Own& o, long long m, int r, int c, int g, int l32) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = acc[8 * h + j] * p.back;
    if constexpr (POLY) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = j & 1 ? hi_f32<false>(o.hi[h][j >> 1]) + hi_f32<false>(o.lo[h][j >> 1])
                              : lo_f32<false>(o.hi[h][j >> 1]) + lo_f32<false>(o.lo[h][j >> 1]);
        const int at_r = r + 16 * h + 4 * g + (j & 3) + (j & 4) * 2;
        f[j] = __builtin_fmaf(p.cc, f[j], __builtin_fmaf(p.cb, x * p.cg, at_r == c + l32 ? p.ca : 0.f));
      }
    }
    u32x4 hi, lo;
    split8(f, p.scale, hi, lo);
    u16* at = p.out + m * kMat + muon_chunk<N2>(c + l32, r / 16 + h, g);
    *(u32x4*)at = hi;
    *(u32x4*)(at + N2 * N2) = lo;
  }
}

// 32 x 64 tiles of out, 32 x 32 and half of the inner dimension a wave, whose loads are all in flight at once; blockIdx.y
// picks one of two independent products
template <bool POLY>
__global__ void __launch_bounds__(256) prod256_kernel(Prod256 p0, Prod256 p1, long long matrices) {
  __shared__ f32x4 half[2][4][64];
  const Prod256 p = blockIdx.y == 0 ? p0 : p1;
  const int lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, wave = (int)threadIdx.x >> 6;
  long long m;
  int tile;
  if (!place<32>(matrices, &m, &tile)) return;
  const int side = wave & 1, k0 = (wave >> 1) * (N2 / 2);
  const int r0 = (tile >> 2) * 32, c0 = (tile & 3) * 64 + side * 32;
  const u16* A = p.a + m * kMat + muon_chunk<N2>(r0 + l32, k0 / 16, g);
  const u16* B = p.b + m * kMat + muon_chunk<N2>(c0 + l32, k0 / 16, g);
  constexpr int KS = N2 / 32;
  u32x4 ah[KS], al[KS], bh[KS], bl[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    ah[k] = *(const u32x4*)(A + 512 * k);
    al[k] = *(const u32x4*)(A + N2 * N2 + 512 * k);
    bh[k] = *(const u32x4*)(B + 512 * k);
    bl[k] = *(const u32x4*)(B + N2 * N2 + 512 * k);
  }
  Own own;
  if (POLY && wave < 2) own256(own, p, m, r0, c0, g, l32);
  __builtin_amdgcn_sched_barrier(0);
  f32x16 acc = zero16();
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    acc = mfma<false>(al[k], bh[k], acc);
    acc = mfma<false>(ah[k], bl[k], acc);
    acc = mfma<false>(ah[k], bh[k], acc);
  }
  if (wave >= 2)
#pragma unroll
    for (int q = 0; q < 4; ++q) half[side][q][lane] = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (wave >= 2) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 v = half[side][q][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[4 * q + j] += v[j];
  }
  finish256<POLY>(p, acc, own, m, r0, c0, g, l32);
}

// The same in tiles of 128 x 128, 64 x 64 a wave, for many matrices: the operands go through LDS, each once for a workgroup, and
// three workgroups a CU hide each other's beginnings and ends. A step has 16 of the inner dimension, 16 runs of 1 KB, four a
// wave. 0.165 us a matrix, 610 TFLOP/s of 16-bit products (waves that load their own operands: 0.195; two workgroups a CU with a
// step more ahead: 0.17)
constexpr int kWideAhead = 3, kWideStep = 16 * 1024;
template <bool POLY>
__global__ void __launch_bounds__(256, 3) prod256_wide_kernel(Prod256 p0, Prod256 p1, long long matrices) {
  const Prod256 p = blockIdx.y == 0 ? p0 : p1;
  const int lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  long long m;
  int tile;
  if (!place<4>(matrices, &m, &tile)) return;
  const int tr = tile >> 1, tc = tile & 1, wr = wave & 1, wc = wave >> 1;
  constexpr int KS = N2 / 16, PF = kWideAhead;
  // waves 0 and 1 bring the first and second terms of A, the others B's
  const i32x4 src = make_rsrc_words((wave < 2 ? p.a : p.b) + m * kMat, kMat * 2);
  const unsigned from = (unsigned)((wave & 1) * (N2 * N2 * 2) + (wave < 2 ? tr : tc) * (4 * KS * 1024) + lane * 16);
  const auto bring = [&](int k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) buf_load16_lds(src, from + (unsigned)((j * KS + k) * 1024), k % PF * kWideStep + (wave * 4 + j) * 1024);
  };
  Own own[4];  // (before the runs, whose waits count what comes behind them)
  if constexpr (POLY) {
#pragma unroll
    for (int i = 0; i < 4; ++i) own256(own[i], p, m, tr * 128 + wr * 64 + 32 * (i >> 1), tc * 128 + wc * 64 + 32 * (i & 1), g, l32);
  }
#pragma unroll
  for (int k = 0; k < PF - 1; ++k) bring(k);
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = zero16();
  static_for<KS>([&](auto step) {
    constexpr int k = decltype(step)::value;
    wait_vmcnt<4 * (KS - 1 - k < PF - 2 ? KS - 1 - k : PF - 2)>();  // this wave's runs of step k
    __builtin_amdgcn_s_waitcnt(0xC07F);                             // lgkmcnt(0): the reads of step k - 1, whose place is taken next
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (k + PF - 1 < KS) bring(k + PF - 1);
    const int at = k % PF * kWideStep + lane * 16;
    u32x4 a[2][2], b[2][2];  // [term][block]
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[e][i] = lds_read16(at + (e * 4 + 2 * wr + i) * 1024);
        b[e][i] = lds_read16(at + (8 + e * 4 + 2 * wc + i) * 1024);
      }
#pragma unroll
    for (int e = 0; e < 3; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma<false>(a[e == 0][i], b[e == 1][j], acc[i][j]);
  });
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      finish256<POLY>(p, acc[i][j], own[2 * i + j], m, tr * 128 + wr * 64 + 32 * i, tc * 128 + wc * 64 + 32 * j, g, l32);
}

hipError_t steps_256(long long matrices, const float* G0, int parts, u16* P, MuonInfo* info, const MuonSteps& s, void* ws,
                      hipStream_t st) {
  const size_t one = (size_t)matrices * kMat;
  u16* G = (u16*)ws;
  u16 *Q = G + one, *T = Q + one, *R = T + one;
  hipLaunchKernelGGL(sum256_kernel, dim3(place_blocks<16>(matrices)), dim3(256), 0, st, G0, parts, G, info, s, matrices);
  hipError_t e = hipGetLastError();
  const auto run = [&](auto POLY, const Prod256& a, const Prod256* b) {
    constexpr bool poly = decltype(POLY)::value;
    if (e != hipSuccess) return;
    // (16 matrices 7.4 us, in the smaller tiles 5.8; 32 8.6 and 9.4; 64 13.5 and 17; two products of 16 8.5 and 10.7)
    if (matrices * (b ? 2 : 1) >= 32)
      hipLaunchKernelGGL(prod256_wide_kernel<poly>, dim3(place_blocks<4>(matrices), b ? 2 : 1), dim3(256), kWideAhead * kWideStep, st, a,
                         b ? *b : a, matrices);
    else
      hipLaunchKernelGGL(prod256_kernel<poly>, dim3(place_blocks<32>(matrices), b ? 2 : 1), dim3(256), 0, st, a, b ? *b : a, matrices);
    e = hipGetLastError();
  };
  constexpr std::true_type poly{};
  constexpr std::false_type plain{};
  // P_k, the product of the steps' polynomials so far, takes turns in R and P, the last one in P; the first step's Q is P_0
  const auto pk = [&](int k) { return (s.steps - 1 - k) % 2 == 0 ? P : R; };
  for (int k = 0; k < s.steps; ++k) {
    const float sg = s.g_scale[k], sq = s.q_scale[k];
    u16* q = k == 0 ? pk(0) : Q;
    const bool last = k + 1 == s.steps;
    run(poly, Prod256{G, G, q, 1.f / sg / sg, sq, s.a[k], s.b[k], s.c[k], 1.f / sg}, nullptr);
    Prod256 next{};
    if (k > 0) next = Prod256{q, pk(k - 1), pk(k), 1.f / sq / s.p_scale[k - 1], s.p_scale[k], 0.f, 0.f, 0.f, 0.f};
    if (last) {
      if (k > 0) run(plain, next, nullptr);
      break;
    }
    const float stt = sg * sq * 0x1p-14f;  // G Q has G's bound times Q's
    run(plain, Prod256{G, q, T, 1.f / sg / sq, stt, 0.f, 0.f, 0.f, 0.f}, k > 0 ? &next : nullptr);
    run(plain, Prod256{q, T, G, 1.f / sq / stt, s.g_scale[k + 1], 0.f, 0.f, 0.f, 0.f}, nullptr);
  }
  return e;
}

// As many matrices at once as leave all that the launches pass on in the last cache (192: 200 MB): a product of 342 at once
// takes 76 us, of 171 33
long long at_once(long long matrices) {
  const long long parts = (matrices + 191) / 192;
  return parts ? (matrices + parts - 1) / parts : 0;
}

hipError_t launch_256(long long matrices, const float* G0, int parts, u16* P, MuonInfo* info, const MuonSteps& s, void* ws,
                      hipStream_t st) {
  const long long chunk = at_once(matrices);
  for (long long m = 0; m < matrices; m += chunk) {
    const long long n = matrices - m < chunk ? matrices - m : chunk;
    const hipError_t e = steps_256(n, G0 + m * parts * (N2 * N2), parts, P + m * kMat, info + m, s, ws, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

size_t muon_iter_ws_bytes(int NP, long long matrices) {
  return NP == 256 ? (size_t)at_once(matrices) * kMat * 4 * sizeof(u16) : 0;
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

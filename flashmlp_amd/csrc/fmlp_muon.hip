// Stacks of matrices orthogonalised by Newton-Schulz products, and the optimizer's step around it, for gfx950.
//
//   m' = mu m + (1 - mu) g;  u = m' or (1 - mu) g + mu m';  X = u / (|u| + eps);  X <- q(X X^T) X, `steps` times
//   w' = w (1 - decay) - lr X
//
// The steps are taken on the Gram matrix of the smaller side n (fmlp_muon_iter.hip), so a matrix n x e is read twice
// whatever their number: once for G = u u^T, which also writes m', and once for P u, which makes u again from g and m' and
// goes straight into the weights. X X^T X ... on the matrices themselves would read and write them every step and take
// 5 (4 n n e + 2 n^3) FLOP where this takes 3 n n e + 17 n^3 (counting G as symmetric).
//
// Both passes are bound by HBM. A workgroup walks tiles of the whole small side by 8192 / n columns of the long one:
// coalesced loads of the next tile into registers while the matrix instructions work on this one's 16-bit terms in LDS.
// Terms: G of 16-bit values needs one (the products are exact); of 32-bit ones three bf16 terms, six products, whose
// error is below that of the fp32 sums, at any scale. P u takes fp16 terms, two of P and one (16-bit u) or two of u, scaled by
// powers of two: |u| is known by then.
//
// The long side is contiguous (WIDE) or the small one is (TALL): the same tile, once read along rows and once with the
// transposing LDS reads, the other way round in the second pass.
#include <algorithm>
#include <cmath>
#include <vector>

#include "fmlp_muon_device.h"

namespace fmlp {
namespace {

constexpr int kTable = 64;
struct Ref {
  const void* x;
  void* m;
  void* out;
  int R, C;
  unsigned block0, matrix0;  // the tensor's first workgroup and matrix
  float lr, keep;
  unsigned char x_io, m_io, out_io, pad;
};
struct Table {
  Ref t[kTable];
  int n;
};
static_assert(sizeof(Table) <= 3840, "kernel arguments");

__device__ __forceinline__ const Ref& tensor_of(const Table& t, unsigned b) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.t[mid].block0 <= b) lo = mid;
    else hi = mid - 1;
  }
  return t.t[lo];
}

// 8 elements of any type, as loaded and as floats
struct Raw {
  u32x4 a, b;
};
__device__ __forceinline__ void load_raw(int io, const void* base, long long i, int n, Raw& r) {
  if (io == IO_F32) {
    r.a = load_piece<IO_F32>(base, i, n);
    r.b = load_piece<IO_F32>(base, i + 4, n - 4);
  } else {
    r.a = load_piece<IO_F16>(base, i, n);  // (16 bits of any kind)
  }
}
__device__ __forceinline__ void unpack_raw(int io, const Raw& r, float (&f)[8]) {
  if (io == IO_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = __uint_as_float(r.a[j]);
      f[4 + j] = __uint_as_float(r.b[j]);
    }
  } else if (io == IO_BF16) {
    unpack_piece<IO_BF16>(r.a, f);
  } else {
    unpack_piece<IO_F16>(r.a, f);
  }
}
// rounded to the type, stored, and what was stored
__device__ __forceinline__ void store_rounded(int io, void* base, long long i, int n, float (&f)[8]) {
  if (io == IO_F32) {
    const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
    store_piece<IO_F32>(base, i, n, pack_piece<IO_F32>(lo));
    if (n > 4) store_piece<IO_F32>(base, i + 4, n - 4, pack_piece<IO_F32>(hi));
  } else if (io == IO_BF16) {
    const u32x4 v = pack_piece<IO_BF16>(f);
    store_piece<IO_BF16>(base, i, n, v);
    unpack_piece<IO_BF16>(v, f);
  } else {
    const u32x4 v = pack_piece<IO_F16>(f);
    store_piece<IO_F16>(base, i, n, v);
    unpack_piece<IO_F16>(v, f);
  }
}

template <int NP>
constexpr int kTile = NP == 256 ? 32 : 8192 / NP;  // columns of the long side

// The tile in LDS, 16-bit terms one after the other: WIDE rows of the small side ([NP][KT], units of 16 bytes swapped
// within a row so that 16 rows' units lie on all banks), TALL rows of the long side ([KT][NP], a pitch that spreads the
// transposing reads' four rows).
template <int NP, bool TALL>
struct Tile {
  static constexpr int KT = kTile<NP>;
  static constexpr int ROWS = TALL ? KT : NP, COLS = TALL ? NP : KT;
  static constexpr int UR = COLS / 8;                                            // units of a row
  static constexpr int PITCH = TALL ? NP * 2 + (NP == 32 ? 0 : 64) : KT * 2;     // bytes
  static constexpr int TERM = ROWS * PITCH;
  static constexpr int UNITS = ROWS * UR;  // 1024
  static __device__ __forceinline__ int at(int row, int u) {
    if constexpr (TALL) return row * PITCH + u * 16;
    const int f = UR >= 16 ? row & 15 : UR == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
    return row * PITCH + ((u ^ f) << 4);
  }
  // operand of 32 small indices from s0 and 16 long ones from k0: lane = small index, 8 long ones
  static __device__ __forceinline__ u32x4 by_small(int base, int s0, int k0, int lane) {
    const int g = lane >> 5, l32 = lane & 31;
    if constexpr (!TALL) return lds_read16(base + at(s0 + l32, (k0 >> 3) + g));
    const int G = lane >> 4, i16 = lane & 15;
    const int a = base + (k0 + 8 * g + (i16 >> 2)) * PITCH + (s0 + 16 * (G & 1) + 4 * (i16 & 3)) * 2;
    return cat(lds_read_tr(a), lds_read_tr(a + 4 * PITCH));
  }
  // operand of 32 long indices from l0 and 16 small ones from k0: lane = long index, 8 small ones in the order that a
  // result of the matrix instruction has rows in, and so P: 4 g + {0..3, 8..11}
  static __device__ __forceinline__ u32x4 by_long(int base, int l0, int k0, int lane) {
    const int g = lane >> 5, l32 = lane & 31;
    if constexpr (TALL) return lds_read16(base + at(l0 + l32, (k0 >> 3) + g));  // (put_by_long's order)
    // rows k0 + 4 g .., columns l0 + 16 (G & 1) ..: 8-byte halves of the swapped units
    const int G = lane >> 4, i16 = lane & 15;
    const int row = k0 + 4 * g + (i16 >> 2), col = l0 + 16 * (G & 1) + 4 * (i16 & 3);
    const int a = base + at(row, col >> 3) + (col & 4) * 2, b = base + at(row + 8, col >> 3) + (col & 4) * 2;
    return cat(lds_read_tr(a), lds_read_tr(b));
  }
  // 8 elements of unit u of a row where by_long finds them: TALL, halves of 4 in P's order
  static __device__ __forceinline__ void put_by_long(int base, int row, int u, const u32x4& v) {
    if constexpr (TALL) {
      const int to = base + at(row, u & ~1) + (u & 1) * 8;
      lds_write8(to, u32x2{v[0], v[1]});
      lds_write8(to + 16, u32x2{v[2], v[3]});
    } else {
      lds_write16(base + at(row, u), v);
    }
  }
};

// a thread's unit q of a tile from long index l0: its row, the first of its 8 columns, the element in the matrix, and how many
// of the 8 are there
template <int NP, bool TALL, int THREADS>
struct Piece {
  int row, u, n;
  long long i;
  __device__ __forceinline__ Piece(int q, long long l0, int R, int C) {
    using T = Tile<NP, TALL>;
    const int id = q * THREADS + (int)threadIdx.x;
    row = id / T::UR;
    u = id % T::UR;
    const long long r = TALL ? l0 + row : row, c = TALL ? u * 8 : l0 + u * 8;
    n = r < R ? (int)min(8LL, C - c) : 0;
    i = r * C + c;
  }
};

template <int TERMS, bool BF>
__device__ __forceinline__ f32x16 mfma_terms(const u32x4 (&a)[TERMS], const u32x4 (&b)[TERMS], f32x16 c) {
  if constexpr (TERMS == 3) {
    c = mfma<BF>(a[2], b[0], c);
    c = mfma<BF>(a[0], b[2], c);
    c = mfma<BF>(a[1], b[1], c);
    c = mfma<BF>(a[1], b[0], c);
    c = mfma<BF>(a[0], b[1], c);
  }
  return mfma<BF>(a[0], b[0], c);
}

// three bf16 terms of 8 values
__device__ __forceinline__ void split3(const float (&f)[8], u32x4 (&t)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = f[2 * j], b = f[2 * j + 1];
    t[0][j] = pack2<true>(a, b);
    a -= lo_f32<true>(t[0][j]);
    b -= hi_f32<true>(t[0][j]);
    t[1][j] = pack2<true>(a, b);
    a -= lo_f32<true>(t[1][j]);
    b -= hi_f32<true>(t[1][j]);
    t[2][j] = pack2<true>(a, b);
  }
}

// Gram matrices: `parts` workgroups a matrix, each a range of the long side, their partial sums whole and symmetric.
// TERMS 1: x as it is (BF its type); 3: u in fp32, from x and m.
template <int NP, bool TALL, int TERMS, bool BF>
__global__ void __launch_bounds__(256) gram_kernel(Table tab, float* __restrict__ G, int parts, float mu, float nu, int nesterov) {
  using T = Tile<NP, TALL>;
  constexpr int KT = T::KT, RB = NP / 32, PAIRS = RB * (RB + 1) / 2;
  constexpr int KQ = NP <= 64 ? 4 : 1;                   // waves that share the long side's 16s of a tile
  constexpr int MP = KQ == 4 ? PAIRS : (PAIRS + 3) / 4;  // tile pairs of a wave
  constexpr int Q = T::UNITS / 256;
  const Ref& t = tensor_of(tab, blockIdx.x);
  const unsigned local = blockIdx.x - t.block0;
  const long long h = local / (unsigned)parts;
  const int part = (int)(local % (unsigned)parts);
  const int R = t.R, C = t.C;
  const long long L = TALL ? R : C, tiles = (L + KT - 1) / KT, per = (tiles + parts - 1) / parts;
  const long long t0 = part * per, t1 = min(tiles, t0 + per);
  const size_t es_x = t.x_io == IO_F32 ? 4 : 2, es_m = t.m_io == IO_F32 ? 4 : 2;
  const char* X = (const char*)t.x + (size_t)h * R * C * es_x;
  char* M = t.m ? (char*)t.m + (size_t)h * R * C * es_m : nullptr;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

  // the wave's pairs of 32-row blocks, i <= j
  int pi[MP], pj[MP];
  f32x16 acc[MP];
#pragma unroll
  for (int p = 0; p < MP; ++p) {
    int id = KQ == 4 ? p : min(p * 4 + wave, PAIRS - 1), i = 0;
    while (id >= RB - i) {
      id -= RB - i;
      ++i;
    }
    pi[p] = i;
    pj[p] = i + id;
    acc[p] = zero16();
  }

  Raw x[Q], m[TERMS == 3 ? Q : 1];
  const auto load = [&](long long tile) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, 256> at(q, tile * KT, R, C);
      if constexpr (TERMS == 3) {
        load_raw(t.x_io, X, at.i, at.n, x[q]);
        if (M) load_raw(t.m_io, M, at.i, at.n, m[q]);
      } else {
        x[q].a = load_piece<IO_F16>(X, at.i, at.n);
      }
    }
  };
  const auto put = [&](long long tile) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, 256> at(q, tile * KT, R, C);
      const int o = T::at(at.row, at.u);
      if constexpr (TERMS == 3) {
        float f[8];
        unpack_raw(t.x_io, x[q], f);
        if (M) {
          float v[8];
          unpack_raw(t.m_io, m[q], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(mu, v[j], nu * f[j]);
          store_rounded(t.m_io, M, at.i, at.n, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = nesterov ? __builtin_fmaf(mu, v[j], nu * f[j]) : v[j];
        }
        u32x4 s[3];
        split3(f, s);
#pragma unroll
        for (int k = 0; k < 3; ++k) lds_write16(k * T::TERM + o, s[k]);
      } else {
        lds_write16(o, x[q].a);
      }
    }
  };

  if (t0 < t1) load(t0);
  for (long long tile = t0; tile < t1; ++tile) {
    put(tile);
    __syncthreads();
    if (tile + 1 < t1) load(tile + 1);
#pragma unroll
    for (int k = 0; k < KT / 16 / KQ; ++k) {
      const int k0 = 16 * (KQ == 4 ? k * 4 + wave : k);
#pragma unroll
      for (int p = 0; p < MP; ++p) {
        u32x4 a[TERMS], b[TERMS];
#pragma unroll
        for (int e = 0; e < TERMS; ++e) {
          a[e] = T::by_small(e * T::TERM, pi[p] * 32, k0, lane);
          b[e] = T::by_small(e * T::TERM, pj[p] * 32, k0, lane);
        }
        acc[p] = mfma_terms<TERMS, BF>(a, b, acc[p]);
      }
    }
    __syncthreads();
  }

  if constexpr (KQ == 4) {
    // the four waves' sums, in order
    float* scr = (float*)fmlp_lds;
    static_assert(3 * MP * 4096 <= 3 * 8192 * 2, "the sums fit a tile's three terms");
    if (wave > 0)
#pragma unroll
      for (int p = 0; p < MP; ++p)
#pragma unroll
        for (int i = 0; i < 16; ++i) scr[(((wave - 1) * MP + p) * 16 + i) * 64 + lane] = acc[p][i];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int p = 0; p < MP; ++p)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[p][i] += scr[((w * MP + p) * 16 + i) * 64 + lane];
  }
  float* dst = G + ((size_t)(t.matrix0 + h) * parts + part) * (NP * NP);
  const int g = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int p = 0; p < MP; ++p) {
    if (KQ == 1 && p * 4 + wave >= PAIRS) continue;
    const int c = pj[p] * 32 + l32, r = pi[p] * 32 + 4 * g;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *(float4*)(dst + (size_t)c * NP + r + 8 * q) = float4{acc[p][4 * q], acc[p][4 * q + 1], acc[p][4 * q + 2], acc[p][4 * q + 3]};
      if (pi[p] != pj[p])
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[(size_t)(r + 8 * q + j) * NP + c] = acc[p][4 * q + j];
    }
  }
}

// O = P u, and what becomes of it. XT: terms of u. Waves: a block of 32 small indices and CT of 32 long ones each.
template <int NP, bool TALL, int XT>
__global__ void __launch_bounds__(NP == 256 ? 512 : 256)
apply_kernel(Table tab, const u16* __restrict__ P, const MuonInfo* __restrict__ info, int parts, float mu, float nu, int nesterov,
             int update) {
  using T = Tile<NP, TALL>;
  constexpr int THREADS = NP == 256 ? 512 : 256;
  constexpr int KT = T::KT, RB = NP / 32, CT = NP == 256 ? 1 : 2, KS = NP / 16, Q = T::UNITS / THREADS;
  constexpr int OPITCH = T::COLS + 4;  // floats between the result's rows in LDS
  const Ref& t = tensor_of(tab, blockIdx.x);
  const unsigned local = blockIdx.x - t.block0;
  const long long h = local / (unsigned)parts;
  const int part = (int)(local % (unsigned)parts);
  const int R = t.R, C = t.C;
  const long long L = TALL ? R : C, tiles = (L + KT - 1) / KT, per = (tiles + parts - 1) / parts;
  const long long t0 = part * per, t1 = min(tiles, t0 + per);
  if (t0 >= t1) return;
  const size_t es_x = t.x_io == IO_F32 ? 4 : 2, es_m = t.m_io == IO_F32 ? 4 : 2, es_o = t.out_io == IO_F32 ? 4 : 2;
  const char* X = (const char*)t.x + (size_t)h * R * C * es_x;
  const char* M = t.m ? (const char*)t.m + (size_t)h * R * C * es_m : nullptr;
  char* O = (char*)t.out + (size_t)h * R * C * es_o;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  const int s0 = (wave % RB) * 32, c0 = wave / RB * CT * 32;
  const MuonInfo fo = info[t.matrix0 + h];

  // the wave's rows of P
  u32x4 ph[KS], pl[KS];
  const u16* src = P + (size_t)(t.matrix0 + h) * (2 * NP * NP) + muon_chunk<NP>(s0 + l32, 0, g);
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    ph[k] = *(const u32x4*)(src + 512 * k);
    pl[k] = *(const u32x4*)(src + NP * NP + 512 * k);
  }

  Raw x[Q], m[Q], w[Q];
  const auto load = [&](long long tile) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
      load_raw(t.x_io, X, at.i, at.n, x[q]);
      if (M) load_raw(t.m_io, M, at.i, at.n, m[q]);
    }
  };
  float* res = (float*)fmlp_lds;  // the result takes the tile's place
  load(t0);
  for (long long tile = t0; tile < t1; ++tile) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
      float f[8];
      unpack_raw(t.x_io, x[q], f);
      if (M) {
        float v[8];
        unpack_raw(t.m_io, m[q], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = nesterov ? __builtin_fmaf(mu, v[j], nu * f[j]) : v[j];
      }
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = f[2 * j] * fo.u_scale, b = f[2 * j + 1] * fo.u_scale;
        hi[j] = pack2<false>(a, b);
        if constexpr (XT == 2) lo[j] = pack2<false>(a - lo_f32<false>(hi[j]), b - hi_f32<false>(hi[j]));
      }
      T::put_by_long(0, at.row, at.u, hi);
      if constexpr (XT == 2) T::put_by_long(T::TERM, at.row, at.u, lo);
    }
    __syncthreads();
    if (update) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
        load_raw(t.out_io, O, at.i, at.n, w[q]);
      }
    }
    if (tile + 1 < t1) load(tile + 1);
    f32x16 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = zero16();
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const u32x4 xh = T::by_long(0, c0 + c * 32, 16 * k, lane);
        // (WIDE: rows of the result are the small side; TALL: the long one. Lanes are the other, contiguous in memory)
        const auto one = [&](const u32x4& p, const u32x4& v) { acc[c] = TALL ? mfma<false>(v, p, acc[c]) : mfma<false>(p, v, acc[c]); };
        if constexpr (XT == 2) one(ph[k], T::by_long(T::TERM, c0 + c * 32, 16 * k, lane));
        one(pl[k], xh);
        one(ph[k], xh);
      }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i >> 2) + 4 * g + (i & 3);
        const int row = TALL ? c0 + c * 32 + r : s0 + r, col = TALL ? s0 + l32 : c0 + c * 32 + l32;
        res[row * OPITCH + col] = acc[c][i] * fo.factor;
      }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 v = *(const float4*)(res + at.row * OPITCH + at.u * 8 + j);
        f[j] = v.x;
        f[j + 1] = v.y;
        f[j + 2] = v.z;
        f[j + 3] = v.w;
      }
      if (update) {
        float v[8];
        unpack_raw(t.out_io, w[q], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __builtin_fmaf(-t.lr, f[j], v[j] * t.keep);
      }
      store_rounded(t.out_io, O, at.i, at.n, f);
    }
    __syncthreads();
  }
}

template <int NP, bool TALL, int TERMS, bool BF>
hipError_t run_gram(const Table& tab, unsigned blocks, float* G, int parts, const MuonCall& c, hipStream_t st) {
  using T = Tile<NP, TALL>;
  constexpr int lds = std::max(TERMS * T::TERM, NP <= 64 ? 3 * NP / 32 * (NP / 32 + 1) / 2 * 4096 : 0);
  auto k = gram_kernel<NP, TALL, TERMS, BF>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(blocks), dim3(256), lds, st, tab, G, parts, c.mu, c.nu, c.nesterov);
  return hipGetLastError();
}
template <int NP, bool TALL, int XT>
hipError_t run_apply(const Table& tab, unsigned blocks, const u16* P, const MuonInfo* info, int parts, const MuonCall& c,
                     int update, hipStream_t st) {
  using T = Tile<NP, TALL>;
  constexpr int lds = std::max(XT * T::TERM, T::ROWS * (T::COLS + 4) * 4);
  auto k = apply_kernel<NP, TALL, XT>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(blocks), dim3(NP == 256 ? 512 : 256), lds, st, tab, P, info, parts, c.mu, c.nu, c.nesterov, update);
  return hipGetLastError();
}

// f(NP, TALL) as constants
template <typename F>
hipError_t by_shape(int NP, bool tall, F f) {
  const auto t = [&](auto n) { return tall ? f(n, std::true_type{}) : f(n, std::false_type{}); };
  switch (NP) {
    case 32: return t(std::integral_constant<int, 32>{});
    case 64: return t(std::integral_constant<int, 64>{});
    case 128: return t(std::integral_constant<int, 128>{});
    default: return t(std::integral_constant<int, 256>{});
  }
}

int padded(const MuonTensor& t) {
  const int n = std::min(t.R, t.C);
  return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256;
}
// what decides a tensor's kernels: padded small side, orientation, the terms and type of its Gram matrix
struct Kind {
  int NP;
  bool tall;
  int terms;  // 1: 16-bit values as they are
  bool bf;
  bool operator==(const Kind& o) const { return NP == o.NP && tall == o.tall && terms == o.terms && bf == o.bf; }
};
Kind kind_of(const MuonTensor& t) {
  const bool raw = t.m == nullptr && t.x_io != IO_F32;
  return Kind{padded(t), t.R > t.C, raw ? 1 : 3, !raw || t.x_io == IO_BF16};
}

// The matrices of one padded size: their Gram matrices and what comes of them go through the workspace together.
struct Group {
  int NP;
  long long matrices, tiles;  // tiles: of the longest one
  int gram_parts, apply_parts;
  size_t g_off, p_off, info_off, iter_off, end;
};
Group group_of(int NP, int n, const MuonTensor* t, int cus) {
  Group r{};
  r.NP = NP;
  const int KT = NP == 256 ? 32 : 8192 / NP;
  for (int i = 0; i < n; ++i)
    if (t[i].H > 0 && t[i].R > 0 && t[i].C > 0 && padded(t[i]) == NP) {
      r.matrices += t[i].H;
      r.tiles = std::max(r.tiles, ((long long)std::max(t[i].R, t[i].C) + KT - 1) / KT);
    }
  if (r.matrices == 0) return r;
  // three workgroups a CU at least, as far as there are tiles; of Gram matrices no more than pay: a tile takes about
  // 2.5 us, a part's sums are written and read at about 4 TB/s (8 matrices of 256 x 1024: 32 parts 18 + 46 us, 9 PARTS9)
  const long long want = (3LL * cus + r.matrices - 1) / r.matrices;
  const double part_us = (double)r.matrices * NP * NP * 8 / 4e6;
  const long long pays = std::max(1LL, std::llround(std::sqrt((double)r.tiles * 2.5 / part_us)));
  r.gram_parts = (int)std::max(1LL, std::min(std::min(want, pays), r.tiles));
  r.apply_parts = (int)std::max(1LL, std::min(want, r.tiles));
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  r.p_off = up((size_t)r.matrices * r.gram_parts * NP * NP * 4);
  r.info_off = r.p_off + up((size_t)r.matrices * NP * NP * 4);
  r.iter_off = r.info_off + up((size_t)r.matrices * sizeof(MuonInfo));
  r.end = r.iter_off + up(muon_iter_ws_bytes(NP, r.matrices));
  return r;
}
constexpr int kSizes[4] = {32, 64, 128, 256};

// Powers of two that bring each stage's values to at most 2^14 as fp16: bounds of the eigenvalues of G, Q and P from
// the steps' polynomials over the range that G's have, which is [0, 1] at first. Returns the range after the steps.
double set_steps(MuonSteps* s, const MuonCall& c, int first, int steps, bool normalise, double range) {
  s->steps = steps;
  s->normalise = normalise;
  s->eps = c.eps;
  double p = 1;
  const auto scale = [](double bound) {
    int e = 0;
    if (!(bound < 1e30)) bound = 1e30;
    (void)std::frexp(std::max(bound, 1e-30), &e);
    return std::ldexp(1.f, 14 - e);
  };
  for (int k = 0; k < steps; ++k) {
    const float* v = c.abc[first + k];
    s->a[k] = v[0];
    s->b[k] = v[1];
    s->c[k] = v[2];
    double q = 0, next = 0;
    const int N = 512;
    for (int i = 0; i <= N; ++i) {
      const double l = range * 1.02 * i / N, y = v[0] + l * (v[1] + l * v[2]);
      q = std::max(q, std::fabs(y));
      next = std::max(next, l * y * y);
    }
    q *= 1.02;
    p *= q;
    s->g_scale[k] = scale(range * 1.02);
    s->q_scale[k] = scale(q);
    s->p_scale[k] = scale(p);
    range = next * 1.02;
  }
  return range;
}

struct Pass {
  const void* x;
  void* m;
  void* out;
  int x_io, m_io, out_io, update;
};

}  // namespace

MuonPlan muon_plan(int n, const MuonTensor* t, const MuonCall& c, int num_cus) {
  MuonPlan p{};
  for (int NP : kSizes) {
    const Group g = group_of(NP, n, t, num_cus);
    if (g.matrices) p.ws_bytes = std::max(p.ws_bytes, g.end);
  }
  // more steps than a Gram matrix serves: the matrices between the stages in fp32, in the result where that is fp32
  size_t between = 0;
  if (c.steps > c.stage)
    for (int i = 0; i < n; ++i)
      if (c.update || t[i].out_io != IO_F32) between += ((size_t)t[i].H * t[i].R * t[i].C * 4 + 255) / 256 * 256;
  p.ws_bytes += between;
  return p;
}

hipError_t launch_muon(int n, const MuonTensor* t, const MuonCall& c, int num_cus, void* ws, hipStream_t st) {
  size_t shared = 0;
  for (int NP : kSizes) {
    const Group g = group_of(NP, n, t, num_cus);
    if (g.matrices) shared = std::max(shared, g.end);
  }
  char* between0 = (char*)ws + shared;
  for (int NP : kSizes) {
    const Group gr = group_of(NP, n, t, num_cus);
    if (gr.matrices == 0) continue;
    float* G = (float*)ws;
    u16* P = (u16*)((char*)ws + gr.p_off);
    MuonInfo* info = (MuonInfo*)((char*)ws + gr.info_off);
    double range = 1;
    for (int first = 0; first < c.steps; first += c.stage) {
      const int steps = std::min(c.stage, c.steps - first);
      const bool start = first == 0, last = first + steps == c.steps;
      MuonSteps s{};
      range = set_steps(&s, c, first, steps, start, range);
      const auto pass_of = [&](int i, char* y) {
        Pass p{t[i].x, t[i].m, t[i].out, t[i].x_io, t[i].m_io, t[i].out_io, c.update};
        const bool own = !c.update && t[i].out_io == IO_F32;  // the result holds what is between the stages
        void* b = own ? t[i].out : (void*)y;
        if (!start) p = Pass{b, nullptr, p.out, IO_F32, 0, p.out_io, p.update};
        if (!last) {
          p.out = b;
          p.out_io = IO_F32;
          p.update = 0;
        }
        return p;
      };
      // f(kind, table, workgroups, update) for tables of tensors of one kind
      const auto tables = [&](int parts, bool gram, auto f) -> hipError_t {
        std::vector<Kind> done;
        for (int a = 0; a < n; ++a) {
          if (t[a].H == 0 || t[a].R == 0 || t[a].C == 0 || padded(t[a]) != NP) continue;
          const auto kind_at = [&](int i) {
            MuonTensor u = t[i];
            if (!start) {
              u.m = nullptr;
              u.x_io = IO_F32;
            }
            return kind_of(u);
          };
          const Kind k = kind_at(a);
          if (std::find(done.begin(), done.end(), k) != done.end()) continue;
          done.push_back(k);
          Table tab{};
          long long blocks = 0, matrix = 0;
          char* y = between0;
          const auto flush = [&]() -> hipError_t {
            const hipError_t e = tab.n ? f(k, tab, (unsigned)blocks) : hipSuccess;
            tab.n = 0;
            blocks = 0;
            return e;
          };
          for (int i = 0; i < n; ++i) {
            char* mine = y;
            if (c.steps > c.stage && (c.update || t[i].out_io != IO_F32)) y += ((size_t)t[i].H * t[i].R * t[i].C * 4 + 255) / 256 * 256;
            if (t[i].H == 0 || t[i].R == 0 || t[i].C == 0 || padded(t[i]) != NP) continue;
            const long long first_matrix = matrix;
            matrix += t[i].H;
            if (i < a || !(kind_at(i) == k)) continue;
            const long long b = t[i].H * parts;
            if (b > 0x7fffffffLL) return hipErrorInvalidValue;
            if (tab.n == kTable || blocks + b > 0x7fffffffLL) {
              const hipError_t e = flush();
              if (e != hipSuccess) return e;
            }
            const Pass p = pass_of(i, mine);
            Ref& r = tab.t[tab.n++];
            r = Ref{p.x, p.m, p.out, t[i].R, t[i].C, (unsigned)blocks, (unsigned)first_matrix, t[i].lr, t[i].keep,
                    (unsigned char)p.x_io, (unsigned char)p.m_io, (unsigned char)p.out_io, 0};
            blocks += b;
          }
          const hipError_t e = flush();
          if (e != hipSuccess) return e;
        }
        (void)gram;
        return hipSuccess;
      };
      hipError_t e = tables(gr.gram_parts, true, [&](const Kind& k, const Table& tab, unsigned blocks) {
        return by_shape(NP, k.tall, [&](auto np, auto tall) {
          constexpr int N = decltype(np)::value;
          constexpr bool L = decltype(tall)::value;
          if (k.terms == 3) return run_gram<N, L, 3, true>(tab, blocks, G, gr.gram_parts, c, st);
          return k.bf ? run_gram<N, L, 1, true>(tab, blocks, G, gr.gram_parts, c, st)
                      : run_gram<N, L, 1, false>(tab, blocks, G, gr.gram_parts, c, st);
        });
      });
      if (e == hipSuccess) e = launch_muon_iter(NP, gr.matrices, G, gr.gram_parts, P, info, s, (char*)ws + gr.iter_off, st);
      if (e == hipSuccess)
        e = tables(gr.apply_parts, false, [&](const Kind& k, const Table& tab, unsigned blocks) {
          return by_shape(NP, k.tall, [&](auto np, auto tall) {
            constexpr int N = decltype(np)::value;
            constexpr bool L = decltype(tall)::value;
            const int update = c.update && last;
            return k.terms == 3 ? run_apply<N, L, 2>(tab, blocks, P, info, gr.apply_parts, c, update, st)
                                : run_apply<N, L, 1>(tab, blocks, P, info, gr.apply_parts, c, update, st);
          });
        });
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

}  // namespace fmlp

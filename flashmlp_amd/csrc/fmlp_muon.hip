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
// Measured: 2304 matrices of 128 x 1024 (302 M fp32 weights and momenta, bf16 gradients) 1.75 ms, 24 bytes an element at 4.1 TB/s
// where a copy reaches 5.2; matrix instructions 31 % and vector ones 37 % of the SIMDs' cycles, which the steps and the
// terms take beside the stream. One step instead of five: 4.5 TB/s. Three matrices of 12 x 64 x 768: 35 us in three launches, half
// of it the steps' chain. Tried and not kept: the second pass from the last tile on (512 matrices 447 -> 428 us, 1536 1222 ->
// 1238), half of the first round's workgroups started later (no change).
//
// The long side is contiguous (WIDE) or the small one is (TALL): the same tile, once read along rows and once with the
// transposing LDS reads, the other way round in the second pass.
#include <algorithm>
#include <type_traits>

#include "fmlp_muon_device.h"

namespace fmlp {
namespace {

__device__ __forceinline__ const MuonRef& tensor_of(const MuonTable& t, unsigned b) {
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
// rounded to the type
__device__ __forceinline__ void pack_raw(int io, const float (&f)[8], Raw& r) {
  if (io == IO_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.a[j] = __float_as_uint(f[j]);
      r.b[j] = __float_as_uint(f[4 + j]);
    }
  } else if (io == IO_BF16) {
    r.a = pack_piece<IO_BF16>(f);
  } else {
    r.a = pack_piece<IO_F16>(f);
  }
}

// A matrix in memory, or none. VEC: rows of whole 16-byte vectors, less than 2^31 bytes: 8 elements are there or not, and loads
// and stores are the same instructions for every type and place (what is not there is an offset beyond the buffer's end).
// Branches around them have the compiler wait for each load where the paths join again: 302 M weights in matrices of 128 x 1024
// 2114 us so, 1877 with these.
template <bool VEC>
struct Mat;
template <>
struct Mat<true> {
  Rsrc r;
  int io;
  __device__ __forceinline__ Mat(const void* stack, int type, long long h, int R, int C) : io(type) {
    const int bytes = R * C * (io == IO_F32 ? 4 : 2);
    r = make_rsrc((const char*)stack + (stack ? (size_t)h * bytes : 0), stack ? bytes : 0);
  }
  __device__ __forceinline__ unsigned offset(long long i, int n) const { return n > 0 ? (unsigned)i << (io == IO_F32 ? 2 : 1) : BUF_OOB; }
  __device__ __forceinline__ void load(long long i, int n, Raw& v) const {
    const unsigned o = offset(i, n);
    v.a = buf_load16(r, o);
    v.b = buf_load16(r, io == IO_F32 ? o + 16 : BUF_OOB);
  }
  __device__ __forceinline__ u32x4 load16(long long i, int n) const { return buf_load16(r, n > 0 ? (unsigned)i << 1 : BUF_OOB); }
  __device__ __forceinline__ void store(long long i, int n, const Raw& v) const {
    const unsigned o = offset(i, n);
    __builtin_amdgcn_raw_buffer_store_b128(v.a, r, (int)o, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(v.b, r, (int)(io == IO_F32 ? o + 16 : BUF_OOB), 0, 0);
  }
};
template <>
struct Mat<false> {
  char* base;
  int io;
  __device__ __forceinline__ Mat(const void* stack, int type, long long h, int R, int C)
      : base(stack ? (char*)stack + (size_t)h * R * C * (type == IO_F32 ? 4 : 2) : nullptr), io(type) {}
  __device__ __forceinline__ void load(long long i, int n, Raw& v) const {
    if (base == nullptr) return;
    if (io == IO_F32) {
      v.a = load_piece<IO_F32>(base, i, n);
      v.b = load_piece<IO_F32>(base, i + 4, n - 4);
    } else {
      v.a = load_piece<IO_F16>(base, i, n);  // (16 bits of any kind)
    }
  }
  __device__ __forceinline__ u32x4 load16(long long i, int n) const { return load_piece<IO_F16>(base, i, n); }
  __device__ __forceinline__ void store(long long i, int n, const Raw& v) const {
    if (io == IO_F32) {
      store_piece<IO_F32>(base, i, n, v.a);
      store_piece<IO_F32>(base, i + 4, n - 4, v.b);
    } else {
      store_piece<IO_F16>(base, i, n, v.a);
    }
  }
};

template <int NP>
constexpr int kTile = NP == 256 ? 32 : 8192 / NP;  // columns of the long side

// The tile in LDS, 16-bit terms one after the other: WIDE rows of the small side ([NP][KT], units of 16 bytes swapped
// within a row so that 16 rows' units lie on all banks), TALL rows of the long side ([KT][NP], a pitch that spreads the
// transposing reads' four rows).
template <int NP, bool TALL, int KT_ = kTile<NP>>
struct Tile {
  static constexpr int KT = KT_;
  static constexpr int ROWS = TALL ? KT : NP, COLS = TALL ? NP : KT;
  static constexpr int UR = COLS / 8;                                            // units of a row
  static constexpr int PITCH = TALL ? NP * 2 + (NP == 32 ? 0 : 64) : KT * 2;     // bytes
  static constexpr int TERM = ROWS * PITCH;
  static constexpr int UNITS = ROWS * UR;
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

// A workgroup's matrix, and the tiles of it that are its own.
struct Part {
  long long h, t0, t1;
  int part;
};
template <int NP, bool TALL>
__device__ __forceinline__ Part part_of(const MuonRef& t, int parts, unsigned block) {
  const unsigned local = block - t.block0;
  Part p;
  p.h = local / (unsigned)parts;
  p.part = (int)(local % (unsigned)parts);
  const long long L = TALL ? t.R : t.C, tiles = (L + kTile<NP> - 1) / kTile<NP>, per = (tiles + parts - 1) / parts;
  p.t0 = p.part * per;
  p.t1 = min(tiles, p.t0 + per);
  return p;
}
// The 32 x 32 tiles i <= j of a Gram matrix among a workgroup's waves, so that each reads few operands for its tiles.
//   NP = 256, eight waves: rows i0 = wave / 2 and 7 - i0 have nine tiles; one wave takes i0's first five, the other the rest.
//   NP = 128, four waves: rows i0 = wave / 2 and 3 - i0 have five; the two waves that have them share the long side's 16s.
//   Below, every wave has all tiles and a quarter of the 16s.
template <int NP>
struct Pairs {
  static constexpr int WAVES = NP == 256 ? 8 : 4, RB = NP / 32, KQ = NP == 256 ? 1 : NP == 128 ? 2 : 4;
  static constexpr int MP = NP == 256 ? 5 : NP == 128 ? 6 : RB * (RB + 1) / 2;  // sums (128: row i0's by column, then the other's from 2 on)
  // tile p of the wave: row, column, whether it has it
  static __device__ __forceinline__ int i0(int wave) { return wave / 2; }
  static __device__ __forceinline__ int kq(int wave) { return wave % KQ; }
  static __device__ __forceinline__ int row(int p, int wave) {
    if constexpr (NP == 256) return (wave & 1) == 0 || p < 3 - i0(wave) ? i0(wave) : 7 - i0(wave);
    else if constexpr (NP == 128) return p < RB ? i0(wave) : RB - 1 - i0(wave);
    else return p < RB ? 0 : 1;
  }
  static __device__ __forceinline__ int col(int p, int wave) {
    if constexpr (NP == 256) return (wave & 1) == 0 ? i0(wave) + p : p < 3 - i0(wave) ? i0(wave) + 5 + p : 4 + p;
    else return p < RB ? p : p - RB + RB / 2;
  }
  static __device__ __forceinline__ bool has(int p, int wave) {
    if constexpr (NP == 256) return (wave & 1) == 0 || p < 4;
    else return col(p, wave) >= row(p, wave);
  }
};

// The wave's tiles of G over the data tiles [t0, t1), and with a momentum m' on the way. With KQ = 4 the sums are wave
// 0's. TERMS 1: x as it is (BF its type); 3: u in fp32, from x and m.
template <int NP, bool TALL, int TERMS, bool BF, bool VEC>
__device__ __forceinline__ void gram_tiles(f32x16 (&acc)[Pairs<NP>::MP], const MuonRef& t, const Part& part, float mu, float nu,
                                           int nesterov, int wave) {
  using T = Tile<NP, TALL>;
  constexpr int THREADS = Pairs<NP>::WAVES * 64, KT = T::KT, KQ = Pairs<NP>::KQ, MP = Pairs<NP>::MP, Q = T::UNITS / THREADS;
  const int R = t.R, C = t.C, lane = (int)threadIdx.x & 63;
  const long long t0 = part.t0, t1 = part.t1;
  const Mat<VEC> X(t.x, t.x_io, part.h, R, C), M(t.m, t.m_io, part.h, R, C);
  const bool momentum = t.m != nullptr;
#pragma unroll
  for (int p = 0; p < MP; ++p) acc[p] = zero16();

  Raw x[Q], m[TERMS == 3 ? Q : 1];
  const auto load = [&](long long tile, int q) {
    const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
    if constexpr (TERMS == 3) {
      X.load(at.i, at.n, x[q]);
      M.load(at.i, at.n, m[q]);
    } else {
      x[q].a = X.load16(at.i, at.n);
    }
  };
  const auto put = [&](long long tile, int q) {
    const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
    const int o = T::at(at.row, at.u);
    if constexpr (TERMS == 3) {
      float f[8];
      unpack_raw(X.io, x[q], f);
      if (momentum) {
        float v[8];
        unpack_raw(M.io, m[q], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(mu, v[j], nu * f[j]);
        pack_raw(M.io, v, m[q]);
        M.store(at.i, at.n, m[q]);
        unpack_raw(M.io, m[q], v);  // (as it is stored)
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
  };

  if (t0 < t1)
#pragma unroll
    for (int q = 0; q < Q; ++q) load(t0, q);
  using PR = Pairs<NP>;
  for (long long tile = t0; tile < t1; ++tile) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {  // the next tile's loads go out as soon as their registers are free
      put(tile, q);
      if (tile + 1 < t1) load(tile + 1, q);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KT / 16 / KQ; ++k) {
      const int k0 = 16 * (k * KQ + PR::kq(wave));
      const auto fetch = [&](int block, u32x4 (&v)[TERMS]) {
#pragma unroll
        for (int e = 0; e < TERMS; ++e) v[e] = T::by_small(e * T::TERM, block * 32, k0, lane);
      };
      if constexpr (NP == 256) {
        u32x4 a[TERMS], b[TERMS];
        fetch(PR::row(0, wave), a);
#pragma unroll
        for (int p = 0; p < MP; ++p) {
          if (!PR::has(p, wave)) continue;
          if (p > 0 && PR::row(p, wave) != PR::row(p - 1, wave)) fetch(PR::row(p, wave), a);
          fetch(PR::col(p, wave), b);
          acc[p] = mfma_terms<TERMS, BF>(a, b, acc[p]);
        }
      } else if constexpr (NP == 128) {
        u32x4 a[TERMS], c[TERMS];
        fetch(PR::i0(wave), a);
        fetch(PR::RB - 1 - PR::i0(wave), c);
#pragma unroll
        for (int j = 0; j < PR::RB; ++j) {
          if (j < PR::i0(wave)) continue;
          u32x4 b[TERMS];
          fetch(j, b);
          acc[j] = mfma_terms<TERMS, BF>(a, b, acc[j]);
          if (j >= PR::RB / 2)
            if (j >= PR::RB - 1 - PR::i0(wave)) acc[PR::RB / 2 + j] = mfma_terms<TERMS, BF>(c, b, acc[PR::RB / 2 + j]);
        }
      } else {
        u32x4 b[PR::RB][TERMS];
#pragma unroll
        for (int j = 0; j < PR::RB; ++j) fetch(j, b[j]);
#pragma unroll
        for (int p = 0; p < MP; ++p) acc[p] = mfma_terms<TERMS, BF>(b[PR::row(p, 0)], b[p < PR::RB ? p : 1], acc[p]);
      }
    }
    __syncthreads();
  }

  if constexpr (KQ > 1) {
    // the sums of the waves that shared, in order: the first one's
    float* scr = (float*)fmlp_lds;
    const int kq = PR::kq(wave), set = wave / KQ * (KQ - 1);
    if (kq > 0)
#pragma unroll
      for (int p = 0; p < MP; ++p)
#pragma unroll
        for (int i = 0; i < 16; ++i) scr[(((set + kq - 1) * MP + p) * 16 + i) * 64 + lane] = acc[p][i];
    __syncthreads();
    if (kq == 0)
#pragma unroll
      for (int w = 0; w < KQ - 1; ++w)
#pragma unroll
        for (int p = 0; p < MP; ++p)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[p][i] += scr[(((set + w) * MP + p) * 16 + i) * 64 + lane];
    __syncthreads();
  }
}
template <int NP, bool TALL, int TERMS>
constexpr int gram_lds() {
  return std::max(TERMS * Tile<NP, TALL>::TERM, (Pairs<NP>::WAVES - Pairs<NP>::WAVES / Pairs<NP>::KQ) * Pairs<NP>::MP * 4096);
}

// the wave's tiles as both halves of a symmetric matrix, rows `pitch` floats apart
template <int NP>
__device__ __forceinline__ void store_gram(const f32x16 (&acc)[Pairs<NP>::MP], float* dst, int pitch, int wave,
                                           int lane) {
  const int g = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int p = 0; p < Pairs<NP>::MP; ++p) {
    if (Pairs<NP>::kq(wave) > 0 || !Pairs<NP>::has(p, wave)) continue;
    const int bi = Pairs<NP>::row(p, wave), bj = Pairs<NP>::col(p, wave);
    const int c = bj * 32 + l32, r = bi * 32 + 4 * g;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *(float4*)(dst + (size_t)c * pitch + r + 8 * q) = float4{acc[p][4 * q], acc[p][4 * q + 1], acc[p][4 * q + 2], acc[p][4 * q + 3]};
      if (bi != bj)
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[(size_t)(r + 8 * q + j) * pitch + c] = acc[p][4 * q + j];
    }
  }
}

// Gram matrices: `parts` workgroups a matrix, each a range of the long side, their partial sums whole and symmetric.
template <int NP, int TERMS, bool BF, bool VEC>
__global__ void __launch_bounds__(Pairs<NP>::WAVES * 64) gram_kernel(MuonTable tab, float* __restrict__ G, int parts, float mu, float nu, int nesterov) {
  const unsigned block = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);  // (where the steps read a matrix's sums)
  const MuonRef& t = tensor_of(tab, block);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  f32x16 acc[Pairs<NP>::MP];
  Part p;
  const auto run = [&](auto TALL) {
    constexpr bool L = decltype(TALL)::value;
    p = part_of<NP, L>(t, parts, block);
    gram_tiles<NP, L, TERMS, BF, VEC>(acc, t, p, mu, nu, nesterov, wave);
  };
  if (t.R > t.C) run(std::true_type{});
  else run(std::false_type{});
  store_gram<NP>(acc, G + ((size_t)(t.matrix0 + p.h) * parts + p.part) * (NP * NP), NP, wave, lane);
}

// The same for few matrices of 256: 64 x 64 tiles i <= j of a Gram matrix, `parts` workgroups each, which have a range of the long
// side by 64. Waves: a 32 x 32 quarter of the tile and half of the long side's 16s, and the next values into the other buffer's terms.
// m' is in memory already (momentum_kernel). 8 x 256 x 1024 fp32 13.7 us, 7.5 of them there with the shortest long side too.
template <bool TALL, int TERMS, bool BF, bool VEC>
__device__ __forceinline__ void gram_tile(const MuonRef& t, unsigned block, float* __restrict__ G, int parts, float mu, float nu,
                                          int nesterov) {
  using T = Tile<64, TALL, 64>;
  constexpr int KT = T::KT, BLOCK = TERMS * T::TERM;
  static_assert(T::UNITS == 512, "one for each thread");
  const unsigned local = block - t.block0;
  const long long h = local / (unsigned)(kMuonGramTiles * parts);
  const int part = (int)(local / kMuonGramTiles % (unsigned)parts), tile = (int)(local % kMuonGramTiles);
  const int bi = tile < 4 ? 0 : tile < 7 ? 1 : tile < 9 ? 2 : 3, bj = tile - (bi * (7 - bi)) / 2;
  const int R = t.R, C = t.C, small = TALL ? C : R, lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), qr = (wave >> 1) & 1, qc = wave & 1, half = wave >> 2;
  const long long L = TALL ? R : C, tiles = (L + KT - 1) / KT, per = (tiles + parts - 1) / parts;
  const long long t0 = part * per, t1 = bj * 64 < small ? min(tiles, t0 + per) : t0;
  const Mat<VEC> X(t.x, t.x_io, h, R, C), M(t.m, t.m_io, h, R, C);
  const bool momentum = t.m != nullptr, two = bi != bj, has = two || qr <= qc;

  constexpr int AHEAD = 2;
  Raw x[AHEAD][2], m[AHEAD][TERMS == 3 ? 2 : 1];
  const int row = (int)threadIdx.x / T::UR, u = (int)threadIdx.x % T::UR;
  const auto load = [&](long long k, Raw (&xs)[2], Raw (&ms)[TERMS == 3 ? 2 : 1]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int s0 = (b ? bj : bi) * 64;
      const long long r = TALL ? k * KT + row : s0 + row, c = TALL ? s0 + u * 8 : k * KT + u * 8, i = r * C + c;
      const int n = k < t1 && (!b || two) && r < R ? (int)max(0LL, min(8LL, C - c)) : 0;
      if constexpr (TERMS == 3) {
        X.load(i, n, xs[b]);
        M.load(i, n, ms[b]);
      } else {
        xs[b].a = X.load16(i, n);
      }
    }
  };
  const auto put = [&](int buffer, const Raw (&xs)[2], const Raw (&ms)[TERMS == 3 ? 2 : 1]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b && !two) continue;
      const int o = (2 * buffer + b) * BLOCK + T::at(row, u);
      if constexpr (TERMS == 3) {
        float f[8];
        unpack_raw(X.io, xs[b], f);
        if (momentum) {
          float v[8];
          unpack_raw(M.io, ms[b], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = nesterov ? __builtin_fmaf(mu, v[j], nu * f[j]) : v[j];
        }
        u32x4 s[3];
        split3(f, s);
#pragma unroll
        for (int e = 0; e < 3; ++e) lds_write16(e * T::TERM + o, s[e]);
      } else {
        lds_write16(o, xs[b].a);
      }
    }
  };
  f32x16 acc = zero16();
  const auto multiply = [&](int buffer) {
    if (!has) return;
#pragma unroll
    for (int j = 0; j < KT / 32; ++j) {
      const int k0 = 16 * (half * (KT / 32) + j);
      u32x4 a[TERMS], b[TERMS];
#pragma unroll
      for (int e = 0; e < TERMS; ++e) {
        a[e] = T::by_small(2 * buffer * BLOCK + e * T::TERM, qr * 32, k0, lane);
        b[e] = T::by_small((2 * buffer + (two ? 1 : 0)) * BLOCK + e * T::TERM, qc * 32, k0, lane);
      }
      acc = mfma_terms<TERMS, BF>(a, b, acc);
    }
  };
  load(t0, x[0], m[0]);
  load(t0 + 1, x[1], m[1]);
  put(0, x[0], m[0]);
  load(t0 + 2, x[0], m[0]);
  __syncthreads();
  for (long long k = t0; k < t1; k += 2) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {  // (past the end: zeros)
      multiply(p);
      put(1 - p, x[1 - p], m[1 - p]);
      load(k + p + 3, x[1 - p], m[1 - p]);
      __syncthreads();
    }
  }
  float* scr = (float*)fmlp_lds + (wave & 3) * 1024 + lane;
  if (half)
#pragma unroll
    for (int i = 0; i < 16; ++i) scr[i * 64] = acc[i];
  __syncthreads();
  if (half || !has) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] += scr[i * 64];
  const int g = lane >> 5, l32 = lane & 31, c = bj * 64 + qc * 32 + l32, r = bi * 64 + qr * 32 + 4 * g;
  float* dst = G + ((size_t)(t.matrix0 + h) * parts + part) * (256 * 256);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    *(float4*)(dst + c * 256 + r + 8 * q) = float4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    if (two || qr != qc)
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[(r + 8 * q + j) * 256 + c] = acc[4 * q + j];
  }
}
template <int TERMS, bool BF, bool VEC>
__global__ void __launch_bounds__(512) gram_tile_kernel(MuonTable tab, float* __restrict__ G, int parts, float mu, float nu, int nesterov) {
  const unsigned block = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);  // (a matrix on one XCD's L2: each value is read four times)
  const MuonRef& t = tensor_of(tab, block);
  if (t.R > t.C) gram_tile<true, TERMS, BF, VEC>(t, block, G, parts, mu, nu, nesterov);
  else gram_tile<false, TERMS, BF, VEC>(t, block, G, parts, mu, nu, nesterov);
}

// m' = mu m + nu x, `parts` workgroups a matrix
template <bool VEC>
__global__ void __launch_bounds__(256) momentum_kernel(MuonTable tab, int parts, float mu, float nu) {
  const MuonRef& t = tensor_of(tab, blockIdx.x);
  const unsigned local = blockIdx.x - t.block0;
  const Mat<VEC> X(t.x, t.x_io, local / (unsigned)parts, t.R, t.C), M(t.m, t.m_io, local / (unsigned)parts, t.R, t.C);
  const long long n = (long long)t.R * t.C;
  for (long long i = ((long long)(local % (unsigned)parts) * 256 + threadIdx.x) * 8; i < n; i += (long long)parts * 2048) {
    const int there = (int)min(8LL, n - i);
    Raw x, m;
    X.load(i, there, x);
    M.load(i, there, m);
    float f[8], v[8];
    unpack_raw(X.io, x, f);
    unpack_raw(M.io, m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(mu, v[j], nu * f[j]);
    pack_raw(M.io, v, m);
    M.store(i, there, m);
  }
}

// O = P u over the data tiles [t0, t1), and what becomes of it. XT: terms of u. Waves: a block of 32 small indices, whose rows of P
// are ph and pl, and CT of 32 long ones each.
template <int NP, bool TALL, int XT, bool VEC>
__device__ __forceinline__ void apply_tiles(const u32x4 (&ph)[NP / 16], const u32x4 (&pl)[NP / 16], const MuonRef& t, const Part& part,
                                            MuonInfo fo, float mu, float nu, int nesterov, int update, float keep, int wave) {
  using T = Tile<NP, TALL>;
  constexpr int THREADS = NP == 256 ? 512 : 256;
  constexpr int KT = T::KT, RB = NP / 32, CT = NP == 256 ? 1 : 2, KS = NP / 16, Q = T::UNITS / THREADS;
  constexpr int OPITCH = T::COLS + 4;  // floats between the result's rows in LDS
  const int R = t.R, C = t.C, lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int s0 = (wave % RB) * 32, c0 = wave / RB * CT * 32;
  const long long t0 = part.t0, t1 = part.t1;
  const Mat<VEC> X(t.x, t.x_io, part.h, R, C), M(t.m, t.m_io, part.h, R, C), O(t.out, t.out_io, part.h, R, C);
  const bool momentum = t.m != nullptr;
  Raw x[Q], m[Q], w[Q];
  const auto load = [&](long long tile, int q) {
    const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
    X.load(at.i, at.n, x[q]);
    M.load(at.i, at.n, m[q]);
  };
  float* res = (float*)fmlp_lds;  // the result takes the tile's place
#pragma unroll
  for (int q = 0; q < Q; ++q) load(t0, q);
  for (long long tile = t0; tile < t1; ++tile) {
    if (update) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
        O.load(at.i, at.n, w[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const Piece<NP, TALL, THREADS> at(q, tile * KT, R, C);
      float f[8];
      unpack_raw(X.io, x[q], f);
      if (momentum) {
        float v[8];
        unpack_raw(M.io, m[q], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = nesterov ? __builtin_fmaf(mu, v[j], nu * f[j]) : v[j];
      }
      if (tile + 1 < t1) load(tile + 1, q);
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
        unpack_raw(O.io, w[q], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __builtin_fmaf(-t.lr, f[j], v[j] * keep);
      }
      pack_raw(O.io, f, w[q]);
      O.store(at.i, at.n, w[q]);
    }
    __syncthreads();
  }
}
template <int NP, bool TALL, int XT>
constexpr int apply_lds() {
  return std::max(XT * Tile<NP, TALL>::TERM, Tile<NP, TALL>::ROWS * (Tile<NP, TALL>::COLS + 4) * 4);
}

template <int NP, int XT, bool VEC>
__global__ void __launch_bounds__(NP == 256 ? 512 : 256)
apply_kernel(MuonTable tab, const u16* __restrict__ P, const MuonInfo* __restrict__ info, int parts, float mu, float nu, int nesterov,
             int update, float keep) {
  const unsigned block = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);  // (a matrix's P on one XCD's L2)
  const MuonRef& t = tensor_of(tab, block);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const auto run = [&](auto TALL) {
    constexpr bool L = decltype(TALL)::value;
    const Part p = part_of<NP, L>(t, parts, block);
    if (p.t0 >= p.t1) return;
    u32x4 ph[NP / 16], pl[NP / 16];
    const u16* src = P + (size_t)(t.matrix0 + p.h) * (2 * NP * NP) + muon_chunk<NP>((wave % (NP / 32)) * 32 + (lane & 31), 0, lane >> 5);
#pragma unroll
    for (int k = 0; k < NP / 16; ++k) {
      ph[k] = *(const u32x4*)(src + 512 * k);
      pl[k] = *(const u32x4*)(src + NP * NP + 512 * k);
    }
    apply_tiles<NP, L, XT, VEC>(ph, pl, t, p, info[t.matrix0 + p.h], mu, nu, nesterov, update, keep, wave);
  };
  if (t.R > t.C) run(std::true_type{});
  else run(std::false_type{});
}

// ---------------------------------------------------------------------------------------------
// a workgroup a matrix from end to end, NP <= 128
// ---------------------------------------------------------------------------------------------
// byte offset of 16-byte unit u of row r of a [NP][NP] fp16 matrix: units are swapped within a row so that 16
// consecutive rows' units lie on all banks
template <int NP>
__device__ __forceinline__ int unit_off(int r, int u) {
  constexpr int UR = NP / 8;  // units of a row
  const int f = UR >= 16 ? r & 15 : UR == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  return r * (NP * 2) + ((u ^ f) << 4);
}

// A wave's 32 columns of a matrix as both fp16 terms: unit (tile t, half h) of the lane of column n and half g holds
// rows 32 t + 16 h + 4 g + {0..3, 8..11}, the order that a result has them in
template <int NP>
struct Cols {
  u32x4 hi[NP / 16], lo[NP / 16];
};
template <int NP>
__device__ __forceinline__ void pack_cols(const f32x16 (&v)[NP / 32], float s, Cols<NP>& c) {
#pragma unroll
  for (int t = 0; t < NP / 32; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[t][8 * h + j];
      split8(f, s, c.hi[2 * t + h], c.lo[2 * t + h]);
    }
}
// the columns as rows of the left operand
template <int NP>
__device__ __forceinline__ void put_left(const Cols<NP>& c, int n, int g) {
#pragma unroll
  for (int k = 0; k < NP / 16; ++k) {
    const int at = unit_off<NP>(n, 2 * k + g);
    lds_write16(at, c.hi[k]);
    lds_write16(NP * NP * 2 + at, c.lo[k]);
  }
}

// out = (left operand in LDS) * b, in the terms' scales. A step has 16 of the inner dimension for two tiles of rows: their
// operands are read a step ahead.
template <int NP>
__device__ __forceinline__ void product(f32x16 (&out)[NP / 32], const Cols<NP>& b, int g, int l32) {
  constexpr int RB = NP / 32, TP = RB < 2 ? RB : 2, PAIRS = RB / TP, STEPS = NP / 16 * PAIRS;
  u32x4 ah[2][TP], al[2][TP];
  const auto fetch = [&](int j) {
    const int k = j / PAIRS, p = j % PAIRS;
#pragma unroll
    for (int t = 0; t < TP; ++t) {
      const int at = unit_off<NP>(l32, 2 * k + g) + (p * TP + t) * (32 * NP * 2);
      ah[j & 1][t] = lds_read16(at);
      al[j & 1][t] = lds_read16(NP * NP * 2 + at);
    }
  };
  fetch(0);
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    const int k = j / PAIRS, p = j % PAIRS;
    if (j + 1 < STEPS) fetch(j + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma<false>(al[j & 1][t], b.hi[k], k == 0 ? zero16() : out[p * TP + t]);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma<false>(ah[j & 1][t], b.lo[k], out[p * TP + t]);
#pragma unroll
    for (int t = 0; t < TP; ++t) out[p * TP + t] = mfma<false>(ah[j & 1][t], b.hi[k], out[p * TP + t]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Gram matrix, steps and result of one matrix: two workgroups a CU, one of which streams while the other is at its steps (2304
// matrices of 128 x 1024 in launches of their own: 2232 us, 475 of them steps; here 1.75 ms). The steps are those of
// fmlp_muon_iter.hip with 32 columns a wave (the first NP / 32 waves), which reads a left operand half as often. NP = 128 spills 44
// registers of 256, between the passes.
template <int NP, int TERMS, bool BF, bool VEC>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
whole_kernel(MuonTable tab, MuonSteps s, float mu, float nu, int nesterov, int update, float keep) {
  constexpr int RB = NP / 32, GP = NP + 4, SCR = NP * GP * 4;  // LDS: G or the left operand, then the waves' sums
  const MuonRef& t = tensor_of(tab, blockIdx.x);
  const bool tall = t.R > t.C;
  const Part part = tall ? part_of<NP, true>(t, 1, blockIdx.x) : part_of<NP, false>(t, 1, blockIdx.x);
  const int lane = (int)threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = wave * 32 + l32;
  float* lds = (float*)fmlp_lds;
  {
    f32x16 acc[Pairs<NP>::MP];
    if (tall) gram_tiles<NP, true, TERMS, BF, VEC>(acc, t, part, mu, nu, nesterov, wave);
    else gram_tiles<NP, false, TERMS, BF, VEC>(acc, t, part, mu, nu, nesterov, wave);
    store_gram<NP>(acc, lds, GP, wave, lane);
  }
  __syncthreads();
  const bool on = wave < RB;
  f32x16 v[RB];
  const auto diagonal = [&](int tile, int i) { return tile == wave && 8 * (i >> 2) + 4 * g + (i & 3) == l32; };
  float d = 0.f;
  if (on) {
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 f = *(const float4*)(lds + n * GP + 32 * r + 8 * q + 4 * g);
        v[r][4 * q] = f.x;
        v[r][4 * q + 1] = f.y;
        v[r][4 * q + 2] = f.z;
        v[r][4 * q + 3] = f.w;
      }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (diagonal(r, i)) d = v[r][i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
    if (lane == 0) *(float*)(fmlp_lds + SCR + 4 * wave) = d;
  }
  __syncthreads();
  float trace = 0.f;
#pragma unroll
  for (int w = 0; w < RB; ++w) trace += *(const float*)(fmlp_lds + SCR + 4 * w);
  float inv;
  const MuonInfo fo = info_of(trace, s, s.p_scale[s.steps - 1], &inv);
  Cols<NP> G, P;
  if (on) {
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) v[r][i] = v[r][i] * inv * inv;
    pack_cols<NP>(v, s.g_scale[0], G);
  }
  for (int k = 0; k < s.steps; ++k) {
    const float sg = s.g_scale[k], sq = s.q_scale[k], st = sg * sq * 0x1p-14f;
    const bool last = k + 1 == s.steps;
    if (on) put_left<NP>(G, n, g);
    __syncthreads();
    if (on) {
      product<NP>(v, G, g, l32);
      const float cc = s.c[k] / sg / sg, cb = s.b[k] / sg, ca = s.a[k];
#pragma unroll
      for (int u = 0; u < NP / 16; ++u) {
        float f[8];
        const u32x4 gh = G.hi[u], gl = G.lo[u];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = j & 1 ? hi_f32<false>(gh[j >> 1]) + hi_f32<false>(gl[j >> 1])
                                : lo_f32<false>(gh[j >> 1]) + lo_f32<false>(gl[j >> 1]);
          const int i = 8 * (u & 1) + j;
          f[j] = __builtin_fmaf(cc, v[u >> 1][i], __builtin_fmaf(cb, x, diagonal(u >> 1, i) ? ca : 0.f));
        }
        split8(f, sq, G.hi[u], G.lo[u]);
      }
      if (!last) product<NP>(v, G, g, l32);
    }
    __syncthreads();
    if (on) put_left<NP>(G, n, g);
    __syncthreads();
    if (on) {
      if (k == 0) P = G;
      if (!last) pack_cols<NP>(v, st / sg / sq, G);
      if (k > 0) {
        product<NP>(v, P, g, l32);
        pack_cols<NP>(v, s.p_scale[k] / sq / s.p_scale[k - 1], P);
      }
      if (!last) {
        product<NP>(v, G, g, l32);
        pack_cols<NP>(v, s.g_scale[k + 1] / sq / st, G);
      }
    }
    __syncthreads();
  }
  // every wave's rows of P
  if (on) put_left<NP>(P, n, g);
  __syncthreads();
  u32x4 ph[NP / 16], pl[NP / 16];
  const int row = (wave % RB) * 32 + l32;
#pragma unroll
  for (int k = 0; k < NP / 16; ++k) {
    ph[k] = lds_read16(unit_off<NP>(row, 2 * k + g));
    pl[k] = lds_read16(NP * NP * 2 + unit_off<NP>(row, 2 * k + g));
  }
  __syncthreads();
  constexpr int XT = TERMS == 3 ? 2 : 1;
  if (tall) apply_tiles<NP, true, XT, VEC>(ph, pl, t, part, fo, mu, nu, nesterov, update, keep, wave);
  else apply_tiles<NP, false, XT, VEC>(ph, pl, t, part, fo, mu, nu, nesterov, update, keep, wave);
}

template <int NP, int TERMS>
constexpr int both_gram_lds() {
  return std::max(gram_lds<NP, true, TERMS>(), gram_lds<NP, false, TERMS>());
}
template <int NP, int XT>
constexpr int both_apply_lds() {
  return std::max(apply_lds<NP, true, XT>(), apply_lds<NP, false, XT>());
}
// f(terms of G, whether they are bf16, whole vectors) as constants
template <typename F>
hipError_t by_kind(const MuonKind& k, F f) {
  const auto v = [&](auto terms, auto bf) { return k.vec ? f(terms, bf, std::true_type{}) : f(terms, bf, std::false_type{}); };
  if (k.terms == 3) return v(std::integral_constant<int, 3>{}, std::true_type{});
  return k.bf ? v(std::integral_constant<int, 1>{}, std::true_type{}) : v(std::integral_constant<int, 1>{}, std::false_type{});
}
template <int LDS, typename K, typename... A>
hipError_t launch(K k, std::atomic<unsigned long long>& done, unsigned blocks, int threads, hipStream_t st, A... args) {
  const hipError_t e = set_lds_once((const void*)k, LDS, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(blocks), dim3(threads), LDS, st, args...);
  return hipGetLastError();
}

}  // namespace

template <int NP>
hipError_t muon_gram(const MuonKind& kind, const MuonTable& tab, unsigned blocks, float* G, int parts, const MuonCall& c, hipStream_t st) {
  return by_kind(kind, [&](auto T, auto B, auto V) {
    constexpr int TERMS = decltype(T)::value;
    static std::atomic<unsigned long long> done{0};
    return launch<both_gram_lds<NP, TERMS>()>(gram_kernel<NP, TERMS, decltype(B)::value, decltype(V)::value>, done, blocks,
                                              Pairs<NP>::WAVES * 64, st, tab, G, parts, c.mu, c.nu, c.nesterov);
  });
}
template <int NP>
hipError_t muon_apply(const MuonKind& kind, const MuonTable& tab, unsigned blocks, const unsigned short* P, const MuonInfo* info,
                      int parts, const MuonCall& c, int update, hipStream_t st) {
  return by_kind(kind, [&](auto T, auto B, auto V) -> hipError_t {
    constexpr int XT = decltype(T)::value == 3 ? 2 : 1;
    if constexpr (XT == 1 && !decltype(B)::value) {
      return hipErrorInvalidValue;  // (16-bit values of either type are one kind here: muon_apply's callers say bf)
    } else {
      static std::atomic<unsigned long long> done{0};
      return launch<both_apply_lds<NP, XT>()>(apply_kernel<NP, XT, decltype(V)::value>, done, blocks, NP == 256 ? 512 : 256, st, tab, P,
                                              info, parts, c.mu, c.nu, c.nesterov, update, c.keep);
    }
  });
}
template <int NP>
hipError_t muon_whole(const MuonKind& kind, const MuonTable& tab, unsigned blocks, const MuonSteps& s, const MuonCall& c, int update,
                      hipStream_t st) {
  return by_kind(kind, [&](auto T, auto B, auto V) {
    constexpr int TERMS = decltype(T)::value;
    constexpr int lds = std::max(std::max(both_gram_lds<NP, TERMS>(), both_apply_lds<NP, TERMS == 3 ? 2 : 1>()), NP * (NP + 4) * 4 + 16);
    static_assert(lds <= 80 * 1024, "two workgroups a CU");
    static std::atomic<unsigned long long> done{0};
    return launch<lds>(whole_kernel<NP, TERMS, decltype(B)::value, decltype(V)::value>, done, blocks, 256, st, tab, s, c.mu, c.nu,
                       c.nesterov, update, c.keep);
  });
}

#if FMLP_MUON_PART == 256
hipError_t muon_gram_tiles(const MuonKind& kind, const MuonTable& tab, unsigned blocks, float* G, int parts, const MuonCall& c,
                           hipStream_t st) {
  return by_kind(kind, [&](auto T, auto B, auto V) {
    constexpr int TERMS = decltype(T)::value;
    constexpr int lds = 4 * TERMS * std::max(Tile<64, true, 64>::TERM, Tile<64, false, 64>::TERM);
    static_assert(lds <= 160 * 1024 && lds >= 4 * 4096, "the terms, then half of the sums");
    static std::atomic<unsigned long long> done{0};
    return launch<lds>(gram_tile_kernel<TERMS, decltype(B)::value, decltype(V)::value>, done, blocks, 512, st, tab, G, parts, c.mu, c.nu,
                       c.nesterov);
  });
}
hipError_t muon_momentum(const MuonKind& kind, const MuonTable& tab, unsigned blocks, int parts, const MuonCall& c, hipStream_t st) {
  if (kind.vec) hipLaunchKernelGGL(momentum_kernel<true>, dim3(blocks), dim3(256), 0, st, tab, parts, c.mu, c.nu);
  else hipLaunchKernelGGL(momentum_kernel<false>, dim3(blocks), dim3(256), 0, st, tab, parts, c.mu, c.nu);
  return hipGetLastError();
}
#endif

// this part's kernels
template hipError_t muon_gram<FMLP_MUON_PART>(const MuonKind&, const MuonTable&, unsigned, float*, int, const MuonCall&, hipStream_t);
template hipError_t muon_apply<FMLP_MUON_PART>(const MuonKind&, const MuonTable&, unsigned, const unsigned short*, const MuonInfo*, int,
                                               const MuonCall&, int, hipStream_t);
#if FMLP_MUON_PART <= 128
template hipError_t muon_whole<FMLP_MUON_PART>(const MuonKind&, const MuonTable&, unsigned, const MuonSteps&, const MuonCall&, int,
                                               hipStream_t);
#endif

}  // namespace fmlp

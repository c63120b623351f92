// Gated MLP backward for gfx950, 16-bit io: dX = dG Wg^T + dU Wu^T, with
//   G = X Wg, U = X Wu, dH = dO W2^T, dG = dH U act'(G), dU = dH act(G)    recomputed per chunk of E.
//
// The forward's shape (fmlp_gated_fwd.hip): a wave owns 32 rows, whose X and dO stay in registers as the B
// operands of Gt, Ut = W^T X^T and dHt = W2 dO^T (one lane per row); dG and dU, rounded to the io type, are
// then A operands of dX as they come. The columns of a chunk are taken in the order that swaps bits 2 and 3 of
// their index, so that a lane's 8 k-slots of dX are 8 consecutive columns and Wg^T, Wu^T are read as 16-byte
// pieces of the same LDS tiles that the transposed reads take.
//
// Bound by matrix and vector issue: a chunk has 5 D / 16 products and 16 activations with their derivatives a
// lane. Phases of a chunk, one product and a share of vector work a step:
//     G(c+1)               | dG(c), dU(c) from dH, U, act, act' of c
//     dX += dG Wg^T + ..   | act, act' of c + 1
//     U(c+1), dH(c+1)      | the rest of them
// H=32 B=16384 D=128 E=1024 bf16 SiLU 600 us, 1145 TFLOP/s executed, products 61 % and vector instructions 50 % of the
// SIMDs' cycles at 1.76 GHz. Everything is recomputed, so that the backward's memory stays O(weights); dG and dU stored
// by the weight gradients' kernel and read here (2.1 GB there and back, 6 D / 16 products and the activations less) is
// not built and not measured.
#include <algorithm>
#include <type_traits>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

template <bool BF16, int D, int DG, int ACT, int NW, int ES, int NS, int OC>
__global__ void __launch_bounds__(NW * ES * 64) __attribute__((amdgpu_waves_per_eu(OC, OC)))
gated_dx_kernel(const u16* __restrict__ X, const u16* __restrict__ Wg, const u16* __restrict__ Wu,
                const u16* __restrict__ W2, const u16* __restrict__ dO, void* __restrict__ dX, int B, int E, int ldw,
                long long sx, long long sdo, int H, int T, int xs, int nct, int outf32,
                float* __restrict__ ws) {
  constexpr int NT = NW * 64, KS = DG / 16, NTN = D / 32, NPR = 4 * D / NT, NLD = 3 * NPR;
  constexpr int SLOT = 192 * D, WU = 64 * D, W2O = 128 * D, PF = NS - 1;
  // D = 256 runs lone waves: a chunk's loads stand one by one between products, which hides their address work
  // (H=8 B=8192 E=1024 bf16 170 -> 165 us); short chunks lose by the later issue (D = 32, a wave alone: 7.3 -> 8.3 us)
  constexpr bool SPREAD = D == 256;
  static_assert(NPR * NT == 4 * D && NS >= 3 && NLD * (PF - 2) < 64, "chunk loads");
  const int lane = threadIdx.x & 63;
  const int part = ES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  const int tid = threadIdx.x - part * NT;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = lane >> 4, i16 = lane & 15, g = lane >> 5, l32 = lane & 31;

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
  const int NC = (ce - cb + ES - 1) / ES;
  const int c0 = cb + part * NC, e_end = min(E, min(ce, c0 + NC) * 32);
  const int RB = part * NS * SLOT;
  const u16* Xh = X + (size_t)h * sx;
  const u16* dOh = dO + (size_t)h * sdo;
  const u16* Wgh = Wg + (size_t)h * DG * ldw;
  const u16* Wuh = Wu + (size_t)h * DG * ldw;
  const u16* W2h = W2 + (size_t)h * E * DG;
  const int b_wave = (bt * NW + wave) * 32;

  // chunk loads. Wg, Wu: row r (a column d) of four 16-byte pieces, piece q at place q ^ (r / 4 % 4); W2: blocks
  // [32 rows e][32 columns d] likewise. LDS place p takes the piece that belongs there.
  int colq[NPR];
  unsigned o1[NPR], o2[NPR];
#pragma unroll
  for (int k = 0; k < NPR; ++k) {
    const unsigned p = (unsigned)(tid + k * NT), q = (p & 3u) ^ ((p >> 4) & 3u);
    colq[k] = (int)q * 8;
    o1[k] = (p >> 2) * (unsigned)ldw * 2u + q * 16u;
    o2[k] = ((p >> 2) & 31u) * (DG * 2u) + (p >> 7) * 64u + q * 16u;
    if (DG < D) {
      if ((p >> 2) >= (unsigned)DG) o1[k] = BUF_OOB;
      if (q * 8u >= (unsigned)DG) o2[k] = BUF_OOB;
    }
  }
  struct Dst {
    i32x4 r[3];
    int lim, at;
  };
  auto chunk_at = [&](int c, int slot) {
    const int cg = c0 + c, lim = e_end - cg * 32;
    const int rem = clamp0(DG * ldw * 2 - 64 * cg, 0x7fffffff);
    return Dst{{make_rsrc_words(Wgh + (size_t)cg * 32, rem), make_rsrc_words(Wuh + (size_t)cg * 32, rem),
                make_rsrc_words(W2h + (size_t)cg * 32 * DG, clamp0(lim, 32) * DG * 2)},
               lim,
               RB + slot * SLOT + wave * 1024};
  };
  auto load_piece = [&](const Dst& d, int q) {
    const int k = q / 3, m = q % 3;
    buf_load16_lds(d.r[m], m == 2 ? o2[k] : colq[k] < d.lim ? o1[k] : BUF_OOB, d.at + m * WU + k * NT * 16);
  };
  auto load_chunk = [&](int c, int slot) {
    const Dst d = chunk_at(c, slot);
#pragma unroll
    for (int q = 0; q < NLD; ++q) load_piece(d, q);
  };
  auto sync = [&](auto N) {
    wait_vmcnt<decltype(N)::value>();
    if constexpr (NW > 1) {
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
    }
    asm volatile("" ::: "memory");
  };

  u32x4 xr[KS], dr[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int b = b_wave + l32;
    xr[k] = dr[k] = u32x4{0u, 0u, 0u, 0u};
    if (b < B) {
      xr[k] = *(const u32x4*)(Xh + (size_t)b * DG + k * 16 + g * 8);
      dr[k] = *(const u32x4*)(dOh + (size_t)b * DG + k * 16 + g * 8);
    }
  }
#pragma unroll
  for (int c = 0; c < PF; ++c) load_chunk(c, c);

  // transposed reads of Wg, Wu (rows d = 16 k + 8 g + 4 r + i16 / 4; columns: block i16 % 4 of four with its two
  // bits swapped), r = 0, 1; 16-byte reads of their rows d = 32 nt + l32, columns 16 s + 8 g ..; of W2's rows e
  // (bits 2 and 3 of l32 swapped), columns 16 k + 8 g ..
  const int cb4 = ((i16 & 1) << 1) | ((i16 >> 1) & 1);
  int aT[2], aR[2], aW[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = 8 * g + 4 * r + (i16 >> 2);
    aT[r] = row * 64 + (((2 * (G & 1) + (cb4 >> 1)) ^ (2 * g + r)) << 4) + ((cb4 & 1) << 3);
    aR[r] = l32 * 64 + (((2 * r + g) ^ ((l32 >> 2) & 3)) << 4);
    const int e = (l32 & 19) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
    aW[r] = W2O + e * 64 + (((2 * r + g) ^ ((e >> 2) & 3)) << 4);
  }
  auto opT = [&](int base, int k) { return cat(lds_read_tr(base + aT[0] + k * 1024), lds_read_tr(base + aT[1] + k * 1024)); };
  auto opR = [&](int base, int s, int nt) { return lds_read16(base + aR[s] + nt * 2048); };
  auto opW = [&](int base, int k) { return lds_read16(base + aW[k & 1] + (k >> 1) * 2048); };

  f32x16 o[NTN], zg, zu, dh;
  float sv[16], fv[16];
  u32x4 pg[2], pu[2];
#pragma unroll
  for (int nt = 0; nt < NTN; ++nt) o[nt] = zero16();

  sync(std::integral_constant<int, NLD*(PF > 2 ? PF - 2 : 0)>{});
  zg = zu = dh = zero16();
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    zg = mfma<BF16>(opT(RB, k), xr[k], zg);
    zu = mfma<BF16>(opT(RB + WU, k), xr[k], zu);
    dh = mfma<BF16>(opW(RB, k), dr[k], dh);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) act_hf<ACT>(zg[e], sv[e], fv[e]);

  auto iter = [&](auto MORE, int c, int cur, int nxt, int far) {
    constexpr bool M = decltype(MORE)::value;
    Dst dst;
    if constexpr (M && SPREAD) dst = chunk_at(c + PF, far);
    constexpr int N1 = M ? KS : 0, N2 = 4 * NTN, NOPS = 3 * N1 + N2;
    const int b1 = RB + nxt * SLOT, b2 = RB + cur * SLOT;
    auto fetch = [&](int j) {
      if (j < N1) return opT(b1, j);
      if (j < N1 + N2) {
        const int i = j - N1, m = i & 1, nt = (i >> 1) % NTN, s = (i >> 1) / NTN;
        return opR(b2 + m * WU, s, nt);
      }
      const int i = j - N1 - N2;
      return i < N1 ? opT(b1 + WU, i) : opW(b1, i - N1);
    };
    constexpr int PD = 2;
    u32x4 ring[PD + 1];
#pragma unroll
    for (int j = 0; j < PD; ++j) ring[j] = fetch(j);
    __builtin_amdgcn_sched_barrier(0);
    auto make_d = [&](int e) {
      if ((e & 1) == 0) return;
      const float g0 = dh[e - 1] * fv[e - 1] * zu[e - 1], g1 = dh[e] * fv[e] * zu[e];
      pg[e >> 3][(e >> 1) & 3] = pack2<BF16>(g0, g1);
      pu[e >> 3][(e >> 1) & 3] = pack2<BF16>(dh[e - 1] * sv[e - 1], dh[e] * sv[e]);
    };
    if constexpr (!M) {
#pragma unroll
      for (int e = 0; e < 16; ++e) make_d(e);
    }
    static_for<NOPS>([&](auto J) {
      constexpr int j = decltype(J)::value;
      const u32x4 op = ring[j % (PD + 1)];
      if constexpr (j + PD < NOPS) ring[(j + PD) % (PD + 1)] = fetch(j + PD);
      if constexpr (j < N1) {
        zg = mfma<BF16>(op, xr[j], j == 0 ? zero16() : zg);
#pragma unroll
        for (int e = 16 * j / N1; e < 16 * (j + 1) / N1; ++e) make_d(e);
      } else {
        constexpr int i = j - N1, i2 = i - N2;
        if constexpr (i < N2) {
          constexpr int nt = (i >> 1) % NTN, s = (i >> 1) / NTN;
          o[nt] = mfma<BF16>((i & 1) == 0 ? pg[s] : pu[s], op, o[nt]);
        } else if constexpr (i2 < N1) {
          zu = mfma<BF16>(op, xr[i2], i2 == 0 ? zero16() : zu);
        } else {
          dh = mfma<BF16>(op, dr[i2 - N1], i2 == N1 ? zero16() : dh);
        }
        if constexpr (M) {
          constexpr int NV = N2 + 2 * N1;
#pragma unroll
          for (int e = 16 * i / NV; e < 16 * (i + 1) / NV; ++e) act_hf<ACT>(zg[e], sv[e], fv[e]);
        }
      }
      if constexpr (M && SPREAD && j < NLD) load_piece(dst, j);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int cur = 0;
  for (int c = 0; c + 1 < NC; ++c) {
    const int nxt = cur + 1 == NS ? 0 : cur + 1, far = cur == 0 ? NS - 1 : cur - 1;
    if (!SPREAD || b_wave >= B) load_chunk(c + PF, far);
    if (b_wave < B) iter(std::true_type{}, c, cur, nxt, far);  // a wave without rows only loads
    sync(std::integral_constant<int, NLD*(PF - 2)>{});
    cur = nxt;
  }
  if (b_wave < B) iter(std::false_type{}, 0, cur, cur, cur);

  wait_vmcnt<0>();  // chunks past the last are still landing, as zeros
  if constexpr (ES > 1) {
    asm volatile("" ::: "memory");
    __syncthreads();
    const int at = wave * (NTN * 4096) + (part > 0 ? part - 1 : 0) * (NW * NTN * 4096);
    static_assert((ES - 1) * NW * NTN * 4096 <= ES * NS * SLOT, "the partial tiles fit the rings");
    if (part > 0) {
#pragma unroll
      for (int nt = 0; nt < NTN; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          lds_write16(at + ((nt * 4 + q) * 64 + lane) * 16,
                      u32x4{__float_as_uint(o[nt][4 * q]), __float_as_uint(o[nt][4 * q + 1]),
                            __float_as_uint(o[nt][4 * q + 2]), __float_as_uint(o[nt][4 * q + 3])});
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int p = 1; p < ES; ++p)
#pragma unroll
      for (int nt = 0; nt < NTN; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x4 v = lds_read16(at + (p - 1) * (NW * NTN * 4096) + ((nt * 4 + q) * 64 + lane) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][4 * q + j] += __uint_as_float(v[j]);
        }
  }
  if (xs > 1)
    store_rows<BF16, D, DG>(o, ws, (size_t)blockIdx.x * (NW * 32) * DG, B - bt * NW * 32, wave * 32, g, l32, 1);
  else
    store_rows<BF16, D, DG>(o, dX, (size_t)h * B * DG, B, b_wave, g, l32, outf32);
}

struct Args {
  const GatedArgs& a;
  const GatedFwdPlan& p;
  hipStream_t st;
};

template <bool BF16, int D, int DG, int ACT, int FORM>
hipError_t launch(const Args& q) {
  constexpr GatedForm F = gated_form(D, FORM, true);
  static_assert(gated_form_fits(D, F), "the plan's workgroups a CU");
  constexpr int lds = F.es * F.ns * 192 * D;
  auto k = gated_dx_kernel<BF16, D, DG, ACT, F.nw, F.es, F.ns, F.oc>;
  static std::atomic<unsigned long long> done{0};
  hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  const GatedArgs& a = q.a;
  const long long grid = q.p.tiles * q.p.xs;
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * F.nw * F.es), lds, q.st, (const u16*)a.x, (const u16*)a.wg,
                     (const u16*)a.wu, (const u16*)a.w2, (const u16*)a.dout, a.dx, (int)a.B, (int)a.E, (int)a.ldw,
                     (long long)a.sx, (long long)a.sdo, (int)a.H, (int)(q.p.tiles / a.H), q.p.xs, q.p.nct, a.out_f32, (float*)a.ws);
  if ((e = hipGetLastError()) != hipSuccess || q.p.xs == 1) return e;
  return launch_tile_reduce((const float*)a.ws, a.dx, BF16, (int)a.B, DG, 32 * F.nw, (int)a.H, (int)(q.p.tiles / a.H),
                            q.p.xs, (int)q.p.tiles, a.out_f32, q.st);
}

template <bool BF16, int D, int DG, int ACT>
hipError_t by_form(const Args& q) {
  if constexpr (D <= 128)
    if (q.p.form == 2) return launch<BF16, D, DG, ACT, 2>(q);
  if constexpr (D == 128)
    if (q.p.form == 1) return launch<BF16, D, DG, ACT, 1>(q);
  return launch<BF16, D, DG, ACT, 0>(q);
}
template <bool BF16, int D, int DG = D>
hipError_t by_act(const Args& q) {
  switch (q.a.act) {
    case ACT_SILU: return by_form<BF16, D, DG, ACT_SILU>(q);
    case ACT_LEAKY: return by_form<BF16, D, DG, ACT_LEAKY>(q);
    case ACT_SIGMOID: return by_form<BF16, D, DG, ACT_SIGMOID>(q);
    default: return by_form<BF16, D, DG, ACT_NONE>(q);
  }
}
template <bool BF16>
hipError_t by_d(const Args& q) {
  switch (q.a.D) {
    case 16: return by_act<BF16, 32, 16>(q);
    case 32: return by_act<BF16, 32>(q);
    case 64: return by_act<BF16, 64>(q);
    case 128: return by_act<BF16, 128>(q);
    default: return by_act<BF16, 256>(q);
  }
}

}  // namespace

hipError_t launch_gated_dx(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st) {
  if (p.tiles <= 0) return hipSuccess;
  const Args q{a, p, st};
  return a.io == IO_BF16 ? by_d<true>(q) : by_d<false>(q);
}

}  // namespace fmlp

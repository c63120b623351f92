// Gated MLP backward for gfx950, 16-bit io: the weight gradients
//   dWg = X^T dG, dWu = X^T dU, dW2 = h^T dO,   with  G = X Wg, U = X Wu, dH = dO W2^T,
//   h = act(G) U, dG = dH U act'(G), dU = dH act(G)   recomputed per 32-row subtile.
//
// A wave owns 32 columns of E and, at D <= 128, all of D: its three gradient tiles (3 D / 32 accumulators of 16
// values) and its columns of the weights stay in registers over the whole row range. G, U and dH come out with one
// lane per column of E, which is the operand layout of the gradients' products, so h, dG and dU (rounded to the
// io type) never leave registers. The four waves of a workgroup share the rows: X and dO subtiles land in an LDS
// ring by buffer loads, swizzled so that the row reads (operands of G, U, dH) and the transposed reads (operands
// of the gradients) are both free of bank conflicts. D = 256: dw256_rows.
//
// Bound by matrix and vector issue: a subtile has 6 D / 16 products and 16 activations with their derivatives a lane.
// One product and a share of vector work a step (D <= 128):
//     G(i+1)     | dG(i), dU(i) packed
//     gradients of subtile i, U(i+1)  | act, act' of i + 1
//     dH(i+1)    | h(i+1) packed, U act'
// H=32 B=16384 D=128 E=1024 bf16 SiLU 694 us, 1189 TFLOP/s executed, products 60 % and vector instructions 50 % of the
// cycles at 1.87 GHz (one wave a SIMD: they take turns; spreading the activations' stages over the steps, or reading
// operands further ahead, changed nothing). Weights from LDS instead of registers 767 us at D = 128; at D = 64, where
// they leave room for two programs a CU, 234 us at H=8 B=16384 E=2048.
// Rows are split over nS programs where the columns of E alone leave CUs idle; their fp32 partials are added in
// order by a second launch.
#include <algorithm>
#include <type_traits>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

// Waves of a workgroup: EW groups of 32 columns of E times DP parts of D. NS ring slots; OC waves per SIMD; WREG: the
// weights are held in registers, else in LDS.
struct Form {
  int ew, dp, ns, oc;
  bool wreg;
};
__host__ __device__ constexpr Form dw_form(int D) {
  if (D == 256) return {2, 2, 4, 1, true};
  return D == 128 ? Form{4, 1, 4, 1, true} : Form{4, 1, 4, 2, D == 32};
}
// LDS: the ring, then at D <= 128 the tiles of Wg and Wu (for the start only where registers hold them) and W2's (not
// there), at D = 256 the waves' partial sums
__host__ __device__ constexpr int dw_lds(int D) {
  const Form f = dw_form(D);
  return f.ns * 128 * D + (D == 256 ? 4 * 6144 : 128 * D * f.ew + (f.wreg ? 0 : 64 * D * f.ew));
}

template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 32) return (r >> 2) & 3;
  else return (int)swz16<D == 64 ? 64 : 128>((unsigned)r);
}

// D = 256: a wave owns 32 columns of E and half of D: of the weights (in registers), of the contractions over d and of
// the gradients. The two waves of a column group share a subtile's sums and activations: each gives the other its half
// sums of 16 rows, activates the 16 rows it keeps (rows are read in such an order that these are the low half of its
// accumulators), and hands back h, dG and dU. One step of the loop:
//     half sums of i + 1        | act, act', h, dG, dU of this wave's rows of i, stored for the other wave
//     barrier 1                 | (all have left subtile i - 1: i + 3 is loaded in its place)
//     gradients of i, own rows  | the other wave's h, dG, dU read, half sums of i + 1 stored
//     barrier 2                 | (i + 2 is there)
//     gradients of i, its rows  | half sums of i + 1 read and added
// H=8 B=8192 E=1024 bf16 SiLU 228 us (903 TFLOP/s of 12 u); both waves summing over all of D 290, all sums exchanged and
// both activating 283, an element's activation in one step 241; operands read 3 to 8 steps ahead within 1 %. A subtile
// takes about 1.6 us, of which its 48 products are 0.85.
template <bool BF16, int ACT>
__device__ __forceinline__ void dw256_rows(f32x16 (&ag)[4], f32x16 (&au)[4], f32x16 (&a2)[4], const u16* Xh, const u16* dOh,
                                           const u16* __restrict__ Wg, const u16* __restrict__ Wu,
                                           const u16* __restrict__ W2, int E, int ldw, int h, int e0, int r0, int r1,
                                           int wave, int dp) {
  constexpr int D = 256, DH = 128, KS = DH / 16, NTO = DH / 32, ROWB = 2 * D, PPR = D / 8, SLOT = 128 * D, DOO = 64 * D;
  constexpr int NS = dw_form(D).ns, NPR = D / 64, NLD = 2 * NPR, EX = NS * SLOT;
  static_assert(NS == 4, "the loop's waits");
  const int tid = threadIdx.x, lane = tid & 63, d0 = dp * DH;
  const int NSUB = max(0, (r1 - r0 + 31) >> 5);
  const int G = lane >> 4, i16 = lane & 15, g = lane >> 5, l32 = lane & 31;
  auto barrier = [&]() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // ---- weights: rows d0 .. of Wg, Wu as [128][32] tiles of this wave's own in the ring's place ----
  u32x4 wg[KS], wu[KS], w2[KS];
  {
    const int lim = E - e0, rem = clamp0((D - d0) * ldw * 2 - 2 * e0, 0x7fffffff), at = wave * 16384;
    const size_t base = ((size_t)h * D + d0) * ldw + e0;
    const i32x4 rg = make_rsrc_words(Wg + base, rem), ru = make_rsrc_words(Wu + base, rem);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const unsigned p = (unsigned)(k * 64 + lane), q = (p & 3u) * 8u;
      const unsigned o = (int)q < lim ? (p >> 2) * (unsigned)ldw * 2u + q * 2u : BUF_OOB;
      buf_load16_lds(rg, o, at + k * 1024);
      buf_load16_lds(ru, o, at + 8192 + k * 1024);
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      w2[k] = u32x4{0u, 0u, 0u, 0u};
      if (e0 + l32 < E) w2[k] = *(const u32x4*)(W2 + ((size_t)h * E + e0 + l32) * D + d0 + k * 16 + g * 8);
    }
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    const int a = at + (8 * g + (i16 >> 2)) * 64 + 32 * (G & 1) + 8 * (i16 & 3);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      wg[k] = cat(lds_read_tr(a + k * 1024), lds_read_tr(a + k * 1024 + 256));
      wu[k] = cat(lds_read_tr(a + 8192 + k * 1024), lds_read_tr(a + 8192 + k * 1024 + 256));
    }
    barrier();  // before the ring's loads land on the tiles
  }

  unsigned so[NPR];
#pragma unroll
  for (int k = 0; k < NPR; ++k) {
    const int p = k * 256 + tid, r = p / PPR, q = (p % PPR) ^ swz<D>(r);
    so[k] = (unsigned)(r * D * 2 + q * 16);
  }
  auto load_piece = [&](int i, int slot, int k) {  // k = 0 .. NLD - 1
    const int b = r0 + 32 * i, n = clamp0(r1 - b, 32) * D * 2;
    buf_load16_lds(make_rsrc_words((k & 1 ? dOh : Xh) + (size_t)b * D, n), so[k >> 1],
                   slot * SLOT + wave * 1024 + (k & 1) * DOO + (k >> 1) * 4096);
  };
  auto load_sub = [&](int i, int slot) {
#pragma unroll
    for (int k = 0; k < NLD; ++k) load_piece(i, slot, k);
  };
  load_sub(0, 0);
  load_sub(1, 1);
  load_sub(2, 2);
  int ro[KS], to[NTO][2];
  const int row = l32 ^ (16 * dp);  // own rows first
#pragma unroll
  for (int k = 0; k < KS; ++k) ro[k] = row * ROWB + (((2 * (dp * KS + k) + g) ^ swz<D>(row)) << 4);
#pragma unroll
  for (int n = 0; n < NTO; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int rr = 8 * r + 4 * g + (i16 >> 2), q = 4 * (dp * NTO + n) + 2 * (G & 1) + ((i16 & 3) >> 1);
      to[n][r] = rr * ROWB + ((q ^ swz<D>(rr)) << 4) + ((i16 & 1) << 3);
    }
  const int own = dp * 16 * ROWB, its = 16 * ROWB - own;
  auto opCol = [&](int a, int n) { return cat(lds_read_tr(a + to[n][0]), lds_read_tr(a + to[n][1])); };

  // A wave's 6 KB: its half sums for the other wave, which puts the other's h, dG and dU there once it has read them
  const int mine = EX + wave * 6144 + lane * 16, other = EX + (wave ^ 2) * 6144 + lane * 16;
  f32x16 y[3];         // half sums of G, U, dH
  float z[3][8];       // G, U, dH of the own rows
  u32x4 po[3], pi[3];  // h, dG, dU of the own rows and of the other wave's
  auto give = [&](int k) {  // k = 0 .. 5
    const f32x16& u = y[k >> 1];
    const int j = 8 + 4 * (k & 1);
    lds_write16(mine + k * 1024, u32x4{__float_as_uint(u[j]), __float_as_uint(u[j + 1]), __float_as_uint(u[j + 2]),
                                       __float_as_uint(u[j + 3])});
  };
  auto add = [&](int k, u32x4 u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) z[k >> 1][4 * (k & 1) + j] = y[k >> 1][4 * (k & 1) + j] + __uint_as_float(u[j]);
  };
  float ez, sv, fv, hv, gv, uv;  // an element between its thirds; an even one's h, dG and dU until the odd one's are there
  auto element = [&](int e, int third) {
    if (third == 0) {
      ez = act_den<ACT>(z[0][e]);
    } else if (third == 1) {
      act_hf_den<ACT>(z[0][e], ez, sv, fv);
    } else {
      const float a = sv * z[1][e], b = z[2][e] * (fv * z[1][e]), c = z[2][e] * sv;
      if (e & 1) {
        po[0][e >> 1] = pack2<BF16>(hv, a);
        po[1][e >> 1] = pack2<BF16>(gv, b);
        po[2][e >> 1] = pack2<BF16>(uv, c);
      } else {
        hv = a;
        gv = b;
        uv = c;
      }
    }
  };
  auto give_packs = [&]() {
#pragma unroll
    for (int k = 0; k < 3; ++k) lds_write16(other + k * 1024, po[k]);
  };
  // subtile sub in slot cur, the next in slot nxt (M: there is such a subtile)
  auto iter = [&](auto MORE, int sub, int cur, int nxt) {
    constexpr bool M = decltype(MORE)::value;
    constexpr int N1 = M ? 3 * KS : 0, N2 = 3 * NTO, NOPS = N1 + 2 * N2;
    constexpr int B1 = N1 + 3, B2 = N1 + N2 + 3;  // steps that the barriers stand before
    const int b1 = nxt * SLOT, b2 = cur * SLOT;
    auto fetch = [&](auto J) -> u32x4 {
      constexpr int j = decltype(J)::value;
      if constexpr (j < N1) {
        if constexpr (j % 3 == 0) return lds_read16(b1 + ro[j / 3]);
        else if constexpr (j % 3 == 2) return lds_read16(b1 + DOO + ro[j / 3]);
        else return u32x4{0u, 0u, 0u, 0u};
      } else {
        constexpr int i = j - N1, m = i % 3, n = i / 3 % NTO;
        const int a = b2 + (i < N2 ? own : its);
        if constexpr (m == 0) return opCol(a, n);
        else if constexpr (m == 2) return opCol(a + DOO, n);
        else return u32x4{0u, 0u, 0u, 0u};
      }
    };
    constexpr int PD = 4;
    u32x4 ring[PD + 1], xt, sums[6];
    static_for<PD>([&](auto J) { ring[J] = fetch(J); });
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!M) {
#pragma unroll
      for (int e = 0; e < 24; ++e) element(e / 3, e % 3);
      give_packs();
    }
    static_for<NOPS>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if constexpr (M && j == N1) give_packs();
      if constexpr (j == B1) {
        barrier();
#pragma unroll
        for (int k = 0; k < 3; ++k) pi[k] = lds_read16(mine + k * 1024);
      }
      if constexpr (M && j == B2) {
        wait_vmcnt<NLD>();  // subtile sub + 2
        barrier();
      }
      const u32x4 op = ring[j % (PD + 1)];
      if constexpr (j + PD < NOPS) ring[(j + PD) % (PD + 1)] = fetch(std::integral_constant<int, j + PD>{});
      if constexpr (j < N1) {
        constexpr int c = j % 3, k = j / 3;
        if constexpr (c == 0) xt = op;
        y[c] = mfma<BF16>(c == 1 ? xt : op, c == 0 ? wg[k] : c == 1 ? wu[k] : w2[k], k == 0 ? zero16() : y[c]);
        element(j / 3, j % 3);
      } else {
        constexpr int i = j - N1, m = i % 3, n = i / 3 % NTO, half = i / N2;
        const u32x4(&p)[3] = half ? pi : po;
        if constexpr (m == 0) {
          xt = op;
          ag[n] = mfma<BF16>(p[1], xt, ag[n]);
        } else if constexpr (m == 1) {
          au[n] = mfma<BF16>(p[2], xt, au[n]);
        } else {
          a2[n] = mfma<BF16>(op, p[0], a2[n]);
        }
        if constexpr (M && j > B1 && j <= B1 + 6) give(j - B1 - 1);
        if constexpr (M && j >= B1 && j < B1 + NLD) load_piece(sub + 3, (cur + NS - 1) & (NS - 1), j - B1);
        if constexpr (M && j >= B2 && j < B2 + 3) {
          sums[2 * (j - B2)] = lds_read16(other + (2 * (j - B2)) * 1024);
          sums[2 * (j - B2) + 1] = lds_read16(other + (2 * (j - B2) + 1) * 1024);
        }
        if constexpr (M && j >= NOPS - 3) {
          add(2 * (j - NOPS + 3), sums[2 * (j - NOPS + 3)]);
          add(2 * (j - NOPS + 3) + 1, sums[2 * (j - NOPS + 3) + 1]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  if (NSUB > 0) {
    wait_vmcnt<2 * NLD>();  // subtile 0
    barrier();
#pragma unroll
    for (int c = 0; c < 3; ++c) y[c] = zero16();
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const u32x4 x = lds_read16(ro[k]);
      y[0] = mfma<BF16>(x, wg[k], y[0]);
      y[1] = mfma<BF16>(x, wu[k], y[1]);
      y[2] = mfma<BF16>(lds_read16(DOO + ro[k]), w2[k], y[2]);
    }
#pragma unroll
    for (int k = 0; k < 6; ++k) give(k);
    wait_vmcnt<NLD>();  // subtile 1
    barrier();
#pragma unroll
    for (int k = 0; k < 6; ++k) add(k, lds_read16(other + k * 1024));
    int cur = 0;
    for (int i = 0; i + 1 < NSUB; ++i) {
      const int nxt = (cur + 1) & (NS - 1);
      iter(std::true_type{}, i, cur, nxt);
      cur = nxt;
    }
    iter(std::false_type{}, 0, cur, cur);
  }
}

template <bool BF16, int D, int DG, int ACT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(dw_form(D).oc, dw_form(D).oc)))
gated_dw_kernel(const u16* __restrict__ X, const u16* __restrict__ Wg, const u16* __restrict__ Wu,
                const u16* __restrict__ W2, const u16* __restrict__ dO, void* __restrict__ dWg, void* __restrict__ dWu,
                void* __restrict__ dW2, int H, int B, int E, int ldw, long long sx, long long sdo, int nE, int nS,
                int rows_per_split, float scale, float* __restrict__ ws) {
  constexpr Form F = dw_form(D);
  constexpr int EW = F.ew, DP = F.dp, NS = F.ns, PF = NS - 1;
  constexpr bool WREG = F.wreg;
  constexpr int KS = DG / 16, NTO = D / 32 / DP, ROWB = 2 * D, PPR = D / 8, SLOT = 128 * D, DOO = 64 * D;
  constexpr int NPR = D >= 64 ? D / 64 : 1, NLD = D >= 64 ? 2 * NPR : 1;  // loads a thread for X (and dO)
  constexpr int WL = NS * SLOT, W2L = WL + 128 * D * EW;
  static_assert(EW * DP == 4 && NLD * PF < 64 && dw_lds(D) <= 160 * 1024, "form");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = lane >> 4, i16 = lane & 15, g = lane >> 5, l32 = lane & 31;

  const unsigned t = (unsigned)xcd_remap(blockIdx.x, gridDim.x);
  const int et = (int)(t % (unsigned)nE);
  const unsigned hs = t / (unsigned)nE;
  const int s = (int)(hs % (unsigned)nS), h = (int)(hs / (unsigned)nS);
  const int eg = DP == 1 ? wave : wave & (EW - 1), dp = DP == 1 ? 0 : wave / EW;
  const int e0 = (et * EW + eg) * 32, d0 = dp * NTO * 32;
  const int r0 = s * rows_per_split, r1 = min(B, r0 + rows_per_split), NSUB = max(0, (r1 - r0 + 31) >> 5);
  const u16* Xh = X + (size_t)h * sx;
  const u16* dOh = dO + (size_t)h * sdo;
  f32x16 ag[NTO], au[NTO], a2[NTO];
#pragma unroll
  for (int n = 0; n < NTO; ++n) ag[n] = au[n] = a2[n] = zero16();
  auto barrier = [&]() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  if constexpr (D == 256) {
    dw256_rows<BF16, ACT>(ag, au, a2, Xh, dOh, Wg, Wu, W2, E, ldw, h, e0, r0, r1, wave, dp);
  } else {
    const u16* Wgh = Wg + (size_t)h * DG * ldw;
    const u16* Wuh = Wu + (size_t)h * DG * ldw;
    const u16* W2h = W2 + (size_t)h * E * DG;

    // ---- weights: this wave's columns of Wg, Wu as [D][32] tiles through LDS ----
    u32x4 wg[WREG ? KS : 1], wu[WREG ? KS : 1], w2[WREG ? KS : 1];
    const int laneA = (8 * g + (i16 >> 2)) * 64 + 32 * (G & 1) + 8 * (i16 & 3);
    const int wt[2] = {WL + wave * 64 * D, WL + 64 * D * EW + wave * 64 * D};
    auto opWt = [&](int m, int k) {
      const int a = wt[m] + laneA + k * 1024;
      return cat(lds_read_tr(a), lds_read_tr(a + 256));
    };
    {
      const int lim = E - e0, rem = clamp0(DG * ldw * 2 - 2 * e0, 0x7fffffff);
      const i32x4 rg = make_rsrc_words(Wgh + e0, rem), ru = make_rsrc_words(Wuh + e0, rem);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const unsigned p = (unsigned)(k * 64 + lane), q = (p & 3u) * 8u;
        const unsigned o = (int)q < lim && (p >> 2) < (unsigned)DG ? (p >> 2) * (unsigned)ldw * 2u + q * 2u : BUF_OOB;
        buf_load16_lds(rg, o, wt[0] + k * 1024);
        buf_load16_lds(ru, o, wt[1] + k * 1024);
      }
      if constexpr (WREG) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          w2[k] = u32x4{0u, 0u, 0u, 0u};
          if (e0 + l32 < E) w2[k] = *(const u32x4*)(W2h + (size_t)(e0 + l32) * DG + k * 16 + g * 8);
        }
      } else {  // rows e of the whole E-tile, swizzled as the subtiles are
        const int eb = et * EW * 32;
        const i32x4 r2 = make_rsrc_words(W2h + (size_t)eb * DG, clamp0(E - eb, EW * 32) * DG * 2);
#pragma unroll
        for (int i = 0; i < EW * 32 * PPR / 256; ++i) {
          const int p = i * 256 + tid, r = p / PPR, q = (p % PPR) ^ swz<D>(r);
          buf_load16_lds(r2, q * 8 < DG ? (unsigned)(r * DG * 2 + q * 16) : BUF_OOB, W2L + i * 4096 + wave * 1024);
        }
      }
    }
    // ---- subtiles: X and dO rows r0 + 32 i .., 16-byte piece q of row r at place q ^ swz(r) ----
    unsigned so[NPR];
#pragma unroll
    for (int k = 0; k < NPR; ++k) {
      const int p = D >= 64 ? k * 256 + tid : tid & 127, r = p / PPR, q = (p % PPR) ^ swz<D>(r);
      so[k] = q * 8 < DG ? (unsigned)(r * DG * 2 + q * 16) : BUF_OOB;
    }
    auto load_sub = [&](int i, int slot) {
      const int b = r0 + 32 * i, n = clamp0(r1 - b, 32) * DG * 2;
      const i32x4 rx = make_rsrc_words(Xh + (size_t)b * DG, n), rd = make_rsrc_words(dOh + (size_t)b * DG, n);
      const int at = slot * SLOT + wave * 1024;
      if constexpr (D < 64) {  // waves 0 and 1 load X, 2 and 3 dO
        i32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_readfirstlane(wave < 2 ? rx[j] : rd[j]);
        buf_load16_lds(r, so[0], at);
      } else {
#pragma unroll
        for (int k = 0; k < NPR; ++k) {
          buf_load16_lds(rx, so[k], at + k * 4096);
          buf_load16_lds(rd, so[k], at + DOO + k * 4096);
        }
      }
    };
    auto load_first = [&]() {
#pragma unroll
      for (int i = 0; i < PF; ++i) load_sub(i, i);
    };
    load_first();
    if constexpr (WREG) {
      wait_vmcnt<NLD * PF>();  // the weights' tiles (a wave's own)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        wg[k] = opWt(0, k);
        wu[k] = opWt(1, k);
      }
    }
    // row reads (row l32, columns 16 k + 8 g ..) and transposed reads (rows 16 s + 8 r + 4 g + i16 / 4, columns
    // 32 nt + 16 (G % 2) + 4 (i16 % 4) ..)
    int ro[KS], to[NTO][2];
#pragma unroll
    for (int k = 0; k < KS; ++k) ro[k] = l32 * ROWB + (((2 * k + g) ^ swz<D>(l32)) << 4);
#pragma unroll
    for (int n = 0; n < NTO; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 8 * r + 4 * g + (i16 >> 2), q = 4 * n + 2 * (G & 1) + ((i16 & 3) >> 1);
        to[n][r] = row * ROWB + ((q ^ swz<D>(row)) << 4) + ((i16 & 1) << 3);
      }
    auto opRow = [&](int base, int k) { return lds_read16(base + ro[k]); };
    auto opCol = [&](int base, int s2, int n) {
      const int a = base + s2 * 16 * ROWB;
      return cat(lds_read_tr(a + to[n][0]), lds_read_tr(a + to[n][1]));
    };
    auto weight = [&](int m, int k) -> u32x4 {
      if constexpr (WREG) return m == 0 ? wg[k] : m == 1 ? wu[k] : w2[k];
      return m == 2 ? lds_read16(W2L + wave * 32 * ROWB + ro[k]) : opWt(m, k);
    };

    f32x16 zg, zu, dh;
    float sv[16], fv[16];
    u32x4 ph[2], pg[2], pu[2];
    if (NSUB > 0) {
      wait_vmcnt<NLD*(PF > 2 ? PF - 2 : 0)>();
      barrier();
      zg = zu = dh = zero16();
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x = opRow(0, k);
        zg = mfma<BF16>(x, weight(0, k), zg);
        zu = mfma<BF16>(x, weight(1, k), zu);
        dh = mfma<BF16>(opRow(DOO, k), weight(2, k), dh);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) act_hf<ACT>(zg[e], sv[e], fv[e]);
      auto make_h = [&](int e) {
        fv[e] *= zu[e];
        if (e & 1) ph[e >> 3][(e >> 1) & 3] = pack2<BF16>(sv[e - 1] * zu[e - 1], sv[e] * zu[e]);
      };
      auto make_d = [&](int e) {
        if ((e & 1) == 0) return;
        pg[e >> 3][(e >> 1) & 3] = pack2<BF16>(dh[e - 1] * fv[e - 1], dh[e] * fv[e]);
        pu[e >> 3][(e >> 1) & 3] = pack2<BF16>(dh[e - 1] * sv[e - 1], dh[e] * sv[e]);
      };
#pragma unroll
      for (int e = 0; e < 16; ++e) make_h(e);

      // subtile i in `cur`, i + 1 in `nxt`; M: there is a subtile i + 1
      auto iter = [&](auto MORE, int cur, int nxt) {
        constexpr bool M = decltype(MORE)::value;
        constexpr int N1 = M ? KS : 0, N2 = 6 * NTO, NOPS = 3 * N1 + N2;
        const int b1 = nxt * SLOT, b2 = cur * SLOT;
        // products: G, then (s, n) of the three gradients (one operand for dWg and dWu), then U, then dH
        struct Op {
          u32x4 a, w;
        };
        auto fetch = [&](auto J) {
          constexpr int j = decltype(J)::value, i = j - N1, i2 = i - N2, i3 = i2 - N1;
          Op op;
          if constexpr (i < 0) {
            op.a = opRow(b1, j);
            if constexpr (!WREG) op.w = weight(0, j);
          } else if constexpr (i2 < 0) {
            constexpr int m = i % 3, n = i / 3 % NTO, s2 = i / 3 / NTO;
            if constexpr (m == 0) op.a = opCol(b2, s2, n);
            if constexpr (m == 2) op.a = opCol(b2 + DOO, s2, n);
          } else if constexpr (i3 < 0) {
            op.a = opRow(b1, i2);
            if constexpr (!WREG) op.w = weight(1, i2);
          } else {
            op.a = opRow(b1 + DOO, i3);
            if constexpr (!WREG) op.w = weight(2, i3);
          }
          return op;
        };
        constexpr int PD = 2;
        Op ring[PD + 1];
        static_for<PD>([&](auto J) { ring[J] = fetch(J); });
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!M) {
#pragma unroll
          for (int e = 0; e < 16; ++e) make_d(e);
        }
        u32x4 xt;  // the operand that dWg and dWu share
        static_for<NOPS>([&](auto J) {
          constexpr int j = decltype(J)::value, i = j - N1, i2 = i - N2, i3 = i2 - N1;
          const Op op = ring[j % (PD + 1)];
          if constexpr (j + PD < NOPS) ring[(j + PD) % (PD + 1)] = fetch(std::integral_constant<int, j + PD>{});
          if constexpr (i < 0) {
            zg = mfma<BF16>(op.a, WREG ? wg[WREG ? j : 0] : op.w, j == 0 ? zero16() : zg);
#pragma unroll
            for (int e = 16 * j / N1; e < 16 * (j + 1) / N1; ++e) make_d(e);
          } else if constexpr (i2 < 0) {
            constexpr int m = i % 3, n = i / 3 % NTO, s2 = i / 3 / NTO;
            if constexpr (m == 0) {
              xt = op.a;
              ag[n] = mfma<BF16>(pg[s2], xt, ag[n]);
            } else if constexpr (m == 1) {
              au[n] = mfma<BF16>(pu[s2], xt, au[n]);
            } else {
              a2[n] = mfma<BF16>(op.a, ph[s2], a2[n]);
            }
          } else if constexpr (i3 < 0) {
            zu = mfma<BF16>(op.a, WREG ? wu[WREG ? i2 : 0] : op.w, i2 == 0 ? zero16() : zu);
          } else {
            dh = mfma<BF16>(op.a, WREG ? w2[WREG ? i3 : 0] : op.w, i3 == 0 ? zero16() : dh);
#pragma unroll
            for (int e = 16 * i3 / N1; e < 16 * (i3 + 1) / N1; ++e) make_h(e);
          }
          if constexpr (M && i >= 0 && i3 < 0) {
            constexpr int NV = N2 + N1;
#pragma unroll
            for (int e = 16 * i / NV; e < 16 * (i + 1) / NV; ++e) act_hf<ACT>(zg[e], sv[e], fv[e]);
          }
          __builtin_amdgcn_sched_barrier(0);
        });
      };
      int cur = 0;
      for (int i = 0; i + 1 < NSUB; ++i) {
        const int nxt = cur + 1 == NS ? 0 : cur + 1, far = cur == 0 ? NS - 1 : cur - 1;
        load_sub(i + PF, far);
        if (e0 < E) iter(std::true_type{}, cur, nxt);  // a wave past the last column only loads
        wait_vmcnt<NLD*(PF - 2)>();  // subtile i + 2
        barrier();
        cur = nxt;
      }
      if (e0 < E) iter(std::false_type{}, cur, cur);
    }
  }
  wait_vmcnt<0>();  // subtiles past the last are still landing, as zeros

  // ---- dWg, dWu tiles: lane = row d, values along e; dW2 tiles: lane = row e, values along d ----
  if (nS > 1) {  // fp32 partials as the accumulators lie: 1 KB per store
    float4* part = (float4*)ws + ((((size_t)s * H + h) * nE + et) * 4 + wave) * (3 * NTO * 256) + lane;
#pragma unroll
    for (int m = 0; m < 3; ++m)
#pragma unroll
      for (int n = 0; n < NTO; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& t = m == 0 ? ag[n] : m == 1 ? au[n] : a2[n];
          part[((m * NTO + n) * 4 + q) * 64] = float4{t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]};
        }
    return;
  }
#pragma unroll
  for (int n = 0; n < NTO; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      ag[n][i] *= scale;
      au[n][i] *= scale;
      a2[n][i] *= scale;
    }
  // through LDS, so that rows leave as whole 16-byte pieces: 2-byte stores from the accumulators' layout took 8 of the
  // 18 us of a program with one subtile (H=32 B=4 D=128 E=1024)
  barrier();  // the ring is read
  const int area = wave * 2048 * NTO;
  auto fence = [&]() {  // the area belongs to this wave alone: its own reads and writes in order
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
  };
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int n = 0; n < NTO; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& t = m == 0 ? ag[n] : au[n];
        lds_write8(area + (n * 32 + l32) * 64 + ((q ^ ((l32 >> 2) & 3)) << 4) + g * 8,
                   u32x2{pack2<BF16>(t[4 * q], t[4 * q + 1]), pack2<BF16>(t[4 * q + 2], t[4 * q + 3])});
      }
    fence();
    u16* out = (u16*)(m == 0 ? dWg : dWu);
#pragma unroll
    for (int i = 0; i < 2 * NTO; ++i) {
      const int p = i * 64 + lane, r = p >> 2, e = e0 + ((p & 3) ^ ((r >> 2) & 3)) * 8;
      const u32x4 v = lds_read16(area + p * 16);
      if (d0 + r < DG && e < E) {
        u16* at = out + ((size_t)h * DG + d0 + r) * E + e;
        if ((E & 7) == 0) {
          *(u32x4*)at = v;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (e + j < E) at[j] = (u16)(v[j >> 1] >> (16 * (j & 1)));
        }
      }
    }
    fence();
  }
  constexpr int PW = 4 * NTO;  // pieces of a row of the dW2 tiles
#pragma unroll
  for (int n = 0; n < NTO; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lds_write8(area + l32 * (PW * 16) + (((n * 4 + q) ^ (l32 & (PW - 1))) << 4) + g * 8,
                 u32x2{pack2<BF16>(a2[n][4 * q], a2[n][4 * q + 1]), pack2<BF16>(a2[n][4 * q + 2], a2[n][4 * q + 3])});
  fence();
#pragma unroll
  for (int i = 0; i < 2 * NTO; ++i) {
    const int p = i * 64 + lane, r = p / PW, d = d0 + ((p % PW) ^ (r & (PW - 1))) * 8;
    const u32x4 v = lds_read16(area + p * 16);
    if (e0 + r < E && d < DG) *(u32x4*)((u16*)dW2 + ((size_t)h * E + e0 + r) * DG + d) = v;
  }
}

// Sum of the row splits' partials in order: four values of one accumulator a thread, along a row of the gradient.
template <bool BF16, int D, int DG>
__global__ void __launch_bounds__(256) gated_dw_reduce(const float* __restrict__ ws, u16* __restrict__ dWg,
                                                       u16* __restrict__ dWu, u16* __restrict__ dW2, int E, int nE,
                                                       long long quads, int nS, float scale) {
  constexpr Form F = dw_form(D);
  constexpr int NTO = D / 32 / F.dp;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;  // (quads is a multiple of 256)
  const float4* src = (const float4*)ws + id;
  float4 v = src[0];
  for (int s = 1; s < nS; ++s) {
    const float4 u = src[(size_t)s * quads];
    v.x += u.x;
    v.y += u.y;
    v.z += u.z;
    v.w += u.w;
  }
  const int lane = (int)(id & 63), q = (int)(id >> 6) & 3;
  long long t = id >> 8;
  const int n = (int)(t % NTO);
  t /= NTO;
  const int m = (int)(t % 3);
  t /= 3;
  const int wave = (int)(t & 3);
  t >>= 2;
  const int et = (int)(t % nE), eg = F.dp == 1 ? wave : wave & (F.ew - 1), dp = F.dp == 1 ? 0 : wave / F.ew;
  const size_t h = (size_t)(t / nE);
  const int e0 = (et * F.ew + eg) * 32, d0 = (dp * NTO + n) * 32, l32 = lane & 31, along = 8 * q + 4 * (lane >> 5);
  const u32x2 w = {pack2<BF16>(v.x * scale, v.y * scale), pack2<BF16>(v.z * scale, v.w * scale)};
  if (m == 2) {
    const int e = e0 + l32, d = d0 + along;
    if (e < E && d < DG) *(u32x2*)(dW2 + (h * E + e) * DG + d) = w;
  } else {
    const int d = d0 + l32, e = e0 + along;
    if (d >= DG || e >= E) return;
    u16* at = (m == 0 ? dWg : dWu) + (h * DG + d) * E + e;
    if ((E & 3) == 0) {
      *(u32x2*)at = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e + j < E) at[j] = (u16)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

struct Args {
  const GatedArgs& a;
  const GatedDwPlan& p;
  hipStream_t st;
};

template <bool BF16, int D, int DG, int ACT>
hipError_t launch(const Args& q) {
  auto k = gated_dw_kernel<BF16, D, DG, ACT>;
  constexpr int lds = dw_lds(D);
  static std::atomic<unsigned long long> done{0};
  hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  const GatedArgs& a = q.a;
  hipLaunchKernelGGL(k, dim3((unsigned)q.p.programs), dim3(256), lds, q.st, (const u16*)a.x, (const u16*)a.wg,
                     (const u16*)a.wu, (const u16*)a.w2, (const u16*)a.dout, a.dwg, a.dwu, a.dw2, (int)a.H, (int)a.B,
                     (int)a.E, (int)a.ldw, (long long)a.sx, (long long)a.sdo, q.p.nE, q.p.nS, q.p.rows_per_split,
                     a.dw_scale, (float*)a.ws);
  if ((e = hipGetLastError()) != hipSuccess || q.p.nS == 1) return e;
  const long long quads = (long long)a.H * q.p.nE * 4 * (3 * (D / 32 / dw_form(D).dp) * 256);
  hipLaunchKernelGGL((gated_dw_reduce<BF16, D, DG>), dim3((unsigned)(quads / 256)), dim3(256), 0, q.st, (const float*)a.ws,
                     (u16*)a.dwg, (u16*)a.dwu, (u16*)a.dw2, (int)a.E, q.p.nE, quads, q.p.nS, a.dw_scale);
  return hipGetLastError();
}
template <bool BF16, int D, int DG = D>
hipError_t by_act(const Args& q) {
  switch (q.a.act) {
    case ACT_SILU: return launch<BF16, D, DG, ACT_SILU>(q);
    case ACT_LEAKY: return launch<BF16, D, DG, ACT_LEAKY>(q);
    case ACT_SIGMOID: return launch<BF16, D, DG, ACT_SIGMOID>(q);
    default: return launch<BF16, D, DG, ACT_NONE>(q);
  }
}
template <bool BF16>
hipError_t by_d(const Args& q) {
#if FMLP_GATED_DW_PART == 128
  return by_act<BF16, 128>(q);
#else
  switch (q.a.D) {
    case 16: return by_act<BF16, 32, 16>(q);
    case 32: return by_act<BF16, 32>(q);
    case 64: return by_act<BF16, 64>(q);
    default: return by_act<BF16, 256>(q);
  }
#endif
}

}  // namespace

// Built in two parts: D = 128, whose accumulators fill half the registers, with matrix products that write vector
// registers (build.py); the others with the compiler's choice.
#if FMLP_GATED_DW_PART == 128
hipError_t launch_gated_dw128(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st) {
  const Args q{a, p, st};
  return a.io == IO_BF16 ? by_d<true>(q) : by_d<false>(q);
}
#else
GatedDwPlan gated_dw_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole) {
  const int DT = D < 32 ? 32 : (int)D;
  const Form F = dw_form(DT);
  GatedDwPlan p{};
  p.nE = (int)((E + 32 * F.ew - 1) / (32 * F.ew));
  const long long base = H * p.nE, slots = (long long)std::max(num_cus, 1) * F.oc, subs = (B + 31) / 32;
  const size_t tile_bytes = (size_t)4 * (3 * (DT / 32 / F.dp) * 256) * sizeof(float4);  // a program's partials
  // Measured: a program takes fixed_us and, for a subtile, sub_us alone on its CU or full_us on a full device (two a
  // CU at D <= 64, where they gain little on each other: vector issue is shared; one CU with two sets the time). A
  // split adds the sum's launch and the partials' bytes. H=8 B=2048 D=128 E=512: 79 us unsplit, 34 split in eight.
  const double sub_us = DT == 32 ? 0.61 : DT == 64 ? 0.86 : DT == 128 ? 1.15 : 1.35;
  const double full_us = DT == 32 ? 0.96 : DT == 64 ? 1.66 : DT == 128 ? 1.45 : 1.55;
  const double fixed_us = DT <= 64 ? 5.0 : 8.0;
  double best = 0;
  p.nS = 1;
  p.rows_per_split = (int)std::max<long long>(subs * 32, 32);
  for (long long n = 1; n <= (whole ? 1 : 64) && (n == 1 || n <= subs / 2); ++n) {
    const long long per = (subs + n - 1) / n, m = per > 0 ? (subs + per - 1) / per : 1;
    if (m != n && n > 1) continue;
    const long long full = base * n / slots, rest = base * n % slots;
    double t = (double)full * (fixed_us + full_us * (double)per);
    const double share = (double)((rest * F.oc + slots - 1) / slots) / (double)F.oc;  // of a CU's programs, the fullest's
    if (rest > 0) t += fixed_us + (double)per * std::max(sub_us, F.oc > 1 ? full_us * share : full_us * (double)rest / (double)slots);
    if (n > 1) t += 5.0 + (double)(tile_bytes * (size_t)(base * n)) * 2.0 / 6.5e6;
    if (best == 0 || t < best) {
      best = t;
      p.nS = (int)n;
      p.rows_per_split = (int)std::max<long long>(per * 32, 32);
    }
  }
  p.programs = base * p.nS;
  p.ws_bytes = p.nS > 1 ? (size_t)p.programs * tile_bytes : 0;
  return p;
}

hipError_t launch_gated_dw(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st) {
  if (p.programs <= 0) return hipSuccess;
  if (a.D == 128) return launch_gated_dw128(a, p, st);
  const Args q{a, p, st};
  return a.io == IO_BF16 ? by_d<true>(q) : by_d<false>(q);
}
#endif

}  // namespace fmlp

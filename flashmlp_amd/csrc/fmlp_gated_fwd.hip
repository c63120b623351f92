// Gated MLP forward for gfx950, 16-bit io:  O = (act(X Wg) * (X Wu)) W2  per head in one launch.
//
// A wave owns 32 rows, whose X stays in registers as the B operand of Gt = Wg^T X^T and Ut = Wu^T X^T; both
// come out with one lane per row, which is the A operand of O += h W2, so h = act(G) U (rounded to the io
// type there) never leaves registers. E is walked in chunks of 32 columns: Wg, Wu [D][32] and W2
// [D/32][32][32] land in an LDS ring by buffer loads that need no registers, and are read with
// ds_read_b64_tr_b16, which turns the row-major tiles into operands.
//
// Bound by matrix and vector issue: a chunk has D/4 products (32 clocks each, D / 16 for G and for U, D / 16
// for O) and 16 activations a lane. One wave carries three phases per chunk, each step one product and
// its share of vector work, so that neither waits for the other:
//     G(c+1) products  | h(c) = s(c) U(c), packed            s = act(G)
//     O += h(c) W2(c)  | s(c+1), first part
//     U(c+1) products  | s(c+1), the rest
// which keeps 56 values of state instead of the 80 that whole chunks in flight would take: two waves a SIMD
// fit at D = 128 (three at D = 64, one at D = 256).
//
// Measured (bf16 SiLU): H=32 B=16384 D=128 E=1024 393 us, 1049 TFLOP/s, products 54 % and vector instructions 47 % of
// the SIMDs' cycles at 1.86 GHz: they take turns, and the card is at its power limit. Forms with the operands read
// three or four products ahead, or with 64 rows a wave (half the LDS reads), measured the same.
//
// Grids that leave CUs idle split E: over ES sets of NW waves of a workgroup (each walks its own chunks through
// a ring of its own; the partial tiles are added through LDS in order), and over xs workgroups, whose fp32
// partial tiles go through the workspace and are added in order by a second launch.
#include <algorithm>
#include <type_traits>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

// D: tile width (32 to 256); DG: columns in memory (D, or 16 with D = 32); NW waves (32 rows each) per E part; ES
// parts; NS ring slots; OC waves per SIMD
template <bool BF16, int D, int DG, int ACT, int NW, int ES, int NS, int OC>
__global__ void __launch_bounds__(NW * ES * 64) __attribute__((amdgpu_waves_per_eu(OC, OC)))
gated_fwd_kernel(const u16* __restrict__ X, const u16* __restrict__ Wg, const u16* __restrict__ Wu,
                 const u16* __restrict__ W2, void* __restrict__ O, int B, int E, int ldw, long long sx, int H, int T,
                 int xs, int nct, int outf32, float* __restrict__ ws) {
  constexpr int NT = NW * 64, KS = DG / 16, NTN = D / 32, NPR = 4 * D / NT, NLD = 3 * NPR;
  constexpr int SLOT = 192 * D, WU = 64 * D, W2O = 128 * D, PF = NS - 1;
  // D = 256 runs lone waves: a chunk's loads stand one by one between products, which hides their address work
  // (H=8 B=8192 E=1024 bf16 122 -> 119 us); short chunks lose by the later issue (D = 32, a wave alone: 6.1 -> 6.8 us)
  constexpr bool SPREAD = D == 256;
  static_assert(NPR * NT == 4 * D && NS >= 3 && NLD * (PF - 2) < 64, "chunk loads");
  const int lane = threadIdx.x & 63;
  const int part = ES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  const int tid = threadIdx.x - part * NT;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = lane >> 4, i16 = lane & 15, g = lane >> 5, l32 = lane & 31;

  // this workgroup's rows and its chunks [cb, ce); this part's are c0 .. c0 + NC - 1, zeros past c1
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
  const u16* Wgh = Wg + (size_t)h * DG * ldw;
  const u16* Wuh = Wu + (size_t)h * DG * ldw;
  const u16* W2h = W2 + (size_t)h * E * DG;
  const int b_wave = (bt * NW + wave) * 32;

  // chunk loads: piece p (16 bytes) of Wg and Wu is row p / 4, columns 8 (p % 4) ..; of W2 block p / 128, row
  // (p / 4) % 32, the same columns. Columns past E and chunks past the last land as zeros.
  int colq[NPR];
  unsigned o1[NPR], o2[NPR];
#pragma unroll
  for (int k = 0; k < NPR; ++k) {
    const unsigned p = (unsigned)(tid + k * NT);
    colq[k] = (int)(p & 3u) * 8;
    o1[k] = (p >> 2) * (unsigned)ldw * 2u + (p & 3u) * 16u;
    o2[k] = ((p >> 2) & 31u) * (DG * 2u) + (p >> 7) * 64u + (p & 3u) * 16u;
    if (DG < D) {
      if ((p >> 2) >= (unsigned)DG) o1[k] = BUF_OOB;
      if ((p & 3u) * 8u >= (unsigned)DG) o2[k] = BUF_OOB;
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
  // at most N of this wave's loads in flight; a part of one wave reads nothing that others load
  auto sync = [&](auto N) {
    wait_vmcnt<decltype(N)::value>();
    if constexpr (NW > 1) {
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
    }
    asm volatile("" ::: "memory");
  };

  u32x4 xr[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int b = b_wave + l32;
    xr[k] = u32x4{0u, 0u, 0u, 0u};
    if (b < B) xr[k] = *(const u32x4*)(Xh + (size_t)b * DG + k * 16 + g * 8);
  }
#pragma unroll
  for (int c = 0; c < PF; ++c) load_chunk(c, c);

  // operand addresses of the transposed reads (16-lane group G, lane i16: row i16 / 4, columns 4 (i16 % 4) ..)
  const int laneA = (8 * g + (i16 >> 2)) * 64 + 32 * (G & 1) + 8 * (i16 & 3);
  const int laneB = W2O + (4 * g + (i16 >> 2)) * 64 + 32 * (G & 1) + 8 * (i16 & 3);
  auto opA = [&](int base, int k) { return cat(lds_read_tr(base + laneA + k * 1024), lds_read_tr(base + laneA + k * 1024 + 256)); };
  auto opB = [&](int base, int s, int nt) {
    const int a = base + laneB + nt * 2048 + s * 1024;
    return cat(lds_read_tr(a), lds_read_tr(a + 512));
  };

  f32x16 o[NTN], zg, zu;
  float sv[16];
  u32x4 h0, h1;
#pragma unroll
  for (int nt = 0; nt < NTN; ++nt) o[nt] = zero16();

  sync(std::integral_constant<int, NLD*(PF > 2 ? PF - 2 : 0)>{});  // chunks 0 and 1 (0 alone would do)
  zg = zu = zero16();
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    zg = mfma<BF16>(opA(RB, k), xr[k], zg);
    zu = mfma<BF16>(opA(RB + WU, k), xr[k], zu);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) sv[e] = act_f<ACT>(zg[e]);

  // chunk c in `cur`, chunk c + 1 in `nxt`; more: there is a chunk c + 1
  auto iter = [&](auto MORE, int c, int cur, int nxt, int far) {
    constexpr bool M = decltype(MORE)::value;
    Dst dst;
    if constexpr (M && SPREAD) dst = chunk_at(c + PF, far);
    constexpr int N1 = M ? KS : 0, N2 = 2 * NTN, NOPS = 2 * N1 + N2;
    const int b1 = RB + nxt * SLOT, b2 = RB + cur * SLOT;
    auto fetch = [&](int j) {
      if (j < N1) return opA(b1, j);
      if (j < N1 + N2) return opB(b2, (j - N1) / NTN, (j - N1) % NTN);
      return opA(b1 + WU, j - N1 - N2);
    };
    constexpr int PD = 2;  // operands are read two products ahead
    u32x4 ring[PD + 1];
#pragma unroll
    for (int j = 0; j < PD; ++j) ring[j] = fetch(j);
    __builtin_amdgcn_sched_barrier(0);
    // h(c): while G(c + 1) is computed, or before the last products
    auto make_h = [&](int e) {
      if ((e & 1) == 0) return;
      const unsigned pk = pack2<BF16>(sv[e - 1] * zu[e - 1], sv[e] * zu[e]);
      if (e < 8) h0[(e >> 1) & 3] = pk;
      else h1[(e >> 1) & 3] = pk;
    };
    if constexpr (!M) {
#pragma unroll
      for (int e = 0; e < 16; ++e) make_h(e);
    }
#pragma unroll
    for (int j = 0; j < NOPS; ++j) {
      const u32x4 op = ring[j % (PD + 1)];
      if (j + PD < NOPS) ring[(j + PD) % (PD + 1)] = fetch(j + PD);
      if (j < N1) {
        zg = mfma<BF16>(op, xr[j], j == 0 ? zero16() : zg);
#pragma unroll
        for (int e = 16 * j / (N1 > 0 ? N1 : 1); e < 16 * (j + 1) / (N1 > 0 ? N1 : 1); ++e) make_h(e);
      } else {
        if (j < N1 + N2) {
          const int s = (j - N1) / NTN, nt = (j - N1) % NTN;
          o[nt] = mfma<BF16>(s == 0 ? h0 : h1, op, o[nt]);
        } else {
          const int k = j - N1 - N2;
          zu = mfma<BF16>(op, xr[k], k == 0 ? zero16() : zu);
        }
        if constexpr (M) {
          constexpr int NV = N1 + N2;
#pragma unroll
          for (int e = 16 * (j - N1) / NV; e < 16 * (j - N1 + 1) / NV; ++e) sv[e] = act_f<ACT>(zg[e]);
        }
      }
      if (M && SPREAD && j < NLD) load_piece(dst, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int cur = 0;
  for (int c = 0; c + 1 < NC; ++c) {
    const int nxt = cur + 1 == NS ? 0 : cur + 1, far = cur == 0 ? NS - 1 : cur - 1;
    if (!SPREAD || b_wave >= B) load_chunk(c + PF, far);
    // (chunk c + 1 landed before the last barrier; a wave without rows only loads)
    if (b_wave < B) iter(std::true_type{}, c, cur, nxt, far);
    sync(std::integral_constant<int, NLD*(PF - 2)>{});  // chunk c + 2
    cur = nxt;
  }
  if (b_wave < B) iter(std::false_type{}, 0, cur, cur, cur);

  if constexpr (ES > 1) {
    wait_vmcnt<0>();  // chunks past the last are still landing, as zeros
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
  } else {
    wait_vmcnt<0>();
  }
  if (xs > 1)
    store_rows<BF16, D, DG>(o, ws, (size_t)blockIdx.x * (NW * 32) * DG, B - bt * NW * 32, wave * 32, g, l32, 1);
  else
    store_rows<BF16, D, DG>(o, O, (size_t)h * B * DG, B, b_wave, g, l32, outf32);
}

struct Args {
  const GatedArgs& a;
  const GatedFwdPlan& p;
  hipStream_t st;
};

template <bool BF16, int D, int DG, int ACT, int FORM>
hipError_t launch(const Args& q) {
  constexpr GatedForm F = gated_form(D, FORM, false);
  static_assert(gated_form_fits(D, F), "the plan's workgroups a CU");
  constexpr int lds = F.es * F.ns * 192 * D;
  auto k = gated_fwd_kernel<BF16, D, DG, ACT, F.nw, F.es, F.ns, F.oc>;
  static std::atomic<unsigned long long> done{0};
  hipError_t e = set_lds_once((const void*)k, lds, done);
  if (e != hipSuccess) return e;
  const GatedArgs& a = q.a;
  const long long grid = q.p.tiles * q.p.xs;
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * F.nw * F.es), lds, q.st, (const u16*)a.x, (const u16*)a.wg,
                     (const u16*)a.wu, (const u16*)a.w2, a.o, (int)a.B, (int)a.E, (int)a.ldw, (long long)a.sx, (int)a.H,
                     (int)(q.p.tiles / a.H), q.p.xs, q.p.nct, a.out_f32, (float*)a.ws);
  if ((e = hipGetLastError()) != hipSuccess || q.p.xs == 1) return e;
  return launch_tile_reduce((const float*)a.ws, a.o, BF16, (int)a.B, DG, 32 * F.nw, (int)a.H, (int)(q.p.tiles / a.H),
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

GatedFwdPlan gated_fwd_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool dx, bool whole) {
  const int DT = D < 32 ? 32 : (int)D;
  const long long N = num_cus > 0 ? num_cus : 1, nch = (E + 31) / 32;
  GatedFwdPlan best{};
  double best_us = 0;
  for (int form = 0; form < 3; ++form) {
    const GatedForm F = gated_form(DT, form, dx);
    if (F.nw == 0) continue;
    const long long tiles = H * ((B + 32 * F.nw - 1) / (32 * F.nw));
    for (long long want = 1; want <= (whole ? 1 : 16) && want <= nch; ++want) {
      const long long nct = (nch + want - 1) / want, xs = (nch + nct - 1) / nct;
      if (xs != want) continue;
      // full rounds of F.per_cu workgroups a CU, and what is left; a split adds a launch and the partials' bytes
      const long long slots = N * F.per_cu, full = tiles * xs / slots, rest = tiles * xs % slots;
      const double steps = (dx ? 1.4 : 1.0) * (double)((nct + F.es - 1) / F.es);
      double us = (double)full * (F.fixed_us + F.full_us * steps);
      const double share = F.per_cu == 1 ? (double)rest / (double)slots : (double)((rest + N - 1) / N) / (double)F.per_cu;
      if (rest > 0) us += F.fixed_us + steps * std::max(F.chunk_us, F.full_us * share);
      if (xs > 1) us += 2.8 + (double)(H * B * D * xs) * 8.0 / 4.8e6;
      if (best_us == 0 || us < best_us) {
        best_us = us;
        best.form = form;
        best.tiles = tiles;
        best.xs = (int)xs;
        best.nct = (int)nct;
        best.ws_bytes = xs > 1 ? (size_t)(tiles * xs) * 32 * F.nw * D * sizeof(float) : 0;
      }
    }
  }
  return best;
}

hipError_t launch_gated_fwd(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st) {
  if (p.tiles <= 0) return hipSuccess;
  const Args q{a, p, st};
  return a.io == IO_BF16 ? by_d<true>(q) : by_d<false>(q);
}

}  // namespace fmlp

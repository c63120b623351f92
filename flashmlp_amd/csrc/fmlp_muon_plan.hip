// Host side of the orthogonalised updates: which kernels take a call's stacks of matrices, the workspace they share and the scales of
// their terms.
#include <algorithm>
#include <cmath>
#include <vector>

#include "fmlp_muon.h"

namespace fmlp {
namespace {

int padded(const MuonTensor& t) {
  const int n = std::min(t.R, t.C);
  return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256;
}
MuonKind kind_of(const MuonTensor& t) {
  const bool raw = t.m == nullptr && t.x_io != IO_F32;
  const auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool vec = t.C % 8 == 0 && (long long)t.R * t.C < 1LL << 29 && whole(t.x) && whole(t.m) && whole(t.out);
  return MuonKind{raw ? 1 : 3, !raw || t.x_io == IO_BF16, vec};
}

// The matrices of one padded size: their Gram matrices and what comes of them go through the workspace together.
struct Group {
  int NP;
  long long matrices, tiles;  // tiles: of the longest one
  bool momentum, raw;  // a matrix has a momentum; all are of 16 bits and have none
  bool whole;  // a workgroup a matrix from end to end: no workspace
  bool by_tiles;  // of the Gram matrices
  int gram_parts, apply_parts;
  size_t g_off, p_off, info_off, iter_off, end;
};
Group group_of(int NP, int n, const MuonTensor* t, int cus) {
  Group r{};
  r.NP = NP;
  r.raw = true;
  const int KT = NP == 256 ? 32 : 8192 / NP;
  for (int i = 0; i < n; ++i)
    if (t[i].H > 0 && t[i].R > 0 && t[i].C > 0 && padded(t[i]) == NP) {
      r.matrices += t[i].H;
      r.momentum |= t[i].m != nullptr;
      r.raw &= kind_of(t[i]).terms == 1;
      r.tiles = std::max(r.tiles, ((long long)std::max(t[i].R, t[i].C) + KT - 1) / KT);
    }
  if (r.matrices == 0) return r;
  // Below about a matrix for each CU (NP = 128) or three for two, CUs idle that parts of matrices would fill. Muon step in fp32 whole
  // and in parts: 128 x 1024, 128 matrices 198 and 176 us, 256 251 and 279, 512 443 and 477, 768 664 and 785; 64 x 768,
  // 256 matrices 81 and 80 us, 384 99 and 108, 512 113 and 135
  r.whole = NP <= 128 && 2 * r.matrices >= (NP == 128 ? 2 : 3) * cus;
  if (r.whole) return r;
  if (NP < 256) {
    // Three workgroups a CU at least, as far as there are tiles. Of Gram matrices no more than pay: a tile takes about 3 us (16-bit
    // values as they are 1.5), and of a part's sums each matrix's are read by one workgroup of the steps (about 40 KB a us; 16
    // matrices of 128 x 1024 in 10 parts 11 us and 18 for the reading)
    const long long want = (3LL * cus + r.matrices - 1) / r.matrices;
    const long long pays = std::max(1LL, std::llround(std::sqrt((double)r.tiles * (r.raw ? 1.5 : 3) / (NP * NP * 4 / 4e4))));
    r.gram_parts = (int)std::max(1LL, std::min(std::min(want, pays), r.tiles));
    r.apply_parts = (int)std::max(1LL, std::min(want, r.tiles));
  } else {
    // A workgroup a CU at a time, so whole rounds of them: the number with the least of rounds, tiles (5 us) and, for Gram
    // matrices, the parts' sums (written and read at about 4 TB/s), for results the reading of P. (Three a CU for results and
    // the square root for Gram matrices, as above: 64 matrices of 256 x 1024 fp32 438 us, Muon step 376; so 375 and 335)
    const auto best = [&](double fixed_us, double part_us) {
      long long at = 1;
      double least = 1e300;
      for (long long p = 1; p <= std::min(r.tiles, std::max(1LL, 3LL * cus / r.matrices)); ++p) {
        const double us = (double)((r.matrices * p + cus - 1) / cus) * (fixed_us + 5.0 * ((r.tiles + p - 1) / p)) + part_us * p;
        if (us < least) least = us, at = p;
      }
      return (int)at;
    };
    r.gram_parts = best(3, (double)r.matrices * NP * NP * 8 / 4e6);
    r.apply_parts = best(4, 0);
  }
  // Few Gram matrices of 256 by tiles: fewer parts and sums to pass on, but every value is brought into terms four times (not so
  // 16-bit ones, which are their own), and m' takes a launch. Whole and by tiles, 256 x 1024: fp32 orthogonalised, 8 matrices 146 and
  // 104 us, 16 173 and 171, 32 266 and 277; bf16, 8 104 and 76, 64 260 and 257, 128 477 and 481; the Muon step, 8 116 and
  // 98, 16 139 and 146
  if (NP == 256 && r.matrices <= (r.raw ? cus / 2 : r.momentum ? cus / 32 : cus / 20)) {
    const long long fill = cus / (r.matrices * kMuonGramTiles), blocks = (r.tiles + 1) / 2;  // (64 columns)
    r.by_tiles = true;
    r.gram_parts = (int)std::max(1LL, std::min(fill, blocks));
  }
  // as many as have tiles where each takes as many as the first: 16 tiles in 5 parts are 4, 4, 4, 4 and none
  const auto even = [](long long tiles, int parts) {
    const long long each = (tiles + parts - 1) / parts;
    return (int)((tiles + each - 1) / each);
  };
  r.gram_parts = even(r.by_tiles ? (r.tiles + 1) / 2 : r.tiles, r.gram_parts);
  r.apply_parts = even(r.tiles, r.apply_parts);
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  r.p_off = up((size_t)r.matrices * r.gram_parts * NP * NP * 4);
  r.info_off = r.p_off + up((size_t)r.matrices * NP * NP * 4);
  r.iter_off = r.info_off + up((size_t)r.matrices * sizeof(MuonInfo));
  r.end = r.iter_off + up(muon_iter_ws_bytes(NP, r.matrices));
  return r;
}
constexpr int kSizes[4] = {32, 64, 128, 256};

// Powers of two that bring a stage's values to at most 2^14 as fp16, a quarter of its range: G's, Q's and P's elements are at most
// their largest eigenvalues. What is 2^-16 of such a bound still has 22 bits, what is below an error of 2^-39 of it.
void set_steps(MuonSteps* s, const MuonCall& c, int first, int steps, bool normalise) {
  s->steps = steps;
  s->normalise = normalise;
  s->eps = c.eps;
  double p = 1;
  const auto scale = [](double bound) {
    int e = 0;
    (void)std::frexp(std::max(bound, 0x1p-32), &e);  // (products of scales stay within fp32)
    return std::ldexp(1.f, 14 - e);
  };
  for (int k = 0; k < steps; ++k) {
    s->a[k] = c.abc[first + k][0];
    s->b[k] = c.abc[first + k][1];
    s->c[k] = c.abc[first + k][2];
    p *= c.q[first + k];
    s->g_scale[k] = scale(c.range[first + k]);
    s->q_scale[k] = scale(c.q[first + k]);
    s->p_scale[k] = scale(p);
  }
}

bool empty(const MuonTensor& t) { return t.H == 0 || t.R == 0 || t.C == 0; }

// A stage's tensors of one padded size: what it reads and writes of each, and the number of the first matrix.
struct Item {
  MuonTensor t;
  MuonKind kind;
  long long matrix0;
};

// f(kind, table, workgroups) for tables of items of one kind, `parts` workgroups a matrix, and no more of 512 threads than a launch
// holds
template <typename F>
hipError_t for_tables(const std::vector<Item>& items, int parts, bool any_type, F f) {
  for (int code = 0; code < 8; ++code) {  // (kinds in a fixed order)
    const MuonKind k{code & 1 ? 3 : 1, (code & 2) != 0, (code & 4) != 0};
    MuonTable tab{};
    long long blocks = 0;
    for (size_t i = 0; i <= items.size(); ++i) {
      const bool end = i == items.size();
      const Item* it = end ? nullptr : &items[i];
      if (!end && !(it->kind.terms == k.terms && (any_type || it->kind.bf == k.bf) && it->kind.vec == k.vec)) continue;
      if (!end && any_type && !k.bf) continue;  // (both 16-bit types at once)
      const long long b = end ? 0 : it->t.H * parts;
      constexpr long long most = kLaunchThreads / 512;
      if (b > most) return hipErrorInvalidValue;
      if (tab.n > 0 && (end || tab.n == kMuonTable || blocks + b > most)) {
        const hipError_t e = f(k, tab, (unsigned)blocks);
        if (e != hipSuccess) return e;
        tab.n = 0;
        blocks = 0;
      }
      if (end) break;
      const MuonTensor& t = it->t;
      tab.t[tab.n++] = MuonRef{t.x, t.m, t.out, t.R, t.C, (unsigned)blocks, (unsigned)it->matrix0, t.lr,
                               (unsigned char)t.x_io, (unsigned char)t.m_io, (unsigned char)t.out_io, 0};
      blocks += b;
    }
  }
  return hipSuccess;
}

size_t between_bytes(const MuonTensor& t, const MuonCall& c) {
  // matrices between stages are in fp32: in the result where that is what it is
  if (c.stages <= 1 || (!c.update && t.out_io == IO_F32)) return 0;
  return ((size_t)t.H * t.R * t.C * 4 + 255) / 256 * 256;
}

// The call's stacks of one padded size, or runs of a stack's matrices, that go through the workspace together.
struct Batch {
  std::vector<MuonTensor> t;
  Group g;
  size_t between, end;  // bytes before the matrices between stages, and of it all
};
// In even batches of 1024 matrices of 256 at most, whose Gram matrices and P are 512 MB (a Muon step of 2048 of
// 256 x 300 takes 7.6 ms, at once 7.6; of 4096 15.2 and 15.1); of as many of the others as have a launch of a workgroup each.
constexpr long long kBatch256 = 1024, kBatch = kLaunchThreads / 512;
std::vector<Batch> batches_of(int NP, int n, const MuonTensor* t, const MuonCall& c, int cus) {
  long long matrices = 0;
  for (int i = 0; i < n; ++i)
    if (!empty(t[i]) && padded(t[i]) == NP) matrices += t[i].H;
  std::vector<Batch> out;
  if (matrices == 0) return out;
  const long long most = NP == 256 ? kBatch256 : kBatch, number = (matrices + most - 1) / most, each = (matrices + number - 1) / number;
  long long room = 0;
  for (int i = 0; i < n; ++i) {
    if (empty(t[i]) || padded(t[i]) != NP) continue;
    const auto bytes = [](int io) { return io == IO_F32 ? 4 : 2; };
    for (long long h = 0; h < t[i].H;) {
      if (room == 0) {
        out.emplace_back();
        room = each;
      }
      MuonTensor v = t[i];
      v.H = std::min(t[i].H - h, room);
      const size_t at = (size_t)h * t[i].R * t[i].C;
      v.x = (const char*)v.x + at * bytes(v.x_io);
      if (v.m != nullptr) v.m = (char*)v.m + at * bytes(v.m_io);
      v.out = (char*)v.out + at * bytes(v.out_io);
      v.between = out.back().between;
      out.back().between += between_bytes(v, c);
      out.back().t.push_back(v);
      h += v.H;
      room -= v.H;
    }
  }
  for (Batch& b : out) {
    b.g = group_of(NP, (int)b.t.size(), b.t.data(), cus);
    b.end = b.g.end + b.between;
    b.between = b.g.end;
  }
  return out;
}

}  // namespace

// The eigenvalues of the first G are in [0, 1], those after a step in [0, r'], r' the largest l q(l)^2 on [0, r]: at an end or
// where its derivative q (a + 3 b l + 5 c l^2) vanishes. (Taken where they are: with two hundredths more a step, a schedule whose
// polynomials grow fast behind r had bounds of 1e11 after four steps, and its values vanished below them.)
void muon_bounds(MuonCall* c) {
  double r = 1;
  c->range[0] = r;
  for (int k = 0; k < c->steps; ++k) {
    const double a = c->abc[k][0], b = c->abc[k][1], d = c->abc[k][2];
    const auto q = [&](double l) { return a + l * (b + l * d); };
    double most = std::max(std::fabs(q(0)), std::fabs(q(r))), next = r * q(r) * q(r);
    const auto at = [&](double l) {
      if (!(l > 0 && l < r)) return;
      most = std::max(most, std::fabs(q(l)));
      next = std::max(next, l * q(l) * q(l));
    };
    if (d != 0) {
      const double root = std::sqrt(std::max(9 * b * b - 20 * a * d, 0.0));
      at(-b / (2 * d));
      at((-3 * b + root) / (10 * d));
      at((-3 * b - root) / (10 * d));
    } else if (b != 0) {
      at(-a / (3 * b));
    }
    c->q[k] = most;
    c->range[k + 1] = r = next;
  }
}

MuonPlan muon_plan(int n, const MuonTensor* t, const MuonCall& c, int num_cus) {
  MuonPlan p{};
  for (int NP : kSizes)
    for (const Batch& b : batches_of(NP, n, t, c, num_cus)) p.ws_bytes = std::max(p.ws_bytes, b.end);
  return p;
}

static hipError_t launch_batch(int NP, const Batch& b, const MuonCall& c, void* ws, hipStream_t st) {
  const Group& gr = b.g;
  float* G = (float*)ws;
  unsigned short* P = (unsigned short*)((char*)ws + gr.p_off);
  MuonInfo* info = (MuonInfo*)((char*)ws + gr.info_off);
  for (int stage = 0; stage < c.stages; ++stage) {
    const int first = c.first[stage], steps = c.first[stage + 1] - first;
    const bool start = stage == 0, last = stage + 1 == c.stages;
    const int update = c.update && last;
    MuonSteps s{};
    set_steps(&s, c, first, steps, start);
    std::vector<Item> items;
    long long matrix = 0;
    for (MuonTensor v : b.t) {
      void* y = between_bytes(v, c) ? (void*)((char*)ws + b.between + v.between) : v.out;
      if (!start) {
        v.x = y;
        v.m = nullptr;
        v.x_io = IO_F32;
      }
      if (!last) {
        v.out = y;
        v.out_io = IO_F32;
      }
      items.push_back(Item{v, kind_of(v), matrix});
      matrix += v.H;
    }
    hipError_t e;
    if (gr.whole) {
      e = for_tables(items, 1, false, [&](const MuonKind& k, const MuonTable& tab, unsigned blocks) {
        return NP == 32   ? muon_whole<32>(k, tab, blocks, s, c, update, st)
               : NP == 64 ? muon_whole<64>(k, tab, blocks, s, c, update, st)
                          : muon_whole<128>(k, tab, blocks, s, c, update, st);
      });
      if (e != hipSuccess) return e;
      continue;
    }
    e = hipSuccess;
    if (gr.by_tiles) {
      // (all have a momentum, or none has)
      if (items[0].t.m != nullptr)
        e = for_tables(items, gr.apply_parts, false, [&](const MuonKind& k, const MuonTable& tab, unsigned blocks) {
          return muon_momentum(k, tab, blocks, gr.apply_parts, c, st);
        });
      if (e == hipSuccess)
        e = for_tables(items, kMuonGramTiles * gr.gram_parts, false, [&](const MuonKind& k, const MuonTable& tab, unsigned blocks) {
          return muon_gram_tiles(k, tab, blocks, G, gr.gram_parts, c, st);
        });
    }
    else e = for_tables(items, gr.gram_parts, false, [&](const MuonKind& k, const MuonTable& tab, unsigned blocks) {
      return NP == 32    ? muon_gram<32>(k, tab, blocks, G, gr.gram_parts, c, st)
             : NP == 64  ? muon_gram<64>(k, tab, blocks, G, gr.gram_parts, c, st)
             : NP == 128 ? muon_gram<128>(k, tab, blocks, G, gr.gram_parts, c, st)
                         : muon_gram<256>(k, tab, blocks, G, gr.gram_parts, c, st);
    });
    if (e == hipSuccess) e = launch_muon_iter(NP, gr.matrices, G, gr.gram_parts, P, info, s, (char*)ws + gr.iter_off, st);
    if (e == hipSuccess)
      e = for_tables(items, gr.apply_parts, true, [&](const MuonKind& k, const MuonTable& tab, unsigned blocks) {
        return NP == 32    ? muon_apply<32>(k, tab, blocks, P, info, gr.apply_parts, c, update, st)
               : NP == 64  ? muon_apply<64>(k, tab, blocks, P, info, gr.apply_parts, c, update, st)
               : NP == 128 ? muon_apply<128>(k, tab, blocks, P, info, gr.apply_parts, c, update, st)
                           : muon_apply<256>(k, tab, blocks, P, info, gr.apply_parts, c, update, st);
      });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_muon(int n, const MuonTensor* t, const MuonCall& c, int num_cus, void* ws, hipStream_t st) {
  for (int NP : kSizes)
    for (const Batch& b : batches_of(NP, n, t, c, num_cus)) {
      const hipError_t e = launch_batch(NP, b, c, ws, st);
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}

}  // namespace fmlp

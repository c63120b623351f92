// Host-side launch descriptors of the orthogonalised updates (fmlp_muon.hip, fmlp_muon_iter.hip).
#pragma once
#include "fmlp_launch.h"

namespace fmlp {

constexpr int kMuonMaxSmall = 256;  // the smaller side of a matrix
constexpr int kMuonMaxSteps = 10;

// A stack of H matrices R x C, dense. x (and, with a momentum, m) are read; out is written: the orthogonalised matrices,
// or with `update` the weights.
struct MuonTensor {
  const void* x;
  void* m;    // momentum, or null
  void* out;
  long long H;
  int R, C;
  int x_io, m_io, out_io;  // IoType
  float lr;                // update: keep out - lr O
  size_t between;          // launch_muon: where its matrices are between stages
};

// What a call does with every tensor: u = x, or with momenta m' = mu m + nu x, u = m' or (nesterov) nu x + mu m';
// X = u / (|u| + eps); q(l) = a + b l + c l^2 for each step.
struct MuonCall {
  float mu, nu, keep;
  int nesterov, update;
  float eps;
  int steps;
  float abc[kMuonMaxSteps][3];
  int stages;                    // of steps taken on one Gram matrix
  int first[kMuonMaxSteps + 1];  // their first steps, then `steps`
  // largest eigenvalue of G before each step and after the last one, largest |q| of each step (muon_bounds)
  double range[kMuonMaxSteps + 1], q[kMuonMaxSteps];
};
// Sets range and q from the steps' polynomials.
void muon_bounds(MuonCall* c);

// Bytes of workspace and where things are in it, for the call's tensors.
struct MuonPlan {
  size_t ws_bytes;
};
MuonPlan muon_plan(int n, const MuonTensor* t, const MuonCall& c, int num_cus);
hipError_t launch_muon(int n, const MuonTensor* t, const MuonCall& c, int num_cus, void* ws, hipStream_t st);

// ---- between the two translation units ----
// Steps on NP x NP Gram matrices, NP 32 to 256: G (`parts` partial sums each, fp32, whole and symmetric) to P, the product
// of the steps' polynomials, as two fp16 terms times p_scale ([NP][NP] first terms, then second ones, a matrix after the
// other), and for each matrix info = {scale of the values u for fp16 terms, factor of the products}.
struct MuonSteps {
  int steps;
  float a[kMuonMaxSteps], b[kMuonMaxSteps], c[kMuonMaxSteps];
  float g_scale[kMuonMaxSteps], q_scale[kMuonMaxSteps], p_scale[kMuonMaxSteps];  // powers of two, for fp16 terms
  int normalise;
  float eps;
};
struct MuonInfo {
  float u_scale, factor;
};
// Tensors of a launch, in its arguments.
constexpr int kMuonTable = 76;
struct MuonRef {
  const void* x;
  void* m;
  void* out;
  int R, C;
  unsigned block0, matrix0;  // the tensor's first workgroup and matrix
  float lr;
  unsigned char x_io, m_io, out_io, pad;
};
struct MuonTable {
  MuonRef t[kMuonTable];
  int n;
};
static_assert(sizeof(MuonTable) <= 3712, "kernel arguments");
// What decides a tensor's kernels beside its padded small side: the terms and type of its Gram matrix's operands (1: 16-bit values as
// they are, 3: bf16 terms of 32-bit ones), and whether its rows are whole 16-byte vectors.
struct MuonKind {
  int terms;
  bool bf, vec;
};
// `parts` workgroups a matrix: partial Gram matrices (and m'); the result from P; all of it by one workgroup a matrix
// (NP <= 128)
template <int NP>
hipError_t muon_gram(const MuonKind& kind, const MuonTable& tab, unsigned blocks, float* G, int parts, const MuonCall& c, hipStream_t st);
// NP = 256: the same with `parts` workgroups for each of a matrix's kMuonGramTiles tiles, m' being there already, and m' alone
constexpr int kMuonGramTiles = 10;
hipError_t muon_gram_tiles(const MuonKind& kind, const MuonTable& tab, unsigned blocks, float* G, int parts, const MuonCall& c,
                           hipStream_t st);
hipError_t muon_momentum(const MuonKind& kind, const MuonTable& tab, unsigned blocks, int parts, const MuonCall& c, hipStream_t st);
template <int NP>
hipError_t muon_apply(const MuonKind& kind, const MuonTable& tab, unsigned blocks, const unsigned short* P, const MuonInfo* info,
                      int parts, const MuonCall& c, int update, hipStream_t st);
template <int NP>
hipError_t muon_whole(const MuonKind& kind, const MuonTable& tab, unsigned blocks, const MuonSteps& s, const MuonCall& c, int update,
                      hipStream_t st);

size_t muon_iter_ws_bytes(int NP, long long matrices);
hipError_t launch_muon_iter(int NP, long long matrices, const float* G, int parts, unsigned short* P, MuonInfo* info,
                            const MuonSteps& s, void* ws, hipStream_t st);

}  // namespace fmlp

// Host-side launch descriptors of the experts' operators: routing, the plan of a sort by expert, and the copies
// between tokens and experts' rows.
#pragma once
#include "fmlp_launch.h"

namespace fmlp {

constexpr int64_t kMaxExperts = 1024;  // the plan's counters of a workgroup's waves stay within LDS
constexpr int64_t kMaxChoices = 32;    // of a token: the choices of a workgroup's rows go through LDS

struct RouteArgs {
  const void* logits;  // (T, N), rows `stride` elements apart
  float* weights;      // (T, k)
  int32_t* experts;    // (T, k)
  const float* dweights;  // backward: (T, k)
  void* dlogits;          // backward: (T, N) dense
  long long T, stride;
  int N, k, normalize, io;
};
hipError_t launch_route_fwd(const RouteArgs& a, hipStream_t st);
hipError_t launch_route_bwd(const RouteArgs& a, hipStream_t st);

// The sort of M assignments by expert: chunks of `threads` times `items` assignments, a workgroup each; with more than one, their
// histograms ([chunks][N]) take ws_bytes. scan: these are summed up in a launch of its own.
struct ExpertPlan {
  long long chunks;
  int threads, items;
  bool scan;
  size_t ws_bytes;
};
ExpertPlan expert_plan(int64_t M, int64_t N);
hipError_t launch_expert_plan(const void* experts, bool wide, long long M, int N, long long capacity, int32_t* slots,
                              int32_t* counts, const ExpertPlan& p, void* ws, hipStream_t st);

// Tokens (T, D) and experts' rows (N, capacity, D); slots (T, k): the row of each assignment, -1 for none.
struct ExpertCopyArgs {
  const void* x;         // tokens that are read, rows `stride` elements apart
  const void* rows_in;   // experts' rows that are read
  void* rows_out;        // experts' rows that are written, or null
  void* o;               // tokens that are written
  const float* weights;  // (T, k), or null: ones
  float* dweights;       // (T, k), or null
  const int32_t* slots;
  const int32_t* counts;  // (N): assignments of each expert; rows behind them are zeros
  long long T, N, capacity, D, stride;
  int k, io;
};
// rows_out[slot] = weight x, zeros behind; dweights = <rows_in[slot], x>
hipError_t launch_expert_scatter(const ExpertCopyArgs& a, hipStream_t st);
// o = sum over a token's choices of weight rows_in[slot]
hipError_t launch_expert_gather(const ExpertCopyArgs& a, hipStream_t st);

}  // namespace fmlp

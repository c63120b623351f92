// Host-side launch descriptors of the gated block's operators: the gated MLP, the join of a block
// with its residual stream, and gradient clipping.
#pragma once
#include <vector>

#include "fmlp_launch.h"

namespace fmlp {

// Status reporting and device facts shared by the C-ABI translation units (fmlp_abi.cpp).
int abi_fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int abi_ok();
int abi_num_cus(int* out);

// One run of memory of a call over many tensors: what tensor i writes, or what of it is only read.
struct MemRange {
  uintptr_t lo, hi;
  int i;
  bool write;
};
// Workgroups write in no order: memory that a call writes and that another of its ranges holds too would be a race.
// Sorts the ranges and sets two such tensors' indices.
bool mem_overlap(std::vector<MemRange>& r, int* a, int* b);

// Gated MLP: X, dO (H, B, D) with dense rows and any head stride, Wg, Wu (H, D, E) with row pitch
// ldw, W2 (H, E, D), outputs dense.
struct GatedArgs {
  const void* x;
  const void* wg;
  const void* wu;
  const void* w2;
  const void* dout;
  void* o;
  void* dx;
  void* dwg;
  void* dwu;
  void* dw2;
  int64_t H, B, D, E;
  int64_t ldw;      // row pitch of wg and wu in elements (E, or E rounded up to a 16-byte vector)
  int64_t sx, sdo;  // elements between the heads of x and of dout
  int io;           // IoType
  int act;
  int num_cus;
  void* ws;
  size_t ws_bytes;
  int out_f32;      // o and dx as fp32 sums (FMLP_OUT_F32)
  float dw_scale;   // factor of the weight gradients
};

// Rows of E elements of both matrices copied to rows of ldw elements (whole 16-byte vectors, zeros behind the
// last element), one after the other at dst, in one launch (fmlp_gated_util.hip).
hipError_t launch_gated_pad(const void* wg, const void* wu, void* dst, int64_t rows, int64_t E, int64_t ldw, int es,
                            hipStream_t st);

// dst[i] = scale * sum over H of src[h][i] (n values, a multiple of 4), rounded to io (fmlp_gated_util.hip).
hipError_t launch_head_sum(const float* src, void* dst, int64_t n, int64_t H, float scale, int io, hipStream_t st);

// 16-bit io on LDS-staged kernels (fmlp_gated_fwd.hip). Forms of the row kernels: nw waves of 32 rows in each of es
// sets that take every chunk of a part of E, ns ring slots a set, oc waves per SIMD; nw = 0: no such form.
// per_cu workgroups run at once on a CU. A workgroup takes fixed_us and, for a chunk of each set, chunk_us alone or
// its share of full_us when the CU is full: the forward's measured times, dX's over the 1.4 that it takes as long on
// most (dx; at D = 64 it runs two waves a SIMD where the forward runs three: H=16 E=2048 dX of 256 row tiles 54 us, of 512
// 92, of 768 137).
struct GatedForm {
  int nw, es, ns, oc, per_cu;
  double chunk_us, full_us, fixed_us;
};
constexpr GatedForm gated_form(int D, int form, bool dx) {
  if (D == 32)
    return form == 0 ? GatedForm{2, 1, 4, 3, 6, 0.35, 1.2, 4.5} : form == 2 ? GatedForm{1, 4, 4, 1, 1, 0.45, 0.5, 4} : GatedForm{};
  if (D == 64)
    return form == 0   ? dx ? GatedForm{4, 1, 4, 2, 2, 0.55, 0.94, 4} : GatedForm{4, 1, 4, 3, 3, 0.5, 1.35, 4}
           : form == 2 ? GatedForm{2, 4, 3, 2, 1, 0.9, dx ? 1.1 : 0.95, 4}
                       : GatedForm{};
  if (D == 128)
    return form == 0   ? GatedForm{8, 1, 4, 2, 1, 0.94, 1.45, 6}
           : form == 1 ? GatedForm{4, 2, 3, 2, 1, 1.1, 1.45, 6}
                       : GatedForm{2, 2, 3, 1, 1, 1.0, 1.16, 5};
  return form == 0 ? GatedForm{4, 1, 3, 1, 1, 1.3, 1.55, 4.2} : GatedForm{};
}

// per_cu workgroups fit the waves of the CU's four SIMDs, and its LDS
constexpr bool gated_form_fits(int D, GatedForm f) {
  return f.per_cu * f.nw * f.es <= 4 * f.oc && f.per_cu * f.es * f.ns * 192 * D <= 160 * 1024;
}

// `tiles` row tiles of a form, each split over xs workgroups of nct chunks of 32 columns, whose fp32 partials
// take ws_bytes when xs > 1.
struct GatedFwdPlan {
  int form;
  long long tiles;
  int xs, nct;
  size_t ws_bytes;
};
// (whole: no split and no partials, for calls whose workspace does not hold them; likewise below)
GatedFwdPlan gated_fwd_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool dx, bool whole);
hipError_t launch_gated_fwd(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st);
// dX on the same forms and plan (fmlp_gated_dx.hip)
hipError_t launch_gated_dx(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st);

// dW programs (fmlp_gated_dw.hip): nE tiles of E and nS ranges of rows a head, whose fp32 partials
// ([nS][dWg, dWu, dW2]) take ws_bytes when nS > 1.
struct GatedDwPlan {
  int nE, nS, rows_per_split;
  long long programs;
  size_t ws_bytes;
};
GatedDwPlan gated_dw_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole);
hipError_t launch_gated_dw(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st);
hipError_t launch_gated_dw128(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st);

// fp32 io (fmlp_gated_f32.hip): tiles of 128 rows, E-tiles of 128 columns (32 at D = 256).
GatedFwdPlan gated32_rows_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole);
GatedDwPlan gated32_dw_plan(int64_t H, int64_t B, int64_t D, int64_t E, int num_cus, bool whole);
hipError_t launch_gated32_fwd(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st);
hipError_t launch_gated32_dx(const GatedArgs& a, const GatedFwdPlan& p, hipStream_t st);
hipError_t launch_gated32_dw(const GatedArgs& a, const GatedDwPlan& p, hipStream_t st);

// A block's join (fmlp_join.hip): the stream r (B, C), C = H D; o, y and their gradients (head, row, column)
// with unit column stride. Pointers that are null leave their part out: o (no block output: only y is
// taken from r), w_post, gate, w_pre (factors of one), r_out, y (results nobody asked for), and in the
// backward dy, dr_out (gradients that are zero), dr, d_o, dw_post, dgate, dw_pre (not asked for).
struct JoinArgs {
  const void* r;  // backward: null, or what r' is computed from again, rows r_sr apart
  const void* o;
  const void* w_post;
  const void* gate;  // (groups, C): row g for rows g rows_per_gate ..
  const void* w_pre;
  void* r_out;  // forward: r' (dense rows); backward without r: the r' that was saved, rows r_sr apart
  void* y;
  float* rs_o;  // (B) 1 / rms of o and of r', written by the forward (or null) and read by the backward
  float* rs_r;
  const void* dr_out;
  const void* dy;
  void* dr;   // dense rows
  void* d_o;
  void* dw_post;
  void* dgate;
  void* dw_pre;
  long long B, C, D, groups, rows_per_gate;
  long long row0;  // the forward launch's first row
  long long r_sr, dr_sr, o_sh, o_sr, y_sh, y_sr, do_sh, do_sr;  // element strides (y's: of dy in the backward)
  float scale, eps;
  int io;       // IoType of o, y, the weights and the gate
  int r_f32;    // the stream is fp32 beside 16-bit io
  int post;     // o is normalised
  int aligned;  // D % 8 == 0, every pointer 16-byte aligned and every stride a multiple of 16 bytes
};

// Backward units (fmlp_join.hip): `parts` per gate group, or groups_per_unit whole groups each.
struct JoinPlan {
  long long units, groups_per_unit, rows_per_part;
  int parts;
  bool gate_partials;
  size_t off_pre, off_post, off_gate, ws_bytes;
  float* pre;
  float* post;
  float* gate;
};
struct JoinSum {
  const float* src;
  void* dst;
  int rows, groups;
};
struct JoinReduce {
  JoinSum t[3];
};
constexpr int64_t kJoinMaxC = 16384;  // 1024 threads of two vectors of 8 columns
JoinPlan join_plan(int64_t B, int64_t C, int64_t groups, bool dpre, bool dpost, bool dgate, int num_cus);
hipError_t launch_join_fwd(const JoinArgs& a, hipStream_t st);
hipError_t launch_join_bwd(const JoinArgs& a, JoinPlan p, void* ws, hipStream_t st);

// Gradient norm and clipping (fmlp_clip.hip): n tensors of `numel` elements; io / out_io IoType codes. outs[i]
// null: nothing is written; equal to grads[i]: in place. ws: clip_plan's bytes.
struct ClipTensor {
  const void* grad;
  void* out;
  long long numel;
  int io, out_io;
};
struct ClipPlan {
  long long chunk;   // elements per workgroup
  long long blocks;  // workgroups over all tensors
  size_t ws_bytes;   // one double per workgroup and the coefficient
};
ClipPlan clip_plan(int n, const int64_t* numel, int num_cus);
hipError_t launch_clip(int n, const ClipTensor* t, const ClipPlan& p, bool clip, float max_norm, float* norm, void* ws,
                       hipStream_t st);

}  // namespace fmlp

// C ABI of the gated block's operators (declared in include/flashmlp.h): argument validation and
// dispatch, as fmlp_abi.cpp does for the MLP. No allocation, no synchronisation.
#include "../../include/flashmlp.h"
#include "fmlp_block.h"

#include <algorithm>
#include <new>
#include <vector>

#define FMLP_EXPORT extern "C" __attribute__((visibility("default")))

using fmlp::abi_fail;
using fmlp::abi_ok;

namespace {

constexpr int kGatedFlags = FMLP_BWD_NO_DX | FMLP_BWD_NO_DW | FMLP_OUT_F32;

int io_of(int dtype) { return dtype & ~kGatedFlags; }
size_t elem_bytes(int io) { return io == FMLP_DTYPE_F32 ? 4 : 2; }

int check_vec(const void* p, const char* name, bool needed) {
  if (!needed) return FMLP_OK;
  if (p == nullptr) return abi_fail(FMLP_ERR_INVALID_ARG, "%s is NULL", name);
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%s is not 16-byte aligned", name);
  return FMLP_OK;
}

int check_gated(int64_t H, int64_t B, int64_t D, int64_t E, int dtype, int act) {
  if (H < 0 || B < 0 || D < 0 || E < 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "negative dimension (H=%lld B=%lld D=%lld E=%lld)", (long long)H, (long long)B,
                    (long long)D, (long long)E);
  const int io = io_of(dtype);
  if (io != FMLP_DTYPE_F16 && io != FMLP_DTYPE_BF16 && io != FMLP_DTYPE_F32)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", dtype);
  if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "hidden dimension D=%lld: supported D are 16, 32, 64, 128 and 256",
                    (long long)D);
  if (E < 1) return abi_fail(FMLP_ERR_UNSUPPORTED, "intermediate dimension E=%lld: must be positive", (long long)E);
  if (B > (1LL << 30) || E > (1LL << 30) || H > (1LL << 30))
    return abi_fail(FMLP_ERR_INVALID_ARG, "dimension too large (H=%lld B=%lld E=%lld)", (long long)H, (long long)B,
                    (long long)E);
  if (D * (E + 8) * 4 > 0x7fffffffLL)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "per-head weight slice D*E=%lld values exceeds 512 Mi", (long long)(D * E));
  if (H * ((B + 31) / 32) + H * ((E + 31) / 32) * 64 > 0x7fffffffLL)
    return abi_fail(FMLP_ERR_INVALID_ARG, "problem too large for one launch");
  if (act < FMLP_ACT_NONE || act > FMLP_ACT_SIGMOID) return abi_fail(FMLP_ERR_INVALID_ARG, "activation code %d", act);
  return FMLP_OK;
}

int check_head_stride(int64_t s, const char* name, int64_t H, size_t es) {
  if (s < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "%s head stride is negative (%lld)", name, (long long)s);
  if (H > 1 && (s * (int64_t)es) % 16 != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%s head stride %lld is no multiple of 16 bytes", name, (long long)s);
  return FMLP_OK;
}

// Wg and Wu where rows of E elements are no whole 16-byte vectors: padded copies at the workspace's start
size_t gated_pad_bytes(int64_t H, int64_t D, int64_t E, int io) {
  const int es = (int)elem_bytes(io);
  const int64_t ldw = fmlp::w1_pitch(E, es);
  return ldw == E ? 0 : ((size_t)(2 * H * D * ldw) * es + 255) / 256 * 256;
}
hipError_t gated_pad(fmlp::GatedArgs* a, hipStream_t st) {
  const int es = a->io == fmlp::IO_F32 ? 4 : 2;
  a->ldw = fmlp::w1_pitch(a->E, es);
  if (a->ldw == a->E) return hipSuccess;
  const size_t one = (size_t)(a->H * a->D * a->ldw) * es, all = (2 * one + 255) / 256 * 256;
  char* ws = (char*)a->ws;
  const hipError_t e = fmlp::launch_gated_pad(a->wg, a->wu, ws, a->H * a->D, a->E, a->ldw, es, st);
  a->wg = ws;
  a->wu = ws + one;
  a->ws = ws + all;
  a->ws_bytes -= all;
  return e;
}
int check_ws(const void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need))
    return abi_fail(FMLP_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws ? have : (size_t)0, need);
  return FMLP_OK;
}
fmlp::GatedFwdPlan rows_plan(int64_t H, int64_t B, int64_t D, int64_t E, int io, int cus, bool dx, bool whole = false) {
  return io == FMLP_DTYPE_F32 ? fmlp::gated32_rows_plan(H, B, D, E, cus, whole)
                              : fmlp::gated_fwd_plan(H, B, D, E, cus, dx, whole);
}
fmlp::GatedDwPlan dw_plan(int64_t H, int64_t B, int64_t D, int64_t E, int io, int cus, bool whole = false) {
  return io == FMLP_DTYPE_F32 ? fmlp::gated32_dw_plan(H, B, D, E, cus, whole) : fmlp::gated_dw_plan(H, B, D, E, cus, whole);
}
// the same for what is left of the workspace behind the padded weights: whole tiles where the partials do not fit
fmlp::GatedFwdPlan rows_plan(const fmlp::GatedArgs& a, int io, bool dx) {
  const fmlp::GatedFwdPlan p = rows_plan(a.H, a.B, a.D, a.E, io, a.num_cus, dx);
  return p.ws_bytes <= a.ws_bytes ? p : rows_plan(a.H, a.B, a.D, a.E, io, a.num_cus, dx, true);
}
fmlp::GatedDwPlan dw_plan(const fmlp::GatedArgs& a, int io) {
  const fmlp::GatedDwPlan p = dw_plan(a.H, a.B, a.D, a.E, io, a.num_cus);
  return p.ws_bytes <= a.ws_bytes ? p : dw_plan(a.H, a.B, a.D, a.E, io, a.num_cus, true);
}

int io_type(int io) { return io == FMLP_DTYPE_F32 ? fmlp::IO_F32 : io == FMLP_DTYPE_BF16 ? fmlp::IO_BF16 : fmlp::IO_F16; }

}  // namespace

namespace fmlp {

bool mem_overlap(std::vector<MemRange>& r, int* a, int* b) {
  const auto by_lo = [](const MemRange& x, const MemRange& y) { return x.lo < y.lo; };
  if (!std::is_sorted(r.begin(), r.end(), by_lo)) std::sort(r.begin(), r.end(), by_lo);
  const MemRange *w = nullptr, *any = nullptr;  // those that reach furthest so far
  for (const MemRange& x : r) {
    const MemRange* o = x.write ? any : w;
    if (o != nullptr && x.lo < o->hi) {
      *a = std::min(x.i, o->i);
      *b = std::max(x.i, o->i);
      return true;
    }
    if (any == nullptr || x.hi > any->hi) any = &x;
    if (x.write && (w == nullptr || x.hi > w->hi)) w = &x;
  }
  return false;
}

}  // namespace fmlp

FMLP_EXPORT size_t fmlp_gated_min_workspace_bytes(int64_t H, int64_t D, int64_t E, int dtype) {
  if (check_gated(H, 0, D, E, dtype, 0)) return 0;
  return gated_pad_bytes(H, D, E, io_of(dtype));
}

FMLP_EXPORT size_t fmlp_gated_fwd_workspace_bytes(int64_t H, int64_t B, int64_t D, int64_t E, int dtype) {
  int cus = 0;
  dtype &= ~FMLP_OUT_F32;
  if (check_gated(H, B, D, E, dtype, 0) || fmlp::abi_num_cus(&cus)) return 0;
  return gated_pad_bytes(H, D, E, dtype) + rows_plan(H, B, D, E, dtype, cus, false).ws_bytes;
}

namespace {

// the row sums' and the tile sums' partials share the workspace behind the padded weights
size_t gated_bwd_ws(int64_t H, int64_t B, int64_t D, int64_t E, int dtype, int cus) {
  const int io = io_of(dtype);
  const size_t dw = (dtype & FMLP_BWD_NO_DW) ? 0 : dw_plan(H, B, D, E, io, cus).ws_bytes;
  const size_t dx = (dtype & FMLP_BWD_NO_DX) ? 0 : rows_plan(H, B, D, E, io, cus, true).ws_bytes;
  return gated_pad_bytes(H, D, E, io) + (dw > dx ? dw : dx);
}

}  // namespace

FMLP_EXPORT size_t fmlp_gated_bwd_workspace_bytes(int64_t H, int64_t B, int64_t D, int64_t E, int dtype) {
  int cus = 0;
  if (check_gated(H, B, D, E, dtype, 0) || fmlp::abi_num_cus(&cus)) return 0;
  return gated_bwd_ws(H, B, D, E, dtype, cus);
}

FMLP_EXPORT int fmlp_gated_fwd(const void* x, const void* wg, const void* wu, const void* w2, void* o, int64_t H,
                               int64_t B, int64_t D, int64_t E, int64_t x_head_stride, int dtype, int act,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const bool out_f32 = (dtype & FMLP_OUT_F32) != 0;
  dtype &= ~FMLP_OUT_F32;
  if (dtype & kGatedFlags)
    return abi_fail(FMLP_ERR_INVALID_ARG, "FMLP_BWD_NO_DX / FMLP_BWD_NO_DW apply to the backward only");
  int st = check_gated(H, B, D, E, dtype, act);
  if (st) return st;
  const bool rows = H > 0 && B > 0;
  if ((st = check_head_stride(x_head_stride, "x", H, elem_bytes(dtype))) || (st = check_vec(x, "x", rows)) ||
      (st = check_vec(wg, "wg", H > 0)) || (st = check_vec(wu, "wu", H > 0)) || (st = check_vec(w2, "w2", H > 0)) ||
      (st = check_vec(o, "o", rows)) || (st = check_vec(workspace, "workspace", workspace != nullptr)))
    return st;
  if (!rows) return abi_ok();
  fmlp::GatedArgs a{};
  a.x = x;
  a.wg = wg;
  a.wu = wu;
  a.w2 = w2;
  a.o = o;
  a.H = H;
  a.B = B;
  a.D = D;
  a.E = E;
  a.ldw = E;
  a.sx = x_head_stride;
  a.io = io_type(dtype);
  a.act = act;
  a.out_f32 = out_f32 ? 1 : 0;
  a.dw_scale = 1.f;
  a.ws = workspace;
  a.ws_bytes = workspace != nullptr ? workspace_bytes : 0;
  if ((st = fmlp::abi_num_cus(&a.num_cus))) return st;
  const hipStream_t hs = (hipStream_t)stream;
  if ((st = check_ws(workspace, workspace_bytes, gated_pad_bytes(H, D, E, dtype)))) return st;
  hipError_t e = gated_pad(&a, hs);
  const fmlp::GatedFwdPlan p = rows_plan(a, dtype, false);
  if (e == hipSuccess) e = a.io == fmlp::IO_F32 ? fmlp::launch_gated32_fwd(a, p, hs) : fmlp::launch_gated_fwd(a, p, hs);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "gated forward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

FMLP_EXPORT int fmlp_gated_bwd(const void* x, const void* wg, const void* wu, const void* w2, const void* dout,
                               void* dx, void* dwg, void* dwu, void* dw2, int64_t H, int64_t B, int64_t D, int64_t E,
                               int64_t x_head_stride, int64_t dout_head_stride, int dtype, int act, float dw_scale,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_gated(H, B, D, E, dtype, act);
  if (st) return st;
  const bool rows = H > 0 && B > 0, want_dx = (dtype & FMLP_BWD_NO_DX) == 0, want_dw = (dtype & FMLP_BWD_NO_DW) == 0;
  const size_t es = elem_bytes(io_of(dtype));
  if ((st = check_head_stride(x_head_stride, "x", H, es)) || (st = check_head_stride(dout_head_stride, "dout", H, es)) ||
      (st = check_vec(x, "x", rows)) || (st = check_vec(dout, "dout", rows)) || (st = check_vec(wg, "wg", H > 0)) ||
      (st = check_vec(wu, "wu", H > 0)) || (st = check_vec(w2, "w2", H > 0)) ||
      (st = check_vec(dx, "dx", rows && want_dx)) || (st = check_vec(dwg, "dwg", H > 0 && want_dw)) ||
      (st = check_vec(dwu, "dwu", H > 0 && want_dw)) || (st = check_vec(dw2, "dw2", H > 0 && want_dw)) ||
      (st = check_vec(workspace, "workspace", workspace != nullptr)))
    return st;
  if (H == 0) return abi_ok();
  fmlp::GatedArgs a{};
  a.x = x;
  a.wg = wg;
  a.wu = wu;
  a.w2 = w2;
  a.dout = dout;
  a.dx = dx;
  a.dwg = dwg;
  a.dwu = dwu;
  a.dw2 = dw2;
  a.H = H;
  a.B = B;
  a.D = D;
  a.E = E;
  a.ldw = E;
  a.sx = x_head_stride;
  a.sdo = dout_head_stride;
  a.out_f32 = (dtype & FMLP_OUT_F32) ? 1 : 0;
  a.dw_scale = dw_scale;
  a.io = io_type(io_of(dtype));
  a.act = act;
  a.ws = workspace;
  a.ws_bytes = workspace != nullptr ? workspace_bytes : 0;
  if ((st = fmlp::abi_num_cus(&a.num_cus))) return st;
  const hipStream_t hs = (hipStream_t)stream;
  const int io = io_of(dtype);
  hipError_t e = hipSuccess;
  if (want_dw || want_dx) {
    if ((st = check_ws(workspace, workspace_bytes, gated_pad_bytes(H, D, E, io)))) return st;
    e = gated_pad(&a, hs);
    if (e == hipSuccess && want_dw) {
      const fmlp::GatedDwPlan p = dw_plan(a, io);
      e = a.io == fmlp::IO_F32 ? fmlp::launch_gated32_dw(a, p, hs) : fmlp::launch_gated_dw(a, p, hs);
    }
    if (e == hipSuccess && want_dx) {
      const fmlp::GatedFwdPlan p = rows_plan(a, io, true);
      e = a.io == fmlp::IO_F32 ? fmlp::launch_gated32_dx(a, p, hs) : fmlp::launch_gated_dx(a, p, hs);
    }
  }
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "gated backward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

FMLP_EXPORT int fmlp_head_sum(const float* src, void* dst, int64_t H, int64_t n, float scale, int dtype, void* stream) {
  if (H < 1 || H > (1LL << 30) || n < 0 || n % 4 != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "H=%lld n=%lld: at least one head, n a multiple of 4", (long long)H, (long long)n);
  if (dtype != FMLP_DTYPE_F16 && dtype != FMLP_DTYPE_BF16 && dtype != FMLP_DTYPE_F32)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", dtype);
  int st;
  if ((st = check_vec(src, "src", n > 0)) || (st = check_vec(dst, "dst", n > 0))) return st;
  const hipError_t e = fmlp::launch_head_sum(src, dst, n, H, scale, io_type(dtype), (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "head sum launch: %s", hipGetErrorString(e));
  return abi_ok();
}

// ---------------------------------------------------------------------------------------------
// join
// ---------------------------------------------------------------------------------------------
namespace {

// a pointer of the call, aligned to its elements; *vec is cleared where it is not a 16-byte vector's
int join_ptr(const void* p, const char* name, bool needed, size_t es, int* vec) {
  if (p == nullptr) return needed ? abi_fail(FMLP_ERR_INVALID_ARG, "%s is NULL", name) : FMLP_OK;
  if ((reinterpret_cast<uintptr_t>(p) % es) != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%s is not %zu-byte aligned", name, es);
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) *vec = 0;
  return FMLP_OK;
}

int join_stride(int64_t s, const char* name, bool used, size_t es, int* vec) {
  if (!used) return FMLP_OK;
  if (s < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "%s stride is negative (%lld)", name, (long long)s);
  if ((s * (int64_t)es) % 16 != 0) *vec = 0;
  return FMLP_OK;
}

int check_join(const fmlp_join* j, bool bwd, fmlp::JoinArgs* a) {
  if (j == nullptr) return abi_fail(FMLP_ERR_INVALID_ARG, "the call's description is NULL");
  if (j->B < 0 || j->H < 1 || j->D < 1 || j->groups < 1)
    return abi_fail(FMLP_ERR_INVALID_ARG, "dimensions B=%lld H=%lld D=%lld groups=%lld", (long long)j->B, (long long)j->H,
                    (long long)j->D, (long long)j->groups);
  if (j->dtype != FMLP_DTYPE_F16 && j->dtype != FMLP_DTYPE_BF16 && j->dtype != FMLP_DTYPE_F32)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", j->dtype);
  if (j->r_dtype != j->dtype && j->r_dtype != FMLP_DTYPE_F32)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "stream dtype code %d: the blocks' dtype or fp32", j->r_dtype);
  if (j->H > fmlp::kJoinMaxC || j->D > fmlp::kJoinMaxC || j->H * j->D > fmlp::kJoinMaxC)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "%lld x %lld columns: at most %lld", (long long)j->H, (long long)j->D,
                    (long long)fmlp::kJoinMaxC);
  if (j->B > 0x7fffffffLL) return abi_fail(FMLP_ERR_INVALID_ARG, "too many rows (%lld)", (long long)j->B);
  if (j->B % j->groups != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%lld rows are no multiple of the gate's %lld", (long long)j->B,
                    (long long)j->groups);
  if (!(j->eps >= 0)) return abi_fail(FMLP_ERR_INVALID_ARG, "eps is negative or NaN");
  if (!j->post && j->w_post) return abi_fail(FMLP_ERR_INVALID_ARG, "w_post without the post norm");
  const size_t es = elem_bytes(j->dtype), rs = elem_bytes(j->r_dtype);
  const bool rows = j->B > 0, has_o = j->o != nullptr, has_y = bwd ? j->dy != nullptr : j->y != nullptr;
  if (rows && !bwd && !has_y && j->r_out == nullptr) return abi_fail(FMLP_ERR_INVALID_ARG, "no output is asked for");
  if (rows && !has_o && (j->w_post || j->gate)) return abi_fail(FMLP_ERR_INVALID_ARG, "w_post or gate without o");
  if (rows && !has_y && j->w_pre && !bwd) return abi_fail(FMLP_ERR_INVALID_ARG, "w_pre without y");
  // the backward of a 16-bit stream with r makes the unrounded r' again
  const bool from_r = bwd && j->r && has_o && has_y && j->r_dtype != FMLP_DTYPE_F32;
  int vec = j->D % 8 == 0 ? 1 : 0, st;
  if ((st = join_ptr(bwd && !from_r ? nullptr : j->r, "r", rows && !bwd, rs, &vec)) || (st = join_ptr(j->o, "o", false, es, &vec)) ||
      (st = join_ptr(j->w_post, "w_post", false, es, &vec)) || (st = join_ptr(j->gate, "gate", false, es, &vec)) ||
      (st = join_ptr(j->w_pre, "w_pre", false, es, &vec)) ||
      (st = join_ptr(j->r_out, "r_out", rows && bwd && has_y && !from_r, rs, &vec)) ||
      (st = join_ptr(j->y, "y", false, es, &vec)) || (st = join_stride(j->r_stride, "r", true, rs, &vec)) ||
      (st = join_stride(j->o_head_stride, "o head", has_o && j->H > 1, es, &vec)) ||
      (st = join_stride(j->o_row_stride, "o row", has_o, es, &vec)) ||
      (st = join_stride(j->y_head_stride, "y head", has_y && j->H > 1, es, &vec)) ||
      (st = join_stride(j->y_row_stride, "y row", has_y, es, &vec)))
    return st;
  if (bwd) {
    int v4 = 1;
    if ((st = join_ptr(j->dr_out, "dr_out", false, rs, &vec)) || (st = join_ptr(j->dy, "dy", false, es, &vec)) ||
        (st = join_ptr(j->dr, "dr", false, rs, &vec)) || (st = join_ptr(j->d_o, "d_o", false, es, &vec)) ||
        (st = join_ptr(j->dw_post, "dw_post", false, es, &vec)) || (st = join_ptr(j->dgate, "dgate", false, es, &vec)) ||
        (st = join_ptr(j->dw_pre, "dw_pre", false, es, &vec)) ||
        (st = join_stride(j->dr_out_stride, "dr_out", j->dr_out != nullptr, rs, &vec)) ||
        (st = join_stride(j->d_o_head_stride, "d_o head", j->d_o != nullptr && j->H > 1, es, &vec)) ||
        (st = join_stride(j->d_o_row_stride, "d_o row", j->d_o != nullptr, es, &vec)) ||
        (st = join_ptr(j->rs_o, "rs_o", rows && has_o && j->post, 4, &v4)) ||
        (st = join_ptr(j->rs_r, "rs_r", rows && has_y, 4, &v4)))
      return st;
    if (rows && !has_o && (j->d_o || j->dw_post || j->dgate)) return abi_fail(FMLP_ERR_INVALID_ARG, "gradients of o's part without o");
    if (j->dw_post && !j->post) return abi_fail(FMLP_ERR_INVALID_ARG, "dw_post without the post norm");
  }
  a->r = bwd && !from_r ? nullptr : j->r;
  a->o = j->o;
  a->w_post = j->w_post;
  a->gate = j->gate;
  a->w_pre = j->w_pre;
  a->r_out = j->r_out;
  a->y = j->y;
  a->rs_o = j->rs_o;
  a->rs_r = j->rs_r;
  a->dr_out = j->dr_out;
  a->dy = j->dy;
  a->dr = j->dr;
  a->d_o = j->d_o;
  a->dw_post = j->dw_post;
  a->dgate = j->dgate;
  a->dw_pre = j->dw_pre;
  a->B = j->B;
  a->C = j->H * j->D;
  a->D = j->D;
  a->groups = j->groups;
  a->rows_per_gate = j->B / j->groups;
  a->r_sr = j->r_stride;
  a->dr_sr = j->dr_out_stride;
  a->o_sh = j->o_head_stride;
  a->o_sr = j->o_row_stride;
  a->y_sh = j->y_head_stride;
  a->y_sr = j->y_row_stride;
  a->do_sh = j->d_o_head_stride;
  a->do_sr = j->d_o_row_stride;
  a->scale = j->scale;
  a->eps = j->eps;
  a->io = io_type(j->dtype);
  a->r_f32 = j->r_dtype == FMLP_DTYPE_F32 && j->dtype != FMLP_DTYPE_F32;
  a->post = j->post ? 1 : 0;
  a->aligned = vec;
  return FMLP_OK;
}

int join_bwd_plan(const fmlp_join* j, const fmlp::JoinArgs& a, fmlp::JoinPlan* p) {
  int cus = 0;
  const int st = fmlp::abi_num_cus(&cus);
  if (st) return st;
  *p = fmlp::join_plan(a.B, a.C, j->groups, j->dw_pre != nullptr, j->dw_post != nullptr, j->dgate != nullptr, cus);
  return FMLP_OK;
}

}  // namespace

FMLP_EXPORT int fmlp_join_fwd(const fmlp_join* j, void* stream) {
  fmlp::JoinArgs a{};
  const int st = check_join(j, false, &a);
  if (st) return st;
  const hipError_t e = fmlp::launch_join_fwd(a, (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "join forward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

FMLP_EXPORT size_t fmlp_join_bwd_workspace_bytes(const fmlp_join* j) {
  fmlp::JoinArgs a{};
  fmlp::JoinPlan p{};
  if (check_join(j, true, &a) || join_bwd_plan(j, a, &p)) return 0;
  return p.ws_bytes;
}

FMLP_EXPORT int fmlp_join_bwd(const fmlp_join* j, void* workspace, size_t workspace_bytes, void* stream) {
  fmlp::JoinArgs a{};
  fmlp::JoinPlan p{};
  int st;
  if ((st = check_join(j, true, &a)) || (st = join_bwd_plan(j, a, &p)) ||
      (st = check_vec(workspace, "workspace", workspace != nullptr)))
    return st;
  if (p.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < p.ws_bytes))
    return abi_fail(FMLP_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0,
                    p.ws_bytes);
  const hipError_t e = fmlp::launch_join_bwd(a, p, workspace, (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "join backward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

// ---------------------------------------------------------------------------------------------
// gradient norm and clipping
// ---------------------------------------------------------------------------------------------
namespace {

int clip_impl(int n, const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
              const int* out_dtypes, bool clip, float max_norm, float* norm, void* ws, size_t ws_bytes, void* stream) {
  if (n < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "%d tensors", n);
  if (n > 0 && (grads == nullptr || numels == nullptr || dtypes == nullptr || (clip && (outs == nullptr || out_dtypes == nullptr))))
    return abi_fail(FMLP_ERR_INVALID_ARG, "tensor arrays must not be NULL");
  if (norm == nullptr || (reinterpret_cast<uintptr_t>(norm) & 3u) != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "norm is NULL or not 4-byte aligned");
  if (clip && !(max_norm >= 0)) return abi_fail(FMLP_ERR_INVALID_ARG, "max_norm is negative or NaN");
  std::vector<fmlp::ClipTensor> t;
  std::vector<fmlp::MemRange> ranges;
  try {
    t.resize((size_t)n);
    if (clip) ranges.reserve(2 * (size_t)n);
  } catch (const std::bad_alloc&) {
    return abi_fail(FMLP_ERR_INVALID_ARG, "no host memory for %d tensors", n);
  }
  for (int i = 0; i < n; ++i) {
    const int ins[2] = {dtypes[i], clip ? out_dtypes[i] : dtypes[i]};
    for (int d : ins)
      if (d != FMLP_DTYPE_F16 && d != FMLP_DTYPE_BF16 && d != FMLP_DTYPE_F32)
        return abi_fail(FMLP_ERR_UNSUPPORTED, "tensor %d: dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", i, d);
    if (numels[i] < 0 || numels[i] > (1LL << 40))
      return abi_fail(FMLP_ERR_INVALID_ARG, "tensor %d: %lld elements", i, (long long)numels[i]);
    const void* g = grads[i];
    void* o = clip ? outs[i] : nullptr;
    if (numels[i] > 0) {
      if (g == nullptr || (reinterpret_cast<uintptr_t>(g) % elem_bytes(ins[0])) != 0)
        return abi_fail(FMLP_ERR_INVALID_ARG, "gradient %d is NULL or not aligned to its elements", i);
      if (clip && (o == nullptr || (reinterpret_cast<uintptr_t>(o) % elem_bytes(ins[1])) != 0))
        return abi_fail(FMLP_ERR_INVALID_ARG, "output %d is NULL or not aligned to its elements", i);
    }
    t[(size_t)i] = fmlp::ClipTensor{g, o, numels[i], io_type(ins[0]), io_type(ins[1])};
    if (clip && numels[i] > 0) {
      const uintptr_t gi = reinterpret_cast<uintptr_t>(g), oi = reinterpret_cast<uintptr_t>(o);
      ranges.push_back(fmlp::MemRange{oi, oi + (uintptr_t)numels[i] * elem_bytes(ins[1]), i, true});
      if (g != o || ins[0] != ins[1]) ranges.push_back(fmlp::MemRange{gi, gi + (uintptr_t)numels[i] * elem_bytes(ins[0]), i, false});
    }
  }
  int one, two;
  if (clip && fmlp::mem_overlap(ranges, &one, &two))
    return abi_fail(FMLP_ERR_INVALID_ARG, "the output of tensor %d or %d overlaps a tensor of the call", one, two);
  int cus = 0, st;
  if ((st = fmlp::abi_num_cus(&cus))) return st;
  const fmlp::ClipPlan p = fmlp::clip_plan(n, numels, cus);
  if ((st = check_vec(ws, "workspace", true))) return st;
  if (ws_bytes < p.ws_bytes)
    return abi_fail(FMLP_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, p.ws_bytes);
  const hipError_t e = fmlp::launch_clip(n, t.data(), p, clip, max_norm, norm, ws, (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "gradient clipping launch: %s", hipGetErrorString(e));
  return abi_ok();
}

}  // namespace

FMLP_EXPORT size_t fmlp_clip_workspace_bytes(int n, const int64_t* numels) {
  int cus = 0;
  if (n < 0 || (n > 0 && numels == nullptr) || fmlp::abi_num_cus(&cus)) return 0;
  for (int i = 0; i < n; ++i)
    if (numels[i] < 0 || numels[i] > (1LL << 40)) return 0;
  return fmlp::clip_plan(n, numels, cus).ws_bytes;
}

FMLP_EXPORT int fmlp_grad_norm(int n, const void* const* grads, const int64_t* numels, const int* dtypes, float* norm,
                               void* workspace, size_t workspace_bytes, void* stream) {
  return clip_impl(n, grads, nullptr, numels, dtypes, nullptr, false, 0.f, norm, workspace, workspace_bytes, stream);
}

FMLP_EXPORT int fmlp_clip_grads(int n, const void* const* grads, void* const* outs, const int64_t* numels,
                                const int* dtypes, const int* out_dtypes, float max_norm, float* norm, void* workspace,
                                size_t workspace_bytes, void* stream) {
  return clip_impl(n, grads, outs, numels, dtypes, out_dtypes, true, max_norm, norm, workspace, workspace_bytes, stream);
}

// C ABI of the gated block's operators (declared in include/flashmlp.h): argument validation and
// dispatch, as fmlp_abi.cpp does for the MLP. No allocation, no synchronisation.
#include "../../include/flashmlp.h"
#include "fmlp_block.h"

#define FMLP_EXPORT extern "C" __attribute__((visibility("default")))

using fmlp::abi_fail;
using fmlp::abi_ok;

namespace {

constexpr int kGatedFlags = FMLP_BWD_NO_DX | FMLP_BWD_NO_DW;

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

int io_type(int io) { return io == FMLP_DTYPE_F32 ? fmlp::IO_F32 : io == FMLP_DTYPE_BF16 ? fmlp::IO_BF16 : fmlp::IO_F16; }

}  // namespace

FMLP_EXPORT size_t fmlp_gated_fwd_workspace_bytes(int64_t H, int64_t B, int64_t D, int64_t E, int dtype) {
  (void)H, (void)B, (void)D, (void)E, (void)dtype;
  return 0;
}

FMLP_EXPORT size_t fmlp_gated_bwd_workspace_bytes(int64_t H, int64_t B, int64_t D, int64_t E, int dtype) {
  (void)H, (void)B, (void)D, (void)E, (void)dtype;
  return 0;
}

FMLP_EXPORT int fmlp_gated_fwd(const void* x, const void* wg, const void* wu, const void* w2, void* o, int64_t H,
                               int64_t B, int64_t D, int64_t E, int64_t x_head_stride, int dtype, int act,
                               void* workspace, size_t workspace_bytes, void* stream) {
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
  a.ws = workspace;
  a.ws_bytes = workspace != nullptr ? workspace_bytes : 0;
  if ((st = fmlp::abi_num_cus(&a.num_cus))) return st;
  const hipError_t e = fmlp::launch_gated_gen_fwd(a, (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "gated forward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

FMLP_EXPORT int fmlp_gated_bwd(const void* x, const void* wg, const void* wu, const void* w2, const void* dout,
                               void* dx, void* dwg, void* dwu, void* dw2, int64_t H, int64_t B, int64_t D, int64_t E,
                               int64_t x_head_stride, int64_t dout_head_stride, int dtype, int act, void* workspace,
                               size_t workspace_bytes, void* stream) {
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
  a.io = io_type(io_of(dtype));
  a.act = act;
  a.ws = workspace;
  a.ws_bytes = workspace != nullptr ? workspace_bytes : 0;
  if ((st = fmlp::abi_num_cus(&a.num_cus))) return st;
  hipError_t e = hipSuccess;
  if (want_dw) e = fmlp::launch_gated_gen_dw(a, (hipStream_t)stream);
  if (e == hipSuccess && want_dx) e = fmlp::launch_gated_gen_dx(a, (hipStream_t)stream);
  if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "gated backward launch: %s", hipGetErrorString(e));
  return abi_ok();
}

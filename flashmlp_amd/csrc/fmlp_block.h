// Host-side launch descriptors of the gated block's operators: the gated MLP, the join of a block
// with its residual stream, and gradient clipping.
#pragma once
#include "fmlp_launch.h"

namespace fmlp {

// Status reporting and device facts shared by the C-ABI translation units (fmlp_abi.cpp).
int abi_fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int abi_ok();
int abi_num_cus(int* out);

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
};

// The kernels that read their operands from global memory (fmlp_gated_gen.hip): every io type and D.
hipError_t launch_gated_gen_fwd(const GatedArgs& a, hipStream_t st);
hipError_t launch_gated_gen_dx(const GatedArgs& a, hipStream_t st);
hipError_t launch_gated_gen_dw(const GatedArgs& a, hipStream_t st);

}  // namespace fmlp

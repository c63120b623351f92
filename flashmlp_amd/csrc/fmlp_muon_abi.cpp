// C ABI of the orthogonalised updates (declared in include/flashmlp.h): argument validation and dispatch. No device
// allocation, no synchronisation.
#include "../../include/flashmlp.h"
#include "fmlp_block.h"
#include "fmlp_muon.h"

#include <algorithm>
#include <new>
#include <vector>

#define FMLP_EXPORT extern "C" __attribute__((visibility("default")))

using fmlp::abi_fail;
using fmlp::abi_ok;

namespace {

// Steps on one Gram matrix. Rounding of it at the smallest eigenvalues grows by q(0)^2 = a^2 a step, 12 for the usual a = 3.44, until
// they are of the size of one. bf16 results hide a growth of 2e4 before the stage's last step: five usual steps, whose results are
// off by 4e-6 to 4e-4 in norm and up to 1.4e-3 at a singular value (64 x 64 to 256 x 1024, noise around a low rank and spectra
// of one to five decades; a bf16 result's rounding is 1.7e-3, at a singular value 1.6 to 3e-3). Five steps of a schedule that
// begins with a = 8.3, 2e5, were off by up to 2.4e-3 and 1.5e-2, in three and two 4e-5 and 3e-4; of one that grows 3e4 5.9e-4 and 3e-3.
// An fp32 result has two steps on the first Gram matrix, where the first of them grows little enough (a up to 4), and from there on
// a Gram matrix for each step. Off from 64 bits in norm, that and fp32 products of the matrices themselves (64 x 64 to 256 x 1024):
// noise around a low rank 0.7 to 1.3e-6 and 1.0 to 2.5e-6, singular values that fall evenly over two to five decades 1.0 to 5.7e-6
// and 1.0 to 5.9e-6 (two steps, then three: 8 to 36e-6 emulated, 2 2 1: 3.5 to 10e-6), a schedule that begins with a = 8.3
// 2.3 to 19e-6 and 2.2 to 16e-6 (there with two steps first up to seven times the products).
void set_stages(fmlp::MuonCall* c, int dtype) {
  const int steps = c->steps;
  if (dtype == FMLP_DTYPE_F32) {
    const bool two = steps > 1 && c->q[0] * c->q[0] <= 16;
    c->stages = steps - two;
    c->first[0] = 0;
    for (int i = 1; i <= c->stages; ++i) c->first[i] = i + two;
    return;
  }
  // as few even ones as are of five steps at most and grow no further
  for (c->stages = (steps + 4) / 5; c->stages <= steps; ++c->stages) {
    const int n = c->stages;
    bool fits = true;
    for (int i = 0; i <= n; ++i) c->first[i] = (steps * i + n - 1) / n;
    for (int i = 0; i < n; ++i) {
      double grow = 1;
      for (int k = c->first[i]; k + 1 < c->first[i + 1]; ++k) grow *= c->q[k] * c->q[k];
      fits = fits && grow <= 2e4;
    }
    if (fits) break;
  }
}

bool known_dtype(int d) { return d == FMLP_DTYPE_F16 || d == FMLP_DTYPE_BF16 || d == FMLP_DTYPE_F32; }
int io_type(int d) { return d == FMLP_DTYPE_F32 ? fmlp::IO_F32 : d == FMLP_DTYPE_BF16 ? fmlp::IO_BF16 : fmlp::IO_F16; }
size_t elem_bytes(int d) { return d == FMLP_DTYPE_F32 ? 4 : 2; }

int check_stack(int64_t H, int64_t R, int64_t C, int i) {
  if (H < 0 || R < 0 || C < 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "stack %d: negative dimension (H=%lld R=%lld C=%lld)", i, (long long)H, (long long)R,
                    (long long)C);
  if (std::min(R, C) > fmlp::kMuonMaxSmall)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "stack %d: matrices of %lld x %lld: the smaller side is at most %d", i, (long long)R,
                    (long long)C, fmlp::kMuonMaxSmall);
  // (2^40 elements are 2 TB at least)
  if (R > 0x3fffffffLL || C > 0x3fffffffLL || H > (1LL << 40) / std::max<int64_t>(1, R * C))
    return abi_fail(FMLP_ERR_INVALID_ARG, "stack %d: dimension too large (H=%lld R=%lld C=%lld)", i, (long long)H, (long long)R,
                    (long long)C);
  return FMLP_OK;
}

int check_ptr(const void* p, const char* name, int i, size_t align) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) % align) != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%s of stack %d is NULL or not aligned to its elements", name, i);
  return FMLP_OK;
}

int check_steps(int steps) {
  if (steps < 1 || steps > fmlp::kMuonMaxSteps)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "%d steps: 1 to %d", steps, fmlp::kMuonMaxSteps);
  return FMLP_OK;
}
int set_call(fmlp::MuonCall* c, int steps, const float* coefficients, float eps, int dtype) {
  int st = check_steps(steps);
  if (st) return st;
  if (coefficients == nullptr) return abi_fail(FMLP_ERR_INVALID_ARG, "coefficients is NULL");
  if (!(eps >= 0)) return abi_fail(FMLP_ERR_INVALID_ARG, "eps is negative or NaN");
  for (int i = 0; i < 3 * steps; ++i) {
    if (!(coefficients[i] >= -1e4f && coefficients[i] <= 1e4f))
      return abi_fail(FMLP_ERR_INVALID_ARG, "coefficient %d is beyond 1e4 or NaN", i);
    c->abc[i / 3][i % 3] = coefficients[i];
  }
  c->eps = eps;
  c->steps = steps;
  fmlp::muon_bounds(c);
  set_stages(c, dtype);
  // what the terms of the steps hold: G's eigenvalues, and those of each stage's product of polynomials
  constexpr double most = 65536;
  for (int i = 0; i < c->stages; ++i) {
    double p = 1;
    for (int k = c->first[i]; k < c->first[i + 1]; ++k)
      if (!((p *= c->q[k]) <= most) || (k + 1 < steps && !(c->range[k + 1] <= most)))
        return abi_fail(FMLP_ERR_UNSUPPORTED, "coefficients of step %d: singular values up to one may grow too far (above 2^8, or 2^16 times)", k);
  }
  return FMLP_OK;
}

// the stages of a workspace's query; without coefficients those that take the most, which is any number above one
int query_call(fmlp::MuonCall* c, int steps, const float* coefficients, int dtype) {
  if (coefficients != nullptr) return set_call(c, steps, coefficients, 0.f, dtype);
  const int st = check_steps(steps);
  c->stages = c->steps = steps;
  return st;
}
// weights take the update at lr: as exact as a 16-bit result
constexpr int kUpdate = FMLP_DTYPE_BF16;

size_t plan_bytes(int n, const fmlp::MuonTensor* t, const fmlp::MuonCall& c, int cus) {
  try {
    return fmlp::muon_plan(n, t, c, cus).ws_bytes;
  } catch (const std::bad_alloc&) {  // (the call refuses)
    return 0;
  }
}

int run(int n, const fmlp::MuonTensor* t, const fmlp::MuonCall& c, void* ws, size_t ws_bytes, void* stream, const char* what) {
  int cus = 0, st;
  if ((st = fmlp::abi_num_cus(&cus))) return st;
  try {
    const fmlp::MuonPlan p = fmlp::muon_plan(n, t, c, cus);
    if (p.ws_bytes > 0 && (ws == nullptr || ws_bytes < p.ws_bytes))
      return abi_fail(FMLP_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.ws_bytes);
    if ((reinterpret_cast<uintptr_t>(ws) & 15u) != 0) return abi_fail(FMLP_ERR_INVALID_ARG, "workspace is not 16-byte aligned");
    const hipError_t e = fmlp::launch_muon(n, t, c, cus, ws, (hipStream_t)stream);
    if (e != hipSuccess) return abi_fail(FMLP_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
  } catch (const std::bad_alloc&) {
    return abi_fail(FMLP_ERR_INVALID_ARG, "no host memory for %d stacks", n);
  }
  return abi_ok();
}

fmlp::MuonTensor stack_of(int64_t H, int64_t R, int64_t C) {
  fmlp::MuonTensor t{};
  t.H = H;
  t.R = (int)R;
  t.C = (int)C;
  return t;
}

}  // namespace

FMLP_EXPORT size_t fmlp_orthogonalize_workspace_bytes_for(int64_t H, int64_t R, int64_t C, int dtype, int steps,
                                                          const float* coefficients) {
  int cus = 0;
  fmlp::MuonCall c{};
  if (check_stack(H, R, C, 0) || !known_dtype(dtype) || query_call(&c, steps, coefficients, dtype) || fmlp::abi_num_cus(&cus)) return 0;
  fmlp::MuonTensor t = stack_of(H, R, C);
  t.x_io = t.out_io = io_type(dtype);
  return plan_bytes(1, &t, c, cus);
}

FMLP_EXPORT size_t fmlp_orthogonalize_workspace_bytes(int64_t H, int64_t R, int64_t C, int dtype, int steps) {
  return fmlp_orthogonalize_workspace_bytes_for(H, R, C, dtype, steps, nullptr);
}

FMLP_EXPORT int fmlp_orthogonalize(const void* x, void* out, int64_t H, int64_t R, int64_t C, int dtype, int steps,
                                   const float* coefficients, float eps, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  int st = check_stack(H, R, C, 0);
  if (st) return st;
  if (!known_dtype(dtype)) return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", dtype);
  fmlp::MuonCall c{};
  if ((st = set_call(&c, steps, coefficients, eps, dtype))) return st;
  if (H == 0 || R == 0 || C == 0) return abi_ok();
  const size_t es = elem_bytes(dtype), bytes = (size_t)H * (size_t)R * (size_t)C * es;
  if ((st = check_ptr(x, "x", 0, es)) || (st = check_ptr(out, "out", 0, es))) return st;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(out);
  if (a != b && a < b + bytes && b < a + bytes) return abi_fail(FMLP_ERR_INVALID_ARG, "out overlaps x");
  fmlp::MuonTensor t = stack_of(H, R, C);
  t.x = x;
  t.out = out;
  t.x_io = t.out_io = io_type(dtype);
  return run(1, &t, c, workspace, workspace_bytes, stream, "orthogonalisation");
}

namespace {

int take(int n, const fmlp_muon_tensor* tensors, double lr, bool pointers, std::vector<fmlp::MuonTensor>* out,
         std::vector<fmlp::MemRange>* ranges) {
  if (n < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "%d stacks", n);
  if (n > 0 && tensors == nullptr) return abi_fail(FMLP_ERR_INVALID_ARG, "tensors is NULL");
  try {
    out->reserve((size_t)n);
    if (pointers) ranges->reserve(3 * (size_t)n);
  } catch (const std::bad_alloc&) {
    return abi_fail(FMLP_ERR_INVALID_ARG, "no host memory for %d stacks", n);
  }
  for (int i = 0; i < n; ++i) {
    const fmlp_muon_tensor& v = tensors[i];
    int st = check_stack(v.H, v.R, v.C, i);
    if (st) return st;
    for (int d : {v.w_dtype, v.g_dtype, v.m_dtype})
      if (!known_dtype(d)) return abi_fail(FMLP_ERR_UNSUPPORTED, "stack %d: dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", i, d);
    fmlp::MuonTensor t = stack_of(v.H, v.R, v.C);
    const size_t numel = (size_t)v.H * (size_t)v.R * (size_t)v.C;
    if (numel == 0) continue;
    if (pointers) {
      if ((st = check_ptr(v.w, "the weights", i, elem_bytes(v.w_dtype))) ||
          (st = check_ptr(v.g, "the gradient", i, elem_bytes(v.g_dtype))) ||
          (st = check_ptr(v.m, "the momentum", i, elem_bytes(v.m_dtype))))
        return st;
      const auto range = [&](const void* p, int dtype, bool write) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        ranges->push_back(fmlp::MemRange{a, a + numel * elem_bytes(dtype), i, write});
      };
      range(v.w, v.w_dtype, true);
      range(v.m, v.m_dtype, true);
      range(v.g, v.g_dtype, false);
    }
    t.x = v.g;
    t.m = v.m;
    t.out = v.w;
    t.x_io = io_type(v.g_dtype);
    t.m_io = io_type(v.m_dtype);
    t.out_io = io_type(v.w_dtype);
    t.lr = (float)(lr * (double)v.scale);
    out->push_back(t);
  }
  return FMLP_OK;
}

}  // namespace

FMLP_EXPORT size_t fmlp_muon_workspace_bytes_for(int n, const fmlp_muon_tensor* tensors, int steps, const float* coefficients) {
  int cus = 0;
  std::vector<fmlp::MuonTensor> t;
  fmlp::MuonCall c{};
  if (query_call(&c, steps, coefficients, kUpdate) || take(n, tensors, 0, false, &t, nullptr) || fmlp::abi_num_cus(&cus)) return 0;
  c.update = 1;
  for (fmlp::MuonTensor& v : t)
    if (v.m == nullptr) v.m = &c;  // (a momentum whose address is not known yet)
  return plan_bytes((int)t.size(), t.data(), c, cus);
}

FMLP_EXPORT size_t fmlp_muon_workspace_bytes(int n, const fmlp_muon_tensor* tensors, int steps) {
  return fmlp_muon_workspace_bytes_for(n, tensors, steps, nullptr);
}

FMLP_EXPORT int fmlp_muon_step(int n, const fmlp_muon_tensor* tensors, double lr, double momentum, int nesterov,
                               double weight_decay, int steps, const float* coefficients, float eps, void* workspace,
                               size_t workspace_bytes, void* stream) {
  fmlp::MuonCall c{};
  int st = set_call(&c, steps, coefficients, eps, kUpdate);
  if (st) return st;
  if (!(lr >= 0) || !(weight_decay >= 0) || !(momentum >= 0 && momentum <= 1))
    return abi_fail(FMLP_ERR_INVALID_ARG, "lr or weight_decay is negative or NaN, or momentum outside [0, 1]");
  std::vector<fmlp::MuonTensor> t;
  std::vector<fmlp::MemRange> ranges;
  if ((st = take(n, tensors, lr, true, &t, &ranges))) return st;
  int one, two;
  if (fmlp::mem_overlap(ranges, &one, &two))
    return abi_fail(FMLP_ERR_INVALID_ARG, "the weights or momenta of stack %d or %d overlap another tensor of the call", one, two);
  if (t.empty()) return abi_ok();
  c.mu = (float)momentum;
  c.nu = (float)(1.0 - momentum);
  c.nesterov = nesterov != 0;
  c.keep = (float)(1.0 - lr * weight_decay);
  c.update = 1;
  return run((int)t.size(), t.data(), c, workspace, workspace_bytes, stream, "muon step");
}

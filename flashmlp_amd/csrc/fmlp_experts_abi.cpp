// C ABI of the experts' operators (declared in include/flashmlp.h): argument validation and dispatch, as
// fmlp_block_abi.cpp does for the gated block. No allocation, no synchronisation.
#include "../../include/flashmlp.h"
#include "fmlp_block.h"
#include "fmlp_experts.h"

#define FMLP_EXPORT extern "C" __attribute__((visibility("default")))

using fmlp::abi_fail;
using fmlp::abi_ok;

namespace {

constexpr int64_t kMaxRows = 0x7fffffffLL;

bool known_dtype(int d) { return d == FMLP_DTYPE_F16 || d == FMLP_DTYPE_BF16 || d == FMLP_DTYPE_F32; }
int io_type(int d) { return d == FMLP_DTYPE_F32 ? fmlp::IO_F32 : d == FMLP_DTYPE_BF16 ? fmlp::IO_BF16 : fmlp::IO_F16; }
size_t elem_bytes(int d) { return d == FMLP_DTYPE_F32 ? 4 : 2; }

int check_ptr(const void* p, const char* name, bool needed, size_t align) {
  if (p == nullptr) return needed ? abi_fail(FMLP_ERR_INVALID_ARG, "%s is NULL", name) : FMLP_OK;
  if ((reinterpret_cast<uintptr_t>(p) % align) != 0)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%s is not %zu-byte aligned", name, align);
  return FMLP_OK;
}

int check_counts(int64_t T, int64_t N, int64_t k) {
  if (T < 0 || N < 1 || k < 1)
    return abi_fail(FMLP_ERR_INVALID_ARG, "dimensions T=%lld N=%lld k=%lld", (long long)T, (long long)N, (long long)k);
  if (N > fmlp::kMaxExperts)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "%lld experts: at most %lld", (long long)N, (long long)fmlp::kMaxExperts);
  if (k > fmlp::kMaxChoices)
    return abi_fail(FMLP_ERR_UNSUPPORTED, "%lld experts a token: at most %lld", (long long)k, (long long)fmlp::kMaxChoices);
  if (T > kMaxRows / k) return abi_fail(FMLP_ERR_INVALID_ARG, "too many tokens (%lld x %lld)", (long long)T, (long long)k);
  return FMLP_OK;
}

int check_route(const void* logits, bool needed, int64_t T, int64_t N, int64_t row_stride, int64_t k, int dtype) {
  int st = check_counts(T, N, k);
  if (st) return st;
  if (k > N) return abi_fail(FMLP_ERR_INVALID_ARG, "%lld of %lld experts a token", (long long)k, (long long)N);
  if (!known_dtype(dtype)) return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", dtype);
  if (row_stride < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "row stride is negative (%lld)", (long long)row_stride);
  return check_ptr(logits, "logits", needed && T > 0, elem_bytes(dtype));
}

int check_rows(int64_t T, int64_t k, int64_t N, int64_t capacity, int64_t D, int dtype) {
  int st = check_counts(T, N, k);
  if (st) return st;
  if (capacity < 0 || D < 1)
    return abi_fail(FMLP_ERR_INVALID_ARG, "dimensions capacity=%lld D=%lld", (long long)capacity, (long long)D);
  if (D > (1LL << 24)) return abi_fail(FMLP_ERR_UNSUPPORTED, "%lld columns: at most 2^24", (long long)D);
  if (capacity > kMaxRows / N)
    return abi_fail(FMLP_ERR_INVALID_ARG, "%lld experts of %lld rows: more than 2^31 - 1", (long long)N, (long long)capacity);
  if (!known_dtype(dtype)) return abi_fail(FMLP_ERR_UNSUPPORTED, "dtype code %d: fp16 (0), bf16 (1) or fp32 (2)", dtype);
  return FMLP_OK;
}

int finish(hipError_t e, const char* what) {
  return e == hipSuccess ? abi_ok() : abi_fail(FMLP_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

}  // namespace

FMLP_EXPORT int fmlp_route_fwd(const void* logits, float* weights, int32_t* experts, int64_t T, int64_t N, int64_t row_stride,
                               int64_t k, int normalize, int dtype, void* stream) {
  int st;
  if ((st = check_route(logits, true, T, N, row_stride, k, dtype)) || (st = check_ptr(weights, "weights", T > 0, 4)) ||
      (st = check_ptr(experts, "experts", T > 0, 4)))
    return st;
  fmlp::RouteArgs a{};
  a.logits = logits;
  a.weights = weights;
  a.experts = experts;
  a.T = T;
  a.stride = row_stride;
  a.N = (int)N;
  a.k = (int)k;
  a.normalize = normalize != 0;
  a.io = io_type(dtype);
  return finish(fmlp::launch_route_fwd(a, (hipStream_t)stream), "route forward");
}

FMLP_EXPORT int fmlp_route_bwd(const void* logits, const float* weights, const int32_t* experts, const float* dweights,
                               void* dlogits, int64_t T, int64_t N, int64_t row_stride, int64_t k, int normalize, int dtype,
                               void* stream) {
  int st;
  if ((st = check_route(logits, normalize == 0, T, N, row_stride, k, dtype)) ||
      (st = check_ptr(weights, "weights", T > 0, 4)) || (st = check_ptr(experts, "experts", T > 0, 4)) ||
      (st = check_ptr(dweights, "dweights", T > 0, 4)) || (st = check_ptr(dlogits, "dlogits", T > 0, elem_bytes(dtype))))
    return st;
  fmlp::RouteArgs a{};
  a.logits = logits;
  a.weights = const_cast<float*>(weights);
  a.experts = const_cast<int32_t*>(experts);
  a.dweights = dweights;
  a.dlogits = dlogits;
  a.T = T;
  a.stride = row_stride;
  a.N = (int)N;
  a.k = (int)k;
  a.normalize = normalize != 0;
  a.io = io_type(dtype);
  return finish(fmlp::launch_route_bwd(a, (hipStream_t)stream), "route backward");
}

FMLP_EXPORT size_t fmlp_expert_plan_workspace_bytes(int64_t T, int64_t k, int64_t N) {
  return check_counts(T, N, k) ? 0 : fmlp::expert_plan(T * k, N).ws_bytes;
}

FMLP_EXPORT int fmlp_expert_plan(const void* experts, int index_bytes, int32_t* slots, int32_t* counts, int64_t T, int64_t k,
                                 int64_t N, int64_t capacity, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_rows(T, k, N, capacity, 1, FMLP_DTYPE_F32);
  if (st) return st;
  if (index_bytes != 4 && index_bytes != 8)
    return abi_fail(FMLP_ERR_INVALID_ARG, "experts of %d bytes: 4 or 8", index_bytes);
  if ((st = check_ptr(experts, "experts", T > 0, (size_t)index_bytes)) || (st = check_ptr(slots, "slots", T > 0, 4)) ||
      (st = check_ptr(counts, "counts", true, 4)) || (st = check_ptr(workspace, "workspace", false, 4)))
    return st;
  const fmlp::ExpertPlan p = fmlp::expert_plan(T * k, N);
  if (p.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < p.ws_bytes))
    return abi_fail(FMLP_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, p.ws_bytes);
  return finish(fmlp::launch_expert_plan(experts, index_bytes == 8, T * k, (int)N, capacity, slots, counts, p, workspace,
                                         (hipStream_t)stream),
                "expert plan");
}

FMLP_EXPORT int fmlp_expert_scatter(const void* x, int64_t x_row_stride, const float* weights, const int32_t* slots,
                                    const int32_t* counts, const void* rows_in, void* rows_out, float* dweights, int64_t T,
                                    int64_t k, int64_t N, int64_t capacity, int64_t D, int dtype, void* stream) {
  int st = check_rows(T, k, N, capacity, D, dtype);
  if (st) return st;
  const size_t es = elem_bytes(dtype);
  const bool rows = capacity > 0;
  if (x_row_stride < 0) return abi_fail(FMLP_ERR_INVALID_ARG, "x row stride is negative (%lld)", (long long)x_row_stride);
  if (rows_out == nullptr && dweights == nullptr && rows) return abi_fail(FMLP_ERR_INVALID_ARG, "no output is asked for");
  if ((st = check_ptr(x, "x", T > 0, es)) || (st = check_ptr(weights, "weights", false, 4)) ||
      (st = check_ptr(slots, "slots", T > 0, 4)) || (st = check_ptr(counts, "counts", rows && rows_out != nullptr, 4)) ||
      (st = check_ptr(rows_in, "rows_in", rows && T > 0 && dweights != nullptr, es)) ||
      (st = check_ptr(rows_out, "rows_out", false, es)) || (st = check_ptr(dweights, "dweights", false, 4)))
    return st;
  fmlp::ExpertCopyArgs a{};
  a.x = x;
  a.rows_in = rows_in;
  a.rows_out = rows ? rows_out : nullptr;
  a.weights = weights;
  a.dweights = dweights;
  a.slots = slots;
  a.counts = counts;
  a.T = T;
  a.N = N;
  a.capacity = capacity;
  a.D = D;
  a.stride = x_row_stride;
  a.k = (int)k;
  a.io = io_type(dtype);
  if (a.rows_out == nullptr && dweights == nullptr) return abi_ok();
  return finish(fmlp::launch_expert_scatter(a, (hipStream_t)stream), "expert scatter");
}

FMLP_EXPORT int fmlp_expert_gather(const void* rows, const float* weights, const int32_t* slots, void* o, int64_t T, int64_t k,
                                   int64_t N, int64_t capacity, int64_t D, int dtype, void* stream) {
  int st = check_rows(T, k, N, capacity, D, dtype);
  if (st) return st;
  const size_t es = elem_bytes(dtype);
  if ((st = check_ptr(rows, "rows", T > 0 && capacity > 0, es)) || (st = check_ptr(weights, "weights", false, 4)) ||
      (st = check_ptr(slots, "slots", T > 0, 4)) || (st = check_ptr(o, "o", T > 0, es)))
    return st;
  fmlp::ExpertCopyArgs a{};
  a.rows_in = rows;
  a.o = o;
  a.weights = weights;
  a.slots = slots;
  a.T = T;
  a.N = N;
  a.capacity = capacity;
  a.D = D;
  a.k = (int)k;
  a.io = io_type(dtype);
  return finish(fmlp::launch_expert_gather(a, (hipStream_t)stream), "expert gather");
}

// Tokens sorted by expert and back, for gfx950.
//
//   plan:     assignment i = t k + j of token t has its expert's position p = number of earlier assignments to the same
//             expert, and the slot e capacity + p, or -1 where p >= capacity or its expert is out of [0, N)
//   scatter:  rows[slot(t, j)] = w(t, j) x(t), zeros behind an expert's last row; dw(t, j) = <rows_in[slot(t, j)], x(t)>
//   gather:   o(t) = sum over j of w(t, j) rows[slot(t, j)], in fp32 in the order of j, rounded once
//
// The plan is a stable counting sort: positions follow the tokens' order whatever the workgroups' order. Chunks of
// assignments are counted first; then each chunk adds what the chunks before it have of every expert, its waves' counts
// follow one another, and a wave's 64 assignments find those of their own expert by one ballot for each bit of it.
//
// The copies are bound by HBM. A token has a group of lanes, 16 bytes a lane; it is read once and written to its k rows (dispatch), so
// that no inverse map is needed: what is left of an expert's capacity is filled with zeros by workgroups of their own.
//
// Measured, 2^19 tokens of 128 bf16 columns, 32 experts of 40960 rows, 2 a token: plan 18 us (2 launches), scatter 82 (470 MB,
// 5.7 TB/s), gather 75-83 (403 MB, 4.9 to 5.4 TB/s), scatter with weights and their gradient 138 (737 MB, 5.3 TB/s); a copy reaches 5.2.
// Loads without branches around them (dropped choices read some row and throw it away) measured the same.
#include <algorithm>

#include "fmlp_experts.h"
#include "fmlp_vec.h"

namespace fmlp {
namespace {

// ---------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------
constexpr int kItems = 16;  // assignments of a lane, at most; a power of two

// expert of assignment i, -1 for none; past the last one too, whose load is then the last one's (a branch around it would have
// every load waited for before the next)
template <bool WIDE>
__device__ __forceinline__ int expert_at(const void* experts, long long i, long long M, int N) {
  const long long at = i < M ? i : M - 1;
  long long e;
  if constexpr (WIDE) e = ((const long long*)experts)[at];
  else e = ((const int*)experts)[at];
  return i < M && e >= 0 && e < N ? (int)e : -1;
}

template <bool WIDE, int ITEMS>
__global__ void __launch_bounds__(256) plan_count_kernel(const void* experts, long long M, int N, int* hist) {
  extern __shared__ int plan_lds[];
  const long long i0 = (long long)blockIdx.x * (256 * ITEMS) + threadIdx.x;
  int ex[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) ex[u] = expert_at<WIDE>(experts, i0 + u * 256, M, N);
  for (int e = threadIdx.x; e < N; e += 256) plan_lds[e] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (ex[u] >= 0) atomicAdd(&plan_lds[ex[u]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < N; e += 256) hist[(long long)blockIdx.x * N + e] = plan_lds[e];
}

__global__ void __launch_bounds__(256) plan_none_kernel(int* counts, int N) {
  for (int e = threadIdx.x; e < N; e += 256) counts[e] = 0;
}

// hist[c][e] = the sum of hist[c'][e] over c' < c, a wave an expert
__global__ void __launch_bounds__(256) plan_scan_kernel(int* hist, long long chunks, int N) {
  const int e = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = (int)threadIdx.x & 63;
  if (e >= N) return;
  int base = 0;
  for (long long c0 = 0; c0 < chunks; c0 += 256) {
    int v[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // four chunks a lane
      const long long c = c0 + lane * 4 + j;
      v[j] = c < chunks ? hist[c * N + e] : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += v[j];
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    int at = base + upto - sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long c = c0 + lane * 4 + j;
      if (c < chunks) hist[c * N + e] = at;
      at += v[j];
    }
    base += __shfl(upto, 63, 64);
  }
}

// THREADS * ITEMS assignments of workgroup blockIdx.x. hist: null for one workgroup; else every chunk's counts, or where
// `scanned` what the chunks before it have.
template <bool WIDE, int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) plan_kernel(const void* experts, long long M, int N, int bits, long long capacity,
                                                       int* slots, int* counts, const int* hist, int scanned) {
  extern __shared__ int plan_lds[];  // [waves][N]: the wave's counts, then its next position of each expert; [N] what is before
  constexpr int W = THREADS / 64;
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
  int* mine = plan_lds + wave * N;
  int* before = plan_lds + W * N;
  const long long i0 = ((long long)blockIdx.x * W + wave) * (64 * ITEMS) + lane;
  int ex[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) ex[u] = expert_at<WIDE>(experts, i0 + u * 64, M, N);
  for (int e = threadIdx.x; e < (W + 1) * N; e += THREADS) plan_lds[e] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (ex[u] >= 0) atomicAdd(&mine[ex[u]], 1);
  if (hist != nullptr) {
    if (scanned) {
      for (int e = threadIdx.x; e < N; e += THREADS) before[e] = hist[(long long)blockIdx.x * N + e];
    } else {
      // the chunks before this one, dealt to as many groups of threads as there are for the experts
      int lanes = 1;
      while (lanes < N) lanes <<= 1;
      const int parts = THREADS / min(lanes, THREADS), e = (int)threadIdx.x & (lanes - 1), part = (int)threadIdx.x / min(lanes, THREADS);
      for (int e1 = e; e1 < N; e1 += THREADS) {
        int sum = 0;
#pragma unroll 8
        for (int c = part; c < (int)blockIdx.x; c += parts) sum += hist[(long long)c * N + e1];
        if (sum) atomicAdd(&before[e1], sum);
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < N; e += THREADS) {
    int at = before[e];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int n = plan_lds[w * N + e];
      plan_lds[w * N + e] = at;
      at += n;
    }
    if (blockIdx.x + 1 == gridDim.x) counts[e] = at;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int e = ex[u];
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long v = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? v : ~v;
    }
    const long long i = i0 + u * 64;
    const int rank = __popcll(same & ((1ull << lane) - 1));
    int base = 0;
    if (e >= 0) {
      base = mine[e];
      // (the wave's lanes have all read before the last one of each expert writes: one wave's LDS operations keep
      // their order)
      asm volatile("" ::: "memory");
      if ((same >> lane) == 1) mine[e] = base + rank + 1;
    }
    asm volatile("" ::: "memory");
    if (i < M) {
      const long long p = (long long)base + rank;
      slots[i] = e >= 0 && p < capacity ? (int)(e * capacity + p) : -1;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------------------------
constexpr int kFillBytes = 65536;  // of a workgroup that fills with zeros

// Zeros behind expert e's rows, in chunk c of `chunk` rows.
template <int IO>
__device__ __forceinline__ void fill_rows(const ExpertCopyArgs& a, long long e, long long r0, long long chunk) {
  const long long r1 = min(a.capacity, r0 + chunk);
  const long long from = max(r0, (long long)max(a.counts[e], 0));
  if (from >= r1) return;
  constexpr int E = kPiece<IO>;
  const long long i1 = (e * a.capacity + r1) * a.D;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (long long i = (e * a.capacity + from) * a.D + threadIdx.x * E; i < i1; i += 256 * E)
    store_piece<IO>(a.rows_out, i, i1 - i < E ? (int)(i1 - i) : E, zero);
}

// KB: choices of a token in flight; 1 << lg lanes a token. rows_out and dweights may each be null.
template <int IO, int KB, bool W, bool DOT>
__global__ void __launch_bounds__(256) scatter_kernel(ExpertCopyArgs a, int lg, unsigned fill_blocks, unsigned fill_chunks,
                                                      long long fill_rows_each) {
  if (blockIdx.x < fill_blocks) {
    fill_rows<IO>(a, blockIdx.x / fill_chunks, (long long)(blockIdx.x % fill_chunks) * fill_rows_each, fill_rows_each);
    return;
  }
  constexpr int E = kPiece<IO>;
  const int L = 1 << lg, lane = (int)threadIdx.x & (L - 1);
  const long long t = (long long)(blockIdx.x - fill_blocks) * (256 >> lg) + (threadIdx.x >> lg);
  const bool there = t < a.T;
  const long long x0 = there ? t * a.stride : 0, n_rows = a.N * a.capacity;
  const int D = (int)a.D, k = a.k;
  for (int j0 = 0; j0 < k; j0 += KB) {
    int slot[KB];
    float w[KB], dot[KB];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      slot[j] = there && j0 + j < k ? a.slots[t * k + j0 + j] : -1;
      if (slot[j] >= n_rows) slot[j] = -1;
      if constexpr (W) w[j] = slot[j] >= 0 ? a.weights[t * k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    for (int d = lane * E; d < D; d += L * E) {
      const int n = there ? D - d : 0;
      const u32x4 v = load_piece<IO>(a.x, x0 + d, n);
      float f[E];
      if constexpr (W || DOT) unpack_piece<IO>(v, f);
      if constexpr (DOT) {
        u32x4 r[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j)
          r[j] = load_piece<IO>(a.rows_in, slot[j] >= 0 ? (long long)slot[j] * D + d : 0, slot[j] >= 0 ? n : 0);
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          float q[E];
          unpack_piece<IO>(r[j], q);
#pragma unroll
          for (int i = 0; i < E; ++i) dot[j] = __builtin_fmaf(q[i], f[i], dot[j]);
        }
      }
      if (!DOT || a.rows_out != nullptr) {
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          if (slot[j] < 0) continue;
          if constexpr (W) {
            float q[E];
#pragma unroll
            for (int i = 0; i < E; ++i) q[i] = w[j] * f[i];
            store_piece<IO>(a.rows_out, (long long)slot[j] * D + d, n, pack_piece<IO>(q));
          } else {
            store_piece<IO>(a.rows_out, (long long)slot[j] * D + d, n, v);
          }
        }
      }
    }
    if constexpr (DOT) {
#pragma unroll
      for (int j = 0; j < KB; ++j)
        for (int s = 1; s < L; s <<= 1) dot[j] += __shfl_xor(dot[j], s, 64);
      if (there && lane == 0)
#pragma unroll
        for (int j = 0; j < KB; ++j)
          if (j0 + j < k) a.dweights[t * k + j0 + j] = slot[j] >= 0 ? dot[j] : 0.f;  // (0 infinity is no 0)
    }
  }
}

template <int IO, int KB, bool W>
__global__ void __launch_bounds__(256) gather_kernel(ExpertCopyArgs a, int lg) {
  constexpr int E = kPiece<IO>;
  const int L = 1 << lg, lane = (int)threadIdx.x & (L - 1);
  const long long t = (long long)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
  if (t >= a.T) return;
  const long long n_rows = a.N * a.capacity;
  const int D = (int)a.D, k = a.k;
  for (int d = lane * E; d < D; d += L * E) {
    float acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += KB) {
      u32x4 r[KB];
      float w[KB];
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        const int slot = j0 + j < k ? a.slots[t * k + j0 + j] : -1;
        const bool in = slot >= 0 && slot < n_rows;
        w[j] = !in ? 0.f : W ? a.weights[t * k + j0 + j] : 1.f;
        r[j] = load_piece<IO>(a.rows_in, in ? (long long)slot * D + d : 0, in ? D - d : 0);
      }
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        float q[E];
        unpack_piece<IO>(r[j], q);
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = W ? __builtin_fmaf(w[j], q[i], acc[i]) : acc[i] + q[i];
      }
    }
    store_piece<IO>(a.o, t * D + d, D - d, pack_piece<IO>(acc));
  }
}

// lanes of a token: its 16-byte pieces up to a wave
int lanes_log2(long long D, int io) {
  const long long e = io == IO_F32 ? 4 : 8;
  int lg = 0;
  while (lg < 6 && (e << lg) < D) ++lg;
  return lg;
}

template <typename F>
void by_io(int io, F f) {
  if (io == IO_F32) f(std::integral_constant<int, IO_F32>{});
  else if (io == IO_BF16) f(std::integral_constant<int, IO_BF16>{});
  else f(std::integral_constant<int, IO_F16>{});
}
template <typename F>
void by_choices(int k, F f) {
  if (k == 1) f(std::integral_constant<int, 1>{});
  else if (k == 2) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}

}  // namespace

ExpertPlan expert_plan(int64_t M, int64_t N) {
  ExpertPlan p{};
  // One workgroup of 16 waves does all where a lane has at most 4 items: no second launch. Else about 256 workgroups, whose
  // lanes' items follow one another: 16384 assignments by one workgroup 14 us, by 64 9.
  p.threads = M <= 1024 * 4 ? 1024 : 256;
  const long long per = p.threads == 1024 ? 1024 : 65536;
  p.items = 1;
  while (p.items < kItems && p.items * per < M) p.items *= 2;
  p.chunks = p.threads == 1024 ? 1 : (M + 256 * p.items - 1) / (256 * p.items);
  p.ws_bytes = p.chunks > 1 ? (size_t)(p.chunks * N) * sizeof(int) : 0;
  // The workgroups add up the chunks before them themselves where that is at most 32 rounds of their 256 threads (M = 196608, N = 12:
  // 14 us, with a scan in a launch of its own 15.6); a scan takes over from there (M = 2^20, N = 256: 28 us without, 20 with it).
  long long lanes = 1;
  while (lanes < N) lanes <<= 1;
  p.scan = p.chunks > 1 && p.chunks * lanes > 32 * 256;
  return p;
}

hipError_t launch_expert_plan(const void* experts, bool wide, long long M, int N, long long capacity, int32_t* slots,
                              int32_t* counts, const ExpertPlan& p, void* ws, hipStream_t st) {
  int bits = 0;
  while ((1 << bits) < N) ++bits;
  int* hist = p.chunks > 1 ? (int*)ws : nullptr;
  const dim3 grid((unsigned)p.chunks);
  hipError_t e = hipSuccess;
  const auto run = [&](auto WIDE, auto THREADS, auto ITEMS) {
    constexpr bool V = decltype(WIDE)::value;
    constexpr int TH = decltype(THREADS)::value, IT = decltype(ITEMS)::value;
    if (hist != nullptr) {
      hipLaunchKernelGGL((plan_count_kernel<V, IT>), grid, dim3(256), (size_t)N * 4, st, experts, M, N, hist);
      if ((e = hipGetLastError()) != hipSuccess) return;
      if (p.scan) {
        hipLaunchKernelGGL(plan_scan_kernel, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, st, hist, p.chunks, N);
        if ((e = hipGetLastError()) != hipSuccess) return;
      }
    }
    const size_t lds = ((size_t)TH / 64 + 1) * N * 4;
    auto k = plan_kernel<V, TH, IT>;
    static std::atomic<unsigned long long> done{0};
    if (lds > 65536 && (e = set_lds_once((const void*)k, 17 * (int)kMaxExperts * 4, done)) != hipSuccess) return;
    hipLaunchKernelGGL(k, grid, dim3(TH), lds, st, experts, M, N, bits, capacity, slots, counts, hist, (int)p.scan);
    e = hipGetLastError();
  };
  const auto by_items = [&](auto WIDE) {
    const auto one = [&](auto THREADS, auto ITEMS) { run(WIDE, THREADS, ITEMS); };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    using I16 = std::integral_constant<int, kItems>;
    using T256 = std::integral_constant<int, 256>;
    using T1024 = std::integral_constant<int, 1024>;
    if (p.threads == 1024) {
      if (p.items == 1) one(T1024{}, I1{});
      else if (p.items == 2) one(T1024{}, I2{});
      else one(T1024{}, I4{});
    } else if (p.items == 1) one(T256{}, I1{});
    else if (p.items == 2) one(T256{}, I2{});
    else if (p.items == 4) one(T256{}, I4{});
    else if (p.items == 8) one(T256{}, I8{});
    else one(T256{}, I16{});
  };
  if (M == 0) {  // (nothing to read; the counts are zeros)
    hipLaunchKernelGGL(plan_none_kernel, dim3(1), dim3(256), 0, st, counts, N);
    return hipGetLastError();
  }
  if (wide) by_items(std::true_type{});
  else by_items(std::false_type{});
  return e;
}

// Tokens of a launch: those beyond kLaunchThreads' (2^25 of more than 512 bytes) take another.
ExpertCopyArgs from_token(const ExpertCopyArgs& all, long long t0, long long most) {
  const long long es = all.io == IO_F32 ? 4 : 2;
  ExpertCopyArgs a = all;
  a.T = std::min(most, all.T - t0);
  a.x = (const char*)all.x + t0 * all.stride * es;
  if (all.o) a.o = (char*)all.o + t0 * all.D * es;
  a.slots += t0 * all.k;
  if (all.weights) a.weights += t0 * all.k;
  if (all.dweights) a.dweights += t0 * all.k;
  return a;
}

hipError_t launch_expert_scatter(const ExpertCopyArgs& all, hipStream_t st) {
  const int lg = lanes_log2(all.D, all.io);
  const long long per = 256 >> lg, most = kLaunchThreads / 256;
  const long long row_bytes = all.D * (all.io == IO_F32 ? 4 : 2);
  const long long chunk = std::max(1LL, kFillBytes / row_bytes);
  const long long chunks = all.rows_out != nullptr ? (all.capacity + chunk - 1) / chunk : 0;
  if (chunks * all.N >= most) return hipErrorInvalidValue;  // (2^23 times 64 KB)
  for (long long t0 = 0; t0 < all.T || t0 == 0; t0 += most * per) {
    const ExpertCopyArgs a = from_token(all, t0, most * per);
    const long long fill = t0 == 0 ? chunks * a.N : 0, grid = (a.T + per - 1) / per + fill;
    if (grid == 0) return hipSuccess;
    by_io(a.io, [&](auto IO) {
      by_choices(a.k, [&](auto KB) {
        constexpr int I = decltype(IO)::value, K = decltype(KB)::value;
        const auto go = [&](auto k) {
          hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(256), 0, st, a, lg, (unsigned)fill, (unsigned)std::max(chunks, 1LL), chunk);
        };
        if (a.dweights != nullptr) a.weights ? go(scatter_kernel<I, K, true, true>) : go(scatter_kernel<I, K, false, true>);
        else a.weights ? go(scatter_kernel<I, K, true, false>) : go(scatter_kernel<I, K, false, false>);
      });
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_expert_gather(const ExpertCopyArgs& all, hipStream_t st) {
  const int lg = lanes_log2(all.D, all.io);
  const long long per = 256 >> lg, most = kLaunchThreads / 256 * per;
  for (long long t0 = 0; t0 < all.T; t0 += most) {
    const ExpertCopyArgs a = from_token(all, t0, most);
    const dim3 grid((unsigned)((a.T + per - 1) / per));
    by_io(a.io, [&](auto IO) {
      by_choices(a.k, [&](auto KB) {
        constexpr int I = decltype(IO)::value, K = decltype(KB)::value;
        if (a.weights) hipLaunchKernelGGL((gather_kernel<I, K, true>), grid, dim3(256), 0, st, a, lg);
        else hipLaunchKernelGGL((gather_kernel<I, K, false>), grid, dim3(256), 0, st, a, lg);
      });
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace fmlp

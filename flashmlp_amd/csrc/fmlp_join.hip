// A block's output joined to its residual stream, and the next block's input taken from it, on gfx950.
//
//   n = o rsqrt(mean(o^2) + eps)     p = n w_post           (post norm; without it p = o)
//   r' = r + s gate p                                        (stream; without o, r' = r)
//   y = r' rsqrt(mean(r'^2) + eps) w_pre                     (pre norm of the next block)
//
// and the gradients, with m = r' rs_r, dm = dy w_pre:
//   dr = dr' + rs_r (dm - m mean(dm m))                      dw_pre  = sum_rows dy m
//   dp = s gate dr                                           dgate   = sum_{rows of a group} s dr p
//   do = rs_o (dn - n mean(dn n)),  dn = dp w_post           dw_post = sum_rows dp n
//
// One pass over the data each way: a row's C = heads x D columns stay in registers between the sums
// that need all of them and the results, so that the forward reads o and r and writes r' and y, and the
// backward reads r (or r'), o, dr', dy and writes dr, do. o and y are head-major (H, B, D), the layout of the
// MLP kernels, or rows of C columns; the transposition costs nothing, a vector of 8 columns lies in one
// head. Both are bound by HBM bytes; sums are fp32. 16384 x 4096 bf16: forward 112 us (537 MB, 4.8 TB/s), backward 188
// (805 MB, 4.3 TB/s; from the rounded r' 177) and 6 for the column sums; a copy of 1 GiB reaches 5.0 TB/s. Four rows: 5.9 us a call, all launch.
// The backward keeps a row's data and three column sums in registers, which 128 do not always hold: 2 spill at 1024 to
// 8192 columns of a 16-bit stream, 8 to 20 of an fp32 one past 4096, 186 to 276 with two vectors a thread (8192 x 16384 bf16: 1700 us,
// 0.95 TB/s), and 52 to 209 (two vectors: 335 to 1220) element by element past 1024 columns. Element by element every column also
// finds its head by a division: 4096 x (32 x 100) forward 47 us, backward 129 (1.2 TB/s), by vectors (32 x 104) 27 and 47.
#include <algorithm>

#include "fmlp_block.h"
#include "fmlp_device.h"

namespace fmlp {
namespace {

template <int IO>
struct Elem {
  typedef u16 T;
};
template <>
struct Elem<IO_F32> {
  typedef float T;
};

template <int IO>
__device__ __forceinline__ float wide(typename Elem<IO>::T v) {
  if constexpr (IO == IO_F32) return v;
  else return to_f32<IO == IO_BF16>(v);
}
template <int IO>
__device__ __forceinline__ typename Elem<IO>::T narrow(float v) {
  if constexpr (IO == IO_F32) return v;
  else return from_f32<IO == IO_BF16>(v);
}

// 8 elements as they are in memory
template <int IO>
struct Vec {
  u32x4 v[IO == IO_F32 ? 2 : 1];
  __device__ __forceinline__ float get(int j) const {
    if constexpr (IO == IO_F32) return __uint_as_float(v[j >> 2][j & 3]);
    else return (j & 1) ? hi_f32<IO == IO_BF16>(v[0][j >> 1]) : lo_f32<IO == IO_BF16>(v[0][j >> 1]);
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    static_assert(IO != IO_F32, "16-bit elements");
    constexpr bool BF = IO == IO_BF16;
    v[0] = u32x4{pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7])};
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& q : v) q = u32x4{0u, 0u, 0u, 0u};
  }
};

// what was computed from v is not kept: the compiler takes v for new (no instruction)
template <int IO>
__device__ __forceinline__ void forget(Vec<IO>& v) {
#pragma unroll
  for (auto& q : v.v) asm volatile("" : "+v"(q));
}

// A row's columns over the tpr threads that own it. Vectors (ALIGNED): thread t's vector k holds columns
// 8 (t + k tpr) .. + 7. Else element j of it is column t + (8 k + j) tpr, read and written by itself.
template <bool ALIGNED>
__device__ __forceinline__ int column(int t, int tpr, int k, int j) {
  return ALIGNED ? 8 * (t + k * tpr) + j : t + (8 * k + j) * tpr;
}

// where a row of o, y, do, dy lies: head stride sh and row stride sr in elements, D columns a head
struct HeadRows {
  long long sh, sr;
  int D;
};

template <int IO, bool ALIGNED>
__device__ __forceinline__ Vec<IO> load_row(const void* base, long long row_off, int C, int t, int tpr, int k) {
  typedef typename Elem<IO>::T T;
  Vec<IO> r;
  r.zero();
  const T* p = (const T*)base + row_off;
  if constexpr (ALIGNED) {
    const int c = column<true>(t, tpr, k, 0);
    if (c < C) {
#pragma unroll
      for (unsigned q = 0; q < sizeof(r.v) / 16; ++q) r.v[q] = ((const u32x4*)(p + c))[q];
    }
  } else {
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(t, tpr, k, j);
      e[j] = c < C ? p[c] : (T)0;
    }
    __builtin_memcpy(r.v, e, sizeof(e));
  }
  return r;
}

template <int IO, bool ALIGNED>
__device__ __forceinline__ Vec<IO> load_heads(const void* base, HeadRows hr, long long row, int C, int t, int tpr, int k) {
  typedef typename Elem<IO>::T T;
  Vec<IO> r;
  r.zero();
  const T* p = (const T*)base + row * hr.sr;
  if constexpr (ALIGNED) {
    const int c = column<true>(t, tpr, k, 0);
    if (c < C) {
      const int h = (int)((unsigned)c / (unsigned)hr.D);
      const T* q0 = p + h * hr.sh + (c - h * hr.D);
#pragma unroll
      for (unsigned q = 0; q < sizeof(r.v) / 16; ++q) r.v[q] = ((const u32x4*)q0)[q];
    }
  } else {
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(t, tpr, k, j);
      const int h = (int)((unsigned)c / (unsigned)hr.D);
      e[j] = c < C ? p[h * hr.sh + (c - h * hr.D)] : (T)0;
    }
    __builtin_memcpy(r.v, e, sizeof(e));
  }
  return r;
}

template <int IO>
__device__ __forceinline__ void store8(typename Elem<IO>::T* p, const float (&f)[8]) {
  if constexpr (IO == IO_F32) {
    ((float4*)p)[0] = float4{f[0], f[1], f[2], f[3]};
    ((float4*)p)[1] = float4{f[4], f[5], f[6], f[7]};
  } else {
    constexpr bool BF = IO == IO_BF16;
    *(u32x4*)p = u32x4{pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7])};
  }
}

template <int IO, bool ALIGNED>
__device__ __forceinline__ void store_row(void* base, long long row_off, int C, int t, int tpr, int k, const float (&f)[8]) {
  typedef typename Elem<IO>::T T;
  T* p = (T*)base + row_off;
  if constexpr (ALIGNED) {
    const int c = column<true>(t, tpr, k, 0);
    if (c < C) store8<IO>(p + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(t, tpr, k, j);
      if (c < C) p[c] = narrow<IO>(f[j]);
    }
  }
}

template <int IO, bool ALIGNED>
__device__ __forceinline__ void store_heads(void* base, HeadRows hr, long long row, int C, int t, int tpr, int k,
                                            const float (&f)[8]) {
  typedef typename Elem<IO>::T T;
  T* p = (T*)base + row * hr.sr;
  if constexpr (ALIGNED) {
    const int c = column<true>(t, tpr, k, 0);
    if (c < C) {
      const int h = (int)((unsigned)c / (unsigned)hr.D);
      store8<IO>(p + h * hr.sh + (c - h * hr.D), f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(t, tpr, k, j);
      const int h = (int)((unsigned)c / (unsigned)hr.D);
      if (c < C) p[h * hr.sh + (c - h * hr.D)] = narrow<IO>(f[j]);
    }
  }
}

// Sum over the threads of a row: one wave, or all waves of the workgroup through `part` (one float per
// wave). Every thread gets the same bits: the waves' sums are added in wave order.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <bool MULTI>
__device__ __forceinline__ float row_sum(float v, float* part, int nw) {
  v = wave_sum(v);
  if constexpr (!MULTI) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < nw; ++w) s += part[w];
  return s;
}

// ---------------------------------------------------------------------------------
// Forward. MULTI: a row per workgroup of blockDim.x threads; else a row per wave. VPT vectors of 8 columns
// per thread. Every load of a row is requested before the first sum needs one.
// ---------------------------------------------------------------------------------
template <int IO, int RIO, int VPT, bool ALIGNED, bool MULTI>
__global__ void __launch_bounds__(MULTI ? 1024 : 256) join_fwd_kernel(JoinArgs a) {
  __shared__ float part[2][16];
  const int tpr = MULTI ? (int)blockDim.x : 64, t = MULTI ? (int)threadIdx.x : (int)(threadIdx.x & 63);
  const int nw = blockDim.x >> 6, C = (int)a.C;
  const long long row = a.row0 + (MULTI ? (long long)blockIdx.x : (long long)blockIdx.x * nw + (threadIdx.x >> 6));
  if (row >= a.B) return;  // (a whole wave; MULTI workgroups never)
  const HeadRows ho{a.o_sh, a.o_sr, (int)a.D}, hy{a.y_sh, a.y_sr, (int)a.D};
  const float rc = 1.0f / (float)C;
  Vec<RIO> r[VPT];
  Vec<IO> o[VPT], wq[VPT], gq[VPT], wp[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (a.o) o[k] = load_heads<IO, ALIGNED>(a.o, ho, row, C, t, tpr, k);
    r[k] = load_row<RIO, ALIGNED>(a.r, row * a.r_sr, C, t, tpr, k);
  }
  const long long grow = a.gate ? row / a.rows_per_gate * a.C : 0;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (a.w_post) wq[k] = load_row<IO, ALIGNED>(a.w_post, 0, C, t, tpr, k);
    if (a.gate) gq[k] = load_row<IO, ALIGNED>(a.gate, grow, C, t, tpr, k);
    if (a.w_pre) wp[k] = load_row<IO, ALIGNED>(a.w_pre, 0, C, t, tpr, k);
  }
  float f[VPT][8];
  float ro = 1.f;
  if (a.o && a.post) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = __builtin_fmaf(o[k].get(j), o[k].get(j), s);
    ro = 1.0f / sqrtf(__builtin_fmaf(row_sum<MULTI>(s, part[0], nw), rc, a.eps));
    if (a.rs_o && t == 0) a.rs_o[row] = ro;
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = r[k].get(j);
      if (a.o) {
        float p = o[k].get(j) * ro;
        if (a.w_post) p *= wq[k].get(j);
        if (a.gate) p *= gq[k].get(j);
        v = __builtin_fmaf(a.scale, p, v);
      }
      f[k][j] = v;
      s = __builtin_fmaf(v, v, s);
    }
    if (a.r_out) store_row<RIO, ALIGNED>(a.r_out, row * a.C, C, t, tpr, k, f[k]);
  }
  if (!a.y) return;
  const float rr = 1.0f / sqrtf(__builtin_fmaf(row_sum<MULTI>(s, part[1], nw), rc, a.eps));
  if (a.rs_r && t == 0) a.rs_r[row] = rr;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[k][j] = f[k][j] * rr * (a.w_pre ? wp[k].get(j) : 1.0f);
    store_heads<IO, ALIGNED>(a.y, hy, row, C, t, tpr, k, f[k]);
  }
}

// ---------------------------------------------------------------------------------
// Backward. A worker (a workgroup when MULTI, else a wave) walks the rows [r0, r1) of its unit, keeping its
// columns' sums of dw_pre, dw_post and dgate in registers, and stores them as its row of the partial arrays;
// join_reduce_kernel adds the workgroups' rows in order (a workgroup's four waves are added first). Units never cross a gate group unless they hold
// whole groups, whose dgate rows are then stored as they end.
// ---------------------------------------------------------------------------------
// MULTI = 2: more than 512 threads. A 16-bit stream's rows of up to 512 threads run two workgroups a CU, within 128
// registers; an fp32 stream's data do not fit those, and one workgroup requests the next row's data ahead instead
// (16384 x 4096, sums' launch included, from the rounded r': bf16 177 us, with the next row ahead 189 at two workgroups and 194 at one;
// fp32 stream, 4096 x 2048: 42 us, 53 the first way).
__host__ __device__ constexpr bool join_ahead(int RIO, int VPT, int MULTI) { return RIO == IO_F32 && VPT == 1 && MULTI == 1; }
template <int IO, int RIO, int VPT, bool ALIGNED, int MULTI>
__global__ void __launch_bounds__(MULTI == 2 ? 1024 : MULTI ? 512 : 256, MULTI == 1 && !join_ahead(RIO, VPT, MULTI) ? 4 : 1)
join_bwd_kernel(JoinArgs a, JoinPlan p) {
  constexpr bool AHEAD = join_ahead(RIO, VPT, MULTI);
  __shared__ float part[2][2][16];
  const int tpr = MULTI ? (int)blockDim.x : 64, t = MULTI ? (int)threadIdx.x : (int)(threadIdx.x & 63);
  const int nw = blockDim.x >> 6, C = (int)a.C;
  const long long unit = MULTI ? (long long)blockIdx.x : (long long)blockIdx.x * nw + (threadIdx.x >> 6);
  const HeadRows ho{a.o_sh, a.o_sr, (int)a.D}, hy{a.y_sh, a.y_sr, (int)a.D}, hd{a.do_sh, a.do_sr, (int)a.D};
  const float rc = 1.0f / (float)C;
  // the unit's rows: part `unit % parts` of a group, or `groups_per_unit` whole groups
  long long r0, r1;
  const long long T = a.rows_per_gate;
  if (p.parts > 1) {
    const long long g = unit / p.parts, q = unit % p.parts;
    r0 = g * T + min(T, q * p.rows_per_part);
    r1 = min(g * T + T, r0 + p.rows_per_part);
  } else {
    r0 = min(a.B, unit * p.groups_per_unit * T);
    r1 = min(a.B, r0 + p.groups_per_unit * T);
  }
  Vec<IO> wq[VPT], gq[VPT], wp[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (a.w_post) wq[k] = load_row<IO, ALIGNED>(a.w_post, 0, C, t, tpr, k);
    if (a.w_pre) wp[k] = load_row<IO, ALIGNED>(a.w_pre, 0, C, t, tpr, k);
  }
  float s_pre[VPT][8], s_post[VPT][8], s_gate[VPT][8];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) s_pre[k][j] = s_post[k][j] = s_gate[k][j] = 0.f;
  long long in_group = 0;  // rows of the current group done by this unit
  // a row's data, where they fit requested while the row before it is worked on
  struct Row {
    Vec<RIO> r2[VPT], dr[VPT];
    Vec<IO> dy[VPT], o[VPT];
    float rr, ro;
  };
  auto load = [&](long long row, Row& x) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (a.dy) {
        x.dy[k] = load_heads<IO, ALIGNED>(a.dy, hy, row, C, t, tpr, k);
        x.r2[k] = load_row<RIO, ALIGNED>(RIO != IO_F32 && a.r ? a.r : a.r_out, row * a.r_sr, C, t, tpr, k);
      }
      if (a.dr_out) x.dr[k] = load_row<RIO, ALIGNED>(a.dr_out, row * a.dr_sr, C, t, tpr, k);
      if (a.o) x.o[k] = load_heads<IO, ALIGNED>(a.o, ho, row, C, t, tpr, k);
    }
    if (a.dy) x.rr = a.rs_r[row];
    x.ro = a.o && a.post ? a.rs_o[row] : 1.f;
  };
  Row next;
  if (AHEAD && r0 < r1) load(r0, next);
  for (long long row = r0; row < r1; ++row) {
    const int db = (int)(row & 1);  // the row sums' buffers alternate: one barrier a sum
    if (!AHEAD) load(row, next);
    Row x = next;
    const auto &r2 = x.r2, &dr = x.dr;
    if constexpr (RIO != IO_F32)  // (the weights stay packed)
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (a.w_post) forget(wq[k]);
        if (a.w_pre) forget(wp[k]);
      }
    const auto &dy = x.dy, &o = x.o;
    if (AHEAD && row + 1 < r1) load(row + 1, next);
    if (a.gate && in_group == 0) {
      const long long grow = row / T * a.C;
#pragma unroll
      for (int k = 0; k < VPT; ++k) gq[k] = load_row<IO, ALIGNED>(a.gate, grow, C, t, tpr, k);
    }
    float d[VPT][8];  // the stream's gradient
    if (a.dy) {
      const float rr = x.rr;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = r2[k].get(j);
        if constexpr (RIO != IO_F32) {
          // A 16-bit stream's unrounded r' is made again where r is given: dw_pre's error is then its own rounding (with
          // the rounded r' 1.4 times that; 16384 x 4096 bf16: step 297 -> 306 us). Below, beside the row's mean, the
          // rounded one is enough, in half the registers; what is unpacked here is not kept across the sum
          // (kept, 8 more registers spill: 333 us).
          if (a.r) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float q = o[k].get(j) * x.ro;
              if (a.w_post) q *= wq[k].get(j);
              if (a.gate) q *= gq[k].get(j);
              v[j] = __builtin_fmaf(a.scale, q, v[j]);
            }
            x.r2[k].put(v);
            forget(x.o[k]);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float m = v[j] * rr, g = dy[k].get(j);
          const float dm = a.w_pre ? g * wp[k].get(j) : g;
          s_pre[k][j] = __builtin_fmaf(g, m, s_pre[k][j]);
          s = __builtin_fmaf(dm, m, s);
          d[k][j] = dm;
        }
      }
      const float mean = row_sum<(MULTI > 0)>(s, part[db][0], nw) * rc;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float m = r2[k].get(j) * rr;
          d[k][j] = __builtin_fmaf(rr, d[k][j] - m * mean, a.dr_out ? dr[k].get(j) : 0.f);
        }
    } else {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) d[k][j] = a.dr_out ? dr[k].get(j) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (a.dr) store_row<RIO, ALIGNED>(a.dr, row * a.C, C, t, tpr, k, d[k]);
    if (a.o) {
      const float ro = x.ro;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float n = o[k].get(j) * ro, w = a.w_post ? wq[k].get(j) : 1.f, sd = a.scale * d[k][j];
          s_gate[k][j] = __builtin_fmaf(sd, n * w, s_gate[k][j]);
          const float dp = a.gate ? sd * gq[k].get(j) : sd;
          s_post[k][j] = __builtin_fmaf(dp, n, s_post[k][j]);
          const float dn = dp * w;
          s = __builtin_fmaf(dn, n, s);
          d[k][j] = dn;
        }
      if (a.d_o) {
        if (a.post) {
          const float mean = row_sum<(MULTI > 0)>(s, part[db][1], nw) * rc;
#pragma unroll
          for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) d[k][j] = ro * (d[k][j] - o[k].get(j) * ro * mean);
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) store_heads<IO, ALIGNED>(a.d_o, hd, row, C, t, tpr, k, d[k]);
      }
      if (p.parts == 1 && a.dgate && ++in_group == T) {  // the group ends here: its sums are whole
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          store_row<IO, ALIGNED>(a.dgate, row / T * a.C, C, t, tpr, k, s_gate[k]);
#pragma unroll
          for (int j = 0; j < 8; ++j) s_gate[k][j] = 0.f;
        }
        in_group = 0;
      } else if (p.parts > 1) {
        in_group = 1;
      }
    }
  }
  if constexpr (MULTI == 0) {  // the four waves' sums in wave order, through LDS
    __shared__ float sum[3][VPT * 8 * 64];
    const int w = threadIdx.x >> 6;
    const auto fold = [&](float (&v)[VPT][8]) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (w > 0) sum[w - 1][(k * 8 + j) * 64 + t] = v[k][j];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] += sum[i][(k * 8 + j) * 64 + t];
    };
    if (p.pre) fold(s_pre);
    if (p.post) fold(s_post);
    if (p.gate) fold(s_gate);
    if (w > 0) return;
  }
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const long long at = (long long)blockIdx.x * a.C;
    if (p.pre) store_row<IO_F32, ALIGNED>(p.pre, at, C, t, tpr, k, s_pre[k]);
    if (p.post) store_row<IO_F32, ALIGNED>(p.post, at, C, t, tpr, k, s_post[k]);
    if (p.gate) store_row<IO_F32, ALIGNED>(p.gate, at, C, t, tpr, k, s_gate[k]);
  }
}

// Column sums of n rows of partials, group by group (rows [g n, g n + n) give out[g]). A workgroup owns 64
// columns; its 16 waves take every 16th row each, their sums are added in wave order.
template <int IO>
__global__ void __launch_bounds__(1024) join_reduce_kernel(JoinReduce q, int C, int col_blocks) {
  __shared__ float part[16][64];
  int b = blockIdx.x, what = 0;
  while (b >= q.t[what].groups * col_blocks) b -= q.t[what++].groups * col_blocks;
  const JoinSum u = q.t[what];
  const int g = b / col_blocks, c = (b % col_blocks) * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const float* src = u.src + (size_t)g * u.rows * C + c;
  float s = 0.f;
  if (c < C) {
    int i = w;
    for (; i + 7 * 16 < u.rows; i += 8 * 16) {  // eight rows requested at once: 26 -> 9 us at 512 rows of 3 x 4096
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = src[(size_t)(i + 16 * j) * C];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < u.rows; i += 16) s += src[(size_t)i * C];
  }
  part[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w != 0 || c >= C) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += part[i][threadIdx.x];
  ((typename Elem<IO>::T*)u.dst)[(size_t)g * C + c] = narrow<IO>(v);
}

// Threads of a row and vectors of 8 columns per thread.
struct RowShape {
  int vpt;
  bool multi;
  int threads;
};

template <typename F>
hipError_t by_shape(int vpt, F f) {
  return vpt == 1 ? f(std::integral_constant<int, 1>{}) : f(std::integral_constant<int, 2>{});
}

// One wave a row up to 1024 columns, beyond a workgroup of as many threads as the row has vectors (two a thread past
// 8192 columns).
RowShape row_shape(int64_t C) {
  const int vecs = (int)((C + 7) / 8);
  if (vecs <= 128) return {vecs <= 64 ? 1 : 2, false, 256};
  const int vpt = vecs <= 1024 ? 1 : 2;
  return {vpt, true, (vecs + vpt * 64 - 1) / (vpt * 64) * 64};
}

// Rows beyond kLaunchThreads' (2^25 rows of up to 1024 columns) take another launch.
template <int IO, int RIO>
hipError_t fwd_launch(const JoinArgs& a, const RowShape& s, long long grid, hipStream_t st) {
  return by_shape(s.vpt, [&](auto V) {
    constexpr int VPT = decltype(V)::value;
    const dim3 g((unsigned)grid), b((unsigned)s.threads);
    if (a.aligned) {
      if (s.multi) hipLaunchKernelGGL((join_fwd_kernel<IO, RIO, VPT, true, true>), g, b, 0, st, a);
      else hipLaunchKernelGGL((join_fwd_kernel<IO, RIO, VPT, true, false>), g, b, 0, st, a);
    } else {
      if (s.multi) hipLaunchKernelGGL((join_fwd_kernel<IO, RIO, VPT, false, true>), g, b, 0, st, a);
      else hipLaunchKernelGGL((join_fwd_kernel<IO, RIO, VPT, false, false>), g, b, 0, st, a);
    }
    return hipGetLastError();
  });
}

template <int IO, int RIO>
hipError_t fwd_t(JoinArgs a, hipStream_t st) {
  const RowShape s = row_shape(a.C);
  const int per = s.multi ? 1 : 4;  // rows of a workgroup
  const long long most = kLaunchThreads / s.threads;
  for (a.row0 = 0; a.row0 < a.B; a.row0 += most * per) {
    const long long left = (a.B - a.row0 + per - 1) / per;
    const hipError_t e = fwd_launch<IO, RIO>(a, s, std::min(left, most), st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int IO, int RIO>
hipError_t bwd_t(const JoinArgs& a, const JoinPlan& p, hipStream_t st) {
  const RowShape s = row_shape(a.C);
  const long long grid = s.multi ? p.units : (p.units + 3) / 4;
  if (grid > 0) {
    const hipError_t e = by_shape(s.vpt, [&](auto V) {
      constexpr int VPT = decltype(V)::value;
      const dim3 g((unsigned)grid), b((unsigned)s.threads);
      const auto run = [&](auto A) {
        constexpr bool AL = decltype(A)::value;
        if (!s.multi) hipLaunchKernelGGL((join_bwd_kernel<IO, RIO, VPT, AL, 0>), g, b, 0, st, a, p);
        else if (VPT == 1 && s.threads <= 512) hipLaunchKernelGGL((join_bwd_kernel<IO, RIO, 1, AL, 1>), g, b, 0, st, a, p);
        else hipLaunchKernelGGL((join_bwd_kernel<IO, RIO, VPT, AL, 2>), g, b, 0, st, a, p);
      };
      if (a.aligned) run(std::true_type{});
      else run(std::false_type{});
      return hipGetLastError();
    });
    if (e != hipSuccess) return e;
  }
  JoinReduce q{};
  int n = 0;
  long long groups = 0;
  const auto add = [&](const float* src, void* dst, long long rows, long long g) {
    if (dst == nullptr) return;
    q.t[n++] = JoinSum{src, dst, (int)rows, (int)g};
    groups += g;
  };
  const int per = s.multi ? 1 : 4;  // units of a workgroup
  add(p.pre, a.dw_pre, grid, 1);
  add(p.post, a.dw_post, grid, 1);
  if (p.gate) add(p.gate, a.dgate, p.parts / per, a.groups);
  else if (a.B == 0) add(nullptr, a.dgate, 0, a.groups);  // (sums of no rows)
  if (n == 0) return hipSuccess;
  const int col_blocks = (int)((a.C + 63) / 64);
  hipLaunchKernelGGL(join_reduce_kernel<IO>, dim3((unsigned)(groups * col_blocks)), dim3(1024), 0, st, q, (int)a.C,
                     col_blocks);
  return hipGetLastError();
}

}  // namespace

JoinPlan join_plan(int64_t B, int64_t C, int64_t groups, bool dpre, bool dpost, bool dgate, int num_cus) {
  JoinPlan p{};
  const long long T = groups > 0 ? B / groups : 0;
  const RowShape s = row_shape(C);
  // workers that fill the device twice over: two workgroups a CU, or eight waves
  const long long want = (long long)num_cus * (s.multi ? 2 : 8);
  const long long rows = std::max<long long>(1, (B + want - 1) / want);
  p.parts = 1;
  p.groups_per_unit = 1;
  if (T > 0 && rows < T) {
    p.parts = (int)((T + rows - 1) / rows);
    p.rows_per_part = (T + p.parts - 1) / p.parts;
    p.parts = (int)((T + p.rows_per_part - 1) / p.rows_per_part);
    if (!s.multi) p.parts = (p.parts + 3) / 4 * 4;  // a workgroup's four units in one group (the last ones may be empty)
    p.units = groups * p.parts;
  } else if (T > 0) {
    p.groups_per_unit = rows / T;
    p.units = (groups + p.groups_per_unit - 1) / p.groups_per_unit;
  }
  size_t at = 0;
  const size_t one = (size_t)(s.multi ? p.units : (p.units + 3) / 4) * C * sizeof(float);
  const auto take = [&](bool on) {
    const size_t off = at;
    if (on) at += (one + 255) / 256 * 256;
    return off;
  };
  p.off_pre = take(dpre);
  p.off_post = take(dpost);
  p.gate_partials = dgate && p.parts > 1;
  p.off_gate = take(p.gate_partials);
  p.ws_bytes = at;
  return p;
}

hipError_t launch_join_fwd(const JoinArgs& a, hipStream_t st) {
  if (a.B <= 0) return hipSuccess;
  if (a.io == IO_F32) return fwd_t<IO_F32, IO_F32>(a, st);
  if (a.io == IO_BF16) return a.r_f32 ? fwd_t<IO_BF16, IO_F32>(a, st) : fwd_t<IO_BF16, IO_BF16>(a, st);
  return a.r_f32 ? fwd_t<IO_F16, IO_F32>(a, st) : fwd_t<IO_F16, IO_F16>(a, st);
}

hipError_t launch_join_bwd(const JoinArgs& a, JoinPlan p, void* ws, hipStream_t st) {
  p.pre = a.dw_pre ? (float*)((char*)ws + p.off_pre) : nullptr;
  p.post = a.dw_post ? (float*)((char*)ws + p.off_post) : nullptr;
  p.gate = p.gate_partials ? (float*)((char*)ws + p.off_gate) : nullptr;
  if (a.io == IO_F32) return bwd_t<IO_F32, IO_F32>(a, p, st);
  if (a.io == IO_BF16) return a.r_f32 ? bwd_t<IO_BF16, IO_F32>(a, p, st) : bwd_t<IO_BF16, IO_BF16>(a, p, st);
  return a.r_f32 ? bwd_t<IO_F16, IO_F32>(a, p, st) : bwd_t<IO_F16, IO_F16>(a, p, st);
}

}  // namespace fmlp

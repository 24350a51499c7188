// Layer norm over the last dimension, forward and backward (sm_100a).
//
//   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xhat * w + b
//   dx = rstd * (gw - mean(gw) - xhat * mean(gw * xhat)),  gw = g * w
//   dw = sum over rows of g * xhat,  db = sum over rows of g
//
// Both passes are bound by HBM: x (and g) are read once, y (or dx) written once.  A row lives in the
// registers of the threads that share it (a part of a warp, a warp, or a block for wide rows), so the
// variance is the two-pass one, over differences from the mean.  The backward pass keeps each
// thread's share of dw and db in registers over all the rows that it sees; a block adds its groups
// in a fixed order and writes one partial row, and a second kernel adds the blocks' rows in theirs, so
// the gradients do not depend on timing.  All sums are fp32; the values are rounded once, on output.
// Rows wider than the register paths hold take loops that read the row once per pass.
//
// Measured on one B200: forward 819,200 x 256 fp16 127 us (6.6 TB/s, a plain copy's rate); backward
// 204,800 x 256 bf16 71 us (4.4 TB/s), its sums' second kernel 4; 5,003 x 771 fp32 9 and 10 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "rbq_internal.cuh"

namespace rbq {
namespace {

constexpr int kNormThreads = 256;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Vec {
  T e[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC])
{
  const Vec<T, VEC> x = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = to_f(x.e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Vec<T, VEC>& x, float (&v)[VEC])
{
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = to_f(x.e[i]);
}
// A thread's own ring of row pieces in shared memory, filled by asynchronous 16-byte copies.  A thread
// reads only what it copied itself, so waiting for its copies is all the order that is needed; rows
// outside the matrix are filled with zeros.  The bytes on their way cost no registers.
template <typename T, int VEC, int CH, int TPR, int DEPTH>
struct RowRing {
  uint4 (*slot)[kNormThreads];  // [DEPTH * CH]
  const T* p;
  int64_t rows;
  int d, i;
  __device__ __forceinline__ void ask(int64_t r, int stage) const
  {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * TPR + i) * VEC;
      const bool in = r < rows && col < d;
      const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&slot[stage * CH + c][threadIdx.x]);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? p + r * d + col : p), "r"(in ? 16 : 0)
                   : "memory");
    }
  }
  __device__ __forceinline__ void take(int stage, float (&v)[CH][VEC]) const
  {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const uint4 raw = slot[stage * CH + c][threadIdx.x];
      unpack<T, VEC>(*reinterpret_cast<const Vec<T, VEC>*>(&raw), v[c]);
    }
  }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void ring_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Keeps x packed: the compiler would unpack loop-invariant values once and hold twice the registers.
template <typename T, int VEC>
__device__ __forceinline__ void keep_packed(Vec<T, VEC>& x)
{
  static_assert(sizeof(Vec<T, VEC>) % 4 == 0 || VEC == 1, "whole registers");
  if (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) asm volatile("" : "+r"(reinterpret_cast<uint32_t*>(&x)[k]));
  }
}
// A thread's pieces of row r of a [rows, d] matrix, as they lie in memory; zeros outside.
template <typename T, int VEC, int CH, int TPR>
__device__ __forceinline__ void fetch(const T* p, int64_t r, int64_t rows, int d, int i, Vec<T, VEC> (&x)[CH])
{
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * TPR + i) * VEC;
    if (r < rows && col < d)
      x[c] = *reinterpret_cast<const Vec<T, VEC>*>(p + r * d + col);
    else
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[c].e[e] = from_f<T>(0.0f);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC])
{
  Vec<T, VEC> x;
#pragma unroll
  for (int i = 0; i < VEC; ++i) x.e[i] = from_f<T>(v[i]);
  *reinterpret_cast<Vec<T, VEC>*>(p) = x;
}

// Sum over the TPR threads that share a row (TPR = kNormThreads: the block).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s_red)
{
  if (TPR <= 32) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // the last sum has been read
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; ++w) t += s_red[w];
  return t;
}

// sum / d, rounded as a division would: the product with the rounded 1 / d, corrected once by its residual
// (Markstein's method).  An infinite sum has no residual (infinity - infinity) and stays as it is.
__device__ __forceinline__ float over(float sum, float d, float inv_d)
{
  const float q = sum * inv_d, rest = fmaf(-q, d, sum);
  return rest == rest ? fmaf(rest, inv_d, q) : q;
}

// TPR threads to a row; thread i of a row holds CH pieces of VEC values, piece c at column
// (c * TPR + i) * VEC.  Few threads with several pieces each need fewer shuffles and scalar steps per row
// than a warp with one piece each.
template <typename T, typename P, int VEC, int CH, int TPR>
__global__ void __launch_bounds__(kNormThreads)
    norm_kernel(const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int d, float eps)
{
  __shared__ float s_red[kNormThreads / 32];
  constexpr int kRows = kNormThreads / TPR;
  // The thread's parameters stay in registers, as they lie in memory.  (From shared memory they took
  // most of the load-store unit's cycles, and as fp32 registers half the warps.)
  constexpr bool kHold = CH * VEC <= 16;
  const int i = threadIdx.x % TPR;
  const float fd = (float)d, inv_d = 1.0f / fd;
  const int64_t step = (int64_t)gridDim.x * kRows;
  // Rows on their way while one is worked on: kDepth - 1 in the ring, one in registers where the pieces are not
  // of 16 bytes or too many.
  constexpr bool kRing = VEC * sizeof(T) == 16 && CH <= 2;
  constexpr int kDepth = 4;
  __shared__ uint4 s_ring[kRing ? kDepth * CH : 1][kRing ? kNormThreads : 1];
  const RowRing<T, VEC, CH, TPR, kDepth> ring{reinterpret_cast<uint4(*)[kNormThreads]>(s_ring), x, rows, d, i};
  const int64_t mine = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  int stage = 0;
  Vec<T, VEC> next[CH];
  if (kRing) {
#pragma unroll
    for (int k = 0; k < kDepth - 1; ++k) {
      ring.ask(mine + k * step, k);
      ring_commit();
    }
  } else {
    fetch<T, VEC, CH, TPR>(x, mine, rows, d, i, next);
  }
  Vec<P, VEC> wv[CH], bv[CH];
  if (kHold) {
    fetch<P, VEC, CH, TPR>(w, 0, 1, d, i, wv);
    fetch<P, VEC, CH, TPR>(b, 0, 1, d, i, bv);
  }
  // whole warps run every round, so that the shuffles see all lanes
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += step) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool live = r < rows;
    float v[CH][VEC];
    float sum = 0.0f;
    if (kRing) {
      ring.ask(r + (kDepth - 1) * step, (stage + kDepth - 1) % kDepth);
      ring_commit();
      ring_wait<kDepth - 1>();
      ring.take(stage, v);
      stage = (stage + 1) % kDepth;
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) unpack<T, VEC>(next[c], v[c]);
      fetch<T, VEC, CH, TPR>(x, r + step, rows, d, i, next);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += v[c][e];
    const float mean = over(row_sum<TPR>(sum, s_red), fd, inv_d);
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if ((c * TPR + i) * VEC < d) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[c][e] -= mean;
          sq = fmaf(v[c][e], v[c][e], sq);
        }
      }
    }
    const float rstd = rsqrtf(over(row_sum<TPR>(sq, s_red), fd, inv_d) + eps);
    if (live) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + i) * VEC;
        if (col < d) {
          float wc[VEC], bc[VEC];
          if (kHold) {
            keep_packed(wv[c]);
            keep_packed(bv[c]);
            unpack<P, VEC>(wv[c], wc);
            unpack<P, VEC>(bv[c], bc);
          } else {
            load_vec<P, VEC>(w + col, wc);
            load_vec<P, VEC>(b + col, bc);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[c][e] = fmaf(v[c][e] * rstd, wc[e], bc[e]);
          store_vec<T, VEC>(y + r * d + col, v[c]);
        }
      }
      if (i == 0) {
        mean_out[r] = mean;
        rstd_out[r] = rstd;
      }
    }
  }
  if (kRing) ring_wait<0>();
}

// part[block][2][d]: this block's share of dw and db.  Rows on their way lie in shared memory: in
// registers they cost a quarter of the warps (204,800 rows of 256: 71 us, 77 that way, 73 with none ahead).
template <typename T, typename P, int VEC, int CH, int TPR>
__global__ void __launch_bounds__(kNormThreads, CH * VEC <= 8 ? 4 : 1)
    norm_grad_kernel(const T* __restrict__ g, const T* __restrict__ x, const P* __restrict__ w,
                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                     float* __restrict__ part, int64_t rows, int d)
{
  extern __shared__ float s_part[];  // [2][d], rows shared by TPR < kNormThreads threads only
  __shared__ float s_red[kNormThreads / 32];
  constexpr int kRows = kNormThreads / TPR;
  constexpr bool kHold = CH * VEC <= 16;
  const int i = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float fd = (float)d, inv_d = 1.0f / fd;
  const int64_t step = (int64_t)gridDim.x * kRows;
  float dw[CH][VEC], db[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[c][e] = db[c][e] = 0.0f;
  Vec<P, VEC> wv[CH];
  if (kHold) fetch<P, VEC, CH, TPR>(w, 0, 1, d, i, wv);
  constexpr bool kRing = VEC * sizeof(T) == 16 && CH <= 2;
  constexpr int kDepth = 4 / (CH <= 2 ? CH : 2);
  __shared__ uint4 s_ring[kRing ? 2 * kDepth * CH : 1][kRing ? kNormThreads : 1];
  uint4(*ring_slots)[kNormThreads] = reinterpret_cast<uint4(*)[kNormThreads]>(s_ring);
  const RowRing<T, VEC, CH, TPR, kDepth> ring_x{ring_slots, x, rows, d, i}, ring_g{ring_slots + kDepth * CH, g, rows, d, i};
  const int64_t mine = (int64_t)blockIdx.x * kRows + group;
  int stage = 0;
  float next_mean = 0.0f, next_rstd = 0.0f;
  if (kRing) {
#pragma unroll
    for (int k = 0; k < kDepth - 1; ++k) {
      ring_x.ask(mine + k * step, k);
      ring_g.ask(mine + k * step, k);
      ring_commit();
    }
    if (mine < rows) next_mean = __ldg(mean_in + mine), next_rstd = __ldg(rstd_in + mine);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += step) {
    const int64_t r = r0 + group;
    const bool live = r < rows;
    float mean, rstd, xh[CH][VEC], gw[CH][VEC];
    float a = 0.0f, b = 0.0f;
    if (kRing) {
      ring_x.ask(r + (kDepth - 1) * step, (stage + kDepth - 1) % kDepth);
      ring_g.ask(r + (kDepth - 1) * step, (stage + kDepth - 1) % kDepth);
      ring_commit();
      mean = next_mean, rstd = next_rstd;
      if (r + step < rows) next_mean = __ldg(mean_in + r + step), next_rstd = __ldg(rstd_in + r + step);
      ring_wait<kDepth - 1>();
      ring_x.take(stage, xh);
      ring_g.take(stage, gw);
      stage = (stage + 1) % kDepth;
    } else {
      mean = live ? __ldg(mean_in + r) : 0.0f, rstd = live ? __ldg(rstd_in + r) : 0.0f;
      Vec<T, VEC> xr[CH], gr[CH];
      fetch<T, VEC, CH, TPR>(x, r, rows, d, i, xr);
      fetch<T, VEC, CH, TPR>(g, r, rows, d, i, gr);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        unpack<T, VEC>(xr[c], xh[c]);
        unpack<T, VEC>(gr[c], gw[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * TPR + i) * VEC;
      if (live && col < d) {
        float wc[VEC];
        if (kHold) {
          keep_packed(wv[c]);
          unpack<P, VEC>(wv[c], wc);
        } else {
          load_vec<P, VEC>(w + col, wc);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          xh[c][e] = (xh[c][e] - mean) * rstd;
          dw[c][e] = fmaf(gw[c][e], xh[c][e], dw[c][e]);
          db[c][e] += gw[c][e];
          gw[c][e] *= wc[e];
          a += gw[c][e];
          b = fmaf(gw[c][e], xh[c][e], b);
        }
      }
    }
    if (dx == nullptr) continue;
    a = over(row_sum<TPR>(a, s_red), fd, inv_d);
    b = over(row_sum<TPR>(b, s_red), fd, inv_d);
    if (live) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + i) * VEC;
        if (col < d) {
          float o[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = rstd * (gw[c][e] - a - xh[c][e] * b);
          store_vec<T, VEC>(dx + r * d + col, o);
        }
      }
    }
  }
  if (kRing) ring_wait<0>();
  if (part == nullptr) return;
  float* out = part + (int64_t)blockIdx.x * 2 * d;
  if (TPR < 32) {  // the warp's rows
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
#pragma unroll
        for (int o = TPR; o < 32; o <<= 1) {
          dw[c][e] += __shfl_xor_sync(0xffffffffu, dw[c][e], o);
          db[c][e] += __shfl_xor_sync(0xffffffffu, db[c][e], o);
        }
      }
  }
  if (TPR == kNormThreads) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * TPR + i) * VEC;
      if (col < d) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          out[col + e] = dw[c][e];
          out[d + col + e] = db[c][e];
        }
      }
    }
    return;
  }
  for (int k = 0; k < kNormThreads / 32; ++k) {  // the warps in their order
    if ((int)(threadIdx.x >> 5) == k && (threadIdx.x & 31) < TPR) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + i) * VEC;
        if (col < d) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            s_part[col + e] = (k ? s_part[col + e] : 0.0f) + dw[c][e];
            s_part[d + col + e] = (k ? s_part[d + col + e] : 0.0f) + db[c][e];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int j = threadIdx.x; j < 2 * d; j += kNormThreads) out[j] = s_part[j];
}

// Rows wider than the register paths: a block per row, the row read once per pass.
template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
    norm_wide_kernel(const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                     float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int d, float eps)
{
  __shared__ float s_red[kNormThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * d;
    float sum = 0.0f, sq = 0.0f;
    for (int j = threadIdx.x; j < d; j += kNormThreads) sum += to_f(xr[j]);
    const float mean = row_sum<kNormThreads>(sum, s_red) / (float)d;
    for (int j = threadIdx.x; j < d; j += kNormThreads) {
      const float c = to_f(xr[j]) - mean;
      sq = fmaf(c, c, sq);
    }
    const float rstd = rsqrtf(row_sum<kNormThreads>(sq, s_red) / (float)d + eps);
    for (int j = threadIdx.x; j < d; j += kNormThreads)
      y[r * d + j] = from_f<T>(fmaf((to_f(xr[j]) - mean) * rstd, to_f(w[j]), to_f(b[j])));
    if (threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}
template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
    norm_wide_grad_kernel(const T* __restrict__ g, const T* __restrict__ x, const P* __restrict__ w,
                          const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                          int64_t rows, int d)
{
  __shared__ float s_red[kNormThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * d, *gr = g + r * d;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float a = 0.0f, b = 0.0f;
    for (int j = threadIdx.x; j < d; j += kNormThreads) {
      const float gw = to_f(gr[j]) * to_f(w[j]);
      a += gw;
      b = fmaf(gw, (to_f(xr[j]) - mean) * rstd, b);
    }
    a = row_sum<kNormThreads>(a, s_red) / (float)d;
    b = row_sum<kNormThreads>(b, s_red) / (float)d;
    for (int j = threadIdx.x; j < d; j += kNormThreads) {
      const float gw = to_f(gr[j]) * to_f(w[j]);
      dx[r * d + j] = from_f<T>(rstd * (gw - a - (to_f(xr[j]) - mean) * rstd * b));
    }
  }
}
// Shares of dw and db of such rows: thread = column, block y = a share of the rows.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
    norm_wide_sums_kernel(const T* __restrict__ g, const T* __restrict__ x, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, float* __restrict__ part, int64_t rows, int d)
{
  const int64_t c = (int64_t)blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= d) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = rows * blockIdx.y / gridDim.y, e = rows * (blockIdx.y + 1) / gridDim.y; r < e; ++r) {
    const float gv = to_f(g[r * d + c]);
    dw = fmaf(gv, (to_f(x[r * d + c]) - __ldg(mean_in + r)) * __ldg(rstd_in + r), dw);
    db += gv;
  }
  part[(int64_t)blockIdx.y * 2 * d + c] = dw;
  part[(int64_t)blockIdx.y * 2 * d + d + c] = db;
}

// dw and db from the blocks' shares: 32 interleaved runs of blocks, then the runs in their order.
template <typename P>
__global__ void __launch_bounds__(1024) norm_parts_kernel(const float* __restrict__ part, int parts, int d, P* __restrict__ dw,
                                                          P* __restrict__ db)
{
  __shared__ float s_sum[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < 2 * (int64_t)d) {
#pragma unroll 4
    for (int p = run; p < parts; p += 32) t += part[(int64_t)p * 2 * d + c];
  }
  s_sum[run][lane] = t;
  __syncthreads();
  if (run == 0 && c < 2 * (int64_t)d) {
#pragma unroll
    for (int k = 1; k < 32; ++k) t += s_sum[k][lane];
    if (c < d) {
      if (dw != nullptr) dw[c] = from_f<P>(t);
    } else if (db != nullptr) {
      db[c - d] = from_f<P>(t);
    }
  }
}

// How a row is shared: vec values per load (16 bytes, or one where the width or an address does not
// allow that), tpr threads per row, ch loads per thread; tpr = 0: wider than the register paths.  For rows that a
// block holds ch is the next size up, so that no thread steps over more than half of its loads (200 M values in
// rows of 1,953 fp32: 644 us with 32 loads, 293 with 8; of 2,048 fp16: 369 with 4, 166 with 1).  Narrower rows of
// single values have one size for widths to 32 and one to 256, and step over more.
struct Plan {
  int vec, tpr, ch;
};
Plan plan_of(int d, int esize, bool vector, bool backward)
{
  const int vec = vector ? 16 / esize : 1;
  const int loads = (d + vec - 1) / vec;
  if (vector) {
    if (loads <= 8) return {vec, 8, 1};
    if (loads <= 16) return {vec, 8, 2};
    // the backward pass holds five values per column: half the pieces, for as many warps on an SM
    if (loads <= 32) return backward ? Plan{vec, 32, 1} : Plan{vec, 16, 2};
    if (loads <= 64) return Plan{vec, 32, 2};
    if (loads <= 128) return {vec, 32, 4};
    if (loads <= kNormThreads) return {vec, kNormThreads, 1};
    if (loads <= 2 * kNormThreads) return {vec, kNormThreads, 2};
    if (loads <= 4 * kNormThreads) return {vec, kNormThreads, 4};
    if (vec == 4 && loads <= 8 * kNormThreads) return {vec, kNormThreads, 8};
  } else {
    if (loads <= 32) return {vec, 8, 4};
    if (loads <= 256) return {vec, 32, 8};
    if (loads <= 4 * kNormThreads) return {vec, kNormThreads, 4};
    if (loads <= 8 * kNormThreads) return {vec, kNormThreads, 8};
    if (loads <= 16 * kNormThreads) return {vec, kNormThreads, 16};
    if (loads <= 32 * kNormThreads) return {vec, kNormThreads, 32};
  }
  return {vec, 0, 0};
}

// Blocks of a kernel that runs over its rows in rounds: those that an SM holds at once (kMostBlocks at
// most), and no more than there are rows for.  With `rounds` there are as many times that many as leave
// each block about so many rounds: SMs get through memory traffic at different rates, and blocks that start
// as others end even that out (forward pass, 819,200 x 256: 159 us in one wave, 127 in 16).  The backward
// pass writes sums for every block and gains nothing (71 us, 72 in two waves).
constexpr int kMostBlocks = 8, kRounds = 6;
template <typename T, typename P, int VEC, int CH, int TPR, int PASS>
struct Kernel;  // names a kernel
template <typename Name, typename K>
int blocks_for(K kernel, size_t smem, int64_t rows, int tpr, int rounds)
{
  // one for every Name and all devices (the library runs on one architecture); smem is that of its widest rows
  static std::atomic<int> per_sm{0};
  int n = per_sm.load();
  if (n == 0) {
    RBQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kNormThreads, smem));
    n = std::max(1, std::min(n, kMostBlocks));
    per_sm.store(n);
  }
  const int64_t work = ceil_div(rows, kNormThreads / tpr), wave = (int64_t)device_sm_count() * n;
  const int64_t waves = rounds > 0 ? std::max<int64_t>(1, std::min<int64_t>(64, work / (wave * rounds))) : 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(work, wave * waves));
}

template <typename T, typename P>
void run_forward(const T* x, const P* w, const P* b, T* y, float* mean, float* rstd, int64_t rows, int d, float eps,
                 bool vector, cudaStream_t s)
{
  const Plan p = plan_of(d, (int)sizeof(T), vector, false);
  constexpr int V = 16 / (int)sizeof(T);
#define RBQ_NORM(VEC, CH, TPR)                                                                                      \
  norm_kernel<T, P, VEC, CH, TPR>                                                                                   \
      <<<blocks_for<Kernel<T, P, VEC, CH, TPR, 0>>(norm_kernel<T, P, VEC, CH, TPR>, 0, rows, TPR, kRounds), kNormThreads, 0, \
         s>>>(x, w, b, y, mean, rstd, rows, d, eps)
  if (p.tpr == 0)
    norm_wide_kernel<T, P><<<(unsigned)std::min<int64_t>(rows, (int64_t)device_sm_count() * kMostBlocks), kNormThreads, 0, s>>>(
        x, w, b, y, mean, rstd, rows, d, eps);
  else if (p.vec == 1 && p.tpr == 8)
    RBQ_NORM(1, 4, 8);
  else if (p.vec == 1 && p.tpr == 32)
    RBQ_NORM(1, 8, 32);
  else if (p.vec == 1)
    p.ch == 4    ? RBQ_NORM(1, 4, kNormThreads)
    : p.ch == 8  ? RBQ_NORM(1, 8, kNormThreads)
    : p.ch == 16 ? RBQ_NORM(1, 16, kNormThreads)
                 : RBQ_NORM(1, 32, kNormThreads);
  else if (p.tpr == 8)
    p.ch == 1 ? RBQ_NORM(V, 1, 8) : RBQ_NORM(V, 2, 8);
  else if (p.tpr == 16)
    RBQ_NORM(V, 2, 16);
  else if (p.tpr == 32)
    p.ch == 2 ? RBQ_NORM(V, 2, 32) : RBQ_NORM(V, 4, 32);
  else
    p.ch == 1   ? RBQ_NORM(V, 1, kNormThreads)
    : p.ch == 2 ? RBQ_NORM(V, 2, kNormThreads)
    : p.ch == 4 ? RBQ_NORM(V, 4, kNormThreads)
                : RBQ_NORM(V, (V == 4 ? 8 : 4), kNormThreads);  // fp32 rows only
#undef RBQ_NORM
  RBQ_LAUNCHED();
}

template <typename T, typename P>
void run_backward(const T* g, const T* x, const P* w, const float* mean, const float* rstd, T* dx, P* dw, P* db, float* part,
                  int64_t rows, int d, bool vector, cudaStream_t s)
{
  const Plan p = plan_of(d, (int)sizeof(T), vector, true);
  constexpr int V = 16 / (int)sizeof(T);
  int blocks = (int)std::min<int64_t>(rows, (int64_t)device_sm_count() * kMostBlocks);  // of the wide kernels
  const bool sums = dw != nullptr || db != nullptr;
  float* out = sums ? part : nullptr;
  const size_t smem = sums && p.tpr && p.tpr < kNormThreads ? (size_t)2 * d * sizeof(float) : 0;
#define RBQ_NORM(VEC, CH, TPR)                                                                                          \
  (blocks = blocks_for<Kernel<T, P, VEC, CH, TPR, 1>>(norm_grad_kernel<T, P, VEC, CH, TPR>,                              \
                                                    TPR < kNormThreads ? 2 * sizeof(float) * CH * TPR * VEC : 0, rows, TPR, 0), \
   norm_grad_kernel<T, P, VEC, CH, TPR><<<blocks, kNormThreads, smem, s>>>(g, x, w, mean, rstd, dx, out, rows, d))
  if (p.tpr == 0) {
    if (dx != nullptr) {
      norm_wide_grad_kernel<T, P><<<blocks, kNormThreads, 0, s>>>(g, x, w, mean, rstd, dx, rows, d);
      RBQ_LAUNCHED();
    }
    if (sums) {
      norm_wide_sums_kernel<T><<<dim3((unsigned)ceil_div(d, kNormThreads), blocks), kNormThreads, 0, s>>>(
          g, x, mean, rstd, part, rows, d);
      RBQ_LAUNCHED();
    }
  } else {
    if (p.vec == 1 && p.tpr == 8)
      RBQ_NORM(1, 4, 8);
    else if (p.vec == 1 && p.tpr == 32)
      RBQ_NORM(1, 8, 32);
    else if (p.vec == 1)
      p.ch == 4    ? RBQ_NORM(1, 4, kNormThreads)
    : p.ch == 8  ? RBQ_NORM(1, 8, kNormThreads)
    : p.ch == 16 ? RBQ_NORM(1, 16, kNormThreads)
                 : RBQ_NORM(1, 32, kNormThreads);
    else if (p.tpr == 8)
      p.ch == 1 ? RBQ_NORM(V, 1, 8) : RBQ_NORM(V, 2, 8);
    else if (p.tpr == 32)
      p.ch == 1 ? RBQ_NORM(V, 1, 32) : p.ch == 2 ? RBQ_NORM(V, 2, 32) : RBQ_NORM(V, 4, 32);
    else
      p.ch == 1   ? RBQ_NORM(V, 1, kNormThreads)
      : p.ch == 2 ? RBQ_NORM(V, 2, kNormThreads)
      : p.ch == 4 ? RBQ_NORM(V, 4, kNormThreads)
                : RBQ_NORM(V, (V == 4 ? 8 : 4), kNormThreads);  // fp32 rows only
    RBQ_LAUNCHED();
  }
#undef RBQ_NORM
  if (sums) {
    norm_parts_kernel<P><<<(unsigned)ceil_div(2 * (int64_t)d, 32), 1024, 0, s>>>(part, blocks, d, dw, db);
    RBQ_LAUNCHED();
  }
}

bool aligned16(std::initializer_list<const void*> ps)
{
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  return true;
}

}  // namespace

// Parameters are of the rows' type or fp32.  16-byte loads need a width of whole loads (of fp32
// parameters too: twice as many bytes) and aligned addresses; else one value at a time.
void launch_layer_norm(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int d,
                       float eps, int dtype, int param_dtype, cudaStream_t s)
{
  const bool vec = d % (dtype == RBQ_F32 ? 4 : 8) == 0 && aligned16({x, w, b, y});
#define RBQ_RUN(T, P) run_forward<T, P>((const T*)x, (const P*)w, (const P*)b, (T*)y, mean, rstd, rows, d, eps, vec, s)
  if (dtype == RBQ_F32)
    RBQ_RUN(float, float);
  else if (dtype == RBQ_F16)
    param_dtype == RBQ_F32 ? RBQ_RUN(__half, float) : RBQ_RUN(__half, __half);
  else
    param_dtype == RBQ_F32 ? RBQ_RUN(__nv_bfloat16, float) : RBQ_RUN(__nv_bfloat16, __nv_bfloat16);
#undef RBQ_RUN
}

int64_t layer_norm_workspace(int64_t rows, int d)
{
  return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)device_sm_count() * kMostBlocks)) * 2 * d * (int64_t)sizeof(float);
}

void launch_layer_norm_backward(const void* g, const void* x, const void* w, const float* mean, const float* rstd, void* dx,
                                void* dw, void* db, float* part, int64_t rows, int d, int dtype, int param_dtype,
                                cudaStream_t s)
{
  const bool vec = d % (dtype == RBQ_F32 ? 4 : 8) == 0 && aligned16({g, x, w, dx});
#define RBQ_RUN(T, P) \
  run_backward<T, P>((const T*)g, (const T*)x, (const P*)w, mean, rstd, (T*)dx, (P*)dw, (P*)db, part, rows, d, vec, s)
  if (dtype == RBQ_F32)
    RBQ_RUN(float, float);
  else if (dtype == RBQ_F16)
    param_dtype == RBQ_F32 ? RBQ_RUN(__half, float) : RBQ_RUN(__half, __half);
  else
    param_dtype == RBQ_F32 ? RBQ_RUN(__nv_bfloat16, float) : RBQ_RUN(__nv_bfloat16, __nv_bfloat16);
#undef RBQ_RUN
}

}  // namespace rbq

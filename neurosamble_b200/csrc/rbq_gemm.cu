// Matrix products on the 5th-generation tensor cores (tcgen05, sm_100a) with the epilogues of the
// read encoder's operators: the linear layer y = act(x w^T + b) + residual and its gradients, and
// the softmax loss of embeddings against a bank, whose logits never leave the SM.
//
//   D[M, N] = sum_k A[m, k] B[n, k]     A, B fp16 or bf16, fp32 accumulators in tensor memory
//
// Either operand may be stored with k contiguous ("K-major": x, w, q, the bank) or with its own
// rows contiguous ("MN-major": the same matrices inside a gradient, where the sum runs over the
// stored rows); the tensor cores read both, so no operand is ever transposed in memory.
//
// CTA, persistent over output tiles: one warp streams 64-wide k-blocks of A and B by TMA into a ring
// of shared-memory stages (128-byte swizzle, zero fill past the edges), one warp issues the MMAs into
// one of two accumulators (2 x BN of the 512 TMEM columns), and BN / 64 warpgroups take 64 columns each
// of the finished one; thread r of a group owns row r (TMEM lane r).  The accumulator is free again
// as soon as its columns are in registers, and the epilogue's arithmetic runs beside the next tiles'
// MMAs, with four warps per scheduler to hide its latencies.
//
// Two shapes.  CG = 2, products with enough tiles for every SM pair: two CTAs of a cluster share a
// 256 x 256 tile (cta_group::2), each holding 128 rows of A and 128 of B per stage, so that a CTA
// takes 64 operand bytes per MMA clock out of L2 where one with a 128 x 256 tile of its own takes 96.  The
// leader CTA issues the MMAs for both.  CG = 1, the smaller ones: a CTA takes a 128 x 128 tile.
//
// Output and input tiles of the epilogue pass through 128-byte swizzled staging rows: by TMA where the
// matrix allows it (rows a multiple of 16 bytes apart), else by coalesced loads and stores of the warp
// that owns the rows.
//
// Measured on one B200 (CUDA time; cuBLAS alone on the same product in brackets, where taken): linear
// 819,200 x 256 -> 1,024 in fp16 0.47 ms without, 0.66 with GELU (0.50; HBM floor 0.32); 819,200 x 1,024
// -> 256 0.41 (0.39); 8,192^3 0.82 (0.70: its tiles are better ordered for L2).  Loss of 8,192 queries
// against 200,000 x 256: forward 0.72 ms (1.17 PFLOP/s), backward 2.4 ms.  In loops of these the card
// runs into its 1,000 W limit at 1.3 to 1.7 GHz.
//
// Long sums with few output tiles (weight gradients) are cut along k instead: every CTA takes an equal
// run of k-blocks through the tiles laid end to end, writes what it has of a tile to an fp32 slab of that
// tile, and a second kernel adds a tile's slabs in their order, so results do not depend on timing.
//
// Every mbarrier wait is bounded: on time-out the kernel records a code in g_op_err, all roles stop
// touching memory, copies in flight are waited for (bounded), TMEM is freed and the kernel returns.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "rbq_internal.cuh"
#include "rbq_tc.cuh"

namespace rbq {
namespace {

constexpr int kBM = 128;       // output rows of a tile (TMEM lanes)
constexpr int kBK = 64;        // reduction values per stage: one 128-byte row of 16-bit values
constexpr int kStageOut = kBM * 128;          // one staging buffer: 128 rows of 128 bytes
constexpr int kSlabCols = 16;                 // a slab's: 128 rows of 64 bytes, which leaves room for one more stage
constexpr int kSlabOut = kBM * kSlabCols * 4;
constexpr uint32_t kOpWaitLimit = 1u << 22;   // polls; each suspends for up to some microseconds
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGradScale = 16384.0f;        // power of two, see GradRows

__device__ int g_op_err;

// Column sums of the gradient kernel's output (the bias's gradient) are taken in fp32, before its rounding to 16
// bits: a sum of many terms of either sign may be small beside them, and their roundings are not.  A row's values lie
// in one thread, so the 32 rows of a warp pass 16 columns at a time through the staging rows that held the extra
// input of these columns (consumed by then): lane l adds columns 2 (l % 8) and the next over rows 8 (l / 8).., in
// registers for as long as the CTA stays in one column of tiles.  Tiles run down the columns for that, so a CTA (or
// pair) visits each column of tiles once at most and writes one row of sums per warp for it:
//   sums[((cta * CG + rank) * 4 + warp) * N + column]
// Rows past the last add zeros: g is 0 there, and the slope finite but in columns whose bias is NaN, of which nothing
// is left anyway.  51,200 x 256 -> 1,024 with GELU: 72 us, 67 with sums of the rounded values; four columns to a lane
// spill (74).  A pass of its own over the output took a third of the kernel.
enum Epilogue {
  kEpiLinear,  // out = act(alpha * acc + bias) + extra
  kEpiActGrad, // out = extra * act'(acc + bias)
  kEpiSlab,    // fp32 slab of a part of k, written or added to
  kEpiLse,     // per row and tile: max and sum of exp of the scaled logits, without the target's
  kEpiProb,    // out = gradient of the loss with respect to the logits, scaled
};

struct GemmArgs {
  int64_t M = 0;
  int N = 0;
  int tiles_m = 0, tiles_n = 0, kblocks = 0;
  int run = 1, units = 0;  // see UnitWalk
  int len_fast = 0, len_slow = 0, step_fast = 0, step_slow = 0;
  int ctas = 0;  // or pairs
  int m_fast = 0;        // tile order: rows of tiles vary fastest, else columns
  int a_mn = 0, b_mn = 0;  // operand stored with its rows contiguous
  uint32_t idesc = 0;
  // epilogue matrices
  int extra_tma = 1, out_tma = 1;  // staging moves by TMA; else by the warps from / to the pointers below
  const void* bias = nullptr;   // [N]
  const void* extra = nullptr;  // [M, N]
  void* out = nullptr;          // [M, N]
  int has_extra = 0;
  int64_t ld_extra = 0, ld_out = 0;  // of the warps' own moves
  float alpha = 1.0f;
  const float* alpha_dev = nullptr;  // further factor held on the device
  float* sums = nullptr;  // kEpiActGrad: column sums of out before its rounding, see above
  int slab_rows = 0;     // rows between slabs
  int slab_add = 0;      // add to what the slab holds
  // softmax loss: rows are queries, columns bank rows col0 + n
  float c2 = 0.0f;       // scale * log2(e)
  int64_t col0 = 0;
  const int64_t* target = nullptr;   // [M]
  float2* partial = nullptr;         // [runs * groups, M] (max, sum) of a group's columns, base 2
  const float4* rows = nullptr;      // [M] GradRows
};

// What the gradient of a row's logits needs: lse in base 2, the row's weight w = g_i / max|g| times a
// scale of at most kGradScale (0: the row takes no part) and the value at the target, expm1(-loss) * w.
//   d loss_i / d s_ij = p_ij - [j = t_i],   p_ij - 1 = expm1(-loss_i) at the target
// The gradient of the logits is rounded to the operands' 16 bits, since it is the operand of the two
// products that follow; what that takes off the target's entry, the largest of its row, is added to dq by
// itself (at_rest, see loss_operands_kernel).  |p - 1| <= 1, so with |w| <= 2^14 nothing overflows in fp16 and
// probabilities down to 2^-27 keep all 11 bits; the factor max|g| * scale / w returns in fp32.
struct GradRows {
  float lse2, w, at_target, at_rest;
};

__device__ __forceinline__ float ex2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: 8-row atoms 1024 bytes apart (stride
// offset).  MN-major: an atom is 64 values of the rows by 8 of k; the next 8 of k are 1024 bytes
// on (stride offset), the next 64 rows one whole k-block on, kBK * 128 bytes (leading offset).
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int mn)
{
  const uint32_t lead = mn ? kBK * 128u : 16u;
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
  if (CG == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// Arrives on `bar` of this CTA, or of both CTAs of the pair, once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar)
{
  if (CG == 1)
    tc_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

// Tile load whose bytes are counted on `bar`, a barrier of the pair's leader.
template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
  if (CG == 1)
    tma_load_2d(dst, map, x, y, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// The leader's copy of a shared-memory address, in the cluster's window.
__device__ __forceinline__ uint32_t leader_addr(uint32_t addr)
{
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}

template <int CG>
__device__ __forceinline__ void arrive_leader(uint32_t bar)
{
  if (CG == 1)
    mbar_arrive(bar);
  else
    // what the arrival orders is TMEM reads, and the tcgen05 fence before it has
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
}

__device__ __forceinline__ void cluster_sync()
{
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Bounded wait that gives up once any role has failed.
__device__ __forceinline__ bool op_wait(uint32_t bar, uint32_t parity, volatile int* fail)
{
  for (uint32_t it = 0; it < kOpWaitLimit; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 255u) == 255u && *fail) return false;
  }
  return false;
}

// Bounded wait for copies or MMAs in flight after a failure.
__device__ __forceinline__ void op_drain(uint32_t bar, uint32_t parity)
{
  volatile int never = 0;
  op_wait(bar, parity, &never);
}

__device__ __forceinline__ void fail_with(volatile int* fail, int code)
{
  *fail = 1;
  atomicExch(&g_op_err, code);
}

__device__ __forceinline__ void group_sync(int wg) { asm volatile("bar.sync %0, 128;" ::"r"(wg + 1) : "memory"); }

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y)
{
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, uint32_t src, int x, int y)
{
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <typename T>
struct Pack;
template <>
struct Pack<__half> {
  static __device__ __forceinline__ uint32_t two(float a, float b)
  {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 get(uint32_t u)
  {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  static __device__ __forceinline__ float one(__half h) { return __half2float(h); }
  static __device__ __forceinline__ __half from(float f) { return __float2half_rn(f); }
};
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t two(float a, float b)
  {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 get(uint32_t u)
  {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 h) { return __bfloat162float(h); }
  static __device__ __forceinline__ __nv_bfloat16 from(float f) { return __float2bfloat16_rn(f); }
};

__device__ __forceinline__ float max_nan(float a, float b)
{
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// GELU z Phi(z) = max(z, 0) - t(w), w = |z|, with the tail t(w) = w Phi(-w); its slope Phi(z) + z phi(z) is
// s(w) = Phi(-w) - w phi(w) for z <= 0 and 1 - s(w) for z > 0.  Both are e^{-w^2 / 2} times a smooth function of w,
// whose zeros are taken out as factors:
//   t(w) = e^{-w^2 / 2} w P(w),   s(w) = e^{-w^2 / 2} (w0 - w) Q(w),   s(w0) = 0
// so that polynomials for P and Q hold the relative error of the tails, which 16-bit outputs show to the last
// bit (at z = -5 an absolute error of 8e-7 is half the value).  Own minimax fits by linear programming, in
// powers of -w.  What they add to the one rounding of the output, in units of that: 0.14 (value) and 0.16 (slope) in
// fp16, 0.21 and 0.18 in bf16 up to w = 5; past it, in fp16, as much and 0.32 down to the subnormal values (a value is
// 0 from w = 6, and a slope past 8 times any gradient); in bf16, whose exponents reach w = 13.1, 0.79 and 0.82.
// Their absolute error stays under 3e-6 (1 + w).  From w = 13.2 on the exponential is 0.
// bf16's value past w = 6.5 is a constant times an exponential: w P(w) rises by 1.8 % from there to 13, and the
// exponential of (1 - 2.6e-4) w^2 / 2 rises along with it (P on [0, 6.5] makes up for that).  Without that the
// polynomial took two terms more, in powers of 4.75 - w to keep it from cancelling: 15 % more of the layer's time
// than the absolute fit named below, where this one takes 3 %.
// On one B200, 819,200 x 256 -> 1,024 in fp16: 660 us; polynomials for an absolute error of 8e-7, one term shorter,
// 641; erff and expf 1.85 times as long as those.  The slope's kernel, 51,200 x 256 -> 1,024: 72 us, 67 with one for an
// absolute error of 4e-6.
__device__ __forceinline__ uint64_t gauss2(uint64_t z, float c = -0.72134752f)  // 2^{c z^2}, e^{-z^2 / 2} unless told
{
  const float2 t = split(mul2(mul2(z, z), pair(c, c)));
  return pair(ex2(t.x), ex2(t.y));
}
template <int N>
__device__ __forceinline__ uint64_t horner2(const float (&c)[N], uint64_t x)
{
  uint64_t r = pair(c[N - 1], c[N - 1]);
#pragma unroll
  for (int i = N - 2; i >= 0; --i) r = fma2(r, x, pair(c[i], c[i]));
  return r;
}
// (-w, -w) of two values, w at most `end`
__device__ __forceinline__ uint64_t minus_abs(float2 v, float end)
{
  return pair(fmaxf(-fabsf(v.x), -end), fmaxf(-fabsf(v.y), -end));
}
template <typename T, int ACT>
__device__ __forceinline__ float2 act_of(uint64_t z)
{
  const float2 v = split(z);
  if (ACT == RBQ_ACT_RELU) return make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
  if (ACT == RBQ_ACT_GELU) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const float half[10] = {0.499972373f,  0.398479819f,  0.247432157f,   0.126111999f,   0.0520200133f,
                            0.0164886173f, 0.0037531869f, 0.000565699709f, 4.99067755e-05f, 1.93591131e-06f};
    const float bf16[10] = {0.499914378f,  0.397714943f,   0.244145826f,   0.119834676f,   0.0455746762f,
                            0.0126912659f, 0.00243611634f, 0.000300497486f, 2.12530103e-05f, 6.51733785e-07f};
    const uint64_t nw = minus_abs(v, kHalf ? 6.0f : 6.5f), g = kHalf ? gauss2(z) : gauss2(z, -0.721159995f);
    const uint64_t p = kHalf ? horner2(half, nw) : horner2(bf16, nw);
    return split(fma2(mul2(g, nw), p, pair(fmaxf(v.x, 0.0f), fmaxf(v.y, 0.0f))));
  }
  return v;
}
template <typename T, int ACT>
__device__ __forceinline__ float2 act_slope(uint64_t z)
{
  const float2 v = split(z);
  if (ACT == RBQ_ACT_RELU)
    return make_float2(v.x > 0.0f ? 1.0f : (v.x != v.x ? v.x : 0.0f), v.y > 0.0f ? 1.0f : (v.y != v.y ? v.y : 0.0f));
  if (ACT == RBQ_ACT_GELU) {
    const float root = 0.751791525f;
    uint64_t nw, p;
    if (std::is_same<T, __half>::value) {
      const float c[10] = {0.66507566f,    0.176510572f,   0.096318841f,    0.0434494428f,   0.015321183f,
                           0.00392379053f, 0.00068282726f, 7.52700944e-05f, 4.69856604e-06f, 1.25869008e-07f};
      nw = minus_abs(v, 8.0f);
      p = horner2(c, nw);
    } else {
      const float c[11] = {0.66507411f,    0.176427275f,    0.095736444f,    0.0421805046f,   0.0141140036f,  0.0033448264f,
                           0.000535338011f, 5.57655512e-05f, 3.59613659e-06f, 1.29842135e-07f, 2.00207539e-09f};
      nw = minus_abs(v, 13.25f);
      p = horner2(c, nw);
    }
    const float2 t = split(mul2(mul2(gauss2(z), add2(nw, pair(root, root))), p));
    return make_float2(v.x > 0.0f ? 1.0f - t.x : t.x, v.y > 0.0f ? 1.0f - t.y : t.y);
  }
  return make_float2(1.0f, 1.0f);
}

struct Tile {
  int m, n;
};
// Steps through a CTA's (or pair's) tiles in order; every role walks the same sequence.  A unit of work is
// a run of `run` tiles next to each other in one row of tiles (one tile but for the loss's forward pass);
// units vary fastest along the shorter side of the product.  A step adds the grid's size to the unit's
// (fast, slow) digits: no division, which every thread of the epilogue would pay for at each tile.
struct UnitWalk {
  const GemmArgs& a;
  int fast, slow, r;
  __device__ __forceinline__ UnitWalk(const GemmArgs& args, int first) : a(args), r(0)
  {
    slow = first / a.len_fast;
    fast = first - slow * a.len_fast;
  }
  __device__ __forceinline__ bool live() const { return slow < a.len_slow; }
  __device__ __forceinline__ Tile tile() const
  {
    return a.m_fast ? Tile{fast, slow * a.run + r} : Tile{slow, fast * a.run + r};
  }
  __device__ __forceinline__ bool run_starts() const { return r == 0; }
  __device__ __forceinline__ bool run_ends() const
  {
    return r + 1 == a.run || (a.m_fast ? slow : fast) * a.run + r + 1 == a.tiles_n;
  }
  __device__ __forceinline__ int k_begin() const { return 0; }
  __device__ __forceinline__ int k_end() const { return a.kblocks; }
  __device__ __forceinline__ int slab() const { return 0; }
  __device__ __forceinline__ void next()
  {
    if (!run_ends()) {
      ++r;
      return;
    }
    r = 0;
    fast += a.step_fast;
    slow += a.step_slow;
    if (fast >= a.len_fast) fast -= a.len_fast, ++slow;
  }
};
// The k-blocks of all tiles, column by column, laid end to end: CTA p of P takes [T p / P, T (p + 1) / P) of
// the T of them.  Its part of a tile is the tile's slab number p - (the first CTA that has a part of it).
__host__ __device__ __forceinline__ int64_t first_cta(int64_t at, int64_t ctas, int64_t total)
{
  return ((at + 1) * ctas - 1) / total;  // the last p with T p / P <= at
}
struct RangeWalk {
  const GemmArgs& a;
  int64_t at, end;
  int cta, t, k;  // tile and k-block of `at`
  __device__ __forceinline__ RangeWalk(const GemmArgs& args, int first) : a(args), cta(first)
  {
    const int64_t total = (int64_t)a.tiles_m * a.tiles_n * a.kblocks;
    at = total * first / a.ctas;
    end = total * (first + 1) / a.ctas;
    t = (int)(at / a.kblocks);
    k = (int)(at - (int64_t)t * a.kblocks);
  }
  __device__ __forceinline__ bool live() const { return at < end; }
  __device__ __forceinline__ Tile tile() const { return Tile{t % a.tiles_m, t / a.tiles_m}; }
  __device__ __forceinline__ bool run_starts() const { return true; }
  __device__ __forceinline__ bool run_ends() const { return true; }
  __device__ __forceinline__ int k_begin() const { return k; }
  __device__ __forceinline__ int k_end() const { return (int)min((int64_t)a.kblocks, k + end - at); }
  __device__ __forceinline__ int slab() const
  {
    return cta - (int)first_cta((int64_t)t * a.kblocks, a.ctas, (int64_t)a.tiles_m * a.tiles_n * a.kblocks);
  }
  __device__ __forceinline__ void next()
  {
    at += k_end() - k;
    ++t;
    k = 0;
  }
};

template <int EPI, int CG>
struct Shape {
  static constexpr int kBN = 128 * CG;             // columns of a tile and of its accumulator
  static constexpr int kGroups = kBN / 64;         // epilogue warpgroups
  static constexpr int kThreads = kGroups * 128 + 64;
  static constexpr int kLoadWarp = kGroups * 4, kMmaWarp = kLoadWarp + 1;
  static constexpr int kOperands = 2 * kBM * 128;  // a CTA's share of a stage: 128 rows of A, 128 of B
  // Staging buffers per group: none in the loss's forward pass, which writes no tile; two where an extra
  // input streams in for every tile (its load then overlaps the tile before), else one.
  static constexpr int kBufs = EPI == kEpiLse ? 0 : EPI == kEpiActGrad ? 2 : 1;
  static constexpr int kBufBytes = EPI == kEpiSlab ? kSlabOut : kStageOut;
  static constexpr int kOutBytes = kGroups * kBufs * kBufBytes;
  // Stages, staging, [2][BN] bias values, barriers: as many stages as 227 KB hold, all of it in dynamic
  // shared memory, which starts on the 1,024 bytes that the swizzle wants when there is no other.
  static constexpr int kTail = 2 * kBN * 4 + 256;
  static constexpr int kFit = (227 * 1024 - kTail - kOutBytes) / kOperands;
  static constexpr int kStages = kFit < 7 ? kFit : 7;
  static constexpr int kBytes = kStages * kOperands + kOutBytes + kTail;
  static_assert((2 * kStages + 4 + kGroups * 2) * 8 + 8 <= 256, "barriers");
};

// The warp's 32 staging rows <-> a matrix of 16-bit values whose rows no TMA can address, 64 columns from
// `col`: a lane has columns lane and lane + 32, so that an access covers 64 bytes in a row.  BATCH rows are on
// their way at a time: 200,000 x 300 -> 333 with a residual takes 278 us, row by row in pairs of columns 499.
// Eight rows of loads gain 20 us there but cost the other products their registers (aligned GELU training 143
// -> 151).  4-byte accesses, rows that start between them shifted over the lanes, were slower (495).
template <bool LOAD, int BATCH>
__device__ __forceinline__ void move_rows(unsigned char* buf, void* mat, int64_t row0, int64_t M, int64_t ld, int col, int N,
                                          int warp_row, int lane)
{
  const bool in0 = col + lane < N, in1 = col + lane + 32 < N;
  uint16_t* g = reinterpret_cast<uint16_t*>(mat) + (row0 + warp_row) * ld + col + lane;
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += BATCH, g += BATCH * ld) {
    const int row = warp_row + r0, rows = (int)min((int64_t)BATCH, M - row0 - row);
    auto at = [&](int r, int half) {
      return reinterpret_cast<uint16_t*>(buf + (row + r) * 128 + (((lane >> 3) + half * 4) ^ ((row + r) & 7)) * 16 +
                                         (lane & 7) * 2);
    };
    uint16_t v[BATCH], w[BATCH];
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
      const bool in = r < rows;
      v[r] = LOAD ? (in && in0 ? g[r * ld] : 0) : *at(r, 0);
      w[r] = LOAD ? (in && in1 ? g[r * ld + 32] : 0) : *at(r, 1);
    }
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
      if (LOAD) {
        *at(r, 0) = v[r];
        *at(r, 1) = w[r];
      } else if (r < rows) {
        if (in0) g[r * ld] = v[r];
        if (in1) g[r * ld + 32] = w[r];
      }
    }
  }
}

template <int EPI, typename T, int CG, int ACT>
__global__ void __launch_bounds__(Shape<EPI, CG>::kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ GemmArgs a)
{
  using S = Shape<EPI, CG>;
  using Walk = typename std::conditional<EPI == kEpiSlab, RangeWalk, UnitWalk>::type;
  constexpr int BN = S::kBN, kLoadWarp = S::kLoadWarp, kMmaWarp = S::kMmaWarp, kGroups = S::kGroups;
  extern __shared__ __align__(1024) unsigned char gemm_smem[];
  unsigned char* base = gemm_smem;
  if (smem_u32(base) & 1023u) {  // the swizzle pattern is taken from the address bits
    if (threadIdx.x == 0) atomicExch(&g_op_err, 7);
    return;
  }
  unsigned char* staging = base + S::kStages * S::kOperands;
  float* s_bias = reinterpret_cast<float*>(staging + S::kOutBytes);  // [2][BN]: this tile's and the next one's
  unsigned long long* s_full = reinterpret_cast<unsigned long long*>(s_bias + 2 * BN);
  unsigned long long *s_empty = s_full + S::kStages, *s_done = s_empty + S::kStages, *s_free = s_done + 2, *s_x = s_free + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_x + kGroups * 2);
  int* s_fail = reinterpret_cast<int*>(s_tmem + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 2 ? (int)(blockIdx.x & 1) : 0;  // in the pair; 0 leads
  const int first_unit = blockIdx.x / CG;
  if (warp == kMmaWarp) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                   "r"((uint32_t)(2 * BN)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                   "r"((uint32_t)(2 * BN)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_done[i]), 1);
      mbar_init(smem_u32(&s_free[i]), kGroups * 4 * CG);  // one arrival per epilogue warp of the pair
    }
    for (int i = 0; i < kGroups * 2; ++i) mbar_init(smem_u32(&s_x[i]), 1);
    *s_fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG == 2) cluster_sync();  // the pair's barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *s_tmem;
  volatile int* fail = s_fail;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
      int st = 0, done = 0;  // stage of the next k-block; k-blocks asked for (kStages at most are counted)
      uint32_t lap = 0;      // parity of the ring's laps
      bool ok = true;
      const uint32_t full0 = CG == 2 ? leader_addr(smem_u32(&s_full[0])) : smem_u32(&s_full[0]);
      for (Walk w(a, first_unit); w.live() && ok; w.next()) {
        const Tile tl = w.tile();
        const int m0 = (tl.m * CG + rank) * kBM, n0 = tl.n * BN + rank * 128;  // this CTA's rows of A and of B
        for (int kb = w.k_begin(), ke = w.k_end(); kb < ke; ++kb) {
          if (done == S::kStages && !op_wait(smem_u32(&s_empty[st]), lap ^ 1, fail)) {
            fail_with(fail, 1);
            ok = false;
            break;
          }
          const uint32_t full = full0 + st * 8;
          const uint32_t sa = smem_u32(base) + st * S::kOperands, sb = sa + kBM * 128;
          if (rank == 0) mbar_expect_tx(smem_u32(&s_full[st]), (uint32_t)(CG * S::kOperands));
          const int k0 = kb * kBK;
          if (a.a_mn) {
#pragma unroll
            for (int j = 0; j < 2; ++j) load_tile<CG>(sa + j * kBK * 128, &tmA, m0 + j * 64, k0, full);
          } else {
            load_tile<CG>(sa, &tmA, k0, m0, full);
          }
          if (a.b_mn) {
#pragma unroll
            for (int j = 0; j < 2; ++j) load_tile<CG>(sb + j * kBK * 128, &tmB, n0 + j * 64, k0, full);
          } else {
            load_tile<CG>(sb, &tmB, k0, n0, full);
          }
          if (done < S::kStages) ++done;
          if (++st == S::kStages) st = 0, lap ^= 1;
        }
      }
      // The last lap.  The pair's MMAs arrive on both CTAs' barriers: all have before this one's shared
      // memory goes away.  After a failure the copies in flight land first (the leader's barriers count
      // those of both CTAs).
      for (int i = 0; i < done; ++i) {
        if (st == 0) st = S::kStages, lap ^= 1;
        --st;
        if (!*fail && !op_wait(smem_u32(&s_empty[st]), lap, fail)) fail_with(fail, 6);
        if (*fail && rank == 0) op_drain(smem_u32(&s_full[st]), lap);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    if (lane == 0 && rank == 0) {
      // One thread issues every MMA: descriptors are one addition each.
      const uint32_t a_step = (a.a_mn ? 16 * 128 : 32) >> 4, b_step = (a.b_mn ? 16 * 128 : 32) >> 4;  // 16 values of k
      const uint64_t a_desc = operand_desc(smem_u32(base), a.a_mn), b_desc = operand_desc(smem_u32(base) + kBM * 128, a.b_mn);
      int st = 0, i = 0;
      uint32_t lap = 0;
      bool ok = true, any = false;
      for (Walk w(a, first_unit); w.live() && ok; w.next(), ++i) {
        const int acc = i & 1;
        if (i >= 2 && !op_wait(smem_u32(&s_free[acc]), (uint32_t)(((i >> 1) - 1) & 1), fail)) {
          fail_with(fail, 2);
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + acc * BN;
        uint32_t into = 0;  // the first MMA overwrites the accumulator
        for (int left = w.k_end() - w.k_begin(); left > 0; --left) {
          if (!op_wait(smem_u32(&s_full[st]), lap, fail)) {
            fail_with(fail, 3);
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t ad = a_desc + st * (S::kOperands >> 4), bd = b_desc + st * (S::kOperands >> 4);
#pragma unroll
          for (int ks = 0; ks < kBK / 16; ++ks) {
            mma_f16<CG>(d, ad + ks * a_step, bd + ks * b_step, a.idesc, into);
            into = 1;
          }
          commit<CG>(smem_u32(&s_empty[st]));
          any = true;
          if (++st == S::kStages) st = 0, lap ^= 1;
        }
        if (ok) commit<CG>(smem_u32(&s_done[acc]));
      }
      // MMAs still running after a failure end before TMEM is freed: the last commit follows them.
      if (*fail && any) {
        if (st == 0) st = S::kStages, lap ^= 1;
        op_drain(smem_u32(&s_empty[st - 1]), lap);
      }
    }
    __syncwarp();
  } else {
    const int wg = warp >> 2, quarter = warp & 3;
    const int gt = tid & 127;  // thread of the group = accumulator lane = output row
    const bool leader = gt == 0;
    constexpr bool kElement = EPI == kEpiLinear || EPI == kEpiActGrad;
    unsigned char* bufs = staging + wg * S::kBufs * S::kBufBytes;
    float* bias = s_bias + wg * 64;
    bool dead = false;  // a wait failed: keep the barriers in step, touch nothing
    int c = 0;          // staging tile, counted over the group's run: buffer c % kBufs
    auto buf_of = [&](int k) { return bufs + (S::kBufs == 2 ? (k & 1) * kStageOut : 0); };
    auto bar_of = [&](int k) { return smem_u32(&s_x[wg * 2 + (S::kBufs == 2 ? k & 1 : 0)]); };
    auto parity_of = [&](int k) { return (uint32_t)((S::kBufs == 2 ? k >> 1 : k) & 1); };

    // The extra inputs of the group's tiles arrive by TMA, in order; `ask` is the next tile to ask for.
    const bool extra_tma = kElement && a.has_extra && a.extra_tma;
    int loaded = 0;
    Walk ask(a, first_unit);
    auto ask_extra = [&]() {
      while (ask.live() && ask.tile().n * BN + wg * 64 >= a.N) ask.next();
      if (!ask.live()) return;
      const Tile tl = ask.tile();
      mbar_expect_tx(bar_of(loaded), (uint32_t)kStageOut);
      tma_load_2d(smem_u32(buf_of(loaded)), &tmX, tl.n * BN + wg * 64, (tl.m * CG + rank) * kBM, bar_of(loaded));
      ++loaded;
      ask.next();
    };
    if (extra_tma && leader) ask_extra();

    // What a thread needs of the next tile besides the accumulator is read one tile ahead.
    float next_bias = 0.0f;
    int64_t next_target = -1;
    float4 next_rows = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto read_ahead = [&](const Walk& w) {
      if (!w.live()) return;
      const Tile tl = w.tile();
      const int64_t row = (int64_t)(tl.m * CG + rank) * kBM + gt;
      if (kElement) {
        const int col = tl.n * BN + wg * 64 + gt;
        next_bias = a.bias != nullptr && gt < 64 && col < a.N ? Pack<T>::one(reinterpret_cast<const T*>(a.bias)[col]) : 0.0f;
      }
      if (EPI == kEpiLse || EPI == kEpiProb) next_target = row < a.M ? __ldg(a.target + row) : -1;
      if (EPI == kEpiProb) next_rows = row < a.M ? __ldg(a.rows + row) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    Walk w(a, first_unit);
    read_ahead(w);
    uint64_t sums[4] = {};  // of columns 16 i + 2 (lane % 8) and the next of the group, over the lane's rows
    int sums_n = -1;        // the column of tiles that they belong to
    const int sum_at = quarter * 4096 + (lane >> 3) * 1024 + (lane & 7) * 8;  // first of the lane's 8 rows
    auto write_sums = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 two = split(sums[i]);
        float e[2] = {two.x, two.y};
        const int col = sums_n * BN + wg * 64 + i * 16 + (lane & 7) * 2;
        float* at = a.sums + ((int64_t)(first_unit * CG + rank) * 4 + quarter) * a.N + col;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) e[k] += __shfl_xor_sync(0xffffffffu, e[k], o);
          if (lane < 8 && col + k < a.N) at[k] = e[k];
        }
      }
    };
    if (kElement) {
      if (gt < 64) bias[gt] = next_bias;
      group_sync(wg);
    }
    float alpha = a.alpha;
    if (a.alpha_dev != nullptr) alpha *= __ldg(a.alpha_dev);
    float m = -INFINITY, l = 0.0f;  // of the run of tiles so far (kEpiLse)

    for (int i = 0; w.live(); ++i) {
      const Tile tl = w.tile();
      const int acc = i & 1;
      const uint32_t acc_addr = tmem + acc * BN + wg * 64 + ((uint32_t)(quarter * 32) << 16);
      const int64_t m0 = (int64_t)(tl.m * CG + rank) * kBM;
      const int n0 = tl.n * BN + wg * 64;
      const int64_t row = m0 + gt;
      const int64_t tj = next_target < 0 ? -1 : next_target - a.col0 - n0;  // the target's column here, if it is one
      const GradRows gr{next_rows.x, next_rows.y, next_rows.z, next_rows.w};
      const bool some = n0 < a.N;  // the group's columns lie in the matrix
      const bool first_of_run = w.run_starts(), last_of_run = w.run_ends();
      const int slab = w.slab();
      w.next();
      read_ahead(w);
      if (!dead) {
        const bool ok = op_wait(smem_u32(&s_done[acc]), (uint32_t)((i >> 1) & 1), fail);
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) fail_with(fail, 4);
          dead = true;
        }
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // The share is read 32 columns at a time (64 at once spilled registers), the accumulator free after
      // the second read.
      auto read_half = [&](int h, float (&v)[32]) {
        if (!dead && some) tc_ld32(acc_addr + h * 32, v);
        if (h == 1) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_leader<CG>(smem_u32(&s_free[acc]));
        }
      };

      if (EPI == kEpiLse) {
        if (first_of_run) m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[32];
          read_half(h, v);
          if (dead || !some) continue;
          const int64_t th = tj - h * 32;
          if (__any_sync(0xffffffffu, (uint64_t)th < 32u)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = e == th ? -INFINITY : v[e];
          }
          if (n0 + h * 32 + 32 > a.N) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = n0 + h * 32 + e < a.N ? v[e] : -INFINITY;
          }
          float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int e = 4; e < 32; ++e) top[e & 3] = fmaxf(top[e & 3], v[e]);
          const float mn = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.c2);
          const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing but masked logits so far
          const uint64_t c2 = pair(a.c2, a.c2), nref = pair(-ref, -ref);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = split(fma2(pair(v[e], v[e + 1]), c2, nref));
            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair(ex2(x.x), ex2(x.y)));
          }
          const float2 t2 = split(add2(sum[0], sum[1]));
          l = fmaf(l, ex2(m - ref), t2.x + t2.y);
          m = mn;
        }
        if (last_of_run && !dead && row < a.M)
          a.partial[(int64_t)(tl.n / a.run * kGroups + wg) * a.M + row] = make_float2(m, l);
        continue;
      }
      // The next tile's bias, beside this one's; the group's barriers below publish it.
      const float* tile_bias = bias + (i & 1) * BN;
      if (kElement && gt < 64) bias[((i + 1) & 1) * BN + gt] = next_bias;
      if (!some) {
        float v[32];
        read_half(1, v);
        if (kElement) group_sync(wg);
        continue;
      }

      if (EPI == kEpiSlab) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[32];
          read_half(h, v);
#pragma unroll
          for (int q = 0; q < 32 / kSlabCols; ++q) {
            const int col = n0 + h * 32 + q * kSlabCols;
            if (col < a.N) {
              if (leader) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              group_sync(wg);  // the buffer's last store has been read
              if (!dead) {
                float4* at = reinterpret_cast<float4*>(bufs + gt * kSlabCols * 4);
#pragma unroll
                for (int k = 0; k < kSlabCols / 4; ++k) {
                  const float* e = v + q * kSlabCols + 4 * k;
                  at[k ^ ((gt >> 1) & 3)] = make_float4(e[0], e[1], e[2], e[3]);  // 64-byte swizzle
                }
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              group_sync(wg);
              if (leader && !dead && !*fail && m0 < a.M) {  // a pair's second half may lie past the last row
                const int y = slab * a.slab_rows + (int)m0;
                if (a.slab_add)
                  tma_add_2d(&tmO, smem_u32(bufs), col, y);
                else
                  tma_store_2d(&tmO, smem_u32(bufs), col, y);
              }
            }
          }
        }
        continue;
      }

      unsigned char* buf = buf_of(c);
      if (extra_tma) {
        if (S::kBufs == 2 && leader && !dead) {  // the next tile's, into the buffer whose store has been read
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          ask_extra();
        }
        if (!dead) {
          const bool ok = op_wait(bar_of(c), parity_of(c), fail);
          if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0) fail_with(fail, 5);
            dead = true;
          }
        }
      } else {
        if (a.out_tma) {
          if (leader) {
            if (S::kBufs == 2)
              asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            else
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
          group_sync(wg);  // the buffer's last store has been read
        }
        if (kElement && a.has_extra) {
          if (!dead)
            move_rows<true, 4>(buf, const_cast<void*>(a.extra), m0, a.M, a.ld_extra, n0, a.N, quarter * 32,
                               lane);
          __syncwarp();
        }
      }
      if (EPI == kEpiActGrad && a.sums != nullptr && tl.n != sums_n) {
        if (sums_n >= 0 && !dead) write_sums();
        sums_n = tl.n;
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] = 0;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        read_half(h, v);
        if (dead) continue;
        uint4* at = reinterpret_cast<uint4*>(buf + gt * 128);
        if (EPI == kEpiProb) {
          const uint64_t c2 = pair(a.c2, a.c2), nlse = pair(-gr.lse2, -gr.lse2), wt = pair(gr.w, gr.w);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = split(fma2(pair(v[e], v[e + 1]), c2, nlse));
            const float2 y = split(mul2(pair(ex2(x.x), ex2(x.y)), wt));
            v[e] = y.x;
            v[e + 1] = y.y;
          }
          const int64_t th = tj - h * 32;
          if (__any_sync(0xffffffffu, gr.w == 0.0f || (uint64_t)th < 32u)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)  // a row that takes no part gives zeros, whatever its logits
              v[e] = gr.w == 0.0f ? 0.0f : e == th ? gr.at_target : v[e];
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int slot = (h * 4 + k) ^ (gt & 7);
          float* o = v + k * 8;
          if (kElement) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (EPI == kEpiActGrad || a.has_extra) x = at[slot];
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
            const uint64_t al = pair(alpha, alpha);
            const ulonglong2* bp = reinterpret_cast<const ulonglong2*>(tile_bias + h * 32 + k * 8);
            const ulonglong2 b01 = bp[0], b23 = bp[1];
            const uint64_t b[4] = {b01.x, b01.y, b23.x, b23.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t z = fma2(pair(o[2 * e], o[2 * e + 1]), al, b[e]);
              if (EPI == kEpiActGrad) {
                const float2 f = act_slope<T, ACT>(z), g = Pack<T>::get(xs[e]);
                o[2 * e] = g.x * f.x;
                o[2 * e + 1] = g.y * f.y;
              } else {
                const float2 f = act_of<T, ACT>(z);
                o[2 * e] = f.x;
                o[2 * e + 1] = f.y;
                if (a.has_extra) {
                  const float2 r = Pack<T>::get(xs[e]);
                  o[2 * e] += r.x;
                  o[2 * e + 1] += r.y;
                }
              }
            }
          }
          if (EPI != kEpiActGrad)
            at[slot] = make_uint4(Pack<T>::two(o[0], o[1]), Pack<T>::two(o[2], o[3]), Pack<T>::two(o[4], o[5]),
                                  Pack<T>::two(o[6], o[7]));
        }
        if (EPI == kEpiActGrad) {
          if (a.sums != nullptr) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              if (q == 1) __syncwarp();  // the columns before have been read
              float4* to = reinterpret_cast<float4*>(at);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float* e = v + q * 16 + k * 4;
                to[(h * 4 + k) ^ (gt & 7)] = make_float4(e[0], e[1], e[2], e[3]);
              }
              __syncwarp();
#pragma unroll
              for (int r = 0; r < 8; ++r)
                sums[h * 2 + q] = add2(sums[h * 2 + q], *reinterpret_cast<const uint64_t*>(
                                                            buf + (sum_at ^ (h * 64) ^ (r * 16)) + r * 128));
            }
            __syncwarp();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float* o = v + k * 8;
            at[(h * 4 + k) ^ (gt & 7)] = make_uint4(Pack<T>::two(o[0], o[1]), Pack<T>::two(o[2], o[3]),
                                                    Pack<T>::two(o[4], o[5]), Pack<T>::two(o[6], o[7]));
          }
        }
      }
      if (a.out_tma) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        group_sync(wg);
        if (leader && !dead && !*fail) {
          // A pair's second half may lie past the last row: an empty group then, since the waits above count
          // one group per tile and would else take this tile's for that of the tile before.
          if (m0 < a.M)
            tma_store_2d(&tmO, smem_u32(buf), n0, (int)m0);
          else
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          if (S::kBufs == 1 && extra_tma) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            ask_extra();
          }
        }
      } else {
        __syncwarp();
        if (!dead) move_rows<false, 8>(buf, a.out, m0, a.M, a.ld_out, n0, a.N, quarter * 32, lane);
        group_sync(wg);
      }
      ++c;
    }
    if (EPI == kEpiActGrad && a.sums != nullptr && sums_n >= 0 && !dead) write_sums();
    if (leader) {
      // after a failure: extra inputs in flight land before the shared memory goes away
      if (S::kBufs > 0 && *fail && loaded > 0)
        for (int k = (loaded > S::kBufs ? loaded - S::kBufs : 0); k < loaded; ++k) op_drain(bar_of(k), parity_of(k));
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (CG == 2) cluster_sync();  // the pair is done with each other's barriers and TMEM
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN)));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN)));
  }
}

// ---------------------------------------------------------------------------------------
// Small kernels around the products.
// ---------------------------------------------------------------------------------------

// Rows of `cols` 16-bit values -> rows `ld` apart (ld a multiple of 8, so that TMA can address them).  A thread
// makes 16 bytes of the copy.
__global__ void pad_rows_kernel(const uint16_t* __restrict__ src, int64_t rows, int cols, int ld,
                                uint16_t* __restrict__ dst)
{
  const int per = ld / 8;
  for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < rows; r += (int64_t)gridDim.x * blockDim.y) {
    for (int i = threadIdx.x; i < per; i += blockDim.x) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i * 8 + e < cols ? src[r * cols + i * 8 + e] : 0u;
      *reinterpret_cast<uint4*>(dst + r * ld + i * 8) =
          make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
  }
}

// out[m, n] = alpha * sum over the tile's slabs in ascending order, + extra [m, n] if there is one; slab rows are ld
// (multiple of 4) apart.
// With `ctas` the slabs of a tile are those of the CTAs that had a part of it (RangeWalk), else all of them.
struct SlabTiles {
  int slabs, tile, tiles_m, kblocks, ctas;  // tile: rows and columns of one
  int64_t total;                            // k-blocks of all tiles
};
template <typename T>
__global__ void add_slabs_kernel(const float* __restrict__ slabs, SlabTiles st, int64_t slab_stride, int64_t rows, int cols,
                                 int ld, float alpha, const float* __restrict__ alpha_dev, const T* __restrict__ extra,
                                 T* __restrict__ out)
{
  if (alpha_dev != nullptr) alpha *= __ldg(alpha_dev);
  const int quads = ld / 4;
  const int64_t total = rows * quads;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    int n = st.slabs;
    if (st.ctas > 0) {
      const int64_t at = ((int64_t)(c / st.tile) * st.tiles_m + r / st.tile) * st.kblocks;
      n = (int)(first_cta(at + st.kblocks - 1, st.ctas, st.total) - first_cta(at, st.ctas, st.total)) + 1;
    }
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(slabs + s * slab_stride + r * ld + c);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    T* o = out + r * cols + c;
    float e[4] = {alpha * sum.x, alpha * sum.y, alpha * sum.z, alpha * sum.w};
    if ((cols & 3) == 0) {
      if (extra != nullptr) {
        const uint2 x = *reinterpret_cast<const uint2*>(extra + r * cols + c);
        const float2 a = Pack<T>::get(x.x), b = Pack<T>::get(x.y);
        e[0] += a.x, e[1] += a.y, e[2] += b.x, e[3] += b.y;
      }
      *reinterpret_cast<uint2*>(o) = make_uint2(Pack<T>::two(e[0], e[1]), Pack<T>::two(e[2], e[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) o[j] = Pack<T>::from(extra != nullptr ? e[j] + Pack<T>::one(extra[r * cols + c + j]) : e[j]);
    }
  }
}

// Column sums of Z [rows, cols] (rows ld apart, ld a multiple of 8): block y sums its share of the
// rows into part[y][cols]; a second kernel adds the parts in their order.
constexpr int kColThreads = 256, kColGroup = 32;  // 32 lanes of 8 columns, 8 rows at a time
template <typename T>
__global__ void __launch_bounds__(kColThreads) column_sums_kernel(const T* __restrict__ Z, int64_t rows, int cols, int64_t ld,
                                                                  float* __restrict__ part)
{
  __shared__ float s_sum[kColThreads / kColGroup][kColGroup * 8 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (blockIdx.x * kColGroup + lane) * 8;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float sum[8] = {};
  if (c0 < cols) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += kColThreads / kColGroup) {
      const uint4 v = *reinterpret_cast<const uint4*>(Z + r * ld + c0);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = Pack<T>::get(u[e]);
        sum[2 * e] += f.x;
        sum[2 * e + 1] += f.y;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) s_sum[warp][lane * 8 + e] = sum[e];
  __syncthreads();
  const int c = blockIdx.x * kColGroup * 8 + threadIdx.x;
  if (c < cols) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kColThreads / kColGroup; ++w) t += s_sum[w][threadIdx.x];
    part[(int64_t)blockIdx.y * cols + c] = t;
  }
}
// The parts' columns in 32 interleaved runs, then the runs in their order.  Parts are rows of `cols`
// floats; with tiles > 0 they are the gradient kernel's sums, `each` rows from each of `ctas` CTAs (or
// pairs) that walked `tiles` tiles of `width` columns down each column, and those of a CTA that no tile
// of a column fell to are left out.
template <typename T>
__global__ void __launch_bounds__(1024) add_parts_kernel(const float* __restrict__ part, int parts, int cols, int tiles, int width,
                                                         int ctas, int each, T* __restrict__ out)
{
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  __shared__ float s_sum[32][33];
  float t = 0.0f;
  if (c < cols) {
    const int first = tiles > 0 ? (int)((int64_t)(c / width) * tiles % ctas) : 0;  // CTA of the column's first unit
#pragma unroll 4
    for (int p = run; p < parts; p += 32) {
      bool here = true;
      if (tiles > 0) {
        const int ahead = p / each - first;  // units to the CTA's first one in this column
        here = (ahead < 0 ? ahead + ctas : ahead) < tiles;
      }
      if (here) t += part[(int64_t)p * cols + c];
    }
  }
  s_sum[run][lane] = t;
  __syncthreads();
  if (run == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += s_sum[i][lane];
    out[c] = Pack<T>::from(t);
  }
}

// Softmax loss of 32 rows per block from the tiles' (max, sum) pairs.  Warp w first gathers every
// 32nd tile of all 32 rows (lane = row), then finishes row w.  The target's logit is a dot product of
// its own: with rest = log sum_{j != t} e^{s_j}, the loss log(1 + e^{rest - s_t}) of a row that has
// learnt its target is a small number that lse - s_t would lose.  The few values per row are held in
// 64 bits.
template <typename T>
__global__ void __launch_bounds__(1024) loss_rows_kernel(const float2* __restrict__ partial, int tiles, int64_t n,
                                                         const T* __restrict__ q, int64_t ldq, const T* __restrict__ bank,
                                                         int64_t ldb, int d, int64_t v, const int64_t* __restrict__ target,
                                                         float scale, float* __restrict__ loss, float* __restrict__ lse)
{
  __shared__ float s_m[32][33], s_l[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * 32;
  float m = -INFINITY, l = 0.0f;
  if (r0 + lane < n) {
    for (int t = warp; t < tiles; t += 32) {
      const float2 p = partial[(int64_t)t * n + r0 + lane];
      const float mn = fmaxf(m, p.x), ref = mn == -INFINITY ? 0.0f : mn;
      l = l * ex2(m - ref) + p.y * ex2(p.x - ref);
      m = mn;
    }
  }
  s_m[warp][lane] = m;
  s_l[warp][lane] = l;
  __syncthreads();
  const int64_t row = r0 + warp;
  if (row >= n) return;
  m = s_m[lane][warp];
  l = s_l[lane][warp];
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.0f : top;
  l *= ex2(m - ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const int64_t t = target[row];
  const bool valid = t >= 0 && t < v;
  double dot = 0.0;
  if (valid)
    for (int j = lane; j < d; j += 32)
      dot += (double)Pack<T>::one(q[row * ldq + j]) * (double)Pack<T>::one(bank[t * ldb + j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if (lane == 0) {
    const double rest = (double)top * 0.69314718055994531 + log((double)l);  // -inf: no other row
    double out = 0.0, total = rest;
    if (valid) {
      const double own = (double)scale * dot, u = rest - own;
      out = fmax(u, 0.0) + log1p(exp(-fabs(u)));
      if (u != u) out = u;
      total = own + out;
    }
    loss[row] = (float)out;
    lse[row] = (float)total;
  }
}

// Largest finite |g| of the rows that take part (1 if all are 0), and the scale of the logits' gradient: kGradScale
// times one of eight factors in (1/2, 1].  A bank row's gradient is mostly the entries of the queries that it is the target
// of, whose rounding does not average out the way the others' do; rows that have learnt about as much have entries
// of about one mantissa, and a factor that moves it up towards the next power of two halves the rounding.  The
// factor is the one with the least squared rounding of the target's entries over the first rows.  A row whose g
// is infinite or NaN has a weight that is: its own gradient and the bank's are lost, the other rows' are not.
constexpr int kScaleTries = 8;
constexpr int64_t kScaleRows = 16384;
template <typename T>
__global__ void __launch_bounds__(1024) grad_top_kernel(const float* __restrict__ g, const int64_t* __restrict__ target,
                                                        const float* __restrict__ loss, int64_t n, int64_t v, float scale,
                                                        float* __restrict__ out)
{
  __shared__ float s_red[32][kScaleTries];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    const int64_t t = target[i];
    if (t >= 0 && t < v && isfinite(g[i])) top = fmaxf(top, fabsf(g[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_red[warp][0] = top;
  __syncthreads();
  for (int w = 0; w < 32; ++w) top = fmaxf(top, s_red[w][0]);
  if (top == 0.0f) top = 1.0f;
  __syncthreads();
  float err[kScaleTries] = {};
  for (int64_t i = threadIdx.x; i < n && i < kScaleRows; i += 1024) {
    const int64_t t = target[i];
    if (t < 0 || t >= v || g[i] == 0.0f || !isfinite(g[i])) continue;
    const float at = expm1f(-loss[i]) * (g[i] / top * kGradScale);
#pragma unroll
    for (int k = 0; k < kScaleTries; ++k) {
      const float f = 1.0f - (float)k / (2 * kScaleTries), x = at * f;
      const float e = (Pack<T>::one(Pack<T>::from(x)) - x) / (f * kGradScale);
      err[k] = fmaf(e, e, err[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kScaleTries; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) err[k] += __shfl_xor_sync(0xffffffffu, err[k], o);
    if (lane == 0) s_red[warp][k] = err[k];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float least = INFINITY, factor = 1.0f;
    for (int k = 0; k < kScaleTries; ++k) {
      float sum = 0.0f;
      for (int w = 0; w < 32; ++w) sum += s_red[w][k];
      if (sum < least) least = sum, factor = 1.0f - (float)k / (2 * kScaleTries);
    }
    out[0] = top;
    out[1] = top * (scale / (kGradScale * factor));
    out[2] = kGradScale * factor;
  }
}
template <typename T>
__global__ void grad_rows_kernel(const float* __restrict__ g, const int64_t* __restrict__ target,
                                 const float* __restrict__ loss, const float* __restrict__ lse, int64_t n, int64_t v,
                                 const float* __restrict__ top, float4* __restrict__ rows)
{
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t t = target[i];
  float w = 0.0f;
  if (t >= 0 && t < v && g[i] != 0.0f) w = g[i] / top[0] * top[2];
  const float at = w == 0.0f ? 0.0f : expm1f(-loss[i]) * w;
  rows[i] = make_float4(lse[i] * kLog2e, w, at, at - Pack<T>::one(Pack<T>::from(at)));
}

// What the products of the loss's gradient read beside the logits' gradient:
//   kept [n, ld]: q with zeros in the rows that take no part.  They meet zeros of the logits' gradient in the bank's
//     sums, and zero times an infinity or NaN that such a row may hold (a batch's padding) would spoil every row of
//     dbank.  Rows ld apart, a multiple of 8.
//   rest [n, d]: what the rounding of the target's entry takes off dq, at_rest * k_target times the products' factor.
//     That entry is as large as all the others of its row together, so its rounding does not average out as theirs
//     do, and where a bank's rows lie close to the target the products' sum is far smaller than the entry: without
//     this dq was up to 1.8 times as far off as fp32 torch's.  (The bank's gradient keeps the rounding: there such
//     entries come from different queries.)
// A thread has eight values of a row.
template <typename T>
__global__ void loss_operands_kernel(const T* __restrict__ q, const T* __restrict__ bank, const int64_t* __restrict__ target,
                                     const float4* __restrict__ rows, const float* __restrict__ top, int64_t n, int d, int ld,
                                     uint16_t* __restrict__ kept, T* __restrict__ rest)
{
  const int per = ld / 8;
  const bool whole = d == ld;  // rows of whole 16-byte pieces
  for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < n; r += (int64_t)gridDim.x * blockDim.y) {
    const float4 row = rows[r];
    const float f = row.w * top[1];
    const bool add = row.w != 0.0f;  // the row takes part, so its target lies in the bank
    const uint16_t* from = reinterpret_cast<const uint16_t*>(q) + r * d;
    const uint16_t* key = reinterpret_cast<const uint16_t*>(bank) + (add ? target[r] * d : 0);
    for (int i = threadIdx.x; i < per; i += blockDim.x) {
      uint4 x = make_uint4(0, 0, 0, 0), k = x;
      uint32_t *xs = &x.x, *ks = &k.x;
      if (whole) {
        if (row.y != 0.0f) x = *reinterpret_cast<const uint4*>(from + i * 8);
        if (add) k = *reinterpret_cast<const uint4*>(key + i * 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = i * 8 + e < d;
          if (in && row.y != 0.0f) xs[e / 2] |= (uint32_t)from[i * 8 + e] << (e & 1) * 16;
          if (in && add) ks[e / 2] |= (uint32_t)key[i * 8 + e] << (e & 1) * 16;
        }
      }
      *reinterpret_cast<uint4*>(kept + r * ld + i * 8) = x;
      if (rest == nullptr) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 two = Pack<T>::get(ks[e]);
        ks[e] = add ? Pack<T>::two(f * two.x, f * two.y) : 0u;
      }
      uint16_t* to = reinterpret_cast<uint16_t*>(rest) + r * d + i * 8;
      if (whole) {
        *reinterpret_cast<uint4*>(to) = k;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i * 8 + e < d) to[e] = (uint16_t)(ks[e / 2] >> (e & 1) * 16);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------
constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A row-major matrix [rows, cols] with rows ld values apart.
struct Matrix {
  const void* p;
  int64_t rows, cols, ld;
};

CUtensorMap tile_map(const void* p, CUtensorMapDataType type, int esize, int64_t rows, int64_t cols, int64_t ld, int box_cols,
                     int box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B)
{
  CUtensorMap m;
  // The encoder is a driver call and wants the device's context bound to this host thread, which
  // a thread that has made no runtime call yet (autograd's) lacks.
  thread_local int bound = -1;
  int dev = 0;
  RBQ_CUDA(cudaGetDevice(&dev));
  if (bound != dev) {
    RBQ_CUDA(cudaSetDevice(dev));
    bound = dev;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * esize};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = tensor_map_encoder()(&m, type, 2, const_cast<void*>(p), dims, strides, box, estr,
                                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RBQ_CHECK(r == CUDA_SUCCESS, RBQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return m;
}

template <typename T>
constexpr CUtensorMapDataType map_type()
{
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}
// 64 columns by `box_rows` rows of an operand or output.
template <typename T>
CUtensorMap matrix_map(const Matrix& m, int box_rows)
{
  return tile_map(m.p, map_type<T>(), 2, m.rows, m.cols, m.ld, 64, box_rows);
}

template <int EPI, typename T, int CG, int ACT>
void launch_gemm(GemmArgs& a, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                 cudaStream_t s)
{
  using S = Shape<EPI, CG>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit has been raised
  int dev = 0;
  RBQ_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    RBQ_CUDA(cudaFuncSetAttribute(gemm_kernel<EPI, T, CG, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg{};
  if (EPI != kEpiSlab) a.ctas = std::min(a.units, device_sm_count() / CG);
  a.step_fast = a.ctas % a.len_fast;
  a.step_slow = a.ctas / a.len_fast;
  cfg.gridDim = dim3((unsigned)(CG * a.ctas));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  RBQ_CUDA(cudaLaunchKernelEx(&cfg, gemm_kernel<EPI, T, CG, ACT>, ta, tb, tx, to, a));
  RBQ_LAUNCHED();
}

// One product.  A is [M, K] (or [K, M] with a_mn), B [N, K] (or [K, N] with b_mn); cg as in the kernel.
template <int EPI, typename T, int ACT = RBQ_ACT_NONE>
void gemm(GemmArgs a, Matrix A, bool a_mn, Matrix B, bool b_mn, int cg, const CUtensorMap* tx, const CUtensorMap* to,
          cudaStream_t s)
{
  a.M = a_mn ? A.cols : A.rows;
  a.N = (int)(b_mn ? B.cols : B.rows);
  const int64_t K = a_mn ? A.rows : A.cols;
  a.a_mn = a_mn;
  a.b_mn = b_mn;
  const int64_t tm = ceil_div(a.M, kBM * cg), tn = ceil_div(a.N, 128 * cg), kb = ceil_div(K, kBK);
  RBQ_CHECK(tm * tn < (1ll << 31) && K < (1ll << 31) && a.M < (1ll << 31) - 256, RBQ_ERR_INVALID,
            "matrix product: sizes too large");
  a.tiles_m = (int)tm;
  a.tiles_n = (int)tn;
  a.kblocks = (int)kb;
  // The operand with fewer tiles stays in L2 while the other streams by once; column sums want columns.
  a.m_fast = tm <= tn || a.sums != nullptr;
  const int runs = (int)ceil_div(tn, a.run);
  a.len_fast = a.m_fast ? (int)tm : runs;
  a.len_slow = a.m_fast ? runs : (int)tm;
  a.units = a.len_fast * a.len_slow;
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  a.idesc = (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
            ((uint32_t)(128 * cg >> 3) << 17) | ((uint32_t)(kBM * cg >> 4) << 24);
  const CUtensorMap ta = matrix_map<T>(A, a_mn ? kBK : 128), tb = matrix_map<T>(B, b_mn ? kBK : 128);
  const CUtensorMap& x = tx ? *tx : ta;
  const CUtensorMap& o = to ? *to : ta;
  if (cg == 2)
    launch_gemm<EPI, T, 2, ACT>(a, ta, tb, x, o, s);
  else
    launch_gemm<EPI, T, 1, ACT>(a, ta, tb, x, o, s);
}

// CTAs of a tile: pairs with 256 x 256 tiles where there is one for every SM pair, else single CTAs
// with 128 x 128 tiles, which spread a small product over four times as many SMs.
int group_size(int64_t M, int64_t N) { return N > 128 && ceil_div(M, 256) * ceil_div(N, 256) >= device_sm_count() / 2 ? 2 : 1; }

// Carves aligned pieces out of the caller's workspace; with no workspace it only counts.
struct Carver {
  char* base;
  int64_t used = 0;
  explicit Carver(void* p) : base(static_cast<char*>(p)) {}
  template <typename U>
  U* take(int64_t count)
  {
    U* p = base ? reinterpret_cast<U*>(base + used) : nullptr;
    used += round_up(std::max<int64_t>(count, 1) * (int64_t)sizeof(U), 1024);
    return p;
  }
};

// Blocks of 256 threads, each with eight values of a row.
struct RowBlocks {
  dim3 block;
  unsigned blocks;
  RowBlocks(int64_t rows, int ld)
  {
    int x = 8;  // threads to a row
    while (x < 256 && x < ld / 8) x *= 2;
    block = dim3(x, 256 / x);
    blocks = (unsigned)std::min<int64_t>(ceil_div(rows, block.y), (int64_t)device_sm_count() * 16);
  }
};

void pad_rows(const void* src, int64_t rows, int cols, int ld, void* dst, cudaStream_t s)
{
  const RowBlocks l(rows, ld);
  pad_rows_kernel<<<l.blocks, l.block, 0, s>>>(static_cast<const uint16_t*>(src), rows, cols, ld,
                                               static_cast<uint16_t*>(dst));
  RBQ_LAUNCHED();
}

// The matrix itself where TMA can address its rows, else a padded copy in the workspace.
Matrix addressable(const void* p, int64_t rows, int cols, Carver& ws, bool run, cudaStream_t s)
{
  if (cols % 8 == 0) return Matrix{p, rows, cols, cols};
  const int ld = (int)round_up(cols, 8);
  uint16_t* copy = ws.take<uint16_t>(rows * ld);
  if (run) pad_rows(p, rows, cols, ld, copy, s);
  return Matrix{copy, rows, cols, ld};
}

// How out[M, N] = alpha * A B^T with a long sum is computed: at once, where its tiles fill the SMs to nine
// tenths or the sum is short, else through slabs.  A CTA takes 8 k-blocks at least, to be worth its
// prologue and its slab.
struct SlabPlan {
  bool direct;
  int cg, ctas, slabs, tiles_m, kblocks;
  int64_t rows, ld, total;  // rows and their distance in a slab; k-blocks of all tiles
  int64_t floats() const { return direct ? 0 : (int64_t)slabs * rows * ld; }
};
SlabPlan plan_slabs(int64_t M, int N, int64_t K, bool must_add)
{
  SlabPlan p;
  p.cg = N > 128 && M > 128 ? 2 : 1;
  const int64_t slots = device_sm_count() / p.cg, tm = ceil_div(M, kBM * p.cg), tiles = tm * ceil_div(N, 128 * p.cg);
  p.tiles_m = (int)tm;
  p.kblocks = (int)ceil_div(K, kBK);
  p.total = tiles * p.kblocks;
  p.direct = !must_add && (p.kblocks <= 8 || tiles * 10 >= ceil_div(tiles, slots) * slots * 9);
  p.ctas = (int)std::min(slots, std::max(tiles, p.total / 8));
  p.slabs = (int)std::min<int64_t>(p.ctas, (p.kblocks - 1) / (p.total / p.ctas) + 2);
  p.rows = round_up(M, kBM);
  p.ld = round_up(N, 4);
  RBQ_CHECK(p.direct || p.slabs * p.rows < (1ll << 31), RBQ_ERR_INVALID, "matrix product: sizes too large");
  return p;
}
template <typename T>
void slab_gemm(const SlabPlan& p, Matrix A, bool a_mn, Matrix B, bool b_mn, float* slabs, bool add, cudaStream_t s)
{
  const int64_t N = b_mn ? B.cols : B.rows;
  GemmArgs a;
  a.ctas = p.ctas;
  a.slab_rows = (int)p.rows;
  a.slab_add = add;
  const CUtensorMap to = tile_map(slabs, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.slabs * p.rows, N, p.ld, kSlabCols, kBM,
                                  CU_TENSOR_MAP_SWIZZLE_64B);
  gemm<kEpiSlab, T>(a, A, a_mn, B, b_mn, p.cg, nullptr, &to, s);
}
// `all`: every slab holds a sum (of zeros at least), else those of RangeWalk.
template <typename T>
void add_slabs(const SlabPlan& p, const float* slabs, bool all, int64_t M, int N, float alpha, const float* alpha_dev,
               const T* extra, T* out, cudaStream_t s)
{
  const int64_t blocks = std::min<int64_t>(ceil_div(M * (p.ld / 4), 256), (int64_t)device_sm_count() * 8);
  const SlabTiles st{p.slabs, 128 * p.cg, p.tiles_m, p.kblocks, all ? 0 : p.ctas, p.total};
  add_slabs_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(slabs, st, p.rows * p.ld, M, N, (int)p.ld, alpha, alpha_dev,
                                                         extra, out);
  RBQ_LAUNCHED();
}

// out[M, N] (dense) = alpha_dev * A B^T (+ extra [M, N]), written by the product's own epilogue.
template <typename T>
void store_gemm(Matrix A, bool a_mn, Matrix B, bool b_mn, int cg, const float* alpha_dev, const T* extra, T* out,
                cudaStream_t s)
{
  const int64_t M = a_mn ? A.cols : A.rows, N = b_mn ? B.cols : B.rows;
  GemmArgs a;
  a.alpha_dev = alpha_dev;
  a.extra = extra;
  a.has_extra = extra != nullptr;
  a.out = out;
  a.ld_extra = a.ld_out = N;
  a.extra_tma = a.out_tma = N % 8 == 0;
  CUtensorMap tx{}, to{};
  if (a.out_tma) {
    to = matrix_map<T>(Matrix{out, M, N, N}, kBM);
    tx = extra ? matrix_map<T>(Matrix{extra, M, N, N}, kBM) : to;
  }
  gemm<kEpiLinear, T>(a, A, a_mn, B, b_mn, cg, a.out_tma ? &tx : nullptr, a.out_tma ? &to : nullptr, s);
}

template <typename T>
void linear_forward(const T* x, const T* w, const T* bias, const T* residual, T* y, int64_t m, int k, int n, int act,
                    Carver& ws, bool run, cudaStream_t s)
{
  const Matrix X = addressable(x, m, k, ws, run, s), W = addressable(w, n, k, ws, run, s);
  if (!run) return;
  GemmArgs a;
  a.bias = bias;
  a.extra = residual;
  a.has_extra = residual != nullptr;
  a.out = y;
  a.ld_extra = a.ld_out = n;
  a.extra_tma = a.out_tma = n % 8 == 0;
  CUtensorMap tx{}, to{};
  if (a.out_tma) {
    to = matrix_map<T>(Matrix{y, m, n, n}, kBM);
    tx = residual ? matrix_map<T>(Matrix{residual, m, n, n}, kBM) : to;
  }
  const int cg = group_size(m, n);
  const CUtensorMap *px = a.out_tma ? &tx : nullptr, *po = a.out_tma ? &to : nullptr;
  if (act == RBQ_ACT_GELU)
    gemm<kEpiLinear, T, RBQ_ACT_GELU>(a, X, false, W, false, cg, px, po, s);
  else if (act == RBQ_ACT_RELU)
    gemm<kEpiLinear, T, RBQ_ACT_RELU>(a, X, false, W, false, cg, px, po, s);
  else
    gemm<kEpiLinear, T>(a, X, false, W, false, cg, px, po, s);
}

// dz = g * act'(x w^T + b) recomputes the layer's product: for the encoder's widths (k = 256) that
// reads and writes less than keeping z, and no rounding of z enters the gradient.  dz is rounded to
// the operands' 16 bits, as the operand of the two products dx = dz w and dw = dz^T x; the sums of
// all of them are fp32.
template <typename T>
void linear_backward(const T* g, const T* x, const T* w, const T* bias, T* dx, T* dw, T* dbias, int64_t m, int k, int n,
                     int act, Carver& ws, bool run, cudaStream_t s)
{
  const Matrix X = addressable(x, m, k, ws, run, s), W = addressable(w, n, k, ws, run, s);
  Matrix Z;
  const int cg = group_size(m, n);
  // With an activation the gradient kernel leaves 4 rows of n sums per CTA; without one dz is g, summed by a pass.
  const bool fused = act != RBQ_ACT_NONE;
  const int64_t tiles_m = ceil_div(m, kBM * cg), tiles_n = ceil_div(n, 128 * cg);
  const int ctas = (int)std::min<int64_t>(tiles_m * tiles_n, device_sm_count() / cg);
  const int gx = (int)ceil_div(n, kColGroup * 8);
  const int parts = fused ? ctas * cg * 4
                          : (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(m, 64), ceil_div(4 * device_sm_count(), gx)));
  float* part = ws.take<float>((int64_t)parts * n);
  if (act == RBQ_ACT_NONE) {
    Z = addressable(g, m, n, ws, run, s);
  } else {
    const int64_t ld = round_up(n, 8);
    Z = Matrix{ws.take<T>(m * ld), m, n, ld};
    if (run) {
      GemmArgs a;
      a.bias = bias;
      a.extra = g;
      a.has_extra = 1;
      a.ld_extra = n;
      a.extra_tma = n % 8 == 0;
      a.sums = fused && dbias ? part : nullptr;
      CUtensorMap tx{};
      if (a.extra_tma) tx = matrix_map<T>(Matrix{g, m, n, n}, kBM);
      const CUtensorMap to = matrix_map<T>(Z, kBM), *px = a.extra_tma ? &tx : nullptr, *po = &to;
      if (act == RBQ_ACT_GELU)
        gemm<kEpiActGrad, T, RBQ_ACT_GELU>(a, X, false, W, false, cg, px, po, s);
      else
        gemm<kEpiActGrad, T, RBQ_ACT_RELU>(a, X, false, W, false, cg, px, po, s);
    }
  }
  const SlabPlan plan = plan_slabs(n, k, m, false);
  float* slabs = ws.take<float>(plan.floats());
  if (!run) return;
  if (dx) store_gemm<T>(Z, false, W, true, group_size(m, k), nullptr, nullptr, dx, s);
  if (dw && plan.direct) store_gemm<T>(Z, true, X, true, plan.cg, nullptr, nullptr, dw, s);
  if (dw && !plan.direct) {
    slab_gemm<T>(plan, Z, true, X, true, slabs, false, s);
    add_slabs<T>(plan, slabs, false, n, k, 1.0f, nullptr, nullptr, dw, s);
  }
  if (dbias) {
    if (!fused) {
      column_sums_kernel<T><<<dim3(gx, parts), kColThreads, 0, s>>>(static_cast<const T*>(Z.p), m, n, Z.ld, part);
      RBQ_LAUNCHED();
    }
    add_parts_kernel<T><<<(unsigned)ceil_div(n, 32), 1024, 0, s>>>(part, parts, n, fused ? (int)tiles_m : 0, 128 * cg, ctas,
                                                                  4 * cg, dbias);
    RBQ_LAUNCHED();
  }
}

template <typename T>
void loss_forward(const T* q, const T* bank, const int64_t* target, int64_t n, int64_t v, int d, float scale, float* loss,
                  float* lse, Carver& ws, bool run, cudaStream_t s)
{
  const Matrix Q = addressable(q, n, d, ws, run, s), B = addressable(bank, v, d, ws, run, s);
  const int cg = group_size(n, v);
  // Runs of up to 16 tiles write one partial row each, but leave enough of them to even out over the SMs.
  const int64_t tiles_m = ceil_div(n, kBM * cg), tiles_n = ceil_div(v, 128 * cg);
  const int length = (int)std::max<int64_t>(1, std::min<int64_t>(16, tiles_m * tiles_n / (8 * (device_sm_count() / cg))));
  const int64_t tiles = 2 * cg * ceil_div(tiles_n, length);
  float2* partial = ws.take<float2>(tiles * n);
  if (!run) return;
  GemmArgs a;
  a.run = length;
  a.c2 = scale * kLog2e;
  a.target = target;
  a.partial = partial;
  gemm<kEpiLse, T>(a, Q, false, B, false, cg, nullptr, nullptr, s);
  loss_rows_kernel<T><<<(unsigned)ceil_div(n, 32), 1024, 0, s>>>(partial, (int)tiles, n, q, d, bank, d, d, v, target, scale,
                                                                 loss, lse);
  RBQ_LAUNCHED();
}

// The gradient of the logits exists one piece of the bank at a time, 16-bit values [n, piece] of at most
// kPieceBytes.  Pieces that stay in L2 (64 MB) cost more in short kernels than the traffic they save:
// 8,192 queries x 200,000 rows x 256, the three products of the backward pass and the adding: 2.71 ms in
// pieces of 256 MB, 2.49 of 512, 2.41 of 640, 2.42 of 1,024, 2.46 of 2,048 (3.6 of 64 with an earlier
// kernel).
constexpr int64_t kPieceBytes = 640ll << 20;
int64_t piece_columns(int64_t n, int64_t v)
{
  const int64_t most = std::max<int64_t>(1, kPieceBytes / (2 * n) / 256);  // in tiles of 256 columns
  // whole rounds of the SM pairs for the bank's gradient, where a piece holds one; the last piece is shorter
  const int64_t pairs = device_sm_count() / 2, whole = most >= pairs ? most / pairs * pairs : most;
  return std::min(whole, ceil_div(v, 256)) * 256;
}

template <typename T>
void loss_backward(const float* g, const T* q, const T* bank, const int64_t* target, const float* loss, const float* lse,
                   int64_t n, int64_t v, int d, float scale, T* dq, T* dbank, Carver& ws, bool run, cudaStream_t s)
{
  const int ldq = (int)round_up(d, 8);
  uint16_t* kept = ws.take<uint16_t>(n * ldq);
  T* rest = ws.take<T>(n * d);
  const Matrix Q{kept, n, d, ldq}, B = addressable(bank, v, d, ws, run, s);
  const int64_t piece = std::min(piece_columns(n, v), round_up(v, 8));
  float* top = ws.take<float>(3);
  float4* rows = ws.take<float4>(n);
  const int64_t ld = round_up(piece, 8);
  T* prob = ws.take<T>(n * ld);
  // The queries' gradient is summed over the pieces, in slabs that start from zero; the last piece may be
  // shorter than the others.
  const bool pieces = v > piece;
  const int64_t whole = std::min(piece, v), last = (v - 1) % piece + 1;
  SlabPlan pq = plan_slabs(n, d, whole, pieces), pq_last = plan_slabs(n, d, last, pieces);
  pq.slabs = pq_last.slabs = std::max(pq.slabs, pq_last.slabs);
  float* slabs_q = ws.take<float>(pq.floats());
  const SlabPlan pb = plan_slabs(whole, d, n, false), pb_last = plan_slabs(last, d, n, false);
  float* slabs_b = ws.take<float>(std::max(pb.floats(), pb_last.floats()));
  if (!run) return;
  grad_top_kernel<T><<<1, 1024, 0, s>>>(g, target, loss, n, v, scale, top);
  RBQ_LAUNCHED();
  grad_rows_kernel<T><<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(g, target, loss, lse, n, v, top, rows);
  RBQ_LAUNCHED();
  const RowBlocks l(n, ldq);
  loss_operands_kernel<T><<<l.blocks, l.block, 0, s>>>(q, bank, target, rows, top, n, d, ldq, kept, dq ? rest : nullptr);
  RBQ_LAUNCHED();
  if (dq && pieces) RBQ_CUDA(cudaMemsetAsync(slabs_q, 0, pq.floats() * sizeof(float), s));
  for (int64_t v0 = 0; v0 < v; v0 += piece) {
    const int64_t cols = std::min(piece, v - v0);
    const Matrix Bp{static_cast<const T*>(B.p) + v0 * B.ld, cols, d, B.ld};
    const Matrix P{prob, n, cols, ld};
    GemmArgs a;
    a.c2 = scale * kLog2e;
    a.col0 = v0;
    a.target = target;
    a.rows = rows;
    const CUtensorMap to = matrix_map<T>(P, kBM);
    gemm<kEpiProb, T>(a, Q, false, Bp, false, group_size(n, cols), nullptr, &to, s);
    const bool at_last = v0 + piece >= v;
    if (dq && pq.direct) store_gemm<T>(P, false, Bp, true, pq.cg, top + 1, rest, dq, s);
    if (dq && !pq.direct) slab_gemm<T>(at_last ? pq_last : pq, P, false, Bp, true, slabs_q, pieces, s);
    if (dbank) {
      const SlabPlan& p = at_last ? pb_last : pb;
      if (p.direct) {
        store_gemm<T>(P, true, Q, true, p.cg, top + 1, nullptr, dbank + v0 * d, s);
      } else {
        slab_gemm<T>(p, P, true, Q, true, slabs_b, false, s);
        add_slabs<T>(p, slabs_b, false, cols, d, 1.0f, top + 1, nullptr, dbank + v0 * d, s);
      }
    }
  }
  if (dq && !pq.direct) add_slabs<T>(pq, slabs_q, pieces, n, d, 1.0f, top + 1, rest, dq, s);
}

}  // namespace

// ---------------------------------------------------------------------------------------
// Launchers (arguments checked by the C ABI).  With ws == nullptr they launch nothing and return
// the workspace they need.
// ---------------------------------------------------------------------------------------
int64_t launch_linear(const void* x, const void* w, const void* bias, const void* residual, void* y, int64_t m, int k, int n,
                      int dtype, int act, void* ws, bool run, cudaStream_t s)
{
  Carver c(ws);
  if (dtype == RBQ_F16)
    linear_forward<__half>((const __half*)x, (const __half*)w, (const __half*)bias, (const __half*)residual, (__half*)y, m, k,
                           n, act, c, run, s);
  else
    linear_forward<__nv_bfloat16>((const __nv_bfloat16*)x, (const __nv_bfloat16*)w, (const __nv_bfloat16*)bias,
                                  (const __nv_bfloat16*)residual, (__nv_bfloat16*)y, m, k, n, act, c, run, s);
  return c.used;
}

int64_t launch_linear_backward(const void* g, const void* x, const void* w, const void* bias, void* dx, void* dw, void* dbias,
                               int64_t m, int k, int n, int dtype, int act, void* ws, bool run, cudaStream_t s)
{
  Carver c(ws);
  if (dtype == RBQ_F16)
    linear_backward<__half>((const __half*)g, (const __half*)x, (const __half*)w, (const __half*)bias, (__half*)dx,
                            (__half*)dw, (__half*)dbias, m, k, n, act, c, run, s);
  else
    linear_backward<__nv_bfloat16>((const __nv_bfloat16*)g, (const __nv_bfloat16*)x, (const __nv_bfloat16*)w,
                                   (const __nv_bfloat16*)bias, (__nv_bfloat16*)dx, (__nv_bfloat16*)dw,
                                   (__nv_bfloat16*)dbias, m, k, n, act, c, run, s);
  return c.used;
}

int64_t launch_softmax_loss(const void* q, const void* bank, const int64_t* target, int64_t n, int64_t v, int d, float scale,
                            int dtype, float* loss, float* lse, void* ws, bool run, cudaStream_t s)
{
  Carver c(ws);
  if (dtype == RBQ_F16)
    loss_forward<__half>((const __half*)q, (const __half*)bank, target, n, v, d, scale, loss, lse, c, run, s);
  else
    loss_forward<__nv_bfloat16>((const __nv_bfloat16*)q, (const __nv_bfloat16*)bank, target, n, v, d, scale, loss, lse, c,
                                run, s);
  return c.used;
}

int64_t launch_softmax_loss_backward(const float* g, const void* q, const void* bank, const int64_t* target,
                                     const float* loss, const float* lse, int64_t n, int64_t v, int d, float scale, int dtype,
                                     void* dq, void* dbank, void* ws, bool run, cudaStream_t s)
{
  Carver c(ws);
  if (dtype == RBQ_F16)
    loss_backward<__half>(g, (const __half*)q, (const __half*)bank, target, loss, lse, n, v, d, scale, (__half*)dq,
                          (__half*)dbank, c, run, s);
  else
    loss_backward<__nv_bfloat16>(g, (const __nv_bfloat16*)q, (const __nv_bfloat16*)bank, target, loss, lse, n, v, d, scale,
                                 (__nv_bfloat16*)dq, (__nv_bfloat16*)dbank, c, run, s);
  return c.used;
}

int take_op_error()
{
  int code = 0;
  RBQ_CUDA(cudaMemcpyFromSymbol(&code, g_op_err, sizeof(int)));
  if (code) {
    const int zero = 0;
    RBQ_CUDA(cudaMemcpyToSymbol(g_op_err, &zero, sizeof(int)));
  }
  return code;
}

}  // namespace rbq

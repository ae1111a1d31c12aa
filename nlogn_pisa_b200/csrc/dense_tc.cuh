// Building blocks shared by the tensor-core kernels of dense attention.
#pragma once

#include <type_traits>

#include "dense_attn.cuh"
#include "tc.cuh"

namespace pisa {

constexpr int kRows = 128;   // queries of a tile, keys of a tile

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
         "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
         "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(x0), "r"(x1), "r"(x2), "r"(x3) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// A CTA's waits: whether one of them has expired, and how many tries (of a
// microsecond each) any of them makes.
struct WaitFlag {
  int expired;
  uint32_t tries;
  __device__ __forceinline__ void init(uint32_t most = kWaitTries) {
    expired = 0;
    tries = most;
  }
};

// Waits for the phase with parity `phase & 1` of `bar`, flag->tries
// microseconds at most (tries that suspend a microsecond each).  An expired wait
// sets flag->expired and returns false, as does a wait of a CTA whose flag is set.  Warps with
// collective work do not leave their loops on a false result, which their
// lanes need not share: they go on, store NaN, and each further wait is short.
static __device__ __noinline__ bool wait_long(uint32_t addr, uint32_t parity, WaitFlag* flag) {
  const uint32_t tries = flag->tries;
#pragma unroll 1
  for (uint32_t i = 0; i < tries; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return true;
    if ((i & 255) == 255 && *static_cast<volatile int*>(&flag->expired)) return false;
  }
  *static_cast<volatile int*>(&flag->expired) = 1;
  return false;
}
__device__ __forceinline__ bool wait_phase(uint64_t* bar, int phase, WaitFlag* flag) {
  const uint32_t addr = tc::smem_u32(bar), parity = uint32_t(phase & 1);
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(addr), "r"(parity) : "memory");
  return done ? true : wait_long(addr, parity, flag);
}

// True in one lane of a converged warp.  The MMA warps run their control flow
// and waits as a whole and issue under this predicate: values then stay in the
// uniform registers that MMA operands come from.  (With one lane running the
// role alone, an MMA took about 110 cycles to issue.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Shared-memory operand descriptors as (low word: address and leading offset,
// high word: the rest); steps along K only change the low word.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);   // 8-row groups 1024 B apart, version 1, 128-byte swizzle

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      :: "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh) : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
      :: "r"(d), "r"(a), "r"(b_low), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh) : "memory");
}

// D = A B^T over DP dims of two K-major tiles of 128 rows in shared memory.
// (Loops over 64-dim chunks stay rolled here and below: the softmax warps sweep
// the instruction caches, and every line of the MMA warp's code is fetched
// again each step.)
template <int DP>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  uint32_t al = desc_low(a, 16), bl = desc_low(b, 16);
#pragma unroll 1
  for (int c = 0; c < DP / 64; ++c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) mma_ss(d, al + s * 2, bl + s * 2, idesc, c + s > 0);
    al += kRows * 128 / 16;
    bl += kRows * 128 / 16;
  }
}

// D (+)= A B over the first `steps` * 16 rows of the MN-major tile B; A in TMEM,
// 8 columns per step, the second four steps `gap` columns after the first.
__device__ __forceinline__ void mma_cols(uint32_t d, uint32_t a, uint32_t gap, uint32_t b, uint32_t idesc, int steps,
                                         bool accumulate) {
  uint32_t bl = desc_low(b, kRows * 128);
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (4 * c + s < steps) mma_ts(d, a + s * 8, bl + s * (16 * 128 / 16), idesc, accumulate || c + s > 0);
    a += gap;
    bl += 4 * (16 * 128 / 16);
  }
}

// (a * b) on two lanes at once
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Untiled bulk copy into shared memory: both addresses on 16 bytes, `bytes` a
// multiple of 16; completion counts on `mbar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(src), "r"(bytes), "r"(tc::smem_u32(mbar)) : "memory");
}

// Zero rows [first, last) of a [DP/64][128 rows][128 B] operand tile, one warp.
template <int DP>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first, int last, int lane) {
  for (int f = lane; f < (last - first) * DP / 8; f += 32) {
    const int r = first + f / (DP / 8), s = f % (DP / 8);
    st_shared16(tile + (s >> 3) * kRows * 128 + r * 128 + (s & 7) * 16, 0, 0, 0, 0);
  }
}

// This warp's 32 TMEM lanes x W columns, rounded to T, to the first `rows` rows
// of global memory (row r at out + r * stride, columns past `cols` dropped)
// through `stage` (32 * W * 2 bytes of shared memory of this warp).  With
// `empty` zeros are stored in their place.
template <typename T, int W>
__device__ __forceinline__ void store_lanes(uint32_t taddr, bool empty, float mul, uint32_t stage, T* out, int64_t stride,
                                            int rows, int cols, int lane) {
  constexpr int SEG = W / 8;
#pragma unroll
  for (int c = 0; c < W; c += 32) {
    float o[32];
    if (empty) {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0.f;
    } else {
      tc::tmem_ld32(taddr + c, o);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int seg = c / 8 + s;
      st_shared16(stage + (lane * SEG + (seg ^ (lane & (SEG - 1) & 7))) * 16, pack2<T>(o[8 * s] * mul, o[8 * s + 1] * mul),
                  pack2<T>(o[8 * s + 2] * mul, o[8 * s + 3] * mul), pack2<T>(o[8 * s + 4] * mul, o[8 * s + 5] * mul),
                  pack2<T>(o[8 * s + 6] * mul, o[8 * s + 7] * mul));
    }
  }
  __syncwarp();
  for (int f = lane; f < rows * SEG; f += 32) {
    const int r = f / SEG, seg = f % SEG;
    const uint4 v = ld_shared16(stage + (r * SEG + (seg ^ (r & (SEG - 1) & 7))) * 16);
    if (seg * 8 < cols) *reinterpret_cast<uint4*>(out + r * stride + seg * 8) = v;
  }
}

// Largest of 64 values by four chains of three-input maxima.
__device__ __forceinline__ float max_of(const float (&v)[64]) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = v[i];
#pragma unroll
  for (int i = 4; i < 60; i += 8) {
#pragma unroll
    for (int c = 0; c < 4; ++c) m[c] = tc::max3f(m[c], v[i + 2 * c], v[i + 2 * c + 1]);
  }
  return fmaxf(tc::max3f(m[0], v[60], v[61]), fmaxf(tc::max3f(m[1], v[62], v[63]), fmaxf(m[2], m[3])));
}

// Largest of two values, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair on the FMA and integer pipes, beside the special-function
// unit: x = j + f with |f| <= 1/2 by adding and taking away 1.5 * 2^23 + 127
// (the sum's low bits then are the exponent field of 2^j), 2^f by a polynomial
// of degree 4 fitted for least relative error on that range (iteratively
// reweighted least squares), 2.7e-6, against 2^-9 and 2^-12 of the rounding to
// bf16 or fp16 that follows.  For x <= 100; below -126 it stays at 2^-126, so
// hidden elements are set to zero afterwards.
__device__ __forceinline__ float2 ex2_pair(float2 x) {
  const float2 magic = make_float2(12583039.f, 12583039.f), minus = make_float2(-12583039.f, -12583039.f);
  x = make_float2(max_nan(x.x, -126.f), max_nan(x.y, -126.f));
  const float2 t = tc::add2(x, magic);
  const float2 f = tc::fma2(tc::add2(t, minus), make_float2(-1.f, -1.f), x);
  float2 p = tc::fma2(make_float2(0.009570105f, 0.009570105f), f, make_float2(0.05591787f, 0.05591787f));
  p = tc::fma2(p, f, make_float2(0.24024744f, 0.24024744f));
  p = tc::fma2(p, f, make_float2(0.6931218f, 0.6931218f));
  p = tc::fma2(p, f, make_float2(0.9999993f, 0.9999993f));
  return mul2(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}

// 2^x of pair number `i`: `poly` pairs of every eight by polynomial, spread out.
__device__ __forceinline__ float2 ex2_mixed(float2 x, int i, int poly) {
  const bool by_poly = (i % 8 + 1) * poly / 8 > (i % 8) * poly / 8;
  return by_poly ? ex2_pair(x) : make_float2(tc::ex2f(x.x), tc::ex2f(x.y));
}

constexpr float kRescale = 8.f;   // base-2 growth of a row maximum that moves it

// One tile of 128 scores of this thread's row (TMEM columns ts ..): updates the
// row's maximum m and weight sum l (base-2 logits), rescales O (DP columns at
// `to`) when the maximum moves, and leaves P, rounded to T, in the first 64
// columns of the scores' place.  Keys past `lim` are hidden.  The caller waits
// for the stores (tmem_wait_st) and hands P on.
template <typename T, int DP>
__device__ __forceinline__ void softmax_tile(uint32_t ts, uint32_t to, float sl, bool first, int lim, float& m, float& l) {
  uint32_t s0[64], s1[64];
  tc::tmem_ld64_nowait(ts, s0);
  tc::tmem_ld64_nowait(ts + 64, s1);
  tc::tmem_wait_ld2(s0, s1);
  float x0[64], x1[64];
#pragma unroll
  for (int c = 0; c < 64; ++c) {
    x0[c] = __uint_as_float(s0[c]);
    x1[c] = __uint_as_float(s1[c]);
  }
  if (lim < kRows - 1) {
#pragma unroll
    for (int c = 0; c < 64; ++c) {
      if (c > lim) x0[c] = -INFINITY;
      if (c + 64 > lim) x1[c] = -INFINITY;
    }
  }
  const float top = fmaxf(max_of(x0), max_of(x1)) * sl;
  if (first) {
    m = top;
  } else if (__any_sync(kFull, top > m + kRescale)) {
    const float next = fmaxf(m, top);
    const float alpha = next == -INFINITY ? 1.f : tc::ex2f(m - next);
    m = next;
    l *= alpha;
#pragma unroll
    for (int c = 0; c < DP; c += 16) {
      float o[16];
      uint32_t r[16];
      tc::tmem_ld16(to + c, o);
#pragma unroll
      for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(o[e] * alpha);
      tc::tmem_st16(to + c, r);
    }
  }
  const float ref = m == -INFINITY ? 0.f : m;
  const float2 k2 = make_float2(sl, sl), c2 = make_float2(-ref, -ref);
  uint32_t w[32];
  float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float2 p = tc::fma2(make_float2(x0[c], x0[c + 1]), k2, c2);
    p = make_float2(tc::ex2f(p.x), tc::ex2f(p.y));
    sum0 = tc::add2(sum0, p);
    w[c / 2] = pack2<T>(p.x, p.y);
  }
  tmem_st32(ts, w);
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float2 p = tc::fma2(make_float2(x1[c], x1[c + 1]), k2, c2);
    p = make_float2(tc::ex2f(p.x), tc::ex2f(p.y));
    sum1 = tc::add2(sum1, p);
    w[c / 2] = pack2<T>(p.x, p.y);
  }
  tmem_st32(ts + 32, w);
  l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
}

// OR of `mine` over `count` threads that meet at hardware barrier `id`.
__device__ __forceinline__ bool any_of(int id, int count, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbar.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "r"(uint32_t(mine)), "r"(id), "r"(count) : "memory");
  return r != 0;
}

// Half a tile's scores (64 keys) of this thread's row; another warp of the same
// quarter holds the row's other half.  As softmax_tile, with the halves'
// maxima exchanged through `other` (128 rows x 2) only when one of the tile's
// 256 threads needs a new maximum.  `ts`: TMEM of the half's scores, whose
// first 32 columns receive P; `to`: the half of O's columns that this thread
// rescales.  Keys past `lim` (of the half) are hidden.
template <typename T, int DP>
__device__ __forceinline__ void softmax_half(uint32_t ts, uint32_t to, float sl, bool first, int lim, int barrier,
                                             float (*other)[kRows], int half, int row, float& m, float& l) {
  float x[64];
  tc::tmem_ld64(ts, x);
  if (lim < 63) {
#pragma unroll
    for (int c = 0; c < 64; ++c)
      if (c > lim) x[c] = -INFINITY;
  }
  const float top = max_of(x) * sl;
  if (any_of(barrier, 256, first || top > m + kRescale)) {
    other[half][row] = top;
    tc::named_sync(barrier, 256);
    const float next = fmaxf(m, fmaxf(top, other[half ^ 1][row]));
    const float alpha = next == -INFINITY ? 1.f : tc::ex2f(m - next);
    m = next;
    if (!first) {
      l *= alpha;
#pragma unroll 1
      for (int c = 0; c < DP / 2; c += 16) {
        float o[16];
        uint32_t r[16];
        tc::tmem_ld16(to + c, o);
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(o[e] * alpha);
        tc::tmem_st16(to + c, r);
      }
    }
  }
  const float ref = m == -INFINITY ? 0.f : m;
  const float2 k2 = make_float2(sl, sl), c2 = make_float2(-ref, -ref);
  float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[16];
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      float2 p = tc::fma2(make_float2(x[32 * h + c], x[32 * h + c + 1]), k2, c2);
      float2 q = tc::fma2(make_float2(x[32 * h + c + 2], x[32 * h + c + 3]), k2, c2);
      p = make_float2(tc::ex2f(p.x), tc::ex2f(p.y));
      q = make_float2(tc::ex2f(q.x), tc::ex2f(q.y));
      sum0 = tc::add2(sum0, p);
      sum1 = tc::add2(sum1, q);
      w[c / 2] = pack2<T>(p.x, p.y);
      w[c / 2 + 1] = pack2<T>(q.x, q.y);
    }
    tmem_st16(ts + 16 * h, w);
  }
  l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
}

}  // namespace pisa

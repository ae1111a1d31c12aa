// The norms after one branch of a decoder block and before the next, fused
// with the branch's gate and the residual scale, and their gradient.
//
// For a row of D elements with rms(v) = sqrt(mean(v^2) + eps):
//   y' = y / rms(y) * p          (p: post weight; without it y' = y)
//   h  = a x + b g y'            (a, b: scales; g: gate, or 1)
//   n  = h / rms(h) * w.
// Backward, with v = h / rms(h), z = y / rms(y), from dh and dn:
//   dw = sum over rows of dn v,    t = dh + (dn w - v mean(dn w v)) / rms(h),
//   dx = a t,    dg = b t y'  (summed over the rows that share it),
//   s = b t g,   dp = sum of s z,   dy = (s p - z mean(s p z)) / rms(y)  (or s).
// Everything is held in fp32; each output is rounded once, the int8 form of n
// from its fp32 value.
//
// Bound by HBM: forward reads x and y (and a gate per token) and writes h and
// n, backward reads dh, dn, x, y and writes dx, dy.  The backward computes h
// again, as the forward had it before its rounding: the sums of dw and dp would
// carry the rounding of a stored h.  A team of threads holds its
// row in registers, so every operand is read once; the two row sums follow one
// another and other teams of the SM fill their waits.  Arithmetic is on pairs
// (f32x2): the backward, bound by instruction issue and barriers, went from 50 to
// 45 us with it.
//
// Measured, bf16: 32768 rows of 4096 forward 165 us (6.5 TB/s); 16384 rows of 1024,
// norms on both sides and a gate: forward 27 us (5.0 TB/s), backward 43 and 5 for
// the parameters (4.6 TB/s; issue slots 54 % busy, 16 warps per SM at 126
// registers; 5 or 6 CTAs per SM spill: 58 and 86 us); the second norm alone (no
// gate, no post weight) 19 and 37 us.  8192 rows of 4096 backward 100 us, the second
// norm alone 76 (one CTA of 512 threads per SM, which waits at its barrier).  Odd
// widths read elements one by one: 8193 rows of 1001 fp16 with a gate per token 25
// and 54 us (3.2 and 2.4 TB/s).  Their backward in fp32 spills 104 to 152 bytes per
// thread, that of aligned fp32 rows over 1024 elements 24, of 16-bit odd ones 8.
#include "rows.cuh"

namespace pisa {

namespace {

struct NormArgs {
  const void* x;
  int64_t x_st;
  const void* y;          // branch, or NULL: h = x
  int64_t y_st;
  const void* gate;       // or NULL
  int64_t gate_st;
  uint32_t gate_rows;     // consecutive rows that share a gate row, 0: each row has its own in the tensors' type
  const void* post;       // or NULL
  const void* w;
  int gate_f32, post_f32, w_f32;
  int64_t rows;
  int D;
  float a, b, eps, inv_d;
  void* h;
  void* n;                // or NULL with n_q
  int8_t* n_q;
  int64_t n_q_st;
  float* n_scale;
  float* stats;           // [rows][2]: 1 / rms of the branch and of h, or NULL
  // backward
  const void* dh;         // or NULL: zero
  const void* dn;
  void* dx;
  void* dy;
  void* dgate;
  float* partial;         // [teams][sums][D]
  float* means;           // wide rows: [rows][2]
  int combine;            // the teams of a CTA leave one partial
  int sums, sum_post, sum_gate;   // rows of a partial: weight 0, then post and gate where they are summed
  uint32_t share_rows, share_teams;   // rows of a share (one gate row's, or all), teams of a share
  uint32_t teams, cols;   // teams in all, CTAs of a gradient row
  void* dw;
  void* dpost;
};

template <typename T, int TPR, int NV, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1;
  __shared__ float red[TPR < 32 ? 1 : 2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x % TPR;
  int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TPR;
  const bool live = row < a.rows;
  // larger teams are CTAs with a row each; of smaller ones a warp without any row leaves, teams without one read and store nothing
  if (TPR < 32 ? !__any_sync(kFull, live) : !live) return;
  if (!live) row = 0;
  const int D = live ? a.D : 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_st;
  Raw8<T> x[NV], y[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) x[j] = load_piece<T, TPR, A>(xr, j, t, D);
  float h[NV][8];
  float inv_y = 1.f;
  if (a.y) {
    const T* yr = static_cast<const T*>(a.y) + row * a.y_st;
#pragma unroll
    for (int j = 0; j < NV; ++j) y[j] = load_piece<T, TPR, A>(yr, j, t, D);
    if (a.post) {
      float2 sum = both(0.f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[8];
        widen8<T>(y[j], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum = pair_fma(pair_at(f, k), pair_at(f, k), sum);
      }
      inv_y = rsqrtf(team_reduce<TPR, false>(sum.x + sum.y, red, set) * a.inv_d + a.eps);
    }
    const char* gr = static_cast<const char*>(a.gate);
    if (gr) gr += int64_t(a.gate_rows ? uint32_t(row) / a.gate_rows : uint32_t(row)) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T)));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[8], p[8];
      widen8<T>(x[j], h[j]);
      widen8<T>(y[j], f);
      if (a.post) {
        param_piece<T, TPR, A>(a.post, a.post_f32, j, t, D, p);
#pragma unroll
        for (int k = 0; k < 4; ++k) set_pair(f, k, pair_mul(pair_mul(pair_at(f, k), both(inv_y)), pair_at(p, k)));
      }
      if (gr) {
        param_piece<T, TPR, A>(gr, a.gate_f32, j, t, D, p);
#pragma unroll
        for (int k = 0; k < 4; ++k) set_pair(f, k, pair_mul(pair_at(f, k), pair_at(p, k)));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        set_pair(h[j], k, pair_fma(both(a.b), pair_at(f, k), pair_mul(both(a.a), pair_at(h[j], k))));
    }
    T* hr = static_cast<T*>(a.h) + row * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece<T, TPR, A>(hr, j, t, D, h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) widen8<T>(x[j], h[j]);
  }
  float2 sum = both(0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = pair_fma(pair_at(h[j], k), pair_at(h[j], k), sum);
  const float inv_h = rsqrtf(team_reduce<TPR, false>(sum.x + sum.y, red, set) * a.inv_d + a.eps);
  if (a.stats && t == 0 && live) {
    a.stats[2 * row] = inv_y;
    a.stats[2 * row + 1] = inv_h;
  }
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float w[8];
    param_piece<T, TPR, A>(a.w, a.w_f32, j, t, D, w);
#pragma unroll
    for (int k = 0; k < 4; ++k) set_pair(h[j], k, pair_mul(pair_mul(pair_at(h[j], k), both(inv_h)), pair_at(w, k)));
    if (a.n_q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = larger(top, fabsf(h[j][e]));
    }
  }
  if (a.n_q) {
    // places past the row's end hold 0 * inv_h * 0: NaN where eps is 0 and the row is, as its values are
    top = team_reduce<TPR, true>(top, red, set);
    const Scale8 s(top);
    int8_t* qr = a.n_q + row * a.n_q_st;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece_s8<T, TPR, A>(qr, j, t, D, h[j], top < INFINITY, s.inv);
    if (t == 0 && live) a.n_scale[row] = s.scale;
  } else {
    T* nr = static_cast<T*>(a.n) + row * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece<T, TPR, A>(nr, j, t, D, h[j]);
  }
}

// The backward for wider rows in two passes: the two means of every row, and
// then columns, of which a thread keeps 8 over many rows without a barrier.  It
// reads the operands twice; one pass with the parameters' sums in shared memory
// took 275 us for 4096 rows of 8192 (bf16), these two take 64 and 82.
// Means of a row: of dn w v, and of s p z (as in norm_bwd_row_kernel).
constexpr int kWideThreads = 256, kSlab = 1024;   // columns of a CTA of the second pass

template <typename T, bool A>
__global__ void __launch_bounds__(kWideThreads) norm_means_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TPR = kWideThreads, STEP = TPR * 8;
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x, D = a.D;
  const int64_t row = blockIdx.x;
  const float2 stats = reinterpret_cast<const float2*>(a.stats)[row];
  const char* gr = static_cast<const char*>(a.gate);
  if (gr) gr += int64_t(a.gate_rows ? uint32_t(row) / a.gate_rows : uint32_t(row)) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T)));
  const int w_size = a.w_f32 ? 4 : int(sizeof(T)), p_size = a.post_f32 ? 4 : int(sizeof(T)), g_size = a.gate_f32 ? 4 : int(sizeof(T));
  float sum1 = 0.f, sum2 = 0.f, sum3 = 0.f;
#pragma unroll 2
  for (int c = 0; c < D; c += STEP) {
    const int width = min(STEP, D - c);
    float v[8], s[8], f[8], q[8];
    widen8<T>(load_piece<T, TPR, A>(static_cast<const T*>(a.x) + row * a.x_st + c, 0, t, width), v);
    widen8<T>(load_piece<T, TPR, A>(static_cast<const T*>(a.dn) + row * D + c, 0, t, width), s);
    param_piece<T, TPR, A>(static_cast<const char*>(a.w) + int64_t(c) * w_size, a.w_f32, 0, t, width, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= a.a;
      s[e] *= f[e];
      q[e] = 0.f;
    }
    if (a.y) {
      widen8<T>(load_piece<T, TPR, A>(static_cast<const T*>(a.y) + row * a.y_st + c, 0, t, width), q);
      if (a.post) {
        param_piece<T, TPR, A>(static_cast<const char*>(a.post) + int64_t(c) * p_size, a.post_f32, 0, t, width, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] *= stats.x * f[e];
      }
      if (gr) {
        param_piece<T, TPR, A>(gr + int64_t(c) * g_size, a.gate_f32, 0, t, width, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] *= f[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] *= a.b;
        v[e] += q[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= stats.y;
      sum1 = fmaf(s[e], v[e], sum1);
    }
    if (a.post) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
      if (a.dh) widen8<T>(load_piece<T, TPR, A>(static_cast<const T*>(a.dh) + row * D + c, 0, t, width), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum2 = fmaf(q[e], fmaf(stats.y, s[e], f[e]), sum2);
        sum3 = fmaf(q[e], v[e], sum3);
      }
    }
  }
  sum1 = team_reduce<TPR, false>(sum1, red, set);
  const float mean = sum1 * a.inv_d;
  float mean_y = 0.f;
  if (a.post) {
    sum2 = team_reduce<TPR, false>(sum2, red, set);
    sum3 = team_reduce<TPR, false>(sum3, red, set);
    mean_y = fmaf(-mean * stats.y, sum3, sum2) * a.inv_d;
  }
  if (t == 0) reinterpret_cast<float2*>(a.means)[row] = make_float2(mean, mean_y);
}

template <typename T, bool A>
__global__ void __launch_bounds__(128) norm_columns_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TPR = 128;
  const int t = threadIdx.x, D = a.D;
  const uint32_t slabs = uint32_t((D + kSlab - 1) / kSlab), team = blockIdx.x / slabs;
  const int c0 = int(blockIdx.x - team * slabs) * kSlab, width = min(kSlab, D - c0);
  const uint32_t share = team / a.share_teams, first = team - share * a.share_teams;
  const int64_t begin = int64_t(share) * a.share_rows;
  const bool token_gate = a.gate && !a.gate_rows;
  const char* gr = static_cast<const char*>(a.gate);
  const int g_size = a.gate_f32 ? 4 : int(sizeof(T));
  float w[8], p[8], g[8], dw[8], dp[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = dp[e] = dg[e] = 0.f, p[e] = g[e] = 1.f;
  param_piece<T, TPR, A>(static_cast<const char*>(a.w) + int64_t(c0) * (a.w_f32 ? 4 : int(sizeof(T))), a.w_f32, 0, t, width, w);
  if (a.post)
    param_piece<T, TPR, A>(static_cast<const char*>(a.post) + int64_t(c0) * (a.post_f32 ? 4 : int(sizeof(T))), a.post_f32, 0, t, width, p);
  if (gr && !token_gate)
    param_piece<T, TPR, A>(gr + (int64_t(uint32_t(begin) / a.gate_rows) * a.gate_st + c0) * g_size, a.gate_f32, 0, t, width, g);
  Raw8<T> x, y, dn, dh, gt;
  float2 stats, means;
  auto fetch = [&](int64_t row) {
    x = load_piece<T, TPR, A>(static_cast<const T*>(a.x) + row * a.x_st + c0, 0, t, width);
    dn = load_piece<T, TPR, A>(static_cast<const T*>(a.dn) + row * D + c0, 0, t, width);
    if (a.dh) dh = load_piece<T, TPR, A>(static_cast<const T*>(a.dh) + row * D + c0, 0, t, width);
    if (a.y) y = load_piece<T, TPR, A>(static_cast<const T*>(a.y) + row * a.y_st + c0, 0, t, width);
    if (token_gate) gt = load_piece<T, TPR, A>(reinterpret_cast<const T*>(gr) + row * a.gate_st + c0, 0, t, width);
    stats = reinterpret_cast<const float2*>(a.stats)[row];
    means = reinterpret_cast<const float2*>(a.means)[row];
  };
  fetch(begin + first);
  for (int64_t i = first; i < a.share_rows; i += a.share_teams) {
    const int64_t row = begin + i;
    float z[8], v[8], s[8], d[8];
    widen8<T>(x, v);
    widen8<T>(dn, s);
    if (a.dh) {
      widen8<T>(dh, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = 0.f;
    }
    if (a.y) widen8<T>(y, z);
    if (token_gate) widen8<T>(gt, g);
    const float2 st = stats, m = means;
    if (i + a.share_teams < a.share_rows) fetch(row + a.share_teams);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= a.a;
      if (a.y) {
        if (a.post) z[e] *= st.x;
        v[e] = fmaf(a.b * g[e], z[e] * p[e], v[e]);
      }
      v[e] *= st.y;
      dw[e] = fmaf(s[e], v[e], dw[e]);
      s[e] = fmaf(fmaf(-v[e], m.x, s[e] * w[e]), st.y, d[e]);
      d[e] = a.a * s[e];
      s[e] *= a.b;
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dx) + row * D + c0, 0, t, width, d);
    if (!a.y) continue;
    if (gr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d[e] = s[e] * (z[e] * p[e]);
        dg[e] += d[e];
        s[e] *= g[e];
      }
      if (token_gate) store_piece<T, TPR, A>(static_cast<T*>(a.dgate) + row * D + c0, 0, t, width, d);
    }
    if (a.post) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dp[e] = fmaf(s[e], z[e], dp[e]);
        s[e] = fmaf(-z[e], m.y, s[e] * p[e]) * st.x;
      }
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dy) + row * D + c0, 0, t, width, s);
  }
  float* out = a.partial + int64_t(team) * a.sums * D + c0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = column<T, TPR, A>(0, e, t);
    if (c < width) {
      out[c] = dw[e];
      if (a.sum_post) out[a.sum_post * int64_t(D) + c] = dp[e];
      if (a.sum_gate) out[a.sum_gate * int64_t(D) + c] = dg[e];
    }
  }
}

// The backward for rows that a team holds with 8 elements per thread.  A team
// keeps the parameters and their running sums in registers, and the next rows'
// operands are on their way while it works on one: aligned rows through a ring
// in shared memory, of which each thread fills and reads its own columns, others
// through registers.  One barrier per row: the second norm's sum follows from
// three that need no other,
//   mean(s p z) with s = b g t  is  S2 - mean(dn w v) / rms(h) S3,
//   S2 = mean(q (dh + dn w / rms(h))), S3 = mean(q v), q = b g p z.
template <typename T, int TPR>
struct Ring {
  static constexpr int THREADS = TPR < 128 ? 128 : TPR, PIECES = sizeof(T) / 2;      // 16-byte pieces of 8 elements
  static constexpr int ROWS = sizeof(T) == 2 ? 4 : THREADS < 512 ? 3 : 2;            // rows in flight or in use
  static int bytes(bool token_gate) { return ROWS * THREADS * (16 * PIECES * (token_gate ? 5 : 4) + 8); }
  uint32_t base, tensors;
  __device__ __forceinline__ uint32_t at(int slot, int k) const { return base + ((slot * tensors + k) * PIECES * THREADS + threadIdx.x) * 16; }
  __device__ __forceinline__ uint32_t stats(int slot) const {
    return base + ROWS * tensors * PIECES * THREADS * 16 + (slot * THREADS + threadIdx.x) * 8;
  }
  __device__ __forceinline__ void fill(int slot, int k, const T* row, int t, int D) const {
    // columns past the row's end are zeros: nothing is read
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = column<T, TPR, true>(0, 4 * i, t);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(at(slot, k) + i * THREADS * 16),
                   "l"(row + (c < D ? c : 0)), "r"(c < D ? 16 : 0) : "memory");
    }
  }
  __device__ __forceinline__ Raw8<T> take(int slot, int k) const {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.v[i].x), "=r"(r.v[i].y), "=r"(r.v[i].z), "=r"(r.v[i].w)
                   : "r"(at(slot, k) + i * THREADS * 16) : "memory");
    return r;
  }
};

template <typename T, int TPR, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR <= 128 ? 4 : TPR == 256 ? 2 : 1)
norm_bwd_row_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1, W = TPR / 32;
  using R = Ring<T, TPR>;
  extern __shared__ __align__(16) uint8_t ring_bytes[];
  __shared__ __align__(16) float red[2][W > 1 ? 4 * W : 4];
  int set = 0;
  const int t = threadIdx.x % TPR, D = a.D;
  const uint32_t team = blockIdx.x * TEAMS + threadIdx.x / TPR;
  const uint32_t share = team / a.share_teams, first = team - share * a.share_teams;
  const int64_t begin = int64_t(share) * a.share_rows;
  // teams of a warp or less that come after the last have no rows
  const int64_t end = begin < a.rows ? int64_t(a.share_rows) : 0;
  const bool token_gate = a.gate && !a.gate_rows;
  const char* gr = static_cast<const char*>(a.gate);
  float w[8], p[8], g[8], dw[8], dp[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = dp[e] = dg[e] = 0.f, p[e] = g[e] = 1.f;
  param_piece<T, TPR, A>(a.w, a.w_f32, 0, t, D, w);
  if (a.post) param_piece<T, TPR, A>(a.post, a.post_f32, 0, t, D, p);
  // the rows of a share have one gate row
  if (gr && !token_gate && end)
    param_piece<T, TPR, A>(gr + int64_t(uint32_t(begin) / a.gate_rows) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T))), a.gate_f32, 0, t,
                           D, g);
  struct Row {
    Raw8<T> x, y, dn, dh, g;
    float inv_y, inv_h;
  };
  Row next;
  const R ring{uint32_t(__cvta_generic_to_shared(ring_bytes)), token_gate ? 5u : 4u};
  const T* xs = static_cast<const T*>(a.x);
  const T* ys = static_cast<const T*>(a.y);
  const T* gs = reinterpret_cast<const T*>(gr);
  const T* dns = static_cast<const T*>(a.dn);
  const T* dhs = static_cast<const T*>(a.dh);
  auto fetch = [&](int64_t row, int slot) {
    if constexpr (A) {
      ring.fill(slot, 0, xs + row * a.x_st, t, D);
      ring.fill(slot, 1, dns + row * D, t, D);
      if (dhs) ring.fill(slot, 2, dhs + row * D, t, D);
      if (ys) ring.fill(slot, 3, ys + row * a.y_st, t, D);
      if (token_gate) ring.fill(slot, 4, gs + row * a.gate_st, t, D);
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(ring.stats(slot)), "l"(a.stats + 2 * row) : "memory");
    } else {
      next.x = load_piece<T, TPR, A>(xs + row * a.x_st, 0, t, D);
      next.dn = load_piece<T, TPR, A>(dns + row * D, 0, t, D);
      if (dhs) next.dh = load_piece<T, TPR, A>(dhs + row * D, 0, t, D);
      if (ys) next.y = load_piece<T, TPR, A>(ys + row * a.y_st, 0, t, D);
      if (token_gate) next.g = load_piece<T, TPR, A>(gs + row * a.gate_st, 0, t, D);
      next.inv_y = a.stats[2 * row];
      next.inv_h = a.stats[2 * row + 1];
    }
  };
  int slot = 0;
  if constexpr (A) {
#pragma unroll
    for (int i = 0; i < R::ROWS - 1; ++i) {
      const int64_t at = int64_t(first) + int64_t(i) * a.share_teams;
      if (at < end) fetch(begin + at, i);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  } else if (first < end) {
    fetch(begin + first, 0);
  }
  const float2 scale_a = both(a.a), scale_b = both(a.b);
  // teams of a warp take as many turns, so that its shuffles meet
  const int64_t turns = TPR < 32 ? (int64_t(a.share_rows) + a.share_teams - 1) / a.share_teams : 0;
  int64_t turn = 0;
  for (int64_t i = first; TPR < 32 ? turn < turns : i < end; i += a.share_teams, ++turn) {
    const bool live = TPR >= 32 || i < end;
    const int64_t row = live ? begin + i : 0;
    Row r;
    if constexpr (A) {
      // the slot of the row before: its values are in use no more
      const int64_t ahead = i + int64_t(R::ROWS - 1) * a.share_teams;
      if (ahead < end) fetch(begin + ahead, slot ? slot - 1 : R::ROWS - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group %0;" :: "n"(R::ROWS - 1) : "memory");
      r.x = ring.take(slot, 0);
      r.dn = ring.take(slot, 1);
      if (dhs) r.dh = ring.take(slot, 2);
      if (ys) r.y = ring.take(slot, 3);
      if (token_gate) r.g = ring.take(slot, 4);
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r.inv_y), "=f"(r.inv_h) : "r"(ring.stats(slot)) : "memory");
      if (++slot == R::ROWS) slot = 0;
    } else {
      r = next;
      if (i + a.share_teams < end) fetch(row + a.share_teams, 0);
    }
    if (!live) {   // all zeros: nothing is added
#pragma unroll
      for (int k = 0; k < int(sizeof(T) / 2); ++k) r.x.v[k] = r.dn.v[k] = r.dh.v[k] = r.y.v[k] = r.g.v[k] = make_uint4(0, 0, 0, 0);
      r.inv_y = r.inv_h = 0.f;
    }
    float z[8], v[8], s[8], d[8];
    float2 sum1 = both(0.f), sum2 = both(0.f), sum3 = both(0.f);
    widen8<T>(r.x, v);
    widen8<T>(r.dn, s);
    if (dhs) {
      widen8<T>(r.dh, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = 0.f;
    }
    if (token_gate) widen8<T>(r.g, g);
    if (ys) widen8<T>(r.y, z);
    const float2 inv_h = both(r.inv_h);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 hv = pair_mul(scale_a, pair_at(v, k)), q = both(0.f);
      if (ys) {
        float2 zz = pair_at(z, k);
        if (a.post) {
          zz = pair_mul(zz, both(r.inv_y));
          set_pair(z, k, zz);
        }
        q = pair_mul(scale_b, pair_mul(pair_at(g, k), pair_mul(zz, pair_at(p, k))));
        hv = pair_add(hv, q);
      }
      hv = pair_mul(hv, inv_h);
      const float2 n = pair_at(s, k), sw = pair_mul(n, pair_at(w, k));
      set_pair(dw, k, pair_fma(n, hv, pair_at(dw, k)));
      sum1 = pair_fma(sw, hv, sum1);
      if (a.post) {
        sum2 = pair_fma(q, pair_fma(inv_h, sw, pair_at(d, k)), sum2);
        sum3 = pair_fma(q, hv, sum3);
      }
      set_pair(v, k, hv);
      set_pair(s, k, sw);
    }
    float sums[3] = {sum1.x + sum1.y, sum2.x + sum2.y, sum3.x + sum3.y};
    if constexpr (TPR < 32 || (TPR > 128 && sizeof(T) == 2)) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (k && !a.post) break;
#pragma unroll
        for (int o = TPR < 32 ? TPR / 2 : 16; o > 0; o >>= 1) sums[k] += __shfl_xor_sync(kFull, sums[k], o);
      }
      if constexpr (W > 1) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
          for (int k = 0; k < 3; ++k) red[set][k * W + (threadIdx.x >> 5)] = sums[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          if (k && !a.post) break;
          sums[k] = red[set][k * W];
#pragma unroll
          for (int x = 1; x < W; ++x) sums[k] += red[set][k * W + x];
        }
        set ^= 1;
      }
    } else {
      // Three sums in six shuffles: halves of the warp carry different ones on (16384 x 1024 43 us, 45 with fifteen;
      // 16-bit teams of 256 and 512 threads have no registers left for it: 54 and 112 us against 48 and 100).
      const bool hi = threadIdx.x & 16, mid = threadIdx.x & 8;
      float u = hi ? sums[1] : sums[0], v1 = hi ? sums[0] : sums[1];
      u += __shfl_xor_sync(kFull, v1, 16);                                  // lanes 0-15: sum 0, 16-31: sum 1
      const float third = sums[2] + __shfl_xor_sync(kFull, sums[2], 16);
      float k = mid ? third : u;
      k += __shfl_xor_sync(kFull, mid ? u : third, 8);                      // lanes 0-7: sum 0, 16-23: sum 1, 8-15 and 24-31: sum 2
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) k += __shfl_xor_sync(kFull, k, o);
      if constexpr (W > 1) {
        if ((threadIdx.x & 7) == 0 && (threadIdx.x & 24) != 24) red[set][4 * (threadIdx.x >> 5) + ((threadIdx.x & 8) ? 2 : (threadIdx.x & 16) >> 4)] = k;
        __syncthreads();
        float4 all = *reinterpret_cast<const float4*>(&red[set][0]);
#pragma unroll
        for (int x = 1; x < W; ++x) {
          const float4 more = *reinterpret_cast<const float4*>(&red[set][4 * x]);
          all.x += more.x;
          all.y += more.y;
          all.z += more.z;
        }
        sums[0] = all.x;
        sums[1] = all.y;
        sums[2] = all.z;
        set ^= 1;
      } else {
        sums[0] = __shfl_sync(kFull, k, 0);
        sums[1] = __shfl_sync(kFull, k, 16);
        sums[2] = __shfl_sync(kFull, k, 8);
      }
    }
    const float mean = sums[0] * a.inv_d, mean_y = fmaf(-mean * inv_h.x, sums[2], sums[1]) * a.inv_d;
    const int width = live ? D : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = pair_fma(pair_fma(pair_at(v, k), both(-mean), pair_at(s, k)), inv_h, pair_at(d, k));
      set_pair(d, k, pair_mul(scale_a, x));
      set_pair(s, k, pair_mul(scale_b, x));
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dx) + row * D, 0, t, width, d);
    if (!ys) continue;
    if (gr) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = pair_mul(pair_at(s, k), pair_mul(pair_at(z, k), pair_at(p, k)));
        set_pair(d, k, x);
        set_pair(dg, k, pair_add(pair_at(dg, k), x));
        set_pair(s, k, pair_mul(pair_at(s, k), pair_at(g, k)));
      }
      if (token_gate) store_piece<T, TPR, A>(static_cast<T*>(a.dgate) + row * D, 0, t, width, d);
    }
    if (a.post) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 zz = pair_at(z, k), x = pair_at(s, k);
        set_pair(dp, k, pair_fma(x, zz, pair_at(dp, k)));
        set_pair(s, k, pair_mul(pair_fma(zz, both(-mean_y), pair_mul(x, pair_at(p, k))), both(r.inv_y)));
      }
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dy) + row * D, 0, t, width, s);
  }
  if (TEAMS > 1 && a.combine) {
    // all teams serve the same rows' sums: one partial per CTA, added in the order of the teams
    float* buf = reinterpret_cast<float*>(ring_bytes);     // [TEAMS][sums][D]
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* mine = buf + int(threadIdx.x / TPR) * a.sums * D;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<T, TPR, A>(0, e, t);
      if (c < D) {
        mine[c] = dw[e];
        if (a.sum_post) mine[a.sum_post * D + c] = dp[e];
        if (a.sum_gate) mine[a.sum_gate * D + c] = dg[e];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.sums * D; c += R::THREADS) {
      float v = buf[c];
#pragma unroll
      for (int k = 1; k < TEAMS; ++k) v += buf[k * a.sums * D + c];
      a.partial[int64_t(blockIdx.x) * a.sums * D + c] = v;
    }
    return;
  }
  if (!end) return;
  float* out = a.partial + int64_t(team) * a.sums * D;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = column<T, TPR, A>(0, e, t);
    if (c < D) {
      out[c] = dw[e];
      if (a.sum_post) out[a.sum_post * int64_t(D) + c] = dp[e];
      if (a.sum_gate) out[a.sum_gate * int64_t(D) + c] = dg[e];
    }
  }
}

// The parameters' gradients from the teams' partials, added in a fixed order:
// 32 columns of one gradient row per CTA, a warp for every 32nd partial.  The
// rows: dw and dp over all teams, then dg of every share over its own.
template <typename T>
__global__ void __launch_bounds__(1024) norm_sum_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t r = blockIdx.x / a.cols;
  const int c = (blockIdx.x - r * a.cols) * 32 + lane;
  const uint32_t whole = a.sum_post ? 2 : 1;      // rows that all teams share
  const bool is_gate = r >= whole;
  const uint32_t count = is_gate ? a.share_teams : a.teams;
  const int64_t from = is_gate ? int64_t(r - whole) * a.share_teams : 0, stride = int64_t(a.sums) * a.D;
  float v = 0.f;
  if (c < a.D) {
    const float* at = a.partial + from * stride + (is_gate ? a.sum_gate : r ? a.sum_post : 0) * int64_t(a.D) + c;
#pragma unroll 8
    for (uint32_t p = warp; p < count; p += 32) v += at[p * stride];
  }
  buf[warp][lane] = v;
  __syncthreads();
  if (warp || c >= a.D) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) v += buf[i][lane];
  const int64_t at = (is_gate ? int64_t(r - whole) * a.D : 0) + c;
  void* out = is_gate ? a.dgate : r ? a.dpost : a.dw;
  if (is_gate ? a.gate_f32 : r ? a.post_f32 : a.w_f32) static_cast<float*>(out)[at] = v;
  else static_cast<T*>(out)[at] = from_f32<T>(v);
}

constexpr int64_t kMaxWidth = 16384;

template <typename T, int TPR, int NV>
int launch_fwd(const NormArgs& a, bool aligned, cudaStream_t s) {
  constexpr int threads = TPR < 128 ? 128 : TPR, teams = threads / TPR;
  const unsigned ctas = unsigned((a.rows + teams - 1) / teams);
  if (aligned) norm_fwd_kernel<T, TPR, NV, true><<<ctas, threads, 0, s>>>(a);
  else norm_fwd_kernel<T, TPR, NV, false><<<ctas, threads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int fwd(const NormArgs& a, bool aligned, cudaStream_t s) {
  if (a.D <= 64) return launch_fwd<T, 8, 1>(a, aligned, s);
  if (a.D <= 128) return launch_fwd<T, 16, 1>(a, aligned, s);
  if (a.D <= 256) return launch_fwd<T, 32, 1>(a, aligned, s);
  if (a.rows <= 2 * sm_count()) {
    // few rows: more threads each, whose chain of loads, sums and stores is shorter (64 x 4096: 4.3 us, with 128 threads 8.2)
    if (a.D <= 1024) return launch_fwd<T, 128, 1>(a, aligned, s);
    if (a.D <= 4096) return launch_fwd<T, 512, 1>(a, aligned, s);
    return launch_fwd<T, 1024, 2>(a, aligned, s);
  }
  if (a.D <= 512) return launch_fwd<T, 32, 2>(a, aligned, s);
  if (a.D <= 1024) return launch_fwd<T, 32, 4>(a, aligned, s);
  if (a.D <= 2048) return launch_fwd<T, 128, 2>(a, aligned, s);
  if (a.D <= 4096) return launch_fwd<T, 128, 4>(a, aligned, s);
  if (a.D <= 8192) return launch_fwd<T, 512, 2>(a, aligned, s);
  return launch_fwd<T, 1024, 2>(a, aligned, s);
}

// Teams of the backward by width: their threads, CTAs, and the partials that they leave.
struct Plan {
  int teams_per_cta, combine;
  uint32_t share_rows, share_teams;
  int64_t shares, teams, ctas, partials, means_bytes;
};

Plan make_plan(int64_t rows, int64_t D, int64_t share_rows) {
  Plan p{};
  const int tpr = D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 128;
  p.teams_per_cta = tpr < 128 ? 128 / tpr : 1;
  const int64_t slabs = D <= 4096 ? 1 : (D + kSlab - 1) / kSlab, sms = sm_count();
  const int64_t most = D <= 1024 ? sms * 4 * p.teams_per_cta : D <= 2048 ? sms * 2 : D <= 4096 ? sms : (4 * sms + slabs - 1) / slabs;
  p.share_rows = uint32_t(share_rows);
  p.shares = rows / share_rows;
  const int64_t each = most / p.shares;
  p.share_teams = uint32_t(each < 1 ? 1 : each < share_rows ? each : share_rows);
  p.teams = p.shares * p.share_teams;
  p.ctas = (p.teams + p.teams_per_cta - 1) / p.teams_per_cta * slabs;
  p.combine = p.shares == 1 && p.teams_per_cta > 1;
  p.partials = p.combine ? p.ctas : p.teams;
  p.means_bytes = D <= 4096 ? 0 : (rows * 8 + 255) / 256 * 256;
  return p;
}

template <typename T, int TPR>
int launch_bwd_row(const NormArgs& a, const Plan& p, bool aligned, cudaStream_t s) {
  constexpr int threads = TPR < 128 ? 128 : TPR;
  if (aligned) {
    const int smem = Ring<T, TPR>::bytes(a.gate && !a.gate_rows);   // holds the teams' sums in the end: 12 KB at most
    if (int rc = allow_smem<norm_bwd_row_kernel<T, TPR, true>>(Ring<T, TPR>::bytes(true), "norm backward smem attribute")) return rc;
    norm_bwd_row_kernel<T, TPR, true><<<unsigned(p.ctas), threads, smem, s>>>(a);
  } else {
    const int smem = a.combine ? int(sizeof(float)) * 3 * 8 * threads : 0;
    norm_bwd_row_kernel<T, TPR, false><<<unsigned(p.ctas), threads, smem, s>>>(a);
  }
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int launch_bwd_wide(const NormArgs& a, const Plan& p, bool aligned, cudaStream_t s) {
  if (aligned) norm_means_kernel<T, true><<<unsigned(a.rows), kWideThreads, 0, s>>>(a);
  else norm_means_kernel<T, false><<<unsigned(a.rows), kWideThreads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  if (aligned) norm_columns_kernel<T, true><<<unsigned(p.ctas), 128, 0, s>>>(a);
  else norm_columns_kernel<T, false><<<unsigned(p.ctas), 128, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int bwd(NormArgs a, const Plan& p, bool aligned, cudaStream_t s) {
  int rc;
  if (a.D <= 64) rc = launch_bwd_row<T, 8>(a, p, aligned, s);
  else if (a.D <= 128) rc = launch_bwd_row<T, 16>(a, p, aligned, s);
  else if (a.D <= 256) rc = launch_bwd_row<T, 32>(a, p, aligned, s);
  else if (a.D <= 1024) rc = launch_bwd_row<T, 128>(a, p, aligned, s);
  else if (a.D <= 2048) rc = launch_bwd_row<T, 256>(a, p, aligned, s);
  else if (a.D <= 4096) rc = launch_bwd_row<T, 512>(a, p, aligned, s);
  else rc = launch_bwd_wide<T>(a, p, aligned, s);
  if (rc) return rc;
  a.teams = uint32_t(p.partials);
  a.cols = uint32_t((a.D + 31) / 32);
  const int64_t rows = 1 + (a.sum_post ? 1 : 0) + (a.sum_gate ? p.shares : 0);
  if (p.combine) a.share_teams = a.teams;
  norm_sum_kernel<T><<<unsigned(a.cols * rows), 1024, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

int check(const void* x, int64_t x_st, const void* y, const void* gate, int64_t gate_rows, int gate_dtype, const void* post,
          int post_dtype, const void* w, int w_dtype, int dtype, int64_t rows, int64_t D, float a, float b, float eps) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if ((w_dtype != dtype && w_dtype != PISA_F32) || (post && post_dtype != dtype && post_dtype != PISA_F32))
    return fail(PISA_ERR_UNSUPPORTED, "norm weights must be FP32 or the tensors' type");
  if (rows <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (D > kMaxWidth) return fail(PISA_ERR_UNSUPPORTED, "rows of more than 16384 elements are not supported");
  if (rows >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (!(eps >= 0.f) || std::isinf(eps)) return fail(PISA_ERR_INVALID, "eps must be finite and not negative");
  if (!std::isfinite(a) || !std::isfinite(b)) return fail(PISA_ERR_INVALID, "scales must be finite");
  if (!x || !w) return fail(PISA_ERR_INVALID, "x and weight are required");
  if (!y && (gate || post)) return fail(PISA_ERR_INVALID, "a gate and a post weight belong to a branch");
  if (gate) {
    if (gate_dtype != dtype && (gate_dtype != PISA_F32 || gate_rows == 0))
      return fail(PISA_ERR_UNSUPPORTED, "the gate must have the tensors' type, or FP32 where rows share it");
    if (gate_rows < 0 || gate_rows > rows || (gate_rows && rows % gate_rows))
      return fail(PISA_ERR_INVALID, "gate rows must divide the rows");
    if (gate_rows && (rows / gate_rows + 2) * ((D + 31) / 32) >= (int64_t(1) << 31))
      return fail(PISA_ERR_UNSUPPORTED, "too many gate rows");
  }
  return PISA_OK;
}

bool param_on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

}  // namespace pisa

extern "C" {

int pisa_residual_norm(const void* x, int64_t x_st, const void* branch, int64_t branch_st, const void* gate, int64_t gate_st,
                       int64_t gate_rows, int gate_dtype, const void* post_weight, int post_dtype, const void* weight,
                       int weight_dtype, int dtype, int64_t rows, int64_t D, float residual_scale, float branch_scale,
                       float eps, void* h, void* n, int8_t* n_q, int64_t n_q_st, float* n_scale, float* stats,
                       pisa_stream_t stream) {
  using namespace pisa;
  if (int rc = check(x, x_st, branch, gate, gate_rows, gate_dtype, post_weight, post_dtype, weight, weight_dtype, dtype, rows, D,
                     residual_scale, branch_scale, eps))
    return rc;
  if ((branch && !h) || (!n && !n_q) || (n_q && !n_scale)) return fail(PISA_ERR_INVALID, "the outputs are required");
  if (n && n_q) return fail(PISA_ERR_INVALID, "the norm is written in its type or in 8 bits");
  if (n_q && !rows_on16(n_q, rows, n_q_st)) return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must start on 16 bytes");
  NormArgs a{};
  a.x = x; a.x_st = x_st; a.y = branch; a.y_st = branch_st;
  a.gate = gate; a.gate_st = gate_st; a.gate_rows = uint32_t(gate_rows); a.gate_f32 = gate_dtype == PISA_F32;
  a.post = post_weight; a.post_f32 = post_dtype == PISA_F32; a.w = weight; a.w_f32 = weight_dtype == PISA_F32;
  a.rows = rows; a.D = int(D); a.a = residual_scale; a.b = branch_scale; a.eps = eps; a.inv_d = 1.f / float(D);
  a.h = h; a.n = n; a.n_q = n_q; a.n_q_st = n_q_st; a.n_scale = n_scale; a.stats = stats;
  const int es = dtype == PISA_F32 ? 4 : 2;
  const bool aligned = D % 8 == 0 && rows_on16(x, rows, x_st * es) && (!branch || (rows_on16(branch, rows, branch_st * es) && param_on16(h))) &&
                       (!gate || rows_on16(gate, gate_rows ? rows / gate_rows : rows, gate_st * (a.gate_f32 ? 4 : es))) && param_on16(n) &&
                       param_on16(weight) && param_on16(post_weight);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PISA_F32) return fwd<float>(a, aligned, s);
  if (dtype == PISA_BF16) return fwd<__nv_bfloat16>(a, aligned, s);
  return fwd<__half>(a, aligned, s);
}

int64_t pisa_residual_norm_bwd_workspace_bytes(int64_t rows, int64_t D, int64_t gate_rows) {
  using namespace pisa;
  if (rows <= 0 || D <= 0 || D > kMaxWidth || gate_rows < 0 || (gate_rows && rows % gate_rows)) return -1;
  const Plan p = make_plan(rows, D, gate_rows ? gate_rows : rows);
  return p.means_bytes + int64_t(sizeof(float)) * 3 * D * p.partials;
}

int pisa_residual_norm_bwd(const void* dh, const void* dn, const void* x, int64_t x_st, const void* branch, int64_t branch_st,
                           const void* gate, int64_t gate_st, int64_t gate_rows, int gate_dtype, const void* post_weight,
                           int post_dtype, const void* weight, int weight_dtype, int dtype, int64_t rows, int64_t D,
                           float residual_scale, float branch_scale, const float* stats, void* dx, void* dbranch, void* dgate,
                           void* dpost_weight, void* dweight, void* workspace, int64_t workspace_bytes, pisa_stream_t stream) {
  using namespace pisa;
  if (int rc = check(x, x_st, branch, gate, gate_rows, gate_dtype, post_weight, post_dtype, weight, weight_dtype, dtype, rows, D,
                     residual_scale, branch_scale, 0.f))
    return rc;
  if (!dn || !stats || !dx || !dweight || (branch && !dbranch) || (gate && !dgate) || (post_weight && !dpost_weight))
    return fail(PISA_ERR_INVALID, "the gradients and the forward's statistics are required");
  if (reinterpret_cast<uintptr_t>(stats) & 7u) return fail(PISA_ERR_INVALID, "statistics must start on 8 bytes");
  const bool shared = gate && gate_rows;
  const Plan p = make_plan(rows, D, shared ? gate_rows : rows);
  if (p.ctas >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "too many gate rows");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7u) || workspace_bytes < pisa_residual_norm_bwd_workspace_bytes(rows, D, gate ? gate_rows : 0))
    return fail(PISA_ERR_INVALID, "workspace too small or not on 8 bytes");
  NormArgs a{};
  a.x = x; a.x_st = x_st; a.y = branch; a.y_st = branch_st;
  a.gate = gate; a.gate_st = gate_st; a.gate_rows = uint32_t(gate_rows); a.gate_f32 = gate_dtype == PISA_F32;
  a.post = post_weight; a.post_f32 = post_dtype == PISA_F32; a.w = weight; a.w_f32 = weight_dtype == PISA_F32;
  a.rows = rows; a.D = int(D); a.a = residual_scale; a.b = branch_scale; a.inv_d = 1.f / float(D);
  a.stats = const_cast<float*>(stats);
  a.dh = dh; a.dn = dn; a.dx = dx; a.dy = dbranch; a.dgate = dgate;
  a.means = static_cast<float*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.means_bytes);
  a.combine = p.combine;
  a.dw = dweight; a.dpost = dpost_weight;
  a.sums = 1;
  if (post_weight) a.sum_post = a.sums++;
  if (shared) a.sum_gate = a.sums++;
  a.share_rows = p.share_rows; a.share_teams = p.share_teams;
  const int es = dtype == PISA_F32 ? 4 : 2;
  const bool aligned = D % 8 == 0 && rows_on16(x, rows, x_st * es) && (!branch || rows_on16(branch, rows, branch_st * es)) &&
                       (!gate || rows_on16(gate, gate_rows ? rows / gate_rows : rows, gate_st * (a.gate_f32 ? 4 : es))) && param_on16(dh) &&
                       param_on16(dn) && param_on16(dx) && param_on16(dbranch) && param_on16(dgate) && param_on16(weight) &&
                       param_on16(post_weight);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PISA_F32) return bwd<float>(a, p, aligned, s);
  if (dtype == PISA_BF16) return bwd<__nv_bfloat16>(a, p, aligned, s);
  return bwd<__half>(a, p, aligned, s);
}

}  // extern "C"

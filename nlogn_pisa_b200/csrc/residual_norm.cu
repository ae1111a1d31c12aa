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
// another and other teams of the SM fill their waits.
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
  int sums, sum_post, sum_gate;   // rows of a partial: weight 0, then post and gate where they are summed
  uint32_t share_rows, share_teams;   // rows of a share (one gate row's, or all), teams of a share
  uint32_t teams, cols;   // teams in all, CTAs of a gradient row
  void* dw;
  void* dpost;
};

template <typename T, int TPR, int NV, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1;
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x % TPR, D = a.D;
  const int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TPR;
  if (row >= a.rows) return;                      // a whole warp: larger teams are CTAs with a row each
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
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[8];
        widen8<T>(y[j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(f[e], f[e], sum);
      }
      inv_y = rsqrtf(team_reduce<TPR, false>(sum, red, set) * a.inv_d + a.eps);
    }
    const char* gr = static_cast<const char*>(a.gate);
    if (gr) gr += int64_t(a.gate_rows ? uint32_t(row) / a.gate_rows : uint32_t(row)) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T)));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[8], p[8];
      widen8<T>(x[j], h[j]);
      widen8<T>(y[j], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= inv_y;
      if (a.post) {
        param_piece<T, TPR, A>(a.post, a.post_f32, j, t, D, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= p[e];
      }
      if (gr) {
        param_piece<T, TPR, A>(gr, a.gate_f32, j, t, D, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= p[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = fmaf(a.b, f[e], a.a * h[j][e]);
    }
    T* hr = static_cast<T*>(a.h) + row * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece<T, TPR, A>(hr, j, t, D, h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) widen8<T>(x[j], h[j]);
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[j][e], h[j][e], sum);
  const float inv_h = rsqrtf(team_reduce<TPR, false>(sum, red, set) * a.inv_d + a.eps);
  if (a.stats && t == 0) {
    a.stats[2 * row] = inv_y;
    a.stats[2 * row + 1] = inv_h;
  }
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float w[8];
    param_piece<T, TPR, A>(a.w, a.w_f32, j, t, D, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[j][e] = h[j][e] * inv_h * w[e];
      top = max_nan(top, fabsf(h[j][e]));
    }
  }
  if (a.n_q) {
    // places past the row's end hold 0 * inv_h * 0: NaN where eps is 0 and the row is, as its values are
    top = team_reduce<TPR, true>(top, red, set);
    const Scale8 s(top);
    int8_t* qr = a.n_q + row * a.n_q_st;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece_s8<TPR, A>(qr, j, t, D, h[j], top < INFINITY, s.inv);
    if (t == 0) a.n_scale[row] = s.scale;
  } else {
    T* nr = static_cast<T*>(a.n) + row * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece<T, TPR, A>(nr, j, t, D, h[j]);
  }
}

// A team's running sums of one parameter's gradient for wide rows: in shared
// memory, where each thread touches its own columns only.
template <int TPR, bool A>
struct Sums {
  float* at;
  __device__ __forceinline__ void add(int j, int t, int D, const float (&x)[8], const float (&y)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<TPR, A>(j, e, t);
      if (c < D) at[c] = fmaf(x[e], y[e], at[c]);
    }
  }
};

// The backward for wider rows, a CTA each, their operands read as they are needed.
template <typename T, int TPR, int NV, bool A>
__global__ void __launch_bounds__(TPR) norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ float sums[];
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x, D = a.D;
  const uint32_t team = blockIdx.x;
  const uint32_t share = team / a.share_teams, first = team - share * a.share_teams;
  const int64_t begin = int64_t(share) * a.share_rows;
  Sums<TPR, A> dw{sums}, dp{sums + a.sum_post * D}, dg{sums + a.sum_gate * D};
  for (int c = t; c < a.sums * D; c += TPR) sums[c] = 0.f;
  __syncthreads();
  for (uint32_t i = first; i < a.share_rows; i += a.share_teams) {
    const int64_t row = begin + i;
    Raw8<T> x[NV], dn[NV], dh[NV], y[NV];
    const T* xr = static_cast<const T*>(a.x) + row * a.x_st;
    const T* dnr = static_cast<const T*>(a.dn) + row * D;
    const T* dhr = static_cast<const T*>(a.dh) + row * D;
    const T* yr = static_cast<const T*>(a.y) + row * a.y_st;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = load_piece<T, TPR, A>(xr, j, t, D);
      dn[j] = load_piece<T, TPR, A>(dnr, j, t, D);
      if (a.dh) dh[j] = load_piece<T, TPR, A>(dhr, j, t, D);
      if (a.y) y[j] = load_piece<T, TPR, A>(yr, j, t, D);
    }
    const float inv_y = a.stats[2 * row], inv_h = a.stats[2 * row + 1];
    const char* gr = static_cast<const char*>(a.gate);
    if (gr) gr += int64_t(a.gate_rows ? uint32_t(row) / a.gate_rows : uint32_t(row)) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T)));
    float s[NV][8], v[NV][8], g[NV][8], dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[8];
      widen8<T>(x[j], v[j]);
      if (a.y) {
        float f[8];
        widen8<T>(y[j], f);
        if (a.post) {
          param_piece<T, TPR, A>(a.post, a.post_f32, j, t, D, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = f[e] * inv_y * w[e];
        }
        if (gr) {
          param_piece<T, TPR, A>(gr, a.gate_f32, j, t, D, g[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= g[j][e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = fmaf(a.b, f[e], a.a * v[j][e]);
      }
      param_piece<T, TPR, A>(a.w, a.w_f32, j, t, D, w);
      widen8<T>(dn[j], s[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= inv_h;
      dw.add(j, t, D, s[j], v[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[j][e] *= w[e];
        dot = fmaf(s[j][e], v[j][e], dot);
      }
    }
    float mean = team_reduce<TPR, false>(dot, red, set) * a.inv_d;
    T* dxr = static_cast<T*>(a.dx) + row * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float d[8];
      if (a.dh) {
        widen8<T>(dh[j], d);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[j][e] = fmaf(fmaf(-v[j][e], mean, s[j][e]), inv_h, d[e]);
        d[e] = a.a * s[j][e];
        s[j][e] *= a.b;
      }
      store_piece<T, TPR, A>(dxr, j, t, D, d);
    }
    if (!a.y) continue;
    dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float p[8];
      widen8<T>(y[j], v[j]);
      if (a.post) {
        param_piece<T, TPR, A>(a.post, a.post_f32, j, t, D, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= inv_y;
      }
      if (gr) {
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = a.post ? v[j][e] * p[e] : v[j][e];
        if (a.sum_gate) {
          dg.add(j, t, D, s[j], u);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] *= s[j][e];
          store_piece<T, TPR, A>(static_cast<T*>(a.dgate) + row * D, j, t, D, u);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] *= g[j][e];
      }
      if (a.post) {
        dp.add(j, t, D, s[j], v[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[j][e] *= p[e];
          dot = fmaf(s[j][e], v[j][e], dot);
        }
      }
    }
    if (a.post) {
      mean = team_reduce<TPR, false>(dot, red, set) * a.inv_d;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = fmaf(-v[j][e], mean, s[j][e]) * inv_y;
    }
    T* dyr = static_cast<T*>(a.dy) + row * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_piece<T, TPR, A>(dyr, j, t, D, s[j]);
  }
  __syncthreads();
  float* out = a.partial + int64_t(team) * a.sums * D;
  for (int c = t; c < a.sums * D; c += TPR) out[c] = sums[c];
}

// The backward for rows that a team holds with 8 elements per thread.  A team
// keeps the parameters and their running sums in registers, and the next row's
// operands are on their way while it works on one.  One barrier per row: the
// second norm's sum follows from three that need no other,
//   mean(s p z) with s = b g t  is  S2 - mean(dn w v) / rms(h) S3,
//   S2 = mean(q (dh + dn w / rms(h))), S3 = mean(q v), q = b g p z.
template <typename T, int TPR, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_bwd_row_kernel(const __grid_constant__ NormArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1, W = TPR / 32;
  __shared__ float red[2][3][W];
  int set = 0;
  const int t = threadIdx.x % TPR, D = a.D;
  const uint32_t team = blockIdx.x * TEAMS + threadIdx.x / TPR;
  const uint32_t share = team / a.share_teams, first = team - share * a.share_teams;
  const int64_t begin = int64_t(share) * a.share_rows;
  if (begin >= a.rows) return;                    // a whole warp
  const bool token_gate = a.gate && !a.gate_rows;
  const char* gr = static_cast<const char*>(a.gate);
  float w[8], p[8], g[8], dw[8], dp[8], dg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = dp[e] = dg[e] = 0.f, p[e] = g[e] = 1.f;
  param_piece<T, TPR, A>(a.w, a.w_f32, 0, t, D, w);
  if (a.post) param_piece<T, TPR, A>(a.post, a.post_f32, 0, t, D, p);
  // the rows of a share have one gate row
  if (gr && !token_gate)
    param_piece<T, TPR, A>(gr + int64_t(uint32_t(begin) / a.gate_rows) * a.gate_st * (a.gate_f32 ? 4 : int(sizeof(T))), a.gate_f32, 0, t,
                           D, g);
  struct Row {
    Raw8<T> x, y, dn, dh, g;
    float inv_y, inv_h;
  };
  Row next;
  auto fetch = [&](int64_t row) {
    next.x = load_piece<T, TPR, A>(static_cast<const T*>(a.x) + row * a.x_st, 0, t, D);
    next.dn = load_piece<T, TPR, A>(static_cast<const T*>(a.dn) + row * D, 0, t, D);
    if (a.dh) next.dh = load_piece<T, TPR, A>(static_cast<const T*>(a.dh) + row * D, 0, t, D);
    if (a.y) next.y = load_piece<T, TPR, A>(static_cast<const T*>(a.y) + row * a.y_st, 0, t, D);
    if (token_gate) next.g = load_piece<T, TPR, A>(reinterpret_cast<const T*>(gr) + row * a.gate_st, 0, t, D);
    next.inv_y = a.stats[2 * row];
    next.inv_h = a.stats[2 * row + 1];
  };
  fetch(begin + first);
  for (uint32_t i = first; i < a.share_rows; i += a.share_teams) {
    const int64_t row = begin + i;
    const Row r = next;
    if (a.share_rows - i > a.share_teams) fetch(row + a.share_teams);
    float z[8], v[8], s[8], d[8], sums[3] = {0.f, 0.f, 0.f};
    widen8<T>(r.x, v);
    widen8<T>(r.dn, s);
    if (a.dh) {
      widen8<T>(r.dh, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = 0.f;
    }
    if (token_gate) widen8<T>(r.g, g);
    if (a.y) {
      widen8<T>(r.y, z);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (a.post) z[e] *= r.inv_y;
        v[e] = fmaf(a.b, g[e] * (z[e] * p[e]), a.a * v[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= r.inv_h;
      dw[e] = fmaf(s[e], v[e], dw[e]);
      s[e] *= w[e];
      sums[0] = fmaf(s[e], v[e], sums[0]);
      if (a.post) {
        const float q = a.b * g[e] * (p[e] * z[e]);
        sums[1] = fmaf(q, fmaf(r.inv_h, s[e], d[e]), sums[1]);
        sums[2] = fmaf(q, v[e], sums[2]);
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (k && !a.post) break;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sums[k] += __shfl_xor_sync(kFull, sums[k], o);
    }
    if constexpr (W > 1) {
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < 3; ++k) red[set][k][threadIdx.x >> 5] = sums[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (k && !a.post) break;
        sums[k] = red[set][k][0];
#pragma unroll
        for (int x = 1; x < W; ++x) sums[k] += red[set][k][x];
      }
      set ^= 1;
    }
    const float mean = sums[0] * a.inv_d, mean_y = fmaf(-mean * r.inv_h, sums[2], sums[1]) * a.inv_d;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] = fmaf(fmaf(-v[e], mean, s[e]), r.inv_h, d[e]);
      d[e] = a.a * s[e];
      s[e] *= a.b;
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dx) + row * D, 0, t, D, d);
    if (!a.y) continue;
    if (gr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d[e] = s[e] * (z[e] * p[e]);
        dg[e] += d[e];
        s[e] *= g[e];
      }
      if (token_gate) store_piece<T, TPR, A>(static_cast<T*>(a.dgate) + row * D, 0, t, D, d);
    }
    if (a.post) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dp[e] = fmaf(s[e], z[e], dp[e]);
        s[e] = fmaf(-z[e], mean_y, s[e] * p[e]) * r.inv_y;
      }
    }
    store_piece<T, TPR, A>(static_cast<T*>(a.dy) + row * D, 0, t, D, s);
  }
  float* out = a.partial + int64_t(team) * a.sums * D;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = column<TPR, A>(0, e, t);
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
  if (a.D <= 256) return launch_fwd<T, 32, 1>(a, aligned, s);
  if (a.D <= 512) return launch_fwd<T, 32, 2>(a, aligned, s);
  if (a.D <= 1024) return launch_fwd<T, 32, 4>(a, aligned, s);
  if (a.D <= 2048) return launch_fwd<T, 128, 2>(a, aligned, s);
  if (a.D <= 4096) return launch_fwd<T, 128, 4>(a, aligned, s);
  if (a.D <= 8192) return launch_fwd<T, 256, 4>(a, aligned, s);
  return launch_fwd<T, 512, 4>(a, aligned, s);
}

// Teams of the backward: their threads and CTAs per SM by width.
struct Plan {
  int tpr, teams_per_cta, ctas;
  uint32_t share_rows, share_teams;
  int64_t shares, teams;
};

Plan make_plan(int64_t rows, int64_t D, int64_t share_rows) {
  Plan p{};
  p.tpr = D <= 256 ? 32 : D <= 1024 ? 128 : D <= 2048 ? 256 : 512;
  p.teams_per_cta = p.tpr < 128 ? 128 / p.tpr : 1;
  const int64_t most = int64_t(sm_count()) * (D <= 256 ? 16 : D <= 1024 ? 4 : D <= 2048 ? 2 : 1);
  p.share_rows = uint32_t(share_rows);
  p.shares = rows / share_rows;
  const int64_t each = most / p.shares;
  p.share_teams = uint32_t(each < 1 ? 1 : each < share_rows ? each : share_rows);
  p.teams = p.shares * p.share_teams;
  p.ctas = int((p.teams + p.teams_per_cta - 1) / p.teams_per_cta);
  return p;
}

template <typename T, int TPR>
int launch_bwd_row(const NormArgs& a, const Plan& p, bool aligned, cudaStream_t s) {
  constexpr int threads = TPR < 128 ? 128 : TPR;
  if (aligned) norm_bwd_row_kernel<T, TPR, true><<<unsigned(p.ctas), threads, 0, s>>>(a);
  else norm_bwd_row_kernel<T, TPR, false><<<unsigned(p.ctas), threads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int NV, bool A>
int launch_bwd(const NormArgs& a, const Plan& p, cudaStream_t s) {
  if (int rc = allow_smem<norm_bwd_kernel<T, 512, NV, A>>(int(sizeof(float)) * 3 * NV * 4096, "norm backward smem attribute")) return rc;
  norm_bwd_kernel<T, 512, NV, A><<<unsigned(p.ctas), 512, sizeof(float) * a.sums * a.D, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int bwd(NormArgs a, const Plan& p, bool aligned, cudaStream_t s) {
  int rc;
  if (a.D <= 256) rc = launch_bwd_row<T, 32>(a, p, aligned, s);
  else if (a.D <= 1024) rc = launch_bwd_row<T, 128>(a, p, aligned, s);
  else if (a.D <= 2048) rc = launch_bwd_row<T, 256>(a, p, aligned, s);
  else if (a.D <= 4096) rc = launch_bwd_row<T, 512>(a, p, aligned, s);
  else if (a.D <= 8192) rc = aligned ? launch_bwd<T, 2, true>(a, p, s) : launch_bwd<T, 2, false>(a, p, s);
  else rc = aligned ? launch_bwd<T, 4, true>(a, p, s) : launch_bwd<T, 4, false>(a, p, s);
  if (rc) return rc;
  a.teams = uint32_t(p.teams);
  a.cols = uint32_t((a.D + 31) / 32);
  const int64_t rows = 1 + (a.sum_post ? 1 : 0) + (a.sum_gate ? p.shares : 0);
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
  return int64_t(sizeof(float)) * 3 * D * make_plan(rows, D, gate_rows ? gate_rows : rows).teams;
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
  const bool shared = gate && gate_rows;
  const Plan p = make_plan(rows, D, shared ? gate_rows : rows);
  if (!workspace || workspace_bytes < pisa_residual_norm_bwd_workspace_bytes(rows, D, gate ? gate_rows : 0))
    return fail(PISA_ERR_INVALID, "workspace too small");
  NormArgs a{};
  a.x = x; a.x_st = x_st; a.y = branch; a.y_st = branch_st;
  a.gate = gate; a.gate_st = gate_st; a.gate_rows = uint32_t(gate_rows); a.gate_f32 = gate_dtype == PISA_F32;
  a.post = post_weight; a.post_f32 = post_dtype == PISA_F32; a.w = weight; a.w_f32 = weight_dtype == PISA_F32;
  a.rows = rows; a.D = int(D); a.a = residual_scale; a.b = branch_scale; a.inv_d = 1.f / float(D);
  a.stats = const_cast<float*>(stats);
  a.dh = dh; a.dn = dn; a.dx = dx; a.dy = dbranch; a.dgate = dgate;
  a.partial = static_cast<float*>(workspace);
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

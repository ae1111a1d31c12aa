// Attention of every query over all keys of its sequence (causal or not), and
// its gradient, on the FMA pipes: fp32 tensors, and 16-bit heads wider than
// 128, which the tensor-core kernels do not hold.
//
// With s_ij = scale q_i . k_j over the keys that query i sees,
//   l_i = sum_j exp(s_ij - m_i),  out_i = sum_j exp(s_ij - m_i) v_j / l_i,
//   lse_i = m_i + ln l_i   (no visible key: out_i = 0, lse_i = -inf).
// Backward, with P = exp(s - lse), delta_i = dout_i . out_i and
// dS = scale P (dout v - delta):
//   dq = dS k,   dk = dS^T q,   dv = P^T dout   (dk, dv summed over the G
// query heads of a KV head).  Forward and dq walk the key tiles of a query
// tile, dk / dv walk the query tiles of a key tile: no atomics, so results do
// not vary from run to run.
//
// Bound by FP32 FMAs.  Tiles of R*16 x R*16 scores, a thread computes R x R
// of them from shared memory rows padded by 16 bytes (the 8 rows that a
// quarter of a warp reads then fall in different banks) and R rows x DP/16
// columns of each output.  Rows outside the sequence are staged as zeros and
// products with hidden keys are skipped, not multiplied by zero, so
// infinities and NaN in hidden places reach nothing.
//
// Measured: two fp32 sequences of 1500 and 2596, 4 heads of 64: forward 186 us,
// dq 320 us, dk and dv 359 us, 25, 22 and 26 TFLOP/s or a third of the FMA pipes'
// rate.  Four heads make few tiles, and the longest causal ones end the launch.
#include <type_traits>

#include "dense_attn.cuh"
#include "tc.cuh"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr size_t kOnePerSm = 116 * 1024;   // more than half an SM's shared memory

// rows x DP tile of `src` (row stride `stride` elements) into fp32 shared
// memory, zero past `valid` rows and past D columns
template <typename T, int DP, int LD>
__device__ __forceinline__ void stage(float* dst, const T* src, int64_t stride, int rows, int valid, int D) {
  constexpr int VN = Vec<T>::N, SEG = DP / VN;
  for (int i = threadIdx.x; i < rows * SEG; i += kThreads) {
    const int r = i / SEG, c = (i - r * SEG) * VN;
    float v[VN];
#pragma unroll
    for (int e = 0; e < VN; ++e) v[e] = 0.f;
    if (r < valid && c < D) load_vec<T>(src + r * stride + c, v);
#pragma unroll
    for (int e = 0; e < VN; e += 4)
      *reinterpret_cast<float4*>(dst + r * LD + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
}

// The same tile by asynchronous copies (fp32); the caller waits for the group.
template <int DP, int LD>
__device__ __forceinline__ void stage_async(float* dst, const float* src, int64_t stride, int rows, int valid, int D) {
  constexpr int SEG = DP / 4;
  for (int i = threadIdx.x; i < rows * SEG; i += kThreads) {
    const int r = i / SEG, c = (i - r * SEG) * 4;
    const bool real = r < valid && c < D;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 :: "r"(tc::smem_u32(dst + r * LD + c)), "l"(real ? src + r * stride + c : src), "r"(real ? 16 : 0) : "memory");
  }
}

// Two tiles that a loop consumes one after the other (keys and values, or
// queries and dout).  fp32: the next pair is copied while this one is used, in
// the second of two buffers; one CTA per SM then starts its tiles in falling
// order of their work.  Otherwise: converted into the one buffer in between.
template <typename T, int DP, bool FITS = true> struct Pair {
  static constexpr bool async = std::is_same<T, float>::value, ahead = async && FITS;
  static constexpr int LD = DP + 4, BUFFERS = ahead ? 2 : 1;

  template <int BT>
  __device__ __forceinline__ static void fetch(float* buffer, const T* a, int64_t a_st, int da, const T* b, int64_t b_st,
                                               int db, int valid) {
    if constexpr (async) {
      stage_async<DP, LD>(buffer, a, a_st, BT, valid, da);
      stage_async<DP, LD>(buffer + BT * LD, b, b_st, BT, valid, db);
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else {
      stage<T, DP, LD>(buffer, a, a_st, BT, valid, da);
      stage<T, DP, LD>(buffer + BT * LD, b, b_st, BT, valid, db);
    }
  }
  __device__ __forceinline__ static void arrived() {
    if constexpr (async) asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }
};

// acc[i][j] += a row (ty*R + i) . b row (tx + 16 j), pairs of dims at a time
template <int R, int DP, int LD>
__device__ __forceinline__ void rows_dot(const float* a, const float* b, int ty, int tx, float (&acc)[R][R]) {
  float2 sum[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) sum[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[R], y[R];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty * R + i) * LD + d);
#pragma unroll
    for (int j = 0; j < R; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * LD + d);
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        sum[i][j] = tc::fma2(make_float2(x[i].x, x[i].y), make_float2(y[j].x, y[j].y), sum[i][j]);
        sum[i][j] = tc::fma2(make_float2(x[i].z, x[i].w), make_float2(y[j].z, y[j].w), sum[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] += sum[i][j].x + sum[i][j].y;
}

// acc[i][c] += sum_j w[ty*R + i][j] x[j][columns of tx]; a weight outside
// [lo[i], hi[i]] is skipped when `partial`.  Columns of tx: 4 from tx*4 + 64 c.
// Four keys per step: a row of weights is one 16-byte load.  Rows of w past
// `count` (to a multiple of four) are skipped as well.
template <int R, int DP, int LD, int LP>
__device__ __forceinline__ void rows_sum(const float* w, const float* x, int count, int ty, int tx, bool partial,
                                         const int (&lo)[R], const int (&hi)[R], float2 (&acc)[R][DP / 32]) {
  const int whole = partial ? 0 : count & ~3;
#pragma unroll 2
  for (int j = 0; j < whole; j += 4) {
    float4 p[R];
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = *reinterpret_cast<const float4*>(w + (ty * R + i) * LP + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 y = *reinterpret_cast<const float4*>(x + (j + e) * LD + tx * 4 + 64 * c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float v = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
          acc[i][2 * c] = tc::fma2(make_float2(v, v), make_float2(y.x, y.y), acc[i][2 * c]);
          acc[i][2 * c + 1] = tc::fma2(make_float2(v, v), make_float2(y.z, y.w), acc[i][2 * c + 1]);
        }
      }
    }
  }
  for (int j = whole; j < count; ++j) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(x + j * LD + tx * 4 + 64 * c);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (partial && (j < lo[i] || j > hi[i])) continue;
        const float v = w[(ty * R + i) * LP + j];
        acc[i][2 * c] = tc::fma2(make_float2(v, v), make_float2(y.x, y.y), acc[i][2 * c]);
        acc[i][2 * c + 1] = tc::fma2(make_float2(v, v), make_float2(y.z, y.w), acc[i][2 * c + 1]);
      }
    }
  }
}

template <int DP> struct Tile {
  static constexpr int R = DP <= 128 ? 4 : 2;   // 256 dims: tiles of 32 keep four of them in shared memory
  static constexpr int BT = R * 16, LD = DP + 4, LP = BT + 4;
};

template <typename T, int R, int DP>
__device__ __forceinline__ void store_rows(T* dst, int64_t stride, int valid, int D, int ty, int tx,
                                           const float2 (&acc)[R][DP / 32], const float (&mul)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty * R + i;
    if (r >= valid) continue;
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = tx * 4 + 64 * c + e;
        const float2 v = acc[i][2 * c + e / 2];
        if (d < D) dst[r * stride + d] = from_f32<T>((e & 1 ? v.y : v.x) * mul[i]);
      }
    }
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) dense_fwd_kernel(const __grid_constant__ DenseAttnArgs a) {
  using S = Tile<DP>;
  constexpr int R = S::R, BT = S::BT, LD = S::LD, LP = S::LP;
  extern __shared__ __align__(16) float smem[];
  using P = Pair<T, DP>;
  float* qs = smem;
  float* ps = qs + BT * LD;
  float* ring = ps + BT * LP;
  // later query tiles, which see more keys, first
  const int index = int(gridDim.x) - 1 - int(blockIdx.x);
  const int slot = index / a.Hq, hq = index - slot * a.Hq, h = hq / a.G;
  const SeqTile t = seq_tile(a, slot, BT, false);
  const int q0 = t.tile * BT;
  if (q0 >= t.q_len) return;
  const int valid = min(BT, t.q_len - q0);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + int64_t(t.q_begin + q0) * a.q_st + hq * a.q_sh;
  const T* kp = static_cast<const T*>(a.k) + t.b * a.k_sb + int64_t(t.k_begin) * a.k_st + h * a.k_sh;
  const T* vp = static_cast<const T*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin) * a.v_st + h * a.v_sh;
  stage<T, DP, LD>(qs, qp, a.q_st, BT, valid, a.D);
  const float sl = a.scale * kLog2e;
  float2 acc[R][DP / 32];
  float m[R], l[R];
  int last[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    last[i] = last_visible(a, t, q0 + ty * R + i);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = make_float2(0.f, 0.f);
  }
  const int end = last_visible(a, t, q0 + valid - 1) + 1, full = last_visible(a, t, q0) + 1;
  auto fetch = [&](int j0, int buffer) {
    P::template fetch<BT>(ring + buffer * 2 * BT * LD, kp + int64_t(j0) * a.k_st, a.k_st, a.D, vp + int64_t(j0) * a.v_st,
                          a.v_st, a.Dv, min(BT, t.k_len - j0));
  };
  if (P::ahead && end > 0) fetch(0, 0);
  int buffer = 0;
  for (int j0 = 0; j0 < end; j0 += BT) {
    const int nk = min(BT, t.k_len - j0);
    if (!P::ahead) {
      __syncthreads();
      fetch(j0, 0);
    }
    P::arrived();
    if (P::ahead && j0 + BT < end) fetch(j0 + BT, buffer ^ 1);
    const float* ks = ring + buffer * 2 * BT * LD;
    const float* vs = ks + BT * LD;
    if (P::ahead) buffer ^= 1;
    float s[R][R] = {};
    rows_dot<R, DP, LD>(qs, ks, ty, tx, s);
    int lo[R], hi[R];
    bool grown = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      lo[i] = 0;
      hi[i] = last[i] - j0;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        s[i][j] = tx + 16 * j <= hi[i] ? s[i][j] * sl : -INFINITY;
        grown = grown || s[i][j] > m[i];
      }
    }
    // the rows' maxima move in few tiles: one vote instead of the shuffles
    if (__any_sync(kFull, grown)) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float top = m[i];
#pragma unroll
        for (int j = 0; j < R; ++j) top = fmaxf(top, s[i][j]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
        const float corr = top == -INFINITY ? 1.f : exp2f(m[i] - top);
        m[i] = top;
        l[i] *= corr;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) acc[i][c] = make_float2(acc[i][c].x * corr, acc[i][c].y * corr);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const float p = exp2f(s[i][j] - base);
        ps[(ty * R + i) * LP + tx + 16 * j] = p;
        l[i] += p;                          // this thread's share of the row's sum
      }
    }
    __syncwarp();   // the rows of ps that a warp reads are its own
    rows_sum<R, DP, LD, LP>(ps, vs, min(nk, end - j0), ty, tx, j0 + BT > full, lo, hi, acc);
  }
  float inv[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(kFull, l[i], o);
    inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    const int r = ty * R + i;
    if (a.lse && tx == 0 && r < valid)
      a.lse[(int64_t(t.b) * a.T + t.q_begin + q0 + r) * a.Hq + hq] =
          l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
  T* op = static_cast<T*>(a.out) + ((int64_t(t.b) * a.T + t.q_begin + q0) * a.Hq + hq) * a.Dv;
  store_rows<T, R, DP>(op, int64_t(a.Hq) * a.Dv, valid, a.Dv, ty, tx, acc, inv);
  if (a.out_low) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        const float2 v = make_float2(acc[i][c].x * inv[i], acc[i][c].y * inv[i]);
        acc[i][c] = make_float2(v.x - to_f32<T>(from_f32<T>(v.x)), v.y - to_f32<T>(from_f32<T>(v.y)));
      }
      inv[i] = 1.f;
    }
    T* lp = static_cast<T*>(a.out_low) + ((int64_t(t.b) * a.T + t.q_begin + q0) * a.Hq + hq) * a.Dv;
    store_rows<T, R, DP>(lp, int64_t(a.Hq) * a.Dv, valid, a.Dv, ty, tx, acc, inv);
  }
}

// delta = dout . (out + out_low) per row, one warp per row
template <typename T>
__global__ void __launch_bounds__(128) dense_delta_kernel(const T* __restrict__ dout, const T* __restrict__ out,
                                                          const T* __restrict__ low, float* __restrict__ delta,
                                                          int64_t rows, int Dv, int* status) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *status = PISA_OK;
  constexpr int VN = Vec<T>::N;
  const int64_t r = blockIdx.x * int64_t(4) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  float acc = 0.f;
  for (int d = lane * VN; d < Dv; d += 32 * VN) {
    float x[VN], y[VN];
    load_vec<T>(dout + r * Dv + d, x);
    load_vec<T>(out + r * Dv + d, y);
#pragma unroll
    for (int e = 0; e < VN; ++e) acc = fmaf(x[e], y[e], acc);
    if (low) {
      load_vec<T>(low + r * Dv + d, y);
#pragma unroll
      for (int e = 0; e < VN; ++e) acc = fmaf(x[e], y[e], acc);
    }
  }
  acc = warp_sum(acc);
  if (lane == 0) delta[r] = acc;
}

// Base-2 lse of a row for the recomputed weights; a row without weight (lse
// -inf) gets +inf, which makes them all zero.
__device__ __forceinline__ float lse_base2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// P and dS of one score element: base-2 logit minus base-2 lse
__device__ __forceinline__ float2 prob_grad(float s, float dp, float sl, float lse2, float delta, float scale,
                                            bool visible) {
  const float p = visible ? exp2f(fmaf(s, sl, -lse2)) : 0.f;
  return make_float2(p, visible ? scale * p * (dp - delta) : 0.f);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) dense_dq_kernel(const __grid_constant__ DenseAttnArgs a) {
  using S = Tile<DP>;
  constexpr int R = S::R, BT = S::BT, LD = S::LD, LP = S::LP;
  extern __shared__ __align__(16) float smem[];
  float* qs = smem;
  using P = Pair<T, DP>;
  float* os = qs + BT * LD;
  float* ds = os + BT * LD;
  float* ring = ds + BT * LP;
  const int index = int(gridDim.x) - 1 - int(blockIdx.x);
  const int slot = index / a.Hq, hq = index - slot * a.Hq, h = hq / a.G;
  const SeqTile t = seq_tile(a, slot, BT, false);
  const int q0 = t.tile * BT;
  if (q0 >= t.q_len) return;
  const int valid = min(BT, t.q_len - q0);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int64_t row0 = (int64_t(t.b) * a.T + t.q_begin + q0) * a.Hq + hq;
  const T* kp = static_cast<const T*>(a.k) + t.b * a.k_sb + int64_t(t.k_begin) * a.k_st + h * a.k_sh;
  const T* vp = static_cast<const T*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin) * a.v_st + h * a.v_sh;
  stage<T, DP, LD>(qs, static_cast<const T*>(a.q) + t.b * a.q_sb + int64_t(t.q_begin + q0) * a.q_st + hq * a.q_sh,
                   a.q_st, BT, valid, a.D);
  stage<T, DP, LD>(os, static_cast<const T*>(a.dout) + row0 * a.Dv, int64_t(a.Hq) * a.Dv, BT, valid, a.Dv);
  const float sl = a.scale * kLog2e;
  float2 acc[R][DP / 32];
  float lse2[R], delta[R];
  int last[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty * R + i;
    last[i] = r < valid ? last_visible(a, t, q0 + r) : -1;
    lse2[i] = r < valid ? lse_base2(a.lse_in[row0 + int64_t(r) * a.Hq]) : 0.f;
    delta[i] = r < valid ? a.delta[row0 + int64_t(r) * a.Hq] : 0.f;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = make_float2(0.f, 0.f);
  }
  const int end = last_visible(a, t, q0 + valid - 1) + 1, full = last_visible(a, t, q0) + 1;
  auto fetch = [&](int j0, int buffer) {
    P::template fetch<BT>(ring + buffer * 2 * BT * LD, kp + int64_t(j0) * a.k_st, a.k_st, a.D, vp + int64_t(j0) * a.v_st,
                          a.v_st, a.Dv, min(BT, t.k_len - j0));
  };
  if (P::ahead && end > 0) fetch(0, 0);
  int buffer = 0;
  for (int j0 = 0; j0 < end; j0 += BT) {
    const int nk = min(BT, t.k_len - j0);
    if (!P::ahead) {
      __syncthreads();
      fetch(j0, 0);
    }
    P::arrived();
    if (P::ahead && j0 + BT < end) fetch(j0 + BT, buffer ^ 1);
    const float* ks = ring + buffer * 2 * BT * LD;
    const float* vs = ks + BT * LD;
    if (P::ahead) buffer ^= 1;
    float s[R][R] = {}, dp[R][R] = {};
    rows_dot<R, DP, LD>(qs, ks, ty, tx, s);
    rows_dot<R, DP, LD>(os, vs, ty, tx, dp);
    int lo[R], hi[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      lo[i] = 0;
      hi[i] = last[i] - j0;
#pragma unroll
      for (int j = 0; j < R; ++j)
        ds[(ty * R + i) * LP + tx + 16 * j] =
            prob_grad(s[i][j], dp[i][j], sl, lse2[i], delta[i], a.scale, tx + 16 * j <= hi[i]).y;
    }
    __syncwarp();
    rows_sum<R, DP, LD, LP>(ds, ks, min(nk, end - j0), ty, tx, j0 + BT > full || valid < BT, lo, hi, acc);
  }
  float one[R];
#pragma unroll
  for (int i = 0; i < R; ++i) one[i] = 1.f;
  store_rows<T, R, DP>(static_cast<T*>(a.dq) + row0 * a.D, int64_t(a.Hq) * a.D, valid, a.D, ty, tx, acc, one);
}

// 128 dims: six operand tiles and the two of weights pass the shared memory
template <typename T, int DP> using KvPair = Pair<T, DP, DP != 128>;

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) dense_dkv_kernel(const __grid_constant__ DenseAttnArgs a) {
  using S = Tile<DP>;
  constexpr int R = S::R, BT = S::BT, LD = S::LD, LP = S::LP;
  extern __shared__ __align__(16) float smem[];
  float* ks = smem;
  float* vs = ks + BT * LD;
  using P = KvPair<T, DP>;
  float* ps = vs + BT * LD;      // P^T: key rows, query columns
  float* ds = ps + BT * LP;      // dS^T
  float* ring = ds + BT * LP;
  __shared__ float lse_s[2][64], delta_s[2][64];
  const int slot = int(blockIdx.x) / a.H, h = int(blockIdx.x) - slot * a.H;   // early keys, seen by most queries, first
  const SeqTile t = seq_tile(a, slot, BT, true);
  const int j0 = t.tile * BT;
  if (j0 >= t.k_len) return;
  const int valid = min(BT, t.k_len - j0);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  stage<T, DP, LD>(ks, static_cast<const T*>(a.k) + t.b * a.k_sb + int64_t(t.k_begin + j0) * a.k_st + h * a.k_sh,
                   a.k_st, BT, valid, a.D);
  stage<T, DP, LD>(vs, static_cast<const T*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin + j0) * a.v_st + h * a.v_sh,
                   a.v_st, BT, valid, a.Dv);
  const float sl = a.scale * kLog2e;
  float2 dk[R][DP / 32], dv[R][DP / 32];
  int first[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty * R + i;
    first[i] = r < valid ? first_seeing(a, t, j0 + r) : t.q_len;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) dk[i][c] = dv[i][c] = make_float2(0.f, 0.f);
  }
  const int begin = first_seeing(a, t, j0) / BT * BT, full = first_seeing(a, t, j0 + valid - 1);
  auto fetch = [&](int g, int q0, int buffer) {
    const int hq = h * a.G + g, nq = min(BT, t.q_len - q0);
    const int64_t row0 = (int64_t(t.b) * a.T + t.q_begin + q0) * a.Hq + hq;
    P::template fetch<BT>(ring + buffer * 2 * BT * LD,
                          static_cast<const T*>(a.q) + t.b * a.q_sb + int64_t(t.q_begin + q0) * a.q_st + hq * a.q_sh, a.q_st,
                          a.D, static_cast<const T*>(a.dout) + row0 * a.Dv, int64_t(a.Hq) * a.Dv, a.Dv, nq);
    if (threadIdx.x < BT) {
      const bool real = int(threadIdx.x) < nq;
      lse_s[buffer][threadIdx.x] = real ? lse_base2(a.lse_in[row0 + int64_t(threadIdx.x) * a.Hq]) : 0.f;
      delta_s[buffer][threadIdx.x] = real ? a.delta[row0 + int64_t(threadIdx.x) * a.Hq] : 0.f;
    }
  };
  int buffer = 0;
  if (P::ahead && begin < t.q_len) fetch(0, begin, 0);
  for (int g = 0; g < a.G; ++g) {
    for (int q0 = begin; q0 < t.q_len; q0 += BT) {
      const int nq = min(BT, t.q_len - q0), now = buffer;
      if (!P::ahead) {
        __syncthreads();
        fetch(g, q0, 0);
      }
      P::arrived();
      if (P::ahead) {
        buffer ^= 1;
        if (q0 + BT < t.q_len) fetch(g, q0 + BT, buffer);
        else if (g + 1 < a.G) fetch(g + 1, begin, buffer);
      }
      const float* qs = ring + now * 2 * BT * LD;
      const float* os = qs + BT * LD;
      float s[R][R] = {}, dp[R][R] = {};
      rows_dot<R, DP, LD>(ks, qs, ty, tx, s);
      rows_dot<R, DP, LD>(vs, os, ty, tx, dp);
      int lo[R], hi[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        lo[i] = first[i] - q0;
        hi[i] = nq - 1;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const int c = tx + 16 * j;
          const float2 pg = prob_grad(s[i][j], dp[i][j], sl, lse_s[now][c], delta_s[now][c], a.scale, c >= lo[i] && c <= hi[i]);
          ps[(ty * R + i) * LP + c] = pg.x;
          ds[(ty * R + i) * LP + c] = pg.y;
        }
      }
      __syncwarp();
      const bool partial = q0 < full || valid < BT;
      rows_sum<R, DP, LD, LP>(ps, os, nq, ty, tx, partial, lo, hi, dv);
      rows_sum<R, DP, LD, LP>(ds, qs, nq, ty, tx, partial, lo, hi, dk);
    }
  }
  float one[R];
#pragma unroll
  for (int i = 0; i < R; ++i) one[i] = 1.f;
  const int64_t row0 = (int64_t(t.b) * a.N + t.k_begin + j0) * a.H + h;
  store_rows<T, R, DP>(static_cast<T*>(a.dk) + row0 * a.D, int64_t(a.H) * a.D, valid, a.D, ty, tx, dk, one);
  store_rows<T, R, DP>(static_cast<T*>(a.dv) + row0 * a.Dv, int64_t(a.H) * a.Dv, valid, a.Dv, ty, tx, dv, one);
}

template <auto Kernel>
int launch(int64_t blocks, size_t smem, const DenseAttnArgs& a, cudaStream_t s) {
  if (blocks >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (int rc = allow_smem<Kernel>(int(smem), "dense attention smem attribute")) return rc;
  Kernel<<<unsigned(blocks), kThreads, smem, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int fwd_t(const DenseAttnArgs& a, cudaStream_t s) {
  using L = Tile<DP>;
  const int64_t slots = seq_slots(a.cu_q, a.B, a.T, a.sequences, L::BT);
  size_t smem = sizeof(float) * L::BT * ((1 + 2 * Pair<T, DP>::BUFFERS) * L::LD + L::LP);
  if (Pair<T, DP>::ahead && smem < kOnePerSm) smem = kOnePerSm;
  return launch<dense_fwd_kernel<T, DP>>(slots * a.Hq, smem, a, s);
}

template <typename T, int DP>
int bwd_t(const DenseAttnArgs& a, cudaStream_t s) {
  using L = Tile<DP>;
  const int64_t rows = int64_t(a.B) * a.T * a.Hq;
  if ((rows + 3) / 4 >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  dense_delta_kernel<T><<<unsigned((rows + 3) / 4), 128, 0, s>>>(static_cast<const T*>(a.dout),
                                                                 static_cast<const T*>(a.o), static_cast<const T*>(a.o_low),
                                                                 a.delta, rows, a.Dv, a.status);
  PISA_CHECK_LAUNCH();
  int rc = launch<dense_dq_kernel<T, DP>>(seq_slots(a.cu_q, a.B, a.T, a.sequences, L::BT) * a.Hq,
                  sizeof(float) * L::BT * ((2 + 2 * Pair<T, DP>::BUFFERS) * L::LD + L::LP), a, s);
  if (rc) return rc;
  return launch<dense_dkv_kernel<T, DP>>(seq_slots(a.cu_q, a.B, a.N, a.sequences, L::BT) * a.H,
                sizeof(float) * L::BT * ((2 + 2 * KvPair<T, DP>::BUFFERS) * L::LD + 2 * L::LP), a, s);
}

template <typename T>
int by_dim(const DenseAttnArgs& a, bool bwd, cudaStream_t s) {
  const int d = a.D > a.Dv ? a.D : a.Dv;
  if (d <= 64) return bwd ? bwd_t<T, 64>(a, s) : fwd_t<T, 64>(a, s);
  if (d <= 128) return bwd ? bwd_t<T, 128>(a, s) : fwd_t<T, 128>(a, s);
  return bwd ? bwd_t<T, 256>(a, s) : fwd_t<T, 256>(a, s);
}

int by_type(const DenseAttnArgs& a, int dtype, bool bwd, cudaStream_t s) {
  if (dtype == PISA_F32) return by_dim<float>(a, bwd, s);
  if (dtype == PISA_BF16) return by_dim<__nv_bfloat16>(a, bwd, s);
  return by_dim<__half>(a, bwd, s);
}

}  // namespace

int dense_attn_fwd_simt(const DenseAttnArgs& a, int dtype, cudaStream_t stream) {
  return by_type(a, dtype, false, stream);
}
int dense_attn_bwd_simt(const DenseAttnArgs& a, int dtype, cudaStream_t stream) {
  return by_type(a, dtype, true, stream);
}

}  // namespace pisa

// Norm of every query and key head with the split-half position rotation in
// the same pass, and its gradient.
//
// For a head row x of D elements, with u = x / sqrt(mean(x^2) + eps), the
// weight w (one per tensor, D elements) and the angle a_i = position *
// frequency_i (one fp32 product), i < D/2:
//   y = u w,  out_i = y_i cos a_i - y_{i+D/2} sin a_i,
//             out_{i+D/2} = y_i sin a_i + y_{i+D/2} cos a_i.
// Backward, with g = the inverse rotation of dout:
//   dw = sum over rows of g u,   h = g w,
//   dx = (h - u mean(h u)) / sqrt(mean(x^2) + eps).
// Everything is held in fp32 and rounded once to the output's type.
//
// Both directions are bound by HBM: forward reads x and writes out, backward
// reads x and dout and writes dx.  A lane holds V consecutive elements of the
// first half of a row and the V that rotate with them, so the rotation stays
// in registers and a row's sums are a few shuffles; a token's cosines and
// sines are computed once per CTA in shared memory and serve all its heads.
// Lanes keep their columns over all rows they visit, so dw accumulates in
// registers; each CTA stores one partial row and a second launch adds the
// partials in a fixed order (no atomics: results do not vary from run to run).
#include "dense_attn.cuh"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct NormSide {
  const void* x;
  int64_t sb, st, sh;   // element strides of x
  const void* dout;     // backward: contiguous gradient of out
  void* out;            // contiguous out, or dx
  const void* w;
  void* dw;
  int w_f32;            // weight is fp32 (else the tensors' type)
};

struct NormArgs {
  NormSide q, k;
  const float* freq;
  const int64_t* positions;
  int64_t pos_sb, pos_offset;
  int64_t rows;          // B * T tokens
  int T, Hq, H, D, half, lanes, lg_lanes;  // lanes per head row (a power of two)
  int tokens_per_cta;
  float eps;
  float* partial;        // backward: [CTAs][2][D]
};

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T e[V]; };

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32<T>(r.e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = r;
}

template <typename T>
__device__ __forceinline__ float weight_at(const NormSide& s, int i) {
  return s.w_f32 ? static_cast<const float*>(s.w)[i] : to_f32<T>(static_cast<const T*>(s.w)[i]);
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// cos and sin of the CTA's tokens into shared memory (float2 per pair)
__device__ __forceinline__ void fill_angles(const NormArgs& a, int64_t row0, int count, float2* table) {
  for (int i = threadIdx.x; i < count * a.half; i += kThreads) {
    const int tok = i / a.half, p = i - tok * a.half;
    const int64_t row = row0 + tok;
    const int64_t b = row / a.T, t = row - b * a.T;
    const int64_t pos = a.positions ? a.positions[b * a.pos_sb + t] : a.pos_offset + t;
    float s, c;
    sincosf(float(pos) * a.freq[p], &s, &c);
    table[i] = make_float2(c, s);
  }
}

template <typename T, int V, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_rotary_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ float2 table[];   // [tokens_per_cta][half]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_warp = 32 >> a.lg_lanes;           // head rows of one warp step
  const int sub = lane >> a.lg_lanes, col = (lane & (a.lanes - 1)) * V;
  const bool active = col < a.half;                // lanes past the row's columns idle
  const int heads = a.Hq + a.H, groups = (heads + per_warp - 1) / per_warp;
  float wq[2][V], wk[2][V], dq[2][V], dk[2][V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int d = col + i + s * a.half;
      wq[s][i] = active ? weight_at<T>(a.q, d) : 0.f;
      wk[s][i] = active ? weight_at<T>(a.k, d) : 0.f;
      dq[s][i] = dk[s][i] = 0.f;
    }
  }
  const float inv_d = 1.f / float(a.D);
  for (int64_t row0 = int64_t(blockIdx.x) * a.tokens_per_cta; row0 < a.rows;
       row0 += int64_t(gridDim.x) * a.tokens_per_cta) {
    const int count = int(min64(a.tokens_per_cta, a.rows - row0));
    __syncthreads();
    fill_angles(a, row0, count, table);
    __syncthreads();
    for (int item = warp; item < count * groups; item += kWarps) {
      const int tok = item / groups, head = (item - tok * groups) * per_warp + sub;
      const int64_t row = row0 + tok;
      const bool is_q = head < a.Hq, live = active && head < heads;
      const NormSide& s = is_q ? a.q : a.k;
      const int h = is_q ? head : head - a.Hq;
      const int64_t out_at = (row * (is_q ? a.Hq : a.H) + h) * a.D + col;
      float x0[V], x1[V], g0[V], g1[V];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) x0[i] = x1[i] = g0[i] = g1[i] = 0.f;
      if (live) {
        const int64_t b = row / a.T, t = row - b * a.T;
        const T* xp = static_cast<const T*>(s.x) + b * s.sb + t * s.st + h * s.sh + col;
        load<T, V>(xp, x0);
        load<T, V>(xp + a.half, x1);
        if constexpr (BWD) {
          const T* gp = static_cast<const T*>(s.dout) + out_at;
          load<T, V>(gp, g0);
          load<T, V>(gp + a.half, g1);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum += x0[i] * x0[i] + x1[i] * x1[i];
      const float inv = rsqrtf(group_sum(sum, a.lanes) * inv_d + a.eps);
      const float2* cs = table + tok * a.half + col;
      if constexpr (!BWD) {
        if (live) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 t = cs[i];
            const float y0 = x0[i] * inv * (is_q ? wq[0][i] : wk[0][i]);
            const float y1 = x1[i] * inv * (is_q ? wq[1][i] : wk[1][i]);
            x0[i] = y0 * t.x - y1 * t.y;
            x1[i] = y0 * t.y + y1 * t.x;
          }
          T* op = static_cast<T*>(s.out) + out_at;
          store<T, V>(op, x0);
          store<T, V>(op + a.half, x1);
        }
      } else {
        float dot = 0.f;
        if (live) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 t = cs[i];
            const float r0 = g0[i] * t.x + g1[i] * t.y, r1 = g1[i] * t.x - g0[i] * t.y;
            x0[i] *= inv;
            x1[i] *= inv;
            if (is_q) {
              dq[0][i] += r0 * x0[i];
              dq[1][i] += r1 * x1[i];
            } else {
              dk[0][i] += r0 * x0[i];
              dk[1][i] += r1 * x1[i];
            }
            g0[i] = r0 * (is_q ? wq[0][i] : wk[0][i]);
            g1[i] = r1 * (is_q ? wq[1][i] : wk[1][i]);
            dot += g0[i] * x0[i] + g1[i] * x1[i];
          }
        }
        dot = group_sum(dot, a.lanes) * inv_d;
        if (live) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            g0[i] = (g0[i] - x0[i] * dot) * inv;
            g1[i] = (g1[i] - x1[i] * dot) * inv;
          }
          T* op = static_cast<T*>(s.out) + out_at;
          store<T, V>(op, g0);
          store<T, V>(op + a.half, g1);
        }
      }
    }
  }
  if constexpr (BWD) {
    // the CTA's partial dw: lane groups, then warps, in a fixed order
    __syncthreads();
    float* buf = reinterpret_cast<float*>(table);   // [kWarps][2][D]
    for (int o = a.lanes; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          dq[s][i] += __shfl_xor_sync(kFull, dq[s][i], o);
          dk[s][i] += __shfl_xor_sync(kFull, dk[s][i], o);
        }
      }
    }
    if (sub == 0 && active) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          buf[(warp * 2 + 0) * a.D + col + i + s * a.half] = dq[s][i];
          buf[(warp * 2 + 1) * a.D + col + i + s * a.half] = dk[s][i];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += buf[w * 2 * a.D + i];
      a.partial[int64_t(blockIdx.x) * 2 * a.D + i] = v;
    }
  }
}

// dw: the CTAs' partials of one column, summed by a warp.
template <typename T>
__global__ void __launch_bounds__(128) norm_weight_kernel(const float* __restrict__ partial, int parts, int D,
                                                          void* dqw, int q_f32, void* dkw, int k_f32) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= 2 * D) return;
  float v = 0.f;
  for (int p = lane; p < parts; p += 32) v += partial[int64_t(p) * 2 * D + i];
  v = warp_sum(v);
  if (lane) return;
  void* out = i < D ? dqw : dkw;
  const int f32 = i < D ? q_f32 : k_f32, d = i < D ? i : i - D;
  if (f32) static_cast<float*>(out)[d] = v;
  else static_cast<T*>(out)[d] = from_f32<T>(v);
}

int max_ctas() { return sm_count() * 4; }

template <typename T, int V>
int launch(NormArgs a, bool bwd, cudaStream_t s) {
  a.lanes = next_pow2(a.half / V);
  a.lg_lanes = 0;
  while ((1 << a.lg_lanes) < a.lanes) ++a.lg_lanes;
  const int most = max_ctas();
  // one token per CTA while that leaves no CTA a second turn, four beyond
  a.tokens_per_cta = a.rows <= most ? 1 : 4;
  const int64_t work = (a.rows + a.tokens_per_cta - 1) / a.tokens_per_cta;
  const size_t table = sizeof(float2) * a.tokens_per_cta * a.half;
  if (bwd) {
    const int ctas = int(min64(work, most));
    const size_t smem = table > sizeof(float) * kWarps * 2 * a.D ? table : sizeof(float) * kWarps * 2 * a.D;
    norm_rotary_kernel<T, V, true><<<ctas, kThreads, smem, s>>>(a);
    PISA_CHECK_LAUNCH();
    norm_weight_kernel<T><<<(2 * a.D + 3) / 4, 128, 0, s>>>(a.partial, ctas, a.D, a.q.dw, a.q.w_f32, a.k.dw,
                                                            a.k.w_f32);
    PISA_CHECK_LAUNCH();
    return PISA_OK;
  }
  norm_rotary_kernel<T, V, false><<<unsigned(work), kThreads, table, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

int dispatch(const NormArgs& a, int dtype, bool bwd, cudaStream_t s) {
  // 16-byte accesses when a half row is a whole number of them, 8-byte otherwise
  if (dtype == PISA_F32) return launch<float, 4>(a, bwd, s);
  if (dtype == PISA_BF16)
    return a.half % 8 ? launch<__nv_bfloat16, 4>(a, bwd, s) : launch<__nv_bfloat16, 8>(a, bwd, s);
  return a.half % 8 ? launch<__half, 4>(a, bwd, s) : launch<__half, 8>(a, bwd, s);
}

bool rows16(const void* p, int64_t es, int64_t sb, int64_t st, int64_t sh) {
  const int64_t v = 16 / es;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && sb % v == 0 && st % v == 0 && sh % v == 0;
}

int check(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
          int64_t k_sh, const void* qw, const void* kw, const float* freq, int dtype, int w_dtype, int64_t B, int64_t T,
          int64_t Hq, int64_t H, int64_t D) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (w_dtype != dtype && w_dtype != PISA_F32) return fail(PISA_ERR_UNSUPPORTED, "norm weights must be FP32 or the tensors' type");
  if (B <= 0 || T <= 0 || Hq <= 0 || H <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (D % 8 || D > 256) return fail(PISA_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 256");
  if (B * T >= (int64_t(1) << 31) || Hq + H >= (1 << 16)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (!q || !k || !qw || !kw || !freq) return fail(PISA_ERR_INVALID, "q, k, the weights and frequency are required");
  const int64_t es = dtype == PISA_F32 ? 4 : 2;
  if (!rows16(q, es, q_sb, q_st, q_sh) || !rows16(k, es, k_sb, k_st, k_sh))
    return fail(PISA_ERR_UNSUPPORTED, "q and k rows must be 16-byte aligned");
  return PISA_OK;
}

NormArgs make_args(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                   int64_t k_sh, const void* qw, const void* kw, int w_f32, const float* freq, const int64_t* positions,
                   int64_t positions_sb, int64_t position_offset, int64_t B, int64_t T, int64_t Hq, int64_t H,
                   int64_t D, float eps) {
  NormArgs a{};
  a.q.x = q; a.q.sb = q_sb; a.q.st = q_st; a.q.sh = q_sh; a.q.w = qw; a.q.w_f32 = w_f32;
  a.k.x = k; a.k.sb = k_sb; a.k.st = k_st; a.k.sh = k_sh; a.k.w = kw; a.k.w_f32 = w_f32;
  a.freq = freq; a.positions = positions; a.pos_sb = positions_sb; a.pos_offset = position_offset;
  a.rows = B * T; a.T = int(T); a.Hq = int(Hq); a.H = int(H); a.D = int(D); a.half = int(D / 2);
  a.eps = eps;
  return a;
}

}  // namespace

}  // namespace pisa

extern "C" {

int pisa_qk_norm_rotary(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                        int64_t k_st, int64_t k_sh, const void* q_weight, const void* k_weight, int weight_dtype,
                        const float* frequency, const int64_t* positions, int64_t positions_sb,
                        int64_t position_offset, int dtype, int64_t B, int64_t T, int64_t Hq, int64_t H, int64_t D,
                        float eps, void* q_out, void* k_out, pisa_stream_t stream) {
  int rc = pisa::check(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight, frequency, dtype, weight_dtype, B,
                       T, Hq, H, D);
  if (rc) return rc;
  if (!q_out || !k_out) return pisa::fail(PISA_ERR_INVALID, "q_out and k_out are required");
  pisa::NormArgs a = pisa::make_args(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight,
                                     weight_dtype == PISA_F32, frequency, positions, positions_sb, position_offset, B,
                                     T, Hq, H, D, eps);
  a.q.out = q_out;
  a.k.out = k_out;
  return pisa::dispatch(a, dtype, false, static_cast<cudaStream_t>(stream));
}

int64_t pisa_qk_norm_rotary_bwd_workspace_bytes(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || T <= 0 || D <= 0) return -1;
  return int64_t(sizeof(float)) * 2 * D * pisa::min64(B * T, pisa::max_ctas());
}

int pisa_qk_norm_rotary_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                            int64_t k_st, int64_t k_sh, const void* dq_out, const void* dk_out, const void* q_weight,
                            const void* k_weight, int weight_dtype, const float* frequency, const int64_t* positions,
                            int64_t positions_sb, int64_t position_offset, int dtype, int64_t B, int64_t T, int64_t Hq,
                            int64_t H, int64_t D, float eps, void* dq, void* dk, void* dq_weight, void* dk_weight,
                            void* workspace, int64_t workspace_bytes, pisa_stream_t stream) {
  int rc = pisa::check(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight, frequency, dtype, weight_dtype, B,
                       T, Hq, H, D);
  if (rc) return rc;
  if (!dq_out || !dk_out || !dq || !dk || !dq_weight || !dk_weight)
    return pisa::fail(PISA_ERR_INVALID, "the gradients are required");
  if (!workspace || workspace_bytes < pisa_qk_norm_rotary_bwd_workspace_bytes(B, T, D))
    return pisa::fail(PISA_ERR_INVALID, "workspace too small");
  pisa::NormArgs a = pisa::make_args(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight,
                                     weight_dtype == PISA_F32, frequency, positions, positions_sb, position_offset, B,
                                     T, Hq, H, D, eps);
  a.q.dout = dq_out; a.q.out = dq; a.q.dw = dq_weight;
  a.k.dout = dk_out; a.k.out = dk; a.k.dw = dk_weight;
  a.partial = static_cast<float*>(workspace);
  return pisa::dispatch(a, dtype, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

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
// in registers and a row's sums are a few shuffles.  A CTA's turn is a run of
// tokens of one batch row: their cosines and sines are computed once into
// shared memory and serve all heads, and offsets inside a turn are two
// 32-bit products.  Arithmetic is on pairs (f32x2): with single operations the
// forward was bound by instruction issue (337 instructions per warp and step).
// Each warp requests U rows before it works on the first.
// Lanes keep their columns over all rows they visit, so dw accumulates in
// registers; each CTA stores one partial row and a second launch adds the
// partials in a fixed order (no atomics: results do not vary from run to run).
//
// Measured: 32768 tokens of 32 query and 8 key heads of 128, bf16, forward: 126
// us, 5.3 TB/s; training block of four sequences of 4096, 16 + 16 heads of 64:
// forward 30 us (4.5 TB/s), backward 52 us (3.9 TB/s) and 2.6 us for dw.  Rows
// in flight per warp and CTAs per SM, forward of the first and forward and
// backward of the second: U = 2 with 4 CTAs (forward) and 2 (backward) as kept;
// U = 2 with 3: 130 us; U = 3 with 3: 122, 36 and 56 us; U = 4 with 3: 129 us.
#include <cmath>

#include "dense_tc.cuh"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct NormSide {
  const void* x;
  int64_t sb;
  int st, sh;           // element strides of x
  const void* dout;     // backward: contiguous gradient of out
  void* out;            // contiguous out, or dx
  const void* w;
  void* dw;
  int w_f32;            // weight is fp32 (else the tensors' type)
  int heads;
  FastDiv groups;       // warp steps of a token
  int ctas;             // backward: CTAs of this side
};

struct NormArgs {
  NormSide side[2];      // q, k
  const float* freq;
  const int64_t* positions;
  int64_t pos_sb, pos_offset;
  int T, D, half, lg_lanes;              // lanes per head row: a power of two
  int tokens, turns;                     // tokens of a turn, turns in all
  FastDiv per_row;                       // turns of a batch row
  float eps;
  float* partial;        // backward: [CTAs of q, then of k][D]
};

// V elements as loaded, and as pairs of floats.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { uint32_t w[sizeof(T) * V / 4]; };

template <typename T, int V>
__device__ __forceinline__ void widen(const Pack<T, V>& r, float2 (&v)[V / 2]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      v[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      v[i] = make_float2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
    } else {
      v[i] = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float2 (&v)[V / 2]) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      r.w[2 * i] = __float_as_uint(v[i].x);
      r.w[2 * i + 1] = __float_as_uint(v[i].y);
    } else {
      r.w[i] = pack2<T>(v[i].x, v[i].y);
    }
  }
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
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }

// Cosines and sines of `count` tokens from t0 of batch row b, ordered so that
// the lanes of a row read consecutive 16-byte words (cos, cos, sin, sin): pairs
// V c + i and V c + i + 1 (i even) of a token are word i / 2 * lanes + c.
template <int V>
__device__ __forceinline__ void fill_angles(const NormArgs& a, int b, int t0, int count, int lanes, float* table) {
  const int lg = a.lg_lanes + (V == 8 ? 3 : 2);      // pairs of a token, padded to lanes * V
  for (int i = threadIdx.x; i < count << lg; i += kThreads) {
    const int tok = i >> lg, p = i - (tok << lg);
    if (p >= a.half) continue;
    const int64_t pos = a.positions ? a.positions[b * a.pos_sb + t0 + tok] : a.pos_offset + t0 + tok;
    float s, c;
    sincosf(float(pos) * a.freq[p], &s, &c);
    float* at = table + (tok << (lg + 1)) + (p % V / 2 * lanes + p / V) * 4 + (p & 1);
    at[0] = c;
    at[2] = s;
  }
}

// The rows of one side in one turn.
template <typename T, int V, bool BWD>
__device__ __forceinline__ void turn_rows(const NormArgs& a, const NormSide& s, int b, int t0, int count, const float* table,
                                          const float2 (&w)[2][V / 2], float2 (&dw)[2][V / 2]) {
  constexpr int U = 2;                             // rows requested ahead
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = 1 << a.lg_lanes, per_warp = 32 >> a.lg_lanes;   // head rows of one warp step
  const int sub = lane >> a.lg_lanes, c = lane & (lanes - 1), col = c * V;
  const int heads = s.heads, groups = int(s.groups.d);
  const bool active = col < a.half;                // lanes past the row's columns idle
  const T* x_base = static_cast<const T*>(s.x) + b * s.sb + int64_t(t0) * s.st + col;
  const int64_t out_base = (int64_t(b) * a.T + t0) * heads * a.D + col;
  T* o_base = static_cast<T*>(s.out) + out_base;
  const T* g_base = static_cast<const T*>(s.dout) + out_base;
  const int step_tok = int(s.groups.div(kWarps)), step_grp = kWarps - step_tok * groups;
  int tok = int(s.groups.div(uint32_t(warp))), grp = warp - tok * groups;
  const float inv_d = 1.f / float(a.D);
  while (tok < count) {
    Pack<T, V> x[U][2], g[BWD ? U : 1][2];
    int token[U], head[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      head[u] = grp * per_warp + sub;
      live[u] = tok < count && active && head[u] < heads;
      // rows that are not there are zeros (they add nothing to dw) and use the first token's angles
      token[u] = live[u] ? tok : 0;
      x[u][0] = x[u][1] = Pack<T, V>{};
      if constexpr (BWD) g[u][0] = g[u][1] = Pack<T, V>{};
      if (live[u]) {
        const T* xp = x_base + int64_t(tok) * s.st + int64_t(head[u]) * s.sh;
        x[u][0] = *reinterpret_cast<const Pack<T, V>*>(xp);
        x[u][1] = *reinterpret_cast<const Pack<T, V>*>(xp + a.half);
        if constexpr (BWD) {
          const T* gp = g_base + int64_t(tok * heads + head[u]) * a.D;
          g[u][0] = *reinterpret_cast<const Pack<T, V>*>(gp);
          g[u][1] = *reinterpret_cast<const Pack<T, V>*>(gp + a.half);
        }
      }
      tok += step_tok;
      grp += step_grp;
      if (grp >= groups) {
        grp -= groups;
        ++tok;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 x0[V / 2], x1[V / 2], sum = make_float2(0.f, 0.f);
      widen<T, V>(x[u][0], x0);
      widen<T, V>(x[u][1], x1);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) sum = tc::fma2(x1[i], x1[i], tc::fma2(x0[i], x0[i], sum));
      const float size = group_sum(sum.x + sum.y, lanes) * inv_d + a.eps;
      const float inv = live[u] ? rsqrtf(size) : 0.f;   // rows that are not there add nothing, also with eps 0
      const float2 inv2 = make_float2(inv, inv);
      const float4* cs = reinterpret_cast<const float4*>(table + token[u] * 2 * lanes * V) + (active ? c : 0);
      T* op = o_base + int64_t(token[u] * heads + head[u]) * a.D;
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float4 t = cs[i * lanes];
          const float2 co = make_float2(t.x, t.y), si = make_float2(t.z, t.w);
          const float2 y0 = mul2(mul2(x0[i], inv2), w[0][i]), y1 = mul2(mul2(x1[i], inv2), w[1][i]);
          x0[i] = tc::fma2(neg2(y1), si, mul2(y0, co));
          x1[i] = tc::fma2(y1, co, mul2(y0, si));
        }
        if (live[u]) {
          store<T, V>(op, x0);
          store<T, V>(op + a.half, x1);
        }
      } else {
        float2 g0[V / 2], g1[V / 2], dot = make_float2(0.f, 0.f);
        widen<T, V>(g[u][0], g0);
        widen<T, V>(g[u][1], g1);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float4 t = cs[i * lanes];
          const float2 co = make_float2(t.x, t.y), si = make_float2(t.z, t.w);
          const float2 r0 = tc::fma2(g1[i], si, mul2(g0[i], co)), r1 = tc::fma2(neg2(g0[i]), si, mul2(g1[i], co));
          x0[i] = mul2(x0[i], inv2);
          x1[i] = mul2(x1[i], inv2);
          dw[0][i] = tc::fma2(r0, x0[i], dw[0][i]);
          dw[1][i] = tc::fma2(r1, x1[i], dw[1][i]);
          g0[i] = mul2(r0, w[0][i]);
          g1[i] = mul2(r1, w[1][i]);
          dot = tc::fma2(g1[i], x1[i], tc::fma2(g0[i], x0[i], dot));
        }
        const float mean = group_sum(dot.x + dot.y, lanes) * -inv_d;
        const float2 mean2 = make_float2(mean, mean);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          g0[i] = mul2(tc::fma2(x0[i], mean2, g0[i]), inv2);
          g1[i] = mul2(tc::fma2(x1[i], mean2, g1[i]), inv2);
        }
        if (live[u]) {
          store<T, V>(op, g0);
          store<T, V>(op + a.half, g1);
        }
      }
    }
  }
}

// Forward: a CTA per turn does q and k.  Backward: the CTAs of each side take
// its turns in steps (one side's dw at a time fits the registers).
template <typename T, int V, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? 2 : 4) norm_rotary_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ __align__(16) float table[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = 1 << a.lg_lanes;
  const int col = (lane & (lanes - 1)) * V;
  const int first = BWD && int(blockIdx.x) >= a.side[0].ctas ? 1 : 0, end = BWD ? first + 1 : 2;
  const int cta = int(blockIdx.x) - (BWD && first ? a.side[0].ctas : 0);
  const int stride = BWD ? a.side[first].ctas : int(gridDim.x);
  float2 w[2][V / 2], dw[2][V / 2];
  auto load_weights = [&](const NormSide& s) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const int d = col + 2 * i + x * a.half;
        w[x][i] = col < a.half ? make_float2(weight_at<T>(s, d), weight_at<T>(s, d + 1)) : make_float2(0.f, 0.f);
        dw[x][i] = make_float2(0.f, 0.f);
      }
    }
  };
  if constexpr (BWD) load_weights(a.side[first]);
  for (int turn = cta; turn < a.turns; turn += stride) {
    const int b = int(a.per_row.div(uint32_t(turn))), t0 = (turn - b * int(a.per_row.d)) * a.tokens;
    const int count = min(a.tokens, a.T - t0);
    __syncthreads();
    fill_angles<V>(a, b, t0, count, lanes, table);
    __syncthreads();
    for (int x = first; x < end; ++x) {
      if constexpr (!BWD) load_weights(a.side[x]);
      turn_rows<T, V, BWD>(a, a.side[x], b, t0, count, table, w, dw);
    }
  }
  if constexpr (BWD) {
    // the CTA's partial dw: lane groups, then warps, in a fixed order
    __syncthreads();
    float* buf = table;   // [kWarps][D]
    for (int o = lanes; o < 32; o <<= 1) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          dw[x][i].x += __shfl_xor_sync(kFull, dw[x][i].x, o);
          dw[x][i].y += __shfl_xor_sync(kFull, dw[x][i].y, o);
        }
      }
    }
    if (lane < lanes && col < a.half) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          buf[warp * a.D + col + 2 * i + x * a.half] = dw[x][i].x;
          buf[warp * a.D + col + 2 * i + 1 + x * a.half] = dw[x][i].y;
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) v += buf[x * a.D + i];
      a.partial[int64_t(blockIdx.x) * a.D + i] = v;
    }
  }
}

// dw: the CTAs' partials of one column, summed by a warp.
template <typename T>
__global__ void __launch_bounds__(128) norm_weight_kernel(const __grid_constant__ NormArgs a) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= 2 * a.D) return;
  const int which = i < a.D ? 0 : 1, d = which ? i - a.D : i, begin = which ? a.side[0].ctas : 0;
  float v = 0.f;
#pragma unroll 4
  for (int p = lane; p < a.side[which].ctas; p += 32) v += a.partial[int64_t(begin + p) * a.D + d];
  v = warp_sum(v);
  if (lane) return;
  if (a.side[which].w_f32) static_cast<float*>(a.side[which].dw)[d] = v;
  else static_cast<T*>(a.side[which].dw)[d] = from_f32<T>(v);
}

int max_ctas() { return sm_count() * 4; }

template <typename T, int V>
int launch(NormArgs a, int64_t B, bool bwd, cudaStream_t s) {
  const int lanes = next_pow2(a.half / V), sms = sm_count();
  while ((1 << a.lg_lanes) < lanes) ++a.lg_lanes;
  int steps = 0;   // warp steps of a token
  for (int x = 0; x < 2; ++x) {
    const int groups = (a.side[x].heads + (32 >> a.lg_lanes) - 1) >> (5 - a.lg_lanes);
    a.side[x].groups = FastDiv::make(uint32_t(groups));
    steps += groups;
  }
  // a turn of about sixteen rows per warp, with at most 16 KB of angles, while
  // there are tokens for two CTAs per SM; single tokens for the smallest calls
  const int64_t most = min64(min64(16 * kWarps / steps, 2048 / (lanes * V)), B * a.T / (2 * sms));
  const int64_t per_row = (a.T + (most < 1 ? 1 : most) - 1) / (most < 1 ? 1 : most);
  a.tokens = int((a.T + per_row - 1) / per_row);
  a.per_row = FastDiv::make(uint32_t((a.T + a.tokens - 1) / a.tokens));
  a.turns = int(B * a.per_row.d);
  size_t smem = sizeof(float2) * a.tokens * lanes * V;
  if (!bwd) {
    norm_rotary_kernel<T, V, false><<<unsigned(a.turns), kThreads, smem, s>>>(a);
    PISA_CHECK_LAUNCH();
    return PISA_OK;
  }
  if (smem < sizeof(float) * kWarps * a.D) smem = sizeof(float) * kWarps * a.D;
  // the CTAs of two per SM, shared out by the sides' rows
  const int64_t heads = a.side[0].heads + a.side[1].heads;
  for (int x = 0; x < 2; ++x) {
    const int64_t share = (2 * sms * a.side[x].heads + heads - 1) / heads;
    a.side[x].ctas = int(min64(a.turns, share));
  }
  norm_rotary_kernel<T, V, true><<<unsigned(a.side[0].ctas + a.side[1].ctas), kThreads, smem, s>>>(a);
  PISA_CHECK_LAUNCH();
  norm_weight_kernel<T><<<(2 * a.D + 3) / 4, 128, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

int dispatch(const NormArgs& a, int64_t B, int dtype, bool bwd, cudaStream_t s) {
  // 16-byte accesses when a half row is a whole number of them, 8-byte otherwise
  if (dtype == PISA_F32) return launch<float, 4>(a, B, bwd, s);
  if (dtype == PISA_BF16)
    return a.half % 8 ? launch<__nv_bfloat16, 4>(a, B, bwd, s) : launch<__nv_bfloat16, 8>(a, B, bwd, s);
  return a.half % 8 ? launch<__half, 4>(a, B, bwd, s) : launch<__half, 8>(a, B, bwd, s);
}

// The stride of a dimension of one element may hold anything.
bool rows16(const void* p, int64_t es, int64_t B, int64_t T, int64_t H, int64_t sb, int64_t st, int64_t sh) {
  const int64_t v = 16 / es;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (B == 1 || sb % v == 0) && (T == 1 || st % v == 0) &&
         (H == 1 || sh % v == 0);
}

int check(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
          int64_t k_sh, const void* qw, const void* kw, const float* freq, int dtype, int w_dtype, int64_t B, int64_t T,
          int64_t Hq, int64_t H, int64_t D, float eps) {
  if (!(eps >= 0.f) || std::isinf(eps)) return fail(PISA_ERR_INVALID, "eps must be finite and not negative");
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (w_dtype != dtype && w_dtype != PISA_F32) return fail(PISA_ERR_UNSUPPORTED, "norm weights must be FP32 or the tensors' type");
  if (B <= 0 || T <= 0 || Hq <= 0 || H <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (D % 8 || D > 256) return fail(PISA_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 256");
  if (B * T >= (int64_t(1) << 30) || Hq + H >= (1 << 16)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  constexpr int64_t wide = int64_t(1) << 31;
  if ((T > 1 && (q_st >= wide || k_st >= wide)) || (Hq > 1 && q_sh >= wide) || (H > 1 && k_sh >= wide))
    return fail(PISA_ERR_UNSUPPORTED, "token and head strides must be below 2^31 elements");
  if (!q || !k || !qw || !kw || !freq) return fail(PISA_ERR_INVALID, "q, k, the weights and frequency are required");
  const int64_t es = dtype == PISA_F32 ? 4 : 2;
  if (!rows16(q, es, B, T, Hq, q_sb, q_st, q_sh) || !rows16(k, es, B, T, H, k_sb, k_st, k_sh))
    return fail(PISA_ERR_UNSUPPORTED, "q and k rows must be 16-byte aligned");
  return PISA_OK;
}

NormArgs make_args(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                   int64_t k_sh, const void* qw, const void* kw, int w_f32, const float* freq, const int64_t* positions,
                   int64_t positions_sb, int64_t position_offset, int64_t T, int64_t Hq, int64_t H,
                   int64_t D, float eps) {
  NormArgs a{};
  NormSide& sq = a.side[0];
  NormSide& sk = a.side[1];
  sq.x = q; sq.sb = q_sb; sq.st = int(q_st); sq.sh = int(q_sh); sq.w = qw; sq.w_f32 = w_f32; sq.heads = int(Hq);
  sk.x = k; sk.sb = k_sb; sk.st = int(k_st); sk.sh = int(k_sh); sk.w = kw; sk.w_f32 = w_f32; sk.heads = int(H);
  a.freq = freq; a.positions = positions; a.pos_sb = positions_sb; a.pos_offset = position_offset;
  a.T = int(T); a.D = int(D); a.half = int(D / 2);
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
                       T, Hq, H, D, eps);
  if (rc) return rc;
  if (!q_out || !k_out) return pisa::fail(PISA_ERR_INVALID, "q_out and k_out are required");
  pisa::NormArgs a = pisa::make_args(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight,
                                     weight_dtype == PISA_F32, frequency, positions, positions_sb, position_offset,
                                     T, Hq, H, D, eps);
  a.side[0].out = q_out;
  a.side[1].out = k_out;
  return pisa::dispatch(a, B, dtype, false, static_cast<cudaStream_t>(stream));
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
                       T, Hq, H, D, eps);
  if (rc) return rc;
  if (!dq_out || !dk_out || !dq || !dk || !dq_weight || !dk_weight)
    return pisa::fail(PISA_ERR_INVALID, "the gradients are required");
  if (!workspace || workspace_bytes < pisa_qk_norm_rotary_bwd_workspace_bytes(B, T, D))
    return pisa::fail(PISA_ERR_INVALID, "workspace too small");
  pisa::NormArgs a = pisa::make_args(q, q_sb, q_st, q_sh, k, k_sb, k_st, k_sh, q_weight, k_weight,
                                     weight_dtype == PISA_F32, frequency, positions, positions_sb, position_offset,
                                     T, Hq, H, D, eps);
  a.side[0].dout = dq_out; a.side[0].out = dq; a.side[0].dw = dq_weight;
  a.side[1].dout = dk_out; a.side[1].out = dk; a.side[1].dw = dk_weight;
  a.partial = static_cast<float*>(workspace);
  return pisa::dispatch(a, B, dtype, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

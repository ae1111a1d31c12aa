// The gated product of a feed-forward layer, its inputs kept in 8 bits for the
// backward, and its form for 8-bit products.
//
//   a = silu(g) u = g s(g) u,   s(g) = 1 / (1 + exp(-g)).
// Backward from da, with g and u as they were kept:
//   du = da g s(g),   dg = da u s(g) (1 + g (1 - s(g))).
// Kept in 8 bits, every group of 128 elements of a row has one fp32 scale
// (Scale8); the backward reads the bytes and widens them in registers, so the
// 16-bit inputs need not live until then.
//
// Bound by HBM: per element of a 16-bit layer the forward moves 4 bytes in and
// 2 out, and 2 more for the kept bytes; the backward 4 in and 4 out.  Sixteen
// threads share a group: 8 elements each, a group's maximum is four shuffles.
// Close behind is instruction issue: with the group's index by 64-bit division,
// single operations and a quotient per thread the two passes took 75 and 71 us
// for 16384 x 2816 in bf16, now 58 and 59 (6.3 TB/s); 8191 x 11264 in fp16 takes
// 112 and 113, and 16384 x 2817, whose rows are read element by element, 106 and
// 148.  Teams with one group and few bytes in flight: 73 us, with two 68.  Without
// kept bytes 16384 x 2816 takes 38 and 70 us in bf16, 86 and 140 in fp32; with them
// 118 and 122 in fp32; as 8-bit rows 48 (bf16) and 79 (fp32).  fp32 rows of more than
// 16384 spill 56 to 80 bytes per thread (4096 x 32768: 242 us, 5.0 TB/s).
// Arithmetic is fp32; exponentials and reciprocals are the exact ones for fp32 and
// the fast forms for 16-bit tensors.  There s(x) is off by about 2^-24 (8 + |x|) of
// itself (the exponent's product is rounded), 5e-6 at x = -80, before a rounding of
// 2^-9 or 2^-12; below x = -87.3, where s(x) is under the smallest normal number, it
// is 0.
#include "rows.cuh"

namespace pisa {

namespace {

struct GluArgs {
  const void* g;
  int64_t g_st;
  const void* u;
  int64_t u_st;
  int64_t rows;
  uint32_t items;         // groups of all rows
  int D;
  FastDiv groups;         // groups of 128 of a row
  void* out;              // contiguous [rows, D]
  int8_t* g_q;            // kept bytes, rows q_st apart, and scales [rows, groups]
  int8_t* u_q;
  int64_t q_st;
  float* g_scale;
  float* u_scale;
  // backward
  const void* dout;
  int64_t dout_st;
  void* dg;
  void* du;
  // 8-bit rows of the product
  int8_t* a_q;
  int64_t a_q_st;
  float* a_scale;
};

__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// s(x) of a pair.
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  if constexpr (std::is_same<T, float>::value) {
    return make_float2(1.f / (1.f + expf(-x.x)), 1.f / (1.f + expf(-x.y)));
  } else {
    constexpr float kLog2e = 1.4426950408889634f;
    const float2 y = pair_mul(x, both(-kLog2e)), z = pair_add(make_float2(fast_ex2(y.x), fast_ex2(y.y)), both(1.f));
    return make_float2(fast_rcp(z.x), fast_rcp(z.y));
  }
}

// Maximum over the sixteen threads of a group, NaN if any is.
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = larger(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

constexpr int kGluThreads = 256, kGluTeams = kGluThreads / 16;

// Where group `u` of a team's U lies; a group past the last has no elements.
template <int U>
struct GluGroup {
  uint32_t at;
  int64_t row;
  int first, width;
  __device__ __forceinline__ GluGroup(const GluArgs& a, int u) {
    const uint32_t item = (blockIdx.x * U + u) * kGluTeams + (threadIdx.x >> 4);
    const bool live = item < a.items;
    at = live ? item : 0;
    row = a.groups.div(at);
    first = int(at - uint32_t(row) * a.groups.d) * kGroup;
    width = live ? min(kGroup, a.D - first) : 0;
  }
};

// Sixteen threads per group; all of a thread's loads are under way before its first use.
template <typename T, int U, bool A, bool KEEP>
__global__ void __launch_bounds__(kGluThreads) glu_fwd_kernel(const __grid_constant__ GluArgs a) {
  const int t = threadIdx.x & 15;
  Raw8<T> gr[U], ur[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const GluGroup<U> n(a, i);
    gr[i] = load_piece<T, 16, A>(static_cast<const T*>(a.g) + n.row * a.g_st + n.first, 0, t, n.width);
    ur[i] = load_piece<T, 16, A>(static_cast<const T*>(a.u) + n.row * a.u_st + n.first, 0, t, n.width);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const GluGroup<U> n(a, i);
    float g[8], u[8], o[8];
    widen8<T>(gr[i], g);
    widen8<T>(ur[i], u);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = pair_at(g, k);
      set_pair(o, k, pair_mul(pair_mul(x, sigmoid2<T>(x)), pair_at(u, k)));
    }
    store_piece<T, 16, A>(static_cast<T*>(a.out) + n.row * a.D + n.first, 0, t, n.width, o);
    if constexpr (KEEP) {
      const float top_g = group_max(largest8<T>(gr[i], g)), top_u = group_max(largest8<T>(ur[i], u));
      // Scale8 of both: its four quotients are four lanes' (a quotient costs more than a shuffle)
      const float m = fmaxf(t & 1 ? top_u : top_g, kTiny), r = __fdiv_rn(t & 2 ? m : 127.f, t & 2 ? 127.f : m);
      const int team = threadIdx.x & 16;
      const bool fine_g = top_g < INFINITY, fine_u = top_u < INFINITY;
      store_piece_s8<T, 16, A>(a.g_q + n.row * a.q_st + n.first, 0, t, n.width, g, fine_g, __shfl_sync(kFull, r, team));
      store_piece_s8<T, 16, A>(a.u_q + n.row * a.q_st + n.first, 0, t, n.width, u, fine_u, __shfl_sync(kFull, r, team + 1));
      if (n.width && (t & ~1) == 2) (t & 1 ? a.u_scale : a.g_scale)[n.at] = (t & 1 ? fine_u : fine_g) ? r : __int_as_float(0x7fffffff);
    }
  }
}

template <typename T, int U, bool A, bool KEPT>
__global__ void __launch_bounds__(kGluThreads) glu_bwd_kernel(const __grid_constant__ GluArgs a) {
  const int t = threadIdx.x & 15;
  Raw8<T> dr[U], gr[U], ur[U];
  uint2 gq[U], uq[U];
  float gs[U], us[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const GluGroup<U> n(a, i);
    dr[i] = load_piece<T, 16, A>(static_cast<const T*>(a.dout) + n.row * a.dout_st + n.first, 0, t, n.width);
    if constexpr (KEPT) {
      gq[i] = load_piece_s8<T, 16, A>(a.g_q + n.row * a.q_st + n.first, t, n.width);
      uq[i] = load_piece_s8<T, 16, A>(a.u_q + n.row * a.q_st + n.first, t, n.width);
      gs[i] = a.g_scale[n.at];
      us[i] = a.u_scale[n.at];
    } else {
      gr[i] = load_piece<T, 16, A>(static_cast<const T*>(a.g) + n.row * a.g_st + n.first, 0, t, n.width);
      ur[i] = load_piece<T, 16, A>(static_cast<const T*>(a.u) + n.row * a.u_st + n.first, 0, t, n.width);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const GluGroup<U> n(a, i);
    float d[8], g[8], u[8], o[8];
    if constexpr (KEPT) {
      widen8_s8(gq[i], gs[i], g);
      widen8_s8(uq[i], us[i], u);
    } else {
      widen8<T>(gr[i], g);
      widen8<T>(ur[i], u);
    }
    widen8<T>(dr[i], d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = pair_at(g, k), s = sigmoid2<T>(x), y = pair_mul(x, s), v = pair_at(u, k), e = pair_at(d, k);
      if (a.out) set_pair(o, k, pair_mul(y, v));
      // s (1 + x (1 - s)) with 1 - s as 1 + (-1) s
      const float2 slope = pair_mul(s, pair_fma(x, pair_fma(s, both(-1.f), both(1.f)), both(1.f)));
      set_pair(u, k, pair_mul(pair_mul(e, v), slope));
      set_pair(g, k, pair_mul(e, y));
    }
    store_piece<T, 16, A>(static_cast<T*>(a.dg) + n.row * a.D + n.first, 0, t, n.width, u);
    store_piece<T, 16, A>(static_cast<T*>(a.du) + n.row * a.D + n.first, 0, t, n.width, g);
    if (a.out) store_piece<T, 16, A>(static_cast<T*>(a.out) + n.row * a.D + n.first, 0, t, n.width, o);
  }
}

// The product in 8 bits with one scale per row: a team holds the row.
template <typename T, int TPR, int NV, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) glu_row_kernel(const __grid_constant__ GluArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1;
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x % TPR, D = a.D;
  const int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TPR;
  if (row >= a.rows) return;                      // a whole warp
  Raw8<T> g[NV], u[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    g[j] = load_piece<T, TPR, A>(static_cast<const T*>(a.g) + row * a.g_st, j, t, D);
    u[j] = load_piece<T, TPR, A>(static_cast<const T*>(a.u) + row * a.u_st, j, t, D);
  }
  float o[NV][8], top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[8];
    widen8<T>(g[j], f);
    widen8<T>(u[j], o[j]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = pair_at(f, k);
      set_pair(o[j], k, pair_mul(pair_mul(x, sigmoid2<T>(x)), pair_at(o[j], k)));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = larger(top, fabsf(o[j][e]));
  }
  top = team_reduce<TPR, true>(top, red, set);
  const Scale8 s(top);
  int8_t* qr = a.a_q + row * a.a_q_st;
#pragma unroll
  for (int j = 0; j < NV; ++j) store_piece_s8<T, TPR, A>(qr, j, t, D, o[j], top < INFINITY, s.inv);
  if (t == 0) a.a_scale[row] = s.scale;
}

template <typename T, int TPR, int NV>
int launch_row(const GluArgs& a, bool aligned, cudaStream_t s) {
  constexpr int threads = TPR < 128 ? 128 : TPR, teams = threads / TPR;
  const unsigned ctas = unsigned((a.rows + teams - 1) / teams);
  if (aligned) glu_row_kernel<T, TPR, NV, true><<<ctas, threads, 0, s>>>(a);
  else glu_row_kernel<T, TPR, NV, false><<<ctas, threads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int rows8(const GluArgs& a, bool aligned, cudaStream_t s) {
  if (a.D <= 256) return launch_row<T, 32, 1>(a, aligned, s);
  if (a.D <= 1024) return launch_row<T, 128, 1>(a, aligned, s);
  if (a.D <= 4096) return launch_row<T, 256, 2>(a, aligned, s);
  if (a.D <= 16384) return launch_row<T, 512, 4>(a, aligned, s);
  return launch_row<T, 1024, 4>(a, aligned, s);
}

template <typename T, int U, bool KEEP, bool BWD>
int launch_groups(const GluArgs& a, bool aligned, cudaStream_t s) {
  constexpr int64_t per = kGluTeams * U;
  const unsigned ctas = unsigned((a.items + per - 1) / per);
  if constexpr (BWD) {
    if (aligned) glu_bwd_kernel<T, U, true, KEEP><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_bwd_kernel<T, U, false, KEEP><<<ctas, kGluThreads, 0, s>>>(a);
  } else {
    if (aligned) glu_fwd_kernel<T, U, true, KEEP><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_fwd_kernel<T, U, false, KEEP><<<ctas, kGluThreads, 0, s>>>(a);
  }
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

// Four groups per team where that still gives every SM four CTAs, else one.
template <typename T, bool BWD>
int groups(const GluArgs& a, bool aligned, cudaStream_t s) {
  const bool many = a.items >= uint32_t(4 * kGluTeams * 4 * sm_count());
  if (a.g_q) return many ? launch_groups<T, 4, true, BWD>(a, aligned, s) : launch_groups<T, 1, true, BWD>(a, aligned, s);
  return many ? launch_groups<T, 4, false, BWD>(a, aligned, s) : launch_groups<T, 1, false, BWD>(a, aligned, s);
}

template <typename T>
int fwd(const GluArgs& a, bool aligned, cudaStream_t s) {
  return a.a_q ? rows8<T>(a, aligned, s) : groups<T, false>(a, aligned, s);
}

template <typename T>
int bwd(const GluArgs& a, bool aligned, cudaStream_t s) {
  return groups<T, true>(a, aligned, s);
}

int check(int dtype, int64_t rows, int64_t D) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (rows <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (rows >= (int64_t(1) << 31) || D >= (int64_t(1) << 30) || rows * ((D + kGroup - 1) / kGroup) >= (int64_t(1) << 31) - 256)
    return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  return PISA_OK;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

}  // namespace pisa

extern "C" {

int pisa_swiglu(const void* gate, int64_t gate_st, const void* up, int64_t up_st, int dtype, int64_t rows, int64_t D, void* out,
                int8_t* gate_q, int8_t* up_q, int64_t q_st, float* gate_scale, float* up_scale, int8_t* out_q, int64_t out_q_st,
                float* out_scale, pisa_stream_t stream) {
  using namespace pisa;
  if (int rc = check(dtype, rows, D)) return rc;
  if (!gate || !up) return fail(PISA_ERR_INVALID, "gate and up are required");
  if (out_q ? (out || gate_q || !out_scale) : !out)
    return fail(PISA_ERR_INVALID, "the product is written in its type, with kept bytes or without, or in 8 bits");
  if ((gate_q || up_q) && (!gate_q || !up_q || !gate_scale || !up_scale))
    return fail(PISA_ERR_INVALID, "kept bytes and scales come together");
  if (out_q && D > 32768) return fail(PISA_ERR_UNSUPPORTED, "8-bit rows of more than 32768 elements are not supported");
  if ((gate_q && (!rows_on16(gate_q, rows, q_st) || !rows_on16(up_q, rows, q_st))) || (out_q && !rows_on16(out_q, rows, out_q_st)))
    return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must start on 16 bytes");
  GluArgs a{};
  a.g = gate; a.g_st = gate_st; a.u = up; a.u_st = up_st; a.rows = rows; a.D = int(D);
  a.groups = FastDiv::make(uint32_t((D + kGroup - 1) / kGroup)); a.items = uint32_t(rows) * a.groups.d;
  a.out = out; a.g_q = gate_q; a.u_q = up_q; a.q_st = q_st; a.g_scale = gate_scale; a.u_scale = up_scale;
  a.a_q = out_q; a.a_q_st = out_q_st; a.a_scale = out_scale;
  const int es = dtype == PISA_F32 ? 4 : 2;
  const bool aligned = D % 8 == 0 && rows_on16(gate, rows, gate_st * es) && rows_on16(up, rows, up_st * es) && on16(out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PISA_F32) return fwd<float>(a, aligned, s);
  if (dtype == PISA_BF16) return fwd<__nv_bfloat16>(a, aligned, s);
  return fwd<__half>(a, aligned, s);
}

int pisa_swiglu_bwd(const void* dout, int64_t dout_st, const void* gate, int64_t gate_st, const void* up, int64_t up_st,
                    const int8_t* gate_q, const int8_t* up_q, int64_t q_st, const float* gate_scale, const float* up_scale,
                    int dtype, int64_t rows, int64_t D, void* dgate, void* dup, void* out, pisa_stream_t stream) {
  using namespace pisa;
  if (int rc = check(dtype, rows, D)) return rc;
  if (gate_q ? (!up_q || !gate_scale || !up_scale) : (!gate || !up))
    return fail(PISA_ERR_INVALID, "gate and up are required, or their kept bytes and scales");
  if (!dout || !dgate || !dup) return fail(PISA_ERR_INVALID, "the gradients are required");
  if (gate_q && (!rows_on16(gate_q, rows, q_st) || !rows_on16(up_q, rows, q_st)))
    return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must start on 16 bytes");
  GluArgs a{};
  a.g = gate; a.g_st = gate_st; a.u = up; a.u_st = up_st; a.rows = rows; a.D = int(D);
  a.groups = FastDiv::make(uint32_t((D + kGroup - 1) / kGroup)); a.items = uint32_t(rows) * a.groups.d;
  a.out = out; a.g_q = const_cast<int8_t*>(gate_q); a.u_q = const_cast<int8_t*>(up_q); a.q_st = q_st;
  a.g_scale = const_cast<float*>(gate_scale); a.u_scale = const_cast<float*>(up_scale);
  a.dout = dout; a.dout_st = dout_st; a.dg = dgate; a.du = dup;
  const int es = dtype == PISA_F32 ? 4 : 2;
  const bool aligned = D % 8 == 0 && rows_on16(dout, rows, dout_st * es) && on16(dgate) && on16(dup) && on16(out) &&
                       (gate_q || (rows_on16(gate, rows, gate_st * es) && rows_on16(up, rows, up_st * es)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PISA_F32) return bwd<float>(a, aligned, s);
  if (dtype == PISA_BF16) return bwd<__nv_bfloat16>(a, aligned, s);
  return bwd<__half>(a, aligned, s);
}

}  // extern "C"

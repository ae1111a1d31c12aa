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
// Arithmetic is fp32; exponentials and reciprocals are the fast forms for
// 16-bit tensors (errors of a few 2^-22 before a rounding of 2^-9 or 2^-12) and
// the exact ones for fp32.
#include "rows.cuh"

namespace pisa {

namespace {

struct GluArgs {
  const void* g;
  int64_t g_st;
  const void* u;
  int64_t u_st;
  int64_t rows;
  int D;
  uint32_t groups;        // groups of 128 of a row
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

template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (std::is_same<T, float>::value) return 1.f / (1.f + expf(-x));
  else return __fdividef(1.f, 1.f + __expf(-x));   // 0 where the sum passes 2^126
}

// Maximum over the sixteen threads of a group, NaN if any is.
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

__device__ __forceinline__ float largest8(const float (&f)[8]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(f[e]));
  return top;
}

// The eight kept values of a thread.  A group of a row is a row of 128 to its sixteen threads.
template <bool A>
__device__ __forceinline__ void load8(const int8_t* q, float scale, int t, int width, float (&f)[8]) {
  uint2 r = make_uint2(0, 0);
  if constexpr (A) {
    if (t * 8 < width) asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(q + t * 8));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<16, A>(0, e, t);
      const uint32_t b = c < width ? uint8_t(q[c]) : 0;
      if (e < 4) r.x |= b << (8 * e);
      else r.y |= b << (8 * (e - 4));
    }
  }
  float lo[4], hi[4];
  unpack_s8(r.x, lo);
  unpack_s8(r.y, hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = lo[e] * scale;
    f[4 + e] = hi[e] * scale;
  }
}

constexpr int kGluThreads = 256;

// Sixteen threads per group of a row; whole warps run on (the maxima need them) with nothing to load or store.
template <typename T, bool A, bool KEEP>
__global__ void __launch_bounds__(kGluThreads) glu_fwd_kernel(const __grid_constant__ GluArgs a) {
  const int t = threadIdx.x & 15;
  const int64_t item = int64_t(blockIdx.x) * (kGluThreads / 16) + (threadIdx.x >> 4);
  const bool live = item < a.rows * a.groups;
  const uint64_t at = live ? uint64_t(item) : 0;
  const int64_t row = int64_t(at / a.groups);
  const int first = int(at - uint64_t(row) * a.groups) * kGroup;
  const int width = live ? min(kGroup, a.D - first) : 0;
  const Raw8<T> gr = load_piece<T, 16, A>(static_cast<const T*>(a.g) + row * a.g_st + first, 0, t, width);
  const Raw8<T> ur = load_piece<T, 16, A>(static_cast<const T*>(a.u) + row * a.u_st + first, 0, t, width);
  float g[8], u[8], o[8];
  widen8<T>(gr, g);
  widen8<T>(ur, u);
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = g[e] * sigmoid<T>(g[e]) * u[e];
  store_piece<T, 16, A>(static_cast<T*>(a.out) + row * a.D + first, 0, t, width, o);
  if constexpr (KEEP) {
    const float top_g = group_max(largest8(g)), top_u = group_max(largest8(u));
    const Scale8 sg(top_g), su(top_u);
    store_piece_s8<16, A>(a.g_q + row * a.q_st + first, 0, t, width, g, top_g < INFINITY, sg.inv);
    store_piece_s8<16, A>(a.u_q + row * a.q_st + first, 0, t, width, u, top_u < INFINITY, su.inv);
    if (live && t == 0) {
      a.g_scale[at] = sg.scale;
      a.u_scale[at] = su.scale;
    }
  }
}

template <typename T, bool A, bool KEPT>
__global__ void __launch_bounds__(kGluThreads) glu_bwd_kernel(const __grid_constant__ GluArgs a) {
  const int t = threadIdx.x & 15;
  const int64_t item = int64_t(blockIdx.x) * (kGluThreads / 16) + (threadIdx.x >> 4);
  if (item >= a.rows * a.groups) return;
  const int64_t row = int64_t(uint64_t(item) / a.groups);
  const int first = int(item - row * a.groups) * kGroup, width = min(kGroup, a.D - first);
  const Raw8<T> dr = load_piece<T, 16, A>(static_cast<const T*>(a.dout) + row * a.dout_st + first, 0, t, width);
  float d[8], g[8], u[8], o[8];
  if constexpr (KEPT) {
    load8<A>(a.g_q + row * a.q_st + first, a.g_scale[item], t, width, g);
    load8<A>(a.u_q + row * a.q_st + first, a.u_scale[item], t, width, u);
  } else {
    widen8<T>(load_piece<T, 16, A>(static_cast<const T*>(a.g) + row * a.g_st + first, 0, t, width), g);
    widen8<T>(load_piece<T, 16, A>(static_cast<const T*>(a.u) + row * a.u_st + first, 0, t, width), u);
  }
  widen8<T>(dr, d);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float s = sigmoid<T>(g[e]), y = g[e] * s;
    if (a.out) o[e] = y * u[e];
    u[e] = d[e] * u[e] * s * fmaf(g[e], 1.f - s, 1.f);
    g[e] = d[e] * y;
  }
  store_piece<T, 16, A>(static_cast<T*>(a.dg) + row * a.D + first, 0, t, width, u);
  store_piece<T, 16, A>(static_cast<T*>(a.du) + row * a.D + first, 0, t, width, g);
  if (a.out) store_piece<T, 16, A>(static_cast<T*>(a.out) + row * a.D + first, 0, t, width, o);
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
    for (int e = 0; e < 8; ++e) o[j][e] *= f[e] * sigmoid<T>(f[e]);
    top = max_nan(top, largest8(o[j]));
  }
  top = team_reduce<TPR, true>(top, red, set);
  const Scale8 s(top);
  int8_t* qr = a.a_q + row * a.a_q_st;
#pragma unroll
  for (int j = 0; j < NV; ++j) store_piece_s8<TPR, A>(qr, j, t, D, o[j], top < INFINITY, s.inv);
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

template <typename T>
int fwd(const GluArgs& a, bool aligned, cudaStream_t s) {
  if (a.a_q) return rows8<T>(a, aligned, s);
  const int64_t items = a.rows * a.groups, per = kGluThreads / 16;
  const unsigned ctas = unsigned((items + per - 1) / per);
  if (a.g_q) {
    if (aligned) glu_fwd_kernel<T, true, true><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_fwd_kernel<T, false, true><<<ctas, kGluThreads, 0, s>>>(a);
  } else {
    if (aligned) glu_fwd_kernel<T, true, false><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_fwd_kernel<T, false, false><<<ctas, kGluThreads, 0, s>>>(a);
  }
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int bwd(const GluArgs& a, bool aligned, cudaStream_t s) {
  const int64_t items = a.rows * a.groups, per = kGluThreads / 16;
  const unsigned ctas = unsigned((items + per - 1) / per);
  if (a.g_q) {
    if (aligned) glu_bwd_kernel<T, true, true><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_bwd_kernel<T, false, true><<<ctas, kGluThreads, 0, s>>>(a);
  } else {
    if (aligned) glu_bwd_kernel<T, true, false><<<ctas, kGluThreads, 0, s>>>(a);
    else glu_bwd_kernel<T, false, false><<<ctas, kGluThreads, 0, s>>>(a);
  }
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

int check(int dtype, int64_t rows, int64_t D) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (rows <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (rows >= (int64_t(1) << 31) || D >= (int64_t(1) << 30) || rows * ((D + kGroup - 1) / kGroup) >= (int64_t(1) << 34))
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
  a.groups = uint32_t((D + kGroup - 1) / kGroup);
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
  a.groups = uint32_t((D + kGroup - 1) / kGroup);
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

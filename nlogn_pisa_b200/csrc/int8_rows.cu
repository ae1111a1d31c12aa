// Tensors in 8 bits: a row, or every group of 128 elements of it, as signed
// bytes with one fp32 scale (Scale8 in rows.cuh has the rounding).
//
// Rows serve 8-bit products (a scale per token or output channel), groups keep
// activations for the backward.  Both are bound by HBM: 16-bit elements in, a
// byte out (and back): 16384 rows of 4096 in bf16 take 29 us (6.9 TB/s: the bytes
// stay in L2 for the product that follows), in fp32 40, one row of 1024 2.1 us.
// Groups, of which a team has one and its loads in flight: 46 us, back 37 (4.4 and
// 5.5 TB/s), in fp32 48 and 51.
#include "rows.cuh"

namespace pisa {

namespace {

struct RowArgs {
  const void* x;
  int64_t x_st;
  int64_t rows;
  uint32_t items;         // groups of all rows
  int64_t D;
  FastDiv groups;
  int8_t* q;
  int64_t q_st;
  float* scale;
  void* out;
  int* status;            // cleared on the way, or NULL
};

// A team holds the row.
template <typename T, int TPR, int NV, bool A>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) row_kernel(const __grid_constant__ RowArgs a) {
  constexpr int TEAMS = TPR < 128 ? 128 / TPR : 1;
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int t = threadIdx.x % TPR, D = int(a.D);
  const int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TPR;
  if (a.status && row == 0 && t == 0) *a.status = PISA_OK;
  if (row >= a.rows) return;                      // a whole warp
  const T* xr = static_cast<const T*>(a.x) + row * a.x_st;
  Raw8<T> x[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) x[j] = load_piece<T, TPR, A>(xr, j, t, D);
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[8];
    widen8<T>(x[j], f);
    top = larger(top, largest8<T>(x[j], f));
  }
  top = team_reduce<TPR, true>(top, red, set);
  const Scale8 s(top);
  int8_t* qr = a.q + row * a.q_st;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[8];
    widen8<T>(x[j], f);
    store_piece_s8<T, TPR, A>(qr, j, t, D, f, top < INFINITY, s.inv);
  }
  if (t == 0) a.scale[row] = s.scale;
}

// Rows too long for registers are read twice, in pieces of 8 times 512 elements.
template <typename T, bool A>
__global__ void __launch_bounds__(512) long_row_kernel(const __grid_constant__ RowArgs a) {
  constexpr int TPR = 512, STEP = TPR * 8;
  __shared__ float red[2 * (TPR / 32)];
  int set = 0;
  const int64_t row = blockIdx.x;
  if (a.status && row == 0 && threadIdx.x == 0) *a.status = PISA_OK;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_st;
  float top = 0.f;
  for (int64_t at = 0; at < a.D; at += STEP) {
    float f[8];
    widen8<T>(load_piece<T, TPR, A>(xr + at, 0, threadIdx.x, int(min64(STEP, a.D - at))), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = larger(top, fabsf(f[e]));
  }
  top = team_reduce<TPR, true>(top, red, set);
  const Scale8 s(top);
  int8_t* qr = a.q + row * a.q_st;
  for (int64_t at = 0; at < a.D; at += STEP) {
    const int left = int(min64(STEP, a.D - at));
    float f[8];
    widen8<T>(load_piece<T, TPR, A>(xr + at, 0, threadIdx.x, left), f);
    store_piece_s8<T, TPR, A>(qr + at, 0, threadIdx.x, left, f, top < INFINITY, s.inv);
  }
  if (threadIdx.x == 0) a.scale[row] = s.scale;
}

template <typename T, int TPR, int NV>
int launch_row(const RowArgs& a, bool aligned, cudaStream_t s) {
  constexpr int threads = TPR < 128 ? 128 : TPR, teams = threads / TPR;
  const unsigned ctas = unsigned((a.rows + teams - 1) / teams);
  if (aligned) row_kernel<T, TPR, NV, true><<<ctas, threads, 0, s>>>(a);
  else row_kernel<T, TPR, NV, false><<<ctas, threads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int rows8(const RowArgs& a, bool aligned, cudaStream_t s) {
  if (a.D <= 256) return launch_row<T, 32, 1>(a, aligned, s);
  if (a.D <= 1024) return launch_row<T, 32, 4>(a, aligned, s);
  if (a.D <= 4096) return launch_row<T, 128, 4>(a, aligned, s);
  if (a.D <= 16384) return launch_row<T, 512, 4>(a, aligned, s);
  if (aligned) long_row_kernel<T, true><<<unsigned(a.rows), 512, 0, s>>>(a);
  else long_row_kernel<T, false><<<unsigned(a.rows), 512, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

constexpr int kThreads = 256;

// Groups: sixteen threads each.
template <typename T, bool A, bool BACK>
__global__ void __launch_bounds__(kThreads) group_kernel(const __grid_constant__ RowArgs a) {
  const int t = threadIdx.x & 15;
  const uint32_t item = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  const bool live = item < a.items;
  const uint32_t at = live ? item : 0;
  const int64_t row = a.groups.div(at), first = int64_t(at - uint32_t(row) * a.groups.d) * kGroup;
  const int width = live ? int(min64(kGroup, a.D - first)) : 0;
  int8_t* qr = a.q + row * a.q_st + first;
  float f[8];
  if constexpr (BACK) {
    widen8_s8(load_piece_s8<T, 16, A>(qr, t, width), a.scale[at], f);
    store_piece<T, 16, A>(static_cast<T*>(a.out) + row * a.D + first, 0, t, width, f);
  } else {
    const Raw8<T> x = load_piece<T, 16, A>(static_cast<const T*>(a.x) + row * a.x_st + first, 0, t, width);
    widen8<T>(x, f);
    float top = largest8<T>(x, f);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(kFull, top, o));
    const Scale8 s(top);
    store_piece_s8<T, 16, A>(qr, 0, t, width, f, top < INFINITY, s.inv);
    if (live && t == 0) a.scale[at] = s.scale;
  }
}

template <typename T, bool BACK>
int groups8(const RowArgs& a, bool aligned, cudaStream_t s) {
  const int64_t items = a.rows * a.groups.d, per = kThreads / 16;
  const unsigned ctas = unsigned((items + per - 1) / per);
  if (aligned) group_kernel<T, true, BACK><<<ctas, kThreads, 0, s>>>(a);
  else group_kernel<T, false, BACK><<<ctas, kThreads, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

int check(const void* x, const int8_t* q, int64_t q_st, const float* scale, int dtype, int64_t rows, int64_t D) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (rows <= 0 || D <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (rows >= (int64_t(1) << 31) || D >= (int64_t(1) << 31) || rows * ((D + kGroup - 1) / kGroup) >= (int64_t(1) << 31) - 256)
    return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (!x || !q || !scale) return fail(PISA_ERR_INVALID, "the tensor, its bytes and scales are required");
  if (!rows_on16(q, rows, q_st)) return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must start on 16 bytes");
  return PISA_OK;
}

RowArgs make_args(int64_t rows, int64_t D, int8_t* q, int64_t q_st, float* scale) {
  RowArgs a{};
  a.rows = rows; a.D = D; a.groups = FastDiv::make(uint32_t((D + kGroup - 1) / kGroup)); a.items = uint32_t(rows) * a.groups.d; a.q = q; a.q_st = q_st; a.scale = scale;
  return a;
}

}  // namespace

int quantize_rows(const void* x, int64_t x_st, int dtype, int64_t rows, int64_t D, int8_t* q, int64_t q_st, float* scale, int* status,
                  cudaStream_t s) {
  if (int rc = check(x, q, q_st, scale, dtype, rows, D)) return rc;
  RowArgs a = make_args(rows, D, q, q_st, scale);
  a.x = x; a.x_st = x_st; a.status = status;
  const bool aligned = D % 8 == 0 && rows_on16(x, rows, x_st * (dtype == PISA_F32 ? 4 : 2));
  if (dtype == PISA_F32) return rows8<float>(a, aligned, s);
  if (dtype == PISA_BF16) return rows8<__nv_bfloat16>(a, aligned, s);
  return rows8<__half>(a, aligned, s);
}

}  // namespace pisa

extern "C" {

int pisa_quantize_int8(const void* x, int64_t x_st, int dtype, int64_t rows, int64_t D, int grouped, int8_t* q, int64_t q_st,
                       float* scale, pisa_stream_t stream) {
  using namespace pisa;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!grouped) return quantize_rows(x, x_st, dtype, rows, D, q, q_st, scale, nullptr, s);
  if (int rc = check(x, q, q_st, scale, dtype, rows, D)) return rc;
  RowArgs a = make_args(rows, D, q, q_st, scale);
  a.x = x; a.x_st = x_st;
  const bool aligned = D % 8 == 0 && rows_on16(x, rows, x_st * (dtype == PISA_F32 ? 4 : 2));
  if (dtype == PISA_F32) return groups8<float, false>(a, aligned, s);
  if (dtype == PISA_BF16) return groups8<__nv_bfloat16, false>(a, aligned, s);
  return groups8<__half, false>(a, aligned, s);
}

int pisa_restore_int8(const int8_t* q, int64_t q_st, const float* scale, int dtype, int64_t rows, int64_t D, void* out,
                      pisa_stream_t stream) {
  using namespace pisa;
  if (int rc = check(out, q, q_st, scale, dtype, rows, D)) return rc;
  RowArgs a = make_args(rows, D, const_cast<int8_t*>(q), q_st, const_cast<float*>(scale));
  a.out = out;
  const bool aligned = D % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PISA_F32) return groups8<float, true>(a, aligned, s);
  if (dtype == PISA_BF16) return groups8<__nv_bfloat16, true>(a, aligned, s);
  return groups8<__half, true>(a, aligned, s);
}

}  // extern "C"

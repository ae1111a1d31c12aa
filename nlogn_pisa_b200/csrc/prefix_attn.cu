// Attention of a step's newest tokens (one or a few per sequence) over the
// keys of a prefix that every sequence of the batch shares and the sequence's
// own cache: one softmax over both.  Token t of T sees the whole prefix and
// own keys 0 .. length - T + t.
//
// The keys are split along their length; a split's partial (m, l, o) of a row,
//   m = max s_j,  l = sum 2^(s_j - m),  o = sum 2^(s_j - m) v_j   (base 2),
// joins the others in a second launch: out = sum w o / sum w l with
// w = 2^(m - max m).  The prefix is one key range for the query rows of the
// whole batch, so its keys and values are read once for all of them; own
// caches are read once each.  This file holds the form on the FMA pipes (fp32
// tensors and heads wider than 128) and the joining launch.  The FMA form loads
// a tile, waits and computes in turn, and its latencies bound it: in fp32 64
// sequences of 1 to 2048 keys (8 heads of 128) take 458 us and the prefix of 8192
// that they share 319 us, against 73 and 10 us for their bytes.  The join is bound by
// its reads (L2 mostly), whose start overlaps the launch before it.
#include "prefix_attn.cuh"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;   // keys of one staged tile
constexpr int kCombineWarps = 8;

template <typename T, int DP, int LD>
__device__ __forceinline__ void stage_row(float* dst, const T* src, bool real, int c, int D) {
  constexpr int VN = Vec<T>::N;
  float v[VN];
#pragma unroll
  for (int e = 0; e < VN; ++e) v[e] = 0.f;
  if (real && c < D) load_vec<T>(src + c, v);
#pragma unroll
  for (int e = 0; e < VN; e += 4) *reinterpret_cast<float4*>(dst + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
}

// One CTA: 16 R query rows of one KV head (row = token * G + head of the
// group) against the keys of one split.  Row of thread ty*R + i, keys
// tx + 16 j, output columns tx*4 + 64 c.
template <typename T, int DP, int R>
__global__ void __launch_bounds__(kThreads) prefix_simt_kernel(const __grid_constant__ PrefixArgs a, bool prefix) {
  constexpr int BR = 16 * R, LD = DP + 4, LP = kKeys + 1, VN = Vec<T>::N, SEG = DP / VN;
  extern __shared__ __align__(16) float smem[];
  if (blockIdx.x + blockIdx.y + blockIdx.z + threadIdx.x == 0) *a.status = PISA_OK;
  float* qs = smem;
  float* ks = qs + BR * LD;   // keys, then the values of the same tile
  float* ps = ks + kKeys * LD;
  const int split = blockIdx.x / a.H, h = blockIdx.x % a.H, b = blockIdx.z;
  const int rows = (prefix ? a.B * a.T : a.T) * a.G, r0 = blockIdx.y * BR;
  const int length = prefix ? a.P : own_length(a, b);
  int begin, end;
  split_range(length, split, prefix ? a.prefix_chunk : a.own_chunk, begin, end);
  const T* kp = prefix ? static_cast<const T*>(a.pk) + h * a.pk_sh : static_cast<const T*>(a.k) + b * a.k_sb + h * a.k_sh;
  const T* vp = prefix ? static_cast<const T*>(a.pv) + h * a.pv_sh : static_cast<const T*>(a.v) + b * a.v_sb + h * a.v_sh;
  const int64_t k_st = prefix ? a.pk_st : a.k_st, v_st = prefix ? a.pv_st : a.v_st;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  for (int i = threadIdx.x; i < BR * SEG; i += kThreads) {
    const int r = i / SEG, c = (i - r * SEG) * VN, row = r0 + r;
    const int tok = row / a.G, g = row - tok * a.G;
    const int qb = prefix ? tok / a.T : b, qt = prefix ? tok - qb * a.T : tok;
    stage_row<T, DP, LD>(qs + r * LD, static_cast<const T*>(a.q) + qb * a.q_sb + qt * a.q_st + (h * a.G + g) * a.q_sh,
                         row < rows, c, a.D);
  }
  const float sl = a.scale * kLog2e;
  float acc[R][DP / 16], m[R], l[R];
  int last[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + ty * R + i;
    m[i] = -INFINITY;
    l[i] = 0.f;
    last[i] = row >= rows ? -1 : prefix ? a.P - 1 : length - a.T + row / a.G;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  for (int j0 = begin; j0 < end; j0 += kKeys) {
    const int nk = min(kKeys, end - j0);
    __syncthreads();
    for (int i = threadIdx.x; i < kKeys * SEG; i += kThreads) {
      const int r = i / SEG, c = (i - r * SEG) * VN;
      stage_row<T, DP, LD>(ks + r * LD, kp + int64_t(j0 + r) * k_st, r < nk, c, a.D);
    }
    __syncthreads();
    float s[R][4] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(qs + (ty * R + i) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(x.x, y[j].x, fmaf(x.y, y[j].y, fmaf(x.z, y[j].z, fmaf(x.w, y[j].w, s[i][j]))));
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float top = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = j0 + tx + 16 * j <= last[i] ? s[i][j] * sl : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
      const float base = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[i] - base);
      float sum = 0.f;
      m[i] = top;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - base);
        ps[(ty * R + i) * LP + tx + 16 * j] = p;
        sum += p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      l[i] = l[i] * corr + sum;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) acc[i][c] *= corr;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kKeys * SEG; i += kThreads) {
      const int r = i / SEG, c = (i - r * SEG) * VN;
      stage_row<T, DP, LD>(ks + r * LD, vp + int64_t(j0 + r) * v_st, r < nk, c, a.Dv);
    }
    __syncthreads();
    for (int j = 0; j < nk; ++j) {
      float p[R];
#pragma unroll
      for (int i = 0; i < R; ++i) p[i] = ps[(ty * R + i) * LP + j];
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 y = *reinterpret_cast<const float4*>(ks + j * LD + tx * 4 + 64 * c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (j0 + j > last[i]) continue;   // hidden values reach nothing, whatever they hold
          acc[i][4 * c + 0] = fmaf(p[i], y.x, acc[i][4 * c + 0]);
          acc[i][4 * c + 1] = fmaf(p[i], y.y, acc[i][4 * c + 1]);
          acc[i][4 * c + 2] = fmaf(p[i], y.z, acc[i][4 * c + 2]);
          acc[i][4 * c + 3] = fmaf(p[i], y.w, acc[i][4 * c + 3]);
        }
      }
    }
  }
  const int slots = a.prefix_splits + a.own_splits, slot = prefix ? split : a.prefix_splits + split;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + ty * R + i;
    if (row >= rows) continue;
    const int tok = row / a.G, g = row - tok * a.G;
    const int64_t at = (int64_t(prefix ? 0 : b) * a.T + tok) * a.Hq + h * a.G + g;   // tok counts b * T + t in the prefix
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    if (slots == 1) {
      if (tx == 0 && a.lse) a.lse[at] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
    } else if (tx == 0) {
      a.part_ml[at * slots + slot] = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = tx * 4 + 64 * c + e;
        if (d >= a.Dv) continue;
        if (slots == 1) static_cast<T*>(a.out)[at * a.Dv + d] = from_f32<T>(acc[i][4 * c + e] * inv);
        else a.part_o[(at * slots + slot) * a.Dv + d] = acc[i][4 * c + e];
      }
    }
  }
}

// Joins the slots of a row that were written: all prefix splits, and the own
// splits that hold keys (one at least).  One CTA per row; its warps take the
// slots in turn, a lane 4 columns (and 4 more past 128), and join through
// shared memory: with a few hundred rows the work is a few loads deep, not a
// chain of them.
template <typename T>
__global__ void prefix_combine_kernel(const __grid_constant__ PrefixArgs a) {
  __shared__ float4 part[kCombineWarps][2][32];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  const int slots = a.prefix_splits + a.own_splits;
  const int ranges = (own_length(a, int(row / (int64_t(a.T) * a.Hq))) + a.own_chunk - 1) / a.own_chunk;
  const float2* ml = a.part_ml + row * slots;
  const float* po = a.part_o + row * slots * a.Dv + lane * 4;
  cudaGridDependencySynchronize();   // the partials are complete from here on
  // slots: the prefix's ranges, then, from prefix_splits on, the own cache's
  const int shared = a.tile_ctas ? a.status[1] : a.prefix_splits, used = shared + max(1, ranges);
  auto place = [&](int s) { return s < shared ? s : s - shared + a.prefix_splits; };
  float top = -INFINITY;
  for (int s = lane; s < used; s += 32) {
    const float2 x = ml[place(s)];
    if (x.y != 0.f) top = fmaxf(top, x.x);
  }
  top = warp_max(top);
  // slots without weight are left out, whatever their partial holds
  float total = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int s0 = 0; s0 < used; s0 += 32) {
    const float2 x = s0 + lane < used ? ml[place(s0 + lane)] : make_float2(0.f, 0.f);
    const float weight = x.y == 0.f ? 0.f : exp2f(x.x - top);   // of slot s0 + lane
    total = fmaf(weight, x.y, total);
    const uint32_t heavy = __ballot_sync(kFull, x.y != 0.f);
#pragma unroll 4
    for (int i = warp; i < min(32, used - s0); i += warps) {
      const float w = __shfl_sync(kFull, weight, i);
      if (!(heavy >> i & 1)) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (lane * 4 + 128 * c >= a.Dv) continue;
        const float4 o = __ldcs(reinterpret_cast<const float4*>(po + int64_t(place(s0 + i)) * a.Dv + 128 * c));
        acc[c].x = fmaf(w, o.x, acc[c].x);
        acc[c].y = fmaf(w, o.y, acc[c].y);
        acc[c].z = fmaf(w, o.z, acc[c].z);
        acc[c].w = fmaf(w, o.w, acc[c].w);
      }
    }
  }
  total = warp_sum(total);
  if (a.lse && threadIdx.x == 0) a.lse[row] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
  part[warp][0][lane] = acc[0];
  part[warp][1][lane] = acc[1];
  __syncthreads();
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int d = threadIdx.x; d < a.Dv; d += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += reinterpret_cast<const float*>(part[w])[d];
    static_cast<T*>(a.out)[row * a.Dv + d] = from_f32<T>(v * inv);
  }
}

template <typename T, int DP, int R>
int launch(const PrefixArgs& a, bool prefix, cudaStream_t s) {
  constexpr int BR = 16 * R;
  const size_t smem = sizeof(float) * (BR * (DP + 4) + kKeys * (DP + 4) + BR * (kKeys + 1));
  if (int rc = allow_smem<prefix_simt_kernel<T, DP, R>>(int(smem), "prefix attention smem attribute")) return rc;
  const int64_t rows = int64_t(prefix ? a.B : 1) * a.T * a.G;
  // heads of a key range side by side: their rows share DRAM pages
  const dim3 grid(unsigned((prefix ? a.prefix_splits : a.own_splits) * a.H), unsigned((rows + BR - 1) / BR),
                  unsigned(prefix ? 1 : a.B));
  prefix_simt_kernel<T, DP, R><<<grid, kThreads, smem, s>>>(a, prefix);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int segments(const PrefixArgs& a, cudaStream_t s) {
  // 64-row tiles once a KV head has more than 16 query rows: fewer passes over the keys
  int rc = PISA_OK;
  if (a.prefix_splits) rc = int64_t(a.B) * a.T * a.G > 16 ? launch<T, DP, 4>(a, true, s) : launch<T, DP, 1>(a, true, s);
  if (rc == PISA_OK && a.own_splits)
    rc = int64_t(a.T) * a.G > 16 ? launch<T, DP, 4>(a, false, s) : launch<T, DP, 1>(a, false, s);
  return rc;
}

template <typename T>
int by_dim(const PrefixArgs& a, cudaStream_t s) {
  const int d = a.D > a.Dv ? a.D : a.Dv;
  if (d <= 64) return segments<T, 64>(a, s);
  if (d <= 128) return segments<T, 128>(a, s);
  return segments<T, 256>(a, s);
}

template <typename T>
int combine(const PrefixArgs& a, cudaStream_t s) {
  const int slots = a.prefix_splits + a.own_splits;
  const int warps = slots > 32 ? kCombineWarps : kCombineWarps / 2;
  return launch_after(prefix_combine_kernel<T>, dim3(unsigned(int64_t(a.B) * a.T * a.Hq)), warps * 32, 0, a, s);
}

}  // namespace

int prefix_attn_simt(const PrefixArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == PISA_F32) return by_dim<float>(a, stream);
  if (dtype == PISA_BF16) return by_dim<__nv_bfloat16>(a, stream);
  return by_dim<__half>(a, stream);
}

int prefix_combine(const PrefixArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == PISA_F32) return combine<float>(a, stream);
  if (dtype == PISA_BF16) return combine<__nv_bfloat16>(a, stream);
  return combine<__half>(a, stream);
}

}  // namespace pisa

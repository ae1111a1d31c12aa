// Shared-prefix decode attention on mma.sync, for 16-bit tensors with heads of
// at most 128 dims (formulas and partial results in prefix_attn.cu).
//
// A decode step reads every key and value once for a handful of query rows,
// so it is bound by HBM; the kernel's task is to keep loads in flight.  A warp
// takes 16 query rows (8 are enough up to G * T = 8) and 16 keys per step and
// loads keys and values straight into the registers that the MMAs read:
//  - a contraction may visit the dims in any order, so the B operand of
//    S = Q K^T takes the 8 consecutive dims (16 bytes) that a thread loads of
//    a key row as its operands of two steps; Q is loaded the same way;
//  - the columns of O may stand in any order, so the B operand of O += P V
//    takes 8 consecutive dims of four key rows, whose halves two byte
//    permutations pair up.
// There is no shared-memory staging and no barrier in the loop; the next
// step's keys are requested when this step's scores are done, its values when
// this step's products are.  Each warp keeps its own running maximum and sum;
// the warps that share query rows join at the end.
//
// Hidden keys: scores are selected away, and value rows past the last key
// that every row sees are zeroed in registers; the up to T - 1 newer keys
// that only later tokens see are added row by row.
#include "dense_tc.cuh"
#include "prefix_attn.cuh"

namespace pisa {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kStep = 16;                 // keys of a warp's step

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(kFull, v, 1));
  return fmaxf(v, __shfl_xor_sync(kFull, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(kFull, v, 1);
  return v + __shfl_xor_sync(kFull, v, 2);
}

// Thread (g, t) = (lane / 4, lane % 4).  HALVES: 16-row fragments' halves in
// use (1: rows 0-7 only).  row_warps: warps of the CTA with query rows of
// their own; the other factor of kWarps splits the keys of a step.
template <typename T, int DP, int HALVES>
__global__ void __launch_bounds__(kThreads) prefix_mma_kernel(const __grid_constant__ PrefixArgs a, bool prefix, int row_warps) {
  constexpr int KC = DP / 32, VC = DP / 64, NT = DP / 8;   // 16-byte loads of a key / value row per thread, O tiles
  constexpr int BR = 8 * HALVES;
  extern __shared__ __align__(16) float smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, h = blockIdx.z % a.H, b = prefix ? 0 : blockIdx.z / a.H;
  const int rows = (prefix ? a.B * a.T : a.T) * a.G;
  const int r0 = (int(blockIdx.y) * row_warps + warp % row_warps) * BR;
  const int key_warps = kWarps / row_warps, key_warp = warp / row_warps;
  const int length = prefix ? a.P : own_length(a, b);
  int begin, end;
  split_range(length, split, prefix ? a.prefix_splits : a.own_splits, kWarps * kStep, begin, end);
  const int shared = prefix ? length : length - a.T + 1;   // keys before this one are seen by every row
  const T* kp = prefix ? static_cast<const T*>(a.pk) + h * a.pk_sh : static_cast<const T*>(a.k) + b * a.k_sb + h * a.k_sh;
  const T* vp = prefix ? static_cast<const T*>(a.pv) + h * a.pv_sh : static_cast<const T*>(a.v) + b * a.v_sb + h * a.v_sh;
  const int64_t k_st = prefix ? a.pk_st : a.k_st, v_st = prefix ? a.pv_st : a.v_st;

  uint4 q[HALVES][KC];
  int last[HALVES];
#pragma unroll
  for (int i = 0; i < HALVES; ++i) {
    const int row = r0 + g + 8 * i, tok = row / a.G, hq = h * a.G + row - tok * a.G;
    const int qb = prefix ? tok / a.T : b, qt = prefix ? tok - qb * a.T : tok;
    last[i] = row >= rows ? -1 : prefix ? length - 1 : length - a.T + tok;
    const T* qp = static_cast<const T*>(a.q) + qb * a.q_sb + qt * a.q_st + hq * a.q_sh;
#pragma unroll
    for (int c = 0; c < KC; ++c)
      q[i][c] = row < rows && 32 * c + 8 * t < a.D ? *reinterpret_cast<const uint4*>(qp + 32 * c + 8 * t) : make_uint4(0, 0, 0, 0);
  }
  const float sl = a.scale * kLog2e;
  float o[NT][4], m[HALVES], l[HALVES];
#pragma unroll
  for (int i = 0; i < HALVES; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

  uint4 k[2][KC], v[4][VC];
  // keys 8 i + g of the step at j; rows past the end repeat the last one (their scores are selected away)
  auto load_k = [&](int j) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const T* p = kp + int64_t(min(j + 8 * i + g, end - 1)) * k_st + 8 * t;
#pragma unroll
      for (int c = 0; c < KC; ++c)
        k[i][c] = 32 * c + 8 * t < a.D ? __ldg(reinterpret_cast<const uint4*>(p + 32 * c)) : make_uint4(0, 0, 0, 0);
    }
  };
  // values of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9; zero from key min(end, shared) on
  const int seen = min(end, shared);
  auto load_v = [&](int j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = j + 2 * t + (i & 1) + 8 * (i >> 1);
      const T* p = vp + int64_t(key) * v_st + 8 * g;
#pragma unroll
      for (int c = 0; c < VC; ++c)
        v[i][c] = key < seen && 64 * c + 8 * g < a.Dv ? __ldg(reinterpret_cast<const uint4*>(p + 64 * c)) : make_uint4(0, 0, 0, 0);
    }
  };
  const int stride = key_warps * kStep;
  int j = begin + key_warp * kStep;
  if (r0 < rows && j < end) {
    load_k(j);
    load_v(j);
    for (; j < end; j += stride) {
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const uint4 lo = q[0][c], hi = HALVES == 2 ? q[HALVES - 1][c] : make_uint4(0, 0, 0, 0);
          mma16816<T>(s[i], lo.x, hi.x, lo.y, hi.y, k[i][c].x, k[i][c].y);
          mma16816<T>(s[i], lo.z, hi.z, lo.w, hi.w, k[i][c].z, k[i][c].w);
        }
      }
      if (j + stride < end) load_k(j + stride);
      const bool partial = j + kStep > seen;    // keys past the end, or seen by some rows only
      uint32_t p[2][HALVES];                    // P of key tiles 0 and 1 as A operands
      float alpha[HALVES], pf[2][HALVES][2];
      bool moved = false;
#pragma unroll
      for (int i = 0; i < HALVES; ++i) {
        float x[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[n][e] = s[n][2 * i + e] * sl;
            const int key = j + 8 * n + 2 * t + e;
            if (partial && (key > last[i] || key >= end)) x[n][e] = -INFINITY;
          }
        }
        const float top = quad_max(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])));
        const float to = fmaxf(m[i], top), ref = to == -INFINITY ? 0.f : to;
        alpha[i] = m[i] == -INFINITY ? 0.f : tc::ex2f(m[i] - ref);
        moved = moved || to > m[i];
        m[i] = to;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            pf[n][i][e] = tc::ex2f(x[n][e] - ref);
            sum += pf[n][i][e];
            const int key = j + 8 * n + 2 * t + e;
            if (partial && key >= seen) x[n][e] = 0.f;      // added row by row below
            else x[n][e] = pf[n][i][e];
          }
          p[n][i] = pack2<T>(x[n][0], x[n][1]);
        }
        l[i] = l[i] * alpha[i] + sum;    // this thread's share of the row's sum
      }
      if (__any_sync(kFull, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < HALVES; ++i) {
            o[n][2 * i] *= alpha[i];
            o[n][2 * i + 1] *= alpha[i];
          }
        }
      }
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const uint32_t* v0 = &v[0][c].x;
        const uint32_t* v1 = &v[1][c].x;
        const uint32_t* v2 = &v[2][c].x;
        const uint32_t* v3 = &v[3][c].x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {   // O tile 8 c + e: dims 64 c + 8 g + e
          const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
          mma16816<T>(o[8 * c + e], p[0][0], HALVES == 2 ? p[0][HALVES - 1] : 0u, p[1][0], HALVES == 2 ? p[1][HALVES - 1] : 0u,
                      __byte_perm(v0[e / 2], v1[e / 2], sel), __byte_perm(v2[e / 2], v3[e / 2], sel));
        }
      }
      if (j + stride < end) load_v(j + stride);
      if (partial) {
        for (int key = max(j, shared); key < min(j + kStep, end); ++key) {
          const int x = key - j, src = (lane & ~3) | ((x & 7) >> 1);
#pragma unroll
          for (int i = 0; i < HALVES; ++i) {
            const float w0 = x < 8 ? pf[0][i][0] : pf[1][i][0], w1 = x < 8 ? pf[0][i][1] : pf[1][i][1];
            const float w = __shfl_sync(kFull, x & 1 ? w1 : w0, src);
            if (key > last[i]) continue;
            // O tile n, columns 2 t and 2 t + 1: dims 64 c + 16 t + e and 8 more
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int d = 64 * (n / 8) + 16 * t + (n & 7);
              if (d < a.Dv) o[n][2 * i] = fmaf(w, to_f32<T>(vp[int64_t(key) * v_st + d]), o[n][2 * i]);
              if (d + 8 < a.Dv) o[n][2 * i + 1] = fmaf(w, to_f32<T>(vp[int64_t(key) * v_st + d + 8]), o[n][2 * i + 1]);
            }
          }
        }
      }
    }
  }
  // Join the warps that share query rows: (m, l) per row and O through shared memory.
  float* so = smem;                                        // [kWarps][BR][DP + 4]
  float2* sml = reinterpret_cast<float2*>(so + kWarps * BR * (DP + 4));   // [kWarps][BR]
#pragma unroll
  for (int i = 0; i < HALVES; ++i) {
    const int row = g + 8 * i;
    const float sum = quad_sum(l[i]);
    if (t == 0) sml[warp * BR + row] = make_float2(m[i], sum);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int d = 64 * (n / 8) + 16 * t + (n & 7);
      so[(warp * BR + row) * (DP + 4) + d] = o[n][2 * i];
      so[(warp * BR + row) * (DP + 4) + d + 8] = o[n][2 * i + 1];
    }
  }
  __syncthreads();
  const int slots = a.prefix_splits + a.own_splits, slot = prefix ? split : a.prefix_splits + split;
  for (int x = threadIdx.x; x < row_warps * BR * (DP / 4); x += kThreads) {
    const int d = x % (DP / 4) * 4, r = x / (DP / 4) % BR, rw = x / (DP / 4) / BR;
    const int row = (int(blockIdx.y) * row_warps + rw) * BR + r;
    if (row >= rows || d >= a.Dv) continue;
    float top = -INFINITY;
    for (int w = 0; w < key_warps; ++w) top = fmaxf(top, sml[(w * row_warps + rw) * BR + r].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int w = 0; w < key_warps; ++w) {
      const int at = (w * row_warps + rw) * BR + r;
      const float2 y = sml[at];
      if (y.y == 0.f) continue;            // no keys, or only weightless ones
      const float f = tc::ex2f(y.x - ref);
      const float4 z = *reinterpret_cast<const float4*>(so + at * (DP + 4) + d);
      sum = fmaf(f, y.y, sum);
      acc.x = fmaf(f, z.x, acc.x);
      acc.y = fmaf(f, z.y, acc.y);
      acc.z = fmaf(f, z.z, acc.z);
      acc.w = fmaf(f, z.w, acc.w);
    }
    const int tok = row / a.G, hq = h * a.G + row - tok * a.G;
    const int64_t at = (int64_t(b) * a.T + tok) * a.Hq + hq;   // in the prefix tok counts b * T + t
    if (slots == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const uint2 w = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.Dv + d) = w;
      if (d == 0 && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    } else {
      *reinterpret_cast<float4*>(a.part_o + (at * slots + slot) * a.Dv + d) = acc;
      if (d == 0) a.part_ml[at * slots + slot] = make_float2(top, sum);
    }
  }
}

template <typename T, int DP, int HALVES>
int launch(const PrefixArgs& a, bool prefix, cudaStream_t s) {
  constexpr int BR = 8 * HALVES;
  const int64_t rows = int64_t(prefix ? a.B : 1) * a.T * a.G, blocks = (rows + BR - 1) / BR;
  const int row_warps = blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
  constexpr int smem = kWarps * BR * ((DP + 4) * 4 + 8);
  static_assert(smem <= 48 * 1024, "fits the default shared memory");
  const dim3 grid(unsigned(prefix ? a.prefix_splits : a.own_splits), unsigned((blocks + row_warps - 1) / row_warps),
                  unsigned((prefix ? 1 : a.B) * a.H));
  prefix_mma_kernel<T, DP, HALVES><<<grid, kThreads, smem, s>>>(a, prefix, row_warps);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int segment(const PrefixArgs& a, bool prefix, cudaStream_t s) {
  // rows 8-15 of the fragments are left out when no KV head has them: half the
  // accumulator registers, so more warps and more loads in flight
  return int64_t(prefix ? a.B : 1) * a.T * a.G <= 8 ? launch<T, DP, 1>(a, prefix, s) : launch<T, DP, 2>(a, prefix, s);
}

template <typename T, int DP>
int segments(const PrefixArgs& a, cudaStream_t s) {
  int rc = PISA_OK;
  if (a.prefix_splits) rc = segment<T, DP>(a, true, s);
  if (rc == PISA_OK && a.own_splits) rc = segment<T, DP>(a, false, s);
  return rc;
}

template <typename T>
int by_dim(const PrefixArgs& a, cudaStream_t s) {
  return a.D <= 64 && a.Dv <= 64 ? segments<T, 64>(a, s) : segments<T, 128>(a, s);
}

}  // namespace

int prefix_attn_mma(const PrefixArgs& a, int dtype, cudaStream_t stream) {
  return dtype == PISA_BF16 ? by_dim<__nv_bfloat16>(a, stream) : by_dim<__half>(a, stream);
}

}  // namespace pisa

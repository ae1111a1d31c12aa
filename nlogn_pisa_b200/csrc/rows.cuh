// Row-wise building blocks of the decoder block's operators: threads that share
// a row, its sums and maxima, and the 8-bit form of a row or of a group of it.
//
// A team of TPR threads holds a row in registers, NV pieces of 8 elements per
// thread.  Where every row starts on 16 bytes and its width is a multiple of 8
// (A), piece j of thread t is 8 consecutive elements, in fp32 two times 4 of them,
// so that a warp's 16-byte accesses lie side by side; otherwise its elements lie
// TPR apart, so that a warp still touches consecutive ones.
#pragma once

#include <cmath>
#include <type_traits>

#include "dense_attn.cuh"
#include "internal.h"

namespace pisa {

// Smallest magnitude that an 8-bit scale follows: below it 127 / max would overflow.
constexpr float kTiny = 7.88860905221011805e-31f;   // 2^-100
constexpr int kGroup = 128;                          // elements that share a scale of a kept activation

// 8 elements as loaded.
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };

template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(r.v[i].x);
      f[4 * i + 1] = __uint_as_float(r.v[i].y);
      f[4 * i + 2] = __uint_as_float(r.v[i].z);
      f[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
  } else {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const float (&f)[8]) {
  Raw8<T> r;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.v[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                          __float_as_uint(f[4 * i + 3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    r.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

// Arithmetic on pairs: one instruction for two fp32 results.
__device__ __forceinline__ float2 pair_fma(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 pair_mul(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 pair_add(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 pair_at(const float (&f)[8], int i) { return make_float2(f[2 * i], f[2 * i + 1]); }
__device__ __forceinline__ void set_pair(float (&f)[8], int i, float2 v) {
  f[2 * i] = v.x;
  f[2 * i + 1] = v.y;
}

// Data that is read once: past L1.
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Column of element e of piece j.
template <typename T, int TPR, bool A>
__device__ __forceinline__ int column(int j, int e, int t) {
  if constexpr (!A) return (j * 8 + e) * TPR + t;
  else if constexpr (sizeof(T) == 2) return (j * TPR + t) * 8 + e;
  else return ((2 * j + e / 4) * TPR + t) * 4 + e % 4;
}

// Piece j of a row of D elements; elements past its end are zeros.
template <typename T, int TPR, bool A>
__device__ __forceinline__ Raw8<T> load_piece(const T* row, int j, int t, int D) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) r.v[i] = make_uint4(0, 0, 0, 0);
  if constexpr (A) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) {
      const int c = column<T, TPR, A>(j, 4 * i, t);
      if (c < D) r.v[i] = load_stream(row + c);
    }
  } else {
    uint32_t w[2 * sizeof(T)];
#pragma unroll
    for (int i = 0; i < int(2 * sizeof(T)); ++i) w[i] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<T, TPR, A>(j, e, t);
      if (c < D) {
        if constexpr (sizeof(T) == 4) asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[e]) : "l"(row + c));
        else {
          uint16_t h;
          asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(h) : "l"(row + c));
          w[e / 2] |= uint32_t(h) << (e % 2 * 16);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) r.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  return r;
}

template <typename T, int TPR, bool A>
__device__ __forceinline__ void store_piece(T* row, int j, int t, int D, const float (&f)[8]) {
  if constexpr (A) {
    const Raw8<T> r = narrow8<T>(f);
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) {
      const int c = column<T, TPR, A>(j, 4 * i, t);
      if (c < D) *reinterpret_cast<uint4*>(row + c) = r.v[i];
    }
  } else {
    T* at = row + column<T, TPR, A>(j, 0, t);
    const Raw8<T> r = narrow8<T>(f);
    const T* e = reinterpret_cast<const T*>(&r);
    if (TPR > 16 && (j + 1) * 8 * TPR <= D) {   // a whole piece for all threads: no test per element
#pragma unroll
      for (int i = 0; i < 8; ++i) at[i * TPR] = e[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (column<T, TPR, A>(j, i, t) < D) at[i * TPR] = e[i];
    }
  }
}

// Piece j of a parameter row in fp32 or in the tensors' type (cached: many rows read it).
template <typename T, int TPR, bool A>
__device__ __forceinline__ void param_piece(const void* p, int f32, int j, int t, int D, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0.f;
  if constexpr (A) {
    if (f32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = column<T, TPR, A>(j, 4 * i, t);
        if (c >= D) continue;
        const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c));
        f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
      }
    } else if constexpr (sizeof(T) == 2) {
      const int c = column<T, TPR, A>(j, 0, t);
      if (c >= D) return;
      Raw8<T> r;
      r.v[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + c));
      widen8<T>(r, f);
    }
  } else {
    if (f32) {
      const float* at = static_cast<const float*>(p) + column<T, TPR, A>(j, 0, t);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (column<T, TPR, A>(j, e, t) < D) f[e] = __ldg(at + e * TPR);
    } else {
      const T* at = static_cast<const T*>(p) + column<T, TPR, A>(j, 0, t);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (column<T, TPR, A>(j, e, t) < D) f[e] = to_f32<T>(__ldg(at + e * TPR));
    }
  }
}

// Larger of two, NaN if either is.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum (or maximum, NaN if any is) of a team's values, the same in all its
// threads and in every run.  Teams of more than a warp are whole CTAs; `red`
// holds two sets of TPR / 32 floats that calls use in turn (`set`), so that one
// barrier per call is enough.
template <int TPR, bool MAX>
__device__ __forceinline__ float team_reduce(float v, float* red, int& set) {
#pragma unroll
  for (int o = TPR < 32 ? TPR / 2 : 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(kFull, v, o);
    v = MAX ? larger(v, w) : v + w;
  }
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    float* at = red + set * W;
    set ^= 1;
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    v = at[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = MAX ? larger(v, at[i]) : v + at[i];
  }
  return v;
}

// The 8-bit form of values whose largest magnitude is `top`: q = round(x * inv)
// to the nearest (ties to even), x ~ q * scale, each step one fp32 result:
//   m = max(top, 2^-100), inv = 127 / m, scale = m / 127.
// Values that hold an infinity or NaN are zeros under a scale of NaN: they read
// back as NaN.
struct Scale8 {
  float inv, scale;
  __device__ __forceinline__ explicit Scale8(float top) {
    const float m = fmaxf(top, kTiny);
    const bool fine = top < INFINITY;
    inv = fine ? __fdiv_rn(127.f, m) : 0.f;
    scale = fine ? __fdiv_rn(m, 127.f) : __int_as_float(0x7fffffff);
  }
};

// Eight rounded values as bytes.  Adding 1.5 * 2^23 leaves the nearest integer
// (ties to even, as the sum's rounding) in the low bits of the sum.  The product
// is rounded before: as pairs the two steps became one multiply-add, whose single
// rounding differs next to ties.
__device__ __forceinline__ uint2 pack8_s8(const float (&f)[8], float inv) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], inv), 12582912.f));
  return make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
}

// Largest magnitude of a thread's 8 values, NaN if any is: 16-bit values in
// their packed form.
template <typename T>
__device__ __forceinline__ float largest8(const Raw8<T>& r, const float (&f)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = larger(top, fabsf(f[e]));
    return top;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
    return larger(__low2float(m), __high2float(m));
  } else {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
    return larger(__low2float(m), __high2float(m));
  }
}

template <typename T, int TPR, bool A>
__device__ __forceinline__ void store_piece_s8(int8_t* row, int j, int t, int D, const float (&f)[8], bool fine, float inv) {
  const uint2 bytes = pack8_s8(f, inv);
  const uint32_t lo = fine ? bytes.x : 0, hi = fine ? bytes.y : 0;
  if constexpr (A) {
    const int c = column<T, TPR, A>(j, 0, t), c4 = column<T, TPR, A>(j, 4, t);
    if constexpr (sizeof(T) == 2) {
      if (c < D) *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
    } else {
      if (c < D) *reinterpret_cast<uint32_t*>(row + c) = lo;
      if (c4 < D) *reinterpret_cast<uint32_t*>(row + c4) = hi;
    }
  } else {
    int8_t* at = row + column<T, TPR, A>(j, 0, t);
    if (TPR > 16 && (j + 1) * 8 * TPR <= D) {   // a whole piece for all threads: no test per element
#pragma unroll
      for (int e = 0; e < 8; ++e) at[e * TPR] = int8_t((e < 4 ? lo >> (8 * e) : hi >> (8 * (e - 4))) & 255u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (column<T, TPR, A>(j, e, t) < D) at[e * TPR] = int8_t((e < 4 ? lo >> (8 * e) : hi >> (8 * (e - 4))) & 255u);
    }
  }
}

// Piece 0 of kept bytes, zeros past their end, and as floats.
template <typename T, int TPR, bool A>
__device__ __forceinline__ uint2 load_piece_s8(const int8_t* row, int t, int D) {
  uint2 r = make_uint2(0, 0);
  if constexpr (A) {
    const int c = column<T, TPR, A>(0, 0, t), c4 = column<T, TPR, A>(0, 4, t);
    if constexpr (sizeof(T) == 2) {
      if (c < D) asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(row + c));
    } else {
      if (c < D) asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(r.x) : "l"(row + c));
      if (c4 < D) asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(r.y) : "l"(row + c4));
    }
  } else {
    const uint8_t* at = reinterpret_cast<const uint8_t*>(row) + column<T, TPR, A>(0, 0, t);
    uint32_t b[8];
    if (8 * TPR <= D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = __ldg(at + e * TPR);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = column<T, TPR, A>(0, e, t) < D ? __ldg(at + e * TPR) : 0;
    }
    r.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
    r.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
  }
  return r;
}
// A byte b in the low bits of 0x4B000000 | (b ^ 128) is the float 2^23 + 128 + b.
__device__ __forceinline__ void widen8_s8(const uint2& q, float scale, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (i < 2 ? q.x : q.y) ^ 0x80808080u;
    const float2 x = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, i % 2 ? 0x7442 : 0x7440)),
                                 __uint_as_float(__byte_perm(u, 0x4B000000u, i % 2 ? 0x7443 : 0x7441)));
    set_pair(f, i, pair_mul(pair_add(x, both(-8388736.f)), both(scale)));
  }
}

// Host: whether a row view starts every row on 16 bytes (the stride of a single row may hold anything).
inline bool rows_on16(const void* p, int64_t rows, int64_t stride_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows == 1 || stride_bytes % 16 == 0);
}

}  // namespace pisa

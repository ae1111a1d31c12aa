// Building blocks shared by the tensor-core kernels of dense attention.
#pragma once

#include <type_traits>

#include "dense_attn.cuh"
#include "tc.cuh"

namespace pisa {

constexpr int kRows = 128;   // queries of a tile, keys of a tile

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
         "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
         "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(x0), "r"(x1), "r"(x2), "r"(x3) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// (a * b) on two lanes at once
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Untiled bulk copy into shared memory: both addresses on 16 bytes, `bytes` a
// multiple of 16; completion counts on `mbar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(src), "r"(bytes), "r"(tc::smem_u32(mbar)) : "memory");
}

// Zero rows [first, last) of a [DP/64][128 rows][128 B] operand tile, one warp.
template <int DP>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first, int last, int lane) {
  for (int f = lane; f < (last - first) * DP / 8; f += 32) {
    const int r = first + f / (DP / 8), s = f % (DP / 8);
    st_shared16(tile + (s >> 3) * kRows * 128 + r * 128 + (s & 7) * 16, 0, 0, 0, 0);
  }
}

// This warp's 32 TMEM lanes x W columns, rounded to T, to the first `rows` rows
// of global memory (row r at out + r * stride, columns past `cols` dropped)
// through `stage` (32 * W * 2 bytes of shared memory of this warp).  With
// `empty` zeros are stored in their place.
template <typename T, int W>
__device__ __forceinline__ void store_lanes(uint32_t taddr, bool empty, float mul, uint32_t stage, T* out, int64_t stride,
                                            int rows, int cols, int lane) {
  constexpr int SEG = W / 8;
#pragma unroll
  for (int c = 0; c < W; c += 32) {
    float o[32];
    if (empty) {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0.f;
    } else {
      tc::tmem_ld32(taddr + c, o);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int seg = c / 8 + s;
      st_shared16(stage + (lane * SEG + (seg ^ (lane & (SEG - 1) & 7))) * 16, pack2<T>(o[8 * s] * mul, o[8 * s + 1] * mul),
                  pack2<T>(o[8 * s + 2] * mul, o[8 * s + 3] * mul), pack2<T>(o[8 * s + 4] * mul, o[8 * s + 5] * mul),
                  pack2<T>(o[8 * s + 6] * mul, o[8 * s + 7] * mul));
    }
  }
  __syncwarp();
  for (int f = lane; f < rows * SEG; f += 32) {
    const int r = f / SEG, seg = f % SEG;
    const uint4 v = ld_shared16(stage + (r * SEG + (seg ^ (r & (SEG - 1) & 7))) * 16);
    if (seg * 8 < cols) *reinterpret_cast<uint4*>(out + r * stride + seg * 8) = v;
  }
}

}  // namespace pisa

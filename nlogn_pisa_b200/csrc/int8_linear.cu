// Products of 8-bit tensors with a scale per token and per output channel.
//
//   y[t, o] = ws[o] xs[t] sum_k w[o, k] x[t, k] + bias[o],
// with int32 sums, which are exact for K < 2^17.
//
// tcgen05 tiles (kind::i8): 128 output channels are the rows of a tile and up
// to BN tokens its columns, so a warp's lanes are 32 consecutive channels of every
// token it stores and rows of any length leave without a detour.  K goes in
// blocks of 128 bytes, a 128-byte-swizzled TMA box of each operand per stage.
// Warp 0 loads, warp 1 issues the MMAs, warps 2 to 9 scale and store; two
// accumulators in TMEM let a tile's stores run under the next tile's products.
//
// Many tokens are bound by the tensor cores (and, back to back, by power), few by
// HBM and the start of a launch: 16384 x 4096 x 11264 takes 437 to 449 us (3.4
// PTOP/s, tensor pipe 86 % busy on a smaller case), 64 tokens over 4096 x 16384
// 14.7 us (4.7 TB/s), one token in bytes over 1024 x 5632 5.4 us.  Tiles of short K are bound
// by their stores: 30000 x 512 x 2000 49 us (65 with a test per store).
//
// A few floating tokens are rounded by the storing warps of every CTA, which
// keep their bytes in shared memory for all of its tiles, while the first weights
// arrive: one launch instead of two.
//
// Where the tiles are fewer than the SMs, a cluster of CTAs shares each: every
// CTA sums a range of K, leaves its int32 sums in shared memory, and takes a
// share of the tile's tokens, for which it adds all ranges' sums (integers: in
// any order the same).
#include <cudaTypedefs.h>

#include "dense_tc.cuh"
#include "rows.cuh"

namespace pisa {

// pisa_quantize_int8 of rows, which clears a status word on its way (int8_rows.cu)
int quantize_rows(const void* x, int64_t x_st, int dtype, int64_t rows, int64_t D, int8_t* q, int64_t q_st, float* scale, int* status,
                  cudaStream_t s);

namespace {

constexpr int kM = 128;          // output channels of a tile
constexpr int kStepBytes = 128;  // bytes of K per stage
constexpr int kThreads = 320;    // a warp of loads, one of products, eight of stores
constexpr int kSmem = 220 * 1024;

struct LinArgs {
  CUtensorMap tm_w, tm_x;
  const float* w_scale;
  const float* x_scale;
  const void* bias;     // or NULL
  int bias_f32;
  int T, O, steps;      // steps: K in blocks of 128 bytes
  int bn;               // tokens of a tile, a multiple of 16
  uint32_t tiles_o, tiles;
  uint32_t split;       // CTAs that share a tile
  uint32_t tries;
  void* out;
  int* status;
  // floating tokens that the kernel rounds itself
  const void* x;
  int64_t x_st;
  int x_dtype, x_wide, K;   // x_wide: rows start on 16 bytes and K is a multiple of 8
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint64_t* mbar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(tc::smem_u32(mbar)) : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T of signed bytes, 32 of K.
__device__ __forceinline__ void mma_i8(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, p;\n\t}"
      :: "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh) : "memory");
}

// Instruction descriptor of kind::i8: int32 sums of signed bytes, both operands K-major.
__device__ __forceinline__ uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

constexpr int kRoundTokens = 16, kRoundSteps = 48;   // tokens that a CTA rounds itself, steps of K that it holds of them

// ROUND: stages hold weights only, the tokens' bytes lie behind them.
template <int BN, bool ROUND = false>
struct Tile {
  static constexpr int A_BYTES = kM * kStepBytes, B_BYTES = BN * kStepBytes, STAGE = A_BYTES + (ROUND ? 0 : B_BYTES);
  static constexpr int STAGES = ROUND ? 7 : (kSmem - 1024) / STAGE < 10 ? (kSmem - 1024) / STAGE : 10;
  static constexpr int SMEM = STAGES * STAGE + (ROUND ? kRoundSteps * B_BYTES : 0) + 1024;
  static constexpr int COLS = BN < 32 ? 32 : BN;             // TMEM columns of an accumulator
};

// Pieces p, p + step, ... (U of 8 elements) of a token, zeros past its end.
template <typename X, bool WIDE, int U>
__device__ __forceinline__ void token_pieces(const X* row, int p, int step, int K, Raw8<X> (&r)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (p + u * step) * 8;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < int(sizeof(X) / 2); ++i)
        r[u].v[i] = c < K ? __ldg(reinterpret_cast<const uint4*>(row + c) + i) : make_uint4(0, 0, 0, 0);
    } else {
      X e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = c + i < K ? row[c + i] : from_f32<X>(0.f);
      r[u] = *reinterpret_cast<const Raw8<X>*>(e);
    }
  }
}

// The storing warps (256 threads, as many for each token) round the tokens as
// pisa_quantize_int8 does; the bytes of steps k0 .. k1 - 1 go to 128-byte-swizzled
// tiles of 16 rows from `at` on, scales to `scale`.  Rows past the last token are
// not written: no one stores their products.
template <typename X, bool WIDE>
__device__ __forceinline__ void round_tokens(const LinArgs& a, uint32_t at, int k0, int k1, float* scale, float* red) {
  constexpr int U = 16 / int(sizeof(X));
  int lg = 0;
  while ((1 << lg) < a.T) ++lg;
  const int id = int(threadIdx.x) - 64, each = 256 >> lg, row = id / each, t = id % each;
  const X* x = static_cast<const X*>(a.x) + int64_t(min(row, a.T - 1)) * a.x_st;
  float top = 0.f;
  for (int p = t; p * 8 < a.K; p += U * each) {
    Raw8<X> r[U];
    token_pieces<X, WIDE, U>(x, p, each, a.K, r);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      widen8<X>(r[u], f);
      top = larger(top, largest8<X>(r[u], f));
    }
  }
  for (int o = min(each, 32) / 2; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(kFull, top, o));
  if (each > 32) {
    if ((id & 31) == 0) red[id >> 5] = top;
    tc::named_sync(1, 256);
    for (int w = row * each >> 5; w < (row + 1) * each >> 5; ++w) top = larger(top, red[w]);
  }
  const Scale8 s(top);
  if (t == 0) scale[row] = s.scale;
  if (row < a.T) {
    for (int p = k0 * 16 + t; p < k1 * 16; p += U * each) {
      Raw8<X> r[U];
      token_pieces<X, WIDE, U>(x, p, each, a.K, r);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int n = p + u * each;
        if (n >= k1 * 16) break;
        float f[8];
        widen8<X>(r[u], f);
        uint2 q = pack8_s8(f, s.inv);
        if (!(top < INFINITY)) q = make_uint2(0, 0);
        const uint32_t to = at + uint32_t((n >> 4) - k0) * (kRoundTokens * kStepBytes) + tc::swizzle128(row, (n & 15) >> 1) + (n & 1) * 8;
        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" :: "r"(to), "r"(q.x), "r"(q.y) : "memory");
      }
    }
  }
  tc::fence_async_smem();
}
template <typename X>
__device__ __forceinline__ void round_tokens(const LinArgs& a, uint32_t at, int k0, int k1, float* scale, float* red) {
  if (a.x_wide) round_tokens<X, true>(a, at, k0, k1, scale, red);
  else round_tokens<X, false>(a, at, k0, k1, scale, red);
}
__device__ __forceinline__ void round_tokens(const LinArgs& a, uint32_t at, int k0, int k1, float* scale, float* red, uint64_t* ready) {
  if (a.x_dtype == PISA_F32) round_tokens<float>(a, at, k0, k1, scale, red);
  else if (a.x_dtype == PISA_BF16) round_tokens<__nv_bfloat16>(a, at, k0, k1, scale, red);
  else round_tokens<__half>(a, at, k0, k1, scale, red);
  tc::named_sync(1, 256);
  if ((threadIdx.x & 31) == 0) tc::mbar_arrive(ready);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 tokens of one channel per lane, stored token by token: 32 consecutive
// channels per warp.  `whole`: all 32 tokens and channels exist (the warp takes
// one path without a test per store; those cost half of its instructions).
template <typename T>
__device__ __forceinline__ void store_columns(const float (&v)[32], T* out, int64_t O, int t, int T_, int o, int O_, bool pairs,
                                              bool whole) {
  if constexpr (sizeof(T) == 2) {
    if (pairs) {
      // neighbouring lanes swap, so that each holds both channels of a pair for every other token
      const bool odd = threadIdx.x & 1;
      const uint32_t pick = odd ? 0x3276u : 0x5410u;
      T* at = out + int64_t(t + odd) * O + (o & ~1);
      uint32_t r[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t own = pack2<T>(v[2 * j], v[2 * j + 1]);
        r[j] = __byte_perm(own, __shfl_xor_sync(kFull, own, 1), pick);
      }
      if (whole) {
#pragma unroll
        for (int j = 0; j < 16; ++j, at += 2 * O) *reinterpret_cast<uint32_t*>(at) = r[j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j, at += 2 * O)
          if (t + 2 * j + odd < T_ && o < O_) *reinterpret_cast<uint32_t*>(at) = r[j];
      }
      return;
    }
  }
  T* at = out + int64_t(t) * O + o;
  if (whole) {
#pragma unroll
    for (int j = 0; j < 32; ++j, at += O) *at = from_f32<T>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j, at += O)
      if (t + j < T_ && o < O_) *at = from_f32<T>(v[j]);
  }
}

// 32 columns of a finished tile, scaled and stored for tokens t .. t1 - 1 (columns past the tile's tokens are not the product's).
template <typename T>
__device__ __forceinline__ void store_tile(const LinArgs& a, uint32_t tmem, const float* xs, float ws, float bias, int t, int t1, int o,
                                           bool pairs) {
  float v[32];
  tc::tmem_ld32(tmem, v);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 s = *reinterpret_cast<const float4*>(xs + j);
    v[j] = fmaf(float(__float_as_int(v[j])) * ws, s.x, bias);
    v[j + 1] = fmaf(float(__float_as_int(v[j + 1])) * ws, s.y, bias);
    v[j + 2] = fmaf(float(__float_as_int(v[j + 2])) * ws, s.z, bias);
    v[j + 3] = fmaf(float(__float_as_int(v[j + 3])) * ws, s.w, bias);
  }
  const bool whole = t + 32 <= t1 && (o | 31) < a.O;
  store_columns<T>(v, static_cast<T*>(a.out), a.O, t, t1, o, a.O, pairs, whole);
}

template <typename T, int BN, bool ROUND>
__global__ void __launch_bounds__(kThreads) int8_linear_kernel(const __grid_constant__ LinArgs a) {
  using L = Tile<BN, ROUND>;
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES], acc_full[2], acc_empty[2], drained, x_ready;
  __shared__ uint32_t slot;
  __shared__ WaitFlag wait;
  __shared__ __align__(16) float s_xs[8][BN < 32 ? 32 : BN];
  __shared__ float s_scale[kRoundTokens], s_red[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (tc::smem_u32(raw) + 1023u) & ~1023u;
  auto load = [&](int st, int k, uint32_t tt, uint32_t to) {
    const uint32_t at = base + st * L::STAGE;
    tc::mbar_arrive_expect_tx(&full[st], uint32_t(L::A_BYTES + (ROUND ? 0 : a.bn * kStepBytes)));
    tma_load_2d(at, &a.tm_w, k * kStepBytes, int(to) * kM, &full[st]);
    if (!ROUND) tma_load_2d(at + L::A_BYTES, &a.tm_x, k * kStepBytes, int(tt) * a.bn, &full[st]);
  };
  if (warp == 0 && lane == 0) {
    prefetch_map(&a.tm_w);
    if (!ROUND) prefetch_map(&a.tm_x);
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 8);
    }
    tc::mbar_init(&drained, 1);
    tc::mbar_init(&x_ready, 8);
    tc::fence_barrier_init();
    wait.init(a.tries);
    // the first stages are on their way while the others get ready (the first tile of a CTA always exists)
    const uint32_t tt = blockIdx.x / a.tiles_o, to = blockIdx.x - tt * a.tiles_o;
    for (int k = 0; k < min(L::STAGES, a.steps); ++k) load(k, k, tt, to);
  }
  if (warp == 1) tc::tmem_alloc(&slot, 2 * L::COLS);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = slot, x_at = base + L::STAGES * L::STAGE;
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int loads = min(L::STAGES, a.steps), st = loads % L::STAGES, k = loads;
      uint32_t phase = loads == L::STAGES ? 0 : 1;
      for (uint32_t tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x, k = 0) {
        const uint32_t tt = tile / a.tiles_o, to = tile - tt * a.tiles_o;
        for (; k < a.steps; ++k) {
          if (!(ok = wait_phase(&empty[st], int(phase), &wait))) break;
          load(st, k, tt, to);
          ++loads;
          if (++st == L::STAGES) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      // nothing may arrive after the CTA's end: the stages in use have been
      // handed back (after an expired wait: their copies have landed)
      for (int x = max(0, loads - L::STAGES); x < loads; ++x)
        wait_phase(ok ? &empty[x % L::STAGES] : &full[x % L::STAGES], x / L::STAGES, &wait);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t idesc = idesc_i8(kM, a.bn);
    int st = 0, n = 0;
    uint32_t phase = 0;
    if (ROUND) ok = wait_phase(&x_ready, 0, &wait);
    for (uint32_t tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x, ++n) {
      const int buf = n & 1;
      if (n >= 2) ok = wait_phase(&acc_empty[buf], (n >> 1) - 1, &wait);
      tc::fence_after_sync();
      const uint32_t d = tmem + buf * L::COLS;
#pragma unroll 1
      for (int k = 0; k < a.steps; ++k) {
        ok = wait_phase(&full[st], int(phase), &wait) && ok;
        if (!__all_sync(kFull, ok)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        if (leader) {
          const uint32_t al = desc_low(base + st * L::STAGE, 16), bl = desc_low(ROUND ? x_at + k * L::B_BYTES : base + st * L::STAGE + L::A_BYTES, 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) mma_i8(d, al + 2 * i, bl + 2 * i, idesc, k > 0 || i > 0);
          tc::mma_commit(&empty[st]);
          if (k + 1 == a.steps) tc::mma_commit(&acc_full[buf]);
        }
        __syncwarp();
        if (++st == L::STAGES) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    if (!__all_sync(kFull, ok)) {
      if (leader) tc::mma_commit(&drained);
      wait_phase(&drained, 0, &wait);
    }
    __syncwarp();
  } else {
    // TMEM lanes that this warp may read; two warps share them, with every other 32 tokens each
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    float* xs = s_xs[warp - 2];
    const bool pairs = (a.O & 1) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0;
    if (ROUND) round_tokens(a, x_at, 0, a.steps, s_scale, s_red, &x_ready);
    int n = 0;
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++n) {
      const int buf = n & 1;
      const uint32_t tt = tile / a.tiles_o, to = tile - tt * a.tiles_o;
      const int t0 = int(tt) * a.bn, t1 = min(a.T, t0 + a.bn), o = int(to) * kM + quarter * 32 + lane;
      __syncwarp();
      for (int i = half * 32 + lane; i < a.bn; i += 64) xs[i] = t0 + i < a.T ? (ROUND ? s_scale[i] : a.x_scale[t0 + i]) : 0.f;
      const float ws = o < a.O ? a.w_scale[o] : 0.f;
      float bias = 0.f;
      if (a.bias && o < a.O) bias = a.bias_f32 ? static_cast<const float*>(a.bias)[o] : to_f32<T>(static_cast<const T*>(a.bias)[o]);
      __syncwarp();
      ok = wait_phase(&acc_full[buf], n >> 1, &wait) && ok;
      if (!__all_sync(kFull, ok)) break;
      tc::fence_after_sync();
#pragma unroll 1
      for (int c = half * 32; c < a.bn; c += 64) store_tile<T>(a, tmem + buf * L::COLS + c + lanes, xs + c, ws, bias, t0 + c, t1, o, pairs);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (threadIdx.x == 0 && wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == 1) tc::tmem_free(tmem, 2 * L::COLS);
}

// ---------------------------------------------------------------------------
// Tiles of 256 channels for pairs of CTAs: each loads its 128 channels and half
// of the tokens, and one issues MMAs (cta_group::2) that read both shared
// memories and sum each CTA's channels in its own TMEM.  A pair moves two thirds
// of the bytes per product of two separate tiles of 128 x 256.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t leader_address(const void* p) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(tc::smem_u32(p)));
  return at;
}
// Into this CTA's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(mbar) : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, p;\n\t}"
      :: "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(uint32_t(accumulate)), "r"(kDescHigh) : "memory");
}
// Arrive on `mbar` of both CTAs once the pair's MMAs so far have completed.
__device__ __forceinline__ void commit_pair(uint64_t* mbar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               :: "r"(tc::smem_u32(mbar)), "h"(uint16_t(3)) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t mbar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(mbar) : "memory");
}

struct PairTile {
  static constexpr int A_BYTES = kM * kStepBytes, B_BYTES = 128 * kStepBytes, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 6, SMEM = STAGES * STAGE + 1024, COLS = 256;
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads) int8_linear_pair_kernel(const __grid_constant__ LinArgs a) {
  using L = PairTile;
  extern __shared__ __align__(16) uint8_t raw[];
  // full and acc_empty are the leader's; the other CTA counts on them from afar
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t slot;
  __shared__ WaitFlag wait;
  __shared__ __align__(16) float s_xs[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t rank = blockIdx.x & 1, pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  if (warp == 0 && lane == 0) {
    prefetch_map(&a.tm_w);
    prefetch_map(&a.tm_x);
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 16);
    }
    tc::mbar_init(&drained, 1);
    tc::fence_barrier_init();
    wait.init(a.tries);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(tc::smem_u32(&slot)), "r"(2 * L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = slot;
  const int half_tokens = a.bn / 2;
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      const uint32_t stage_bytes = uint32_t(2 * (L::A_BYTES + half_tokens * kStepBytes));   // of both CTAs
      int st = 0, loads = 0;
      uint32_t phase = 1;
      for (uint32_t tile = first; tile < a.tiles && ok; tile += pairs) {
        const uint32_t tt = tile / a.tiles_o, to = tile - tt * a.tiles_o;
        const int o = int(to * 2 + rank) * kM, t = int(tt) * a.bn + int(rank) * half_tokens;
        for (int k = 0; k < a.steps; ++k) {
          if (!(ok = wait_phase(&empty[st], int(phase), &wait))) break;
          const uint32_t at = base + st * L::STAGE, bar = leader_address(&full[st]);
          if (rank == 0) tc::mbar_arrive_expect_tx(&full[st], stage_bytes);
          tma_load_2d_pair(at, &a.tm_w, k * kStepBytes, o, bar);
          tma_load_2d_pair(at + L::A_BYTES, &a.tm_x, k * kStepBytes, t, bar);
          ++loads;
          if (++st == L::STAGES) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      // Nothing may arrive after the pair's end, which both CTAs reach together:
      // stages have been handed back to both; after an expired wait the leader
      // sees both CTAs' copies land, or waits its limit out.
      if (ok || rank == 0)
        for (int x = max(0, loads - L::STAGES); x < loads; ++x)
          wait_phase(ok ? &empty[x % L::STAGES] : &full[x % L::STAGES], x / L::STAGES, &wait);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      const uint32_t idesc = idesc_i8(2 * kM, a.bn);
      int st = 0, n = 0;
      uint32_t phase = 0;
      for (uint32_t tile = first; tile < a.tiles && ok; tile += pairs, ++n) {
        const int buf = n & 1;
        if (n >= 2) ok = wait_phase(&acc_empty[buf], (n >> 1) - 1, &wait);
        tc::fence_after_sync();
        const uint32_t d = tmem + buf * L::COLS;
#pragma unroll 1
        for (int k = 0; k < a.steps; ++k) {
          ok = wait_phase(&full[st], int(phase), &wait) && ok;
          if (!__all_sync(kFull, ok)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          if (leader) {
            const uint32_t al = desc_low(base + st * L::STAGE, 16), bl = desc_low(base + st * L::STAGE + L::A_BYTES, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma_i8_pair(d, al + 2 * i, bl + 2 * i, idesc, k > 0 || i > 0);
            commit_pair(&empty[st]);
            if (k + 1 == a.steps) commit_pair(&acc_full[buf]);
          }
          __syncwarp();
          if (++st == L::STAGES) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      if (!__all_sync(kFull, ok)) {
        if (leader) commit_pair(&drained);
        wait_phase(&drained, 0, &wait);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    float* xs = s_xs[warp - 2];
    const bool pairwise = (a.O & 1) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0;
    int n = 0;
    for (uint32_t tile = first; tile < a.tiles; tile += pairs, ++n) {
      const int buf = n & 1;
      const uint32_t tt = tile / a.tiles_o, to = tile - tt * a.tiles_o;
      const int t0 = int(tt) * a.bn, t1 = min(a.T, t0 + a.bn), o = int(to * 2 + rank) * kM + quarter * 32 + lane;
      __syncwarp();
      for (int i = half * 32 + lane; i < a.bn; i += 64) xs[i] = t0 + i < a.T ? a.x_scale[t0 + i] : 0.f;
      const float ws = o < a.O ? a.w_scale[o] : 0.f;
      float bias = 0.f;
      if (a.bias && o < a.O) bias = a.bias_f32 ? static_cast<const float*>(a.bias)[o] : to_f32<T>(static_cast<const T*>(a.bias)[o]);
      __syncwarp();
      ok = wait_phase(&acc_full[buf], n >> 1, &wait) && ok;
      if (!__all_sync(kFull, ok)) break;
      tc::fence_after_sync();
#pragma unroll 1
      for (int c = half * 32; c < a.bn; c += 64) store_tile<T>(a, tmem + buf * L::COLS + c + lanes, xs + c, ws, bias, t0 + c, t1, o, pairwise);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(leader_address(&acc_empty[buf]));
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (threadIdx.x == 0 && wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  cluster_sync();   // the other CTA's signals have arrived, its reads of this one's shared memory are done
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(2 * L::COLS) : "memory");
}

__device__ __forceinline__ int4 load_peer(uint32_t addr, int rank) {
  int4 v;
  asm volatile("{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %4, %5;\n\tld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [at];\n\t}"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "r"(rank));
  return v;
}

// A warp's tokens c, c + step, ... below c1 of a tile split over S ranges of K:
// four channels per lane, the sums of several tokens on their way at a time.
template <typename T, int S>
__device__ __forceinline__ void join(const LinArgs& a, const float* x_scale, uint32_t base, int c, int c1, int step, int64_t t0, int o) {
  constexpr int U = S == 8 ? 2 : 4;
  const int lane = threadIdx.x & 31, left = a.O - o;
  float ws[4], bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ws[i] = i < left ? a.w_scale[o + i] : 0.f;
    bias[i] = 0.f;
    if (a.bias && i < left)
      bias[i] = a.bias_f32 ? static_cast<const float*>(a.bias)[o + i] : to_f32<T>(static_cast<const T*>(a.bias)[o + i]);
  }
  const bool wide = left >= 4 && a.O % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & (4 * sizeof(T) - 1)) == 0;
  for (; c < c1; c += U * step) {
    int4 v[U][S];
    float xs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(c + u * step, c1 - 1);
      xs[u] = x_scale[at];
#pragma unroll
      for (int r = 0; r < S; ++r) v[u][r] = load_peer(base + uint32_t(at * kM + lane * 4) * 4, r);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * step >= c1) break;
      int4 sum = v[u][0];
#pragma unroll
      for (int r = 1; r < S; ++r) {
        sum.x += v[u][r].x;
        sum.y += v[u][r].y;
        sum.z += v[u][r].z;
        sum.w += v[u][r].w;
      }
      const float y[4] = {fmaf(float(sum.x) * ws[0], xs[u], bias[0]), fmaf(float(sum.y) * ws[1], xs[u], bias[1]),
                          fmaf(float(sum.z) * ws[2], xs[u], bias[2]), fmaf(float(sum.w) * ws[3], xs[u], bias[3])};
      T* out = static_cast<T*>(a.out) + (t0 + c + u * step) * a.O + o;
      if (wide) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
        else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) out[i] = from_f32<T>(y[i]);
      }
    }
  }
}

// One tile per cluster of a.split CTAs.
template <typename T, int BN, bool ROUND>
__global__ void __launch_bounds__(kThreads) int8_linear_split_kernel(const __grid_constant__ LinArgs a) {
  using L = Tile<BN, ROUND>;
  static_assert(BN * kM * 4 <= L::STAGES * L::STAGE && (!ROUND || BN == kRoundTokens), "the sums take the stages' place");
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES], acc_full, drained, x_ready;
  __shared__ uint32_t slot;
  __shared__ WaitFlag wait;
  __shared__ float s_scale[kRoundTokens], s_red[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t tile = blockIdx.x / a.split, rank = blockIdx.x - tile * a.split;   // rank: clusters are runs of a.split CTAs
  const uint32_t tt = tile / a.tiles_o, to = tile - tt * a.tiles_o;
  const int k0 = int(int64_t(a.steps) * rank / a.split), k1 = int(int64_t(a.steps) * (rank + 1) / a.split);
  auto load = [&](int st, int k) {
    const uint32_t at = base + st * L::STAGE;
    tc::mbar_arrive_expect_tx(&full[st], uint32_t(L::A_BYTES + (ROUND ? 0 : a.bn * kStepBytes)));
    tma_load_2d(at, &a.tm_w, k * kStepBytes, int(to) * kM, &full[st]);
    if (!ROUND) tma_load_2d(at + L::A_BYTES, &a.tm_x, k * kStepBytes, int(tt) * a.bn, &full[st]);
  };
  const int early = min(L::STAGES, k1 - k0);
  if (warp == 0 && lane == 0) {
    prefetch_map(&a.tm_w);
    if (!ROUND) prefetch_map(&a.tm_x);
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&acc_full, 1);
    tc::mbar_init(&drained, 1);
    tc::mbar_init(&x_ready, 8);
    tc::fence_barrier_init();
    wait.init(a.tries);
    for (int i = 0; i < early; ++i) load(i, k0 + i);   // on their way while the others get ready
  }
  if (warp == 1) tc::tmem_alloc(&slot, L::COLS);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = slot, x_at = base + L::STAGES * L::STAGE;
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int loads = early, st = loads % L::STAGES;
      uint32_t phase = loads == L::STAGES ? 0 : 1;
      for (int k = k0 + early; k < k1; ++k) {
        if (!(ok = wait_phase(&empty[st], int(phase), &wait))) break;
        load(st, k);
        ++loads;
        if (++st == L::STAGES) {
          st = 0;
          phase ^= 1;
        }
      }
      for (int x = max(0, loads - L::STAGES); x < loads; ++x)
        wait_phase(ok ? &empty[x % L::STAGES] : &full[x % L::STAGES], x / L::STAGES, &wait);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t idesc = idesc_i8(kM, a.bn);
    int st = 0;
    uint32_t phase = 0;
    if (ROUND) ok = wait_phase(&x_ready, 0, &wait);
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
      ok = wait_phase(&full[st], int(phase), &wait) && ok;
      if (!__all_sync(kFull, ok)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      if (leader) {
        const uint32_t al = desc_low(base + st * L::STAGE, 16), bl = desc_low(ROUND ? x_at + (k - k0) * L::B_BYTES : base + st * L::STAGE + L::A_BYTES, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_i8(tmem, al + 2 * i, bl + 2 * i, idesc, k > k0 || i > 0);
        tc::mma_commit(&empty[st]);
        if (k + 1 == k1) tc::mma_commit(&acc_full);
      }
      __syncwarp();
      if (++st == L::STAGES) {
        st = 0;
        phase ^= 1;
      }
    }
    if (!__all_sync(kFull, ok)) {
      if (leader) tc::mma_commit(&drained);
      wait_phase(&drained, 0, &wait);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const uint32_t mine = base + (quarter * 32 + lane) * 4;      // sums: [token][channel]
    if (ROUND) round_tokens(a, x_at, k0, k1, s_scale, s_red, &x_ready);
    // the sums' products are done, so every stage has been read
    ok = wait_phase(&acc_full, 0, &wait);
    tc::fence_after_sync();
    if (__all_sync(kFull, ok)) {
#pragma unroll 1
      for (int c = (warp - 2) >> 2 << 4; c < a.bn; c += 32) {
        float v[16];
        tc::tmem_ld16(tmem + c + (uint32_t(quarter * 32) << 16), v);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          asm volatile("st.shared.f32 [%0], %1;" :: "r"(mine + uint32_t(c + j) * (kM * 4)), "f"(v[j]) : "memory");
      }
    }
    __syncwarp();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (threadIdx.x == 0 && wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == 1) tc::tmem_free(tmem, L::COLS);
  cluster_sync();
  const int64_t t0 = int64_t(tt) * a.bn;
  const int c0 = int(a.bn * rank / a.split), c1 = int(min64(a.bn * (rank + 1) / a.split, a.T - t0)), o = int(to) * kM + lane * 4;
  const float* x_scale = ROUND ? s_scale : a.x_scale + t0;
  if (a.split == 2) join<T, 2>(a, x_scale, base, c0 + warp, c1, kThreads / 32, t0, o);
  else if (a.split == 4) join<T, 4>(a, x_scale, base, c0 + warp, c1, kThreads / 32, t0, o);
  else join<T, 8>(a, x_scale, base, c0 + warp, c1, kThreads / 32, t0, o);
  cluster_sync();   // no CTA leaves while another reads its sums
}

// 2-D map over rows of bytes: a box of 128 bytes of `box` rows, 128-byte
// swizzle; bytes past a row's end and rows past the last read as zero.
int byte_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int64_t stride, uint32_t box) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  if (!encode) return fail(PISA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {cuuint64_t(K), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride)};
  const cuuint32_t boxes[2] = {cuuint32_t(kStepBytes), box}, steps[2] = {1u, 1u};
  for (int tries = 0; tries < 2; ++tries) {
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, steps,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return PISA_OK;
    // a thread whose first CUDA call this is has no context until a runtime call binds the device's
    if (cudaFree(nullptr) != cudaSuccess) return fail(PISA_ERR_CUDA, "no CUDA context");
  }
  return fail(PISA_ERR_UNSUPPORTED, "tensor map encoding rejected the operand layout");
}

struct Operands {
  const void* x;
  int64_t x_st;
  const void* w;
  int64_t w_st, K;
};

// Tokens of a tile of at most `most`: as many for each tile, in whole sixteens.
int tile_tokens(int64_t T, int most) {
  const int64_t tiles = (T + most - 1) / most;
  return int(((T + tiles - 1) / tiles + 15) / 16 * 16);
}

template <typename T, int BN, bool ROUND = false>
int launch(LinArgs a, const Operands& m, int split, cudaStream_t s) {
  using L = Tile<BN, ROUND>;
  a.bn = tile_tokens(a.T, BN);
  int rc = byte_map(&a.tm_w, m.w, a.O, m.K, m.w_st, kM);
  if (!ROUND && rc == PISA_OK) rc = byte_map(&a.tm_x, m.x, a.T, m.K, m.x_st, uint32_t(a.bn));
  if (rc) return rc;
  a.tiles_o = uint32_t((a.O + kM - 1) / kM);
  const int64_t tiles = int64_t(a.tiles_o) * ((a.T + a.bn - 1) / a.bn);
  if (tiles >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  a.tiles = uint32_t(tiles);
  a.split = uint32_t(split);
  if (split == 1) {
    if ((rc = allow_smem<int8_linear_kernel<T, BN, ROUND>>(L::SMEM, "8-bit product smem attribute"))) return rc;
    int8_linear_kernel<T, BN, ROUND><<<unsigned(min64(tiles, sm_count())), kThreads, L::SMEM, s>>>(a);
    PISA_CHECK_LAUNCH();
    return PISA_OK;
  }
  if ((rc = allow_smem<int8_linear_split_kernel<T, BN, ROUND>>(L::SMEM, "8-bit product smem attribute"))) return rc;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = unsigned(split);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.gridDim = dim3(unsigned(tiles * split));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = L::SMEM;
  config.stream = s;
  config.attrs = &cluster;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, int8_linear_split_kernel<T, BN, ROUND>, a) != cudaSuccess) return fail_cuda(cudaGetLastError(), "8-bit product");
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T>
int launch_pairs(LinArgs a, const Operands& m, cudaStream_t s) {
  a.bn = (tile_tokens(a.T, 256) + 31) / 32 * 32;      // halves of whole sixteens
  int rc = byte_map(&a.tm_w, m.w, a.O, m.K, m.w_st, kM);
  if (rc == PISA_OK) rc = byte_map(&a.tm_x, m.x, a.T, m.K, m.x_st, uint32_t(a.bn / 2));
  if (rc == PISA_OK) rc = allow_smem<int8_linear_pair_kernel<T>>(PairTile::SMEM, "8-bit product smem attribute");
  if (rc) return rc;
  a.tiles_o = uint32_t((a.O + 2 * kM - 1) / (2 * kM));
  const int64_t tiles = int64_t(a.tiles_o) * ((a.T + a.bn - 1) / a.bn);
  if (tiles >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  a.tiles = uint32_t(tiles);
  int8_linear_pair_kernel<T><<<unsigned(2 * min64(tiles, (sm_count() + 1) / 2)), kThreads, PairTile::SMEM, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

// Tokens of a tile (at most), CTAs that share one, and whether pairs of CTAs take tiles of 256 channels (split 0).
struct Shape {
  int bn, split;
};

// The form with the least estimated time.  The estimates, in microseconds, are
// fits of measurements over tiles, splits and shapes (1 to 32768 tokens, K 16 to
// 16384, 96 to 60000 channels): a step of 128 bytes of K takes 0.235 + 0.00065 per
// token of the tile (16 tokens 0.245, 256 tokens 0.40), of a pair's tile 0.20 +
// 0.0005 (256 tokens 0.33), and all tiles' operands no less than HBM takes for
// them; storing a tile takes 0.75 + 0.0095 per token, a pair's 1 + 0.011, mostly under
// the next tile's steps; a split costs 1.3 and 0.008 per token, and clusters of 8
// fit on three quarters of the SMs.  Both sides of each choice: 16384 x 4096 x
// 11264 takes 499 us in single tiles and 437 in pairs, 8192 x 1024 x 5632 takes 45.6
// and 46.8; one token over 4096 x 4096 takes 11.6 us unsplit and 8.4 split by 4,
// over 1024 x 5632 5.7 and 6.8 (split by 2); 5110 x 64 x 3392 takes 13.9 us in tiles
// of 256 tokens and 34.1 of 32, 326 x 128 x 1088 takes 5.1 and 3.7.
Shape choose(int64_t T, int64_t O, int64_t steps, bool pairs = true) {
  const int64_t sms = sm_count();
  const double memory = double(T + O) * double(steps * kStepBytes) / 6.5e6;
  Shape best{256, 1};
  double least = 1e30;
  const auto consider = [&](int most, int split, int64_t ctas, int64_t room, double step, double store, double fixed) {
    const int64_t waves = (ctas + room - 1) / room;
    const double work = double((steps + (split > 1 ? split : 1) - 1) / (split > 1 ? split : 1)) * step;
    const double all = double(waves) * (work > store ? work + 0.1 * store : store + 0.1 * work);
    const double cost = fixed + store + (all > memory ? all : memory);
    if (cost < least) {
      least = cost;
      best = {most, split};
    }
  };
  for (int most = 16; most <= 256; most *= 2) {
    const int bn = tile_tokens(T, most);
    if (most > 16 && bn <= most / 2) break;
    const int64_t tiles = (O + kM - 1) / kM * ((T + bn - 1) / bn);
    for (int split = 1; split <= 8; split *= 2) {
      if (split > steps || (split > 1 && tiles * split > (split == 8 ? sms * 3 / 4 : sms))) break;
      consider(most, split, tiles * split, sms, 0.235 + 0.00065 * bn, 0.75 + 0.0095 * bn, split > 1 ? 5.3 + 0.008 * bn : 4.0);
    }
  }
  const int bn = (tile_tokens(T, 256) + 31) / 32 * 32;
  if (pairs) consider(256, 0, (O + 2 * kM - 1) / (2 * kM) * ((T + bn - 1) / bn), (sms + 1) / 2, 0.20 + 0.0005 * bn, 1.0 + 0.011 * bn, 4.5);
  return best;
}

// Whether the product's kernel rounds floating tokens itself, and its split: few
// elements, since every CTA reads them all, and no more steps per CTA than its
// shared memory holds.  Replayed in a graph, weights from HBM and tokens as the
// step before left them in L2, one launch takes less than rounding and product in
// two: 1024 -> 5632 6.5 us against 7.5 for one token, 7.3 and 7.7 for 16, 4096 ->
// 4096 9.6 and 10.7, 1024 -> 50257 14.0 and 15.4; of 33 sizes only 4 tokens of 4096 ->
// 16384 lose (17.4 and 17.1).  The host spends 14 us on one launch and 21 on two.
// Tokens that come from HBM too cost each CTA a wait of their own: 1024 -> 5632 9.7
// us for one and 10.2 for 16, where the two kernels alone take 2.1 + 5.9.
int rounds_itself(int64_t T, int64_t K, int64_t O) {
  if (T > kRoundTokens || T * K > 16384) return 0;
  const int64_t steps = (K + kStepBytes - 1) / kStepBytes;
  const Shape c = choose(T, O, steps, false);
  return (steps + c.split - 1) / c.split <= kRoundSteps ? c.split : 0;
}

template <typename T>
int dispatch(const LinArgs& a, const Operands& m, cudaStream_t s) {
  if (a.x) return launch<T, kRoundTokens, true>(a, m, rounds_itself(a.T, a.K, a.O), s);
  const Shape c = choose(a.T, a.O, a.steps);
  if (c.split == 0) return launch_pairs<T>(a, m, s);
  switch (c.bn) {
    case 16: return launch<T, 16>(a, m, c.split, s);
    case 32: return launch<T, 32>(a, m, c.split, s);
    case 64: return launch<T, 64>(a, m, c.split, s);
    case 128: return launch<T, 128>(a, m, c.split, s);
    default: return launch<T, 256>(a, m, c.split, s);
  }
}

}  // namespace

}  // namespace pisa

extern "C" {

// workspace: status word, then (floating x, unless the product's kernel rounds it) the tokens' scales and bytes
int64_t pisa_int8_linear_workspace_bytes(int64_t T, int64_t K, int64_t O, int x_dtype) {
  if (T <= 0 || K <= 0 || O <= 0 || x_dtype < PISA_F32 || x_dtype > PISA_S8) return -1;
  if (x_dtype == PISA_S8 || pisa::rounds_itself(T, K, O)) return 256;
  return 256 + (T * 4 + 255) / 256 * 256 + T * ((K + 15) / 16 * 16);
}

int pisa_int8_linear(const void* x, int64_t x_st, int x_dtype, const float* x_scale, const int8_t* weight, int64_t weight_st,
                     const float* weight_scale, const void* bias, int bias_dtype, int out_dtype, int64_t T, int64_t K, int64_t O,
                     void* out, void* workspace, int64_t workspace_bytes, pisa_stream_t stream) {
  using namespace pisa;
  const bool bytes = x_dtype == PISA_S8;
  if (out_dtype < PISA_F32 || out_dtype > PISA_F16 || x_dtype < PISA_F32 || x_dtype > PISA_S8)
    return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (bias && bias_dtype != out_dtype && bias_dtype != PISA_F32)
    return fail(PISA_ERR_UNSUPPORTED, "the bias must be FP32 or the output's type");
  if (T <= 0 || K <= 0 || O <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (K >= (int64_t(1) << 17)) return fail(PISA_ERR_UNSUPPORTED, "sums of 131072 or more products may not fit 32 bits");
  if (T >= (int64_t(1) << 31) - 256 || O >= (int64_t(1) << 31) - 256) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (!x || (bytes && !x_scale) || !weight || !weight_scale || !out)
    return fail(PISA_ERR_INVALID, "operands, scales and out are required");
  const int64_t row_bytes = (K + 15) / 16 * 16;
  if (T == 1 && bytes) x_st = row_bytes;          // the stride of a single row may hold anything
  if (O == 1) weight_st = row_bytes;
  if ((bytes && ((reinterpret_cast<uintptr_t>(x) & 15u) || x_st % 16)) || (reinterpret_cast<uintptr_t>(weight) & 15u) || weight_st % 16)
    return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must start on 16 bytes");
  if ((bytes && x_st < K) || weight_st < K) return fail(PISA_ERR_UNSUPPORTED, "8-bit rows must not overlap");
  const bool own = !bytes && rounds_itself(T, K, O);   // no workspace but for the status word
  if (workspace ? workspace_bytes < pisa_int8_linear_workspace_bytes(T, K, O, x_dtype) : !bytes && !own)
    return fail(PISA_ERR_INVALID, "workspace too small");
  if (!bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u)) return fail(PISA_ERR_INVALID, "workspace must start on 16 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LinArgs a{};
  a.status = static_cast<int*>(workspace);
  Operands m{x, x_st, weight, weight_st, K};
  if (bytes || own) {
    if (own) {
      a.x = x; a.x_st = x_st; a.x_dtype = x_dtype; a.K = int(K);
      a.x_wide = K % 8 == 0 && rows_on16(x, T, x_st * (x_dtype == PISA_F32 ? 4 : 2));
    }
    if (workspace) {
      cudaError_t e = cudaMemsetAsync(workspace, 0, 256, s);
      if (e != cudaSuccess) return fail_cuda(e, "status clear");
    }
  } else {
    float* scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
    int8_t* values = static_cast<int8_t*>(workspace) + 256 + (T * 4 + 255) / 256 * 256;
    if (int rc = quantize_rows(x, x_st, x_dtype, T, K, values, row_bytes, scale, a.status, s)) return rc;
    x_scale = scale;
    m.x = values;
    m.x_st = row_bytes;
  }
  a.w_scale = weight_scale; a.x_scale = x_scale; a.bias = bias; a.bias_f32 = bias_dtype == PISA_F32;
  a.T = int(T); a.O = int(O); a.steps = int((K + kStepBytes - 1) / kStepBytes);
  a.tries = wait_tries(a.steps);
  a.out = out;
  if (out_dtype == PISA_F32) return dispatch<float>(a, m, s);
  if (out_dtype == PISA_BF16) return dispatch<__nv_bfloat16>(a, m, s);
  return dispatch<__half>(a, m, s);
}

}  // extern "C"

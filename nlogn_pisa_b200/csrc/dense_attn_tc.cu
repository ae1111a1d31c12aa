// Dense attention forward on the tensor cores: 16-bit tensors, heads of at
// most 128 dims (formulas in dense_attn.cu).
//
// One CTA holds two tiles of 128 consecutive queries of one head and walks
// the keys of their sequence in tiles of 128:
//   MMA 1  S = Q K^T   (M = 128 queries, N = 128 keys)  -> TMEM
//   softmax in registers, two threads per query row, 64 keys each (no
//          shuffles); P rounded to the input type overwrites S in TMEM
//   MMA 2  O += P V    (A = P from TMEM, B = V with keys along K) -> TMEM
// The two query tiles take turns: while eight warps turn tile 0's scores into
// weights, the tensor core works for tile 1.  A tile's step is a chain (S,
// softmax, P V), so its length decides: two threads per row halve the softmax
// part and give every scheduler four warps to hide its latencies with.  Warps
// 0-7 and 8-15 are the two tiles' softmax warps, warp 16 issues the MMAs, warp
// 17 the TMA loads (a ring of value and key tiles).  TMEM: S/P of both tiles
// and O of both fill 512 columns at 128 dims.
//
// The running maximum only moves when a row's new maximum passes the one in
// use by 2^8: weights up to 256 are as exact in 16-bit floating point as
// weights up to 1, and O in TMEM is rescaled a few times per row instead of
// once per key tile.  P is rounded to the input type because the second MMA
// takes its operands so; sums of weights are taken before that rounding, in
// fp32.
//
// Hidden keys of a tile weigh zero, but zero times an infinite or NaN value
// is NaN.  A row whose output holds NaN although its weights do not is
// therefore summed again over its visible keys alone (row_again); rows past
// the sequence's end need nothing (they are not stored).
#include "dense_tc.cuh"

namespace pisa {

namespace {

constexpr int kMmaWarp = 16, kLoadWarp = 17;
constexpr int kThreads = 576;

struct FwdTcArgs {
  CUtensorMap tm_q, tm_k, tm_v;             // boxes of 64 dims x 128 rows of one head
  DenseAttnArgs d;
  int bf16;
};

template <int DP> struct FwdTile {
  static constexpr int CH = DP / 64;                    // 64-dim chunks
  static constexpr int BYTES = kRows * DP * 2;          // one operand tile
  // ring stages of the values of one key tile and the keys of the next; three
  // of 64 dims also keep a second CTA off the SM's TMEM
  static constexpr int STAGES = DP == 128 ? 2 : 3;
  static constexpr int SMEM = (2 + 2 * STAGES) * BYTES + 1024;
};

// Output row of query `i` summed over its visible keys alone, by one warp,
// with the row's maximum m and weight sum l (base 2): acc[e] of column
// lane + 32 e.  Stops once every column is NaN.
template <typename T, int DP>
__device__ __noinline__ void row_again(const DenseAttnArgs& a, const SeqTile& t, int hq, int i, float m, float l,
                                       float (&acc)[DP / 32]) {
  const int lane = threadIdx.x & 31, h = hq / a.G;
  const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + int64_t(t.q_begin + i) * a.q_st + hq * a.q_sh;
  const T* kp = static_cast<const T*>(a.k) + t.b * a.k_sb + int64_t(t.k_begin) * a.k_st + h * a.k_sh;
  const T* vp = static_cast<const T*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin) * a.v_st + h * a.v_sh;
  const float sl = a.scale * kLog2e;
  float q[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) {
    q[e] = lane + 32 * e < a.D ? to_f32<T>(qp[lane + 32 * e]) : 0.f;
    acc[e] = 0.f;
  }
  const int last = last_visible(a, t, i);
  for (int j = 0; j <= last; ++j) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e)
      if (lane + 32 * e < a.D) s = fmaf(q[e], to_f32<T>(kp[j * a.k_st + lane + 32 * e]), s);
    const float p = exp2f(fmaf(warp_sum(s), sl, -m));
    bool all = true;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
      if (lane + 32 * e < a.Dv) {
        acc[e] = fmaf(p, to_f32<T>(vp[j * a.v_st + lane + 32 * e]), acc[e]);
        all = all && isnan(acc[e]);
      }
    }
    if (__all_sync(kFull, all)) break;
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) acc[e] *= inv;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) dense_fwd_tc_kernel(const __grid_constant__ FwdTcArgs args) {
  using L = FwdTile<DP>;
  const DenseAttnArgs& a = args.d;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_addr = base, kv_addr = base + 2 * L::BYTES;
  __shared__ uint64_t q_full[2], kv_full[L::STAGES], kv_empty[L::STAGES], s_full[2], p_full[2], o_done[2], drained;
  __shared__ float s_other[2][2][kRows];      // the halves' maxima, at the end their sums
  __shared__ uint32_t tmem_slot;
  __shared__ int s_fail;
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  // the last query tiles, which see the most keys, first; heads of a tile side by side
  const int index = int(gridDim.x) - 1 - int(blockIdx.x);
  const int slot = index / a.Hq, hq = index - slot * a.Hq;
  const SeqTile t = seq_tile(a, slot, 2 * kRows, false);
  const int q0 = t.tile * 2 * kRows;
  if (q0 >= t.q_len) return;
  // key tiles that each query tile visits
  int tiles[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = q0 + i * kRows, rows = min(kRows, t.q_len - first);
    tiles[i] = rows > 0 ? (last_visible(a, t, first + rows - 1) + kRows) / kRows : 0;
  }
  const int most = max(tiles[0], tiles[1]);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&q_full[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 8);
      tc::mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
    }
    tc::mbar_init(&drained, 1);
    s_fail = 0;
    tc::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(kFull, tmem_slot, 0);
  // TMEM columns: S/P of the two tiles, then their O
  const uint32_t tS = tmem, tO = tmem + 256;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      const int h = hq / a.G;
      for (int i = 0; i < 2; ++i) {
        if (!tiles[i]) continue;
        tc::mbar_arrive_expect_tx(&q_full[i], L::BYTES);
        for (int c = 0; c < L::CH; ++c)
          tc::tma_load_4d(q_addr + i * L::BYTES + c * kRows * 128, &args.tm_q, c * 64, hq, t.q_begin + q0 + i * kRows, t.b,
                          &q_full[i]);
      }
      for (int j = 0; j <= most; ++j) {   // V_{j-1} and K_j
        const int st = j % L::STAGES;
        if (most == 0) break;
        if (!wait_phase(&kv_empty[st], (j / L::STAGES) + 1, &s_fail)) {
          // the copies in flight land before the CTA ends
          for (int x = max(0, j - L::STAGES); x < j; ++x) wait_phase(&kv_full[x % L::STAGES], x / L::STAGES, &s_fail);
          break;
        }
        const uint32_t v = kv_addr + st * 2 * L::BYTES, k = v + L::BYTES;
        tc::mbar_arrive_expect_tx(&kv_full[st], (int(j > 0) + int(j < most)) * L::BYTES);
#pragma unroll 1
        for (int c = 0; c < L::CH; ++c) {
          if (j < most)
            tc::tma_load_4d(k + c * kRows * 128, &args.tm_k, c * 64, h, t.k_begin + j * kRows, t.b, &kv_full[st]);
          if (j > 0)
            tc::tma_load_4d(v + c * kRows * 128, &args.tm_v, c * 64, h, t.k_begin + (j - 1) * kRows, t.b, &kv_full[st]);
        }
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    const uint32_t id_s = tc::idesc_f16(kRows, kRows, args.bf16), id_o = tc::idesc_f16(kRows, DP, args.bf16, 1);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) {
      if (ok && !wait_phase(bar, phase, &s_fail)) ok = false;
    };
    if (tiles[0]) wait(&q_full[0], 0);
    if (tiles[1]) wait(&q_full[1], 0);
    for (int j = 0; j <= most && most > 0 && __all_sync(kFull, ok); ++j) {
      const int st = j % L::STAGES;
      const uint32_t v = kv_addr + st * 2 * L::BYTES, k = v + L::BYTES;
      wait(&kv_full[st], j / L::STAGES);      // V_{j-1} and K_j
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int own = i ? tiles[1] : tiles[0];
        if (j >= 1 && j <= own) wait(&p_full[i], j - 1);
        tc::fence_after_sync();
        if (leader && ok) {
          if (j >= 1 && j <= own) {           // O += P V of key tile j - 1
            mma_cols(tO + i * DP, tS + i * 128, 64, v, id_o, kRows / 16, j > 1);
            if (j == own) tc::mma_commit(&o_done[i]);
          }
          if (j < own) {                      // S = Q K^T of key tile j
            mma_rows<DP>(tS + i * 128, q_addr + i * L::BYTES, k, id_s);
            tc::mma_commit(&s_full[i]);
          }
        }
        __syncwarp();
      }
      // a stage that no later tile takes is not handed back: nothing may arrive after the CTA's end
      if (leader && ok && j + L::STAGES <= most) tc::mma_commit(&kv_empty[st]);
    }
    if (!ok && leader) {
      tc::mma_commit(&drained);
      wait_phase(&drained, 0, &s_fail);
    }
    __syncwarp();
  } else {
    const int i = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
    const int qi = q0 + i * kRows + row;             // query of this thread
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tS + i * 128 + half * 64 + lanes, to = tO + i * DP + half * (DP / 2) + lanes;
    const bool real = qi < t.q_len;
    const int last = (real ? last_visible(a, t, qi) : -1) - half * 64;
    const float sl = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;                    // base-2 logits; l: of this half's keys
    bool ok = true;
    const int own = i ? tiles[1] : tiles[0];
    const int full = (last_visible(a, t, q0 + i * kRows) + 1) / kRows;   // key tiles that every row sees whole
    for (int j = 0; j < own; ++j) {
      ok = wait_phase(&s_full[i], j, &s_fail) && ok;
      tc::fence_after_sync();
      softmax_half<T, DP>(ts, to, sl, j == 0, j >= full ? last - j * kRows : kRows, 1 + i, s_other[i], half, row, m, l);
      tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[i]);
    }
    // O / l: each half stores its columns, through its share of the query
    // tile's shared memory (the tile's last S is complete before o_done)
    const bool any = own > 0;
    if (any) {
      ok = wait_phase(&o_done[i], 0, &s_fail) && ok;
      tc::fence_after_sync();
      s_other[i][half][row] = l;
      tc::named_sync(1 + i, 256);
      l += s_other[i][half ^ 1][row];
    }
    const float inv = !ok ? NAN : l == 0.f ? 0.f : 1.f / l;
    constexpr int W = DP / 2, SEG = W / 8;           // columns of a half, their 16-byte segments
    const uint32_t stage = q_addr + i * L::BYTES + (half * 4 + quarter) * 32 * W * 2;
    const int64_t row0 = int64_t(t.b) * a.T + t.q_begin + q0 + i * kRows + quarter * 32;
    const int rows = min(32, t.q_len - (q0 + i * kRows + quarter * 32));
    // pass 0 stores the rounded output, pass 1 what the rounding dropped
#pragma unroll 1
    for (int pass = 0; pass < (a.out_low ? 2 : 1); ++pass) {
      bool wild = false;
#pragma unroll 1
      for (int c = 0; c < W; c += 16) {
        float o[16];
        if (any) {
          tc::tmem_ld16(to + c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          wild = wild || isnan(o[e]);
          o[e] = l == 0.f && ok ? 0.f : o[e] * inv;
          if (pass) o[e] -= to_f32<T>(from_f32<T>(o[e]));
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int seg = c / 8 + s;
          st_shared16(stage + (lane * SEG + (seg ^ (lane & (SEG - 1)))) * 16, pack2<T>(o[8 * s], o[8 * s + 1]),
                      pack2<T>(o[8 * s + 2], o[8 * s + 3]), pack2<T>(o[8 * s + 4], o[8 * s + 5]),
                      pack2<T>(o[8 * s + 6], o[8 * s + 7]));
        }
      }
      __syncwarp();
      uint32_t again = __ballot_sync(kFull, ok && real && wild && l != 0.f && !isnan(l));
      while (again) {
        const int r = __ffs(again) - 1;
        again &= again - 1;
        float acc[DP / 32];
        row_again<T, DP>(a, t, hq, q0 + i * kRows + quarter * 32 + r, __shfl_sync(kFull, m, r), __shfl_sync(kFull, l, r),
                         acc);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) {
          const int d = lane + 32 * e - half * W;
          T v = from_f32<T>(acc[e]);
          if (pass) v = from_f32<T>(acc[e] - to_f32<T>(v));
          if (d >= 0 && d < W)
            asm volatile("st.shared.b16 [%0], %1;"
                         :: "r"(stage + (r * SEG + ((d >> 3) ^ (r & (SEG - 1)))) * 16 + (d & 7) * 2),
                            "h"(*reinterpret_cast<const uint16_t*>(&v)) : "memory");
        }
        __syncwarp();
      }
      T* out = static_cast<T*>(pass ? a.out_low : a.out) + half * W;
      for (int f = lane; f < rows * SEG; f += 32) {
        const int r = f / SEG, seg = f % SEG;
        const uint4 v = ld_shared16(stage + (r * SEG + (seg ^ (r & (SEG - 1)))) * 16);
        if (half * W + seg * 8 < a.Dv) *reinterpret_cast<uint4*>(out + ((row0 + r) * a.Hq + hq) * a.Dv + seg * 8) = v;
      }
      __syncwarp();
    }
    if (a.lse && real && half == 0)
      a.lse[(row0 + lane) * a.Hq + hq] = !ok ? NAN : l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (tid == 0 && s_fail && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == kMmaWarp) tc::tmem_free(tmem, 512);
}

template <typename T, int DP>
int fwd_t(const FwdTcArgs& a, cudaStream_t s) {
  using L = FwdTile<DP>;
  const int64_t blocks = seq_slots(a.d.cu_q, a.d.B, a.d.T, a.d.sequences, 2 * kRows) * a.d.Hq;
  if (blocks >= (int64_t(1) << 31)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (int rc = allow_smem<dense_fwd_tc_kernel<T, DP>>(L::SMEM, "dense attention smem attribute")) return rc;
  dense_fwd_tc_kernel<T, DP><<<unsigned(blocks), kThreads, L::SMEM, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

}  // namespace

bool dense_attn_tc_eligible(const DenseAttnArgs& a, int dtype) {
  return dtype != PISA_F32 && a.D <= 128 && a.Dv <= 128;
}

int dense_attn_fwd_tc(const DenseAttnArgs& d, int dtype, cudaStream_t stream) {
  FwdTcArgs a{};
  a.d = d;
  a.bf16 = dtype == PISA_BF16;
  int rc = dense_tensor_map(&a.tm_q, d.q, dtype, d.B, d.T, d.Hq, d.D, d.q_sb, d.q_st, d.q_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_k, d.k, dtype, d.B, d.N, d.H, d.D, d.k_sb, d.k_st, d.k_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_v, d.v, dtype, d.B, d.N, d.H, d.Dv, d.v_sb, d.v_st, d.v_sh, kRows);
  if (rc) return rc;
  const bool narrow = d.D <= 64 && d.Dv <= 64;
  if (dtype == PISA_BF16) return narrow ? fwd_t<__nv_bfloat16, 64>(a, stream) : fwd_t<__nv_bfloat16, 128>(a, stream);
  return narrow ? fwd_t<__half, 64>(a, stream) : fwd_t<__half, 128>(a, stream);
}

}  // namespace pisa

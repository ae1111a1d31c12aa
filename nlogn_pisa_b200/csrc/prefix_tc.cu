// The shared prefix of decode attention on the tensor cores, for batches with
// many query rows per KV head (formulas and partial results in
// prefix_attn.cu; the pipeline is that of dense_attn_tc.cu).
//
// The prefix is the same for every sequence, so the query rows of the whole
// batch (token by token, the G heads of a KV head side by side) form ordinary
// tiles of up to 128 rows, and its keys and values are read once for 256 of
// them.  One CTA takes a range of keys of one KV head.  With two row tiles or
// more, its two tiles share the stream of keys; with one, both halves hold the
// same rows and take every other key tile, so that the tensor core still
// works for one half while the other half's weights are computed, and their
// results join in shared memory.  The number of ranges follows from the own
// caches' lengths (prefix_share): CTAs without a range leave at once.
//
// Measured: 64 tokens of 32 query heads over 8192 shared keys (8 heads of 128):
// 18 us with all SMs for 8.6 GFLOP and 34 MB, 53 us on the few that end with the
// own caches' stream; 16 tokens over 65536: 48 us for 268 MB (5.5 TB/s) with all,
// 70 us beside the stream.  The streaming kernel reads a shared prefix once per 16 query rows: 195
// us for the first of these, which is why more than 16 rows come here.
#include "dense_tc.cuh"
#include "prefix_attn.cuh"

namespace pisa {

namespace {

constexpr int kMmaWarp = 8, kLoadWarp = 9, kThreads = 320;

struct PrefixTcArgs {
  CUtensorMap tm_q;                  // [B * T tokens, Hq, D], box of 64 dims x G heads x tokens of a tile
  CUtensorMap tm_k, tm_v;            // prefix, boxes of 64 dims x 128 keys of one head
  PrefixArgs p;
  int tokens, tiles;                 // tokens of a row tile, row tiles
  int bf16;
};

template <int DP> struct PrefixTile {
  static constexpr int CH = DP / 64, BYTES = kRows * DP * 2;
  static constexpr int STAGES = DP == 128 ? 4 : 6;      // 64 dims: also keeps a second CTA off the SM's TMEM
  static constexpr int SMEM = (2 + STAGES) * BYTES + 1024;
  static_assert(STAGES * BYTES >= kRows * (DP + 4) * 4, "half 1's output fits the ring");
};

__device__ __forceinline__ void st_global32(float* p, const float* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) prefix_tc_kernel(const __grid_constant__ PrefixTcArgs args) {
  using L = PrefixTile<DP>;
  const PrefixArgs& a = args.p;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_addr = base, kv_addr = base + 2 * L::BYTES;
  float* join = reinterpret_cast<float*>(smem_raw + (kv_addr - tc::smem_u32(smem_raw)));   // [128][DP + 4], after the ring's use
  __shared__ uint64_t q_full[2], kv_full[L::STAGES], kv_empty[L::STAGES], s_full[2], p_full[2], o_done[2], drained;
  __shared__ float2 join_ml[kRows];
  __shared__ int64_t s_own[kThreads / 32];
  __shared__ uint32_t tmem_slot;
  __shared__ WaitFlag s_wait;
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  cudaTriggerProgrammaticLaunchCompletion();   // the own caches' kernel may be scheduled
  // half a second before any wait can expire
  if (blockIdx.x + blockIdx.y + tid == 0) *a.status = PISA_OK;
  const int h = blockIdx.x % a.H, split = blockIdx.x / a.H;
  int64_t own = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) own += b0 + tid < a.B ? own_length(a, b0 + tid) : 0;
  for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(kFull, own, o);
  if (lane == 0) s_own[warp] = own;
  __syncthreads();
  own = 0;
  for (int w = 0; w < kThreads / 32; ++w) own += s_own[w];
  const PrefixShare share = prefix_share(a, own);
  if (blockIdx.x + blockIdx.y + tid == 0) a.status[1] = share.ranges;
  if (split >= share.ranges) return;
  const bool dual = args.tiles == 1;            // one row tile: the halves take every other key tile
  int begin, end;
  split_range(a.P, split, share.chunk, begin, end);
  const int keys = (end - begin + kRows - 1) / kRows;      // key tiles, at least one
  const int row_tile[2] = {dual ? 0 : int(blockIdx.y) * 2, dual ? 0 : int(blockIdx.y) * 2 + 1};
  const int steps[2] = {dual ? (keys + 1) / 2 : keys, dual ? keys / 2 : row_tile[1] < args.tiles ? keys : 0};
  const int most = max(steps[0], steps[1]);
  // ring position of the keys of half i's step s (its values: one more)
  auto position = [&](int i, int s) { return dual ? 2 * (2 * s + i) : 2 * s; };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&q_full[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 4);
      tc::mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
    }
    tc::mbar_init(&drained, 1);
    s_wait.init();
    tc::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(kFull, tmem_slot, 0);
  const uint32_t tS = tmem, tO = tmem + 256;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      const uint32_t q_bytes = uint32_t(args.tokens) * a.G * 128 * L::CH;
      for (int i = 0; i < 2; ++i) {
        if (!steps[i]) continue;
        tc::mbar_arrive_expect_tx(&q_full[i], q_bytes);
        for (int c = 0; c < L::CH; ++c)
          tc::tma_load_4d(q_addr + i * L::BYTES + c * kRows * 128, &args.tm_q, c * 64, h * a.G, row_tile[i] * args.tokens, 0,
                          &q_full[i]);
      }
      for (int n = 0; n < 2 * keys; ++n) {   // K0 V0 K1 V1 ...
        const int st = n % L::STAGES;
        if (!wait_phase(&kv_empty[st], (n / L::STAGES) + 1, &s_wait)) {
          // the copies in flight land before the CTA ends
          for (int x = max(0, n - L::STAGES); x < n; ++x) wait_phase(&kv_full[x % L::STAGES], x / L::STAGES, &s_wait);
          break;
        }
        tc::mbar_arrive_expect_tx(&kv_full[st], L::BYTES);
        const CUtensorMap* map = n & 1 ? &args.tm_v : &args.tm_k;
        for (int c = 0; c < L::CH; ++c)
          tc::tma_load_4d(kv_addr + st * L::BYTES + c * kRows * 128, map, c * 64, h, begin + (n >> 1) * kRows, 0, &kv_full[st]);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    const uint32_t id_s = tc::idesc_f16(kRows, kRows, args.bf16), id_o = tc::idesc_f16(kRows, DP, args.bf16, 1);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) { ok = wait_phase(bar, phase, &s_wait) && ok; };
    const int last = steps[1] ? 1 : 0;            // the half that hands a shared stage back
    for (int s = 0; s <= most && __all_sync(kFull, ok); ++s) {
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int own = i ? steps[1] : steps[0];
        // a stage that no later tile takes is not handed back: nothing may arrive after the CTA's end
        if (s >= 1 && s <= own) {                 // O += P V of step s - 1
          const int pos = position(i, s - 1) + 1, st = pos % L::STAGES;
          if (dual || i == 0) wait(&kv_full[st], pos / L::STAGES);
          wait(&p_full[i], s - 1);
          tc::fence_after_sync();
          if (leader && ok) {
            mma_cols(tO + i * DP, tS + i * 128, 32, kv_addr + st * L::BYTES, id_o, kRows / 16, s > 1);
            if (s == own) tc::mma_commit(&o_done[i]);
            if ((dual || i == last) && pos + L::STAGES < 2 * keys) tc::mma_commit(&kv_empty[st]);
          }
        }
        if (s < own) {                            // S = Q K^T of step s
          const int pos = position(i, s), st = pos % L::STAGES;
          if (s == 0) wait(&q_full[i], 0);
          if (dual || i == 0) wait(&kv_full[st], pos / L::STAGES);
          tc::fence_after_sync();
          if (leader && ok) {
            mma_rows<DP>(tS + i * 128, q_addr + i * L::BYTES, kv_addr + st * L::BYTES, id_s);
            tc::mma_commit(&s_full[i]);
            if ((dual || i == last) && pos + L::STAGES < 2 * keys) tc::mma_commit(&kv_empty[st]);
          }
        }
        __syncwarp();
      }
    }
    if (!__all_sync(kFull, ok)) {
      if (leader) tc::mma_commit(&drained);
      wait_phase(&drained, 0, &s_wait);
    }
    __syncwarp();
  } else {
    const int i = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tS + i * 128 + lanes, to = tO + i * DP + lanes;
    const float sl = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int s = 0; s < steps[i]; ++s) {
      ok = wait_phase(&s_full[i], s, &s_wait) && ok;
      tc::fence_after_sync();
      const int first = begin + (dual ? 2 * s + i : s) * kRows;
      softmax_tile<T, DP>(ts, to, sl, s == 0, end - 1 - first, m, l);
      tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[i]);
    }
    if (steps[i]) ok = wait_phase(&o_done[i], 0, &s_wait) && ok;
    tc::fence_after_sync();
    if (!ok) l = NAN;
    // half 1's result joins half 0's when they hold the same rows
    float mul = 1.f, mul1 = 0.f;
    if (dual) {
      if (i == 1) {
        // the ring is free once half 0's last product is done, too
        if (!wait_phase(&o_done[0], 0, &s_wait)) l = NAN;
        if (steps[1]) {
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            float o[32];
            tc::tmem_ld32(to + c, o);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(join + row * (DP + 4) + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        join_ml[row] = make_float2(m, l);
      }
      tc::named_sync(1, 256);
      if (i == 0) {
        const float2 x = join_ml[row];
        const float top = fmaxf(m, x.x), ref = top == -INFINITY ? 0.f : top;
        mul = m == -INFINITY ? 0.f : tc::ex2f(m - ref);
        mul1 = x.y == 0.f ? 0.f : tc::ex2f(x.x - ref);
        l = l * mul + (x.y == 0.f ? 0.f : x.y * mul1);
        m = top;
      }
    }
    const int tok = row_tile[i] * args.tokens + row / a.G, hq = h * a.G + row % a.G;
    const bool real = steps[i] && !(dual && i == 1) && row < args.tokens * a.G && tok < a.B * a.T;
    const int slots = a.prefix_splits + a.own_splits;
    const int64_t at = (int64_t(tok) * a.Hq + hq) * slots + split;
    if (steps[i] && !(dual && i == 1)) {
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        tc::tmem_ld32(to + c, o);
        if (dual) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 x = mul1 == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                         : *reinterpret_cast<const float4*>(join + row * (DP + 4) + c + e);
            o[e] = o[e] * mul + x.x * mul1;
            o[e + 1] = o[e + 1] * mul + x.y * mul1;
            o[e + 2] = o[e + 2] * mul + x.z * mul1;
            o[e + 3] = o[e + 3] * mul + x.w * mul1;
          }
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (real && c + e < a.Dv) st_global32(a.part_o + at * a.Dv + c + e, o + e);
      }
      if (real) a.part_ml[at] = make_float2(m, l);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (tid == 0 && s_wait.expired) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == kMmaWarp) tc::tmem_free(tmem, 512);
}

template <typename T, int DP>
int launch(const PrefixTcArgs& a, cudaStream_t s) {
  using L = PrefixTile<DP>;
  if (int rc = allow_smem<prefix_tc_kernel<T, DP>>(L::SMEM, "prefix attention smem attribute")) return rc;
  prefix_tc_kernel<T, DP><<<dim3(unsigned(a.p.prefix_splits * a.p.H), unsigned((a.tiles + 1) / 2)), kThreads, L::SMEM, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

}  // namespace

int prefix_attn_tc(const PrefixArgs& p, int dtype, cudaStream_t stream) {
  PrefixTcArgs a{};
  a.p = p;
  a.bf16 = dtype == PISA_BF16;
  a.tokens = kRows / p.G;
  const int64_t tokens = int64_t(p.B) * p.T;
  a.tiles = int((tokens + a.tokens - 1) / a.tokens);
  int64_t st = p.T == 1 ? p.q_sb : p.q_st;
  int64_t sh = p.Hq == 1 ? p.D : p.q_sh;
  if (tokens == 1) st = p.Hq * sh;
  int rc = thread_tensor_map(&a.tm_q, p.q, dtype, 1, tokens, p.Hq, p.D, 0, st, sh, uint32_t(p.G), uint32_t(a.tokens));
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_k, p.pk, dtype, 1, p.P, p.H, p.D, 0, p.pk_st, p.pk_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_v, p.pv, dtype, 1, p.P, p.H, p.Dv, 0, p.pv_st, p.pv_sh, kRows);
  if (rc) return rc;
  const bool narrow = p.D <= 64 && p.Dv <= 64;
  if (dtype == PISA_BF16) return narrow ? launch<__nv_bfloat16, 64>(a, stream) : launch<__nv_bfloat16, 128>(a, stream);
  return narrow ? launch<__half, 64>(a, stream) : launch<__half, 128>(a, stream);
}

}  // namespace pisa

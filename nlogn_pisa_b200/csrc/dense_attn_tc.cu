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
// 17 the TMA loads (a ring of value and key tiles), warp 18 finds the next
// item.  TMEM: S/P of both tiles and O of both fill 512 columns at 128 dims.
//
// One persistent CTA per SM takes items in turn, those that meet the most keys
// first; the loads and first scores of an item overlap the output of the one
// before.  (A CTA per item paid for its start, and packed sequences in their own
// order ended in a few long tiles.)
//
// The running maximum only moves when a row's new maximum passes the one in
// use by 2^8: weights up to 256 are as exact in 16-bit floating point as
// weights up to 1, and O in TMEM is rescaled a few times per row instead of
// once per key tile.  P is rounded to the input type because the second MMA
// takes its operands so; sums of weights are taken before that rounding, in
// fp32.
//
// Hidden keys of a tile weigh zero, but zero times an infinite or NaN value
// is NaN.  Only the last key tiles of an item (at most three) hide keys from
// any of its rows.  Their values pass through warp 18, which zeroes rows that
// are not finite before the products read them and lists those that some row
// of the item may see; the rows that do add them again in fp32 when they are
// stored.  That is at most 256 keys per row, whatever the length.
//
// The tensor core's fp32 accumulator truncates: over many keys of like weight
// the output falls short, by about 2e-4 of itself at 65536 keys, 0.002 at a
// million and 0.17 at 2^26.  Every 65536 keys O therefore moves from TMEM into fp32
// workspace, summed there on the FMA pipes.  Where a backward follows it does so
// every 8192 keys: delta inherits the loss, and dQ, a sum whose terms cancel,
// multiplies it (65536 keys of like weight, k and v with a mean of half their
// deviation: error of dQ 0.013 of its norm, now 0.002).
//
// Measured: one prompt of 16384, 32 query and 8 key heads of 128: 1685 us, 1305
// TFLOP/s; a training block of four sequences of 4096, 16 heads of 64: 204 us,
// 674 TFLOP/s.  A step of both tiles (128 keys) takes about 3170 cycles at 128
// dims, of which the two products need 2048: the rest is the chain of a tile's
// softmax (about 1780 cycles) that the other tile's products do not cover.  At
// 64 dims the exponentials (one per score, 16 a cycle) take as long as the
// products at 128 dims and bound the step.  Exponentials by polynomial for 1/8
// to 4/8 of the scores gained nothing here.
#include "dense_tc.cuh"

namespace pisa {

namespace {

constexpr int kSoftWarps = 16, kMmaWarp = 16, kLoadWarp = 17, kPlanWarp = 18;
constexpr int kThreads = 608;
// key tiles after which O leaves TMEM: in inference, and before a backward
constexpr int kKeepTiles = 512, kKeepTilesTrain = 64;
constexpr int kListWords = 3 * kRows / 32;   // the key tiles of an item that hide keys: three at most

struct FwdTcArgs {
  CUtensorMap tm_q, tm_k, tm_v;             // boxes of 64 dims x 128 rows of one head
  DenseAttnArgs d;
  int items;                                // slots of query tile pairs x heads
  int keep_tiles;
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

// 16 columns (8 registers of pairs) to global memory; those past `left` are not there.
template <typename T>
__device__ __forceinline__ void store16(T* p, const uint32_t (&r)[8], int left) {
  if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
  } else {
    if (left > 0) *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    if (left > 8) *reinterpret_cast<uint4*>(p + 8) = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// Adds the listed values to 16 columns (from `col`) of this thread's row: those
// of query `i`, with the row's maximum m (base 2), over the listed keys that it
// sees.  Bit b of list[w] is key first + 32 w + b.
template <typename T>
__device__ __noinline__ void add_listed(const DenseAttnArgs& a, const SeqTile& t, int hq, int i, float m, const uint32_t* list,
                                        int first, int col, float (&o)[16]) {
  const int h = hq / a.G, last = last_visible(a, t, i);
  const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + int64_t(t.q_begin + i) * a.q_st + hq * a.q_sh;
  const T* kp = static_cast<const T*>(a.k) + t.b * a.k_sb + int64_t(t.k_begin) * a.k_st + h * a.k_sh;
  const T* vp = static_cast<const T*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin) * a.v_st + h * a.v_sh;
  const float sl = a.scale * kLog2e;
  for (int w = 0; w < kListWords; ++w) {
    for (uint32_t left = list[w]; left; left &= left - 1) {
      const int j = first + 32 * w + __ffs(left) - 1;
      if (j > last) continue;
      float s = 0.f;
      for (int d = 0; d < a.D; d += 8) {
        float x[8], y[8];
        load_vec<T>(qp + d, x);
        load_vec<T>(kp + j * a.k_st + d, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
      }
      const float p = exp2f(fmaf(s, sl, -m));
#pragma unroll
      for (int c = 0; c < 16; c += 8) {
        if (col + c >= a.Dv) continue;
        float v[8];
        load_vec<T>(vp + j * a.v_st + col + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c + e] = fmaf(p, v[e], o[c + e]);
      }
    }
  }
}

// Workspace of the outputs on their way, by CTA, query tile and half of the
// columns: [W / 4][128 rows][4], then the row maxima (base 2) that they refer to.
template <int W> __device__ __forceinline__ float* kept_at(const DenseAttnArgs& a, int i, int half) {
  return a.kept + ((int64_t(blockIdx.x) * 2 + i) * 2 + half) * kRows * (W + 1);
}
template <int W> __device__ __forceinline__ float kept_factor(const float* at, int row, float m) {
  const float of = at[W * kRows + row];
  return of == m ? 1.f : exp2f(of - m);
}
__device__ __forceinline__ float4* kept_columns(float* at, int row, int c) {
  return reinterpret_cast<float4*>(at + c * kRows + row * 4);
}

// Adds W columns of O (TMEM `to`) with row maximum m to the workspace and clears them; one warp.
template <int W> __device__ __noinline__ void keep(uint32_t to, float* at, int row, bool first, float m) {
  const float f = first ? 0.f : kept_factor<W>(at, row, m);
#pragma unroll 1
  for (int c = 0; c < W; c += 16) {
    float o[16];
    const uint32_t zero[16] = {};
    tc::tmem_ld16(to + c, o);
    tmem_st16(to + c, zero);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float4* x = kept_columns(at, row, c + e);
      const float4 y = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *x;
      *x = make_float4(fmaf(y.x, f, o[e]), fmaf(y.y, f, o[e + 1]), fmaf(y.z, f, o[e + 2]), fmaf(y.w, f, o[e + 3]));
    }
  }
  at[W * kRows + row] = m;
  tmem_wait_st();
}

// One work item: the pair of query tiles of one head.  The scheduler warp hands
// items out one ahead of their use.
struct Work {
  SeqTile t;
  int hq;        // -1: no more work
  int tiles[2];  // key tiles that each query tile visits
  int seen[2];   // keys that every row of each query tile sees
  __device__ __forceinline__ int most() const { return max(tiles[0], tiles[1]); }
  // keys that every row of the query tiles that visit key tile j sees
  __device__ __forceinline__ int seen_by_all(int j) const { return tiles[0] > j ? seen[0] : seen[1]; }
  __device__ __forceinline__ bool hides(int j) const { return seen_by_all(j) < (j + 1) * kRows; }
  // the first key tile that hides keys; those from `most` on are not visited
  __device__ __forceinline__ int first_hiding() const { return seen_by_all(0) / kRows; }
};

// Does one of the 16-byte words of 16-bit elements hold an infinity or a NaN?
// Zero times such an element is NaN and stays in the sum.
template <typename T> struct Wild {
  using T2 = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
  T2 sum;
  __device__ __forceinline__ Wild() { *reinterpret_cast<uint32_t*>(&sum) = 0; }
  __device__ __forceinline__ void add(const uint4& v) {
    T2 zero;
    *reinterpret_cast<uint32_t*>(&zero) = 0;
    const T2* x = reinterpret_cast<const T2*>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __hfma2(x[e], zero, sum);
  }
  __device__ __forceinline__ bool any() const { return isnan(to_f32<T>(sum.x)) || isnan(to_f32<T>(sum.y)); }
};

// Rows [first, 128) of a value tile ([DP/64][128 rows][128 B]) that hold an
// infinity or a NaN become zeros; those before `real` are marked in list
// (128 bits).  One warp; true if a row was changed.
template <typename T, int DP>
__device__ __forceinline__ bool silence(uint32_t tile, int first, int real, uint32_t* list, int lane) {
  Wild<T> wild;
#pragma unroll 1
  for (int c = 0; c < DP / 64; ++c) {
#pragma unroll 8
    for (int r = first & ~3; r < kRows; r += 4)
      wild.add(ld_shared16(tile + c * kRows * 128 + (r + lane / 8) * 128 + lane % 8 * 16));
  }
  if (!__any_sync(kFull, wild.any())) return false;
  bool changed = false;
  for (int r = first; r < kRows; ++r) {
    const uint32_t at = tile + lane / 8 * kRows * 128 + r * 128 + lane % 8 * 16;
    Wild<T> row;
    if (lane < DP / 8) row.add(ld_shared16(at));
    if (!__any_sync(kFull, row.any())) continue;
    if (lane < DP / 8) st_shared16(at, 0, 0, 0, 0);
    if (lane == 0 && r < real) list[r / 32] |= 1u << (r % 32);
    changed = true;
  }
  return changed;
}

// KEEP: a sequence may pass args.keep_tiles key tiles (a kernel of its own: the
// code beside the steps costs short sequences 3 %).
template <typename T, int DP, bool KEEP>
__global__ void __launch_bounds__(kThreads, 1) dense_fwd_tc_kernel(const __grid_constant__ FwdTcArgs args) {
  using L = FwdTile<DP>;
  const DenseAttnArgs& a = args.d;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_addr = base, kv_addr = base + 2 * L::BYTES;
  __shared__ uint64_t w_full[2], w_empty[2], q_full[2], q_empty[2], kv_full[L::STAGES], kv_empty[L::STAGES];
  __shared__ uint64_t kv_raw[L::STAGES], checked[2];   // values that hide keys, before their check; an item's checks
  __shared__ uint64_t s_full[2], p_full[2], o_done[2], o_free[2], drained;
  __shared__ float s_other[2][2][kRows];      // the halves' maxima, at the end their sums
  __shared__ uint32_t s_list[2][kListWords];  // an item's keys with values that are not finite, from its first hiding tile on
  __shared__ int s_listed[2];
  __shared__ Work s_work[2];
  __shared__ uint32_t tmem_slot;
  __shared__ WaitFlag s_wait;
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&w_full[i], 1);
      tc::mbar_init(&w_empty[i], kSoftWarps + 2);
      tc::mbar_init(&q_full[i], 1);
      tc::mbar_init(&q_empty[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], kSoftWarps / 2);
      tc::mbar_init(&o_done[i], 1);
      tc::mbar_init(&o_free[i], kSoftWarps / 2);
      tc::mbar_init(&checked[i], 1);
    }
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_raw[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
    }
    tc::mbar_init(&drained, 1);
    s_wait.init(a.tries);
    tc::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(kFull, tmem_slot, 0);
  // TMEM columns: S/P of the two tiles, then their O
  const uint32_t tS = tmem, tO = tmem + 256;
  bool ok = true;
  // the next item (every lane of the calling warp), handed back when read
  auto take = [&](int n) {
    ok = wait_phase(&w_full[n & 1], n >> 1, &s_wait) && ok;
    Work w = s_work[n & 1];
    __syncwarp();
    if (lane == 0 && ok) tc::mbar_arrive(&w_empty[n & 1]);
    if (!__all_sync(kFull, ok)) w.hq = -1;
    return w;
  };

  if (warp == kPlanWarp) {
    const int slots = args.items / a.Hq;
    const bool ranked = a.cu_q != nullptr && a.sequences < kRanked;
    int n = 0, loads = 0;                      // items; ring positions of the items that were checked
    uint32_t uses = 0;                         // parity of the unchecked loads that each ring slot has held
    Work before;                               // the item before
    before.hq = -1;
    // the values of item n's tiles that hide keys
    auto check = [&](const Work& w, int slot) {
      if (lane < kListWords) s_list[slot][lane] = 0;
      __syncwarp();
      bool listed = false;
      const int from = w.first_hiding(), most = w.most();
      for (int j = from; j < most; ++j) {
        if (!w.hides(j)) continue;
        const int st = (loads + j + 1) % L::STAGES;
        ok = wait_phase(&kv_raw[st], int(uses >> st), &s_wait) && ok;
        uses ^= 1u << st;
        if (!__all_sync(kFull, ok)) return;
        if (silence<T, DP>(kv_addr + st * 2 * L::BYTES, max(0, w.seen_by_all(j) - j * kRows), w.t.k_len - j * kRows,
                           s_list[slot] + (j - from) * (kRows / 32), lane)) {
          listed = true;
          tc::fence_async_smem();
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&kv_full[st]);
      }
      if (most > 0) loads += most + 1;
      if (lane == 0) {
        s_listed[slot] = listed;
        tc::mbar_arrive(&checked[slot]);
      }
    };
    for (int round = 0;; ++round) {
      // items are in falling order of their work: every other round goes
      // backwards, or the first CTA would draw the longest of every round
      const int g = int(gridDim.x), c = int(blockIdx.x), r = round * g + (round & 1 ? g - 1 - c : c);
      Work w;
      w.hq = -1;
      if (r < args.items) {
        const int slot = r / a.Hq;             // heads of a tile side by side
        w.hq = r - slot * a.Hq;
        w.t = ranked ? tile_ranked(a, slot, 2 * kRows, false) : seq_tile(a, slots - 1 - slot, 2 * kRows, false);
        const int q0 = w.t.tile * 2 * kRows;
        if (q0 >= w.t.q_len) {
          if (!ranked) continue;               // a slot without rows
          w.hq = -1;                           // ranks end here
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int first = q0 + i * kRows, rows = min(kRows, w.t.q_len - first);
          w.tiles[i] = rows > 0 ? (last_visible(a, w.t, first + rows - 1) + kRows) / kRows : 0;
          w.seen[i] = last_visible(a, w.t, first) + 1;
        }
      }
      ok = wait_phase(&w_empty[n & 1], (n >> 1) + 1, &s_wait) && ok;
      if (!__all_sync(kFull, ok)) w.hq = -1;
      if (lane == 0) {
        s_work[n & 1] = w;
        tc::mbar_arrive(&w_full[n & 1]);
      }
      __syncwarp();
      // the next item is known by now: its loads follow those that wait here
      if (before.hq >= 0 && __all_sync(kFull, ok)) check(before, (n & 1) ^ 1);
      if (w.hq < 0) break;
      before = w;
      ++n;
    }
  } else if (warp == kLoadWarp) {
    int st = 0, uses[2] = {0, 0};              // ring slot; items that used each query tile
    uint32_t phase = 0, raw = 0, raws = 0;     // bit st: the last load of slot st is unchecked; parity of those
    int loads = 0;
    for (int n = 0;; ++n) {
      const Work w = take(n);
      if (w.hq < 0) break;
      if (lane == 0) {
        const int h = w.hq / a.G, most = w.most();
#pragma unroll 1
        for (int j = 0; j <= most && most > 0 && ok; ++j) {   // V_{j-1} and K_j; the queries before K_0
          if (j == 0) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
              if (!w.tiles[i]) continue;
              ok = wait_phase(&q_empty[i], uses[i] + 1, &s_wait) && ok;
              if (!ok) break;
              ++uses[i];
              tc::mbar_arrive_expect_tx(&q_full[i], L::BYTES);
              for (int c = 0; c < L::CH; ++c)
                tc::tma_load_4d(q_addr + i * L::BYTES + c * kRows * 128, &args.tm_q, c * 64, w.hq,
                                w.t.q_begin + (w.t.tile * 2 + i) * kRows, w.t.b, &q_full[i]);
            }
          }
          ok = ok && wait_phase(&kv_empty[st], int(phase) + 1, &s_wait);
          if (!ok) break;
          const uint32_t v = kv_addr + st * 2 * L::BYTES, k = v + L::BYTES;
          const bool unchecked = j > 0 && w.hides(j - 1);
          uint64_t* bar = unchecked ? &kv_raw[st] : &kv_full[st];
          raw = (raw & ~(1u << st)) | uint32_t(unchecked) << st;
          raws ^= uint32_t(unchecked) << st;
          tc::mbar_arrive_expect_tx(bar, (int(j > 0) + int(j < most)) * L::BYTES);
#pragma unroll 1
          for (int c = 0; c < L::CH; ++c) {
            if (j < most) tc::tma_load_4d(k + c * kRows * 128, &args.tm_k, c * 64, h, w.t.k_begin + j * kRows, w.t.b, bar);
            if (j > 0) tc::tma_load_4d(v + c * kRows * 128, &args.tm_v, c * 64, h, w.t.k_begin + (j - 1) * kRows, w.t.b, bar);
          }
          ++loads;
          if (++st == L::STAGES) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      ok = __all_sync(kFull, ok);
    }
    if (lane == 0) {
      // nothing may arrive after the CTA's end: every stage and query tile has
      // been handed back (after an expired wait: the copies in flight have landed)
      for (int x = max(0, loads - L::STAGES); x < loads; ++x) {
        const int y = x % L::STAGES;
        if (!ok && (raw >> y & 1)) wait_phase(&kv_raw[y], int(raws >> y & 1) + 1, &s_wait);
        else wait_phase(ok ? &kv_empty[y] : &kv_full[y], x / L::STAGES, &s_wait);
      }
      for (int i = 0; i < 2; ++i)
        if (uses[i]) wait_phase(ok ? &q_empty[i] : &q_full[i], uses[i] - 1, &s_wait);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    const uint32_t id_s = tc::idesc_f16(kRows, kRows, args.bf16), id_o = tc::idesc_f16(kRows, DP, args.bf16, 1);
    int st = 0;
    uint32_t phase = 0, p_phase = 0;                          // bit i: of query tile i
    int uses[2] = {0, 0};                                     // items that used each query tile
    auto next_stage = [&]() {
      if (leader && ok) tc::mma_commit(&kv_empty[st]);
      if (++st == L::STAGES) {
        st = 0;
        phase ^= 1;
      }
    };
    for (int n = 0;; ++n) {
      const Work w = take(n);
      if (w.hq < 0) break;
      const int most = w.most();
      if (most == 0) continue;
      ok = wait_phase(&kv_full[st], int(phase), &s_wait) && ok;   // K_0
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int own = i ? w.tiles[1] : w.tiles[0];
        if (own == 0) continue;
        ok = wait_phase(&q_full[i], i ? uses[1] : uses[0], &s_wait) && ok;
        tc::fence_after_sync();
        if (leader && ok) {
          mma_rows<DP>(tS + i * 128, q_addr + i * L::BYTES, kv_addr + (2 * st + 1) * L::BYTES, id_s);
          tc::mma_commit(&s_full[i]);
          if (own == 1) tc::mma_commit(&q_empty[i]);
        }
        __syncwarp();
      }
      next_stage();
      // the tiles' O of the item before has been read out
      for (int i = 0; i < 2; ++i) {
        if (w.tiles[i] == 0) continue;
        if (uses[i] > 0) ok = wait_phase(&o_free[i], uses[i] - 1, &s_wait) && ok;
        ++uses[i];
      }
      for (int j = 1; j <= most && __all_sync(kFull, ok); ++j) {
        const uint32_t v = kv_addr + st * 2 * L::BYTES, k = v + L::BYTES;
        ok = wait_phase(&kv_full[st], int(phase), &s_wait) && ok;      // V_{j-1} and K_j
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int own = i ? w.tiles[1] : w.tiles[0];
          if (j > own) continue;
          ok = wait_phase(&p_full[i], int(p_phase >> i), &s_wait) && ok;
          p_phase ^= 1u << i;
          tc::fence_after_sync();
          if (leader && ok) {
            mma_cols(tO + i * DP, tS + i * 128, 64, v, id_o, kRows / 16, j > 1);   // O += P V of key tile j - 1
            if (j < own) {                      // S = Q K^T of key tile j
              mma_rows<DP>(tS + i * 128, q_addr + i * L::BYTES, k, id_s);
              tc::mma_commit(&s_full[i]);
              if (j + 1 == own) tc::mma_commit(&q_empty[i]);
            } else {
              tc::mma_commit(&o_done[i]);
            }
          }
          __syncwarp();
        }
        next_stage();
      }
    }
    if (!__all_sync(kFull, ok)) {
      if (leader) tc::mma_commit(&drained);
      wait_phase(&drained, 0, &s_wait);
    }
    __syncwarp();
  } else {
    const int i = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    constexpr int W = DP / 2;                        // columns of a half
    const uint32_t ts = tS + i * 128 + half * 64 + lanes, to = tO + i * DP + half * W + lanes;
    const float sl = a.scale * kLog2e;
    int step = 0, done = 0;                          // score tiles and items of this query tile so far
    for (int n = 0;; ++n) {
      // the item stays in shared memory while it is worked on: registers are short
      ok = wait_phase(&w_full[n & 1], n >> 1, &s_wait) && ok;
      const Work& w = s_work[n & 1];
      if (w.hq < 0 || !__all_sync(kFull, ok)) break;
      int last, own, full;                           // full: key tiles that every row sees whole
      {
        const SeqTile t = w.t;
        const int q0 = (t.tile * 2 + i) * kRows;
        last = (q0 + row < t.q_len ? last_visible(a, t, q0 + row) : -1) - half * 64;
        full = (last_visible(a, t, q0) + 1) / kRows;
        own = w.tiles[i];
      }
      float m = -INFINITY, l = 0.f;                  // base-2 logits; l: of this half's keys
      for (int j = 0; j < own; ++j, ++step) {
        ok = wait_phase(&s_full[i], step, &s_wait) && ok;
        tc::fence_after_sync();
        if constexpr (KEEP) {                        // with these scores, O of the tiles before is complete
          if (j > 0 && (j & (args.keep_tiles - 1)) == 0) keep<W>(to, kept_at<W>(a, i, half), row, j == args.keep_tiles, m);
        }
        softmax_half<T, DP>(ts, to, sl, j == 0, j >= full ? last - j * kRows : kRows, 1 + i, s_other[i], half, row, m, l);
        tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&p_full[i]);
      }
      if (own > 0) {
        ok = wait_phase(&o_done[i], done++, &s_wait) && ok;
        tc::fence_after_sync();
        s_other[i][half][row] = l;
        tc::named_sync(1 + i, 256);
        l += s_other[i][half ^ 1][row];
      }
      ok = wait_phase(&checked[n & 1], n >> 1, &s_wait) && ok;
      const bool listed = s_listed[n & 1];
      const SeqTile t = w.t;
      const int hq = w.hq, qi = (t.tile * 2 + i) * kRows + row;   // query of this thread
      const int list_first = listed ? w.first_hiding() * kRows : 0;
      const bool real = qi < t.q_len;
      __syncwarp();
      if (lane == 0 && !listed) tc::mbar_arrive(&w_empty[n & 1]);   // a list is handed back after its use
      // O / l, stored by each thread for its half of the row (128 or 64
      // consecutive bytes); pass 1 stores what the rounding dropped
      const float inv = !ok ? NAN : l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (int64_t(t.b) * a.T + t.q_begin + qi) * a.Hq + hq;
#pragma unroll 1
      for (int c = 0; c < W; c += 16) {
        float o[16];
        if (own > 0) {
          tc::tmem_ld16(to + c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
        }
        if constexpr (KEEP) {
          if (own > args.keep_tiles) {
            float* at_kept = kept_at<W>(a, i, half);
            const float f = kept_factor<W>(at_kept, row, m);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 x = *kept_columns(at_kept, row, c + e);
              o[e] = fmaf(x.x, f, o[e]);
              o[e + 1] = fmaf(x.y, f, o[e + 1]);
              o[e + 2] = fmaf(x.z, f, o[e + 2]);
              o[e + 3] = fmaf(x.w, f, o[e + 3]);
            }
          }
        }
        if (listed && real && l != 0.f) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = o[e];
          add_listed<T>(a, t, hq, qi, m, s_list[n & 1], list_first, half * W + c, x);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = x[e];
        }
        __syncwarp();
        uint32_t r[8], d[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float x = l == 0.f && ok ? 0.f : o[e] * inv, y = l == 0.f && ok ? 0.f : o[e + 1] * inv;
          r[e / 2] = pack2<T>(x, y);
          d[e / 2] = pack2<T>(x - to_f32<T>(from_f32<T>(x)), y - to_f32<T>(from_f32<T>(y)));
        }
        const int col = half * W + c;
        if (real) {
          store16<T>(static_cast<T*>(a.out) + at * a.Dv + col, r, a.Dv - col);
          if (a.out_low) store16<T>(static_cast<T*>(a.out_low) + at * a.Dv + col, d, a.Dv - col);
        }
      }
      if (own > 0) {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&o_free[i]);
      }
      if (listed) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&w_empty[n & 1]);
      }
      if (a.lse && real && half == 0) a.lse[at] = !ok ? NAN : l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (tid == 0 && s_wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == kMmaWarp) tc::tmem_free(tmem, 512);
}

template <typename T, int DP, bool KEEP>
int fwd_keep(FwdTcArgs a, cudaStream_t s) {
  using L = FwdTile<DP>;
  const int64_t items = seq_slots(a.d.cu_q, a.d.B, a.d.T, a.d.sequences, 2 * kRows) * a.d.Hq;
  if (items >= (int64_t(1) << 30)) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  a.items = int(items);
  if (int rc = allow_smem<dense_fwd_tc_kernel<T, DP, KEEP>>(L::SMEM, "dense attention smem attribute")) return rc;
  dense_fwd_tc_kernel<T, DP, KEEP><<<unsigned(min64(items, sm_count())), kThreads, L::SMEM, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int fwd_t(const FwdTcArgs& a, cudaStream_t s) {
  return a.d.kept && a.d.N > a.keep_tiles * kRows ? fwd_keep<T, DP, true>(a, s) : fwd_keep<T, DP, false>(a, s);
}

}  // namespace

int64_t dense_fwd_kept_bytes(int64_t N, int64_t D, int64_t Dv) {
  if (N <= int64_t(kKeepTilesTrain) * kRows) return 0;
  return int64_t(sm_count()) * 2 * 2 * kRows * ((D <= 64 && Dv <= 64 ? 32 : 64) + 1) * int64_t(sizeof(float));
}

bool dense_attn_tc_eligible(const DenseAttnArgs& a, int dtype) {
  return dtype != PISA_F32 && a.D <= 128 && a.Dv <= 128;
}

int dense_attn_fwd_tc(const DenseAttnArgs& d, int dtype, cudaStream_t stream) {
  FwdTcArgs a{};
  a.d = d;
  a.d.tries = wait_tries((int64_t(d.N) + kRows - 1) / kRows);
  a.bf16 = dtype == PISA_BF16;
  a.keep_tiles = d.out_low ? kKeepTilesTrain : kKeepTiles;
  int rc = dense_tensor_map(&a.tm_q, d.q, dtype, d.B, d.T, d.Hq, d.D, d.q_sb, d.q_st, d.q_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_k, d.k, dtype, d.B, d.N, d.H, d.D, d.k_sb, d.k_st, d.k_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_v, d.v, dtype, d.B, d.N, d.H, d.Dv, d.v_sb, d.v_st, d.v_sh, kRows);
  if (rc) return rc;
  const bool narrow = d.D <= 64 && d.Dv <= 64;
  if (dtype == PISA_BF16) return narrow ? fwd_t<__nv_bfloat16, 64>(a, stream) : fwd_t<__nv_bfloat16, 128>(a, stream);
  return narrow ? fwd_t<__half, 64>(a, stream) : fwd_t<__half, 128>(a, stream);
}

}  // namespace pisa

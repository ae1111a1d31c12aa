// Dense attention backward on the tensor cores: 16-bit tensors, heads of at
// most 128 dims (formulas in dense_attn.cu).  Three launches:
//
// 1. Row statistics: -lse and -scale * delta (fp16: -delta) of every query (delta = dout .
//    out, with the part of out that its rounding dropped: it would add half
//    again to the rounding errors of dQ and dK), base 2, in tiles of 128
//    queries of one sequence and head.  Rows past a sequence's end and rows
//    without keys get lse = +inf, so their weights are zero below.  The same
//    launch lists the tiles in falling order of their work for the next two.
// 2. dK, dV: an item is 128 keys of a KV head, over the query tiles that see
//    them, for each of the G query heads (the statistics enter S^T and dP^T
//    as one more step of their products):
//      MMA  S^T  = K Q^T       (M = 128 keys, N = 128 queries)  -> TMEM
//      MMA  dP^T = V dO^T                                       -> TMEM
//      P^T = 2^(S^T - lse), dS^T = P^T (dP^T - delta) scale, a thread per key
//      row and 64 queries; both return to TMEM as 16-bit operands
//      MMA  dV += P^T dO,  dK += dS^T Q   (A from TMEM, B with queries along K)
// 3. dQ: an item is 128 queries of a query head, over their key tiles:
//      S = Q K^T, dP = dO V^T, dS as above, dQ += dS K.
//
// Recomputing S and dP in launch 3 costs two more products than one kernel
// that adds dQ tiles into memory, but every sum stays in TMEM: no atomics, no
// fp32 copy of dQ, and results do not vary from run to run.  P and dS are
// rounded to the input type because the MMAs take their operands so.  In fp16 dS
// leaves the scale to the stores and carries a power of two instead, one per
// sequence and KV head, that brings the largest possible dS just under the
// type's range (launch 0 finds the largest finite |dout| and |v|; |dP - delta|
// is at most twice their product times the dims).  Otherwise dS, about scale |dout|
// / keys, falls below fp16's normal range: with dout of 1e-3, 2048 keys and 64
// dims dQ and dK had an error of 0.0066 of their norm, now 0.00034 (a
// once-rounded result: 0.00027).  P, about 1 / keys, is taken times 2^15 in launch
// 2 for the same reason (262144 keys: error of dV 0.0044, now below 0.0009).
// bf16 has fp32's range and keeps the scale in dS and P as it is.
//
// Rows of the last, ragged tile of a sequence belong to other sequences: the
// products that sum over them take only the 16-row steps that hold real rows,
// and a warp zeroes the rest of the last step in shared memory first (a weight
// of zero would not silence an infinite or NaN value).
//
// The tensor core's fp32 accumulator truncates, 2e-4 of a sum over 65536 rows of
// one sign and with their number.  Items of more than 512 tiles therefore come in
// parts: the sums of a part move from TMEM into fp32 workspace and the last part
// stores them (1048576 query rows of a KV head: error of dV in fp16 0.003 of its
// norm, now 0.0003).
//
// Measured: four sequences of 4096, 16 heads of 64: statistics 28 us, dK/dV 329
// us (836 TFLOP/s), dQ 226 us (912); packed documents of 1 to 4096 tokens, 32
// query and 8 key heads of 128: 54, 305 (1267) and 300 us (967).  At 64 dims the
// tensor pipe is busy 45 % of the time and the softmax warps issue in 45 to 50 %
// of the cycles: a tile's chain of exponentials, rounding and the TMEM round
// trip bounds it.  Not kept: sixteen softmax warps (dK/dV 340 us at 64 dims, 316
// at 128); the scale left out of a bf16 dS and applied to dK (328 and 306 us);
// a share of the tiles fixed per CTA (340 at 128 dims, before the statistics
// moved into the products).
#include "dense_tc.cuh"

namespace pisa {

namespace {

constexpr int kMmaWarp = 8, kLoadWarp = 9, kTrimWarp = 10;
constexpr int kThreads = 352;
// Pairs of every eight whose exponential is a polynomial.  The softmax warps of
// a CTA do the same phase at the same time, so the special-function unit bounds
// one phase and idles in the other.  Training block, four sequences of 4096, 16
// heads of 64: dK/dV 353 us with 0, 345 with 1, 346 with 2, 340 with 3, 348 with
// 4; dQ 235, 231, 226, 232 and 238.
constexpr int kPolyKv = 3, kPolyQ = 2;

constexpr int kPart = 512;               // tiles of an item's part

// Statistics of a query tile: -lse (base 2) and -scale * delta (fp16: -delta) of its rows in
// fp32, then 16 bytes per row for the products of launch 2 (see mma_stat).
constexpr int kStat = 2 * kRows + kRows * 4, kStatBytes = kRows * 16;

struct BwdTcArgs {
  CUtensorMap tm_q, tm_k, tm_v, tm_do;   // boxes of 64 dims x 128 rows of one head
  DenseAttnArgs d;
  float* stats;                          // [Hq][q_slots][kStat]
  SeqTile* order;                        // query tiles, then key tiles, in falling order of their work
  int* counters;                         // items of launches 2 and 3 drawn past each CTA's first
  uint32_t* range;                       // fp16: bits of the largest |dout| and |v| by sequence and KV head
  int64_t q_slots, k_slots;
  int bf16;
};

template <int DP> struct BwdTile {
  static constexpr int BYTES = kRows * DP * 2;
  // ring of operand tiles (Q dO Q dO ... or K V K V ...): 64 dims leave room
  // for three pairs, which also keeps a second CTA off the SM's TMEM
  static constexpr int RING = DP == 128 ? 4 : 6;
  // with statistics and the outputs' staging
  static constexpr int DKV_SMEM = (2 + RING) * BYTES + (RING / 2 + 3) * kStatBytes + 8 * 32 * 64 + 1024;
  static constexpr int DQ_SMEM = (3 + RING) * BYTES + 1024;
};

__device__ __forceinline__ float* stat_tile(const BwdTcArgs& a, int hq, int64_t slot) {
  return a.stats + (hq * a.q_slots + slot) * kStat;
}

// Factor of the scores in base 2, never quite zero (the statistics are divided by it).
__device__ __forceinline__ float base2_scale(const DenseAttnArgs& a) {
  return fmaxf(a.scale * kLog2e, 1e-30f);
}

// This thread's place in the workspace of sums on their way: [columns / 4][128 rows][4] by CTA and side.
template <int W> __device__ __forceinline__ float* kept_at(const DenseAttnArgs& a, int side, int row) {
  return a.kept + (int64_t(blockIdx.x) * 2 + side) * kRows * W + row * 4;
}
// W columns of a part's sums (TMEM `from`): added to the workspace, and back into TMEM for the last part.  One warp.
template <int W> __device__ __noinline__ void keep_part(uint32_t from, float* at, bool first, bool last) {
#pragma unroll 1
  for (int c = 0; c < W; c += 16) {
    float o[16];
    uint32_t r[16];
    tc::tmem_ld16(from + c, o);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float4* x = reinterpret_cast<float4*>(at + (c + e) * kRows);
      const float4 y = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *x;
      const float4 sum = make_float4(y.x + o[e], y.y + o[e + 1], y.z + o[e + 2], y.w + o[e + 3]);
      if (!last) *x = sum;
      r[e] = __float_as_uint(sum.x);
      r[e + 1] = __float_as_uint(sum.y);
      r[e + 2] = __float_as_uint(sum.z);
      r[e + 3] = __float_as_uint(sum.w);
    }
    if (last) tmem_st16(from + c, r);
  }
  if (last) tmem_wait_st();
}

template <typename T> constexpr bool kHalf = std::is_same<T, __half>::value;
// P of launch 2 carries 2^kWeightShift: its largest, 2^15, is within fp16's range.
template <typename T> constexpr int kWeightShift = kHalf<T> ? 15 : 0;

// Launch 0 (fp16): a CTA per query tile (dout) or key tile (v) and KV head; 17 us
// for four sequences of 4096 tokens of 16 heads of 64 (67 MB).
// Elements that are not finite are left out: they reach their own rows anyway.
__global__ void __launch_bounds__(128) dense_range_kernel(const __grid_constant__ BwdTcArgs args) {
  const DenseAttnArgs& a = args.d;
  const bool keys = int64_t(blockIdx.x) >= args.q_slots;
  const int h = blockIdx.y;
  const SeqTile t = seq_tile(a, int(keys ? blockIdx.x - args.q_slots : blockIdx.x), kRows, keys);
  const int first = t.tile * kRows, rows = min(kRows, (keys ? t.k_len : t.q_len) - first);
  const int words = (keys ? 1 : a.G) * a.Dv / 8;       // of a row, side by side
  const int64_t stride = keys ? a.v_st : int64_t(a.Hq) * a.Dv;
  const __half* at = keys ? static_cast<const __half*>(a.v) + t.b * a.v_sb + int64_t(t.k_begin + first) * a.v_st + h * a.v_sh
                          : static_cast<const __half*>(a.dout) +
                                ((int64_t(t.b) * a.T + t.q_begin + first) * a.Hq + int64_t(h) * a.G) * a.Dv;
  uint32_t most = 0;                                   // of the low and the high halves
  for (int i = threadIdx.x; i < rows * words; i += 128) {
    const int r = i / words;
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(at + r * stride + (i - r * words) * 8));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t size = w[e] & 0x7fff7fffu;
      most = __vmaxu2(most, size & ~__vcmpgeu2(size, 0x7c007c00u));
    }
  }
  most = __reduce_max_sync(kFull, max(most & 0xffffu, most >> 16));
  if (threadIdx.x % 32 == 0 && most) atomicMax(args.range + (int64_t(t.seq) * a.H + h) * 2 + int(keys), most);
}

// The factor of dS in the type's range: 2^15 over the next power of two above its bound.
template <typename T>
__device__ __forceinline__ float grad_factor(const BwdTcArgs& args, int seq, int h) {
  if constexpr (!kHalf<T>) return args.d.scale;
  const uint32_t* at = args.range + (int64_t(seq) * args.d.H + h) * 2;
  const float bound = 2.f * float(args.d.Dv) * __half2float(__ushort_as_half(uint16_t(at[0]))) *
                      __half2float(__ushort_as_half(uint16_t(at[1])));
  return bound == 0.f ? 1.f : __uint_as_float((127u + 15u + 126u - (__float_as_uint(bound) >> 23)) << 23);
}
// What dS with that factor still lacks, at the stores of dQ and dK.
template <typename T>
__device__ __forceinline__ float grad_rest(const BwdTcArgs& args, float factor) {
  return kHalf<T> ? args.d.scale / factor : 1.f;
}

// x = three bf16 values, to 24 bits
__device__ __forceinline__ uint2 three_parts(float x) {
  const __nv_bfloat16 hi = __float2bfloat16_rn(x);
  const float rest = x - __bfloat162float(hi);
  const __nv_bfloat16 mid = __float2bfloat16_rn(rest);
  const __nv_bfloat16 lo = __float2bfloat16_rn(rest - __bfloat162float(mid));
  return make_uint2(__bfloat16_as_ushort(hi) | uint32_t(__bfloat16_as_ushort(mid)) << 16, __bfloat16_as_ushort(lo));
}

// D += the row statistic of column j in every lane: one more step of the
// product, whose A rows hold ones at the statistic's three parts and zeros
// elsewhere and whose B rows are the tile's 16 bytes (the second 16 bytes of
// both are `zeros`, the leading offset away).  The steps before had operands of
// the input type; this one's are bf16 for either, as fp16 lacks the range.
// Bound by shared-memory reads otherwise: a thread per key row needs the
// statistics of all 64 columns, 512 cycles per tile and statistic.
__device__ __forceinline__ void mma_stat(uint32_t d, uint32_t a, uint32_t b, uint32_t zeros) {
  constexpr uint32_t kPlainHigh = (128u >> 4) | (1u << 14);   // 8-row groups 128 B apart, version 1, no swizzle
  asm volatile(
      "{\n\t.reg .b64 a, b;\n\t.reg .pred p;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.eq.u32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      :: "r"(d), "r"(desc_low(a, zeros - a)), "r"(desc_low(b, zeros - b)), "r"(tc::idesc_f16(kRows, kRows, 1)), "r"(kPlainHigh)
      : "memory");
}

// Launch 1: kStatTokens queries x all heads per CTA, DP/8 lanes per row, each
// with U rows requested at a time (bound by HBM: reads dout, out and out_low).
constexpr int kStatTokens = 8;

template <typename T, int DP>
__global__ void __launch_bounds__(256) dense_stats_kernel(const __grid_constant__ BwdTcArgs args) {
  constexpr int LANES = DP / 8, PER = 256 / LANES, U = 4;   // rows of the CTA at a time
  const DenseAttnArgs& a = args.d;
  const int slot = blockIdx.x;
  if (blockIdx.y == kRows / kStatTokens) {
    // the order of the tiles in the launches that follow: eight ranks per CTA
    if (slot == 0 && threadIdx.x == 0) {
      *a.status = PISA_OK;
      args.counters[0] = args.counters[1] = 0;
    }
    const int64_t r = slot * int64_t(8) + threadIdx.x / 32, all = args.q_slots + args.k_slots;
    if (r >= all) return;
    const bool by_keys = r >= args.q_slots;
    const int rank = int(by_keys ? r - args.q_slots : r);
    const SeqTile t = a.cu_q != nullptr && a.sequences < kRanked ? tile_ranked(a, rank, kRows, by_keys)
                      : seq_tile(a, by_keys ? rank : int(args.q_slots) - 1 - rank, kRows, by_keys);
    if (threadIdx.x % 32 == 0) args.order[r] = t;
    return;
  }
  const SeqTile t = seq_tile(a, slot, kRows, false);
  const int q0 = t.tile * kRows;
  if (slot >= args.q_slots || q0 >= t.q_len) return;
  const int lane = threadIdx.x % LANES, d = lane * 8, token0 = blockIdx.y * kStatTokens;
  const T* out = static_cast<const T*>(a.o);
  const T* low = static_cast<const T*>(a.o_low);
  const T* dout = static_cast<const T*>(a.dout);
  const int64_t first = (int64_t(t.b) * a.T + t.q_begin + q0 + token0) * a.Hq;   // row of the CTA's first
  const int rows = kStatTokens * a.Hq, real = (t.q_len - q0 - token0) * a.Hq;     // consecutive in memory
  for (int x0 = threadIdx.x / LANES; x0 < rows; x0 += U * PER) {
    uint4 u[U], v[U], w[U];
    float lse[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int x = x0 + i * PER;
      u[i] = v[i] = w[i] = make_uint4(0, 0, 0, 0);
      lse[i] = -INFINITY;
      if (x < rows && x < real) {
        lse[i] = a.lse_in[first + x];
        if (d < a.Dv) {
          const int64_t at = (first + x) * a.Dv + d;
          u[i] = __ldg(reinterpret_cast<const uint4*>(dout + at));
          v[i] = __ldg(reinterpret_cast<const uint4*>(out + at));
          if (low) w[i] = __ldg(reinterpret_cast<const uint4*>(low + at));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int x = x0 + i * PER;
      const T* ue = reinterpret_cast<const T*>(&u[i]);
      const T* ve = reinterpret_cast<const T*>(&v[i]);
      const T* we = reinterpret_cast<const T*>(&w[i]);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(to_f32<T>(ue[e]), to_f32<T>(ve[e]) + to_f32<T>(we[e]), dot);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
      if (lane == 0 && x < rows) {
        const int token = x / a.Hq;
        float* tile = stat_tile(args, x - token * a.Hq, slot);
        const int row = token0 + token;
        const float nlse = -lse[i] * kLog2e, sl = base2_scale(a);
        const bool dead = lse[i] == -INFINITY;
        tile[row] = dead ? -INFINITY : nlse;
        tile[kRows + row] = kHalf<T> ? -dot : -dot * a.scale;
        const uint2 m = three_parts(dead ? -0x1p127f : (nlse + float(kWeightShift<T>)) / sl), d3 = three_parts(-dot);
        reinterpret_cast<uint4*>(tile + 2 * kRows)[row] = make_uint4(m.x, m.y, d3.x, d3.y);
      }
    }
  }
}

// One operand tile of a head: DP/64 boxes on `bar`, issued by one thread.
template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int head, int row, int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tc::tma_load_4d(dst + c * kRows * 128, map, c * 64, head, row, b, bar);
}

struct Wait {
  WaitFlag* flag;
  bool ok = true;
  __device__ __forceinline__ bool operator()(uint64_t* bar, int phase) {   // one thread
    if (ok && !wait_phase(bar, phase, flag)) ok = false;
    return ok;
  }
  // a warp with collective work: it goes on after an expired wait
  __device__ __forceinline__ void warp(uint64_t* bar, int phase) { ok = wait_phase(bar, phase, flag) && ok; }
};

// Launches 2 and 3 run one persistent CTA per SM.  Items come from a counter in
// falling order of their work: the loading thread draws the next one when it
// has issued the last load of the current one, so that the next item's loads
// and first scores overlap the outputs before them.  (A CTA per item paid 7000
// cycles for its start and end; a fixed share per CTA left packed documents
// with four heads to a group 17 % above the mean.)  Which CTA takes an item
// changes nothing in its result.  All phases and ring positions run on across
// items.
template <typename Item> struct Queue {
  uint64_t full[2], empty[2];
  Item item[2];
  __device__ __forceinline__ void init() {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 10);   // MMA, trimming and eight softmax warps
    }
  }
  __device__ __forceinline__ void put(int n, const Item& w, Wait& wait) {   // one thread
    if (!wait(&empty[n & 1], (n >> 1) + 1)) return;
    item[n & 1] = w;
    tc::mbar_arrive(&full[n & 1]);
  }
  // item n (every lane of the calling warp), handed back when read
  __device__ __forceinline__ Item take(int n, Wait& wait, int lane) {
    wait.warp(&full[n & 1], n >> 1);
    Item w = item[n & 1];
    __syncwarp();
    if (lane == 0 && wait.ok) tc::mbar_arrive(&empty[n & 1]);
    if (!__all_sync(kFull, wait.ok)) w.head = -1;
    return w;
  }
};

// Draws positions of the list until `visit` accepts one; false at its end.
template <typename F> __device__ __forceinline__ bool draw(int n, int items, int* counter, F visit) {
  for (bool first = n == 0;; first = false) {
    const int at = first ? int(blockIdx.x) : int(gridDim.x) + atomicAdd(counter, 1);
    if (at >= items) return false;
    if (visit(at)) return true;
  }
}

// The next part of item w, of which `left` tiles are left (0: w is a new item).
template <typename Item> __device__ __forceinline__ void next_part(Item& w, int& left) {
  if (left == 0) {
    left = w.head < 0 ? 0 : w.total;
    w.part_from = 0;
  } else {
    w.part_from += w.total;
  }
  w.total = min(left, kPart);
  left -= w.total;
  w.part_last = left == 0;
}

// Launch 2.  An item: key tile, KV head.
struct DkvItem {
  SeqTile t;
  int head;                           // < 0: no item
  int first_tile, end_tile;           // query tiles that see a key of the tile
  int per_head, total, tail;          // their number, with all heads of the group; real rows of the last one
  float factor;                       // of dS
  int part_from;                      // of a part: its first tile (`total` counts the part's)
  bool part_last;                     // no part follows
  template <bool PARTS> __device__ __forceinline__ int from() const { return PARTS ? part_from : 0; }
  template <bool PARTS> __device__ __forceinline__ bool last() const { return !PARTS || part_last; }
};

template <typename T> __device__ __forceinline__ DkvItem dkv_item(const BwdTcArgs& args, int n) {
  const DenseAttnArgs& a = args.d;
  DkvItem w;
  const bool found = draw(n, int(args.k_slots * a.H), args.counters, [&](int at) {
    const int slot = at / a.H, j0 = (w.t = args.order[args.q_slots + slot]).tile * kRows;
    if (j0 >= w.t.k_len) return false;   // a slot without rows
    w.head = at - slot * a.H;
    const int first = first_seeing(a, w.t, j0);
    w.first_tile = first / kRows;
    w.end_tile = (w.t.q_len + kRows - 1) / kRows;
    w.per_head = first < w.t.q_len ? w.end_tile - w.first_tile : 0;
    w.total = w.per_head * a.G;
    w.tail = w.t.q_len - (w.end_tile - 1) * kRows;
    w.factor = grad_factor<T>(args, w.t.seq, w.head);
    return true;
  });
  if (!found) w.head = -1;
  return w;
}

// PARTS: items may pass kPart tiles (kernels of their own: the others have no registers to spare).
template <typename T, int DP, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1) dense_dkv_tc_kernel(const __grid_constant__ BwdTcArgs args) {
  using L = BwdTile<DP>;
  const DenseAttnArgs& a = args.d;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t k_addr = base, v_addr = base + L::BYTES, ring = base + 2 * L::BYTES;
  // statistics, the rows that pick each of them, zeros
  const uint32_t stat_addr = ring + L::RING * L::BYTES, pick_lse = stat_addr + L::RING / 2 * kStatBytes;
  const uint32_t pick_delta = pick_lse + kStatBytes, zeros = pick_delta + kStatBytes, out_addr = zeros + kStatBytes;
  __shared__ uint64_t kv_full, kv_empty, full[L::RING], raw[L::RING], empty[L::RING];
  __shared__ uint64_t s_full, p_full, dp_full, ds_full, done, drained;
  __shared__ Queue<DkvItem> queue;
  __shared__ uint32_t tmem_slot;
  __shared__ WaitFlag s_wait;
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    tc::mbar_init(&kv_full, 1);
    tc::mbar_init(&kv_empty, 1);
    for (int i = 0; i < L::RING; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&raw[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&s_full, 1);
    tc::mbar_init(&p_full, 8);
    tc::mbar_init(&dp_full, 1);
    tc::mbar_init(&ds_full, 8);
    tc::mbar_init(&done, 1);
    tc::mbar_init(&drained, 1);
    queue.init();
    s_wait.init(a.tries);
    tc::fence_barrier_init();
  }
  if (warp < 4) {
    constexpr uint32_t kOne = 0x3F80;   // 1 in bf16
    st_shared16(pick_lse + tid * 16, kOne | kOne << 16, kOne, 0, 0);
    st_shared16(pick_delta + tid * 16, 0, 0, kOne | kOne << 16, kOne);
    st_shared16(zeros + tid * 16, 0, 0, 0, 0);
    tc::fence_async_smem();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(kFull, tmem_slot, 0);
  const uint32_t tS = tmem, tP = tmem + 128, tV = tmem + 256, tK = tmem + 256 + DP;
  Wait wait{&s_wait};
  // tile n of an item: query head h*G + n / per_head, query tile first_tile +
  // n % per_head; one ring position holds its Q (and statistics), the next its dO

  if (warp == kLoadWarp) {
    if (lane == 0) {
      int pos = 0, used = 0;          // ring position; items with queries so far
      DkvItem w;
      int left = 0, drawn = 0;        // tiles of the drawn item that no part took yet; items drawn
      for (int n = 0; wait.ok; ++n) {
        if (!PARTS || left == 0) w = dkv_item<T>(args, drawn++);
        if constexpr (PARTS) next_part(w, left);
        queue.put(n, w, wait);
        if (w.head < 0) break;
        if (w.total == 0) continue;
        if (!wait(&kv_empty, used + 1)) break;
        tc::mbar_arrive_expect_tx(&kv_full, 2 * L::BYTES);
        load_tile<DP>(k_addr, &args.tm_k, w.head, w.t.k_begin + w.t.tile * kRows, w.t.b, &kv_full);
        load_tile<DP>(v_addr, &args.tm_v, w.head, w.t.k_begin + w.t.tile * kRows, w.t.b, &kv_full);
        ++used;
        int g = w.template from<PARTS>() / w.per_head, qt = w.first_tile + w.template from<PARTS>() % w.per_head;
        for (int i = 0; i < w.total && wait.ok; ++i) {
          const bool ragged = w.tail < kRows && qt + 1 == w.end_tile;
          const int row = w.t.q_begin + qt * kRows, hq = w.head * a.G + g;
#pragma unroll
          for (int x = 0; x < 2; ++x, ++pos) {
            const int st = pos % L::RING;
            if (!wait(&empty[st], (pos / L::RING) + 1)) break;
            uint64_t* bar = ragged ? &raw[st] : &full[st];   // rows of a ragged tile pass through the trimming warp
            tc::mbar_arrive_expect_tx(bar, L::BYTES + (x == 0 ? kStatBytes : 0));
            load_tile<DP>(ring + st * L::BYTES, x == 0 ? &args.tm_q : &args.tm_do, hq, row, w.t.b, bar);
            if (x == 0)
              bulk_load(stat_addr + (st / 2) * kStatBytes, stat_tile(args, hq, query_slot(a, w.t, qt, kRows)) + 2 * kRows,
                        kStatBytes, bar);
          }
          if (++qt == w.end_tile) { qt = w.first_tile; ++g; }
        }
      }
      if (!wait.ok) {                 // the copies in flight land before the CTA ends
        if (used) wait_phase(&kv_full, used - 1, &s_wait);
        for (int x = max(0, pos - L::RING); x < pos; ++x) wait_phase(&full[x % L::RING], x / L::RING, &s_wait);
      }
    }
    __syncwarp();
  } else if (warp == kTrimWarp) {
    int start = 0;                    // the item's first ring position
    uint32_t uses = 0;                // parity of the ragged tiles that each ring slot has held
    for (int i = 0;; ++i) {
      const DkvItem w = queue.take(i, wait, lane);
      if (w.head < 0) break;
      if (w.total > 0 && w.tail < kRows) {
        for (int n = w.per_head - 1 - w.template from<PARTS>() % w.per_head; n < w.total; n += w.per_head) {
          for (int x = 0; x < 2; ++x) {
            const int st = (start + 2 * n + x) % L::RING;
            wait.warp(&raw[st], uses >> st);
            uses ^= 1u << st;
            zero_rows<DP>(ring + st * L::BYTES, w.tail, (w.tail + 15) & ~15, lane);
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0 && wait.ok) tc::mbar_arrive(&full[st]);
          }
        }
      }
      start += 2 * w.total;
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    const uint32_t id_s = tc::idesc_f16(kRows, kRows, args.bf16), id_o = tc::idesc_f16(kRows, DP, args.bf16, 1);
    int st = 0, tile = 0, used = 0;   // slot of a tile's Q (its dO is in the next one); tiles and items so far
    uint32_t phase = 0;               // the slot's phase
    for (int i = 0;; ++i) {
      const DkvItem w = queue.take(i, wait, lane);
      if (w.head < 0) break;
      const int total = w.total, per_head = w.per_head, tail = w.tail;
      // per query tile: S and dP are issued one round ahead of the products
      // that use them, each after the last use of its TMEM columns
      if (total > 0) {
        wait.warp(&kv_full, used);
        wait.warp(&full[st], int(phase));
        tc::fence_after_sync();
        if (leader) {
          mma_rows<DP>(tS, k_addr, ring + st * L::BYTES, id_s);
          mma_stat(tS, pick_lse, stat_addr + (st >> 1) * kStatBytes, zeros);
          tc::mma_commit(&s_full);
        }
        wait.warp(&full[st + 1], int(phase));
        tc::fence_after_sync();
        if (leader) {
          mma_rows<DP>(tP, v_addr, ring + (st + 1) * L::BYTES, id_s);
          mma_stat(tP, pick_delta, stat_addr + (st >> 1) * kStatBytes, zeros);
          tc::mma_commit(&dp_full);
          if (total == 1) tc::mma_commit(&kv_empty);
        }
        ++used;
      }
      int left = total > 0 ? per_head - w.template from<PARTS>() % per_head : 0;   // tiles to the head's last one
      for (int n = 0; n < total && __all_sync(kFull, wait.ok); ++n, ++tile) {
        const bool rag = tail < kRows && left == 1;
        left = left == 1 ? per_head : left - 1;
        const int steps = rag ? (tail + 15) / 16 : kRows / 16;
        const uint32_t q = ring + st * L::BYTES;
        const int next = st + 2 == L::RING ? 0 : st + 2;
        const uint32_t next_phase = next ? phase : phase ^ 1;
        wait.warp(&p_full, tile);     // and the outputs of the item before have been read
        tc::fence_after_sync();
        if (leader) {
          mma_cols(tV, tS, 64, q + L::BYTES, id_o, steps, n > 0);
          tc::mma_commit(&empty[st + 1]);
        }
        if (n + 1 < total) {
          wait.warp(&full[next], int(next_phase));
          tc::fence_after_sync();
          if (leader) {
            mma_rows<DP>(tS, k_addr, ring + next * L::BYTES, id_s);
            mma_stat(tS, pick_lse, stat_addr + (next >> 1) * kStatBytes, zeros);
            tc::mma_commit(&s_full);
          }
        }
        wait.warp(&ds_full, tile);
        tc::fence_after_sync();
        if (leader) {
          mma_cols(tK, tP, 64, q, id_o, steps, n > 0);
          tc::mma_commit(&empty[st]);
          if (n + 1 == total) tc::mma_commit(&done);
        }
        if (n + 1 < total) {
          wait.warp(&full[next + 1], int(next_phase));
          tc::fence_after_sync();
          if (leader) {
            mma_rows<DP>(tP, v_addr, ring + (next + 1) * L::BYTES, id_s);
            mma_stat(tP, pick_delta, stat_addr + (next >> 1) * kStatBytes, zeros);
            tc::mma_commit(&dp_full);
            if (n + 2 == total) tc::mma_commit(&kv_empty);
          }
        }
        st = next;
        phase = next_phase;
      }
    }
    if (leader) tc::mma_commit(&drained);
    wait_phase(&drained, 0, &s_wait);
    __syncwarp();
  } else {
    const int side = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;   // key row, queries 64*side ..
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tS + lanes + side * 64, tp = tP + lanes + side * 64;
    const float2 sl2 = make_float2(base2_scale(a), base2_scale(a));
    int tile = 0, used = 0, item = 0;
    DkvItem w = queue.take(item, wait, lane);
    while (w.head >= 0) {
      const int j0 = w.t.tile * kRows;
      const float factor = kHalf<T> ? w.factor / float(1 << kWeightShift<T>) : w.factor;
      const float2 sc2 = make_float2(factor, factor);
      const int first = first_seeing(a, w.t, j0 + row), whole = first_seeing(a, w.t, j0 + kRows - 1);
      int qt = w.first_tile + (w.total > 0 ? w.template from<PARTS>() % w.per_head : 0);
      for (int n = 0; n < w.total; ++n, ++tile) {
        wait.warp(&s_full, tile);
        tc::fence_after_sync();
        float p[64];
        uint32_t x16[32];
        tc::tmem_ld64(ts, p);
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 u = ex2_mixed(mul2(make_float2(p[c], p[c + 1]), sl2), c / 2, kPolyKv);
          p[c] = u.x;
          p[c + 1] = u.y;
        }
        const bool edge = qt * kRows < whole || (w.tail < kRows && qt + 1 == w.end_tile);
        if (edge) {
          // queries before column `low` do not see the key, those from `high` on are not the sequence's
          const int low = first - qt * kRows - side * 64, high = w.t.q_len - qt * kRows - side * 64;
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c < low || c >= high) p[c] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 2) x16[c / 2] = pack2<T>(p[c], p[c + 1]);
        tmem_st32(ts, x16);
        tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&p_full);
        wait.warp(&dp_full, tile);
        tc::fence_after_sync();
        float dp[64];
        tc::tmem_ld64(tp, dp);
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 u = mul2(mul2(make_float2(dp[c], dp[c + 1]), sc2), make_float2(p[c], p[c + 1]));
          dp[c] = u.x;
          dp[c + 1] = u.y;
        }
        if (edge) {   // without weight no gradient, whatever dP holds there
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (p[c] == 0.f) dp[c] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 2) x16[c / 2] = pack2<T>(dp[c], dp[c + 1]);
        tmem_st32(tp, x16);
        tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ds_full);
        if (++qt == w.end_tile) qt = w.first_tile;
      }
      const DkvItem next = queue.take(++item, wait, lane);
      if (w.total > 0) wait.warp(&done, used++);
      tc::fence_after_sync();
      // warps of side 0 store dV, of side 1 dK, 32 columns at a time
      const int rows = min(32, w.t.k_len - (j0 + quarter * 32)), cols = side ? a.D : a.Dv;
      const int64_t at = (int64_t(w.t.b) * a.N + w.t.k_begin + j0 + quarter * 32) * a.H + w.head;
      T* to = static_cast<T*>(side ? a.dk : a.dv) + at * cols;
      const float rest = !wait.ok ? NAN : side ? grad_rest<T>(args, w.factor) : 1.f / float(1 << kWeightShift<T>);
      if constexpr (PARTS) {
        if (w.part_from > 0 || !w.part_last)
          keep_part<DP>((side ? tK : tV) + lanes, kept_at<DP>(a, side, row), w.part_from == 0, w.part_last);
      }
#pragma unroll 1
      for (int c = 0; c < DP && w.template last<PARTS>(); c += 32) {
        store_lanes<T, 32>((side ? tK : tV) + lanes + c, w.total == 0, rest, out_addr + warp * 32 * 64, to + c,
                           int64_t(a.H) * cols, rows, cols - c, lane);
        __syncwarp();
      }
      w = next;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (tid == 0 && s_wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == kMmaWarp) tc::tmem_free(tmem, 512);
}

// Launch 3.  An item: query tile, query head.
struct DqItem {
  SeqTile t;
  int head;                           // < 0: no item
  int valid, total, tail;             // real rows; key tiles, and the real rows of the last one
  float factor;                       // of dS
  int part_from;                      // of a part: its first key tile (`total` counts the part's)
  bool part_last;                     // no part follows
  template <bool PARTS> __device__ __forceinline__ int from() const { return PARTS ? part_from : 0; }
  template <bool PARTS> __device__ __forceinline__ bool last() const { return !PARTS || part_last; }
};

template <typename T> __device__ __forceinline__ DqItem dq_item(const BwdTcArgs& args, int n) {
  const DenseAttnArgs& a = args.d;
  DqItem w;
  const bool found = draw(n, int(args.q_slots * a.Hq), args.counters + 1, [&](int at) {
    const int slot = at / a.Hq;
    w.t = args.order[slot];
    w.valid = min(kRows, w.t.q_len - w.t.tile * kRows);
    if (w.valid <= 0) return false;      // a slot without rows
    w.head = at - slot * a.Hq;
    const int keys = last_visible(a, w.t, w.t.tile * kRows + w.valid - 1) + 1;
    w.total = (keys + kRows - 1) / kRows;
    w.tail = min(kRows, w.t.k_len - (w.total - 1) * kRows);
    w.factor = grad_factor<T>(args, w.t.seq, w.head / a.G);
    return true;
  });
  if (!found) w.head = -1;
  return w;
}

template <typename T, int DP, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1) dense_dq_tc_kernel(const __grid_constant__ BwdTcArgs args) {
  using L = BwdTile<DP>;
  const DenseAttnArgs& a = args.d;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_addr = base, o_addr = base + L::BYTES, out_addr = base + 2 * L::BYTES, ring = base + 3 * L::BYTES;
  __shared__ uint64_t q_full, q_empty, full[L::RING], raw[L::RING], empty[L::RING];
  __shared__ uint64_t s_full[2], dp_full, dp_free, ds_full, done, drained;
  __shared__ Queue<DqItem> queue;
  __shared__ uint32_t tmem_slot;
  __shared__ WaitFlag s_wait;
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    tc::mbar_init(&q_full, 1);
    tc::mbar_init(&q_empty, 1);
    for (int i = 0; i < L::RING; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&raw[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&s_full[0], 1);
    tc::mbar_init(&s_full[1], 1);
    tc::mbar_init(&dp_full, 1);
    tc::mbar_init(&dp_free, 8);
    tc::mbar_init(&ds_full, 8);
    tc::mbar_init(&done, 1);
    tc::mbar_init(&drained, 1);
    queue.init();
    s_wait.init(a.tries);
    tc::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(kFull, tmem_slot, 0);
  const uint32_t tS = tmem, tP = tmem + 256, tQ = tmem + 384;   // two S, whose dS overwrites it; dP; dQ
  Wait wait{&s_wait};

  if (warp == kLoadWarp) {
    if (lane == 0) {
      int pos = 0, used = 0;                    // ring position; items with keys so far
      DqItem w;
      int left = 0, drawn = 0;                  // tiles of the drawn item that no part took yet; items drawn
      for (int n = 0; wait.ok; ++n) {
        if (!PARTS || left == 0) w = dq_item<T>(args, drawn++);
        if constexpr (PARTS) next_part(w, left);
        queue.put(n, w, wait);
        if (w.head < 0) break;
        if (w.total <= 0) continue;
        const int h = w.head / a.G;
        if (!wait(&q_empty, used + 1)) break;
        tc::mbar_arrive_expect_tx(&q_full, 2 * L::BYTES);
        load_tile<DP>(q_addr, &args.tm_q, w.head, w.t.q_begin + w.t.tile * kRows, w.t.b, &q_full);
        load_tile<DP>(o_addr, &args.tm_do, w.head, w.t.q_begin + w.t.tile * kRows, w.t.b, &q_full);
        ++used;
        for (int x = 0; x < 2 * w.total; ++x, ++pos) {   // K0 V0 K1 V1 ...
          const int st = pos % L::RING;
          if (!wait(&empty[st], (pos / L::RING) + 1)) break;
          // keys of a ragged last tile pass through the trimming warp
          uint64_t* bar = x == 2 * w.total - 2 && w.template last<PARTS>() && w.tail < kRows ? &raw[st] : &full[st];
          tc::mbar_arrive_expect_tx(bar, L::BYTES);
          load_tile<DP>(ring + st * L::BYTES, x & 1 ? &args.tm_v : &args.tm_k, h, w.t.k_begin + (w.template from<PARTS>() + (x >> 1)) * kRows, w.t.b, bar);
        }
      }
      if (!wait.ok) {   // the copies in flight land before the CTA ends
        if (used) wait_phase(&q_full, used - 1, &s_wait);
        for (int x = max(0, pos - L::RING); x < pos; ++x) wait_phase(&full[x % L::RING], x / L::RING, &s_wait);
      }
    }
    __syncwarp();
  } else if (warp == kTrimWarp) {
    int pos = 0;
    uint32_t uses = 0;                          // parity of the ragged tiles that each ring slot has held
    for (int i = 0;; ++i) {
      const DqItem w = queue.take(i, wait, lane);
      if (w.head < 0) break;
      if (w.total <= 0) continue;
      pos += 2 * w.total;
      if (w.tail >= kRows || !w.template last<PARTS>()) continue;
      const int st = (pos - 2) % L::RING;
      wait.warp(&raw[st], uses >> st);
      uses ^= 1u << st;
      zero_rows<DP>(ring + st * L::BYTES, w.tail, (w.tail + 15) & ~15, lane);
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0 && wait.ok) tc::mbar_arrive(&full[st]);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    const uint32_t id_s = tc::idesc_f16(kRows, kRows, args.bf16), id_o = tc::idesc_f16(kRows, DP, args.bf16, 1);
    int st = 0, tile = 0, used = 0;             // slot of a tile's K (its V is in the next one); tiles and items so far
    uint32_t phase = 0;
    for (int i = 0;; ++i) {
      const DqItem w = queue.take(i, wait, lane);
      if (w.head < 0) break;
      const int total = w.total, steps = w.template last<PARTS>() ? (w.tail + 15) / 16 : kRows / 16;
      if (total > 0) {
        wait.warp(&q_full, used);
        wait.warp(&full[st], int(phase));
        tc::fence_after_sync();
        if (leader) {                           // the buffers' last readers: products and warps waited for before
          mma_rows<DP>(tS + (tile & 1) * 128, q_addr, ring + st * L::BYTES, id_s);
          tc::mma_commit(&s_full[tile & 1]);
        }
        wait.warp(&full[st + 1], int(phase));
        tc::fence_after_sync();
        if (leader) {
          mma_rows<DP>(tP, o_addr, ring + (st + 1) * L::BYTES, id_s);
          tc::mma_commit(&dp_full);
          tc::mma_commit(&empty[st + 1]);
          if (total == 1) tc::mma_commit(&q_empty);
        }
        ++used;
      }
      for (int n = 0; n < total && __all_sync(kFull, wait.ok); ++n, ++tile) {
        const int next = st + 2 == L::RING ? 0 : st + 2;
        const uint32_t next_phase = next ? phase : phase ^ 1;
        if (n + 1 < total) {
          wait.warp(&full[next], int(next_phase));
          tc::fence_after_sync();
          if (leader) {                         // its buffer held dS of the tile before, whose product was issued
            mma_rows<DP>(tS + ((tile + 1) & 1) * 128, q_addr, ring + next * L::BYTES, id_s);
            tc::mma_commit(&s_full[(tile + 1) & 1]);
          }
          wait.warp(&dp_free, tile);            // dP is in registers
          wait.warp(&full[next + 1], int(next_phase));
          tc::fence_after_sync();
          if (leader) {
            mma_rows<DP>(tP, o_addr, ring + (next + 1) * L::BYTES, id_s);
            tc::mma_commit(&dp_full);
            tc::mma_commit(&empty[next + 1]);
            if (n + 2 == total) tc::mma_commit(&q_empty);
          }
        }
        wait.warp(&ds_full, tile);              // and the dQ of the item before has been read
        tc::fence_after_sync();
        if (leader) {
          mma_cols(tQ, tS + (tile & 1) * 128, 64, ring + st * L::BYTES, id_o, n + 1 == total ? steps : kRows / 16, n > 0);
          tc::mma_commit(&empty[st]);
          if (n + 1 == total) tc::mma_commit(&done);
        }
        st = next;
        phase = next_phase;
      }
    }
    if (leader) tc::mma_commit(&drained);
    wait_phase(&drained, 0, &s_wait);
    __syncwarp();
  } else {
    const int side = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;   // query row, keys 64*side ..
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const float2 sl2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
    int tile = 0, used = 0, item = 0;
    float nlse = -INFINITY, ndel = 0.f;
    auto statistics = [&](const DqItem& w) {
      nlse = -INFINITY;
      ndel = 0.f;
      if (w.head >= 0 && row < w.valid) {
        const float* st = stat_tile(args, w.head, query_slot(a, w.t, w.t.tile, kRows));
        nlse = st[row];
        ndel = kHalf<T> ? st[kRows + row] * w.factor : st[kRows + row];
      }
    };
    DqItem w = queue.take(item, wait, lane);
    statistics(w);
    while (w.head >= 0) {
      const int q0 = w.t.tile * kRows;
      const float2 nlse2 = make_float2(nlse, nlse), ndel2 = make_float2(ndel, ndel), sc2 = make_float2(w.factor, w.factor);
      const int last = row < w.valid ? last_visible(a, w.t, q0 + row) : -1;
      const int whole = (last_visible(a, w.t, q0) + 1) / kRows;   // key tiles that every row sees whole
      for (int n = 0; n < w.total; ++n, ++tile) {
        const uint32_t ts = tS + (tile & 1) * 128 + lanes + side * 64;
        wait.warp(&s_full[tile & 1], tile >> 1);
        tc::fence_after_sync();
        float p[64], dp[64];
        tc::tmem_ld64(ts, p);
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 u = ex2_mixed(tc::fma2(make_float2(p[c], p[c + 1]), sl2, nlse2), c / 2, kPolyQ);
          p[c] = u.x;
          p[c + 1] = u.y;
        }
        wait.warp(&dp_full, tile);
        tc::fence_after_sync();
        tc::tmem_ld64(tP + lanes + side * 64, dp);
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&dp_free);
        uint32_t x[32];
        const int lim = last - (w.template from<PARTS>() + n) * kRows - side * 64;
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 u = mul2(tc::fma2(make_float2(dp[c], dp[c + 1]), sc2, ndel2), make_float2(p[c], p[c + 1]));
          dp[c] = u.x;
          dp[c + 1] = u.y;
        }
        if (w.template from<PARTS>() + n >= whole) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c > lim) dp[c] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 2) x[c / 2] = pack2<T>(dp[c], dp[c + 1]);
        tmem_st32(ts, x);
        tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ds_full);
      }
      const DqItem next = queue.take(++item, wait, lane);
      statistics(next);
      if (w.total > 0) wait.warp(&done, used++);
      tc::fence_after_sync();
      // each side stores half of the columns
      const int rows = min(32, w.valid - quarter * 32);
      const int64_t at = (int64_t(w.t.b) * a.T + w.t.q_begin + q0 + quarter * 32) * a.Hq + w.head;
      if constexpr (PARTS) {
        if (w.part_from > 0 || !w.part_last)
          keep_part<DP / 2>(tQ + lanes + side * (DP / 2), kept_at<DP / 2>(a, side, row), w.part_from == 0, w.part_last);
      }
      if (w.template last<PARTS>())
        store_lanes<T, DP / 2>(tQ + lanes + side * (DP / 2), w.total <= 0, wait.ok ? grad_rest<T>(args, w.factor) : NAN,
                               out_addr + warp * 32 * DP, static_cast<T*>(a.dq) + at * a.D + side * (DP / 2),
                               int64_t(a.Hq) * a.D, rows, a.D - side * (DP / 2), lane);
      __syncwarp();
      w = next;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (tid == 0 && s_wait.expired && a.status) atomicExch(a.status, PISA_ERR_TIMEOUT);
  if (warp == kMmaWarp) tc::tmem_free(tmem, 512);
}

template <auto Kernel>
int launch(int64_t blocks, int smem, const BwdTcArgs& a, cudaStream_t s) {
  if (int rc = allow_smem<Kernel>(smem, "dense attention smem attribute")) return rc;
  Kernel<<<unsigned(blocks), kThreads, smem, s>>>(a);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int bwd_t(const BwdTcArgs& a, cudaStream_t s) {
  const DenseAttnArgs& d = a.d;
  const int64_t wide = a.q_slots > (a.q_slots + a.k_slots + 7) / 8 ? a.q_slots : (a.q_slots + a.k_slots + 7) / 8;
  dense_stats_kernel<T, DP><<<dim3(unsigned(wide), kRows / kStatTokens + 1), 256, 0, s>>>(a);
  PISA_CHECK_LAUNCH();
  const int64_t kv_ctas = min64(a.k_slots * d.H, sm_count()), q_ctas = min64(a.q_slots * d.Hq, sm_count());
  int rc = d.kept ? launch<dense_dkv_tc_kernel<T, DP, true>>(kv_ctas, BwdTile<DP>::DKV_SMEM, a, s)
                  : launch<dense_dkv_tc_kernel<T, DP, false>>(kv_ctas, BwdTile<DP>::DKV_SMEM, a, s);
  if (rc) return rc;
  return d.kept ? launch<dense_dq_tc_kernel<T, DP, true>>(q_ctas, BwdTile<DP>::DQ_SMEM, a, s)
                : launch<dense_dq_tc_kernel<T, DP, false>>(q_ctas, BwdTile<DP>::DQ_SMEM, a, s);
}

}  // namespace

namespace {
// Entries of `range`: two per sequence (and one for the rows past the last) and KV head.
int64_t range_entries(bool packed, int64_t B, int64_t H, int64_t sequences) { return 2 * H * (packed ? sequences + 1 : B); }
// Sums on their way, where an item may pass kPart tiles: its bytes, behind the rest.
int64_t kept_bytes(int64_t T, int64_t N, int64_t G, int64_t D, int64_t Dv) {
  const int64_t most = int64_t(kPart) * kRows;
  if ((T + kRows) * G <= most && N <= most) return 0;
  return int64_t(sm_count()) * 2 * kRows * (D <= 64 && Dv <= 64 ? 64 : 128) * int64_t(sizeof(float));
}
// Bytes of the statistics, the list of tiles, the counters and `range`; the sums
// on their way begin there (on 16 bytes, as the workspace does).
int64_t kept_offset(bool packed, int dtype, int64_t B, int64_t T, int64_t N, int64_t Hq, int64_t H, int64_t sequences) {
  const int64_t q = seq_slots(packed, B, T, sequences, kRows), k = seq_slots(packed, B, N, sequences, kRows);
  const int64_t words = 2 + (dtype == PISA_F16 ? range_entries(packed, B, H, sequences) : 0);
  const int64_t bytes = q * Hq * kStat * int64_t(sizeof(float)) + (q + k) * int64_t(sizeof(SeqTile)) + words * int64_t(sizeof(int));
  return (bytes + 15) / 16 * 16;
}
}  // namespace

int64_t dense_bwd_workspace(bool packed, int dtype, int64_t B, int64_t T, int64_t N, int64_t Hq, int64_t H, int64_t D,
                            int64_t Dv, int64_t sequences) {
  return kept_offset(packed, dtype, B, T, N, Hq, H, sequences) + kept_bytes(T, N, Hq / H, D, Dv);
}

int dense_attn_bwd_tc(const DenseAttnArgs& d, int dtype, cudaStream_t stream) {
  BwdTcArgs a{};
  a.d = d;
  // an item of dK/dV visits the query tiles of a whole group, one of dQ the key tiles
  const int64_t q_tiles = (int64_t(d.T) + kRows - 1) / kRows * d.G, k_tiles = (int64_t(d.N) + kRows - 1) / kRows;
  a.d.tries = wait_tries(q_tiles > k_tiles ? q_tiles : k_tiles);
  a.bf16 = dtype == PISA_BF16;
  a.stats = d.delta;
  a.q_slots = seq_slots(d.cu_q, d.B, d.T, d.sequences, kRows);
  a.k_slots = seq_slots(d.cu_q, d.B, d.N, d.sequences, kRows);
  a.order = reinterpret_cast<SeqTile*>(d.delta + a.q_slots * d.Hq * kStat);
  a.counters = reinterpret_cast<int*>(a.order + a.q_slots + a.k_slots);
  if (a.q_slots * d.Hq >= (int64_t(1) << 31) - 4096 || a.k_slots * d.H >= (int64_t(1) << 31) - 4096) return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (kept_bytes(d.T, d.N, d.G, d.D, d.Dv))
    a.d.kept = reinterpret_cast<float*>(reinterpret_cast<char*>(d.delta) +
                                        kept_offset(d.cu_q, dtype, d.B, d.T, d.N, d.Hq, d.H, d.sequences));
  if (dtype == PISA_F16) {
    a.range = reinterpret_cast<uint32_t*>(a.counters + 2);
    const cudaError_t e = cudaMemsetAsync(a.range, 0, range_entries(d.cu_q, d.B, d.H, d.sequences) * sizeof(int), stream);
    if (e != cudaSuccess) return fail_cuda(e, "range clear");
    dense_range_kernel<<<dim3(unsigned(a.q_slots + a.k_slots), unsigned(d.H)), 128, 0, stream>>>(a);
    PISA_CHECK_LAUNCH();
  }
  int rc = dense_tensor_map(&a.tm_q, d.q, dtype, d.B, d.T, d.Hq, d.D, d.q_sb, d.q_st, d.q_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_k, d.k, dtype, d.B, d.N, d.H, d.D, d.k_sb, d.k_st, d.k_sh, kRows);
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_v, d.v, dtype, d.B, d.N, d.H, d.Dv, d.v_sb, d.v_st, d.v_sh, kRows);
  const int64_t st = int64_t(d.Hq) * d.Dv;
  if (rc == PISA_OK) rc = dense_tensor_map(&a.tm_do, d.dout, dtype, d.B, d.T, d.Hq, d.Dv, d.T * st, st, d.Dv, kRows);
  if (rc) return rc;
  const bool narrow = d.D <= 64 && d.Dv <= 64;
  if (dtype == PISA_BF16) return narrow ? bwd_t<__nv_bfloat16, 64>(a, stream) : bwd_t<__nv_bfloat16, 128>(a, stream);
  return narrow ? bwd_t<__half, 64>(a, stream) : bwd_t<__half, 128>(a, stream);
}

}  // namespace pisa

// Shared declarations of the dense (full) attention kernels: the operands,
// and the mapping from a grid slot to a tile of one sequence.
#pragma once

#include <atomic>

#include "internal.h"

namespace pisa {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DenseAttnArgs {
  const void* q;
  int64_t q_sb, q_st, q_sh;
  const void* k;
  int64_t k_sb, k_st, k_sh;
  const void* v;
  int64_t v_sb, v_st, v_sh;
  // packed sequences (B = 1): cumulative lengths of the queries and of the
  // keys, `sequences` + 1 entries of cu_bytes each; null: every batch row is
  // one sequence whose first query sits at position query_offset
  const void* cu_q;
  const void* cu_k;
  int cu_bytes, sequences;
  int64_t query_offset;
  int B, T, N, Hq, H, G, D, Dv;
  float scale;
  int causal;
  void* out;        // [B, T, Hq, Dv]
  void* out_low;    // same shape: the part of the output that rounding dropped, or null
  float* lse;       // [B, T, Hq] or null
  int* status;      // device status word or null
  float* kept;      // tensor-core forms: workspace of outputs on their way, or null
  uint32_t tries;   // of a wait (tensor-core forms), from wait_tries
  // backward
  const void* o;    // the forward's output, contiguous
  const void* o_low;  // its dropped part, or null
  const void* dout; // contiguous
  const float* lse_in;
  float* delta;     // workspace: [B, T, Hq] row dot products of dout and out (FMA form), row statistics (tensor-core form)
  void* dq;
  void* dk;
  void* dv;
};

// Tries of a wait, a microsecond each: half a second, and more where a wait may
// last as long as an item of that many tiles (some wait for the whole item
// before them; a tile takes 1 to 2 us).
constexpr uint32_t kWaitTries = 1u << 19;
inline uint32_t wait_tries(int64_t tiles) { return kWaitTries + uint32_t(tiles < (1 << 27) ? 8 * tiles : 1 << 30); }

// Multiprocessors of the current device, asked once per device.
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Lets a kernel use `smem` bytes of dynamic shared memory, once per device.
template <auto Kernel>
int allow_smem(int smem, const char* where) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return PISA_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail_cuda(e, where);
  if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  return PISA_OK;
}

// Tile `tile` of one sequence.  Queries q_begin .. q_begin + q_len and keys
// k_begin .. k_begin + k_len of batch row b; query i sits at position
// shift + i, key j at position j.
struct SeqTile {
  int b, seq, tile, q_begin, q_len, k_begin, k_len;
  int64_t shift;
};

__device__ __forceinline__ int cu_at(const void* cu, int bytes, int i, int most) {
  const int64_t v = bytes == 4 ? int64_t(static_cast<const int32_t*>(cu)[i]) : static_cast<const int64_t*>(cu)[i];
  return int(v < 0 ? 0 : v > most ? most : v);
}

// First row of sequence s; s == sequences stands for the rows after the last
// sequence, which no key (or no query) meets.
__device__ __forceinline__ int seq_begin(const DenseAttnArgs& a, const void* cu, int most, int s) {
  return s == 0 ? 0 : cu_at(cu, a.cu_bytes, s, most);
}
__device__ __forceinline__ int seq_end(const DenseAttnArgs& a, const void* cu, int most, int s, int begin) {
  return s >= a.sequences ? most : max(begin, cu_at(cu, a.cu_bytes, s + 1, most));
}

// Packed sequences need no table of tiles: sequence s owns the slots from
// floor(begin_s / rows) + s, of which there are at least ceil(len_s / rows)
// before the next sequence's, so a binary search over the cumulative lengths
// finds a slot's sequence.  Entries that are not in order leave rows without
// a slot but never lead outside the tensors (every value is clamped, and the
// search keeps base(lo) <= slot).
__host__ __device__ __forceinline__ int64_t seq_slots(bool packed, int64_t batch, int64_t total, int64_t sequences,
                                                      int64_t rows) {
  return packed ? total / rows + sequences + 1 : batch * ((total + rows - 1) / rows);
}

__device__ __forceinline__ SeqTile seq_tile(const DenseAttnArgs& a, int slot, int rows, bool by_keys) {
  SeqTile t;
  const int total = by_keys ? a.N : a.T;
  if (a.cu_q == nullptr) {
    t.tile = slot / a.B;   // equal tiles of all batch rows side by side
    t.b = slot - t.tile * a.B;
    t.seq = t.b;
    t.q_begin = t.k_begin = 0;
    t.q_len = a.T;
    t.k_len = a.N;
    t.shift = a.query_offset;
    return t;
  }
  const void* cu = by_keys ? a.cu_k : a.cu_q;
  int lo = 0, hi = a.sequences;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seq_begin(a, cu, total, mid) / rows + mid <= slot) lo = mid;
    else hi = mid - 1;
  }
  t.b = 0;
  t.seq = lo;
  t.q_begin = seq_begin(a, a.cu_q, a.T, lo);
  t.k_begin = seq_begin(a, a.cu_k, a.N, lo);
  t.q_len = seq_end(a, a.cu_q, a.T, lo, t.q_begin) - t.q_begin;
  t.k_len = seq_end(a, a.cu_k, a.N, lo, t.k_begin) - t.k_begin;
  t.tile = slot - ((by_keys ? t.k_begin : t.q_begin) / rows + lo);
  if (lo >= a.sequences) {
    if (by_keys) t.q_len = 0;
    else t.k_len = 0;
  }
  t.shift = int64_t(t.k_len) - t.q_len;
  return t;
}

// Tile of rank `rank` when all sequences' query (or key) tiles are ordered by
// the tiles they meet, most first (one warp; fewer than kRanked packed
// sequences).  CTAs take ranks in turn: long tiles start early and short ones
// fill the end.  A lane knows a few sequences; how many tiles cost at least c
// is a sum of closed forms, and bisection finds the cost of the rank: some 300
// instructions and no table.  No rows (q_len or k_len 0): past every tile.
constexpr int kRanked = 128;

__device__ __forceinline__ SeqTile tile_ranked(const DenseAttnArgs& a, int rank, int rows, bool by_keys) {
  constexpr int PER = kRanked / 32;
  const int lane = threadIdx.x & 31;
  // sequence lane + 32 i: its tiles, the cost of the largest, and x with x - c tiles of cost c or more
  int tiles[PER], top[PER], x[PER];
  int most = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = lane + 32 * i;
    tiles[i] = top[i] = x[i] = 0;
    if (s > a.sequences) continue;
    const int qb = seq_begin(a, a.cu_q, a.T, s), kb = seq_begin(a, a.cu_k, a.N, s);
    const int ql = seq_end(a, a.cu_q, a.T, s, qb) - qb, kl = seq_end(a, a.cu_k, a.N, s, kb) - kb;
    tiles[i] = ((by_keys ? kl : ql) + rows - 1) / rows;
    if (s == a.sequences || ql == 0 || kl == 0) continue;      // rows that meet nothing cost nothing
    const int ahead = max(0, kl - ql) / rows, q_tiles = (ql + rows - 1) / rows;
    top[i] = by_keys ? q_tiles : a.causal ? ahead + tiles[i] : (kl + rows - 1) / rows;
    x[i] = ahead + q_tiles + 1;
    most = max(most, top[i]);
  }
  auto at_least = [&](int i, int c) {
    if (c <= 0) return tiles[i];
    return c > top[i] ? 0 : a.causal ? max(0, min(tiles[i], x[i] - c)) : tiles[i];
  };
  auto count = [&](int c) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += at_least(i, c);
    return int(__reduce_add_sync(kFull, unsigned(n)));
  };
  int lo = 0, hi = int(__reduce_max_sync(kFull, unsigned(most)));
  SeqTile t{};
  if (rank >= count(0)) return t;
  while (lo < hi) {         // the largest cost that more than `rank` tiles reach
    const int mid = (lo + hi + 1) >> 1;
    if (count(mid) > rank) lo = mid;
    else hi = mid - 1;
  }
  int left = rank - count(lo + 1), seq = 0, tile = 0;
  bool found = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {   // the tiles of that cost, in sequence order
    const int n = at_least(i, lo) - at_least(i, lo + 1);
    int up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(kFull, up, o);
      if (lane >= o) up += y;
    }
    const unsigned who = __ballot_sync(kFull, !found && left >= up - n && left < up);
    if (who) {
      const int src = __ffs(who) - 1;
      seq = src + 32 * i;
      // larger costs lie at later query tiles, and at earlier key tiles
      tile = __shfl_sync(kFull, (by_keys ? at_least(i, lo + 1) : tiles[i] - at_least(i, lo)) + left - (up - n), src);
      found = true;
    }
    left -= __shfl_sync(kFull, up, 31);
  }
  t.seq = seq;
  t.q_begin = seq_begin(a, a.cu_q, a.T, seq);
  t.k_begin = seq_begin(a, a.cu_k, a.N, seq);
  t.q_len = seq_end(a, a.cu_q, a.T, seq, t.q_begin) - t.q_begin;
  t.k_len = seq_end(a, a.cu_k, a.N, seq, t.k_begin) - t.k_begin;
  if (seq >= a.sequences) {
    if (by_keys) t.q_len = 0;
    else t.k_len = 0;
  }
  t.tile = tile;
  t.shift = int64_t(t.k_len) - t.q_len;
  return t;
}

// Slot of query tile `tile` (of `rows` queries) of t's sequence: the inverse of seq_tile.
__device__ __forceinline__ int query_slot(const DenseAttnArgs& a, const SeqTile& t, int tile, int rows) {
  return a.cu_q == nullptr ? tile * a.B + t.b : t.q_begin / rows + t.seq + tile;
}

// Keys that query i of the tile's sequence sees: 0 .. last (-1: none).
__device__ __forceinline__ int last_visible(const DenseAttnArgs& a, const SeqTile& t, int i) {
  const int64_t last = a.causal ? min64(t.shift + i, int64_t(t.k_len) - 1) : int64_t(t.k_len) - 1;
  return last < -1 ? -1 : int(last);
}

// First query of the sequence that sees key j (q_len: none).
__device__ __forceinline__ int first_seeing(const DenseAttnArgs& a, const SeqTile& t, int j) {
  if (!a.causal) return 0;
  const int64_t first = int64_t(j) - t.shift;
  return int(first < 0 ? 0 : first > t.q_len ? t.q_len : first);
}

// make_tensor_map from any host thread: the encoding wants a current context,
// which a thread whose first CUDA call this is (autograd's, a server's) does
// not have until a runtime call binds the device's.
inline int thread_tensor_map(CUtensorMap* map, const void* base, int dtype, int64_t B, int64_t T, int64_t H, int64_t D,
                             int64_t sb, int64_t st, int64_t sh, uint32_t box_h, uint32_t box_t) {
  if (make_tensor_map(map, base, dtype, B, T, H, D, sb, st, sh, box_h, box_t) == PISA_OK) return PISA_OK;
  if (cudaFree(nullptr) != cudaSuccess) return fail(PISA_ERR_CUDA, "no CUDA context");
  return make_tensor_map(map, base, dtype, B, T, H, D, sb, st, sh, box_h, box_t);
}

// make_tensor_map with a box of `rows` tokens of one head; strides of
// dimensions of one element, which may hold anything, are replaced.
inline int dense_tensor_map(CUtensorMap* map, const void* base, int dtype, int64_t B, int64_t T, int64_t H, int64_t D,
                            int64_t sb, int64_t st, int64_t sh, uint32_t rows) {
  if (H == 1) sh = D;
  if (T == 1) st = H * sh;
  return thread_tensor_map(map, base, dtype, B, T, H, D, sb, st, sh, 1, rows);
}

// 16-bit tensors of at most 128 dims: tensor-core kernels
bool dense_attn_tc_eligible(const DenseAttnArgs& a, int dtype);
int dense_attn_fwd_tc(const DenseAttnArgs& a, int dtype, cudaStream_t stream);
// workspace for outputs on their way over more than 8192 keys; 0 for fewer
int64_t dense_fwd_kept_bytes(int64_t N, int64_t D, int64_t Dv);
// a.delta: dense_bwd_workspace(...) bytes
int64_t dense_bwd_workspace(bool packed, int dtype, int64_t B, int64_t T, int64_t N, int64_t Hq, int64_t H, int64_t D,
                            int64_t Dv, int64_t sequences);
int dense_attn_bwd_tc(const DenseAttnArgs& a, int dtype, cudaStream_t stream);

int dense_attn_fwd_simt(const DenseAttnArgs& a, int dtype, cudaStream_t stream);
int dense_attn_bwd_simt(const DenseAttnArgs& a, int dtype, cudaStream_t stream);

}  // namespace pisa

// Shared-prefix decode attention for 16-bit tensors with heads of at most 128
// dims and up to 16 query rows per KV head and pass (formulas and partial
// results in prefix_attn.cu).
//
// A decode step reads every key and value once for a handful of query rows:
// it is bound by HBM, and the kernel's task is an unbroken stream of loads.
// One persistent CTA per SM walks work items (a range of keys of one KV head
// for 8 or 16 query rows).  One warp issues TMA loads of 64-key tiles, keys
// and values, into a ring that runs on across items (128 KB);
// eight warps compute, four per tile, 16 keys each, on mma.sync: the query
// rows are too few for a tensor-core tile of 128.
//   S^T = K Q^T     keys along the MMA's 16 rows, query rows along its 8 columns
//   O^T += V^T P^T  dims along the 16 rows; V^T by transposing ldmatrix
// P^T leaves the first MMA key by thread group and enters the second query row
// by thread group: an 8 x 8 transpose of the packed weights in registers.  A
// warp's running maximum moves only when a score passes it by 2^8 (weights up
// to 256 are as exact in 16-bit floating point), so the usual tile needs one
// vote instead of a maximum over the threads.  The warps join through shared
// memory at the end of an item.
//
// Items: the prefix's key ranges, then the own caches' ranges that hold keys,
// counted on the device from the lengths (no CTA draws empty ranges).  Heads of
// a range are neighbours, so their rows meet in the same DRAM pages.
//
// Hidden keys: scores are selected away, and value rows past the last key
// that every row sees are masked out of the operand registers (zero times an
// infinite or NaN value is NaN); the up to T - 1 newer keys that only later
// tokens see are added row by row.
//
// Measured: 64 sequences over caches of 1 to 2048 keys (8 heads of 128, 240 MB)
// beside a shared prefix of 8192: 57 us on the SMs that the prefix leaves, 66 us
// for the whole step; 16 sequences of 5 to 4096 keys beside 65536 shared ones: 73
// and 90 us (5.7 TB/s for both kernels together).  The caches alone stream at 4.9
// TB/s.  One sequence of 700 keys: 4.4 us and 3.9 us for the join.
#include "dense_tc.cuh"
#include "prefix_attn.cuh"

namespace pisa {

namespace {

constexpr int kTile = 64;                        // keys of a ring stage
constexpr int kComputeWarps = 8, kLoadWarp = 8, kThreads = (kComputeWarps + 1) * 32;
constexpr int kTable = 1024;                     // entries of the table of own ranges

struct StreamArgs {
  CUtensorMap tm_k, tm_v, tm_pk, tm_pv;          // boxes of 64 dims x 64 keys of one head
  PrefixArgs p;
  int prefix_items;                              // key ranges x row blocks x heads of the prefix done here
  int prefix_blocks, own_blocks;                 // row blocks of a KV head
  int per_entry;                                 // sequences of a table entry
  bool after_tiles;                              // follows the prefix's tile kernel, which it shares nothing with
};

template <int DP, int NR> struct Stream {
  static constexpr int CH = DP / 64, BR = 8 * NR;
  static constexpr int OPERAND = kTile * DP * 2, STAGE = 2 * OPERAND;
  static constexpr int JOIN = kComputeWarps * BR * ((DP + 4) * 4 + 8);   // the warps' O, m and l
  // an even number: a stage always belongs to the same four warps, which then
  // wait for every phase of its barriers (parities cannot be taken for others)
  static constexpr int STAGES = DP == 64 ? 8 : 4;
  static_assert(STAGES % 2 == 0, "stages alternate between the two groups of warps");
  static constexpr int SMEM = STAGES * STAGE + JOIN + 1024;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 8 x 8 transpose of 16-bit elements: thread (g, t) gives row g, columns 2t
// and 2t + 1, and takes rows 2t and 2t + 1 of column g.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Over the eight thread groups g.
__device__ __forceinline__ float groups_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float groups_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Key ranges of sequence b's own cache: at least one, which may be empty.
__device__ __forceinline__ int own_ranges(const PrefixArgs& a, int b) {
  return max(1, (own_length(a, b) + a.own_chunk - 1) / a.own_chunk);
}

struct Item {
  bool prefix;
  int b, h, block, split, length, begin, end;
};

// Item `i` of the list; `table` holds the own ranges before each entry's sequences.
__device__ __forceinline__ Item item_at(const StreamArgs& s, const int* table, int i) {
  const PrefixArgs& a = s.p;
  Item x;
  x.prefix = i < s.prefix_items;
  if (!x.prefix) i -= s.prefix_items;
  const int blocks = x.prefix ? s.prefix_blocks : s.own_blocks;
  x.h = i % a.H;
  i /= a.H;
  x.block = i % blocks;
  i /= blocks;
  x.b = 0;
  if (!x.prefix) {
    int lo = 0, hi = (a.B + s.per_entry - 1) / s.per_entry - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (table[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    i -= table[lo];
    x.b = lo * s.per_entry;
    for (int n; x.b + 1 < a.B && i >= (n = own_ranges(a, x.b)); ++x.b) i -= n;
  }
  x.split = i;
  x.length = x.prefix ? a.P : own_length(a, x.b);
  split_range(x.length, i, x.prefix ? a.prefix_chunk : a.own_chunk, x.begin, x.end);
  return x;
}

template <typename T, int DP, int NR>
__global__ void __launch_bounds__(kThreads, 1) prefix_stream_kernel(const __grid_constant__ StreamArgs args) {
  using L = Stream<DP, NR>;
  constexpr int MT = DP / 16, BR = L::BR;
  const PrefixArgs& a = args.p;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023) & ~1023u;
  float* so = reinterpret_cast<float*>(smem_raw + (base - tc::smem_u32(smem_raw)) + L::STAGES * L::STAGE);  // [warps][BR][DP + 4]
  float2* sml = reinterpret_cast<float2*>(so + kComputeWarps * BR * (DP + 4));                              // [warps][BR]
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES];
  __shared__ int table[kTable + 1];
  __shared__ int ctas;                         // that take items: the others find the prefix's tiles on their SM
  __shared__ WaitFlag s_wait;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cudaTriggerProgrammaticLaunchCompletion();   // the joining launch may be scheduled
  // half a second before any wait can expire
  if (!args.after_tiles && blockIdx.x + tid == 0) *a.status = PISA_OK;

  // own ranges before each table entry (an exclusive scan by one warp)
  const int entries = (a.B + args.per_entry - 1) / args.per_entry;
  if (warp == 0) {
    int sum = 0;
    int64_t keys = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const int e = e0 + lane;
      int n = 0;
      if (e < entries)
        for (int b = e * args.per_entry; b < min(a.B, (e + 1) * args.per_entry); ++b) {
          n += own_ranges(a, b);
          keys += own_length(a, b);
        }
      int up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFull, up, o);
        if (lane >= o) up += y;
      }
      if (e < entries) table[e] = sum + up - n;
      sum += __shfl_sync(kFull, up, 31);
    }
    for (int o = 16; o > 0; o >>= 1) keys += __shfl_xor_sync(kFull, keys, o);
    if (lane == 0) {
      table[entries] = sum;
      ctas = args.after_tiles ? min(int(gridDim.x), prefix_share(a, keys).own_ctas) : int(gridDim.x);
    }
  } else if (tid == 32) {
    for (int i = 0; i < L::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 4);
    }
    s_wait.init();
    tc::fence_barrier_init();
  }
  __syncthreads();
  const int items = int(blockIdx.x) < ctas ? args.prefix_items + table[entries] * args.own_blocks * a.H : 0;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      int n = 0;   // tiles issued so far
      bool ok = true;
      for (int i = blockIdx.x; i < items && ok; i += ctas) {
        const Item x = item_at(args, table, i);
        const CUtensorMap* mk = x.prefix ? &args.tm_pk : &args.tm_k;
        const CUtensorMap* mv = x.prefix ? &args.tm_pv : &args.tm_v;
        for (int j = x.begin; j < x.end; j += kTile, ++n) {
          const int st = n % L::STAGES;
          if (!wait_phase(&empty[st], (n / L::STAGES) + 1, &s_wait)) { ok = false; break; }
          tc::mbar_arrive_expect_tx(&full[st], L::STAGE);
          const uint32_t k = base + st * L::STAGE, v = k + L::OPERAND;
#pragma unroll
          for (int c = 0; c < L::CH; ++c) {
            tc::tma_load_4d(k + c * kTile * 128, mk, c * 64, x.h, j, x.b, &full[st]);
            tc::tma_load_4d(v + c * kTile * 128, mv, c * 64, x.h, j, x.b, &full[st]);
          }
        }
      }
      // after an expired wait: the copies in flight land before the CTA ends
      if (!ok)
        for (int x = max(0, n - L::STAGES); x < n; ++x) wait_phase(&full[x % L::STAGES], x / L::STAGES, &s_wait);
    }
  } else {
    const int g = lane >> 2, t = lane & 3, sub = warp & 3, side = warp >> 2;   // 16 keys of the CTA's even or odd tiles
    const float sl = a.scale * kLog2e;
    const int slots = a.prefix_splits + a.own_splits;
    bool ok = true;
    int n = 0;   // tiles of the items before
    for (int i = blockIdx.x; i < items; i += ctas) {
      const Item x = item_at(args, table, i);
      const int rows = (x.prefix ? a.B * a.T : a.T) * a.G, r0 = x.block * BR;
      const int shared = x.prefix ? x.length : x.length - a.T + 1;   // keys before this one are seen by every row
      const int seen = min(x.end, shared);
      const T* vp = x.prefix ? static_cast<const T*>(a.pv) + x.h * a.pv_sh
                             : static_cast<const T*>(a.v) + x.b * a.v_sb + x.h * a.v_sh;
      const int64_t v_st = x.prefix ? a.pv_st : a.v_st;
      // query row 8 r + g as the B operand; the rows whose scores this thread
      // holds are 8 r + 2 t and 8 r + 2 t + 1
      uint32_t q[NR][MT][2];
      int last[NR][2];
      float o[NR][MT][4], m[NR][2], l[NR][2];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = r0 + 8 * r + g, tok = row / a.G, hq = x.h * a.G + row - tok * a.G;
        const int qb = x.prefix ? tok / a.T : x.b, qt = x.prefix ? tok - qb * a.T : tok;
        const T* qp = static_cast<const T*>(a.q) + qb * a.q_sb + qt * a.q_st + hq * a.q_sh;
#pragma unroll
        for (int s = 0; s < MT; ++s) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = 16 * s + 8 * e + 2 * t;
            q[r][s][e] = row < rows && d < a.D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
          }
          o[r][s][0] = o[r][s][1] = o[r][s][2] = o[r][s][3] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int mine = r0 + 8 * r + 2 * t + e;
          last[r][e] = mine >= rows ? -1 : x.prefix ? x.length - 1 : x.length - a.T + mine / a.G;
          m[r][e] = -INFINITY;
          l[r][e] = 0.f;
        }
      }
      const int tiles = (x.end - x.begin + kTile - 1) / kTile;
      for (int u = (n ^ side) & 1; u < tiles; u += 2) {   // tiles n + u of this side's parity
        const int st = (n + u) % L::STAGES;
        ok = wait_phase(&full[st], (n + u) / L::STAGES, &s_wait) && ok;
        const uint32_t kt = base + st * L::STAGE + sub * 16 * 128, vt = kt + L::OPERAND;
        const int j = x.begin + u * kTile + sub * 16;      // first key of this warp
        if (j < x.end) {
          float s[NR][4];
#pragma unroll
          for (int r = 0; r < NR; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            const int row = lane & 15, seg = (c & 3) * 2 + (lane >> 4);
            uint32_t k[4];
            ldmatrix4(k, kt + (c >> 2) * kTile * 128 + row * 128 + ((seg ^ (row & 7)) << 4));
#pragma unroll
            for (int r = 0; r < NR; ++r) mma16816<T>(s[r], k, q[r][c][0], q[r][c][1]);
          }
          const bool partial = j + 16 > seen;              // keys past the end, or seen by some rows only
          bool grown = false;
#pragma unroll
          for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {                  // key g (e < 2) or g + 8 of row 8 r + 2 t + (e & 1)
              s[r][e] *= sl;
              const int key = j + g + 8 * (e >> 1);
              if (partial && (key > last[r][e & 1] || key >= x.end)) s[r][e] = -INFINITY;
              grown = grown || s[r][e] > m[r][e & 1] + 8.f;
            }
          }
          if (__any_sync(kFull, grown)) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float to = fmaxf(m[r][e], groups_max(fmaxf(s[r][e], s[r][2 + e])));
                const float alpha = m[r][e] == -INFINITY ? 0.f : tc::ex2f(m[r][e] - to);
                m[r][e] = to;
                l[r][e] *= alpha;
#pragma unroll
                for (int c = 0; c < MT; ++c) {
                  o[r][c][e] *= alpha;
                  o[r][c][2 + e] *= alpha;
                }
              }
            }
          }
          uint32_t p[NR][2];                               // P^T of keys 0-7 and 8-15 as B operands
#pragma unroll
          for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ref = m[r][e & 1] == -INFINITY ? 0.f : m[r][e & 1];
              s[r][e] = tc::ex2f(s[r][e] - ref);
            }
            l[r][0] += s[r][0] + s[r][2];                  // this thread's share of the rows' sums
            l[r][1] += s[r][1] + s[r][3];
            // weights of keys that only some rows see join row by row below
            p[r][0] = transpose8(!partial || j + g < seen ? pack2<T>(s[r][0], s[r][1]) : 0u);
            p[r][1] = transpose8(!partial || j + 8 + g < seen ? pack2<T>(s[r][2], s[r][3]) : 0u);
          }
          // operand registers hold keys 2 t and 2 t + 1 (and 8 more) as a pair
          const int k0 = j + 2 * t;
          const uint32_t low = (k0 < seen ? 0xffffu : 0u) | (k0 + 1 < seen ? 0xffff0000u : 0u);
          const uint32_t high = (k0 + 8 < seen ? 0xffffu : 0u) | (k0 + 9 < seen ? 0xffff0000u : 0u);
#pragma unroll
          for (int c = 0; c < MT; ++c) {                   // dims 16 c + g and 16 c + 8 + g
            const int row = (lane & 7) + (lane >> 4) * 8, seg = (c & 3) * 2 + ((lane >> 3) & 1);
            uint32_t v[4];
            ldmatrix4_trans(v, vt + (c >> 2) * kTile * 128 + row * 128 + ((seg ^ (row & 7)) << 4));
            if (partial) {
              v[0] &= low;
              v[1] &= low;
              v[2] &= high;
              v[3] &= high;
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) mma16816<T>(o[r][c], v, p[r][0], p[r][1]);
          }
          if (partial) {
            for (int key = max(j, shared); key < min(j + 16, x.end); ++key) {
              const int y = key - j, src = (y & 7) * 4 + t;
#pragma unroll
              for (int r = 0; r < NR; ++r) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float w0 = __shfl_sync(kFull, s[r][e], src), w1 = __shfl_sync(kFull, s[r][2 + e], src);
                  if (key > last[r][e]) continue;
                  const float w = y < 8 ? w0 : w1;
#pragma unroll
                  for (int c = 0; c < MT; ++c) {
                    const int d = 16 * c + g;
                    if (d < a.Dv) o[r][c][e] = fmaf(w, to_f32<T>(vp[int64_t(key) * v_st + d]), o[r][c][e]);
                    if (d + 8 < a.Dv) o[r][c][2 + e] = fmaf(w, to_f32<T>(vp[int64_t(key) * v_st + d + 8]), o[r][c][2 + e]);
                  }
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0 && ok) tc::mbar_arrive(&empty[st]);
      }
      n += tiles;
      // Join: (m, l) per row and O of the eight warps through shared memory.
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = warp * BR + 8 * r + 2 * t + e;
          const float sum = groups_sum(ok ? l[r][e] : NAN);
          if (g == 0) sml[at] = make_float2(m[r][e], sum);
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            so[at * (DP + 4) + 16 * c + g] = o[r][c][e];
            so[at * (DP + 4) + 16 * c + 8 + g] = o[r][c][2 + e];
          }
        }
      }
      tc::named_sync(1, kComputeWarps * 32);
      const int slot = x.prefix ? x.split : a.prefix_splits + x.split;
      for (int y = tid; y < BR * (DP / 4); y += kComputeWarps * 32) {
        const int d = y % (DP / 4) * 4, r = y / (DP / 4), row = r0 + r;
        if (row >= rows || d >= a.Dv) continue;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kComputeWarps; ++w) top = fmaxf(top, sml[w * BR + r].x);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kComputeWarps; ++w) {
          const float2 ml = sml[w * BR + r];
          if (ml.y == 0.f) continue;                       // no keys, or only weightless ones
          const float f = tc::ex2f(ml.x - ref);
          const float4 z = *reinterpret_cast<const float4*>(so + (w * BR + r) * (DP + 4) + d);
          sum = fmaf(f, ml.y, sum);
          acc.x = fmaf(f, z.x, acc.x);
          acc.y = fmaf(f, z.y, acc.y);
          acc.z = fmaf(f, z.z, acc.z);
          acc.w = fmaf(f, z.w, acc.w);
        }
        const int tok = row / a.G, hq = x.h * a.G + row - tok * a.G;
        const int64_t at = (int64_t(x.b) * a.T + tok) * a.Hq + hq;   // in the prefix tok counts b * T + t
        if (slots == 1) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.Dv + d) =
              make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
          if (d == 0 && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
        } else {
          *reinterpret_cast<float4*>(a.part_o + (at * slots + slot) * a.Dv + d) = acc;
          if (d == 0) a.part_ml[at * slots + slot] = make_float2(top, sum);
        }
      }
      tc::named_sync(1, kComputeWarps * 32);
    }
  }
  __syncthreads();
  if (tid == 0 && s_wait.expired) atomicExch(a.status, PISA_ERR_TIMEOUT);
  // scheduled while the prefix's tiles drain, whose partials the joining launch
  // reads too: this kernel ends after that one
  cudaGridDependencySynchronize();
}

template <typename T, int DP, int NR>
int launch(const StreamArgs& s, int sms, cudaStream_t stream) {
  using L = Stream<DP, NR>;
  const PrefixArgs& a = s.p;
  if (int rc = allow_smem<prefix_stream_kernel<T, DP, NR>>(L::SMEM, "prefix attention smem attribute")) return rc;
  const int64_t most = s.prefix_items + int64_t(a.B) * a.own_splits * s.own_blocks * a.H;
  const dim3 grid(unsigned(min64(sms, most)));
  if (s.after_tiles) return launch_after(prefix_stream_kernel<T, DP, NR>, grid, kThreads, L::SMEM, s, stream);
  prefix_stream_kernel<T, DP, NR><<<grid, kThreads, L::SMEM, stream>>>(s);
  PISA_CHECK_LAUNCH();
  return PISA_OK;
}

template <typename T, int DP>
int by_rows(StreamArgs s, bool prefix, int sms, cudaStream_t stream) {
  const PrefixArgs& a = s.p;
  const int64_t own_rows = int64_t(a.T) * a.G, prefix_rows = a.B * own_rows;
  // 8 rows per pass when no KV head has more: half the registers and join
  // buffers; 16 otherwise: half the passes over the keys
  const int br = (prefix ? prefix_rows : own_rows) <= 8 ? 8 : 16;
  s.own_blocks = int((own_rows + br - 1) / br);
  s.prefix_blocks = int((prefix_rows + br - 1) / br);
  const int64_t items = int64_t(prefix ? a.prefix_splits : 0) * s.prefix_blocks * a.H;
  if (items + int64_t(a.B) * a.own_splits * s.own_blocks * a.H >= (int64_t(1) << 31))
    return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  s.prefix_items = int(items);
  s.per_entry = (a.B + kTable - 1) / kTable;
  return br == 8 ? launch<T, DP, 1>(s, sms, stream) : launch<T, DP, 2>(s, sms, stream);
}

}  // namespace

int prefix_attn_mma(const PrefixArgs& a, int dtype, bool prefix, int sms, cudaStream_t stream) {
  StreamArgs s{};
  s.p = a;
  s.after_tiles = a.prefix_splits > 0 && !prefix;
  int rc = dense_tensor_map(&s.tm_k, a.k, dtype, a.B, a.cap, a.H, a.D, a.k_sb, a.k_st, a.k_sh, kTile);
  if (rc == PISA_OK) rc = dense_tensor_map(&s.tm_v, a.v, dtype, a.B, a.cap, a.H, a.Dv, a.v_sb, a.v_st, a.v_sh, kTile);
  if (rc == PISA_OK && prefix) rc = dense_tensor_map(&s.tm_pk, a.pk, dtype, 1, a.P, a.H, a.D, 0, a.pk_st, a.pk_sh, kTile);
  if (rc == PISA_OK && prefix) rc = dense_tensor_map(&s.tm_pv, a.pv, dtype, 1, a.P, a.H, a.Dv, 0, a.pv_st, a.pv_sh, kTile);
  if (rc) return rc;
  const bool narrow = a.D <= 64 && a.Dv <= 64;
  if (dtype == PISA_BF16)
    return narrow ? by_rows<__nv_bfloat16, 64>(s, prefix, sms, stream) : by_rows<__nv_bfloat16, 128>(s, prefix, sms, stream);
  return narrow ? by_rows<__half, 64>(s, prefix, sms, stream) : by_rows<__half, 128>(s, prefix, sms, stream);
}

}  // namespace pisa

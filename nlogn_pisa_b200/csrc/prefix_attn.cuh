// Shared declarations of the decode attention over a shared prefix and each
// sequence's own cache.
#pragma once

#include "dense_attn.cuh"

namespace pisa {

struct PrefixArgs {
  const void* q;                 // [B, T, Hq, D]
  int64_t q_sb, q_st, q_sh;
  const void* k;                 // own caches [B, cap, H, D]
  int64_t k_sb, k_st, k_sh;
  const void* v;
  int64_t v_sb, v_st, v_sh;
  const void* lengths;           // [B] valid own keys, this step's T included
  int len_bytes;
  const void* pk;                // prefix [P, H, D]
  int64_t pk_st, pk_sh;
  const void* pv;
  int64_t pv_st, pv_sh;
  int B, T, Hq, H, G, D, Dv, cap, P;
  float scale;
  void* out;                     // [B, T, Hq, Dv]
  float* lse;                    // [B, T, Hq] or null
  // partial results of every (query row, slot): prefix splits first, then own
  // splits; with one slot in all the kernels write `out` directly
  int prefix_splits, own_splits, prefix_chunk, own_chunk;
  float* part_o;                 // [rows][slots][Dv], sum_j 2^(s_j - m) v_j
  float2* part_ml;               // [rows][slots], (m, l) with base-2 logits
  int* status;                   // device status word, cleared by block 0 of the first launch
  // prefix in 128-row tiles: CTAs of one key range (0: another form, whose
  // ranges are prefix_splits), multiprocessors; the number of ranges that the
  // tiles' kernel settled on follows the status word
  int tile_ctas, sms;
};

// Key ranges that a prefix in 128-row tiles needs: the tensor core's accumulator
// truncates, and passes 1e-4 of its sum over 65536 keys of like weight.
__host__ __device__ __forceinline__ int least_ranges(int64_t keys) { return int((keys + 65535) / 65536); }

__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
  const int64_t n = a.len_bytes == 4 ? int64_t(static_cast<const int32_t*>(a.lengths)[b])
                                     : static_cast<const int64_t*>(a.lengths)[b];
  return int(n < 0 ? 0 : n > a.cap ? a.cap : n);
}

// Keys of split `i`: [begin, end), empty past the sequence's length.  A split
// has the same number of keys in every sequence (chosen for the caches'
// capacity): no CTA has more to do than another.
__device__ __forceinline__ void split_range(int keys, int i, int chunk, int& begin, int& end) {
  begin = int(min64(keys, int64_t(i) * chunk));
  end = int(min64(keys, int64_t(i) * chunk + chunk));
}

// Key ranges of a prefix in 128-row tiles, at most prefix_splits, from the own
// caches' total length.  Both kernels read at the same rate per multiprocessor,
// so the prefix takes as many of them as make both end together, and the own
// caches the rest from the start.  Times in 128-key tiles of a head; a range
// starts and stores its rows in about 5.  (64 sequences of 1 to 2048 keys over
// 8192 shared ones, 8 heads of 128: 66 us for the step, 76 with one wave of
// prefix tiles before the own caches.)
struct PrefixShare {
  int ranges, chunk, own_ctas;   // own_ctas: CTAs that read the own caches
};

__device__ __forceinline__ PrefixShare prefix_share(const PrefixArgs& a, int64_t own_keys) {
  const float own = float(own_keys) / 128.f * a.H * ((a.T * a.G + 15) / 16), prefix = float(a.P) / 128.f;
  PrefixShare best{a.prefix_splits, 0, a.sms};
  float least = prefix / a.prefix_splits + 5.f + own / a.sms;   // one after the other
  // prefix / r + 5 = own / (sms - r * tile_ctas), solved for r
  const float c = float(a.tile_ctas), b = 5.f * a.sms - c * prefix - own, root = sqrtf(b * b + 20.f * c * prefix * a.sms);
  const int at = int(b > 0.f ? (b + root) / (10.f * c) : 2.f * prefix * a.sms / (root - b));
  for (int i = 0; i < 2; ++i) {
    const int r = min(max(at + i, least_ranges(a.P)), a.prefix_splits);
    const int rest = a.sms - r * a.tile_ctas;
    if (rest < 1) break;
    const float time = fmaxf(prefix / r + 5.f, own / rest);
    if (time < least) {
      least = time;
      best.ranges = r;
      best.own_ctas = rest;
    }
  }
  best.chunk = ((a.P + best.ranges - 1) / best.ranges + 127) / 128 * 128;
  best.ranges = (a.P + best.chunk - 1) / best.chunk;
  return best;
}

// Launches a kernel that may be scheduled while the stream's previous kernel
// drains: it waits in the kernel (cudaGridDependencySynchronize), before the
// first access to what that kernel writes.
template <typename A>
int launch_after(void (*kernel)(A), dim3 grid, int threads, size_t smem, const A& args, cudaStream_t stream) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(unsigned(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args);
  count_launch();
  return e == cudaSuccess ? PISA_OK : fail_cuda(e, "prefix attention launch");
}

int prefix_attn_simt(const PrefixArgs& a, int dtype, cudaStream_t stream);
// 16-bit tensors of at most 128 dims
// (own caches, and the prefix where `prefix`)
int prefix_attn_mma(const PrefixArgs& a, int dtype, bool prefix, int sms, cudaStream_t stream);
// the prefix alone, G <= 128, tokens of q a whole stride apart
int prefix_attn_tc(const PrefixArgs& a, int dtype, cudaStream_t stream);
int prefix_combine(const PrefixArgs& a, int dtype, cudaStream_t stream);

}  // namespace pisa

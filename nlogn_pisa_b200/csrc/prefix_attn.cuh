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
};

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

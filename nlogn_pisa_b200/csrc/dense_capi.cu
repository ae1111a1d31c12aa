// C entry points of dense attention (whole prompts, and decode over a shared
// prefix): argument checks, workspace layout and the choice of kernel.
#include <algorithm>
#include <cmath>

#include "dense_attn.cuh"
#include "prefix_attn.cuh"

namespace pisa {

namespace {

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Rows of a [B, T, H, D] view start on 16 bytes; the stride of a dimension of
// one element may hold anything.
bool rows16(const void* p, int dtype, int64_t B, int64_t T, int64_t H, int64_t sb, int64_t st, int64_t sh) {
  const int64_t v = dtype == PISA_F32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (B == 1 || sb % v == 0) && (T == 1 || st % v == 0) &&
         (H == 1 || sh % v == 0);
}
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_common(int dtype, int64_t Hq, int64_t H, int64_t D, int64_t Dv, float scale) {
  if (dtype < PISA_F32 || dtype > PISA_F16) return fail(PISA_ERR_UNSUPPORTED, "the kernels support FP16, BF16 and FP32");
  if (Hq <= 0 || H <= 0 || D <= 0 || Dv <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (Hq % H) return fail(PISA_ERR_INVALID, "a whole number of query heads per KV head is required");
  if (D % 8 || Dv % 8 || D > 256 || Dv > 256)
    return fail(PISA_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 256");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(PISA_ERR_INVALID, "scale must be positive and finite");
  return PISA_OK;
}

int check_dense(const DenseAttnArgs& a, int dtype, int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t Dv,
                int64_t N, int64_t sequences) {
  if (int rc = check_common(dtype, Hq, H, D, Dv, a.scale)) return rc;
  if (B <= 0 || Tq <= 0 || N <= 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  constexpr int64_t most = (int64_t(1) << 31) - 1;
  if (Tq > most - 4096 || N > most - 4096 || B > most || Hq > 65535 || sequences > most / 2 || B * Tq * Hq > most * 4)
    return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (!a.q || !a.k || !a.v) return fail(PISA_ERR_INVALID, "q, k and v are required");
  if (!rows16(a.q, dtype, B, Tq, Hq, a.q_sb, a.q_st, a.q_sh) || !rows16(a.k, dtype, B, N, H, a.k_sb, a.k_st, a.k_sh) ||
      !rows16(a.v, dtype, B, N, H, a.v_sb, a.v_st, a.v_sh))
    return fail(PISA_ERR_UNSUPPORTED, "q, k and v rows must be 16-byte aligned");
  if (a.cu_q || a.cu_k) {
    if (!a.cu_q || !a.cu_k || sequences < 1) return fail(PISA_ERR_INVALID, "cumulative lengths of queries and keys are required");
    if (a.cu_bytes != 4 && a.cu_bytes != 8) return fail(PISA_ERR_INVALID, "cumulative lengths must be int32 or int64");
    if (B != 1) return fail(PISA_ERR_INVALID, "packed inputs require batch size one");
  } else if (a.causal && (a.query_offset < 0 || a.query_offset + Tq > N)) {
    return fail(PISA_ERR_INVALID, "queries must refer to positions within their key sequence");
  }
  return PISA_OK;
}

struct PrefixPlan {
  int64_t prefix_splits, own_splits, prefix_chunk, own_chunk, ml_off, o_off, total;
  bool tiles;   // the prefix runs in 128-row tiles
};

bool prefix_mma(int dtype, int64_t D, int64_t Dv) { return dtype != PISA_F32 && D <= 128 && Dv <= 128; }

// Ranges of keys.  FMA form: two CTAs per SM, at least 256 keys each.  16-bit
// forms: the prefix's tiles in one wave of CTAs; the streaming kernel in one
// wave at least (of 64 keys or more), and ranges of about 512 keys where that
// makes no more than eight per SM: sequences of different lengths then fill the
// CTAs evenly (64 sequences of 1 to 2048 keys, 8 KV heads of 128: 55 us with
// ranges of 256, 49 with 512, 51 with 1024 or 2048).
PrefixPlan plan_prefix(int64_t B, int64_t T, int64_t Hq, int64_t H, int64_t D, int64_t Dv, int64_t cap, int64_t P, int dtype) {
  PrefixPlan p{};
  const bool mma = prefix_mma(dtype, D, Dv);
  const int64_t sms = sm_count(), G = Hq / H, rows = B * T * Hq;
  auto ranges = [](int64_t keys, int64_t count, int64_t least, int64_t* chunk) {
    *chunk = std::max<int64_t>(1, ((keys + count - 1) / count + least - 1) / least) * least;
    return std::max<int64_t>(1, (keys + *chunk - 1) / *chunk);
  };
  if (mma) {
    auto stream = [&](int64_t keys, int64_t items, int64_t* chunk) {
      const int64_t most = std::min((keys + 511) / 512, (8 * sms + items - 1) / items);
      return ranges(keys, std::max((sms + items - 1) / items, most), 64, chunk);
    };
    p.own_splits = stream(cap, B * H * ((T * G + 15) / 16), &p.own_chunk);
    if (P == 0 && cap <= 512) p.own_splits = ranges(cap, 1, 64, &p.own_chunk);   // short caches: nothing to join
    // more than 16 query rows per KV head: tiles of 128 rows, else the stream
    p.tiles = P > 0 && B * T * G > 16 && G <= 128;
    const int64_t tokens = p.tiles ? 128 / G : 1, tiles = (B * T + tokens - 1) / tokens;
    if (p.tiles)
      p.prefix_splits = ranges(P, std::max<int64_t>(least_ranges(P), sms / (H * ((tiles + 1) / 2))), 128, &p.prefix_chunk);
    else if (P > 0) p.prefix_splits = stream(P, H * ((B * T * G + 15) / 16), &p.prefix_chunk);
  } else {
    auto count = [&](int64_t items) { return (2 * sms + items - 1) / items; };
    p.own_splits = ranges(cap, count(B * H * ((T * G + 63) / 64)), 256, &p.own_chunk);
    p.prefix_splits = P > 0 ? ranges(P, count(H * ((B * T * G + 63) / 64)), 256, &p.prefix_chunk) : 0;
  }
  const int64_t slots = p.own_splits + p.prefix_splits;
  p.ml_off = 256;
  p.o_off = p.ml_off + (slots > 1 ? round256(rows * slots * 8) : 0);
  p.total = p.o_off + (slots > 1 ? rows * slots * Dv * 4 : 0);
  return p;
}

}  // namespace

}  // namespace pisa

using namespace pisa;

extern "C" {

int64_t pisa_full_attn_fwd_workspace_bytes(int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t Dv,
                                           int64_t N, int64_t sequences, int dtype) {
  if (B <= 0 || Tq <= 0 || Hq <= 0 || H <= 0 || D <= 0 || Dv <= 0 || N <= 0 || sequences < 0 || dtype < PISA_F32 ||
      dtype > PISA_F16)
    return -1;
  return 256 + (dtype == PISA_F32 || D > 128 || Dv > 128 ? 0 : dense_fwd_kept_bytes(N, D, Dv));
}

int pisa_full_attn_fwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                       int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh,
                       const void* cu_seqlens_q, const void* cu_seqlens_k, int cu_bytes, int64_t sequences,
                       int64_t query_offset, int dtype, int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D,
                       int64_t Dv, int64_t N, float scale, int causal, void* out, void* out_low, float* lse,
                       void* workspace, int64_t workspace_bytes, pisa_stream_t stream) {
  DenseAttnArgs a{};
  a.q = q; a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k = k; a.k_sb = k_sb; a.k_st = k_st; a.k_sh = k_sh;
  a.v = v; a.v_sb = v_sb; a.v_st = v_st; a.v_sh = v_sh;
  a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k; a.cu_bytes = cu_bytes;
  a.query_offset = query_offset; a.scale = scale; a.causal = causal ? 1 : 0;
  if (int rc = check_dense(a, dtype, B, Tq, Hq, H, D, Dv, N, sequences)) return rc;
  if (!out) return fail(PISA_ERR_INVALID, "out is required");
  a.sequences = int(sequences);
  a.B = int(B); a.T = int(Tq); a.N = int(N); a.Hq = int(Hq); a.H = int(H); a.G = int(Hq / H);
  a.D = int(D); a.Dv = int(Dv);
  a.out = out; a.lse = lse;
  a.out_low = dtype == PISA_F32 ? nullptr : out_low;
  if (!on16(out) || !on16(out_low))
    return fail(PISA_ERR_UNSUPPORTED, "out and out_low must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (workspace) {
    if (workspace_bytes < 256) return fail(PISA_ERR_INVALID, "workspace too small");
    cudaError_t e = cudaMemsetAsync(workspace, 0, 256, s);
    if (e != cudaSuccess) return fail_cuda(e, "status clear");
    a.status = static_cast<int*>(workspace);
    const int64_t whole = pisa_full_attn_fwd_workspace_bytes(B, Tq, Hq, H, D, Dv, N, sequences, dtype);
    if (whole > 256 && workspace_bytes >= whole && on16(workspace)) a.kept = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  }
  return dense_attn_tc_eligible(a, dtype) ? dense_attn_fwd_tc(a, dtype, s) : dense_attn_fwd_simt(a, dtype, s);
}

int64_t pisa_full_attn_bwd_workspace_bytes(int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t Dv,
                                           int64_t N, int64_t sequences, int dtype) {
  if (B <= 0 || Tq <= 0 || Hq <= 0 || H <= 0 || D <= 0 || Dv <= 0 || N <= 0 || sequences < 0 || dtype < PISA_F32 ||
      dtype > PISA_F16)
    return -1;
  if (dtype == PISA_F32 || D > 128 || Dv > 128) return 256 + B * Tq * Hq * 4;
  return 256 + dense_bwd_workspace(sequences > 0, dtype, B, Tq, N, Hq, H, D, Dv, sequences);
}

int pisa_full_attn_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
                       int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh,
                       const void* out, const void* out_low, const void* dout, const float* lse,
                       const void* cu_seqlens_q, const void* cu_seqlens_k, int cu_bytes, int64_t sequences, int64_t query_offset, int dtype,
                       int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t Dv, int64_t N, float scale,
                       int causal, void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes,
                       pisa_stream_t stream) {
  DenseAttnArgs a{};
  a.q = q; a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k = k; a.k_sb = k_sb; a.k_st = k_st; a.k_sh = k_sh;
  a.v = v; a.v_sb = v_sb; a.v_st = v_st; a.v_sh = v_sh;
  a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k; a.cu_bytes = cu_bytes;
  a.query_offset = query_offset; a.scale = scale; a.causal = causal ? 1 : 0;
  if (int rc = check_dense(a, dtype, B, Tq, Hq, H, D, Dv, N, sequences)) return rc;
  if (!out || !dout || !lse || !dq || !dk || !dv) return fail(PISA_ERR_INVALID, "out, dout, lse and the gradients are required");
  if (!on16(out) || !on16(dout) || !on16(out_low))
    return fail(PISA_ERR_UNSUPPORTED, "out, out_low and dout must be 16-byte aligned");
  a.sequences = int(sequences);
  a.B = int(B); a.T = int(Tq); a.N = int(N); a.Hq = int(Hq); a.H = int(H); a.G = int(Hq / H);
  a.D = int(D); a.Dv = int(Dv);
  a.o = out; a.o_low = dtype == PISA_F32 ? nullptr : out_low; a.dout = dout; a.lse_in = lse; a.dq = dq; a.dk = dk; a.dv = dv;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(PISA_ERR_INVALID, "workspace must be 16-byte aligned");
  if (!workspace ||
      workspace_bytes < pisa_full_attn_bwd_workspace_bytes(B, Tq, Hq, H, D, Dv, N, cu_seqlens_q ? sequences : 0, dtype))
    return fail(PISA_ERR_INVALID, "workspace too small");
  a.status = static_cast<int*>(workspace);   // cleared by the first launch, which waits for nothing
  a.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  return dense_attn_tc_eligible(a, dtype) ? dense_attn_bwd_tc(a, dtype, s) : dense_attn_bwd_simt(a, dtype, s);
}

int64_t pisa_prefix_attn_workspace_bytes(int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t Dv,
                                         int64_t capacity, int64_t prefix, int dtype) {
  if (B <= 0 || Tq <= 0 || Hq <= 0 || H <= 0 || Hq % H || D <= 0 || Dv <= 0 || capacity <= 0 || prefix < 0 ||
      dtype < PISA_F32 || dtype > PISA_F16)
    return -1;
  return plan_prefix(B, Tq, Hq, H, D, Dv, capacity, prefix, dtype).total;
}

int pisa_prefix_attn(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                     int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* lengths,
                     int length_bytes, const void* prefix_k, int64_t pk_st, int64_t pk_sh, const void* prefix_v,
                     int64_t pv_st, int64_t pv_sh, int dtype, int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D,
                     int64_t Dv, int64_t capacity, int64_t prefix, float scale, void* out, float* lse, void* workspace,
                     int64_t workspace_bytes, pisa_stream_t stream) {
  if (int rc = check_common(dtype, Hq, H, D, Dv, scale)) return rc;
  if (B <= 0 || Tq <= 0 || capacity <= 0 || prefix < 0) return fail(PISA_ERR_INVALID, "nonempty tensors are required");
  if (!q || !k || !v || !lengths || !out) return fail(PISA_ERR_INVALID, "q, k, v, lengths and out are required");
  if (prefix > 0 && (!prefix_k || !prefix_v)) return fail(PISA_ERR_INVALID, "prefix keys and values are required");
  if (length_bytes != 4 && length_bytes != 8) return fail(PISA_ERR_INVALID, "lengths must be int32 or int64");
  constexpr int64_t most = (int64_t(1) << 31) - 4097;
  if (capacity > most || prefix > most || B > 65535 || Hq > 65535 || B * Tq * (Hq / H) > 65535 * 16 || B * Tq * Hq > most)
    return fail(PISA_ERR_UNSUPPORTED, "tensor too large");
  if (B > 1 && Tq > 1 && q_sb != Tq * q_st)
    return fail(PISA_ERR_UNSUPPORTED, "the tokens of q must be a single stride apart over batch and tokens");
  if (!rows16(q, dtype, B, Tq, Hq, q_sb, q_st, q_sh) || !rows16(k, dtype, B, capacity, H, k_sb, k_st, k_sh) ||
      !rows16(v, dtype, B, capacity, H, v_sb, v_st, v_sh) ||
      (prefix > 0 && (!rows16(prefix_k, dtype, 1, prefix, H, 0, pk_st, pk_sh) ||
                      !rows16(prefix_v, dtype, 1, prefix, H, 0, pv_st, pv_sh))))
    return fail(PISA_ERR_UNSUPPORTED, "q, k and v rows must be 16-byte aligned");
  const PrefixPlan plan = plan_prefix(B, Tq, Hq, H, D, Dv, capacity, prefix, dtype);
  if ((reinterpret_cast<uintptr_t>(workspace) & 31u) != 0) return fail(PISA_ERR_INVALID, "workspace must be 32-byte aligned");
  if (!workspace || workspace_bytes < plan.total) return fail(PISA_ERR_INVALID, "workspace too small");
  char* ws = static_cast<char*>(workspace);
  PrefixArgs a{};
  a.q = q; a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k = k; a.k_sb = k_sb; a.k_st = k_st; a.k_sh = k_sh;
  a.v = v; a.v_sb = v_sb; a.v_st = v_st; a.v_sh = v_sh;
  a.lengths = lengths; a.len_bytes = length_bytes;
  a.pk = prefix_k; a.pk_st = pk_st; a.pk_sh = pk_sh;
  a.pv = prefix_v; a.pv_st = pv_st; a.pv_sh = pv_sh;
  a.B = int(B); a.T = int(Tq); a.Hq = int(Hq); a.H = int(H); a.G = int(Hq / H); a.D = int(D); a.Dv = int(Dv);
  a.cap = int(capacity); a.P = int(prefix);
  a.scale = scale; a.out = out; a.lse = lse;
  a.prefix_splits = int(plan.prefix_splits); a.own_splits = int(plan.own_splits);
  a.prefix_chunk = int(plan.prefix_chunk); a.own_chunk = int(plan.own_chunk);
  a.status = reinterpret_cast<int*>(ws);
  a.sms = sm_count();
  if (plan.tiles) {
    const int64_t tokens = 128 / a.G, tiles = (B * Tq + tokens - 1) / tokens;
    a.tile_ctas = int(H * ((tiles + 1) / 2));
  }
  a.part_ml = reinterpret_cast<float2*>(ws + plan.ml_off);
  a.part_o = reinterpret_cast<float*>(ws + plan.o_off);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (prefix_mma(dtype, D, Dv)) {
    if (plan.tiles)
      if (int rc = prefix_attn_tc(a, dtype, s)) return rc;
    if (int rc = prefix_attn_mma(a, dtype, prefix > 0 && !plan.tiles, sm_count(), s)) return rc;
  } else if (int rc = prefix_attn_simt(a, dtype, s)) {
    return rc;
  }
  return a.prefix_splits + a.own_splits > 1 ? prefix_combine(a, dtype, s) : PISA_OK;
}

}  // extern "C"

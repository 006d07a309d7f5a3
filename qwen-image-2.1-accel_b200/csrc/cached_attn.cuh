// What the attention kernels over the INT8 prefix cache share: parameters, key
// enumeration, and the per-key numbers of the softmax.
//
//   o_i = sum_j exp(c q_i.k_j) v_j / sum_j exp(c q_i.k_j)
//
// over the request's cached tokens j < lengths[b] (k_j = ks_j kc_j, v_j = vs_j
// vc_j with INT8 codes kc, vc) and its fresh bf16 tokens, each only where
// key_valid is set. A query with no key writes zeros.
//
// No scale is left in the inner loop of either kind of kernel, and masks cost
// (almost) nothing. On the tensor cores of the larger forms the keys are f16 rows
// scaled by powers of two per tile (cached_attn_tc.cuh). In the 16-row form the codes
// themselves are the operands (every INT8 value is exact in f16) and both scales
// move into the exponent, so that a key costs one fused multiply-add per score:
//   t_ij = (c log2e ks_j) (q_i.kc_j) + log2 vs_j
//   w_ij = 2^(t_ij - M_i)               the weight of the code vc_j
//   o_i  = sum_j w_ij vc_j / sum_j w_ij / vs_j
// There a masked or missing key has (0, -inf, 0) for (c log2e ks, log2 vs, 1/vs) and
// zero rows, so its w is exactly 0 whatever its memory holds.
// M_i is a running maximum that may lag the true one by 2^7 (the weights then
// exceed 1, which f16 holds), so the accumulators are rescaled rarely.
#pragma once

#include "qia_common.cuh"

namespace qia {

constexpr int kCaD = 128;

struct CachedAttn {
  const __nv_bfloat16* q;       // [B, Sq, H, 128], strides (b, s, h)
  const __nv_bfloat16* k;       // fresh rows [B, Sk, Hkv, 128]
  const __nv_bfloat16* v;
  __nv_bfloat16* out;           // [B, Sq, H, 128]
  const int8_t* kc;             // [B, Hkv, capacity, 128]
  const int8_t* vc;
  const float* ks;              // [B, Hkv, capacity]
  const float* vs;
  const int* lengths;           // [B]
  const uint8_t* key_valid;     // [B, extent + Sk], or null
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh, mask_sb;
  int sq, sk, heads, kv_heads, share, capacity, extent;   // share = heads / kv_heads
  float scale_log2;             // c log2(e)
};

// Cached tokens of request b that the call may read.
__device__ __forceinline__ int cached_len(const CachedAttn& p, int b) {
  return max(0, min(__ldg(p.lengths + b), p.extent));
}

struct KeyScalars {
  float sk, lsv, rsv;   // c log2e ks, log2 vs, 1 / vs
};

// vs below 2^-90 is taken as 2^-90: sums of w / vs then stay in range. A zero row
// (scale 0) has zero codes, so any vs gives the same value: 2^-60, which leaves the
// running maximum to the rows that count (with 1, f16 weights of rows with scales
// below 2^-22 vanished beside it) and its own part of the sum above fp32's smallest
// number beside rows with scales up to 2^50.
__device__ __forceinline__ KeyScalars key_scalars(const CachedAttn& p, float ks, float vs, bool valid) {
  KeyScalars r;
  const float v = vs == 0.0f ? 8.673617380e-19f : fmaxf(vs, 8.077935669e-28f);
  r.sk = valid ? p.scale_log2 * ks : 0.0f;
  float lg, rc;                 // (relative errors below 2^-21)
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rc) : "f"(v));
  r.lsv = valid ? (vs == vs ? lg : vs) : -INFINITY;
  r.rsv = valid ? rc : 0.0f;
  return r;
}

// The forms by query rows per K/V head (seq_q * share): one 16-row tile
// (cached_attn.cu); up to two 128-row tiles over many keys (cached_attn_tiles.cu);
// more, or few keys (cached_attn_wide.cu, which needs a workspace).
int launch_cached_rows(const CachedAttn& p, int batch, cudaStream_t st);
int launch_cached_tiles(const CachedAttn& p, int batch, cudaStream_t st);
int launch_cached_wide(const CachedAttn& p, int batch, void* workspace, cudaStream_t st);
bool cached_use_wide(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t kv_heads, int64_t share, int64_t extent);
int64_t cached_wide_workspace(int64_t batch, int64_t seq_k, int64_t kv_heads, int64_t extent);

__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace qia

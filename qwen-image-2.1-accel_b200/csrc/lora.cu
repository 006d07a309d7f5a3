// Low-rank adapters of many requests beside a shared projection:
//   y[b, s] = base[b, s] + scale_i * B_i (A_i x[b, s]),   i = ids[b]
// with A_i [r_i, in], B_i [out, r_i] of adapter i; ids[b] < 0: y = base.
// A is stored [adapters, r_pad, in] and B [adapters, out, r_pad], bf16, rows and
// columns past the adapter's own rank ignored. fp32 accumulation throughout,
// one rounding of y to bf16.
//
// lora_tokens_kernel: few tokens per request. The weights are what is read (2
// bytes per product), each by one CTA of a cluster that serves one request: the
// cluster's warps share the rank rows of A (and, for small ranks, slices of the
// contraction), every partial sum is stored into all CTAs' shared memory, and
// after one cluster barrier each CTA computes its slice of the outputs. One
// launch, fixed summation order.
#include "cluster.cuh"

namespace qia {
namespace {

constexpr int kLoraMaxRank = 128;
constexpr int kTokWarps = 8;

struct Lora {
  const __nv_bfloat16* x;      // [B, S, in]
  const __nv_bfloat16* base;   // [B, S, out]
  __nv_bfloat16* y;            // [B, S, out]
  const __nv_bfloat16* a;      // [n, r_pad, in]
  const __nv_bfloat16* b;      // [n, out, r_pad]
  const int* ranks;            // [n]
  const float* scales;         // [n]
  const int* ids;              // [B]
  int64_t x_sb, x_ss, base_sb, base_ss, y_sb, y_ss;
  int batch, seq, in, out, adapters, r_pad;
};

// The request's adapter, or -1; an id past the table is recorded and ignored.
__device__ __forceinline__ int lora_id(const Lora& p, int b, int* err) {
  const int id = __ldg(p.ids + b);
  if (id < p.adapters) return id;
  if (threadIdx.x == 0 && err) atomicExch(err, QIA_ERR_INVALID);
  return -1;
}

template <int TS>
__global__ void __launch_bounds__(kTokWarps * 32) lora_tokens_kernel(const __grid_constant__ Lora p, int* err) {
  // partial sums of A x: [slice of the contraction][token][rank]; slices x rank <= kTokWarps * cluster (or rank)
  __shared__ float part[TS * (kLoraMaxRank > kTokWarps * 8 ? kLoraMaxRank : kTokWarps * 8)];
  cluster_arrive();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = int(cluster_size()), cta = int(cluster_rank());
  const int chunk = blockIdx.x / ctas, b = blockIdx.y;
  const int s0 = chunk * TS, live = min(TS, p.seq - s0);
  const int id = lora_id(p, b, err);
  const int rank = id < 0 ? 0 : min(max(__ldg(p.ranks + id), 0), p.r_pad);
  const __nv_bfloat16* x = p.x + b * p.x_sb + int64_t(s0) * p.x_ss;

  int slices = 1;
  while (slices < 8 && rank * slices * 2 <= kTokWarps * ctas) slices *= 2;
  const int groups = p.in / 8;
  cluster_wait();   // every CTA runs: its shared memory may be stored to
  for (int item = warp * ctas + cta; item < rank * slices; item += kTokWarps * ctas) {
    const int r = item / slices, slice = item % slices;
    const uint4* arow = reinterpret_cast<const uint4*>(p.a + (int64_t(id) * p.r_pad + r) * p.in);
    float acc[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t) acc[t] = 0.0f;
    const int per = (groups + slices - 1) / slices;
    const int end = min(groups, (slice + 1) * per);
#pragma unroll 4
    for (int i = slice * per + lane; i < end; i += 32) {
      float w[8];
      unpack8(__ldg(arow + i), w);
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        if (t < live) {
          float f[8];
          unpack8(__ldg(reinterpret_cast<const uint4*>(x + t * p.x_ss) + i), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[t] = fmaf(w[e], f[e], acc[t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TS; ++t) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
      if (lane < ctas) st_cluster_f32(cluster_map(&part[(slice * TS + t) * rank + r], lane), acc[t]);
    }
  }
  cluster_sync();
  // the slices of a rank are added in order, into slice 0
  for (int i = threadIdx.x; i < TS * rank; i += blockDim.x) {
    float sum = part[i];
    for (int k = 1; k < slices; ++k) sum += part[k * TS * rank + i];
    part[i] = sum * __ldg(p.scales + id);
  }
  __syncthreads();

  // ---- outputs: `lanes` lanes of eight ranks each per output, 32 outputs per warp and round
  int lanes = 1;
  while (lanes * 8 < rank) lanes *= 2;
  const int per_round = 32 / lanes, group = lane / lanes, sub = lane % lanes;
  const int blocks = (p.out + 31) / 32;
  for (int ob = cta * kTokWarps + warp; ob < blocks; ob += ctas * kTokWarps) {
    float mine[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t) mine[t] = 0.0f;
    if (rank) {
      for (int j = 0; j < lanes; ++j) {
        const int o = ob * 32 + j * per_round + group;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 0.0f;
        if (o < p.out && sub * 8 < rank)
          unpack8(__ldg(reinterpret_cast<const uint4*>(p.b + (int64_t(id) * p.out + o) * p.r_pad) + sub), w);
#pragma unroll
        for (int t = 0; t < TS; ++t) {
          float v = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (sub * 8 + e < rank) v = fmaf(w[e], part[t * rank + sub * 8 + e], v);
          for (int k = 1; k < lanes; k *= 2) v += __shfl_xor_sync(0xffffffffu, v, k);
          v = __shfl_sync(0xffffffffu, v, (lane % per_round) * lanes);
          if (lane / per_round == j) mine[t] = v;
        }
      }
    }
    const int o = ob * 32 + lane;
    if (o < p.out) {
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        if (t < live) {
          const float v = bf16_to_f32(p.base[b * p.base_sb + int64_t(s0 + t) * p.base_ss + o]) + mine[t];
          p.y[b * p.y_sb + int64_t(s0 + t) * p.y_ss + o] = f32_to_bf16(v);
        }
      }
    }
  }
}

int launch_tokens(const Lora& p, cudaStream_t st) {
  const bool one = p.seq == 1;
  const int64_t chunks = one ? 1 : (int64_t(p.seq) + 7) / 8;
  // four CTAs of 256 threads per SM at most; a cluster has work for at most out / 256 of them
  int ctas = 1;
  while (ctas < 8 && chunks * p.batch * ctas < 4 * sm_count() && ctas * kTokWarps * 32 < p.out) ctas *= 2;
  const dim3 grid(unsigned(chunks * ctas), unsigned(p.batch));
  if (one) return launch_cluster("qia_lora_add", lora_tokens_kernel<1>, grid, kTokWarps * 32, 0, ctas, st, p,
                                 device_error_word());
  return launch_cluster("qia_lora_add", lora_tokens_kernel<8>, grid, kTokWarps * 32, 0, ctas, st, p,
                        device_error_word());
}

}  // namespace
}  // namespace qia

using namespace qia;

extern "C" int64_t qia_lora_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int qia_lora_add(const void* x, const void* base, void* y, const void* a, const void* b, const void* ranks,
                            const void* scales, const void* ids, int64_t batch, int64_t seq, int64_t in_features,
                            int64_t out_features, int64_t adapters, int64_t r_pad, const int64_t* strides,
                            void* workspace, void* stream) {
  const char* who = "qia_lora_add";
  if (!x || !base || !y || !a || !b || !ranks || !scales || !ids || !strides)
    return set_error(QIA_ERR_INVALID, "%s: null pointer", who);
  if (batch <= 0 || seq < 0 || in_features <= 0 || out_features <= 0 || adapters <= 0 || r_pad <= 0)
    return set_error(QIA_ERR_INVALID, "%s: batch=%lld seq=%lld in=%lld out=%lld adapters=%lld r_pad=%lld", who,
                     (long long)batch, (long long)seq, (long long)in_features, (long long)out_features,
                     (long long)adapters, (long long)r_pad);
  if (in_features % 8 || out_features % 8 || r_pad % 8 || r_pad > kLoraMaxRank || in_features > (1 << 20) ||
      out_features > (1 << 20) || batch > 65535 || seq > (1 << 20) || adapters > 65535)
    return set_error(QIA_ERR_UNSUPPORTED,
                     "%s: batch=%lld seq=%lld in=%lld out=%lld (multiples of 8) r_pad=%lld (a multiple of 8 to 128)", who,
                     (long long)batch, (long long)seq, (long long)in_features, (long long)out_features,
                     (long long)r_pad);
  if (!aligned(x, 16) || !aligned(base, 16) || !aligned(y, 16) || !aligned(a, 16) || !aligned(b, 16) ||
      !aligned(ranks, 4) || !aligned(scales, 4) || !aligned(ids, 4))
    return set_error(QIA_ERR_ALIGNMENT, "%s: misaligned pointer", who);
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8)
      return set_error(QIA_ERR_ALIGNMENT, "%s: stride %lld is not a multiple of 8", who, (long long)strides[i]);
  (void)workspace;
  if (seq == 0) return QIA_OK;
  Lora p;
  p.x = (const __nv_bfloat16*)x;
  p.base = (const __nv_bfloat16*)base;
  p.y = (__nv_bfloat16*)y;
  p.a = (const __nv_bfloat16*)a;
  p.b = (const __nv_bfloat16*)b;
  p.ranks = (const int*)ranks;
  p.scales = (const float*)scales;
  p.ids = (const int*)ids;
  int64_t* dst[6] = {&p.x_sb, &p.x_ss, &p.base_sb, &p.base_ss, &p.y_sb, &p.y_ss};
  for (int i = 0; i < 6; ++i) *dst[i] = strides[i];
  p.batch = int(batch);
  p.seq = int(seq);
  p.in = int(in_features);
  p.out = int(out_features);
  p.adapters = int(adapters);
  p.r_pad = int(r_pad);
  return launch_tokens(p, as_stream(stream));
}

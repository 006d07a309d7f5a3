// Low-rank adapters of many requests beside a shared projection:
//   y[b, s] = base[b, s] + scale_i * B_i (A_i x[b, s]),   i = ids[b]
// with A_i [r_i, in], B_i [out, r_i] of adapter i; ids[b] < 0: y = base.
// A is stored [adapters, r_pad, in] and B [adapters, out, r_pad], bf16, rows and
// columns past the adapter's own rank ignored. fp32 accumulation throughout,
// one rounding of y to bf16. The padding of A and B holds zeros.
//
// Two forms. lora_tokens_kernel: few tokens per request. The weights are what is read (2
// bytes per product), each by one CTA of a cluster that serves one request: the
// cluster's warps share the rank rows of A (and, for small ranks, slices of the
// contraction), every partial sum is stored into all CTAs' shared memory, and
// after one cluster barrier each CTA computes its slice of the outputs. One
// launch, fixed summation order.
//
// lora_shrink_kernel + lora_expand_kernel: many tokens per request, on tcgen05.
// Both are bound by the bytes of x and of base and y, so a CTA is a stream of
// TMA tiles with as much in flight as fits, and the products hide behind it:
//   shrink  t = scale_i A_i x for 128 tokens, the contraction split over a
//           cluster until the CTAs fill the device; partial sums are added
//           through distributed shared memory in rank order; t is rounded to
//           bf16 once (the operand type of the second product: at most 2^-9 of
//           each |t_r B_r|, below the rounding of y where |B t| <= |y|);
//   expand  y = base + B_i t for 128 tokens x 128 outputs: base arrives by TMA,
//           is added to the accumulator in place in shared memory and leaves by
//           a TMA store. Launched as a dependent of shrink: its base and B tiles
//           load while shrink still runs.
// x, base and y are three-dimensional maps (channel, token, request), so a tile
// never crosses into another request and ragged edges are zero-filled or cut.
#include <cudaTypedefs.h>

#include <mutex>

#include "cluster.cuh"
#include "sm100.cuh"

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

// ------------------------------------------------------------------ many tokens
constexpr int kShrinkStages = 5;
constexpr int kShrinkX = 128 * 64 * 2;    // x tile of a stage: 128 tokens x 64 channels

__host__ __device__ constexpr int shrink_rank(int r_pad) { return (r_pad + 15) / 16 * 16; }   // N of the product
__host__ __device__ constexpr int shrink_stage(int r_pad) { return kShrinkX + shrink_rank(r_pad) * 128; }
__host__ __device__ constexpr int shrink_sums(int r_pad) { return 128 * (shrink_rank(r_pad) + 4) * 4; }
__host__ __device__ constexpr int shrink_smem(int r_pad) {
  return kShrinkStages * ((shrink_stage(r_pad) + 1023) / 1024 * 1024) + 256 + 1024;
}
static_assert(shrink_sums(kLoraMaxRank) <= kShrinkStages * kShrinkX, "the sums reuse the stages");

constexpr uint32_t idesc_bf16(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ uint32_t tmem_cols(int n) { return n <= 32 ? 32u : n <= 64 ? 64u : 128u; }

// grid (token tiles x cluster, requests), 192 threads: warps 0-3 epilogue, 4 TMA, 5 MMA
__global__ void __launch_bounds__(192)
lora_shrink_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a,
                   const __grid_constant__ Lora p, __nv_bfloat16* t, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n = shrink_rank(p.r_pad), stage_bytes = (shrink_stage(p.r_pad) + 1023) / 1024 * 1024;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kShrinkStages * stage_bytes);
  uint64_t* empty = full + kShrinkStages;
  uint64_t* acc_full = empty + kShrinkStages;
  uint64_t* drain = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int s0 = blockIdx.x / splits * 128, b = blockIdx.y;
  grid_launch_dependents();
  const int id = lora_id(p, b, err);
  if (id < 0) return;                      // (all CTAs of the cluster serve one request)
  const int blocks = (p.in + 63) / 64, per = (blocks + splits - 1) / splits;
  const int first = min(blocks, split * per), count = min(blocks, first + per) - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kShrinkStages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    mbar_init(smem_u32(acc_full), 1);
    mbar_init(smem_u32(drain), 1);
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), tmem_cols(n));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 4) {
    if (lane == 0) {
      int issued = 0;
      bool ok = true;
      for (int i = 0; i < count; ++i) {
        const int st = i % kShrinkStages;
        if (!mbar_wait(smem_u32(&empty[st]), ((i / kShrinkStages) & 1) ^ 1, err)) { ok = false; break; }
        const uint32_t dst = smem_u32(smem + st * stage_bytes), bar = smem_u32(&full[st]);
        mbar_arrive_expect_tx(bar, uint32_t(kShrinkX + n * 128));
        tma_load_3d(dst, &tm_x, bar, (first + i) * 64, s0, b);
        tma_load_3d(dst + kShrinkX, &tm_a, bar, (first + i) * 64, 0, id);
        issued = i + 1;
      }
      if (!ok)   // let queued copies land before the shared memory is released
        for (int i = max(0, issued - kShrinkStages); i < issued; ++i)
          mbar_wait(smem_u32(&full[i % kShrinkStages]), (i / kShrinkStages) & 1, nullptr, 100000000ull);
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      bool ok = true;
      const uint32_t idesc = idesc_bf16(0) | (uint32_t(n >> 3) << 17);
      for (int i = 0; i < count; ++i) {
        const int st = i % kShrinkStages;
        if (!mbar_wait(smem_u32(&full[st]), (i / kShrinkStages) & 1, err)) { ok = false; break; }
        tc_fence_after();
        const uint64_t xd = smem_desc_k_sw128(smem_u32(smem + st * stage_bytes));
        const uint64_t ad = smem_desc_k_sw128(smem_u32(smem + st * stage_bytes + kShrinkX));
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(tmem, xd + uint64_t(2 * k), ad + uint64_t(2 * k), idesc, (i | k) != 0);
        tc_commit(smem_u32(&empty[st]));
      }
      if (ok) tc_commit(smem_u32(acc_full));
      tc_commit(smem_u32(drain));
      mbar_wait(smem_u32(drain), 0, ok ? err : nullptr, 100000000ull);
    }
    __syncwarp();
  } else {
    // the sums of this CTA's slice, one token per thread, over the stages (all
    // read once the accumulator is complete)
    const bool got = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_full), 0, err)) && count > 0;
    tc_fence_after();
    const int row = warp * 32 + lane;
    float4* dst = reinterpret_cast<float4*>(smem + row * (n + 4) * 4);
    for (int c = 0; c < n; c += 16) {
      uint32_t v[16];
      if (got) {
        tc_ld_32x32b_x16(tmem + (uint32_t(warp * 32) << 16) + uint32_t(c), v);
        tc_wait_ld();
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        dst[c / 4 + e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                     __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols(n));
  }
  cluster_sync();
  // ---- join the slices: this CTA finishes 128 / splits tokens, eight ranks per piece
  const int rank = min(__ldg(p.ranks + id), p.r_pad), groups = p.r_pad / 8, rows = 128 / splits;
  const float scale = __ldg(p.scales + id);
  for (int i = threadIdx.x; i < rows * groups; i += blockDim.x) {
    const int row = split * rows + i / groups, g = i % groups;
    if (s0 + row >= p.seq) continue;
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < splits; ++k) {
      const uint32_t src = cluster_map(smem + row * (n + 4) * 4 + g * 32, uint32_t(k));
      const float4 lo = ld_cluster_f32x4(src), hi = ld_cluster_f32x4(src + 16);
      f[0] += lo.x; f[1] += lo.y; f[2] += lo.z; f[3] += lo.w;
      f[4] += hi.x; f[5] += hi.y; f[6] += hi.z; f[7] += hi.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = g * 8 + e < rank ? f[e] * scale : 0.0f;
    reinterpret_cast<uint4*>(t + (int64_t(b) * p.seq + s0 + row) * p.r_pad)[g] = pack8(f);
  }
  cluster_sync();
}

constexpr int kExpandN = 128;
constexpr int kExpandBase = 128 * kExpandN * 2;         // 32 KB: two 64-output panels
__host__ __device__ constexpr int expand_panels(int r_pad) { return (r_pad + 63) / 64; }
__host__ __device__ constexpr int expand_smem(int r_pad) { return kExpandBase + expand_panels(r_pad) * 32768 + 128 + 1024; }

// grid (output tiles, token tiles, requests), 160 threads: warps 0-3 epilogue, 4 TMA and MMA
__global__ void __launch_bounds__(160)
lora_expand_kernel(const __grid_constant__ CUtensorMap tm_t, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_base, const __grid_constant__ CUtensorMap tm_y,
                   const __grid_constant__ Lora p, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int panels = expand_panels(p.r_pad);
  uint8_t* t_tile = smem + kExpandBase;
  uint8_t* b_tile = t_tile + panels * 16384;
  uint64_t* bars = reinterpret_cast<uint64_t*>(b_tile + panels * 16384);
  uint64_t* base_full = bars;
  uint64_t* b_full = bars + 1;
  uint64_t* t_full = bars + 2;
  uint64_t* acc_full = bars + 3;
  uint64_t* drain = bars + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int o0 = blockIdx.x * kExpandN, s0 = blockIdx.y * 128, b = blockIdx.z;
  const int id = __ldg(p.ids + b);
  const bool adapt = id >= 0 && id < p.adapters;
  if (!adapt && p.base == p.y) {                        // nothing to add, nothing to copy
    grid_wait();
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) mbar_init(smem_u32(&bars[i]), 1);
    fence_barrier_init();
  }
  if (warp == 4 && adapt) tmem_alloc(smem_u32(tmem_slot), kExpandN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 4) {
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(base_full), kExpandBase);
      for (int h = 0; h < 2; ++h)
        tma_load_3d(smem_u32(smem + h * 16384), &tm_base, smem_u32(base_full), o0 + h * 64, s0, b);
      if (adapt) {
        mbar_arrive_expect_tx(smem_u32(b_full), uint32_t(panels) * 16384u);
        for (int h = 0; h < panels; ++h)
          tma_load_3d(smem_u32(b_tile + h * 16384), &tm_b, smem_u32(b_full), h * 64, o0, id);
        grid_wait();                                    // t is complete
        mbar_arrive_expect_tx(smem_u32(t_full), uint32_t(panels) * 16384u);
        for (int h = 0; h < panels; ++h)
          tma_load_3d(smem_u32(t_tile + h * 16384), &tm_t, smem_u32(t_full), h * 64, s0, b);
        const bool got_b = mbar_wait(smem_u32(b_full), 0, err);
        const bool ok = mbar_wait(smem_u32(t_full), 0, err) && got_b;
        if (ok) {
          tc_fence_after();
          const int steps = (min(__ldg(p.ranks + id), p.r_pad) + 15) / 16;
          for (int k = 0; k < steps; ++k) {
            const uint64_t off = uint64_t(((k >> 2) * 16384 + (k & 3) * 32) >> 4);
            tc_mma_f16_ss(tmem, smem_desc_k_sw128(smem_u32(t_tile)) + off, smem_desc_k_sw128(smem_u32(b_tile)) + off,
                          idesc_bf16(kExpandN), k > 0);
          }
          tc_commit(smem_u32(acc_full));
        }
        tc_commit(smem_u32(drain));
        mbar_wait(smem_u32(drain), 0, ok ? err : nullptr, 100000000ull);
      }
    }
    __syncwarp();
  } else {
    bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(base_full), 0, err));
    if (adapt) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_full), 0, err)) && ok;
      tc_fence_after();
      const int row = warp * 32 + lane;
      if (ok) {
#pragma unroll
        for (int c = 0; c < kExpandN; c += 32) {
          uint32_t v[32];
          tc_ld_32x32b_x32(tmem + (uint32_t(warp * 32) << 16) + uint32_t(c), v);
          tc_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int piece = (c & 63) / 8 + q;
            uint4* at = reinterpret_cast<uint4*>(smem + (c >> 6) * 16384 + row * 128 + ((piece ^ (row & 7)) << 4));
            float f[8];
            unpack8(*at, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += __uint_as_float(v[8 * q + e]);
            *at = pack8(f);
          }
        }
        fence_proxy_async_shared();
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (threadIdx.x == 0 && ok) {
      if (!adapt) grid_wait();     // (this grid may not end before the one it depends on)
      for (int h = 0; h < 2; ++h)
        if (o0 + h * 64 < p.out) tma_store_3d(&tm_y, smem_u32(smem + h * 16384), o0 + h * 64, s0, b);
      tma_store_commit();
      tma_store_wait();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 && adapt) {
    tc_fence_after();
    tmem_dealloc(tmem, kExpandN);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 lora_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(q);
  });
  return fn;
}

// bf16 [d2, d1, d0] with element strides (s2, s1, 1), box {64, rows, 1}, 128-byte swizzle
int make_map(CUtensorMap* map, const void* base, int64_t d0, int64_t d1, int64_t d2, int64_t s1, int64_t s2, int rows) {
  auto fn = lora_encode_fn();
  if (!fn) return set_error(QIA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {cuuint64_t(d0), cuuint64_t(d1), cuuint64_t(d2)};
  cuuint64_t strides[2] = {cuuint64_t(s1 * 2), cuuint64_t(s2 * 2)};
  cuuint32_t box[3] = {64u, cuuint32_t(rows), 1u};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(QIA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
  return QIA_OK;
}

int launch_tiles(const Lora& p, void* workspace, cudaStream_t st) {
  static const bool ready =
      cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           shrink_smem(kLoraMaxRank)) == cudaSuccess &&
      cudaFuncSetAttribute(lora_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           expand_smem(kLoraMaxRank)) == cudaSuccess;
  if (!ready) return set_error(QIA_ERR_CUDA, "qia_lora_add: cudaFuncSetAttribute failed");
  __nv_bfloat16* t = (__nv_bfloat16*)workspace;
  CUtensorMap tm_x, tm_a, tm_t, tm_b, tm_base, tm_y;
  int rc = make_map(&tm_x, p.x, p.in, p.seq, p.batch, p.x_ss, p.x_sb, 128);
  if (!rc) rc = make_map(&tm_a, p.a, p.in, p.r_pad, p.adapters, p.in, int64_t(p.r_pad) * p.in, shrink_rank(p.r_pad));
  if (!rc) rc = make_map(&tm_t, t, p.r_pad, p.seq, p.batch, p.r_pad, int64_t(p.seq) * p.r_pad, 128);
  if (!rc) rc = make_map(&tm_b, p.b, p.r_pad, p.out, p.adapters, p.r_pad, int64_t(p.out) * p.r_pad, kExpandN);
  if (!rc) rc = make_map(&tm_base, p.base, p.out, p.seq, p.batch, p.base_ss, p.base_sb, 128);
  if (!rc) rc = make_map(&tm_y, p.y, p.out, p.seq, p.batch, p.y_ss, p.y_sb, 128);
  if (rc) return rc;
  const int64_t tiles = (int64_t(p.seq) + 127) / 128;
  const int blocks = (p.in + 63) / 64;
  // the contraction is split until the CTAs fill the device, down to two stages' worth each
  int splits = 1;
  while (splits < 8 && tiles * p.batch * splits < sm_count() && blocks >= 4 * splits * 2) splits *= 2;
  rc = launch_cluster("lora_shrink_kernel", lora_shrink_kernel, dim3(unsigned(tiles * splits), unsigned(p.batch)), 192,
                      size_t(shrink_smem(p.r_pad)), splits, st, tm_x, tm_a, p, t, device_error_word());
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((p.out + kExpandN - 1) / kExpandN), unsigned(tiles), unsigned(p.batch));
  cfg.blockDim = dim3(160);
  cfg.dynamicSmemBytes = size_t(expand_smem(p.r_pad));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, lora_expand_kernel, tm_t, tm_b, tm_base, tm_y, p, device_error_word());
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(QIA_ERR_CUDA, "lora_expand_kernel: %s", cudaGetErrorString(e));
  }
  return QIA_OK;
}

// Few tokens per request, or a broadcast row or request (a zero stride, which
// a tensor map does not take).
bool use_tokens(int64_t batch, int64_t seq, const Lora& p) {
  if (seq <= 8) return true;
  return p.x_ss <= 0 || p.base_ss <= 0 || p.y_ss <= 0 ||
         (batch > 1 && (p.x_sb <= 0 || p.base_sb <= 0 || p.y_sb <= 0));
}

}  // namespace
}  // namespace qia

using namespace qia;

extern "C" int64_t qia_lora_workspace_bytes(int64_t batch, int64_t seq, int64_t r_pad) {
  return seq <= 8 || batch <= 0 || r_pad <= 0 ? 0 : batch * seq * r_pad * 2;   // t of the two-kernel form
}

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
  if (use_tokens(batch, seq, p)) return launch_tokens(p, as_stream(stream));
  if (!workspace || !aligned(workspace, 16))
    return set_error(QIA_ERR_INVALID, "%s: the workspace is null or misaligned", who);
  // (a request that is alone needs no request stride: any value that a map takes)
  if (batch == 1) p.x_sb = p.base_sb = p.y_sb = 8;
  return launch_tiles(p, workspace, as_stream(stream));
}

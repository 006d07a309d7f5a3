// Low-rank adapters of many requests beside a shared projection:
//   y[b, s] = base[b, s] + scale_i * B_i (A_i x[b, s]),   i = ids[b]
// with A_i [r_i, in], B_i [out, r_i] of adapter i; ids[b] < 0: y = base.
// A is stored [adapters, r_pad, in] and B [adapters, out, r_pad], bf16, with zeros
// past an adapter's own rank. fp32 accumulation throughout, one rounding of y to bf16.
//
// Two forms, chosen by their estimated times (plan_tokens, tiles_us).
// lora_tokens_kernel: eight tokens of a request, or eight single-token requests of
// one adapter, are the columns of m16n8k16 products whose rows are weights: the
// weights are what is read (2 bytes per product), straight from global memory into
// the operand registers of the warp that uses them, and the call is a chain of
// latencies -- id, rows of A, exchange, rows of B (requested before the exchange), y.
// A cluster of up to eight CTAs serves eight tokens: its warps share the 16-row
// blocks of A and slices of the contraction, every partial sum is stored into all
// CTAs' shared memory, and after one cluster barrier each CTA computes its slice of
// the outputs with t = scale A x as a sum of two bf16 numbers (2^-17 of t). One
// launch, fixed summation order. (With one lane per weight row and fp32 FMAs the
// same schedule executed ten times the instructions.) 32 single tokens, 4096 -> 4096,
// rank 64, eight adapters: 9.3 us, 5 us of them launch and latency; 4 x 77 tokens,
// 12288 -> 4096, rank 16: 11.3 us.
//
// lora_shrink_kernel + lora_expand_kernel: many tokens per request, on tcgen05.
// Both are bound by the bytes of x and of base and y, so a CTA is a stream of
// TMA tiles with as much in flight as fits, and the products hide behind it (four
// requests of 4096 tokens, 4096 -> 12288, rank 64: 168 us, 86 % of the copy's rate:
// shrink 31 us, its bytes 21; expand the rest, its bytes 123):
//   shrink  t = scale_i A_i x for 128 tokens, the contraction split over a
//           cluster until the CTAs fill the device; partial sums are added
//           through distributed shared memory in rank order; t is rounded to
//           bf16 once (the operand type of the second product: at most 2^-8 of
//           each |t_r B_r|, below the rounding of y where |B t| <= |y|; the token
//           form keeps two parts, so precision goes with the form);
//   expand  y = base + B_i t for 128 tokens x 128 outputs: base arrives by TMA,
//           is added to the accumulator in place in shared memory and leaves by
//           a TMA store. Launched as a dependent of shrink: its base and B tiles
//           load while shrink still runs.
// x, base and y are three-dimensional maps (channel, token, request), so a tile
// never crosses into another request and ragged edges are zero-filled or cut.
#include <cudaTypedefs.h>

#include <cmath>
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

constexpr int kTokens = 8;                      // tokens per cluster
constexpr int kMaxSlices = 16;
constexpr int kSums = kMaxSlices * 64;          // slices x ranks: at most 64 warps, 16 ranks each

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Slices of the contraction: the cluster's warps over the 16-row blocks of A.
__host__ __device__ __forceinline__ int token_slices(int r_pad, int ctas, int chunks) {
  const int blocks = (r_pad + 15) / 16, n = kTokWarps * ctas / blocks, most = chunks < kMaxSlices ? chunks : kMaxSlices;
  return n < 1 ? 1 : n < most ? n : most;
}

// kSteps: 16-rank steps of r_pad (2, 4 or 8); a warp has the rows of B of
// up to four blocks of outputs in flight.
template <int kSteps>
__global__ void __launch_bounds__(kTokWarps * 32, 2) lora_tokens_kernel(const __grid_constant__ Lora p, int* err) {
  constexpr int kPre = 8;                       // chunks of 32 channels (of 16 rows) in flight
  constexpr int kRounds = kSteps == 8 ? 2 : 4;
  __shared__ __align__(16) float part[kSums * kTokens];                       // [slice][rank][token]
  __shared__ __align__(16) __nv_bfloat16 t_hi[kTokens][kLoraMaxRank + 8], t_lo[kTokens][kLoraMaxRank + 8];
  __shared__ int col_b[kTokens], col_n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int ctas = int(cluster_size()), cta = int(cluster_rank()), b = blockIdx.y;
  // ---- the columns: eight tokens of request b, or, of single-token requests, b
  // and the next seven with the same adapter (the others of the eight leave it to
  // the first of them, so the weights are read once)
  const int s0 = int(blockIdx.x) / ctas * kTokens;
  const int raw = __ldg(p.ids + b);
  if (p.seq == 1) {
    if (warp == 0) {
      int rank = 0, found = 0;
      for (int i0 = 0; i0 < p.batch && found < kTokens; i0 += 32) {
        const int i = i0 + lane, d = b - i0;
        const uint32_t same = __ballot_sync(0xffffffffu, i < p.batch && __ldg(p.ids + i) == raw);
        const uint32_t later = d <= 0 ? same : d >= 32 ? 0u : same & (0xffffffffu << d);
        const int at = found + __popc(later & ((1u << lane) - 1u));
        if (((later >> lane) & 1) && at < kTokens) col_b[at] = i;
        rank += __popc(same ^ later);
        found += __popc(later);
      }
      if (lane == 0) col_n = rank % kTokens ? 0 : min(found, kTokens);
    }
    __syncthreads();
    if (col_n == 0) return;              // (the same in every CTA of the cluster)
  } else {
    if (threadIdx.x < kTokens) col_b[threadIdx.x] = b;
    if (threadIdx.x == 0) col_n = min(kTokens, p.seq - s0);
    __syncthreads();
  }
  cluster_arrive();
  const int live = col_n, id = lora_id(p, b, err), at = max(id, 0);
  // element offset of column `col` in a tensor of strides (sb, ss)
  const auto column = [&](int col, int64_t sb, int64_t ss) {
    return col_b[col] * sb + (p.seq == 1 ? int64_t(0) : int64_t(s0 + col) * ss);
  };
  const __nv_bfloat16* x = p.x + column(min(g, live - 1), p.x_sb, p.x_ss);

  // ---- A x: 16 rows x this warp's slice; the products take channels 8 c .. 8 c + 7
  // of a chunk from every c. The rows are requested before the adapter's rank is
  // known (they exist up to r_pad).
  const int blocks = (p.r_pad + 15) / 16, chunks = (p.in + 31) / 32, slices = token_slices(p.r_pad, ctas, chunks);
  const int per = (chunks + slices - 1) / slices, ranks16 = blocks * 16;
  const int items = id < 0 ? 0 : blocks * slices;
  for (int item = warp * ctas + cta; item < items; item += kTokWarps * ctas) {
    const int block = item % blocks, slice = item / blocks, end = min(chunks, (slice + 1) * per);
    const uint4* row0 = reinterpret_cast<const uint4*>(p.a + (int64_t(at) * p.r_pad + min(16 * block + g, p.r_pad - 1)) * p.in);
    const uint4* row1 =
        reinterpret_cast<const uint4*>(p.a + (int64_t(at) * p.r_pad + min(16 * block + g + 8, p.r_pad - 1)) * p.in);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = slice * per; k0 < end; k0 += kPre) {
      uint4 a0[kPre], a1[kPre], xv[kPre];
#pragma unroll
      for (int k = 0; k < kPre; ++k) {
        const int i = (k0 + k) * 4 + c;
        const bool held = k0 + k < end && i * 8 < p.in;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        a0[k] = held ? __ldg(row0 + i) : zero;
        a1[k] = held ? __ldg(row1 + i) : zero;
        xv[k] = held && g < live ? __ldg(reinterpret_cast<const uint4*>(x) + i) : zero;
      }
#pragma unroll
      for (int k = 0; k < kPre; ++k) {
        mma_bf16(acc, a0[k].x, a1[k].x, a0[k].y, a1[k].y, xv[k].x, xv[k].y);
        mma_bf16(acc, a0[k].z, a1[k].z, a0[k].w, a1[k].w, xv[k].z, xv[k].w);
      }
    }
    if (item == warp * ctas + cta) cluster_wait();   // every CTA runs: its shared memory may be stored to
    if (2 * c < live) {
      float* dst = part + (slice * ranks16 + 16 * block + g) * kTokens + 2 * c;
      for (int r = 0; r < ctas; ++r) {
        const uint32_t peer = cluster_map(dst, uint32_t(r));
        st_cluster_f32x2(peer, acc[0], acc[1]);
        st_cluster_f32x2(peer + 8 * kTokens * 4, acc[2], acc[3]);
      }
    }
  }
  if (warp * ctas + cta >= items) cluster_wait();

  // ---- rows of B and base of kRounds blocks of 16 outputs: channels 16 k + 4 c .. + 3 of every c
  const int rank = id < 0 ? 0 : min(max(__ldg(p.ranks + at), 0), p.r_pad), steps = (rank + 15) / 16;
  const float scale = __ldg(p.scales + at);
  // (this cluster's share of the outputs: blockIdx.z of gridDim.z)
  const int all_blocks = (p.out + 15) / 16, share = (all_blocks + int(gridDim.z) - 1) / int(gridDim.z);
  const int first_block = int(blockIdx.z) * share, out_blocks = min(all_blocks, first_block + share);
  const int out_end = min(p.out, out_blocks * 16), stride = ctas * kTokWarps;
  int64_t col_base[2], col_y[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    col_base[e] = column(min(2 * c + e, live - 1), p.base_sb, p.base_ss);
    col_y[e] = column(min(2 * c + e, live - 1), p.y_sb, p.y_ss);
  }
  uint2 w[kRounds][kSteps][2];
  float base[kRounds][2][2];
  const auto load = [&](int first) {
#pragma unroll
    for (int q = 0; q < kRounds; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int o = (first + q * stride) * 16 + g + 8 * h;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          w[q][k][h] = k < steps && 16 * k + 4 * c < p.r_pad && o < out_end
                           ? __ldg(reinterpret_cast<const uint2*>(p.b + (int64_t(at) * p.out + o) * p.r_pad + 16 * k + 4 * c))
                           : make_uint2(0u, 0u);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          base[q][h][e] = o < out_end && 2 * c + e < live ? bf16_to_f32(p.base[col_base[e] + o]) : 0.0f;
      }
  };
  int ob = first_block + cta * kTokWarps + warp;
  load(ob);
  cluster_sync();
  for (int i = threadIdx.x; i < ranks16 * kTokens; i += blockDim.x) {
    const int r = i / kTokens, tok = i % kTokens;
    float sum = 0.0f;
    if (tok < live && r < rank)
      for (int k = 0; k < slices; ++k) sum += part[(k * ranks16 + r) * kTokens + tok];
    sum *= scale;
    const __nv_bfloat16 hi = f32_to_bf16(sum);
    t_hi[tok][r] = hi;
    t_lo[tok][r] = f32_to_bf16(sum - bf16_to_f32(hi));
  }
  __syncthreads();
  uint2 th[kSteps], tl[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    th[k] = tl[k] = make_uint2(0u, 0u);
    if (k < steps) {
      th[k] = *reinterpret_cast<const uint2*>(&t_hi[g][16 * k + 4 * c]);
      tl[k] = *reinterpret_cast<const uint2*>(&t_lo[g][16 * k + 4 * c]);
    }
  }
  while (ob < out_blocks) {
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        if (k < steps) {
          mma_bf16(acc, w[q][k][0].x, w[q][k][1].x, w[q][k][0].y, w[q][k][1].y, th[k].x, th[k].y);
          mma_bf16(acc, w[q][k][0].x, w[q][k][1].x, w[q][k][0].y, w[q][k][1].y, tl[k].x, tl[k].y);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int o = (ob + q * stride) * 16 + g + 8 * h, tok = 2 * c + e;
          if (o < out_end && tok < live)
            p.y[col_y[e] + o] = f32_to_bf16(base[q][h][e] + acc[2 * h + e]);
        }
    }
    ob += kRounds * stride;
    if (ob < out_blocks) load(ob);
  }
}

// How the token form would run: CTAs of a cluster, clusters that share the outputs
// of a group of eight tokens (each computes t), and about how long, in us. A
// cluster takes 5 us and its weights, 31 MB / ms and CTA; beyond four fifths of an SM's
// worth of CTAs two share an SM (1.4 times as long), beyond 1.85 there is another
// wave; and L2 gives about 4 MB / us. On a B200, 4096 -> 12288 at rank 128, one token:
// 22 us without sharing, 10 with six clusters; 12288 -> 4096 at rank 16, 4 x 77
// tokens: 15.8 us in clusters of eight (two waves), 11.3 in clusters of four.
struct TokenPlan {
  int ctas, shares;
  float us;
};

TokenPlan plan_tokens(const Lora& p) {
  int64_t groups = int64_t(p.batch) * ((p.seq + kTokens - 1) / kTokens);
  if (p.seq == 1) {      // requests of one adapter go together
    const int64_t most = int64_t(p.batch) / kTokens + p.adapters + 1;
    groups = groups < most ? groups : most;
  }
  TokenPlan best = {1, 1, INFINITY};
  // (a CTA has work for its warps down to 128 outputs or 256 channels)
  for (int ctas = 1; ctas <= 8 && (ctas == 1 || ctas * kTokWarps * 8 < p.out || ctas * kTokWarps * 16 < p.in); ctas *= 2) {
    const int pass = ctas * kTokWarps * (p.r_pad <= 64 ? 4 : 2) * 16;     // outputs that a cluster has in flight
    for (int shares = 1; shares <= 8 && (shares - 1) * pass < p.out; ++shares) {
      const float n = float(groups) * ctas * shares, sms = float(sm_count());
      const float mb = p.r_pad * 2e-6f * (p.in + float(p.out) / shares);
      const float us = fmaxf((n <= 0.8f * sms ? 1.0f : 1.4f * ceilf(n / (1.85f * sms))) * (5.0f + 32.0f * mb / ctas),
                             5.0f + 0.25f * float(groups) * shares * mb);
      if (us < best.us) best = {ctas, shares, us};
    }
  }
  return best;
}

int launch_tokens(const Lora& p, const TokenPlan& plan, cudaStream_t st) {
  const int64_t chunks = (int64_t(p.seq) + kTokens - 1) / kTokens;
  const dim3 grid(unsigned(chunks * plan.ctas), unsigned(p.batch), unsigned(plan.shares));
  const auto run = [&](auto kernel) {
    return launch_cluster("qia_lora_add", kernel, grid, kTokWarps * 32, 0, plan.ctas, st, p, device_error_word());
  };
  return p.r_pad <= 32 ? run(lora_tokens_kernel<2>) : p.r_pad <= 64 ? run(lora_tokens_kernel<4>) : run(lora_tokens_kernel<8>);
}

// ------------------------------------------------------------------ many tokens
constexpr int kShrinkX = 128 * 64 * 2;    // x tile of a stage: 128 tokens x 64 channels

__host__ __device__ constexpr int shrink_rank(int r_pad) { return (r_pad + 15) / 16 * 16; }   // N of the product
__host__ __device__ constexpr int shrink_stage(int r_pad) { return kShrinkX + shrink_rank(r_pad) * 128; }
__host__ __device__ constexpr int shrink_sums(int r_pad) { return 128 * (shrink_rank(r_pad) + 4) * 4; }
// Stages of a CTA: two CTAs per SM.
__host__ __device__ constexpr int shrink_stages(int r_pad) {
  return 110 * 1024 / shrink_stage(r_pad) < 6 ? 110 * 1024 / shrink_stage(r_pad) : 6;
}
__host__ __device__ constexpr int shrink_smem(int r_pad) { return shrink_stages(r_pad) * shrink_stage(r_pad) + 256 + 1024; }
static_assert((2 * 6 + 2) * 8 + 4 <= 256, "barriers of six stages and the TMEM address");
static_assert(shrink_sums(kLoraMaxRank) <= shrink_stages(kLoraMaxRank) * shrink_stage(kLoraMaxRank) &&
                  shrink_sums(64) <= shrink_stages(64) * shrink_stage(64),
              "the sums reuse the stages");
static_assert(shrink_stage(8) % 1024 == 0 && shrink_stage(kLoraMaxRank) % 1024 == 0, "swizzled tiles are 1 KB aligned");

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
  const int n = shrink_rank(p.r_pad), stage_bytes = shrink_stage(p.r_pad), stages = shrink_stages(p.r_pad);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
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
    for (int i = 0; i < stages; ++i) {
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
      int st = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      // x is read once: above 16 MB (an eighth of L2) it leaves L2 first, so that base
      // and y stay. On a B200 (us, as usual / first): 4096 tokens of 12288 channels (101 MB)
      // 40.6 / 36.9, of 4096 (34 MB) 29.0 / 27.7; 666 of 12288 (16 MB) 15.5 / 15.9, 800 of
      // 4096 (7 MB) 15.5 / 16.0.
      const uint64_t policy = l2_policy(int64_t(p.batch) * p.seq * p.in * 2 > (16 << 20));
      for (int i = 0; i < count; ++i) {
        if (!mbar_wait(smem_u32(&empty[st]), phase ^ 1, err)) { ok = false; break; }
        const uint32_t dst = smem_u32(smem + st * stage_bytes), bar = smem_u32(&full[st]);
        mbar_arrive_expect_tx(bar, uint32_t(kShrinkX + n * 128));
        tma_load_3d(dst, &tm_x, bar, (first + i) * 64, s0, b, policy);
        tma_load_3d(dst + kShrinkX, &tm_a, bar, (first + i) * 64, 0, id);
        ++issued;
        if (++st == stages) { st = 0; phase ^= 1; }
      }
      if (!ok)   // let queued copies land before the shared memory is released
        for (int i = max(0, issued - stages); i < issued; ++i)
          mbar_wait(smem_u32(&full[i % stages]), (i / stages) & 1, nullptr, 100000000ull);
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      bool ok = true;
      int st = 0;
      uint32_t phase = 0;
      const uint32_t idesc = idesc_bf16(0) | (uint32_t(n >> 3) << 17);
      for (int i = 0; i < count; ++i) {
        if (!mbar_wait(smem_u32(&full[st]), phase, err)) { ok = false; break; }
        tc_fence_after();
        const uint64_t xd = smem_desc_k_sw128(smem_u32(smem + st * stage_bytes));
        const uint64_t ad = smem_desc_k_sw128(smem_u32(smem + st * stage_bytes + kShrinkX));
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(tmem, xd + uint64_t(2 * k), ad + uint64_t(2 * k), idesc, (i | k) != 0);
        tc_commit(smem_u32(&empty[st]));
        if (++st == stages) { st = 0; phase ^= 1; }
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
static_assert(5 * 8 + 4 <= 128, "barriers and the TMEM address");

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
          // (one step at least: t is zero past the rank, and the accumulator has to be written)
          const int steps = max(1, (min(__ldg(p.ranks + id), p.r_pad) + 15) / 16);
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
  static std::atomic<uint64_t> shrink_allowed, expand_allowed;
  int rc = allow_launch("qia_lora_add", lora_shrink_kernel, 112 * 1024, &shrink_allowed, true);
  if (!rc) rc = allow_launch("qia_lora_add", lora_expand_kernel, expand_smem(kLoraMaxRank), &expand_allowed);
  if (rc) return rc;
  __nv_bfloat16* t = (__nv_bfloat16*)workspace;
  CUtensorMap tm_x, tm_a, tm_t, tm_b, tm_base, tm_y;
  rc = make_map(&tm_x, p.x, p.in, p.seq, p.batch, p.x_ss, p.x_sb, 128);
  if (!rc) rc = make_map(&tm_a, p.a, p.in, p.r_pad, p.adapters, p.in, int64_t(p.r_pad) * p.in, shrink_rank(p.r_pad));
  if (!rc) rc = make_map(&tm_t, t, p.r_pad, p.seq, p.batch, p.r_pad, int64_t(p.seq) * p.r_pad, 128);
  if (!rc) rc = make_map(&tm_b, p.b, p.r_pad, p.out, p.adapters, p.r_pad, int64_t(p.out) * p.r_pad, kExpandN);
  if (!rc) rc = make_map(&tm_base, p.base, p.out, p.seq, p.batch, p.base_ss, p.base_sb, 128);
  if (!rc) rc = make_map(&tm_y, p.y, p.out, p.seq, p.batch, p.y_ss, p.y_sb, 128);
  if (rc) return rc;
  const int64_t tiles = (int64_t(p.seq) + 127) / 128;
  const int blocks = (p.in + 63) / 64;
  // The contraction is split until the CTAs fill the device, down to eight
  // 64-channel blocks each, while the clusters run at once: two CTAs per SM, one
  // with clusters of sixteen (4096 -> 4096 at rank 64, eight requests of 333 tokens:
  // 24.2 us, 21.4 in fewer CTAs; sixteen of 77: 19.5 us, 27.1 in clusters of
  // sixteen, which take two waves; 12288 -> 4096, four of 77: 14.2 us in sixteen
  // splits, 16.3 in eight).
  static std::atomic<int> resident[17];
  const int64_t requests = tiles * p.batch;
  int splits = 1;
  while (splits < 16 && requests * splits < sm_count() && blocks >= 8 * splits * 2 &&
         requests <= (splits < 8 ? 2 : 1) *
                         resident_clusters(lora_shrink_kernel, 192, shrink_smem(p.r_pad), 2 * splits, resident))
    splits *= 2;
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
  count_launch();
  return QIA_OK;
}

// A broadcast row or request: a zero stride, which a tensor map does not take.
bool broadcast(const Lora& p) {
  return p.x_ss <= 0 || p.base_ss <= 0 || p.y_ss <= 0 ||
         (p.batch > 1 && (p.x_sb <= 0 || p.base_sb <= 0 || p.y_sb <= 0));
}

// About how long the two kernels take, in us: two launches, the contraction's
// length, the 128-token tiles and their weights, and the tokens of a tile. Measured on a B200
// (us, token form / two kernels): 12288 -> 4096, rank 16, 64 tokens: one request 7.2 /
// 13.5, four 8.4 / 14.1, sixteen 22.4 / 21.8; 4096 -> 4096, rank 64: one 9.0 / 12.3,
// four 13.7 / 12.9, eight 25.6 / 13.6; 4096 -> 12288, rank 128, one request: 16 tokens
// 10.3 / 12.6, 64 18.0 / 14.8. Up to eight tokens the token form was never slower.
float tiles_us(const Lora& p) {
  const float tiles = float(int64_t(p.batch) * ((p.seq + 127) / 128));
  return 8.0f + 3e-4f * p.in + tiles * (0.25f + 0.33f * (p.r_pad * 2e-6f * (float(p.in) + p.out))) +
         0.027f * float(p.seq < 128 ? p.seq : 128);
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
  const TokenPlan plan = plan_tokens(p);
  if (seq <= kTokens || broadcast(p)) return launch_tokens(p, plan, as_stream(stream));
  if (!workspace || !aligned(workspace, 16))
    return set_error(QIA_ERR_INVALID, "%s: the workspace is null or misaligned", who);
  if (plan.us <= tiles_us(p)) return launch_tokens(p, plan, as_stream(stream));
  // (a request that is alone needs no request stride: any value that a map takes)
  if (batch == 1) p.x_sb = p.base_sb = p.y_sb = 8;
  return launch_tiles(p, workspace, as_stream(stream));
}

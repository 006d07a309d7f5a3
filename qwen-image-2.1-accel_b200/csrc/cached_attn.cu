// Attention of few query rows over the INT8 prefix cache, and the entry point
// of the cached attention.
//
// cached_attn_rows_kernel: a tile of 16 query rows (token-major over the heads
// that share a K/V head) against a slice of the keys. What bounds it is the
// cache's bytes (one per element), so everything is arranged around streaming
// them once: every warp keeps a ring of kRowsRing 16-key steps (4 KB of codes
// each) in flight with cp.async into shared memory of its own -- no barrier
// between warps -- and reads 16-byte pieces back with no bank conflicts (piece
// p of row r is stored at p ^ (r & 7)). Each thread takes contiguous bytes and
// the contraction is permuted instead:
//   * q.k: thread c = lane % 4 holds channels [32c, 32c + 32) of key lane / 4,
//     and step j of the eight m16n8k16 products takes channels 32c + 4j .. + 3
//     of every c (the query fragments are loaded in the same order);
//   * p.v: thread g = lane / 4 holds channels [16g, 16g + 16) of four keys, and
//     product t of sixteen takes channel 16g + t of every g.
// INT8 -> f16 is two byte permutes and one subtraction per four codes: byte
// u = code + 128 under exponent byte 0x64 is the f16 1024 + u.
//
// Warps take 16-key steps of the CTA's slice in turn, each with a running
// maximum and sum of its own; the CTA joins its warps in shared memory and the
// CTAs of a cluster (which split the keys) join through distributed shared
// memory, in rank order: one launch, no workspace, results that do not depend
// on timing.
#include "cached_attn.cuh"
#include "cluster.cuh"

#include <cuda_fp16.h>

namespace qia {
namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsTile = 16;          // query rows per CTA
constexpr int kRowsStep = 16;          // keys per warp step
constexpr int kRowsRing = 4;           // steps in flight per warp
constexpr int kRowsCodes = 2 * kRowsStep * kCaD;            // K, then V codes of a step
constexpr int kRowsStage = kRowsCodes + 2 * kRowsStep * 4;  // and their scales
// f16 weights: w = 2^(t - M + 8) <= 2^15 while t <= M + 7, so the accumulators
// are rescaled only when a score passes its maximum by more than 7.
constexpr float kRowsBias = 8.0f, kRowsLag = 7.0f;

// The rings are done when the joining begins.
union RowsSmem {
  uint8_t ring[kRowsWarps][kRowsRing][kRowsStage];
  struct {
  float o[kRowsWarps][kRowsTile][kCaD + 4];
  float m[kRowsWarps][kRowsTile], l[kRowsWarps][kRowsTile];
  float om[kRowsTile][kCaD + 4];        // the CTA's joined rows, read by the cluster
  float mm[kRowsTile], lm[kRowsTile];
  };
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// codes (c0, c1) in bytes `sel` of the biased word -> f16 pair
__device__ __forceinline__ uint32_t code_pair(uint32_t biased, uint32_t sel) {
  return hsub2(prmt(biased, 0x64646464u, sel), 0x64806480u);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(smem))), "l"(gmem)
               : "memory");
}
__device__ __forceinline__ void cp_async4(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(uint32_t(__cvta_generic_to_shared(smem))), "l"(gmem)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 2^e with max|x| in [2^e, 2^(e+1)), e clamped to [-90, 126], and its inverse:
// a bf16 row times the inverse is exact in f16 down to 2^-24 of its maximum.
__device__ __forceinline__ void pow2_scale(uint32_t amax_bits, float& up, float& inv) {
  int e = int(amax_bits >> 23) - 127;
  e = min(max(e, -90), 126);
  up = __uint_as_float(uint32_t(e + 127) << 23);
  inv = __uint_as_float(uint32_t(127 - e) << 23);
}

__device__ __forceinline__ uint32_t absmax8(const uint4& v, uint32_t m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
  return m;
}

__global__ void __launch_bounds__(kRowsWarps * 32, 3) cached_attn_rows_kernel(const __grid_constant__ CachedAttn p) {
  extern __shared__ __align__(16) uint8_t rows_smem[];
  RowsSmem& sm = *reinterpret_cast<RowsSmem*>(rows_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int tile = blockIdx.x / splits, kvh = blockIdx.y, b = blockIdx.z;
  const int rows = p.sq * p.share;
  const int len = cached_len(p, b);
  const int cached_steps = (len + kRowsStep - 1) / kRowsStep;
  const int steps = cached_steps + (p.sk + kRowsStep - 1) / kRowsStep;
  const int per = (steps + splits - 1) / splits;
  const int step_end = min(steps, (split + 1) * per);

  const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
  const int8_t* kc = p.kc + head_row * kCaD;
  const int8_t* vc = p.vc + head_row * kCaD;
  const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;
  // key of this thread's V row i (of four), and of its score columns
  const auto vkey = [&](int i) { return 2 * c + (i & 1) + (i >> 1) * 8; };

  // ---- the warp's ring of cached steps: step0, step0 + kRowsWarps, ...
  const int cached_end = min(step_end, cached_steps);
  const int step0 = split * per + warp;
  const int mine_n = step0 < cached_end ? (cached_end - step0 + kRowsWarps - 1) / kRowsWarps : 0;
  const auto issue = [&](int i) {
    if (i < mine_n) {
      uint8_t* st = sm.ring[warp][i % kRowsRing];
      const int k0 = (step0 + i * kRowsWarps) * kRowsStep;
      // (keys past the length: any held row, weight 0)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int row = r4 * 4 + (lane >> 3), piece = lane & 7, at = row * kCaD + ((piece ^ (row & 7)) << 4);
        const int64_t src = int64_t(min(k0 + row, len - 1)) * kCaD + piece * 16;
        cp_async16(st + at, kc + src);
        cp_async16(st + kRowsCodes / 2 + at, vc + src);
      }
      cp_async4(st + kRowsCodes + lane * 4, (lane < 16 ? p.ks : p.vs) + head_row + min(k0 + (lane & 15), len - 1));
    }
    cp_async_commit();      // (an empty group keeps the count)
  };
  const auto mask_of = [&](int i) {   // of key lane % 16 of step i
    const int key = (step0 + i * kRowsWarps) * kRowsStep + (lane & 15);
    return i < mine_n && key < len && (!mask || __ldg(mask + key) != 0);
  };
#pragma unroll
  for (int i = 0; i < kRowsRing - 1; ++i) issue(i);
  bool valid = mask_of(0);

  // ---- query fragments, normalised per row by a power of two (f16 operands)
  uint32_t qa[8][4];
  float qup[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = tile * kRowsTile + g + 8 * r;
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows) {
      const __nv_bfloat16* src = p.q + b * p.q_sb + int64_t(row / p.share) * p.q_ss +
                                 int64_t(kvh * p.share + row % p.share) * p.q_sh + 32 * c;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = absmax8(x[i], m);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float inv;
    pow2_scale(m, qup[r], inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[8];
      unpack8(x[i], f);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        qa[2 * i + j][r] = cvt_f16x2(f[4 * j] * inv, f[4 * j + 1] * inv);
        qa[2 * i + j][r + 2] = cvt_f16x2(f[4 * j + 2] * inv, f[4 * j + 3] * inv);
      }
    }
  }

  float o[16][4];
#pragma unroll
  for (int t = 0; t < 16; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[t][e] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  // softmax of one step's scores s[nt][..] and p.v over four V rows given as
  // f16 pair producers
  const auto absorb = [&](float (&s)[2][4], const KeyScalars& mine, auto&& vpair) {
    float sk[4], lsv[4], rsv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sk[i] = __shfl_sync(0xffffffffu, mine.sk, vkey(i));
      lsv[i] = __shfl_sync(0xffffffffu, mine.lsv, vkey(i));
      rsv[i] = __shfl_sync(0xffffffffu, mine.rsv, vkey(i));
    }
    float t[2][4];   // [row][key]
    bool grow = false;
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) t[r][i] = fmaf(s[i >> 1][2 * r + (i & 1)] * qup[r], sk[i], lsv[i]);
      float x = fmaxf(fmaxf(t[r][0], t[r][1]), fmaxf(t[r][2], t[r][3]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      top[r] = x;
      grow |= x > m[r] + kRowsLag;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float mn = top[r] > m[r] + kRowsLag ? top[r] : m[r];
        const float f = m[r] == mn ? 1.0f : ex2_ftz(m[r] - mn);   // (m = -inf: 0)
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int tt = 0; tt < 16; ++tt) {
          o[tt][2 * r] *= f;
          o[tt][2 * r + 1] *= f;
        }
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float base = m[r] == -INFINITY ? 0.0f : m[r] - kRowsBias;
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = ex2_ftz(t[r][i] - base);
        l[r] = fmaf(w[i], rsv[i], l[r]);
      }
      pa[r] = cvt_f16x2(w[0], w[1]);
      pa[r + 2] = cvt_f16x2(w[2], w[3]);
    }
#pragma unroll
    for (int tt = 0; tt < 16; ++tt) mma_f16(o[tt], pa, vpair(0, tt), vpair(1, tt));
  };

  // ---- cached keys
  for (int i = 0; i < mine_n; ++i) {
    cp_async_wait<kRowsRing - 2>();
    __syncwarp();
    issue(i + kRowsRing - 1);              // into the slot of step i - 1, which every lane has read
    const bool next_valid = mask_of(i + 1);
    const uint8_t* st = sm.ring[warp][i % kRowsRing];
    const float* scales = reinterpret_cast<const float*>(st + kRowsCodes);
    const KeyScalars mine = key_scalars(p, scales[lane & 15], scales[16 + (lane & 15)], valid);
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(st + (nt * 8 + g) * kCaD + (((2 * c + h) ^ g) << 4));
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u = w[j] ^ 0x80808080u;
          mma_f16(s[nt], qa[4 * h + j], code_pair(u, 0x4140), code_pair(u, 0x4342));
        }
      }
    }
    // channel t of two V rows: interleave the rows' bytes, then widen
    uint32_t il[2][8];
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      const uint8_t* v0 = st + kRowsCodes / 2 + vkey(2 * pr) * kCaD + ((g ^ (2 * c)) << 4);
      const uint8_t* v1 = st + kRowsCodes / 2 + vkey(2 * pr + 1) * kCaD + ((g ^ (2 * c + 1)) << 4);
      const uint4 x = *reinterpret_cast<const uint4*>(v0), y = *reinterpret_cast<const uint4*>(v1);
      const uint32_t xa[4] = {x.x, x.y, x.z, x.w}, ya[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        il[pr][2 * k] = prmt(xa[k], ya[k], 0x5140) ^ 0x80808080u;
        il[pr][2 * k + 1] = prmt(xa[k], ya[k], 0x7362) ^ 0x80808080u;
      }
    }
    absorb(s, mine, [&](int pr, int tt) { return code_pair(il[pr][tt >> 1], (tt & 1) ? 0x4342 : 0x4140); });
    valid = next_valid;
  }
  cp_async_wait<0>();
  int step = step0 + mine_n * kRowsWarps;

  // ---- fresh keys: rows normalised by a power of two each, then as above
  for (; step < step_end; step += kRowsWarps) {
    const int k0 = (step - cached_steps) * kRowsStep;
    const auto fresh_ok = [&](int key) { return key < p.sk && (!mask || mask[p.extent + key] != 0); };
    float s[2][4], kup[2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int key = k0 + nt * 8 + g;
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = make_uint4(0u, 0u, 0u, 0u);
      if (fresh_ok(key)) {
        const uint4* src = reinterpret_cast<const uint4*>(p.k + b * p.k_sb + int64_t(key) * p.k_ss + kvh * p.k_sh + 32 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __ldg(src + i);
      }
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = absmax8(x[i], mx);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      float inv;
      pow2_scale(mx, kup[nt], inv);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[8];
        unpack8(x[i], f);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          mma_f16(s[nt], qa[2 * i + j], cvt_f16x2(f[4 * j] * inv, f[4 * j + 1] * inv),
                  cvt_f16x2(f[4 * j + 2] * inv, f[4 * j + 3] * inv));
      }
    }
    float vf[4][16], vup[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k0 + vkey(i);
      uint4 x[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
      if (fresh_ok(key)) {
        const uint4* src = reinterpret_cast<const uint4*>(p.v + b * p.v_sb + int64_t(key) * p.v_ss + kvh * p.v_sh + 16 * g);
        x[0] = __ldg(src);
        x[1] = __ldg(src + 1);
      }
      uint32_t mx = absmax8(x[1], absmax8(x[0], 0));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      float inv;
      pow2_scale(mx, vup[i], inv);
      unpack8(x[0], vf[i]);
      unpack8(x[1], vf[i] + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) vf[i][e] *= inv;
    }
    // lane j < 16 collects key j's scales from the threads that hold them
    const int j = lane & 15;
    float ks = 0.0f, vs = 0.0f;
    {
      const float k_lo = __shfl_sync(0xffffffffu, kup[0], (j & 7) * 4), k_hi = __shfl_sync(0xffffffffu, kup[1], (j & 7) * 4);
      ks = j < 8 ? k_lo : k_hi;
      float part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) part[i] = __shfl_sync(0xffffffffu, vup[i], (j & 7) >> 1);
      vs = j < 8 ? ((j & 1) ? part[1] : part[0]) : ((j & 1) ? part[3] : part[2]);
    }
    const KeyScalars mine = key_scalars(p, ks, vs, fresh_ok(k0 + j));
    absorb(s, mine, [&](int pr, int tt) { return cvt_f16x2(vf[2 * pr][tt], vf[2 * pr + 1][tt]); });
  }

  // ---- join the warps
  __syncthreads();          // (every ring is done)
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = g + 8 * r;
    if (c == 0) {
      sm.m[warp][row] = m[r];
      sm.l[warp][row] = l[r];
    }
    // product t, columns 2c and 2c + 1: channels 32c + t and 32c + 16 + t
#pragma unroll
    for (int t4 = 0; t4 < 4; ++t4) {
      float4* dst = reinterpret_cast<float4*>(&sm.o[warp][row][32 * c + 4 * t4]);
      dst[0] = make_float4(o[4 * t4][2 * r], o[4 * t4 + 1][2 * r], o[4 * t4 + 2][2 * r], o[4 * t4 + 3][2 * r]);
      dst[4] = make_float4(o[4 * t4][2 * r + 1], o[4 * t4 + 1][2 * r + 1], o[4 * t4 + 2][2 * r + 1],
                           o[4 * t4 + 3][2 * r + 1]);
    }
  }
  __syncthreads();
  const int live = min(kRowsTile, rows - tile * kRowsTile);
  for (int row = warp; row < live; row += kRowsWarps) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) mx = fmaxf(mx, sm.m[w][row]);
    float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float f = sm.m[w][row] == -INFINITY ? 0.0f : ex2_ftz(sm.m[w][row] - mx);
      sum = fmaf(sm.l[w][row], f, sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sm.o[w][row][lane + 32 * i], f, acc[i]);
    }
    if (lane == 0) {
      sm.mm[row] = mx;
      sm.lm[row] = sum;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm.om[row][lane + 32 * i] = acc[i];
  }
  cluster_sync();
  // ---- join the splits: CTA `split` of the cluster writes every splits-th row
  // when there are rows enough, else every splits-th channel group
  const int pieces = live * 32;   // (row, four channels)
  for (int i = split * int(blockDim.x) + int(threadIdx.x); i < pieces; i += splits * int(blockDim.x)) {
    const int row = i >> 5, ch = (i & 31) * 4;
    float mx = -INFINITY;
    for (int r = 0; r < splits; ++r) mx = fmaxf(mx, ld_cluster_f32(cluster_map(&sm.mm[row], r)));
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int r = 0; r < splits; ++r) {
      const float mr = ld_cluster_f32(cluster_map(&sm.mm[row], r));
      const float f = mr == -INFINITY ? 0.0f : ex2_ftz(mr - mx);
      sum = fmaf(ld_cluster_f32(cluster_map(&sm.lm[row], r)), f, sum);
      const float4 x = ld_cluster_f32x4(cluster_map(&sm.om[row][ch], r));
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    // no key at all: zeros (a NaN sum still divides, and stays NaN)
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int grow = tile * kRowsTile + row;
    __nv_bfloat16* dst = p.out + b * p.o_sb + int64_t(grow / p.share) * p.o_ss +
                         int64_t(kvh * p.share + grow % p.share) * p.o_sh + ch;
    const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    *reinterpret_cast<uint2*>(dst) = pack4(f);
  }
  cluster_sync();   // no CTA leaves while another reads its shared memory
}

}  // namespace

int launch_cached_rows(const CachedAttn& p, int batch, cudaStream_t st) {
  static const int smem = [] {
    return cudaFuncSetAttribute(cached_attn_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(sizeof(RowsSmem))) == cudaSuccess ? int(sizeof(RowsSmem)) : -1;
  }();
  if (smem < 0) return set_error(QIA_ERR_CUDA, "qia_cached_attention: cudaFuncSetAttribute failed");
  const int64_t tiles = (int64_t(p.sq) * p.share + kRowsTile - 1) / kRowsTile;
  const int64_t groups = tiles * p.kv_heads * batch;
  const int steps = (p.extent + kRowsStep - 1) / kRowsStep + (p.sk + kRowsStep - 1) / kRowsStep;
  // The keys are split as finely as leaves every warp two steps, up to a cluster
  // of eight, but not into a second wave that would be nearly empty: past one
  // wave (three CTAs per SM) only where that leaves several.
  const int64_t slots = 3 * int64_t(sm_count());
  int splits = 1;
  for (int s = 2; s <= 8; ++s) {
    if (steps < 2 * s * kRowsWarps) break;
    if (groups * s <= slots || groups * s >= 2 * slots || groups * (s - 1) > slots) splits = s;
  }
  const int64_t gx = tiles * splits;
  if (gx > 0x7fffffff) return set_error(QIA_ERR_UNSUPPORTED, "qia_cached_attention: too many query rows");
  return launch_cluster("qia_cached_attention", cached_attn_rows_kernel,
                        dim3(unsigned(gx), unsigned(p.kv_heads), unsigned(batch)), kRowsWarps * 32, size_t(smem),
                        splits, st, p);
}

}  // namespace qia

using namespace qia;

// The rows that share a K/V head fill one 16-row tile.
static bool use_rows(int64_t seq_q, int64_t share) { return seq_q * share <= 16; }

extern "C" int64_t qia_cached_attention_workspace_bytes(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t heads,
                                                        int64_t kv_heads, int64_t extent) {
  if (batch <= 0 || seq_q <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || heads / kv_heads > 128 ||
      use_rows(seq_q, heads / kv_heads) || !cached_use_wide(seq_q, heads / kv_heads))
    return 0;
  return cached_wide_workspace(batch, seq_k, kv_heads, extent);
}

extern "C" int qia_cached_attention(const void* q, const void* k, const void* v, const void* k_codes,
                                    const void* v_codes, const void* k_scales, const void* v_scales,
                                    const void* lengths, const void* key_valid, void* out, int64_t batch,
                                    int64_t seq_q, int64_t seq_k, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                    int64_t capacity, int64_t extent, const int64_t* strides, int64_t mask_stride,
                                    float sm_scale, void* workspace, void* stream) {
  const char* who = "qia_cached_attention";
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !lengths || !out || !strides)
    return set_error(QIA_ERR_INVALID, "%s: null pointer", who);
  if (seq_k > 0 && (!k || !v)) return set_error(QIA_ERR_INVALID, "%s: seq_k=%lld without k and v", who, (long long)seq_k);
  if (head_dim != kCaD) return set_error(QIA_ERR_UNSUPPORTED, "%s: head_dim=%lld (only 128)", who, (long long)head_dim);
  if (batch <= 0 || seq_q < 0 || seq_k < 0 || heads <= 0 || kv_heads <= 0 || capacity <= 0 || extent < 0 ||
      extent > capacity)
    return set_error(QIA_ERR_INVALID, "%s: batch=%lld seq_q=%lld seq_k=%lld heads=%lld kv_heads=%lld extent=%lld of %lld",
                     who, (long long)batch, (long long)seq_q, (long long)seq_k, (long long)heads, (long long)kv_heads,
                     (long long)extent, (long long)capacity);
  if (heads % kv_heads)
    return set_error(QIA_ERR_INVALID, "%s: heads=%lld is not a multiple of kv_heads=%lld", who, (long long)heads,
                     (long long)kv_heads);
  if (heads / kv_heads > 128 || kv_heads > 65535 || batch > 65535 || seq_q > (1 << 20) || seq_k > (1 << 20) ||
      capacity > (1 << 30))
    return set_error(QIA_ERR_UNSUPPORTED, "%s: batch=%lld seq_q=%lld seq_k=%lld heads=%lld/%lld capacity=%lld", who,
                     (long long)batch, (long long)seq_q, (long long)seq_k, (long long)heads, (long long)kv_heads,
                     (long long)capacity);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(k_codes, 16) ||
      !aligned(v_codes, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4) || !aligned(lengths, 4))
    return set_error(QIA_ERR_ALIGNMENT, "%s: misaligned pointer", who);
  for (int i = 0; i < 12; ++i)
    if (strides[i] % 8)
      return set_error(QIA_ERR_ALIGNMENT, "%s: stride %lld is not a multiple of 8", who, (long long)strides[i]);
  if (seq_q == 0) return QIA_OK;
  CachedAttn p;
  p.q = (const __nv_bfloat16*)q;
  p.k = (const __nv_bfloat16*)k;
  p.v = (const __nv_bfloat16*)v;
  p.out = (__nv_bfloat16*)out;
  p.kc = (const int8_t*)k_codes;
  p.vc = (const int8_t*)v_codes;
  p.ks = (const float*)k_scales;
  p.vs = (const float*)v_scales;
  p.lengths = (const int*)lengths;
  p.key_valid = (const uint8_t*)key_valid;
  int64_t* dst[12] = {&p.q_sb, &p.q_ss, &p.q_sh, &p.k_sb, &p.k_ss, &p.k_sh,
                      &p.v_sb, &p.v_ss, &p.v_sh, &p.o_sb, &p.o_ss, &p.o_sh};
  for (int i = 0; i < 12; ++i) *dst[i] = strides[i];
  p.mask_sb = mask_stride;
  p.sq = int(seq_q);
  p.sk = int(seq_k);
  p.heads = int(heads);
  p.kv_heads = int(kv_heads);
  p.share = int(heads / kv_heads);
  p.capacity = int(capacity);
  p.extent = int(extent);
  p.scale_log2 = (sm_scale > 0.0f ? sm_scale : 0.08838834764831845f) * 1.4426950408889634f;
  // rows that share a K/V head fill one 16-row tile, or the tensor-core tiles
  if (use_rows(seq_q, p.share)) return launch_cached_rows(p, int(batch), as_stream(stream));
  if (!cached_use_wide(seq_q, p.share)) return launch_cached_tiles(p, int(batch), as_stream(stream));
  return launch_cached_wide(p, int(batch), workspace, as_stream(stream));
}

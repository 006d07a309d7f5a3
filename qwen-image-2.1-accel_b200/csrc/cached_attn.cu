// Attention of few query rows over the INT8 prefix cache, and the entry point
// of the cached attention.
//
// cached_attn_rows_kernel: a tile of up to 8 or 16 query rows (token-major over
// the heads that share a K/V head) against a slice of the keys. What bounds it is
// the cache's bytes (one per element) and, next, the instructions that widen
// them, so the keys are the rows of the matrix products (m16n8k16 with the
// queries as its eight columns) and are streamed once: every warp keeps the next
// K or V half of a 32-key step in flight with cp.async into shared memory of its
// own -- no barrier between warps -- and the contraction is permuted so that each
// thread reads contiguous bytes:
//   * row (mt, g, half) of the two score tiles of a step, g = lane / 4, is key
//     4 g + 2 mt + half, so a thread owns the scores of four adjacent keys;
//   * k.q: thread (g, c = lane % 4) holds channels [32 c, +32) of its keys, and
//     product j of eight takes channels 32 c + 4 j .. + 3 of every c (the query
//     fragments are loaded in the same order);
//   * v.p: the weights are transposed in registers (movmatrix), which leaves
//     thread c the keys 8 c .. 8 c + 7; thread (g, c) holds channels [16 g, +16)
//     of them, and product t of eight takes channels 16 g + 2 t, + 1 of every g.
// Piece p (16 bytes) of row r is stored at p ^ swizzle(r): no bank conflicts in
// either read. INT8 -> f16 is two byte permutes and one subtraction per four
// codes: byte u = code + 128 under exponent byte 0x64 is the f16 1024 + u.
//
// Warps take 32-key steps of the CTA's slice in turn, each with a running
// maximum and sum of its own; the CTA joins its warps in shared memory and the
// CTAs of a cluster (which split the keys) join through distributed shared
// memory, in a fixed order: one launch, no workspace, results that do not depend
// on timing.
//
// On a B200, sixteen requests of 4097 to 16391 tokens, 32 / 8 heads, one token: 73 us,
// 5.8 TB/s (89 % of the copy's rate). 32 heads over 4229 tokens: 12.6 us for 35
// MB, of them 4.8 us launch, query, one fresh key and joining; the rest is latency,
// with seven warps per SM. (Clusters of up to sixteen and five CTAs per SM were
// slower, eight warps per CTA no faster.)
#include "cached_attn.cuh"
#include "cluster.cuh"

#include <cuda_fp16.h>

namespace qia {
namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsStep = 32;          // keys per warp step
constexpr int kRowsHalf = kRowsStep * (kCaD + 4);   // K (or V) codes of a step and their scales
// f16 weights: w = 2^(t - M + 8) <= 2^15 while t <= M + 7, so the accumulators
// are rescaled only when a score passes its maximum by more than 7.
constexpr float kRowsBias = 8.0f, kRowsLag = 7.0f;

// The staged steps are done when the joining begins.
template <int ROWS, int DEPTH>
union RowsSmem {
  struct {
    uint8_t half[kRowsWarps][2][DEPTH][kRowsHalf];
    float key[kRowsWarps][3][kRowsStep];   // the softmax's numbers of a step's keys
  };
  struct {
    float o[kRowsWarps][ROWS][kCaD + 4];
    float m[kRowsWarps][ROWS], l[kRowsWarps][ROWS];
    float om[ROWS][kCaD + 4];              // the CTA's joined rows, read by the cluster
    float mm[ROWS], lm[ROWS];
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

__device__ __forceinline__ int rows_swizzle(int row) { return ((row >> 2) & 1) ^ (((row >> 3) & 3) << 1); }

// Transposes an 8 x 8 matrix of f16 held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// NT: column tiles of eight query rows; DEPTH: steps that a warp holds, the next
// DEPTH - 1 whole and the halves of one more in flight.
template <int NT, int DEPTH>
__global__ void __launch_bounds__(kRowsWarps * 32, NT == 1 && DEPTH == 1 ? 4 : 3)
cached_attn_rows_kernel(const __grid_constant__ CachedAttn p) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(16) uint8_t rows_smem[];
  RowsSmem<ROWS, DEPTH>& sm = *reinterpret_cast<RowsSmem<ROWS, DEPTH>*>(rows_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = p.sq * p.share;                     // (one tile: at most ROWS)
  const int len = cached_len(p, b);
  const int cached_steps = (len + kRowsStep - 1) / kRowsStep;
  const int steps = cached_steps + (p.sk + kRowsStep - 1) / kRowsStep;
  const int per = (steps + splits - 1) / splits;
  const int step_end = min(steps, (split + 1) * per);

  const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
  const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;

  // ---- the warp's cached steps: step0, step0 + kRowsWarps, ...; z: 0 K, 1 V
  const int cached_end = min(step_end, cached_steps);
  const int step0 = split * per + warp;
  const int mine_n = step0 < cached_end ? (cached_end - step0 + kRowsWarps - 1) / kRowsWarps : 0;
  const auto issue = [&](int i, int z) {
    if (i < mine_n) {
      uint8_t* st = sm.half[warp][z][i % DEPTH];
      const int k0 = (step0 + i * kRowsWarps) * kRowsStep;
      const int8_t* codes = (z ? p.vc : p.kc) + head_row * kCaD;
      // (keys past the length: any held row, weight 0)
#pragma unroll
      for (int r8 = 0; r8 < 8; ++r8) {
        const int row = r8 * 4 + (lane >> 3), piece = lane & 7;
        cp_async16(st + row * kCaD + ((piece ^ rows_swizzle(row)) << 4),
                   codes + int64_t(min(k0 + row, len - 1)) * kCaD + piece * 16);
      }
      cp_async4(st + kRowsStep * kCaD + lane * 4, (z ? p.vs : p.ks) + head_row + min(k0 + lane, len - 1));
    }
    cp_async_commit();      // (an empty group keeps the count)
  };
  const auto mask_of = [&](int i) {   // of key `lane` of step i
    const int key = (step0 + i * kRowsWarps) * kRowsStep + lane;
    return i < mine_n && key < len && (!mask || __ldg(mask + key) != 0);
  };
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
    issue(i, 0);
    issue(i, 1);
  }
  bool valid = mask_of(0);

  // ---- query fragments, normalised per row by a power of two (f16 operands):
  // thread (g, c) holds channels [32 c, +32) of row 8 nt + g
  uint32_t qb[NT][8][2];
  float qup[NT][2];                    // of the rows whose scores it owns, 8 nt + 2 c + e
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = 8 * nt + g;
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
    float up, inv;
    pow2_scale(m, up, inv);
#pragma unroll
    for (int e = 0; e < 2; ++e) qup[nt][e] = __shfl_sync(0xffffffffu, up, 4 * (2 * c + e));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[8];
      unpack8(x[i], f);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        qb[nt][2 * i + j][0] = cvt_f16x2(f[4 * j] * inv, f[4 * j + 1] * inv);
        qb[nt][2 * i + j][1] = cvt_f16x2(f[4 * j + 2] * inv, f[4 * j + 3] * inv);
      }
    }
  }

  float o[NT][8][4];      // [..][t]: channels 16 g + 2 t (+ 1), rows 8 nt + 2 c (+ 1)
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][t][e] = 0.0f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.0f;
  }

  // The softmax of a step's scores s[nt][mt] -> transposed weights: column
  // fragments of two products of 16 keys (mt); `mine`: key `lane`'s numbers.
  const auto softmax = [&](float (&s)[NT][2][4], const KeyScalars& mine, uint32_t (&pb)[NT][2][2]) {
    float* key = sm.key[warp][0];
    __syncwarp();                  // (the previous step's reads are done)
    key[lane] = mine.sk;
    key[kRowsStep + lane] = mine.lsv;
    key[2 * kRowsStep + lane] = mine.rsv;
    __syncwarp();
    const float4 sk4 = *reinterpret_cast<const float4*>(key + 4 * g);
    const float4 lsv4 = *reinterpret_cast<const float4*>(key + kRowsStep + 4 * g);
    const float4 rsv4 = *reinterpret_cast<const float4*>(key + 2 * kRowsStep + 4 * g);
    const float sk[4] = {sk4.x, sk4.y, sk4.z, sk4.w}, lsv[4] = {lsv4.x, lsv4.y, lsv4.z, lsv4.w};
    const float rsv[4] = {rsv4.x, rsv4.y, rsv4.z, rsv4.w};
    float t[NT][2][4], top[NT][2];   // [..][row e][key 4 g + i], i = 2 mt + half
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          t[nt][e][i] = fmaf(s[nt][i >> 1][2 * (i & 1) + e] * qup[nt][e], sk[i], lsv[i]);
        float x = fmaxf(fmaxf(t[nt][e][0], t[nt][e][1]), fmaxf(t[nt][e][2], t[nt][e][3]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
        top[nt][e] = x;
        grow |= x > m[nt][e] + kRowsLag;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mn = top[nt][e] > m[nt][e] + kRowsLag ? top[nt][e] : m[nt][e];
          const float f = m[nt][e] == mn ? 1.0f : ex2_ftz(m[nt][e] - mn);   // (m = -inf: 0)
          m[nt][e] = mn;
          l[nt][e] *= f;
#pragma unroll
          for (int tt = 0; tt < 8; ++tt) {
            o[nt][tt][e] *= f;
            o[nt][tt][2 + e] *= f;
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[nt][e] == -INFINITY ? 0.0f : m[nt][e] - kRowsBias;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[e][i] = ex2_ftz(t[nt][e][i] - base);
          l[nt][e] = fmaf(w[e][i], rsv[i], l[nt][e]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pb[nt][i >> 1][i & 1] = transpose8x8(cvt_f16x2(w[0][i], w[1][i]));
    }
  };

  // ---- cached keys
  for (int i = 0; i < mine_n; ++i) {
    cp_async_wait<2 * DEPTH - 1>();        // K
    __syncwarp();
    const uint8_t* kst = sm.half[warp][0][i % DEPTH];
    const uint8_t* vst = sm.half[warp][1][i % DEPTH];
    const float ks = reinterpret_cast<const float*>(kst + kRowsStep * kCaD)[lane];
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][mt][e] = 0.0f;
      const int row = 4 * g + 2 * mt;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(kst + row * kCaD + (((2 * c + h) ^ rows_swizzle(row)) << 4));
        const uint4 y =
            *reinterpret_cast<const uint4*>(kst + (row + 1) * kCaD + (((2 * c + h) ^ rows_swizzle(row + 1)) << 4));
        const uint32_t xa[4] = {x.x, x.y, x.z, x.w}, ya[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u = xa[j] ^ 0x80808080u, v = ya[j] ^ 0x80808080u;
          const uint32_t a[4] = {code_pair(u, 0x4140), code_pair(v, 0x4140), code_pair(u, 0x4342), code_pair(v, 0x4342)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt][mt], a, qb[nt][4 * h + j][0], qb[nt][4 * h + j][1]);
        }
      }
    }
    __syncwarp();
    issue(i + DEPTH, 0);                   // (every lane has read K)
    const bool next_valid = mask_of(i + 1);
    cp_async_wait<2 * DEPTH - 1>();        // V
    __syncwarp();
    const float vs = reinterpret_cast<const float*>(vst + kRowsStep * kCaD)[lane];
    uint32_t pb[NT][2][2];
    softmax(s, key_scalars(p, ks, vs, valid), pb);
    valid = next_valid;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      // columns of the transposed weights: keys 8 c + 2 mt + half and + 4; the
      // rows' bytes are interleaved, then widened
      uint32_t il[2][8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = 8 * c + 2 * mt + half;
        const uint4 x = *reinterpret_cast<const uint4*>(vst + row * kCaD + ((g ^ rows_swizzle(row)) << 4));
        const uint4 y = *reinterpret_cast<const uint4*>(vst + (row + 4) * kCaD + ((g ^ rows_swizzle(row + 4)) << 4));
        const uint32_t xa[4] = {x.x, x.y, x.z, x.w}, ya[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          il[half][2 * k] = prmt(xa[k], ya[k], 0x5140) ^ 0x80808080u;
          il[half][2 * k + 1] = prmt(xa[k], ya[k], 0x7362) ^ 0x80808080u;
        }
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t a[4] = {code_pair(il[0][t], 0x4140), code_pair(il[0][t], 0x4342), code_pair(il[1][t], 0x4140),
                               code_pair(il[1][t], 0x4342)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][t], a, pb[nt][mt][0], pb[nt][mt][1]);
      }
    }
    __syncwarp();
    issue(i + DEPTH, 1);                   // (every lane has read V)
  }
  cp_async_wait<0>();
  int step = step0 + mine_n * kRowsWarps;

  // ---- fresh keys: rows normalised by a power of two each, then as above
  for (; step < step_end; step += kRowsWarps) {
    const int k0 = (step - cached_steps) * kRowsStep;
    const auto fresh_ok = [&](int key) { return key < p.sk && (!mask || mask[p.extent + key] != 0); };
    const auto row_of = [&](int z, int key) {
      return z ? p.v + b * p.v_sb + int64_t(key) * p.v_ss + kvh * p.v_sh : p.k + b * p.k_sb + int64_t(key) * p.k_ss + kvh * p.k_sh;
    };
    // lane j holds key j's scales: they are found first, four rows at a time, eight
    // lanes per row (a row at a time, sixteen fresh keys took 7 us)
    float up[2] = {1.0f, 1.0f}, inv[2] = {1.0f, 1.0f};
#pragma unroll 1
    for (int j0 = 0; j0 < min(kRowsStep, p.sk - k0); j0 += 4) {
      const int key = k0 + j0 + (lane >> 3);
      const bool held = fresh_ok(key);
      uint4 x[2][2];
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          x[z][i] = held ? __ldg(reinterpret_cast<const uint4*>(row_of(z, key)) + 2 * (lane & 7) + i)
                         : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        uint32_t m = absmax8(x[z][1], absmax8(x[z][0], 0u));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = __shfl_sync(0xffffffffu, m, 8 * (lane & 3));
        if (lane >> 2 == j0 >> 2) {
          pow2_scale(m, up[z], inv[z]);
          if (m == 0) up[z] = 0.0f;        // (as of a cached zero row)
        }
      }
    }
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][mt][e] = 0.0f;
      float f_inv[2];
      bool held[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = 4 * g + 2 * mt + half;
        f_inv[half] = __shfl_sync(0xffffffffu, inv[0], row);
        held[half] = fresh_ok(k0 + row);
      }
      if (!__any_sync(0xffffffffu, held[0] || held[1])) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2][8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = 4 * g + 2 * mt + half;
          unpack8(held[half] ? __ldg(reinterpret_cast<const uint4*>(row_of(0, k0 + row)) + 4 * c + i)
                             : make_uint4(0u, 0u, 0u, 0u), f[half]);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[half][e] *= f_inv[half];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t a[4] = {cvt_f16x2(f[0][4 * j], f[0][4 * j + 1]), cvt_f16x2(f[1][4 * j], f[1][4 * j + 1]),
                                 cvt_f16x2(f[0][4 * j + 2], f[0][4 * j + 3]), cvt_f16x2(f[1][4 * j + 2], f[1][4 * j + 3])};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt][mt], a, qb[nt][2 * i + j][0], qb[nt][2 * i + j][1]);
        }
      }
    }
    uint32_t pb[NT][2][2];
    softmax(s, key_scalars(p, up[0], up[1], fresh_ok(k0 + lane)), pb);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float v_inv[4];                      // keys 8 c + 2 mt + {0, 4, 1, 5}
      bool held[4], any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 8 * c + 2 * mt + (e >> 1) + 4 * (e & 1);
        v_inv[e] = __shfl_sync(0xffffffffu, inv[1], row);
        held[e] = fresh_ok(k0 + row);
        any |= held[e];
      }
      if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q) {        // channels 16 g + 8 q .. + 7
        float f[4][8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 8 * c + 2 * mt + (e >> 1) + 4 * (e & 1);
          unpack8(held[e] ? __ldg(reinterpret_cast<const uint4*>(row_of(1, k0 + row)) + 2 * g + q)
                          : make_uint4(0u, 0u, 0u, 0u), f[e]);
#pragma unroll
          for (int x = 0; x < 8; ++x) f[e][x] *= v_inv[e];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t a[4] = {cvt_f16x2(f[0][2 * t], f[1][2 * t]), cvt_f16x2(f[0][2 * t + 1], f[1][2 * t + 1]),
                                 cvt_f16x2(f[2][2 * t], f[3][2 * t]), cvt_f16x2(f[2][2 * t + 1], f[3][2 * t + 1])};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * q + t], a, pb[nt][mt][0], pb[nt][mt][1]);
        }
      }
    }
  }

  // ---- join the warps
  __syncthreads();          // (the staged steps are done)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 8 * nt + 2 * c + e;
      float sum = l[nt][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (g == 0) {
        sm.m[warp][row] = m[nt][e];
        sm.l[warp][row] = sum;
      }
#pragma unroll
      for (int t = 0; t < 8; t += 2)
        *reinterpret_cast<float4*>(&sm.o[warp][row][16 * g + 2 * t]) =
            make_float4(o[nt][t][e], o[nt][t][2 + e], o[nt][t + 1][e], o[nt][t + 1][2 + e]);
    }
  __syncthreads();
  // a warp per row, four channels per lane
  const int live = min(ROWS, rows);
  const auto write = [&](int row, const float (&acc)[4], float sum) {
    // no key at all: zeros (a NaN sum still divides, and stays NaN)
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float f[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    *reinterpret_cast<uint2*>(p.out + b * p.o_sb + int64_t(row / p.share) * p.o_ss +
                              int64_t(kvh * p.share + row % p.share) * p.o_sh + 4 * lane) = pack4(f);
  };
#pragma unroll 1
  for (int row = warp; row < live; row += kRowsWarps) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) mx = fmaxf(mx, sm.m[w][row]);
    float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float f = sm.m[w][row] == -INFINITY ? 0.0f : ex2_ftz(sm.m[w][row] - mx);
      const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][row][4 * lane]);
      sum = fmaf(sm.l[w][row], f, sum);
      acc[0] = fmaf(x.x, f, acc[0]);
      acc[1] = fmaf(x.y, f, acc[1]);
      acc[2] = fmaf(x.z, f, acc[2]);
      acc[3] = fmaf(x.w, f, acc[3]);
    }
    if (splits == 1) {
      write(row, acc, sum);
      continue;
    }
    if (lane == 0) {
      sm.mm[row] = mx;
      sm.lm[row] = sum;
    }
    *reinterpret_cast<float4*>(&sm.om[row][4 * lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  }
  if (splits == 1) return;
  cluster_sync();
  // ---- join the splits, the rows shared out over the CTAs: lane r (mod 8) holds the
  // numbers of CTA r, and all remote reads of a row are in flight at once (with a
  // thread per row and four channels, reading CTA after CTA, 32 heads over 4229
  // tokens took 0.9 us longer)
#pragma unroll 1
  for (int row = warp * splits + split; row < live; row += kRowsWarps * splits) {
    const int from = lane & 7;
    float m = -INFINITY, l = 0.0f;
    if (from < splits) {
      m = ld_cluster_f32(cluster_map(&sm.mm[row], from));
      l = ld_cluster_f32(cluster_map(&sm.lm[row], from));
    }
    float4 x[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      x[r] = r < splits ? ld_cluster_f32x4(cluster_map(&sm.om[row][4 * lane], r)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float mx = m;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float f = m == -INFINITY ? 0.0f : ex2_ftz(m - mx);
    float sum = l * f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float fr = __shfl_sync(0xffffffffu, f, r);
      acc[0] = fmaf(x[r].x, fr, acc[0]);
      acc[1] = fmaf(x[r].y, fr, acc[1]);
      acc[2] = fmaf(x[r].z, fr, acc[2]);
      acc[3] = fmaf(x[r].w, fr, acc[3]);
    }
    write(row, acc, sum);
  }
  cluster_sync();   // no CTA leaves while another reads its shared memory
}

// The shortest schedule of the keys over clusters of up to eight CTAs, in warp
// steps: the waves of resident clusters, each a warp's share of the steps plus the
// fixed part of a CTA (launch, query, joining), which costs as much as about six
// of them.
struct RowsPlan {
  int64_t cost;
  int splits;
};

template <int NT, int DEPTH>
int plan_rows(int64_t groups, int steps, RowsPlan* plan) {
  constexpr int smem = int(sizeof(RowsSmem<8 * NT, DEPTH>));
  static std::atomic<uint64_t> allowed;
  const int rc = allow_launch("qia_cached_attention", cached_attn_rows_kernel<NT, DEPTH>, smem, &allowed);
  if (rc) return rc;
  static std::atomic<int> resident[17];
  *plan = {INT64_MAX, 1};
  for (int s = 1; s <= 8 && (s == 1 || s <= steps); ++s) {
    const int64_t slots = resident_clusters(cached_attn_rows_kernel<NT, DEPTH>, kRowsWarps * 32, smem, s, resident);
    if (slots == 0) continue;
    const int64_t cost = (groups + slots - 1) / slots * ((steps + s * kRowsWarps - 1) / (s * kRowsWarps) + 6);
    if (cost < plan->cost) *plan = {cost, s};
  }
  return QIA_OK;
}

template <int NT, int DEPTH>
int run_rows(const CachedAttn& p, int batch, int splits, cudaStream_t st) {
  return launch_cluster("cached_attn_rows_kernel", cached_attn_rows_kernel<NT, DEPTH>,
                        dim3(unsigned(splits), unsigned(p.kv_heads), unsigned(batch)), kRowsWarps * 32,
                        sizeof(RowsSmem<8 * NT, DEPTH>), splits, st, p);
}

}  // namespace

// Up to eight rows: with few groups the device is not full, and a warp's own depth
// hides the latency (three CTAs per SM); with many, one more CTA per SM does it
// better. On a B200 (us, deep / shallow): 32 heads of one request, one row, 16384
// tokens 29.2 / 31.6, 333 5.4 / 5.5; sixteen requests of 8 K/V heads, four rows: 333
// 7.6 / 8.1, 4229 31.1 / 30.8, 16384 96.2 / 94.7. More rows leave no registers for
// depth (32 heads, sixteen rows: 1111 tokens 11.7 / 10.9, 16384 44.7 / 42.6).
int launch_cached_rows(const CachedAttn& p, int batch, cudaStream_t st) {
  const int64_t groups = int64_t(p.kv_heads) * batch;
  const int steps = (p.extent + kRowsStep - 1) / kRowsStep + (p.sk + kRowsStep - 1) / kRowsStep;
  RowsPlan deep, wide;
  if (int64_t(p.sq) * p.share > 8) {
    const int rc = plan_rows<2, 1>(groups, steps, &wide);
    return rc ? rc : run_rows<2, 1>(p, batch, wide.splits, st);
  }
  int rc = plan_rows<1, 2>(groups, steps, &deep);
  if (!rc) rc = plan_rows<1, 1>(groups, steps, &wide);
  if (rc) return rc;
  return deep.cost <= wide.cost ? run_rows<1, 2>(p, batch, deep.splits, st) : run_rows<1, 1>(p, batch, wide.splits, st);
}

}  // namespace qia

using namespace qia;

// The rows that share a K/V head fill one 16-row tile. On a B200 (us, this form / the
// larger ones): 32 heads, one request, one row: 16 tokens 4.5 / 10.9, 333 5.4 / 13.0,
// 16384 29.2 / 66; sixteen rows: 16 9.0 / 11.5, 1111 10.9 / 19.1, 16384 42.6 / 66; four
// requests of sixteen rows: 16 9.7 / 15.1, 4229 44.8 / 71.
static bool use_rows(int64_t seq_q, int64_t share) { return seq_q * share <= 16; }

extern "C" int64_t qia_cached_attention_workspace_bytes(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t heads,
                                                        int64_t kv_heads, int64_t extent) {
  if (batch <= 0 || seq_q <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || heads / kv_heads > 128 ||
      use_rows(seq_q, heads / kv_heads) || !cached_use_wide(batch, seq_q, seq_k, kv_heads, heads / kv_heads, extent))
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
  if (use_rows(seq_q, p.share)) return launch_cached_rows(p, int(batch), as_stream(stream));
  if (!cached_use_wide(batch, seq_q, seq_k, kv_heads, p.share, extent)) return launch_cached_tiles(p, int(batch), as_stream(stream));
  return launch_cached_wide(p, int(batch), workspace, as_stream(stream));
}

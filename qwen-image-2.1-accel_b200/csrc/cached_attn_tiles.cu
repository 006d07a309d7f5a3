// Attention of some tens to some hundreds of query rows over the INT8 prefix
// cache (at most two tiles of 128 rows per request and K/V head), on tcgen05.
//
// Roles (512 threads, one CTA per SM):
//   warps 0-3, 4-7  softmax groups 0 and 1 (a query row per thread): scores from
//                   TMEM, weights back into TMEM;
//   warp 8          issues the MMAs;
//   warps 9-15      operand writers: INT8 codes -> bf16 (exact), fresh bf16 rows
//                   copied, into the swizzled shared-memory tiles, and the
//                   per-key numbers of the softmax.
// A key tile is 128 keys. K and V tiles (32 KB each) have two stages. TMEM:
// scores of group i at columns [128 i, +128), its bf16 weights over the first 64
// of them (the A operand of P.V), accumulators at 256 + 128 i. The groups own
// the two query tiles of the CTA and see every key tile, or, when there is only
// one query tile, both work on it with the even and the odd key tiles.
//
// The issuer runs, per softmax group: P(j).V(j), as each half of P(j) is stored,
// then Q.K of the group's next key tile, so while one group's products run, the
// other group's softmax works. MMAs of one thread complete in order: the next
// Q.K may overwrite the scores that hold P(j), and once its scores are there,
// the accumulators hold all of P.V up to j and the softmax may rescale them
// (only when a row's maximum grew by more than 2^8, see cached_attn.cuh).
//
// Both products take the codes themselves; the softmax multiplies scores by
// c log2e ks_j and weights by vs_j in fp32. Tiles whose keys all take part skip
// the mask; fresh ones have no scales and touch no per-key number at all (the
// broadcast reads of those share the shared-memory port with the operands).
//
// INT8 -> bf16: byte b under exponent byte 0x43; x = 128 + (b & 0x7f) and
// c = 128 (b >= 0) or 256 (b < 0, exponent + 1) are bf16 patterns, x - c = b.
//
// Keys may be split over a cluster, which joins through distributed shared
// memory in rank order (no workspace, fixed order). Every wait is bounded (1 s)
// and reports QIA_ERR_TIMEOUT through the device error word.
#include "cached_attn_tc.cuh"

namespace qia {
namespace {

constexpr int kThreads = 512;
constexpr int kWriters = 7;                     // operand-writer warps: arrivals of a written tile
constexpr int kScalarBytes = 3 * 128 * 4;       // [sk | vs | bias][128] f32
constexpr int kSmemML = kSmemTail + kScalarRing * kScalarBytes;   // m, l of 256 rows (joining)
constexpr int kSmemBars = kSmemML + 2 * 256 * 4;
constexpr int kSmemBytes = kSmemBars + 256 + 1024;
// registers of a softmax thread and of any other: 256 x 160 + 256 x 96 = 512 x 128, what the block starts with
constexpr int kSoftmaxRegs = 160, kOtherRegs = 96;
constexpr float kTilesLag = 8.0f;
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);   // B (V) is MN-major
// kinds of a key tile, in the order of what the softmax has to read
constexpr int kFreshFull = 0, kCachedFull = 1, kMasked = 2;

__device__ __forceinline__ void cp_async16_zfill(uint32_t smem, const void* gmem, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// bf16 pair of two codes of `w` (bytes picked by `sel`)
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t w, uint32_t sel) {
  const uint32_t t = __byte_perm(w, 0x43434343u, sel);
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t & 0xff7fff7fu), "r"(t & 0xff80ff80u));
  return r;
}

// The 128 scores of a row in registers -> their maximum, and for tiles with
// per-key numbers also t = s * sk (+ bias) in place.
template <int KIND>
__device__ __forceinline__ float row_scores(uint32_t (&s)[128], const float* scal, float c) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 128; i += 4) {
    if (KIND != kFreshFull) {
      const float4 sk = *reinterpret_cast<const float4*>(scal + i);
      uint64_t t0 = f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
      uint64_t t1 = f2_pack(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
      if (KIND == kMasked) {
        const float4 bias = *reinterpret_cast<const float4*>(scal + 256 + i);
        t0 = f2_fma(t0, f2_pack(sk.x, sk.y), f2_pack(bias.x, bias.y));
        t1 = f2_fma(t1, f2_pack(sk.z, sk.w), f2_pack(bias.z, bias.w));
      } else {
        t0 = f2_mul(t0, f2_pack(sk.x, sk.y));
        t1 = f2_mul(t1, f2_pack(sk.z, sk.w));
      }
      float a, b;
      f2_unpack(t0, a, b);
      s[i] = __float_as_uint(a);
      s[i + 1] = __float_as_uint(b);
      f2_unpack(t1, a, b);
      s[i + 2] = __float_as_uint(a);
      s[i + 3] = __float_as_uint(b);
    }
    mx[(i / 4) & 3] = max3(mx[(i / 4) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    mx[(i / 4 + 2) & 3] = max3(mx[(i / 4 + 2) & 3], __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
  }
  const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
  return KIND == kFreshFull ? top * c : top;
}

// Weights of 64 keys (half h): w = 2^(t - m), their sum into l, and w (times vs
// of cached keys) as bf16 pairs.
template <int KIND>
__device__ __forceinline__ void row_weights(const uint32_t (&s)[128], int h, const float* scal, float c, float neg_m,
                                            uint64_t (&l)[2], uint32_t (&w)[32]) {
  const uint64_t c2 = f2_pack(c, c), n2 = f2_pack(neg_m, neg_m);
#pragma unroll
  for (int k = 0; k < 64; k += 4) {
    const int i = h * 64 + k;
    float4 vs;
    if (KIND != kFreshFull) vs = *reinterpret_cast<const float4*>(scal + 128 + i);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint64_t x = f2_pack(__uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
      float a, b;
      f2_unpack(KIND == kFreshFull ? f2_fma(x, c2, n2) : f2_add(x, n2), a, b);
      a = ex2_ftz(a);
      b = ex2_ftz(b);
      l[e] = f2_add(l[e], f2_pack(a, b));
      if (KIND != kFreshFull) f2_unpack(f2_mul(f2_pack(a, b), e ? f2_pack(vs.z, vs.w) : f2_pack(vs.x, vs.y)), a, b);
      w[k / 2 + e] = cvt_bf16x2(a, b);
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
cached_attn_tiles_kernel(const __grid_constant__ CachedAttn p, const __grid_constant__ TileGrid tp, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBars);
  uint64_t* k_full = bars;            // [2] operand writers -> issuer
  uint64_t* v_full = bars + 2;        // [2]
  uint64_t* k_empty = bars + 4;       // [2] issuer -> operand writers
  uint64_t* v_empty = bars + 6;       // [2]
  uint64_t* scal_full = bars + 8;     // [4] operand writers -> softmax
  uint64_t* s_full = bars + 12;       // [2] scores of group i
  uint64_t* p_full = bars + 14;       // [2][2] weights of group i, half h, stored
  uint64_t* o_full = bars + 18;
  uint64_t* drain = bars + 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int group = tp.first_group + int(blockIdx.x) / splits;
  const int pair = group % tp.pairs, kvh = group / tp.pairs % p.kv_heads, b = group / tp.pairs / p.kv_heads;
  const int n_tiles = min(2, tp.q_tiles - 2 * pair);   // query tiles of this CTA
  const bool duo = n_tiles == 1;                       // the groups share one: even and odd key tiles
  const int len = cached_len(p, b);
  const int cached_tiles = (len + 127) / 128;
  const int all_tiles = cached_tiles + (p.sk + 127) / 128;
  const int per = (all_tiles + splits - 1) / splits;
  const int first = min(all_tiles, split * per), n = min(all_tiles, first + per) - first;   // this CTA's key tiles

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&k_full[i]), kWriters);
      mbar_init(smem_u32(&v_full[i]), kWriters);
      mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&v_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&p_full[i]), 4);
    for (int i = 0; i < kScalarRing; ++i) mbar_init(smem_u32(&scal_full[i]), kWriters);
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(drain), 1);
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(smem_u32(tmem_slot), 512);
  // ---- query tiles (rows past the end are zeros)
  const int tile_rows = tp.tokens_per_tile * p.share;
  for (int i = threadIdx.x; i < n_tiles * kTileRows * 16; i += kThreads) {
    const int tile = i >> 11, row = (i >> 4) & 127, piece = i & 15;
    const int token = (2 * pair + tile) * tp.tokens_per_tile + row / p.share;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row < tile_rows && token < p.sq)
      v = __ldg(reinterpret_cast<const uint4*>(p.q + b * p.q_sb + int64_t(token) * p.q_ss +
                                               int64_t(kvh * p.share + row % p.share) * p.q_sh) + piece);
    st_shared_v4(sbase + kSmemQ + tile * kTileBytes + tile_offset(row, piece), v.x, v.y, v.z, v.w);
  }
  fence_proxy_async_shared();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // key tiles of softmax group w: the it-th is it (both groups), or 2 it + w
  const auto tiles_of = [&](int w) { return duo ? (n - w + 1) / 2 : n; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ------------------------------------------------------------ MMA issuer
      // (warp-uniform control, one elected lane: see cached_attn_wide.cu)
      if (n > 0) {
        const bool lead = elect_one();
        const auto wait = [&](uint64_t* bar, int parity) {
          const bool got = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), uint32_t(parity), err));
          tc_fence_after();
          return got;
        };
        const auto commit = [&](uint64_t* bar) {
          if (lead) tc_commit(smem_u32(bar));
        };
        const auto qk = [&](int w, int j) {
          const uint64_t qd = smem_desc_k_sw128(sbase + kSmemQ + (duo ? 0 : w) * kTileBytes);
          const uint64_t kd = smem_desc_k_sw128(sbase + kSmemKV + (j & 1) * 2 * kTileBytes);
          if (lead) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint64_t off = uint64_t(((kk >> 2) * kPanel + (kk & 3) * 32) >> 4);
              tc_mma_f16_ss(tmem + uint32_t(128 * w), qd + off, kd + off, kIdescS, kk > 0);
            }
            tc_commit(smem_u32(&s_full[w]));
          }
        };
        const auto wait_k = [&](int j) { return wait(&k_full[j & 1], (j >> 1) & 1); };
        // P.V of group w's it-th key tile j, in halves of 64 keys as they are stored
        const auto pv = [&](int w, int it, int j) {
          const uint64_t vd = smem_desc_mn_sw128(sbase + kSmemKV + ((j & 1) * 2 + 1) * kTileBytes, kPanel);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!wait(&p_full[2 * w + h], it & 1)) return false;
            if (lead) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {   // 16 keys: two 8-key groups of 1 KB
                const int kk = 4 * h + k;
                tc_mma_f16_ts(tmem + uint32_t(256 + 128 * w), tmem + uint32_t(128 * w + 8 * kk),
                              vd + uint64_t(128 * kk), kIdescO, kk > 0 || it > 0);
              }
            }
          }
          return true;
        };
        bool ok = true;
        if (duo) {
          for (int j = 0; j < 2 && j < n && ok; ++j) {
            ok = wait_k(j);
            if (ok) qk(j, j);
            if (ok) commit(&k_empty[j]);
          }
          for (int j = 0; j < n && ok; ++j) {
            ok = wait(&v_full[j & 1], (j >> 1) & 1) && pv(j & 1, j >> 1, j);
            if (!ok) break;
            commit(&v_empty[j & 1]);
            if (j + 2 < n) {
              ok = wait_k(j + 2);
              if (!ok) break;
              qk(j & 1, j + 2);
              commit(&k_empty[j & 1]);
            }
          }
        } else {
          ok = wait_k(0);
          if (ok) {
            qk(0, 0);
            qk(1, 0);
            commit(&k_empty[0]);
          }
          for (int j = 0; j < n && ok; ++j) {
            ok = wait(&v_full[j & 1], (j >> 1) & 1);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              ok = ok && pv(w, j, j);
              if (ok && j + 1 < n) {
                ok = w > 0 || wait_k(j + 1);
                if (ok) qk(w, j + 1);
              }
            }
            if (!ok) break;
            commit(&v_empty[j & 1]);
            if (j + 1 < n) commit(&k_empty[(j + 1) & 1]);
          }
        }
        if (ok) commit(o_full);
        commit(drain);
        mbar_wait(smem_u32(drain), 0, ok ? err : nullptr, 100000000ull);
      }
    } else {
      // ------------------------------------------------------- operand writers
      const int t = threadIdx.x - 32 * 9;
      const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
      const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;
      const int cached_n = max(0, min(n, cached_tiles - first));   // cached tiles of this CTA
      // codes of half tile u (2 j: K of tile j, 2 j + 1: V): eight threads per
      // row, 28 rows per step
      constexpr int kSteps = 5;
      const int trow = t >> 3;
      const auto load_codes = [&](int u, uint4 (&c)[kSteps]) {
        const int k0 = (first + (u >> 1)) * 128;
        const int8_t* src = ((u & 1) ? p.vc : p.kc) + head_row * kCaD + (t & 7) * 16;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int key = min(k0 + i * 28 + trow, len - 1);   // (past the length: any held row, weight 0)
          c[i] = __ldg(reinterpret_cast<const uint4*>(src + int64_t(key) * kCaD));
        }
      };
      const auto store_codes = [&](uint32_t slot, const uint4 (&c)[kSteps]) {
        const int piece = (t & 7) * 2;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int row = i * 28 + trow;
          if (row >= kTileRows) break;
          const uint32_t a0 = codes_bf16x2(c[i].x, 0x4140), a1 = codes_bf16x2(c[i].x, 0x4342);
          const uint32_t a2 = codes_bf16x2(c[i].y, 0x4140), a3 = codes_bf16x2(c[i].y, 0x4342);
          const uint32_t b0 = codes_bf16x2(c[i].z, 0x4140), b1 = codes_bf16x2(c[i].z, 0x4342);
          const uint32_t b2 = codes_bf16x2(c[i].w, 0x4140), b3 = codes_bf16x2(c[i].w, 0x4342);
          // the upper four lanes of a row write their second piece first: the
          // eight lanes of a store phase then hit eight different bank groups
          const bool up = t & 4;
          st_shared_v4(slot + tile_offset(row, piece + up), up ? b0 : a0, up ? b1 : a1, up ? b2 : a2, up ? b3 : a3);
          st_shared_v4(slot + tile_offset(row, piece + !up), up ? a0 : b0, up ? a1 : b1, up ? a2 : b2, up ? a3 : b3);
        }
      };
      // the softmax's numbers of key tile j, one key per thread
      float ks = 1.0f, vs = 1.0f;
      bool valid = false;
      const auto load_scalars = [&](int j) {
        const int tile = first + j;
        ks = vs = 1.0f;
        if (tile < cached_tiles) {
          const int key = tile * 128 + t;
          valid = key < len && t < 128;
          if (valid) {
            ks = __ldg(p.ks + head_row + key);
            vs = __ldg(p.vs + head_row + key);
            valid = !mask || __ldg(mask + key) != 0;
          }
        } else {
          const int key = (tile - cached_tiles) * 128 + t;
          valid = key < p.sk && t < 128 && (!mask || __ldg(mask + p.extent + key) != 0);
        }
      };
      const auto store_scalars = [&](int j) {
        if (t < 128) {
          float* dst = reinterpret_cast<float*>(smem + kSmemTail + (j % kScalarRing) * kScalarBytes) + t;
          dst[0] = valid ? p.scale_log2 * ks : 0.0f;
          dst[128] = valid ? vs : 0.0f;
          dst[256] = valid ? 0.0f : -INFINITY;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scal_full[j % kScalarRing]));
      };
      const auto publish = [&](int u) {
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32((u & 1) ? &v_full[(u >> 1) & 1] : &k_full[(u >> 1) & 1]));
      };
      const auto wait_slot = [&](int u) {
        const int j = u >> 1;
        return __all_sync(0xffffffffu, mbar_wait(smem_u32((u & 1) ? &v_empty[j & 1] : &k_empty[j & 1]),
                                                 ((j >> 1) & 1) ^ 1, err));
      };
      uint4 cur[kSteps];
      bool ok = true;
      if (n > 0) load_scalars(0);
      if (cached_n > 0) load_codes(0, cur);
      int u = 0;
      for (; u < 2 * cached_n && ok; ++u) {
        uint4 next[kSteps];
        if (u + 1 < 2 * cached_n) load_codes(u + 1, next);
        const int j = u >> 1;
        ok = wait_slot(u);
        if (!ok) break;
        store_codes(sbase + kSmemKV + uint32_t((j & 1) * 2 + (u & 1)) * kTileBytes, cur);
        publish(u);
        if (!(u & 1)) {
          store_scalars(j);
        } else if (j + 1 < n) {
          load_scalars(j + 1);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) cur[i] = next[i];
      }
      // fresh tiles: bf16 rows copied as they are (masked and missing rows as
      // zeros); a tile is published one step later, when its copies have landed
      bool pending = false;
      for (; u < 2 * n && ok; ++u) {
        const int j = u >> 1, k0 = (first + j - cached_tiles) * 128;
        ok = wait_slot(u);
        if (!ok) break;
        if (pending) {
          cp_async_wait();
          publish(u - 1);
        }
        const uint32_t slot = sbase + kSmemKV + uint32_t((j & 1) * 2 + (u & 1)) * kTileBytes;
        const __nv_bfloat16* src = (u & 1) ? p.v + b * p.v_sb + kvh * p.v_sh : p.k + b * p.k_sb + kvh * p.k_sh;
        const int64_t ss = (u & 1) ? p.v_ss : p.k_ss;
        for (int row = t >> 4; row < kTileRows; row += 14) {
          const int piece = t & 15, key = k0 + row;
          const bool held = key < p.sk && (!mask || __ldg(mask + p.extent + key) != 0);
          cp_async16_zfill(slot + tile_offset(row, piece), src + int64_t(held ? key : 0) * ss + piece * 8, held);
        }
        pending = true;
        if (!(u & 1)) {
          store_scalars(j);
          if (j + 1 < n) load_scalars(j + 1);
        }
      }
      cp_async_wait();
      if (pending && ok) publish(u - 1);
    }
  } else {
    // ----------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + uint32_t(128 * w), t_o = tmem + t_lane + uint32_t(256 + 128 * w);
    const float c = p.scale_log2;
    const int count = tiles_of(w);
    bool ok = true;
    float m = -INFINITY;
    uint64_t l2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
    for (int it = 0; it < count; ++it) {
      const int j = duo ? 2 * it + w : it;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[w]), it & 1, err) &&
                                       mbar_wait(smem_u32(&scal_full[j % kScalarRing]), (j / kScalarRing) & 1, err));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        tc_ld_32x32b_x32(t_s + uint32_t(q * 32), *reinterpret_cast<uint32_t(*)[32]>(&s[q * 32]));
      const float* scal = reinterpret_cast<const float*>(smem + kSmemTail + (j % kScalarRing) * kScalarBytes);
      const int tile = first + j, tail = tile < cached_tiles ? len - tile * 128 : p.sk - (tile - cached_tiles) * 128;
      const int kind = p.key_valid || tail < 128 ? kMasked : tile < cached_tiles ? kCachedFull : kFreshFull;
      tc_wait_ld();
      const float top = kind == kFreshFull    ? row_scores<kFreshFull>(s, scal, c)
                        : kind == kCachedFull ? row_scores<kCachedFull>(s, scal, c)
                                              : row_scores<kMasked>(s, scal, c);
      const bool grow = top > m + kTilesLag;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2_ftz(m - top) : 1.0f;   // (m = -inf: 0)
        if (grow) m = top;
        l2[0] = f2_mul(l2[0], f2_pack(f, f));
        l2[1] = f2_mul(l2[1], f2_pack(f, f));
        if (it > 0) {
#pragma unroll 1
          for (int q = 0; q < 8; ++q) {
            uint32_t o[16];
            tc_ld_32x32b_x16(t_o + uint32_t(q * 16), o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc_st_32x32b_x16(t_o + uint32_t(q * 16), o);
          }
        }
      }
      const float neg_m = m == -INFINITY ? 0.0f : -m;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t x[32];
        if (kind == kFreshFull) row_weights<kFreshFull>(s, h, scal, c, neg_m, l2, x);
        else row_weights<kCachedFull>(s, h, scal, c, neg_m, l2, x);
        tc_st_32x32b_x32(t_s + uint32_t(32 * h), x);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[2 * w + h]));
      }
    }
    float la, lb;
    f2_unpack(f2_add(l2[0], l2[1]), la, lb);
    const float l = la + lb;
    bool have = ok && count > 0;       // the accumulators hold something
    if (ok && n > 0) have = __all_sync(0xffffffffu, mbar_wait(smem_u32(o_full), 0, err)) && have;
    tc_fence_after();
    // ------------------------------------------------------------------ output
    const int row = (warp & 3) * 32 + lane;
    const int token = (2 * pair + w) * tp.tokens_per_tile + row / p.share;
    if (splits == 1 && !duo)
      store_row(t_o, have, l, row < tile_rows && token < p.sq,
                p.out + b * p.o_sb + int64_t(token) * p.o_ss + int64_t(kvh * p.share + row % p.share) * p.o_sh);
    else
      stage_row(t_o, have, m, l, sbase, reinterpret_cast<float*>(smem + kSmemML), w * kTileRows + row);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (splits > 1 || duo)     // (the same in every CTA of a cluster)
    join_rows(p, tp, sbase, sbase + kSmemML, splits, split, duo ? 2 : 1, n_tiles, pair, kvh, b);
}

}  // namespace

int launch_cached_tiles(const CachedAttn& p, int batch, cudaStream_t st) {
  static const bool ready = cudaFuncSetAttribute(cached_attn_tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSmemBytes) == cudaSuccess;
  if (!ready) return set_error(QIA_ERR_CUDA, "qia_cached_attention: cudaFuncSetAttribute failed");
  TileGrid g = tile_grid(p);
  const int64_t groups = int64_t(g.pairs) * p.kv_heads * batch;
  if (groups > 0x0fffffff) return set_error(QIA_ERR_UNSUPPORTED, "qia_cached_attention: too many query rows");
  static std::atomic<int> resident[17];
  return launch_waves(
      groups, (p.extent + 127) / 128 + (p.sk + 127) / 128,
      [&](int s) { return resident_clusters(cached_attn_tiles_kernel, kThreads, kSmemBytes, s, resident); },
      [&](int64_t first, int64_t count, int splits, bool) {
        g.first_group = int(first);
        return launch_cluster("cached_attn_tiles_kernel", cached_attn_tiles_kernel, dim3(unsigned(count * splits)),
                              kThreads, size_t(kSmemBytes), splits, st, p, g, device_error_word());
      });
}

}  // namespace qia

// Attention of many query rows over the INT8 prefix cache: 256 query rows per
// CTA on tcgen05.
//
// Roles (512 threads, one CTA per SM; warps 13-15 only fill the warpgroup):
//   warps 0-3, 4-7  softmax of query tile 0 / 1 (128 rows each, a row per
//                   thread): scores from TMEM, weights back into TMEM;
//   warps 8-11      operand writers: INT8 codes -> bf16 (exact), fresh bf16 rows
//                   copied, into the swizzled shared-memory tiles, and the
//                   three per-key numbers of the softmax;
//   warp 12         issues the MMAs.
// A key tile is 128 keys. K and V tiles (32 KB each) have two stages. TMEM:
// scores of tile i at columns [128 i, +128), its bf16 weights over the first 64
// of them (the A operand of P.V), accumulators at 256 + 128 i.
//
// The issuer runs, for key tile j and query tile i:  P_i(j).V(j), then
// Q_i.K(j+1), so while one tile's products run, the other tile's softmax works.
// MMAs of one thread complete in order: Q_i.K(j+1) may overwrite the scores that
// hold P_i(j), and once the scores of j+1 are there, the accumulators hold all
// of P.V up to j and the softmax may rescale them (only when a row's maximum
// grew by more than 2^8, see cached_attn.cuh).
//
// What bounds it: per key tile and query tile 2 x 512 tensor cycles and 1024
// cycles of exponentials per SM, with 4.5 instructions per score on four
// schedulers close behind; INT8 -> bf16 costs two instructions per code, spread
// over the 256 rows of the CTA.
//
// INT8 -> bf16: byte b under exponent byte 0x43; x = 128 + (b & 0x7f) and
// c = 128 (b >= 0) or 256 (b < 0, exponent + 1) are bf16 patterns, x - c = b.
//
// Keys may be split over a cluster, which joins through distributed shared
// memory in rank order (no workspace, fixed order). Every wait is bounded (1 s)
// and reports QIA_ERR_TIMEOUT through the device error word.
#include "cached_attn.cuh"
#include "cluster.cuh"
#include "sm100.cuh"

namespace qia {
namespace {

constexpr int kTileRows = 128;                 // query rows per tile, keys per tile
constexpr int kTileBytes = kTileRows * kCaD * 2;   // 32 KB: two 64-channel panels of 16 KB
constexpr int kPanel = kTileBytes / 2;
constexpr int kSmemQ = 0;
constexpr int kSmemKV = 2 * kTileBytes;        // stage s: K at 2 s, V at 2 s + 1
constexpr int kScalarRing = 4;
constexpr int kSmemScal = kSmemKV + 4 * kTileBytes;                   // [ring][sk | lsv | rsv][128] f32
constexpr int kSmemML = kSmemScal + kScalarRing * 3 * 128 * 4;        // m, l of 256 rows (cluster join)
constexpr int kSmemBars = kSmemML + 2 * 256 * 4;
constexpr int kTilesSmem = kSmemBars + 256 + 1024;
constexpr int kTilesThreads = 512;   // (a multiple of four warps: the register split below is per warpgroup)
constexpr float kTilesLag = 8.0f;
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);   // B (V) is MN-major

__device__ __forceinline__ void cp_async16_zfill(uint32_t smem, const void* gmem, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// bf16 pair of two codes of `w` (bytes picked by `sel`)
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t w, uint32_t sel) {
  const uint32_t t = __byte_perm(w, 0x43434343u, sel);
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t & 0xff7fff7fu), "r"(t & 0xff80ff80u));
  return r;
}

// Shared-memory offset of 16-byte piece `piece` (0..15) of row `row` in a tile.
__device__ __forceinline__ uint32_t tile_offset(int row, int piece) {
  return uint32_t((piece >> 3) * kPanel + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

struct TilesParams {
  CachedAttn a;
  int tokens_per_tile;   // query tokens in a tile of 128 rows: 128 / share
  int q_tiles;           // tiles of the request
};

__global__ void __launch_bounds__(kTilesThreads, 1)
cached_attn_tiles_kernel(const __grid_constant__ TilesParams tp, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const CachedAttn& p = tp.a;
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBars);
  uint64_t* k_full = bars;            // [2] operand writers -> issuer
  uint64_t* v_full = bars + 2;        // [2]
  uint64_t* k_empty = bars + 4;       // [2] issuer -> operand writers
  uint64_t* v_empty = bars + 6;       // [2]
  uint64_t* scal_full = bars + 8;     // [4] operand writers -> softmax
  uint64_t* s_full = bars + 12;       // [2] scores of query tile i
  uint64_t* p_full = bars + 14;       // [2] weights of query tile i stored
  uint64_t* o_full = bars + 16;
  uint64_t* drain = bars + 17;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int pair = blockIdx.x / splits, kvh = blockIdx.y, b = blockIdx.z;
  const int n_tiles = min(2, tp.q_tiles - 2 * pair);   // query tiles of this CTA
  const int len = cached_len(p, b);
  const int cached_tiles = (len + 127) / 128;
  const int all_tiles = cached_tiles + (p.sk + 127) / 128;
  const int per = (all_tiles + splits - 1) / splits;
  const int first = min(all_tiles, split * per), n = min(all_tiles, first + per) - first;   // this CTA's key tiles

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&k_full[i]), 4);
      mbar_init(smem_u32(&v_full[i]), 4);
      mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&v_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 4);
    }
    for (int i = 0; i < kScalarRing; ++i) mbar_init(smem_u32(&scal_full[i]), 4);
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(drain), 1);
    fence_barrier_init();
  }
  if (warp == 12) tmem_alloc(smem_u32(tmem_slot), 512);
  // ---- query tiles (rows past the end are zeros)
  const int tile_rows = tp.tokens_per_tile * p.share;
  for (int i = threadIdx.x; i < 2 * kTileRows * 16; i += kTilesThreads) {
    const int tile = i >> 11, row = (i >> 4) & 127, piece = i & 15;
    const int token = (2 * pair + tile) * tp.tokens_per_tile + row / p.share;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (tile < n_tiles && row < tile_rows && token < p.sq)
      v = __ldg(reinterpret_cast<const uint4*>(p.q + b * p.q_sb + int64_t(token) * p.q_ss +
                                               int64_t(kvh * p.share + row % p.share) * p.q_sh) + piece);
    st_shared_v4(sbase + kSmemQ + tile * kTileBytes + tile_offset(row, piece), v.x, v.y, v.z, v.w);
  }
  fence_proxy_async_shared();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  float m = -INFINITY, l = 0.0f;
  bool have = false;               // the accumulators hold something
  if (warp >= 12) {
    // -------------------------------------------------------------- MMA issuer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 12 && lane == 0 && n > 0) {
      bool ok = true;
      const auto qk = [&](int i, int j) {
        const uint64_t qd = smem_desc_k_sw128(sbase + kSmemQ + i * kTileBytes);
        const uint64_t kd = smem_desc_k_sw128(sbase + kSmemKV + (j & 1) * 2 * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint64_t off = uint64_t(((kk >> 2) * kPanel + (kk & 3) * 32) >> 4);
          tc_mma_f16_ss(tmem + uint32_t(128 * i), qd + off, kd + off, kIdescS, kk > 0);
        }
        tc_commit(smem_u32(&s_full[i]));
      };
      const auto pv = [&](int i, int j) {
        const uint64_t vd = smem_desc_mn_sw128(sbase + kSmemKV + ((j & 1) * 2 + 1) * kTileBytes, kPanel);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)   // 16 keys: two 8-key groups of 1 KB
          tc_mma_f16_ts(tmem + uint32_t(256 + 128 * i), tmem + uint32_t(128 * i + 8 * kk), vd + uint64_t(128 * kk),
                        kIdescO, (j | kk) != 0);
      };
      ok = mbar_wait(smem_u32(&k_full[0]), 0, err);
      tc_fence_after();
      if (ok) {
        for (int i = 0; i < n_tiles; ++i) qk(i, 0);
        tc_commit(smem_u32(&k_empty[0]));
      }
      for (int j = 0; j < n && ok; ++j) {
        ok = mbar_wait(smem_u32(&v_full[j & 1]), (j >> 1) & 1, err);
        for (int i = 0; i < n_tiles && ok; ++i) {
          ok = mbar_wait(smem_u32(&p_full[i]), j & 1, err);
          if (ok && i == 0 && j + 1 < n) ok = mbar_wait(smem_u32(&k_full[(j + 1) & 1]), ((j + 1) >> 1) & 1, err);
          if (!ok) break;
          tc_fence_after();
          pv(i, j);
          if (j + 1 < n) qk(i, j + 1);
        }
        if (!ok) break;
        tc_commit(smem_u32(&v_empty[j & 1]));
        if (j + 1 < n) tc_commit(smem_u32(&k_empty[(j + 1) & 1]));
      }
      if (ok) tc_commit(smem_u32(o_full));
      tc_commit(smem_u32(drain));
      mbar_wait(smem_u32(drain), 0, ok ? err : nullptr, 100000000ull);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // --------------------------------------------------------- operand writers
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    const int t = threadIdx.x - 256;
    const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
    const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;
    const int cached_n = max(0, min(n, cached_tiles - first));   // cached tiles of this CTA
    // codes of half tile u (2 j: K of tile j, 2 j + 1: V): eight 16-byte pieces, eight threads per row
    const auto load_codes = [&](int u, uint4 (&c)[8]) {
      const int k0 = (first + (u >> 1)) * 128;
      const int8_t* src = ((u & 1) ? p.vc : p.kc) + head_row * kCaD + (t & 7) * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = min(k0 + i * 16 + (t >> 3), len - 1);   // (past the length: any held row, weight 0)
        c[i] = __ldg(reinterpret_cast<const uint4*>(src + int64_t(key) * kCaD));
      }
    };
    const auto load_scalars = [&](int j, float& ks, float& vs, bool& valid) {
      const int tile = first + j;
      ks = vs = 1.0f;
      if (tile < cached_tiles) {
        const int key = tile * 128 + t;
        valid = key < len && (!mask || mask[key] != 0);
        if (key < len) {
          ks = __ldg(p.ks + head_row + key);
          vs = __ldg(p.vs + head_row + key);
        }
      } else {
        const int key = (tile - cached_tiles) * 128 + t;
        valid = key < p.sk && (!mask || mask[p.extent + key] != 0);
      }
    };
    const auto store_scalars = [&](int j, float ks, float vs, bool valid) {
      const KeyScalars k = key_scalars(p, ks, vs, valid);
      float* dst = reinterpret_cast<float*>(smem + kSmemScal) + (j % kScalarRing) * 384 + t;
      dst[0] = k.sk;
      dst[128] = k.lsv;
      dst[256] = k.rsv;
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
    uint4 cur[8];
    float ks = 1.0f, vs = 1.0f;
    bool valid = false, ok = true;
    if (n > 0) load_scalars(0, ks, vs, valid);
    if (cached_n > 0) load_codes(0, cur);
    int u = 0;
    for (; u < 2 * cached_n && ok; ++u) {
      uint4 next[8];
      if (u + 1 < 2 * cached_n) load_codes(u + 1, next);
      const int j = u >> 1;
      ok = wait_slot(u);
      if (!ok) break;
      const uint32_t slot = sbase + kSmemKV + uint32_t((j & 1) * 2 + (u & 1)) * kTileBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 16 + (t >> 3), piece = (t & 7) * 2;
        const uint32_t a0 = codes_bf16x2(cur[i].x, 0x4140), a1 = codes_bf16x2(cur[i].x, 0x4342);
        const uint32_t a2 = codes_bf16x2(cur[i].y, 0x4140), a3 = codes_bf16x2(cur[i].y, 0x4342);
        const uint32_t b0 = codes_bf16x2(cur[i].z, 0x4140), b1 = codes_bf16x2(cur[i].z, 0x4342);
        const uint32_t b2 = codes_bf16x2(cur[i].w, 0x4140), b3 = codes_bf16x2(cur[i].w, 0x4342);
        // the upper four lanes of a row write their second piece first: the
        // eight lanes of a store phase then hit eight different bank groups
        if (t & 4) {
          st_shared_v4(slot + tile_offset(row, piece + 1), b0, b1, b2, b3);
          st_shared_v4(slot + tile_offset(row, piece), a0, a1, a2, a3);
        } else {
          st_shared_v4(slot + tile_offset(row, piece), a0, a1, a2, a3);
          st_shared_v4(slot + tile_offset(row, piece + 1), b0, b1, b2, b3);
        }
      }
      if (!(u & 1)) {
        store_scalars(j, ks, vs, valid);
      } else if (j + 1 < n) {
        load_scalars(j + 1, ks, vs, valid);
      }
      publish(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) cur[i] = next[i];
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
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = i * 8 + (t >> 4), piece = t & 15, key = k0 + row;
        const bool held = key < p.sk && (!mask || mask[p.extent + key] != 0);
        cp_async16_zfill(slot + tile_offset(row, piece), src + int64_t(held ? key : 0) * ss + piece * 8, held);
      }
      pending = true;
      if (!(u & 1)) {
        store_scalars(j, ks, vs, valid);
        if (j + 1 < n) load_scalars(j + 1, ks, vs, valid);
      }
    }
    cp_async_wait();
    if (pending && ok) publish(u - 1);
  } else {
    // ----------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int tile = warp >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + uint32_t(128 * tile), t_o = tmem + t_lane + uint32_t(256 + 128 * tile);
    bool ok = tile < n_tiles;
    uint64_t l0 = f2_pack(0.0f, 0.0f), l1 = l0;
    for (int j = 0; j < n && ok; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[tile]), j & 1, err) &&
                                       mbar_wait(smem_u32(&scal_full[j % kScalarRing]), (j / kScalarRing) & 1, err));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tc_ld_32x32b_x32(t_s + uint32_t(c * 32), *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
      tc_wait_ld();
      const uint32_t scal = sbase + kSmemScal + uint32_t((j % kScalarRing) * 384 * 4);
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int c = 0; c < 128; c += 4) {
        const float4 sk = ld_shared_f4(scal + c * 4), lv = ld_shared_f4(scal + 512 + c * 4);
        float t0, t1, t2, t3;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), f2_pack(sk.x, sk.y),
                         f2_pack(lv.x, lv.y)), t0, t1);
        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), f2_pack(sk.z, sk.w),
                         f2_pack(lv.z, lv.w)), t2, t3);
        mx0 = fmaxf(mx0, fmaxf(t0, t1));
        mx1 = fmaxf(mx1, fmaxf(t2, t3));
        s[c] = __float_as_uint(t0);
        s[c + 1] = __float_as_uint(t1);
        s[c + 2] = __float_as_uint(t2);
        s[c + 3] = __float_as_uint(t3);
      }
      const float top = fmaxf(mx0, mx1);
      const bool grow = top > m + kTilesLag;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2_ftz(m - top) : 1.0f;   // (m = -inf: 0)
        if (grow) m = top;
        l0 = f2_mul(l0, f2_pack(f, f));
        l1 = f2_mul(l1, f2_pack(f, f));
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tc_ld_32x32b_x32(t_o + uint32_t(c * 32), o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc_st_32x32b_x32(t_o + uint32_t(c * 32), o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : -m;
      const uint64_t base2 = f2_pack(base, base);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          const int i = h * 64 + c;
          const float4 rv = ld_shared_f4(scal + 1024 + i * 4);
          float w0, w1, w2, w3;
          f2_unpack(f2_add(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), base2), w0, w1);
          f2_unpack(f2_add(f2_pack(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), base2), w2, w3);
          w0 = ex2_ftz(w0);
          w1 = ex2_ftz(w1);
          w2 = ex2_ftz(w2);
          w3 = ex2_ftz(w3);
          l0 = f2_fma(f2_pack(w0, w1), f2_pack(rv.x, rv.y), l0);
          l1 = f2_fma(f2_pack(w2, w3), f2_pack(rv.z, rv.w), l1);
          w[c / 2] = cvt_bf16x2(w0, w1);
          w[c / 2 + 1] = cvt_bf16x2(w2, w3);
        }
        tc_st_32x32b_x32(t_s + uint32_t(32 * h), w);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_full[tile]));
    }
    float a, c;
    f2_unpack(f2_add(l0, l1), a, c);
    l = a + c;
    have = ok && n > 0;
    if (have) have = __all_sync(0xffffffffu, mbar_wait(smem_u32(o_full), 0, err));
    tc_fence_after();
    // ------------------------------------------------------------------ output
    const int row = (warp & 3) * 32 + lane;
    const int token = (2 * pair + tile) * tp.tokens_per_tile + row / p.share;
    const bool live = tile < n_tiles && row < tile_rows && token < p.sq;
    if (splits == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.o_sb + int64_t(token) * p.o_ss +
                                            int64_t(kvh * p.share + row % p.share) * p.o_sh);
#pragma unroll 1
      for (int c4 = 0; c4 < 4; ++c4) {
        uint32_t o[32];
        if (have) {
          tc_ld_32x32b_x32(t_o + uint32_t(c4 * 32), o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (live) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[q * 8 + e]) * inv;
            dst[c4 * 4 + q] = pack8(f);
          }
        }
      }
    } else if (tile < n_tiles) {
      // this CTA's rows into the K/V stages (every MMA that read them is done),
      // 16-byte pieces swizzled by the row so that a warp's stores spread
      const int r = tile * kTileRows + row;
      float* ml = reinterpret_cast<float*>(smem + kSmemML);
      ml[r] = m;
      ml[256 + r] = l;
#pragma unroll 1
      for (int c4 = 0; c4 < 4; ++c4) {
        uint32_t o[32];
        if (have) {
          tc_ld_32x32b_x32(t_o + uint32_t(c4 * 32), o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
          st_shared_v4(sbase + kSmemKV + r * 512 + (((c4 * 8 + q) ^ (r & 31)) << 4), o[4 * q], o[4 * q + 1],
                       o[4 * q + 2], o[4 * q + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (splits == 1) return;
  cluster_sync();
  // ---- join the splits: (row, four channels) pieces shared out over the CTAs
  const int pieces = n_tiles * kTileRows * 32;
  const uint32_t ml0 = sbase + kSmemML;
  for (int i = split * kTilesThreads + int(threadIdx.x); i < pieces; i += splits * kTilesThreads) {
    const int r = i >> 5, q = i & 31, tile = r >> 7, row = r & 127;
    const int token = (2 * pair + tile) * tp.tokens_per_tile + row / p.share;
    if (row >= tile_rows || token >= p.sq) continue;
    float mx = -INFINITY;
    for (int k = 0; k < splits; ++k) {
      uint32_t peer;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(ml0 + uint32_t(r * 4)), "r"(k));
      mx = fmaxf(mx, ld_cluster_f32(peer));
    }
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < splits; ++k) {
      uint32_t peer, data;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(ml0 + uint32_t(r * 4)), "r"(k));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                   : "=r"(data)
                   : "r"(sbase + kSmemKV + uint32_t(r * 512 + ((q ^ (r & 31)) << 4))), "r"(k));
      const float mk = ld_cluster_f32(peer);
      const float f = mk == -INFINITY ? 0.0f : ex2_ftz(mk - mx);
      sum = fmaf(ld_cluster_f32(peer + 1024), f, sum);
      const float4 x = ld_cluster_f32x4(data);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    *reinterpret_cast<uint2*>(p.out + b * p.o_sb + int64_t(token) * p.o_ss +
                              int64_t(kvh * p.share + row % p.share) * p.o_sh + 4 * q) = pack4(f);
  }
  cluster_sync();
}

}  // namespace

int launch_cached_tiles(const CachedAttn& p, int batch, cudaStream_t st) {
  static const bool ready = cudaFuncSetAttribute(cached_attn_tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kTilesSmem) == cudaSuccess;
  if (!ready) return set_error(QIA_ERR_CUDA, "qia_cached_attention: cudaFuncSetAttribute failed");
  TilesParams tp;
  tp.a = p;
  tp.tokens_per_tile = kTileRows / p.share;
  tp.q_tiles = (p.sq + tp.tokens_per_tile - 1) / tp.tokens_per_tile;
  const int64_t pairs = (tp.q_tiles + 1) / 2;
  const int64_t groups = pairs * p.kv_heads * batch;
  const int tiles = (p.extent + 127) / 128 + (p.sk + 127) / 128;
  // splits of the keys: the count with the shortest schedule, in key tiles --
  // waves of one CTA per SM, each its share of the keys plus the fixed part of
  // a CTA (prologue, epilogue; twice that when it also joins)
  int splits = 1;
  double best = 1e30;
  for (int s = 1; s <= 8 && s <= (tiles > 0 ? tiles : 1); s *= 2) {
    const double waves = double((groups * s + sm_count() - 1) / sm_count());
    const double cost = waves * ((tiles + s - 1) / s + (s == 1 ? 2.0 : 4.0));
    if (cost < best) {
      best = cost;
      splits = s;
    }
  }
  if (pairs * splits > 0x7fffffff) return set_error(QIA_ERR_UNSUPPORTED, "qia_cached_attention: too many query rows");
  return launch_cluster("qia_cached_attention", cached_attn_tiles_kernel,
                        dim3(unsigned(pairs * splits), unsigned(p.kv_heads), unsigned(batch)), kTilesThreads,
                        size_t(kTilesSmem), splits, st, tp, device_error_word());
}

}  // namespace qia

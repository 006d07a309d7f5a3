// Attention of some tens to some hundreds of query rows over the INT8 prefix
// cache (at most two tiles of 128 rows per request and K/V head), on tcgen05,
// converting the codes as it goes: numerics, tiles and joining as in
// cached_attn_tc.cuh.
//
// Roles (512 threads, one CTA per SM):
//   warps 0-3, 4-7  softmax groups 0 and 1 (a query row per thread): scores from
//                   TMEM, weights back into TMEM;
//   warp 8          issues the MMAs;
//   warps 9-15      operand writers: codes and fresh rows -> f16 in the swizzled
//                   shared-memory tiles, and the tiles' numbers.
// A key tile is 128 keys. K and V tiles (32 KB each) have two stages. TMEM:
// scores of group i at columns [128 i, +128), its weights over the first 64 of
// them (the A operand of P.V), accumulators at 256 + 128 i. The groups own the two
// query tiles of the CTA and see every key tile, or, when there is only one query
// tile, both work on it with the even and the odd key tiles.
//
// The issuer runs, per softmax group: P(j).V(j), as each half of P(j) is stored,
// then Q.K of the group's next key tile, so while one group's products run, the
// other group's softmax works. MMAs of one thread complete in order: the next
// Q.K may overwrite the scores that hold P(j), and once its scores are there,
// the accumulators hold all of P.V up to j and the softmax may rescale them.
//
// Keys may be split over a cluster, which joins through distributed shared
// memory in rank order (no workspace, fixed order). Every wait is bounded (1 s)
// and reports QIA_ERR_TIMEOUT through the device error word.
#include "cached_attn_tc.cuh"

namespace qia {
namespace {

constexpr int kThreads = 512;
constexpr int kWriters = 7;                     // operand-writer warps: arrivals of a written tile
constexpr int kSmemQScale = kSmemTail + kScalarRing * kInfoBytes;   // 2^e_i of 256 rows
constexpr int kSmemML = kSmemQScale + 256 * 4;                      // m, l of 256 rows (joining)
constexpr int kSmemFactor = kSmemML + 2 * 256 * 4;                  // [writer][K, V][128] scale 2^-e of a tile's keys
constexpr int kSmemSlots = kSmemFactor + kWriters * 2 * 128 * 4;    // [writer] maxima
constexpr int kSmemStage = kSmemSlots + 64;                         // codes of half a tile in flight
constexpr int kStageBytes = kTileRows * kCaD;
constexpr int kSmemBars = kSmemStage + kStageBytes;
constexpr int kSmemBytes = kSmemBars + 256 + 1024;
// registers of a softmax thread and of any other: 256 x 160 + 256 x 96 = 512 x 128, what the block starts with
constexpr int kSoftmaxRegs = 160, kOtherRegs = 96;

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

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
  uint64_t* info_full = bars + 8;     // [4] first operand writer -> softmax
  uint64_t* s_full = bars + 12;       // [2] scores of group i
  uint64_t* p_full = bars + 14;       // [2][2] weights of group i, half h, stored
  uint64_t* o_full = bars + 18;
  uint64_t* drain = bars + 19;
  uint64_t* q_full = bars + 20;       // softmax -> issuer
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);

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
    for (int i = 0; i < kScalarRing; ++i) mbar_init(smem_u32(&info_full[i]), 1);
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(drain), 1);
    mbar_init(smem_u32(q_full), 8);
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

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
        bool ok = wait(q_full, 0);
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
          ok = ok && wait_k(0);
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
      const int t = threadIdx.x - 32 * 9, writer = warp - 9;
      const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
      const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;
      const int cached_n = max(0, min(n, cached_tiles - first));   // cached tiles of this CTA
      float* factor = reinterpret_cast<float*>(smem + kSmemFactor) + writer * 256;
      // z: 0 K, 1 V. Codes: eight threads per row, 28 rows per step, through
      // pieces of a staging buffer private to the warp, with cp.async: two halves of a
      // tile in flight where the second query tile's space is free, one otherwise.
      // (With plain loads a warp waits for all of its outstanding loads at the
      // first use of any: 5300 cycles per tile.)
      constexpr int kSteps = 5;
      const int trow = t >> 3, depth = duo ? 2 : 1;
      const uint32_t stage = duo ? sbase + kSmemQ + kTileBytes : sbase + kSmemStage;
      const auto issue = [&](int u) {      // half u: K (even) or V of tile u / 2
        if (u < 2 * cached_n) {
          const int k0 = (first + (u >> 1)) * 128;
          const int8_t* src = ((u & 1) ? p.vc : p.kc) + head_row * kCaD + (t & 7) * 16;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int row = i * 28 + trow;
            if (row < kTileRows)   // (past the length: any held row, factor 0)
              cp_async16(stage + uint32_t(duo ? (u & 1) * kStageBytes : 0) + uint32_t(row * kCaD + (t & 7) * 16),
                         src + int64_t(min(k0 + row, len - 1)) * kCaD);
          }
        }
        cp_async_commit();      // (an empty group keeps the count)
      };
      // Eight codes (one 16-byte f16 piece) per thread and row: sixteen threads per
      // row read what their warp staged.
      const auto take_codes = [&](int u, uint2 (&c)[2 * kSteps]) {
        if (duo) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2 * kSteps; ++i) {
          const int row = (i >> 1) * 28 + writer * 4 + (i & 1) * 2 + (lane >> 4);
          const uint32_t at = stage + uint32_t(duo ? (u & 1) * kStageBytes : 0) + uint32_t(row * kCaD + (lane & 15) * 8);
          c[i] = make_uint2(0u, 0u);
          if (row < kTileRows)
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c[i].x), "=r"(c[i].y) : "r"(at) : "memory");
        }
        __syncwarp();
        issue(u + depth);
      };
      const auto slot_of = [&](int j, int z) { return sbase + kSmemKV + uint32_t((j & 1) * 2 + z) * kTileBytes; };
      const auto store_codes = [&](int j, int z, const uint2 (&c)[2 * kSteps]) {
        const uint32_t slot = slot_of(j, z);
#pragma unroll
        for (int i = 0; i < 2 * kSteps; ++i) {
          const int row = (i >> 1) * 28 + writer * 4 + (i & 1) * 2 + (lane >> 4);
          if (row >= kTileRows) break;
          const float a = factor[z * 128 + row];
          const uint2 x = widen4(c[i].x, a), y = widen4(c[i].y, a);
          st_shared_v4(slot + tile_offset(row, lane & 15), x.x, x.y, y.x, y.y);
        }
      };
      const auto publish = [&](int j, int z) {
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(z ? &v_full[j & 1] : &k_full[j & 1]));
      };
      const auto wait_slot = [&](int j, int z) {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(z ? &v_empty[j & 1] : &k_empty[j & 1]), ((j >> 1) & 1) ^ 1, err));
      };
      // (ring slot j % 4: tile j - 4 was done before V of j - 3 left)
      const auto store_info = [&](int j, int e, int f, const uint32_t (&bits)[4]) {
        if (writer == 0 && lane == 0) {
          TileInfo* info = reinterpret_cast<TileInfo*>(smem + kSmemTail + (j % kScalarRing) * kInfoBytes);
          info->c = p.scale_log2 * pow2f(e);
          info->f = float(f);
          info->inv_f = pow2f(-f);
          info->all = (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu;
#pragma unroll
          for (int i = 0; i < 4; ++i) info->valid[i] = bits[i];
          mbar_arrive(smem_u32(&info_full[j % kScalarRing]));
        }
      };
      // ---- cached tiles. Every writer warp keeps the scales of the tile's keys
      // (keys lane + 32 i), so that no writer waits for another.
      float ks[4], vs[4];
      bool valid[4];
      const auto load_scales = [&](int j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (first + j) * 128 + 32 * i + lane;
          ks[i] = __ldg(p.ks + head_row + min(key, len - 1));
          vs[i] = __ldg(p.vs + head_row + min(key, len - 1));
          valid[i] = key < len && (!mask || __ldg(mask + key) != 0);
        }
      };
      uint2 codes[2 * kSteps];
      bool ok = true;
      for (int u = 0; u < depth; ++u) issue(u);
      if (cached_n > 0) load_scales(0);
      int j = 0;
      for (; j < cached_n; ++j) {
        uint32_t mk = 0, mv = 0, bits[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bits[i] = __ballot_sync(0xffffffffu, valid[i]);
          if (!valid[i]) ks[i] = vs[i] = 0.0f;
          mk = max(mk, magnitude(ks[i]));
          mv = max(mv, magnitude(vs[i]));
        }
        const int e = code_exponent(__reduce_max_sync(0xffffffffu, mk), kLowK);
        const int f = code_exponent(__reduce_max_sync(0xffffffffu, mv), kLowV);
        store_info(j, e, f, bits);
        __syncwarp();                        // (the previous tile's factors were read)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          factor[32 * i + lane] = ks[i] * pow2f(-e);
          factor[128 + 32 * i + lane] = vs[i] * pow2f(-f);
        }
        __syncwarp();
        if (j + 1 < cached_n) load_scales(j + 1);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          take_codes(2 * j + z, codes);
          ok = ok && wait_slot(j, z);
          if (ok) {
            store_codes(j, z, codes);
            publish(j, z);
          }
        }
        if (!ok) break;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      // ---- fresh tiles: the exponents come from the rows themselves (sixteen
      // threads per row, 14 rows per step)
      constexpr int kFresh = 10;
      uint32_t* slots = reinterpret_cast<uint32_t*>(smem + kSmemSlots);
      for (; j < n && ok; ++j) {
        const int k0 = (first + j - cached_tiles) * 128, piece = t & 15;
        uint32_t bits[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 32 * i + lane;
          bits[i] = __ballot_sync(0xffffffffu, key < p.sk && (!mask || __ldg(mask + p.extent + key) != 0));
        }
        const auto load_rows = [&](int z, uint4 (&c)[kFresh]) {
          const __nv_bfloat16* src = z ? p.v + b * p.v_sb + kvh * p.v_sh : p.k + b * p.k_sb + kvh * p.k_sh;
          const int64_t ss = z ? p.v_ss : p.k_ss;
#pragma unroll
          for (int i = 0; i < kFresh; ++i) {
            const int row = i * 14 + (t >> 4);
            const uint32_t word = row < 32 ? bits[0] : row < 64 ? bits[1] : row < 96 ? bits[2] : bits[3];
            c[i] = row < kTileRows && ((word >> (row & 31)) & 1)
                       ? __ldg(reinterpret_cast<const uint4*>(src + int64_t(k0 + row) * ss) + piece)
                       : make_uint4(0u, 0u, 0u, 0u);
          }
        };
        const auto exponent = [&](const uint4 (&c)[kFresh], int lo) {
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < kFresh; ++i) m = finite_max8(c[i], m);
          m = __reduce_max_sync(0xffffffffu, m);
          asm volatile("bar.sync 1, 224;" ::: "memory");      // (the slots' last readers are done)
          if (lane == 0) slots[writer] = m;
          asm volatile("bar.sync 1, 224;" ::: "memory");
#pragma unroll
          for (int i = 0; i < kWriters; ++i) m = max(m, slots[i]);
          return tile_exponent(m, lo);
        };
        const auto store_rows = [&](int z, const uint4 (&c)[kFresh], float a) {
          const uint32_t slot = slot_of(j, z);
#pragma unroll
          for (int i = 0; i < kFresh; ++i) {
            const int row = i * 14 + (t >> 4);
            const uint4 h = narrow8(c[i], a);
            if (row < kTileRows) st_shared_v4(slot + tile_offset(row, piece), h.x, h.y, h.z, h.w);
          }
        };
        uint4 c[kFresh];
        load_rows(1, c);
        const int f = exponent(c, kLowV);
        load_rows(0, c);
        const int e = exponent(c, kLowK);
        store_info(j, e, f, bits);
        // (a warp whose wait gives up leaves the others: their named barriers do
        // not depend on it beyond this tile's, which it has passed)
        ok = wait_slot(j, 0);
        if (ok) {
          store_rows(0, c, pow2f(-e));
          publish(j, 0);
          load_rows(1, c);
          ok = wait_slot(j, 1);
        }
        if (ok) {
          store_rows(1, c, pow2f(-f));
          publish(j, 1);
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      for (; j < n; ++j)    // the barriers of tiles that were given up
        if (j >= cached_n)
          for (int i = 0; i < 4; ++i) asm volatile("bar.sync 1, 224;" ::: "memory");
    }
  } else {
    // ----------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + uint32_t(128 * w), t_o = tmem + t_lane + uint32_t(256 + 128 * w);
    const int q_tile = duo ? 0 : w;
    float* scale = reinterpret_cast<float*>(smem + kSmemQScale) + q_tile * kTileRows;
    if (duo) load_queries<256>(p, tp, sbase + kSmemQ, scale, 2 * pair, threadIdx.x, kvh, b, q_full);
    else load_queries<128>(p, tp, sbase + kSmemQ + w * kTileBytes, scale, 2 * pair + w, threadIdx.x & 127, kvh, b, q_full);
    asm volatile("bar.sync 2, 256;" ::: "memory");       // (the rows' scales)
    const float q_up = scale[row];
    const int count = duo ? (n - w + 1) / 2 : n;       // key tiles of this group
    bool ok = true;
    RowState st = {-INFINITY, 0.0f};
    for (int it = 0; it < count; ++it) {
      const int j = duo ? 2 * it + w : it;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[w]), it & 1, err) &&
                                       mbar_wait(smem_u32(&info_full[j % kScalarRing]), (j / kScalarRing) & 1, err));
      if (!ok) break;
      tc_fence_after();
      softmax_tile(t_s, t_o, reinterpret_cast<const TileInfo*>(smem + kSmemTail + (j % kScalarRing) * kInfoBytes), q_up,
                   it == 0, st, &p_full[2 * w], lane);
    }
    bool have = ok && count > 0;       // the accumulators hold something
    if (ok && n > 0) have = __all_sync(0xffffffffu, mbar_wait(smem_u32(o_full), 0, err)) && have;
    tc_fence_after();
    const int token = (2 * pair + w) * tp.tokens_per_tile + row / p.share;
    if (splits == 1 && !duo)
      store_row(t_o, have, st.l, row < tp.tokens_per_tile * p.share && token < p.sq,
                p.out + b * p.o_sb + int64_t(token) * p.o_ss + int64_t(kvh * p.share + row % p.share) * p.o_sh);
    else
      stage_row(t_o, have, st.m, st.l, sbase, reinterpret_cast<float*>(smem + kSmemML), w * kTileRows + row);
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
  static std::atomic<uint64_t> allowed;
  const int rc = allow_launch("qia_cached_attention", cached_attn_tiles_kernel, kSmemBytes, &allowed);
  if (rc) return rc;
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

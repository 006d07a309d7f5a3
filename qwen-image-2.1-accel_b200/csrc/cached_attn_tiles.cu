// Attention of some tens to some hundreds of query rows over the INT8 prefix
// cache (at most two tiles of 128 rows per request and K/V head), on tcgen05,
// converting the codes as it goes: numerics, tiles and joining as in
// cached_attn_tc.cuh.
//
// Roles (896 threads, one CTA per SM):
//   warps 0-3, 4-7  softmax groups 0 and 1 (a query row per thread): scores from
//                   TMEM, weights back into TMEM;
//   warps 8-15, 16-23  operand writers of K and of V: codes and fresh rows -> f16 in
//                   the swizzled shared-memory tiles;
//   warp 24         issues the MMAs;
//   warp 25         copies the codes to shared memory ahead of the writers, 64 keys of
//                   K or V (8 KB, contiguous) per bulk copy;
//   warp 26         the cached tiles' numbers and the factors of their keys.
// A key tile is 128 keys; the fresh tiles come first, converted while the query
// rows load and the first codes are on their way (7000 cycles at the end of a CTA
// otherwise). K and V tiles (32 KB each) have two stages. TMEM:
// scores of group i at columns [128 i, +128), its weights over the first 64 of
// them (the A operand of P.V), accumulators at 256 + 128 i. The groups own the two
// query tiles of the CTA and see every key tile, or, when there is only one query
// tile, both work on it with the even and the odd key tiles (and the second query
// tile's space holds more copies in flight).
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
//
// What bounds it: with one query tile, the writers and the softmax about equally
// (2250 cycles of work per operand tile, 4200 for the softmax of every second key
// tile: 3100 cycles per 128 keys, 2.4 TB/s of codes); with two, the softmax, which
// sees every tile. Both are instruction issue: seven warps per scheduler, nine
// instructions per four codes. Four requests of 77 rows, 32 heads, on a B200: 8192
// cached tokens 117 to 122 us, 1024 25 us, 16 12 us (seven writer warps, each with its own
// copies and factors in unrolled code: 150, 28 and 13 us; eight in one team: 155,
// 30 and 15 us; pieces of the scores read ahead while others are used: 119, 25 and
// 14 us).
#include "cached_attn_tc.cuh"

namespace qia {
namespace {

constexpr int kThreads = 896;
constexpr int kWriters = 8;                     // operand-writer warps of K, and of V: arrivals of a written tile
constexpr int kInfoRing = 8;
constexpr int kUnitKeys = 64, kUnitBytes = kUnitKeys * kCaD;        // codes per bulk copy
constexpr int kUnits = 3, kDuoUnits = kUnits + kTileBytes / kUnitBytes;
constexpr int kSmemQScale = kSmemTail + kInfoRing * kInfoBytes;     // 2^e_i of 256 rows
constexpr int kSmemML = kSmemQScale + 256 * 4;                      // m, l of 256 rows (joining)
constexpr int kSmemFactor = kSmemML + 2 * 256 * 4;                  // [2 tiles][K, V][128] scale 2^-e of a tile's keys
constexpr int kSmemSlots = kSmemFactor + 2 * 256 * 4;               // [2 tiles][K, V][writer] maxima
constexpr int kSmemBars = kSmemSlots + 2 * 2 * kWriters * 4;
constexpr int kBars = 55;
// the TMEM address, read after the setup barrier: nothing that is written from then
// on (the codes in flight) may share its bytes
constexpr int kSmemTmem = kSmemBars + kBars * 8;
constexpr int kSmemStage = kSmemBars + 512;                         // codes in flight
constexpr int kSmemBytes = kSmemStage + kUnits * kUnitBytes + 1024;
static_assert(kSmemTmem + 4 <= kSmemStage, "the TMEM address has a place of its own");
static_assert(kSmemStage % 16 == 0 && kSmemBytes <= 227 * 1024, "shared memory");
// registers of a softmax thread, a writer and any other: 256 x 112 + 512 x 56 + 128 x 48 = 63488 of the
// 896 x 72 that the block starts with
constexpr int kSoftmaxRegs = 112, kWriterRegs = 56, kOtherRegs = 48;
static_assert(256 * kSoftmaxRegs + 512 * kWriterRegs + 128 * kOtherRegs <= kThreads * 72, "register split");

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
  uint64_t* info_full = bars + 40;    // [8] a tile's numbers -> softmax
  uint64_t* s_full = bars + 12;       // [2] scores of group i
  uint64_t* p_full = bars + 14;       // [2][2] weights of group i, half h, stored
  uint64_t* o_full = bars + 18;
  uint64_t* drain = bars + 19;
  uint64_t* q_full = bars + 20;       // softmax -> issuer
  // bulk copies -> operand writers, [7] for K and for V: a parity wait only tells the
  // phase from the one before, so a team's barriers count its own uses of a unit alone
  // (with one barrier per unit, a team could take the other's copy, still on its way,
  // for its own)
  uint64_t* stage_full_k = bars + 21;
  uint64_t* stage_full_v = bars + 48;
  uint64_t* stage_empty = bars + 28;  // [7] operand writers -> bulk copies
  uint64_t* factor_full = bars + 35;  // [2] factors of tile j % 2
  uint64_t* factor_empty = bars + 37; // [2]
  uint64_t* fresh_done = bars + 39;   // K and V writers are past the fresh tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmemTmem);

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
  const int cached_n = max(0, min(n, cached_tiles - first)), fresh_n = n - cached_n;         // tiles 0 .. fresh_n - 1: fresh
  const int64_t head_row = (int64_t(b) * p.kv_heads + kvh) * p.capacity;
  const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb : nullptr;
  const int units = duo ? kDuoUnits : kUnits;
  const auto unit_at = [&](int s) {
    return s < kUnits ? sbase + uint32_t(kSmemStage + s * kUnitBytes)
                      : sbase + uint32_t(kSmemQ + kTileBytes + (s - kUnits) * kUnitBytes);
  };
  // The numbers of tile j that come from K (z = 0) or V, by one thread each. Ring
  // slot j % 8: K of tile j - 1 (for a cached tile, K and V of j - 2) is written, so
  // Q.K of j - 4 was issued, after P.V of j - 6: the softmax has read those of j - 8.
  const auto store_info = [&](int j, int z, int e, const uint32_t (&bits)[4]) {
    TileInfo* info = reinterpret_cast<TileInfo*>(smem + kSmemTail + (j % kInfoRing) * kInfoBytes);
    if (z) {
      info->f = float(e);
      info->inv_f = pow2f(-e);
    } else {
      info->c = p.scale_log2 * pow2f(e);
      info->all = (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu;
#pragma unroll
      for (int i = 0; i < 4; ++i) info->valid[i] = bits[i];
    }
    mbar_arrive(smem_u32(&info_full[j % kInfoRing]));
  };

  if (warp < 8) {
    if (duo) fetch_queries<256>(p, tp, sbase + kSmemQ, 2 * pair, threadIdx.x, kvh, b);
    else fetch_queries<128>(p, tp, sbase + kSmemQ + (warp >> 2) * kTileBytes, 2 * pair + (warp >> 2), threadIdx.x & 127, kvh, b);
  }
  // a barrier per thread (one thread for all of them took a microsecond)
  if (threadIdx.x >= 256 && threadIdx.x < 256 + kBars) {
    const int i = threadIdx.x - 256;
    const int arrivals = i < 4 || (i >= 28 && i < 35) || i == 20 ? kWriters      // k_full, v_full, stage_empty; q_full
                         : i >= 14 && i < 18                     ? 4             // p_full
                         : i == 37 || i == 38                    ? 2 * kWriters  // factor_empty
                         : i >= 39 && i < 48                     ? 2             // fresh_done, info_full
                                                                 : 1;
    mbar_init(smem_u32(&bars[i]), uint32_t(arrivals));
    fence_barrier_init();
  }
  if (warp == 24) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 24) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 24) {
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
    } else if (warp == 25 && lane == 0) {
      // ------------------------------------------------------------ bulk copies
      // (only held rows are read; what the buffer keeps past the length has factor 0)
      int st = 0, u = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (; u < 4 * cached_n; ++u) {          // K, V of tile u / 4 in halves
        ok = mbar_wait(smem_u32(&stage_empty[st]), phase ^ 1, err);
        if (!ok) break;
        const int k0 = (first + (u >> 2)) * kTileRows + (u & 1) * kUnitKeys, rows = max(0, min(len - k0, kUnitKeys));
        const uint32_t full = smem_u32(((u & 2) ? stage_full_v : stage_full_k) + st);
        mbar_arrive_expect_tx(full, uint32_t(rows * kCaD));
        if (rows > 0)
          bulk_load(unit_at(st), ((u & 2) ? p.vc : p.kc) + (head_row + k0) * kCaD, uint32_t(rows * kCaD), full);
        if (++st == units) { st = 0; phase ^= 1; }
      }
      if (!ok)   // let queued copies land before the shared memory is released
        for (int i = max(0, u - units); i < u; ++i) {
          uint32_t uses = 0;                   // of the unit by that team before
          for (int k = i % units; k < i; k += units) uses += ((k ^ i) & 2) == 0;
          mbar_wait(smem_u32(((i & 2) ? stage_full_v : stage_full_k) + i % units), uses & 1, nullptr, 100000000ull);
        }
    } else if (warp == 26) {
      // ---------------------------------------- numbers and factors of cached tiles
      // (keys lane + 32 i; the next tile's scales are requested before this one's are used)
      float* factors = reinterpret_cast<float*>(smem + kSmemFactor);
      float ks[4], vs[4];
      bool valid[4];
      const auto load_scales = [&](int j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (first + j) * kTileRows + 32 * i + lane;
          ks[i] = __ldg(p.ks + head_row + min(key, len - 1));
          vs[i] = __ldg(p.vs + head_row + min(key, len - 1));
          valid[i] = key < len && (!mask || __ldg(mask + key) != 0);
        }
      };
      if (cached_n > 0) load_scales(0);
#pragma unroll 1
      for (int j = 0; j < cached_n; ++j) {
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
        // (the factors of tile j - 2 were used; the ring of numbers is not more than its length ahead)
        bool ok = mbar_wait(smem_u32(&factor_empty[j & 1]), ((j >> 1) & 1) ^ 1, err);
        if (j == 0 && fresh_n > kInfoRing / 2) ok = ok && mbar_wait(smem_u32(fresh_done), 0, err);
        if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          factors[(j & 1) * 256 + 32 * i + lane] = code_factor(ks[i] * pow2f(-e));
          factors[(j & 1) * 256 + 128 + 32 * i + lane] = code_factor(vs[i] * pow2f(-f));
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&factor_full[j & 1]));
          store_info(fresh_n + j, 0, e, bits);
          store_info(fresh_n + j, 1, f, bits);
        }
        if (j + 1 < cached_n) load_scales(j + 1);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // --------------------------------------------------------- operand writers
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWriterRegs));
    const int writer = (warp - 8) & 7, z = (warp - 8) >> 3, t = writer * 32 + lane, piece = lane & 15;   // z: 0 K, 1 V
    uint64_t* full = z ? v_full : k_full;
    uint64_t* empty = z ? v_empty : k_empty;
    const uint32_t slots0 = sbase + uint32_t(kSmemKV + z * kTileBytes);      // tile j in stage j % 2
    const auto publish = [&](int j) {
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&full[j & 1]));
    };
    bool ok = true;
    // ---- fresh tiles: the exponent comes from the rows themselves (sixteen
    // threads per row, 16 rows per step; one named barrier per tile and operand, passed
    // whether or not a wait gave up)
    uint32_t* slots = reinterpret_cast<uint32_t*>(smem + kSmemSlots);
    const __nv_bfloat16* src = z ? p.v + b * p.v_sb + kvh * p.v_sh : p.k + b * p.k_sb + kvh * p.k_sh;
    const int64_t ss = z ? p.v_ss : p.k_ss;
#pragma unroll 1
    for (int j = 0; j < fresh_n; ++j) {
      const int k0 = (first + cached_n + j - cached_tiles) * kTileRows;
      uint32_t bits[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = k0 + 32 * i + lane;
        bits[i] = __ballot_sync(0xffffffffu, key < p.sk && (!mask || __ldg(mask + p.extent + key) != 0));
      }
      uint4 c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 16 + (t >> 4);
        c[i] = (bits[i >> 1] >> (row & 31)) & 1
                   ? __ldg(reinterpret_cast<const uint4*>(src + int64_t(k0 + row) * ss) + piece)
                   : make_uint4(0u, 0u, 0u, 0u);
      }
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = finite_max8(c[i], m);
      m = __reduce_max_sync(0xffffffffu, m);
      // (a slot is written again two tiles on: every writer has read it before the barrier between)
      uint32_t* mine = slots + ((j & 1) * 2 + z) * kWriters;
      if (lane == 0) mine[writer] = m;
      asm volatile("bar.sync %0, 256;" ::"r"(3 + z) : "memory");
#pragma unroll
      for (int i = 0; i < kWriters; ++i) m = max(m, mine[i]);
      const int e = tile_exponent(m, z ? kLowV : kLowK);
      if (ok && t == 0) store_info(j, z, e, bits);
      ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[j & 1]), ((j >> 1) & 1) ^ 1, err));
      if (ok) {
        const uint32_t slot = slots0 + uint32_t((j & 1) * 2 * kTileBytes);
        const float a = pow2f(-e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 x = narrow8(c[i], a);
          st_shared_v4(slot + tile_offset(i * 16 + (t >> 4), piece), x.x, x.y, x.z, x.w);
        }
        publish(j);
      }
    }
    if (fresh_n > 0 && t == 0) mbar_arrive(smem_u32(fresh_done));
    // ---- cached tiles: eight rows per warp and unit, sixteen threads (of eight
    // codes, one 16-byte piece) per row, in a short loop: the instruction cache has to
    // hold it beside the softmax. Its steps are latencies (waits, loads, the proxy
    // fence), which sixteen warps hide.
    const int row0 = 8 * writer + (lane >> 4);
    const uint32_t code_at = uint32_t(row0 * kCaD + piece * 8);
    const float* factors = reinterpret_cast<const float*>(smem + kSmemFactor) + z * 128 + row0;
    uint64_t* stage_full = z ? stage_full_v : stage_full_k;
    int st = 2 * z;
    uint32_t phases = 0;                     // bit st: of the team's next use of that unit
#pragma unroll 1
    for (int u = 0; u < 2 * cached_n; ++u) {
      const int i0 = u >> 1, j = fresh_n + i0, h = u & 1;
      if (h == 0)
        ok = ok && mbar_wait(smem_u32(&factor_full[i0 & 1]), (i0 >> 1) & 1, err) &&
             mbar_wait(smem_u32(&empty[j & 1]), ((j >> 1) & 1) ^ 1, err);
      ok = ok && mbar_wait(smem_u32(&stage_full[st]), (phases >> st) & 1, err);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      phases ^= 1u << st;
      const uint32_t from = unit_at(st) + code_at;
      uint2 codes[4];
      float a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(codes[i].x), "=r"(codes[i].y) : "r"(from + uint32_t(i * 2 * kCaD))
                     : "memory");
        a[i] = factors[(i0 & 1) * 256 + h * kUnitKeys + 2 * i];
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&stage_empty[st]));
        if (h == 1) mbar_arrive(smem_u32(&factor_empty[i0 & 1]));
      }
      const uint32_t slot = slots0 + uint32_t((j & 1) * 2 * kTileBytes + h * kUnitKeys * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float off = widen_offset(a[i]);
        const uint2 x = widen4(codes[i].x, a[i], off), y = widen4(codes[i].y, a[i], off);
        st_shared_v4(slot + tile_offset(row0 + 2 * i, piece), x.x, x.y, y.x, y.y);
      }
      if (h == 1) publish(j);
      st += h ? 3 : 1;                       // (the other operand's units lie between)
      if (st >= units) st -= units;
    }
  } else {
    // ----------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + uint32_t(128 * w), t_o = tmem + t_lane + uint32_t(256 + 128 * w);
    const int q_tile = duo ? 0 : w;
    float* scale = reinterpret_cast<float*>(smem + kSmemQScale) + q_tile * kTileRows;
    if (duo) convert_queries<256>(sbase + kSmemQ, scale, threadIdx.x, q_full);
    else convert_queries<128>(sbase + kSmemQ + w * kTileBytes, scale, threadIdx.x & 127, q_full);
    asm volatile("bar.sync 2, 256;" ::: "memory");       // (the rows' scales)
    const float q_up = scale[row];
    const int count = duo ? (n - w + 1) / 2 : n;       // key tiles of this group
    bool ok = true;
    RowState st = {-INFINITY, 0.0f};
    for (int it = 0; it < count; ++it) {
      const int j = duo ? 2 * it + w : it;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[w]), it & 1, err) &&
                                       mbar_wait(smem_u32(&info_full[j % kInfoRing]), (j / kInfoRing) & 1, err));
      if (!ok) break;
      tc_fence_after();
      softmax_tile<false>(t_s, t_o, reinterpret_cast<const TileInfo*>(smem + kSmemTail + (j % kInfoRing) * kInfoBytes), q_up,
                   it == 0, st, &p_full[2 * w], lane, [] {}, [] {});
    }
    bool have = ok && count > 0;       // the accumulators hold something
    if (ok && n > 0) have = __all_sync(0xffffffffu, mbar_wait(smem_u32(o_full), 0, err)) && have;
    tc_fence_after();
    if (splits == 1 && !duo)
      store_rows(p, tp, sbase + uint32_t(kSmemQ + w * kTileBytes), t_o, have, st.l, 2 * pair + w, row, kvh, b);
    else
      stage_row(t_o, have, st.m, st.l, sbase, reinterpret_cast<float*>(smem + kSmemML), w * kTileRows + row);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 24) {
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

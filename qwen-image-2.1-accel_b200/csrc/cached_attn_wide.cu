// Attention of many query rows over the INT8 prefix cache (more than two query
// tiles per request and K/V head): the keys are widened once, then every group
// of 256 query rows streams them by TMA.
//
// cached_widen_kernel writes, per (request, K/V head), the cached and the fresh
// keys as the f16 rows of cached_attn_tc.cuh and their tiles' numbers. It moves 3
// bytes per code, once, instead of converting the codes again in every CTA.
//
// Roles (384 threads, one CTA per SM): warps 0-3 and 4-7 softmax of the two query
// tiles (a row per thread), warp 8 issues the MMAs, warp 9 the TMA loads. TMEM:
// scores of tile i at columns [128 i, +128), its f16 weights over the first 64 of
// them (the A operand of P.V), accumulators at 256 + 128 i. The issuer runs, per
// query tile: P(j).V(j), as each half of P(j) is stored, then Q.K(j+1), so while
// one tile's products run, the other tile's softmax works. MMAs of one thread
// complete in order: Q.K(j+1) may overwrite the scores that hold P(j), and once
// its scores are there, the accumulators hold all of P.V up to j and the softmax
// may rescale them (only when a row's maximum grew by more than 2^7; f16 weights
// are at most 2^15).
//
// The warps of the two groups that share a scheduler take their exponentials in
// turn: both at once, each runs at half the unit's rate and then both wait for the
// tensor cores (4096 rows over 8325 keys, 32 heads: 559 us without turns on a card
// that took 530 to 547 with them; 528 to 558 over several cards).
//
// What bounds it: the chain scores, softmax, weights, product of each query tile. Per
// key tile and SM the tensor cores need 2050 cycles for both, the exponentials 2048;
// a tile's softmax takes about 2050 and its next scores come some 1300 later (they
// overwrite the weights, so Q.K has to wait for P.V). On a B200, 4096 rows over
// 4229 + 4096 keys, 32 heads: 1.1 PFLOP/s after 37 us of widening. Measured and left
// out: steps of 64 keys with two score buffers in the same columns (products of 64
// keys read the queries twice as often, 777 cycles instead of 514 per 128 keys: 587 us
// at best); an issuer per query tile (613 us without turns, 552 with); a third or a
// quarter of the exponentials as cubics on the FMA pipes (580, 571 us).
#include "cached_attn_tc.cuh"

namespace qia {
namespace {

constexpr int kThreads = 384;
constexpr int kSmemQScale = kSmemTail + kScalarRing * kInfoBytes;   // 2^e_i of 256 rows
constexpr int kSmemML = kSmemQScale + 256 * 4;                      // m, l of 256 rows (joining)
constexpr int kSmemBars = kSmemML + 2 * 256 * 4;
constexpr int kBars = 29;
constexpr int kSmemTmem = kSmemBars + kBars * 8;                    // the TMEM address
constexpr int kSmemBytes = kSmemBars + 256 + 1024;
static_assert(kSmemTmem + 4 <= kSmemBars + 256 && kSmemBytes <= 227 * 1024, "shared memory");
// registers of a softmax thread and of any other: 256 x 208 + 128 x 88 = 384 x 168, what the block starts with
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
struct Widened {
  __half* k;             // [B Hkv, tiles * 128, 128]: cached_cap cached tiles, then the fresh ones
  __half* v;
  TileInfo* info;        // [B Hkv, tiles]
  int cached_cap, tiles;
};

// Maximum of |x| over the block as bits (NaN and infinity above every number); 256 threads.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slots) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = slots[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, slots[i]);
  return m;
}

// One CTA per (tile, K/V head, request).
__global__ void __launch_bounds__(256, 3) cached_widen_kernel(const __grid_constant__ CachedAttn p,
                                                           const __grid_constant__ Widened w) {
  __shared__ float factor[2][128];
  __shared__ uint32_t slots[2][8], valid_bits[4];
  const int tile = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  grid_launch_dependents();
  const bool cached = tile < w.cached_cap;
  const int end = cached ? cached_len(p, b) : p.sk, k0 = (cached ? tile : tile - w.cached_cap) * 128;
  if (k0 >= end) return;
  const int group = b * p.kv_heads + kvh;
  const int64_t head_row = int64_t(group) * p.capacity, out_row = (int64_t(group) * w.tiles + tile) * 128;
  const uint8_t* mask = p.key_valid ? p.key_valid + b * p.mask_sb + (cached ? 0 : p.extent) : nullptr;
  if (t < 128) {
    const bool valid = k0 + t < end && (!mask || __ldg(mask + k0 + t) != 0);
    const uint32_t bits = __ballot_sync(0xffffffffu, valid);
    if ((t & 31) == 0) valid_bits[t >> 5] = bits;
  }
  int e[2];
  if (cached) {
    uint4 c[2][4];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int8_t* src = (z ? p.vc : p.kc) + head_row * kCaD;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = k0 + i * 32 + (t >> 3);
        c[z][i] = key < end ? __ldg(reinterpret_cast<const uint4*>(src + int64_t(key) * kCaD) + (t & 7))
                            : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    // thread t: K's scale of key t, or V's of key t - 128
    const int key = k0 + (t & 127);
    const float s = key < end ? __ldg((t < 128 ? p.ks : p.vs) + head_row + key) : 0.0f;
    __syncthreads();
    const float mine = (valid_bits[(t & 127) >> 5] >> (t & 31)) & 1 ? s : 0.0f;
    const uint32_t mag = magnitude(mine);
    const uint32_t mk = block_max(t < 128 ? mag : 0u, slots[0]), mv = block_max(t < 128 ? 0u : mag, slots[1]);
    e[0] = code_exponent(mk, kLowK);
    e[1] = code_exponent(mv, kLowV);
    factor[t >> 7][t & 127] = code_factor(mine * pow2f(-e[t >> 7]));
    __syncthreads();
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = i * 32 + (t >> 3);
        const float a = factor[z][row], off = widen_offset(a);
        const uint2 x = widen4(c[z][i].x, a, off), y = widen4(c[z][i].y, a, off);
        const uint2 u = widen4(c[z][i].z, a, off), v = widen4(c[z][i].w, a, off);
        st_global_v8((z ? w.v : w.k) + (out_row + row) * kCaD + 16 * (t & 7), make_uint4(x.x, x.y, y.x, y.y),
                     make_uint4(u.x, u.y, v.x, v.y));
      }
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const __nv_bfloat16* src = z ? p.v + b * p.v_sb + kvh * p.v_sh : p.k + b * p.k_sb + kvh * p.k_sh;
      const int64_t ss = z ? p.v_ss : p.k_ss;
      uint4 c[8];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 16 + (t >> 4);
        c[i] = (valid_bits[row >> 5] >> (row & 31)) & 1
                   ? __ldg(reinterpret_cast<const uint4*>(src + int64_t(k0 + row) * ss) + (t & 15))
                   : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) m = finite_max8(c[i], m);
      e[z] = tile_exponent(block_max(m, slots[z]), z ? kLowV : kLowK);
      const float a = pow2f(-e[z]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 16 + (t >> 4);
        reinterpret_cast<uint4*>((z ? w.v : w.k) + (out_row + row) * kCaD)[t & 15] = narrow8(c[i], a);
      }
    }
  }
  if (t == 0) {
    TileInfo info;
    info.c = p.scale_log2 * pow2f(e[0]);
    info.f = float(e[1]);
    info.inv_f = pow2f(-e[1]);
    info.all = (valid_bits[0] & valid_bits[1] & valid_bits[2] & valid_bits[3]) == 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 4; ++i) info.valid[i] = valid_bits[i];
    w.info[int64_t(group) * w.tiles + tile] = info;
  }
}

__global__ void __launch_bounds__(kThreads, 1)
cached_attn_wide_kernel(const __grid_constant__ CachedAttn p, const __grid_constant__ TileGrid tp,
                        const __grid_constant__ Widened wd, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBars);
  uint64_t* k_full = bars;            // [2] TMA -> issuer
  uint64_t* v_full = bars + 2;        // [2]
  uint64_t* k_empty = bars + 4;       // [2] issuer -> TMA
  uint64_t* v_empty = bars + 6;       // [2]
  uint64_t* info_full = bars + 8;     // [4] TMA -> softmax
  uint64_t* s_full = bars + 12;       // [2] scores of query tile i
  uint64_t* p_full = bars + 14;       // [2][2] weights of query tile i, half h, stored
  uint64_t* o_full = bars + 18;
  uint64_t* drain = bars + 19;
  uint64_t* q_full = bars + 20;       // softmax -> issuer
  uint64_t* turn = bars + 21;         // [2][4] warp k of group i takes its exponentials
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmemTmem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), split = int(cluster_rank());
  const int group = tp.first_group + int(blockIdx.x) / splits;
  const int pair = group % tp.pairs, kvh = group / tp.pairs % p.kv_heads, b = group / tp.pairs / p.kv_heads;
  const int n_tiles = min(2, tp.q_tiles - 2 * pair);   // query tiles of this CTA
  const int len = cached_len(p, b);
  const int cached_tiles = (len + 127) / 128;
  const int all_tiles = cached_tiles + (p.sk + 127) / 128;
  const int per = (all_tiles + splits - 1) / splits;
  const int first = min(all_tiles, split * per), n = min(all_tiles, first + per) - first;   // this CTA's key tiles

  if (warp < 4 * n_tiles)
    fetch_queries<128>(p, tp, sbase + kSmemQ + (warp >> 2) * kTileBytes, 2 * pair + (warp >> 2), threadIdx.x & 127, kvh, b);
  if (threadIdx.x == 256) {
    for (int i = 0; i < 12; ++i) mbar_init(smem_u32(&bars[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&s_full[i]), 1);
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&p_full[i]), 4);
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(drain), 1);
    mbar_init(smem_u32(q_full), 4 * n_tiles);
    for (int i = 0; i < 8; ++i) mbar_init(smem_u32(&turn[i]), 1);
    fence_barrier_init();
    if (wd.tiles) {                        // (a call without keys has no maps)
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
  }
  if (warp == 9) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ------------------------------------------------------------ MMA issuer
      // The whole warp runs the schedule and one elected lane issues: with warp-
      // uniform control the descriptors stay in uniform registers (issued from a
      // one-lane branch, a product of 128 x 128 x 128 took 611 cycles, not 512).
      if (n > 0) {
        const bool lead = elect_one();
        const auto wait = [&](uint64_t* bar, int parity) {
          const bool got = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), uint32_t(parity), err));
          tc_fence_after();
          return got;
        };
        const auto qk = [&](int i, int j) {
          const uint64_t qd = smem_desc_k_sw128(sbase + kSmemQ + i * kTileBytes);
          const uint64_t kd = smem_desc_k_sw128(sbase + kSmemKV + (j & 1) * 2 * kTileBytes);
          if (lead) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint64_t off = uint64_t(((kk >> 2) * kPanel + (kk & 3) * 32) >> 4);
              tc_mma_f16_ss(tmem + uint32_t(128 * i), qd + off, kd + off, kIdescS, kk > 0);
            }
            tc_commit(smem_u32(&s_full[i]));
          }
        };
        // half h (64 keys) of P.V of query tile i and key tile j
        const auto pv = [&](int i, int j, int h) {
          const uint64_t vd = smem_desc_mn_sw128(sbase + kSmemKV + ((j & 1) * 2 + 1) * kTileBytes, kPanel);
          if (lead) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {   // 16 keys: two 8-key groups of 1 KB
              const int kk = 4 * h + k;
              tc_mma_f16_ts(tmem + uint32_t(256 + 128 * i), tmem + uint32_t(128 * i + 8 * kk), vd + uint64_t(128 * kk),
                            kIdescO, kk > 0 || j > 0);
            }
          }
        };
        const auto commit = [&](uint64_t* bar) {
          if (lead) tc_commit(smem_u32(bar));
        };
        bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
        if (ok) {
          for (int i = 0; i < n_tiles; ++i) qk(i, 0);
          commit(&k_empty[0]);
        }
        for (int j = 0; j < n && ok; ++j) {
          ok = wait(&v_full[j & 1], (j >> 1) & 1);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (i < n_tiles && ok) {
              ok = wait(&p_full[2 * i], j & 1);
              if (ok) pv(i, j, 0);
              ok = ok && wait(&p_full[2 * i + 1], j & 1);
              if (ok) pv(i, j, 1);
              if (ok && j + 1 < n) {
                ok = i > 0 || wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
                if (ok) qk(i, j + 1);
              }
            }
          }
          if (!ok) break;
          commit(&v_empty[j & 1]);
          if (j + 1 < n) commit(&k_empty[(j + 1) & 1]);
        }
        if (ok) commit(o_full);
        commit(drain);
        mbar_wait(smem_u32(drain), 0, ok ? err : nullptr, 100000000ull);
      }
    } else if (warp == 9 && lane == 0) {
      // ---------------------------------------------------------- TMA producer
      const int64_t bh = int64_t(b) * p.kv_heads + kvh;
      bool ok = true;
      // the keys are widened. A CTA without key tiles waits too: this grid may not end
      // before the one it depends on, since a launch of the remaining groups is
      // ordered behind this grid alone
      grid_wait();
      int issued = 0;
      for (int u = 0; u < 2 * n && ok; ++u) {
        const int j = u >> 1, st = j & 1;
        const int tile = first + j < cached_tiles ? first + j : wd.cached_cap + first + j - cached_tiles;
        if (!(u & 1)) {                      // (ring slot j % 4: tile j - 4 was done before V of j - 3 left)
          const uint32_t bar = smem_u32(&info_full[j % kScalarRing]);
          mbar_arrive_expect_tx(bar, kInfoBytes);
          bulk_load(sbase + kSmemTail + uint32_t(j % kScalarRing) * kInfoBytes, wd.info + bh * wd.tiles + tile,
                    kInfoBytes, bar);
        }
        ok = mbar_wait(smem_u32((u & 1) ? &v_empty[st] : &k_empty[st]), ((j >> 1) & 1) ^ 1, err);
        if (!ok) break;
        const uint32_t bar = smem_u32((u & 1) ? &v_full[st] : &k_full[st]);
        const uint32_t slot = sbase + kSmemKV + uint32_t(st * 2 + (u & 1)) * kTileBytes;
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int h = 0; h < 2; ++h)
          tma_load_2d(slot + uint32_t(h * kPanel), (u & 1) ? &tm_v : &tm_k, bar, h * 64, int((bh * wd.tiles + tile) * 128));
        issued = u + 1;
      }
      if (!ok) {   // let queued copies land before the shared memory is released
        for (int u = max(0, issued - 4); u < issued; ++u)
          mbar_wait(smem_u32((u & 1) ? &v_full[(u >> 1) & 1] : &k_full[(u >> 1) & 1]), (u >> 2) & 1, nullptr,
                    100000000ull);
        for (int j = max(0, (issued + 1) / 2 - kScalarRing); j <= issued / 2; ++j)
          mbar_wait(smem_u32(&info_full[j % kScalarRing]), (j / kScalarRing) & 1, nullptr, 100000000ull);
      }
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + uint32_t(128 * w), t_o = tmem + t_lane + uint32_t(256 + 128 * w);
    float* scale = reinterpret_cast<float*>(smem + kSmemQScale) + w * kTileRows;
    if (w < n_tiles)
      convert_queries<128>(sbase + kSmemQ + w * kTileBytes, scale, threadIdx.x & 127, q_full);
    bool ok = w < n_tiles;
    if (ok) asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");   // (the rows' scales)
    const float q_up = scale[row];
    RowState st = {-INFINITY, 0.0f};
    for (int j = 0; j < n && ok; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[w]), j & 1, err) &&
                                       mbar_wait(smem_u32(&info_full[j % kScalarRing]), (j / kScalarRing) & 1, err));
      if (!ok) break;
      tc_fence_after();
      softmax_tile<true>(t_s, t_o, reinterpret_cast<const TileInfo*>(smem + kSmemTail + (j % kScalarRing) * kInfoBytes), q_up,
                   j == 0, st, &p_full[2 * w], lane,
                   [&] {      // (group 0 first: its first wait is for the phase before the first)
                     if (n_tiles > 1)
                       ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&turn[4 * w + (warp & 3)]), (j & 1) ^ (w ^ 1), err));
                   },
                   [&] {
                     if (n_tiles > 1 && lane == 0) mbar_arrive(smem_u32(&turn[4 * (w ^ 1) + (warp & 3)]));
                   });
    }
    const bool have = ok && n > 0 && __all_sync(0xffffffffu, mbar_wait(smem_u32(o_full), 0, err));
    tc_fence_after();
    if (w < n_tiles) {
      if (splits == 1)
        store_rows(p, tp, sbase + uint32_t(kSmemQ + w * kTileBytes), t_o, have, st.l, 2 * pair + w, row, kvh, b);
      else
        stage_row(t_o, have, st.m, st.l, sbase, reinterpret_cast<float*>(smem + kSmemML), w * kTileRows + row);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (splits > 1) join_rows(p, tp, sbase, sbase + kSmemML, splits, split, 1, n_tiles, pair, kvh, b);
}

PFN_cuTensorMapEncodeTiled_v12000 wide_encode_fn() {
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

// f16 [rows, 128], boxes of 128 rows x 64 channels
int make_rows_map(CUtensorMap* map, const void* base, int64_t rows) {
  auto fn = wide_encode_fn();
  if (!fn) return set_error(QIA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {cuuint64_t(kCaD), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(kCaD * 2)};
  cuuint32_t box[2] = {64u, 128u};
  cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(QIA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
  return QIA_OK;
}

}  // namespace

// Widening once, or converting in every CTA (cached_attn_tiles.cu). From three
// query tiles per request and K/V head on, several CTAs would convert the same keys.
// Up to two, widening costs its bytes (5 per code, against 1) and saves the CTA's
// conversion, so it is for few keys: up to 320 key tiles in all. On a B200 (us, widened /
// in place): 32 heads of one request, 256 rows: 16 + 256 keys (96 tiles) 15.6 / 19.5,
// 1024 + 256 (320) 25.0 / 24.9, 4229 + 256 (1152) 49.4 / 44.2; 8 K/V heads, 40 rows of
// four: 1024 + 40 (72) 16.8 / 19.7, 4229 (280) 26.3 / 30.6, 8192 (520) 35.7 / 39.1; 128
// heads of four requests, 77 rows: 128 + 77 (256) 15.1 / 15.3, 512 (640) 23.6 / 21.5,
// 8192 (8320) 232 / 123.
bool cached_use_wide(int64_t batch, int64_t seq_q, int64_t seq_k, int64_t kv_heads, int64_t share, int64_t extent) {
  const int64_t per = kTileRows / share;
  return (seq_q + per - 1) / per > 2 ||
         batch * kv_heads * ((extent + kTileRows - 1) / kTileRows + (seq_k + kTileRows - 1) / kTileRows) <= 320;
}

int64_t cached_wide_workspace(int64_t batch, int64_t seq_k, int64_t kv_heads, int64_t extent) {
  return batch * kv_heads * ((extent + 127) / 128 + (seq_k + 127) / 128) * (2 * kTileBytes + kInfoBytes);
}

int launch_cached_wide(const CachedAttn& p, int batch, void* workspace, cudaStream_t st) {
  const char* who = "qia_cached_attention";
  static std::atomic<uint64_t> allowed;
  int rc = allow_launch(who, cached_attn_wide_kernel, kSmemBytes, &allowed);
  if (rc) return rc;
  TileGrid g = tile_grid(p);
  const int64_t groups = int64_t(g.pairs) * p.kv_heads * batch, heads = int64_t(batch) * p.kv_heads;
  Widened wd = {};
  wd.cached_cap = (p.extent + 127) / 128;
  wd.tiles = wd.cached_cap + (p.sk + 127) / 128;
  const int64_t rows = heads * wd.tiles * 128;
  if (groups > 0x0fffffff || rows > 0x7fffffff)
    return set_error(QIA_ERR_UNSUPPORTED, "%s: too many rows for one call", who);
  CUtensorMap tm_k = {}, tm_v = {};
  if (wd.tiles) {
    if (!workspace || !aligned(workspace, 128))
      return set_error(QIA_ERR_INVALID, "%s: the workspace is null or misaligned", who);
    wd.k = (__half*)workspace;
    wd.v = wd.k + rows * kCaD;
    wd.info = (TileInfo*)(wd.v + rows * kCaD);
    rc = make_rows_map(&tm_k, wd.k, rows);
    if (!rc) rc = make_rows_map(&tm_v, wd.v, rows);
    if (rc) return rc;
    cached_widen_kernel<<<dim3(unsigned(wd.tiles), unsigned(p.kv_heads), unsigned(batch)), 256, 0, st>>>(p, wd);
    rc = check_launch("cached_widen_kernel");
    if (rc) return rc;
    count_launch();
  }
  static std::atomic<int> resident[17];
  return launch_waves(
      groups, wd.tiles,
      [&](int s) { return resident_clusters(cached_attn_wide_kernel, kThreads, kSmemBytes, s, resident); },
      [&](int64_t first, int64_t count, int splits, bool follows) {
        g.first_group = int(first);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(count * splits));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemBytes;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(splits);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        // the first launch follows the widening: its prologue overlaps it
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = follows && wd.tiles ? 2 : 1;
        const cudaError_t e =
            cudaLaunchKernelEx(&cfg, cached_attn_wide_kernel, p, g, wd, tm_k, tm_v, device_error_word());
        if (e != cudaSuccess) {
          cudaGetLastError();
          return set_error(QIA_ERR_CUDA, "cached_attn_wide_kernel: %s", cudaGetErrorString(e));
        }
        count_launch();
        return int(QIA_OK);
      });
}

}  // namespace qia

// What the two tensor-core forms of the cached attention share: tile layout in
// shared memory, the output of a CTA's rows and their joining over a cluster,
// and the schedule of the query groups. (The kernels: cached_attn_tiles.cu for
// requests of at most two query tiles, cached_attn_wide.cu for larger ones.)
#pragma once

#include <cudaTypedefs.h>

#include <mutex>

#include "cached_attn.cuh"
#include "cluster.cuh"
#include "sm100.cuh"

namespace qia {

constexpr int kTileRows = 128;                     // query rows per tile, keys per tile
constexpr int kTileBytes = kTileRows * kCaD * 2;   // 32 KB: two 64-channel panels of 16 KB
constexpr int kPanel = kTileBytes / 2;
constexpr int kSmemQ = 0;
constexpr int kSmemKV = 2 * kTileBytes;            // stage s: K at 2 s, V at 2 s + 1
constexpr int kSmemTail = kSmemKV + 4 * kTileBytes;
constexpr int kScalarRing = 4;

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Shared-memory offset of 16-byte piece `piece` (0..15) of row `row` in a tile.
__device__ __forceinline__ uint32_t tile_offset(int row, int piece) {
  return uint32_t((piece >> 3) * kPanel + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}

// Query tiles and groups: a tile is 128 / share tokens of all heads that share a
// K/V head; a group is a pair of tiles of one (request, K/V head).
struct TileGrid {
  int tokens_per_tile;
  int q_tiles, pairs;    // tiles of a request, and pairs of them
  int first_group;       // group = (request, K/V head, pair), pairs fastest
};

inline TileGrid tile_grid(const CachedAttn& p) {
  TileGrid g = {};
  g.tokens_per_tile = kTileRows / p.share;
  g.q_tiles = (p.sq + g.tokens_per_tile - 1) / g.tokens_per_tile;
  g.pairs = (g.q_tiles + 1) / 2;
  return g;
}

// A softmax thread's row of accumulators (128 TMEM columns from t_o) / l -> out.
__device__ __forceinline__ void store_row(uint32_t t_o, bool have, float l, bool live, __nv_bfloat16* row) {
  // no key at all: zeros (a NaN sum still divides, and stays NaN)
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint4* dst = reinterpret_cast<uint4*>(row);
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    uint32_t o[32];
    if (have) {
      tc_ld_32x32b_x32(t_o + uint32_t(q * 32), o);
      tc_wait_ld();
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0u;
    }
    if (live) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[h * 8 + e]) * inv;
        dst[q * 4 + h] = pack8(f);
      }
    }
  }
}

// The same row into shared memory for joining: over the K/V stages (every MMA
// that read them is done), 16-byte pieces swizzled by the row so that a warp's
// stores spread; its maximum and sum into `ml` ([256] each).
__device__ __forceinline__ void stage_row(uint32_t t_o, bool have, float m, float l, uint32_t sbase, float* ml, int r) {
  ml[r] = have ? m : -INFINITY;
  ml[256 + r] = have ? l : 0.0f;
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    uint32_t o[32];
    if (have) {
      tc_ld_32x32b_x32(t_o + uint32_t(q * 32), o);
      tc_wait_ld();
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0u;
    }
#pragma unroll
    for (int h = 0; h < 8; ++h)
      st_shared_v4(sbase + kSmemKV + r * 512 + (((q * 8 + h) ^ (r & 31)) << 4), o[4 * h], o[4 * h + 1], o[4 * h + 2],
                   o[4 * h + 3]);
  }
}

// Joins the splits of a cluster and, where `sets` is 2, both groups of one query
// tile (rows r and r + 128): (row, four channels) pieces shared out over the
// CTAs, read through distributed shared memory, added in rank order.
__device__ __forceinline__ void join_rows(const CachedAttn& p, const TileGrid& g, uint32_t sbase, uint32_t ml, int splits,
                                          int split, int sets, int n_tiles, int pair, int kvh, int b) {
  cluster_sync();
  const int tile_rows = g.tokens_per_tile * p.share, pieces = n_tiles * kTileRows * 32;
  for (int i = split * int(blockDim.x) + int(threadIdx.x); i < pieces; i += splits * int(blockDim.x)) {
    const int r = i >> 5, q = i & 31, tile = r >> 7, row = r & 127;
    const int token = (2 * pair + tile) * g.tokens_per_tile + row / p.share;
    if (row >= tile_rows || token >= p.sq) continue;
    float mx = -INFINITY;
    for (int k = 0; k < splits * sets; ++k)
      mx = fmaxf(mx, ld_cluster_f32(cluster_addr(ml + uint32_t((r + k % sets * kTileRows) * 4), k / sets)));
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < splits * sets; ++k) {
      const int rk = r + k % sets * kTileRows;
      const uint32_t at = cluster_addr(ml + uint32_t(rk * 4), k / sets);
      const float mk = ld_cluster_f32(at);
      const float f = mk == -INFINITY ? 0.0f : ex2_ftz(mk - mx);
      sum = fmaf(ld_cluster_f32(at + 1024), f, sum);
      const float4 x = ld_cluster_f32x4(
          cluster_addr(sbase + kSmemKV + uint32_t(rk * 512 + ((q ^ (rk & 31)) << 4)), k / sets));
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

// ----------------------------------------------------------------------- host
// Runs `groups` groups of `tiles` key tiles: whole waves of one CTA per SM
// unsplit; what is left over splits its keys so that it fills the device, when
// that is shorter (in key tiles, with the fixed part of a CTA -- prologue and
// output -- as two, joining as two more). launch(first group, count, splits,
// whether it is the call's first).
template <class Resident, class Launch>
int launch_waves(int64_t groups, int tiles, Resident&& resident, Launch&& launch) {
  const int64_t whole = groups / sm_count() * sm_count();
  const int rest = int(groups - whole);
  int splits = 1;
  const auto cost = [&](int s) { return (tiles + s - 1) / s + (s > 1 ? 4 : 2); };
  for (int s = 2; s <= 8 && s <= tiles && rest > 0; ++s)
    if (rest <= resident(s) && cost(s) < cost(splits)) splits = s;
  if (splits == 1 || whole == 0) return launch(int64_t(0), groups, splits, true);
  const int rc = launch(int64_t(0), whole, 1, true);
  return rc ? rc : launch(whole, int64_t(rest), splits, false);
}

}  // namespace qia

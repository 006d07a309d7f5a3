// What the two tensor-core forms of the cached attention share: tile layout in
// shared memory, the output of a CTA's rows and their joining over a cluster,
// and the schedule of the query groups. (The kernels: cached_attn_tiles.cu for
// requests of at most two query tiles, cached_attn_wide.cu for larger ones.)
#pragma once

#include <cuda_fp16.h>
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

// The numerics of both forms. Keys are f16 rows, each tile of 128 keys scaled by
// powers of two of its own:
//   kw_j = ks_j kc_j 2^-e,  vw_j = vs_j vc_j 2^-f     (masked keys: zeros)
// with the tile's largest |ks|, |vs| just inside 2^14. f16 keeps eleven bits down
// to 2^-28 of that, an eighth of bf16's rounding, and no factor is left per key:
// with x = q_i . kw_j (q_i scaled by a power of two per row),
//   t_ij = x c_i + f,  c_i = c log2e 2^(e + e_i)        log2 of the weight of vw_j
//   w_ij = 2^(t_ij - M_i + 8)
//   o_i  = sum_j w_ij vw_j / sum_tiles 2^-f sum_j w_ij
// so a score costs half a maximum, half a multiply-add, one exponential, half an
// addition and half a conversion, and the softmax reads 32 bytes per tile. (With
// the scales as per-key numbers in shared memory, a step of 256 x 128 scores took
// 5700 cycles instead of 4200: the broadcast reads compete with the MMA operands.)
// The accumulators are rescaled only when a row's maximum grew by more than 2^7
// (f16 weights are at most 2^15).
constexpr float kBias = 8.0f, kLag = 7.0f;
constexpr uint32_t kIdescS = (1u << 4) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);   // f16 x f16 -> f32
constexpr uint32_t kIdescO = kIdescS | (1u << 16);   // B (V) is MN-major

// A tile of 128 keys: the softmax's numbers and which keys take part.
constexpr int kInfoBytes = 32;
struct __align__(16) TileInfo {
  float c, f, inv_f;     // c log2e 2^e, f, 2^-f
  uint32_t all;          // every key takes part
  uint32_t valid[4];
};
static_assert(sizeof(TileInfo) == kInfoBytes, "bulk copy size");

__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A key's factor, kept to 15 bits (2^-15 of the scale, a sixteenth of the f16
// rounding): its products with the offset below and with a code are then exact.
__device__ __forceinline__ float code_factor(float x) {
  return x == x ? __uint_as_float((__float_as_uint(x) + 256u) & 0xfffffe00u) : x;
}

// Four codes (a word of INT8) times a -> four f16: byte u = code + 128 in the
// second byte of 0x47000000 is the float 2^15 + u, and (2^15 + u) a - (2^15 + 128) a
// is one multiply-add.
__device__ __forceinline__ uint2 widen4(uint32_t w, float a, float off) {
  const uint32_t u = w ^ 0x80808080u;
  const uint64_t a2 = f2_pack(a, a), off2 = f2_pack(off, off);
  float x[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t t = f2_pack(__uint_as_float(__byte_perm(u, 0x47000000u, 0x7404 + 0x20 * i)),
                               __uint_as_float(__byte_perm(u, 0x47000000u, 0x7414 + 0x20 * i)));
    f2_unpack(f2_fma(t, a2, off2), x[2 * i], x[2 * i + 1]);
  }
  return make_uint2(cvt_f16x2(x[0], x[1]), cvt_f16x2(x[2], x[3]));
}
__device__ __forceinline__ float widen_offset(float a) { return -32896.0f * a; }

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

// Exponent e with max 2^-e in [2^13, 2^14) for a maximum given as bits; kept in
// a range where c 2^(e + e_i) and 2^+-f stay normal (rows beyond it only lose
// bits: below 2^-44 they no longer matter to a score, above they saturate f16
// to infinity at 2^106). Of INT8 rows: the maximum scale, |code| < 2^7.
__device__ __forceinline__ int tile_exponent(uint32_t bits, int lo) {
  return min(max(int(bits >> 23) - 127 - 13, lo), 90);
}
constexpr int kLowK = -30, kLowV = -90;
__device__ __forceinline__ int code_exponent(uint32_t scale_bits, int lo) { return tile_exponent(scale_bits + (7u << 23), lo); }

// |x| as bits of a number that may set a tile's exponent: a NaN does not.
__device__ __forceinline__ uint32_t magnitude(float x) { return x == x ? __float_as_uint(x) & 0x7fffffffu : 0u; }

// The largest finite magnitude of eight bf16 values.
__device__ __forceinline__ uint32_t finite_max8(const uint4& v, uint32_t m) {
  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t lo = (x[q] << 16) & 0x7fffffffu, hi = x[q] & 0x7fff0000u;
    m = max(m, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
  }
  return m;
}

__device__ __forceinline__ uint4 narrow8(const uint4& v, float a) {   // eight bf16 values times a -> f16
  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
  const uint64_t a2 = f2_pack(a, a);
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_unpack(f2_mul(f2_pack(bf16_lo(x[i]), bf16_hi(x[i])), a2), lo, hi);
    h[i] = cvt_f16x2(lo, hi);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

// Query tiles and groups: a tile is 128 / share tokens of all heads that share a
// K/V head; a group is a pair of tiles of one (request, K/V head).
struct TileGrid {
  int tokens_per_tile;
  int q_tiles, pairs;    // tiles of a request, and pairs of them
  int first_group;       // group = (request, K/V head, pair), pairs fastest
  uint32_t share_inv;    // 2^16 / share rounded up: (row * share_inv) >> 16 = row / share for rows below 128
};

inline TileGrid tile_grid(const CachedAttn& p) {
  TileGrid g = {};
  g.tokens_per_tile = kTileRows / p.share;
  g.q_tiles = (p.sq + g.tokens_per_tile - 1) / g.tokens_per_tile;
  g.pairs = (g.q_tiles + 1) / 2;
  g.share_inv = uint32_t((65536 + p.share - 1) / p.share);
  return g;
}

// A query tile into shared memory as f16, each row scaled by a power of two 2^e_i
// (rows past the end are zeros), by THREADS threads (`t`; sixteen per row), in two
// steps: fetch_queries asks for the rows where they will stay, all at once, before
// the block's barriers and TMEM are set up; convert_queries converts them in place,
// with 2^e_i into scale[128], and announces them on q_full by every warp. Both are
// short loops (with the rows in registers and everything unrolled, a first CTA spent
// up to 16000 cycles here, most of them waiting for its own instructions).
template <int THREADS>
__device__ __forceinline__ void fetch_queries(const CachedAttn& p, const TileGrid& g, uint32_t slot, int tile, int t,
                                              int kvh, int b) {
  constexpr int kRows = THREADS / 16, kLoads = kTileRows / kRows;
  static_assert(kRows % 8 == 0, "the swizzle of a thread's rows is the same");
  const int tile_rows = g.tokens_per_tile * p.share, row0 = t >> 4, piece = t & 15;
  const uint32_t at = slot + tile_offset(row0, piece);
  const __nv_bfloat16* src = p.q + b * p.q_sb + int64_t(kvh * p.share) * p.q_sh + 8 * piece;
#pragma unroll 4
  for (int i = 0; i < kLoads; ++i) {
    const int row = i * kRows + row0, part = int((uint32_t(row) * g.share_inv) >> 16);
    const int token = tile * g.tokens_per_tile + part;
    const bool held = row < tile_rows && token < p.sq;
    const __nv_bfloat16* from = held ? src + int64_t(token) * p.q_ss + int64_t(row - part * p.share) * p.q_sh : p.q;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + uint32_t(i * kRows * 128)), "l"(from),
                 "r"(held ? 16 : 0)
                 : "memory");
  }
}

template <int THREADS>
__device__ __forceinline__ void convert_queries(uint32_t slot, float* scale, int t, uint64_t* q_full) {
  constexpr int kRows = THREADS / 16, kLoads = kTileRows / kRows;
  const int row0 = t >> 4, piece = t & 15;
  const uint32_t at = slot + tile_offset(row0, piece);
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < kLoads; i += 8) {
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v[k].x), "=r"(v[k].y), "=r"(v[k].z), "=r"(v[k].w)
                   : "r"(at + uint32_t((i + k) * kRows * 128))
                   : "memory");
    uint32_t m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m[k] = __vmaxu2(__vmaxu2(abs_bf16x2(v[k].x), abs_bf16x2(v[k].y)), __vmaxu2(abs_bf16x2(v[k].z), abs_bf16x2(v[k].w)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < 8; ++k) m[k] = __vmaxu2(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = min(max(int(max(m[k] & 0xffffu, m[k] >> 16) >> 7) - 127, -80), 120);
      if (piece == 0) scale[(i + k) * kRows + row0] = pow2f(e);
      const uint4 h = narrow8(v[k], pow2f(-e));
      st_shared_v4(at + uint32_t((i + k) * kRows * 128), h.x, h.y, h.z, h.w);
    }
  }
  fence_proxy_async_shared();
  __syncwarp();
  if ((t & 31) == 0) mbar_arrive(smem_u32(q_full));
}

struct RowState {
  float m, l;
};

__device__ __forceinline__ float max_of(const uint32_t (&s)[128]) {
  float mx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(s[i]);
#pragma unroll
  for (int i = 4; i < 124; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
#pragma unroll
  for (int k = 0; k < 2; ++k) mx[k] = max3(mx[k], __uint_as_float(s[124 + 2 * k]), __uint_as_float(s[125 + 2 * k]));
  return fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
}

__device__ __forceinline__ float max_of(const uint32_t (&s)[64]) {
  float mx[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) mx[k] = __uint_as_float(s[k]);
#pragma unroll
  for (int i = 4; i < 60; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
#pragma unroll
  for (int k = 0; k < 2; ++k) mx[k] = max3(mx[k], __uint_as_float(s[60 + 2 * k]), __uint_as_float(s[61 + 2 * k]));
  return fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
}

// 32 keys' scores of a row, those that take no part (clear bits) at -infinity.
__device__ __forceinline__ void drop_keys(uint32_t* s, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!((bits >> i) & 1)) s[i] = 0xff800000u;
}

// 64 scores of a row -> weights 2^(s c + n1), summed into sum[2], as f16 at TMEM column t.
__device__ __forceinline__ void weigh64(const uint32_t* s, float c, float n1, uint64_t (&sum)[2], uint32_t t) {
  const uint64_t c2 = f2_pack(c, c), n2 = f2_pack(n1, n1);
  uint32_t x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a, b;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, n2), a, b);
    a = ex2_ftz(a);
    b = ex2_ftz(b);
    sum[i & 1] = f2_add(sum[i & 1], f2_pack(a, b));
    x[i] = cvt_f16x2(a, b);
  }
  tc_st_32x32b_x32(t, x);
}

// One softmax step of a thread's row: the 128 scores at TMEM column t_s -> f16
// weights over the first 64 columns, each half announced on p_full[h]; `fresh`:
// the row's accumulators (t_o) hold nothing yet. kHold: the scores stay in
// registers between their maximum and their weights (the wide form: 208 registers a
// thread); otherwise they are read twice, 64 at a time, in loops (the form that
// converts codes: its writers need the registers, and the instruction cache has to
// hold three streams).
//
// Keys that take no part have zero rows, so their score is exactly 0 and their
// weight 2^(f - M + 8) changes nothing but the sum: where every row of the warp
// has a positive score -- its maximum is then a key's that takes part -- they cost
// one subtraction per tile (at most 128 times the largest weight: seven bits of
// fp32). Otherwise their scores are set to -infinity (450 cycles a tile more).
// begin() comes before the exponentials, end() after them.
template <bool kHold, class Begin, class End>
__device__ __forceinline__ void softmax_tile(uint32_t t_s, uint32_t t_o, const TileInfo* info, float q_up, bool fresh,
                                             RowState& st, uint64_t* p_full, int lane, Begin&& begin, End&& end) {
  uint32_t s[kHold ? 128 : 64];
  bool drop = false;
  const auto load = [&](int h, uint32_t* dst) {       // 64 scores
    tc_ld_32x32b_x32(t_s + uint32_t(h * 64), *reinterpret_cast<uint32_t(*)[32]>(dst));
    tc_ld_32x32b_x32(t_s + uint32_t(h * 64 + 32), *reinterpret_cast<uint32_t(*)[32]>(dst + 32));
  };
  const auto reload = [&](int h) {
    load(h, s);
    tc_wait_ld();
    if (drop) {
      drop_keys(s, info->valid[2 * h]);
      drop_keys(s + 32, info->valid[2 * h + 1]);
    }
  };
  const auto maximum = [&] {
    float m = -INFINITY;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      reload(h);
      m = fmaxf(m, max_of(*reinterpret_cast<const uint32_t(*)[64]>(s)));
    }
    return m;
  };
  float raw, missing = 0.0f;
  if constexpr (kHold) {
    load(0, s);
    load(1, s + 64);
  }
  const float4 num = *reinterpret_cast<const float4*>(info);
  const float c = num.x * q_up, f = num.y;
  if constexpr (kHold) {
    tc_wait_ld();
    raw = max_of(s);
  } else {
    raw = maximum();
  }
  if (!__float_as_uint(num.w)) {         // some keys take no part
    if (__all_sync(0xffffffffu, raw > 0.0f)) {
      const uint4 bits = *reinterpret_cast<const uint4*>(info->valid);
      missing = float(128 - __popc(bits.x) - __popc(bits.y) - __popc(bits.z) - __popc(bits.w));
    } else if constexpr (kHold) {
#pragma unroll
      for (int q = 0; q < 4; ++q) drop_keys(s + 32 * q, info->valid[q]);
      raw = max_of(s);
    } else {
      drop = true;
      raw = maximum();
    }
  }
  const float top = fmaf(raw, c, f);
  const bool grow = top > st.m + kLag;
  if (__any_sync(0xffffffffu, grow)) {
    const float r = grow ? ex2_ftz(st.m - top) : 1.0f;   // (m = -inf: 0)
    if (grow) st.m = top;
    st.l *= r;
    if (!fresh) {
#pragma unroll 1
      for (int q = 0; q < 8; ++q) {
        uint32_t o[16];
        tc_ld_32x32b_x16(t_o + uint32_t(q * 16), o);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * r);
        tc_st_32x32b_x16(t_o + uint32_t(q * 16), o);
      }
    }
  }
  const float n1 = f + kBias - (st.m == -INFINITY ? 0.0f : st.m);
  uint64_t sum[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
  begin();
#pragma unroll(kHold ? 2 : 1)
  for (int h = 0; h < 2; ++h) {
    if constexpr (!kHold) reload(h);
    weigh64(kHold ? s + 64 * h : s, c, n1, sum, t_s + uint32_t(32 * h));
    if (h == 1) end();
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&p_full[h]));
  }
  float a, b;
  f2_unpack(f2_add(sum[0], sum[1]), a, b);
  a += b;
  // (only there: 2^n1 is at most 2^15 beside a positive score, infinite far below zero)
  if (missing > 0.0f) a = fmaf(-missing, ex2_ftz(n1), a);
  st.l = fmaf(a, num.z, st.l);
}

// A softmax warp's 32 rows of accumulators (a row per thread, 128 TMEM columns from
// t_o) / l -> out, by way of the query tile's space (every MMA that read it is
// done), so that a store instruction writes two whole rows (a row per thread, 16
// bytes of 32 rows at once, took 6800 cycles).
__device__ __forceinline__ void store_rows(const CachedAttn& p, const TileGrid& g, uint32_t slot, uint32_t t_o, bool have,
                                           float l, int tile, int row, int kvh, int b) {
  // no key at all: zeros (a NaN sum still divides, and stays NaN)
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
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
    for (int h = 0; h < 4; ++h) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[h * 8 + e]) * inv;
      const uint4 v = pack8(f);
      st_shared_v4(slot + uint32_t(row * 256 + (((q * 4 + h) ^ (row & 15)) << 4)), v.x, v.y, v.z, v.w);
    }
  }
  __syncwarp();
  const int lane = row & 31, piece = lane & 15;
  __nv_bfloat16* out = p.out + b * p.o_sb + int64_t(kvh * p.share) * p.o_sh + 8 * piece;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = (row & ~31) + 2 * i + (lane >> 4), part = int((uint32_t(r) * g.share_inv) >> 16);
    const int token = tile * g.tokens_per_tile + part;
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(slot + uint32_t(r * 256 + ((piece ^ (r & 15)) << 4)))
                 : "memory");
    if (r < g.tokens_per_tile * p.share && token < p.sq)
      *reinterpret_cast<uint4*>(out + int64_t(token) * p.o_ss + int64_t(r - part * p.share) * p.o_sh) = v;
  }
}

// A softmax thread's row into shared memory for joining: over the K/V stages (every MMA
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
// tile (rows r and r + 128), the rows in turn to the CTAs: the parts' maxima and
// sums into a table in the query tiles' space, all remote reads at once; the parts'
// factors, a thread per row; then a warp per row, in a fixed order. What bounds it
// is distributed shared memory, 14 bytes per cycle and SM: about 7000 cycles for two
// query tiles over four CTAs.
__device__ __forceinline__ void join_rows(const CachedAttn& p, const TileGrid& g, uint32_t sbase, uint32_t ml, int splits,
                                          int split, int sets, int n_tiles, int pair, int kvh, int b) {
  cluster_sync();
  float* table = static_cast<float*>(__cvta_shared_to_generic(sbase + kSmemQ));   // [m, l][part][row of this CTA]
  const int rows = n_tiles * kTileRows, parts = splits * sets, second = sets - 1;
  for (int i = threadIdx.x; i < parts * 256; i += blockDim.x) {
    const int k = i >> 8, r = (i & 255) * splits + split;
    if (r >= rows) continue;
    const uint32_t at = cluster_addr(ml + uint32_t((r + (k & second) * kTileRows) * 4), k >> second);
    table[i] = ld_cluster_f32(at);
    table[4096 + i] = ld_cluster_f32(at + 1024);
  }
  __syncthreads();
  for (int i = threadIdx.x; i * splits + split < rows; i += blockDim.x) {
    float mx = -INFINITY, sum = 0.0f;
    for (int k = 0; k < parts; ++k) mx = fmaxf(mx, table[k * 256 + i]);
    for (int k = 0; k < parts; ++k) {
      const float m = table[k * 256 + i], f = m == -INFINITY ? 0.0f : ex2_ftz(m - mx);
      sum = fmaf(table[4096 + k * 256 + i], f, sum);
      table[k * 256 + i] = f;
    }
    table[4096 + i] = sum == 0.0f ? 0.0f : 1.0f / sum;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;       // four channels
  __nv_bfloat16* out = p.out + b * p.o_sb + int64_t(kvh * p.share) * p.o_sh + 4 * lane;
#pragma unroll 1
  for (int i = threadIdx.x >> 5; i * splits + split < rows; i += blockDim.x >> 5) {
    const int r = i * splits + split, row = r & 127, part = int((uint32_t(row) * g.share_inv) >> 16);
    const int token = (2 * pair + (r >> 7)) * g.tokens_per_tile + part;
    if (row >= g.tokens_per_tile * p.share || token >= p.sq) continue;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const int rk = r + (k & second) * kTileRows;
      const float4 x =
          ld_cluster_f32x4(cluster_addr(sbase + kSmemKV + uint32_t(rk * 512 + ((lane ^ (rk & 31)) << 4)), k >> second));
      const float f = table[k * 256 + i];
      acc[0] = fmaf(x.x, f, acc[0]);
      acc[1] = fmaf(x.y, f, acc[1]);
      acc[2] = fmaf(x.z, f, acc[2]);
      acc[3] = fmaf(x.w, f, acc[3]);
    }
    const float inv = table[4096 + i];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    *reinterpret_cast<uint2*>(out + int64_t(token) * p.o_ss + int64_t(row - part * p.share) * p.o_sh) = pack4(acc);
  }
  if (splits > 1) cluster_sync();   // no CTA leaves while another reads its shared memory
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

// The INT8 prefix cache: K/V rows quantised as they are written, and cached
// rows read back to bf16.
//
// A row is one token of one head, x[0..127]. With a = max|x|:
//   scale = a / 127,  code_d = rint(x_d * (127 / a))  in [-127, 127]
// (both divides IEEE; an all-zero row has scale 0 and zero codes; a row that
// holds a NaN or an infinity has scale NaN, so reading it back gives NaN). The
// row reads back as bf16(code_d * scale).
//
// Layout: codes [batch, kv_heads, capacity, 128] int8 and scales [batch,
// kv_heads, capacity] f32, head-major, so that an attention CTA streams the
// tokens of its head as one contiguous run. The bf16 rows are token-major
// ([batch, seq, heads, 128], any 16-byte aligned strides).
//
// Both kernels only move bytes (3 per element and direction plus 4 per row); their
// instructions have to stay out of the way (no integer conversions, one divide
// per row). One row is 16 lanes x 16 bytes on the bf16 side, so every access is a
// whole line. A CTA takes 16 tokens of 8 heads (write) or 32 of 4 (read): the
// scales of a head go out in runs of 64 bytes, and a thread has eight (four) rows
// in flight. Two prefixes of 8325 tokens, 32 heads, on a B200: written in 62 us
// (6.7 TB/s; 67 us with 4 heads per CTA, 82 with 2), read back in 65 us (6.4 TB/s;
// 82 us with 16-byte stores).
#include "qia_common.cuh"

namespace qia {
namespace {

constexpr int kKvD = 128;
constexpr int kWriteHeads = 8, kReadHeads = 4;   // heads per CTA
constexpr int kWriteTok = 16;    // tokens per CTA of the write kernel (one per half-warp)
constexpr int kReadTok = 32;     // tokens per CTA of the read kernel (one per 8 lanes)

struct KvCache {
  int8_t* codes[2];   // K, V
  float* scales[2];
  int* lengths;       // tokens held per request
  int capacity, heads;
};

struct KvRows {
  __nv_bfloat16* x[2];
  int64_t sb[2], ss[2], sh[2];
};

// Rows [0, seq) of every request go to tokens [start, start + seq), start the
// request's length when `append`. Tokens past the capacity are dropped and
// recorded in the device error word. The lengths are updated by CTA 0 (fixed
// start: nobody reads them) or by the CTA that finishes last (append: every
// CTA has read its start before it takes a ticket).
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvRows src, const __grid_constant__ KvCache c, int batch, int seq, int start,
                                                       int append, unsigned* ticket, int* err) {
  const int h0 = blockIdx.x * kWriteHeads, b = blockIdx.z >> 1, which = blockIdx.z & 1;
  const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int s = blockIdx.y * kWriteTok + half;
  const int first = append ? *reinterpret_cast<volatile const int*>(c.lengths + b) : start;
  const int t = first + s;
  const bool held = s < seq && first >= 0 && t < c.capacity;
  if (s < seq && !held && lane == 0 && err) atomicExch(err, QIA_ERR_INVALID);
  const __nv_bfloat16* x = src.x[which] + b * src.sb[which] + int64_t(s) * src.ss[which];
  uint4 v[kWriteHeads];
#pragma unroll
  for (int i = 0; i < kWriteHeads; ++i)
    v[i] = held && h0 + i < c.heads ? __ldg(reinterpret_cast<const uint4*>(x + (h0 + i) * src.sh[which]) + lane)
                                    : make_uint4(0u, 0u, 0u, 0u);
  // max of |x| on pairs of bf16 patterns: NaN and infinity compare above every
  // number; lane i of the sixteen keeps row i's and does its two divides
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kWriteHeads; ++i) {
    uint32_t m = __vmaxu2(__vmaxu2(abs_bf16x2(v[i].x), abs_bf16x2(v[i].y)), __vmaxu2(abs_bf16x2(v[i].z), abs_bf16x2(v[i].w)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == i) top = m;
  }
  const uint32_t bits = max(top << 16, top & 0xffff0000u);
  const bool finite = bits < 0x7f800000u;
  // (127 / amax overflows below amax = 2^-121: bounded, so that 0 * inv stays 0;
  // a row that is not finite gets zero codes and the scale NaN)
  const float my_inv = finite && bits ? fminf(__fdiv_rn(127.0f, __uint_as_float(bits)), 3.402823466e38f) : 0.0f;
  const int64_t row0 = (int64_t(b) * c.heads + h0) * c.capacity + t;
  if (lane < kWriteHeads && held && h0 + lane < c.heads)
    c.scales[which][row0 + int64_t(lane) * c.capacity] =
        finite ? __fdiv_rn(__uint_as_float(bits), 127.0f) : __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int i = 0; i < kWriteHeads; ++i) {
    const float inv = __shfl_sync(0xffffffffu, my_inv, i, 16);
    const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    const uint64_t magic = f2_pack(12582912.0f, 12582912.0f);
    uint32_t w[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // x * inv rounded to the nearest integer (|x * inv| <= 127 and a rounding)
      // in the low byte of x * inv + 1.5 2^23 (scalar products: a packed pair of
      // them would be contracted with the addition into one rounding)
      float y[4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        f2_unpack(f2_add(f2_pack(__fmul_rn(bf16_lo(u[2 * q + e]), inv), __fmul_rn(bf16_hi(u[2 * q + e]), inv)), magic),
                  y[2 * e], y[2 * e + 1]);
      w[q] = __byte_perm(__byte_perm(__float_as_uint(y[0]), __float_as_uint(y[1]), 0x0040),
                         __byte_perm(__float_as_uint(y[2]), __float_as_uint(y[3]), 0x0040), 0x5410);
    }
    if (inv == 0.0f) w[0] = w[1] = 0u;     // (an infinity times 0)
    if (held && h0 + i < c.heads)
      reinterpret_cast<uint2*>(c.codes[which] + (row0 + int64_t(i) * c.capacity) * kKvD)[lane] = make_uint2(w[0], w[1]);
  }
  if (!append) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
      for (int i = threadIdx.x; i < batch; i += blockDim.x) c.lengths[i] = min(start + seq, c.capacity);
    return;
  }
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned total = gridDim.x * gridDim.y * gridDim.z;
    last = atomicAdd(ticket, 1u) == total - 1;
  }
  __syncthreads();
  if (last) {
    for (int i = threadIdx.x; i < batch; i += blockDim.x)
      c.lengths[i] = min(*reinterpret_cast<volatile int*>(c.lengths + i) + seq, c.capacity);
    if (threadIdx.x == 0) *ticket = 0;
  }
}

// Tokens [first, first + n) of every request to bf16 rows [0, n); rows past a
// request's length are zeros.
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvCache c, const __grid_constant__ KvRows dst, int first, int n,
                                                      bool wide) {
  const int h0 = blockIdx.x * kReadHeads, b = blockIdx.z >> 1, which = blockIdx.z & 1;
  const int s = blockIdx.y * kReadTok + (threadIdx.x >> 3), lane = threadIdx.x & 7;
  if (s >= n) return;
  const int t = first + s;
  const bool held = t < min(__ldg(c.lengths + b), c.capacity);
  uint4 v[kReadHeads];
  float sc[kReadHeads];
#pragma unroll
  for (int i = 0; i < kReadHeads; ++i) {
    const int64_t row = (int64_t(b) * c.heads + h0 + i) * c.capacity + t;
    const bool have = held && h0 + i < c.heads;
    v[i] = have ? __ldg(reinterpret_cast<const uint4*>(c.codes[which] + row * kKvD) + lane) : make_uint4(0u, 0u, 0u, 0u);
    sc[i] = have ? __ldg(c.scales[which] + row) : 0.0f;
  }
  __nv_bfloat16* x = dst.x[which] + b * dst.sb[which] + int64_t(s) * dst.ss[which];
#pragma unroll
  for (int i = 0; i < kReadHeads; ++i) {
    if (h0 + i >= c.heads) break;
    // byte u = code + 128 under 0x4B0000 is the float 2^23 + u (an integer
    // conversion per code would be the bound, at a sixteenth of the issue rate)
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    const uint64_t off = f2_pack(-8388736.0f, -8388736.0f), sc2 = f2_pack(sc[i], sc[i]);
    float f[16];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const uint32_t u = w[e >> 2] ^ 0x80808080u;
      const uint64_t code = f2_add(f2_pack(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + (e & 3))),
                                           __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7541 + (e & 3)))), off);
      f2_unpack(f2_mul(code, sc2), f[e], f[e + 1]);
    }
    uint4* out = reinterpret_cast<uint4*>(x + (h0 + i) * dst.sh[which]) + 2 * lane;
    if (wide) {
      st_global_v8(out, pack8(f), pack8(f + 8));
    } else {
      out[0] = pack8(f);
      out[1] = pack8(f + 8);
    }
  }
}

int check_cache(const char* who, const void* kc, const void* vc, const void* ks, const void* vs, const void* lengths,
                int64_t batch, int64_t seq, int64_t heads, int64_t capacity, int64_t head_dim) {
  if (!kc || !vc || !ks || !vs || !lengths) return set_error(QIA_ERR_INVALID, "%s: null pointer", who);
  if (head_dim != kKvD) return set_error(QIA_ERR_UNSUPPORTED, "%s: head_dim=%lld (only 128)", who, (long long)head_dim);
  if (batch <= 0 || heads <= 0 || capacity <= 0 || seq < 0)
    return set_error(QIA_ERR_INVALID, "%s: batch=%lld seq=%lld heads=%lld capacity=%lld", who, (long long)batch,
                     (long long)seq, (long long)heads, (long long)capacity);
  if (batch > 32767 || heads > 65536 || capacity > (1 << 30) || seq > 1000000)
    return set_error(QIA_ERR_UNSUPPORTED, "%s: batch=%lld seq=%lld heads=%lld capacity=%lld", who, (long long)batch,
                     (long long)seq, (long long)heads, (long long)capacity);
  if (!aligned(kc, 16) || !aligned(vc, 16) || !aligned(ks, 4) || !aligned(vs, 4) || !aligned(lengths, 4))
    return set_error(QIA_ERR_ALIGNMENT, "%s: misaligned pointer", who);
  return QIA_OK;
}

int make_rows(KvRows* r, const char* who, const void* k, const void* v, const int64_t* st) {
  if (!k || !v || !st) return set_error(QIA_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16)) return set_error(QIA_ERR_ALIGNMENT, "%s: misaligned rows", who);
  for (int i = 0; i < 6; ++i)
    if (st[i] % 8) return set_error(QIA_ERR_ALIGNMENT, "%s: stride %lld is not a multiple of 8", who, (long long)st[i]);
  r->x[0] = (__nv_bfloat16*)k;
  r->x[1] = (__nv_bfloat16*)v;
  for (int i = 0; i < 2; ++i) {
    r->sb[i] = st[3 * i];
    r->ss[i] = st[3 * i + 1];
    r->sh[i] = st[3 * i + 2];
  }
  return QIA_OK;
}

KvCache make_cache(void* kc, void* vc, void* ks, void* vs, void* lengths, int64_t capacity, int64_t heads) {
  KvCache c;
  c.codes[0] = (int8_t*)kc;
  c.codes[1] = (int8_t*)vc;
  c.scales[0] = (float*)ks;
  c.scales[1] = (float*)vs;
  c.lengths = (int*)lengths;
  c.capacity = int(capacity);
  c.heads = int(heads);
  return c;
}

}  // namespace
}  // namespace qia

using namespace qia;

extern "C" int qia_kv_cache_write(const void* k, const void* v, void* k_codes, void* v_codes, void* k_scales,
                                  void* v_scales, void* lengths, int64_t batch, int64_t seq, int64_t heads,
                                  int64_t head_dim, int64_t capacity, int64_t start, const int64_t* strides,
                                  void* ticket, void* stream) {
  const char* who = "qia_kv_cache_write";
  int rc = check_cache(who, k_codes, v_codes, k_scales, v_scales, lengths, batch, seq, heads, capacity, head_dim);
  if (rc) return rc;
  const bool append = start < 0;
  if (append && !ticket) return set_error(QIA_ERR_INVALID, "%s: an append needs a ticket word", who);
  if (!append && start > capacity - seq)
    return set_error(QIA_ERR_INVALID, "%s: tokens %lld+%lld exceed the capacity %lld", who, (long long)start,
                     (long long)seq, (long long)capacity);
  if (seq == 0 && append) return QIA_OK;
  KvRows rows = {};
  rc = seq ? make_rows(&rows, who, k, v, strides) : QIA_OK;   // (no rows: only the lengths are set)
  if (rc) return rc;
  const int64_t tiles = seq ? (seq + kWriteTok - 1) / kWriteTok : 1;
  const dim3 grid(unsigned((heads + kWriteHeads - 1) / kWriteHeads), unsigned(tiles), unsigned(2 * batch));
  kv_write_kernel<<<grid, 256, 0, as_stream(stream)>>>(
      rows, make_cache(k_codes, v_codes, k_scales, v_scales, lengths, capacity, heads), int(batch), int(seq),
      append ? 0 : int(start), append, (unsigned*)ticket, device_error_word());
  rc = check_launch(who);
  if (!rc) count_launch();
  return rc;
}

extern "C" int qia_kv_cache_read(const void* k_codes, const void* v_codes, const void* k_scales, const void* v_scales,
                                 const void* lengths, void* k, void* v, int64_t batch, int64_t first, int64_t tokens,
                                 int64_t heads, int64_t head_dim, int64_t capacity, const int64_t* strides,
                                 void* stream) {
  const char* who = "qia_kv_cache_read";
  int rc = check_cache(who, k_codes, v_codes, k_scales, v_scales, lengths, batch, tokens, heads, capacity, head_dim);
  if (rc) return rc;
  if (first < 0 || first > capacity - tokens)
    return set_error(QIA_ERR_INVALID, "%s: tokens %lld+%lld of capacity %lld", who, (long long)first,
                     (long long)tokens, (long long)capacity);
  if (tokens == 0) return QIA_OK;
  KvRows rows;
  rc = make_rows(&rows, who, k, v, strides);
  if (rc) return rc;
  // whole 32-byte sectors per store where the rows allow it
  bool wide = aligned(k, 32) && aligned(v, 32);
  for (int i = 0; i < 6; ++i) wide = wide && strides[i] % 16 == 0;
  const dim3 grid(unsigned((heads + kReadHeads - 1) / kReadHeads), unsigned((tokens + kReadTok - 1) / kReadTok),
                  unsigned(2 * batch));
  kv_read_kernel<<<grid, 256, 0, as_stream(stream)>>>(
      make_cache((void*)k_codes, (void*)v_codes, (void*)k_scales, (void*)v_scales, (void*)lengths, capacity, heads),
      rows, int(first), int(tokens), wide);
  rc = check_launch(who);
  if (!rc) count_launch();
  return rc;
}

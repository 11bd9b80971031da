// kvquant.hip -- rows of keys and values into a cache of 8 bits, and back.
//
// A row of one KV head (head_dim entries x) is held as int8 entries and one f32 scale: with a = max |x|,
// scale = a / 127 and entry = x / scale, each rounded to nearest once (the entry to a whole number, from the
// quotient rounded to f32); it reads back as entry * scale. A row of zeros has scale 0; a row with a non-finite entry has
// scale NaN and entries 0, so that it reads back as NaN and reaches the outputs that see it, and no others.
//
// G lanes share a row, eight entries each (8 bytes of the cache a lane: a row of 256 is written by half a wave in one
// piece); the largest magnitude is taken over the bit patterns, where infinities and NaN come out on top. Bound by
// the rows' bytes for prompts and by the launch and two trips to memory for one token. Measured, 4 KV heads of 256: one token
// written and read back 6.7 to 8.3 us (kernels 2.4 and 1.9); 4 prompts, 12287 bf16 rows inside q, k, v rows, written and
// read back as f32 47.5 us: 19.2 (76 MB: 4.0 TB/s; by divisions instead of kvq_four 24.2) and 21.5 (126 MB: 5.9 TB/s); 16
// caches of 8192 rows read back as bf16 144 us (810 MB: 5.6 TB/s; a large copy 4.6); 77 rows of 8 heads of 128 read back
// 3.8 to 4.1 us.
#include "rbt_device.h"
#include "rbt_internal.h"

namespace rbt {

__device__ __forceinline__ float kvq_ld(const void *p, long i, int b16) {
  return b16 ? rbt_bf16_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

__device__ __forceinline__ int kvq_entry(float x, float scale) {
  const float r = rintf(__fdiv_rn(x, scale));
  return (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// Four entries, packed, where the scale lies in [2^-60, 2^60] and r = 1 / scale rounded to nearest: x r is within two steps
// of the quotient, the first correction by its remainder (which an fma gives exactly) brings it within one, and
// the second one rounds it as a division would (Markstein 1990). A quotient whose remainder underflows is below
// 2^-40, an entry of 0 either way. Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves its
// last eight bits in the sum's; |x / scale| <= 127 (1 + 2^-23), so nothing has to be cut.
__device__ __forceinline__ uint32_t kvq_four(const float *x, float scale, float r) {
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    float q = x[e] * r;
    q = fmaf(fmaf(-q, scale, x[e]), r, q);
    q = fmaf(fmaf(-q, scale, x[e]), r, q);
    o[e] = __float_as_uint(q + 12582912.0f);
  }
  const uint32_t lo = __builtin_amdgcn_perm(o[1], o[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(o[3], o[2], 0x04000c0cu);
  return lo | hi;
}

// What a row's largest magnitude (as bits) makes of it: the scale, and whether its entries are to be formed.
__device__ __forceinline__ bool kvq_scale(uint32_t top, float &scale) {
  const bool finite = top < 0x7f800000u;
  scale = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __uint_as_float(0x7fc00000u);
  return finite && scale > 0.0f;
}

// The workgroup's sequence: rows n from row `at` of the cache on; false where its numbers do not fit.
__device__ __forceinline__ bool kvq_fits(const KvqArgs &a, int b, int &n, int &at) {
  n = a.n_rows ? a.n_rows[b] : a.T;
  at = a.len ? a.len[b] : 0;
  if (n >= 0 && n <= a.T && at >= 0 && at <= a.cap - n) return true;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.bad = 1;
  return false;
}

// grid (workgroups of a sequence, sequences). A unit is a row of one head and side; `per` units at a time.
template <bool VEC>
__global__ __launch_bounds__(256) void k_kv_quant(KvqArgs a, int G) {
  const int b = blockIdx.y, gl = threadIdx.x % G, gr = threadIdx.x / G, per = 256 / G;
  int n, at;
  if (!kvq_fits(a, b, n, at)) return;
  const long units = 2L * n * a.K;
  for (long u = (long)blockIdx.x * per + gr; u < units; u += (long)gridDim.x * per) {
    const int side = u >= (long)n * a.K;
    const unsigned r = (unsigned)(u - (side ? (long)n * a.K : 0)), j = r / a.K, h = r - j * a.K;
    const void *src = side ? a.v : a.k;
    const long so = b * a.seq + j * a.row + h * a.head, to = (((long)b * a.cap + at + j) * a.K + h);
    int8_t *dst = (side ? a.vc : a.kc) + to * a.hd;
    float *sc = (side ? a.vs : a.ks) + to;
    uint32_t top = 0;
    float scale;
    if constexpr (VEC) {
      float x[8];
      const bool in = 8 * gl < a.hd;
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = 0.0f;
      if (in && a.x16) {
        const rbt_u4 v = *(const rbt_u4 *)((const uint16_t *)src + so + 8 * gl);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[2 * e] = __uint_as_float(v[e] << 16);
          x[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
        }
      } else if (in) {
        const float4 v = *(const float4 *)((const float *)src + so + 8 * gl);
        const float4 w = *(const float4 *)((const float *)src + so + 8 * gl + 4);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      for (int d = 1; d < G; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
      const bool form = kvq_scale(top, scale);
      uint32_t o[2] = {0, 0};
      if (form && scale >= 0x1p-60f && scale <= 0x1p60f) {
        const float r = __fdiv_rn(1.0f, scale);
        o[0] = kvq_four(x, scale, r);
        o[1] = kvq_four(x + 4, scale, r);
      } else if (form) {
#pragma unroll
        for (int e = 0; e < 8; e++) o[e >> 2] |= ((uint32_t)kvq_entry(x[e], scale) & 0xffu) << (8 * (e & 3));
      }
      if (in) *(uint2 *)(dst + 8 * gl) = make_uint2(o[0], o[1]);
    } else {
      for (int i = gl; i < a.hd; i += G) top = max(top, __float_as_uint(kvq_ld(src, so + i, a.x16)) & 0x7fffffffu);
      for (int d = 1; d < G; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
      const bool form = kvq_scale(top, scale);
      for (int i = gl; i < a.hd; i += G) dst[i] = form ? (int8_t)kvq_entry(kvq_ld(src, so + i, a.x16), scale) : 0;
    }
    if (gl == 0) *sc = scale;
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void k_kv_dequant(KvqArgs a, int G) {
  const int b = blockIdx.y, gl = threadIdx.x % G, gr = threadIdx.x / G, per = 256 / G;
  int n, at;
  if (!kvq_fits(a, b, n, at)) return;
  const long units = 2L * n * a.K;
  for (long u = (long)blockIdx.x * per + gr; u < units; u += (long)gridDim.x * per) {
    const int side = u >= (long)n * a.K;
    const unsigned r = (unsigned)(u - (side ? (long)n * a.K : 0)), j = r / a.K, h = r - j * a.K;
    const long from = (((long)b * a.cap + at + j) * a.K + h), to = b * a.seq + j * a.row + h * a.head;
    const int8_t *src = (side ? a.vc : a.kc) + from * a.hd;
    const float scale = (side ? a.vs : a.ks)[from];
    void *dst = side ? a.vo : a.ko;
    if constexpr (VEC) {
      if (8 * gl >= a.hd) continue;
      const uint2 v = *(const uint2 *)(src + 8 * gl);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = (float)(int8_t)((e < 4 ? v.x : v.y) >> (8 * (e & 3))) * scale;
      if (a.x16) {
        rbt_u4 o;
#pragma unroll
        for (int e = 0; e < 4; e++)
          o[e] = (uint32_t)rbt_f32_bf16(x[2 * e]) | (uint32_t)rbt_f32_bf16(x[2 * e + 1]) << 16;
        *(rbt_u4 *)((uint16_t *)dst + to + 8 * gl) = o;
      } else {
        *(float4 *)((float *)dst + to + 8 * gl) = make_float4(x[0], x[1], x[2], x[3]);
        *(float4 *)((float *)dst + to + 8 * gl + 4) = make_float4(x[4], x[5], x[6], x[7]);
      }
    } else {
      for (int i = gl; i < a.hd; i += G) {
        const float x = (float)src[i] * scale;
        if (a.x16)
          ((uint16_t *)dst)[to + i] = rbt_f32_bf16(x);
        else
          ((float *)dst)[to + i] = x;
      }
    }
  }
}

hipError_t launch_kvq(const Ctx &c, const KvqArgs &a, int B, bool read) {
  // whole eights of entries at aligned places: 16-byte loads of the rows, 8-byte ones of the cache
  const int xs = a.x16 ? 2 : 4;
  const void *x[2] = {read ? a.ko : (void *)a.k, read ? a.vo : (void *)a.v};
  bool vec = a.hd % 8 == 0 && a.hd <= 512 && (a.seq | a.row | a.head) * xs % 16 == 0 &&
             (((uintptr_t)a.kc | (uintptr_t)a.vc) & 7) == 0 && (((uintptr_t)x[0] | (uintptr_t)x[1]) & 15) == 0;
  const int lanes = vec ? a.hd / 8 : a.hd;
  int G = 1;
  while (G < lanes && G < 64) G *= 2;
  const int per = 256 / G;
  const long units = 2L * a.T * a.K;
  const long want = std::max(1L, 32L * c.num_cu / B);
  const dim3 grid((unsigned)std::min((units + per - 1) / per, want), B);
  if (read)
    launch_k(c, vec ? k_kv_dequant<true> : k_kv_dequant<false>, grid, dim3(256), a, G);
  else
    launch_k(c, vec ? k_kv_quant<true> : k_kv_quant<false>, grid, dim3(256), a, G);
  return hipGetLastError();
}

}  // namespace rbt

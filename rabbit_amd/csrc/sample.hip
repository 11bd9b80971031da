// sample.hip -- tokens and probabilities from logits: temperature, top-k, top-p, min-p, one draw.
//
// With m the largest logit, w_i = exp((x_i - m) / t). The entries' order is by `ord`, 64 bits: the logit's bits turned so
// that larger ones come first, then the index. top-k, top-p and min-p each keep a run from the front of the order, so
// what is kept are the entries up to one `ord`, found digit by digit.
//
// Weights are summed in whole numbers of 2^-S (S = 62 less the vocabulary's bits, at most 45): such sums do not depend on
// their order or on how the row was split, so equal calls give equal tokens, and a draw differs from one in real numbers
// only where u is within 2^-S times the number of entries of a border. (Sums in fp32 would move every border by 1e-7.)
#include "rbt_device.h"
#include "rbt_internal.h"

namespace rbt {

typedef unsigned long long u64;

// A logit's bits, larger logits first; NaN counts as -inf, and -0 as 0.
__device__ __forceinline__ uint32_t smp_key(float x) {
  if (!(x > -INFINITY)) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float smp_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu);
}

struct SmpRow {
  const void *x;
  int x16, V, S;  // 2^S units in a weight of 1
  double m, inv_t, min_p;
  __device__ __forceinline__ float at(int i) const {
    return x16 ? rbt_bf16_f32(((const uint16_t *)x)[i]) : ((const float *)x)[i];
  }
};

// exp(y), y <= 0: 2^(k/32) from a table times a Taylor polynomial of what is left (at most ln 2 / 64: the seventh
// term is below 2^-52).
__device__ __forceinline__ void smp_table(double *tab) {
  if (threadIdx.x < 32) tab[threadIdx.x] = exp2((double)threadIdx.x * 0.03125);
}
__device__ __forceinline__ double smp_exp(double y, const double *tab) {
  if (!(y > -690.0)) return 0.0;
  const double k = rint(y * 46.16624130844683);
  const double r = fma(k, -7.247021293269686e-19, fma(k, -0.02166084939249829, y));
  const int n = (int)k;
  double p = fma(r, 1.0 / 720.0, 1.0 / 120.0);
  p = fma(r, p, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return ldexp(tab[n & 31] * p, n >> 5);
}
__device__ __forceinline__ double smp_weight(const SmpRow &r, float x, const double *tab) {
  return smp_exp(((double)x - r.m) * r.inv_t, tab);
}
// in units of 2^-S, to the nearest (w <= 1, S <= 45)
__device__ __forceinline__ u64 smp_mass(const SmpRow &r, double w) {
  return (u64)__double_as_longlong(ldexp(w, r.S) + 0x1p52) & 0xfffffffffffffull;
}

struct SmpSet {  // a row's settings
  int k;
  double t, top_p, min_p, u;
};
__device__ __forceinline__ bool smp_set(const SampleArgs &a, int r, SmpSet &s) {
  const float t = a.temp ? a.temp[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f, q = a.min_p ? a.min_p[r] : 0.0f, u = a.u[r];
  s.k = a.top_k ? a.top_k[r] : 0;
  s.t = t;
  s.top_p = p;
  s.min_p = q;
  s.u = u;
  const bool ok = t >= 0.0f && t < INFINITY && s.k >= 0 && p >= 0.0f && p <= 1.0f && q >= 0.0f && q <= 1.0f && u >= 0.0f && u < 1.0f;
  if (t == 0.0f) {  // greedy: the first of the order
    s.k = 1;
    s.t = 1.0;
  }
  return ok;
}

__device__ __forceinline__ uint32_t smp_wave_min(uint32_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = min(v, (uint32_t)__shfl_xor((int)v, d, 64));
  return v;
}
__device__ __forceinline__ u64 smp_wave_sum(u64 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += (u64)__shfl_xor((long long)v, d, 64);
  return v;
}
__device__ __forceinline__ u64 smp_wave_scan(u64 v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 x = (u64)__shfl_up((long long)v, d, 64);
    if (lane >= d) v += x;
  }
  return v;
}

// One workgroup per row, entry by entry.
constexpr int SMP_NT = 1024;
struct SmpShared {
  double tab[32];
  u64 mass[256], wsum[SMP_NT / 64], pre[2];
  unsigned cnt[256], wmin[SMP_NT / 64];
  int digit, tok;
};

// The first `ord` of the row at which the running count of the order reaches k (k > 0) or, among entries up to `most`, the
// running mass reaches `target`; and the mass up to it.
__device__ u64 smp_select(const SmpRow &r, SmpShared &sh, unsigned k, double target, u64 most, u64 &mass_to) {
  const int t = threadIdx.x;
  u64 pre = 0, before = 0;
  unsigned nbefore = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (shift == 24) {  // indexes are below 2^24
      continue;
    }
    for (int i = t; i < 256; i += blockDim.x) sh.mass[i] = 0, sh.cnt[i] = 0;
    __syncthreads();
    for (int i = t; i < r.V; i += blockDim.x) {
      const float x = r.at(i);
      const u64 o = (u64)smp_key(x) << 32 | (unsigned)i;
      const bool in = shift == 56 || o >> (shift + 8) == pre >> (shift + 8);
      if (in && o <= most) {
        const int d = (int)(o >> shift & 255);
        atomicAdd(&sh.cnt[d], 1u);
        const u64 w = smp_mass(r, smp_weight(r, x, sh.tab));
        if (w) atomicAdd(&sh.mass[d], w);
      }
    }
    __syncthreads();
    if (t == 0) {
      int d = 0;
      for (; d < 255; d++) {
        const bool there = k ? nbefore + sh.cnt[d] >= k : (double)(before + sh.mass[d]) >= target;
        if (there && sh.cnt[d]) break;
        nbefore += sh.cnt[d];
        before += sh.mass[d];
      }
      sh.digit = d;
      sh.pre[0] = before;
      sh.pre[1] = nbefore;
    }
    __syncthreads();
    pre |= (u64)sh.digit << shift;
    before = sh.pre[0];
    nbefore = (unsigned)sh.pre[1];
    if (shift == 0) mass_to = before + sh.mass[sh.digit];
    __syncthreads();
  }
  return pre;
}

__global__ __launch_bounds__(SMP_NT) void k_sample_any(SampleArgs a) {
  __shared__ SmpShared sh;
  const int row = blockIdx.x, t = threadIdx.x, w = t >> 6, lane = t & 63;
  SmpRow r{(const char *)a.x + (long)row * a.stride * (a.x16 ? 2 : 4), a.x16, a.V, a.S, 0.0, 0.0, 0.0};
  SmpSet s;
  const bool ok = smp_set(a, row, s);
  smp_table(sh.tab);
  uint32_t top = 0xffffffffu;
  for (int i = t; i < r.V; i += SMP_NT) top = min(top, smp_key(r.at(i)));
  top = smp_wave_min(top);
  if (lane == 0) sh.wmin[w] = top;
  __syncthreads();
  for (int i = 0; i < SMP_NT / 64; i++) top = min(top, sh.wmin[i]);
  const float m = smp_value(top);
  float *probs = a.probs ? a.probs + (long)row * r.V : nullptr;
  if (!ok || !(fabsf(m) < INFINITY)) {
    if (t == 0) {
      a.tokens[row] = -1;
      if (!ok) *a.bad = 1;
    }
    if (probs)
      for (int i = t; i < r.V; i += SMP_NT) probs[i] = 0.0f;
    return;
  }
  r.m = m;
  r.inv_t = 1.0 / s.t;
  u64 most = ~0ull, mass = 0;
  const bool by_k = s.k > 0 && s.k < r.V;
  if (by_k) most = smp_select(r, sh, s.k, 0.0, most, mass);
  auto total = [&]() {
    u64 v = 0;
    for (int i = t; i < r.V; i += SMP_NT) {
      const float x = r.at(i);
      const double wt = smp_weight(r, x, sh.tab);
      if (((u64)smp_key(x) << 32 | (unsigned)i) <= most && wt >= r.min_p) v += smp_mass(r, wt);
    }
    v = smp_wave_sum(v);
    __syncthreads();
    if (lane == 0) sh.wsum[w] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < SMP_NT / 64; i++) v += sh.wsum[i];
    return v;
  };
  if (s.top_p < 1.0) {
    if (!by_k) mass = total();
    most = smp_select(r, sh, 0, s.top_p * (double)mass, most, mass);
  }
  r.min_p = s.min_p;
  const u64 all = total();
  const double target = s.u * (double)all, scale = ldexp(1.0, r.S) / (double)all;
  u64 run = 0;
  if (t == 0) sh.tok = INT32_MAX;
  __syncthreads();
  for (int i0 = 0; i0 < r.V; i0 += SMP_NT) {
    const int i = i0 + t;
    double wt = 0.0;
    if (i < r.V) {
      const float x = r.at(i);
      wt = smp_weight(r, x, sh.tab);
      if (((u64)smp_key(x) << 32 | (unsigned)i) > most || !(wt >= r.min_p)) wt = 0.0;
      if (probs) probs[i] = (float)(wt * scale);
    }
    const u64 in = smp_wave_scan(smp_mass(r, wt));
    if (lane == 63) sh.wsum[w] = in;
    __syncthreads();
    u64 mine = run + in;
    for (int j = 0; j < w; j++) mine += sh.wsum[j];
    if (i < r.V && (double)mine > target) atomicMin(&sh.tok, i);
    for (int j = 0; j < SMP_NT / 64; j++) run += sh.wsum[j];
    __syncthreads();
    if (!probs && sh.tok != INT32_MAX) break;
  }
  if (t == 0) a.tokens[row] = sh.tok;
}

size_t sample_scratch(const Ctx &c, size_t n, int V) { return 256; }

hipError_t launch_sample(const Ctx &c, SampleArgs a, size_t n, void *scratch) {
  int bits = 0;
  while (bits < 31 && (1L << bits) < a.V) bits++;
  a.S = std::min(45, 62 - bits);
  launch_k(c, k_sample_any, dim3((unsigned)n), dim3(SMP_NT), a);
  return hipGetLastError();
}

}  // namespace rbt

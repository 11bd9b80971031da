// sample.hip -- tokens and probabilities from logits: temperature, top-k, top-p, min-p, one draw.
//
// With m the largest logit, w_i = exp((x_i - m) / t). The entries' order is by `ord`, 64 bits: the logit's bits turned so
// that larger ones come first, then the index. top-k, top-p and min-p each keep a run from the front of the order, so
// what is kept are the entries up to one `ord`.
//
// Weights are summed in whole numbers of 2^-S (S = 62 less the vocabulary's bits, at most 45): such sums do not depend on
// their order or on how the row was split, so equal calls give equal tokens, and a draw differs from one in real numbers
// only where u is within 2^-S times the number of entries of a border. (Sums in fp32 would move every border by 1e-7.)
//
// How the thresholds are found:
//   top-k of up to three quarters of the row's parts (some threads' entries), which have a largest entry each; at least k
//     entries are as large as the k-th of those, and few more, so those go to a list.
//   else 512 buckets of (m - x) / t, with counts and rounded masses, tell the buckets where the thresholds may lie, and
//     those buckets' entries go to a list.
//   The list (at most SMP_LIST) is sorted, summed up, and every threshold found in it. Without thresholds there is none.
//   A row whose list would be longer is taken digit by digit of `ord`, by one workgroup: seven passes over the row for top-k,
//     seven for top-p, and the draw's. Such are thousands of equal logits; rows without spikes, where one bucket at top-p's
//     threshold holds more than the list (normal logits of deviation 1, top-p 0.9, from some 100000 entries on); and rows with
//     fewer finite logits than top-k, whose parts' largest run out so that all entries are listed. Right, and slow. Measured, one
//     row, us, with the list and digit by digit: 32000 entries 18 and 290 (masked to 20 tokens, top-k 50) to 760 (equal
//     logits, top-k 2500 and top-p), 131072 entries 24 to 76 and 1820 to 3620, 248320 26 to 38 and 3400 to 6540, 2^20 40 and
//     14200 to 27000; 64 rows of 131072 38 to 128 and 4480 to 9700.
//
//   k_sample_one   rows of up to 32768 entries, and any rows where there are enough for the chip: a workgroup of 16 waves
//                  per row does all of it, and the probabilities, in one launch.
//   k_sample_top, k_sample_cut, k_sample_list, k_sample_probs   longer rows in G chunks, a workgroup each: the chunk's
//                  largest entries; the list or the buckets; the buckets' list; the probabilities. No workgroup waits for
//                  another: the last one of a row to arrive goes on.
#include "rbt_device.h"
#include "rbt_internal.h"

namespace rbt {

typedef unsigned long long u64;

constexpr int SMP_NT = 256, SMP_ONE = 1024;  // threads of a chunk's workgroup, of a row's
constexpr int SMP_NB = 512, SMP_LIST = 2048, SMP_GMAX = 32, SMP_PARTS = 64;

// A logit's bits, larger logits first; NaN counts as -inf, and -0 as 0.
__device__ __forceinline__ uint32_t smp_key(float x) {
  if (!(x > -INFINITY)) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float smp_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu);
}
__device__ __forceinline__ u64 smp_ord(float x, int i) { return (u64)smp_key(x) << 32 | (unsigned)i; }

struct SmpRow {
  const void *x;
  int x16, V, S;  // 2^S units in a weight of 1
  double m, inv_t;
  __device__ __forceinline__ float at(int i) const {
    return x16 ? rbt_bf16_f32(((const uint16_t *)x)[i]) : ((const float *)x)[i];
  }
};
__device__ __forceinline__ SmpRow smp_row(const SampleArgs &a, int row) {
  return {(const char *)a.x + (long)row * a.stride * (a.x16 ? 2 : 4), a.x16, a.V, a.S, 0.0, 0.0};
}

struct SmpSet {  // a row's settings
  int k;
  double t, top_p, min_p, u;
  bool ok, by_k, by_p, by_m;
};
__device__ __forceinline__ SmpSet smp_set(const SampleArgs &a, int r) {
  SmpSet s;
  const float t = a.temp ? a.temp[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f, q = a.min_p ? a.min_p[r] : 0.0f, u = a.u[r];
  s.k = a.top_k ? a.top_k[r] : 0;
  s.t = t;
  s.top_p = p;
  s.min_p = q;
  s.u = u;
  s.ok = t >= 0.0f && t < INFINITY && s.k >= 0 && p >= 0.0f && p <= 1.0f && q >= 0.0f && q <= 1.0f && u >= 0.0f && u < 1.0f;
  if (t == 0.0f) {  // greedy: the first of the order
    s.k = 1;
    s.t = 1.0;
  }
  s.by_k = s.k > 0 && s.k < a.V;
  s.by_p = p < 1.0f;
  s.by_m = q > 0.0f;
  return s;
}

// ---- weights ---------------------------------------------------------------------------------------
// 2^(k / 128)
__device__ const double SMP_POW[128] = {
    0x1.0000000000000p+0, 0x1.0163da9fb3335p+0, 0x1.02c9a3e778061p+0, 0x1.04315e86e7f85p+0,
    0x1.059b0d3158574p+0, 0x1.0706b29ddf6dep+0, 0x1.0874518759bc8p+0, 0x1.09e3ecac6f383p+0,
    0x1.0b5586cf9890fp+0, 0x1.0cc922b7247f7p+0, 0x1.0e3ec32d3d1a2p+0, 0x1.0fb66affed31bp+0,
    0x1.11301d0125b51p+0, 0x1.12abdc06c31ccp+0, 0x1.1429aaea92de0p+0, 0x1.15a98c8a58e51p+0,
    0x1.172b83c7d517bp+0, 0x1.18af9388c8deap+0, 0x1.1a35beb6fcb75p+0, 0x1.1bbe084045cd4p+0,
    0x1.1d4873168b9aap+0, 0x1.1ed5022fcd91dp+0, 0x1.2063b88628cd6p+0, 0x1.21f49917ddc96p+0,
    0x1.2387a6e756238p+0, 0x1.251ce4fb2a63fp+0, 0x1.26b4565e27cddp+0, 0x1.284dfe1f56381p+0,
    0x1.29e9df51fdee1p+0, 0x1.2b87fd0dad990p+0, 0x1.2d285a6e4030bp+0, 0x1.2ecafa93e2f56p+0,
    0x1.306fe0a31b715p+0, 0x1.32170fc4cd831p+0, 0x1.33c08b26416ffp+0, 0x1.356c55f929ff1p+0,
    0x1.371a7373aa9cbp+0, 0x1.38cae6d05d866p+0, 0x1.3a7db34e59ff7p+0, 0x1.3c32dc313a8e5p+0,
    0x1.3dea64c123422p+0, 0x1.3fa4504ac801cp+0, 0x1.4160a21f72e2ap+0, 0x1.431f5d950a897p+0,
    0x1.44e086061892dp+0, 0x1.46a41ed1d0057p+0, 0x1.486a2b5c13cd0p+0, 0x1.4a32af0d7d3dep+0,
    0x1.4bfdad5362a27p+0, 0x1.4dcb299fddd0dp+0, 0x1.4f9b2769d2ca7p+0, 0x1.516daa2cf6642p+0,
    0x1.5342b569d4f82p+0, 0x1.551a4ca5d920fp+0, 0x1.56f4736b527dap+0, 0x1.58d12d497c7fdp+0,
    0x1.5ab07dd485429p+0, 0x1.5c9268a5946b7p+0, 0x1.5e76f15ad2148p+0, 0x1.605e1b976dc09p+0,
    0x1.6247eb03a5585p+0, 0x1.6434634ccc320p+0, 0x1.6623882552225p+0, 0x1.68155d44ca973p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6c012750bdabfp+0, 0x1.6dfb23c651a2fp+0, 0x1.6ff7df9519484p+0,
    0x1.71f75e8ec5f74p+0, 0x1.73f9a48a58174p+0, 0x1.75feb564267c9p+0, 0x1.780694fde5d3fp+0,
    0x1.7a11473eb0187p+0, 0x1.7c1ed0130c132p+0, 0x1.7e2f336cf4e62p+0, 0x1.80427543e1a12p+0,
    0x1.82589994cce13p+0, 0x1.8471a4623c7adp+0, 0x1.868d99b4492edp+0, 0x1.88ac7d98a6699p+0,
    0x1.8ace5422aa0dbp+0, 0x1.8cf3216b5448cp+0, 0x1.8f1ae99157736p+0, 0x1.9145b0b91ffc6p+0,
    0x1.93737b0cdc5e5p+0, 0x1.95a44cbc8520fp+0, 0x1.97d829fde4e50p+0, 0x1.9a0f170ca07bap+0,
    0x1.9c49182a3f090p+0, 0x1.9e86319e32323p+0, 0x1.a0c667b5de565p+0, 0x1.a309bec4a2d33p+0,
    0x1.a5503b23e255dp+0, 0x1.a799e1330b358p+0, 0x1.a9e6b5579fdbfp+0, 0x1.ac36bbfd3f37ap+0,
    0x1.ae89f995ad3adp+0, 0x1.b0e07298db666p+0, 0x1.b33a2b84f15fbp+0, 0x1.b59728de5593ap+0,
    0x1.b7f76f2fb5e47p+0, 0x1.ba5b030a1064ap+0, 0x1.bcc1e904bc1d2p+0, 0x1.bf2c25bd71e09p+0,
    0x1.c199bdd85529cp+0, 0x1.c40ab5fffd07ap+0, 0x1.c67f12e57d14bp+0, 0x1.c8f6d9406e7b5p+0,
    0x1.cb720dcef9069p+0, 0x1.cdf0b555dc3fap+0, 0x1.d072d4a07897cp+0, 0x1.d2f87080d89f2p+0,
    0x1.d5818dcfba487p+0, 0x1.d80e316c98398p+0, 0x1.da9e603db3285p+0, 0x1.dd321f301b460p+0,
    0x1.dfc97337b9b5fp+0, 0x1.e264614f5a129p+0, 0x1.e502ee78b3ff6p+0, 0x1.e7a51fbc74c83p+0,
    0x1.ea4afa2a490dap+0, 0x1.ecf482d8e67f1p+0, 0x1.efa1bee615a27p+0, 0x1.f252b376bba97p+0,
    0x1.f50765b6e4540p+0, 0x1.f7bfdad9cbe14p+0, 0x1.fa7c1819e90d8p+0, 0x1.fd3c22b8f71f1p+0,
};
__device__ __forceinline__ void smp_table(double *tab) {
  if (threadIdx.x < 128) tab[threadIdx.x] = SMP_POW[threadIdx.x];
}
// exp(y) times 2^sh for y in [-690, 0]: 2^(k/128) from the table times a Taylor polynomial of what is left (at most
// ln 2 / 256: the fifth term is below 2^-49), and a whole power of two in the exponent's bits (which stay in range for sh
// of 0 and y >= -690, and for sh up to 45). k is read off a sum with 1.5 * 2^52 instead of converted.
__device__ __forceinline__ double smp_exp(double y, int sh, const double *tab) {
  const double big = 0x1.8p52, kb = fma(y, 184.6649652337873, big);
  const int n = (int)(unsigned)__double_as_longlong(kb);
  const double r = fma(kb - big, -0.0054152123481245725, y);
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  const long long v = __double_as_longlong(tab[n & 127] * p);
  return __longlong_as_double(v + ((long long)((n >> 7) + sh) << 52));
}
__device__ __forceinline__ double smp_weight(const SmpRow &r, float x, const double *tab) {
  const double y = ((double)x - r.m) * r.inv_t;
  return y > -690.0 ? smp_exp(y, 0, tab) : 0.0;
}
// The weight in units of 2^-S, to the nearest (w <= 1, S <= 45; e^-34 is below 2^-46).
__device__ __forceinline__ u64 smp_mass(const SmpRow &r, float x, const double *tab) {
  const double y = ((double)x - r.m) * r.inv_t;
  return y > -34.0 ? (u64)__double_as_longlong(smp_exp(y, r.S, tab) + 0x1p52) & 0xfffffffffffffull : 0;
}

__device__ __forceinline__ u64 smp_units(const SmpRow &r, double w) {
  return (u64)__double_as_longlong(ldexp(w, r.S) + 0x1p52) & 0xfffffffffffffull;
}

// The bucket of a logit: 24ths of (m - x) / t, never falling along the order; the last holds all from 21.3 on.
__device__ __forceinline__ float smp_scale(double t) { return fminf(24.0f / (float)t, 1e30f); }
__device__ __forceinline__ int smp_bucket(float m, float x, float cf) {
  return x > -INFINITY ? (int)fminf((m - x) * cf, 511.0f) : 511;
}

// ---- the row's entries -----------------------------------------------------------------------------
// Entries lo .. hi - 1 of the row, NT threads side by side: four(i, x) for aligned fours, one(i, x) for the up to three
// before and after them. Two fours of a thread are taken at once and the next two are on their way; more copies of
// what is done with them only make longer programs, whose first run from memory takes longer than the row (with eight
// fours at once k_sample_one had 119 KB, and 1500 entries took 27 us).
template <int NT, typename F4, typename F1>
__device__ __forceinline__ void smp_fours(const SmpRow &r, int lo, int hi, F4 four, F1 one) {
  const int t = threadIdx.x;
  const int a0 = min(hi, lo + (-(int)(((uintptr_t)r.x >> (r.x16 ? 1 : 2)) + lo) & 3)), n = (hi - a0) >> 2, a1 = a0 + 4 * n;
  auto load = [&](int q, float (&x)[4]) {
    const int i = a0 + 4 * min(q, n - 1);
    if (r.x16) {
      const uint2 v = *(const uint2 *)((const uint16_t *)r.x + i);
      x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
      x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
    } else {
      const float4 v = *(const float4 *)((const float *)r.x + i);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
  };
  float x[2][4], y[2][4];
  if (t < n) {
    load(t, y[0]);
    load(t + NT, y[1]);
  }
#pragma unroll 1
  for (int q = t; q < n; q += 2 * NT) {
#pragma unroll
    for (int e = 0; e < 4; e++) x[0][e] = y[0][e], x[1][e] = y[1][e];
    load(q + 2 * NT, y[0]);
    load(q + 3 * NT, y[1]);
    four(a0 + 4 * q, x[0]);
    if (q + NT < n) four(a0 + 4 * (q + NT), x[1]);
  }
  const int e = t < a0 - lo ? lo + t : a1 + t - (a0 - lo);
  if (e < hi) one(e, r.at(e));
}
template <int NT, typename F>
__device__ __forceinline__ void smp_each(const SmpRow &r, int lo, int hi, F f) {
  smp_fours<NT>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) f(i + e, x[e]);
  }, f);
}

// ---- over the workgroup ----------------------------------------------------------------------------
struct SmpRed {
  u64 w[SMP_ONE / 64];
};
__device__ __forceinline__ u64 smp_wave_sum(u64 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += (u64)__shfl_xor((long long)v, d, 64);
  return v;
}
template <int NT>
__device__ __forceinline__ u64 smp_sum(u64 v, SmpRed &red) {
  v = smp_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) v += red.w[i];
  return v;
}
template <int NT>
__device__ __forceinline__ u64 smp_scan(u64 v, u64 &all, SmpRed &red) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 x = (u64)__shfl_up((long long)v, d, 64);
    if (lane >= d) v += x;
  }
  __syncthreads();
  if (lane == 63) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    if (i < (int)(threadIdx.x >> 6)) v += red.w[i];
    all += red.w[i];
  }
  return v;
}
template <int NT>
__device__ __forceinline__ u64 smp_least(u64 v, SmpRed &red) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = min(v, (u64)__shfl_xor((long long)v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red.w[0];
#pragma unroll
  for (int i = 1; i < NT / 64; i++) v = min(v, red.w[i]);
  return v;
}

// A thread's first entry of the order (~0: none above -inf).
template <int NT>
__device__ __forceinline__ u64 smp_best(const SmpRow &r, int lo, int hi) {
  float best = -INFINITY;
  int at = 0;
  smp_each<NT>(r, lo, hi, [&](int i, float x) {
    if (x > best || (x == best && i < at)) best = x, at = i;
  });
  return best > -INFINITY ? smp_ord(best, at) : ~0ull;
}

// A key that at least k of n <= 64 N keys (of parts of the row; in LDS) are not above, and few more: bit by bit to the
// largest value that fewer than k keys are below, or to one that a few more than k are. By one wave: a barrier for
// every bit cost 5 us.
template <int N>
__device__ __forceinline__ unsigned smp_kth(const unsigned *key, int n, int k) {
  __shared__ unsigned got;
  const int t = threadIdx.x;
  if (t < 64) {
    unsigned mine[N], lo = 0;
#pragma unroll
    for (int i = 0; i < N; i++) mine[i] = t + 64 * i < n ? key[t + 64 * i] : 0xffffffffu;
#pragma unroll 1
    for (int b = 31; b >= 0; b--) {
      const unsigned x = lo | 1u << b;
      float f = 0.0f;  // (whole numbers)
#pragma unroll
      for (int i = 0; i < N; i++) f += mine[i] < x ? 1.0f : 0.0f;
      const int c = (int)__int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(rbt_group_sum<64>(f))));
      if (c >= k && c <= k + k / 4 + 8) {
        lo = x - 1;
        break;
      }
      if (c < k) lo = x;
    }
    if (t == 0) got = lo;
  }
  __syncthreads();
  return got;
}

// ---- the list --------------------------------------------------------------------------------------
struct SmpFind {
  u64 ord[SMP_LIST], run[SMP_LIST];  // the list in order, its masses summed up to each
};
struct SmpSlow {
  u64 mass[256];
  unsigned cnt[256];
  u64 before, nbefore;
  int digit;
};
union SmpLds {
  SmpFind f;
  SmpSlow slow;
  u64 hist[SMP_NB + 1];
};
// Where the thresholds are: the list holds the n1 entries of buckets b0 .. b1, which cnt0 come before, and those of
// bucket kb where it lies beyond (top-k's, which cntk come before).
struct SmpCut {
  int b0, b1, kb, n1, n, cnt0, cntk;
  bool beyond;
};

// The list's n entries (f.ord, any order) put in order, and the thresholds found in it; mass0 and massk lie before
// buckets b0 and kb, `whole` is the row's mass (~0: the list is all that counts). Returns the last kept entry (-1: none of
// the list), with kept mass `total`.
template <int NT>
__device__ __forceinline__ int smp_find(const SmpRow &r, const SmpSet &s, const double *tab, SmpFind &f, int n, const SmpCut &c, u64 mass0,
                                        u64 massk, u64 whole, u64 &total, SmpRed &red) {
  __shared__ int ip, im;
  const int t = threadIdx.x, n1 = c.n1;
  int n2 = 64;
  while (n2 < n) n2 *= 2;
#pragma unroll 1
  for (int i = n + t; i < n2; i += NT) f.ord[i] = ~0ull;
  if (t == 0) ip = n1, im = n1 - 1;
  __syncthreads();
  u64 run = 0;
  if (n2 <= 256) {
    // every entry counts those before it and their masses; NT / n2 threads share an entry's
    const int i = t % n2;
    u64 *mass = f.ord + SMP_LIST / 2, *sum = f.run + SMP_LIST / 2, *at = sum + 256;
    const u64 o = f.ord[i];
    const double w = smp_weight(r, i < n ? smp_value((uint32_t)(o >> 32)) : -INFINITY, tab);
    if (t < n2) {
      mass[i] = smp_units(r, w);
      sum[i] = at[i] = 0;
    }
    __syncthreads();
    u64 v = 0, before = 0;
#pragma unroll 4
    for (int j = t / n2; j < n; j += NT / n2) {
      const bool in = f.ord[j] <= o;
      v += in ? mass[j] : 0;
      before += in;
    }
    if (NT > n2) {
      atomicAdd(&sum[i], v);
      atomicAdd(&at[i], before);
      __syncthreads();
      v = sum[i];
      before = at[i];
    }
    __syncthreads();
    if (t < n) {
      const int to = (int)before - 1;
      f.ord[to] = o;
      f.run[to] = v;
      if (to < n1 && !(w >= s.min_p)) atomicMin(&im, to - 1);
    }
    __syncthreads();
    run = f.run[n - 1];
  } else {
    // bitonic, padded to a power of two; steps of up to 64 stay within a wave's 128 entries
#pragma unroll 1
    for (int len = 2; len <= n2; len *= 2)
#pragma unroll 1
      for (int d = len / 2; d; d /= 2) {
#pragma unroll 1
        for (int i = t; i < n2 / 2; i += NT) {
          const int x = 2 * i - (i & (d - 1)), y = x + d;
          const u64 p = f.ord[x], q = f.ord[y];
          if ((p > q) == !(x & len)) f.ord[x] = q, f.ord[y] = p;
        }
        if (d > 64 || (d == 1 && len > 64))
          __syncthreads();
        else
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      }
    __syncthreads();
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += NT) {
      const int i = i0 + t;
      const double w = smp_weight(r, i < n ? smp_value((uint32_t)(f.ord[i] >> 32)) : -INFINITY, tab);
      u64 all;
      const u64 up = run + smp_scan<NT>(smp_units(r, w), all, red);
      if (i < n) f.run[i] = up;
      // (weights fall along the order: the first that is too light)
      if (i < n1 && !(w >= s.min_p) && (i == 0 || smp_value((uint32_t)(f.ord[i] >> 32)) != smp_value((uint32_t)(f.ord[i - 1] >> 32))))
        atomicMin(&im, i - 1);
      run += all;
    }
    __syncthreads();
  }
  int last = n1 - 1;
  u64 left = whole == ~0ull ? run : whole;  // the mass that top-k leaves
  if (s.by_k && !c.beyond) {
    last = s.k - 1 - c.cnt0;
    left = mass0 + f.run[last];
  } else if (s.by_k) {
    left = massk + f.run[n1 + s.k - 1 - c.cntk] - (n1 ? f.run[n1 - 1] : 0);
  }
  if (s.by_p) {
    const double target = s.top_p * (double)left;
#pragma unroll 1
    for (int i = t; i < n1; i += NT)  // (the first that reaches it: one thread's)
      if ((double)(mass0 + f.run[i]) >= target && (i == 0 || !((double)(mass0 + f.run[i - 1]) >= target))) ip = i;
    __syncthreads();
    last = min(last, ip);
  }
  last = min(last, min(im, n1 - 1));
  total = mass0 + (last >= 0 ? f.run[last] : 0);
  return last;
}

// The draw's border: a running mass passes u times the whole where it is above this. In whole numbers, since sums past 2^53
// are rounded as doubles, and a border that lies in one chunk by rounded sums need not lie in its entries.
__device__ __forceinline__ u64 smp_left(const SmpSet &s, u64 total) { return (u64)(s.u * (double)total); }

// Where nothing is kept before the list: the draw among its entries up to `last`, in the order of their indexes.
template <int NT>
__device__ __forceinline__ int smp_draw_list(const SmpFind &f, int last, u64 left) {
  __shared__ u64 first;
  const int t = threadIdx.x;
  if (t == 0) first = ~0ull;
  __syncthreads();
  for (int i = t; i <= last; i += NT) {
    const unsigned at = (unsigned)f.ord[i];
    u64 run = 0, before = 0;
#pragma unroll 2
    for (int j = 0; j <= last; j++) {
      const u64 up = f.run[j];
      if ((unsigned)f.ord[j] <= at) run += up - before;
      before = up;
    }
    if (run > left) atomicMin(&first, (u64)at);
  }
  __syncthreads();
  return first == ~0ull ? -1 : (int)first;
}

// The least index in [lo, hi) at which the running mass of entries up to thr passes `left`: every wave sums a part of it,
// then the workgroup looks through the part where it passes, four entries a thread.
template <int NT>
__device__ __forceinline__ int smp_draw(const SmpRow &r, const double *tab, int lo, int hi, u64 thr, u64 left, SmpRed &red) {
  __shared__ int found;
  constexpr int W = NT / 64, UN = 8;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, part = (hi - lo + W - 1) / W;
  auto kept = [&](float x, int i) { return smp_ord(x, i) <= thr ? smp_mass(r, x, tab) : 0; };
  u64 sum = 0;
  const int end = min(hi, lo + (w + 1) * part);
#pragma unroll 1
  for (int i = lo + w * part + lane; i < end; i += 64 * UN) {
    float x[UN];
#pragma unroll
    for (int e = 0; e < UN; e++) x[e] = r.at(min(i + 64 * e, hi - 1));
#pragma unroll
    for (int e = 0; e < UN; e++)
      if (i + 64 * e < end) sum += kept(x[e], i + 64 * e);
  }
  sum = smp_wave_sum(sum);
  __syncthreads();
  if (lane == 0) red.w[w] = sum;
  if (t == 0) found = INT32_MAX;
  __syncthreads();
  u64 run = 0;
  int q = -1;
#pragma unroll
  for (int i = 0; i < W; i++) {
    if (q < 0 && run + red.w[i] > left) q = i;
    if (q < 0) run += red.w[i];
  }
  if (q < 0) return -1;  // (not reached: u below 1 times the whole is below the whole)
  const int e1 = min(hi, lo + (q + 1) * part);
#pragma unroll 1
  for (int i0 = lo + q * part; i0 < e1; i0 += 4 * NT) {
    const int i = i0 + 4 * t;
    u64 m[4], all;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = r.at(min(i + e, hi - 1));
      m[e] = i + e < e1 ? kept(x, i + e) : 0;
    }
    const u64 mine = (m[0] + m[1]) + (m[2] + m[3]), up = run + smp_scan<NT>(mine, all, red);
    if (up > left && up - mine <= left) {  // this thread's (one's alone)
      u64 at = up - mine;
      int e = 0;
#pragma unroll
      for (; e < 3; e++) {
        at += m[e];
        if (at > left) break;
      }
      found = i + e;
    }
    run += all;
    __syncthreads();
    if (found != INT32_MAX) return found;
  }
  return -1;
}

// ---- digit by digit --------------------------------------------------------------------------------
// The first `ord` of the row at which the running count of the order reaches k (k > 0) or, among entries up to `most`, the
// running mass reaches `target`; and the mass up to it.
template <int NT>
__device__ __noinline__ u64 smp_select(const SmpRow &r, const double *tab, SmpSlow &sh, unsigned k, double target, u64 most, u64 &mass_to) {
  const int t = threadIdx.x;
  u64 pre = 0, before = 0;
  unsigned nbefore = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (shift == 24) continue;  // indexes are below 2^24
    for (int i = t; i < 256; i += NT) sh.mass[i] = 0, sh.cnt[i] = 0;
    __syncthreads();
    for (int i = t; i < r.V; i += NT) {
      const float x = r.at(i);
      const u64 o = smp_ord(x, i);
      if ((shift == 56 || o >> (shift + 8) == pre >> (shift + 8)) && o <= most) {
        const int d = (int)(o >> shift & 255);
        atomicAdd(&sh.cnt[d], 1u);
        const u64 w = smp_mass(r, x, tab);
        if (w) atomicAdd(&sh.mass[d], w);
      }
    }
    __syncthreads();
    if (t == 0) {
      int held = 0;  // the last digit with any entry
      u64 mb = before, hm = before;
      unsigned nb = nbefore, hn = nbefore;
      for (int d = 0; d < 256; d++) {
        if (!sh.cnt[d]) continue;
        held = d;
        hm = mb;
        hn = nb;
        if (k ? nb + sh.cnt[d] >= k : (double)(mb + sh.mass[d]) >= target) break;
        nb += sh.cnt[d];
        mb += sh.mass[d];
      }
      sh.digit = held;
      sh.before = hm;
      sh.nbefore = hn;
    }
    __syncthreads();
    pre |= (u64)sh.digit << shift;
    before = sh.before;
    nbefore = (unsigned)sh.nbefore;
    if (shift == 0) mass_to = before + sh.mass[sh.digit];
    __syncthreads();
  }
  return pre;
}
template <int NT>
__device__ __forceinline__ u64 smp_slow(const SmpRow &r, const SmpSet &s, const double *tab, SmpSlow &sh, u64 &total, SmpRed &red) {
  const int t = threadIdx.x;
  u64 thr = ~0ull, mass = 0, sum = 0, last = 0;
  if (s.by_k) {
    thr = smp_select<NT>(r, tab, sh, s.k, 0.0, thr, mass);
  } else if (s.by_p) {
    for (int i = t; i < r.V; i += NT) mass += smp_mass(r, r.at(i), tab);
    mass = smp_sum<NT>(mass, red);
  }
  if (s.by_p) thr = smp_select<NT>(r, tab, sh, 0, s.top_p * (double)mass, thr, mass);
  for (int i = t; i < r.V; i += NT) {
    const float x = r.at(i);
    const u64 o = smp_ord(x, i);
    if (o <= thr && (!s.by_m || smp_weight(r, x, tab) >= s.min_p)) {
      sum += smp_mass(r, x, tab);
      last = max(last, o);
    }
  }
  total = smp_sum<NT>(sum, red);
  if (s.by_m) thr = ~smp_least<NT>(~last, red);  // the last that is heavy enough
  return thr;
}

// ---- buckets ---------------------------------------------------------------------------------------
// A bucket's word: its count in the low cb bits, above them its entries' masses / 2^sh, each cut to a whole number.
struct SmpUnits {
  int cb, sh;
};
// Where the thresholds may lie, from the buckets' words (two of them, v, in each of the first 256 threads) and the row's
// mass `all`. hist is scratch.
template <int NT>
__device__ __forceinline__ SmpCut smp_cut(const SmpSet &s, int V, const SmpUnits &un, const u64 (&v)[2], u64 all, u64 *hist, SmpRed &red) {
  __shared__ int kb_s, p0_s, p1_s, held_s;
  const int t = threadIdx.x;
  const bool in = NT == 256 || t < 256;
  u64 rest;
  const u64 upto = smp_scan<NT>(in ? v[0] + v[1] : 0, rest, red);
  __syncthreads();
  if (in) {
    hist[2 * t + 1] = upto - v[1];
    hist[2 * t] = upto - v[1] - v[0];
  }
  if (t == 0) {
    hist[SMP_NB] = rest;
    kb_s = p0_s = p1_s = SMP_NB;
    held_s = 0;
  }
  __syncthreads();
  const unsigned one = (1u << un.cb) - 1;
  auto cnt = [&](int b) { return b == SMP_NB ? V : (int)((unsigned)hist[b] & one); };
  // the mass before bucket b, in units of 2^(sh - S): at least, and below
  auto low = [&](int b) { return (double)(hist[b] >> un.cb); };
  auto high = [&](int b) { return b == SMP_NB ? ldexp((double)all, -un.sh) + 1.0 : low(b) + (double)cnt(b); };
  if (s.by_k && in)
    for (int e = 0; e < 2; e++)
      if (cnt(2 * t + e) < s.k && cnt(2 * t + e + 1) >= s.k) kb_s = 2 * t + e;
  __syncthreads();
  const int kb = kb_s;
  if (s.by_p && in) {  // of the mass that top-k leaves
    const double whole0 = s.by_k ? low(kb) : ldexp((double)all, -un.sh), whole1 = s.by_k ? high(kb + 1) : whole0;
    for (int e = 0; e < 2; e++) {  // (the first of those that reach it: one thread's)
      const int b = 2 * t + e;
      if (high(b + 1) >= s.top_p * whole0 && (b == 0 || !(high(b) >= s.top_p * whole0))) p0_s = b;
      if (low(b + 1) >= s.top_p * whole1 && (b == 0 || !(low(b) >= s.top_p * whole1))) p1_s = b;
    }
  }
  __syncthreads();
  int b0 = s.by_p ? min(p0_s, kb) : kb, b1 = s.by_p ? min(p1_s, kb) : kb;
  if (s.by_m) {  // the bucket of the least weight, and its neighbours for their rounding
    // (temperatures past which buckets do not follow the weights: smp_scale cuts 24 / t, or logits up to 21.3 t apart pass
    // f32. Any bucket may then hold the least weight)
    const bool all_of_them = s.t < 0x1p-90 || s.t > 0x1p120;
    const int b = all_of_them ? 0 : (int)fmin(-log(s.min_p) * 24.0, 600.0);
    b0 = min(b0, max(b - 1, 0));
    b1 = min(b1, all_of_them ? SMP_NB : b + 1);
  }
  b0 = min(b0, SMP_NB - 1);
  b1 = min(b1, SMP_NB - 1);
  if (cnt(b1 + 1) == cnt(b0)) {  // no entry near min_p: the threshold is the last of the bucket before
    if (in)
      for (int e = 0; e < 2; e++)
        if (2 * t + e < b0 && cnt(2 * t + e + 1) > cnt(2 * t + e)) atomicMax(&held_s, 2 * t + e);
    __syncthreads();
    b0 = held_s;  // (the largest logit is in bucket 0)
  }
  SmpCut c;
  c.b0 = b0;
  c.b1 = b1;
  c.kb = s.by_k ? kb : -1;
  c.beyond = s.by_k && kb > b1;
  c.cnt0 = cnt(b0);
  c.cntk = s.by_k ? cnt(kb) : 0;
  c.n1 = cnt(b1 + 1) - c.cnt0;
  c.n = c.n1 + (c.beyond ? cnt(kb + 1) - c.cntk : 0);
  __syncthreads();
  return c;
}
__device__ __forceinline__ SmpCut smp_cut_all(int n) { return {0, SMP_NB - 1, -1, n, n, 0, 0, false}; }

typedef float smp_f4 __attribute__((ext_vector_type(4), aligned(4)));  // (stores of four words want four bytes' alignment)
template <int NT>
__device__ __forceinline__ void smp_probs(const SampleArgs &a, const SmpRow &r, int row, int lo, int hi, u64 thr, u64 total, const double *tab) {
  const double scale = total ? ldexp(1.0, a.S) / (double)total : 0.0;
  float *to = a.probs + (long)row * a.V;
  auto p = [&](int i, float x) { return total && smp_ord(x, i) <= thr ? (float)(smp_weight(r, x, tab) * scale) : 0.0f; };
  smp_fours<NT>(r, lo, hi, [&](int i, const float (&x)[4]) {
    *(smp_f4 *)(to + i) = smp_f4{p(i, x[0]), p(i + 1, x[1]), p(i + 2, x[2]), p(i + 3, x[3])};
  }, [&](int i, float x) { to[i] = p(i, x); });
}

// ---- a workgroup per row -----------------------------------------------------------------------------
__global__ __launch_bounds__(SMP_ONE) void k_sample_one(SampleArgs a, SmpUnits un) {
  constexpr int NT = SMP_ONE;
  __shared__ SmpLds lds;
  __shared__ double tab[128];
  __shared__ SmpRed red;
  __shared__ unsigned here;
  const int row = blockIdx.x, t = threadIdx.x, V = a.V;
  SmpRow r = smp_row(a, row);
  const SmpSet s = smp_set(a, row);
  smp_table(tab);
  if (t == 0) here = 0;
  const u64 mine = smp_best<NT>(r, 0, V), top = smp_least<NT>(mine, red);
  const float m = smp_value((uint32_t)(top >> 32));
  const bool none = !s.ok || top == ~0ull || !(fabsf(m) < INFINITY);
  u64 thr = top, total = none ? 0 : 1ull << a.S;
  int tok = none ? -1 : (int)(unsigned)top;
  r.m = m;
  r.inv_t = 1.0 / s.t;
  if (!none && s.k != 1) {
    unsigned n;
    auto gather = [&](auto take) {
      __syncthreads();
      smp_each<NT>(r, 0, V, [&](int i, float x) {
        if (take(x)) {
          const unsigned at = atomicAdd(&here, 1u);
          if (at < SMP_LIST) lds.f.ord[at] = smp_ord(x, i);
        }
      });
      __syncthreads();
      n = here;
    };
    bool slow = false, drawn = false;
    if (s.by_k && s.k <= NT / 2 * 3 / 4) {  // (more parts than that make longer lists)
      unsigned key = (unsigned)(mine >> 32), *keys = (unsigned *)lds.f.run;
      key = min(key, (unsigned)__shfl_xor((int)key, 1, 64));
      if (t % 2 == 0) keys[t / 2] = key;
      __syncthreads();
      const unsigned most = smp_kth<NT / 128>(keys, NT / 2, s.k);
      gather([&](float x) { return smp_key(x) <= most; });
      slow = n > SMP_LIST;
      if (!slow) {
        const int last = smp_find<NT>(r, s, tab, lds.f, n, smp_cut_all(n), 0, 0, ~0ull, total, red);
        thr = lds.f.ord[last];
        tok = last < NT ? smp_draw_list<NT>(lds.f, last, smp_left(s, total))
                        : smp_draw<NT>(r, tab, 0, V, thr, smp_left(s, total), red);
      }
    } else {
      const bool any = s.by_k || s.by_p || s.by_m;
      const float cf = smp_scale(s.t);
      for (int i = t; i <= SMP_NB; i += NT) lds.hist[i] = 0;
      __syncthreads();
      u64 sum = 0;
      smp_each<NT>(r, 0, V, [&](int, float x) {
        const u64 v = smp_mass(r, x, tab);
        sum += v;
        const int b = smp_bucket(m, x, cf);
        if (any && b < SMP_NB - 1) atomicAdd(&lds.hist[b], (v >> un.sh) << un.cb | 1);
      });
      const u64 all = smp_sum<NT>(sum, red);
      thr = ~0ull;
      total = all;
      if (any) {
        const u64 v[2] = {t < 256 ? lds.hist[2 * t] : 0, t < 256 ? lds.hist[2 * t + 1] : 0};
        const SmpCut c = smp_cut<NT>(s, V, un, v, all, lds.hist, red);
        slow = c.n > SMP_LIST;
        if (!slow) {
          u64 sum0 = 0, sumk = 0;
          gather([&](float x) {
            const int b = smp_bucket(m, x, cf);
            if (b < c.b0 || (c.beyond && b < c.kb)) {
              const u64 w = smp_mass(r, x, tab);
              if (b < c.b0) sum0 += w;
              sumk += w;
            }
            return (b >= c.b0 && b <= c.b1) || b == c.kb;
          });
          sum0 = smp_sum<NT>(sum0, red);
          sumk = smp_sum<NT>(sumk, red);
          const int last = smp_find<NT>(r, s, tab, lds.f, n, c, sum0, sumk, all, total, red);
          thr = last >= 0 ? lds.f.ord[last] : lds.f.ord[0] - 1;
          if (sum0 == 0 && last < NT) {
            tok = smp_draw_list<NT>(lds.f, last, smp_left(s, total));
            drawn = true;
          }
        }
      }
      if (!slow && !drawn) tok = smp_draw<NT>(r, tab, 0, V, thr, smp_left(s, total), red);
    }
    if (slow) {
      thr = smp_slow<NT>(r, s, tab, lds.slow, total, red);
      tok = smp_draw<NT>(r, tab, 0, V, thr, smp_left(s, total), red);
    }
  }
  if (t == 0) {
    a.tokens[row] = tok;
    if (!s.ok) *a.bad = 1;
  }
  if (a.probs) smp_probs<NT>(a, r, row, 0, V, thr, total, tab);
}

// ---- a row in chunks -----------------------------------------------------------------------------------
enum { SMP_DONE = 0, SMP_FIND = 1, SMP_SLOW = 2 };
struct SmpState {  // a row between launches
  u64 thr, total;  // kept: entries up to thr, their mass (0: none, token -1)
  int mode;
  unsigned n;      // list entries so far
  SmpCut c;
};
struct SmpWork {  // scratch of up to CNT_N rows
  u64 *top, *hist, *cert, *list;  // [rows, G], [rows, G, SMP_NB], [rows, 2, G], [rows, SMP_LIST]
  unsigned *part;                 // [rows, G, SMP_PARTS]
  SmpState *state;
  unsigned *arrive;               // arrival counters, left at 0
  int G, len, row0;               // chunks of a row, entries of a chunk (a multiple of 4), first row
  SmpUnits un;
};

template <typename T>
__device__ __forceinline__ void smp_put(T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T smp_get(const T *p) {
  return __hip_atomic_load(const_cast<T *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the row's last; what its threads put before is then at the device's coherence point.
__device__ __forceinline__ bool smp_last(const SmpWork &k, int row) {
  __shared__ int last;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(k.arrive + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (unsigned)k.G;
    if (last) __hip_atomic_store(k.arrive + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last;
}

__global__ __launch_bounds__(SMP_NT) void k_sample_top(SampleArgs a, SmpWork k) {
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  const SmpRow r = smp_row(a, k.row0 + row);
  const u64 mine = smp_best<SMP_NT>(r, lo, hi);
  unsigned key = (unsigned)(mine >> 32);
  key = min(key, (unsigned)__shfl_xor((int)key, 1, 64));
  key = min(key, (unsigned)__shfl_xor((int)key, 2, 64));
  const long chunk = (long)row * k.G + g;
  if (t % 4 == 0) k.part[chunk * SMP_PARTS + t / 4] = key;
  const u64 top = smp_least<SMP_NT>(mine, red);
  if (t == 0) {
    k.top[chunk] = top;
    if (g == 0) k.state[row].n = 0;
  }
}

// The chunk where the running mass passes `left`, and the mass before it.
__device__ __forceinline__ int smp_chunk(const u64 *mass, int G, u64 left, u64 &before) {
  before = 0;
  for (int g = 0; g < G; g++) {
    if (before + mass[g] > left) return g;
    before += mass[g];
  }
  return -1;
}
__device__ __forceinline__ int smp_draw_chunk(const SmpRow &r, const SmpWork &k, const double *tab, const u64 *mass, u64 thr, u64 left,
                                              SmpRed &red) {
  u64 before;
  const int ch = smp_chunk(mass, k.G, left, before);
  return ch < 0 ? -1 : smp_draw<SMP_NT>(r, tab, ch * k.len, min(r.V, (ch + 1) * k.len), thr, left - before, red);
}
// The token: of the list up to `last`, and of what lies before it (mass0, by chunks in `chunk`).
__device__ __forceinline__ int smp_token(const SmpRow &r, const SmpWork &k, const SmpSet &s, const double *tab, const SmpFind &f, int last,
                                         u64 thr, u64 total, u64 mass0, u64 *chunk, SmpRed &red) {
  const u64 left = smp_left(s, total);
  if (mass0 == 0 && last < SMP_NT) return smp_draw_list<SMP_NT>(f, last, left);
  for (int i = threadIdx.x; i <= last; i += SMP_NT) {
    const u64 v = f.run[i] - (i ? f.run[i - 1] : 0);
    if (v) atomicAdd(&chunk[(int)((unsigned)f.ord[i] / (unsigned)k.len)], v);
  }
  __syncthreads();
  return smp_draw_chunk(r, k, tab, chunk, thr, left, red);
}
__device__ __forceinline__ void smp_finish(const SampleArgs &a, SmpState &st, int row, int tok, u64 thr, u64 total) {
  if (threadIdx.x == 0) {
    a.tokens[row] = tok;
    st.mode = SMP_DONE;
    st.thr = thr;
    st.total = total;
  }
}

// The entries of [lo, hi) that `take` wants, appended to the row's list: by the last workgroup the whole list is in lds.
// Its length goes past SMP_LIST where it does not fit. `then` runs before the workgroup's arrival. False for the
// workgroups that are not the last.
template <typename F, typename H>
__device__ __forceinline__ bool smp_gather(const SmpRow &r, const SmpWork &k, SmpState &st, int row, int lo, int hi, SmpFind &f, unsigned &n,
                                           F take, H then) {
  __shared__ unsigned here, base;
  const int t = threadIdx.x;
  if (t == 0) here = 0;
  __syncthreads();
  smp_each<SMP_NT>(r, lo, hi, [&](int i, float x) {
    if (take(x)) {
      const unsigned at = atomicAdd(&here, 1u);
      if (at < SMP_LIST) f.ord[at] = smp_ord(x, i);
    }
  });
  __syncthreads();
  n = here;
  then();
  u64 *list = k.list + (long)row * SMP_LIST;
  if (t == 0 && n) base = __hip_atomic_fetch_add(&st.n, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (unsigned i = t; i < min(n, (unsigned)SMP_LIST); i += SMP_NT)
    if (base + i < SMP_LIST) smp_put(list + base + i, f.ord[i]);
  if (!smp_last(k, row)) return false;
  const u64 ahead = smp_get(list + t);  // (the first ones beside their number)
  n = smp_get(&st.n);
  if (t < n) f.ord[t] = ahead;
  for (unsigned i = t + SMP_NT; i < min(n, (unsigned)SMP_LIST); i += SMP_NT) f.ord[i] = smp_get(list + i);
  __syncthreads();
  return true;
}

__global__ __launch_bounds__(SMP_NT) void k_sample_cut(SampleArgs a, SmpWork k) {
  constexpr int NT = SMP_NT;
  __shared__ SmpLds lds;
  __shared__ double tab[128];
  __shared__ u64 cert[SMP_GMAX];
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x, G = k.G, np = G * SMP_PARTS;
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  SmpRow r = smp_row(a, gr);
  const u64 top1 = t < G ? k.top[(long)row * G + t] : ~0ull;
  unsigned *keys = (unsigned *)lds.f.run;
  for (int i = t; i < np; i += NT) keys[i] = k.part[(long)row * np + i];
  const SmpSet s = smp_set(a, gr);
  smp_table(tab);
  const u64 top = smp_least<NT>(top1, red);
  const float m = smp_value((uint32_t)(top >> 32));
  SmpState &st = k.state[row];
  const bool none = !s.ok || top == ~0ull || !(fabsf(m) < INFINITY);
  if (none || s.k == 1) {  // nothing to draw from, or one entry
    if (g == 0) {
      if (!s.ok && t == 0) *a.bad = 1;
      smp_finish(a, st, gr, none ? -1 : (int)(unsigned)top, top, none ? 0 : 1ull << a.S);
    }
    return;
  }
  r.m = m;
  r.inv_t = 1.0 / s.t;
  if (s.by_k && s.k <= min(np * 3 / 4, SMP_LIST / 4)) {
    const unsigned most = smp_kth<SMP_GMAX * SMP_PARTS / 64>(keys, np, s.k);
    unsigned n;
    if (!smp_gather(r, k, st, row, lo, hi, lds.f, n, [&](float x) { return smp_key(x) <= most; }, [] {})) return;
    if (n <= SMP_LIST) {
      u64 total;
      const int last = smp_find<NT>(r, s, tab, lds.f, n, smp_cut_all(n), 0, 0, ~0ull, total, red);
      if (t < G) cert[t] = 0;
      __syncthreads();
      const u64 thr = lds.f.ord[last];
      smp_finish(a, st, gr, smp_token(r, k, s, tab, lds.f, last, thr, total, 0, cert, red), thr, total);
    } else if (t == 0) {
      st.mode = SMP_SLOW;
    }
    return;
  }
  for (int i = t; i <= SMP_NB; i += NT) lds.hist[i] = 0;
  __syncthreads();
  const float cf = smp_scale(s.t);
  u64 sum = 0;
  const bool any = s.by_k || s.by_p || s.by_m;
  smp_each<NT>(r, lo, hi, [&](int, float x) {
    const u64 v = smp_mass(r, x, tab);
    sum += v;
    const int b = smp_bucket(m, x, cf);
    if (any && b < SMP_NB - 1) atomicAdd(&lds.hist[b], (v >> k.un.sh) << k.un.cb | 1);  // (the last is what is left)
  });
  sum = smp_sum<NT>(sum, red);
  u64 *mine = k.cert + (long)row * 2 * G;
  if (t == 0) smp_put(mine + g, sum);
  const long at = (long)row * G * SMP_NB;
  if (any)
    for (int b = t; b < SMP_NB; b += NT) smp_put(k.hist + at + (long)g * SMP_NB + b, lds.hist[b]);
  if (!smp_last(k, row)) return;
  if (t < G) cert[t] = smp_get(mine + t);
  u64 v[2] = {0, 0};
  if (any) {
    constexpr int UN = 8;  // chunks whose loads are on their way at once
    for (int j0 = 0; j0 < G; j0 += UN) {
      u64 x[UN][2];
#pragma unroll
      for (int j = 0; j < UN; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) x[j][e] = smp_get(k.hist + at + (long)min(j0 + j, G - 1) * SMP_NB + 2 * t + e);
#pragma unroll
      for (int j = 0; j < UN; j++)
        if (j0 + j < G) v[0] += x[j][0], v[1] += x[j][1];
    }
  }
  __syncthreads();
  u64 all = 0;
  for (int j = 0; j < G; j++) all += cert[j];
  if (!any) {
    smp_finish(a, st, gr, smp_draw_chunk(r, k, tab, cert, ~0ull, smp_left(s, all), red), ~0ull, all);
    return;
  }
  const SmpCut c = smp_cut<NT>(s, a.V, k.un, v, all, lds.hist, red);
  if (t == 0) {
    st.mode = c.n > SMP_LIST ? SMP_SLOW : SMP_FIND;
    st.total = all;
    st.c = c;
    st.n = 0;
  }
}

__global__ __launch_bounds__(SMP_NT) void k_sample_list(SampleArgs a, SmpWork k) {
  constexpr int NT = SMP_NT;
  __shared__ SmpLds lds;
  __shared__ double tab[128];
  __shared__ u64 chunk[SMP_GMAX];
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x, G = k.G;
  SmpState &st = k.state[row];
  const int mode = st.mode;
  if (mode == SMP_DONE || (mode == SMP_SLOW && g)) return;
  const SmpCut c = st.c;
  const u64 all = st.total;
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  SmpRow r = smp_row(a, gr);
  const SmpSet s = smp_set(a, gr);
  smp_table(tab);
  const u64 top = smp_least<NT>(t < G ? k.top[(long)row * G + t] : ~0ull, red);
  const float m = smp_value((uint32_t)(top >> 32));
  r.m = m;
  r.inv_t = 1.0 / s.t;
  if (mode == SMP_SLOW) {
    u64 total;
    const u64 thr = smp_slow<NT>(r, s, tab, lds.slow, total, red);
    smp_finish(a, st, gr, smp_draw<NT>(r, tab, 0, a.V, thr, smp_left(s, total), red), thr, total);
    return;
  }
  const float cf = smp_scale(s.t);
  // the masses before the listed buckets, and before top-k's where that is another
  u64 sum0 = 0, sumk = 0, *mine = k.cert + (long)row * 2 * G;
  unsigned n;
  const bool last_one = smp_gather(r, k, st, row, lo, hi, lds.f, n, [&](float x) {
    const int b = smp_bucket(m, x, cf);
    if (b < c.b0 || (c.beyond && b < c.kb)) {
      const u64 v = smp_mass(r, x, tab);
      if (b < c.b0) sum0 += v;
      sumk += v;
    }
    return (b >= c.b0 && b <= c.b1) || b == c.kb;
  }, [&] {
    sum0 = smp_sum<NT>(sum0, red);
    sumk = smp_sum<NT>(sumk, red);
    if (t == 0) smp_put(mine + g, sum0), smp_put(mine + G + g, sumk);
  });
  if (!last_one) return;
  u64 v0 = 0, vk = 0;
  if (t < G) {  // (the chunks' masses are read by all after the sums' barriers)
    v0 = smp_get(mine + t);
    vk = smp_get(mine + G + t);
    chunk[t] = v0;
  }
  const u64 mass0 = smp_sum<NT>(v0, red), massk = smp_sum<NT>(vk, red);
  u64 total;
  const int last = smp_find<NT>(r, s, tab, lds.f, (int)min(n, (unsigned)SMP_LIST), c, mass0, massk, all, total, red);
  const u64 thr = last >= 0 ? lds.f.ord[last] : lds.f.ord[0] - 1;
  smp_finish(a, st, gr, smp_token(r, k, s, tab, lds.f, last, thr, total, mass0, chunk, red), thr, total);
}

__global__ __launch_bounds__(SMP_NT) void k_sample_probs(SampleArgs a, SmpWork k) {
  constexpr int NT = SMP_NT;
  __shared__ double tab[128];
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x;
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  SmpRow r = smp_row(a, gr);
  const SmpSet s = smp_set(a, gr);
  smp_table(tab);
  const u64 thr = k.state[row].thr, total = k.state[row].total, top = smp_least<NT>(t < k.G ? k.top[(long)row * k.G + t] : ~0ull, red);
  r.m = smp_value((uint32_t)(top >> 32));
  r.inv_t = 1.0 / s.t;
  smp_probs<NT>(a, r, gr, lo, hi, thr, total, tab);
}

// Chunks of a row (1: a workgroup per row): some 1024 workgroups in all, of 4096 entries or a little less at the least.
static int smp_chunks(const Ctx &c, long rows, int V) {
  if (V <= 32 * SMP_ONE || rows >= c.num_cu) return 1;
  return (int)std::max(2L, std::min({(long)SMP_GMAX, (V + 4095L) / 4096, 4L * c.num_cu / rows}));
}
static size_t smp_carve(const Ctx &c, size_t n, int V, char *base, SmpWork *k) {
  const long rows = std::min<long>(n, CNT_N), G = smp_chunks(c, n, V);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *p = base + at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  SmpWork w{};
  w.G = (int)G;
  if (G > 1) {
    w.len = (int)(((V + G - 1) / G + 3) & ~3L);
    w.top = (u64 *)take(rows * G * 8);
    w.cert = (u64 *)take(rows * 2 * G * 8);
    w.part = (unsigned *)take(rows * G * SMP_PARTS * 4);
    w.state = (SmpState *)take(rows * sizeof(SmpState));
    w.list = (u64 *)take(rows * SMP_LIST * 8);
    w.hist = (u64 *)take(rows * G * SMP_NB * 8);
  }
  w.arrive = c.d_cnt;
  if (k) *k = w;
  return at;
}
size_t sample_scratch(const Ctx &c, size_t n, int V) { return smp_carve(c, n, V, nullptr, nullptr); }

hipError_t launch_sample(const Ctx &c, SampleArgs a, size_t n, void *scratch) {
  int bits = 0;
  while (bits < 31 && (1L << bits) < a.V) bits++;
  a.S = std::min(45, 62 - bits);
  SmpWork k;
  smp_carve(c, n, a.V, (char *)scratch, &k);
  // a bucket's count is at most 2^bits, its mass V of 2^(S - sh)
  k.un.cb = bits + 1;
  k.un.sh = a.S - std::min(30, 63 - k.un.cb - bits);
  if (k.G == 1) {
    launch_k(c, k_sample_one, dim3((unsigned)n), dim3(SMP_ONE), a, k.un);
    return hipGetLastError();
  }
  // (fewer rows than CUs, and so than counters)
  const dim3 grid(k.G, (unsigned)n), block(SMP_NT);
  launch_k(c, k_sample_top, grid, block, a, k);
  launch_k(c, k_sample_cut, grid, block, a, k);
  if (a.top_k || a.top_p || a.min_p) launch_k(c, k_sample_list, grid, block, a, k);
  if (a.probs) launch_k(c, k_sample_probs, grid, block, a, k);
  return hipGetLastError();
}

}  // namespace rbt

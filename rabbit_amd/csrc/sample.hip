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
  double m, inv_t;
  __device__ __forceinline__ float at(int i) const {
    return x16 ? rbt_bf16_f32(((const uint16_t *)x)[i]) : ((const float *)x)[i];
  }
};

// exp(y), y <= 0, times 2^sh: 2^(k/32) from a table times a Taylor polynomial of what is left (at most ln 2 / 64: the
// sixth term is below 2^-48).
__device__ __forceinline__ void smp_table(double *tab) {
  if (threadIdx.x < 32) tab[threadIdx.x] = exp2((double)threadIdx.x * 0.03125);
}
__device__ __forceinline__ double smp_exp(double y, int sh, const double *tab) {
  const double k = rint(y * 46.16624130844683);
  const double r = fma(k, -7.247021293269686e-19, fma(k, -0.02166084939249829, y));
  const int n = (int)k;
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return ldexp(tab[n & 31] * p, (n >> 5) + sh);
}
__device__ __forceinline__ double smp_weight(const SmpRow &r, float x, const double *tab) {
  const double y = ((double)x - r.m) * r.inv_t;
  return y > -690.0 ? smp_exp(y, 0, tab) : 0.0;
}
// The weight in units of 2^-S, to the nearest (w <= 1, S <= 45).
__device__ __forceinline__ u64 smp_round(double w) {
  return (u64)__double_as_longlong(w + 0x1p52) & 0xfffffffffffffull;
}
__device__ __forceinline__ u64 smp_mass(const SmpRow &r, float x, const double *tab) {
  const double y = ((double)x - r.m) * r.inv_t;
  return y > -34.0 ? smp_round(smp_exp(y, r.S, tab)) : 0;  // (e^-34 is below 2^-46)
}

// The bucket of a logit: 24ths of (m - x) / t, never falling along the order; the last holds all from 21.3 on.
__device__ __forceinline__ float smp_scale(double t) { return fminf(24.0f / (float)t, 1e30f); }
__device__ __forceinline__ int smp_bucket(float m, float x, float cf) {
  return x > -INFINITY ? (int)fminf((m - x) * cf, 511.0f) : 511;
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

// A row is cut in G chunks, a workgroup each, over three launches (no workgroup waits for another; the last one of a row
// to arrive goes on):
//   k_sample_top   the chunk's first entry of the order, and the largest logits of 64 parts of it
//   k_sample_cut   with the row's m. top-k of up to 512: at least k entries are as large as the k-th of all chunks' part
//                  maxima, and few more, so those go to a list, and the last workgroup sorts it, finds every threshold in it
//                  and draws. Else the counts and rounded masses of 512 buckets of (m - x) / t, of which the last workgroup
//                  takes those where the thresholds may lie; without thresholds it draws.
//   k_sample_list  the entries of those buckets as a list, the masses of those before; the last workgroup goes on as above,
//                  and draws the chunk by the chunks' masses, then the entry.
//   k_sample_probs the probabilities, where they are wanted.
// A row whose list would be longer than SMP_LIST (thousands of equal logits; a temperature that leaves all mass in one
// bucket) is taken by one workgroup digit by digit. Rows of up to SMP_LIST entries are lists as they are.
constexpr int SMP_NT = 256, SMP_NB = 512, SMP_LIST = 2048, SMP_GMAX = 32, SMP_PARTS = 64, SMP_KMAX = 512;
enum { SMP_DONE = 0, SMP_FIND = 1, SMP_SLOW = 2 };

struct SmpState {  // a row between launches
  u64 thr, total;  // kept: entries up to thr, their mass (0: none, token -1)
  int mode, b0, b1, kb;  // listed: buckets b0 .. b1, and kb
  int cnt0, cntk, n1;  // entries before b0, before kb, in b0 .. b1
  unsigned n;          // list entries so far
};
struct SmpWork {  // scratch of up to CNT_N rows
  u64 *top, *hist, *cert, *list;  // [rows, G], [rows, G, SMP_NB], [rows, 2, G], [rows, SMP_LIST]
  unsigned *part;                 // [rows, G, SMP_PARTS]
  SmpState *state;
  unsigned *arrive;               // arrival counters, left at 0
  int G, len, row0;               // chunks of a row, entries of a chunk (a multiple of 4), first row
  int cb, sh;                     // buckets: count in the low cb bits, above them mass / 2^sh
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
    last = 1;
    if (k.G > 1) {
      last = __hip_atomic_fetch_add(k.arrive + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (unsigned)k.G;
      if (last) __hip_atomic_store(k.arrive + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  return last;
}

// Entries lo .. hi - 1 of the row, four in a row at a time per thread: f(first index, four values), with -inf for those
// outside [lo, hi). The fours begin at aligned places; UN loads of a thread are on their way at once.
template <int UN, typename F>
__device__ __forceinline__ void smp_each(const SmpRow &r, int lo, int hi, F f) {
  const int pad = (int)(((uintptr_t)r.x >> (r.x16 ? 1 : 2)) + lo) & 3;
  for (int i0 = lo - pad + 4 * threadIdx.x; i0 < hi; i0 += UN * 4 * SMP_NT) {
    float x[UN][4];
#pragma unroll
    for (int k = 0; k < UN; k++) {
      const int i = i0 + k * 4 * SMP_NT;
      if (i >= lo && i + 4 <= hi) {
        if (r.x16) {
          const uint2 v = *(const uint2 *)((const uint16_t *)r.x + i);
          x[k][0] = __uint_as_float(v.x << 16), x[k][1] = __uint_as_float(v.x & 0xffff0000u);
          x[k][2] = __uint_as_float(v.y << 16), x[k][3] = __uint_as_float(v.y & 0xffff0000u);
        } else {
          const float4 v = *(const float4 *)((const float *)r.x + i);
          x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[k][e] = i + e >= lo && i + e < hi ? r.at(i + e) : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < UN; k++)
      if (i0 + k * 4 * SMP_NT < hi) f(i0 + k * 4 * SMP_NT, x[k]);
  }
}

__device__ __forceinline__ u64 smp_ord(float x, int i) { return (u64)smp_key(x) << 32 | (unsigned)i; }

__device__ __forceinline__ SmpRow smp_row(const SampleArgs &a, int row) {
  return {(const char *)a.x + (long)row * a.stride * (a.x16 ? 2 : 4), a.x16, a.V, a.S, 0.0, 0.0};
}

// The workgroup's sum (in every thread), its inclusive scan, its least.
struct SmpRed {
  u64 w[SMP_NT / 64];
};
__device__ __forceinline__ u64 smp_sum(u64 v, SmpRed &red) {
  v = smp_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < SMP_NT / 64; i++) v += red.w[i];
  return v;
}
__device__ __forceinline__ u64 smp_scan(u64 v, u64 &all, SmpRed &red) {
  v = smp_wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int i = 0; i < SMP_NT / 64; i++) {
    if (i < (int)(threadIdx.x >> 6)) v += red.w[i];
    all += red.w[i];
  }
  return v;
}
__device__ __forceinline__ u64 smp_least(u64 v, SmpRed &red) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = min(v, (u64)__shfl_xor((long long)v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red.w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red.w[0];
#pragma unroll
  for (int i = 1; i < SMP_NT / 64; i++) v = min(v, red.w[i]);
  return v;
}

__global__ __launch_bounds__(SMP_NT) void k_sample_top(SampleArgs a, SmpWork k) {
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  const SmpRow r = smp_row(a, k.row0 + row);
  float best = -INFINITY;  // (the first of equal ones: indexes rise)
  int at = 0;
  smp_each<8>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (x[e] > best) best = x[e], at = i + e;
  });
  const u64 mine = best > -INFINITY ? smp_ord(best, at) : ~0ull;
  unsigned key = (unsigned)(mine >> 32);
  key = min(key, (unsigned)__shfl_xor((int)key, 1, 64));
  key = min(key, (unsigned)__shfl_xor((int)key, 2, 64));
  const long chunk = (long)row * k.G + g;
  if (t % 4 == 0) k.part[chunk * SMP_PARTS + t / 4] = key;
  const u64 top = smp_least(mine, red);
  if (t == 0) {
    k.top[chunk] = top;
    if (g == 0) k.state[row].n = 0;
  }
}

// The least index in [lo, hi) at which the running mass of entries up to thr passes `left`; every wave first sums its
// quarter, then the workgroup scans the one where it passes.
__device__ __forceinline__ int smp_draw(const SmpRow &r, const double *tab, int lo, int hi, u64 thr, double left, SmpRed &red) {
  __shared__ int found;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, part = ((hi - lo + 3) / 4 + 3) & ~3;
  u64 v = 0;
  for (int i = lo + w * part + lane; i < min(hi, lo + (w + 1) * part); i += 64) {
    const float x = r.at(i);
    if (smp_ord(x, i) <= thr) v += smp_mass(r, x, tab);
  }
  v = smp_wave_sum(v);
  __syncthreads();
  if (lane == 0) red.w[w] = v;
  if (t == 0) found = INT32_MAX;
  __syncthreads();
  u64 run = 0;
  int q = -1;
  for (int i = 0; i < SMP_NT / 64; i++) {
    if (q < 0 && (double)(run + red.w[i]) > left) q = i;
    if (q < 0) run += red.w[i];
  }
  if (q < 0) return -1;  // (u below 1 times the whole is below the whole)
  const int end = min(hi, lo + (q + 1) * part);
  for (int i0 = lo + q * part; i0 < end; i0 += 4 * SMP_NT) {
    u64 mine[4], sum = 0, all;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = i0 + 4 * t + e;
      const float x = i < end ? r.at(i) : -INFINITY;
      mine[e] = i < end && smp_ord(x, i) <= thr ? smp_mass(r, x, tab) : 0;
      sum += mine[e];
    }
    u64 at = run + smp_scan(sum, all, red) - sum;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      at += mine[e];
      if ((double)at > left) {
        atomicMin(&found, i0 + 4 * t + e);
        break;
      }
    }
    run += all;
    __syncthreads();
    if (found != INT32_MAX) return found;
  }
  return -1;
}

// The chunk where the running mass passes `left`, and the mass before it.
__device__ __forceinline__ int smp_chunk(const u64 *mass, int G, double left, u64 &before) {
  before = 0;
  for (int g = 0; g < G; g++) {
    if ((double)(before + mass[g]) > left) return g;
    before += mass[g];
  }
  return -1;
}

// ---- one workgroup for a whole row ---------------------------------------------------------------
struct SmpSlow {
  u64 mass[256];
  unsigned cnt[256];
  u64 before, nbefore;
  int digit;
};
// The first `ord` of the row at which the running count of the order reaches k (k > 0) or, among entries up to `most`, the
// running mass reaches `target`; and the mass up to it.
__device__ u64 smp_select(const SmpRow &r, const double *tab, SmpSlow &sh, unsigned k, double target, u64 most, u64 &mass_to) {
  const int t = threadIdx.x;
  u64 pre = 0, before = 0;
  unsigned nbefore = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (shift == 24) continue;  // indexes are below 2^24
    for (int i = t; i < 256; i += SMP_NT) sh.mass[i] = 0, sh.cnt[i] = 0;
    __syncthreads();
    for (int i = t; i < r.V; i += SMP_NT) {
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
      int d = 0, held = 0;  // held: the last digit with any entry
      u64 mb = before, hm = before;
      unsigned nb = nbefore, hn = nbefore;
      for (; d < 256; d++) {
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

struct SmpFind {
  u64 ord[SMP_LIST], run[SMP_LIST];  // the list in order, its masses summed up to each
};
union SmpLds {
  SmpFind f;
  SmpSlow slow;
  struct {
    u64 hist[SMP_NB + 1];
    unsigned key[SMP_GMAX * SMP_PARTS];
  } cut;
};

// The list's n entries (in lds.f.ord, any order) put in order, the thresholds found among the first n1 of them, which
// begin after cnt0 entries and a mass of mass0; and top-k's entry, where it lies beyond (n1 and cntk, massk) or
// among them. Returns the last kept entry (-1: none of the list), with kept mass `total`.
__device__ int smp_find(const SmpRow &r, const SmpSet &s, const double *tab, SmpFind &f, int n, int n1, bool by_k, bool beyond, int cnt0,
                        int cntk, u64 mass0, u64 massk, u64 whole, u64 &total, SmpRed &red) {
  __shared__ int ip, im;
  const int t = threadIdx.x;
  int n2 = 2;
  while (n2 < n) n2 *= 2;
  for (int i = n + t; i < n2; i += SMP_NT) f.ord[i] = ~0ull;
  if (t == 0) ip = n1, im = -1;
  __syncthreads();
  for (int len = 2; len <= n2; len *= 2)  // bitonic, padded to a power of two
    for (int d = len / 2; d; d /= 2) {
      for (int i = t; i < n2 / 2; i += SMP_NT) {
        const int x = (i / d) * 2 * d + i % d, y = x + d;
        const u64 p = f.ord[x], q = f.ord[y];
        if ((p > q) == !(x & len)) f.ord[x] = q, f.ord[y] = p;
      }
      __syncthreads();
    }
  u64 run = 0;
  for (int i0 = 0; i0 < n; i0 += SMP_NT) {
    const int i = i0 + t;
    const float x = i < n ? smp_value((uint32_t)(f.ord[i] >> 32)) : -INFINITY;
    u64 all;
    const u64 up = run + smp_scan(smp_mass(r, x, tab), all, red);
    if (i < n) f.run[i] = up;
    if (i < n1 && (s.min_p == 0.0 || smp_weight(r, x, tab) >= s.min_p)) atomicMax(&im, i);
    run += all;
  }
  __syncthreads();
  int last = n1 - 1;
  u64 left = whole == ~0ull ? run : whole;  // the mass that top-k leaves (~0: the list is all there is)
  if (by_k && !beyond) {
    last = s.k - 1 - cnt0;
    left = mass0 + f.run[last];
  } else if (by_k) {
    left = massk + f.run[n1 + s.k - 1 - cntk] - (n1 ? f.run[n1 - 1] : 0);
  }
  if (s.top_p < 1.0) {
    const double target = s.top_p * (double)left;
    for (int i = t; i < n1; i += SMP_NT)
      if ((double)(mass0 + f.run[i]) >= target) atomicMin(&ip, i);
    __syncthreads();
    last = min(last, ip);
  }
  last = min(last, min(im, n1 - 1));
  total = mass0 + (last >= 0 ? f.run[last] : 0);
  return last;
}

// Where nothing is kept before the list: the draw among its entries up to `last`, in the order of their indexes.
__device__ int smp_draw_list(const SmpFind &f, int last, double left) {
  __shared__ u64 first;
  const int t = threadIdx.x;
  if (t == 0) first = ~0ull;
  __syncthreads();
  for (int i = t; i <= last; i += SMP_NT) {
    const unsigned at = (unsigned)f.ord[i];
    u64 run = 0, before = 0;
    for (int j = 0; j <= last; j++) {
      const u64 up = f.run[j];
      if ((unsigned)f.ord[j] <= at) run += up - before;
      before = up;
    }
    if ((double)run > left) atomicMin(&first, (u64)at);
  }
  __syncthreads();
  return first == ~0ull ? -1 : (int)first;
}

// The token: of the list up to `last`, and of what lies before it (mass0, by chunks in `chunk`).
__device__ int smp_token(const SmpRow &r, const SmpWork &k, const SmpSet &s, const double *tab, const SmpFind &f, int last, u64 thr,
                         u64 total, u64 mass0, u64 *chunk, SmpRed &red) {
  const double left = s.u * (double)total;
  if (mass0 == 0 && last < 256) return smp_draw_list(f, last, left);
  for (int i = threadIdx.x; i <= last; i += SMP_NT) {
    const u64 v = f.run[i] - (i ? f.run[i - 1] : 0);
    if (v) atomicAdd(&chunk[(int)((unsigned)f.ord[i] / (unsigned)k.len)], v);
  }
  __syncthreads();
  u64 before;
  const int ch = smp_chunk(chunk, k.G, left, before);
  return ch < 0 ? -1 : smp_draw(r, tab, ch * k.len, min(r.V, (ch + 1) * k.len), thr, left - (double)before, red);
}

// The k-th smallest of n keys in LDS, bit by bit.
__device__ unsigned smp_kth(const unsigned *key, int n, int k, SmpRed &red) {
  const int t = threadIdx.x;
  unsigned mine[SMP_GMAX * SMP_PARTS / SMP_NT], lo = 0;
#pragma unroll
  for (int i = 0; i < SMP_GMAX * SMP_PARTS / SMP_NT; i++) mine[i] = t + i * SMP_NT < n ? key[t + i * SMP_NT] : 0xffffffffu;
  // the largest value that fewer than k keys are below
  for (int b = 31; b >= 0; b--) {
    const unsigned x = lo | 1u << b;
    int c = 0;
#pragma unroll
    for (int i = 0; i < SMP_GMAX * SMP_PARTS / SMP_NT; i++) c += __popcll(__ballot(mine[i] < x));
    unsigned *cnt = (unsigned *)red.w + (b & 1) * (SMP_NT / 64);  // (two sets in turn: one barrier a bit)
    if ((t & 63) == 0) cnt[t >> 6] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int i = 0; i < SMP_NT / 64; i++) c += cnt[i];
    if (c < k) lo = x;
  }
  __syncthreads();
  return lo;
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
template <int UN, typename F, typename H>
__device__ bool smp_gather(const SmpRow &r, const SmpWork &k, SmpState &st, int row, int lo, int hi, SmpFind &f, unsigned &n, F take, H then) {
  __shared__ unsigned here, base;
  const int t = threadIdx.x;
  if (t == 0) here = 0;
  __syncthreads();
  smp_each<UN>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (take(x[e]) && i + e >= lo && i + e < hi) {
        const unsigned at = atomicAdd(&here, 1u);
        if (at < SMP_LIST) f.ord[at] = smp_ord(x[e], i + e);
      }
  });
  __syncthreads();
  n = here;
  then();
  if (k.G == 1) return true;
  u64 *list = k.list + (long)row * SMP_LIST;
  if (t == 0 && n) base = __hip_atomic_fetch_add(&st.n, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (unsigned i = t; i < min(n, (unsigned)SMP_LIST); i += SMP_NT)
    if (base + i < SMP_LIST) smp_put(list + base + i, f.ord[i]);
  if (!smp_last(k, row)) return false;
  n = smp_get(&st.n);
  for (unsigned i = t; i < min(n, (unsigned)SMP_LIST); i += SMP_NT) f.ord[i] = smp_get(list + i);
  __syncthreads();
  return true;
}

__global__ __launch_bounds__(SMP_NT) void k_sample_cut(SampleArgs a, SmpWork k) {
  __shared__ SmpLds lds;
  __shared__ double tab[32];
  __shared__ u64 cert[SMP_GMAX];
  __shared__ SmpRed red;
  __shared__ int kb_s, p0_s, p1_s, held_s;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x, G = k.G;
  SmpRow r = smp_row(a, gr);
  SmpSet s;
  const u64 top1 = t < G ? k.top[(long)row * G + t] : ~0ull;
  const bool ok = smp_set(a, gr, s);
  smp_table(tab);
  const u64 top = smp_least(top1, red);
  const float m = smp_value((uint32_t)(top >> 32));
  SmpState &st = k.state[row];
  const bool none = !ok || top == ~0ull || !(fabsf(m) < INFINITY);
  if (none || s.k == 1) {  // nothing to draw from, or one entry
    if (g == 0) {
      if (!ok && t == 0) *a.bad = 1;
      smp_finish(a, st, gr, none ? -1 : (int)(unsigned)top, top, none ? 0 : 1ull << a.S);
    }
    return;
  }
  r.m = m;
  r.inv_t = 1.0 / s.t;
  const bool by_k = s.k > 0 && s.k < a.V, by_p = s.top_p < 1.0, by_m = s.min_p > 0.0;
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len), np = G * SMP_PARTS;
  const bool whole = a.V <= SMP_LIST;
  if (whole || (by_k && s.k <= min(SMP_KMAX, np))) {
    unsigned most = ~0u, n;
    if (!whole) {
      for (int i = t; i < np; i += SMP_NT) lds.cut.key[i] = k.part[(long)row * np + i];
      __syncthreads();
      most = smp_kth(lds.cut.key, np, s.k, red);
    }
    if (!smp_gather<8>(r, k, st, row, lo, hi, lds.f, n, [&](float x) { return smp_key(x) <= most; }, [] {})) return;
    if (n <= SMP_LIST) {
      u64 total;
      const int last = smp_find(r, s, tab, lds.f, n, n, by_k, false, 0, 0, 0, 0, ~0ull, total, red);
      if (t < G) cert[t] = 0;
      __syncthreads();
      const u64 thr = lds.f.ord[last];
      smp_finish(a, st, gr, smp_token(r, k, s, tab, lds.f, last, thr, total, 0, cert, red), thr, total);
    } else if (t == 0) {
      st.mode = SMP_SLOW;
    }
    return;
  }
  for (int i = t; i <= SMP_NB; i += SMP_NT) lds.cut.hist[i] = 0;
  __syncthreads();
  const float cf = smp_scale(s.t);
  u64 sum = 0;
  const bool any = by_k || by_p || by_m;
  smp_each<4>(r, lo, hi, [&](int, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const u64 v = smp_mass(r, x[e], tab);
      sum += v;
      const int b = smp_bucket(m, x[e], cf);
      if (any && b < SMP_NB - 1) atomicAdd(&lds.cut.hist[b], (v >> k.sh) << k.cb | 1);  // (the last is what is left)
    }
  });
  sum = smp_sum(sum, red);
  u64 *mine = k.cert + (long)row * 2 * G;
  if (t == 0) G > 1 ? smp_put(mine + g, sum) : (void)(cert[0] = sum);
  const long at = (long)row * G * SMP_NB;
  if (G > 1 && any)
    for (int b = t; b < SMP_NB; b += SMP_NT) smp_put(k.hist + at + (long)g * SMP_NB + b, lds.cut.hist[b]);
  if (!smp_last(k, row)) return;
  if (G > 1 && t < G) cert[t] = smp_get(mine + t);
  // the row's buckets, two a thread, and what lies before each
  u64 v[2] = {lds.cut.hist[2 * t], lds.cut.hist[2 * t + 1]};
  if (G > 1 && any) {
    v[0] = v[1] = 0;
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
  u64 all = 0, before;
  for (int j = 0; j < G; j++) all += cert[j];
  if (!any) {
    const double left = s.u * (double)all;
    const int ch = smp_chunk(cert, G, left, before);
    const int tok = ch < 0 ? -1 : smp_draw(r, tab, ch * k.len, min(a.V, (ch + 1) * k.len), ~0ull, left - (double)before, red);
    smp_finish(a, st, gr, tok, ~0ull, all);
    return;
  }
  u64 rest;
  const u64 upto = smp_scan(v[0] + v[1], rest, red);
  __syncthreads();
  u64 *hist = lds.cut.hist;
  hist[2 * t + 1] = upto - v[1];
  hist[2 * t] = upto - v[1] - v[0];
  if (t == 0) {
    hist[SMP_NB] = rest;
    kb_s = p0_s = p1_s = SMP_NB;
    held_s = 0;
  }
  __syncthreads();
  const unsigned one = (1u << k.cb) - 1;
  auto cnt = [&](int b) { return b == SMP_NB ? (unsigned)a.V : (unsigned)hist[b] & one; };
  // the mass before bucket b, in units of 2^(sh - S): at least, and below
  auto low = [&](int b) { return (double)(hist[b] >> k.cb); };
  auto high = [&](int b) { return b == SMP_NB ? ldexp((double)all, -k.sh) + 1.0 : low(b) + (double)cnt(b); };
  if (by_k)
    for (int e = 0; e < 2; e++)
      if (cnt(2 * t + e) < (unsigned)s.k && cnt(2 * t + e + 1) >= (unsigned)s.k) kb_s = 2 * t + e;
  __syncthreads();
  const int kb = kb_s;
  if (by_p) {  // of the mass that top-k leaves
    const double whole0 = by_k ? low(kb) : ldexp((double)all, -k.sh), whole1 = by_k ? high(kb + 1) : whole0;
    for (int e = 0; e < 2; e++) {
      if (high(2 * t + e + 1) >= s.top_p * whole0) atomicMin(&p0_s, 2 * t + e);
      if (low(2 * t + e + 1) >= s.top_p * whole1) atomicMin(&p1_s, 2 * t + e);
    }
  }
  __syncthreads();
  int b0 = by_p ? min(p0_s, kb) : kb, b1 = by_p ? min(min(p1_s, kb), SMP_NB - 1) : kb;
  if (by_m) {  // the bucket of the least weight, and its neighbours for their rounding
    const int b = (int)fmin(-log(s.min_p) * 24.0, 600.0);
    b0 = min(b0, max(b - 1, 0));
    b1 = min(b1, min(b + 1, SMP_NB - 1));
  }
  b0 = min(b0, SMP_NB - 1);
  if (cnt(b1 + 1) == cnt(b0)) {  // no entry near min_p: the threshold is the last of the bucket before
    for (int e = 0; e < 2; e++)
      if (2 * t + e < b0 && cnt(2 * t + e + 1) > cnt(2 * t + e)) atomicMax(&held_s, 2 * t + e);
    __syncthreads();
    b0 = held_s;  // (the largest logit is in bucket 0)
  }
  if (t == 0) {
    const unsigned n1 = cnt(b1 + 1) - cnt(b0), nk = by_k && kb > b1 ? cnt(kb + 1) - cnt(kb) : 0;
    st.mode = n1 + nk > SMP_LIST ? SMP_SLOW : SMP_FIND;
    st.total = all;
    st.b0 = b0;
    st.b1 = b1;
    st.kb = by_k ? kb : -1;
    st.n1 = (int)n1;
    st.cnt0 = (int)cnt(b0);
    st.cntk = by_k ? (int)cnt(kb) : 0;
    st.n = 0;
  }
}

__global__ __launch_bounds__(SMP_NT) void k_sample_list(SampleArgs a, SmpWork k) {
  __shared__ SmpLds lds;
  __shared__ double tab[32];
  __shared__ u64 chunk[SMP_GMAX];
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x, G = k.G;
  SmpState &st = k.state[row];
  const int mode = st.mode;
  if (mode == SMP_DONE || (mode == SMP_SLOW && g)) return;
  SmpRow r = smp_row(a, gr);
  SmpSet s;
  smp_set(a, gr, s);
  smp_table(tab);
  const u64 top = smp_least(t < G ? k.top[(long)row * G + t] : ~0ull, red);
  const float m = smp_value((uint32_t)(top >> 32));
  r.m = m;
  r.inv_t = 1.0 / s.t;
  const bool by_k = s.k > 0 && s.k < a.V, by_p = s.top_p < 1.0, by_m = s.min_p > 0.0;
  if (mode == SMP_SLOW) {
    u64 thr = ~0ull, mass = 0, total = 0, last = 0;
    if (by_k) {
      thr = smp_select(r, tab, lds.slow, s.k, 0.0, thr, mass);
    } else if (by_p) {
      for (int i = t; i < a.V; i += SMP_NT) mass += smp_mass(r, r.at(i), tab);
      mass = smp_sum(mass, red);
    }
    if (by_p) thr = smp_select(r, tab, lds.slow, 0, s.top_p * (double)mass, thr, mass);
    for (int i = t; i < a.V; i += SMP_NT) {
      const float x = r.at(i);
      const u64 o = smp_ord(x, i);
      if (o <= thr && (!by_m || smp_weight(r, x, tab) >= s.min_p)) {
        total += smp_mass(r, x, tab);
        last = max(last, o);
      }
    }
    total = smp_sum(total, red);
    if (by_m) thr = ~smp_least(~last, red);  // the last that is heavy enough
    smp_finish(a, st, gr, smp_draw(r, tab, 0, a.V, thr, s.u * (double)total, red), thr, total);
    return;
  }
  const int b0 = st.b0, b1 = st.b1, kb = st.kb, n1 = st.n1, cnt0 = st.cnt0, cntk = st.cntk;
  const u64 all = st.total;
  const bool beyond = by_k && kb > b1;
  const float cf = smp_scale(s.t);
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  // the masses before the listed buckets, and before top-k's where that is another
  u64 sum0 = 0, sumk = 0, *mine = k.cert + (long)row * 2 * G;
  unsigned n;
  const bool last_one = smp_gather<8>(r, k, st, row, lo, hi, lds.f, n, [&](float x) {
    const int b = smp_bucket(m, x, cf);
    if (b < b0 || (beyond && b < kb)) {
      const u64 v = smp_mass(r, x, tab);
      if (b < b0) sum0 += v;
      sumk += v;
    }
    return (b >= b0 && b <= b1) || b == kb;
  }, [&]() {
    sum0 = smp_sum(sum0, red);
    sumk = smp_sum(sumk, red);
    if (t == 0) smp_put(mine + g, sum0), smp_put(mine + G + g, sumk);
  });
  if (!last_one) return;
  u64 v0 = 0, vk = 0;
  if (t < G) {  // (the chunks' masses are read by all after the sums' barriers)
    v0 = smp_get(mine + t);
    vk = smp_get(mine + G + t);
    chunk[t] = v0;
  }
  const u64 mass0 = smp_sum(v0, red), massk = smp_sum(vk, red);
  u64 total;
  const int last = smp_find(r, s, tab, lds.f, (int)min(n, (unsigned)SMP_LIST), n1, by_k, beyond, cnt0, cntk, mass0, massk, all, total, red);
  const u64 thr = last >= 0 ? lds.f.ord[last] : lds.f.ord[0] - 1;
  const int tok = smp_token(r, k, s, tab, lds.f, last, thr, total, mass0, chunk, red);
  smp_finish(a, st, gr, tok, thr, total);
}

typedef float smp_f4 __attribute__((ext_vector_type(4), aligned(4)));  // (stores of four words want four bytes' alignment)
__global__ __launch_bounds__(SMP_NT) void k_sample_probs(SampleArgs a, SmpWork k) {
  __shared__ double tab[32];
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x;
  SmpRow r = smp_row(a, gr);
  SmpSet s;
  smp_set(a, gr, s);
  smp_table(tab);
  const u64 top = smp_least(t < k.G ? k.top[(long)row * k.G + t] : ~0ull, red), thr = k.state[row].thr, total = k.state[row].total;
  r.m = smp_value((uint32_t)(top >> 32));
  r.inv_t = 1.0 / s.t;
  const double scale = total ? ldexp(1.0, a.S) / (double)total : 0.0;
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  float *to = a.probs + (long)gr * a.V;
  smp_each<4>(r, lo, hi, [&](int i, const float (&x)[4]) {
    float p[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
      p[e] = total && smp_ord(x[e], i + e) <= thr ? (float)(smp_weight(r, x[e], tab) * scale) : 0.0f;
    if (i >= lo && i + 4 <= hi) {
      *(smp_f4 *)(to + i) = smp_f4{p[0], p[1], p[2], p[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (i + e >= lo && i + e < hi) to[i + e] = p[e];
    }
  });
}

// Chunks of a row: some 1024 workgroups in all, of at least 2048 entries each.
static int smp_chunks(const Ctx &c, long rows, int V) {
  return (int)std::max(1L, std::min({(long)SMP_GMAX, (V + 2047L) / 2048, 4L * c.num_cu / rows}));
}
static size_t smp_carve(const Ctx &c, size_t n, int V, char *base, SmpWork *k) {
  const long rows = std::min<long>(n, CNT_N), G = smp_chunks(c, rows, V);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *p = base + at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  SmpWork w{};
  w.G = (int)G;
  w.len = (int)(((V + G - 1) / G + 3) & ~3L);
  w.top = (u64 *)take(rows * G * 8);
  w.cert = (u64 *)take(rows * 2 * G * 8);
  w.part = (unsigned *)take(rows * G * SMP_PARTS * 4);
  w.state = (SmpState *)take(rows * sizeof(SmpState));
  w.list = (u64 *)take(G > 1 ? rows * SMP_LIST * 8 : 0);
  w.hist = (u64 *)take(G > 1 ? rows * G * SMP_NB * 8 : 0);
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
  k.cb = bits + 1;
  k.sh = a.S - std::min(30, 63 - k.cb - bits);
  for (size_t r0 = 0; r0 < n; r0 += CNT_N) {
    k.row0 = (int)r0;
    const int rows = (int)std::min<size_t>(CNT_N, n - r0);
    const dim3 grid(k.G, rows), block(SMP_NT);
    launch_k(c, k_sample_top, grid, block, a, k);
    launch_k(c, k_sample_cut, grid, block, a, k);
    if (a.V > SMP_LIST && (a.top_k || a.top_p || a.min_p)) launch_k(c, k_sample_list, grid, block, a, k);
    if (a.probs) launch_k(c, k_sample_probs, grid, block, a, k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace rbt

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

// The bucket of a logit: sixteenths of (m - x) / t, never falling along the order.
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
//   k_sample_top   the chunk's first entry of the order
//   k_sample_hist  with the row's m, the counts and masses of 512 buckets of (m - x) / t, a sixteenth wide (the last is
//                  all from 32 on). The last workgroup sums the chunks' and finds the buckets where the
//                  thresholds lie; without thresholds it draws.
//   k_sample_list  the entries of those buckets into a list (at most SMP_LIST). The last workgroup sorts it, finds
//                  the thresholds in it, and draws: the chunk by the chunks' masses, then the entry. A row whose list
//                  would be longer (thousands of equal logits; a temperature that leaves all mass in one bucket) is taken by one
//                  workgroup digit by digit.
//   k_sample_probs the probabilities, where they are wanted.
constexpr int SMP_NT = 256, SMP_NB = 512, SMP_LIST = 2048, SMP_GMAX = 64;
enum { SMP_DONE = 0, SMP_FIND = 1, SMP_SLOW = 2 };

struct SmpState {  // a row between launches
  u64 thr, total;  // kept: entries up to thr, their mass (0: none, token -1)
  u64 mass0, massk;  // mass before bucket b0, before bucket kb
  int mode, b0, b1, kb;  // listed: buckets b0 .. b1, and kb
  int cnt0, cntk, n1;  // entries before b0, before kb, in b0 .. b1
  unsigned n;          // list entries so far
};
struct SmpWork {  // scratch of up to CNT_N rows
  u64 *top, *mass, *cert, *list;  // [rows, G], [rows, G, SMP_NB], [rows, G], [rows, SMP_LIST]
  unsigned *cnt;                  // [rows, G, SMP_NB]
  SmpState *state;
  unsigned *arrive;               // arrival counters, left at 0
  int G, len, row0;               // chunks of a row, entries of a chunk (a multiple of 4), first row
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

// Entries lo .. hi - 1 of the row, four in a row at a time per thread: f(first index, four values); past hi the values
// are -inf. UN loads of a thread are on their way at once.
template <bool QUADS, int UN, typename F>
__device__ __forceinline__ void smp_each(const SmpRow &r, int lo, int hi, F f) {
  for (int i0 = lo + 4 * threadIdx.x; i0 < hi; i0 += UN * 4 * SMP_NT) {
    float x[UN][4];
#pragma unroll
    for (int k = 0; k < UN; k++) {
      const int i = i0 + k * 4 * SMP_NT;
      if (QUADS && i + 4 <= hi) {
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
        for (int e = 0; e < 4; e++) x[k][e] = i + e < hi ? r.at(i + e) : -INFINITY;
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

template <bool QUADS>
__global__ __launch_bounds__(SMP_NT) void k_sample_top(SampleArgs a, SmpWork k) {
  __shared__ SmpRed red;
  const int g = blockIdx.x, row = blockIdx.y, lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  const SmpRow r = smp_row(a, k.row0 + row);
  u64 top = ~0ull;
  smp_each<QUADS, 8>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) top = min(top, smp_ord(x[e], i + e));
  });
  top = smp_least(top, red);
  if (threadIdx.x == 0) k.top[(long)row * k.G + g] = top;
}

// The least index in [lo, hi) at which the running mass of entries up to thr passes `left`; every wave first sums its
// quarter, then the workgroup scans the one where it passes.
template <bool QUADS>
__device__ int smp_draw(const SmpRow &r, const double *tab, int lo, int hi, u64 thr, double left, SmpRed &red) {
  __shared__ int found;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, part = ((hi - lo + 3) / 4 + 3) & ~3;
  u64 v = 0;
  for (int i = lo + w * part + lane; i < min(hi, lo + (w + 1) * part); i += 64) {
    const float x = r.at(i);
    if (smp_ord(x, i) <= thr) v += smp_mass(r, smp_weight(r, x, tab));
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
      mine[e] = i < end && smp_ord(x, i) <= thr ? smp_mass(r, smp_weight(r, x, tab)) : 0;
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

template <bool QUADS>
__global__ __launch_bounds__(SMP_NT) void k_sample_hist(SampleArgs a, SmpWork k) {
  __shared__ double tab[32];
  __shared__ u64 mass[SMP_NB + 1], cert[SMP_GMAX];
  __shared__ unsigned cnt[SMP_NB + 1];
  __shared__ SmpRed red;
  __shared__ int kb_s, p0_s, p1_s, held_s;
  const int g = blockIdx.x, row = blockIdx.y, gr = k.row0 + row, t = threadIdx.x, G = k.G;
  SmpRow r = smp_row(a, gr);
  SmpSet s;
  const bool ok = smp_set(a, gr, s);
  smp_table(tab);
  for (int i = t; i <= SMP_NB; i += SMP_NT) mass[i] = 0, cnt[i] = 0;
  const u64 top = smp_least(t < G ? k.top[(long)row * G + t] : ~0ull, red);
  const float m = smp_value((uint32_t)(top >> 32));
  SmpState &st = k.state[row];
  if (!ok || !(fabsf(m) < INFINITY) || s.k == 1) {  // nothing to draw from, or one entry
    if (g == 0 && t == 0) {
      const bool none = !ok || !(fabsf(m) < INFINITY);
      if (!ok) *a.bad = 1;
      a.tokens[gr] = none ? -1 : (int)(unsigned)top;
      st.mode = SMP_DONE;
      st.thr = top;
      st.total = none ? 0 : 1ull << a.S;
    }
    return;
  }
  r.m = m;
  r.inv_t = 1.0 / s.t;
  const float cf = fminf(16.0f / (float)s.t, 1e30f);
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  smp_each<QUADS, 4>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int b = smp_bucket(m, x[e], cf);
      const u64 v = smp_mass(r, smp_weight(r, x[e], tab));
      if (v) atomicAdd(&mass[b], v);
      if (b < SMP_NB - 1) atomicAdd(&cnt[b], 1u);  // (the last bucket's is what is left of the row)
    }
  });
  __syncthreads();
  if (G > 1) {
    const long at = ((long)row * G + g) * SMP_NB;
    for (int b = t; b < SMP_NB; b += SMP_NT) {
      smp_put(k.mass + at + b, mass[b]);
      smp_put(k.cnt + at + b, cnt[b]);
    }
  }
  if (!smp_last(k, row)) return;
  // the row's buckets, two a thread, and what lies before each
  u64 v[2] = {mass[2 * t], mass[2 * t + 1]};
  unsigned c[2] = {cnt[2 * t], cnt[2 * t + 1]};
  if (G > 1) {
    v[0] = v[1] = 0;
    c[0] = c[1] = 0;
    const long at = (long)row * G * SMP_NB + 2 * t;
    constexpr int UN = 8;  // chunks whose loads are on their way at once
    for (int j0 = 0; j0 < G; j0 += UN) {
      u64 x[UN][2];
      unsigned y[UN][2];
#pragma unroll
      for (int j = 0; j < UN; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const long from = at + (long)min(j0 + j, G - 1) * SMP_NB + e;
          x[j][e] = smp_get(k.mass + from);
          y[j][e] = smp_get(k.cnt + from);
        }
#pragma unroll
      for (int j = 0; j < UN; j++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (j0 + j < G) v[e] += x[j][e], c[e] += y[j][e];
    }
  }
  u64 all, any;
  const u64 upto = smp_scan(v[0] + v[1], all, red), cupto = smp_scan((u64)c[0] + c[1], any, red);
  __syncthreads();
  mass[2 * t + 1] = upto - v[1];
  mass[2 * t] = upto - v[1] - v[0];
  cnt[2 * t + 1] = (unsigned)(cupto - c[1]);
  cnt[2 * t] = (unsigned)(cupto - c[1] - c[0]);
  if (t == 0) {
    mass[SMP_NB] = all;
    cnt[SMP_NB] = a.V;
    kb_s = p0_s = p1_s = SMP_NB;
    held_s = 0;
  }
  __syncthreads();
  const bool by_k = s.k > 0 && s.k < a.V, by_p = s.top_p < 1.0, by_m = s.min_p > 0.0;
  if (by_k)
    for (int e = 0; e < 2; e++)
      if (cnt[2 * t + e] < (unsigned)s.k && cnt[2 * t + e + 1] >= (unsigned)s.k) kb_s = 2 * t + e;
  __syncthreads();
  const int kb = kb_s;
  if (by_p) {  // of the mass that top-k leaves, known up to its last bucket
    const double f0 = s.top_p * (double)mass[by_k ? kb : SMP_NB], f1 = s.top_p * (double)mass[by_k ? kb + 1 : SMP_NB];
    for (int e = 0; e < 2; e++) {
      if ((double)mass[2 * t + e + 1] >= f0) atomicMin(&p0_s, 2 * t + e);
      if ((double)mass[2 * t + e + 1] >= f1) atomicMin(&p1_s, 2 * t + e);
    }
  } else if (t == 0) {
    p0_s = p1_s = kb;
  }
  __syncthreads();
  int b0 = p0_s, b1 = p1_s;
  if (by_m) {  // the bucket of the least weight, and its neighbours for their rounding
    const int b = (int)fmin(-log(s.min_p) * 16.0, 600.0);
    b0 = min(b0, max(b - 1, 0));
    b1 = min(b1, min(b + 1, SMP_NB - 1));
  }
  const bool list = b0 < SMP_NB;
  if (list && cnt[b1 + 1] == cnt[b0]) {  // no entry near min_p: the threshold is the last of the bucket before
    for (int e = 0; e < 2; e++)
      if (2 * t + e < b0 && cnt[2 * t + e + 1] > cnt[2 * t + e]) atomicMax(&held_s, 2 * t + e);
    __syncthreads();
    b0 = held_s;  // (the largest logit is in bucket 0)
  }
  const int n1 = list ? cnt[b1 + 1] - cnt[b0] : 0, nk = list && by_k && kb > b1 ? cnt[kb + 1] - cnt[kb] : 0;
  if (t == 0) {
    st.mode = !list ? SMP_DONE : n1 + nk > SMP_LIST ? SMP_SLOW : SMP_FIND;
    st.thr = ~0ull;
    st.total = all;
    st.b0 = b0;
    st.b1 = b1;
    st.kb = by_k ? kb : -1;
    st.n1 = n1;
    st.n = 0;
    if (list) {
      st.mass0 = mass[b0];
      st.cnt0 = cnt[b0];
      if (by_k) st.massk = mass[kb], st.cntk = cnt[kb];
    }
  }
  if (list && n1 + nk > SMP_LIST) return;
  // the chunks' masses below the listed buckets
  if (G > 1) {
    const int w = t >> 6, lane = t & 63;
    for (int j = w; j < G; j += SMP_NT / 64) {
      u64 x = 0;
      const long at = ((long)row * G + j) * SMP_NB;
      for (int b = lane; b < min(b0, SMP_NB); b += 64) x += smp_get(k.mass + at + b);
      x = smp_wave_sum(x);
      if (lane == 0) {
        cert[j] = x;
        k.cert[(long)row * G + j] = x;
      }
    }
  } else if (t == 0) {
    cert[0] = k.cert[row] = mass[min(b0, SMP_NB)];
  }
  __syncthreads();
  if (list) return;
  u64 before;
  const double left = s.u * (double)all;
  const int ch = smp_chunk(cert, G, left, before);
  const int tok = ch < 0 ? -1 : smp_draw<QUADS>(r, tab, ch * k.len, min(a.V, (ch + 1) * k.len), ~0ull, left - (double)before, red);
  if (t == 0) a.tokens[gr] = tok;
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
        const u64 w = smp_mass(r, smp_weight(r, x, tab));
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
union SmpListLds {
  SmpFind f;
  SmpSlow slow;
};

template <bool QUADS>
__global__ __launch_bounds__(SMP_NT) void k_sample_list(SampleArgs a, SmpWork k) {
  __shared__ SmpListLds lds;
  __shared__ double tab[32];
  __shared__ u64 chunk[SMP_GMAX];
  __shared__ SmpRed red;
  __shared__ unsigned n_s, base_s;
  __shared__ int ip_s, im_s;
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
    u64 thr = ~0ull, mass = st.total;
    if (by_k) thr = smp_select(r, tab, lds.slow, s.k, 0.0, thr, mass);
    if (by_p) thr = smp_select(r, tab, lds.slow, 0, s.top_p * (double)mass, thr, mass);
    u64 total = 0, last = 0;
    for (int i = t; i < a.V; i += SMP_NT) {
      const float x = r.at(i);
      const double wt = smp_weight(r, x, tab);
      const u64 o = smp_ord(x, i);
      if (o <= thr && wt >= s.min_p) {
        total += smp_mass(r, wt);
        last = max(last, o);
      }
    }
    total = smp_sum(total, red);
    if (by_m) thr = ~smp_least(~last, red);  // the last that is heavy enough
    const int tok = smp_draw<QUADS>(r, tab, 0, a.V, thr, s.u * (double)total, red);
    if (t == 0) {
      a.tokens[gr] = tok;
      st.thr = thr;
      st.total = total;
    }
    return;
  }
  if (t == 0) n_s = 0;
  __syncthreads();
  const int b0 = st.b0, b1 = st.b1, kb = st.kb, n1 = st.n1;
  const float cf = fminf(16.0f / (float)s.t, 1e30f);
  const int lo = min(a.V, g * k.len), hi = min(a.V, lo + k.len);
  smp_each<QUADS, 8>(r, lo, hi, [&](int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int b = smp_bucket(m, x[e], cf);
      if (((b >= b0 && b <= b1) || b == kb) && i + e < hi) {
        const unsigned at = atomicAdd(&n_s, 1u);
        if (at < SMP_LIST) lds.f.ord[at] = smp_ord(x[e], i + e);
      }
    }
  });
  __syncthreads();
  unsigned n = min(n_s, (unsigned)SMP_LIST);
  u64 *list = k.list + (long)row * SMP_LIST;
  if (G > 1) {
    if (t == 0 && n) base_s = __hip_atomic_fetch_add(&st.n, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (unsigned i = t; i < n; i += SMP_NT)
      if (base_s + i < SMP_LIST) smp_put(list + base_s + i, lds.f.ord[i]);
    if (!smp_last(k, row)) return;
    n = min(smp_get(&st.n), (unsigned)SMP_LIST);
    for (unsigned i = t; i < n; i += SMP_NT) lds.f.ord[i] = smp_get(list + i);
  }
  // in order (bitonic, padded to a power of two)
  int n2 = 2;
  while (n2 < (int)n) n2 *= 2;
  for (int i = n + t; i < n2; i += SMP_NT) lds.f.ord[i] = ~0ull;
  __syncthreads();
  for (int len = 2; len <= n2; len *= 2)
    for (int d = len / 2; d; d /= 2) {
      for (int i = t; i < n2 / 2; i += SMP_NT) {
        const int x = (i / d) * 2 * d + i % d, y = x + d;
        const u64 p = lds.f.ord[x], q = lds.f.ord[y];
        if ((p > q) == !(x & len)) lds.f.ord[x] = q, lds.f.ord[y] = p;
      }
      __syncthreads();
    }
  // masses up to each entry; the last of b0 .. b1 that is heavy enough
  if (t == 0) ip_s = n1, im_s = -1;
  u64 run = 0;
  for (int i0 = 0; i0 < (int)n; i0 += SMP_NT) {
    const int i = i0 + t;
    const double wt = i < (int)n ? smp_weight(r, smp_value((uint32_t)(lds.f.ord[i] >> 32)), tab) : 0.0;
    u64 all;
    const u64 up = run + smp_scan(i < (int)n ? smp_mass(r, wt) : 0, all, red);
    if (i < (int)n) lds.f.run[i] = up;
    if (i < n1 && wt >= s.min_p) atomicMax(&im_s, i);
    run += all;
  }
  __syncthreads();
  int last = n1 - 1;
  u64 kept = st.total;  // mass that top-k leaves
  if (by_k) {
    if (kb <= b1) {
      last = s.k - 1 - st.cnt0;
      kept = st.mass0 + lds.f.run[last];
    } else {
      kept = st.massk + lds.f.run[n1 + s.k - 1 - st.cntk] - (n1 ? lds.f.run[n1 - 1] : 0);
    }
  }
  if (by_p) {
    const double target = s.top_p * (double)kept;
    for (int i = t; i < n1; i += SMP_NT)
      if ((double)(st.mass0 + lds.f.run[i]) >= target) atomicMin(&ip_s, i);
    __syncthreads();
    last = min(last, ip_s);
  }
  if (by_m) last = min(last, im_s);
  last = min(last, n1 - 1);
  const u64 total = st.mass0 + (last >= 0 ? lds.f.run[last] : 0), thr = last >= 0 ? lds.f.ord[last] : lds.f.ord[0] - 1;
  for (int j = t; j < G; j += SMP_NT) chunk[j] = k.cert[(long)row * G + j];
  __syncthreads();
  for (int i = t; i <= last; i += SMP_NT) {
    const u64 v = lds.f.run[i] - (i ? lds.f.run[i - 1] : 0);
    if (v) atomicAdd(&chunk[(int)((unsigned)lds.f.ord[i] / (unsigned)k.len)], v);
  }
  __syncthreads();
  u64 before;
  const double left = s.u * (double)total;
  const int ch = smp_chunk(chunk, G, left, before);
  const int tok = ch < 0 ? -1 : smp_draw<QUADS>(r, tab, ch * k.len, min(a.V, (ch + 1) * k.len), thr, left - (double)before, red);
  if (t == 0) {
    a.tokens[gr] = tok;
    st.thr = thr;
    st.total = total;
  }
}

template <bool QUADS>
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
  const bool quads = a.V % 4 == 0 && (uintptr_t)a.probs % 16 == 0;
  smp_each<QUADS, 4>(r, lo, hi, [&](int i, const float (&x)[4]) {
    float p[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
      p[e] = total && smp_ord(x[e], i + e) <= thr ? (float)(smp_weight(r, x[e], tab) * scale) : 0.0f;
    if (quads && i + 4 <= hi) {
      *(float4 *)(to + i) = make_float4(p[0], p[1], p[2], p[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (i + e < hi) to[i + e] = p[e];
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
  w.cert = (u64 *)take(rows * G * 8);
  w.state = (SmpState *)take(rows * sizeof(SmpState));
  w.list = (u64 *)take(rows * SMP_LIST * 8);
  w.mass = (u64 *)take(G > 1 ? rows * G * SMP_NB * 8 : 0);
  w.cnt = (unsigned *)take(G > 1 ? rows * G * SMP_NB * 4 : 0);
  w.arrive = c.d_cnt;
  if (k) *k = w;
  return at;
}
size_t sample_scratch(const Ctx &c, size_t n, int V) { return smp_carve(c, n, V, nullptr, nullptr); }

template <bool QUADS>
static void run_sample(const Ctx &c, const SampleArgs &a, const SmpWork &k, int rows) {
  const dim3 grid(k.G, rows), block(SMP_NT);
  launch_k(c, k_sample_top<QUADS>, grid, block, a, k);
  launch_k(c, k_sample_hist<QUADS>, grid, block, a, k);
  if (a.top_k || a.top_p || a.min_p) launch_k(c, k_sample_list<QUADS>, grid, block, a, k);
  if (a.probs) launch_k(c, k_sample_probs<QUADS>, grid, block, a, k);
}

hipError_t launch_sample(const Ctx &c, SampleArgs a, size_t n, void *scratch) {
  int bits = 0;
  while (bits < 31 && (1L << bits) < a.V) bits++;
  a.S = std::min(45, 62 - bits);
  SmpWork k;
  smp_carve(c, n, a.V, (char *)scratch, &k);
  const bool quads = a.stride % 4 == 0 && (uintptr_t)a.x % (a.x16 ? 8 : 16) == 0;
  for (size_t r0 = 0; r0 < n; r0 += CNT_N) {
    k.row0 = (int)r0;
    const int rows = (int)std::min<size_t>(CNT_N, n - r0);
    quads ? run_sample<true>(c, a, k, rows) : run_sample<false>(c, a, k, rows);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace rbt

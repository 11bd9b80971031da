// drafts.hip -- several drafted tokens at once: rotary positions, verification, the accepted rows' move.
//
//   k_rope / k_rope_any  per token and head row: optional (1 + w) RMSNorm (qwen38/attention.rs:138-143), then
//                        the rotation of the entries [start, start + d) by pos * inv_freq
//                        (attention.rs:160-172), from f32 or bf16 to f32 or bf16.
//   k_tree_pos           a node's position: the sequence's length plus the node's depth.
//   k_verify             rejection of drafted tokens against the target's distribution.
//   k_commit             the standing nodes' rows of every layer's draft buffers to its cache.
//
// Products and sums round on their own (-ffp-contract=off).
#include "rbt_device.h"
#include "rbt_internal.h"

namespace rbt {

// ---- rotary positions --------------------------------------------------------------------------
__device__ __forceinline__ void rope_angle(const RopeArgs &a, int pos, int j, float &cs, float &sn) {
  double x = (double)pos * a.inv[j];
  if (a.angle_f32) x = (double)__fmul_rn((float)pos, (float)a.inv[j]);  // as k_gqa_prep rounds it
  double s, c;
  rbt_sincos_d(x, s, c);
  cs = (float)(c * (double)a.factor);
  sn = (float)(s * (double)a.factor);
}

__device__ __forceinline__ int rope_part_of(const RopeArgs &a, int row) {
  int p = 0;
  for (int i = 1; i < a.n_parts; i++)
    if (row >= a.part[i].row0) p = i;
  return p;
}

// Any shape, stride and alignment: one wave per row, entry by entry through LDS.
__global__ __launch_bounds__(256) void k_rope_any(RopeArgs a) {
  __shared__ float cs[512], sn[512], rows[4][1024];
  const int t = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int pos = a.pos[t];
  if (pos < 0) return;
  for (int j = threadIdx.x; j < a.rd / 2; j += 256) rope_angle(a, pos, j, cs[j], sn[j]);
  __syncthreads();
  for (int r = blockIdx.y * 4 + w; r < a.n_rows; r += 4 * gridDim.y) {
    const RopePartD &p = a.part[rope_part_of(a, r)];
    const int h = r - p.row0;
    const long so = (long)t * p.sts + (long)h * p.shs, dof = (long)t * p.dts + (long)h * p.dhs;
    float *x = rows[w];
    double ss = 0.0;
    for (int i = lane; i < a.hd; i += 64) {
      const float v = p.s16 ? rbt_bf16_f32(((const uint16_t *)p.src)[so + i]) : ((const float *)p.src)[so + i];
      ss += (double)v * (double)v;
      x[i] = v;
    }
    if (p.norm) {
      ss = rbt_wave_sum_d(ss);
      const float rr = __fdiv_rn(1.0f, rbt_sqrt_rn(__fadd_rn((float)(ss / (double)a.hd), a.eps)));
      for (int i = lane; i < a.hd; i += 64) x[i] = __fmul_rn(x[i], __fmul_rn(rr, __fadd_rn(1.0f, p.norm[i])));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    const int half = a.rd / 2;
    for (int i = lane; i < a.hd; i += 64) {
      float v = x[i];
      const int k = i - a.start;
      if (p.rotate && k >= 0 && k < a.rd) {
        const int j = a.pairs ? k >> 1 : k < half ? k : k - half;
        const bool first = a.pairs ? !(k & 1) : k < half;
        const int d = a.pairs ? 1 : half;
        const float y = x[first ? i + d : i - d];
        const float vc = __fmul_rn(v, cs[j]), ys = __fmul_rn(y, sn[j]);
        v = first ? __fsub_rn(vc, ys) : __fadd_rn(vc, ys);
      }
      if (p.d16)
        ((uint16_t *)p.dst)[dof + i] = rbt_f32_bf16(v);
      else
        ((float *)p.dst)[dof + i] = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  }
}

// Rows of whole quads (four entries), 16-byte loads. G lanes share a row, each holding U units of two quads: in the
// half layout a rotated pair of quads (j, j + d/2), else two quads of the two halves of the rest. A workgroup takes
// one token (or a part of its rows), 256 / G rows of one tensor at a time; the angles are formed once per
// workgroup, in 64 bits, while the first rows travel.
// Bound by the rows' bytes for prompts: 4095 tokens of 72 rows x 192 f32 in 92 us, 4.9 TB/s in and out (a 4 GiB copy
// reaches 4.75); 158 us while a pass mixed the tensors, whose descriptions then came through vector loads ahead
// of every row. For one token, by the launch and two round trips to memory (5.2 us).
__device__ __forceinline__ float4 rope_ld(const RopePartD &p, long at) {
  if (!p.s16) return *(const float4 *)((const float *)p.src + at);
  const uint2 v = *(const uint2 *)((const uint16_t *)p.src + at);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ void rope_st(const RopePartD &p, long at, float4 v) {
  if (!p.d16) {
    *(float4 *)((float *)p.dst + at) = v;
  } else {
    uint2 o;
    o.x = (uint32_t)rbt_f32_bf16(v.x) | (uint32_t)rbt_f32_bf16(v.y) << 16;
    o.y = (uint32_t)rbt_f32_bf16(v.z) | (uint32_t)rbt_f32_bf16(v.w) << 16;
    *(uint2 *)((uint16_t *)p.dst + at) = o;
  }
}

template <int U>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a, int G) {
  __shared__ __attribute__((aligned(16))) float cs[512], sn[512];
  const int t = blockIdx.x, gl = threadIdx.x % G, gr = threadIdx.x / G, per = 256 / G;
  const int pos = a.pos[t];
  if (pos < 0) return;
  const int nq = a.hd / 4, sq = a.start / 4;
  float4 x[U][2];
  int q[U][2], pi = 0, h = 0;
  // A pass takes `per` rows of one part (its numbers then are the workgroup's, in scalar registers). Loads this
  // lane's quads of pass k; false past the last pass.
  auto load = [&](int k) {
    for (pi = 0; pi < a.n_parts; pi++) {
      const int np = (a.part[pi].heads + per - 1) / per;
      if (k < np) break;
      k -= np;
    }
    if (pi == a.n_parts) return false;
    const RopePartD &p = a.part[pi];
    h = k * per + gr;
    const long so = (long)t * p.sts + (long)h * p.shs;
    const int hq = p.rotate && !a.pairs ? a.rd / 8 : 0, nr = nq - 2 * hq, n2 = (nr + 1) / 2;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = gl + G * u, m = i - hq, m1 = m + n2;
      if (i < hq) {
        q[u][0] = sq + i;
        q[u][1] = sq + hq + i;
      } else {
        q[u][0] = m < n2 ? (m < sq || !hq ? m : m + 2 * hq) : -1;
        q[u][1] = m < n2 && m1 < nr ? (m1 < sq || !hq ? m1 : m1 + 2 * hq) : -1;
      }
      if (h >= p.heads) q[u][0] = q[u][1] = -1;
#pragma unroll
      for (int e = 0; e < 2; e++)
        x[u][e] = q[u][e] >= 0 ? rope_ld(p, so + 4 * q[u][e]) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return true;
  };
  int k = blockIdx.y;
  bool any = load(k);
  for (int j = threadIdx.x; j < a.rd / 2; j += 256) rope_angle(a, pos, j, cs[j], sn[j]);
  __syncthreads();
  for (; any; any = load(k += gridDim.y)) {
    const RopePartD &p = a.part[pi];
    const long dof = (long)t * p.dts + (long)h * p.dhs;
    if (p.norm) {
      double ss = 0.0;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float4 v = x[u][e];
          ss += ((double)v.x * (double)v.x + (double)v.y * (double)v.y) +
                ((double)v.z * (double)v.z + (double)v.w * (double)v.w);
        }
      for (int d = 1; d < G; d <<= 1) ss += __shfl_xor(ss, d, 64);
      const float rr = __fdiv_rn(1.0f, rbt_sqrt_rn(__fadd_rn((float)(ss / (double)a.hd), a.eps)));
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          if (q[u][e] < 0) continue;
          const float *w = p.norm + 4 * q[u][e];
          float4 &v = x[u][e];
          v.x = __fmul_rn(v.x, __fmul_rn(rr, __fadd_rn(1.0f, w[0])));
          v.y = __fmul_rn(v.y, __fmul_rn(rr, __fadd_rn(1.0f, w[1])));
          v.z = __fmul_rn(v.z, __fmul_rn(rr, __fadd_rn(1.0f, w[2])));
          v.w = __fmul_rn(v.w, __fmul_rn(rr, __fadd_rn(1.0f, w[3])));
        }
    }
    if (p.rotate && !a.pairs) {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (gl + G * u < a.rd / 8) {
          const float4 c = *(const float4 *)(cs + 4 * (gl + G * u)), s = *(const float4 *)(sn + 4 * (gl + G * u));
          const float4 v = x[u][0], y = x[u][1];
          float4 &a0 = x[u][0], &a1 = x[u][1];
          a0.x = __fsub_rn(__fmul_rn(v.x, c.x), __fmul_rn(y.x, s.x));
          a0.y = __fsub_rn(__fmul_rn(v.y, c.y), __fmul_rn(y.y, s.y));
          a0.z = __fsub_rn(__fmul_rn(v.z, c.z), __fmul_rn(y.z, s.z));
          a0.w = __fsub_rn(__fmul_rn(v.w, c.w), __fmul_rn(y.w, s.w));
          a1.x = __fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(v.x, s.x));
          a1.y = __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(v.y, s.y));
          a1.z = __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(v.z, s.z));
          a1.w = __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(v.w, s.w));
        }
    } else if (p.rotate) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int j = 2 * (q[u][e] - sq);  // the quad's first pair
          if (q[u][e] < sq || j >= a.rd / 2) continue;
          const float4 v = x[u][e];
          x[u][e] = make_float4(__fsub_rn(__fmul_rn(v.x, cs[j]), __fmul_rn(v.y, sn[j])),
                                __fadd_rn(__fmul_rn(v.y, cs[j]), __fmul_rn(v.x, sn[j])),
                                __fsub_rn(__fmul_rn(v.z, cs[j + 1]), __fmul_rn(v.w, sn[j + 1])),
                                __fadd_rn(__fmul_rn(v.w, cs[j + 1]), __fmul_rn(v.z, sn[j + 1])));
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (q[u][e] >= 0) rope_st(p, dof + 4 * q[u][e], x[u][e]);
  }
}

// Whether every row, of every part, is made of aligned quads.
static bool rope_quads(const RopeArgs &a) {
  if (a.hd % 4 || a.start % 4 || a.rd % (a.pairs ? 4 : 8)) return false;
  for (int i = 0; i < a.n_parts; i++) {
    const RopePartD &p = a.part[i];
    if ((p.sts | p.shs | p.dts | p.dhs) % 4) return false;
    if ((uintptr_t)p.src % (p.s16 ? 8 : 16) || (uintptr_t)p.dst % (p.d16 ? 8 : 16)) return false;
  }
  return true;
}

hipError_t launch_rope(const Ctx &c, const RopeArgs &a, int s) {
  // a token's rows over several workgroups where there are few tokens: four per CU in all
  const int want = std::max(1, 4 * c.num_cu / std::max(1, s));
  if (rope_quads(a)) {
    const int units = (a.hd / 4 + 1) / 2;
    int G = 1;
    while (G < units && G < 64) G *= 2;
    int passes = 0;
    for (int i = 0; i < a.n_parts; i++) passes += (a.part[i].heads * G + 255) / 256;
    const dim3 grid(s, std::min(passes, want));
    if (units <= 64)
      launch_k(c, k_rope<1>, grid, dim3(256), a, G);
    else
      launch_k(c, k_rope<2>, grid, dim3(256), a, G);
  } else {
    launch_k(c, k_rope_any, dim3(s, std::min((a.n_rows + 3) / 4, want)), dim3(256), a);
  }
  return hipGetLastError();
}

// ---- tree positions ------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_tree_pos(const int *__restrict__ parent, const int *__restrict__ n_nodes,
                                                  const int *__restrict__ len, int T, int *__restrict__ pos,
                                                  int *__restrict__ bad) {
  __shared__ int par[TREE_MAX];
  const int b = blockIdx.x, t = threadIdx.x;
  int n = n_nodes[b], L = len[b];
  if (n < 0 || n > T || L < 0 || L > INT32_MAX - max(n - 1, 0)) {
    if (t == 0) *bad = 1;
    n = 0;
  }
  if (t < n) {
    int p = parent[(long)b * T + t];
    if (p < -1 || p >= t) {
      *bad = 1;
      p = -1;
    }
    par[t] = p;
  }
  __syncthreads();
  if (t >= T) return;
  int d = 0;
  if (t < n)
    for (int p = par[t]; p >= 0; p = par[p]) d++;
  pos[(long)b * T + t] = t < n ? L + d : -1;
}

hipError_t launch_tree_pos(const Ctx &c, const int *parent, const int *n_nodes, const int *len, int B, int T, int *pos,
                           int *bad) {
  launch_k(c, k_tree_pos, dim3(B), dim3(256), parent, n_nodes, len, T, pos, bad);
  return hipGetLastError();
}

// ---- verification --------------------------------------------------------------------------------
// The walk reads p and q of every node's token under the node's parent, gathered once, and takes a step per test;
// only a rejected child (given q) and the draw need a pass over the vocabulary. A launch holds G workgroups per
// sequence: each takes the walk to its first pass by itself (the same numbers in the same order: the same walk),
// sums its chunk of the residual, and the last one to arrive goes on: it adds the chunks in order, continues the
// walk, and either draws from the chunks at hand or leaves the state for the next launch's pass. In the last
// launch it makes whatever passes are left by itself. No workgroup waits for another.
// Chains, and drafts without q, need one pass and so one launch. Sums are in 64 bits, and as their order is fixed
// the drawn token is too. Bound by trips to memory that follow one another (count, tokens, their p and q, the
// pass, the arrival, the sums, the draw), not by bytes: a chain of five over 32000 entries takes 12.7 us, one over
// 131072 entries 13, sixteen of them 21; sixteen trees of 32 nodes 66 to 84 by their walks in six launches, of
// which most end at once (one workgroup per sequence for all of it: 26 and, for the trees, 191 where six launches take 80).
constexpr int VF_NT = 256, VF_G = 64, VF_ROUNDS = 6;  // threads per workgroup, chunks and launches at most

struct VerifyRow {
  const float *p, *q;  // the current node's rows (q may be null)
  double c;
  const int *gone;  // without q: tokens that count as 0
  int n_gone;
  __device__ __forceinline__ double of(float pv, float qv, int i) const {
    double r = (double)pv;
    if (q) r = r - c * (double)qv;
    for (int k = 0; k < n_gone; k++)
      if (gone[k] == i) return 0.0;
    return r > 0.0 ? r : 0.0;
  }
  __device__ __forceinline__ double at(int i) const { return of(p[i], q ? q[i] : 0.0f, i); }
};

// The workgroup's sum of [lo, hi), in every thread; quads: rows and lo are aligned to 16 bytes.
__device__ double vf_sum(const VerifyRow &row, int lo, int hi, bool quads, double *red) {
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  double acc = 0.0;
  if (quads) {
    constexpr int UN = 4;
    const int he = lo + ((hi - lo) & ~3);
    for (int i0 = lo + 4 * t; i0 < he; i0 += UN * 4 * VF_NT) {
      float4 pv[UN], qv[UN];
#pragma unroll
      for (int k = 0; k < UN; k++) pv[k] = *(const float4 *)(row.p + min(i0 + k * 4 * VF_NT, he - 4));
#pragma unroll
      for (int k = 0; k < UN; k++)
        qv[k] = row.q ? *(const float4 *)(row.q + min(i0 + k * 4 * VF_NT, he - 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < UN; k++) {
        const int i = i0 + k * 4 * VF_NT;
        if (i < he)
          acc += (row.of(pv[k].x, qv[k].x, i) + row.of(pv[k].y, qv[k].y, i + 1)) +
                 (row.of(pv[k].z, qv[k].z, i + 2) + row.of(pv[k].w, qv[k].w, i + 3));
      }
    }
    lo = he;
  }
  constexpr int UN = 8;
  for (int i0 = lo + t; i0 < hi; i0 += UN * VF_NT) {
    float pv[UN], qv[UN];
#pragma unroll
    for (int k = 0; k < UN; k++) pv[k] = row.p[min(i0 + k * VF_NT, hi - 1)];
#pragma unroll
    for (int k = 0; k < UN; k++) qv[k] = row.q ? row.q[min(i0 + k * VF_NT, hi - 1)] : 0.0f;
#pragma unroll
    for (int k = 0; k < UN; k++)
      if (i0 + k * VF_NT < hi) acc += row.of(pv[k], qv[k], i0 + k * VF_NT);
  }
  acc = rbt_wave_sum_d(acc);
  __syncthreads();
  if (lane == 0) red[w] = acc;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void vf_put(double *p, double v) {
  __hip_atomic_store((unsigned long long *)p, (unsigned long long)__double_as_longlong(v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double vf_get(double *p) {
  return __longlong_as_double(
      (long long)__hip_atomic_load((unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

__global__ __launch_bounds__(VF_NT) void k_verify(VerifyArgs a, int round, int last_round) {
  __shared__ int par[TREE_MAX], tok[TREE_MAX], way[TREE_MAX], gone[TREE_MAX];
  __shared__ float px[TREE_MAX], qx[TREE_MAX], us[TREE_MAX];
  __shared__ double red[4], sums[VF_G];
  __shared__ VerifyState st;
  __shared__ int n_gone, found, is_last;
  const int b = blockIdx.y, ch = blockIdx.x, G = gridDim.x, t = threadIdx.x, lane = t & 63, V = a.V;
  int n = a.n_nodes[b];
  if (n < 0 || n > a.T) {
    if (t == 0) *a.bad = 1;
    n = 0;
  }
  if (n == 0) {
    if (ch || round) return;
    for (int j = t; j < a.T; j += VF_NT) a.path[(long)b * a.T + j] = -1;
    if (t == 0) a.n_path[b] = 0, a.next[b] = -1;
    return;
  }
  if (t == 0) {
    if (round)
      st = a.state[b];
    else
      st = VerifyState{0.0, 1.0, 0, 0, 1, 1, 0};
    n_gone = 0;
    way[0] = 0;
  }
  __syncthreads();
  if (st.done) return;
  const int np0 = round ? st.np : 0;  // standing nodes that an earlier launch wrote
  const float *pb = a.p + (long)b * a.T * V, *qb = a.q ? a.q + (long)b * a.T * V : nullptr;
  auto tables = [&]() {
    if (t < n) {
      int pr = a.parent[(long)b * a.T + t], x = a.tokens[(long)b * a.T + t];
      us[t] = a.u[(long)b * a.T + t];
      if (pr < -1 || pr >= t) {
        *a.bad = 1;
        pr = -1;
      }
      if (t > 0 && (x < 0 || x >= V)) {
        *a.bad = 1;
        x = -1;
      }
      const bool ok = t > 0 && pr >= 0 && x >= 0;
      par[t] = ok ? pr : -1;  // a node without a token of the vocabulary is nobody's child
      tok[t] = x;
      px[t] = ok ? pb[(long)pr * V + x] : 0.0f;
      qx[t] = ok && qb ? qb[(long)pr * V + x] : 1.0f;
    }
    __syncthreads();
  };
  // wave 0: tests children until one is rejected (st.need = 1) or none is left (0)
  auto walk = [&]() {
    if (t < 64) {
      int pk[TREE_MAX / 64], cur = st.cur, at = st.at, np = st.np, ng = n_gone, nd = 0;
      double c = st.c, S = st.mass;
#pragma unroll
      for (int k = 0; k < TREE_MAX / 64; k++) pk[k] = lane + 64 * k < n ? par[lane + 64 * k] : -1;
      for (;;) {
        int i = -1;
#pragma unroll
        for (int k = TREE_MAX / 64 - 1; k >= 0; k--) {
          const unsigned long long m = __ballot(pk[k] == cur && lane + 64 * k > at);
          if (m) i = 64 * k + __ffsll((long long)m) - 1;
        }
        if (i < 0) break;
        at = i;
        const double q = (double)qx[i];
        double r = (double)px[i];
        if (qb) {
          r = r - c * q;
        } else {
          for (int k = 0; k < ng; k++)
            if (gone[k] == tok[i]) r = 0.0;
        }
        r = r > 0.0 ? r : 0.0;
        if ((double)us[i] * (S * q) < r) {
          cur = i;
          if (lane == 0) way[np - np0] = i;
          np++;
          c = 0.0;
          S = 1.0;
          ng = 0;
        } else if (qb) {
          c = c + S;
          nd = 1;
          break;
        } else {
          S = S - r;
          if (lane == 0) gone[ng] = tok[i];
          ng++;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        }
      }
      if (lane == 0) {
        st = VerifyState{c, S, cur, at, np, nd, 0};
        n_gone = ng;
      }
    }
    __syncthreads();
  };
  if (!round) {
    tables();
    walk();
  }
  const bool quads = V % 4 == 0 && (((uintptr_t)a.p | (uintptr_t)a.q) & 15) == 0;
  const int len = ((V + G - 1) / G + 3) & ~3, lo = min(V, ch * len), hi = min(V, lo + len);
  auto row_of = [&]() {
    return VerifyRow{pb + (long)st.cur * V, st.c > 0.0 ? qb + (long)st.cur * V : nullptr, st.c, gone, n_gone};
  };
  VerifyRow row = row_of();
  double s = lo < hi ? vf_sum(row, lo, hi, quads, red) : 0.0;
  if (t == 0) {
    is_last = 1;
    if (G > 1) {
      vf_put(a.part + b * VF_G + ch, s);
      __builtin_amdgcn_s_waitcnt(0);  // the sum is at the device's coherence point before its announcement
      const unsigned old = __hip_atomic_fetch_add(a.cnt + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      is_last = old + 1 == (unsigned)G;
      if (is_last) __hip_atomic_store(a.cnt + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      sums[0] = s;
    }
  }
  __syncthreads();
  if (!is_last) return;
  if (G > 1 && t < G) sums[t] = vf_get(a.part + b * VF_G + t);
  if (round) tables();
  __syncthreads();
  for (;;) {
    double S = 0.0;
    for (int k = 0; k < G; k++) S += sums[k];
    if (st.need) {  // the pass was for a rejected child
      const int cur0 = st.cur;
      const double c0 = st.c;
      __syncthreads();
      if (t == 0) st.mass = S;
      __syncthreads();
      walk();
      if (!st.need && st.cur == cur0 && st.c == c0) break;  // no child is left: the draw is from this residual
    } else {
      break;
    }
    // another residual
    if (!last_round) {
      for (int j = np0 + t; j < st.np; j += VF_NT) a.path[(long)b * a.T + j] = way[j - np0];
      if (t == 0) a.state[b] = st;
      return;
    }
    row = row_of();
    for (int k = 0; k < G; k++) {
      const int l0 = min(V, k * len), h0 = min(V, l0 + len);
      const double x = l0 < h0 ? vf_sum(row, l0, h0, quads, red) : 0.0;
      if (t == 0) sums[k] = x;
    }
    __syncthreads();
    if (!st.need) break;
  }
  const int np = st.np;
  for (int j = np0 + t; j < a.T; j += VF_NT) a.path[(long)b * a.T + j] = j < np ? way[j - np0] : -1;
  if (t == 0) {
    a.n_path[b] = np;
    if (!last_round) a.state[b].done = 1;
  }
  // the draw: the chunk, then the entry, where the running sum passes u times the whole
  row = row_of();
  double tot = 0.0;
  for (int k = 0; k < G; k++) tot += sums[k];
  if (!(tot > 0.0)) {  // an empty residual: p itself
    row = VerifyRow{row.p, nullptr, 0.0, gone, 0};
    tot = 0.0;
    for (int k = 0; k < G; k++) {
      const int l0 = min(V, k * len), h0 = min(V, l0 + len);
      const double x = l0 < h0 ? vf_sum(row, l0, h0, quads, red) : 0.0;
      if (t == 0) sums[k] = x;
      tot += x;
    }
    __syncthreads();
  }
  if (!(tot > 0.0) || tot > 1.7e308) {
    if (t == 0) a.next[b] = -1;
    return;
  }
  double left = (double)us[0] * tot;
  int k = -1, last = 0;
  double before = 0.0, lb = 0.0, run = 0.0;
  for (int j = 0; j < G; j++) {
    const double x = sums[j];
    if (x > 0.0) {
      last = j;
      lb = run;
    }
    if (k < 0 && run + x > left) {
      k = j;
      before = run;
    }
    run += x;
  }
  if (k < 0) {  // rounding left none: the last one with any mass
    k = last;
    before = lb;
  }
  left -= before;
  // blocks of eight entries a thread, in order
  constexpr int E = 8;
  const int l0 = k * len, h0 = min(V, l0 + len), w = t >> 6;
  int tail = -1;  // this thread's last entry with any mass
  for (int b0 = l0; b0 < h0; b0 += E * VF_NT) {
    const int i0 = b0 + t * E;
    float pv[E], qv[E];
    double r[E], mine = 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) pv[e] = row.p[min(i0 + e, V - 1)];
#pragma unroll
    for (int e = 0; e < E; e++) qv[e] = row.q ? row.q[min(i0 + e, V - 1)] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      r[e] = i0 + e < h0 ? row.of(pv[e], qv[e], i0 + e) : 0.0;
      mine += r[e];
      if (r[e] > 0.0) tail = i0 + e;
    }
    const double in = rbt_wave_scan_d(mine), up = __shfl_up(in, 1, 64);
    __syncthreads();
    if (lane == 63) red[w] = in;
    if (t == 0) found = INT32_MAX;
    __syncthreads();
    double base = lane ? up : 0.0;
    for (int j = 0; j < w; j++) base += red[j];
    if (mine > 0.0 && base + mine > left) {
      int at = -1;  // (the thread's last entry with any mass where rounding lets none pass)
#pragma unroll
      for (int e = E - 1; e >= 0; e--)
        if (at < 0 && r[e] > 0.0) at = i0 + e;
      double sum = base;
#pragma unroll
      for (int e = 0; e < E; e++) {
        sum += r[e];
        if (r[e] > 0.0 && sum > left && at > i0 + e) at = i0 + e;
      }
      atomicMin(&found, at);
    }
    __syncthreads();
    if (found != INT32_MAX) break;
    left -= (red[0] + red[1]) + (red[2] + red[3]);
  }
  if (found == INT32_MAX) {  // rounding: the chunk's last entry with any mass
    __syncthreads();
    if (t == 0) found = -1;
    __syncthreads();
    if (tail >= 0) atomicMax(&found, tail);
    __syncthreads();
  }
  if (t == 0) a.next[b] = found;
}

int verify_chunks(const Ctx &c, int B, int V) {
  // 4096 entries each: sixteen trees over 131072 entries take 80 us so, 90 with 2048 (the arrivals queue on their
  // counter), 95 with 8192 and 133 with 16384 (the pass itself)
  return std::max(1, std::min({VF_G, (V + 4095) / 4096, 8 * c.num_cu / B}));
}
size_t verify_scratch(int B) { return (size_t)B * (VF_G * sizeof(double) + sizeof(VerifyState)); }

hipError_t launch_verify(const Ctx &c, VerifyArgs a, int B, int max_children, void *scratch) {
  a.part = (double *)scratch;
  a.state = (VerifyState *)(a.part + (size_t)B * VF_G);
  a.cnt = c.d_cnt;
  const int G = verify_chunks(c, B, a.V), rounds = !a.q || max_children == 1 ? 1 : VF_ROUNDS;
  for (int r = 0; r < rounds; r++) launch_k(c, k_verify, dim3(G, B), dim3(VF_NT), a, r, (int)(r == rounds - 1));
  return hipGetLastError();
}

// ---- commit --------------------------------------------------------------------------------------
// grid (sequences, sides of the launch's layers); U: the unit of the copy. The K and V rows of up to 32 layers go in
// one launch: three rows of 23 layers 3-4 us (the launch), 32 sequences' (28 MB in and out) 6-7 us, against one launch
// per layer and side.
template <typename U>
__global__ __launch_bounds__(256) void k_commit(CommitArgs a, const int *__restrict__ path, const int *__restrict__ n_path,
                                                const int *__restrict__ len, int T, int cap, int row_units,
                                                int *__restrict__ len_out, int *__restrict__ bad) {
  __shared__ int way[TREE_MAX];
  const int b = blockIdx.x, t = threadIdx.x;
  const int n = n_path[b], L = len[b];
  bool ok = n >= 0 && n <= T && L >= 0 && L <= cap - n;
  if (ok && t < n) {
    way[t] = path[(long)b * T + t];
    ok = way[t] >= 0 && way[t] < T;
  }
  ok = !__syncthreads_or(!ok);
  if (blockIdx.y == 0 && t == 0) {
    len_out[b] = ok ? L + n : L;
    if (!ok) *bad = 1;
  }
  if (!ok || a.sides == 0) return;
  U *dst = (U *)a.dst[blockIdx.y] + ((long)b * cap + L) * row_units;
  const U *src = (const U *)a.src[blockIdx.y] + (long)b * T * row_units;
  for (int i = t; i < n * row_units; i += 256) {
    const int j = i / row_units;
    dst[i] = src[(long)way[j] * row_units + (i - j * row_units)];
  }
}

hipError_t launch_commit(const Ctx &c, const CommitArgs &a, int unit, const int *path, const int *n_path, const int *len,
                         int B, int T, int cap, int row_units, int *len_out, int *bad) {
  const dim3 grid(B, std::max(1, a.sides));
  auto k = unit == 16 ? k_commit<uint4> : unit == 4 ? k_commit<uint32_t> : k_commit<uint16_t>;
  launch_k(c, k, grid, dim3(256), a, path, n_path, len, T, cap, row_units, len_out, bad);
  return hipGetLastError();
}

}  // namespace rbt

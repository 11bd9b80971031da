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
        v = first ? __fsub_rn(__fmul_rn(v, cs[j]), __fmul_rn(y, sn[j])) : __fadd_rn(__fmul_rn(v, cs[j]), __fmul_rn(y, sn[j]));
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
      for (int e = 0; e < 2; e++) x[u][e] = q[u][e] >= 0 ? rope_ld(p, so + 4 * q[u][e]) : make_float4(0.f, 0.f, 0.f, 0.f);
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
          ss += ((double)v.x * (double)v.x + (double)v.y * (double)v.y) + ((double)v.z * (double)v.z + (double)v.w * (double)v.w);
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
          v = make_float4(__fmul_rn(v.x, __fmul_rn(rr, __fadd_rn(1.0f, w[0]))), __fmul_rn(v.y, __fmul_rn(rr, __fadd_rn(1.0f, w[1]))),
                          __fmul_rn(v.z, __fmul_rn(rr, __fadd_rn(1.0f, w[2]))), __fmul_rn(v.w, __fmul_rn(rr, __fadd_rn(1.0f, w[3]))));
        }
    }
    if (p.rotate && !a.pairs) {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (gl + G * u < a.rd / 8) {
          const float4 c = *(const float4 *)(cs + 4 * (gl + G * u)), s = *(const float4 *)(sn + 4 * (gl + G * u));
          const float4 v = x[u][0], y = x[u][1];
          x[u][0] = make_float4(__fsub_rn(__fmul_rn(v.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(v.y, c.y), __fmul_rn(y.y, s.y)),
                                __fsub_rn(__fmul_rn(v.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(v.w, c.w), __fmul_rn(y.w, s.w)));
          x[u][1] = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(v.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(v.y, s.y)),
                                __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(v.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(v.w, s.w)));
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
    if ((p.sts | p.shs | p.dts | p.dhs) % 4 || (uintptr_t)p.src % (p.s16 ? 8 : 16) || (uintptr_t)p.dst % (p.d16 ? 8 : 16))
      return false;
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
  if (n < 0 || n > T || L < 0) {
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
// One workgroup per sequence. The walk needs p and q of each node's token under the node's parent, gathered
// once; a rejected child needs the mass of the residual, one pass over the vocabulary.
constexpr int VF_NT = 1024, VF_W = VF_NT / 64;

struct VerifyRow {
  const float *p, *q;  // the current node's rows (q may be null)
  double c;
  const int *gone;  // without q: tokens that count as 0
  int n_gone;
  __device__ double at(int i) const {
    double r = (double)p[i];
    if (q) r = r - c * (double)q[i];
    for (int k = 0; k < n_gone; k++)
      if (gone[k] == i) return 0.0;
    return r > 0.0 ? r : 0.0;
  }
};

// Sums of [lo, hi) in VF_W contiguous segments (seg entries each) into sums; every thread returns the whole.
__device__ double vf_sums(const VerifyRow &row, int lo, int hi, int seg, double *sums) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int s0 = lo + w * seg, s1 = min(hi, s0 + seg);
  double acc = 0.0;
  for (int i = s0 + lane; i < s1; i += 64) acc += row.at(i);
  acc = rbt_wave_sum_d(acc);
  __syncthreads();
  if (lane == 0) sums[w] = acc;
  __syncthreads();
  double tot = 0.0;
  for (int k = 0; k < VF_W; k++) tot += sums[k];
  return tot;
}

__global__ __launch_bounds__(VF_NT) void k_verify(const int *__restrict__ tokens, const int *__restrict__ parent,
                                                  const int *__restrict__ n_nodes, const float *__restrict__ p,
                                                  const float *__restrict__ q, const float *__restrict__ u, int T, int V,
                                                  int *__restrict__ path, int *__restrict__ n_path,
                                                  int *__restrict__ next, int *__restrict__ bad) {
  __shared__ int par[TREE_MAX], tok[TREE_MAX], way[TREE_MAX], gone[TREE_MAX];
  __shared__ float px[TREE_MAX], qx[TREE_MAX], us[TREE_MAX];
  __shared__ double sums[VF_W], st_c, st_s;
  __shared__ int st_cur, st_i, st_need, st_np, st_gone, found;
  const int b = blockIdx.x, t = threadIdx.x;
  int n = n_nodes[b];
  if (n < 0 || n > T) {
    if (t == 0) *bad = 1;
    n = 0;
  }
  const float *pb = p + (long)b * T * V, *qb = q ? q + (long)b * T * V : nullptr;
  if (t < n) {
    int pr = parent[(long)b * T + t], x = tokens[(long)b * T + t];
    if (pr < -1 || pr >= t) {
      *bad = 1;
      pr = -1;
    }
    if (t > 0 && (x < 0 || x >= V)) {
      *bad = 1;
      x = -1;
    }
    par[t] = t == 0 ? -1 : pr;
    tok[t] = x;
    us[t] = u[(long)b * T + t];
    const bool ok = t > 0 && pr >= 0 && x >= 0;
    px[t] = ok ? pb[(long)pr * V + x] : 0.0f;
    qx[t] = ok && qb ? qb[(long)pr * V + x] : ok ? 1.0f : 0.0f;
  }
  if (t == 0) {
    st_cur = 0;
    st_c = 0.0;
    st_s = 1.0;
    st_i = 1;
    st_np = n > 0;
    st_gone = 0;
    way[0] = 0;
  }
  __syncthreads();
  for (;;) {
    if (t == 0) {
      int i = st_i, cur = st_cur;
      st_need = 0;
      for (; i < n; i++) {
        if (par[i] != cur) continue;
        const double c = st_c, S = st_s;
        double r = (double)px[i];
        if (q) {
          r = r - c * (double)qx[i];
        } else {
          for (int k = 0; k < st_gone; k++)
            if (gone[k] == tok[i]) r = 0.0;
        }
        r = r > 0.0 ? r : 0.0;
        if ((double)us[i] * (S * (double)qx[i]) < r) {
          cur = i;
          way[st_np++] = i;
          st_c = 0.0;
          st_s = 1.0;
          st_gone = 0;
        } else if (tok[i] < 0) {
          // a token outside the vocabulary leaves the residual as it is
        } else if (q) {
          st_c = c + S;
          st_need = 1;
          i++;
          break;
        } else {
          st_s = S - r;
          gone[st_gone++] = tok[i];
        }
      }
      st_i = i;
      st_cur = cur;
    }
    __syncthreads();
    const int need = st_need;
    if (!need) break;
    const VerifyRow row{pb + (long)st_cur * V, qb + (long)st_cur * V, st_c, gone, 0};
    const double S = vf_sums(row, 0, V, (V + VF_W - 1) / VF_W, sums);
    __syncthreads();
    if (t == 0) st_s = S;
    __syncthreads();
  }
  const int np = st_np;
  for (int j = t; j < T; j += VF_NT) path[(long)b * T + j] = j < np ? way[j] : -1;
  if (t == 0) n_path[b] = np;
  if (n == 0) {
    if (t == 0) next[b] = -1;
    return;
  }
  // the draw: the segment, then the entry, where the running sum passes u times the whole
  const int cur = st_cur;
  VerifyRow row{pb + (long)cur * V, qb && st_c > 0.0 ? qb + (long)cur * V : nullptr, st_c, gone, st_gone};
  int lo = 0, hi = V, seg = (V + VF_W - 1) / VF_W;
  double tot = vf_sums(row, lo, hi, seg, sums);
  if (!(tot > 0.0)) {
    row = VerifyRow{pb + (long)cur * V, nullptr, 0.0, gone, 0};
    tot = vf_sums(row, lo, hi, seg, sums);
  }
  if (!(tot > 0.0) || tot > 1.7e308) {
    if (t == 0) next[b] = -1;
    return;
  }
  double left = (double)us[0] * tot;
  for (;;) {
    // the first segment whose end passes `left`; rounding may leave none: then the last one with any mass
    int k = -1, last = 0;
    double before = 0.0, lb = 0.0, run = 0.0;
    for (int j = 0; j < VF_W; j++) {
      if (sums[j] > 0.0) {
        last = j;
        lb = run;
      }
      if (k < 0 && run + sums[j] > left) {
        k = j;
        before = run;
      }
      run += sums[j];
    }
    if (k < 0) {
      k = last;
      before = lb;
    }
    left -= before;
    lo = lo + k * seg;
    hi = min(hi, lo + seg);
    if (hi - lo <= VF_NT) break;
    seg = (hi - lo + VF_W - 1) / VF_W;
    vf_sums(row, lo, hi, seg, sums);
  }
  const int i = lo + t, w = t >> 6, lane = t & 63;
  const double r = i < hi ? row.at(i) : 0.0;
  const double in = rbt_wave_scan_d(r);
  __syncthreads();
  if (lane == 63) sums[w] = in;
  if (t == 0) found = INT32_MAX;
  __syncthreads();
  double run = in;
  for (int k = 0; k < w; k++) run += sums[k];
  if (r > 0.0 && run > left) atomicMin(&found, i);
  __syncthreads();
  if (found == INT32_MAX) {  // rounding: the last entry with any mass
    __syncthreads();
    if (t == 0) found = -1;
    __syncthreads();
    if (r > 0.0) atomicMax(&found, i);
    __syncthreads();
  }
  if (t == 0) next[b] = found;
}

hipError_t launch_verify(const Ctx &c, const int *tokens, const int *parent, const int *n_nodes, const float *p,
                         const float *q, const float *u, int B, int T, int V, int *path, int *n_path, int *next, int *bad) {
  launch_k(c, k_verify, dim3(B), dim3(VF_NT), tokens, parent, n_nodes, p, q, u, T, V, path, n_path, next, bad);
  return hipGetLastError();
}

// ---- commit --------------------------------------------------------------------------------------
// grid (sequences, sides of the launch's layers); U: the unit of the copy.
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

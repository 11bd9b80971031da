// tree.hip -- attention of a tree of drafted tokens per sequence over the sequence's cache.
//
// Node i of sequence b sees the len[b] committed rows, itself and its ancestors: with s_j = scale q . k_j over
// those, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), times sigmoid(gate) (qwen38/attention.rs:190-226).
#include "rbt_device.h"
#include "rbt_internal.h"

namespace rbt {

__device__ __forceinline__ float tree_ld(const void *p, long i, int b16) {
  return b16 ? rbt_bf16_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

// Whether the sequence's numbers fit; what does not is reported once per sequence.
__device__ __forceinline__ bool tree_fits(const TreeArgs &a, int b, int &n, int &L) {
  n = a.n_nodes[b];
  L = a.len[b];
  if (n >= 0 && n <= a.T && L >= 0 && L <= a.cap) return true;
  if (threadIdx.x == 0) *a.bad = 1;
  return false;
}

// Any shape: one workgroup per (query head, node, sequence), 256 keys at a time with the running maximum and
// sum. Thread t takes key t's score, then entries t, t + 256, ... of the output; rows that the node does not
// see are passed over.
__global__ __launch_bounds__(256) void k_tree_any(TreeArgs a) {
  __shared__ float q[1024], pr[256], red[4];
  __shared__ int par[TREE_MAX];
  __shared__ uint8_t sees[TREE_MAX];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  int n, L;
  if (!tree_fits(a, b, n, L) || i >= n) return;
  const int kv = h / (a.H / a.K), hd = a.hd;
  const long row = (long)a.K * hd, qi = (((long)b * a.T + i) * a.H + h) * hd;
  for (int e = t; e < hd; e += 256) q[e] = a.q[qi + e];
  if (t < n) {
    int p = a.parent[(long)b * a.T + t];
    if (p < -1 || p >= t) {
      *a.bad = 1;
      p = -1;
    }
    par[t] = p;
    sees[t] = 0;
  }
  __syncthreads();
  if (t == 0)
    for (int j = i; j >= 0; j = par[j]) sees[j] = 1;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int total = L + i + 1;  // no later node is an ancestor
  for (int k0 = 0; k0 < total; k0 += 256) {
    const int j = k0 + t;
    float s = -INFINITY;
    if (j < total && (j < L || sees[j - L])) {
      const void *src = j < L ? a.kc : a.kd;
      const long at = (j < L ? (long)b * a.cap + j : (long)b * a.T + (j - L)) * row + (long)kv * hd;
      float d = 0.0f;
      for (int e = 0; e < hd; e++) d = fmaf(q[e], tree_ld(src, at + e, a.kv16), d);
      s = d * a.scale;
    }
    const float wm = rbt_wave_max_f(s);
    if ((t & 63) == 0) red[t >> 6] = wm;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float f = mn == -INFINITY ? 1.0f : expf(m - mn);
    const float p = s == -INFINITY ? 0.0f : expf(s - mn);
    pr[t] = p;
    __syncthreads();
    const float ws = rbt_group_sum<64>(p);
    if ((t & 63) == 0) red[t >> 6] = ws;
    __syncthreads();
    l = l * f + ((red[0] + red[1]) + (red[2] + red[3]));
    m = mn;
    const int nk = min(256, total - k0);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int e = t + 256 * c;
      if (e >= hd) break;
      float o = acc[c] * f;
      for (int jj = 0; jj < nk; jj++) {
        const int j2 = k0 + jj;
        if (j2 >= L && !sees[j2 - L]) continue;
        const void *src = j2 < L ? a.vc : a.vd;
        const long at = (j2 < L ? (long)b * a.cap + j2 : (long)b * a.T + (j2 - L)) * row + (long)kv * hd;
        o = fmaf(pr[jj], tree_ld(src, at + e, a.kv16), o);
      }
      acc[c] = o;
    }
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const int e = t + 256 * c;
    if (e >= hd) break;
    float o = acc[c] / l;
    if (a.gate) o = __fmul_rn(o, rbt_sigmoid(a.gate[((long)b * a.T + i) * a.gts + (long)h * a.ghs + e]));
    a.out[qi + e] = o;
  }
}

hipError_t launch_tree(const Ctx &c, const TreeArgs &a) {
  launch_k(c, k_tree_any, dim3(a.H, a.T, a.B), dim3(256), a);
  return hipGetLastError();
}

}  // namespace rbt

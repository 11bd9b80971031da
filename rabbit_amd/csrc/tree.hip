// tree.hip -- attention of a tree of drafted tokens per sequence over the sequence's cache.
//
// Node i of sequence b sees the len[b] committed rows, itself and its ancestors: with s_j = scale q . k_j over
// those, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), times sigmoid(gate) (qwen38/attention.rs:190-226).
//
//   k_tree       head dims 64, 128, 192, 256: one pass over a piece of the cache and the drafted rows on the matrix
//                cores, with the running maximum and sum; writes the output, or the piece's partial sums
//   k_tree_join  the pieces' partial sums joined
//   k_tree_any   any head dim: fp32 multiply-adds, one workgroup per query head and node
// Sequences behind shared prefixes (rbt_gqa_prefix_d) take two passes: over each prefix once, its sequences' rows in tiles
// as one long sequence's, and over the sequences' own rows; both leave partial sums.
//   k_tree_both    the two passes in one launch, where that is faster
//   k_prefix_join  a sequence's own pieces and its prefix's joined
//
// Bounds and times (64 query heads over 4 KV heads of 256, one MI355X):
//   64 nodes over 32749 bf16 rows: 292-314 us, of them 280-290 in k_tree: 412 GFLOP of bf16 products, 1.4 PFLOP/s (a
//     large library product reaches 1.2); the matrix cores are busy 63% of the cycles, at a clock that the load holds
//     near 2 GHz.
//   16 trees of 12 to 24 nodes over 4096 to 8192 bf16 rows: 353-368 us, k_tree 324-337; the products as above, and
//     row tiles that a sequence fills in part.
//   32 sequences of one node over 2048 to 4096 rows, 32 query heads over 8 KV heads: 41 us for bf16 rows of 64, 90 for
//     bf16 of 128, 88 and 189 for f32: the caches at 4.3 to 4.9 TB/s.
//   one node over 32768 bf16 rows: 35 us, k_tree 26 (134 MB: 5.1 TB/s); over 513 rows: 13.3 us, two launches of one
//     trip to memory each; five nodes over 4096 f32 rows: 32 us.
//   64 users, 512 own bf16 rows each, behind 8192 shared: 119-126 us (the products of three bf16 parts at the rate of a large
//     library product 94); 8 with 300 own behind 1500: 27 us.
//   32 users, 1000 own int8 rows each, behind 32749 shared: 157-172 us, in the pass over the prefix 117-128 by events around
//     the launch and 133-137 under a profiler (its int8 products at the rate of a large library product 118; vector
//     instructions issue in 60% of the busy cycles, the matrix cores work in 37%, mostly one after the other);
//     16 with up to 8192 own rows: 73-78 us (bytes at a large copy's rate 45), k_tree 63-69: CUs are busy for 65% of the
//     launch (pieces of one length, sequences of unequal ones), their waves wait 58% of the time (two of four compute).
//   One chunk of 256 nodes behind 8192 rows: 364 us bf16, 296 int8 (419 GFLOP or GOP: 371 and 237 at a library product's rate).
#include "rbt_device.h"
#include "rbt_internal.h"

#include <atomic>
#include <cmath>

namespace rbt {

__device__ __forceinline__ float tree_ld(const void *p, long i, int b16) {
  return b16 ? rbt_bf16_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

// Whether a sequence of n nodes behind L own rows is one that is attended to: the passes and the joins ask alike.
__device__ __forceinline__ bool tree_valid(const TreeArgs &a, int n, int L) {
  return n >= 0 && n <= a.T && L >= 0 && L <= a.cap - (a.in_cache ? n : 0);
}
// The sequence's numbers; those that are not valid are reported once per sequence.
__device__ __forceinline__ bool tree_fits(const TreeArgs &a, int b, int &n, int &L) {
  n = a.n_nodes[b];
  L = a.len[b];
  if (tree_valid(a, n, L)) return true;
  if (threadIdx.x == 0) *a.bad = 1;
  return false;
}

// The prefix of sequence b, in every thread of the workgroup: its number (-1: none), its first sequence and its rows.
// False where the prefixes' first sequences do not follow each other within the batch, or the prefix is longer than its
// cache.
__device__ __forceinline__ bool tree_prefix(const TreeArgs &a, int b, int &g, int &f, int &P) {
  __shared__ int found[3];
  g = -1;
  f = P = 0;
  if (a.G == 0) return true;
  if (threadIdx.x == 0) found[0] = -1;
  __syncthreads();
  bool ok = true;
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) {
    const int f0 = a.first[i], f1 = a.first[i + 1], n = a.prefix_len[i];
    ok = ok && f0 >= 0 && f0 <= f1 && f1 <= a.B;
    if (f0 <= b && b < f1) {
      found[0] = i;
      found[1] = f0;
      found[2] = n;
    }
  }
  ok = !__syncthreads_or(!ok);
  if (ok && found[0] >= 0) {
    g = found[0];
    f = found[1];
    P = found[2];
    ok = P >= 0 && P <= a.pcap;
  }
  if (!ok && threadIdx.x == 0) *a.bad = 1;
  return ok;
}

// Entries e .. e + 3 of a row: v / l, times sigmoid of the gate.
__device__ __forceinline__ void tree_store(const TreeArgs &a, int b, int i, int h, int e, float4 v, float l) {
  float o[4] = {v.x / l, v.y / l, v.z / l, v.w / l};
  if (a.gate) {
    const float *g = a.gate + ((long)b * a.T + i) * a.gts + (long)h * a.ghs + e;
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = __fmul_rn(o[k], rbt_sigmoid(g[k]));
  }
  *(float4 *)(a.out + (((long)b * a.T + i) * a.H + h) * a.hd + e) = make_float4(o[0], o[1], o[2], o[3]);
}

// Any shape: one workgroup per (query head, node, sequence), 256 keys at a time with the running maximum and
// sum, the prefix's first. Thread t takes key t's score, then entries t, t + 256, ... of the output; rows that the
// node does not see are passed over.
struct TreeRow {
  const void *p;       // the row's first entry
  const float *scale;  // of 8-bit rows
};
template <bool NEW>
__device__ __forceinline__ TreeRow tree_row(const TreeArgs &a, bool v, int b, int g, int P, int L, int kv, long j) {
  const void *base;
  const float *sc;
  long at;
  if (NEW && j < P) {
    base = v ? a.vp : a.kp;
    sc = v ? a.vps : a.kps;
    at = (long)g * a.pcap + j;
  } else if (j < (long)P + L || (NEW && a.in_cache)) {
    base = v ? a.vc : a.kc;
    sc = v ? a.vcs : a.kcs;
    at = (long)b * a.cap + (j - P);
  } else {
    base = v ? a.vd : a.kd;
    sc = v ? a.vds : a.kds;
    at = (long)b * a.T + (j - P - L);
  }
  at = at * a.K + kv;
  return {(const char *)base + at * a.hd * (NEW && a.kv8 ? 1 : a.kv16 ? 2 : 4), NEW && a.kv8 ? sc + at : nullptr};
}
template <bool NEW>
__device__ __forceinline__ float tree_at(const TreeArgs &a, const TreeRow &r, int e) {
  return NEW && a.kv8 ? (float)((const int8_t *)r.p)[e] * *r.scale : tree_ld(r.p, e, a.kv16);
}

// NEW: with prefixes, 8-bit rows or nodes in the cache.
template <bool NEW>
__global__ __launch_bounds__(256) void k_tree_any(TreeArgs a) {
  __shared__ float q[1024], pr[256], red[4];
  __shared__ int par[TREE_MAX];
  __shared__ uint8_t sees[TREE_MAX];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  int n, L, g = -1, f0 = 0, P = 0;
  if (!tree_fits(a, b, n, L) || i >= n) return;
  if (NEW && !tree_prefix(a, b, g, f0, P)) return;
  const int kv = h / (a.H / a.K), hd = a.hd;
  const long qi = (((long)b * a.T + i) * a.H + h) * hd;
  for (int e = t; e < hd; e += 256) q[e] = a.q[qi + e];
  if (t < n) {
    int p = a.parent ? a.parent[(long)b * a.T + t] : t - 1;
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
  const long old = (long)P + L, total = old + i + 1;  // no later node is an ancestor
  for (long k0 = 0; k0 < total; k0 += 256) {
    const long j = k0 + t;
    float s = -INFINITY;
    if (j < total && (j < old || sees[j - old])) {
      const TreeRow r = tree_row<NEW>(a, false, b, g, P, L, kv, j);
      float d = 0.0f;
      for (int e = 0; e < hd; e++) d = fmaf(q[e], tree_at<NEW>(a, r, e), d);
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
    const int nk = (int)min(256L, total - k0);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int e = t + 256 * c;
      if (e >= hd) break;
      float o = acc[c] * f;
      for (int jj = 0; jj < nk; jj++) {
        const long j2 = k0 + jj;
        if (j2 >= old && !sees[j2 - old]) continue;
        o = fmaf(pr[jj], tree_at<NEW>(a, tree_row<NEW>(a, true, b, g, P, L, kv, j2), e), o);
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

// ---- on the matrix cores -----------------------------------------------------------------------------
// The rows of a KV head are its nodes times its query heads (row r = node * n_rep + head), sixteen per wave. With
// keys on the M side, S^T = K Q^T leaves each lane four keys of one row (column n = lane % 16), which is the B operand
// that O^T = V^T P^T wants if V's rows are taken in the same order: the probabilities never leave their lane, and
// the running maximum and sum of a row are the lane's own (joined over the four lanes of a column).
//   bf16 caches: q and p are split into three bf16 parts that hold their 24 bits exactly (by truncation: 8 bits
//     each), so every product is exact and only the fp32 sums round, at three times the products.
//   f32 caches, one or two row tiles: fp32 MFMAs, which keep up with memory there (32 rows: 128 cycles a key of
//     the 157 that its 2 KB take a CU's share of the bandwidth).
//   f32 caches, more row tiles: keys and values are split too, once per workgroup on their way into LDS, at six
//     products. All four are rounded to nearest part by part, so that the middle part is at most 2^-8 of the whole and
//     the last 2^-17, and the three products left out come to 2^-24 of theirs at most, of either sign (parts by
//     truncation are of one sign and twice and four times as long: 2^-21, always towards zero). 64 nodes over 8192 rows
//     187 us, 307 with fp32 MFMAs.
// A workgroup of RW x KW waves takes RW row tiles and one piece of the keys: KW groups of waves share out each
// stage's keys (few rows: every wave has its own keys; many rows: every wave has its own rows, up to eight waves: with
// four, two workgroups per CU, 64 nodes over 32749 rows took 348 us against 311). Stages of TK keys land in LDS by
// direct loads (global_load_lds, 16 bytes per lane), two stages in turn: while one is multiplied the next is in
// flight. (Split rows pass through registers, and have one buffer: its 96 KB at head_dim 256 leave no room.)
// Wave priorities that let one wave of a SIMD run ahead of the other changed nothing (297 us either way).
typedef float tf4 __attribute__((ext_vector_type(4)));
typedef short ts4 __attribute__((ext_vector_type(4)));
typedef __bf16 tb8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) ts4 tree_lds_s4;

// 64 lanes' 16 bytes at p (each its own) to LDS at `base` (the wave's) + 16 lane. m0 is a register that the compiler
// reserves: it keeps nothing there from one statement to the next, and warns of it in a list of clobbers.
__device__ __forceinline__ void tree_dma(const void *p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(p) : "memory");
}
// 64 lanes' 4 bytes, to `base` + 4 lane.
__device__ __forceinline__ void tree_dma4(const void *p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(base), "v"(p) : "memory");
}

// x = hi + mid + lo, each with its low 16 bits zero (fp32 has 24 significant bits, each part 8): for products with bf16
// rows, of which all three are kept.
__device__ __forceinline__ void tree_split(float x, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
  hi = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(hi);
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid));
}
// The high halves of a and b as two bf16 (a low).
__device__ __forceinline__ uint32_t tree_pack(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// a and b rounded to the nearest bf16 (a low).
typedef float tf2 __attribute__((ext_vector_type(2)));
typedef __bf16 tb2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t tree_cvt(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((tf2{a, b}), tb2));
}
// a and b each as the sum of three bf16, the first two rounded to nearest: exact from 2^-110 on, since the first leaves
// 16 significant bits and the second 7. WIDE: a first part that would round to infinity stays the largest bf16, which
// leaves no more bits; infinities and NaN give a NaN. (Rounding by integers instead of conversions: 8 sequences of 16
// nodes 329 us, 321 with conversions. A check of the stage for numbers that large instead of WIDE: 325.)
template <bool WIDE>
__device__ __forceinline__ void tree_round(float a, float b, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
  constexpr float top = 0x1.fep127f;
  hi = WIDE ? tree_cvt(__builtin_amdgcn_fmed3f(a, -top, top), __builtin_amdgcn_fmed3f(b, -top, top)) : tree_cvt(a, b);
  a -= __uint_as_float(hi << 16);
  b -= __uint_as_float(hi & 0xffff0000u);
  mid = tree_cvt(a, b);
  lo = tree_pack(__float_as_uint(a - __uint_as_float(mid << 16)),
                 __float_as_uint(b - __uint_as_float(mid & 0xffff0000u)));
}

// Over a column's four lanes (lane % 16): a swap of rows, then of halves, leaves both sides' values in every lane,
// without the LDS trip of a shuffle.
struct TreePair { float a, b; };
__device__ __forceinline__ TreePair tree_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return {__uint_as_float(p[0]), __uint_as_float(p[1])};
}
__device__ __forceinline__ TreePair tree_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return {__uint_as_float(p[0]), __uint_as_float(p[1])};
}
__device__ __forceinline__ float tree_xor_max(float v) {
  TreePair p = tree_rows(v);
  p = tree_halves(fmaxf(p.a, p.b));
  return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float tree_xor_sum(float v) {
  TreePair p = tree_rows(v);
  p = tree_halves(p.a + p.b);
  return p.a + p.b;
}

// How keys and values reach the matrix cores: bf16 as they are, f32 as they are, f32 in three bf16 parts.
// KV_PARTS4: by workgroups of four waves, several of them on a CU, for batches of up to four row tiles at head dims 64
// and 128. 12 nodes of 32 query heads over 8 KV heads of 128: 32 sequences of up to 4096 rows 246 us with eight waves,
// 207 with four, but one of 8192 rows (16 nodes) 27.6 and 30.9, where loading a stage is what it waits for.
// KV_I8: 8-bit rows with a scale each, see tree_digits below.
enum { KV_BF16 = 0, KV_F32 = 1, KV_PARTS = 2, KV_PARTS4 = 3, KV_I8 = 4 };
constexpr bool tree_parts(int kv) { return kv == KV_PARTS || kv == KV_PARTS4; }

// Workgroups of eight waves, one on a CU; else of four, two or more.
constexpr bool tree_wide(int kv, int kw) { return kw == 1 && kv != KV_PARTS4; }

// Keys per stage.
constexpr int tree_tk(int kv, int kw) { return kv == KV_I8 && kw == 1 ? 128 : kv == KV_BF16 || kv == KV_I8 ? 64 : 32; }

template <int HD, int KV, int KW = 1>
struct TreeTile {
  static constexpr int ROWB = HD * (KV == KV_F32 ? 4 : KV == KV_I8 ? 1 : 2), CH = ROWB / 16;  // bytes and chunks of a row in LDS
  static constexpr int GROW = HD * (KV == KV_BF16 ? 2 : KV == KV_I8 ? 1 : 4);  // bytes of a row of the cache
  static constexpr int TK = tree_tk(KV, KW);
  static constexpr int PART = TK * ROWB, SIDE = PART * (tree_parts(KV) ? 3 : 1);
  static constexpr int STAGE = 2 * SIDE + (KV == KV_I8 ? 8 * TK : 0);       // K, then V, then 8-bit rows' scales of K and V
  static constexpr int LDS = tree_parts(KV) ? STAGE : 2 * STAGE;
  static constexpr int INSTR = TK * CH / 64;                                // 1 KB loads per side
  static_assert(TK * CH % 64 == 0 && CH % (KV == KV_I8 ? 4 : 8) == 0, "whole loads");
  // Where chunk c of row r lies in its row: c ^ k_turn(r), c ^ v_turn(r). The LDS serves 256 bytes a cycle from 64
  // banks, to lanes 0-3, 12-15, 20-23 and 24-27 of a 16-byte read (four such sets) or to half a wave of an 8-byte
  // one; the turns spread the rows of each set over all banks. (Turns within 128 bytes made every read take
  // two cycles: half of the LDS's cycles at 64 nodes over 32749 rows.)
  static constexpr bool WIDE = CH % 16 == 0;  // rows of whole 256 bytes; others begin half a cycle apart
  static __device__ __forceinline__ int k_turn(int r) {
    return WIDE ? r & 15 : CH % 8 == 0 ? r & 7 : -(r >> 2) & 3;  // (rows of 64 and 192 bytes: four, or a multiple, to a cycle)
  }
  static __device__ __forceinline__ int v_turn(int r) {
    // (a 16-lane read of 8-bit values takes rows 0-3 and 16-19 of its column's four)
    if constexpr (KV == KV_I8)
      return WIDE ? (r & 7) | (r >> 4 & 1) << 3 : CH % 8 == 0 ? (r >> 1 & 3) | (r >> 4 & 1) << 2 : (r >> 2 & 1) | (r >> 4 & 1) << 1;
    return KV == KV_F32 ? 0 : WIDE ? (r & 7) << 1 : (r >> 1 & 3) << 1;
  }
};

// A row's node, row / n_rep: magic = ceil(2^32 / n_rep), exact since row * n_rep < 2^32 (at most 2^20 rows and 2^12
// query heads).
__device__ __forceinline__ int tree_div(int row, const TreeArgs &a) {
  return a.R == 1 ? row : (int)__umulhi(row, a.magic);
}

// Keys of a piece and pieces of a sequence of L committed rows; one longer than expected takes larger pieces.
__device__ __forceinline__ void tree_pieces(const TreeArgs &a, int L, int TK, unsigned &per, unsigned &np) {
  per = a.per;
  np = 1;
  if (a.pieces == 1 && L > 0) {
    per = L;
  } else if (L > 0) {
    if ((unsigned)L > (unsigned long long)per * a.pieces)
      per = (((unsigned)L + a.pieces - 1) / a.pieces + TK - 1) / TK * TK;
    np = ((unsigned)L + per - 1) / per;
  }
}

// 8-bit rows. Their entries go to the matrix cores as they are (v_mfma_i32_16x16x64_i8, at twice the rate of bf16), and
// so do three digits of each query and probability: a number x is taken as the whole number X nearest to x f, where f
// brings the row's largest |x| to just below 2^23, and X = 65536 d2 + 256 d1 + d0 with digits in -128..127. A digit's
// products and sums are exact (256 * 128 * 127 at most, below 2^22). So a score is exact up to the query's rounding (half of 2^-22 of its largest entry), and the sum over a
// stage's values up to the probabilities' (half of 2^-22 of the stage's largest probability times scale); f32 sums
// over stages. A key's scale multiplies its score, a value's its probability. Three products at twice the
// rate are half of what bf16 rows take.
constexpr float TREE_TOP = 8355711.0f;           // 127 * 65536 + 127 * 256 + 127
constexpr float TREE_BIAS = 8421504.0f;          // 128 in every digit: those of X + TREE_BIAS are not negative
constexpr float TREE_FIT = TREE_TOP / 0x1p23f;   // [2^22, 2^23) times this is at most TREE_TOP

// Byte k of four words as digit words; the words hold X + TREE_BIAS in [2^23, 2^24) as floats (X not negative), so
// that bits 0-22 are that less 2^23: byte 2 is the digit itself, bytes 1 and 0 are 128 more than theirs.
__device__ __forceinline__ void tree_digits(const uint32_t (&w)[4], uint32_t &d2, uint32_t &d1, uint32_t &d0) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x0c0c0602u);
  d0 = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
  d1 = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u;
  d2 = __builtin_amdgcn_perm(d, c, 0x05040100u);
}
typedef int ti4 __attribute__((ext_vector_type(4)));
typedef int ti2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) ti2 tree_lds_i2;
// Sums start from the bits of C = 1.5 * 2^23, so that one of n (within 2^22) holds the bits of C + n and needs no
// conversion (which takes the time of four instructions). With s2, s1, s0 read so, 256 s2 - K + s1 is
// 256 n2 + n1 - C / 256 for K = 257 C + C / 256 (all but the last sum exact), and 256 times that plus s0 is the whole.
__device__ __forceinline__ ti4 tree_zero() { return ti4{0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000}; }
__device__ __forceinline__ float tree_high(int s2, int s1) {
  return fmaf(__int_as_float(s2), 256.0f, -0xc0c0c000p0f) + __int_as_float(s1);
}

// The prefix and its tile of 16 rw rows that flat tile `rt` of a pass over the prefixes is. A prefix's tiles begin at
// (f TR + g (U - 1)) / U, with f its first sequence and U = 16 rw: at least its own number from the one before.
__device__ __forceinline__ int tree_tile0(const TreeArgs &a, int f, int g, int U) {
  return (f * a.T * a.R + g * (U - 1)) / U;
}
__device__ __forceinline__ bool tree_group(const TreeArgs &a, int rt, int &g, int &f0, int &f1, int &L) {
  const int lane = threadIdx.x & 63, U = 16 * a.rw;
  for (int i0 = 0; i0 < a.G; i0 += 64) {
    const int i = min(i0 + lane, a.G - 1), x0 = a.first[i], x1 = a.first[i + 1], n = a.len[i];
    const bool in = x0 >= 0 && x0 < x1 && x1 <= a.B && tree_tile0(a, x0, i, U) <= rt && rt < tree_tile0(a, x1, i + 1, U);
    const unsigned long long m = __ballot(in);
    if (m) {
      const int l = __ffsll((long long)m) - 1;
      g = __builtin_amdgcn_readlane(i, l);
      f0 = __builtin_amdgcn_readlane(x0, l);
      f1 = __builtin_amdgcn_readlane(x1, l);
      L = __builtin_amdgcn_readlane(n, l);
      return true;
    }
  }
  return false;
}

// Workgroup (bx, by, bz) of a pass.
template <int HD, int KV, int KW>
__device__ __forceinline__ void tree_pass(const TreeArgs &a, int bx, int by, int bz) {
  using TT = TreeTile<HD, KV, KW>;
  constexpr bool I8 = KV == KV_I8;
  constexpr bool B16 = KV != KV_F32, PARTS = tree_parts(KV);  // values' tiles of 16 entries; split rows
  constexpr int ROWB = TT::ROWB, CH = TT::CH, TK = TT::TK, SK = TK / KW, NT = SK / 16;
  static_assert(!I8 || SK == 128 || SK == 32, "whole products");
  static_assert(!PARTS || KW == 1, "one group of waves");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ int par[TREE_MAX];
  __shared__ uint32_t vis[128][TREE_MAX / 32];  // per node of the row tile: which drafted rows it sees
  __shared__ uint32_t dirty[TREE_MAX / 32];     // drafted rows with non-finite values
  __shared__ float ml[KW > 1 ? 4 : 1][2][16];

  // workgroup -> (row tile, piece, KV head, sequence); with several row tiles the workgroups that share keys are
  // consecutive ones of an XCD (id % 8)
  int piece = bx, rt = 0, kv = by, b = bz;
  if (a.tiles > 1) {
    const unsigned id = bx, g = id / 8 / a.tiles * 8 + id % 8, KB = a.K * a.seqs;
    if (g >= a.pieces * KB) return;
    rt = id / 8 % a.tiles;
    piece = g / KB;
    const unsigned r = g - piece * KB;
    b = r / a.K;
    kv = r - b * a.K;
  }
  int n, L, node0 = b * a.T;  // nodes, rows of the cache, first node's place among all
  const int R = a.R, RW = a.rw;
  long unit = (((long)piece * a.seqs + b) * a.K + kv) * a.t16;  // of the partial sums' 16-row tiles
  if (a.pre) {  // the cache is a prefix, the nodes are those of all its sequences
    int f0, f1;
    if (!tree_group(a, rt, b, f0, f1, L)) return;
    if (L <= 0 || L > a.cap) return;  // (reported where the parts are joined)
    rt -= tree_tile0(a, f0, b, 16 * RW);
    unit += tree_tile0(a, f0, b, 16);
    node0 = f0 * a.T;
    n = (f1 - f0) * a.T;
  } else if (!tree_fits(a, b, n, L)) {
    return;
  }
  const int rows = n * R;
  const int NW = blockDim.x >> 6;
  const int row0 = rt * RW * 16;
  if (row0 >= rows) return;
  unsigned per, np;
  tree_pieces(a, L, TK, per, np);
  if (piece >= (int)np) return;
  const int k0 = piece * per, nc = min(L - k0, (int)per);  // cache rows k0 .. k0 + nc - 1, then drafted rows
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int rg = KW == 1 ? w : w % RW, kgp = KW == 1 ? 0 : w / RW, col = lane & 15, kg = lane >> 4;
  const int node_lo = tree_div(row0, a), node_hi = tree_div(min(rows, row0 + RW * 16) - 1, a);
  const int nd = !a.pre && piece == (int)np - 1 ? node_hi + 1 : 0;  // drafted rows: those up to the tile's last node
  const int keys = nc + nd, st_n = (keys + TK - 1) / TK;

  const long seq_row = (long)a.K * TT::GROW;  // bytes from a row to the next
  const long at_c = ((long)b * a.cap + k0) * a.K + kv, at_d = (a.in_cache ? (long)b * a.cap + L : (long)b * a.T) * a.K + kv;
  const long off_c = at_c * TT::GROW, off_d = at_d * TT::GROW;
  const char *kc = (const char *)a.kc + off_c, *vc = (const char *)a.vc + off_c;
  const char *kd = (const char *)a.kd + off_d, *vd = (const char *)a.vd + off_d;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;

  // keys s TK .. of the piece into buffer s & 1; rows past the last one repeat it
  auto issue = [&](int s) {
    const int base = s * TK;
    const uint32_t to = lds0 + (s & 1) * TT::STAGE;
    if (base + TK <= nc) {
      for (int i = w; i < TT::INSTR; i += NW) {
        const int u = i * 64 + lane, r = u / CH, c = u - r * CH;
        const long at = (long)(base + r) * seq_row;
        tree_dma(kc + at + (c ^ TT::k_turn(r)) * 16, to + i * 1024);
        tree_dma(vc + at + (c ^ TT::v_turn(r)) * 16, to + TT::SIDE + i * 1024);
      }
    } else {
      for (int i = w; i < TT::INSTR; i += NW) {
        const int u = i * 64 + lane, r = u / CH, c = u - r * CH, j = min(base + r, keys - 1);
        const long at = (long)(j < nc ? j : j - nc) * seq_row;
        tree_dma((j < nc ? kc : kd) + at + (c ^ TT::k_turn(r)) * 16, to + i * 1024);
        tree_dma((j < nc ? vc : vd) + at + (c ^ TT::v_turn(r)) * 16, to + TT::SIDE + i * 1024);
      }
    }
    if constexpr (I8)
      for (int i = w; i < 2 * TK / 64; i += NW) {
        constexpr int per = TK / 64;
        const bool v = i >= per;
        const int j = min(base + (v ? i - per : i) * 64 + lane, keys - 1);
        const float *from = j < nc ? (v ? a.vcs : a.kcs) + at_c : (v ? a.vds : a.kds) + at_d;
        tree_dma4(from + (long)(j < nc ? j : j - nc) * a.K, to + 2 * TT::SIDE + i * 256);
      }
  };
  // key i of the piece holds a non-finite value (one past the last repeats it)
  auto mark = [&](int i) { atomicOr(&dirty[(min(i, keys - 1) - nc) >> 5], 1u << ((min(i, keys - 1) - nc) & 31)); };

  // split rows: a thread's quads of the stage, K's then V's, on their way
  constexpr int PNT = KV == KV_PARTS4 ? 256 : 512, UN = PARTS ? TK * HD / 4 / PNT : 1;
  static_assert(!PARTS || TK * HD / 4 == UN * PNT, "whole quads");
  float4 raw[2][UN];
  // Lane numbers formed anew in every stage of split rows of 256: kept from stage to stage, the addresses made of them
  // push queries out of the registers, and the reloads wait for the rows on their way.
  auto again = [](int x) {
    if constexpr (PARTS && HD == 256) asm volatile("" : "+v"(x));
    return x;
  };
  auto fetch = [&](int s) {
    if ((s + 1) * TK <= nc) {  // 32 rows are at most 2^27 bytes: a 32-bit offset per lane from the stage's first row
      const char *k0 = kc + (long)s * TK * seq_row, *v0 = vc + (long)s * TK * seq_row;
#pragma unroll
      for (int k = 0; k < UN; k++) {
        constexpr int Q = HD / 4, whole = PNT % Q == 0;
        const unsigned u = whole ? t : k * PNT + t, r = u / Q;
        const unsigned at = r * (unsigned)seq_row + (u - r * Q) * 16;
        const long up = whole ? k * (PNT / Q) * seq_row : 0;
        raw[0][k] = *(const float4 *)(k0 + up + at);
        raw[1][k] = *(const float4 *)(v0 + up + at);
      }
      return;
    }
    const int t0 = again(t);
#pragma unroll
    for (int k = 0; k < UN; k++) {
      const int u = k * PNT + t0, r = u / (HD / 4), j = min(s * TK + r, keys - 1);
      const long at = (long)(j < nc ? j : j - nc) * seq_row + (u - r * (HD / 4)) * 16;
      raw[0][k] = *(const float4 *)((j < nc ? kc : kd) + at);
      raw[1][k] = *(const float4 *)((j < nc ? vc : vd) + at);
    }
  };
  // the quads in three parts to LDS; non-finite drafted values are taken out (see below)
  auto split = [&](int s) {
    const int t0 = again(t);
    const bool drafted = nd > 1 && (s + 1) * TK > nc;
#pragma unroll
    for (int k = 0; k < UN; k++) {
      const int u = k * PNT + t0, r = u / (HD / 4), c = u - r * (HD / 4);
#pragma unroll
      for (int side = 0; side < 2; side++) {
        float v[4] = {raw[side][k].x, raw[side][k].y, raw[side][k].z, raw[side][k].w};
        if (side && drafted && s * TK + r >= nc) {
          bool hit = false;
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (!(fabsf(v[e]) < INFINITY)) v[e] = 0.0f, hit = true;
          if (hit) mark(s * TK + r);
        }
        uint32_t o[3][2];
#pragma unroll
        for (int e = 0; e < 2; e++) tree_round<true>(v[2 * e], v[2 * e + 1], o[0][e], o[1][e], o[2][e]);
        const int at = (c >> 1) ^ (side ? TT::v_turn(r) : TT::k_turn(r));
        char *to = smem + side * TT::SIDE + r * ROWB + at * 16 + (c & 1) * 8;
#pragma unroll
        for (int p = 0; p < 3; p++) *(uint2 *)(to + p * TT::PART) = make_uint2(o[p][0], o[p][1]);
      }
    }
  };
  if constexpr (PARTS)
    fetch(0);
  else
    issue(0);

  // this lane's row, and its query in the B operand's layout
  const bool active = rg < RW && kgp < KW && row0 + rg * 16 < rows;  // a wave without rows or keys only loads
  const int row = row0 + rg * 16 + col, rc = min(row, rows - 1);
  const int node = tree_div(rc, a), head = kv * R + (rc - node * R);
  const long qrow = (long)(node0 + node) * a.H + head;
  const float *qp = a.q + qrow * HD;
  tb8 qb[B16 && !I8 ? HD / 32 : 1][3];
  float4 qf[B16 ? 1 : HD / 16];
  ti4 qd[I8 ? HD / 64 : 1][3];
  float qs = 1.0f;  // what a score's whole number stands for, in powers of two
  if constexpr (I8) {
    float4 x[HD / 64][4];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < HD / 64; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[s][i] = *(const float4 *)(qp + 64 * s + 16 * kg + 4 * i);
        const float4 v = x[s][i];
        top = max(max(max(top, __float_as_uint(v.x) & 0x7fffffffu), __float_as_uint(v.y) & 0x7fffffffu),
                  max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
      }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    const float most = __uint_as_float(top);
    int e = __builtin_amdgcn_frexp_expf(most);  // most in [2^(e - 1), 2^e)
    if (__builtin_amdgcn_ldexpf(most, 23 - e) > TREE_TOP) e++;
    e = max(e, -100);
    const bool whole = top < 0x7f800000u;
    // (the scale's sign goes to the query, zeros for a scale of 0; the factor stays above 0 for hidden keys' sake)
    qs = whole ? fmaxf(fabsf(a.scale) * 1.44269504088896341f * __builtin_amdgcn_ldexpf(1.0f, e - 23), 0x1p-126f) : __uint_as_float(0x7fc00000u);
    const float sign = a.scale < 0.0f ? -1.0f : a.scale > 0.0f ? 1.0f : 0.0f;
#pragma unroll
    for (int s = 0; s < HD / 64; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float v[4] = {x[s][i].x, x[s][i].y, x[s][i].z, x[s][i].w};
        uint32_t u[4], d2, d1, d0;
#pragma unroll
        for (int k = 0; k < 4; k++)
          u[k] = whole ? (uint32_t)((int)rintf(__builtin_amdgcn_ldexpf(v[k] * sign, 23 - e)) + (int)TREE_BIAS) : (uint32_t)TREE_BIAS;
        tree_digits(u, d2, d1, d0);
        qd[s][0][i] = (int)d0;
        qd[s][1][i] = (int)d1;
        qd[s][2][i] = (int)(d2 ^ 0x80808080u);
      }
  } else if constexpr (B16) {
#pragma unroll
    for (int s = 0; s < HD / 32; s++) {
      const float4 x = *(const float4 *)(qp + 32 * s + 8 * kg), y = *(const float4 *)(qp + 32 * s + 8 * kg + 4);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      if constexpr (PARTS) {
        uint32_t o[3][4];
#pragma unroll
        for (int e = 0; e < 4; e++) tree_round<true>(v[2 * e], v[2 * e + 1], o[0][e], o[1][e], o[2][e]);
#pragma unroll
        for (int p = 0; p < 3; p++) qb[s][p] = __builtin_bit_cast(tb8, rbt_u4{o[p][0], o[p][1], o[p][2], o[p][3]});
      } else {
        uint32_t o[3][8];
#pragma unroll
        for (int e = 0; e < 8; e++) tree_split(v[e], o[0][e], o[1][e], o[2][e]);
#pragma unroll
        for (int p = 0; p < 3; p++)
          qb[s][p] = __builtin_bit_cast(tb8, rbt_u4{tree_pack(o[p][0], o[p][1]), tree_pack(o[p][2], o[p][3]),
                                                    tree_pack(o[p][4], o[p][5]), tree_pack(o[p][6], o[p][7])});
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < HD / 16; s++) qf[s] = *(const float4 *)(qp + 16 * s + 4 * kg);
  }
  if (nd > 0) {
    if (t < TREE_MAX / 32) dirty[t] = 0;
    for (int j = t; j < n; j += blockDim.x) {
      int p = a.parent ? a.parent[(long)b * a.T + j] : j - 1;
      if (p < -1 || p >= j) {
        *a.bad = 1;
        p = -1;
      }
      par[j] = p;
    }
    lds_barrier();
    for (int i = node_lo + t; i <= node_hi; i += blockDim.x) {
      for (int x = 0; x < TREE_MAX / 32; x++) vis[i - node_lo][x] = 0;
      for (int j = i; j >= 0; j = par[j]) vis[i - node_lo][j >> 5] |= 1u << (j & 31);
    }
    // (read after the barrier of the first drafted stage)
  }

  const float c1 = a.scale * 1.44269504088896341f;  // scores in powers of two
  float m = -INFINITY, l = 0.0f;
  float gone = 0.0f;  // NaN where a value's scale was not finite
  tf4 o[HD / 16];
#pragma unroll
  for (int x = 0; x < HD / 16; x++) o[x] = tf4{0.f, 0.f, 0.f, 0.f};

  for (int s = 0; s < st_n; s++) {
    char *kt = smem + (PARTS ? 0 : (s & 1) * TT::STAGE), *vt = kt + TT::SIDE;
    const int base = s * TK;
    if constexpr (PARTS) {
      lds_barrier();  // the last stage's readers are done
      split(s);
      if (s + 1 < st_n) fetch(s + 1);
      lds_barrier();
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();  // the stage has landed, and the other buffer's readers are done
      if (s + 1 < st_n) issue(s + 1);
    }
    if (!PARTS && !I8 && nd > 1 && base + TK > nc) {
      // a value that some rows do not see must not meet their zero probabilities: non-finite ones are taken
      // out of the tile (its repeated last row too) and make NaNs at the end of the rows that do see them
      for (int u = t + max(nc - base, 0) * CH; u < TK * CH; u += blockDim.x) {
        const int r = u / CH;
        uint32_t *x = (uint32_t *)(vt + u * 16);
        bool hit = false;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t v = x[e];
          if constexpr (B16) {
            if ((v & 0x7f80u) == 0x7f80u) v &= 0xffff0000u, hit = true;
            if ((v & 0x7f800000u) == 0x7f800000u) v &= 0xffffu, hit = true;
          } else {
            if ((v & 0x7f800000u) == 0x7f800000u) v = 0, hit = true;
          }
          if (hit) x[e] = v;
        }
        if (hit) mark(base + r);
      }
      lds_barrier();
    }

    if (!active) continue;

    // scores: lane (col, kg) gets keys 16 x + 4 kg + i of its row
    tf4 sc[NT];
#pragma unroll
    for (int x = 0; x < NT; x++) sc[x] = tf4{0.f, 0.f, 0.f, 0.f};
    const char *kb = kt + (kgp * SK + col) * ROWB;
    // byte of chunk 4 st + kg in the lane's rows (rows 16 apart turn alike): a few offsets per lane and a constant
    constexpr int KP = TT::WIDE ? 4 : CH % 8 == 0 ? 2 : 1;
    auto kc_at = [&](int st) { return ((4 * (st % KP) + kg) ^ TT::k_turn(col)) * 16 + st / KP * KP * 64; };
    constexpr int NP = PARTS ? 3 : 1;  // parts of a key or value
    const float *ks = (const float *)(kt + 2 * TT::SIDE) + kgp * SK + 4 * kg, *vs = ks + TK;  // 8-bit rows' scales
    if constexpr (I8) {
      // a tile of 16 keys at a time: its reads go out a tile ahead, and a tile's sums are put together while the
      // next one's multiply
      constexpr int NS = HD / 64;
      ti4 kf[2][NS], d[2][3];
      float4 k4[2];
      float kq[4] = {0.f, 0.f, 0.f, 0.f};
      auto read = [&](int x) {
        k4[x & 1] = *(const float4 *)(ks + 16 * x);
#pragma unroll
        for (int st = 0; st < NS; st++) kf[x & 1][st] = *(const ti4 *)(kb + x * 16 * ROWB + kc_at(st));
      };
      read(0);
#pragma unroll
      for (int x = 0; x <= NT; x++) {
        if (x + 1 < NT) read(x + 1);
        __builtin_amdgcn_sched_barrier(0);
        if (x < NT) {
#pragma unroll
          for (int p = 0; p < 3; p++) d[x & 1][p] = tree_zero();
#pragma unroll
          for (int st = 0; st < NS; st++)
#pragma unroll
            for (int p = 2; p >= 0; p--)
              d[x & 1][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[x & 1][st], qd[st][p], d[x & 1][p], 0, 0, 0);
        }
        if (x > 0) {
          const int y = x - 1;
          const float kk[4] = {kq[0], kq[1], kq[2], kq[3]};
#pragma unroll
          for (int i = 0; i < 4; i++)
            sc[y][i] = fmaf(tree_high(d[y & 1][2][i], d[y & 1][1][i]), 256.0f, __int_as_float(d[y & 1][0][i])) * kk[i];
        }
        if (x < NT) {
          kq[0] = k4[x & 1].x, kq[1] = k4[x & 1].y, kq[2] = k4[x & 1].z, kq[3] = k4[x & 1].w;
        }
      }
    } else if constexpr (B16) {
      // a step: 32 entries of one part for up to two tiles of keys, the next step's read while this one's multiply.
      // Small parts first; of two split operands the three products that come to 2^-24 at most are left out.
      constexpr int XS = NT > 1 ? 2 : 1, QS = HD / 32 * NP * (NT / XS);
      tb8 kf[2][XS];
      auto read = [&](int i, tb8(&to)[XS]) {
        const int st = i / (NP * (NT / XS)), f = NP - 1 - i / (NT / XS) % NP, x = i % (NT / XS) * XS;
#pragma unroll
        for (int e = 0; e < XS; e++) to[e] = *(const tb8 *)(kb + f * TT::PART + (x + e) * 16 * ROWB + kc_at(st));
      };
      read(0, kf[0]);
#pragma unroll
      for (int i = 0; i < QS; i++) {
        if (i + 1 < QS) read(i + 1, kf[(i + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        const int st = i / (NP * (NT / XS)), f = NP - 1 - i / (NT / XS) % NP, x = i % (NT / XS) * XS;
#pragma unroll
        for (int p = 2 - f; p >= 0; p--)
#pragma unroll
          for (int e = 0; e < XS; e++)
            sc[x + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i & 1][e], qb[st][p], sc[x + e], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int st = 0; st < HD / 16; st++) {
        float4 kf[NT];
#pragma unroll
        for (int x = 0; x < NT; x++) kf[x] = *(const float4 *)(kb + x * 16 * ROWB + kc_at(st));
#pragma unroll
        for (int x = 0; x < NT; x++) sc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x].x, qf[st].x, sc[x], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < NT; x++) sc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x].y, qf[st].y, sc[x], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < NT; x++) sc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x].z, qf[st].z, sc[x], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < NT; x++) sc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x].w, qf[st].w, sc[x], 0, 0, 0);
      }
    }
    float mt = -INFINITY;
    uint32_t hid = 0;  // the lane's keys that its row does not see
    if (base + TK > nc) {
      const int kfirst = base + kgp * SK + 4 * kg - nc;  // drafted row of the lane's first key, below 0 in the cache
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int j = kfirst + 16 * x + i;
          const bool see = j < 0 || (j < nd && (vis[node - node_lo][min(j, TREE_MAX - 1) >> 5] >> (j & 31) & 1));
          sc[x][i] = see ? (I8 ? sc[x][i] : sc[x][i] * c1) : -INFINITY;
          if (I8 && !see) hid |= 1u << (4 * x + i);
        }
    } else if constexpr (!I8) {
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) sc[x][i] *= c1;
    }
#pragma unroll
    for (int x = 0; x < NT; x++) mt = fmaxf(mt, fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3])));
    mt = tree_xor_max(mt);
    mt = fmaxf(m, I8 ? mt * qs : mt);
    // (8-bit rows: only past 2^8, their probabilities' digits being made for each stage's largest)
    if (__any(I8 ? mt > m + 8.0f : mt > m)) {
      if (I8 && !(mt > m + 8.0f)) mt = m;
      const float f = mt == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mt);
      l *= f;
#pragma unroll
      for (int x = 0; x < HD / 16; x++) o[x] *= f;
      m = mt;
    }
    const float ms = m == -INFINITY ? 0.0f : m;
    // (8-bit rows: m is a rounded product and the fused difference from it is not. Past 2^20 they would be apart by more than
    // 2^-4, by anything at scores of 2^32: the products there are rounded first. Row by row: a wave's rows are of several
    // users, and of padding nodes)
    float step = qs;
    const bool far = I8 && fabsf(ms) > 0x1p20f;
    if (I8 && __any(far)) {
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) sc[x][i] = far ? sc[x][i] * qs : sc[x][i];
      step = far ? 1.0f : qs;
    }
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        sc[x][i] = __builtin_amdgcn_exp2f(I8 ? fmaf(sc[x][i], step, -ms) : sc[x][i] - ms);
        l += sc[x][i];
      }

    // values
    if constexpr (I8) {
      float pv[NT][4], mx = 0.0f;
#pragma unroll
      for (int x = 0; x < NT; x++) {
        const float4 v4 = *(const float4 *)(vs + 16 * x);
        pv[x][0] = v4.x, pv[x][1] = v4.y, pv[x][2] = v4.z, pv[x][3] = v4.w;
      }
      if (base + TK > nc) {
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) pv[x][i] = hid >> (4 * x + i) & 1 ? 0.0f : pv[x][i];
      }
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          pv[x][i] *= sc[x][i];
          mx = fmaxf(mx, pv[x][i]);
        }
      // scales that are not finite, two a lane
      const float2 two = *(const float2 *)((const float *)(kt + 2 * TT::SIDE) + TK + kgp * SK + 2 * (lane % (SK / 2)));
      if (__any(!(fabsf(two.x) + fabsf(two.y) < INFINITY))) {
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!(hid >> (4 * x + i) & 1) && !(fabsf(vs[16 * x + i]) < INFINITY)) gone = __uint_as_float(0x7fc00000u);
      }
      mx = tree_xor_max(mx);
      const int e = max(__builtin_amdgcn_frexp_expf(mx), -100);
      const float f = __builtin_amdgcn_ldexpf(TREE_FIT, 23 - e), inv = __builtin_amdgcn_ldexpf(1.0f / TREE_FIT, e - 23);
      uint32_t pd[3][NT];
#pragma unroll
      for (int x = 0; x < NT; x++) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __float_as_uint(fmaf(pv[x][i], f, TREE_BIAS));  // rounded to a whole number
        tree_digits(u, pd[2][x], pd[1][x], pd[0][x]);
      }
      const int j = (lane & 15) >> 1, vr = 16 * (j >> 2) + 4 * kg + (j & 3), turn = TT::v_turn(vr);
      const char *vb = vt + (kgp * SK + vr) * ROWB + (lane & 1) * 8;
      constexpr int VP = TT::WIDE ? 16 : CH % 8 == 0 ? 8 : 4;
      const float inv256 = inv * 256.0f;
      // a tile's reads go out ahead, and its sums are added while the next one's multiply
      constexpr int ND = HD / 16, AHEAD = NT == 2 ? 2 : 1, NR = NT / 2;
      ti2 vf[AHEAD + 1][NR];
      ti4 d[2][3];
      auto read = [&](int dt) {
        const char *at = vb + (dt / VP * VP + ((dt % VP) ^ turn)) * 16;
#pragma unroll
        for (int h = 0; h < NR; h++)
          vf[dt % (AHEAD + 1)][h] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((tree_lds_i2 *)(at + h * 32 * ROWB));
      };
#pragma unroll
      for (int dt = 0; dt < AHEAD; dt++) read(dt);
#pragma unroll
      for (int dt = 0; dt <= ND; dt++) {
        if (dt + AHEAD < ND) read(dt + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        if (dt < ND) {
          const ti2 *v = vf[dt % (AHEAD + 1)];
#pragma unroll
          for (int p = 2; p >= 0; p--) {
            if constexpr (NT == 2) {
              d[dt & 1][p] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                  __builtin_bit_cast(long, v[0]), __builtin_bit_cast(long, ti2{(int)pd[p][0], (int)pd[p][1]}),
                  tree_zero(), 0, 0, 0);
            } else {
              d[dt & 1][p] = tree_zero();
            }
          }
          if constexpr (NT > 2) {
#pragma unroll
            for (int h = 0; h < NT / 4; h++)
#pragma unroll
              for (int p = 2; p >= 0; p--)
                d[dt & 1][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    ti4{v[2 * h].x, v[2 * h].y, v[2 * h + 1].x, v[2 * h + 1].y},
                    ti4{(int)pd[p][4 * h], (int)pd[p][4 * h + 1], (int)pd[p][4 * h + 2], (int)pd[p][4 * h + 3]},
                    d[dt & 1][p], 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (dt > 0) {
          const ti4 *e = d[(dt - 1) & 1];
#pragma unroll
          for (int i = 0; i < 4; i++)
            o[dt - 1][i] = fmaf(tree_high(e[2][i], e[1][i]), inv256, fmaf(__int_as_float(e[0][i]), inv, o[dt - 1][i]));
        }
      }
    } else if constexpr (B16) {
      const int cv = again(lane) & 15, xr = cv >> 2;
      const char *vb = vt + (kgp * SK + 4 * kg + xr) * ROWB + (cv & 1) * 8 + ((cv >> 1) & 1) * 16;
      constexpr int VP = TT::WIDE ? 8 : 4;
      const int turn = TT::v_turn(4 * kg + xr) >> 1;
      uint32_t pp[NT][3][2];
#pragma unroll
      for (int x = 0; x < NT; x++) {
        if constexpr (PARTS) {
#pragma unroll
          for (int i = 0; i < 2; i++)
            tree_round<false>(sc[x][2 * i], sc[x][2 * i + 1], pp[x][0][i], pp[x][1][i], pp[x][2][i]);
        } else {
          uint32_t h[3][4];
#pragma unroll
          for (int i = 0; i < 4; i++) tree_split(sc[x][i], h[0][i], h[1][i], h[2][i]);
#pragma unroll
          for (int p = 0; p < 3; p++) {
            pp[x][p][0] = tree_pack(h[p][0], h[p][1]);
            pp[x][p][1] = tree_pack(h[p][2], h[p][3]);
          }
        }
      }
      // a step: one part of 32 keys (16 where the wave has no more) for two tiles of entries
      constexpr int XS = NT > 1 ? 2 : 1, VS = HD / 32 * (NT / XS) * NP;
      ts4 vf[2][2][XS];
      auto read = [&](int i, ts4(&to)[2][XS]) {
        const int dt = i / (NP * (NT / XS)) * 2, x = i / NP % (NT / XS) * XS, f = NP - 1 - i % NP;
#pragma unroll
        for (int d = 0; d < 2; d++)
#pragma unroll
          for (int e = 0; e < XS; e++) {
            const int tile = (dt + d) / VP * VP + (((dt + d) % VP) ^ turn);
            to[d][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (tree_lds_s4 *)(vb + tile * 32 + f * TT::PART + (x + e) * 16 * ROWB));
          }
      };
      read(0, vf[0]);
#pragma unroll
      for (int i = 0; i < VS; i++) {
        if (i + 1 < VS) read(i + 1, vf[(i + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        const int dt = i / (NP * (NT / XS)) * 2, x = i / NP % (NT / XS) * XS, f = NP - 1 - i % NP;
#pragma unroll
        for (int p = 2 - f; p >= 0; p--)
#pragma unroll
          for (int d = 0; d < 2; d++) {
            if constexpr (XS == 2) {
              struct { ts4 lo, hi; } vv{vf[i & 1][d][0], vf[i & 1][d][1]};
              const rbt_u4 pv{pp[x][p][0], pp[x][p][1], pp[x + 1][p][0], pp[x + 1][p][1]};
              o[dt + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tb8, vv),
                                                                  __builtin_bit_cast(tb8, pv), o[dt + d], 0, 0, 0);
            } else {
              struct { uint32_t x, y; } pv{pp[0][p][0], pp[0][p][1]};
              o[dt + d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf[i & 1][d][0], __builtin_bit_cast(ts4, pv),
                                                                    o[dt + d], 0, 0, 0);
            }
          }
      }
    } else {
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const char *vb = vt + (kgp * SK + 16 * x + 4 * kg + i) * ROWB + col * 16;
#pragma unroll
          for (int dt = 0; dt < HD / 64; dt++) {
            const float4 v = *(const float4 *)(vb + dt * 256);
            o[4 * dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x, sc[x][i], o[4 * dt], 0, 0, 0);
            o[4 * dt + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.y, sc[x][i], o[4 * dt + 1], 0, 0, 0);
            o[4 * dt + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.z, sc[x][i], o[4 * dt + 2], 0, 0, 0);
            o[4 * dt + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.w, sc[x][i], o[4 * dt + 3], 0, 0, 0);
          }
        }
    }
  }

  if constexpr (I8) {
    gone = tree_xor_sum(gone);
#pragma unroll
    for (int d = 0; d < HD / 16; d++) o[d] += gone;
  } else if (nd > 1) {  // the non-finite values that were taken out, for the rows that see them; none in a healthy step
    for (int x = 0; x < TREE_MAX / 32; x++)
      for (uint32_t bits = dirty[x]; bits; bits &= bits - 1) {
        const int j = 32 * x + __ffs(bits) - 1;
        if (!active || !(vis[node - node_lo][x] >> (j & 31) & 1)) continue;
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int at = B16 ? 16 * d + 4 * kg + e : 64 * (d >> 2) + 16 * kg + 4 * e + (d & 3);
            const float v = tree_ld(vd + j * seq_row, at, KV == KV_BF16);
            o[d][e] += fabsf(v) < INFINITY ? 0.0f : v - v;
          }
      }
  }

  // the column's four lanes hold parts of the row's sum
  l = tree_xor_sum(l);
  const bool direct = np == 1 && !a.joined;
  // partial sums lie by 16-row tiles in the order of the lanes: quad 64 d + lane holds row col's entries
  // 16 d + 4 kg .. + 3, so that they are written and read in whole lines
  unit += rt * RW + rg;
  float *po = a.part + unit * 16 * HD;
  float2 *pm = a.part_ml + unit * 16;
  // entry e of value tile d is entry at(d, e) of the head
  if constexpr (KW > 1) {
    // join the key groups in LDS: every group's O and l scaled to the row's largest maximum
    constexpr int ST = HD + 4;
    if (kgp < KW && kg == 0) {
      ml[w][0][col] = m;
      ml[w][1][col] = l;
    }
    lds_barrier();
    float M = -INFINITY;
    for (int k = 0; k < KW; k++) M = fmaxf(M, ml[k * RW + rg][0][col]);
    const float Ms = M == -INFINITY ? 0.0f : M;
    const float f = __builtin_amdgcn_exp2f(m - Ms);
    float *oj = (float *)smem;
#pragma unroll
    for (int d = 0; d < HD / 16; d++) {
      if (kgp >= KW) break;
      float *to = oj + (w * 16 + col) * ST;
      if constexpr (B16) {
        *(float4 *)(to + 16 * d + 4 * kg) = make_float4(o[d][0] * f, o[d][1] * f, o[d][2] * f, o[d][3] * f);
      } else {
        const int g = d & ~3, e = d & 3;
        *(float4 *)(to + 16 * g + 16 * kg + 4 * e) =
            make_float4(o[g][e] * f, o[g + 1][e] * f, o[g + 2][e] * f, o[g + 3][e] * f);
      }
    }
    lds_barrier();
    // the waves of a row tile (those that only loaded too) share its rows' entries
    constexpr int Q4 = HD / 4;
    for (int u = kgp * 64 + lane; u < 16 * Q4; u += 64 * (NW / RW)) {
      const int r = u / Q4, e = u - r * Q4, rr = row0 + rg * 16 + r;
      if (rr >= rows) continue;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float Mr = -INFINITY, lr = 0.0f;
      for (int k = 0; k < KW; k++) {
        const float4 x = *(const float4 *)(oj + ((k * RW + rg) * 16 + r) * ST + 4 * e);
        v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
        Mr = fmaxf(Mr, ml[k * RW + rg][0][r]);
      }
      const float Mrs = Mr == -INFINITY ? 0.0f : Mr;
      for (int k = 0; k < KW; k++) lr += ml[k * RW + rg][1][r] * __builtin_amdgcn_exp2f(ml[k * RW + rg][0][r] - Mrs);
      if (direct) {
        const int nodr = tree_div(rr, a), hdr = kv * R + (rr - nodr * R);
        tree_store(a, b, nodr, hdr, 4 * e, v, lr);
      } else {
        *(float4 *)(po + ((e >> 2) * 64 + (e & 3) * 16 + r) * 4) = v;
        if (e == 0) pm[r] = make_float2(Mr, lr);
      }
    }
  } else {
    static_assert(B16, "the values' tiles are 16 entries wide");
    if (!active) return;
#pragma unroll
    for (int d = 0; d < HD / 16; d++) {
      const float4 v = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
      if (!direct)
        *(float4 *)(po + (d * 64 + lane) * 4) = v;
      else if (row < rows)
        tree_store(a, b, node, head, 16 * d + 4 * kg, v, l);
    }
    if (!direct && kg == 0) pm[col] = make_float2(m, l);
  }
}

template <int HD, int KV, int KW>
__global__ __launch_bounds__(tree_wide(KV, KW) ? 512 : 256, tree_wide(KV, KW) ? 1 : 2)
void k_tree(TreeArgs a) {
  tree_pass<HD, KV, KW>(a, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The pass over the prefixes (its first np workgroups) and the sequences' own in one launch: many rows against few, so
// that the second's trips to memory run beside the first's products where the chip has room for both (8 users behind 1500
// rows 36.7 -> 27.8 us, 11 trees of five behind 1001 f32 rows 34.6 -> 31.8).
template <int HD, int KVP, int KV, int KW>
__global__ __launch_bounds__(512, 1) void k_tree_both(TreeArgs p, TreeArgs a, int np) {
  const int id = blockIdx.x;
  if (id < np) {
    if (p.tiles > 1)
      tree_pass<HD, KVP, 1>(p, id, 0, 0);
    else
      tree_pass<HD, KVP, 1>(p, id % p.pieces, id / p.pieces, 0);
  } else {
    const int i = id - np, r = i / a.pieces;
    tree_pass<HD, KV, KW>(a, i - r * a.pieces, r % a.K, r / a.K);
  }
}

// The pieces of 16 rows joined. WP = 1: a workgroup takes 64 entries of the rows, 16 per wave; WP = 4: 16 entries, its
// waves take every fourth piece each and their sums are added in order. Lane by lane as the partial sums lie.
template <int WP>
__global__ __launch_bounds__(256) void k_tree_join(TreeArgs a, int TK) {
  __shared__ float wt[256][16], red[16][16];
  __shared__ float4 sum[WP > 1 ? 4 : 1][64];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, col = lane & 15, kv = blockIdx.y, b = blockIdx.z;
  const int nd = a.hd / 16, tile = WP > 1 ? blockIdx.x / nd : blockIdx.x * 4 / nd;
  const int d = WP > 1 ? blockIdx.x - tile * nd : blockIdx.x * 4 - tile * nd + w;
  const long ps = (long)a.B * a.K * a.t16, unit = ((long)b * a.K + kv) * a.t16 + tile;
  // Thread t takes row t % 16's maxima and sums (of up to 256 pieces: all are loaded at once, and so are this wave's
  // first partial outputs), ahead of the sequence's own numbers: pieces that it does not have are read, not used (one
  // node over 513 rows 13.6 -> 13.3 us, 64 over 32749 330 -> 328, on one MI355X in turn).
  const int r = t & 15, j0 = t >> 4, most = a.pieces - 1;
  float2 x[16];
#pragma unroll
  for (int k = 0; k < 16; k++)
    if (16 * k <= most) x[k] = a.part_ml[(min(j0 + 16 * k, most) * ps + unit) * 16 + r];
  constexpr int PF = 8;
  const int first = WP > 1 ? w : 0;
  const float *po = a.part + unit * 16 * a.hd + (d * 64 + lane) * 4;
  float4 y[PF];
#pragma unroll
  for (int k = 0; k < PF; k++) y[k] = *(const float4 *)(po + min(first + k * WP, most) * ps * 16 * a.hd);
  const int n = a.n_nodes[b], L = a.len[b];
  if (!tree_valid(a, n, L) || tile * 16 >= n * a.R) return;
  unsigned per, pieces;
  tree_pieces(a, L, TK, per, pieces);
  const int np = (int)pieces;
  if (np <= 1) return;
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < 16; k++)
    if (j0 + 16 * k < np) M = fmaxf(M, x[k].x);
  red[j0][r] = M;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; k++) M = fmaxf(M, red[k][r]);
  const float Ms = M == -INFINITY ? 0.0f : M;
  float l = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const int j = j0 + 16 * k;
    if (j >= np) break;
    const float f = __builtin_amdgcn_exp2f(x[k].x - Ms);
    wt[j][r] = f;
    l += x[k].y * f;
  }
  __syncthreads();
  red[j0][r] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; k++) l += red[k][col];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float4 y, int j) {
    const float f = wt[j][col];
    v = make_float4(v.x + y.x * f, v.y + y.y * f, v.z + y.z * f, v.w + y.w * f);
  };
#pragma unroll
  for (int k = 0; k < PF; k++)
    if (first + k * WP < np) add(y[k], first + k * WP);
#pragma unroll 8
  for (int j = first + PF * WP; j < np; j += WP) add(*(const float4 *)(po + j * ps * 16 * a.hd), j);
  if constexpr (WP > 1) {
    sum[w][lane] = v;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < 4; k++) {
      const float4 y = sum[k][lane];
      v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
    }
  }
  const int row = tile * 16 + col, i = tree_div(row, a);
  if (i < n) tree_store(a, b, i, kv * a.R + (row - i * a.R), 16 * d + 4 * (lane >> 4), v, l);
}

// What the pieces of a sequence and those of its prefix left, joined: a workgroup takes 16 rows of a sequence and 64
// entries, 16 per wave. `a` is the sequences' pass, `p` the prefixes'. Bound by trips to memory: the sequence's own sums, its
// gate and its numbers are asked for at once, then the prefix's sums, whose place the numbers tell.
__global__ __launch_bounds__(256) void k_prefix_join(TreeArgs a, TreeArgs p) {
  __shared__ float wt[512][16], red[16][16];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, col = lane & 15, kg = lane >> 4, kv = blockIdx.y, b = blockIdx.z;
  const int nd = a.hd / 16, tile = blockIdx.x * 4 / nd, d = blockIdx.x * 4 - tile * nd + w, TR = a.T * a.R;
  const long ps = (long)a.B * a.K * a.t16, pp = (long)p.K * p.t16, own = ((long)b * a.K + kv) * a.t16 + tile;
  const int r = t & 15, j0 = t >> 4, most = a.pieces - 1;
  // the first pieces' maxima, sums and outputs (of pieces that the sequence does not have too: read, not used)
  constexpr int PO = 4, PP = 16;
  const float *po = a.part + own * 16 * a.hd + (d * 64 + lane) * 4;
  const float2 ml0 = a.part_ml[(min(j0, most) * ps + own) * 16 + r];
  float4 yo[PO], yp[PP];
#pragma unroll
  for (int k = 0; k < PO; k++) yo[k] = *(const float4 *)(po + min(k, most) * ps * 16 * a.hd);
  const int row = tile * 16 + col, i = tree_div(row, a), h = kv * a.R + (row - i * a.R), e = 16 * d + 4 * kg;
  float gate[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.gate && i < a.T) {
    const float *g = a.gate + ((long)b * a.T + i) * a.gts + (long)h * a.ghs + e;
#pragma unroll
    for (int k = 0; k < 4; k++) gate[k] = g[k];
  }
  const int n = a.n_nodes[b], L = a.len[b];
  int g, f0, P;
  if (!tree_prefix(p, b, g, f0, P)) return;
  if (!tree_valid(a, n, L) || tile * 16 >= n * a.R) return;
  unsigned per, u1, u2 = 0;
  tree_pieces(a, L, a.tk, per, u1);
  if (P > 0) tree_pieces(p, P, p.tk, per, u2);
  const int n1 = (int)u1, n2 = (int)u2, np = n1 + n2;
  // row r of the tile among the prefix's partial sums
  const long pu = (long)kv * p.t16 + tree_tile0(p, f0, max(g, 0), 16);
  const int x0 = (b - f0) * TR + tile * 16, last = (b - f0) * TR + n * a.R - 1;
  const int xr = min(x0 + r, last), xc = min(x0 + col, last);
  const float *pq = p.part + (pu + xc / 16) * 16 * a.hd + (d * 64 + kg * 16 + xc % 16) * 4;
  const float2 *pm = p.part_ml + (pu + xr / 16) * 16 + xr % 16;
  float2 ml1 = make_float2(-INFINITY, 0.0f);
  if (n2 > 0) {
    ml1 = pm[min(j0, n2 - 1) * pp * 16];
#pragma unroll
    for (int k = 0; k < PP; k++) yp[k] = *(const float4 *)(pq + min(k, n2 - 1) * pp * 16 * a.hd);
  }
  float M = j0 < n1 ? ml0.x : -INFINITY;
  if (j0 < n2) M = fmaxf(M, ml1.x);
  for (int j = j0 + 16; j < n1; j += 16) M = fmaxf(M, a.part_ml[(j * ps + own) * 16 + r].x);
  for (int j = j0 + 16; j < n2; j += 16) M = fmaxf(M, pm[j * pp * 16].x);
  red[j0][r] = M;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; k++) M = fmaxf(M, red[k][r]);
  const float Ms = M == -INFINITY ? 0.0f : M;
  float l = 0.0f;
  auto weigh = [&](int at, float2 x) {
    const float f = __builtin_amdgcn_exp2f(x.x - Ms);
    wt[at][r] = f;
    l += x.y * f;
  };
  if (j0 < n1) weigh(j0, ml0);
  for (int j = j0 + 16; j < n1; j += 16) weigh(j, a.part_ml[(j * ps + own) * 16 + r]);
  if (j0 < n2) weigh(n1 + j0, ml1);
  for (int j = j0 + 16; j < n2; j += 16) weigh(n1 + j, pm[j * pp * 16]);
  __syncthreads();
  red[j0][r] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; k++) l += red[k][col];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float4 y, int j) {
    const float f = wt[j][col];
    v = make_float4(v.x + y.x * f, v.y + y.y * f, v.z + y.z * f, v.w + y.w * f);
  };
#pragma unroll
  for (int k = 0; k < PO; k++)
    if (k < n1) add(yo[k], k);
#pragma unroll 8
  for (int j = PO; j < n1; j++) add(*(const float4 *)(po + j * ps * 16 * a.hd), j);
#pragma unroll
  for (int k = 0; k < PP; k++)
    if (k < n2) add(yp[k], n1 + k);
#pragma unroll 8
  for (int j = PP; j < n2; j++) add(*(const float4 *)(pq + j * pp * 16 * a.hd), n1 + j);
  if (i >= n) return;
  float o[4] = {v.x / l, v.y / l, v.z / l, v.w / l};
  if (a.gate) {
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = __fmul_rn(o[k], rbt_sigmoid(gate[k]));
  }
  *(float4 *)(a.out + (((long)b * a.T + i) * a.H + h) * a.hd + e) = make_float4(o[0], o[1], o[2], o[3]);
}

// Workgroups of `threads` that a CU holds at once (their LDS and registers), asked once per kernel and size.
template <int HD, int KV, int KW>
static int tree_per_cu(int threads) {
  static std::atomic<int> known[9];  // by waves, up to 8
  std::atomic<int> &k = known[threads / 64];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_tree<HD, KV, KW>, threads,
                                                     TreeTile<HD, KV, KW>::LDS) !=
        hipSuccess) {
      (void)hipGetLastError();
      n = 1;
    }
    n = std::max(n, 1);
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}
template <int KV, int KW>
static int tree_per_cu(int hd, int threads) {
  return hd == 64    ? tree_per_cu<64, KV, KW>(threads)
         : hd == 128 ? tree_per_cu<128, KV, KW>(threads)
         : hd == 192 ? tree_per_cu<192, KV, KW>(threads)
                     : tree_per_cu<256, KV, KW>(threads);
}

// Threads of a workgroup.
static int tree_threads(const TreeArgs &a) {
  return a.kw > 1 || a.four ? 256 : a.kv16 || a.kv8 ? 64 * a.rw : 512;
}

// Pieces and row tiles for a call on the matrix cores.
bool tree_plan(const Ctx &c, TreeArgs &a) {
  a.rw = a.kw = a.tiles = a.pieces = 1;
  a.four = 0;
  int rw = 1, kw = 1;
  a.tiled = a.hd == 64 || a.hd == 128 || a.hd == 192 || a.hd == 256;
  if (!a.tiled) return true;
  // (a pass over prefixes: row tiles of a prefix of average size)
  const int R = a.H / a.K, t16 = a.pre ? (int)(((long)a.B * a.T * R + 16L * a.G - 1) / (16L * a.G)) : (a.T * R + 15) / 16;
  a.seqs = a.pre ? 1 : a.B;
  a.t16 = t16;
  a.R = R;
  a.magic = R == 1 ? 0 : (unsigned)((0x100000000ull + R - 1) / R);
  if (t16 <= 2) {
    rw = t16;
    kw = a.kv16 ? 4 / rw : 2;
  } else {
    kw = 1;
    a.tiles = (t16 + 7) / 8;
    rw = (t16 + a.tiles - 1) / a.tiles;
  }
  a.tiles = (t16 + rw - 1) / rw;
  a.rw = rw;
  a.kw = kw;
  if (a.pre) {
    a.tiles = (int)(((long)a.B * a.T * R + a.G * (16L * rw - 1)) / (16 * rw));
    a.t16 = (int)(((long)a.B * a.T * R + 15L * a.G) / 16);
  }
  a.tk = tree_tk(a.kv8 ? KV_I8 : a.kv16 ? KV_BF16 : KV_F32, kw);
  const int TK = a.tk, seqs = a.pre ? a.G : a.B;
  // Pieces by the time they should take, in microseconds. A workgroup starts and ends in 7 and takes `stage` per stage
  // (measured at head_dim 256, where a CU holds one; it goes with the head dim), and several pieces cost a second
  // launch and a write and read of their rows' partial sums. Equal sequences end together, so their workgroups count
  // by whole rounds of the chip; those of a batch are of any length: past one round they fill it evenly, at about
  // 0.8 of the longest each, and the last ones are waited for. A batch at a smaller head dim runs `hold` workgroups
  // beside each other on a CU: a stage is then mostly waiting, all but `busy` of it, and grows less with the head
  // dim, until the caches pass at 5.0 TB/s (sequences taken at three quarters of the longest; a sixth less with one
  // workgroup per CU, and evenly only where every CU has as many). One sequence keeps the first model, whatever its
  // head dim: with the batches' it took 5 to 13% longer. Measured over bf16 rows at head_dim 256: one node
  // over 4096 rows 113 us in one piece, 27 in 8, 17 in 32, 17 in 64; 64 nodes over 32749 rows 527 in 4, 311 in 8, 326
  // in 16, 368 in 32; 16 sequences of one node over 3000 to 6000 rows 186 in 1, 65 in 4, 74 in 8, 86 in 16. And with
  // 32 query heads over 8 KV heads, 32 sequences of up to 4096 rows (one piece fills every CU once): one node over
  // f32 rows of 128 254 in 1, 189 in 2, 212 in 8, of 64 183 in 1, 88 in 3, 102 in 8; 12 nodes over bf16 rows of 128
  // 133 in 1, 113 in 2, 124 in 8, of 64 90 in 1, 60 in 3, 66 in 8.
  const bool wide = rw > 4;  // two waves on a SIMD
  const double ncu = c.num_cu, base = (double)a.tiles * a.K * a.seqs;
  const double most = std::ceil((double)(a.max_len + (a.pre ? 0 : a.T)) / TK);
  const double part = a.hd / 256.0;
  // (from eight stages a CU on, a point between two measured ones: three sequences of 1001 rows, one and a half a CU,
  // 15.2 us with eight waves, 15.6 with four; eight of 4096, 32 a CU, 72 and 63)
  a.four = !a.kv16 && !a.kv8 && kw == 1 && a.hd <= 128 && rw <= 4 && seqs > 1 && base * most >= 8 * ncu;
  double stage, busy = 1.0, hold = 1.0;
  if (seqs == 1) {
    stage = (kw > 1 ? (a.kv8 ? 1.0 : a.kv16 ? 1.6 : 2.6) : a.kv8 ? (wide ? 5.0 : 3.0) : a.kv16 ? (wide ? 4.4 : 2.6) : (wide ? 6.5 : 4.0)) * part;
  } else if (kw > 1) {
    stage = (a.kv8 ? 1.0 : a.kv16 ? 1.6 : 2.6) * (0.3 + 0.7 * part);
    busy = 0.25;
    hold = a.kv8 ? tree_per_cu<KV_I8, 2>(a.hd, 256)
           : a.kv16 ? (kw == 4 ? tree_per_cu<KV_BF16, 4>(a.hd, 256) : tree_per_cu<KV_BF16, 2>(a.hd, 256))
                  : tree_per_cu<KV_F32, 2>(a.hd, 256);
  } else if (a.kv8) {
    stage = (wide ? 5.0 : 3.0) * (0.3 + 0.7 * part);
    busy = wide ? 0.9 : 0.6;
    hold = tree_per_cu<KV_I8, 1>(a.hd, tree_threads(a));
  } else if (a.kv16) {
    stage = (wide ? 4.4 : 2.6) * (0.3 + 0.7 * part);
    busy = wide ? 0.9 : 0.4;
    hold = tree_per_cu<KV_BF16, 1>(a.hd, tree_threads(a));
  } else {
    stage = (a.hd == 256 ? (wide ? 6.5 : 4.0) : (wide ? 4.4 : 3.6)) * (0.1 + 0.9 * part);
    busy = wide ? 0.9 : 0.65;
    hold = !a.four      ? tree_per_cu<KV_PARTS, 1>(a.hd, 512)
           : a.hd == 64 ? tree_per_cu<64, KV_PARTS4, 1>(256)
                        : tree_per_cu<128, KV_PARTS4, 1>(256);
  }
  const double bytes = (double)a.seqs * a.K * a.t16 * 16 * a.hd * 8.0;
  const double pass = seqs > 1 ? 0.75 * seqs * a.K * a.max_len * a.hd * (a.kv8 ? 2.0 : a.kv16 ? 4.0 : 8.0) / 5.0e6 : 0.0;
  double best = 0.0;
  long pieces = 1;
  auto consider = [&](long p) {
    // (partial sums of at most 256 MiB)
    if (p < 1 || p > 256 || (p > 1 && (p > most || bytes * p > 2.0 * (256u << 20)))) return;
    const double groups = base * p, rounds = groups / (ncu * hold), beside = std::min(hold, std::ceil(groups / ncu));
    const double one = 7.0 + stage * std::max(1.0, beside * busy) * std::ceil(most / p);
    double t = rounds <= 1.0 ? one : seqs == 1 ? std::ceil(rounds) * one : (0.8 * rounds + 0.4) * one;
    const double uneven = rounds > 1.0 ? 1.0 : beside * ncu / groups;
    t = std::max(t, pass * uneven * (hold > 1.0 && groups <= ncu ? 1.2 : 1.0));
    if (p > 1) t += 4.0 + bytes * p / 1.2e7;
    if (best == 0.0 || t < best) best = t, pieces = p;
  };
  consider(1);
  for (long p = 2; p <= 256; p += p < 16 ? 1 : p / 8) consider(p);
  for (int k = 1; k <= 4; k++) consider((long)(k * ncu * hold / base));
  a.per = (unsigned)((long)((most + pieces - 1) / pieces) * TK);
  a.pieces = (int)std::max(1L, (a.max_len + a.per - 1) / (long)a.per);
  // a launch holds fewer than 2^32 threads in x
  if (a.tiles > 1 && ((long)a.pieces * a.K * a.seqs + 7) / 8 * 8 * a.tiles > (1L << 23) - 1) return false;
  return true;
}

size_t tree_part_floats(const TreeArgs &a) {
  return a.pieces > 1 || a.joined ? (size_t)a.pieces * a.seqs * a.K * a.t16 * 16 * (a.hd + 2) : 0;
}

template <int HD, int KV, int KW>
static hipError_t run_tree(const Ctx &c, const TreeArgs &a) {
  constexpr int lds = TreeTile<HD, KV, KW>::LDS;
  static_assert(4 * 16 * (HD + 4) * 4 <= lds || KW == 1, "the key groups' join fits the stages' LDS");
  const long groups = (long)a.pieces * a.K * a.seqs;
  const long blocks = (groups + 7) / 8 * 8 * a.tiles;
  const dim3 grid = a.tiles > 1 ? dim3((unsigned)blocks) : dim3(a.pieces, a.K, a.seqs);
  launch_ks(c, k_tree<HD, KV, KW>, grid, dim3(tree_threads(a)), (unsigned)lds, a);
  return hipGetLastError();
}

template <int HD>
static hipError_t run_tree_hd(const Ctx &c, const TreeArgs &a) {
  if (a.kv8)
    return a.kw == 2 ? run_tree<HD, KV_I8, 2>(c, a) : run_tree<HD, KV_I8, 1>(c, a);
  if (a.kv16)
    return a.kw == 4   ? run_tree<HD, KV_BF16, 4>(c, a)
           : a.kw == 2 ? run_tree<HD, KV_BF16, 2>(c, a)
                       : run_tree<HD, KV_BF16, 1>(c, a);
  if constexpr (HD <= 128)
    if (a.four) return run_tree<HD, KV_PARTS4, 1>(c, a);
  return a.kw == 2 ? run_tree<HD, KV_F32, 2>(c, a) : run_tree<HD, KV_PARTS, 1>(c, a);
}

static hipError_t run_tree_pass(const Ctx &c, const TreeArgs &a) {
  return a.hd == 64 ? run_tree_hd<64>(c, a) : a.hd == 128 ? run_tree_hd<128>(c, a)
         : a.hd == 192 ? run_tree_hd<192>(c, a) : run_tree_hd<256>(c, a);
}

hipError_t launch_tree(const Ctx &c, const TreeArgs &a) {
  if (!a.tiled) {
    const bool plain = a.parent && !a.kv8 && !a.in_cache && a.G == 0;
    launch_k(c, plain ? k_tree_any<false> : k_tree_any<true>, dim3(a.H, a.T, a.B), dim3(256), a);
    return hipGetLastError();
  }
  const hipError_t e = run_tree_pass(c, a);
  if (e != hipSuccess || a.pieces == 1) return e;
  // few rows, many pieces: the pieces too over the waves
  if (a.pieces > 4 && (long)a.t16 * a.K * a.B <= 256)
    launch_k(c, k_tree_join<4>, dim3(a.t16 * (a.hd / 16), a.K, a.B), dim3(256), a, a.tk);
  else
    launch_k(c, k_tree_join<1>, dim3(a.t16 * (a.hd / 64), a.K, a.B), dim3(256), a, a.tk);
  return hipGetLastError();
}

void tree_prefix_args(const TreeArgs &a, TreeArgs &p) {
  p = a;
  p.pre = 1;
  p.kc = a.kp;
  p.vc = a.vp;
  p.kcs = a.kps;
  p.vcs = a.vps;
  p.len = a.prefix_len;
  p.cap = a.pcap;
  p.max_len = a.max_prefix;
  p.in_cache = 0;
  p.joined = 1;
}

// False: two launches are better. (8-bit rows of 192 or 256 at more workgroups than CUs: the prefixes' stages of 128
// keys leave a CU one workgroup, where a pass over own rows by itself has two. 32 users behind 8000 int8 rows 80 us,
// 90 in one launch; with bf16 rows of 256, one workgroup a CU in both, 64 behind 4096 86.5 and 84.2, 8 behind
// 6000 43.8 and 36.7; with rows of 128, 64 behind 4096 54.2 and 49.2, 32 behind 8000 int8 ones 56.2 and 55.5.)
template <int HD, int KVP, int KV, int KW>
static bool run_tree_both(const Ctx &c, const TreeArgs &p, const TreeArgs &a) {
  constexpr int lp = TreeTile<HD, KVP, 1>::LDS, la = TreeTile<HD, KV, KW>::LDS, lds = lp > la ? lp : la;
  const long groups = (long)p.pieces * p.K, np = p.tiles > 1 ? (groups + 7) / 8 * 8 * p.tiles : groups;
  const long own = (long)a.pieces * a.K * a.B;
  if (np + own >= 1L << 22 || (KV == KV_I8 && HD > 128 && np + own > c.num_cu)) return false;
  const int threads = std::max(tree_threads(p), tree_threads(a));
  launch_ks(c, k_tree_both<HD, KVP, KV, KW>, dim3((unsigned)(np + own)), dim3(threads), (unsigned)lds, p, a, (int)np);
  return true;
}
template <int HD>
static bool run_tree_both_hd(const Ctx &c, const TreeArgs &p, const TreeArgs &a) {
  // (where the prefixes have three row tiles or more, a sequence one, or two in int8 and f32)
  if (p.kw != 1 || p.four || a.kw != (a.kv16 ? 4 : 2) || a.tiles != 1) return false;
  return a.kv8    ? run_tree_both<HD, KV_I8, KV_I8, 2>(c, p, a)
         : a.kv16 ? run_tree_both<HD, KV_BF16, KV_BF16, 4>(c, p, a)
                  : run_tree_both<HD, KV_PARTS, KV_F32, 2>(c, p, a);
}

hipError_t launch_prefix(const Ctx &c, const TreeArgs &a, const TreeArgs &p) {
  const bool one = a.hd == 64    ? run_tree_both_hd<64>(c, p, a)
                   : a.hd == 128 ? run_tree_both_hd<128>(c, p, a)
                   : a.hd == 192 ? run_tree_both_hd<192>(c, p, a)
                                 : run_tree_both_hd<256>(c, p, a);
  hipError_t e = one ? hipGetLastError() : run_tree_pass(c, p);
  if (!one && e == hipSuccess) e = run_tree_pass(c, a);
  if (e != hipSuccess) return e;
  const int tiles = (a.T * a.R + 15) / 16;
  launch_k(c, k_prefix_join, dim3(tiles * (a.hd / 64), a.K, a.B), dim3(256), a, p);
  return hipGetLastError();
}

}  // namespace rbt

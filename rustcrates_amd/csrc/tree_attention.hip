// tree_attention.hip — attention of a tree of drafted tokens over the KV cache.
//
// Each node of a sequence's tree attends over the committed rows and over its
// own ancestors among the drafted ones, whose rows lie behind the committed
// ones in the cache (TreeAttn in serving.hpp has the formula).  A node at depth
// g stands where an ordinary decode step would put the g-th next token, so its
// bias column is kv_len + g and a chain of nodes gives what decode steps give.
// A row that a node does not see never enters its sums, finite or not.
//
// k_tree_split: one block per (chunk of slots, head, sequence, up to 16 NG
// nodes).  Its four waves are NG groups of 16 nodes by 4 / NG that share the
// chunk's 16-slot tiles, each with a running maximum and sum (one pass over the
// keys and values):
//   S^T = K Q^T   Re(q k) is a real product of length 2 dh: (kr, ki) with
//                 (qr, -qi) scaled.  A lane holds key row lane % 16 and, of each
//                 four complex columns, lane / 16: one 16-byte load feeds two MFMAs.
//   O^T += V^T P^T  element e of S^T's tile is slot 4 e + lane / 16 of node
//                 lane % 16, which is the B operand of the e-th step: the
//                 weights go from one product to the next in their registers.
// So keys and values go straight from memory to the matrix cores, each once per
// wave, and LDS holds the queries alone, in the order the lanes read them.  A
// tile's keys are requested once the last tile's scores are formed, its values
// once the last tile's output is.  Waves, then chunks (k_tree_join) are merged
// by their maxima.
#include <algorithm>
#include <cmath>

#include "attn_run.hpp"
#include "serving.hpp"

namespace mitok {

// chunk partials: max, sum and unnormalised output of a node, and the scores
// of the weighed nodes
struct TreeWs {
  double* m = nullptr;   // [B][H][n][nsplit]
  double* l = nullptr;
  double2* o = nullptr;  // [B][H][n][nsplit][dh] (nsplit > 1)
  double* x = nullptr;   // [B][H][T][weigh]
};

// A block's place: chunk entry * H + head, and its first node.
struct TreeAt {
  int b, h, bh, L, cnt, t0, t1, s, n0;
  const unsigned long long* seen;  // of the sequence's nodes
  const int* depth;
  __device__ __forceinline__ TreeAt(const TreeAttn& a, const TreePlan& p, const OpTable& own, int nodes) {
    const int e = blockIdx.x / a.H;
    const int4 c = op_array<int4>(a.tab, own, p.chunks)[e];
    b = __builtin_amdgcn_readfirstlane(c.x);
    t0 = __builtin_amdgcn_readfirstlane(c.y);
    t1 = __builtin_amdgcn_readfirstlane(c.z);
    s = __builtin_amdgcn_readfirstlane(c.w);
    h = blockIdx.x - e * a.H;
    bh = b * a.H + h;
    L = op_int(a.tab, own, a.kv_len, b);
    cnt = op_int(a.tab, own, a.count, b);
    seen = op_array<unsigned long long>(a.tab, own, a.seen) + (long)b * a.n * a.words;
    depth = op_array<int>(a.tab, own, a.depth) + (long)b * a.n;
    n0 = blockIdx.y * nodes;
  }
  // rows of nodes [n0, n0 + nodes) that are not used: zero, by the sequence's first chunk
  __device__ __forceinline__ void clear(const TreeAttn& a, int nodes) const {
    if (s) return;
    const int from = max(n0, cnt), rows = min(n0 + nodes, a.n) - from;
    for (int x = threadIdx.x; x < rows * a.dh; x += 256)
      a.out[((long)b * a.n + from + x / a.dh) * a.ldo + (long)h * a.dh + x % a.dh] = make_double2(0.0, 0.0);
  }
};

// Bits e of a tile's slots t + 4 e + kq that node i sees; a tile of committed slots: all
__device__ __forceinline__ unsigned tree_sees(const TreeAttn& a, const TreeAt& at, int t, int kq, int i) {
  if (t + 16 <= at.L) return 15u;
  unsigned vis = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = t + 4 * e + kq - at.L;
    bool see = j < 0;
    if (j >= 0 && j < at.cnt && i < at.cnt) see = (at.seen[i * a.words + (j >> 6)] >> (j & 63)) & 1;
    if (see) vis |= 1u << e;
  }
  return vis;
}
// the biases of slots t + 4 e + kq (0 without any)
__device__ __forceinline__ void tree_bias(const TreeAttn& a, const TreeAt& at, int t, int kq, double (&bf)[4]) {
  const double* bias = a.bias + (long)at.h * a.bias_stride;
  if (!a.bias) return;
  if (t + 16 <= at.L) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bf[e] = ld_glb(bias + t + kq + 4 * e);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    int col = min(t + 4 * e + kq, at.t1 - 1);
    if (col >= at.L) col = at.L + at.depth[col - at.L];
    bf[e] = bias[col];
  }
}
// the weighed nodes' scores, [slot][node]
__device__ __forceinline__ void tree_scores(const TreeAttn& a, const TreePlan& p, const TreeWs& ws, const TreeAt& at,
                                            int t, int kq, int i, const v4d& s) {
  if (i >= a.weigh) return;
  double* x = ws.x + ((long)at.bh * p.T + t) * a.weigh + (uint32_t)(kq * a.weigh + i);
  if (t + 16 <= at.t1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) *(MITOK_GLOBAL double*)(x + 4 * e * (uint32_t)a.weigh) = s[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (t + 4 * e + kq < at.t1) x[4 * e * (uint32_t)a.weigh] = s[e];
}

// A node's output row element: final where the sequence has one chunk, else the chunk's part.
__device__ __forceinline__ void tree_put(const TreeAttn& a, const TreePlan& p, const TreeWs& ws, const TreeAt& at, int k,
                                         int e, double2 v, double sum) {
  if (p.nsplit == 1) a.out[((long)at.b * a.n + k) * a.ldo + (long)at.h * a.dh + e] = make_double2(v.x / sum, v.y / sum);
  else ws.o[(((long)at.bh * a.n + k) * p.nsplit + at.s) * a.dh + e] = v;
}
__device__ __forceinline__ void tree_put_sum(const TreeAttn& a, const TreePlan& p, const TreeWs& ws, const TreeAt& at,
                                             int i, double m, double l) {
  if (i >= at.cnt || (p.nsplit == 1 && i >= a.weigh)) return;
  const long x = ((long)at.bh * a.n + i) * p.nsplit + at.s;
  ws.m[x] = m;
  ws.l[x] = l;
}

// What bounds it: the bytes of keys and values where a tile has one or few
// nodes (64 sequences of 12 heads and 400 to 511 rows, head dim 64, one node:
// 725 MB in 140 us, 5.1 TB/s, as a large copy runs); with 16 nodes 182 MB in 51
// us, a block's start and end (8 us of its 50) and the longest sequence.  One
// node takes the matrix instructions too: the 15 unused rows cost nothing that
// the memory does not hide.  Above head dim 64 a tile's rows no longer fit the
// registers ahead of it and are requested among its products, which wait for
// them: 32 sequences of 16 nodes, 8 heads of 128, 362 MB in 210 us.  Above 128
// the outputs alone fill the registers (272 VGPRs spilled): 4 heads of 256, the
// same bytes in 320 us.
template <int DHP, int NG, bool FULL>
__global__ __launch_bounds__(256, DHP <= 128 ? 2 : 1) void k_tree_split(TreeAttn a, TreePlan p, TreeWs ws, OpTable own) {
  constexpr int KG = 4 / NG;       // waves that share a node group's slots
  constexpr int U = DHP / 4;       // 16-byte key loads of a lane per tile, two MFMAs each
  constexpr int CT = DHP / 16;     // 16-column tiles of the values
  constexpr bool PRE = DHP <= 64;  // the next tile's rows wait in registers
  constexpr int OSTR = DHP + 1;    // LDS row of a node's output: nodes in different banks
  constexpr int PARTS = DHP <= 64 ? KG : 1;  // LDS holds this many waves' outputs of each node group
  constexpr size_t Q_BYTES = (size_t)NG * U * 64 * sizeof(double2);
  constexpr size_t O_BYTES = (size_t)PARTS * NG * 16 * OSTR * sizeof(double2);
  __shared__ __align__(16) unsigned char lds[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
  __shared__ double sm[4][16], sl[4][16], sum[NG][16];
  double2* qs = (double2*)lds;  // [NG][U][64], then outputs [PARTS][NG * 16][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ng = wave % NG, kg = wave / NG;
  const int node = lane & 15, kq = lane >> 4, dh = a.dh;
  const TreeAt at(a, p, own, 16 * NG);
  at.clear(a, 16 * NG);
  if (at.n0 >= at.cnt) return;
  const int t0 = at.t0, t1 = at.t1;
  const double2* K = a.kc + (long)at.bh * a.ctx * dh;
  const double2* V = a.vc + (long)at.bh * a.ctx * dh;
  const int i = at.n0 + 16 * ng + node;  // this lane's node
  const double2* qw = qs + ng * U * 64 + lane;

  // a tile's key row of this lane and its value rows 4 q + kq; a slot past the
  // end reads the last one's, with weight 0.  Padded columns: keys of 0 (0 times
  // an infinity would be NaN), and value columns that nobody reads.
  const auto key_at = [&](int t, int u) {
    const uint32_t x = (uint32_t)min(node, t1 - 1 - t) * (uint32_t)dh + kq;
    if (!FULL && 4 * u + kq >= dh) return make_double2(0.0, 0.0);
    return ld_glb(K + (long)t * dh + x + 4 * u);
  };
  const auto value_at = [&](int t, int q, int c) {
    const uint32_t x = (uint32_t)min(4 * q + kq, t1 - 1 - t) * (uint32_t)dh;
    if (FULL) return ld_glb(V + (long)t * dh + (x + node) + 16 * c);
    return ld_glb(V + (long)t * dh + (x + (uint32_t)min(node + 16 * c, dh - 1)));
  };
  double2 kf[PRE ? U : 1], vf[PRE ? 4 : 1][PRE ? CT : 1];
  double bf[4] = {0.0, 0.0, 0.0, 0.0};
  const auto load_keys = [&](int t) {
    if constexpr (PRE) {
#pragma unroll
      for (int u = 0; u < U; ++u) kf[u] = key_at(t, u);
    }
    tree_bias(a, at, t, kq, bf);
  };
  const auto load_values = [&](int t) {
    if constexpr (PRE) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int c = 0; c < CT; ++c) vf[q][c] = value_at(t, q, c);
    }
  };
  int t = t0 + 16 * kg;
  if (t < t1) {
    load_keys(t);
    load_values(t);
  }
  // the queries, behind the first tile's loads
  for (int x = tid; x < NG * U * 64; x += 256) {
    const int ln = x & 63, u = (x >> 6) % U, g = x / (64 * U);
    const int r = at.n0 + 16 * g + (ln & 15), e = 4 * u + (ln >> 4);
    double2 q = make_double2(0.0, 0.0);
    if (r < at.cnt && e < dh) q = a.q[((long)at.b * a.n + r) * a.ldq + (long)at.h * dh + e];
    qs[x] = make_double2(q.x * a.scale, -q.y * a.scale);
  }
  __syncthreads();

  AttnRun<DHP> run;
  for (; t < t1; t += 16 * KG) {
    v4d s = {0.0, 0.0, 0.0, 0.0}, z = s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const double2 k = PRE ? kf[PRE ? u : 0] : key_at(t, u), q = qw[u * 64];
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(k.x, q.x, s, 0, 0, 0);
      z = __builtin_amdgcn_mfma_f64_16x16x4f64(k.y, q.y, z, 0, 0, 0);
      if (u % (PRE ? 4 : 16) == (PRE ? 3 : 15)) __builtin_amdgcn_sched_barrier(0);  // so many operands at a time in registers
    }
    const unsigned vis = tree_sees(a, at, t, kq, i);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = (vis >> e & 1) && t + 4 * e + kq < t1 ? s[e] + z[e] + bf[e] : -INFINITY;
    tree_scores(a, p, ws, at, t, kq, i, s);
    const bool more = t + 16 * KG < t1;
    if (more) load_keys(t + 16 * KG);
    run.soften(s);
    const bool drafted = t + 16 > at.L;
    bool fine = true;
    if (PRE && drafted) {
#pragma unroll
      for (int q = 0; q < (PRE ? 4 : 0); ++q)
#pragma unroll
        for (int c = 0; c < CT; ++c) fine &= attn_finite(vf[q][c]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        double2 v = PRE ? vf[PRE ? q : 0][PRE ? c : 0] : value_at(t, q, c);
        if (!PRE && drafted) fine &= attn_finite(v);
        run.output(s, q, c, v);
      }
      if (!PRE) __builtin_amdgcn_sched_barrier(0);
    }
    if (more) load_values(t + 16 * KG);
    if (__ballot(!fine)) run.add_left_out([&](int k) { return V + (long)(t + k) * dh; }, dh, t1 - t, s, vis);
  }

  // the waves of a node group, rescaled to their common maximum and added in order
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) sm[wave][node] = run.m, sl[wave][node] = run.l;
  __syncthreads();  // and the queries' last read
  double M = -INFINITY;
#pragma unroll
  for (int g = 0; g < KG; ++g) M = fmax(M, sm[g * NG + ng][node]);
  const double base = M == -INFINITY ? 0.0 : M;
  double Ls = 0.0;
#pragma unroll
  for (int g = 0; g < KG; ++g) Ls += sl[g * NG + ng][node] * exp(sm[g * NG + ng][node] - base);
  const double f = exp(run.m - base);
#pragma unroll
  for (int g = 0; g < KG; g += PARTS) {
    if (kg / PARTS * PARTS == g && i < at.cnt) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          double2* to = os + ((kg - g) * NG * 16 + 16 * ng + node) * OSTR + 16 * c + 4 * e + kq;
          const double2 v = make_double2(run.o_re[c][e] * f, run.o_im[c][e] * f);
          *to = g ? cadd(*to, v) : v;
        }
    }
    __syncthreads();
  }
  if (kg == 0 && kq == 0) {
    sum[ng][node] = Ls;
    tree_put_sum(a, p, ws, at, i, M, Ls);
  }
  __syncthreads();
  for (int x = tid; x < min(16 * NG, at.cnt - at.n0) * dh; x += 256) {
    const int r = x / dh, e = x - r * dh;
    double2 v = os[r * OSTR + e];
#pragma unroll
    for (int g = 1; g < PARTS; ++g) v = cadd(v, os[(g * NG * 16 + r) * OSTR + e]);
    tree_put(a, p, ws, at, at.n0 + r, e, v, sum[r >> 4][r & 15]);
  }
}

// 33 nodes and more: every wave has 16 nodes of its own and the block's tiles
// are shared.  A wave requests a quarter of the next tile, in the order the
// matrix cores take it, among the first products of the current one and leaves
// it in LDS after the last: a load has most of a tile's time to arrive.  The queries
// wait in registers.  Bound by double MFMAs and the softmax's double arithmetic,
// which take turns on a SIMD: 4 sequences of 12 heads, 1964 to 2048 slots and 64
// nodes at head dim 64 take 90 us, 48% of it MFMAs (the padded products alone
// are 44 us).  Head dim 128, whose queries and outputs leave 11 VGPRs spilled
// (26 padded) at one wave a SIMD, takes 222 us for twice the products.  Tiles of
// a wave's own would be read four times through the caches.
template <int DHP, bool FULL>
__global__ __launch_bounds__(256, DHP <= 64 ? 2 : 1) void k_tree_shared(TreeAttn a, TreePlan p, TreeWs ws, OpTable own) {
  constexpr int U = DHP / 4, CT = DHP / 16;
  constexpr int F = U + 4 * CT;    // 1 KB fragments of a tile: keys [U], values [4][CT]
  constexpr int PER = F / 4;       // of each wave
  constexpr int OSTR = DHP + 1;
  constexpr size_t T_BYTES = 2 * (size_t)F * 64 * sizeof(double2), O_BYTES = (size_t)64 * OSTR * sizeof(double2);
  __shared__ __align__(16) unsigned char lds[T_BYTES > O_BYTES ? T_BYTES : O_BYTES];
  __shared__ double sum[64];
  __shared__ int left_out;  // some value stayed out of a tile
  double2* tiles = (double2*)lds;  // [2][F][64], then outputs [64][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int node = lane & 15, kq = lane >> 4, dh = a.dh;
  const TreeAt at(a, p, own, 64);
  at.clear(a, 64);
  if (at.n0 >= at.cnt) return;
  const int t0 = at.t0, t1 = at.t1;
  const double2* K = a.kc + (long)at.bh * a.ctx * dh;
  const double2* V = a.vc + (long)at.bh * a.ctx * dh;
  const int i = at.n0 + 16 * wave + node;
  // This wave's fragments of the tile at t: value columns 16 c + lane % 16 of row
  // 4 q + kq, and keys, of which four lanes load 64 bytes of a row (a quarter
  // wave then touches 4 lines, not 16) and leave them where the products' lanes
  // read them; kq's rotation of the row keeps both sides off shared banks.
  // Padding as in k_tree_split.
  const int krow = lane >> 2, kcol = lane & 3;
  const int kput = kcol * 16 + ((krow + 4 * kcol) & 15), kget = kq * 16 + ((node + 4 * kq) & 15);
  double2 next[PER];
  const auto fetch_one = [&](int t, int j) {
    if (j < U / 4) {
      const int u = wave * (U / 4) + j;
      const uint32_t x = (uint32_t)min(krow, t1 - 1 - t) * (uint32_t)dh + kcol + 4 * u;
      next[j] = FULL || 4 * u + kcol < dh ? ld_glb(K + (long)t * dh + x) : make_double2(0.0, 0.0);
    } else {
      const int c = j - U / 4;
      const uint32_t x = (uint32_t)min(4 * wave + kq, t1 - 1 - t) * (uint32_t)dh;
      next[j] = ld_glb(V + (long)t * dh + (x + (FULL ? node + 16 * c : min(node + 16 * c, dh - 1))));
    }
  };
  // into LDS; values of the nodes' own slots that are not finite stay out
  const auto leave = [&](int buf, int t) {
    if (t + 16 > at.L) {
      bool fine = true;
#pragma unroll
      for (int c = 0; c < CT; ++c) fine &= attn_finite(next[U / 4 + c]);
      if (!fine) left_out = 1;
    }
    double2* to = tiles + buf * F * 64;
#pragma unroll
    for (int j = 0; j < U / 4; ++j) to[(wave * (U / 4) + j) * 64 + kput] = next[j];
#pragma unroll
    for (int c = 0; c < CT; ++c) to[(U + wave * CT + c) * 64 + lane] = next[U / 4 + c];
  };
  if (tid == 0) left_out = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) fetch_one(t0, j);
  double2 qf[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = 4 * u + kq;
    double2 q = make_double2(0.0, 0.0);
    if (i < at.cnt && e < dh) q = a.q[((long)at.b * a.n + i) * a.ldq + (long)at.h * dh + e];
    qf[u] = make_double2(q.x * a.scale, -q.y * a.scale);
  }
  __syncthreads();
  leave(0, t0);
  __syncthreads();

  AttnRun<DHP> run;
  int buf = 0;
  for (int t = t0; t < t1; t += 16, buf ^= 1) {
    const double2* tile = tiles + buf * F * 64;
    double bf[4] = {0.0, 0.0, 0.0, 0.0};
    tree_bias(a, at, t, kq, bf);
    const int tn = min(t + 16, t1 - 1);  // the next tile's loads, spread over the products
    v4d s = {0.0, 0.0, 0.0, 0.0}, z = s;
#pragma unroll
    for (int g = 0; g < U / 4; ++g) {
#pragma unroll
      for (int j = 0; j < PER / (U / 4); ++j) fetch_one(tn, g * (PER / (U / 4)) + j);
      double2 k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = tile[(4 * g + j) * 64 + kget];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = __builtin_amdgcn_mfma_f64_16x16x4f64(k[j].x, qf[4 * g + j].x, s, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f64_16x16x4f64(k[j].y, qf[4 * g + j].y, z, 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const unsigned vis = tree_sees(a, at, t, kq, i);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = (vis >> e & 1) && t + 4 * e + kq < t1 ? s[e] + z[e] + bf[e] : -INFINITY;
    tree_scores(a, p, ws, at, t, kq, i, s);
    run.soften(s);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int c = 0; c < CT; ++c) run.output(s, q, c, tile[(U + q * CT + c) * 64 + lane]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (t + 16 > at.L && left_out) run.add_left_out([&](int k) { return V + (long)(t + k) * dh; }, dh, t1 - t, s, vis);
    leave(buf ^ 1, t + 16);  // read by nobody since the last barrier (after the last tile: by nobody at all)
    __syncthreads();
  }
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) {
    sum[16 * wave + node] = run.l;
    tree_put_sum(a, p, ws, at, i, run.m, run.l);
  }
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      os[(16 * wave + node) * OSTR + 16 * c + 4 * e + kq] = make_double2(run.o_re[c][e], run.o_im[c][e]);
  __syncthreads();
  for (int x = tid; x < min(64, at.cnt - at.n0) * dh; x += 256) {
    const int r = x / dh, e = x - r * dh;
    tree_put(a, p, ws, at, at.n0 + r, e, os[r * OSTR + e], sum[r]);
  }
}

// Joins the chunks: blocks y < oparts the outputs, the others the weights of
// 256 slots, or of TREE_SLOTS and 16 lanes to a slot where many nodes are
// weighed; a grid of at most TREE_PARTS such blocks walks a longer cache.
// Bound by its launch where little was split (4 us), else by the parts and
// scores it reads: 23 us for 64 weighed nodes of 48 heads and 2000 slots (49 MB
// of scores) and their parts of ten chunks (32 MB).  Joining in the
// last chunk's block instead was slower throughout (one token 28 -> 30 us a
// call, 64 sequences 164 -> 175): the parts then pass the XCD's own cache.
constexpr int TREE_FEW = 4, TREE_SLOTS = 64, TREE_PARTS = 16384;
__global__ __launch_bounds__(256) void k_tree_join(TreeAttn a, TreePlan p, TreeWs ws, int oparts, OpTable own) {
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, tid = threadIdx.x;
  const int L = op_int(a.tab, own, a.kv_len, b), cnt = op_int(a.tab, own, a.count, b), T = cnt ? L + cnt : 0;
  const int ns = op_int(a.tab, own, p.splits, b);
  if ((int)blockIdx.y < oparts) {
    const int x = blockIdx.y * 256 + tid, i = x / a.dh, e = x - i * a.dh;
    if (i >= cnt) return;
    const long at = ((long)bh * a.n + i) * p.nsplit;
    double M = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < ns; ++s) M = fmax(M, ws.m[at + s]);
    const double base = M == -INFINITY ? 0.0 : M;
    double l = 0.0;
    double2 v = make_double2(0.0, 0.0);
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
      const double f = exp(ws.m[at + s] - base);
      const double2 o = ws.o[(at + s) * a.dh + e];
      l += ws.l[at + s] * f;
      v = make_double2(v.x + o.x * f, v.y + o.y * f);
    }
    a.out[((long)b * a.n + i) * a.ldo + (long)h * a.dh + e] = make_double2(v.x / l, v.y / l);
    return;
  }
  const int few = min(a.weigh, cnt), per = a.weigh <= TREE_FEW ? 256 : TREE_SLOTS, step = gridDim.y - oparts;
  if ((long)(blockIdx.y - oparts) * per >= T) return;
  __shared__ double sM[TREE_MAX_NODES], sR[TREE_MAX_NODES];  // maximum and 1 / sum
  for (int i = tid; i < few; i += 256) {
    const long at = ((long)bh * a.n + i) * p.nsplit;
    double M = -INFINITY, l = 0.0;
#pragma unroll 4
    for (int s = 0; s < ns; ++s) M = fmax(M, ws.m[at + s]);
#pragma unroll 4
    for (int s = 0; s < ns; ++s) l += ws.l[at + s] * exp(ws.m[at + s] - (M == -INFINITY ? 0.0 : M));
    sM[i] = M;
    sR[i] = 1.0 / l;
  }
  __syncthreads();
  const auto add = [&](int t, double w) {
    double* to = a.weights + (long)bh * a.ctx + t;
    *to = t < L ? *to + w : w;
  };
  // a slot that a node does not see has score -inf; a node without a softmax
  // (a score NaN or infinite, its sum NaN, or none above -inf, its sum 0) is NaN
  // at the slots it sees, as its output is
  const auto weight = [&](int t, int i, double x) {
    if (x != -INFINITY || isfinite(sR[i])) return exp(x - sM[i]) * sR[i];
    const int j = t - L;
    const auto* seen = op_array<unsigned long long>(a.tab, own, a.seen) + ((long)b * a.n + i) * a.words;
    const bool see = j < 0 || ((seen[j >> 6] >> (j & 63)) & 1);
    return see ? (double)NAN : 0.0;
  };
  const double* xs = ws.x + (long)bh * p.T * a.weigh;
  for (int from = (blockIdx.y - oparts) * per; from < T; from += step * per) {
    if (a.weigh <= TREE_FEW) {
      const int t = from + tid;
      if (t >= T) return;
      double w = 0.0;
      for (int i = 0; i < few; ++i) w += weight(t, i, xs[(long)t * a.weigh + i]);
      add(t, w);
      continue;
    }
    double w[TREE_SLOTS / 16] = {};
    for (int i = tid & 15; i < few; i += 16) {
      double x[TREE_SLOTS / 16];
#pragma unroll
      for (int k = 0; k < TREE_SLOTS / 16; ++k) x[k] = xs[(long)min(from + 16 * k + (tid >> 4), T - 1) * a.weigh + i];
#pragma unroll
      for (int k = 0; k < TREE_SLOTS / 16; ++k) w[k] += weight(min(from + 16 * k + (tid >> 4), T - 1), i, x[k]);
    }
#pragma unroll
    for (int k = 0; k < TREE_SLOTS / 16; ++k) {
      const int t = from + 16 * k + (tid >> 4);
      const double all = row16_sum(w[k]);
      if (t < T && (tid & 15) == 0) add(t, all);
    }
  }
}

// Chunks of the least estimated time.  A block's tile takes 2.3 us of a SIMD at
// head dim 64 (64 MFMAs and the softmax), half as much again alone, or its
// bytes' time at 5.2 TB/s where every place of the chip is busy; 8 us go to a
// block's start and end, and the parts of a split pass through memory twice.
// Whole rounds run at the average length, the last at its longest.  Measured,
// us, head dim 64: 32 sequences of 144 to 512 slots and 16 nodes 69 in chunks of
// 64, 57 of 128, 47 of 256, 50 whole; 64 of 400 to 512 and one node 157 of 128,
// 146 of 256, 149 whole.  Other widths go by the same figures in proportion,
// which nothing was fitted to there.
TreePlan tree_plan(const TreeAttn& a, const int* kv_len, const int* count, std::vector<int>& lists) {
  TreePlan p;
  p.ng = a.n <= 16 || a.dh > 128 ? 1 : a.n <= 32 ? 2 : 4;
  const int groups = (a.n + 16 * p.ng - 1) / (16 * p.ng), unit = 64 / p.ng;  // slots that its waves take at a time
  const double places = a.dh <= 64 || (a.dh <= 128 && p.ng < 4) ? 512.0 : 256.0;  // blocks the chip holds at once
  std::vector<int> len(a.B);
  double all = 0.0;  // units of the call
  for (int b = 0; b < a.B; ++b) {
    len[b] = count[b] ? kv_len[b] + count[b] : 0;
    p.T = std::max(p.T, len[b]);
    all += (len[b] + unit - 1) / unit;
  }
  const double row = (double)a.H * groups, tile = 0.7 + 1.6 * a.dh / 64;
  const double unit_mb_us = unit * a.dh * 32 / 5.2e6 / groups;
  const int most = std::max(1, (p.T + unit - 1) / unit);
  int each = 1;  // units of a chunk
  if (all * row > places) {
    double least = 1e300;
    int last = 0;
    for (int k : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32}) {
      const int c = (most + k - 1) / k, slots = c * unit;
      if (c == last) continue;
      last = c;
      double blocks = 0.0;
      for (int b = 0; b < a.B; ++b) blocks += std::max(1, (len[b] + slots - 1) / slots);
      const bool split = blocks > a.B;
      blocks *= row;
      const double full = std::floor(blocks / places), rest = blocks - full * places;
      const double work = all * row / blocks;  // units of a block, on average
      double cost = full * (3.0 + work * std::max(2.0 * tile * places / 512.0, places * unit_mb_us));
      if (rest > 0.0) cost += 8.0 + std::max(c * tile * (rest > 256.0 ? 2.0 : 1.45), rest * work * unit_mb_us);
      if (split) cost += blocks * 16 * std::min(p.ng * 16, a.n) * a.dh * 2 / 5.2e6;
      if (cost < least) least = cost, each = c;
    }
  }
  std::vector<int> splits(a.B);
  std::vector<int4> list;
  for (int b = 0; b < a.B; ++b) {
    const int units = std::max(1, (len[b] + unit - 1) / unit), k = (units + each - 1) / each;
    const int slots = (units + k - 1) / k * unit;
    int s = 0;
    for (int t0 = 0; s == 0 || t0 < len[b]; t0 += slots) list.push_back(make_int4(b, t0, std::min(len[b], t0 + slots), s++));
    splits[b] = s;
    p.nsplit = std::max(p.nsplit, s);
  }
  std::stable_sort(list.begin(), list.end(), [](const int4& x, const int4& y) { return x.z - x.y > y.z - y.y; });
  lists.resize((lists.size() + 3) & ~(size_t)3);
  p.entries = (int)list.size();
  p.chunks = (uint32_t)(lists.size() * sizeof(int));
  for (const int4& e : list) lists.insert(lists.end(), {e.x, e.y, e.z, e.w});
  p.splits = (uint32_t)(lists.size() * sizeof(int));
  lists.insert(lists.end(), splits.begin(), splits.end());
  return p;
}

static size_t tree_layout(const TreeAttn& a, const TreePlan& p, char* base, TreeWs& ws) {
  const size_t rows = (size_t)a.B * a.H * a.n * p.nsplit;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  ws.m = (double*)take(rows * sizeof(double));
  ws.l = (double*)take(rows * sizeof(double));
  if (p.nsplit > 1) ws.o = (double2*)take(rows * a.dh * sizeof(double2));
  if (a.weigh > 0) ws.x = (double*)take((size_t)a.B * a.H * p.T * a.weigh * sizeof(double));
  return at;
}

size_t tree_ws_bytes(const TreeAttn& a, const TreePlan& p) {
  TreeWs ws;
  return tree_layout(a, p, nullptr, ws);
}

template <int DHP, bool FULL>
static void launch_split(hipStream_t st, const TreeAttn& a, const TreePlan& p, const TreeWs& ws, const OpTable& own) {
  const dim3 grid((unsigned)((long)p.entries * a.H), (a.n + 16 * p.ng - 1) / (16 * p.ng));
  const auto go = [&](auto kern) { MITOK_LAUNCH(kern, grid, dim3(256), 0, st, a, p, ws, own); };
  if constexpr (DHP <= 128) {
    if (p.ng == 4) return go(k_tree_shared<DHP, FULL>);
    if (p.ng == 2) return go(k_tree_split<DHP, 2, FULL>);
  }
  go(k_tree_split<DHP, 1, FULL>);
}

void tree_attention(hipStream_t st, const TreeAttn& a, const TreePlan& p, const OpTable& own) {
  TreeWs ws;
  tree_layout(a, p, (char*)a.ws, ws);
  const auto width = [&](auto padded, auto whole, int dhp) { a.dh == dhp ? whole(st, a, p, ws, own) : padded(st, a, p, ws, own); };
  if (a.dh <= 16) width(launch_split<16, false>, launch_split<16, true>, 16);
  else if (a.dh <= 32) width(launch_split<32, false>, launch_split<32, true>, 32);
  else if (a.dh <= 64) width(launch_split<64, false>, launch_split<64, true>, 64);
  else if (a.dh <= 128) width(launch_split<128, false>, launch_split<128, true>, 128);
  else width(launch_split<256, false>, launch_split<256, true>, 256);
  const int oparts = p.nsplit > 1 ? (a.n * a.dh + 255) / 256 : 0;
  const int per = a.weigh <= TREE_FEW ? 256 : TREE_SLOTS;
  const int wparts = a.weights && a.weigh > 0 ? std::min((p.T + per - 1) / per, TREE_PARTS) : 0;
  if (oparts + wparts)
    hipLaunchKernelGGL(k_tree_join, dim3((unsigned)(a.B * a.H), oparts + wparts), dim3(256), 0, st, a, p, ws, oparts, own);
}

}  // namespace mitok

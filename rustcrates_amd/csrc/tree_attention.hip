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
// D[i][j] of a 16x16 tile sits at lane j + 16 * (i % 4), element i / 4.
#include <algorithm>

#include "serving.hpp"

namespace mitok {

// chunk partials: max and sum of (row of the workspace, node), and the
// unnormalised output; scores of the weighed nodes [B][H][T][weigh]
struct TreeWs {
  double* m = nullptr;  // [B][H][n][nsplit]
  double* l = nullptr;
  double2* o = nullptr;  // [B][H][n][nsplit][dh] (nsplit > 1)
  double* x = nullptr;   // [B][H][T][weigh]
};
struct TreePlan {
  int ng = 1, nsplit = 1, ch = 64, T = 0;
  TreeWs ws;
};

template <int DHP, int NG, bool FULL>
__global__ __launch_bounds__(256, DHP <= 128 ? 2 : 1) void k_tree_split(TreeAttn a, TreePlan p) {
  constexpr int KG = 4 / NG;    // waves that share a node group's slots
  constexpr int U = DHP / 4;    // 16-byte key loads of a lane per tile, two MFMAs each
  constexpr int CT = DHP / 16;  // 16-column tiles of the values
  constexpr bool PRE = DHP <= 64;  // the next tile's rows wait in registers
  constexpr int OSTR = DHP + 1;    // LDS row of a node's output: nodes in different banks
  constexpr size_t Q_BYTES = (size_t)NG * U * 64 * sizeof(double2), O_BYTES = (size_t)NG * 16 * OSTR * sizeof(double2);
  __shared__ __align__(16) unsigned char lds[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
  __shared__ double sm[4][16], sl[4][16];
  double2* qs = (double2*)lds;  // [NG][U][64], then the merged outputs [NG * 16][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ng = wave % NG, kg = wave / NG;
  const int node = lane & 15, kq = lane >> 4;
  const int chunk = blockIdx.x % p.nsplit, bh = blockIdx.x / p.nsplit, b = bh / a.H, h = bh - b * a.H;
  const int n0 = blockIdx.y * 16 * NG, dh = a.dh;
  const int L = a.kv_len[b], cnt = a.count[b], T = cnt ? L + cnt : 0;
  const int t0 = chunk * p.ch, t1 = min(T, t0 + p.ch);
  if (n0 >= cnt || t0 >= T) {
    // unused nodes give zero; a chunk past the sequence leaves nothing to join
    if (chunk == 0)
      for (int x = tid; x < 16 * NG * dh; x += 256) {
        const int i = n0 + x / dh, e = x % dh;
        if (i < a.n && i >= cnt) a.out[((long)b * a.n + i) * a.ldo + (long)h * dh + e] = make_double2(0.0, 0.0);
      }
    return;
  }
  const double2* K = a.kc + (long)bh * a.ctx * dh;
  const double2* V = a.vc + (long)bh * a.ctx * dh;
  const double* bias = a.bias ? a.bias + (long)h * a.bias_stride : nullptr;
  const int i = n0 + 16 * ng + node;  // this lane's node

  for (int x = tid; x < NG * U * 64; x += 256) {
    const int ln = x & 63, u = (x >> 6) % U, g = x / (64 * U);
    const int r = n0 + 16 * g + (ln & 15), e = 4 * u + (ln >> 4);
    double2 q = make_double2(0.0, 0.0);
    if (r < cnt && e < dh) q = a.q[((long)b * a.n + r) * a.ldq + (long)h * dh + e];
    qs[x] = make_double2(q.x * a.scale, -q.y * a.scale);
  }
  __syncthreads();
  const double2* qw = qs + ng * U * 64 + lane;

  v4d o_re[CT], o_im[CT];
  double m = -INFINITY, l = 0.0;  // of this lane's node; l over this lane's slots alone
#pragma unroll
  for (int c = 0; c < CT; ++c) o_re[c] = o_im[c] = v4d{0.0, 0.0, 0.0, 0.0};

  // a tile's key row of this lane and its value rows 4 q + kq; a row past
  // `end` is row end - 1, with weight 0.  Padded columns: keys of 0 (0 times an
  // infinity would be NaN), and value columns that nobody reads.
  const auto key_at = [&](int t, int u, int end) {
    const uint32_t at = (uint32_t)min(node, end - 1 - t) * (uint32_t)dh + kq;
    if (!FULL && 4 * u + kq >= dh) return make_double2(0.0, 0.0);
    return ld_glb(K + (long)t * dh + at + 4 * u);
  };
  const auto value_at = [&](int t, int q, int c, int end) {
    const uint32_t at = (uint32_t)min(4 * q + kq, end - 1 - t) * (uint32_t)dh;
    if (FULL) return ld_glb(V + (long)t * dh + (at + node) + 16 * c);
    return ld_glb(V + (long)t * dh + (at + (uint32_t)min(node + 16 * c, dh - 1)));
  };
  const auto score = [&](v4d& s, int u, double2 k) {
    const double2 q = qw[u * 64];
    s = __builtin_amdgcn_mfma_f64_16x16x4f64(k.x, q.x, s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f64_16x16x4f64(k.y, q.y, s, 0, 0, 0);
  };
  const auto keep_scores = [&](const v4d& s, int t, int end) {
    if (i >= a.weigh) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t + 4 * e + kq < end) p.ws.x[((long)bh * p.T + t + 4 * e + kq) * a.weigh + i] = s[e];
  };
  // the running maximum and sum take a tile's scores, which become its weights
  const auto soften = [&](v4d& s) {
    double x, y;
    pair16_f64(fmax(fmax(s[0], s[1]), fmax(s[2], s[3])), x, y);
    pair32_f64(fmax(x, y), x, y);
    const double mn = fmax(m, fmax(x, y));
    const double base = mn == -INFINITY ? 0.0 : mn;  // nothing seen yet: every weight e^-inf = 0
    const double keep = exp(m - base);
    m = mn;
    double ls = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = exp(s[e] - base);
      ls += s[e];
    }
    l = l * keep + ls;
#pragma unroll
    for (int c = 0; c < CT; ++c) o_re[c] *= keep, o_im[c] *= keep;
  };
  const auto output = [&](const v4d& s, int q, int c, double2 v) {
    o_re[c] = __builtin_amdgcn_mfma_f64_16x16x4f64(v.x, s[q], o_re[c], 0, 0, 0);
    o_im[c] = __builtin_amdgcn_mfma_f64_16x16x4f64(v.y, s[q], o_im[c], 0, 0, 0);
  };

  // committed slots: every node sees them
  const int tc = min(t1, L);
  {
    double2 kf[PRE ? U : 1], vf[PRE ? 4 : 1][PRE ? CT : 1];
    double bf[4] = {0.0, 0.0, 0.0, 0.0};
    const auto load_keys = [&](int t) {
      if constexpr (PRE) {
#pragma unroll
        for (int u = 0; u < U; ++u) kf[u] = key_at(t, u, tc);
      }
      if (bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bf[e] = bias[min(t + 4 * e + kq, tc - 1)];
      }
    };
    const auto load_values = [&](int t) {
      if constexpr (PRE) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int c = 0; c < CT; ++c) vf[q][c] = value_at(t, q, c, tc);
      }
    };
    int t = t0 + 16 * kg;
    if (t < tc) {
      load_keys(t);
      load_values(t);
    }
    for (; t < tc; t += 16 * KG) {
      v4d s = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        score(s, u, PRE ? kf[PRE ? u : 0] : key_at(t, u, tc));
        if (u % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four queries at a time in registers
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = t + 4 * e + kq < tc ? s[e] + bf[e] : -INFINITY;
      keep_scores(s, t, tc);
      const bool more = t + 16 * KG < tc;
      if (more || !PRE) load_keys(t + (more ? 16 * KG : 0));
      soften(s);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int c = 0; c < CT; ++c) output(s, q, c, PRE ? vf[PRE ? q : 0][PRE ? c : 0] : value_at(t, q, c, tc));
        if (!PRE) __builtin_amdgcn_sched_barrier(0);
      }
      if (more) load_values(t + 16 * KG);
    }
  }

  // the nodes' own slots: a node sees its ancestors and itself
  for (int t = max(t0, L) + 16 * kg; t < t1; t += 16 * KG) {
    v4d s = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      score(s, u, key_at(t, u, t1));
      if (u % 8 == 7) __builtin_amdgcn_sched_barrier(0);
    }
    unsigned vis = 0;  // bit e: slot t + 4 e + kq is seen by this lane's node
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = t + 4 * e + kq - L;
      const bool see = j < t1 - L && i < cnt && ((a.seen[((long)b * a.n + i) * a.words + (j >> 6)] >> (j & 63)) & 1);
      if (see) vis |= 1u << e;
      if (see && bias) s[e] += bias[L + a.depth[(long)b * a.n + j]];
      if (!see) s[e] = -INFINITY;
    }
    keep_scores(s, t, t1);
    soften(s);
    // values that are not finite are left out of the products, where 0 times
    // them is NaN in the rows of the nodes that do not see them ...
    bool bad = false;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        double2 v = value_at(t, q, c, t1);
        const bool nx = !isfinite(v.x), ny = !isfinite(v.y);
        bad |= nx || ny;
        if (nx) v.x = 0.0;
        if (ny) v.y = 0.0;
        output(s, q, c, v);
        if (c % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    // ... and added to the others: output column 16 c + 4 e + kq, slot by slot
    if (__ballot(bad)) {
      for (int k = 0; k < 16 && t + k < t1; ++k) {
        const int from = node + 16 * (k & 3), q = k >> 2;
        const double pk = __shfl(q == 0 ? s[0] : q == 1 ? s[1] : q == 2 ? s[2] : s[3], from);
        const bool see = (__shfl((int)vis, from) >> q) & 1;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = 16 * c + 4 * e + kq;
            if (see && col < dh) {
              const double2 v = V[(long)(t + k) * dh + col];
              if (!isfinite(v.x)) o_re[c][e] += pk * v.x;
              if (!isfinite(v.y)) o_im[c][e] += pk * v.y;
            }
          }
      }
    }
  }

  // the waves of a node group, rescaled to their common maximum and added in order
  l = xor32_sum(xor16_sum(l));
  if (kq == 0) sm[wave][node] = m, sl[wave][node] = l;
  __syncthreads();  // and the queries' last read
  double M = -INFINITY;
#pragma unroll
  for (int g = 0; g < KG; ++g) M = fmax(M, sm[g * NG + ng][node]);
  const double base = M == -INFINITY ? 0.0 : M;
  double Ls = 0.0;
#pragma unroll
  for (int g = 0; g < KG; ++g) Ls += sl[g * NG + ng][node] * exp(sm[g * NG + ng][node] - base);
  const double f = exp(m - base);
#pragma unroll
  for (int g = 0; g < KG; ++g) {
    if (kg == g) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          double2* at = os + (16 * ng + node) * OSTR + 16 * c + 4 * e + kq;
          const double2 v = make_double2(o_re[c][e] * f, o_im[c][e] * f);
          *at = g ? cadd(*at, v) : v;
        }
    }
    __syncthreads();
  }
  if (kg == 0 && kq == 0) {
    sl[ng][node] = Ls;
    if (i < cnt && (p.nsplit > 1 || i < a.weigh)) {
      const long at = ((long)bh * a.n + i) * p.nsplit + chunk;
      p.ws.m[at] = M;
      p.ws.l[at] = Ls;
    }
  }
  __syncthreads();
  for (int x = tid; x < 16 * NG * dh; x += 256) {
    const int r = x / dh, e = x - r * dh, k = n0 + r;
    if (k >= a.n) break;
    const double2 v = os[r * OSTR + e];
    if (p.nsplit == 1) {
      const double w = sl[r >> 4][r & 15];
      a.out[((long)b * a.n + k) * a.ldo + (long)h * dh + e] = k < cnt ? make_double2(v.x / w, v.y / w) : make_double2(0.0, 0.0);
    } else if (k < cnt) {
      p.ws.o[(((long)bh * a.n + k) * p.nsplit + chunk) * dh + e] = v;
    } else if (chunk == 0) {
      a.out[((long)b * a.n + k) * a.ldo + (long)h * dh + e] = make_double2(0.0, 0.0);
    }
  }
}

// Joins the chunks: blocks y < oparts the outputs, the others the weights of
// 256 / 16 slots each (or 256 where few nodes are weighed).
constexpr int TREE_FEW = 4;
__global__ __launch_bounds__(256) void k_tree_join(TreeAttn a, TreePlan p, int oparts) {
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, tid = threadIdx.x;
  const int L = a.kv_len[b], cnt = a.count[b], T = cnt ? L + cnt : 0;
  const int ns = (T + p.ch - 1) / p.ch;
  if ((int)blockIdx.y < oparts) {
    const int x = blockIdx.y * 256 + tid, i = x / a.dh, e = x - i * a.dh;
    if (i >= cnt) return;
    const long at = ((long)bh * a.n + i) * p.nsplit;
    double M = -INFINITY;
    for (int s = 0; s < ns; ++s) M = fmax(M, p.ws.m[at + s]);
    const double base = M == -INFINITY ? 0.0 : M;
    double l = 0.0;
    double2 v = make_double2(0.0, 0.0);
    for (int s = 0; s < ns; ++s) {
      const double f = exp(p.ws.m[at + s] - base);
      const double2 o = p.ws.o[(at + s) * a.dh + e];
      l += p.ws.l[at + s] * f;
      v = make_double2(v.x + o.x * f, v.y + o.y * f);
    }
    a.out[((long)b * a.n + i) * a.ldo + (long)h * a.dh + e] = make_double2(v.x / l, v.y / l);
    return;
  }
  const int few = min(a.weigh, cnt);
  __shared__ double sM[TREE_MAX_NODES], sL[TREE_MAX_NODES];
  for (int i = tid; i < few; i += 256) {
    const long at = ((long)bh * a.n + i) * p.nsplit;
    double M = -INFINITY, l = 0.0;
    for (int s = 0; s < ns; ++s) M = fmax(M, p.ws.m[at + s]);
    for (int s = 0; s < ns; ++s) l += p.ws.l[at + s] * exp(p.ws.m[at + s] - (M == -INFINITY ? 0.0 : M));
    sM[i] = M;
    sL[i] = l;
  }
  __syncthreads();
  const int part = blockIdx.y - oparts;
  const auto add = [&](int t, double w) {
    double* to = a.weights + (long)bh * a.ctx + t;
    *to = t < L ? *to + w : w;
  };
  // a slot that a node does not see has score -inf; a node without any weight
  // (maximum -inf) is NaN at the slots it sees, as its output is
  const auto weight = [&](int t, int i) {
    const double x = p.ws.x[((long)bh * p.T + t) * a.weigh + i];
    if (x != -INFINITY || sM[i] != -INFINITY) return exp(x - sM[i]) / sL[i];
    const int j = t - L;
    const bool see = j < 0 || ((a.seen[((long)b * a.n + i) * a.words + (j >> 6)] >> (j & 63)) & 1);
    return see ? (double)NAN : 0.0;
  };
  if (a.weigh <= TREE_FEW) {
    const int t = part * 256 + tid;
    if (t >= T) return;
    double w = 0.0;
    for (int i = 0; i < few; ++i) w += weight(t, i);
    add(t, w);
  } else {
    const int t = part * 16 + (tid >> 4);
    double w = 0.0;
    if (t < T)
      for (int i = tid & 15; i < few; i += 16) w += weight(t, i);
    w = row16_sum(w);
    if (t < T && (tid & 15) == 0) add(t, w);
  }
}

// Node groups per block: as many as there are nodes for, where LDS holds their
// queries.  Chunks: as many as fill the chip twice over, of at least one tile
// per wave.
static TreePlan tree_plan(const TreeAttn& a) {
  TreePlan p;
  const int most = a.dh <= 64 ? 4 : a.dh <= 128 ? 2 : 1;
  p.ng = a.n <= 16 ? 1 : std::min(most, a.n <= 32 ? 2 : 4);
  p.T = a.T_max;
  const long blocks = (long)a.B * a.H * ((a.n + 16 * p.ng - 1) / (16 * p.ng));
  const int tiles = std::max(1, (p.T + 63) / 64);
  p.nsplit = (int)std::max<long>(1, std::min<long>(std::min(tiles, 64), (1024 + blocks - 1) / blocks));
  p.ch = (tiles + p.nsplit - 1) / p.nsplit * 64;
  p.nsplit = std::max(1, (p.T + p.ch - 1) / p.ch);
  return p;
}

static size_t tree_layout(const TreeAttn& a, TreePlan& p, char* base) {
  const size_t rows = (size_t)a.B * a.H * a.n * p.nsplit;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  p.ws.m = (double*)take(rows * sizeof(double));
  p.ws.l = (double*)take(rows * sizeof(double));
  if (p.nsplit > 1) p.ws.o = (double2*)take(rows * a.dh * sizeof(double2));
  if (a.weigh > 0) p.ws.x = (double*)take((size_t)a.B * a.H * p.T * a.weigh * sizeof(double));
  return at;
}

size_t tree_ws_bytes(const TreeAttn& a) {
  TreePlan p = tree_plan(a);
  return tree_layout(a, p, nullptr);
}

template <int DHP, bool FULL>
static void launch_split_of(hipStream_t st, const TreeAttn& a, const TreePlan& p) {
  const dim3 grid((unsigned)((long)a.B * a.H * p.nsplit), (a.n + 16 * p.ng - 1) / (16 * p.ng));
  const auto go = [&](auto kern) { MITOK_LAUNCH(kern, grid, dim3(256), 0, st, a, p); };
  if constexpr (DHP <= 64)
    if (p.ng == 4) return go(k_tree_split<DHP, 4, FULL>);
  if constexpr (DHP <= 128)
    if (p.ng == 2) return go(k_tree_split<DHP, 2, FULL>);
  go(k_tree_split<DHP, 1, FULL>);
}

template <int DHP>
static void launch_split(hipStream_t st, const TreeAttn& a, const TreePlan& p) {
  if (a.dh == DHP) launch_split_of<DHP, true>(st, a, p);
  else launch_split_of<DHP, false>(st, a, p);
}

void tree_attention(hipStream_t st, const TreeAttn& a) {
  TreePlan p = tree_plan(a);
  tree_layout(a, p, (char*)a.ws);
  if (a.dh <= 16) launch_split<16>(st, a, p);
  else if (a.dh <= 32) launch_split<32>(st, a, p);
  else if (a.dh <= 64) launch_split<64>(st, a, p);
  else if (a.dh <= 128) launch_split<128>(st, a, p);
  else launch_split<256>(st, a, p);
  const int oparts = p.nsplit > 1 ? (a.n * a.dh + 255) / 256 : 0;
  const int per = a.weigh <= TREE_FEW ? 256 : 16;
  const int wparts = a.weights && a.weigh > 0 ? (p.T + per - 1) / per : 0;
  if (oparts + wparts)
    hipLaunchKernelGGL(k_tree_join, dim3((unsigned)(a.B * a.H), oparts + wparts), dim3(256), 0, st, a, p, oparts);
}

}  // namespace mitok

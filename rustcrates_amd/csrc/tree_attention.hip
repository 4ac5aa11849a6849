// tree_attention.hip — attention of a tree of drafted tokens over the KV cache.
//
// Each node of a sequence's tree attends over the committed rows and over its
// own ancestors among the drafted ones, whose rows lie behind the committed
// ones in the cache (TreeAttn in serving.hpp has the formula).  A node at depth
// g stands where an ordinary decode step would put the g-th next token, so its
// bias column is kv_len + g and a chain of nodes gives what decode steps give.
// A row that a node does not see never enters its sums, finite or not.
#include "serving.hpp"

namespace mitok {

// One block per (node, head, sequence): each wave walks every fourth visible
// slot with a running maximum and sum, lane e holding columns e, e + 64, ...
__global__ __launch_bounds__(256) void k_tree_rows(TreeAttn a, double* __restrict__ ml) {
  constexpr int EC = TREE_MAX_DH / 64;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dh = a.dh;
  double2* out = a.out + ((long)b * a.n + i) * a.ldo + (long)h * dh;
  if (i >= a.count[b]) {
    for (int e = threadIdx.x; e < dh; e += 256) out[e] = make_double2(0.0, 0.0);
    return;
  }
  const long lane_bh = (long)b * a.H + h;
  const double2* K = a.kc + lane_bh * a.ctx * dh;
  const double2* V = a.vc + lane_bh * a.ctx * dh;
  const double2* q = a.q + ((long)b * a.n + i) * a.ldq + (long)h * dh;
  const unsigned long long* seen = a.seen + ((long)b * a.n + i) * a.words;
  const int L = a.kv_len[b], T = L + i + 1;  // ancestors come before their nodes
  double2 qv[EC], o[EC];
#pragma unroll
  for (int c = 0; c < EC; ++c) {
    const int e = lane + 64 * c;
    qv[c] = e < dh ? q[e] : make_double2(0.0, 0.0);
    o[c] = make_double2(0.0, 0.0);
  }
  double m = -INFINITY, l = 0.0;
  for (int t = wave; t < T; t += 4) {
    const int j = t - L;
    if (j >= 0 && !((seen[j >> 6] >> (j & 63)) & 1)) continue;
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < EC; ++c) {
      const int e = lane + 64 * c;
      if (e < dh) {
        const double2 k = K[(long)t * dh + e];
        s += qv[c].x * k.x - qv[c].y * k.y;
      }
    }
    s = wave_sum(s) * a.scale;
    if (a.bias) s += a.bias[(long)h * a.bias_stride + (j < 0 ? t : L + a.depth[(long)b * a.n + j])];
    const double mn = s > m || isnan(s) ? s : m;
    const double keep = m == -INFINITY ? 0.0 : exp(m - mn), p = mn == -INFINITY ? 0.0 : exp(s - mn);
    m = mn;
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < EC; ++c) {
      const int e = lane + 64 * c;
      if (e < dh) {
        const double2 v = V[(long)t * dh + e];
        o[c].x = o[c].x * keep + p * v.x;
        o[c].y = o[c].y * keep + p * v.y;
      }
    }
  }
  __shared__ double sm[4], sl[4];
  __shared__ double2 so[4][TREE_MAX_DH];
  if (lane == 0) sm[wave] = m, sl[wave] = l;
#pragma unroll
  for (int c = 0; c < EC; ++c) so[wave][lane + 64 * c] = o[c];
  __syncthreads();
  double M = sm[0];
  for (int w = 1; w < 4; ++w) M = sm[w] > M || isnan(sm[w]) ? sm[w] : M;
  double f[4], sum = 0.0;
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.0 : exp(sm[w] - M);
    sum += sl[w] * f[w];
  }
  for (int e = threadIdx.x; e < dh; e += 256) {
    double2 v = make_double2(0.0, 0.0);
    for (int w = 0; w < 4; ++w)
      if (f[w] != 0.0) v = make_double2(v.x + so[w][e].x * f[w], v.y + so[w][e].y * f[w]);
    out[e] = make_double2(v.x / sum, v.y / sum);
  }
  if (threadIdx.x == 0) {
    double* at = ml + (lane_bh * a.n + i) * 2;
    at[0] = M;
    at[1] = sum;
  }
}

// The first `weigh` nodes' softmax weights, one wave per slot, in node order.
__global__ __launch_bounds__(256) void k_tree_weights(TreeAttn a, const double* __restrict__ ml) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, dh = a.dh;
  const int L = a.kv_len[b], n = a.count[b];
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= L + n) return;
  const long lane_bh = (long)b * a.H + h;
  const double2* k = a.kc + (lane_bh * a.ctx + t) * dh;
  const int j = t - L;
  double w = 0.0;
  for (int i = 0; i < min(a.weigh, n); ++i) {
    if (j >= 0 && !((a.seen[((long)b * a.n + i) * a.words + (j >> 6)] >> (j & 63)) & 1)) continue;
    const double2* q = a.q + ((long)b * a.n + i) * a.ldq + (long)h * dh;
    double s = 0.0;
    for (int e = lane; e < dh; e += 64) s += q[e].x * k[e].x - q[e].y * k[e].y;
    s = wave_sum(s) * a.scale;
    if (a.bias) s += a.bias[(long)h * a.bias_stride + (j < 0 ? t : L + a.depth[(long)b * a.n + j])];
    const double* at = ml + (lane_bh * a.n + i) * 2;
    w += exp(s - at[0]) / at[1];
  }
  if (lane == 0) {
    double* to = a.weights + lane_bh * a.ctx + t;
    *to = j < 0 ? *to + w : w;
  }
}

size_t tree_ws_bytes(const TreeAttn& a) { return (size_t)a.B * a.H * a.n * 2 * sizeof(double); }

void tree_attention(hipStream_t st, const TreeAttn& a) {
  double* ml = (double*)a.ws;
  MITOK_LAUNCH(k_tree_rows, dim3(a.n, a.H, a.B), dim3(256), 0, st, a, ml);
  if (a.weights && a.weigh > 0 && a.T_max > 0)
    hipLaunchKernelGGL(k_tree_weights, dim3((a.T_max + 3) / 4, a.H, a.B), dim3(256), 0, st, a, ml);
}

}  // namespace mitok

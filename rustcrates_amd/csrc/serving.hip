// serving.hip — the other operators of a serving loop: rows evicted from the KV
// cache by the attention they received, and the rules that turn logits into a
// token (penalties for repeated tokens, biases, a mask of allowed tokens).
#include "serving.hpp"

namespace mitok {

// ===========================================================================
// eviction
// ===========================================================================
// a double as an integer of the same order; NaN is the least, -0 equals +0
__device__ __forceinline__ unsigned long long order_key(double w) {
  if (isnan(w)) return 0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(w + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// One block per (head, sequence).  A slot between the sinks and the recent rows
// stays if fewer than keep - sinks - recent others come before it (larger
// weight, or equal and a lower slot); a scan gives the kept slots their places.
__global__ __launch_bounds__(1024) void k_evict_select(EvictSelect e) {
  __shared__ int total[16], carry;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int L = e.kv_len[b];
  const double* w = e.w + ((long)b * e.H + h) * e.ctx;
  uint32_t* kept = e.kept + ((long)b * e.H + h) * e.keep;
  const int lo = e.sinks, hi = L - e.recent, most = e.keep - e.sinks - e.recent;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int t0 = 0; t0 < L; t0 += 1024) {
    const int t = t0 + tid;
    bool stay = t < L;
    if (stay && L > e.keep && t >= lo && t < hi) {
      const unsigned long long mine = order_key(w[t]);
      int before = 0;
      for (int s = lo; s < hi; ++s) {
        const unsigned long long k = order_key(w[s]);
        before += k > mine || (k == mine && s < t) ? 1 : 0;
      }
      stay = before < most;
    }
    const unsigned long long vote = __ballot(stay);
    if (lane == 0) total[wave] = __popcll(vote);
    __syncthreads();
    int at = carry + __popcll(vote & ((1ull << lane) - 1));
    for (int x = 0; x < wave; ++x) at += total[x];
    if (stay) kept[at] = (uint32_t)t;
    __syncthreads();
    if (tid == 0)
      for (int x = 0; x < 16; ++x) carry += total[x];
    __syncthreads();
  }
  for (int r = min(L, e.keep) + tid; r < e.keep; r += 1024) kept[r] = NO_ROW;
}

void evict_select(hipStream_t st, const EvictSelect& e) {
  hipLaunchKernelGGL(k_evict_select, dim3(e.H, e.B), dim3(1024), 0, st, e);
}

// One block per (head, sequence), 64 rows at a time: read, then written.  Kept
// slots ascend, so a row moves to a place at or before its own and no write
// reaches a row that a later step reads: in place is as good as to another cache.
__global__ __launch_bounds__(256) void k_cache_move(CacheMove m) {
  const int h = blockIdx.x, b = blockIdx.y, dh = m.dh;
  const long bh = (long)b * m.H + h;
  const uint32_t* idx = m.idx + b * m.idx_b + h * m.idx_h;
  const int base = m.base ? m.base[b] : 0, rows = m.rows[b];
  const double2* src[2] = {m.k + (bh * m.ctx + base) * dh, m.v + (bh * m.ctx + base) * dh};
  double2* dst[2] = {m.ko + (bh * m.ctx_out + base) * dh, m.vo + (bh * m.ctx_out + base) * dh};
  for (int r = 0; r < rows; ++r) {
    const long s = idx[r];
    double2 x[2];
    double w = 0.0;
    const int e = threadIdx.x;
    if (e < dh)
      for (int p = 0; p < 2; ++p) x[p] = src[p][s * dh + e];
    if (e == 0 && m.w) w = m.w[bh * m.ctx + base + s];
    __syncthreads();
    if (e < dh)
      for (int p = 0; p < 2; ++p) dst[p][(long)r * dh + e] = x[p];
    if (e == 0 && m.w) m.wo[bh * m.ctx_out + base + r] = w;
    __syncthreads();
  }
}

void cache_move(hipStream_t st, const CacheMove& m) {
  if (m.rows_max <= 0) return;
  hipLaunchKernelGGL(k_cache_move, dim3(m.H, m.B), dim3(256), 0, st, m);
}

__global__ void k_zero_weights(double* w, int H, long ctx, const int* from, const int* to) {
  const int h = blockIdx.y, b = blockIdx.z;
  const long t = from[b] + (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (t < to[b]) w[((long)b * H + h) * ctx + t] = 0.0;
}

void zero_weights(hipStream_t st, double* w, int B, int H, long ctx, const int* from, const int* to, int most) {
  if (most <= 0) return;
  hipLaunchKernelGGL(k_zero_weights, dim3((most + 255) / 256, H, B), dim3(256), 0, st, w, H, ctx, from, to);
}

__global__ void k_pick_ids(const uint32_t* ids, int n, const int* last, int B, uint32_t* dec_ids) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < B && last[b] >= 0) dec_ids[b] = ids[(long)b * n + last[b]];
}

void pick_ids(hipStream_t st, const uint32_t* ids, int n, const int* last, int B, uint32_t* dec_ids) {
  hipLaunchKernelGGL(k_pick_ids, dim3((B + 255) / 256), dim3(256), 0, st, ids, n, last, B, dec_ids);
}

// ===========================================================================
// logits to a token
// ===========================================================================
__device__ __forceinline__ void set_err(uint32_t* err, int word) {
  __hip_atomic_store(err + word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

constexpr int LR_CHUNK = 4096;
int logit_chunks(int V) { return (V + LR_CHUNK - 1) / LR_CHUNK; }

// One block per row, a chunk of the vocabulary at a time: the chunk's
// occurrences in the history and its last bias entry are gathered in LDS
// (integer atomics, so their order does not show), then its logits are read,
// changed, written and compared.
__global__ __launch_bounds__(256) void k_logit_rules(LogitRules r) {
  __shared__ uint32_t count[LR_CHUNK], entry[LR_CHUNK];
  __shared__ double sv[4];
  __shared__ int si[4];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = r.V;
  if (r.row_mask && !r.row_mask[row]) {
    if (tid == 0 && r.ids) r.ids[row] = NO_TOKEN;
    return;
  }
  const double* x = r.x + (long)row * V;
  double theta = 1.0, presence = 0.0, frequency = 0.0;
  if (r.penalties) {
    theta = r.penalties[3 * (long)row];
    presence = r.penalties[3 * (long)row + 1];
    frequency = r.penalties[3 * (long)row + 2];
    if (tid == 0 && !(theta > 0.0 && isfinite(theta) && isfinite(presence) && isfinite(frequency)))
      set_err(r.err, OE_BAD_PENALTY);
  }
  const int hist = r.penalties ? r.hist : 0;
  double bv = -INFINITY;
  int bi = -1;
  for (int c0 = 0; c0 < V; c0 += LR_CHUNK) {
    const int len = min(LR_CHUNK, V - c0);
    for (int i = tid; i < len; i += 256) count[i] = entry[i] = 0;
    __syncthreads();
    for (int i = tid; i < hist; i += 256) {
      const uint32_t t = r.history[(long)row * r.hist + i];
      if (t != NO_TOKEN && t >= (uint32_t)V) set_err(r.err, OE_BAD_TOKEN);
      if (t - (uint32_t)c0 < (uint32_t)len) atomicAdd(&count[t - c0], 1u);
    }
    for (int i = tid; i < r.nb; i += 256) {
      const uint32_t t = r.bias_ids[(long)row * r.nb + i];
      if (t != NO_TOKEN && t >= (uint32_t)V) set_err(r.err, OE_BAD_TOKEN);
      if (t - (uint32_t)c0 < (uint32_t)len) atomicMax(&entry[t - c0], (uint32_t)i + 1);
    }
    __syncthreads();
    for (int i = tid; i < len; i += 256) {
      const int t = c0 + i;
      double y = x[t];
      const uint32_t c = count[i], en = entry[i];
      if (c) {
        y = y > 0.0 ? y / theta : y * theta;
        y -= frequency * (double)c + presence;
      }
      if (en) y += r.bias[(long)row * r.nb + en - 1];
      const bool ok = !r.allowed || (r.allowed[(long)row * ((V + 31) / 32) + (t >> 5)] >> (t & 31)) & 1;
      if (!ok) y = -INFINITY;
      if (r.out) r.out[(long)row * V + t] = y;
      if (ok) {
        if (isnan(y)) set_err(r.err, OE_NAN);
        argmax_combine(bv, bi, y, t);
      }
    }
    __syncthreads();
  }
  wave_argmax(bv, bi);
  if (lane == 0) sv[wave] = bv, si[wave] = bi;
  __syncthreads();
  if (tid == 0 && r.ids) {
    for (int w = 1; w < 4; ++w) argmax_combine(bv, bi, sv[w], si[w]);
    r.ids[row] = bv > -INFINITY ? (uint32_t)bi : NO_TOKEN;  // nothing allowed is above -inf
  }
}

void logit_rules(hipStream_t st, const LogitRules& r) {
  hipLaunchKernelGGL(k_logit_rules, dim3(r.rows), dim3(256), 0, st, r);
}

}  // namespace mitok

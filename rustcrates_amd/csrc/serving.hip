// serving.hip — the other operators of a serving loop: rows evicted from the KV
// cache by the attention they received, and the rules that turn logits into a
// token (penalties for repeated tokens, biases, a mask of allowed tokens).
#include <algorithm>

#include "serving.hpp"

namespace mitok {

// ===========================================================================
// eviction
// ===========================================================================
// a double as an integer of the same order, at least 2; NaN is 1, -0 equals +0
__device__ __forceinline__ unsigned long long order_key(double w) {
  if (isnan(w)) return 1ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(w + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// One block per (head, sequence).  The least key that stays is sought between
// the smallest and the largest: each round counts the keys at or above three
// values that quarter the range (a compare and a ballot per key, held in
// registers), and the search ends once as many as have to stay lie above one:
// about 10 rounds for weights that differ, 33 at most.  Of equal least keys the lowest slots
// stay; scans over the slots give ranks and places.  NK: slots per thread, 0:
// any number, read again each round.  Bound by the rounds' latency, a barrier
// each, not by the 8 bytes of a slot: 48 heads of 2048 slots 11.5 us, 256 of
// up to 512 7.5, 4 of 320 5.3.  Sorting would order what only has to be
// divided; quartering the range instead of halving it saves half the barriers.
// Blocks of 8 waves take 6.2 us for the 320, of 16 waves 18.6 for the 2048.
template <int NK>
__global__ __launch_bounds__(256) void k_evict_select(EvictSelect e, OpTable own) {
  __shared__ unsigned long long ext[2][4];
  __shared__ int4 part[2][4];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int L = op_int(e.tab, own, e.kv_len, b);
  const double* w = e.w + ((long)b * e.H + h) * e.ctx;
  uint32_t* kept = e.kept + ((long)b * e.H + h) * e.keep;
  for (int r = min(L, e.keep) + tid; r < e.keep; r += 256) kept[r] = NO_ROW;
  if (L <= e.keep) {
    for (int t = tid; t < L; t += 256) kept[t] = (uint32_t)t;
    return;
  }
  const int lo = e.sinks, hi = L - e.recent, most = e.keep - e.sinks - e.recent;
  const int nk = NK ? NK : (L + 255) / 256;
  unsigned long long held[NK ? NK : 1];
  // slots between the sinks and the recent rows; the others never count (0)
  const auto load = [&](int k) {
    const int t = 256 * k + tid;
    return t >= lo && t < hi ? order_key(w[t]) : 0ull;
  };
  const auto key = [&](int k) { return NK ? held[NK ? k : 0] : load(k); };
  if constexpr (NK > 0) {
#pragma unroll
    for (int k = 0; k < NK; ++k) held[k] = load(k);
  }
  int round = 0;
  // keys at or above each of three values, in the whole block
  const auto count = [&](const unsigned long long (&least)[3], int (&c)[3]) {
    c[0] = c[1] = c[2] = 0;
#pragma unroll NK ? NK : 1
    for (int k = 0; k < nk; ++k)
#pragma unroll
      for (int j = 0; j < 3; ++j) c[j] += __popcll(__ballot(key(k) >= least[j]));
    if (lane == 0) part[round & 1][wave] = make_int4(c[0], c[1], c[2], 0);
    __syncthreads();
    c[0] = c[1] = c[2] = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int4 q = part[round & 1][v];
      c[0] += q.x, c[1] += q.y, c[2] += q.z;
    }
    ++round;
  };
  // count(>= low) >= most > count(>= high)
  unsigned long long low = ~0ull, high = 0;
#pragma unroll NK ? NK : 1
  for (int k = 0; k < nk; ++k) {
    const unsigned long long x = key(k);
    if (x) low = min(low, x);
    high = max(high, x);
  }
  for (int d = 32; d; d >>= 1) {
    low = min(low, (unsigned long long)__shfl_xor((long long)low, d));
    high = max(high, (unsigned long long)__shfl_xor((long long)high, d));
  }
  if (lane == 0) ext[0][wave] = low, ext[1][wave] = high;
  __syncthreads();
  low = min(min(ext[0][0], ext[0][1]), min(ext[0][2], ext[0][3]));
  high = max(max(ext[1][0], ext[1][1]), max(ext[1][2], ext[1][3])) + 1;  // a key is below 2^64 - 1
  int equal = 0;  // of the keys == low, how many stay
  if (most == 0) {
    low = ~0ull;
  } else {
    bool found = false;
    while (!found && high - low > 1) {
      const unsigned long long q = (high - low) / 4;
      const unsigned long long at[3] = {low + q, low + 2 * q, low + 3 * q + (high - low) % 4 / 2};
      int c[3];
      count(at, c);
      unsigned long long next = low;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (c[j] >= most) next = at[j];
        else high = min(high, at[j]);
        if (c[j] == most) found = true;  // and low is the largest such, so none below it stays
      }
      low = next;
    }
    equal = L;
    if (!found) {
      const unsigned long long above[3] = {low + 1, low + 1, low + 1};
      int c[3];
      count(above, c);
      equal = most - c[0];
    }
  }
  const unsigned long long below = (1ull << lane) - 1;
  // a running number over the slots, whose 256 of step k vote `v`: what comes
  // before this lane's, given the waves' votes of the step, and the total so far
  const auto before = [&](const int4& votes, unsigned long long v, int& so_far) {
    const int w[4] = {votes.x, votes.y, votes.z, votes.w};
    int at = so_far + __popcll(v & below);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x < wave) at += w[x];
      so_far += w[x];
    }
    return at;
  };
  const auto certain = [&](int k) {  // stays whatever the ties
    const int t = 256 * k + tid;
    return t < L && (t < lo || t >= hi || key(k) > low);
  };
  int ties = 0, all = 0;
  if constexpr (NK > 0) {
    __shared__ int4 eq[NK], st[NK];
    unsigned stays = 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int n = __popcll(__ballot(held[k] == low));
      if (lane == 0) ((int*)&eq[k])[wave] = n;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const bool tied = held[k] == low;
      const int rank = before(eq[k], __ballot(tied), ties);
      if (certain(k) || (tied && rank < equal)) stays |= 1u << k;
      const int n = __popcll(__ballot(stays >> k & 1));
      if (lane == 0) ((int*)&st[k])[wave] = n;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int at = before(st[k], __ballot(stays >> k & 1), all);
      if (stays >> k & 1) kept[at] = (uint32_t)(256 * k + tid);
    }
  } else {
    __shared__ int4 eq, st;
    for (int k = 0; k < nk; ++k) {
      const bool tied = key(k) == low;
      const unsigned long long v = __ballot(tied);
      if (lane == 0) ((int*)&eq)[wave] = __popcll(v);
      __syncthreads();
      const int rank = before(eq, v, ties);
      const bool stay = certain(k) || (tied && rank < equal);
      const unsigned long long w2 = __ballot(stay);
      if (lane == 0) ((int*)&st)[wave] = __popcll(w2);
      __syncthreads();
      const int at = before(st, w2, all);
      if (stay) kept[at] = (uint32_t)(256 * k + tid);
    }
  }
}

// keys in registers up to the widest context of a layer (6144); the smallest
// variant that holds the call's slots
void evict_select(hipStream_t st, const EvictSelect& e, const OpTable& own) {
  const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(e.H, e.B), dim3(256), 0, st, e, own); };
  if (e.T_max <= 512) go(k_evict_select<2>);
  else if (e.T_max <= 2048) go(k_evict_select<8>);
  else if (e.T_max <= 6144) go(k_evict_select<24>);
  else go(k_evict_select<0>);
}

constexpr int MV_PER = 8;  // 16-byte elements of a thread in flight
__device__ __forceinline__ void st_stream(double2* p, double2 v) {
  v2d x = {v.x, v.y};
  __builtin_nontemporal_store(x, (MITOK_GLOBAL v2d*)p);
}

// To another cache: 256 * MV_PER elements of one (head, sequence)'s keys (y 0)
// or values (y 1) per block, each read once and written once.  Bound by HBM:
// 32 sequences of 8 heads, 256 rows of 64 kept, 270 MB in 49.5 us (5.4 TB/s);
// 48 heads, 1024 rows, 201 MB in 37.8 us (5.3 TB/s).  A row's 1 KB is one
// wave's load, so rows picked here and there cost no bandwidth.
__global__ __launch_bounds__(256) void k_cache_copy(CacheMove m, int parts, OpTable own) {
  const int bh = blockIdx.x / parts, part = blockIdx.x % parts, b = bh / m.H, h = bh - b * m.H, dh = m.dh;
  const int base = m.based ? op_int(m.tab, own, m.base, b) : 0, rows = op_int(m.tab, own, m.rows, b);
  const uint32_t* idx = m.idx + b * m.idx_b + h * m.idx_h;
  if (blockIdx.y == 2) {
    for (int r = part * 256 + threadIdx.x; r < rows; r += parts * 256)
      m.wo[(long)bh * m.ctx_out + base + r] = m.w[(long)bh * m.ctx + base + idx[r]];
    return;
  }
  const double2* src = (blockIdx.y ? m.v : m.k) + ((long)bh * m.ctx + base) * dh;
  double2* dst = (blockIdx.y ? m.vo : m.ko) + ((long)bh * m.ctx_out + base) * dh;
  const long all = (long)rows * dh;
  const long x0 = (long)part * (256 * MV_PER) + threadIdx.x;
  if (x0 >= all) return;
  int r = (int)(x0 / dh), e = (int)(x0 - (long)r * dh);
  const int dr = 256 / dh, de = 256 - dr * dh;
  double2 v[MV_PER];
#pragma unroll
  for (int k = 0; k < MV_PER; ++k) {
    if (r < rows) v[k] = ld_stream(src + (long)idx[r] * dh + e);
    r += dr;
    e += de;
    if (e >= dh) e -= dh, ++r;
  }
#pragma unroll
  for (int k = 0; k < MV_PER; ++k)
    if (x0 + 256 * k < all) st_stream(dst + x0 + 256 * k, v[k]);
}

// In place: a block moves one 8-wide slice of the columns (a cache line) of one
// (head, sequence)'s keys or values, 32 * MV_PER rows at a time: all read, then
// all written.  The slots ascend, so a row moves to a place at or before its
// own, and no write reaches a row that a later step reads.  The sizes above in
// place: 49.6 and 36.4 us, the same 5.4 TB/s.  Only columns can be shared out
// among blocks without a wait between them: a block of rows would overwrite
// what another has still to read.
__global__ __launch_bounds__(256) void k_cache_pack(CacheMove m, int slices, OpTable own) {
  const int bh = blockIdx.x / slices, sl = blockIdx.x % slices, b = bh / m.H, h = bh - b * m.H, dh = m.dh;
  const int base = m.based ? op_int(m.tab, own, m.base, b) : 0, rows = op_int(m.tab, own, m.rows, b);
  const uint32_t* idx = m.idx + b * m.idx_b + h * m.idx_h;
  if (blockIdx.y == 2) {
    if (sl) return;
    double* w = m.wo + (long)bh * m.ctx + base;
    for (int r0 = 0; r0 < rows; r0 += 256) {
      const int r = r0 + threadIdx.x;
      const double x = r < rows ? w[idx[r]] : 0.0;
      __syncthreads();
      if (r < rows) w[r] = x;
      __syncthreads();
    }
    return;
  }
  MITOK_GLOBAL v2d* at = (MITOK_GLOBAL v2d*)((blockIdx.y ? m.vo : m.ko) + ((long)bh * m.ctx + base) * dh);
  const int e = sl * 8 + (threadIdx.x & 7), q = threadIdx.x >> 3;
  const bool in = e < dh;
  for (int r0 = 0; r0 < rows; r0 += 32 * MV_PER) {
    v2d v[MV_PER];
    unsigned move = 0;
#pragma unroll
    for (int k = 0; k < MV_PER; ++k) {
      const int r = r0 + 32 * k + q;
      const int from = r < rows ? (int)idx[r] : r;
      v[k] = v2d{0.0, 0.0};
      if (in && from != r) {
        move |= 1u << k;
        v[k] = at[(long)from * dh + e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MV_PER; ++k)
      if (move >> k & 1) at[(long)(r0 + 32 * k + q) * dh + e] = v[k];
    __syncthreads();
  }
}

void cache_move(hipStream_t st, const CacheMove& m, const OpTable& own) {
  if (m.rows_max <= 0) return;
  const unsigned y = m.w ? 3 : 2;
  if (m.ko == m.k) {
    const int slices = (m.dh + 7) / 8;
    hipLaunchKernelGGL(k_cache_pack, dim3((unsigned)(m.B * m.H * slices), y), dim3(256), 0, st, m, slices, own);
  } else {
    const int parts = (int)(((long)m.rows_max * m.dh + 256 * MV_PER - 1) / (256 * MV_PER));
    hipLaunchKernelGGL(k_cache_copy, dim3((unsigned)((long)m.B * m.H * parts), y), dim3(256), 0, st, m, parts, own);
  }
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
__device__ __forceinline__ bool bad_penalties(const LogitRules& r, long row) {
  const double *p = r.penalties + 3 * row;
  return !(p[0] > 0.0 && isfinite(p[0]) && isfinite(p[1]) && isfinite(p[2]));
}

// Logits in place would be lost to a caller whose ids or penalties are refused,
// so those are looked at before the first of them changes: 2.5 us more for one row
// of 4096 and a history of 48, 3.7 for 512 rows of 50280 and 512.  Bound by the
// launch; the word holds the number of the call, so nothing has to clear it.
__global__ __launch_bounds__(256) void k_logit_check(LogitRules r) {
  for (long row = blockIdx.x; row < r.rows; row += gridDim.x) {
    bool bad = false;
    for (int i = threadIdx.x; i < r.hist; i += 256) {
      const uint32_t t = r.history[row * r.hist + i];
      bad |= t != NO_TOKEN && t >= (uint32_t)r.V;
    }
    for (int i = threadIdx.x; i < r.nb; i += 256) {
      const uint32_t t = r.bias_ids[row * r.nb + i];
      bad |= t != NO_TOKEN && t >= (uint32_t)r.V;
    }
    const bool pen = threadIdx.x == 0 && r.penalties && bad_penalties(r, row);
    if (bad) set_word(r.err, OE_BAD_TOKEN);
    if (pen) set_word(r.err, OE_BAD_PENALTY);
    if (bad || pen) __hip_atomic_store(r.refused, r.call, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

void logit_check(hipStream_t st, const LogitRules& r) {
  hipLaunchKernelGGL(k_logit_check, dim3(std::min(r.rows, 65536)), dim3(256), 0, st, r);
}

// tokens per block: 2048, or 1024 where that leaves most of the chip idle
constexpr int LR_WIDE = 2048, LR_NARROW = 1024;
int logit_chunks(int V) { return (V + LR_NARROW - 1) / LR_NARROW; }

// two logits of a row, whose start is aligned to one
typedef double v2row __attribute__((ext_vector_type(2), aligned(8)));

// One block per (chunk of the vocabulary, row).  Its logits are requested first;
// the chunk's occurrences in the history and its last bias entry are gathered
// in LDS meanwhile (integer atomics, so their order does not show); then each
// logit is changed, written and compared, so it is read once and written once.
// The row's last block joins the chunks' maxima.  Bound by HBM on many rows
// (512 rows of 50280, 512 tokens of history: 412 MB in 86 us, 4.8 TB/s; each of
// a row's 25 blocks reads the row's history), by its chain of loads, LDS
// atomics and the join on few (one row of 4096 6.4 us, 7 of 31999 9.5).  Of 4096
// tokens a block, half as many of which a CU holds, 92 us; one logit to a load
// and store 99 us at either size.
template <int CH>
__global__ __launch_bounds__(256) void k_logit_rules(LogitRules r, int row0) {
  constexpr int PER = CH / 512;  // pairs of a thread
  __shared__ __align__(16) uint32_t count[CH], entry[CH];
  __shared__ uint32_t words[CH / 32];
  __shared__ double sv[4];
  __shared__ int si[4];
  if (r.refused && *r.refused == r.call) return;
  const int row = row0 + blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = r.V;
  const int c0 = blockIdx.x * CH, len = min(CH, V - c0);
  if (r.row_mask && !r.row_mask[row]) {
    if (tid == 0 && c0 == 0 && r.ids) r.ids[row] = NO_TOKEN;
    return;
  }
  const double* x = r.x + (long)row * V + c0;
  v2row y[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = 2 * (tid + 256 * k);
    y[k] = v2row{0.0, 0.0};
    if (i + 1 < len) y[k] = __builtin_nontemporal_load((const MITOK_GLOBAL v2row*)(x + i));
    else if (i < len) y[k].x = x[i];
  }
  double theta = 1.0, presence = 0.0, frequency = 0.0;
  if (r.penalties) {
    theta = r.penalties[3 * (long)row];
    presence = r.penalties[3 * (long)row + 1];
    frequency = r.penalties[3 * (long)row + 2];
    if (tid == 0 && bad_penalties(r, row)) set_word(r.err, OE_BAD_PENALTY);
  }
  const bool ruled = r.hist > 0 || r.nb > 0;
  if (ruled) {
    for (int i = tid; i < CH / 4; i += 256) ((uint4*)count)[i] = ((uint4*)entry)[i] = make_uint4(0, 0, 0, 0);
  }
  if (r.allowed)
    for (int i = tid; i < (len + 31) / 32; i += 256) words[i] = r.allowed[(long)row * ((V + 31) / 32) + c0 / 32 + i];
  __syncthreads();
  if (ruled) {
    for (int i = tid; i < r.hist; i += 256) {
      const uint32_t t = r.history[(long)row * r.hist + i];
      if (t != NO_TOKEN && t >= (uint32_t)V) set_word(r.err, OE_BAD_TOKEN);
      if (t - (uint32_t)c0 < (uint32_t)len) atomicAdd(&count[t - c0], 1u);
    }
    for (int i = tid; i < r.nb; i += 256) {
      const uint32_t t = r.bias_ids[(long)row * r.nb + i];
      if (t != NO_TOKEN && t >= (uint32_t)V) set_word(r.err, OE_BAD_TOKEN);
      if (t - (uint32_t)c0 < (uint32_t)len) atomicMax(&entry[t - c0], (uint32_t)i + 1);
    }
    __syncthreads();
  }
  double bv = -INFINITY;
  int bi = -1;
  bool nan = false;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = 2 * (tid + 256 * k);
    if (i >= len) break;
    uint2 c = make_uint2(0, 0), en = c;
    if (ruled) c = *(const uint2*)(count + i), en = *(const uint2*)(entry + i);
    const uint32_t ok = r.allowed ? words[i >> 5] >> (i & 31) : 3u;
    const auto change = [&](double v, uint32_t times, uint32_t at, bool may) {
      if (times) {
        v = v > 0.0 ? v / theta : v * theta;
        v -= frequency * (double)times + presence;
      }
      if (at) v += r.bias[(long)row * r.nb + at - 1];
      return may ? v : -INFINITY;
    };
    y[k].x = change(y[k].x, c.x, en.x, ok & 1);
    nan |= isnan(y[k].x);
    argmax_combine(bv, bi, y[k].x, c0 + i);
    double* out = r.out + (long)row * V + c0 + i;
    if (i + 1 < len) {
      y[k].y = change(y[k].y, c.y, en.y, ok & 2);
      nan |= isnan(y[k].y);
      argmax_combine(bv, bi, y[k].y, c0 + i + 1);
      if (r.out) __builtin_nontemporal_store(y[k], (MITOK_GLOBAL v2row*)out);
    } else if (r.out) {
      *out = y[k].x;
    }
  }
  if (__ballot(nan) && lane == 0) set_word(r.err, OE_NAN);
  if (!r.ids) return;
  wave_argmax(bv, bi);
  if (lane == 0) sv[wave] = bv, si[wave] = bi;
  __syncthreads();
  const int chunks = gridDim.x;
  if (tid == 0) {
    for (int w = 1; w < 4; ++w) argmax_combine(bv, bi, sv[w], si[w]);
    if (chunks == 1) r.ids[row] = bv > -INFINITY ? (uint32_t)bi : NO_TOKEN;  // nothing allowed is above -inf
    else {
      st_dev(r.part_v + (long)row * chunks + blockIdx.x, bv);
      st_dev(r.part_i + (long)row * chunks + blockIdx.x, bi);
    }
  }
  if (chunks == 1 || !arrive_last(r.counters + blockIdx.y, chunks)) return;
  if (wave == 0) {
    bv = -INFINITY;
    bi = -1;
    for (int c = lane; c < chunks; c += 64)
      argmax_combine(bv, bi, ld_dev(r.part_v + (long)row * chunks + c), ld_dev(r.part_i + (long)row * chunks + c));
    wave_argmax(bv, bi);
    if (lane == 0) r.ids[row] = bv > -INFINITY ? (uint32_t)bi : NO_TOKEN;
  }
}

void logit_rules(hipStream_t st, const LogitRules& r) {
  // us a call, narrow / wide: 32 rows of 32000 (512 wide blocks) 28.8 / 24.6
  const bool wide = (long)((r.V + LR_WIDE - 1) / LR_WIDE) * r.rows >= 512;
  const int chunks = wide ? (r.V + LR_WIDE - 1) / LR_WIDE : logit_chunks(r.V);
  for (int row0 = 0; row0 < r.rows; row0 += 32768) {  // a counter per row of a launch
    const dim3 grid(chunks, std::min(r.rows - row0, 32768));
    if (wide) hipLaunchKernelGGL(k_logit_rules<LR_WIDE>, grid, dim3(256), 0, st, r, row0);
    else hipLaunchKernelGGL(k_logit_rules<LR_NARROW>, grid, dim3(256), 0, st, r, row0);
  }
}

}  // namespace mitok

// paged_attention.hip — attention of a chunk of new tokens over a paged cache
// (PagedAttn in paged.hpp has the formula).
//
// A tile of 16 slots lies in one page, so a wave looks its page up once a tile,
// one tile ahead of the loads that need it.  New rows are read from the caller's
// rows, not from the pages they are also stored to, so nothing waits for the
// stores and one launch does both.
#include <algorithm>
#include <cmath>

#include "attn_run.hpp"
#include "paged.hpp"

namespace mitok {

// chunk partials: max, sum and unnormalised output of a row
struct PagedWs {
  double* m = nullptr;   // [B][H][n][nsplit]
  double* l = nullptr;
  double2* o = nullptr;  // [B][H][n][nsplit][dh]
};

// A block's place (chunk entry * H + head) and the sequence's pages.
struct PagedAt {
  int b, h, bh, L, cnt, t0, t1, s, n0;
  bool split;
  const uint32_t* table;
  int tiles;       // of a page
  uint32_t magic;  // x / tiles as umulhi(x, magic), x below 2^26
  __device__ __forceinline__ PagedAt(const PagedAttn& a, const PagedPlan& p, const OpTable& own, int rows) {
    const int e = blockIdx.x / a.H;
    const int4 c = op_array<int4>(a.tab, own, p.chunks)[e];
    b = __builtin_amdgcn_readfirstlane(c.x);
    t0 = __builtin_amdgcn_readfirstlane(c.y);
    t1 = __builtin_amdgcn_readfirstlane(c.z);
    const int w = __builtin_amdgcn_readfirstlane(c.w);
    split = w & 1;
    s = (w >> 1) & 31;
    n0 = (w >> 6) * rows;
    h = blockIdx.x - e * a.H;
    bh = b * a.H + h;
    L = op_int(a.tab, own, a.kv_len, b);
    cnt = op_int(a.tab, own, a.count, b);
    t1 = min(t1, L + min(n0 + rows, cnt));
    table = a.table + (long)b * a.max_pages;
    tiles = a.page_rows / PAGE_TILE;
    magic = 0xFFFFFFFFu / (uint32_t)tiles + 1;
  }
  // the page of a tile (its number among the sequence's pages and its id); an
  // id that is none sets the error word and reads page 0
  __device__ __forceinline__ int page(const PagedAttn& a, int t, uint32_t& id) const {
    const uint32_t x = (uint32_t)t / PAGE_TILE, p = tiles == 1 ? x : __umulhi(x, magic);
    id = __builtin_amdgcn_readfirstlane(ld_glb(table + p));
    if (id >= a.pages) {
      set_word(a.err, PE_BAD_PAGE);
      id = 0;
    }
    return (int)p;
  }
};

// A tile's rows in their page, or among the new rows from slot L on.
struct PagedTile {
  const double2 *k, *v, *kn, *vn;  // of the tile's first slot
  int fresh;                       // rows from here on are new ones
  long step;
  __device__ __forceinline__ PagedTile() {}
  __device__ __forceinline__ PagedTile(const PagedAttn& a, const PagedAt& at, int t, int page, uint32_t id) {
    const long in = (((long)id * a.H + at.h) * a.page_rows + (t - page * a.page_rows)) * a.dh;
    const long nw = (long)at.b * a.new_b + (long)(t - at.L) * a.new_row + (long)at.h * a.new_head;
    k = a.kp + in;
    v = a.vp + in;
    kn = a.kn + nw;
    vn = a.vn + nw;
    fresh = at.L - t;
    step = a.new_row;
  }
  __device__ __forceinline__ const double2* key(int r, int dh) const { return r >= fresh ? kn + r * step : k + (uint32_t)r * (uint32_t)dh; }
  __device__ __forceinline__ const double2* value(int r, int dh) const { return r >= fresh ? vn + r * step : v + (uint32_t)r * (uint32_t)dh; }
};

// What the first block of a group of rows does besides: its new rows go to
// their pages, and its output rows past the sequence's last are zero.
__device__ __forceinline__ void paged_store(const PagedAttn& a, const PagedAt& at, int rows) {
  if (at.s) return;
  const int last = min(at.n0 + rows, at.cnt), dh = a.dh;
  for (int x = threadIdx.x; x < (last - at.n0) * dh; x += 256) {
    const int r = at.n0 + x / dh, e = x % dh, slot = at.L + r;
    const long from = (long)at.b * a.new_b + (long)r * a.new_row + (long)at.h * a.new_head + e;
    const uint32_t id = at.table[slot / a.page_rows];
    if (id >= a.pages) {
      set_word(a.err, PE_BAD_PAGE);
      continue;
    }
    if (a.stamp && at.h == 0 && e == 0 && (slot % a.page_rows == 0 || r == at.n0)) {
      const uint32_t who = (uint32_t)at.b << 16 | (uint32_t)(slot / a.page_rows & 0xFFFF);
      const unsigned long long mine = (unsigned long long)a.call << 32 | who, had = atomicExch(a.stamp + id, mine);
      if (had >> 32 == a.call && had != mine) set_word(a.err, PE_SHARED_PAGE);
    }
    const long to = (((long)id * a.H + at.h) * a.page_rows + slot % a.page_rows) * dh + e;
    a.kp[to] = a.kn[from];
    a.vp[to] = a.vn[from];
  }
  const int from = max(at.n0, at.cnt), idle = min(at.n0 + rows, a.n) - from;
  for (int x = threadIdx.x; x < idle * dh; x += 256)
    a.out[((long)at.b * a.n + from + x / dh) * a.ldo + (long)at.h * dh + x % dh] = make_double2(0.0, 0.0);
}

// the biases of slots t + 4 e + kq for new row i (0 without any)
__device__ __forceinline__ void paged_bias(const PagedAttn& a, const PagedAt& at, int t, int kq, int i, double (&bf)[4]) {
  if (!a.bias) return;
  const double* bias = a.bias + (long)at.h * a.bias_stride + (long)(at.L + min(i, at.cnt - 1)) * a.bias_row;
#pragma unroll
  for (int e = 0; e < 4; ++e) bf[e] = ld_glb(bias + min(t + 4 * e + kq, at.t1 - 1));
}

// Bits e of a tile's slots t + 4 e + kq that new row i sees
__device__ __forceinline__ unsigned paged_sees(const PagedAt& at, int t, int kq, int i) {
  const int past = min(at.t1, at.L + min(i, at.cnt - 1) + 1) - t - kq;  // slots kq, kq + 4, .. below past + kq
  return past <= 0 ? 0u : past > 12 ? 15u : (1u << ((past + 3) >> 2)) - 1u;
}

// A row's output element: final where the group has one chunk, else the chunk's part.
__device__ __forceinline__ void paged_put(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at, int i,
                                          int e, double2 v, double sum) {
  if (!at.split) a.out[((long)at.b * a.n + i) * a.ldo + (long)at.h * a.dh + e] = make_double2(v.x / sum, v.y / sum);
  else ws.o[(((long)at.bh * a.n + i) * p.nsplit + at.s) * a.dh + e] = v;
}
__device__ __forceinline__ void paged_put_sum(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at,
                                              int i, double m, double l) {
  if (i >= at.cnt || !at.split) return;
  const long x = ((long)at.bh * a.n + i) * p.nsplit + at.s;
  ws.m[x] = m;
  ws.l[x] = l;
}

// Up to 32 new rows: one block per (chunk of slots, head, sequence, 16 NG rows).
// Its four waves are NG groups of 16 rows by 4 / NG that share the chunk's tiles,
// each with a running maximum and sum, one pass over the keys and values:
//   S^T = K Q^T   Re(q k) is a real product of length 2 dh: (kr, ki) with
//                 (qr, -qi) scaled.  A lane holds key row lane % 16 and, of each
//                 four complex columns, lane / 16: one 16-byte load feeds two MFMAs.
//   O^T += V^T P^T  element e of S^T's tile is slot 4 e + lane / 16 of row
//                 lane % 16, which is the B operand of the e-th step.
// Keys and values go from memory to the matrix cores without LDS, which holds
// the queries in the order the lanes read them.
template <int DHP, int NG, bool FULL>
__global__ __launch_bounds__(256, DHP <= 128 ? 2 : 1) void k_paged_split(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
  constexpr int KG = 4 / NG;       // waves that share a group's slots
  constexpr int U = DHP / 4;       // 16-byte key loads of a lane per tile, two MFMAs each
  constexpr int CT = DHP / 16;     // 16-column tiles of the values
  constexpr bool PRE = DHP <= 64;  // the next tile's rows wait in registers
  constexpr int OSTR = DHP + 1;    // LDS row of an output: rows in different banks
  constexpr int PARTS = DHP <= 64 ? KG : 1;  // LDS holds this many waves' outputs of each group
  constexpr size_t Q_BYTES = (size_t)NG * U * 64 * sizeof(double2);
  constexpr size_t O_BYTES = (size_t)PARTS * NG * 16 * OSTR * sizeof(double2);
  __shared__ __align__(16) unsigned char lds[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
  __shared__ double sm[4][16], sl[4][16], sum[NG][16];
  double2* qs = (double2*)lds;  // [NG][U][64], then outputs [PARTS][NG * 16][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ng = wave % NG, kg = wave / NG;
  const int row = lane & 15, kq = lane >> 4, dh = a.dh;
  const PagedAt at(a, p, own, 16 * NG);
  paged_store(a, at, 16 * NG);
  if (at.n0 >= at.cnt) return;
  const int t0 = at.t0, t1 = at.t1;
  const int i = at.n0 + 16 * ng + row;  // this lane's new row
  const double2* qw = qs + ng * U * 64 + lane;

  double2 kf[PRE ? U : 1], vf[PRE ? 4 : 1][PRE ? CT : 1];
  double bf[4] = {0.0, 0.0, 0.0, 0.0};
  // a slot past the end reads the last one's row, with weight 0.  Padded columns:
  // keys of 0 (0 times an infinity would be NaN), value columns that nobody reads.
  const auto key_at = [&](const double2* k, int u) {
    if (!FULL && 4 * u + kq >= dh) return make_double2(0.0, 0.0);
    return ld_glb(k + 4 * u + kq);
  };
  const auto value_at = [&](const double2* v, int c) { return ld_glb(v + (FULL ? row + 16 * c : min(row + 16 * c, dh - 1))); };
  const auto key_row = [&](const PagedTile& tl, int t) { return tl.key(min(row, t1 - 1 - t), dh); };
  const auto value_row = [&](const PagedTile& tl, int t, int q) { return tl.value(min(4 * q + kq, t1 - 1 - t), dh); };
  const auto load_keys = [&](const PagedTile& tl, int t) {
    if constexpr (PRE) {
      const double2* k = key_row(tl, t);
#pragma unroll
      for (int u = 0; u < U; ++u) kf[u] = key_at(k, u);
    }
    paged_bias(a, at, t, kq, i, bf);
  };
  const auto load_values = [&](const PagedTile& tl, int t) {
    if constexpr (PRE) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const double2* v = value_row(tl, t, q);
#pragma unroll
        for (int c = 0; c < CT; ++c) vf[q][c] = value_at(v, c);
      }
    }
  };
  int t = t0 + 16 * kg;
  PagedTile tile, next;
  uint32_t id = 0;
  int pg = 0;
  if (t < t1) {
    pg = at.page(a, t, id);
    tile = PagedTile(a, at, t, pg, id);
    load_keys(tile, t);
    load_values(tile, t);
    if (t + 16 * KG < t1) pg = at.page(a, t + 16 * KG, id);
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
    const bool more = t + 16 * KG < t1;
    if (more) next = PagedTile(a, at, t + 16 * KG, pg, id);
    if (t + 32 * KG < t1) pg = at.page(a, t + 32 * KG, id);
    v4d s = {0.0, 0.0, 0.0, 0.0}, z = s;
    const double2* k0 = PRE ? nullptr : key_row(tile, t);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const double2 k = PRE ? kf[PRE ? u : 0] : key_at(k0, u), q = qw[u * 64];
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(k.x, q.x, s, 0, 0, 0);
      z = __builtin_amdgcn_mfma_f64_16x16x4f64(k.y, q.y, z, 0, 0, 0);
      if (u % (PRE ? 4 : 16) == (PRE ? 3 : 15)) __builtin_amdgcn_sched_barrier(0);  // so many operands at a time in registers
    }
    const unsigned vis = paged_sees(at, t, kq, i);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = vis >> e & 1 ? s[e] + z[e] + bf[e] : -INFINITY;
    if (more) load_keys(next, t + 16 * KG);
    run.soften(s);
    const bool edge = t + 15 > at.L + at.n0;  // some row does not see some slot
    bool fine = true;
    if (PRE && edge) {
#pragma unroll
      for (int q = 0; q < (PRE ? 4 : 0); ++q)
#pragma unroll
        for (int c = 0; c < CT; ++c) fine &= attn_finite(vf[q][c]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const double2* v0 = PRE ? nullptr : value_row(tile, t, q);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        double2 v = PRE ? vf[PRE ? q : 0][PRE ? c : 0] : value_at(v0, c);
        if (!PRE && edge) fine &= attn_finite(v);
        run.output(s, q, c, v);
      }
      if (!PRE) __builtin_amdgcn_sched_barrier(0);
    }
    if (more) load_values(next, t + 16 * KG);
    if (__ballot(!fine)) run.add_left_out([&](int k) { return tile.value(k, dh); }, dh, t1 - t, s, vis);
    tile = next;
  }

  // the waves of a group, rescaled to their common maximum and added in order
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) sm[wave][row] = run.m, sl[wave][row] = run.l;
  __syncthreads();  // and the queries' last read
  double M = -INFINITY;
#pragma unroll
  for (int g = 0; g < KG; ++g) M = fmax(M, sm[g * NG + ng][row]);
  const double base = M == -INFINITY ? 0.0 : M;
  double Ls = 0.0;
#pragma unroll
  for (int g = 0; g < KG; ++g) Ls += sl[g * NG + ng][row] * exp(sm[g * NG + ng][row] - base);
  const double f = exp(run.m - base);
#pragma unroll
  for (int g = 0; g < KG; g += PARTS) {
    if (kg / PARTS * PARTS == g && i < at.cnt) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          double2* to = os + ((kg - g) * NG * 16 + 16 * ng + row) * OSTR + 16 * c + 4 * e + kq;
          const double2 v = make_double2(run.o_re[c][e] * f, run.o_im[c][e] * f);
          *to = g ? cadd(*to, v) : v;
        }
    }
    __syncthreads();
  }
  if (kg == 0 && kq == 0) {
    sum[ng][row] = Ls;
    paged_put_sum(a, p, ws, at, i, M, Ls);
  }
  __syncthreads();
  for (int x = tid; x < min(16 * NG, at.cnt - at.n0) * dh; x += 256) {
    const int r = x / dh, e = x - r * dh;
    double2 v = os[r * OSTR + e];
#pragma unroll
    for (int g = 1; g < PARTS; ++g) v = cadd(v, os[(g * NG * 16 + r) * OSTR + e]);
    paged_put(a, p, ws, at, at.n0 + r, e, v, sum[r >> 4][r & 15]);
  }
}

// 33 new rows and more: every wave has 16 rows of its own and the block's tiles
// are shared through LDS.  A wave requests a quarter of the next tile, in the
// order the matrix cores take it, among the first products of the current one
// and leaves it in LDS after the last.  The queries wait in registers.  A wave
// whose rows lie before a tile leaves its products out.
template <int DHP, bool FULL>
__global__ __launch_bounds__(256, DHP <= 64 ? 2 : 1) void k_paged_tile(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
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
  const int row = lane & 15, kq = lane >> 4, dh = a.dh;
  const PagedAt at(a, p, own, 64);
  paged_store(a, at, 64);
  if (at.n0 >= at.cnt) return;
  const int t0 = at.t0, t1 = at.t1;
  const int i = at.n0 + 16 * wave + row;
  // This wave's fragments of the tile at t: value columns 16 c + lane % 16 of row
  // 4 q + kq, and keys, of which four lanes load 64 bytes of a row (a quarter
  // wave then touches 4 lines, not 16) and leave them where the products' lanes
  // read them; kq's rotation of the row keeps both sides off shared banks.
  const int krow = lane >> 2, kcol = lane & 3;
  const int kput = kcol * 16 + ((krow + 4 * kcol) & 15), kget = kq * 16 + ((row + 4 * kq) & 15);
  double2 next[PER];
  const double2 *kfrom = nullptr, *vfrom = nullptr;
  const auto rows_of = [&](const PagedTile& tl, int t) {
    kfrom = tl.key(min(krow, t1 - 1 - t), dh) + kcol + wave * U;
    vfrom = tl.value(min(4 * wave + kq, t1 - 1 - t), dh);
  };
  const auto fetch_one = [&](int j) {
    if (j < U / 4) next[j] = FULL || wave * U + 4 * j + kcol < dh ? ld_glb(kfrom + 4 * j) : make_double2(0.0, 0.0);
    else next[j] = ld_glb(vfrom + (FULL ? row + 16 * (j - U / 4) : min(row + 16 * (j - U / 4), dh - 1)));
  };
  // into LDS; values of the new rows' own slots that are not finite stay out
  const auto leave = [&](int buf, int t) {
    if (t + 15 > at.L + at.n0) {
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
  if (t0 >= t1) return;  // not where the plan is the call's own
  uint32_t id;
  int pg = at.page(a, t0, id);
  PagedTile tile(a, at, t0, pg, id), ahead = tile;
  rows_of(tile, t0);
#pragma unroll
  for (int j = 0; j < PER; ++j) fetch_one(j);
  if (t0 + 16 < t1) pg = at.page(a, t0 + 16, id);
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
    const double2* lt = tiles + buf * F * 64;
    const bool more = t + 16 < t1;
    if (more) {
      ahead = PagedTile(a, at, t + 16, pg, id);
      rows_of(ahead, t + 16);  // after the last tile: that one's rows again, read by nobody
    }
    if (t + 32 < t1) pg = at.page(a, t + 32, id);
    const bool mine = t <= at.L + at.n0 + 16 * wave + 15 && at.n0 + 16 * wave < at.cnt;  // some row of this wave sees the tile
    double bf[4] = {0.0, 0.0, 0.0, 0.0};
    v4d s = {0.0, 0.0, 0.0, 0.0}, z = s;
    if (mine) paged_bias(a, at, t, kq, i, bf);
#pragma unroll
    for (int g = 0; g < U / 4; ++g) {
#pragma unroll
      for (int j = 0; j < PER / (U / 4); ++j) fetch_one(g * (PER / (U / 4)) + j);
      if (!mine) continue;
      double2 k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = lt[(4 * g + j) * 64 + kget];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = __builtin_amdgcn_mfma_f64_16x16x4f64(k[j].x, qf[4 * g + j].x, s, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f64_16x16x4f64(k[j].y, qf[4 * g + j].y, z, 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (mine) {
      const unsigned vis = paged_sees(at, t, kq, i);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = vis >> e & 1 ? s[e] + z[e] + bf[e] : -INFINITY;
      run.soften(s);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int c = 0; c < CT; ++c) run.output(s, q, c, lt[(U + q * CT + c) * 64 + lane]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (t + 15 > at.L + at.n0 && left_out) run.add_left_out([&](int k) { return tile.value(k, dh); }, dh, t1 - t, s, vis);
    }
    leave(buf ^ 1, t + 16);  // read by nobody since the last barrier (after the last tile: by nobody at all)
    tile = ahead;
    __syncthreads();
  }
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) {
    sum[16 * wave + row] = run.l;
    paged_put_sum(a, p, ws, at, i, run.m, run.l);
  }
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      os[(16 * wave + row) * OSTR + 16 * c + 4 * e + kq] = make_double2(run.o_re[c][e], run.o_im[c][e]);
  __syncthreads();
  for (int x = tid; x < min(64, at.cnt - at.n0) * dh; x += 256) {
    const int r = x / dh, e = x - r * dh;
    paged_put(a, p, ws, at, at.n0 + r, e, os[r * OSTR + e], sum[r]);
  }
}

// Joins the chunks of the rows whose group was split.
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
  const int cnt = op_int(a.tab, own, a.count, b);
  const int* splits = op_array<int>(a.tab, own, p.splits) + (long)b * p.groups;
  for (long x = (long)blockIdx.y * 256 + threadIdx.x; x < (long)cnt * a.dh; x += (long)gridDim.y * 256) {
    const int i = (int)(x / a.dh), e = (int)(x - (long)i * a.dh);
    const int ns = splits[i / (16 * p.ng)];
    if (ns == 1) continue;
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
  }
}

PagedPlan paged_plan(const PagedAttn& a, const int* kv_len, const int* count, std::vector<int>& lists) {
  PagedPlan p;
  p.ng = a.n <= 16 || a.dh > 128 ? 1 : a.n <= 32 ? 2 : 4;
  const int rows = 16 * p.ng, unit = 64 / p.ng;  // slots that a block's waves take at a time
  p.groups = (a.n + rows - 1) / rows;
  const double places = a.dh <= 64 || (a.dh <= 128 && p.ng < 4) ? 512.0 : 256.0;  // blocks the chip holds at once
  // the slots that a group's rows see, 0 without rows
  const auto seen = [&](int b, int g) { return g * rows < count[b] ? kv_len[b] + std::min((g + 1) * rows, count[b]) : 0; };
  int longest = 0;
  double all = 0.0;  // units of the call
  for (int b = 0; b < a.B; ++b)
    for (int g = 0; g < p.groups; ++g) {
      const int len = seen(b, g);
      longest = std::max(longest, len);
      all += (len + unit - 1) / unit;
    }
  const double tile = 0.7 + 1.6 * a.dh / 64, unit_mb_us = unit * a.dh * 32 / 5.2e6 / p.groups;
  const int most = std::max(1, (longest + unit - 1) / unit);
  int each = 1;  // units of a chunk
  if (all * a.H > places) {
    double least = 1e300;
    int last = 0;
    for (int k : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32}) {
      const int c = (most + k - 1) / k, slots = c * unit;
      if (c == last) continue;
      last = c;
      double blocks = 0.0;
      for (int b = 0; b < a.B; ++b)
        for (int g = 0; g < p.groups; ++g) blocks += std::max(1, (seen(b, g) + slots - 1) / slots);
      const bool split = blocks > (double)a.B * p.groups;
      blocks *= a.H;
      const double full = std::floor(blocks / places), rest = blocks - full * places;
      const double work = all * a.H / blocks;  // units of a block, on average
      double cost = full * (3.0 + work * std::max(2.0 * tile * places / 512.0, places * unit_mb_us));
      if (rest > 0.0) cost += 8.0 + std::max(c * tile * (rest > 256.0 ? 2.0 : 1.45), rest * work * unit_mb_us);
      if (split) cost += blocks * 16 * std::min(rows, a.n) * a.dh * 2 / 5.2e6;
      if (cost < least) least = cost, each = c;
    }
  }
  each = std::max(each, (most + PAGED_MAX_SPLIT - 1) / PAGED_MAX_SPLIT);
  std::vector<int> splits;
  std::vector<int4> list;
  for (int b = 0; b < a.B; ++b)
    for (int g = 0; g < p.groups; ++g) {
      const int len = seen(b, g), units = std::max(1, (len + unit - 1) / unit), k = (units + each - 1) / each;
      const int slots = (units + k - 1) / k * unit, n = std::max(1, (len + slots - 1) / slots);
      for (int s = 0; s < n; ++s) list.push_back(make_int4(b, s * slots, std::min(len, (s + 1) * slots), g * 64 + s * 2 + (n > 1)));
      splits.push_back(n);
      p.nsplit = std::max(p.nsplit, n);
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

static size_t paged_layout(const PagedAttn& a, const PagedPlan& p, char* base, PagedWs& ws) {
  if (p.nsplit == 1) return 0;
  const size_t rows = (size_t)a.B * a.H * a.n * p.nsplit;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  ws.m = (double*)take(rows * sizeof(double));
  ws.l = (double*)take(rows * sizeof(double));
  ws.o = (double2*)take(rows * a.dh * sizeof(double2));
  return at;
}

size_t paged_ws_bytes(const PagedAttn& a, const PagedPlan& p) {
  PagedWs ws;
  return paged_layout(a, p, nullptr, ws);
}

template <int DHP, bool FULL>
static void launch_paged(hipStream_t st, const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const OpTable& own) {
  const dim3 grid((unsigned)((long)p.entries * a.H));
  const auto go = [&](auto kern) { MITOK_LAUNCH(kern, grid, dim3(256), 0, st, a, p, ws, own); };
  if constexpr (DHP <= 128) {
    if (p.ng == 4) return go(k_paged_tile<DHP, FULL>);
    if (p.ng == 2) return go(k_paged_split<DHP, 2, FULL>);
  }
  go(k_paged_split<DHP, 1, FULL>);
}

void paged_attention(hipStream_t st, const PagedAttn& a, const PagedPlan& p, const OpTable& own) {
  PagedWs ws;
  paged_layout(a, p, (char*)a.ws, ws);
  const auto width = [&](auto padded, auto whole, int dhp) { a.dh == dhp ? whole(st, a, p, ws, own) : padded(st, a, p, ws, own); };
  if (a.dh <= 16) width(launch_paged<16, false>, launch_paged<16, true>, 16);
  else if (a.dh <= 32) width(launch_paged<32, false>, launch_paged<32, true>, 32);
  else if (a.dh <= 64) width(launch_paged<64, false>, launch_paged<64, true>, 64);
  else if (a.dh <= 128) width(launch_paged<128, false>, launch_paged<128, true>, 128);
  else width(launch_paged<256, false>, launch_paged<256, true>, 256);
  if (p.nsplit > 1) {
    const unsigned parts = (unsigned)std::min<long>(((long)a.n * a.dh + 255) / 256, 4096);
    hipLaunchKernelGGL(k_paged_join, dim3((unsigned)(a.B * a.H), parts), dim3(256), 0, st, a, p, ws, own);
  }
}

}  // namespace mitok

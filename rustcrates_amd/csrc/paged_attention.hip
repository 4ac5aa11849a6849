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

// partials of the groups that were cut: max, sum and unnormalised output of a row
struct PagedWs {
  double* m = nullptr;   // [H][part rows]
  double* l = nullptr;
  double2* o = nullptr;  // [H][part rows][dh]
};

// A piece of work: a head's new rows n0.. of a sequence over slots [t0, t1).
struct PagedAt {
  int b, h, L, cnt, t0, t1, n0;
  int part;  // its rows' place among the partials, -1: the group has one piece
  const uint32_t* table;
  int tiles;       // of a page
  uint32_t magic;  // x / tiles as umulhi(x, magic), x below 2^26
  const double2 *kn, *vn;  // slot 0 of the new rows, had they one
  __device__ __forceinline__ PagedAt(const PagedAttn& a, const PagedPlan& p, const OpTable& own, int piece, int head) {
    const int4 c = op_array<int4>(a.tab, own, p.pieces)[piece];
    const int d = op_array<int>(a.tab, own, p.places)[piece];
    h = head;
    b = __builtin_amdgcn_readfirstlane(c.x);
    n0 = __builtin_amdgcn_readfirstlane(c.y);
    t0 = __builtin_amdgcn_readfirstlane(c.z);
    part = __builtin_amdgcn_readfirstlane(d);
    L = op_int(a.tab, own, a.kv_len, b);
    cnt = op_int(a.tab, own, a.count, b);
    t1 = min(__builtin_amdgcn_readfirstlane(c.w), L + min(n0 + p.rows, cnt));
    rest(a);
  }
  __device__ __forceinline__ PagedAt(const PagedAttn& a, int sequence, int head, int len, int rows, int from, int to)
      : b(sequence), h(head), L(len), cnt(rows), t0(from), t1(to), n0(0), part(-1) {
    rest(a);
  }
  __device__ __forceinline__ void rest(const PagedAttn& a) {
    table = a.table + (long)b * a.max_pages;
    tiles = a.page_rows / PAGE_TILE;
    magic = 0xFFFFFFFFu / (uint32_t)tiles + 1;
    const long nw = (long)b * a.new_b + (long)h * a.new_head - (long)L * a.new_row;
    kn = a.kn + nw;
    vn = a.vn + nw;
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

// A tile's rows: in their page, or from slot L on among the new rows.
struct PagedTile {
  long in;  // of the tile's first slot
  int t;
  __device__ __forceinline__ PagedTile() {}
  __device__ __forceinline__ PagedTile(const PagedAttn& a, const PagedAt& at, int slot, int page, uint32_t id)
      : in((((long)id * a.H + at.h) * a.page_rows + (slot - page * a.page_rows)) * a.dh), t(slot) {}
  __device__ __forceinline__ const double2* key(const PagedAttn& a, const PagedAt& at, int r) const {
    return t + r >= at.L ? at.kn + (long)(t + r) * a.new_row : a.kp + in + (uint32_t)r * (uint32_t)a.dh;
  }
  __device__ __forceinline__ const double2* value(const PagedAttn& a, const PagedAt& at, int r) const {
    return t + r >= at.L ? at.vn + (long)(t + r) * a.new_row : a.vp + in + (uint32_t)r * (uint32_t)a.dh;
  }
};

// What the first piece of a group of rows does besides: its new rows go to
// their pages, and its output rows past the sequence's last are zero.
__device__ __forceinline__ void paged_store(const PagedAttn& a, const PagedAt& at, int rows) {
  if (at.t0) return;
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

// A row's output element: final where the group has one piece, else the piece's part.
__device__ __forceinline__ void paged_put(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at, int i,
                                          int e, double2 v, double sum) {
  if (at.part < 0) a.out[((long)at.b * a.n + i) * a.ldo + (long)at.h * a.dh + e] = make_double2(v.x / sum, v.y / sum);
  else ws.o[((long)at.h * p.part_rows + at.part + i - at.n0) * a.dh + e] = v;
}
__device__ __forceinline__ void paged_put_sum(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at,
                                              int i, double m, double l) {
  if (i >= at.cnt || at.part < 0) return;
  const long x = (long)at.h * p.part_rows + at.part + i - at.n0;
  ws.m[x] = m;
  ws.l[x] = l;
}

// Up to 32 rows of a sequence.  The four waves are NG groups of 16 rows by 4 / NG that
// share the chunk's tiles, each with a running maximum and sum, one pass over the
// keys and values:
//   S^T = K Q^T   Re(q k) is a real product of length 2 dh: (kr, ki) with
//                 (qr, -qi) scaled.  A lane holds key row lane % 16 and, of each
//                 four complex columns, lane / 16: one 16-byte load feeds two MFMAs.
//   O^T += V^T P^T  element e of S^T's tile is slot 4 e + lane / 16 of row
//                 lane % 16, which is the B operand of the e-th step.
// Keys and values go from memory to the matrix cores without LDS, which holds
// the queries in the order the lanes read them.  Bound by the bytes of keys and values:
// 64 sequences of one row, 12 heads, 400 to 511 slots of head dim 64, 721 MB in 138 us
// (5.2 TB/s); one sequence of 160 slots and 8 heads 10.4 us, a block's chain of
// lookups, loads and merges.
template <int DHP>
constexpr size_t split_lds(int ng) {
  return std::max((size_t)ng * (DHP / 4) * 64 * sizeof(double2), (size_t)(DHP <= 64 ? 4 / ng : 1) * ng * 16 * (DHP + 1) * sizeof(double2));
}
struct PagedSums {  // in LDS
  double m[4][16], l[4][16], sum[64];
  int left_out;  // some value stayed out of a tile
};
template <int DHP, int NG, bool FULL>
__device__ __forceinline__ void paged_split(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at,
                                            unsigned char* lds, PagedSums& sh) {
  constexpr int KG = 4 / NG;       // waves that share a group's slots
  constexpr int U = DHP / 4;       // 16-byte key loads of a lane per tile, two MFMAs each
  constexpr int CT = DHP / 16;     // 16-column tiles of the values
  constexpr bool PRE = DHP <= 64;  // the next tile's rows wait in registers
  constexpr int OSTR = DHP + 1;    // LDS row of an output: rows in different banks
  constexpr int PARTS = DHP <= 64 ? KG : 1;  // LDS holds this many waves' outputs of each group
  double2* qs = (double2*)lds;  // [NG][U][64], then outputs [PARTS][NG * 16][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ng = wave % NG, kg = wave / NG;
  const int row = lane & 15, kq = lane >> 4, dh = a.dh;
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
  const auto key_row = [&](const PagedTile& tl, int t) { return tl.key(a, at, min(row, t1 - 1 - t)); };
  const auto value_row = [&](const PagedTile& tl, int t, int q) { return tl.value(a, at, min(4 * q + kq, t1 - 1 - t)); };
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
    if (__ballot(!fine)) run.add_left_out([&](int k) { return tile.value(a, at, k); }, dh, t1 - t, s, vis);
    tile = next;
  }

  // the waves of a group, rescaled to their common maximum and added in order
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) sh.m[wave][row] = run.m, sh.l[wave][row] = run.l;
  __syncthreads();  // and the queries' last read
  double M = -INFINITY;
#pragma unroll
  for (int g = 0; g < KG; ++g) M = fmax(M, sh.m[g * NG + ng][row]);
  const double base = M == -INFINITY ? 0.0 : M;
  double Ls = 0.0;
#pragma unroll
  for (int g = 0; g < KG; ++g) Ls += sh.l[g * NG + ng][row] * exp(sh.m[g * NG + ng][row] - base);
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
    sh.sum[16 * ng + row] = Ls;
    paged_put_sum(a, p, ws, at, i, M, Ls);
  }
  __syncthreads();
  for (int x = tid; x < min(16 * NG, at.cnt - at.n0) * dh; x += 256) {
    const int r = x / dh, e = x - r * dh;
    double2 v = os[r * OSTR + e];
#pragma unroll
    for (int g = 1; g < PARTS; ++g) v = cadd(v, os[(g * NG * 16 + r) * OSTR + e]);
    paged_put(a, p, ws, at, at.n0 + r, e, v, sh.sum[r]);
  }
}

// More than 32 rows of a sequence: every wave has 16 rows of its own and the block's
// tiles are shared through LDS.  A wave requests a quarter of the next tile, in the
// order the matrix cores take it, among the first products of the current one
// and leaves it in LDS after the last.  The queries wait in registers.  A wave
// whose rows lie before a tile leaves its products out.  Bound by a wave's waits between
// its MFMAs (33% of its time: LDS reads, the barrier a tile, loads), which two waves a
// SIMD hide in part.  Three sequences of 12 heads of 64, inputs changing from call to
// call: 193 to 700 rows behind 774 to 1024 slots 237 us, of which the matrix cores are
// busy for 112 (219 us where the inputs stay); 392 to 700 behind 568 to 1024 302 us, 145
// busy.
template <int DHP>
constexpr size_t tile_lds() {  // keys [U] and values [4][CT] in 1 KB fragments, twice; then outputs [64][DHP + 1]
  return std::max(2 * (size_t)(DHP / 2) * 64 * sizeof(double2), (size_t)64 * (DHP + 1) * sizeof(double2));
}
template <int DHP, bool FULL>
__device__ __forceinline__ void paged_tile(const PagedAttn& a, const PagedPlan& p, const PagedWs& ws, const PagedAt& at,
                                           unsigned char* lds, PagedSums& sh) {
  constexpr int U = DHP / 4, CT = DHP / 16;
  constexpr int F = U + 4 * CT;    // 1 KB fragments of a tile: keys [U], values [4][CT]
  constexpr int PER = F / 4;       // of each wave
  constexpr int OSTR = DHP + 1;
  double2* tiles = (double2*)lds;  // [2][F][64], then outputs [64][OSTR]
  double2* os = (double2*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, kq = lane >> 4, dh = a.dh;
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
    kfrom = tl.key(a, at, min(krow, t1 - 1 - t)) + kcol + wave * U;
    vfrom = tl.value(a, at, min(4 * wave + kq, t1 - 1 - t));
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
      if (!fine) sh.left_out = 1;
    }
    double2* to = tiles + buf * F * 64;
#pragma unroll
    for (int j = 0; j < U / 4; ++j) to[(wave * (U / 4) + j) * 64 + kput] = next[j];
#pragma unroll
    for (int c = 0; c < CT; ++c) to[(U + wave * CT + c) * 64 + lane] = next[U / 4 + c];
  };
  if (tid == 0) sh.left_out = 0;
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
      if (t + 15 > at.L + at.n0 && sh.left_out) run.add_left_out([&](int k) { return tile.value(a, at, k); }, dh, t1 - t, s, vis);
    }
    leave(buf ^ 1, t + 16);  // read by nobody since the last barrier (after the last tile: by nobody at all)
    tile = ahead;
    __syncthreads();
  }
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) {
    sh.sum[16 * wave + row] = run.l;
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
    paged_put(a, p, ws, at, at.n0 + r, e, os[r * OSTR + e], sh.sum[r]);
  }
}

// One new row each of up to 16 sequences of equal length, head dims up to 64: one
// block per (bunch of sequences, head).  Sequences whose tables begin with the same
// pages are beams of one prompt: a tile of those pages is read once, and its products
// are those of all of them, a column of the matrix cores each.  The other tiles are
// each one sequence's; the products' other columns get weight 0.  Which tiles are
// shared is read off the tables, whatever the caller took them for: a run of
// sequences holds in common the pages up to the first in which a neighbour differs.
// 32 prompts of 4 beams, 200 to 248 slots of which 128 are shared, 8 heads: the 256
// blocks take the longest bunch's time, 67 us (4.1 TB/s of the 275 MB that have to be
// read), with eight waves each, two a SIMD; a call 85 us against 89 with four waves
// where the inputs change from call to call, 74 against 82 where they stay.  512 blocks of
// single sequences' pieces and more read 470 MB and take longer than either.  More
// blocks than CUs stand two on a CU with four waves: 64 prompts of 8 beams 258 us a call,
// 253 with eight waves, where the inputs change, 216 and 226 where they stay.
struct BeamRuns {  // in LDS
  int4 at[32];     // tiles [x, y) of all from tile z of sequence w & 15 for columns w >> 8
  int n;
};
template <int DHP, bool FULL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_paged_beams(PagedAttn a, PagedPlan p, OpTable own) {
  constexpr int U = DHP / 4, CT = DHP / 16, OSTR = DHP + 1;
  __shared__ __align__(16) unsigned char lds[std::max((size_t)U * 64, (size_t)WAVES * 16 * OSTR) * sizeof(double2)];
  __shared__ double sm[WAVES][16], sl[WAVES][16], sums[16];
  __shared__ BeamRuns runs;
  __shared__ int same[16];  // pages in common with the sequence before
  double2* qs = (double2*)lds;  // [U][64], then outputs [waves][16][OSTR]
  double2* os = (double2*)lds;
  const int bunch = blockIdx.x / a.H, h = blockIdx.x - bunch * a.H;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, kq = lane >> 4, dh = a.dh;
  const int4 mine = op_array<int4>(a.tab, own, p.pieces)[bunch];
  const int b0 = __builtin_amdgcn_readfirstlane(mine.x), m = __builtin_amdgcn_readfirstlane(mine.y);
  const int L = op_int(a.tab, own, a.kv_len, b0), tiles = L / PAGE_TILE + 1;
  for (int k = wave; k < m; k += WAVES) {
    PagedAt at(a, b0 + k, h, L, 1, 0, L + 1);
    if (lane == 0) same[k] = 0;
    if (k) {  // whole pages of rows that both have
      const int pages = L / a.page_rows;
      int c = 0;
      for (int j0 = 0; j0 < pages; j0 += 64) {
        const bool differ = j0 + lane < pages && at.table[j0 + lane] != at.table[j0 + lane - a.max_pages];
        const unsigned long long v = __ballot(differ);
        if (v) {
          c = j0 + __ffsll(v) - 1;
          break;
        }
        c = min(pages, j0 + 64);
      }
      if (lane == 0) same[k] = c;
    }
  }
  for (int k = 0; k < m; ++k) {
    const PagedAt at(a, b0 + k, h, L, 1, 0, L + 1);
    paged_store(a, at, 1);
  }
  // the queries, [sequence] where k_paged_split has [row]
  for (int x = tid; x < U * 64; x += 64 * WAVES) {
    const int r = x & 15, e = 4 * (x >> 6) + (x & 63) / 16;
    double2 q = make_double2(0.0, 0.0);
    if (r < m && e < dh) q = a.q[(long)(b0 + r) * a.n * a.ldq + (long)h * dh + e];
    qs[x] = make_double2(q.x * a.scale, -q.y * a.scale);
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0, done = 0;
    const auto add = [&](int from, int to, int sequence, unsigned columns) {
      if (to <= from) return;
      runs.at[n++] = make_int4(done, done + to - from, from, sequence | (int)(columns << 8));
      done += to - from;
    };
    for (int k = 0, end; k < m; k = end) {
      int pages = INT32_MAX;
      for (end = k + 1; end < m && same[end] > 0; ++end) pages = min(pages, same[end]);
      const int shared = end > k + 1 ? pages * (a.page_rows / PAGE_TILE) : 0;
      add(0, shared, k, ((1u << (end - k)) - 1) << k);
      for (int i = k; i < end; ++i) add(shared, tiles, i, 1u << i);
    }
    runs.n = n;
  }
  __syncthreads();
  const int all = __builtin_amdgcn_readfirstlane(runs.at[runs.n - 1].y);

  // tile v of the bunch; v grows from call to call
  struct Place {
    PagedTile tile;
    const double2 *kn, *vn;
    unsigned columns;
    __device__ __forceinline__ const double2* key(const PagedAttn& a, int r, int L) const {
      return tile.t + r >= L ? kn : a.kp + tile.in + (uint32_t)r * (uint32_t)a.dh;
    }
    __device__ __forceinline__ const double2* value(const PagedAttn& a, int r, int L) const {
      return tile.t + r >= L ? vn : a.vp + tile.in + (uint32_t)r * (uint32_t)a.dh;
    }
  };
  int run_at = 0;
  const auto place = [&](int v) {
    int4 r = runs.at[run_at];
    while (v >= __builtin_amdgcn_readfirstlane(r.y)) r = runs.at[++run_at];
    const int w = __builtin_amdgcn_readfirstlane(r.w), t = 16 * (v - __builtin_amdgcn_readfirstlane(r.x) + __builtin_amdgcn_readfirstlane(r.z));
    const PagedAt at(a, b0 + (w & 15), h, L, 1, 0, L + 1);
    uint32_t id;
    const int pg = at.page(a, t, id);
    Place x;
    x.tile = PagedTile(a, at, t, pg, id);
    x.kn = at.kn + (long)L * a.new_row;
    x.vn = at.vn + (long)L * a.new_row;
    x.columns = (unsigned)w >> 8;
    return x;
  };
  double2 kf[U], vf[4][CT];
  double bf[4] = {0.0, 0.0, 0.0, 0.0};
  const auto load_keys = [&](const Place& x) {
    const double2* k = x.key(a, min(row, L - x.tile.t), L);
#pragma unroll
    for (int u = 0; u < U; ++u) kf[u] = FULL || 4 * u + kq < dh ? ld_glb(k + 4 * u + kq) : make_double2(0.0, 0.0);
    if (a.bias) {
      const double* bias = a.bias + (long)h * a.bias_stride + (long)L * a.bias_row;
#pragma unroll
      for (int e = 0; e < 4; ++e) bf[e] = ld_glb(bias + min(x.tile.t + 4 * e + kq, L));
    }
  };
  const auto load_values = [&](const Place& x) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const double2* v = x.value(a, min(4 * q + kq, L - x.tile.t), L);
#pragma unroll
      for (int c = 0; c < CT; ++c) vf[q][c] = ld_glb(v + (FULL ? row + 16 * c : min(row + 16 * c, dh - 1)));
    }
  };
  AttnRun<DHP> run;
  int v = wave;
  Place now, ahead;
  if (v < all) {
    now = place(v);
    load_keys(now);
    load_values(now);
    ahead = place(min(v + WAVES, all - 1));
  }
  const double2* qw = qs + lane;
  for (; v < all; v += WAVES) {
    v4d s = {0.0, 0.0, 0.0, 0.0}, z = s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const double2 k = kf[u], q = qw[u * 64];
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(k.x, q.x, s, 0, 0, 0);
      z = __builtin_amdgcn_mfma_f64_16x16x4f64(k.y, q.y, z, 0, 0, 0);
      if (u % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // so many operands at a time in registers
    }
    const bool column = now.columns >> row & 1;
    const int t = now.tile.t;
    unsigned vis = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool see = column && t + 4 * e + kq <= L;
      vis |= (unsigned)see << e;
      s[e] = see ? s[e] + z[e] + bf[e] : -INFINITY;
    }
    const bool more = v + WAVES < all;
    if (more) load_keys(ahead);
    run.soften(s);
    bool fine = true;  // 0 times what is not finite is NaN in the other columns
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < CT; ++c) fine &= attn_finite(vf[q][c]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < CT; ++c) run.output(s, q, c, vf[q][c]);
    if (more) load_values(ahead);
    if (__ballot(!fine)) run.add_left_out([&](int k) { return now.value(a, k, L); }, dh, L + 1 - t, s, vis);
    now = ahead;
    if (more) ahead = place(min(v + 2 * WAVES, all - 1));
  }
  // the waves, rescaled to their common maximum and added in order
  run.l = xor32_sum(xor16_sum(run.l));
  if (kq == 0) sm[wave][row] = run.m, sl[wave][row] = run.l;
  __syncthreads();  // and the queries' last read
  double M = -INFINITY, sum = 0.0;
#pragma unroll
  for (int g = 0; g < WAVES; ++g) M = fmax(M, sm[g][row]);
  const double base = M == -INFINITY ? 0.0 : M, f = exp(run.m - base);
#pragma unroll
  for (int g = 0; g < WAVES; ++g) sum += sl[g][row] * exp(sm[g][row] - base);
  if (row < m)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        os[(wave * 16 + row) * OSTR + 16 * c + 4 * e + kq] = make_double2(run.o_re[c][e] * f, run.o_im[c][e] * f);
  if (wave == 0 && kq == 0) sums[row] = sum;
  __syncthreads();
  for (int x = tid; x < m * dh; x += 64 * WAVES) {
    const int r = x / dh, e = x - r * dh;
    double2 o = os[r * OSTR + e];
#pragma unroll
    for (int g = 1; g < WAVES; ++g) o = cadd(o, os[(g * 16 + r) * OSTR + e]);
    a.out[(long)(b0 + r) * a.n * a.ldo + (long)h * dh + e] = make_double2(o.x / sums[r], o.y / sums[r]);
  }
}

// One block per (piece, head).
template <int DHP, int NG, bool FULL>
__global__ __launch_bounds__(256, DHP <= 128 ? 2 : 1) void k_paged_split(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
  __shared__ __align__(16) unsigned char lds[split_lds<DHP>(NG)];
  __shared__ PagedSums sh;
  const int piece = blockIdx.x / a.H;
  const PagedAt at(a, p, own, piece, blockIdx.x - piece * a.H);
  paged_store(a, at, p.rows);
  if (at.n0 < at.cnt) paged_split<DHP, NG, FULL>(a, p, ws, at, lds, sh);
}

// One block per (range of pieces, head).
template <int DHP, bool FULL>
__global__ __launch_bounds__(256, DHP <= 64 ? 2 : 1) void k_paged_tile(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
  __shared__ __align__(16) unsigned char lds[tile_lds<DHP>()];
  __shared__ PagedSums sh;
  const int range = blockIdx.x / a.H, head = blockIdx.x - range * a.H;
  const int end = op_int(a.tab, own, p.ranges, range + 1);
  for (int piece = op_int(a.tab, own, p.ranges, range); piece < end; ++piece) {
    const PagedAt at(a, p, own, piece, head);
    paged_store(a, at, p.rows);
    if (at.n0 >= at.cnt) continue;
    paged_tile<DHP, FULL>(a, p, ws, at, lds, sh);
    __syncthreads();  // LDS is the next piece's
  }
}

// Joins the partials of the rows whose group was cut.  Bound by their bytes: 504 blocks'
// pieces of up to 64 rows 14 to 18 us; one token 4 us, the launch.
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan p, PagedWs ws, OpTable own) {
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
  const int cnt = op_int(a.tab, own, a.count, b);
  const int2* cuts = op_array<int2>(a.tab, own, p.cuts) + (long)b * p.groups;
  for (long x = (long)blockIdx.y * 256 + threadIdx.x; x < (long)cnt * a.dh; x += (long)gridDim.y * 256) {
    const int i = (int)(x / a.dh), e = (int)(x - (long)i * a.dh);
    const int g = i / p.rows, ns = cuts[g].y, rows = min(p.rows, a.n);
    if (ns == 1) continue;
    const long at = (long)h * p.part_rows + cuts[g].x + i - g * p.rows;
    // four parts at a time, all their loads at once
    double M = -INFINITY, l = 0.0;
    double2 v = make_double2(0.0, 0.0);
    for (int s0 = 0; s0 < ns; s0 += 4) {
      double m[4], ls[4];
      double2 o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long x = at + (long)min(s0 + k, ns - 1) * rows;
        m[k] = s0 + k < ns ? ws.m[x] : -INFINITY;
        ls[k] = ws.l[x];
        o[k] = ws.o[x * a.dh + e];
      }
      const double top = fmax(fmax(fmax(m[0], m[1]), fmax(m[2], m[3])), M), base = top == -INFINITY ? 0.0 : top;
      const double keep = exp(M - base);
      M = top;
      l *= keep;
      v = make_double2(v.x * keep, v.y * keep);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (s0 + k >= ns) break;
        const double f = exp(m[k] - base);
        l += ls[k] * f;
        v = make_double2(v.x + o[k].x * f, v.y + o[k].y * f);
      }
    }
    a.out[((long)b * a.n + i) * a.ldo + (long)h * a.dh + e] = make_double2(v.x / l, v.y / l);
  }
}

// A step is what a block's four waves take at a time, 64 MFMAs each at head dim 64.
// Up to 32 rows a piece is a block, and all have at most so many steps: of the least
// estimated time.  A block's step takes 2.3 us of a SIMD at head dim 64 (64 MFMAs and
// the softmax), half as much again alone, or its bytes' time at 5.2 TB/s where every
// place of the chip is busy; 8 us go to a block's start and end, and the partials
// pass through memory twice.  Other widths go by the same figures in proportion.
// With more rows a block takes as many steps as any other, of as many groups as that
// needs: up to 700 rows of three sequences behind 555 to 1024 slots, 12 heads, take 352 us
// a call in blocks of 14 steps at most, 291 in 504 blocks of equal steps (inputs changing
// from call to call).
PagedPlan paged_plan(const PagedAttn& a, const int* kv_len, const int* count, std::vector<int>& lists) {
  PagedPlan p;
  p.ng = a.n <= 16 || a.dh > 128 ? 1 : a.n <= 32 ? 2 : 4;
  p.rows = 16 * p.ng;
  p.groups = (a.n + p.rows - 1) / p.rows;
  const int unit = 64 / p.ng;  // slots of a step
  const bool even = p.ng == 4;
  struct Group {
    int b, n0, len, steps;  // slots that its rows see (0 without rows), at most 2^26 steps
  };
  std::vector<Group> groups;
  long steps = 0;
  int longest = 1;
  for (int b = 0; b < a.B; ++b)
    for (int g = 0; g < p.groups; ++g) {
      const int n0 = g * p.rows, rows = std::min(p.rows, count[b] - n0), len = rows > 0 ? kv_len[b] + n0 + rows : 0;
      groups.push_back({b, n0, len, std::max(1, (len + unit - 1) / unit)});
      steps += groups.back().steps;
      longest = std::max(longest, groups.back().steps);
    }
  // One row of many sequences: neighbours of equal length may be beams that share
  // pages, which are then read once.  In bunches where that leaves a block for
  // three of four CUs: 16 prompts of 16 beams, 12 heads, take 324 us a call so in 192
  // blocks, 375 in 384 of 11 and 5 sequences.  Sequences of one length that share nothing
  // lose nothing by it there (64 of 480 slots, 12 heads: 171 us, 173 in 264 blocks).
  // A bunch is one block however long it is, and what it shares is not known here: one
  // that holds 1.9 times a CU's even share of all rows or more is cut into smaller ones,
  // and where pairs are too long yet, no bunch is formed.  us a call, 12 heads, with
  // 90% / 50% / none of the slots shared: 16 of 2000 slots beside 42 pairs of 100 to 141
  // 172 / 194 / 234 so (pieces by slots), 173 / 253 / 335 in pairs (2.0 even shares), 423 /
  // 1181 / 2108 in one bunch; 16 prompts of 16 beams, 100 to 500 slots (1.8), 138 / 313 /
  // 521 whole, 172 / 351 / 571 in bunches of 13 and 3.
  if (a.n == 1 && a.dh <= 64 && std::all_of(count, count + a.B, [](int c) { return c == 1; }))
    for (int most = 16; most > 1 && !p.beams; --most) {
      std::vector<int4> bunches;
      for (int b = 0, end; b < a.B; b = end) {
        for (end = b + 1; end < a.B && end < b + most && kv_len[end] == kv_len[b]; ++end) {}
        bunches.push_back(make_int4(b, end - b, 0, 0));
      }
      if (3 * bunches.size() > 2 * (size_t)a.B) break;
      if (bunches.size() * a.H < 192) continue;
      long longest = 0, all = 0;  // tiles
      for (const int4& x : bunches) {
        const long tiles = (long)x.y * (kv_len[x.x] / PAGE_TILE + 1);
        longest = std::max(longest, tiles);
        all += tiles;
      }
      if (longest * 256 > 1.9 * all * a.H) continue;
      std::stable_sort(bunches.begin(), bunches.end(),
                       [&](const int4& x, const int4& y) { return (long)x.y * kv_len[x.x] > (long)y.y * kv_len[y.x]; });
      p.beams = true;
      p.blocks = (int)bunches.size();
      lists.resize((lists.size() + 3) & ~(size_t)3);
      p.pieces = (uint32_t)(lists.size() * sizeof(int));
      for (const int4& x : bunches) lists.insert(lists.end(), {x.x, x.y, 0, 0});
    }
  if (p.beams) return p;
  const double places = a.dh <= 64 || (a.dh <= 128 && p.ng < 4) ? 512.0 : 256.0;  // blocks the chip holds at once
  int each = 1;  // steps of a piece
  if (!even && (double)steps * a.H > places) {
    const double tile_us = 0.7 + 1.6 * a.dh / 64, step_mb_us = unit * a.dh * 32 / 5.2e6 / p.groups;
    double least = 1e300;
    int last = 0;
    for (int k : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32}) {
      const int c = (longest + k - 1) / k;
      if (c == last) continue;
      last = c;
      double blocks = 0.0;
      for (const Group& g : groups) blocks += (g.steps + c - 1) / c;
      const bool cut = blocks > (double)groups.size();
      blocks *= a.H;
      const double full = std::floor(blocks / places), rest = blocks - full * places;
      const double work = (double)steps * a.H / blocks;  // steps of a block, on average
      double cost = full * (3.0 + work * std::max(2.0 * tile_us * places / 512.0, places * step_mb_us));
      if (rest > 0.0) cost += 8.0 + std::max(c * tile_us * (rest > 256.0 ? 2.0 : 1.45), rest * work * step_mb_us);
      if (cut) cost += blocks * 16 * std::min(p.rows, a.n) * a.dh * 2 / 5.2e6;
      if (cost < least) least = cost, each = c;
    }
  }
  const long ranges = std::min<long>(steps, std::max<long>(1, (long)places / a.H));
  // pieces of one group a block where that costs no more than the two steps that another piece does
  bool own_block = !even;
  if (even) {
    long c = (steps + ranges - 1) / ranges;  // past 32 bits where many groups have long caches
    const long bar = c + 2;
    const auto blocks = [&] {
      long n = 0;
      for (const Group& g : groups) n += (g.steps + c - 1) / c;
      return n;
    };
    while (c < bar && blocks() > ranges) ++c;
    own_block = blocks() <= ranges;
    if (own_block) each = (int)c;
    else each = INT32_MAX;
  }
  const auto cut = [&](auto&& piece) {
    long done = 0, range = 0;
    for (size_t g = 0; g < groups.size(); ++g) {
      const int n = own_block ? (groups[g].steps + each - 1) / each : 1, same = (groups[g].steps + n - 1) / n;
      for (int from = 0; from < groups[g].steps;) {
        int take = std::min(same, groups[g].steps - from);
        if (!own_block) {
          while (steps * (range + 1) / ranges <= done) ++range;
          take = (int)std::min<long>(groups[g].steps - from, steps * (range + 1) / ranges - done);
        }
        piece(g, range, from, take);
        if (own_block) ++range;
        from += take;
        done += take;
      }
    }
  };
  std::vector<int> of(groups.size(), 0), next(groups.size(), 0), cuts, ends = {0}, places_of;
  std::vector<int4> pieces;
  cut([&](size_t g, long, int, int) { ++of[g]; });
  for (size_t g = 0; g < groups.size(); ++g) {
    cuts.insert(cuts.end(), {p.part_rows, of[g]});
    if (of[g] > 1) p.part_rows += of[g] * std::min(p.rows, a.n);
  }
  cut([&](size_t g, long range, int from, int take) {
    const Group& x = groups[g];
    while ((long)ends.size() <= range) ends.push_back((int)pieces.size());
    pieces.push_back(make_int4(x.b, x.n0, from * unit, std::min(x.len, (from + take) * unit)));
    places_of.push_back(of[g] > 1 ? cuts[2 * g] + next[g]++ * std::min(p.rows, a.n) : -1);
  });
  ends.push_back((int)pieces.size());
  p.blocks = even ? (int)ends.size() - 1 : (int)pieces.size();
  if (!even) {  // the longest first
    std::vector<int> order(pieces.size());
    for (size_t k = 0; k < order.size(); ++k) order[k] = (int)k;
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return pieces[x].w - pieces[x].z > pieces[y].w - pieces[y].z; });
    const std::vector<int4> was = pieces;
    const std::vector<int> at = places_of;
    for (size_t k = 0; k < order.size(); ++k) pieces[k] = was[order[k]], places_of[k] = at[order[k]];
  }
  const auto put = [&](const int* v, size_t n) {
    lists.resize((lists.size() + 3) & ~(size_t)3);
    const uint32_t at = (uint32_t)(lists.size() * sizeof(int));
    lists.insert(lists.end(), v, v + n);
    return at;
  };
  p.pieces = put((const int*)pieces.data(), 4 * pieces.size());
  p.places = put(places_of.data(), places_of.size());
  if (even) p.ranges = put(ends.data(), ends.size());
  if (p.part_rows) p.cuts = put(cuts.data(), cuts.size());
  return p;
}

static size_t paged_layout(const PagedAttn& a, const PagedPlan& p, char* base, PagedWs& ws) {
  if (!p.part_rows) return 0;
  const size_t rows = (size_t)a.H * p.part_rows;
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
  const dim3 grid((unsigned)((long)p.blocks * a.H));
  const auto go = [&](auto kern) { MITOK_LAUNCH(kern, grid, dim3(256), 0, st, a, p, ws, own); };
  if constexpr (DHP <= 64)
    if (p.beams) {
      const auto bunches = [&](auto kern, int waves) { MITOK_LAUNCH(kern, grid, dim3(64 * waves), 0, st, a, p, own); };
      return grid.x <= 256 ? bunches(k_paged_beams<DHP, FULL, 8>, 8) : bunches(k_paged_beams<DHP, FULL, 4>, 4);
    }
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
  if (p.part_rows) {
    const unsigned parts = (unsigned)std::min<long>(((long)a.n * a.dh + 255) / 256, 4096);
    hipLaunchKernelGGL(k_paged_join, dim3((unsigned)(a.B * a.H), parts), dim3(256), 0, st, a, p, ws, own);
  }
}

}  // namespace mitok

// beams.hip — beams on a paged cache: sequences that take other sequences' pages
// (ForkPages in paged.hpp), and the best continuations of a group of beams
// (BeamSelect).
#include <algorithm>

#include "paged.hpp"
#include "rank_bins.hpp"

namespace mitok {

// ===========================================================================
// forks
// ===========================================================================
// held [3][pages]: a page's holders among the new sequences, how many of them
// write behind their rows in it, and n minus the first of these.  The plan's
// second kernel reads them and leaves zeros.
size_t fork_held_words(uint32_t pages) { return 3 * (size_t)pages; }

struct ForkWs {
  uint32_t* table;  // [n][max_pages] the parents' pages
  uint32_t* len;    // [n] rows
  uint32_t* room;   // [n] rows to grow
  uint32_t* start;  // [n] first free page taken, among the list
  uint32_t* copy;   // [n] 1: the last page is copied
  uint32_t* free;   // [pages] free pages, as many as are taken
};
static size_t fork_layout(uint32_t n, uint32_t max_pages, uint32_t pages, char* base, ForkWs& w) {
  size_t at = 0;
  const auto take = [&](size_t words) {
    char* q = base ? base + at : nullptr;
    at += (words * sizeof(uint32_t) + 255) & ~(size_t)255;
    return (uint32_t*)q;
  };
  w.len = take(n);
  w.room = take(n);
  w.start = take(n);
  w.copy = take(n);
  w.free = take(pages);
  w.table = take((size_t)n * max_pages);
  return at;
}
size_t fork_ws_bytes(uint32_t n, uint32_t max_pages, uint32_t pages) {
  ForkWs w;
  return fork_layout(n, max_pages, pages, nullptr, w);
}

// A new sequence's parent, its rows and its room; one that is refused holds nothing.
struct ForkOne {
  uint32_t p, len = 0, room = 0;
  __device__ __forceinline__ ForkOne(const ForkPages& f, uint32_t i) {
    p = f.parents ? f.parents[i] : i;
    if (p == NO_ROW) return;
    if (p >= f.old) {
      refuse(f, PE_BAD_PARENT);
      return;
    }
    len = f.lens[p];
    room = f.grow ? f.grow[i] : f.grow_all;
    if ((uint64_t)len + room > (uint64_t)f.max_pages * f.page_rows) refuse(f, PE_BAD_LENGTH);
  }
  __device__ __forceinline__ void refuse(const ForkPages& f, int word) {
    len = room = 0;
    set_word(f.err, word);
    *f.refused = f.call;  // the same value, whoever writes it
  }
};
// its page j, and what that does to the page's counts
__device__ __forceinline__ void fork_hold(const ForkPages& f, const ForkWs& w, uint32_t i, uint32_t p, uint32_t j, uint32_t had,
                                          bool writes) {
  const uint32_t id = f.table[(size_t)p * f.max_pages + j];
  w.table[(size_t)i * f.max_pages + j] = id;
  if (id >= f.pages) {
    set_word(f.err, PE_BAD_PAGE);
    *f.refused = f.call;
    return;
  }
  atomicAdd(f.held + id, 1u);
  if (writes && j + 1 == had) {
    atomicAdd(f.held + f.pages + id, 1u);
    atomicMax(f.held + 2 * (size_t)f.pages + id, f.n - i);
  }
}

// One block per new sequence.
__global__ __launch_bounds__(256) void k_fork_take(ForkPages f, ForkWs w) {
  const uint32_t i = blockIdx.x, tid = threadIdx.x;
  const ForkOne x(f, i);
  const uint32_t had = (x.len + f.page_rows - 1) / f.page_rows;
  for (uint32_t j = tid; j < had; j += 256) fork_hold(f, w, i, x.p, j, had, x.room > 0 && x.len % f.page_rows);
  if (tid == 0) {
    w.len[i] = x.len;
    w.room[i] = x.room;
  }
}

// what comes before this thread's number in the block's order, and the block's sum
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* part, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) part[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
  for (int k = 0; k < 16; ++k) {
    if (k < wave) before += part[k];
    all += part[k];
  }
  __syncthreads();
  return before + x - v;
}

// One block: which last pages are copied, where each sequence's share of the free
// pages starts, and the list of these.  Leaves the counts at zero.
// SMALL: what k_fork_take does, too.
constexpr uint32_t FORK_SMALL = 1024;  // table entries, one of a thread
template <bool SMALL>
__global__ __launch_bounds__(1024) void k_fork_assign(ForkPages f, ForkWs w) {
  __shared__ uint32_t part[16];
  const uint32_t tid = threadIdx.x;
  if constexpr (SMALL) {
    __shared__ uint32_t from[1024], lens[1024], rooms[1024];
    if (tid < f.n) {
      const ForkOne x(f, tid);
      from[tid] = x.p;
      w.len[tid] = lens[tid] = x.len;
      w.room[tid] = rooms[tid] = x.room;
    }
    __syncthreads();
    for (uint32_t x = tid; x < f.n * f.max_pages; x += 1024) {
      const uint32_t i = x / f.max_pages, j = x - i * f.max_pages, had = (lens[i] + f.page_rows - 1) / f.page_rows;
      if (j < had) fork_hold(f, w, i, from[i], j, had, rooms[i] > 0 && lens[i] % f.page_rows);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the counts are there before any wave reads them
    __syncthreads();
  }
  uint32_t total = 0, all;
  for (uint32_t i0 = 0; i0 < f.n; i0 += 1024) {
    const uint32_t i = i0 + tid;
    uint32_t copy = 0, need = 0;
    if (i < f.n) {
      const uint32_t len = w.len[i], room = w.room[i];
      const uint32_t had = (len + f.page_rows - 1) / f.page_rows;
      need = (len + room + f.page_rows - 1) / f.page_rows - had;
      if (room > 0 && len % f.page_rows) {
        const uint32_t id = w.table[(size_t)i * f.max_pages + had - 1];
        if (id < f.pages) {
          const bool all_write = ld_dev(f.held + f.pages + id) == ld_dev(f.held + id), first = ld_dev(f.held + 2 * (size_t)f.pages + id) == f.n - i;
          copy = !(all_write && first);
        }
      }
    }
    const uint32_t before = block_before(copy + need, part, all);
    if (i < f.n) {
      w.start[i] = total + before;
      w.copy[i] = copy;
    }
    total += all;
  }
  uint32_t found = 0;
  for (uint32_t p0 = 0; p0 < f.pages; p0 += 1024) {
    const uint32_t id = p0 + tid;
    const bool is_free = id < f.pages && ld_dev(f.held + id) == 0;
    if (id < f.pages) f.held[id] = f.held[f.pages + id] = f.held[2 * (size_t)f.pages + id] = 0;
    if (found < total) {
      const uint32_t at = found + block_before(is_free ? 1u : 0u, part, all);
      if (is_free && at < total) w.free[at] = id;
      found += all;
    }
  }
  if (tid == 0 && found < total) {
    set_word(f.err, PE_NO_PAGES);
    *f.refused = f.call;
  }
}

// y 0: the new tables and lengths; others, of one layer's keys or values: the
// used rows of a copied page, head by head (a head's rows are contiguous).  Bound by
// HBM: 12 layers of 12 heads of 64 and pages of 32 rows, 64 sequences, 41 us at about 6
// TB/s, read and written.
constexpr int FC_PER = 4;
__global__ __launch_bounds__(256) void k_fork_commit(ForkPages f, ForkWs w, PagePool pool, int parts, int commit) {
  if (*f.refused == f.call) return;
  const uint32_t i = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x;
  const uint32_t len = w.len[i], copy = w.copy[i], start = w.start[i];
  const uint32_t had = (len + f.page_rows - 1) / f.page_rows;
  if (commit && blockIdx.y == 0) {
    if (part) return;
    const uint32_t then = (len + w.room[i] + f.page_rows - 1) / f.page_rows;
    for (uint32_t j = tid; j < f.max_pages; j += 256) {
      uint32_t id = NO_PAGE;
      if (j < had) id = copy && j + 1 == had ? w.free[start] : w.table[(size_t)i * f.max_pages + j];
      else if (j < then) id = w.free[start + copy + j - had];
      f.table_out[(size_t)i * f.max_pages + j] = id;
    }
    if (tid == 0) f.lens_out[i] = len;
    return;
  }
  if (!copy) return;
  const int y = blockIdx.y - commit, layer = y >> 1, dh = pool.dh;
  const size_t page = (size_t)pool.H * f.page_rows * dh;
  double2* x = (y & 1 ? pool.v : pool.k) + (size_t)layer * f.pages * page;
  const double2* src = x + (size_t)w.table[(size_t)i * f.max_pages + had - 1] * page;
  double2* dst = x + (size_t)w.free[start] * page;
  const uint32_t each = (len % f.page_rows) * dh, all = each * pool.H, skip = f.page_rows * dh - each;
  for (uint32_t e = part * 256 + tid; e < all; e += parts * 256) {
    const size_t at = e + (size_t)(e / each) * skip;
    dst[at] = src[at];
  }
}

static ForkWs fork_ws(const ForkPages& f) {
  ForkWs w;
  fork_layout(f.n, f.max_pages, f.pages, (char*)f.ws, w);
  return w;
}

void fork_plan(hipStream_t st, const ForkPages& f) {
  const ForkWs w = fork_ws(f);
  // us a call, one block / two launches: 4 sequences with 32 entries each 22.9 / 24.4, 128 37.3 / 36.0
  if ((uint64_t)f.n * f.max_pages <= FORK_SMALL) {
    hipLaunchKernelGGL(k_fork_assign<true>, dim3(1), dim3(1024), 0, st, f, w);
    return;
  }
  hipLaunchKernelGGL(k_fork_take, dim3(f.n), dim3(256), 0, st, f, w);
  hipLaunchKernelGGL(k_fork_assign<false>, dim3(1), dim3(1024), 0, st, f, w);
}

void fork_copy(hipStream_t st, const ForkPages& f, const PagePool& pool, bool commit) {
  const ForkWs w = fork_ws(f);
  const size_t most = (size_t)pool.H * (f.page_rows - 1) * pool.dh;  // elements of a copy
  const int parts = (int)std::clamp<size_t>((most + 256 * FC_PER - 1) / (256 * FC_PER), 1, 32);
  hipLaunchKernelGGL(k_fork_commit, dim3(f.n * parts, 2 * pool.layers + (commit ? 1 : 0)), dim3(256), 0, st, f, w, pool, parts,
                     commit ? 1 : 0);
}

// ===========================================================================
// selection
// ===========================================================================
// A row is cut into pieces, a wave each: the sum of its exponentials, and the maximum
// of each quarter, the share of 16 lanes.  Of the K best quarters by their maxima each
// holds a continuation at least as good as the least of those maxima, so no
// continuation below that bound is among the K best: the logits are read once, and of
// them again only the quarters whose maximum reaches the bound.
struct BeamWs {
  double* m;  // [rows][pieces][4]
  double* s;  // [rows][pieces] of e^(x - the largest of the four)
};
// Logits of a piece: 512, or 256 where that leaves most of the chip idle.
static int beam_piece(const BeamSelect& b) { return (long)b.groups * b.beams * ((b.V + 511) / 512) >= 2048 ? 512 : 256; }
static size_t beam_layout(const BeamSelect& b, char* base, BeamWs& w) {
  const size_t n = (size_t)b.groups * b.beams * ((b.V + 255) / 256);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  w.m = (double*)take(4 * n * sizeof(double));
  w.s = (double*)take(n * sizeof(double));
  return at;
}
size_t beam_ws_bytes(const BeamSelect& b) {
  BeamWs w;
  return beam_layout(b, nullptr, w);
}

// two logits of a row, whose start is aligned to one
typedef double v2logit __attribute__((ext_vector_type(2), aligned(8)));

// a row without logits to read: ended, or of score -inf
__device__ __forceinline__ bool beam_idle(const BeamSelect& b, long row) {
  return b.scores[row] == -INFINITY || (b.done && b.done[row]);
}

// The quarter at t0 of a row: a lane of 16 takes logits t0 + 32 k + 2 (lane % 16) and the one
// behind, -inf past the row.  No branch between the loads, so that whoever waits for
// them waits for them alone.
__device__ __forceinline__ int beam_token(int t0, int k) { return t0 + 32 * k + 2 * (threadIdx.x & 15); }
template <int PER>
__device__ __forceinline__ void beam_load(const double* row, int V, int t0, v2logit (&v)[PER]) {
  if (V < 2) {
    for (int k = 0; k < PER; ++k) v[k] = v2logit{beam_token(t0, k) == 0 ? row[0] : -INFINITY, -INFINITY};
    return;
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = *(const MITOK_GLOBAL v2logit*)(row + min(beam_token(t0, k), V - 2));
}
template <int PER>
__device__ __forceinline__ void beam_cut(int V, int t0, v2logit (&v)[PER]) {
  if (V < 2) return;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int t = beam_token(t0, k);
    if (t + 1 >= V) v[k] = v2logit{t < V ? v[k].y : -INFINITY, -INFINITY};  // the last two were read
  }
}

// e^x for x <= 0 within a unit in the last place: x = k ln 2 + r, |r| <= ln 2 / 2 (ln 2
// as a double and the rest of it), then Taylor's polynomial of degree 13 in r, whose
// remainder r^14 / 14! is below 5e-18.  18 double operations: the range checks of the
// library's exp cost a third more.
__device__ __forceinline__ double exp_below(double x) {
  x = fmax(x, -1100.0);  // e^-1100 is 0
  const double k = rint(x * 0x1.71547652b82fep+0);
  const double r = fma(-k, 0x1.abc9e3b39803fp-56, fma(-k, 0x1.62e42fefa39efp-1, x));
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)k);
}

// Bound by the bytes and, beside them, by 20 double operations a logit: 192 rows of
// 50280, 67 MB of live rows in 15.9 us (4.2 TB/s), where a read with the maxima alone
// takes 12.  Waves that walk several pieces, the next one's loads in flight, took 22.
template <int PER>
__global__ __launch_bounds__(256) void k_beam_pieces(BeamSelect b, BeamWs w, int pieces, uint32_t blocks) {
  const int lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x / blocks;
  const int piece = (int)(blockIdx.x - row * blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (piece >= pieces || beam_idle(b, row)) return;
  const int t0 = piece * 128 * PER + (lane >> 4) * 32 * PER;
  v2logit v[PER];
  beam_load(b.x + (long)row * b.V, b.V, t0, v);
  beam_cut(b.V, t0, v);
  double m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    bad |= !(v[k].x < INFINITY) || !(v[k].y < INFINITY);  // NaN, or an infinity that leaves no distribution
    m = fmax(m, fmax(v[k].x, v[k].y));
  }
  if (__ballot(bad) && lane == 0) set_word(b.err, PE_BAD_SCORE);
  m = row16_max(m);
  const long at = (long)row * pieces + piece;
  if ((lane & 15) == 0) w.m[4 * at + (lane >> 4)] = m;
  double x, y;
  pair16_f64(m, x, y);
  pair32_f64(fmax(x, y), x, y);
  m = fmax(x, y);
  double s = 0.0;
  if (m > -INFINITY) {
#pragma unroll
    for (int k = 0; k < PER; ++k) s += exp_below(v[k].x - m) + exp_below(v[k].y - m);
  }
  s = wave_sum(s);
  if (lane == 0) w.s[at] = s;
}

// the order of continuations: rank, then the lower row, the larger logit, the lower token
struct Cont {
  double rank, x;
  int row, t;
};
__device__ __forceinline__ bool before(const Cont& a, const Cont& b) {  // without branches
  const bool later = (a.x > b.x) | ((a.x == b.x) & (a.t < b.t));
  const bool tied = (a.row < b.row) | ((a.row == b.row) & later);
  return (a.rank > b.rank) | ((a.rank == b.rank) & tied);
}
// the first of a wave's continuations (each lane's own), in every lane
__device__ __forceinline__ void wave_first(Cont& c) {
  for (int d = 32; d; d >>= 1) {
    Cont o;
    o.rank = __shfl_xor(c.rank, d);
    o.x = __shfl_xor(c.x, d);
    o.row = __shfl_xor(c.row, d);
    o.t = __shfl_xor(c.t, d);
    if (before(o, c)) c = o;
  }
}

// sum of a row of 16 lanes
__device__ __forceinline__ int row16_sumi(int v) {
  v += dpp_i32<DPP_XOR1>(v);
  v += dpp_i32<DPP_XOR2>(v);
  v += dpp_i32<DPP_HALF_MIRROR>(v);
  return v + dpp_i32<DPP_MIRROR>(v);
}

// One block per group.  A histogram of the quarters' maxima gives a bound that K of
// them reach; the continuations that reach it are listed, and a continuation's
// place is how many of the list come before it.  Where the list is too long (few
// quarters, or logits close together), a histogram of what reached the bound gives
// a closer one; where that cannot part them (equal ranks), K rounds over the
// quarters find one continuation each.  A finite mask over whole quarters opens the
// first range so far that one bin has all live ones: 83 us a call instead of 32 for
// 32 x 4 rows of 32000 with a sixth allowed.  Bound by that chain's latency, a memory round
// trip or a few barriers a link: 7.4 us for 4 rows of 4096, 12 for 12 rows of 50280 and
// 24 kept (K rounds of a block-wide maximum took 120).
constexpr int BS_LIST = 512, BS_PARTS = 4096, BS_WAVES = 16;
constexpr int BS_GROUPS = 1 << 21;  // of a launch, which has fewer than 2^32 threads
constexpr int BS_HELD = 5;  // of a thread's quarters, maxima that wait in registers (5120: 12 rows of 50280 logits); later ones are read anew
template <int PER>
__global__ __launch_bounds__(1024) void k_beam_pick(BeamSelect b, BeamWs w, int pieces, int first) {
  __shared__ double lse[1024], had[1024], scale[1024];  // of the group's rows; lse NaN: ended
  __shared__ Cont part[BS_WAVES], list[BS_LIST];
  __shared__ int plist[BS_PARTS];
  __shared__ __align__(16) int bins[BB_BINS];  // read by fours
  __shared__ double lows[BS_WAVES], highs[BS_WAVES];
  __shared__ int sums[BS_WAVES], nparts, listed;
  const int g = first + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = b.beams, K = b.keep;
  const int parts = 4 * pieces, E = R * parts;  // quarters of a row, of the group
  const long row0 = (long)g * R;
  // what the rows need, requested at once; an idle row's has no meaning and is left out
  double held[BS_HELD];
#pragma unroll
  for (int k = 0; k < BS_HELD; ++k) held[k] = tid + 1024 * k < E ? w.m[row0 * parts + tid + 1024 * k] : -INFINITY;
  for (int r = wave; r < R; r += BS_WAVES) {
    const long row = row0 + r;
    const double score = b.scores[row], f = b.scale ? b.scale[row] : 1.0;
    const bool ended = b.done && b.done[row];
    const auto largest = [&](int c) {
      const double* q = w.m + 4 * (row * pieces + c);
      return fmax(fmax(q[0], q[1]), fmax(q[2], q[3]));
    };
    double mc[2], sc[2], m = -INFINITY, s = 0.0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = lane + 64 * k;
      mc[k] = c < pieces ? largest(c) : -INFINITY;
      sc[k] = c < pieces ? w.s[row * pieces + c] : 0.0;
    }
    if (score > -INFINITY && !ended) {
      m = fmax(mc[0], mc[1]);
      for (int c = lane + 128; c < pieces; c += 64) m = fmax(m, largest(c));
      m = wave_max(m);
      if (m > -INFINITY) {
        s = sc[0] * exp_below(mc[0] - m) + sc[1] * exp_below(mc[1] - m);
        for (int c = lane + 128; c < pieces; c += 64) s += w.s[row * pieces + c] * exp_below(largest(c) - m);
        s = wave_sum(s);
      }
    }
    if (lane == 0) {
      if (isnan(score) || score == INFINITY) set_word(b.err, PE_BAD_SCORE);
      if (!(f > 0.0 && f < INFINITY)) set_word(b.err, PE_BAD_SCALE);
      had[r] = score;
      scale[r] = f;
      lse[r] = ended ? NAN : m > -INFINITY ? m + log(s) : 0.0;  // a row that allows nothing: every logit stays -inf
    }
  }
  if (tid == 0) nparts = 0;
  __syncthreads();
  const Cont none = {-INFINITY, -INFINITY, INT32_MAX, INT32_MAX};
  const auto rank_of = [&](int r, double x) { return (had[r] + (x - lse[r])) * scale[r]; };
  // the best rank of a quarter, of its maximum; an ended row's one continuation is its first quarter's
  const auto top = [&](int e, double x) -> double {
    const int r = e / parts;
    if (had[r] == -INFINITY) return -INFINITY;
    if (isnan(lse[r])) return e - r * parts ? -INFINITY : had[r] * scale[r];
    return rank_of(r, x);
  };
  const auto look = [&](int e) { return top(e, w.m[row0 * parts + e]); };
#pragma unroll
  for (int k = 0; k < BS_HELD; ++k) held[k] = tid + 1024 * k < E ? top(tid + 1024 * k, held[k]) : -INFINITY;
  // this thread's quarters and their best ranks above -inf
  const auto tops = [&](auto&& f) {
#pragma unroll
    for (int k = 0; k < BS_HELD; ++k)
      if (held[k] > -INFINITY) f(tid + 1024 * k, held[k]);
    for (int e = tid + 1024 * BS_HELD; e < E; e += 1024) {
      const double t = look(e);
      if (t > -INFINITY) f(e, t);
    }
  };
  // smallest, largest and number of the block's ranks above -inf
  const auto extent = [&](double& lo, double& hi, int& n) {
    const double l = wave_max(-lo), h = wave_max(hi);
    int a, b;
    pair16_i32(row16_sumi(n), a, b);
    pair32_i32(a + b, a, b);
    __syncthreads();
    if (lane == 0) lows[wave] = l, highs[wave] = h, sums[wave] = a + b;
    __syncthreads();
    lo = -row16_max(lows[lane & 15]);
    hi = row16_max(highs[lane & 15]);
    n = row16_sumi(sums[lane & 15]);
  };
  // the highest bin that K ranks reach, once they are counted in `bins`: every wave
  // on its own, a lane four bins from the highest down
  const auto bound = [&]() {
    __syncthreads();
    const int4 q = ((const int4*)bins)[BB_BINS / 4 - 1 - lane];
    const int own = q.x + q.y + q.z + q.w;
    int upto = own;
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    const int from = __ffsll((unsigned long long)__ballot(upto >= K)) - 1;  // K ranks are counted
    int level = BB_BINS - 4 - 4 * lane, above = upto - own + q.w;
    if (above >= K) level += 3;
    else if ((above += q.z) >= K) level += 2;
    else if (above + q.y >= K) level += 1;
    level = __shfl(level, from);
    __syncthreads();  // before anybody counts anew
    return level;
  };
  double lo = INFINITY, hi = -INFINITY;
  int n = 0;
  tops([&](int, double t) { lo = fmin(lo, t), hi = fmax(hi, t), ++n; });
  if (tid < BB_BINS) bins[tid] = 0;
  extent(lo, hi, n);
  RankBins in(lo, hi);
  int least = -1;  // continuations of this bin and above are listed; those below every maximum are in bin -1 or 0
  if (n > K) {
    tops([&](int, double t) { atomicAdd(&bins[in.of(t)], 1); });
    least = bound();
  }
  tops([&](int e, double t) {
    if (in.of(t) < least) return;
    const int at = atomicAdd(&nparts, 1);
    if (at < BS_PARTS) plist[at] = e;
  });
  __syncthreads();
  const bool all_parts = nparts > BS_PARTS;
  const int np = all_parts ? E : nparts;
  // every continuation of the listed quarters that reaches the bound
  const auto visit = [&](auto&& f) {
    for (int p = tid >> 4; p < np; p += 4 * BS_WAVES) {
      const int e = all_parts ? p : plist[p], r = e / parts, t0 = (e - r * parts) * 32 * PER;
      if (all_parts && !(look(e) > -INFINITY)) continue;
      if (isnan(lse[r])) {
        const Cont c = {had[r] * scale[r], 0.0, r, -1};
        if ((lane & 15) == 0 && in.of(c.rank) >= least) f(c);
        continue;
      }
      v2logit v[PER];
      beam_load(b.x + (row0 + r) * b.V, b.V, t0, v);
      beam_cut(b.V, t0, v);
#pragma unroll
      for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const double x = h ? v[k].y : v[k].x;
          const Cont c = {rank_of(r, x), x, r, beam_token(t0, k) + h};
          if (c.rank > -INFINITY && in.of(c.rank) >= least) f(c);
        }
    }
  };
  const auto put = [&](int j, const Cont& c) {
    const long at = (long)g * K + j;
    const bool there = c.rank > -INFINITY;
    b.parents[at] = there ? (uint32_t)(row0 + c.row) : NO_ROW;
    b.tokens[at] = there && c.t >= 0 ? (uint32_t)c.t : NO_TOKEN;
    b.best[at] = !there ? -INFINITY : c.t < 0 ? had[c.row] : had[c.row] + (c.x - lse[c.row]);
  };
  for (int round = 0;; ++round) {
    if (tid == 0) listed = 0;
    __syncthreads();
    visit([&](const Cont& c) {
      const int at = atomicAdd(&listed, 1);
      if (at < BS_LIST) list[at] = c;
    });
    __syncthreads();
    if (listed <= BS_LIST || round == 4) break;
    // a closer bound among what reached this one
    lo = INFINITY, hi = -INFINITY, n = 0;
    visit([&](const Cont& c) { lo = fmin(lo, c.rank), hi = fmax(hi, c.rank), ++n; });
    extent(lo, hi, n);
    if (!(lo < hi)) break;
    const RankBins closer(lo, hi);
    if (tid < BB_BINS) bins[tid] = 0;
    __syncthreads();
    visit([&](const Cont& c) { atomicAdd(&bins[closer.of(c.rank)], 1); });
    least = bound();
    in = closer;
  }
  if (listed <= BS_LIST) {  // a wave to a continuation, a lane to another it is compared with
    const int m = listed;
    for (int i = wave; i < m; i += BS_WAVES) {
      const Cont c = list[i];
      int at = 0;
      for (int j0 = 0; j0 < m; j0 += 64) {
        const Cont o = list[min(j0 + lane, m - 1)];
        at += __popcll(__ballot(j0 + lane < m && before(o, c)));
      }
      if (at < K && lane == 0) put(at, c);
    }
    if (tid >= m && tid < K) put(tid, none);
    return;
  }
  Cont last = none;
  for (int j = 0; j < K; ++j) {
    Cont best = none;
    visit([&](const Cont& c) {
      if (before(c, best) && (!j || before(last, c))) best = c;
    });
    wave_first(best);
    __syncthreads();
    if (lane == 0) part[wave] = best;
    __syncthreads();
    last = part[0];
    for (int k = 1; k < BS_WAVES; ++k)
      if (before(part[k], last)) last = part[k];
    if (tid == 0) put(j, last);
  }
}

void beam_select(hipStream_t st, const BeamSelect& b) {
  BeamWs w;
  beam_layout(b, (char*)b.ws, w);
  const int piece = beam_piece(b), pieces = (b.V + piece - 1) / piece;
  const uint32_t blocks = (uint32_t)(pieces + 3) / 4;
  const dim3 grid((unsigned)(b.groups * b.beams) * blocks);  // the caller sees to fewer than 2^24
  const auto run = [&](auto piece_kern, auto pick_kern) {
    hipLaunchKernelGGL(piece_kern, grid, dim3(256), 0, st, b, w, pieces, blocks);
    for (int g = 0; g < b.groups; g += BS_GROUPS)
      hipLaunchKernelGGL(pick_kern, dim3(std::min(BS_GROUPS, b.groups - g)), dim3(1024), 0, st, b, w, pieces, g);
  };
  if (piece == 512) run(k_beam_pieces<4>, k_beam_pick<4>);
  else run(k_beam_pieces<2>, k_beam_pick<2>);
}

__global__ __launch_bounds__(256) void k_beam_advance(BeamAdvance a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.groups * a.keep) return;
  const int g = i / a.keep;
  const uint32_t r = a.parents[i], t = a.tokens[i];
  uint32_t done = 0, len = 0, id = 0, from = (uint32_t)(g * a.beams);
  if (r != NO_ROW) {
    const bool had = a.done && a.done[r];
    done = had || t == a.end;
    len = (a.len ? a.len[r] : 0u) + (had ? 0u : 1u);
    id = had ? a.end : t;
    from = r;
    if (!done) __hip_atomic_fetch_add(a.live, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  a.done_out[i] = done;
  a.len_out[i] = len;
  a.scale_out[i] = pow((double)(done ? len : len + 1), -a.power);
  a.ids[i] = id < (uint32_t)a.V ? id : 0u;
  a.from[i] = from;
}

void beam_advance(hipStream_t st, const BeamAdvance& a) {
  hipLaunchKernelGGL(k_beam_advance, dim3((a.groups * a.keep + 255) / 256), dim3(256), 0, st, a);
}

}  // namespace mitok

// beams.hip — beams on a paged cache: sequences that take other sequences' pages
// (ForkPages in paged.hpp), and the best continuations of a group of beams
// (BeamSelect).
#include <algorithm>

#include "paged.hpp"

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

// One block per new sequence: its parent's rows and pages, and what it does to
// the counts of those.  A sequence that is refused holds nothing.
__global__ __launch_bounds__(256) void k_fork_take(ForkPages f, ForkWs w) {
  const uint32_t i = blockIdx.x, tid = threadIdx.x;
  const uint32_t p = f.parents ? f.parents[i] : i;
  uint32_t len = 0, room = 0;
  bool bad = false;
  if (p != NO_ROW) {
    if (p >= f.old) {
      bad = true;
      if (tid == 0) set_word(f.err, PE_BAD_PARENT);
    } else {
      len = f.lens[p];
      room = f.grow ? f.grow[i] : f.grow_all;
      if ((uint64_t)len + room > (uint64_t)f.max_pages * f.page_rows) {
        bad = true;
        len = room = 0;
        if (tid == 0) set_word(f.err, PE_BAD_LENGTH);
      }
    }
  }
  const uint32_t had = (len + f.page_rows - 1) / f.page_rows;
  const bool writes = room > 0 && len % f.page_rows;
  for (uint32_t j = tid; j < had; j += 256) {
    const uint32_t id = f.table[(size_t)p * f.max_pages + j];
    w.table[(size_t)i * f.max_pages + j] = id;
    if (id >= f.pages) {
      bad = true;
      set_word(f.err, PE_BAD_PAGE);
      continue;
    }
    atomicAdd(f.held + id, 1u);
    if (writes && j + 1 == had) {
      atomicAdd(f.held + f.pages + id, 1u);
      atomicMax(f.held + 2 * (size_t)f.pages + id, f.n - i);
    }
  }
  if (tid == 0) {
    w.len[i] = len;
    w.room[i] = room;
  }
  if (bad) *f.refused = f.call;  // the same value, whoever writes it
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
__global__ __launch_bounds__(1024) void k_fork_assign(ForkPages f, ForkWs w) {
  __shared__ uint32_t part[16];
  const uint32_t tid = threadIdx.x;
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
          const bool all_write = f.held[f.pages + id] == f.held[id], first = f.held[2 * (size_t)f.pages + id] == f.n - i;
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
    const bool is_free = id < f.pages && f.held[id] == 0;
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
// used rows of a copied page, head by head (a head's rows are contiguous).
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
  hipLaunchKernelGGL(k_fork_take, dim3(f.n), dim3(256), 0, st, f, w);
  hipLaunchKernelGGL(k_fork_assign, dim3(1), dim3(1024), 0, st, f, w);
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
// A row is cut into pieces of BS_PIECE logits, a wave each: its maximum, the
// first token that has it, and the sum of exponentials below that.  Of the K best
// pieces by their maxima none of the other pieces' logits can be among the K
// best, nor any logit that comes after the least of those K maxima: so the
// logits are read once, and of them again only K pieces.
constexpr int BS_PER = 8, BS_PIECE = 64 * BS_PER;
struct BeamWs {
  double* m;  // [rows][pieces]
  double* s;
  int* at;
};
static int beam_pieces(int V) { return (V + BS_PIECE - 1) / BS_PIECE; }
static size_t beam_layout(const BeamSelect& b, char* base, BeamWs& w) {
  const size_t n = (size_t)b.groups * b.beams * beam_pieces(b.V);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  w.m = (double*)take(n * sizeof(double));
  w.s = (double*)take(n * sizeof(double));
  w.at = (int*)take(n * sizeof(int));
  return at;
}
size_t beam_ws_bytes(const BeamSelect& b) {
  BeamWs w;
  return beam_layout(b, nullptr, w);
}

// the larger value, of equal ones the lower index; NaN never wins
__device__ __forceinline__ void first_max(double& v, int& i, double ov, int oi) {
  if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
}
template <int CTRL>
__device__ __forceinline__ void first_max_dpp(double& v, int& i) {
  first_max(v, i, dpp_f64<CTRL>(v), dpp_i32<CTRL>(i));
}
__device__ __forceinline__ void wave_first_max(double& v, int& i) {
  first_max_dpp<DPP_XOR1>(v, i);
  first_max_dpp<DPP_XOR2>(v, i);
  first_max_dpp<DPP_HALF_MIRROR>(v, i);
  first_max_dpp<DPP_MIRROR>(v, i);
  double a, b;
  int ia, ib;
  pair16_f64(v, a, b);
  pair16_i32(i, ia, ib);
  first_max(a, ia, b, ib);
  pair32_f64(a, v, b);
  pair32_i32(ia, i, ib);
  first_max(v, i, b, ib);
}

// a row without logits to read: ended, or of score -inf
__device__ __forceinline__ bool beam_idle(const BeamSelect& b, long row) {
  return b.scores[row] == -INFINITY || (b.done && b.done[row]);
}

__global__ __launch_bounds__(256) void k_beam_pieces(BeamSelect b, BeamWs w, int pieces, long waves) {
  const int lane = threadIdx.x & 63;
  const long step = (long)gridDim.x * 4;
  for (long x = (long)blockIdx.x * 4 + (threadIdx.x >> 6); x < waves; x += step) {
    const long row = x / pieces;
    const int piece = (int)(x - row * pieces), t0 = piece * BS_PIECE;
    if (beam_idle(b, row)) continue;
    const double* p = b.x + row * b.V;
    double v[BS_PER];
#pragma unroll
    for (int k = 0; k < BS_PER; ++k) {
      const int t = t0 + 64 * k + lane;
      v[k] = t < b.V ? __builtin_nontemporal_load((const MITOK_GLOBAL double*)(p + t)) : -INFINITY;
    }
    double m = -INFINITY;
    int at = INT32_MAX;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < BS_PER; ++k) {
      bad |= !(v[k] < INFINITY);  // NaN, or an infinity that leaves no distribution
      first_max(m, at, v[k], t0 + 64 * k + lane);
    }
    if (__ballot(bad) && lane == 0) set_word(b.err, PE_BAD_SCORE);
    wave_first_max(m, at);
    double s = 0.0;
    if (m > -INFINITY) {
#pragma unroll
      for (int k = 0; k < BS_PER; ++k) s += exp(v[k] - m);
    }
    s = wave_sum(s);
    if (lane == 0) {
      w.m[x] = m;
      w.s[x] = s;
      w.at[x] = at;
    }
  }
}

// the order of continuations: rank, then the lower row, the larger logit, the lower token
struct Cont {
  double rank, x;
  int row, t;
};
__device__ __forceinline__ bool before(const Cont& a, const Cont& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.row != b.row) return a.row < b.row;
  if (a.x != b.x) return a.x > b.x;
  return a.t < b.t;
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

// One block per group.  Each round finds the first continuation after the last
// one found: K rounds over the pieces' maxima give the K best pieces and the
// bound, then the logits of those that do not come after the bound are listed
// and each one's place is how many come before it.  Where the list overflows
// (many equal logits, or fewer pieces than K), K rounds over the pieces' logits.
constexpr int BS_LIST = 1024;
__global__ __launch_bounds__(256) void k_beam_pick(BeamSelect b, BeamWs w, int pieces) {
  __shared__ double lse[1024];  // of the group's rows
  __shared__ Cont part[4], list[BS_LIST], chosen[BEAM_MAX_KEEP];
  __shared__ int listed;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = b.beams, K = b.keep;
  const long row0 = (long)g * R;
  for (int r = wave; r < R; r += 4) {
    const long row = row0 + r;
    const double had = b.scores[row];
    if (lane == 0) {
      if (isnan(had) || had == INFINITY) set_word(b.err, PE_BAD_SCORE);
      if (b.scale && !(b.scale[row] > 0.0 && b.scale[row] < INFINITY)) set_word(b.err, PE_BAD_SCALE);
    }
    if (beam_idle(b, row)) continue;
    double m = -INFINITY, s = 0.0;
    for (int c = lane; c < pieces; c += 64) m = fmax(m, w.m[row * pieces + c]);
    m = wave_max(m);
    if (m > -INFINITY) {
      for (int c = lane; c < pieces; c += 64) s += w.s[row * pieces + c] * exp(w.m[row * pieces + c] - m);
      s = wave_sum(s);
    }
    if (lane == 0) lse[r] = m > -INFINITY ? m + log(s) : 0.0;  // a row that allows nothing: every logit stays -inf
  }
  if (tid == 0) listed = 0;
  __syncthreads();
  const auto cont = [&](int r, double x, int t) {
    Cont c;
    c.row = r;
    c.x = x;
    c.t = t;
    c.rank = (b.scores[row0 + r] + (x - lse[r])) * (b.scale ? b.scale[row0 + r] : 1.0);
    return c;
  };
  const Cont none = {-INFINITY, -INFINITY, INT32_MAX, INT32_MAX};
  // entry e of the group's pieces: its best continuation; an ended row's one continuation is its first piece's
  const auto entry = [&](int e) {
    const int r = e / pieces, c = e - r * pieces;
    const long row = row0 + r;
    if (b.scores[row] == -INFINITY) return none;
    if (b.done && b.done[row]) {
      if (c) return none;
      Cont o = {b.scores[row] * (b.scale ? b.scale[row] : 1.0), 0.0, r, -1};
      return o;
    }
    return cont(r, w.m[row * pieces + c], w.at[row * pieces + c]);
  };
  // the first of what comes after `last`, of all the block's threads
  const auto next = [&](Cont best) {
    wave_first(best);
    if (lane == 0) part[wave] = best;
    __syncthreads();
    best = part[0];
    for (int k = 1; k < 4; ++k)
      if (before(part[k], best)) best = part[k];
    __syncthreads();
    return best;
  };
  int n = 0;  // pieces chosen
  for (; n < K; ++n) {
    Cont best = none;
    for (int e = tid; e < R * pieces; e += 256) {
      const Cont c = entry(e);
      if (c.rank > -INFINITY && before(c, best) && (!n || before(chosen[n - 1], c))) best = c;
    }
    best = next(best);
    if (best.rank == -INFINITY) break;
    if (tid == 0) chosen[n] = best;
    __syncthreads();
  }
  const Cont bound = n == K ? chosen[K - 1] : none;
  // the continuations of a chosen piece, this thread's
  const auto each = [&](int k, auto&& f) {
    const Cont p = chosen[k];
    if (p.t < 0) {
      if (tid == 0) f(p);
      return;
    }
    const int t0 = p.t / BS_PIECE * BS_PIECE;
    for (int t = t0 + tid; t < min(t0 + BS_PIECE, b.V); t += 256) {
      const Cont c = cont(p.row, b.x[(row0 + p.row) * b.V + t], t);
      if (c.rank > -INFINITY) f(c);
    }
  };
  for (int k = 0; k < n; ++k)
    each(k, [&](const Cont& c) {
      if (before(bound, c)) return;
      const int at = atomicAdd(&listed, 1);
      if (at < BS_LIST) list[at] = c;
    });
  __syncthreads();
  const auto put = [&](int j, const Cont& c) {
    const long at = (long)g * K + j;
    const bool there = c.rank > -INFINITY;
    b.parents[at] = there ? (uint32_t)(row0 + c.row) : NO_ROW;
    b.tokens[at] = there && c.t >= 0 ? (uint32_t)c.t : NO_TOKEN;
    b.best[at] = !there ? -INFINITY : c.t < 0 ? b.scores[row0 + c.row] : b.scores[row0 + c.row] + (c.x - lse[c.row]);
  };
  if (listed <= BS_LIST) {
    for (int i = tid; i < listed; i += 256) {
      const Cont c = list[i];
      int at = 0;
      for (int j = 0; j < listed; ++j) at += before(list[j], c);
      if (at < K) put(at, c);
    }
    for (int j = listed + tid; j < K; j += 256) put(j, none);
    return;
  }
  Cont last = none;
  for (int j = 0; j < K; ++j) {
    Cont best = none;
    for (int k = 0; k < n; ++k)
      each(k, [&](const Cont& c) {
        if (before(c, best) && (!j || before(last, c))) best = c;
      });
    last = next(best);
    if (tid == 0) put(j, last);
    if (last.rank == -INFINITY) {
      for (int i = j + 1 + tid; i < K; i += 256) put(i, none);
      return;
    }
  }
}

void beam_select(hipStream_t st, const BeamSelect& b) {
  BeamWs w;
  beam_layout(b, (char*)b.ws, w);
  const int pieces = beam_pieces(b.V);
  const long waves = (long)b.groups * b.beams * pieces;
  hipLaunchKernelGGL(k_beam_pieces, dim3((unsigned)std::min<long>((waves + 3) / 4, 65536)), dim3(256), 0, st, b, w, pieces, waves);
  hipLaunchKernelGGL(k_beam_pick, dim3(b.groups), dim3(256), 0, st, b, w, pieces);
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

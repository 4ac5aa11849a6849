// paged.hpp — launch wrappers of the operators of a beam search on a paged
// cache: attention of a chunk of new tokens (paged_attention.hip), forks of
// sequences with their pages and the selection over beams and vocabulary
// (beams.hip).
//
// As in kernels.hpp, every wrapper enqueues on `st` and neither synchronises
// nor allocates.
#pragma once

#include "serving.hpp"

namespace mitok {

constexpr int PAGE_TILE = 16;       // a page holds a multiple of so many rows, so a tile of slots lies in one
constexpr int PAGE_MAX_ROWS = 1024;
constexpr uint32_t NO_PAGE = 0xFFFFFFFFu;

// words of these operators' kernels, as OpErrWord
enum PageErrWord : int {
  PE_BAD_PAGE = 0, PE_BAD_PARENT = 1, PE_BAD_LENGTH = 2, PE_NO_PAGES = 3, PE_SHARED_PAGE = 4,
  PE_BAD_SCORE = 5, PE_BAD_SCALE = 6, PE_WORDS = 8
};

// ---- attention of a chunk of new tokens over a paged cache ----
// Sequence b holds kv_len[b] rows: slot t in row t % page_rows of page
// table[b][t / page_rows].  Its count[b] new rows go to the slots behind them,
// and new row i sees the slots up to its own, kv_len[b] + i:
//   s(i, t) = Re(q_i . k_t) * scale + bias[h][row(i)][t],
//   row(i) = kv_len[b] + i, or 0 where bias_row is
//   out_i = sum_t softmax(s(i, .))_t v_t; rows past count[b] are zero
struct PagedAttn {
  const double2* q = nullptr;  // [B][n][ldq]; head h at column h * dh
  long ldq = 0;
  const double2* kn = nullptr;  // the new rows: sequence, row and head these strides apart
  const double2* vn = nullptr;
  long new_b = 0, new_row = 0, new_head = 0;
  double2* kp = nullptr;  // [pages][H][page_rows][dh]
  double2* vp = nullptr;
  const uint32_t* table = nullptr;  // [B][max_pages]
  int max_pages = 0, page_rows = 0;
  uint32_t pages = 0;
  const double* bias = nullptr;  // or null
  long bias_stride = 0, bias_row = 0;
  const char* tab = nullptr;  // the host's arrays (OpTable)
  uint32_t kv_len = 0;        // int [B]
  uint32_t count = 0;         // int [B]
  int B = 0, n = 0, H = 0, dh = 0;
  double scale = 1.0;
  double2* out = nullptr;  // [B][n][ldo]
  long ldo = 0;
  void* ws = nullptr;  // paged_ws_bytes
  // [pages] or null: the call, the sequence and which of its pages last stored to
  // a page, which tells two that store to the same in one call
  unsigned long long* stamp = nullptr;
  uint32_t call = 0;
  uint32_t* err = nullptr;  // PageErrWord
};
// How a call's work is cut up, from its lengths: groups of `rows` new rows, and
// ranges of pieces of them, a block each (for every head).  The lists are appended
// to `lists`; pieces, ranges and cuts are their byte offsets, once the lists' own
// place is known.  A plan also serves shorter sequences of up to 32 rows each: a
// piece ends where the sequence does.
struct PagedPlan {
  bool beams = false;   // a piece is a bunch of sequences of one row: the first one, how many
  int ng = 1;           // groups of 16 rows that a block's waves have of their own
  int rows = 16;        // 16 ng
  int groups = 1;       // of a sequence
  int blocks = 0;       // of a head
  int part_rows = 0;    // rows of the pieces of groups that were cut
  uint32_t pieces = 0;  // int4 each: sequence, first row, first slot, end
  uint32_t places = 0;  // int each: place of its rows among the partials, or -1
  uint32_t ranges = 0;  // int [blocks + 1] (ng 4): a block's pieces
  uint32_t cuts = 0;    // int2 [B][groups] (part_rows > 0): place of the first piece's rows, pieces
};
PagedPlan paged_plan(const PagedAttn& a, const int* kv_len, const int* count, std::vector<int>& lists);
size_t paged_ws_bytes(const PagedAttn& a, const PagedPlan& p);
void paged_attention(hipStream_t st, const PagedAttn& a, const PagedPlan& p, const OpTable& own);

// ---- sequences that take other sequences' pages ----
// New sequence i takes the rows of old sequence parents[i] (or none: NO_ROW) and
// room for grow[i] more.  Pages are shared, but a sequence that grows writes
// behind its rows: a part-filled last page that another new sequence holds too
// is copied to a free page (its used rows, in every layer), except for the first
// of its holders if all of them grow from it as their last page.  Free is what
// no new sequence holds; free pages are taken in ascending order, sequence by
// sequence, a copy before the room.  An error leaves everything as it was.
struct ForkPages {
  const uint32_t* table = nullptr;  // [old][max_pages]
  const uint32_t* lens = nullptr;   // [old] rows
  const uint32_t* parents = nullptr;  // [n], or null: i itself
  const uint32_t* grow = nullptr;     // [n], or null: grow_all each
  uint32_t grow_all = 0;
  uint32_t* table_out = nullptr;      // [n][max_pages]; NO_PAGE behind a sequence's last
  uint32_t* lens_out = nullptr;       // [n] rows, without the room; both may be the inputs
  uint32_t old = 0, n = 0, max_pages = 0, page_rows = 0, pages = 0;
  uint32_t* held = nullptr;  // fork_held_words(pages), zero between calls
  void* ws = nullptr;        // fork_ws_bytes
  uint32_t* refused = nullptr;  // a device word that holds `call` where an input is refused
  uint32_t call = 0;
  uint32_t* err = nullptr;   // PageErrWord
};
size_t fork_held_words(uint32_t pages);
size_t fork_ws_bytes(uint32_t n, uint32_t max_pages, uint32_t pages);
// A pool whose copies fork_copy makes: `layers` of [pages][H][page_rows][dh]
struct PagePool {
  double2* k = nullptr;
  double2* v = nullptr;
  int layers = 1, H = 0, dh = 0;
};
// the new tables and lengths, and the list of copies in the workspace
void fork_plan(hipStream_t st, const ForkPages& f);
// the copies of one pool; several pools of one plan may follow it
void fork_copy(hipStream_t st, const ForkPages& f, const PagePool& pool, bool commit);

// ---- the best continuations of a group of beams ----
// Of the continuations (row, token) of each group's `beams` rows the `keep` of
// largest rank:
//   score(r, t) = scores[r] + x[r][t] - log sum_u exp x[r][u],
//   rank = score * scale[r]
// in a row the larger logit first, equal ones the lower token, between rows the
// larger rank, equal ones the lower row.  A row with done[r] has one
// continuation, no token, of score scores[r]; one of score -inf has none.
constexpr int BEAM_MAX_KEEP = 64;
struct BeamSelect {
  const double* x = nullptr;  // [groups * beams][V]
  const double* scores = nullptr;
  const uint32_t* done = nullptr;  // or null
  const double* scale = nullptr;   // or null: 1
  int groups = 0, beams = 0, V = 0, keep = 0;
  uint32_t* parents = nullptr;  // [groups][keep]: the row (of all), NO_ROW where there is no continuation
  uint32_t* tokens = nullptr;   // NO_TOKEN there and of done rows
  double* best = nullptr;       // scores, -inf there
  void* ws = nullptr;           // beam_ws_bytes
  uint32_t* err = nullptr;      // PageErrWord
};
size_t beam_ws_bytes(const BeamSelect& s);
void beam_select(hipStream_t st, const BeamSelect& s);

// From a step's selection to the next step's rows, one per new beam (n =
// groups * keep): what it feeds, whether it has ended and after how many tokens,
// and the factor its continuations are ranked by, (tokens then)^-power.  A beam
// without a continuation goes on as a copy of its group's first row, of score -inf.
struct BeamAdvance {
  const uint32_t* parents = nullptr;  // the selection's
  const uint32_t* tokens = nullptr;
  const uint32_t* done = nullptr;  // of the rows selected from, or null: none has ended
  const uint32_t* len = nullptr;   // their tokens, or null: 0
  int groups = 0, beams = 0, keep = 0, V = 0;
  uint32_t end = NO_TOKEN;
  double power = 0.0;
  uint32_t* done_out = nullptr;
  uint32_t* len_out = nullptr;
  double* scale_out = nullptr;
  uint32_t* ids = nullptr;      // the token fed
  uint32_t* from = nullptr;     // the row whose pages it takes
  uint32_t* live = nullptr;     // += beams that go on
};
void beam_advance(hipStream_t st, const BeamAdvance& a);

}  // namespace mitok

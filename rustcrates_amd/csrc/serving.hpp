// serving.hpp — launch wrappers of the operators of a serving loop over the KV
// cache: attention of drafted token trees (tree_attention.hip), eviction of
// cached rows and the rules that turn logits into a token (serving.hip).
//
// As in kernels.hpp, every wrapper enqueues on `st` and neither synchronises
// nor allocates.
#pragma once

#include <vector>

#include "kernels.hpp"

namespace mitok {

// Words a kernel sets and the host reads once the stream is idle (pinned host
// memory: no copy back).  Plain stores of 1, so any number of lanes may set one.
enum OpErrWord : int { OE_BAD_TOKEN = 0, OE_NAN = 1, OE_BAD_PENALTY = 2, OE_WORDS = 4 };
__device__ __forceinline__ void set_word(uint32_t* err, int word) {
  __hip_atomic_store(err + word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// The host's small arrays of a call (lengths, trees, lists), at byte offsets of
// one table: in the kernels' own arguments where they fit, which saves the
// upload's 3 us, else in device memory (`tab` of the operator's struct).
struct OpTable {
  static constexpr size_t ROOM = 2032;
  alignas(16) unsigned char at[ROOM];
};

constexpr int TREE_MAX_NODES = 256;
constexpr int TREE_WORDS = TREE_MAX_NODES / 64;
constexpr int TREE_MAX_DH = 256;

// ---- attention of a tree of drafted tokens ----
// Node i of sequence b sits in cache slot kv_len[b] + i and sees the slots
// before kv_len[b], its ancestors and itself:
//   s(i, t) = Re(q_i . k_t) * scale + bias[h][column(t)],
//   column(t) = t, or kv_len[b] + depth(j) for node j's slot
//   out_i = sum_t softmax(s(i, .))_t v_t
// weights (if not null): [b][h][t] += the sum over the first `weigh` nodes of
// their softmax weights at the committed slots, = at the nodes' slots.
struct TreeAttn {
  const double2* q = nullptr;  // [B][n][ldq]; head h at column h * dh
  long ldq = 0;
  const double2* kc = nullptr;  // [B][H][ctx][dh]
  const double2* vc = nullptr;
  const double* bias = nullptr;  // [H][bias_stride] or null
  long bias_stride = 0;
  const char* tab = nullptr;  // the table, or null: the kernels' arguments
  uint32_t seen = 0;          // 64-bit [B][n][words]: bit j of a node: itself or an ancestor
  uint32_t kv_len = 0;        // int [B]
  uint32_t count = 0;         // int [B] nodes used; rows past them are zero
  uint32_t depth = 0;         // int [B][n]
  int words = 1;
  int B = 0, n = 0, H = 0, dh = 0, ctx = 0;
  double scale = 1.0;
  int weigh = 0;
  double* weights = nullptr;  // [B][H][ctx]
  double2* out = nullptr;     // [B][n][ldo]
  long ldo = 0;
  void* ws = nullptr;  // tree_ws_bytes
};
// How a call's work is cut up, from its lengths (host arrays): each sequence's
// slots in chunks, the longest first.  The lists are appended to `lists`;
// chunks and splits are their offsets, once the lists' own place is known.
struct TreePlan {
  int ng = 1;      // groups of 16 nodes per block
  int entries = 0; // chunks of all sequences
  int nsplit = 1;  // the most of one sequence
  int T = 0;       // the most slots of one sequence
  uint32_t chunks = 0;  // int4 [entries]: sequence, first slot, end, index in the sequence
  uint32_t splits = 0;  // int [B] chunks of each sequence
};
TreePlan tree_plan(const TreeAttn& a, const int* kv_len, const int* count, std::vector<int>& lists);
size_t tree_ws_bytes(const TreeAttn& a, const TreePlan& p);
void tree_attention(hipStream_t st, const TreeAttn& a, const TreePlan& p, const OpTable& own);

// ---- rows of a cache moved to its front, or to another cache's ----
struct CacheMove {
  const double2* k = nullptr;  // [B][H][ctx][dh]
  const double2* v = nullptr;
  const double* w = nullptr;  // [B][H][ctx] weights, or null
  double2* ko = nullptr;      // [B][H][ctx_out][dh]; the same pointers: in place
  double2* vo = nullptr;
  double* wo = nullptr;
  int B = 0, H = 0, dh = 0;
  long ctx = 0, ctx_out = 0;
  const char* tab = nullptr;      // the table, or null: the kernels' arguments
  uint32_t base = 0;              // int [B] slot that both sides count from
  bool based = false;             // (else 0)
  const uint32_t* idx = nullptr;  // row r of (b, h) comes from slot base + idx[b * idx_b + h * idx_h + r]; ascending
  long idx_b = 0, idx_h = 0;
  uint32_t rows = 0;  // int [B] rows moved
  int rows_max = 0;
};
void cache_move(hipStream_t st, const CacheMove& m, const OpTable& own);

// ---- which rows an eviction keeps ----
// Of kv_len[b] rows, `keep` stay where there are more: the first `sinks`, the
// last `recent` and the others of largest weight (equal ones and NaN, which
// counts as less than any number: the lowest slot first).  kept
// [B][H][keep]: their slots ascending, then NO_ROW; rows [B]: min(kv_len, keep).
constexpr uint32_t NO_ROW = 0xFFFFFFFFu;
struct EvictSelect {
  const double* w = nullptr;  // [B][H][ctx]
  const char* tab = nullptr;
  uint32_t kv_len = 0;  // int [B] in the table
  int B = 0, H = 0;
  long ctx = 0;
  int T_max = 0;
  int keep = 0, sinks = 0, recent = 0;
  uint32_t* kept = nullptr;
};
void evict_select(hipStream_t st, const EvictSelect& e, const OpTable& own);

// w[b][h][from[b] .. to[b]) = 0
void zero_weights(hipStream_t st, double* w, int B, int H, long ctx, const int* from, const int* to, int most);
// dec_ids[b] = ids[b * n + last[b]] where last[b] >= 0
void pick_ids(hipStream_t st, const uint32_t* ids, int n, const int* last, int B, uint32_t* dec_ids);

// ---- logits to a token ----
constexpr uint32_t NO_TOKEN = 0xFFFFFFFFu;
struct LogitRules {
  const double* x = nullptr;  // [rows][V]
  int rows = 0, V = 0;
  const uint32_t* history = nullptr;  // [rows][hist] token ids, NO_TOKEN entries skipped
  int hist = 0;
  const double* penalties = nullptr;  // [rows][3]: repetition, presence, frequency
  const uint32_t* bias_ids = nullptr;  // [rows][nb], NO_TOKEN entries skipped; of equal ids the last counts
  const double* bias = nullptr;
  int nb = 0;
  const uint32_t* allowed = nullptr;   // [rows][(V + 31) / 32] bits
  const uint32_t* row_mask = nullptr;  // [rows] or null: rows with 0 are skipped, their id NO_TOKEN
  double* out = nullptr;               // [rows][V] or null; x itself: in place
  uint32_t* ids = nullptr;             // [rows] or null
  double* part_v = nullptr;            // [rows][logit_chunks(V)]
  int* part_i = nullptr;
  uint32_t* counters = nullptr;  // SYNC_COUNTERS words, zero
  uint32_t* err = nullptr;       // OpErrWord
  // in place: a device word that holds `call` where logit_check refused the
  // rules; no logit is changed then
  uint32_t* refused = nullptr;
  uint32_t call = 0;
};
int logit_chunks(int V);
// the ids and penalties of every row, before logit_rules changes any (r.refused)
void logit_check(hipStream_t st, const LogitRules& r);
void logit_rules(hipStream_t st, const LogitRules& r);

// an array of the table; the same value for every lane of a wave where `i` is
template <class T>
__device__ __forceinline__ const T* op_array(const char* tab, const OpTable& own, uint32_t at) {
  return (const T*)((tab ? tab : (const char*)own.at) + at);
}
__device__ __forceinline__ int op_int(const char* tab, const OpTable& own, uint32_t at, int i) {
  return __builtin_amdgcn_readfirstlane(op_array<int>(tab, own, at)[i]);
}

}  // namespace mitok

// Shared by the kernels of tq_attend: queries of one token or of many per sequence against the stored
// tokens, with a sliding window and first tokens that stay visible.
//
// Query token i of sequence s stands at position p = N_s - n_s + i (N_s tokens stored, the newest n_s of
// them are the queries' own) and sees the tokens j <= p with j < sinks or j > p - window.  The rows of a
// (sequence, KV head) unit are numbered i * G + g: neighbouring rows see nearly the same tokens, so a tile
// of rows reads the codes once for all query heads of the group.
//
// The kernels for few rows and the general ones leave states (m, l, o[D]) per (unit, row, split): m in units of
// log 2, o un-normalised; of the first ns_cold splits in the values' code space, of the others in the original basis.  A
// combine kernel merges them in split order, applies the inverse rotation once and rounds to the output's type.
// (Those for many rows have states of their own, all in code space.)
#pragma once

#include <limits.h>

#include "common.cuh"
#include "decode_generic.cuh"  // TQ_SCORE_LOG2, tq_exp2

// The states of a shared beginning as its form leaves them: [head][rows][ns][TQ_SLOT_STRIDE], the first ns_cold of them in code
// space; of a flagged head the general form's two, [head][rows][2][2 + D].
struct SharedStates {
  const float* slots;  // null: none
  const int32_t* left;
  const float* general;
  int32_t ns_cold, ns;
};
constexpr int TQ_SLOT_STRIDE = 4 + TQ_D;  // M, L, -, -, o

struct AttendArgs {
  tq_geom g;
  const uint8_t* pages;
  const void* hot_k;
  const void* hot_v;
  const uint32_t* pool_dec;
  const uint16_t* pool_val;
  const PageMeta* page_meta;
  const int32_t* seq_len;  // of the layer
  const Tables* tables;
  int32_t* status;
  const void* q;
  int64_t q_seq, q_tok, q_head;  // strides in elements
  void* out;                     // [seq_count][n_tokens][n_q_heads][D] of q_dtype
  const int32_t* q_lens;         // [seq_count] or null: n_tokens everywhere
  float* partials;               // per unit, unit_stride floats apart: [row][ns_cold + ns_hot][2 + D]
  int64_t unit_stride;
  void* plan;                    // the rows form's
  int32_t hot_cost;              // and its division of work: of a window tile
  // flags of the kernels for many rows, per unit: not zero, the unit is left to the general form (null: none)
  const int32_t* left;
  int32_t layer, seq_begin, seq_count, n_tokens, q_dtype;
  int32_t window, sinks;  // window: INT_MAX without one
  int32_t ns_cold, ns_hot;
  int32_t rows;  // of a unit: n_tokens * group
  int32_t device, sm_count;
  // listed: of the blocks a query token sees those on its list alone, [seq_count][n_tokens][n_kv_heads][n_list]
  const int32_t* list;
  int32_t n_list, listed;
  // A shared beginning: the queries of all sequences are those of one, the prefix, and see all that it holds (whole); the merge
  // leaves states (M, L, o[D]), o in the original basis, [unit][rows][2 + D].  The sequences' own part then takes them
  // into its merge: row r of a unit of head h has the state [h][before_rows][2 + D] at s * rows + r.
  int32_t whole;
  float* states;
  const float* before;
  int64_t before_rows;
  SharedStates shared;  // or its states, unmerged
  int32_t no_window;    // the rows form: the pages alone, and no merge
  int32_t wait_limit, withhold;  // test hook of the form for many rows (tq_debug_wait); 0 and -1 otherwise
};

// What a sequence holds and where its queries stand.
struct AttendSeq {
  int n;         // tokens stored
  int cold;      // of them in blocks
  int q_n;       // query tokens
  int first;     // position of query token 0
};
TQ_DEV AttendSeq attend_seq(const AttendArgs& a, int s) {
  AttendSeq r;
  r.n = a.seq_len[a.layer * a.g.n_seqs + a.seq_begin + s];
  r.cold = n_cold_blocks(r.n, a.g.hot_window, a.g.block_tokens) * a.g.block_tokens;
  r.q_n = a.q_lens == nullptr ? a.n_tokens : min(max(a.q_lens[s], 0), a.n_tokens);
  r.first = a.whole ? r.n : r.n - r.q_n;
  return r;
}
// position of a row's token; -1: the row sees nothing
TQ_DEV int attend_position(const AttendArgs& a, const AttendSeq& s, int row) {
  const int i = row / a.g.group;
  return i < s.q_n ? max(s.first + i, -1) : -1;
}
// first token of a position's window
TQ_DEV int attend_window(const AttendArgs& a, int p) { return max(p - a.window + 1, 0); }

// The tiles of `size` tokens of [base, end) that rows from position p_lo to p_hi see any of: those of the
// first tokens, then those of the window.  Tile t covers base + t * size ...
struct AttendTiles {
  int head, first, n;  // tiles 0 .. head - 1, then first .. first + n - 1
  TQ_DEV int count() const { return head + n; }
  TQ_DEV int at(int i) const { return i < head ? i : first + i - head; }
};
TQ_DEV AttendTiles attend_tiles(const AttendArgs& a, int base, int end, int size, int p_lo, int p_hi) {
  AttendTiles t = {0, 0, 0};
  const int last = min(end, p_hi + 1) - 1;  // last token seen
  if (p_hi < 0 || last < base) return t;
  const int w = attend_window(a, max(p_lo, 0));
  t.first = max(w - base, 0) / size;
  t.n = max((last - base) / size + 1 - t.first, 0);
  const int sink = min(a.sinks, last + 1) - base;
  t.head = sink > 0 ? min((sink + size - 1) / size, t.first) : 0;
  return t;
}

// ---- attention of listed blocks: every query token and KV head has a list of its own
TQ_DEV const int32_t* attend_list(const AttendArgs& a, int s, int i, int head) {
  return a.list + (((size_t)s * a.n_tokens + i) * a.g.n_kv_heads + head) * a.n_list;
}
// Entries of a list that count: a list ends at the first one that is not above the one before, or no block of the sequence
// (by a whole warp).
TQ_DEV int attend_listed(const AttendArgs& a, const int32_t* list, int blocks) {
  const int lane = threadIdx.x & 31;
  for (int k0 = 0; k0 < a.n_list; k0 += 32) {
    const int k = k0 + lane;
    const int v = k < a.n_list ? list[k] : -1, before = k > 0 && k < a.n_list ? list[k - 1] : -1;
    const uint32_t in = __ballot_sync(0xffffffffu, v > before && v < blocks);
    if (in != 0xffffffffu) return k0 + __ffs(~in) - 1;
  }
  return a.n_list;
}

TQ_DEV float* attend_partial(const AttendArgs& a, int unit, int row, int split) {
  return a.partials + (size_t)unit * a.unit_stride + ((size_t)row * (a.ns_cold + a.ns_hot) + split) * TQ_PART_STRIDE;
}

// The weight of a state in a merge whose maximum is `by`; a state without a sum takes no part, one whose sum is no number does.
TQ_DEV float attend_weight(float m, float l, float by) { return l == 0.0f ? 0.0f : m > -INFINITY ? tq_exp2(m - by) : 1.0f; }
// The state of a row's shared beginning, null where the row has no token of its own.
TQ_DEV const float* attend_before(const AttendArgs& a, int s, int head, int row) {
  if (a.before == nullptr || attend_position(a, attend_seq(a, s), row) < 0) return nullptr;
  return a.before + ((size_t)head * a.before_rows + (size_t)s * a.rows + row) * TQ_PART_STRIDE;
}
// Channel e of a merged row (maximum M, sum of weights L, sum of weighted values o) as the call's result.  PLAIN: no states of a
// shared beginning, neither given nor wanted.
template <bool PLAIN = false>
TQ_DEV void attend_result(const AttendArgs& a, int s, int head, int row, int e, float M, float L, float o) {
  const tq_geom& g = a.g;
  if (!PLAIN && a.states != nullptr) {
    float* to = a.states + ((size_t)(s * g.n_kv_heads + head) * a.rows + row) * TQ_PART_STRIDE;
    if (e == 0) *(float2*)to = make_float2(M, L);
    to[2 + e] = o;
    return;
  }
  if (const float* x = PLAIN ? nullptr : attend_before(a, s, head, row)) {
    const float top = fmaxf(M, x[0]), by = top > -INFINITY ? top : 0.0f;
    const float w = attend_weight(M, L, by), wx = attend_weight(x[0], x[1], by);
    L = (w != 0.0f ? L * w : 0.0f) + (wx != 0.0f ? x[1] * wx : 0.0f);
    o = (w != 0.0f ? o * w : 0.0f) + (wx != 0.0f ? x[2 + e] * wx : 0.0f);
  }
  const float v = L == 0.0f ? 0.0f : o / L;
  const int G = g.group;
  const size_t to = (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D + e;
  if (a.q_dtype == TQ_F32) ((float*)a.out)[to] = v;
  else if (a.q_dtype == TQ_F16) ((__half*)a.out)[to] = __float2half_rn(v);
  else ((__nv_bfloat16*)a.out)[to] = __float2bfloat16_rn(v);
}

TQ_DEV float attend_ld(const void* p, size_t i, int dt) {
  if (dt == TQ_F32) return ((const float*)p)[i];
  if (dt == TQ_F16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}

// Sets a kernel's dynamic shared memory once per device (again by a second thread at worst).
template <class K>
int attend_shared(K kernel, size_t bytes, int device, bool (&done)[64]) {
  if (device >= 0 && device < 64 && done[device]) return TQ_OK;
  TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  if (device >= 0 && device < 64) done[device] = true;
  return TQ_OK;
}

// The most tokens that one of these sequences may hold when a call's kernels run
int tq_most_tokens(const tq_ctx* ctx, int layer, int seq_begin, int seq_count, cudaStream_t st);
int tq_launch_attend_general(const AttendArgs& a, cudaStream_t st);
int tq_launch_attend_combine(const AttendArgs& a, cudaStream_t st);
// ---- the rows form's division of its work
constexpr int AR_SEQS = 64;        // sequences of a launch
// How long a strip takes, by whether operands are pairs (the measurements are beside the kernel)
TQ_HD constexpr int ar_cost(bool split) { return split ? 8 : 4; }
TQ_DEV int64_t ar_div(int64_t x, int64_t y) {  // (mostly of numbers that fit 32 bits)
  return (x | y) >> 32 == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}
// How a launch divides its work; the first CTA leaves it for the merge.
struct ArPlan {
  int64_t share;
  int64_t cum[AR_SEQS + 1];
  int4 seq[AR_SEQS];  // strips, window tiles and row tiles of a sequence
};
constexpr int TQ_ROWS_TILE = 8;  // query rows of a tile
// Few rows, 256-token blocks of per-channel keys, queries on 16-byte boundaries; the merge too.
struct AttendRowsPlan {
  int ns_cold, ns_hot;  // slots of a row's states
  int seqs;             // most sequences of a launch
  int hot_cost;         // of a window tile, for AttendArgs
  size_t plan_bytes;    // at a.plan
};
AttendRowsPlan tq_attend_rows_plan(const AttendArgs& a, int tokens);
int tq_launch_attend_rows(const AttendArgs& a, cudaStream_t st);
// 16-bit queries, per-channel keys: everything in one, the merge too; `cap` tiles of tokens per unit have room
constexpr int TQ_ATTEND_TILE = 80;  // tokens of a tile
size_t tq_attend_tiles_bytes(const AttendArgs& a, int units, int cap, int splits);
int tq_launch_attend_tiles(const AttendArgs& a, void* workspace, int cap, int splits, cudaStream_t st);
// A shared beginning: 16-bit queries, 256-token blocks of per-channel keys; the states
void tq_attend_shared_plan(const AttendArgs& a, int tokens, int* ns_cold, int* ns_hot);
size_t tq_attend_shared_bytes(const AttendArgs& a);
// `merged`: to a.states; else *as gets a.shared for those who merge it with theirs
int tq_launch_attend_shared(const AttendArgs& a, void* workspace, bool merged, SharedStates* as, cudaStream_t st);
// The last part of such a call where the sequences' queries are few rows of the window's 16-bit type: window and merge
int tq_launch_attend_window(const AttendArgs& a, int blocks_tile, cudaStream_t st);

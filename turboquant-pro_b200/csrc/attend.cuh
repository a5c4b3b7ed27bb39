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
  r.first = r.n - r.q_n;
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

TQ_DEV float* attend_partial(const AttendArgs& a, int unit, int row, int split) {
  return a.partials + (size_t)unit * a.unit_stride + ((size_t)row * (a.ns_cold + a.ns_hot) + split) * TQ_PART_STRIDE;
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

int tq_launch_attend_general(const AttendArgs& a, cudaStream_t st);
int tq_launch_attend_combine(const AttendArgs& a, cudaStream_t st);
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

// tq_attend: checks, the choice of a form, the division of the work, the workspace.
#include <algorithm>

#include "attend.cuh"

// The most tokens a sequence of the call may hold when the kernels run: the host's lengths, or the
// capacity where the launch is captured, since a replay may find longer sequences.
int tq_most_tokens(const tq_ctx* ctx, int layer, int seq_begin, int seq_count, cudaStream_t st) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone)
    return ctx->g.max_tokens_per_seq;
  int n = 0;
  for (int s = seq_begin; s < seq_begin + seq_count; ++s)
    n = std::max(n, ctx->len[(size_t)layer * ctx->g.n_seqs + s]);
  return n;
}

namespace {

constexpr size_t AT_ONE_GO = (size_t)1 << 30;  // workspace that a call asks for at most, unless one
                                               // sequence needs more

enum Form { GENERAL, ROWS, TILES, SHARED, WINDOW };
struct Plan {
  Form form;
  int ns_cold, ns_hot;
  int hot_cost;      // ROWS: of a window tile, in the division of the work
  int cap, splits;   // TILES: tiles that a (sequence, KV head) has room for, splits of them
  int seqs;          // most sequences of a launch
  size_t fixed_bytes, seq_bytes;  // workspace: of a launch, of a sequence
};

// A call: the caller's arguments, the blocks on its lists (listed), and the parts of a call with a shared beginning (see
// AttendArgs).
struct Call : tq_attend_args {
  const int32_t* list;
  int32_t n_list;
  bool listed, whole, merges;  // merges: the sequences' own part of a call with a shared beginning, which merges the states
  float* states;
  const float* before;
  int64_t before_rows;
  SharedStates shared;  // the prefix's states, not merged
  SharedStates* keep;   // of the prefix's part: they are to stay so
};
Call plain_call(const tq_attend_args* r) {
  Call c = {};
  (tq_attend_args&)c = *r;
  return c;
}
// The sequences from `s` on, `n` of them.
Call part_of(const tq_ctx* ctx, const Call& r, int s, int n) {
  const tq_geom& g = ctx->g;
  const size_t esz = elem_size(r.q_dtype);
  Call part = r;
  part.seq_begin = r.seq_begin + s;
  part.seq_count = n;
  part.q = (const uint8_t*)r.q + (int64_t)s * r.q_seq_stride * (int64_t)esz;
  part.out = (uint8_t*)r.out + (size_t)s * r.n_tokens * g.n_q_heads * TQ_D * esz;
  part.q_lens = r.q_lens == nullptr ? nullptr : r.q_lens + s;
  part.before = r.before == nullptr ? nullptr : r.before + (size_t)s * r.n_tokens * g.group * TQ_PART_STRIDE;
  if (r.shared.slots != nullptr) {
    const size_t row = (size_t)s * r.n_tokens * g.group;
    part.shared.slots += row * r.shared.ns * TQ_SLOT_STRIDE;
    part.shared.general += row * 2 * TQ_PART_STRIDE;
  }
  part.list = r.list == nullptr ? nullptr : r.list + (size_t)s * r.n_tokens * g.n_kv_heads * r.n_list;
  return part;
}

int check_args(tq_ctx* ctx, const tq_attend_args* r) {
  TQ_REQUIRE(ctx != nullptr && r != nullptr, TQ_ERR_INVALID, "null argument");
  const tq_geom& g = ctx->g;
  TQ_REQUIRE(r->layer >= 0 && r->layer < g.n_layers, TQ_ERR_INVALID, "bad layer");
  TQ_REQUIRE(r->seq_begin >= 0 && r->seq_count >= 0 && (int64_t)r->seq_begin + r->seq_count <= g.n_seqs,
             TQ_ERR_INVALID, "sequence range out of bounds");
  TQ_REQUIRE(r->n_tokens >= 0 && (int64_t)r->n_tokens * g.group <= (1 << 30), TQ_ERR_INVALID,
             "n_tokens out of range");
  TQ_REQUIRE(r->window >= 0 && r->sinks >= 0, TQ_ERR_INVALID, "window and sinks must not be negative");
  TQ_REQUIRE(r->q_dtype == TQ_F32 || r->q_dtype == TQ_F16 || r->q_dtype == TQ_BF16, TQ_ERR_INVALID,
             "bad q_dtype");
  const int64_t step = 16 / elem_size(r->q_dtype);
  TQ_REQUIRE(r->q_seq_stride % step == 0 && r->q_tok_stride % step == 0 && r->q_head_stride % step == 0 &&
                 (uintptr_t)r->q % 16 == 0 && (uintptr_t)r->out % 16 == 0,
             TQ_ERR_INVALID, "q, its strides and out must be aligned to 16 bytes");
  if (ctx->sm_count == 0)
    TQ_CUDA(cudaDeviceGetAttribute(&ctx->sm_count, cudaDevAttrMultiProcessorCount, ctx->device));
  return TQ_OK;
}

// The form that does a call soonest.  16-bit queries: few rows do best where their keys and values are decoded row
// tile by row tile (ROWS), many where they are decoded once into the operands of tcgen05 products (TILES); between
// them goes what was measured over 600 to 32768 tokens, 1 to 32 sequences and 4 to 32 KV heads.  With W tokens
// seen, times sequences and KV heads, in thousands, and tiles of eight rows, in microseconds (bfloat16 | float16):
//   ROWS 25 + (0.085 | 0.165) W tiles        TILES 50 + (0.42 | 0.64) W
// e.g. one sequence of 8192, 8 KV heads, bfloat16: 64 rows 68 against 76, 128 rows 108 against 77; of 32768: 32 rows
// 100 against 149, 64 rows 177 against 150; 8 of 8192: 204 against 264, 393 against 266.  ROWS is written for blocks of
// 256 tokens.  With others it is between TILES and, up to 64 rows, GENERAL:
//   GENERAL up to 16 rows 26 + 0.9 W, above 40 + 1.7 W
// (8 KV heads, bfloat16, GENERAL against TILES: one sequence, a window of 100: 4 rows 17 and 38, 64 rows 32 and 41; one
// of 1000: 4 rows 37 and 52, 32 rows 57 and 53, 64 rows 66 and 55; one of 4000: 61 and 58, 89 and 60, 98 and 61.)
// float32 queries, which TILES would round: ROWS up to 48 rows, GENERAL above (ROWS against GENERAL, four
// sequences of 8000, 8 KV heads: 32 rows 222 and 344, 48: 311 and 351, 64: 394 and 361, 128: 740 and 693; eight of 2000, 32
// KV heads: 32 rows 527 and 666, 64: 1100 and 729).
// Listed blocks differ from token to token: ROWS, where the blocks are those it is written for, tile of rows by tile.  The window is the
// same for all tokens of a sequence: WINDOW takes it in tiles of 16 rows instead, for a kernel more, where ROWS would spend more
// than 14 us on it by the above (27 x 8 heads of 5 x 8 rows, float16, 2 blocks: 210 us without, 141 with; 20 x 8 of 16 x 4 rows,
// bfloat16: 98 and 48; 8 x 4 of 5 x 7 rows, 24 blocks: 70 and 74; 1 x 8 of 4 rows, 16 blocks: 28 and 43).
Form choose(const tq_ctx* ctx, const Call* r, int n) {
  const tq_geom& g = ctx->g;
  const int rows = r->n_tokens * g.group;
  const bool channels = g.key_mode != TQ_KEYS_POLAR && !ctx->force_generic, blocks = g.block_tokens == 256;
  if (!channels) return GENERAL;
  const bool window = r->q_dtype != TQ_F32 && r->q_dtype == g.kv_dtype;
  if (r->listed) {
    const double w = (double)std::min(n, g.hot_window) * r->seq_count * g.n_kv_heads * r->n_tokens * ((g.group + 7) / 8) / 1000.0;
    return !blocks ? GENERAL : window && (r->q_dtype == TQ_F16 ? 0.165 : 0.085) * w > 14.0 ? WINDOW : ROWS;
  }
  // A shared beginning: SHARED, however many rows.  SHARED and TILES, the whole call, us, 8 KV heads of 4, by rows a head: bfloat16 on
  // 8192 tokens 256 rows 53 and 129, 1280 145 and 208, 2048 243 and 237, 4096 526 and 383, 32768 2942 and 1673; on 2000 tokens 2048
  // 120 and 170, 4096 297 and 273; on 32768 768 217 and 270, 2048 510 and 496, 4096 1080 and 848; float16 on 8192 512 119 and 173, 1280
  // 269 and 253, 4096 858 and 470.  So prompts behind a beginning, from some 2000 rows a head on (float16: 1000), wait for a rule.
  if (r->whole && blocks && r->q_dtype != TQ_F32) return SHARED;
  // (and the merge of its states with few rows: a window of their type, and what blocks the sequences have by the rows form)
  if (r->merges && blocks && rows <= 64 && window) return WINDOW;
  if (r->q_dtype == TQ_F32) return blocks && rows <= 48 ? ROWS : GENERAL;
  const double seen = r->window == 0 ? n : std::min((double)n, (double)r->window + r->n_tokens + r->sinks);
  const double w = seen * r->seq_count * g.n_kv_heads / 1000.0;
  const bool f16 = r->q_dtype == TQ_F16;
  const double tiles = 50.0 + (f16 ? 0.64 : 0.42) * w;
  if (!blocks) return rows <= 64 && (rows <= 16 ? 26.0 + 0.9 * w : 40.0 + 1.7 * w) <= tiles ? GENERAL : TILES;
  return 25.0 + (f16 ? 0.165 : 0.085) * w * ((rows + 7) / 8) <= tiles ? ROWS : TILES;
}

// Splits of the tokens: enough CTAs for the GPU, of what is visible in the longest sequence, in blocks and in
// the window.
Plan make_plan(const tq_ctx* ctx, const Call* r, cudaStream_t st) {
  const tq_geom& g = ctx->g;
  Plan p = {};
  p.seqs = INT_MAX;
  const int n = tq_most_tokens(ctx, r->layer, r->seq_begin, r->seq_count, st), rows = r->n_tokens * g.group;
  const int nb = n_cold_blocks(n, g.hot_window, g.block_tokens);
  p.form = choose(ctx, r, n);
  const int sm_count = ctx->sm_count;
  if (p.form == SHARED) {
    AttendArgs a = {};
    a.g = g;
    a.rows = rows;
    a.q_dtype = r->q_dtype;
    a.sm_count = sm_count;
    tq_attend_shared_plan(a, n, &a.ns_cold, &a.ns_hot);
    p.ns_cold = a.ns_cold, p.ns_hot = a.ns_hot;
    p.seq_bytes = tq_attend_shared_bytes(a);
    return p;
  }
  if (p.form == TILES) {
    constexpr int TILE = TQ_ATTEND_TILE;
    const int64_t all = std::max<int64_t>((n + TILE - 1) / TILE, 1);
    auto seen = [&](int64_t tokens) {  // tiles that so many neighbouring query tokens see
      return r->window == 0 ? all
                            : std::min<int64_t>(all, ((int64_t)r->window + tokens + 2 * TILE - 2) / TILE +
                                                         ((int64_t)r->sinks + TILE - 1) / TILE);
    };
    p.cap = (int)seen(r->n_tokens);
    // splits of a tile of rows: as many as bring the rounds of CTAs nearest to even (with four tiles' time for
    // what a CTA does besides)
    const int64_t each = seen(256 / g.group + 1), ctas = (int64_t)r->seq_count * g.n_kv_heads * ((rows + 255) / 256);
    int64_t best = INT64_MAX;
    for (int k = 1; k <= 32 && k <= each; ++k) {
      const int64_t time = (ctas * k + sm_count - 1) / sm_count * ((each + k - 1) / k + 4);
      if (time < best) best = time, p.splits = k;
    }
    AttendArgs a = {};
    a.g = g;
    a.rows = rows;
    a.q_dtype = r->q_dtype;
    p.seq_bytes = tq_attend_tiles_bytes(a, g.n_kv_heads, p.cap, p.splits);
    return p;
  }
  if (p.form == WINDOW && n <= g.hot_window) {  // no blocks
    p.seq_bytes = 256;
    return p;
  }
  if (p.form == ROWS || p.form == WINDOW) {
    AttendArgs a = {};
    a.no_window = p.form == WINDOW;
    a.g = g;
    a.rows = rows;
    a.seq_count = r->seq_count;
    a.n_tokens = r->n_tokens;
    a.window = r->window == 0 ? INT_MAX : r->window;
    a.sinks = r->sinks;
    a.q_dtype = r->q_dtype;
    a.sm_count = sm_count;
    a.n_list = r->n_list, a.listed = r->listed;
    const AttendRowsPlan rp = tq_attend_rows_plan(a, n);
    p.ns_cold = rp.ns_cold, p.ns_hot = rp.ns_hot, p.hot_cost = rp.hot_cost;
    p.seqs = rp.seqs;
    p.fixed_bytes = rp.plan_bytes;
    p.seq_bytes = (size_t)g.n_kv_heads * rows * (p.ns_cold + p.ns_hot) * TQ_PART_STRIDE * 4;
    return p;
  }
  const int row_tile = rows <= 16 || r->listed ? 16 : 64;
  constexpr int cold_size = 64, hot_size = 64;
  // tokens in blocks that the rows of a tile can see
  const int64_t in_blocks = (int64_t)nb * g.block_tokens;
  const int64_t seen = r->listed         ? std::min<int64_t>(in_blocks, (int64_t)r->n_list * g.block_tokens)
                       : r->window == 0 ? in_blocks
                                        : std::min<int64_t>(in_blocks, (int64_t)r->window + row_tile / g.group + r->sinks + cold_size);
  const int64_t cold = (seen + cold_size - 1) / cold_size;
  const int64_t hot = (std::min<int64_t>(g.hot_window, n) + hot_size - 1) / hot_size;
  const int64_t tiles = r->listed ? r->n_tokens : (rows + row_tile - 1) / row_tile;
  const int64_t ctas = std::max<int64_t>((int64_t)r->seq_count * g.n_kv_heads * tiles, 1);
  const int64_t want = std::min<int64_t>(std::max<int64_t>((4 * sm_count + ctas - 1) / ctas, 1), 64);
  const int64_t each = (std::max<int64_t>(cold + hot, 1) + want - 1) / want;
  p.ns_cold = (int)((cold + each - 1) / each);
  p.ns_hot = (int)std::max<int64_t>((hot + each - 1) / each, 1);
  // (the kernels go by the lengths on the device: blocks always have a split where there can be any)
  if (p.ns_cold == 0 && n_cold_blocks(g.max_tokens_per_seq, g.hot_window, g.block_tokens) > 0) p.ns_cold = 1;
  p.seq_bytes = (size_t)g.n_kv_heads * rows * (p.ns_cold + p.ns_hot) * TQ_PART_STRIDE * 4;
  return p;
}

size_t least_bytes(const Plan& p) { return p.fixed_bytes + p.seq_bytes; }

// The sequences of `r` by a plan that its workspace has room for, as many at once as it has.
int run(tq_ctx* ctx, const Call* r, const Plan& p, cudaStream_t st) {
  const tq_geom& g = ctx->g;
  const int at_once =
      (int)std::min({(r->workspace_bytes - p.fixed_bytes) / p.seq_bytes, (size_t)r->seq_count, (size_t)p.seqs});
  AttendArgs a = {};
  a.g = g;
  a.pages = (const uint8_t*)ctx->b.pages;
  a.hot_k = ctx->b.hot_k;
  a.hot_v = ctx->b.hot_v;
  a.pool_dec = (const uint32_t*)ctx->b.pool_dec;
  a.pool_val = (const uint16_t*)ctx->b.pool_val;
  a.page_meta = (const PageMeta*)ctx->b.page_meta;
  a.seq_len = (const int32_t*)((const uint8_t*)ctx->b.state + state_len_off(g));
  a.status = (int32_t*)((uint8_t*)ctx->b.state + state_status_off(g));
  a.tables = (const Tables*)ctx->b.tables;
  a.q_seq = r->q_seq_stride, a.q_tok = r->q_tok_stride, a.q_head = r->q_head_stride;
  a.plan = r->workspace;
  a.partials = (float*)((uint8_t*)r->workspace + p.fixed_bytes);
  a.layer = r->layer;
  a.n_tokens = r->n_tokens;
  a.q_dtype = r->q_dtype;
  a.window = r->window == 0 ? INT_MAX : r->window;
  a.sinks = r->sinks;
  a.ns_cold = p.ns_cold, a.ns_hot = p.ns_hot, a.hot_cost = p.hot_cost;
  a.rows = r->n_tokens * g.group;
  a.device = ctx->device, a.sm_count = ctx->sm_count;
  a.wait_limit = ctx->wait_limit, a.withhold = ctx->withhold_tile;
  a.unit_stride = (int64_t)a.rows * (p.ns_cold + p.ns_hot) * TQ_PART_STRIDE;
  a.n_list = r->n_list, a.listed = r->listed;
  a.whole = r->whole, a.states = r->states, a.before_rows = r->before_rows;
  for (int s = 0; s < r->seq_count; s += at_once) {
    const Call part = part_of(ctx, *r, s, std::min(at_once, r->seq_count - s));
    a.seq_begin = part.seq_begin, a.seq_count = part.seq_count;
    a.q = part.q, a.out = part.out, a.q_lens = part.q_lens, a.list = part.list, a.before = part.before, a.shared = part.shared;
    if (p.form == WINDOW) {
      a.no_window = 1;
      int rc = p.ns_cold > 0 ? tq_launch_attend_rows(a, st) : TQ_OK;
      if (rc == TQ_OK) rc = tq_launch_attend_window(a, TQ_ROWS_TILE, st);
      if (rc != TQ_OK) return rc;
      ctx->last_launches += p.ns_cold > 0 ? 2 : 1;
      continue;
    }
    if (p.form == SHARED) {
      SharedStates as;
      const int rc = tq_launch_attend_shared(a, r->workspace, r->keep == nullptr, &as, st);
      if (rc != TQ_OK) return rc;
      if (r->keep != nullptr) *r->keep = as;
      ctx->last_launches += r->keep != nullptr ? 2 : 3;
      continue;
    }
    if (p.form == TILES) {
      const int rc = tq_launch_attend_tiles(a, r->workspace, p.cap, p.splits, st);
      if (rc != TQ_OK) return rc;
      ctx->last_launches += 4;
      continue;
    }
    if (p.form == ROWS) {
      const int rc = tq_launch_attend_rows(a, st);
      if (rc != TQ_OK) return rc;
      ctx->last_launches += 2;
      continue;
    }
    int rc = tq_launch_attend_general(a, st);
    if (rc != TQ_OK) return rc;
    rc = tq_launch_attend_combine(a, st);
    if (rc != TQ_OK) return rc;
    ctx->last_launches += 2;
  }
  return TQ_OK;
}

int workspace_of(tq_ctx* ctx, const Call& r, void* stream, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_ERR_INVALID, "null argument");
  const Plan p = make_plan(ctx, &r, (cudaStream_t)stream);
  const size_t n = std::max<size_t>(AT_ONE_GO / std::max<size_t>(p.seq_bytes, 1), 1);
  *bytes = align_up(p.fixed_bytes + std::min({n, (size_t)r.seq_count, (size_t)p.seqs}) * p.seq_bytes, 256);
  return TQ_OK;
}

int attend(tq_ctx* ctx, const Call& r, void* stream) {
  if (r.seq_count == 0 || r.n_tokens == 0) return TQ_OK;
  TQ_REQUIRE(r.q != nullptr && r.out != nullptr, TQ_ERR_INVALID, "q and out must be device pointers");
  TQ_REQUIRE(r.workspace != nullptr && (uintptr_t)r.workspace % 256 == 0, TQ_ERR_INVALID,
             "workspace must be a device pointer aligned to 256 bytes");
  TQ_CUDA(cudaSetDevice(ctx->device));
  cudaStream_t st = (cudaStream_t)stream;
  const Plan all = make_plan(ctx, &r, st);
  if (r.workspace_bytes >= least_bytes(all)) {
    ctx->last_launches = 0;
    return run(ctx, &r, all, st);
  }
  // Even one sequence needs more in the form that suits all of them: half as many, planned by themselves, and so on
  // (another form may suit them).  Looked through before anything is launched.
  for (const bool launch : {false, true}) {
    if (launch) ctx->last_launches = 0;
    for (int s = 0, n = 0; s < r.seq_count; s += n) {
      n = r.seq_count - s;
      Plan p;
      for (;;) {
        const Call part = part_of(ctx, r, s, n);
        p = make_plan(ctx, &part, st);
        if (r.workspace_bytes >= least_bytes(p)) break;
        TQ_REQUIRE(n > 1, TQ_ERR_CAPACITY, "workspace smaller than tq_attend_workspace asks for one sequence");
        n = (n + 1) / 2;
      }
      if (!launch) continue;
      const Call part = part_of(ctx, r, s, n);
      const int rc = run(ctx, &part, p, st);
      if (rc != TQ_OK) return rc;
    }
  }
  return TQ_OK;
}

int check_listed(const tq_attend_args* r, const int32_t* blocks, int32_t n_blocks) {
  TQ_REQUIRE(r->window == 0 && r->sinks == 0, TQ_ERR_INVALID, "listed blocks take the place of a window");
  TQ_REQUIRE(n_blocks >= 0, TQ_ERR_INVALID, "n_blocks must not be negative");
  TQ_REQUIRE(blocks != nullptr || n_blocks == 0 || r->seq_count == 0 || r->n_tokens == 0, TQ_ERR_INVALID,
             "blocks must be a device pointer");
  return TQ_OK;
}

Call listed_call(const tq_attend_args* r, const int32_t* blocks, int32_t n_blocks) {
  Call c = plain_call(r);
  c.list = blocks, c.n_list = n_blocks, c.listed = true;
  return c;
}

// A call with a shared beginning, in two parts: the queries of all sequences as those of one, on the prefix, and the
// sequences' own tokens, whose merge takes the prefix's states in: one a row, or, where both parts have the forms that can,
// all of them as they are.
struct Shared {
  Call prefix, own;
  size_t states, of_prefix, of_own;  // bytes
  bool direct;                       // the states are not merged in between
};
int check_shared(const tq_ctx* ctx, const tq_attend_args* r, int32_t prefix) {
  TQ_REQUIRE(r->window == 0 && r->sinks == 0, TQ_ERR_INVALID, "a window and a shared beginning do not go together");
  TQ_REQUIRE(prefix >= 0 && prefix < ctx->g.n_seqs && (prefix < r->seq_begin || prefix >= r->seq_begin + r->seq_count),
             TQ_ERR_INVALID, "prefix must be a sequence of the context that is none of the call's own");
  TQ_REQUIRE((int64_t)r->seq_count * r->n_tokens * ctx->g.group <= (1 << 30), TQ_ERR_INVALID, "too many query tokens in a call");
  TQ_REQUIRE(r->seq_count <= 1 || r->n_tokens <= 1 || r->q_seq_stride == r->n_tokens * r->q_tok_stride, TQ_ERR_INVALID,
             "with a shared beginning the queries of a sequence must follow those of the one before");
  return TQ_OK;
}
// Sequences s .. s + n - 1 of the call
Shared shared_part(const tq_ctx* ctx, const tq_attend_args* r, int32_t prefix, int s, int n) {
  const tq_geom& g = ctx->g;
  Shared c;
  c.own = c.prefix = part_of(ctx, plain_call(r), s, n);
  const int tokens = n * r->n_tokens;
  Call& p = c.prefix;
  p.seq_begin = prefix, p.seq_count = 1, p.n_tokens = tokens;
  if (r->n_tokens == 1) p.q_tok_stride = r->q_seq_stride;
  p.q_lens = nullptr;
  p.whole = true;
  c.states = align_up((size_t)g.n_kv_heads * tokens * g.group * TQ_PART_STRIDE * 4, 256);
  c.own.before_rows = (int64_t)tokens * g.group;
  return c;
}
// Bytes of a part's workspace; where it is, and how the parts go together.
int shared_plan(tq_ctx* ctx, const tq_attend_args* r, cudaStream_t st, Shared* c) {
  c->own.merges = make_plan(ctx, &c->prefix, st).form == SHARED;
  int rc = workspace_of(ctx, c->prefix, st, &c->of_prefix);
  if (rc == TQ_OK) rc = workspace_of(ctx, c->own, st, &c->of_own);
  if (rc != TQ_OK) return rc;
  const Plan own = make_plan(ctx, &c->own, st);
  c->direct = c->own.merges && (own.form == ROWS || own.form == WINDOW) && c->of_own >= least_bytes(own);
  uint8_t* w = (uint8_t*)r->workspace;
  c->prefix.workspace = w, c->prefix.workspace_bytes = c->of_prefix;
  c->own.workspace = w + c->of_prefix, c->own.workspace_bytes = c->of_own;
  if (c->direct) {
    c->states = 0;
    return TQ_OK;
  }
  c->prefix.states = (float*)(w + c->of_prefix + c->of_own);
  c->own.before = c->prefix.states;
  return TQ_OK;
}
// Bytes that the call needs in rounds of n sequences.
int shared_bytes(tq_ctx* ctx, const tq_attend_args* r, int32_t prefix, int n, cudaStream_t st, size_t* bytes) {
  *bytes = 0;
  for (int s = 0; s < r->seq_count; s += n) {
    Shared c = shared_part(ctx, r, prefix, s, std::min(n, r->seq_count - s));
    const int rc = shared_plan(ctx, r, st, &c);
    if (rc != TQ_OK) return rc;
    *bytes = std::max(*bytes, c.of_prefix + c.of_own + c.states);
  }
  return TQ_OK;
}
// The most sequences a round for which `most` bytes do; one at least.
int shared_rounds(tq_ctx* ctx, const tq_attend_args* r, int32_t prefix, size_t most, cudaStream_t st, int* n, size_t* bytes) {
  *n = std::max(r->seq_count, 1);
  for (;; *n = (*n + 1) / 2) {
    const int rc = shared_bytes(ctx, r, prefix, *n, st, bytes);
    if (rc != TQ_OK || *bytes <= most || *n == 1) return rc;
  }
}

}  // namespace

extern "C" int32_t tq_attend_prefix_workspace(tq_ctx* ctx, const tq_attend_args* r, int32_t prefix, void* stream,
                                              size_t* bytes) {
  int rc = check_args(ctx, r);
  if (rc == TQ_OK) rc = check_shared(ctx, r, prefix);
  if (rc != TQ_OK) return rc;
  TQ_REQUIRE(bytes != nullptr, TQ_ERR_INVALID, "null argument");
  int n;
  return shared_rounds(ctx, r, prefix, AT_ONE_GO, (cudaStream_t)stream, &n, bytes);
}

extern "C" int32_t tq_attend_prefix(tq_ctx* ctx, const tq_attend_args* r, int32_t prefix, void* stream) {
  int rc = check_args(ctx, r);
  if (rc == TQ_OK) rc = check_shared(ctx, r, prefix);
  if (rc != TQ_OK || r->seq_count == 0 || r->n_tokens == 0) return rc;
  TQ_REQUIRE(r->workspace != nullptr && (uintptr_t)r->workspace % 256 == 0, TQ_ERR_INVALID,
             "workspace must be a device pointer aligned to 256 bytes");
  int n;
  size_t bytes;
  rc = shared_rounds(ctx, r, prefix, r->workspace_bytes, (cudaStream_t)stream, &n, &bytes);
  if (rc != TQ_OK) return rc;
  TQ_REQUIRE(bytes <= r->workspace_bytes, TQ_ERR_CAPACITY, "workspace smaller than tq_attend_prefix_workspace asks for one sequence");
  int launches = 0;
  for (int s = 0; s < r->seq_count; s += n) {
    Shared c = shared_part(ctx, r, prefix, s, std::min(n, r->seq_count - s));
    rc = shared_plan(ctx, r, (cudaStream_t)stream, &c);
    if (rc != TQ_OK) return rc;
    if (c.direct) c.prefix.keep = &c.own.shared;
    for (const Call* x : {&c.prefix, &c.own}) {
      rc = attend(ctx, *x, stream);
      if (rc != TQ_OK) return rc;
      launches += ctx->last_launches;
    }
  }
  ctx->last_launches = launches;
  return TQ_OK;
}

extern "C" int32_t tq_attend_workspace(tq_ctx* ctx, const tq_attend_args* r, void* stream, size_t* bytes) {
  const int rc = check_args(ctx, r);
  return rc != TQ_OK ? rc : workspace_of(ctx, plain_call(r), stream, bytes);
}

extern "C" int32_t tq_attend(tq_ctx* ctx, const tq_attend_args* r, void* stream) {
  const int rc = check_args(ctx, r);
  return rc != TQ_OK ? rc : attend(ctx, plain_call(r), stream);
}

extern "C" int32_t tq_attend_blocks_workspace(tq_ctx* ctx, const tq_attend_args* r, int32_t n_blocks, void* stream,
                                              size_t* bytes) {
  int rc = check_args(ctx, r);
  if (rc == TQ_OK) rc = check_listed(r, (const int32_t*)r, n_blocks);  // (pointers are not looked at)
  return rc != TQ_OK ? rc : workspace_of(ctx, listed_call(r, nullptr, n_blocks), stream, bytes);
}

extern "C" int32_t tq_attend_blocks(tq_ctx* ctx, const tq_attend_args* r, const int32_t* blocks, int32_t n_blocks,
                                    void* stream) {
  int rc = check_args(ctx, r);
  if (rc == TQ_OK) rc = check_listed(r, blocks, n_blocks);
  return rc != TQ_OK ? rc : attend(ctx, listed_call(r, blocks, n_blocks), stream);
}

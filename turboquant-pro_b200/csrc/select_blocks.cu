// Which blocks of a sequence a query token is worth attending, per KV head, by what the pages hold per channel anyway.
//
// A key of a block, outliers aside, lies on the block's grid: between mean + lo * scale and mean + hi * scale in every
// channel (NF4: lo, hi = -1, 1; uniform: 0, 15).  The score of a block is the sum over the group's query heads of the
// largest q . k that this allows,
//   sum_g sum_d max(q_gd (mu_d + lo s_d), q_gd (mu_d + hi s_d)) = sum_d (P_d + N_d) mu_d + (hi P_d + lo N_d) s_d,
// with P = sum_g max(q, 0), N = sum_g min(q, 0): two multiply-adds per channel, however large the group.  In 64
// bits, so that two blocks that are nearly as good come in the same order whoever adds them up, and their places do not depend on
// the order of a sum.
//
// A cluster of up to eight CTAs takes one (sequence, KV head) and up to eight query tokens: the CTAs divide the
// blocks, sixteen lanes two blocks and two tokens at a time, and leave the scores in the shared memory of the CTA that chooses
// for the token (in the workspace where they do not fit).  Up to 128 blocks are counted, a thread a block; of more the choice is
// a radix selection from the highest bit in which the scores differ on: the threshold, eight bits at a time, then
// the indices above it in order.
//
// What bounds it is not its bytes (a 28th of a page) but its own steps one after the other, each from a cold cache: the launch of
// a cluster, queries, blocks, choice.  8 heads of 31 blocks, one token: 7.3 us (2900 cycles to the queries' sums, 1800 for the
// scores, 2000 for the choice); 128 units of 3 to 127 blocks: 11.5 us; 16 units of 512 blocks, five tokens: 17.5 us, 24.3 with
// one block and one token at a time, where the sums were read from shared memory four times as often.
#include <cooperative_groups.h>

#include <algorithm>

#include "attend.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int SB_THREADS = 256, SB_WARPS = SB_THREADS / 32;
constexpr int SB_TOKENS = 8;                 // query tokens of a cluster
constexpr int SB_LANES = 16;                 // lanes of a block
constexpr int SB_SWEEP = 2 * SB_THREADS / SB_LANES;  // blocks of a CTA at once, two a thread
constexpr int SB_COUNTED = 128;              // blocks up to which the choice is by counting
constexpr size_t SB_SHARED = 96 * 1024;      // most bytes of queries and scores in shared memory

typedef unsigned long long u64;
constexpr u64 SB_ALWAYS = ~0ull;             // order key of a block that is chosen in any case

struct SelectArgs {
  tq_geom g;
  const uint8_t* pages;
  const int32_t* seq_len;  // of the layer
  tq_select_args r;
  double lo, hi;           // ends of the grid
  u64* scores;             // [cluster][token][cap], or null: shared memory
  int cap;                 // blocks that there is room for
  int tokens, groups, cluster;  // tokens of a cluster, groups of tokens, CTAs of a cluster
};

// ascending with the score; what is no number comes last
TQ_DEV u64 sb_key(double x) {
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return x == x ? (b >> 63 ? ~b : b | 1ull << 63) : 0ull;
}

// a channel's place in a row of 128: lane l of a block's 16 has channels 4 l + 0 .. 3 and 64 + 4 l + 0 .. 3, and what the 16 read
// at once is 256 bytes in a row
TQ_DEV int sb_place(int d) { return (d & 64) | (d & 2) << 4 | (d & 60) >> 1 | (d & 1); }

struct SelectShared {
  uint32_t hist[256];
  u64 most[SB_WARPS], least[SB_WARPS];
  uint32_t ties[SB_WARPS], taken[SB_WARPS];
  uint32_t digit, above, at;
  int own[SB_TOKENS];  // block of a token's position, or -1
};

// The n highest of keys[0 .. m), ties to the lowest index, their indices in order to out[0 .. n), and -1 behind them.
TQ_DEV void sb_choose(const u64* keys, int m, int n, int always, int32_t* out, SelectShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (m <= n) {
    for (int i = tid; i < n; i += SB_THREADS) out[i] = i < m ? i : -1;
    return;
  }
  if (m <= SB_COUNTED) {  // a thread a key: how many come before it
    const u64 mine = tid < m ? keys[tid] : 0ull;
    int before = 0;
    if (32 * warp < m) {
#pragma unroll 4
      for (int j = 0; j < m; ++j) {
        const u64 k = keys[j];
        before += k > mine || (k == mine && j < tid);
      }
    }
    const bool in = tid < m && before < n;
    const uint32_t of_in = __ballot_sync(0xffffffffu, in);
    __syncthreads();  // (the choice before has been read)
    if (lane == 0) sh.taken[warp] = __popc(of_in);
    __syncthreads();
    int to = __popc(of_in & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) to += sh.taken[w];
    if (in) out[to] = tid;
    return;
  }
  // chosen: (key & mask) above `prefix`, and of those at it the first `need`
  u64 mask = 0ull, prefix = 0ull;
  uint32_t need = n;
  if (always >= n) {
    mask = prefix = SB_ALWAYS;
  } else {
    need -= always;
    u64 most = 0ull, least = SB_ALWAYS;  // bits that any has, that all have
    for (int i = tid; i < m; i += SB_THREADS) {
      const u64 k = keys[i];
      if (k != SB_ALWAYS) most |= k, least &= k;
    }
    auto both = [](u64 x, auto f) { return (u64)f((uint32_t)(x >> 32)) << 32 | f((uint32_t)x); };
    most = both(most, [](uint32_t v) { return __reduce_or_sync(0xffffffffu, v); });
    least = both(least, [](uint32_t v) { return __reduce_and_sync(0xffffffffu, v); });
    __syncthreads();  // (the choice before has been read)
    if (lane == 0) sh.most[warp] = most, sh.least[warp] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SB_WARPS; ++w) most |= sh.most[w], least &= sh.least[w];
    int bits = 64 - __clzll((long long)(most ^ least));  // those above are all the same
    if (bits < 64) mask = ~0ull << bits, prefix = most & mask;
    while (bits > 0) {
      const int shift = max(bits - 8, 0);
      const u64 field = (1ull << (bits - shift)) - 1ull;
      if (tid < 256) sh.hist[tid] = 0u;
      __syncthreads();
      for (int i = tid; i < m; i += SB_THREADS) {
        const u64 k = keys[i];
        if (k != SB_ALWAYS && (k & mask) == prefix) atomicAdd(&sh.hist[k >> shift & field], 1u);
      }
      __syncthreads();
      if (warp == 0) {  // the digit with which the keys from the highest on reach `need`
        uint32_t mine[8], sum = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // lane 0 has the highest digits
          mine[j] = sh.hist[255 - 8 * lane - j];
          sum += mine[j];
        }
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        uint32_t before = upto - sum;
        if (before < need && need <= upto) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (before < need && need <= before + mine[j]) {
              sh.digit = 255 - 8 * lane - j, sh.above = before, sh.at = mine[j];
            }
            before += mine[j];
          }
        }
      }
      __syncthreads();
      need -= sh.above;
      prefix |= (u64)sh.digit << shift;
      mask |= field << shift;
      bits = shift;
      if (sh.at == need) break;  // all that are left are chosen
    }
  }
  uint32_t ties = 0u, taken = 0u;  // of the indices before these
  for (int i0 = 0; i0 < m; i0 += SB_THREADS) {
    const int i = i0 + tid;
    const u64 k = i < m ? keys[i] : 0ull;
    const bool over = i < m && ((k & mask) > prefix || (k == SB_ALWAYS && prefix != SB_ALWAYS));
    const bool tie = i < m && !over && (k & mask) == prefix;
    const uint32_t of_tie = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1u;
    __syncthreads();  // (those before have been read)
    if (lane == 0) sh.ties[warp] = __popc(of_tie);
    __syncthreads();
    uint32_t rank = ties + __popc(of_tie & below);
#pragma unroll
    for (int w = 0; w < SB_WARPS; ++w) {
      const uint32_t c = sh.ties[w];
      if (w < warp) rank += c;
      ties += c;
    }
    const bool in = over || (tie && rank < need);
    const uint32_t of_in = __ballot_sync(0xffffffffu, in);
    if (lane == 0) sh.taken[warp] = __popc(of_in);
    __syncthreads();
    uint32_t to = taken + __popc(of_in & below);
#pragma unroll
    for (int w = 0; w < SB_WARPS; ++w) {
      const uint32_t c = sh.taken[w];
      if (w < warp) to += c;
      taken += c;
    }
    if (in && to < (uint32_t)n) out[to] = i;
  }
}

template <int DT>
__global__ void __launch_bounds__(SB_THREADS, 2) select_blocks_kernel(SelectArgs a) {
  extern __shared__ __align__(16) uint8_t sb_smem[];
  __shared__ SelectShared sh;
  const tq_geom& g = a.g;
  const tq_select_args& r = a.r;
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = blockIdx.x % a.cluster, id = blockIdx.x / a.cluster;
  const int unit = id / a.groups, t0 = id % a.groups * a.tokens, tokens = min(a.tokens, r.n_tokens - t0);
  const int H = g.n_kv_heads, G = g.group, s = unit / H, head = unit % H, S = g.block_tokens;
  double* const of_mean = (double*)sb_smem;              // [tokens][128]: P + N
  double* const of_scale = of_mean + a.tokens * TQ_D;    // hi P + lo N
  u64* const mine = (u64*)(of_scale + a.tokens * TQ_D);  // scores of tokens rank, rank + cluster, ...
  // all of the queries on their way at once (a thread waits for a few heads of one token at a time)
  constexpr int LINES = TQ_D * (DT == TQ_F32 ? 4 : 2) / 64;
  for (int i = tid; i < tokens * G * LINES; i += SB_THREADS) {
    const int64_t at = (int64_t)s * r.q_seq_stride + (int64_t)(t0 + i / LINES / G) * r.q_tok_stride +
                       (int64_t)(head * G + i / LINES % G) * r.q_head_stride + i % LINES * (TQ_D / LINES);
    asm volatile("prefetch.global.L2 [%0];" ::"l"((const uint8_t*)r.q + at * (DT == TQ_F32 ? 4 : 2)));
  }
  const int n = a.seq_len[(size_t)r.layer * g.n_seqs + r.seq_begin + s];
  const int q_n = r.q_lens == nullptr ? r.n_tokens : min(max(r.q_lens[s], 0), r.n_tokens);
  const int nb = min(n_cold_blocks(n, g.hot_window, S), a.cap);
  // blocks that begin at a token's position or before
  auto position = [&](int t) { return t0 + t < q_n ? n - q_n + t0 + t : -1; };
  auto candidates = [&](int t) {
    const int p = position(t);
    return p < 0 ? 0 : min(nb, p / S + 1);
  };

  cg::cluster_group cluster = cg::this_cluster();
  auto there = cluster.barrier_arrive();  // (before another CTA's shared memory is written, it has to be there)
  // the first blocks' lines, on their way while the queries are summed (pages that there may be, whatever the length)
  const int sub = lane % SB_LANES;
  const uint8_t* const pages = a.pages + page_offset(g, r.layer, r.seq_begin + s, head, 0);
  float4 m4[2][2], s4[2][2];  // [block][channels]
  auto fetch = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* page = pages + (size_t)min(b + i * (SB_SWEEP / 2), a.cap - 1) * g.page_bytes + 16 * sub;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m4[i][j] = *(const float4*)(page + g.mean_off + 256 * j);
        s4[i][j] = *(const float4*)(page + g.scale_off + 256 * j);
      }
    }
  };
  if (g.max_blocks > 0) fetch(rank * SB_SWEEP + tid / SB_LANES);
  if (tid < tokens) sh.own[tid] = position(tid) < 0 ? -1 : position(tid) / S;
  // (a half-warp has 16 channels and every second head of the group)
#pragma unroll 2
  for (int i = tid; i < tokens * 2 * TQ_D; i += SB_THREADS) {
    const int t = i / (2 * TQ_D), d = i / 32 % 8 * 16 + lane % 16;
    const int64_t at = (int64_t)s * r.q_seq_stride + (int64_t)(t0 + t) * r.q_tok_stride +
                       (int64_t)(head * G) * r.q_head_stride + d;
    double up = 0.0, down = 0.0;
#pragma unroll 4
    for (int k = lane / 16; k < G; k += 2) {
      const float x = attend_ld(r.q, (size_t)(at + k * r.q_head_stride), DT);
      up += x > 0.0f ? (double)x : 0.0;
      down += x > 0.0f ? 0.0 : (double)x;
    }
    up += __shfl_xor_sync(0xffffffffu, up, 16), down += __shfl_xor_sync(0xffffffffu, down, 16);
    const int to = t * TQ_D + sb_place(d);
    if (lane < 16) of_mean[to] = up + down;
    else of_scale[to] = a.hi * up + a.lo * down;
  }
  __syncthreads();
  cluster.barrier_wait(std::move(there));

  // ---- scores: sixteen lanes two blocks
  auto scores_of = [&](int t) -> u64* {
    if (a.scores != nullptr) return a.scores + ((size_t)id * a.tokens + t) * a.cap;
    return (u64*)cluster.map_shared_rank(mine, t & (a.cluster - 1)) + (size_t)(t >> (31 - __clz(a.cluster))) * a.cap;
  };
  const int last = min(tokens, q_n - t0) - 1, most = last >= 0 ? candidates(last) : 0;
  for (int b0 = rank * SB_SWEEP; b0 < most; b0 += a.cluster * SB_SWEEP) {
    const int b = b0 + tid / SB_LANES;
    if (b0 != rank * SB_SWEEP) fetch(b);
    double md[2][8], sd[2][8];  // (converted once, not for each token)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        md[i][4 * j] = m4[i][j].x, md[i][4 * j + 1] = m4[i][j].y, md[i][4 * j + 2] = m4[i][j].z, md[i][4 * j + 3] = m4[i][j].w;
        sd[i][4 * j] = s4[i][j].x, sd[i][4 * j + 1] = s4[i][j].y, sd[i][4 * j + 2] = s4[i][j].z, sd[i][4 * j + 3] = s4[i][j].w;
      }
    // two tokens at a time: four sums, so that none waits for itself, from what is read of the queries once
#pragma unroll 1
    for (int t = 0; t < tokens; t += 2) {
      double x[2][2] = {};  // [block][token]
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = (k == 0 ? t : min(t + 1, tokens - 1)) * TQ_D + 32 * j + 2 * sub;
          const double2 u = *(const double2*)(of_mean + at), v = *(const double2*)(of_scale + at);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[i][k] = fma(u.x, md[i][2 * j], x[i][k]), x[i][k] = fma(u.y, md[i][2 * j + 1], x[i][k]);
            x[i][k] = fma(v.x, sd[i][2 * j], x[i][k]), x[i][k] = fma(v.y, sd[i][2 * j + 1], x[i][k]);
          }
        }
      // over the block's lanes; each half keeps a block, each quarter a token of it
      const int of_block = sub >> 3, of_token = sub >> 2 & 1;
      double y[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        y[k] = (of_block ? x[1][k] : x[0][k]) + __shfl_xor_sync(0xffffffffu, of_block ? x[0][k] : x[1][k], 8);
      double z = (of_token ? y[1] : y[0]) + __shfl_xor_sync(0xffffffffu, of_token ? y[0] : y[1], 4);
      z += __shfl_xor_sync(0xffffffffu, z, 2);
      z += __shfl_xor_sync(0xffffffffu, z, 1);
      const int at_t = t + of_token, at_b = b + of_block * (SB_SWEEP / 2);
      if ((sub & 3) == 0 && at_t < tokens && at_b < nb)
        scores_of(at_t)[at_b] = at_b < r.first || at_b == sh.own[at_t] ? SB_ALWAYS : sb_key(z);
    }
  }
  cluster.sync();

  // ---- the choice, the tokens divided over the CTAs
  for (int t = rank; t < tokens; t += a.cluster) {
    const int m = candidates(t), p = position(t), own = p >= 0 ? p / S : -1;
    const int first = min(r.first, m);
    const int always = first + (own >= first && own < m ? 1 : 0);
    int32_t* out = r.out + (((size_t)s * r.n_tokens + t0 + t) * H + head) * r.n_blocks;
    const u64* keys = a.scores != nullptr ? a.scores + ((size_t)id * a.tokens + t) * a.cap
                                          : mine + (size_t)(t / a.cluster) * a.cap;
    sb_choose(keys, m, r.n_blocks, always, out, sh);
  }
}

struct Plan {
  int cap, tokens, groups, cluster;
  bool shared;
  size_t shared_bytes, bytes;
};

int check_select(tq_ctx* ctx, const tq_select_args* r) {
  TQ_REQUIRE(ctx != nullptr && r != nullptr, TQ_ERR_INVALID, "null argument");
  const tq_geom& g = ctx->g;
  TQ_REQUIRE(g.key_mode != TQ_KEYS_POLAR, TQ_ERR_UNSUPPORTED, "blocks are selected by the keys' per-channel grids: polar keys have none");
  TQ_REQUIRE(r->layer >= 0 && r->layer < g.n_layers, TQ_ERR_INVALID, "bad layer");
  TQ_REQUIRE(r->seq_begin >= 0 && r->seq_count >= 0 && (int64_t)r->seq_begin + r->seq_count <= g.n_seqs,
             TQ_ERR_INVALID, "sequence range out of bounds");
  TQ_REQUIRE(r->n_tokens >= 0 && (int64_t)r->n_tokens * g.group <= (1 << 30), TQ_ERR_INVALID,
             "n_tokens out of range");
  TQ_REQUIRE(r->n_blocks >= 1, TQ_ERR_INVALID, "n_blocks must be at least 1");
  TQ_REQUIRE(r->first >= 0, TQ_ERR_INVALID, "first must not be negative");
  TQ_REQUIRE(r->q_dtype == TQ_F32 || r->q_dtype == TQ_F16 || r->q_dtype == TQ_BF16, TQ_ERR_INVALID, "bad q_dtype");
  if (ctx->sm_count == 0)
    TQ_CUDA(cudaDeviceGetAttribute(&ctx->sm_count, cudaDevAttrMultiProcessorCount, ctx->device));
  return TQ_OK;
}

Plan make_plan(const tq_ctx* ctx, const tq_select_args* r, cudaStream_t st) {
  const tq_geom& g = ctx->g;
  Plan p;
  p.cap = std::max(n_cold_blocks(tq_most_tokens(ctx, r->layer, r->seq_begin, r->seq_count, st), g.hot_window, g.block_tokens), 1);
  p.tokens = std::min(std::max(r->n_tokens, 1), SB_TOKENS);
  p.groups = (r->n_tokens + p.tokens - 1) / p.tokens;
  // as many CTAs a cluster as have blocks to score and the GPU has room for, two an SM
  const int64_t clusters = (int64_t)r->seq_count * g.n_kv_heads * p.groups;
  p.cluster = 1;
  while (p.cluster < 8 && p.cluster * SB_SWEEP < p.cap && clusters * p.cluster * 2 <= 2 * ctx->sm_count) p.cluster *= 2;
  const size_t queries = (size_t)p.tokens * TQ_D * 2 * sizeof(double);
  const size_t keys = (size_t)((p.tokens + p.cluster - 1) / p.cluster) * p.cap * sizeof(u64);
  p.shared = queries + keys <= SB_SHARED;
  p.shared_bytes = queries + (p.shared ? keys : 0);
  p.bytes = p.shared ? 0 : (size_t)clusters * p.tokens * p.cap * sizeof(u64);
  return p;
}

template <int DT>
int launch(const tq_ctx* ctx, const SelectArgs& a, const Plan& p, int grid, cudaStream_t st) {
  static bool done[64];
  const int rc = attend_shared(select_blocks_kernel<DT>, SB_SHARED, ctx->device, done);
  if (rc != TQ_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(SB_THREADS);
  cfg.dynamicSmemBytes = p.shared_bytes;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TQ_CUDA(cudaLaunchKernelEx(&cfg, select_blocks_kernel<DT>, a));
  return TQ_OK;
}

}  // namespace

extern "C" int32_t tq_select_blocks_workspace(tq_ctx* ctx, const tq_select_args* r, void* stream, size_t* bytes) {
  const int rc = check_select(ctx, r);
  if (rc != TQ_OK) return rc;
  TQ_REQUIRE(bytes != nullptr, TQ_ERR_INVALID, "null argument");
  *bytes = make_plan(ctx, r, (cudaStream_t)stream).bytes;
  return TQ_OK;
}

extern "C" int32_t tq_select_blocks(tq_ctx* ctx, const tq_select_args* r, void* stream) {
  const int rc = check_select(ctx, r);
  if (rc != TQ_OK) return rc;
  if (r->seq_count == 0 || r->n_tokens == 0) return TQ_OK;
  const tq_geom& g = ctx->g;
  TQ_REQUIRE(r->q != nullptr && r->out != nullptr, TQ_ERR_INVALID, "q and out must be device pointers");
  cudaStream_t st = (cudaStream_t)stream;
  const Plan p = make_plan(ctx, r, st);
  TQ_REQUIRE(p.bytes == 0 || (r->workspace != nullptr && (uintptr_t)r->workspace % 256 == 0), TQ_ERR_INVALID,
             "workspace must be a device pointer aligned to 256 bytes");
  TQ_REQUIRE(r->workspace_bytes >= p.bytes, TQ_ERR_CAPACITY, "workspace smaller than tq_select_blocks_workspace asks for");
  const int64_t grid = (int64_t)r->seq_count * g.n_kv_heads * p.groups * p.cluster;
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (sequence, head, query token) items in a call");
  TQ_CUDA(cudaSetDevice(ctx->device));
  SelectArgs a;
  a.g = g;
  a.pages = (const uint8_t*)ctx->b.pages;
  a.seq_len = (const int32_t*)((const uint8_t*)ctx->b.state + state_len_off(g));
  a.r = *r;
  a.lo = g.key_mode == TQ_KEYS_UNIFORM ? 0.0 : -1.0, a.hi = g.key_mode == TQ_KEYS_UNIFORM ? 15.0 : 1.0;
  a.scores = p.shared ? nullptr : (u64*)r->workspace;
  a.cap = p.cap, a.tokens = p.tokens, a.groups = p.groups, a.cluster = p.cluster;
  const int rc2 = r->q_dtype == TQ_F32 ? launch<TQ_F32>(ctx, a, p, (int)grid, st)
                  : r->q_dtype == TQ_F16 ? launch<TQ_F16>(ctx, a, p, (int)grid, st)
                                         : launch<TQ_BF16>(ctx, a, p, (int)grid, st);
  if (rc2 != TQ_OK) return rc2;
  ctx->last_launches = 1;
  return TQ_OK;
}

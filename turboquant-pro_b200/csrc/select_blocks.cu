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
// blocks, eight lanes a block (a 128-byte line of scales, one of zero-points at a time, for all tokens), and leave the scores
// in the shared memory of the CTA that chooses for the token (in the workspace where they do not fit).  The choice is
// a radix selection from the highest bit in which the scores differ on: the threshold, eight bits at a time,
// then the indices above it in order.
#include <cooperative_groups.h>

#include <algorithm>

#include "attend.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int SB_THREADS = 256, SB_WARPS = SB_THREADS / 32;
constexpr int SB_TOKENS = 8;                 // query tokens of a cluster
constexpr int SB_LANES = 8;                  // lanes of a block
constexpr int SB_SWEEP = SB_THREADS / SB_LANES;  // blocks of a CTA at once
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

struct SelectShared {
  uint32_t hist[256];
  u64 most[SB_WARPS], least[SB_WARPS];
  uint32_t ties[SB_WARPS], taken[SB_WARPS];
  uint32_t digit, above, at;
};

// The n highest of keys[0 .. m), ties to the lowest index, their indices in order to out[0 .. n), and -1 behind them.
TQ_DEV void sb_choose(const u64* keys, int m, int n, int always, int32_t* out, SelectShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (m <= n) {
    for (int i = tid; i < n; i += SB_THREADS) out[i] = i < m ? i : -1;
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
      sh.hist[tid] = 0u;
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
  const int n = a.seq_len[(size_t)r.layer * g.n_seqs + r.seq_begin + s];
  const int q_n = r.q_lens == nullptr ? r.n_tokens : min(max(r.q_lens[s], 0), r.n_tokens);
  const int nb = min(n_cold_blocks(n, g.hot_window, S), a.cap);
  // blocks that begin at a token's position or before
  auto position = [&](int t) { return t0 + t < q_n ? n - q_n + t0 + t : -1; };
  auto candidates = [&](int t) {
    const int p = position(t);
    return p < 0 ? 0 : min(nb, p / S + 1);
  };

  for (int i = tid; i < tokens * TQ_D; i += SB_THREADS) {
    const int t = i / TQ_D, d = i % TQ_D;
    const int64_t at = (int64_t)s * r.q_seq_stride + (int64_t)(t0 + t) * r.q_tok_stride +
                       (int64_t)(head * G) * r.q_head_stride + d;
    double up = 0.0, down = 0.0;
    for (int k = 0; k < G; ++k) {
      const float x = attend_ld(r.q, (size_t)(at + k * r.q_head_stride), r.q_dtype);
      up += x > 0.0f ? (double)x : 0.0;
      down += x > 0.0f ? 0.0 : (double)x;
    }
    of_mean[i] = up + down;
    of_scale[i] = a.hi * up + a.lo * down;
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();  // (every CTA of the cluster is there)

  // ---- scores: eight lanes a block
  auto scores_of = [&](int t) -> u64* {
    if (a.scores != nullptr) return a.scores + ((size_t)id * a.tokens + t) * a.cap;
    return (u64*)cluster.map_shared_rank(mine, t % a.cluster) + (size_t)(t / a.cluster) * a.cap;
  };
  const int last = min(tokens, q_n - t0) - 1, most = last >= 0 ? candidates(last) : 0;
  const int sub = lane % SB_LANES;
  for (int b0 = rank * SB_SWEEP; b0 < most; b0 += a.cluster * SB_SWEEP) {
    const int b = b0 + tid / SB_LANES;
    const uint8_t* page = a.pages + page_offset(g, r.layer, r.seq_begin + s, head, min(b, nb - 1));
    float4 m4[4], s4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m4[j] = *(const float4*)(page + g.mean_off + (32 * j + 4 * sub) * 4);
      s4[j] = *(const float4*)(page + g.scale_off + (32 * j + 4 * sub) * 4);
    }
    for (int t = 0; t < tokens; ++t) {
      double x = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double2* u = (const double2*)(of_mean + t * TQ_D + 32 * j + 4 * sub);
        const double2* v = (const double2*)(of_scale + t * TQ_D + 32 * j + 4 * sub);
        const double2 u0 = u[0], u1 = u[1], v0 = v[0], v1 = v[1];
        x = fma(u0.x, (double)m4[j].x, x), x = fma(u0.y, (double)m4[j].y, x);
        x = fma(u1.x, (double)m4[j].z, x), x = fma(u1.y, (double)m4[j].w, x);
        x = fma(v0.x, (double)s4[j].x, x), x = fma(v0.y, (double)s4[j].y, x);
        x = fma(v1.x, (double)s4[j].z, x), x = fma(v1.y, (double)s4[j].w, x);
      }
#pragma unroll
      for (int o = 1; o < SB_LANES; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (sub == 0 && b < nb) {
        const int p = position(t);
        scores_of(t)[b] = b < r.first || b == p / S ? SB_ALWAYS : sb_key(x);
      }
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
  static bool done[64];
  const int rc2 = attend_shared(select_blocks_kernel, SB_SHARED, ctx->device, done);
  if (rc2 != TQ_OK) return rc2;
  SelectArgs a;
  a.g = g;
  a.pages = (const uint8_t*)ctx->b.pages;
  a.seq_len = (const int32_t*)((const uint8_t*)ctx->b.state + state_len_off(g));
  a.r = *r;
  a.lo = g.key_mode == TQ_KEYS_UNIFORM ? 0.0 : -1.0, a.hi = g.key_mode == TQ_KEYS_UNIFORM ? 15.0 : 1.0;
  a.scores = p.shared ? nullptr : (u64*)r->workspace;
  a.cap = p.cap, a.tokens = p.tokens, a.groups = p.groups, a.cluster = p.cluster;
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
  TQ_CUDA(cudaLaunchKernelEx(&cfg, select_blocks_kernel, a));
  ctx->last_launches = 1;
  return TQ_OK;
}

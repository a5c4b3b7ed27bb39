// Root-mean-square norm of every query and key head and the rotation by the token's position, in one pass:
//   y = x * rsqrt(mean x^2 + eps) * weight        (x itself without a weight)
//   channels i and i + r/2 (i < r/2) turn by  position * inv_freq[i]
// what a model does to q and k between their projections and the cache.
//
// A warp holds a head: four channels a lane, loaded and stored as one 8- or 16-byte word; the sum of squares
// is five shuffles, the partner channels come from the lane r/8 further.  The angles of a token are the same
// for all heads, so a CTA takes one token and forms them once: position * inv_freq / 2 pi in 64 bits, of which
// only the fraction counts (a 32-bit angle of position 10^6 is off by 0.06), then one sincospi in float32.
// Sums, norm and rotation are float32, rounded once.
//
// Bound by memory for prompts, by launch and latency for single tokens.
#include "common.cuh"

namespace {

constexpr int NR_THREADS = 256;

struct RopeArgs {
  tq_rope r;
  const int32_t* seq_len;  // positions of the tokens that follow what is stored; null: r.positions
};

// elements 4 * lane .. + 3 of a row
template <int DT>
TQ_DEV void nr_load(const void* row, int64_t at, bool vec, float (&x)[4]) {
  using T = typename Elem<DT>::type;
  const T* p = (const T*)row + at;
  if constexpr (DT == TQ_F32) {
    if (vec) {
      const float4 v = *(const float4*)p;
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      return;
    }
  } else if (vec) {
    const uint2 v = *(const uint2*)p;
    const T* e = (const T*)&v;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Elem<DT>::ld(e, i);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = Elem<DT>::ld(p, i);
}
TQ_DEV float nr_round(float x, float*) { return x; }
TQ_DEV __half nr_round(float x, __half*) { return __float2half_rn(x); }
TQ_DEV __nv_bfloat16 nr_round(float x, __nv_bfloat16*) { return __float2bfloat16_rn(x); }
template <int DT>
TQ_DEV void nr_store(void* row, int64_t at, const float (&x)[4]) {
  using T = typename Elem<DT>::type;
  struct alignas(4 * sizeof(T)) V4 { T v[4]; } v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = nr_round(x[i], (T*)nullptr);
  *(V4*)((T*)row + at) = v;
}
TQ_DEV float nr_weight(const void* w, int i, int dt) {
  if (dt == TQ_F32) return ((const float*)w)[i];
  if (dt == TQ_F16) return __half2float(((const __half*)w)[i]);
  return __bfloat162float(((const __nv_bfloat16*)w)[i]);
}

template <int DT>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(RopeArgs a, int vec) {
  __shared__ __align__(16) float cos_s[TQ_D / 2], sin_s[TQ_D / 2];
  const tq_rope& r = a.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int s = blockIdx.x / r.n_tokens, t = blockIdx.x % r.n_tokens;
  const int half = r.rotary_dim / 2, heads = r.n_q_heads + r.n_kv_heads;
  constexpr int N = 4;  // heads of a warp in flight
  float x[N][4];
  auto row_of = [&](int h, int64_t& at) -> const void* {
    const bool is_q = h < r.n_q_heads;
    at = is_q ? (int64_t)s * r.q_seq_stride + (int64_t)t * r.q_tok_stride + (int64_t)h * r.q_head_stride
              : (int64_t)s * r.k_seq_stride + (int64_t)t * r.k_tok_stride +
                    (int64_t)(h - r.n_q_heads) * r.k_head_stride;
    at += 4 * lane;
    return is_q ? r.q : r.k;
  };
  auto fetch = [&](int h0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + i * (NR_THREADS / 32);
      if (h < heads) {
        int64_t at;
        const void* row = row_of(h, at);
        nr_load<DT>(row, at, vec, x[i]);
      }
    }
  };
  fetch(warp);  // (the loads are on their way while the angles are formed)
  if (tid < half) {
    int64_t p;
    if (a.seq_len != nullptr) p = (int64_t)a.seq_len[s] + t;
    else {
      const int64_t at = (int64_t)s * r.pos_seq_stride + (int64_t)t * r.pos_tok_stride;
      p = r.pos_bits == 64 ? ((const int64_t*)r.positions)[at] : (int64_t)((const int32_t*)r.positions)[at];
    }
    const double turns = (double)p * ((double)r.inv_freq[tid] * 0.15915494309189533577);
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    cos_s[tid] = cs;
    sin_s[tid] = sn;
  }
  float wq[4], wk[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wq[i] = r.q_weight != nullptr ? nr_weight(r.q_weight, 4 * lane + i, r.weight_dtype) : 1.0f;
    wk[i] = r.k_weight != nullptr ? nr_weight(r.k_weight, 4 * lane + i, r.weight_dtype) : 1.0f;
  }
  __syncthreads();
  // this lane's channels: the first ones of their pairs, the second ones, or not turned at all
  const int ch = 4 * lane;
  const bool low = ch < half, turns = ch < 2 * half;
  const int pair = turns ? (low ? ch : ch - half) : 0, other = turns ? (low ? lane + half / 4 : lane - half / 4) : lane;
  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = turns ? cos_s[pair + i] : 1.0f;
    sn[i] = turns ? (low ? -sin_s[pair + i] : sin_s[pair + i]) : 0.0f;
  }
  for (int h0 = warp; h0 < heads; h0 += N * (NR_THREADS / 32)) {
    if (h0 != warp) fetch(h0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + i * (NR_THREADS / 32);
      if (h >= heads) break;  // (the whole warp)
      const bool is_q = h < r.n_q_heads;
      if ((is_q ? r.q_weight : r.k_weight) != nullptr) {
        float ss = (x[i][0] * x[i][0] + x[i][1] * x[i][1]) + (x[i][2] * x[i][2] + x[i][3] * x[i][3]);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float f = 1.0f / sqrtf(ss * (1.0f / TQ_D) + r.eps);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[i][c] *= f * (is_q ? wq[c] : wk[c]);
      }
      float y[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float z = __shfl_sync(0xffffffffu, x[i][c], other);
        y[c] = turns ? fmaf(x[i][c], cs[c], z * sn[c]) : x[i][c];
      }
      const int64_t tok = (int64_t)s * r.n_tokens + t;
      if (is_q) nr_store<DT>(r.q_out, (tok * r.n_q_heads + h) * TQ_D + 4 * lane, y);
      else nr_store<DT>(r.k_out, (tok * r.n_kv_heads + h - r.n_q_heads) * TQ_D + 4 * lane, y);
    }
  }
}

int check_rope(const tq_rope* r, bool stored) {
  TQ_REQUIRE(r != nullptr, TQ_ERR_INVALID, "null argument");
  TQ_REQUIRE(r->n_seqs >= 0 && r->n_tokens >= 0, TQ_ERR_INVALID, "n_seqs and n_tokens must not be negative");
  TQ_REQUIRE(r->n_q_heads >= 0 && r->n_kv_heads >= 0 && (int64_t)r->n_q_heads + r->n_kv_heads <= 1 << 20,
             TQ_ERR_INVALID, "head counts out of range");
  TQ_REQUIRE(r->dtype == TQ_F32 || r->dtype == TQ_F16 || r->dtype == TQ_BF16, TQ_ERR_INVALID, "bad dtype");
  TQ_REQUIRE(r->weight_dtype == TQ_F32 || r->weight_dtype == TQ_F16 || r->weight_dtype == TQ_BF16,
             TQ_ERR_INVALID, "bad weight_dtype");
  TQ_REQUIRE(r->rotary_dim >= 0 && r->rotary_dim <= TQ_D && r->rotary_dim % 8 == 0, TQ_ERR_UNSUPPORTED,
             "rotary_dim must be a multiple of 8, at most 128");
  TQ_REQUIRE(r->eps >= 0.0f, TQ_ERR_INVALID, "eps must not be negative");
  TQ_REQUIRE((int64_t)r->n_seqs * r->n_tokens <= INT32_MAX, TQ_ERR_UNSUPPORTED,
             "more than 2^31 - 1 tokens in a call");
  if (r->n_seqs == 0 || r->n_tokens == 0) return TQ_OK;
  TQ_REQUIRE((r->n_q_heads == 0 || (r->q && r->q_out)) && (r->n_kv_heads == 0 || (r->k && r->k_out)),
             TQ_ERR_INVALID, "q, k and their outputs must be device pointers");
  TQ_REQUIRE(r->rotary_dim == 0 || r->inv_freq, TQ_ERR_INVALID, "inv_freq must be a device pointer");
  TQ_REQUIRE(r->rotary_dim == 0 || stored || (r->positions && (r->pos_bits == 32 || r->pos_bits == 64)),
             TQ_ERR_INVALID, "positions must be a device pointer to 32- or 64-bit integers");
  TQ_REQUIRE(((uintptr_t)r->q_out | (uintptr_t)r->k_out) % (4 * elem_size(r->dtype)) == 0, TQ_ERR_INVALID,
             "q_out and k_out must be aligned to four elements");
  return TQ_OK;
}

int launch(const tq_rope* r, const int32_t* seq_len, cudaStream_t st) {
  const int64_t tokens = (int64_t)r->n_seqs * r->n_tokens;
  if (tokens == 0 || r->n_q_heads + r->n_kv_heads == 0) return TQ_OK;
  const int word = 4 * elem_size(r->dtype);
  const bool vec = ((uintptr_t)r->q | (uintptr_t)r->k) % word == 0 &&
                   ((r->q_seq_stride | r->q_tok_stride | r->q_head_stride | r->k_seq_stride |
                     r->k_tok_stride | r->k_head_stride) & 3) == 0;
  RopeArgs a = {*r, seq_len};
  switch (r->dtype) {
    case TQ_F32: norm_rope_kernel<TQ_F32><<<(int)tokens, NR_THREADS, 0, st>>>(a, vec); break;
    case TQ_F16: norm_rope_kernel<TQ_F16><<<(int)tokens, NR_THREADS, 0, st>>>(a, vec); break;
    default: norm_rope_kernel<TQ_BF16><<<(int)tokens, NR_THREADS, 0, st>>>(a, vec); break;
  }
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

}  // namespace

extern "C" int32_t tq_norm_rope(const tq_rope* r, int32_t device, void* stream) {
  const int rc = check_rope(r, false);
  if (rc != TQ_OK) return rc;
  TQ_CUDA(cudaSetDevice(device));
  return launch(r, nullptr, (cudaStream_t)stream);
}

extern "C" int32_t tq_ctx_norm_rope(tq_ctx* ctx, int32_t layer, int32_t seq_begin, const tq_rope* r,
                                    void* stream) {
  TQ_REQUIRE(ctx != nullptr && layer >= 0 && layer < ctx->g.n_layers, TQ_ERR_INVALID, "bad context or layer");
  const int rc = check_rope(r, true);
  if (rc != TQ_OK) return rc;
  const tq_geom& g = ctx->g;
  TQ_REQUIRE(r->n_q_heads == g.n_q_heads && r->n_kv_heads == g.n_kv_heads, TQ_ERR_INVALID,
             "head counts do not match the context");
  TQ_REQUIRE(seq_begin >= 0 && r->n_seqs >= 0 && (int64_t)seq_begin + r->n_seqs <= g.n_seqs, TQ_ERR_INVALID,
             "sequence range out of bounds");
  TQ_CUDA(cudaSetDevice(ctx->device));
  const int32_t* len = (const int32_t*)((const uint8_t*)ctx->b.state + state_len_off(g)) +
                       (size_t)layer * g.n_seqs + seq_begin;
  return launch(r, len, (cudaStream_t)stream);
}

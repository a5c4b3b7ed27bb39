// Root-mean-square norm of every query and key head and the rotation by the token's position, in one pass:
//   y = x * rsqrt(mean x^2 + eps) * weight        (x itself without a weight)
//   channels i and i + r/2 (i < r/2) turn by  position * inv_freq[i]
// what a model does to q and k between their projections and the cache.
//
// A lane holds 16 bytes of a head, so a warp two heads of 16-bit elements or one of float32.  The sum of squares
// goes over the head's lanes with shuffles; the partner channels come, still packed, from the lane half a
// rotation further.  What a token's heads have in common is formed once per token: position * inv_freq / 2 pi in
// 64 bits, of which only the fraction counts (a 32-bit angle of position 10^6 is off by 0.06), one sincospi in
// float32, and the weights times cosines and sines, so that a channel costs two multiply-adds.  Sums, norm and
// rotation are float32, rounded once.
//
// Positions of several axes (time, height, width): every frequency has the number of the axis whose position it goes
// by, one more load per angle.
//
// A CTA of eight warps takes one token of few, or up to eight, a warp each, whose angles are one step of the CTA.
// Bound by launch and latency for single tokens (4 us); for prompts by reading and writing q and k, at 68 to 80 % of
// a plain copy's rate (8 x 2048 tokens of 32 + 8 heads, bfloat16: 75 us, 4.5 TB/s), and the unpacking, shuffles and
// packing between them.
#include <atomic>

#include "common.cuh"

namespace {

constexpr int NR_THREADS = 256;

struct RopeArgs {
  tq_rope r;
  const int32_t* seq_len;  // positions of the tokens that follow what is stored; null: r.positions
  const int32_t* before;   // and behind so many tokens of a prefix (null: none)
  tq_rope_axes x;          // x.axes null: a position each
};

TQ_DEV float nr_weight(const void* w, int i, int dt) {
  if (dt == TQ_F32) return ((const float*)w)[i];
  if (dt == TQ_F16) return __half2float(((const __half*)w)[i]);
  return __bfloat162float(((const __nv_bfloat16*)w)[i]);
}
// two float32 at once
TQ_DEV uint64_t nr_f2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
TQ_DEV uint64_t nr_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
TQ_DEV uint64_t nr_mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// the elements of a 16-byte word
template <int DT>
TQ_DEV void nr_unpack(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == TQ_F32) {
      x[i] = __uint_as_float(w[i]);
    } else if (DT == TQ_F16) {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int DT>
TQ_DEV uint4 nr_pack(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == TQ_F32) {
      w[i] = __float_as_uint(x[i]);
    } else if (DT == TQ_F16) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *(const uint32_t*)&h;
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *(const uint32_t*)&h;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 16 bytes of a row, by elements where rows may lie anywhere
template <int DT, bool VEC>
TQ_DEV uint4 nr_load(const typename Elem<DT>::type* p) {
  using T = typename Elem<DT>::type;
  if constexpr (VEC) {
    return *(const uint4*)p;
  } else {
    union { uint4 v; T e[16 / sizeof(T)]; } u;
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) u.e[i] = p[i];
    return u.v;
  }
}

// A head's elements as one lane holds them: 16 bytes, with what the lane knows of them.
template <int DT>
struct NrLane {
  static constexpr int E = 16 / (int)sizeof(typename Elem<DT>::type);
  static constexpr int LPH = TQ_D / E, HPW = 32 / LPH;  // lanes of a head, heads of a warp
  int lane, hl, ch, half, partner;
  bool low, turned;
  float own[E], other[E];  // y = f * (x * own + partner * other), f the norm's factor
};

// PAIRED: a lane's partner channels are all of one lane (half the rotation is a multiple of a lane's channels);
// otherwise they come one by one.
template <int DT, bool PAIRED>
TQ_DEV void nr_factors(NrLane<DT>& n, const float* w, const float* cos_s, const float* sin_s) {
  constexpr int E = NrLane<DT>::E;
  if (PAIRED) {
    const int pr = n.turned ? (n.low ? n.ch : n.ch - n.half) : 0, oc = n.turned ? (n.low ? n.ch + n.half : n.ch - n.half) : n.ch;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 c4 = *(const float4*)(cos_s + pr + i), s4 = *(const float4*)(sin_s + pr + i);
      const float4 w4 = *(const float4*)(w + n.ch + i), o4 = *(const float4*)(w + oc + i);
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
      const float a[4] = {w4.x, w4.y, w4.z, w4.w}, o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        n.own[i + j] = n.turned ? a[j] * c[j] : a[j];
        n.other[i + j] = n.turned ? (n.low ? -s[j] : s[j]) * o[j] : 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = n.ch + i;
      const bool lo = c < n.half, in = c < 2 * n.half;
      const int pr = in ? (lo ? c : c - n.half) : 0, oc = in ? (lo ? c + n.half : c - n.half) : c;
      n.own[i] = in ? w[c] * cos_s[pr] : w[c];
      n.other[i] = in ? (lo ? -sin_s[pr] : sin_s[pr]) * w[oc] : 0.0f;
    }
  }
}
template <int DT, bool PAIRED>
TQ_DEV uint4 nr_head(const NrLane<DT>& n, const uint4& raw, bool normed, float eps) {
  constexpr int E = NrLane<DT>::E, LPH = NrLane<DT>::LPH;
  float x[E], z[E], y[E];
  nr_unpack<DT>(raw, x);
  float f = 1.0f;
  if (normed) {
    uint64_t sq = 0ull;
#pragma unroll
    for (int c = 0; c < E; c += 2) sq = nr_fma2(nr_f2(x[c], x[c + 1]), nr_f2(x[c], x[c + 1]), sq);
    float ss = __uint_as_float((uint32_t)sq) + __uint_as_float((uint32_t)(sq >> 32));
#pragma unroll
    for (int d = LPH / 2; d >= 1; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    f = rsqrtf(fmaf(ss, 1.0f / TQ_D, eps));
  }
  if (PAIRED) {
    uint4 o;
    o.x = __shfl_sync(0xffffffffu, raw.x, n.partner), o.y = __shfl_sync(0xffffffffu, raw.y, n.partner);
    o.z = __shfl_sync(0xffffffffu, raw.z, n.partner), o.w = __shfl_sync(0xffffffffu, raw.w, n.partner);
    if (!n.turned) o = make_uint4(0u, 0u, 0u, 0u);
    nr_unpack<DT>(o, z);
  } else {
#pragma unroll
    for (int c = 0; c < E; ++c) {
      // the channel's partner: element (oc % E) of its lane, whichever that is
      const int d = n.ch + c, oc = d < n.half ? d + n.half : d < 2 * n.half ? d - n.half : d;
      z[c] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = __shfl_sync(0xffffffffu, x[e], n.hl * LPH + oc / E);
        if (oc % E == e && d < 2 * n.half) z[c] = v;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < E; c += 2) {
    const uint64_t v = nr_mul2(nr_f2(f, f), nr_fma2(nr_f2(x[c], x[c + 1]), nr_f2(n.own[c], n.own[c + 1]),
                                                    nr_mul2(nr_f2(z[c], z[c + 1]), nr_f2(n.other[c], n.other[c + 1]))));
    y[c] = __uint_as_float((uint32_t)v), y[c + 1] = __uint_as_float((uint32_t)(v >> 32));
  }
  return nr_pack<DT>(y);
}

// MORE: several axes, or a prefix
template <int DT, bool PAIRED, bool VEC, bool MORE>
__global__ void __launch_bounds__(NR_THREADS, 3) norm_rope_kernel(RopeArgs a, int tokens, int per_cta) {
  using T = typename Elem<DT>::type;
  using Lane = NrLane<DT>;
  constexpr int HPW = Lane::HPW;
  constexpr int N = 4;  // query items of a warp in flight, and one of keys
  __shared__ __align__(16) float cos_s[8][TQ_D / 2], sin_s[8][TQ_D / 2], weight_s[2][TQ_D];
  static_assert(NR_THREADS == 2 * TQ_D, "a thread per weight");
  const tq_rope& r = a.r;
  const int tid = threadIdx.x, warp = tid >> 5;
  const int wpt = NR_THREADS / 32 / per_cta;  // warps of a token
  const int mine = warp / wpt, sub = warp % wpt;
  const uint32_t tok = blockIdx.x * (uint32_t)per_cta + mine;  // (at most 2^31 + 7)
  const bool active = tok < (uint32_t)tokens;
  const uint32_t s = active ? tok / (uint32_t)r.n_tokens : 0u, t = active ? tok - s * (uint32_t)r.n_tokens : 0u;
  Lane n;
  n.lane = tid & 31;
  n.hl = n.lane / Lane::LPH, n.ch = n.lane % Lane::LPH * Lane::E, n.half = r.rotary_dim / 2;
  n.low = n.ch < n.half, n.turned = n.ch < 2 * n.half;
  n.partner = !PAIRED || !n.turned ? n.lane : n.low ? n.lane + n.half / Lane::E : n.lane - n.half / Lane::E;
  // this lane's head of item 0; the items of a warp are `step` heads apart
  const int h0 = sub * HPW + n.hl, step = wpt * HPW;
  const T* q = (const T*)r.q + ((int64_t)s * r.q_seq_stride + (int64_t)t * r.q_tok_stride + h0 * r.q_head_stride + n.ch);
  const T* k = (const T*)r.k + ((int64_t)s * r.k_seq_stride + (int64_t)t * r.k_tok_stride + h0 * r.k_head_stride + n.ch);
  const int64_t q_step = step * r.q_head_stride, k_step = step * r.k_head_stride;

  uint4 raw[N], raw_k = make_uint4(0u, 0u, 0u, 0u);
  auto fetch = [&](int h) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (active && h + i * step < r.n_q_heads) raw[i] = nr_load<DT, VEC>(q);
      q += q_step;
    }
  };
  fetch(h0);  // (on their way while the angles are formed)
  if (active && h0 < r.n_kv_heads) raw_k = nr_load<DT, VEC>(k);
  {
    const void* w = tid < TQ_D ? r.q_weight : r.k_weight;
    weight_s[tid / TQ_D][tid % TQ_D] = w == nullptr ? 1.0f : nr_weight(w, tid % TQ_D, r.weight_dtype);
  }
  for (int i = tid; i < per_cta * n.half; i += NR_THREADS) {
    const int u = i / n.half, f = i - u * n.half;
    const uint32_t tk = blockIdx.x * (uint32_t)per_cta + u;
    if (tk >= (uint32_t)tokens) break;
    const uint32_t us = tk / (uint32_t)r.n_tokens, ut = tk - us * (uint32_t)r.n_tokens;
    int64_t p;
    if (a.seq_len != nullptr) {
      p = (int64_t)a.seq_len[us] + ut;
      if (MORE && a.before != nullptr) p += *a.before;
    } else {
      int64_t at = (int64_t)us * r.pos_seq_stride + (int64_t)ut * r.pos_tok_stride;
      if (MORE && a.x.axes != nullptr) at += min((int)a.x.axes[f], a.x.n_axes - 1) * a.x.pos_axis_stride;
      p = r.pos_bits == 64 ? ((const int64_t*)r.positions)[at] : (int64_t)((const int32_t*)r.positions)[at];
    }
    const double turns = (double)p * ((double)r.inv_freq[f] * 0.15915494309189533577);
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    cos_s[u][f] = cs;
    sin_s[u][f] = sn;
  }
  __syncthreads();
  if (!active) return;

  T* out = (T*)r.q_out + (((int64_t)tok * r.n_q_heads + h0) * TQ_D + n.ch);
  nr_factors<DT, PAIRED>(n, weight_s[0], cos_s[mine], sin_s[mine]);
  for (int h = h0; h - n.hl < r.n_q_heads; h += N * step) {  // (a warp's lanes stay together)
    if (h != h0) fetch(h);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (h - n.hl + i * step >= r.n_q_heads) break;
      const uint4 y = nr_head<DT, PAIRED>(n, raw[i], r.q_weight != nullptr, r.eps);
      if (h + i * step < r.n_q_heads) *(uint4*)out = y;
      out += step * TQ_D;
    }
  }
  out = (T*)r.k_out + (((int64_t)tok * r.n_kv_heads + h0) * TQ_D + n.ch);
  nr_factors<DT, PAIRED>(n, weight_s[1], cos_s[mine], sin_s[mine]);
  for (int h = h0; h - n.hl < r.n_kv_heads; h += step) {
    const uint4 x = raw_k;
    k += k_step;
    if (h + step < r.n_kv_heads) raw_k = nr_load<DT, VEC>(k);
    const uint4 y = nr_head<DT, PAIRED>(n, x, r.k_weight != nullptr, r.eps);
    if (h < r.n_kv_heads) *(uint4*)out = y;
    out += step * TQ_D;
  }
}

template <int DT, bool PAIRED>
void start(const RopeArgs& a, int tokens, int sm_count, bool vec, cudaStream_t st) {
  // The fewest tokens a CTA with which all are resident at once, three an SM: another round of them costs more than a
  // warp's longer work, and that more than the angles of more tokens a thread.  us for 1 | 2 | 4 | 8 tokens a CTA (32 + 8
  // heads, bfloat16): 64 tokens 3.7 | 4.2 | 5.5 | 8.5, 600: 8.3 |
  // 6.3 | 6.9 | 8.6, 1700: 17.1 | 11.6 | 9.1 | 11.1, 6000: 62 | 41 | 34 | 32.
  const int resident = 3 * sm_count;
  int per_cta = 1;
  while (per_cta < NR_THREADS / 32 && tokens > per_cta * resident) per_cta *= 2;
  const int grid = (int)(((int64_t)tokens + per_cta - 1) / per_cta);
  const bool more = a.before != nullptr || a.x.axes != nullptr;
  const auto kernel = vec ? more ? norm_rope_kernel<DT, PAIRED, true, true> : norm_rope_kernel<DT, PAIRED, true, false>
                          : more ? norm_rope_kernel<DT, PAIRED, false, true> : norm_rope_kernel<DT, PAIRED, false, false>;
  kernel<<<grid, NR_THREADS, 0, st>>>(a, tokens, per_cta);
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
  TQ_REQUIRE(((uintptr_t)r->q_out | (uintptr_t)r->k_out) % 16 == 0, TQ_ERR_INVALID,
             "q_out and k_out must be aligned to 16 bytes");
  return TQ_OK;
}

int launch(const tq_rope* r, const int32_t* seq_len, const int32_t* before, const tq_rope_axes& x, int device,
           cudaStream_t st) {
  const int tokens = r->n_seqs * r->n_tokens;
  if (tokens == 0 || r->n_q_heads + r->n_kv_heads == 0) return TQ_OK;
  static std::atomic<int> counts[64];  // (asked for once per device)
  int sms = device >= 0 && device < 64 ? counts[device].load(std::memory_order_relaxed) : 0;
  if (sms == 0) {
    TQ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    if (device >= 0 && device < 64) counts[device].store(sms, std::memory_order_relaxed);
  }
  const int e = 16 / elem_size(r->dtype);
  const bool vec = ((uintptr_t)r->q | (uintptr_t)r->k) % 16 == 0 &&
                   ((r->q_seq_stride | r->q_tok_stride | r->q_head_stride | r->k_seq_stride |
                     r->k_tok_stride | r->k_head_stride) & (e - 1)) == 0;
  RopeArgs a = {*r, seq_len, before, x};
  const bool paired = r->rotary_dim / 2 % e == 0;
  switch (r->dtype) {
    case TQ_F32: start<TQ_F32, true>(a, tokens, sms, vec, st); break;
    case TQ_F16: paired ? start<TQ_F16, true>(a, tokens, sms, vec, st) : start<TQ_F16, false>(a, tokens, sms, vec, st); break;
    default: paired ? start<TQ_BF16, true>(a, tokens, sms, vec, st) : start<TQ_BF16, false>(a, tokens, sms, vec, st);
  }
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

}  // namespace

extern "C" int32_t tq_norm_rope(const tq_rope* r, int32_t device, void* stream) {
  return tq_norm_rope_axes(r, nullptr, device, stream);
}

extern "C" int32_t tq_norm_rope_axes(const tq_rope* r, const tq_rope_axes* x, int32_t device, void* stream) {
  const int rc = check_rope(r, false);
  if (rc != TQ_OK) return rc;
  TQ_REQUIRE(x == nullptr || ((x->axes != nullptr || r->rotary_dim == 0) && x->n_axes >= 1), TQ_ERR_INVALID,
             "axes must be a device pointer, and n_axes at least 1");
  TQ_CUDA(cudaSetDevice(device));
  return launch(r, nullptr, nullptr, x == nullptr ? tq_rope_axes{} : *x, device, (cudaStream_t)stream);
}

extern "C" int32_t tq_ctx_norm_rope(tq_ctx* ctx, int32_t layer, int32_t seq_begin, const tq_rope* r, void* stream) {
  return tq_ctx_norm_rope_after(ctx, layer, seq_begin, -1, r, stream);
}

extern "C" int32_t tq_ctx_norm_rope_after(tq_ctx* ctx, int32_t layer, int32_t seq_begin, int32_t prefix,
                                          const tq_rope* r, void* stream) {
  TQ_REQUIRE(ctx != nullptr && layer >= 0 && layer < ctx->g.n_layers, TQ_ERR_INVALID, "bad context or layer");
  const int rc = check_rope(r, true);
  if (rc != TQ_OK) return rc;
  const tq_geom& g = ctx->g;
  TQ_REQUIRE(r->n_q_heads == g.n_q_heads && r->n_kv_heads == g.n_kv_heads, TQ_ERR_INVALID,
             "head counts do not match the context");
  TQ_REQUIRE(seq_begin >= 0 && r->n_seqs >= 0 && (int64_t)seq_begin + r->n_seqs <= g.n_seqs, TQ_ERR_INVALID,
             "sequence range out of bounds");
  TQ_REQUIRE(prefix == -1 || (prefix >= 0 && prefix < g.n_seqs && (prefix < seq_begin || prefix >= seq_begin + r->n_seqs)),
             TQ_ERR_INVALID, "prefix must be a sequence of the context that is none of the call's own");
  TQ_CUDA(cudaSetDevice(ctx->device));
  const int32_t* len = (const int32_t*)((const uint8_t*)ctx->b.state + state_len_off(g)) + (size_t)layer * g.n_seqs;
  return launch(r, len + seq_begin, prefix < 0 ? nullptr : len + prefix, tq_rope_axes{}, ctx->device,
                (cudaStream_t)stream);
}

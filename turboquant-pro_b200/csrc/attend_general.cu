// Attention of many query tokens on the codes, general form: float32 arithmetic on the CUDA cores, every
// key format, block length, query group and type; and the merge of the splits' states for all forms.
//
// A CTA takes a tile of query rows of one (sequence, KV head) and one split of the token tiles that these
// rows see.  A tile of 64 tokens is dequantised into shared memory once and attended by all rows of the
// CTA:  k = mean + scale * grid[code], outliers put over it;  v = norm * centroid[code] in code space
// (PolarQuant keys likewise, against the rotated query);  window tokens as they are.  A thread owns RPT rows
// x 4 tokens of the scores and RPT rows x 8 channels of the sums; the running maximum and sum of a row
// live in the registers of the 16 threads that share it.
//
// A value that is not finite must not reach rows that do not see its token (0 * inf): a tile that holds
// one is summed with the masked products left out one by one.
//
// Bound by the FP32 pipe (46 %) and the loads that feed it (issue slots 62 %) at two CTAs an SM (large calls: 200 tokens of
// 28 query heads on 3 x 6850 tokens of 4 KV heads, float32, 2.17 ms: 27 TFLOP/s), and by the chain of loads of the
// dequantisation into shared memory (few rows).
#include <algorithm>

#include "attend.cuh"

namespace {

constexpr int AG_THREADS = 256;
constexpr int AG_T = 64;            // tokens of a tile
constexpr int AG_KS = TQ_D + 4;     // floats per row of keys, values and queries
constexpr int AG_PS = AG_T + 4;     // floats per row of probabilities

struct AgFixed {
  float k[AG_T][AG_KS];  // and, when the scores have been formed, the probabilities: two CTAs an SM have room then
  float v[AG_T][AG_KS];
  float grid[16], cent[16];
};
// 32 channels of a window row, 16 bytes at a time; whether all are numbers and finite
TQ_DEV bool ag_row(const void* rows, size_t at, int dt, float* to) {
  bool ok = true;
  if (dt == TQ_F32) {
    const float4* from = (const float4*)((const float*)rows + at);
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
      const float4 x = from[i];
      *(float4*)(to + 4 * i) = x;
      ok &= isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
    }
    return ok;
  }
  const uint4* from = (const uint4*)((const uint16_t*)rows + at);
#pragma unroll 2
  for (int i = 0; i < 4; ++i) {
    const uint4 u = from[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 f;
      if (dt == TQ_F16) f = __half22float2(*(const __half2*)&w[j]);
      else f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
      *(float2*)(to + 8 * i + 2 * j) = f;
      ok &= isfinite(f.x) && isfinite(f.y);
    }
  }
  return ok;
}
template <int RPT>
struct AgShared : AgFixed {
  float q[16 * RPT][AG_KS];
};
static_assert(64 * AG_PS <= AG_T * AG_KS, "the probabilities' place");

// The value-layout codes of token `t` of a block, channels d0 .. d0 + 31, times `f`.
TQ_DEV void ag_codes(const uint8_t* codes, int bits, int t, int d0, const float* cent, float f, float* to) {
  const uint8_t* grp = codes + (size_t)(t >> 4) * v_group_bytes(bits);
#pragma unroll 4
  for (int i = 0; i < 32; ++i) to[i] = f * cent[v_get_code(grp, bits, t & 15, d0 + i)];
}
// The same of all 16 tokens of a group: a warp's lanes expand their records.
TQ_DEV void ag_group(const uint8_t* grp, int bits, int lane, const float* cent, const float* norms,
                     float (*to)[AG_KS]) {
  const int r = lane >> 2, c = lane & 3;
  uint32_t w[9];
  if (bits == 4) {
    const uint4 x = *(const uint4*)(grp + lane * 16), y = *(const uint4*)(grp + 512 + lane * 16);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint2 x = *(const uint2*)(grp + i * 256 + lane * 8);
      w[2 * i] = x.x, w[2 * i + 1] = x.y;
    }
    w[6] = w[7] = 0u;
  }
  w[8] = 0u;
#pragma unroll
  for (int p = 0; p < 32; ++p) {
    const int t = 2 * c + 8 * (p & 1), d = r + 8 * (p >> 1);
    uint32_t lo, hi;
    if (bits == 4) {
      const uint32_t b = w[p >> 2] >> (8 * (p & 3));
      lo = b & 15, hi = (b >> 4) & 15;
    } else {
      const uint32_t b = __funnelshift_r(w[6 * p >> 5], w[(6 * p >> 5) + 1], (6 * p) & 31);
      lo = b & 7, hi = (b >> 3) & 7;
    }
    to[t][d] = norms[t] * cent[lo];
    to[t + 1][d] = norms[t + 1] * cent[hi];
  }
}

// A tile of rows and a split of its tokens.
template <int RPT>
TQ_DEV void ag_item(const AttendArgs& a, int row_tiles, int item, AgShared<RPT>& sh) {
  constexpr int RT = 16 * RPT;
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ty = tid >> 4, tx = tid & 15;
  const int ns = a.ns_cold + a.ns_hot;
  const int split = item % ns, rt = item / ns % row_tiles, unit = item / ns / row_tiles;
  if (a.left != nullptr && a.left[unit] == 0) return;
  const int H = g.n_kv_heads, G = g.group, S = g.block_tokens, vb = g.value_bits;
  const int s = unit / H, head = unit % H, row0 = rt * RT;
  const AttendSeq sq = attend_seq(a, s);
  const bool polar = g.key_mode == TQ_KEYS_POLAR, is_cold = split < a.ns_cold;
  const size_t uix = unit_index(g, a.layer, a.seq_begin + s, head);

  if (tid < 16) {
    sh.grid[tid] = a.tables->grid[tid];
    sh.cent[tid] = a.tables->centroids[tid];
  }
  // ---- query rows, in units that make scores logarithms to base 2
  for (int i = tid; i < RT * TQ_D; i += AG_THREADS) {
    const int r = i / TQ_D, d = i % TQ_D, row = row0 + r;
    float x = 0.0f;
    if (row < a.rows)
      x = attend_ld(a.q, (size_t)((int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok +
                                  (int64_t)(head * G + row % G) * a.q_head + d), a.q_dtype);
    sh.q[r][d] = tq_scaled<true>(x);
  }
  if (polar && is_cold) {  // codes of keys are met by the rotated query: q @ Pi^T
    __syncthreads();
    constexpr int N = RT * TQ_D / AG_THREADS;
    float y[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * AG_THREADS, r = i / TQ_D, e = i % TQ_D;
      float x = 0.0f;
      for (int d = 0; d < TQ_D; ++d) x = fmaf(sh.q[r][d], a.tables->pi_t[d * TQ_D + e], x);
      y[k] = x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * AG_THREADS;
      sh.q[i / TQ_D][i % TQ_D] = y[k];
    }
  }

  // ---- the token tiles of this split
  const int i_lo = row0 / G, i_hi = min(min(row0 + RT, a.rows) - 1, sq.q_n * G - 1) / G;
  const int p_lo = sq.first + i_lo, p_hi = i_lo < sq.q_n ? sq.first + i_hi : -1;
  const int base = is_cold ? 0 : sq.cold, end = is_cold ? sq.cold : sq.n;
  const AttendTiles tl = attend_tiles(a, base, end, AG_T, p_lo, p_hi);
  const int part = is_cold ? split : split - a.ns_cold, parts = is_cold ? a.ns_cold : a.ns_hot;
  const int k_lo = (int)((long)tl.count() * part / parts), k_hi = (int)((long)tl.count() * (part + 1) / parts);

  int pos[RPT], win[RPT];
  float m[RPT], l[RPT], o[RPT][8];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int row = row0 + ty * RPT + r;
    pos[r] = row < a.rows ? attend_position(a, sq, row) : -1;
    win[r] = attend_window(a, pos[r]);
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.0f;
  }

  for (int k = k_lo; k < k_hi; ++k) {
    const int t0 = base + tl.at(k) * AG_T, t1 = min(t0 + AG_T, end);
    __syncthreads();
    bool odd = false;  // a value that is not finite
    {
      const int t = t0 + (tid & 63), d0 = (tid >> 6) * 32;
      float* kr = &sh.k[tid & 63][d0];
      float* vr = &sh.v[tid & 63][d0];
      if (t >= t1) {
#pragma unroll
        for (int i = 0; i < 32; ++i) kr[i] = vr[i] = 0.0f;
      } else if (!is_cold) {
        const size_t at = hot_offset_elems(g, a.layer, a.seq_begin + s, head) +
                          (size_t)(t % g.hot_cap) * TQ_D + d0;
        ag_row(a.hot_k, at, g.kv_dtype, kr);
        odd |= !ag_row(a.hot_v, at, g.kv_dtype, vr);
      } else {
        const int b = t / S, slot = t - b * S;
        const uint8_t* page = a.pages + page_offset(g, a.layer, a.seq_begin + s, head, b);
        if (polar) {
          ag_codes(page, vb, slot, d0, sh.cent, ((const float*)(page + g.scale_off))[slot], kr);
        } else {
          const uint4 cw = *(const uint4*)(page + slot * (TQ_D / 2) + d0 / 2);
          const uint32_t w[4] = {cw.x, cw.y, cw.z, cw.w};
          const float* sc = (const float*)(page + g.scale_off) + d0;
          const float* mu = (const float*)(page + g.mean_off) + d0;
#pragma unroll 4
          for (int i = 0; i < 32; i += 4) {
            const float4 x = *(const float4*)(sc + i), y = *(const float4*)(mu + i);
            const uint32_t c = w[i >> 3] >> (4 * (i & 7));
            kr[i] = fmaf(x.x, sh.grid[c & 15], y.x);
            kr[i + 1] = fmaf(x.y, sh.grid[(c >> 4) & 15], y.y);
            kr[i + 2] = fmaf(x.z, sh.grid[(c >> 8) & 15], y.z);
            kr[i + 3] = fmaf(x.w, sh.grid[(c >> 12) & 15], y.w);
          }
        }
        const float norm = ((const float*)(page + g.norm_off))[slot];
        odd |= !isfinite(norm);
        if (S % TQ_GROUP_TOK != 0) ag_codes(page + g.v_off, vb, slot, d0, sh.cent, norm, vr);
      }
    }
    if (is_cold && S % TQ_GROUP_TOK == 0 && warp < AG_T / TQ_GROUP_TOK) {
      const int t = t0 + warp * TQ_GROUP_TOK, b = t / S, slot = t - b * S;
      if (t < t1) {  // (blocks are whole groups, and so is what is in blocks)
        const uint8_t* page = a.pages + page_offset(g, a.layer, a.seq_begin + s, head, b);
        ag_group(page + g.v_off + (size_t)(slot >> 4) * v_group_bytes(vb), vb, lane, sh.cent,
                 (const float*)(page + g.norm_off) + slot, &sh.v[warp * TQ_GROUP_TOK]);
      }
    }
    odd = __syncthreads_or(odd);
    if (is_cold && g.outlier_k > 0) {
      // (a block at a time by all, or, where a tile has several, by a warp each: their lists' places are loads that
      // depend on one another)
      const bool many = S < AG_T;
      for (int b = t0 / S + (many ? warp : 0); b * S < t1; b += many ? AG_THREADS / 32 : 1) {
        const PageMeta pm = a.page_meta[uix * g.max_blocks + b];
        const size_t slab = uix * (size_t)g.pool_entries + pm.off;
        for (uint32_t e = many ? lane : tid; e < pm.cnt; e += many ? 32 : AG_THREADS) {
          const uint32_t w = a.pool_dec[slab + e];
          const int t = b * S + (int)(w >> 24);
          if (t >= t0 && t < t1)
            sh.k[t - t0][(w >> 16) & 127] = __half2float(__ushort_as_half(a.pool_val[slab + e]));
        }
      }
      __syncthreads();
    }

    float (*const prob)[AG_PS] = (float (*)[AG_PS])&sh.k[0][0];
    // ---- scores: rows ty * RPT .., tokens tx + 16 j
    float x[RPT][4];
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[r][j] = 0.0f;
    // (sixteen channels at a time: a sum over all 128 in a row would be rounded at its full size 128 times)
#pragma unroll 1
    for (int d0 = 0; d0 < TQ_D; d0 += 16) {
      float y[RPT][4];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[r][j] = 0.0f;
#pragma unroll
      for (int d = d0; d < d0 + 16; d += 4) {
        float4 kk[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[j] = *(const float4*)&sh.k[tx + 16 * j][d];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          const float4 qq = *(const float4*)&sh.q[ty * RPT + r][d];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[r][j] = fmaf(qq.x, kk[j].x, fmaf(qq.y, kk[j].y, fmaf(qq.z, kk[j].z, fmaf(qq.w, kk[j].w, y[r][j]))));
        }
      }
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[r][j] += y[r][j];
    }
    __syncthreads();  // (the keys have been read)
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      bool sees[4];
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + tx + 16 * j;
        sees[j] = t < t1 && t <= pos[r] && (t >= win[r] || t < a.sinks);
        if (sees[j]) top = fmaxf(top, x[r][j]);
      }
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      top = fmaxf(m[r], top);
      // (a maximum of -inf: nothing seen yet, or scores that are no numbers, which stay so)
      const float by = top > -INFINITY ? top : 0.0f;
      const float down = tq_exp2(m[r] - by);
      m[r] = top;
      l[r] *= down;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= down;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = sees[j] ? tq_exp2(x[r][j] - by) : 0.0f;
        l[r] += p;
        prob[ty * RPT + r][tx + 16 * j] = odd && !sees[j] ? -1.0f : p;
      }
    }
    __syncwarp();  // (a row's sixteen threads are in one warp)

    // ---- sums: rows ty * RPT .., channels 4 tx .. + 3 and 64 + 4 tx .. + 3
    if (!odd) {
#pragma unroll 2
      for (int t = 0; t < AG_T; t += 4) {
        float4 pp[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) pp[r] = *(const float4*)&prob[ty * RPT + r][t];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float4 va = *(const float4*)&sh.v[t + u][4 * tx], vc = *(const float4*)&sh.v[t + u][64 + 4 * tx];
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const float p = u == 0 ? pp[r].x : u == 1 ? pp[r].y : u == 2 ? pp[r].z : pp[r].w;
            o[r][0] = fmaf(p, va.x, o[r][0]), o[r][1] = fmaf(p, va.y, o[r][1]);
            o[r][2] = fmaf(p, va.z, o[r][2]), o[r][3] = fmaf(p, va.w, o[r][3]);
            o[r][4] = fmaf(p, vc.x, o[r][4]), o[r][5] = fmaf(p, vc.y, o[r][5]);
            o[r][6] = fmaf(p, vc.z, o[r][6]), o[r][7] = fmaf(p, vc.w, o[r][7]);
          }
        }
      }
    } else {
      for (int t = 0; t < AG_T; ++t)
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          const float p = prob[ty * RPT + r][t];
          if (p < 0.0f) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            o[r][e] = fmaf(p, sh.v[t][(e >> 2) * 64 + 4 * tx + (e & 3)], o[r][e]);
        }
    }
  }

#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int row = row0 + ty * RPT + r;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
    if (row >= a.rows) continue;
    float* to = attend_partial(a, unit, row, split);
    if (tx == 0) *(float2*)to = make_float2(m[r], l[r]);
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      *(float2*)(to + 2 + (e >> 2) * 64 + 4 * tx + (e & 3)) = make_float2(o[r][e], o[r][e + 1]);
  }
}

template <int RPT>
__global__ void __launch_bounds__(AG_THREADS, 2) attend_general_kernel(AttendArgs a, int row_tiles) {
  extern __shared__ __align__(16) uint8_t ag_smem[];
  ag_item(a, row_tiles, (int)blockIdx.x, *(AgShared<RPT>*)ag_smem);
}
// Only the (sequence, KV head) units that the form for many rows has left: hardly ever one, so that a CTA per SM looks
// through the flags first (a CTA per item, that finds its own unset, took 7.5 us for 2048 tokens of 8 KV heads).
template <int RPT>
__global__ void __launch_bounds__(AG_THREADS) attend_left_kernel(AttendArgs a, int row_tiles, int items) {
  extern __shared__ __align__(16) uint8_t ag_smem[];
  bool any = false;
  for (int i = threadIdx.x; i < a.seq_count * a.g.n_kv_heads; i += AG_THREADS) any |= a.left[i] != 0;
  if (!__syncthreads_or(any)) return;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    ag_item(a, row_tiles, (int)item, *(AgShared<RPT>*)ag_smem);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// Merge of a row's states, a CTA per row and a thread per channel.  The splits are visited in order, so the result
// depends on nothing else; a state without a sum takes no part, one whose sum is not a number does.  (Sixteen rows
// a CTA, which read Pi once for all, took longer at every number of rows: by 157 us for 128 rows of 4000
// tokens, by 10 us for 51200 rows with a window of 64.)
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(TQ_D) attend_combine_kernel(AttendArgs a) {
  const tq_geom& g = a.g;
  const int e = threadIdx.x, unit = blockIdx.x / a.rows, row = blockIdx.x % a.rows;
  const int ns = a.ns_cold + a.ns_hot, H = g.n_kv_heads, G = g.group, s = unit / H, head = unit % H;
  __shared__ float cs[TQ_D];
  float M = -INFINITY, L = 0.0f, C = 0.0f, Y = 0.0f;
  const float* p = attend_partial(a, unit, row, 0);
  for (int i = 0; i < ns; ++i) M = fmaxf(M, p[(size_t)i * TQ_PART_STRIDE]);
  const float by = M > -INFINITY ? M : 0.0f;
  for (int i = 0; i < ns; ++i) {
    const float* x = p + (size_t)i * TQ_PART_STRIDE;
    const float li = x[1];
    if (li == 0.0f) continue;
    const float w = x[0] > -INFINITY ? tq_exp2(x[0] - by) : 1.0f;
    L += li * w;
    if (i < a.ns_cold) C += x[2 + e] * w;
    else Y += x[2 + e] * w;
  }
  cs[e] = C;
  __syncthreads();
  float y = 0.0f;
  for (int d0 = 0; d0 < TQ_D; d0 += 16) {  // (sums of sums: a chain of 128 roundings would show in float32)
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < 16; ++d) z = fmaf(cs[d0 + d], a.tables->pi[(d0 + d) * TQ_D + e], z);
    y += z;
  }
  const size_t at = (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D + e;
  const float x = L == 0.0f ? 0.0f : (y + Y) / L;
  if (a.q_dtype == TQ_F32) ((float*)a.out)[at] = x;
  else if (a.q_dtype == TQ_F16) ((__half*)a.out)[at] = __float2half_rn(x);
  else ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(x);
}

template <int RPT>
int launch_general(const AttendArgs& a, cudaStream_t st) {
  const int row_tiles = (a.rows + 16 * RPT - 1) / (16 * RPT);
  const int64_t grid = (int64_t)a.seq_count * a.g.n_kv_heads * row_tiles * (a.ns_cold + a.ns_hot);
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (sequence, head, query row) tiles in a call");
  static bool done[64], left_done[64];
  if (a.left != nullptr) {
    const int rc = attend_shared(attend_left_kernel<RPT>, sizeof(AgShared<RPT>), a.device, left_done);
    if (rc != TQ_OK) return rc;
    attend_left_kernel<RPT><<<(int)std::min<int64_t>(grid, a.sm_count), AG_THREADS, sizeof(AgShared<RPT>), st>>>(
        a, row_tiles, (int)grid);
    TQ_CUDA(cudaGetLastError());
    return TQ_OK;
  }
  const int rc = attend_shared(attend_general_kernel<RPT>, sizeof(AgShared<RPT>), a.device, done);
  if (rc != TQ_OK) return rc;
  attend_general_kernel<RPT><<<(int)grid, AG_THREADS, sizeof(AgShared<RPT>), st>>>(a, row_tiles);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

}  // namespace

// Tiles of 16 rows, or of 64 with a fourth of the loads per product: 4 to 16 rows 54 to 56 us against 69 to 71 (4000
// float32 tokens, 8 KV heads), 32 rows 94 against 73, 64 rows 160 against 77.
int tq_launch_attend_general(const AttendArgs& a, cudaStream_t st) {
  return a.rows <= 16 ? launch_general<1>(a, st) : launch_general<4>(a, st);
}

int tq_launch_attend_combine(const AttendArgs& a, cudaStream_t st) {
  const int64_t grid = (int64_t)a.seq_count * a.g.n_kv_heads * a.rows;
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (sequence, head, query row) tiles in a call");
  attend_combine_kernel<<<(int)grid, TQ_D, 0, st>>>(a);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

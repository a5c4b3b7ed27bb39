// Attention of many query rows per KV head on the codes: prompt chunks.  The products run on tcgen05 with the
// accumulators in tensor memory.  Three kernels:
//
// attend_stage_kernel   the tokens that any row sees, 128 at a time, from codes to the two shared-memory images
//     that tcgen05 takes as operands (fp16, K-major core matrices of 8 rows x 16 bytes), written to the workspace
//     once instead of once per tile of rows:
//       keys    (mean + scale * grid[code] - c) / 16, outliers put over it.  c is one vector per (sequence, KV head),
//               the zero-point of its first block: it moves all scores of a row alike, so the softmax does not
//               see it, and large constant channels do not eat the half-precision digits.  The 16 keeps keys to 10^6
//               in fp16's range.
//       values  transposed, in code space: norm * centroid[code], window tokens rotated into that space; all times
//               the power of two that takes the tile's largest norm below 2^15, whose exponent is kept.
//     What is not a number, or too large even so, sets the flag of its (sequence, KV head), which the general kernel
//     then does.
// attend_tiles_kernel   256 rows of a (sequence, KV head) per CTA against a split of these tiles.  S = Q K^T into tensor
//     memory; two groups of 128 threads, a thread per row, make the probabilities and put them back over S as fp16;
//     O += P V with P as the operand in tensor memory.  The groups work on different halves of the rows, so that the
//     tensor cores have one's products while the other's softmax runs.  A tile's exponent is added to its scores, so
//     that the running maximum is that of probability * value and fp16 holds what counts.  The maximum is only
//     renewed (and O rescaled) when it has grown by 2^8 since.
// attend_tiles_combine_kernel   merges the splits, rotates the sums back (sum @ Pi), rounds.
//
// Queries are fp16 in shared memory, each row scaled by a power of two, which is exact for both 16-bit types.
// SPLIT (float16 queries): keys and values as pairs hi + lo, so that only the probabilities are rounded to fp16 and the
// result is off by about its own rounding; bfloat16 queries take the hi parts alone (2^-12 against 2^-9).
#include <algorithm>

#include "attend.cuh"
#include "encode.cuh"  // mbarrier, descriptors, commit

namespace {

constexpr int TI_T = 128;                    // tokens of a tile
constexpr int TI_ROWS = 256;                 // rows of a CTA
constexpr int TI_IMAGE = TI_T * TQ_D * 2;    // bytes of an operand image
constexpr int TI_LBO = TI_T * 16, TI_SBO = 128;
constexpr int TI_SLOTS = 5;                  // images in shared memory
constexpr int TI_THREADS = 320;              // two softmax groups, a warp that issues, a warp that loads
constexpr float TI_KEY = 16.0f;              // keys are divided by it
constexpr float TI_LIFT = 7.0f, TI_GROW = 8.0f;  // probabilities reach 2^(7 + 8) at most
constexpr int TI_WAIT = 1 << 21;             // probes of a wait, a microsecond or two each at most

struct TileArgs {
  uint8_t* images;    // [unit][cap][K hi, (K lo,) V hi, (V lo)]
  float* exponent;    // [unit][cap]
  int32_t* left;      // [unit]
  float* sums;        // per unit, unit_stride floats apart: [split][row tile][channel][256]
  float* stats;       // [unit][split][row tile][2][256]
  int cap;            // tiles a unit has room for
  int splits, row_tiles;
};

// the tiles of a unit that any row of the call sees
TQ_DEV AttendTiles unit_tiles(const AttendArgs& a, const AttendSeq& sq) {
  return attend_tiles(a, 0, sq.n, TI_T, sq.first, sq.q_n > 0 ? sq.n - 1 : -1);
}

TQ_DEV float ti_lift(float x, int top, float& exponent) {  // 2^(top - floor(log2 x)), and the exponent of its inverse
  const int e = min(max((int)(__float_as_uint(x) >> 23 & 255u), 64), 254);
  exponent = (float)(e - 127 - top);
  return __int_as_float((254 + top - e) << 23);
}

TQ_DEV uint32_t ti_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
TQ_DEV uint32_t ti_rest(float a, float b, uint32_t hi) {  // what the pair's rounding dropped
  const float2 f = __half22float2(*(const __half2*)&hi);
  return ti_pair(a - f.x, b - f.y);
}

constexpr int TS_THREADS = 256;
constexpr int TS_VS = TQ_D + 4;  // floats per row of window values
template <bool SPLIT>
struct StageShared {
  alignas(16) uint8_t k[SPLIT ? 2 : 1][TI_IMAGE];
  float v[TI_T][TS_VS];
  float center[TQ_D], grid[16], cent[16], norm[TI_T];
  float top[TS_THREADS / 32];
};

template <bool SPLIT>
__global__ void __launch_bounds__(TS_THREADS) attend_stage_kernel(AttendArgs a, TileArgs ta) {
  extern __shared__ __align__(16) uint8_t ts_smem[];
  StageShared<SPLIT>& sh = *(StageShared<SPLIT>*)ts_smem;
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // (the last tiles first: the window's take longest)
  const int unit = blockIdx.x / ta.cap, s = unit / g.n_kv_heads, head = unit % g.n_kv_heads;
  const AttendSeq sq = attend_seq(a, s);
  const AttendTiles tl = unit_tiles(a, sq);
  const int idx = tl.count() - 1 - (int)(blockIdx.x % ta.cap);
  if (tl.count() > ta.cap) {
    if (idx == tl.count() - 1 && tid == 0) ta.left[unit] = 1;
    return;
  }
  if (idx < 0) return;
  const int S = g.block_tokens, vb = g.value_bits;
  const int t0 = tl.at(idx) * TI_T, t1 = min(t0 + TI_T, sq.n);
  const size_t uix = unit_index(g, a.layer, a.seq_begin + s, head);
  const uint8_t* const pages = a.pages + page_offset(g, a.layer, a.seq_begin + s, head, 0);
  const size_t ring = hot_offset_elems(g, a.layer, a.seq_begin + s, head);

  if (tid < 16) {
    sh.grid[tid] = a.tables->grid[tid];
    sh.cent[tid] = a.tables->centroids[tid];
  }
  if (tid < TQ_D) {  // uniform grids count from their zero-point on: their middle
    float c = 0.0f;
    if (sq.cold > 0) {
      c = ((const float*)(pages + g.mean_off))[tid];
      if (g.key_mode == TQ_KEYS_UNIFORM) c = fmaf(7.5f, ((const float*)(pages + g.scale_off))[tid], c);
      if (!isfinite(c)) c = 0.0f;
    }
    sh.center[tid] = c;
  }
  __syncthreads();
  bool odd = false;
  {  // ---- keys: a thread has half a token
    const int row = tid & 127, h = tid >> 7, t = t0 + row;
    auto put = [&](int chunk, const float (&x)[8]) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = x[2 * i] * (1.0f / TI_KEY), q = x[2 * i + 1] * (1.0f / TI_KEY);
        odd |= !(fabsf(p) <= 65504.0f) || !(fabsf(q) <= 65504.0f);
        hi[i] = ti_pair(p, q);
        if (SPLIT) lo[i] = ti_rest(p, q, hi[i]);
      }
      *(uint4*)(sh.k[0] + chunk * TI_LBO + row * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if (SPLIT) *(uint4*)(sh.k[SPLIT] + chunk * TI_LBO + row * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    };
    if (t < sq.cold) {
      const int b = t / S, slot = t - b * S;
      const uint8_t* page = pages + (size_t)b * g.page_bytes;
      const float* sc = (const float*)(page + g.scale_off);
      const float* mu = (const float*)(page + g.mean_off);
      const uint4 c0 = *(const uint4*)(page + slot * (TQ_D / 2) + 32 * h);
      const uint4 c1 = *(const uint4*)(page + slot * (TQ_D / 2) + 32 * h + 16);
      const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 64 * h + 8 * i;
        const float4 s0 = *(const float4*)(sc + d), s1 = *(const float4*)(sc + d + 4);
        const float4 m0 = *(const float4*)(mu + d), m1 = *(const float4*)(mu + d + 4);
        const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
        const float mm[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(ss[e], sh.grid[w[i] >> (4 * e) & 15], mm[e] - sh.center[d + e]);
        put(8 * h + i, x);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 64 * h + 8 * i;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = t < t1 ? attend_ld(a.hot_k, ring + (size_t)(t % g.hot_cap) * TQ_D + d + e, g.kv_dtype) - sh.center[d + e] : 0.0f;
        put(8 * h + i, x);
      }
    }
  }
  __syncthreads();
  if (g.outlier_k > 0) {
    for (int b = t0 / S; b * S < min(t1, sq.cold); ++b) {
      const PageMeta pm = a.page_meta[uix * g.max_blocks + b];
      const size_t slab = uix * (size_t)g.pool_entries + pm.off;
      for (uint32_t e = tid; e < pm.cnt; e += TS_THREADS) {
        const uint32_t w = a.pool_dec[slab + e];
        const int t = b * S + (int)(w >> 24), ch = (w >> 16) & 127;
        if (t < t0 || t >= t1) continue;
        const float x = (__half2float(__ushort_as_half(a.pool_val[slab + e])) - sh.center[ch]) * (1.0f / TI_KEY);
        odd |= !(fabsf(x) <= 65504.0f);
        const int at = (ch >> 3) * TI_LBO + (t - t0) * 16 + (ch & 7) * 2;
        const __half hi = __float2half_rn(x);
        *(__half*)(sh.k[0] + at) = hi;
        if (SPLIT) *(__half*)(sh.k[SPLIT] + at) = __float2half_rn(x - __half2float(hi));
      }
    }
  }

  // ---- values: norms, the tile's power of two
  const bool hot = t1 > sq.cold;  // some tokens are of the window
  if (hot) {
    for (int i = tid; i < TI_T * (TQ_D / 4); i += TS_THREADS) {
      const int row = i / (TQ_D / 4), d = i % (TQ_D / 4) * 4, t = t0 + row;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (t >= sq.cold && t < t1) {
        const size_t at = ring + (size_t)(t % g.hot_cap) * TQ_D + d;
        x = make_float4(attend_ld(a.hot_v, at, g.kv_dtype), attend_ld(a.hot_v, at + 1, g.kv_dtype),
                        attend_ld(a.hot_v, at + 2, g.kv_dtype), attend_ld(a.hot_v, at + 3, g.kv_dtype));
      }
      *(float4*)&sh.v[row][d] = x;
    }
  }
  __syncthreads();
  uint8_t* const images = ta.images + ((size_t)unit * ta.cap + idx) * (SPLIT ? 4 : 2) * TI_IMAGE;
  {
    float norm = 0.0f;
    if (tid < TI_T) {
      const int t = t0 + tid;
      if (t < sq.cold) {
        const int b = t / S;
        norm = ((const float*)(pages + (size_t)b * g.page_bytes + g.norm_off))[t - b * S];
      } else if (t < t1) {
        float x = 0.0f;
        for (int d = 0; d < TQ_D; ++d) x = fmaf(sh.v[tid][d], sh.v[tid][d], x);
        norm = sqrtf(x);
      }
      odd |= !isfinite(norm);
      sh.norm[tid] = norm;
    }
    float top = fabsf(norm);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sh.top[warp] = top;
  }
  for (int i = tid; i < TI_IMAGE / 16; i += TS_THREADS) {  // (the keys are complete)
    *(uint4*)(images + 16 * i) = *(const uint4*)(sh.k[0] + 16 * i);
    if (SPLIT) *(uint4*)(images + TI_IMAGE + 16 * i) = *(const uint4*)(sh.k[SPLIT] + 16 * i);
  }
  odd = __syncthreads_or(odd);
  if (odd && tid == 0) ta.left[unit] = 1;
  float top = 0.0f, exponent;
#pragma unroll
  for (int w = 0; w < TS_THREADS / 32; ++w) top = fmaxf(top, sh.top[w]);
  const float up = ti_lift(top, 14, exponent);
  if (tid == 0) ta.exponent[(size_t)unit * ta.cap + idx] = exponent;
  uint8_t* const v_hi = images + (SPLIT ? 2 : 1) * TI_IMAGE;
  uint8_t* const v_lo = v_hi + TI_IMAGE;
  if (!hot && S % TQ_GROUP_TOK == 0) {
    // a warp expands the records of a group of 16 tokens: two tokens of a channel are a word of the image
    const int t = t0 + warp * TQ_GROUP_TOK, b = t / S, slot = t - b * S, r = lane >> 2, c = lane & 3;
    if (t < t1) {
      const uint8_t* grp = pages + (size_t)b * g.page_bytes + g.v_off + (size_t)(slot >> 4) * v_group_bytes(vb);
      uint32_t w[9];
      if (vb == 4) {
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
      float nv[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) nv[h][x] = sh.norm[warp * TQ_GROUP_TOK + 8 * h + 2 * c + x] * up;
#pragma unroll
      for (int p = 0; p < 32; ++p) {
        const int h = p & 1, d = r + 8 * (p >> 1);
        uint32_t ca, cb;
        if (vb == 4) {
          const uint32_t by = w[p >> 2] >> (8 * (p & 3));
          ca = by & 15, cb = by >> 4 & 15;
        } else {
          const uint32_t by = __funnelshift_r(w[6 * p >> 5], w[(6 * p >> 5) + 1], (6 * p) & 31);
          ca = by & 7, cb = by >> 3 & 7;
        }
        const float x = nv[h][0] * sh.cent[ca], y = nv[h][1] * sh.cent[cb];
        const uint32_t hi = ti_pair(x, y);
        const int at = (2 * warp + h) * TI_LBO + d * 16 + 4 * c;
        *(uint32_t*)(v_hi + at) = hi;
        if (SPLIT) *(uint32_t*)(v_lo + at) = ti_rest(x, y, hi);
      }
    } else {
#pragma unroll 4
      for (int p = 0; p < 32; ++p) {
        const int at = (2 * warp + (p & 1)) * TI_LBO + (r + 8 * (p >> 1)) * 16 + 4 * c;
        *(uint32_t*)(v_hi + at) = 0u;
        if (SPLIT) *(uint32_t*)(v_lo + at) = 0u;
      }
    }
  } else {
    // a thread has 8 tokens x 8 channels: window tokens v @ Pi^T, tokens of blocks from their codes
    const int ty = tid >> 4, tx = tid & 15;
    float x[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
    if (hot) {
#pragma unroll 2
      for (int d = 0; d < TQ_D; ++d) {
        const float4 p0 = *(const float4*)&a.tables->pi_t[d * TQ_D + 8 * tx], p1 = *(const float4*)&a.tables->pi_t[d * TQ_D + 8 * tx + 4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = sh.v[8 * ty + i][d];
          x[i][0] = fmaf(v, p0.x, x[i][0]), x[i][1] = fmaf(v, p0.y, x[i][1]);
          x[i][2] = fmaf(v, p0.z, x[i][2]), x[i][3] = fmaf(v, p0.w, x[i][3]);
          x[i][4] = fmaf(v, p1.x, x[i][4]), x[i][5] = fmaf(v, p1.y, x[i][5]);
          x[i][6] = fmaf(v, p1.z, x[i][6]), x[i][7] = fmaf(v, p1.w, x[i][7]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = t0 + 8 * ty + i;
      if (t < sq.cold) {
        const int b = t / S, slot = t - b * S;
        const uint8_t* grp = pages + (size_t)b * g.page_bytes + g.v_off + (size_t)(slot >> 4) * v_group_bytes(vb);
        const float norm = sh.norm[8 * ty + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = norm * sh.cent[v_get_code(grp, vb, slot & 15, 8 * tx + e)];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = x[2 * i][e] * up, q = x[2 * i + 1][e] * up;
        hi[i] = ti_pair(p, q);
        if (SPLIT) lo[i] = ti_rest(p, q, hi[i]);
      }
      const int at = ty * TI_LBO + (8 * tx + e) * 16;
      *(uint4*)(v_hi + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if (SPLIT) *(uint4*)(v_lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------
struct TiShared {
  alignas(128) uint8_t q[2][TI_IMAGE];
  alignas(128) uint8_t kv[TI_SLOTS][TI_IMAGE];
  unsigned long long full[TI_SLOTS], empty[TI_SLOTS], q_ready, s_full[2], p_full[2], o_done[2];
  uint32_t tmem;
};

TQ_DEV void ti_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
TQ_DEV void ti_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(ta), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
#define TI_R8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
#define TI_W8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
TQ_DEV void ti_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : TI_W8(r, 0), TI_W8(r, 8), TI_W8(r, 16), TI_W8(r, 24)
      : "r"(addr)
      : "memory");
}
TQ_DEV void ti_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      TI_R8(r, 0), TI_R8(r, 8), TI_R8(r, 16), TI_R8(r, 24)
      : "memory");
}
TQ_DEV void ti_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
TQ_DEV void ti_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
TQ_DEV void ti_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
TQ_DEV void ti_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <bool SPLIT>
__global__ void __launch_bounds__(TI_THREADS, 1) attend_tiles_kernel(AttendArgs a, TileArgs ta) {
  extern __shared__ __align__(128) uint8_t ti_smem[];
  TiShared& sh = *(TiShared*)ti_smem;
  constexpr int PARTS = SPLIT ? 2 : 1;  // images of keys, and of values
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % ta.splits, rt = blockIdx.x / ta.splits % ta.row_tiles;
  const int unit = blockIdx.x / ta.splits / ta.row_tiles;
  if (ta.left[unit] != 0) return;
  const int G = g.group, s = unit / g.n_kv_heads, head = unit % g.n_kv_heads, row0 = rt * TI_ROWS;
  const AttendSeq sq = attend_seq(a, s);
  const AttendTiles ul = unit_tiles(a, sq);
  const int i_lo = row0 / G, i_hi = min(min(row0 + TI_ROWS, a.rows) - 1, sq.q_n * G - 1) / G;
  const int p_lo = sq.first + i_lo, p_hi = i_lo < sq.q_n ? sq.first + i_hi : -1;
  const AttendTiles tl = attend_tiles(a, 0, sq.n, TI_T, p_lo, p_hi);
  const int k_lo = (int)((long)tl.count() * split / ta.splits), n = (int)((long)tl.count() * (split + 1) / ta.splits) - k_lo;
  const int groups = a.rows - row0 > 128 ? 2 : 1;  // halves of the rows that there are

  const uint32_t q_bar = enc_smem(&sh.q_ready);
  if (tid == 0) {
    for (int i = 0; i < TI_SLOTS; ++i) {
      mbar_init(enc_smem(&sh.full[i]), 1);
      mbar_init(enc_smem(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(enc_smem(&sh.s_full[i]), 1);
      mbar_init(enc_smem(&sh.p_full[i]), 128);
      mbar_init(enc_smem(&sh.o_done[i]), 1);
    }
    mbar_init(q_bar, 128 * groups);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(enc_smem(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ti_fence_before();
  __syncthreads();
  ti_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)&sh.tmem;

  // Bounded waits: one that runs out sets the status bit, and the thread then waits for nothing more.
  const int limit = TI_WAIT;
  bool gave_up = false;
  auto wait = [&](unsigned long long* bar, unsigned parity) {
    const uint32_t at = enc_smem(bar);
    for (int i = 0; !gave_up && !mbar_try_wait(at, parity);)
      if (++i >= limit) {
        atomicOr(a.status, TQ_STATUS_WAIT_TIMEOUT);
        gave_up = true;
      }
  };

  if (warp == 9) {
    // ---- loads: K V of tile after tile through the ring
    if (lane == 0) {
      const uint8_t* images = ta.images + (size_t)unit * ta.cap * 2 * PARTS * TI_IMAGE;
      int c = 0;
      for (int k = 0; k < n; ++k) {
        const int t = tl.at(k_lo + k), slot_of = t < ul.head ? t : ul.head + t - ul.first;
        const uint8_t* from = images + (size_t)slot_of * 2 * PARTS * TI_IMAGE;
        for (int i = 0; i < 2 * PARTS; ++i, ++c) {
          const int slot = c % TI_SLOTS;
          if (c >= TI_SLOTS) wait(&sh.empty[slot], (c / TI_SLOTS - 1) & 1);
          if (gave_up) break;
          const uint32_t bar = enc_smem(&sh.full[slot]);
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(TI_IMAGE) : "memory");
          asm volatile(
              "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                  enc_smem(sh.kv[slot])),
              "l"(from + (size_t)i * TI_IMAGE), "r"(TI_IMAGE), "r"(bar)
              : "memory");
        }
      }
      // (the copies have all landed before the CTA's memory goes)
      gave_up = false;
      for (int i = max(c - TI_SLOTS, 0); i < c; ++i) wait(&sh.full[i % TI_SLOTS], (i / TI_SLOTS) & 1);
    }
  } else if (warp == 8) {
    // ---- products
    if (lane == 0 && n > 0) {
      constexpr uint32_t idesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint64_t STEP = 2 * TI_LBO >> 4;  // 16 deep
      auto image = [&](int c) { return umma_desc_k_major(enc_smem(sh.kv[c % TI_SLOTS]), TI_LBO, TI_SBO); };
      auto landed = [&](int c) { wait(&sh.full[c % TI_SLOTS], (c / TI_SLOTS) & 1); };
      // scores of half x against the keys of tile k
      auto scores = [&](int x, int k) {
        const uint64_t q = umma_desc_k_major(enc_smem(sh.q[x]), TI_LBO, TI_SBO);
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) {
          const uint64_t b = image(2 * PARTS * k + i);
#pragma unroll
          for (int j = 0; j < 8; ++j) ti_mma(tmem + 128 * x, q + j * STEP, b + j * STEP, idesc, i < PARTS - 1 || j > 0);
        }
        umma_commit(enc_smem(&sh.s_full[x]));
      };
      auto release = [&](int c) {  // the parts of an operand, once the products issued so far are done
        for (int i = 0; i < PARTS; ++i) umma_commit(enc_smem(&sh.empty[(c + i) % TI_SLOTS]));
      };
      wait(&sh.q_ready, 0);
      for (int i = 0; i < PARTS; ++i) landed(i);
      ti_fence_after();
      for (int x = 0; x < groups; ++x) scores(x, 0);
      release(0);
      for (int k = 0; k < n; ++k) {
        const int cv = 2 * PARTS * k + PARTS, ck = cv + PARTS;  // values of this tile, keys of the next
        for (int i = 0; i < PARTS; ++i) landed(cv + i);
        if (k + 1 < n)
          for (int i = 0; i < PARTS; ++i) landed(ck + i);
        for (int x = 0; x < groups; ++x) {
          wait(&sh.p_full[x], k & 1);
          ti_fence_after();
#pragma unroll
          for (int i = PARTS - 1; i >= 0; --i) {
            const uint64_t b = image(cv + i);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              ti_mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * j, b + j * STEP, idesc, k > 0 || i < PARTS - 1 || j > 0);
          }
          umma_commit(enc_smem(&sh.o_done[x]));
          if (x == groups - 1) release(cv);
          if (k + 1 < n) {
            // the next scores take the place of the probabilities that these products read
            wait(&sh.o_done[x], k & 1);
            scores(x, k + 1);
          }
        }
        if (k + 1 < n) release(ck);
      }
      gave_up = false;  // (nor are products under way then)
      for (int x = 0; x < groups; ++x) wait(&sh.o_done[x], (n - 1) & 1);
    }
  } else if (warp < 4 * groups) {
    // ---- a thread per row
    const int x = warp >> 2, r = tid & 127, row = row0 + tid;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + 128 * x + lanes, to = tmem + 256 + 128 * x + lanes;
    float factor;
    {
      uint4 raw[16];
      const bool there = row < a.rows;
      const uint16_t* q = (const uint16_t*)a.q + ((int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok +
                                                  (int64_t)(head * G + row % G) * a.q_head);
#pragma unroll
      for (int i = 0; i < 16; ++i) raw[i] = there ? *(const uint4*)(q + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
      auto pair = [&](uint32_t w) -> float2 {
        if (a.q_dtype == TQ_F16) return __half22float2(*(const __half2*)&w);
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      };
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair(w[j]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      float exponent;
      const float up = ti_lift(top, 13, exponent);
      factor = tq_scaled<true>(TI_KEY * exp2f(exponent));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair(w[j]);
          h[j] = ti_pair(f.x * up, f.y * up);
        }
        *(uint4*)(sh.q[x] + i * TI_LBO + r * 16) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_bar);
    }
    const int p = row < a.rows ? attend_position(a, sq, row) : -1, w = attend_window(a, p);
    // rows of this CTA: the earliest one that sees anything, the latest window
    const bool whole = row0 + TI_ROWS <= a.rows && i_lo < sq.q_n && (row0 + TI_ROWS - 1) / G < sq.q_n && p_lo >= 0;
    const int w_hi = attend_window(a, max(p_hi, 0));
    float m = -INFINITY, l = 0.0f;
    for (int k = 0; k < n; ++k) {
      const int t = tl.at(k_lo + k), t0 = t * TI_T;
      const float e = ta.exponent[(size_t)unit * ta.cap + (t < ul.head ? t : ul.head + t - ul.first)];
      wait(&sh.s_full[x], k & 1);
      gave_up = __any_sync(0xffffffffu, gave_up);
      ti_fence_after();
      uint32_t v[128];
#pragma unroll
      for (int i = 0; i < 4; ++i) ti_ld32(ts + 32 * i, v + 32 * i);
      ti_wait_ld();
      if (!(whole && t0 + TI_T - 1 <= p_lo && (t0 >= w_hi || t0 + TI_T <= a.sinks))) {
        const int hi = min(p, sq.n - 1) - t0, lo = w - t0, sk = a.sinks - t0;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > hi || (i < lo && i >= sk)) v[i] = 0xff800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[i]));
      const float now = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), factor, e);
      const bool grown = now > m + TI_GROW;  // (also from -inf)
      float down = 1.0f;
      if (grown) {
        down = tq_exp2(m - now);
        m = now;
      }
      if (k > 0 && __any_sync(0xffffffffu, grown)) {
        wait(&sh.o_done[x], (k - 1) & 1);
        gave_up = __any_sync(0xffffffffu, gave_up);
        ti_fence_after();
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          uint32_t o[32];
          ti_ld32(to + 32 * i, o);
          ti_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * down);
          ti_st32(to + 32 * i, o);
        }
      }
      const float off = TI_LIFT + e - (m > -INFINITY ? m : 0.0f);
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t h[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float y = tq_exp2(fmaf(__uint_as_float(v[64 * i + 2 * j]), factor, off));
          const float z = tq_exp2(fmaf(__uint_as_float(v[64 * i + 2 * j + 1]), factor, off));
          sum[j & 3] += y + z;
          h[j] = ti_pair(y, z);
        }
        ti_st32(ts + 32 * i, h);
      }
      ti_wait_st();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.p_full[x]));
      l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), exp2f(-e), l * down);
    }
    // the row's state: [channel][row], neighbouring threads side by side
    const size_t part = ((size_t)unit * ta.splits + split) * ta.row_tiles + rt;
    float* stats = ta.stats + part * 2 * TI_ROWS + tid;
    stats[0] = n > 0 ? m - TI_LIFT : -INFINITY;
    stats[TI_ROWS] = l;
    if (n > 0) {
      wait(&sh.o_done[x], (n - 1) & 1);
      gave_up = __any_sync(0xffffffffu, gave_up);
      ti_fence_after();
      float* sums = ta.sums + (size_t)unit * a.unit_stride + ((size_t)split * ta.row_tiles + rt) * TI_ROWS * TQ_D + tid;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        uint32_t o[32];
        ti_ld32(to + 32 * i, o);
        ti_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) sums[(32 * i + j) * TI_ROWS] = __uint_as_float(o[j]);
      }
    }
  }
  __syncwarp();
  ti_fence_before();
  __syncthreads();
  if (warp == 8) {
    ti_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------
// 64 rows of a unit: the splits' sums in order, sum @ Pi, over the sum of the weights.
constexpr int TC_ROWS = 64, TC_THREADS = 256, TC_S = TC_ROWS + 4;
__global__ void __launch_bounds__(TC_THREADS) attend_tiles_combine_kernel(AttendArgs a, TileArgs ta, int tiles) {
  __shared__ __align__(16) float c[TQ_D][TC_S];
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, unit = blockIdx.x / tiles, row0 = blockIdx.x % tiles * TC_ROWS;
  const int H = g.n_kv_heads, G = g.group, s = unit / H, head = unit % H;
  const int rows = min(TC_ROWS, a.rows - row0);
  if (ta.left[unit] != 0) {  // the general kernel's states: blocks and window, the latter not in code space
    for (int i = tid; i < rows * TQ_D; i += TC_THREADS) {
      const int r = i / TQ_D, e = i % TQ_D, row = row0 + r;
      const float* p = attend_partial(a, unit, row, 0);
      const float* q = p + TQ_PART_STRIDE;
      const float M = fmaxf(p[0], q[0]), by = M > -INFINITY ? M : 0.0f;
      const float wp = p[1] == 0.0f ? 0.0f : p[0] > -INFINITY ? tq_exp2(p[0] - by) : 1.0f;
      const float wq = q[1] == 0.0f ? 0.0f : q[0] > -INFINITY ? tq_exp2(q[0] - by) : 1.0f;
      float x = 0.0f;
      if (wp != 0.0f)
        for (int d = 0; d < TQ_D; ++d) x = fmaf(p[2 + d] * wp, a.tables->pi[d * TQ_D + e], x);
      if (wq != 0.0f) x = fmaf(q[2 + e], wq, x);
      const float L = (wp != 0.0f ? p[1] * wp : 0.0f) + (wq != 0.0f ? q[1] * wq : 0.0f);
      x = L == 0.0f ? 0.0f : x / L;
      const size_t at = (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D + e;
      if (a.q_dtype == TQ_F16) ((__half*)a.out)[at] = __float2half_rn(x);
      else ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(x);
    }
    return;
  }
  const int rt = row0 / TI_ROWS, in = row0 % TI_ROWS;
  {
    const int r = tid % TC_ROWS, d0 = tid / TC_ROWS * (TQ_D * TC_ROWS / TC_THREADS);
    float M = -INFINITY, L = 0.0f;
    float x[TQ_D * TC_ROWS / TC_THREADS];
    constexpr int N = TQ_D * TC_ROWS / TC_THREADS;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.0f;
    if (r < rows) {
      for (int i = 0; i < ta.splits; ++i)
        M = fmaxf(M, ta.stats[((((size_t)unit * ta.splits + i) * ta.row_tiles + rt) * 2) * TI_ROWS + in + r]);
      const float by = M > -INFINITY ? M : 0.0f;
      for (int i = 0; i < ta.splits; ++i) {
        const size_t part = ((size_t)unit * ta.splits + i) * ta.row_tiles + rt;
        const float mi = ta.stats[part * 2 * TI_ROWS + in + r], li = ta.stats[(part * 2 + 1) * TI_ROWS + in + r];
        if (li == 0.0f) continue;
        const float w = mi > -INFINITY ? tq_exp2(mi - by) : 1.0f;
        L += li * w;
        const float* from = ta.sums + (size_t)unit * a.unit_stride + (((size_t)i * ta.row_tiles + rt) * TQ_D + d0) * TI_ROWS + in + r;
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = fmaf(from[k * TI_ROWS], w, x[k]);
      }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int k = 0; k < N; ++k) c[d0 + k][r] = x[k] * inv;
  }
  __syncthreads();
  // a thread has 4 rows x 8 channels
  const int ty = tid >> 4, tx = tid & 15;
  float y[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = 0.0f;
#pragma unroll 4
  for (int d = 0; d < TQ_D; ++d) {
    const float4 r4 = *(const float4*)&c[d][4 * ty];
    const float4 p0 = *(const float4*)&a.tables->pi[d * TQ_D + 8 * tx], p1 = *(const float4*)&a.tables->pi[d * TQ_D + 8 * tx + 4];
    const float rr[4] = {r4.x, r4.y, r4.z, r4.w}, pp[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = fmaf(rr[i], pp[e], y[i][e]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i, row = row0 + r;
    if (r >= rows) continue;
    const size_t at = (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D + 8 * tx;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.q_dtype == TQ_F16) {
        w[e] = ti_pair(y[i][2 * e], y[i][2 * e + 1]);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(y[i][2 * e], y[i][2 * e + 1]);
        w[e] = *(const uint32_t*)&h;
      }
    }
    *(uint4*)((uint16_t*)a.out + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

struct Layout {
  size_t images, exponent, left, stats, sums, total;
  int64_t unit_stride;  // floats
};
Layout layout(const AttendArgs& a, int units, int cap, int splits) {
  const bool pairs = a.q_dtype == TQ_F16;
  const int row_tiles = (a.rows + TI_ROWS - 1) / TI_ROWS;
  Layout l;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t x = at;
    at += align_up(n, 256);
    return x;
  };
  l.images = take((size_t)units * cap * (pairs ? 4 : 2) * TI_IMAGE);
  l.exponent = take((size_t)units * cap * 4);
  l.left = take((size_t)units * 4);
  l.stats = take((size_t)units * splits * row_tiles * TI_ROWS * 2 * 4);
  // a unit's sums, or, if it is left to the general kernel, two states a row
  l.unit_stride = std::max((int64_t)splits * row_tiles * TI_ROWS * TQ_D, (int64_t)a.rows * 2 * TQ_PART_STRIDE);
  l.sums = take((size_t)units * l.unit_stride * 4);
  l.total = at;
  return l;
}

template <bool SPLIT>
int launch(const AttendArgs& a, const TileArgs& ta, int units, cudaStream_t st) {
  TQ_CUDA(cudaFuncSetAttribute(attend_stage_kernel<SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)sizeof(StageShared<SPLIT>)));
  TQ_CUDA(cudaFuncSetAttribute(attend_tiles_kernel<SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)sizeof(TiShared)));
  TQ_CUDA(cudaMemsetAsync(ta.left, 0, (size_t)units * 4, st));
  attend_stage_kernel<SPLIT><<<units * ta.cap, TS_THREADS, sizeof(StageShared<SPLIT>), st>>>(a, ta);
  TQ_CUDA(cudaGetLastError());
  attend_tiles_kernel<SPLIT><<<units * ta.splits * ta.row_tiles, TI_THREADS, sizeof(TiShared), st>>>(a, ta);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

}  // namespace

size_t tq_attend_tiles_bytes(const AttendArgs& a, int units, int cap, int splits) {
  return layout(a, units, cap, splits).total;
}

int tq_launch_attend_tiles(const AttendArgs& base, void* workspace, int cap, int splits, cudaStream_t st) {
  AttendArgs a = base;
  const int units = a.seq_count * a.g.n_kv_heads;
  const Layout l = layout(a, units, cap, splits);
  uint8_t* w = (uint8_t*)workspace;
  TileArgs ta;
  ta.images = w + l.images;
  ta.exponent = (float*)(w + l.exponent);
  ta.left = (int32_t*)(w + l.left);
  ta.sums = (float*)(w + l.sums);
  ta.stats = (float*)(w + l.stats);
  ta.cap = cap;
  ta.splits = splits;
  ta.row_tiles = (a.rows + TI_ROWS - 1) / TI_ROWS;
  const int64_t most = (int64_t)units * std::max(cap, splits * ta.row_tiles);
  const int tiles = (a.rows + TC_ROWS - 1) / TC_ROWS;
  TQ_REQUIRE(most <= INT_MAX && (int64_t)units * tiles <= INT_MAX, TQ_ERR_UNSUPPORTED,
             "too many (sequence, head, query row) tiles in a call");
  a.left = ta.left;
  a.ns_cold = a.ns_hot = 1;
  a.partials = ta.sums;
  a.unit_stride = l.unit_stride;
  int rc = a.q_dtype == TQ_F16 ? launch<true>(a, ta, units, st) : launch<false>(a, ta, units, st);
  if (rc != TQ_OK) return rc;
  rc = tq_launch_attend_general(a, st);
  if (rc != TQ_OK) return rc;
  attend_tiles_combine_kernel<<<units * tiles, TC_THREADS, 0, st>>>(a, ta, tiles);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

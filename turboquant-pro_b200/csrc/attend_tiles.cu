// Attention of many query rows per KV head on the codes: prompt chunks.  The products run on tcgen05 with the
// accumulators in tensor memory.  Three kernels:
//
// attend_stage_kernel   the tokens that any row sees, 80 at a time, from codes to the two shared-memory images
//     that tcgen05 takes as operands (fp16, K-major core matrices of 8 rows x 16 bytes), written to the workspace
//     once instead of once per tile of rows:
//       keys    mean + scale * grid[code] - c, outliers put over it.  c is one vector per (sequence, KV head),
//               the zero-point of its first block: it moves all scores of a row alike, so the softmax does not
//               see it, and large constant channels do not eat the half-precision digits.  All times the power of
//               two that takes the tile's largest below 2^15; its inverse is kept, for the scores.
//       values  transposed, in code space: norm * centroid[code], window tokens rotated into that space; all times
//               the power of two that takes the tile's largest norm below 2^15, whose exponent is kept.
//     What is not a number, keys beyond 2^20, and a token whose keys or values lie below 2^-20 of the tile's largest (zeros
//     aside: its digits would fall out of fp16) set the flag of their (sequence, KV head), which the general kernel
//     then does.
// attend_tiles_kernel   256 rows of a (sequence, KV head) per CTA against a split of these tiles, in two halves of 128 rows.
//     S = Q K^T into tensor memory; a group of 128 threads per half, a thread per row, makes the probabilities and
//     puts them back as fp16; O += P V with P as the operand in tensor memory.  Of its 512 columns a half has
//     80 for scores, 40 for probabilities and 128 for the sums: that is what sets the tile.  (With 128 tokens the
//     probabilities had to go over the scores, so that the next scores waited for the product that read them: a chain of
//     3 800 cycles a tile, in which neither the tensor cores nor the softmax were busy for more than half.)  As it is
//     the next scores are formed while the exponentials of these are.  A warp per half issues, one loads.
//     A tile's exponent is added to its scores, so that the running maximum is that of probability * value and fp16
//     holds what counts.  The maximum is only renewed (and O rescaled) when it has grown by 2^8 since.
// attend_tiles_combine_kernel   merges the splits, rotates the sums back (sum @ Pi), rounds.
//
// Measured, 8 KV heads of 4 query heads, bfloat16, by the clock that the power cap leaves: 2048 tokens on 32768 1 103 to
// 1 130 us, of which stage 83, tiles 914 to 935 (70 to 71 % of the rate of a large library product of as many
// operations, 4.3 GB/ms of operands from L2), merge 66; 512 tokens on 16384 210 us: 52, 141, 16; 777 float16 ones with a
// window of 2000 106 us: 18, 63, 22.  What bounds the tiles: a half's chain of waits, fetch, maximum and exponentials, 2
// 000 cycles of a period of 2 200, is covered by the other half alone.  Products (1 280 cycles a tile) have the tensor
// pipe busy for 56 % and exponentials (16 a cycle and SM: as long, but for the quarter that goes over the multiply-add
// units) the special-function units for 43 %: neither is full.  (An even division over the SMs, whose parts went on
// through a CTA's tiles of rows, took as long for 512 tokens on 148 SMs as this does on 128, at 1.65 GHz.)  Shares of
// exponentials on the multiply-add units of 1, 2, 3, 4, 5 eighths, before the keys had a power of two per tile: 899,
// 907, 923, 958, 994 us at 2048 tokens and 66.9, 64.7, 66.1, 67.0, 68.1 for 777 float16 ones.
//
// Queries are fp16 in shared memory, each row scaled by a power of two, which is exact for both 16-bit types (from 2^-27
// of a row's largest on).  SPLIT (float16 queries): keys and values as pairs hi + lo, so that only the probabilities
// are rounded to fp16 and the result is off by about its own rounding (2.4e-4 in 2-norms against 64 bits, where rounding the
// exact result gives 2.1e-4).  Bfloat16 queries take the hi parts alone, 2^-11 at worst against the half step of their type,
// 2^-8: scores of a deviation of five, with channels 20 times the others, are then off by 1e-3, and the result by 2.0 to
// 2.2e-3 instead of 1.65e-3; pairs would double the products.
#include <algorithm>

#include "attend.cuh"
#include "encode.cuh"  // mbarrier, descriptors, commit

namespace {

constexpr int TI_T = TQ_ATTEND_TILE;         // tokens of a tile
constexpr int TI_ROWS = 256;                 // rows of a CTA
constexpr int TI_IMAGE = TI_T * TQ_D * 2;    // bytes of an operand image of keys or values
constexpr int TI_QIMAGE = 128 * TQ_D * 2;    // and of a half's queries
constexpr int TI_KLBO = TI_T * 16, TI_LBO = TQ_D * 16, TI_SBO = 128;  // from eight K to the next: keys; queries, values
constexpr int TI_SLOTS = 8;                  // images in shared memory
constexpr int TI_SOFTMAX = 256;              // softmax threads: one a row
constexpr int TI_THREADS = TI_SOFTMAX + 96;  // and two warps that issue, a warp that loads
constexpr int TI_S = 0, TI_P = TI_T, TI_HALF = 128, TI_O = 256;  // columns: scores, probabilities of a half, sums
constexpr float TI_KEY_MOST = 0x1p20f, TI_LEAST = 0x1p-20f;  // largest key; least part of a tile's largest
constexpr float TI_LIFT = 7.0f, TI_GROW = 8.0f;  // probabilities reach 2^(7 + 8) at most
constexpr int TI_POLY = 2;                   // of eight pairs of exponentials, those on the multiply-add units
constexpr int TI_WAIT = 1 << 21;             // probes of a wait
static_assert(TI_P + TI_T / 2 <= TI_HALF && 2 * TI_HALF <= TI_O && TI_T % 16 == 0, "tensor memory's columns");

struct TileArgs {
  uint8_t* images;    // [unit][cap][K hi, (K lo,) V hi, (V lo)]
  float2* exponent;   // [unit][cap]: of the values; the keys' factor
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

// 2^(top - floor(log2 x)), and the exponent of its inverse; what is below 2^-63, or 2^(least - 127), counts as that
TQ_DEV float ti_lift(float x, int top, float& exponent, int least = 64) {
  const int e = min(max((int)(__float_as_uint(x) >> 23 & 255u), least), 254);
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

TQ_DEV void tc_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (a NaN stays)
TQ_DEV float ti_max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
constexpr int TS_THREADS = 4 * TI_T;  // four a token; two warps per 16 tokens of values
constexpr int TS_PITCH = TQ_D * 2 + 16;  // bytes per row of window values
constexpr int TS_VT = 16;         // window tokens that are rotated at a time
struct StageShared {
  alignas(16) float k[TQ_D / 4][TI_T][4];  // four channels a plane; afterwards rows of window values, as pairs hi + lo
  alignas(16) float center[TQ_D];
  float grid[16], cent[16], norm[TI_T];
  float top[TS_THREADS / 32], k_top[TS_THREADS / 32], part_top[4][TI_T];
};
static_assert(2 * TS_VT * TS_PITCH <= 2 * TI_IMAGE, "the window values' place");

// eight neighbouring elements of a window row
TQ_DEV void ts_ld8(const void* p, size_t at, int dt, float (&x)[8]) {
  if (dt == TQ_F32) {
    const float4 u = *(const float4*)((const float*)p + at), v = *(const float4*)((const float*)p + at + 4);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    return;
  }
  const uint4 u = *(const uint4*)((const uint16_t*)p + at);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == TQ_F16) {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <bool SPLIT>
__global__ void __launch_bounds__(TS_THREADS, SPLIT ? 2 : 3) attend_stage_kernel(AttendArgs a, TileArgs ta) {
  extern __shared__ __align__(16) uint8_t ts_smem[];
  StageShared& sh = *(StageShared*)ts_smem;
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
  const bool hot = t1 > sq.cold;  // some tokens are of the window

  // what is used later, on its way: the tile's first block's list, this thread's quarter of a token's codes
  PageMeta first = {0, 0};
  if (g.outlier_k > 0 && t0 < sq.cold) first = a.page_meta[uix * g.max_blocks + t0 / S];
  const int krow = tid % TI_T, kq = tid / TI_T, kt = t0 + krow, kb = kt / S, kslot = kt - kb * S;
  const uint8_t* const kpage = pages + (size_t)kb * g.page_bytes;
  uint4 codes = {0u, 0u, 0u, 0u};
  if (kt < sq.cold) codes = *(const uint4*)(kpage + kslot * (TQ_D / 2) + 16 * kq);
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
  bool odd = false;
  {  // ---- norms of the values: four threads a token
    const int row = tid >> 2, t = t0 + row;
    float norm = 0.0f;
    if (t < sq.cold) {
      const int b = t / S;
      norm = ((const float*)(pages + (size_t)b * g.page_bytes + g.norm_off))[t - b * S];
    }
    if (hot) {
      float ss = 0.0f;
      if (t >= sq.cold && t < t1) {
        const size_t at = ring + (size_t)(t % g.hot_cap) * TQ_D + (tid & 3) * (TQ_D / 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[8];
          ts_ld8(a.hot_v, at + 8 * i, g.kv_dtype, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        }
      }
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      if (t >= sq.cold) norm = sqrtf(ss);
    }
    odd |= !isfinite(norm);
    if ((tid & 3) == 0) sh.norm[row] = norm;
    float top = fabsf(norm);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sh.top[warp] = top;
  }
  __syncthreads();
  float most = 0.0f;
  {  // ---- keys: a thread has a quarter of a token
    auto put = [&](int chunk, const float (&x)[8]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) most = ti_max3_nan(most, fabsf(x[2 * i]), fabsf(x[2 * i + 1]));
      *(float4*)sh.k[2 * chunk][krow] = make_float4(x[0], x[1], x[2], x[3]);
      *(float4*)sh.k[2 * chunk + 1][krow] = make_float4(x[4], x[5], x[6], x[7]);
    };
    if (kt < sq.cold) {
      const float* sc = (const float*)(kpage + g.scale_off);
      const float* mu = (const float*)(kpage + g.mean_off);
      const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * kq + 8 * i;
        const float4 s0 = *(const float4*)(sc + d), s1 = *(const float4*)(sc + d + 4);
        const float4 m0 = *(const float4*)(mu + d), m1 = *(const float4*)(mu + d + 4);
        const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
        const float mm[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
        const float4 z0 = *(const float4*)&sh.center[d], z1 = *(const float4*)&sh.center[d + 4];
        const float zz[8] = {z0.x, z0.y, z0.z, z0.w, z1.x, z1.y, z1.z, z1.w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(ss[e], sh.grid[w[i] >> (4 * e) & 15], mm[e] - zz[e]);
        put(4 * kq + i, x);
      }
    } else {
      const size_t at = ring + (size_t)(kt % g.hot_cap) * TQ_D + 32 * kq;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[8];
        if (kt < t1) {
          ts_ld8(a.hot_k, at + 8 * i, g.kv_dtype, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= sh.center[32 * kq + 8 * i + e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        }
        put(4 * kq + i, x);
      }
    }
    odd |= !(most < TI_KEY_MOST);
    sh.part_top[kq][krow] = most;
  }
  __syncthreads();
  const float token_top =
      tid < TI_T ? fmaxf(fmaxf(sh.part_top[0][tid], sh.part_top[1][tid]), fmaxf(sh.part_top[2][tid], sh.part_top[3][tid])) : 0.0f;
  if (g.outlier_k > 0) {
    for (int b = t0 / S; b * S < min(t1, sq.cold); ++b) {
      const PageMeta pm = b == t0 / S ? first : a.page_meta[uix * g.max_blocks + b];
      const size_t slab = uix * (size_t)g.pool_entries + pm.off;
#pragma unroll 3
      for (uint32_t e = tid; e < pm.cnt; e += TS_THREADS) {
        const uint32_t w = a.pool_dec[slab + e];
        const __half val = __ushort_as_half(a.pool_val[slab + e]);
        const int t = b * S + (int)(w >> 24), ch = (w >> 16) & 127;
        if (t < t0 || t >= t1) continue;
        const float x = __half2float(val) - sh.center[ch];
        odd |= !(fabsf(x) < TI_KEY_MOST);
        most = fmaxf(most, fabsf(x));
        sh.k[ch >> 2][t - t0][ch & 3] = x;
      }
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) sh.k_top[warp] = most;
  odd = __syncthreads_or(odd);
  if (odd && tid == 0) ta.left[unit] = 1;
#pragma unroll
  for (int w = 0; w < TS_THREADS / 32; ++w) most = fmaxf(most, sh.k_top[w]);
  if (token_top > 0.0f && token_top < most * TI_LEAST) ta.left[unit] = 1;
  // (from 2^-30 on: the factor times a row's own stays a number above zero)
  float k_exponent;
  const float k_up = ti_lift(most, 14, k_exponent, 97);
  uint8_t* const images = ta.images + ((size_t)unit * ta.cap + idx) * (SPLIT ? 4 : 2) * TI_IMAGE;
#pragma unroll
  for (int i = tid; i < TI_IMAGE / 16; i += TS_THREADS) {  // eight channels of a token
    const int chunk = i / TI_T, row = i - chunk * TI_T;
    const float4 x = *(const float4*)sh.k[2 * chunk][row], y = *(const float4*)sh.k[2 * chunk + 1][row];
    const uint4 hi = {ti_pair(x.x * k_up, x.y * k_up), ti_pair(x.z * k_up, x.w * k_up), ti_pair(y.x * k_up, y.y * k_up),
                      ti_pair(y.z * k_up, y.w * k_up)};
    *(uint4*)(images + 16 * i) = hi;
    if (SPLIT)
      *(uint4*)(images + TI_IMAGE + 16 * i) =
          make_uint4(ti_rest(x.x * k_up, x.y * k_up, hi.x), ti_rest(x.z * k_up, x.w * k_up, hi.y),
                     ti_rest(y.x * k_up, y.y * k_up, hi.z), ti_rest(y.z * k_up, y.w * k_up, hi.w));
  }

  // ---- values
  float top = 0.0f, exponent;
#pragma unroll
  for (int w = 0; w < TS_THREADS / 32; ++w) top = fmaxf(top, sh.top[w]);
  const float up = ti_lift(top, 14, exponent);
  if (tid < TI_T && sh.norm[tid] != 0.0f && fabsf(sh.norm[tid]) < top * TI_LEAST) ta.left[unit] = 1;
  if (tid == 0) ta.exponent[(size_t)unit * ta.cap + idx] = make_float2(exponent, exp2f(k_exponent));
  uint8_t* const v_hi = images + (SPLIT ? 2 : 1) * TI_IMAGE;
  uint8_t* const v_lo = v_hi + TI_IMAGE;
  if (!hot && S % TQ_GROUP_TOK == 0) {
    // two warps expand the records of a group of 16 tokens: two tokens of a channel are a word of the image
    const int grp_i = warp >> 1, part = warp & 1, t = t0 + grp_i * TQ_GROUP_TOK, b = t / S, slot = t - b * S;
    const int r = lane >> 2, c = lane & 3;
    const bool there = t < t1;
    const uint8_t* grp = pages + (size_t)(there ? b : 0) * g.page_bytes + g.v_off + (size_t)(there ? slot >> 4 : 0) * v_group_bytes(vb);
    uint32_t w[4];  // pairs 16 part .. + 15
    if (vb == 4) {
      const uint4 x = *(const uint4*)(grp + part * 512 + lane * 16);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      // the record's 24 bytes; these pairs are words 3 part .. + 2
      const uint2 r0 = *(const uint2*)(grp + lane * 8), r1 = *(const uint2*)(grp + 256 + lane * 8), r2 = *(const uint2*)(grp + 512 + lane * 8);
      w[0] = part ? r1.y : r0.x, w[1] = part ? r2.x : r0.y, w[2] = part ? r2.y : r1.x, w[3] = 0u;
    }
    float nv[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x) nv[h][x] = there ? sh.norm[grp_i * TQ_GROUP_TOK + 8 * h + 2 * c + x] * up : 0.0f;
#pragma unroll
    for (int p = 0; p < 16; ++p) {
      const int h = p & 1, d = r + 8 * (8 * part + (p >> 1));
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
      const int at = (2 * grp_i + h) * TI_LBO + d * 16 + 4 * c;
      *(uint32_t*)(v_hi + at) = hi;
      if (SPLIT) *(uint32_t*)(v_lo + at) = ti_rest(x, y, hi);
    }
    return;
  }
  // Window tokens are rotated, v @ Pi^T, on mma.sync: 16 tokens at a time as pairs hi + lo are the B operand, a warp's 16
  // output channels, whose rows of Pi are pairs too, the A operand.  Tokens of blocks in the same tile come
  // from their codes one by one.
  uint8_t* const vs = (uint8_t*)sh.k;
  const int q = lane >> 2, c = lane & 3;
#pragma unroll 1
  for (int n0 = 0; n0 < TI_T; n0 += TS_VT) {
    float d[TS_VT / 8][4];
#pragma unroll
    for (int nt = 0; nt < TS_VT / 8; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[nt][i] = 0.0f;
    if (t0 + n0 + TS_VT > sq.cold && t0 + n0 < t1) {
      __syncthreads();  // (the keys, or the rows before, have been read)
      if (tid < TS_VT * 16) {
        const int row = tid >> 4, ch = (tid & 15) * 8, t = t0 + n0 + row;
        float v[8];
        if (t >= sq.cold && t < t1) {
          ts_ld8(a.hot_v, ring + (size_t)(t % g.hot_cap) * TQ_D + ch, g.kv_dtype, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = ti_pair(v[2 * i] * up, v[2 * i + 1] * up);
          lo[i] = ti_rest(v[2 * i] * up, v[2 * i + 1] * up, hi[i]);
        }
        *(uint4*)(vs + row * TS_PITCH + 2 * ch) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *(uint4*)(vs + (TS_VT + row) * TS_PITCH + 2 * ch) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      __syncthreads();
      if (warp < 8)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = *(const float2*)&a.tables->pi[(16 * warp + q + 8 * (i & 1)) * TQ_D + 16 * k + 2 * c + 8 * (i >> 1)];
          ph[i] = ti_pair(x.x * 256.0f, x.y * 256.0f);
          pl[i] = ti_rest(x.x * 256.0f, x.y * 256.0f, ph[i]);
        }
#pragma unroll
        for (int nt = 0; nt < TS_VT / 8; ++nt) {
          const uint8_t* at = vs + (8 * nt + q) * TS_PITCH + 32 * k + 4 * c;
          const uint32_t h0 = *(const uint32_t*)at, h1 = *(const uint32_t*)(at + 16);
          const uint32_t l0 = *(const uint32_t*)(at + TS_VT * TS_PITCH), l1 = *(const uint32_t*)(at + TS_VT * TS_PITCH + 16);
          tc_mma(d[nt], pl, h0, h1);
          tc_mma(d[nt], ph, l0, l1);
          tc_mma(d[nt], ph, h0, h1);
        }
      }
    }
    if (warp >= 8) continue;
#pragma unroll
    for (int nt = 0; nt < TS_VT / 8; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {  // channels q, q + 8 of the warp's sixteen; tokens 2 c, 2 c + 1
        const int ch = 16 * warp + q + 8 * y, n = n0 + 8 * nt + 2 * c;
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int t = t0 + n + e;
          x[e] = d[nt][2 * y + e] * (1.0f / 256.0f);
          if (t < sq.cold) {
            const int b = t / S, slot = t - b * S;
            const uint8_t* grp = pages + (size_t)b * g.page_bytes + g.v_off + (size_t)(slot >> 4) * v_group_bytes(vb);
            x[e] = sh.norm[n + e] * up * sh.cent[v_get_code(grp, vb, slot & 15, ch)];
          }
        }
        const uint32_t hi = ti_pair(x[0], x[1]);
        const int at = (n >> 3) * TI_LBO + ch * 16 + (n & 7) * 2;
        *(uint32_t*)(v_hi + at) = hi;
        if (SPLIT) *(uint32_t*)(v_lo + at) = ti_rest(x[0], x[1], hi);
      }
  }
}

// ---------------------------------------------------------------------------------------------------
struct TiShared {
  alignas(128) uint8_t q[2][TI_QIMAGE];
  alignas(128) uint8_t kv[TI_SLOTS][TI_IMAGE];
  unsigned long long full[TI_SLOTS], empty[TI_SLOTS], q_ready[2], s_full[2], s_read[2], p_full[2], o_done[2],
      drained[2];
  uint32_t tmem;
};
static_assert(sizeof(TiShared) <= 227 * 1024, "shared memory of one CTA");

// (accumulate: known where the call stands, so that no predicate has to be formed)
template <bool ACC>
TQ_DEV void ti_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
               "l"(da), "l"(db), "r"(idesc), "n"(ACC ? 1 : 0)
               : "memory");
}
template <bool ACC>
TQ_DEV void ti_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
               "r"(ta), "l"(db), "r"(idesc), "n"(ACC ? 1 : 0)
               : "memory");
}
TQ_DEV bool ti_elect() {  // one thread of the (converged) warp
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(on));
  return on != 0;
}
// (without a time to sleep: the waiting threads have little slack)
TQ_DEV bool ti_try_wait(uint32_t bar, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
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
TQ_DEV void ti_ld16(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : TI_W8(r, 0), TI_W8(r, 8)
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
TQ_DEV void ti_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), TI_R8(r, 0) : "memory");
}
TQ_DEV float ti_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// pairs of floats in one register pair
TQ_DEV uint64_t ti_u2(uint32_t a, uint32_t b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "r"(a), "r"(b));
  return y;
}
TQ_DEV uint64_t ti_f2(float a, float b) { return ti_u2(__float_as_uint(a), __float_as_uint(b)); }
TQ_DEV float2 ti_floats(uint64_t x) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
  return y;
}
TQ_DEV uint64_t ti_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
TQ_DEV uint64_t ti_add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
// 2^x on the special-function units, which do 16 a cycle and SM; and on the multiply-add units: x = n + f with n whole
// and |f| <= 1/2, a polynomial of degree 4 for 2^f (Remez exchange on the relative error: 2.6e-6 at all six extrema), n
// added to its exponent.  Both together finish sooner than either.  The polynomial takes what is below 2^-120 for
// that.
TQ_DEV float ti_exp2(float x) {  // (results below 2^-126 are zero: nothing next to the row's largest, and one instruction)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
TQ_DEV float2 ti_exp2_unit(uint64_t x) {
  const float2 y = ti_floats(x);
  return make_float2(ti_exp2(y.x), ti_exp2(y.y));
}
TQ_DEV float2 ti_exp2_poly(uint64_t x) {
  const float2 y = ti_floats(x);
  const uint64_t z = ti_f2(fmaxf(y.x, -120.0f), fmaxf(y.y, -120.0f));
  const uint64_t n = ti_add2(z, ti_f2(12582912.0f, 12582912.0f));  // 1.5 * 2^23: whole numbers in the low bits
  const uint64_t f = ti_fma2(ti_add2(n, ti_f2(-12582912.0f, -12582912.0f)), ti_f2(-1.0f, -1.0f), z);
  uint64_t p = ti_fma2(ti_f2(0.009570101791435913f, 0.009570101791435913f), f, ti_f2(0.05591786030999481f, 0.05591786030999481f));
  p = ti_fma2(p, f, ti_f2(0.24024744830820266f, 0.24024744830820266f));
  p = ti_fma2(p, f, ti_f2(0.6931218147384395f, 0.6931218147384395f));
  p = ti_fma2(p, f, ti_f2(0.9999992614448223f, 0.9999992614448223f));
  const float2 m = ti_floats(n), w = ti_floats(p);
  return make_float2(__uint_as_float(__float_as_uint(w.x) + (__float_as_uint(m.x) << 23)),
                     __uint_as_float(__float_as_uint(w.y) + (__float_as_uint(m.y) << 23)));
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

  if (tid == 0) {
    for (int i = 0; i < TI_SLOTS; ++i) {
      mbar_init(enc_smem(&sh.full[i]), 1);
      mbar_init(enc_smem(&sh.empty[i]), groups);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(enc_smem(&sh.s_full[i]), 1);
      mbar_init(enc_smem(&sh.q_ready[i]), 128);
      mbar_init(enc_smem(&sh.s_read[i]), 128);
      mbar_init(enc_smem(&sh.p_full[i]), 128);
      mbar_init(enc_smem(&sh.o_done[i]), 1);
      mbar_init(enc_smem(&sh.drained[i]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == TI_SOFTMAX / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(enc_smem(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ti_fence_before();
  __syncthreads();
  ti_fence_after();
  constexpr uint32_t tmem = 0;  // (all 512 columns are this CTA's: they begin at the first)

  // Bounded waits: one that runs out sets the status bit, and the thread then waits for nothing more and starts no
  // copies or products; those under way are waited for (with the full limit) before the CTA's memory goes.
  const int limit = a.wait_limit > 0 ? a.wait_limit : TI_WAIT;
  bool gave_up = false;
  auto wait_for = [&](unsigned long long* bar, unsigned parity, int most) {
    const uint32_t at = enc_smem(bar);
    for (int i = 0; !gave_up && !ti_try_wait(at, parity);)
      if (++i >= most) {
        atomicOr(a.status, TQ_STATUS_WAIT_TIMEOUT);
        gave_up = true;
      }
  };
  auto wait = [&](unsigned long long* bar, unsigned parity) { wait_for(bar, parity, limit); };

  if (warp == TI_SOFTMAX / 32 + 2) {
    // ---- loads: K V of tile after tile through the ring
    if (lane == 0) {
      const uint8_t* images = ta.images + (size_t)unit * ta.cap * 2 * PARTS * TI_IMAGE;
      const int held = blockIdx.x == 0 ? a.withhold : -1;  // test hook: an image that is never copied
      int c = 0;
      for (int k = 0; k < n && !gave_up; ++k) {
        const int t = tl.at(k_lo + k), slot_of = t < ul.head ? t : ul.head + t - ul.first;
        const uint8_t* from = images + (size_t)slot_of * 2 * PARTS * TI_IMAGE;
        for (int i = 0; i < 2 * PARTS; ++i, ++c) {
          const int slot = c % TI_SLOTS;
          if (c >= TI_SLOTS) wait(&sh.empty[slot], (c / TI_SLOTS - 1) & 1);
          if (gave_up) break;
          if (c == held) continue;
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
      for (int i = max(c - TI_SLOTS, 0); i < c; ++i)
        if (i != held) wait_for(&sh.full[i % TI_SLOTS], (i / TI_SLOTS) & 1, TI_WAIT);
    }
  } else if (warp >= TI_SOFTMAX / 32) {
    // ---- products of half x
    // The whole warp runs this, one thread issues.  What the products take are constants or the same in all lanes to
    // the compiler's knowledge (the shuffle), so that it lies in uniform registers: fetched there product by product,
    // each took about a hundred cycles to issue, more than its execution.
    const int x = warp - TI_SOFTMAX / 32, n_u = __shfl_sync(0xffffffffu, x < groups ? n : 0, 0);
    if (n_u > 0) {
      constexpr uint32_t s_desc = (1u << 4) | ((uint32_t)(TI_T >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t o_desc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint64_t KSTEP = 2 * TI_KLBO >> 4, STEP = 2 * TI_LBO >> 4;  // 16 deep
      const uint64_t q = umma_desc_k_major(enc_smem(sh.q[0]), TI_LBO, TI_SBO) + (uint64_t)(x * (TI_QIMAGE >> 4));
      const uint64_t k0 = umma_desc_k_major(enc_smem(sh.kv[0]), TI_KLBO, TI_SBO);
      const uint64_t v0 = umma_desc_k_major(enc_smem(sh.kv[0]), TI_LBO, TI_SBO);
      const uint32_t ds = tmem + TI_S + TI_HALF * x, dp = tmem + TI_P + TI_HALF * x, d_o = tmem + TI_O + 128 * x;
      auto image = [&](int c) { return (uint64_t)((uint32_t)(c % TI_SLOTS) * (TI_IMAGE >> 4)); };
      auto wait_all = [&](unsigned long long* bar, unsigned parity) {  // (the warp stays together)
        wait(bar, parity);
        gave_up = __any_sync(0xffffffffu, gave_up);
      };
      auto landed = [&](int c) { wait_all(&sh.full[c % TI_SLOTS], (c / TI_SLOTS) & 1); };
      auto release = [&](int c) {  // an operand's parts, once the products issued so far are done (the issuing thread)
#pragma unroll
        for (int i = 0; i < PARTS; ++i) umma_commit(enc_smem(&sh.empty[(c + i) % TI_SLOTS]));
      };
      // scores against the keys of tile k
      auto scores = [&](int k) {
        const int c = 2 * PARTS * k;
        uint64_t b[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) b[i] = k0 + image(c + i);
        if (ti_elect()) {
          ti_mma<false>(ds, q, b[PARTS - 1], s_desc);
#pragma unroll
          for (int j = 1; j < 8; ++j) ti_mma<true>(ds, q + j * STEP, b[PARTS - 1] + j * KSTEP, s_desc);
          if (SPLIT)
#pragma unroll
            for (int j = 0; j < 8; ++j) ti_mma<true>(ds, q + j * STEP, b[0] + j * KSTEP, s_desc);
          umma_commit(enc_smem(&sh.s_full[x]));
          release(c);
        }
        __syncwarp();
      };
      // O += P V
      auto values = [&](int k) {
        const int c = 2 * PARTS * k + PARTS;
        uint64_t b[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) b[i] = v0 + image(c + i);
        if (ti_elect()) {
          if (k == 0) ti_mma_ts<false>(d_o, dp, b[PARTS - 1], o_desc);
          else ti_mma_ts<true>(d_o, dp, b[PARTS - 1], o_desc);
#pragma unroll
          for (int j = 1; j < TI_T / 16; ++j) ti_mma_ts<true>(d_o, dp + 8 * j, b[PARTS - 1] + j * STEP, o_desc);
          if (SPLIT)
#pragma unroll
            for (int j = 0; j < TI_T / 16; ++j) ti_mma_ts<true>(d_o, dp + 8 * j, b[0] + j * STEP, o_desc);
          umma_commit(enc_smem(&sh.o_done[x]));
          release(c);
        }
        __syncwarp();
      };
      wait_all(&sh.q_ready[x], 0);
      for (int i = 0; i < PARTS; ++i) landed(i);
      ti_fence_after();
      if (!gave_up) scores(0);
#pragma unroll 1
      for (int k = 0; k < n_u && !gave_up; ++k) {
        if (k + 1 < n_u) {
          for (int i = 0; i < PARTS; ++i) landed(2 * PARTS * (k + 1) + i);
          wait_all(&sh.s_read[x], k & 1);  // (this tile's scores are in registers)
          if (gave_up) break;
          ti_fence_after();
          scores(k + 1);
        }
        for (int i = 0; i < PARTS; ++i) landed(2 * PARTS * k + PARTS + i);
        wait_all(&sh.p_full[x], k & 1);
        if (gave_up) break;
        ti_fence_after();
        values(k);
      }
      // (nor are products under way when the CTA's memory goes: a barrier of one phase tells, however many of the
      // others' there have been)
      if (ti_elect()) umma_commit(enc_smem(&sh.drained[x]));
      __syncwarp();
      gave_up = false;
      wait_for(&sh.drained[x], 0, TI_WAIT);
    }
  } else if (warp < 4 * groups) {
    // ---- a thread per row
    const int x = warp >> 2, r = tid & 127, row = row0 + 128 * x + r;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + TI_S + TI_HALF * x + lanes, tp = tmem + TI_P + TI_HALF * x + lanes;
    const uint32_t to = tmem + TI_O + 128 * x + lanes;
    auto settled = [&](unsigned long long* bar, unsigned parity) {
      wait(bar, parity);
      __syncwarp();
      ti_fence_after();
    };
    float factor;
    {
      uint4 raw[16];
      const bool there = row < a.rows;
      const uint16_t* q = (const uint16_t*)a.q + ((int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok +
                                                  (int64_t)(head * G + row % G) * a.q_head);
#pragma unroll
      for (int i = 0; i < 16; ++i) raw[i] = there ? *(const uint4*)(q + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
      auto pair = [&](uint32_t w) -> float2 {
        if (SPLIT) return __half22float2(*(const __half2*)&w);
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
      factor = tq_scaled<true>(exp2f(exponent));
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
      mbar_arrive(enc_smem(&sh.q_ready[x]));
    }
    const int p = row < a.rows ? attend_position(a, sq, row) : -1, w = attend_window(a, p);
    // whether all rows of this CTA see a tile goes by their earliest position and latest window
    const bool whole = row0 + TI_ROWS <= a.rows && i_lo < sq.q_n && (row0 + TI_ROWS - 1) / G < sq.q_n && p_lo >= 0;
    const int w_hi = attend_window(a, max(p_hi, 0));
    const float2* const exponents = ta.exponent + (size_t)unit * ta.cap;
    auto tile_of = [&](int k) { return tl.at(k_lo + min(k, n - 1)); };
    auto exponent_of = [&](int t) { return exponents[t < ul.head ? t : ul.head + t - ul.first]; };
    float m = -INFINITY, l = 0.0f;
    int t = n > 0 ? tile_of(0) : 0;
    float2 of_tile = n > 0 ? exponent_of(t) : make_float2(0.0f, 0.0f);
    if (groups == 2 && x == 1 && n > 0) asm volatile("bar.arrive 1, 256;" ::: "memory");
    for (int k = 0; k < n; ++k) {
      const int t0 = t * TI_T;
      // (the next tile's exponent and factor, on their way from memory while this one is done)
      const int t_next = tile_of(k + 1);
      const float2 next = exponent_of(t_next);
      const float e = of_tile.x, by = factor * of_tile.y;
      settled(&sh.s_full[x], k & 1);
      uint32_t v[TI_T];
      ti_ld32(ts, v);
      ti_ld32(ts + 32, v + 32);
      ti_ld16(ts + 64, v + 64);
      ti_wait_ld();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.s_read[x]));
      const bool open = whole && t0 + TI_T - 1 <= p_lo && (t0 >= w_hi || t0 + TI_T <= a.sinks);
      if (!open) {
        const int hi = min(p, sq.n - 1) - t0, lo = w - t0, sk = a.sinks - t0;
#pragma unroll
        for (int i = 0; i < TI_T; ++i)
          if (i > hi || (i < lo && i >= sk)) v[i] = 0xff800000u;
      }
      float top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) top[i] = fmaxf(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
#pragma unroll
      for (int i = 16; i < TI_T; i += 2)
        top[i / 2 & 7] = ti_max3(top[i / 2 & 7], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
      top[0] = ti_max3(top[0], top[1], top[2]);
      top[3] = ti_max3(top[3], top[4], top[5]);
      top[0] = ti_max3(ti_max3(top[0], top[3], top[6]), top[7], -INFINITY);
      const float now = fmaf(top[0], by, e);
      const bool grown = now > m + TI_GROW;  // (also from -inf)
      float down = 1.0f;
      if (grown) {
        down = tq_exp2(m - now);
        m = now;
      }
      const bool rescaled = k > 0 && __any_sync(0xffffffffu, grown);
      if (rescaled) {
        settled(&sh.o_done[x], (k - 1) & 1);
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
      if (k > 0 && !rescaled) settled(&sh.o_done[x], (k - 1) & 1);  // (the probabilities before have been used)
      // The halves take turns at their exponentials, which fill the unit for them (16 a cycle and SM): while one is at
      // them, the other waits for its scores, fetches them and finds their largest.  Left to themselves both did the
      // same at the same time (950 us for 2048 tokens on 32768; with turns 907, both before the keys' power of two).
      if (groups == 2) asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");
      const float off = TI_LIFT + e - (m > -INFINITY ? m : 0.0f);
      const uint64_t factor2 = ti_f2(by, by), off2 = ti_f2(off, off);
      uint64_t sum[2] = {0ull, 0ull};
      uint32_t h[TI_T / 2];
      if (open) {
#pragma unroll
        for (int j = 0; j < TI_T / 2; ++j) {
          const uint64_t y = ti_fma2(ti_u2(v[2 * j], v[2 * j + 1]), factor2, off2);
          const float2 z = j % 8 < TI_POLY ? ti_exp2_poly(y) : ti_exp2_unit(y);
          sum[j & 1] = ti_add2(sum[j & 1], ti_f2(z.x, z.y));
          h[j] = ti_pair(z.x, z.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < TI_T / 2; ++j) {
          const float2 z = ti_exp2_unit(ti_fma2(ti_u2(v[2 * j], v[2 * j + 1]), factor2, off2));
          sum[j & 1] = ti_add2(sum[j & 1], ti_f2(z.x, z.y));
          h[j] = ti_pair(z.x, z.y);
        }
      }
      ti_st32(tp, h);
      ti_st8(tp + 32, h + 32);
      if (groups == 2 && (x == 0 || k + 1 < n)) asm volatile("bar.arrive %0, 256;" ::"r"(2 - x) : "memory");
      ti_wait_st();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.p_full[x]));
      const float2 s2 = ti_floats(ti_add2(sum[0], sum[1]));
      l = fmaf(s2.x + s2.y, exp2f(-e), l * down);
      t = t_next, of_tile = next;
    }
    // the row's state: [channel][row], neighbouring threads side by side
    const size_t at = ((size_t)unit * ta.splits + split) * ta.row_tiles + rt;
    float* stats = ta.stats + at * 2 * TI_ROWS + 128 * x + r;
    stats[0] = n > 0 ? m - TI_LIFT : -INFINITY;
    stats[TI_ROWS] = l;
    if (n > 0) {
      settled(&sh.o_done[x], (n - 1) & 1);
      float* sums = ta.sums + (size_t)unit * a.unit_stride + ((size_t)split * ta.row_tiles + rt) * TQ_D * TI_ROWS + 128 * x + r;
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
  if (warp == TI_SOFTMAX / 32) {
    ti_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------
// The splits' sums in order, over the sum of the weights, times Pi.  CTAs take tiles of 64 rows in turn.  The
// merged rows go to shared memory as fp16 pairs hi + lo, each row scaled by a power of two, and through mma.sync as the
// B operand against Pi^T, whose pairs lie there too, a warp taking 16 channels of the output: hi * hi + hi * lo +
// lo * hi, good to 2^-22, with an accumulator each.
constexpr int TC_ROWS = 64, TC_THREADS = 256;
struct CombineShared {
  alignas(128) uint8_t ph[TQ_D * 256], pl[TQ_D * 256], hi[TC_ROWS * 256], lo[TC_ROWS * 256];
  float top[TC_THREADS / 32][TC_ROWS], inv[TC_ROWS];
};
// Byte of eight neighbouring columns of a row: neither eight rows in a row nor every fourth of 32 share a bank.
TQ_DEV int tc_at(int row, int c8) { return row * 256 + ((c8 ^ (row >> 2 & 7) ^ (row & 3) << 1) << 4); }
TQ_DEV void tc_ldmatrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__global__ void __launch_bounds__(TC_THREADS, 2) attend_tiles_combine_kernel(AttendArgs a, TileArgs ta, int tiles, int total) {
  extern __shared__ __align__(128) uint8_t tc_smem[];
  CombineShared& sh = *(CombineShared*)tc_smem;
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, q = lane >> 2, c = lane & 3;
  const int H = g.n_kv_heads, G = g.group;
  for (int i = tid; i < TQ_D * 16; i += TC_THREADS) {  // (read behind the tile's first barrier)
    const int row = i >> 4, c8 = i & 15;
    const float4 u = *(const float4*)&a.tables->pi_t[row * TQ_D + 8 * c8], v = *(const float4*)&a.tables->pi_t[row * TQ_D + 8 * c8 + 4];
    const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = ti_pair(x[2 * k] * 256.0f, x[2 * k + 1] * 256.0f);
      l[k] = ti_rest(x[2 * k] * 256.0f, x[2 * k + 1] * 256.0f, h[k]);
    }
    *(uint4*)(sh.ph + tc_at(row, c8)) = make_uint4(h[0], h[1], h[2], h[3]);
    *(uint4*)(sh.pl + tc_at(row, c8)) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const int unit = item / tiles, row0 = item % tiles * TC_ROWS, s = unit / H, head = unit % H;
    const int rows = min(TC_ROWS, a.rows - row0);
    auto out_at = [&](int row) {
      return (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D;
    };
    if (ta.left[unit] != 0) {  // the general kernel's states: blocks and window, the latter not in code space
      for (int i = tid; i < rows * TQ_D; i += TC_THREADS) {
        const int e = i % TQ_D, row = row0 + i / TQ_D;
        const float* x = attend_partial(a, unit, row, 0);
        const float* y = x + TQ_PART_STRIDE;
        const float M = fmaxf(x[0], y[0]), by = M > -INFINITY ? M : 0.0f;
        const float wx = x[1] == 0.0f ? 0.0f : x[0] > -INFINITY ? tq_exp2(x[0] - by) : 1.0f;
        const float wy = y[1] == 0.0f ? 0.0f : y[0] > -INFINITY ? tq_exp2(y[0] - by) : 1.0f;
        float o = 0.0f;
        if (wx != 0.0f)
          for (int d = 0; d < TQ_D; ++d) o = fmaf(x[2 + d] * wx, a.tables->pi[d * TQ_D + e], o);
        if (wy != 0.0f) o = fmaf(y[2 + e], wy, o);
        const float L = (wx != 0.0f ? x[1] * wx : 0.0f) + (wy != 0.0f ? y[1] * wy : 0.0f);
        o = L == 0.0f ? 0.0f : o / L;
        if (a.q_dtype == TQ_F16) ((__half*)a.out)[out_at(row) + e] = __float2half_rn(o);
        else ((__nv_bfloat16*)a.out)[out_at(row) + e] = __float2bfloat16_rn(o);
      }
      continue;
    }
    // a thread: eight channels of four rows
    const int rt = row0 / TI_ROWS, in = row0 % TI_ROWS, r4 = tid % 16 * 4, c8 = tid / 16;
    float x[4][8], L[4] = {0.0f, 0.0f, 0.0f, 0.0f}, M[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
    const float* stats = ta.stats + ((size_t)unit * ta.splits * ta.row_tiles + rt) * 2 * TI_ROWS + in + r4;
    const size_t step = (size_t)ta.row_tiles * 2 * TI_ROWS;
    const float* sums = ta.sums + (size_t)unit * a.unit_stride + ((size_t)rt * TQ_D + c8 * 8) * TI_ROWS + in + r4;
    for (int i = 0; i < ta.splits; ++i) {
      const float4 m = *(const float4*)(stats + i * step);
      M[0] = fmaxf(M[0], m.x), M[1] = fmaxf(M[1], m.y), M[2] = fmaxf(M[2], m.z), M[3] = fmaxf(M[3], m.w);
    }
#pragma unroll 2
    for (int i = 0; i < ta.splits; ++i) {
      const float4 m4 = *(const float4*)(stats + i * step), l4 = *(const float4*)(stats + i * step + TI_ROWS);
      const float* from = sums + (size_t)i * ta.row_tiles * TI_ROWS * TQ_D;
      float4 f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = *(const float4*)(from + k * TI_ROWS);
      const float m[4] = {m4.x, m4.y, m4.z, m4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (a split that saw nothing of the row may not have written its sums)
        if (l[j] == 0.0f) continue;
        const float w = m[j] > -INFINITY ? tq_exp2(m[j] - (M[j] > -INFINITY ? M[j] : 0.0f)) : 1.0f;
        L[j] += l[j] * w;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[j][k] = fmaf(j == 0 ? f[k].x : j == 1 ? f[k].y : j == 2 ? f[k].z : f[k].w, w, x[j][k]);
      }
    }
    float top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top[j] = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) top[j] = fmaxf(top[j], fabsf(x[j][k]));
      top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
    }
    __syncthreads();  // (the tile before has been read)
    if (lane < 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) sh.top[warp][r4 + j] = top[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float t = 0.0f, exponent;
#pragma unroll
      for (int i = 0; i < TC_THREADS / 32; ++i) t = fmaxf(t, sh.top[i][r4 + j]);
      const float up = ti_lift(t, 13, exponent);
      if (c8 == 0) sh.inv[r4 + j] = L[j] == 0.0f ? 0.0f : exp2f(exponent - 8.0f) / L[j];
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = x[j][2 * i] * up, v = x[j][2 * i + 1] * up;
        h[i] = ti_pair(u, v);
        l[i] = ti_rest(u, v, h[i]);
      }
      *(uint4*)(sh.hi + tc_at(r4 + j, c8)) = make_uint4(h[0], h[1], h[2], h[3]);
      *(uint4*)(sh.lo + tc_at(r4 + j, c8)) = make_uint4(l[0], l[1], l[2], l[3]);
    }
    __syncthreads();
    uint32_t ph[8][4], pl[8][4];  // A: rows = output channels 16 warp .., k = input channels
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = tc_at(16 * warp + (lane & 15), 2 * k + (lane >> 4));
      tc_ldmatrix(ph[k], enc_smem(sh.ph + at));
      tc_ldmatrix(pl[k], enc_smem(sh.pl + at));
    }
#pragma unroll 2
    for (int nt = 0; nt < TC_ROWS / 8; ++nt) {
      if (8 * nt >= rows) break;
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f}, d1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, d2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t h[4], l[4];
        const int at = tc_at(8 * nt + (lane & 7), 2 * k + (lane >> 3));
        tc_ldmatrix(h, enc_smem(sh.hi + at));
        tc_ldmatrix(l, enc_smem(sh.lo + at));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          tc_mma(d1, pl[k + i], h[2 * i], h[2 * i + 1]);
          tc_mma(d2, ph[k + i], l[2 * i], l[2 * i + 1]);
          tc_mma(d, ph[k + i], h[2 * i], h[2 * i + 1]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] += d1[i] + d2[i];
      // channels q, q + 8 of the warp's sixteen; rows 2 c, 2 c + 1
      const float f0 = sh.inv[8 * nt + 2 * c], f1 = sh.inv[8 * nt + 2 * c + 1];
      uint32_t w[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float u = d[2 * y] * f0, v = d[2 * y + 1] * f1;
        if (a.q_dtype == TQ_F16) {
          w[y] = ti_pair(u, v);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(u, v);
          w[y] = *(const uint32_t*)&h;
        }
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w[y]) : "r"(w[y]));
      }
      const int row = 8 * nt + q;  // now two neighbouring channels of row q
      if (row < rows) {
        uint16_t* to = (uint16_t*)a.out + out_at(row0 + row) + 16 * warp + 2 * c;
        *(uint32_t*)to = w[0];
        *(uint32_t*)(to + 8) = w[1];
      }
    }
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
  l.exponent = take((size_t)units * cap * 8);
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
  static bool stage_done[64], tiles_done[64];
  int rc = attend_shared(attend_stage_kernel<SPLIT>, sizeof(StageShared), a.device, stage_done);
  if (rc == TQ_OK) rc = attend_shared(attend_tiles_kernel<SPLIT>, sizeof(TiShared), a.device, tiles_done);
  if (rc != TQ_OK) return rc;
  TQ_CUDA(cudaMemsetAsync(ta.left, 0, (size_t)units * 4, st));
  attend_stage_kernel<SPLIT><<<units * ta.cap, TS_THREADS, sizeof(StageShared), st>>>(a, ta);
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
  ta.exponent = (float2*)(w + l.exponent);
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
  static bool combine_done[64];
  rc = attend_shared(attend_tiles_combine_kernel, sizeof(CombineShared), a.device, combine_done);
  if (rc != TQ_OK) return rc;
  attend_tiles_combine_kernel<<<std::min(units * tiles, 2 * a.sm_count), TC_THREADS, sizeof(CombineShared), st>>>(a, ta, tiles, units * tiles);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

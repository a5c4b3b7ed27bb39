// Attention of few query rows per KV head on the codes: single tokens, drafts to verify, small chunks.
// 256-token blocks with per-channel keys; the products on mma.sync (m16n8k16) with the codes as the A operand,
// straight from a table into registers, and NT tiles of eight query rows as the B operand.
//
// A CTA of eight warps takes one (sequence, KV head), one tile of rows and one split of the pages that
// these rows see (first tokens, then the window).  Pages come in whole with cp.async, the next one while this one is
// attended; a warp attends 32 of the page's 256 tokens:
//   weights  w = q * scale, scaled by a power of two per row, as an fp16 pair hi + lo in the layout of the
//            B operand, and the zero-points' part of the score, q . mean: once per page, a row per warp;
//   scores   a byte of key codes (two channels) is one look-up; hi * w and lo * w accumulate apart;
//   mask     by position, where a row of the tile does not see the whole strip;
//   softmax  running maximum and sum per row and warp, in units of log 2;
//   values   probability * norm, scaled by a power of two per row and strip, transposed in registers into the
//            B operand; two tokens' codes of a channel are one look-up.  The sums of a strip start from zero and are
//            added in float32.
//
// SPLIT (float32 and float16 queries): the table's entries are hi + lo pairs too, hi * hi of 16 channels is added
// up in float32 registers, and outliers count with their exact stored value: as exact as float32 arithmetic.
// bfloat16 queries leave the table's lo part out (2^-12 of a level; their own step is 2^-8), and take the outliers
// from the page's list by token, which holds their distance from the grid in fp16.
//
// The uncompressed window is converted, 128 tokens at a time, to fp16 rows in shared memory (hi, and lo with
// SPLIT), each token scaled by a power of two, and goes through the same steps with ldmatrix.  A tile that holds
// an infinity or a NaN is attended term by term instead: products with masked tokens would spread it.
//
// Bound by the issue slots of look-ups and products; at one row tile the codes are read once.
#include "attend.cuh"

namespace {

constexpr int AR_THREADS = 256, AR_WARPS = 8;
constexpr int AR_S = 256;          // tokens of a page
constexpr int AR_STRIP = 32;       // of them, a warp's
constexpr int AR_HOT = 128;        // window tokens of a tile
constexpr int AR_PITCH = TQ_D * 2 + 16;  // bytes of a converted row
constexpr int AR_LIST = 1024;      // outliers of a page that are copied ahead (640 is usual)

template <int NT, bool SPLIT, int VB>
struct ArShape {
  static constexpr int N = 8 * NT;                     // query rows
  static constexpr int NV = VB == 4 ? 256 : 64;
  // copies of a table side by side: 16 pairs fill a half warp's banks; of single words as many as leave
  // room for two CTAs on an SM
  static constexpr int REP = SPLIT ? 16 : (VB == 4 ? 8 : 16);
  static constexpr int ENTRY = REP * (SPLIT ? 8 : 4);  // bytes of an entry, copies and all
  static constexpr int LUTK = 256 * ENTRY, LUTV = NV * ENTRY;
  static constexpr int PAGE = AR_S * TQ_D / 2 + AR_S * TQ_D * VB / 8 + AR_S * 4 + 2 * TQ_D * 4 + TQ_TAIL_BYTES;
  static constexpr int LIST = SPLIT ? AR_LIST * 6 : 0;
  static constexpr int STAGE = PAGE + LIST;
  static constexpr int COLD = LUTK + LUTV + 2 * STAGE;
  static constexpr int HOT = AR_HOT * AR_PITCH * (SPLIT ? 4 : 2) + AR_HOT * 8;
  static constexpr int AREA = COLD > HOT ? COLD : HOT;
  static constexpr int WROW = 33 * 16;                 // bytes of a k-step's B fragments, padded
};

template <int NT, bool SPLIT, int VB>
struct ArShared {
  using Sh = ArShape<NT, SPLIT, VB>;
  alignas(128) uint8_t area[Sh::AREA];
  alignas(16) uint8_t w[NT][8][Sh::WROW];  // [tile][k-step][lane] {b0 hi, b1 hi, b0 lo, b1 lo}
  alignas(16) float corr[AR_S][Sh::N];     // outliers' part of the scores; at the end the merged sums
  alignas(16) float q[TQ_D][Sh::N];        // row q_row(d): channel d
  float bias[Sh::N], inv[Sh::N];
  float m[AR_WARPS][Sh::N], l[AR_WARPS][Sh::N];
  int pos[Sh::N], win[Sh::N];
  float grid[16], cent[16];
};

TQ_DEV void ar_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}
TQ_DEV uint32_t ar_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
// a * x and b * y as fp16 pairs hi + lo; lo takes what the products' rounding drops, too
TQ_DEV void ar_split(float a, float x, float b, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a * x, b * y);
  const float2 f = __half22float2(h);
  hi = *(const uint32_t*)&h;
  lo = ar_pair(fmaf(a, x, -f.x), fmaf(b, y, -f.y));
}
TQ_DEV uint32_t ar_transpose(uint32_t v) {  // of an 8x8 matrix of 16-bit elements
  uint32_t o;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
  return o;
}
// 2^(top - floor(log2 x)) and its inverse; zero, denormals, infinities and NaN count as the nearest ordinary
// exponent
TQ_DEV float ar_lift(float x, int top, float& inverse) {
  const int e = min(max((int)(__float_as_uint(x) >> 23 & 255u), 32), 254);
  inverse = __int_as_float((e - top) << 23);
  return __int_as_float((254 + top - e) << 23);
}
TQ_DEV uint32_t ar_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
TQ_DEV void ar_cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ar_smem(dst)), "l"(src) : "memory");
}
TQ_DEV void ar_cp8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(ar_smem(dst)), "l"(src) : "memory");
}
TQ_DEV void ar_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
TQ_DEV uint32_t ar_lut1(uint32_t addr) {  // (the tables do not change: not volatile)
  uint32_t v;
  asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
TQ_DEV uint2 ar_lut2(uint32_t addr) {
  uint2 v;
  asm("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
template <bool TRANS>
TQ_DEV void ar_ldm(uint32_t (&a)[4], uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
}

template <int NT, bool SPLIT, int VB>
__global__ void __launch_bounds__(AR_THREADS, !SPLIT&& NT == 1 ? 2 : 1)
    attend_rows_kernel(AttendArgs a, int row_tiles) {
  using Sh = ArShape<NT, SPLIT, VB>;
  constexpr int N = Sh::N;
  constexpr int VGB = TQ_GROUP_TOK * TQ_D * VB / 8;
  extern __shared__ __align__(128) uint8_t ar_shared[];
  ArShared<NT, SPLIT, VB>& sh = *(ArShared<NT, SPLIT, VB>*)ar_shared;
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int ns = a.ns_cold + a.ns_hot;
  const int split = blockIdx.x % ns, rt = blockIdx.x / ns % row_tiles, unit = blockIdx.x / ns / row_tiles;
  const int H = g.n_kv_heads, G = g.group;
  const int s = unit / H, head = unit - s * H, row0 = rt * N;
  const AttendSeq sq = attend_seq(a, s);
  const bool is_cold = split < a.ns_cold;
  const size_t uix = unit_index(g, a.layer, a.seq_begin + s, head);

  // ---- what this CTA attends
  const int i_lo = row0 / G, i_hi = min(min(row0 + N, a.rows) - 1, sq.q_n * G - 1) / G;
  const int p_lo = sq.first + i_lo, p_hi = i_lo < sq.q_n ? sq.first + i_hi : -1;
  const int base = is_cold ? 0 : sq.cold, end = is_cold ? sq.cold : sq.n, size = is_cold ? AR_S : AR_HOT;
  const AttendTiles tl = attend_tiles(a, base, end, size, p_lo, p_hi);
  const int part = is_cold ? split : split - a.ns_cold, parts = is_cold ? a.ns_cold : a.ns_hot;
  const int k_lo = (int)((long)tl.count() * part / parts), k_hi = (int)((long)tl.count() * (part + 1) / parts);

  // ---- pages on their way
  uint8_t* const stages = sh.area + Sh::LUTK + Sh::LUTV;
  const uint8_t* const pages = a.pages + page_offset(g, a.layer, a.seq_begin + s, head, 0);
  auto meta_of = [&](int k) -> PageMeta {
    PageMeta pm = {0, 0};
    if (SPLIT && g.outlier_k > 0 && k < k_hi) pm = a.page_meta[uix * g.max_blocks + tl.at(k)];
    return pm;
  };
  auto listed = [&](const PageMeta& pm) { return pm.cnt <= (uint32_t)AR_LIST && (pm.off & 3u) == 0u; };
  auto fetch = [&](int k, const PageMeta& pm) {
    uint8_t* to = stages + (k & 1) * Sh::STAGE;
    const uint8_t* from = pages + (size_t)tl.at(k) * g.page_bytes;
    for (int i = tid; i < Sh::PAGE / 16; i += AR_THREADS) ar_cp16(to + 16 * i, from + 16 * i);
    if (SPLIT && listed(pm)) {
      const size_t slab = uix * (size_t)g.pool_entries + pm.off;
      const int n4 = (int)(pm.cnt + 3) / 4;  // (slices are whole fours, and slabs whole sixty-fours, of entries)
      for (int i = tid; i < n4; i += AR_THREADS) {
        ar_cp16(to + Sh::PAGE + 16 * i, a.pool_dec + slab + 4 * i);
        ar_cp8(to + Sh::PAGE + 4 * AR_LIST + 8 * i, a.pool_val + slab + 4 * i);
      }
    }
  };
  PageMeta meta[2];
  if (is_cold && k_lo < k_hi) {
    meta[k_lo & 1] = meta_of(k_lo);
    fetch(k_lo, meta[k_lo & 1]);
    ar_commit();
    meta[(k_lo + 1) & 1] = meta_of(k_lo + 1);
  }

  // ---- tables, queries
  if (tid < 16) {
    sh.grid[tid] = a.tables->grid[tid];
    sh.cent[tid] = a.tables->centroids[tid];
  }
  for (int i = tid; i < N; i += AR_THREADS) {
    const int row = row0 + i;
    sh.pos[i] = row < a.rows ? attend_position(a, sq, row) : -1;
    sh.win[i] = attend_window(a, sh.pos[i]);
  }
  float qv[NT][4];  // rows warp, warp + 8, ...: channels 4 lane .. + 3, times the scores' unit
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + 8 * t + warp;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = 0.0f;
      if (row < a.rows)
        x = attend_ld(a.q, (size_t)((int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok +
                                    (int64_t)(head * G + row % G) * a.q_head + 4 * lane + i), a.q_dtype);
      qv[t][i] = tq_scaled<true>(x);
      sh.q[q_row(4 * lane + i)][8 * t + warp] = qv[t][i];
    }
  }
  __syncthreads();
  float inv_k = 1.0f, inv_v = 1.0f;
  if (is_cold && k_lo < k_hi) {
    float max_k = 0.0f, max_v = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      max_k = fmaxf(max_k, fabsf(sh.grid[i]));
      max_v = fmaxf(max_v, fabsf(sh.cent[i]));
    }
    const float up_k = ar_lift(max_k, 7, inv_k), up_v = ar_lift(max_v, 7, inv_v);
    for (int e = tid; e < 256 + Sh::NV; e += AR_THREADS) {
      uint32_t hi, lo;
      uint4* to;
      if (e < 256) {
        ar_split(sh.grid[e & 15], up_k, sh.grid[e >> 4], up_k, hi, lo);
        to = (uint4*)(sh.area + e * Sh::ENTRY);
      } else {
        const int b = e - 256;
        ar_split(sh.cent[b & ((1 << VB) - 1)], up_v, sh.cent[b >> VB], up_v, hi, lo);
        to = (uint4*)(sh.area + Sh::LUTK + b * Sh::ENTRY);
      }
#pragma unroll
      for (int i = 0; i < Sh::ENTRY / 16; ++i)
        to[(i + lane) % (Sh::ENTRY / 16)] = SPLIT ? make_uint4(hi, lo, hi, lo) : make_uint4(hi, hi, hi, hi);
    }
  }

  // rows 8 t + 2 c + x are this lane's columns
  float acc[NT][8][4], m_run[NT][2], l_run[NT][2];
  int first_pos = INT_MAX, last_win = 0;  // the earliest row that sees anything; the latest window
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][mt][i] = 0.0f;
#pragma unroll
    for (int x = 0; x < 2; ++x) m_run[t][x] = -INFINITY, l_run[t][x] = 0.0f;
  }
  for (int i = 0; i < N; ++i) {
    first_pos = min(first_pos, row0 + i < a.rows ? sh.pos[i] : INT_MAX);
    last_win = max(last_win, sh.win[i]);
  }

  // From the scores of `tiles` times 16 tokens from `t0` on to the B operand of their values: maximum and sum go
  // on, probability * nv is scaled by a power of two per row.
  auto softmax = [&](float (&sc)[2][NT][4], int t0, int t_end, int tiles, const float (&nv)[2][2],
                     uint32_t (&ph)[2][NT][2], uint32_t (&pl)[2][NT][2], float (&inv_n)[NT][2]) {
    const bool open = t0 + 16 * tiles <= t_end && t0 + 16 * tiles - 1 <= first_pos &&
                      (t0 >= last_win || t0 + 16 * tiles <= a.sinks);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t hidden = tiles == 1 ? 0xcu : 0u;  // (only one tile of 16)
        if (!open) {
          const int p = sh.pos[8 * t + 2 * c + x], w = sh.win[8 * t + 2 * c + x];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int j = t0 + 16 * h + 8 * y + r;
              if (j >= t_end || j > p || (j < w && j >= a.sinks)) hidden |= 1u << (2 * h + y);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (!(hidden >> (2 * h + y) & 1u)) top = fmaxf(top, sc[h][t][2 * y + x]);
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(m_run[t][x], top);
        // (-inf: nothing seen yet, or scores that are no numbers, which stay so)
        const float by = top > -INFINITY ? top : 0.0f, down = tq_exp2(m_run[t][x] - by);
        float sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float e = hidden >> (2 * h + y) & 1u ? 0.0f : tq_exp2(sc[h][t][2 * y + x] - by);
            sum += e;
            sc[h][t][2 * y + x] = e;
            most = fmaxf(most, fabsf(e * nv[h][y]));
          }
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        m_run[t][x] = top;
        l_run[t][x] = fmaf(l_run[t][x], down, sum);
        const float up = ar_lift(most, 13, inv_n[t][x]);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          acc[t][mt][x] *= down;
          acc[t][mt][2 + x] *= down;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) sc[h][t][2 * y + x] *= up;
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t hi, lo;
          // (a hidden token's norm may be anything)
          const float n0 = sc[h][t][2 * y] == 0.0f ? 0.0f : nv[h][y], n1 = sc[h][t][2 * y + 1] == 0.0f ? 0.0f : nv[h][y];
          ar_split(sc[h][t][2 * y], n0, sc[h][t][2 * y + 1], n1, hi, lo);
          ph[h][t][y] = ar_transpose(hi);
          if (SPLIT) pl[h][t][y] = ar_transpose(lo);
        }
  };
  // acc += values (A: channels 16 mt .. + 15 of a group's tokens) * probabilities
  auto add_values = [&](int mt, const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&ph)[NT][2],
                        const uint32_t (&pl)[NT][2], const float (&inv_n)[NT][2], float by) {
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float d[4];
      if (SPLIT) {
        ar_mma(d, al, ph[t][0], ph[t][1], zero);
        ar_mma(d, ah, pl[t][0], pl[t][1], d);
        ar_mma(d, ah, ph[t][0], ph[t][1], d);
      } else {
        ar_mma(d, ah, ph[t][0], ph[t][1], zero);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][mt][i] = fmaf(d[i], inv_n[t][i & 1] * by, acc[t][mt][i]);
    }
  };
  // hi (and lo) of a row's four channels as B operands, scaled so that the largest is just below 2^14
  auto row_lift = [&](const float (&w)[4], float& inverse) -> float {
    float mx = fmaxf(fmaxf(fabsf(w[0]), fabsf(w[1])), fmaxf(fabsf(w[2]), fabsf(w[3])));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    return ar_lift(mx, 13, inverse);
  };

  if (is_cold) {
    const uint32_t lutk = ar_smem(sh.area) + (lane % Sh::REP) * (SPLIT ? 8 : 4);
    const uint32_t lutv = lutk + Sh::LUTK;
    for (int k = k_lo; k < k_hi; ++k) {
      const uint8_t* page = stages + (k & 1) * Sh::STAGE;
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();  // the page has landed; the one before it, its weights and corrections have been read
      const PageMeta pm = meta[k & 1];
      if (k + 1 < k_hi) {
        fetch(k + 1, meta[(k + 1) & 1]);
        ar_commit();
        meta[k & 1] = meta_of(k + 2);
      }
      {  // weights: k-step j of lane group c takes channels 32 c + 4 j .. + 3
        const float4 s4 = *(const float4*)(page + g.scale_off + 16 * lane);
        const float4 m4 = *(const float4*)(page + g.mean_off + 16 * lane);
        const float sc[4] = {s4.x, s4.y, s4.z, s4.w}, mu[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float w[4], b = 0.0f, inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = qv[t][i] * sc[i];
            b = fmaf(qv[t][i], mu[i], b);
          }
          const float up = row_lift(w, inv);
#pragma unroll
          for (int o = 16; o >= 1; o >>= 1) b += __shfl_xor_sync(0xffffffffu, b, o);
          uint4 f;
          ar_split(qv[t][0] * up, sc[0], qv[t][1] * up, sc[1], f.x, f.z);
          ar_split(qv[t][2] * up, sc[2], qv[t][3] * up, sc[3], f.y, f.w);
          *(uint4*)(sh.w[t][lane & 7] + (4 * warp + (lane >> 3)) * 16) = f;
          if (lane == 0) {
            sh.bias[8 * t + warp] = b;
            sh.inv[8 * t + warp] = inv * inv_k;
          }
        }
      }
      const PageHeader* hdr = (const PageHeader*)(page + g.hdr_off);
      auto add_corr = [&](float (&e)[N], float delta, int qrow) {
#pragma unroll
        for (int x = 0; x < N; x += 4) {
          const float4 q4 = *(const float4*)&sh.q[qrow][x];
          e[x] = fmaf(q4.x, delta, e[x]), e[x + 1] = fmaf(q4.y, delta, e[x + 1]);
          e[x + 2] = fmaf(q4.z, delta, e[x + 2]), e[x + 3] = fmaf(q4.w, delta, e[x + 3]);
        }
      };
      // (columns of a token's row in an order that spreads eight tokens over the banks)
      auto put_corr = [&](int tok, const float (&e)[N]) {
#pragma unroll
        for (int x = 0; x < N; x += 4)
          *(float4*)&sh.corr[tok][x ^ (4 * (tok >> 2 & 1))] = make_float4(e[x], e[x + 1], e[x + 2], e[x + 3]);
      };
      if (g.outlier_k > 0) {
        float e[N];
#pragma unroll
        for (int x = 0; x < N; ++x) e[x] = 0.0f;
        if (SPLIT) {
          // the pool's list, ordered by token: the thread that holds a token's first entry adds up all of them
          put_corr(tid, e);
          __syncthreads();
          const uint32_t* dec;
          const uint16_t* val;
          if (listed(pm)) {
            dec = (const uint32_t*)(page + Sh::PAGE);
            val = (const uint16_t*)(page + Sh::PAGE + 4 * AR_LIST);
          } else {
            dec = a.pool_dec + uix * (size_t)g.pool_entries + pm.off;
            val = a.pool_val + uix * (size_t)g.pool_entries + pm.off;
          }
          for (uint32_t i = tid; i < pm.cnt; i += AR_THREADS) {
            const int tok = (int)(dec[i] >> 24);
            if (i > 0 && (int)(dec[i - 1] >> 24) == tok) continue;
#pragma unroll
            for (int x = 0; x < N; ++x) e[x] = 0.0f;
            for (uint32_t j = i; j < pm.cnt && (int)(dec[j] >> 24) == tok; ++j) {
              const int ch = (dec[j] >> 16) & 127;
              const float on_grid = sh.grid[page[tok * (TQ_D / 2) + (ch >> 1)] >> (4 * (ch & 1)) & 15];
              const float sc = ((const float*)(page + g.scale_off))[ch], mu = ((const float*)(page + g.mean_off))[ch];
              // what the weights' part gives is taken off, and the value itself put in
              add_corr(e, fmaf(-sc, on_grid, __half2float(__ushort_as_half(val[j])) - mu), q_row(ch));
            }
            put_corr(tok, e);
          }
        } else {
          const uint8_t* col = page + g.hdr_off + TQ_ELL_COL_OFF;
          const uint16_t* delta = (const uint16_t*)(page + g.hdr_off + TQ_ELL_OFF);
          const bool spilled = (hdr->flags & TQ_PAGE_SPILLED) != 0;
          if (!spilled) {
#pragma unroll
            for (int j = 0; j < TQ_ELL_SLOTS; ++j)
              add_corr(e, __half2float(__ushort_as_half(delta[j * AR_S + tid])), col[j * AR_S + tid]);
          }
          put_corr(tid, e);
          __syncwarp();
          // the rest of the list, ordered by token, as above
          const uint32_t* list = (const uint32_t*)(page + g.hdr_off + TQ_OVF_OFF);
          int e0 = hdr->ovf_start[warp >> 1], e1 = hdr->ovf_start[(warp >> 1) + 1];
          if (spilled) {
            list = a.pool_dec + uix * (size_t)g.pool_entries + hdr->off;
            e0 = 0, e1 = (int)hdr->cnt;
          }
          for (int i = e0 + lane; i < e1; i += 32) {
            uint32_t v = list[i];
            const int tok = (int)(v >> 24);
            if (tok >> 5 != warp || (i > e0 && (int)(list[i - 1] >> 24) == tok)) continue;
#pragma unroll
            for (int x = 0; x < N; ++x) e[x] = sh.corr[tok][x ^ (4 * (tok >> 2 & 1))];
            for (int j = i;;) {
              add_corr(e, __half2float(__ushort_as_half((unsigned short)(v & 0xffffu))), q_row((v >> 16) & 127));
              if (++j >= e1) break;
              v = list[j];
              if ((int)(v >> 24) != tok) break;
            }
            put_corr(tok, e);
          }
        }
      }
      __syncthreads();  // weights and corrections are there

      // ---- this warp's 32 tokens
      const int ts = AR_STRIP * warp, t0 = tl.at(k) * AR_S + ts;
      if (t0 > p_hi || (t0 + AR_STRIP <= attend_window(a, max(p_lo, 0)) && t0 >= a.sinks)) continue;  // (no row sees any)
      float sc[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t kw[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint4 v = *(const uint4*)(page + (ts + 16 * h + 8 * x + r) * (TQ_D / 2) + c * 16);
          kw[x][0] = v.x, kw[x][1] = v.y, kw[x][2] = v.z, kw[x][3] = v.w;
        }
        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float sum[NT][4], low[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] = low[t][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // tokens r, r + 8; bytes 2 j, 2 j + 1
            const uint32_t b = __byte_perm(kw[x & 1][j >> 1], 0, 0x4440 + 2 * (j & 1) + (x >> 1));
            if (SPLIT) {
              const uint2 v = ar_lut2(lutk + b * Sh::ENTRY);
              ah[x] = v.x, al[x] = v.y;
            } else {
              ah[x] = ar_lut1(lutk + b * Sh::ENTRY);
            }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4 w = *(const uint4*)(sh.w[t][j] + lane * 16);
            if (SPLIT) {
              float d[4];
              ar_mma(d, ah, w.x, w.y, zero);
              ar_mma(low[t], al, w.x, w.y, low[t]);
              ar_mma(low[t], ah, w.z, w.w, low[t]);
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[t][i] += d[i];
            } else {
              ar_mma(sum[t], ah, w.x, w.y, sum[t]);
              ar_mma(low[t], ah, w.z, w.w, low[t]);
            }
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = 8 * t + 2 * c + (i & 1), tok = ts + 16 * h + 8 * (i >> 1) + r;
            float x = fmaf(sum[t][i] + low[t][i], sh.inv[n], sh.bias[n]);
            if (g.outlier_k > 0) x += sh.corr[tok][n ^ (4 * (tok >> 2 & 1))];
            sc[h][t][i] = x;
          }
      }
      float nv[2][2], inv_n[NT][2];
      uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) nv[h][y] = ((const float*)(page + g.norm_off))[ts + 16 * h + 8 * y + r];
      softmax(sc, t0, end, 2, nv, ph, pl, inv_n);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* grp = page + g.v_off + (2 * warp + h) * VGB;
        uint32_t rec[9];
        if (VB == 4) {
          const uint4 x = *(const uint4*)(grp + lane * 16), y = *(const uint4*)(grp + 512 + lane * 16);
          rec[0] = x.x, rec[1] = x.y, rec[2] = x.z, rec[3] = x.w;
          rec[4] = y.x, rec[5] = y.y, rec[6] = y.z, rec[7] = y.w;
        } else {
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            const uint2 v = *(const uint2*)(grp + 256 * x + lane * 8);
            rec[2 * x] = v.x, rec[2 * x + 1] = v.y;
          }
          rec[6] = 0u;
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // channels r, r + 8; tokens 0-7, 8-15: pairs 4 mt, 4 mt + 2, 4 mt + 1, 4 mt + 3 of the record
            const int pr = 4 * mt + 2 * (x & 1) + (x >> 1);
            uint32_t b;
            if (VB == 4) b = __byte_perm(rec[pr >> 2], 0, 0x4440 + (pr & 3));
            else b = __funnelshift_r(rec[6 * pr >> 5], rec[(6 * pr >> 5) + 1], (6 * pr) & 31) & 63u;
            if (SPLIT) {
              const uint2 v = ar_lut2(lutv + b * Sh::ENTRY);
              ah[x] = v.x, al[x] = v.y;
            } else {
              ah[x] = ar_lut1(lutv + b * Sh::ENTRY);
            }
          }
          add_values(mt, ah, al, ph[h], pl[h], inv_n, inv_v);
        }
      }
    }
  } else {
    // ---- the uncompressed window: rows as fp16, natural order of channels
    uint8_t* const kh = sh.area;
    uint8_t* const vh = kh + AR_HOT * AR_PITCH;
    uint8_t* const kl = vh + AR_HOT * AR_PITCH;  // (SPLIT)
    uint8_t* const vl = kl + AR_HOT * AR_PITCH;
    float* const k_inv = (float*)(sh.area + AR_HOT * AR_PITCH * (SPLIT ? 4 : 2));
    float* const v_inv = k_inv + AR_HOT;
    {  // the queries as B operand: k-step j takes channels 16 j ..
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float inv;
        const float up = row_lift(qv[t], inv);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t hi, lo;
          ar_split(qv[t][2 * x], up, qv[t][2 * x + 1], up, hi, lo);
          const int d = (4 * lane + 2 * x) & 15;  // channels d, d + 1 of the step: word d / 8 of lane (d % 8) / 2
          uint32_t* to = (uint32_t*)(sh.w[t][lane >> 2] + (4 * warp + (d & 7) / 2) * 16) + (d >> 3);
          to[0] = hi, to[2] = lo;
        }
        if (lane == 0) sh.inv[8 * t + warp] = inv;
      }
    }
    const size_t ring = hot_offset_elems(g, a.layer, a.seq_begin + s, head);
    for (int k = k_lo; k < k_hi; ++k) {
      const int t0 = base + tl.at(k) * AR_HOT;
      __syncthreads();  // the tile before has been read
      bool odd = false;
      // sixteen threads a row, eight channels each; rows of two threads' half warps side by side
#pragma unroll 1
      for (int i = 0; i < AR_HOT / 16; ++i) {
        const int row = 16 * i + (tid >> 4), ch = 8 * (tid & 15), t = t0 + row;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          float x[8];
          if (t < end) {
            const void* src = kv ? a.hot_v : a.hot_k;
            const size_t at = ring + (size_t)(t % g.hot_cap) * TQ_D + ch;
            if (g.kv_dtype == TQ_F32) {
              const float4 u = *(const float4*)((const float*)src + at), v = *(const float4*)((const float*)src + at + 4);
              x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
            } else {
              const uint4 u = *(const uint4*)((const uint16_t*)src + at);
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if (g.kv_dtype == TQ_F16) {
                  const float2 f = __half22float2(*(const __half2*)&w[y]);
                  x[2 * y] = f.x, x[2 * y + 1] = f.y;
                } else {
                  x[2 * y] = __uint_as_float(w[y] << 16), x[2 * y + 1] = __uint_as_float(w[y] & 0xffff0000u);
                }
              }
            }
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) x[y] = 0.0f;
          }
          float mx = 0.0f;
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            mx = fmaxf(mx, fabsf(x[y]));
            odd |= !isfinite(x[y]);
          }
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          float inv;
          const float up = ar_lift(mx, 13, inv);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) ar_split(x[2 * y], up, x[2 * y + 1], up, hi[y], lo[y]);
          *(uint4*)((kv ? vh : kh) + row * AR_PITCH + 2 * ch) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if (SPLIT) *(uint4*)((kv ? vl : kl) + row * AR_PITCH + 2 * ch) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          if ((tid & 15) == 0) (kv ? v_inv : k_inv)[row] = inv;
        }
      }
      odd = __syncthreads_or(odd);

      const int ts = 16 * warp, tw = t0 + ts;
      if (odd) {  // term by term
        for (int j = 0; j < 16; ++j) {
          const int tok = tw + j;
          if (tok >= end) break;
          const size_t at = ring + (size_t)(tok % g.hot_cap) * TQ_D;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int n = 8 * t + 2 * c + x;
              if (tok > sh.pos[n] || (tok < sh.win[n] && tok >= a.sinks)) continue;
              float dot = 0.0f;
              for (int d = 0; d < TQ_D; ++d) dot = fmaf(sh.q[q_row(d)][n], attend_ld(a.hot_k, at + d, g.kv_dtype), dot);
              const float top = fmaxf(m_run[t][x], dot), by = top > -INFINITY ? top : 0.0f;
              const float down = tq_exp2(m_run[t][x] - by), e = tq_exp2(dot - by);
              m_run[t][x] = top;
              l_run[t][x] = l_run[t][x] * down + (r == 0 ? e : 0.0f);
#pragma unroll
              for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                  acc[t][mt][2 * y + x] = fmaf(e, attend_ld(a.hot_v, at + 16 * mt + 8 * y + r, g.kv_dtype),
                                               acc[t][mt][2 * y + x] * down);
            }
        }
        continue;
      }
      if (tw >= end || tw > p_hi || (tw + 16 <= attend_window(a, max(p_lo, 0)) && tw >= a.sinks)) continue;
      float sc[2][NT][4];
      {
        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float sum[NT][4], low[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] = low[t][i] = sc[1][t][i] = 0.0f;
        const uint32_t at = (ts + (lane & 15)) * AR_PITCH + (lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t ah[4], al[4];
          ar_ldm<false>(ah, ar_smem(kh) + at + 32 * j);
          if (SPLIT) ar_ldm<false>(al, ar_smem(kl) + at + 32 * j);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4 w = *(const uint4*)(sh.w[t][j] + lane * 16);
            if (SPLIT) {
              float d[4];
              ar_mma(d, ah, w.x, w.y, zero);
              ar_mma(low[t], al, w.x, w.y, low[t]);
              ar_mma(low[t], ah, w.z, w.w, low[t]);
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[t][i] += d[i];
            } else {
              ar_mma(sum[t], ah, w.x, w.y, sum[t]);
              ar_mma(low[t], ah, w.z, w.w, low[t]);
            }
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[0][t][i] = (sum[t][i] + low[t][i]) * sh.inv[8 * t + 2 * c + (i & 1)] * k_inv[ts + 8 * (i >> 1) + r];
      }
      float inv_n[NT][2];
      const float nv[2][2] = {{v_inv[ts + r], v_inv[ts + 8 + r]}, {0.0f, 0.0f}};
      uint32_t ph[2][NT][2], pl[2][NT][2];
      softmax(sc, tw, end, 1, nv, ph, pl, inv_n);
      const uint32_t at = (ts + (lane & 7) + (lane >> 4) * 8) * AR_PITCH + (lane >> 3 & 1) * 16;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        uint32_t ah[4], al[4];
        ar_ldm<true>(ah, ar_smem(vh) + at + 32 * mt);
        if (SPLIT) ar_ldm<true>(al, ar_smem(vl) + at + 32 * mt);
        add_values(mt, ah, al, ph[0], pl[0], inv_n, 1.0f);
      }
    }
  }

  // ---- the warps' states become one
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) l_run[t][x] += __shfl_xor_sync(0xffffffffu, l_run[t][x], o);
      if (r == 0) {
        sh.m[warp][8 * t + 2 * c + x] = m_run[t][x];
        sh.l[warp][8 * t + 2 * c + x] = l_run[t][x];
      }
    }
  __syncthreads();
  float* const sums = (float*)sh.area;  // [warp][N rows][128], two bits of the channel by the row
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int n = 8 * t + 2 * c + x;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < AR_WARPS; ++w) M = fmaxf(M, sh.m[w][n]);
      const float by = M > -INFINITY ? M : 0.0f;
      const float f = l_run[t][x] == 0.0f ? 0.0f : m_run[t][x] > -INFINITY ? tq_exp2(m_run[t][x] - by) : 1.0f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          sums[(warp * N + n) * TQ_D + ((16 * mt + 8 * y + r) ^ (8 * c))] =
              l_run[t][x] == 0.0f ? 0.0f : acc[t][mt][2 * y + x] * f;
    }
  __syncthreads();
  for (int i = tid; i < N * TQ_D; i += AR_THREADS) {
    const int n = i / TQ_D, d = i % TQ_D;
    if (row0 + n >= a.rows) break;
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < AR_WARPS; ++w) x += sums[(w * N + n) * TQ_D + (d ^ (8 * (n >> 1 & 3)))];
    float* to = attend_partial(a, unit, row0 + n, split);
    to[2 + d] = x;
    if (d == 0) {
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < AR_WARPS; ++w) M = fmaxf(M, sh.m[w][n]);
      const float by = M > -INFINITY ? M : 0.0f;
#pragma unroll
      for (int w = 0; w < AR_WARPS; ++w)
        if (sh.l[w][n] != 0.0f) L += sh.m[w][n] > -INFINITY ? sh.l[w][n] * tq_exp2(sh.m[w][n] - by) : sh.l[w][n];
      to[0] = M;
      to[1] = L;
    }
  }
}

template <int NT, bool SPLIT, int VB>
int launch_rows(const AttendArgs& a, cudaStream_t st) {
  using Shared = ArShared<NT, SPLIT, VB>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of one CTA");
  static_assert(SPLIT || NT > 1 || sizeof(Shared) <= 113 * 1024, "two CTAs on an SM");
  static_assert(AR_WARPS * 8 * NT * TQ_D * 4 <= ArShape<NT, SPLIT, VB>::AREA, "the sums' place");
  const int row_tiles = (a.rows + 8 * NT - 1) / (8 * NT);
  const int64_t grid = (int64_t)a.seq_count * a.g.n_kv_heads * row_tiles * (a.ns_cold + a.ns_hot);
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (sequence, head, query row) tiles in a call");
  TQ_REQUIRE((ArShape<NT, SPLIT, VB>::PAGE <= a.g.page_bytes), TQ_ERR_INVALID, "page size");
  TQ_CUDA(cudaFuncSetAttribute(attend_rows_kernel<NT, SPLIT, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)sizeof(Shared)));
  attend_rows_kernel<NT, SPLIT, VB><<<(int)grid, AR_THREADS, sizeof(Shared), st>>>(a, row_tiles);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

template <int NT, bool SPLIT>
int launch_rows(const AttendArgs& a, cudaStream_t st) {
  return a.g.value_bits == 4 ? launch_rows<NT, SPLIT, 4>(a, st) : launch_rows<NT, SPLIT, 3>(a, st);
}

}  // namespace

int tq_attend_rows_tile(int rows) { return rows <= 8 ? 8 : 16; }

int tq_launch_attend_rows(const AttendArgs& a, cudaStream_t st) {
  const bool one = tq_attend_rows_tile(a.rows) == 8;
  if (a.q_dtype == TQ_BF16) return one ? launch_rows<1, false>(a, st) : launch_rows<2, false>(a, st);
  return one ? launch_rows<1, true>(a, st) : launch_rows<2, true>(a, st);
}

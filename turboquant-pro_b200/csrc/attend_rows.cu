// Attention of few query rows per KV head on the codes: single tokens, drafts to verify, small chunks.
// 256-token blocks with per-channel keys; the products on mma.sync (m16n8k16) with the codes as the A operand,
// straight from a table into registers, and NT tiles of eight query rows as the B operand.
//
// Persistent CTAs of eight warps.  The pages that the rows of each (sequence, KV head, row tile) see, first tokens,
// then the window, and after them its tiles of the uncompressed window, form one list that is cut into shares of
// equal cost, one per CTA, so ragged batches and every number of heads balance; where a share enters or leaves a
// row tile, or goes from pages to the window, the CTA writes a state, and the merge sums these.  Items come
// in whole with cp.async, the next one while this one is attended.  Of a page's 256 tokens a warp attends 32:
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
// The uncompressed window, 64 tokens at a time: 16-bit rows are the A operand as they are, in their own type
// (ldmatrix), so that only the other operand is split: the query is exact in one part for 16-bit queries of that type
// or of bfloat16 in fp16, and has as many as it needs otherwise; probabilities have one part in fp16 (two with SPLIT)
// and two in bfloat16 (three).  float32 rows, 32 at a time, are split into fp16 pairs as they are read.  A tile that
// holds an infinity or a NaN is attended term by term instead (products with masked tokens and with low parts would
// spread it), and so is one of float32 keys beyond fp16's range.
//
// Bound by the issue slots of look-ups and products; at one row tile the codes are read once.
#include <algorithm>

#include "attend.cuh"

namespace {

constexpr int AR_THREADS = 256, AR_WARPS = 8;
constexpr int AR_S = 256;          // tokens of a page
constexpr int AR_STRIP = 32;       // of them, a warp's
constexpr int AR_HOT = 64, AR_HOT32 = 32;  // window tokens of a tile: 16-bit rows, float32 rows
constexpr int AR_PITCH = TQ_D * 2 + 16, AR_PITCH32 = TQ_D * 4 + 16;  // bytes of a window row in shared memory
constexpr int AR_COST = 4;         // a page takes the time of so many tiles of the window
constexpr int AR_SEQS = 64;        // sequences of a launch
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
  static constexpr int STAGE = PAGE + LIST;            // a page, or a tile of the window
  static constexpr int WROW = 33 * 16;                 // bytes of a k-step's B fragments, padded
  static constexpr int QROW = TQ_D * (SPLIT ? 4 : 2);  // bytes of a query as it comes, at most
};
static_assert(2 * AR_HOT * AR_PITCH <= ArShape<1, false, 3>::PAGE && 2 * AR_HOT32 * AR_PITCH32 <= ArShape<1, false, 3>::PAGE,
              "a tile of the window in a page's place");
static_assert(AR_WARPS * 8 * TQ_D * 4 <= ArShape<1, false, 3>::PAGE, "the warps' sums of eight rows in a page's place");

template <int NT, bool SPLIT, int VB>
struct ArShared {
  using Sh = ArShape<NT, SPLIT, VB>;
  alignas(128) uint8_t lut[Sh::LUTK + Sh::LUTV];
  alignas(128) uint8_t stage[2][Sh::STAGE];
  alignas(16) uint8_t q_raw[Sh::N * Sh::QROW];  // the next rows' queries
  alignas(16) uint8_t w[NT][8][Sh::WROW];       // [tile][k-step][lane] {b0 hi, b1 hi, b0 lo, b1 lo}
  alignas(16) uint2 w3[SPLIT ? NT : 1][SPLIT ? 8 : 1][32];  // third parts (bfloat16 windows)
  alignas(16) float corr[AR_S][Sh::N];          // outliers' part of the scores
  alignas(16) float q[TQ_D][Sh::N];             // row q_row(d): channel d
  float bias[Sh::N], inv[Sh::N];
  float m[AR_WARPS][Sh::N], l[AR_WARPS][Sh::N];
  int pos[Sh::N], win[Sh::N];
  float grid[16], cent[16], top[AR_WARPS];
  int most[2];                                  // pages and window tiles of the longest row
  int2 seq[AR_SEQS];                            // tokens, query tokens
  int cum[AR_SEQS + 1];                         // work before each sequence, per row
};

TQ_DEV void ar_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}
TQ_DEV void ar_mma_bf(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
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
// the same of a and b as PARTS bfloat16 parts
template <int PARTS>
TQ_DEV void ar_split_bf(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    w[i] = *(const uint32_t*)&h;
    a -= __uint_as_float(w[i] << 16);
    b -= __uint_as_float(w[i] & 0xffff0000u);
  }
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
TQ_DEV void ar_cp16_or_zero(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ar_smem(dst)), "l"(src), "r"(there ? 16 : 0)
               : "memory");
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

// A sequence's work in a launch: its pages (first tokens, then the window), then its tiles of the uncompressed
// window; the same for all of its heads and row tiles.
struct ArWork {
  AttendTiles page, hot;
  int cold;  // tokens in blocks
  TQ_DEV int items() const { return page.count() + hot.count(); }
  TQ_DEV int cost() const { return AR_COST * page.count() + hot.count(); }
};
TQ_DEV ArWork ar_work(const AttendArgs& a, int n, int q_n) {
  ArWork w;
  w.cold = n_cold_blocks(n, a.g.hot_window, AR_S) * AR_S;
  const int p_lo = n - q_n, p_hi = q_n > 0 ? n - 1 : -1;
  w.page = attend_tiles(a, 0, w.cold, AR_S, p_lo, p_hi);
  w.hot = attend_tiles(a, w.cold, n, a.g.kv_dtype == TQ_F32 ? AR_HOT32 : AR_HOT, p_lo, p_hi);
  return w;
}

// How a launch divides its work; the first CTA leaves it for the merge.
struct ArPlan {
  int64_t share;
  int cum[AR_SEQS + 1];
};

// An item of the list.
struct ArItem {
  int s, row, it;  // sequence, row (head * row tiles + tile), item of the row
  int64_t at;      // the cost of what is before it
};

template <int NT, bool SPLIT, int VB>
__global__ void __launch_bounds__(AR_THREADS, !SPLIT&& NT == 1 ? 2 : 1)
    attend_rows_kernel(AttendArgs a, int row_tiles) {
  using Sh = ArShape<NT, SPLIT, VB>;
  constexpr int N = Sh::N;
  constexpr int VGB = TQ_GROUP_TOK * TQ_D * VB / 8;
  extern __shared__ __align__(128) uint8_t ar_shared[];
  ArShared<NT, SPLIT, VB>& sh = *(ArShared<NT, SPLIT, VB>*)ar_shared;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int H = g.n_kv_heads, G = g.group, rows_per_seq = H * row_tiles;
  const bool q32 = a.q_dtype == TQ_F32, hot32 = g.kv_dtype == TQ_F32;
  const int hot_size = hot32 ? AR_HOT32 : AR_HOT;

  // ---- the work before every sequence
  if (tid < 16) {
    sh.grid[tid] = a.tables->grid[tid];
    sh.cent[tid] = a.tables->centroids[tid];
  }
  if (warp == 0) {
    constexpr int PER = AR_SEQS / 32;
    int sum = 0, most_page = 0, most_hot = 0, cost[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      cost[i] = 0;
      if (s < a.seq_count) {
        const AttendSeq sq = attend_seq(a, s);
        sh.seq[s] = make_int2(sq.n, sq.q_n);
        const ArWork w = ar_work(a, sq.n, sq.q_n);
        cost[i] = w.cost();
        most_page = max(most_page, w.page.count());
        most_hot = max(most_hot, w.hot.count());
      }
      sum += cost[i];
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    if (lane == 31) sh.cum[AR_SEQS] = before;
    before -= sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sh.cum[lane * PER + i] = before;
      before += cost[i];
    }
    most_page = __reduce_max_sync(0xffffffffu, most_page);
    most_hot = __reduce_max_sync(0xffffffffu, most_hot);
    if (lane == 0) sh.most[0] = most_page, sh.most[1] = most_hot;
  }
  __syncthreads();
  // Shares of equal cost: what starts in [k share, (k + 1) share) is CTA k's.  A row's pages then meet at most
  // AR_COST * (pages - 1) / share + 2 CTAs, its window tiles (tiles - 1) / share + 2, which have to fit their slots.
  const int64_t total = (int64_t)sh.cum[AR_SEQS] * rows_per_seq;
  // (at least a page's cost: otherwise CTAs between two pages would have slots, but nothing to put there)
  int64_t share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)AR_COST);
  share = max(share, (int64_t)((AR_COST * sh.most[0] + a.ns_cold - 3) / (a.ns_cold - 2)));
  share = max(share, (int64_t)((sh.most[1] + a.ns_hot - 3) / (a.ns_hot - 2)));
  if (blockIdx.x == 0) {
    ArPlan* plan = (ArPlan*)a.plan;
    if (tid == 0) plan->share = share;
    for (int i = tid; i <= AR_SEQS; i += AR_THREADS) plan->cum[i] = sh.cum[i];
  }
  const int64_t lo = share * blockIdx.x, hi = min(lo + share, total);
  if (lo >= total) return;

  auto work_of = [&](int s) { return ar_work(a, sh.seq[s].x, sh.seq[s].y); };
  ArItem cur;
  {  // the first item that starts at lo or after it
    int x = 0, y = a.seq_count - 1;
    while (x < y) {  // the last sequence that starts at lo or before it
      const int mid = (x + y + 1) >> 1;
      if ((int64_t)sh.cum[mid] * rows_per_seq <= lo) x = mid;
      else y = mid - 1;
    }
    const ArWork w = work_of(x);
    const int64_t in = lo - (int64_t)sh.cum[x] * rows_per_seq;
    const int cost = w.cost(), off = (int)(in % cost), pages = AR_COST * w.page.count();
    cur.s = x;
    cur.row = (int)(in / cost);
    cur.it = off < pages ? (off + AR_COST - 1) / AR_COST : w.page.count() + off - pages;
    cur.at = lo - off + (off < pages ? AR_COST * cur.it : off);
    if (cur.it == w.items()) {  // (off lies in the last page of a row without a window)
      cur.it = 0;
      ++cur.row;
    }
  }
  auto settle = [&](ArItem& i) {  // rows past the sequence's last: the next sequence that has any work
    while (i.row >= rows_per_seq) {
      i.row = 0;
      do ++i.s;
      while (i.s < a.seq_count && sh.cum[i.s + 1] == sh.cum[i.s]);
      if (i.s >= a.seq_count) break;
    }
  };
  auto after = [&](const ArItem& i) {
    const ArWork w = work_of(i.s);
    ArItem n = i;
    n.at += i.it < w.page.count() ? AR_COST : 1;
    if (++n.it >= w.items()) {
      n.it = 0;
      ++n.row;
      settle(n);
    }
    return n;
  };
  settle(cur);
  if (cur.at >= hi) return;

  // ---- copies
  auto unit_of = [&](const ArItem& i) {
    return unit_index(g, a.layer, a.seq_begin + i.s, i.row / row_tiles);
  };
  auto meta_of = [&](const ArItem& i) -> PageMeta {
    PageMeta pm = {0, 0};
    if (SPLIT && g.outlier_k > 0 && i.at < hi) {
      const ArWork w = work_of(i.s);
      if (i.it < w.page.count()) pm = a.page_meta[unit_of(i) * g.max_blocks + w.page.at(i.it)];
    }
    return pm;
  };
  auto listed = [&](const PageMeta& pm) { return pm.cnt <= (uint32_t)AR_LIST && (pm.off & 3u) == 0u; };
  auto fetch = [&](const ArItem& i, const PageMeta& pm, uint8_t* to) {
    const ArWork w = work_of(i.s);
    const size_t u = unit_of(i);
    if (i.it < w.page.count()) {
      const uint8_t* from = a.pages + (u * g.max_blocks + w.page.at(i.it)) * (size_t)g.page_bytes;
      for (int k = tid; k < Sh::PAGE / 16; k += AR_THREADS) ar_cp16(to + 16 * k, from + 16 * k);
      if (SPLIT && listed(pm)) {
        const size_t slab = u * (size_t)g.pool_entries + pm.off;
        const int n4 = (int)(pm.cnt + 3) / 4;  // (slices are whole fours, and slabs whole sixty-fours, of entries)
        for (int k = tid; k < n4; k += AR_THREADS) {
          ar_cp16(to + Sh::PAGE + 16 * k, a.pool_dec + slab + 4 * k);
          ar_cp8(to + Sh::PAGE + 4 * AR_LIST + 8 * k, a.pool_val + slab + 4 * k);
        }
      }
    } else {
      const int t0 = w.cold + w.hot.at(i.it - w.page.count()) * hot_size, n = sh.seq[i.s].x;
      const size_t ring = u * (size_t)g.hot_cap * TQ_D;
      const int pieces = hot32 ? 32 : 16, pitch = hot32 ? AR_PITCH32 : AR_PITCH, esz = hot32 ? 4 : 2;
      for (int k = tid; k < hot_size * pieces; k += AR_THREADS) {
        const int row = k / pieces, at = (k - row * pieces) * 16, t = t0 + row;
        const size_t from = (ring + (size_t)(t % g.hot_cap) * TQ_D) * esz + at;
        ar_cp16_or_zero(to + row * pitch + at, (const uint8_t*)a.hot_k + from, t < n);
        ar_cp16_or_zero(to + (hot_size + row) * pitch + at, (const uint8_t*)a.hot_v + from, t < n);
      }
    }
  };
  auto fetch_q = [&](const ArItem& i) {
    const int head = i.row / row_tiles, row0 = i.row % row_tiles * N, pieces = q32 ? 32 : 16, esz = q32 ? 4 : 2;
    for (int k = tid; k < N * pieces; k += AR_THREADS) {
      const int n = k / pieces, at = (k - n * pieces) * 16, row = row0 + n;
      const bool there = row < a.rows;
      const int64_t from = there ? (int64_t)i.s * a.q_seq + (int64_t)(row / G) * a.q_tok +
                                       (int64_t)(head * G + row % G) * a.q_head
                                 : 0;
      ar_cp16_or_zero(sh.q_raw + n * Sh::QROW + at, (const uint8_t*)a.q + from * esz + at, there);
    }
  };
  int st = 0;
  PageMeta pm = meta_of(cur);
  fetch(cur, pm, sh.stage[0]);
  fetch_q(cur);
  ar_commit();
  ArItem nxt = after(cur);
  PageMeta pm_next = meta_of(nxt);

  // ---- tables of pairs
  float inv_k, inv_v;
  {
    float max_k = 0.0f, max_v = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      max_k = fmaxf(max_k, fabsf(sh.grid[i]));
      max_v = fmaxf(max_v, fabsf(sh.cent[i]));
    }
    const float up_k = ar_lift(max_k, 7, inv_k), up_v = ar_lift(max_v, 7, inv_v);
    for (int e = tid; e < 256 + Sh::NV; e += AR_THREADS) {
      uint32_t hi2, lo2;
      uint4* to;
      if (e < 256) {
        ar_split(sh.grid[e & 15], up_k, sh.grid[e >> 4], up_k, hi2, lo2);
        to = (uint4*)(sh.lut + e * Sh::ENTRY);
      } else {
        const int b = e - 256;
        ar_split(sh.cent[b & ((1 << VB) - 1)], up_v, sh.cent[b >> VB], up_v, hi2, lo2);
        to = (uint4*)(sh.lut + Sh::LUTK + b * Sh::ENTRY);
      }
#pragma unroll
      for (int i = 0; i < Sh::ENTRY / 16; ++i)
        to[(i + lane) % (Sh::ENTRY / 16)] = SPLIT ? make_uint4(hi2, lo2, hi2, lo2) : make_uint4(hi2, hi2, hi2, hi2);
    }
  }

  // rows 8 t + 2 c + x are this lane's columns
  float qv[NT][4];  // rows warp, warp + 8, ...: channels 4 lane .. + 3, times the scores' unit
  float acc[NT][8][4], m_run[NT][2], l_run[NT][2];
  int first_pos = 0, last_win = 0, p_lo = 0, p_hi = 0;  // of the row tile: see `start_row`
  auto reset = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][mt][i] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x) m_run[t][x] = -INFINITY, l_run[t][x] = 0.0f;
    }
  };
  // four channels of a row of q_raw
  auto raw_q = [&](int n, float (&x)[4]) {
    const uint8_t* p = sh.q_raw + n * Sh::QROW + 4 * lane * (q32 ? 4 : 2);
    if (SPLIT && q32) {
      const float4 v = *(const float4*)p;
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const uint2 v = *(const uint2*)p;
      if (SPLIT) {
        const float2 u = __half22float2(*(const __half2*)&v.x), w = __half22float2(*(const __half2*)&v.y);
        x[0] = u.x, x[1] = u.y, x[2] = w.x, x[3] = w.y;
      } else {
        x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
      }
    }
  };
  // (between two barriers of an item; what it writes is read after the second)
  auto start_row = [&](const ArItem& i) {
    AttendSeq sq;
    sq.n = sh.seq[i.s].x, sq.q_n = sh.seq[i.s].y;
    sq.first = sq.n - sq.q_n;
    sq.cold = 0;
    const int row0 = i.row % row_tiles * N, last = min(min(row0 + N, a.rows), sq.q_n * G) - 1;
    p_lo = sq.first + row0 / G;
    p_hi = last >= row0 ? sq.first + last / G : -1;
    // whether a tile of tokens is seen by all rows of the tile: from the earliest row, and the latest window
    first_pos = min(row0 + N, a.rows) - 1 <= last ? p_lo : -1;
    last_win = attend_window(a, max(p_hi, 0));
    if (tid < N) {
      sh.pos[tid] = row0 + tid < a.rows ? attend_position(a, sq, row0 + tid) : -1;
      sh.win[tid] = attend_window(a, sh.pos[tid]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      raw_q(8 * t + warp, qv[t]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qv[t][k] = tq_scaled<true>(qv[t][k]);
        sh.q[q_row(4 * lane + k)][8 * t + warp] = qv[t][k];
      }
    }
  };
  auto row_max = [&](const float (&w)[4]) -> float {
    float mx = fmaxf(fmaxf(fabsf(w[0]), fabsf(w[1])), fmaxf(fabsf(w[2]), fabsf(w[3])));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    return mx;
  };
  // whether tokens t0 .. t1 - 1 are seen by every row of the tile, and by none
  auto open_to_all = [&](int t0, int t1) { return t1 - 1 <= first_pos && (t0 >= last_win || t1 <= a.sinks); };
  auto open_to_none = [&](int t0, int t1) {
    return t0 > p_hi || (t1 <= attend_window(a, max(p_lo, 0)) && t0 >= a.sinks);
  };

  // From the scores of `tiles` times 16 tokens from `t0` on to their probabilities: maximum and sum go on, the
  // probability stays in `sc`, times a power of two that takes the row's largest probability * nv below 2^14.
  auto softmax = [&](float (&sc)[2][NT][4], int t0, int t_end, int tiles, const float (&nv)[2][2], float (&inv_n)[NT][2]) {
    const bool open = t0 + 16 * tiles <= t_end && open_to_all(t0, t0 + 16 * tiles);
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
  };
  auto scaled_add = [&](float (&to)[4], const float (&d)[4], const float (&inv)[2], float by) {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = fmaf(d[i], inv[i & 1] * by, to[i]);
  };
  const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};

  // ---- a page: weights and corrections, then, past a barrier, this warp's 32 tokens
  const uint32_t lutk = ar_smem(sh.lut) + (lane % Sh::REP) * (SPLIT ? 8 : 4);
  const uint32_t lutv = lutk + Sh::LUTK;
  auto page_prepare = [&](const uint8_t* page, const PageMeta& pm, size_t u) {
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
        const float up = ar_lift(row_max(w), 13, inv);
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
    if (g.outlier_k == 0) return;
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
        dec = a.pool_dec + u * (size_t)g.pool_entries + pm.off;
        val = a.pool_val + u * (size_t)g.pool_entries + pm.off;
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
        list = a.pool_dec + u * (size_t)g.pool_entries + hdr->off;
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
  };
  auto page_attend = [&](const uint8_t* page, int first, int cold) {
    const int ts = AR_STRIP * warp, t0 = first + ts;
    if (open_to_none(t0, t0 + AR_STRIP)) return;
    float sc[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t kw[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint4 v = *(const uint4*)(page + (ts + 16 * h + 8 * x + r) * (TQ_D / 2) + c * 16);
        kw[x][0] = v.x, kw[x][1] = v.y, kw[x][2] = v.z, kw[x][3] = v.w;
      }
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
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int y = 0; y < 2; ++y) nv[h][y] = ((const float*)(page + g.norm_off))[ts + 16 * h + 8 * y + r];
    softmax(sc, t0, cold, 2, nv, inv_n);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t hi2, lo2;
          // (a hidden token's norm may be anything)
          const float n0 = sc[h][t][2 * y] == 0.0f ? 0.0f : nv[h][y], n1 = sc[h][t][2 * y + 1] == 0.0f ? 0.0f : nv[h][y];
          ar_split(sc[h][t][2 * y], n0, sc[h][t][2 * y + 1], n1, hi2, lo2);
          ph[t][y] = ar_transpose(hi2);
          if (SPLIT) pl[t][y] = ar_transpose(lo2);
        }
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
          scaled_add(acc[t][mt], d, inv_n[t], inv_v);
        }
      }
    }
  };

  // ---- a tile of the uncompressed window
  // the raw queries as B operand, in natural order of channels: k-step j takes channels 16 j ..
  auto hot_weights = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[4], inv = 1.0f;
      raw_q(8 * t + warp, x);
      const bool bf = g.kv_dtype == TQ_BF16;
      const float up = bf ? 1.0f : ar_lift(row_max(x), 13, inv);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t w[3] = {0u, 0u, 0u};
        if (bf) ar_split_bf<SPLIT ? 3 : 1>(x[2 * k], x[2 * k + 1], w);
        else ar_split(x[2 * k], up, x[2 * k + 1], up, w[0], w[1]);
        const int d = (4 * lane + 2 * k) & 15;  // channels d, d + 1 of the step: word d / 8 of lane (d % 8) / 2
        uint32_t* to = (uint32_t*)(sh.w[t][lane >> 2] + (4 * warp + (d & 7) / 2) * 16) + (d >> 3);
        to[0] = w[0], to[2] = w[1];
        if (SPLIT) ((uint32_t*)&sh.w3[t][lane >> 2][4 * warp + (d & 7) / 2])[d >> 3] = w[2];
      }
      if (lane == 0) sh.inv[8 * t + warp] = inv;
    }
  };
  // Whether the tile has to go term by term, and (float32) the power of two for its values.  Has a barrier.
  auto hot_check = [&](const uint8_t* tile, float& v_up, float& v_inv) -> bool {
    bool odd = false;
    v_up = v_inv = 1.0f;
    if (hot32) {
      float top = 0.0f, top_k = 0.0f;
      for (int k = tid; k < AR_HOT32 * 32; k += AR_THREADS) {
        const int at = k / 32 * AR_PITCH32 + k % 32 * 16;
        const float4 x = *(const float4*)(tile + at), y = *(const float4*)(tile + AR_HOT32 * AR_PITCH32 + at);
        top_k = fmaxf(top_k, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        top = fmaxf(top, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
        odd |= !(fabsf(x.x) + fabsf(x.y) + fabsf(x.z) + fabsf(x.w) + fabsf(y.x) + fabsf(y.y) + fabsf(y.z) + fabsf(y.w) < INFINITY);
      }
      odd |= top_k > 65504.0f;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) sh.top[warp] = top;
      odd = __syncthreads_or(odd);
#pragma unroll
      for (int w = 0; w < AR_WARPS; ++w) top = fmaxf(top, sh.top[w]);
      v_up = ar_lift(top, 13, v_inv);
    } else {
      const uint32_t ones = g.kv_dtype == TQ_F16 ? 0x7c007c00u : 0x7f807f80u;
      for (int k = tid; k < AR_HOT * 16; k += AR_THREADS) {
        const uint4 x = *(const uint4*)(tile + (AR_HOT + k / 16) * AR_PITCH + k % 16 * 16);
        // (an exponent of ones in either half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = (i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w) & ones;
          odd |= (w & 0xffffu) == (ones & 0xffffu) || w >> 16 == ones >> 16;
        }
      }
      odd = __syncthreads_or(odd);
    }
    return odd;
  };
  auto hot_terms = [&](int t0, int n, size_t ring) {  // this warp's tokens of the tile, term by term
    const int per = hot_size / AR_WARPS;
    for (int j = 0; j < per; ++j) {
      const int tok = t0 + per * warp + j;
      if (tok >= n) break;
      const size_t at = ring + (size_t)(tok % g.hot_cap) * TQ_D;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 8 * t + 2 * c + x;
          if (tok > sh.pos[row] || (tok < sh.win[row] && tok >= a.sinks)) continue;
          float dot = 0.0f;
          for (int d = 0; d < TQ_D; ++d) dot = fmaf(sh.q[q_row(d)][row], attend_ld(a.hot_k, at + d, g.kv_dtype), dot);
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
  };
  auto hot_attend = [&](const uint8_t* tile, int first, int n, float v_up, float v_inv) {
    const int ts = 16 * warp, t0 = first + ts;
    if (ts >= hot_size || t0 >= n || open_to_none(t0, t0 + 16)) return;
    const bool bf = g.kv_dtype == TQ_BF16;
    float sc[2][NT][4], sum[NT][4], low[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] = low[t][i] = sc[1][t][i] = 0.0f;
    const uint32_t k_at = ar_smem(tile) + (ts + (lane & 15)) * AR_PITCH + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t ah[4], al[4] = {0u, 0u, 0u, 0u};
      if (hot32) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 f = *(const float2*)(tile + (ts + r + 8 * (x & 1)) * AR_PITCH32 + (16 * j + 2 * c + 8 * (x >> 1)) * 4);
          ar_split(f.x, 1.0f, f.y, 1.0f, ah[x], al[x]);
        }
      } else {
        ar_ldm<false>(ah, k_at + 32 * j);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 w = *(const uint4*)(sh.w[t][j] + lane * 16);
        if (bf) {
          if (SPLIT) {
            const uint2 w3 = sh.w3[t][j][lane];
            float d[4];
            ar_mma_bf(d, ah, w.x, w.y, zero);
            ar_mma_bf(low[t], ah, w.z, w.w, low[t]);
            ar_mma_bf(low[t], ah, w3.x, w3.y, low[t]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[t][i] += d[i];
          } else {
            ar_mma_bf(sum[t], ah, w.x, w.y, sum[t]);
          }
        } else {
          float d[4];
          ar_mma(d, ah, w.x, w.y, zero);
          if (SPLIT || hot32) {
            ar_mma(low[t], ah, w.z, w.w, low[t]);
            if (hot32) ar_mma(low[t], al, w.x, w.y, low[t]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] += d[i];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sc[0][t][i] = tq_scaled<true>((sum[t][i] + low[t][i]) * sh.inv[8 * t + 2 * c + (i & 1)]);
    float inv_n[NT][2];
    const float nv[2][2] = {{1.0f, 1.0f}, {0.0f, 0.0f}};
    softmax(sc, t0, n, 1, nv, inv_n);
    uint32_t p[NT][2][3] = {};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (bf) ar_split_bf<SPLIT ? 3 : 2>(sc[0][t][2 * y], sc[0][t][2 * y + 1], p[t][y]);
        else ar_split(sc[0][t][2 * y], 1.0f, sc[0][t][2 * y + 1], 1.0f, p[t][y][0], p[t][y][1]);
#pragma unroll
        for (int k = 0; k < (SPLIT ? 3 : 2); ++k) p[t][y][k] = ar_transpose(p[t][y][k]);
      }
    const uint8_t* v = tile + hot_size * (hot32 ? AR_PITCH32 : AR_PITCH);
    const uint32_t v_at = ar_smem(v) + (ts + (lane & 7) + (lane >> 4) * 8) * AR_PITCH + (lane >> 3 & 1) * 16;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      uint32_t ah[4], al[4] = {0u, 0u, 0u, 0u};
      if (hot32) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // channels r, r + 8; tokens 2 c, 2 c + 1, and 8 further
          const float* f = (const float*)(v + (ts + 2 * c + 8 * (x >> 1)) * AR_PITCH32) + 16 * mt + r + 8 * (x & 1);
          ar_split(f[0], v_up, f[AR_PITCH32 / 4], v_up, ah[x], al[x]);
        }
      } else {
        ar_ldm<true>(ah, v_at + 32 * mt);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float d[4];
        if (bf) {
          if (SPLIT) {
            ar_mma_bf(d, ah, p[t][0][2], p[t][1][2], zero);
            ar_mma_bf(d, ah, p[t][0][1], p[t][1][1], d);
          } else {
            ar_mma_bf(d, ah, p[t][0][1], p[t][1][1], zero);
          }
          ar_mma_bf(d, ah, p[t][0][0], p[t][1][0], d);
        } else {
          ar_mma(d, ah, p[t][0][1], p[t][1][1], zero);
          if (hot32) ar_mma(d, al, p[t][0][0], p[t][1][0], d);
          ar_mma(d, ah, p[t][0][0], p[t][1][0], d);
        }
        scaled_add(acc[t][mt], d, inv_n[t], v_inv);
      }
    }
  };

  // ---- the warps' states become one: `work` has room for the sums of eight rows of every warp
  auto flush = [&](const ArItem& i, const ArWork& w, bool hot, uint8_t* room) {
    const int head = i.row / row_tiles, row0 = i.row % row_tiles * N, unit = i.s * H + head;
    const int64_t begin = (int64_t)sh.cum[i.s] * rows_per_seq + (int64_t)i.row * w.cost();
    const int slot = hot ? a.ns_cold + (int)(blockIdx.x - (begin + AR_COST * w.page.count()) / share)
                         : (int)(blockIdx.x - begin / share);
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
    float* const sums = (float*)room;  // [warp][8 rows][128], two bits of the channel by the row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      __syncthreads();  // (the item, or the eight rows before, have been read)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int n = 8 * t + 2 * c + x;
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < AR_WARPS; ++k) M = fmaxf(M, sh.m[k][n]);
        const float by = M > -INFINITY ? M : 0.0f;
        const float f = l_run[t][x] == 0.0f ? 0.0f : m_run[t][x] > -INFINITY ? tq_exp2(m_run[t][x] - by) : 1.0f;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            sums[(warp * 8 + 2 * c + x) * TQ_D + ((16 * mt + 8 * y + r) ^ (8 * c))] =
                l_run[t][x] == 0.0f ? 0.0f : acc[t][mt][2 * y + x] * f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8 * TQ_D / AR_THREADS; ++k) {
        const int n = k * (AR_THREADS / TQ_D) + tid / TQ_D, d = tid % TQ_D;
        if (row0 + 8 * t + n >= a.rows) break;
        float x = 0.0f;
#pragma unroll
        for (int u = 0; u < AR_WARPS; ++u) x += sums[(u * 8 + n) * TQ_D + (d ^ (8 * (n >> 1)))];
        float* to = attend_partial(a, unit, row0 + 8 * t + n, slot);
        to[2 + d] = x;
        if (d == 0) {
          float M = -INFINITY, L = 0.0f;
#pragma unroll
          for (int u = 0; u < AR_WARPS; ++u) M = fmaxf(M, sh.m[u][8 * t + n]);
          const float by = M > -INFINITY ? M : 0.0f;
#pragma unroll
          for (int u = 0; u < AR_WARPS; ++u)
            if (sh.l[u][8 * t + n] != 0.0f)
              L += sh.m[u][8 * t + n] > -INFINITY ? sh.l[u][8 * t + n] * tq_exp2(sh.m[u][8 * t + n] - by) : sh.l[u][8 * t + n];
          to[0] = M;
          to[1] = L;
        }
      }
    }
  };

  // ---- the share, item by item
  bool new_row = true, new_kind = true;
  for (;;) {
    uint8_t* const item = sh.stage[st];
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the item has landed; the one before it, and what was made for it, has been read
    const ArWork w = work_of(cur.s);
    const bool hot = cur.it >= w.page.count(), more = nxt.at < hi;
    if (more) {
      fetch(nxt, pm_next, sh.stage[st ^ 1]);
      ar_commit();
    }
    if (new_row) {
      start_row(cur);
      if (!hot) __syncthreads();  // (the corrections of a page read the queries before its barrier)
    }
    if (new_kind) reset();
    const size_t u = unit_of(cur);
    const int first = hot ? w.cold + w.hot.at(cur.it - w.page.count()) * hot_size : w.page.at(cur.it) * AR_S;
    float v_up = 1.0f, v_inv = 1.0f;
    bool odd = false;
    if (hot) {
      if (new_kind) hot_weights();
      odd = hot_check(item, v_up, v_inv);
    } else {
      page_prepare(item, pm, u);
      __syncthreads();
    }
    const ArItem nn = more ? after(nxt) : nxt;
    const PageMeta pm_nn = more ? meta_of(nn) : pm_next;
    const bool row_ends = !more || nxt.row != cur.row || nxt.s != cur.s;
    if (more && row_ends) {
      fetch_q(nxt);
      ar_commit();
    }
    if (hot) {
      if (odd) hot_terms(first, sh.seq[cur.s].x, u * (size_t)g.hot_cap * TQ_D);
      else hot_attend(item, first, sh.seq[cur.s].x, v_up, v_inv);
    } else {
      page_attend(item, first, w.cold);
    }
    const bool kind_ends = row_ends || (!hot && nxt.it >= w.page.count());
    if (kind_ends) flush(cur, w, hot, item);
    if (!more) break;
    new_row = row_ends;
    new_kind = kind_ends;
    cur = nxt, nxt = nn;
    pm = pm_next, pm_next = pm_nn;
    st ^= 1;
  }
}

// ---------------------------------------------------------------------------------------------------
// Merge of the states: four rows at a time, a group of 128 threads each, which sums the row's slots in order; then all
// 512 threads rotate the four sums of pages, a quarter of the input channels each, whose rows of Pi they hold
// in registers from before the states were there.
// ---------------------------------------------------------------------------------------------------
constexpr int AC_THREADS = 512;

__global__ void __launch_bounds__(AC_THREADS) attend_rows_combine_kernel(AttendArgs a, int row_tiles, int tile, int total) {
  __shared__ __align__(16) float cs[TQ_D][4], ys[4][4][TQ_D];
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, e = tid % TQ_D, h = tid / TQ_D;
  const int H = g.n_kv_heads, G = g.group;
  float pi[TQ_D / 4];
#pragma unroll
  for (int d = 0; d < TQ_D / 4; ++d) pi[d] = a.tables->pi[(32 * h + d) * TQ_D + e];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ArPlan* plan = (const ArPlan*)a.plan;
  const int64_t share = plan->share;
  for (int r0 = blockIdx.x * 4; r0 < total; r0 += gridDim.x * 4) {
    const int at = r0 + h;
    float hot = 0.0f, L = 0.0f, x = 0.0f;
    int s = 0, head = 0, row = 0;
    if (at < total) {
      row = at % a.rows;
      const int unit = at / a.rows;
      s = unit / H, head = unit - s * H;
      const AttendSeq sq = attend_seq(a, s);
      const ArWork w = ar_work(a, sq.n, sq.q_n);
      const int64_t begin = (int64_t)plan->cum[s] * H * row_tiles + (int64_t)(head * row_tiles + row / tile) * w.cost();
      const int pages = w.page.count(), hots = w.hot.count();
      const int64_t middle = begin + AR_COST * pages;
      const int nc = pages > 0 ? (int)((middle - AR_COST) / share - begin / share) + 1 : 0;
      const int nh = hots > 0 ? (int)((middle + hots - 1) / share - middle / share) + 1 : 0;
      const float* base = attend_partial(a, unit, row, 0);
      auto slot = [&](int i) { return base + (size_t)(i < nc ? i : a.ns_cold + i - nc) * TQ_PART_STRIDE; };
      float M = -INFINITY;
#pragma unroll 8
      for (int i = 0; i < nc + nh; ++i) M = fmaxf(M, slot(i)[0]);
      const float by = M > -INFINITY ? M : 0.0f;
#pragma unroll 8
      for (int i = 0; i < nc + nh; ++i) {
        const float* p = slot(i);
        const float mi = p[0], li = p[1], v = p[2 + e];
        const float f = li == 0.0f ? 0.0f : mi > -INFINITY ? tq_exp2(mi - by) : 1.0f;
        if (f == 0.0f && li == 0.0f) continue;
        L += li * f;
        if (i < nc) x += v * f;
        else hot += v * f;
      }
    }
    cs[e][h] = x;
    __syncthreads();
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < TQ_D / 4; ++d) {
      const float4 v = *(const float4*)cs[32 * h + d];
      y[0] = fmaf(v.x, pi[d], y[0]), y[1] = fmaf(v.y, pi[d], y[1]);
      y[2] = fmaf(v.z, pi[d], y[2]), y[3] = fmaf(v.w, pi[d], y[3]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) ys[h][k][e] = y[k];
    __syncthreads();
    if (at < total) {
      const float o = (ys[0][h][e] + ys[1][h][e]) + (ys[2][h][e] + ys[3][h][e]) + hot;
      const float v = L == 0.0f ? 0.0f : o / L;
      const size_t to = (((size_t)s * a.n_tokens + row / G) * g.n_q_heads + head * G + row % G) * TQ_D + e;
      if (a.q_dtype == TQ_F32) ((float*)a.out)[to] = v;
      else if (a.q_dtype == TQ_F16) ((__half*)a.out)[to] = __float2half_rn(v);
      else ((__nv_bfloat16*)a.out)[to] = __float2bfloat16_rn(v);
    }
  }
}

template <int NT, bool SPLIT, int VB>
int launch_rows(const AttendArgs& a, int sm_count, cudaStream_t st) {
  using Shared = ArShared<NT, SPLIT, VB>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of one CTA");
  static_assert(SPLIT || NT > 1 || sizeof(Shared) <= 113 * 1024, "two CTAs on an SM");
  constexpr int PER_SM = !SPLIT && NT == 1 ? 2 : 1;
  const int row_tiles = (a.rows + 8 * NT - 1) / (8 * NT);
  const int64_t all = (int64_t)a.seq_count * a.g.n_kv_heads * a.rows;
  TQ_REQUIRE(all <= INT_MAX - 4 * AC_THREADS, TQ_ERR_UNSUPPORTED, "too many query rows in a call");
  TQ_REQUIRE((ArShape<NT, SPLIT, VB>::PAGE <= a.g.page_bytes), TQ_ERR_INVALID, "page size");
  TQ_CUDA(cudaFuncSetAttribute(attend_rows_kernel<NT, SPLIT, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)sizeof(Shared)));
  attend_rows_kernel<NT, SPLIT, VB><<<PER_SM * sm_count, AR_THREADS, sizeof(Shared), st>>>(a, row_tiles);
  TQ_CUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((all + 3) / 4, 2 * sm_count));
  cfg.blockDim = dim3(AC_THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TQ_CUDA(cudaLaunchKernelEx(&cfg, attend_rows_combine_kernel, a, row_tiles, 8 * NT, (int)all));
  return TQ_OK;
}

template <int NT, bool SPLIT>
int launch_rows(const AttendArgs& a, int sm_count, cudaStream_t st) {
  return a.g.value_bits == 4 ? launch_rows<NT, SPLIT, 4>(a, sm_count, st) : launch_rows<NT, SPLIT, 3>(a, sm_count, st);
}

}  // namespace

AttendRowsPlan tq_attend_rows_plan(const AttendArgs& a, int tokens, int sm_count) {
  const tq_geom& g = a.g;
  AttendRowsPlan p;
  const int nt = a.rows <= 8 ? 1 : 2;
  p.seqs = AR_SEQS;
  p.plan_bytes = align_up(sizeof(ArPlan), 256);
  // Slots for the states of a row: what its work meets at the shares of this call, and a few more (the kernel
  // makes the shares larger where they would not do).
  const int nb = n_cold_blocks(tokens, g.hot_window, AR_S);
  const int64_t pages = a.window == INT_MAX
                            ? nb
                            : std::min<int64_t>(nb, ((int64_t)a.window + a.n_tokens + 510) / 256 + (a.sinks + 255) / 256);
  const int64_t size = g.kv_dtype == TQ_F32 ? AR_HOT32 : AR_HOT;
  const int64_t hot = (std::min(tokens, g.hot_window) + size - 1) / size;
  const int64_t rows = (int64_t)std::min(a.seq_count, AR_SEQS) * g.n_kv_heads * ((a.rows + 8 * nt - 1) / (8 * nt));
  const int64_t ctas = (int64_t)sm_count * (a.q_dtype == TQ_BF16 && nt == 1 ? 2 : 1);
  const int64_t share = std::max<int64_t>((AR_COST * pages + hot) * rows / 2 / ctas, AR_COST);  // (others may be shorter)
  p.ns_cold = (int)std::min<int64_t>(AR_COST * pages / share + 3, 64);
  p.ns_hot = (int)std::min<int64_t>(hot / share + 3, 32);
  return p;
}

int tq_launch_attend_rows(const AttendArgs& a, int sm_count, cudaStream_t st) {
  if (a.q_dtype == TQ_BF16)
    return a.rows <= 8 ? launch_rows<1, false>(a, sm_count, st) : launch_rows<2, false>(a, sm_count, st);
  return a.rows <= 8 ? launch_rows<1, true>(a, sm_count, st) : launch_rows<2, true>(a, sm_count, st);
}

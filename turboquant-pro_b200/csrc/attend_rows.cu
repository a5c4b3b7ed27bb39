// Attention of few query rows per KV head on the codes: single tokens, drafts to verify, small chunks.
// 256-token blocks with per-channel keys; the products on mma.sync (m16n8k16) with the codes as the A operand,
// straight from a table into registers, and NT tiles of eight query rows as the B operand.
//
// Persistent CTAs, one an SM; every warp works alone, without barriers.  The 64-token strips of pages that the rows
// of each (sequence, KV head, row tile) see, first tokens, then the window, and after them the 32-token tiles of the
// uncompressed window, form one list that is cut into shares of equal cost, one per warp, so ragged batches and every
// number of heads balance; where a share leaves a row tile, or goes from pages to the window, the warp writes a
// state, and the merge sums these.  What a warp needs of a strip comes with cp.async into its own piece of shared
// memory, the key half of the next one while the values of this one are summed and the other way round:
//   weights  w = q * scale, scaled by a power of two per row, as fp16 pairs hi + lo in the registers of the B
//            operand, and the zero-points' part of the score, q . mean: once per page;
//   scores   a byte of key codes (two channels) is one look-up; hi * w and lo * w accumulate apart;
//   mask     by position, where a row of the tile does not see the whole strip;
//   softmax  running maximum and sum per row, in units of log 2, once per strip;
//   values   probability * norm, scaled by a power of two per row and strip, transposed in registers into the
//            B operand; two tokens' codes of a channel are one look-up.  The sums of a strip start from zero and are
//            added in float32.
// (With eight warps on a page, its weights in shared memory and a CTA per pair of heads it took twice as long: a
// page cost five barriers and twice the instructions.)
//
// SPLIT (float32 and float16 queries): the table's entries are hi + lo pairs too, hi * hi of 16 channels is added
// up in float32 registers, and outliers count with their exact stored value: as exact as float32 arithmetic.
// bfloat16 queries leave the table's lo part out (2^-11 of a level at worst, against the half step of their own type, 2^-8),
// and take the outliers from the page's list by token, which holds their distance from the grid in fp16: 1.6 to 1.95e-3 off
// (2-norms, 64 bits), a tenth more at most than rounding the exact result (1.57 to 1.75e-3: the spread is that of calls with few rows).
//
// The uncompressed window: 16-bit rows are the A operand as they are, in their own type (ldmatrix), so that only the
// other operand is split: a query that is exact in that type has one part, others as many as they need;
// probabilities have two parts in fp16 and in bfloat16 (three there with SPLIT).  float32 rows are split into fp16 pairs
// as they are read, each times a power of two of its own.  A tile that holds an infinity or a NaN is
// attended term by term instead (products with masked tokens and with low parts would spread it); of 16-bit keys, one
// whose scores are no numbers.
//
// Bound by look-ups, products and their latencies at twelve warps an SM: 44 % of the issue slots (29 % and 22 % with pairs, at
// eight warps, on short windows; 46 % on 32 listed blocks a row tile, where a scheduler's two warps have 4.4 cycles between
// instructions), a tenth of the waiting for instructions (a fifth for float32 windows: the code of all formats is long); at one
// row tile the codes are read once.  Measured, 8 KV heads, one token: 16 sequences of 8192 with a window of 4096 72.5 us, of
// these the merge's tail 10; 8 sequences of 8000 and five tokens, three row tiles, 100 us; one sequence, window 1024, 19 us, a
// chain of latencies.
#include <algorithm>

#include "attend.cuh"

namespace {

constexpr int AR_S = 256;          // tokens of a page
// Tiles of eight query rows that a warp takes at once: with two it takes twice the registers, eight warps an SM
// instead of twelve, and as long per row (18 000 cycles a strip against 13 000: 2 250 and 1 080 an SM).
constexpr int NT = 1;
constexpr int AR_STRIP = 64;       // of them, in an item of the list
constexpr int AR_HOT = 32;         // window tokens of an item
constexpr int AR_PITCH = TQ_D * 2 + 16, AR_PITCH32 = TQ_D * 4 + 16;  // bytes of a window row in shared memory
// How long a strip takes, by whether operands are pairs, and a tile of the window beside it.  Measured, tile to strip, us
// (8 KV heads of 4 query heads, one token, unless said):
//   bfloat16 on 16-bit windows   2:4, 3:4, 4:4: 16 x 8192 tokens 76, 72, 79; 8 x 8000 and five tokens 100, 99, 108; 8 x
//     3000 of 32 KV heads of one 73, 70, 76; 64 x 1500, window 700, 79, 82, 88; 32 x 700 39, 36, 35; 1 x 600 23, 23, 18
//   float16 and float32 on 16-bit windows   2:8, 3:8, 4:8, 6:8: 8 x 8192 83, 79, 79, 80; 64 x 700 73, 80, 82, 87; 16 x 3000
//     float32 on bfloat16 75, 71, 72, 72
//   bfloat16 on float32 windows   3:4, 4:4, 5:4, 6:4: 16 x 2000 of 4 x 7, two tokens, 63, 55, 59, 58; 32 x 700 -, 65, 69, 72
//   float16 and float32 on float32 windows   4:8, 6:8, 8:8, 10:8: 8 x 3000 of 32 x 1 177, 155, 148, 153; 4 x 20000, two
//     tokens, 106, 90, 85, 84; 16 x 3000 float16 98, 88, 82, 89; 32 x 700 76, 70, 72, 80; 1 x 600 35, 35, 24, 24.  Half of
//     that (HALF_HOT) where every warp then has one share of a strip's length, and would not otherwise: 1 x 2500 of 32 x 1,
//     window 2000, 39, 43, 44, -.  (The kernel cannot choose: that took 1.5 to 4 us of its prologue.)
inline int ar_hot_cost(int q_dtype, int kv_dtype) { return kv_dtype != TQ_F32 ? 3 : q_dtype == TQ_BF16 ? 4 : 8; }
constexpr int HALF_HOT = 4;
constexpr int AR_LIST = 256;       // outliers of a strip that are copied ahead (160 is usual)

template <bool SPLIT, int VB>
struct ArShape {
  static constexpr int N = 8 * NT;                     // query rows
  static constexpr int NV = VB == 4 ? 256 : 64;
  static constexpr int WARPS = SPLIT ? 8 : 12;         // as many as have room
  // sixteen copies of a table side by side: pairs fill a half warp's banks
  static constexpr int ENTRY = 16 * (SPLIT ? 8 : 4);   // bytes of an entry, copies and all
  static constexpr int LUTK = 256 * ENTRY, LUTV = NV * ENTRY;
};

// A warp's strip of a page, or the values of a tile of the window in its place.
template <bool SPLIT, int VB>
struct alignas(16) ArWarp {
  uint8_t keys[AR_STRIP * TQ_D / 2];
  uint16_t delta[TQ_ELL_SLOTS][AR_STRIP];
  uint8_t col[TQ_ELL_SLOTS][AR_STRIP];
  float scale[4][36], mean[4][36];  // 32 channels a row (the pad spreads a lane's rows over the banks)
  PageHeader hdr;
  uint32_t ovf[TQ_OVF_CAP];
  uint8_t values[AR_STRIP * TQ_D * VB / 8];
  float norms[AR_STRIP];
  uint32_t dec[SPLIT ? AR_LIST : 4];
  uint16_t val[SPLIT ? AR_LIST : 8];
  float corr[32][8 * NT];           // outliers' part of the scores of 32 tokens
  uint8_t q[TQ_D][8 * NT * (SPLIT ? 4 : 2)];  // row q_row(d): channel d
};
static_assert(AR_HOT * AR_PITCH <= 6528 + 64 * TQ_D * 3 / 8 + 256 && 16 * AR_PITCH32 <= 6528 + 64 * TQ_D * 3 / 8 + 256, "a tile of the window in a strip's place");

template <bool SPLIT, int VB>
struct ArShared {
  using Sh = ArShape<SPLIT, VB>;
  alignas(128) uint8_t lut[Sh::LUTK + Sh::LUTV];
  ArWarp<SPLIT, VB> warp[Sh::WARPS];
  float grid[16], cent[16];
  int2 seq[AR_SEQS];                            // tokens, query tokens
  int64_t cum[AR_SEQS + 1];                     // the cost of the sequences before
  int most[2];                                  // strips and window tiles of the longest row
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
// tq_scaled of a score, less `by`, without a rounding at the score's full size
TQ_DEV float ar_exponent(float x, float by) {
  constexpr TqFactor f{TQ_SCORE_LOG2};
  constexpr float hi = f.hi, lo = f.lo;
  return fmaf(x, lo, fmaf(x, hi, -by));
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
template <int N>
struct ArTiles {
  static constexpr int value = N;
};
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

// A sequence's work in a launch: its strips of pages (first tokens, then the window), then its tiles of the uncompressed
// window; the same for all of its heads and row tiles.
struct ArWork {
  AttendTiles strip, hot;
  int cold;  // tokens in blocks
  TQ_DEV int items() const { return strip.count() + hot.count(); }
  TQ_DEV int cost(int of_strip, int of_hot) const { return of_strip * strip.count() + of_hot * hot.count(); }
};
// What a call is: AR_LISTS, blocks that differ by query token and KV head; AR_BEGINNING, a part of one with a shared beginning that is
// not done as others are (queries behind all tokens, or the window done elsewhere).  Instances of their own: with what these take
// in it the kernel of plain calls spilled 72 bytes more, and 24 ragged float16 sequences took 82 us instead of 79.
enum ArKind { AR_PLAIN, AR_LISTS, AR_BEGINNING };
// AR_LISTS: as many strips as a list can have, whether it has them or not, for every query token and head alike.
template <ArKind KIND>
TQ_DEV ArWork ar_work(const AttendArgs& a, int n, int q_n) {
  ArWork w;
  w.cold = n_cold_blocks(n, a.g.hot_window, AR_S) * AR_S;
  const bool whole = KIND == AR_BEGINNING && a.whole, no_window = KIND != AR_PLAIN && a.no_window;
  const int p_lo = whole ? n : n - q_n, p_hi = q_n > 0 ? (whole ? n + q_n : n) - 1 : -1;
  w.strip = KIND == AR_LISTS ? AttendTiles{0, 0, p_hi >= 0 ? min(a.n_list, w.cold / AR_S) * (AR_S / AR_STRIP) : 0}
                             : attend_tiles(a, 0, w.cold, AR_STRIP, p_lo, p_hi);
  w.hot = no_window ? AttendTiles{0, 0, 0} : attend_tiles(a, w.cold, n, AR_HOT, p_lo, p_hi);
  return w;
}
// row tiles of a sequence that have query tokens
// (AR_LISTS: a tile has rows of one query token alone)
template <ArKind KIND>
TQ_DEV int ar_tiles(const AttendArgs& a, int q_n, int n) {
  return KIND == AR_LISTS ? q_n * ((a.g.group + n - 1) / n) : (q_n * a.g.group + n - 1) / n;
}

template <bool SPLIT, int VB, ArKind KIND>
__global__ void __launch_bounds__(32 * ArShape<SPLIT, VB>::WARPS, 1) attend_rows_kernel(AttendArgs a) {
  using Sh = ArShape<SPLIT, VB>;
  constexpr bool LIST = KIND == AR_LISTS;
  constexpr int N = Sh::N, WARPS = Sh::WARPS, THREADS = 32 * WARPS, COST = ar_cost(SPLIT);
  constexpr int VGB = TQ_GROUP_TOK * TQ_D * VB / 8;
  extern __shared__ __align__(128) uint8_t ar_shared[];
  ArShared<SPLIT, VB>& sh = *(ArShared<SPLIT, VB>*)ar_shared;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int H = g.n_kv_heads, G = g.group;
  const bool q32 = a.q_dtype == TQ_F32;
  ArWarp<SPLIT, VB>& my = sh.warp[warp];

  // ---- the work before every sequence
  if (tid < 16) {
    sh.grid[tid] = a.tables->grid[tid];
    sh.cent[tid] = a.tables->centroids[tid];
  }
  if (warp == 0) {
    constexpr int PER = AR_SEQS / 32;
    int most_strip = 0, most_hot = 0;
    int64_t cost[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      cost[i] = 0;
      if (s < a.seq_count) {
        const AttendSeq sq = attend_seq(a, s);
        sh.seq[s] = make_int2(sq.n, sq.q_n);
        const ArWork w = ar_work<KIND>(a, sq.n, sq.q_n);
        cost[i] = (int64_t)w.cost(COST, a.hot_cost) * (H * ar_tiles<KIND>(a, sq.q_n, N));
        most_strip = max(most_strip, w.strip.count());
        most_hot = max(most_hot, w.hot.count());
      }
      sum += cost[i];
    }
    int64_t before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    if (lane == 31) sh.cum[AR_SEQS] = before;
    before -= sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sh.cum[lane * PER + i] = before;
      before += cost[i];
    }
    most_strip = __reduce_max_sync(0xffffffffu, most_strip);
    most_hot = __reduce_max_sync(0xffffffffu, most_hot);
    if (lane == 0) sh.most[0] = most_strip, sh.most[1] = most_hot;
  }
  __syncthreads();
  // Shares of equal cost: what starts in [k share, (k + 1) share) is warp k's.  A row's strips then meet at most
  // COST * (strips - 1) / share + 2 warps, its window tiles likewise, which have to fit their slots; and
  // no share is smaller than a strip's cost, so that every warp between a row's first and last has a part.
  const int workers = gridDim.x * WARPS;
  const int64_t total = sh.cum[AR_SEQS];
  int64_t share = max((total + workers - 1) / workers, (int64_t)COST);
  share = max(share, (int64_t)((COST * sh.most[0] + a.ns_cold - 3) / (a.ns_cold - 2)));
  if (KIND == AR_PLAIN || a.ns_hot > 0) share = max(share, (int64_t)((a.hot_cost * sh.most[1] + a.ns_hot - 3) / (a.ns_hot - 2)));
  if (blockIdx.x == 0) {
    ArPlan* plan = (ArPlan*)a.plan;
    if (tid == 0) plan->share = share;
    for (int i = tid; i <= AR_SEQS; i += THREADS) plan->cum[i] = sh.cum[i];
    for (int i = tid; i < a.seq_count; i += THREADS) {
      const ArWork w = ar_work<KIND>(a, sh.seq[i].x, sh.seq[i].y);
      plan->seq[i] = make_int4(w.strip.count(), w.hot.count(), ar_tiles<KIND>(a, sh.seq[i].y, N), 0);
    }
  }
  // (neighbouring shares go to different SMs: where there are few, each has one to itself)
  const int64_t me = (int64_t)warp * gridDim.x + blockIdx.x;
  if (share * blockIdx.x >= total) return;  // (the whole CTA)


  // ---- where the share begins: sequence, head, row tile, item
  int64_t at = share * me;
  const int64_t stop = min(at + share, total);
  bool more = at < total;
  int s = 0, head = 0, rt = 0, it = 0, row_items = 0, row_strips = 0, row_tiles = 1;
  ArWork w;
  auto enter_seq = [&]() {
    w = ar_work<KIND>(a, sh.seq[s].x, sh.seq[s].y);
    row_strips = w.strip.count();
    row_items = w.items();
    row_tiles = ar_tiles<KIND>(a, sh.seq[s].y, N);
  };
  int64_t begin = 0;  // the cost of what is before this row
  if (more) {
    int x = 0, y = a.seq_count - 1;
    while (x < y) {  // the last sequence that starts here or before
      const int mid = (x + y + 1) >> 1;
      if (sh.cum[mid] <= at) x = mid;
      else y = mid - 1;
    }
    s = x;
    enter_seq();
    const uint32_t cost = (uint32_t)w.cost(COST, a.hot_cost);
    // (a sequence's cost may pass 32 bits, a row's does not)
    const int64_t in = at - sh.cum[s];
    const int row = in >> 31 == 0 ? (int)((uint32_t)in / cost) : (int)(in / cost);
    const int off = (int)(in - (int64_t)row * cost), strips = COST * row_strips;
    begin = at - off;
    head = row / row_tiles, rt = row - head * row_tiles;
    if (off < strips) {
      it = (off + COST - 1) / COST;
      at = begin + COST * it;
    } else {
      const int k = (off - strips + a.hot_cost - 1) / a.hot_cost;
      it = row_strips + k;
      at = begin + strips + a.hot_cost * k;
    }
  }
  auto next_row = [&]() {  // false: there is none
    begin += w.cost(COST, a.hot_cost);
    at = begin;
    it = 0;
    if (++rt < row_tiles) return true;
    rt = 0;
    if (++head < H) return true;
    head = 0;
    do ++s;
    while (s < a.seq_count && sh.cum[s + 1] == sh.cum[s]);
    if (s >= a.seq_count) return false;
    enter_seq();
    return true;
  };
  if (more && it == row_items) more = next_row();  // (it began within the last item of a row)
  more = more && at < stop;

  // ---- copies
  size_t uix = 0;
  uint32_t list_at = 0, list_end = 0;  // SPLIT: the strip's first entry of the page's list, the list's end
  const uint8_t* page = nullptr;
  const int32_t* list = nullptr;  // LIST: the row tile's blocks
  int row_valid = 0;              // and strips of these
  auto strip_at = [&](int i) { return LIST ? 4 * list[i >> 2] + (i & 3) : w.strip.at(i); };
  auto page_of = [&](int i) { return a.pages + (uix * g.max_blocks + (strip_at(i) >> 2)) * (size_t)g.page_bytes; };
  auto copy_keys = [&](const uint8_t* from, int t0, uint32_t first) {  // t0: of the strip in its page
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ar_cp16(my.keys + (32 * i + lane) * 16, from + t0 * (TQ_D / 2) + (32 * i + lane) * 16);
    ar_cp16(&my.scale[lane >> 3][(lane & 7) * 4], from + g.scale_off + lane * 16);
    ar_cp16(&my.mean[lane >> 3][(lane & 7) * 4], from + g.mean_off + lane * 16);
    if (SPLIT) {
      // (the list's slice is whole fours of entries, and its slab whole sixty-fours: pieces of four)
      const uint32_t base = first & ~3u;
      const size_t slab = uix * (size_t)g.pool_entries;
#pragma unroll
      for (int i = 0; i < AR_LIST / 128; ++i) {
        const uint32_t e = base + 4 * (32 * i + lane);
        if (e < list_end) {
          ar_cp16(my.dec + 4 * (32 * i + lane), a.pool_dec + slab + e);
          ar_cp8(my.val + 4 * (32 * i + lane), a.pool_val + slab + e);
        }
      }
    } else {
      const uint8_t* ed = from + g.hdr_off + TQ_ELL_OFF;      // 8 pieces a slot
      const uint8_t* ec = from + g.hdr_off + TQ_ELL_COL_OFF;  // 4 pieces a slot
      ar_cp16((uint8_t*)my.delta + lane * 16, ed + (lane >> 3) * (AR_S * 2) + t0 * 2 + (lane & 7) * 16);
      if (lane < 16) ar_cp16((uint8_t*)my.col + lane * 16, ec + (lane >> 2) * AR_S + t0 + (lane & 3) * 16);
      if (lane < 4) ar_cp16((uint8_t*)&my.hdr + lane * 16, from + g.hdr_off + lane * 16);
      else ar_cp16(my.ovf + (lane - 4) * 4, from + g.hdr_off + TQ_OVF_OFF + (lane - 4) * 16);
    }
  };
  auto copy_values = [&](const uint8_t* from, int t0) {
    const uint8_t* src = from + g.v_off + (size_t)(t0 / TQ_GROUP_TOK) * VGB;
#pragma unroll
    for (int i = 0; i < 4 * VGB / 512; ++i) ar_cp16(my.values + (32 * i + lane) * 16, src + (32 * i + lane) * 16);
    if (lane < 16) ar_cp16(my.norms + lane * 4, from + g.norm_off + t0 * 4 + lane * 16);
  };
  static_assert(sizeof(PageHeader) == 64 && TQ_OVF_CAP * 4 == 28 * 16, "pieces of the tail");
  // SPLIT: the list of the page of item i, and its first entry of token t0 or a later one
  auto open_list = [&](int i, int t0) {
    if (!SPLIT || g.outlier_k == 0) return;
    const PageMeta pm = a.page_meta[uix * g.max_blocks + (strip_at(i) >> 2)];
    list_end = pm.off + pm.cnt;
    uint32_t lo = pm.off, hi = list_end;
    const uint32_t* dec = a.pool_dec + uix * (size_t)g.pool_entries;
    if (t0 > 0)
      while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((int)(dec[mid] >> 24) < t0) lo = mid + 1;
        else hi = mid;
      }
    list_at = lo;
  };

  // ---- rows 8 t + 2 c + x are this lane's columns
  float acc[NT][8][4], m_run[NT][2], l_run[NT][2];
  int pos[NT][2], win[NT][2];
  int first_pos = 0, last_win = 0, p_lo = 0, p_hi = 0, row0 = 0;
  int token_end = 0;  // LIST: the row behind those of the tile's query token
  auto rows_end = [&]() { return LIST ? token_end : a.rows; };
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
  // the rows' queries in shared memory as they are; float32 ones are asked for as scores' units where they are used
  auto q_at = [&](int qrow, int n) -> float {
    if (SPLIT) return ((const float*)my.q[qrow])[n];
    return __uint_as_float((uint32_t)((const uint16_t*)my.q[qrow])[n] << 16);
  };
  // A row tile's queries and positions; in two parts, so that other work can go on while the queries come.
  float4 q_raw[N * (SPLIT ? 1 : 0) + 1];
  uint2 q_half[N];
  auto fetch_row = [&]() {
    uix = unit_index(g, a.layer, a.seq_begin + s, head);
    row0 = rt * N;
    if (LIST) {
      const int per = (G + N - 1) / N, token = rt / per;
      row0 = token * G + (rt - token * per) * N, token_end = (token + 1) * G;
      list = attend_list(a, s, token, head);
      row_valid = (AR_S / AR_STRIP) * attend_listed(a, list, w.cold / AR_S);
    }
    int i = row0 / G, k = row0 - i * G;  // query token and head of the group
    const int64_t from = (int64_t)s * a.q_seq + (int64_t)(head * G) * a.q_head + 4 * lane;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t e = from + (int64_t)i * a.q_tok + (int64_t)k * a.q_head;
      const bool there = row0 + n < rows_end();
      if (SPLIT && q32) q_raw[n] = there ? *(const float4*)((const float*)a.q + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      else q_half[n] = there ? *(const uint2*)((const uint16_t*)a.q + e) : make_uint2(0u, 0u);
      if (++k == G) k = 0, ++i;
    }
  };
  auto start_row = [&]() {
    const int n = sh.seq[s].x, q_n = sh.seq[s].y, first = KIND == AR_BEGINNING && a.whole ? n : n - q_n;
    const int last = min(min(row0 + N, rows_end()), q_n * G) - 1;
    p_lo = first + row0 / G;
    p_hi = last >= row0 ? first + last / G : -1;
    // whether tokens are seen by all rows of the tile goes by its earliest row and its latest window
    first_pos = min(row0 + N, rows_end()) - 1 <= last ? p_lo : -1;
    last_win = attend_window(a, max(p_hi, 0));
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = row0 + 8 * t + 2 * c + x;
        pos[t][x] = row <= last ? max(first + row / G, -1) : -1;
        win[t][x] = attend_window(a, pos[t][x]);
      }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (SPLIT) {
        float4 x = q_raw[k];
        if (!q32) {
          const float2 u = __half22float2(*(const __half2*)&q_half[k].x), f = __half22float2(*(const __half2*)&q_half[k].y);
          x = make_float4(u.x, u.y, f.x, f.y);
        }
        ((float*)my.q[q_row(4 * lane)])[k] = x.x, ((float*)my.q[q_row(4 * lane + 1)])[k] = x.y;
        ((float*)my.q[q_row(4 * lane + 2)])[k] = x.z, ((float*)my.q[q_row(4 * lane + 3)])[k] = x.w;
      } else {
        const uint2 x = q_half[k];
        ((uint16_t*)my.q[q_row(4 * lane)])[k] = (uint16_t)x.x, ((uint16_t*)my.q[q_row(4 * lane + 1)])[k] = (uint16_t)(x.x >> 16);
        ((uint16_t*)my.q[q_row(4 * lane + 2)])[k] = (uint16_t)x.y, ((uint16_t*)my.q[q_row(4 * lane + 3)])[k] = (uint16_t)(x.y >> 16);
      }
    }
    __syncwarp();
  };
  auto open_to_all = [&](int t0, int t1) { return t1 - 1 <= first_pos && (t0 >= last_win || t1 <= a.sinks); };
  auto open_to_none = [&](int t0, int t1) {
    return t0 > p_hi || (t1 <= attend_window(a, max(p_lo, 0)) && t0 >= a.sinks);
  };
  const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  // From the scores (q . k as it is) of TILES times 16 tokens from `t0` on to their probabilities: maximum and sum go
  // on, in units of log 2 (taken to the exponent in one multiply-add: a score in these units would be rounded once
  // more at its full size), the probability stays in `sc`, times a power of two that takes the row's largest probability * nv below 2^14.
  auto softmax = [&](auto& sc, int t0, int t_end, auto tiles, const auto& nv, float (&inv_n)[NT][2]) {
    constexpr int TILES = decltype(tiles)::value;
    const bool open = t0 + 16 * TILES <= t_end && open_to_all(t0, t0 + 16 * TILES);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t hidden = 0u;
        if (!open) {
#pragma unroll
          for (int h = 0; h < TILES; ++h)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int j = t0 + 16 * h + 8 * y + r;
              if (j >= t_end || j > pos[t][x] || (j < win[t][x] && j >= a.sinks)) hidden |= 1u << (2 * h + y);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < TILES; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (!(hidden >> (2 * h + y) & 1u)) top = fmaxf(top, sc[h][t][2 * y + x]);
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(m_run[t][x], tq_scaled<true>(top));
        // (-inf: nothing seen yet, or scores that are no numbers, which stay so)
        const float by = top > -INFINITY ? top : 0.0f, down = tq_exp2(m_run[t][x] - by);
        float sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int h = 0; h < TILES; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float e = hidden >> (2 * h + y) & 1u ? 0.0f : tq_exp2(ar_exponent(sc[h][t][2 * y + x], by));
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
        for (int h = 0; h < TILES; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) sc[h][t][2 * y + x] *= up;
      }
  };

  // ---- a strip of a page
  float inv_k, inv_v;  // of the tables
  const uint32_t lutk = ar_smem(sh.lut) + (lane & 15) * (SPLIT ? 8 : 4), lutv = lutk + Sh::LUTK;
  uint32_t bh[NT][8][2], bl[NT][8][2];  // weights: k-step j takes channels 32 c + 4 j .. + 3, column r is row 8 t + r
  float bias[NT][2], inv[NT][2];
  auto weights = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx = 0.0f;
      float4 b4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 s4 = *(const float4*)&my.scale[c][4 * j], m4 = *(const float4*)&my.mean[c][4 * j];
        const int d = 32 * c + 4 * j, n = 8 * t + r;
        const float q0 = q_at(q_row(d), n), q1 = q_at(q_row(d + 1), n), q2 = q_at(q_row(d + 2), n), q3 = q_at(q_row(d + 3), n);
        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(q0 * s4.x), fabsf(q1 * s4.y)), fmaxf(fabsf(q2 * s4.z), fabsf(q3 * s4.w))));
        b4.x = fmaf(q0, m4.x, b4.x), b4.y = fmaf(q1, m4.y, b4.y);
        b4.z = fmaf(q2, m4.z, b4.z), b4.w = fmaf(q3, m4.w, b4.w);
      }
      float b = (b4.x + b4.y) + (b4.z + b4.w);
      b += __shfl_xor_sync(0xffffffffu, b, 1);
      b += __shfl_xor_sync(0xffffffffu, b, 2);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      float i0;
      const float up = ar_lift(mx, 13, i0);
      i0 *= inv_k;
#pragma unroll
      for (int x = 0; x < 2; ++x) {  // of rows 2 c + x
        bias[t][x] = __shfl_sync(0xffffffffu, b, 8 * c + 4 * x);
        inv[t][x] = __shfl_sync(0xffffffffu, i0, 8 * c + 4 * x);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 s4 = *(const float4*)&my.scale[c][4 * j];
        const int d = 32 * c + 4 * j, n = 8 * t + r;
        ar_split(q_at(q_row(d), n) * up, s4.x, q_at(q_row(d + 1), n) * up, s4.y, bh[t][j][0], bl[t][j][0]);
        ar_split(q_at(q_row(d + 2), n) * up, s4.z, q_at(q_row(d + 3), n) * up, s4.w, bh[t][j][1], bl[t][j][1]);
      }
    }
  };
  auto add_corr = [&](float (&e)[N], float delta, int qrow) {
#pragma unroll
    for (int x = 0; x < N; x += 4) {
      if (SPLIT) {
        const float4 q4 = *(const float4*)((const float*)my.q[qrow] + x);
        e[x] = fmaf(q4.x, delta, e[x]), e[x + 1] = fmaf(q4.y, delta, e[x + 1]);
        e[x + 2] = fmaf(q4.z, delta, e[x + 2]), e[x + 3] = fmaf(q4.w, delta, e[x + 3]);
      } else {
        const uint2 q4 = *(const uint2*)((const uint16_t*)my.q[qrow] + x);
        e[x] = fmaf(__uint_as_float(q4.x << 16), delta, e[x]);
        e[x + 1] = fmaf(__uint_as_float(q4.x & 0xffff0000u), delta, e[x + 1]);
        e[x + 2] = fmaf(__uint_as_float(q4.y << 16), delta, e[x + 2]);
        e[x + 3] = fmaf(__uint_as_float(q4.y & 0xffff0000u), delta, e[x + 3]);
      }
    }
  };
  // (columns of a token's row in an order that spreads eight tokens over the banks)
  auto put_corr = [&](int tok, const float (&e)[N]) {
#pragma unroll
    for (int x = 0; x < N; x += 4)
      *(float4*)&my.corr[tok][x ^ (4 * (tok >> 2 & 1))] = make_float4(e[x], e[x + 1], e[x + 2], e[x + 3]);
  };
  // the outliers' part of the scores of tokens 32 half .. + 31 of the strip, which begins at token ts of its page
  uint32_t list_next = 0;
  auto corrections = [&](int half, int ts) {
    float e[N];
#pragma unroll
    for (int x = 0; x < N; ++x) e[x] = 0.0f;
    __syncwarp();  // (those before have been read)
    if (SPLIT) {
      // the pool's list, ordered by token: the lane that holds a token's first entry adds up all of them
      put_corr(lane, e);
      __syncwarp();
      const uint32_t base = list_at & ~3u;  // of what has been copied
      const size_t slab = uix * (size_t)g.pool_entries;
      auto dec_at = [&](uint32_t i) { return i - base < (uint32_t)AR_LIST ? my.dec[i - base] : a.pool_dec[slab + i]; };
      auto val_at = [&](uint32_t i) { return i - base < (uint32_t)AR_LIST ? my.val[i - base] : a.pool_val[slab + i]; };
      const int t0 = ts + 32 * half;
      const uint32_t first = half == 0 ? list_at : list_next;
      bool go = true;
      for (uint32_t i = first; go; i += 32) {
        const uint32_t k = i + lane;
        const int tok = k < list_end ? (int)(dec_at(k) >> 24) - t0 : 32;
        const uint32_t in = __ballot_sync(0xffffffffu, tok < 32);
        go = in == 0xffffffffu;
        if (!go) list_next = i + __popc(in);
        if (tok >= 32 || (k > first && (int)(dec_at(k - 1) >> 24) - t0 == tok)) continue;
#pragma unroll
        for (int x = 0; x < N; ++x) e[x] = 0.0f;
        for (uint32_t j = k; j < list_end; ++j) {
          const uint32_t u = dec_at(j);
          if ((int)(u >> 24) - t0 != tok) break;
          const int ch = (u >> 16) & 127;
          const float on_grid = sh.grid[my.keys[(tok + 32 * half) * (TQ_D / 2) + (ch >> 1)] >> (4 * (ch & 1)) & 15];
          // what the weights' part gives is taken off, and the value itself put in
          add_corr(e, fmaf(-my.scale[ch >> 5][ch & 31], on_grid, __half2float(__ushort_as_half(val_at(j))) - my.mean[ch >> 5][ch & 31]),
                   q_row(ch));
        }
        put_corr(tok, e);
      }
      __syncwarp();
      return;
    }
    const bool spilled = (my.hdr.flags & TQ_PAGE_SPILLED) != 0;
    const int tok = 32 * half + lane;
    if (!spilled) {
#pragma unroll
      for (int j = 0; j < TQ_ELL_SLOTS; ++j) add_corr(e, __half2float(__ushort_as_half(my.delta[j][tok])), my.col[j][tok]);
    }
    put_corr(lane, e);
    __syncwarp();
    // the rest of the list, ordered by token, as above
    const uint32_t* list = my.ovf;
    int e0 = my.hdr.ovf_start[ts >> 6], e1 = my.hdr.ovf_start[(ts >> 6) + 1];
    if (spilled) {
      list = a.pool_dec + uix * (size_t)g.pool_entries + my.hdr.off;
      e0 = 0, e1 = (int)my.hdr.cnt;
    }
    for (int i = e0 + lane; i < e1; i += 32) {
      uint32_t v = list[i];
      const int tk = (int)(v >> 24);
      if (tk >> 5 != (ts >> 5) + half || (i > e0 && (int)(list[i - 1] >> 24) == tk)) continue;
#pragma unroll
      for (int x = 0; x < N; ++x) e[x] = my.corr[tk & 31][x ^ (4 * (tk >> 2 & 1))];
      for (int j = i;;) {
        add_corr(e, __half2float(__ushort_as_half((unsigned short)(v & 0xffffu))), q_row((v >> 16) & 127));
        if (++j >= e1) break;
        v = list[j];
        if ((int)(v >> 24) != tk) break;
      }
      put_corr(tk & 31, e);
    }
    __syncwarp();
  };
  // scores of tokens 32 half .. + 31 of the strip
  auto strip_scores = [&](float (&sc)[2][NT][4], int half, int ts) {
    if (g.outlier_k > 0) corrections(half, ts);
    // (a loop, here and of the values: unrolled, the code did not fit the instruction caches)
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      uint32_t kw[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint4 v = *(const uint4*)(my.keys + (32 * half + 16 * h + 8 * x + r) * (TQ_D / 2) + c * 16);
        kw[x][0] = v.x, kw[x][1] = v.y, kw[x][2] = v.z, kw[x][3] = v.w;
      }
      float sum[NT][4], low[NT][4], pair[NT][4];
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
          if (SPLIT) {
            float d[4];
            ar_mma(d, ah, bh[t][j][0], bh[t][j][1], zero);
            ar_mma(low[t], al, bh[t][j][0], bh[t][j][1], low[t]);
            ar_mma(low[t], ah, bl[t][j][0], bl[t][j][1], low[t]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // (32 channels at a time)
              if (j & 1) sum[t][i] += pair[t][i] + d[i];
              else pair[t][i] = d[i];
            }
          } else {
            ar_mma(sum[t], ah, bh[t][j][0], bh[t][j][1], sum[t]);
            ar_mma(low[t], ah, bl[t][j][0], bl[t][j][1], low[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 8 * t + 2 * c + (i & 1), tok = 16 * h + 8 * (i >> 1) + r;
          // (small parts first)
          float x = bias[t][i & 1];
          if (g.outlier_k > 0) x += my.corr[tok][n ^ (4 * (tok >> 2 & 1))];
          sc[0][t][i] = sc[1][t][i];
          sc[1][t][i] = fmaf(sum[t][i], inv[t][i & 1], fmaf(low[t][i], inv[t][i & 1], x));
        }
    }
  };
  auto strip_values = [&](float (&sc)[2][NT][4], int half, const float (&nv)[2][2], const float (&inv_n)[NT][2]) {
    float f[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) f[t][0] = inv_n[t][0] * inv_v, f[t][1] = inv_n[t][1] * inv_v;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t hi, lo;
          // (a hidden token's norm may be anything)
          const float v = h == 0 ? nv[0][y] : nv[1][y];
          const float n0 = sc[0][t][2 * y] == 0.0f ? 0.0f : v, n1 = sc[0][t][2 * y + 1] == 0.0f ? 0.0f : v;
          ar_split(sc[0][t][2 * y], n0, sc[0][t][2 * y + 1], n1, hi, lo);
          sc[0][t][2 * y] = sc[1][t][2 * y], sc[0][t][2 * y + 1] = sc[1][t][2 * y + 1];
          ph[t][y] = ar_transpose(hi);
          if (SPLIT) pl[t][y] = ar_transpose(lo);
        }
      const uint8_t* grp = my.values + (2 * half + h) * VGB;
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
          uint32_t off;
          if (VB == 4) {
            off = __byte_perm(rec[pr >> 2], 0, 0x4440 + (pr & 3)) * Sh::ENTRY;
          } else {  // the 6-bit field at bit 6 pr, moved to where it is the entry's offset
            constexpr int UP = SPLIT ? 7 : 6;
            static_assert(VB == 4 || Sh::ENTRY == 1 << UP, "an entry's size");
            const int bit = 6 * pr, wd = bit >> 5, b = bit & 31;
            const uint32_t v = b < UP         ? rec[wd] << (UP - b)
                               : b > 26       ? __funnelshift_r(rec[wd], rec[wd + 1], b - UP)
                                              : rec[wd] >> (b - UP);
            off = v & (63u << UP);
          }
          if (SPLIT) {
            const uint2 v = ar_lut2(lutv + off);
            ah[x] = v.x, al[x] = v.y;
          } else {
            ah[x] = ar_lut1(lutv + off);
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
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][mt][i] = fmaf(d[i], f[t][i & 1], acc[t][mt][i]);
        }
      }
    }
  };

  // ---- a tile of the uncompressed window: 32 tokens.  KIND: TQ_F16, TQ_BF16, TQ_F32.
  uint32_t b3[SPLIT ? NT : 1][SPLIT ? 8 : 1][2];  // third parts of the queries (bfloat16 windows)
  // the queries as B operand, channels in the order of the weights
  auto hot_weights = [&]() {
    const bool bf = g.kv_dtype == TQ_BF16;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx = 0.0f, i0 = 1.0f, up = 1.0f;
#pragma unroll
      for (int k = 0; k < 32; ++k) mx = fmaxf(mx, fabsf(q_at(q_row(32 * c + k), 8 * t + r)));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (!bf) up = ar_lift(mx, 13, i0);
#pragma unroll
      for (int x = 0; x < 2; ++x) inv[t][x] = __shfl_sync(0xffffffffu, i0, 8 * c + 4 * x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int d = 32 * c + 4 * j + 2 * k;
          const float x = q_at(q_row(d), 8 * t + r), y = q_at(q_row(d + 1), 8 * t + r);
          if (bf) {
            uint32_t p[3] = {0u, 0u, 0u};
            ar_split_bf<SPLIT ? 3 : 1>(x, y, p);
            bh[t][j][k] = p[0], bl[t][j][k] = p[1];
            if (SPLIT) b3[t][j][k] = p[2];
          } else {
            ar_split(x, up, y, up, bh[t][j][k], bl[t][j][k]);
          }
        }
    }
  };
  size_t ring = 0;   // elements before the row of slot 0
  int slot0 = 0;     // slot of the tile's first token
  auto hot_row = [&](int i) {  // elements before the row of the tile's token i
    const int k = slot0 + i;
    return ring + (size_t)((k >= g.hot_cap ? k - g.hot_cap : k) * TQ_D);
  };
  auto hot_terms = [&](int t0, int n) {  // term by term
#pragma unroll 1
    for (int tok = t0; tok < min(t0 + AR_HOT, n); ++tok) {
      const size_t from = hot_row(tok - t0);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (tok > pos[t][x] || (tok < win[t][x] && tok >= a.sinks)) continue;
          float dot = 0.0f;
#pragma unroll 1
          for (int d = 0; d < TQ_D; ++d) dot = fmaf(q_at(q_row(d), 8 * t + 2 * c + x), attend_ld(a.hot_k, from + d, g.kv_dtype), dot);
          dot = tq_scaled<true>(dot);
          const float top = fmaxf(m_run[t][x], dot), by = top > -INFINITY ? top : 0.0f;
          const float down = tq_exp2(m_run[t][x] - by), e = tq_exp2(dot - by);
          m_run[t][x] = top;
          l_run[t][x] = l_run[t][x] * down + (r == 0 ? e : 0.0f);
#pragma unroll
          for (int mt = 0; mt < 8; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              acc[t][mt][2 * y + x] = fmaf(e, attend_ld(a.hot_v, from + 16 * mt + 8 * y + r, g.kv_dtype),
                                           acc[t][mt][2 * y + x] * down);
        }
    }
  };
  auto hot_attend = [&](int t0, int n, auto kind) {
    constexpr int KIND = decltype(kind)::value;
    constexpr bool BF = KIND == TQ_BF16, F32 = KIND == TQ_F32;
    uint8_t* const rows = my.keys;
    // values on their way: all 32 tokens, or the first 16 of float32
    auto fetch_values = [&](int h) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = F32 ? 16 * h + i : 2 * i + (lane >> 4);
        if (F32)
          ar_cp16_or_zero(rows + i * AR_PITCH32 + lane * 16, (const float*)a.hot_v + hot_row(row) + lane * 4, t0 + row < n);
        else
          ar_cp16_or_zero(rows + row * AR_PITCH + (lane & 15) * 16, (const uint16_t*)a.hot_v + hot_row(row) + (lane & 15) * 8,
                          t0 + row < n);
      }
      ar_commit();
    };
    fetch_values(0);
    bool odd = false;
    // float32 rows: a power of two per token (and its inverse), so that the pairs' digits depend neither on its size nor on
    // that of the others, hidden ones among them
    auto row_lift = [&](const float* from, float& inverse) {  // of 32 channels, this lane's
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 v = ((const float4*)from)[j];
        top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        odd |= !(fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < INFINITY);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      return ar_lift(top, 13, inverse);
    };
    float nv[2][2] = {{1.0f, 1.0f}, {1.0f, 1.0f}}, v_up[2][2];  // values of tokens 16 h + 8 y + r
    float sc[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // a lane's keys are channels 32 c .. + 31 of tokens r and r + 8
      float sum[NT][4], low[NT][4], pair[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[t][i] = low[t][i] = 0.0f;
      uint32_t kw[2][F32 ? 1 : 16];
      const void* row[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const size_t from = hot_row(min(16 * h + 8 * x + r, n - 1 - t0)) + 32 * c;  // (past the end: hidden whatever its key)
        row[x] = F32 ? (const void*)((const float*)a.hot_k + from) : (const void*)((const uint16_t*)a.hot_k + from);
        if (!F32)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4 v = ((const uint4*)row[x])[k];
            kw[x][4 * k] = v.x, kw[x][4 * k + 1] = v.y, kw[x][4 * k + 2] = v.z, kw[x][4 * k + 3] = v.w;
          }
      }
      float k_up[2] = {1.0f, 1.0f}, k_inv[2] = {1.0f, 1.0f};
      if (F32)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const size_t from = hot_row(min(16 * h + 8 * x + r, n - 1 - t0)) + 32 * c;
          k_up[x] = row_lift((const float*)a.hot_k + from, k_inv[x]);
          v_up[h][x] = row_lift((const float*)a.hot_v + from, nv[h][x]);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t ah[4], al[4] = {0u, 0u, 0u, 0u};
        if (F32) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float4 v = ((const float4*)row[x])[j];
            ar_split(v.x, k_up[x], v.y, k_up[x], ah[x], al[x]);
            ar_split(v.z, k_up[x], v.w, k_up[x], ah[2 + x], al[2 + x]);
          }
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) ah[x] = kw[x & 1][F32 ? 0 : 2 * j + (x >> 1)];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float d[4];
          if (BF) {
            ar_mma_bf(d, ah, bh[t][j][0], bh[t][j][1], zero);
            if (SPLIT) {
              ar_mma_bf(low[t], ah, bl[t][j][0], bl[t][j][1], low[t]);
              ar_mma_bf(low[t], ah, b3[t][j][0], b3[t][j][1], low[t]);
            }
          } else {
            ar_mma(d, ah, bh[t][j][0], bh[t][j][1], zero);
            if (SPLIT || F32) ar_mma(low[t], ah, bl[t][j][0], bl[t][j][1], low[t]);
            if (F32) ar_mma(low[t], al, bh[t][j][0], bh[t][j][1], low[t]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (j & 1) sum[t][i] += pair[t][i] + d[i];
            else pair[t][i] = d[i];
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = (sum[t][i] + low[t][i]) * inv[t][i & 1] * (F32 ? k_inv[i >> 1] : 1.0f);
          sc[h][t][i] = x;
          // An infinite key is no number next to a part that is zero, where the score may be -inf, a weight of zero.
          // (Rows of padding may hold anything: they do not count.)
          if (!F32) odd |= !(x == x) && pos[t][i & 1] >= 0;
        }
    }
    if (!F32) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      // an exponent of ones in either half of a word carries into the sign's place
      constexpr uint32_t ONE = KIND == TQ_F16 ? 0x04000400u : 0x00800080u;
      uint32_t carry = 0u;
#pragma unroll
      for (int i = 0; i < AR_HOT / 2; ++i) {
        const uint4 x = *(const uint4*)(rows + (2 * i + (lane >> 4)) * AR_PITCH + (lane & 15) * 16);
        carry |= ((x.x & 0x7fff7fffu) + ONE) | ((x.y & 0x7fff7fffu) + ONE) | ((x.z & 0x7fff7fffu) + ONE) | ((x.w & 0x7fff7fffu) + ONE);
      }
      odd |= (carry & 0x80008000u) != 0u;
    }
    if (__any_sync(0xffffffffu, odd)) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      hot_terms(t0, n);
      return;
    }
    float inv_n[NT][2];
    softmax(sc, t0, n, ArTiles<2>(), nv, inv_n);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (F32) {
        if (h == 1) {
          __syncwarp();  // (the first 16 have been read)
          fetch_values(1);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
      uint32_t p[NT][2][3] = {};
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (BF) ar_split_bf<SPLIT ? 3 : 2>(sc[h][t][2 * y], sc[h][t][2 * y + 1], p[t][y]);
          else ar_split(sc[h][t][2 * y], nv[h][y], sc[h][t][2 * y + 1], nv[h][y], p[t][y][0], p[t][y][1]);
#pragma unroll
          for (int k = 0; k < (BF && SPLIT ? 3 : 2); ++k) p[t][y][k] = ar_transpose(p[t][y][k]);
        }
      float up[2][2] = {};  // of tokens 2 c, 2 c + 1, and 8 further
      if (F32)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int k = 0; k < 2; ++k) up[y][k] = __shfl_sync(0xffffffffu, v_up[h][y], 8 * c + 4 * k);
      const uint32_t v_at = ar_smem(rows) + (16 * h + (lane & 7) + (lane >> 4) * 8) * AR_PITCH + (lane >> 3 & 1) * 16;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        uint32_t ah[4], al[4] = {0u, 0u, 0u, 0u};
        if (F32) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // channels r, r + 8; tokens 2 c, 2 c + 1, and 8 further
            const float* f = (const float*)(rows + (2 * c + 8 * (x >> 1)) * AR_PITCH32) + 16 * mt + r + 8 * (x & 1);
            ar_split(f[0], up[x >> 1][0], f[AR_PITCH32 / 4], up[x >> 1][1], ah[x], al[x]);
          }
        } else {
          ar_ldm<true>(ah, v_at + 32 * mt);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float d[4];
          if (BF) {
            if (SPLIT) {
              ar_mma_bf(d, ah, p[t][0][2], p[t][1][2], zero);
              ar_mma_bf(d, ah, p[t][0][1], p[t][1][1], d);
            } else {
              ar_mma_bf(d, ah, p[t][0][1], p[t][1][1], zero);
            }
            ar_mma_bf(d, ah, p[t][0][0], p[t][1][0], d);
          } else if (SPLIT || F32) {
            ar_mma(d, ah, p[t][0][1], p[t][1][1], zero);
            if (F32) ar_mma(d, al, p[t][0][0], p[t][1][0], d);
            ar_mma(d, ah, p[t][0][0], p[t][1][0], d);
          } else {
            ar_mma(d, ah, p[t][0][0], p[t][1][0], zero);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][mt][i] = fmaf(d[i], inv_n[t][i & 1], acc[t][mt][i]);
        }
      }
    }
  };

  // ---- a state
  auto flush = [&](bool hot) {
    const int64_t from = hot ? begin + COST * row_strips : begin;
    const int slot = (hot ? a.ns_cold : 0) + (int)(me - ar_div(from, share));
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) l_run[t][x] += __shfl_xor_sync(0xffffffffu, l_run[t][x], o);
        const int row = row0 + 8 * t + 2 * c + x;
        if (row >= rows_end()) continue;
        float* to = attend_partial(a, s * H + head, row, slot);
        if (r == 0) *(float2*)to = make_float2(m_run[t][x], l_run[t][x]);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
#pragma unroll
          for (int y = 0; y < 2; ++y) to[2 + 16 * mt + 8 * y + r] = acc[t][mt][2 * y + x];
      }
  };

  // ---- the share, item by item
  int strip = 0, ts = 0;  // a strip of the row, its first token in its page
  auto open_strips = [&]() {
    strip = strip_at(it), ts = (strip & 3) * AR_STRIP;
    page = page_of(it);
    open_list(it, ts);
    copy_keys(page, ts, list_at);
    ar_commit();
    copy_values(page, ts);
    ar_commit();
  };
  if (more) {  // (on their way while the tables are made)
    fetch_row();
    if (it < (LIST ? row_valid : row_strips)) open_strips();
  }
  {  // tables of pairs
    float max_k = 0.0f, max_v = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      max_k = fmaxf(max_k, fabsf(sh.grid[i]));
      max_v = fmaxf(max_v, fabsf(sh.cent[i]));
    }
    const float up_k = ar_lift(max_k, 7, inv_k), up_v = ar_lift(max_v, 7, inv_v);
    for (int e = tid; e < 256 + Sh::NV; e += THREADS) {
      uint32_t hi, lo;
      uint4* to;
      if (e < 256) {
        ar_split(sh.grid[e & 15], up_k, sh.grid[e >> 4], up_k, hi, lo);
        to = (uint4*)(sh.lut + e * Sh::ENTRY);
      } else {
        const int b = e - 256;
        ar_split(sh.cent[b & ((1 << VB) - 1)], up_v, sh.cent[b >> VB], up_v, hi, lo);
        to = (uint4*)(sh.lut + Sh::LUTK + b * Sh::ENTRY);
      }
#pragma unroll
      for (int i = 0; i < Sh::ENTRY / 16; ++i)
        to[(i + lane) % (Sh::ENTRY / 16)] = SPLIT ? make_uint4(hi, lo, hi, lo) : make_uint4(hi, hi, hi, hi);
    }
  }
  __syncthreads();  // (the last one)
  bool opened = true;
  while (more) {
    // a row tile's strips, then its tiles of the window, as far as the share goes
    if (!opened) {
      fetch_row();
      if (it < (LIST ? row_valid : row_strips)) open_strips();
    }
    opened = false;
    start_row();
    if (it < row_strips) {
      reset();
      bool new_page = true;
      while (!LIST || it < row_valid) {
        at += COST;
        const int i1 = it + 1;
        const bool last = i1 >= (LIST ? row_valid : row_strips) || at >= stop;
        const int next = last ? strip : strip_at(i1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // the key half has landed
        __syncwarp();
        if (new_page) weights();
        if (SPLIT) list_next = 0xffffffffu;
        // (32 tokens at a time: a loop of 64 did not fit the instruction caches)
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int t0 = strip * AR_STRIP + 32 * half;
          const bool seen = !open_to_none(t0, t0 + 32);
          float sc[2][NT][4] = {};
          if (seen || (SPLIT && half == 0)) strip_scores(sc, half, ts);  // (SPLIT: the second half's list begins where the first's ends)
          if (half == 1) {
            __syncwarp();  // the key half has been read
            if (!last) {
              const int nt = (next & 3) * AR_STRIP;
              const bool turn = next >> 2 != strip >> 2;  // another page
              const bool follows = !turn && next == strip + 1 && list_next != 0xffffffffu && seen;
              if (turn) page = page_of(i1);
              if (follows) list_at = list_next;
              else open_list(i1, nt);
              copy_keys(page, nt, list_at);
            }
            ar_commit();
            asm volatile("cp.async.wait_group 1;" ::: "memory");
          } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");  // the value half has landed
          }
          __syncwarp();
          if (seen) {
            float nv[2][2], inv_n[NT][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int y = 0; y < 2; ++y) nv[h][y] = my.norms[32 * half + 16 * h + 8 * y + r];
            softmax(sc, t0, w.cold, ArTiles<2>(), nv, inv_n);
            strip_values(sc, half, nv, inv_n);
          }
        }
        __syncwarp();  // the value half has been read
        if (!last) copy_values(page, (next & 3) * AR_STRIP);
        ar_commit();
        it = i1;
        if (last) break;
        new_page = next >> 2 != strip >> 2;
        strip = next, ts = (next & 3) * AR_STRIP;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      if (LIST && it < row_strips && at < stop) {  // (what the list does not have)
        const int64_t left = min((stop - at + COST - 1) / COST, (int64_t)(row_strips - it));
        it += (int)left, at += COST * left;
      }
      flush(false);
      more = at < stop;
    }
    if (more && it < row_items) {
      reset();
      hot_weights();
      const int n = sh.seq[s].x;
      ring = uix * (size_t)g.hot_cap * TQ_D;
#pragma unroll 1
      for (; it < row_items && at < stop; ++it, at += a.hot_cost) {
        const int t0 = w.cold + w.hot.at(it - row_strips) * AR_HOT;
        slot0 = t0 % g.hot_cap;
        if (open_to_none(t0, min(t0 + AR_HOT, n))) continue;
        if (g.kv_dtype == TQ_BF16) hot_attend(t0, n, ArTiles<TQ_BF16>());
        else if (g.kv_dtype == TQ_F16) hot_attend(t0, n, ArTiles<TQ_F16>());
        else hot_attend(t0, n, ArTiles<TQ_F32>());
        __syncwarp();  // the rows have been read
      }
      flush(true);
      more = at < stop;
    }
    if (more) more = next_row();
  }
}

// ---------------------------------------------------------------------------------------------------
// Merge of the states: a row's slots are summed in order by groups of 128 threads, a thread per channel; the pages' sum is
// then rotated by all 512 threads, a quarter of the input channels each, whose rows of Pi they hold in registers
// from before the states were there.  ROWS = 4: a group per row, four rows at a time; ROWS = 1 (few rows, which
// then have many slots): every group takes a fourth of the row's slots.
// ---------------------------------------------------------------------------------------------------
constexpr int AC_THREADS = 512;

// (PLAIN: neither lists nor a shared beginning.  Code that a call goes through once is waited for: with what these take in it, a cold
// call on 1000 tokens of 8 KV heads took 28.7 us instead of 27.7.)
template <int ROWS, bool PLAIN>
__global__ void __launch_bounds__(AC_THREADS, 2) attend_rows_combine_kernel(AttendArgs a, int tile, int total) {
  __shared__ __align__(16) float cs[TQ_D][4], ys[4][ROWS][TQ_D], hs[4][TQ_D], ls[4][TQ_D], ms[4];
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, e = tid % TQ_D, h = tid / TQ_D;
  const int H = g.n_kv_heads, G = g.group, cost = ar_cost(a.q_dtype != TQ_BF16);
  float pi[TQ_D / 4];
#pragma unroll
  for (int d = 0; d < TQ_D / 4; ++d) pi[d] = a.tables->pi[(32 * h + d) * TQ_D + e];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ArPlan* plan = (const ArPlan*)a.plan;
  const int64_t share = plan->share;
  for (int r0 = blockIdx.x * ROWS; r0 < total; r0 += gridDim.x * ROWS) {
    const int at = r0 + (ROWS == 4 ? h : 0);
    float hot = 0.0f, L = 0.0f, x = 0.0f, M = -INFINITY;
    int s = 0, head = 0, row = 0;
    if (at < total) {
      row = at % a.rows;
      const int unit = at / a.rows;
      s = unit / H, head = unit - s * H;
      const int4 seq = plan->seq[s];
      const int64_t before = plan->cum[s];
      const int rt = !PLAIN && a.listed ? row / G * ((G + tile - 1) / tile) + row % G / tile : row / tile;
      if (rt < seq.z) {
        const int64_t begin = before + (int64_t)(head * seq.z + rt) * (cost * seq.x + a.hot_cost * seq.y);
        const int64_t middle = begin + cost * seq.x;
        const int nc = seq.x > 0 ? (int)(ar_div(middle - cost, share) - ar_div(begin, share)) + 1 : 0;
        const int nh = seq.y > 0 ? (int)(ar_div(middle + a.hot_cost * (seq.y - 1), share) - ar_div(middle, share)) + 1 : 0;
        const float* base = attend_partial(a, unit, row, 0);
        constexpr int BATCH = 4, STEP = ROWS == 4 ? 1 : 4;
        for (int i0 = ROWS == 4 ? 0 : h; i0 < nc + nh; i0 += BATCH * STEP) {
          float m[BATCH], l[BATCH], v[BATCH];
          float top = M;
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + k * STEP;
            m[k] = -INFINITY, l[k] = v[k] = 0.0f;
            if (i < nc + nh) {
              const float* p = base + (size_t)(i < nc ? i : a.ns_cold + i - nc) * TQ_PART_STRIDE;
              m[k] = p[0], l[k] = p[1], v[k] = p[2 + e];
            }
          }
#pragma unroll
          for (int k = 0; k < BATCH; ++k) top = fmaxf(top, m[k]);
          const float by = top > -INFINITY ? top : 0.0f, down = M > -INFINITY ? tq_exp2(M - by) : 1.0f;
          L *= down, x *= down, hot *= down;
          M = top;
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            if (l[k] == 0.0f) continue;
            const float f = m[k] > -INFINITY ? tq_exp2(m[k] - by) : 1.0f;
            L = fmaf(l[k], f, L);
            if (i0 + k * STEP < nc) x = fmaf(v[k], f, x);
            else hot = fmaf(v[k], f, hot);
          }
        }
        if (ROWS == 1) {  // the four groups to one maximum
          if (e == 0) ms[h] = M;
          __syncthreads();
          const float top = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), by = top > -INFINITY ? top : 0.0f;
          const float down = M > -INFINITY ? tq_exp2(M - by) : 1.0f;
          L *= down, x *= down, hot *= down;
          M = top;
        }
      }
    }
    cs[e][h] = x;
    if (ROWS == 1) hs[h][e] = hot, ls[h][e] = L;
    __syncthreads();
    float y[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) y[k] = 0.0f;
#pragma unroll
    for (int d = 0; d < TQ_D / 4; ++d) {
      const float4 v = *(const float4*)cs[32 * h + d];
      if constexpr (ROWS == 4) {
        y[0] = fmaf(v.x, pi[d], y[0]), y[1] = fmaf(v.y, pi[d], y[1]);
        y[2] = fmaf(v.z, pi[d], y[2]), y[3] = fmaf(v.w, pi[d], y[3]);
      } else {
        y[0] = fmaf((v.x + v.y) + (v.z + v.w), pi[d], y[0]);
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) ys[h][k][e] = y[k];
    __syncthreads();
    if (at < total && (ROWS == 4 || h == 0)) {
      if (ROWS == 1) {
        hot = (hs[0][e] + hs[1][e]) + (hs[2][e] + hs[3][e]);
        L = (ls[0][e] + ls[1][e]) + (ls[2][e] + ls[3][e]);
      }
      const int k = ROWS == 4 ? h : 0;
      const float o = (ys[0][k][e] + ys[1][k][e]) + (ys[2][k][e] + ys[3][k][e]) + hot;
      attend_result<PLAIN>(a, s, head, row, e, M, L, o);
    }
    if (ROWS == 1) __syncthreads();  // (the sums have been read)
  }
}

// The same with the states of a shared beginning, of which there may be tens a row: eight rows at a time, two warps a row, a lane
// four channels, and eight states of each on their way at once.  (Merged by a kernel of their own before, 64 x 8 x 8 rows cost 25 us
// more, 32 x 8 x 4 rows 10.)
constexpr int AM_THREADS = 512, AM_ROWS = 8;
__global__ void __launch_bounds__(AM_THREADS, 1) attend_rows_merge_kernel(AttendArgs a, int tile, int total) {
  __shared__ __align__(16) float cs[AM_ROWS][TQ_D], hs[AM_ROWS][TQ_D], ys[4][AM_ROWS][TQ_D];
  __shared__ float ms[AM_ROWS], ls[AM_ROWS];
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e = tid % TQ_D, h = tid / TQ_D;
  const int H = g.n_kv_heads, cost = ar_cost(a.q_dtype != TQ_BF16);
  float pi[TQ_D / 4];
#pragma unroll
  for (int d = 0; d < TQ_D / 4; ++d) pi[d] = a.tables->pi[(32 * h + d) * TQ_D + e];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ArPlan* plan = (const ArPlan*)a.plan;
  const int64_t share = plan->share;
  const int in = warp >> 1, half = warp & 1;
  for (int r0 = blockIdx.x * AM_ROWS; r0 < total; r0 += gridDim.x * AM_ROWS) {
    const int at = r0 + in;
    float M = -INFINITY, L = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, hot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto weigh = [&](float top) {  // to the maximum `top`
      const float by = top > -INFINITY ? top : 0.0f, down = M > -INFINITY ? tq_exp2(M - by) : 1.0f;
      L *= down;
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] *= down, hot[c] *= down;
      M = top;
      return by;
    };
    if (at < total) {
      const int row = at % a.rows, unit = at / a.rows, s = unit / H, head = unit - s * H;
      const int4 seq = plan->seq[s];
      const int64_t before = plan->cum[s];
      const float* of_prefix = nullptr;
      int np = 0, np_cold = 0, stride = TQ_SLOT_STRIDE, skip = 4;
      if (attend_position(a, attend_seq(a, s), row) >= 0) {
        const size_t of = (size_t)head * a.before_rows + (size_t)s * a.rows + row;
        const bool general = a.shared.left[head] != 0;
        np = general ? 2 : a.shared.ns, np_cold = general ? 1 : a.shared.ns_cold;
        if (general) stride = TQ_PART_STRIDE, skip = 2;
        of_prefix = general ? a.shared.general + of * 2 * TQ_PART_STRIDE : a.shared.slots + of * np * TQ_SLOT_STRIDE;
      }
      int nc = 0, nh = 0;
      if (row / tile < seq.z) {  // (slots as in the kernel above)
        const int64_t begin = before + (int64_t)(head * seq.z + row / tile) * (cost * seq.x + a.hot_cost * seq.y);
        const int64_t middle = begin + cost * seq.x;
        nc = seq.x > 0 ? (int)(ar_div(middle - cost, share) - ar_div(begin, share)) + 1 : 0;
        nh = seq.y > 0 ? (int)(ar_div(middle + a.hot_cost * (seq.y - 1), share) - ar_div(middle, share)) + 1 : 0;
      }
      const float* own = attend_partial(a, unit, row, 0);
      constexpr int BATCH = 8;
      for (int i0 = half; i0 < np + nc + nh; i0 += 2 * BATCH) {
        float2 ml[BATCH], u[BATCH], v[BATCH];
        float top = M;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          ml[k] = make_float2(-INFINITY, 0.0f), u[k] = v[k] = make_float2(0.0f, 0.0f);
          const int i = i0 + 2 * k, o = i - np;
          if (o < nc + nh) {
            const float* p = o < 0 ? of_prefix + (size_t)i * stride : own + (size_t)(o < nc ? o : a.ns_cold + o - nc) * TQ_PART_STRIDE;
            ml[k] = *(const float2*)p;
            p += (o < 0 ? skip : 2) + 4 * lane;
            u[k] = *(const float2*)p, v[k] = *(const float2*)(p + 2);
          }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) top = fmaxf(top, ml[k].x);
        const float by = weigh(top);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float f = attend_weight(ml[k].x, ml[k].y, by);
          if (f == 0.0f) continue;
          const int i = i0 + 2 * k;
          const float y[4] = {u[k].x, u[k].y, v[k].x, v[k].y};
          L = fmaf(ml[k].y, f, L);
          if (i < np ? i < np_cold : i - np < nc) {
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = fmaf(y[c], f, x[c]);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) hot[c] = fmaf(y[c], f, hot[c]);
          }
        }
      }
    }
    // the second warp's to the first's
    if (half == 1) {
      *(float4*)&cs[in][4 * lane] = make_float4(x[0], x[1], x[2], x[3]);
      *(float4*)&hs[in][4 * lane] = make_float4(hot[0], hot[1], hot[2], hot[3]);
      if (lane == 0) ms[in] = M, ls[in] = L;
    }
    __syncthreads();
    if (half == 0) {
      const float m = ms[in], l = ls[in], by = weigh(fmaxf(M, m)), f = attend_weight(m, l, by);
      const float4 u = *(const float4*)&cs[in][4 * lane], v = *(const float4*)&hs[in][4 * lane];
      if (f != 0.0f) {
        L = fmaf(l, f, L);
        x[0] = fmaf(u.x, f, x[0]), x[1] = fmaf(u.y, f, x[1]), x[2] = fmaf(u.z, f, x[2]), x[3] = fmaf(u.w, f, x[3]);
        hot[0] = fmaf(v.x, f, hot[0]), hot[1] = fmaf(v.y, f, hot[1]), hot[2] = fmaf(v.z, f, hot[2]), hot[3] = fmaf(v.w, f, hot[3]);
      }
      *(float4*)&cs[in][4 * lane] = make_float4(x[0], x[1], x[2], x[3]);
      *(float4*)&hs[in][4 * lane] = make_float4(hot[0], hot[1], hot[2], hot[3]);
      __syncwarp();
      if (lane == 0) ms[in] = M, ls[in] = L;
    }
    __syncthreads();
    float y[AM_ROWS];
#pragma unroll
    for (int k = 0; k < AM_ROWS; ++k) y[k] = 0.0f;
#pragma unroll
    for (int d = 0; d < TQ_D / 4; d += 4)
#pragma unroll
      for (int k = 0; k < AM_ROWS; ++k) {
        const float4 v = *(const float4*)&cs[k][32 * h + d];
        y[k] = fmaf(v.x, pi[d], y[k]), y[k] = fmaf(v.y, pi[d + 1], y[k]);
        y[k] = fmaf(v.z, pi[d + 2], y[k]), y[k] = fmaf(v.w, pi[d + 3], y[k]);
      }
#pragma unroll
    for (int k = 0; k < AM_ROWS; ++k) ys[h][k][e] = y[k];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AM_ROWS / 4; ++i) {
      const int k = 4 * i + h;
      if (r0 + k >= total) break;
      const int row = (r0 + k) % a.rows, unit = (r0 + k) / a.rows, s = unit / H;
      attend_result(a, s, unit - s * H, row, e, ms[k], ls[k], (ys[0][k][e] + ys[1][k][e]) + (ys[2][k][e] + ys[3][k][e]) + hs[k][e]);
    }
    __syncthreads();  // (the rows have been read)
  }
}

template <bool SPLIT, int VB, ArKind KIND>
int launch_rows(const AttendArgs& a, cudaStream_t st) {
  using Shared = ArShared<SPLIT, VB>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of one CTA");
  const int64_t all = (int64_t)a.seq_count * a.g.n_kv_heads * a.rows;
  TQ_REQUIRE(all <= INT_MAX - 4 * AC_THREADS, TQ_ERR_UNSUPPORTED, "too many query rows in a call");
  static bool done[64];
  const int rc = attend_shared(attend_rows_kernel<SPLIT, VB, KIND>, sizeof(Shared), a.device, done);
  if (rc != TQ_OK) return rc;
  attend_rows_kernel<SPLIT, VB, KIND><<<a.sm_count, 32 * ArShape<SPLIT, VB>::WARPS, sizeof(Shared), st>>>(a);
  TQ_CUDA(cudaGetLastError());
  if (a.no_window) return TQ_OK;  // (the merge is another's)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  // A CTA per row while these are two an SM at most, else groups of threads with four rows at a time, in turn.  Whole
  // calls, 4000 tokens: 32 rows 29 us against 47, 256 rows 36 against 50; 8 x 1000 tokens: 256 rows 25 against 30, 512
  // rows 30 and 30, 1024 rows 44 against 35.
  const bool few = all <= 2 * a.sm_count;
  if (a.shared.slots != nullptr) {
    cfg.gridDim = dim3((unsigned)std::min<int64_t>((all + AM_ROWS - 1) / AM_ROWS, a.sm_count));
    cfg.blockDim = dim3(AM_THREADS);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TQ_CUDA(cudaLaunchKernelEx(&cfg, attend_rows_merge_kernel, a, 8 * NT, (int)all));
    return TQ_OK;
  }
  cfg.gridDim = dim3((unsigned)(few ? all : std::min<int64_t>((all + 3) / 4, 2 * a.sm_count)));
  cfg.blockDim = dim3(AC_THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const bool plain = !a.listed && a.states == nullptr && a.before == nullptr;
  const auto kernel = few ? plain ? attend_rows_combine_kernel<1, true> : attend_rows_combine_kernel<1, false>
                          : plain ? attend_rows_combine_kernel<4, true> : attend_rows_combine_kernel<4, false>;
  TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, 8 * NT, (int)all));
  return TQ_OK;
}

}  // namespace

AttendRowsPlan tq_attend_rows_plan(const AttendArgs& a, int tokens) {
  const tq_geom& g = a.g;
  AttendRowsPlan p;
  p.seqs = AR_SEQS;
  p.plan_bytes = align_up(sizeof(ArPlan), 256);
  // Slots for the states of a row: what its work meets at the shares of this call where the other sequences are
  // half as long, and a few more (the kernel makes the shares larger where they would not do).
  const int64_t in_blocks = (int64_t)n_cold_blocks(tokens, g.hot_window, AR_S) * AR_S;
  const int64_t seen = a.window == INT_MAX ? in_blocks : std::min<int64_t>(in_blocks, (int64_t)a.window + a.n_tokens + 128);
  const int64_t strips = a.listed ? std::min<int64_t>(a.n_list, in_blocks / AR_S) * (AR_S / AR_STRIP)
                                  : (seen + AR_STRIP - 1) / AR_STRIP + (std::min<int64_t>(a.sinks, in_blocks) + AR_STRIP - 1) / AR_STRIP;
  const int64_t hot = a.no_window ? 0 : (std::min(tokens, g.hot_window) + AR_HOT - 1) / AR_HOT;
  const int64_t tiles = a.listed ? (int64_t)a.n_tokens * ((g.group + 8 * NT - 1) / (8 * NT)) : (a.rows + 8 * NT - 1) / (8 * NT);
  const int64_t rows = (int64_t)std::min(a.seq_count, AR_SEQS) * g.n_kv_heads * tiles;
  const int64_t workers = (int64_t)a.sm_count * (a.q_dtype == TQ_BF16 ? ArShape<false, 3>::WARPS : ArShape<true, 3>::WARPS);
  const int cost = ar_cost(a.q_dtype != TQ_BF16);
  int hot_cost = ar_hot_cost(a.q_dtype, g.kv_dtype);
  if (hot_cost > HALF_HOT) {  // (by what the longest sequence's rows see, as ar_work has it)
    const int64_t room = workers * cost;
    const int64_t w = a.window == INT_MAX ? 0 : std::max<int64_t>((int64_t)tokens - a.n_tokens - a.window + 1, 0), first = w / AR_STRIP;
    const int64_t n_strips = a.listed ? strips : std::max<int64_t>(in_blocks / AR_STRIP - first, 0) +
                             std::min<int64_t>((std::min<int64_t>(a.sinks, in_blocks) + AR_STRIP - 1) / AR_STRIP, first);
    const int64_t n_hot = (tokens - in_blocks + AR_HOT - 1) / AR_HOT - std::max<int64_t>(w - in_blocks, 0) / AR_HOT;
    if (rows * (cost * n_strips + hot_cost * n_hot) > room && rows * (cost * n_strips + HALF_HOT * n_hot) <= room) hot_cost = HALF_HOT;
  }
  p.hot_cost = hot_cost;
  const int64_t share = std::max<int64_t>((cost * strips + hot_cost * hot) * ((rows + 1) / 2) / workers, cost);
  p.ns_cold = (int)std::min<int64_t>(cost * strips / share + 3, 1024);
  p.ns_hot = a.no_window ? 0 : (int)std::min<int64_t>(hot_cost * hot / share + 3, 64);
  return p;
}

template <ArKind KIND>
static int launch_form(const AttendArgs& a, cudaStream_t st) {
  if (a.q_dtype == TQ_BF16) return a.g.value_bits == 4 ? launch_rows<false, 4, KIND>(a, st) : launch_rows<false, 3, KIND>(a, st);
  return a.g.value_bits == 4 ? launch_rows<true, 4, KIND>(a, st) : launch_rows<true, 3, KIND>(a, st);
}

int tq_launch_attend_rows(const AttendArgs& a, cudaStream_t st) {
  if (a.listed) return launch_form<AR_LISTS>(a, st);
  return a.whole || a.no_window ? launch_form<AR_BEGINNING>(a, st) : launch_form<AR_PLAIN>(a, st);
}

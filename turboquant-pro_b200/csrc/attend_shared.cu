// Attention of many sequences' queries on a beginning that they share: every row of a KV head sees every token of one sequence.
// 16-bit queries, 256-token blocks with per-channel keys; the products run on tcgen05 with the accumulators in tensor
// memory.
//
// attend_shared_kernel   a CTA takes up to 256 rows of a head (SPLIT: 128) and a part of the prefix, 64 tokens at a time.
//     Eight warps turn codes into the two operands in shared memory (fp16, K-major core matrices of 8 rows x 16
//     bytes); a warp per half of 128 rows issues S = Q K^T and O += P V; a thread per row makes the probabilities, which
//     stay in tensor memory.  Codes are decoded where they are used: the operands, four times as large, never leave the SM.
//       keys    (mean - c + scale * grid[code]) times a power of two per CTA, two channels a look-up and one multiply-add in
//               float32, outliers put over it.  c is one vector per head, the zero-point of the first block: it moves all
//               scores of a row alike; what it takes off goes back into the state's maximum.
//       values  in code space, norm * centroid[code] times a power of two per tile: two tokens of a channel a look-up.
//     A row's error is that of its scores, and theirs comes from channels many times as wide as the others (half precision
//     rounds a key of 60 by up to 0.016): the eight widest of a head's first page have a second part, a product step of
//     its own.  The same 32768 tokens with three channels 20 times the others: 2.5e-3 -> 1.7e-3 off, rounding the exact
//     result gives 1.65e-3.
//     The uncompressed window is the work of CTAs of its own, whose sums are in the original basis.
//     Pages whose grids span more than 2^20 in a CTA's part, an outlier that is 64 times its grid, window tokens below 2^-20 of
//     their tile's largest, and what is no number set the flag of their head, which the general kernel then does.
//     What bounds it: 64 tokens take 3000 cycles for 256 rows (32768 tokens, 8 heads of 512 rows: 130 us, 0.53 PFLOP/s; 8192 and 128
//     rows 33 us; float16, 12345 tokens, 4 heads of 231 rows: 40).  The makers are busy for 2000 of them, the exponentials of
//     the two halves for 1150 each, the products for 1090, and a ring of three stages, for which there is shared memory, ties
//     them together; 49 % of the issue slots are used (58 % of those of cycles in which an SM has work).  Exponentials of both halves at once, or more of them on the
//     multiply-add units, measured the same.  Why 256 rows: codes are decoded once for all of a CTA's rows, and
//     tensor memory holds two halves' scores, probabilities and sums.
// attend_shared_merge_kernel   for other forms of the sequences' own tokens than few rows: merges a row's states in order,
//     rotates what is in code space, and leaves one state a row.
#include <algorithm>

#include "attend_tc.cuh"

namespace {

constexpr int PX_T = 64;                     // tokens of a tile: a strip of a page
constexpr int PX_S = 256;                    // tokens of a page
constexpr int PX_IMAGE = PX_T * TQ_D * 2, PX_QIMAGE = 128 * TQ_D * 2;
constexpr int PX_KLBO = PX_T * 16, PX_LBO = TQ_D * 16, PX_SBO = 128;  // from eight K to the next: keys; queries, values
// Warps: eight of softmax, two that issue products, two that put the outliers over the keys, eight that make operands.  A
// thread's registers, 96 at launch, are divided anew by warpgroup: 120, 64 and 88 (two, one and two groups: 480 = 5 x 96).
constexpr int PX_SOFTMAX = 256, PX_ISSUE = 128, PX_MAKERS = 256, PX_THREADS = PX_SOFTMAX + PX_ISSUE + PX_MAKERS;
#define PX_REGISTERS(how, n) asm volatile("setmaxnreg." how ".sync.aligned.u32 " n ";")
constexpr int PX_P = PX_T, PX_HALF = 128, PX_O = 256;  // tensor memory's columns, as in the form for many rows
constexpr int PX_STRIDE = TQ_SLOT_STRIDE;    // floats of a state
constexpr int PX_TOP = 8;                    // a page's largest key on the grid is lifted to 2^8 .. 2^9
constexpr int PX_LIST = 7;                   // outliers of a tile that a lane holds (160 of a tile are usual)
constexpr int PX_WIDE = 8;                   // channels whose keys are two parts
constexpr int PX_WLBO = PX_T * 16, PX_WIMAGE = 2 * PX_WLBO, PX_QWLBO = 128 * 16, PX_QWIMAGE = 2 * PX_QWLBO;

template <bool SPLIT>
struct PxShape {
  static constexpr int HALVES = SPLIT ? 1 : 2, ROWS = 128 * HALVES;
  static constexpr int PARTS = SPLIT ? 2 : 1;      // images of keys, and of values
  static constexpr int STAGES = SPLIT ? 2 : 3;
};
template <bool SPLIT, int VB>
struct PxShared {
  using Sh = PxShape<SPLIT>;
  static constexpr int WIDE = SPLIT ? 0 : 1;
  static constexpr int ENTRY_K = 128, ENTRY_V = VB == 4 ? 64 : 128;  // bytes of a table's entry, copies and all
  alignas(128) uint8_t q[Sh::HALVES][PX_QIMAGE];
  alignas(128) uint8_t kv[Sh::STAGES][2 * Sh::PARTS][PX_IMAGE];
  // the second parts of the wide channels (a step of 16 channels, the other eight of which stay zero), and their queries
  alignas(128) uint8_t wide[Sh::STAGES][WIDE ? PX_WIMAGE : 128], q_wide[Sh::HALVES][WIDE ? PX_QWIMAGE : 128];
  float levels[32];                          // of the keys' grid, of the values' codebook
  uint8_t wide_of[TQ_D];                     // a channel's place among the wide ones, or 255: none
  int wide_at[PX_WIDE];
  alignas(128) uint8_t lut_k[256 * ENTRY_K], lut_v[(VB == 4 ? 256 : 64) * ENTRY_V];
  alignas(16) float center[TQ_D];
  float2 of_tile[Sh::STAGES];                // the values' exponent, the keys' factor
  float top[2][8];
  float k_up;                                // the factor of the CTA's keys
  unsigned long long on_grid[Sh::STAGES], k_full[Sh::STAGES], v_full[Sh::STAGES], empty[Sh::STAGES];
  unsigned long long q_ready[2], s_full[2], s_read[2], p_full[2], o_done[2], drained[2];
  uint32_t tmem;
};

struct PrefixArgs {
  int32_t* left;   // [head]
  float* slots;    // [head][rows][ns][PX_STRIDE]
  int ns_cold, ns_hot, row_tiles;
};

TQ_DEV uint64_t px_lds64(uint32_t at) {
  uint64_t v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(at));  // (volatile, here and below: so that a batch stays one)
  return v;
}
TQ_DEV uint32_t px_lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
TQ_DEV void px_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
TQ_DEV void px_makers() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
static_assert(PX_MAKERS == 256 && PX_SOFTMAX == 256, "barriers");

template <bool SPLIT, int VB>
__global__ void __launch_bounds__(PX_THREADS, 1) attend_shared_kernel(AttendArgs a, PrefixArgs pa) {
  using Sh = PxShape<SPLIT>;
  using Shared = PxShared<SPLIT, VB>;
  constexpr int PARTS = Sh::PARTS, STAGES = Sh::STAGES, ROWS = Sh::ROWS;
  constexpr int VGB = TQ_GROUP_TOK * TQ_D * VB / 8;
  extern __shared__ __align__(128) uint8_t px_smem[];
  Shared& sh = *(Shared*)px_smem;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ns = pa.ns_cold + pa.ns_hot;
  const int split = blockIdx.x % ns, rt = blockIdx.x / ns % pa.row_tiles, head = blockIdx.x / ns / pa.row_tiles;
  const int G = g.group, row0 = rt * ROWS;
  const AttendSeq sq = attend_seq(a, 0);
  const bool hot = split >= pa.ns_cold;
  const int tiles = hot ? (sq.n - sq.cold + PX_T - 1) / PX_T : sq.cold / PX_T;
  const int part = hot ? split - pa.ns_cold : split, parts = hot ? pa.ns_hot : pa.ns_cold;
  const int k_lo = (int)((long)tiles * part / parts), n = (int)((long)tiles * (part + 1) / parts) - k_lo;
  auto slot_of = [&](int row) { return pa.slots + (((size_t)head * a.rows + row) * ns + split) * PX_STRIDE; };
  if (n == 0) {
    for (int r = tid; r < min(ROWS, a.rows - row0); r += PX_THREADS) *(float2*)slot_of(row0 + r) = make_float2(-INFINITY, 0.0f);
    return;
  }
  const bool listed = !hot && g.outlier_k > 0;  // two warps put the outliers over the keys
  const int held = blockIdx.x == 0 ? a.withhold : -1;  // test hook: a tile whose keys are never handed over
  const int groups = Sh::HALVES == 2 && a.rows - row0 > 128 ? 2 : 1;  // halves of the rows that there are
  const uint8_t* const pages = a.pages + page_offset(g, a.layer, a.seq_begin, head, 0);

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(enc_smem(&sh.on_grid[i]), PX_MAKERS / 32);
      mbar_init(enc_smem(&sh.k_full[i]), listed ? 1 : PX_MAKERS / 32);
      mbar_init(enc_smem(&sh.v_full[i]), PX_MAKERS / 32);
      mbar_init(enc_smem(&sh.empty[i]), groups);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(enc_smem(&sh.q_ready[i]), 128);
      mbar_init(enc_smem(&sh.s_full[i]), 1);
      mbar_init(enc_smem(&sh.s_read[i]), 128);
      mbar_init(enc_smem(&sh.p_full[i]), 128);
      mbar_init(enc_smem(&sh.o_done[i]), 1);
      mbar_init(enc_smem(&sh.drained[i]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == PX_SOFTMAX / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(enc_smem(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---- what the roles need, in two steps: from memory, and from what is then in shared memory.  (Loops, not unrolled: code that
  // runs once is waited for from memory, 700 instructions for 10 000 cycles.)  Queries: a thread per row.
  float factor = 0.0f, shift = 0.0f;  // of a row's scores; what the keys' common vector takes off them
  if (warp < 4 * groups) {
    const int row = row0 + tid;
    const bool there = row < a.rows;
    const uint16_t* q = (const uint16_t*)a.q;
    if (there) q += (int64_t)(row / G) * a.q_tok + (int64_t)(head * G + row % G) * a.q_head;
    const uint32_t to = enc_smem(sh.q[warp >> 2] + (tid & 127) * 16);
#pragma unroll 2
    for (int i = 0; i < 16; ++i)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * PX_LBO), "l"(q + 8 * i), "r"(there ? 16 : 0)
                   : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");  // (each thread its own row)
  } else if (warp >= PX_SOFTMAX / 32 && warp < (PX_SOFTMAX + PX_ISSUE) / 32) {
    const int d = tid - PX_SOFTMAX;
    static_assert(PX_ISSUE == TQ_D, "a thread per channel");
    sh.center[d] = sq.cold > 0 ? ti_center(g, pages, d) : 0.0f;
    const float scale = sq.cold > 0 ? ((const float*)(pages + g.scale_off))[d] : 0.0f;
    ((float*)sh.kv[0])[d] = scale < INFINITY ? scale : 0.0f;  // (numbers: places below are a permutation)
  } else if (warp >= (PX_SOFTMAX + PX_ISSUE) / 32 && tid < PX_SOFTMAX + PX_ISSUE + 32) {
    const int i = tid & 31;
    sh.levels[i] = i < 16 ? a.tables->grid[i] : a.tables->centroids[i - 16];
  }
  ti_fence_before();
  __syncthreads();
  ti_fence_after();
  if (warp < 4 * groups) {
    uint8_t* const from = sh.q[warp >> 2] + (tid & 127) * 16;
    auto pairs = [&](const uint4& w, float2 (&f)[4]) {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = SPLIT ? __half22float2(*(const __half2*)&u[j])
                     : make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u));
    };
    float top = 0.0f;
    uint64_t part[2] = {0ull, 0ull};
#pragma unroll 2
    for (int i = 0; i < 16; ++i) {
      float2 f[4];
      pairs(*(const uint4*)(from + i * PX_LBO), f);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float4 z = *(const float4*)&sh.center[8 * i + 2 * j];
        top = ti_max3(ti_max3(top, fabsf(f[j].x), fabsf(f[j].y)), fabsf(f[j + 1].x), fabsf(f[j + 1].y));
        part[0] = ti_fma2(ti_f2(f[j].x, f[j].y), ti_f2(z.x, z.y), part[0]);
        part[1] = ti_fma2(ti_f2(f[j + 1].x, f[j + 1].y), ti_f2(z.z, z.w), part[1]);
      }
    }
    const float2 of_center = ti_floats(ti_add2(part[0], part[1]));
    shift = tq_scaled<true>(of_center.x + of_center.y);
    float exponent;
    const float up = ti_lift(top, 13, exponent);
    factor = tq_scaled<true>(exp2f(exponent));
#pragma unroll 2
    for (int i = 0; i < 16; ++i) {
      float2 f[4];
      pairs(*(const uint4*)(from + i * PX_LBO), f);
      *(uint4*)(from + i * PX_LBO) = make_uint4(ti_pair(f[0].x * up, f[0].y * up), ti_pair(f[1].x * up, f[1].y * up),
                                                ti_pair(f[2].x * up, f[2].y * up), ti_pair(f[3].x * up, f[3].y * up));
    }
  } else if (warp >= (PX_SOFTMAX + PX_ISSUE) / 32) {
    if (!hot) {  // tables: an entry's copies side by side, so that the lanes of a look-up meet different banks
      const int pt = tid - PX_SOFTMAX - PX_ISSUE;
      for (int e = pt; e < 256 * 8; e += PX_MAKERS) {  // two copies at a time
        const int b = e >> 3;
        const float x = sh.levels[b & 15], y = sh.levels[b >> 4];
        *(float4*)(sh.lut_k + e * 16) = make_float4(x, y, x, y);
      }
      constexpr int NV = VB == 4 ? 256 : 64, PER = Shared::ENTRY_V / 16;
      for (int e = pt; e < NV * PER; e += PX_MAKERS) {
        const int b = e / PER;
        const float x = sh.levels[16 + (b & ((1 << VB) - 1))], y = sh.levels[16 + (b >> VB)];
        if (SPLIT) {
          *(float4*)(sh.lut_v + e * 16) = make_float4(x, y, x, y);
        } else {
          const uint32_t h = ti_pair(x, y);
          *(uint4*)(sh.lut_v + e * 16) = make_uint4(h, h, h, h);
        }
      }
    }
  } else if (!SPLIT && warp >= PX_SOFTMAX / 32) {
    // the widest channels, the lower of two equal ones first
    const int d = tid - PX_SOFTMAX;
    const float* scales = (const float*)sh.kv[0];
    const float mine = scales[d];
    int place = 0;
#pragma unroll 4
    for (int i = 0; i < TQ_D; i += 4) {
      const float4 x = *(const float4*)(scales + i);
      place += (x.x > mine || (x.x == mine && i < d)) + (x.y > mine || (x.y == mine && i + 1 < d)) +
               (x.z > mine || (x.z == mine && i + 2 < d)) + (x.w > mine || (x.w == mine && i + 3 < d));
    }
    sh.wide_of[d] = place < PX_WIDE ? place : 255;
    if (place < PX_WIDE) sh.wide_at[place] = d;
    for (int i = d; i < STAGES * PX_WIMAGE / 16; i += PX_ISSUE) ((uint4*)sh.wide)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = d; i < Sh::HALVES * PX_QWIMAGE / 16; i += PX_ISSUE) ((uint4*)sh.q_wide)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  px_fence();
  __syncthreads();
  constexpr uint32_t tmem = 0;  // (all 512 columns are this CTA's: they begin at the first)

  // Bounded waits: one that runs out sets the status bit, and the thread then waits for nothing more and starts no
  // products; those under way are waited for (with the full limit) before the CTA's memory goes.
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

  auto hand_over = [&](unsigned long long* bar) {  // operands, by a warp
    px_fence();
    __syncwarp();
    if (lane == 0) mbar_arrive(enc_smem(bar));
  };

  if (warp >= (PX_SOFTMAX + PX_ISSUE) / 32) {
    // ---- the makers of the operands
    PX_REGISTERS("dec", "88");
    const int pt = tid - PX_SOFTMAX - PX_ISSUE, pw = pt >> 5;
    const int token = pt & (PX_T - 1), quarter = pt / PX_T;  // of a token: 32 channels (window), two wide channels
    bool odd = false;
    auto put_key = [&](uint8_t* to, int chunk, int token, const float (&x)[8]) {  // eight channels of a token
      const uint4 hi = {ti_pair(x[0], x[1]), ti_pair(x[2], x[3]), ti_pair(x[4], x[5]), ti_pair(x[6], x[7])};
      *(uint4*)(to + chunk * PX_KLBO + token * 16) = hi;
      if (SPLIT)
        *(uint4*)(to + PX_IMAGE + chunk * PX_KLBO + token * 16) =
            make_uint4(ti_rest(x[0], x[1], hi.x), ti_rest(x[2], x[3], hi.y), ti_rest(x[4], x[5], hi.z), ti_rest(x[6], x[7], hi.w));
    };
    const int wide0 = SPLIT ? 0 : sh.wide_at[2 * quarter], wide1 = SPLIT ? 0 : sh.wide_at[2 * quarter + 1];
    auto put_wide = [&](int stage, float x, float y) {  // lifted keys of channels wide0 and wide1
      *(uint32_t*)(sh.wide[stage] + token * 16 + 4 * quarter) = ti_rest(x, y, ti_pair(x, y));
    };
    if (!hot) {
      // two warps expand the records of a group of 16 tokens; a lane: pairs 16 half .. + 15 of a record
      const int grp = pw >> 1, half = pw & 1, r = lane >> 2, c = lane & 3;
      // Keys: a thread has eight channels, whose scales and zero-points stay in registers, of four tokens; neighbouring lanes
      // have neighbouring tokens, so that eight of them write 128 bytes in a row.
      const int chunk = 4 * (pw & 3) + (lane >> 3), token0 = 32 * (pw >> 2) + (lane & 7);
      // What a tile needs is on its way while the tile before it is made.  (Without conditions: a value that may or may not have
      // been loaded is moved, and so waited for, at once.)
      uint32_t codes[4], wide_codes[2] = {0u, 0u}, rec[4];
      float2 norm2[2], norm_of;  // of the group; of tokens 2 lane, 2 lane + 1 of the strip
      float4 scale4[2], mean4[2];
      auto page_of = [&](int j) { return pages + (size_t)(j >> 2) * g.page_bytes; };
      auto fetch_keys = [&](int j) {
        const uint8_t* row = page_of(j) + (j & 3) * PX_T * (TQ_D / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[i] = *(const uint32_t*)(row + (token0 + 8 * i) * (TQ_D / 2) + 4 * chunk);
        if (!SPLIT)
          wide_codes[0] = row[token * (TQ_D / 2) + (wide0 >> 1)], wide_codes[1] = row[token * (TQ_D / 2) + (wide1 >> 1)];
      };
      auto fetch_norms = [&](int j) { norm_of = *(const float2*)(page_of(j) + g.norm_off + ((j & 3) * PX_T + 2 * lane) * 4); };
      auto fetch_values = [&](int j) {
        const uint8_t* from = page_of(j) + g.v_off + (size_t)((j & 3) * (PX_T / TQ_GROUP_TOK) + grp) * VGB;
        if (VB == 4) {
          const uint4 x = *(const uint4*)(from + half * 512 + lane * 16);
          rec[0] = x.x, rec[1] = x.y, rec[2] = x.z, rec[3] = x.w;
        } else {  // words 3 half .. + 2 of the record's six, two of which are side by side
          const uint8_t* at = from + lane * 8;
          rec[0] = *(const uint32_t*)(at + (half ? 256 + 4 : 0)), rec[1] = *(const uint32_t*)(at + (half ? 512 : 4));
          rec[2] = *(const uint32_t*)(at + (half ? 512 + 4 : 256)), rec[3] = 0u;
        }
        const float* norms = (const float*)(page_of(j) + g.norm_off) + (j & 3) * PX_T + 16 * grp + 2 * c;
        norm2[0] = *(const float2*)norms, norm2[1] = *(const float2*)(norms + 8);
      };
      auto fetch_page = [&](int j) {
        const float* s = (const float*)(page_of(j) + g.scale_off) + 8 * chunk;
        const float* m = (const float*)(page_of(j) + g.mean_off) + 8 * chunk;
        scale4[0] = *(const float4*)s, scale4[1] = *(const float4*)(s + 4);
        mean4[0] = *(const float4*)m, mean4[1] = *(const float4*)(m + 4);
      };
      fetch_page(k_lo);
      fetch_keys(k_lo);
      fetch_norms(k_lo);
      fetch_values(k_lo);
      // ---- the largest and the least that a channel of the CTA's pages may have
      float k_up, k_factor;
      {
        float most = 0.0f, least = INFINITY;
        const float gridmost = g.key_mode == TQ_KEYS_UNIFORM ? 15.0f : 1.0f;
        const float4 z4 = *(const float4*)&sh.center[4 * lane];
        for (int j = (k_lo & ~3) + 4 * pw; j < k_lo + n; j += 4 * (PX_MAKERS / 32)) {
          const float4 s4 = *(const float4*)(page_of(j) + g.scale_off + lane * 16);
          const float4 m4 = *(const float4*)(page_of(j) + g.mean_off + lane * 16);
          const float s[4] = {s4.x, s4.y, s4.z, s4.w}, m[4] = {m4.x - z4.x, m4.y - z4.y, m4.z - z4.z, m4.w - z4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = fmaf(fabsf(s[i]), gridmost, fabsf(m[i]));
            odd |= !(x < TI_KEY_MOST);
            most = fmaxf(most, x);
            if (x > 0.0f) least = fminf(least, x);
          }
        }
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
        if (lane == 0) sh.top[0][pw] = most, sh.top[1][pw] = least;
        px_makers();
#pragma unroll
        for (int i = 0; i < PX_MAKERS / 32; ++i) most = fmaxf(most, sh.top[0][i]), least = fminf(least, sh.top[1][i]);
        odd |= least < most * TI_LEAST;
        float exponent;
        k_up = ti_lift(most, PX_TOP, exponent, 97);
        k_factor = exp2f(exponent);
        if (pt == 0) sh.k_up = k_up;  // (the outliers' warps read it behind the first tile)
      }
      uint64_t s2[4], m2[4];
      float of_wide[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // scale and zero-point of the wide channels
#pragma unroll 1
      for (int k = 0; k < n; ++k) {
        const int j = k_lo + k, stage = k % STAGES, next = min(j + 1, k_lo + n - 1);
        if (k == 0 || (j & 3) == 0) {
          const float4 z0 = *(const float4*)&sh.center[8 * chunk], z1 = *(const float4*)&sh.center[8 * chunk + 4];
          s2[0] = ti_f2(scale4[0].x * k_up, scale4[0].y * k_up), s2[1] = ti_f2(scale4[0].z * k_up, scale4[0].w * k_up);
          s2[2] = ti_f2(scale4[1].x * k_up, scale4[1].y * k_up), s2[3] = ti_f2(scale4[1].z * k_up, scale4[1].w * k_up);
          m2[0] = ti_f2((mean4[0].x - z0.x) * k_up, (mean4[0].y - z0.y) * k_up);
          m2[1] = ti_f2((mean4[0].z - z0.z) * k_up, (mean4[0].w - z0.w) * k_up);
          m2[2] = ti_f2((mean4[1].x - z1.x) * k_up, (mean4[1].y - z1.y) * k_up);
          m2[3] = ti_f2((mean4[1].z - z1.z) * k_up, (mean4[1].w - z1.w) * k_up);
          if (!SPLIT) {
            const float* s = (const float*)(page_of(j) + g.scale_off);
            const float* m = (const float*)(page_of(j) + g.mean_off);
            of_wide[0] = s[wide0] * k_up, of_wide[1] = s[wide1] * k_up;
            of_wide[2] = (m[wide0] - sh.center[wide0]) * k_up, of_wide[3] = (m[wide1] - sh.center[wide1]) * k_up;
          }
        }
        if (k >= STAGES) wait(&sh.empty[stage], (k / STAGES - 1) & 1);
        __syncwarp();
        uint8_t* const ki = sh.kv[stage][0];
        uint8_t* const vi = sh.kv[stage][PARTS];
        float v_up;
        {
          const float x = fabsf(norm_of.x), y = fabsf(norm_of.y);
          odd |= !(x < INFINITY) || !(y < INFINITY);
          const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(x, y))));
          odd |= (x > 0.0f && x < most * TI_LEAST) || (y > 0.0f && y < most * TI_LEAST);
          float exponent;
          v_up = ti_lift(most, 14, exponent);
          if (pt == 0) sh.of_tile[stage] = make_float2(exponent, k_factor);
        }
        fetch_norms(next);
        {  // ---- keys
          const uint32_t lut = enc_smem(sh.lut_k) + (lane & 15) * 8;
#pragma unroll
          for (int i0 = 0; i0 < 4; i0 += 2) {  // (two tokens' look-ups at once)
            uint64_t y[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) y[i][e] = px_lds64(__byte_perm(codes[i0 + i], 0, 0x4440 + e) * 128 + lut);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = ti_floats(ti_fma2(y[i][e], s2[e], m2[e]));
                x[2 * e] = f.x, x[2 * e + 1] = f.y;
              }
              put_key(ki, chunk, token0 + 8 * (i0 + i), x);
            }
          }
          if (!SPLIT) {
            const float x = __uint_as_float(px_lds32(lut + (wide_codes[0] >> (4 * (wide0 & 1)) & 15u) * 128));
            const float y = __uint_as_float(px_lds32(lut + (wide_codes[1] >> (4 * (wide1 & 1)) & 15u) * 128));
            put_wide(stage, fmaf(x, of_wide[0], of_wide[2]), fmaf(y, of_wide[1], of_wide[3]));
          }
        }
        if (listed) hand_over(&sh.on_grid[stage]);
        else if (k != held) hand_over(&sh.k_full[stage]);
        fetch_keys(next);
        if ((next & 3) == 0) fetch_page(next);
        {  // ---- values
          const uint32_t lut = enc_smem(sh.lut_v) + (lane % (SPLIT ? Shared::ENTRY_V / 8 : Shared::ENTRY_V / 4)) * (SPLIT ? 8 : 4);
          uint32_t n2[2];
          uint64_t f2[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            n2[h] = ti_pair(norm2[h].x * v_up, norm2[h].y * v_up);
            f2[h] = ti_f2(norm2[h].x * v_up, norm2[h].y * v_up);
          }
          constexpr int AT_ONCE = SPLIT ? 4 : 8;
#pragma unroll
          for (int p0 = 0; p0 < 16; p0 += AT_ONCE) {
            uint64_t y[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
              const int p = p0 + i, at = 6 * p;
              const uint32_t code = VB == 4 ? __byte_perm(rec[p >> 2], 0, 0x4440 + (p & 3))
                                            : __funnelshift_r(rec[at >> 5], rec[min((at >> 5) + 1, 3)], at & 31) & 63u;
              y[i] = SPLIT ? px_lds64(code * Shared::ENTRY_V + lut) : px_lds32(code * Shared::ENTRY_V + lut);
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
              const int p = p0 + i, h = p & 1, d = r + 8 * (8 * half + (p >> 1));
              uint8_t* const to = vi + (2 * grp + h) * PX_LBO + d * 16 + 4 * c;
              if (SPLIT) {
                const float2 f = ti_floats(ti_fma2(y[i], f2[h], 0ull));
                const uint32_t hi = ti_pair(f.x, f.y);
                *(uint32_t*)to = hi;
                *(uint32_t*)(to + PX_IMAGE) = ti_rest(f.x, f.y, hi);
              } else {
                const uint32_t w = (uint32_t)y[i];
                const __half2 v = __hmul2(*(const __half2*)&w, *(const __half2*)&n2[h]);
                *(uint32_t*)to = *(const uint32_t*)&v;
              }
            }
          }
        }
        fetch_values(next);
        hand_over(&sh.v_full[stage]);
      }
    } else {
      // ---- the uncompressed window: a thread has a quarter of a token's channels
      const size_t ring = hot_offset_elems(g, a.layer, a.seq_begin, head);
      float(*const part_top)[4][PX_T] = (float(*)[4][PX_T])sh.lut_k;  // (the window has no use for the tables)
      // the largest of a tile; whether a token lies far below it, or something is no number
      auto largest = [&](float most, int which) {
        part_top[which][quarter][token] = most;
        const float mine = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        if (lane == 0) sh.top[which][pw] = mine;
        px_makers();
        float top = 0.0f, of_token = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sh.top[which][i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) of_token = fmaxf(of_token, part_top[which][i][token]);
        odd |= of_token > 0.0f && of_token < top * TI_LEAST;
        return top;
      };
#pragma unroll 1
      for (int k = 0; k < n; ++k) {
        const int stage = k % STAGES, t = sq.cold + (k_lo + k) * PX_T + token;
        if (k >= STAGES) wait(&sh.empty[stage], (k / STAGES - 1) & 1);
        __syncwarp();
        uint8_t* const ki = sh.kv[stage][0];
        uint8_t* const vi = sh.kv[stage][PARTS];
        const size_t row = ring + (size_t)(t % g.hot_cap) * TQ_D, at = row + 32 * quarter;
        const bool there = t < sq.n;
        float x[4][8], most = 0.0f, exponent, k_exponent, of_wide[2] = {0.0f, 0.0f};
        if (!SPLIT && there) {
          of_wide[0] = attend_ld(a.hot_k, row + wide0, g.kv_dtype);
          of_wide[1] = attend_ld(a.hot_k, row + wide1, g.kv_dtype);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (there) ti_ld8(a.hot_k, at + 8 * i, g.kv_dtype, x[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[i][e] = there ? x[i][e] - sh.center[32 * quarter + 8 * i + e] : 0.0f;
            odd |= !(fabsf(x[i][e]) < TI_KEY_MOST);
            most = fmaxf(most, fabsf(x[i][e]));
          }
        }
        const float k_up = ti_lift(largest(most, 0), 14, k_exponent, 97);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] *= k_up;
          put_key(ki, 4 * quarter + i, token, x[i]);
        }
        if (!SPLIT)
          put_wide(stage, there ? (of_wide[0] - sh.center[wide0]) * k_up : 0.0f, there ? (of_wide[1] - sh.center[wide1]) * k_up : 0.0f);
        most = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (there) ti_ld8(a.hot_v, at + 8 * i, g.kv_dtype, x[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[i][e] = there ? x[i][e] : 0.0f;
            odd |= !(fabsf(x[i][e]) < INFINITY);
            most = fmaxf(most, fabsf(x[i][e]));
          }
        }
        const float v_up = ti_lift(largest(most, 1), 14, exponent);
        if (pt == 0) sh.of_tile[stage] = make_float2(exponent, exp2f(k_exponent));
        if (k != held) hand_over(&sh.k_full[stage]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = x[i][e] * v_up;
            const __half hi = __float2half_rn(y);
            uint8_t* const to = vi + (token >> 3) * PX_LBO + (32 * quarter + 8 * i + e) * 16 + (token & 7) * 2;
            *(__half*)to = hi;
            if (SPLIT) *(__half*)(to + PX_IMAGE) = __float2half_rn(y - __half2float(hi));
          }
        hand_over(&sh.v_full[stage]);
      }
    }
    if (odd) pa.left[head] = 1;
  } else if (warp >= PX_SOFTMAX / 32) {
    // (the whole warpgroup, and where its paths part, not before: the compiler allocates by what it sees on a path)
    PX_REGISTERS("dec", "64");
    if (warp >= PX_SOFTMAX / 32 + 2) {
    // ---- outliers: two warps, a tile each in turn, put the entries of the page's list, which is ordered by token, over its keys
    if (listed) {
      const int hw = warp - PX_SOFTMAX / 32 - 2;
      const size_t uix = unit_index(g, a.layer, a.seq_begin, head);
      float k_up = 0.0f;
      bool odd = false;
      wait(&sh.on_grid[0], 0);  // (the factor is there)
      __syncwarp();
      k_up = sh.k_up;
      const PageMeta* const metas = a.page_meta + uix * g.max_blocks;
      // Where a tile's entries begin: behind the last of 32 samples of the page's list that is before it.  (The samples are those of
      // a page, and they are asked for ahead, as are its place and length: three loads that wait for one another otherwise.)
      PageMeta meta = {0, 0}, meta_next = {0, 0};
      int sample = 4;
      auto open_page = [&]() {
        const uint32_t e = lane * ((meta.cnt + 31) / 32);
        sample = 4;
        if (e < meta.cnt) sample = (int)(a.pool_dec[uix * (size_t)g.pool_entries + meta.off + e] >> 30);
      };
      if (hw < n) {
        meta = metas[(k_lo + hw) >> 2];
        open_page();
      }
#pragma unroll 1
      for (int k = hw; k < n; k += 2) {
        const int j = k_lo + k, stage = k % STAGES, strip = j & 3;
        const uint32_t* const dec = a.pool_dec + uix * (size_t)g.pool_entries + meta.off;
        const uint16_t* const val = a.pool_val + uix * (size_t)g.pool_entries + meta.off;
        const int before = __popc(__ballot_sync(0xffffffffu, sample < strip));
        const uint32_t first = before > 0 ? (before - 1) * ((meta.cnt + 31) / 32) : 0u;
        uint32_t key[PX_LIST], rest[PX_LIST];
#pragma unroll
        for (int i = 0; i < PX_LIST; ++i) {
          key[i] = rest[i] = 0u;
          const uint32_t at = first + 32 * i + lane;
          if (at < meta.cnt) key[i] = dec[at], rest[i] = val[at];
        }
        const bool turn = k + 2 < n && (j + 2) >> 2 != j >> 2;
        if (turn) meta_next = metas[(j + 2) >> 2];
        // (whether the last entry held may be followed by more of the tile's)
        const bool more = __shfl_sync(0xffffffffu, first + 32 * PX_LIST < meta.cnt && (int)(key[PX_LIST - 1] >> 30) <= strip, 31);
        // An entry as it is put: its place in the tile's image | the key; the key's second part | the channel's place among the
        // wide ones, or 256: none of the tile's.
        auto prepare = [&](uint32_t& key, uint32_t& rest, bool there) {
          const uint32_t t = key >> 24, ch = key >> 16 & 127u;
          const float x = (__half2float(__ushort_as_half((unsigned short)rest)) - sh.center[ch]) * k_up;
          there = there && t >> 6 == (uint32_t)strip;
          odd |= there && !(fabsf(x) < 32768.0f);
          const __half hi = __float2half_rn(x), lo = __float2half_rn(x - __half2float(hi));
          key = (ch >> 3) * PX_KLBO + (t & (PX_T - 1)) * 16 + (ch & 7u) * 2 | (uint32_t)__half_as_ushort(hi) << 16;
          rest = (uint32_t)__half_as_ushort(lo) << 16 | (there ? sh.wide_of[ch] : 256u);
        };
        static_assert(16 * PX_KLBO <= 65536 && PX_KLBO == 1024, "an entry's place");
        uint8_t* const ki = sh.kv[stage][0];
        uint8_t* const wi = sh.wide[stage];
        auto put = [&](uint32_t key, uint32_t rest) {
          const uint32_t place = rest & 511u;
          if (place < 256u) {
            *(uint16_t*)(ki + (key & 0xffffu)) = (uint16_t)(key >> 16);
            if (SPLIT) *(uint16_t*)(ki + PX_IMAGE + (key & 0xffffu)) = (uint16_t)(rest >> 16);
          }
          if (!SPLIT && place < PX_WIDE) *(uint16_t*)(wi + (key & 0x3f0u) + 2 * place) = (uint16_t)(rest >> 16);
        };
#pragma unroll
        for (int i = 0; i < PX_LIST; ++i) prepare(key[i], rest[i], first + 32 * i + lane < meta.cnt);
        wait(&sh.on_grid[stage], (k / STAGES) & 1);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PX_LIST; ++i) put(key[i], rest[i]);
        if (more)
          for (uint32_t at = first + 32 * PX_LIST + lane; at < meta.cnt; at += 32) {
            uint32_t x = dec[at], y = val[at];
            if ((int)(x >> 30) > strip) break;
            prepare(x, y, true);
            put(x, y);
          }
        __syncwarp();
        if (k != held) hand_over(&sh.k_full[stage]);
        if (turn) {
          meta = meta_next;
          open_page();
        }
      }
      if (odd) pa.left[head] = 1;
    }
    } else {
    // ---- products of half x: the whole warp runs this, one thread issues
    const int x = warp - PX_SOFTMAX / 32, n_u = __shfl_sync(0xffffffffu, x < groups ? n : 0, 0);
    if (n_u > 0) {
      constexpr uint32_t s_desc = (1u << 4) | ((uint32_t)(PX_T >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t o_desc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint64_t KSTEP = 2 * PX_KLBO >> 4, STEP = 2 * PX_LBO >> 4;  // 16 deep
      const uint64_t q = umma_desc_k_major(enc_smem(sh.q[0]), PX_LBO, PX_SBO) + (uint64_t)(x * (PX_QIMAGE >> 4));
      const uint64_t k0 = umma_desc_k_major(enc_smem(sh.kv[0][0]), PX_KLBO, PX_SBO);
      const uint64_t v0 = umma_desc_k_major(enc_smem(sh.kv[0][PARTS]), PX_LBO, PX_SBO);
      const uint64_t q_wide = umma_desc_k_major(enc_smem(sh.q_wide[0]), PX_QWLBO, PX_SBO) + (uint64_t)(x * (PX_QWIMAGE >> 4));
      const uint64_t k_wide = umma_desc_k_major(enc_smem(sh.wide[0]), PX_WLBO, PX_SBO);
      const uint32_t ds = tmem + PX_HALF * x, dp = tmem + PX_P + PX_HALF * x, d_o = tmem + PX_O + 128 * x;
      auto image = [&](int k, int part) {
        return (uint64_t)((uint32_t)(k % STAGES) * (2 * PARTS * PX_IMAGE >> 4) + part * (PX_IMAGE >> 4));
      };
      auto wait_all = [&](unsigned long long* bar, unsigned parity) {  // (the warp stays together)
        wait(bar, parity);
        gave_up = __any_sync(0xffffffffu, gave_up);
      };
      auto scores = [&](int k) {
        uint64_t b[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) b[i] = k0 + image(k, i);
        if (ti_elect()) {
          ti_mma<false>(ds, q, b[PARTS - 1], s_desc);
#pragma unroll
          for (int j = 1; j < 8; ++j) ti_mma<true>(ds, q + j * STEP, b[PARTS - 1] + j * KSTEP, s_desc);
          if (SPLIT)
#pragma unroll
            for (int j = 0; j < 8; ++j) ti_mma<true>(ds, q + j * STEP, b[0] + j * KSTEP, s_desc);
          else
            ti_mma<true>(ds, q_wide, k_wide + (uint64_t)((uint32_t)(k % STAGES) * (PX_WIMAGE >> 4)), s_desc);
          umma_commit(enc_smem(&sh.s_full[x]));
        }
        __syncwarp();
      };
      auto values = [&](int k) {
        uint64_t b[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) b[i] = v0 + image(k, i);
        if (ti_elect()) {
          if (k == 0) ti_mma_ts<false>(d_o, dp, b[PARTS - 1], o_desc);
          else ti_mma_ts<true>(d_o, dp, b[PARTS - 1], o_desc);
#pragma unroll
          for (int j = 1; j < PX_T / 16; ++j) ti_mma_ts<true>(d_o, dp + 8 * j, b[PARTS - 1] + j * STEP, o_desc);
          if (SPLIT)
#pragma unroll
            for (int j = 0; j < PX_T / 16; ++j) ti_mma_ts<true>(d_o, dp + 8 * j, b[0] + j * STEP, o_desc);
          umma_commit(enc_smem(&sh.o_done[x]));
          umma_commit(enc_smem(&sh.empty[k % STAGES]));  // (both operands: the scores were formed before)
        }
        __syncwarp();
      };
      wait_all(&sh.q_ready[x], 0);
      wait_all(&sh.k_full[0], 0);
      ti_fence_after();
      if (!gave_up) scores(0);
#pragma unroll 1
      for (int k = 0; k < n_u && !gave_up; ++k) {
        if (k + 1 < n_u) {
          wait_all(&sh.k_full[(k + 1) % STAGES], ((k + 1) / STAGES) & 1);
          wait_all(&sh.s_read[x], k & 1);  // (this tile's scores are in registers)
          if (gave_up) break;
          ti_fence_after();
          scores(k + 1);
        }
        wait_all(&sh.v_full[k % STAGES], (k / STAGES) & 1);
        wait_all(&sh.p_full[x], k & 1);
        if (gave_up) break;
        ti_fence_after();
        values(k);
      }
      // (no products are under way when the CTA's memory goes)
      if (ti_elect()) umma_commit(enc_smem(&sh.drained[x]));
      __syncwarp();
      gave_up = false;
      wait_for(&sh.drained[x], 0, TI_WAIT);
    }
    }
  } else {
    PX_REGISTERS("inc", "120");
    if (warp < 4 * groups) {
    // ---- a thread per row
    const int x = warp >> 2, r = tid & 127, row = row0 + 128 * x + r;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + PX_HALF * x + lanes, tp = tmem + PX_P + PX_HALF * x + lanes;
    const uint32_t to = tmem + PX_O + 128 * x + lanes;
    auto settled = [&](unsigned long long* bar, unsigned parity) {
      wait(bar, parity);
      __syncwarp();
      ti_fence_after();
    };
    {
      if (!SPLIT)
#pragma unroll
        for (int i = 0; i < PX_WIDE; ++i) {
          const int d = sh.wide_at[i];
          *(uint16_t*)(sh.q_wide[x] + r * 16 + 2 * i) = *(const uint16_t*)(sh.q[x] + (d >> 3) * PX_LBO + r * 16 + (d & 7) * 2);
        }
      px_fence();
      mbar_arrive(enc_smem(&sh.q_ready[x]));
    }
    float m = -INFINITY, l = 0.0f;
    if (groups == 2 && x == 1) asm volatile("bar.arrive 1, 256;" ::: "memory");
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      wait(&sh.k_full[k % STAGES], (k / STAGES) & 1);
      const float2 of_tile = sh.of_tile[k % STAGES];
      const float e = of_tile.x, by = factor * of_tile.y;
      settled(&sh.s_full[x], k & 1);
      uint32_t v[PX_T];
      ti_ld32(ts, v);
      ti_ld32(ts + 32, v + 32);
      ti_wait_ld();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.s_read[x]));
      if (hot) {
        const int there = sq.n - sq.cold - (k_lo + k) * PX_T;
        if (there < PX_T)
#pragma unroll
          for (int i = 0; i < PX_T; ++i)
            if (i >= there) v[i] = 0xff800000u;
      }
      float top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) top[i] = fmaxf(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
#pragma unroll
      for (int i = 16; i < PX_T; i += 2)
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
      if (k > 0) settled(&sh.o_done[x], (k - 1) & 1);  // (the probabilities before have been used)
      if (rescaled) {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          uint32_t o[16];
          ti_ld16(to + 16 * i, o);
          ti_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * down);
          ti_st8(to + 16 * i, o);
          ti_st8(to + 16 * i + 8, o + 8);
        }
      }
      if (groups == 2) asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");
      const float off = TI_LIFT + e - (m > -INFINITY ? m : 0.0f);
      const uint64_t factor2 = ti_f2(by, by), off2 = ti_f2(off, off);
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int i = 0; i < PX_T / 2; i += 8) {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t y = ti_fma2(ti_u2(v[2 * (i + j)], v[2 * (i + j) + 1]), factor2, off2);
          const float2 z = ti_exp2_unit(y);
          sum[j & 1] = ti_add2(sum[j & 1], ti_f2(z.x, z.y));
          h[j] = ti_pair(z.x, z.y);
        }
        ti_st8(tp + i, h);
      }
      if (groups == 2 && (x == 0 || k + 1 < n)) asm volatile("bar.arrive %0, 256;" ::"r"(2 - x) : "memory");
      ti_wait_st();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.p_full[x]));
      const float2 s2 = ti_floats(ti_add2(sum[0], sum[1]));
      l = fmaf(s2.x + s2.y, exp2f(-e), l * down);
    }
    settled(&sh.o_done[x], (n - 1) & 1);
    if (row < a.rows) *(float2*)slot_of(row) = make_float2(m - TI_LIFT + shift, l);
    // The sums go through the queries' place, which the warp's rows have 64 columns at a time, so that half a warp writes 256
    // bytes of a row in a row.  (The scores' products, which read it, are long done; the other half has a place of its own.)
    uint8_t* const place = sh.q[x] + (warp & 3) * 8192;
    auto at = [&](int r, int c4) { return (float4*)(place + r * 256 + ((c4 ^ (r & 15)) << 4)); };
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t o[16];
        ti_ld16(to + 64 * half + 16 * i, o);
        ti_wait_ld();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *at(lane, 4 * i + j) = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]),
                                             __uint_as_float(o[4 * j + 3]));
      }
      __syncwarp();
      const int first = row0 + 128 * x + 32 * (warp & 3) + (lane >> 4);
#pragma unroll 4
      for (int i = 0; i < 32; i += 2)
        if (first + i < a.rows) *(float4*)(slot_of(first + i) + 4 + 64 * half + 4 * (lane & 15)) = *at(i + (lane >> 4), lane & 15);
      __syncwarp();
    }
    }
  }
  __syncwarp();
  ti_fence_before();
  __syncthreads();
  if (warp == PX_SOFTMAX / 32) {
    ti_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------
// Merge of a row's states: a group of 128 threads a row, four rows at a time, a thread per channel; the sums in code space are
// then rotated by all 512 threads, a quarter of the input channels each, whose rows of Pi they hold in registers.
constexpr int PM_THREADS = 512;
__global__ void __launch_bounds__(PM_THREADS, 2) attend_shared_merge_kernel(AttendArgs a, PrefixArgs pa) {
  __shared__ __align__(16) float cs[TQ_D][4], ys[4][4][TQ_D];
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, e = tid % TQ_D, h = tid / TQ_D, total = g.n_kv_heads * a.rows;
  float pi[TQ_D / 4];
#pragma unroll
  for (int d = 0; d < TQ_D / 4; ++d) pi[d] = a.tables->pi[(32 * h + d) * TQ_D + e];
  for (int r0 = blockIdx.x * 4; r0 < total; r0 += gridDim.x * 4) {
    const int at = r0 + h;
    float M = -INFINITY, L = 0.0f, x = 0.0f, hot = 0.0f;
    if (at < total) {
      const int head = at / a.rows, row = at - head * a.rows;
      const bool general = pa.left[head] != 0;  // (its two states)
      const int nc = general ? 1 : pa.ns_cold, ns = general ? 2 : nc + pa.ns_hot, skip = general ? 2 : 4;
      const int step = general ? TQ_PART_STRIDE : PX_STRIDE;
      const float* base = general ? attend_partial(a, head, row, 0) : pa.slots + ((size_t)head * a.rows + row) * ns * PX_STRIDE;
      constexpr int BATCH = 4;
      for (int i0 = 0; i0 < ns; i0 += BATCH) {
        float m[BATCH], l[BATCH], v[BATCH], top = M;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          m[k] = -INFINITY, l[k] = v[k] = 0.0f;
          if (i0 + k < ns) {
            const float* p = base + (size_t)(i0 + k) * step;
            m[k] = p[0], l[k] = p[1], v[k] = p[skip + e];
          }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) top = fmaxf(top, m[k]);
        const float by = top > -INFINITY ? top : 0.0f, down = M > -INFINITY ? tq_exp2(M - by) : 1.0f;
        L *= down, x *= down, hot *= down;
        M = top;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float f = attend_weight(m[k], l[k], by);
          if (f == 0.0f) continue;
          L = fmaf(l[k], f, L);
          if (i0 + k < nc) x = fmaf(v[k], f, x);
          else hot = fmaf(v[k], f, hot);
        }
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
      float* to = a.states + (size_t)at * TQ_PART_STRIDE;
      if (e == 0) *(float2*)to = make_float2(M, L);
      to[2 + e] = (ys[0][h][e] + ys[1][h][e]) + (ys[2][h][e] + ys[3][h][e]) + hot;
    }
  }
}

struct Layout {
  size_t left, slots, partials, total;
};
Layout layout(const AttendArgs& a) {
  Layout l;
  const size_t rows = (size_t)a.g.n_kv_heads * a.rows;
  l.left = 0;
  l.slots = align_up((size_t)a.g.n_kv_heads * 4, 256);
  l.partials = align_up(l.slots + rows * (a.ns_cold + a.ns_hot) * PX_STRIDE * 4, 256);
  l.total = align_up(l.partials + rows * 2 * TQ_PART_STRIDE * 4, 256);
  return l;
}

template <bool SPLIT, int VB>
int launch(const AttendArgs& a, const PrefixArgs& pa, cudaStream_t st) {
  using Shared = PxShared<SPLIT, VB>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of one CTA");
  static bool done[64];
  const int rc = attend_shared(attend_shared_kernel<SPLIT, VB>, sizeof(Shared), a.device, done);
  if (rc != TQ_OK) return rc;
  const int64_t grid = (int64_t)a.g.n_kv_heads * pa.row_tiles * (pa.ns_cold + pa.ns_hot);
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (head, query row) tiles in a call");
  attend_shared_kernel<SPLIT, VB><<<(int)grid, PX_THREADS, sizeof(Shared), st>>>(a, pa);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}
int rows_of_cta(const AttendArgs& a) { return a.q_dtype == TQ_F16 ? PxShape<true>::ROWS : PxShape<false>::ROWS; }

}  // namespace

// Splits of the blocks and of the window, one of whose tiles takes as long as two: of as many as fill the GPU once, twice .. those
// with the least time, with six tiles' time for what a CTA does besides.
void tq_attend_shared_plan(const AttendArgs& a, int tokens, int* ns_cold, int* ns_hot) {
  const tq_geom& g = a.g;
  const int64_t cold = (int64_t)n_cold_blocks(tokens, g.hot_window, PX_S) * (PX_S / PX_T);
  const int64_t hot = std::max((std::min(tokens, g.hot_window) + PX_T - 1) / PX_T, 1);
  const int64_t units = (int64_t)g.n_kv_heads * ((a.rows + rows_of_cta(a) - 1) / rows_of_cta(a));
  int64_t best = INT64_MAX;
  *ns_cold = *ns_hot = 1;
  for (int rounds = 1; rounds <= 8; ++rounds) {
    const int64_t ctas = std::min<int64_t>(rounds * (int64_t)a.sm_count / std::max<int64_t>(units, 1), 256);  // of a unit
    if (ctas < 2) continue;
    int64_t each = std::max<int64_t>((cold + 2 * hot + ctas - 1) / ctas, 1), nc, nh;  // tiles of a CTA
    for (;; ++each) {
      nc = std::max<int64_t>((cold + each - 1) / each, 1), nh = std::min((2 * hot + each - 1) / each, hot);
      if (nc + nh <= ctas) break;
    }
    if (rounds * (each + 6) < best) best = rounds * (each + 6), *ns_cold = (int)nc, *ns_hot = (int)nh;
  }
}

size_t tq_attend_shared_bytes(const AttendArgs& a) { return layout(a).total; }

int tq_launch_attend_shared(const AttendArgs& base, void* workspace, bool merged, SharedStates* as,
                            cudaStream_t st) {
  AttendArgs a = base;
  const Layout l = layout(a);
  uint8_t* w = (uint8_t*)workspace;
  PrefixArgs pa;
  pa.left = (int32_t*)(w + l.left);
  pa.slots = (float*)(w + l.slots);
  pa.ns_cold = a.ns_cold, pa.ns_hot = a.ns_hot;
  pa.row_tiles = (a.rows + rows_of_cta(a) - 1) / rows_of_cta(a);
  TQ_REQUIRE((int64_t)a.g.n_kv_heads * a.rows <= INT_MAX - 4 * PM_THREADS, TQ_ERR_UNSUPPORTED, "too many query rows in a call");
  TQ_CUDA(cudaMemsetAsync(pa.left, 0, (size_t)a.g.n_kv_heads * 4, st));
  int rc;
  if (a.q_dtype == TQ_F16) rc = a.g.value_bits == 4 ? launch<true, 4>(a, pa, st) : launch<true, 3>(a, pa, st);
  else rc = a.g.value_bits == 4 ? launch<false, 4>(a, pa, st) : launch<false, 3>(a, pa, st);
  if (rc != TQ_OK) return rc;
  a.left = pa.left;
  a.ns_cold = a.ns_hot = 1;
  a.partials = (float*)(w + l.partials);
  a.unit_stride = (int64_t)a.rows * 2 * TQ_PART_STRIDE;
  rc = tq_launch_attend_general(a, st);
  if (rc != TQ_OK) return rc;
  *as = {pa.slots, pa.left, a.partials, pa.ns_cold, pa.ns_cold + pa.ns_hot};
  if (!merged) return TQ_OK;
  const int64_t rows = (int64_t)a.g.n_kv_heads * a.rows;
  attend_shared_merge_kernel<<<(int)std::min<int64_t>((rows + 3) / 4, 2 * a.sm_count), PM_THREADS, 0, st>>>(a, pa);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

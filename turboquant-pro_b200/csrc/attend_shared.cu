// Attention of many sequences' queries on a beginning that they share: every row of a KV head sees every token of one sequence.
// 16-bit queries, 256-token blocks with per-channel keys; the products run on tcgen05 with the accumulators in tensor
// memory.
//
// attend_shared_kernel   a CTA takes up to 256 rows of a head (SPLIT: 128) and a part of the prefix, 64 tokens at a time.
//     Eight warps turn codes into the two operands in shared memory (fp16, K-major core matrices of 8 rows x 16
//     bytes); a warp per half of 128 rows issues S = Q K^T and O += P V; a thread per row makes the probabilities, which
//     stay in tensor memory.  Codes are decoded where they are used: the operands, four times as large, never leave the SM.
//       keys    (mean - c + scale * grid[code]) times a power of two per page, two channels a look-up and one multiply-add in
//               float32, outliers put over it.  c is one vector per head, the zero-point of the first block: it moves all
//               scores of a row alike; what it takes off goes back into the state's maximum.
//       values  in code space, norm * centroid[code] times a power of two per tile: two tokens of a channel a look-up.
//     The uncompressed window is the work of CTAs of its own, whose sums are in the original basis.
//     A page whose grid spans more than 2^20, an outlier that is 64 times its grid, window tokens below 2^-20 of their
//     tile's largest, and what is no number set the flag of their head, which the general kernel then does.
// attend_shared_merge_kernel   merges a row's states in order, rotates what is in code space, and leaves one state a row.
#include <algorithm>

#include "attend_tc.cuh"

namespace {

constexpr int PX_T = 64;                     // tokens of a tile: a strip of a page
constexpr int PX_S = 256;                    // tokens of a page
constexpr int PX_IMAGE = PX_T * TQ_D * 2, PX_QIMAGE = 128 * TQ_D * 2;
constexpr int PX_KLBO = PX_T * 16, PX_LBO = TQ_D * 16, PX_SBO = 128;  // from eight K to the next: keys; queries, values
constexpr int PX_SOFTMAX = 256, PX_MAKERS = 256, PX_THREADS = PX_SOFTMAX + 64 + PX_MAKERS;
constexpr int PX_P = PX_T, PX_HALF = 128, PX_O = 256;  // tensor memory's columns, as in the form for many rows
constexpr int PX_POLY = 2;                   // of eight pairs of exponentials, those on the multiply-add units
constexpr int PX_STRIDE = 4 + TQ_D;          // floats of a state: M, L, -, -, o
constexpr int PX_TOP = 8;                    // a page's largest key on the grid is lifted to 2^8 .. 2^9
constexpr int PX_LIST = 3;                   // entries of a page's list that a thread holds

template <bool SPLIT>
struct PxShape {
  static constexpr int HALVES = SPLIT ? 1 : 2, ROWS = 128 * HALVES;
  static constexpr int PARTS = SPLIT ? 2 : 1;      // images of keys, and of values
  static constexpr int STAGES = SPLIT ? 2 : 3;
};
template <bool SPLIT, int VB>
struct PxShared {
  using Sh = PxShape<SPLIT>;
  static constexpr int ENTRY_K = 128, ENTRY_V = VB == 4 ? 64 : 128;  // bytes of a table's entry, copies and all
  alignas(128) uint8_t q[Sh::HALVES][PX_QIMAGE];
  alignas(128) uint8_t kv[Sh::STAGES][2 * Sh::PARTS][PX_IMAGE];
  alignas(128) uint8_t lut_k[256 * ENTRY_K], lut_v[(VB == 4 ? 256 : 64) * ENTRY_V];
  alignas(16) float scale[2][TQ_D], mean[2][TQ_D], center[TQ_D];  // of a page, lifted
  float2 of_tile[Sh::STAGES];                // the values' exponent, the keys' factor
  float part_top[2][4][PX_T], top[2][8];
  unsigned long long k_full[Sh::STAGES], v_full[Sh::STAGES], empty[Sh::STAGES], q_ready[2], s_full[2], s_read[2], p_full[2],
      o_done[2], drained[2];
  uint32_t tmem;
};

struct PrefixArgs {
  int32_t* left;   // [head]
  float* slots;    // [head][rows][ns][PX_STRIDE]
  int ns_cold, ns_hot, row_tiles;
};

TQ_DEV uint64_t px_lds64(uint32_t at) {
  uint64_t v;
  asm("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(at));
  return v;
}
TQ_DEV uint32_t px_lds32(uint32_t at) {
  uint32_t v;
  asm("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
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
  const int groups = Sh::HALVES == 2 && a.rows - row0 > 128 ? 2 : 1;  // halves of the rows that there are
  const uint8_t* const pages = a.pages + page_offset(g, a.layer, a.seq_begin, head, 0);

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(enc_smem(&sh.k_full[i]), PX_MAKERS / 32);
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
  // ---- tables: an entry's copies side by side, so that the lanes of a look-up meet different banks
  if (!hot) {
    for (int e = tid; e < 256 * 8; e += PX_THREADS) {  // two copies at a time
      const int b = e >> 3;
      const float x = a.tables->grid[b & 15], y = a.tables->grid[b >> 4];
      *(float4*)(sh.lut_k + e * 16) = make_float4(x, y, x, y);
    }
    constexpr int NV = VB == 4 ? 256 : 64, PER = Shared::ENTRY_V / 16;
    for (int e = tid; e < NV * PER; e += PX_THREADS) {
      const int b = e / PER;
      const float x = a.tables->centroids[b & ((1 << VB) - 1)], y = a.tables->centroids[b >> VB];
      if (SPLIT) {
        *(float4*)(sh.lut_v + e * 16) = make_float4(x, y, x, y);
      } else {
        const uint32_t h = ti_pair(x, y);
        *(uint4*)(sh.lut_v + e * 16) = make_uint4(h, h, h, h);
      }
    }
  }
  if (tid < TQ_D) sh.center[tid] = sq.cold > 0 ? ti_center(g, pages, tid) : 0.0f;
  ti_fence_before();
  __syncthreads();
  ti_fence_after();
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

  if (warp >= PX_SOFTMAX / 32 + 2) {
    // ---- the makers of the operands
    const int pt = tid - PX_SOFTMAX - 64, pw = pt >> 5;
    const int token = pt & (PX_T - 1), quarter = pt / PX_T;  // keys: 32 channels of a token
    const int held = blockIdx.x == 0 ? a.withhold : -1;      // test hook: a tile whose keys are never handed over
    bool odd = false;
    auto hand_over = [&](unsigned long long* bar) {
      px_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(enc_smem(bar));
    };
    auto put_key = [&](uint8_t* to, int chunk, const float (&x)[8]) {
      const uint4 hi = {ti_pair(x[0], x[1]), ti_pair(x[2], x[3]), ti_pair(x[4], x[5]), ti_pair(x[6], x[7])};
      *(uint4*)(to + chunk * PX_KLBO + token * 16) = hi;
      if (SPLIT)
        *(uint4*)(to + PX_IMAGE + chunk * PX_KLBO + token * 16) =
            make_uint4(ti_rest(x[0], x[1], hi.x), ti_rest(x[2], x[3], hi.y), ti_rest(x[4], x[5], hi.z), ti_rest(x[6], x[7], hi.w));
    };
    if (!hot) {
      const size_t uix = unit_index(g, a.layer, a.seq_begin, head);
      const uint32_t* const dec = a.pool_dec + uix * (size_t)g.pool_entries;
      const uint16_t* const val = a.pool_val + uix * (size_t)g.pool_entries;
      const PageMeta* const metas = a.page_meta + uix * g.max_blocks;
      const bool listed = g.outlier_k > 0;
      const float gridmost = g.key_mode == TQ_KEYS_UNIFORM ? 15.0f : 1.0f;
      // two warps expand the records of a group of 16 tokens; a lane: pairs 16 half .. + 15 of a record
      const int grp = pw >> 1, half = pw & 1, r = lane >> 2, c = lane & 3;
      uint4 codes;
      uint32_t rec[4];
      float2 norm2[2];
      float2 norm_of;  // of tokens 2 lane, 2 lane + 1 of the strip
      PageMeta meta = {0, 0};
      auto fetch = [&](int j) {  // strip j's, on their way
        const uint8_t* page = pages + (size_t)(j >> 2) * g.page_bytes;
        const int ts = (j & 3) * PX_T;
        codes = *(const uint4*)(page + (ts + token) * (TQ_D / 2) + 16 * quarter);
        const uint8_t* from = page + g.v_off + (size_t)((ts >> 4) + grp) * VGB;
        if (VB == 4) {
          const uint4 x = *(const uint4*)(from + half * 512 + lane * 16);
          rec[0] = x.x, rec[1] = x.y, rec[2] = x.z, rec[3] = x.w;
        } else {  // the record's 24 bytes; these pairs are words 3 half .. + 2
          const uint2 r0 = *(const uint2*)(from + (half ? 256 : 0) + lane * 8), r1 = *(const uint2*)(from + (half ? 512 : 256) + lane * 8);
          rec[0] = half ? r0.y : r0.x, rec[1] = half ? r1.x : r0.y, rec[2] = half ? r1.y : r1.x, rec[3] = 0u;
        }
        const float* norms = (const float*)(page + g.norm_off) + ts;
        norm2[0] = *(const float2*)(norms + 16 * grp + 2 * c), norm2[1] = *(const float2*)(norms + 16 * grp + 8 + 2 * c);
        norm_of = *(const float2*)(norms + 2 * lane);
      };
      float k_up = 1.0f, k_factor = 1.0f;
      uint32_t of_list[PX_LIST];
      uint16_t of_val[PX_LIST];
      if (listed) meta = metas[k_lo >> 2];
      fetch(k_lo);
      int turn = 0;  // of the page's place in shared memory
#pragma unroll 1
      for (int k = 0; k < n; ++k) {
        const int j = k_lo + k, stage = k % STAGES;
        const uint8_t* const page = pages + (size_t)(j >> 2) * g.page_bytes;
        if (k == 0 || (j & 3) == 0) {
          // ---- a page: its scales and zero-points, its list
          turn ^= 1;
          const float4 s4 = *(const float4*)(page + g.scale_off + lane * 16), m4 = *(const float4*)(page + g.mean_off + lane * 16);
          if (listed) {
            if (k > 0) meta = metas[j >> 2];
#pragma unroll
            for (int i = 0; i < PX_LIST; ++i) {
              const uint32_t e = pt + PX_MAKERS * i;
              of_list[i] = 0xffffffffu, of_val[i] = 0;
              if (e < meta.cnt) of_list[i] = dec[meta.off + e], of_val[i] = val[meta.off + e];
            }
          }
          const float4 z4 = *(const float4*)&sh.center[4 * lane];
          const float s[4] = {s4.x, s4.y, s4.z, s4.w}, m[4] = {m4.x - z4.x, m4.y - z4.y, m4.z - z4.z, m4.w - z4.w};
          float most = 0.0f, least = INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = fmaf(fabsf(s[i]), gridmost, fabsf(m[i]));
            odd |= !(x < TI_KEY_MOST);
            most = fmaxf(most, x);
            if (x > 0.0f) least = fminf(least, x);
          }
          most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
          odd |= least < most * TI_LEAST;
          float exponent;
          k_up = ti_lift(most, PX_TOP, exponent, 97);
          k_factor = exp2f(exponent);
          if (pw == 0) {
            *(float4*)&sh.scale[turn][4 * lane] = make_float4(s[0] * k_up, s[1] * k_up, s[2] * k_up, s[3] * k_up);
            *(float4*)&sh.mean[turn][4 * lane] = make_float4(m[0] * k_up, m[1] * k_up, m[2] * k_up, m[3] * k_up);
          }
          px_makers();
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
        {  // ---- keys
          const uint32_t lut = enc_smem(sh.lut_k) + (lane & 15) * 8;
          const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
          const uint32_t of_scale = enc_smem(&sh.scale[turn][32 * quarter]), of_mean = enc_smem(&sh.mean[turn][32 * quarter]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint64_t s[4], m[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              asm("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(s[2 * e]), "=l"(s[2 * e + 1]) : "r"(of_scale + 32 * i + 16 * e));
              asm("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(m[2 * e]), "=l"(m[2 * e + 1]) : "r"(of_mean + 32 * i + 16 * e));
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t off = (e == 0 ? w[i] << 7 : w[i] >> (8 * e - 7)) & 0x7f80u;
              const float2 f = ti_floats(ti_fma2(px_lds64(lut + off), s[e], m[e]));
              x[2 * e] = f.x, x[2 * e + 1] = f.y;
            }
            put_key(ki, 4 * quarter + i, x);
          }
        }
        uint32_t vw[4] = {rec[0], rec[1], rec[2], rec[3]};
        const float2 nv[2] = {norm2[0], norm2[1]};
        if (k + 1 < n) fetch(j + 1);
        if (listed) {
          px_makers();  // (the grid's part is there)
          auto put = [&](uint32_t e, uint16_t v) {
            const int t = (int)(e >> 24), ch = (int)(e >> 16) & 127;
            if (t >> 6 != (j & 3)) return;
            const float x = (__half2float(__ushort_as_half(v)) - sh.center[ch]) * k_up;
            odd |= !(fabsf(x) < 32768.0f);
            const __half hi = __float2half_rn(x);
            uint8_t* to = ki + (ch >> 3) * PX_KLBO + (t & (PX_T - 1)) * 16 + (ch & 7) * 2;
            *(__half*)to = hi;
            if (SPLIT) *(__half*)(to + PX_IMAGE) = __float2half_rn(x - __half2float(hi));
          };
#pragma unroll
          for (int i = 0; i < PX_LIST; ++i)
            if (pt + PX_MAKERS * i < meta.cnt) put(of_list[i], of_val[i]);
          for (uint32_t e = pt + PX_MAKERS * PX_LIST; e < meta.cnt; e += PX_MAKERS) put(dec[meta.off + e], val[meta.off + e]);
        }
        if (k != held) hand_over(&sh.k_full[stage]);
        {  // ---- values
          const uint32_t lut = enc_smem(sh.lut_v) + (lane % (SPLIT ? Shared::ENTRY_V / 8 : Shared::ENTRY_V / 4)) * (SPLIT ? 8 : 4);
          uint32_t n2[2];
          uint64_t f2[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            n2[h] = ti_pair(nv[h].x * v_up, nv[h].y * v_up);
            f2[h] = ti_f2(nv[h].x * v_up, nv[h].y * v_up);
          }
#pragma unroll
          for (int p = 0; p < 16; ++p) {
            const int h = p & 1, d = r + 8 * (8 * half + (p >> 1));
            uint32_t off;
            if (VB == 4) off = ((p & 3) == 0 ? vw[p >> 2] << 6 : vw[p >> 2] >> (8 * (p & 3) - 6)) & 0x3fc0u;
            else off = (__funnelshift_r(vw[6 * p >> 5], vw[min((6 * p >> 5) + 1, 3)], (6 * p) & 31) & 63u) * Shared::ENTRY_V;
            uint8_t* const to = vi + (2 * grp + h) * PX_LBO + d * 16 + 4 * c;
            if (SPLIT) {
              const float2 f = ti_floats(ti_fma2(px_lds64(lut + off), f2[h], 0ull));
              const uint32_t hi = ti_pair(f.x, f.y);
              *(uint32_t*)to = hi;
              *(uint32_t*)(to + PX_IMAGE) = ti_rest(f.x, f.y, hi);
            } else {
              const uint32_t y = px_lds32(lut + off);
              const __half2 v = __hmul2(*(const __half2*)&y, *(const __half2*)&n2[h]);
              *(uint32_t*)to = *(const uint32_t*)&v;
            }
          }
        }
        hand_over(&sh.v_full[stage]);
      }
    } else {
      // ---- the uncompressed window: a thread has a quarter of a token's channels
      const size_t ring = hot_offset_elems(g, a.layer, a.seq_begin, head);
      // the largest of a tile; whether a token lies far below it, or something is no number
      auto largest = [&](float most, int which) {
        sh.part_top[which][quarter][token] = most;
        const float mine = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        if (lane == 0) sh.top[which][pw] = mine;
        px_makers();
        float top = 0.0f, of_token = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sh.top[which][i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) of_token = fmaxf(of_token, sh.part_top[which][i][token]);
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
        const size_t at = ring + (size_t)(t % g.hot_cap) * TQ_D + 32 * quarter;
        float x[4][8], most = 0.0f, exponent, k_exponent;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (t < sq.n) ti_ld8(a.hot_k, at + 8 * i, g.kv_dtype, x[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[i][e] = t < sq.n ? x[i][e] - sh.center[32 * quarter + 8 * i + e] : 0.0f;
            odd |= !(fabsf(x[i][e]) < TI_KEY_MOST);
            most = fmaxf(most, fabsf(x[i][e]));
          }
        }
        const float k_up = ti_lift(largest(most, 0), 14, k_exponent, 97);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] *= k_up;
          put_key(ki, 4 * quarter + i, x[i]);
        }
        most = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (t < sq.n) ti_ld8(a.hot_v, at + 8 * i, g.kv_dtype, x[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[i][e] = t < sq.n ? x[i][e] : 0.0f;
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
    // ---- products of half x: the whole warp runs this, one thread issues
    const int x = warp - PX_SOFTMAX / 32, n_u = __shfl_sync(0xffffffffu, x < groups ? n : 0, 0);
    if (n_u > 0) {
      constexpr uint32_t s_desc = (1u << 4) | ((uint32_t)(PX_T >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t o_desc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint64_t KSTEP = 2 * PX_KLBO >> 4, STEP = 2 * PX_LBO >> 4;  // 16 deep
      const uint64_t q = umma_desc_k_major(enc_smem(sh.q[0]), PX_LBO, PX_SBO) + (uint64_t)(x * (PX_QIMAGE >> 4));
      const uint64_t k0 = umma_desc_k_major(enc_smem(sh.kv[0][0]), PX_KLBO, PX_SBO);
      const uint64_t v0 = umma_desc_k_major(enc_smem(sh.kv[0][PARTS]), PX_LBO, PX_SBO);
      const uint32_t ds = tmem + PX_HALF * x, dp = tmem + PX_P + PX_HALF * x, d_o = tmem + PX_O + 128 * x;
      auto image = [&](int k, int part) { return (uint64_t)((uint32_t)(k % STAGES) * (2 * PARTS * PX_IMAGE >> 4) + part * (PX_IMAGE >> 4)); };
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
  } else if (warp < 4 * groups) {
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
    float factor, shift;
    {
      uint4 raw[16];
      const bool there = row < a.rows;
      const uint16_t* q = (const uint16_t*)a.q + ((int64_t)(row / G) * a.q_tok + (int64_t)(head * G + row % G) * a.q_head);
#pragma unroll
      for (int i = 0; i < 16; ++i) raw[i] = there ? *(const uint4*)(q + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
      auto pair = [&](uint32_t w) -> float2 {
        if (SPLIT) return __half22float2(*(const __half2*)&w);
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      };
      float top = 0.0f, part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair(w[j]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          // what the keys' common vector takes off this row's scores
          part[j] = fmaf(f.x, sh.center[8 * i + 2 * j], fmaf(f.y, sh.center[8 * i + 2 * j + 1], part[j]));
        }
      }
      shift = tq_scaled<true>((part[0] + part[1]) + (part[2] + part[3]));
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
        *(uint4*)(sh.q[x] + i * PX_LBO + r * 16) = make_uint4(h[0], h[1], h[2], h[3]);
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
      uint32_t h[PX_T / 2];
#pragma unroll
      for (int j = 0; j < PX_T / 2; ++j) {
        const uint64_t y = ti_fma2(ti_u2(v[2 * j], v[2 * j + 1]), factor2, off2);
        const float2 z = j % 8 < PX_POLY ? ti_exp2_poly(y) : ti_exp2_unit(y);
        sum[j & 1] = ti_add2(sum[j & 1], ti_f2(z.x, z.y));
        h[j] = ti_pair(z.x, z.y);
      }
      ti_st32(tp, h);
      if (groups == 2 && (x == 0 || k + 1 < n)) asm volatile("bar.arrive %0, 256;" ::"r"(2 - x) : "memory");
      ti_wait_st();
      ti_fence_before();
      mbar_arrive(enc_smem(&sh.p_full[x]));
      const float2 s2 = ti_floats(ti_add2(sum[0], sum[1]));
      l = fmaf(s2.x + s2.y, exp2f(-e), l * down);
    }
    settled(&sh.o_done[x], (n - 1) & 1);
    float* const slot = slot_of(min(row, a.rows - 1));
    if (row < a.rows) *(float2*)slot = make_float2(m - TI_LIFT + shift, l);
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      uint32_t o[16];
      ti_ld16(to + 16 * i, o);
      ti_wait_ld();
      if (row < a.rows)
#pragma unroll
        for (int j = 0; j < 16; j += 4) *(uint4*)(slot + 4 + 16 * i + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
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

// Splits of the blocks and of the window: as many as bring the rounds of CTAs nearest to even, with six tiles' time for what a
// CTA does besides.
void tq_attend_shared_plan(const AttendArgs& a, int tokens, int* ns_cold, int* ns_hot) {
  const tq_geom& g = a.g;
  const int64_t cold = (int64_t)n_cold_blocks(tokens, g.hot_window, PX_S) * (PX_S / PX_T);
  const int64_t hot = (std::min(tokens, g.hot_window) + PX_T - 1) / PX_T;
  const int64_t units = (int64_t)g.n_kv_heads * ((a.rows + rows_of_cta(a) - 1) / rows_of_cta(a));
  int64_t best = INT64_MAX;
  *ns_cold = *ns_hot = 1;
  for (int64_t each = 1; each <= std::max(cold, hot); ++each) {  // tiles of a CTA
    const int64_t nc = std::max<int64_t>((cold + each - 1) / each, 1), nh = std::max<int64_t>((hot + each - 1) / each, 1);
    if (nc + nh > 256) continue;
    const int64_t time = (units * (nc + nh) + a.sm_count - 1) / a.sm_count * (each + 6);
    if (time < best) best = time, *ns_cold = (int)nc, *ns_hot = (int)nh;
  }
}

size_t tq_attend_shared_bytes(const AttendArgs& a) { return layout(a).total; }

int tq_launch_attend_shared(const AttendArgs& base, void* workspace, cudaStream_t st) {
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
  const int64_t rows = (int64_t)a.g.n_kv_heads * a.rows;
  attend_shared_merge_kernel<<<(int)std::min<int64_t>((rows + 3) / 4, 2 * a.sm_count), PM_THREADS, 0, st>>>(a, pa);
  TQ_CUDA(cudaGetLastError());
  return TQ_OK;
}

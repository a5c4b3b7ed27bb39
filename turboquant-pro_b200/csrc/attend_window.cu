// The last kernel of a call with a shared beginning or on listed blocks: attention of a sequence's query rows on its uncompressed
// window (all that most sequences have behind a long beginning, and what all tokens share of calls whose blocks differ from
// token to token), and the merge with the states of the beginning and of the sequence's own blocks, if it has any.
// 16-bit queries and a window of their type.
//
// A CTA has 8 or 16 rows of a (sequence, KV head); its four warps take tiles of 32 tokens in turn and work alone: keys and values
// come with cp.async, the next tile's keys while this one's values are summed and the other way round; S = Q K^T and O += P V on
// mma.sync (m16n8k16) with the rows as they are, so that products are exact; probabilities are pairs hi + lo (float16: of 2^14
// times their size; behind a first token that has no value and all but 1e-3 of the weight, results were 6.9e-4 off without that).
// The four states are merged in shared memory, with those of memory; what is in code space is rotated by Pi.
//   An infinity or a NaN among the values spoils sums of rows that do not see it (0 * inf), and those of its low parts: a warp whose
// sums are not all finite does its tiles again, term by term.
//   What bounds it: latencies of one thing after the other.  64 sequences with windows of up to 500 tokens, 8 KV heads of 8 rows, ten
// states a row: 41 us, two waves of CTAs of 20 us each: lengths and queries 5900 cycles, window 11400, merge 10000, rotation 7800.
// 32 x 8 heads of 4 rows 22 us, 4 x 8 12.5.  (The form for few rows, whose kernel is made for blocks, took 27 us for the windows
// of 4 sequences and 45 for those of 64, 8 KV heads, and its merge 10 and 28.)  Rotating four rows at a time cost 4 us more of the 41.
#include <algorithm>

#include "attend.cuh"

namespace {

constexpr int AW_THREADS = 128, AW_WARPS = 4, AW_ROWS = 16, AW_T = 32;
constexpr int AW_PITCH = TQ_D * 2 + 16;  // bytes of a row in shared memory
constexpr int AW_TILE = AW_T * AW_PITCH;
struct AwShared {
  alignas(16) uint8_t kv[AW_WARPS][2][AW_TILE];  // keys; values.  Afterwards a warp's sums
  float m[AW_WARPS][AW_ROWS], l[AW_WARPS][AW_ROWS], of_l[AW_ROWS];
};
static_assert(AW_ROWS * (TQ_D + 4) * 4 <= AW_TILE, "a warp's sums in its keys' place, the merged rows in the values'");

TQ_DEV uint32_t aw_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <bool BF>
TQ_DEV void aw_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
TQ_DEV uint64_t aw_f2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
TQ_DEV uint64_t aw_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
template <bool TRANS>
TQ_DEV void aw_ldm(uint32_t (&r)[4], uint32_t at) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool BF>
TQ_DEV void aw_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    hi = *(const uint32_t*)&h;
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
    lo = *(const uint32_t*)&r;
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    hi = *(const uint32_t*)&h;
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    lo = *(const uint32_t*)&r;
  }
}

template <bool BF>
__global__ void __launch_bounds__(AW_THREADS, 3) attend_window_kernel(AttendArgs a, int row_tiles, int tile, int blocks_tile) {
  constexpr float LIFT = BF ? 0.0f : 14.0f;  // float16: probabilities are 2^14 at most, and small ones keep their digits
  extern __shared__ __align__(16) uint8_t aw_shared[];
  AwShared& sh = *(AwShared*)aw_shared;
  const tq_geom& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int rt = blockIdx.x % row_tiles, unit = blockIdx.x / row_tiles, H = g.n_kv_heads, G = g.group;
  const int s = unit / H, head = unit - s * H, row0 = rt * tile, rows = min(tile, a.rows - row0);
  const AttendSeq sq = attend_seq(a, s);
  const size_t ring = hot_offset_elems(g, a.layer, a.seq_begin + s, head);
  // the latest position of the tile's rows: tokens behind it count for nothing
  const int last = min(row0 + rows, sq.q_n * G) - 1;
  const int end = last >= row0 ? min(sq.n, sq.first + last / G + 1) : sq.cold;
  const int tiles = max(end - sq.cold + AW_T - 1, 0) / AW_T;

  auto fetch = [&](int t, int which) {  // a tile's keys (0) or values (1)
    const uint32_t to = aw_smem(sh.kv[warp][which]) + (lane >> 4) * AW_PITCH + (lane & 15) * 16;
    const uint16_t* const from = (const uint16_t*)(which == 0 ? a.hot_k : a.hot_v) + ring + (lane & 15) * 8;
    const int first = sq.cold + t * AW_T + (lane >> 4);
    int slot = first % g.hot_cap;
#pragma unroll 4
    for (int i = 0; i < AW_T; i += 2) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * AW_PITCH), "l"(from + slot * TQ_D),
                   "r"(first + i < end ? 16 : 0)
                   : "memory");
      slot = slot + 2 >= g.hot_cap ? slot + 2 - g.hot_cap : slot + 2;
    }
  };
  auto commit = [&]() { asm volatile("cp.async.commit_group;" ::: "memory"); };
  if (warp < tiles) fetch(warp, 0);
  commit();
  if (warp < tiles) fetch(warp, 1);
  commit();

  // rows r and r + 8: queries (the A operand), positions
  uint32_t q[8][4];
  int pos[2];
  const uint16_t* q_at[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = row0 + r + 8 * x;
    const bool there = r + 8 * x < rows;
    pos[x] = there ? attend_position(a, sq, row) : -1;
    q_at[x] = (const uint16_t*)a.q;
    if (there) q_at[x] += (int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok + (int64_t)(head * G + row % G) * a.q_head;
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int y = 0; y < 2; ++y) q[k][x + 2 * y] = pos[x] >= 0 ? *(const uint32_t*)(q_at[x] + 16 * k + 8 * y + 2 * c) : 0u;
  }
  float acc[16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
  const uint32_t k_at = aw_smem(sh.kv[warp][0]) + ((lane & 7) + (lane >> 4) * 8) * AW_PITCH + (lane >> 3 & 1) * 16;
  const uint32_t v_at = aw_smem(sh.kv[warp][1]) + (lane & 15) * AW_PITCH + (lane >> 4) * 16;
#pragma unroll 1
  for (int t = warp; t < tiles; t += AW_WARPS) {
    const int j0 = sq.cold + t * AW_T;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    float sc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[i][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t b[4];
        aw_ldm<false>(b, k_at + 8 * i * AW_PITCH + 32 * k);
        aw_mma<BF>(sc[i], q[k], b[0], b[1]);
        aw_mma<BF>(sc[i + 1], q[k], b[2], b[3]);
      }
    __syncwarp();  // (the keys have been read)
    if (t + AW_WARPS < tiles) fetch(t + AW_WARPS, 0);
    commit();
    // tokens 8 i + 2 c + y of the tile; scores in units of log 2
    float down[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float& v = sc[i][2 * x + y];
          v = j0 + 8 * i + 2 * c + y <= pos[x] ? tq_scaled<true>(v) : -INFINITY;
          top = fmaxf(top, v);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[x]);
      const float by = top > -INFINITY ? top : 0.0f, low = by - LIFT;
      down[x] = tq_exp2(m[x] - by);
      m[x] = top;
      l[x] *= down[x];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float p = tq_exp2(sc[i][2 * x + y] - low);
          sc[i][2 * x + y] = p;
          l[x] += p;
        }
    }
    uint32_t ph[2][4], pl[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int x = 0; x < 2; ++x) aw_parts<BF>(sc[2 * k + y][2 * x], sc[2 * k + y][2 * x + 1], ph[k][x + 2 * y], pl[k][x + 2 * y]);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i][0] *= down[0], acc[i][1] *= down[0], acc[i][2] *= down[1], acc[i][3] *= down[1];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        uint32_t b[4];
        aw_ldm<true>(b, v_at + 16 * k * AW_PITCH + 16 * i);
        aw_mma<BF>(acc[i], pl[k], b[0], b[1]);
        aw_mma<BF>(acc[i], ph[k], b[0], b[1]);
        aw_mma<BF>(acc[i + 1], pl[k], b[2], b[3]);
        aw_mma<BF>(acc[i + 1], ph[k], b[2], b[3]);
      }
    __syncwarp();  // (the values have been read)
    if (t + AW_WARPS < tiles) fetch(t + AW_WARPS, 1);
    commit();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
  // ---- a warp's state to shared memory
  float* const sums = (float*)sh.kv[warp][0];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= pos[e >> 1] >= 0 && !(fabsf(acc[i][e]) < INFINITY);
  if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
    for (int k = 0; k < rows; ++k) {  // a row; a lane has channels lane, lane + 32 ..
      const int row = row0 + k, p = attend_position(a, sq, row);
      const int64_t at = (int64_t)s * a.q_seq + (int64_t)(row / G) * a.q_tok + (int64_t)(head * G + row % G) * a.q_head;
      float top = -INFINITY, sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
      for (int t = warp; t < tiles; t += AW_WARPS)
#pragma unroll 1
        for (int j = sq.cold + t * AW_T; j < min(sq.cold + (t + 1) * AW_T, min(end, p + 1)); ++j) {
          const size_t from = ring + (size_t)(j % g.hot_cap) * TQ_D;
          float dot = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dot = fmaf(attend_ld(a.q, (size_t)(at + lane + 32 * i), a.q_dtype),
                       attend_ld(a.hot_k, from + lane + 32 * i, g.kv_dtype), dot);
#pragma unroll
          for (int d = 16; d >= 1; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
          dot = tq_scaled<true>(dot);
          const float now = fmaxf(top, dot), by = now > -INFINITY ? now : 0.0f, f = tq_exp2(top - by), e = tq_exp2(dot - by);
          top = now;
          sum = fmaf(sum, f, e);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = fmaf(e, attend_ld(a.hot_v, from + lane + 32 * i, g.kv_dtype), o[i] * f);
        }
      __syncwarp();
      if (lane == 0) sh.m[warp][k] = top, sh.l[warp][k] = sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[k * (TQ_D + 4) + lane + 32 * i] = o[i];
    }
  } else {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (c == 0) sh.m[warp][r + 8 * x] = m[x] - LIFT, sh.l[warp][r + 8 * x] = l[x];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        *(float2*)&sums[(r + 8 * x) * (TQ_D + 4) + 8 * i + 2 * c] = make_float2(acc[i][2 * x], acc[i][2 * x + 1]);
    }
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- the merge: a warp a row, a lane four channels, ten states of memory on their way at once
  float(*const xs)[TQ_D] = (float(*)[TQ_D])sh.kv[0][1];  // rows in code space, in the original basis
  float(*const hs)[TQ_D] = (float(*)[TQ_D])sh.kv[1][1];
  const bool behind = a.shared.slots != nullptr, general = behind && a.shared.left[head] != 0;  // (general: its two states)
  const int np = general ? 2 : behind ? a.shared.ns : 0, np_cold = general ? 1 : a.shared.ns_cold;
  const int stride = general ? TQ_PART_STRIDE : TQ_SLOT_STRIDE, skip = general ? 2 : 4;
  const size_t of_unit = (size_t)head * a.before_rows + (size_t)s * a.rows;
  const float* const prefix = (general ? a.shared.general : a.shared.slots) + of_unit * np * stride;
#pragma unroll 1
  for (int k = warp; k < rows; k += AW_WARPS) {
    const int row = row0 + k;
    float M = fmaxf(fmaxf(sh.m[0][k], sh.m[1][k]), fmaxf(sh.m[2][k], sh.m[3][k])), L = 0.0f;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, hot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < AW_WARPS; ++w) {
      const float f = attend_weight(sh.m[w][k], sh.l[w][k], M > -INFINITY ? M : 0.0f);
      if (f == 0.0f) continue;
      const float4 v = *(const float4*)&((const float*)sh.kv[w][0])[k * (TQ_D + 4) + 4 * lane];
      L = fmaf(sh.l[w][k], f, L);
      hot[0] = fmaf(v.x, f, hot[0]), hot[1] = fmaf(v.y, f, hot[1]), hot[2] = fmaf(v.z, f, hot[2]), hot[3] = fmaf(v.w, f, hot[3]);
    }
    // those of the beginning, then those of the sequence's own blocks; the first nc of them in code space.  (One loop for both:
    // code that a warp goes through once is waited for.)
#pragma unroll 1
    for (int own = 0; own < 2; ++own) {
      const float* base = prefix + (size_t)row * np * stride;
      int n = attend_position(a, sq, row) >= 0 ? np : 0, step = stride, head_of = skip, nc = np_cold;
      if (own == 1) {
        if (a.ns_cold == 0) break;
        const ArPlan* plan = (const ArPlan*)a.plan;
        const int4 seq = plan->seq[s];
        const int of_row = a.listed ? row / G * ((G + blocks_tile - 1) / blocks_tile) + row % G / blocks_tile : row / blocks_tile;
        n = 0;
        if (seq.x > 0 && of_row < seq.z) {
          const int cost = ar_cost(a.q_dtype != TQ_BF16);
          const int64_t begin = plan->cum[s] + (int64_t)(head * seq.z + of_row) * cost * seq.x;
          n = (int)(ar_div(begin + cost * (seq.x - 1), plan->share) - ar_div(begin, plan->share)) + 1;
        }
        base = attend_partial(a, unit, row, 0), step = TQ_PART_STRIDE, head_of = 2, nc = n;
      }
      constexpr int BATCH = 10;
#pragma unroll 1
      for (int i0 = 0; i0 < n; i0 += BATCH) {
        float2 ml[BATCH], u[BATCH], v[BATCH];
        float top = M;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          ml[i] = make_float2(-INFINITY, 0.0f), u[i] = v[i] = make_float2(0.0f, 0.0f);
          if (i0 + i < n) {
            const float* p = base + (size_t)(i0 + i) * step;
            ml[i] = *(const float2*)p;
            u[i] = *(const float2*)(p + head_of + 4 * lane), v[i] = *(const float2*)(p + head_of + 4 * lane + 2);
          }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) top = fmaxf(top, ml[i].x);
        const float by = top > -INFINITY ? top : 0.0f, down = M > -INFINITY ? tq_exp2(M - by) : 1.0f;
        M = top;
        L *= down;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= down, hot[e] *= down;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const float f = attend_weight(ml[i].x, ml[i].y, by);
          if (f == 0.0f) continue;
          L = fmaf(ml[i].y, f, L);
          const float y[4] = {u[i].x, u[i].y, v[i].x, v[i].y};
          const float fx = i0 + i < nc ? f : 0.0f, fh = i0 + i < nc ? 0.0f : f;
          if (fx != 0.0f)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], fx, x[e]);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) hot[e] = fmaf(y[e], fh, hot[e]);
        }
      }
    }
    *(float4*)&xs[k][4 * lane] = make_float4(x[0], x[1], x[2], x[3]);
    *(float4*)&hs[k][4 * lane] = make_float4(hot[0], hot[1], hot[2], hot[3]);
    if (lane == 0) sh.of_l[k] = L;
  }
  __syncthreads();
  // ---- the rotation: a thread a channel, eight rows at a time
  const int e = tid;
#pragma unroll 1
  for (int k0 = 0; k0 < rows; k0 += 8) {
    uint64_t y[8];  // (even and odd channels)
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = 0ull;
#pragma unroll 1
    for (int d = 0; d < TQ_D; d += 32) {
      uint64_t pi[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) pi[i] = aw_f2(a.tables->pi[(d + 2 * i) * TQ_D + e], a.tables->pi[(d + 2 * i + 1) * TQ_D + e]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k == 4 && rows - k0 <= 4) break;
        uint64_t z = 0ull;  // (32 at a time: a sum over all 128 in a row would be rounded at its full size 128 times)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          uint64_t u, v;
          asm("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(u), "=l"(v) : "r"(aw_smem(&xs[k0 + k][d + 2 * i])) : "memory");
          z = aw_fma2(u, pi[i], z);
          z = aw_fma2(v, pi[i + 1], z);
        }
        y[k] = aw_fma2(z, aw_f2(1.0f, 1.0f), y[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)  // (rows that there are not: of no use, and in place)
      hs[k0 + k][e] += __uint_as_float((uint32_t)y[k]) + __uint_as_float((uint32_t)(y[k] >> 32));
  }
  int i = row0 / G, gh = row0 - i * G;  // query token and head of the group
  size_t to = (((size_t)s * a.n_tokens + i) * g.n_q_heads + head * G + gh) * TQ_D + e;
#pragma unroll 1
  for (int k = 0; k < rows; ++k) {
    const float L = sh.of_l[k], v = L == 0.0f ? 0.0f : hs[k][e] / L;
    if (BF) ((__nv_bfloat16*)a.out)[to] = __float2bfloat16_rn(v);
    else ((__half*)a.out)[to] = __float2half_rn(v);
    to += TQ_D;
    if (++gh == G) gh = 0, to += (size_t)(g.n_q_heads - G) * TQ_D;
  }
}

}  // namespace

int tq_launch_attend_window(const AttendArgs& a, int blocks_tile, cudaStream_t st) {
  // Tiles of 16 rows, the products' own size, or of 8 while all CTAs are resident at once, three an SM: the merge, rows by rows, then
  // takes half as long (11 x 4 heads of 21 rows: 34 us with 16).
  const int64_t units = (int64_t)a.seq_count * a.g.n_kv_heads;
  const int tile = units * ((a.rows + 7) / 8) <= 3 * a.sm_count ? 8 : AW_ROWS, row_tiles = (a.rows + tile - 1) / tile;
  const int64_t grid = (int64_t)a.seq_count * a.g.n_kv_heads * row_tiles;
  TQ_REQUIRE(grid <= INT_MAX, TQ_ERR_UNSUPPORTED, "too many (sequence, head, query row) tiles in a call");
  const bool bf = a.q_dtype == TQ_BF16;
  static bool done[2][64];
  const auto kernel = bf ? attend_window_kernel<true> : attend_window_kernel<false>;
  // The kernel reads lengths, queries and windows before it waits for the one that it starts under.  So that has to be one of this
  // call, whose first comes behind what is in the stream in full order.  Where there is none (lists, and no sequence with a block)
  // what it would start under is another call's: a ring writer, say, that has not written yet.
  const bool behind_own = a.ns_cold > 0 || a.shared.slots != nullptr;
  const int rc = attend_shared(kernel, sizeof(AwShared), a.device, done[bf]);
  if (rc != TQ_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(AW_THREADS);
  cfg.dynamicSmemBytes = sizeof(AwShared);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = behind_own ? 1 : 0;
  TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, row_tiles, tile, blocks_tile));
  return TQ_OK;
}

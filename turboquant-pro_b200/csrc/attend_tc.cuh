// Shared by the forms of attention whose products run on tcgen05 with the accumulators in tensor memory: instructions,
// powers of two that lift operands into half precision, exponentials.
#pragma once

#include "attend.cuh"
#include "encode.cuh"  // mbarrier, descriptors, commit

constexpr float TI_KEY_MOST = 0x1p20f, TI_LEAST = 0x1p-20f;  // largest key; least part of a tile's largest
constexpr float TI_LIFT = 7.0f, TI_GROW = 8.0f;  // probabilities reach 2^(7 + 8) at most
constexpr int TI_WAIT = 1 << 21;             // probes of a wait

// The vector that is taken off all keys of a (sequence, KV head): what its first block's channels are around.  (Uniform grids
// count from their zero-point on: their middle.)
TQ_DEV float ti_center(const tq_geom& g, const uint8_t* page, int d) {
  float c = ((const float*)(page + g.mean_off))[d];
  if (g.key_mode == TQ_KEYS_UNIFORM) c = fmaf(7.5f, ((const float*)(page + g.scale_off))[d], c);
  return isfinite(c) ? c : 0.0f;
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

// eight neighbouring elements of a window row
TQ_DEV void ti_ld8(const void* p, size_t at, int dt, float (&x)[8]) {
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
#define TI_W8(v, i) \
  "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
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


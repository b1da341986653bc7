// What the 16-bit kernels of linear layers share: loads from tensor memory and shared memory, activations, the epilogue's arithmetic.
// Everything is in an unnamed namespace: each translation unit gets its own copy.
#pragma once
#include "linear.cuh"
#include "tcgen05_common.cuh"

namespace {

__device__ __forceinline__ uint32_t bar(uint64_t* b) { return smem_u32(b); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_shared(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ------------------------------------------------------------------ activations, two numbers at a time

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger of two numbers; what is no number stays so.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// Normal distribution's function at v <= 0 as an exponential of a polynomial: log2 of it is a smooth curve near a parabola, fitted by
// least largest error (degree 7) from -6.5 on: within 9e-6 of the value, a fiftieth of half a step of 16-bit results at least.  Before
// that, where it is below 4e-11, the polynomial falls as the function does, to 0.  (The library's error function takes three times the
// instructions, of which this kernel has its fill.)
constexpr float GELU_END = -64.f;   // where it is 0, and so that infinity times it is none
__device__ __forceinline__ float2 normal_tail(float2 v) {
  float2 p = both(1.75778337e-06f);
  p = __ffma2_rn(p, v, both(5.99367486e-05f));
  p = __ffma2_rn(p, v, both(0.000916364603f));
  p = __ffma2_rn(p, v, both(0.00844739377f));
  p = __ffma2_rn(p, v, both(0.0538245253f));
  p = __ffma2_rn(p, v, both(-0.458615661f));
  p = __ffma2_rn(p, v, both(1.15118015f));
  p = __ffma2_rn(p, v, both(-1.00000381f));
  return make_float2(exp2_fast(p.x), exp2_fast(p.y));
}
// -|z|, the polynomial's end at least; what is no number stays so.
__device__ __forceinline__ float2 below_zero(float2 z) { return make_float2(max_nan(-fabsf(z.x), GELU_END), max_nan(-fabsf(z.y), GELU_END)); }
// -(Phi(v) + v phi(v)) / exp(-v^2 / 2) at v <= 0, the slope of GELU there: a polynomial of degree 7, fitted so that its largest error
// times the exponential is least (4e-6; the slope itself reaches 1.13).
__device__ __forceinline__ float2 slope_tail(float2 v) {
  float2 p = both(-0.000168556944f);
  p = __ffma2_rn(p, v, both(-0.00231906539f));
  p = __ffma2_rn(p, v, both(-0.0139235854f));
  p = __ffma2_rn(p, v, both(-0.0499400012f));
  p = __ffma2_rn(p, v, both(-0.12582691f));
  p = __ffma2_rn(p, v, both(-0.247959629f));
  p = __ffma2_rn(p, v, both(-0.797662377f));
  p = __ffma2_rn(p, v, both(-0.499996036f));
  return p;
}
__device__ __forceinline__ float2 logistic(float2 z) {
  const float2 e = __fmul2_rn(z, both(-1.4426950408889634f));
  const float2 d = __fadd2_rn(both(1.f), make_float2(exp2_fast(e.x), exp2_fast(e.y)));
  return make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
}

template <int ACT> __device__ __forceinline__ float2 activate(float2 z) {
  if (ACT == WCN_ACT_RELU) return make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f));
  if (ACT == WCN_ACT_SILU) return __fmul2_rn(z, logistic(z));
  if (ACT == WCN_ACT_GELU) {   // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const float2 v = below_zero(z);
    return __ffma2_rn(v, normal_tail(v), make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f)));
  }
  return z;
}
// dy act'(z)
template <int ACT> __device__ __forceinline__ float2 through(float2 dy, float2 z) {
  if (ACT == WCN_ACT_RELU) return make_float2(z.x > 0.f ? dy.x : 0.f, z.y > 0.f ? dy.y : 0.f);
  if (ACT == WCN_ACT_SILU) {
    const float2 p = logistic(z), q = __ffma2_rn(p, both(-1.f), both(1.f));
    return __fmul2_rn(dy, __fmul2_rn(p, __ffma2_rn(z, q, both(1.f))));
  }
  if (ACT == WCN_ACT_GELU) {
    const float2 v = below_zero(z);
    const float2 e = __fmul2_rn(__fmul2_rn(v, both(-0.72134752044448170f)), v);
    const float2 w = __ffma2_rn(make_float2(exp2_fast(e.x), exp2_fast(e.y)), slope_tail(v), both(0.5f));   // slope at |z| - 1/2
    return __fmul2_rn(dy, __fadd2_rn(make_float2(copysignf(w.x, z.x), copysignf(w.y, z.y)), both(0.5f)));
  }
  return dy;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float2 v) {
  if (BF16) {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16> __device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF16> __device__ __forceinline__ float number(uint16_t v) {
  return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// `keys`: in shared memory.  Sixteen numbers of one row: v = A B^T + bias on entry, the result's on exit; add: as many in 16 bits.
template <int ACT, bool GRAD, bool BF16, bool MORE>   // MORE: there may be dropout or a sum
__device__ __forceinline__ void finish(const wcn_linear_product& q, const PhiloxKeys* keys, float2 (&v)[8], const uint4 (&add)[2], int64_t row, int col) {
  const bool drop = MORE && q.drop.least != 0, sum = MORE && !GRAD && q.add;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint32_t a[4] = {add[b].x, add[b].y, add[b].z, add[b].w};
    float2 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = GRAD ? unpack2<BF16>(a[i]) : activate<ACT>(v[4 * b + i]);
    if (drop) drop_eight(q.drop, *keys, (uint32_t)col / 8 + b, (uint64_t)row, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * b + i] = GRAD ? through<ACT>(t[i], v[4 * b + i]) : sum ? __fadd2_rn(t[i], unpack2<BF16>(a[i])) : t[i];
  }
}

}  // namespace

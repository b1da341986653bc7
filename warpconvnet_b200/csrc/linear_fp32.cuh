// Activations of linear layers in fp32.  Everything is in an unnamed namespace: each translation unit gets its own copy.
#pragma once
#include "linear.cuh"

namespace {

__device__ __forceinline__ float reciprocal(float x) {   // within 2^-23 of it
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Normal distribution: the function at z, and exp(-z^2 / 2).  At u = -|z| the function is the exponential times a curve that has no steep
// places, a polynomial of degree 9 in 1 / (1 + 0.35 |u|) that was fitted by least largest error relative to it (3e-8; evaluated in fp32
// 3.3e-7, 0.8e-7 in the mean).  Before -14, where it is below the end of fp32, it is what it is there.  No branches: those of the
// library's function, eight numbers of a thread one after the other, took as long as three times the products.
struct Normal {
  float function, density, u;   // u: z, at most 14 from 0
};
__device__ __forceinline__ Normal normal(float z) {
  Normal n;
  const float u = fminf(fabsf(z), 14.f), h = u * u, t = reciprocal(fmaf(0.35f, u, 1.f));
  float e = expf(-0.5f * h);
  e = fmaf(e, -0.5f * fmaf(u, u, -h), e);   // (what the square was rounded by)
  float p = -0.0280455314f;
  p = fmaf(p, t, 0.138257608f);
  p = fmaf(p, t, -0.242944166f);
  p = fmaf(p, t, 0.143102035f);
  p = fmaf(p, t, -0.0105960881f);
  p = fmaf(p, t, 0.0992779881f);
  p = fmaf(p, t, 0.121809669f);
  p = fmaf(p, t, 0.139477521f);
  p = fmaf(p, t, 0.139662862f);
  p = fmaf(p, t, -1.88678132e-06f);
  p *= e;
  n.function = z > 0.f ? 1.f - p : p;
  n.density = e;
  n.u = z != z ? z : copysignf(u, z);
  return n;
}

template <int ACT> __device__ __forceinline__ float activate(float z) {
  if (ACT == WCN_ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if (ACT == WCN_ACT_SILU) return z * reciprocal(1.f + expf(-z));
  if (ACT == WCN_ACT_GELU) {
    const Normal n = normal(z);
    return (z < -14.f ? n.u : z) * n.function;
  }
  return z;
}
// dy act'(z)
template <int ACT> __device__ __forceinline__ float through(float dy, float z) {
  if (ACT == WCN_ACT_RELU) return z > 0.f ? dy : 0.f;
  if (ACT == WCN_ACT_SILU) {
    const float e = expf(-fabsf(z)), r = reciprocal(1.f + e), p = z > 0.f ? r : e * r, rest = z > 0.f ? e * r : r;   // (1 - p would be z 2^-24 off)
    return dy * (p * fmaf(z, rest, 1.f));
  }
  if (ACT == WCN_ACT_GELU) {
    const Normal n = normal(z);
    return dy * fmaf(n.u, 0.3989422804014327f * n.density, n.function);
  }
  return dy;
}

}  // namespace

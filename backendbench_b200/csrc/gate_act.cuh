// The activations of a gated projection pair, with their slopes (fp32).
//
//   silu       g s(g)                      s (1 + g (1 - s))               s(z) = 1 / (1 + e^-z)
//   gelu       g P(g), P the normal cdf    P(g) + g e^(-g^2 / 2) / sqrt(2 pi)
//   gelu_tanh  g s(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3): (1 + tanh z) / 2 is s(2 z)
//   relu       g for g > 0, else 0; NaN stays NaN
//   sigmoid    s(g)                        s (1 - s)
//
// s(z) is 1 / (1 + t) for z >= 0 and t / (1 + t) below, t = e^-|z|: a denominator of 1 to 2. (1 + e^-z overflows below -88.7, and the fast quotient
// gives 0 for denominators above 2^126, below -87.3, where s is 2^-127 and g s times a large u is not small.) Below -87.3 t is subnormal, and resolved to
// 2^-149; below -103.9 it is 0.
//
// `fast` goes with 16-bit results: its exponential is off by 2 + 1.173 |z| units in the last place of fp32 (2^-19 at |z| = 10, 2^-16.4 at 80), its quotient by
// two, against the 2^-8 or 2^-11 of the rounding that follows. `exact` goes with fp32 ones. The normal cdf is CUDA's
// own function, which does not cancel on the negative side as 1 + erf does.
#pragma once

#include "b200_common.cuh"

namespace b200 {

// v s(z)
template <bool FAST> __device__ __forceinline__ float gate_times_sigmoid(float v, float z) {
  const float t = FAST ? __expf(-fabsf(z)) : expf(-fabsf(z)), w = z < 0.f ? v * t : v;
  return FAST ? __fdividef(w, 1.f + t) : w / (1.f + t);
}
template <bool FAST> __device__ __forceinline__ float gate_sigmoid(float z) { return gate_times_sigmoid<FAST>(1.f, z); }
__device__ __forceinline__ float gelu_tanh_arg(float g) { return 1.5957691216057308f * (g + 0.044715f * g * g * g); }  // 2 z

struct ActSilu {
  template <bool FAST> static __device__ __forceinline__ float f(float g) { return gate_times_sigmoid<FAST>(g, g); }
  template <bool FAST> static __device__ __forceinline__ void both(float g, float& a, float& d) {
    const float s = gate_sigmoid<FAST>(g);
    a = g * s;
    d = s * (1.f + g * (1.f - s));
  }
  __device__ __forceinline__ float fast(float g) const { return f<true>(g); }
  __device__ __forceinline__ float exact(float g) const { return f<false>(g); }
};
struct ActGelu {
  template <bool FAST> static __device__ __forceinline__ float f(float g) { return g * normcdff(g); }
  template <bool FAST> static __device__ __forceinline__ void both(float g, float& a, float& d) {
    const float c = normcdff(g), e = -0.5f * g * g;
    a = g * c;
    d = c + g * 0.3989422804014327f * (FAST ? __expf(e) : expf(e));
  }
  __device__ __forceinline__ float fast(float g) const { return f<true>(g); }
  __device__ __forceinline__ float exact(float g) const { return f<false>(g); }
};
struct ActGeluTanh {
  template <bool FAST> static __device__ __forceinline__ float f(float g) { return gate_times_sigmoid<FAST>(g, gelu_tanh_arg(g)); }
  template <bool FAST> static __device__ __forceinline__ void both(float g, float& a, float& d) {
    const float s = gate_sigmoid<FAST>(gelu_tanh_arg(g));
    a = g * s;
    // beyond 30 the slope is 0 or 1 to the last bit, and g^2 stays finite
    const float h = g < -30.f ? -30.f : g > 30.f ? 30.f : g;
    d = s + h * s * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * h * h);
  }
  __device__ __forceinline__ float fast(float g) const { return f<true>(g); }
  __device__ __forceinline__ float exact(float g) const { return f<false>(g); }
};
struct ActRelu {
  template <bool FAST> static __device__ __forceinline__ float f(float g) { return g <= 0.f ? 0.f : g; }
  template <bool FAST> static __device__ __forceinline__ void both(float g, float& a, float& d) {
    a = g <= 0.f ? 0.f : g;
    d = g <= 0.f ? 0.f : 1.f;
  }
  __device__ __forceinline__ float fast(float g) const { return f<true>(g); }
  __device__ __forceinline__ float exact(float g) const { return f<false>(g); }
};
struct ActSigmoid {
  template <bool FAST> static __device__ __forceinline__ float f(float g) { return gate_sigmoid<FAST>(g); }
  template <bool FAST> static __device__ __forceinline__ void both(float g, float& a, float& d) {
    a = gate_sigmoid<FAST>(g);
    d = a * (1.f - a);
  }
  __device__ __forceinline__ float fast(float g) const { return f<true>(g); }
  __device__ __forceinline__ float exact(float g) const { return f<false>(g); }
};

// `body` with the activation as its argument: one look per tile or thread, not one per value
#pragma nv_exec_check_disable
template <typename F> __host__ __device__ __forceinline__ void gate_act_each(int act, F body) {
  switch (act) {
    case B200_ACT_SILU: body(ActSilu{}); break;
    case B200_ACT_GELU: body(ActGelu{}); break;
    case B200_ACT_GELU_TANH: body(ActGeluTanh{}); break;
    case B200_ACT_RELU: body(ActRelu{}); break;
    default: body(ActSigmoid{}); break;
  }
}

}  // namespace b200

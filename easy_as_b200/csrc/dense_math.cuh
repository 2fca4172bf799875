// dense_math.cuh — activations, their derivatives and 16-bit conversions of the dense-layer kernels.
//
//   none       z                          1
//   relu       max(z, 0)                  z > 0
//   gelu       z Phi(z)                   Phi(z) + z phi(z)
//   gelu_tanh  z s(q), q = 2c(z + a z^3)  s(q) + z s(q) s(-q) 2c(1 + 3 a z^2)      c = sqrt(2/pi), a = 0.044715
//   silu       z s(z)                     s(z) + z s(z) s(-z)
//   sigmoid    s(z)                       s(z) s(-z)
//
// with s the logistic function and Phi, phi the normal distribution and its density.  s(-z) is computed
// beside s(z) from the same exponential, not as 1 - s(z), which would cancel.  All in f32; exp is
// __expf (2 + 1.17 |z| ulp: under 2^-16 relative wherever s is a normal f32), far below the 2^-9
// or 2^-12 of the 16-bit result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace dense {

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4, kSigmoid = 5, kActs = 6 };
enum Type { kF16 = 0, kBF16 = 1, kTypes = 2 };

// s(z) and s(-z) = 1 - s(z).  e = exp(-|z|) <= 1, so nothing overflows.
__device__ __forceinline__ void logistic(float z, float& p, float& q) {
  const float e = __expf(-fabsf(z));
  const float r = __fdividef(1.0f, 1.0f + e);
  const float small = e * r;
  p = z < 0 ? small : r;
  q = z < 0 ? r : small;
}

constexpr float kGeluC2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// Phi(z) and e = exp(-z^2 / 2), which its density shares.  The tail 1 - Phi(|z|) is e times a smooth
// function that falls like 1 / |z|: a polynomial without constant term in t = 1 / (1 + 0.3606 |z|), the
// form of Hastings' approximations of the error function, here of degree 7 with coefficients fitted
// to the least relative error (1.2e-6 for |z| < 13 in f32).  So the tail of a negative z is as exact
// as its exponential, where 1 + erf(z / sqrt 2) would cancel; 14 instructions, against about 50 of
// erfcf (the backward pass of 4096 x 8192 pre-activations took 89 us with it, where its bytes take 31).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  e = __expf(-0.5f * z * z);
  const float t = __fdividef(1.0f, fmaf(0.36062446f, fabsf(z), 1.0f));
  float p = fmaf(t, 4.724989589e-02f, -1.795671291e-01f);
  p = fmaf(t, p, 1.792224294e-01f);
  p = fmaf(t, p, 2.752668697e-02f);
  p = fmaf(t, p, 1.395329766e-01f);
  p = fmaf(t, p, 1.420761715e-01f);
  p = fmaf(t, p, 1.439587504e-01f);
  const float tail = e * (t * p);
  return z < 0 ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == kRelu) {
    return z < 0 ? 0.0f : z;  // NaN stays NaN
  } else if constexpr (ACT == kGelu) {
    float e;
    return z * normal_cdf(z, e);
  } else if constexpr (ACT == kGeluTanh) {
    float p, q;
    logistic(kGeluC2 * z * (1.0f + kGeluA * z * z), p, q);
    return z * p;
  } else if constexpr (ACT == kSilu) {
    float p, q;
    logistic(z, p, q);
    return z * p;
  } else if constexpr (ACT == kSigmoid) {
    float p, q;
    logistic(z, p, q);
    return p;
  }
  return z;
}

// An infinite z is what f16 holds of a finite pre-activation past 65504: the value and the slope are the ones
// of far values (0 and 0 to the left, where the formula's -inf x 0 is none; slope 1 to the right).
template <int ACT>
__device__ __forceinline__ void act_and_slope(float z, float& v, float& d) {
  v = z;
  d = 1.0f;
  float p, q;
  // (both of them pass NaN by; p and cdf keep it)
  const float left = fmaxf(z, -3.402823466e38f), far = fminf(left, 3.402823466e38f);
  if constexpr (ACT == kRelu) {
    v = z < 0 ? 0.0f : z;
    d = z > 0 ? 1.0f : (z <= 0 ? 0.0f : z);
  } else if constexpr (ACT == kGelu) {
    float e;
    const float cdf = normal_cdf(z, e);
    v = left * cdf;
    d = cdf + far * (0.39894228040143268f * e);
  } else if constexpr (ACT == kGeluTanh) {
    const float z2 = fminf(z * z, 1e4f);  // past it s(z) s(-z) is 0 and the bracket must not be infinite
    logistic(kGeluC2 * z * (1.0f + kGeluA * z2), p, q);
    v = left * p;
    d = p + far * p * q * (kGeluC2 * (1.0f + 3.0f * kGeluA * z2));
  } else if constexpr (ACT == kSilu) {
    logistic(z, p, q);
    v = left * p;
    d = p * (1.0f + far * q);
  } else if constexpr (ACT == kSigmoid) {
    logistic(z, p, q);
    v = p;
    d = p * q;
  }
}

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t h) {
  if constexpr (BF16) return __uint_as_float((uint32_t)h << 16);
  return __half2float(__ushort_as_half(h));
}

template <bool BF16>
__device__ __forceinline__ uint16_t to_16(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}

// two values in one word, the first in the low half
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

// Runs `f` with the activation as a compile-time constant.
template <typename F>
__device__ __forceinline__ void with_act(int a, F&& f) {
  switch (a) {
    case kRelu: f(std::integral_constant<int, kRelu>()); break;
    case kGelu: f(std::integral_constant<int, kGelu>()); break;
    case kGeluTanh: f(std::integral_constant<int, kGeluTanh>()); break;
    case kSilu: f(std::integral_constant<int, kSilu>()); break;
    case kSigmoid: f(std::integral_constant<int, kSigmoid>()); break;
    default: f(std::integral_constant<int, kNone>()); break;
  }
}

// 16-bit values s .. s + 7 of the 16 in two neighbouring words of 16 bytes.
__device__ __forceinline__ uint4 shift8(const uint4& a, const uint4& b, int s) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 6; ++j) w[j] = s & 4 ? w[j + 2] : w[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) w[j] = s & 2 ? w[j + 1] : w[j];
  const int bits = (s & 1) * 16;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// v with zeros behind its first n of 8 values.
__device__ __forceinline__ uint4 first8(const uint4& v, int n) {
  auto mask = [&](int j) { return n >= 2 * j + 2 ? 0xffffffffu : n == 2 * j + 1 ? 0xffffu : 0u; };
  return make_uint4(v.x & mask(0), v.y & mask(1), v.z & mask(2), v.w & mask(3));
}

// The first n of 8 values (zeros behind them) from any address: the one or two aligned words of 16 bytes
// that hold them, shifted together.  fetch() only loads, so that several can be under way before the
// first get().  A word that reaches out of the matrix's own memory [lo, hi) is left out, and its
// values are read one by one.
struct Gather8 {
  uint4 a, b;
  const uint16_t* p;
  int n, s;
  bool inside;

  __device__ __forceinline__ void fetch(const uint16_t* from, int count, const uint16_t* lo, const uint16_t* hi) {
    p = from, n = count;
    s = (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
    const uint16_t* word = p - s;
    const bool two = s + min(n, 8) > 8;
    inside = word >= lo && word + (two ? 16 : 8) <= hi;
    a = b = make_uint4(0, 0, 0, 0);
    if (inside && n > 0) a = *reinterpret_cast<const uint4*>(word);
    if (inside && two) b = reinterpret_cast<const uint4*>(word)[1];
  }
  __device__ __forceinline__ uint4 get() const {
    uint4 v = shift8(a, b, s);
    if (!inside) {
      auto one = [&](int j) { return j < n ? (uint32_t)p[j] : 0u; };
      v = make_uint4(one(0) | one(1) << 16, one(2) | one(3) << 16, one(4) | one(5) << 16, one(6) | one(7) << 16);
    }
    return first8(v, n);
  }
};

}  // namespace dense

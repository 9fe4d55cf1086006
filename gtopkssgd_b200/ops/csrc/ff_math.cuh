// What the kernels of the feed-forward operators (K6 layer norm, K7 8-bit activations, K8 matrix products) share:
// element types, vectors of them, activations with their slopes, and the 8-bit block format.
//
// All arithmetic is in f32; a value is rounded once, where it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace gtk {

enum ElemType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActCount = 5 };

inline int elem_bytes(int type) { return type == kF32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements that move with one access of sizeof(T) * N bytes (two or more of 16 where that is longer).
template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};
// Two neighbours of a 16-bit type at a time: an instruction each to unpack, one for both to pack.
__device__ __forceinline__ void unpack2(uint32_t u, float* a, float* b, __nv_bfloat16) {
  *a = __uint_as_float(u << 16);
  *b = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float* a, float* b, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  *a = f.x;
  *b = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <typename T, int N>
__device__ __forceinline__ void to_f32(const Vec<T, N>& x, float (&out)[N]) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < N; i += 2) unpack2(w[i / 2], &out[i], &out[i + 1], T{});
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_f32(x.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[N]) {
  const Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(p);
  to_f32<T, N>(x, out);
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[N]) {
  Vec<T, N> x;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < N; i += 2) w[i / 2] = pack2(in[i], in[i + 1], T{});
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = from_f32<T>(in[i]);
  }
  *reinterpret_cast<Vec<T, N>*>(p) = x;
}

// ---- activations ---------------------------------------------------------------------------------------------
// On tiles of a matrix product these are the larger part of the epilogue's instructions, and of an element-wise pass
// in 16 bits they, not the bytes, set the time (erff and expf: 240 us for 16384 x 8192, of which the bytes are 100).  So
// each is written with one exponential and one reciprocal of the special-function unit, a few units of 2^-24 off.
constexpr float kSqrt2OverPi = 0.79788456080286536f;     // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;
constexpr float kLog2E = 1.44269504088896341f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two values that are multiplied and added by one instruction; what follows is written for these and for single ones.
struct Two {
  unsigned long long u;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void parts(Two x, float* a, float* b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x.u)); }
__device__ __forceinline__ Two vmul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ Two vfma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ Two vadd(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
template <typename V>
__device__ __forceinline__ V vset(float c) {
  if constexpr (sizeof(V) == 8) return two(c, c);
  else return c;
}
__device__ __forceinline__ float vtotal(float x) { return x; }
__device__ __forceinline__ float vtotal(Two x) {
  float a, b;
  parts(x, &a, &b);
  return a + b;
}
// Element, or pair of elements, i of an array, and back.
template <typename V>
__device__ __forceinline__ V vget(const float* v, int i) {
  if constexpr (sizeof(V) == 8) return two(v[2 * i], v[2 * i + 1]);
  else return v[i];
}
__device__ __forceinline__ void vput(float* v, int i, float x) { v[i] = x; }
__device__ __forceinline__ void vput(float* v, int i, Two x) { parts(x, v + 2 * i, v + 2 * i + 1); }
template <int N>
using Wide = std::conditional_t<N % 2 == 0, Two, float>;   // what N elements are computed in

template <typename F>
__device__ __forceinline__ float each(float x, F&& f) { return f(x); }
template <typename F>
__device__ __forceinline__ Two each(Two x, F&& f) {
  float a, b;
  parts(x, &a, &b);
  return two(f(a), f(b));
}
template <typename V>
__device__ __forceinline__ V vexp2(V x) { return each(x, [](float v) { return exp2_fast(v); }); }
template <typename V>
__device__ __forceinline__ V vrcp(V x) { return each(x, [](float v) { return rcp_fast(v); }); }
template <typename V>
__device__ __forceinline__ V vabs(V x) { return each(x, [](float v) { return fabsf(v); }); }
__device__ __forceinline__ float vwhere_negative(float z, float a, float b) { return z < 0.f ? a : b; }
__device__ __forceinline__ Two vwhere_negative(Two z, Two a, Two b) {
  float z0, z1, a0, a1, b0, b1;
  parts(z, &z0, &z1);
  parts(a, &a0, &a1);
  parts(b, &b0, &b1);
  return two(z0 < 0.f ? a0 : b0, z1 < 0.f ? a1 : b1);
}

// 1 / (1 + e^-(c z))
template <typename V>
__device__ __forceinline__ V sigmoid(V z, float c) {
  const V e = vexp2(vmul(z, vset<V>(-kLog2E * c)));
  return vrcp(vfma(e, vset<V>(1.f), vset<V>(1.f)));
}

// The normal distribution's Phi(z), and e^(-z^2 / 2), which it contains: Phi(-|z|) = e^(-z^2 / 2) t (b1 + t (b2 + ...)),
// t = 1 / (1 + p |z| / sqrt 2), Abramowitz and Stegun 7.1.26 for the error function with its coefficients halved; 7.5e-8
// off at most.
template <typename V>
__device__ __forceinline__ V normal_cdf(V z, V* bell) {
  const V t = vrcp(vfma(vabs(z), vset<V>(0.3275911f * 0.70710678118654752f), vset<V>(1.f)));
  const V g = vexp2(vmul(vmul(z, z), vset<V>(-0.5f * kLog2E)));
  V p = vfma(t, vset<V>(0.5f * 1.061405429f), vset<V>(0.5f * -1.453152027f));
  p = vfma(t, p, vset<V>(0.5f * 1.421413741f));
  p = vfma(t, p, vset<V>(0.5f * -0.284496736f));
  p = vfma(t, p, vset<V>(0.5f * 0.254829592f));
  const V tail = vmul(vmul(p, t), g);
  *bell = g;
  return vwhere_negative(z, tail, vfma(tail, vset<V>(-1.f), vset<V>(1.f)));
}

// 2 sqrt(2 / pi) (z + c z^3): (1 + tanh u) / 2 = 1 / (1 + e^-2u)
template <typename V>
__device__ __forceinline__ V tanh_argument(V z) {
  return vmul(z, vfma(vmul(z, z), vset<V>(2.f * kSqrt2OverPi * kGeluCubic), vset<V>(2.f * kSqrt2OverPi)));
}

template <int ACT, typename V>
__device__ __forceinline__ V act_value(V z) {
  if constexpr (ACT == kActRelu) return vwhere_negative(z, vset<V>(0.f), z);  // a NaN stays one
  if constexpr (ACT == kActGelu) {
    V bell;
    return vmul(z, normal_cdf(z, &bell));
  }
  if constexpr (ACT == kActGeluTanh) return vmul(z, sigmoid(tanh_argument(z), 1.f));
  if constexpr (ACT == kActSilu) return vmul(z, sigmoid(z, 1.f));
  return z;
}

// d act(z) / dz, and act(z) itself, which shares its work.
template <int ACT, typename V>
__device__ __forceinline__ V act_slope(V z, V* value) {
  if constexpr (ACT == kActRelu) {
    *value = vwhere_negative(z, vset<V>(0.f), z);
    return each(z, [](float v) { return v > 0.f ? 1.f : 0.f; });
  }
  if constexpr (ACT == kActGelu) {
    V bell;
    const V cdf = normal_cdf(z, &bell);
    *value = vmul(z, cdf);
    return vfma(vmul(z, vset<V>(0.39894228040143268f)), bell, cdf);   // 1 / sqrt(2 pi)
  }
  if constexpr (ACT == kActGeluTanh) {
    const V s = sigmoid(tanh_argument(z), 1.f);
    const V h = vmul(z, s);
    *value = h;
    // s + t du, t = h (1 - s), du = 2 sqrt(2 / pi) (1 + 3 c z^2); t first, which is 0 before z^2 leaves f32's range
    const V t = vmul(h, vfma(s, vset<V>(-1.f), vset<V>(1.f)));
    return vfma(vmul(vmul(t, z), z), vset<V>(6.f * kSqrt2OverPi * kGeluCubic), vfma(t, vset<V>(2.f * kSqrt2OverPi), s));
  }
  if constexpr (ACT == kActSilu) {
    const V s = sigmoid(z, 1.f);
    const V h = vmul(z, s);
    *value = h;
    return vfma(h, vfma(s, vset<V>(-1.f), vset<V>(1.f)), s);   // s (1 + z (1 - s))
  }
  *value = z;
  return vset<V>(1.f);
}

// N values in place; and slopes times what is in g, z becoming the values.
template <int ACT, int N>
__device__ __forceinline__ void act_values(float (&z)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) parts(act_value<ACT>(two(z[i], z[i + 1])), &z[i], &z[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = act_value<ACT>(z[i]);
  }
}
template <int ACT, int N>
__device__ __forceinline__ void act_slopes(float (&g)[N], float (&z)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      Two value;
      const Two slope = act_slope<ACT>(two(z[i], z[i + 1]), &value);
      parts(vmul(two(g[i], g[i + 1]), slope), &g[i], &g[i + 1]);
      parts(value, &z[i], &z[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float value;
      g[i] *= act_slope<ACT>(z[i], &value);
      z[i] = value;
    }
  }
}

// Calls f with the activation's number as a type.
template <int A>
using ActConst = std::integral_constant<int, A>;
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case kActRelu: f(ActConst<kActRelu>{}); break;
    case kActGelu: f(ActConst<kActGelu>{}); break;
    case kActGeluTanh: f(ActConst<kActGeluTanh>{}); break;
    case kActSilu: f(ActConst<kActSilu>{}); break;
    default: f(ActConst<kActNone>{}); break;
  }
}

// ---- 8 bits: blocks of 32 along a row ----------------------------------------------------------------------------
// A block stores one byte, e + 127, with e the least integer (at least -127) for which max|x| <= 127 * 2^e; a value
// is q = rint(x * 2^-e), |q| <= 127, and stands for q * 2^e.  Both scalings are by powers of two, so that only rint
// rounds and the codes do not depend on the precision they are computed in.  Byte 255: the block held a NaN or an
// infinity and every value of it stands for NaN.  In the last step, 2^122, codes stop at 63: 64 would stand for 2^128.
constexpr int kBlock8 = 32;
constexpr uint32_t kBlock8NaN = 255u, kBlock8Last = 249u;

// abs_bits: the largest bit pattern of |x| in the block.
__device__ __forceinline__ uint32_t block8_byte(uint32_t abs_bits) {
  if (abs_bits >= 0x7f800000u) return kBlock8NaN;
  // |x| = m * 2^E with m in [1, 2): e = E - 6 where m <= 127/64 (mantissa bits up to 0x7e0000), else E - 5
  const int e = (int)((abs_bits + (0x7fffffu - 0x7e0000u)) >> 23) - 127 - 6;
  return (uint32_t)(e < -127 ? 0 : e + 127);
}
// 2^(byte - 127) for byte 0 .. 254, NaN for 255
__device__ __forceinline__ float block8_scale(uint32_t byte) {
  return __uint_as_float(byte == kBlock8NaN ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}
// 2^-(byte - 127), for the bytes 0 .. 249 (255: something)
__device__ __forceinline__ float block8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// The largest magnitude of three, NaN where one is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Four codes in a word, for bytes below kBlock8Last: adding 1.5 * 2^23 rounds to an integer, whose low byte it leaves in
// the low byte of the sum.
__device__ __forceinline__ uint32_t block8_codes(float a, float b, float c, float d, float inverse) {
  constexpr float kMagic = 12582912.f;
  const uint32_t ia = __float_as_uint(fmaf(a, inverse, kMagic)), ib = __float_as_uint(fmaf(b, inverse, kMagic));
  const uint32_t ic = __float_as_uint(fmaf(c, inverse, kMagic)), id = __float_as_uint(fmaf(d, inverse, kMagic));
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}
// What the four codes of a word stand for: byte + 128 becomes the low byte of 2^23, from which 2^23 + 128 is taken and the
// rest scaled, both exactly.  (One multiply-add of what is scaled already would take it past f32's range from 2^105 on.)
__device__ __forceinline__ void block8_values(uint32_t codes, float scale, float* v) {
  const uint32_t u = codes ^ 0x80808080u;
  const Two back = vset<Two>(-8388736.f), by = vset<Two>(scale);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const Two q = two(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + i)));
    parts(vmul(vadd(q, back), by), v + i, v + i + 1);
  }
}
__device__ __forceinline__ int block8_code(float x, uint32_t byte) {
  const int q = __float2int_rn(x * block8_inverse(byte));
  return byte < kBlock8Last ? q : byte == kBlock8NaN ? 0 : max(-63, min(63, q));
}

// ---- f32 as three bf16 pieces ---------------------------------------------------------------------------------------
// Three bf16 pieces whose sum is v to 24 bits: each is the nearest to what the ones before left.  The first is cut
// instead of rounded where rounding would overflow; a NaN or an infinity is all in the first.
__device__ __forceinline__ void split3(float v, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(v);
  if (isinf(__bfloat162float(p[0])) && !isinf(v)) p[0] = __float2bfloat16_rz(v);
  float left = v - __bfloat162float(p[0]);
  if (!(fabsf(v) <= 3.402823466e38f)) left = 0.f;
  p[1] = __float2bfloat16_rn(left);
  p[2] = __float2bfloat16_rn(left - __bfloat162float(p[1]));
}
// The lower products' sum on top of one that has the first pieces' products.  Where that is no longer finite it is the result:
// the first piece has its value's sign and is zero only where it is, but an infinity, and what leaves f32's range, may meet
// lower pieces that are zero or of the other sign.
__device__ __forceinline__ float add_lower(float sum, float lower) { return fabsf(sum) <= 3.402823466e38f ? sum + lower : sum; }

// ---- f32 as two f16 pieces -----------------------------------------------------------------------------------------
// The power of two by which values whose largest magnitude has these bits are scaled: it then lies in [2^14, 2^15).
// Values down to 2^-17 of the largest keep 22 bits, smaller ones are off by 2^-40 of it at most.
__device__ __forceinline__ int pair_shift(uint32_t most) {
  const int shift = 14 + 127 - (int)(most >> 23);
  return most == 0u || most >= 0x7f800000u ? 0 : shift > 126 ? 126 : shift;
}

}  // namespace gtk

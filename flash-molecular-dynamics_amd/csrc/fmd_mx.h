// Block-scaled numbers (32 columns of a row share a power of two) and the bf16 planes the products are made of.
//
//   4 bits   value = e2m1 * 2^(byte-127)            e2m1 in {0,.5,1,1.5,2,3,4,6}, two to a byte, even column low
//   8 bits   value = int8 / 64 * 2^(byte-127)       int8 in [-127,127]
//
// byte = max(floor(log2 amax) - (4 bits: 2, 8 bits: 0), -127) + 127; a block that holds an Inf or a NaN gets byte 255
// and stands for NaN.  Scaling by a power of two is exact, so the codes are a function of the input's bits alone.
//
// Planes: an fp32 value is the exact sum of three bf16 (truncation keeps 8 significant bits at a time), an fp16 value of
// two, a bf16 value and every 4- or 8-bit block value is one.  A product of plane sums keeps the plane pairs (i, j) with
// i + j < max(planes): what is dropped is below the last kept plane's last bit.  bf16 has fp32's range, so no operand
// needs a scale of its own.  Where every operand is fp16 or a function of fp16 values that stays in its range (a wide layer's
// training products), one fp16 plane does the work of two bf16 ones; the 8-bit value of an fp16 number is one itself.
//
// Operands that are computed (tanh(x), tanh of an 8-bit value, a gradient times tanh') are no such sums.  fp32 has its three planes for
// them, a narrow 16-bit layer two: 2^-15 of the value.  A wide 16-bit layer has one plane of its type for them, two bf16 ones for an fp16
// gradient times tanh': they are rounded to the type once more, as a layer of separate 16-bit operations would, because a second
// plane doubles the products.  8192 x 4096 -> 1024 bf16 under tanh, us a call: forward 128, with two planes 228; backward 290, 418; 2.2e-3
// from the exact result, 1.7e-3.  4096 x 4096 -> 4096 with 4-bit weights backward 192, 303.  1294 x 6196 -> 2319 fp16, a training step
// with one fp16 plane 277, with two bf16 planes of everything 573; 2.7e-4 from the exact result, 2.1e-4.
#pragma once
#include "fmd_common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct mx_bf16 { uint16_t u; };  // bf16 in memory

template <class T> struct MxType;
template <> struct MxType<float> {
  static constexpr int planes = 3;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct MxType<_Float16> {
  static constexpr int planes = 2;
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float v) { return (_Float16)v; }
};
template <> struct MxType<mx_bf16> {
  static constexpr int planes = 1;
  static __device__ __forceinline__ float to(mx_bf16 v) { return __builtin_bit_cast(float, (uint32_t)v.u << 16); }
  static __device__ __forceinline__ mx_bf16 from(float v) {  // nearest even
    const __bf16 b = (__bf16)v;
    return mx_bf16{__builtin_bit_cast(uint16_t, b)};
  }
};

static inline int64_t mx_blocks(int64_t k) { return (k + 31) / 32; }
static inline int64_t mx_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// pairs (i, j) of planes whose product is kept, the smallest first
struct MxPairs { int n; int8_t a[6], b[6]; };
static inline MxPairs mx_pairs(int pa, int pb) {
  MxPairs p{};
  const int top = pa > pb ? pa : pb;
  for (int s = top - 1; s >= 0; --s)
    for (int i = 0; i < pa; ++i) {
      const int j = s - i;
      if (j >= 0 && j < pb) { p.a[p.n] = (int8_t)i; p.b[p.n] = (int8_t)j; ++p.n; }
    }
  return p;
}

// ---- scales ---------------------------------------------------------------------------------------------------------
// scale byte of a block from the largest bit pattern of |x| (an unsigned maximum: a NaN's pattern is above Inf's)
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  // floor(log2) of a subnormal is below every exponent the byte can hold
  const int e = (int)(top >> 23) - (BITS == 4 ? 2 : 0);  // biased by 127 already
  return e > 0 ? (uint32_t)e : 0u;
}
// 2^(byte-127) as fp32 (byte 0: the subnormal 2^-127; byte 255: NaN)
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// four 8-bit codes of a block, the first in the low byte.  64 x / 2^E is exact; adding 1.5 * 2^23 rounds it to nearest even and
// leaves the integer in the low bits
__device__ __forceinline__ uint32_t mx_codes8(float x0, float x1, float x2, float x3, uint32_t byte) {
  const int e = 133 - (int)byte;
  auto bits = [e](float x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(__builtin_ldexpf(x, e), -127.f, 127.f) + 12582912.f);
  };
  const uint32_t lo = __builtin_amdgcn_perm(bits(x1), bits(x0), 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits(x3), bits(x2), 0x0c0c0400u);
  return byte == 255u ? 0u : lo | hi << 16;
}
__device__ __forceinline__ float mx_value8(int code, uint32_t byte) {
  return byte == 255u ? __builtin_nanf("") : __builtin_ldexpf((float)code, (int)byte - 133);
}
// eight 4-bit codes (columns 0..7 from the low bits up) of a block of the given scale value
__device__ __forceinline__ uint32_t mx_codes4(const float (&v)[8], float scale) {
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], scale, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], scale, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], scale, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], scale, 3);
  return o;
}
// eight 4-bit codes as bf16 (exact: e2m1 has two significant bits)
__device__ __forceinline__ u32x4 mx_bf16_from4(uint32_t codes, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}

// 1 / (e^{2|x|} + 1), what tanh and tanh' are made of
__device__ __forceinline__ float mx_sigma(float x) { return __builtin_amdgcn_rcpf(__expf(2.0f * fabsf(x)) + 1.0f); }
// tanh without a branch: 1 - 2 t, t = mx_sigma(x), from |x| = 1/4 up (absolute error 8e-8), the odd Taylor polynomial to x^9 below
// (the next term is 2e-9 of it there), so that small values keep their relative accuracy
__device__ __forceinline__ float mx_tanh(float x, float t) {
  const float x2 = x * x;
  const float p = x * (1.0f + x2 * (-0.33333334f + x2 * (0.13333334f + x2 * (-0.053968254f + x2 * 0.021869488f))));
  const float y = copysignf(1.0f - 2.0f * t, x);
  return fabsf(x) < 0.25f ? p : y;  // a NaN takes the second and stays one
}
__device__ __forceinline__ float mx_tanh(float x) { return mx_tanh(x, mx_sigma(x)); }
// tanh' = 1 - tanh^2 = 4 t (1 - t): no digits cancel, so that it keeps its relative accuracy as tanh goes to one.  What is lost is the
// exponent's rounding, 3 |x| units in the last place.  (1 - y^2 of an fp32 y is off by 28 % at |x| = 8.5.)
__device__ __forceinline__ float mx_dtanh_of(float t) { return 4.0f * t * (1.0f - t); }

// v times tanh' of an 8-bit value.  The product is rounded to fp32 before anything else is made of it (the compiler would form
// it and round it to 16 bits in one instruction here and two there), so that every kernel gives the same bits.
__device__ __forceinline__ float mx_times_dtanh(float v, int code, uint32_t byte) {
  float r = v * mx_dtanh_of(mx_sigma(mx_value8(code, byte)));
  asm("" : "+v"(r));
  return r;
}

// tanh' as a 16-bit layer keeps it for its backward pass, in 16 bits.  It has no sign and is at most one, which leaves 4 bits of exponent
// and 12 of fraction: half a step is 2^-13 of the value, or 2^-27 below 2^-14 (sums beyond 5.5).  The code is the value times 2^-112 as fp32
// holds it -- its subnormal numbers are the small values --, rounded to the 12th bit of the fraction; 0xf000 is one, what is above a NaN.
// As fp16 it costs the gradients of an fp16 layer 2.9e-4 against 2.1e-4 of theirs.  500000 x 64 -> 128 fp16 forward and backward, us a
// call: as fp16 91 + 112, like this 94 + 110, as fp32, half as many bytes again, 142 for the second.
struct mx_dact { uint16_t u; };
template <> struct MxType<mx_dact> {
  static __device__ __forceinline__ float to(mx_dact v) {
    return v.u > 0xf000u ? __builtin_nanf("") : __builtin_bit_cast(float, (uint32_t)v.u << 11) * 0x1p112f;
  }
  // from tanh' 2^-112.  A NaN's exponent is all ones, its quiet bit set: 0xf800 and above
  static __device__ __forceinline__ mx_dact from(float v) { return mx_dact{(uint16_t)((__builtin_bit_cast(uint32_t, v) + 0x400u) >> 11)}; }
};
__device__ __forceinline__ float mx_keep_dtanh_of(float t) { return t * 0x1p-110f * (1.0f - t); }

// a wave-uniform value that the compiler takes for a new one: what is computed from it stays where it is used, in scalar
// registers, instead of becoming dozens of loop-invariant vector registers
__device__ __forceinline__ int mx_here(int v) {
  asm volatile("" : "+s"(v));
  return v;
}

// ---- planes -----------------------------------------------------------------------------------------------------------
// two fp32 values -> one dword of bf16 pairs per plane.  Cutting off the low half keeps 8 significant bits and cannot
// overflow; the remainder is exact.  x == hi for an Inf, whose remainder is then 0 and not Inf - Inf; a NaN whose low
// half alone is set leaves a NaN remainder, so no NaN is lost.
template <int P>
__device__ __forceinline__ void mx_split2(float x, float y, uint32_t (&out)[P]) {
  if constexpr (P == 1) {  // one plane: rounded to nearest even
    bf16x2 b;
    b[0] = (__bf16)x;
    b[1] = (__bf16)y;
    out[0] = __builtin_bit_cast(uint32_t, b);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t ux = __builtin_bit_cast(uint32_t, x), uy = __builtin_bit_cast(uint32_t, y);
      out[p] = __builtin_amdgcn_perm(uy, ux, 0x07060302u);
      if (p + 1 < P) {
        const float hx = __builtin_bit_cast(float, ux & 0xffff0000u), hy = __builtin_bit_cast(float, uy & 0xffff0000u);
        x = x == hx ? 0.f : x - hx;
        y = y == hy ? 0.f : y - hy;
      }
    }
  }
}
// P = 0: one plane of fp16
template <int P>
__device__ __forceinline__ void mx_split8(const float (&v)[8], u32x4 (&out)[P ? P : 1]) {
  if constexpr (P == 0) {
    f16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (_Float16)v[i];
    out[0] = __builtin_bit_cast(u32x4, o);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t o[P ? P : 1];
    mx_split2<P ? P : 1>(v[2 * i], v[2 * i + 1], o);
#pragma unroll
    for (int p = 0; p < P; ++p) out[p][i] = o[p];
  }
}

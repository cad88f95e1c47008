// Block quantisation along the rows and back (formats: fmd_mx.h).
//
// A thread holds 8 columns, four neighbouring lanes a block of 32: the block's largest magnitude is an unsigned maximum of
// the bit patterns over the four lanes.  One pass: read x once, write codes and scales once.  Bound by memory.
#include "fmd_mx.h"

namespace {

template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t c0, int64_t k, bool vec, float (&v)[8]) {
  if (vec && c0 + 8 <= k) {
    T t[8];
    if constexpr (sizeof(T) == 4) {
      *(u32x4*)&t[0] = *(const u32x4*)(row + c0);
      *(u32x4*)&t[4] = *(const u32x4*)(row + c0 + 4);
    } else {
      *(u32x4*)&t[0] = *(const u32x4*)(row + c0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = MxType<T>::to(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < k ? MxType<T>::to(row[c0 + i]) : 0.f;
  }
}

// lay8: where the scale byte of (row, block) goes.  0: [row][blocks].  1: [block/8][row][8], the order in which the product
// kernel reads them (rows = `rows`)
template <class T, int BITS>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t m, int64_t k, int64_t nb, int vec,
                                                       uint32_t* __restrict__ codes, uint8_t* __restrict__ scales, int lay8) {
  const int64_t total = m * nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / (nb * 4), q = t - row * (nb * 4);
    float v[8];
    load8<T>(x + row * k, q * 8, k, vec != 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    // total is a multiple of 4 and so is a wave's first t: the four lanes of a block are always active together
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    const uint32_t byte = mx_scale_byte<BITS>(top);
    if constexpr (BITS == 4) {
      const float s = byte == 255u ? 1.f : mx_scale_value(byte);
      uint32_t c = mx_codes4(v, s);
      codes[t] = byte == 255u ? 0u : c;
    } else {
      uint32_t c[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i >> 2] |= (uint32_t)(mx_code8(v[i], byte) & 255) << (8 * (i & 3));
      *(u32x2*)(codes + 2 * t) = u32x2{c[0], c[1]};
    }
    if ((q & 3) == 0) {
      const int64_t b = q >> 2;
      uint8_t* to = scales + (lay8 ? ((b >> 3) * m + row) * 8 + (b & 7) : row * nb + b);
      *to = (uint8_t)byte;
      if (lay8 && b == nb - 1)
        for (int i = 1; i < 8 - (int)(b & 7); ++i) to[i] = 0;
    }
  }
}

template <class T, int BITS>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                         int64_t m, int64_t k, int64_t nb, int vec, T* __restrict__ out) {
  const int64_t total = m * nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / (nb * 4), q = t - row * (nb * 4), c0 = q * 8;
    if (c0 >= k) continue;
    const uint32_t byte = scales[row * nb + (q >> 2)];
    float v[8];
    if constexpr (BITS == 4) {
      const u32x4 b = mx_bf16_from4(codes[t], mx_scale_value(byte));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, i & 1 ? b[i >> 1] & 0xffff0000u : b[i >> 1] << 16);
    } else {
      const u32x2 c = *(const u32x2*)(codes + 2 * t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx_value8((int)(int8_t)(c[i >> 2] >> (8 * (i & 3))), byte);
    }
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = MxType<T>::from(v[i]);
    T* p = out + row * k + c0;
    if (vec && c0 + 8 <= k) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((u32x4*)p)[i] = ((const u32x4*)o)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < k) p[i] = o[i];
    }
  }
}

int grid_for(int64_t threads) {
  const int64_t g = (threads + 255) / 256;
  return (int)(g < 256 * 16 ? g : 256 * 16);
}

template <int BITS>
int quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, int lay8, hipStream_t s) {
  if (m < 0 || k < 1 || dtype < 0 || dtype > 2) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!x || !codes || !scales || ((uintptr_t)x & 15) || ((uintptr_t)codes & 15)) return FMD_EINVAL;
  const int64_t nb = mx_blocks(k);
  const int g = grid_for(m * nb * 4), vec = dtype == FMD_F32 ? k % 4 == 0 : k % 8 == 0;
  if (dtype == FMD_F32)
    quantize_kernel<float, BITS><<<g, 256, 0, s>>>((const float*)x, m, k, nb, vec, (uint32_t*)codes, (uint8_t*)scales, lay8);
  else if (dtype == FMD_F16)
    quantize_kernel<_Float16, BITS><<<g, 256, 0, s>>>((const _Float16*)x, m, k, nb, vec, (uint32_t*)codes, (uint8_t*)scales, lay8);
  else
    quantize_kernel<mx_bf16, BITS><<<g, 256, 0, s>>>((const mx_bf16*)x, m, k, nb, vec, (uint32_t*)codes, (uint8_t*)scales, lay8);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

template <int BITS>
int dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype, hipStream_t s) {
  if (m < 0 || k < 1 || dtype < 0 || dtype > 2) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!out || !codes || !scales || ((uintptr_t)out & 15) || ((uintptr_t)codes & 15)) return FMD_EINVAL;
  const int64_t nb = mx_blocks(k);
  const int g = grid_for(m * nb * 4), vec = dtype == FMD_F32 ? k % 4 == 0 : k % 8 == 0;
  if (dtype == FMD_F32)
    dequantize_kernel<float, BITS><<<g, 256, 0, s>>>((const uint32_t*)codes, (const uint8_t*)scales, m, k, nb, vec, (float*)out);
  else if (dtype == FMD_F16)
    dequantize_kernel<_Float16, BITS><<<g, 256, 0, s>>>((const uint32_t*)codes, (const uint8_t*)scales, m, k, nb, vec, (_Float16*)out);
  else
    dequantize_kernel<mx_bf16, BITS><<<g, 256, 0, s>>>((const uint32_t*)codes, (const uint8_t*)scales, m, k, nb, vec, (mx_bf16*)out);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

}  // namespace

int mx_quantize4_for_product(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, hipStream_t s) {
  return quantize<4>(x, dtype, m, k, codes, scales, 1, s);
}

extern "C" int fmd_mxfp4_quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, void* stream) {
  return quantize<4>(x, dtype, m, k, codes, scales, 0, fmd_stream(stream));
}
extern "C" int fmd_mxfp4_dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype,
                                    void* stream) {
  return dequantize<4>(codes, scales, m, k, out, dtype, fmd_stream(stream));
}
extern "C" int fmd_mxint8_quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, void* stream) {
  return quantize<8>(x, dtype, m, k, codes, scales, 0, fmd_stream(stream));
}
extern "C" int fmd_mxint8_dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype,
                                     void* stream) {
  return dequantize<8>(codes, scales, m, k, out, dtype, fmd_stream(stream));
}

// Block quantisation along the rows and back (formats: fmd_mx.h).
//
// A thread holds 8 columns, four neighbouring lanes a block of 32: the block's largest magnitude is an unsigned maximum of
// the bit patterns over the four lanes.  One pass: read x once, write codes and scales once.  Bound by memory:
// 8192 x 8192 bf16 in 4 bits in 33 us, 5.1 TB/s, back in 29 us, 5.9 TB/s (a large copy runs at 5.0).
#include "fmd_mx.h"

namespace {

// Rows whose length is no multiple of 16 bytes: a workgroup moves ROWS whole rows, which are (32 rows, any length) a multiple of
// 16 bytes of memory, in 16-byte pieces through LDS and takes its columns from there.  (1882048 x 50 fp32 in 4 bits, quantising /
// back to bf16: 121 / 125 us with single values from memory, 97 / 64 us like this: 4.5 / 4.0 TB/s.)
constexpr int ROWS = 32, STAGE = 32 * 1024;  // most LDS of a workgroup; it asks for what its rows take

template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t c0, int64_t k, bool vec, float (&v)[8]) {
  if (vec && c0 + 8 <= k) {
    T t[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((u32x4*)t)[i] = *(const u32x4*)(row + c0 + i * (16 / sizeof(T)));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = MxType<T>::to(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool there = c0 + i < k;  // the load itself is unconditional, of a value that exists
      const float x = MxType<T>::to(row[there ? c0 + i : 0]);
      v[i] = there ? x : 0.f;
    }
  }
}

struct QuantArgs {
  int64_t m, k, nb;
  int vec;
  uint32_t* codes;
  uint8_t* scales;
};

// PRODUCT: where the scale byte of (row, block) goes.  false: [row][blocks].  true: [block/8][block&1][row][4] with
// the rows rounded up to 4, as the product kernel reads them.  The four lanes of a block are always active together
template <int BITS, bool PRODUCT>
__device__ __forceinline__ void quantize8(const QuantArgs& a, int64_t row, int64_t q, const float (&v)[8]) {
  const int64_t t = row * a.nb * 4 + q;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  const uint32_t byte = mx_scale_byte<BITS>(top);
  if constexpr (BITS == 4) {
    const uint32_t c = mx_codes4(v, byte == 255u ? 1.f : mx_scale_value(byte));
    a.codes[t] = byte == 255u ? 0u : c;
  } else {
    *(u32x2*)(a.codes + 2 * t) = u32x2{mx_codes8(v[0], v[1], v[2], v[3], byte), mx_codes8(v[4], v[5], v[6], v[7], byte)};
  }
  if ((q & 3) == 0) {
    const int64_t b = q >> 2;
    if constexpr (PRODUCT) {
      const int64_t pad = (a.m + 3) & ~(int64_t)3;
      auto at = [&](int64_t i) { return a.scales + (((i >> 3) * 2 + (i & 1)) * pad + row) * 4 + (i >> 1 & 3); };
      *at(b) = (uint8_t)byte;
      if (b == a.nb - 1)
        for (int64_t i = b + 1; i & 7; ++i) *at(i) = 0;
    } else {
      a.scales[row * a.nb + b] = (uint8_t)byte;
    }
  }
}

template <class T, int BITS, bool PRODUCT>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, const QuantArgs a) {
  const int64_t total = a.m * a.nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / (a.nb * 4), q = t - row * (a.nb * 4);
    float v[8];
    load8<T>(x + row * a.k, q * 8, a.k, a.vec != 0, v);
    quantize8<BITS, PRODUCT>(a, row, q, v);
  }
}

template <class T, int BITS, bool PRODUCT>
__global__ __launch_bounds__(256) void quantize_staged_kernel(const T* __restrict__ x, const QuantArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int k = (int)a.k, q4 = (int)a.nb * 4;
  const int64_t groups = (a.m + ROWS - 1) / ROWS;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const int64_t row0 = g * ROWS;
    const int rows = (int)(a.m - row0 < ROWS ? a.m - row0 : ROWS), bytes = rows * k * (int)sizeof(T);
    const char* from = (const char*)(x + row0 * k);
    for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16) {
      if (i + 16 <= bytes) *(u32x4*)(lds + i) = *(const u32x4*)(from + i);
      else
        for (int e = i; e < bytes; e += (int)sizeof(T)) *(T*)(lds + e) = *(const T*)(from + e);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < rows * q4; t += 256) {
      const int row = t / q4, q = t - row * q4;
      float v[8];
      load8<T>((const T*)lds + row * k, q * 8, k, false, v);
      quantize8<BITS, PRODUCT>(a, row0 + row, q, v);
    }
    __syncthreads();
  }
}

template <int BITS>
__device__ __forceinline__ void dequantize8(const QuantArgs& a, int64_t row, int64_t q, float (&v)[8]) {
  const int64_t t = row * a.nb * 4 + q;
  const uint32_t byte = a.scales[row * a.nb + (q >> 2)];
  if constexpr (BITS == 4) {
    const u32x4 b = mx_bf16_from4(a.codes[t], mx_scale_value(byte));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, i & 1 ? b[i >> 1] & 0xffff0000u : b[i >> 1] << 16);
  } else {
    const u32x2 c = *(const u32x2*)(a.codes + 2 * t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_value8((int)(int8_t)(c[i >> 2] >> (8 * (i & 3))), byte);
  }
}

template <class T, int BITS>
__global__ __launch_bounds__(256) void dequantize_kernel(const QuantArgs a, T* __restrict__ out) {
  const int64_t total = a.m * a.nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / (a.nb * 4), q = t - row * (a.nb * 4), c0 = q * 8;
    if (c0 >= a.k) continue;
    float v[8];
    dequantize8<BITS>(a, row, q, v);
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = MxType<T>::from(v[i]);
    T* p = out + row * a.k + c0;
    if (a.vec && c0 + 8 <= a.k) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((u32x4*)p)[i] = ((const u32x4*)o)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < a.k) p[i] = o[i];
    }
  }
}

template <class T, int BITS>
__global__ __launch_bounds__(256) void dequantize_staged_kernel(const QuantArgs a, T* __restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int k = (int)a.k, q4 = (int)a.nb * 4;
  const int64_t groups = (a.m + ROWS - 1) / ROWS;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const int64_t row0 = g * ROWS;
    const int rows = (int)(a.m - row0 < ROWS ? a.m - row0 : ROWS), bytes = rows * k * (int)sizeof(T);
    for (int t = threadIdx.x; t < rows * q4; t += 256) {
      const int row = t / q4, q = t - row * q4;
      if (q * 8 >= k) continue;
      float v[8];
      dequantize8<BITS>(a, row0 + row, q, v);
      T* to = (T*)lds + row * k + q * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (q * 8 + i < k) to[i] = MxType<T>::from(v[i]);
    }
    __syncthreads();
    char* to = (char*)(out + row0 * k);
    for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16) {
      if (i + 16 <= bytes) *(u32x4*)(to + i) = *(const u32x4*)(lds + i);
      else
        for (int e = i; e < bytes; e += (int)sizeof(T)) *(T*)(to + e) = *(const T*)(lds + e);
    }
    __syncthreads();
  }
}

int grid_for(int64_t threads) {
  const int64_t g = (threads + 255) / 256;
  return (int)(g < 256 * 16 ? g : 256 * 16);
}

template <class T, int BITS, bool PRODUCT>
void run_quantize(const T* x, QuantArgs a, hipStream_t s) {
  a.vec = a.k * sizeof(T) % 16 == 0;
  if (!a.vec && a.k * (int64_t)sizeof(T) * ROWS <= STAGE) {
    const int64_t groups = (a.m + ROWS - 1) / ROWS;
    quantize_staged_kernel<T, BITS, PRODUCT><<<(int)(groups < 8192 ? groups : 8192), 256, (int)mx_up(a.k * sizeof(T) * ROWS, 16), s>>>(x, a);
  } else {
    quantize_kernel<T, BITS, PRODUCT><<<grid_for(a.m * a.nb * 4), 256, 0, s>>>(x, a);
  }
}

template <class T, int BITS>
void run_dequantize(QuantArgs a, T* out, hipStream_t s) {
  a.vec = a.k * sizeof(T) % 16 == 0;
  if (!a.vec && a.k * (int64_t)sizeof(T) * ROWS <= STAGE) {
    const int64_t groups = (a.m + ROWS - 1) / ROWS;
    dequantize_staged_kernel<T, BITS><<<(int)(groups < 8192 ? groups : 8192), 256, (int)mx_up(a.k * sizeof(T) * ROWS, 16), s>>>(a, out);
  } else {
    dequantize_kernel<T, BITS><<<grid_for(a.m * a.nb * 4), 256, 0, s>>>(a, out);
  }
}

template <int BITS, bool PRODUCT = false>
int quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, hipStream_t s) {
  if (m < 0 || k < 1 || dtype < 0 || dtype > 2) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!x || !codes || !scales || ((uintptr_t)x & 15) || ((uintptr_t)codes & 15)) return FMD_EINVAL;
  const QuantArgs a{m, k, mx_blocks(k), 0, (uint32_t*)codes, (uint8_t*)scales};
  if (dtype == FMD_F32) run_quantize<float, BITS, PRODUCT>((const float*)x, a, s);
  else if (dtype == FMD_F16) run_quantize<_Float16, BITS, PRODUCT>((const _Float16*)x, a, s);
  else run_quantize<mx_bf16, BITS, PRODUCT>((const mx_bf16*)x, a, s);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

template <int BITS>
int dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype, hipStream_t s) {
  if (m < 0 || k < 1 || dtype < 0 || dtype > 2) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!out || !codes || !scales || ((uintptr_t)out & 15) || ((uintptr_t)codes & 15)) return FMD_EINVAL;
  const QuantArgs a{m, k, mx_blocks(k), 0, (uint32_t*)codes, (uint8_t*)scales};
  if (dtype == FMD_F32) run_dequantize<float, BITS>(a, (float*)out, s);
  else if (dtype == FMD_F16) run_dequantize<_Float16, BITS>(a, (_Float16*)out, s);
  else run_dequantize<mx_bf16, BITS>(a, (mx_bf16*)out, s);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

}  // namespace

int mx_quantize4_for_product(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, hipStream_t s) {
  return quantize<4, true>(x, dtype, m, k, codes, scales, s);
}

extern "C" int fmd_mxfp4_quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, void* stream) {
  return quantize<4>(x, dtype, m, k, codes, scales, fmd_stream(stream));
}
extern "C" int fmd_mxfp4_dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype,
                                    void* stream) {
  return dequantize<4>(codes, scales, m, k, out, dtype, fmd_stream(stream));
}
extern "C" int fmd_mxint8_quantize(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, void* stream) {
  return quantize<8>(x, dtype, m, k, codes, scales, fmd_stream(stream));
}
extern "C" int fmd_mxint8_dequantize(const void* codes, const void* scales, int64_t m, int64_t k, void* out, int dtype,
                                     void* stream) {
  return dequantize<8>(codes, scales, m, k, out, dtype, fmd_stream(stream));
}

// A few rows through a wide layer with 4-bit weights: y[m,n] = f(x^ W^T + b), m at most 64.
//
// All there is to do is to read the weights once, 17 bytes for 32 of them, so nothing may stand between the loads: a workgroup
// takes 16 rows of W whole, its eight waves every eighth run of four blocks, and each lane holds a block (16 bytes, one load)
// with its scale, four runs on their way at a time.  The 16 x 16 matrix instructions take a lane's block as it is: W's rows on
// one side, up to 16 rows of x on the other -- as 4-bit blocks that the lane quantises itself, or as bf16 planes against the
// weight's exact bf16 values.  Rows of x that do not exist cost matrix time that is free here.  The waves' sums meet in LDS and
// are added in a fixed order: one launch, no workspace.
//
// Bound by the latency of two rounds of loads: 4096 x 4096 for one row in 5.8 us (1.5 TB/s of weights) repeated in a graph, 7 to 8.5 by
// itself between other work.  Against the general product, us a call in a graph, bf16 x / x in 4 bits: 1 row of 1000 x 1000 4.1 / 4.1 and
// 13.5 / 10.6, of 4096 x 4096 5.8 / 6.0 and 38 / 14.5; 64 rows of 1000 x 1000 7.9 / 8.4 and 16.4 / 13.3, of 4096 x 4096 19.1 / 19.6 and
// 34.7 / 18.5: more rows are the product's.
#include "fmd_mx_host.h"

namespace {

constexpr int WAVES = 8;

struct RowsArgs {
  const void* x;
  const uint8_t *codes, *scales;
  MxEpilogue e;
  int m, n, k, nb, vec;
};

// 32 columns of a row of x as they lie in memory
template <class T>
struct Block {
  static constexpr int PER = 16 / sizeof(T), N = 32 / PER;
  u32x4 v[N];
  __device__ __forceinline__ void load(const RowsArgs& a, int row, int b) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = u32x4{0, 0, 0, 0};
    if (row >= a.m || b >= a.nb) return;
    const T* p = (const T*)a.x + (int64_t)row * a.k + b * 32;
    if (a.vec && b * 32 + 32 <= a.k) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = *(const u32x4*)(p + i * PER);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const bool there = b * 32 + i < a.k;  // the load itself is unconditional, of a value that exists
        const T* at = there ? p + i : p;
        if constexpr (sizeof(T) == 4) v[i / PER][i % PER] = there ? *(const uint32_t*)at : 0u;
        else v[i / PER][i % PER / 2] |= (there ? (uint32_t) * (const uint16_t*)at : 0u) << 16 * (i & 1);
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = v[i / PER][sizeof(T) == 4 ? i % PER : i % PER / 2];
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, u);
    else return MxType<T>::to(__builtin_bit_cast(T, (uint16_t)(u >> 16 * (i & 1))));
  }
};

template <class T, bool BOTH, int MT>
__global__ __launch_bounds__(64 * WAVES) void rows_kernel(const RowsArgs a) {
  constexpr int P = MxType<T>::planes, DEPTH = MT == 1 ? 4 : MT == 2 ? 2 : 1;
  __shared__ f32x4 lds[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, row = n0 + i;
  const int runs = (a.nb + 3) >> 2;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int r0 = wave; r0 < runs; r0 += WAVES * DEPTH) {
    u32x4 w[DEPTH];
    uint32_t s[DEPTH];
    constexpr bool AHEAD = MT == 1;  // x, too, before anything is waited for; more rows are read where they are used
    Block<T> x[AHEAD ? DEPTH : 1];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int b = (r0 + d * WAVES) * 4 + q;
      if constexpr (AHEAD) x[d].load(a, i, b);
      w[d] = u32x4{0, 0, 0, 0};
      s[d] = 0;
      if (row < a.n && b < a.nb) {
        w[d] = *(const u32x4*)(a.codes + ((int64_t)row * a.nb + b) * 16);
        s[d] = a.scales[(int64_t)row * a.nb + b];
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int b = (r0 + d * WAVES) * 4 + q;
      if (r0 + d * WAVES >= runs) break;  // the whole wave
      bf16x8 fw[4];
      if constexpr (!BOTH) {
        const float sv = mx_scale_value(s[d]);
        const int behind = a.k - b * 32;  // the codes behind the last column count as zeros whatever they are
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int valid = min(max(behind - 8 * g, 0), 8);
          fw[g] = __builtin_bit_cast(bf16x8, mx_bf16_from4(valid ? w[d][g] & (0xffffffffu >> (32 - 4 * valid)) : 0u, sv));
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float v[32];
        if constexpr (!AHEAD) x[0].load(a, t * 16 + i, b);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = x[AHEAD ? d : 0].get(e);
        if constexpr (BOTH) {
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 32; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
          const uint32_t byte = mx_scale_byte<4>(top);
          const float sv = byte == 255u ? 1.f : mx_scale_value(byte);
          i32x8 fx = {};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = v[8 * g + e];
            fx[g] = byte == 255u ? 0 : (int)mx_codes4(o, sv);
          }
          const i32x8 fw = {(int)w[d][0], (int)w[d][1], (int)w[d][2], (int)w[d][3], 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, acc[t], 4, 4, 0, (int)s[d], 0, (int)byte);
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = v[8 * g + e];
            u32x4 fx[P];
            mx_split8<P>(o, fx);
#pragma unroll
            for (int p = P - 1; p >= 0; --p)
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[g], __builtin_bit_cast(bf16x8, fx[p]), acc[t], 0, 0, 0);
          }
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) lds[wave][t][lane] = acc[t];
  __syncthreads();
  // lane (row of x, group of four rows of W) of each tile: one output a thread
  for (int o = threadIdx.x; o < MT * 256; o += 64 * WAVES) {
    const int t = o >> 8, m = t * 16 + ((o >> 4) & 15), c = o & 15, n = n0 + c;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += ((const float*)&lds[w][t][((c >> 2) << 4) + ((o >> 4) & 15)])[c & 3];
    if (m >= a.m || n >= a.n) continue;
    if (a.e.bias) v += MxType<T>::to(((const T*)a.e.bias)[n]);
    const int64_t at = (int64_t)m * a.n + n;
    if (a.e.tanh) {
      const float t = mx_sigma(v);
      if (a.e.dact) ((mx_dact*)a.e.dact)[at] = MxType<mx_dact>::from(mx_keep_dtanh_of(t));
      v = mx_tanh(v, t);
    }
    ((T*)a.e.out)[at] = MxType<T>::from(v);
  }
}

template <class T, bool BOTH>
int run(RowsArgs a, hipStream_t s) {
  a.vec = ((uintptr_t)a.x & 15) == 0 && a.k * sizeof(T) % 16 == 0;
  const int grid = (a.n + 15) / 16;
  if (a.m <= 16) rows_kernel<T, BOTH, 1><<<grid, 64 * WAVES, 0, s>>>(a);
  else if (a.m <= 32) rows_kernel<T, BOTH, 2><<<grid, 64 * WAVES, 0, s>>>(a);
  else rows_kernel<T, BOTH, 4><<<grid, 64 * WAVES, 0, s>>>(a);
  return hipGetLastError() == hipSuccess ? FMD_OK : FMD_ELAUNCH;
}

template <class T>
int run(const RowsArgs& a, bool both, hipStream_t s) {
  return both ? run<T, true>(a, s) : run<T, false>(a, s);
}

}  // namespace

bool mx_rows_fits(int64_t m) { return m <= 64; }

int mx_rows(const void* x, int dtype, const void* codes, const void* scales, bool both, int64_t m, int64_t n, int64_t k,
            const MxEpilogue& e, hipStream_t s) {
  const RowsArgs a{x, (const uint8_t*)codes, (const uint8_t*)scales, e, (int)m, (int)n, (int)k, (int)mx_blocks(k), 0};
  if (dtype == FMD_F32) return run<float>(a, both, s);
  if (dtype == FMD_F16) return run<_Float16>(a, both, s);
  return run<mx_bf16>(a, both, s);
}

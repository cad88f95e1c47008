// Weight and bias gradients: gw[k,n] = sum over rows p(x8)[.,k] g[.,n], gb[n] = sum g[.,n], x8 in 8-bit blocks.
//
// gradient_kernel, for narrow layers (k and n at most 256, in parts of 128 x 128) over many rows.  The contraction runs over the
// rows, so a matrix fragment wants 8 rows of one column in a lane.  Lane i of a half wave takes columns NT*i .. NT*i+NT-1 of g (one
// 16-byte load a row) and KT*i .. of the checkpoint; over 8 rows that is one fragment for each of its columns, with no
// transposition through LDS: which matrix column a lane stands for is free, and the result is stored back in the same order.  A
// wave holds all of gw in its accumulators (up to 128 x 128: 256 of a lane's 512 registers, one wave a SIMD) and takes 16 rows a
// step, the next step's rows already on their way.  The waves of a workgroup add up in LDS, the workgroups in a second kernel, in a
// fixed order.  Bound by reading g and the checkpoint once: 262144 x 128 x 128 fp32 under tanh in 116 us, 1.5 TB/s (the 6 products of
// a term and the tanh come on top of the bytes), bf16 92 us, the sums' kernel included.
//
// gradient_tile_kernel, for few rows and any width.  A workgroup makes one 32 x 32 tile of gw from a slice of the rows; its eight
// waves take 16 rows each in turn.  g and the checkpoint are read once for every tile beside or below, from the caches, but a
// few rows spread over many workgroups, and a workgroup has 16 sums a lane to bring together instead of 256.  Bound by latency while
// the rows are few (269 x 128 x 128 fp32: 5.7 us), by those reads later.
#include <type_traits>

#include "fmd_mx_host.h"

namespace {

constexpr int WAVES = 4;
constexpr uint32_t NOWHERE = 0x40000000u;  // behind the end of every descriptor: 16 rows of at most 2^20 fp32 are 2^26 bytes
typedef __amdgpu_buffer_rsrc_t Rows;

struct GradArgs {
  const void* g;
  const uint8_t *codes, *scales;
  float* part;  // [slice][32 KT + 1][32 NT]; the last row: bias
  int64_t m;
  int k, n, nb, vec;  // of gw's part that a launch makes (nb: of all columns)
  int ld, n0, block0;  // columns of g; the part's first column and block of the checkpoint
};

__device__ __forceinline__ Rows rows_of(const void* p, int64_t row0, int64_t m, int row_bytes) {
  const int64_t left = m - row0;
  const int n = left < 16 ? (left > 0 ? (int)left : 0) : 16;
  return __builtin_amdgcn_make_buffer_rsrc((char*)p + row0 * row_bytes, 0, n * row_bytes, 0x00020000);
}

// workgroups a CU: two where half the registers are enough
template <class T, int KT> constexpr int PER_CU = sizeof(T) == 2 && KT == 2 ? 2 : 1;

// planes of p(x8): one holds the 8 bits themselves, their tanh is not rounded to bf16 first (193688 x 128 x 128 bf16 168 us a call either
// way, 500 x 1000 x 1000 87 against 89)
template <class T, bool TANH> constexpr int KEPT_PLANES = !TANH ? 1 : MxType<T>::planes < 2 ? 2 : MxType<T>::planes;

template <class T, bool TANH, int KT, int NT>
__global__ __launch_bounds__(64 * WAVES, (PER_CU<T, KT>)) void gradient_kernel(const GradArgs a) {
  constexpr int PA = KEPT_PLANES<T, TANH>, PB = MxType<T>::planes, TOP = PA > PB ? PA : PB, S = sizeof(T);
  constexpr int W = NT * S / 4;                    // dwords of a lane's columns in a row of g
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 31, h = lane >> 5;
  const int k0 = KT * j, n0 = NT * j;
  const int steps = (int)((a.m + 15) >> 4), stride = gridDim.x * WAVES;  // m is at most 2^34

  uint32_t g_raw[8][W], s_raw[8];
  uint32_t c_raw[8];
  const int block = a.block0 + (k0 >> 5);
  const bool kept = a.codes && k0 < a.k && block < a.nb;  // the bias's gradient alone needs no checkpoint
  const uint32_t c_off = kept ? (uint32_t)((8 * h * a.nb + a.block0) * 32 + k0) : NOWHERE;
  const uint32_t s_off = kept ? (uint32_t)(8 * h * a.nb + block) : NOWHERE;
  auto fetch = [&](int step) {
    const int64_t row0 = (int64_t)step * 16;
    const Rows g = rows_of(a.g, row0, a.m, a.ld * S), c = rows_of(a.codes, row0, a.m, a.nb * 32), s = rows_of(a.scales, row0, a.m, a.nb);
    const int gs = mx_here(a.ld * S), nbs = mx_here(a.nb);
    const uint32_t at = (uint32_t)(8 * h * a.ld + a.n0 + n0) * S;
    if (a.vec) {
      const uint32_t off = n0 < a.n ? at : NOWHERE;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if constexpr (W == 4) *(u32x4*)g_raw[r] = __builtin_amdgcn_raw_buffer_load_b128(g, off + r * gs, 0, 0);
        else if constexpr (W == 2) *(u32x2*)g_raw[r] = __builtin_amdgcn_raw_buffer_load_b64(g, off + r * gs, 0, 0);
        else g_raw[r][0] = __builtin_amdgcn_raw_buffer_load_b32(g, off + r * gs, 0, 0);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if constexpr (S == 4) {
            g_raw[r][w] = __builtin_amdgcn_raw_buffer_load_b32(g, n0 + w < a.n ? at + 4 * w + r * gs : NOWHERE, 0, 0);
          } else {
            const uint32_t lo = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(g, n0 + 2 * w < a.n ? at + 4 * w + r * gs : NOWHERE, 0, 0);
            const uint32_t hi = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(g, n0 + 2 * w + 1 < a.n ? at + 4 * w + 2 + r * gs : NOWHERE, 0, 0);
            g_raw[r][w] = lo | hi << 16;
          }
        }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (KT == 4) c_raw[r] = __builtin_amdgcn_raw_buffer_load_b32(c, c_off + r * 32 * nbs, 0, 0);
      else c_raw[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(c, c_off + r * 32 * nbs, 0, 0);
      s_raw[r] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(s, s_off + r * nbs, 0, 0);
    }
  };
  auto g_value = [&](int r, int t) {
    if constexpr (S == 4) return __builtin_bit_cast(float, g_raw[r][t]);
    else if constexpr (std::is_same<T, mx_bf16>::value)
      return __builtin_bit_cast(float, t & 1 ? g_raw[r][t >> 1] & 0xffff0000u : g_raw[r][t >> 1] << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(g_raw[r][t >> 1] >> 16 * (t & 1)));
  };

  f32x16 acc[KT][NT];
  float bias[NT] = {};
#pragma unroll
  for (int i = 0; i < KT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][t][r] = 0.f;

  int step = wave * gridDim.x + blockIdx.x;
  if (step < steps) fetch(step);
  for (; step < steps; step += stride) {
    u32x4 fa[KT][PA], fb[NT][PB];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float x = mx_value8((int)(int8_t)(c_raw[r] >> 8 * i), s_raw[r]);
        v[r] = TANH ? mx_tanh(x) : x;
      }
      mx_split8<PA>(v, fa[i]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = g_value(r, t);
      mx_split8<PB>(v, fb[t]);
      bias[t] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    if (step + stride < steps) fetch(step + stride);
#pragma unroll
    for (int sum = TOP - 1; sum >= 0; --sum)
#pragma unroll
      for (int p = 0; p < PA; ++p)
        if (sum - p >= 0 && sum - p < PB)
#pragma unroll
          for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              acc[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa[i][p]),
                                                                  __builtin_bit_cast(bf16x8, fb[t][sum - p]), acc[i][t], 0, 0, 0);
  }

  // the waves add up in LDS, one after the other: [register][lane], then the bias
  constexpr int REGS = KT * NT * 16;
  for (int w = 0; w < WAVES; ++w) {
    if (wave == w) {
      float* mine = lds + lane;
#pragma unroll
      for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          // keeps the 256 sums of a full tile where they are: the compiler would copy all of them out before the loop
          // (the nops: a matrix result is read at the earliest 18 states after its instruction)
          if constexpr (KT * NT == 16) asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[i][t]));
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float* to = mine + ((i * NT + t) * 16 + r) * 64;
            *to = w ? *to + acc[i][t][r] : acc[i][t][r];
          }
          __builtin_amdgcn_sched_barrier(0);  // a tile at a time, or the compiler holds all of them twice
        }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float v = fmd_xor32_sum(bias[t]);
        float* to = lds + REGS * 64 + n0 + t;
        if (h == 0) *to = w ? *to + v : v;
      }
    }
    __syncthreads();
  }
  float* part = a.part + (int64_t)blockIdx.x * (32 * KT + 1) * (32 * NT);
  for (int at = threadIdx.x; at < 32 * KT * 32 * NT; at += 64 * WAVES) {
    const int k = at / (32 * NT), n = at % (32 * NT), i = k % KT, row = k / KT, t = n % NT;
    part[at] = lds[((i * NT + t) * 16 + (row & 3) + 4 * (row >> 3)) * 64 + 32 * (row >> 2 & 1) + n / NT];
  }
  if (threadIdx.x < 32 * NT) part[32 * KT * 32 * NT + threadIdx.x] = lds[REGS * 64 + threadIdx.x];
}

constexpr int TILE_WAVES = 8;

template <class T, bool TANH>
__global__ __launch_bounds__(64 * TILE_WAVES) void gradient_tile_kernel(const GradArgs a, T* __restrict__ gw, T* __restrict__ gb) {
  constexpr int PA = KEPT_PLANES<T, TANH>, PB = MxType<T>::planes, TOP = PA > PB ? PA : PB, S = sizeof(T);
  __shared__ float lds[TILE_WAVES][17][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 31, h = lane >> 5;
  const int block = blockIdx.x, k = block * 32 + j, n = blockIdx.y * 32 + j;  // 32 columns of the checkpoint: one block
  const int steps = (int)((a.m + 15) >> 4), stride = gridDim.z * TILE_WAVES;

  uint32_t g_raw[8], c_raw[8], s_raw[8];
  const uint32_t g_off = n < a.n ? (uint32_t)(8 * h * a.n + n) * S : NOWHERE;
  const uint32_t c_off = a.codes ? (uint32_t)(8 * h * a.nb * 32 + k) : NOWHERE, s_off = a.codes ? (uint32_t)(8 * h * a.nb + block) : NOWHERE;
  auto fetch = [&](int step) {
    const int64_t row0 = (int64_t)step * 16;
    const Rows g = rows_of(a.g, row0, a.m, a.n * S), c = rows_of(a.codes, row0, a.m, a.nb * 32), s = rows_of(a.scales, row0, a.m, a.nb);
    const int gs = mx_here(a.n * S), nbs = mx_here(a.nb);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (S == 4) g_raw[r] = __builtin_amdgcn_raw_buffer_load_b32(g, g_off + r * gs, 0, 0);
      else g_raw[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(g, g_off + r * gs, 0, 0);
      c_raw[r] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(c, c_off + r * 32 * nbs, 0, 0);
      s_raw[r] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(s, s_off + r * nbs, 0, 0);
    }
  };
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  float bias = 0.f;
  int step = blockIdx.z * TILE_WAVES + wave;
  if (step < steps) fetch(step);
  for (; step < steps; step += stride) {
    u32x4 fa[PA], fb[PB];
    float v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float x = mx_value8((int)(int8_t)c_raw[r], s_raw[r]);
      v[r] = TANH ? mx_tanh(x) : x;
    }
    mx_split8<PA>(v, fa);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (S == 4) v[r] = __builtin_bit_cast(float, g_raw[r]);
      else v[r] = MxType<T>::to(__builtin_bit_cast(T, (uint16_t)g_raw[r]));
    }
    mx_split8<PB>(v, fb);
    bias += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    if (step + stride < steps) fetch(step + stride);
#pragma unroll
    for (int sum = TOP - 1; sum >= 0; --sum)
#pragma unroll
      for (int p = 0; p < PA; ++p)
        if (sum - p >= 0 && sum - p < PB)
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa[p]), __builtin_bit_cast(bf16x8, fb[sum - p]), acc, 0,
                                                        0, 0);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) lds[wave][r][lane] = acc[r];
  lds[wave][16][lane] = bias;
  __syncthreads();
  // (register, lane) of the tile: row of gw 8 (r >> 2) + 4 h + (r & 3), column j; r = 16: the bias, halves to be added
  float* part = a.part ? a.part + (int64_t)blockIdx.z * (a.k + 1) * a.n : nullptr;
  for (int o = threadIdx.x; o < 17 * 64; o += 64 * TILE_WAVES) {
    const int r = o >> 6, l = o & 63, col = blockIdx.y * 32 + (l & 31);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < TILE_WAVES; ++w) v += lds[w][r][l];
    if (r == 16) {
      v = fmd_xor32_sum(v);  // one wave holds this row
      if (block || l >= 32 || col >= a.n) continue;
      if (part) part[a.k * a.n + col] = v;
      else if (gb) gb[col] = MxType<T>::from(v);
    } else {
      const int row = block * 32 + (r & 3) + 8 * (r >> 2) + 4 * (l >> 5);
      if (row >= a.k || col >= a.n) continue;
      if (part) part[row * a.n + col] = v;
      else if (gw) gw[(int64_t)row * a.n + col] = MxType<T>::from(v);
    }
  }
}

// gw and gb from the slices: 16 outputs a workgroup, 16 groups of slices each, added in a fixed order
template <class T>
__global__ __launch_bounds__(256) void gradient_sum_kernel(const float* __restrict__ part, int slices, int rows, int pitch, int k, int n, int ld,
                                                           T* __restrict__ gw, T* __restrict__ gb) {
  __shared__ float lds[16][17];
  const int at = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
  const int row = at / n, col = at - row * n;  // row k: the bias
  const bool want = row < k ? gw != nullptr : row == k && gb != nullptr;
  float v = 0.f;
  if (want) {
    const float* p = part + (int64_t)(row < k ? row : rows) * pitch + col;
    const int64_t slice = (int64_t)(rows + 1) * pitch;
    const int s1 = slices * (q + 1) / 16;
#pragma unroll 8
    for (int s = slices * q / 16; s < s1; ++s) v += p[s * slice];
  }
  lds[q][threadIdx.x & 15] = v;
  __syncthreads();
  if (q == 0 && want) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += lds[i][threadIdx.x];
    if (row < k) gw[(int64_t)row * ld + col] = MxType<T>::from(v);
    else gb[col] = MxType<T>::from(v);
  }
}

template <class T, bool TANH, int KT, int NT>
int launch(const GradArgs& a, int slices, hipStream_t s) {
  constexpr int bytes = (KT * NT * 16 * 64 + 32 * NT) * 4;
  static_assert(bytes * PER_CU<T, KT> <= 160 * 1024, "LDS of a CU");
  if (mx_allow_lds(&gradient_kernel<T, TANH, KT, NT>, bytes) != hipSuccess) return FMD_ELAUNCH;
  gradient_kernel<T, TANH, KT, NT><<<slices, 64 * WAVES, bytes, s>>>(a);
  return hipGetLastError() == hipSuccess ? FMD_OK : FMD_ELAUNCH;
}

template <class T, bool TANH>
int by_width(const GradArgs& a, int slices, hipStream_t s) {
  if (a.k <= 64) return a.n <= 64 ? launch<T, TANH, 2, 2>(a, slices, s) : launch<T, TANH, 2, 4>(a, slices, s);
  return a.n <= 64 ? launch<T, TANH, 4, 2>(a, slices, s) : launch<T, TANH, 4, 4>(a, slices, s);
}

// part by part of at most 128 x 128, one after the other in the same workspace.  The bias's sums come with the first parts along k; for
// them alone (the same bits as beside gw) the others are left out
template <class T>
int run(GradArgs a, bool tanh, int slices, void* gw, void* gb, hipStream_t s) {
  const int k = a.k, n = a.n;
  for (int k0 = 0; k0 < (gw ? k : 1); k0 += 128)
    for (int n0 = 0; n0 < n; n0 += 128) {
      a.k = k - k0 < 128 ? k - k0 : 128, a.n = n - n0 < 128 ? n - n0 : 128, a.n0 = n0, a.block0 = k0 / 32;
      const int nt = a.n <= 64 ? 2 : 4, rows = a.k <= 64 ? 64 : 128;
      a.vec = ((uintptr_t)a.g & 15) == 0 && a.n % nt == 0 && n % nt == 0;
      const int rc = tanh ? by_width<T, true>(a, slices, s) : by_width<T, false>(a, slices, s);
      if (rc != FMD_OK) return rc;
      gradient_sum_kernel<T><<<((a.k + 1) * a.n + 15) / 16, 256, 0, s>>>(a.part, slices, rows, 32 * nt, a.k, a.n, n,
                                                                         gw ? (T*)gw + (int64_t)k0 * n + n0 : nullptr,
                                                                         gb && k0 == 0 ? (T*)gb + n0 : nullptr);
      if (hipGetLastError() != hipSuccess) return FMD_ELAUNCH;
    }
  return FMD_OK;
}

// workgroups along the rows: one step of 16 rows for each wave at least, what fits the chip at once at most
int slices_for(int dtype, int64_t m, int64_t k) {
  const int64_t s = (m + 16 * WAVES - 1) / (16 * WAVES), most = k <= 64 && dtype != FMD_F32 ? 512 : 256;  // of the first part, the largest
  return (int)(s < most ? s : most);
}

// Which kernel: a tile at a time while the rows are few; it reads a narrow layer's rows once for each 32 columns of the other side,
// the parts' kernel once for each 128, and general products write both operands anew.  Tiles against the other, us, tanh, with sums:
//   narrow: 1000 x 128 x 128 fp32 8.1 / 50, 65536 fp32 46 / 70, 98304 71 / 77 (bf16 55 / 67), 131072 85 / 85 (bf16 70 / 72), 262144
//           160 / 117 (bf16 135 / 92); 98304 x 256 x 200 264 / 306, x 64 x 256 64 / 60
//   wide:   500 x 1000 x 1000 fp32 23 / 41 (bf16 17 / 29), 1000 40 / 48 (30 / 34), 2000 75 / 63 (56 / 39); 64 x 1024 x 4096 bf16 15 / 16,
//           128 21 / 18, 300 36 / 21; 5000 x 300 x 300 32 / 58
constexpr int64_t FEW = 98304, FEW_PRODUCTS = (int64_t)1 << 29;
bool by_tiles(int64_t m, int64_t n, int64_t k) { return k <= 256 && n <= 256 ? m <= FEW : m * n <= FEW_PRODUCTS / k; }
// Rows in parts: two steps of 16 for each wave at least, and none up to 512 rows, where the sum over parts is a launch too many (400 x
// 128 x 128 fp32: 7.1 in one, 8.0 in two; 1000: 13.6 in one, 8.0 in four)
int tile_slices(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = ((k + 31) / 32) * ((n + 31) / 32), s = (m + 32 * TILE_WAVES - 1) / (32 * TILE_WAVES), most = (512 + tiles - 1) / tiles;
  return (int)(m <= 512 ? 1 : s < most ? s : most);
}

template <class T>
int run_tiles(GradArgs a, bool tanh, void* gw, void* gb, hipStream_t s) {
  const int slices = tile_slices(a.m, a.n, a.k);
  if (slices == 1) a.part = nullptr;
  const dim3 grid(gw ? (a.k + 31) / 32 : 1, (a.n + 31) / 32, slices);  // the bias's sums are the first block's
  if (tanh) gradient_tile_kernel<T, true><<<grid, 64 * TILE_WAVES, 0, s>>>(a, (T*)gw, (T*)gb);
  else gradient_tile_kernel<T, false><<<grid, 64 * TILE_WAVES, 0, s>>>(a, (T*)gw, (T*)gb);
  if (slices > 1) gradient_sum_kernel<T><<<((a.k + 1) * a.n + 15) / 16, 256, 0, s>>>(a.part, slices, a.k, a.n, a.k, a.n, a.n, (T*)gw, (T*)gb);
  return hipGetLastError() == hipSuccess ? FMD_OK : FMD_ELAUNCH;
}

}  // namespace

bool mx_gradient_fits(int64_t m, int64_t n, int64_t k) { return (k <= 256 && n <= 256) || by_tiles(m, n, k); }

int64_t mx_gradient_bytes(int dtype, int64_t m, int64_t n, int64_t k) {
  if (by_tiles(m, n, k)) return tile_slices(m, n, k) > 1 ? (int64_t)tile_slices(m, n, k) * (k + 1) * n * 4 : 0;
  return (int64_t)slices_for(dtype, m, k) * ((k <= 64 ? 64 : 128) + 1) * (n <= 64 ? 64 : 128) * 4;
}

int mx_gradient(const void* g, const uint8_t* codes, const uint8_t* scales, bool tanh, int dtype, int64_t m, int64_t n, int64_t k,
                void* gw, void* gb, void* workspace, hipStream_t s) {
  const GradArgs a{g, codes, scales, (float*)workspace, m, (int)k, (int)n, (int)mx_blocks(k), 0, (int)n, 0, 0};
  if (by_tiles(m, n, k)) {
    if (dtype == FMD_F32) return run_tiles<float>(a, tanh, gw, gb, s);
    if (dtype == FMD_F16) return run_tiles<_Float16>(a, tanh, gw, gb, s);
    return run_tiles<mx_bf16>(a, tanh, gw, gb, s);
  }
  const int slices = slices_for(dtype, m, k);
  if (dtype == FMD_F32) return run<float>(a, tanh, slices, gw, gb, s);
  if (dtype == FMD_F16) return run<_Float16>(a, tanh, slices, gw, gb, s);
  return run<mx_bf16>(a, tanh, slices, gw, gb, s);
}

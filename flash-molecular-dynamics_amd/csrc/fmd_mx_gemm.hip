// The general product of block-scaled layers: any sizes, any type.
//
//   1. lay the operands out as K-contiguous rows of 128-byte tiles: bf16 planes (fmd_mx.h) for 32- and 16-bit operands and
//      for 8-bit checkpoints, the 4-bit codes themselves where both operands are in 4 bits
//   2. C = A B^T on the matrix cores, tile by tile
//   3. where the rows of C are too few to fill the chip, the contraction is split and the parts are summed in a fixed order
//
// The transforms (tanh, the gradient's tanh', dequantisation) happen in step 1, once per element, or in the epilogue.
//
// 8192 x 8192 x 4096 in 150 us from 4-bit operands (3.7 PF), matrix pipe busy 48 % of the time, no bank conflicts, waves waiting 45 % of
// theirs: the barrier of each tile, where its loads have to have landed, bounds it.  bf16 8192 x 1024 x 4096, with the small tile, in 101 us
// (0.68 PF, matrix pipe 51 %); bf16 4096 x 4096 x 4096 against 4-bit weights in 126 us (1.09 PF), the planes' kernels included.
#include <type_traits>

#include "fmd_mx_host.h"

namespace {

// =====================================================================================================================
// operand sources: eight neighbouring columns of one row as fp32
// =====================================================================================================================
template <class T, bool TANH>
struct SrcDense {
  const T* p;
  int64_t cols;
  bool vec;
  __device__ __forceinline__ void load(int64_t row, int64_t c0, float (&v)[8]) const {
    const T* r = p + row * cols;
    if (vec && c0 + 8 <= cols) {
      T t[8];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((u32x4*)t)[i] = *(const u32x4*)(r + c0 + i * (16 / sizeof(T)));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = MxType<T>::to(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? MxType<T>::to(r[c0 + i]) : 0.f;
    }
    if constexpr (TANH)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx_tanh(v[i]);  // tanh(0) = 0: padding stays zero
  }
};
// a gradient times the derivative of the activation behind it.  AUX 1: aux = y in fp32, factor 1 - y^2; 2: aux = the factor as mx_dact
template <class T, int AUX>
struct SrcGrad {
  const T* p;
  const void* aux;
  int64_t cols;
  bool vec;
  __device__ __forceinline__ void load(int64_t row, int64_t c0, float (&v)[8]) const {
    SrcDense<T, false>{p, cols, vec}.load(row, c0, v);
    if constexpr (AUX == 1) {
      float y[8];
      SrcDense<float, false>{(const float*)aux, cols, vec}.load(row, c0, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= 1.f - y[i] * y[i];
    } else if constexpr (AUX == 2) {
      float d[8];
      SrcDense<mx_dact, false>{(const mx_dact*)aux, cols, vec}.load(row, c0, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= d[i];
    }
  }
};
// 8-bit checkpoint; codes [row][32 nb] are padded with zeros
template <bool TANH>
struct SrcI8 {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t cols, nb;
  __device__ __forceinline__ void load(int64_t row, int64_t c0, float (&v)[8]) const {
    if (c0 >= cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      return;
    }
    const u32x2 c = *(const u32x2*)(codes + (row * nb) * 32 + c0);
    const uint32_t byte = scales[row * nb + (c0 >> 5)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = mx_value8((int)(int8_t)(c[i >> 2] >> (8 * (i & 3))), byte);
      v[i] = c0 + i < cols ? (TANH ? mx_tanh(x) : x) : 0.f;
    }
  }
};
struct SrcFp4 {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t cols, nb;
  __device__ __forceinline__ void load(int64_t row, int64_t c0, float (&v)[8]) const {
    if (c0 >= cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      return;
    }
    const uint32_t c = *(const uint32_t*)(codes + (row * nb) * 16 + (c0 >> 1));
    const u32x4 b = mx_bf16_from4(c, mx_scale_value(scales[row * nb + (c0 >> 5)]));
#pragma unroll
    for (int i = 0; i < 8; ++i)  // columns behind the last one hold whatever the caller's codes hold there
      v[i] = c0 + i < cols ? __builtin_bit_cast(float, i & 1 ? b[i >> 1] & 0xffff0000u : b[i >> 1] << 16) : 0.f;
  }
};

// rows x cols -> planes [P][rows][pad] (pad = cols rounded up to 64, zeros behind cols)
template <class S, int P>
__global__ __launch_bounds__(256) void planes_kernel(S src, int64_t rows, int64_t pad, uint16_t* __restrict__ out) {
  const int64_t per = pad >> 3, total = rows * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / per, c0 = (t - row * per) * 8;
    float v[8];
    src.load(row, c0, v);
    constexpr int N = P ? P : 1;
    u32x4 o[N];
    mx_split8<P>(v, o);
#pragma unroll
    for (int p = 0; p < N; ++p) *(u32x4*)(out + (int64_t)p * rows * pad + row * pad + c0) = o[p];
  }
}

// the same of p(x), and x in 8-bit blocks (four neighbouring lanes hold a block and are active together: pad is a multiple of 64)
template <class T, bool TANH, int P>
__global__ __launch_bounds__(256) void planes_keep_kernel(SrcDense<T, false> src, int64_t rows, int64_t pad, uint16_t* __restrict__ out,
                                                          int64_t nb, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t per = pad >> 3, total = rows * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / per, q = t - row * per, b = q >> 2;
    float v[8];
    src.load(row, q * 8, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    const uint32_t byte = mx_scale_byte<8>(top);
    if (b < nb) {
      *(u32x2*)(codes + (row * nb + b) * 32 + (q & 3) * 8) =
          u32x2{mx_codes8(v[0], v[1], v[2], v[3], byte), mx_codes8(v[4], v[5], v[6], v[7], byte)};
      if ((q & 3) == 0) scales[row * nb + b] = (uint8_t)byte;
    }
    if constexpr (TANH)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx_tanh(v[i]);
    constexpr int N = P ? P : 1;
    u32x4 o[N];
    mx_split8<P>(v, o);
#pragma unroll
    for (int p = 0; p < N; ++p) *(u32x4*)(out + (int64_t)p * rows * pad + row * pad + q * 8) = o[p];
  }
}

// rows x cols -> planes [P][cols][pad] of the transposed matrix (pad = rows rounded up to 64, zeros behind rows); 64 x 64 tiles
// through LDS, rows 66 halves apart so that neither side meets a bank twice more than it has to
template <class S, int P>
__global__ __launch_bounds__(256) void planes_t_kernel(S src, int64_t rows, int64_t cols, int64_t pad, uint16_t* __restrict__ out) {
  constexpr int N = P ? P : 1;
  __shared__ uint32_t tile[N][64][33];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (t >> 3) + 32 * i, c = (t & 7) * 8;
    float v[8];
    if (r0 + r < rows) {
      src.load(r0 + r, c0 + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    u32x4 o[N];
    mx_split8<P>(v, o);
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[p][r][(c >> 1) + j] = o[p][j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = (t >> 3) + 32 * i, r = (t & 7) * 8;
    if (c0 + c >= cols) continue;
#pragma unroll
    for (int p = 0; p < N; ++p) {
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = tile[p][r + 2 * j][c >> 1], hi = tile[p][r + 2 * j + 1][c >> 1];
        o[j] = c & 1 ? __builtin_amdgcn_perm(hi, lo, 0x07060302u) : __builtin_amdgcn_perm(hi, lo, 0x05040100u);
      }
      *(u32x4*)(out + ((int64_t)p * cols + c0 + c) * pad + r0 + r) = o;
    }
  }
}

// scales [rows][nb] -> [tile of 8 blocks][half][row][4], zeros behind nb: block 2 s + half of a tile is byte s, what one half of a wave
// needs in the four steps of a tile
__global__ __launch_bounds__(256) void scale_tiles_kernel(const uint8_t* __restrict__ s, int64_t rows, int64_t pad, int64_t nb, int64_t kt,
                                                          uint32_t* __restrict__ out) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < rows * kt * 2; t += (int64_t)gridDim.x * 256) {
    const int64_t q = t / rows, row = t - q * rows;
    uint32_t v = 0;
    for (int i = 0; i < 4; ++i) {
      const int64_t b = (q >> 1) * 8 + 2 * i + (q & 1);
      if (b < nb) v |= (uint32_t)s[row * nb + b] << (8 * i);
    }
    out[q * pad + row] = v;
  }
}

// =====================================================================================================================
// C[m,n] = epi(A B^T + bias): BM x BN tiles, TM x TN matrix tiles of 32 x 32 per wave, K tiles of 128 bytes a row
// (64 bf16 or 256 4-bit elements), two LDS buffers filled by direct loads one tile ahead.
//
// LDS: lines of two rows, 16 slots of 16 bytes (all 64 banks).  Granule q of row r is in slot ((r & 1) * 8 + q) ^ ((r / T) & 15) of
// line r / 2, T (even) the matrix tiles per wave in that direction: the 32 lanes of a fragment read rows T*lane + t, so 16
// neighbouring lanes meet 16 different slots.  That row order also gives a lane T neighbouring columns of C.  (With the two rows
// of a line swizzled apart, half the banks served a read: 4 conflict cycles on 4.)
// =====================================================================================================================
struct GemmArgs {
  const char *a, *b;
  int64_t a_plane, b_plane, a_pitch, b_pitch;  // bytes
  const char *sa, *sb;                         // 4-bit operands: scales [tile][half][row][4]
  int m, n, kt, granules, tiles_m, tiles_n, splits, npairs;
  uint32_t pa, pb;                             // planes of pair i: bits 2i, 2i+1
  MxEpilogue e;
  float* partial;  // [splits][m][n], or null: the epilogue writes C
};

template <class T>
__device__ __forceinline__ void finish_one(const MxEpilogue& e, int64_t row, int64_t col, int64_t ld, float v) {
  if (e.bias) v += MxType<T>::to(((const T*)e.bias)[col]);
  if (e.tanh) {
    const float t = mx_sigma(v);
    if (e.dact) ((mx_dact*)e.dact)[row * ld + col] = MxType<mx_dact>::from(mx_keep_dtanh_of(t));
    v = mx_tanh(v, t);
  }
  if (e.codes8) v = mx_times_dtanh(v, (int)(int8_t)e.codes8[row * e.nb8 * 32 + col], e.scales8[row * e.nb8 + (col >> 5)]);
  ((T*)e.out)[row * ld + col] = MxType<T>::from(v);
}

enum { FMT_BF16, FMT_FP4, FMT_F16 };

template <class T, int FMT, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(64 * WM * WN) void gemm_kernel(const GemmArgs g) {
  constexpr bool FP4 = FMT == FMT_FP4;
  static_assert(TM % 2 == 0 && TN % 2 == 0, "two rows of a line belong to one lane");
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NW = WM * WN, SLOTS = (BM + BN) * 8, LOADS = SLOTS / (64 * NW);
  __shared__ __attribute__((aligned(16))) char lds[2 * (BM + BN) * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  // one XCD gets a run of neighbouring tiles (workgroups are dealt to the eight XCDs in turn), eight tile rows at a time
  int bid = blockIdx.x;
  const int tiles = g.tiles_m * g.tiles_n;
  if ((tiles & 7) == 0) bid = (bid & 7) * (tiles >> 3) + (bid >> 3);
  const int group = 8 * g.tiles_n, first = bid / group * 8, high = min(8, g.tiles_m - first);
  const int m0 = (first + bid % group % high) * BM, n0 = bid % group / high * BN;
  const int split = blockIdx.y;
  const int all = g.npairs * g.kt, begin = (int)((int64_t)all * split / g.splits), end = (int)((int64_t)all * (split + 1) / g.splits);

  // this wave's direct loads: byte offset of (row, granule) and the granule's number
  int64_t off[LOADS];
  int gran[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const bool is_a = (i * NW + wave) * 64 < BM * 8;  // uniform: BM * 8 is a multiple of 64
    const int slot = (i * NW + wave) * 64 + lane - (is_a ? 0 : BM * 8), line = slot >> 4;
    const int id = (slot & 15) ^ ((is_a ? 2 * line / TM : 2 * line / TN) & 15), rr = 2 * line + (id >> 3);
    gran[i] = id & 7;
    const int row = is_a ? min(m0 + rr, g.m - 1) : min(n0 + rr, g.n - 1);
    off[i] = (int64_t)row * (is_a ? g.a_pitch : g.b_pitch) + (FP4 ? 0 : gran[i] * 16);
  }
  auto issue = [&](int pair, int t, char* buf) {
    // 4-bit rows may end inside a tile: the granules behind stand for the last one again, under scales of 2^-127 on either side
    const char *pa = g.a + (FP4 ? 0 : (int64_t)t * 128), *pb = g.b + (FP4 ? 0 : (int64_t)t * 128);
    if constexpr (!FP4) pa += (g.pa >> 2 * pair & 3) * g.a_plane, pb += (g.pb >> 2 * pair & 3) * g.b_plane;
    auto direct = [&](int i, const char* src) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                       (__attribute__((address_space(3))) void*)(buf + (i * NW + wave) * 1024), 16, 0, 0);
    };
    auto place = [&](int i) { return ((i * NW + wave) * 64 < BM * 8 ? pa : pb) + off[i]; };
    // one straight line, so that the loads can be laid between the matrix instructions
#pragma unroll
    for (int i = 0; i < LOADS; ++i) direct(i, place(i) + (FP4 ? (uint32_t)min(t * 8 + gran[i], g.granules - 1) * 16 : 0));
  };
  f32x16 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

  // scales: the TM (TN) neighbouring rows of a lane, four steps each, in one load
  typedef uint32_t ScalesA __attribute__((ext_vector_type(TM)));
  typedef uint32_t ScalesB __attribute__((ext_vector_type(TN)));
  ScalesA sa_next;
  ScalesB sb_next;
  const int pad_m = (g.m + 3) & ~3, pad_n = (g.n + 3) & ~3;
  const int64_t off_sa = 4 * ((int64_t)h * pad_m + min(m0 + (wm * 32 + j) * TM, pad_m - TM));
  const int64_t off_sb = 4 * ((int64_t)h * pad_n + min(n0 + (wn * 32 + j) * TN, pad_n - TN));
  auto load_scales = [&](int t) {
    if constexpr (FP4) {
      sa_next = *(const ScalesA*)(g.sa + (int64_t)t * pad_m * 8 + off_sa);
      sb_next = *(const ScalesB*)(g.sb + (int64_t)t * pad_n * 8 + off_sb);
    }
  };
  ScalesA sa;
  ScalesB sb;
  auto take_scales = [&]() {
    if constexpr (FP4) sa = sa_next, sb = sb_next;
  };
  auto compute = [&](const char* buf, auto between) {  // between: what is done once the matrix unit has work
    const char* la = buf + (wm * 32 + j) * TM * 128;
    const char* lb = buf + BM * 128 + (wn * 32 + j) * TN * 128;
    // the fragments of the next step are read while this one's matrix instructions run
    u32x4 fa[2][TM], fb[2][TN];
    auto read = [&](int s) {
      const int q = s * 2 + h, at = (q ^ (j & 15)) * 16, odd = ((8 + q) ^ (j & 15)) * 16;
#pragma unroll
      for (int a = 0; a < TM; ++a) fa[s & 1][a] = *(const u32x4*)(la + (a >> 1) * 256 + (a & 1 ? odd : at));
#pragma unroll
      for (int b = 0; b < TN; ++b) fb[s & 1][b] = *(const u32x4*)(lb + (b >> 1) * 256 + (b & 1 ? odd : at));
    };
    read(0);
    // the compiler keeps this order: the next step's fragments on their way before a step's matrix instructions, no two of which in a
    // row add to the same sums; the next tile's loads amid the first step
#define MX_STEP(s, BETWEEN)                                                                                                 \
  {                                                                                                                         \
    if (s < 3) read(s + 1);                                                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                                      \
    _Pragma("unroll") for (int a = 0; a < TM; ++a) _Pragma("unroll") for (int b = 0; b < TN; ++b) {                         \
      const u32x4 ua = fa[s & 1][a], ub = fb[s & 1][b];                                                                     \
      if constexpr (FP4) {                                                                                                  \
        const i32x8 xa = {(int)ua[0], (int)ua[1], (int)ua[2], (int)ua[3], 0, 0, 0, 0};                                      \
        const i32x8 xb = {(int)ub[0], (int)ub[1], (int)ub[2], (int)ub[3], 0, 0, 0, 0};                                      \
        acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xa, xb, acc[a][b], 4, 4, s, (int)sa[a], s, (int)sb[b]); \
      } else if constexpr (FMT == FMT_F16) {                                                                                \
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, ua), __builtin_bit_cast(f16x8, ub),    \
                                                           acc[a][b], 0, 0, 0);                                             \
      } else {                                                                                                              \
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ua), __builtin_bit_cast(bf16x8, ub), \
                                                            acc[a][b], 0, 0, 0);                                            \
      }                                                                                                                     \
      if (a == TM / 2 - 1 && b == TN - 1) {                                                                                 \
        __builtin_amdgcn_sched_barrier(0);                                                                                  \
        BETWEEN;                                                                                                            \
        __builtin_amdgcn_sched_barrier(0);                                                                                  \
      }                                                                                                                     \
    }                                                                                                                       \
    __builtin_amdgcn_sched_barrier(0);                                                                                      \
  }
    MX_STEP(0, between())
    MX_STEP(1, ) MX_STEP(2, ) MX_STEP(3, )
#undef MX_STEP
  };

  int pair = begin / g.kt, t = begin - pair * g.kt, half = 0;
  if (begin < end) {
    issue(pair, t, lds);
    load_scales(t);
  }
  for (int it = begin; it < end; ++it) {
    // this tile has landed for every wave, and every wave is done with the other buffer
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    take_scales();
    compute(lds + half, [&]() {
      // behind the last tile the same one once more, into a buffer that nobody reads
      t += it + 1 < end;
      const int wrap = !FP4 && t == g.kt;  // 4-bit operands: one pair
      t = wrap ? 0 : t;
      pair += wrap;
      issue(pair, t, lds + ((BM + BN) * 128 - half));
      load_scales(t);
    });
    half = (BM + BN) * 128 - half;
  }
  __builtin_amdgcn_s_waitcnt(0);  // no load is left on its way into LDS when the workgroup ends

  // A lane's TN columns are neighbours: stored together where every row starts on a multiple of them.  Tiles that lie inside C are
  // stored without comparisons.
  const int64_t ld = g.n, col = n0 + (wn * 32 + j) * TN, row0 = m0 + (wm * 32 + 4 * h) * TM;
  auto epilogue = [&](auto inside_) {
    constexpr bool INSIDE = decltype(inside_)::value;
    auto row_of = [&](int a, int r) { return row0 + ((r & 3) + 8 * (r >> 2)) * TM + a; };
    auto write = [&](auto* p, const float (&v)[TN]) {  // p: (row, col) of the output
      using U = typename std::remove_reference<decltype(*p)>::type;
      if constexpr (INSIDE) {
        struct alignas(sizeof(U) * TN) Vec { U e[TN]; } o;
#pragma unroll
        for (int b = 0; b < TN; ++b) o.e[b] = MxType<U>::from(v[b]);
        *(Vec*)p = o;
      } else {
#pragma unroll
        for (int b = 0; b < TN; ++b)
          if (col + b < g.n) p[b] = MxType<U>::from(v[b]);
      }
    };
    auto each = [&](auto finish) {
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t row = row_of(a, r);
          if (!INSIDE && row >= g.m) continue;
          float v[TN];
#pragma unroll
          for (int b = 0; b < TN; ++b) v[b] = acc[a][b][r];
          finish(row * ld + col, v);
        }
    };
    if (g.partial) {
      float* const p = g.partial + (int64_t)split * g.m * ld;
      each([&](int64_t at, float (&v)[TN]) { write(p + at, v); });
    } else if (g.e.codes8) {
#pragma unroll
      for (int a = 0; a < TM; ++a) {
        // the checkpoint's values of 16 rows before any of them is used: one latency for all
        uint32_t code[16], byte[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t row = INSIDE ? row_of(a, r) : min(row_of(a, r), (int64_t)g.m - 1);
          const int64_t at = INSIDE || col < g.n ? col : 0;  // col is a multiple of TN: one block
          code[r] = TN == 4 ? *(const uint32_t*)(g.e.codes8 + row * g.e.nb8 * 32 + at) : *(const uint16_t*)(g.e.codes8 + row * g.e.nb8 * 32 + at);
          byte[r] = g.e.scales8[row * g.e.nb8 + (at >> 5)];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (!INSIDE && (row_of(a, r) >= g.m || col >= g.n)) continue;
          float v[TN];
#pragma unroll
          for (int b = 0; b < TN; ++b) v[b] = mx_times_dtanh(acc[a][b][r], (int)(int8_t)(code[r] >> 8 * b), byte[r]);
          write((T*)g.e.out + row_of(a, r) * ld + col, v);
        }
      }
    } else {
      float bias[TN] = {};
      if (g.e.bias)
#pragma unroll
        for (int b = 0; b < TN; ++b)
          if (INSIDE || col + b < g.n) bias[b] = MxType<T>::to(((const T*)g.e.bias)[col + b]);
      if (g.e.tanh) {
        each([&](int64_t at, float (&v)[TN]) {
          float t[TN];
#pragma unroll
          for (int b = 0; b < TN; ++b) {
            t[b] = mx_sigma(v[b] + bias[b]);
            v[b] = mx_tanh(v[b] + bias[b], t[b]);
          }
          write((T*)g.e.out + at, v);
          if (g.e.dact) {
#pragma unroll
            for (int b = 0; b < TN; ++b) t[b] = mx_keep_dtanh_of(t[b]);
            write((mx_dact*)g.e.dact + at, t);
          }
        });
      } else {
        each([&](int64_t at, float (&v)[TN]) {
#pragma unroll
          for (int b = 0; b < TN; ++b) v[b] += bias[b];
          write((T*)g.e.out + at, v);
        });
      }
    }
  };
  if (m0 + BM <= g.m && n0 + BN <= g.n && g.n % TN == 0) epilogue(std::true_type{});
  else epilogue(std::false_type{});
}

// out = epi(sum over parts), in the parts' order
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ parts, int64_t count, int64_t m, int64_t n,
                                                        MxEpilogue e) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < m * n; t += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int64_t s = 0; s < count; ++s) v += parts[s * m * n + t];
    const int64_t row = t / n;
    finish_one<T>(e, row, t - row * n, n, v);
  }
}

// parts[0] = sum over parts, in the parts' order
__global__ __launch_bounds__(256) void fold_parts_kernel(float* parts, int64_t count, int64_t elements) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < elements; t += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int64_t s = 0; s < count; ++s) v += parts[s * elements + t];
    parts[t] = v;
  }
}

// column sums of a gradient: part [blockIdx.y] of 64 columns
template <class S>
__global__ __launch_bounds__(256) void column_sums_kernel(S src, int64_t rows, int64_t cols, int64_t rows_per_part,
                                                          float* __restrict__ part) {
  __shared__ float lds[32][64];
  const int t = threadIdx.x, c = (t & 7) * 8;
  const int64_t c0 = (int64_t)blockIdx.x * 64, r0 = (int64_t)blockIdx.y * rows_per_part;
  const int64_t r1 = min(rows, r0 + rows_per_part);
  float s[8] = {};
  for (int64_t r = r0 + (t >> 3); r < r1; r += 32) {
    float v[8];
    if (c0 + c < cols) {
      src.load(r, c0 + c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[t >> 3][c + i] = s[i];
  __syncthreads();
  if (t < 64 && c0 + t < cols) {
    float v = 0.f;
    for (int i = 0; i < 32; ++i) v += lds[i][t];
    part[(int64_t)blockIdx.y * cols + c0 + t] = v;
  }
}

// their totals: four columns, 64 groups of parts, in a fixed order
template <class T>
__global__ __launch_bounds__(256) void column_parts_kernel(const float* __restrict__ part, int count, int64_t cols, T* __restrict__ out) {
  __shared__ float lds[64][4];
  const int64_t col = (int64_t)blockIdx.x * 4 + (threadIdx.x & 3);
  const int q = threadIdx.x >> 2;
  float v = 0.f;
  if (col < cols) {
    const int s1 = count * (q + 1) / 64;
#pragma unroll 4
    for (int s = count * q / 64; s < s1; ++s) v += part[s * cols + col];
  }
  lds[q][threadIdx.x & 3] = v;
  __syncthreads();
  if (q == 0 && col < cols) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += lds[i][threadIdx.x];
    out[col] = MxType<T>::from(v);
  }
}

int grid_for(int64_t threads) {
  const int64_t g = (threads + 255) / 256;
  return (int)(g < 1 ? 1 : g < 8192 ? g : 8192);
}

template <class S, int P>
void run_planes(S src, int64_t rows, int64_t pad, void* out, hipStream_t s) {
  planes_kernel<S, P><<<grid_for(rows * (pad >> 3)), 256, 0, s>>>(src, rows, pad, (uint16_t*)out);
}
template <class S, int P>
void run_planes_t(S src, int64_t rows, int64_t cols, int64_t pad, void* out, hipStream_t s) {
  const dim3 grid((unsigned)(pad / 64), (unsigned)((cols + 63) / 64));
  planes_t_kernel<S, P><<<grid, 256, 0, s>>>(src, rows, cols, pad, (uint16_t*)out);
}

bool vec_ok(const void* p, int64_t cols, int size) { return ((uintptr_t)p & 15) == 0 && cols * size % 16 == 0; }

}  // namespace

// ---- host ------------------------------------------------------------------------------------------------------------
void mx_planes(const MxSource& q, int64_t rows, int64_t cols, bool transposed, void* out, hipStream_t s) {
  if (rows < 1) return;
  const int64_t pad = mx_up(transposed ? rows : cols, 64);
#define MX_RUN(S, P, ...)                                                        \
  do {                                                                           \
    if (transposed) run_planes_t<S, P>(S __VA_ARGS__, rows, cols, pad, out, s);  \
    else run_planes<S, P>(S __VA_ARGS__, rows, pad, out, s);                     \
  } while (0)
#define MX_TYPED(T, P)                                                                                                   \
  do {                                                                                                                   \
    const bool vec = vec_ok(q.p, cols, sizeof(T));                                                                       \
    if (q.kind == MX_SRC_DENSE) MX_RUN(MX_ARG(SrcDense<T, false>), P, {(const T*)q.p, cols, vec});                       \
    else if (q.kind == MX_SRC_TANH) MX_RUN(MX_ARG(SrcDense<T, true>), P, {(const T*)q.p, cols, vec});                    \
    else if (q.kind == MX_SRC_GRAD_Y)                                                                                    \
      MX_RUN(MX_ARG(SrcGrad<T, 1>), P, {(const T*)q.p, q.aux, cols, vec && vec_ok(q.aux, cols, 4)});                     \
    else if (q.kind == MX_SRC_GRAD_D)                                                                                    \
      MX_RUN(MX_ARG(SrcGrad<T, 2>), P, {(const T*)q.p, q.aux, cols, vec && vec_ok(q.aux, cols, 2)});                     \
    else if (q.kind == MX_SRC_I8_TANH)                                                                                   \
      MX_RUN(SrcI8<true>, P, {(const uint8_t*)q.p, (const uint8_t*)q.aux, cols, mx_blocks(cols)});                       \
  } while (0)
#define MX_ARG(...) __VA_ARGS__
  if (q.kind == MX_SRC_I8 && q.half) MX_RUN(SrcI8<false>, 0, {(const uint8_t*)q.p, (const uint8_t*)q.aux, cols, mx_blocks(cols)});
  else if (q.kind == MX_SRC_I8) MX_RUN(SrcI8<false>, 1, {(const uint8_t*)q.p, (const uint8_t*)q.aux, cols, mx_blocks(cols)});
  else if (q.kind == MX_SRC_FP4) MX_RUN(SrcFp4, 1, {(const uint8_t*)q.p, (const uint8_t*)q.aux, cols, mx_blocks(cols)});
  else if (q.dtype == FMD_F32) MX_TYPED(float, 3);
  else if (q.half) MX_TYPED(_Float16, 0);
  else if (q.dtype == FMD_F16) MX_TYPED(_Float16, 2);
  else MX_TYPED(mx_bf16, 1);
#undef MX_RUN
#undef MX_TYPED
#undef MX_ARG
}

void mx_planes_keep(const MxSource& q, int64_t rows, int64_t cols, void* out, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  const int64_t pad = mx_up(cols, 64), nb = mx_blocks(cols);
  const int grid = grid_for(rows * (pad >> 3));
#define MX_TYPED(T, P)                                                                                                            \
  do {                                                                                                                            \
    const SrcDense<T, false> src{(const T*)q.p, cols, vec_ok(q.p, cols, sizeof(T))};                                              \
    if (q.kind == MX_SRC_TANH) planes_keep_kernel<T, true, P><<<grid, 256, 0, s>>>(src, rows, pad, (uint16_t*)out, nb, codes, scales); \
    else planes_keep_kernel<T, false, P><<<grid, 256, 0, s>>>(src, rows, pad, (uint16_t*)out, nb, codes, scales);                 \
  } while (0)
  if (q.dtype == FMD_F32) MX_TYPED(float, 3);
  else if (q.dtype == FMD_F16) MX_TYPED(_Float16, 0);
  else MX_TYPED(mx_bf16, 1);
#undef MX_TYPED
}

void mx_scale_tiles(const void* scales, int64_t rows, int64_t nb, void* out, hipStream_t s) {
  const int64_t kt = (nb + 7) / 8;
  scale_tiles_kernel<<<grid_for(rows * kt * 2), 256, 0, s>>>((const uint8_t*)scales, rows, mx_up(rows, 4), nb, kt, (uint32_t*)out);
}

// The large tile reads each operand half as often and is worth it once its workgroups fill three quarters of the chip; else the small
// tile, and the contraction in parts.  Calls with 4096 columns of x, us, bf16 planes / both in 4 bits, large against small:
//   2560 x 4096 (160 large tiles) 133 / 81 against 125 / 48;  2816 x 4352 (187) 153 / 82 against 141 / 55;
//   8192 x 1536 (192) 120 / 51 against 135 / 57;  3840 x 4096 (240) 122 / 48 against 148 / 55;  4096 x 4096 (256) 126 / 51 against 147 / 57
MxProductPlan mx_product_plan(int64_t m, int64_t n, int64_t kt, int npairs) {
  MxProductPlan p{};
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128);
  p.big = big >= 192;
  p.tiles = p.big ? big : small;
  const int64_t its = kt * npairs;
  int64_t s = p.tiles >= 192 ? 1 : 512 / p.tiles;
  if (s > its / 4) s = its / 4;
  if (s > 64) s = 64;
  p.splits = p.most = (int)(s < 1 ? 1 : s);
  return p;
}

template <class T, int FMT>
static void launch_gemm(const GemmArgs& g, bool big, hipStream_t s) {
  const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits);
  if (big) gemm_kernel<T, FMT, 2, 4, 4, 2><<<grid, 512, 0, s>>>(g);
  else gemm_kernel<T, FMT, 2, 2, 2, 2><<<grid, 256, 0, s>>>(g);
}

void mx_product(const MxOperand& a, const MxOperand& b, int64_t m, int64_t n, int64_t kt, const MxProductPlan& plan, int dtype,
                const MxEpilogue& e, float* parts, hipStream_t s) {
  GemmArgs g{};
  g.a = (const char*)a.p, g.b = (const char*)b.p;
  g.a_plane = a.plane, g.b_plane = b.plane, g.a_pitch = a.pitch, g.b_pitch = b.pitch;
  g.sa = (const char*)a.scales, g.sb = (const char*)b.scales;
  g.m = (int)m, g.n = (int)n, g.kt = (int)kt, g.granules = (int)(a.pitch / 16);
  const int side = plan.big ? 256 : 128;
  g.tiles_m = (int)((m + side - 1) / side), g.tiles_n = (int)((n + side - 1) / side), g.splits = plan.splits;
  const MxPairs pairs = mx_pairs(a.planes, b.planes);
  g.npairs = pairs.n;
  for (int i = 0; i < pairs.n; ++i) g.pa |= (uint32_t)pairs.a[i] << 2 * i, g.pb |= (uint32_t)pairs.b[i] << 2 * i;
  g.e = e;
  g.partial = parts;
  const bool f32 = parts || dtype == FMD_F32;
  if (a.scales) {
    if (f32) launch_gemm<float, FMT_FP4>(g, plan.big, s);
    else if (dtype == FMD_F16) launch_gemm<_Float16, FMT_FP4>(g, plan.big, s);
    else launch_gemm<mx_bf16, FMT_FP4>(g, plan.big, s);
  } else if (a.half) {
    if (f32) launch_gemm<float, FMT_F16>(g, plan.big, s);
    else launch_gemm<_Float16, FMT_F16>(g, plan.big, s);
  } else {
    if (f32) launch_gemm<float, FMT_BF16>(g, plan.big, s);
    else if (dtype == FMD_F16) launch_gemm<_Float16, FMT_BF16>(g, plan.big, s);
    else launch_gemm<mx_bf16, FMT_BF16>(g, plan.big, s);
  }
}

void mx_sum_parts(const float* parts, int64_t count, int64_t m, int64_t n, int dtype, const MxEpilogue& e, hipStream_t s) {
  if (dtype == FMD_F32) sum_parts_kernel<float><<<grid_for(m * n), 256, 0, s>>>(parts, count, m, n, e);
  else if (dtype == FMD_F16) sum_parts_kernel<_Float16><<<grid_for(m * n), 256, 0, s>>>(parts, count, m, n, e);
  else sum_parts_kernel<mx_bf16><<<grid_for(m * n), 256, 0, s>>>(parts, count, m, n, e);
}

void mx_fold_parts(float* parts, int64_t count, int64_t elements, hipStream_t s) {
  fold_parts_kernel<<<grid_for(elements), 256, 0, s>>>(parts, count, elements);
}

void mx_column_sums(const MxSource& q, int64_t rows, int64_t cols, int64_t parts, float* out, hipStream_t s) {
  const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)parts);
  const int64_t per = (rows + parts - 1) / parts;
#define MX_TYPED(T)                                                                                                        \
  do {                                                                                                                     \
    const bool vec = vec_ok(q.p, cols, sizeof(T));                                                                         \
    if (q.kind == MX_SRC_DENSE)                                                                                            \
      column_sums_kernel<<<grid, 256, 0, s>>>(SrcDense<T, false>{(const T*)q.p, cols, vec}, rows, cols, per, out);         \
    else if (q.kind == MX_SRC_GRAD_Y)                                                                                      \
      column_sums_kernel<<<grid, 256, 0, s>>>(SrcGrad<T, 1>{(const T*)q.p, q.aux, cols, vec && vec_ok(q.aux, cols, 4)},    \
                                              rows, cols, per, out);                                                       \
    else                                                                                                                   \
      column_sums_kernel<<<grid, 256, 0, s>>>(SrcGrad<T, 2>{(const T*)q.p, q.aux, cols, vec && vec_ok(q.aux, cols, 2)},    \
                                              rows, cols, per, out);                                                       \
  } while (0)
  if (q.dtype == FMD_F32) MX_TYPED(float);
  else if (q.dtype == FMD_F16) MX_TYPED(_Float16);
  else MX_TYPED(mx_bf16);
#undef MX_TYPED
}

void mx_column_totals(const float* parts, int64_t count, int64_t cols, int dtype, void* out, hipStream_t s) {
  const unsigned grid = (unsigned)((cols + 3) / 4);
  if (dtype == FMD_F32) column_parts_kernel<float><<<grid, 256, 0, s>>>(parts, (int)count, cols, (float*)out);
  else if (dtype == FMD_F16) column_parts_kernel<_Float16><<<grid, 256, 0, s>>>(parts, (int)count, cols, (_Float16*)out);
  else column_parts_kernel<mx_bf16><<<grid, 256, 0, s>>>(parts, (int)count, cols, (mx_bf16*)out);
}

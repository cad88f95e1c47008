// Narrow layers over many rows: out[m,o] = epi(pro(in)[m,c] V[c,o] (+ bias)), c and o at most 256.  One pass over the rows.
//
// These layers are bound by memory (a row of 128 + 128 fp32 is 1 KB against 32 K multiply-adds), so everything a row needs
// happens between its one read and its one write: the activation or the gradient's factor, the cut into planes, the 4- or
// 8-bit quantisation, the product, bias, tanh, tanh'.
//
// A workgroup keeps the whole weight in LDS in the order of the matrix fragments; a wave owns 32 rows at a time and shares
// nothing with the others, so the loop has no barrier.  The rows of a wave's next 64 columns are on their way in registers
// while the current ones are computed; they pass through 32 x 64 values of LDS that belong to the wave, from coalesced
// rows to the layout in which lane (row, half) holds 32 neighbouring columns -- a whole block: its largest value, codes and
// scale need no other lane.  The contraction may run in any order as long as both operands agree, so step s of a 64-column
// chunk takes columns 8s..8s+7 of either half.  Output column NT*lane + tile: a lane's NT results are neighbours, and a
// store of one register per tile writes two whole rows.
//
// Measured: 1882048 x 50 -> 128 fp32 under tanh, 4-bit weights 271 us (4.9 TB/s; a large copy runs at 5.0), with an 8-bit checkpoint of
// x 278, the gradient back through tanh' and the bias's sums 501 (4.6 TB/s); 1000000 x 128 -> 128 bf16 150 and 171 (5.1 and 4.5 TB/s).
// Against the general product, us a call in a graph: 256 x 128 x 128 bf16 3.6 / 9.0 (fp32 5.1 / 12), 34432 rows 9 / 15 (12 / 25), 193688
// rows 20 / 58 (34 / 154); 256 x 256: 4096 rows 9.3 / 12 (14 / 27), 193688 rows 53 / 78 (107 / 231); both operands in 4 bits at
// 256 x 256: 4096 rows 6.8 / 8.7, 193688 51 / 50, and 34432 24 / 18, the one shape where the product is ahead.
#include <type_traits>

#include "fmd_mx_host.h"

namespace {

constexpr int WAVES = 8;
enum { PRO_ID, PRO_TANH_IN, PRO_GRAD_Y, PRO_GRAD_D };
enum { W_DENSE, W_FP4, W_FP4_BOTH, W_FP4_ACROSS };  // across: the contraction runs over the weight's rows
enum { EPI_ACT, EPI_DTANH };

struct LayerArgs {
  const void *in, *aux, *w, *bias;
  const uint8_t* wscales;
  void *out, *dact;
  uint8_t *codes8, *scales8;  // EPI_DTANH: read, [row][32 nb8]; else written unless null
  void* totals;
  float* sums;                // column sums of the (multiplied) input, [workgroup][c], or null
  int64_t m, sk, sn;          // sk, sn: strides of a dense weight
  int c, o, vec, wvec, tanh, nb8;
};

// an operand that is computed here has a second plane in bf16: one would round it to the layer's type before the product does
// (193688 x 128 x 128 bf16 under tanh, us a call: forward 56 against 53, backward of a 4-bit layer 79 against 81)
template <class T, int WK, int PRO = PRO_ID> struct LayerPlanes {
  static constexpr int in = WK == W_FP4_BOTH ? 1 : PRO != PRO_ID && MxType<T>::planes == 1 ? 2 : MxType<T>::planes;
  static constexpr int w = WK == W_DENSE ? MxType<T>::planes : 1;
};

// Rows through buffer descriptors: a tile's descriptor ends behind the last row, so rows past the end read as zeros and are
// not written, without a comparison; a lane whose column does not exist uses an offset behind every descriptor's end.
typedef __amdgpu_buffer_rsrc_t Rows;
constexpr uint32_t NOWHERE = 0x40000000u;
__device__ __forceinline__ Rows rows_of(const void* p, int64_t row0, int64_t m, int row_bytes) {
  const int64_t left = m - row0;
  const int n = left < 32 ? (left > 0 ? (int)left : 0) : 32;
  return __builtin_amdgcn_make_buffer_rsrc((char*)p + row0 * row_bytes, 0, n * row_bytes, 0x00020000);
}

// 32 rows x 64 columns in registers: pieces of 16 bytes where the rows allow it, else single values (lane = column)
template <class T>
struct Raw {
  static constexpr int S = sizeof(T), PIECES = S == 4 ? 8 : 4, PER_ROW = 64 * S / 16, PER = 16 / S;
  u32x4 v[8];  // 8 or 4 pieces, or 32 single values
  __device__ __forceinline__ void load(Rows rows, int c, int col0, bool vec, int lane) {
    const int cs = mx_here(c * S);
    if (vec) {
      const int col = col0 + lane % PER_ROW * PER;
      const uint32_t off = col < c ? (uint32_t)(lane / PER_ROW * c + col) * S : NOWHERE;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        v[i] = __builtin_amdgcn_raw_buffer_load_b128(rows, off + i * (64 / PER_ROW) * cs, 0, 0);
    } else {
      const uint32_t off = col0 + lane < c ? (uint32_t)(col0 + lane) * S : NOWHERE;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if constexpr (S == 4) v[i >> 2][i & 3] = __builtin_amdgcn_raw_buffer_load_b32(rows, off + i * cs, 0, 0);
        else v[i >> 2][i & 3] = __builtin_amdgcn_raw_buffer_load_b16(rows, off + i * cs, 0, 0);
      }
    }
  }
  static __device__ __forceinline__ float value(uint32_t u) {
    if constexpr (S == 4) return __builtin_bit_cast(float, u);
    else return MxType<T>::to(__builtin_bit_cast(T, (uint16_t)u));
  }
};

// What a lane writes there in one type, others read in another: words that the compiler takes for any type's
typedef uint16_t any16 __attribute__((may_alias));
typedef uint32_t any32 __attribute__((may_alias));
typedef u32x4 any128 __attribute__((may_alias));
// A wave's accesses of LDS are done in their order; the compiler, which sees one lane's addresses, keeps that order across this
__device__ __forceinline__ void between_lanes() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// LDS of a wave, 32 rows x 64 values: row r's piece q of 16 bytes at position q ^ s(r), so that neither the rows' writes nor
// the lanes' reads (a row each) meet a bank twice
template <class T>
struct Pass {
  static constexpr int S = sizeof(T), PER = 16 / S, ROW = 64 * S;
  static __device__ __forceinline__ int swz(int r) { return S == 4 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ void put(char* lds, const Raw<T>& raw, bool vec, int lane) {
    using R = Raw<T>;
    if (vec) {
#pragma unroll
      for (int i = 0; i < R::PIECES; ++i) {
        const int r = i * (64 / R::PER_ROW) + lane / R::PER_ROW, q = lane % R::PER_ROW;
        *(any128*)(lds + r * ROW + (q ^ swz(r)) * 16) = raw.v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        char* to = lds + i * ROW + ((lane / PER) ^ swz(i)) * 16 + (lane % PER) * S;
        if constexpr (S == 4) *(any32*)to = raw.v[i >> 2][i & 3];
        else *(any16*)to = (uint16_t)raw.v[i >> 2][i & 3];
      }
    }
  }
  // the sum of a column over the rows
  static __device__ __forceinline__ float column(const char* lds, int col) {
    float s[4] = {};
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const char* at = lds + r * ROW + ((col / PER) ^ swz(r)) * 16 + col % PER * S;
      T v;
      if constexpr (S == 4) v = __builtin_bit_cast(T, (uint32_t) * (const any32*)at);
      else v = __builtin_bit_cast(T, (uint16_t) * (const any16*)at);
      s[r & 3] += MxType<T>::to(v);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
  // the 32 columns of (row, half)
  static __device__ __forceinline__ void get(const char* lds, int row, int h, float (&x)[32]) {
    constexpr int N = ROW / 32;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u32x4 u = *(const any128*)(lds + row * ROW + ((h * N + i) ^ swz(row)) * 16);
      T t[PER];
      *(u32x4*)t = u;
#pragma unroll
      for (int e = 0; e < PER; ++e) x[i * PER + e] = MxType<T>::to(t[e]);
    }
  }
};

// a gradient and its factor, multiplied in fp32 on the way into LDS.  T = float: aux = y, factor 1 - y^2; else aux = the factor
template <class T>
__device__ __forceinline__ void put_product(char* lds, const Raw<T>& g, const Raw<typename std::conditional<sizeof(T) == 4, float, mx_dact>::type>& aux,
                                            bool vec, int lane) {
  using A = typename std::conditional<sizeof(T) == 4, float, mx_dact>::type;
  using R = Raw<T>;
  auto factor = [](float v) { return sizeof(T) == 4 ? 1.f - v * v : v; };
  if (vec) {
#pragma unroll
    for (int i = 0; i < R::PIECES; ++i) {
      const int r = i * (64 / R::PER_ROW) + lane / R::PER_ROW, q = lane % R::PER_ROW;
      T gv[R::PER];
      A av[R::PER];
      *(u32x4*)gv = g.v[i];
      *(u32x4*)av = aux.v[i];
#pragma unroll
      for (int k = 0; k < R::PER / 4; ++k) {
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = MxType<T>::to(gv[4 * k + e]) * factor(MxType<A>::to(av[4 * k + e]));
        *(any128*)(lds + r * 256 + ((q * (R::PER / 4) + k) ^ Pass<float>::swz(r)) * 16) = __builtin_bit_cast(u32x4, o);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      *(any32*)(lds + i * 256 + ((lane >> 2) ^ Pass<float>::swz(i)) * 16 + (lane & 3) * 4) =
          __builtin_bit_cast(uint32_t, Raw<T>::value(g.v[i >> 2][i & 3]) * factor(Raw<A>::value(aux.v[i >> 2][i & 3])));
  }
}

template <class T, int WK, int NT>
__device__ __forceinline__ void fill_weight(const LayerArgs& a, int o0, char* lds) {
  const int chunks = (a.c + 63) >> 6;
  constexpr int P = LayerPlanes<T, WK>::w;
  if constexpr (WK == W_FP4_BOTH) {  // [chunk][tile][64 lanes] codes, then scales
    const int nb = (a.c + 31) >> 5;
    for (int u = threadIdx.x; u < chunks * NT * 64; u += 64 * WAVES) {
      const int lane = u & 63, t = (u >> 6) % NT, ch = (u >> 6) / NT;
      const int n = o0 + NT * (lane & 31) + t, b = ch * 2 + (lane >> 5);
      u32x4 code = {0, 0, 0, 0};
      uint32_t s = 0;
      if (n < a.o && b < nb) {
        code = *(const u32x4*)((const char*)a.w + ((int64_t)n * nb + b) * 16);
        s = a.wscales[(int64_t)n * nb + b];
      }
      *(u32x4*)(lds + u * 16) = code;
      *(uint32_t*)(lds + chunks * NT * 1024 + u * 4) = s;
    }
  } else if constexpr (WK == W_DENSE) {  // [chunk][step][plane][tile][64 lanes] of 8 bf16
    // the loads of four units first: one latency for all of them
    constexpr int MORE = 4;
    const T* w = (const T*)a.w;
    const int units = chunks * 4 * NT * 64;
    for (int u0 = threadIdx.x; u0 < units; u0 += 64 * WAVES * MORE) {
      T raw[MORE][8];
#pragma unroll
      for (int i = 0; i < MORE; ++i) {
        const int u = u0 + i * 64 * WAVES, lane = u & 63, t = (u >> 6) % NT, cs = (u >> 6) / NT;
        const int n = o0 + NT * (lane & 31) + t, k0 = (cs >> 2) * 64 + (lane >> 5) * 32 + (cs & 3) * 8;
        if (a.wvec && n < a.o && k0 + 8 <= a.c) {  // the contraction is contiguous
#pragma unroll
          for (int e = 0; e < (int)sizeof(T) / 2; ++e) ((u32x4*)raw[i])[e] = ((const u32x4*)(w + (int64_t)n * a.sn + k0))[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) raw[i][e] = u < units && n < a.o && k0 + e < a.c ? w[(int64_t)(k0 + e) * a.sk + n * a.sn] : T{};
        }
      }
#pragma unroll
      for (int i = 0; i < MORE; ++i) {
        const int u = u0 + i * 64 * WAVES, lane = u & 63, t = (u >> 6) % NT, cs = (u >> 6) / NT;
        if (u >= units) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = MxType<T>::to(raw[i][e]);
        u32x4 f[P];
        mx_split8<P>(v, f);
#pragma unroll
        for (int p = 0; p < P; ++p) *(u32x4*)(lds + (((cs * P + p) * NT + t) * 64 + lane) * 16) = f[p];
      }
    }
  } else {
    for (int u = threadIdx.x; u < chunks * 4 * NT * 64; u += 64 * WAVES) {
      const int lane = u & 63, t = (u >> 6) % NT, cs = (u >> 6) / NT;
      const int n = o0 + NT * (lane & 31) + t, k0 = (cs >> 2) * 64 + (lane >> 5) * 32 + (cs & 3) * 8;
      u32x4 f[1];
      if constexpr (WK == W_FP4) {
        const int nb = (a.c + 31) >> 5, b = k0 >> 5;
        f[0] = u32x4{0, 0, 0, 0};
        if (n < a.o && b < nb) {
          uint32_t code = *(const uint32_t*)((const char*)a.w + ((int64_t)n * nb + b) * 16 + (k0 & 31) / 2);
          const int valid = a.c - k0;  // columns behind the last one count as zeros whatever the caller's codes hold
          if (valid < 8) code = valid > 0 ? code & ((1u << 4 * valid) - 1) : 0u;
          f[0] = mx_bf16_from4(code, mx_scale_value(a.wscales[(int64_t)n * nb + b]));
        }
      } else {  // weight row k, column n
        const int nb = (a.o + 31) >> 5;
        uint32_t byte[8], scale[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool there = n < a.o && k0 + i < a.c;
          const int64_t r = there ? (int64_t)(k0 + i) * nb + (n >> 5) : 0;
          byte[i] = there ? ((const uint8_t*)a.w)[r * 16 + ((n & 31) >> 1)] : 0u;
          scale[i] = there ? a.wscales[r] : 0u;
        }
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const u32x4 q = mx_bf16_from4(n & 1 ? byte[i] >> 4 : byte[i] & 15u, mx_scale_value(scale[i]));
          v[i] = __builtin_bit_cast(float, q[0] << 16);
        }
        mx_split8<1>(v, f);
      }
      *(u32x4*)(lds + ((cs * NT + t) * 64 + lane) * 16) = f[0];
    }
  }
}

template <class T, int PRO>
constexpr int pass_bytes() {  // LDS of a wave on the way from rows to lanes
  return 32 * 64 * (PRO == PRO_GRAD_Y || PRO == PRO_GRAD_D ? 4 : (int)sizeof(T));
}

template <class T, int PRO, int WK, int EPI, int NT>
__global__ __launch_bounds__(64 * WAVES, 2) void layer_kernel(const LayerArgs a) {
  constexpr int PA = LayerPlanes<T, WK, PRO>::in, PB = LayerPlanes<T, WK>::w, TOP = PA > PB ? PA : PB;
  using AuxT = typename std::conditional<sizeof(T) == 4, float, mx_dact>::type;
  constexpr bool AUX = PRO == PRO_GRAD_Y || PRO == PRO_GRAD_D;
  constexpr int S = sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 31, h = lane >> 5;
  const int chunks = (a.c + 63) >> 6;
  const bool vec = a.vec;
  char* const own = lds + wave * pass_bytes<T, PRO>();
  char* const wl = lds + WAVES * pass_bytes<T, PRO>();
  const int o0 = blockIdx.y * 32 * NT;  // few rows: the outputs are shared out, too
  fill_weight<T, WK, NT>(a, o0, wl);

  const int tiles = (int)((a.m + 31) >> 5), stride = gridDim.x * WAVES;
  Raw<T> raw;
  Raw<AuxT> raw_aux;
  auto fetch = [&](int tile, int ch) {
    raw.load(rows_of(a.in, (int64_t)tile * 32, a.m, a.c * S), a.c, ch * 64, vec, lane);
    if constexpr (AUX) raw_aux.load(rows_of(a.aux, (int64_t)tile * 32, a.m, a.c * (int)sizeof(AuxT)), a.c, ch * 64, vec, lane);
  };
  int tile = wave * gridDim.x + blockIdx.x, ch = 0;  // few tiles: one a workgroup first
  if (tile < tiles) fetch(tile, 0);
  float bias[NT] = {};
  if (EPI == EPI_ACT && a.bias)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (o0 + NT * j + t < a.o) bias[t] = MxType<T>::to(((const T*)a.bias)[o0 + NT * j + t]);
  __syncthreads();

  f32x16 acc[NT];
  float sums[4] = {};  // columns lane, 64 + lane, ..
  while (tile < tiles) {
    const int64_t row0 = (int64_t)tile * 32;
    if (ch == 0)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    {
      float x[32];
      between_lanes();
      if constexpr (AUX) {
        put_product<T>(own, raw, raw_aux, vec, lane);
        between_lanes();
        Pass<float>::get(own, j, h, x);
      } else {
        Pass<T>::put(own, raw, vec, lane);
        between_lanes();
        Pass<T>::get(own, j, h, x);
      }
      if (WK == W_FP4_ACROSS && a.sums) {
        const float v = Pass<typename std::conditional<AUX, float, T>::type>::column(own, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] += i == ch ? v : 0.f;
      }
      const int next_tile = ch + 1 < chunks ? tile : tile + stride, next_ch = ch + 1 < chunks ? ch + 1 : 0;
      if (next_tile < tiles) fetch(next_tile, next_ch);
      if (EPI == EPI_ACT && WK == W_DENSE && a.codes8 && blockIdx.y == 0) {
        const int64_t row = row0 + j;
        const int b = ch * 2 + h;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
        const uint32_t byte = mx_scale_byte<8>(top);
        if (row < a.m && b < a.nb8) {
          u32x4 q[2];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            q[i >> 2][i & 3] = mx_codes8(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], byte);
          }
          u32x4* to = (u32x4*)(a.codes8 + (row * a.nb8 + b) * 32);
          to[0] = q[0];
          to[1] = q[1];
          a.scales8[row * a.nb8 + b] = (uint8_t)byte;
        }
      }
      if constexpr (PRO == PRO_TANH_IN)
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = mx_tanh(x[i]);
      if constexpr (WK == W_FP4_BOTH) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
        const uint32_t byte = mx_scale_byte<4>(top);
        const float s = byte == 255u ? 1.f : mx_scale_value(byte);
        i32x8 fa = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = x[8 * i + e];
          fa[i] = byte == 255u ? 0 : (int)mx_codes4(v, s);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const u32x4 u = *(const u32x4*)(wl + ((ch * NT + t) * 64 + lane) * 16);
          const i32x8 fb = {(int)u[0], (int)u[1], (int)u[2], (int)u[3], 0, 0, 0, 0};
          const int sb = *(const int*)(wl + chunks * NT * 1024 + ((ch * NT + t) * 64 + lane) * 4);
          acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa, fb, acc[t], 4, 4, 0, (int)byte, 0, sb);
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = x[8 * s + e];
          u32x4 fa[PA];
          mx_split8<PA>(v, fa);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            u32x4 fb[PB];
#pragma unroll
            for (int p = 0; p < PB; ++p) fb[p] = *(const u32x4*)(wl + ((((ch * 4 + s) * PB + p) * NT + t) * 64 + lane) * 16);
#pragma unroll
            for (int sum = TOP - 1; sum >= 0; --sum)  // the smallest products first
#pragma unroll
              for (int p = 0; p < PA; ++p)
                if (sum - p >= 0 && sum - p < PB)
                  acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa[p]),
                                                                   __builtin_bit_cast(bf16x8, fb[sum - p]), acc[t], 0, 0, 0);
          }
        }
      }
    }
    if (++ch < chunks) continue;
    ch = 0;
    tile += stride;
    const int col = o0 + NT * j, os = mx_here(a.o), nbs = mx_here(a.nb8);
    const bool whole = a.o % NT == 0;
    // v of one row into out (U = T) or dact (U = mx_dact); a lane's columns in one store where every row starts on a multiple of NT
    auto write = [&](auto zero, Rows rows, int r, const float (&v)[NT]) {
      using U = decltype(zero);
      constexpr int SU = sizeof(U);
      const uint32_t voff = (col < a.o ? (uint32_t)(4 * h * a.o + col) * SU : NOWHERE) + ((r & 3) + 8 * (r >> 2)) * os * SU;
      if (whole) {
        U e[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) e[t] = MxType<U>::from(v[t]);
        if constexpr (SU * NT == 16) __builtin_amdgcn_raw_buffer_store_b128(*(u32x4*)e, rows, voff, 0, 0);
        else if constexpr (SU * NT == 8) __builtin_amdgcn_raw_buffer_store_b64(*(u32x2*)e, rows, voff, 0, 0);
        else if constexpr (SU * NT == 4) __builtin_amdgcn_raw_buffer_store_b32(*(uint32_t*)e, rows, voff, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(*(uint16_t*)e, rows, voff, 0, 0);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t off = col + t < a.o ? voff + t * SU : NOWHERE;
          const U e = MxType<U>::from(v[t]);
          if constexpr (SU == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, e), rows, off, 0, 0);
          else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, e), rows, off, 0, 0);
        }
      }
    };
    const Rows out = rows_of(a.out, row0, a.m, a.o * S);
    if constexpr (EPI == EPI_DTANH) {
      const Rows codes = rows_of(a.codes8, row0, a.m, a.nb8 * 32), scales = rows_of(a.scales8, row0, a.m, a.nb8);
      const uint32_t at = col < a.o ? (uint32_t)(4 * h * a.nb8 * 32 + col) : NOWHERE;  // col is a multiple of NT: one block
      const uint32_t sat = col < a.o ? (uint32_t)(4 * h * a.nb8 + (col >> 5)) : NOWHERE;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = (r & 3) + 8 * (r >> 2);
        uint32_t q;
        if constexpr (NT == 4) q = __builtin_amdgcn_raw_buffer_load_b32(codes, at + row * 32 * nbs, 0, 0);
        else if constexpr (NT == 1) q = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(codes, at + row * 32 * nbs, 0, 0);
        else q = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(codes, at + row * 32 * nbs, 0, 0);
        const uint32_t byte = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(scales, sat + row * nbs, 0, 0);
        float v[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) v[t] = mx_times_dtanh(acc[t][r], (int)(int8_t)(q >> 8 * t), byte);
        write(T{}, out, r, v);
      }
    } else {
      const Rows dact = a.dact ? rows_of(a.dact, row0, a.m, a.o * 2) : rows_of(a.out, a.m, a.m, 0);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) v[t] = acc[t][r] + bias[t];
        if ((WK == W_FP4 || WK == W_FP4_BOTH) && a.tanh) {  // the others have none
          float u[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            u[t] = mx_sigma(v[t]);
            v[t] = mx_tanh(v[t], u[t]);
          }
          if (a.dact) {
#pragma unroll
            for (int t = 0; t < NT; ++t) u[t] = mx_keep_dtanh_of(u[t]);
            write(mx_dact{}, dact, r, u);
          }
        }
        write(T{}, out, r, v);
      }
    }
  }
  if constexpr (WK == W_FP4_ACROSS) {
    if (a.sums && blockIdx.y == 0) {  // the waves' sums, in order
      __syncthreads();
      float* all = (float*)lds;
#pragma unroll
      for (int i = 0; i < 4; ++i) all[wave * 256 + 64 * i + lane] = sums[i];
      __syncthreads();
      if ((int)threadIdx.x < a.c) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += all[w * 256 + threadIdx.x];
        a.sums[(int64_t)blockIdx.x * a.c + threadIdx.x] = v;
      }
    }
  }
}

// column totals from the workgroups' sums: four columns, 64 groups of workgroups, in a fixed order
template <class T>
__global__ __launch_bounds__(256) void column_totals_kernel(const float* __restrict__ sums, int count, int c, T* __restrict__ out) {
  __shared__ float lds[64][4];
  const int col = blockIdx.x * 4 + (threadIdx.x & 3), q = threadIdx.x >> 2;
  float v = 0.f;
  if (col < c) {
    const int s1 = count * (q + 1) / 64;
#pragma unroll 8
    for (int s = count * q / 64; s < s1; ++s) v += sums[s * c + col];  // at most 512 x 256
  }
  lds[q][threadIdx.x & 3] = v;
  __syncthreads();
  if (q == 0 && col < c) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += lds[i][threadIdx.x];
    out[col] = MxType<T>::from(v);
  }
}

template <class T, int PRO, int WK, int NT>
int lds_bytes(int c) {
  const int chunks = (c + 63) >> 6;
  return WAVES * pass_bytes<T, PRO>() + (WK == W_FP4_BOTH ? chunks * NT * 64 * 20 : chunks * 4 * NT * 1024 * LayerPlanes<T, WK>::w);
}
constexpr int LDS = 160 * 1024;

template <class T, int PRO, int WK, int EPI, int NT>
int launch(const LayerArgs& a, hipStream_t s) {
  const int bytes = lds_bytes<T, PRO, WK, NT>(a.c);
  if (bytes > LDS) return FMD_EINVAL;
  if (mx_allow_lds(&layer_kernel<T, PRO, WK, EPI, NT>, LDS) != hipSuccess) return FMD_ELAUNCH;
  const int64_t tiles = (a.m + 31) / 32, full = 256 * (bytes <= LDS / 2 ? 2 : 1);
  const int grid = (int)(tiles < full ? tiles : full);
  layer_kernel<T, PRO, WK, EPI, NT><<<dim3(grid, (a.o + 32 * NT - 1) / (32 * NT)), 64 * WAVES, bytes, s>>>(a);
  if (WK == W_FP4_ACROSS && a.sums) column_totals_kernel<T><<<(a.c + 3) / 4, 256, 0, s>>>(a.sums, grid, a.c, (T*)a.totals);
  return hipGetLastError() == hipSuccess ? FMD_OK : FMD_ELAUNCH;
}

template <class T, int PRO, int WK, int EPI>
int by_width(const LayerArgs& a, hipStream_t s) {
  // A tile of rows is 10 us from one end to the other: up to 64 of them, every 32 outputs get workgroups of their own (269 rows,
  // 128 x 128, fp32: 11.1 us against 18.2); from there on the rows fill the chip (34432 rows: 43 against 25)
  if ((a.m + 31) / 32 <= 64) return launch<T, PRO, WK, EPI, 1>(a, s);
  // 128 outputs a workgroup, which read the rows once for each 128, where their weight fits LDS (fp32 beyond 128 columns: 64)
  return a.o <= 64 || lds_bytes<T, PRO, WK, 4>(a.c) > LDS ? launch<T, PRO, WK, EPI, 2>(a, s) : launch<T, PRO, WK, EPI, 4>(a, s);
}

template <class T>
int by_kind(LayerArgs a, const MxLayer& l, hipStream_t s) {
  a.vec = ((uintptr_t)a.in & 15) == 0 && a.c * sizeof(T) % 16 == 0 &&
          (!a.aux || (((uintptr_t)a.aux & 15) == 0 && a.c * (l.pro == MX_SRC_GRAD_Y ? 4 : 2) % 16 == 0));
  a.wvec = a.sk == 1 && ((uintptr_t)a.w & 15) == 0 && a.sn * sizeof(T) % 16 == 0;
  if (l.weight == MX_WEIGHT_FP4) return by_width<T, PRO_ID, W_FP4, EPI_ACT>(a, s);
  if (l.weight == MX_WEIGHT_FP4_BOTH) return by_width<T, PRO_ID, W_FP4_BOTH, EPI_ACT>(a, s);
  if (l.weight == MX_WEIGHT_FP4_ACROSS) {
    if (l.pro == MX_SRC_DENSE) return by_width<T, PRO_ID, W_FP4_ACROSS, EPI_ACT>(a, s);
    if constexpr (sizeof(T) == 4) return by_width<T, PRO_GRAD_Y, W_FP4_ACROSS, EPI_ACT>(a, s);
    else return by_width<T, PRO_GRAD_D, W_FP4_ACROSS, EPI_ACT>(a, s);
  }
  if (l.dtanh) return by_width<T, PRO_ID, W_DENSE, EPI_DTANH>(a, s);
  if (l.pro == MX_SRC_TANH) return by_width<T, PRO_TANH_IN, W_DENSE, EPI_ACT>(a, s);
  return by_width<T, PRO_ID, W_DENSE, EPI_ACT>(a, s);
}

}  // namespace

int64_t mx_layer_sums_bytes(int64_t m, int64_t c) { return (m < 512 * 32 ? (m + 31) / 32 : 512) * c * 4; }
bool mx_layer_fits(int64_t c, int64_t o) { return c <= 256 && o <= 256; }

int mx_layer(const MxLayer& l, int dtype, int64_t m, int64_t c, int64_t o, hipStream_t s) {
  LayerArgs a{};
  a.in = l.in, a.aux = l.aux, a.w = l.w, a.wscales = (const uint8_t*)l.wscales, a.bias = l.e.bias;
  a.out = l.e.out, a.dact = l.e.dact, a.tanh = l.e.tanh;
  a.codes8 = l.codes8, a.scales8 = l.scales8, a.nb8 = (int)mx_blocks(l.dtanh ? o : c);
  a.sums = l.sums, a.totals = l.totals;
  a.m = m, a.c = (int)c, a.o = (int)o, a.sk = l.sk, a.sn = l.sn;
  if (dtype == FMD_F32) return by_kind<float>(a, l, s);
  if (dtype == FMD_F16) return by_kind<_Float16>(a, l, s);
  return by_kind<mx_bf16>(a, l, s);
}

// What the translation units of the block-scaled layers share on the host side.
#pragma once
#include "fmd_mx.h"

struct MxEpilogue {            // v = acc (+ bias) (tanh) (* tanh'(8-bit value)) -> out
  const void* bias;            // in out's type, or null
  void* out;
  void* dact;                  // tanh' as mx_dact, or null
  const uint8_t *codes8, *scales8;  // [row][32 nb8], [row][nb8], or null
  int64_t nb8;
  int tanh;
};

enum { MX_SRC_DENSE, MX_SRC_TANH, MX_SRC_GRAD_Y, MX_SRC_GRAD_D, MX_SRC_I8, MX_SRC_I8_TANH, MX_SRC_FP4 };
struct MxSource {
  int kind, dtype;      // dtype: of p where it is dense, of the planes for 8 bits under tanh
  const void *p, *aux;  // aux: y or its derivative, or the scales
  bool half;            // one plane of fp16 instead of bf16 planes
};

struct MxOperand {  // K-contiguous rows
  const void* p;
  int64_t plane, pitch;  // bytes
  int planes;
  const void* scales;  // 4-bit operand: [tile of 8 blocks][half][row][4], else null
  bool half;           // the plane is fp16
};

struct MxProductPlan {
  int64_t tiles;
  int splits, most;  // parts of the contraction; what a shorter one of the same shape has at most
  bool big;
};

// rows x cols (or its transposed) as bf16 planes [planes][rows][cols up to 64]
void mx_planes(const MxSource& q, int64_t rows, int64_t cols, bool transposed, void* out, hipStream_t s);
// p(x) (kind: MX_SRC_DENSE or _TANH) as planes, and x in 8-bit blocks, from one read
void mx_planes_keep(const MxSource& q, int64_t rows, int64_t cols, void* out, uint8_t* codes, uint8_t* scales, hipStream_t s);
void mx_scale_tiles(const void* scales, int64_t rows, int64_t nb, void* out, hipStream_t s);
int mx_quantize4_for_product(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, hipStream_t s);
MxProductPlan mx_product_plan(int64_t m, int64_t n, int64_t kt, int npairs);
void mx_product(const MxOperand& a, const MxOperand& b, int64_t m, int64_t n, int64_t kt, const MxProductPlan& plan, int dtype,
                const MxEpilogue& e, float* parts, hipStream_t s);
void mx_sum_parts(const float* parts, int64_t count, int64_t m, int64_t n, int dtype, const MxEpilogue& e, hipStream_t s);
void mx_fold_parts(float* parts, int64_t count, int64_t elements, hipStream_t s);
void mx_column_totals(const float* parts, int64_t count, int64_t cols, int dtype, void* out, hipStream_t s);
void mx_column_sums(const MxSource& q, int64_t rows, int64_t cols, int64_t parts, float* out, hipStream_t s);

// a layer of at most 256 x 256 in one pass over the rows (fmd_mx_layer.hip)
enum { MX_WEIGHT_DENSE, MX_WEIGHT_FP4, MX_WEIGHT_FP4_BOTH, MX_WEIGHT_FP4_ACROSS };
struct MxLayer {
  const void *in, *aux;
  int pro;                     // MX_SRC_DENSE, _TANH, _GRAD_Y, _GRAD_D
  const void *w, *wscales;
  int weight;
  int64_t sk, sn;              // dense weight: strides of the contraction and of the outputs
  uint8_t *codes8, *scales8;   // written (null: not kept), or read for dtanh
  bool dtanh;
  MxEpilogue e;                // bias, out, dact, tanh
  float* sums;                 // MX_WEIGHT_FP4_ACROSS: workspace of mx_layer_sums_bytes for the input's column totals, or null
  void* totals;
};
int64_t mx_layer_sums_bytes(int64_t m, int64_t c);
bool mx_layer_fits(int64_t c, int64_t o);
int mx_layer(const MxLayer& l, int dtype, int64_t m, int64_t c, int64_t o, hipStream_t s);

// gw [k,n] and gb [n] (either may be null) of a narrow layer, or of few rows (fmd_mx_gradient.hip)
bool mx_gradient_fits(int64_t m, int64_t n, int64_t k);
int64_t mx_gradient_bytes(int dtype, int64_t m, int64_t n, int64_t k);
int mx_gradient(const void* g, const uint8_t* codes, const uint8_t* scales, bool tanh, int dtype, int64_t m, int64_t n, int64_t k,
                void* gw, void* gb, void* workspace, hipStream_t s);

// at most 64 rows through a layer with 4-bit weights of any width (fmd_mx_rows.hip)
bool mx_rows_fits(int64_t m);
int mx_rows(const void* x, int dtype, const void* codes, const void* scales, bool both, int64_t m, int64_t n, int64_t k,
            const MxEpilogue& e, hipStream_t s);

// the dynamic-LDS ceiling of a kernel, raised once on each device
template <class K>
hipError_t mx_allow_lds(K kernel, int bytes) {
  static bool done[64] = {};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev >= 0 && dev < 64 && done[dev]) return hipSuccess;
  e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

static inline int mx_dtype_size(int dtype) { return dtype == FMD_F32 ? 4 : 2; }
// a wide layer's products of 16-bit operands alone: one plane of their own type, to which computed ones are rounded (fmd_mx.h)
static inline bool mx_half(int dtype) { return dtype == FMD_F16; }
static inline int mx_own_planes(int dtype) { return dtype == FMD_F32 ? 3 : 1; }
static inline int mx_dtype_planes(int dtype) { return dtype == FMD_F32 ? 3 : dtype == FMD_F16 ? 2 : 1; }

// workspace laid out by the same code that uses it: with a null base it only counts
struct MxArena {
  char* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += mx_up(bytes, 256);
    return p;
  }
};

// What the translation units of the block-scaled layers share on the host side.
#pragma once
#include "fmd_mx.h"

struct MxEpilogue {            // v = acc (+ bias) (tanh) (* tanh'(8-bit value)) -> out
  const void* bias;            // in out's type, or null
  void* out;
  void* dact;                  // fp16 1 - tanh^2, or null
  const uint8_t *codes8, *scales8;  // [row][32 nb8], [row][nb8], or null
  int64_t nb8;
  int tanh;
};

enum { MX_SRC_DENSE, MX_SRC_TANH, MX_SRC_GRAD_Y, MX_SRC_GRAD_D, MX_SRC_I8, MX_SRC_I8_TANH, MX_SRC_FP4 };
struct MxSource {
  int kind, dtype;      // dtype: of p where it is dense, of the planes for 8 bits under tanh
  const void *p, *aux;  // aux: y or its derivative, or the scales
};

struct MxOperand {  // K-contiguous rows
  const void* p;
  int64_t plane, pitch;  // bytes
  int planes;
  const void* scales;  // 4-bit operand: [tile][row][8], else null
};

struct MxProductPlan {
  int64_t tiles;
  int splits;
  bool big;
};

// rows x cols (or its transposed) as bf16 planes [planes][rows][cols up to 64]
void mx_planes(const MxSource& q, int64_t rows, int64_t cols, bool transposed, void* out, hipStream_t s);
void mx_scale_tiles(const void* scales, int64_t rows, int64_t nb, void* out, hipStream_t s);
int mx_quantize4_for_product(const void* x, int dtype, int64_t m, int64_t k, void* codes, void* scales, hipStream_t s);
MxProductPlan mx_product_plan(int64_t m, int64_t n, int64_t kt, int npairs);
void mx_product(const MxOperand& a, const MxOperand& b, int64_t m, int64_t n, int64_t kt, const MxProductPlan& plan, int dtype,
                const MxEpilogue& e, float* parts, hipStream_t s);
void mx_sum_parts(const float* parts, int64_t count, int64_t m, int64_t n, int dtype, const MxEpilogue& e, hipStream_t s);
void mx_column_sums(const MxSource& q, int64_t rows, int64_t cols, int64_t parts, float* out, hipStream_t s);

static inline int mx_dtype_size(int dtype) { return dtype == FMD_F32 ? 4 : 2; }
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

// Entry points of the block-scaled layers: which kernels a call takes, and its workspace.
#include "fmd_mx_host.h"

namespace {

constexpr int64_t CHUNK_BYTES = (int64_t)128 << 20;  // planes of one chunk of rows: they stay in the last-level cache between the
                                                     // kernel that writes them and the product, and bound the workspace
// rows of a chunk: a multiple of 256, so that only the last one ends inside a tile
int64_t chunk_rows(int64_t m, int64_t row_bytes) {
  int64_t r = CHUNK_BYTES / row_bytes / 256 * 256;
  if (r < 1024) r = 1024;
  return r < m ? r : m;
}

const void* at(const void* p, int64_t elements, int size) { return p ? (const char*)p + elements * size : nullptr; }

MxEpilogue rows_of(const MxEpilogue& e, int64_t r0, int64_t n, int dtype) {
  MxEpilogue o = e;
  o.out = (void*)at(e.out, r0 * n, mx_dtype_size(dtype));
  o.dact = (void*)at(e.dact, r0 * n, 2);
  o.codes8 = (const uint8_t*)at(e.codes8, r0 * e.nb8 * 32, 1);
  o.scales8 = (const uint8_t*)at(e.scales8, r0 * e.nb8, 1);
  return o;
}

// out[m,n] = epi(A B^T), A = q [m,k] as planes, B already laid out; codes, scales: where q's 8-bit blocks go, or null; run = false
// only counts the workspace
void product_of_rows(MxArena& ar, bool run, MxSource q, int64_t m, int64_t k, const MxOperand& b, int64_t n, int dtype,
                     const MxEpilogue& e, hipStream_t s, uint8_t* codes = nullptr, uint8_t* scales = nullptr) {
  const int pa = q.half ? 1 : mx_dtype_planes(dtype);
  const int64_t pad = mx_up(k, 64), kt = pad / 64, rows = chunk_rows(m, pa * pad * 2);
  const MxProductPlan plan = mx_product_plan(rows, n, kt, mx_pairs(pa, b.planes).n);
  void* planes = ar.take(pa * rows * pad * 2);
  float* parts = plan.splits > 1 ? (float*)ar.take(plan.splits * rows * n * 4) : nullptr;
  if (!run) return;
  const int size = mx_dtype_size(q.dtype), aux = q.kind == MX_SRC_GRAD_Y ? 4 : 2;
  for (int64_t r0 = 0; r0 < m; r0 += rows) {
    const int64_t c = m - r0 < rows ? m - r0 : rows;
    MxSource part = q;
    part.p = at(q.p, r0 * k, size), part.aux = at(q.aux, r0 * k, aux);
    if (codes) mx_planes_keep(part, c, k, planes, codes + r0 * mx_blocks(k) * 32, scales + r0 * mx_blocks(k), s);
    else mx_planes(part, c, k, false, planes, s);
    const MxOperand a{planes, c * pad * 2, pad * 2, pa, nullptr, q.half};
    const MxEpilogue ep = rows_of(e, r0, n, dtype);
    mx_product(a, b, c, n, kt, plan, dtype, ep, parts, s);
    if (parts) mx_sum_parts(parts, plan.splits, c, n, dtype, ep, s);
  }
}

// out[k,n] = A^T B summed over the rows of A = qa [m,k] and B = qb [m,n], chunk by chunk in the order of the rows.  At most `room` of
// the chunks' parts are held; where there are more, those held are folded into the first, which the next ones follow: the order of the
// sums, and so their bits, do not depend on it.  Four at least, so that a fold serves three chunks (16384 x 8192 x 8192 fp32 23.1 ms
// against 23.0 with all of them held, 131072 x 8192 x 4096 bf16 18.8 against 18.6: 1.1 GiB of workspace for 2.1, 0.6 for 3.3).
void product_over_rows(MxArena& ar, bool run, MxSource qa, int pa, int64_t k, MxSource qb, int64_t n, int64_t m, int dtype, void* out,
                       hipStream_t s) {
  const int pb = mx_own_planes(dtype);
  const bool half = mx_half(dtype);
  const int64_t rows = chunk_rows(m, 2 * (pa * k + pb * n));
  const int64_t pad = mx_up(rows, 64), chunks = (m + rows - 1) / rows;
  const MxProductPlan plan = mx_product_plan(k, n, pad / 64, mx_pairs(pa, pb).n);
  void* ta = ar.take(pa * k * pad * 2);
  void* tb = ar.take(pb * n * pad * 2);
  int64_t room = CHUNK_BYTES / (k * n * 4);  // a chunk in parts has 33 MB of them at most (mx_product_plan)
  if (room < 4) room = 4;
  if (room > chunks * plan.most) room = chunks * plan.most;
  float* parts = room > 1 ? (float*)ar.take(room * k * n * 4) : nullptr;
  int64_t count = 0;  // the last chunk is shorter and may have fewer parts
  if (!run) return;
  const int64_t nb = mx_blocks(k);
  const MxEpilogue e{nullptr, out, nullptr, nullptr, nullptr, 0, 0};
  for (int64_t i = 0; i < chunks; ++i) {
    const int64_t r0 = i * rows, c = m - r0 < rows ? m - r0 : rows, cpad = mx_up(c, 64);
    MxSource a = qa, b = qb;
    a.p = at(qa.p, r0 * nb * 32, 1), a.aux = at(qa.aux, r0 * nb, 1);
    b.p = at(qb.p, r0 * n, mx_dtype_size(qb.dtype));
    mx_planes(a, c, k, true, ta, s);
    mx_planes(b, c, n, true, tb, s);
    const MxProductPlan here = c == rows ? plan : mx_product_plan(k, n, cpad / 64, mx_pairs(pa, pb).n);
    if (count + here.splits > room) {
      mx_fold_parts(parts, count, k * n, s);
      count = 1;
    }
    mx_product({ta, k * cpad * 2, cpad * 2, pa, nullptr, half}, {tb, n * cpad * 2, cpad * 2, pb, nullptr, half}, k, n, cpad / 64, here, dtype, e,
               parts ? parts + count * k * n : nullptr, s);
    count += here.splits;
  }
  if (parts) mx_sum_parts(parts, count, k, n, dtype, e, s);
}

void sum_over_rows(MxArena& ar, bool run, const MxSource& q, int64_t m, int64_t n, int dtype, void* out, hipStream_t s) {
  int64_t parts = (m + 255) / 256;
  const int64_t most = 4096 / ((n + 63) / 64);
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  float* p = (float*)ar.take(parts * n * 4);
  if (!run) return;
  mx_column_sums(q, m, n, parts, p, s);
  mx_column_totals(p, parts, n, dtype, out, s);
}

// The four calls below return the bytes of their workspace, or below zero the error of a launch that asked for it (which takes it
// from the runtime: what is not handed on is lost).
// ---- y = f(x^ W^T + b), W in 4-bit blocks -----------------------------------------------------------------------------
struct Fp4Linear {
  const void *x, *codes, *scales;
  int dtype;
  int64_t m, n, k;
  bool both;
  MxEpilogue e;
};

int64_t fp4_forward(const Fp4Linear& c, void* base, bool run, hipStream_t s) {
  MxArena ar{(char*)base, 0};
  if (mx_layer_fits(c.k, c.n)) {
    if (run)
      return mx_layer({c.x, nullptr, MX_SRC_DENSE, c.codes, c.scales, c.both ? MX_WEIGHT_FP4_BOTH : MX_WEIGHT_FP4, 0, 0, nullptr, nullptr, false,
                       c.e, nullptr, nullptr}, c.dtype, c.m, c.k, c.n, s);
    return 0;
  }
  if (mx_rows_fits(c.m)) {
    return run ? mx_rows(c.x, c.dtype, c.codes, c.scales, c.both, c.m, c.n, c.k, c.e, s) : 0;
  }
  const int64_t nb = mx_blocks(c.k);
  if (c.both) {
    const int64_t kt = (nb + 7) / 8;
    const MxProductPlan plan = mx_product_plan(c.m, c.n, kt, 1);
    void* xc = ar.take(c.m * nb * 16);
    void* xs = ar.take(mx_up(c.m, 4) * kt * 8);
    void* ws = ar.take(mx_up(c.n, 4) * kt * 8);
    float* parts = plan.splits > 1 ? (float*)ar.take(plan.splits * c.m * c.n * 4) : nullptr;
    if (run) {
      if (const int rc = mx_quantize4_for_product(c.x, c.dtype, c.m, c.k, xc, xs, s)) return rc;
      mx_scale_tiles(c.scales, c.n, nb, ws, s);
      mx_product({xc, 0, nb * 16, 1, xs, false}, {c.codes, 0, nb * 16, 1, ws, false}, c.m, c.n, kt, plan, c.dtype, c.e, parts, s);
      if (parts) mx_sum_parts(parts, plan.splits, c.m, c.n, c.dtype, c.e, s);
    }
  } else {
    const int64_t pad = mx_up(c.k, 64);
    void* w = ar.take(c.n * pad * 2);
    if (run) mx_planes({MX_SRC_FP4, FMD_BF16, c.codes, c.scales, false}, c.n, c.k, false, w, s);
    product_of_rows(ar, run, {MX_SRC_DENSE, c.dtype, c.x, nullptr, false}, c.m, c.k, {w, c.n * pad * 2, pad * 2, 1, nullptr, false}, c.n, c.dtype,
                    c.e, s);
  }
  return ar.used;
}

struct Fp4Backward {
  const void *g, *aux, *codes, *scales;
  void *gx, *gb;
  int dtype, kind;
  int64_t m, n, k;
};

int64_t fp4_backward(const Fp4Backward& c, void* base, bool run, bool want_gx, bool want_gb, hipStream_t s) {
  MxArena ar{(char*)base, 0};
  const MxSource g{c.kind, c.dtype, c.g, c.aux, false};
  const MxEpilogue to_gx{nullptr, c.gx, nullptr, nullptr, nullptr, 0, 0};
  if (want_gx && mx_layer_fits(c.n, c.k)) {
    float* sums = want_gb ? (float*)ar.take(mx_layer_sums_bytes(c.m, c.n)) : nullptr;
    if (run)
      return mx_layer({c.g, c.aux, c.kind, c.codes, c.scales, MX_WEIGHT_FP4_ACROSS, 0, 0, nullptr, nullptr, false, to_gx, sums, c.gb}, c.dtype, c.m,
               c.n, c.k, s);
    return ar.used;
  } else if (want_gx) {
    const int64_t pad = mx_up(c.n, 64);
    void* w = ar.take(c.k * pad * 2);
    if (run) mx_planes({MX_SRC_FP4, FMD_BF16, c.codes, c.scales, false}, c.n, c.k, true, w, s);
    product_of_rows(ar, run, g, c.m, c.n, {w, c.k * pad * 2, pad * 2, 1, nullptr, false}, c.k, c.dtype, to_gx, s);
  }
  if (want_gb) sum_over_rows(ar, run, g, c.m, c.n, c.dtype, c.gb, s);
  return ar.used;
}

// ---- y = p(x) W + b, x kept in 8-bit blocks ---------------------------------------------------------------------------
struct Kept {
  const void *x, *w, *g;
  uint8_t *codes, *scales;
  void *gx, *gw, *gb;
  int dtype;
  int64_t m, n, k;
  bool tanh;
  MxEpilogue e;
};

int64_t kept_forward(const Kept& c, void* base, bool run, hipStream_t s) {
  MxArena ar{(char*)base, 0};
  if (mx_layer_fits(c.k, c.n)) {
    if (run)
      return mx_layer({c.x, nullptr, c.tanh ? MX_SRC_TANH : MX_SRC_DENSE, c.w, nullptr, MX_WEIGHT_DENSE, c.n, 1, c.codes, c.scales, false, c.e, nullptr, nullptr},
               c.dtype, c.m, c.k, c.n, s);
    return 0;
  }
  const int p = mx_own_planes(c.dtype);
  const bool half = mx_half(c.dtype);
  const int64_t pad = mx_up(c.k, 64);
  void* w = ar.take(p * c.n * pad * 2);
  if (run) mx_planes({MX_SRC_DENSE, c.dtype, c.w, nullptr, half}, c.k, c.n, true, w, s);
  product_of_rows(ar, run, {c.tanh ? MX_SRC_TANH : MX_SRC_DENSE, c.dtype, c.x, nullptr, half}, c.m, c.k,
                  {w, c.n * pad * 2, pad * 2, p, nullptr, half}, c.n, c.dtype, c.e, s, c.codes, c.scales);
  return ar.used;
}

int64_t kept_backward(const Kept& c, void* base, bool run, bool want_gx, bool want_gw, bool want_gb, hipStream_t s) {
  MxArena ar{(char*)base, 0};
  const int p = mx_own_planes(c.dtype);
  const bool half = mx_half(c.dtype);
  const MxSource g{MX_SRC_DENSE, c.dtype, c.g, nullptr, half};
  const bool narrow = mx_layer_fits(c.n, c.k);
  if (want_gx && narrow) {
    if (run) {
      const int rc = mx_layer({c.g, nullptr, MX_SRC_DENSE, c.w, nullptr, MX_WEIGHT_DENSE, 1, c.n, c.tanh ? c.codes : nullptr,
                               c.tanh ? c.scales : nullptr, c.tanh, {nullptr, c.gx, nullptr, nullptr, nullptr, 0, 0}, nullptr, nullptr},
                              c.dtype, c.m, c.n, c.k, s);
      if (rc) return rc;
    }
  } else if (want_gx) {
    const int64_t pad = mx_up(c.n, 64);
    void* w = ar.take(p * c.k * pad * 2);
    if (run) mx_planes({MX_SRC_DENSE, c.dtype, c.w, nullptr, half}, c.k, c.n, false, w, s);
    MxEpilogue e{nullptr, c.gx, nullptr, nullptr, nullptr, 0, 0};
    if (c.tanh) e.codes8 = c.codes, e.scales8 = c.scales, e.nb8 = mx_blocks(c.k);
    product_of_rows(ar, run, g, c.m, c.n, {w, c.k * pad * 2, pad * 2, p, nullptr, half}, c.k, c.dtype, e, s);
  }
  if ((want_gw || want_gb) && mx_gradient_fits(c.m, c.n, c.k)) {  // the bias's sums come along
    const int64_t bytes = mx_gradient_bytes(c.dtype, c.m, c.n, c.k);
    void* part = bytes ? ar.take(bytes) : nullptr;
    if (run) return mx_gradient(c.g, c.codes, c.scales, c.tanh, c.dtype, c.m, c.n, c.k, c.gw, c.gb, part, s);
    return ar.used;
  }
  if (want_gw)
    product_over_rows(ar, run, {c.tanh ? MX_SRC_I8_TANH : MX_SRC_I8, c.dtype, c.codes, c.scales, half}, c.tanh ? p : 1, c.k, g, c.n, c.m,
                      c.dtype, c.gw, s);
  if (want_gb) sum_over_rows(ar, run, g, c.m, c.n, c.dtype, c.gb, s);
  return ar.used;
}

// Up to 2^20 a side of a weight (grids of 64 and 32 columns count in 16 bits), 2^34 rows (steps of 16 count in 32) and 2^38 elements
// a matrix (at most 2^22 + 2^21 tiles of a product: fewer than 2^32 threads); the rows of a 4-bit x go through one product.
bool bad_sizes(int dtype, int64_t m, int64_t n, int64_t k, bool both = false) {
  const int64_t side = (int64_t)1 << 20, most = (int64_t)1 << 38;
  return dtype < 0 || dtype > 2 || m < 0 || n < 1 || k < 1 || m > (int64_t)1 << (both ? 29 : 34) || n > side || k > side ||
         m * n > most || m * k > most || n * k > most;
}
bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

}  // namespace

extern "C" int64_t fmd_mxfp4_linear_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k, int quantize_input) {
  if (bad_sizes(dtype, m, n, k, quantize_input != 0)) return FMD_EINVAL;
  if (m == 0) return 0;
  Fp4Linear c{nullptr, nullptr, nullptr, dtype, m, n, k, quantize_input != 0, {}};
  return fp4_forward(c, nullptr, false, nullptr);
}

extern "C" int fmd_mxfp4_linear(const void* x, int dtype, const void* codes, const void* scales, const void* bias, void* y, void* dact,
                                int64_t m, int64_t n, int64_t k, int tanh, int quantize_input, void* workspace, void* stream) {
  if (bad_sizes(dtype, m, n, k, quantize_input != 0)) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!x || !codes || !scales || !y || off16(x) || off16(codes) || off16(y) || off16(workspace) || off16(dact) || (dact && !tanh)) return FMD_EINVAL;
  const Fp4Linear c{x, codes, scales, dtype, m, n, k, quantize_input != 0, {bias, y, dact, nullptr, nullptr, 0, tanh}};
  if (!workspace && fp4_forward(c, nullptr, false, nullptr)) return FMD_EINVAL;
  if (const int64_t rc = fp4_forward(c, workspace, true, fmd_stream(stream)); rc < 0) return (int)rc;
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

extern "C" int64_t fmd_mxfp4_linear_bwd_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k, int want_gx, int want_gbias) {
  if (bad_sizes(dtype, m, n, k)) return FMD_EINVAL;
  Fp4Backward c{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, dtype, MX_SRC_DENSE, m, n, k};
  return fp4_backward(c, nullptr, false, want_gx && m, want_gbias, nullptr);
}

extern "C" int fmd_mxfp4_linear_bwd(const void* g, int dtype, const void* aux, int aux_kind, const void* codes, const void* scales,
                                    void* gx, void* gbias, int64_t m, int64_t n, int64_t k, void* workspace, void* stream) {
  if (bad_sizes(dtype, m, n, k) || aux_kind < 0 || aux_kind > 2 || (aux_kind == FMD_AUX_Y) != (aux_kind && dtype == FMD_F32))
    return FMD_EINVAL;
  if (m && (!g || off16(g) || (aux_kind && (!aux || off16(aux))) || (gx && (!codes || !scales || off16(gx) || off16(codes)))))
    return FMD_EINVAL;
  if (!gx && !gbias) return FMD_OK;
  if (off16(workspace)) return FMD_EINVAL;
  const int kind = aux_kind == FMD_AUX_Y ? MX_SRC_GRAD_Y : aux_kind == FMD_AUX_DACT ? MX_SRC_GRAD_D : MX_SRC_DENSE;
  const Fp4Backward c{g, aux, codes, scales, gx, gbias, dtype, kind, m, n, k};
  if (!workspace && fp4_backward(c, nullptr, false, gx && m, gbias, nullptr)) return FMD_EINVAL;
  if (const int64_t rc = fp4_backward(c, workspace, true, gx && m, gbias, fmd_stream(stream)); rc < 0) return (int)rc;
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

extern "C" int64_t fmd_linear_ckpt8_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k) {
  if (bad_sizes(dtype, m, n, k)) return FMD_EINVAL;
  if (m == 0) return 0;
  Kept c{};
  c.dtype = dtype, c.m = m, c.n = n, c.k = k;
  return kept_forward(c, nullptr, false, nullptr);
}

extern "C" int fmd_linear_ckpt8(const void* x, int dtype, const void* w, const void* bias, void* y, void* codes, void* scales, int64_t m,
                                int64_t n, int64_t k, int tanh, void* workspace, void* stream) {
  if (bad_sizes(dtype, m, n, k) || (codes != nullptr) != (scales != nullptr)) return FMD_EINVAL;
  if (m == 0) return FMD_OK;
  if (!x || !w || !y || off16(x) || off16(w) || off16(y) || off16(codes) || off16(workspace)) return FMD_EINVAL;
  Kept c{};
  c.x = x, c.w = w, c.codes = (uint8_t*)codes, c.scales = (uint8_t*)scales, c.dtype = dtype, c.m = m, c.n = n, c.k = k, c.tanh = tanh != 0;
  c.e = {bias, y, nullptr, nullptr, nullptr, 0, 0};
  if (!workspace && kept_forward(c, nullptr, false, nullptr)) return FMD_EINVAL;
  if (const int64_t rc = kept_forward(c, workspace, true, fmd_stream(stream)); rc < 0) return (int)rc;
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

extern "C" int64_t fmd_linear_ckpt8_bwd_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k, int tanh, int want_gx, int want_gw,
                                                        int want_gbias) {
  if (bad_sizes(dtype, m, n, k)) return FMD_EINVAL;
  if (m == 0) return 0;
  Kept c{};
  c.dtype = dtype, c.m = m, c.n = n, c.k = k, c.tanh = tanh != 0;
  return kept_backward(c, nullptr, false, want_gx, want_gw, want_gbias, nullptr);
}

extern "C" int fmd_linear_ckpt8_bwd(const void* g, int dtype, const void* codes, const void* scales, const void* w, void* gx, void* gw,
                                    void* gbias, int64_t m, int64_t n, int64_t k, int tanh, void* workspace, void* stream) {
  if (bad_sizes(dtype, m, n, k) || m == 0) return FMD_EINVAL;
  if (!gx && !gw && !gbias) return FMD_OK;
  const bool kept = gw || (gx && tanh);
  if (!g || off16(g) || off16(workspace) || off16(gw) || (gx && (!w || off16(w) || off16(gx))) || (kept && (!codes || !scales || off16(codes))))
    return FMD_EINVAL;
  Kept c{};
  c.g = g, c.w = w, c.codes = (uint8_t*)codes, c.scales = (uint8_t*)scales, c.gx = gx, c.gw = gw, c.gb = gbias;
  c.dtype = dtype, c.m = m, c.n = n, c.k = k, c.tanh = tanh != 0;
  if (!workspace && kept_backward(c, nullptr, false, gx, gw, gbias, nullptr)) return FMD_EINVAL;
  if (const int64_t rc = kept_backward(c, workspace, true, gx, gw, gbias, fmd_stream(stream)); rc < 0) return (int)rc;
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

// mx4_abi.cu — entry points of the MXFP4 operators (declared in include/oxg_b200.h): argument checks and one
// launch each. They keep nothing between calls and use no workspace, so calls on different streams, and
// captured graphs, are independent of one another; the products share only the context's error word.
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/oxg_b200.h"
#include "ctx_internal.h"
#include "mx4.h"

namespace oxg {

namespace {
// Words given back, oldest first: a graph that outlives its context may still write to that context's word, so one
// is used again only when all have been in use.
std::mutex words_lock;
int words_back[kMx4ErrWords], back_first = 0, back_n = 0;  // a ring
int words_new = 0;
}  // namespace

int mx4_word_take() {
  std::lock_guard<std::mutex> g(words_lock);
  if (words_new < kMx4ErrWords - 1) return words_new++;
  if (back_n == 0) return kMx4ErrWords - 1;  // the last one is shared by what comes beyond
  const int w = words_back[back_first];
  back_first = (back_first + 1) % kMx4ErrWords;
  --back_n;
  return w;
}

void mx4_word_give(int word) {
  if (word < 0 || word >= kMx4ErrWords - 1) return;
  int unread;
  if (mx4_take_error(word, &unread) != cudaSuccess) return;  // not known to be clear: it stays unused
  std::lock_guard<std::mutex> g(words_lock);
  words_back[(back_first + back_n++) % kMx4ErrWords] = word;
}

int mx4_check_error(oxg_ctx *ctx, int word) {
  if (word < 0) return OXG_OK;
  int h = 0;
  const cudaError_t st = mx4_take_error(word, &h);
  if (st != cudaSuccess) return ctx_error(ctx, OXG_ERR_CUDA, cudaGetErrorString(st));
  if (h == kMx4ErrCounts)
    return ctx_error(ctx, OXG_ERR_SHAPE,
                     "oxg_mxfp4_grouped_matmul: a group's count was negative, or the counts added up to more rows than there are");
  if (h) return ctx_error(ctx, OXG_ERR_TIMEOUT, "a pipeline wait of an MXFP4 product timed out");
  return OXG_OK;
}

}  // namespace oxg

namespace {

int fail(oxg_ctx *ctx, int status, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return oxg::ctx_error(ctx, status, buf);
}

struct DevGuard {
  int prev = -1, dev;
  explicit DevGuard(int d) : dev(d) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DevGuard() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
};

template <class F>
int run(oxg_ctx *ctx, const char *name, F &&fn) {
  DevGuard g(oxg::ctx_device(ctx));
  const cudaError_t st = oxg::ctx_launch(ctx, name, fn);
  if (st == cudaSuccess) return OXG_OK;
  return fail(ctx, st == cudaErrorMemoryAllocation ? OXG_ERR_OOM : OXG_ERR_CUDA, "%s launch: %s (%s)", name, cudaGetErrorName(st),
              cudaGetErrorString(st));
}

bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

int quantize(oxg_ctx *ctx, oxg::Mx4QuantArgs &a, int dtype, bool swiglu) {
  const size_t width = swiglu ? 2 : 1, size = dtype == OXG_DTYPE_F32 ? 4 : 2;
  if (dtype != OXG_DTYPE_F32 && dtype != OXG_DTYPE_BF16 && dtype != OXG_DTYPE_F16)
    return fail(ctx, OXG_ERR_INVALID_ARG, "unknown element type %d", dtype);
  if (a.rule != OXG_MX_FLOOR && a.rule != OXG_MX_NOCLIP) return fail(ctx, OXG_ERR_INVALID_ARG, "unknown scale rule %d", a.rule);
  if (a.tiled != OXG_SCALES_ROWS && a.tiled != OXG_SCALES_TILED)
    return fail(ctx, OXG_ERR_INVALID_ARG, "unknown scale layout %d", a.tiled);
  if (a.cols % 32 != 0) return fail(ctx, OXG_ERR_SHAPE, "cols must be divisible by 32, got %zu", a.cols);
  if (a.cols > 0x7FFFFFE0u) return fail(ctx, OXG_ERR_SHAPE, "cols must be below 2^31, got %zu", a.cols);
  if (a.rows == 0 || a.cols == 0) return OXG_OK;
  if (a.rows > 1 && a.ld < width * a.cols)
    return fail(ctx, OXG_ERR_SHAPE, "ld must be at least the %zu elements of a row, got %zu", width * a.cols, a.ld);
  const size_t pitch = a.ld > width * a.cols ? a.ld : width * a.cols;
  if (pitch > SIZE_MAX / 8 / a.rows) return fail(ctx, OXG_ERR_SHAPE, "rows * ld overflows: %zu x %zu", a.rows, pitch);
  if (!a.x || !a.blocks || !a.scales) return fail(ctx, OXG_ERR_INVALID_ARG, "input, blocks and scales must be non-NULL");
  if (!aligned(a.x, size)) return fail(ctx, OXG_ERR_INVALID_ARG, "the input must be aligned to its elements");
  if (!aligned(a.blocks, 4)) return fail(ctx, OXG_ERR_INVALID_ARG, "blocks must be 4-byte aligned");
  if (!aligned(a.row_scale, 4)) return fail(ctx, OXG_ERR_INVALID_ARG, "row_scale must be 4-byte aligned");
  return run(ctx, swiglu ? "swiglu_quantize_mxfp4" : "quantize_mxfp4", [&] {
    return oxg::launch_mx4_quantize(a, dtype, swiglu, oxg::ctx_n_sms(ctx), oxg::ctx_stream(ctx));
  });
}

constexpr int kMost = 0x7FFFFE00;  // 32-bit numbers with room for a tile

int product(oxg_ctx *ctx, oxg::Mx4GemmArgs &a, int out_dtype) {
  if (a.m < 0 || a.n < 0) return fail(ctx, OXG_ERR_SHAPE, "m and n must not be negative, got %d and %d", a.m, a.n);
  if (a.m > kMost || a.n > kMost || a.k > kMost)
    return fail(ctx, OXG_ERR_SHAPE, "m, n and k must be at most %d, got %d, %d and %d", kMost, a.m, a.n, a.k);
  if (a.k <= 0 || a.k % 32) return fail(ctx, OXG_ERR_SHAPE, "k must be a positive multiple of 32, got %d", a.k);
  if (out_dtype != OXG_DTYPE_F32 && out_dtype != OXG_DTYPE_BF16)
    return fail(ctx, OXG_ERR_INVALID_ARG, "the output must be f32 or bf16, got element type %d", out_dtype);
  if (a.m == 0 || a.n == 0 || a.groups == 0) return OXG_OK;
  if (a.m > 1 && a.ldo < (size_t)a.n) return fail(ctx, OXG_ERR_SHAPE, "ldo must be at least n = %d, got %zu", a.n, a.ldo);
  if (a.ldo > SIZE_MAX / 8 / (size_t)a.m) return fail(ctx, OXG_ERR_SHAPE, "m * ldo overflows: %d x %zu", a.m, a.ldo);
  if (!a.a || !a.a_scales || !a.b || !a.b_scales || !a.out)
    return fail(ctx, OXG_ERR_INVALID_ARG, "blocks, scales and out must be non-NULL");
  if (!aligned(a.a, 16) || !aligned(a.b, 16)) return fail(ctx, OXG_ERR_INVALID_ARG, "blocks must be 16-byte aligned");
  if (!aligned(a.a_scales, 4) || !aligned(a.b_scales, 4))
    return fail(ctx, OXG_ERR_INVALID_ARG, "tiled scales must be 4-byte aligned");
  if (!aligned(a.bias, 2)) return fail(ctx, OXG_ERR_INVALID_ARG, "bias must be 2-byte aligned");
  a.out_bf16 = out_dtype == OXG_DTYPE_BF16;
  if (!aligned(a.out, a.out_bf16 ? 2 : 4)) return fail(ctx, OXG_ERR_INVALID_ARG, "out must be aligned to its elements");
  a.err_word = oxg::ctx_mx4_word(ctx);
  return run(ctx, a.counts ? "mxfp4_grouped_matmul" : "mxfp4_matmul",
             [&] { return oxg::launch_mx4_gemm(a, oxg::ctx_n_sms(ctx), oxg::ctx_stream(ctx)); });
}

}  // namespace

extern "C" {

int oxg_quantize_mxfp4(oxg_ctx *ctx, const void *x, int dtype, size_t rows, size_t cols, size_t ld, const float *row_scale,
                       int scale_rule, int scale_layout, uint8_t *blocks, uint8_t *scales) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  oxg::Mx4QuantArgs a{};
  a.x = x;
  a.ld = ld;
  a.rows = rows;
  a.cols = cols;
  a.row_scale = row_scale;
  a.rule = scale_rule;
  a.tiled = scale_layout;
  a.blocks = blocks;
  a.scales = scales;
  return quantize(ctx, a, dtype, false);
}

int oxg_swiglu_quantize_mxfp4(oxg_ctx *ctx, const void *gate_up, int dtype, size_t rows, size_t cols, size_t ld, float alpha,
                              float limit, int scale_rule, int scale_layout, uint8_t *blocks, uint8_t *scales) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  if (!(limit > 0.f)) return fail(ctx, OXG_ERR_INVALID_ARG, "limit must be positive, got %g", (double)limit);
  oxg::Mx4QuantArgs a{};
  a.x = gate_up;
  a.ld = ld;
  a.rows = rows;
  a.cols = cols;
  a.rule = scale_rule;
  a.tiled = scale_layout;
  a.alpha = alpha;
  a.limit = limit;
  a.blocks = blocks;
  a.scales = scales;
  return quantize(ctx, a, dtype, true);
}

int oxg_mxfp4_tile_scales(oxg_ctx *ctx, const uint8_t *scales, size_t n_groups, size_t rows, size_t cols, uint8_t *tiled) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  if (cols % 32 != 0) return fail(ctx, OXG_ERR_SHAPE, "cols must be divisible by 32, got %zu", cols);
  if (cols > 0x7FFFFFE0u) return fail(ctx, OXG_ERR_SHAPE, "cols must be below 2^31, got %zu", cols);
  if (n_groups == 0 || rows == 0 || cols == 0) return OXG_OK;
  if (rows > SIZE_MAX / cols || n_groups > SIZE_MAX / (rows * cols))
    return fail(ctx, OXG_ERR_SHAPE, "n_groups * rows * cols overflows: %zu x %zu x %zu", n_groups, rows, cols);
  if (!scales || !tiled) return fail(ctx, OXG_ERR_INVALID_ARG, "scales and tiled must be non-NULL");
  if (!aligned(tiled, 4)) return fail(ctx, OXG_ERR_INVALID_ARG, "tiled must be 4-byte aligned");
  return run(ctx, "mxfp4_tile_scales", [&] {
    return oxg::launch_mx4_tile_scales(scales, n_groups, rows, cols, tiled, oxg::ctx_n_sms(ctx), oxg::ctx_stream(ctx));
  });
}

int oxg_mxfp4_matmul(oxg_ctx *ctx, const uint8_t *a_blocks, const uint8_t *a_scales, int m, const uint8_t *b_blocks,
                     const uint8_t *b_scales, int n, int k, const uint16_t *bias, void *out, int out_dtype, size_t ldo) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  oxg::Mx4GemmArgs a{};
  a.m = m;
  a.n = n;
  a.k = k;
  a.a = a_blocks;
  a.a_scales = reinterpret_cast<const uint32_t *>(a_scales);
  a.b = b_blocks;
  a.b_scales = reinterpret_cast<const uint32_t *>(b_scales);
  a.bias = bias;
  a.out = out;
  a.ldo = ldo;
  return product(ctx, a, out_dtype);
}

int oxg_mxfp4_grouped_matmul(oxg_ctx *ctx, const uint8_t *a_blocks, const uint8_t *a_scales, int m, const int32_t *counts_dev,
                             int n_groups, const uint8_t *b_blocks, const uint8_t *b_scales, int n, int k, const uint16_t *bias,
                             void *out, int out_dtype, size_t ldo) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  if (n_groups < 0 || n_groups > oxg::kMx4MaxGroups)
    return fail(ctx, OXG_ERR_SHAPE, "n_groups must be in [0, %d], got %d", oxg::kMx4MaxGroups, n_groups);
  if (n_groups > 0 && !counts_dev) return fail(ctx, OXG_ERR_INVALID_ARG, "counts must be non-NULL");
  if (!aligned(counts_dev, 4)) return fail(ctx, OXG_ERR_INVALID_ARG, "counts must be 4-byte aligned");
  oxg::Mx4GemmArgs a{};
  a.m = m;
  a.n = n;
  a.k = k;
  a.groups = n_groups;
  a.counts = counts_dev;
  a.a = a_blocks;
  a.a_scales = reinterpret_cast<const uint32_t *>(a_scales);
  a.b = b_blocks;
  a.b_scales = reinterpret_cast<const uint32_t *>(b_scales);
  a.bias = bias;
  a.out = out;
  a.ldo = ldo;
  return product(ctx, a, out_dtype);
}

// Not part of the interface: either product with a kernel of the caller's choice (-1: the library's own), for tests that
// hold every kernel to the same sizes. ran: the kernel taken and the CTAs that split its K. groups < 0: not grouped.
__attribute__((visibility("default"))) int oxgtest_mxfp4_product(oxg_ctx *ctx, const uint8_t *a_blocks, const uint8_t *a_scales,
                                                                 int m, const int32_t *counts_dev, int groups,
                                                                 const uint8_t *b_blocks, const uint8_t *b_scales, int n, int k,
                                                                 const uint16_t *bias, void *out, int out_dtype, size_t ldo,
                                                                 int kernel, int ranks, int *ran) {
  if (!ctx) return fail(nullptr, OXG_ERR_INVALID_ARG, "ctx is NULL");
  if (kernel < oxg::kMx4Auto || kernel > oxg::kMx4Split) return fail(ctx, OXG_ERR_INVALID_ARG, "unknown kernel %d", kernel);
  if (groups > oxg::kMx4MaxGroups || (groups > 0 && !counts_dev))
    return fail(ctx, OXG_ERR_INVALID_ARG, "groups without counts, or too many");
  oxg::Mx4GemmArgs a{};
  a.m = m;
  a.n = n;
  a.k = k;
  a.groups = groups < 0 ? 1 : groups;
  a.counts = groups < 0 ? nullptr : counts_dev;
  a.a = a_blocks;
  a.a_scales = reinterpret_cast<const uint32_t *>(a_scales);
  a.b = b_blocks;
  a.b_scales = reinterpret_cast<const uint32_t *>(b_scales);
  a.bias = bias;
  a.out = out;
  a.ldo = ldo;
  a.kernel = kernel;
  a.ranks = ranks;
  a.ran = ran;
  return product(ctx, a, out_dtype);
}

}  // extern "C"

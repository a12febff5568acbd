// mx4.h — host-side launchers of the MXFP4 operators: quantisation
// (mx4_quant.cu) and the products of two MXFP4 operands (mx4_gemm.cu).
// Internal to the library.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace oxg {

#ifdef __CUDACC__
// The MXFP4 kernels are launched as programmatic dependents and let their own dependents start at once: the next
// one's launch and setup then overlap this one's end. Every thread that touches memory which an earlier kernel
// may have written, or writes any, first waits for all of the earlier kernel; through that kernel's own wait
// this covers every kernel before it.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Loads of what an earlier kernel may have written, for behind that wait: this kernel may have been resident while
// the earlier one still wrote, so the non-coherent path (ld.global.nc, __ldg), which is for data that nothing writes
// while a kernel runs, is not for them. It costs the same (8192 x 2880 quantised from bf16: 10.9 us with
// either, 64 x 201088 x 2880 product: 61.4).
__device__ __forceinline__ uint4 ld_stream_v4(const void *p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_u32(const void *p) {
  uint32_t r;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_u32_if(bool go, const void *p) {  // 0 where not
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "mov.b32 %0, 0;\n\t"
      "@q ld.global.u32 %0, [%1];\n\t}"
      : "=&r"(r)
      : "l"(p), "r"((int)go));
  return r;
}
__device__ __forceinline__ float ld_f32(const float *p) { return __uint_as_float(ld_u32(p)); }
__device__ __forceinline__ uint16_t ld_u16(const void *p) {
  uint16_t r;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_u8(const void *p) {
  uint32_t r;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
#endif

// Element types and scale rules and layouts, as the public header numbers them.
enum { kMx4F32 = 0, kMx4Bf16 = 1, kMx4F16 = 2 };
enum { kMx4Floor = 0, kMx4NoClip = 1 };
enum { kMx4ScaleRows = 0, kMx4ScaleTiled = 1 };

struct Mx4QuantArgs {
  const void *x = nullptr;           // [rows, cols] (SwiGLU: [rows, 2 cols], gate and up interleaved)
  size_t ld = 0;                     // elements from one row to the next
  size_t rows = 0, cols = 0;         // of the quantised matrix; cols a multiple of 32
  size_t scale_rows = 0;             // rows of the tiled scales (set by the launch)
  const float *row_scale = nullptr;  // [rows] factors, or null
  int rule = kMx4Floor;
  int tiled = 0;
  float alpha = 0.f, limit = 0.f;    // SwiGLU
  uint8_t *blocks = nullptr;         // [rows, cols / 2], 4-byte aligned
  uint8_t *scales = nullptr;         // [rows, cols / 32], or tiled [ceil(cols / 128), rows, 4]
};
cudaError_t launch_mx4_quantize(const Mx4QuantArgs &a, int dtype, bool swiglu, int n_sms, cudaStream_t stream);

// Scale rows [groups, rows, cols / 32] -> tiled [groups, ceil(cols / 128), rows, 4].
cudaError_t launch_mx4_tile_scales(const uint8_t *src, size_t groups, size_t rows, size_t cols, uint8_t *dst, int n_sms,
                                   cudaStream_t stream);

constexpr int kMx4MaxGroups = 1024;
// Error words of the products: part of the library's module on every device, so that a context's word costs no
// allocation and a captured launch may outlive the context that it was captured with.
constexpr int kMx4ErrWords = 4096;
// Error-word codes of the products.
constexpr int kMx4ErrWait = 81;    // a pipeline wait ran out
constexpr int kMx4ErrCounts = 85;  // a negative group count, or counts beyond the rows there are

// The products' kernels: single CTAs, pairs of them, clusters that split K.
enum { kMx4Auto = -1, kMx4Few = 0, kMx4Pair = 1, kMx4Split = 2 };

struct Mx4GemmArgs {
  int m = 0, n = 0, k = 0;           // activation rows, weight rows (per group), reduction length
  int groups = 1;
  const int32_t *counts = nullptr;   // [groups] rows of each group (device), or null: one group of m rows
  const uint8_t *a = nullptr;        // [m, k / 2] codes
  const uint32_t *a_scales = nullptr;  // [ceil(k / 128), m]
  const uint8_t *b = nullptr;        // [groups, n, k / 2] codes
  const uint32_t *b_scales = nullptr;  // [groups, ceil(k / 128), n]
  const uint16_t *bias = nullptr;    // [groups, n] bf16, or null
  void *out = nullptr;               // [m, ldo]
  size_t ldo = 0;
  int out_bf16 = 0;                  // else f32
  int err_word = 0;                  // below kMx4ErrWords
  int kernel = kMx4Auto, ranks = 0;  // for tests: this kernel whatever the sizes; CTAs that split K
  int *ran = nullptr;                // for tests: the kernel taken, and its ranks
};
cudaError_t launch_mx4_gemm(const Mx4GemmArgs &a, int n_sms, cudaStream_t stream);
// Reads an error word of the current device, and clears it where it is set. Waits for nothing but itself.
cudaError_t mx4_take_error(int word, int *code);

}  // namespace oxg

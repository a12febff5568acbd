// mx4_quant.cu — floating-point rows to MXFP4, alone or behind the clamped SwiGLU.
//
// A block of 32 elements with largest magnitude t gets the scale
//   floor rule:   s = 2^(floor(log2 t) - 2)       (t / s in [4, 8): what lies above 6 becomes 6)
//   noclip rule:  twice that where t > 1.5 * 2^floor(log2 t)   (t / s in (3, 6]: nothing clips)
// but at least 2^-126, so that the byte 0, which means 0.0 to the dequantisation and 2^-127 to the tensor
// cores, never comes up, and at most 2^125, so that what was finite reads back finite (4 * 2^126 would not
// in f32 or bf16). Each element becomes the E2M1 value nearest to x / s, ties to the even code
// (cvt.rn.satfinite.e2m1x2; x / s is exact, s being a power of two). A block that holds an infinity or a
// NaN becomes codes 0 under scale byte 255, which reads as NaN everywhere.
//
// Bound: HBM. A thread owns 8 consecutive elements (one 16-byte load of 16-bit types, two of f32) and a
// block is four neighbouring lanes, which share the largest magnitude by two shuffles; the codes leave as
// one 4-byte word per thread. Each thread issues 64 bytes of loads before it works on the first; a block takes
// one contiguous run of chunks and ends.
#include "common.cuh"
#include "mx4.h"

namespace oxg {
namespace {

constexpr int kThreads = 128;  // SwiGLU prompt from bf16: 85 us, against 95 with 256 threads, 107 with 512 and 100 with 64

template <int T>
struct Elem;
template <>
struct Elem<kMx4F32> {
  static constexpr int kBytes = 4;
};
template <>
struct Elem<kMx4Bf16> {
  static constexpr int kBytes = 2;
};
template <>
struct Elem<kMx4F16> {
  static constexpr int kBytes = 2;
};

// N consecutive elements as raw 16-byte words. Without VEC (a base or a row pitch off the 16-byte grid)
// they are read one by one.
template <int T, int N, bool VEC>
struct Raw {
  static constexpr int kWords = N * Elem<T>::kBytes / 16;
  uint4 w[kWords];
  __device__ __forceinline__ void load(const void *p) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = ld_stream_v4(static_cast<const uint4 *>(p) + i);
    } else if (Elem<T>::kBytes == 4) {
      uint32_t *d = reinterpret_cast<uint32_t *>(w);
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = ld_u32(static_cast<const uint32_t *>(p) + i);
    } else {
      uint32_t *d = reinterpret_cast<uint32_t *>(w);
      const uint16_t *s = static_cast<const uint16_t *>(p);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) d[i] = (uint32_t)ld_u16(s + 2 * i) | ((uint32_t)ld_u16(s + 2 * i + 1) << 16);
    }
  }
  __device__ __forceinline__ void values(float (&v)[N]) const {
    const uint32_t *d = reinterpret_cast<const uint32_t *>(w);
    if (T == kMx4F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __uint_as_float(d[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (T == kMx4Bf16) {
          v[2 * i] = __uint_as_float(d[i] << 16);
          v[2 * i + 1] = __uint_as_float(d[i] & 0xFFFF0000u);
        } else {
          const float2 f = unpack_f16x2(d[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  }
};

// Two f32 operations in one instruction (each rounded on its own).
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Eight values to four code bytes, element 0 in the lowest half byte.
__device__ __forceinline__ uint32_t e2m1_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint32_t pack_scaled(const float (&v)[8], float f) {
  float r[8];
  const uint64_t f2 = pair(f, f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 t = halves(mul2(pair(v[i], v[i + 1]), f2));
    r[i] = t.x;
    r[i + 1] = t.y;
  }
  return e2m1_pack8(r);
}

// Scale byte of a block from the f32 bits of its largest magnitude (finite).
__device__ __forceinline__ int scale_byte(uint32_t top, int rule) {
  const int b = (int)(top >> 23) - 2 + ((rule == kMx4NoClip && (top & 0x7FFFFFu) > 0x400000u) ? 1 : 0);
  return b < 1 ? 1 : (b > 252 ? 252 : b);
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// max and min that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// f32 bits of a block's largest magnitude (NaN if it holds one), shared by its four lanes
__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
  float t = max3_abs_nan(max3_abs_nan(v[0], v[1], v[2]), max3_abs_nan(v[3], v[4], v[5]), max_nan(fabsf(v[6]), fabsf(v[7])));
  t = max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
  return __float_as_uint(max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2)));
}

__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], int rule, int *byte) {
  const uint32_t top = block_top(v);
  if (top >= 0x7F800000u) {
    *byte = 255;
    return 0u;
  }
  *byte = scale_byte(top, rule);
  return pack_scaled(v, inverse_scale(*byte));
}

// The clamped SwiGLU in f64, correct to far below an f32 rounding.
__device__ __forceinline__ double swiglu_f64(float gf, float uf, float alpha, float limit) {
  const double g = gf > limit ? limit : gf, u = uf < -limit ? -limit : (uf > limit ? limit : uf);
  return g * (1.0 / (1.0 + exp(-(double)alpha * g))) * (u + 1.0);
}

// Eight SwiGLU outputs from their gate / up pairs, quantised as the exact values would be. The f32 value comes
// from the hardware's exponential and reciprocal (expf and the IEEE quotient: 210 us for 32768 x 2880 from bf16).
// For x = -alpha g <= 40 its relative error stays below kTol = 2^-17 = 128 2^-24: log2 e, -alpha log2 e and its
// product with g are rounded, 2.5 2^-24 |x| in e^x; ex2 adds 2^-22, the reciprocal 2^-23, the sum, u + 1 and two
// products 2^-24 each, 110 2^-24 in all, as long as nothing leaves f32's normal range. What does is off by 2^-150
// (1 + limit) at most, which is nothing to a block whose scale is 2^-100 or more while limit <= 2^18, and to
// one that is zero throughout (its exact values lie below the smallest scale's first border). So where the
// block's largest magnitude or a scaled element lies within kTol of a border between two scales or two codes
// (the latter seen by rounding both (1 - kTol) and (1 + kTol) times the value), or where one of these conditions
// does not hold, the block's four lanes evaluate it again in f64: about 1 block in 300 of normally distributed
// inputs. The codes then do not depend on which exponential computed them. Gates far out cost more: 32768 x 2880 from
// bf16 takes 93 us (tiled scales) with gates of deviation 2, 124 with 5, 312 with 8 and 470 where every block has one
// below -23.
constexpr float kTol = 0x1p-17f;
__device__ __forceinline__ uint32_t swiglu_quantize8_f64(const float (&gu)[16], float alpha, float limit, int rule, int *byte,
                                                      uint32_t lanes) {
  double h[8], top = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = swiglu_f64(gu[2 * i], gu[2 * i + 1], alpha, limit);
    top = top != top || fabs(h[i]) <= top ? top : fabs(h[i]);  // a NaN stays
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    const double other = __shfl_xor_sync(lanes, top, o);
    top = top != top || other <= top ? top : other;
  }
  if (!(top < 0x1p128)) {  // what f32 does not hold
    *byte = 255;
    return 0u;
  }
  const long long bits = __double_as_longlong(top);
  int b = (int)(bits >> 52) - 1023 + 127 - 2;
  if (rule == kMx4NoClip && (bits & 0xFFFFFFFFFFFFFll) > 0x8000000000000ll) b += 1;
  *byte = b = b < 1 ? 1 : (b > 252 ? 252 : b);
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double r = scalbn(fabs(h[i]), 127 - b);
    const uint32_t c = (r > 0.25) + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5.0);
    w |= (c | (signbit(h[i]) ? 8u : 0u)) << (4 * i);
  }
  return w;
}
__device__ __forceinline__ uint32_t swiglu_quantize8(const float (&gu)[16], float alpha, float limit, int rule, int *byte) {
  const float c = -alpha * 1.4426950408889634f;  // e^(-alpha g) = 2^(c g)
  const uint64_t one = pair(1.f, 1.f), c2 = pair(c, c);
  float h[8];
  uint64_t sum2 = 0ull;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t g = pair(min_nan(gu[2 * i], limit), min_nan(gu[2 * i + 2], limit));
    const uint64_t u = pair(max_nan(min_nan(gu[2 * i + 1], limit), -limit), max_nan(min_nan(gu[2 * i + 3], limit), -limit));
    const float2 x = halves(mul2(c2, g));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
    const uint64_t e2 = pair(e.x, e.y);
    const float2 d = halves(add2(one, e2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
    const float2 v = halves(mul2(mul2(g, pair(r.x, r.y)), add2(u, one)));
    h[i] = v.x;
    h[i + 1] = v.y;
    sum2 = add2(sum2, e2);
  }
  const float sum = halves(sum2).x + halves(sum2).y;
  bool close = sum > 0x1p57f;  // some x beyond 40 (40 log2 e > 57)
  if (!(limit <= 0x1p18f)) {   // without a clamp that means something, every gate that is neither 0 nor ordinary
#pragma unroll
    for (int i = 0; i < 8; ++i) close |= fabsf(gu[2 * i]) < 0x1p-40f && gu[2 * i] != 0.f;
  }
  const uint32_t top = block_top(h);
  const bool finite = top < 0x7F800000u;
  close |= top == 0x7F800000u;            // an overflow, perhaps only of the f32 arithmetic
  close |= top - 1u < (29u << 23) - 1u;   // scales below 2^-100, but for a block of zeros
  close |= ((top + 128u) & 0x3FFFFFu) < 256u;  // within 128 2^-23 of a power of two or of 1.5 times one
  *byte = finite ? scale_byte(top, rule) : 255;
  const float inv = inverse_scale(finite ? *byte : 1);
  const uint32_t w = pack_scaled(h, inv * (1.0f - kTol));
  close |= w != pack_scaled(h, inv * (1.0f + kTol));
  const uint32_t lanes = 0xFu << (threadIdx.x & 28);
  if ((__ballot_sync(0xFFFFFFFFu, close) & lanes) != 0u)  // the four lanes of a block go together
    return swiglu_quantize8_f64(gu, alpha, limit, rule, byte, lanes);
  return finite ? w : 0u;
}

// n / d for n below 2^32 by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994): the compiler's division costs as much as a chunk's arithmetic.
struct Div {
  uint32_t d, mul, shift;
  explicit Div(uint32_t d_) : d(d_) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) ++l;
    mul = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
    shift = l ? l - 1 : 0;
    if (d == 1) mul = 0;
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    if (d == 1) return n;
    const uint32_t t = __umulhi(mul, n);
    return (t + ((n - t) >> 1)) >> shift;
  }
};

// How rows lie: one after another with scales in rows and no factors (a chunk's place is its number), on the
// 16-byte grid with any pitch, or anyhow.
enum Lay { kFlat, kGrid, kAny };

template <int T, bool SWIGLU, Lay LAY, int UNR>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(const Mx4QuantArgs a, uint32_t n_chunks, const Div per_row) {
  constexpr int N = SWIGLU ? 16 : 8;
  launch_dependents();
  wait_prerequisites();
  // every lane of a warp goes through the shuffles below; chunks come in fours, so blocks stay whole
  const uint32_t c0 = blockIdx.x * (UNR * kThreads) + threadIdx.x;
  Raw<T, N, LAY != kAny> raw[UNR];
  uint32_t row[UNR], col[UNR];
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const uint32_t c = c0 + u * kThreads;
    if (LAY != kFlat) {
      row[u] = per_row.quotient(c);
      col[u] = c - row[u] * per_row.d;
    }
    const size_t at = LAY == kFlat ? (size_t)c * N : row[u] * a.ld + (size_t)col[u] * N;
    if (c < n_chunks)
      raw[u].load(static_cast<const uint8_t *>(a.x) + at * Elem<T>::kBytes);
    else
#pragma unroll
      for (int i = 0; i < Raw<T, N, LAY != kAny>::kWords; ++i) raw[u].w[i] = make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const uint32_t c = c0 + u * kThreads;
    float v[N];
    raw[u].values(v);
    int byte;
    uint32_t w;
    if constexpr (SWIGLU) {
      w = swiglu_quantize8(v, a.alpha, a.limit, a.rule, &byte);
    } else {
      if (LAY != kFlat && a.row_scale) {
        const float f = c < n_chunks ? ld_f32(a.row_scale + row[u]) : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fmul_rn(v[i], f);
      }
      w = quantize8(v, a.rule, &byte);
    }
    if (c >= n_chunks) continue;
    reinterpret_cast<uint32_t *>(a.blocks)[c] = w;
    if ((c & 3) == 0) {
      if (LAY == kFlat || !a.tiled) {
        a.scales[c >> 2] = (uint8_t)byte;
      } else {
        const uint32_t kb = col[u] >> 2;
        uint8_t *d = a.scales + ((size_t)(kb >> 2) * a.scale_rows + row[u]) * 4;
        d[kb & 3] = (uint8_t)byte;
        if (col[u] + 4 == per_row.d)  // zero where the row ends inside a 128-element stretch
          for (uint32_t j = (kb & 3) + 1; j < 4; ++j) d[j] = 0;
      }
    }
  }
}

// One thread per 4-byte word, consecutive rows side by side in the output.
__global__ void __launch_bounds__(kThreads)
    mx4_tile_scales_kernel(const uint8_t *src, size_t n_words, size_t rows, uint32_t kb, uint32_t words, uint32_t *dst) {
  launch_dependents();
  wait_prerequisites();
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n_words; i += (size_t)gridDim.x * kThreads) {
    const size_t r = i % rows, q = i / rows, g = q / words;
    const uint32_t b0 = (uint32_t)(q - g * words) * 4;
    const uint8_t *s = src + (g * rows + r) * kb + b0;
    uint32_t w = 0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      if (b0 + j < kb) w |= ld_u8(s + j) << (8 * j);
    dst[i] = w;
  }
}

template <class... P, class... A>
cudaError_t launch_dependent(void (*kernel)(P...), unsigned grid, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
template <int T, bool SWIGLU, Lay LAY, int UNR>
cudaError_t launch_unr(const Mx4QuantArgs &a, cudaStream_t stream) {
  const uint32_t n_chunks = (uint32_t)(a.rows * (a.cols / 8));
  return launch_dependent(mx4_quantize_kernel<T, SWIGLU, LAY, UNR>, (n_chunks + UNR * kThreads - 1) / (UNR * kThreads), stream,
                          a, n_chunks, Div((uint32_t)(a.cols / 8)));
}
template <int T, bool SWIGLU, Lay LAY>
cudaError_t launch_lay(Mx4QuantArgs a, int n_sms, cudaStream_t stream) {
  // 64 bytes of loads in flight per thread, once there is a chunk for every thread that fits the GPU
  constexpr int UNR = 4 / (Elem<T>::kBytes / 2) / (SWIGLU ? 2 : 1);
  const size_t width = a.cols * (SWIGLU ? 2 : 1) * Elem<T>::kBytes;
  // 32-bit chunk numbers: a kernel takes the rows of at most 2^31 chunks (34 GB of bf16)
  const size_t most = ((size_t)1 << 31) / (a.cols / 8), rows = a.rows;
  a.scale_rows = rows;
  for (size_t r = 0; r < rows; r += most) {
    a.rows = rows - r < most ? rows - r : most;
    const cudaError_t st = a.rows * (a.cols / 8) <= (size_t)n_sms * 2048 ? launch_unr<T, SWIGLU, LAY, 1>(a, stream)
                                                                        : launch_unr<T, SWIGLU, LAY, UNR>(a, stream);
    if (st) return st;
    a.x = static_cast<const uint8_t *>(a.x) + a.rows * (a.ld * Elem<T>::kBytes > width ? a.ld * Elem<T>::kBytes : width);
    a.blocks += a.rows * (a.cols / 2);
    a.scales += a.rows * (a.tiled ? 4 : a.cols / 32);
    if (a.row_scale) a.row_scale += a.rows;
  }
  return cudaSuccess;
}
template <int T, bool SWIGLU>
cudaError_t launch_op(const Mx4QuantArgs &a, int n_sms, cudaStream_t stream) {
  if ((uintptr_t)a.x % 16 != 0 || (a.rows > 1 && a.ld * Elem<T>::kBytes % 16 != 0)) return launch_lay<T, SWIGLU, kAny>(a, n_sms, stream);
  const bool flat = (a.rows == 1 || a.ld == a.cols * (SWIGLU ? 2 : 1)) && !a.tiled && !a.row_scale;
  return flat ? launch_lay<T, SWIGLU, kFlat>(a, n_sms, stream) : launch_lay<T, SWIGLU, kGrid>(a, n_sms, stream);
}
template <int T>
cudaError_t launch_typed(const Mx4QuantArgs &a, bool swiglu, int n_sms, cudaStream_t stream) {
  return swiglu ? launch_op<T, true>(a, n_sms, stream) : launch_op<T, false>(a, n_sms, stream);
}

}  // namespace

cudaError_t launch_mx4_quantize(const Mx4QuantArgs &a, int dtype, bool swiglu, int n_sms, cudaStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return cudaSuccess;
  if (dtype == kMx4F32) return launch_typed<kMx4F32>(a, swiglu, n_sms, stream);
  if (dtype == kMx4Bf16) return launch_typed<kMx4Bf16>(a, swiglu, n_sms, stream);
  return launch_typed<kMx4F16>(a, swiglu, n_sms, stream);
}

cudaError_t launch_mx4_tile_scales(const uint8_t *src, size_t groups, size_t rows, size_t cols, uint8_t *dst, int n_sms,
                                   cudaStream_t stream) {
  const uint32_t kb = (uint32_t)(cols / 32), words = (kb + 3) / 4;
  const size_t n_words = groups * rows * words;
  if (n_words == 0) return cudaSuccess;
  const size_t want = (n_words + kThreads - 1) / kThreads, cap = (size_t)n_sms * 32;
  return launch_dependent(mx4_tile_scales_kernel, (unsigned)(want < cap ? want : cap), stream, src, n_words, rows, kb, words,
                          reinterpret_cast<uint32_t *>(dst));
}

}  // namespace oxg

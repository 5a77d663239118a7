// What the normalisation and checkpoint kernels share: 8 channels of a pixel as one access in any storage type, the
// activations and their derivatives, the walk of a block over pixels x channels, and the 8-bit block format.
#pragma once
#include "common.h"

namespace miseg {

struct bf16s {};                                  // storage types
struct f16s {};
struct f32s {};

template <typename T> struct Vec8 { uint4 v; };   // 8 values as they lie in memory
template <> struct Vec8<f32s> { uint4 v, w; };

template <typename T> struct Elem { static constexpr int bytes = 2; };
template <> struct Elem<f32s> { static constexpr int bytes = 4; };

template <typename T> __device__ __forceinline__ Vec8<T> load8(const char* p) {
  Vec8<T> r;
  r.v = *reinterpret_cast<const uint4*>(p);
  if constexpr (Elem<T>::bytes == 4) r.w = *reinterpret_cast<const uint4*>(p + 16);
  return r;
}
template <typename T> __device__ __forceinline__ void store8(char* p, const Vec8<T>& r) {
  *reinterpret_cast<uint4*>(p) = r.v;
  if constexpr (Elem<T>::bytes == 4) *reinterpret_cast<uint4*>(p + 16) = r.w;
}

typedef __attribute__((ext_vector_type(2))) _Float16 nf16x2;
__device__ __forceinline__ float f16lo(unsigned v) { return (float)__builtin_bit_cast(nf16x2, v)[0]; }
__device__ __forceinline__ float f16hi(unsigned v) { return (float)__builtin_bit_cast(nf16x2, v)[1]; }
__device__ __forceinline__ unsigned f16pack(float lo, float hi) {
  nf16x2 b = {(_Float16)lo, (_Float16)hi};        // nearest even; out of range becomes infinity, which a loss scaler has to see
  return __builtin_bit_cast(unsigned, b);
}

template <typename T> __device__ __forceinline__ void unpack8(float (&f)[8], const Vec8<T>& r) {
  const unsigned u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, bf16s)) { f[2 * i] = bf16lo_to_f32(u[i]); f[2 * i + 1] = bf16hi_to_f32(u[i]); }
    else if constexpr (__is_same(T, f16s)) { f[2 * i] = f16lo(u[i]); f[2 * i + 1] = f16hi(u[i]); }
    else f[i] = __uint_as_float(u[i]);
  }
  if constexpr (__is_same(T, f32s)) {
    f[4] = __uint_as_float(r.w.x); f[5] = __uint_as_float(r.w.y);
    f[6] = __uint_as_float(r.w.z); f[7] = __uint_as_float(r.w.w);
  }
}
// results are rounded once, to nearest even, where they leave
template <typename T> __device__ __forceinline__ Vec8<T> pack8(const float (&f)[8]) {
  Vec8<T> r;
  if constexpr (__is_same(T, bf16s)) {
    r.v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else if constexpr (__is_same(T, f16s)) {
    r.v = make_uint4(f16pack(f[0], f[1]), f16pack(f[2], f[3]), f16pack(f[4], f[5]), f16pack(f[6], f[7]));
  } else {
    r.v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    r.w = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
  }
  return r;
}

// ---- activations: 0 none, 1 relu, 2 silu
enum { NA_NONE = 0, NA_RELU = 1, NA_SILU = 2 };
__device__ __forceinline__ float sigmoid_f32(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
template <int ACT> __device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == NA_RELU) return z < 0.f ? 0.f : z;            // a NaN stays one
  if constexpr (ACT == NA_SILU) return z * sigmoid_f32(z);
  return z;
}
template <int ACT> __device__ __forceinline__ float act_bwd(float z, float dy) {   // dy * act'(z)
  if constexpr (ACT == NA_RELU) return z > 0.f ? dy : 0.f;
  if constexpr (ACT == NA_SILU) {
    const float s = sigmoid_f32(z);
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}

// ---- pixels x channels over a grid: blockIdx = (pixel chunk, channel slab, image).  A slab is `cw` groups of 8
// channels, a multiple of 4 so that the four lanes of a 32-channel block are neighbours; a block's 256 threads are
// `rows` pixels x cw groups, and a thread keeps its 8 channels for its whole walk.
constexpr int kNormThreads = 256;
struct NormGrid {
  int cw, ny, rows;                                // groups of 8 channels per slab, slabs, pixels per sweep
  int chunk, blocks;                               // pixels per block (a multiple of rows), blocks per image
};

// Blocks enough to fill the chip (`want` in all), but none with less than `least` sweeps.
static inline NormGrid norm_grid(long long N, long long pixels, int C, int want, int least) {
  NormGrid g;
  const int c8 = ((C + 31) / 32) * 4;
  g.ny = (c8 + 63) / 64;
  g.cw = ((c8 + g.ny - 1) / g.ny + 3) / 4 * 4;
  g.rows = kNormThreads / g.cw;
  long long b = (want + N * g.ny - 1) / (N * g.ny);
  const long long most = (pixels + (long long)g.rows * least - 1) / ((long long)g.rows * least);
  if (b > most) b = most;
  if (b < 1) b = 1;
  long long chunk = (pixels + b - 1) / b;
  chunk = (chunk + g.rows - 1) / g.rows * g.rows;
  g.chunk = (int)chunk;
  g.blocks = (int)((pixels + chunk - 1) / chunk);
  return g;
}

struct NormWalk {
  long long p0, p1;                                // pixels of this block
  int c, r, n;                                     // first channel, pixel of the sweep, image
  bool active;
  __device__ __forceinline__ NormWalk(const NormGrid& g, long long pixels, int C) {
    r = threadIdx.x / g.cw;
    c = (blockIdx.y * g.cw + threadIdx.x - r * g.cw) * 8;
    n = blockIdx.z;
    p0 = (long long)blockIdx.x * g.chunk;
    p1 = p0 + g.chunk < pixels ? p0 + g.chunk : pixels;
    active = r < g.rows && c < C;
  }
};

__device__ __forceinline__ void load_coef(float (&f)[8], const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// ---- the 8-bit block format: 32 consecutive channels of a pixel share a bf16 scale, bf16(amax / 127).
// code = rint(v / scale): |code| <= 127 because the scale's rounding moves amax / scale by at most 2^-9 of 127, less than
// half a step.  Below 2^-119 the scale would be a subnormal number and its reciprocal infinite: such a block is zero.  A
// value that is not finite makes the scale NaN, so that all of its block reads back as NaN and an overflow is not lost.
struct Quant8 { uint2 codes; bf16_t scale; };
__device__ __forceinline__ Quant8 quantise8(const float (&v)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {                    // magnitudes compared as integers: a NaN is above infinity
    const unsigned b = __float_as_uint(v[j]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const unsigned b = (unsigned)__shfl_xor((int)m, o, 4);
    m = b > m ? b : m;
  }
  Quant8 q;
  const float amax = __uint_as_float(m);
  float s = amax < 0x1p-119f ? 0.f : amax / 127.f;
  q.scale = m >= 0x7f800000u ? (bf16_t)0x7fc0 : f32_to_bf16(s);
  s = bf16_to_f32(q.scale);
  const float inv = s > 0.f ? 1.f / s : 0.f;       // 0 for a zero and for a NaN scale
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = inv > 0.f ? rintf(v[j] * inv) : 0.f;
    w[j >> 2] |= ((unsigned)(int)f & 0xffu) << (8 * (j & 3));
  }
  q.codes = make_uint2(w[0], w[1]);
  return q;
}
__device__ __forceinline__ void dequantise8(float (&v)[8], uint2 codes, float s) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)(int)(signed char)((j < 4 ? codes.x : codes.y) >> (8 * (j & 3))) * s;
}

// y may be x itself, or another channel range of the same buffer; any other overlap would be read after it was written.
static inline bool views_clash(const void* a, long long apix, long long aimg, const void* b, long long bpix, long long bimg,
                               long long N, long long pixels, int C, int bytes) {
  if (!a || !b) return false;
  const char *pa = (const char*)a, *pb = (const char*)b;
  const long long ea = ((N - 1) * aimg + (pixels - 1) * apix + C) * bytes, eb = ((N - 1) * bimg + (pixels - 1) * bpix + C) * bytes;
  if (pa + ea <= pb || pb + eb <= pa) return false;
  if (apix != bpix || (N > 1 && aimg != bimg)) return true;
  if (pa == pb) return false;
  long long d = pa < pb ? pb - pa : pa - pb;
  if (N > 1 && aimg < pixels * apix) return true;
  return d < (long long)C * bytes || d + (long long)C * bytes > apix * bytes;
}

}  // namespace miseg

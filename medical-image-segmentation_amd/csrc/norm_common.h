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

// NT: the line is not kept in the caches (nontemporal).  Of 157 MB read twice, a second pass that also writes 157 MB takes
// 38 us when the first left them in the 256 MB memory-side cache, 56 us when they come from HBM.
typedef __attribute__((ext_vector_type(4))) unsigned nt_u32x4;
template <bool NT> __device__ __forceinline__ uint4 load16(const char* p) {
  if constexpr (NT) {
    const nt_u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const nt_u32x4*>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
  }
  return *reinterpret_cast<const uint4*>(p);
}
template <bool NT> __device__ __forceinline__ void store16(char* p, uint4 v) {
  if constexpr (NT) {
    const nt_u32x4 w = {v.x, v.y, v.z, v.w};
    __builtin_nontemporal_store(w, reinterpret_cast<nt_u32x4*>(p));
  } else {
    *reinterpret_cast<uint4*>(p) = v;
  }
}
template <typename T, bool NT = false> __device__ __forceinline__ Vec8<T> load8(const char* p) {
  Vec8<T> r;
  r.v = load16<NT>(p);
  if constexpr (Elem<T>::bytes == 4) r.w = load16<NT>(p + 16);
  return r;
}
template <typename T, bool NT = false> __device__ __forceinline__ void store8(char* p, const Vec8<T>& r) {
  store16<NT>(p, r.v);
  if constexpr (Elem<T>::bytes == 4) store16<NT>(p + 16, r.w);
}
// 8 codes
typedef __attribute__((ext_vector_type(2))) unsigned nt_u32x2;
template <bool NT> __device__ __forceinline__ uint2 load_codes(const signed char* p) {
  if constexpr (NT) {
    const nt_u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const nt_u32x2*>(p));
    return make_uint2(v.x, v.y);
  }
  return *reinterpret_cast<const uint2*>(p);
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
  if constexpr (ACT == NA_RELU) return __builtin_elementwise_maximum(z, 0.f);   // a NaN stays one
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
// channels, at most 64 (a multiple of 4 where 32-channel blocks are written, so that their four lanes are neighbours); a
// block's 256 threads are `rows` pixels x cw groups, and a thread keeps its 8 channels for its whole walk.
constexpr int kNormThreads = 256;
struct NormGrid {
  int cw, ny, rows;                                // groups of 8 channels per slab, slabs, pixels per sweep
  int chunk, blocks;                               // pixels per block (a multiple of rows), blocks per image
};

// Blocks enough to fill the chip (`want` in all and no more, or the last ones run alone: 197 MB of statistics 35 us with 504
// blocks, 42 with 516, when 512 are two a CU), none with less than `least` sweeps unless there are few of them anyway.
static inline NormGrid norm_grid(long long N, long long pixels, int C, int want, int least, bool whole32 = false) {
  NormGrid g;
  const int unit = whole32 ? 4 : 1, c8 = (C / 8 + unit - 1) / unit * unit;
  g.ny = (c8 + 63) / 64;
  g.cw = ((c8 + g.ny - 1) / g.ny + unit - 1) / unit * unit;
  g.rows = kNormThreads / g.cw;
  const long long sweeps = (pixels + g.rows - 1) / g.rows, all = sweeps * N * g.ny;
  if (all < (long long)least * 1024) least = (int)(all / 1024) + 1;
  long long b = want / (N * g.ny);
  const long long most = (sweeps + least - 1) / least;
  if (b < 1) b = 1;
  if (b > most) b = most;
  long long chunk = (pixels + b - 1) / b;
  chunk = (chunk + g.rows - 1) / g.rows * g.rows;
  g.chunk = (int)chunk;
  g.blocks = (int)((pixels + chunk - 1) / chunk);
  return g;
}

struct NormWalk {
  int p0, p1;                                      // pixels of this block
  int c, r, n;                                     // first channel, pixel of the sweep, image
  bool active;
  __device__ __forceinline__ NormWalk(const NormGrid& g, int block, int pixels, int C) {
    r = threadIdx.x / g.cw;
    c = (blockIdx.y * g.cw + threadIdx.x - r * g.cw) * 8;
    n = blockIdx.z;
    p0 = block * g.chunk;
    p1 = p0 + g.chunk < pixels ? p0 + g.chunk : pixels;
    active = r < g.rows && c < C;
  }
};

__device__ __forceinline__ void load_coef(float (&f)[8], const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// Parameters of 8 channels, `none` where there are none; a slice of a flat parameter buffer need not be aligned.
__device__ __forceinline__ void load_param(float (&f)[8], const float* p, int c, float none) {
  if (p && ((uintptr_t)p & 15) == 0) {
    load_coef(f, p + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p ? p[c + j] : none;
  }
}
__device__ __forceinline__ void store_coef(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
// A layer's parameters, and where a call leaves what it read of them (or nowhere).
struct NormParams {
  const float *gamma, *beta;
  float *gamma_kept, *beta_kept;
  __device__ __forceinline__ void keep(int c) const {
    float f[8];
    if (gamma_kept) { load_param(f, gamma, c, 1.f); store_coef(gamma_kept + c, f); }
    if (beta_kept) { load_param(f, beta, c, 0.f); store_coef(beta_kept + c, f); }
  }
};

// ---- the 8-bit block format: 32 consecutive channels of a pixel share a bf16 scale, bf16(amax / 127).
// code = rint(v / scale): |code| <= 127 because the scale's rounding moves amax / scale by at most 2^-8 of 127, to 127.496,
// less than half a step.  Below 2^-119 the scale would be a subnormal number and its reciprocal infinite: such a block is zero.  A
// value that is not finite makes the scale NaN, so that all of its block reads back as NaN and an overflow is not lost.
struct Quant8 { uint2 codes; bf16_t scale; };
// The definition's operations are single 32-bit roundings: m / 127 and 1 / scale, here by a reciprocal and a correction
// (equal to the rounded quotient for every magnitude that is kept and for every bf16 scale), v * (1 / scale), and rint, by
// adding 1.5 * 2^23: the sum's lowest byte is the code.  No product may be contracted into a sum, except in corrections.
__device__ __forceinline__ Quant8 quantise8(const float (&v)[8]) {
#pragma clang fp contract(off)
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
  float s = amax * (1.f / 127.f);
  s = fmaf(fmaf(-127.f, s, amax), 1.f / 127.f, s);
  q.scale = m >= 0x7f800000u ? (bf16_t)0x7fc0 : amax < 0x1p-119f ? (bf16_t)0 : f32_to_bf16(s);
  s = bf16_to_f32(q.scale);
  float inv = __builtin_amdgcn_rcpf(s);
  inv = fmaf(fmaf(-s, inv, 1.f), inv, inv);
  unsigned w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float t = v[4 * h + j] * inv;
      b[j] = __float_as_uint(t + 12582912.f);
    }
    w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400),
                                 0x05040100);
    if (!(s > 0.f)) w[h] = 0;                      // a zero or NaN scale
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
  if ((pixels > 1 && apix != bpix) || (N > 1 && aimg != bimg)) return true;
  if (pa == pb) return false;
  const long long d = pa < pb ? pb - pa : pa - pb;
  if (pixels == 1) {                               // the pixel stride has no meaning: images lie where pixels do otherwise
    if (N == 1) return true;
    apix = aimg;
  } else if (N > 1 && aimg < pixels * apix) {
    return true;
  }
  return d < (long long)C * bytes || d + (long long)C * bytes > apix * bytes;
}

}  // namespace miseg

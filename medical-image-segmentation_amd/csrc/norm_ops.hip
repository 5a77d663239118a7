// Group normalisation with an activation on channels-last tensors, forward and backward, and activation checkpoints in
// 8 bits: their writing, their reading, and the backward pass out of them.
#include "norm_common.h"

namespace miseg {

// ------------------------------------------------------------------------------------------------ forward statistics
// Per block and channel: mean and sum of squared differences from it.  A thread sums (x - k) and (x - k)^2 with k its own
// first value, so that an offset of the channel that is large against its spread does not cancel; threads and blocks are
// joined by counts, means and sums of squares.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void gn_stats_kernel(const char* x, long long xps, long long ximg, int pixels,
                                                                int C, NormGrid g, float2* __restrict__ part) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  __shared__ float lmean[kNormThreads * 8], lm2[kNormThreads * 8];
  __shared__ int lcount[kNormThreads];
  __shared__ double2 lsum[kNormThreads];
  NormWalk w(g, blockIdx.x, pixels, C);
  float k[8], s1[8], s2[8];
  int count = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) k[j] = s1[j] = s2[j] = 0.f;
  int px = w.p0 + w.r;
  if (w.active && px < w.p1) {
    const char* xp = x + (w.n * ximg + px * xps + w.c) * ES;
    const long long step = g.rows * xps * ES;
    unpack8(k, load8<T>(xp));
    for (; px < w.p1; px += U * g.rows, xp += U * step) {
      Vec8<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (px + u * g.rows < w.p1) v[u] = load8<T>(xp + u * step);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (px + u * g.rows < w.p1) {
          float f[8];
          unpack8(f, v[u]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float d = f[j] - k[j];
            s1[j] += d;
            s2[j] = fmaf(d, d, s2[j]);
          }
          ++count;
        }
    }
  }
  const float rc = count ? 1.f / (float)count : 0.f;
  if ((int)threadIdx.x == w.r * g.cw) lcount[w.r] = count;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lmean[threadIdx.x * 8 + j] = k[j] + s1[j] * rc;
    lm2[threadIdx.x * 8 + j] = s2[j] - s1[j] * s1[j] * rc;
  }
  __syncthreads();
  // channel i of the slab from `parts` threads, then from one
  const int wide = g.cw * 8, parts = wide < kNormThreads ? kNormThreads / wide : 1;
  for (int i0 = 0; i0 < wide; i0 += kNormThreads) {
    const int i = i0 + (int)threadIdx.x % wide, q = (int)threadIdx.x / wide;
    double sum = 0, sq = 0;
    if (q < parts && i < wide)
      for (int r = q; r < g.rows; r += parts) {
        const double m = lmean[r * wide + i], n = lcount[r];
        sum += n * m;
        sq += lm2[r * wide + i] + n * m * m;
      }
    if (parts > 1) {
      lsum[threadIdx.x] = make_double2(sum, sq);
      __syncthreads();
      if (q == 0)
        for (int t = 1; t < parts; ++t) {
          sum += lsum[t * wide + i].x;
          sq += lsum[t * wide + i].y;
        }
    }
    const int c = blockIdx.y * wide + i;
    if (q == 0 && i < wide && c < C) {
      const double mean = sum / (w.p1 - w.p0);
      part[((long long)w.n * gridDim.x + blockIdx.x) * C + c] = make_float2((float)mean, (float)(sq - sum * mean));
    }
  }
}

// Sum over the 256 threads of a block, in every thread.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// One block per (group, image): the blocks' statistics of the group's channels in 64 bits, then the coefficients.
__global__ __launch_bounds__(kNormThreads) void gn_finalize_kernel(const float2* __restrict__ part, int blocks, int chunk,
                                                                   long long pixels, int C, int groups,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, float eps,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   float* __restrict__ scale, float* __restrict__ shift,
                                                                   float* __restrict__ qs, float* __restrict__ qt) {
  __shared__ double lds[4];
  const int w = C / groups, g = blockIdx.x, n = blockIdx.y;
  double s = 0, q = 0;
  const int entries = blocks * w, last = (int)(pixels - (long long)(blocks - 1) * chunk);
  const float2* pp = part + (long long)n * blocks * C + g * w;
  constexpr int U = 8;                             // loads in flight: the kernel waits for nothing else
  for (int e0 = threadIdx.x; e0 < entries; e0 += U * kNormThreads) {
    float2 v[U];
    int count[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kNormThreads, b = e / w;
      count[u] = e >= entries ? 0 : b == blocks - 1 ? last : chunk;
      v[u] = e < entries ? pp[(long long)b * C + (e - b * w)] : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const double n = count[u], m = v[u].x;
      s += n * m;
      q += (double)v[u].y + n * m * m;
    }
  }
  s = block_sum(s, lds);
  q = block_sum(q, lds);
  const double count = (double)pixels * w, m = s / count;
  double var = q / count - m * m;
  if (var < 0) var = 0;
  const double r = 1.0 / sqrt(var + (double)eps);
  if (threadIdx.x == 0) {
    mean[n * groups + g] = (float)m;
    rstd[n * groups + g] = (float)r;
  }
  for (int i = threadIdx.x; i < w; i += kNormThreads) {
    const int c = g * w + i;
    const double a = gamma ? gamma[c] * r : r;
    scale[(long long)n * C + c] = (float)a;
    shift[(long long)n * C + c] = (float)((beta ? beta[c] : 0.0) - m * a);
    if (qs) {
      qs[(long long)n * C + c] = (float)r;
      qt[(long long)n * C + c] = (float)(-m * r);
    }
  }
}

// ---------------------------------------------------------------------------- one pass: activated result, checkpoint
// y = act(x a + b) and the checkpoint of x s + t (of x without s), either or both.  Coefficients per channel, `cimg` from
// one image's to the next's.  A block makes one sweep of U pixels per thread where there is work for 32768 blocks: short
// blocks keep more loads and stores in flight than long walks (operand of 4 x 960 x 1280 x 64 out of 8 bits: 200 us with
// 4096 blocks, 158 with 32768).  x is read for the last time here and y is read by another kernel: neither stays in the
// caches.  The last pixels come first, as they are the likeliest to be in the caches still.
struct PassArgs {
  const char* x;
  char* y;
  signed char* codes;
  bf16_t* scales;
  const float *a, *b, *s, *t;
  long long xps, ximg, yps, yimg, cimg;
  int pixels, C;
  NormGrid g;
};

template <typename T, int ACT, bool Y, bool Q>
__global__ __launch_bounds__(kNormThreads) void norm_pass_kernel(PassArgs p) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  NormWalk w(p.g, gridDim.x - 1 - blockIdx.x, p.pixels, p.C);
  if (w.r >= p.g.rows) return;                    // lanes past the last channel stay for the exchange in quantise8
  float a[8], b[8], s[8], t[8];
  if (w.active) {
    if (Y) { load_coef(a, p.a + w.n * p.cimg + w.c); load_coef(b, p.b + w.n * p.cimg + w.c); }
    if (Q && p.s) { load_coef(s, p.s + w.n * p.cimg + w.c); load_coef(t, p.t + w.n * p.cimg + w.c); }
  }
  const int blocks32 = (p.C + 31) >> 5, rows = p.g.rows;
  int px = w.p0 + w.r;
  const char* xp = p.x + (w.n * p.ximg + px * p.xps + w.c) * ES;
  char* yp = p.y + (w.n * p.yimg + px * p.yps + w.c) * ES;
  const long long row = (long long)w.n * p.pixels + px, xstep = rows * p.xps * ES, ystep = rows * p.yps * ES;
  signed char* cp = p.codes + row * p.C + w.c;
  bf16_t* sp = p.scales + row * blocks32 + (w.c >> 5);
  const int cstep = rows * p.C, sstep = rows * blocks32;
  for (; px < w.p1; px += U * rows) {
    Vec8<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (w.active && px + u * rows < w.p1) v[u] = load8<T, true>(xp + u * xstep);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (px + u * rows >= w.p1) break;
      float f[8], o[8];
      if (w.active) unpack8(f, v[u]);
      if (Y && w.active) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = act_fwd<ACT>(fmaf(f[j], a[j], b[j]));
        store8<T, true>(yp + u * ystep, pack8<T>(o));
      }
      if constexpr (Q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = !w.active ? 0.f : p.s ? fmaf(f[j], s[j], t[j]) : f[j];
        const Quant8 q = quantise8(o);
        if (w.active) {
          *reinterpret_cast<uint2*>(cp + u * cstep) = q.codes;
          if ((w.c & 31) == 0) sp[u * sstep] = q.scale;
        }
      }
    }
    xp += U * xstep;
    yp += U * ystep;
    cp += U * cstep;
    sp += U * sstep;
  }
}

// ------------------------------------------------------------------------------------------------ checkpoint, read back
// y = act(code * scale * a + b), or code * scale without a.
struct ReadArgs {
  const signed char* codes;
  const bf16_t* scales;
  char* y;
  const float *a, *b;
  long long yps, yimg, cimg;
  int pixels, C;
  NormGrid g;
};

template <typename T, int ACT, bool AFF>
__global__ __launch_bounds__(kNormThreads) void checkpoint_read_kernel(ReadArgs p) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  NormWalk w(p.g, blockIdx.x, p.pixels, p.C);
  if (!w.active) return;
  float a[8], b[8];
  if (AFF) { load_coef(a, p.a + w.n * p.cimg + w.c); load_coef(b, p.b + w.n * p.cimg + w.c); }
  const int blocks32 = (p.C + 31) >> 5, rows = p.g.rows;
  int px = w.p0 + w.r;
  const long long row = (long long)w.n * p.pixels + px, ystep = rows * p.yps * ES;
  const signed char* cp = p.codes + row * p.C + w.c;
  const bf16_t* sp = p.scales + row * blocks32 + (w.c >> 5);
  char* yp = p.y + (w.n * p.yimg + px * p.yps + w.c) * ES;
  const int cstep = rows * p.C, sstep = rows * blocks32;
  for (; px < w.p1; px += U * rows) {
    uint2 q[U];
    bf16_t s[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (px + u * rows < w.p1) {
        q[u] = load_codes<true>(cp + u * cstep);
        s[u] = sp[u * sstep];
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (px + u * rows >= w.p1) break;
      float f[8];
      dequantise8(f, q[u], bf16_to_f32(s[u]));
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = act_fwd<ACT>(AFF ? fmaf(f[j], a[j], b[j]) : f[j]);
      store8<T, true>(yp + u * ystep, pack8<T>(f));
    }
    cp += U * cstep;
    sp += U * sstep;
    yp += U * ystep;
  }
}

// ------------------------------------------------------------------------------------------------ backward
// g = dy act'(z), z = x a + b.  One fma gives the sign of z exactly, so the ReLU's mask is that of the forward pass.  With
// the checkpoint z = xhat gamma + beta, and code * scale is exact in 32 bits (7 + 8 significand bits).
struct BwdArgs {
  const char *x, *dy;
  char* dx;
  const signed char* codes;
  const bf16_t* scales;
  const float *mean, *rstd, *a, *b, *gamma, *beta; // mean, rstd [N][groups]; a, b [N][C]; gamma, beta [C] (checkpoint)
  const float *cm, *cp, *cq;                       // [N][C], second pass: dx = a g + (x - cm) cp + cq
  const double2* sums;                             // [N][C], all images: second pass, where the parameters' gradients are due
  float *dgamma, *dbeta;
  long long xps, ximg, dps, dimg, ops, oimg;
  int pixels, C, groups, images;
  NormGrid g;
};

template <typename T, bool CK> struct BwdLoad {
  Vec8<T> x, dy;
};
template <typename T> struct BwdLoad<T, true> {
  uint2 codes;
  bf16_t scale;
  Vec8<T> dy;
};

// Where a thread's next pixels lie.
template <typename T, bool CK> struct BwdFrom {
  const char *x, *dy;
  const signed char* codes;
  const bf16_t* scales;
  long long xstep, dstep;
  int cstep, sstep;
  __device__ __forceinline__ BwdFrom(const BwdArgs& p, const NormWalk& w) {
    constexpr int ES = Elem<T>::bytes;
    const int px = w.p0 + w.r, blocks32 = (p.C + 31) >> 5;
    if constexpr (CK) {
      const long long row = (long long)w.n * p.pixels + px;
      codes = p.codes + row * p.C + w.c;
      scales = p.scales + row * blocks32 + (w.c >> 5);
      cstep = p.g.rows * p.C;
      sstep = p.g.rows * blocks32;
    } else {
      x = p.x + (w.n * p.ximg + px * p.xps + w.c) * ES;
      xstep = p.g.rows * p.xps * ES;
    }
    dy = p.dy + (w.n * p.dimg + px * p.dps + w.c) * ES;
    dstep = p.g.rows * p.dps * ES;
  }
  // XNT, DNT: keep x (the codes), dy out of the caches
  template <bool XNT, bool DNT> __device__ __forceinline__ void load(BwdLoad<T, CK>& l, int u) const {
    if constexpr (CK) {
      l.codes = load_codes<XNT>(codes + u * cstep);
      l.scale = scales[u * sstep];
    } else {
      l.x = load8<T, XNT>(x + u * xstep);
    }
    l.dy = load8<T, DNT>(dy + u * dstep);
  }
  __device__ __forceinline__ void next(int u) {
    if constexpr (CK) {
      codes += u * cstep;
      scales += u * sstep;
    } else {
      x += u * xstep;
    }
    dy += u * dstep;
  }
};

// Coefficients of z for this thread's channels.
template <bool CK>
__device__ __forceinline__ void bwd_coef(float (&za)[8], float (&zb)[8], const BwdArgs& p, const NormWalk& w) {
  if constexpr (CK) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      za[j] = p.gamma ? p.gamma[w.c + j] : 1.f;
      zb[j] = p.beta ? p.beta[w.c + j] : 0.f;
    }
  } else {
    load_coef(za, p.a + (long long)w.n * p.C + w.c);
    load_coef(zb, p.b + (long long)w.n * p.C + w.c);
  }
}

// First pass: per block and channel sum g and sum g xhat.  XNT: x does not stay in the caches, as it and dy together are more
// than they hold.
template <typename T, int ACT, bool CK, bool XNT>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_reduce_kernel(BwdArgs p, float2* __restrict__ part) {
  constexpr int U = 4;
  __shared__ float l1[kNormThreads * 8], l2[kNormThreads * 8];
  __shared__ double2 lsum[kNormThreads];
  NormWalk w(p.g, blockIdx.x, p.pixels, p.C);
  float s1[8], s2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s1[j] = s2[j] = 0.f;
  if (w.active) {
    float za[8], zb[8], m[8], rs[8];
    bwd_coef<CK>(za, zb, p, w);
    if constexpr (!CK) {
      const int width = p.C / p.groups;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = w.n * p.groups + (w.c + j) / width;
        m[j] = p.mean[at];
        rs[j] = p.rstd[at];
      }
    }
    BwdFrom<T, CK> from(p, w);
    const int rows = p.g.rows;
    for (int px = w.p0 + w.r; px < w.p1; px += U * rows, from.next(U)) {
      BwdLoad<T, CK> l[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (px + u * rows < w.p1) from.template load<XNT, false>(l[u], u);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (px + u * rows < w.p1) {
          float f[8], d[8];
          unpack8(d, l[u].dy);
          if constexpr (CK) dequantise8(f, l[u].codes, bf16_to_f32(l[u].scale));
          else unpack8(f, l[u].x);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float gj = act_bwd<ACT>(fmaf(f[j], za[j], zb[j]), d[j]);
            s1[j] += gj;
            s2[j] = fmaf(gj, CK ? f[j] : f[j] - m[j], s2[j]);
          }
        }
    }
    if constexpr (!CK) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s2[j] *= rs[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    l1[threadIdx.x * 8 + j] = s1[j];
    l2[threadIdx.x * 8 + j] = s2[j];
  }
  __syncthreads();
  const int wide = p.g.cw * 8, parts = wide < kNormThreads ? kNormThreads / wide : 1;
  for (int i0 = 0; i0 < wide; i0 += kNormThreads) {
    const int i = i0 + (int)threadIdx.x % wide, q = (int)threadIdx.x / wide;
    double a = 0, b = 0;
    if (q < parts && i < wide)
      for (int r = q; r < p.g.rows; r += parts) {
        a += l1[r * wide + i];
        b += l2[r * wide + i];
      }
    if (parts > 1) {
      lsum[threadIdx.x] = make_double2(a, b);
      __syncthreads();
      if (q == 0)
        for (int t = 1; t < parts; ++t) {
          a += lsum[t * wide + i].x;
          b += lsum[t * wide + i].y;
        }
    }
    const int c = blockIdx.y * wide + i;
    if (q == 0 && i < wide && c < p.C)
      part[((long long)w.n * gridDim.x + blockIdx.x) * p.C + c] = make_float2((float)a, (float)b);
  }
}

// One block per (group, image): the channels' sums over the blocks, then over the group, in 64 bits.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_finalize_kernel(BwdArgs p, const float2* __restrict__ part, int blocks,
                                                                       int ckpt, double2* __restrict__ sums, float* __restrict__ cm,
                                                                       float* __restrict__ cp, float* __restrict__ cq) {
  __shared__ double r1[kNormThreads], r2[kNormThreads], lds[4];
  const int w = p.C / p.groups, g = blockIdx.x, n = blockIdx.y;
  const int wide = w < kNormThreads ? w : kNormThreads, lanes = kNormThreads / wide;
  const int ci = threadIdx.x % wide, li = threadIdx.x / wide;
  double k1 = 0, k2 = 0;
  for (int c0 = 0; c0 < w; c0 += wide) {
    const int c = g * w + c0 + ci;
    double a = 0, b = 0;
    if (li < lanes && c0 + ci < w)
#pragma unroll 8
      for (int k = li; k < blocks; k += lanes) {
        const float2 v = part[((long long)n * blocks + k) * p.C + c];
        a += v.x;
        b += v.y;
      }
    r1[threadIdx.x] = a;
    r2[threadIdx.x] = b;
    __syncthreads();
    for (int left = lanes; left > 1;) {
      const int half = (left + 1) >> 1;
      if (li + half < left) {
        r1[threadIdx.x] += r1[threadIdx.x + half * wide];
        r2[threadIdx.x] += r2[threadIdx.x + half * wide];
      }
      __syncthreads();
      left = half;
    }
    if (li == 0 && c0 + ci < w) {
      const double a1 = r1[threadIdx.x], a2 = r2[threadIdx.x], sc = p.a[(long long)n * p.C + c];
      sums[(long long)n * p.C + c] = make_double2(a1, a2);
      k1 += sc * a1;
      k2 += sc * a2;
    }
    __syncthreads();
  }
  const double count = (double)p.pixels * w;
  k1 = block_sum(k1, lds) / count;
  k2 = block_sum(k2, lds) / count;
  const float m = p.mean[n * p.groups + g], rs = p.rstd[n * p.groups + g];
  for (int i = threadIdx.x; i < w; i += kNormThreads) {
    const long long at = (long long)n * p.C + g * w + i;
    cm[at] = m;
    cp[at] = (float)(ckpt ? -k2 : -k2 * rs);
    cq[at] = (float)-k1;
  }
}

// The parameters' gradients: the images' sums.
__device__ __forceinline__ void gn_bwd_params(const double2* sums, int images, int C, int c, float* dgamma, float* dbeta) {
  double a = 0, b = 0;
#pragma unroll 8
  for (int n = 0; n < images; ++n) {
    const double2 v = sums[(long long)n * C + c];
    a += v.x;
    b += v.y;
  }
  if (dbeta) dbeta[c] = (float)a;
  if (dgamma) dgamma[c] = (float)b;
}

// Second pass: dx = a g + (x - cm) cp + cq.  With `sums`, the blocks past the last pixels add up the parameters' gradients.
template <typename T, int ACT, bool CK>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_apply_kernel(BwdArgs p) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  if ((int)blockIdx.x == p.g.blocks) {
    if (blockIdx.z == 0)
      for (int i = threadIdx.x; i < p.g.cw * 8; i += kNormThreads)
        if (const int c = blockIdx.y * p.g.cw * 8 + i; c < p.C) gn_bwd_params(p.sums, p.images, p.C, c, p.dgamma, p.dbeta);
    return;
  }
  NormWalk w(p.g, p.g.blocks - 1 - blockIdx.x, p.pixels, p.C);
  if (!w.active) return;
  float za[8], zb[8], a[8], m[8], kp[8], kq[8];
  const long long cat = (long long)w.n * p.C + w.c;
  bwd_coef<CK>(za, zb, p, w);
  load_coef(a, p.a + cat);
  load_coef(kp, p.cp + cat);
  load_coef(kq, p.cq + cat);
  if constexpr (!CK) load_coef(m, p.cm + cat);
  BwdFrom<T, CK> from(p, w);
  const int rows = p.g.rows;
  int px = w.p0 + w.r;
  char* op = p.dx + (w.n * p.oimg + px * p.ops + w.c) * ES;
  const long long ostep = rows * p.ops * ES;
  for (; px < w.p1; px += U * rows, from.next(U), op += U * ostep) {
    BwdLoad<T, CK> l[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (px + u * rows < w.p1) from.template load<true, true>(l[u], u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (px + u * rows >= w.p1) break;
      float f[8], d[8];
      unpack8(d, l[u].dy);
      if constexpr (CK) dequantise8(f, l[u].codes, bf16_to_f32(l[u].scale));
      else unpack8(f, l[u].x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float gj = act_bwd<ACT>(fmaf(f[j], za[j], zb[j]), d[j]);
        d[j] = fmaf(a[j], gj, fmaf(CK ? f[j] : f[j] - m[j], kp[j], kq[j]));
      }
      store8<T, true>(op + u * ostep, pack8<T>(d));
    }
  }
}

// ------------------------------------------------------------------------------------------------ launches
static int storage_of(int dtype, int fmt) { return dtype == MISEG_DT_F32 ? 2 : fmt == MISEG_FMT_F16 ? 1 : 0; }
static int act_of(int act) { return act == MISEG_ACT_RELU ? NA_RELU : act == MISEG_ACT_SILU ? NA_SILU : NA_NONE; }

// f(type tag, activation constant) for the storage type and activation of a call
template <int A> struct ActTag { static constexpr int act = A; };
template <typename T, typename F> static void by_act(int act, F f) {
  if (act == NA_RELU) f(T{}, ActTag<NA_RELU>{});
  else if (act == NA_SILU) f(T{}, ActTag<NA_SILU>{});
  else f(T{}, ActTag<NA_NONE>{});
}
template <typename F> static void by_type_act(int storage, int act, F f) {
  if (storage == 0) by_act<bf16s>(act, f);
  else if (storage == 1) by_act<f16s>(act, f);
  else by_act<f32s>(act, f);
}

#define NORM_CHECK_COMMON(name, d)                                                                                            \
  MISEG_CHECK_ARG((d)->dtype == MISEG_DT_BF16 || (d)->dtype == MISEG_DT_F32, name ": dtype %d", (d)->dtype);                  \
  MISEG_CHECK_ARG((d)->fmt == MISEG_FMT_BF16 || (d)->fmt == MISEG_FMT_F16, name ": fmt %d", (d)->fmt);                        \
  MISEG_CHECK_ARG((d)->act == MISEG_ACT_NONE || (d)->act == MISEG_ACT_RELU || (d)->act == MISEG_ACT_SILU, name ": act %d",    \
                  (d)->act);                                                                                                  \
  MISEG_CHECK_ARG((d)->N > 0 && (d)->N <= 65535 && (d)->pixels > 0 && (d)->C > 0 && ((d)->C & 7) == 0 && (d)->C <= 65536,     \
                  name ": N = %d (1..65535), pixels = %lld, C = %d (a multiple of 8, at most 65536)", (d)->N,                 \
                  (long long)(d)->pixels, (d)->C);                                                                            \
  MISEG_CHECK_ARG((d)->pixels < (1LL << 31) / 4, name ": %lld pixels in an image are too many", (long long)(d)->pixels)

static bool good_view(const void* p, int pix, long long img, long long N, long long pixels, int C, int bytes) {
  const int per = 16 / bytes;                      // elements in 16 bytes
  return p && ((uintptr_t)p & 15) == 0 && pix >= C && pix % per == 0 && img % per == 0 && img >= 0 &&
         (N == 1 || img >= (pixels - 1) * pix + C);
}
static bool good_coef(const void* p) { return ((uintptr_t)p & 15) == 0; }
static int bytes_of(int dtype) { return dtype == MISEG_DT_F32 ? 4 : 2; }

constexpr int kStatBlocks = 512, kStatLeast = 8;   // blocks of a reduction, sweeps in the smallest of them
constexpr int kPassBlocks = 32768, kPassLeast = 4; // the same for a pass that only streams
// Images are taken one launch after the other in steps whose tensors stay in the memory-side cache (256 MB) from the first
// pass to the second.
constexpr long long kCacheBytes = 200000000;

static int images_per_step(long long N, long long image_bytes) {
  const long long n = kCacheBytes / image_bytes;
  return (int)(n < 1 ? 1 : n < N ? n : N);
}

static long long round_up(long long v) { return (v + 255) / 256 * 256; }

// The blocks' partial sums, for steps of any number of images: norm_grid gives at most max(want, images x slabs) + images x
// slabs - 1 blocks over all slabs, and a block writes cw * 8 channels at most.
static long long gn_partials(long long N, long long pixels, int C) {
  const NormGrid g = norm_grid(1, pixels, C, kStatBlocks, 1);
  const long long slab = 8LL * g.cw * 8, most = (long long)((pixels + g.rows - 1) / g.rows) * N * g.ny;
  const long long blocks = kStatBlocks + 2 * N * g.ny;
  return round_up(slab * (blocks < most ? blocks : most));
}

static long long gn_workspace(long long N, long long pixels, int C, int backward) {
  const long long part = gn_partials(N, pixels, C), coef = round_up(4LL * N * C);
  return backward ? part + 2 * round_up(8LL * N * C) + 3 * coef : part + 2 * coef;
}

static void launch_pass(const PassArgs& p, int N, int storage, int act, hipStream_t s) {
  const dim3 grid(p.g.blocks, p.g.ny, N);
  by_type_act(storage, act, [&](auto t, auto a) {
    typedef decltype(t) T;
    constexpr int A = decltype(a)::act;
    if (p.y && p.codes) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, true>), grid, dim3(kNormThreads), 0, s, p);
    else if (p.y) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, false>), grid, dim3(kNormThreads), 0, s, p);
    else if constexpr (A == NA_NONE)
      hipLaunchKernelGGL((norm_pass_kernel<T, NA_NONE, false, true>), grid, dim3(kNormThreads), 0, s, p);
  });
}

int launch_group_norm_fwd(const miseg_group_norm_desc* d, hipStream_t s) {
  NORM_CHECK_COMMON("group_norm_act", d);
  const int bytes = bytes_of(d->dtype);
  MISEG_CHECK_ARG(d->groups > 0 && d->C % d->groups == 0, "group_norm_act: %d channels in %d groups", d->C, d->groups);
  MISEG_CHECK_ARG(good_view(d->x, d->x_pix, d->x_img, d->N, d->pixels, d->C, bytes) &&
                  good_view(d->y, d->y_pix, d->y_img, d->N, d->pixels, d->C, bytes),
                  "group_norm_act: x and y must be 16-byte aligned with strides of whole 16 bytes that hold C channels");
  MISEG_CHECK_ARG(!views_clash(d->x, d->x_pix, d->x_img, d->y, d->y_pix, d->y_img, d->N, d->pixels, d->C, bytes),
                  "group_norm_act: y overlaps x without being x or another channel range of its buffer");
  MISEG_CHECK_ARG(d->mean && d->rstd && d->scale && d->shift && good_coef(d->scale) && good_coef(d->shift),
                  "group_norm_act: mean, rstd, scale and shift are needed, scale and shift 16-byte aligned");
  MISEG_CHECK_ARG(d->eps >= 0.f, "group_norm_act: eps = %g", (double)d->eps);
  MISEG_CHECK_ARG(!d->codes == !d->code_scales && ((uintptr_t)d->codes & 7) == 0 && ((uintptr_t)d->code_scales & 1) == 0,
                  "group_norm_act: codes and code_scales go together, 8-byte and 2-byte aligned");
  const long long need = gn_workspace(d->N, d->pixels, d->C, 0);
  MISEG_CHECK_ARG(d->workspace && good_coef(d->workspace) && d->workspace_bytes >= need,
                  "group_norm_act: the workspace must be 16-byte aligned and hold %lld bytes (%lld given)", need,
                  (long long)d->workspace_bytes);
  const int storage = storage_of(d->dtype, d->fmt);
  char* ws = (char*)d->workspace;
  float2* part = (float2*)ws;
  ws += gn_partials(d->N, d->pixels, d->C);
  float *qs = nullptr, *qt = nullptr;
  if (d->codes) {
    qs = (float*)ws;
    qt = (float*)(ws + round_up(4LL * d->N * d->C));
  }
  const int step = images_per_step(d->N, d->pixels * d->C * bytes);
  for (int n0 = 0; n0 < d->N; n0 += step) {
    const int n = d->N - n0 < step ? d->N - n0 : step;
    const char* x = (const char*)d->x + n0 * d->x_img * bytes;
    const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
    const NormGrid g = norm_grid(n, d->pixels, d->C, kStatBlocks, kStatLeast);
    by_type_act(storage, NA_NONE, [&](auto t, auto) {
      hipLaunchKernelGGL((gn_stats_kernel<decltype(t)>), dim3(g.blocks, g.ny, n), dim3(kNormThreads), 0, s, x,
                         (long long)d->x_pix, d->x_img, (int)d->pixels, d->C, g, part);
    });
    hipLaunchKernelGGL(gn_finalize_kernel, dim3(d->groups, n), dim3(kNormThreads), 0, s, part, g.blocks, g.chunk, d->pixels,
                       d->C, d->groups, d->gamma, d->beta, d->eps, d->mean + gat, d->rstd + gat, d->scale + cat,
                       d->shift + cat, qs, qt);
    PassArgs p{x, (char*)d->y + n0 * d->y_img * bytes, (signed char*)d->codes, (bf16_t*)d->code_scales, d->scale + cat,
               d->shift + cat, qs, qt, d->x_pix, d->x_img, d->y_pix, d->y_img, d->C, (int)d->pixels, d->C,
               norm_grid(n, d->pixels, d->C, kPassBlocks, kPassLeast)};
    if (p.codes) {
      p.codes += n0 * d->pixels * d->C;
      p.scales += n0 * d->pixels * ((d->C + 31) / 32);
    }
    launch_pass(p, n, storage, act_of(d->act), s);
  }
  MISEG_CHECK_HIP(hipGetLastError());
  return MISEG_OK;
}

int launch_group_norm_bwd(const miseg_group_norm_bwd_desc* d, hipStream_t s) {
  NORM_CHECK_COMMON("group_norm_act_bwd", d);
  const int bytes = bytes_of(d->dtype);
  MISEG_CHECK_ARG(d->groups > 0 && d->C % d->groups == 0, "group_norm_act_bwd: %d channels in %d groups", d->C, d->groups);
  MISEG_CHECK_ARG(!d->codes == !d->code_scales && !d->codes != !d->x,
                  "group_norm_act_bwd: either x, or codes and code_scales");
  MISEG_CHECK_ARG(((uintptr_t)d->codes & 7) == 0 && ((uintptr_t)d->code_scales & 1) == 0,
                  "group_norm_act_bwd: codes and code_scales must be 8-byte and 2-byte aligned");
  MISEG_CHECK_ARG((d->codes || good_view(d->x, d->x_pix, d->x_img, d->N, d->pixels, d->C, bytes)) &&
                  good_view(d->dy, d->dy_pix, d->dy_img, d->N, d->pixels, d->C, bytes) &&
                  good_view(d->dx, d->dx_pix, d->dx_img, d->N, d->pixels, d->C, bytes),
                  "group_norm_act_bwd: x, dy and dx must be 16-byte aligned with strides of whole 16 bytes that hold C channels");
  MISEG_CHECK_ARG(!views_clash(d->x, d->x_pix, d->x_img, d->dx, d->dx_pix, d->dx_img, d->N, d->pixels, d->C, bytes) &&
                  !views_clash(d->dy, d->dy_pix, d->dy_img, d->dx, d->dx_pix, d->dx_img, d->N, d->pixels, d->C, bytes),
                  "group_norm_act_bwd: dx overlaps x or dy without being it or another channel range of its buffer");
  MISEG_CHECK_ARG(d->mean && d->rstd && d->scale && d->shift && good_coef(d->scale) && good_coef(d->shift),
                  "group_norm_act_bwd: mean, rstd, scale and shift are needed, scale and shift 16-byte aligned");
  const long long need = gn_workspace(d->N, d->pixels, d->C, 1);
  MISEG_CHECK_ARG(d->workspace && good_coef(d->workspace) && d->workspace_bytes >= need,
                  "group_norm_act_bwd: the workspace must be 16-byte aligned and hold %lld bytes (%lld given)", need,
                  (long long)d->workspace_bytes);
  const int storage = storage_of(d->dtype, d->fmt), act = act_of(d->act);
  const bool ck = d->codes != nullptr;
  char* ws = (char*)d->workspace;
  float2* part = (float2*)ws;
  ws += gn_partials(d->N, d->pixels, d->C);
  double2* sums = (double2*)ws;
  ws += 2 * round_up(8LL * d->N * d->C);
  const long long coef = round_up(4LL * d->N * d->C);
  float *cm = (float*)ws, *cp = (float*)(ws + coef), *cq = (float*)(ws + 2 * coef);
  const long long dbytes = d->pixels * d->C * bytes, xbytes = ck ? d->pixels * (d->C + 2 * ((d->C + 31) / 32)) : dbytes;
  // both stay in the cache if they can; else dy alone; else the last pixels of both
  const bool alone = xbytes + dbytes > kCacheBytes && dbytes <= kCacheBytes;
  const int step = images_per_step(d->N, alone ? dbytes : xbytes + dbytes);
  for (int n0 = 0; n0 < d->N; n0 += step) {
    const int n = d->N - n0 < step ? d->N - n0 : step;
    const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
    BwdArgs p{(const char*)d->x + n0 * d->x_img * bytes, (const char*)d->dy + n0 * d->dy_img * bytes,
              (char*)d->dx + n0 * d->dx_img * bytes, (const signed char*)d->codes, (const bf16_t*)d->code_scales,
              d->mean + gat, d->rstd + gat, d->scale + cat, d->shift + cat, d->gamma, d->beta, cm, cp, cq, nullptr,
              d->dgamma, d->dbeta, d->x_pix, d->x_img, d->dy_pix, d->dy_img, d->dx_pix, d->dx_img, (int)d->pixels, d->C,
              d->groups, d->N, norm_grid(n, d->pixels, d->C, kStatBlocks, kStatLeast)};
    if (ck) {
      p.codes += n0 * d->pixels * d->C;
      p.scales += n0 * d->pixels * ((d->C + 31) / 32);
    }
    const int blocks = p.g.blocks;
    by_type_act(storage, act, [&](auto t, auto a) {
      typedef decltype(t) T;
      constexpr int A = decltype(a)::act;
      const dim3 grid(blocks, p.g.ny, n);
      if (ck && alone) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, true, true>), grid, dim3(kNormThreads), 0, s, p, part);
      else if (ck) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, true, false>), grid, dim3(kNormThreads), 0, s, p, part);
      else if (alone) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, false, true>), grid, dim3(kNormThreads), 0, s, p, part);
      else hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, false, false>), grid, dim3(kNormThreads), 0, s, p, part);
    });
    hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3(d->groups, n), dim3(kNormThreads), 0, s, p, part, blocks, ck ? 1 : 0,
                       sums + cat, cm, cp, cq);
    p.g = norm_grid(n, d->pixels, d->C, kPassBlocks, kPassLeast);
    const bool params = n0 + n == d->N && (d->dgamma || d->dbeta);
    if (params) p.sums = sums;
    by_type_act(storage, act, [&](auto t, auto a) {
      typedef decltype(t) T;
      constexpr int A = decltype(a)::act;
      const dim3 grid(p.g.blocks + (params ? 1 : 0), p.g.ny, n);
      if (ck) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, true>), grid, dim3(kNormThreads), 0, s, p);
      else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, false>), grid, dim3(kNormThreads), 0, s, p);
    });
  }
  MISEG_CHECK_HIP(hipGetLastError());
  return MISEG_OK;
}

int launch_checkpoint8_write(const miseg_checkpoint8_desc* d, hipStream_t s) {
  NORM_CHECK_COMMON("checkpoint8_write", d);
  const int bytes = bytes_of(d->dtype);
  MISEG_CHECK_ARG(good_view(d->x, d->x_pix, d->x_img, d->N, d->pixels, d->C, bytes),
                  "checkpoint8_write: x must be 16-byte aligned with strides of whole 16 bytes that hold C channels");
  MISEG_CHECK_ARG(d->codes && d->code_scales && ((uintptr_t)d->codes & 7) == 0 && ((uintptr_t)d->code_scales & 1) == 0,
                  "checkpoint8_write: codes and code_scales are needed, 8-byte and 2-byte aligned");
  MISEG_CHECK_ARG(!d->code_a == !d->code_b && !d->y_a == !d->y_b, "checkpoint8_write: coefficients go in pairs");
  MISEG_CHECK_ARG(good_coef(d->code_a) && good_coef(d->code_b) && good_coef(d->y_a) && good_coef(d->y_b) &&
                  (d->coef_img & 3) == 0 && d->coef_img >= 0, "checkpoint8_write: coefficients must be 16-byte aligned");
  MISEG_CHECK_ARG(!d->y == !d->y_a, "checkpoint8_write: y takes its coefficients y_a and y_b");
  MISEG_CHECK_ARG(d->y || d->act == MISEG_ACT_NONE, "checkpoint8_write: an activation belongs to y");
  MISEG_CHECK_ARG(!d->y || (good_view(d->y, d->y_pix, d->y_img, d->N, d->pixels, d->C, bytes) &&
                            !views_clash(d->x, d->x_pix, d->x_img, d->y, d->y_pix, d->y_img, d->N, d->pixels, d->C, bytes)),
                  "checkpoint8_write: y must be a view like x, and be x, another channel range of its buffer or apart from it");
  PassArgs p{(const char*)d->x, (char*)d->y, (signed char*)d->codes, (bf16_t*)d->code_scales, d->y_a, d->y_b, d->code_a,
             d->code_b, d->x_pix, d->x_img, d->y_pix, d->y_img, d->coef_img, (int)d->pixels, d->C,
             norm_grid(d->N, d->pixels, d->C, kPassBlocks, kPassLeast)};
  launch_pass(p, d->N, storage_of(d->dtype, d->fmt), act_of(d->act), s);
  MISEG_CHECK_HIP(hipGetLastError());
  return MISEG_OK;
}

int launch_checkpoint8_read(const miseg_checkpoint8_desc* d, hipStream_t s) {
  NORM_CHECK_COMMON("checkpoint8_read", d);
  const int bytes = bytes_of(d->dtype);
  MISEG_CHECK_ARG(good_view(d->y, d->y_pix, d->y_img, d->N, d->pixels, d->C, bytes),
                  "checkpoint8_read: y must be 16-byte aligned with strides of whole 16 bytes that hold C channels");
  MISEG_CHECK_ARG(d->codes && d->code_scales && ((uintptr_t)d->codes & 7) == 0 && ((uintptr_t)d->code_scales & 1) == 0,
                  "checkpoint8_read: codes and code_scales are needed, 8-byte and 2-byte aligned");
  MISEG_CHECK_ARG(!d->y_a == !d->y_b && good_coef(d->y_a) && good_coef(d->y_b) && (d->coef_img & 3) == 0 && d->coef_img >= 0,
                  "checkpoint8_read: coefficients go in pairs, 16-byte aligned");
  ReadArgs p{(const signed char*)d->codes, (const bf16_t*)d->code_scales, (char*)d->y, d->y_a, d->y_b, d->y_pix,
             d->y_img, d->coef_img, (int)d->pixels, d->C, norm_grid(d->N, d->pixels, d->C, kPassBlocks, kPassLeast)};
  const dim3 grid(p.g.blocks, p.g.ny, d->N);
  by_type_act(storage_of(d->dtype, d->fmt), act_of(d->act), [&](auto t, auto a) {
    typedef decltype(t) T;
    constexpr int A = decltype(a)::act;
    if (p.a) hipLaunchKernelGGL((checkpoint_read_kernel<T, A, true>), grid, dim3(kNormThreads), 0, s, p);
    else hipLaunchKernelGGL((checkpoint_read_kernel<T, A, false>), grid, dim3(kNormThreads), 0, s, p);
  });
  MISEG_CHECK_HIP(hipGetLastError());
  return MISEG_OK;
}

long long group_norm_workspace(int N, long long pixels, int C, int backward) {
  if (N <= 0 || N > 65535 || pixels <= 0 || pixels >= (1LL << 31) / 4 || C <= 0 || (C & 7) || C > 65536) {
    set_error("group_norm_workspace: N = %d, pixels = %lld, C = %d", N, pixels, C);
    return MISEG_E_INVALID_ARG;
  }
  return gn_workspace(N, pixels, C, backward);
}

}  // namespace miseg

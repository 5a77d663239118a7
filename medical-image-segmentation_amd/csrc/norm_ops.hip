// Group normalisation with an activation on channels-last tensors, forward and backward, and activation checkpoints in
// 8 bits: their writing, their reading, and the backward pass out of them.
#include "norm_common.h"

namespace miseg {

// Sweeps whose pixels are all there go without a check per load.
struct WholeTag { constexpr operator bool() const { return true; } };
struct PartTag { constexpr operator bool() const { return false; } };

// ------------------------------------------------------------------------------------------------ sums over a block
// Threads in segments of `lanes`, a power of two up to 64 or a multiple of 64: the sums over a segment, in its first thread.
// Every thread of the block calls; `waves` holds one entry per wave.
struct Segments {
  int lanes, seg, t;
  __device__ __forceinline__ Segments(int threads, int segments) {
    const int most = threads / segments;
    lanes = most >= 64 ? most & ~63 : 1 << (31 - __clz(most));
    seg = threadIdx.x / lanes;
    t = threadIdx.x - seg * lanes;
  }
  __device__ __forceinline__ double2 sum(double2 v, double2* waves) const {
    for (int o = lanes < 64 ? lanes >> 1 : 32; o > 0; o >>= 1) {
      v.x += __shfl_xor(v.x, o, 64);
      v.y += __shfl_xor(v.y, o, 64);
    }
    if (lanes > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) waves[wave] = v;
      __syncthreads();
      if (t == 0)
        for (int i = 1; i < lanes >> 6; ++i) {
          v.x += waves[wave + i].x;
          v.y += waves[wave + i].y;
        }
    }
    return v;
  }
};

// f(j, table[group of channel first + j]) for the 8 channels of a thread, `first` a multiple of 8 counted from a group's start.
template <typename V, typename F>
__device__ __forceinline__ void each_group(const V* table, int first, int width, F f) {
  int g = first / width;
  if ((width & 7) == 0) {
    const V v = table[g];
#pragma unroll
    for (int j = 0; j < 8; ++j) f(j, v);
    return;
  }
  int left = width - (first - g * width);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f(j, table[g]);
    if (--left == 0) {
      left = width;
      ++g;
    }
  }
}

// Coefficients of z = x a + b for channels c.. of groups whose (mean, rstd) are in `stat`, where channel c is number `first`.
__device__ __forceinline__ void affine_coef(float (&a)[8], float (&b)[8], const double2* stat, int first, int width,
                                            const float* gamma, const float* beta, int c) {
  load_param(a, gamma, c, 1.f);
  load_param(b, beta, c, 0.f);
  each_group(stat, first, width, [&](int j, double2 q) {
    const double sc = a[j] * q.y;
    a[j] = (float)sc;
    b[j] = (float)(b[j] - q.x * sc);
  });
}
// Of xhat = x s + t.
__device__ __forceinline__ void unit_coef(float (&s)[8], float (&t)[8], const double2* stat, int first, int width) {
  each_group(stat, first, width, [&](int j, double2 q) {
    s[j] = (float)q.y;
    t[j] = (float)(-q.x * q.y);
  });
}

// Per column the sums over `blocks` of f(block, partial) as out[c], C columns of partials in rows of `pitch`; 256 threads.
// Loads are issued by fours: the partials were written by other chiplets, and a round trip takes about a microsecond.
template <typename V, typename F>
__device__ __forceinline__ void column_sums(double2* out, double2* tree, const V* part, int blocks, int C, int pitch,
                                            F f) {
  constexpr int U = 4;
  const int wide = C < kNormThreads ? C : kNormThreads, parts = kNormThreads / wide;
  const int i = threadIdx.x % wide, share = threadIdx.x / wide;
  for (int c0 = 0; c0 < C; c0 += wide) {
    const int c = c0 + i;
    double2 sum = make_double2(0, 0);
    if (share < parts && c < C)
      for (int k0 = share; k0 < blocks; k0 += U * parts) {
        V v[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k0 + u * parts < blocks) v[u] = part[(long long)(k0 + u * parts) * pitch + c];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k0 + u * parts < blocks) {
            const double2 t = f(k0 + u * parts, v[u]);
            sum.x += t.x;
            sum.y += t.y;
          }
      }
    tree[threadIdx.x] = sum;
    __syncthreads();
    for (int left = parts; left > 1;) {
      const int half = (left + 1) >> 1;
      if (share + half < left) {
        tree[threadIdx.x].x += tree[threadIdx.x + half * wide].x;
        tree[threadIdx.x].y += tree[threadIdx.x + half * wide].y;
      }
      __syncthreads();
      left = half;
    }
    if (share == 0 && c < C) out[c] = tree[threadIdx.x];
    __syncthreads();
  }
}
// group[g] = sum over its channels of chan, which holds `channels` from number `first` of group 0 on.
__device__ __forceinline__ void group_sums(double2* group, const double2* chan, double2* waves, int groups, int width,
                                           int first, int channels) {
  auto from = [&](int g) { return g == 0 ? 0 : g * width - first; };
  auto to = [&](int g) { return (g + 1) * width - first < channels ? (g + 1) * width - first : channels; };
  if (width <= 16) {
    for (int g = threadIdx.x; g < groups; g += kNormThreads) {
      double2 sum = make_double2(0, 0);
      for (int e = from(g); e < to(g); ++e) {
        sum.x += chan[e].x;
        sum.y += chan[e].y;
      }
      group[g] = sum;
    }
  } else {
    const Segments sg(kNormThreads, groups);
    double2 sum = make_double2(0, 0);
    if (sg.seg < groups)
      for (int e = from(sg.seg) + sg.t; e < to(sg.seg); e += sg.lanes) {
        sum.x += chan[e].x;
        sum.y += chan[e].y;
      }
    sum = sg.sum(sum, waves);
    if (sg.seg < groups && sg.t == 0) group[sg.seg] = sum;
  }
  __syncthreads();
}
constexpr int kSlabChannels = 512;                 // of norm_grid's widest slab

// A block's partial sums a group, [image][block][slab][pitch]: a slab, which may cut a group at either end, holds those of the
// groups from first() on, each over the channels of the group that lie in it.
struct GroupCuts {
  int slab, width, pitch, C;
  __device__ __forceinline__ GroupCuts(const NormGrid& g, int C, int width) : slab(g.cw * 8), width(width), C(C) {
    const int most = (slab + width - 2) / width + 1, groups = C / width;
    pitch = g.ny == 1 || most > groups ? groups : most;
  }
  __device__ __forceinline__ int first(int y) const { return y * slab / width; }
  __device__ __forceinline__ int end(int y) const { return (y + 1) * slab < C ? (y + 1) * slab : C; }
  __device__ __forceinline__ int groups(int y) const { return (end(y) - 1) / width - first(y) + 1; }
  __device__ __forceinline__ int channels(int g, int y) const {
    const int from = g * width > y * slab ? g * width : y * slab, to = (g + 1) * width < end(y) ? (g + 1) * width : end(y);
    return to - from;
  }
  // slabs that hold channels of group g
  __device__ __forceinline__ int from_slab(int g) const { return g * width / slab; }
  __device__ __forceinline__ int slabs(int g) const { return ((g + 1) * width - 1) / slab - from_slab(g) + 1; }
};

// ------------------------------------------------------------------------------------------------ forward statistics
// Per block and channel: mean and sum of squared differences from it.  A thread sums (x - k) and (x - k)^2 with k its own
// first value, so that an offset of the channel that is large against its spread does not cancel; threads and blocks are
// joined by counts, means and sums of squares, a partial a group of the slab, also where slabs cut groups (120 x 160 x 1536 in
// one group: the finalisation takes 6 us; with a partial a channel it takes 294).
// Bound by reading x: 157 MB in 30 us (5.3 TB/s).  512 blocks, two a CU, read as fast as 2048 and leave a quarter of the
// partials: the finalisation of 960 x 1280 x 64 takes 4.9 us, 17 with 2048.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void gn_stats_kernel(const char* x, long long xps, long long ximg, int pixels,
                                                                int C, int width, NormGrid g, float2* __restrict__ part) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  __shared__ double2 chan[kSlabChannels], group[kSlabChannels], waves[kNormThreads / 64];
  __shared__ float lmean[kNormThreads * 8], lm2[kNormThreads * 8];
  __shared__ int lcount[kNormThreads];
  __shared__ double2 lsum[kNormThreads];
  NormWalk w(g, blockIdx.x, pixels, C);
  float k[8], s1[8], s2[8];
  int count = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) k[j] = s1[j] = s2[j] = 0.f;
  const int px = w.p0 + w.r;
  if (w.active && px < w.p1) {
    const char* xp = x + (w.n * ximg + px * xps + w.c) * ES;
    const long long step = g.rows * xps * ES;
    unpack8(k, load8<T>(xp));
    auto sweep = [&](auto whole, int left) {
      Vec8<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (whole || u * g.rows < left) v[u] = load8<T>(xp + u * step);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!whole && u * g.rows >= left) break;
        float f[8];
        unpack8(f, v[u]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = f[j] - k[j];
          s1[j] += d;
          s2[j] = fmaf(d, d, s2[j]);
        }
      }
    };
    for (int at = w.p0; at < w.p1; at += U * g.rows, xp += U * step) {
      if (at + U * g.rows <= w.p1) sweep(WholeTag{}, 0);
      else sweep(PartTag{}, w.p1 - at - w.r);
    }
    count = (w.p1 - px + g.rows - 1) / g.rows;
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
    if (q == 0 && i < wide) chan[i] = make_double2(sum, sq);
  }
  __syncthreads();
  const GroupCuts cuts(g, C, width);
  const int y = blockIdx.y, g0 = cuts.first(y), groups = cuts.groups(y);
  const double2* from = chan;
  if (width > 1) {
    group_sums(group, chan, waves, groups, width, y * wide - g0 * width, cuts.end(y) - y * wide);
    from = group;
  }
  float2* out = part + (((long long)w.n * gridDim.x + blockIdx.x) * g.ny + y) * cuts.pitch;
  for (int e = threadIdx.x; e < groups; e += kNormThreads) {
    const double mean = from[e].x / ((double)(w.p1 - w.p0) * cuts.channels(g0 + e, y));
    out[e] = make_float2((float)mean, (float)(from[e].y - from[e].x * mean));
  }
}

// Sum over the threads of a block, in every thread.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int i = 1; i < kNormThreads / 64; ++i) v += lds[i];
  return v;
}

// One block per (group, image): the blocks' statistics of the group's channels in 64 bits, then the coefficients.
__global__ __launch_bounds__(kNormThreads) void gn_finalize_kernel(const float2* __restrict__ part, NormGrid grid,
                                                                   long long pixels, int C, int groups, NormParams param,
                                                                   float eps,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   float* __restrict__ scale, float* __restrict__ shift,
                                                                   float* __restrict__ qs, float* __restrict__ qt) {
  __shared__ double lds[kNormThreads / 64];
  const int w = C / groups, g = blockIdx.x, n = blockIdx.y;
  double s = 0, q = 0;
  const GroupCuts cuts(grid, C, w);
  const int y0 = cuts.from_slab(g), ys = cuts.slabs(g), blocks = grid.blocks, entries = blocks * ys;
  const int last = (int)(pixels - (long long)(blocks - 1) * grid.chunk);
  const float2* pp = part + (long long)n * blocks * grid.ny * cuts.pitch + g;
  constexpr int U = 4;                             // loads in flight: the kernel waits for nothing else
  for (int e0 = threadIdx.x; e0 < entries; e0 += U * kNormThreads) {
    float2 v[U];
    double count[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kNormThreads, b = e / ys, y = y0 + e - b * ys;
      count[u] = e >= entries ? 0. : (double)(b == blocks - 1 ? last : grid.chunk) * cuts.channels(g, y);
      v[u] = e < entries ? pp[((long long)b * grid.ny + y) * cuts.pitch - cuts.first(y)] : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const double m = v[u].x;
      s += count[u] * m;
      q += (double)v[u].y + count[u] * m * m;
    }
  }
  s = block_sum(s, lds);
  q = block_sum(q, lds);
  const double count = (double)pixels * w, m = s / count;
  double var = q / count - m * m;
  if (var < 0) var = 0;
  const double r = 1.0 / sqrt(var + (double)eps);
  if (threadIdx.x == 0) {
    mean[(long long)n * groups + g] = (float)m;
    rstd[(long long)n * groups + g] = (float)r;
  }
  for (int i = threadIdx.x; i < w; i += kNormThreads) {
    const int c = g * w + i;
    const float gm = param.gamma ? param.gamma[c] : 1.f, bt = param.beta ? param.beta[c] : 0.f;
    const double a = gm * r;
    scale[(long long)n * C + c] = (float)a;
    shift[(long long)n * C + c] = (float)(bt - m * a);
    if (n == 0 && param.gamma_kept) param.gamma_kept[c] = gm;
    if (n == 0 && param.beta_kept) param.beta_kept[c] = bt;
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
// Bound by memory: 157 MB in, out of the memory-side cache, and 157 MB out in 46 us (6.8 TB/s); with the checkpoint (4 x 240
// x 320 x 128) 199 MB in 31 us (6.4 TB/s), with SiLU as without.
struct PassArgs {
  const char* x;
  char* y;
  signed char* codes;
  bf16_t* scales;
  const float *a, *b, *s, *t;
  long long xps, ximg, yps, yimg, cimg;
  int pixels, C;
  NormGrid g;
  // FIN: group normalisation out of the partial statistics
  const float2* part = nullptr;
  int part_blocks = 0, part_chunk = 0, groups = 0;
  NormParams param = {};
  float *mean = nullptr, *rstd = nullptr, *scale = nullptr, *shift = nullptr;
  float eps = 0.f;
};

// The statistics of the groups of image n out of the blocks' (a partial a group) as (mean, rstd), and those of block 0 to
// memory.  Every block adds them up for itself, which saves a launch.
__device__ __forceinline__ void pass_statistics(const PassArgs& p, int n, double2* group) {
  __shared__ double2 tree[kNormThreads];
  const int last = p.pixels - (p.part_blocks - 1) * p.part_chunk, width = p.C / p.groups;
  column_sums(group, tree, p.part + (long long)n * p.part_blocks * p.groups, p.part_blocks, p.groups, p.groups,
              [&](int k, float2 v) {
                const double count = (double)(k == p.part_blocks - 1 ? last : p.part_chunk) * width, m = v.x;
                return make_double2(count * m, (double)v.y + count * m * m);
              });
  const double rcount = 1.0 / ((double)p.pixels * width);
  for (int g = threadIdx.x; g < p.groups; g += kNormThreads) {
    const double m = group[g].x * rcount;
    double var = group[g].y * rcount - m * m;
    if (var < 0) var = 0;
    const double rs = 1.0 / sqrt(var + (double)p.eps);
    group[g] = make_double2(m, rs);
    if (blockIdx.x == 0) {
      p.mean[n * p.groups + g] = (float)m;
      p.rstd[n * p.groups + g] = (float)rs;
    }
  }
  __syncthreads();
}

template <typename T, int ACT, bool Y, bool Q, bool FIN>
__global__ __launch_bounds__(kNormThreads) void norm_pass_kernel(PassArgs p) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  NormWalk w(p.g, gridDim.x - 1 - blockIdx.x, p.pixels, p.C);
  float a[8], b[8], s[8], t[8];
  if constexpr (FIN) {
    __shared__ double2 group[kSlabChannels];
    pass_statistics(p, w.n, group);
    if (w.active) {
      affine_coef(a, b, group, w.c, p.C / p.groups, p.param.gamma, p.param.beta, w.c);
      if (Q) unit_coef(s, t, group, w.c, p.C / p.groups);
      if (blockIdx.x == 0 && w.r == 0) {
        store_coef(p.scale + (long long)w.n * p.C + w.c, a);
        store_coef(p.shift + (long long)w.n * p.C + w.c, b);
        if (w.n == 0) p.param.keep(w.c);
      }
    }
  }
  if (w.r >= p.g.rows) return;                    // lanes past the last channel stay for the exchange in quantise8
  if (!FIN && w.active) {
    if (Y) { load_coef(a, p.a + w.n * p.cimg + w.c); load_coef(b, p.b + w.n * p.cimg + w.c); }
    if (Q && p.s) { load_coef(s, p.s + w.n * p.cimg + w.c); load_coef(t, p.t + w.n * p.cimg + w.c); }
  }
  if (!Q && !w.active) return;
  const int blocks32 = (p.C + 31) >> 5, rows = p.g.rows;
  const int px = w.p0 + w.r;
  const char* xp = p.x + (w.n * p.ximg + px * p.xps + w.c) * ES;
  char* yp = p.y + (w.n * p.yimg + px * p.yps + w.c) * ES;
  const long long row = (long long)w.n * p.pixels + px, xstep = rows * p.xps * ES, ystep = rows * p.yps * ES;
  signed char* cp = p.codes + row * p.C + w.c;
  bf16_t* sp = p.scales + row * blocks32 + (w.c >> 5);
  const int cstep = rows * p.C, sstep = rows * blocks32;
  const bool first = w.active && (w.c & 31) == 0;
  // left: pixels of this thread's column that are left; whole: all of a sweep's are there
  auto sweep = [&](auto whole, int left) {
    Vec8<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((!Q || w.active) && (whole || u * rows < left)) v[u] = load8<T, true>(xp + u * xstep);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!whole && u * rows >= left) break;
      float f[8], o[8];
      unpack8(f, v[u]);
      if constexpr (Y) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = act_fwd<ACT>(fmaf(f[j], a[j], b[j]));
        if (!Q || w.active) store8<T, true>(yp + u * ystep, pack8<T>(o));
      }
      if constexpr (Q) {
        if (FIN || p.s) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = fmaf(f[j], s[j], t[j]);
        }
        if (!w.active) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = 0.f;
        }
        const Quant8 q = quantise8(f);
        if (w.active) *reinterpret_cast<uint2*>(cp + u * cstep) = q.codes;
        if (first) sp[u * sstep] = q.scale;
      }
    }
  };
  for (int at = w.p0; at < w.p1; at += U * rows) {
    if (at + U * rows <= w.p1) sweep(WholeTag{}, 0);
    else sweep(PartTag{}, w.p1 - at - w.r);
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
  const int px = w.p0 + w.r;
  const long long row = (long long)w.n * p.pixels + px, ystep = rows * p.yps * ES;
  const signed char* cp = p.codes + row * p.C + w.c;
  const bf16_t* sp = p.scales + row * blocks32 + (w.c >> 5);
  char* yp = p.y + (w.n * p.yimg + px * p.yps + w.c) * ES;
  const int cstep = rows * p.C, sstep = rows * blocks32;
  auto sweep = [&](auto whole, int left) {
    uint2 q[U];
    bf16_t s[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (whole || u * rows < left) {
        q[u] = load_codes<true>(cp + u * cstep);
        s[u] = sp[u * sstep];
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!whole && u * rows >= left) break;
      float f[8];
      dequantise8(f, q[u], bf16_to_f32(s[u]));
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = act_fwd<ACT>(AFF ? fmaf(f[j], a[j], b[j]) : f[j]);
      store8<T, true>(yp + u * ystep, pack8<T>(f));
    }
  };
  for (int at = w.p0; at < w.p1; at += U * rows) {
    if (at + U * rows <= w.p1) sweep(WholeTag{}, 0);
    else sweep(PartTag{}, w.p1 - at - w.r);
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
  const float *cm, *cz, *cp, *cq;                  // [N][C], second pass: dx = a g + (x - cm) cp + cq (checkpoint: a g +
                                                   // xhat cp + cq, z = xhat cm + cz)
  const double2* sums;                             // [N][C], all images: second pass, where the parameters' gradients are due
  float *dgamma, *dbeta;
  long long xps, ximg, dps, dimg, ops, oimg;
  int pixels, C, groups, images;
  NormGrid g;
  const float2 *part, *gpart;                      // FIN: the blocks' sums a channel and a group, `part_blocks` an image
  int part_blocks;
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
    load_param(za, p.gamma, w.c, 1.f);
    load_param(zb, p.beta, w.c, 0.f);
  } else {
    load_coef(za, p.a + (long long)w.n * p.C + w.c);
    load_coef(zb, p.b + (long long)w.n * p.C + w.c);
  }
}

constexpr int kParamChannels = 16;                 // of a block that adds up partial sums by channels
// First pass: per block and channel sum g and sum g xhat; with `gpart` also per group, times the channels' a.
// XNT: x does not stay in the caches, as it and dy together are more than they hold.  Bound by reading: 157 MB (two images of
// 480 x 640 x 64, x and dy) in 30 us, 241 MB (codes and dy of 960 x 1280 x 64) in 41 us (5.9 TB/s).
template <typename T, int ACT, bool CK, bool XNT>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_reduce_kernel(BwdArgs p, float2* __restrict__ part,
                                                                     float2* __restrict__ gpart) {
  constexpr int U = 4;
  __shared__ double2 chan[kSlabChannels], group[kSlabChannels], waves[kNormThreads / 64];
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
      each_group(p.mean + (long long)w.n * p.groups, w.c, width, [&](int j, float v) { m[j] = v; });
      each_group(p.rstd + (long long)w.n * p.groups, w.c, width, [&](int j, float v) { rs[j] = v; });
    }
    BwdFrom<T, CK> from(p, w);
    const int rows = p.g.rows;
    auto sweep = [&](auto whole, int left) {
      BwdLoad<T, CK> l[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (whole || u * rows < left) from.template load<XNT, false>(l[u], u);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!whole && u * rows >= left) break;
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
    };
    for (int at = w.p0; at < w.p1; at += U * rows, from.next(U)) {
      if (at + U * rows <= w.p1) sweep(WholeTag{}, 0);
      else sweep(PartTag{}, w.p1 - at - w.r);
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
    if (q == 0 && i < wide && c < p.C) {
      part[((long long)w.n * gridDim.x + blockIdx.x) * p.C + c] = make_float2((float)a, (float)b);
      if (gpart) {
        const double sc = p.a[(long long)w.n * p.C + c];
        chan[i] = make_double2(sc * a, sc * b);
      }
    }
  }
  if (gpart) {
    const GroupCuts cuts(p.g, p.C, p.C / p.groups);
    const int y = blockIdx.y, g0 = cuts.first(y), groups = cuts.groups(y);
    __syncthreads();
    group_sums(group, chan, waves, groups, cuts.width, y * wide - g0 * cuts.width, cuts.end(y) - y * wide);
    float2* out = gpart + (((long long)w.n * gridDim.x + blockIdx.x) * p.g.ny + y) * cuts.pitch;
    for (int g = threadIdx.x; g < groups; g += kNormThreads) out[g] = make_float2((float)group[g].x, (float)group[g].y);
  }
}

// Coefficients of the second pass from the group's mean g a (k1) and mean g a xhat (k2).
__device__ __forceinline__ void bwd_share(const BwdArgs& p, int n, int c, double k1, double k2, float m, float rs, int ckpt,
                                          float* cm, float* cz, float* cp, float* cq) {
  const long long at = (long long)n * p.C + c;
  cm[at] = !ckpt ? m : p.gamma ? p.gamma[c] : 1.f;
  if (ckpt) cz[at] = p.beta ? p.beta[c] : 0.f;
  cp[at] = (float)(ckpt ? -k2 : -k2 * rs);
  cq[at] = (float)-k1;
}

// One block per (group, image): the channels' sums over the blocks, then over the group, in 64 bits.  Latency: 5 us, 7 from 8192
// partial sums a group on.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_finalize_kernel(BwdArgs p, const float2* __restrict__ part, int blocks,
                                                                      int ckpt, double2* __restrict__ sums,
                                                                      float* __restrict__ cm, float* __restrict__ cz,
                                                                      float* __restrict__ cp, float* __restrict__ cq) {
  __shared__ double r1[kNormThreads], r2[kNormThreads], lds[kNormThreads / 64];
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
  const float m = p.mean[(long long)n * p.groups + g], rs = p.rstd[(long long)n * p.groups + g];
  for (int i = threadIdx.x; i < w; i += kNormThreads) bwd_share(p, n, g * w + i, k1, k2, m, rs, ckpt, cm, cz, cp, cq);
}

// The same where a group has more than 16384 partial sums, from the groups' partials of the blocks, by 16 channels of an image:
// one group of 464 channels out of 127 blocks 9 us and 3 in the first pass, 21 in one block of 1024 threads; of 1536
// channels out of 83 blocks 8 us, 38.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_finalize_wide_kernel(BwdArgs p, const float2* __restrict__ part,
                                                                           int blocks, int ckpt, double2* __restrict__ sums,
                                                                           float* __restrict__ cm, float* __restrict__ cz,
                                                                           float* __restrict__ cp, float* __restrict__ cq) {
  __shared__ double2 chan[kParamChannels], tree[kNormThreads];
  __shared__ double lds[kNormThreads / 64];
  const int c0 = blockIdx.x * kParamChannels, n = blockIdx.y;
  const int channels = p.C - c0 < kParamChannels ? p.C - c0 : kParamChannels;
  const GroupCuts cuts(p.g, p.C, p.C / p.groups);
  column_sums(chan, tree, part + (long long)n * blocks * p.C + c0, blocks, channels, p.C,
              [](int, float2 v) { return make_double2(v.x, v.y); });
  if ((int)threadIdx.x < channels) sums[(long long)n * p.C + c0 + threadIdx.x] = chan[threadIdx.x];
  const double count = (double)p.pixels * cuts.width;
  const float2* gpart = p.gpart + (long long)n * blocks * p.g.ny * cuts.pitch;
  for (int g = c0 / cuts.width; g * cuts.width < c0 + channels; ++g) {
    const int y0 = cuts.from_slab(g), ys = cuts.slabs(g);
    const float m = p.mean[(long long)n * p.groups + g], rs = p.rstd[(long long)n * p.groups + g];
    double k1 = 0, k2 = 0;
    for (int e = threadIdx.x; e < blocks * ys; e += kNormThreads) {
      const int y = y0 + e % ys;
      const float2 v = gpart[((long long)(e / ys) * p.g.ny + y) * cuts.pitch + g - cuts.first(y)];
      k1 += v.x;
      k2 += v.y;
    }
    k1 = block_sum(k1, lds) / count;
    k2 = block_sum(k2, lds) / count;
    const int c = c0 + threadIdx.x;
    if ((int)threadIdx.x < channels && c / cuts.width == g) bwd_share(p, n, c, k1, k2, m, rs, ckpt, cm, cz, cp, cq);
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

template <bool CK>
__device__ __forceinline__ void group_bwd_coef(float (&za)[8], float (&zb)[8], float (&m)[8], float (&rs)[8], const BwdArgs& p,
                                               int n, int c, int width) {
  if constexpr (CK) {
    load_param(za, p.gamma, c, 1.f);
    load_param(zb, p.beta, c, 0.f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = 0.f;
      rs[j] = 1.f;
    }
  } else {
    load_coef(za, p.a + (long long)n * p.C + c);
    load_coef(zb, p.b + (long long)n * p.C + c);
    each_group(p.mean + (long long)n * p.groups, c, width, [&](int j, float v) { m[j] = v; });
    each_group(p.rstd + (long long)n * p.groups, c, width, [&](int j, float v) { rs[j] = v; });
  }
}
// kp and kq of the second pass from the groups' sums; kp holds rstd (1 for a checkpoint).
__device__ __forceinline__ void share_coef(float (&kp)[8], float (&kq)[8], const double2* group, int first, int width, int pixels) {
  const double rcount = 1.0 / ((double)pixels * width);
  each_group(group, first, width, [&](int j, double2 k) {
    kp[j] = (float)(-k.y * rcount * kp[j]);
    kq[j] = (float)(-k.x * rcount);
  });
}

template <typename T, int ACT, bool CK>
__device__ __forceinline__ void bwd_apply(const BwdArgs& p, const NormWalk& w, const float (&a)[8], const float (&za)[8],
                                          const float (&zb)[8], const float (&m)[8], const float (&kp)[8],
                                          const float (&kq)[8]) {
  constexpr int ES = Elem<T>::bytes, U = 4;
  BwdFrom<T, CK> from(p, w);
  const int rows = p.g.rows;
  const int px = w.p0 + w.r;
  char* op = p.dx + (w.n * p.oimg + px * p.ops + w.c) * ES;
  const long long ostep = rows * p.ops * ES;
  auto sweep = [&](auto whole, int left) {
    BwdLoad<T, CK> l[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (whole || u * rows < left) from.template load<true, true>(l[u], u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!whole && u * rows >= left) break;
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
  };
  for (int at = w.p0; at < w.p1; at += U * rows, from.next(U), op += U * ostep) {
    if (at + U * rows <= w.p1) sweep(WholeTag{}, 0);
    else sweep(PartTag{}, w.p1 - at - w.r);
  }
}

// Second pass: dx = a g + (x - cm) cp + cq.  With dgamma or dbeta due, the blocks past the last pixels add them up.
// FIN: every block adds up the groups' sums of its image for itself, which saves a launch.
// Bound by memory: 157 MB out of the memory-side cache and 79 MB out in 34 us (6.9 TB/s); 84 MB of codes from HBM, 157 MB of
// dy and 157 MB out in 59 us (6.8 TB/s; 75 with scalar loads of the parameters in every block).
template <typename T, int ACT, bool CK, bool FIN>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_apply_kernel(BwdArgs p) {
  if constexpr (FIN) {
    __shared__ double2 group[kSlabChannels], tree[kNormThreads];
    const auto plain = [](int, float2 v) { return make_double2(v.x, v.y); };
    if ((int)blockIdx.x >= p.g.blocks) {
      if (blockIdx.z != 0) return;
      const int c0 = ((int)blockIdx.x - p.g.blocks) * kParamChannels;
      const int channels = p.C - c0 < kParamChannels ? p.C - c0 : kParamChannels;
      column_sums(group, tree, p.part + c0, p.images * p.part_blocks, channels, p.C, plain);
      if ((int)threadIdx.x < channels) {
        if (p.dbeta) p.dbeta[c0 + threadIdx.x] = (float)group[threadIdx.x].x;
        if (p.dgamma) p.dgamma[c0 + threadIdx.x] = (float)group[threadIdx.x].y;
      }
      return;
    }
    const int n = blockIdx.z, width = p.C / p.groups;
    column_sums(group, tree, p.gpart + (long long)n * p.part_blocks * p.groups, p.part_blocks, p.groups, p.groups, plain);
    NormWalk w(p.g, p.g.blocks - 1 - blockIdx.x, p.pixels, p.C);
    if (!w.active) return;
    float za[8], zb[8], a[8], m[8], kp[8], kq[8];
    group_bwd_coef<CK>(za, zb, m, kp, p, n, w.c, width);
    if constexpr (CK) load_coef(a, p.a + (long long)n * p.C + w.c);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = za[j];
    share_coef(kp, kq, group, w.c, width, p.pixels);
    bwd_apply<T, ACT, CK>(p, w, a, za, zb, m, kp, kq);
  } else {
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
    load_coef(a, p.a + cat);
    if constexpr (CK) {
      load_coef(za, p.cm + cat);
      load_coef(zb, p.cz + cat);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) za[j] = a[j];
      load_coef(zb, p.b + cat);
      load_coef(m, p.cm + cat);
    }
    load_coef(kp, p.cp + cat);
    load_coef(kq, p.cq + cat);
    bwd_apply<T, ACT, CK>(p, w, a, za, zb, m, kp, kq);
  }
}

// ------------------------------------------------------------------------------------------------ small maps
// A block takes all pixels of some groups of one image and keeps them in registers between the statistics and the result:
// one launch, x read once.  A thread holds up to V pixels of its 8 channels.
struct SmallGrid {
  int threads;                                     // per block; 0: the map is too large
  int slab, slabs;                                 // channels of a block (whole groups, whole 8s), blocks per image
  int cw, rows;                                    // groups of 8 channels and pixels of a sweep
};
constexpr int kSmallThreads[2] = {256, 1024}, kSmallBack[2] = {256, 512};

// Neighbouring slabs share 128-byte lines: blocks 8 apart, which the hardware deals to one chiplet and its L2, take them.
__device__ __forceinline__ int small_block(int blocks) {
  const int per = blocks >> 3, b = blockIdx.x;
  return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}

struct SmallFwdArgs {
  const char* x;
  char* y;
  signed char* codes;
  bf16_t* scales;
  NormParams param;
  float *mean, *rstd, *a, *b;
  long long xps, ximg, yps, yimg;
  int pixels, C, groups, act, blocks;
  float eps;
  SmallGrid g;
};

template <typename T, int ACT, int V>
__device__ __forceinline__ void small_fwd_finish(char* yp, long long yps, const Vec8<T> (&v)[V], const float (&a)[8],
                                                 const float (&b)[8], int r, int rows, int pixels) {
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int px = r + u * rows;
    if (px >= pixels) break;
    float f[8];
    unpack8(f, v[u]);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = act_fwd<ACT>(fmaf(f[j], a[j], b[j]));
    store8<T>(yp + px * yps * Elem<T>::bytes, pack8<T>(f));
  }
}

template <typename T, bool Q, int TB, int V>
__global__ __launch_bounds__(TB) void gn_small_fwd_kernel(SmallFwdArgs p) {
  constexpr int ES = Elem<T>::bytes;
  __shared__ float2 part[TB * 8];
  __shared__ double2 stat[TB], waves[TB / 64];
  const int tid = threadIdx.x, id = small_block(p.blocks), n = id / p.g.slabs, c0 = (id - n * p.g.slabs) * p.g.slab;
  const int channels = p.C - c0 < p.g.slab ? p.C - c0 : p.g.slab, width = p.C / p.groups;
  const int rows = p.g.rows, cw = p.g.cw, r = tid / cw, l = tid - r * cw, c = c0 + l * 8;
  const bool active = r < rows && l * 8 < channels;
  Vec8<T> v[V];
  const char* xp = p.x + (n * p.ximg + c) * ES;
#pragma unroll
  for (int u = 0; u < V; ++u)
    if (active && r + u * rows < p.pixels) v[u] = load8<T>(xp + (r + u * rows) * p.xps * ES);
  // pixels of row r: every + (r < over)
  const int every = p.pixels / rows, over = p.pixels - every * rows;
  const int bits = width & 7 ? width & 3 ? width & 1 ? 0 : 1 : 2 : 3, merge = 1 << bits;   // channels of a thread in one group
  if (active) {
    float k[8], s1[8], s2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = s1[j] = s2[j] = 0.f;
    if (r < p.pixels) unpack8(k, v[0]);
#pragma unroll
    for (int u = 1; u < V; ++u) {
      if (r + u * rows >= p.pixels) break;
      float f[8];
      unpack8(f, v[u]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = f[j] - k[j];
        s1[j] += d;
        s2[j] = fmaf(d, d, s2[j]);
      }
    }
    // to means and sums of squares around them, then channels of a group joined by twos: equal counts
    const int count = every + (r < over ? 1 : 0);
    const float rc = count ? 1.f / (float)count : 0.f;
    float join = 0.5f * (float)count;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      k[j] += s1[j] * rc;
      s2[j] -= s1[j] * s1[j] * rc;
    }
#pragma unroll
    for (int size = 1; size < 8; size *= 2)
      if (merge > size) {
#pragma unroll
        for (int j = 0; j < 8; j += 2 * size) {
          const float d = k[j + size] - k[j];
          s2[j] += s2[j + size] + d * d * join;
          k[j] = 0.5f * (k[j] + k[j + size]);
        }
        join *= 2.f;
      }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((j & (merge - 1)) == 0) part[tid * (8 >> bits) + (j >> bits)] = make_float2(k[j], s2[j]);
  }
  __syncthreads();
  // the threads' statistics of a group: a row has `entry` of them, each of `merge` channels
  const int ng = channels / width, entry = width >> bits, pitch = cw * (8 >> bits);
  const Segments sg(TB, ng);
  double2 sum = make_double2(0, 0);
  if (sg.seg < ng) {
    int row = sg.t / entry, ch = sg.t - row * entry;
    const int drow = sg.lanes / entry, dch = sg.lanes - drow * entry, last = rows < p.pixels ? rows : p.pixels;
    while (row < last) {
      const float2 q = part[row * pitch + sg.seg * entry + ch];
      const double count = (every + (row < over ? 1 : 0)) * merge, m = q.x;
      sum.x += count * m;
      sum.y += (double)q.y + count * m * m;
      row += drow;
      ch += dch;
      if (ch >= entry) {
        ch -= entry;
        ++row;
      }
    }
  }
  sum = sg.sum(sum, waves);
  if (sg.seg < ng && sg.t == 0) {
    const double rcount = 1.0 / ((double)p.pixels * width), m = sum.x * rcount;
    double var = sum.y * rcount - m * m;
    if (var < 0) var = 0;
    const double rs = 1.0 / sqrt(var + (double)p.eps);
    const long long at = (long long)n * p.groups + c0 / width + sg.seg;
    p.mean[at] = (float)m;
    p.rstd[at] = (float)rs;
    stat[sg.seg] = make_double2(m, rs);
  }
  __syncthreads();
  if (active) {
    float a[8], b[8];
    affine_coef(a, b, stat, l * 8, width, p.param.gamma, p.param.beta, c);
    if (r == 0) {
      store_coef(p.a + (long long)n * p.C + c, a);
      store_coef(p.b + (long long)n * p.C + c, b);
      if (n == 0) p.param.keep(c);
    }
    char* yp = p.y + (n * p.yimg + c) * ES;
    if (p.act == NA_RELU) small_fwd_finish<T, NA_RELU, V>(yp, p.yps, v, a, b, r, rows, p.pixels);
    else if (p.act == NA_SILU) small_fwd_finish<T, NA_SILU, V>(yp, p.yps, v, a, b, r, rows, p.pixels);
    else small_fwd_finish<T, NA_NONE, V>(yp, p.yps, v, a, b, r, rows, p.pixels);
  }
  if constexpr (Q) {
    if (r >= rows) return;                        // whole quads of lanes: the others stay for the exchange in quantise8
    float qs[8], qt[8];
    unit_coef(qs, qt, stat, active ? l * 8 : 0, width);
    const int blocks32 = (p.C + 31) >> 5;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int px = r + u * rows;
      if (px >= p.pixels) break;
      float f[8];
      unpack8(f, v[u]);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = active ? fmaf(f[j], qs[j], qt[j]) : 0.f;
      const Quant8 q = quantise8(f);
      if (active) {
        const long long row = (long long)n * p.pixels + px;
        *reinterpret_cast<uint2*>(p.codes + row * p.C + c) = q.codes;
        if ((c & 31) == 0) p.scales[row * blocks32 + (c >> 5)] = q.scale;
      }
    }
  }
}

// Backward: x (or its codes) and dy stay in registers.  One image writes the parameters' gradients, several their sums.
struct SmallBwdArgs {
  BwdArgs p;
  double2* sums;
  int act, blocks;
  SmallGrid g;
};

template <typename T, int ACT, bool CK, int V>
__device__ __forceinline__ void small_bwd_sums(float (&s1)[8], float (&s2)[8], const BwdLoad<T, CK> (&v)[V],
                                               const float (&za)[8], const float (&zb)[8], const float (&m)[8], int r, int rows,
                                               int pixels) {
#pragma unroll
  for (int u = 0; u < V; ++u) {
    if (r + u * rows >= pixels) break;
    float f[8], d[8];
    unpack8(d, v[u].dy);
    if constexpr (CK) dequantise8(f, v[u].codes, bf16_to_f32(v[u].scale));
    else unpack8(f, v[u].x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gj = act_bwd<ACT>(fmaf(f[j], za[j], zb[j]), d[j]);
      s1[j] += gj;
      s2[j] = fmaf(gj, CK ? f[j] : f[j] - m[j], s2[j]);
    }
  }
}
template <typename T, int ACT, bool CK, int V>
__device__ __forceinline__ void small_bwd_finish(char* op, long long ops, const BwdLoad<T, CK> (&v)[V], const float (&a)[8],
                                                 const float (&za)[8], const float (&zb)[8], const float (&m)[8],
                                                 const float (&kp)[8], const float (&kq)[8], int r, int rows, int pixels) {
  constexpr int ES = Elem<T>::bytes;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int px = r + u * rows;
    if (px >= pixels) break;
    float f[8], d[8];
    unpack8(d, v[u].dy);
    if constexpr (CK) dequantise8(f, v[u].codes, bf16_to_f32(v[u].scale));
    else unpack8(f, v[u].x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gj = act_bwd<ACT>(fmaf(f[j], za[j], zb[j]), d[j]);
      d[j] = fmaf(a[j], gj, fmaf(CK ? f[j] : f[j] - m[j], kp[j], kq[j]));
    }
    store8<T>(op + px * ops * ES, pack8<T>(d));
  }
}

template <typename T, bool CK, int TB, int V>
__global__ __launch_bounds__(TB) void gn_small_bwd_kernel(SmallBwdArgs q) {
  constexpr int ES = Elem<T>::bytes;
  __shared__ float2 part[TB * 8];
  __shared__ double2 tree[TB], chan[TB], waves[TB / 64];
  const BwdArgs& p = q.p;
  const int tid = threadIdx.x, id = small_block(q.blocks), n = id / q.g.slabs, c0 = (id - n * q.g.slabs) * q.g.slab;
  const int channels = p.C - c0 < q.g.slab ? p.C - c0 : q.g.slab, width = p.C / p.groups;
  const int rows = q.g.rows, cw = q.g.cw, r = tid / cw, l = tid - r * cw, c = c0 + l * 8;
  const bool active = r < rows && l * 8 < channels;
  BwdLoad<T, CK> v[V];
  if (active) {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int px = r + u * rows;
      if (px >= p.pixels) break;
      if constexpr (CK) {
        const long long row = (long long)n * p.pixels + px;
        v[u].codes = load_codes<false>(p.codes + row * p.C + c);
        v[u].scale = p.scales[row * ((p.C + 31) >> 5) + (c >> 5)];
      } else {
        v[u].x = load8<T>(p.x + (n * p.ximg + px * p.xps + c) * ES);
      }
      v[u].dy = load8<T>(p.dy + (n * p.dimg + px * p.dps + c) * ES);
    }
  }
  if (active) {
    float za[8], zb[8], m[8], rs[8], s1[8], s2[8];
    group_bwd_coef<CK>(za, zb, m, rs, p, n, c, width);
#pragma unroll
    for (int j = 0; j < 8; ++j) s1[j] = s2[j] = 0.f;
    if (q.act == NA_RELU) small_bwd_sums<T, NA_RELU, CK, V>(s1, s2, v, za, zb, m, r, rows, p.pixels);
    else if (q.act == NA_SILU) small_bwd_sums<T, NA_SILU, CK, V>(s1, s2, v, za, zb, m, r, rows, p.pixels);
    else small_bwd_sums<T, NA_NONE, CK, V>(s1, s2, v, za, zb, m, r, rows, p.pixels);
#pragma unroll
    for (int j = 0; j < 8; ++j) part[j * TB + tid] = make_float2(s1[j], s2[j] * rs[j]);
  }
  __syncthreads();
  // per channel, by `parts` threads each; slot = j * cw + l
  const int used = rows < p.pixels ? rows : p.pixels, slots = cw * 8, parts = TB / slots;
  const int slot = tid % slots, share = tid / slots, sj = slot / cw, sl = slot - sj * cw, ch = sl * 8 + sj;
  double2 sum = make_double2(0, 0);
  if (share < parts && ch < channels)
    for (int row = share; row < used; row += parts) {
      const float2 e = part[sj * TB + row * cw + sl];
      sum.x += e.x;
      sum.y += e.y;
    }
  tree[tid] = sum;
  __syncthreads();
  for (int left = parts; left > 1;) {
    const int half = (left + 1) >> 1;
    if (share + half < left) {
      tree[tid].x += tree[tid + half * slots].x;
      tree[tid].y += tree[tid + half * slots].y;
    }
    __syncthreads();
    left = half;
  }
  if (tid < slots && ch < channels) {
    const long long at = (long long)n * p.C + c0 + ch;
    const double2 e = tree[tid];
    if (p.images == 1) {
      if (p.dbeta) p.dbeta[c0 + ch] = (float)e.x;
      if (p.dgamma) p.dgamma[c0 + ch] = (float)e.y;
    } else {
      q.sums[at] = e;
    }
    const double sc = p.a[at];
    chan[ch] = make_double2(sc * e.x, sc * e.y);
  }
  __syncthreads();
  // per group
  const int ng = channels / width;
  const Segments sg(TB, ng);
  sum = make_double2(0, 0);
  if (sg.seg < ng)
    for (int e = sg.t; e < width; e += sg.lanes) {
      sum.x += chan[sg.seg * width + e].x;
      sum.y += chan[sg.seg * width + e].y;
    }
  sum = sg.sum(sum, waves);
  if (sg.seg < ng && sg.t == 0) tree[sg.seg] = sum;
  __syncthreads();
  if (!active) return;
  float za[8], zb[8], m[8], a[8], kp[8], kq[8];   // read again rather than held over the exchange: registers are short
  group_bwd_coef<CK>(za, zb, m, kp, p, n, c, width);
  if constexpr (CK) load_coef(a, p.a + (long long)n * p.C + c);
  else
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = za[j];
  share_coef(kp, kq, tree, l * 8, width, p.pixels);
  char* op = p.dx + (n * p.oimg + c) * ES;
  if (q.act == NA_RELU) small_bwd_finish<T, NA_RELU, CK, V>(op, p.ops, v, a, za, zb, m, kp, kq, r, rows, p.pixels);
  else if (q.act == NA_SILU) small_bwd_finish<T, NA_SILU, CK, V>(op, p.ops, v, a, za, zb, m, kp, kq, r, rows, p.pixels);
  else small_bwd_finish<T, NA_NONE, CK, V>(op, p.ops, v, a, za, zb, m, kp, kq, r, rows, p.pixels);
}

// The parameters' gradients by 16 channels.  Latency: 2 to 4 us; 3000 images of 16 channels 24 us, 100 with a thread a channel.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_params_kernel(const double2* __restrict__ sums, int images, int C,
                                                                     float* dgamma, float* dbeta) {
  __shared__ double2 chan[kParamChannels], tree[kNormThreads];
  const int c0 = blockIdx.x * kParamChannels, channels = C - c0 < kParamChannels ? C - c0 : kParamChannels;
  column_sums(chan, tree, sums + c0, images, channels, C, [](int, double2 v) { return v; });
  if ((int)threadIdx.x >= channels) return;
  if (dbeta) dbeta[c0 + threadIdx.x] = (float)chan[threadIdx.x].x;
  if (dgamma) dgamma[c0 + threadIdx.x] = (float)chan[threadIdx.x].y;
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

constexpr int kStatBlocks = 512, kStatLeast = 8;   // blocks of a reduction, sweeps in the smallest of them (4, 16: the same)
constexpr int kPassBlocks = 32768, kPassLeast = 4; // the same for a pass that only streams
// Images are taken one launch after the other in steps whose tensors stay in the memory-side cache (256 MB) from the first
// pass to the second.
constexpr long long kCacheBytes = 200000000;

// Registers hold V vectors of 8 values a thread, in blocks of 256 threads or of 1024 (backward: 512, whose threads have twice
// the registers: x, dy and the coefficients of 1024 spilled).
template <typename T> struct SmallHold { static constexpr int fwd[2] = {8, 16}, bwd[2] = {4, 16}; };
template <> struct SmallHold<f32s> { static constexpr int fwd[2] = {4, 8}, bwd[2] = {2, 8}; };

static int gcd_int(int a, int b) { return b ? gcd_int(b, a % b) : a; }

// One launch pays where few pixels meet few channels: a load of a slab narrower than a line keeps a lane for every line, so
// a block's time grows with its pixels (fp32, 3 x 61 x 83 x 40 in slabs of 8: 17 us in one launch, 10 in two).  bf16, calls in a
// replayed graph, one launch | the better of two and three: forward 1..8 x 15 x 20 x 512 5.2 to 5.5 us | 9.2 to 10.5, 1..8 x 32 x
// 64 x 64 6.9 to 7.4 | 8.4 to 9.1, 1..8 x 32 x 64 x 512 8.9 to 13.3 | 11.9 to 16.8; backward with the launch that adds up the
// parameters, 2 x 30 x 40 x 512 11.9 | 12.5, 8 x 30 x 40 x 512 14.9 | 19.8, 1 x 30 x 40 x 64 8.5 | 9.2.  It loses on narrow maps
// of many pixels, backward with several images (2 x 30 x 40 x 64 10.8 | 9.4) and forward with a checkpoint (1 x 20 x 30 x 64 10.5 |
// 9.1, 1 x 32 x 64 x 64 16.1 | 9.3), where a launch less for the host stands against it.  Slabs are the widest of whole groups
// and whole 8s (32s where 32-channel blocks are written) that a block can hold, up to 64 channels, while 256 blocks are left.
constexpr int kSmallPixels = 2048;
static SmallGrid small_grid(long long N, long long pixels, int C, int groups, bool whole32, const int (&threads)[2],
                            const int (&hold)[2]) {
  SmallGrid g{};
  if (pixels > kSmallPixels) return g;
  const int width = C / groups, whole = whole32 ? 32 : 8;
  long long unit = (long long)width / gcd_int(width, whole) * whole;
  if (unit > C) unit = C;
  auto columns = [&](long long slab) { return whole32 ? (slab + 31) / 32 * 4 : slab / 8; };
  auto fits = [&](long long slab, int k) {
    if (columns(slab) * 8 > threads[k]) return false;
    const long long rows = threads[k] / columns(slab);
    return (pixels + rows - 1) / rows <= hold[k];
  };
  auto blocks = [&](long long slab) { return N * ((C + slab - 1) / slab); };
  if (!fits(unit, 0) && !fits(unit, 1)) return g;
  long long slab = unit;
  while (slab * 2 <= C && slab * 2 <= 64 && (fits(slab * 2, 0) || fits(slab * 2, 1)) && blocks(slab * 2) >= 256) slab *= 2;
  g.threads = threads[fits(slab, 0) ? 0 : 1];
  g.slab = (int)slab;
  g.slabs = (int)((C + slab - 1) / slab);
  g.cw = (int)columns(slab);
  g.rows = g.threads / g.cw;
  return g;
}

// Images that one launch of the small form takes: at most 2^32 threads in a direction of a grid.
static int small_images(const SmallGrid& g) {
  const long long n = ((1LL << 32) - 1) / g.threads / g.slabs;
  return (int)(n < 65535 ? n : 65535);
}

// Partial sums of a group that one block adds up (10 thousand: 7 us, as the chip); more are left to the whole chip.
constexpr int kWidePartials = 16384;

static int images_per_step(long long N, long long image_bytes) {
  const long long n = kCacheBytes / image_bytes;
  return (int)(n < 1 ? 1 : n < N ? n : N);
}

// Whether an image's partial sums are few enough for every block of the second pass to add them up itself: 4096 of them
// (32 KB), from blocks that read at most 128 KB of x each.  Two launches with a gap between them for three; in a replayed graph
// 3 x 61 x 83 x 72 forward 10 us (three launches: 11.5), out of 8 bits 10.5 (13.1).  Upwards of 2 x 60 x 80 x 256 (forward 14.1 us,
// 11.9) and 240 x 320 x 64 (17.1, 14.1; backward the same) three launches are shorter on the GPU and 3.6 us longer on the host.
// With 64 KB a block 120 x 160 x 256 would take three (14.1 us for 17.8), with 256 KB nothing here changes.  Passes of 512 blocks:
// 4 x 120 x 160 x 128 with a checkpoint 28.6 us (25.9); of 2048: its backward out of 8 bits 28.6 (26.1).
constexpr int kFewEntries = 4096, kFewBlocks = 512, kFewPass = 1024;
constexpr long long kFewBytes = 128 << 10;
static bool few_partials(long long N, long long pixels, int C, int groups, int bytes, NormGrid& g) {
  if (C > kSlabChannels) return false;
  const long long most = kFewEntries / groups, spread = (kFewBlocks + N - 1) / N;
  g = norm_grid(1, pixels, C, 1, 1);
  const long long deep = (pixels + 4 * g.rows - 1) / (4 * g.rows);     // blocks of the four sweeps that are in flight together
  const long long some = spread < most ? spread : most;
  g = norm_grid(1, pixels, C, (int)(deep < some ? deep : some), 1);
  return (long long)g.chunk * C * bytes <= kFewBytes;
}

static long long round_up(long long v) { return (v + 255) / 256 * 256; }

// The blocks' partial sums, for steps of any number of images: norm_grid gives at most max(want, images x slabs) blocks over
// all slabs, and a block writes cw * 8 channels at most.
static long long gn_partials(long long N, long long pixels, int C) {
  const NormGrid g = norm_grid(1, pixels, C, kStatBlocks, 1);
  const long long slab = 8LL * g.cw * 8, most = (long long)((pixels + g.rows - 1) / g.rows) * N * g.ny;
  const long long blocks = kStatBlocks + N * g.ny;
  return round_up(slab * (blocks < most ? blocks : most));
}

static SmallGrid small_fwd(long long N, long long pixels, int C, int groups, int dtype, bool checkpoint) {
  const int (&hold)[2] = dtype == MISEG_DT_F32 ? SmallHold<f32s>::fwd : SmallHold<bf16s>::fwd;
  return small_grid(N, pixels, C, groups, checkpoint, kSmallThreads, hold);
}
static SmallGrid small_bwd(long long N, long long pixels, int C, int groups, int dtype) {
  const int (&hold)[2] = dtype == MISEG_DT_F32 ? SmallHold<f32s>::bwd : SmallHold<bf16s>::bwd;
  return small_grid(N, pixels, C, groups, false, kSmallBack, hold);
}

static long long gn_workspace(long long N, long long pixels, int C, int groups, int dtype, int checkpoint, int backward) {
  const long long part = gn_partials(N, pixels, C), coef = round_up(4LL * N * C), sums = 2 * round_up(8LL * N * C);
  if (!backward) return small_fwd(N, pixels, C, groups, dtype, checkpoint).threads ? 0 : part + (checkpoint ? 2 * coef : 0);
  if (small_bwd(N, pixels, C, groups, dtype).threads) return N > 1 ? sums : 0;
  return sums + part + 4 * coef + part;            // the groups' partial sums are at most as many as the channels'

}

static void launch_pass(const PassArgs& p, int N, int storage, int act, hipStream_t s) {
  const dim3 grid(p.g.blocks, p.g.ny, N);
  by_type_act(storage, act, [&](auto t, auto a) {
    typedef decltype(t) T;
    constexpr int A = decltype(a)::act;
    if (p.part && p.codes) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, true, true>), grid, dim3(kNormThreads), 0, s, p);
    else if (p.part) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, false, true>), grid, dim3(kNormThreads), 0, s, p);
    else if (p.y && p.codes) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, true, false>), grid, dim3(kNormThreads), 0, s, p);
    else if (p.y) hipLaunchKernelGGL((norm_pass_kernel<T, A, true, false, false>), grid, dim3(kNormThreads), 0, s, p);
    else if constexpr (A == NA_NONE)
      hipLaunchKernelGGL((norm_pass_kernel<T, NA_NONE, false, true, false>), grid, dim3(kNormThreads), 0, s, p);
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
  MISEG_CHECK_ARG(good_coef(d->gamma_kept) && good_coef(d->beta_kept),
                  "group_norm_act: gamma_kept and beta_kept must be 16-byte aligned");
  MISEG_CHECK_ARG(d->eps >= 0.f, "group_norm_act: eps = %g", (double)d->eps);
  MISEG_CHECK_ARG(!d->codes == !d->code_scales && ((uintptr_t)d->codes & 7) == 0 && ((uintptr_t)d->code_scales & 1) == 0,
                  "group_norm_act: codes and code_scales go together, 8-byte and 2-byte aligned");
  const long long need = gn_workspace(d->N, d->pixels, d->C, d->groups, d->dtype, d->codes != nullptr, 0);
  MISEG_CHECK_ARG(!need || (d->workspace && good_coef(d->workspace) && d->workspace_bytes >= need),
                  "group_norm_act: the workspace must be 16-byte aligned and hold %lld bytes (%lld given)", need,
                  (long long)d->workspace_bytes);
  const int storage = storage_of(d->dtype, d->fmt);
  const NormParams param{d->gamma, d->beta, d->gamma_kept, d->beta_kept};
  const SmallGrid sg = small_fwd(d->N, d->pixels, d->C, d->groups, d->dtype, d->codes != nullptr);
  if (sg.threads) {
    const int most = small_images(sg);
    for (int n0 = 0; n0 < d->N; n0 += most) {
      const int n = d->N - n0 < most ? d->N - n0 : most;
      const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
      SmallFwdArgs p{(const char*)d->x + n0 * d->x_img * bytes, (char*)d->y + n0 * d->y_img * bytes, (signed char*)d->codes,
                     (bf16_t*)d->code_scales, n0 ? NormParams{d->gamma, d->beta, nullptr, nullptr} : param, d->mean + gat,
                     d->rstd + gat, d->scale + cat, d->shift + cat, d->x_pix, d->x_img, d->y_pix, d->y_img, (int)d->pixels,
                     d->C, d->groups, act_of(d->act), n * sg.slabs, d->eps, sg};
      if (p.codes) {
        p.codes += n0 * d->pixels * d->C;
        p.scales += n0 * d->pixels * ((d->C + 31) / 32);
      }
      const dim3 grid(p.blocks), block(sg.threads);
      by_type_act(storage, NA_NONE, [&](auto t, auto) {
        typedef decltype(t) T;
        typedef SmallHold<T> H;
        if (sg.threads == kSmallThreads[0]) {
          if (d->codes) hipLaunchKernelGGL((gn_small_fwd_kernel<T, true, kSmallThreads[0], H::fwd[0]>), grid, block, 0, s, p);
          else hipLaunchKernelGGL((gn_small_fwd_kernel<T, false, kSmallThreads[0], H::fwd[0]>), grid, block, 0, s, p);
        } else {
          if (d->codes) hipLaunchKernelGGL((gn_small_fwd_kernel<T, true, kSmallThreads[1], H::fwd[1]>), grid, block, 0, s, p);
          else hipLaunchKernelGGL((gn_small_fwd_kernel<T, false, kSmallThreads[1], H::fwd[1]>), grid, block, 0, s, p);
        }
      });
    }
    MISEG_CHECK_HIP(hipGetLastError());
    return MISEG_OK;
  }
  char* ws = (char*)d->workspace;
  float2* part = (float2*)ws;
  ws += gn_partials(d->N, d->pixels, d->C);
  float *qs = nullptr, *qt = nullptr;
  if (d->codes) {
    qs = (float*)ws;
    qt = (float*)(ws + round_up(4LL * d->N * d->C));
  }
  if (NormGrid g; few_partials(d->N, d->pixels, d->C, d->groups, bytes, g)) {
    by_type_act(storage, NA_NONE, [&](auto t, auto) {
      hipLaunchKernelGGL((gn_stats_kernel<decltype(t)>), dim3(g.blocks, g.ny, d->N), dim3(kNormThreads), 0, s,
                         (const char*)d->x, (long long)d->x_pix, d->x_img, (int)d->pixels, d->C, d->C / d->groups, g, part);
    });
    PassArgs p{(const char*)d->x, (char*)d->y, (signed char*)d->codes, (bf16_t*)d->code_scales, nullptr, nullptr, nullptr,
               nullptr, d->x_pix, d->x_img, d->y_pix, d->y_img, d->C, (int)d->pixels, d->C,
               norm_grid(d->N, d->pixels, d->C, kFewPass, kPassLeast, d->codes != nullptr), part, g.blocks, g.chunk,
               d->groups, param, d->mean, d->rstd, d->scale, d->shift, d->eps};
    launch_pass(p, d->N, storage, act_of(d->act), s);
    MISEG_CHECK_HIP(hipGetLastError());
    return MISEG_OK;
  }
  const int step = images_per_step(d->N, d->pixels * d->C * bytes);
  for (int n0 = 0; n0 < d->N; n0 += step) {
    const int n = d->N - n0 < step ? d->N - n0 : step;
    const char* x = (const char*)d->x + n0 * d->x_img * bytes;
    const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
    const NormGrid g = norm_grid(n, d->pixels, d->C, kStatBlocks, kStatLeast);
    by_type_act(storage, NA_NONE, [&](auto t, auto) {
      hipLaunchKernelGGL((gn_stats_kernel<decltype(t)>), dim3(g.blocks, g.ny, n), dim3(kNormThreads), 0, s, x,
                         (long long)d->x_pix, d->x_img, (int)d->pixels, d->C, d->C / d->groups, g, part);
    });
    hipLaunchKernelGGL(gn_finalize_kernel, dim3(d->groups, n), dim3(kNormThreads), 0, s, part, g, d->pixels, d->C,
                       d->groups, n0 ? NormParams{d->gamma, d->beta, nullptr, nullptr} : param, d->eps, d->mean + gat, d->rstd + gat, d->scale + cat, d->shift + cat,
                       qs, qt);
    PassArgs p{x, (char*)d->y + n0 * d->y_img * bytes, (signed char*)d->codes, (bf16_t*)d->code_scales, d->scale + cat,
               d->shift + cat, qs, qt, d->x_pix, d->x_img, d->y_pix, d->y_img, d->C, (int)d->pixels, d->C,
               norm_grid(n, d->pixels, d->C, kPassBlocks, kPassLeast, d->codes != nullptr)};
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
  const long long need = gn_workspace(d->N, d->pixels, d->C, d->groups, d->dtype, d->codes != nullptr, 1);
  MISEG_CHECK_ARG(!need || (d->workspace && good_coef(d->workspace) && d->workspace_bytes >= need),
                  "group_norm_act_bwd: the workspace must be 16-byte aligned and hold %lld bytes (%lld given)", need,
                  (long long)d->workspace_bytes);
  const int storage = storage_of(d->dtype, d->fmt), act = act_of(d->act);
  const bool ck = d->codes != nullptr;
  char* ws = (char*)d->workspace;
  double2* sums = (double2*)ws;
  const SmallGrid sg = small_bwd(d->N, d->pixels, d->C, d->groups, d->dtype);
  if (sg.threads) {
    const int most = small_images(sg);
    for (int n0 = 0; n0 < d->N; n0 += most) {
      const int n = d->N - n0 < most ? d->N - n0 : most;
      const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
      SmallBwdArgs q{{(const char*)d->x + n0 * d->x_img * bytes, (const char*)d->dy + n0 * d->dy_img * bytes,
                      (char*)d->dx + n0 * d->dx_img * bytes, (const signed char*)d->codes, (const bf16_t*)d->code_scales,
                      d->mean + gat, d->rstd + gat, d->scale + cat, d->shift + cat, d->gamma, d->beta, nullptr, nullptr,
                      nullptr, nullptr, nullptr, d->dgamma, d->dbeta, d->x_pix, d->x_img, d->dy_pix, d->dy_img, d->dx_pix,
                      d->dx_img, (int)d->pixels, d->C, d->groups, d->N, NormGrid{}, nullptr, nullptr, 0},
                     sums + cat, act, n * sg.slabs, sg};
      if (ck) {
        q.p.codes += n0 * d->pixels * d->C;
        q.p.scales += n0 * d->pixels * ((d->C + 31) / 32);
      }
      const dim3 grid(q.blocks), block(sg.threads);
      by_type_act(storage, NA_NONE, [&](auto t, auto) {
        typedef decltype(t) T;
        typedef SmallHold<T> H;
        if (sg.threads == kSmallBack[0]) {
          if (ck) hipLaunchKernelGGL((gn_small_bwd_kernel<T, true, kSmallBack[0], H::bwd[0]>), grid, block, 0, s, q);
          else hipLaunchKernelGGL((gn_small_bwd_kernel<T, false, kSmallBack[0], H::bwd[0]>), grid, block, 0, s, q);
        } else {
          if (ck) hipLaunchKernelGGL((gn_small_bwd_kernel<T, true, kSmallBack[1], H::bwd[1]>), grid, block, 0, s, q);
          else hipLaunchKernelGGL((gn_small_bwd_kernel<T, false, kSmallBack[1], H::bwd[1]>), grid, block, 0, s, q);
        }
      });
    }
    if (d->N > 1 && (d->dgamma || d->dbeta))
      hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((d->C + kParamChannels - 1) / kParamChannels), dim3(kNormThreads), 0, s, sums,
                         d->N, d->C, d->dgamma, d->dbeta);
    MISEG_CHECK_HIP(hipGetLastError());
    return MISEG_OK;
  }
  ws += 2 * round_up(8LL * d->N * d->C);
  float2* part = (float2*)ws;
  ws += gn_partials(d->N, d->pixels, d->C);
  const long long coef = round_up(4LL * d->N * d->C);
  float *cm = (float*)ws, *cz = (float*)(ws + coef), *cp = (float*)(ws + 2 * coef), *cq = (float*)(ws + 3 * coef);
  NormGrid few{};
  const bool fin = few_partials(d->N, d->pixels, d->C, d->groups, bytes, few);
  const long long dbytes = d->pixels * d->C * bytes, xbytes = ck ? d->pixels * (d->C + 2 * ((d->C + 31) / 32)) : dbytes;
  // both stay in the cache if they can; else dy alone; else the last pixels of both
  const bool alone = xbytes + dbytes > kCacheBytes && dbytes <= kCacheBytes;
  float2* gspace = (float2*)(ws + 4 * coef);
  const int step = fin ? d->N : images_per_step(d->N, alone ? dbytes : xbytes + dbytes);
  for (int n0 = 0; n0 < d->N; n0 += step) {
    const int n = d->N - n0 < step ? d->N - n0 : step;
    const long long cat = (long long)n0 * d->C, gat = (long long)n0 * d->groups;
    BwdArgs p{(const char*)d->x + n0 * d->x_img * bytes, (const char*)d->dy + n0 * d->dy_img * bytes,
              (char*)d->dx + n0 * d->dx_img * bytes, (const signed char*)d->codes, (const bf16_t*)d->code_scales,
              d->mean + gat, d->rstd + gat, d->scale + cat, d->shift + cat, d->gamma, d->beta, cm, cz, cp, cq, nullptr,
              d->dgamma, d->dbeta, d->x_pix, d->x_img, d->dy_pix, d->dy_img, d->dx_pix, d->dx_img, (int)d->pixels, d->C,
              d->groups, d->N, fin ? few : norm_grid(n, d->pixels, d->C, kStatBlocks, kStatLeast), part, gspace, few.blocks};
    if (ck) {
      p.codes += n0 * d->pixels * d->C;
      p.scales += n0 * d->pixels * ((d->C + 31) / 32);
    }
    const int blocks = p.g.blocks;
    const bool wide = !fin && (long long)blocks * (d->C / d->groups) > kWidePartials;
    float2* gpart = fin || wide ? gspace : nullptr;
    by_type_act(storage, act, [&](auto t, auto a) {
      typedef decltype(t) T;
      constexpr int A = decltype(a)::act;
      const dim3 grid(blocks, p.g.ny, n), block(kNormThreads);
      if (ck && alone) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, true, true>), grid, block, 0, s, p, part, gpart);
      else if (ck) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, true, false>), grid, block, 0, s, p, part, gpart);
      else if (alone) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, false, true>), grid, block, 0, s, p, part, gpart);
      else hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, A, false, false>), grid, block, 0, s, p, part, gpart);
    });
    if (wide)
      hipLaunchKernelGGL(gn_bwd_finalize_wide_kernel, dim3((d->C + kParamChannels - 1) / kParamChannels, n), dim3(kNormThreads),
                         0, s, p, part, blocks, ck ? 1 : 0, sums + cat, cm, cz, cp, cq);
    else if (!fin)
      hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3(d->groups, n), dim3(kNormThreads), 0, s, p, part, blocks, ck ? 1 : 0,
                         sums + cat, cm, cz, cp, cq);
    p.g = norm_grid(n, d->pixels, d->C, fin ? kFewPass : kPassBlocks, kPassLeast);
    const bool params = n0 + n == d->N && (d->dgamma || d->dbeta);
    if (params) p.sums = sums;
    by_type_act(storage, act, [&](auto t, auto a) {
      typedef decltype(t) T;
      constexpr int A = decltype(a)::act;
      const dim3 grid(p.g.blocks + (!params ? 0 : fin ? (d->C + kParamChannels - 1) / kParamChannels : 1), p.g.ny, n);
      if (ck && fin) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, true, true>), grid, dim3(kNormThreads), 0, s, p);
      else if (ck) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, true, false>), grid, dim3(kNormThreads), 0, s, p);
      else if (fin) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, false, true>), grid, dim3(kNormThreads), 0, s, p);
      else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A, false, false>), grid, dim3(kNormThreads), 0, s, p);
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
             norm_grid(d->N, d->pixels, d->C, kPassBlocks, kPassLeast, true)};
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

long long group_norm_workspace(int N, long long pixels, int C, int groups, int dtype, int checkpoint, int backward) {
  if (N <= 0 || N > 65535 || pixels <= 0 || pixels >= (1LL << 31) / 4 || C <= 0 || (C & 7) || C > 65536 || groups <= 0 ||
      C % groups || (dtype != MISEG_DT_BF16 && dtype != MISEG_DT_F32)) {
    set_error("group_norm_workspace: N = %d, pixels = %lld, C = %d, groups = %d, dtype = %d", N, pixels, C, groups, dtype);
    return MISEG_E_INVALID_ARG;
  }
  return gn_workspace(N, pixels, C, groups, dtype, checkpoint, backward);
}

}  // namespace miseg

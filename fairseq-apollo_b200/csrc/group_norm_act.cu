// Group norm over a sequence with an activation, channels last, forward and backward.
//
//   xhat = (x - mean) rstd, z = xhat scale + beta, y = z sigmoid(z)
//   dz = dy s (1 + z (1 - s)), s = sigmoid(z);  dn = dz scale
//   dx = rstd (dn - mean(dn) - xhat mean(dn xhat)),  dgamma = sum dz xhat,  dbeta = sum dz
//
// A block takes a tile of whole groups (channels side by side, a 16-byte vector of them to a thread) and a run of steps.
// First pass: statistics (backward: the two sums of every channel), over the block, written as one partial result per run.
// Second pass: every block folds the partial results of its groups, in their order, and does the elementwise part.  A sequence of
// one run needs no partial results: the same block does both, in one launch.
//
// Bound: HBM, each value once: the second pass goes backwards, over what the first has just left in L2, and a call that is larger
// than that goes through L2 in pieces of sequences and tiles.
//
// Statistics: a thread adds up d = x - p and d^2 with p the first value of its run.  p being one of the n values, the squares about
// it are at most n + 1 times those about the mean, so n <= kRun bounds what their difference loses; such entries are then joined by
// counts, means and squared deviations: the mean of all first, then the deviations about it.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "tma.cuh"

namespace mega {

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 64;        // steps of a thread at most
constexpr int kBatch = 4;       // rows that a thread loads at once
constexpr int kGroups = 256;    // groups of a tile at most (a vector or more each, or the 128 bytes of a narrow tile)

struct GnArgs {
  const void *x, *dy;
  void* out;
  long long xsb, xsl, gsb, gsl, osb, osl;
  const float *gamma, *beta;
  const unsigned char* mask;
  int B, L, D, G, size;        // size: channels of a group
  int ng, tiles;               // groups of a tile, tiles of a row
  int steps, runs;             // steps of a block, blocks of a sequence
  int first, slices;           // this launch: (sequence, tile) pairs first .. first + slices
  float eps, offset;
  int silu;
  long long* count;
  float *mean, *rstd;
  float *part, *chan;          // partial results of a run: of its groups (3 or 2 values), backward: of its channels (2)
  float *dgamma, *dbeta;
  int params;                  // blocks behind the others that add up dgamma, dbeta
};

// kV channels in a register or four
template <typename T, int kV>
struct Vec {
  static constexpr int kBytes = kV * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  unsigned w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
    }
  }
  __device__ __forceinline__ void get(float (&f)[kV]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kV; ++j) f[j] = __uint_as_float(w[j]);
    } else {
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int j = 0; j < kV; ++j) f[j] = Elem<T>::ld_shared(e + j);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[kV]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kV; ++j) w[j] = __float_as_uint(f[j]);
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int j = 0; j < kV; ++j) Elem<T>::st(e + j, f[j]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 4)
      *reinterpret_cast<unsigned*>(p) = w[0];
    else
      *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
  }
};

// sigmoid(z): fp32 with the full-range exponential and division, 16-bit types with the approximate ones (relative 2^-22 or so)
template <typename T>
__device__ __forceinline__ float sig(float z) {
  return sizeof(T) == 4 ? 1.f / (1.f + expf(-z)) : rcp_approx(1.f + __expf(-z));
}

// What a block works on.
template <int kV>
struct Where {
  int b, tile, run, c0, chans, groups, t0, t1;   // first channel, channels, groups; steps
  int nv, lanes, v, r;                           // vectors of a row, rows at once; this thread's vector and row
  bool on;
  __device__ __forceinline__ Where(const GnArgs& a, int slice, int run_) {
    b = slice / a.tiles, tile = slice % a.tiles, run = run_;
    c0 = tile * a.ng * a.size;
    groups = min(a.ng, a.G - tile * a.ng);
    chans = groups * a.size;
    t0 = run * a.steps, t1 = min(t0 + a.steps, a.L);
    nv = a.ng * a.size / kV;
    lanes = kThreads / nv;
    r = threadIdx.x / nv, v = threadIdx.x - r * nv;
    on = r < lanes && v * kV < chans;
  }
};

struct Sums {
  float a[2][kThreads * 8];   // [row of the block][channel of the tile]
  float n[kThreads];
  float g[3][kGroups];        // of a group: mean, rstd; backward the two sums
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// calls f(row, step, live) for the thread's rows of the block, live: not padded; loads go ahead, kN at a time
template <typename T, int kV, int kOps, int kN, typename Load, typename F>
__device__ __forceinline__ void rows(const GnArgs& a, const Where<kV>& p, bool back, Load&& load, F&& f) {
  const unsigned char* mask = a.mask ? a.mask + (long long)p.b * a.L : nullptr;
  const int total = p.t1 - p.t0, mine = p.on && p.r < total ? (total - p.r + p.lanes - 1) / p.lanes : 0;
  const int first = back ? p.t0 + p.r + (mine - 1) * p.lanes : p.t0 + p.r, step = back ? -p.lanes : p.lanes;
  int k = 0;
  if (mask == nullptr) {
    for (; k + kN <= mine; k += kN) {
      Vec<T, kV> v[kN][kOps];
#pragma unroll
      for (int u = 0; u < kN; ++u) load(v[u], first + (k + u) * step);
#pragma unroll
      for (int u = 0; u < kN; ++u) f(v[u], first + (k + u) * step, true);
    }
  }
  for (; k < mine; k += kN) {
    Vec<T, kV> v[kN][kOps];
    bool live[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      const int t = first + (k + u) * step;
      live[u] = k + u < mine && !(mask && mask[t]);
      if (live[u]) load(v[u], t);
    }
#pragma unroll
    for (int u = 0; u < kN; ++u)
      if (k + u < mine) f(v[u], first + (k + u) * step, live[u]);
  }
}

// ---- forward -----------------------------------------------------------------------------------
// Statistics of n values, means m[k] of counts c[k] and squared deviations q[k]: mean = sum c m / n, then sum q + c (m - mean)^2.
//
// Of the tile's groups over the block's steps -> s.g: steps, mean, squared deviations of all channels over their number.
// kOne: a vector lies in one group; its values are then one entry.
template <typename T, int kV, bool kOne>
__device__ __forceinline__ void moments(const GnArgs& a, const Where<kV>& p, Sums& s) {
  constexpr int kE = kOne ? 1 : kV;   // entries that a thread leaves
  const T* x = (const T*)a.x + p.b * a.xsb + p.c0 + p.v * kV;
  float cnt = 0.f, pv[kV], S[kV], Q[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) S[j] = Q[j] = pv[j] = 0.f;
  rows<T, kV, 1, kBatch>(a, p, false, [&](Vec<T, kV>(&v)[1], int t) { v[0].load(x + t * a.xsl); },
                         [&](Vec<T, kV>(&v)[1], int, bool live) {
                           if (!live) return;
                           float f[kV];
                           v[0].get(f);
                           if (cnt == 0.f) {
#pragma unroll
                             for (int j = 0; j < kV; ++j) pv[j] = f[j];
                           }
                           cnt += 1.f;
#pragma unroll
                           for (int j = 0; j < kV; ++j) {
                             const float d = f[j] - pv[j];
                             S[j] += d;
                             Q[j] = fmaf(d, d, Q[j]);
                           }
                         });
  const float inv = cnt > 0.f ? 1.f / cnt : 0.f;
  const int width = p.nv * kE;
  if (p.r < p.lanes) {
    float m[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const float d = S[j] * inv;
      m[j] = pv[j] + d;
      Q[j] = not_negative(fmaf(-S[j], d, Q[j]));
    }
    if (kOne) {
      float mean = 0.f, q = 0.f;
#pragma unroll
      for (int j = 0; j < kV; ++j) mean += m[j];
      mean *= 1.f / kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) q += fmaf(cnt * (m[j] - mean), m[j] - mean, Q[j]);
      m[0] = mean, Q[0] = q;
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      s.a[0][p.r * width + p.v * kE + j] = m[j];
      s.a[1][p.r * width + p.v * kE + j] = Q[j];
    }
    if (p.v == 0) s.n[p.r] = cnt;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, per = a.size * kE / kV;   // entries of a row and group
  float n = 0.f;
  for (int r = lane; r < p.lanes; r += 32) n += s.n[r];
  n = warp_sum(n);
  const float over = n > 0.f ? 1.f / (n * (float)per) : 0.f;
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    float sum = 0.f, dev = 0.f;
    for (int e = lane; e < p.lanes * per; e += 32) {
      const int r = e / per;
      sum = fmaf(s.n[r], s.a[0][r * width + g * per + e - r * per], sum);
    }
    const float mean = warp_sum(sum) * over;
    for (int e = lane; e < p.lanes * per; e += 32) {
      const int r = e / per, at = r * width + g * per + e - r * per;
      const float d = s.a[0][at] - mean, c = s.n[r] * (float)(kV / kE);
      if (c > 0.f) dev += fmaf(c * d, d, s.a[1][at]);   // (an empty row has no mean)
    }
    dev = warp_sum(dev);
    if (lane == 0) {
      s.g[0][g] = n;
      s.g[1][g] = mean;
      s.g[2][g] = dev / (float)a.size;
    }
  }
  __syncthreads();
}

// (steps, mean, squared deviations) -> (mean, rstd), written once
template <int kV>
__device__ __forceinline__ void finish(const GnArgs& a, const Where<kV>& p, Sums& s, bool write) {
  for (int g = threadIdx.x; g < p.groups; g += kThreads) {
    const float n = s.g[0][g], m = n > 0.f ? s.g[1][g] : 0.f, r = rsqrtf((n > 0.f ? s.g[2][g] / n : 0.f) + a.eps);
    s.g[0][g] = m;
    s.g[1][g] = r;
    if (write) {
      const long long at = (long long)p.b * a.G + p.tile * a.ng + g;
      a.mean[at] = m;
      a.rstd[at] = r;
      if (p.tile == 0 && g == 0) a.count[p.b] = (long long)n;
    }
  }
  __syncthreads();
}

// the group of a thread's j-th channel
template <int kV, bool kOne>
__device__ __forceinline__ int group_of(const GnArgs& a, const Where<kV>& p, int j) {
  return p.on ? (p.v * kV + (kOne ? 0 : j)) / a.size : 0;
}

template <typename T, int kV, bool kOne>
__device__ __forceinline__ void apply(const GnArgs& a, const Where<kV>& p, const Sums& s) {
  constexpr int kE = kOne ? 1 : kV;
  float m[kE], scale[kV], beta[kV];
#pragma unroll
  for (int j = 0; j < kE; ++j) m[j] = s.g[0][group_of<kV, kOne>(a, p, j)];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    scale[j] = p.on ? s.g[1][group_of<kV, kOne>(a, p, j)] * (a.gamma[p.c0 + p.v * kV + j] + a.offset) : 0.f;
    beta[j] = p.on ? a.beta[p.c0 + p.v * kV + j] : 0.f;
  }
  const T* x = (const T*)a.x + p.b * a.xsb + p.c0 + p.v * kV;
  T* y = (T*)a.out + p.b * a.osb + p.c0 + p.v * kV;
  rows<T, kV, 1, kBatch>(a, p, true, [&](Vec<T, kV>(&v)[1], int t) { v[0].load(x + t * a.xsl); },
                         [&](Vec<T, kV>(&v)[1], int t, bool live) {
                           float f[kV];
                           Vec<T, kV> o;
                           v[0].get(f);
#pragma unroll
                           for (int j = 0; j < kV; ++j) {
                             const float z = fmaf(f[j] - m[kOne ? 0 : j], scale[j], beta[j]);
                             f[j] = live ? (a.silu ? z * sig<T>(z) : z) : 0.f;
                           }
                           o.set(f);
                           o.store(y + t * a.osl);
                         });
}

// the partial results of the tile's groups, of every run (steps, mean, squared deviations)
__device__ __forceinline__ void fold(const GnArgs& a, int b, int tile, int groups, Sums& s) {
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < groups; g += kThreads / 32) {
    const float* q = a.part + (((long long)b * a.G + tile * a.ng + g) * a.runs) * 3;
    float n = 0.f, sum = 0.f, dev = 0.f;
    for (int r = lane; r < a.runs; r += 32) {
      n += q[3 * r];
      sum = fmaf(q[3 * r], q[3 * r + 1], sum);
    }
    n = warp_sum(n), sum = warp_sum(sum);
    const float mean = n > 0.f ? sum / n : 0.f;
    for (int r = lane; r < a.runs; r += 32) {
      const float d = q[3 * r + 1] - mean;
      if (q[3 * r] > 0.f) dev += fmaf(q[3 * r] * d, d, q[3 * r + 2]);
    }
    dev = warp_sum(dev);
    if (lane == 0) s.g[0][g] = n, s.g[1][g] = mean, s.g[2][g] = dev;
  }
  __syncthreads();
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_first_kernel(GnArgs a) {
  __shared__ Sums s;
  pdl_wait();
  const Where<kV> p(a, a.first + blockIdx.y, blockIdx.x);
  moments<T, kV, kOne>(a, p, s);
  if (a.runs == 1) {
    finish(a, p, s, true);
    apply<T, kV, kOne>(a, p, s);
  } else {
    for (int g = threadIdx.x; g < p.groups; g += kThreads) {
      float* q = a.part + (((long long)p.b * a.G + p.tile * a.ng + g) * a.runs + p.run) * 3;
      q[0] = s.g[0][g], q[1] = s.g[1][g], q[2] = s.g[2][g];
    }
  }
  pdl_next();
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_second_kernel(GnArgs a) {
  __shared__ Sums s;
  const int slice = a.slices - 1 - blockIdx.y, run = a.runs - 1 - blockIdx.x;
  const Where<kV> p(a, a.first + slice, run);
  pdl_wait();
  fold(a, p.b, p.tile, p.groups, s);
  finish(a, p, s, run == 0);
  apply<T, kV, kOne>(a, p, s);
  pdl_next();
}

// ---- backward --------------------------------------------------------------------------------
// dz of d = x - mean, with scale = rstd (gamma [+ 1])
template <typename T>
__device__ __forceinline__ float slope_of(float d, float dy, float scale, float beta, bool silu) {
  if (!silu) return dy;
  const float z = fmaf(d, scale, beta), g = sig<T>(z);
  return dy * (g * fmaf(z, 1.f - g, 1.f));
}

template <typename T, int kV, bool kOne>
struct Back {
  static constexpr int kE = kOne ? 1 : kV;
  const T *x, *dy;
  float m[kE], scale[kV], beta[kV];
  __device__ __forceinline__ Back(const GnArgs& a, const Where<kV>& p) {
    const long long at = (long long)p.b * a.G + p.tile * a.ng;
    x = (const T*)a.x + p.b * a.xsb + p.c0 + p.v * kV;
    dy = (const T*)a.dy + p.b * a.gsb + p.c0 + p.v * kV;
#pragma unroll
    for (int j = 0; j < kE; ++j) m[j] = a.mean[at + group_of<kV, kOne>(a, p, j)];
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      scale[j] = p.on ? a.rstd[at + group_of<kV, kOne>(a, p, j)] * (a.gamma[p.c0 + p.v * kV + j] + a.offset) : 0.f;
      beta[j] = p.on ? a.beta[p.c0 + p.v * kV + j] : 0.f;
    }
  }
  __device__ __forceinline__ void load(const GnArgs& a, Vec<T, kV> (&v)[2], int t) const {
    v[0].load(x + t * a.xsl);
    v[1].load(dy + t * a.gsl);
  }
};

// sums of dz and dz xhat of every channel over the block's steps -> a.chan, of dn and dn xhat of every group -> s.g[0], s.g[1]
template <typename T, int kV, bool kOne>
__device__ __forceinline__ void sums(const GnArgs& a, const Where<kV>& p, Sums& s) {
  float S[kV], Q[kV];   // (Q: of dz d, xhat being rstd d)
#pragma unroll
  for (int j = 0; j < kV; ++j) S[j] = Q[j] = 0.f;
  {
    const Back<T, kV, kOne> k(a, p);
    rows<T, kV, 2, kBatch / 2>(a, p, false, [&](Vec<T, kV>(&v)[2], int t) { k.load(a, v, t); },
                               [&](Vec<T, kV>(&v)[2], int, bool live) {
                                 if (!live) return;
                                 float f[kV], g[kV];
                                 v[0].get(f);
                                 v[1].get(g);
#pragma unroll
                                 for (int j = 0; j < kV; ++j) {
                                   const float d = f[j] - k.m[kOne ? 0 : j], dz = slope_of<T>(d, g[j], k.scale[j], k.beta[j], a.silu);
                                   S[j] += dz;
                                   Q[j] = fmaf(dz, d, Q[j]);
                                 }
                               });
  }
  const int width = p.nv * kV;
  if (p.r < p.lanes) {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      s.a[0][p.r * width + p.v * kV + j] = S[j];
      s.a[1][p.r * width + p.v * kV + j] = Q[j];
    }
  }
  __syncthreads();
  // rows of the block: some threads to a channel, each every parts-th row, into that part's row
  const int parts = min(max(1, kThreads / width), p.lanes);
  for (int e = threadIdx.x; e < parts * width; e += kThreads) {
    const int part = e / width, c = e - part * width;
    float u = 0.f, q = 0.f;
    for (int r = part; r < p.lanes; r += parts) u += s.a[0][r * width + c], q += s.a[1][r * width + c];
    s.a[0][e] = u;
    s.a[1][e] = q;
  }
  __syncthreads();
  const long long row = ((long long)p.b * a.runs + p.run) * 2 * a.D, at = (long long)p.b * a.G + p.tile * a.ng;
  for (int c = threadIdx.x; c < p.chans; c += kThreads) {
    float u = 0.f, q = 0.f;
    for (int k = 0; k < parts; ++k) u += s.a[0][k * width + c], q += s.a[1][k * width + c];
    q *= a.rstd[at + c / a.size];
    a.chan[row + p.c0 + c] = u;
    a.chan[row + a.D + p.c0 + c] = q;
    const float w = a.gamma[p.c0 + c] + a.offset;
    s.a[0][c] = u * w;   // (this thread alone has read the place)
    s.a[1][c] = q * w;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    float u = 0.f, q = 0.f;
    for (int c = lane; c < a.size; c += 32) u += s.a[0][g * a.size + c], q += s.a[1][g * a.size + c];
    u = warp_sum(u), q = warp_sum(q);
    if (lane == 0) s.g[0][g] = u, s.g[1][g] = q;
  }
  __syncthreads();
}

// sums of dn, dn xhat in s.g[0], s.g[1] -> dx = rstd dn - rstd mean(dn) - d rstd^2 mean(dn xhat)
template <typename T, int kV, bool kOne>
__device__ __forceinline__ void grads(const GnArgs& a, const Where<kV>& p, const Sums& s) {
  constexpr int kE = kOne ? 1 : kV;
  const Back<T, kV, kOne> k(a, p);
  const float n = (float)a.count[p.b] * (float)a.size, inv = n > 0.f ? 1.f / n : 0.f;
  float m1[kE], m2[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    const int g = group_of<kV, kOne>(a, p, j);
    const float r = a.rstd[(long long)p.b * a.G + p.tile * a.ng + g];
    m1[j] = s.g[0][g] * inv * r;
    m2[j] = s.g[1][g] * inv * r * r;
  }
  T* dx = (T*)a.out + p.b * a.osb + p.c0 + p.v * kV;
  rows<T, kV, 2, kBatch / 2>(a, p, true, [&](Vec<T, kV>(&v)[2], int t) { k.load(a, v, t); },
                             [&](Vec<T, kV>(&v)[2], int t, bool live) {
                               float f[kV], g[kV];
                               Vec<T, kV> o;
                               v[0].get(f);
                               v[1].get(g);
#pragma unroll
                               for (int j = 0; j < kV; ++j) {
                                 const float d = f[j] - k.m[kOne ? 0 : j], dz = slope_of<T>(d, g[j], k.scale[j], k.beta[j], a.silu);
                                 f[j] = live ? fmaf(dz, k.scale[j], -m1[kOne ? 0 : j]) - d * m2[kOne ? 0 : j] : 0.f;
                               }
                               o.set(f);
                               o.store(dx + t * a.osl);
                             });
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_sums_kernel(GnArgs a) {
  __shared__ Sums s;
  pdl_wait();
  const Where<kV> p(a, a.first + blockIdx.y, blockIdx.x);
  sums<T, kV, kOne>(a, p, s);
  if (a.runs == 1) {
    grads<T, kV, kOne>(a, p, s);
  } else {
    const long long at = (long long)p.b * a.G + p.tile * a.ng;
    for (int g = threadIdx.x; g < p.groups; g += kThreads) {
      float* q = a.part + ((at + g) * a.runs + p.run) * 2;
      q[0] = s.g[0][g], q[1] = s.g[1][g];
    }
  }
  pdl_next();
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_grads_kernel(GnArgs a) {
  __shared__ Sums s;
  const int slice = a.slices - 1 - blockIdx.y, run = a.runs - 1 - blockIdx.x, lane = threadIdx.x & 31;
  const Where<kV> p(a, a.first + slice, run);
  pdl_wait();
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    const float* q = a.part + (((long long)p.b * a.G + p.tile * a.ng + g) * a.runs) * 2;
    float u = 0.f, w = 0.f;
    for (int r = lane; r < a.runs; r += 32) u += q[2 * r], w += q[2 * r + 1];
    u = warp_sum(u), w = warp_sum(w);
    if (lane == 0) s.g[0][g] = u, s.g[1][g] = w;
  }
  __syncthreads();
  grads<T, kV, kOne>(a, p, s);
  pdl_next();
}

// dgamma, dbeta of 32 channels: the partial results of all sequences and runs, 32 rows at a time
__global__ void __launch_bounds__(1024) gn_params_kernel(GnArgs a) {
  __shared__ float part[2][32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  const long long n = (long long)a.B * a.runs;
  pdl_wait();
  float u = 0.f, q = 0.f;
  if (d < a.D) {
#pragma unroll 4
    for (long long r = w; r < n; r += 32) {
      u += a.chan[r * 2 * a.D + d];
      q += a.chan[r * 2 * a.D + a.D + d];
    }
  }
  part[0][w][lane] = u;
  part[1][w][lane] = q;
  __syncthreads();
  u = warp_sum(part[0][lane][w]), q = warp_sum(part[1][lane][w]);
  if (lane == 0 && blockIdx.x * 32 + w < a.D) {
    a.dbeta[blockIdx.x * 32 + w] = u;
    a.dgamma[blockIdx.x * 32 + w] = q;
  }
  pdl_next();
}

// ---- groups of more channels than a block's threads span -------------------------------------------
// One block per sequence and group takes the sums, an elementwise pass follows: each value is read three times.  Taken by
// groups of more than 2048 channels in 16-bit types (1024 in fp32), fewer where vectors are shorter.
__device__ float block_sum(float v) {   // the sum in every thread
  __shared__ float part[8];
  __syncthreads();
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < 8; ++w) v += part[w];
  return v;
}

// calls f(step, channel of the group) for what is not padded of this block's group
template <typename F>
__device__ __forceinline__ void wide_each(const GnArgs& a, F&& f) {
  const unsigned char* mask = a.mask ? a.mask + (long long)blockIdx.y * a.L : nullptr;
  for (int t = 0; t < a.L; ++t) {
    if (mask && mask[t]) continue;
    for (int c = threadIdx.x; c < a.size; c += kThreads) f(t, blockIdx.x * a.size + c);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_wide_stats_kernel(GnArgs a) {
  const int g = blockIdx.x, b = blockIdx.y;
  const T* x = (const T*)a.x + b * a.xsb;
  int live = 0;
  float s = 0.f, q = 0.f;
  for (int t = threadIdx.x; t < a.L; t += kThreads) live += !(a.mask && a.mask[(long long)b * a.L + t]);
  const float n = block_sum((float)live), inv = n > 0.f ? 1.f / (n * (float)a.size) : 0.f;
  // (runs of steps are joined, so that a long sequence's sums do not grow past their addends)
  float part = 0.f;
  int in = 0;
  wide_each(a, [&](int t, int c) {
    part += Elem<T>::ld(x + t * a.xsl + c);
    if (++in == kRun) s += part, part = 0.f, in = 0;
  });
  const float m = block_sum(s + part) * inv;
  part = 0.f, in = 0;
  wide_each(a, [&](int t, int c) {
    const float d = Elem<T>::ld(x + t * a.xsl + c) - m;
    part = fmaf(d, d, part);
    if (++in == kRun) q += part, part = 0.f, in = 0;
  });
  q = block_sum(q + part) * inv;
  if (threadIdx.x == 0) {
    a.mean[(long long)b * a.G + g] = m;
    a.rstd[(long long)b * a.G + g] = rsqrtf(q + a.eps);
    if (g == 0) a.count[b] = (long long)n;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_wide_apply_kernel(GnArgs a) {
  const int t = blockIdx.x, b = blockIdx.y;
  const T* x = (const T*)a.x + b * a.xsb + t * a.xsl;
  T* y = (T*)a.out + b * a.osb + t * a.osl;
  const bool pad = a.mask && a.mask[(long long)b * a.L + t];
  for (int d = threadIdx.x; d < a.D; d += kThreads) {
    const long long at = (long long)b * a.G + d / a.size;
    const float z = pad ? 0.f : fmaf((Elem<T>::ld(x + d) - a.mean[at]) * a.rstd[at], a.gamma[d] + a.offset, a.beta[d]);
    Elem<T>::st(y + d, a.silu ? z * sig<T>(z) : z);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_wide_sums_kernel(GnArgs a) {
  const int b = blockIdx.y;
  const long long at = (long long)b * a.G + blockIdx.x;
  const float m = a.mean[at], r = a.rstd[at];
  float s = 0.f, q = 0.f, u = 0.f, v = 0.f;
  int in = 0;
  wide_each(a, [&](int t, int d) {
    const float w = a.gamma[d] + a.offset;
    const float e = Elem<T>::ld((const T*)a.x + b * a.xsb + t * a.xsl + d) - m;
    const float dn = w * slope_of<T>(e, Elem<T>::ld((const T*)a.dy + b * a.gsb + t * a.gsl + d), r * w, a.beta[d], a.silu);
    u += dn;
    v = fmaf(dn, e * r, v);
    if (++in == kRun) s += u, q += v, u = v = 0.f, in = 0;
  });
  s = block_sum(s + u), q = block_sum(q + v);
  if (threadIdx.x == 0) {
    const float n = (float)a.count[b] * (float)a.size, inv = n > 0.f ? 1.f / n : 0.f;
    a.part[2 * at] = s * inv;
    a.part[2 * at + 1] = q * inv;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_wide_grads_kernel(GnArgs a) {
  const int t = blockIdx.x, b = blockIdx.y;
  const T *x = (const T*)a.x + b * a.xsb + t * a.xsl, *dy = (const T*)a.dy + b * a.gsb + t * a.gsl;
  T* dx = (T*)a.out + b * a.osb + t * a.osl;
  const bool pad = a.mask && a.mask[(long long)b * a.L + t];
  for (int d = threadIdx.x; d < a.D; d += kThreads) {
    const long long at = (long long)b * a.G + d / a.size;
    float o = 0.f;
    if (!pad) {
      const float w = a.gamma[d] + a.offset;
      const float e = Elem<T>::ld(x + d) - a.mean[at], r = a.rstd[at];
      const float dz = slope_of<T>(e, Elem<T>::ld(dy + d), r * w, a.beta[d], a.silu);
      o = r * (fmaf(dz, w, -a.part[2 * at]) - e * r * a.part[2 * at + 1]);
    }
    Elem<T>::st(dx + d, o);
  }
}

// the channels' sums over one sequence, 32 channels to a block, as the tiled kernels leave them for a run
template <typename T>
__global__ void __launch_bounds__(kThreads) gn_wide_channels_kernel(GnArgs a) {
  const int lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane, w = threadIdx.x >> 5, b = blockIdx.y;
  float s = 0.f, q = 0.f, u = 0.f, v = 0.f;
  if (d < a.D) {
    const long long at = (long long)b * a.G + d / a.size;
    int in = 0;
    for (int t = w; t < a.L; t += kThreads / 32) {
      if (a.mask && a.mask[(long long)b * a.L + t]) continue;
      const float e = Elem<T>::ld((const T*)a.x + b * a.xsb + t * a.xsl + d) - a.mean[at], r = a.rstd[at];
      const float dz = slope_of<T>(e, Elem<T>::ld((const T*)a.dy + b * a.gsb + t * a.gsl + d), r * (a.gamma[d] + a.offset), a.beta[d], a.silu);
      u += dz;
      v = fmaf(dz, e * r, v);
      if (++in == kRun) s += u, q += v, u = v = 0.f, in = 0;
    }
  }
  __shared__ float part[2][8][32];
  part[0][w][lane] = s + u;
  part[1][w][lane] = q + v;
  __syncthreads();
  if (w == 0 && d < a.D) {
    s = q = 0.f;
    for (int k = 0; k < 8; ++k) s += part[0][k][lane], q += part[1][k][lane];
    a.chan[(long long)b * 2 * a.D + d] = s;
    a.chan[(long long)b * 2 * a.D + a.D + d] = q;
  }
}

// ---- host ------------------------------------------------------------------------------------
int check_gn(int dtype, int B, int L, int D, int G, std::initializer_list<const void*> acts) {
  if (!valid_dtype(dtype)) return MEGA_ERR_DTYPE;
  if (B <= 0 || L <= 0 || D <= 0 || G <= 0 || D % G != 0) return MEGA_ERR_SHAPE;
  if (B > 65535 || G > 65535 || L > 1 << 24) return MEGA_ERR_UNSUPPORTED;   // (counts of steps are fp32)
  for (const void* p : acts)
    if (!aligned_to(p, elem_size(dtype))) return MEGA_ERR_ALIGN;
  return MEGA_OK;
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

struct Plan {
  int ng, tiles, steps, runs, piece;   // piece: slices that a pass leaves in L2 for the next
};
constexpr long long kL2 = 48ll << 20;   // bytes of inputs that the second pass finds in L2

Plan plan_of(int dtype, int B, int L, int D, int G, int vec, bool bwd) {
  const int es = elem_size(dtype), size = D / G, arrays = bwd ? 2 : 1;
  Plan p;
  if (vec == 0) return {G, 1, L, 1, 1};
  // a tile: whole groups and whole vectors, 128 bytes or more of a row where there are as many
  const int unit = vec / gcd(size, vec);
  p.ng = unit;
  while (p.ng < G && p.ng * size * es < 128) p.ng += unit;
  while (p.ng > G) p.ng -= unit;
  if (p.ng <= 0) p.ng = G;   // (D is whole vectors: the row is)
  p.tiles = (G + p.ng - 1) / p.ng;
  const long long slices = (long long)B * p.tiles, row = (long long)p.ng * size * es * arrays;
  // a block's run of steps: some 64 KB, fewer where the device would not be full, one run where a sequence is little more
  long long steps = std::max<long long>(1, (64 << 10) / row);
  const long long blocks = 4 * 148;
  if (slices * ((L + steps - 1) / steps) < blocks) steps = std::max<long long>((L * slices + blocks - 1) / blocks, std::max<long long>(1, (8 << 10) / row));
  if (L <= 2 * steps || (slices >= 296 && L * row <= (256 << 10))) steps = L;
  const int nv = std::max(1, p.ng * size / vec);
  steps = std::min<long long>(steps, (long long)kRun * std::max(1, kThreads / nv));
  p.steps = (int)std::min<long long>(steps, L);
  p.runs = (L + p.steps - 1) / p.steps;
  p.piece = (int)std::min<long long>(slices, std::max<long long>(1, kL2 / (row * L)));
  if (p.runs == 1) p.piece = (int)std::min<long long>(slices, 65535);
  return p;
}

// Channels of a vector: 16 or 4 bytes where all rows start on them and the row is whole vectors, else one; 0 where a block's threads
// do not span the groups that whole vectors make up.
int vec_of(int dtype, int D, int G, std::initializer_list<std::pair<const void*, std::pair<long long, long long>>> ops) {
  const int es = elem_size(dtype), size = D / G;
  auto fits = [&](int bytes) {
    const int v = bytes / es;
    if (D % v != 0 || size / gcd(size, v) > kThreads) return false;
    return std::all_of(ops.begin(), ops.end(), [&](const auto& o) {
      return aligned_to(o.first, bytes) && o.second.first * es % bytes == 0 && o.second.second * es % bytes == 0;
    });
  };
  return fits(16) ? 16 / es : fits(4) ? 4 / es : fits(es) ? 1 : 0;
}

void fill(GnArgs& a, const Plan& p) {
  a.ng = p.ng, a.tiles = p.tiles, a.steps = p.steps, a.runs = p.runs;
}

// first pass, second pass, piece by piece
template <typename First, typename Second>
void passes(First first, Second second, GnArgs a, int slices, int piece, cudaStream_t s) {
  for (int at = 0; at < slices; at += piece) {
    a.first = at;
    a.slices = std::min(piece, slices - at);
    if (at == 0)
      launch(first, dim3(a.runs, a.slices), dim3(kThreads), 0, s, a);
    else
      launch_after(first, dim3(a.runs, a.slices), dim3(kThreads), 0, s, a);
    if (a.runs > 1) launch_after(second, dim3(a.runs, a.slices), dim3(kThreads), 0, s, a);
  }
}
template <typename T, int kV, bool kOne>
void run_one(bool bwd, const GnArgs& a, const Plan& p, cudaStream_t s) {
  const int slices = a.B * p.tiles, piece = std::min(p.piece, 65535);
  if (bwd)
    passes(gn_sums_kernel<T, kV, kOne>, gn_grads_kernel<T, kV, kOne>, a, slices, piece, s);
  else
    passes(gn_first_kernel<T, kV, kOne>, gn_second_kernel<T, kV, kOne>, a, slices, piece, s);
}
template <typename T, int kV>
void run_vec(bool bwd, const GnArgs& a, const Plan& p, cudaStream_t s) {
  if constexpr (kV * sizeof(T) == 16) {
    if (a.size % kV == 0) return run_one<T, kV, true>(bwd, a, p, s);
  }
  run_one<T, kV, kV == 1>(bwd, a, p, s);
}
template <typename T>
void run_gn(bool bwd, int vec, const GnArgs& a, const Plan& p, cudaStream_t s) {
  if (vec == 0) {
    if (bwd) {
      launch(gn_wide_sums_kernel<T>, dim3(a.G, a.B), dim3(kThreads), 0, s, a);
      launch(gn_wide_grads_kernel<T>, dim3(a.L, a.B), dim3(kThreads), 0, s, a);
      launch(gn_wide_channels_kernel<T>, dim3((a.D + 31) / 32, a.B), dim3(kThreads), 0, s, a);
    } else {
      launch(gn_wide_stats_kernel<T>, dim3(a.G, a.B), dim3(kThreads), 0, s, a);
      launch(gn_wide_apply_kernel<T>, dim3(a.L, a.B), dim3(kThreads), 0, s, a);
    }
    return;
  }
  if (vec == 16 / (int)sizeof(T)) return run_vec<T, 16 / (int)sizeof(T)>(bwd, a, p, s);
  if constexpr (sizeof(T) == 2) {
    if (vec == 2) return run_vec<T, 2>(bwd, a, p, s);
  }
  run_vec<T, 1>(bwd, a, p, s);
}

size_t work_bytes(const Plan& p, int B, int D, int G, bool bwd) {
  const size_t parts = (size_t)B * p.runs;
  return 16 + sizeof(float) * (bwd ? parts * 2 * ((size_t)D + G) : parts * 3 * G);
}

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int64_t mega_group_norm_work(int dtype, int B, int L, int D, int num_groups) {
  if (check_gn(dtype, B, L, D, num_groups, {})) return 0;
  size_t most = 0;
  for (int vec : {16 / elem_size(dtype), 4 / elem_size(dtype), 1, 0})
    for (bool bwd : {false, true}) most = std::max(most, work_bytes(plan_of(dtype, B, L, D, num_groups, vec, bwd), B, D, num_groups, bwd));
  return (int64_t)most;
}

extern "C" int mega_group_norm_fwd(const void* x, void* y, int dtype, int B, int L, int D, int64_t xsb, int64_t xsl, int64_t ysb,
                                   int64_t ysl, const float* gamma, const float* beta, const uint8_t* pad_mask, int num_groups,
                                   double eps, unsigned flags, int64_t* count, float* mean, float* rstd, void* work,
                                   mega_stream_t stream) {
  if (!x || !y || !gamma || !beta || !count || !mean || !rstd || !work) return MEGA_ERR_NULL;
  if (int rc = check_gn(dtype, B, L, D, num_groups, {x, y})) return rc;
  if (!aligned_to(work, 16)) return MEGA_ERR_ALIGN;
  GnArgs a = {};
  a.x = x, a.out = y, a.xsb = xsb, a.xsl = xsl, a.osb = ysb, a.osl = ysl, a.gamma = gamma, a.beta = beta, a.mask = pad_mask;
  a.B = B, a.L = L, a.D = D, a.G = num_groups, a.size = D / num_groups;
  a.eps = (float)eps, a.offset = flags & MEGA_GN_OFFSET ? 1.f : 0.f, a.silu = (flags & MEGA_GN_SILU) != 0;
  a.count = (long long*)count, a.mean = mean, a.rstd = rstd, a.part = (float*)work;
  const int vec = vec_of(dtype, D, num_groups, {{x, {xsb, xsl}}, {y, {ysb, ysl}}});
  const Plan p = plan_of(dtype, B, L, D, num_groups, vec, false);
  fill(a, p);
  MEGA_DISPATCH_DTYPE(dtype, run_gn<T>(false, vec, a, p, (cudaStream_t)stream));
  return check_launch("group_norm_fwd");
}

extern "C" int mega_group_norm_bwd(const void* dy, const void* x, void* dx, int dtype, int B, int L, int D, int64_t gsb, int64_t gsl,
                                   int64_t xsb, int64_t xsl, int64_t dsb, int64_t dsl, const float* gamma, const float* beta,
                                   const uint8_t* pad_mask, int num_groups, unsigned flags, const int64_t* count, const float* mean,
                                   const float* rstd, float* dgamma, float* dbeta, void* work, mega_stream_t stream) {
  if (!dy || !x || !dx || !gamma || !beta || !count || !mean || !rstd || !dgamma || !dbeta || !work) return MEGA_ERR_NULL;
  if (int rc = check_gn(dtype, B, L, D, num_groups, {dy, x, dx})) return rc;
  if (!aligned_to(work, 16)) return MEGA_ERR_ALIGN;
  GnArgs a = {};
  a.x = x, a.dy = dy, a.out = dx, a.xsb = xsb, a.xsl = xsl, a.gsb = gsb, a.gsl = gsl, a.osb = dsb, a.osl = dsl;
  a.gamma = gamma, a.beta = beta, a.mask = pad_mask;
  a.B = B, a.L = L, a.D = D, a.G = num_groups, a.size = D / num_groups;
  a.offset = flags & MEGA_GN_OFFSET ? 1.f : 0.f, a.silu = (flags & MEGA_GN_SILU) != 0;
  a.count = (long long*)count, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.dgamma = dgamma, a.dbeta = dbeta;
  const int vec = vec_of(dtype, D, num_groups, {{dy, {gsb, gsl}}, {x, {xsb, xsl}}, {dx, {dsb, dsl}}});
  const Plan p = plan_of(dtype, B, L, D, num_groups, vec, true);
  fill(a, p);
  a.chan = (float*)work, a.part = a.chan + (size_t)B * p.runs * 2 * D;
  MEGA_DISPATCH_DTYPE(dtype, run_gn<T>(true, vec, a, p, (cudaStream_t)stream));
  launch_after(gn_params_kernel, dim3((D + 31) / 32), dim3(1024), 0, stream, a);
  return check_launch("group_norm_bwd");
}

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
// Small calls are held in shared memory by clusters of blocks, in one pass (gn_held_*).
//
// Bound: HBM, but for the held calls with every input twice: what the second pass, which goes backwards, finds in L2 of the first
// saves it little, as its 16 special-function operations to a vector take as long (16 x 4096 x 512 bf16, 32 groups, forward: 17 us
// for the first pass, 26 for the second, which takes 24 of its 67 MB from DRAM, 25 for a copy; 6 x 32768 x 1024 206 us, 0.90 of the
// measured copy rate over the three arrays).  Calls in pieces that fit L2 were slower by their launches (6 x 32768 x 1024 forward 231
// us against 206, backward 446 against 324; a call that fits as it is takes the same).  Of the kernels only the sums of 16-bit groups
// that share a vector spill registers (44 bytes a thread).
//
// Statistics: a thread adds up d = x - p and d^2 with p the first value of its run.  p being one of the n values, the squares about
// it are at most n + 1 times those about the mean, so n <= kRun bounds what their difference loses; such entries are then joined by
// counts, means and squared deviations: the mean of all first, then the deviations about it (Chan's rule, entry after entry with its
// divisions, took the first pass 1.7 us a block).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "gates.cuh"
#include "tma.cuh"

namespace mega {

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 64;        // steps of a thread at most
constexpr int kGroups = 256;    // groups of a tile at most

struct GnArgs {
  const void *x, *dy;
  void* out;
  long long xsb, xsl, gsb, gsl, osb, osl;
  const float *gamma, *beta;
  const unsigned char* mask;
  int B, L, D, G, size;        // size: channels of a group
  int ng, tiles;               // groups of a tile, tiles of a row
  int nv, lanes;               // vectors of a tile's row, rows that a block takes at once
  int steps, runs;             // steps of a block, blocks of a sequence
  float over_nv, over_size, over_vectors;   // reciprocals: of a row's vectors, a group's channels, a group's vectors
  float eps, offset;
  int silu;
  long long* count;
  float *mean, *rstd;
  float *part, *chan;          // partial results of a run: of its groups (3 or 2 values), backward: of its channels (2)
  float *dgamma, *dbeta;
};

// kV neighbouring channels: as pairs of fp32 values (packed arithmetic; with one channel the second of the pair is idle)
template <typename T, int kV>
struct Vec {
  static constexpr int kBytes = kV * (int)sizeof(T), kP = (kV + 1) / 2;
  static __device__ __forceinline__ void fetch(uint32_t slot, const T* p) {   // to shared memory, asynchronously
    static_assert(kBytes == 16 || kBytes == 4, "");
    if (kBytes == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(p) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot), "l"(p) : "memory");
  }
  static __device__ __forceinline__ void read(const char* slot, f32x2 (&f)[kP]) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(slot);
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < kP; ++j) f[j] = sizeof(T) == 4 ? pack2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1])) : two(w[j]);
    } else {
      const unsigned w = *reinterpret_cast<const unsigned*>(slot);
      f[0] = sizeof(T) == 4 ? pack2(__uint_as_float(w), 0.f) : two(w);
    }
  }
  static __device__ __forceinline__ f32x2 two(unsigned w) {   // a pair of 16-bit values
    if constexpr (sizeof(T) == 2) {
      const T* e = reinterpret_cast<const T*>(&w);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      return pack2(Elem<T>::ld_shared(e), Elem<T>::ld_shared(e + 1));
    }
    return 0;
  }
  static __device__ __forceinline__ unsigned one(f32x2 v) {
    float a, b;
    unpack2(v, a, b);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
      return *reinterpret_cast<const unsigned*>(&r);
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ void store(T* p, const f32x2 (&f)[kP]) {
    if constexpr (kV == 1) {
      float a, b;
      unpack2(f[0], a, b);
      Elem<T>::st(p, a);
    } else if constexpr (sizeof(T) == 4) {
      float4 v;
      unpack2(f[0], v.x, v.y);
      unpack2(f[kP - 1], v.z, v.w);
      *reinterpret_cast<float4*>(p) = v;
    } else if constexpr (kBytes == 16) {
      *reinterpret_cast<uint4*>(p) = make_uint4(one(f[0]), one(f[kP > 1 ? 1 : 0]), one(f[kP > 2 ? 2 : 0]), one(f[kP - 1]));
    } else {
      *reinterpret_cast<unsigned*>(p) = one(f[0]);
    }
  }
};
__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }

// sigmoid(z): fp32 with the full-range exponential and division, 16-bit types with the approximate ones (relative 2^-22 or so)
template <typename T>
__device__ __forceinline__ float sig(float z) {
  return sizeof(T) == 4 ? 1.f / (1.f + expf(-z)) : rcp_approx(1.f + __expf(-z));
}
// a / b for 0 <= a < 2^16 and b's reciprocal (off by less than 2^-23 of it: the half keeps the quotient on its side)
__device__ __forceinline__ int quotient(int a, float over) { return __float2int_rd(((float)a + 0.5f) * over); }

// What a block works on.
template <int kV>
struct Where {
  int b, tile, run, c0, chans, groups, t0, t1;   // first channel, channels, groups; steps
  int nv, lanes, v, r;                           // vectors of a row, rows at once; this thread's vector and row
  bool on;
  __device__ __forceinline__ Where(const GnArgs& a, bool back) {
    b = back ? gridDim.z - 1 - blockIdx.z : blockIdx.z;
    tile = back ? gridDim.y - 1 - blockIdx.y : blockIdx.y;
    run = back ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    c0 = tile * a.ng * a.size;
    groups = min(a.ng, a.G - tile * a.ng);
    chans = groups * a.size;
    t0 = run * a.steps, t1 = min(t0 + a.steps, a.L);
    nv = a.nv;
    lanes = a.lanes;
    r = quotient(threadIdx.x, a.over_nv), v = threadIdx.x - r * nv;
    on = r < lanes && v * kV < chans;
  }
};

// Shared memory: every thread's own ring of vectors that are on their way, the block's sums.
constexpr int kRing = 32 << 10;   // bytes of the ring: eight rows of one operand, four of two
constexpr int kHeld = 16, kHeldBack = 12;   // vectors that a thread keeps where a cluster holds a sequence: three blocks fit a multiprocessor
struct Sums {
  float n[kThreads];
  float g[3][kGroups];        // of a group: mean, rstd; backward the two sums
  unsigned bits[kRun * kThreads / 32];   // padded steps of the block
  float a[2 * kThreads * 8];   // two arrays [row of the block][channel of the tile] (or vector, where it is one entry)
};
// behind it the ring, or what is held; a forward pass of one entry to a vector needs an eighth of the arrays
constexpr int kPlaces = (sizeof(Sums) + 15) / 16 * 16, kFewer = kPlaces - 2 * kThreads * 7 * (int)sizeof(float);
// Groups of a held tile at most: a cluster's joined statistics, three values to a group, go to what there is of the arrays then.
constexpr int kHeldGroups = 2 * kThreads / 3;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// the padded steps of the block as bits
template <int kV>
__device__ __forceinline__ void read_mask(const GnArgs& a, const Where<kV>& p, Sums& s) {
  if (a.mask == nullptr) return;
  const unsigned char* mask = a.mask + (long long)p.b * a.L + p.t0;
  const int n = p.t1 - p.t0;
#pragma unroll 8
  for (int i = threadIdx.x; i < (n + 31) / 32 * 32; i += kThreads) {
    const unsigned bits = __ballot_sync(0xffffffffu, i < n && mask[i] != 0);
    if ((threadIdx.x & 31) == 0) s.bits[i >> 5] = bits;
  }
  __syncthreads();
}

// The thread's rows of the block, in order or back.  begin() sets the first of them on their way to the thread's own places in
// shared memory, run(f) calls f(values, address, first, live) for each (live: not padded; address: of the output's vector
// there).  What a block has under way so takes no registers, and begins before what the rows are needed for is known (16 x 4096 x
// 512 bf16, 32 groups: 64 us with rows of the ring asked for in order, 45 with them under way before the launch before has ended).
template <typename T, int kV, int kOps>
struct Walk {
  using V = Vec<T, kV>;
  static constexpr int kP = V::kP, kDepth = kRing / (kThreads * 16 * kOps);
  const T* q[kOps];
  long long hop[kOps], next;
  T* at;
  int mine, start, step, ahead = 0;
  const char* own;
  __device__ __forceinline__ Walk(const GnArgs& a, const Where<kV>& p, char* place, bool back, T* out) {
    const int total = p.t1 - p.t0;
    mine = p.on && p.r < total ? quotient(total - p.r + p.lanes - 1, 1.f / (float)p.lanes) : 0;   // (at most kRun)
    start = back ? p.r + (mine - 1) * p.lanes : p.r, step = back ? -p.lanes : p.lanes;
    const int c = p.c0 + p.v * kV;
    q[0] = (const T*)a.x + p.b * a.xsb + (p.t0 + start) * a.xsl + c, hop[0] = step * a.xsl;
    if (kOps == 2) q[kOps - 1] = (const T*)a.dy + p.b * a.gsb + (p.t0 + start) * a.gsl + c, hop[kOps - 1] = step * a.gsl;
    at = out + p.b * a.osb + (p.t0 + start) * a.osl + c, next = step * a.osl;
    own = place + threadIdx.x * 16;
  }
  __device__ __forceinline__ void fetch(int u) {   // the next row, into place u
    if constexpr (V::kBytes != 2) {
      if (ahead < mine) {
#pragma unroll
        for (int o = 0; o < kOps; ++o) {
          V::fetch(smem_u32(own) + (u * kOps + o) * (kThreads * 16), q[o]);
          q[o] += hop[o];
        }
      }
      ++ahead;
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int u = 0; u < kDepth - 1; ++u) fetch(u);
  }
  template <typename F>
  __device__ __forceinline__ void run(const Sums& s, bool masked, F&& f) {
    auto live = [&](int k) {
      if (!masked) return true;
      const int i = start + k * step;
      return !((s.bits[i >> 5] >> (i & 31)) & 1u);
    };
    if constexpr (V::kBytes == 2) {   // (no copy is that short: eight at a time through registers)
      constexpr int kN = 8 / kOps;
      for (int k = 0; k < mine; k += kN) {
        float v[kN][kOps];
#pragma unroll
        for (int u = 0; u < kN; ++u)
#pragma unroll
          for (int o = 0; o < kOps; ++o) v[u][o] = k + u < mine ? Elem<T>::ld(q[o] + (k + u) * hop[o]) : 0.f;
#pragma unroll
        for (int u = 0; u < kN; ++u) {
          f32x2 w[kOps][kP];
#pragma unroll
          for (int o = 0; o < kOps; ++o) w[o][0] = pack2(v[u][o], 0.f);
          if (k + u < mine) f(w, at, k + u == 0, live(k + u));
          at += next;
        }
      }
    } else {
      auto use = [&](int k, int u) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
        f32x2 w[kOps][kP];
#pragma unroll
        for (int o = 0; o < kOps; ++o) V::read(own + (u * kOps + o) * (kThreads * 16), w[o]);
        f(w, at, k == 0, live(k));
        at += next;
      };
      int k = 0;
      for (; k + kDepth <= mine; k += kDepth) {
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
          use(k + u, u);
          fetch((u + kDepth - 1) % kDepth);
        }
      }
#pragma unroll
      for (int u = 0; u < kDepth - 1; ++u) {
        if (k + u < mine) use(k + u, u);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  }
};

// The same with every row kept: a block's steps are what its threads' places hold, and rows are there for a second run.
template <typename T, int kV, int kOps>
struct Held {
  using V = Vec<T, kV>;
  static constexpr int kP = V::kP, kRows = (kOps == 1 ? kHeld : kHeldBack) / kOps, kSteps = (kRows + 3) / 4;
  int mine, start, step;
  T* to;
  long long next;
  const char* own;
  __device__ __forceinline__ Held(const GnArgs& a, const Where<kV>& p, char* place, T* out) {
    const int total = p.t1 - p.t0, c = p.c0 + p.v * kV;
    mine = p.on && p.r < total ? quotient(total - p.r + p.lanes - 1, 1.f / (float)p.lanes) : 0;   // (at most kRows)
    start = p.r, step = p.lanes;
    own = place + threadIdx.x * 16;
    const T *x = (const T*)a.x + p.b * a.xsb + (p.t0 + start) * a.xsl + c, *dy = nullptr;
    const long long hx = step * a.xsl, hy = kOps == 2 ? step * a.gsl : 0;
    if (kOps == 2) dy = (const T*)a.dy + p.b * a.gsb + (p.t0 + start) * a.gsl + c;
    const uint32_t at = smem_u32(own);
    auto row = [&](int k) {
      V::fetch(at + k * kOps * (kThreads * 16), x);
      x += hx;
      if (kOps == 2) {
        V::fetch(at + (k * kOps + 1) * (kThreads * 16), dy);
        dy += hy;
      }
    };
#pragma unroll
    for (int q = 0; q < kSteps; ++q) {
      if (mine >= min(4 * q + 4, kRows)) {
#pragma unroll
        for (int k = 4 * q; k < min(4 * q + 4, kRows); ++k) row(k);
      } else {
        for (int k = 4 * q; k < mine; ++k) row(k);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    to = out + p.b * a.osb + (p.t0 + start) * a.osl + c, next = step * a.osl;
  }
  template <int kQ, typename F>
  __device__ __forceinline__ void quarter(const Sums& s, bool masked, T*& at, F&& f) {
    if constexpr (kQ < kSteps) {
      constexpr int kEnd = 4 * kQ + 4 < kRows ? 4 * kQ + 4 : kRows;
      asm volatile("cp.async.wait_group %0;" ::"n"(kSteps - 1 - kQ) : "memory");
      auto use = [&](int k, bool live) {
        f32x2 w[kOps][kP];
#pragma unroll
        for (int o = 0; o < kOps; ++o) V::read(own + (k * kOps + o) * (kThreads * 16), w[o]);
        f(w, at, k == 0, live);
        at += next;
      };
      if (mine >= kEnd && !masked) {
#pragma unroll
        for (int k = 4 * kQ; k < kEnd; ++k) use(k, true);
      } else {
#pragma unroll 1
        for (int k = 4 * kQ; k < min(kEnd, mine); ++k) {
          const int i = start + k * step;
          use(k, !(masked && ((s.bits[i >> 5] >> (i & 31)) & 1u)));
        }
      }
      quarter<kQ + 1>(s, masked, at, f);
    }
  }
  template <typename F>
  __device__ __forceinline__ void run(const Sums& s, bool masked, F&& f) {
    T* at = to;
    quarter<0>(s, masked, at, f);
  }
};

// the blocks of a cluster, which share a sequence's steps
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer(const float* p, int rank) {   // a float of another block's shared memory
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// ---- forward -----------------------------------------------------------------------------------
// Statistics of n values, means m[k] of counts c[k] and squared deviations q[k]: mean = sum c m / n, then sum q + c (m - mean)^2.
//
// Of the tile's groups over the block's steps -> s.g: steps, mean, squared deviations of all channels over their number.
// kOne: a vector lies in one group; its values are then one entry.
template <typename T, int kV, bool kOne, typename W>
__device__ __forceinline__ void moments(const GnArgs& a, const Where<kV>& p, Sums& s, W& walk, Walk<T, kV, 1>* then) {
  constexpr int kE = kOne ? 1 : kV, kP = Vec<T, kV>::kP, kPlane = kThreads * kE;   // entries that a thread leaves, pairs
  float cnt = 0.f;
  f32x2 pv[kP], S[kP], Q[kP];
#pragma unroll
  for (int j = 0; j < kP; ++j) S[j] = Q[j] = pv[j] = both(0.f);
  walk.run(s, a.mask != nullptr, [&](f32x2(&f)[1][kP], T*, bool first, bool live) {
    if (!live) return;
    if (a.mask != nullptr ? cnt == 0.f : first) {
#pragma unroll
      for (int j = 0; j < kP; ++j) pv[j] = f[0][j];
    }
    cnt += 1.f;
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      const f32x2 d = sub2(f[0][j], pv[j]);
      S[j] = add2(S[j], d);
      Q[j] = fma2(d, d, Q[j]);
    }
  });
  if (then) then->begin();
  const float inv = cnt > 0.f ? 1.f / cnt : 0.f;
  const int width = p.nv * kE;
  if (p.r < p.lanes) {
    float m[2 * kP], q[2 * kP];
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      float s0, s1, q0, q1;
      unpack2(S[j], s0, s1), unpack2(Q[j], q0, q1), unpack2(pv[j], m[2 * j], m[2 * j + 1]);
      m[2 * j] = fmaf(s0, inv, m[2 * j]), m[2 * j + 1] = fmaf(s1, inv, m[2 * j + 1]);
      q[2 * j] = not_negative(fmaf(-s0 * inv, s0, q0)), q[2 * j + 1] = not_negative(fmaf(-s1 * inv, s1, q1));
    }
    if (kOne) {
      float mean = 0.f, all = 0.f;
#pragma unroll
      for (int j = 0; j < kV; ++j) mean += m[j];
      mean *= 1.f / kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) all += fmaf(cnt * (m[j] - mean), m[j] - mean, q[j]);
      m[0] = mean, q[0] = all;
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      s.a[p.r * width + p.v * kE + j] = m[j];
      s.a[kPlane + p.r * width + p.v * kE + j] = q[j];
    }
    if (p.v == 0) s.n[p.r] = cnt;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, per = kOne ? quotient(a.size, 1.f / kV) : a.size;   // entries of a row and group
  const float over_per = kOne ? a.over_vectors : a.over_size;
  float n = 0.f;
  for (int r = lane; r < p.lanes; r += 32) n += s.n[r];
  n = warp_sum(n);
  const float over = n > 0.f ? 1.f / (n * (float)per) : 0.f;
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    float sum = 0.f, dev = 0.f;
    for (int e = lane; e < p.lanes * per; e += 32) {
      const int r = quotient(e, over_per);
      sum = fmaf(s.n[r], s.a[r * width + g * per + e - r * per], sum);
    }
    const float mean = warp_sum(sum) * over;
    for (int e = lane; e < p.lanes * per; e += 32) {
      const int r = quotient(e, over_per), at = r * width + g * per + e - r * per;
      const float d = s.a[at] - mean, c = s.n[r] * (float)(kV / kE);
      if (c > 0.f) dev += fmaf(c * d, d, s.a[kPlane + at]);   // (an empty row has no mean)
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
  return p.on ? quotient(p.v * kV + (kOne ? 0 : j), a.over_size) : 0;
}
// a pair of the thread's channels: what `of` says for each (0 for the idle one)
template <int kV, typename F>
__device__ __forceinline__ f32x2 pair_of(int j, F&& of) {
  return pack2(of(2 * j), kV == 1 ? 0.f : of(2 * j + 1));
}

// the thread's channels of gamma (+ 1) and beta
template <int kV>
struct Params {
  static constexpr int kP = (kV + 1) / 2;
  f32x2 w[kP], c[kP];
  __device__ __forceinline__ Params(const GnArgs& a, const Where<kV>& p) {
    const float *gamma = a.gamma + p.c0 + p.v * kV, *beta = a.beta + p.c0 + p.v * kV;
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      w[j] = pair_of<kV>(j, [&](int k) { return p.on ? gamma[k] + a.offset : 0.f; });
      c[j] = pair_of<kV>(j, [&](int k) { return p.on ? beta[k] : 0.f; });
    }
  }
};

template <typename T, int kV, bool kOne, typename W>
__device__ __forceinline__ void apply(const GnArgs& a, const Where<kV>& p, Sums& s, W& walk, const Params<kV>& k) {
  constexpr int kP = Vec<T, kV>::kP, kM = kOne ? 1 : kP;
  f32x2 m[kM], scale[kP];
#pragma unroll
  for (int j = 0; j < kM; ++j) m[j] = pair_of<kOne ? 2 : kV>(j, [&](int c) { return s.g[0][group_of<kV, kOne>(a, p, c)]; });
#pragma unroll
  for (int j = 0; j < kP; ++j) scale[j] = mul2(k.w[j], pair_of<kV>(j, [&](int c) { return s.g[1][group_of<kV, kOne>(a, p, c)]; }));
  walk.run(s, a.mask != nullptr, [&](f32x2(&f)[1][kP], T* at, bool, bool live) {
    f32x2 o[kP];
#pragma unroll
    for (int j = 0; j < kP; ++j) o[j] = fma2(sub2(f[0][j], m[kOne ? 0 : j]), scale[j], k.c[j]);
    if (a.silu) {
#pragma unroll
      for (int j = 0; j < kP; ++j) o[j] = mul2(o[j], minus_sigmoid2<T, -1>(o[j]) ^ 0x8000000080000000ull);
    }
    if (!live) {
#pragma unroll
      for (int j = 0; j < kP; ++j) o[j] = both(0.f);
    }
    Vec<T, kV>::store(at, o);
  });
}

// the partial results of the tile's groups, of every run (steps, mean, squared deviations)
__device__ __forceinline__ void fold(const GnArgs& a, int b, int tile, int groups, Sums& s) {
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < groups; g += kThreads / 32) {
    const float* q = a.part + (((long long)b * a.G + tile * a.ng + g) * a.runs) * 3;
    float n = 0.f, sum = 0.f, dev = 0.f, c0 = 0.f, m0 = 0.f, q0 = 0.f;
    if (lane < a.runs) c0 = q[3 * lane], m0 = q[3 * lane + 1], q0 = q[3 * lane + 2];
    n = c0, sum = c0 * m0;
    for (int r = lane + 32; r < a.runs; r += 32) {
      n += q[3 * r];
      sum = fmaf(q[3 * r], q[3 * r + 1], sum);
    }
    n = warp_sum(n), sum = warp_sum(sum);
    const float mean = n > 0.f ? sum / n : 0.f;
    if (c0 > 0.f) dev = fmaf(c0 * (m0 - mean), m0 - mean, q0);
    for (int r = lane + 32; r < a.runs; r += 32) {
      const float d = q[3 * r + 1] - mean;
      if (q[3 * r] > 0.f) dev += fmaf(q[3 * r] * d, d, q[3 * r + 2]);
    }
    dev = warp_sum(dev);
    if (lane == 0) s.g[0][g] = n, s.g[1][g] = mean, s.g[2][g] = dev;
  }
  __syncthreads();
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 4) gn_first_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  pdl_wait();
  const Where<kV> p(a, false);
  Walk<T, kV, 1> walk(a, p, smem + kPlaces, false, (T*)a.out);
  walk.begin();
  pdl_next();
  read_mask(a, p, s);
  if (a.runs == 1) {
    Walk<T, kV, 1> again(a, p, smem + kPlaces, true, (T*)a.out);
    moments<T, kV, kOne>(a, p, s, walk, &again);
    const Params<kV> k(a, p);
    finish(a, p, s, true);
    apply<T, kV, kOne>(a, p, s, again, k);
    return;
  }
  moments<T, kV, kOne>(a, p, s, walk, nullptr);
  for (int g = threadIdx.x; g < p.groups; g += kThreads) {
    float* q = a.part + (((long long)p.b * a.G + p.tile * a.ng + g) * a.runs + p.run) * 3;
    q[0] = s.g[0][g], q[1] = s.g[1][g], q[2] = s.g[2][g];
  }
}

// (what it reads of the caller's is there before the first pass begins, so its rows are on their way before that has ended)
template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 4) gn_second_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  const Where<kV> p(a, true);
  Walk<T, kV, 1> walk(a, p, smem + kPlaces, true, (T*)a.out);
  walk.begin();
  const Params<kV> k(a, p);
  read_mask(a, p, s);
  pdl_wait();
  pdl_next();
  fold(a, p.b, p.tile, p.groups, s);
  finish(a, p, s, p.run == 0);
  apply<T, kV, kOne>(a, p, s, walk, k);
}

// In one pass: a cluster's blocks hold the sequence's steps of the tile, and tell one another their statistics.
template <typename T, int kV>
__global__ void __launch_bounds__(kThreads, 3) gn_held_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  const Where<kV> p(a, false);
  Held<T, kV, 1> rows(a, p, smem + kFewer, (T*)a.out);
  const Params<kV> k(a, p);
  read_mask(a, p, s);
  moments<T, kV, true>(a, p, s, rows, nullptr);
  if (a.runs > 1) {
    cluster_arrive();
    cluster_wait();
    // a lane to a block (their results stay where they are until all have read them, the own ones go to where the counts were)
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
      float n = 0.f, m = 0.f, q = 0.f;
      if (lane < a.runs) n = peer(&s.g[0][g], lane), m = peer(&s.g[1][g], lane), q = peer(&s.g[2][g], lane);
      const float all = warp_sum(n), mean = all > 0.f ? warp_sum(n * m) / all : 0.f;
      const float dev = warp_sum(n > 0.f ? fmaf(n * (m - mean), m - mean, q) : 0.f);
      if (lane == 0) s.a[3 * g] = all, s.a[3 * g + 1] = mean, s.a[3 * g + 2] = dev;
    }
    cluster_arrive();
    cluster_wait();
    for (int g = threadIdx.x; g < p.groups; g += kThreads) s.g[0][g] = s.a[3 * g], s.g[1][g] = s.a[3 * g + 1], s.g[2][g] = s.a[3 * g + 2];
    __syncthreads();
  }
  finish(a, p, s, p.run == 0);
  apply<T, kV, true>(a, p, s, rows, k);
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
  static constexpr int kP = Vec<T, kV>::kP, kM = kOne ? 1 : kP;
  f32x2 m[kM], scale[kP], beta[kP];
  __device__ __forceinline__ Back(const GnArgs& a, const Where<kV>& p) {
    const long long at = (long long)p.b * a.G + p.tile * a.ng;
    const float *mean = a.mean + at, *rstd = a.rstd + at;
    const Params<kV> k(a, p);
#pragma unroll
    for (int j = 0; j < kM; ++j) m[j] = pair_of<kOne ? 2 : kV>(j, [&](int c) { return mean[group_of<kV, kOne>(a, p, c)]; });
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      scale[j] = mul2(k.w[j], pair_of<kV>(j, [&](int c) { return rstd[group_of<kV, kOne>(a, p, c)]; }));
      beta[j] = k.c[j];
    }
  }
  // d = x - mean, and minus dz
  __device__ __forceinline__ void slopes(const GnArgs& a, const f32x2 (&x)[kP], const f32x2 (&dy)[kP], f32x2 (&d)[kP], f32x2 (&ndz)[kP]) const {
#pragma unroll
    for (int j = 0; j < kP; ++j) d[j] = sub2(x[j], m[kOne ? 0 : j]);
    if (a.silu) {
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const f32x2 z = fma2(d[j], scale[j], beta[j]), ns = minus_sigmoid2<T, -1>(z);
        ndz[j] = mul2(mul2(dy[j], ns), add2(fma2(z, ns, z), both(1.f)));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kP; ++j) ndz[j] = dy[j] ^ 0x8000000080000000ull;
    }
  }
};

// sums of dz and dz xhat of every channel over the block's steps -> a.chan, of dn and dn xhat of every group -> s.g[0], s.g[1]
template <typename T, int kV, bool kOne, typename W>
__device__ __forceinline__ void sums(const GnArgs& a, const Where<kV>& p, Sums& s, const Back<T, kV, kOne>& k, W& walk, Walk<T, kV, 2>* then) {
  constexpr int kP = Vec<T, kV>::kP, kPlane = kThreads * kV;
  f32x2 nS[kP], nQ[kP];   // minus the sums of dz and of dz d (xhat being rstd d)
#pragma unroll
  for (int j = 0; j < kP; ++j) nS[j] = nQ[j] = both(0.f);
  walk.run(s, a.mask != nullptr, [&](f32x2(&f)[2][kP], T*, bool, bool live) {
    if (!live) return;
    f32x2 d[kP], ndz[kP];
    k.slopes(a, f[0], f[1], d, ndz);
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      nS[j] = add2(nS[j], ndz[j]);
      nQ[j] = fma2(ndz[j], d[j], nQ[j]);
    }
  });
  if (then) then->begin();
  float S[2 * kP], Q[2 * kP];
#pragma unroll
  for (int j = 0; j < kP; ++j) {
    unpack2(nS[j], S[2 * j], S[2 * j + 1]);
    unpack2(nQ[j], Q[2 * j], Q[2 * j + 1]);
  }
  const int width = p.nv * kV;
  if (p.r < p.lanes) {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      s.a[p.r * width + p.v * kV + j] = -S[j];
      s.a[kPlane + p.r * width + p.v * kV + j] = -Q[j];
    }
  }
  __syncthreads();
  // rows of the block: some threads to a channel, each every parts-th row, into that part's row
  const int parts = min(max(1, quotient(kThreads, 1.f / (float)width)), p.lanes);
  for (int e = threadIdx.x; e < parts * width; e += kThreads) {
    const int part = quotient(e, 1.f / (float)width), c = e - part * width;
    float u = 0.f, q = 0.f;
    for (int r = part; r < p.lanes; r += parts) u += s.a[r * width + c], q += s.a[kPlane + r * width + c];
    s.a[e] = u;
    s.a[kPlane + e] = q;
  }
  __syncthreads();
  const long long row = ((long long)p.b * a.runs + p.run) * 2 * a.D, at = (long long)p.b * a.G + p.tile * a.ng;
  for (int c = threadIdx.x; c < p.chans; c += kThreads) {
    float u = 0.f, q = 0.f;
    for (int k = 0; k < parts; ++k) u += s.a[k * width + c], q += s.a[kPlane + k * width + c];
    q *= a.rstd[at + quotient(c, a.over_size)];
    a.chan[row + p.c0 + c] = u;
    a.chan[row + a.D + p.c0 + c] = q;
    const float w = a.gamma[p.c0 + c] + a.offset;
    s.a[c] = u * w;   // (this thread alone has read the place)
    s.a[kPlane + c] = q * w;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    float u = 0.f, q = 0.f;
    for (int c = lane; c < a.size; c += 32) u += s.a[g * a.size + c], q += s.a[kPlane + g * a.size + c];
    u = warp_sum(u), q = warp_sum(q);
    if (lane == 0) s.g[0][g] = u, s.g[1][g] = q;
  }
  __syncthreads();
}

// sums of dn, dn xhat in s.g[0], s.g[1] -> dx = rstd dn - rstd mean(dn) - d rstd^2 mean(dn xhat)
template <typename T, int kV, bool kOne, typename W>
__device__ __forceinline__ void grads(const GnArgs& a, const Where<kV>& p, Sums& s, const Back<T, kV, kOne>& k, W& walk) {
  constexpr int kP = Vec<T, kV>::kP, kM = kOne ? 1 : kP;
  const float n = (float)a.count[p.b] * (float)a.size, inv = n > 0.f ? 1.f / n : 0.f;
  const float* rstd = a.rstd + (long long)p.b * a.G + p.tile * a.ng;
  f32x2 m1[kM], m2[kM];   // rstd times the one mean, rstd^2 times the other
#pragma unroll
  for (int j = 0; j < kM; ++j) {
    m1[j] = pair_of<kOne ? 2 : kV>(j, [&](int c) {
      const int g = group_of<kV, kOne>(a, p, c);
      return s.g[0][g] * inv * rstd[g];
    });
    m2[j] = pair_of<kOne ? 2 : kV>(j, [&](int c) {
      const int g = group_of<kV, kOne>(a, p, c);
      return s.g[1][g] * inv * rstd[g] * rstd[g];
    });
  }
  walk.run(s, a.mask != nullptr, [&](f32x2(&f)[2][kP], T* at, bool, bool live) {
    f32x2 d[kP], ndz[kP], o[kP];
    k.slopes(a, f[0], f[1], d, ndz);
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      // dz scale - m1 - d m2, the signs turned twice
      const f32x2 v = fma2(ndz[j], k.scale[j], fma2(d[j], m2[kOne ? 0 : j], m1[kOne ? 0 : j]));
      o[j] = live ? v ^ 0x8000000080000000ull : both(0.f);
    }
    Vec<T, kV>::store(at, o);
  });
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_sums_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  pdl_wait();
  const Where<kV> p(a, false);
  Walk<T, kV, 2> walk(a, p, smem + kPlaces, false, (T*)a.out);
  walk.begin();
  pdl_next();
  const Back<T, kV, kOne> k(a, p);
  read_mask(a, p, s);
  if (a.runs == 1) {
    Walk<T, kV, 2> again(a, p, smem + kPlaces, true, (T*)a.out);
    sums<T, kV, kOne>(a, p, s, k, walk, &again);
    grads<T, kV, kOne>(a, p, s, k, again);
    return;
  }
  sums<T, kV, kOne>(a, p, s, k, walk, nullptr);
  const long long at = (long long)p.b * a.G + p.tile * a.ng;
  for (int g = threadIdx.x; g < p.groups; g += kThreads) {
    float* q = a.part + ((at + g) * a.runs + p.run) * 2;
    q[0] = s.g[0][g], q[1] = s.g[1][g];
  }
}

template <typename T, int kV, bool kOne>
__global__ void __launch_bounds__(kThreads, 3) gn_grads_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  const int lane = threadIdx.x & 31;
  const Where<kV> p(a, true);
  Walk<T, kV, 2> walk(a, p, smem + kPlaces, true, (T*)a.out);
  walk.begin();
  const Back<T, kV, kOne> k(a, p);
  read_mask(a, p, s);
  pdl_wait();
  pdl_next();
  for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
    const float* q = a.part + (((long long)p.b * a.G + p.tile * a.ng + g) * a.runs) * 2;
    float u = 0.f, w = 0.f;
    for (int r = lane; r < a.runs; r += 32) u += q[2 * r], w += q[2 * r + 1];
    u = warp_sum(u), w = warp_sum(w);
    if (lane == 0) s.g[0][g] = u, s.g[1][g] = w;
  }
  __syncthreads();
  grads<T, kV, kOne>(a, p, s, k, walk);
}

template <typename T, int kV>
__global__ void __launch_bounds__(kThreads, 3) gn_held_back_kernel(GnArgs a) {
  extern __shared__ __align__(16) char smem[];
  Sums& s = *reinterpret_cast<Sums*>(smem);
  const Where<kV> p(a, false);
  Held<T, kV, 2> rows(a, p, smem + kPlaces, (T*)a.out);
  pdl_next();
  const Back<T, kV, true> k(a, p);
  read_mask(a, p, s);
  sums<T, kV, true>(a, p, s, k, rows, nullptr);
  if (a.runs > 1) {
    cluster_arrive();
    cluster_wait();
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.groups; g += kThreads / 32) {
      float u = 0.f, q = 0.f;
      if (lane < a.runs) u = peer(&s.g[0][g], lane), q = peer(&s.g[1][g], lane);
      u = warp_sum(u), q = warp_sum(q);
      if (lane == 0) s.a[2 * g] = u, s.a[2 * g + 1] = q;
    }
    cluster_arrive();   // (all have read)
    cluster_wait();
    for (int g = threadIdx.x; g < p.groups; g += kThreads) s.g[0][g] = s.a[2 * g], s.g[1][g] = s.a[2 * g + 1];
    __syncthreads();
  }
  grads<T, kV, true>(a, p, s, k, rows);
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
// One block per sequence and group takes the sums, value by value, an elementwise pass follows: each value is read three times.
// Taken where whole groups that are whole vectors together need more than 256 vectors of any length that the rows allow: from 257
// channels to a group on if their number is odd or rows start on odd addresses, from 2056 in 16-bit types (1028 in fp32) if it is a
// multiple of the longest vector.  Bound: that one block, whatever the device has besides (bf16 1 x 8192 x 4096, one group: 26 ms
// forward and 40 backward, in 32 groups 44 and 66 us; 4 x 4096 x 1028, 4 groups: 4.0 and 3.5 ms, 4 x 4096 x 1024 28 and 39 us).
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
  int ng, tiles, steps, runs;
  bool held;   // in one pass, the runs of a sequence a cluster
};
// Bytes of a row of a held tile at least.  A group has 16 or more of them, and a tile takes no more groups than make them up.
constexpr int kHeldRow = 64;
static_assert(kHeldRow / 16 <= kHeldGroups, "a held tile's groups have their places");

Plan plan_of(int dtype, int B, int L, int D, int G, int vec, bool bwd) {
  const int es = elem_size(dtype), size = D / G, arrays = bwd ? 2 : 1, blocks = (bwd ? 3 : 4) * 148;   // (all at once on the device)
  if (vec == 0) return {G, 1, L, 1, false};
  Plan p;
  p.held = false;
  if (vec * es == 16 && size % vec == 0) {
    // Held in one pass where eight blocks hold a sequence's steps of a tile of 64 bytes or more, and all of the call are on the device
    // at once (B = 7, L = 314, D = 768, 16 groups forward and backward 8.6 and 13.9 us, in two passes 10.6 and 17.6; in several
    // waves, which load and compute by turns, B = 32, L = 1024, D = 1024 backward 97 us against 75).
    const int places = bwd ? kHeldBack / 2 : kHeld;
    auto lanes_of = [&](int ng) { return kThreads / (ng * size / vec); };
    auto blocks_of = [&](int ng) { return (L + places * lanes_of(ng) - 1) / (places * lanes_of(ng)); };
    int ng = 1;
    while (ng < G && ng * size * es < kHeldRow) ++ng;
    if (ng * size <= kThreads * vec && blocks_of(ng) <= 8 && (long long)B * ((G + ng - 1) / ng) * blocks_of(ng) <= 3 * 148) {
      p.ng = ng, p.tiles = (G + ng - 1) / ng, p.runs = blocks_of(ng), p.held = true;
      p.steps = (L + p.runs - 1) / p.runs;
      return p;
    }
  }
  // a tile: whole groups and whole vectors, 64 bytes or more of a row where there are as many; up to 256 while runs of eight rows to a
  // thread still fill the device (B = 2, L = 32768, D = 1024, 16 groups, bf16 forward: 81 us with 128 bytes, 76 with 256, 76 with
  // 512), and further while whole sequences do, as a block's fixed part is worth some ten rows of a thread
  const int unit = vec / gcd(size, vec);
  auto tiles_of = [&](int ng) { return (G + ng - 1) / ng; };
  auto most = [&](int ng) { return (long long)B * tiles_of(ng) * std::max<long long>(1, L / (8ll * std::max(1, kThreads / (ng * size / vec)))); };
  p.ng = unit;
  while (p.ng < G && p.ng * size * es < 64) p.ng += unit;
  while (p.ng < G && 2 * p.ng * size <= kThreads * vec && 2 * p.ng <= kGroups &&
         (p.ng * size * es < 256 ? most(2 * p.ng) >= blocks : (long long)B * tiles_of(2 * p.ng) >= blocks))
    p.ng *= 2;
  while (p.ng > G) p.ng -= unit;
  if (p.ng <= 0) p.ng = G;   // (D is whole vectors: the row is)
  p.tiles = tiles_of(p.ng);
  const long long slices = (long long)B * p.tiles;
  const int lanes = std::max(1, kThreads / std::max(1, p.ng * size / vec));
  // runs: as many as fill the device once (or, where a thread's kRun rows are fewer, a whole number of times), of eight rows to a
  // thread at least
  const long long least = (L + (long long)kRun * lanes - 1) / ((long long)kRun * lanes), waves = (least * slices + blocks - 1) / blocks;
  const long long runs = std::max<long long>(least, std::min<long long>(waves * blocks / slices, L / (8ll * lanes)));
  p.steps = (int)((L + runs - 1) / runs);
  p.runs = (L + p.steps - 1) / p.steps;
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

void fill(GnArgs& a, const Plan& p, int vec) {
  a.ng = p.ng, a.tiles = p.tiles, a.steps = p.steps, a.runs = p.runs;
  if (vec == 0) return;
  a.nv = p.ng * a.size / vec, a.lanes = kThreads / a.nv;
  a.over_nv = 1.f / (float)a.nv, a.over_size = 1.f / (float)a.size, a.over_vectors = 1.f / (float)std::max(1, a.size / vec);
}

template <typename First, typename Second>
void passes(First first, Second second, const GnArgs& a, cudaStream_t s) {
  const dim3 grid(a.runs, a.tiles, a.B);
  launch(first, grid, dim3(kThreads), kPlaces + kRing, s, a);
  if (a.runs > 1) launch_after(second, grid, dim3(kThreads), kPlaces + kRing, s, a);
}
template <typename T, int kV, bool kOne>
void run_one(bool bwd, const GnArgs& a, cudaStream_t s) {
  if (bwd)
    passes(gn_sums_kernel<T, kV, kOne>, gn_grads_kernel<T, kV, kOne>, a, s);
  else
    passes(gn_first_kernel<T, kV, kOne>, gn_second_kernel<T, kV, kOne>, a, s);
}
template <typename Kernel>
void launch_held(Kernel kernel, bool bwd, const GnArgs& a, cudaStream_t s) {
  const size_t smem = bwd ? kPlaces + kHeldBack * kThreads * 16 : kFewer + kHeld * kThreads * 16;
  allow_smem(reinterpret_cast<const void*>(kernel), smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.runs, a.tiles, a.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.runs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  g_last_kernel.store("group_norm_held", std::memory_order_relaxed);
}
template <typename T, int kV>
void run_vec(bool bwd, const GnArgs& a, const Plan& p, cudaStream_t s) {
  if constexpr (kV * sizeof(T) == 16) {
    if (p.held) return launch_held(bwd ? gn_held_back_kernel<T, kV> : gn_held_kernel<T, kV>, bwd, a, s);
    if (a.size % kV == 0) return run_one<T, kV, true>(bwd, a, s);
  }
  run_one<T, kV, kV == 1>(bwd, a, s);
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

extern "C" int64_t mega_group_norm_work(int dtype, int B, int L, int D, int num_groups, int backward) {
  if (check_gn(dtype, B, L, D, num_groups, {})) return 0;
  size_t most = 0;   // (of the vectors that addresses may allow)
  for (int vec : {16 / elem_size(dtype), 4 / elem_size(dtype), 1, 0})
    most = std::max(most, work_bytes(plan_of(dtype, B, L, D, num_groups, vec, backward != 0), B, D, num_groups, backward != 0));
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
  fill(a, p, vec);
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
  fill(a, p, vec);
  a.chan = (float*)work, a.part = a.chan + (size_t)B * p.runs * 2 * D;
  MEGA_DISPATCH_DTYPE(dtype, run_gn<T>(true, vec, a, p, (cudaStream_t)stream));
  launch_after(gn_params_kernel, dim3((D + 31) / 32), dim3(1024), 0, stream, a);
  return check_launch("group_norm_bwd");
}

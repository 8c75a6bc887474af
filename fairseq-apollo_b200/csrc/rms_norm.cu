// Root-mean-square norm with a residual: r = x + residual (rounded to the activations' type), y = r rstd (1 + w) with
// rstd = 1 / sqrt(mean(r^2) + eps) over a group of channels.  Backward, with g = dy (1 + w) and the mean over the group,
//   dx = rstd (g - r rstd^2 mean(g r)) + dr        dw = sum over rows of dy r rstd
//
// Nothing but memory bounds it: x, residual, y, r once each.  A row stays in registers between its sum and its outputs, kHeld pieces of
// 16 bytes to a thread, all of them on their way at once: a warp takes a row by itself (no barrier; the pieces of several warps
// cover the memory's latency), eight warps one that a warp cannot hold.  Groups: a row's piece i of lane l holds channels of one
// group, whose lanes are a power of two side by side (their sum is a butterfly over those lanes), or rows of a group count as rows.
// Measured: forward with a residual, 8 x 4096 x 2048 bf16, 85 us or 0.96 of the copy rate; training, 16 x 4096 x 1024 bf16 with a residual,
// 192 us: forward 76, backward 104 (0.8), its shares of dw 8; 2 x 32768 x 1024 fp16 in 16 groups 143 us: the backward's two sums of eight
// lanes for each piece take as long as its memory.
// The backward adds up dw of the rows that a warp walks in registers, then over a block's warps, then over blocks, in a fixed order.
#include <algorithm>

#include "common.cuh"
#include "tma.cuh"

namespace mega {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kSms = 148;

struct Rms {
  const void *x, *res, *dy, *dr;   // backward: x is r
  void *y, *sum;                   // backward: y is dx
  long long xb, xl, rb, rl, yb, yl, sb, sl, gb, gl, hb, hl;
  const float* w;
  float* dw;                       // [blocks][D] partial sums
  long long rows;                  // B L
  int L, D, n, groups;             // n: channels of a group
  float eps, inv;                  // 1 / n
};

template <typename T>
constexpr int kVals = 16 / (int)sizeof(T);   // of a piece
template <typename T>
__device__ __forceinline__ void widen(const uint4& p, float* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(p.x), v[1] = __uint_as_float(p.y), v[2] = __uint_as_float(p.z), v[3] = __uint_as_float(p.w);
  } else {
    const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 narrow(const float* v) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(v[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void store16(void* p, const uint4& v) {
  asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Sum over the threads of a row (kRowWarps warps) or, with `lanes` < 32, over lanes side by side
template <int kRowWarps, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int lanes, float (*smem)[kWarps], int turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (o < lanes)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(~0u, v[i], o);
  if constexpr (kRowWarps > 1) {
    static_assert(kRowWarps == kWarps, "a row is a warp's or a block's");
    float(*s)[kWarps] = smem + turn * N;   // (two places in turn: one barrier a row)
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i][threadIdx.x >> 5] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v[i] += s[i][k];
    }
  }
}

// kHeld: pieces of a row to a thread.  `lanes`: 32: a row is a group; less: lanes of a group (kRowWarps == 1).
template <typename T, int kRowWarps, int kHeld, bool kRes, bool kSplit>
__global__ void __launch_bounds__(kThreads) rms_fwd_kernel(const Rms a, int lanes) {
  constexpr int kV = kVals<T>, kStep = 32 * kRowWarps;
  __shared__ float smem[2][kWarps];
  const int lane = kRowWarps == 1 ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int g0 = blockIdx.y * a.n, pieces = (kSplit ? a.D : a.n) / kV;
  const long long stride = kRowWarps == 1 ? (long long)gridDim.x * kWarps : gridDim.x;
  long long row = kRowWarps == 1 ? (long long)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  for (int turn = 0; row < a.rows; row += stride, turn ^= 1) {
    const long long b = row / a.L, l = row % a.L;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + l * a.xl + g0;
    const T* res = static_cast<const T*>(a.res) + b * a.rb + l * a.rl + g0;
    uint4 p[kHeld], q[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane + i * kStep;
      p[i] = q[i] = make_uint4(0, 0, 0, 0);
      if (at < pieces) {
        p[i] = load16(x + at * kV);
        if (kRes) q[i] = load16(res + at * kV);
      }
    }
    float ss[kSplit ? kHeld : 1];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (kSplit || i == 0) ss[kSplit ? i : 0] = 0.f;
      float v[kV], u[kV];
      widen<T>(p[i], v);
      if (kRes) {
        widen<T>(q[i], u);
#pragma unroll
        for (int j = 0; j < kV; ++j) v[j] += u[j];
        p[i] = narrow<T>(v);
        if (lane + i * kStep < pieces) store16(static_cast<T*>(a.sum) + b * a.sb + l * a.sl + g0 + (lane + i * kStep) * kV, p[i]);
        widen<T>(p[i], v);
      }
#pragma unroll
      for (int j = 0; j < kV; ++j) ss[kSplit ? i : 0] += v[j] * v[j];
    }
    row_sum<kRowWarps>(ss, lanes, smem, turn);
    T* y = static_cast<T*>(a.y) + b * a.yb + l * a.yl + g0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane + i * kStep;
      if (at >= pieces) continue;
      const float rstd = rsqrtf(ss[kSplit ? i : 0] * a.inv + a.eps);
      float v[kV];
      widen<T>(p[i], v);
#pragma unroll
      for (int j = 0; j < kV; j += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(a.w + g0 + at * kV + j));
        v[j] *= rstd * (1.f + w.x), v[j + 1] *= rstd * (1.f + w.y), v[j + 2] *= rstd * (1.f + w.z), v[j + 3] *= rstd * (1.f + w.w);
      }
      store16(y + at * kV, narrow<T>(v));
    }
  }
}

template <typename T, int kRowWarps, int kHeld, bool kRes, bool kSplit>
__global__ void __launch_bounds__(kThreads, kHeld <= 4 ? 2 : 1) rms_bwd_kernel(const Rms a, int lanes) {
  constexpr int kV = kVals<T>, kStep = 32 * kRowWarps;
  __shared__ float smem[4][kWarps];
  extern __shared__ float sums[];   // kRowWarps == 1: [kHeld * 32 * kV]
  const int lane = kRowWarps == 1 ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int g0 = blockIdx.y * a.n, pieces = (kSplit ? a.D : a.n) / kV;
  const long long stride = kRowWarps == 1 ? (long long)gridDim.x * kWarps : gridDim.x;
  long long row = kRowWarps == 1 ? (long long)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  float dw[kHeld][kV];
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
#pragma unroll
    for (int j = 0; j < kV; ++j) dw[i][j] = 0.f;
  for (int turn = 0; row < a.rows; row += stride, turn ^= 1) {
    const long long b = row / a.L, l = row % a.L;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + l * a.xl + g0;
    const T* dy = static_cast<const T*>(a.dy) + b * a.gb + l * a.gl + g0;
    const T* dr = static_cast<const T*>(a.dr) + b * a.hb + l * a.hl + g0;
    uint4 p[kHeld], q[kHeld], h[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane + i * kStep;
      p[i] = q[i] = h[i] = make_uint4(0, 0, 0, 0);
      if (at < pieces) {
        p[i] = load16(x + at * kV);
        q[i] = load16(dy + at * kV);
        if (kRes) h[i] = load16(dr + at * kV);
      }
    }
    constexpr int kSums = kSplit ? 2 * kHeld : 2;
    float s[kSums];   // sum of r^2, of g r
#pragma unroll
    for (int i = 0; i < kSums; ++i) s[i] = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      float v[kV], g[kV];
      widen<T>(p[i], v);
      widen<T>(q[i], g);
      const int at = lane + i * kStep, to = kSplit ? 2 * i : 0;
#pragma unroll
      for (int j = 0; j < kV; j += 4) {
        const float4 w = at < pieces ? __ldg(reinterpret_cast<const float4*>(a.w + g0 + at * kV + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
        s[to] += v[j] * v[j] + v[j + 1] * v[j + 1] + v[j + 2] * v[j + 2] + v[j + 3] * v[j + 3];
        s[to + 1] += (1.f + w.x) * g[j] * v[j] + (1.f + w.y) * g[j + 1] * v[j + 1] + (1.f + w.z) * g[j + 2] * v[j + 2] +
                     (1.f + w.w) * g[j + 3] * v[j + 3];
      }
    }
    row_sum<kRowWarps>(s, lanes, smem, turn);
    T* dx = static_cast<T*>(a.y) + b * a.yb + l * a.yl + g0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane + i * kStep, to = kSplit ? 2 * i : 0;
      if (at >= pieces) continue;
      const float rstd = rsqrtf(s[to] * a.inv + a.eps), along = s[to + 1] * a.inv * rstd * rstd;
      float v[kV], g[kV], u[kV];
      widen<T>(p[i], v);
      widen<T>(q[i], g);
      if (kRes) widen<T>(h[i], u);
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        dw[i][j] += g[j] * (v[j] * rstd);
      }
#pragma unroll
      for (int j = 0; j < kV; j += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(a.w + g0 + at * kV + j));
        const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j + k] = rstd * ((1.f + ww[k]) * g[j + k] - along * v[j + k]) + (kRes ? u[j + k] : 0.f);
      }
      store16(dx + at * kV, narrow<T>(v));
    }
  }
  // this block's share of dw
  float* out = a.dw + (long long)blockIdx.x * a.D + g0;
  if constexpr (kRowWarps == 1) {
    const int warp = threadIdx.x >> 5;
    for (int t = 0; t < kWarps; ++t) {   // (one warp after another: a fixed order)
      if (t == warp)
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            float* s = sums + (lane + i * 32) * kV + j;
            *s = t ? *s + dw[i][j] : dw[i][j];
          }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < pieces * kV; i += kThreads) out[i] = sums[i];
  } else {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane + i * kStep;
      if (at >= pieces) continue;
#pragma unroll
      for (int j = 0; j < kV; ++j) out[at * kV + j] = dw[i][j];
    }
  }
}

// Any width, any alignment: a warp to a (row, group), values one by one, read twice
template <typename T>
__global__ void __launch_bounds__(kThreads) rms_any_fwd_kernel(const Rms a) {
  const int lane = threadIdx.x & 31;
  const long long total = a.rows * a.groups, step = (long long)gridDim.x * kWarps;
  for (long long it = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); it < total; it += step) {
    const long long row = it / a.groups, b = row / a.L, l = row % a.L;
    const int g0 = (int)(it % a.groups) * a.n;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + l * a.xl + g0;
    T* sum = static_cast<T*>(a.sum) + b * a.sb + l * a.sl + g0;
    float ss = 0.f;
    for (int i = lane; i < a.n; i += 32) {
      float v = Elem<T>::ld(x + i);
      if (a.res) {
        T r;
        Elem<T>::st(&r, v + Elem<T>::ld(static_cast<const T*>(a.res) + b * a.rb + l * a.rl + g0 + i));
        sum[i] = r;
        v = Elem<T>::ld_shared(&r);
      }
      ss += v * v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    const float rstd = rsqrtf(ss * a.inv + a.eps);
    T* y = static_cast<T*>(a.y) + b * a.yb + l * a.yl + g0;
    for (int i = lane; i < a.n; i += 32) {
      const float v = a.res ? Elem<T>::ld_shared(sum + i) : Elem<T>::ld(x + i);   // (what this thread wrote)
      Elem<T>::st(y + i, v * rstd * (1.f + __ldg(a.w + g0 + i)));
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(kThreads) rms_any_bwd_kernel(const Rms a, float* rstds) {
  const int lane = threadIdx.x & 31;
  const long long total = a.rows * a.groups, step = (long long)gridDim.x * kWarps;
  for (long long it = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); it < total; it += step) {
    const long long row = it / a.groups, b = row / a.L, l = row % a.L;
    const int g0 = (int)(it % a.groups) * a.n;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + l * a.xl + g0;
    const T* dy = static_cast<const T*>(a.dy) + b * a.gb + l * a.gl + g0;
    float s[2] = {0.f, 0.f};
    for (int i = lane; i < a.n; i += 32) {
      const float v = Elem<T>::ld(x + i);
      s[0] += v * v;
      s[1] += v * Elem<T>::ld(dy + i) * (1.f + __ldg(a.w + g0 + i));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s[0] += __shfl_xor_sync(~0u, s[0], o), s[1] += __shfl_xor_sync(~0u, s[1], o);
    const float rstd = rsqrtf(s[0] * a.inv + a.eps), along = s[1] * a.inv * rstd * rstd;
    if (lane == 0) rstds[it] = rstd;
    T* dx = static_cast<T*>(a.y) + b * a.yb + l * a.yl + g0;
    for (int i = lane; i < a.n; i += 32) {
      const float v = Elem<T>::ld(x + i), g = Elem<T>::ld(dy + i) * (1.f + __ldg(a.w + g0 + i));
      const float h = a.dr ? Elem<T>::ld(static_cast<const T*>(a.dr) + b * a.hb + l * a.hl + g0 + i) : 0.f;
      Elem<T>::st(dx + i, rstd * (g - along * v) + h);
    }
  }
}
// dw of a block's rows: 32 channels, eight rows at a time
template <typename T>
__global__ void __launch_bounds__(kThreads) rms_any_dw_kernel(const Rms a, const float* rstds) {
  __shared__ float part[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.y * 32 + lane;
  float s = 0.f;
  if (c < a.D)
    for (long long row = (long long)blockIdx.x * kWarps + warp; row < a.rows; row += (long long)gridDim.x * kWarps) {
      const long long b = row / a.L, l = row % a.L;
      const float v = Elem<T>::ld(static_cast<const T*>(a.x) + b * a.xb + l * a.xl + c);
      s += Elem<T>::ld(static_cast<const T*>(a.dy) + b * a.gb + l * a.gl + c) * (v * rstds[row * a.groups + c / a.n]);
    }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < a.D) {
    for (int i = 1; i < kWarps; ++i) s += part[i][lane];
    a.dw[(long long)blockIdx.x * a.D + c] = s;
  }
}
// over blocks: a warp's lanes take 32 channels, its block's warps every eighth share
__global__ void __launch_bounds__(kThreads) rms_dw_kernel(const float* part, float* dw, int blocks, int D) {
  __shared__ float sh[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < D)
#pragma unroll 4
    for (int i = warp; i < blocks; i += kWarps) s += part[(long long)i * D + c];
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < D) {
    for (int i = 1; i < kWarps; ++i) s += sh[i][lane];
    dw[c] = s;
  }
}

// How a call is laid out: warps of a row, pieces a thread holds, lanes of a group, rows of a group as rows (grid's second axis);
// held == 0: the kernels for any width
struct Layout {
  int row_warps, held, lanes, groups;
  bool split;
};
Layout layout_of(int size, int D, int groups, bool back) {
  const int v = 16 / size, n = D / groups, gp = n / v;
  if (n % v || (groups > 1 && D % v)) return {0, 0, 32, 1, false};
  auto held = [&](int pieces, int per) {
    const int need = (pieces + per - 1) / per;
    return need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : 0;
  };
  const int all = D / v;
  // The backward holds three arrays and a row's share of dw: beyond four pieces to a thread that leaves a block of eight warps to a
  // multiprocessor, so there a row is a block's (2048 channels in 16 bits: one piece to a thread).
  const int most = back ? 4 : 8;
  if (groups > 1 && gp <= 32 && (gp & (gp - 1)) == 0 && all <= most * 32) return {1, held(all, 32), gp, 1, true};
  if (groups > 1 && gp < 16) return {0, 0, 32, 1, false};
  if (gp <= most * 32) return {1, held(gp, 32), 32, groups, false};
  if (gp <= 8 * kThreads) return {kWarps, held(gp, kThreads), 32, groups, false};
  return {0, 0, 32, 1, false};
}
bool rows16(const void* p, long long a, long long b, int size) { return aligned_to(p, 16) && a * size % 16 == 0 && b * size % 16 == 0; }

int fwd_blocks(const Layout& l, long long rows) {
  const long long want = l.row_warps == 1 ? (rows + kWarps - 1) / kWarps : rows;
  return (int)std::min<long long>(want, 1 << 30);
}
int bwd_blocks(long long rows, int row_warps) {
  const long long want = row_warps == kWarps ? rows : (rows + kWarps - 1) / kWarps;
  return (int)std::max<long long>(1, std::min<long long>(want, 2 * kSms));
}

template <typename T, int RW, int HELD>
void go(const Rms& a, const Layout& l, bool back, int blocks, void* stream) {
  const dim3 grid((unsigned)blocks, (unsigned)l.groups), block(kThreads);
  const size_t smem = back && RW == 1 ? (size_t)HELD * 32 * kVals<T> * sizeof(float) : 0;
#define MEGA_RMS(RES, SPLIT)                                                                       \
  if (back) launch(rms_bwd_kernel<T, RW, HELD, RES, SPLIT>, grid, block, smem, stream, a, l.lanes); \
  else launch(rms_fwd_kernel<T, RW, HELD, RES, SPLIT>, grid, block, 0, stream, a, l.lanes)
  const bool res = back ? a.dr != nullptr : a.res != nullptr;
  if constexpr (RW == 1) {
    if (l.split) {
      if (res) { MEGA_RMS(true, true); } else { MEGA_RMS(false, true); }
      return;
    }
  }
  if (res) { MEGA_RMS(true, false); } else { MEGA_RMS(false, false); }
#undef MEGA_RMS
}
template <typename T>
void dispatch(const Rms& a, const Layout& l, bool back, int blocks, void* stream) {
  if (l.row_warps == 1) {
    switch (l.held) {
      case 1: return go<T, 1, 1>(a, l, back, blocks, stream);
      case 2: return go<T, 1, 2>(a, l, back, blocks, stream);
      case 4: return go<T, 1, 4>(a, l, back, blocks, stream);
      default: return go<T, 1, 8>(a, l, back, blocks, stream);
    }
  }
  switch (l.held) {
    case 1: return go<T, kWarps, 1>(a, l, back, blocks, stream);
    case 2: return go<T, kWarps, 2>(a, l, back, blocks, stream);
    case 4: return go<T, kWarps, 4>(a, l, back, blocks, stream);
    default: return go<T, kWarps, 8>(a, l, back, blocks, stream);
  }
}
int check_shape(int dtype, int B, int L, int D, int groups) {
  if (!valid_dtype(dtype)) return MEGA_ERR_DTYPE;
  if (B <= 0 || L <= 0 || D <= 0 || groups <= 0 || D % groups) return MEGA_ERR_SHAPE;
  if (groups > 65535 || D > 1 << 20) return MEGA_ERR_UNSUPPORTED;   // (grids' second axes)
  return MEGA_OK;
}
Rms base(int B, int L, int D, int groups, const float* w, double eps) {
  Rms a = {};
  a.w = w, a.rows = (long long)B * L, a.L = L, a.D = D, a.groups = groups, a.n = D / groups, a.eps = (float)eps, a.inv = 1.f / (float)a.n;
  return a;
}
constexpr int kAnyBlocks = 4 * kSms;
}  // namespace
}  // namespace mega

using namespace mega;

extern "C" MEGA_API int64_t mega_rms_norm_work(int dtype, int B, int L, int D, int num_groups) {
  if (check_shape(dtype, B, L, D, num_groups)) return 0;
  const long long rows = (long long)B * L;
  // shares of dw, and (where a call's memory is not aligned) 1 / rms of every row
  return (int64_t)sizeof(float) * ((long long)std::max(kAnyBlocks, 2 * kSms) * D + rows * num_groups);
}

extern "C" MEGA_API int mega_rms_norm_fwd(const void* x, const void* residual, void* y, void* sum, int dtype, int B, int L, int D, int64_t xsb,
                                 int64_t xsl, int64_t rsb, int64_t rsl, int64_t ysb, int64_t ysl, int64_t ssb, int64_t ssl, const float* weight,
                                 int num_groups, double eps, mega_stream_t stream) {
  const int bad = check_shape(dtype, B, L, D, num_groups);
  if (bad) return bad;
  if (!x || !y || !weight || (residual && !sum)) return MEGA_ERR_NULL;
  const int size = elem_size(dtype);
  Rms a = base(B, L, D, num_groups, weight, eps);
  a.x = x, a.res = residual, a.y = y, a.sum = sum;
  a.xb = xsb, a.xl = xsl, a.rb = rsb, a.rl = rsl, a.yb = ysb, a.yl = ysl, a.sb = ssb, a.sl = ssl;
  const Layout l = layout_of(size, D, num_groups, false);
  const bool wide = l.held && rows16(x, xsb, xsl, size) && rows16(y, ysb, ysl, size) && aligned_to(weight, 16) &&
                    (!residual || (rows16(residual, rsb, rsl, size) && rows16(sum, ssb, ssl, size)));
  if (wide) {
    MEGA_DISPATCH_DTYPE(dtype, dispatch<T>(a, l, false, fwd_blocks(l, a.rows), stream));
  } else {
    const long long want = (a.rows * num_groups + kWarps - 1) / kWarps;
    MEGA_DISPATCH_DTYPE(dtype, launch(rms_any_fwd_kernel<T>, dim3((unsigned)std::min<long long>(want, 1 << 20)), dim3(kThreads), 0, stream, a));
  }
  return check_launch("rms_norm_fwd");
}

extern "C" MEGA_API int mega_rms_norm_bwd(const void* dy, const void* dr, const void* r, void* dx, int dtype, int B, int L, int D, int64_t gsb,
                                 int64_t gsl, int64_t rgsb, int64_t rgsl, int64_t rsb, int64_t rsl, int64_t dsb, int64_t dsl,
                                 const float* weight, int num_groups, double eps, float* dweight, void* work, mega_stream_t stream) {
  const int bad = check_shape(dtype, B, L, D, num_groups);
  if (bad) return bad;
  if (!dy || !r || !dx || !weight || !dweight || !work) return MEGA_ERR_NULL;
  if (!aligned_to(work, 16)) return MEGA_ERR_ALIGN;
  const int size = elem_size(dtype);
  Rms a = base(B, L, D, num_groups, weight, eps);
  a.x = r, a.dy = dy, a.dr = dr, a.y = dx, a.dw = static_cast<float*>(work);
  a.xb = rsb, a.xl = rsl, a.yb = dsb, a.yl = dsl, a.gb = gsb, a.gl = gsl, a.hb = rgsb, a.hl = rgsl;
  const Layout l = layout_of(size, D, num_groups, true);
  const bool wide = l.held && rows16(r, rsb, rsl, size) && rows16(dx, dsb, dsl, size) && rows16(dy, gsb, gsl, size) && aligned_to(weight, 16) &&
                    (!dr || rows16(dr, rgsb, rgsl, size));
  int blocks;
  if (wide) {
    blocks = bwd_blocks(a.rows, l.row_warps);
    MEGA_DISPATCH_DTYPE(dtype, dispatch<T>(a, l, true, blocks, stream));
  } else {
    const long long want = (a.rows * num_groups + kWarps - 1) / kWarps;
    blocks = (int)std::min<long long>(kAnyBlocks, (a.rows + kWarps - 1) / kWarps);
    float* rstds = a.dw + (long long)kAnyBlocks * D;
    MEGA_DISPATCH_DTYPE(dtype, {
      launch(rms_any_bwd_kernel<T>, dim3((unsigned)std::min<long long>(want, 1 << 20)), dim3(kThreads), 0, stream, a, rstds);
      launch(rms_any_dw_kernel<T>, dim3((unsigned)blocks, (unsigned)((D + 31) / 32)), dim3(kThreads), 0, stream, a, static_cast<const float*>(rstds));
    });
  }
  launch(rms_dw_kernel, dim3((unsigned)((D + 31) / 32)), dim3(kThreads), 0, stream, static_cast<const float*>(work), dweight, blocks, D);
  return check_launch("rms_norm_bwd");
}

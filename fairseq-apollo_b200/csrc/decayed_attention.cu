// Linear attention with a decay for each head: per sequence and head a state S (K, V) in fp32,
//   S_t = a_t S_{t-1} + k_t v_t^T      y_t = scale S_t^T q_t      a = sigmoid(f)
// in chunks of 64 steps.  With G the running sum of log2 a inside a chunk and S the state that enters it,
//   y_i = scale (2^{G_i} S^T q_i + sum_{j <= i} 2^{G_i - G_j} (q_i . k_j) v_j)
//   S'  = 2^{G_64} S + sum_j 2^{G_64 - G_j} k_j v_j^T
// which are four matrix products.  All gradients are the same walk with other operands (R: the gradient of the state):
//   dq: queries dy, keys v, values k, in the order of the forward walk;
//   dk: queries v, keys dy, values q, backwards, a step's decay taking effect behind it (`excl`);
//   dv: queries k, keys q, values dy, the same way.
// The gates' gradient is d log a_t = a_t <R_t, S_{t-1}>.  Over a chunk it is gathered from what passes t: pairs (i >= t > j) inside the
// chunk, steps i >= t that read the state which enters, steps j < t that are read behind the chunk, and what passes all of it.  With
// W_ij = (dy_i . v_j) (q_i . k_j) of a pair with its weight, summed over j by the walk of dq and over i by that of dk, the first is
// sum_{i >= t} of the one less the other (fp32 products both, unrounded: the pairs on one side of t cancel); the next two are sums of
// q_i . dq_i and k_j . dk_j of the parts that come from states, the last is the product of both states, for which the walk of dq leaves
// every chunk's state in the activations' type (fp16: with its scale).  Nothing is carried from chunk to chunk, where roundings would pile
// up, and pairs' sums are not carried past steps that let nothing through.
//
// This file: chunks of 64 steps on mma.sync, for fp32 (three products of TF32 pieces for each), heads of more than 128 keys or values, operands
// that TMA cannot address, and short calls; everything else goes to the form on tcgen05 (decayed_attention_tc.cu).  A block of four warps
// has 64 (32) values of a head; the state stays in its registers in fp32, the next chunk is on its way by cp.async.  What bounds it: the
// rate of mma.sync with few warps to a multiprocessor (8 x 4096 x 16 heads of 64 in bf16 345 us, the time to move q, k, v, y is 41;
// fp32, 4 x 2805 x 7 heads of 50 x 83, rows on 4- and 8-byte boundaries, 284 us for 13).
//
// Resets (and gates so closed that their decay is zero in fp32) are counted rather than summed: a pair with another count between
// its steps has no weight.  Padded steps keep the state and have zeros for keys and values.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "decayed_attention.cuh"
#include "tma.cuh"

namespace mega {
namespace {

constexpr int kC = 64, kWarps = 4, kThreads = 32 * kWarps;

// ---------------------------------------------------------------------------------------------- matrix products
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, const uint32_t* b, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, const uint32_t* b, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma8(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Fragments of A (16 rows) and B (8 columns) for kStep places of the contraction.  fp32 operands go in as two TF32 pieces, 11 bits
// each; of the four products the one of both small pieces (2^-22 of the value) is left out.  Their places are taken in pairs
// (2 t, 2 t + 1) where the instruction has (t, t + 4), on both sides: a sum's order is free, and the layout of results is that of A.
template <typename T>
struct Mma {
  static constexpr int kStep = 16;
  struct A {
    uint32_t r[4];
  };
  struct B {
    uint32_t r[2];
  };
  // rows m0.., places k0.. of a tile with rows of the contraction's axis
  static __device__ __forceinline__ void a_rows(A& a, const T* s, int ld, int m0, int k0, int lane) {
    ldsm4(a.r, smem_u32(s + (m0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8));
  }
  // two fragments (16 columns) of B: columns n0.. are rows of the tile
  static __device__ __forceinline__ void b_rows(B* b, const T* s, int ld, int n0, int k0, int lane) {
    uint32_t r[4];
    ldsm4(r, smem_u32(s + (n0 + (lane & 7) + (lane >> 4) * 8) * ld + k0 + ((lane >> 3) & 1) * 8));
    b[0].r[0] = r[0], b[0].r[1] = r[1], b[1].r[0] = r[2], b[1].r[1] = r[3];
  }
  // the same where the contraction's axis runs over the tile's rows
  static __device__ __forceinline__ void b_cols(B* b, const T* s, int ld, int n0, int k0, int lane) {
    uint32_t r[4];
    ldsm4t(r, smem_u32(s + (k0 + (lane & 15)) * ld + n0 + (lane >> 4) * 8));
    b[0].r[0] = r[0], b[0].r[1] = r[1], b[1].r[0] = r[2], b[1].r[1] = r[3];
  }
  static __device__ __forceinline__ void go(float* c, float*, const A& a, const B& b) { mma16(c, a.r, b.r, T()); }
  // results of 16 columns as A
  static __device__ __forceinline__ void from(A& a, const float (*c)[4]) {
    a.r[0] = pack<T>(c[0][0], c[0][1]), a.r[1] = pack<T>(c[0][2], c[0][3]);
    a.r[2] = pack<T>(c[1][0], c[1][1]), a.r[3] = pack<T>(c[1][2], c[1][3]);
  }
  // A = (w k)^T, rows m0.. of the keys, places of the steps k0..  The state is to keep fp32's places: the product w k goes in as pieces
  // of 8 bits (bf16: three, 24 bits) or 11 (fp16: two, 22; scaled by `up`).
  static constexpr int kPieces = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
  template <typename F>
  static __device__ __forceinline__ void each_weighted(const T* s, int ld, int m0, int k0, const float* w, int lane, F&& fn) {
    uint32_t r[4];
    ldsm4t(r, smem_u32(s + (k0 + (lane & 7) + (lane >> 4) * 8) * ld + m0 + ((lane >> 3) & 1) * 8));
    const int t = lane & 3;
    const float2 w0 = *reinterpret_cast<const float2*>(w + k0 + 2 * t), w1 = *reinterpret_cast<const float2*>(w + k0 + 8 + 2 * t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v = unpack<T>(r[i]);
      const float2 u = i < 2 ? w0 : w1;
      v.x *= u.x, v.y *= u.y;
      fn(i, v);
    }
  }
  // the exponent of the largest one of 16 keys and the chunk's steps
  static __device__ __forceinline__ int largest(const T* s, int ld, int m0, const float* w, int lane) {
    float most = 0.f;
#pragma unroll
    for (int k0 = 0; k0 < kC; k0 += kStep)
      each_weighted(s, ld, m0, k0, w, lane, [&](int, const float2& v) { most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y))); });
    return (int)(__reduce_max_sync(~0u, __float_as_uint(most)) >> 23);
  }
  static __device__ __forceinline__ void a_weighted(A* p, const T* s, int ld, int m0, int k0, const float* w, float up, int lane) {
    each_weighted(s, ld, m0, k0, w, lane, [&](int i, float2 v) {
      if constexpr (kScaled<T>) v.x *= up, v.y *= up;
#pragma unroll
      for (int n = 0; n < kPieces; ++n) {
        p[n].r[i] = pack<T>(v.x, v.y);
        const float2 h = unpack<T>(p[n].r[i]);
        v.x -= h.x, v.y -= h.y;
      }
    });
  }
};
__device__ __forceinline__ void tf32_split(float v, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(v - __uint_as_float(hi)) + 0x1000u;
}
template <>
struct Mma<float> {
  static constexpr int kStep = 8;
  struct A {
    uint32_t h[4], l[4];
  };
  struct B {
    uint32_t h[2], l[2];
  };
  static __device__ __forceinline__ void a_rows(A& a, const float* s, int ld, int m0, int k0, int lane) {
    const float* p = s + (m0 + (lane >> 2)) * ld + k0 + 2 * (lane & 3);
    const float2 u = *reinterpret_cast<const float2*>(p), v = *reinterpret_cast<const float2*>(p + 8 * ld);
    tf32_split(u.x, a.h[0], a.l[0]), tf32_split(v.x, a.h[1], a.l[1]);
    tf32_split(u.y, a.h[2], a.l[2]), tf32_split(v.y, a.h[3], a.l[3]);
  }
  static __device__ __forceinline__ void b_rows(B* b, const float* s, int ld, int n0, int k0, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 u = *reinterpret_cast<const float2*>(s + (n0 + 8 * i + (lane >> 2)) * ld + k0 + 2 * (lane & 3));
      tf32_split(u.x, b[i].h[0], b[i].l[0]), tf32_split(u.y, b[i].h[1], b[i].l[1]);
    }
  }
  static __device__ __forceinline__ void b_cols(B* b, const float* s, int ld, int n0, int k0, int lane) {
    const float* p = s + (k0 + 2 * (lane & 3)) * ld + n0 + (lane >> 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) tf32_split(p[8 * i], b[i].h[0], b[i].l[0]), tf32_split(p[ld + 8 * i], b[i].h[1], b[i].l[1]);
  }
  // The products with a small piece have a sum of their own, x: the accumulator is cut off at each step, at the size of what it holds
  // (4 x 2805 x 7 heads of 50 x 83: outputs 1.0e-6 from 64 bits with one sum, 3.7e-7 with two)
  static __device__ __forceinline__ void go(float* c, float* x, const A& a, const B& b) {
    mma8(x, a.l, b.h);
    mma8(x, a.h, b.l);
    mma8(c, a.h, b.h);
  }
  static __device__ __forceinline__ void from(A& a, const float (*c)[4]) {
    tf32_split(c[0][0], a.h[0], a.l[0]), tf32_split(c[0][2], a.h[1], a.l[1]);
    tf32_split(c[0][1], a.h[2], a.l[2]), tf32_split(c[0][3], a.h[3], a.l[3]);
  }
  static constexpr int kPieces = 1;   // (of 22 bits, as all operands)
  static __device__ __forceinline__ void a_weighted(A* p, const float* s, int ld, int m0, int k0, const float* w, float, int lane) {
    A& hi = *p;
    const int t = lane & 3;
    const float* f = s + (k0 + 2 * t) * ld + m0 + (lane >> 2);
    const float2 u = *reinterpret_cast<const float2*>(w + k0 + 2 * t);
    tf32_split(u.x * f[0], hi.h[0], hi.l[0]), tf32_split(u.x * f[8], hi.h[1], hi.l[1]);
    tf32_split(u.y * f[ld], hi.h[2], hi.l[2]), tf32_split(u.y * f[ld + 8], hi.h[3], hi.l[3]);
  }
};

// ------------------------------------------------------------------------------------------------------- loads
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool there) {
  const int n = there ? BYTES : 0;   // (0: zeros)
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
template <typename T, int D, int VEC>
__device__ __forceinline__ void load_pieces(T* to, const T* from, long long sl, int rows, int d, int tid) {
  constexpr int kPer = D * (int)sizeof(T) / VEC, kLd = D * (int)sizeof(T) + 16;
#pragma unroll 4
  for (int i = tid; i < kC * kPer; i += kThreads) {
    const int r = i / kPer, c = (i % kPer) * VEC;
    if (c < d * (int)sizeof(T))
      copy_async<VEC>(smem_u32(to) + r * kLd + c, reinterpret_cast<const char*>(from + (r < rows ? r : 0) * sl) + c, r < rows);
  }
}
// 64 steps of an operand, zeros behind the last one; columns from d on keep the zeros that are there
template <typename T, int D>
__device__ __forceinline__ void load_tile(T* to, const T* from, long long sl, int rows, int d, int vec, int tid) {
  if (vec == 16) load_pieces<T, D, 16>(to, from, sl, rows, d, tid);
  else if (vec == 8) load_pieces<T, D, 8>(to, from, sl, rows, d, tid);
  else if (vec == 4) load_pieces<T, D, 4>(to, from, sl, rows, d, tid);
  else {
    constexpr int kLd = D + 16 / (int)sizeof(T);
    for (int i = tid; i < kC * D; i += kThreads) {
      const int r = i / D, c = i % D;
      if (c < d) to[r * kLd + c] = r < rows ? from[r * sl + c] : T(0.f);
    }
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// What a chunk's gates come to, by rows of the tile
struct Gates {
  float hi[kC], lo[kC];   // running sum of log2 a, in two pieces
  float weight[kC];       // of a step in the state that leaves
  int count[kC];          // resets so far
  uint8_t pad[kC];
  float enter;            // weight of the state that enters in the one that leaves (0: a reset lies between)
  int padded;
};
__device__ __forceinline__ void gates_put(const Walk& w, Gates& o, const GateIn<2>& in, int lane) {
  const GateOut<2> r = gates_scan<2>(w, in, lane);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = gate_row<2>(w, lane, i);
    o.hi[row] = gate_sum(r.sum[i]);   // (finite)
    o.lo[row] = gate_sum(r.sum[i] - (long long)(o.hi[row] * 0x1p40f));
    o.hi[row] += r.bad;
    o.count[row] = r.count[i];
    o.weight[row] = r.weight[i];
    o.pad[row] = in.pad >> i & 1;
  }
  if (lane == 0) o.enter = r.enter, o.padded = r.padded;
}

// A second sum beside `c` (fp32: see Mma<float>::go), which is added to it at the end; 16-bit types have none
template <typename T, int N>
struct Beside {
  float x[sizeof(T) == 4 ? N : 1][4];
  __device__ __forceinline__ Beside() {
#pragma unroll
    for (int n = 0; n < (sizeof(T) == 4 ? N : 1); ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][i] = 0.f;
  }
  __device__ __forceinline__ float* of(int n) { return x[sizeof(T) == 4 ? n : 0]; }
  __device__ __forceinline__ void join(float (*c)[4]) {
    if constexpr (sizeof(T) == 4)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] += x[n][i];
  }
};

template <typename T, int KD, int VT, int STAGES, bool kX>
struct Shared {
  static constexpr int kLk = KD + 16 / (int)sizeof(T), kLv = VT + 16 / (int)sizeof(T);
  T q[STAGES][kC * kLk], k[STAGES][kC * kLk], v[STAGES][kC * kLv];
  T s[KD * kLv];
  T x[kX ? kC * kLv : 8];
  Gates g[2];
  float sums[kWarps], tops[kWarps];
};

// A state's value in the products: rounded to their type (the state itself stays in fp32 registers; of the three roundings on the way
// to an output it is the one of the share that comes from before the chunk)
template <typename T, int VT>
__device__ __forceinline__ void state_to_shared(T* s, int ld, int row0, const float (*acc)[4], float up, int lane) {
#pragma unroll
  for (int n = 0; n < VT / 8; ++n)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      T* p = s + (row0 + (lane >> 2) + 8 * hf) * ld + n * 8 + 2 * (lane & 3);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(acc[n][2 * hf], acc[n][2 * hf + 1]);
      else if constexpr (kScaled<T>) *reinterpret_cast<uint32_t*>(p) = pack<T>(up * acc[n][2 * hf], up * acc[n][2 * hf + 1]);
      else *reinterpret_cast<uint32_t*>(p) = pack<T>(acc[n][2 * hf], acc[n][2 * hf + 1]);
    }
}

// kOut: outputs; else the state that a segment leaves by itself.  kDots: sums for the gates' gradient.
template <typename T, int KD, int VT, int STAGES, bool kOut, int kDots>
__global__ void __launch_bounds__(kThreads) walk_kernel(const Walk w) {
  using M = Mma<T>;
  using S = Shared<T, KD, VT, STAGES, kDots != 0>;
  extern __shared__ __align__(16) unsigned char raw[];
  S& sh = *reinterpret_cast<S*>(raw);
  constexpr int kLk = S::kLk, kLv = S::kLv, kN = VT / 8, kRows = KD / kWarps, kM = (kRows + 15) / 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int tile = blockIdx.x % w.tiles, bh = (blockIdx.x / w.tiles) % (w.B * w.H), seg = blockIdx.x / w.tiles / (w.B * w.H);
  const int b = bh / w.H, h = bh % w.H;
  const int from = seg * w.per, to = min(from + w.per, w.chunks);   // chunks, in the order of the walk
  const int dv = min(VT, w.v.d - tile * VT);
  const T* qp = static_cast<const T*>(w.q.p) + b * w.q.sb + h * w.q.sh;
  const T* kp = static_cast<const T*>(w.k.p) + b * w.k.sb + h * w.k.sh;
  const T* vp = static_cast<const T*>(w.v.p) + b * w.v.sb + h * w.v.sh + tile * VT;

  for (int i = tid; i < (int)(sizeof(S) / 16); i += kThreads) reinterpret_cast<uint4*>(raw)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();

  // rows of the state that this warp holds: with fewer than 64 keys two warps have none
  const bool holds = warp * 16 * kM < KD;
  float st[kM][kN][4];
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) st[m][n][i] = 0.f;
  auto each_state = [&](auto&& fn) {
    if (!holds) return;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (warp * kM + m) * 16 + g + 8 * (i >> 1), c = n * 8 + 2 * t4 + (i & 1);
          if (r < w.k.d && c < dv) fn(st[m][n][i], r, c);
        }
  };
  const long long s_at = (long long)bh * w.k.d * w.v.d + (long long)tile * VT * w.s_col;
  auto slot = [&](long long n) { return n * w.k.d * VT; };   // states of (segment or group, head, tile): rows of VT values
  if (kOut) {
    if (w.s_in) each_state([&](float& v, int r, int c) { v = w.s_in[s_at + (long long)r * w.s_row + (long long)c * w.s_col]; });
    for (int p = 0; p < seg; ++p) {
      const float fac = w.factor[(long long)p * w.B * w.H + bh];
      const float* l = w.local + slot(((long long)p * w.B * w.H + bh) * w.tiles + tile);
      each_state([&](float& v, int r, int c) { v = (fac == 0.f ? 0.f : fac * v) + l[r * VT + c]; });
    }
  }
  int scale = 0;   // fp16: of the state in shared memory, a power of two
  // the state that enters the next chunk, where all that it is multiplied with finds it
  auto state_out = [&]() {
    if constexpr (kScaled<T>) {
      float top = 0.f;
      if (holds)
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(st[m][n][i]));
      const unsigned bits = __reduce_max_sync(~0u, __float_as_uint(top));
      if (lane == 0) sh.tops[warp] = __uint_as_float(bits);
      __syncthreads();
      unsigned most = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) most = max(most, __float_as_uint(sh.tops[i]));
      scale = scale_of((int)(most >> 23));
    }
    if (holds)
#pragma unroll
      for (int m = 0; m < kM; ++m) state_to_shared<T, VT>(sh.s, kLv, (warp * kM + m) * 16, st[m], two_to(scale), lane);
  };
  if (kOut) state_out();
  float decay = 1.f;   // of the segment so far

  auto tile_of = [&](int c) { return w.rev ? w.chunks - 1 - c : c; };
  auto fetch = [&](int c, int stage) {
    const long long t0 = (long long)tile_of(c) * kC;
    const int rows = (int)min((long long)kC, w.L - t0);
    if (kOut) load_tile<T, KD>(sh.q[stage], qp + t0 * w.q.sl, w.q.sl, rows, w.q.d, w.q.vec, tid);
    load_tile<T, KD>(sh.k[stage], kp + t0 * w.k.sl, w.k.sl, rows, w.k.d, w.k.vec, tid);
    load_tile<T, VT>(sh.v[stage], vp + t0 * w.v.sl, w.v.sl, rows, dv, w.v.vec, tid);
    copies_commit();
  };
  auto fetch_x = [&](int c) {   // (one place: asked for where the last one has been used)
    const long long t0 = (long long)tile_of(c) * kC;
    load_tile<T, VT>(sh.x, static_cast<const T*>(w.x.p) + b * w.x.sb + h * w.x.sh + tile * VT + t0 * w.x.sl, w.x.sl, (int)min((long long)kC, w.L - t0),
                     dv, w.x.vec, tid);
    copies_commit();
  };
  if (kDots) fetch_x(from);
  fetch(from, 0);
  if (warp == 0) gates_put(w, sh.g[from & 1], gates_fetch<T, 2>(w, b, h, tile_of(from), lane), lane);

  for (int c = from; c < to; ++c) {
    const int stage = STAGES == 2 ? (c - from) & 1 : 0;
    const long long t0 = (long long)tile_of(c) * kC;
    const Gates& gt = sh.g[c & 1];
    copies_wait();
    __syncthreads();
    T *qs = sh.q[stage], *ks = sh.k[stage], *vs = sh.v[stage];
    if (gt.padded) {   // (whatever lies at padded steps)
      for (int i = tid; i < kC * KD; i += kThreads)
        if (gt.pad[i / KD]) ks[(i / KD) * kLk + i % KD] = T(0.f);
      for (int i = tid; i < kC * VT; i += kThreads)
        if (gt.pad[i / VT]) {
          vs[(i / VT) * kLv + i % VT] = T(0.f);
          if (kDots) sh.x[(i / VT) * kLv + i % VT] = T(0.f);
        }
      __syncthreads();
    }
    GateIn<2> next;
    if (STAGES == 2 && c + 1 < to) fetch(c + 1, stage ^ 1);
    if (warp == 0 && c + 1 < to) next = gates_fetch<T, 2>(w, b, h, tile_of(c + 1), lane);

    if constexpr (kOut) {
      // ---- the state that enters: written by the walk of dq, and multiplied with the gradient of the one that leaves by that of dk
      if (kDots && gt.enter > (kDots == 1 ? 0.f : kLeast)) {
        T* a = static_cast<T*>(w.anchors) + slot(((long long)bh * w.chunks + tile_of(c)) * w.tiles + tile);
        if (kDots == 1) each_state([&](float& v, int r, int cc) { Elem<T>::st(a + r * VT + cc, kScaled<T> ? two_to(scale) * v : v); });
        else {
          float sum = 0.f;
          each_state([&](float& v, int r, int cc) { sum += v * Elem<T>::ld(a + r * VT + cc); });
#pragma unroll
          for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
          if (lane == 0) sh.sums[warp] = sum;
        }
      }
      // ---- queries times state, queries times keys
      float o[kN][4], p[kC / 8][4];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
#pragma unroll
      for (int n = 0; n < kC / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[n][i] = 0.f;
      constexpr bool kApart = sizeof(T) == 4;   // (fp32: one after the other, as each has a second sum)
      {
        Beside<T, kN> small;
#pragma unroll 4
        for (int k0 = 0; k0 < KD; k0 += M::kStep) {
          typename M::A a;
          typename M::B bb[2];
          M::a_rows(a, qs, kLk, warp * 16, k0, lane);
#pragma unroll
          for (int n = 0; n < kN; n += 2) {
            M::b_cols(bb, sh.s, kLv, n * 8, k0, lane);
            M::go(o[n], small.of(n), a, bb[0]);
            M::go(o[n + 1], small.of(n + 1), a, bb[1]);
          }
          if constexpr (!kApart)
#pragma unroll
            for (int n = 0; n < kC / 8; n += 2)
              if (w.rev ? n / 2 >= warp : n / 2 <= warp) {
                M::b_rows(bb, ks, kLk, n * 8, k0, lane);
                M::go(p[n], nullptr, a, bb[0]);
                M::go(p[n + 1], nullptr, a, bb[1]);
              }
        }
        small.join(o);
      }
      if constexpr (kApart) {
        Beside<T, kC / 8> small;
#pragma unroll 2
        for (int k0 = 0; k0 < KD; k0 += M::kStep) {
          typename M::A a;
          typename M::B bb[2];
          M::a_rows(a, qs, kLk, warp * 16, k0, lane);
#pragma unroll
          for (int n = 0; n < kC / 8; n += 2)
            if (w.rev ? n / 2 >= warp : n / 2 <= warp) {
              M::b_rows(bb, ks, kLk, n * 8, k0, lane);
              M::go(p[n], small.of(n), a, bb[0]);
              M::go(p[n + 1], small.of(n + 1), a, bb[1]);
            }
        }
        small.join(p);
      }
      const int i0 = warp * 16 + g, i1 = i0 + 8;
      const float h0 = gt.hi[i0], h1 = gt.hi[i1], l0 = gt.lo[i0], l1 = gt.lo[i1];
      // (a padded step has no pairs and reads no state: -1 resets)
      const int c0 = gt.pad[i0] ? -1 : gt.count[i0], c1 = gt.pad[i1] ? -1 : gt.count[i1];
      const float unit = kScaled<T> ? two_to(-scale) : 1.f, e0 = w.o_scale * exp2f(h0) * unit, e1 = w.o_scale * exp2f(h1) * unit;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        o[n][0] = c0 ? 0.f : e0 * o[n][0], o[n][1] = c0 ? 0.f : e0 * o[n][1];
        o[n][2] = c1 ? 0.f : e1 * o[n][2], o[n][3] = c1 ? 0.f : e1 * o[n][3];
      }
      // ---- weights of the pairs
#pragma unroll
      for (int n = 0; n < kC / 8; ++n)
        if (w.rev ? n / 2 >= warp : n / 2 <= warp) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = n * 8 + 2 * t4 + (i & 1), r = i < 2 ? i0 : i1;
            const float d = (i < 2 ? h0 : h1) - gt.hi[j] + ((i < 2 ? l0 : l1) - gt.lo[j]);   // (sums of some thousands lie behind closed gates)
            const bool on = (w.rev ? j >= r : j <= r) && gt.count[j] == (i < 2 ? c0 : c1);
            p[n][i] = on ? p[n][i] * (w.p_scale * exp2f(fminf(d, 0.f))) : 0.f;
          }
        }
      if (kDots) {
        // x . out of the part from the state; the pairs' sums: W = (weighted pair) (x . value), the step by itself left out
        float dot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            dot[0] += o[n][i] * Elem<T>::ld_shared(sh.x + i0 * kLv + n * 8 + 2 * t4 + i);
            dot[1] += o[n][2 + i] * Elem<T>::ld_shared(sh.x + i1 * kLv + n * 8 + 2 * t4 + i);
          }
#pragma unroll
        for (int n = 0; n < kC / 8; n += 2)
          if (w.rev ? n / 2 >= warp : n / 2 <= warp) {
            float p2[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p2[0][i] = p2[1][i] = 0.f;
            Beside<T, 2> small;
#pragma unroll 2
            for (int k0 = 0; k0 < VT; k0 += M::kStep) {
              typename M::A a;
              typename M::B bb[2];
              M::a_rows(a, sh.x, kLv, warp * 16, k0, lane);
              M::b_rows(bb, vs, kLv, n * 8, k0, lane);
              M::go(p2[0], small.of(0), a, bb[0]);
              M::go(p2[1], small.of(1), a, bb[1]);
            }
            small.join(p2);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = (n + m) * 8 + 2 * t4 + (i & 1);
                if (j != (i < 2 ? i0 : i1)) dot[2 + (i >> 1)] += p[n + m][i] == 0.f ? 0.f : p[n + m][i] * p2[m][i];
              }
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dot[i] += __shfl_xor_sync(~0u, dot[i], 1);
          dot[i] += __shfl_xor_sync(~0u, dot[i], 2);
        }
        float2* d = w.dots + ((long long)tile * w.B * w.H + bh) * w.L + t0;
        if (t4 == 0 && t0 + i0 < w.L) d[i0] = make_float2(dot[0], dot[2]);
        if (t4 == 0 && t0 + i1 < w.L) d[i1] = make_float2(dot[1], dot[3]);
      }
      // fp16: a power of two for a row's pairs, which its outputs have until they are done
      float back0 = 1.f, back1 = 1.f;
      if constexpr (kScaled<T>) {
        float top0 = 0.f, top1 = 0.f;
#pragma unroll
        for (int n = 0; n < kC / 8; ++n)
          if (w.rev ? n / 2 >= warp : n / 2 <= warp)
            top0 = fmaxf(top0, fmaxf(fabsf(p[n][0]), fabsf(p[n][1]))), top1 = fmaxf(top1, fmaxf(fabsf(p[n][2]), fabsf(p[n][3])));
#pragma unroll
        for (int i = 1; i <= 2; i <<= 1) top0 = fmaxf(top0, __shfl_xor_sync(~0u, top0, i)), top1 = fmaxf(top1, __shfl_xor_sync(~0u, top1, i));
        // (at most 2^60: the share of the state is in the same sum)
        const int up0 = min(scale_of(__float_as_int(top0) >> 23), 60), up1 = min(scale_of(__float_as_int(top1) >> 23), 60);
        const float f0 = two_to(up0), f1 = two_to(up1);
        back0 = two_to(-up0), back1 = two_to(-up1);
#pragma unroll
        for (int n = 0; n < kC / 8; ++n)
          if (w.rev ? n / 2 >= warp : n / 2 <= warp) p[n][0] *= f0, p[n][1] *= f0, p[n][2] *= f1, p[n][3] *= f1;
#pragma unroll
        for (int n = 0; n < kN; ++n) o[n][0] *= f0, o[n][1] *= f0, o[n][2] *= f1, o[n][3] *= f1;
      }
      // ---- weighted pairs times values
      Beside<T, kN> small;
#pragma unroll
      for (int k0 = 0; k0 < kC; k0 += M::kStep)
        if (w.rev ? k0 / 16 >= warp : k0 / 16 <= warp) {
          typename M::A a;
          typename M::B bb[2];
          M::from(a, p + k0 / 8);
#pragma unroll
          for (int n = 0; n < kN; n += 2) {
            M::b_cols(bb, vs, kLv, n * 8, k0, lane);
            M::go(o[n], small.of(n), a, bb[0]);
            M::go(o[n + 1], small.of(n + 1), a, bb[1]);
          }
        }
      small.join(o);
      // ---- outputs
      T* op = static_cast<T*>(w.out) + b * w.ob + h * w.oh + tile * VT;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = hf ? i1 : i0;
        if (t0 + r >= w.L) continue;
        T* row = op + (t0 + r) * w.ol;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const int cc = n * 8 + 2 * t4;
          const float back = hf ? back1 : back0, u = kScaled<T> ? back * o[n][2 * hf] : o[n][2 * hf],
                      v = kScaled<T> ? back * o[n][2 * hf + 1] : o[n][2 * hf + 1];
          if (w.piece >= 2 * (int)sizeof(T)) {
            if (cc < dv) {
              if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(row + cc) = make_float2(u, v);
              else *reinterpret_cast<uint32_t*>(row + cc) = pack<T>(u, v);
            }
          } else {
            if (cc < dv) Elem<T>::st(row + cc, u);
            if (cc + 1 < dv) Elem<T>::st(row + cc + 1, v);
          }
        }
      }
      __syncthreads();   // (the state in shared memory, and x, have been read)
      if (kDots && c + 1 < to) fetch_x(c + 1);
      if (kDots && tid == 0) {
        const long long at = ((long long)bh * w.chunks + tile_of(c)) * w.tiles + tile;
        if (kScaled<T> && kDots == 1) w.units[at] = unit;
        if (kDots == 2) {
          float sum = 0.f;
          for (int i = 0; i < kWarps; ++i) sum += sh.sums[i];
          if (kScaled<T> && gt.enter > kLeast) sum *= w.units[at];
          w.through[at] = gt.enter > kLeast ? gt.enter * sum : 0.f;
        }
      }
    }

    // ---- the state that leaves
    decay *= gt.enter;
    if (holds) {
      const float e = gt.enter;
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        // (a chunk's own sum first: the accumulator of the products is cut off, not rounded, which over a long sequence adds up)
        float add[kN][4];
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) add[n][i] = 0.f;
        Beside<T, kN> small;
        int up = 0;
        if constexpr (kScaled<T>) up = scale_of(M::largest(ks, kLk, (warp * kM + m) * 16, gt.weight, lane));
#pragma unroll
        for (int k0 = 0; k0 < kC; k0 += M::kStep) {
          typename M::A a[M::kPieces];
          typename M::B bb[2];
          M::a_weighted(a, ks, kLk, (warp * kM + m) * 16, k0, gt.weight, two_to(up), lane);
#pragma unroll
          for (int n = 0; n < kN; n += 2) {
            M::b_cols(bb, vs, kLv, n * 8, k0, lane);
#pragma unroll
            for (int p = M::kPieces - 1; p >= 0; --p) {   // (small ones first)
              M::go(add[n], small.of(n), a[p], bb[0]);
              M::go(add[n + 1], small.of(n + 1), a[p], bb[1]);
            }
          }
        }
        small.join(add);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[m][n][i] = (e == 0.f ? 0.f : e * st[m][n][i]) + (kScaled<T> ? two_to(-up) : 1.f) * add[n][i];
        if (kOut && !kScaled<T>) state_to_shared<T, VT>(sh.s, kLv, (warp * kM + m) * 16, st[m], 1.f, lane);
      }
    }
    if constexpr (kOut && kScaled<T>) state_out();
    if (STAGES == 1 && c + 1 < to) {
      __syncthreads();
      fetch(c + 1, 0);
    }
    if (warp == 0 && c + 1 < to) gates_put(w, sh.g[(c + 1) & 1], next, lane);
  }
  if (!kOut) {
    float* l = w.local + slot(((long long)seg * w.B * w.H + bh) * w.tiles + tile);
    each_state([&](float& v, int r, int c) { l[r * VT + c] = v; });
    if (tid == 0 && tile == 0) w.factor[(long long)seg * w.B * w.H + bh] = decay;
  } else if (w.s_out && to == w.chunks) {
    each_state([&](float& v, int r, int c) { w.s_out[s_at + (long long)r * w.s_row + (long long)c * w.s_col] = v; });
  }
}

// ------------------------------------------------------------------------------------------ the gates' gradient
struct GateGrad {
  Walk w;                     // of the forward walk
  const float2 *dq, *dk;      // [tile][B H][L] (part from the state that entered, pairs)
  const float* through;       // [B H][chunk][part]
  int dq_tiles, dk_tiles, parts;
  void* df;
  long long db, dl, dh;
};
// a warp to a chunk of 32 N steps of a head
template <typename T, int N>
__global__ void __launch_bounds__(128) gate_grad_kernel(const GateGrad a) {
  const Walk& w = a.w;
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), bhs = (long long)w.B * w.H;
  if (at >= bhs * w.chunks) return;
  const long long bh = at / w.chunks;
  const int tile = (int)(at % w.chunks), b = (int)(bh / w.H), h = (int)(bh % w.H);
  const GateIn<N> in = gates_fetch<T, N>(w, b, h, tile, lane);
  float through = 0.f;
  for (int i = 0; i < a.parts; ++i) through += a.through[at * a.parts + i];
  // Pairs that end at a step less those that begin at it, reads of the state that entered, what a step leaves behind the chunk.  The first is
  // summed up between steps that let nothing through (resets, and decays below fp32's resolution, 2^-24): pairs on one side of
  // such a step cancel but for roundings, beside which the gradient of a closed gate is next to nothing.
  float pairs[N], reads[N], kept[N], behind = 0.f, before = 0.f, within = 0.f;
  bool cut[N], open = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    pairs[i] = reads[i] = kept[i] = 0.f;
    cut[i] = (in.reset >> i & 1) || (!(in.pad >> i & 1) && log2_gate(in.f[i]) < -24.f);
    const long long t = (long long)tile * (32 * N) + gate_row<N>(w, lane, i);
    if (t >= w.L) continue;
    for (int k = 0; k < a.dq_tiles; ++k) {
      const float2 u = a.dq[(k * bhs + bh) * w.L + t];
      reads[i] += u.x, pairs[i] += u.y;
    }
    for (int k = 0; k < a.dk_tiles; ++k) {
      const float2 u = a.dk[(k * bhs + bh) * w.L + t];
      kept[i] += u.x, pairs[i] -= u.y;
    }
    behind += reads[i], before += kept[i];
  }
#pragma unroll
  for (int i = N - 1; i >= 0; --i) {   // (of the pairs, what reaches the step before this lane's, and whether what is behind them does)
    within += pairs[i];
    if (cut[i]) within = 0.f, open = false;
  }
  float suffix = behind, prefix = before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float u = __shfl_down_sync(~0u, suffix, o), v = __shfl_up_sync(~0u, prefix, o), x = __shfl_down_sync(~0u, within, o);
    const bool y = __shfl_down_sync(~0u, (int)open, o);
    if (lane + o < 32) {
      suffix += u;
      if (open) within += x;
      open = open && y;
    }
    if (lane >= o) prefix += v;
  }
  suffix = __shfl_down_sync(~0u, suffix, 1), prefix = __shfl_up_sync(~0u, prefix, 1);   // (of the lanes behind, before)
  within = __shfl_down_sync(~0u, within, 1);
  if (lane == 31) suffix = within = 0.f;
  if (lane == 0) prefix = 0.f;
#pragma unroll
  for (int i = N - 1; i >= 0; --i) {
    within += pairs[i];
    if (cut[i]) within = 0.f;
    float da = suffix + prefix + through + within;
#pragma unroll
    for (int j = 0; j < N; ++j) da += j >= i ? reads[j] : kept[j];
    const long long t = (long long)tile * (32 * N) + gate_row<N>(w, lane, i);
    if (t >= w.L) continue;
    // log sigmoid(f)' = sigmoid(-f)
    const float v = (in.pad >> i & 1) || (in.reset >> i & 1) || closed(log2_gate(in.f[i])) ? 0.f : da * gate_of<float>(in.f[i]).c;
    const long long to = b * a.db + t * a.dl + h * a.dh;
    if (w.f_dtype == MEGA_F32) static_cast<float*>(a.df)[to] = v;
    else Elem<T>::st(static_cast<T*>(a.df) + to, v);
  }
}
}  // namespace

// ------------------------------------------------------------------------------------------------------- host
namespace {
int vec_of(const void* p, long long sb, long long sl, long long sh, int d, int size, int most) {
  for (int v = most; v > size; v >>= 1) {
    auto fits = [&](long long n) { return n * size % v == 0; };
    if (aligned_to(p, v) && fits(sb) && fits(sl) && fits(sh) && fits(d)) return v;
  }
  return size;
}
// (of an axis with one place the stride is not used)
Operand operand(const mega_decayed_attention_args& a, const void* p, const int64_t* s, int d) {
  Operand o = {p, a.B > 1 ? s[0] : 0, a.L > 1 ? s[1] : 0, a.H > 1 ? s[2] : 0, d, 0};
  o.vec = vec_of(p, o.sb, o.sl, o.sh, d, elem_size(a.dtype), 16);
  return o;
}

int key_tile(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }
int value_tile(int keys) { return key_tile(keys) == 256 ? 32 : 64; }

// How a walk is cut: into tiles of values, and, where (sequence, head, tile)s do not fill the device, the time axis into segments,
// whose states are found first at the price of a second pass over keys and values.
struct Plan {
  bool tc;
  int tiles, chunks, per, segs;
  size_t local, factor, gates, anchors, units, through;   // floats
};
Plan plan_of(bool tc, int dtype, int B, int L, int H, int keys, int values) {
  Plan p;
  p.tc = tc;
  const int c = tc ? kTcChunk : kC, vt = tc ? (values <= 64 ? 64 : 128) : value_tile(keys);
  const long long places = tc ? 148 : 2 * 148;
  p.chunks = (L - 1) / c + 1;   // (L may be the largest there is)
  p.tiles = (values + vt - 1) / vt;
  const long long blocks = (long long)B * H * p.tiles;
  p.per = p.chunks;
  if (blocks * 2 <= places && p.chunks > 1) {
    const long long want = places / blocks;
    p.per = (int)std::max<long long>(1, (p.chunks + want - 1) / want);
  }
  p.segs = (p.chunks + p.per - 1) / p.per;
  const size_t n = (size_t)(p.segs - 1) * B * H, bh = (size_t)B * H;
  auto even = [](size_t n) { return (n + 3) / 4 * 4; };
  p.local = even(n * p.tiles * keys * vt);
  p.factor = even(n);
  p.gates = tc ? bh * p.chunks * (kTcGates / 4) : 0;
  p.anchors = even(bh * p.chunks * p.tiles * keys * vt * elem_size(dtype) / 4 + 1);
  p.units = dtype == MEGA_F16 ? even(bh * p.chunks * p.tiles) : 0;
  p.through = even(bh * p.chunks * std::max(p.tiles, kTcParts));
  return p;
}
bool tc_heads(const mega_decayed_attention_args& a) { return a.dtype != MEGA_F32 && a.K <= kTcMost && a.V <= kTcMost; }

template <typename T, int KD, int VT, int STAGES>
void run_walk(const Walk& w, int dots, void* stream) {
  const long long blocks = (long long)w.tiles * w.B * w.H;
  const size_t plain = sizeof(Shared<T, KD, VT, STAGES, false>), more = sizeof(Shared<T, KD, VT, STAGES, true>);
  if (w.segs > 1) launch(walk_kernel<T, KD, VT, STAGES, false, 0>, dim3((unsigned)(blocks * (w.segs - 1))), dim3(kThreads), plain, stream, w);
  const dim3 grid((unsigned)(blocks * w.segs));
  if (dots == 0) launch(walk_kernel<T, KD, VT, STAGES, true, 0>, grid, dim3(kThreads), plain, stream, w);
  else if (dots == 1) launch(walk_kernel<T, KD, VT, STAGES, true, 1>, grid, dim3(kThreads), more, stream, w);
  else launch(walk_kernel<T, KD, VT, STAGES, true, 2>, grid, dim3(kThreads), more, stream, w);
}
template <typename T>
void run_keys(const Walk& w, int dots, void* stream) {
  switch (key_tile(w.k.d)) {
    case 32: return run_walk<T, 32, 64, 2>(w, dots, stream);
    case 64: return run_walk<T, 64, 64, sizeof(T) == 4 ? 1 : 2>(w, dots, stream);   // (fp32: one place, three blocks to a multiprocessor: 284 us for 381)
    case 128: return run_walk<T, 128, 64, 2>(w, dots, stream);
    default: return run_walk<T, 256, 32, sizeof(T) == 4 ? 1 : 2>(w, dots, stream);
  }
}
// `work`: the plan's local states, factors and gates
int run(int dtype, Walk& w, const Plan& p, int dots, float* work, void* stream) {
  w.tiles = p.tiles, w.per = p.per, w.segs = p.segs, w.chunks = p.chunks;
  if ((long long)p.tiles * w.B * w.H * p.segs > 0x7fffffffLL) return MEGA_ERR_UNSUPPORTED;
  w.gates = work, w.local = work + p.gates, w.factor = w.local + p.local;
  if (p.tc) return tc_walk(dtype, w, dots, stream);
  MEGA_DISPATCH_DTYPE(dtype, run_keys<T>(w, dots, stream));
  return MEGA_OK;
}

int check_args(const mega_decayed_attention_args* a) {
  if (!a) return MEGA_ERR_NULL;
  if (!valid_dtype(a->dtype) || !valid_dtype(a->gate_dtype)) return MEGA_ERR_DTYPE;
  if (a->gate_dtype != MEGA_F32 && a->gate_dtype != a->dtype) return MEGA_ERR_DTYPE;
  if (a->B <= 0 || a->L <= 0 || a->H <= 0 || a->K <= 0 || a->V <= 0) return MEGA_ERR_SHAPE;
  if (a->K > MEGA_ATT_MOST || a->V > MEGA_ATT_MOST || (long long)a->B * a->H > 0x7fffffffLL / 8) return MEGA_ERR_UNSUPPORTED;
  if (!a->q || !a->k || !a->v || !a->f) return MEGA_ERR_NULL;
  const size_t size = elem_size(a->dtype);
  for (const void* p : {a->q, a->k, a->v, (const void*)a->y, a->dy, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
    if (!aligned_to(p, size)) return MEGA_ERR_ALIGN;
  if (!aligned_to(a->f, elem_size(a->gate_dtype)) || !aligned_to(a->df, elem_size(a->gate_dtype))) return MEGA_ERR_ALIGN;
  for (const float* p : {a->h_in, (const float*)a->h_out, a->dh_out, (const float*)a->dh_in})
    if (!aligned_to(p, 4)) return MEGA_ERR_ALIGN;
  const size_t state = (size_t)a->B * a->H * a->K * a->V;
  if (overlap(a->h_in, a->h_out, state) || overlap(a->dh_out, a->dh_in, state)) return MEGA_ERR_UNSUPPORTED;
  return MEGA_OK;
}
void put_out(Walk& w, const mega_decayed_attention_args& a, void* p, const int64_t* s) {
  w.out = p, w.ob = s[0], w.ol = s[1], w.oh = s[2];
  w.piece = vec_of(p, a.B > 1 ? s[0] : 0, a.L > 1 ? s[1] : 0, a.H > 1 ? s[2] : 0, w.v.d, elem_size(a.dtype), 32);
}
Walk base(const mega_decayed_attention_args& a) {
  Walk w = {};
  w.f = a.f, w.fb = a.fs[0], w.fl = a.fs[1], w.fh = a.fs[2], w.f_dtype = a.gate_dtype;
  w.pad = a.pad_mask, w.reset = a.reset_mask;
  w.B = a.B, w.L = a.L, w.H = a.H;
  return w;
}
struct BackPlan {
  Plan dq, dk, dv;
  size_t walk, dots, all;   // floats
};
BackPlan back_plan(const mega_decayed_attention_args& a, bool tc) {
  BackPlan p;
  p.dq = p.dk = plan_of(tc, a.dtype, a.B, a.L, a.H, a.V, a.K);
  p.dv = plan_of(tc, a.dtype, a.B, a.L, a.H, a.K, a.V);
  p.walk = std::max(p.dq.local + p.dq.factor, p.dv.local + p.dv.factor) + p.dq.gates;
  p.dots = ((size_t)a.B * a.H * (tc ? kTcDots : p.dq.tiles) * a.L * 2 + 3) / 4 * 4;
  p.all = p.walk + 2 * p.dots + p.dq.anchors + p.dq.units + p.dq.through;
  return p;
}
// (whether the tensor memory's form takes a call depends on its memory too: room for either)
size_t forward_floats(const mega_decayed_attention_args& a, bool tc) {
  const Plan p = plan_of(tc, a.dtype, a.B, a.L, a.H, a.K, a.V);
  return p.local + p.factor + p.gates;
}
}  // namespace
cudaError_t decayed_attention_read_device_error(int* v, bool reset) { return tc_read_device_error(v, reset); }
}  // namespace mega

using namespace mega;

extern "C" MEGA_API int64_t mega_decayed_attention_work(const mega_decayed_attention_args* a, int backward) {
  if (!a || !valid_dtype(a->dtype) || a->B <= 0 || a->L <= 0 || a->H <= 0 || a->K <= 0 || a->V <= 0 || a->K > MEGA_ATT_MOST || a->V > MEGA_ATT_MOST)
    return 0;
  size_t n = backward ? back_plan(*a, false).all : forward_floats(*a, false);
  if (tc_heads(*a)) n = std::max(n, backward ? back_plan(*a, true).all : forward_floats(*a, true));
  return (int64_t)(n * sizeof(float));
}

extern "C" MEGA_API int mega_decayed_attention_fwd(const mega_decayed_attention_args* a, mega_stream_t stream) {
  const int bad = check_args(a);
  if (bad) return bad;
  if (!a->y) return MEGA_ERR_NULL;
  Walk w = base(*a);
  w.q = operand(*a, a->q, a->qs, a->K), w.k = operand(*a, a->k, a->ks, a->K), w.v = operand(*a, a->v, a->vs, a->V);
  put_out(w, *a, a->y, a->ys);
  const Plan p = plan_of(tc_takes(a->dtype, w), a->dtype, a->B, a->L, a->H, a->K, a->V);
  if (p.local + p.factor + p.gates && !a->work) return MEGA_ERR_NULL;
  if (a->work && !aligned_to(a->work, 16)) return MEGA_ERR_ALIGN;
  w.s_in = a->h_in, w.s_out = a->h_out, w.s_row = a->V, w.s_col = 1;
  w.p_scale = w.o_scale = (float)a->scale, w.s_scale = 1.f;
  w.rev = (a->flags & MEGA_ATT_REVERSE) != 0;
  const int rc = run(a->dtype, w, p, 0, static_cast<float*>(a->work), stream);
  return rc ? rc : check_launch("decayed_attention_fwd");
}

extern "C" MEGA_API int mega_decayed_attention_bwd(const mega_decayed_attention_args* a, mega_stream_t stream) {
  const int bad = check_args(a);
  if (bad) return bad;
  if (!a->dy || !a->dq || !a->dk || !a->dv || !a->df || !a->work) return MEGA_ERR_NULL;
  if (!aligned_to(a->work, 16)) return MEGA_ERR_ALIGN;
  const Operand q = operand(*a, a->q, a->qs, a->K), k = operand(*a, a->k, a->ks, a->K), v = operand(*a, a->v, a->vs, a->V),
                dy = operand(*a, a->dy, a->gs, a->V);
  Walk w = base(*a);
  w.q = dy, w.k = v, w.v = k, w.x = q;
  put_out(w, *a, a->dq, a->dqs);
  Walk wk = base(*a), wv = base(*a);
  wk.q = v, wk.k = dy, wk.v = q, wk.x = k, wv.q = k, wv.k = q, wv.v = dy;
  put_out(wk, *a, a->dk, a->dks), put_out(wv, *a, a->dv, a->dvs);
  const BackPlan p = back_plan(*a, tc_takes(a->dtype, w) && tc_takes(a->dtype, wk) && tc_takes(a->dtype, wv));
  float* at = static_cast<float*>(a->work);
  auto take = [&](size_t n) { float* r = at; at += n; return r; };
  float* walk = take(p.walk);
  float2 *dots_q = reinterpret_cast<float2*>(take(p.dots)), *dots_k = reinterpret_cast<float2*>(take(p.dots));
  float *anchors = take(p.dq.anchors), *units = take(p.dq.units), *through = take(p.dq.through);
  const bool rev = (a->flags & MEGA_ATT_REVERSE) != 0;
  w.s_in = a->h_in, w.s_row = 1, w.s_col = a->V;
  w.p_scale = w.o_scale = (float)a->scale, w.s_scale = 1.f;
  w.rev = rev;
  w.dots = dots_q, w.anchors = anchors, w.units = units;
  int rc = run(a->dtype, w, p.dq, 1, walk, stream);
  if (rc) return rc;
  const Walk forward = w;

  wk.s_in = a->dh_out, wk.s_out = a->dh_in, wk.s_row = 1, wk.s_col = a->V;
  wk.p_scale = wk.s_scale = (float)a->scale, wk.o_scale = 1.f;
  wk.rev = !rev, wk.excl = 1;
  wk.dots = dots_k, wk.anchors = anchors, wk.units = units, wk.through = through;
  rc = run(a->dtype, wk, p.dk, 2, walk, stream);
  if (rc) return rc;

  wv.s_in = a->dh_out, wv.s_row = a->V, wv.s_col = 1;
  wv.p_scale = wv.s_scale = (float)a->scale, wv.o_scale = 1.f;
  wv.rev = !rev, wv.excl = 1, wv.gates_there = 1;   // (those of the walk before, in the same place)
  rc = run(a->dtype, wv, p.dv, 0, walk, stream);
  if (rc) return rc;

  const int tiles = p.dk.tc ? kTcDots : p.dk.tiles;
  const GateGrad gg = {forward, dots_q, dots_k, through, tiles, tiles, p.dk.tc ? kTcParts : p.dk.tiles, a->df, a->dfs[0], a->dfs[1],
                       a->dfs[2]};
  const dim3 grid((unsigned)(((long long)a->B * a->H * forward.chunks + 3) / 4));
  MEGA_DISPATCH_DTYPE(a->dtype, {
    if (p.dk.tc) launch(gate_grad_kernel<T, kTcChunk / 32>, grid, dim3(128), 0, stream, gg);
    else launch(gate_grad_kernel<T, kC / 32>, grid, dim3(128), 0, stream, gg);
  });
  if (p.dk.tc) g_last_kernel.store("decayed_attention_tc", std::memory_order_relaxed);   // (of the walks; the gates' gradient has one form)
  return check_launch("decayed_attention_bwd");
}

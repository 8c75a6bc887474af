// Linear attention with a decay for each head (decayed_attention.cu has the mathematics) on tcgen05 products, for 16-bit activations and
// heads of at most 128 keys and values: chunks of 128 steps, a block to a (sequence, head) or a segment of one.
//
// Per chunk, with rows i, j of the chunk, and keys and values padded to 64 or 128 with zeros:
//   P  = Q K^T                      accumulator P, 128 columns; the weighted pairs go back as 16-bit operand in its first 64
//   O1 = Q S                        S: the state that enters, in shared memory
//   dS = (w K)^T V                  w K in pieces of 8 (bf16, three) or 11 (fp16, two) bits, the first in K's place
//   O2 = (weighted pairs) V
// and y = e O1 + O2 with a row's factor e.  For the gates' gradient also X V^T, in O2's place before it.
// Roles: four warps of pairs and outputs (a thread has a row of the chunk), four or eight of weights and state (a thread has a step's
// keys, then a row of the state, whose fp32 values stay in its registers), one that loads, one for the gates, one for padded steps, one that issues products.  All exchange over
// mbarriers.
//
// Activations lie as TMA leaves them (columns of 64, rows of 128 bytes, swizzled), what the threads write as planes of 16 bytes along
// keys or values, rows one after another.  Both serve with either axis as the contraction, and a thread that owns a row reads and
// writes it without bank conflicts.  (Loads by cp.async, three warps of them, took 140 cycles each and held up every other access to
// shared memory: 213 us where this takes LATER, 8 x 4096 x 16 heads of 64.)
//
// The state is accumulated by each chunk's own sum, which is then added in fp32: a long chain inside the tensor cores' accumulator
// would be cut off, not rounded, thousands of times.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "decayed_attention.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace mega {
namespace {

constexpr int kC = kTcChunk, kPlane = kC * 16;

struct TcGates {
  float sum[kC], weight[kC];   // running sum of log2 a; weight of a step in the state that leaves
  uint8_t count[kC];           // resets so far
  float enter;                 // weight of the state that enters in the one that leaves
  int total;                   // resets
  int pad_[2];
};
// barriers; kQRaw...: what a load completes where padded steps have to be cleared before the rest may see it
enum { kQFull, kQEmpty, kKFull, kKEmpty = kKFull + 2, kVFull = kKEmpty + 2, kVEmpty = kVFull + 2, kXFull = kVEmpty + 2, kXEmpty, kGFull, kGEmpty = kGFull + 2,
       kPDone = kGEmpty + 2, kPReady, kODone, kORead, kSReady, kDsDone, kWReady, kLoFree, kW2Ready, kQRaw, kKRaw, kVRaw = kKRaw + 2, kXRaw = kVRaw + 2, kBars };

// kOut: outputs; else the state that a segment leaves by itself.  kDots: sums for the gates' gradient (1: walk of dq, 2: of dk).
template <typename T, int KD, int VD, bool kOut, int kDots>
struct Lay {
  static constexpr int kTk = KD * kC * 2, kTv = VD * kC * 2, kTs = VD / 8 * KD * 16;
  static constexpr int kPieces = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
  // with heads of 128 x 128 there is no room for the third piece: it takes the second's place when that has been used
  static constexpr bool kSeq = kOut && KD == 128 && VD == 128 && kPieces == 3;
  static constexpr int kVStages = kOut && kDots && KD == 128 && VD == 128 ? 1 : 2;
  static constexpr int kState = VD == 128 ? 8 : 4;                       // warps of weights and state
  static constexpr int kThreads = 32 * (4 + kState + 4);
  // (a product over 128 rows of 64 keys reads on into what follows: no piece and no tile of keys is last)
  static constexpr int kOffLo = 0, kOffLo2 = kOffLo + kTk, kOffK = kOffLo2 + (kPieces == 3 && !kSeq ? kTk : 0), kOffV = kOffK + 2 * kTk,
                       kOffQ = kOffV + kVStages * kTv, kOffX = kOffQ + (kOut ? kTk : 0), kOffS = kOffX + (kDots ? kTv : 0),
                       kOffG = kOffS + (kOut ? kTs : 0), kOffBar = kOffG + 2 * (int)sizeof(TcGates), kOffSlot = kOffBar + kBars * 8, kEnd = kOffSlot + 16;
  static_assert(kEnd <= 227 * 1024, "shared memory");
  static_assert(sizeof(TcGates) % 16 == 0, "gates");
};
// columns of tensor memory
constexpr uint32_t kColP = 0, kColO1 = 128, kColO2 = 256, kColS = 384;

__device__ __forceinline__ bool tried(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// A wait that gives up (after some seconds: never expected) raises `gone`; from then on no wait lasts, and everything runs out on
// whatever the buffers hold.
__device__ __noinline__ void wait_long(uint32_t bar, uint32_t parity, volatile int* gone) {
  const long long start = clock64();
  while (!*gone) {
    if (tried(bar, parity)) return;
    if (clock64() - start > 4000000000LL) {
      g_device_error = 1;
      *gone = 1;
    }
  }
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <int N>
__device__ __forceinline__ void loaded(float (&v)[N]) {   // (the registers of a load from tensor memory, once it has been waited for)
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void sts16(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Products, all over k = 16 places at a time.  d = or += a b; A in shared or tensor memory.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void umma_tm(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool onto) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
               "r"(id), "r"((uint32_t)onto)
               : "memory");
}
// planes whose contraction runs over the rows
__device__ __forceinline__ uint64_t over(uint32_t at, uint32_t plane) { return umma_desc(at, 128, plane); }

// columns of 64: rows whose contraction runs along them, or over the rows
constexpr int kBox = 64 * kC * 2;
__device__ __forceinline__ uint64_t tile_desc(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3fffu) | ((uint64_t)(kBox >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr int kAlong(int k) { return (k / 4 * kBox + k % 4 * 32) / 16; }   // of 16 places
constexpr int kOver(int k) { return k * 2048 / 16; }
// 16 bytes of a row
__device__ __forceinline__ uint32_t piece_of(int row, int c) { return c / 8 * kBox + row * 128 + ((c ^ row) & 7) * 16; }

struct Maps {
  CUtensorMap q, k, v, x;
};
__device__ __forceinline__ void tma_load_4d(uint32_t to, const CUtensorMap* m, int c, int t, int h, int b, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(c), "r"(t), "r"(h), "r"(b), "r"(bar)
               : "memory");
}
// 128 steps of an operand; rows behind the last one and columns it does not have become zeros.  An axis whose stride is 0 has one place.
template <int D>
__device__ __forceinline__ void load_tile(uint32_t to, const CUtensorMap* m, const Operand& o, int t0, int h, int b, uint32_t bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(D * kC * 2) : "memory");
#pragma unroll
  for (int c = 0; c < D; c += 64) tma_load_4d(to + c / 64 * kBox, m, c, t0, o.sh ? h : 0, o.sb ? b : 0, bar);
}
template <int D>
__device__ __forceinline__ void clear_rows(uint32_t at, const uint32_t (&pad)[4], int lane) {
#pragma unroll 1
  for (int k = 0; k < 4; ++k)
    if (pad[k] >> lane & 1)
#pragma unroll
      for (int c = 0; c < D / 8; ++c) sts16(at + piece_of(32 * k + lane, c), make_uint4(0, 0, 0, 0));
}

template <typename T, int KD, int VD, bool kOut, int kDots>
__global__ void __launch_bounds__(Lay<T, KD, VD, kOut, kDots>::kThreads, 1) tc_kernel(const __grid_constant__ Walk w, const __grid_constant__ Maps maps) {
  using L = Lay<T, KD, VD, kOut, kDots>;
  constexpr int kStateWarps = L::kState, kHalves = kStateWarps / 4, kStateThreads = 32 * kStateWarps;
  extern __shared__ __align__(1024) unsigned char smem[];
  int* const slot_ = reinterpret_cast<int*>(smem + L::kOffSlot);   // where tensor memory lies; whether a wait has given up
  volatile int* gone = slot_ + 1;
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bh = blockIdx.x % (w.B * w.H), seg = blockIdx.x / (w.B * w.H), b = bh / w.H, h = bh % w.H;
  const int first = seg * w.per, chunks = min(w.per, w.chunks - first);   // in the order of the walk
  auto bar = [&](int i) { return base + L::kOffBar + i * 8; };
  auto wait = [&](int i, uint32_t parity) {
    if (!tried(bar(i), parity)) wait_long(bar(i), parity, gone);
  };
  auto tile_of = [&](int n) { return w.rev ? w.chunks - 1 - first - n : first + n; };
  auto gates = [&](int n) -> TcGates& { return reinterpret_cast<TcGates*>(smem + L::kOffG)[n & 1]; };

  if (tid == 0) {
    *gone = 0;
    auto init = [&](int i, uint32_t count) { mbar_init(reinterpret_cast<uint64_t*>(smem + L::kOffBar) + i, count); };
    for (int i : {(int)kQFull, (int)kKFull, kKFull + 1, (int)kVFull, kVFull + 1, (int)kXFull, (int)kQRaw, (int)kKRaw, kKRaw + 1, (int)kVRaw, kVRaw + 1, (int)kXRaw})
      init(i, 1);
    for (int i : {(int)kGFull, kGFull + 1}) init(i, 32);
    for (int i : {(int)kQEmpty, (int)kKEmpty, kKEmpty + 1, (int)kVEmpty, kVEmpty + 1, (int)kPDone, (int)kODone, (int)kDsDone, (int)kLoFree}) init(i, 1);
    for (int i : {(int)kXEmpty, (int)kPReady, (int)kORead}) init(i, 128);
    for (int i : {(int)kSReady, (int)kWReady, (int)kW2Ready}) init(i, kStateThreads);
    for (int i : {(int)kGEmpty, kGEmpty + 1}) init(i, kStateThreads + (kOut ? 128 : 0));
    mbar_fence_init();
  }
  if (warp == 0) tm_alloc(smem_u32(slot_), kOut ? 512 : 128);
  tm_before();
  __syncthreads();
  tm_after();
  const uint32_t tm = *reinterpret_cast<volatile uint32_t*>(slot_);
  constexpr uint32_t kCs = kOut ? kColS : 0;

  if (warp < 4) {
    // ================================================================================ pairs and outputs
    if constexpr (kOut) {
      const int i = warp * 32 + lane;
      const uint32_t quarter = tm + ((uint32_t)(warp * 32) << 16);
      for (int n = 0; n < chunks; ++n) {
        const TcGates& g = gates(n);
        const long long t = (long long)tile_of(n) * kC + i;
        wait(kGFull + (n & 1), n >> 1 & 1);
        const float gi = g.sum[i];
        const int ci = g.count[i];
        const bool resets = g.total != 0;
        float inner = 0.f, read = 0.f;
        wait(kPDone, n & 1);
        tm_after();
        auto block = [&](int jb, auto diagonal, auto counted) {
          constexpr bool kDiag = decltype(diagonal)::value, kCount = decltype(counted)::value;
          float v[32], x[kDots ? 32 : 1];
          tm_ld32(quarter + kColP + 32 * jb, v);
          if constexpr (kDots != 0) tm_ld32(quarter + kColO2 + 32 * jb, x);
          tm_wait_ld();
          loaded(v);
          if constexpr (kDots != 0) loaded(x);
          uint32_t word[16];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 gj = *reinterpret_cast<const float4*>(g.sum + 32 * jb + j);
            uchar4 cj;
            if (kCount) cj = *reinterpret_cast<const uchar4*>(g.count + 32 * jb + j);
            const float gg[4] = {gj.x, gj.y, gj.z, gj.w};
            const unsigned char cc[4] = {cj.x, cj.y, cj.z, cj.w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              bool on = true;
              if (kDiag) on = w.rev ? j + m >= lane : j + m <= lane;
              if (kCount) on = on && cc[m] == ci;
              float p = v[j + m] * (w.p_scale * ex2(fminf(gi - gg[m], 0.f)));
              if (kDiag || kCount) p = on ? p : 0.f;
              v[j + m] = p;
              if constexpr (kDots != 0) {
                if (kDiag || kCount) inner += on && !(kDiag && j + m == lane) ? p * x[j + m] : 0.f;
                else inner += p * x[j + m];
              }
            }
            word[j / 2] = pack<T>(v[j], v[j + 1]), word[j / 2 + 1] = pack<T>(v[j + 2], v[j + 3]);
          }
          tm_st8(quarter + kColP + 16 * jb, word);
          tm_st8(quarter + kColP + 16 * jb + 8, word + 8);
        };
#pragma unroll 1
        for (int jb = 0; jb < 4; ++jb) {
          if (w.rev ? jb < warp : jb > warp) {
            uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            tm_st8(quarter + kColP + 16 * jb, zero);
            tm_st8(quarter + kColP + 16 * jb + 8, zero);
          } else if (resets) {
            if (jb == warp) block(jb, std::true_type(), std::true_type());
            else block(jb, std::false_type(), std::true_type());
          } else {
            if (jb == warp) block(jb, std::true_type(), std::false_type());
            else block(jb, std::false_type(), std::false_type());
          }
        }
        tm_wait_st();
        tm_before();
        arrive(bar(kPReady));

        const float e = ci ? 0.f : w.o_scale * ex2(gi);
        if (kDots) wait(kXFull, n & 1);
        wait(kODone, n & 1);
        tm_after();
        char* row = static_cast<char*>(w.out) + (b * w.ob + h * w.oh + t * w.ol) * 2;
#pragma unroll 1
        for (int c = 0; c < VD; c += 32) {
          float o[32], p[32];
          tm_ld32(quarter + kColO1 + c, o);
          tm_ld32(quarter + kColO2 + c, p);
          tm_wait_ld();
          loaded(o);
          loaded(p);
#pragma unroll
          for (int m = 0; m < 32; ++m) o[m] *= e;
          if constexpr (kDots != 0) {
#pragma unroll
            for (int m = 0; m < 32; m += 8) {
              const uint4 u = lds16(base + L::kOffX + piece_of(i, (c + m) / 8));
              const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 x = unpack<T>(uu[k]);
                read += o[m + 2 * k] * x.x + o[m + 2 * k + 1] * x.y;
              }
            }
          }
          uint32_t word[16];
#pragma unroll
          for (int m = 0; m < 16; ++m) word[m] = pack<T>(o[2 * m] + p[2 * m], o[2 * m + 1] + p[2 * m + 1]);
          if (t < w.L) {
            if (w.piece == 32) {
#pragma unroll
              for (int m = 0; m < 16; m += 8)
                if (c + 2 * m < w.v.d)
                  asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + (c + 2 * m) * 2), "r"(word[m]),
                               "r"(word[m + 1]), "r"(word[m + 2]), "r"(word[m + 3]), "r"(word[m + 4]), "r"(word[m + 5]), "r"(word[m + 6]), "r"(word[m + 7])
                               : "memory");
            } else if (w.piece == 16) {
#pragma unroll
              for (int m = 0; m < 16; m += 4)
                if (c + 2 * m < w.v.d) *reinterpret_cast<uint4*>(row + (c + 2 * m) * 2) = make_uint4(word[m], word[m + 1], word[m + 2], word[m + 3]);
            } else {
#pragma unroll
              for (int m = 0; m < 32; ++m)
                if (c + m < w.v.d) *reinterpret_cast<unsigned short*>(row + (c + m) * 2) = (unsigned short)(word[m / 2] >> (16 * (m & 1)));
            }
          }
        }
        tm_before();
        arrive(bar(kORead));
        if (kDots) {
          arrive(bar(kXEmpty));
          if (t < w.L) w.dots[(long long)bh * w.L + t] = make_float2(read, inner);
        }
        arrive(bar(kGEmpty + (n & 1)));
      }
    }
  } else if (warp < 4 + kStateWarps) {
    // ================================================================================ weights and state
    const int sw = warp - 4, row = (sw & 3) * 32 + lane, half = sw >> 2;   // a step, or a key; half: of the planes of keys, of the values
    const uint32_t quarter = tm + ((uint32_t)((sw & 3) * 32) << 16);
    const bool holds = (sw & 3) * 32 < KD;   // (of 64 keys two warps have none)
    constexpr int kPlanes = KD / 8 / kHalves;
    const int col0 = half * 64;
    float st[64];
    const long long s_at = (long long)bh * w.k.d * w.v.d + (long long)row * w.s_row;
    auto slot = [&](long long at) { return (at * w.k.d + row) * VD + col0; };   // a row of a state in the workspace
    const bool mine = holds && row < w.k.d;
#pragma unroll
    for (int c = 0; c < 64; ++c) st[c] = kOut && mine && w.s_in && col0 + c < w.v.d ? w.s_in[s_at + (long long)(col0 + c) * w.s_col] : 0.f;
    if (kOut)
      for (int p = 0; p < seg; ++p) {
        const float fac = w.factor[(long long)p * w.B * w.H + bh];
        const float* l = w.local + slot((long long)p * w.B * w.H + bh);
        if (mine)
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            const float4 u = *reinterpret_cast<const float4*>(l + c);
            const float uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) st[c + k] = (fac == 0.f ? 0.f : fac * st[c + k]) + uu[k];
          }
      }
    // the state as an operand: rounded to 16 bits (the state itself is not)
    auto state_out = [&]() {
      if (holds)
#pragma unroll
        for (int c = 0; c < 64; c += 8)
          sts16(base + L::kOffS + (col0 + c) / 8 * (KD * 16) + row * 16,
                make_uint4(pack<T>(st[c], st[c + 1]), pack<T>(st[c + 2], st[c + 3]), pack<T>(st[c + 4], st[c + 5]), pack<T>(st[c + 6], st[c + 7])));
      fence_proxy_async();
      arrive(bar(kSReady));
    };
    if (kOut) state_out();
    float decay = 1.f;
    for (int n = 0; n < chunks; ++n) {
      const TcGates& g = gates(n);
      wait(kGFull + (n & 1), n >> 1 & 1);
      wait(kKFull + (n & 1), n >> 1 & 1);
      if (kOut) wait(kPDone, n & 1);   // (the pairs' product has read the keys)
      const float wt = g.weight[row], enter = g.enter;
      uint4 last[L::kSeq ? kPlanes : 1];
#pragma unroll
      for (int c = 0; c < kPlanes; ++c) {
        const uint32_t at = (half * kPlanes + c) * kPlane + row * 16, key = base + L::kOffK + (n & 1) * L::kTk + piece_of(row, half * kPlanes + c);
        const uint4 u = lds16(key);
        const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
        uint32_t piece[3][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 v = unpack<T>(uu[k]);
          v.x *= wt, v.y *= wt;
#pragma unroll
          for (int p = 0; p < L::kPieces; ++p) {
            piece[p][k] = pack<T>(v.x, v.y);
            const float2 r = unpack<T>(piece[p][k]);
            v.x -= r.x, v.y -= r.y;
          }
        }
        sts16(key, make_uint4(piece[0][0], piece[0][1], piece[0][2], piece[0][3]));
        sts16(base + L::kOffLo + at, make_uint4(piece[1][0], piece[1][1], piece[1][2], piece[1][3]));
        if constexpr (L::kPieces == 3) {
          const uint4 v = make_uint4(piece[2][0], piece[2][1], piece[2][2], piece[2][3]);
          if constexpr (L::kSeq) last[c] = v;
          else sts16(base + L::kOffLo2 + at, v);
        }
      }
      fence_proxy_async();
      arrive(bar(kWReady));
      if constexpr (kDots != 0) {
        // the state that enters: left by the walk of dq, multiplied with the gradient of the one that leaves by that of dk
        T* a = static_cast<T*>(w.anchors) + slot((long long)bh * w.chunks + tile_of(n));
        if (kDots == 1) {
          if (mine && enter != 0.f)
#pragma unroll
            for (int c = 0; c < 64; c += 8)
              *reinterpret_cast<uint4*>(a + c) =
                  make_uint4(pack<T>(st[c], st[c + 1]), pack<T>(st[c + 2], st[c + 3]), pack<T>(st[c + 4], st[c + 5]), pack<T>(st[c + 6], st[c + 7]));
        } else {
          float s = 0.f;
          if (mine && enter > kLeast)
#pragma unroll
            for (int c = 0; c < 64; c += 8) {
              const uint4 u = *reinterpret_cast<const uint4*>(a + c);
              const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 v = unpack<T>(uu[k]);
                s += st[c + 2 * k] * v.x + st[c + 2 * k + 1] * v.y;
              }
            }
#pragma unroll
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
          if (lane == 0) {
            float* to = w.through + ((long long)bh * w.chunks + tile_of(n)) * kTcParts;
            to[sw] = enter > kLeast ? enter * s : 0.f;
            if (kStateWarps < kTcParts) to[sw + 4] = 0.f;
          }
        }
      }
      if constexpr (L::kSeq) {
        wait(kLoFree, n & 1);
#pragma unroll
        for (int c = 0; c < kPlanes; ++c) sts16(base + L::kOffLo + (half * kPlanes + c) * kPlane + row * 16, last[c]);
        fence_proxy_async();
        arrive(bar(kW2Ready));
      }
      wait(kDsDone, n & 1);
      tm_after();
      if (holds) {
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          tm_ld32(quarter + kCs + col0 + c, v);
          tm_wait_ld();
          loaded(v);
#pragma unroll
          for (int k = 0; k < 32; ++k) st[c + k] = (enter == 0.f ? 0.f : enter * st[c + k]) + v[k];
        }
        tm_before();
      }
      decay *= enter;
      arrive(bar(kGEmpty + (n & 1)));
      if (kOut && n + 1 < chunks) state_out();
    }
    if (!kOut) {
      if (mine) {
        float* l = w.local + slot((long long)seg * w.B * w.H + bh);
#pragma unroll
        for (int c = 0; c < 64; c += 4) *reinterpret_cast<float4*>(l + c) = make_float4(st[c], st[c + 1], st[c + 2], st[c + 3]);
      }
      if (sw == 0 && lane == 0) w.factor[(long long)seg * w.B * w.H + bh] = decay;
    } else if (w.s_out && first + chunks == w.chunks && mine) {
#pragma unroll
      for (int c = 0; c < 64; ++c)
        if (col0 + c < w.v.d) w.s_out[s_at + (long long)(col0 + c) * w.s_col] = st[c];
    }
  } else if (warp == 4 + kStateWarps) {
    // ================================================================================ loads
    if (umma_elect()) {
      constexpr int kS = L::kVStages;
      const bool raw = w.pad != nullptr;
      for (int n = 0; n < chunks; ++n) {
        const int t0 = tile_of(n) * kC, stage = kS == 2 ? n & 1 : 0, use = kS == 2 ? n >> 1 : n;
        if (n > 1) wait(kKEmpty + (n & 1), ((n >> 1) - 1) & 1);
        load_tile<KD>(base + L::kOffK + (n & 1) * L::kTk, &maps.k, w.k, t0, h, b, bar((raw ? kKRaw : kKFull) + (n & 1)));
        auto values = [&]() {
          if (use) wait(kVEmpty + stage, (use - 1) & 1);
          load_tile<VD>(base + L::kOffV + stage * L::kTv, &maps.v, w.v, t0, h, b, bar((raw ? kVRaw : kVFull) + stage));
        };
        if (kS == 2) values();
        if (kOut) {
          if (n) wait(kQEmpty, (n - 1) & 1);
          load_tile<KD>(base + L::kOffQ, &maps.q, w.q, t0, h, b, bar(raw ? kQRaw : kQFull));
        }
        if (kDots) {
          if (n) wait(kXEmpty, (n - 1) & 1);
          load_tile<VD>(base + L::kOffX, &maps.x, w.x, t0, h, b, bar(raw ? kXRaw : kXFull));
        }
        if (kS == 1) values();
      }
    }
    __syncwarp();
  } else if (warp == 5 + kStateWarps) {
    // ================================================================================ gates
    GateIn<4> ahead = gates_fetch<4>(w, b, h, tile_of(0), lane);
    for (int n = 0; n < chunks; ++n) {
      const GateIn<4> in = ahead;
      if (n + 1 < chunks) ahead = gates_fetch<4>(w, b, h, tile_of(n + 1), lane);
      if (n > 1) wait(kGEmpty + (n & 1), ((n >> 1) - 1) & 1);
      const GateOut<4> r = gates_scan<4>(w, in, lane);
      TcGates& g = gates(n);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = gate_row<4>(w, lane, k);
        g.sum[at] = gate_sum(r.sum[k]) + r.bad, g.weight[at] = r.weight[k], g.count[at] = (uint8_t)r.count[k];
      }
      if (lane == 0) g.enter = r.enter, g.total = r.total;
      __syncwarp();
      arrive(bar(kGFull + (n & 1)));
    }
  } else if (warp == 6 + kStateWarps) {
    // ================================================================================ padded steps: whatever lies there becomes zeros
    if (w.pad) {
      for (int n = 0; n < chunks; ++n) {
        const int t0 = tile_of(n) * kC, rows = min(kC, w.L - t0);
        constexpr int kS = L::kVStages;
        const int stage = kS == 2 ? n & 1 : 0, use = kS == 2 ? n >> 1 : n;
        const uint8_t* m = w.pad + (long long)b * w.L + t0;
        uint32_t pad[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) pad[k] = __ballot_sync(~0u, 32 * k + lane < rows && m[32 * k + lane]);
        const bool any = (pad[0] | pad[1] | pad[2] | pad[3]) != 0;
        auto pass = [&](auto width, uint32_t at, int from, int to, uint32_t parity) {
          wait(from, parity);
          if (any) {
            clear_rows<decltype(width)::value>(at, pad, lane);
            fence_proxy_async();
          }
          __syncwarp();
          if (lane == 0) arrive(bar(to));
        };
        using Keys = std::integral_constant<int, KD>;
        using Values = std::integral_constant<int, VD>;
        pass(Keys(), base + L::kOffK + (n & 1) * L::kTk, kKRaw + (n & 1), kKFull + (n & 1), n >> 1 & 1);
        if (kOut) pass(Keys(), base + L::kOffQ, kQRaw, kQFull, n & 1);
        if (kDots && kS == 1) pass(Values(), base + L::kOffX, kXRaw, kXFull, n & 1);
        pass(Values(), base + L::kOffV + stage * L::kTv, kVRaw + stage, kVFull + stage, use & 1);
        if (kDots && kS == 2) pass(Values(), base + L::kOffX, kXRaw, kXFull, n & 1);
      }
    }
  } else {
    // ================================================================================ products
    if (umma_elect()) {
    constexpr uint32_t kPairs = idesc<T>(128, false, false), kRows = idesc<T>(VD, false, true), kBoth = idesc<T>(VD, true, true);
    constexpr int kS = L::kVStages;
    const uint64_t q = tile_desc(base + L::kOffQ), s = over(base + L::kOffS, KD * 16), x = tile_desc(base + L::kOffX);
    const uint64_t lo = over(base + L::kOffLo, kPlane), lo2 = over(base + L::kOffLo2, kPlane);
    for (int n = 0; n < chunks; ++n) {
      const int stage = kS == 2 ? n & 1 : 0, use = kS == 2 ? n >> 1 : n;
      const uint32_t key = base + L::kOffK + (n & 1) * L::kTk, val = base + L::kOffV + stage * L::kTv;
      const uint64_t kt = tile_desc(key), vt = tile_desc(val);
      if constexpr (kOut) {
        wait(kQFull, n & 1);
        wait(kKFull + (n & 1), n >> 1 & 1);
        if (kDots) {
          wait(kXFull, n & 1);
          wait(kVFull + stage, use & 1);
          if (n) wait(kORead, (n - 1) & 1);
        }
        tm_after();
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) umma(tm + kColP, q + kAlong(k), kt + kAlong(k), kPairs, k > 0);
        if (kDots)
#pragma unroll
          for (int k = 0; k < VD / 16; ++k) umma(tm + kColO2, x + kAlong(k), vt + kAlong(k), kPairs, k > 0);
        umma_commit(bar(kPDone));
        wait(kSReady, n & 1);
        if (!kDots && n) wait(kORead, (n - 1) & 1);
        tm_after();
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) umma(tm + kColO1, q + kAlong(k), s + k * 16, kRows, k > 0);
        umma_commit(bar(kQEmpty));
      }
      wait(kWReady, n & 1);
      wait(kVFull + stage, use & 1);
      tm_after();
      if constexpr (L::kPieces == 3 && !L::kSeq)
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma(tm + kCs, lo2 + k * 16, vt + kOver(k), kBoth, k > 0);
#pragma unroll
      for (int k = 0; k < kC / 16; ++k) umma(tm + kCs, lo + k * 16, vt + kOver(k), kBoth, k > 0 || (L::kPieces == 3 && !L::kSeq));
#pragma unroll
      for (int k = 0; k < kC / 16; ++k) umma(tm + kCs, kt + kOver(k), vt + kOver(k), kBoth, true);
      if constexpr (L::kSeq) umma_commit(bar(kLoFree));
      else {
        umma_commit(bar(kDsDone));
        umma_commit(bar(kKEmpty + (n & 1)));
      }
      if constexpr (kOut) {
        wait(kPReady, n & 1);
        tm_after();
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma_tm(tm + kColO2, tm + kColP + k * 8, vt + kOver(k), kRows, k > 0);
        umma_commit(bar(kODone));
      }
      if constexpr (L::kSeq) {
        wait(kW2Ready, n & 1);
        tm_after();
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma(tm + kCs, lo + k * 16, vt + kOver(k), kBoth, true);
        umma_commit(bar(kDsDone));
        umma_commit(bar(kKEmpty + (n & 1)));
      }
      umma_commit(bar(kVEmpty + stage));
    }
    // (nothing of this block's products is on its way when it ends: the last of each kind has been waited for by the other roles, or is)
    const int stage = kS == 2 ? (chunks - 1) & 1 : 0, use = kS == 2 ? (chunks - 1) >> 1 : chunks - 1;
    wait(kVEmpty + stage, use & 1);
    }
    __syncwarp();
  }
  tm_before();
  __syncthreads();
  tm_after();
  if (warp == 0) tm_free(tm, kOut ? 512 : 128);
}

template <typename T, int KD, int VD>
void run(const Walk& w, const Maps& maps, int dots, void* stream) {
  const long long blocks = (long long)w.B * w.H;
  auto go = [&](auto kernel, auto lay, long long n) {
    using L = decltype(lay);
    launch(kernel, dim3((unsigned)n), dim3(L::kThreads), L::kEnd, stream, w, maps);
  };
  if (w.segs > 1) go(tc_kernel<T, KD, VD, false, 0>, Lay<T, KD, VD, false, 0>(), blocks * (w.segs - 1));
  if (dots == 0) go(tc_kernel<T, KD, VD, true, 0>, Lay<T, KD, VD, true, 0>(), blocks * w.segs);
  else if (dots == 1) go(tc_kernel<T, KD, VD, true, 1>, Lay<T, KD, VD, true, 1>(), blocks * w.segs);
  else go(tc_kernel<T, KD, VD, true, 2>, Lay<T, KD, VD, true, 2>(), blocks * w.segs);
}
template <typename T>
void pick(const Walk& w, const Maps& m, int dots, void* stream) {
  if (w.k.d <= 64) w.v.d <= 64 ? run<T, 64, 64>(w, m, dots, stream) : run<T, 64, 128>(w, m, dots, stream);
  else w.v.d <= 64 ? run<T, 128, 64>(w, m, dots, stream) : run<T, 128, 128>(w, m, dots, stream);
}

// (width, step, head, sequence) of an operand; false where TMA cannot address it
bool map_of(CUtensorMap* m, int dtype, const Operand& o, const Walk& w) {
  auto place = [](int n, long long stride) { return (uint64_t)(stride ? n : 1); };
  auto step = [](long long stride) { return stride ? stride : 8; };
  return make_tensor_map_4d(m, dtype, o.p, o.d, w.L, place(w.H, o.sh), place(w.B, o.sb), step(o.sl), step(o.sh), step(o.sb), 64, kC);
}
bool maps_of(Maps* m, int dtype, const Walk& w) {
  if (!map_of(&m->q, dtype, w.q, w) || !map_of(&m->k, dtype, w.k, w) || !map_of(&m->v, dtype, w.v, w)) return false;
  if (!w.x.p) m->x = m->v;
  return !w.x.p || map_of(&m->x, dtype, w.x, w);
}
}  // namespace

bool tc_takes(int dtype, const Walk& w) {
  if (dtype == MEGA_F32 || g_options[OPT_DISABLE_MMA].load()) return false;
  for (const Operand* o : {&w.q, &w.k, &w.v, &w.x})
    if (o->p && (o->d > kTcMost || o->vec < 16 || o->sl < 0 || o->sh < 0 || o->sb < 0 || (o->sl == 0 && w.L > 1))) return false;
  Maps m;   // (what the driver refuses is known before a plan is made)
  return maps_of(&m, dtype, w);
}
int tc_walk(int dtype, const Walk& w, int dots, void* stream) {
  Maps m;
  if (!maps_of(&m, dtype, w)) return MEGA_ERR_UNSUPPORTED;
  dtype == MEGA_BF16 ? pick<__nv_bfloat16>(w, m, dots, stream) : pick<__half>(w, m, dots, stream);
  g_last_kernel.store("decayed_attention_tc", std::memory_order_relaxed);
  return MEGA_OK;
}
cudaError_t tc_read_device_error(int* v, bool reset) { return read_device_error(v, reset); }
}  // namespace mega

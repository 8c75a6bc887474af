// Gated linear recurrence: a decay per step, sequence and channel; forward, backward, single step.
//
//   l_t = sigmoid(-f_t),  h_t = h_{t-1} - l_t h_{t-1} + c_t,  c_t = l_t x_t  or  sigmoid(i_t) x_t
//
// written with the leak l where a gate stands open (f >> 0): it is far below the spacing of floats next to 1, and a decay 1 - l would
// round it to a few bits, the same way at every step.  Where a gate is closed (f << 0) it is the decay k that is small, and 1 - l
// has few of its bits, or none: there h = x + k (h - x), and the gradient of f, k l times the rest, has k as it is.  fp32 calls take the
// smaller of l and k at every step (gate_side2); 16-bit calls l alone, and the sides in segments where a gate is closed that far, which
// the warp looks at first (bf16, the sides in all segments: B = 8, L = 4096, D = 2048 forward 90 us against 74, backward 158 against 124;
// B = 1, L = 65536 216 against 185 and 385 against 304).
//
// A run of steps maps the state that enters it linearly to the one that leaves, h -> h_loc + A h (h_loc: from a zero state,
// A: the product of the decays), and such maps compose, so the time axis is split: a warp takes 64 channels (two to a lane) of
// kS steps, a block kW such segments, a cluster of up to eight blocks as many block tiles, and walks the sequence in
// strides of the cluster.  A segment is walked once, h_loc and A of every step staying in registers; its map goes through
// shared memory to the block's other warps, the block's through distributed shared memory to the cluster's other blocks;
// then y_t = h_loc,t + A_t h for the state h that enters.  Inputs are read once, by cp.async into a ring of the warp's own, so
// the next tile is on its way while this one is worked on and exchanged.
//
// Backward, with q the gradient that flows into the state behind a step: g_t = dy_t + q, q' = k_t g_t, a linear map
// of the same kind walked the other way.  The states are walked again from one that the forward left for each segment.
//   tied gates   dx = l g,  df = k l (h_{t-1} - x) g       input gate s   dx = s g,  df = k l h_{t-1} g,  di = s (1 - s) x g
//
// A reset is a map that ignores what enters: its A is -0 (the decays are never negative), and A = -0 means h_loc alone, so
// that nothing infinite or NaN passes.
//
// Infinities.  As the recurrence has it, an infinite state stays until a reset or the other infinity comes, and a state between two
// large values is no larger than they are.  h - x of such values overflows, an infinity less its leak is NaN, and so is one times a
// product of decays that has underflowed: all of them mark the values behind them as not finite.  Each lane keeps what it has seen
// of that (a product with 0 a round); where it has, one warp goes through the tile's steps in order at the end, and what had come out
// not finite is replaced (0.5 us a step forward and 1 backward, until all is NaN: joining infinite maps as they come cost calls that
// have none 3 to 12 %).
//
// Bound: HBM where the blocks fill the device (B = 64, L = 1024, D = 2048 bf16: forward 134 us, backward 224, 0.92 and 0.91 of the
// measured copy rate over 3 and 5 arrays).  With fewer it is the rounds: a multiprocessor takes some 1.2 us for a block's tile, of
// which the special-function operations of the gates are 0.55 and its instructions 0.6, and an exchange through a cluster adds 0.3
// to 0.7 (B = 8, L = 4096, D = 2048 74 and 124 us; B = 1, L = 65536, D = 2048 184 and 304, 0.67 and 0.67).  Resets cost 3 to 4 % more.
// What was tried there, beside 190 and 305 us at the larger then, and no faster: leaks of the next tile taken while a block waits (203
// and 347, registers); stages of the gates' operations batched over 4, 8 and 16 rows (210, 210, 205); three stages of the ring (198);
// segments of 8 steps and three blocks to a multiprocessor (255); blocks of four warps (better where there are four for each
// multiprocessor and more, worse backward); clusters spread over the multiprocessors by preference.
// Of 128 registers the 16-byte forms spill 8 bytes a thread at most, the 4-byte ones 16; rows of 16-bit values on odd addresses, which
// come through registers, up to 144 backward and 80 forward (B = 32, L = 2000, D = 1001 346 us backward, D = 1000 176).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "gated_recurrence.cuh"
#include "gates.cuh"
#include "tma.cuh"

namespace mega {

namespace {

constexpr int kW = 8;        // segments (warps) of a block: two blocks of 128 registers a thread fit a multiprocessor (kResident)
constexpr int kC = 64;       // channels of a tile: two to a lane, for packed arithmetic; a row is 128 or 256 bytes
constexpr int kStages = 2;   // tiles of a warp's ring (one is worked on while 64 KB a multiprocessor are on their way)

struct RecArgs {
  const void *x, *f, *i, *dy;
  void *y, *dx, *df, *di;
  // strides in elements of the axes before the channels; a walk from the last step has its pointers there and these negative
  long long xsb, xsl, fsb, fsl, isb, isl, ysb, ysl, gsb, gsl, dxb, dxl, dfb, dfl, dib, dil;
  const unsigned char *pad, *reset;
  long long msb, msl;
  const float *h_in, *dh_out;
  float *h_out, *starts, *dh_in;
  int L, D, pairs;   // pairs: whether two floats of a state lie on 8 bytes
  int tiles, units;   // of a row's channels, of the call
};

// Steps of a segment: what h_loc and A of every step (the backward: leak, state and, with an input gate, its two factors) leave of
// 128 registers; fp32 tiles would not fit the shared memory of two blocks otherwise (the backward with an input gate does not with 8
// either).  The forward saves the states that the backward's segments start from.
template <typename T, bool kGate>
constexpr int kBackSteps = sizeof(T) == 4 || kGate ? 8 : 16;
template <typename T>
constexpr int kForwardSteps = sizeof(T) == 4 ? 8 : 16;
// Blocks on a multiprocessor.  The fp32 backward with an input gate has 128 KB of tiles to a block: one, which may have all registers.
template <typename T, bool kGate, bool kBack>
constexpr int kResident = kBack && kGate && sizeof(T) == 4 ? 1 : 2;
template <typename T, bool kGate, bool kBack>
constexpr int kRingBytes = kW * kStages * ((kGate ? 3 : 2) + (kBack ? 1 : 0)) * (kBack ? kBackSteps<T, kGate> : kForwardSteps<T>) * kC * (int)sizeof(T);

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes to the same place in another block's shared memory, counted by the barrier at that block's `bar`
__device__ __forceinline__ void send(float4* p, uint64_t* bar, int rank, float4 v) {
  uint32_t at, to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w), "r"(to)
               : "memory");
}
// What the cluster's blocks sent for this phase has arrived.  Bounded: false, with the error word raised, after about 2 s.
__device__ __forceinline__ bool received(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  const long long start = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity)
        : "memory");
    if (ok) return true;
    if (clock64() - start > 4000000000LL) {
      g_device_error = 1;
      return false;
    }
  }
}
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int valid) {   // the rest of kBytes is zeroed
  if (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ f32x2 neg2(f32x2 v) { return v ^ 0x8000000080000000ull; }

// -sigmoid(-f): minus the leak
template <typename T>
__device__ __forceinline__ f32x2 minus_leak2(f32x2 f) {
  return minus_sigmoid2<T, 1>(f);
}
// Whether every gate is held by the smaller of its sides.  In 16-bit types that is left to segments with a gate so far closed that
// 1 - l loses what a 16-bit value shows of the decay (any_closed).
template <typename T>
constexpr bool kSides = sizeof(T) == 4;
// The least of the gates' arguments that a lane has seen.  1 - l is off by 3 x 2^-24 absolutely (the sum 1 + e and the reciprocal):
// above kLeast by at most 2^-13.7 of the decay (fp16: 2^-15.2), a twenty-sixth (a ninth) of the type's half step.
template <typename T>
struct LeastGate {   // (fp32: none)
  __device__ __forceinline__ void see(const T*) {}
  __device__ __forceinline__ bool closed() const { return false; }
};
template <>
struct LeastGate<__nv_bfloat16> {
  static constexpr float kLeast = -6.f;
  __nv_bfloat162 v = __floats2bfloat162_rn(0.f, 0.f);
  __device__ __forceinline__ void see(const __nv_bfloat16* p) { v = __hmin2(v, *reinterpret_cast<const __nv_bfloat162*>(p)); }
  __device__ __forceinline__ bool closed() const { return fminf(__low2float(v), __high2float(v)) < kLeast; }
};
template <>
struct LeastGate<__half> {
  static constexpr float kLeast = -5.f;
  __half2 v = __floats2half2_rn(0.f, 0.f);
  __device__ __forceinline__ void see(const __half* p) { v = __hmin2(v, *reinterpret_cast<const __half2*>(p)); }
  __device__ __forceinline__ bool closed() const { return fminf(__low2float(v), __high2float(v)) < kLeast; }
};
// sigmoid(i), and sigmoid(i) sigmoid(-i) where the caller asks for it
template <typename T, bool kSlope>
__device__ __forceinline__ f32x2 gate2(f32x2 i, f32x2& slope) {
  const f32x2 e = exp_pair<T, -1>(i), ns = minus_over_one_and(e);
  if (kSlope) {   // s (e s): 1 - s would lose what there is of it when the gate stands open; an infinite e comes with s = 0
    float a, b;
    unpack2(e, a, b);
    slope = mul2(mul2(pack2(fminf(a, 3.4e38f), fminf(b, 3.4e38f)), ns), ns);
  }
  return neg2(ns);
}

// two neighbouring values of shared memory
__device__ __forceinline__ f32x2 two(const float* p) {
  const float2 v = *reinterpret_cast<const float2*>(p);
  return pack2(v.x, v.y);
}
__device__ __forceinline__ f32x2 two(const __nv_bfloat16* p) {
  const unsigned v = *reinterpret_cast<const unsigned*>(p);
  return pack2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ f32x2 two(const __half* p) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(p));
  return pack2(v.x, v.y);
}
// two values to memory: as one word where kPair, `n` of them (0 .. 2) are inside
template <bool kPair>
__device__ __forceinline__ void put(float* p, f32x2 v, int n) {
  float a, b;
  unpack2(v, a, b);
  if (kPair && n == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(a, b);
  } else {
    if (n > 0) p[0] = a;
    if (n > 1) p[1] = b;
  }
}
template <bool kPair>
__device__ __forceinline__ void put(__nv_bfloat16* p, f32x2 v, int n) {
  float a, b;
  unpack2(v, a, b);
  if (kPair && n == 2) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
  } else {
    if (n > 0) p[0] = __float2bfloat16_rn(a);
    if (n > 1) p[1] = __float2bfloat16_rn(b);
  }
}
template <bool kPair>
__device__ __forceinline__ void put(__half* p, f32x2 v, int n) {
  float a, b;
  unpack2(v, a, b);
  if (kPair && n == 2) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
  } else {
    if (n > 0) p[0] = __float2half_rn(a);
    if (n > 1) p[1] = __float2half_rn(b);
  }
}
__device__ __forceinline__ f32x2 minus_zero() { return 0x8000000080000000ull; }

__device__ __forceinline__ f32x2 get_state(const float* p, int n, bool pairs) {
  if (p == nullptr || n == 0) return pack2(0.f, 0.f);
  if (pairs && n == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    return pack2(v.x, v.y);
  }
  return pack2(p[0], n > 1 ? p[1] : 0.f);
}
__device__ __forceinline__ void put_state(float* p, f32x2 v, int n, bool pairs) {
  if (pairs)
    put<true>(p, v, n);
  else
    put<false>(p, v, n);
}

// a map of the state: what a run makes of zero, and the factor of what enters
struct Map {
  f32x2 a, h;
  __device__ __forceinline__ float4 words() const {
    float4 v;
    unpack2(a, v.x, v.y);
    unpack2(h, v.z, v.w);
    return v;
  }
  __device__ __forceinline__ static Map of(float4 v) { return {pack2(v.x, v.y), pack2(v.z, v.w)}; }
  template <bool kReset>
  __device__ __forceinline__ f32x2 operator()(f32x2 in) const {
    f32x2 r = fma2(a, in, h);
    if (kReset) {
      float a0, a1, h0, h1, r0, r1;
      unpack2(a, a0, a1), unpack2(h, h0, h1), unpack2(r, r0, r1);
      r = pack2(__float_as_int(a0) == (int)0x80000000 ? h0 : r0, __float_as_int(a1) == (int)0x80000000 ? h1 : r1);
    }
    return r;
  }
};
// first, then second
template <bool kReset>
__device__ __forceinline__ Map then(const Map& first, const Map& second) {
  Map r = {mul2(first.a, second.a), second.operator()<kReset>(first.h)};
  if (kReset) {
    float b0, b1, r0, r1;
    unpack2(second.a, b0, b1), unpack2(r.a, r0, r1);
    r.a = pack2(__float_as_int(b0) == (int)0x80000000 ? b0 : r0, __float_as_int(b1) == (int)0x80000000 ? b1 : r1);
  }
  return r;
}

// One operand's tiles: [kS][kC] values of a warp, kMode bytes to a copy (2: through registers, for rows of 16-bit values that lie
// on odd ones).
template <typename T, int kS, int kMode>
struct Tile {
  static constexpr int kBytes = kS * kC * (int)sizeof(T);
  static constexpr int kRow = kC * (int)sizeof(T);
  // rows t0 .. t0 + kS of p (at the tile's first channel), of which `rows` are inside, and `chans` channels
  static __device__ __forceinline__ void fetch(char* dst, const T* p, long long stride, int t0, int rows, int chans, int lane) {
    if (kMode == 2) {
      unsigned short v[2 * kS];
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p + (long long)t0 * stride);
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        v[2 * s] = s < rows && lane < chans ? __ldg(q + s * stride + lane) : (unsigned short)0;
        v[2 * s + 1] = s < rows && lane + 32 < chans ? __ldg(q + s * stride + lane + 32) : (unsigned short)0;
      }
      unsigned short* d = reinterpret_cast<unsigned short*>(dst);
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        d[s * kC + lane] = v[2 * s];
        d[s * kC + lane + 32] = v[2 * s + 1];
      }
      return;
    }
    constexpr int kPer = kRow / (kMode == 16 ? 16 : 4);                // copies to a row
    constexpr int kRows = kPer >= 32 ? 1 : 32 / kPer;                 // rows to a round of the warp
    constexpr int kOver = kPer >= 32 ? kPer / 32 : 1;                 // rounds to a row
    const int row = kPer >= 32 ? 0 : lane / kPer, col = (kPer >= 32 ? lane : lane % kPer) * kMode;
    const char* base = reinterpret_cast<const char*>(p);
    const uint32_t to = smem_u32(dst) + row * kRow + col;
    const char* from = base + ((long long)(t0 + row) * stride) * (int)sizeof(T) + col;
    const long long next = stride * (kRows * (int)sizeof(T));
    if (rows == kS && chans == kC) {
#pragma unroll
      for (int s = 0; s < kS; s += kRows) {
#pragma unroll
        for (int o = 0; o < kOver; ++o) copy_async<kMode == 16 ? 16 : 4>(to + s * kRow + o * 32 * kMode, from + o * 32 * kMode, kMode);
        from += next;
      }
      return;
    }
#pragma unroll
    for (int s = 0; s < kS; s += kRows) {
#pragma unroll
      for (int o = 0; o < kOver; ++o) {
        const int left = min(max(chans * (int)sizeof(T) - col - o * 32 * kMode, 0), kMode);
        const int n = s + row < rows ? left : 0;
        copy_async<kMode == 16 ? 16 : 4>(to + s * kRow + o * 32 * kMode, n ? from + o * 32 * kMode : base, n);
      }
      from += next;
    }
  }
};

// The padding (bits 0 ..) and resets (bits 16 ..) of a segment, one byte to a lane; steps behind the end are padded.  The byte is asked
// for a round before flags_of() looks at it, and nothing may look at it earlier: a test beside the load, which the compiler makes when
// it can, waits for memory in every round (B = 8, L = 4096, D = 2048 with resets: forward 89 us, backward 141, without 76 and 127).
__device__ __forceinline__ unsigned flag_byte(const RecArgs& a, int b, int t0, int steps, int lane) {
  const int s = lane & 15, t = t0 + s;
  const unsigned char* mask = lane < 16 ? a.pad : a.reset;
  unsigned v = lane < 16 && s < steps && t >= a.L;
  if (mask != nullptr && s < steps && t < a.L) v = mask[b * a.msb + t * a.msl];
  return v;
}
__device__ __forceinline__ unsigned flags_of(unsigned byte) {
  asm volatile("" : "+r"(byte));
  return __ballot_sync(0xffffffffu, byte != 0);
}

// whether a gate of the warp's segment is closed that far; padded steps do not count
template <typename T, int kS>
__device__ __forceinline__ bool any_closed(const T* f, unsigned flags) {
  if constexpr (kSides<T>) {
    return false;
  } else {
    LeastGate<T> least;
    if ((flags & 0xffffu) == 0) {
#pragma unroll
      for (int s = 0; s < kS; ++s) least.see(f + s * kC);
    } else {
#pragma unroll 1
      for (int s = 0; s < kS; ++s)
        if (!((flags >> s) & 1u)) least.see(f + s * kC);
    }
    return __any_sync(0xffffffffu, least.closed());
  }
}
template <int kS>
__device__ __forceinline__ bool all_padded(unsigned flags) {
  return (flags & ((1u << kS) - 1u)) == (1u << kS) - 1u;
}
// Resets alone: the walks then take them by selections instead of branches (a block waits for its slowest warp, and one of its eight
// segments has a reset in every sixth round at documents of 700 steps).
__device__ __forceinline__ bool only_resets(unsigned flags) { return flags != 0 && (flags & 0xffffu) == 0; }
// whether a reset lies at step s of a segment; at it or before; at it or behind
__device__ __forceinline__ bool cut_at(unsigned flags, int s) { return (flags >> (16 + s)) & 1u; }
__device__ __forceinline__ bool cut_until(unsigned flags, int s) { return (flags >> 16) & ((2u << s) - 1u); }
__device__ __forceinline__ bool cut_from(unsigned flags, int s) { return flags >> (16 + s); }
template <int kS>
__device__ __forceinline__ bool idle(unsigned flags) {   // all padded, and no reset
  return flags == (1u << kS) - 1u;
}

// Where a warp is: its sequence (-1: behind the last), the tile's first channel, its place in time.  Serial: a warp walks a sequence's
// tile by itself, and nobody waits for anybody, which is what many short sequences take.
struct Place {
  int w, lane, b, size, rank, c0;
  __device__ __forceinline__ Place(const RecArgs& a, bool serial) {
    w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (serial) {
      const int unit = blockIdx.x * kW + w;
      b = unit < a.units ? unit / a.tiles : -1;
      c0 = (unit % a.tiles) * kC, size = 1, rank = 0;
    } else {
      b = blockIdx.y, size = cluster_size(), rank = size > 1 ? cluster_rank() : 0, c0 = (blockIdx.x / size) * kC;
    }
  }
};

// What the warps of a block, and the blocks of a cluster, tell one another.  Two of each: a place is written again only after every
// reader has taken part in the round between.
struct Post {
  float4 warps[2][kW][32], blocks[2][8][32];
  f32x2 carry[2][32];
  uint64_t bar[2];
  unsigned odd;   // lanes of the cluster (in its first block) that have seen values that are not finite
};
// (of a multiprocessor's 228 KB of shared memory a block takes 1 KB besides)
template <typename T, bool kGate, bool kBack>
constexpr bool fits() {
  constexpr int block = kRingBytes<T, kGate, kBack> + (int)sizeof(Post) + 1024;
  return kResident<T, kGate, kBack> == (2 * block <= (228 << 10) ? 2 : 1);
}

// Every warp's map -> the state that enters each; `carry` is the state that enters the whole stride, then the next one (in a block
// by itself: in the last warp alone, the others find it here in the next round).  kDir > 0: in the order of warps and ranks, else
// the other way.  A warp reads the maps before its own only: all eight in every warp are a third of the shared memory traffic, and
// their loads, issued together, crowd out the registers.  Returns false once a wait has given up: the rounds go on, without
// waiting.
template <int kDir, bool kReset, bool kFour>
__device__ __forceinline__ bool exchange(const Map& own, f32x2& carry, f32x2& in, Post& post, int round, int w, int lane, int rank, int size,
                                         bool alive) {
  const int at = round & 1, place = kDir > 0 ? w : kW - 1 - w;
  post.warps[at][w][lane] = own.words();
  __syncthreads();
  if (size == 1) {
    if (round > 0 && place < kW - 1) carry = post.carry[at][lane];
    in = carry;
#pragma unroll
    for (int k = 0; k < kW - 1; ++k) {
      if (k >= place) break;
      in = Map::of(post.warps[at][kDir > 0 ? k : kW - 1 - k][lane]).template operator()<kReset>(in);
    }
    if (place == kW - 1) {
      carry = own.operator()<kReset>(in);
      post.carry[at ^ 1][lane] = carry;
    }
    return true;
  }
  Map pre = {pack2(1.f, 1.f), pack2(0.f, 0.f)};
#pragma unroll
  for (int k = 0; k < kW - 1; ++k) {
    if (k >= place) break;
    const Map m = Map::of(post.warps[at][kDir > 0 ? k : kW - 1 - k][lane]);
    pre = k == 0 ? m : then<kReset>(pre, m);
  }
  if (round == 0) cluster_wait();
  if (place == kW - 1) {
    if (lane == 0) mbar_expect_tx(&post.bar[at], size * 512);
    const float4 v = then<kReset>(pre, own).words();
    for (int r = 0; r < size; ++r) send(&post.blocks[at][rank][lane], &post.bar[at], r, v);
  }
  if (place == kW - 1) {
    if (alive) alive = received(&post.bar[at], (round >> 1) & 1);
    if constexpr (kFour) {   // (maps read four at a time)
#pragma unroll
      for (int k0 = 0; k0 < 8; k0 += 4) {
        if (k0 >= size) break;
        float4 m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = kDir > 0 ? k0 + k : size - 1 - k0 - k;
          if (k0 + k < size) m[k] = post.blocks[at][r][lane];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = kDir > 0 ? k0 + k : size - 1 - k0 - k;
          if (r == rank) in = carry;
          if (k0 + k < size) carry = Map::of(m[k]).template operator()<kReset>(carry);
        }
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < size; ++k) {
        const int r = kDir > 0 ? k : size - 1 - k;
        if (r == rank) in = carry;
        carry = Map::of(post.blocks[at][r][lane]).template operator()<kReset>(carry);
      }
    }
    post.carry[at][lane] = in;
  }
  __syncthreads();
  in = pre.operator()<kReset>(post.carry[at][lane]);
  return alive;
}

// ---- values that are not finite ----------------------------------------------------------------
// adds to what a lane has seen: NaN once it was not finite
__device__ __forceinline__ float seen(float odd, f32x2 v) {
  float a, b;
  unpack2(v, a, b);
  return fmaf(a, 0.f, fmaf(b, 0.f, odd));
}
__device__ __forceinline__ unsigned odd_lanes(float odd) {
  return __ballot_sync(0xffffffffu, isnan(odd));
}
// The same of all warps of a block, or of a cluster for its first block, which then may write over what the others have written.
__device__ __forceinline__ unsigned odd_lanes(float odd, Post& post, const Place& p) {
  const unsigned own = odd_lanes(odd);
  if (own && p.lane == 0) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(&post.odd)));
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(at), "r"(own) : "memory");
  }
  if (p.size > 1) {   // (nor does any block's shared memory go before all are through)
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  return post.odd;
}

// which of a lane's values in a run of steps (bit 2 s + j) are not finite; plain loads, as this call has written them
template <int kS, typename T>
__device__ __forceinline__ unsigned not_finite(const T* p, long long stride, int rows, int n) {
  float v[kS][2];
#pragma unroll
  for (int s = 0; s < kS; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) v[s][j] = s < rows && j < n ? Elem<T>::ld_shared(p + s * stride + j) : 0.f;
  unsigned r = 0;
#pragma unroll
  for (int s = 0; s < kS; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) r |= (isfinite(v[s][j]) ? 0u : 1u) << (2 * s + j);
  return r;
}
// the values that `which` asks for
template <typename T>
__device__ __forceinline__ void mend(T* p, unsigned which, const float (&v)[2]) {
  if (which & 1u) Elem<T>::st(p, v[0]);
  if (which & 2u) Elem<T>::st(p + 1, v[1]);
}
__device__ __forceinline__ f32x2 unless_finite(f32x2 v, f32x2 other) {
  float a, b, c, d;
  unpack2(v, a, b), unpack2(other, c, d);
  return pack2(isfinite(a) ? a : c, isfinite(b) ? b : d);
}

// One step of one channel, any values: the gate's two sides, or with an input gate its side and slope, and what it makes of them.
template <typename T, bool kGate>
struct Step {
  float c, side, into, slope;   // side: of the forget gate, the smaller; into: the input gate
  bool open;
  __device__ __forceinline__ Step(float f, float i) {
    float s;
    unpack2(gate_side2<T>(pack2(f, kGate ? i : 0.f)), c, s);
    open = signbit(c), side = fabsf(c), into = signbit(s) ? 1.f + s : s, slope = fabsf(s) * (1.f - fabsf(s));
  }
  // a gate of this value on u; infinite u as it is (an infinity less a part of it, or 0 times it where the gate has underflowed, is
  // NaN), NaN where the gate is
  static __device__ __forceinline__ float on(float r, float u, float gate) { return isinf(u) ? fmaf(gate, 0.f, u) : r; }
  __device__ __forceinline__ float keep(float u) const { return on(fmaf(c, u, open ? u : 0.f), u, c); }
  __device__ __forceinline__ float leak(float u) const { return on(fmaf(-c, u, open ? 0.f : u), u, c); }
  __device__ __forceinline__ float enter(float u) const { return kGate ? on(into * u, u, into) : leak(u); }
  __device__ __forceinline__ float next(float h, float x) const { return keep(h) + enter(x); }
};

// NaN in all of these channels, to the end: there is no reset
__device__ __forceinline__ bool nothing_left(const RecArgs& a, bool mine, const float (&v)[2], int n) {
  return a.reset == nullptr && __all_sync(0xffffffffu, !mine || (isnan(v[0]) && (n < 2 || isnan(v[1]))));
}

// The forward of some lanes' channels, step by step, by a warp; the state behind the last one.  ring: tiles of the warp's own.
template <typename T, bool kGate, int kMode>
__device__ __noinline__ f32x2 forward_again(const RecArgs& a, char* ring, int b, int c0, unsigned lanes) {
  constexpr int kS = kForwardSteps<T>, kSave = kBackSteps<T, kGate>;
  using Op = Tile<T, kS, kMode>;
  const int lane = threadIdx.x & 31, chans = min(a.D - c0, kC), n = min(max(chans - 2 * lane, 0), 2), c = c0 + 2 * lane;
  const int segs = (a.L + kSave - 1) / kSave;
  const bool mine = (lanes >> lane) & 1u;
  const T* op = reinterpret_cast<const T*>(ring) + 2 * lane;
  float h[2] = {0.f, 0.f};
  for (int j = 0; j < n; ++j) h[j] = a.h_in ? a.h_in[(long long)b * a.D + c + j] : 0.f;
#pragma unroll 1
  for (int t0 = 0; t0 < a.L; t0 += kS) {
    const int rows = min(kS, a.L - t0);
    const unsigned flags = flags_of(flag_byte(a, b, t0, kS, lane));   // (and the tile before has been read)
    Op::fetch(ring, (const T*)a.x + b * a.xsb + c0, a.xsl, t0, rows, chans, lane);
    Op::fetch(ring + Op::kBytes, (const T*)a.f + b * a.fsb + c0, a.fsl, t0, rows, chans, lane);
    if (kGate) Op::fetch(ring + 2 * Op::kBytes, (const T*)a.i + b * a.isb + c0, a.isl, t0, rows, chans, lane);
    copies_commit();
    T* y = (T*)a.y + b * a.ysb + t0 * a.ysl + c;
    unsigned which = mine ? not_finite<kS>(y, a.ysl, rows, n) : 0u;
    copies_wait<0>();
    __syncwarp();
    if (mine) {
#pragma unroll 1
      for (int s = 0; s < rows; ++s) {
        if (a.starts && s % kSave == 0) {
          float* p = a.starts + ((long long)b * segs + (t0 + s) / kSave) * a.D + c;
          mend(p, not_finite<1>(p, 0, 1, n), h);
        }
        if ((flags >> (16 + s)) & 1u) h[0] = h[1] = 0.f;
        if (!((flags >> s) & 1u)) {
          float x[2], f[2], i[2] = {0.f, 0.f};
          unpack2(two(op + s * kC), x[0], x[1]), unpack2(two(op + (kS + s) * kC), f[0], f[1]);
          if (kGate) unpack2(two(op + (2 * kS + s) * kC), i[0], i[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) h[j] = Step<T, kGate>(f[j], i[j]).next(h[j], x[j]);
          mend(y, which >> (2 * s), h);
        }
        y += a.ysl;
      }
    }
    if (nothing_left(a, mine, h, n)) break;
  }
  return pack2(h[0], h[1]);
}

// The backward: the states of a segment from the saved one, then its steps in reverse; the gradient of the state that came in.
template <typename T, bool kGate, int kMode>
__device__ __noinline__ f32x2 backward_again(const RecArgs& a, char* ring, int b, int c0, unsigned lanes) {
  constexpr int kS = kBackSteps<T, kGate>, kOps = kGate ? 4 : 3;
  using Op = Tile<T, kS, kMode>;
  static_assert(kS * kC * (int)sizeof(float) <= (kStages - 1) * kOps * Op::kBytes, "states of a segment behind the operands");
  const int lane = threadIdx.x & 31, chans = min(a.D - c0, kC), n = min(max(chans - 2 * lane, 0), 2), c = c0 + 2 * lane;
  const int segs = (a.L + kS - 1) / kS;
  const bool mine = (lanes >> lane) & 1u;
  const T* op = reinterpret_cast<const T*>(ring) + 2 * lane;
  float2* before = reinterpret_cast<float2*>(ring + kOps * Op::kBytes) + lane;
  float q[2] = {0.f, 0.f};
  for (int j = 0; j < n; ++j) q[j] = a.dh_out ? a.dh_out[(long long)b * a.D + c + j] : 0.f;
#pragma unroll 1
  for (int k = segs - 1; k >= 0; --k) {
    const int t0 = k * kS, rows = min(kS, a.L - t0);
    const unsigned flags = flags_of(flag_byte(a, b, t0, kS, lane));
    Op::fetch(ring, (const T*)a.x + b * a.xsb + c0, a.xsl, t0, rows, chans, lane);
    Op::fetch(ring + Op::kBytes, (const T*)a.f + b * a.fsb + c0, a.fsl, t0, rows, chans, lane);
    Op::fetch(ring + 2 * Op::kBytes, (const T*)a.dy + b * a.gsb + c0, a.gsl, t0, rows, chans, lane);
    if (kGate) Op::fetch(ring + 3 * Op::kBytes, (const T*)a.i + b * a.isb + c0, a.isl, t0, rows, chans, lane);
    copies_commit();
    T *dx = (T*)a.dx + b * a.dxb + t0 * a.dxl + c, *df = (T*)a.df + b * a.dfb + t0 * a.dfl + c;
    T* di = kGate ? (T*)a.di + b * a.dib + t0 * a.dil + c : nullptr;
    unsigned bad_x = 0, bad_f = 0, bad_i = 0;
    float h[2] = {0.f, 0.f};
    if (mine) {
      for (int j = 0; j < n; ++j) h[j] = a.starts[((long long)b * segs + k) * a.D + c + j];
      bad_x = not_finite<kS>(dx, a.dxl, rows, n), bad_f = not_finite<kS>(df, a.dfl, rows, n);
      if (kGate) bad_i = not_finite<kS>(di, a.dil, rows, n);
    }
    copies_wait<0>();
    __syncwarp();
    auto gates = [&](int s, float (&f)[2], float (&i)[2]) {
      unpack2(two(op + (kS + s) * kC), f[0], f[1]);
      i[0] = i[1] = 0.f;
      if (kGate) unpack2(two(op + (3 * kS + s) * kC), i[0], i[1]);
    };
    if (mine) {
#pragma unroll 1
      for (int s = 0; s < rows; ++s) {
        if ((flags >> (16 + s)) & 1u) h[0] = h[1] = 0.f;
        before[s * (kC / 2)] = make_float2(h[0], h[1]);
        if ((flags >> s) & 1u) continue;
        float x[2], f[2], i[2];
        gates(s, f, i);
        unpack2(two(op + s * kC), x[0], x[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) h[j] = Step<T, kGate>(f[j], i[j]).next(h[j], x[j]);
      }
#pragma unroll 1
      for (int s = rows - 1; s >= 0; --s) {
        if (!((flags >> s) & 1u)) {
          const float2 hs = before[s * (kC / 2)];
          float x[2], f[2], i[2], g[2], ox[2], of[2], oi[2];
          gates(s, f, i);
          unpack2(two(op + s * kC), x[0], x[1]), unpack2(two(op + (2 * kS + s) * kC), g[0], g[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Step<T, kGate> e(f[j], i[j]);
            const float u = q[j] + g[j], rest = e.on(fmaf(-e.side, u, u), u, e.c), from = j ? hs.y : hs.x;
            // (half of h - x, which may be past the largest value, and twice the side)
            const float half = kGate ? 0.5f * from : fmaf(0.5f, from, -0.5f * x[j]);
            ox[j] = e.enter(u), of[j] = (half * rest) * (2.f * e.side), oi[j] = (x[j] * u) * e.slope;
            q[j] = e.keep(u);
          }
          mend(dx + s * a.dxl, bad_x >> (2 * s), ox);
          mend(df + s * a.dfl, bad_f >> (2 * s), of);
          if (kGate) mend(di + s * a.dil, bad_i >> (2 * s), oi);
        }
        if ((flags >> (16 + s)) & 1u) q[0] = q[1] = 0.f;
      }
    }
    if (nothing_left(a, mine, q, n)) break;
  }
  return pack2(q[0], q[1]);
}

// ---- forward ---------------------------------------------------------------------------------
template <typename T, bool kGate, int kMode, bool kSerial>
__global__ void __launch_bounds__(kW * 32, kResident<T, kGate, false>) rec_fwd_kernel(const __grid_constant__ RecArgs a) {
  constexpr int kS = kForwardSteps<T>, kSave = kBackSteps<T, kGate>, kOps = kGate ? 3 : 2;
  using Op = Tile<T, kS, kMode>;
  static_assert(fits<T, kGate, false>(), "as many blocks as cluster_of reckons with");
  constexpr bool kPair = kMode == 16 || (kMode == 4 && sizeof(T) == 2);
  constexpr bool kFour = kMode == 16 && sizeof(T) == 2;   // (the other forms and the backward have no registers left for it)
  extern __shared__ __align__(16) char smem[];
  __shared__ Post post;
  const Place p(a, kSerial);
  if (kSerial && p.b < 0) return;
  const int w = p.w, lane = p.lane, b = p.b, size = p.size, rank = p.rank, c0 = p.c0, chans = min(a.D - c0, kC);
  const int n = min(max(chans - 2 * lane, 0), 2);
  const long long state = (long long)b * a.D + c0 + 2 * lane;
  const T *x = (const T*)a.x + b * a.xsb + c0, *f = (const T*)a.f + b * a.fsb + c0, *i = kGate ? (const T*)a.i + b * a.isb + c0 : nullptr;
  T* y = (T*)a.y + b * a.ysb + c0 + 2 * lane;
  char* ring = smem + w * (kStages * kOps * Op::kBytes);
  const int stride = kSerial ? kS : size * kW * kS, rounds = (a.L + stride - 1) / stride, segs = (a.L + kSave - 1) / kSave;
  const bool reset = a.reset != nullptr, whole = kPair && chans == kC;
  bool alive = true;

  auto first = [&](int k) { return kSerial ? k * kS : (k * size + rank) * (kW * kS) + w * kS; };
  unsigned flag = flag_byte(a, b, first(0), kS, lane);
  // sets round k's tile on its way and returns its padding and resets, which came a round earlier: a segment of padding is not read
  auto fetch = [&](int k) {
    const unsigned flags = flags_of(flag);
    if (k + 1 < rounds) flag = flag_byte(a, b, first(k + 1), kS, lane);
    const int t0 = first(k), rows = min(max(a.L - t0, 0), kS);
    char* at = ring + (k % kStages) * (kOps * Op::kBytes);
    if (k < rounds && !all_padded<kS>(flags)) {
      const int t = rows > 0 ? t0 : 0;
      Op::fetch(at, x, a.xsl, t, rows, chans, lane);
      Op::fetch(at + Op::kBytes, f, a.fsl, t, rows, chans, lane);
      if (kGate) Op::fetch(at + 2 * Op::kBytes, i, a.isl, t, rows, chans, lane);
    }
    copies_commit();
    return flags;
  };

  if (!kSerial && threadIdx.x == 0) post.odd = 0;   // (added to behind the first round's barriers)
  if (!kSerial && size > 1) {
    if (threadIdx.x == 0) {
      mbar_init(&post.bar[0], 1);
      mbar_init(&post.bar[1], 1);
      mbar_fence_init();
    }
    cluster_arrive();   // (every block has begun, and its barriers are there, before another writes to it)
  }
  f32x2 carry = get_state(a.h_in ? a.h_in + state : nullptr, n, a.pairs);
  float odd = 0.f;   // see seen()
  unsigned flags, next = fetch(0);
  for (int k = 0; k < rounds; ++k) {
    flags = next;
    __syncwarp();   // (the stage that is fetched into next has been read by every lane)
    next = fetch(k + 1);
    copies_wait<kStages - 1>();
    __syncwarp();
    const T* op = reinterpret_cast<const T*>(ring + (k % kStages) * (kOps * Op::kBytes)) + 2 * lane;
    Map loc[kS];
    f32x2 h = pack2(0.f, 0.f), A = pack2(1.f, 1.f);
    const bool closed = (flags & 0xffffu) == 0 && any_closed<T, kS>(op + kS * kC, 0u);   // (padded ones take the sides in any case)
    auto step = [&](int s, auto sides) {
      const T* fs = op + kS * kC + s * kC;
      const f32x2 xv = two(op + s * kC);
      f32x2 in = pack2(0.f, 0.f), none;
      if (kGate) in = gate2<T, false>(two(op + 2 * kS * kC + s * kC), none);
      if constexpr (decltype(sides)::value) {
        const f32x2 c = gate_side2<T>(two(fs)), open = open_bits(c);
        h = kGate ? fma2(in, xv, pass(c, open, h)) : fma2(c, sub2(h, xv), either(open, h, xv));
        A = pass(c, open, A);
      } else {
        const f32x2 nl = minus_leak2<T>(two(fs));
        h = kGate ? fma2(in, xv, fma2(nl, h, h)) : fma2(nl, sub2(h, xv), h);
        A = fma2(nl, A, A);
      }
    };
    constexpr std::bool_constant<kSides<T>> usual;
    auto by_step = [&] {   // with the gates' sides, padded steps among them
      h = pack2(0.f, 0.f), A = pack2(1.f, 1.f);
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        if ((flags >> (16 + s)) & 1u) odd = seen(odd, h), h = pack2(0.f, 0.f), A = minus_zero();
        if (!((flags >> s) & 1u)) {
          const f32x2 before = A;
          step(s, std::true_type{});
          if (before == minus_zero()) A = minus_zero();
        }
        loc[s] = {A, h};
      }
    };
    if (flags == 0 && !closed) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        step(s, usual);
        loc[s] = {A, h};
      }
    } else if (!kSides<T> && flags == 0) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        step(s, std::true_type{});
        loc[s] = {A, h};
      }
    } else if (only_resets(flags) && !closed) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        odd = seen(odd, h);
        h = cut_at(flags, s) ? pack2(0.f, 0.f) : h;
        step(s, usual);
        A = cut_until(flags, s) ? minus_zero() : A;
        loc[s] = {A, h};
      }
    } else if (idle<kS>(flags)) {
      loc[kS - 1] = {A, h};
    } else {
      by_step();
    }
    f32x2 in;
    if (kSerial) {
      in = carry;
      const Map m = idle<kS>(flags) ? Map{pack2(1.f, 1.f), pack2(0.f, 0.f)} : loc[kS - 1];
      carry = reset ? m.operator()<true>(in) : m.operator()<false>(in);
    } else {
      alive = reset ? exchange<1, true, kFour>(loc[kS - 1], carry, in, post, k, w, lane, rank, size, alive)
                    : exchange<1, false, kFour>(loc[kS - 1], carry, in, post, k, w, lane, rank, size, alive);
    }
    odd = seen(seen(odd, h), in);
    const int t0 = first(k);
    if (a.starts) {
#pragma unroll
      for (int s = 0; s < kS; s += kSave) {
        const f32x2 from = s == 0 || idle<kS>(flags) ? in : loc[s > 0 ? s - 1 : 0].operator()<true>(in);
        if (t0 + s < a.L) put_state(a.starts + ((long long)b * segs + (t0 + s) / kSave) * a.D + c0 + 2 * lane, from, n, a.pairs);
      }
    }
    T* yt = y + t0 * a.ysl;
    if (flags == 0 && whole) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        put<kPair>(yt, loc[s].operator()<false>(in), 2);
        yt += a.ysl;
      }
    } else if (only_resets(flags) && whole) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        put<kPair>(yt, cut_until(flags, s) ? loc[s].h : loc[s].operator()<false>(in), 2);
        yt += a.ysl;
      }
    } else if (idle<kS>(flags)) {
#pragma unroll 4
      for (int s = 0; s < min(kS, a.L - t0); ++s) {
        put<kPair>(yt, pack2(0.f, 0.f), n);
        yt += a.ysl;
      }
    } else {
#pragma unroll
      for (int s = 0; s < kS; ++s)
        if (t0 + s < a.L) put<kPair>(yt + s * a.ysl, (flags >> s) & 1u ? pack2(0.f, 0.f) : loc[s].operator()<true>(in), n);
    }
  }
  const Place e = kSerial ? p : Place(a, false);   // (again: it costs registers through the rounds)
  const unsigned again = kSerial ? odd_lanes(odd) : odd_lanes(odd, post, e);
  if (kSerial || (e.rank == 0 && e.w == kW - 1)) {
    const int n = min(max(a.D - e.c0 - 2 * e.lane, 0), 2);
    if (again) {
      const f32x2 last = forward_again<T, kGate, kMode>(a, smem + e.w * (kStages * kOps * Op::kBytes), e.b, e.c0, again);
      if ((again >> e.lane) & 1u) carry = unless_finite(carry, last);
    }
    if (a.h_out) put_state(a.h_out + (long long)e.b * a.D + e.c0 + 2 * e.lane, carry, n, a.pairs);
  }
}

// ---- backward --------------------------------------------------------------------------------
template <typename T, bool kGate, int kMode, bool kSerial>
__global__ void __launch_bounds__(kW * 32, kResident<T, kGate, true>) rec_bwd_kernel(const __grid_constant__ RecArgs a) {
  constexpr int kS = kBackSteps<T, kGate>, kOps = kGate ? 4 : 3;
  using Op = Tile<T, kS, kMode>;
  static_assert(fits<T, kGate, true>(), "as many blocks as cluster_of reckons with");
  constexpr bool kPair = kMode == 16 || (kMode == 4 && sizeof(T) == 2);
  extern __shared__ __align__(16) char smem[];
  __shared__ Post post;
  const Place p(a, kSerial);
  if (kSerial && p.b < 0) return;
  const int w = p.w, lane = p.lane, b = p.b, size = p.size, rank = p.rank, c0 = p.c0, chans = min(a.D - c0, kC);
  const int n = min(max(chans - 2 * lane, 0), 2);
  const long long state = (long long)b * a.D + c0 + 2 * lane;
  const T *x = (const T*)a.x + b * a.xsb + c0, *f = (const T*)a.f + b * a.fsb + c0, *dy = (const T*)a.dy + b * a.gsb + c0;
  const T* i = kGate ? (const T*)a.i + b * a.isb + c0 : nullptr;
  T *dx = (T*)a.dx + b * a.dxb + c0 + 2 * lane, *df = (T*)a.df + b * a.dfb + c0 + 2 * lane;
  T* di = kGate ? (T*)a.di + b * a.dib + c0 + 2 * lane : nullptr;
  char* ring = smem + w * (kStages * kOps * Op::kBytes);
  const int stride = kSerial ? kS : size * kW * kS, rounds = (a.L + stride - 1) / stride, segs = (a.L + kS - 1) / kS;
  const bool reset = a.reset != nullptr, whole = kPair && chans == kC;
  bool alive = true;

  f32x2 start = pack2(0.f, 0.f);
  auto first = [&](int k) { return kSerial ? (rounds - 1 - k) * kS : ((rounds - 1 - k) * size + rank) * (kW * kS) + w * kS; };   // (round k is the k-th from the end)
  unsigned flag = flag_byte(a, b, first(0), kS, lane);
  auto fetch = [&](int k) {
    const unsigned flags = flags_of(flag);
    if (k + 1 < rounds) flag = flag_byte(a, b, first(k + 1), kS, lane);
    const int t0 = first(k), rows = min(max(a.L - t0, 0), kS);
    char* at = ring + (k % kStages) * (kOps * Op::kBytes);
    if (k < rounds && !all_padded<kS>(flags)) {
      const int t = rows > 0 ? t0 : 0;
      Op::fetch(at, x, a.xsl, t, rows, chans, lane);
      Op::fetch(at + Op::kBytes, f, a.fsl, t, rows, chans, lane);
      Op::fetch(at + 2 * Op::kBytes, dy, a.gsl, t, rows, chans, lane);
      if (kGate) Op::fetch(at + 3 * Op::kBytes, i, a.isl, t, rows, chans, lane);
      if (rows > 0) start = get_state(a.starts + ((long long)b * segs + t0 / kS) * a.D + c0 + 2 * lane, n, a.pairs);
    }
    copies_commit();
    return flags;
  };

  if (!kSerial && threadIdx.x == 0) post.odd = 0;   // (added to behind the first round's barriers)
  if (!kSerial && size > 1) {
    if (threadIdx.x == 0) {
      mbar_init(&post.bar[0], 1);
      mbar_init(&post.bar[1], 1);
      mbar_fence_init();
    }
    cluster_arrive();
  }
  f32x2 carry = get_state(a.dh_out ? a.dh_out + state : nullptr, n, a.pairs);
  float odd = 0.f;   // see seen()
  unsigned flags, next = fetch(0);
  for (int k = 0; k < rounds; ++k) {
    flags = next;
    const f32x2 enters = start;
    f32x2 h = enters;
    __syncwarp();
    next = fetch(k + 1);
    copies_wait<kStages - 1>();
    __syncwarp();
    const T* op = reinterpret_cast<const T*>(ring + (k % kStages) * (kOps * Op::kBytes)) + 2 * lane;
    const T* gy = op + 2 * kS * kC;
    // c: minus the leak, with `sides` the smaller side of the gate; v: h_{t-1} - x, with an input gate h_{t-1}
    f32x2 c[kS], v[kS], gate[kGate ? kS : 1], slope[kGate ? kS : 1];
    const bool closed = any_closed<T, kS>(op + kS * kC, flags);
    auto state_step = [&](int s, auto sides) {
      const T* fs = op + kS * kC + s * kC;
      const f32x2 xv = two(op + s * kC);
      if (kGate) gate[s] = gate2<T, true>(two(op + 3 * kS * kC + s * kC), slope[s]);
      v[s] = kGate ? h : sub2(h, xv);
      if constexpr (decltype(sides)::value) {
        c[s] = gate_side2<T>(two(fs));
        const f32x2 open = open_bits(c[s]);
        h = kGate ? fma2(gate[s], xv, pass(c[s], open, h)) : fma2(c[s], v[s], either(open, h, xv));
      } else {
        c[s] = minus_leak2<T>(two(fs));
        h = kGate ? fma2(gate[s], xv, fma2(c[s], h, h)) : fma2(c[s], v[s], h);
      }
    };
    Map m = {pack2(1.f, 1.f), pack2(0.f, 0.f)};
    auto grad_step = [&](int s, auto sides) {
      const f32x2 g = add2(m.h, two(gy + s * kC));
      if constexpr (decltype(sides)::value) {
        const f32x2 open = open_bits(c[s]);
        m.h = pass(c[s], open, g);
        m.a = pass(c[s], open, m.a);
      } else {
        m.h = fma2(c[s], g, g);
        m.a = fma2(c[s], m.a, m.a);
      }
    };
    constexpr std::bool_constant<kSides<T>> usual;
    auto by_step = [&](auto sides) {   // padded steps among them
      h = enters;
      m = {pack2(1.f, 1.f), pack2(0.f, 0.f)};
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        if ((flags >> (16 + s)) & 1u) odd = seen(odd, h), h = pack2(0.f, 0.f);
        c[s] = v[s] = pack2(0.f, 0.f);
        if (kGate) gate[s] = slope[s] = pack2(0.f, 0.f);
        if (!((flags >> s) & 1u)) state_step(s, sides);
      }
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) {
        if (!((flags >> s) & 1u)) {
          const f32x2 before = m.a;
          grad_step(s, sides);
          if (before == minus_zero()) m.a = minus_zero();
        }
        if ((flags >> (16 + s)) & 1u) odd = seen(odd, m.h), m = {minus_zero(), pack2(0.f, 0.f)};
      }
    };
    if (flags == 0 && !closed) {
#pragma unroll
      for (int s = 0; s < kS; ++s) state_step(s, usual);
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) grad_step(s, usual);
    } else if (!kSides<T> && flags == 0) {
#pragma unroll
      for (int s = 0; s < kS; ++s) state_step(s, std::true_type{});
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) grad_step(s, std::true_type{});
    } else if (only_resets(flags) && !closed) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        odd = seen(odd, h);
        h = cut_at(flags, s) ? pack2(0.f, 0.f) : h;
        state_step(s, usual);
      }
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) {
        grad_step(s, usual);
        odd = seen(odd, m.h);
        m.h = cut_at(flags, s) ? pack2(0.f, 0.f) : m.h;
        m.a = cut_from(flags, s) ? minus_zero() : m.a;
      }
    } else if (!idle<kS>(flags)) {
      if (!closed)
        by_step(usual);
      else if constexpr (!kSides<T>)
        by_step(std::true_type{});
    }
    f32x2 q;
    if (kSerial) {
      q = carry;
      carry = reset ? m.operator()<true>(q) : m.operator()<false>(q);
    } else {
      alive = reset ? exchange<-1, true, false>(m, carry, q, post, k, w, lane, rank, size, alive)
                    : exchange<-1, false, false>(m, carry, q, post, k, w, lane, rank, size, alive);
    }
    if (!idle<kS>(flags)) odd = seen(odd, h);   // (an idle segment has not read its state)
    odd = seen(seen(odd, m.h), q);
    const int t0 = first(k);
    T *xt = dx + t0 * a.dxl, *ft = df + t0 * a.dfl, *it = kGate ? di + t0 * a.dil : nullptr;
    auto out_step = [&](int s, auto sides, bool pad, int count) {
      const f32x2 g = add2(q, two(gy + s * kC));
      f32x2 ox, of, oi = pack2(0.f, 0.f);
      // (the gate's side and the slope, which may be subnormal, come last: a product of theirs would be rounded to few bits first)
      if constexpr (decltype(sides)::value) {
        const f32x2 open = open_bits(c[s]), na = c[s] | 0x8000000080000000ull;
        if (!pad) q = pass(c[s], open, g);
        ox = kGate ? mul2(gate[s], g) : hold_back(c[s], open, g);
        of = mul2(mul2(v[s], fma2(na, g, g)), neg2(na));
      } else {
        if (!pad) q = fma2(c[s], g, g);
        ox = kGate ? mul2(gate[s], g) : neg2(mul2(c[s], g));
        of = neg2(mul2(mul2(v[s], q), c[s]));
      }
      if (kGate) oi = mul2(mul2(two(op + s * kC), g), slope[s]);
      if (pad) ox = of = oi = pack2(0.f, 0.f);
      put<kPair>(xt + s * a.dxl, ox, count);
      put<kPair>(ft + s * a.dfl, of, count);
      if (kGate) put<kPair>(it + s * a.dil, oi, count);
    };
    if (flags == 0 && whole && !closed) {
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) out_step(s, usual, false, 2);
    } else if (!kSides<T> && flags == 0 && whole) {
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) out_step(s, std::true_type{}, false, 2);
    } else if (only_resets(flags) && whole && !closed) {
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) {
        out_step(s, usual, false, 2);
        q = cut_at(flags, s) ? pack2(0.f, 0.f) : q;
      }
    } else if (idle<kS>(flags)) {
#pragma unroll 4
      for (int s = 0; s < min(kS, a.L - t0); ++s) {
        put<kPair>(xt, pack2(0.f, 0.f), n);
        put<kPair>(ft, pack2(0.f, 0.f), n);
        if (kGate) put<kPair>(it, pack2(0.f, 0.f), n);
        xt += a.dxl, ft += a.dfl;
        if (kGate) it += a.dil;
      }
    } else {
#pragma unroll
      for (int s = kS - 1; s >= 0; --s) {
        if (t0 + s < a.L) out_step(s, std::true_type{}, (flags >> s) & 1u, n);   // (minus a leak is the side of a gate that stands open)
        if ((flags >> (16 + s)) & 1u) q = pack2(0.f, 0.f);
      }
    }
  }
  const Place e = kSerial ? p : Place(a, false);   // (again: it costs registers through the rounds)
  const unsigned again = kSerial ? odd_lanes(odd) : odd_lanes(odd, post, e);
  if (kSerial || (e.rank == 0 && e.w == 0)) {
    const int n = min(max(a.D - e.c0 - 2 * e.lane, 0), 2);
    if (again) {
      const f32x2 last = backward_again<T, kGate, kMode>(a, smem + e.w * (kStages * kOps * Op::kBytes), e.b, e.c0, again);
      if ((again >> e.lane) & 1u) carry = unless_finite(carry, last);
    }
    if (a.dh_in) put_state(a.dh_in + (long long)e.b * a.D + e.c0 + 2 * e.lane, carry, n, a.pairs);
  }
}

// ---- single step -----------------------------------------------------------------------------
// A value a thread: at serving sizes (64 x 2048) some 2 us, launch and latency; a call through the package takes 6 us of the host.
template <typename T>
__global__ void __launch_bounds__(128) rec_step_kernel(RecArgs a) {
  const int b = blockIdx.y, d = blockIdx.x * 128 + threadIdx.x;
  if (d >= a.D) return;
  const long long at = (long long)b * a.D + d;
  const float h = a.h_in ? a.h_in[at] : 0.f, x = Elem<T>::ld((const T*)a.x + b * a.xsb + d);
  const float f = Elem<T>::ld((const T*)a.f + b * a.fsb + d);
  const float v = a.i ? Step<T, true>(f, Elem<T>::ld((const T*)a.i + b * a.isb + d)).next(h, x) : Step<T, false>(f, 0.f).next(h, x);
  Elem<T>::st((T*)a.y + b * a.ysb + d, v);
  a.h_out[at] = v;
}

// ---- host ------------------------------------------------------------------------------------
int check_rec(int dtype, int B, int L, int D, std::initializer_list<const void*> acts, std::initializer_list<const void*> f32) {
  if (!valid_dtype(dtype)) return MEGA_ERR_DTYPE;
  if (B <= 0 || L <= 0 || D <= 0) return MEGA_ERR_SHAPE;
  // (steps are counted past the end by up to two strides; tiles of all sequences by an int)
  if (B > 65535 || L > INT_MAX - 8192 || ((long long)D + kC - 1) / kC * B > INT_MAX - kW) return MEGA_ERR_UNSUPPORTED;
  for (const void* p : acts)
    if (!aligned_to(p, elem_size(dtype))) return MEGA_ERR_ALIGN;
  for (const void* p : f32)
    if (!aligned_to(p, 4)) return MEGA_ERR_ALIGN;
  return MEGA_OK;
}

struct Operand {
  const void* p;
  long long sb, sl;
  bool on(int bytes, int es) const { return !p || (aligned_to(p, bytes) && sb * es % bytes == 0 && sl * es % bytes == 0); }
};
// bytes of a copy: 16 or 4 where every row of the inputs starts on them (and pairs of outputs on theirs), else 2
int mode_of(int es, std::initializer_list<Operand> in, std::initializer_list<Operand> out) {
  auto all = [&](std::initializer_list<Operand> ops, int bytes) { return std::all_of(ops.begin(), ops.end(), [&](const Operand& o) { return o.on(bytes, es); }); };
  if (all(in, 16) && all(out, 2 * es)) return 16;
  return es == 4 || (all(in, 4) && all(out, 4)) ? 4 : 2;
}

// Blocks to a cluster, 0 for serial warps: what is predicted to take the least time.  A round takes two blocks on a multiprocessor about 2.4 us and one
// block 1.6 (bf16 forward; the other forms' ratios are alike), a cluster's exchange some more; a launch is rounds and one to begin
// with, in as many waves as it has blocks for (the device holds that many clusters at once; half where a multiprocessor holds one
// block, which then always runs by itself: kResident).  Measured, bf16 forward, clusters of 1, 2, 4, 8: B = 8, L = 4096, D = 1024
// 54, 47, 53, 60 us; B = 1, L = 65536, D = 2048 771, 504, 258, 184; B = 8, L = 4096, D = 2048 74, 91, 101, 115; fp32 backward with an
// input gate (one block): B = 2, L = 8192, D = 1024 323, 193, 103, 164; B = 20, L = 1000, D = 320 45, 56, 62, 70.
int cluster_of(int tiles, int B, int L, int steps, int resident) {
  const int forced = g_options[OPT_REC_CLUSTER].load(std::memory_order_relaxed);
  if (forced == 1 || forced == 2 || forced == 4 || forced == 8) return forced;
  const long long units = (long long)tiles * B;
  if (forced == 16) return 0;
  struct Form {
    int size, slots;
    double round;
  };
  constexpr Form kForms[] = {{1, 296, 1.}, {2, 296, 1.2}, {4, 284, 1.25}, {8, 264, 1.3}};
  auto waves_of = [&](long long n, long long slots) {   // the last one takes less where one block runs by itself
    if (resident == 1) return (double)((n + slots / 2 - 1) / (slots / 2));
    const long long last = n % slots;
    return (double)(n / slots) + (last == 0 ? 0. : last <= slots / 2 ? 1.6 / 2.4 : 1.);
  };
  int best = 1;
  double least = 1e300;
  for (const Form& f : kForms) {
    const double cost = waves_of(units * f.size, f.slots) * ((L + f.size * kW * steps - 1) / (f.size * kW * steps) + 1) * f.round;
    if (cost < least * 0.999) least = cost, best = f.size;
  }
  return waves_of(units, 296 * kW) * ((L + steps - 1) / steps + 1) < least ? 0 : best;
}

template <typename Kernel>
void launch_rec(Kernel kernel, int tiles, int B, int cluster, size_t smem, cudaStream_t s, const RecArgs& a) {
  if (cluster == 0) {
    launch(kernel, dim3((a.units + kW - 1) / kW), dim3(kW * 32), smem, s, a);
    g_last_kernel.store("gated_recurrence serial", std::memory_order_relaxed);
    return;
  }
  allow_smem(reinterpret_cast<const void*>(kernel), smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * cluster, B);
  cfg.blockDim = dim3(kW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  g_last_kernel.store("gated_recurrence", std::memory_order_relaxed);
}

template <typename T, bool kGate, int kMode>
void run_mode(bool bwd, int B, RecArgs a, cudaStream_t s) {
  const int steps = bwd ? kBackSteps<T, kGate> : kForwardSteps<T>, tiles = (a.D + kC - 1) / kC;
  const int cluster = cluster_of(tiles, B, a.L, steps, bwd ? kResident<T, kGate, true> : kResident<T, kGate, false>);
  const size_t smem = bwd ? kRingBytes<T, kGate, true> : kRingBytes<T, kGate, false>;
  a.tiles = tiles, a.units = tiles * B;
  if (cluster == 0)
    launch_rec(bwd ? rec_bwd_kernel<T, kGate, kMode, true> : rec_fwd_kernel<T, kGate, kMode, true>, tiles, B, 0, smem, s, a);
  else
    launch_rec(bwd ? rec_bwd_kernel<T, kGate, kMode, false> : rec_fwd_kernel<T, kGate, kMode, false>, tiles, B, cluster, smem, s, a);
}
template <typename T>
void run_rec(bool bwd, int mode, int B, const RecArgs& a, cudaStream_t s) {
  auto go = [&](auto gate) {
    constexpr bool kGate = decltype(gate)::value;
    if (mode == 16) return run_mode<T, kGate, 16>(bwd, B, a, s);
    if constexpr (sizeof(T) == 2) {
      if (mode == 2) return run_mode<T, kGate, 2>(bwd, B, a, s);
    }
    run_mode<T, kGate, 4>(bwd, B, a, s);
  };
  a.i ? go(std::true_type{}) : go(std::false_type{});
}

// operands at the walk's first step, strides in its direction
template <typename P>
void turn(P& p, long long& stride, int L, int es) {
  if (p) p = (P)((const char*)p + (long long)(L - 1) * stride * es);
  stride = -stride;
}

}  // namespace

cudaError_t gated_recurrence_read_device_error(int* v, bool reset) { return read_device_error(v, reset); }

}  // namespace mega

using namespace mega;

extern "C" int mega_gated_recurrence_segment(int dtype, int gated) {
  return !valid_dtype(dtype) ? 0 : dtype == MEGA_F32 ? kBackSteps<float, false> : gated ? kBackSteps<__half, true> : kBackSteps<__half, false>;
}

extern "C" int mega_gated_recurrence_fwd(const void* x, const void* f, const void* i, void* y, int dtype, int B, int L, int D,
                                         int64_t xsb, int64_t xsl, int64_t fsb, int64_t fsl, int64_t isb, int64_t isl, int64_t ysb,
                                         int64_t ysl, const uint8_t* pad_mask, const uint8_t* reset_mask, const float* h_in,
                                         float* h_out, float* starts, unsigned flags, mega_stream_t stream) {
  if (!x || !f || !y) return MEGA_ERR_NULL;
  if (int rc = check_rec(dtype, B, L, D, {x, f, i, y}, {h_in, h_out, starts})) return rc;
  RecArgs a = {};
  a.x = x, a.f = f, a.i = i, a.y = y;
  a.xsb = xsb, a.xsl = xsl, a.fsb = fsb, a.fsl = fsl, a.isb = isb, a.isl = isl, a.ysb = ysb, a.ysl = ysl;
  a.pad = pad_mask, a.reset = reset_mask, a.h_in = h_in, a.h_out = h_out, a.starts = starts;
  a.msb = L, a.msl = 1, a.L = L, a.D = D;
  a.pairs = D % 2 == 0 && aligned_to(h_in, 8) && aligned_to(h_out, 8) && aligned_to(starts, 8);
  const int es = elem_size(dtype), mode = mode_of(es, {{x, xsb, xsl}, {f, fsb, fsl}, {i, isb, isl}}, {{y, ysb, ysl}});
  if (flags & MEGA_REC_REVERSE) {
    turn(a.x, a.xsl, L, es), turn(a.f, a.fsl, L, es), turn(a.i, a.isl, L, es), turn(a.y, a.ysl, L, es);
    if (a.pad) a.pad += L - 1;
    if (a.reset) a.reset += L - 1;
    a.msl = -1;
  }
  MEGA_DISPATCH_DTYPE(dtype, run_rec<T>(false, mode, B, a, (cudaStream_t)stream));
  return check_launch("gated_recurrence_fwd");
}

extern "C" int mega_gated_recurrence_bwd(const void* dy, const void* x, const void* f, const void* i, void* dx, void* df, void* di,
                                         int dtype, int B, int L, int D, int64_t gsb, int64_t gsl, int64_t xsb, int64_t xsl,
                                         int64_t fsb, int64_t fsl, int64_t isb, int64_t isl, int64_t dxb, int64_t dxl, int64_t dfb,
                                         int64_t dfl, int64_t dib, int64_t dil, const uint8_t* pad_mask, const uint8_t* reset_mask,
                                         const float* starts, const float* dh_out, float* dh_in, unsigned flags,
                                         mega_stream_t stream) {
  if (!dy || !x || !f || !dx || !df || !starts || (i && !di)) return MEGA_ERR_NULL;
  if (int rc = check_rec(dtype, B, L, D, {dy, x, f, i, dx, df, di}, {starts, dh_out, dh_in})) return rc;
  RecArgs a = {};
  a.dy = dy, a.x = x, a.f = f, a.i = i, a.dx = dx, a.df = df, a.di = di;
  a.gsb = gsb, a.gsl = gsl, a.xsb = xsb, a.xsl = xsl, a.fsb = fsb, a.fsl = fsl, a.isb = isb, a.isl = isl;
  a.dxb = dxb, a.dxl = dxl, a.dfb = dfb, a.dfl = dfl, a.dib = dib, a.dil = dil;
  a.pad = pad_mask, a.reset = reset_mask, a.starts = const_cast<float*>(starts), a.dh_out = dh_out, a.dh_in = dh_in;
  a.msb = L, a.msl = 1, a.L = L, a.D = D;
  a.pairs = D % 2 == 0 && aligned_to(dh_in, 8) && aligned_to(dh_out, 8) && aligned_to(starts, 8);
  const int es = elem_size(dtype);
  const int mode = mode_of(es, {{dy, gsb, gsl}, {x, xsb, xsl}, {f, fsb, fsl}, {i, isb, isl}}, {{dx, dxb, dxl}, {df, dfb, dfl}, {i ? di : nullptr, dib, dil}});
  if (flags & MEGA_REC_REVERSE) {
    turn(a.dy, a.gsl, L, es), turn(a.x, a.xsl, L, es), turn(a.f, a.fsl, L, es), turn(a.i, a.isl, L, es);
    turn(a.dx, a.dxl, L, es), turn(a.df, a.dfl, L, es), turn(a.di, a.dil, L, es);
    if (a.pad) a.pad += L - 1;
    if (a.reset) a.reset += L - 1;
    a.msl = -1;
  }
  MEGA_DISPATCH_DTYPE(dtype, run_rec<T>(true, mode, B, a, (cudaStream_t)stream));
  return check_launch("gated_recurrence_bwd");
}

extern "C" int mega_gated_recurrence_step(const void* x, const void* f, const void* i, void* y, int dtype, int B, int D, int64_t xsb,
                                          int64_t fsb, int64_t isb, int64_t ysb, const float* h_in, float* h_out,
                                          mega_stream_t stream) {
  if (!x || !f || !y || !h_out) return MEGA_ERR_NULL;
  if (int rc = check_rec(dtype, B, 1, D, {x, f, i, y}, {h_in, h_out})) return rc;
  RecArgs a = {};
  a.x = x, a.f = f, a.i = i, a.y = y, a.xsb = xsb, a.fsb = fsb, a.isb = isb, a.ysb = ysb;
  a.h_in = h_in, a.h_out = h_out, a.L = 1, a.D = D;
  MEGA_DISPATCH_DTYPE(dtype, launch(rec_step_kernel<T>, dim3((D + 127) / 128, B), dim3(128), 0, stream, a));
  return check_launch("gated_recurrence_step");
}

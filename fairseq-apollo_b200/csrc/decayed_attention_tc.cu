// Linear attention with a decay for each head (decayed_attention.cu has the mathematics) on tcgen05 products, for 16-bit activations and
// heads of at most 128 keys and values: chunks of 128 steps, a block to a (sequence, head) or a segment of one.
//
// Per chunk, with rows i, j of the chunk, and keys and values padded to 64 or 128 with zeros:
//   P  = Q K^T                      accumulator P, 128 columns; the weighted pairs go back as 16-bit operand in its first 64
//   O1 = Q S                        S: the state that enters, in shared memory
//   dS = (w K)^T V                  w K in pieces of 8 (bf16, three) or 11 (fp16, two) bits, the first in K's place
//   O2 = (weighted pairs) V
// and y = e O1 + O2 with a row's factor e.  The sums for the gates' gradient are those of x with e O1 and with O2: of the latter, taken from
// the walks of dq and dk, the pairs on one side of a step cancel because both walks round the same weights the same way (but for the one pair
// in some thousand whose weight, two units apart, lies next to a rounding's border: such a pair is off by one rounding).
// Roles: eight warps of pairs and outputs (a thread has half of a row of the chunk), eight of weights and state (a thread has half of a
// step's keys, then half of a row of the state, whose fp32 values stay in its registers), one that loads, one for
// padded steps, and two that issue products: those of pairs, and those with the state (one warp for both takes longer to wait and to issue
// than the tensor cores to compute).  All exchange over mbarriers.
//
// Activations lie as TMA leaves them (columns of 64, rows of 128 bytes, swizzled), what the threads write as planes of 16 bytes along
// keys or values, rows one after another.  Both serve with either axis as the contraction, and a thread that owns a row reads and
// writes it without bank conflicts.  (Loads by cp.async, three warps of them, took 140 cycles each and held up every other access to
// shared memory: they were what bounded it: 209 us, by TMA 135, 8 x 4096 x 16 heads of 64.)
//
// Measured (8 sequences x 4096 steps x 16 heads in bf16, forward, no padding): heads of 64 84 to 88 us, 3.1 TB/s of q, k, v and y; of 128
// 140 us, 3.8 TB/s; the products of chunks on mma.sync (decayed_attention.cu) 345 and 559 us.  What bounds it: a chunk of 64 x 64 heads
// takes 4600 cycles (from the difference to 8192 steps), in which its products keep the tensor cores busy for 1600; 8000 warp instructions at 1.75 a
// cycle and the exchanges between roles (250 cycles a wait) are the rest.  Heads of 128 also saturate shared memory: products read
// 350 KB of operands a chunk at 128 bytes a cycle, and the pieces of keys are 100 KB more (two pieces instead of three: 138 us for 152).
// Steps on the way: gates by a kernel before (123 -> 101 us at 64), two places for pairs (101 -> 91), products from two warps (91 -> 88).
// fp16 is scaled where it enters products (decayed_attention.cuh), for which the roles look their operands through once more and meet: heads of
// 64 100 us (86 without), of 128 153 (131), training at 64 516 (425), at 64 x 128 660 (610).
//
// The state is accumulated by each chunk's own sum, which is then added in fp32: a long chain inside the tensor cores' accumulator
// would be cut off, not rounded, thousands of times.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "decayed_attention.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace mega {
namespace {

constexpr int kC = kTcChunk, kPlane = kC * 16;

// What the gates of a chunk come to.  A pair's weight is one factor of j, from there to the last step of its 32, and
// one of i, from that step on; so is a step's weight in the state that leaves.  Only where the first factor gets too small, or a reset
// lies among those 32 steps, pairs inside them need a power of two each.
struct TcGates {
  int rel[kC];        // running sum of log2 a beyond that at the last of a step's 32, in 2^-18 (at most 32 x 149)
  float col[kC];      // weight of a step at the last of its 32 (0: a reset lies between)
  uint8_t count[kC];  // resets so far
  float base[4];      // running sum of log2 a at the last of 32 steps
  float between[4][4];   // [i][j]: running sum from the last of the 32 steps j to that of i (a difference of sums of thousands, as whole numbers)
  float leave[4];     // weight of the last of 32 steps in the state that leaves
  uint32_t pad[4];    // padded steps
  float enter;        // weight of the state that enters in the one that leaves
  uint8_t apart[4];   // whether resets lie among 32 steps, or their decay is out of range
  uint32_t padded;    // 0: no step is, 2: all are and none resets (which leaves the state as it is)
  uint32_t pad_;
};
static_assert(sizeof(TcGates) == kTcGates, "gates");
__device__ __forceinline__ int last_of(const Walk& w, int block) { return 32 * block + (w.rev ? 0 : 31); }

// They are found before the walk, a warp to a chunk: a warp of the walk itself took 3000 cycles for one and its loads as many again,
// which was most of a chunk's time.
template <typename T>
__global__ void __launch_bounds__(128) tc_gates_kernel(const __grid_constant__ Walk w) {
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_next();   // (the walk waits for this kernel's end where it reads the gates)
  if (at >= (long long)w.B * w.H * w.chunks) return;
  const int bh = (int)(at / w.chunks), tile = (int)(at % w.chunks);
  const GateIn<4> in = gates_fetch<T, 4>(w, bh / w.H, bh % w.H, tile, lane);
  const GateOut<4> r = gates_scan<4>(w, in, lane);
  TcGates& g = static_cast<TcGates*>(w.gates)[at];
  // (eight lanes hold 32 steps; the last of them in the order of the walk is the last one's)
  const long long end = __shfl_sync(~0u, r.sum[3], lane | 7);
  const int there = __shfl_sync(~0u, r.count[3], lane | 7);
  // (cut off alike for the walk that goes the other way, whose sums leave out a step's own gate: differences between steps are the same there)
  const int way = w.excl ? -1 : 1;
  auto place = [&](long long sum) { return (w.excl ? r.all - sum : sum) >> 22; };
  unsigned mask = 0;   // of this lane's rows in their word
  int rel[4];
  float col[4];
  uint8_t count[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int to = w.rev ? 3 - k : k;   // rows ascend
    rel[to] = way * (int)(place(r.sum[k]) - place(end)), count[to] = (uint8_t)r.count[k];
    col[to] = r.count[k] == there && !(in.pad >> k & 1) ? exp2f(gate_sum(end - r.sum[k]) + r.bad) : 0.f;
    mask |= (in.pad >> k & 1) << to;
  }
  const int row = w.rev ? kC - 4 - 4 * lane : 4 * lane, word = row / 32;
  *reinterpret_cast<int4*>(g.rel + row) = make_int4(rel[0], rel[1], rel[2], rel[3]);
  *reinterpret_cast<float4*>(g.col + row) = make_float4(col[0], col[1], col[2], col[3]);
  *reinterpret_cast<uchar4*>(g.count + row) = make_uchar4(count[0], count[1], count[2], count[3]);
  const unsigned lanes = 0xffu << (lane & 24);
  const bool reset = __any_sync(lanes, r.count[0] != there || r.count[1] != there || r.count[2] != there);
  const bool far = __any_sync(lanes, gate_sum(end - r.sum[0]) < (kScaled<T> ? -60.f : -100.f));   // (fp16: besides a scale of up to 2^40)
  mask = __reduce_or_sync(lanes, mask << (row & 31));
  float gap[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) gap[k] = gate_sum(end - __shfl_sync(~0u, end, 8 * (w.rev ? 3 - k : k))) + r.bad;   // (rows ascend)
  if ((lane & 7) == 7) {
    *reinterpret_cast<float4*>(g.between[word]) = make_float4(gap[0], gap[1], gap[2], gap[3]);
    g.apart[word] = reset || far;
    g.base[word] = gate_sum(end) + r.bad;
    g.leave[word] = there == r.total ? w.s_scale * exp2f(gate_sum(r.all - end) + r.bad) : 0.f;
    g.pad[word] = mask;
  }
  const bool all = __all_sync(~0u, in.pad == 15u);
  if (lane == 0) g.enter = r.enter, g.padded = !r.padded ? 0 : all && !r.total ? 2 : 1;
}

// barriers; kQRaw...: what a load completes where padded steps have to be cleared before the rest may see it; kUnit: fp16's scale of the state
enum { kQFull, kQEmpty = kQFull + 3, kQRaw = kQEmpty + 3, kKFull = kQRaw + 3, kKEmpty = kKFull + 3, kKRaw = kKEmpty + 3, kVFull = kKRaw + 3,
       kVEmpty = kVFull + 3, kVRaw = kVEmpty + 3, kXFull = kVRaw + 3, kXEmpty = kXFull + 2, kXRaw = kXEmpty + 2, kGFull = kXRaw + 2, kGEmpty = kGFull + 2,
       kPDone = kGEmpty + 2, kPReady = kPDone + 2, kODone = kPReady + 2, kO1Done, kORead = kO1Done + 2, kSReady = kORead + 2, kDsDone,
       kUnit, kAllDone = kUnit + 4, kWReady = kAllDone + 2, kBars = kWReady + 2 };

// kOut: outputs; else the state that a segment leaves by itself.  kDots: sums for the gates' gradient (1: walk of dq, 2: of dk).
template <typename T, int KD, int VD, bool kOut, int kDots>
struct Lay {
  static constexpr int kTk = KD * kC * 2, kTv = VD * kC * 2, kTs = VD / 8 * KD * 16;
  static constexpr bool kBig = KD == 128 && VD == 128 && kOut;   // heads of 128 x 128: shared memory holds seven of their tiles
  // pieces of weighted keys; beside x there is no room for a third one (which matters to no output but the gradient of the state)
  static constexpr int kPieces = std::is_same<T, __nv_bfloat16>::value && !(kBig && kDots) ? 3 : 2;
  // places of each operand, as shared memory has room
  static constexpr bool kSmall = KD == 64 && VD == 64;
  static constexpr int kQs = kSmall ? 3 : KD == 64 ? (kDots ? 2 : 3) : 1, kKs = kSmall ? 3 : KD == 64 && !kDots ? 3 : 2,
                       kVs = kSmall ? 3 : kBig && kPieces == 3 ? 1 : 2, kXs = kSmall ? 2 : 1;
  static constexpr bool kX = kDots && !kBig;   // x by way of shared memory; else each thread reads its half of a row itself (with one place
                                               // for values instead, the walks of dq and dk took 235 us for 207, 8 x 4096 x 16 heads)
  static constexpr int kThreads = 640;   // 8 warps of pairs and outputs, 8 of weights and state, loads, padding, products (2)
  // Registers of a thread: 96 at launch, 20 warps; where the state takes 64 of them its eight warps have 128, the first eight 88 and
  // the last four 48: 2 x 88 + 2 x 128 + 48 for each four warps, as at launch (5 x 96).
  static constexpr int kRegs = 96;
  static constexpr bool kMove = VD == 128;
  // Columns of tensor memory.  Where they suffice pairs have two places: those of the next chunk are worked on while this one's outputs
  // are on their way.
  static constexpr bool kTwo = kOut && VD == 64;
  static constexpr int kOffLo = 0, kOffLo2 = kOffLo + kTk, kOffK = kOffLo2 + (kPieces == 3 ? kTk : 0), kOffV = kOffK + kKs * kTk,
                       kOffQ = kOffV + kVs * kTv, kOffX = kOffQ + (kOut ? kQs * kTk : 0), kOffS = kOffX + (kX ? kXs * kTv : 0),
                       kOffG = kOffS + (kOut ? kTs : 0), kOffBar = kOffG + 2 * (int)sizeof(TcGates), kOffSlot = kOffBar + kBars * 8,
                       kOffMost = kOffSlot + 16, kOffUnit = kOffMost + 32, kOffPairs = kOffUnit + 4, kEnd = kOffMost + (!kScaled<T> ? 0 : kTwo ? 64 : 48);
  static_assert(kEnd <= 227 * 1024, "shared memory");
  static constexpr uint32_t kColO2 = kTwo ? 384 : 256, kColS = !kOut ? 0 : kTwo ? 448 : 384;
  static __device__ __forceinline__ uint32_t col_p(int n) { return kTwo ? (n & 1) * 128 : 0; }
  static __device__ __forceinline__ uint32_t col_o1(int n) { return kTwo ? 256 + (n & 1) * 64 : 128; }
  static_assert(sizeof(TcGates) % 16 == 0, "gates");
};

__device__ __forceinline__ bool tried(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// A wait that gives up (never expected) raises `gone` and returns false; from then on no wait lasts.  Warps that meet others by name run out on
// whatever the buffers hold; loads and products are issued no more, and what is under way is waited for before the block ends.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* gone, long long limit) {
  if (tried(bar, parity)) return true;
  const long long from = clock64();
#pragma unroll 1
  while (!tried(bar, parity))
    if (*gone || clock64() - from > limit) {
      g_device_error = *gone = 1;
      return false;
    }
  return true;
}
// what the block itself has under way, however short the limit of the other waits is
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity, long long limit) {
  const long long from = clock64();
#pragma unroll 1
  while (!tried(bar, parity) && clock64() - from < 2 * limit + 4000000) {}
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// `THREADS` threads, whole warps, meet
template <int ID, int THREADS>
__device__ __forceinline__ void named_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory"); }
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
__device__ __forceinline__ void tm_ld16(uint32_t at, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
        "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(at)
      : "memory");
}
// chunk n's place among S, and the parity of the barriers of its use of that place
template <int S>
struct Ring {
  static __device__ __forceinline__ int place(int n) { return n % S; }
  static __device__ __forceinline__ uint32_t parity(int n) { return n / S & 1; }
};
template <int N>
__device__ __forceinline__ void tm_load(uint32_t at, float* v) {
  if constexpr (N == 32) tm_ld32(at, v);
  else tm_ld16(at, v);
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

// w v as 16-bit pieces that add up to it.  bf16 (three): the upper, middle and lower eight bits, cut off, which is exact; fp16 (two): what
// rounding leaves is the second.
template <typename T, int PIECES>
__device__ __forceinline__ void split(float2 v, float w, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  v.x *= w, v.y *= w;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    auto upper = [](float f) { return __uint_as_float(__float_as_uint(f) & 0xffff0000u); };
    auto both = [](float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); };
    p0 = both(v.x, v.y);
    v.x -= upper(v.x), v.y -= upper(v.y);
    p1 = PIECES == 2 ? pack<T>(v.x, v.y) : both(v.x, v.y);
    v.x -= upper(v.x), v.y -= upper(v.y);
    p2 = both(v.x, v.y);
  } else {
    p0 = pack<T>(v.x, v.y);
    const float2 r = unpack<T>(p0);
    p1 = pack<T>(v.x - r.x, v.y - r.y);
    p2 = 0;
  }
}

// Products, all over k = 16 places at a time.  d = or += a b; A in shared or tensor memory.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn, int m) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
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
__device__ __forceinline__ void load_tile(uint32_t to, const CUtensorMap* m, const Operand& o, int t0, int h, int b, uint32_t bar, bool go = true) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(D * kC * 2) : "memory");
  if (!go) return;   // (a test: what waits for it gives up)
#pragma unroll
  for (int c = 0; c < D; c += 64) tma_load_4d(to + c / 64 * kBox, m, c, t0, o.sh ? h : 0, o.sb ? b : 0, bar);
}
__device__ __forceinline__ void clear_rows(uint32_t at, int planes, const uint32_t (&pad)[4], int lane) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (pad[k] >> lane & 1)
#pragma unroll 1
      for (int c = 0; c < planes; ++c) sts16(at + piece_of(32 * k + lane, c), make_uint4(0, 0, 0, 0));
}

template <typename T, int KD, int VD, bool kOut, int kDots>
__global__ void __launch_bounds__(Lay<T, KD, VD, kOut, kDots>::kThreads, 1) tc_kernel(const __grid_constant__ Walk w, const __grid_constant__ Maps maps) {
  using L = Lay<T, KD, VD, kOut, kDots>;
  using Qr = Ring<L::kQs>;
  using Kr = Ring<L::kKs>;
  using Vr = Ring<L::kVs>;
  using Xr = Ring<L::kXs>;
  extern __shared__ __align__(1024) unsigned char smem[];
  int* const slot_ = reinterpret_cast<int*>(smem + L::kOffSlot);   // where tensor memory lies; whether a wait has given up
  volatile int* gone = slot_ + 1;
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bh = blockIdx.x % (w.B * w.H), seg = blockIdx.x / (w.B * w.H), b = bh / w.H, h = bh % w.H;
  int first = seg * w.per, chunks = min(w.per, w.chunks - first);   // in the order of the walk
  const bool ends = first + chunks == w.chunks;
  auto bar = [&](int i) { return base + L::kOffBar + i * 8; };
  auto wait = [&](int i, uint32_t parity) { return wait_for(bar(i), parity, gone, w.wait_limit); };
  auto done = [&](int i) {   // (a warp arrives as one: barriers take their threads one after another)
    __syncwarp();
    if (lane == 0) arrive(bar(i));
  };
  auto tile_of = [&](int n) { return w.rev ? w.chunks - 1 - first - n : first + n; };
  auto gates = [&](int n) -> TcGates& { return reinterpret_cast<TcGates*>(smem + L::kOffG)[n & 1]; };

  if (tid == 0) {
    *gone = 0;
#pragma unroll 1
    for (int i = 0; i < kBars; ++i) {
      const bool empty = i == kGEmpty || i == kGEmpty + 1;
      const bool all = i == kXEmpty || i == kXEmpty + 1 || i == kPReady || i == kPReady + 1 || i == kORead || i == kORead + 1 || i == kSReady || i >= kWReady;
      const bool both = kOut && ((i >= kQEmpty && i < kQEmpty + 3) || (i >= kVEmpty && i < kVEmpty + 3));   // (two warps' products read it)
      mbar_init(reinterpret_cast<uint64_t*>(smem + L::kOffBar) + i, both ? 2 : empty ? 16 + (w.pad ? 1 : 0) : all ? (!kOut && i >= kWReady ? 16 : 8) : 1);
    }
    mbar_fence_init();
  }
  if (warp == 16 && umma_elect()) {
    prefetch_tensormap(&maps.k), prefetch_tensormap(&maps.v);
    if (kOut) prefetch_tensormap(&maps.q);
    if (L::kX) prefetch_tensormap(&maps.x);
  }
  if (warp == 0) tm_alloc(smem_u32(slot_), kOut ? 512 : 128);
  tm_before();
  __syncthreads();
  tm_after();
  pdl_wait();   // (all that comes before on the stream)
  if (w.pad) {
    // chunks of nothing but padding at either end of the segment are not walked
    const TcGates* const table = static_cast<const TcGates*>(w.gates) + (long long)bh * w.chunks;
    int* const range = slot_ + 2;
    if (tid == 0) range[0] = chunks, range[1] = -1;
    __syncthreads();
    for (int n = tid; n < chunks; n += L::kThreads)
      if (table[tile_of(n)].padded != 2) {
        atomicMin(range, n);
        atomicMax(range + 1, n);
      }
    __syncthreads();
    const int low = range[0], high = range[1] + 1;
    if constexpr (kOut) {
      const int per_row = w.v.d / 8, all = chunks - max(high - low, 0);
      for (long long k = tid; k < (long long)all * kC * per_row; k += L::kThreads) {
        const int at = (int)(k / (kC * per_row)), n = at < low ? at : at + high - low, r = (int)(k / per_row % kC);
        const long long t = (long long)tile_of(n) * kC + r;
        if (t < w.L) *reinterpret_cast<uint4*>(static_cast<char*>(w.out) + (b * w.ob + h * w.oh + t * w.ol + k % per_row * 8) * 2) = make_uint4(0, 0, 0, 0);
      }
    }
    if (high > low) first += low, chunks = high - low;
    else chunks = 0;
  }
  const uint32_t tm = *reinterpret_cast<volatile uint32_t*>(slot_);

  if constexpr (L::kMove) {   // (the four warps that do little leave registers to those that hold the state)
    if (warp >= 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    else if (warp >= 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  }
  // fp16: the powers of two that w K of a chunk, from `count` planes of a step in each thread, and the state that enters it, whose largest
  // value in this thread is `held`, are multiplied with.  The warps of weights meet for them, each with a byte for its exponents: two sets of
  // them in turn, as a warp may be at the next chunk while another still reads.
  // (Reading the keys once more and meeting costs 856 -> 924 us, training of 2 x 16384 x 16 heads of 64 x 128; the state's scale 9 more.)
  struct Scales {
    int keys, state;
  };
  auto scales = [&](int n, int step, int from, int count, float held) {
    const TcGates& g = gates(n);
    const uint32_t keys = base + L::kOffK + Kr::place(n) * L::kTk;
    __half2 top = __float2half2_rn(0.f);
#pragma unroll 2
    for (int c = from; c < from + count; ++c) {
      const uint4 u = lds16(keys + piece_of(step, c));
      const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&uu[k])));
    }
    const float most = fmaxf(__low2float(top), __high2float(top)) * fabsf(g.col[step] * g.leave[step >> 5]);
    constexpr int kMeet = kOut ? 8 : 16;
    volatile unsigned char* const of = smem + L::kOffMost + (n & 1) * 16;
    const unsigned own = __reduce_max_sync(~0u, __float_as_uint(most)) >> 23;
    const unsigned ours = kOut ? __reduce_max_sync(~0u, __float_as_uint(held)) >> 23 : 0;
    if (lane == 0) {
      of[warp & (kMeet - 1)] = (unsigned char)own;
      if (kOut) of[8 + (warp & 7)] = (unsigned char)ours;
    }
    __syncwarp();
    named_sync<1, 32 * kMeet>();
    const unsigned got = of[lane & 15];   // (16 keys' exponents, or eight and eight states')
    Scales r;
    r.keys = scale_of((int)__reduce_max_sync(~0u, !kOut || (lane & 8) == 0 ? got : 0u));
    r.state = kOut ? scale_of((int)__reduce_max_sync(~0u, lane & 8 ? got : 0u)) : 0;
    return r;
  };
  // w K in pieces, of a step's `count` planes from `from` on
  auto weigh = [&](int n, int step, int from, int count, int up) {
    const TcGates& g = gates(n);
    float wt = g.col[step] * g.leave[step >> 5];
    if constexpr (kScaled<T>) wt *= two_to(up);
    const uint32_t keys = base + L::kOffK + Kr::place(n) * L::kTk;
#pragma unroll 1
    for (int c0 = from; c0 < from + count; c0 += 2) {   // (two at a time: reads first, as none may pass a write)
      uint4 u[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) u[c] = lds16(keys + piece_of(step, c0 + c));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t piece[3][4];
        const uint32_t uu[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) split<T, L::kPieces>(unpack<T>(uu[k]), wt, piece[0][k], piece[1][k], piece[2][k]);
        const int at = c0 + c;
        sts16(keys + piece_of(step, at), make_uint4(piece[0][0], piece[0][1], piece[0][2], piece[0][3]));
        sts16(base + L::kOffLo + at * kPlane + step * 16, make_uint4(piece[1][0], piece[1][1], piece[1][2], piece[1][3]));
        if constexpr (L::kPieces == 3) sts16(base + L::kOffLo2 + at * kPlane + step * 16, make_uint4(piece[2][0], piece[2][1], piece[2][2], piece[2][3]));
      }
    }
    fence_proxy_async();
    done(kWReady + (n & 1));
  };

  if (warp < 8) {
    // ================================================================================ pairs and outputs
    if constexpr (!kOut) {   // (none: the other half of the weighted keys)
      const int step = (warp & 3) * 32 + lane, from = (warp >> 2) * (KD / 16) + KD / 32;
      int up = 0;
#pragma unroll 1
      for (int n = 0; n < chunks; ++n) {
        wait(kGFull + (n & 1), n >> 1 & 1);
        wait(kKFull + Kr::place(n), Kr::parity(n));
        if (n) wait(kDsDone, (n - 1) & 1);   // (the products have read the last chunk's)
        if constexpr (kScaled<T>) up = scales(n, step, from, KD / 32, 0.f).keys;
        weigh(n, step, from, KD / 32, up);
        done(kGEmpty + (n & 1));
      }
    } else {
      constexpr int kW = 32;   // columns at a time (sixteen take longer: 94 us for 86, 8 x 4096 x 16 heads of 64)
      const int rb = warp & 3, half = warp >> 2, i = rb * 32 + lane;   // a row, and half of its pairs and of its outputs
      const uint32_t quarter = tm + ((uint32_t)(rb * 32) << 16);
      float e_next = 0.f, unit_next = 1.f;
      bool live = false;   // (read by the thread itself, x of a padded step must not count)
      auto pairs = [&](int n) {
        const TcGates& g = gates(n);
        wait(kGFull + (n & 1), n >> 1 & 1);
        const int ri = g.rel[i];
        const float gi = g.base[rb] + 0x1p-18f * (float)ri;
        const int ci = g.count[i];
        live = !(g.pad[rb] >> lane & 1);
        e_next = ci || !live ? 0.f : w.o_scale * ex2(gi);
        wait(kPDone + (n & 1), n >> 1 & 1);
        tm_after();
        const int from = max(w.rev ? rb : 0, 2 * half), to = min(w.rev ? 3 : rb, 2 * half + 1);   // blocks of 32 steps that these rows see
        float p_scale = w.p_scale;
        if constexpr (kScaled<T>) {
          // fp16: a power of two for all pairs of the chunk, from the largest one before its weight (at most 2^40: a row's factor may be 2^60).
          // Two sets of bytes in turn where the next chunk's pairs may be under way while another warp still reads.
          float top = 0.f;
#pragma unroll 1
          for (int jb = from; jb <= to; ++jb) {
            float v[32];
            tm_ld32(quarter + L::col_p(n) + 32 * jb, v);
            tm_wait_ld();
            loaded(v);
#pragma unroll
            for (int j = 0; j < 32; ++j) top = fmaxf(top, fabsf(v[j]));
          }
          const unsigned own = __reduce_max_sync(~0u, __float_as_uint(top * fabsf(p_scale))) >> 23;
          volatile unsigned char* const of = smem + L::kOffPairs + (L::kTwo ? (n & 1) * 8 : 0);
          if (lane == 0) of[warp] = (unsigned char)own;
          __syncwarp();
          named_sync<2, 256>();
          const int up = min(scale_of((int)__reduce_max_sync(~0u, (unsigned)of[lane & 7])), 40);
          p_scale *= two_to(up), unit_next = two_to(-up);
        }
        // kW pairs of a row
        auto block = [&](int jb, int k) {
          float v[kW];
          tm_ld32(quarter + L::col_p(n) + 32 * jb + k, v);
          // (one factor above one and one below where the row lies inside the 32 steps: their product is what counts, while both are in range.
          // The row's is then one over its own as a column: both walks' weights agree to two units, however large the sums.)
          const int end = last_of(w, jb), j0 = 32 * jb + k;
          const float col = g.col[i];
          const float f = g.count[end] != ci || (jb == rb && col == 0.f) ? 0.f : jb == rb ? __fdividef(p_scale, col) : p_scale * ex2(g.between[rb][jb] + 0x1p-18f * (float)ri);
          float4 c[kW / 4];
#pragma unroll
          for (int j = 0; j < kW / 4; ++j) c[j] = *reinterpret_cast<const float4*>(g.col + j0 + 4 * j);
          const f32x2 ff = pack2(f, f);
          tm_wait_ld();
          loaded(v);
          // a step by itself has the same weight to the last bit in the walks of dq and dk, whose sums differ by it
          float own = 0.f;
          if constexpr (kDots != 0)
            if (jb == rb)
#pragma unroll
              for (int j = 0; j < kW; ++j) own = j == lane - k ? v[j] * p_scale : own;
          if (jb != rb || !g.apart[jb]) {
#pragma unroll
            for (int j = 0; j < kW / 4; ++j) {
              unpack2(mul2(pack2(v[4 * j], v[4 * j + 1]), mul2(ff, pack2(c[j].x, c[j].y))), v[4 * j], v[4 * j + 1]);
              unpack2(mul2(pack2(v[4 * j + 2], v[4 * j + 3]), mul2(ff, pack2(c[j].z, c[j].w))), v[4 * j + 2], v[4 * j + 3]);
            }
          } else {   // resets among these steps, or a decay by more than 2^-100 (fp16: 2^-60): a power of two for each pair
#pragma unroll
            for (int j = 0; j < kW; ++j) {
              const float p = v[j] * (p_scale * ex2(0x1p-18f * (float)min(ri - g.rel[j0 + j], 0)));
              v[j] = g.count[j0 + j] == ci ? p : 0.f;
            }
          }
          if (jb == rb) {
            const uint32_t seen = (w.rev ? ~0u << lane : ~0u >> (31 - lane)) >> k;
#pragma unroll
            for (int j = 0; j < kW; ++j) v[j] = seen & (1u << j) ? v[j] : 0.f;
            if constexpr (kDots != 0)
#pragma unroll
              for (int j = 0; j < kW; ++j) v[j] = j == lane - k ? own : v[j];
          }
          uint32_t word[kW / 2];
#pragma unroll
          for (int j = 0; j < kW / 2; ++j) word[j] = pack<T>(v[2 * j], v[2 * j + 1]);
          const uint32_t to = quarter + L::col_p(n) + 64 * half + 16 * (jb & 1) + k / 2;   // (in the place of pairs that this warp has read)
#pragma unroll
          for (int j = 0; j < kW / 2; j += 8) tm_st8(to + j, word + j);
        };
        {
#pragma unroll 1
          for (int j = 32 * from; j < 32 * to + 32; j += kW) block(j / 32, j % 32);
          const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
          for (int jb = 2 * half; jb < 2 * half + 2; ++jb)
            if (jb < from || jb > to) {
              tm_st8(quarter + L::col_p(n) + 64 * half + 16 * (jb & 1), zero);
              tm_st8(quarter + L::col_p(n) + 64 * half + 16 * (jb & 1) + 8, zero);
            }
        }
        done(kGEmpty + (n & 1));
        tm_wait_st();
        tm_before();
        done(kPReady + (n & 1));
      };
      auto outputs = [&](int n, float e, float unit) {   // unit: what the pairs' share is to be multiplied with
        const long long t = (long long)tile_of(n) * kC + i;
        float read = 0.f, inner = 0.f;
        constexpr int kUnroll = kDots && !L::kX ? 4 : 1, kHalf = VD / 2, kO = kDots && !L::kX ? 16 : kW;
        uint4 xr[kDots && !L::kX ? kHalf / 8 : 1];
        if constexpr (kDots && !L::kX) {
          const T* xp = static_cast<const T*>(w.x.p) + b * w.x.sb + h * w.x.sh + t * w.x.sl + half * kHalf;
#pragma unroll
          for (int m = 0; m < kHalf / 8; ++m)
            xr[m] = live && t < w.L && half * kHalf + 8 * m < w.x.d ? __ldg(reinterpret_cast<const uint4*>(xp) + m) : make_uint4(0, 0, 0, 0);
        } else if (kDots) {
          wait(kXFull + Xr::place(n), Xr::parity(n));
        }
        wait(kODone, n & 1);
        wait(kO1Done + (n & 1), n >> 1 & 1);
        tm_after();
        if constexpr (kScaled<T>) {
          // (four places: the next state but one waits for these outputs to be read)
          wait(kUnit + (n & 3), n >> 2 & 1);
          e *= two_to(113 - (int)*(volatile unsigned char*)(smem + L::kOffUnit + (n & 3)));
        }
        char* row = static_cast<char*>(w.out) + (b * w.ob + h * w.oh + t * w.ol) * 2;
        const bool apart = __any_sync(~0u, e == 0.f);   // rows that read nothing of the state (which may be infinite: no factor)
#pragma unroll kUnroll
        for (int c0 = 0; c0 < kHalf; c0 += kO) {
          const int c = half * kHalf + c0;
          float o[kO], p[kO];
          tm_load<kO>(quarter + L::col_o1(n) + c, o);
          tm_load<kO>(quarter + L::kColO2 + c, p);
          uint4 u[kDots ? kO / 8 : 1];
          if constexpr (kDots != 0)
#pragma unroll
            for (int m = 0; m < kO / 8; ++m) u[m] = kDots && !L::kX ? xr[kDots && !L::kX ? c0 / 8 + m : 0] : lds16(base + L::kOffX + Xr::place(n) * L::kTv + piece_of(i, c / 8 + m));
          tm_wait_ld();
          loaded(o);
          loaded(p);
          if (apart)
#pragma unroll
            for (int m = 0; m < kO; ++m) o[m] = e == 0.f ? 0.f : o[m];
          if (c0 + kO >= kHalf) {
            tm_before();
            done(kORead + (n & 1));
          }
          uint32_t word[kO / 2];
          const f32x2 ee = pack2(e, e);
          if constexpr (kScaled<T>)
#pragma unroll
            for (int m = 0; m < kO / 2; ++m) unpack2(mul2(pack2(unit, unit), pack2(p[2 * m], p[2 * m + 1])), p[2 * m], p[2 * m + 1]);
#pragma unroll
          for (int m = 0; m < kO / 2; ++m) {
            f32x2 y;
            if constexpr (kDots != 0) {
              const f32x2 own = mul2(ee, pack2(o[2 * m], o[2 * m + 1]));
              const uint32_t uu[4] = {u[m / 4].x, u[m / 4].y, u[m / 4].z, u[m / 4].w};
              const float2 x = unpack<T>(uu[m & 3]);
              unpack2(own, o[2 * m], o[2 * m + 1]);
              read += o[2 * m] * x.x + o[2 * m + 1] * x.y;
              inner += p[2 * m] * x.x + p[2 * m + 1] * x.y;
              y = add2(own, pack2(p[2 * m], p[2 * m + 1]));
            } else {
              y = fma2(ee, pack2(o[2 * m], o[2 * m + 1]), pack2(p[2 * m], p[2 * m + 1]));
            }
            float lo, hi;
            unpack2(y, lo, hi);
            word[m] = pack<T>(lo, hi);
          }
          if (t < w.L) {
            if (w.piece == 32) {
#pragma unroll
              for (int m = 0; m < kO / 2; m += 8)
                if (c + 2 * m < w.v.d)
                  asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + (c + 2 * m) * 2), "r"(word[m]),
                               "r"(word[m + 1]), "r"(word[m + 2]), "r"(word[m + 3]), "r"(word[m + 4]), "r"(word[m + 5]), "r"(word[m + 6]), "r"(word[m + 7])
                               : "memory");
            } else {
#pragma unroll
              for (int m = 0; m < kO / 2; m += 4)
                if (c + 2 * m < w.v.d) *reinterpret_cast<uint4*>(row + (c + 2 * m) * 2) = make_uint4(word[m], word[m + 1], word[m + 2], word[m + 3]);
            }
          }
        }
        if (kDots) {
          if (L::kX) done(kXEmpty + Xr::place(n));
          if (t < w.L) w.dots[((long long)half * w.B * w.H + bh) * w.L + t] = make_float2(read, inner);
        }
      };
      constexpr int kAhead = L::kTwo ? 1 : 0;
#pragma unroll 1
      for (int n = -kAhead; n < chunks; ++n) {
        const float e_now = e_next, unit_now = unit_next;
        if (n + kAhead < chunks) pairs(n + kAhead);
        if (n >= 0) outputs(n, kAhead ? e_now : e_next, kAhead ? unit_now : unit_next);
      }
    }
  } else if (warp < 16) {
    // ================================================================================ weights and state
    constexpr int kCols = VD / 2, kPlanes = KD / 16;
    const int sw = warp - 8, step = (sw & 3) * 32 + lane, half = sw >> 2;   // a step; half: of the planes of keys, of the values
    const uint32_t quarter = tm + ((uint32_t)((sw & 3) * 32) << 16);
    // a key's row of the state: of 64, the tensor cores leave 16 in each warp's lanes
    const int row = KD == 128 ? step : (sw & 3) * 16 + (lane & 15);
    const int col0 = half * kCols;
    float st[kCols];
    const long long s_at = (long long)bh * w.k.d * w.v.d + (long long)row * w.s_row;
    auto slot = [&](long long at) { return (at * w.k.d + row) * VD + col0; };   // a row of a state in the workspace
    const bool holds = KD == 128 || lane < 16, mine = holds && row < w.k.d;
#pragma unroll
    for (int c = 0; c < kCols; ++c) st[c] = 0.f;
    if (kOut && mine && w.s_in) {
      const float* p = w.s_in + s_at + (long long)col0 * w.s_col;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 8)   // (values come in eights)
        if (col0 + c0 < w.v.d)
#pragma unroll
          for (int c = c0; c < c0 + 8; ++c, p += w.s_col) st[c] = *p;
    }
    if (kOut)
      for (int p = 0; p < seg; ++p) {
        const float fac = w.factor[(long long)p * w.B * w.H + bh];
        const float* l = w.local + slot((long long)p * w.B * w.H + bh);
        if (mine)
#pragma unroll
          for (int c = 0; c < kCols; c += 4) {
            const float4 u = *reinterpret_cast<const float4*>(l + c);
            const float uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) st[c + k] = (fac == 0.f ? 0.f : fac * st[c + k]) + uu[k];
          }
      }
    // eight values of the state as an operand: rounded to 16 bits (the state itself is not), fp16 after a scale
    float scale = 1.f;
    auto eight = [&](int c) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = kScaled<T> ? st[c + k] * scale : st[c + k];
      return make_uint4(pack<T>(v[0], v[1]), pack<T>(v[2], v[3]), pack<T>(v[4], v[5]), pack<T>(v[6], v[7]));
    };
    auto state_out = [&]() {
      if (holds)
#pragma unroll
        for (int c = 0; c < kCols; c += 8) sts16(base + L::kOffS + (col0 + c) / 8 * (KD * 16) + row * 16, eight(c));
      fence_proxy_async();
      done(kSReady);
    };
    if (kOut && !kScaled<T>) state_out();
    float decay = 1.f;
    constexpr int kMine = kOut ? kPlanes : kPlanes / 2;
    int up = 0;
    for (int n = 0; n < chunks; ++n) {
      const TcGates& g = gates(n);
      wait(kGFull + (n & 1), n >> 1 & 1);
      wait(kKFull + Kr::place(n), Kr::parity(n));
      if constexpr (kScaled<T>) {
        float held = 0.f;
        if (kOut && holds)
#pragma unroll
          for (int c = 0; c < kCols; ++c) held = fmaxf(held, fabsf(st[c]));
        const Scales r = scales(n, step, half * kPlanes, kMine, held);
        up = r.keys, scale = two_to(r.state);
        if constexpr (kOut) {
          if (sw == 0 && lane == 0) {
            smem[L::kOffUnit + (n & 3)] = (unsigned char)(r.state + 113);
            arrive(bar(kUnit + (n & 3)));
            if (kDots == 1) w.units[(long long)bh * w.chunks + tile_of(n)] = two_to(-r.state);
          }
          state_out();
        }
      }
      if (kOut) wait(kPDone + (n & 1), n >> 1 & 1);   // (the pairs' product has read the keys)
      const float enter = g.enter;
      weigh(n, step, half * kPlanes, kMine, up);
      if constexpr (kDots != 0) {
        // the state that enters: left by the walk of dq, multiplied with the gradient of the one that leaves by that of dk
        T* a = static_cast<T*>(w.anchors) + slot((long long)bh * w.chunks + tile_of(n));
        if (kDots == 1) {
          if (mine && enter != 0.f)
#pragma unroll
            for (int c = 0; c < kCols; c += 8)
              *reinterpret_cast<uint4*>(a + c) = eight(c);
        } else {
          float s = 0.f;
          if (mine && enter > kLeast)
#pragma unroll
            for (int c = 0; c < kCols; c += 8) {
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
            const long long at = (long long)bh * w.chunks + tile_of(n);
            if (kScaled<T> && enter > kLeast) s *= w.units[at];
            w.through[at * kTcParts + sw] = enter > kLeast ? enter * s : 0.f;
          }
        }
      }
      wait(kDsDone, n & 1);
      tm_after();
      {
        if (enter == 0.f)   // (not a factor: what is forgotten may be infinite)
#pragma unroll
          for (int c = 0; c < kCols; ++c) st[c] = 0.f;
        const f32x2 ee = pack2(enter, enter), unit = pack2(two_to(-up), two_to(-up));
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          float v[16];
          tm_ld16(quarter + L::kColS + col0 + c, v);
          tm_wait_ld();
          loaded(v);
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            f32x2 sum = pack2(v[k], v[k + 1]);
            if constexpr (kScaled<T>) sum = mul2(unit, sum);
            unpack2(fma2(ee, pack2(st[c + k], st[c + k + 1]), sum), st[c + k], st[c + k + 1]);
          }
        }
        tm_before();
      }
      decay *= enter;
      done(kGEmpty + (n & 1));
      if (kOut && !kScaled<T> && n + 1 < chunks) state_out();
    }
    if (!kOut) {
      if (mine) {
        float* l = w.local + slot((long long)seg * w.B * w.H + bh);
#pragma unroll
        for (int c = 0; c < kCols; c += 4) *reinterpret_cast<float4*>(l + c) = make_float4(st[c], st[c + 1], st[c + 2], st[c + 3]);
      }
      if (sw == 0 && lane == 0) w.factor[(long long)seg * w.B * w.H + bh] = decay;
    } else if (w.s_out && ends && mine) {
      float* p = w.s_out + s_at + (long long)col0 * w.s_col;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 8)
        if (col0 + c0 < w.v.d)
#pragma unroll
          for (int c = c0; c < c0 + 8; ++c, p += w.s_col) *p = st[c];
    }
  } else if (warp == 16) {
    // ================================================================================ loads
    if (umma_elect()) {
      const TcGates* const table = static_cast<const TcGates*>(w.gates) + (long long)bh * w.chunks;
      bool next = w.pad && chunks && table[tile_of(0)].padded;
      // parity of the uses of kQRaw..., for rings of one, two and three places
      uint32_t uses = 0;
      auto used = [](int n) { return 1u | 2u << (n & 1) | 8u << n % 3; };
      int n = 0, begun = 0;   // where it ended: loads of chunk n that were issued, bits of keys, queries, values, x, gates
#pragma unroll 1
      for (; n < chunks; ++n) {
        const int t0 = tile_of(n) * kC;
        const bool raw = next;   // (the others' loads are seen as they land)
        next = w.pad && n + 1 < chunks && table[tile_of(n + 1)].padded;
        constexpr int kFirst = L::kVs > 1 ? 5 : 1;   // keys, and values where they come next
        if (n >= L::kKs && !wait(kKEmpty + Kr::place(n), Kr::parity(n) ^ 1)) break;
        load_tile<KD>(base + L::kOffK + Kr::place(n) * L::kTk, &maps.k, w.k, t0, h, b, bar((raw ? kKRaw : kKFull) + Kr::place(n)), n != w.withhold);
        auto values = [&]() {
          if (n >= L::kVs && !wait(kVEmpty + Vr::place(n), Vr::parity(n) ^ 1)) return false;
          load_tile<VD>(base + L::kOffV + Vr::place(n) * L::kTv, &maps.v, w.v, t0, h, b, bar((raw ? kVRaw : kVFull) + Vr::place(n)));
          return true;
        };
        if (L::kVs > 1 && !values()) {
          begun = 1;
          break;
        }
        if (kOut) {
          if (n >= L::kQs && !wait(kQEmpty + Qr::place(n), Qr::parity(n) ^ 1)) {
            begun = kFirst;
            break;
          }
          load_tile<KD>(base + L::kOffQ + Qr::place(n) * L::kTk, &maps.q, w.q, t0, h, b, bar((raw ? kQRaw : kQFull) + Qr::place(n)));
        }
        if (n > 1 && !wait(kGEmpty + (n & 1), (n >> 1 & 1) ^ 1)) {
          begun = kFirst | 2;
          break;
        }
        uint64_t* const got = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + kGFull + (n & 1);
        mbar_expect_tx(got, sizeof(TcGates));
        bulk_load_1d(&gates(n), table + tile_of(n), sizeof(TcGates), got);
        if (L::kX) {
          if (n >= L::kXs && !wait(kXEmpty + Xr::place(n), Xr::parity(n) ^ 1)) {
            begun = kFirst | 2 | 16;
            break;
          }
          load_tile<VD>(base + L::kOffX + Xr::place(n) * L::kTv, &maps.x, w.x, t0, h, b, bar((raw ? kXRaw : kXFull) + Xr::place(n)));
        }
        if (L::kVs == 1 && !values()) {
          begun = kFirst | 2 | 16 | 8;
          break;
        }
        if (raw) uses ^= used(n);
      }
      // (the last load of each place lands before the block ends, also where no one has waited for it)
      auto landed = [&](int what, int places, int full, int raw) {
        const int count = n + (begun >> what & 1);
        auto is_raw = [&](int m) { return raw != full && w.pad && table[tile_of(m)].padded; };
        const uint32_t parity = count > n && is_raw(n) ? uses ^ used(n) : uses;
#pragma unroll 1
        for (int m = max(count - places, 0); m < count; ++m) {
          if (what == 0 && m == w.withhold) continue;
          const int place = m % places;
          if (is_raw(m)) settle(bar(raw + place), (parity >> (places == 1 ? 0 : places == 2 ? 1 + place : 3 + place) & 1) ^ 1, w.wait_limit);
          else settle(bar(full + place), m / places & 1, w.wait_limit);
        }
      };
      landed(0, L::kKs, kKFull, kKRaw);
      if (kOut) landed(1, L::kQs, kQFull, kQRaw);
      landed(2, L::kVs, kVFull, kVRaw);
      if (L::kX) landed(3, L::kXs, kXFull, kXRaw);
      landed(4, 2, kGFull, kGFull);
    }
    __syncwarp();
  } else if (warp == 17) {
    // ================================================================================ padded steps: whatever lies there becomes zeros
    if (w.pad) {
      uint32_t used = 0;   // parity of each place's uses by chunks with padding
      auto together = [&](int i, uint32_t parity) { return __all_sync(~0u, wait(i, parity)); };
      bool go = true;
      for (int n = 0; go && n < chunks; ++n) {
        const TcGates& g = gates(n);
        if (!together(kGFull + (n & 1), n >> 1 & 1)) break;
        const uint32_t pad[4] = {g.pad[0], g.pad[1], g.pad[2], g.pad[3]};
        const bool any = g.padded;
        done(kGEmpty + (n & 1));
        if (!any) continue;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {   // keys, queries, values, x (and x before values where those have one place)
          const int what = k < 2 ? k : L::kVs == 1 ? 5 - k : k;
          if ((what == 1 && !kOut) || (what == 3 && !L::kX)) continue;
          const int place = what == 0 ? Kr::place(n) : what == 1 ? Qr::place(n) : what == 2 ? Vr::place(n) : Xr::place(n);
          const int raw = (what == 0 ? kKRaw : what == 1 ? kQRaw : what == 2 ? kVRaw : kXRaw) + place;
          const int full = (what == 0 ? kKFull : what == 1 ? kQFull : what == 2 ? kVFull : kXFull) + place;
          const uint32_t at = base + (what == 0 ? L::kOffK : what == 1 ? L::kOffQ : what == 2 ? L::kOffV : L::kOffX) + place * (what < 2 ? L::kTk : L::kTv);
          go = together(raw, used >> (3 * what + place) & 1);
          if (!go) break;
          used ^= 1u << (3 * what + place);
          clear_rows(at, what < 2 ? KD / 8 : VD / 8, pad, lane);
          fence_proxy_async();
          done(full);
        }
      }
    }
  } else if (warp == 18) {
    // ================================================================================ products of pairs
    if (kOut && umma_elect()) {
      constexpr uint32_t kPairs = idesc<T>(128, false, false, 128), kRows = idesc<T>(VD, false, true, 128);
      constexpr int kAhead = L::kTwo ? 1 : 0;
      bool begun = false;
#pragma unroll 1
      for (int n = -kAhead; n < chunks; ++n) {
        if (const int m = n + kAhead; m < chunks) {
          if (!wait(kQFull + Qr::place(m), Qr::parity(m)) || !wait(kKFull + Kr::place(m), Kr::parity(m))) break;
          // (a barrier tells two phases apart: the warps of weights have seen these products of two chunks ago, not only those of pairs)
          if (m > 1 && !wait(kWReady + (m & 1), (m >> 1 & 1) ^ 1)) break;
          tm_after();
          const uint64_t q = tile_desc(base + L::kOffQ + Qr::place(m) * L::kTk), kt = tile_desc(base + L::kOffK + Kr::place(m) * L::kTk);
#pragma unroll
          for (int k = 0; k < KD / 16; ++k) umma(tm + L::col_p(m), q + kAlong(k), kt + kAlong(k), kPairs, k > 0);
          begun = true;
          umma_commit(bar(kPDone + (m & 1)));
          umma_commit(bar(kQEmpty + Qr::place(m)));
        }
        if (n < 0) continue;
        const uint64_t vt = tile_desc(base + L::kOffV + Vr::place(n) * L::kTv);
        if (!wait(kVFull + Vr::place(n), Vr::parity(n)) || (n && !wait(kORead + ((n - 1) & 1), (n - 1) >> 1 & 1)) ||
            !wait(kPReady + (n & 1), n >> 1 & 1))
          break;
        tm_after();
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma_tm(tm + L::kColO2, tm + L::col_p(n) + k / 4 * 64 + k % 4 * 8, vt + kOver(k), kRows, k > 0);
        umma_commit(bar(kODone));
        umma_commit(bar(kVEmpty + Vr::place(n)));
      }
      if (begun) {   // (nothing of this block's products is on its way when it ends)
        umma_commit(bar(kAllDone));
        settle(bar(kAllDone), 0, w.wait_limit);
      }
    }
    __syncwarp();
  } else {
    // ================================================================================ products of the state
    if (umma_elect()) {
      constexpr uint32_t kRows = idesc<T>(VD, false, true, 128), kBoth = idesc<T>(VD, true, true, KD);
      const uint64_t s = over(base + L::kOffS, KD * 16), lo = over(base + L::kOffLo, kPlane), lo2 = over(base + L::kOffLo2, kPlane);
      bool begun = false;
#pragma unroll 1
      for (int n = 0; n < chunks; ++n) {
        if constexpr (kOut) {
          if (!wait(kQFull + Qr::place(n), Qr::parity(n)) || !wait(kSReady, n & 1)) break;
          if (const int m = L::kTwo ? n - 2 : n - 1; m >= 0 && !wait(kORead + (m & 1), m >> 1 & 1)) break;   // (the place is free)
          tm_after();
          const uint64_t q = tile_desc(base + L::kOffQ + Qr::place(n) * L::kTk);
#pragma unroll
          for (int k = 0; k < KD / 16; ++k) umma(tm + L::col_o1(n), q + kAlong(k), s + k * 16, kRows, k > 0);
          begun = true;
          umma_commit(bar(kO1Done + (n & 1)));
          umma_commit(bar(kQEmpty + Qr::place(n)));
        }
        if (!wait(kVFull + Vr::place(n), Vr::parity(n)) || !wait(kWReady + (n & 1), n >> 1 & 1)) break;
        tm_after();
        const uint64_t kt = tile_desc(base + L::kOffK + Kr::place(n) * L::kTk), vt = tile_desc(base + L::kOffV + Vr::place(n) * L::kTv);
        if constexpr (L::kPieces == 3)
#pragma unroll
          for (int k = 0; k < kC / 16; ++k) umma(tm + L::kColS, lo2 + k * 16, vt + kOver(k), kBoth, k > 0);
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma(tm + L::kColS, lo + k * 16, vt + kOver(k), kBoth, k > 0 || L::kPieces == 3);
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) umma(tm + L::kColS, kt + kOver(k), vt + kOver(k), kBoth, true);
        begun = true;
        umma_commit(bar(kDsDone));
        umma_commit(bar(kKEmpty + Kr::place(n)));
        umma_commit(bar(kVEmpty + Vr::place(n)));
      }
      if (begun) {
        umma_commit(bar(kAllDone + 1));
        settle(bar(kAllDone + 1), 0, w.wait_limit);
      }
    }
    __syncwarp();
  }
  tm_before();
  __syncthreads();
  tm_after();
  if (warp == 0) tm_free(tm, kOut ? 512 : 128);
}

// Whether the compiler gave a kernel the registers that its warps share out among themselves: with fewer they would wait for good.
bool has_registers(const void* kernel, int regs) {
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, kernel) == cudaSuccess) return a.numRegs >= regs;
  cudaGetLastError();
  return false;
}
// The kernels of a walk whose keys and values are padded to KD and VD
template <typename T, int KD, int VD>
struct Width {
  template <bool kOut, int kDots>
  static bool takes() {
    using L = Lay<T, KD, VD, kOut, kDots>;
    return !L::kMove || has_registers(reinterpret_cast<const void*>(+tc_kernel<T, KD, VD, kOut, kDots>), L::kRegs);
  }
  static bool takes_all() {
    static std::atomic<bool> known{false};   // (asked until they do: it costs microseconds)
    if (!known.load(std::memory_order_relaxed) && takes<false, 0>() && takes<true, 0>() && takes<true, 1>() && takes<true, 2>()) known.store(true);
    return known.load(std::memory_order_relaxed);
  }
  template <bool kOut, int kDots>
  static void go(const Walk& w, const Maps& maps, long long n, void* stream) {
    using L = Lay<T, KD, VD, kOut, kDots>;
    launch_after(tc_kernel<T, KD, VD, kOut, kDots>, dim3((unsigned)n), dim3(L::kThreads), L::kEnd, stream, w, maps);
  }
  static void run(const Walk& w, const Maps& maps, int dots, void* stream) {
    const long long blocks = (long long)w.B * w.H;
    if (!w.gates_there) launch(tc_gates_kernel<T>, dim3((unsigned)((blocks * w.chunks + 3) / 4)), dim3(128), 0, stream, w);
    if (w.segs > 1) go<false, 0>(w, maps, blocks * (w.segs - 1), stream);
    if (dots == 0) go<true, 0>(w, maps, blocks * w.segs, stream);
    else if (dots == 1) go<true, 1>(w, maps, blocks * w.segs, stream);
    else go<true, 2>(w, maps, blocks * w.segs, stream);
  }
};
// fn(Width) for a walk's widths
template <typename F>
auto with_width(int dtype, const Walk& w, F&& fn) {
  auto widths = [&](auto zero) {
    using T = decltype(zero);
    if (w.k.d <= 64) return w.v.d <= 64 ? fn(Width<T, 64, 64>()) : fn(Width<T, 64, 128>());
    return w.v.d <= 64 ? fn(Width<T, 128, 64>()) : fn(Width<T, 128, 128>());
  };
  return dtype == MEGA_BF16 ? widths(__nv_bfloat16()) : widths(__half());
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
  // A call of up to 64 steps is half a chunk here and one of the other form: 72 us for 34, 64 sequences x 64 steps x 16 heads of 64, 18.6 for
  // 12.1 with one sequence; at 300 steps it is 23 for 33, at 8 x 1024 33 for 91.
  if (w.L <= kTcChunk / 2) return false;
  if (dtype == MEGA_F32 || g_options[OPT_DISABLE_MMA].load() || w.piece < 16) return false;
  for (const Operand* o : {&w.q, &w.k, &w.v, &w.x})
    if (o->p && (o->d > kTcMost || o->vec < 16 || o->sl < 0 || o->sh < 0 || o->sb < 0 || (o->sl == 0 && w.L > 1))) return false;
  Maps m;   // (what the driver refuses, or the compiler did not give, is known before a plan is made)
  return maps_of(&m, dtype, w) && with_width(dtype, w, [](auto width) { return width.takes_all(); });
}
int tc_walk(int dtype, const Walk& w, int dots, void* stream) {
  Maps m;
  if (!maps_of(&m, dtype, w)) return MEGA_ERR_UNSUPPORTED;
  Walk bounded = w;
  const int limit = g_options[OPT_WAIT_LIMIT].load(), withhold = g_options[OPT_WITHHOLD_LOAD].load();
  bounded.wait_limit = limit > 0 ? (long long)limit : 4000000000LL;
  bounded.withhold = withhold > 0 ? withhold : -1;
  with_width(dtype, w, [&](auto width) { width.run(bounded, m, dots, stream); });
  g_last_kernel.store("decayed_attention_tc", std::memory_order_relaxed);
  return MEGA_OK;
}
cudaError_t tc_read_device_error(int* v, bool reset) { return read_device_error(v, reset); }
}  // namespace mega

// What the forms of linear attention with a decay for each head share (decayed_attention.cu has the mathematics).
#pragma once
#include <type_traits>

#include "common.cuh"

namespace mega {

struct Operand {
  const void* p;
  long long sb, sl, sh;   // strides in elements; the last axis is contiguous
  int d, vec;             // width; bytes of a piece that every row's start and width are multiples of
};

// One walk over the steps of every (sequence, head)
struct Walk {
  Operand q, k, v, x;     // queries, keys, values; x: what the outputs are multiplied with for the gates' gradient
  void* out;
  long long ob, ol, oh;
  int piece;              // bytes of a piece of an output row that every row's start and width are multiples of
  const void* f;
  long long fb, fl, fh;
  int f_dtype;
  const uint8_t *pad, *reset;
  const float* s_in;
  float* s_out;
  int s_row, s_col;       // strides of the states that come in and go out: (keys, values) of this walk
  float2* dots;           // [tile][B H][L]: x . out of the part from the state that entered; the pairs' sum W of a step
  void* anchors;          // [B H][chunk][tile] states that enter a chunk, in the activations' type (written, or read:)
  float* units;           // [B H][chunk][tile]: fp16: what those states are to be multiplied with
  float* through;         // [B H][chunk][part]: what passes the whole chunk
  void* gates;            // [B H][chunk]: what the tensor memory's form reads of the gates
  int gates_there;        // (an earlier walk has left them)
  float *local, *factor;  // states that segments leave by themselves, and their decay
  int B, L, H, tiles, chunks, per, segs;
  float p_scale, o_scale, s_scale;
  int rev, excl;
  long long wait_limit;   // SM cycles after which a wait of the tensor memory's form gives up
  int withhold;           // a test: chunk of each block whose keys are never loaded, or -1
};

// The walk of dq leaves a chunk's state where its weight in the next one is above zero; that of dk, whose sum of the same gates may round
// otherwise, reads it where the weight is well above.
constexpr float kLeast = 1e-35f;

// fp16 has five bits of exponent: what is rounded to it on the way to a product is first multiplied with a power of two that brings the
// largest value to 2^14 or above, and the product's fp32 sum with its inverse.  (Weighted keys as they are would be multiples of 2^-24:
// the state of gradients of 1e-3 was off by 7e-4, of 1e-5 by 6e-2.)  bf16 has fp32's exponents.
template <typename T>
constexpr bool kScaled = std::is_same<T, __half>::value;
// the power, from the biased exponent of the largest value; what is not finite stays as it is
__device__ __forceinline__ int scale_of(int exponent) { return exponent == 255 ? 0 : min(141 - exponent, 100); }
__device__ __forceinline__ float two_to(int n) { return __int_as_float((127 + n) << 23); }

// (gates are of the activations' type or fp32)
template <typename T>
__device__ __forceinline__ float gate_value(const Walk& w, long long at) {
  return w.f_dtype == MEGA_F32 ? __ldg(static_cast<const float*>(w.f) + at) : Elem<T>::ld(static_cast<const T*>(w.f) + at);
}

// The gates of a chunk of 32 N steps, N steps of the walk to a lane
template <int N>
struct GateIn {
  float f[N];
  unsigned pad, reset;
};
template <int N>
__device__ __forceinline__ int gate_row(const Walk& w, int lane, int i) {
  const int p = N * lane + i;
  return w.rev ? 32 * N - 1 - p : p;
}
template <typename T, int N>
__device__ __forceinline__ GateIn<N> gates_fetch(const Walk& w, int b, int h, int tile, int lane) {
  GateIn<N> g;
  g.pad = (1u << N) - 1, g.reset = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    g.f[i] = 0.f;
    const long long t = (long long)tile * (32 * N) + gate_row<N>(w, lane, i);
    if (t >= w.L) continue;
    g.f[i] = gate_value<T>(w, b * w.fb + t * w.fl + h * w.fh);
    if (!w.pad || !w.pad[b * (long long)w.L + t]) g.pad &= ~(1u << i);
    if (w.reset && w.reset[b * (long long)w.L + t]) g.reset |= 1u << i;
  }
  return g;
}
// What they come to: running sum of log2 a (whole numbers of 2^-40: their order does not matter, so both directions agree), resets so far, weight of a step in the state that leaves, and the weight of
// the state that enters in it (0: a reset lies between).  A gate whose decay is below fp32's range counts as a reset.
template <int N>
struct GateOut {
  long long sum[N], all;
  int count[N];
  float weight[N], enter, bad;   // bad: what the sums have to be given besides, 0 or NaN
  int total;
  bool padded;
};
// log2 sigmoid(f), and whether that is no decay but a reset
__device__ __forceinline__ float log2_gate(float f) { return (fminf(f, 0.f) - log1pf(expf(-fabsf(f)))) * 1.44269504f; }
__device__ __forceinline__ bool closed(float g) { return g < -149.f; }
__device__ __forceinline__ float gate_sum(long long s) { return (float)s * 0x1p-40f; }
template <int N>
__device__ __forceinline__ GateOut<N> gates_scan(const Walk& w, const GateIn<N>& in, int lane) {
  long long s[N], sum = 0;
  int c[N], cnt = 0;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float g = in.pad >> i & 1 ? 0.f : log2_gate(in.f[i]);
    c[i] = (in.reset >> i & 1) || closed(g);
    nan = nan || g != g;
    s[i] = c[i] ? 0 : (long long)(g * 0x1p40f);
    sum += s[i], cnt += c[i];
  }
  long long upto = sum;
  int counted = cnt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(~0u, upto, o);
    const int v = __shfl_up_sync(~0u, counted, o);
    if (lane >= o) upto += u, counted += v;
  }
  const float bad = __any_sync(~0u, nan) ? __int_as_float(0x7fffffff) : 0.f;   // (a gate that is NaN: the whole chunk is)
  const long long all = __shfl_sync(~0u, upto, 31);
  GateOut<N> r;
  r.all = all;
  r.total = __shfl_sync(~0u, counted, 31);
  upto -= sum, counted -= cnt;   // (what lies before this lane's steps)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!w.excl) upto += s[i], counted += c[i];
    r.sum[i] = upto, r.count[i] = counted;
    r.weight[i] = counted == r.total && !(in.pad >> i & 1) ? w.s_scale * exp2f(gate_sum(all - upto) + bad) : 0.f;
    if (w.excl) upto += s[i], counted += c[i];
  }
  r.enter = r.total ? 0.f : exp2f(gate_sum(all) + bad);
  r.bad = bad;
  r.padded = __any_sync(~0u, in.pad != 0);
  return r;
}

// The form on tcgen05 products (decayed_attention_tc.cu): 16-bit activations, heads of at most 128 keys and values
constexpr int kTcChunk = 128, kTcMost = 128, kTcParts = 8, kTcDots = 2, kTcGates = 1280;   // shares of Walk::through and Walk::dots
bool tc_takes(int dtype, const Walk& w);
int tc_walk(int dtype, const Walk& w, int dots, void* stream);
cudaError_t tc_read_device_error(int* v, bool reset);
cudaError_t decayed_attention_read_device_error(int* v, bool reset);

}  // namespace mega

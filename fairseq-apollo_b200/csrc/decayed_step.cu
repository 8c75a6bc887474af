// One step of linear attention with a decay for each head: S' = a S + k v^T, y = scale S'^T q, a = sigmoid(f), per sequence and head.
//
// The state is all there is to move (K V values in and out in fp32, against 2 K + 2 V + 1 of activations).  A block takes kCols
// columns (values) of a state, which need nothing of the others: a thread keeps one place of kVec columns and walks the keys in
// strides, so that a warp reads whole rows of the block's columns, and has all its rows under way at once; y is summed over the
// threads of a column in shared memory, in a fixed order.  Measured: 64 sequences x 16 heads of 128 x 128 26.7 us, 5.1 TB/s or 0.78 of the
// copy rate; whole rows of 128 to a block (16 keys to a thread) 28.7.  Small calls are the host's 6 us.
#include <algorithm>

#include "common.cuh"

namespace mega {
namespace {

constexpr int kThreads = 256;

struct Step {
  const void *q, *k, *v, *f;
  long long qb, qh, kb, kh, vb, vh, fb, fh, yb, yh;
  void* y;
  const float* h_in;
  float* h_out;
  int H, K, V, f_dtype;
  float scale;
};

template <int VEC>
struct Piece {
  float v[VEC];
};
template <int VEC>
__device__ __forceinline__ Piece<VEC> load_piece(const float* p) {
  Piece<VEC> r;
  if constexpr (VEC == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}

// LANES threads side by side hold LANES * VEC columns; ROWS: keys that a thread holds at a time
template <typename T, int VEC, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) step_kernel(const Step a) {
  constexpr int kCols = LANES * VEC, kGroups = kThreads / LANES;
  __shared__ float sq[MEGA_ATT_MOST], sk[MEGA_ATT_MOST], part[kGroups][kCols + 1];
  const int tid = threadIdx.x, b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int col = blockIdx.y * kCols + (tid % LANES) * VEC, grp = tid / LANES;
  const bool in = col < a.V;
  const float* s = a.h_in ? a.h_in + (long long)blockIdx.x * a.K * a.V : nullptr;
  float* to = a.h_out + (long long)blockIdx.x * a.K * a.V;
  Piece<VEC> st[ROWS];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = r0 + i * kGroups;
      if (s && in && r < a.K) st[i] = load_piece<VEC>(s + (long long)r * a.V + col);
      else
#pragma unroll
        for (int j = 0; j < VEC; ++j) st[i].v[j] = 0.f;
    }
  };
  fetch(grp);
  const T *q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh, *k = static_cast<const T*>(a.k) + b * a.kb + h * a.kh;
  for (int i = tid; i < a.K; i += kThreads) {
    sq[i] = Elem<T>::ld(q + i);
    sk[i] = Elem<T>::ld(k + i);
  }
  const long long fat = b * a.fb + h * a.fh;
  const float f = a.f_dtype == MEGA_F32 ? __ldg(static_cast<const float*>(a.f) + fat) : Elem<T>::ld(static_cast<const T*>(a.f) + fat);
  const float decay = gate_of<float>(f).s;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + h * a.vh + col;
  float val[VEC], sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) val[j] = in ? Elem<T>::ld(v + j) : 0.f, sum[j] = 0.f;
  __syncthreads();
  for (int r0 = grp; r0 < a.K; r0 += ROWS * kGroups) {
    if (r0 != grp) fetch(r0);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = r0 + i * kGroups;
      if (r >= a.K || !in) continue;
      const float kk = sk[r], qq = sq[r];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        st[i].v[j] = decay * st[i].v[j] + kk * val[j];
        sum[j] += qq * st[i].v[j];
      }
      if constexpr (VEC == 4) *reinterpret_cast<float4*>(to + (long long)r * a.V + col) = make_float4(st[i].v[0], st[i].v[1], st[i].v[2], st[i].v[3]);
      else to[(long long)r * a.V + col] = st[i].v[0];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) part[grp][(tid % LANES) * VEC + j] = sum[j];
  __syncthreads();
  for (int c = tid; c < kCols; c += kThreads) {
    float y = 0.f;
#pragma unroll 8
    for (int i = 0; i < kGroups; ++i) y += part[i][c];
    const int at = blockIdx.y * kCols + c;
    if (at < a.V) Elem<T>::st(static_cast<T*>(a.y) + b * a.yb + h * a.yh + at, a.scale * y);
  }
}

template <typename T>
void run(const Step& a, int B, bool four, void* stream) {
  const dim3 block(kThreads);
  auto grid = [&](int cols) { return dim3((unsigned)(B * a.H), (unsigned)((a.V + cols - 1) / cols)); };
  if (!four) launch(step_kernel<T, 1, 32, 8>, grid(32), block, 0, stream, a);
  else launch(step_kernel<T, 4, 8, 4>, grid(32), block, 0, stream, a);
}
}  // namespace
}  // namespace mega

using namespace mega;

extern "C" MEGA_API int mega_decayed_attention_step(const mega_decayed_attention_args* a, mega_stream_t stream) {
  if (!a) return MEGA_ERR_NULL;
  if (!valid_dtype(a->dtype) || (a->gate_dtype != MEGA_F32 && a->gate_dtype != a->dtype)) return MEGA_ERR_DTYPE;
  if (a->B <= 0 || a->L != 1 || a->H <= 0 || a->K <= 0 || a->V <= 0) return MEGA_ERR_SHAPE;
  if (a->K > MEGA_ATT_MOST || a->V > MEGA_ATT_MOST || (long long)a->B * a->H > 0x7fffffffLL || a->pad_mask || a->reset_mask) return MEGA_ERR_UNSUPPORTED;
  if (!a->q || !a->k || !a->v || !a->f || !a->y || !a->h_out) return MEGA_ERR_NULL;
  for (const void* p : {a->q, a->k, a->v, (const void*)a->y})
    if (!aligned_to(p, elem_size(a->dtype))) return MEGA_ERR_ALIGN;
  if (!aligned_to(a->f, elem_size(a->gate_dtype)) || !aligned_to(a->h_in, 4) || !aligned_to(a->h_out, 4)) return MEGA_ERR_ALIGN;
  const Step s = {a->q, a->k, a->v, a->f, a->qs[0], a->qs[2], a->ks[0], a->ks[2], a->vs[0], a->vs[2], a->fs[0], a->fs[2], a->ys[0], a->ys[2],
                  a->y, a->h_in, a->h_out, a->H, a->K, a->V, a->gate_dtype, (float)a->scale};
  const bool four = a->V % 4 == 0 && aligned_to(a->h_in, 16) && aligned_to(a->h_out, 16);
  MEGA_DISPATCH_DTYPE(a->dtype, run<T>(s, a->B, four, stream));
  return check_launch("decayed_attention_step");
}

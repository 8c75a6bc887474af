// Gated linear recurrence: a decay per step, sequence and channel.
//
//   l_t = sigmoid(-f_t),  h_t = h_{t-1} - l_t h_{t-1} + c_t,  c_t = l_t x_t  or  sigmoid(i_t) x_t
//
// written with the leak l instead of the decay 1 - l: a gate that stands open (f >> 0) has a leak far below the spacing of
// floats next to 1, and 1 - l would round it to a few bits.
#include <algorithm>

#include "common.cuh"

namespace mega {

namespace {

constexpr int kSeg = 16;   // steps between two saved states

struct RecArgs {
  const void *x, *f, *i, *dy;
  void *y, *dx, *df, *di;
  long long xsb, xsl, fsb, fsl, isb, isl, ysb, ysl, gsb, gsl, dxb, dxl, dfb, dfl, dib, dil;
  const unsigned char *pad, *reset;
  const float *h_in, *dh_out;
  float *h_out, *starts, *dh_in;
  int B, L, D, reverse;
};

template <typename T>
__device__ __forceinline__ float leak_of(float f) {
  const float e = 1.f + exp_of<T>(f);
  return sizeof(T) == 4 ? 1.f / e : rcp_approx(e);
}

template <typename T>
__global__ void __launch_bounds__(128) rec_fwd_kernel(RecArgs a) {
  const int b = blockIdx.y, d = blockIdx.x * 128 + threadIdx.x;
  if (d >= a.D) return;
  float h = a.h_in ? a.h_in[(long long)b * a.D + d] : 0.f;
  const int nseg = (a.L + kSeg - 1) / kSeg;
  for (int k = 0; k < a.L; ++k) {
    const int t = a.reverse ? a.L - 1 - k : k;
    if (a.starts && k % kSeg == 0) a.starts[((long long)b * nseg + k / kSeg) * a.D + d] = h;
    if (a.reset && a.reset[(long long)b * a.L + t]) h = 0.f;
    float y = 0.f;
    if (!(a.pad && a.pad[(long long)b * a.L + t])) {
      const float x = Elem<T>::ld((const T*)a.x + b * a.xsb + t * a.xsl + d);
      const float l = leak_of<T>(Elem<T>::ld((const T*)a.f + b * a.fsb + t * a.fsl + d));
      h = a.i ? fmaf(-l, h, fmaf(leak_of<T>(-Elem<T>::ld((const T*)a.i + b * a.isb + t * a.isl + d)), x, h)) : fmaf(l, x - h, h);
      y = h;
    }
    Elem<T>::st((T*)a.y + b * a.ysb + t * a.ysl + d, y);
  }
  if (a.h_out) a.h_out[(long long)b * a.D + d] = h;
}

template <typename T>
__global__ void __launch_bounds__(128) rec_bwd_kernel(RecArgs a) {
  const int b = blockIdx.y, d = blockIdx.x * 128 + threadIdx.x;
  if (d >= a.D) return;
  float q = a.dh_out ? a.dh_out[(long long)b * a.D + d] : 0.f;
  const int nseg = (a.L + kSeg - 1) / kSeg;
  for (int s = nseg - 1; s >= 0; --s) {
    const int n = min(kSeg, a.L - s * kSeg);
    float h = a.starts[((long long)b * nseg + s) * a.D + d];
    float hp[kSeg];
    for (int j = 0; j < n; ++j) {
      const int k = s * kSeg + j, t = a.reverse ? a.L - 1 - k : k;
      if (a.reset && a.reset[(long long)b * a.L + t]) h = 0.f;
      hp[j] = h;
      if (a.pad && a.pad[(long long)b * a.L + t]) continue;
      const float x = Elem<T>::ld((const T*)a.x + b * a.xsb + t * a.xsl + d);
      const float l = leak_of<T>(Elem<T>::ld((const T*)a.f + b * a.fsb + t * a.fsl + d));
      h = a.i ? fmaf(-l, h, fmaf(leak_of<T>(-Elem<T>::ld((const T*)a.i + b * a.isb + t * a.isl + d)), x, h)) : fmaf(l, x - h, h);
    }
    for (int j = n - 1; j >= 0; --j) {
      const int k = s * kSeg + j, t = a.reverse ? a.L - 1 - k : k;
      float dx = 0.f, df = 0.f, di = 0.f;
      if (!(a.pad && a.pad[(long long)b * a.L + t])) {
        const float x = Elem<T>::ld((const T*)a.x + b * a.xsb + t * a.xsl + d);
        const float l = leak_of<T>(Elem<T>::ld((const T*)a.f + b * a.fsb + t * a.fsl + d));
        const float g = q + Elem<T>::ld((const T*)a.dy + b * a.gsb + t * a.gsl + d);
        q = fmaf(-l, g, g);
        if (a.i) {
          const float w = Elem<T>::ld((const T*)a.i + b * a.isb + t * a.isl + d), s1 = leak_of<T>(-w);
          dx = s1 * g;
          df = q * l * hp[j];
          di = dx * leak_of<T>(w) * x;
        } else {
          dx = l * g;
          df = q * l * (hp[j] - x);
        }
      }
      if (a.reset && a.reset[(long long)b * a.L + t]) q = 0.f;
      Elem<T>::st((T*)a.dx + b * a.dxb + t * a.dxl + d, dx);
      Elem<T>::st((T*)a.df + b * a.dfb + t * a.dfl + d, df);
      if (a.i) Elem<T>::st((T*)a.di + b * a.dib + t * a.dil + d, di);
    }
  }
  if (a.dh_in) a.dh_in[(long long)b * a.D + d] = q;
}

template <typename T>
__global__ void __launch_bounds__(128) rec_step_kernel(RecArgs a) {
  const int b = blockIdx.y, d = blockIdx.x * 128 + threadIdx.x;
  if (d >= a.D) return;
  const long long at = (long long)b * a.D + d;
  const float h = a.h_in ? a.h_in[at] : 0.f, x = Elem<T>::ld((const T*)a.x + b * a.xsb + d);
  const float l = leak_of<T>(Elem<T>::ld((const T*)a.f + b * a.fsb + d));
  const float v = a.i ? fmaf(-l, h, fmaf(leak_of<T>(-Elem<T>::ld((const T*)a.i + b * a.isb + d)), x, h)) : fmaf(l, x - h, h);
  Elem<T>::st((T*)a.y + b * a.ysb + d, v);
  a.h_out[at] = v;
}

int check_rec(int dtype, int B, int L, int D, std::initializer_list<const void*> acts, std::initializer_list<const void*> f32) {
  if (!valid_dtype(dtype)) return MEGA_ERR_DTYPE;
  if (B <= 0 || L <= 0 || D <= 0) return MEGA_ERR_SHAPE;
  if (B > 65535) return MEGA_ERR_UNSUPPORTED;
  for (const void* p : acts)
    if (!aligned_to(p, elem_size(dtype))) return MEGA_ERR_ALIGN;
  for (const void* p : f32)
    if (!aligned_to(p, 4)) return MEGA_ERR_ALIGN;
  return MEGA_OK;
}

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int mega_gated_recurrence_segment(int dtype, int gated) { return valid_dtype(dtype) ? kSeg : 0; }

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
  a.B = B, a.L = L, a.D = D, a.reverse = (flags & MEGA_REC_REVERSE) != 0;
  MEGA_DISPATCH_DTYPE(dtype, launch(rec_fwd_kernel<T>, dim3((D + 127) / 128, B), dim3(128), 0, stream, a));
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
  a.B = B, a.L = L, a.D = D, a.reverse = (flags & MEGA_REC_REVERSE) != 0;
  MEGA_DISPATCH_DTYPE(dtype, launch(rec_bwd_kernel<T>, dim3((D + 127) / 128, B), dim3(128), 0, stream, a));
  return check_launch("gated_recurrence_bwd");
}

extern "C" int mega_gated_recurrence_step(const void* x, const void* f, const void* i, void* y, int dtype, int B, int D, int64_t xsb,
                                          int64_t fsb, int64_t isb, int64_t ysb, const float* h_in, float* h_out,
                                          mega_stream_t stream) {
  if (!x || !f || !y || !h_out) return MEGA_ERR_NULL;
  if (int rc = check_rec(dtype, B, 1, D, {x, f, i, y}, {h_in, h_out})) return rc;
  RecArgs a = {};
  a.x = x, a.f = f, a.i = i, a.y = y, a.xsb = xsb, a.fsb = fsb, a.isb = isb, a.ysb = ysb;
  a.h_in = h_in, a.h_out = h_out, a.B = B, a.L = 1, a.D = D;
  MEGA_DISPATCH_DTYPE(dtype, launch(rec_step_kernel<T>, dim3((D + 127) / 128, B), dim3(128), 0, stream, a));
  return check_launch("gated_recurrence_step");
}

// Group norm over a sequence with an activation, channels last, forward and backward.
//
//   xhat = (x - mean) * rstd, z = xhat * scale + beta, y = z * sigmoid(z)
//   dz = dy * s * (1 + z (1 - s)), s = sigmoid(z);  dn = dz * scale
//   dx = rstd * (dn - mean(dn) - xhat * mean(dn * xhat)),  dgamma = sum dz * xhat,  dbeta = sum dz
#include <algorithm>

#include "common.cuh"

namespace mega {

namespace {

struct GnArgs {
  const void *x, *dy;
  void* out;
  long long xsb, xsl, gsb, gsl, osb, osl;
  const float *gamma, *beta;
  const unsigned char* mask;
  int B, L, D, G;
  float eps;
  float offset;
  long long* count;
  float *mean, *rstd;
  float* sums;   // (B, G, 2): mean of dn, of dn xhat
  float *dgamma, *dbeta;
};

// z's activation and its slope
template <bool kSilu>
__device__ __forceinline__ void act_of(float z, float& y, float& slope) {
  if (!kSilu) {
    y = z, slope = 1.f;
    return;
  }
  const float s = 1.f / (1.f + expf(-z));
  y = z * s;
  slope = s * fmaf(z, 1.f - s, 1.f);
}

__device__ float block_sum(float v) {   // 256 threads; the sum in every thread
  __shared__ float part[8];
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < 8; ++w) v += part[w];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) gn_stats_kernel(GnArgs a) {
  const int g = blockIdx.x, b = blockIdx.y, gs = a.D / a.G;
  const T* x = (const T*)a.x + b * a.xsb + (long long)g * gs;
  const unsigned char* mask = a.mask ? a.mask + (long long)b * a.L : nullptr;
  const long long n = (long long)a.L * gs;
  float live = 0.f, s = 0.f;
  for (long long e = threadIdx.x; e < n; e += 256) {
    const int l = (int)(e / gs), c = (int)(e - (long long)l * gs);
    if (mask && mask[l]) continue;
    live += 1.f;
    s += Elem<T>::ld(x + l * a.xsl + c);
  }
  const float num = block_sum(live), inv = num > 0.f ? 1.f / num : 0.f, m = block_sum(s) * inv;
  float q = 0.f;
  for (long long e = threadIdx.x; e < n; e += 256) {
    const int l = (int)(e / gs), c = (int)(e - (long long)l * gs);
    if (mask && mask[l]) continue;
    const float v = Elem<T>::ld(x + l * a.xsl + c) - m;
    q = fmaf(v, v, q);
  }
  q = block_sum(q) * inv;
  if (threadIdx.x == 0) {
    a.mean[(long long)b * a.G + g] = m;
    a.rstd[(long long)b * a.G + g] = rsqrtf(q + a.eps);
    if (g == 0) {
      long long c = a.L;
      for (int l = 0; mask && l < a.L; ++l) c -= mask[l] != 0;
      a.count[b] = c;
    }
  }
}

template <typename T, bool kSilu>
__global__ void __launch_bounds__(256) gn_apply_kernel(GnArgs a) {
  const int l = blockIdx.x, b = blockIdx.y, gs = a.D / a.G;
  const T* x = (const T*)a.x + b * a.xsb + l * a.xsl;
  T* y = (T*)a.out + b * a.osb + l * a.osl;
  const bool pad = a.mask && a.mask[(long long)b * a.L + l];
  for (int d = threadIdx.x; d < a.D; d += 256) {
    const long long at = (long long)b * a.G + d / gs;
    float v = 0.f, slope;
    if (!pad) act_of<kSilu>(fmaf((Elem<T>::ld(x + d) - a.mean[at]) * a.rstd[at], a.gamma[d] + a.offset, a.beta[d]), v, slope);
    Elem<T>::st(y + d, v);
  }
}

// xhat and dz of one value
template <typename T, bool kSilu>
__device__ __forceinline__ float2 grads_of(const GnArgs& a, const T* x, const T* dy, int d, float m, float r) {
  float y, slope;
  const float xh = (Elem<T>::ld(x + d) - m) * r;
  act_of<kSilu>(fmaf(xh, a.gamma[d] + a.offset, a.beta[d]), y, slope);
  return make_float2(xh, Elem<T>::ld(dy + d) * slope);
}

template <typename T, bool kSilu>
__global__ void __launch_bounds__(256) gn_sums_kernel(GnArgs a) {
  const int g = blockIdx.x, b = blockIdx.y, gs = a.D / a.G;
  const long long at = (long long)b * a.G + g, n = (long long)a.L * gs;
  const float m = a.mean[at], r = a.rstd[at];
  float s = 0.f, q = 0.f;
  for (long long e = threadIdx.x; e < n; e += 256) {
    const int l = (int)(e / gs), d = g * gs + (int)(e - (long long)l * gs);
    if (a.mask && a.mask[(long long)b * a.L + l]) continue;
    const float2 v = grads_of<T, kSilu>(a, (const T*)a.x + b * a.xsb + l * a.xsl, (const T*)a.dy + b * a.gsb + l * a.gsl, d, m, r);
    const float dn = v.y * (a.gamma[d] + a.offset);
    s += dn;
    q = fmaf(dn, v.x, q);
  }
  s = block_sum(s), q = block_sum(q);
  if (threadIdx.x == 0) {
    const float num = (float)a.count[b] * gs, inv = num > 0.f ? 1.f / num : 0.f;
    a.sums[2 * at] = s * inv;
    a.sums[2 * at + 1] = q * inv;
  }
}

template <typename T, bool kSilu>
__global__ void __launch_bounds__(256) gn_dx_kernel(GnArgs a) {
  const int l = blockIdx.x, b = blockIdx.y, gs = a.D / a.G;
  const T *x = (const T*)a.x + b * a.xsb + l * a.xsl, *dy = (const T*)a.dy + b * a.gsb + l * a.gsl;
  T* dx = (T*)a.out + b * a.osb + l * a.osl;
  const bool pad = a.mask && a.mask[(long long)b * a.L + l];
  for (int d = threadIdx.x; d < a.D; d += 256) {
    const long long at = (long long)b * a.G + d / gs;
    float o = 0.f;
    if (!pad) {
      const float2 v = grads_of<T, kSilu>(a, x, dy, d, a.mean[at], a.rstd[at]);
      o = a.rstd[at] * (v.y * (a.gamma[d] + a.offset) - a.sums[2 * at] - v.x * a.sums[2 * at + 1]);
    }
    Elem<T>::st(dx + d, o);
  }
}

template <typename T, bool kSilu>
__global__ void __launch_bounds__(256) gn_params_kernel(GnArgs a) {
  const int gs = a.D / a.G, d = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float s = 0.f, q = 0.f;
  if (d < a.D)
    for (int b = 0; b < a.B; ++b) {
      const long long at = (long long)b * a.G + d / gs;
      for (int l = w; l < a.L; l += 8) {
        if (a.mask && a.mask[(long long)b * a.L + l]) continue;
        const float2 v = grads_of<T, kSilu>(a, (const T*)a.x + b * a.xsb + l * a.xsl, (const T*)a.dy + b * a.gsb + l * a.gsl, d,
                                            a.mean[at], a.rstd[at]);
        s += v.y;
        q = fmaf(v.y, v.x, q);
      }
    }
  __shared__ float part[2][8][32];
  part[0][w][threadIdx.x & 31] = s;
  part[1][w][threadIdx.x & 31] = q;
  __syncthreads();
  if (w == 0 && d < a.D) {
    s = q = 0.f;
    for (int k = 0; k < 8; ++k) s += part[0][k][threadIdx.x], q += part[1][k][threadIdx.x];
    a.dbeta[d] = s;
    a.dgamma[d] = q;
  }
}

int check_gn(int dtype, int B, int L, int D, int G, std::initializer_list<const void*> acts) {
  if (!valid_dtype(dtype)) return MEGA_ERR_DTYPE;
  if (B <= 0 || L <= 0 || D <= 0 || G <= 0 || D % G != 0) return MEGA_ERR_SHAPE;
  if (B > 65535 || G > 65535) return MEGA_ERR_UNSUPPORTED;
  for (const void* p : acts)
    if (!aligned_to(p, elem_size(dtype))) return MEGA_ERR_ALIGN;
  return MEGA_OK;
}

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int64_t mega_group_norm_work(int dtype, int B, int L, int D, int num_groups) {
  if (check_gn(dtype, B, L, D, num_groups, {})) return 0;
  return (int64_t)B * num_groups * 2 * sizeof(float);
}

extern "C" int mega_group_norm_fwd(const void* x, void* y, int dtype, int B, int L, int D, int64_t xsb, int64_t xsl, int64_t ysb,
                                   int64_t ysl, const float* gamma, const float* beta, const uint8_t* pad_mask, int num_groups,
                                   double eps, unsigned flags, int64_t* count, float* mean, float* rstd, void* work,
                                   mega_stream_t stream) {
  if (!x || !y || !gamma || !beta || !count || !mean || !rstd || !work) return MEGA_ERR_NULL;
  if (int rc = check_gn(dtype, B, L, D, num_groups, {x, y})) return rc;
  GnArgs a = {};
  a.x = x, a.out = y, a.xsb = xsb, a.xsl = xsl, a.osb = ysb, a.osl = ysl, a.gamma = gamma, a.beta = beta, a.mask = pad_mask;
  a.B = B, a.L = L, a.D = D, a.G = num_groups, a.eps = (float)eps, a.offset = flags & MEGA_GN_OFFSET ? 1.f : 0.f;
  a.count = (long long*)count, a.mean = mean, a.rstd = rstd;
  MEGA_DISPATCH_DTYPE(dtype, {
    launch(gn_stats_kernel<T>, dim3(num_groups, B), dim3(256), 0, stream, a);
    launch(flags & MEGA_GN_SILU ? gn_apply_kernel<T, true> : gn_apply_kernel<T, false>, dim3(L, B), dim3(256), 0, stream, a);
  });
  return check_launch("group_norm_fwd");
}

extern "C" int mega_group_norm_bwd(const void* dy, const void* x, void* dx, int dtype, int B, int L, int D, int64_t gsb, int64_t gsl,
                                   int64_t xsb, int64_t xsl, int64_t dsb, int64_t dsl, const float* gamma, const float* beta,
                                   const uint8_t* pad_mask, int num_groups, unsigned flags, const int64_t* count, const float* mean,
                                   const float* rstd, float* dgamma, float* dbeta, void* work, mega_stream_t stream) {
  if (!dy || !x || !dx || !gamma || !beta || !count || !mean || !rstd || !dgamma || !dbeta || !work) return MEGA_ERR_NULL;
  if (int rc = check_gn(dtype, B, L, D, num_groups, {dy, x, dx})) return rc;
  GnArgs a = {};
  a.x = x, a.dy = dy, a.out = dx, a.xsb = xsb, a.xsl = xsl, a.gsb = gsb, a.gsl = gsl, a.osb = dsb, a.osl = dsl;
  a.gamma = gamma, a.beta = beta, a.mask = pad_mask;
  a.B = B, a.L = L, a.D = D, a.G = num_groups, a.offset = flags & MEGA_GN_OFFSET ? 1.f : 0.f;
  a.count = (long long*)count, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.sums = (float*)work, a.dgamma = dgamma, a.dbeta = dbeta;
  const bool silu = flags & MEGA_GN_SILU;
  MEGA_DISPATCH_DTYPE(dtype, {
    launch(silu ? gn_sums_kernel<T, true> : gn_sums_kernel<T, false>, dim3(num_groups, B), dim3(256), 0, stream, a);
    launch(silu ? gn_dx_kernel<T, true> : gn_dx_kernel<T, false>, dim3(L, B), dim3(256), 0, stream, a);
    launch(silu ? gn_params_kernel<T, true> : gn_params_kernel<T, false>, dim3((D + 31) / 32), dim3(256), 0, stream, a);
  });
  return check_launch("group_norm_bwd");
}

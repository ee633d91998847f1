// groupnorm.hip -- group norm with an activation and an optional residual on channels-last tensors.
// Contract: include/propainter_mi355.h (pp_groupnorm).
//
//   mean = sum x / M, var = sum x^2 / M - mean^2 over the M = HW * C/G values of a group;  y = post(skip + act((x - mean) r gamma + beta))
//
// The sums are held in double (a product of two f32 values is exact there, so sum x^2 / M - mean^2 loses nothing that f32 data
// holds until |mean| / std passes 10^6); f64 multiply-adds run at the rate of f32 ones, far above what memory delivers.  The mean is applied
// as an f32 pair (high, low), so the subtraction is as exact as the data.
#include "bf16_device.h"
#include "pp_host.h"

#include <type_traits>

namespace pp {

struct GroupNormK {
  const void* x;
  void* y;
  const void* skip;
  const float* gamma;
  const float* beta;
  double* partials;  // [N][nchunks][G][2], then the finished statistics [N][G] as (mean high, mean low, 1/std, -) floats
  int64_t x_ldc, y_ldc, skip_ldc, HW;
  int64_t per;  // pixels of a chunk
  int N, C, G, cpg, nchunks, cols, lanes;  // cols: column vectors of a work-group pass, lanes: pixels that it takes at once
  int act, relu_post;
  float eps, act_param;
};

template <typename T, int V>
struct Vec;
template <typename T>
struct Vec<T, 1> {
  static __device__ __forceinline__ void ld(const T* p, float* f) { f[0] = to_f32(*p); }
  static __device__ __forceinline__ void st(T* p, const float* f) { *p = from_f32<T>(f[0]); }
};
template <typename T>
struct Vec<T, 8> {
  static __device__ __forceinline__ void ld(const T* p, float* f) { ld8(p, f); }
  static __device__ __forceinline__ void st(T* p, const float* f) { st8(p, f); }
};
template <>
struct Vec<float, 4> {
  static __device__ __forceinline__ void ld(const float* p, float* f) {
    const f4 v = *reinterpret_cast<const f4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v[i];
  }
  static __device__ __forceinline__ void st(float* p, const float* f) { *reinterpret_cast<f4*>(p) = f4{f[0], f[1], f[2], f[3]}; }
};

__device__ __forceinline__ float norm_act(float v, int act, float param) {
  switch (act) {
    case PP_ACT_RELU: return v > 0.f || v != v ? v : 0.f;
    case PP_ACT_LEAKY: return v > 0.f ? v : v * param;
    case PP_ACT_SIGMOID: return 1.f / (1.f + expf(-v));
    case PP_ACT_TANH: return tanhf(v);
    case PP_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case PP_ACT_SILU: return v / (1.f + expf(-v));
    default: return v;
  }
}

// sums of one chunk of one image, all groups
template <typename T, int V>
__global__ void __launch_bounds__(256) groupnorm_sums_kernel(const GroupNormK k) {
  __shared__ double sh[256 * V * 2];
  const int n = (int)blockIdx.x / k.nchunks, chunk = (int)blockIdx.x - n * k.nchunks;
  const int tid = (int)threadIdx.x;
  const int64_t p0 = (int64_t)chunk * k.per, p1 = p0 + k.per < k.HW ? p0 + k.per : k.HW;
  double* dst = k.partials + ((int64_t)n * k.nchunks + chunk) * k.G * 2;
  const int pl = tid / k.cols, cv = tid - pl * k.cols;
  const int allcols = (k.C + V - 1) / V;
  for (int c0 = 0; c0 < allcols; c0 += k.cols) {
    const int col = c0 + cv;
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0;
    if (pl < k.lanes && col < allcols) {
      const T* base = (const T*)k.x + (int64_t)n * k.HW * k.x_ldc + (int64_t)col * V;
      for (int64_t p = p0 + pl; p < p1; p += k.lanes) {
        float v[V];
        Vec<T, V>::ld(base + p * k.x_ldc, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double d = (double)v[e];
          s[e] += d;
          q[e] += d * d;
        }
      }
    }
    __syncthreads();  // the previous pass's readers
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sh[(tid * V + e) * 2] = s[e];
      sh[(tid * V + e) * 2 + 1] = q[e];
    }
    __syncthreads();
    // groups that touch channels [a, b): thread g % 256 owns group g in every pass, so the running sums need no exchange
    const int a = c0 * V, b = (c0 + k.cols) * V < k.C ? (c0 + k.cols) * V : k.C;
    for (int g = tid; g < k.G; g += 256) {
      const int lo = a > g * k.cpg ? a : g * k.cpg, hi = b < (g + 1) * k.cpg ? b : (g + 1) * k.cpg;
      if (lo >= hi) continue;
      double ss = 0.0, qq = 0.0;
      for (int l = 0; l < k.lanes; ++l)
        for (int c = lo; c < hi; ++c) {
          ss += sh[(l * k.cols * V + c - a) * 2];
          qq += sh[(l * k.cols * V + c - a) * 2 + 1];
        }
      if (lo != g * k.cpg) {
        ss += dst[2 * g];
        qq += dst[2 * g + 1];
      }
      dst[2 * g] = ss;
      dst[2 * g + 1] = qq;
    }
  }
}

__device__ __forceinline__ f4 finish_stats(double s, double q, double m, float eps) {
  const double mean = s / m;
  double var = q / m - mean * mean;
  if (var < 0.0) var = 0.0;  // (a NaN stays one)
  const float hi = (float)mean;
  return f4{hi, (float)(mean - (double)hi), (float)(1.0 / sqrt(var + (double)eps)), 0.f};
}

__global__ void __launch_bounds__(256) groupnorm_finish_kernel(const GroupNormK k) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)k.N * k.G) return;
  const int64_t n = i / k.G, g = i - n * k.G;
  const double* src = k.partials + (n * k.nchunks * k.G + g) * 2;
  double s = 0.0, q = 0.0;
  for (int c = 0; c < k.nchunks; ++c) {
    s += src[(int64_t)c * k.G * 2];
    q += src[(int64_t)c * k.G * 2 + 1];
  }
  reinterpret_cast<f4*>(k.partials + (int64_t)k.N * k.nchunks * k.G * 2)[i] = finish_stats(s, q, (double)k.HW * k.cpg, k.eps);
}

template <typename T, int V>
__global__ void __launch_bounds__(256) groupnorm_apply_kernel(const GroupNormK k) {
  const int n = (int)blockIdx.x / k.nchunks, chunk = (int)blockIdx.x - n * k.nchunks;
  const int tid = (int)threadIdx.x;
  const int64_t p0 = (int64_t)chunk * k.per, p1 = p0 + k.per < k.HW ? p0 + k.per : k.HW;
  const f4* stats = reinterpret_cast<const f4*>(k.partials + (int64_t)k.N * k.nchunks * k.G * 2) + (int64_t)n * k.G;
  const int pl = tid / k.cols, cv = tid - pl * k.cols;
  const int allcols = (k.C + V - 1) / V;
  if (pl >= k.lanes) return;
  for (int col = cv; col < allcols; col += k.cols) {
    float mh[V], ml[V], a[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = col * V + e;
      const f4 st = stats[c / k.cpg];
      mh[e] = st[0];
      ml[e] = st[1];
      a[e] = k.gamma ? st[2] * k.gamma[c] : st[2];
      b[e] = k.beta ? k.beta[c] : 0.f;
    }
    const int64_t px = (int64_t)n * k.HW, c0 = (int64_t)col * V;
    for (int64_t p = p0 + pl; p < p1; p += k.lanes) {
      float v[V], sk[V];
      Vec<T, V>::ld((const T*)k.x + (px + p) * k.x_ldc + c0, v);
      if (k.skip) Vec<T, V>::ld((const T*)k.skip + (px + p) * k.skip_ldc + c0, sk);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = norm_act(((v[e] - mh[e]) - ml[e]) * a[e] + b[e], k.act, k.act_param);
        if (k.skip) v[e] += sk[e];
        if (k.relu_post) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;
      }
      Vec<T, V>::st((T*)k.y + (px + p) * k.y_ldc + c0, v);
    }
  }
}

}  // namespace pp

template <typename T, int V>
static int launch_groupnorm(void* stream, pp::GroupNormK& k) {
  using namespace pp;
  const int allcols = (k.C + V - 1) / V;
  k.cols = allcols < 256 ? allcols : 256;
  k.lanes = 256 / k.cols;
  const dim3 grid((unsigned)(k.N * k.nchunks));
  PP_LAUNCH((groupnorm_sums_kernel<T, V>), grid, dim3(256), 0, stream, k);
  int rc = pp_check_launch("pp_groupnorm(sums)");
  if (rc != PP_OK) return rc;
  PP_LAUNCH(groupnorm_finish_kernel, dim3(pp_blocks_1d((int64_t)k.N * k.G)), dim3(256), 0, stream, k);
  rc = pp_check_launch("pp_groupnorm(finish)");
  if (rc != PP_OK) return rc;
  PP_LAUNCH((groupnorm_apply_kernel<T, V>), grid, dim3(256), 0, stream, k);
  return pp_check_launch("pp_groupnorm(apply)");
}

extern "C" int32_t pp_groupnorm(void* stream, const pp_groupnorm_params* p) {
  using namespace pp;
  if (!p || !p->x || !p->y || !p->partials) return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: null argument");
  if (p->dtype != PP_F32 && p->dtype != PP_F16 && p->dtype != PP_BF16) return pp_fail(PP_ERR_UNSUPPORTED, "pp_groupnorm: dtype");
  if (p->N < 0 || p->HW < 0 || p->C < 1 || p->C > 65536 || p->groups < 1 || p->C % p->groups)
    return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: C must be in [1, 65536] and a multiple of groups");
  if (p->act < PP_ACT_NONE || p->act > PP_ACT_SILU) return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: act");
  if (p->x_ldc < p->C || p->y_ldc < p->C || (p->skip && p->skip_ldc < p->C))
    return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: channel pitch smaller than C");
  if (!(p->eps >= 0.f)) return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: eps must be >= 0");
  if ((uintptr_t)p->partials % 16) return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: partials must be 16-byte aligned");
  if (p->N == 0 || p->HW == 0) return PP_OK;  // nothing to write
  if (p->nchunks < 1 || p->nchunks > p->HW || p->nchunks > (1 << 20) || p->N > (1 << 23) || p->N * p->nchunks >= (1 << 23))
    return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: nchunks must be in [1, HW] and N * nchunks below 2^23");
  GroupNormK k;
  k.x = p->x; k.y = p->y; k.skip = p->skip;
  k.gamma = (const float*)p->gamma; k.beta = (const float*)p->beta;
  k.partials = (double*)p->partials;
  k.x_ldc = p->x_ldc; k.y_ldc = p->y_ldc; k.skip_ldc = p->skip_ldc; k.HW = p->HW;
  k.per = (p->HW + p->nchunks - 1) / p->nchunks;
  k.N = (int)p->N; k.C = (int)p->C; k.G = (int)p->groups; k.cpg = (int)(p->C / p->groups); k.nchunks = (int)p->nchunks;
  k.act = p->act; k.relu_post = p->relu_post; k.eps = p->eps; k.act_param = p->act_param;
  // 16-byte accesses where every row of every tensor allows them, single elements otherwise
  const int V = p->dtype == PP_F32 ? 4 : 8;
  const bool wide = p->C % V == 0 && p->x_ldc % V == 0 && p->y_ldc % V == 0 && (!p->skip || p->skip_ldc % V == 0) &&
                    (((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->skip) % 16) == 0;
  if (p->dtype == PP_F32) return wide ? launch_groupnorm<float, 4>(stream, k) : launch_groupnorm<float, 1>(stream, k);
  if (p->dtype == PP_F16) return wide ? launch_groupnorm<half_t, 8>(stream, k) : launch_groupnorm<half_t, 1>(stream, k);
  return wide ? launch_groupnorm<bf16_t, 8>(stream, k) : launch_groupnorm<bf16_t, 1>(stream, k);
}

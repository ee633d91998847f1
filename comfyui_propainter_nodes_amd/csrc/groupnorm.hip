// groupnorm.hip -- group norm with an activation and an optional residual on channels-last tensors.
// Contract: include/propainter_mi355.h (pp_groupnorm).
//
//   mean = sum x / M, var = sum x^2 / M - mean^2 over the M = HW * C/G values of a group;  y = post(skip + act((x - mean) r gamma + beta))
//
// The sums are held in double, where a product of two f32 values is exact: sum x^2 / M - mean^2 is (mean / std)^2 times a few 2^-53 off, relative to the
// variance.  (65536 f32 values, eps 0: results within 9e-8 of theirs at |mean| / std = 10^4, 4e-7 at 10^5, 2e-5 at 10^6, where f32 data has four
// bits below its standard deviation.)  f64 multiply-adds run at the rate of f32 ones, far above what memory delivers.  The mean is applied
// as an f32 pair (high, low), so the subtraction is as exact as the data.
//
// Bound by memory: 16 x 180 x 320 x 64 f32 with ReLU 149 us -- sums 55 us (236 MB at 4.3 TB/s), apply 82 us (472 MB at 5.8, partly from the
// cache); 16 x 90 x 160 x 96 f32 with a skip 72 us (354 MB at 4.9 TB/s); 16-bit storage with GELU by the vector ALU (6 x 181 x 243 x 320: apply 97 us
// for 338 MB).  A group that fits registers is one launch of 5.4 us (1 x 16 x 16 x 256).
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
  int relu_post, join;
  float eps, act_param;
};

#ifdef PP_EMU
inline float fast_exp2_(float x) { return exp2f(x); }
#else
__device__ __forceinline__ float fast_exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
#endif

// V consecutive elements: as they are loaded, and as floats
template <typename T, int V>
struct Vec {  // 16 bytes
  typedef u4 Raw;
  static_assert(V * sizeof(T) == 16, "");
  static __device__ __forceinline__ Raw ld(const T* p) { return *reinterpret_cast<const u4*>(p); }
  static __device__ __forceinline__ void floats(Raw r, float* f) {
    if constexpr (V == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, (unsigned)r[i]);
    } else {
      ld8(reinterpret_cast<const T*>(&r), f);
    }
  }
  static __device__ __forceinline__ void st(T* p, const float* f) {
    if constexpr (V == 4) *reinterpret_cast<f4*>(p) = f4{f[0], f[1], f[2], f[3]};
    else st8(p, f);
  }
};
template <typename T>
struct Vec<T, 1> {
  typedef T Raw;
  static __device__ __forceinline__ Raw ld(const T* p) { return *p; }
  static __device__ __forceinline__ void floats(Raw r, float* f) { f[0] = to_f32(r); }
  static __device__ __forceinline__ void st(T* p, const float* f) { *p = from_f32<T>(f[0]); }
};

// x Phi(x) = max(x, 0) - z Q(z), z = |x|, Q(z) = erfc(z / sqrt 2) / 2 = exp(-z^2 / 2) R(t), t = 1 / (1 + 0.36 z): R is a polynomial fitted to
// erfcx(z / sqrt 2) / 2 over z in [0, 14], 9e-7 off at most relative to Q (so both tails keep their relative accuracy).  max(x, 0) is
// (x + |x|) / 2, which a NaN passes.
__device__ __forceinline__ float gelu_fast(float x) {
  const float z = fminf(fabsf(x), 20.f);
  const float t = fast_rcp(__builtin_fmaf(z, 0.36f, 1.f));
  float r = 0.04705524072051048f;
  r = __builtin_fmaf(r, t, -0.17976124584674835f);
  r = __builtin_fmaf(r, t, 0.18094944953918457f);
  r = __builtin_fmaf(r, t, 0.02655242383480072f);
  r = __builtin_fmaf(r, t, 0.13971813023090363f);
  r = __builtin_fmaf(r, t, 0.14177265763282776f);
  r = __builtin_fmaf(r, t, 0.14371302723884583f);
  const float u = z * 0.84932180028801907f;  // exp(-z^2 / 2) = 2^(-u^2)
  const float q = fast_exp2_(-u * u) * (r * t);
  return __builtin_fmaf(-z, q, __builtin_fmaf(0.5f, fabsf(x), 0.5f * x));
}

// f32 storage: the library's functions; 16-bit storage: hardware exponential and reciprocal, each a few 2^-24 off.  The rounding of an exponential's
// argument makes the tails worse, in proportion to it: GELU's reach 3e-6 of the value where f16 ends (v = -5.6; to be rounded by up to 2^-11) and
// 2e-5 where bf16 does (v = -13; 2^-8).
template <typename T>
__device__ __forceinline__ float norm_act(float v, int act, float param) {  // act: a compile-time constant or uniform
  constexpr bool kExact = sizeof(T) == 4;
  switch (act) {
    case PP_ACT_RELU: return v > 0.f || v != v ? v : 0.f;
    case PP_ACT_LEAKY: return v > 0.f ? v : v * param;
    case PP_ACT_SIGMOID: return kExact ? 1.f / (1.f + expf(-v)) : sigmoidf_(v);
    case PP_ACT_TANH: return tanhf(v);
    case PP_ACT_GELU: return kExact ? 0.5f * v * (1.f + erff(v * 0.70710678118654752f)) : gelu_fast(v);
    case PP_ACT_SILU: return kExact ? v / (1.f + expf(-v)) : v * sigmoidf_(v);
    default: return v;
  }
}

constexpr int kOwnGroups = 32;  // groups and sums up to which the apply pass joins them itself
constexpr int kOwnSums = 2048;
constexpr int kAhead = 8;  // 16-byte loads of a thread in flight in the sums pass (16 x 180 x 320 x 64 f32: 4 149.4 us, 8 148.4)

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
    auto add = [&](typename Vec<T, V>::Raw raw) __attribute__((always_inline)) {
      float v[V];
      Vec<T, V>::floats(raw, v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double d = (double)v[e];
        s[e] += d;
        q[e] = __builtin_fma(d, d, q[e]);
      }
    };
    if (pl < k.lanes && col < allcols) {
      const T* base = (const T*)k.x + (int64_t)n * k.HW * k.x_ldc + (int64_t)col * V;
      const int64_t step = (int64_t)k.lanes * k.x_ldc;
      int64_t p = p0 + pl;
      const T* at = base + p * k.x_ldc;
      for (; p + (kAhead - 1) * k.lanes < p1; p += kAhead * k.lanes, at += kAhead * step) {
        typename Vec<T, V>::Raw v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = Vec<T, V>::ld(at + u * step);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) add(v[u]);
      }
      for (; p < p1; p += k.lanes, at += step) {
        add(Vec<T, V>::ld(at));
      }
    }
    __syncthreads();  // the previous pass's readers
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sh[(tid * V + e) * 2] = s[e];
      sh[(tid * V + e) * 2 + 1] = q[e];
    }
    __syncthreads();
    // a channel's pixel lanes, then a group's channels: thread g % 256 owns group g in every pass, so the running sums need no exchange
    const int wide = k.cols * V;
    for (int c = tid; c < wide; c += 256) {
      double ss = 0.0, qq = 0.0;
#pragma unroll 4
      for (int l = 0; l < k.lanes; ++l) {
        ss += sh[(l * wide + c) * 2];
        qq += sh[(l * wide + c) * 2 + 1];
      }
      sh[2 * c] = ss;
      sh[2 * c + 1] = qq;
    }
    __syncthreads();
    const int a = c0 * V, b = a + wide < k.C ? a + wide : k.C;
    for (int g = tid; g < k.G; g += 256) {
      const int lo = a > g * k.cpg ? a : g * k.cpg, hi = b < (g + 1) * k.cpg ? b : (g + 1) * k.cpg;
      if (lo >= hi) continue;
      double ss = 0.0, qq = 0.0;
      for (int c = lo; c < hi; ++c) {
        ss += sh[(c - a) * 2];
        qq += sh[(c - a) * 2 + 1];
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

// sum over the lanes of a wave, the same order for every lane
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = __builtin_bit_cast(unsigned, shfl_xor(__builtin_bit_cast(float, (unsigned)u), m));
    const unsigned hi = __builtin_bit_cast(unsigned, shfl_xor(__builtin_bit_cast(float, (unsigned)(u >> 32)), m));
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
  return v;
}

constexpr int kFinishBlocks = 2048;  // 8 work-groups per CU; more (image, group) pairs than they have waves go round again

// a wave per (image, group): its lanes share the chunks
__global__ void __launch_bounds__(256) groupnorm_finish_kernel(const GroupNormK k) {
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < (int64_t)k.N * k.G; i += (int64_t)gridDim.x * 4) {
    const int64_t n = i / k.G, g = i - n * k.G;
    const double* src = k.partials + (n * k.nchunks * k.G + g) * 2;
    double s = 0.0, q = 0.0;
    for (int c = lane_id(); c < k.nchunks; c += 64) {
      s += src[(int64_t)c * k.G * 2];
      q += src[(int64_t)c * k.G * 2 + 1];
    }
    s = wave_sum(s);
    q = wave_sum(q);
    if (lane_id() == 0)
      reinterpret_cast<f4*>(k.partials + (int64_t)k.N * k.nchunks * k.G * 2)[i] = finish_stats(s, q, (double)k.HW * k.cpg, k.eps);
  }
}

// What a vector of V channels needs: ((x - mh) - ml) a + b; with 16-bit storage x - mh is exact to 2^-24 of the larger one and -ml a goes
// into b, one operation less per value.
template <typename T, int V>
struct Affine {
  static constexpr bool kLow = sizeof(T) == 4;
  float mh[V], ml[kLow ? V : 1], a[V], b[V];
  __device__ __forceinline__ void set(const GroupNormK& k, int c, int e, f4 st) {
    mh[e] = st[0];
    a[e] = k.gamma ? st[2] * k.gamma[c] : st[2];
    b[e] = k.beta ? k.beta[c] : 0.f;
    if constexpr (kLow) ml[e] = st[1];
    else b[e] = __builtin_fmaf(-st[1], a[e], b[e]);
  }
  template <int ACT>
  __device__ __forceinline__ void apply(const GroupNormK& k, typename Vec<T, V>::Raw x, typename Vec<T, V>::Raw skip, T* dst) const {
    float v[V], sk[V];
    Vec<T, V>::floats(x, v);
    if (k.skip) Vec<T, V>::floats(skip, sk);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float d = v[e] - mh[e];
      if constexpr (kLow) d -= ml[e];
      v[e] = norm_act<T>(__builtin_fmaf(d, a[e], b[e]), ACT, k.act_param);
      if (k.skip) v[e] += sk[e];
      if (k.relu_post) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;
    }
    Vec<T, V>::st(dst, v);
  }
};

// Chunks are taken in the opposite order of the sums: what they read last is still in the cache.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) groupnorm_apply_kernel(const GroupNormK k) {
  const int id = (int)(gridDim.x - 1 - blockIdx.x), n = id / k.nchunks, chunk = id - n * k.nchunks;
  const int tid = (int)threadIdx.x;
  const int64_t p0 = (int64_t)chunk * k.per, p1 = p0 + k.per < k.HW ? p0 + k.per : k.HW;
  __shared__ f4 own[kOwnGroups];
  __shared__ double sh[512];
  const f4* stats = reinterpret_cast<const f4*>(k.partials + (int64_t)k.N * k.nchunks * k.G * 2) + (int64_t)n * k.G;
  if (k.join) {  // few enough sums: every work-group joins them itself, a launch less
    const int G2 = k.G <= 8 ? 8 : k.G <= 16 ? 16 : 32, g = tid % G2, part = tid / G2, parts = 256 / G2;
    const double* src = k.partials + ((int64_t)n * k.nchunks * k.G + g) * 2;
    double s = 0.0, q = 0.0;
    if (g < k.G) {
#pragma unroll 4
      for (int c = part; c < k.nchunks; c += parts) {
        s += src[(int64_t)c * k.G * 2];
        q += src[(int64_t)c * k.G * 2 + 1];
      }
    }
    sh[2 * tid] = s;
    sh[2 * tid + 1] = q;
    __syncthreads();
    if (tid < k.G) {
      for (int i = 1; i < parts; ++i) {
        s += sh[2 * (tid + i * G2)];
        q += sh[2 * (tid + i * G2) + 1];
      }
      own[tid] = finish_stats(s, q, (double)k.HW * k.cpg, k.eps);
    }
    __syncthreads();
    stats = own;
  }
  const int pl = tid / k.cols, cv = tid - pl * k.cols;
  const int allcols = (k.C + V - 1) / V;
  if (pl >= k.lanes) return;
  for (int col = cv; col < allcols; col += k.cols) {
    Affine<T, V> f;
#pragma unroll
    for (int e = 0; e < V; ++e) f.set(k, col * V + e, e, stats[(col * V + e) / k.cpg]);
    const int64_t px = (int64_t)n * k.HW, c0 = (int64_t)col * V;
    const T* x = (const T*)k.x + px * k.x_ldc + c0;
    const T* skip = (const T*)k.skip + px * k.skip_ldc + c0;
    T* y = (T*)k.y + px * k.y_ldc + c0;
    // (one vector at a time: with 4 in flight a thread holds 139 registers instead of 60 and 6 x 181 x 243 x 320 bf16 with GELU takes 158 us, not 146)
    for (int64_t p = p0 + pl; p < p1; p += k.lanes) {
      const auto v = Vec<T, V>::ld(x + p * k.x_ldc);
      f.template apply<ACT>(k, v, k.skip ? Vec<T, V>::ld(skip + p * k.skip_ldc) : v, y + p * k.y_ldc);
    }
  }
}

// One launch: a work-group keeps all of a group (at most 256 kHeld vectors, each inside the group) in registers between the statistics
// and the values, so x is read once.
constexpr int kHeld = 4;

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) groupnorm_held_kernel(const GroupNormK k) {
  __shared__ double sh[8];
  const int n = (int)blockIdx.x / k.G, g = (int)blockIdx.x - n * k.G;
  const int tid = (int)threadIdx.x, per = k.cpg / V, total = (int)k.HW * per;
  const int64_t px = (int64_t)n * k.HW, c0 = (int64_t)g * k.cpg;
  typename Vec<T, V>::Raw v[kHeld];
  int at[kHeld];
  double s = 0.0, q = 0.0;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    at[u] = tid + 256 * u;
    if (at[u] < total) v[u] = Vec<T, V>::ld((const T*)k.x + (px + at[u] / per) * k.x_ldc + c0 + at[u] % per * V);
  }
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (at[u] < total) {
      float f[V];
      Vec<T, V>::floats(v[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double d = (double)f[e];
        s += d;
        q = __builtin_fma(d, d, q);
      }
    }
  s = wave_sum(s);
  q = wave_sum(q);
  if ((tid & 63) == 0) {
    sh[tid >> 6] = s;
    sh[4 + (tid >> 6)] = q;
  }
  __syncthreads();
  const f4 st = finish_stats(sh[0] + sh[1] + sh[2] + sh[3], sh[4] + sh[5] + sh[6] + sh[7], (double)k.HW * k.cpg, k.eps);
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (at[u] < total) {
      const int64_t p = px + at[u] / per, c = c0 + at[u] % per * V;
      Affine<T, V> f;
#pragma unroll
      for (int e = 0; e < V; ++e) f.set(k, (int)c + e, e, st);
      f.template apply<ACT>(k, v[u], k.skip ? Vec<T, V>::ld((const T*)k.skip + p * k.skip_ldc + c) : v[u], (T*)k.y + p * k.y_ldc + c);
    }
}

}  // namespace pp

template <typename T, int V, int ACT>
static int launch_groupnorm_act(void* stream, pp::GroupNormK& k) {
  using namespace pp;
  // A group's rows are short pieces of the image's, one vector in the worst case: one launch pays while there are few of them in all.  Up to
  // 1024 vectors a group, in us, one launch against more: 32 groups of one vector a pixel, f16: 65536 vectors in all 6.6 / 13.6, 262144
  // 12.7 / 14.0, 524288 20.3 / 15.8; f32: 131072 9.0 / 11.1, 262144 12.0 / 11.1, 524288 19.0 / 12.1.  The limit is set by these.  Wider rows would bear
  // a higher one: 5 vectors a pixel, bf16: 262144 7.8 / 18.9, 524288 13.5 / 19.3, 1048576 24.1 / 27.3, 2097152 43.2 / 34.7; 8 vectors, f32: 524288 9.0 / 13.2.
  // Groups of whole rows (one group): 65536 12.4 / 32.7.
  const int64_t vectors = k.HW * (k.cpg / V);
  if (k.cpg % V == 0 && vectors <= 256 * kHeld && vectors * k.N * k.G <= 400000) {
    PP_LAUNCH((groupnorm_held_kernel<T, V, ACT>), dim3((unsigned)(k.N * k.G)), dim3(256), 0, stream, k);
    return pp_check_launch("pp_groupnorm(held)");
  }
  const int allcols = (k.C + V - 1) / V;
  k.cols = allcols < 256 ? allcols : 256;
  k.lanes = 256 / k.cols;
  k.join = k.G <= kOwnGroups && (int64_t)k.nchunks * k.G <= kOwnSums;
  const dim3 grid((unsigned)(k.N * k.nchunks));
  PP_LAUNCH((groupnorm_sums_kernel<T, V>), grid, dim3(256), 0, stream, k);
  int rc = pp_check_launch("pp_groupnorm(sums)");
  if (rc != PP_OK) return rc;
  if (!k.join) {
    const int64_t blocks = ((int64_t)k.N * k.G + 3) / 4;
    PP_LAUNCH(groupnorm_finish_kernel, dim3((unsigned)(blocks < kFinishBlocks ? blocks : kFinishBlocks)), dim3(256), 0, stream, k);
    rc = pp_check_launch("pp_groupnorm(finish)");
    if (rc != PP_OK) return rc;
  }
  PP_LAUNCH((groupnorm_apply_kernel<T, V, ACT>), grid, dim3(256), 0, stream, k);
  return pp_check_launch("pp_groupnorm(apply)");
}

template <typename T, int V>
static int launch_groupnorm(void* stream, pp::GroupNormK& k, int act) {
  switch (act) {
    case PP_ACT_RELU: return launch_groupnorm_act<T, V, PP_ACT_RELU>(stream, k);
    case PP_ACT_LEAKY: return launch_groupnorm_act<T, V, PP_ACT_LEAKY>(stream, k);
    case PP_ACT_SIGMOID: return launch_groupnorm_act<T, V, PP_ACT_SIGMOID>(stream, k);
    case PP_ACT_TANH: return launch_groupnorm_act<T, V, PP_ACT_TANH>(stream, k);
    case PP_ACT_GELU: return launch_groupnorm_act<T, V, PP_ACT_GELU>(stream, k);
    case PP_ACT_SILU: return launch_groupnorm_act<T, V, PP_ACT_SILU>(stream, k);
    default: return launch_groupnorm_act<T, V, PP_ACT_NONE>(stream, k);
  }
}

extern "C" int32_t pp_groupnorm(void* stream, const pp_groupnorm_params* p) {
  using namespace pp;
  if (!p || !p->x || !p->y || !p->partials) return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: null argument");
  if (p->dtype != PP_F32 && p->dtype != PP_F16 && p->dtype != PP_BF16) return pp_fail(PP_ERR_UNSUPPORTED, "pp_groupnorm: dtype");
  if (p->N < 0 || p->HW < 0 || p->HW > (int64_t)1 << 40 || p->C < 1 || p->C > 65536 || p->groups < 1 || p->C % p->groups)
    return pp_fail(PP_ERR_BAD_ARG, "pp_groupnorm: C must be in [1, 65536] and a multiple of groups, HW at most 2^40");
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
  k.relu_post = p->relu_post; k.eps = p->eps; k.act_param = p->act_param;
  // 16-byte accesses where every row of every tensor allows them, single elements otherwise
  const int V = p->dtype == PP_F32 ? 4 : 8;
  const bool wide = p->C % V == 0 && p->x_ldc % V == 0 && p->y_ldc % V == 0 && (!p->skip || p->skip_ldc % V == 0) &&
                    (((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->skip) % 16) == 0;
  if (p->dtype == PP_F32) return wide ? launch_groupnorm<float, 4>(stream, k, p->act) : launch_groupnorm<float, 1>(stream, k, p->act);
  if (p->dtype == PP_F16) return wide ? launch_groupnorm<half_t, 8>(stream, k, p->act) : launch_groupnorm<half_t, 1>(stream, k, p->act);
  return wide ? launch_groupnorm<bf16_t, 8>(stream, k, p->act) : launch_groupnorm<bf16_t, 1>(stream, k, p->act);
}

// The norm over all gradients of a network and the gradients scaled down to a largest norm.
//
//   total = scale * sqrt(sum over all tensors, all elements of g^2)   or   scale * max |g|
//   coef  = min(1, max_norm / (total + 1e-6)),   out = coef * g
//
// Kin of the multi-tensor optimizer steps (dfhip_fused.hip): the tensors' addresses travel in the kernel argument block, 64
// tensors a launch, so the launches can be captured.  TWO launches for up to 64 tensors: every workgroup of the first leaves
// one partial in double; every workgroup of the second adds ALL partials up by itself, in the same order (the same bits in
// every workgroup and every run; no atomics, no launch for a scalar), and scales its share.
//
// Both launches cut the tensors in the same way, a share of `chunk` elements a workgroup, chunk chosen so that there are
// about 2 048 workgroups: the partials every workgroup re-reads stay at 16 KB out of L2, and a workgroup's share is long
// enough to hide that.  A share that both launches read is found in the Infinity Cache by the second one as long as all
// gradients fit (256 MB).
//
// Bound: HBM, 12 bytes an element (read, read again, write): 403 M elements in 48 arrays 926 us = 5.2 TB/s (norm 311, scale 620; a
// large copy: 5.1).  What fits the Infinity Cache: 62 arrays of 11 MB 5.1 + 6.3 us, four arrays of 0.8 MB 3.4 + 3.8 us, most of it
// the launches.  Going through the shares backwards in the second launch, to meet what the first left in the cache: 924 us.
#include <math.h>

#include <algorithm>

#include "dfhip_internal.h"

using namespace dfhip;

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 64;              // 64 x 28 B of descriptors: inside the 4 KB kernel-argument block
constexpr int64_t kUnit = 4096;           // a share is a multiple of this many elements
constexpr int kShares = 2048;

struct ClipBatch {
  const float* g[kTensors];
  float* out[kTensors];
  int64_t size[kTensors];
  int first[kTensors + 1];                // the workgroup a tensor's shares begin with
  int n;
};

// the tensor a workgroup belongs to: the last t with first[t] <= blk
__device__ __forceinline__ int tensor_of(const ClipBatch& tb, int blk) {
  int lo = 0, hi = tb.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (blk >= tb.first[mid]) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// one element into the running value: squares in double (no square of a float overflows or vanishes there), the largest
// magnitude otherwise -- a NaN wins and stays
template <bool MAX>
__device__ __forceinline__ void take(double& acc, float v) {
  if (MAX) {
    const double a = fabs((double)v);
    acc = (a > acc || a != a) ? a : acc;
  } else {
    acc = fma((double)v, (double)v, acc);
  }
}
template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
  if (MAX) return (b > a || b != b) ? b : a;
  return a + b;
}

// all threads get the workgroup's value; the order of the additions is fixed
template <bool MAX>
__device__ __forceinline__ double block_join(double v, double* sh) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = join<MAX>(v, __shfl_xor(v, off));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; w++) v = join<MAX>(v, sh[w]);
  return v;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void k_clip_norm(ClipBatch tb, int64_t chunk, double* __restrict__ partial) {
  __shared__ double sh[kThreads / 64];
  const int t = tensor_of(tb, blockIdx.x);
  const int64_t lo = (int64_t)((int)blockIdx.x - tb.first[t]) * chunk;
  const int64_t n = min(tb.size[t] - lo, chunk);
  const float* g = tb.g[t] + lo;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t i = 0;
  if ((((uintptr_t)g) & 15) == 0) {
    const float4* g4 = reinterpret_cast<const float4*>(g);
    const int64_t n4 = n >> 2;
    int64_t j = threadIdx.x;
    for (; j + 3 * kThreads < n4; j += 4 * kThreads) {           // four 16-byte loads in flight
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; u++) v[u] = g4[j + u * kThreads];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        take<MAX>(acc[0], v[u].x); take<MAX>(acc[1], v[u].y); take<MAX>(acc[2], v[u].z); take<MAX>(acc[3], v[u].w);
      }
    }
    for (; j < n4; j += kThreads) {
      const float4 v = g4[j];
      take<MAX>(acc[0], v.x); take<MAX>(acc[1], v.y); take<MAX>(acc[2], v.z); take<MAX>(acc[3], v.w);
    }
    i = n4 << 2;
  }
  for (int64_t j = i + threadIdx.x; j < n; j += kThreads) take<MAX>(acc[0], g[j]);
  const double v = block_join<MAX>(join<MAX>(join<MAX>(acc[0], acc[1]), join<MAX>(acc[2], acc[3])), sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void k_clip_scale(ClipBatch tb, int64_t chunk, const double* __restrict__ partial,
                                                         int n_partial, double max_norm, double grad_scale,
                                                         float* __restrict__ norm_out) {
  __shared__ double sh[kThreads / 64];
  double acc = 0.0;
  for (int p = threadIdx.x; p < n_partial; p += kThreads) acc = join<MAX>(acc, partial[p]);
  acc = block_join<MAX>(acc, sh);
  const double total = (MAX ? acc : sqrt(acc)) * grad_scale;
  double c = max_norm / (total + 1e-6);
  c = c > 1.0 ? 1.0 : c;                                         // (a NaN stays one: the gradients say so too)
  const float coef = (float)c;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)total;
  const int t = tensor_of(tb, blockIdx.x);
  const int64_t lo = (int64_t)((int)blockIdx.x - tb.first[t]) * chunk;
  const int64_t n = min(tb.size[t] - lo, chunk);
  const float* g = tb.g[t] + lo;
  float* out = tb.out[t] + lo;
  int64_t i = 0;
  if (((((uintptr_t)g) | ((uintptr_t)out)) & 15) == 0) {
    const float4* g4 = reinterpret_cast<const float4*>(g);
    float4* o4 = reinterpret_cast<float4*>(out);
    const int64_t n4 = n >> 2;
    int64_t j = threadIdx.x;
    for (; j + 3 * kThreads < n4; j += 4 * kThreads) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; u++) v[u] = g4[j + u * kThreads];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        v[u].x *= coef; v[u].y *= coef; v[u].z *= coef; v[u].w *= coef;
        o4[j + u * kThreads] = v[u];
      }
    }
    for (; j < n4; j += kThreads) {
      float4 v = g4[j];
      v.x *= coef; v.y *= coef; v.z *= coef; v.w *= coef;
      o4[j] = v;
    }
    i = n4 << 2;
  }
  for (int64_t j = i + threadIdx.x; j < n; j += kThreads) out[j] = g[j] * coef;
}

}  // namespace

extern "C" {

int dfhip_clip_grad_norm(int n_tensors, const float* const* grads, float* const* outs, const int64_t* sizes, double max_norm,
                         int norm_type, double grad_scale, float* norm) {
  DF_INIT();
  DF_CHECK_ARG(n_tensors >= 0, "clip_grad_norm: negative number of tensors");
  DF_CHECK_ARG(norm_type == DFHIP_NORM_2 || norm_type == DFHIP_NORM_INF, "clip_grad_norm: norm_type is 2 or infinity");
  DF_CHECK_ARG(max_norm >= 0.0, "clip_grad_norm: max_norm must be >= 0");
  DF_CHECK_ARG(grad_scale >= 0.0 && grad_scale <= 3.4e38, "clip_grad_norm: grad_scale must be finite and >= 0");
  DF_CHECK_ARG(norm, "clip_grad_norm: null norm");
  DF_CHECK_ARG(n_tensors == 0 || (grads && outs && sizes), "clip_grad_norm: null table");
  int64_t total = 0;
  for (int i = 0; i < n_tensors; i++) {
    DF_CHECK_ARG(sizes[i] >= 0 && sizes[i] <= ((int64_t)1 << 40), "clip_grad_norm: bad size of tensor %d", i);
    DF_CHECK_ARG(sizes[i] == 0 || (grads[i] && outs[i]), "clip_grad_norm: null tensor %d", i);
    total += sizes[i];
  }
  const int64_t chunk = std::max<int64_t>(1, df_ceil_div(total, kShares * kUnit)) * kUnit;
  int64_t shares = 0;
  for (int i = 0; i < n_tensors; i++) shares += df_ceil_div(sizes[i], chunk);
  if (shares == 0) return dfhip_fill(norm, 1, 0.0f);
  DF_CHECK_ARG(shares <= (1 << 28), "clip_grad_norm: too many tensors");
  double* partial = (double*)workspace((size_t)shares * sizeof(double));
  if (!partial) return DFHIP_OUT_OF_MEMORY;
  ProfScope prof("clip_grad_norm", 3.0 * (double)total, 12.0 * (double)total);
  const bool mx = norm_type == DFHIP_NORM_INF;
  for (int pass = 0; pass < 2; pass++) {
    int64_t base = 0;
    int i = 0;
    bool first_batch = true;
    while (i < n_tensors) {
      ClipBatch tb;
      tb.n = 0;
      int blk = 0;
      for (; i < n_tensors && tb.n < kTensors; i++) {
        if (sizes[i] == 0) continue;
        tb.g[tb.n] = grads[i];
        tb.out[tb.n] = outs[i];
        tb.size[tb.n] = sizes[i];
        tb.first[tb.n] = blk;
        blk += (int)df_ceil_div(sizes[i], chunk);
        tb.n++;
      }
      if (tb.n == 0) break;
      tb.first[tb.n] = blk;
      if (pass == 0) {
        if (mx) DF_LAUNCH(k_clip_norm<true>, dim3(blk), dim3(kThreads), 0, stream(), tb, chunk, partial + base);
        else DF_LAUNCH(k_clip_norm<false>, dim3(blk), dim3(kThreads), 0, stream(), tb, chunk, partial + base);
      } else {
        float* no = first_batch ? norm : nullptr;
        if (mx)
          DF_LAUNCH(k_clip_scale<true>, dim3(blk), dim3(kThreads), 0, stream(), tb, chunk, partial, (int)shares, max_norm,
                    grad_scale, no);
        else
          DF_LAUNCH(k_clip_scale<false>, dim3(blk), dim3(kThreads), 0, stream(), tb, chunk, partial, (int)shares, max_norm,
                    grad_scale, no);
      }
      DF_LAUNCH_CHECK();
      base += blk;
      first_batch = false;
    }
  }
  return DFHIP_OK;
}

}  // extern "C"

// Softmax cross entropy of a linear layer over many classes, without keeping its logits, with its gradient.
//
//   l = x W + b,  row loss = lse(l) - (1 - e) l_t - (e / V) sum_j l_j  for the rows whose target t is not `ignore_index`,
//   loss = sum over those rows (/ their number),  dl = (softmax(l) - (1 - e) onehot(t) - e / V) (/ their number),
//   dx = dl W^T,  dW = x^T dl,  db = column sums of dl.
//
// The rows go through in pieces: the logits of one piece exist at a time, become dl in place and are consumed by the two
// products, so memory does not grow with rows x classes.  The gradients are formed in the forward pass, for an upstream
// gradient of 1: nothing is computed twice (recomputing the logits in a backward pass would be a third more products).
#include <math.h>

#include <algorithm>

#include "dfhip_internal.h"

using namespace dfhip;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kPieceBytes = (int64_t)512 << 20;        // the logits of one piece of the rows

// per call: 0 number of counted rows
__global__ __launch_bounds__(kThreads) void k_lce_count(const float* __restrict__ target, int64_t rows, float ignore,
                                                        float* __restrict__ ctl) {
  __shared__ int sh[kThreads / 64];
  int n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += kThreads) n += target[i] != ignore ? 1 : 0;
#pragma unroll
  for (int off = 32; off; off >>= 1) n += __shfl_xor(n, off);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) ctl[0] = (float)(sh[0] + sh[1] + sh[2] + sh[3]);
}

template <class F>
__device__ __forceinline__ float block_reduce(float v, float* sh, F f) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = f(v, __shfl_xor(v, off));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < kThreads / 64; w++) v = f(v, sh[w]);
  return v;
}

// a workgroup a row: the row's loss, and dl over its logits
__global__ __launch_bounds__(kThreads) void k_lce_rows(float* __restrict__ logits, const float* __restrict__ target,
                                                       const float* __restrict__ ctl, float* __restrict__ rowloss, int64_t V,
                                                       float ignore, float smooth, int mean, int grads) {
  __shared__ float sh[kThreads / 64];
  float* l = logits + (int64_t)blockIdx.x * V;
  const float t = target[blockIdx.x];
  if (t == ignore) {
    if (threadIdx.x == 0) rowloss[blockIdx.x] = 0.0f;
    if (grads)
      for (int64_t v = threadIdx.x; v < V; v += kThreads) l[v] = 0.0f;
    return;
  }
  const bool ok = t >= 0.0f && t < (float)V && t == floorf(t);
  const int64_t ti = ok ? (int64_t)t : 0;
  float m = -INFINITY;
  for (int64_t v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, l[v]);
  m = block_reduce(m, sh, [](float a, float b) { return fmaxf(a, b); });
  float z = 0.0f, s = 0.0f;
  for (int64_t v = threadIdx.x; v < V; v += kThreads) {
    z += expf(l[v] - m);
    s += l[v] - m;
  }
  z = block_reduce(z, sh, [](float a, float b) { return a + b; });
  s = block_reduce(s, sh, [](float a, float b) { return a + b; });
  const float lt = l[ti] - m;
  __syncthreads();                                 // (every thread has read the target's logit before it is overwritten)
  if (threadIdx.x == 0) {
    float r = logf(z) - (1.0f - smooth) * lt;
    if (smooth > 0.0f) r -= smooth * (s / (float)V);
    rowloss[blockIdx.x] = ok ? r : NAN;
  }
  if (!grads) return;
  const float scale = mean ? 1.0f / fmaxf(ctl[0], 1.0f) : 1.0f;
  const float iz = 1.0f / z, q = smooth / (float)V;
  for (int64_t v = threadIdx.x; v < V; v += kThreads) {
    float d = expf(l[v] - m) * iz - q;
    if (v == ti) d -= 1.0f - smooth;
    l[v] = ok ? d * scale : NAN;
  }
}

// loss = sum of the row losses (/ the number of counted rows), in a fixed order
__global__ __launch_bounds__(kThreads) void k_lce_loss(const float* __restrict__ rowloss, const float* __restrict__ ctl,
                                                       float* __restrict__ loss, int64_t rows, int mean) {
  __shared__ float sh[kThreads / 64];
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < rows; i += kThreads) s += rowloss[i];
  s = block_reduce(s, sh, [](float a, float b) { return a + b; });
  if (threadIdx.x == 0) loss[0] = mean ? s / fmaxf(ctl[0], 1.0f) : s;
}

__global__ __launch_bounds__(kThreads) void k_lce_scale(const float* __restrict__ src, const float* __restrict__ scalar,
                                                        float* __restrict__ dst, int64_t n) {
  const float s = scalar[0];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) dst[i] = src[i] * s;
}

struct Held {                                      // a pool block for the duration of a call (its reuse is stream-ordered)
  float* p = nullptr;
  ~Held() { if (p) (void)dfhip_free(p); }
};

}  // namespace

extern "C" {

int dfhip_linear_ce_forward(const float* x, const float* w, const float* bias, const float* target, float* loss, float* dx,
                            float* dw, float* db, int64_t rows, int64_t width, int64_t classes, int64_t ignore_index,
                            double label_smoothing, int mean) {
  DF_INIT();
  DF_CHECK_ARG(rows >= 0 && width >= 1 && classes >= 1, "linear_ce_forward: bad extents (%lld, %lld, %lld)", (long long)rows,
               (long long)width, (long long)classes);
  DF_CHECK_ARG(rows <= 0x7fffffff && width <= 0x7fffffff, "linear_ce_forward: rows and width must be below 2^31");
  DF_CHECK_ARG(classes <= (1 << 24), "linear_ce_forward: at most 2^24 classes (their indices are whole numbers held in fp32)");
  DF_CHECK_ARG(ignore_index >= -(1 << 24) && ignore_index <= (1 << 24), "linear_ce_forward: ignore_index must be within 2^24");
  DF_CHECK_ARG(label_smoothing >= 0.0 && label_smoothing <= 1.0, "linear_ce_forward: label_smoothing must be in [0, 1]");
  DF_CHECK_ARG(loss && w, "linear_ce_forward: null array");
  DF_CHECK_ARG(rows == 0 || (x && target), "linear_ce_forward: null array");
  DF_CHECK_ARG(!db || bias, "linear_ce_forward: a bias gradient without a bias");
  if (rows == 0) {
    int st = dfhip_fill(loss, 1, 0.0f);
    if (st == DFHIP_OK && dw) st = dfhip_fill(dw, width * classes, 0.0f);
    if (st == DFHIP_OK && db) st = dfhip_fill(db, classes, 0.0f);
    return st;
  }
  const bool grads = dx || dw || db;
  const int64_t piece = std::min(rows, std::max<int64_t>(1, kPieceBytes / (4 * classes)));
  Held logits, stats, more;
  int st = dfhip_malloc(piece * classes, &logits.p);
  if (st == DFHIP_OK) st = dfhip_malloc(rows + 1, &stats.p);
  if (st == DFHIP_OK && piece < rows && (dw || db)) st = dfhip_malloc(std::max(dw ? width * classes : 0, classes), &more.p);
  if (st != DFHIP_OK) return st;
  float *ctl = stats.p, *rowloss = stats.p + 1;
  const float ignore = (float)ignore_index;
  DF_LAUNCH(k_lce_count, dim3(1), dim3(kThreads), 0, stream(), target, rows, ignore, ctl);
  DF_LAUNCH_CHECK();
  for (int64_t r0 = 0; r0 < rows; r0 += piece) {
    const int64_t n = std::min(piece, rows - r0);
    st = dfhip_gemm(x + r0 * width, w, bias, logits.p, n, width, classes, 0, 0);
    if (st != DFHIP_OK) return st;
    DF_LAUNCH(k_lce_rows, dim3((unsigned)n), dim3(kThreads), 0, stream(), logits.p, target + r0, ctl, rowloss + r0, classes,
              ignore, (float)label_smoothing, mean, grads ? 1 : 0);
    DF_LAUNCH_CHECK();
    if (dx) st = dfhip_gemm(logits.p, w, nullptr, dx + r0 * width, n, classes, width, 0, 1);
    if (st == DFHIP_OK && dw) {
      st = dfhip_gemm(x + r0 * width, logits.p, nullptr, r0 ? more.p : dw, width, n, classes, 1, 0);
      if (st == DFHIP_OK && r0) st = dfhip_axpy(dw, more.p, 1.0f, width * classes);
    }
    if (st == DFHIP_OK && db) {
      st = dfhip_reduce_axis(logits.p, r0 ? more.p : db, 1, n, classes, 0, 1.0f);
      if (st == DFHIP_OK && r0) st = dfhip_axpy(db, more.p, 1.0f, classes);
    }
    if (st != DFHIP_OK) return st;
  }
  DF_LAUNCH(k_lce_loss, dim3(1), dim3(kThreads), 0, stream(), rowloss, ctl, loss, rows, mean);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

int dfhip_scale_by(const float* src, const float* scalar, float* dst, int64_t n) {
  DF_INIT();
  DF_CHECK_ARG(n >= 0, "scale_by: negative size");
  if (n == 0) return DFHIP_OK;
  DF_CHECK_ARG(src && scalar && dst, "scale_by: null array");
  ProfScope prof("scale_by", 0.0, 8.0 * (double)n);
  DF_LAUNCH(k_lce_scale, dim3((unsigned)std::min<int64_t>(df_ceil_div(n, 4 * kThreads), 4096)), dim3(kThreads), 0, stream(), src,
            scalar, dst, n);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

}  // extern "C"

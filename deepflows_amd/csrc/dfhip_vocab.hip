// Softmax cross entropy of a linear layer over many classes, without keeping its logits, with its gradient.
//
//   l = x W + b,  row loss = lse(l) - (1 - e) l_t - (e / V) sum_j l_j  for the rows whose target t is not `ignore_index`,
//   loss = sum over those rows (/ their number),  dl = (softmax(l) - (1 - e) onehot(t) - e / V) (/ their number),
//   dx = dl W^T,  dW = x^T dl,  db = column sums of dl.
//
// The rows go through in pieces: the logits of one piece exist at a time, become dl in place and are consumed by the two
// products, so memory does not grow with rows x classes.  The gradients are formed in the forward pass, for an upstream
// gradient of 1: nothing is computed twice (recomputing the logits in a backward pass would be a third more products).
//
// The three products run on the fp16 matrix cores with fp32 accuracy (dfhip_splitgemm.h: 23 bits of every element down to 2^-28 of its
// array's largest, of dl down to 2^-29): x and W are converted once a call, dl where it is formed; for few rows, where W's bytes are
// what counts, they run on the fp32 matrix cores (dfhip_fewrows.h, and further
// down).  The launches of a call:
//   k_lce_scan     the largest magnitudes of x (counted rows) and W, finite elements only
//   k_lce_split    x, W -> split arrays; the number of counted rows (a large W may need it twice)
//   per piece:     logits product (+ bias) -> k_lce_rows (losses; dl over the logits, as a split array) -> k_lce_pair: the dx
//                  product and the dW product (db on the side: the column sums of its second operand); with the last piece, the loss
//   without gradients: the product's epilogue leaves what the softmax needs of every 64 logits and the targets' (none is stored),
//                  k_few_rows joins them, k_lce_loss
//
// Measured.  8192 x 1024 x 50001 with gradients, 7.1 ms: logits 2.19 ms and the pair 4.31 ms, 1.15 and 1.17 PFLOP/s of fp16 (the
// library's 8192^3 fp16 product: 1.18; at that rate the three products alone are 6.42 ms, in fp32 16.4), rows 0.68 ms (3.3 GB, 4.8
// TB/s), conversion 0.10.  2048 x 768 x 32000: 0.95 ms; 509 x 512 x 10007: 89 us; 1500 x 1024 x 30011, the loss alone: 0.32 ms.
// Largest error of any result against 64 bits, relative to the result's largest value: 2.1e-6 at 8192 x 1024 x 50001, where the
// fp32 composition (library products) has 5.4e-6; 9e-7 and 4.3e-6 at 2048 x 768 x 32000.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "dfhip_fewrows.h"
#include "dfhip_splitgemm.h"

using namespace dfhip;
using namespace dfhip_split;

namespace {

constexpr int kThreads = 256;
constexpr int kTopDl = 15;                                 // |dl| <= 1: at most 2^15 as a split array
constexpr int kScan = 512;                                 // workgroups (= partial maxima) a tensor
// From this many elements of W on its scale comes from a sample: at 1024 x 16384 the full scan is 11.6 us, the sample 4.6 and the
// launch that looks whether it was enough 4.8; at 1024 x 50001 41 and 5.4 + 4.9.
constexpr int64_t kSampled = (int64_t)16 << 20;
constexpr int64_t kPieceBytes = (int64_t)2 << 30;          // the logits (or the softmax's parts) of one piece of the rows
constexpr int64_t kPieceRows = 1 << 22;                    // a workgroup a row: 2^32 threads a launch are too many

// what the launches of one call hand to each other
struct Ctl {
  float scale;                                             // 1 / number of counted rows, or 1
  int ex, ew;                                              // x = 2^ex * split array, W likewise
  unsigned found;                                          // 0, or W's largest finite magnitude where a sample's scale does not hold it
  float max_x[kScan], max_w[kScan];
};

template <int T, class X, class F>
__device__ __forceinline__ X block_reduce(X v, X* sh, F f) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = f(v, __shfl_xor(v, off));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < T / 64; w++) v = f(v, sh[w]);
  return v;
}
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
  __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
  __device__ __forceinline__ int operator()(int a, int b) const { return a + b; }
};

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028235e38f ? a : 0.0f;                    // (inf and NaN: 0)
}

__device__ __forceinline__ float finite_abs(const float4& v) {
  return fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
}

// workgroups 0 .. kScan-1: x, kScan .. 2 kScan - 1: W.  The rows of x that are not counted are passed over: padding may hold
// anything, and a large value in it would cost the counted rows their low bits.  `sample`: of W every sixteenth piece of 64 elements
// is read; the conversion finds out whether that was enough.
__global__ __launch_bounds__(kThreads) void k_lce_scan(const float* __restrict__ x, int64_t rows, int64_t width,
                                                       const float* __restrict__ target, float ignore,
                                                       const float* __restrict__ w, int64_t nw, int sample, Ctl* __restrict__ ctl) {
  __shared__ float sh[kThreads / 64];
  const bool second = blockIdx.x >= kScan;
  if (blockIdx.x == 0 && threadIdx.x == 0) ctl->found = 0;
  const int blk = (int)blockIdx.x & (kScan - 1);
  float m = 0.0f;
  if (!second) {                                           // a wave takes up to 1 024 elements of one row at a time
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t segs = (width + 1023) >> 10;
    const bool vec = (width & 3) == 0 && (((uintptr_t)x) & 15) == 0;
    for (int64_t it = (int64_t)blk * (kThreads / 64) + wave; it < rows * segs; it += kScan * (kThreads / 64)) {
      const int64_t r = segs == 1 ? it : it / segs;
      const int c0 = (int)(it - r * segs) << 10, n = (int)min(width - c0, (int64_t)1024);
      const float* p = x + r * width + c0;
      const float t = target[r];
      float s = 0.0f;
      if (vec) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int c = u * 256 + lane * 4;
          v[u] = c < n ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < 4; u++) s = fmaxf(s, finite_abs(v[u]));
      } else {
#pragma unroll 4
        for (int c = lane; c < n; c += 64) s = fmaxf(s, finite_abs(p[c]));
      }
      m = t == ignore ? m : fmaxf(m, s);
    }
  } else if (sample) {
    // (64 elements of 1 024, their place among them by a multiplicative hash of the run's number: at one place all would lie on the
    // same few memory channels, and a place that follows the number's last bits repeats from row to row of W where the number of
    // classes is a multiple of 16 384)
    const int64_t runs = nw >> 10, step = kScan * (kThreads / 16);
    const int lane = threadIdx.x & 15;
    int64_t i = (int64_t)blk * (kThreads / 16) + (threadIdx.x >> 4);
    for (; i < runs; i += 4 * step) {
      dfhip_few::f32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int64_t r = min(i + u * step, runs - 1);
        v[u] = *reinterpret_cast<const dfhip_few::f32x4u*>(w + (r << 10) + (((unsigned)r * 2654435769u) >> 28) * 64 + lane * 4);
      }
#pragma unroll
      for (int u = 0; u < 4; u++) m = fmaxf(m, fmaxf(fmaxf(finite_abs(v[u][0]), finite_abs(v[u][1])), fmaxf(finite_abs(v[u][2]), finite_abs(v[u][3]))));
    }
  } else {
    int64_t lo = 0;
    if ((((uintptr_t)w) & 15) == 0) {
      const float4* p4 = reinterpret_cast<const float4*>(w);
      const int64_t n4 = nw >> 2, step = (int64_t)kScan * kThreads;
      int64_t i = (int64_t)blk * kThreads + threadIdx.x;
      for (; i + 3 * step < n4; i += 4 * step) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = p4[i + u * step];
#pragma unroll
        for (int u = 0; u < 4; u++) m = fmaxf(m, finite_abs(v[u]));
      }
      for (; i < n4; i += step) m = fmaxf(m, finite_abs(p4[i]));
      lo = n4 << 2;
    }
    for (int64_t i = lo + (int64_t)blk * kThreads + threadIdx.x; i < nw; i += (int64_t)kScan * kThreads)
      m = fmaxf(m, finite_abs(w[i]));
  }
  m = block_reduce<kThreads>(m, sh, Max());
  if (threadIdx.x == 0) (second ? ctl->max_w : ctl->max_x)[blk] = m;
}

// workgroups [0, bx): x (zeros for the rows that are not counted), [bx, bx + bw): W, the last one: the number of counted rows.  A
// wave takes 512 consecutive cells of the padded array at a time, eight a lane; where rows do not begin on 16 bytes it reads them
// lane by lane and turns them in LDS.
//
// `sample`: W's scale came from a sixteenth of it.  It leaves the largest element seen a factor of four below the largest fp16
// number; larger ones are found on the way, and so is any element that is not zero where the sample held none to take a scale from.
// Should there be any (AGAIN: this kernel's second launch, for W alone, which otherwise ends at once), W is converted once more with
// the scale that it asks for.
constexpr float kHalfMax = 65504.0f;
template <bool AGAIN>
__global__ __launch_bounds__(kThreads) void k_lce_split(const float* __restrict__ x, int64_t rows, int64_t width,
                                                        const float* __restrict__ w, int64_t classes, char* __restrict__ xs,
                                                        char* __restrict__ ws, const float* __restrict__ target, float ignore,
                                                        int mean, int64_t bx, int64_t bw, int sample, Ctl* __restrict__ ctl) {
  __shared__ float sh[kThreads / 64];
  __shared__ int shi[kThreads / 64];
  __shared__ __attribute__((aligned(16))) float turn[kThreads / 64][512];
  if (AGAIN && ctl->found == 0) return;
  if (!AGAIN && blockIdx.x == bx + bw) {
    int n = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < rows; i += kThreads) n += target[i] != ignore ? 1 : 0;
    n = block_reduce<kThreads>(n, shi, Add());
    if (threadIdx.x == 0) ctl->scale = mean ? 1.0f / (float)max(n, 1) : 1.0f;
    return;
  }
  const bool second = blockIdx.x >= bx;
  const float* part = second ? ctl->max_w : ctl->max_x;
  float m = 0.0f;
  if (AGAIN) {
    m = __uint_as_float(ctl->found);
  } else {
#pragma unroll
    for (int u = 0; u < kScan / kThreads; u++) m = fmaxf(m, part[threadIdx.x + u * kThreads]);
    m = block_reduce<kThreads>(m, sh, Max());
  }
  const int e = m > 0.0f ? ilogbf(m) - kTop : 0;
  if (threadIdx.x == 0 && blockIdx.x == (second ? bx : 0)) (second ? ctl->ew : ctl->ex) = e;
  float largest = 0.0f;
  const float* src = second ? w : x;
  char* dst = second ? ws : xs;
  const int64_t nr = second ? width : rows, nc = second ? classes : width;
  const int64_t pr = padded(nr), pc = padded(nc), units = pr * pc / 512;      // (a multiple of 4: the workgroup stays together)
  const int64_t nblk = second ? bw : bx;
  const bool vec = (nc & 3) == 0 && (((uintptr_t)src) & 15) == 0;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int64_t u0 = ((int64_t)blockIdx.x - (second ? bx : 0)) * 4; u0 < units; u0 += nblk * 4) {
    const int64_t first = (u0 + wave) * 512, r0 = first / pc, c0 = first - r0 * pc;
    int64_t r = r0, c = c0 + lane * 8;
    while (c >= pc) { c -= pc; r++; }
    float v[8];
    if (vec) {
      if (r < nr && c + 8 <= nc) {
        const float4 a = *reinterpret_cast<const float4*>(src + r * nc + c), b = *reinterpret_cast<const float4*>(src + r * nc + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (r < nr && c + k < nc) ? src[r * nc + c + k] : 0.0f;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        int64_t rk = r0, ck = c0 + k * 64 + lane;
        while (ck >= pc) { ck -= pc; rk++; }
        v[k] = (rk < nr && ck < nc) ? src[rk * nc + ck] : 0.0f;
      }
      __syncthreads();                             // (the last trip's values have been read)
#pragma unroll
      for (int k = 0; k < 8; k++) turn[wave][k * 64 + lane] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = turn[wave][lane * 8 + k];
    }
    const bool out = !second && r < nr && target[r] == ignore;
    if (!AGAIN && sample && second)
#pragma unroll
      for (int k = 0; k < 8; k++) largest = fmaxf(largest, finite_abs(v[k]));
    half8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      _Float16 h, l;
      split(out ? 0.0f : ldexpf(v[k], -e), h, l);
      hi[k] = h; lo[k] = l;
    }
    char* d = dst + r * pc * 4 + (c >> 5) * 128 + (c & 31) * 2;
    *reinterpret_cast<half8*>(d) = hi;
    *reinterpret_cast<half8*>(d + 64) = lo;
  }
  if (!AGAIN && sample && second) {
    largest = block_reduce<kThreads>(largest, sh, Max());
    // (a largest value: the order does not matter.  Only those that count: 4 096 of these are 33 us)
    const float most = m > 0.0f ? kHalfMax : 0.0f;
    if (threadIdx.x == 0 && ldexpf(largest, -e) > most) atomicMax(&ctl->found, __float_as_uint(largest));
  }
}

// 2^-k, 2^k >= classes: what the terms of a mean over the classes are scaled by, so that no sum of finite ones passes the largest float
__device__ __forceinline__ float mean_scale(int classes) { return ldexpf(1.0f, -(32 - __clz(classes - 1))); }

// A workgroup a row: the row's loss, and dl (times 2^kTopDl) over its logits as a split array.  `cells` is the padded row, a
// multiple of 256; a row that is not counted, or lies behind the last one (blockIdx.x >= rows), becomes zeros.
// U > 0: U groups of eight logits a thread hold the row in registers (T * 8 * U >= cells), one pass over memory each way;
// U = 0: any length, the row read three times.
template <int T, int U>
__global__ __launch_bounds__(T) void k_lce_rows(float* __restrict__ logits, const float* __restrict__ target, int rows,
                                                float* __restrict__ rowloss, int classes, int cells, float ignore, float smooth) {
  __shared__ float sh[T / 64];
  float* l = logits + (int64_t)blockIdx.x * cells;
  const bool exists = (int)blockIdx.x < rows;
  const float t = exists ? target[blockIdx.x] : ignore;
  auto store = [&](int c, const float* v) {                // eight cells from column c (a multiple of 8)
    half8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      _Float16 h, q;
      split(v[k], h, q);
      hi[k] = h; lo[k] = q;
    }
    char* d = reinterpret_cast<char*>(l) + (c >> 5) * 128 + (c & 31) * 2;
    *reinterpret_cast<half8*>(d) = hi;
    *reinterpret_cast<half8*>(d + 64) = lo;
  };
  if (t == ignore) {
    if (threadIdx.x == 0 && exists) rowloss[blockIdx.x] = 0.0f;
    for (int c = threadIdx.x * 4; c < cells; c += T * 4) *reinterpret_cast<float4*>(l + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  const bool ok = t >= 0.0f && t < (float)classes && t == floorf(t);
  const int ti = ok ? (int)t : 0;
  const float lt = l[ti];
  constexpr int UU = U > 0 ? U : 1;
  const int trips = U > 0 ? 1 : (cells + T * 8 - 1) / (T * 8);
  float v[UU][8];
  // (the column is made new for every pass: the compiler otherwise keeps each pass's comparisons of it for the next ones, two
  // masks a group, and spills)
  auto first = [&]() {
    int c0 = (int)threadIdx.x * 8;
    asm volatile("" : "+v"(c0));
    return c0;
  };
  auto load = [&](int trip) {                              // -inf behind the last class
    const int c0 = first();
#pragma unroll
    for (int u = 0; u < UU; u++) {
      const int c = (trip * UU + u) * T * 8 + c0;
      if (c < cells) {
        const float4 a = *reinterpret_cast<const float4*>(l + c), b = *reinterpret_cast<const float4*>(l + c + 4);
        v[u][0] = a.x; v[u][1] = a.y; v[u][2] = a.z; v[u][3] = a.w; v[u][4] = b.x; v[u][5] = b.y; v[u][6] = b.z; v[u][7] = b.w;
      }
      if (c + 8 > classes)                                 // (a branch that few waves take: a mask a value would cost registers)
#pragma unroll
        for (int k = 0; k < 8; k++) v[u][k] = c + k < classes ? v[u][k] : -INFINITY;
    }
  };
  float m = -INFINITY;
  for (int i = 0; i < trips; i++) {
    load(i);
#pragma unroll
    for (int u = 0; u < UU; u++)
#pragma unroll
      for (int k = 0; k < 8; k++) m = fmaxf(m, v[u][k]);   // (passes a NaN over; its exponential makes z one)
  }
  m = block_reduce<T>(m, sh, Max());
  float z = 0.0f, s = 0.0f;
  const float down = mean_scale(classes);
  for (int i = 0; i < trips; i++) {
    if (U == 0) load(i);
    const int c0 = first();
#pragma unroll
    for (int u = 0; u < UU; u++) {
      const int c = (i * UU + u) * T * 8 + c0;
      if (smooth > 0.0f) {
        if (c + 8 <= classes) {
#pragma unroll
          for (int k = 0; k < 8; k++) s = fmaf(v[u][k] - m, down, s);
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++) s = fmaf(c + k < classes ? v[u][k] - m : 0.0f, down, s);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        v[u][k] = exp_of(v[u][k] - m);
        z += v[u][k];
      }
    }
  }
  z = block_reduce<T>(z, sh, Add());
  if (smooth > 0.0f) s = block_reduce<T>(s, sh, Add());
  if (threadIdx.x == 0) {
    float r = logf(z) - (1.0f - smooth) * (lt - m);
    if (smooth > 0.0f) r -= smooth * (s / ((float)classes * down));
    rowloss[blockIdx.x] = ok ? r : NAN;
  }
  const float top = (float)(1 << kTopDl), iz = ok ? top / z : NAN, q = top * (smooth / (float)classes), p1 = top * (1.0f - smooth);
  for (int i = 0; i < trips; i++) {
    if (U == 0) {
      load(i);
#pragma unroll
      for (int u = 0; u < UU; u++)
#pragma unroll
        for (int k = 0; k < 8; k++) v[u][k] = exp_of(v[u][k] - m);
    }
    const int c0 = first();
#pragma unroll
    for (int u = 0; u < UU; u++) {
      const int c = (i * UU + u) * T * 8 + c0;
      if (c < cells) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[u][k] = fmaf(v[u][k], iz, -q);
        if ((unsigned)(ti - c) < 8u)
#pragma unroll
          for (int k = 0; k < 8; k++) v[u][k] -= c + k == ti ? p1 : 0.0f;
        if (c + 8 > classes)
#pragma unroll
          for (int k = 0; k < 8; k++) v[u][k] = c + k < classes ? v[u][k] : 0.0f;
        store(c, v[u]);
      }
    }
  }
}

// loss = sum of the row losses times the scale, in a fixed order; one workgroup of T threads.  In double: a thread adds rows / T values of
// one sign, and in fp32 2 M rows drift by up to 5e-4.
template <int T>
__device__ __forceinline__ void loss_body(const float* __restrict__ rowloss, const Ctl* __restrict__ ctl, float* __restrict__ loss,
                                          int64_t rows, double* sh) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += T) s += (double)rowloss[i];
  s = block_reduce<T>(s, sh, Add());
  if (threadIdx.x == 0) loss[0] = (float)(s * (double)ctl->scale);
}
__global__ __launch_bounds__(1024) void k_lce_loss(const float* __restrict__ rowloss, const Ctl* __restrict__ ctl,
                                                   float* __restrict__ loss, int64_t rows) {
  __shared__ double sh[1024 / 64];
  loss_body<1024>(rowloss, ctl, loss, rows, sh);
}

// The two gradient products of a piece as one launch (they read the same dl; together they leave fewer idle CUs at the end, and a
// small call is one launch shorter): workgroups [0, na): dx, [na, na + nb): dW, and one more for the loss behind the last piece.
struct Pair {
  Gemm a, b;
  int na, nb;
  const float* rowloss;
  const Ctl* ctl;
  float* loss;
  int64_t rows;
};
template <int T, int EPI>
__global__ __launch_bounds__(threads<T>(), waves<T>()) void k_lce_pair(Pair p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int block = (int)blockIdx.x;
  if (block < p.na) gemm_body<T, false, false, EPI_STORE>(p.a, block, lds);
  else if (block < p.na + p.nb) gemm_body<T, true, true, EPI>(p.b, block - p.na, lds);
  else loss_body<threads<T>()>(p.rowloss, p.ctl, p.loss, p.rows, reinterpret_cast<double*>(lds));
}
template <int T, int EPI>
__global__ __launch_bounds__(256) void k_lce_pair_rest(Pair p) {
  constexpr int SLICES = slices<T>();
  const int block = (int)blockIdx.x;
  if (block < p.a.rest * SLICES) rest_body<T, EPI_STORE>(p.a, block);
  else rest_body<T, EPI>(p.b, block - p.a.rest * SLICES);
}

// ---- few rows: W is read as it is (dfhip_fewrows.h) ----------------------------------------------------------------------------
//   k_few_logits   logits (rows, ld), and of every column tile the rows' largest logit, sum of exponentials and sum (row_part)
//   k_few_rows     those joined: row losses; dl (times the mean's factor) over the logits
//   k_few_pair     the dx product, cut along the classes, and the dW product (db on the side); the loss
//   k_few_rest     the parts of dx added up
struct Few {
  dfhip_few::Product logits, dx;
  const float* bias;
  float* l;                                // logits, then dl
  int64_t ld;                              // a multiple of 128
  float* stat;                             // three arrays of (rows, tiles): largest, sum of exponentials, kDown * sum of l - largest
  int tiles, cols;                         // their number and width
  const float* lt;                         // the targets' logits, or NULL: they are in l
  const float* target;
  float ignore, smooth;
  float *dw, *db, *parts, *loss;
  const float* rowloss;
  const Ctl* ctl;
  int width, cuts, cut, n_dx;              // dx: `cuts` ranges of `cut` classes, n_dx workgroups
  int strips, dw_cuts, dw_cut, n_dw;       // dW: strips of few_strip() columns, dw_cuts ranges of dw_cut rows of it
};

template <int RB, int CF, int NW>
__global__ __launch_bounds__(NW * 64) void k_few_logits(Few g) {
  __shared__ dfhip_few::f32x4 lds[dfhip_few::lds_pieces<CF, NW>()];
  // (64 rows a workgroup; a tile's workgroups eight numbers apart, on the same XCD, where W comes out of the L2 for the second)
  const int sets = (g.logits.rows + 63) >> 6, block = (int)blockIdx.x;
  const int tile = (block >> 3) / sets * 8 + (block & 7), row0 = (block >> 3) % sets * 64, n0 = tile * 32 * CF, i = threadIdx.x & 31;
  if (tile >= g.tiles) return;
  dfhip_few::Product p = g.logits;
  p.a += (int64_t)row0 * p.lda;
  p.rows = min(p.rows - row0, 64);
  const int c = n0 + CF * i, over = c - min(c, p.n - CF);  // columns by which this lane's loads were moved back
  float bias[CF];
#pragma unroll
  for (int f = 0; f < CF; f++) bias[f] = g.bias && c + f < p.n ? g.bias[c + f] : 0.0f;
  dfhip_few::across<RB, CF, NW>(p, n0, lds, [&](int row, const float* v) {
    if (row >= p.rows) return;                             // (uniform in the half wave)
    row += row0;
    float w[CF];                                           // -inf behind the last class
#pragma unroll
    for (int f = 0; f < CF; f++) {
      w[f] = -INFINITY;
#pragma unroll
      for (int e = 0; e < CF; e++) w[f] = f + over == e ? v[e] + bias[f] : w[f];
    }
    typedef float vec __attribute__((ext_vector_type(CF)));
    *reinterpret_cast<vec*>(g.l + (int64_t)row * g.ld + c) = *reinterpret_cast<const vec*>(w);
    bool in[CF];
#pragma unroll
    for (int f = 0; f < CF; f++) in[f] = c + f < p.n;
    const RowPart part = row_part<CF, 32>(w, in, g.smooth > 0.0f);
    if (i == 0) store_part(g.stat + (int64_t)row * g.tiles + tile, (int64_t)g.logits.rows * g.tiles, part);
  });
}

// `chunks` workgroups a row, each of which joins the row's tiles for itself; the one that holds the target's column also makes the
// row's loss (nobody else touches that column)
template <bool GRADS, bool COUNT>
__global__ __launch_bounds__(kThreads) void k_few_rows(Few g, int rows, int classes, int mean, int chunk, int chunks,
                                                       float* __restrict__ rowloss, Ctl* __restrict__ ctl) {
  __shared__ float sh[kThreads / 64];
  __shared__ int shi[kThreads / 64];
  const int row = (int)blockIdx.x / chunks, ch = (int)blockIdx.x % chunks;
  const float t = g.target[row];
  float* l = g.l + (int64_t)row * g.ld;
  const int lo = ch * chunk, hi = min(lo + chunk, (int)g.ld);
  float scale = 1.0f;
  if (COUNT) {
    int n = 0;
    for (int k = threadIdx.x; k < rows; k += kThreads) n += g.target[k] != g.ignore ? 1 : 0;
    n = block_reduce<kThreads>(n, shi, Add());
    if (mean) scale = 1.0f / (float)max(n, 1);
    if (blockIdx.x == 0 && threadIdx.x == 0) ctl->scale = scale;
  }
  if (t == g.ignore) {
    if (ch == 0 && threadIdx.x == 0) rowloss[row] = 0.0f;
    if (GRADS)
      for (int c = lo + threadIdx.x * 4; c < hi; c += kThreads * 4) *reinterpret_cast<float4*>(l + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  const float *sm = g.stat + (int64_t)row * g.tiles, *sz = sm + (int64_t)rows * g.tiles, *st = sz + (int64_t)rows * g.tiles;
  const bool ok = t >= 0.0f && t < (float)classes && t == floorf(t);
  const int ti = ok ? (int)t : 0;
  const bool owner = ti >= lo && ti < hi;
  const float lt = owner ? (g.lt ? g.lt[row] : l[ti]) : 0.0f;
  float m = -INFINITY;
#pragma unroll 4
  for (int k = threadIdx.x; k < g.tiles; k += kThreads) m = fmaxf(m, sm[k]);
  m = block_reduce<kThreads>(m, sh, Max());
  float z = 0.0f, s = 0.0f;
  const float down = mean_scale(classes);
#pragma unroll 4
  for (int k = threadIdx.x; k < g.tiles; k += kThreads) z += sz[k] * exp_of(sm[k] - m);
  z = block_reduce<kThreads>(z, sh, Add());
  if (owner && g.smooth > 0.0f) {
    for (int k = threadIdx.x; k < g.tiles; k += kThreads)
      s += sm[k] > -INFINITY ? st[k] * (down / kDown) + (float)min(g.cols, classes - k * g.cols) * down * (sm[k] - m) : -INFINITY;
    s = block_reduce<kThreads>(s, sh, Add());
  }
  if (owner && threadIdx.x == 0) {
    float r = logf(z) - (1.0f - g.smooth) * (lt - m);
    if (g.smooth > 0.0f) r -= g.smooth * (s / ((float)classes * down));
    rowloss[row] = ok ? r : NAN;
  }
  if (!GRADS) return;
  const float iz = ok ? scale / z : NAN, q = scale * (g.smooth / (float)classes), p1 = scale * (1.0f - g.smooth);
  for (int c = lo + threadIdx.x * 4; c < hi; c += kThreads * 4) {
    const float4 a = *reinterpret_cast<const float4*>(l + c);
    float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      v[k] = fmaf(exp_of(v[k] - m), iz, -q);
      if (c + k == ti) v[k] -= p1;
      v[k] = c + k < classes ? v[k] : 0.0f;
    }
    *reinterpret_cast<float4*>(l + c) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

template <int KN>
constexpr int few_strip() { return KN <= 32 ? 512 : 256; }     // columns of dW a workgroup
template <int KN>
__global__ __launch_bounds__(kThreads) void k_few_pair(Few g, int rows, int classes) {
  __shared__ __attribute__((aligned(16))) float lds[4 * 32 * dfhip_few::kPitch];
  constexpr int CF = few_strip<KN>() / 128;
  const int lane = threadIdx.x & 63;
  int block = (int)blockIdx.x;
  if (block < g.n_dx) {
    // (consecutive workgroups go to the eight XCDs in turn: the column tiles of one range of classes on one XCD, side by side,
    // so that dl comes out of its L2)
    const int tiles = (g.width + 127) >> 7, tile = (block >> 3) % tiles, cut = (block >> 3) / tiles * 8 + (block & 7), k0 = cut * g.cut;
    if (cut >= g.cuts) return;
    dfhip_few::along<(KN + 31) / 32>(g.dx, tile * 128, k0, min(k0 + g.cut, classes), lds, g.parts + (int64_t)cut * rows * g.width);
    return;
  }
  block -= g.n_dx;
  if (block < g.n_dw) {
    // (consecutive workgroups go to the eight XCDs in turn; a strip's neighbours share lines where rows begin anywhere: each XCD
    // gets a run of strips)
    const int per = g.n_dw >> 3, id = (block & 7) * per + (block >> 3);
    const int strip = id / g.dw_cuts, cut = id % g.dw_cuts;
    const int n0 = (strip * 4 + (int)(threadIdx.x >> 6)) * 32 * CF, d0 = cut * g.dw_cut;
    if (n0 >= classes || strip >= g.strips) return;
    const uint64_t counted = __ballot(lane < rows && g.target[min(lane, rows - 1)] != g.ignore);
    dfhip_few::outer<KN, CF>(g.logits.a, rows, g.width, g.l, g.ld, g.dw, cut == 0 ? g.db : nullptr, classes, n0, d0,
                         min(d0 + g.dw_cut, g.width), counted);
    return;
  }
  loss_body<kThreads>(g.rowloss, g.ctl, g.loss, rows, reinterpret_cast<double*>(lds));
}

// 64 elements of dx a workgroup, each of its waves a quarter of the parts
__global__ __launch_bounds__(kThreads) void k_few_rest(const float* __restrict__ parts, float* __restrict__ dx, int n, int cuts) {
  __shared__ float sh[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, at = (int)blockIdx.x * 64 + lane;
  const int per = (cuts + 3) / 4, z1 = min(cuts, (wave + 1) * per);
  float v = 0.0f;
  if (at < n) {
    int z = wave * per;
    for (; z + 8 <= z1; z += 8) {
      float q[8];
#pragma unroll
      for (int k = 0; k < 8; k++) q[k] = parts[(int64_t)(z + k) * n + at];
#pragma unroll
      for (int k = 0; k < 8; k++) v += q[k];
    }
    for (; z < z1; z++) v += parts[(int64_t)z * n + at];
  }
  sh[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && at < n) dx[at] = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
}

__global__ __launch_bounds__(kThreads) void k_lce_scale(const float* __restrict__ src, const float* __restrict__ scalar,
                                                        float* __restrict__ dst, int64_t n) {
  const float s = scalar[0];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) dst[i] = src[i] * s;
}

struct Held {                                      // a pool block for the duration of a call (its reuse is stream-ordered)
  float* p = nullptr;
  ~Held() { if (p) (void)dfhip_free(p); }
  int take(int64_t floats) { return p ? DFHIP_OK : dfhip_malloc(floats, &p); }
};

int room(Held& h, int64_t& held, int64_t need) {   // scratch that grows as needed
  if (held >= need) return DFHIP_OK;
  if (h.p) { (void)dfhip_free(h.p); h.p = nullptr; }
  held = need;
  return h.take(need);
}

template <int T, int EPI>
int launch_logits(const Gemm& g) {
  static bool done = false;
  const int st = allow_lds((const void*)k_split_gemm<T, false, true, EPI>, lds_bytes<T>(), done);
  if (st != DFHIP_OK) return st;
  DF_LAUNCH((k_split_gemm<T, false, true, EPI>), dim3((unsigned)groups(g)), dim3(threads<T>()), lds_bytes<T>(), stream(), g);
  DF_LAUNCH_CHECK();
  if (g.rest) {
    DF_LAUNCH((k_split_rest<T, EPI>), dim3((unsigned)g.rest * slices<T>()), dim3(256), 0, stream(), g);
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

template <int T, int EPI>
int launch_pair(const Pair& p) {
  static bool done = false;
  const int st = allow_lds((const void*)k_lce_pair<T, EPI>, lds_bytes<T>(), done);
  if (st != DFHIP_OK) return st;
  DF_LAUNCH((k_lce_pair<T, EPI>), dim3((unsigned)(p.na + p.nb + (p.loss ? 1 : 0))), dim3(threads<T>()), lds_bytes<T>(), stream(), p);
  DF_LAUNCH_CHECK();
  if (p.a.rest + p.b.rest) {
    DF_LAUNCH((k_lce_pair_rest<T, EPI>), dim3((unsigned)(p.a.rest + p.b.rest) * slices<T>()), dim3(256), 0, stream(), p);
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

template <class F>
int with_tile(const Plan& p, F f) {
  if (p.tile == 256) return f(std::integral_constant<int, 256>());
  if (p.tile == 128) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 64>());
}

// The cheapest way through a call's products.  A training loop asks for the same few again and again: the last answers are kept,
// by the sizes alone.
// `dw_rows`: rows of the weight product that are wanted -- width, 1 for the bias gradient alone (a product one tile high of which
// nothing is stored), 0 for neither.
struct Choice {
  int64_t rows, width, classes;
  bool dx;
  int64_t dw_rows;
  Plan logits, a, b;
};
const Choice* choose(int64_t rows, int64_t width, int64_t classes, bool dx, int64_t dw_rows) {
  static thread_local Choice kept[8] = {};
  static thread_local int turn = 0;
  for (const Choice& c : kept)
    if (c.rows == rows && c.width == width && c.classes == classes && c.dx == dx && c.dw_rows == dw_rows && c.logits.tile)
      return &c;
  Choice c = {};
  c.rows = rows; c.width = width; c.classes = classes; c.dx = dx; c.dw_rows = dw_rows;
  double least = 1e300, least_pair = 1e300;
  for (int tile : {256, 128, 64}) {
    Plan l[kWays], a[kWays] = {}, b[kWays] = {};
    // (256 x 128 tiles are for the pair alone: 8192 x 1024 x 50001 7.67 -> 7.16 ms; the logits of 157 x 4274 x 63752 take 847 us with
    // them and 828 without)
    const int nl = tile == 256 ? 0 : ways(tile, rows, classes, (int)df_ceil_div(width, 32), l);
    for (int i = 0; i < nl; i++) {
      const double us = cost_us(&l[i], 1);
      if (us < least) { least = us; c.logits = l[i]; }
    }
    if (!dx && !dw_rows) continue;
    a[0].tile = b[0].tile = tile;                  // (no product)
    const int na = dx ? ways(tile, rows, width, (int)df_ceil_div(classes, 32), a) : 1;
    const int nb = dw_rows ? ways(tile, dw_rows, classes, (int)df_ceil_div(rows, 32), b) : 1;
    for (int i = 0; i < na; i++)
      for (int j = 0; j < nb; j++) {
        Plan both[2] = {a[i], b[j]};
        const double us = dx && dw_rows ? cost_us(both, 2) : cost_us(dx ? &a[i] : &b[j], 1);
        if (us < least_pair) { least_pair = us; c.a = a[i]; c.b = b[j]; }
      }
  }
  if (!c.logits.tile || ((dx || dw_rows) && !c.a.tile)) return nullptr;
  kept[turn] = c;
  const Choice* at = &kept[turn];
  turn = (turn + 1) & 7;
  return at;
}

int rows_pass(float* logits, const float* target, int n, int launch_rows, float* rowloss, int classes, int cells, float ignore,
              float smooth) {
#define ROWS(T, U)                                                                                                        \
  DF_LAUNCH((k_lce_rows<T, U>), dim3((unsigned)launch_rows), dim3(T), 0, stream(), logits, target, n, rowloss, classes,   \
            cells, ignore, smooth)
  if (cells <= 2048) ROWS(256, 1);
  else if (cells <= 4096) ROWS(256, 2);
  else if (cells <= 8192) ROWS(1024, 1);
  else if (cells <= 16384) ROWS(1024, 2);
  else if (cells <= 32768) ROWS(1024, 4);
  else if (cells <= 57344) ROWS(1024, 7);
  else ROWS(1024, 0);
#undef ROWS
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

// Which calls go this way (measured, microseconds, this way / the split products):
//   up to 32 rows: all.  loss and gradients, 32 rows: 256 x 1000 21 / 23, 1024 x 16384 65 / 93, 1024 x 50001 180 / 284,
//     2048 x 99991 691 / 1137; the loss alone: 13 / 18, 27 / 54, 54 / 140, 199 / 540
//   33 to 64 rows, where the fp32 matrix cores begin to count: the loss alone where the reduction is short or W large (64 rows:
//     256 x 1000 15 / 18, 1024 x 1000 22 / 22, 2048 x 1000 34 / 26, 1024 x 5003 25 / 34, 1024 x 50001 85 / 139); with gradients
//     where W is very large (1024 x 34001 220 / 196, 1024 x 50001 277 / 284, 2048 x 50001 513 / 584), and where the launches are
//     what counts, four instead of six (100 x 500 22 / 21, 256 x 1000 24.5 / 24, 512 x 2000 28.6 / 29.5, 64 x 50001 52 / 61, but
//     1024 x 1000 34 / 31, 256 x 16384 47 / 45; the host, where it is slower than the device, saves 5 us of 38)
//   65 to 128 rows: the loss alone over a very large W (128 rows: 1024 x 34001 121 / 106, 1024 x 50001 154 / 139, 2048 x 50001 287 / 278,
//     1024 x 99991 273 / 282, 2048 x 99991 500 / 551, 4096 x 64000 561 / 668; 65 rows 125 / 108 to 549 / 657)
inline bool few_rows(int64_t rows, int64_t width, int64_t classes, bool grads) {
  const int64_t size = width * classes, M = 1 << 20;
  if (classes < 4 || rows > (grads ? 1 : 2) * dfhip_few::kMost) return false;
  if (rows > dfhip_few::kMost) return size >= 128 * M;
  return rows <= 32 || (grads ? size >= 48 * M || (width <= 512 && size <= 7 * M / 2) : size >= 3 * M || width <= 1024);
}

template <int RB>
int few_logits(const Few& g) {
  const dim3 grid((unsigned)(df_ceil_div(g.tiles, 8) * 8 * df_ceil_div(g.logits.rows, 64)));
  if (g.cols == 32) DF_LAUNCH((k_few_logits<RB, 1, 8>), grid, dim3(512), 0, stream(), g);
  else DF_LAUNCH((k_few_logits<RB, 4, 4>), grid, dim3(256), 0, stream(), g);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

int few_rows_forward(const float* x, const float* w, const float* bias, const float* target, float* loss, float* dx, float* dw,
                     float* db, int rows, int width, int classes, float ignore, float smooth, int mean) {
  const bool grads = dx || dw || db;
  const int64_t ld = df_ceil_div(classes, 128) * 128;
  const int cols = df_ceil_div(classes, 128) < num_cus() ? 32 : 128, tiles = (int)df_ceil_div(classes, cols);
  // dx: about two workgroups a CU, at most 256 parts; two windows each at least, one where that makes less than 32 of them
  const int dx_tiles = (int)df_ceil_div(width, 128), windows = (int)df_ceil_div(classes, dfhip_few::kWindow);
  int cuts = std::max(1, std::min(std::min(256, 2 * num_cus() / dx_tiles), std::max((windows + 1) / 2, std::min(windows, 32))));
  const int cut = (int)df_ceil_div(df_ceil_div(classes, cuts), dfhip_few::kWindow) * dfhip_few::kWindow;
  cuts = (int)df_ceil_div(classes, cut);
  Held logits, small, parts;
  const int64_t stats = 3 * (int64_t)rows * tiles;
  int st = small.take((int64_t)(sizeof(Ctl) / 4) + rows + stats);
  if (st == DFHIP_OK) st = logits.take(rows * ld);
  if (st == DFHIP_OK && dx && cuts > 1) st = parts.take((int64_t)cuts * rows * width);
  if (st != DFHIP_OK) return st;
  Ctl* ctl = reinterpret_cast<Ctl*>(small.p);
  float* rowloss = small.p + sizeof(Ctl) / 4;
  Few g = {};
  g.logits = {x, w, width, classes, rows, classes, width};
  g.dx = {logits.p, w, ld, classes, rows, width, classes};
  g.bias = bias;
  g.l = logits.p;
  g.ld = ld;
  g.stat = rowloss + rows;
  g.tiles = tiles;
  g.cols = cols;
  g.target = target;
  g.ignore = ignore;
  g.smooth = smooth;
  g.dw = dw;
  g.db = db;
  g.parts = cuts > 1 ? parts.p : dx;
  g.loss = loss;
  g.rowloss = rowloss;
  g.ctl = ctl;
  g.width = width;
  st = rows <= 32 ? few_logits<1>(g) : few_logits<2>(g);
  if (st != DFHIP_OK) return st;
  const int chunk = grads ? std::max(4096, (int)df_ceil_div(df_ceil_div(ld, 64), 1024) * 1024) : (int)ld;
  const int chunks = (int)df_ceil_div(ld, chunk);
  if (grads)
    DF_LAUNCH((k_few_rows<true, true>), dim3((unsigned)(rows * chunks)), dim3(kThreads), 0, stream(), g, rows, classes, mean, chunk, chunks,
              rowloss, ctl);
  else
    DF_LAUNCH((k_few_rows<false, true>), dim3((unsigned)rows), dim3(kThreads), 0, stream(), g, rows, classes, mean, chunk, chunks, rowloss,
              ctl);
  DF_LAUNCH_CHECK();
  if (!grads) {
    DF_LAUNCH(k_lce_loss, dim3(1), dim3(1024), 0, stream(), rowloss, ctl, loss, (int64_t)rows);
    DF_LAUNCH_CHECK();
    return DFHIP_OK;
  }
  if (dx) {
    g.cuts = cuts;
    g.cut = cut;
    g.n_dx = dx_tiles * (int)df_ceil_div(cuts, 8) * 8;
  }
  if (dw || db) {
    g.strips = (int)df_ceil_div(classes, rows <= 32 ? few_strip<32>() : few_strip<64>());
    // dW: about four workgroups a CU, 32 rows each at least
    const int want = dw ? std::max(1, std::min((int)df_ceil_div(width, 32), 4 * num_cus() / g.strips)) : 1;
    g.dw_cut = (int)df_ceil_div(df_ceil_div(width, want), 32) * 32;
    g.dw_cuts = dw ? (int)df_ceil_div(width, g.dw_cut) : 1;
    g.n_dw = (int)df_ceil_div((int64_t)g.strips * g.dw_cuts, 8) * 8;
  }
  const dim3 grid((unsigned)(g.n_dx + g.n_dw + 1));
#define FEW(KN) DF_LAUNCH((k_few_pair<KN>), grid, dim3(kThreads), 0, stream(), g, rows, classes)
  if (rows <= 8) FEW(8);
  else if (rows <= 32) FEW(32);
  else FEW(64);
#undef FEW
  DF_LAUNCH_CHECK();
  if (dx && cuts > 1) {
    const int n = rows * width;
    DF_LAUNCH(k_few_rest, dim3((unsigned)df_ceil_div(n, 64)), dim3(kThreads), 0, stream(), parts.p, dx, n, cuts);
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

}  // namespace

extern "C" {

int dfhip_linear_ce_forward(const float* x, const float* w, const float* bias, const float* target, float* loss, float* dx,
                            float* dw, float* db, int64_t rows, int64_t width, int64_t classes, int64_t ignore_index,
                            double label_smoothing, int mean) {
  DF_INIT();
  DF_CHECK_ARG(rows >= 0 && width >= 1 && classes >= 1, "linear_ce_forward: bad extents (%lld, %lld, %lld)", (long long)rows,
               (long long)width, (long long)classes);
  DF_CHECK_ARG(rows <= (1 << 30) && width <= (1 << 24), "linear_ce_forward: at most 2^30 rows and a width of 2^24");
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
  if (few_rows(rows, width, classes, grads)) {
    ProfScope prof("linear_ce", (grads ? 6.0 : 2.0) * (double)rows * (double)width * (double)classes,
                   4.0 * ((grads ? 3.0 : 1.0) * (double)width * classes + 2.0 * (double)rows * width));
    return few_rows_forward(x, w, bias, target, loss, dx, dw, db, (int)rows, (int)width, (int)classes, (float)ignore_index,
                            (float)label_smoothing, mean);
  }
  const int64_t np = padded(rows), dp = padded(width), vp = padded(classes);
  // pieces of about the same length, a multiple of 256 rows
  const int64_t row_bytes = grads ? 4 * vp : 12 * df_ceil_div(classes, 32);
  const int64_t cap = std::min<int64_t>(kPieceRows, std::max<int64_t>(256, kPieceBytes / row_bytes / 256 * 256));
  const int64_t pieces = df_ceil_div(rows, cap);
  const int64_t piece = padded(df_ceil_div(rows, pieces));
  Held xs, ws, logits, small, parts;
  int64_t held = 0;
  int st = small.take((int64_t)(sizeof(Ctl) / 4) + rows);
  if (st == DFHIP_OK) st = xs.take(np * dp);
  if (st == DFHIP_OK) st = ws.take(dp * vp);
  if (st == DFHIP_OK) st = logits.take(grads ? piece * vp : piece * (1 + 3 * df_ceil_div(classes, 32)));
  if (st != DFHIP_OK) return st;
  Ctl* ctl = reinterpret_cast<Ctl*>(small.p);
  float* rowloss = small.p + sizeof(Ctl) / 4;
  const float ignore = (float)ignore_index;
  ProfScope prof("linear_ce", (grads ? 6.0 : 2.0) * (double)rows * (double)width * (double)classes,
                 4.0 * (grads ? 2.0 : 1.0) * ((double)rows * width + (double)width * classes));

  const int sample = width * classes >= kSampled;
  DF_LAUNCH(k_lce_scan, dim3(2 * kScan), dim3(kThreads), 0, stream(), x, rows, width, target, ignore, w, width * classes, sample,
            ctl);
  DF_LAUNCH_CHECK();
  const int64_t bx = std::min<int64_t>(np * dp / 2048, 2048), bw = std::min<int64_t>(dp * vp / 2048, 4096);
  DF_LAUNCH((k_lce_split<false>), dim3((unsigned)(bx + bw + 1)), dim3(kThreads), 0, stream(), x, rows, width, w, classes, (char*)xs.p,
            (char*)ws.p, target, ignore, mean, bx, bw, sample, ctl);
  DF_LAUNCH_CHECK();
  if (sample) {
    DF_LAUNCH((k_lce_split<true>), dim3(1024), dim3(kThreads), 0, stream(), x, rows, width, w, classes, (char*)xs.p, (char*)ws.p,
              target, ignore, mean, (int64_t)0, (int64_t)1024, sample, ctl);
    DF_LAUNCH_CHECK();
  }

  for (int64_t r0 = 0; r0 < rows; r0 += piece) {
    const int64_t n = std::min(piece, rows - r0);
    Gemm g = {};
    g.a = (const char*)xs.p + r0 * dp * 4;
    g.lda = dp * 4;
    g.b = (const char*)ws.p;
    g.ldb = vp * 4;
    g.bias = bias;
    g.exp_a = &ctl->ex;
    g.exp_b = &ctl->ew;
    const Choice* how = choose(n, width, classes, dx != nullptr, dw ? width : db ? 1 : 0);
    DF_CHECK_ARG(how, "linear_ce_forward: too many tiles");
    if (grads) {
      g.c = logits.p;
      g.ldc = vp;
    } else {                                       // the softmax's parts instead of the logits
      g.units = (int)df_ceil_div(classes, how->logits.tile == 64 ? unit<64>() : unit<128>());
      g.lt = logits.p;
      g.stat = logits.p + n;
      g.target = target + r0;
      g.sum = label_smoothing > 0.0;
    }
    apply(g, how->logits, n, classes);
    st = room(parts, held, std::max(parts_floats(how->logits), parts_floats(how->a) + parts_floats(how->b)));
    if (st != DFHIP_OK) return st;
    g.parts = parts.p;
    if (how->logits.tile == 128) st = grads ? launch_logits<128, EPI_BIAS>(g) : launch_logits<128, EPI_STATS>(g);
    else st = grads ? launch_logits<64, EPI_BIAS>(g) : launch_logits<64, EPI_STATS>(g);
    if (st != DFHIP_OK) return st;
    if (!grads) {
      Few f = {};
      f.stat = g.stat;
      f.tiles = g.units;
      f.cols = how->logits.tile == 64 ? unit<64>() : unit<128>();
      f.lt = g.lt;
      f.ld = classes;
      f.target = g.target;
      f.ignore = ignore;
      f.smooth = (float)label_smoothing;
      DF_LAUNCH((k_few_rows<false, false>), dim3((unsigned)n), dim3(kThreads), 0, stream(), f, (int)n, (int)classes, mean,
                (int)classes, 1, rowloss + r0, ctl);
      DF_LAUNCH_CHECK();
      continue;
    }
    st = rows_pass(logits.p, target + r0, (int)n, (int)(df_ceil_div(n, 32) * 32), rowloss + r0, (int)classes, (int)vp, ignore,
                   (float)label_smoothing);
    if (st != DFHIP_OK) return st;
    Pair p = {};
    p.a.exp_c = p.b.exp_c = -kTopDl;
    p.a.scale = p.b.scale = &ctl->scale;
    if (dx) {
      p.a.a = (const char*)logits.p;
      p.a.lda = vp * 4;
      p.a.b = (const char*)ws.p;
      p.a.ldb = vp * 4;
      p.a.c = dx + r0 * width;
      p.a.ldc = width;
      p.a.exp_a = &ctl->ew;
      p.a.parts = parts.p;
      apply(p.a, how->a, n, width);
      p.na = groups(p.a);
    }
    if (dw || db) {
      p.b.a = (const char*)xs.p + r0 * dp * 4;
      p.b.lda = dp * 4;
      p.b.b = (const char*)logits.p;
      p.b.ldb = vp * 4;
      p.b.c = dw;
      p.b.ldc = classes;
      p.b.exp_a = &ctl->ex;
      p.b.colsum = db;
      p.b.parts = parts.p + parts_floats(how->a);
      apply(p.b, how->b, width, classes);
      p.nb = groups(p.b);
    }
    if (r0 + n == rows) {
      p.rowloss = rowloss;
      p.ctl = ctl;
      p.loss = loss;
      p.rows = rows;
    }
    st = with_tile(how->a, [&](auto t) {
      constexpr int T = decltype(t)::value;
      return r0 == 0 ? launch_pair<T, EPI_STORE>(p) : launch_pair<T, EPI_ADD>(p);
    });
    if (st != DFHIP_OK) return st;
  }
  if (grads) return DFHIP_OK;
  DF_LAUNCH(k_lce_loss, dim3(1), dim3(1024), 0, stream(), rowloss, ctl, loss, rows);
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

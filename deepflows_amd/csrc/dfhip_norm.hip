// Root-mean-square normalisation over the last axis with the residual's addition, and its gradient.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   n = h r,  g = dy w,  dx = r (g - n mean(g n)) + (what h received from its other readers),  dw = sum over rows of dy n
//
// Bound: HBM.  Forward 16 bytes an element (x, residual in; y, h out), backward 16 (dy, h, the other gradient in; dx out): a
// row is held in registers between the reduction and its use, so every array is touched once.
//
// Layout: a row belongs to a TEAM of threads, four consecutive elements a thread and trip:
//   width <= 128: 16 lanes a row, <= 512: 32 lanes, <= 1024: one wave, <= 4096: four waves, <= 16384 (forward: 32768): sixteen;
//   wider rows: sixteen waves that read the row twice (the second time out of L2).
// Loads and stores are 16 bytes wherever the row begins (the hardware asks for 4-byte alignment only): 4-byte accesses for rows of
// a width that is no multiple of 4 cost 20 % at 1860 x 3578 and 58 % at 315 x 12242 (31 -> 13 us).
// Measured, with residual: 16384 x 4096 both ways 390 us = 5.5 TB/s, 3890 x 3056 forward 29 us = 6.5 TB/s (a large copy: 5.1).
// A thread keeps the same columns for every row its team works on, so the sum over rows of dy n stays in registers until the
// end; the teams of a workgroup meet in LDS, the workgroups' partial rows are added by a second launch in a fixed order.
#include <math.h>

#include <algorithm>

#include "dfhip_internal.h"

using namespace dfhip;

namespace {

constexpr int kThreads = 256;
constexpr int kWide = 1024;
// A launch holds fewer than 2^32 threads: more workgroups than these (of up to 1 024) are several launches.
constexpr int64_t kGroups = 1 << 21;
template <int T> constexpr int threads() { return T > kThreads ? T : kThreads; }

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// four elements of which `left` exist; what does not reads as zero and is not written
__device__ __forceinline__ void load4(float* v, const float* p, int64_t left) {
  if (left >= 4) {
    const float4u t = *reinterpret_cast<const float4u*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = e < left ? p[e] : 0.0f;
  }
}
__device__ __forceinline__ void store4(float* p, const float* v, int64_t left) {
  if (left >= 4) {
    float4u t;
    t.x = v[0]; t.y = v[1]; t.z = v[2]; t.w = v[3];
    *reinterpret_cast<float4u*>(p) = t;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (e < left) p[e] = v[e];
  }
}

// the sum over the T threads of a team, in every one of them (T <= 64: lanes of one wave; more: the workgroup)
template <int T, class X>
__device__ __forceinline__ X team_sum(X v, X* sh) {
#pragma unroll
  for (int off = (T < 64 ? T : 64) / 2; off; off >>= 1) v += __shfl_xor(v, off);
  if (T > 64) {
    __syncthreads();                               // (sh may still be read from the last call)
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < T / 64; w++) v += sh[w];
  }
  return v;
}

// U trips of four elements a thread cover the row: T * U * 4 >= width
template <int T, int U, bool RES>
__global__ __launch_bounds__(threads<T>()) void k_rms_fwd(const float* __restrict__ x, const float* res,
                                                          const float* __restrict__ w, float* __restrict__ y, float* h,
                                                          float* __restrict__ rstd, int64_t rows, int width, double inv, float eps) {
  __shared__ double sh[threads<T>() / 64];
  const int team = threadIdx.x / T, lane = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (threads<T>() / T) + team;
  const bool live = row < rows;                    // (a team whose row does not exist keeps the others company at barriers)
  const int64_t base = (live ? row : 0) * width;
  float v[U][4];
  double ss = 0.0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * 4;
    load4(v[u], x + base + c, width - c);
  }
  if (RES) {
    float r[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * 4;
      load4(r[u], res + base + c, width - c);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * 4;
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] += r[u][e];
      if (live) store4(h + base + c, v[u], width - c);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) ss = fma((double)v[u][e], (double)v[u][e], ss);
  ss = team_sum<T>(ss, sh);
  const float r = (float)(1.0 / sqrt(fma(ss, inv, (double)eps)));
  if (!live) return;
  if (rstd && lane == 0) rstd[row] = r;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * 4;
    float o[4], wv[4];
    if (w) load4(wv, w + c, width - c);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = w ? v[u][e] * r * wv[e] : v[u][e] * r;
    store4(y + base + c, o, width - c);
  }
}

// rows wider than the registers hold: the row twice
template <bool RES>
__global__ __launch_bounds__(kWide) void k_rms_fwd_wide(const float* x, const float* res, const float* __restrict__ w,
                                                        float* __restrict__ y, float* h, float* __restrict__ rstd, int64_t width,
                                                        double inv, float eps) {
  __shared__ double sh[kWide / 64];
  const int64_t base = (int64_t)blockIdx.x * width;
  double ss = 0.0;
  for (int64_t c = (int64_t)threadIdx.x * 4; c < width; c += kWide * 4) {
    float v[4];
    load4(v, x + base + c, width - c);
    if (RES) {
      float r[4];
      load4(r, res + base + c, width - c);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] += r[e];
      store4(h + base + c, v, width - c);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) ss = fma((double)v[e], (double)v[e], ss);
  }
  ss = team_sum<kWide>(ss, sh);
  const float r = (float)(1.0 / sqrt(fma(ss, inv, (double)eps)));
  if (rstd && threadIdx.x == 0) rstd[blockIdx.x] = r;
  const float* s = RES ? h : x;                    // (each thread reads back what it wrote itself)
  for (int64_t c = (int64_t)threadIdx.x * 4; c < width; c += kWide * 4) {
    float v[4], wv[4];
    load4(v, s + base + c, width - c);
    if (w) load4(wv, w + c, width - c);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = w ? v[e] * r * wv[e] : v[e] * r;
    store4(y + base + c, v, width - c);
  }
}

// partial: gridDim.x rows of `width` sums of dy n, or NULL
template <int T, int U>
__global__ __launch_bounds__(threads<T>()) void k_rms_bwd(const float* __restrict__ dy, const float* __restrict__ h,
                                                          const float* __restrict__ rstd, const float* __restrict__ w,
                                                          const float* add, float* dx, float* __restrict__ partial, int64_t rows,
                                                          int width) {
  __shared__ float sh[threads<T>() / 64];
  constexpr int TEAMS = threads<T>() / T;
  __shared__ float meet[TEAMS > 1 ? T * U * 4 * TEAMS : 1];
  const int team = threadIdx.x / T, lane = threadIdx.x % T;
  float sum[U][4], wv[U][4];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * 4;
#pragma unroll
    for (int e = 0; e < 4; e++) { sum[u][e] = 0.0f; wv[u][e] = 1.0f; }
    if (w) load4(wv[u], w + c, width - c);
  }
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  // (the trip count is the workgroup's, so that every thread reaches the barriers of a team of several waves)
  for (int64_t row0 = (int64_t)blockIdx.x * TEAMS; row0 < rows; row0 += step) {
    const bool live = row0 + team < rows;
    const int64_t row = live ? row0 + team : row0;
    const int64_t base = row * width;
    const float r = rstd[row];
    float g[U][4], n[U][4];
    float dot = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * 4;
      load4(g[u], dy + base + c, width - c);
      load4(n[u], h + base + c, width - c);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        n[u][e] *= r;
        if (live) sum[u][e] = fmaf(g[u][e], n[u][e], sum[u][e]);
        g[u][e] *= wv[u][e];
        dot = fmaf(g[u][e], n[u][e], dot);
      }
    if (!dx) continue;
    const float c1 = team_sum<T>(dot, sh) * inv;
    if (live)
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int c = (u * T + lane) * 4;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = r * (g[u][e] - n[u][e] * c1);
        if (add) {
          float a[4];
          load4(a, add + base + c, width - c);
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] += a[e];
        }
        store4(dx + base + c, o, width - c);
      }
  }
  if (!partial) return;
  float* prow = partial + (int64_t)blockIdx.x * width;
  if (TEAMS == 1) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * 4;
      store4(prow + c, sum[u], width - c);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) meet[team * (T * U * 4) + (u * T + lane) * 4 + e] = sum[u][e];
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += threads<T>()) {
    float s = 0.0f;
#pragma unroll
    for (int t = 0; t < TEAMS; t++) s += meet[t * (T * U * 4) + c];
    prow[c] = s;
  }
}

// rows wider than the registers hold: dx alone, a workgroup a row
__global__ __launch_bounds__(kWide) void k_rms_bwd_wide(const float* __restrict__ dy, const float* __restrict__ h,
                                                        const float* __restrict__ rstd, const float* __restrict__ w,
                                                        const float* add, float* dx, int64_t width) {
  __shared__ float sh[kWide / 64];
  const int64_t base = (int64_t)blockIdx.x * width;
  const float r = rstd[blockIdx.x];
  float dot = 0.0f;
  for (int64_t c = (int64_t)threadIdx.x * 4; c < width; c += kWide * 4) {
    float g[4], n[4], wv[4];
    load4(g, dy + base + c, width - c);
    load4(n, h + base + c, width - c);
    if (w) load4(wv, w + c, width - c);
#pragma unroll
    for (int e = 0; e < 4; e++) dot = fmaf(w ? g[e] * wv[e] : g[e], n[e] * r, dot);
  }
  const float c1 = team_sum<kWide>(dot, sh) * (1.0f / (float)width);
  for (int64_t c = (int64_t)threadIdx.x * 4; c < width; c += kWide * 4) {
    float g[4], n[4], wv[4], a[4];
    load4(g, dy + base + c, width - c);
    load4(n, h + base + c, width - c);
    if (w) load4(wv, w + c, width - c);
    if (add) load4(a, add + base + c, width - c);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float o = r * ((w ? g[e] * wv[e] : g[e]) - n[e] * r * c1);
      if (add) o += a[e];
      g[e] = o;
    }
    store4(dx + base + c, g, width - c);
  }
}

// ... and partial sums of dy n over a slice of the rows: blockIdx.x a run of kThreads columns, blockIdx.y a slice
__global__ __launch_bounds__(kThreads) void k_rms_dw_wide(const float* __restrict__ dy, const float* __restrict__ h,
                                                          const float* __restrict__ rstd, float* __restrict__ partial,
                                                          int64_t rows, int64_t width) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= width) return;
  float s = 0.0f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) s = fmaf(dy[row * width + c], h[row * width + c] * rstd[row], s);
  partial[(int64_t)blockIdx.y * width + c] = s;
}

// dw[c] = sum over the partial rows, in the order of the rows within 16 groups and then of the groups; 64 columns a workgroup from
// column `first` on
__global__ __launch_bounds__(1024) void k_rms_dw_sum(const float* __restrict__ partial, float* __restrict__ dw, int n_partial,
                                                     int64_t width, int64_t first) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int64_t c = first + (int64_t)blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (c < width) {
    int p = grp;
    for (; p + 48 < n_partial; p += 64) {          // four loads in flight
      const float a = partial[(int64_t)p * width + c], b = partial[(int64_t)(p + 16) * width + c];
      const float d = partial[(int64_t)(p + 32) * width + c], e = partial[(int64_t)(p + 48) * width + c];
      s = (((s + a) + b) + d) + e;
    }
    for (; p < n_partial; p += 16) s += partial[(int64_t)p * width + c];
  }
  sh[grp][lane] = s;
  __syncthreads();
  if (grp == 0 && c < width) {
#pragma unroll
    for (int g = 1; g < 16; g++) s += sh[g][lane];
    dw[c] = s;
  }
}

// launch(first, n) over [0, total), `most` at a time
template <class F>
int in_pieces(int64_t total, int64_t most, F launch) {
  for (int64_t first = 0; first < total; first += most) {
    launch(first, std::min(total - first, most));
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

template <int T, int U>
int fwd(const float* x, const float* res, const float* w, float* y, float* h, float* rstd, int64_t rows, int64_t width, float eps) {
  constexpr int64_t TEAMS = threads<T>() / T;
  return in_pieces(rows, kGroups * TEAMS, [&](int64_t r0, int64_t n) {
    const dim3 grid((unsigned)df_ceil_div(n, TEAMS)), block(threads<T>());
    const int64_t at = r0 * width;
    float* rs = rstd ? rstd + r0 : nullptr;
    if (res)
      DF_LAUNCH((k_rms_fwd<T, U, true>), grid, block, 0, stream(), x + at, res + at, w, y + at, h + at, rs, n, (int)width,
                1.0 / (double)width, eps);
    else
      DF_LAUNCH((k_rms_fwd<T, U, false>), grid, block, 0, stream(), x + at, nullptr, w, y + at, nullptr, rs, n, (int)width,
                1.0 / (double)width, eps);
  });
}

template <int T, int U>
int bwd(const float* dy, const float* h, const float* rstd, const float* w, const float* add, float* dx, float* partial,
        int blocks, int64_t rows, int64_t width) {
  DF_LAUNCH((k_rms_bwd<T, U>), dim3(blocks), dim3(threads<T>()), 0, stream(), dy, h, rstd, w, add, dx, partial, rows, (int)width);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

// the team of a row of `width` elements: CALL(T, U) of the narrowest form that holds it
#define RMS_FORMS(CALL)                      \
  do {                                       \
    if (width <= 64) return CALL(16, 1);     \
    if (width <= 128) return CALL(16, 2);    \
    if (width <= 256) return CALL(32, 2);    \
    if (width <= 512) return CALL(32, 4);    \
    if (width <= 1024) return CALL(64, 4);   \
    if (width <= 2048) return CALL(256, 2);  \
    if (width <= 4096) return CALL(256, 4);  \
    if (width <= 8192) return CALL(1024, 2); \
    if (width <= 16384) return CALL(1024, 4);\
  } while (0)

int run_fwd(const float* x, const float* res, const float* w, float* y, float* h, float* rstd, int64_t rows, int64_t width,
            float eps) {
#define CALL(T, U) fwd<T, U>(x, res, w, y, h, rstd, rows, width, eps)
  RMS_FORMS(CALL);
  if (width <= 32768) return CALL(1024, 8);        // (the backward pass holds twice as many values a thread: it would spill)
#undef CALL
  return in_pieces(rows, kGroups, [&](int64_t r0, int64_t n) {
    const int64_t at = r0 * width;
    float* rs = rstd ? rstd + r0 : nullptr;
    if (res) DF_LAUNCH(k_rms_fwd_wide<true>, dim3((unsigned)n), dim3(kWide), 0, stream(), x + at, res + at, w, y + at, h + at, rs, width,
                       1.0 / (double)width, eps);
    else DF_LAUNCH(k_rms_fwd_wide<false>, dim3((unsigned)n), dim3(kWide), 0, stream(), x + at, nullptr, w, y + at, nullptr, rs, width,
                   1.0 / (double)width, eps);
  });
}

int run_bwd(const float* dy, const float* h, const float* rstd, const float* w, const float* add, float* dx, float* partial,
            int blocks, int64_t rows, int64_t width) {
#define CALL(T, U) bwd<T, U>(dy, h, rstd, w, add, dx, partial, blocks, rows, width)
  RMS_FORMS(CALL);
#undef CALL
  if (dx) {
    const int st = in_pieces(rows, kGroups, [&](int64_t r0, int64_t n) {
      const int64_t at = r0 * width;
      DF_LAUNCH(k_rms_bwd_wide, dim3((unsigned)n), dim3(kWide), 0, stream(), dy + at, h + at, rstd + r0, w, add ? add + at : nullptr,
                dx + at, width);
    });
    if (st != DFHIP_OK) return st;
  }
  if (partial) {
    DF_LAUNCH(k_rms_dw_wide, dim3((unsigned)df_ceil_div(width, kThreads), (unsigned)blocks), dim3(kThreads), 0, stream(), dy, h,
              rstd, partial, rows, width);
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

int check_shape(const char* name, int64_t rows, int64_t width) {
  DF_CHECK_ARG(rows >= 0 && width >= 1, "%s: rows must be >= 0 and width >= 1", name);
  DF_CHECK_ARG(rows <= 0x7fffffff && width <= 0x7fffffff, "%s: rows and width must be below 2^31", name);
  return DFHIP_OK;
}

}  // namespace

extern "C" {

int dfhip_rms_norm_forward(const float* x, const float* residual, const float* weight, float* y, float* h, float* rstd,
                           int64_t rows, int64_t width, float eps) {
  DF_INIT();
  int st = check_shape("rms_norm_forward", rows, width);
  if (st != DFHIP_OK) return st;
  DF_CHECK_ARG(eps >= 0.0f, "rms_norm_forward: eps must be >= 0");
  if (rows == 0) return DFHIP_OK;
  DF_CHECK_ARG(x && y && (!residual || h), "rms_norm_forward: null array");
  ProfScope prof("rms_norm_fwd", 4.0 * (double)rows * (double)width, (residual ? 16.0 : 8.0) * (double)rows * (double)width);
  return run_fwd(x, residual, weight, y, h, rstd, rows, width, eps);
}

int dfhip_rms_norm_backward(const float* dy, const float* h, const float* rstd, const float* weight, const float* add,
                            float* dx, float* dweight, int64_t rows, int64_t width) {
  DF_INIT();
  int st = check_shape("rms_norm_backward", rows, width);
  if (st != DFHIP_OK) return st;
  DF_CHECK_ARG(dx || dweight, "rms_norm_backward: nothing to compute");
  if (rows == 0) return dweight ? dfhip_fill(dweight, width, 0.0f) : DFHIP_OK;
  DF_CHECK_ARG(dy && h && rstd, "rms_norm_backward: null array");
  ProfScope prof("rms_norm_bwd", 8.0 * (double)rows * (double)width, (add ? 16.0 : 12.0) * (double)rows * (double)width);
  // workgroups that share the rows, and as many partial rows: a team waits for each row's loads, so narrow rows need many of them
  const int64_t teams = width <= 128 ? 16 : width <= 512 ? 8 : width <= 1024 ? 4 : 1;
  const int blocks = (int)std::min<int64_t>(df_ceil_div(rows, teams), (width <= 128 ? 8 : width <= 1024 ? 4 : 2) * num_cus());
  float* partial = nullptr;
  if (dweight) {
    partial = workspace((size_t)blocks * (size_t)width * sizeof(float));
    if (!partial) return DFHIP_OUT_OF_MEMORY;
  }
  st = run_bwd(dy, h, rstd, weight, add, dx, partial, blocks, rows, width);
  if (st != DFHIP_OK || !dweight) return st;
  return in_pieces(width, kGroups * 64, [&](int64_t first, int64_t n) {
    DF_LAUNCH(k_rms_dw_sum, dim3((unsigned)df_ceil_div(n, 64)), dim3(1024), 0, stream(), partial, dweight, blocks, width, first);
  });
}

}  // extern "C"

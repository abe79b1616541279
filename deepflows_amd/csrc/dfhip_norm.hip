// Root-mean-square normalisation over the last axis with the residual's addition, and its gradient.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   n = h r,  g = dy w,  dx = r (g - n mean(g n)) + (what h received from its other readers),  dw = sum over rows of dy n
//
// Bound: HBM.  Forward 16 bytes an element (x, residual in; y, h out), backward 16 (dy, h, the other gradient in; dx out): a
// row is held in registers between the reduction and its use, so every array is touched once.
//
// Layout: a row belongs to a TEAM of threads, a quarter of a wave up to four waves, V consecutive elements a thread and trip:
//   width <= 128: 16 lanes a row, <= 512: 32 lanes, <= 1024: one wave, <= 16384: four waves; wider rows: four waves that read
//   the row twice (the second time out of L2).
// A thread keeps the same columns for every row its team works on, so the sum over rows of dy n stays in registers until the
// end; the teams of a workgroup meet in LDS, the workgroups' partial rows are added by a second launch in a fixed order.
#include <math.h>

#include <algorithm>

#include "dfhip_internal.h"

using namespace dfhip;

namespace {

constexpr int kThreads = 256;

template <int V> struct Vec;
template <> struct Vec<4> { typedef float4 type; };
template <> struct Vec<1> { typedef float type; };

template <int V>
__device__ __forceinline__ void vload(float* v, const float* p) {
  if (V == 4) { const float4 t = *reinterpret_cast<const float4*>(p); v[0] = t.x; v[1 % V] = t.y; v[2 % V] = t.z; v[3 % V] = t.w; }
  else v[0] = p[0];
}
template <int V>
__device__ __forceinline__ void vstore(float* p, const float* v) {
  if (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1 % V], v[2 % V], v[3 % V]);
  else p[0] = v[0];
}

// the sum over the T threads of a team, in every one of them (T <= 64: lanes of one wave; T == kThreads: the workgroup)
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
    for (int w = 1; w < kThreads / 64; w++) v += sh[w];
  }
  return v;
}

// U trips of V elements a thread cover the row: T * U * V >= width
template <int T, int U, int V, bool RES>
__global__ __launch_bounds__(kThreads) void k_rms_fwd(const float* __restrict__ x, const float* res,
                                                      const float* __restrict__ w, float* __restrict__ y, float* h,
                                                      float* __restrict__ rstd, int64_t rows, int width, float eps) {
  __shared__ double sh[kThreads / 64];
  const int team = threadIdx.x / T, lane = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / T) + team;
  const bool live = row < rows;                    // (a team whose row does not exist keeps the others company at barriers)
  const int64_t base = (live ? row : 0) * width;
  float v[U][V];
  double ss = 0.0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * V;
    if (c < width) vload<V>(v[u], x + base + c);
    else
#pragma unroll
      for (int e = 0; e < V; e++) v[u][e] = 0.0f;
  }
  if (RES) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * V;
      if (c < width) {
        float r[V];
        vload<V>(r, res + base + c);
#pragma unroll
        for (int e = 0; e < V; e++) v[u][e] += r[e];
        if (live) vstore<V>(h + base + c, v[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < V; e++) ss = fma((double)v[u][e], (double)v[u][e], ss);
  ss = team_sum<T>(ss, sh);
  const float r = (float)(1.0 / sqrt(ss / (double)width + (double)eps));
  if (!live) return;
  if (rstd && lane == 0) rstd[row] = r;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * V;
    if (c < width) {
      float o[V], wv[V];
      if (w) vload<V>(wv, w + c);
#pragma unroll
      for (int e = 0; e < V; e++) o[e] = w ? v[u][e] * r * wv[e] : v[u][e] * r;
      vstore<V>(y + base + c, o);
    }
  }
}

// rows wider than the registers hold: the row twice
template <int V, bool RES>
__global__ __launch_bounds__(kThreads) void k_rms_fwd_wide(const float* x, const float* res, const float* __restrict__ w,
                                                           float* __restrict__ y, float* h, float* __restrict__ rstd,
                                                           int64_t width, float eps) {
  __shared__ double sh[kThreads / 64];
  const int64_t base = (int64_t)blockIdx.x * width;
  double ss = 0.0;
  for (int64_t c = (int64_t)threadIdx.x * V; c < width; c += kThreads * V) {
    float v[V];
    vload<V>(v, x + base + c);
    if (RES) {
      float r[V];
      vload<V>(r, res + base + c);
#pragma unroll
      for (int e = 0; e < V; e++) v[e] += r[e];
      vstore<V>(h + base + c, v);
    }
#pragma unroll
    for (int e = 0; e < V; e++) ss = fma((double)v[e], (double)v[e], ss);
  }
  ss = team_sum<kThreads>(ss, sh);
  const float r = (float)(1.0 / sqrt(ss / (double)width + (double)eps));
  if (rstd && threadIdx.x == 0) rstd[blockIdx.x] = r;
  const float* s = RES ? h : x;                    // (each thread reads back what it wrote itself)
  for (int64_t c = (int64_t)threadIdx.x * V; c < width; c += kThreads * V) {
    float v[V], wv[V];
    vload<V>(v, s + base + c);
    if (w) vload<V>(wv, w + c);
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = w ? v[e] * r * wv[e] : v[e] * r;
    vstore<V>(y + base + c, v);
  }
}

// partial: gridDim.x rows of `width` sums of dy n, or NULL
template <int T, int U, int V>
__global__ __launch_bounds__(kThreads) void k_rms_bwd(const float* __restrict__ dy, const float* __restrict__ h,
                                                      const float* __restrict__ rstd, const float* __restrict__ w,
                                                      const float* add, float* dx, float* __restrict__ partial, int64_t rows,
                                                      int width) {
  __shared__ float sh[kThreads / 64];
  constexpr int TEAMS = kThreads / T;
  __shared__ float meet[TEAMS > 1 ? T * U * V * TEAMS : 1];
  const int team = threadIdx.x / T, lane = threadIdx.x % T;
  float sum[U][V];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < V; e++) sum[u][e] = 0.0f;
  float wv[U][V];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (u * T + lane) * V;
#pragma unroll
    for (int e = 0; e < V; e++) wv[u][e] = 1.0f;
    if (w && c < width) vload<V>(wv[u], w + c);
  }
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  // (the trip count is the workgroup's, so that every thread reaches the barriers of a four-wave team)
  for (int64_t row0 = (int64_t)blockIdx.x * TEAMS; row0 < rows; row0 += step) {
    const bool live = row0 + team < rows;
    const int64_t row = live ? row0 + team : row0;
    const int64_t base = row * width;
    const float r = rstd[row];
    float g[U][V], n[U][V];
    float dot = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * V;
      if (c < width) {
        vload<V>(g[u], dy + base + c);
        vload<V>(n[u], h + base + c);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) g[u][e] = n[u][e] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < V; e++) {
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
        const int c = (u * T + lane) * V;
        if (c < width) {
          float o[V];
#pragma unroll
          for (int e = 0; e < V; e++) o[e] = r * (g[u][e] - n[u][e] * c1);
          if (add) {
            float a[V];
            vload<V>(a, add + base + c);
#pragma unroll
            for (int e = 0; e < V; e++) o[e] += a[e];
          }
          vstore<V>(dx + base + c, o);
        }
      }
  }
  if (!partial) return;
  float* prow = partial + (int64_t)blockIdx.x * width;
  if (TEAMS == 1) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = (u * T + lane) * V;
      if (c < width)
#pragma unroll
        for (int e = 0; e < V; e++) prow[c + e] = sum[u][e];
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < V; e++) meet[team * (T * U * V) + (u * T + lane) * V + e] = sum[u][e];
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += kThreads) {
    float s = 0.0f;
#pragma unroll
    for (int t = 0; t < TEAMS; t++) s += meet[t * (T * U * V) + c];
    prow[c] = s;
  }
}

// rows wider than the registers hold: dx alone, a workgroup a row
template <int V>
__global__ __launch_bounds__(kThreads) void k_rms_bwd_wide(const float* __restrict__ dy, const float* __restrict__ h,
                                                           const float* __restrict__ rstd, const float* __restrict__ w,
                                                           const float* add, float* dx, int64_t width) {
  __shared__ float sh[kThreads / 64];
  const int64_t base = (int64_t)blockIdx.x * width;
  const float r = rstd[blockIdx.x];
  float dot = 0.0f;
  for (int64_t c = (int64_t)threadIdx.x * V; c < width; c += kThreads * V) {
    float g[V], n[V], wv[V];
    vload<V>(g, dy + base + c);
    vload<V>(n, h + base + c);
    if (w) vload<V>(wv, w + c);
#pragma unroll
    for (int e = 0; e < V; e++) dot = fmaf(w ? g[e] * wv[e] : g[e], n[e] * r, dot);
  }
  const float c1 = team_sum<kThreads>(dot, sh) * (1.0f / (float)width);
  for (int64_t c = (int64_t)threadIdx.x * V; c < width; c += kThreads * V) {
    float g[V], n[V], wv[V], a[V];
    vload<V>(g, dy + base + c);
    vload<V>(n, h + base + c);
    if (w) vload<V>(wv, w + c);
    if (add) vload<V>(a, add + base + c);
#pragma unroll
    for (int e = 0; e < V; e++) {
      float o = r * ((w ? g[e] * wv[e] : g[e]) - n[e] * r * c1);
      if (add) o += a[e];
      g[e] = o;
    }
    vstore<V>(dx + base + c, g);
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

// dw[c] = sum over the partial rows, in the order of the rows within 16 groups and then of the groups; 64 columns a workgroup
__global__ __launch_bounds__(1024) void k_rms_dw_sum(const float* __restrict__ partial, float* __restrict__ dw, int n_partial,
                                                     int64_t width) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
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

template <int T, int U, int V>
int fwd(const float* x, const float* res, const float* w, float* y, float* h, float* rstd, int64_t rows, int64_t width, float eps) {
  const dim3 grid((unsigned)df_ceil_div(rows, kThreads / T));
  if (res) DF_LAUNCH((k_rms_fwd<T, U, V, true>), grid, dim3(kThreads), 0, stream(), x, res, w, y, h, rstd, rows, (int)width, eps);
  else DF_LAUNCH((k_rms_fwd<T, U, V, false>), grid, dim3(kThreads), 0, stream(), x, res, w, y, h, rstd, rows, (int)width, eps);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

template <int T, int U, int V>
int bwd(const float* dy, const float* h, const float* rstd, const float* w, const float* add, float* dx, float* partial,
        int blocks, int64_t rows, int64_t width) {
  DF_LAUNCH((k_rms_bwd<T, U, V>), dim3(blocks), dim3(kThreads), 0, stream(), dy, h, rstd, w, add, dx, partial, rows, (int)width);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

// the team of a row of `width` elements, V elements a load: f(T, U) of the narrowest form that holds it
#define RMS_FORMS(V, CALL)                                                   \
  do {                                                                       \
    const int64_t per = (width + V - 1) / V;                                 \
    if (per <= 16 * (8 / V)) return CALL(16, 8 / V, V);                      \
    if (per <= 32 * (16 / V)) return CALL(32, 16 / V, V);                    \
    if (per <= 64 * (16 / V)) return CALL(64, 16 / V, V);                    \
    if (per <= 256 * (8 / V)) return CALL(256, 8 / V, V);                    \
    if (per <= 256 * (16 / V)) return CALL(256, 16 / V, V);                  \
    if (per <= 256 * (32 / V)) return CALL(256, 32 / V, V);                  \
    if (per <= 256 * (64 / V)) return CALL(256, 64 / V, V);                  \
  } while (0)

template <int V>
int run_fwd(const float* x, const float* res, const float* w, float* y, float* h, float* rstd, int64_t rows, int64_t width,
            float eps) {
#define CALL(T, U, V) fwd<T, U, V>(x, res, w, y, h, rstd, rows, width, eps)
  RMS_FORMS(V, CALL);
#undef CALL
  if (res) DF_LAUNCH((k_rms_fwd_wide<V, true>), dim3((unsigned)rows), dim3(kThreads), 0, stream(), x, res, w, y, h, rstd, width, eps);
  else DF_LAUNCH((k_rms_fwd_wide<V, false>), dim3((unsigned)rows), dim3(kThreads), 0, stream(), x, res, w, y, h, rstd, width, eps);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

template <int V>
int run_bwd(const float* dy, const float* h, const float* rstd, const float* w, const float* add, float* dx, float* partial,
            int blocks, int64_t rows, int64_t width) {
#define CALL(T, U, V) bwd<T, U, V>(dy, h, rstd, w, add, dx, partial, blocks, rows, width)
  RMS_FORMS(V, CALL);
#undef CALL
  if (dx) {
    DF_LAUNCH(k_rms_bwd_wide<V>, dim3((unsigned)rows), dim3(kThreads), 0, stream(), dy, h, rstd, w, add, dx, width);
    DF_LAUNCH_CHECK();
  }
  if (partial) {
    DF_LAUNCH(k_rms_dw_wide, dim3((unsigned)df_ceil_div(width, kThreads), (unsigned)blocks), dim3(kThreads), 0, stream(), dy, h,
              rstd, partial, rows, width);
    DF_LAUNCH_CHECK();
  }
  return DFHIP_OK;
}

bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t a = 0;
  for (const void* p : ps) a |= (uintptr_t)p;
  return (a & 15) == 0;
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
  const bool vec = width % 4 == 0 && aligned16({x, residual, weight, y, residual ? h : nullptr});
  return vec ? run_fwd<4>(x, residual, weight, y, h, rstd, rows, width, eps)
             : run_fwd<1>(x, residual, weight, y, h, rstd, rows, width, eps);
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
  // workgroups that share the rows: two a CU, as many partial rows as workgroups
  const int64_t teams = width <= 128 ? 16 : width <= 512 ? 8 : width <= 1024 ? 4 : 1;
  const int blocks = (int)std::min<int64_t>(df_ceil_div(rows, teams), 2 * num_cus());
  float* partial = nullptr;
  if (dweight) {
    partial = workspace((size_t)blocks * (size_t)width * sizeof(float));
    if (!partial) return DFHIP_OUT_OF_MEMORY;
  }
  const bool vec = width % 4 == 0 && aligned16({dy, h, weight, add, dx});
  st = vec ? run_bwd<4>(dy, h, rstd, weight, add, dx, partial, blocks, rows, width)
           : run_bwd<1>(dy, h, rstd, weight, add, dx, partial, blocks, rows, width);
  if (st != DFHIP_OK || !dweight) return st;
  DF_LAUNCH(k_rms_dw_sum, dim3((unsigned)df_ceil_div(width, 64)), dim3(1024), 0, stream(), partial, dweight, blocks, width);
  DF_LAUNCH_CHECK();
  return DFHIP_OK;
}

}  // extern "C"

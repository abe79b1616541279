// fp32 products of FEW rows (at most 64 a workgroup) with a large matrix W on the fp32 matrix cores.
//
// What bounds them is reading W, or writing a gradient of its size: 32 rows are 64 operations for the 4 bytes of an element, and
// the fp32 matrix cores form 121 in the time that HBM takes for them (153 TFLOP/s, 5.07 TB/s).  So W is read as it is, once a
// product, into the matrix operands: the split products (dfhip_splitgemm.h) read and write it to convert it and read it again, 12
// bytes an element instead of 4 (16 where they read all of it for its scale).
//
// 32 x 32 x 2 MFMA; the order of the reduction is free, so a lane's operands are 16-byte pieces of memory:
//   rows' side       lane (i, h): four elements of row i from k + 4 h: element s belongs to product s, which takes k + s and k + 4 + s
//   W across (K is the row of the storage; x W):     load s: row k + 4 h + s, columns CF i .. CF i + CF - 1, one for each fragment
//   W along  (K runs along the storage; dl W^T):     row i of the storage, elements k + 4 h .. + 3: turned in LDS, see `along`
// A step is eight k.
// Measured: x W of 1 x 2048 x 99991 193 us, of 32 x 1024 x 50001 49 us (4.2 TB/s of W); dl W^T and x^T dl as one launch 367 and 112 us
// (4.5 and 3.7 TB/s of W and dW).
#pragma once
#include "dfhip_internal.h"

namespace dfhip_few {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));      // rows of any width begin on any element
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMost = 64;                          // rows a workgroup; of the gradients, rows in all

// rows x n outputs over kn; `a` (rows, lda), `b` (kn, ldb), along: (n, ldb)
struct Product {
  const float *a, *b;
  int64_t lda, ldb;
  int rows, n, kn;
};

template <int N> struct Vec;
template <> struct Vec<1> { typedef float type; };
template <> struct Vec<2> { typedef float type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct Vec<4> { typedef f32x4u type; };

template <int RB, int CF>
struct Step {
  f32x4 a[RB];
  float b[4][CF];                                  // (product, fragment)
};

// RB blocks of 32 rows, a tile of 32 CF columns from n0 for a workgroup, whose waves divide K; their tiles are joined through LDS.
// `sink(row, v)` gets the joined tile, CF values a lane.
template <int RB, int CF, int NW, class F>
__device__ __forceinline__ void across(const Product& p, int n0, f32x4* lds, F sink) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  f32x16 acc[RB][CF];
#pragma unroll
  for (int rb = 0; rb < RB; rb++)
#pragma unroll
    for (int f = 0; f < CF; f++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[rb][f][r] = 0.0f;
  const float* pa[RB];
#pragma unroll
  for (int rb = 0; rb < RB; rb++) pa[rb] = p.a + (int64_t)min(rb * 32 + i, p.rows - 1) * p.lda + 4 * h;
  // (a lane whose columns pass the last one reads the last ones; the caller puts that right)
  const float* pb = p.b + (int64_t)(4 * h) * p.ldb + min(n0 + CF * i, p.n - CF);
  typedef Step<RB, CF> S;
  auto load = [&](S& q, int k) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
      typedef typename Vec<CF>::type V;
      union { V v; float f[CF]; } u;
      u.v = *reinterpret_cast<const V*>(pb + (int64_t)(k + s) * p.ldb);
#pragma unroll
      for (int f = 0; f < CF; f++) q.b[s][f] = u.f[f];
    }
#pragma unroll
    for (int rb = 0; rb < RB; rb++) q.a[rb] = *reinterpret_cast<const f32x4u*>(pa[rb] + k);
  };
  auto load_end = [&](S& q, int k) {               // a step that passes the end of K: zeros there
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const bool in = k + 4 * h + s < p.kn;
#pragma unroll
      for (int rb = 0; rb < RB; rb++) q.a[rb][s] = in ? pa[rb][k + s] : 0.0f;
#pragma unroll
      for (int f = 0; f < CF; f++) q.b[s][f] = in ? pb[(int64_t)(k + s) * p.ldb + f] : 0.0f;
    }
  };
  auto multiply = [&](const S& q) {
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int rb = 0; rb < RB; rb++)
#pragma unroll
        for (int f = 0; f < CF; f++)
          acc[rb][f] = __builtin_amdgcn_mfma_f32_32x32x2f32(q.a[rb][s], q.b[s][f], acc[rb][f], 0, 0, 0);
  };
  const int steps = (p.kn + 7) / 8, per = (steps + NW - 1) / NW;
  const int first = 8 * min(wave * per, steps), last = 8 * min((wave + 1) * per, steps);
  const int full = (min(last, p.kn) - first) / 8;  // whole steps of this wave; a part of one may follow them
  constexpr int G = 2;                             // steps in flight under as many others
  int t = 0;
  if (full >= G) {
    S q[G], r[G];
#pragma unroll
    for (int j = 0; j < G; j++) load(q[j], first + 8 * j);
    for (; t + G <= full; t += G) {                // (behind the last group: some group again)
      const int k = first + 8 * min(t + G, full - G);
#pragma unroll
      for (int j = 0; j < G; j++) load(r[j], k + 8 * j);
      __builtin_amdgcn_sched_barrier(0);           // (the compiler would move the loads down to their use)
#pragma unroll
      for (int j = 0; j < G; j++) multiply(q[j]);
#pragma unroll
      for (int j = 0; j < G; j++) q[j] = r[j];
    }
  }
  for (; t < full; t++) {
    S q;
    load(q, first + 8 * t);
    multiply(q);
  }
  if (first + 8 * full < min(last, p.kn)) {
    S q;
    load_end(q, first + 8 * full);
    multiply(q);
  }
  // joined: element e of piece q is, in lane (i, h), fragment e % CF of row 8 (r >> 2) + 4 h + (r & 3), r = (4 q + e) / CF
  constexpr int Q = 4 * CF;
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    if (rb) __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; q++) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = acc[rb][e % CF][(4 * q + e) / CF];
      lds[(wave * Q + q) * 64 + lane] = v;
    }
    __syncthreads();
    for (int q = wave; q < Q; q += NW) {
      f32x4 v = lds[q * 64 + lane];
#pragma unroll
      for (int w = 1; w < NW; w++) v += lds[(w * Q + q) * 64 + lane];
#pragma unroll
      for (int j = 0; j < 4 / CF; j++) {
        const int r = q * (4 / CF) + j;
        float o[CF];
#pragma unroll
        for (int f = 0; f < CF; f++) o[f] = v[j * CF + f];
        sink(rb * 32 + 8 * (r >> 2) + 4 * h + (r & 3), o);
      }
    }
  }
}
template <int CF, int NW> constexpr int lds_pieces() { return NW * 4 * CF * 64; }

// A wave's 32 columns of the product with W along (column d is row d of the storage), over the classes [k0, k1): `parts` (rows, n).
// A fragment's lane needs 16 bytes of each of 32 rows of the storage; read like that, every load touches 32 lines, and the lines
// that a chip full of such waves holds open do not fit the L2 (1 x 1024 x 50001: 76 us, 1 x 2048 x 99991: 268; with half as many
// rows a wave 50 and 223, but the rows' side is read more often: 32 rows 343; like this 51, 197, 32 rows 245).  So a wave reads 32 x 64 windows, 256 bytes a row, and turns them
// in LDS of its own (rows 272 bytes apart: sixteen lanes touch every bank once).  All waves of a workgroup go through the same
// classes: the rows' side, (rows, lda) with zeros up to a multiple of 64 classes, comes out of the L1 for three of four.
constexpr int kWindow = 64, kPitch = kWindow + 4;
template <int RB>
__device__ __forceinline__ void along(const Product& p, int n0, int k0, int k1, float* __restrict__ lds, float* __restrict__ parts) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  n0 += wave * 32;
  if (n0 >= p.n) return;
  float* own = lds + wave * 32 * kPitch;
  const int r4 = lane >> 4, c4 = (lane & 15) * 4;
  const float* pb[8];
#pragma unroll
  for (int j = 0; j < 8; j++) pb[j] = p.b + (int64_t)min(n0 + 4 * j + r4, p.n - 1) * p.ldb + c4;
  const float* pa[RB];
#pragma unroll
  for (int rb = 0; rb < RB; rb++) pa[rb] = p.a + (int64_t)min(rb * 32 + i, p.rows - 1) * p.lda + 4 * h;
  f32x4 st[8];
  auto load = [&](int k) {
    if (k + kWindow <= p.kn) {
#pragma unroll
      for (int j = 0; j < 8; j++) st[j] = *reinterpret_cast<const f32x4u*>(pb[j] + k);
    } else {                                       // (zeros behind the last class)
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) st[j][e] = k + c4 + e < p.kn ? pb[j][k + e] : 0.0f;
    }
  };
  f32x16 acc[RB];
#pragma unroll
  for (int rb = 0; rb < RB; rb++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[rb][r] = 0.0f;
  load(k0);
  for (int k = k0; k < k1; k += kWindow) {
#pragma unroll
    for (int j = 0; j < 8; j++) *reinterpret_cast<f32x4*>(own + (4 * j + r4) * kPitch + c4) = st[j];
    if (k + kWindow < k1) load(k + kWindow);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < kWindow / 8; t++) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(own + i * kPitch + 8 * t + 4 * h);
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(pa[rb] + k + 8 * t);
#pragma unroll
        for (int s = 0; s < 4; s++) acc[rb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], acc[rb], 0, 0, 0);
      }
    }
    __builtin_amdgcn_wave_barrier();               // (this window's reads stay in front of the next one's writes)
  }
  if (n0 + i >= p.n) return;
#pragma unroll
  for (int rb = 0; rb < RB; rb++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = rb * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
      if (row < p.rows) parts[(int64_t)row * p.n + n0 + i] = acc[rb][r];
    }
}

// dw (width, classes) = x^T dl for rows [d0, d1) of it and the 32 CF columns from n0 of one wave, db their sums where it is not
// NULL.  dl stays in registers: lane (i, h) holds columns CF i .. CF i + CF - 1 of rows 2 s + h.  `counted`: bit n says whether
// row n takes part (the others of x may hold anything, those behind the last one are not there).
template <int KN, int CF>
__device__ __forceinline__ void outer(const float* __restrict__ x, int rows, int width, const float* __restrict__ dl, int64_t ld,
                                      float* __restrict__ dw, float* __restrict__ db, int classes, int n0, int d0, int d1,
                                      uint64_t counted) {
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  constexpr int S = KN / 2, C = S < 16 ? S : 16;
  typedef typename Vec<CF>::type V;
  union Piece { V v; float f[CF]; };
  float b[S][CF];
  const int c = n0 + CF * i;
#pragma unroll
  for (int s = 0; s < S; s++) {
    const int n = 2 * s + h;
    Piece u;
    u.v = *reinterpret_cast<const V*>(dl + (int64_t)min(n, rows - 1) * ld + c);
#pragma unroll
    for (int f = 0; f < CF; f++) b[s][f] = n < rows ? u.f[f] : 0.0f;
  }
  if (db) {
#pragma unroll
    for (int f = 0; f < CF; f++) {
      float t = b[0][f];
#pragma unroll
      for (int s = 1; s < S; s++) t += b[s][f];
      t += __shfl_xor(t, 32);
      if (h == 0 && c + f < classes) db[c + f] = t;
    }
  }
  if (!dw) return;
  counted >>= h;
  const unsigned words[2] = {(unsigned)counted, (unsigned)(counted >> 32)};
  for (int d = d0; d < d1; d += 32) {
    // (the rows' addresses are formed anew in every trip: kept from one to the next they would take as many registers as dl)
    int last = rows - 1;
    asm volatile("" : "+s"(last));
    const unsigned even = (unsigned)min(d + i, width - 1), odd = even + (unsigned)(h * width);
    f32x16 acc[CF];
#pragma unroll
    for (int f = 0; f < CF; f++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[f][r] = 0.0f;
    float a[2][C];
    auto load = [&](int j) {
#pragma unroll
      for (int s = 0; s < C; s++) {
        const int n = 2 * (j * C + s);
        a[j & 1][s] = (x + (int64_t)min(n, last) * width)[n < last ? odd : even];
      }
    };
    load(0);
#pragma unroll
    for (int j = 0; j < S / C; j++) {
      if (j + 1 < S / C) load(j + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < C; s++) {
        const int at = j * C + s, keep = __builtin_amdgcn_sbfe((int)words[at / 16], 2 * (at % 16), 1);     // all ones, or 0
        const float v = __int_as_float(__float_as_int(a[j & 1][s]) & keep);
#pragma unroll
        for (int f = 0; f < CF; f++) acc[f] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, b[at][f], acc[f], 0, 0, 0);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = d + 8 * (r >> 2) + 4 * h + (r & 3);
      if (row >= width) continue;
      float* out = dw + (int64_t)row * classes + c;
      if (c + CF <= classes) {
        Piece u;
#pragma unroll
        for (int f = 0; f < CF; f++) u.f[f] = acc[f][r];
        *reinterpret_cast<V*>(out) = u.v;
      } else {
#pragma unroll
        for (int f = 0; f < CF; f++)
          if (c + f < classes) out[f] = acc[f][r];
      }
    }
  }
}

}  // namespace dfhip_few

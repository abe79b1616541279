// fp32 products on the fp16 matrix cores: every operand is held as TWO fp16 values that carry 23 bits of it, and a product is formed
// from three of the four partial products, accumulated in fp32.
//
//   v 2^-e = hi + 2^-11 lo,  hi = fp16(v 2^-e),  lo = fp16(2^11 (v 2^-e - hi)):  |error| <= 2^-23 |v|, with a floor of 2^-49 of the
//   array's largest magnitude A, for e such that A 2^-e lies in [2^13, 2^14): lo is a normal number wherever hi is one, down to
//   2^-28 A, and keeps what a hi below that cannot hold.  (Unscaled, lo would leave the normal numbers at 2^-17 A, and elements
//   below 2^-39 A would vanish: the gradient of a class that is hardly ever likely, beside those of the others.)
//   a b = hi hi' + 2^-11 (hi lo' + lo hi')  (+ 2^-22 lo lo' <= 2^-22 |a b|, left out)
// The two sums are two sets of accumulators, joined at the end.
// (The scheme is published: Ootomo and Yokota, "Recovering single precision accuracy from Tensor Cores while surpassing the FP32
// theoretical peak performance", 2022.)  Against fp32 MFMA (157 TFLOP/s) the fp16 rate is 16 times as high, a third of it is left:
// measured error and time beside the caller, dfhip_vocab.hip.
//
// STORAGE ("split array"): a padded row-major array of 4-byte cells, columns in blocks of 32: 128 bytes that hold the block's 32
// hi halves, then its 32 lo halves.  A cell takes as much room as the fp32 value it stands for, so an fp32 array can be converted
// in place block by block, and ONE copy of an array serves as either operand of a product:
//   the reduction runs along the rows of the storage ("K along"): a tile is 128-byte pieces of BM (BN) rows, read as 16-byte fragments;
//   the reduction runs across them ("K across"): a tile is 32 rows of 4 BM (BN) bytes, read with the transposing LDS loads
//   (ds_read_b64_tr_b16: 16 lanes hand in 4 rows x 16 halves, each lane receives the 4 rows of its column).
//
// KERNEL: workgroup tile BM x BN, K step 32, LDS buffers filled by 16-byte global-to-LDS copies issued NS - 1 steps ahead; one
// barrier a step.  32 x 32 x 16 MFMA.  T = 256: 256 x 128 by eight waves of 64 x 64, two buffers, one workgroup a CU; T = 128:
// 128 x 128 by four waves of 64 x 64, two buffers, two workgroups a CU; T = 64: 64 x 64 by four waves of 32 x 32, four buffers (short
// reductions and few tiles wait for memory, not for the matrix cores).
// The second set of accumulators is what the tiles are small for: one set allowed 256 x 256 by waves of 128 x 64, whose operands come
// out of the LDS three quarters as often (8192 x 1024 x 50001: 6.6 ms against 7.07; the power limit sets the clock).  Those waves with
// both sets, one a SIMD (256 x 128 by four): 110 us where eight waves take 96; a third buffer: 99 (256 tiles, 64 steps).
// LDS positions are XOR-permuted at 16-byte granularity by the ROW (the copy's source address is permuted, its LDS side is linear): 16
// lanes that read the same piece of 16 rows, or 32 lanes that read 4 rows transposed, touch every bank once (SQ_LDS_BANK_CONFLICT
// reads 0).
// LDS reads: three products share two fragments a side, so the LDS moves half the bytes an fp16 GEMM of the same rate would.
#pragma once
#include <algorithm>

#include "dfhip_internal.h"

namespace dfhip_split {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTop = 13;                 // the largest magnitude of an operand is scaled into [2^13, 2^14)
constexpr float kLow = 1.0f / 2048;      // what a low half stands for
constexpr int kPad = 256;                // rows and columns of a split array are padded with zeros to a multiple of this

__host__ __device__ inline int64_t padded(int64_t n) { return (n + kPad - 1) / kPad * kPad; }

// one scaled value as hi + kLow lo; what is not finite stays in hi alone
__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  const float r = (v - (float)hi) * (1.0f / kLow);
  lo = (_Float16)(r == r ? r : 0.0f);    // (inf - inf, NaN: no low half)
}

// e^x for x <= 0: 2^(x log2(e)) with the product's rounding error and the constant's own put back to first order (|x| times
// 2^-24 otherwise), results below 2^-126 as 0.  Half the instructions of expf, whose range checks nothing here needs.
__device__ __forceinline__ float exp_of(float x) {
  constexpr double kLog2e = 1.4426950408889634;
  constexpr float hi = (float)kLog2e, lo = (float)(kLog2e - (double)(float)kLog2e);
  x = x < -200.0f ? -200.0f : x;                           // (-inf; a NaN stays one)
  const float t = x * hi, e = fmaf(x, lo, fmaf(x, hi, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, e * 0.6931471805599453f, p);
}

// over LANES (8, 16 or 32) neighbouring lanes, the result in all of them, in the vector unit
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LANES, class F>
__device__ __forceinline__ float lanes_reduce(float v, F f) {
  v = f(v, moved<0xB1>(v));                        // quad_perm 1 0 3 2
  v = f(v, moved<0x4E>(v));                        // quad_perm 2 3 0 1
  v = f(v, moved<0x141>(v));                       // row_half_mirror: the other four of eight
  if (LANES > 8) v = f(v, moved<0x140>(v));        // row_mirror: the other eight of sixteen
  if (LANES > 16) {                                // odd and even rows of sixteen: each pair's even row twice, its odd row twice
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  return v;
}
// What a row of softmax needs of LANES x N of its logits, N a lane: the largest one, the sum of exponentials from there, and (`sum`)
// the sum of l - largest times kDown, in all of the lanes.  w is -inf where there is no class (`in`).  At most 1 / kDown of them: the
// scaled sum of finite values is finite, those of classes that a bias of the type's lowest value masks among them.
constexpr float kDown = 1.0f / 128;
struct RowPart { float m, z, t; };
template <int N, int LANES>
__device__ __forceinline__ RowPart row_part(const float* w, const bool* in, bool sum) {
  static_assert(N * LANES * kDown <= 1.0f, "kDown");
  RowPart p;
  float m = w[0];
#pragma unroll
  for (int f = 1; f < N; f++) m = fmaxf(m, w[f]);
  p.m = lanes_reduce<LANES>(m, [](float a, float b) { return fmaxf(a, b); });
  const float from = p.m > -INFINITY ? p.m : 0.0f; // (all masked: z = 0)
  p.z = p.t = 0.0f;
#pragma unroll
  for (int f = 0; f < N; f++) p.z += exp_of(w[f] - from);
  const auto add = [](float a, float b) { return a + b; };
  p.z = lanes_reduce<LANES>(p.z, add);
  if (sum) {
#pragma unroll
    for (int f = 0; f < N; f++) p.t += in[f] ? (w[f] - from) * kDown : 0.0f;
    p.t = lanes_reduce<LANES>(p.t, add);
  }
  return p;
}
// ... into three arrays `stride` apart
__device__ __forceinline__ void store_part(float* at, int64_t stride, const RowPart& p) {
  at[0] = p.m;
  at[stride] = p.z;
  at[2 * stride] = p.t;
}

enum { EPI_BIAS = 0, EPI_STORE = 1, EPI_ADD = 2, EPI_STATS = 3 };

// Tiles [0, full) are formed by one workgroup each.  The `rest` tiles behind them -- what would be a last round that leaves most
// of the chip idle -- are cut along the reduction into `splits` parts of `ksteps_split` steps; their partial tiles go to `parts`
// and k_split_rest adds them up, in order, and applies the epilogue.
struct Gemm {
  const char *a, *b;                     // split arrays
  int64_t lda, ldb;                      // bytes a storage row
  int tiles_m, tiles_n, full, rest, splits;
  int ksteps, ksteps_split;              // steps of 32 along the reduction, in all and for a part
  float* c;
  int64_t ldc;
  int m, n;                              // EPI_STORE / EPI_ADD: what lies outside is not written; EPI_BIAS: columns with a bias
  const float* bias;                     // EPI_BIAS, or NULL
  const int* exp_a;                      // result = 2^(exp_a + exp_b + exp_c) * scale * accumulator; each NULL or on the device
  const int* exp_b;
  int exp_c;
  const float* scale;
  float* colsum;                         // or NULL: column sums of b (n), scaled by 2^exp_c * scale; added where EPI_ADD (b across)
  float* parts;                          // (rest * splits) x (BM * BN + BN)
  // EPI_STATS: nothing of the product (+ bias) is stored but, of each row's runs of `unit<T>()` columns, row_part's numbers in three
  // arrays of (m, units), and the targets' elements
  float* stat;
  int units, sum;
  const float* target;
  float* lt;
};
template <int T> constexpr int unit() { return T == 64 ? 32 : 64; }      // a wave's columns

// place of a tile: bands of kBand tile rows, down the band first
constexpr int kBand = 4;
__device__ __forceinline__ void place(const Gemm& g, int tile, int& tm, int& tn) {
  const int band = tile / (kBand * g.tiles_n), in = tile - band * kBand * g.tiles_n, high = min(kBand, g.tiles_m - band * kBand);
  tn = in / high;
  tm = band * kBand + in - tn * high;
}

template <int EPI>
__device__ __forceinline__ float bias_of(const Gemm& g, int64_t n) {
  return (EPI == EPI_BIAS || EPI == EPI_STATS) && g.bias && n < g.n ? g.bias[n] : 0.0f;
}
// One value of row m (c: its place) and column n.  STREAM: past the caches, where a wave's stores fill whole lines -- a round of
// 256 workgroups writes 32 MB that nothing reads soon, and the operands' lines stay (1500 x 1024 x 30011 logits written: 373 -> 355 us
// with 256 x 256 tiles).
template <int EPI, bool STREAM>
__device__ __forceinline__ void emit(const Gemm& g, int e, float sc, float bias, int64_t m, int64_t n, float* c, float v) {
  if (EPI != EPI_BIAS && (m >= g.m || n >= g.n)) return;
  v = EPI == EPI_BIAS ? ldexpf(v, e) + bias : ldexpf(v, e) * sc;
  if (EPI == EPI_ADD) *c += v;
  else if (STREAM) __builtin_nontemporal_store(v, c);
  else *c = v;
}
// EPI_STATS for one row: four columns a lane from n
template <int T>
__device__ __forceinline__ void emit_stats(const Gemm& g, int e, const float* bias, int64_t m, int64_t n, const float* v) {
  constexpr int LANES = unit<T>() / 4;
  float w[4];
  bool in[4];
#pragma unroll
  for (int f = 0; f < 4; f++) {
    in[f] = n + f < g.n;
    w[f] = in[f] ? ldexpf(v[f], e) + bias[f] : -INFINITY;
  }
  const RowPart p = row_part<4, LANES>(w, in, g.sum != 0);
  if (m >= g.m) return;
  const int64_t u = n / unit<T>();
  if ((threadIdx.x & (LANES - 1)) == 0 && u < g.units) store_part(g.stat + m * g.units + u, (int64_t)g.m * g.units, p);
  const float t = g.target[m];
#pragma unroll
  for (int f = 0; f < 4; f++)
    if (in[f] && t == (float)(int)(n + f)) g.lt[m] = w[f];
}
// EPI_STATS for a wave's TM x TN tiles from row m0 and column n0: 32 rows at a time through LDS of its own, half a row a lane -- a
// row's sums across the lanes that hold it would be twelve steps for two values, and their code, once for each of 64 rows, longer
// than the instruction cache.
template <int T, int TM, int TN>
__device__ __forceinline__ void wave_stats(const Gemm& g, int e, const float* bias, int64_t m0, int64_t n0, const f32x16 (*acc)[TN],
                                           float* own) {
  static_assert(TN * 32 == unit<T>() && TN * 32 * kDown <= 1.0f, "a run");
  constexpr int PITCH = TN * 32 + 4, HALF = TN * 16;
  const int lane = threadIdx.x & 63, i32 = lane & 31, h = lane >> 5, row = lane >> 1, c0 = (lane & 1) * HALF;
  const int64_t u = n0 / unit<T>();
  const int valid = (int)min(max((int64_t)g.n - n0 - c0, (int64_t)0), (int64_t)HALF);
  bool in[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) in[j] = n0 + j * 32 + i32 < g.n;
  float targets[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) targets[i] = g.target[min(m0 + i * 32 + row, (int64_t)g.m - 1)];
#pragma unroll 1
  for (int i = 0; i < TM; i++) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < TM; k++)
      if (i == k) {
        t = targets[k];
#pragma unroll
        for (int r = 0; r < 16; r++)
#pragma unroll
          for (int j = 0; j < TN; j++)
            own[(8 * (r >> 2) + 4 * h + (r & 3)) * PITCH + j * 32 + i32] = in[j] ? ldexpf(acc[k][j][r], e) + bias[j] : -INFINITY;
      }
    const float* p = own + row * PITCH + c0;
    float w[HALF];
#pragma unroll
    for (int c = 0; c < HALF; c += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + c);
      w[c] = v.x; w[c + 1] = v.y; w[c + 2] = v.z; w[c + 3] = v.w;
    }
    float m = w[0];
#pragma unroll
    for (int c = 1; c < HALF; c++) m = fmaxf(m, w[c]);
    m = fmaxf(m, moved<0xB1>(m));                  // (the row's other half is the neighbour)
    const float from = m > -INFINITY ? m : 0.0f;
    RowPart part = {m, 0.0f, 0.0f};
    if (g.sum) {
#pragma unroll
      for (int c = 0; c < HALF; c++) part.t += c < valid ? (w[c] - from) * kDown : 0.0f;
      part.t += moved<0xB1>(part.t);
    }
#pragma unroll
    for (int c = 0; c < HALF; c++) part.z += exp_of(w[c] - from);
    part.z += moved<0xB1>(part.z);
    const int64_t at = m0 + i * 32 + row;
    if (at < g.m) {
      if ((lane & 1) == 0 && u < g.units) store_part(g.stat + at * g.units + u, (int64_t)g.m * g.units, part);
      const float d = t - (float)(int)(n0 + c0);   // (exact: whole numbers up to 2^24; another target is refused later)
      if (d >= 0.0f && d < (float)valid) g.lt[at] = p[(int)d];
    }
  }
}
template <int EPI>
__device__ __forceinline__ void emit_colsum(const Gemm& g, float sc, int64_t n, float v) {
  if (n >= g.n) return;
  v = ldexpf(v, g.exp_c) * sc;
  g.colsum[n] = EPI == EPI_ADD ? g.colsum[n] + v : v;
}
__device__ __forceinline__ int exponent(const Gemm& g) {
  return g.exp_c + (g.exp_a ? g.exp_a[0] : 0) + (g.exp_b ? g.exp_b[0] : 0);
}

template <int BM, int NW, bool ACROSS>
struct Loader {
  static constexpr int J = BM / 8 / NW;  // 1024-byte copies a wave and step
  static constexpr int ROWS = ACROSS ? 1024 / (BM * 4) : 8;      // storage rows one of them covers
  const char* base;                      // uniform: the wave's first storage row of the next step's tile
  int64_t ld, step;
  unsigned off;                          // this lane's place in the first copy (K across: without its permutation)
  int across;                            // K across: row of the tile this lane copies from, mod 4
  __device__ __forceinline__ void init(const char* p, int64_t ld_, int64_t r0, int kstep0, int wave, int lane) {
    ld = ld_;
    if (ACROSS) {
      const int k = lane * 16 / (BM * 4);          // (0 for BM = 256)
      base = p + ((int64_t)kstep0 * 32 + wave * J * ROWS) * ld + r0 * 4;
      off = (unsigned)(k * ld) + (unsigned)(lane * 16 % (BM * 4));
      across = (wave * J * ROWS + k) & 3;
      step = 32 * ld;
    } else {
      base = p + (r0 + wave * J * ROWS) * ld + (int64_t)kstep0 * 128;
      // (row >> 1) & 7 with row = 8 (wave J + i) + (lane >> 3); J is even, so only i's parity moves it, by 4
      off = (unsigned)((lane >> 3) * ld) + (unsigned)(((lane & 7) ^ ((lane >> 4) & 7)) * 16);
      across = 0;
      step = 128;
    }
  }
  __device__ __forceinline__ void issue(char* lds, int wave) {
    static_assert(ACROSS || J % 2 == 0, "the permutation of the first copy");
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds +
                                                       (unsigned)(wave * J) * 1024u);
#pragma unroll
    for (int i = 0; i < J; i++) {
      const unsigned o = ACROSS ? off ^ (unsigned)(((across + i * ROWS) & 3) << 6) : (i & 1 ? off ^ 64u : off);
      // (written out because the compiler, which cannot tell the buffers apart, waits for the builtin's copies in front of the
      // next LDS read; there is no output register, nothing else here uses m0, and the kernel's own waits and barriers order the
      // copies)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at + i * 1024u), "v"(o),
                   "s"(base + (int64_t)i * ROWS * ld)
                   : "memory");
    }
    base += step;
  }
};

// fragments of T tiles of 32 rows (columns) from row w0 of an LDS tile of BM, for the half step kk (16 of the 32), plane 0 hi / 1 lo
template <int BM, bool ACROSS>
struct Reader {
  int off[4];
  __device__ __forceinline__ void init(int w0, int lane) {
    if (ACROSS) {
      const int k = (lane >> 5) * 8 + ((lane & 15) >> 2);
      const int x = (lane & 15) >> 2;              // k & 3
      const int q = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
#pragma unroll
      for (int par = 0; par < 2; par++)
#pragma unroll
        for (int plane = 0; plane < 2; plane++)
          off[par * 2 + plane] = k * (BM * 4) + (w0 >> 6) * 256 +
                                 (((8 * (par ^ ((w0 >> 5) & 1)) + 4 * plane + q) ^ (x << 2)) << 4) + (lane & 1) * 8;
    } else {
      const int x = ((lane & 31) >> 1) & 7;
#pragma unroll
      for (int kk = 0; kk < 2; kk++)
#pragma unroll
        for (int plane = 0; plane < 2; plane++)
          off[kk * 2 + plane] = (w0 + (lane & 31)) * 128 + (((plane * 4 + kk * 2 + (lane >> 5)) ^ x) << 4);
    }
  }
  // tile i, counted from w0 (where the reduction runs across, w0 is a multiple of 64 or there is tile 0 alone)
  __device__ __forceinline__ half8 get(const char* lds, int i, int kk, int plane) const {
    if (ACROSS) {
      const char* s = lds + off[(i & 1) * 2 + plane] + (i >> 1) * 256 + kk * 16 * (BM * 4);
      const short4v v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)s);
      const short4v v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(s + 4 * (BM * 4)));
      typedef short short8v __attribute__((ext_vector_type(8)));
      const short8v v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(half8, v);
    }
    return *reinterpret_cast<const half8*>(lds + off[kk * 2 + plane] + i * 4096);
  }
};

template <int T> struct Tile;
template <> struct Tile<256> { static constexpr int BM = 256, BN = 128, WM = 4, WN = 2, NS = 2; };
template <> struct Tile<128> { static constexpr int BM = 128, BN = 128, WM = 2, WN = 2, NS = 2; };
template <> struct Tile<64> { static constexpr int BM = 64, BN = 64, WM = 2, WN = 2, NS = 4; };
constexpr int tile_columns(int tile) { return tile == 64 ? 64 : 128; }
template <int T> constexpr int threads() { return Tile<T>::WM * Tile<T>::WN * 64; }
template <int T> constexpr int waves() { return 2; }      // a SIMD: what its registers are shared by
template <int T> constexpr int lds_bytes() { return Tile<T>::NS * (Tile<T>::BM + Tile<T>::BN) * 128; }
template <int T> constexpr int slices() { return Tile<T>::BM * Tile<T>::BN / 1024; }     // workgroups that add up a cut tile's parts
// workgroups of a product
__host__ __device__ inline int groups(const Gemm& g) { return ((g.full + 7) / 8 + (g.rest * g.splits + 7) / 8) * 8; }

template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// the order of a half step for the scheduler: its LDS reads (of the next half) spread evenly over its products
template <int K, int READS, int MULS>
__device__ __forceinline__ void spread() {
  if constexpr (K < READS) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, (K + 1) * MULS / READS - K * MULS / READS, 0);
    spread<K + 1, READS, MULS>();
  }
}

template <int T, bool AX, bool BX, int EPI>
__device__ __forceinline__ void gemm_body(const Gemm& g, const int block, char* lds) {
  constexpr int BM = Tile<T>::BM, BN = Tile<T>::BN, WM = Tile<T>::WM, WN = Tile<T>::WN, NS = Tile<T>::NS;
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128, COPIES = (BM + BN) / 8 / NW;
  static_assert((BM / WM) % 64 == 0 || TM == 1, "Reader");
  static_assert((BN / WN) % 64 == 0 || TN == 1, "Reader");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // consecutive workgroups go to the eight XCDs in turn: each XCD gets a run of consecutive tiles, and the 32 that it works on at a
  // time are 4 x 8 neighbours, which go along the reduction together and share 12 operand tiles in its L2 (a column of 32: 33; of
  // 256 x 128 tiles 2 048 rows of operands, 8 x 4 would be 2 560: 8192 x 1024 x 50001 7.16 -> 7.07 ms)
  const bool whole = block < (g.full + 7) / 8 * 8;
  const int id = whole ? block : block - (g.full + 7) / 8 * 8;
  const int total = whole ? g.full : g.rest * g.splits, per = (total + 7) >> 3;
  const int item = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || item >= total) return;
  const int z = whole ? 0 : item / g.rest, tile = whole ? item : g.full + item % g.rest;
  int tm, tn;
  place(g, tile, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int k0 = whole ? 0 : z * g.ksteps_split, steps = whole ? g.ksteps : min(g.ksteps - k0, g.ksteps_split);
  const int wm = wave / WN * (TM * 32), wn = wave % WN * (TN * 32);
  const bool sums = BX && g.colsum && tm == 0 && wm == 0;

  f32x16 acc[TM][TN], low[TM][TN];                 // hi hi', and hi lo' + lo hi'
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = low[i][j][r] = 0.0f;
  float col[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) col[j] = 0.0f;

  Loader<BM, NW, AX> la;
  Loader<BN, NW, BX> lb;
  la.init(g.a, g.lda, m0, k0, wave, lane);
  lb.init(g.b, g.ldb, n0, k0, wave, lane);
  Reader<BM, AX> ra;
  Reader<BN, BX> rb;
  ra.init(wm, lane);
  rb.init(wn, lane);

  struct Frag { half8 ah[TM], al[TM], bh[TN], bl[TN]; };
  auto read = [&](Frag& f, int stage, int kk) {
    const char* cur = lds + stage * STAGE;
#pragma unroll
    for (int j = 0; j < TN; j++) f.bh[j] = rb.get(cur + ABYTES, j, kk, 0);
#pragma unroll
    for (int i = 0; i < TM; i++) f.al[i] = ra.get(cur, i, kk, 1);
#pragma unroll
    for (int j = 0; j < TN; j++) f.bl[j] = rb.get(cur + ABYTES, j, kk, 1);
#pragma unroll
    for (int i = 0; i < TM; i++) f.ah[i] = ra.get(cur, i, kk, 0);
  };
  auto multiply = [&](const Frag& f) {
    // (the same accumulator comes up again after TM * TN products or more)
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[i], f.bh[j], low[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bl[j], low[i][j], 0, 0, 0);
  };
  auto add_columns = [&](const Frag& f) {          // (a lane holds eight rows of one column)
    if (BX && sums) {
#pragma unroll
      for (int j = 0; j < TN; j++) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) t += fmaf((float)f.bl[j][k], kLow, (float)f.bh[j][k]);
        col[j] += t;
      }
    }
  };

  // A step is two halves of 16.  While one half is multiplied the next one's fragments are read, across the step's end too: the
  // barrier stands in the MIDDLE of a step, where every wave holds the second half in registers.  Behind it the step's buffer is
  // free for the copies of step s + NS, and the first half of step s + 1, whose copies have landed, can be read.
#pragma unroll
  for (int s = 0; s < NS; s++)
    if (s < steps) {
      la.issue(lds + s * STAGE, wave);
      lb.issue(lds + s * STAGE + ABYTES, wave);
    }
  if (NS == 4 && steps >= 4) wait_copies<(NS == 4 ? 3 : 0) * COPIES>();
  else if (NS == 4 && steps == 3) wait_copies<(NS == 4 ? 2 : 0) * COPIES>();
  else if (steps >= 2) wait_copies<COPIES>();
  else wait_copies<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Frag f0, f1;
  read(f0, 0, 0);
  constexpr int READS = TM * 2 * (AX ? 2 : 1) + TN * 2 * (BX ? 2 : 1), MULS = 3 * TM * TN;
  for (int s = 0; s < steps - 1; s++) {
    read(f1, s & (NS - 1), 1);
    multiply(f0);
    spread<0, READS, MULS>();
    add_columns(f0);
    // this wave's copies of step s + 1 have landed (later ones may be under way) and its reads of step s are back
    if (NS == 4 && steps - 2 - s >= 2) wait_copies<(NS == 4 ? 2 : 0) * COPIES>();
    else if (NS == 4 && steps - 2 - s == 1) wait_copies<(NS == 4 ? 1 : 0) * COPIES>();
    else wait_copies<0>();
    static_assert(NS == 2 || NS == 4, "the waits");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + NS < steps) {
      la.issue(lds + (s & (NS - 1)) * STAGE, wave);
      lb.issue(lds + (s & (NS - 1)) * STAGE + ABYTES, wave);
    }
    read(f0, (s + 1) & (NS - 1), 0);
    multiply(f1);
    spread<0, READS, MULS>();
    add_columns(f1);
  }
  read(f1, (steps - 1) & (NS - 1), 1);
  multiply(f0);
  add_columns(f0);
  multiply(f1);
  add_columns(f1);

#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = fmaf(low[i][j][r], kLow, acc[i][j][r]);
  const int e = exponent(g);
  const float sc = g.scale ? g.scale[0] : 1.0f;
  float* part = whole ? nullptr : g.parts + (int64_t)((tile - g.full) * g.splits + z) * (BM * BN + BN);
  if (BX && sums) {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const float t = col[j] + __shfl_xor(col[j], 32);
      if (lane < 32) {
        if (whole) emit_colsum<EPI>(g, sc, n0 + wn + j * 32 + lane, t);
        else part[BM * BN + wn + j * 32 + lane] = t;
      }
    }
  }
  // (rows outermost: an address a row, the columns of a wave's tiles are constants from it)
  if (!whole) {
    float* c0 = part + (wm + 4 * (lane >> 5)) * BN + wn + (lane & 31);
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++)
#pragma unroll
        for (int j = 0; j < TN; j++) c0[(i * 32 + 8 * (r >> 2) + (r & 3)) * BN + j * 32] = acc[i][j][r];
    return;
  }
  const int64_t n = n0 + wn + (lane & 31);
  float bias[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) bias[j] = bias_of<EPI>(g, n + j * 32);
  if constexpr (EPI == EPI_STATS) {
    __syncthreads();                               // (the last step's operands have been read)
    wave_stats<T, TM, TN>(g, e, bias, m0 + wm, n0 + wn, acc, reinterpret_cast<float*>(lds) + wave * (32 * (TN * 32 + 4)));
    return;
  }
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int64_t m = m0 + wm + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
      float* c = g.c + m * g.ldc + n;
#pragma unroll
      for (int j = 0; j < TN; j++) emit<EPI, true>(g, e, sc, bias[j], m, n + j * 32, c + j * 32, acc[i][j][r]);
    }
}

template <int T, bool AX, bool BX, int EPI>
__global__ __launch_bounds__(threads<T>(), waves<T>()) void k_split_gemm(Gemm g) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  gemm_body<T, AX, BX, EPI>(g, (int)blockIdx.x, lds);
}

// the parts of the cut tiles added up: 1024 cells of one tile a workgroup, four a thread
template <int T, int EPI>
__device__ __forceinline__ void rest_body(const Gemm& g, const int block) {
  constexpr int BM = Tile<T>::BM, BN = Tile<T>::BN, SLICES = slices<T>(), CELLS = BM * BN + BN;
  const int t = block / SLICES, slice = block % SLICES, tile = g.full + t;
  int tm, tn;
  place(g, tile, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const float* part = g.parts + (int64_t)t * g.splits * CELLS;
  const int e = exponent(g);
  const float sc = g.scale ? g.scale[0] : 1.0f;
  const int cell = slice * 1024 + (int)threadIdx.x * 4;
  const float* p = part + cell;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  int z = 0;
  for (; z + 8 <= g.splits; z += 8) {              // eight loads in flight
    float4 q[8];
#pragma unroll
    for (int k = 0; k < 8; k++) q[k] = *reinterpret_cast<const float4*>(p + (int64_t)(z + k) * CELLS);
#pragma unroll
    for (int k = 0; k < 8; k++) { v[0] += q[k].x; v[1] += q[k].y; v[2] += q[k].z; v[3] += q[k].w; }
  }
  for (; z < g.splits; z++) {
    const float4 q = *reinterpret_cast<const float4*>(p + (int64_t)z * CELLS);
    v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
  }
  const int64_t n = n0 + cell % BN;
  float bias[4];
#pragma unroll
  for (int k = 0; k < 4; k++) bias[k] = bias_of<EPI>(g, n + k);
  if constexpr (EPI == EPI_STATS) {
    emit_stats<T>(g, e, bias, m0 + cell / BN, n, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; k++) emit<EPI, false>(g, e, sc, bias[k], m0 + cell / BN, n + k, g.c + (m0 + cell / BN) * g.ldc + n + k, v[k]);
  if (g.colsum && tm == 0 && slice == 0 && (int)threadIdx.x < BN) {
    const float* c = part + BM * BN + threadIdx.x;
    float s = 0.0f;
    for (int y = 0; y < g.splits; y++) s += c[(int64_t)y * CELLS];
    emit_colsum<EPI>(g, sc, n0 + threadIdx.x, s);
  }
}

template <int T, int EPI>
__global__ __launch_bounds__(256) void k_split_rest(Gemm g) { rest_body<T, EPI>(g, (int)blockIdx.x); }

// How a product of m x n outputs runs with T x T tiles: which tiles are cut, and into how many parts.
struct Plan { int tile, tiles_m, tiles_n, full, rest, splits, ksteps, ksteps_split; };

// Microseconds of `items` resident workgroups of one step each, measured (a step: 32 along the reduction): a chip full of 256 x 128
// tiles (256 workgroups) 1.4, of 128 x 128 (512) 1.42, of 64 x 64 (512) 0.49; few workgroups 1.0, 0.66 and 0.31.
inline double step_us(int tile, double items) {
  if (tile == 256) return items <= 64 ? 1.0 : 1.0 + 0.4 * (items - 64) / 192;
  const double half = items <= 256 ? items / 256 : 1.0, over = items <= 256 ? 0.0 : (items - 256) / 256;
  return tile == 128 ? 0.66 + 0.15 * half + 0.61 * over : 0.31 + 0.03 * half + 0.15 * over;
}
inline int64_t slots(int tile) { return (tile == 256 ? 1 : 2) * (int64_t)dfhip::num_cus(); }
// one launch of up to two products: their items are handed out in order, each to the workgroup slot that is free first; what is cut
// costs its share of being written and added up, and another launch
inline double cost_us(const Plan* p, int n) {
  const int tile = p[0].tile;
  const int64_t s = slots(tile);
  const double begin = tile == 256 ? 7.0 : tile == 128 ? 4.5 : 3.5;
  int64_t items = 0, parts = 0;
  for (int i = 0; i < n; i++) {
    parts += (int64_t)p[i].rest * p[i].splits;
    items += p[i].full;
  }
  items += parts;
  const double step = step_us(tile, (double)std::min(items, s));
  struct { double t; int64_t k; } free_at[32] = {{0.0, s}};        // k slots are free at t, the earliest first
  int groups = 1;
  double end = 0.0;
  for (int i = 0; i < 2 * n; i++) {
    const Plan& q = p[i / 2];
    int64_t c = i % 2 ? (int64_t)q.rest * q.splits : q.full;
    const double d = (i % 2 ? q.ksteps_split : q.ksteps) * step + begin;
    if (c >= 2 * s) {                              // whole rounds at once
      for (int k = 0; k < groups; k++) free_at[k].t += (double)(c / s - 1) * d;
      c -= (c / s - 1) * s;
    }
    while (c > 0) {
      const int64_t k = std::min(c, free_at[0].k);
      const double t = free_at[0].t + d;
      free_at[0].k -= k;
      if (free_at[0].k == 0) {
        for (int m = 1; m < groups; m++) free_at[m - 1] = free_at[m];
        groups--;
      }
      int at = groups;
      while (at > 0 && free_at[at - 1].t > t) at--;
      if (at > 0 && free_at[at - 1].t == t) free_at[at - 1].k += k;
      else if (groups == 32) free_at[31].k += k;   // (never that many: at most a few classes of items)
      else {
        for (int m = groups; m > at; m--) free_at[m] = free_at[m - 1];
        free_at[at] = {t, k};
        groups++;
      }
      end = std::max(end, t);
      c -= k;
    }
    for (int k = 0; k < groups; k++) end = std::max(end, free_at[k].t);
  }
  return end + (parts ? 5.0 + (double)parts * (tile == 256 ? 0.05 : tile == 128 ? 0.025 : 0.00625) : 0.0);
}
// the ways a product may be cut: not at all; what is left over from whole rounds; every tile
inline int ways(int tile, int64_t m, int64_t n, int steps, Plan* out) {
  const int64_t tm = (m + tile - 1) / tile, bn = tile_columns(tile), tn = (n + bn - 1) / bn, tiles = tm * tn, s = slots(tile);
  if (tiles > (1 << 24)) return 0;
  int count = 0;
  out[count++] = Plan{tile, (int)tm, (int)tn, (int)tiles, 0, 1, steps, steps};
  const int cuts[] = {2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  for (int all = 0; all < 2; all++) {
    const int64_t rest = all ? tiles : tiles % s;
    if (rest == 0 || (all && (tiles > s || rest == tiles % s))) continue;
    for (int c : cuts) {
      if (steps / c < 4 || rest * c > 2 * s) break;
      const int ks = (steps + c - 1) / c, real = (steps + ks - 1) / ks;
      out[count++] = Plan{tile, (int)tm, (int)tn, (int)(tiles - rest), (int)rest, real, steps, ks};
    }
  }
  return count;
}
constexpr int kWays = 24;

inline void apply(Gemm& g, const Plan& p, int64_t m, int64_t n) {
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.full = p.full;
  g.rest = p.rest;
  g.splits = p.splits;
  g.ksteps = p.ksteps;
  g.ksteps_split = p.ksteps_split;
  g.m = g.c || g.stat ? (int)m : 0;                // (column sums alone: nothing of the product is stored)
  g.n = (int)n;
}
inline int64_t parts_floats(const Plan& p) { return (int64_t)p.rest * p.splits * (p.tile * tile_columns(p.tile) + tile_columns(p.tile)); }

// a kernel's LDS beyond 64 KB has to be asked for once
inline int allow_lds(const void* kernel, int bytes, bool& done) {
  if (bytes > 65536 && !done) {
    DF_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done = true;
  }
  return DFHIP_OK;
}

}  // namespace dfhip_split

// Orthogonalisation of matrices by Newton-Schulz products (the Muon update).
//
//   X_0 = G / (|G|_F + eps)             G wide: n <= m (a tall one transposed)
//   A = X X^T,  B = a I + b A + c A A,  X <- B X         `steps` times
//
// Every matrix of a batch runs in the same launches, three a step.  X X^T and
// A A are symmetric: tiles on and above the diagonal are computed and stored
// twice.
//
// Precision.  The products take fp16 operands (11 bits; bf16's 8 would leave
// an error of 1e-2) and add in fp32.  Small singular values grow about 3.4
// times a step, and so does what X loses to rounding in directions without
// signal, so X_0 is two fp16 numbers, 22 bits, and the next ones an fp16 and an
// fp8 one (e4m3) for what that leaves, 15: the products take the first, the
// term a X both.  The last X that is multiplied is fp16 alone, for what it
// loses has no time to grow.  a X takes the fp16 number exactly, by a product
// of its own (ns_update_kernel): on B's diagonal a's rounding, 2^-10, is one of
// every row, and in a matrix of few directions nothing evens that out.  Off by
// so many times what rounding the result costs, for rank 1 / 4 / 64 / full:
// 768 x 2304 1.32 / 1.28 / 1.21 / 1.31, 300 x 300 1.30 / 1.27 / 1.21 / 1.35
// (X_0 in 15 bits, the last two X in 11 and a on the diagonal: 3.31 / 2.35 /
// 2.01 / 1.20, for 4 % less time).
// With up to 64 rows, where few directions share a step's rounding, X, A and
// B are two fp16 numbers each: 1.00, the rounding of the result.
// X is stored times 2^12: its entries stay under 2 and its small ones clear
// of fp16's subnormals.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include <cmath>
#include <limits>

#include "mfma_tile.h"

namespace dlx {

namespace {

constexpr int kTile = 128;            // the smaller output tile
constexpr int kDepth = 64;            // of a stage along k
constexpr float kXScale = 4096.f;
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kNsDiag = 3.4453125f;   // a, rounded to fp16
constexpr int kNormChunk = 1 << 14;   // elements of a partial norm

// k within 16 as operand B wants it next to Frags::tr: quads 0, 2, 1, 3
DLX_DEV constexpr int quad_swap(int k) {
  return (k & ~12) | ((k & 4) << 1) | ((k & 8) >> 1);
}

DLX_DEV float h2f(uint16_t h) { return to_f32<FP16>(FP16{h}); }

// What fp16 leaves of four numbers, as fp8 times 2^6, and back.  X times 2^12
// is under 2^13, so that a low part is at most 2^2 and stays inside e4m3.
constexpr float kLowScale = 64.f;

DLX_DEV uint32_t low_parts(const float* x, const uint16_t* h) {
  float d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] = (x[e] - h2f(h[e])) * kLowScale;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(d[0], d[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(d[2], d[3], w, true);
}

// The same as fp16, unscaled.
template <int N>
DLX_DEV Pack<uint16_t, N> low_halves(const float* x,
                                     const Pack<uint16_t, N>& h) {
  Pack<uint16_t, N> y;
#pragma unroll
  for (int e = 0; e < N; ++e) y.v[e] = from_f32<FP16>(x[e] - h2f(h.v[e])).v;
  return y;
}

DLX_DEV void add_low(float* x, uint32_t low, float by) {
  const f32v2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)low, false);
  const f32v2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)low, true);
  x[0] += by * a[0];
  x[1] += by * a[1];
  x[2] += by * b[0];
  x[3] += by * b[1];
}

// Rows row0.. of [., ld] into an LDS tile of DP columns from col0 on.
template <int ROWS, int DP, int NT>
DLX_DEV void stage_tile(uint16_t* lds, const uint16_t* src, long ld, int row0,
                        int col0) {
  constexpr int CH = DP / 8;
#pragma unroll
  for (int u = 0; u < ROWS * CH / NT; ++u) {
    const int f = u * NT + threadIdx.x;
    const int row = f / CH;
    const int chunk = (f % CH) ^ swizzle<DP>(row);
    copy16_to_lds(src + (row0 + row) * ld + col0 + chunk * 8, lds + f * 8);
  }
}

// V elements at a time: the matrices' size is a multiple of V.  Bound by
// memory: 24 of 1024 x 4096 in fp32, 403 MB in 90 us (4.5 TB/s).
template <typename T, int V>
__global__ __launch_bounds__(256) void ns_norm_kernel(
    const T* __restrict__ g, double* __restrict__ part, long size) {
  __shared__ double red[4];
  const T* p = g + blockIdx.y * size;
  const long i0 = (long)blockIdx.x * kNormChunk;
  const long i1 = i0 + kNormChunk < size ? i0 + kNormChunk : size;
  double s = 0;
#pragma unroll 4
  for (long i = i0 + threadIdx.x * V; i < i1; i += 256 * V) {
    float x[V];
    load_vec<T, V>(p + i, x);
#pragma unroll
    for (int e = 0; e < V; ++e) s += (double)x[e] * (double)x[e];
  }
  for (int off = kWave / 2; off; off >>= 1) s += __shfl_xor(s, off, kWave);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    part[(long)blockIdx.y * gridDim.x + blockIdx.x] =
        red[0] + red[1] + red[2] + red[3];
}

// The partial norms' sum, by all threads.
DLX_DEV double ns_sum(const double* part, int parts, double* red) {
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
  for (int off = kWave / 2; off; off >>= 1) s += __shfl_xor(s, off, kWave);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// What X_0 is of G: times 2^e first, then times f, so that neither leaves fp32
// (a norm of 1e-37 asks for 4e40).  Nothing but zeros has norm and eps of 0.
struct NsScale {
  float f;
  int e;
  DLX_DEV NsScale(double sum, double eps) {
    const double norm = sqrt(sum) + eps;
    f = (float)frexp(norm == 0.0 ? 0.0 : (double)kXScale / norm, &e);
  }
  DLX_DEV float of(float x) const { return ldexpf(x, e) * f; }
};

// G to X_0: scaled, split in two fp16 numbers, padded with zeros, a tall one
// transposed.  A block writes a 64 x 64 tile of X.  Bound by memory: the same
// 24, 403 MB read and 403 written in 135 us
// (6.0 TB/s).
template <typename T, int V>
__global__ __launch_bounds__(256) void ns_split_kernel(
    const T* __restrict__ g, const double* __restrict__ part, int parts,
    uint16_t* __restrict__ xh, uint16_t* __restrict__ xl, int rows, int cols,
    bool tall, int np, int mp, double eps) {
  __shared__ float t[64][65];
  __shared__ double red[4];
  const int b = blockIdx.z;
  const double sum = ns_sum(part + (long)b * parts, parts, red);
  const NsScale by(sum, eps);
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;   // in X
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;     // in G
  const T* gb = g + (long)b * rows * cols;
  constexpr int VR = 64 / V;                              // threads to a row
  const int x = threadIdx.x % VR * V;
#pragma unroll
  for (int r = threadIdx.x / VR; r < 64; r += 256 / VR) {
    float v[V] = {};
    if (r0 + r < rows && c0 + x < cols)
      load_vec<T, V>(gb + (long)(r0 + r) * cols + c0 + x, v);
#pragma unroll
    for (int e = 0; e < V; ++e) t[r][x + e] = by.of(v[e]);
  }
  __syncthreads();
  const int xj = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int r = threadIdx.x >> 4; r < 64; r += 16) {
    const long o = ((long)b * np + i0 + r) * mp + j0 + xj;
    Pack<uint16_t, 4> h;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = tall ? t[xj + e][r] : t[r][xj + e];
      h.v[e] = from_f32<FP16>(v[e]).v;
    }
    *reinterpret_cast<Pack<uint16_t, 4>*>(xh + o) = h;
    if (xl) *reinterpret_cast<Pack<uint16_t, 4>*>(xl + o) = low_halves(v, h);
  }
}

// Output tiles are TILE x TILE, by WM x WN waves.  A tile reads 2 TILE / 64
// bytes for every thousand operations, which 128 leaves to the L2s' rate and
// 256 does not; but 256 leaves few tiles.
template <int TILE> struct Shape;
template <> struct Shape<64> { static constexpr int WM = 2, WN = 2; };
template <> struct Shape<128> { static constexpr int WM = 2, WN = 2; };
template <> struct Shape<256> { static constexpr int WM = 2, WN = 4; };

// out = by (in in^T)              POLY false: A from X
// out = a I + b in + c (in in^T)  POLY true: B from A, columns quad-swapped;
//                                 not SPLIT: less kNsDiag I (ns_update_kernel)
// SPLIT: in and out are two fp16 numbers each (all but the product of the low
// ones is taken), and a matrix has one tile.
// Bound by the main loop where tiles fill the card: 24 of 1024 x 4096, tiles of
// 256: X X^T in 138 us (0.93 PFLOP/s of the ten tiles of sixteen), B from A in
// 56; 12 of 768 x 2304, tiles of 128: 34 and 18 us, 252 tiles on 256 CUs.
template <int TILE, bool POLY, bool SPLIT>
__global__ __launch_bounds__(Shape<TILE>::WM* Shape<TILE>::WN* kWave) void
ns_square_kernel(const uint16_t* __restrict__ in, uint16_t* __restrict__ out,
                 const uint16_t* __restrict__ in_low,
                 uint16_t* __restrict__ out_low, int np, int kp, int pairs) {
  constexpr int WM = Shape<TILE>::WM, WN = Shape<TILE>::WN;
  constexpr int NT = WM * WN * kWave, TS = TILE * kDepth;
  constexpr int FM = TILE / WM / 32, FN = TILE / WN / 32;
  constexpr int BUF = 2 * TS;                 // of one turn
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * BUF];
  const int blk = xcd_block(blockIdx.x, gridDim.x);
  const int batch = blk / pairs;
  int rest = blk - batch * pairs, bi = 0;
  const int nb = np / TILE;
  while (rest >= nb - bi) rest -= nb - bi++;
  const int bj = bi + rest;                   // bj >= bi
  const uint16_t* src = in + (long)batch * np * kp;
  uint16_t* dst = out + (long)batch * np * np;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wr = wid / WN, wc = wid % WN;

  const Frags<kDepth> fr(lds, lane);
  f32x16 acc[FM][FN] = {};
  const int nt = kp / kDepth;
  auto stage = [&](int t) {
    uint16_t* to = lds + (t & 1) * BUF;
    stage_tile<TILE, kDepth, NT>(to, src, kp, bj * TILE, t * kDepth);
    // one tile alone is multiplied by itself
    if (!SPLIT)
      stage_tile<TILE, kDepth, NT>(to + TS, src, kp, bi * TILE, t * kDepth);
    else
      stage_tile<TILE, kDepth, NT>(to + TS, in_low + (long)batch * np * kp, kp,
                                   0, t * kDepth);
  };
  stage(0);
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int la = (t & 1) * BUF, lb = SPLIT ? la : la + TS;
    if (t + 1 < nt) stage(t + 1);
#pragma unroll
    for (int st = 0; st < kDepth / 16; ++st) {
      s16x8 fa[FM], fb[FN];
#pragma unroll
      for (int u = 0; u < FM; ++u)
        fa[u] = fr.row(la + (wr * FM + u) * 32 * kDepth, st);
#pragma unroll
      for (int u = 0; u < FN; ++u)
        fb[u] = fr.row(lb + (wc * FN + u) * 32 * kDepth, st);
#pragma unroll
      for (int u = 0; u < FM; ++u)
#pragma unroll
        for (int v = 0; v < FN; ++v)
          acc[u][v] = mfma32<FP16>(fa[u], fb[v], acc[u][v]);
      if constexpr (SPLIT) {
        s16x8 ga[FM], gb[FN];
#pragma unroll
        for (int u = 0; u < FM; ++u)
          ga[u] = fr.row(la + TS + (wr * FM + u) * 32 * kDepth, st);
#pragma unroll
        for (int u = 0; u < FN; ++u)
          gb[u] = fr.row(la + TS + (wc * FN + u) * 32 * kDepth, st);
#pragma unroll
        for (int u = 0; u < FM; ++u)
#pragma unroll
          for (int v = 0; v < FN; ++v) {
            acc[u][v] = mfma32<FP16>(ga[u], fb[v], acc[u][v]);
            acc[u][v] = mfma32<FP16>(fa[u], gb[v], acc[u][v]);
          }
      }
    }
  }
  constexpr float by = POLY ? kNsC : 1.f / (kXScale * kXScale);
#pragma unroll
  for (int u = 0; u < FM; ++u)
#pragma unroll
    for (int v = 0; v < FN; ++v) {
      const int i = bi * TILE + (wc * FN + v) * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j =
            bj * TILE + (wr * FM + u) * 32 + q * 8 + (lane >> 5) * 4;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[u][v][q * 4 + e] * by;
        if (POLY) {
          const Pack<uint16_t, 4> o =
              *reinterpret_cast<const Pack<uint16_t, 4>*>(src + (long)i * np +
                                                          j);
          Pack<uint16_t, 4> l = {};
          if (SPLIT)
            l = *reinterpret_cast<const Pack<uint16_t, 4>*>(
                in_low + ((long)batch * np + i) * np + j);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] += kNsB * (SPLIT ? h2f(o.v[e]) + h2f(l.v[e]) : h2f(o.v[e])) +
                    (i == j + e ? (SPLIT ? kNsA : kNsA - kNsDiag) : 0.f);
        }
        Pack<uint16_t, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = from_f32<FP16>(x[e]).v;
        const int js = POLY ? quad_swap(j) : j;
        *reinterpret_cast<Pack<uint16_t, 4>*>(dst + (long)i * np + js) = y;
        if (SPLIT)
          *reinterpret_cast<Pack<uint16_t, 4>*>(
              out_low + ((long)batch * np + i) * np + js) = low_halves(x, y);
        if (!SPLIT && bi != bj) {
          const int is = POLY ? quad_swap(i) : i;
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[(long)(j + e) * np + is] = y.v[e];
        }
      }
    }
}

struct NsUpdate {
  const uint16_t *b, *xh;             // b: columns quad-swapped
  const void* xl;                     // X's low part: kFirst fp16, kNext fp8
  uint16_t* yh;                       // the next X, or
  uint8_t* yl;                        // (or none)
  const uint16_t *bw, *xw;            // SPLIT: the low halves
  uint16_t* yw;
  uint16_t* out;                      // the result, bf16
  int np, mp, rows, cols;
  bool tall;
};

enum { kFirst, kNext, kLast };          // steps; one alone is kLast

// B X, and a times the low part of X (the last step's X has none).
// a X takes X's fp16 part exactly: on B's diagonal a would leave every row an
// error of up to 2^-10 of its own, so what lies there is what kNsDiag leaves of
// a, and kNsDiag X is a product more with a diagonal operand, for the 64 rows
// of a wave where the walk over k passes them: 2 FM in FM FN np / 16.
// SPLIT: all but the product of the low halves (a lies on B's diagonal)
// Bound by the main loop: 24 of 1024 x 4096 in 270 us (0.76 PFLOP/s, at best
// 0.84); 12 of 768 x 2304, tiles of 128, in 62 us (0.53 PFLOP/s), and 78 where
// the result is stored transposed, in pieces of 2 bytes.
template <int TILE, int STEP, bool SPLIT>
__global__ __launch_bounds__(Shape<TILE>::WM* Shape<TILE>::WN* kWave) void
ns_update_kernel(NsUpdate a) {
  constexpr int WM = Shape<TILE>::WM, WN = Shape<TILE>::WN;
  constexpr int NT = WM * WN * kWave, TS = TILE * kDepth;
  constexpr int FM = TILE / WM / 32, FN = TILE / WN / 32;
  constexpr int BUF = (SPLIT ? 4 : 2) * TS;   // of one turn
  constexpr bool LAST = STEP == kLast;
  constexpr bool LOW8 = !SPLIT && STEP == kNext, LOW16 = !SPLIT && STEP == kFirst;
  static_assert(SPLIT || FN * 32 == kDepth, "a wave's rows are a stage of k");
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * BUF];
  const int nbi = a.np / TILE, nbj = a.mp / TILE;
  int blk = xcd_block(blockIdx.x, gridDim.x);
  const int batch = blk / (nbi * nbj);
  blk -= batch * nbi * nbj;
  const int bj = blk / nbi, bi = blk - bj * nbi;
  const uint16_t* bm = a.b + (long)batch * a.np * a.np;
  const long xo = (long)batch * a.np * a.mp;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wr = wid / WN, wc = wid % WN;

  const Frags<kDepth> fr(lds, lane);
  const Frags<TILE> fx(lds, lane, wr * FM * 32);
  f32x16 acc[FM][FN] = {};
  const int nt = a.np / kDepth;
  auto stage = [&](uint16_t* to, int t) {
    stage_tile<kDepth, TILE, NT>(to, a.xh + xo, a.mp, t * kDepth, bj * TILE);
    stage_tile<TILE, kDepth, NT>(to + TS, bm, a.np, bi * TILE, t * kDepth);
    if (SPLIT) {
      stage_tile<kDepth, TILE, NT>(to + 2 * TS, a.xw + xo, a.mp, t * kDepth,
                                   bj * TILE);
      stage_tile<TILE, kDepth, NT>(to + 3 * TS,
                                   a.bw + (long)batch * a.np * a.np, a.np,
                                   bi * TILE, t * kDepth);
    }
  };
  stage(lds, 0);
  const int own = bi * (TILE / kDepth) + wc;   // the stage of this wave's rows
  auto step = [&](int t, auto half) {
    constexpr int LX = decltype(half)::value * BUF, LB = LX + TS;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + 1 < nt) stage(lds + (BUF - LX), t + 1);
    unroll<kDepth / 16>([&](auto st) {
      s16x8 fa[FM], fb[FN];
#pragma unroll
      for (int u = 0; u < FN; ++u)
        fb[u] = fr.row(LB + (wc * FN + u) * 32 * kDepth, st);
      fx.template tr<FM, st * 16 * TILE>(fa, LX * 2);
#pragma unroll
      for (int u = 0; u < FM; ++u)
#pragma unroll
        for (int v = 0; v < FN; ++v)
          acc[u][v] = mfma32<FP16>(fa[u], fb[v], acc[u][v]);
      if constexpr (SPLIT) {
        s16x8 g[FM];
        fx.template tr<FM, st * 16 * TILE>(g, (LX + 2 * TS) * 2);
#pragma unroll
        for (int u = 0; u < FM; ++u)
#pragma unroll
          for (int v = 0; v < FN; ++v)
            acc[u][v] = mfma32<FP16>(g[u], fb[v], acc[u][v]);
#pragma unroll
        for (int v = 0; v < FN; ++v) {
          const s16x8 low = fr.row(LX + 3 * TS + (wc * FN + v) * 32 * kDepth, st);
#pragma unroll
          for (int u = 0; u < FM; ++u)
            acc[u][v] = mfma32<FP16>(fa[u], low, acc[u][v]);
        }
      }
    });
    if constexpr (!SPLIT) {
      if (t == own) {
        unroll<kDepth / 16>([&](auto st) {
          // columns 16 st.. of rows 32 (st / 2) + (lane & 31), in tr's order
          s16x8 fa[FM], d;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            d[e] = (st & 1) * 16 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3) ==
                           (lane & 31)
                       ? (short)from_f32<FP16>(kNsDiag).v
                       : (short)0;
          fx.template tr<FM, st * 16 * TILE>(fa, LX * 2);
#pragma unroll
          for (int u = 0; u < FM; ++u)
            acc[u][st / 2] = mfma32<FP16>(fa[u], d, acc[u][st / 2]);
        });
      }
    }
  };
  for (int t = 0; t < nt; t += 2) {
    step(t, std::integral_constant<int, 0>{});
    if (t + 1 < nt) step(t + 1, std::integral_constant<int, 1>{});
  }

  // Through LDS as fp32 rows of X, 32 of each column of waves a turn, so that
  // memory sees whole lines.  Chunk c of 4 in a row lies at c ^ (row & 31).
  float* img = reinterpret_cast<float*>(lds);
  uint16_t* out = LAST ? a.out + (long)batch * a.rows * a.cols : nullptr;
  constexpr int PR = TILE / 8;                 // threads to a row
  using P8 = Pack<uint16_t, 8>;
  const int cj = threadIdx.x % PR * 8;
  const int j = bj * TILE + cj;
  auto place = [&](int row, int chunk) {
    return img + row * TILE + ((chunk ^ (row & 31 & (TILE / 4 - 1))) << 2);
  };
  constexpr int ROWS = NT / PR, TURNS = WN * 32 / ROWS;
  auto row_of = [&](int n) { return threadIdx.x / PR + n * ROWS; };
  auto place_of = [&](int v, int row) {
    return xo + (long)(bi * TILE + (row / 32 * FN + v) * 32 + row % 32) * a.mp +
           j;
  };
#pragma unroll
  for (int v = 0; v < FN; ++v) {
    uint2 low[TURNS] = {};                     // on their way meanwhile
    P8 half_low[TURNS] = {};
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const long o = place_of(v, row_of(n));
      if (LOW8)
        low[n] = *reinterpret_cast<const uint2*>(
            static_cast<const uint8_t*>(a.xl) + o);
      if (LOW16)
        half_low[n] = *reinterpret_cast<const P8*>(
            static_cast<const uint16_t*>(a.xl) + o);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<F32x4*>(
            place(wc * 32 + (lane & 31),
                  ((wr * FM + u) * 32 + q * 8 + (lane >> 5) * 4) >> 2)) =
            F32x4{{acc[u][v][q * 4], acc[u][v][q * 4 + 1],
                   acc[u][v][q * 4 + 2], acc[u][v][q * 4 + 3]}};
    __syncthreads();
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const int row = row_of(n);
      const int i = bi * TILE + (row / 32 * FN + v) * 32 + row % 32;
      const long o = place_of(v, row);
      float x[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const F32x4 y =
            *reinterpret_cast<const F32x4*>(place(row, (cj >> 2) + e));
#pragma unroll
        for (int k = 0; k < 4; ++k) x[e * 4 + k] = y.v[k];
      }
      if (LOW8) {
        add_low(x, low[n].x, kNsA / kLowScale);
        add_low(x + 4, low[n].y, kNsA / kLowScale);
      }
      if (LOW16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += kNsA * h2f(half_low[n].v[e]);
      }
      if (!LAST) {
        P8 yh;
#pragma unroll
        for (int e = 0; e < 8; ++e) yh.v[e] = from_f32<FP16>(x[e]).v;
        *reinterpret_cast<P8*>(a.yh + o) = yh;
        if (SPLIT) {
          *reinterpret_cast<P8*>(a.yw + o) = low_halves(x, yh);
        } else if (a.yl) {
          *reinterpret_cast<uint2*>(a.yl + o) =
              make_uint2(low_parts(x, yh.v), low_parts(x + 4, yh.v + 4));
        }
      } else if (!a.tall) {
        P8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y.v[e] = from_f32<BF16>(x[e] * (1.f / kXScale)).v;
        uint16_t* at = out + (long)i * a.cols + j;
        if (i < a.rows) {
          if (a.cols % 8 == 0 && j < a.cols) {
            *reinterpret_cast<P8*>(at) = y;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (j + e < a.cols) at[e] = y.v[e];
          }
        }
      } else {
        // back into the image: its columns are the result's rows
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<F32x4*>(place(row, (cj >> 2) + e)) = F32x4{
              {x[e * 4], x[e * 4 + 1], x[e * 4 + 2], x[e * 4 + 3]}};
      }
    }
    if (LAST && a.tall) {
      __syncthreads();
      const int row = threadIdx.x % (WN * 32);
      const int c = bi * TILE + (row / 32 * FN + v) * 32 + row % 32;
      for (int jl = threadIdx.x / (WN * 32); jl < TILE; jl += NT / (WN * 32)) {
        const int r = bj * TILE + jl;
        if (r < a.rows && c < a.cols)
          out[(long)r * a.cols + c] =
              from_f32<BF16>(place(row, jl >> 2)[jl & 3] * (1.f / kXScale)).v;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Small matrices (up to 128 x 256): a block holds one and does every step.
// X stays in fp32 in the registers, in the layout of the update's result; its
// fp16 copy, A and B lie in LDS.  With few singular values nothing evens out
// what roundings to fp16 do to them in a step: up to 64 rows X, A and B are
// two fp16 numbers each, and all products but those of two low ones are taken
// (fp16 alone: 64 x 128 off by 1.6 times what rounding the result costs,
// 1 x 5 by up to 14; so by 1.0); up to 128 rows B alone is (1.5; 1.3).
// Bound by the waits between the three products of a step, and in the first
// two by four waves' matrix instructions.  One of 64 x 128: 22 us (fp16 alone
// 15; in seventeen launches 127), 512 of 128 x 256: 245 us (350 for
// 128 x 264, which takes the launches).
// ---------------------------------------------------------------------------

template <typename T, int NP, int MP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void ns_small_kernel(
    const T* __restrict__ g, uint16_t* __restrict__ out, int rows, int cols,
    int steps, double eps) {
  constexpr int TI = NP / 32, TJ = MP / 32;
  constexpr int MINE = (TI * TJ + WAVES - 1) / WAVES;
  constexpr int SQ = (TI * TI + WAVES - 1) / WAVES;
  // the second NP * MP of X and the second NP * NP of A and B: their low
  // parts; B lies in A's place where LDS is short
  constexpr bool ALL = NP == 64, SHARE = NP * MP > 1 << 14;
  constexpr int XS = NP * MP, AS = NP * NP;
  __shared__ __attribute__((aligned(16))) uint16_t lx[ALL ? 2 * XS : XS],
      lb[2 * AS], la_own[SHARE ? 8 : ALL ? 2 * AS : AS];
  uint16_t* la = SHARE ? lb : la_own;
  __shared__ double red[WAVES];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane >> 5;
  const bool tall = rows > cols;
  const int size = rows * cols;
  const T* gb = g + (long)blockIdx.x * size;
  uint16_t* ob = out + (long)blockIdx.x * size;

  // tile u of this wave: rows ti * 32.., columns tj * 32.. of X; register r
  // of a lane: row lane & 31, column 8 (r >> 2) + 4 half + (r & 3)
  f32x16 x[MINE];
  double sum = 0;
#pragma unroll
  for (int u = 0; u < MINE; ++u) {
    const int q = wid + u * WAVES;
    const int i = q % TI * 32 + (lane & 31), j0 = q / TI * 32 + half * 4;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = j0 + 8 * (r >> 2) + (r & 3);
      const int gr = tall ? j : i, gc = tall ? i : j;
      const bool in = q < TI * TJ && gr < rows && gc < cols;
      x[u][r] = in ? to_f32<T>(gb[gr * cols + gc]) : 0.f;
      sum += (double)x[u][r] * (double)x[u][r];
    }
  }
  for (int off = kWave / 2; off; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  if (lane == 0) red[wid] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < WAVES; ++i) sum += red[i];
  const NsScale by(sum, eps);
#pragma unroll
  for (int u = 0; u < MINE; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[u][r] = by.of(x[u][r]);

  auto put = [&](uint16_t* tile, auto dp, auto low, int row, int col,
                 const float* v) {
    constexpr int DP = decltype(dp)::value, LOW = decltype(low)::value;
    using P4 = Pack<uint16_t, 4>;
    P4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = from_f32<FP16>(v[e]).v;
    uint16_t* at = tile + tile_at<DP>(row, col >> 3) + (col & 7);
    *reinterpret_cast<P4*>(at) = y;
    if (LOW) *reinterpret_cast<P4*>(at + LOW) = low_halves(v, y);
  };
  using XW = std::integral_constant<int, MP>;
  using AW = std::integral_constant<int, NP>;
  using XL = std::integral_constant<int, ALL ? XS : 0>;
  using AL = std::integral_constant<int, ALL ? AS : 0>;
  using BL = std::integral_constant<int, AS>;
  const Frags<MP> fx(lx, lane);
  const Frags<NP> fa(la, lane), fb(lb, lane);

  for (int k = 0; k < steps; ++k) {
#pragma unroll
    for (int u = 0; u < MINE; ++u) {
      const int q = wid + u * WAVES;
      if (q >= TI * TJ) break;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float v[4] = {x[u][c * 4], x[u][c * 4 + 1], x[u][c * 4 + 2],
                            x[u][c * 4 + 3]};
        put(lx, XW{}, XL{}, q % TI * 32 + (lane & 31), q / TI * 32 + c * 8 + half * 4,
            v);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < SQ; ++u) {              // A = X X^T
      const int q = wid + u * WAVES;
      if (q >= TI * TI) break;
      const int ti = q % TI * 32, tj = q / TI * 32;
      f32x16 acc = {}, low = {};                // two chains of products
#pragma unroll
      for (int st = 0; st < MP / 16; ++st) {
        const s16x8 f = fx.row(tj * MP, st), h = fx.row(ti * MP, st);
        acc = mfma32<FP16>(f, h, acc);
        if (ALL) {
          low = mfma32<FP16>(fx.row(XS + tj * MP, st), h, low);
          low = mfma32<FP16>(f, fx.row(XS + ti * MP, st), low);
        }
      }
      if (ALL) acc += low;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = acc[c * 4 + e] * (1.f / (kXScale * kXScale));
        put(la, AW{}, AL{}, ti + (lane & 31), tj + c * 8 + half * 4, v);
      }
    }
    __syncthreads();
    f32x16 bt[SQ] = {};
#pragma unroll
    for (int u = 0; u < SQ; ++u) {              // B = b A + c A A
      const int q = wid + u * WAVES;
      if (q >= TI * TI) break;
      const int ti = q % TI * 32, tj = q / TI * 32;
      f32x16 low = {};
#pragma unroll
      for (int st = 0; st < NP / 16; ++st) {
        const s16x8 f = fa.row(tj * NP, st), h = fa.row(ti * NP, st);
        bt[u] = mfma32<FP16>(f, h, bt[u]);
        if (ALL) {
          low = mfma32<FP16>(fa.row(AS + tj * NP, st), h, low);
          low = mfma32<FP16>(f, fa.row(AS + ti * NP, st), low);
        }
      }
      if (ALL) bt[u] += low;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = ti + (lane & 31), j = tj + c * 8 + half * 4;
        const uint16_t* at = la + tile_at<NP>(i, j >> 3) + (j & 7);
        const auto o = *reinterpret_cast<const Pack<uint16_t, 4>*>(at);
        Pack<uint16_t, 4> l = {};
        if (ALL) l = *reinterpret_cast<const Pack<uint16_t, 4>*>(at + AS);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          bt[u][c * 4 + e] =
              kNsC * bt[u][c * 4 + e] +
              kNsB * (ALL ? h2f(o.v[e]) + h2f(l.v[e]) : h2f(o.v[e]));
      }
    }
    if (SHARE) __syncthreads();
#pragma unroll
    for (int u = 0; u < SQ; ++u) {
      const int q = wid + u * WAVES;
      if (q >= TI * TI) break;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float v[4] = {bt[u][c * 4], bt[u][c * 4 + 1], bt[u][c * 4 + 2],
                            bt[u][c * 4 + 3]};
        put(lb, AW{}, BL{}, q % TI * 32 + (lane & 31),
            quad_swap(q / TI * 32 + c * 8 + half * 4), v);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MINE; ++u) {            // X = a X + B X
      const int q = wid + u * WAVES;
      if (q >= TI * TJ) break;
      const Frags<MP> ft(lx, lane, q / TI * 32);
      f32x16 acc = {}, low = {};
      unroll<NP / 16>([&](auto st) {
        s16x8 f[2];
        if constexpr (ALL) ft.template tr_both<st * 16 * MP>(f, XS * 2);
        else ft.template tr<1, st * 16 * MP>(f);
        const s16x8 h = fb.row(q % TI * 32 * NP, st);
        acc = mfma32<FP16>(f[0], h, acc);
        if (ALL) low = mfma32<FP16>(f[1], h, low);
        auto& to = ALL ? low : acc;
        to = mfma32<FP16>(f[0], fb.row(AS + q % TI * 32 * NP, st), to);
      });
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[u][r] = kNsA * x[u][r] + (ALL ? acc[r] + low[r] : acc[r]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < MINE; ++u) {
    const int q = wid + u * WAVES;
    const int i = q % TI * 32 + (lane & 31), j0 = q / TI * 32 + half * 4;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = j0 + 8 * (r >> 2) + (r & 3);
      const int gr = tall ? j : i, gc = tall ? i : j;
      if (q < TI * TJ && gr < rows && gc < cols)
        ob[gr * cols + gc] = from_f32<BF16>(x[u][r] * (1.f / kXScale)).v;
    }
  }
}

template <typename T>
void launch_small(const at::Tensor& g, at::Tensor& out, int batch, int rows,
                  int cols, int steps, double eps, hipStream_t s) {
  const int n = std::min(rows, cols), m = std::max(rows, cols);
  auto go = [&](auto kernel, int waves) {
    kernel<<<batch, waves * kWave, 0, s>>>(
        static_cast<const T*>(g.data_ptr()),
        static_cast<uint16_t*>(out.data_ptr()), rows, cols, steps, eps);
  };
  // waves: so that a lane's share of X is at most 32 registers
  if (n <= 64 && m <= 64) go(ns_small_kernel<T, 64, 64, 4>, 4);
  else if (n <= 64 && m <= 128) go(ns_small_kernel<T, 64, 128, 8>, 8);
  else if (n <= 64) go(ns_small_kernel<T, 64, 256, 8>, 8);
  else if (m <= 128) go(ns_small_kernel<T, 128, 128, 16>, 16);
  else go(ns_small_kernel<T, 128, 256, 16>, 16);
}

template <typename T, int V>
void launch_start(const at::Tensor& g, double* part, int parts, uint16_t* xh,
                  uint16_t* xl, int batch, int rows, int cols, int np, int mp,
                  double eps, hipStream_t s) {
  const T* p = static_cast<const T*>(g.data_ptr());
  ns_norm_kernel<T, V><<<dim3(parts, batch), 256, 0, s>>>(p, part,
                                                          (long)rows * cols);
  const dim3 grid(mp / 64, np / 64, batch);
  ns_split_kernel<T, V><<<grid, 256, 0, s>>>(
      p, part, parts, xh, xl, rows, cols, rows > cols, np, mp, eps);
}

// ---------------------------------------------------------------------------
// What Muon does around it, for matrices of one shape that lie anywhere:
//   v <- mu v + g,  u = g + mu v (nesterov) or v         before
//   p <- (1 - decay) p - step o                          after
// Both stream each array once, bound by memory.  24 of 1024 x 4096 in bf16 with
// fp32 masters: 264 us for 1.41 GB before (5.3 TB/s), 233 us for 1.21 GB after
// (5.2 TB/s); in fp32 294 us for 1.61 GB and 185 us for 1.01 GB.
// ---------------------------------------------------------------------------

constexpr int kMuonList = 48;         // matrices a launch

template <typename T> struct MuonList {
  T* p[kMuonList];                    // gradients, or weights
  float* f[kMuonList];                // momenta, or fp32 masters (or none)
};

template <typename T, int V>
__global__ __launch_bounds__(256) void muon_momentum_kernel(
    MuonList<T> a, float* __restrict__ u, long size, float mu, bool nesterov) {
  const T* g = a.p[blockIdx.y];
  float* v = a.f[blockIdx.y];
  u += (long)blockIdx.y * size;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * V; i < size;
       i += (long)gridDim.x * 256 * V) {
    float x[V], m[V], y[V];
    load_vec<T, V>(g + i, x);
    load_vec<float, V>(v + i, m);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[e] = mu * m[e] + x[e];
      y[e] = nesterov ? x[e] + mu * m[e] : m[e];
    }
    store_vec<float, V>(v + i, m);
    store_vec<float, V>(u + i, y);
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void muon_apply_kernel(
    MuonList<T> a, const BF16* __restrict__ o, long size, float step,
    float keep) {
  T* p = a.p[blockIdx.y];
  float* master = a.f[blockIdx.y];
  o += (long)blockIdx.y * size;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * V; i < size;
       i += (long)gridDim.x * 256 * V) {
    float w[V], x[V];
    if (master) load_vec<float, V>(master + i, w);
    else load_vec<T, V>(p + i, w);
    load_vec<BF16, V>(o + i, x);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = keep * w[e] - step * x[e];
    if (master) store_vec<float, V>(master + i, w);
    store_vec<T, V>(p + i, w);
  }
}

// One launch for each 48 of the matrices; f: as many as p, or none.
template <typename T, typename Launch>
void muon_lists(at::TensorList p, at::TensorList f, long size, Launch launch) {
  for (size_t i0 = 0; i0 < p.size(); i0 += kMuonList) {
    MuonList<T> a{};
    const size_t k = std::min<size_t>(p.size() - i0, kMuonList);
    // elements at a time: what every matrix's place in its bucket allows
    int vec = size % 4 == 0 ? 4 : size % 2 == 0 ? 2 : 1;
    for (size_t i = 0; i < k; ++i) {
      a.p[i] = static_cast<T*>(p[i0 + i].data_ptr());
      a.f[i] = f.empty() ? nullptr : f[i0 + i].data_ptr<float>();
      while (reinterpret_cast<uintptr_t>(a.p[i]) % (vec * sizeof(T)) ||
             reinterpret_cast<uintptr_t>(a.f[i]) % (vec * sizeof(float)))
        vec /= 2;
    }
    const long per = 256 * vec;
    const dim3 grid((unsigned)std::min<long>((size + per - 1) / per, 512),
                    (unsigned)k);
    if (vec == 4) launch(a, grid, std::integral_constant<int, 4>{}, (long)i0);
    else if (vec == 2)
      launch(a, grid, std::integral_constant<int, 2>{}, (long)i0);
    else launch(a, grid, std::integral_constant<int, 1>{}, (long)i0);
  }
}

void muon_check(at::TensorList p, at::TensorList f, const at::Tensor& batch) {
  TORCH_CHECK(batch.dim() == 3 && batch.is_contiguous() &&
                  (size_t)batch.size(0) == p.size() &&
                  (f.empty() || f.size() == p.size()),
              "muon: as many matrices as [batch, rows, cols] holds");
  const long size = batch.size(1) * batch.size(2);
  for (const auto& t : p)
    TORCH_CHECK(t.numel() == size && t.is_contiguous() &&
                    t.scalar_type() == p[0].scalar_type() &&
                    t.device() == batch.device(),
                "muon: the matrices differ in size, type or device");
  for (const auto& t : f)
    TORCH_CHECK(t.numel() == size && t.is_contiguous() &&
                    t.scalar_type() == at::kFloat &&
                    t.device() == batch.device(),
                "muon: momenta and masters are float32, of the matrices' size");
}

}  // namespace

// v <- mu v + g; u [n, rows, cols] fp32: what is orthogonalised
void muon_momentum_impl(at::TensorList g, at::TensorList v, at::Tensor u,
                        double mu, bool nesterov) {
  if (g.empty()) return;
  TORCH_CHECK(u.scalar_type() == at::kFloat && !v.empty(),
              "muon: u is float32, and each matrix has a momentum");
  muon_check(g, v, u);
  const c10::DeviceGuard guard(u.device());
  const long size = u.size(1) * u.size(2);
  if (size == 0) return;
  const auto s = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto tag) {
    using T = decltype(tag);
    muon_lists<T>(g, v, size, [&](auto& a, dim3 grid, auto vec, long i0) {
      muon_momentum_kernel<T, decltype(vec)::value><<<grid, 256, 0, s>>>(
          a, u.data_ptr<float>() + i0 * size, size, (float)mu, nesterov);
    });
  };
  switch (g[0].scalar_type()) {
    case at::kFloat: go(float{}); break;
    case at::kBFloat16: go(BF16{}); break;
    default:
      TORCH_CHECK(false, "muon: unsupported dtype ", g[0].scalar_type());
  }
}

// p (and its fp32 master, where there is one) <- keep p - step o
void muon_apply_impl(at::TensorList p, at::TensorList master,
                     const at::Tensor& o, double step, double keep) {
  if (p.empty()) return;
  TORCH_CHECK(o.scalar_type() == at::kBFloat16, "muon: o is bfloat16");
  muon_check(p, master, o);
  const c10::DeviceGuard guard(o.device());
  const long size = o.size(1) * o.size(2);
  if (size == 0) return;
  const auto s = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto tag) {
    using T = decltype(tag);
    muon_lists<T>(p, master, size, [&](auto& a, dim3 grid, auto vec, long i0) {
      muon_apply_kernel<T, decltype(vec)::value><<<grid, 256, 0, s>>>(
          a, static_cast<const BF16*>(o.data_ptr()) + i0 * size, size,
          (float)step, (float)keep);
    });
  };
  switch (p[0].scalar_type()) {
    case at::kFloat: go(float{}); break;
    case at::kBFloat16: go(BF16{}); break;
    default:
      TORCH_CHECK(false, "muon: unsupported dtype ", p[0].scalar_type());
  }
}

// g: [batch, rows, cols] -> bf16 of the same shape
at::Tensor newton_schulz_impl(const at::Tensor& g_in, int64_t steps,
                              double eps) {
  TORCH_CHECK(g_in.dim() == 3, "newton_schulz: [batch, rows, cols] expected");
  TORCH_CHECK(steps >= 1 && steps <= 100,
              "newton_schulz: 1 to 100 steps, got ", steps);
  TORCH_CHECK(eps >= 0 && std::isfinite(eps),
              "newton_schulz: eps has to be finite and not negative");
  const c10::DeviceGuard guard(g_in.device());
  const auto g = g_in.contiguous();
  const long batch = g.size(0), rows = g.size(1), cols = g.size(2);
  auto out = at::empty(g.sizes(), g.options().dtype(at::kBFloat16));
  if (g.numel() == 0) return out;
  TORCH_CHECK(rows <= (1 << 20) && cols <= (1 << 20) && batch <= 65535,
              "newton_schulz: the matrices are too large or too many");
  // The larger tile where it pads little and its last turn of 256 CUs is
  // nearly full: at most 56 of them, or a sixth of all tiles, without one.  us
  // of five steps, all of 128 / update of 256 / square too:
  //   768 x 768      x 32 684 / 731 / 745   x 56 1095 / 1079 / 1216
  //                  x 48 904 / 900 / 1122  x 128 2489 / 2452 / 2418
  //   768 x 2304     x 8 429 / 414 / 691    x 12 546 / 592 / 853
  //   1024 x 1024    x 17 733 / 828 / 838   x 48 1857 / 1769 / 1752
  //   1024 x 4096    x 4 562 / 544 / 949    x 5 643 / 714 / 1120
  //                  x 12 1379 / 1284 / 1542  x 24 2784 / 2582 / 2504
  //   256 x 256      x 200 388 / 385 / 360
  const long lo = std::min(rows, cols), hi = std::max(rows, cols);
  auto pad = [](long x, long t) { return (x + t - 1) / t * t; };
  const long n256 = pad(lo, 256) / 256, m256 = pad(hi, 256) / 256;
  auto fills = [](long tiles) {
    const long idle = (tiles + 255) / 256 * 256 - tiles;
    return idle <= 56 || idle * 6 <= tiles;
  };
  const bool large = pad(lo, 256) * pad(hi, 256) * 8 <=
                         pad(lo, kTile) * pad(hi, kTile) * 9 &&
                     fills(batch * n256 * m256);
  const bool large_square = large && fills(batch * n256 * (n256 + 1) / 2);
  // Few singular values: nothing evens out what they lose to a step, so X, A
  // and B are two fp16 numbers each, in tiles of 64 (with the parts that more
  // rows get, 40 x 1000 is off by 2.0 times what rounding the result costs,
  // 4 x 400 by up to 2.75, 64 x 512 by 1.4, 128 x 264 by 1.25; so by 1.0; one of
  // 40 x 1000 takes 92 us, in tiles of 128 without it 132).
  const bool wide = lo <= 64;
  const long unit = large ? 256 : wide ? 64 : kTile;
  const long np = pad(lo, unit), mp = pad(hi, unit);
  TORCH_CHECK(batch * (np / 64) * (mp / 64) <=
                      std::numeric_limits<int>::max() &&
                  mp / 64 <= 65535,
              "newton_schulz: the matrices are too large or too many");
  const long parts = (rows * cols + kNormChunk - 1) / kNormChunk;

  const auto s = at::cuda::getCurrentCUDAStream();
  if (std::min(rows, cols) <= 128 && std::max(rows, cols) <= 256) {
    auto small = [&](auto tag) {
      launch_small<decltype(tag)>(g, out, (int)batch, (int)rows, (int)cols,
                                  (int)steps, eps, s);
    };
    switch (g.scalar_type()) {
      case at::kFloat: small(float{}); break;
      case at::kBFloat16: small(BF16{}); break;
      case at::kHalf: small(FP16{}); break;
      default:
        TORCH_CHECK(false, "newton_schulz: unsupported dtype ",
                    g.scalar_type());
    }
    return out;
  }

  const auto half = g.options().dtype(at::kHalf);
  auto x = at::empty({2, batch, np, mp}, half);       // X twice
  // X's low parts: two fp16 (wide); or X_0's fp16, in whose place every second
  // fp8 one follows, and the others' fp8: three bytes an element
  auto low = at::empty({wide ? 4 : 3, batch, np, mp},
                       g.options().dtype(at::kByte));
  auto sq = at::empty({wide ? 4 : 2, batch, np, np}, half);   // A, B
  auto part = at::empty({batch, parts}, g.options().dtype(at::kDouble));
  auto* px = static_cast<uint16_t*>(x.data_ptr());
  auto* pa = static_cast<uint16_t*>(sq.data_ptr());
  auto* pl = static_cast<uint8_t*>(low.data_ptr());
  auto* pw = static_cast<uint16_t*>(low.data_ptr());
  const long xs = batch * np * mp;
  const long as = batch * np * np;
  uint16_t* pb = pa + as;

  auto start = [&](auto tag) {
    using T = decltype(tag);
    // four elements at a time where rows begin on such a border
    const bool v4 = cols % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0;
    (v4 ? launch_start<T, 4> : launch_start<T, 1>)(
        g, part.data_ptr<double>(), (int)parts, px,
        wide || steps > 1 ? pw : nullptr, (int)batch, (int)rows, (int)cols,
        (int)np, (int)mp, eps, s);
  };
  switch (g.scalar_type()) {
    case at::kFloat: start(float{}); break;
    case at::kBFloat16: start(BF16{}); break;
    case at::kHalf: start(FP16{}); break;
    default:
      TORCH_CHECK(false, "newton_schulz: unsupported dtype ", g.scalar_type());
  }
  using Thin = std::integral_constant<int, 64>;
  using Small = std::integral_constant<int, 128>;
  using Large = std::integral_constant<int, 256>;
  using Yes = std::true_type;
  using No = std::false_type;
  auto square = [&](auto tile, auto poly, auto split, const uint16_t* in,
                    uint16_t* to, const uint16_t* in_low, uint16_t* to_low,
                    long depth) {
    constexpr int TILE = decltype(tile)::value;
    constexpr int NT = Shape<TILE>::WM * Shape<TILE>::WN * kWave;
    const long nb = np / TILE, pairs = nb * (nb + 1) / 2;
    ns_square_kernel<TILE, decltype(poly)::value, decltype(split)::value>
        <<<(unsigned)(batch * pairs), NT, 0, s>>>(
            in, to, in_low, to_low, (int)np, (int)depth, (int)pairs);
  };
  auto update = [&](auto tile, auto split, int step, const NsUpdate& u) {
    constexpr int TILE = decltype(tile)::value;
    constexpr int NT = Shape<TILE>::WM * Shape<TILE>::WN * kWave;
    const unsigned blocks = (unsigned)(batch * (np / TILE) * (mp / TILE));
    constexpr bool SPLIT = decltype(split)::value;
    if (step == kLast)
      ns_update_kernel<TILE, kLast, SPLIT><<<blocks, NT, 0, s>>>(u);
    else if (step == kNext)
      ns_update_kernel<TILE, kNext, SPLIT><<<blocks, NT, 0, s>>>(u);
    else                               // SPLIT: the first is like the next
      ns_update_kernel<TILE, SPLIT ? kNext : kFirst, SPLIT>
          <<<blocks, NT, 0, s>>>(u);
  };
  for (int64_t k = 0; k < steps; ++k) {
    uint16_t* cur = px + (k & 1) * xs;
    uint16_t* nxt = px + ((k + 1) & 1) * xs;
    uint16_t* cur_low = wide ? pw + (k & 1) * xs : nullptr;
    uint16_t* a_low = wide ? pa + 2 * as : nullptr;
    uint16_t* b_low = wide ? pa + 3 * as : nullptr;
    if (wide) {
      square(Thin{}, No{}, Yes{}, cur, pa, cur_low, a_low, mp);
      square(Thin{}, Yes{}, Yes{}, pa, pb, a_low, b_low, np);
    } else if (large_square) {
      square(Large{}, No{}, No{}, cur, pa, nullptr, nullptr, mp);
      square(Large{}, Yes{}, No{}, pa, pb, nullptr, nullptr, np);
    } else {
      square(Small{}, No{}, No{}, cur, pa, nullptr, nullptr, mp);
      square(Small{}, Yes{}, No{}, pa, pb, nullptr, nullptr, np);
    }
    // what the last X loses has no time to grow: it has no low part
    auto low_of = [&](int64_t i) { return pl + (i & 1) * 2 * xs; };
    const bool to_low = !wide && k + 2 < steps;
    const NsUpdate u{pb, cur, low_of(k), nxt,
                     to_low ? low_of(k + 1) : nullptr, b_low, cur_low,
                     wide ? pw + ((k + 1) & 1) * xs : nullptr,
                     static_cast<uint16_t*>(out.data_ptr()), (int)np, (int)mp,
                     (int)rows, (int)cols, rows > cols};
    const int which = k + 1 == steps ? kLast : k ? kNext : kFirst;
    if (wide) update(Thin{}, Yes{}, which, u);
    else if (large) update(Large{}, No{}, which, u);
    else update(Small{}, No{}, which, u);
  }
  return out;
}

}  // namespace dlx

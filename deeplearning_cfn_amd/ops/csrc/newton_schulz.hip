// Orthogonalisation of matrices by Newton-Schulz products (the Muon update).
//
//   X_0 = G / (|G|_F + eps)             G wide: n <= m (a tall one transposed)
//   A = X X^T,  B = b A + c A A,  X <- a X + B X         `steps` times
//
// Every matrix of a batch runs in the same launches, three a step.  X X^T and
// A A are symmetric: tiles on and above the diagonal are computed and stored
// twice.
//
// Precision.  The products take fp16 operands (11 bits; bf16's 8 would leave
// an error of 1e-2) and add in fp32.  Small singular values grow about 3.4
// times a step, and what X loses to rounding grows with them, so X is kept as
// a sum of two fp16 numbers (22 bits): the term a X takes both, the products
// the first alone.  B X's rounding lies in the directions where B is large,
// which are those that no longer grow.  Against 64 bits that leaves 4e-4 to
// 2e-3 relative (CPU model of these roundings, five spectra, sizes 64 to
// 768), next to bf16's own 1.7e-3 in the result.  X is stored times 2^12:
// its entries stay under 2 and its small ones clear of fp16's subnormals.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include <cmath>
#include <limits>

#include "mfma_tile.h"

namespace dlx {

namespace {

constexpr int kTile = 128;            // output tile, and what sizes pad to
constexpr int kDepth = 64;            // of a stage along k
constexpr float kXScale = 4096.f;
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kNormChunk = 1 << 16;   // elements of a partial norm

// k within 16 as operand B wants it next to tr_frag: quads 0, 2, 1, 3
DLX_DEV constexpr int quad_swap(int k) {
  return (k & ~12) | ((k & 4) << 1) | ((k & 8) >> 1);
}

DLX_DEV float h2f(uint16_t h) { return to_f32<FP16>(FP16{h}); }

// Rows row0.. of [., ld] into an LDS tile of DP columns from col0 on.
template <int ROWS, int DP>
DLX_DEV void stage_tile(uint16_t* lds, const uint16_t* src, long ld, int row0,
                        int col0) {
  constexpr int CH = DP / 8;
#pragma unroll
  for (int u = 0; u < ROWS * CH / 256; ++u) {
    const int f = u * 256 + threadIdx.x;
    const int row = f / CH;
    const int chunk = (f % CH) ^ (row & 7);
    copy16_to_lds(src + (row0 + row) * ld + col0 + chunk * 8, lds + f * 8);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(
    const T* __restrict__ g, double* __restrict__ part, long size) {
  __shared__ double red[4];
  const T* p = g + blockIdx.y * size;
  const long i0 = (long)blockIdx.x * kNormChunk;
  const long i1 = i0 + kNormChunk < size ? i0 + kNormChunk : size;
  double s = 0;
  for (long i = i0 + threadIdx.x; i < i1; i += 256) {
    const double x = to_f32<T>(p[i]);
    s += x * x;
  }
  for (int off = kWave / 2; off; off >>= 1) s += __shfl_xor(s, off, kWave);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    part[(long)blockIdx.y * gridDim.x + blockIdx.x] =
        red[0] + red[1] + red[2] + red[3];
}

// G to X_0: scaled, split in two, padded with zeros, a tall one transposed.
// A block writes a 64 x 64 tile of X.
template <typename T>
__global__ __launch_bounds__(256) void ns_split_kernel(
    const T* __restrict__ g, const double* __restrict__ part, int parts,
    uint16_t* __restrict__ xh, uint16_t* __restrict__ xl, int rows, int cols,
    bool tall, int np, int mp, float eps) {
  __shared__ float t[64][65];
  const int b = blockIdx.z;
  double sum = 0;
  for (int i = 0; i < parts; ++i) sum += part[(long)b * parts + i];
  const float by = (float)(kXScale / (sqrt(sum) + (double)eps));
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;   // in X
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;     // in G
  const T* gb = g + (long)b * rows * cols;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int r = y; r < 64; r += 4) {
    const bool in = r0 + r < rows && c0 + x < cols;
    t[r][x] =
        in ? to_f32<T>(gb[(long)(r0 + r) * cols + c0 + x]) * by : 0.f;
  }
  __syncthreads();
  for (int r = y; r < 64; r += 4) {
    const float v = tall ? t[x][r] : t[r][x];
    const long o = ((long)b * np + i0 + r) * mp + j0 + x;
    const uint16_t h = from_f32<FP16>(v).v;
    xh[o] = h;
    xl[o] = from_f32<FP16>(v - h2f(h)).v;
  }
}

// out = by (in in^T)              POLY false: A from X
// out = b in + c (in in^T)        POLY true: B from A, columns quad-swapped
template <bool POLY>
__global__ __launch_bounds__(256) void ns_square_kernel(
    const uint16_t* __restrict__ in, uint16_t* __restrict__ out, int np, int kp,
    int pairs) {
  constexpr int TS = kTile * kDepth;
  __shared__ __attribute__((aligned(16))) uint16_t lds[4 * TS];
  const int blk = xcd_block(blockIdx.x, gridDim.x);
  const int batch = blk / pairs;
  int rest = blk - batch * pairs, bi = 0;
  const int nb = np / kTile;
  while (rest >= nb - bi) rest -= nb - bi++;
  const int bj = bi + rest;                   // bj >= bi
  const uint16_t* src = in + (long)batch * np * kp;
  uint16_t* dst = out + (long)batch * np * np;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wr = wid >> 1, wc = wid & 1;

  f32x16 acc[2][2] = {};
  const int nt = kp / kDepth;
  stage_tile<kTile, kDepth>(lds, src, kp, bj * kTile, 0);
  stage_tile<kTile, kDepth>(lds + TS, src, kp, bi * kTile, 0);
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const uint16_t* la = lds + (t & 1) * 2 * TS;
    const uint16_t* lb = la + TS;
    if (t + 1 < nt) {
      uint16_t* nx = lds + ((t + 1) & 1) * 2 * TS;
      stage_tile<kTile, kDepth>(nx, src, kp, bj * kTile, (t + 1) * kDepth);
      stage_tile<kTile, kDepth>(nx + TS, src, kp, bi * kTile, (t + 1) * kDepth);
    }
#pragma unroll
    for (int st = 0; st < kDepth / 16; ++st) {
      s16x8 fa[2], fb[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        fa[u] = row_frag<kDepth>(la, wr * 64 + u * 32, st, lane);
        fb[u] = row_frag<kDepth>(lb, wc * 64 + u * 32, st, lane);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          acc[u][v] = mfma32<FP16>(fa[u], fb[v], acc[u][v]);
    }
  }
  constexpr float by = POLY ? kNsC : 1.f / (kXScale * kXScale);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int i = bi * kTile + wc * 64 + v * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j =
            bj * kTile + wr * 64 + u * 32 + q * 8 + (lane >> 5) * 4;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[u][v][q * 4 + e] * by;
        if (POLY) {
          const Pack<uint16_t, 4> o =
              *reinterpret_cast<const Pack<uint16_t, 4>*>(src + (long)i * np +
                                                          j);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] += kNsB * h2f(o.v[e]);
        }
        Pack<uint16_t, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = from_f32<FP16>(x[e]).v;
        const int js = POLY ? quad_swap(j) : j;
        *reinterpret_cast<Pack<uint16_t, 4>*>(dst + (long)i * np + js) = y;
        if (bi != bj) {
          const int is = POLY ? quad_swap(i) : i;
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[(long)(j + e) * np + is] = y.v[e];
        }
      }
    }
}

struct NsUpdate {
  const uint16_t *b, *xh, *xl;        // b: columns quad-swapped
  uint16_t *yh, *yl;                  // the next X, or
  uint16_t* out;                      // the result, bf16
  int np, mp, rows, cols;
  bool tall;
};

// a X + B X
template <bool LAST>
__global__ __launch_bounds__(256) void ns_update_kernel(NsUpdate a) {
  constexpr int TB = kTile * kDepth, TX = kDepth * kTile;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * (TB + TX)];
  const int nbi = a.np / kTile, nbj = a.mp / kTile;
  int blk = xcd_block(blockIdx.x, gridDim.x);
  const int batch = blk / (nbi * nbj);
  blk -= batch * nbi * nbj;
  const int bj = blk / nbi, bi = blk - bj * nbi;
  const uint16_t* bm = a.b + (long)batch * a.np * a.np;
  const long xo = (long)batch * a.np * a.mp;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wr = wid >> 1, wc = wid & 1;

  f32x16 acc[2][2] = {};
  const int nt = a.np / kDepth;
  stage_tile<kDepth, kTile>(lds, a.xh + xo, a.mp, 0, bj * kTile);
  stage_tile<kTile, kDepth>(lds + TX, bm, a.np, bi * kTile, 0);
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const uint16_t* lx = lds + (t & 1) * (TB + TX);
    const uint16_t* lb = lx + TX;
    if (t + 1 < nt) {
      uint16_t* nx = lds + ((t + 1) & 1) * (TB + TX);
      stage_tile<kDepth, kTile>(nx, a.xh + xo, a.mp, (t + 1) * kDepth,
                                bj * kTile);
      stage_tile<kTile, kDepth>(nx + TX, bm, a.np, bi * kTile,
                                (t + 1) * kDepth);
    }
#pragma unroll
    for (int st = 0; st < kDepth / 16; ++st) {
      s16x8 fa[2], fb[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        fa[u] = tr_frag<kTile>(lx, st * 16, wr * 64 + u * 32, lane);
        fb[u] = row_frag<kDepth>(lb, wc * 64 + u * 32, st, lane);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          acc[u][v] = mfma32<FP16>(fa[u], fb[v], acc[u][v]);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int i = bi * kTile + wc * 64 + v * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j =
            bj * kTile + wr * 64 + u * 32 + q * 8 + (lane >> 5) * 4;
        const long o = xo + (long)i * a.mp + j;
        const Pack<uint16_t, 4> h =
            *reinterpret_cast<const Pack<uint16_t, 4>*>(a.xh + o);
        const Pack<uint16_t, 4> l =
            *reinterpret_cast<const Pack<uint16_t, 4>*>(a.xl + o);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = kNsA * (h2f(h.v[e]) + h2f(l.v[e])) + acc[u][v][q * 4 + e];
        if (!LAST) {
          Pack<uint16_t, 4> yh, yl;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            yh.v[e] = from_f32<FP16>(x[e]).v;
            yl.v[e] = from_f32<FP16>(x[e] - h2f(yh.v[e])).v;
          }
          *reinterpret_cast<Pack<uint16_t, 4>*>(a.yh + o) = yh;
          *reinterpret_cast<Pack<uint16_t, 4>*>(a.yl + o) = yl;
        } else {
          uint16_t* out = a.out + (long)batch * a.rows * a.cols;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t y = from_f32<BF16>(x[e] * (1.f / kXScale)).v;
            const int r = a.tall ? j + e : i, c = a.tall ? i : j + e;
            if (r < a.rows && c < a.cols) out[(long)r * a.cols + c] = y;
          }
        }
      }
    }
}

template <typename T>
void launch_start(const at::Tensor& g, double* part, int parts, uint16_t* xh,
                  uint16_t* xl, int batch, int rows, int cols, int np, int mp,
                  float eps, hipStream_t s) {
  const T* p = static_cast<const T*>(g.data_ptr());
  ns_norm_kernel<T><<<dim3(parts, batch), 256, 0, s>>>(p, part,
                                                       (long)rows * cols);
  ns_split_kernel<T><<<dim3(mp / 64, np / 64, batch), 256, 0, s>>>(
      p, part, parts, xh, xl, rows, cols, rows > cols, np, mp, eps);
}

}  // namespace

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
  auto pad = [](long x) { return (x + kTile - 1) / kTile * kTile; };
  const long np = pad(std::min(rows, cols)), mp = pad(std::max(rows, cols));
  const long nb = np / kTile, pairs = nb * (nb + 1) / 2;
  TORCH_CHECK(batch * nb * (mp / kTile) <= std::numeric_limits<int>::max() &&
                  mp / 64 <= 65535,
              "newton_schulz: the matrices are too large or too many");
  const long parts = (rows * cols + kNormChunk - 1) / kNormChunk;

  const auto half = g.options().dtype(at::kHalf);
  auto x = at::empty({4, batch, np, mp}, half);       // X twice, in two parts
  auto sq = at::empty({2, batch, np, np}, half);      // A, B
  auto part = at::empty({batch, parts}, g.options().dtype(at::kDouble));
  auto* px = static_cast<uint16_t*>(x.data_ptr());
  auto* pa = static_cast<uint16_t*>(sq.data_ptr());
  const long xs = batch * np * mp;
  uint16_t* pb = pa + batch * np * np;
  const auto s = at::cuda::getCurrentCUDAStream();

  auto start = [&](auto tag) {
    launch_start<decltype(tag)>(g, part.data_ptr<double>(), (int)parts, px,
                                px + xs, (int)batch, (int)rows, (int)cols,
                                (int)np, (int)mp, (float)eps, s);
  };
  switch (g.scalar_type()) {
    case at::kFloat: start(float{}); break;
    case at::kBFloat16: start(BF16{}); break;
    case at::kHalf: start(FP16{}); break;
    default:
      TORCH_CHECK(false, "newton_schulz: unsupported dtype ", g.scalar_type());
  }
  for (int64_t k = 0; k < steps; ++k) {
    uint16_t* cur = px + (k & 1) * 2 * xs;
    uint16_t* nxt = px + ((k + 1) & 1) * 2 * xs;
    ns_square_kernel<false><<<(unsigned)(batch * pairs), 256, 0, s>>>(
        cur, pa, (int)np, (int)mp, (int)pairs);
    ns_square_kernel<true><<<(unsigned)(batch * pairs), 256, 0, s>>>(
        pa, pb, (int)np, (int)np, (int)pairs);
    NsUpdate u{pb, cur, cur + xs, nxt, nxt + xs,
               static_cast<uint16_t*>(out.data_ptr()), (int)np, (int)mp,
               (int)rows, (int)cols, rows > cols};
    const unsigned blocks = (unsigned)(batch * nb * (mp / kTile));
    if (k + 1 < steps)
      ns_update_kernel<false><<<blocks, 256, 0, s>>>(u);
    else
      ns_update_kernel<true><<<blocks, 256, 0, s>>>(u);
  }
  return out;
}

}  // namespace dlx

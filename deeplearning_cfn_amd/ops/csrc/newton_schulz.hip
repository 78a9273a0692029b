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
// 2.2e-3 relative (CPU model of these roundings, five spectra, sizes 64 to
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
constexpr int kNormChunk = 1 << 14;   // elements of a partial norm

// k within 16 as operand B wants it next to Frags::tr: quads 0, 2, 1, 3
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
    const int chunk = (f % CH) ^ swizzle<DP>(row);
    copy16_to_lds(src + (row0 + row) * ld + col0 + chunk * 8, lds + f * 8);
  }
}

// V elements at a time: the matrices' size is a multiple of V.
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

// G to X_0: scaled, split in two, padded with zeros, a tall one transposed.
// A block writes a 64 x 64 tile of X.
template <typename T, int V>
__global__ __launch_bounds__(256) void ns_split_kernel(
    const T* __restrict__ g, const double* __restrict__ part, int parts,
    uint16_t* __restrict__ xh, uint16_t* __restrict__ xl, int rows, int cols,
    bool tall, int np, int mp, float eps) {
  __shared__ float t[64][65];
  __shared__ double red[4];
  const int b = blockIdx.z;
  const double sum = ns_sum(part + (long)b * parts, parts, red);
  const float by = (float)(kXScale / (sqrt(sum) + (double)eps));
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
    for (int e = 0; e < V; ++e) t[r][x + e] = v[e] * by;
  }
  __syncthreads();
  const int xj = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int r = threadIdx.x >> 4; r < 64; r += 16) {
    const long o = ((long)b * np + i0 + r) * mp + j0 + xj;
    Pack<uint16_t, 4> h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = tall ? t[xj + e][r] : t[r][xj + e];
      h.v[e] = from_f32<FP16>(v).v;
      l.v[e] = from_f32<FP16>(v - h2f(h.v[e])).v;
    }
    *reinterpret_cast<Pack<uint16_t, 4>*>(xh + o) = h;
    *reinterpret_cast<Pack<uint16_t, 4>*>(xl + o) = l;
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

  const Frags<kDepth> fr(lane);
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
        fa[u] = fr.row(la, wr * 64 + u * 32, st);
        fb[u] = fr.row(lb, wc * 64 + u * 32, st);
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
  const uint16_t *b, *xh, *xl;        // b: columns quad-swapped; xl or none
  uint16_t *yh, *yl;                  // the next X (yl or none), or
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

  const Frags<kDepth> fr(lane);
  const Frags<kTile> fx(lane, wr * 64);
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
        fa[u] = fx.tr(lx, st * 16, u);
        fb[u] = fr.row(lb, wc * 64 + u * 32, st);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          acc[u][v] = mfma32<FP16>(fa[u], fb[v], acc[u][v]);
    }
  }
  // Through LDS as fp32 rows of X, so that memory sees whole lines.  Chunk c
  // of 4 in row i lies at c ^ (i & 31).
  __syncthreads();
  float* img = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int i = wc * 64 + v * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = (wr * 64 + u * 32 + q * 8 + (lane >> 5) * 4) >> 2;
        *reinterpret_cast<F32x4*>(img + i * kTile + ((c ^ (i & 31)) << 2)) =
            F32x4{{acc[u][v][q * 4], acc[u][v][q * 4 + 1],
                   acc[u][v][q * 4 + 2], acc[u][v][q * 4 + 3]}};
      }
    }
  __syncthreads();
  const int cj = (threadIdx.x & 15) * 8;
  const int j = bj * kTile + cj;
#pragma unroll 2
  for (int p = 0; p < kTile / 16; ++p) {
    const int il = p * 16 + (threadIdx.x >> 4);
    const int i = bi * kTile + il;
    const long o = xo + (long)i * a.mp + j;
    using P8 = Pack<uint16_t, 8>;
    const P8 h = *reinterpret_cast<const P8*>(a.xh + o);
    P8 l = {};
    if (a.xl) l = *reinterpret_cast<const P8*>(a.xl + o);
    float x[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const F32x4 y = *reinterpret_cast<const F32x4*>(
          img + il * kTile + ((((cj >> 2) + e) ^ (il & 31)) << 2));
#pragma unroll
      for (int k = 0; k < 4; ++k) x[e * 4 + k] = y.v[k];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float w = h2f(h.v[e]);
      if (a.xl) w += h2f(l.v[e]);
      x[e] += kNsA * w;
    }
    if (!LAST) {
      P8 yh, yl;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        yh.v[e] = from_f32<FP16>(x[e]).v;
        yl.v[e] = from_f32<FP16>(x[e] - h2f(yh.v[e])).v;
      }
      *reinterpret_cast<P8*>(a.yh + o) = yh;
      if (a.yl) *reinterpret_cast<P8*>(a.yl + o) = yl;
    } else {
      P8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        y.v[e] = from_f32<BF16>(x[e] * (1.f / kXScale)).v;
      uint16_t* out = a.out + (long)batch * a.rows * a.cols;
      if (!a.tall) {
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
          *reinterpret_cast<F32x4*>(
              img + il * kTile + ((((cj >> 2) + e) ^ (il & 31)) << 2)) =
              F32x4{{x[e * 4], x[e * 4 + 1], x[e * 4 + 2], x[e * 4 + 3]}};
      }
    }
  }
  if (LAST && a.tall) {
    __syncthreads();
    uint16_t* out = a.out + (long)batch * a.rows * a.cols;
    const int il = (threadIdx.x & 63) * 2;
    for (int jl = threadIdx.x >> 6; jl < kTile; jl += 4) {
      const int r = bj * kTile + jl, c = bi * kTile + il;
      if (r >= a.rows) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = il + e;
        const float x =
            img[i * kTile + (((jl >> 2) ^ (i & 31)) << 2) + (jl & 3)];
        if (c + e < a.cols)
          out[(long)r * a.cols + c + e] =
              from_f32<BF16>(x * (1.f / kXScale)).v;
      }
    }
  }
}

template <typename T, int V>
void launch_start(const at::Tensor& g, double* part, int parts, uint16_t* xh,
                  uint16_t* xl, int batch, int rows, int cols, int np, int mp,
                  float eps, hipStream_t s) {
  const T* p = static_cast<const T*>(g.data_ptr());
  ns_norm_kernel<T, V><<<dim3(parts, batch), 256, 0, s>>>(p, part,
                                                          (long)rows * cols);
  ns_split_kernel<T, V><<<dim3(mp / 64, np / 64, batch), 256, 0, s>>>(
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
    using T = decltype(tag);
    // four elements at a time where rows begin on such a border
    const bool v4 = cols % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0;
    (v4 ? launch_start<T, 4> : launch_start<T, 1>)(
        g, part.data_ptr<double>(), (int)parts, px, px + xs, (int)batch,
        (int)rows, (int)cols, (int)np, (int)mp, (float)eps, s);
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
    // the last two X that are multiplied have one part
    NsUpdate u{pb, cur, k + 2 < steps ? cur + xs : nullptr, nxt,
               k + 3 < steps ? nxt + xs : nullptr,
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

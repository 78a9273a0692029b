// Embedding lookup: a sum of scaled rows of one to four tables, and the
// tables' gradients.
//
//   y[t]    = sum_j c_j W_j[id_j[t]]                 (fp32, rounded once)
//   dW_j[r] = c_j sum_{t : id_j[t] = r} dy[t]        (fp32, rounded once)
//
// Both directions are bound by memory.  The lookup reads each row and
// writes y once, in one launch for all tables.
//
// The gradient sorts the tokens by id and sums each row's tokens in that
// order, so every bit is the same from run to run (no float atomics).
//   1. embed_sort: a block owns a range of ids and looks at ALL tokens; the
//      tokens with smaller ids, counted on the way, are the place where its
//      own begin, so no block waits for another and one launch sorts.  It
//      reads the ids once a block (from L2), which costs less than the
//      launches of a many-pass sort up to about a hundred thousand tokens.
//   2. embed_grad: a wave sums a row of few tokens; a row of kHeavy or more
//      (a mask token, a segment) is cut into pieces, a block each, and the
//      piece that ends last adds them up in their order.
//
// An id outside its table reads nothing: its output row is NaN, and it
// takes no part in the gradient.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include <limits>

#include "seq_common.h"

namespace dlx {

namespace {

constexpr int kMaxTables = 4;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kMaxOwn = 2048;     // ids a sort block owns: 128 KiB of counts
constexpr int kHeavy = 64;        // tokens from which a row is cut in pieces
constexpr int kSlotUnit = 32;     // sorted positions to a piece's slot
constexpr int kMinPiece = 128;    // tokens of a piece
constexpr int kMaxPieces = 256;   // pieces of a row

struct LookupTable {
  const void* ids;
  const void* weight;
  long rows;
  float scale;
  int ids64;
};

struct LookupArgs {
  LookupTable t[kMaxTables];
  int n;
};

DLX_DEV long read_id(const void* ids, int ids64, long i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i]
               : static_cast<const int32_t*>(ids)[i];
}

// Four vectors of a token's row a thread, `tokens` tokens a block.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(
    LookupArgs a, T* __restrict__ y, long n, int width, int nvec,
    uint32_t div_mul, int div_sh, int tokens) {
  const long t0 = (long)blockIdx.x * tokens;
  const int here = (int)(n - t0 < tokens ? n - t0 : tokens);
  const int items = here * nvec;
#pragma unroll 4
  for (int it = threadIdx.x; it < items; it += 256) {
    const int tl = (int)(((uint64_t)it * div_mul) >> div_sh);
    const int c = (it - tl * nvec) * VEC;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    for (int j = 0; j < a.n; ++j) {
      const long id = read_id(a.t[j].ids, a.t[j].ids64, t0 + tl);
      if (id < 0 || id >= a.t[j].rows) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          acc[i] = __builtin_nanf("");
      } else {
        float w[VEC];
        load_vec<T, VEC>(static_cast<const T*>(a.t[j].weight) + id * width + c,
                         w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += a.t[j].scale * w[i];
      }
    }
    store_vec<T, VEC>(y + (t0 + tl) * width + c, acc);
  }
}

struct GradTable {
  const void* ids;
  void* out;            // [rows, width]
  int* order;           // [n] token of each sorted position
  int* first;           // [rows + 1] sorted position where a row begins
  int* slot_row;        // [slots] row of a piece, -1: none
  int* done;            // [slots] pieces of a row that are summed
  float* part;          // [slots, width]
  float scale;
  int ids64;
  int rows;
  int own;              // ids a sort block owns
  int sort0;            // first sort block
  int light0;           // first block of rows of few tokens
};

struct GradArgs {
  GradTable t[kMaxTables];
  int n;
  int slots;            // a table
};

DLX_DEV int piece_tokens(int count) {
  int p = (count + kMaxPieces - 1) / kMaxPieces;
  return p < kMinPiece ? kMinPiece : p;
}

// LDS: counts [wave][own], then 2 * kSortWaves scratch ints.
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(
    GradArgs a, int n) {
  extern __shared__ int lds[];
  int j = 0;
  while (j + 1 < a.n && (int)blockIdx.x >= a.t[j + 1].sort0) ++j;
  const GradTable& tb = a.t[j];
  const int own = tb.own;
  const int lo = ((int)blockIdx.x - tb.sort0) * own;
  const int hi = lo + own < tb.rows ? lo + own : tb.rows;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = threadIdx.x / kWave;
  volatile int* cnt = lds + w * own;
  int* scratch = lds + kSortWaves * own;

  for (int i = threadIdx.x; i < kSortWaves * own; i += kSortThreads)
    lds[i] = 0;
  __syncthreads();

  // a wave's own stretch of the tokens, in whole steps of 64
  const int seg = (n + kSortThreads - 1) / kSortThreads * kWave;
  const int s0 = w * seg;
  const int s1 = s0 + seg < n ? s0 + seg : n;
  int less = 0;
  constexpr int U = 4;
  for (int i0 = s0; i0 < s1; i0 += U * kWave) {
    long id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kWave + lane;
      id[u] = i < s1 ? read_id(tb.ids, tb.ids64, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      less += __popcll(__ballot(id[u] >= 0 && id[u] < lo));
      if (id[u] >= lo && id[u] < hi)
        atomicAdd(lds + w * own + (int)(id[u] - lo), 1);
    }
  }
  if (lane == 0) scratch[w] = less;
  __syncthreads();
  int start = 0;
  for (int i = 0; i < kSortWaves; ++i) start += scratch[i];

  // exclusive scan over (row, wave); two rows a thread
  constexpr int PER = kMaxOwn / kSortThreads;
  int mine[PER], sum = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = threadIdx.x * PER + u;
    mine[u] = 0;
    if (r < own)
      for (int i = 0; i < kSortWaves; ++i) mine[u] += lds[i * own + r];
    sum += mine[u];
  }
  int scan = sum;
  for (int off = 1; off < kWave; off <<= 1) {
    const int up = __shfl_up(scan, off, kWave);
    if (lane >= off) scan += up;
  }
  if (lane == kWave - 1) scratch[kSortWaves + w] = scan;
  __syncthreads();
  int base = start + scan - sum, end = start;
  for (int i = 0; i < kSortWaves; ++i) {
    if (i < w) base += scratch[kSortWaves + i];
    end += scratch[kSortWaves + i];
  }
  const int z0 = start / kSlotUnit;
  const int z1 = hi == tb.rows ? a.slots : end / kSlotUnit;
  for (int i = z0 + threadIdx.x; i < z1; i += kSortThreads) {
    tb.slot_row[i] = -1;
    tb.done[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = threadIdx.x * PER + u;
    if (r < own && lo + r < hi) {
      tb.first[lo + r] = base;
      if (mine[u] >= kHeavy) {
        // count / 32 slots lie inside the row, its pieces are fewer
        const int p = piece_tokens(mine[u]);
        const int k1 = (mine[u] + p - 1) / p;
        for (int k = 0; k < k1; ++k)
          tb.slot_row[base / kSlotUnit + k] = lo + r;
      }
      int at = base;
      for (int i = 0; i < kSortWaves; ++i) {
        const int c = lds[i * own + r];
        lds[i * own + r] = at;
        at += c;
      }
      base += mine[u];
    }
  }
  if (hi == tb.rows && threadIdx.x == 0) tb.first[tb.rows] = end;
  __syncthreads();

  // again over the tokens: lanes of the same id take their places in order
  for (int i0 = s0; i0 < s1; i0 += U * kWave) {
    long id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kWave + lane;
      id[u] = i < s1 ? read_id(tb.ids, tb.ids64, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = id[u] >= lo && id[u] < hi;
      const int r = in ? (int)(id[u] - lo) : -1;
      uint64_t left = __ballot(in);
      while (left) {
        const int f = __ffsll((unsigned long long)left) - 1;
        const int rf = __shfl(r, f, kWave);
        const uint64_t same = __ballot(r == rf);
        const int at = cnt[rf];
        if (r == rf)
          tb.order[at + __popcll(same & ((1ull << lane) - 1))] =
              i0 + u * kWave + lane;
        if (lane == f) cnt[rf] = at + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// The sum of tokens order[p0..p1) of dy, columns c..c+VEC.  p1 - p0 <= 64 a
// turn: a lane holds one token's number and hands it to the others.
template <typename T, int VEC>
DLX_DEV void sum_tokens(const T* __restrict__ dy, const int* __restrict__ order,
                        int p0, int p1, int width, int c, bool on, int lane,
                        float* acc) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  for (int q = p0; q < p1; q += kWave) {
    const int m = p1 - q < kWave ? p1 - q : kWave;
    const int tok = lane < m ? order[q + lane] : 0;
    int k = 0;
    for (; k + 8 <= m; k += 8) {
      float x[8][VEC];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const long t = __builtin_amdgcn_readlane(tok, k + u);
        if (on) load_vec<T, VEC>(dy + t * width + c, x[u]);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += x[u][i];
    }
    for (; k < m; ++k) {
      float x[VEC];
      const long t = __builtin_amdgcn_readlane(tok, k);
      if (on) load_vec<T, VEC>(dy + t * width + c, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += x[i];
    }
  }
}

// Blocks [0, n * slots): pieces of rows of many tokens (they take longest,
// so they begin first); the rest: four rows of few tokens each.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_kernel(
    GradArgs a, const T* __restrict__ dy, int width) {
  __shared__ float red[4][kWave * VEC];
  __shared__ int last;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = threadIdx.x / kWave;
  const int nslots = a.n * a.slots;
  const int step = kWave * VEC;

  if ((int)blockIdx.x >= nslots) {
    const int b = (int)blockIdx.x - nslots;
    int j = 0;
    while (j + 1 < a.n && b >= a.t[j + 1].light0) ++j;
    const GradTable& tb = a.t[j];
    const int r = (b - tb.light0) * 4 + w;
    if (r >= tb.rows) return;
    const int p0 = tb.first[r], p1 = tb.first[r + 1];
    if (p1 - p0 >= kHeavy) return;
    T* out = static_cast<T*>(tb.out) + (long)r * width;
    for (int c0 = 0; c0 < width; c0 += step) {
      const int c = c0 + lane * VEC;
      float acc[VEC];
      sum_tokens<T, VEC>(dy, tb.order, p0, p1, width, c, c < width, lane, acc);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] *= tb.scale;
      if (c < width) store_vec<T, VEC>(out + c, acc);
    }
    return;
  }

  const int j = (int)blockIdx.x / a.slots;
  const int slot = (int)blockIdx.x - j * a.slots;
  const GradTable& tb = a.t[j];
  const int r = tb.slot_row[slot];
  if (r < 0) return;
  const int p0 = tb.first[r], p1 = tb.first[r + 1];
  const int piece = piece_tokens(p1 - p0);
  const int pieces = (p1 - p0 + piece - 1) / piece;
  const int slot0 = p0 / kSlotUnit;
  const int k = slot - slot0;
  const int q0 = p0 + k * piece;
  const int q1 = q0 + piece < p1 ? q0 + piece : p1;
  const int per = (q1 - q0 + 3) / 4;               // a wave's tokens
  const int w0 = q0 + w * per < q1 ? q0 + w * per : q1;
  const int w1 = w0 + per < q1 ? w0 + per : q1;
  T* out = static_cast<T*>(tb.out) + (long)r * width;

  for (int c0 = 0; c0 < width; c0 += step) {
    const int c = c0 + lane * VEC;
    float acc[VEC];
    sum_tokens<T, VEC>(dy, tb.order, w0, w1, width, c, c < width, lane, acc);
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[w][lane * VEC + i] = acc[i];
    __syncthreads();
    if (w == 0 && c < width) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        acc[i] = (red[0][lane * VEC + i] + red[1][lane * VEC + i]) +
                 (red[2][lane * VEC + i] + red[3][lane * VEC + i]);
      if (pieces == 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= tb.scale;
        store_vec<T, VEC>(out + c, acc);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          tb.part[(long)slot * width + c + i] = acc[i];
      }
    }
    __syncthreads();
  }
  if (pieces == 1) return;

  // The piece that ends last adds all of them, in their order.  Every
  // thread's stores are made visible before the count goes up, and the
  // count is seen before the other pieces are read.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(
        tb.done + slot0, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    last = before == pieces - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int kp = (pieces + 3) / 4;
  const int k0 = w * kp < pieces ? w * kp : pieces;
  const int k1 = k0 + kp < pieces ? k0 + kp : pieces;
  for (int c0 = 0; c0 < width; c0 += step) {
    const int c = c0 + lane * VEC;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    if (c < width) {
#pragma unroll 4
      for (int q = k0; q < k1; ++q)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          acc[i] += tb.part[(long)(slot0 + q) * width + c + i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[w][lane * VEC + i] = acc[i];
    __syncthreads();
    if (w == 0 && c < width) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        acc[i] = ((red[0][lane * VEC + i] + red[1][lane * VEC + i]) +
                  (red[2][lane * VEC + i] + red[3][lane * VEC + i])) *
                 tb.scale;
      store_vec<T, VEC>(out + c, acc);
    }
    __syncthreads();
  }
}

void check_ids(const at::Tensor& ids, const at::Tensor& like, int64_t n) {
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "embedding: ids have to be int32 or int64, got ",
              ids.scalar_type());
  TORCH_CHECK(ids.numel() == n, "embedding: the tables' ids differ in number");
  TORCH_CHECK(ids.device() == like.device(),
              "embedding: ids and tables are on different devices");
}

bool aligned16(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

template <typename T, int VEC>
void launch_fwd(const LookupArgs& a, at::Tensor& y, long n, int width,
                hipStream_t s) {
  const int nvec = width / VEC;
  // about 1024 vectors a block; fewer when that leaves the card empty
  long tokens = 1024 / nvec;
  if (tokens > (n + 511) / 512) tokens = (n + 511) / 512;
  if (tokens < 1) tokens = 1;
  // items < 1024 or one token's: it / nvec by multiplication is exact
  int sh = 31;
  while ((1ull << (sh - 31)) < (uint64_t)nvec) ++sh;
  const uint64_t mul = ((1ull << sh) + nvec - 1) / nvec;
  const long blocks = (n + tokens - 1) / tokens;
  TORCH_CHECK(blocks <= std::numeric_limits<int>::max(),
              "embedding: too many tokens");
  embed_fwd_kernel<T, VEC><<<(unsigned)blocks, 256, 0, s>>>(
      a, static_cast<T*>(y.data_ptr()), n, width, nvec, (uint32_t)mul, sh,
      (int)tokens);
}

template <typename T, int VEC>
void launch_grad(const GradArgs& a, const at::Tensor& dy, int width,
                 unsigned blocks, hipStream_t s) {
  embed_grad_kernel<T, VEC><<<blocks, 256, 0, s>>>(
      a, static_cast<const T*>(dy.data_ptr()), width);
}

}  // namespace

// ids: 1..4 index tensors of n elements; tables: [rows, width] each.
// -> [n, width]
at::Tensor embed_sum_fwd_impl(at::TensorList ids_in, at::TensorList tables_in,
                              at::ArrayRef<double> scales) {
  const size_t nt = tables_in.size();
  TORCH_CHECK(nt >= 1 && nt <= kMaxTables, "embedding: 1 to ", kMaxTables,
              " tables, got ", nt);
  TORCH_CHECK(ids_in.size() == nt && scales.size() == nt,
              "embedding: as many ids and scales as tables");
  const at::Tensor& w0 = tables_in[0];
  TORCH_CHECK(w0.dim() == 2, "embedding: a table is [rows, width]");
  const c10::DeviceGuard guard(w0.device());
  const long n = ids_in[0].numel(), width = w0.size(1);
  TORCH_CHECK(width <= (1 << 24), "embedding: a row is too wide");
  std::vector<at::Tensor> hold;
  LookupArgs a{};
  a.n = (int)nt;
  bool vec = true;
  for (size_t j = 0; j < nt; ++j) {
    const at::Tensor& w = tables_in[j];
    TORCH_CHECK(w.dim() == 2 && w.size(1) == width &&
                    w.scalar_type() == w0.scalar_type() &&
                    w.device() == w0.device(),
                "embedding: the tables differ in width, type or device");
    check_ids(ids_in[j], w0, n);
    hold.push_back(ids_in[j].contiguous());
    a.t[j].ids = hold.back().data_ptr();
    a.t[j].ids64 = hold.back().scalar_type() == at::kLong;
    hold.push_back(w.contiguous());
    a.t[j].weight = hold.back().data_ptr();
    a.t[j].rows = w.size(0);
    a.t[j].scale = (float)scales[j];
    vec = vec && aligned16(a.t[j].weight);
  }
  auto y = at::empty({n, width}, w0.options());
  if (n == 0 || width == 0) return y;
  auto s = at::cuda::getCurrentCUDAStream();
  switch (w0.scalar_type()) {
    case at::kBFloat16:
      if (vec && width % 8 == 0) launch_fwd<BF16, 8>(a, y, n, width, s);
      else launch_fwd<BF16, 1>(a, y, n, width, s);
      break;
    case at::kHalf:
      if (vec && width % 8 == 0) launch_fwd<FP16, 8>(a, y, n, width, s);
      else launch_fwd<FP16, 1>(a, y, n, width, s);
      break;
    case at::kFloat:
      if (vec && width % 4 == 0) launch_fwd<float, 4>(a, y, n, width, s);
      else launch_fwd<float, 1>(a, y, n, width, s);
      break;
    default:
      TORCH_CHECK(false, "embedding: unsupported dtype ", w0.scalar_type());
  }
  return y;
}

// dy: [n, width]; rows: of each table -> the tables' gradients in dy's type
std::vector<at::Tensor> embed_sum_bwd_impl(const at::Tensor& dy_in,
                                           at::TensorList ids_in,
                                           at::IntArrayRef rows,
                                           at::ArrayRef<double> scales) {
  const size_t nt = ids_in.size();
  TORCH_CHECK(nt >= 1 && nt <= kMaxTables && rows.size() == nt &&
                  scales.size() == nt,
              "embedding: as many rows and scales as ids, 1 to ", kMaxTables);
  TORCH_CHECK(dy_in.dim() == 2, "embedding: the gradient is [n, width]");
  const c10::DeviceGuard guard(dy_in.device());
  const auto dy = dy_in.contiguous();
  const long n = dy.size(0), width = dy.size(1);
  TORCH_CHECK(width <= (1 << 24) && n <= (1 << 30),
              "embedding: the gradient is too large");
  const long slots = n / kSlotUnit + 1;
  std::vector<at::Tensor> hold, out;
  GradArgs a{};
  a.n = (int)nt;
  a.slots = (int)slots;
  const auto ints = dy.options().dtype(at::kInt);
  long sort_blocks = 0, light_blocks = 0;
  int own_most = 1;
  for (size_t j = 0; j < nt; ++j) {
    check_ids(ids_in[j], dy, n);
    TORCH_CHECK(rows[j] >= 0 && rows[j] < (1ll << 31) - 8,
                "embedding: a table has too many rows");
    out.push_back(at::empty({rows[j], width}, dy.options()));
    GradTable& t = a.t[j];
    t.rows = (int)rows[j];
    // a block a CU; more where a block's counts would not fit its LDS
    long blocks = rows[j] < 256 ? std::max<long>(rows[j], 1) : 256;
    long own = (rows[j] + blocks - 1) / blocks;
    if (own > kMaxOwn) own = kMaxOwn;
    if (own < 1) own = 1;
    blocks = std::max<long>((rows[j] + own - 1) / own, 1);
    own_most = std::max(own_most, (int)own);
    t.own = (int)own;
    t.sort0 = (int)sort_blocks;
    sort_blocks += blocks;
    t.light0 = (int)light_blocks;
    light_blocks += (rows[j] + 3) / 4;
    hold.push_back(ids_in[j].contiguous());
    t.ids = hold.back().data_ptr();
    t.ids64 = hold.back().scalar_type() == at::kLong;
    t.scale = (float)scales[j];
    t.out = out.back().data_ptr();
    hold.push_back(at::empty({n + rows[j] + 1 + 2 * slots}, ints));
    t.order = hold.back().data_ptr<int>();
    t.first = t.order + n;
    t.slot_row = t.first + rows[j] + 1;
    t.done = t.slot_row + slots;
    hold.push_back(at::empty({slots * width}, dy.options().dtype(at::kFloat)));
    t.part = hold.back().data_ptr<float>();
  }
  if (width == 0) return out;
  if (n == 0) {
    for (auto& o : out) o.zero_();
    return out;
  }
  const long blocks = (long)nt * slots + light_blocks;
  TORCH_CHECK(blocks <= std::numeric_limits<int>::max(),
              "embedding: the tables are too large");
  auto s = at::cuda::getCurrentCUDAStream();
  const size_t lds =
      ((size_t)kSortWaves * own_most + 2 * kSortWaves) * sizeof(int);
  embed_sort_kernel<<<(unsigned)sort_blocks, kSortThreads, lds, s>>>(a, (int)n);
  const bool vec = aligned16(dy.data_ptr());
  switch (dy.scalar_type()) {
    case at::kBFloat16:
      if (vec && width % 8 == 0)
        launch_grad<BF16, 8>(a, dy, width, (unsigned)blocks, s);
      else
        launch_grad<BF16, 1>(a, dy, width, (unsigned)blocks, s);
      break;
    case at::kHalf:
      if (vec && width % 8 == 0)
        launch_grad<FP16, 8>(a, dy, width, (unsigned)blocks, s);
      else
        launch_grad<FP16, 1>(a, dy, width, (unsigned)blocks, s);
      break;
    case at::kFloat:
      if (vec && width % 4 == 0)
        launch_grad<float, 4>(a, dy, width, (unsigned)blocks, s);
      else
        launch_grad<float, 1>(a, dy, width, (unsigned)blocks, s);
      break;
    default:
      TORCH_CHECK(false, "embedding: unsupported dtype ", dy.scalar_type());
  }
  return out;
}

}  // namespace dlx

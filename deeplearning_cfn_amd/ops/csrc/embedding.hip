// Embedding lookup: a sum of scaled rows of one to four tables, and the
// tables' gradients.
//
//   y[t]    = sum_j c_j W_j[id_j[t]]                 (fp32, rounded once)
//   dW_j[r] = c_j sum_{t : id_j[t] = r} dy[t]        (fp32, rounded once)
//
// Both directions are bound by memory.  The lookup reads each row and
// writes y once, in one launch for all tables.
//
// The gradient sorts the tokens by id and sums each row's tokens in a fixed
// order, so every bit is the same from run to run (no float atomics).  It is
// the tokens' own up to 65536 of them; of more, a chunk's waves come one after
// the other, each with its tokens.
//   1. Tokens into buckets, id % G (frequent ids are neighbours in a
//      vocabulary, so this spreads them): embed_count counts each of up to
//      64 chunks of the tokens, embed_scatter turns the counts into places
//      and puts every token into its bucket.
//   2. embed_order sorts a bucket by the rest of the id, id / G, a block each.
//   3. embed_grad: a wave sums some rows of few tokens; a row of kHeavy or
//      more (a mask token, a segment) is cut into pieces, a block each.
//   4. embed_join adds up the pieces of a row, in their order.  (One block
//      of the third launch could, the last to finish; but the fence it needs
//      writes back its XCD's whole L2: 81 us instead of 41 for 16384 tokens
//      of 768 in three tables.)
// An id's "place" below is its number in that order, (id % G) * own + id / G.
//
// An id outside its table reads nothing: its output row is NaN, and it
// takes no part in the gradient.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include <algorithm>

#include "seq_common.h"

namespace dlx {

namespace {

constexpr int kMaxTables = 4;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kDirect = 4096;     // tokens up to which no buckets are made
constexpr int kChunks = 64;       // chunks of the tokens, at most
constexpr int kMaxSplit = 11;     // log2 of the buckets, and of a bucket's ids
constexpr int kMaxOwn = 1 << kMaxSplit;
constexpr int kHeavy = 32;        // tokens from which a row is cut in pieces
constexpr int kSlotUnit = 16;     // sorted positions to a piece's slot
constexpr int kPiece = 128;       // tokens of a piece, at least
constexpr int kMaxPieces = 256;   // pieces of a row
constexpr int kLightRows = 4;     // rows of few tokens to a wave

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

// An id as 32 bits without a sign; all ones where it fits no table.
DLX_DEV uint32_t read_id32(const void* ids, int ids64, long i) {
  if (!ids64) return static_cast<const uint32_t*>(ids)[i];
  const uint2 x = static_cast<const uint2*>(ids)[i];
  return x.y ? 0xffffffffu : x.x;
}

// Four vectors of a token's row a thread, `tokens` tokens a block.  Bound by
// memory: 16384 tokens of 768 in bf16, three tables, 25 MB of rows out of the
// largest and 25 MB written in 15 us; 65536 of 1024 in one table, 268 MB in
// 42 us (6.4 TB/s, rows of frequent ids come out of the caches).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(
    LookupArgs a, T* __restrict__ y, long n, int width, int nvec,
    uint32_t div_mul, int div_sh, int tokens) {
  for (long t0 = (long)blockIdx.x * tokens; t0 < n;
       t0 += (long)gridDim.x * tokens) {
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
}

struct GradTable {
  const void* ids;
  void* out;            // [rows, width]
  int* count;           // [buckets, kChunks] tokens
  int* start;           // [buckets + 1] sorted position where one begins
  int2* loose;          // [n] tokens in buckets, with id / G
  int* order;           // [n] token of each sorted position
  int* first;           // [places + 1] sorted position where a place begins
  int* slot_row;        // [slots] place of a piece, -1: none
  int* join_row;        // [joins] place whose pieces are added up, -1: none
  float* part;          // [slots, width]
  float scale;
  int ids64;
  int rows;
  int own;              // ids of a bucket
  int lg;               // log2 of the buckets, G
  int bucket0;          // first block of embed_order
  int light0;           // first block of rows of few tokens
};

struct GradArgs {
  GradTable t[kMaxTables];
  int n;
  int slots, joins;     // a table
};

DLX_DEV int place_id(const GradTable& t, int place) {
  const int b = place / t.own;
  return b + ((place - b * t.own) << t.lg);
}

DLX_DEV int piece_tokens(int count) {
  int p = (count + kMaxPieces - 1) / kMaxPieces;
  return p < kPiece ? kPiece : p;
}

// The lanes of `any` whose number is mine.  The first two numbers are looked
// for one by one (a frequent id fills a bucket nearly alone), the others bit
// by bit.
DLX_DEV uint64_t peers(int r, uint64_t any, int bits) {
  uint64_t same = 0, left = any;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!left) return same;
    const int f = __ffsll((unsigned long long)left) - 1;
    const bool me = r == __builtin_amdgcn_readlane(r, f);
    const uint64_t m = __ballot(me) & any;
    if (me) same = m;
    left &= ~m;
  }
  if (!left) return same;
  uint64_t rest = left;
  for (int b = 0; b < bits; ++b) {
    const uint64_t one = __ballot((r >> b) & 1);
    rest &= (r >> b) & 1 ? one : ~one;
  }
  const uint64_t bit = 1ull << (threadIdx.x & (kWave - 1));
  return left & bit ? rest : same;
}

// Block (c, j): the tokens of chunk c in each bucket of table j.  16384 tokens
// in three tables 3.8 us, 65536 in one 3.5 us: a launch and three waits.
__global__ __launch_bounds__(kSortThreads) void embed_count_kernel(
    GradArgs a, int n, int chunk) {
  __shared__ int h[kMaxOwn];
  const GradTable& tb = a.t[blockIdx.y];
  const int g = 1 << tb.lg;
  for (int i = threadIdx.x; i < g; i += kSortThreads) h[i] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * chunk;
  const int i1 = n - i0 < chunk ? n : i0 + chunk;
  for (int i = i0 + threadIdx.x; i < i1; i += kSortThreads) {
    const uint32_t id = read_id32(tb.ids, tb.ids64, i);
    if (id < (uint32_t)tb.rows) atomicAdd(h + (id & (g - 1)), 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g; i += kSortThreads)
    tb.count[i * kChunks + blockIdx.x] = h[i];
}

// Exclusive sum over a block of kSortThreads; scratch: kSortWaves ints.
DLX_DEV int block_scan(int x, int* scratch) {
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  int s = x;
  for (int off = 1; off < kWave; off <<= 1) {
    const int up = __shfl_up(s, off, kWave);
    if (lane >= off) s += up;
  }
  if (lane == kWave - 1) scratch[w] = s;
  __syncthreads();
  int base = s - x;
  for (int i = 0; i < w; ++i) base += scratch[i];
  __syncthreads();
  return base;
}

// Block (c, j): the tokens of chunk c into table j's buckets.
// 16384 tokens in three tables 8.5 us, 65536 in one 12.5 us: bound by its own
// chain of reads, counts, a scan and a second walk, not by bytes (0.5 MB).
// LDS: counts [wave][bucket], then scratch.
__global__ __launch_bounds__(kSortThreads) void embed_scatter_kernel(
    GradArgs a, int n, int chunk, int chunks) {
  extern __shared__ int lds[];
  const GradTable& tb = a.t[blockIdx.y];
  const int g = 1 << tb.lg, bits = tb.lg;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  volatile int* cnt = lds + w * g;
  int* scratch = lds + kSortWaves * g;
  const int me = blockIdx.x;
  for (int i = threadIdx.x; i < kSortWaves * g; i += kSortThreads) lds[i] = 0;
  __syncthreads();

  const int i0 = me * chunk;
  const int i1 = n - i0 < chunk ? n : i0 + chunk;
  for (int i = i0 + w * kWave; i < i1; i += kSortThreads) {
    const uint32_t id =
        i + lane < i1 ? read_id32(tb.ids, tb.ids64, i + lane) : 0xffffffffu;
    const bool in = id < (uint32_t)tb.rows;
    const int r = in ? (int)(id & (g - 1)) : 0;
    const uint64_t same = peers(r, __ballot(in), bits);
    if (in && !(same & ((1ull << lane) - 1))) cnt[r] = cnt[r] + __popcll(same);
  }
  __syncthreads();

  // two buckets a thread: all chunks' tokens, and those of chunks before me
  constexpr int PER = kMaxOwn / kSortThreads;
  int total[PER], before[PER], sum = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = threadIdx.x * PER + u;
    total[u] = before[u] = 0;
    if (r < g) {
      const int4* p = reinterpret_cast<const int4*>(tb.count + r * kChunks);
      for (int c = 0; c < chunks; c += 4) {
        const int4 x = p[c / 4];
        const int y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c + e < chunks) total[u] += y[e];
          if (c + e < me) before[u] += y[e];
        }
      }
    }
    sum += total[u];
  }
  int base = block_scan(sum, scratch);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = threadIdx.x * PER + u;
    if (r < g) {
      if (me == 0) tb.start[r] = base;
      int at = base + before[u];
      for (int i = 0; i < kSortWaves; ++i) {
        const int c = lds[i * g + r];
        lds[i * g + r] = at;
        at += c;
      }
      if (me == 0 && r == g - 1) tb.start[g] = base + total[u];
    }
    base += total[u];
  }
  __syncthreads();

  for (int i = i0 + w * kWave; i < i1; i += kSortThreads) {
    const uint32_t id =
        i + lane < i1 ? read_id32(tb.ids, tb.ids64, i + lane) : 0xffffffffu;
    const bool in = id < (uint32_t)tb.rows;
    const int r = in ? (int)(id & (g - 1)) : 0;
    const uint64_t same = peers(r, __ballot(in), bits);
    if (in) {
      const uint64_t first = same & ((1ull << lane) - 1);
      const int at = cnt[r];
      tb.loose[at + __popcll(first)] = make_int2(i + lane, (int)(id >> bits));
      if (!first) cnt[r] = at + __popcll(same);
    }
  }
}

// Token number i of a bucket's list, or of all tokens (DIRECT), with its id
// / G; that is -1 behind the end and, of all tokens, in another bucket.
template <bool DIRECT>
DLX_DEV int2 token_at(const GradTable& t, int i, int end, int me, int& less) {
  if (!DIRECT) {
    int2 x = t.loose[i < end ? i : end - 1];
    if (i >= end) x.y = -1;
    return x;
  }
  const uint32_t id =
      i < end ? read_id32(t.ids, t.ids64, i) : 0xffffffffu;
  const bool ok = id < (uint32_t)t.rows;
  const int bucket = (int)(id & ((1u << t.lg) - 1));
  less += __popcll(__ballot(ok && bucket < me));
  return make_int2(i, ok && bucket == me ? (int)(id >> t.lg) : -1);
}

// A bucket's tokens by id / G.  DIRECT: few tokens; every block looks at all
// of them, and those of lower buckets, counted on the way, are the place where
// its own begin, which saves the launches that make the buckets (three tables,
// 4096 tokens of 768: 32 us for a whole gradient, more with buckets).
// Bound by its chain of reads, counts, a scan and a second walk: 16384 tokens
// in three tables 11 us, 65536 in one 15.5 us; two tables of 3001 tokens,
// without buckets, 10 us.
// LDS: counts [wave][own], then scratch.
template <bool DIRECT>
__global__ __launch_bounds__(kSortThreads) void embed_order_kernel(GradArgs a,
                                                                   int n) {
  extern __shared__ int lds[];
  const int blk = (int)blockIdx.x;
  int j = 0;
  while (j + 1 < a.n && blk >= a.t[j + 1].bucket0) ++j;
  const GradTable& tb = a.t[j];
  const int own = tb.own;
  const int me = blk - tb.bucket0;
  const int lo = me * own;
  const bool top = me == (1 << tb.lg) - 1;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  volatile int* cnt = lds + w * own;
  int* scratch = lds + kSortWaves * own;
  for (int i = threadIdx.x; i < kSortWaves * own; i += kSortThreads)
    lds[i] = 0;
  __syncthreads();

  // a wave's own stretch of the list; U times 64 tokens of it on their way
  constexpr int U = 4;
  int start = 0, end = n;
  if (!DIRECT) {
    start = __builtin_amdgcn_readfirstlane(tb.start[me]);
    end = __builtin_amdgcn_readfirstlane(tb.start[me + 1]);
  }
  const int seg = (end - start + kSortThreads - 1) / kSortThreads * kWave;
  const int s0 = start + w * seg < end ? start + w * seg : end;
  const int s1 = s0 + seg < end ? s0 + seg : end;
  const int bits = own > 1 ? 32 - __clz(own - 1) : 0;
  int less = 0, unused = 0;
  // a bucket of one id is in order already (the same: 17.8 -> 13.4 us)
  const bool alone = !DIRECT && own == 1;
  if (alone && threadIdx.x == 0) lds[0] = end - start;
  for (int i = s0; i < s1 && !alone; i += U * kWave) {
    int2 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = token_at<DIRECT>(tb, i + u * kWave + lane, s1, me, less);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = x[u].y;
      const uint64_t any = __ballot(r >= 0);
      if (!any) continue;
      const uint64_t same = peers(r, any, bits);
      if (r >= 0 && !(same & ((1ull << lane) - 1)))
        cnt[r] = cnt[r] + __popcll(same);
    }
  }
  if (DIRECT && lane == 0) scratch[kSortWaves + w] = less;
  __syncthreads();

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
  int first = start;
  if (DIRECT)
    for (int i = 0; i < kSortWaves; ++i) first += scratch[kSortWaves + i];
  int base = first + block_scan(sum, scratch);
  if (DIRECT) {
    if (threadIdx.x == kSortThreads - 1) scratch[kSortWaves] = base + sum;
    __syncthreads();
  }
  const int last = DIRECT ? scratch[kSortWaves] : end;
  // this block's pieces' slots: those that begin between its borders
  const int z1 = top ? a.slots : last / kSlotUnit;
  for (int i = first / kSlotUnit + threadIdx.x; i < z1; i += kSortThreads)
    tb.slot_row[i] = -1;
  // a row of more than one piece owns the first multiple of kPiece in it
  const int y1 = top ? a.joins : (last + kPiece - 1) / kPiece;
  for (int i = (first + kPiece - 1) / kPiece + threadIdx.x; i < y1;
       i += kSortThreads)
    tb.join_row[i] = -1;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = threadIdx.x * PER + u;
    if (r < own) {
      tb.first[lo + r] = base;
      if (mine[u] >= kHeavy) {
        // count / 16 slots lie inside the row, its pieces are fewer
        const int p = piece_tokens(mine[u]);
        const int k1 = (mine[u] + p - 1) / p;
        for (int k = 0; k < k1; ++k)
          tb.slot_row[base / kSlotUnit + k] = lo + r;
        if (k1 > 1) tb.join_row[(base + kPiece - 1) / kPiece] = lo + r;
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
  if (top && threadIdx.x == 0) tb.first[lo + own] = last;
  if (alone) {
#pragma unroll 4
    for (int i = start + threadIdx.x; i < end; i += kSortThreads)
      tb.order[i] = tb.loose[i].x;
    return;
  }
  __syncthreads();

  for (int i = s0; i < s1; i += U * kWave) {
    int2 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = token_at<DIRECT>(tb, i + u * kWave + lane, s1, me, unused);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = x[u].y;
      const uint64_t any = __ballot(r >= 0);
      if (!any) continue;
      const uint64_t same = peers(r, any, bits);
      if (r >= 0) {
        const uint64_t before = same & ((1ull << lane) - 1);
        const int at = cnt[r];
        tb.order[at + __popcll(before)] = x[u].x;
        if (!before) cnt[r] = at + __popcll(same);
      }
    }
  }
}

constexpr int kFlight = 8;          // rows on their way at a time

// The sum of tokens order[p0..p1), VEC columns at `from` in token 0.  64
// tokens a turn: a lane holds one token's number and hands it to the others.
template <typename T, int VEC>
DLX_DEV void sum_tokens(const T* __restrict__ from,
                        const int* __restrict__ order, int p0, int p1,
                        int width, int lane, float* acc) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  for (int q = p0; q < p1; q += kWave) {
    const int m = p1 - q < kWave ? p1 - q : kWave;
    const int tok = lane < m ? order[q + lane] : 0;
    for (int k = 0; k < m; k += kFlight) {
      Pack<T, VEC> x[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const long t =
            __builtin_amdgcn_readlane(tok, k + u < m ? k + u : m - 1);
        x[u] = *reinterpret_cast<const Pack<T, VEC>*>(from + t * width);
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        if (k + u < m) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += to_f32<T>(x[u].v[i]);
        }
    }
  }
}

// Blocks [0, n * slots): pieces of rows of many tokens (they take longest,
// so they begin first); the rest: kLightRows rows of few tokens a wave.
// Columns: blockIdx.y * cols and on, VEC a lane, cols <= 64 * VEC.
// Bound by memory, and by how many rows are on their way: 16384 tokens of 768,
// three tables, 23.4 us for 75 MB read (the second and third time out of the
// caches) and 48 MB written; 65536 of 1024 in one table 54 us for 134 MB read
// in the order of the ids and 63 MB written (3.6 TB/s).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_kernel(
    GradArgs a, const T* __restrict__ dy, int width, int cols) {
  __shared__ float red[4][kWave * VEC];
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nslots = a.n * a.slots;
  const int c0 = blockIdx.y * cols;
  const int c = c0 + lane * VEC;
  const bool on = lane * VEC < cols && c < width;
  // lanes without columns load the first ones: a load under a condition
  // would be waited for before the next one is sent
  const T* from = dy + (on ? c : c0);

  if ((int)blockIdx.x >= nslots) {
    const int b = (int)blockIdx.x - nslots;
    int j = 0;
    while (j + 1 < a.n && b >= a.t[j + 1].light0) ++j;
    const GradTable& tb = a.t[j];
    const int r0 = ((b - tb.light0) * 4 + w) * kLightRows;
    const int places = tb.own << tb.lg;
    if (r0 >= places) return;
    const int nr = places - r0 < kLightRows ? places - r0 : kLightRows;
    // lane i: where place r0 + i begins (lane nr: where the last one ends)
    const int begin = tb.first[r0 + (lane < nr ? lane : nr)];
    int r = 0;
    while (r < nr) {
      int p = __builtin_amdgcn_readlane(begin, r);
      int e = __builtin_amdgcn_readlane(begin, r + 1);
      if (e - p >= kHeavy) {
        ++r;
        continue;
      }
      // the rows up to the next heavy one: their tokens are neighbours
      int r1 = r + 1, p1 = e;
      while (r1 < nr) {
        const int n = __builtin_amdgcn_readlane(begin, r1 + 1);
        if (n - p1 >= kHeavy) break;
        p1 = n;
        ++r1;
      }
      float acc[VEC] = {};
      auto store = [&]() {
        const int id = place_id(tb, r0 + r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= tb.scale;
        if (on && id < tb.rows)
          store_vec<T, VEC>(static_cast<T*>(tb.out) + (long)id * width + c, acc);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
        ++r;
        if (r < r1) e = __builtin_amdgcn_readlane(begin, r + 1);
      };
      for (; p < p1; p += kWave) {
        const int m = p1 - p < kWave ? p1 - p : kWave;
        const int tok = lane < m ? tb.order[p + lane] : 0;
        for (int k = 0; k < m; k += kFlight) {
          Pack<T, VEC> x[kFlight];
#pragma unroll
          for (int u = 0; u < kFlight; ++u) {
            const long t =
                __builtin_amdgcn_readlane(tok, k + u < m ? k + u : m - 1);
            x[u] = *reinterpret_cast<const Pack<T, VEC>*>(from + t * width);
          }
#pragma unroll
          for (int u = 0; u < kFlight; ++u)
            if (k + u < m) {
              while (e <= p + k + u) store();
#pragma unroll
              for (int i = 0; i < VEC; ++i) acc[i] += to_f32<T>(x[u].v[i]);
            }
        }
      }
      while (r < r1) store();
    }
    return;
  }

  const int j = (int)blockIdx.x / a.slots;
  const int slot = (int)blockIdx.x - j * a.slots;
  const GradTable& tb = a.t[j];
  const int r = __builtin_amdgcn_readfirstlane(tb.slot_row[slot]);
  if (r < 0) return;
  const int p0 = __builtin_amdgcn_readfirstlane(tb.first[r]);
  const int p1 = __builtin_amdgcn_readfirstlane(tb.first[r + 1]);
  const int piece = piece_tokens(p1 - p0);
  const int pieces = (p1 - p0 + piece - 1) / piece;
  const int k = slot - p0 / kSlotUnit;
  const int q0 = p0 + k * piece;
  const int q1 = q0 + piece < p1 ? q0 + piece : p1;
  const int per = (q1 - q0 + 3) / 4;               // a wave's tokens
  const int w0 = __builtin_amdgcn_readfirstlane(q0 + w * per < q1 ? q0 + w * per
                                                                  : q1);
  const int w1 = w0 + per < q1 ? w0 + per : q1;
  float acc[VEC];
  sum_tokens<T, VEC>(from, tb.order, w0, w1, width, lane, acc);
#pragma unroll
  for (int i = 0; i < VEC; ++i) red[w][lane * VEC + i] = acc[i];
  __syncthreads();
  for (int i = threadIdx.x; i < cols && c0 + i < width; i += 256) {
    const float x = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    if (pieces == 1)
      static_cast<T*>(tb.out)[(long)place_id(tb, r) * width + c0 + i] =
          from_f32<T>(x * tb.scale);
    else
      tb.part[(long)slot * width + c0 + i] = x;
  }
}

// Rows of more than one piece: the pieces' sums, in their order.  A block
// takes 64 columns, a wave a quarter of the pieces.  5 us: a launch.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(GradArgs a,
                                                         int width) {
  __shared__ float red[4][kWave];
  const GradTable& tb = a.t[blockIdx.y];
  const int r = tb.join_row[blockIdx.x];
  if (r < 0) return;
  const int p0 = tb.first[r], p1 = tb.first[r + 1];
  const int piece = piece_tokens(p1 - p0);
  const int pieces = (p1 - p0 + piece - 1) / piece;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = threadIdx.x / kWave;
  const int c = blockIdx.z * kWave + lane;
  const int per = (pieces + 3) / 4;
  const int k1 = (w + 1) * per < pieces ? (w + 1) * per : pieces;
  const float* part = tb.part + (long)(p0 / kSlotUnit) * width;
  float x = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int k = w * per; k < k1; ++k) x += part[(long)k * width + c];
  }
  red[w][lane] = x;
  __syncthreads();
  if (w == 0 && c < width)
    static_cast<T*>(tb.out)[(long)place_id(tb, r) * width + c] = from_f32<T>(
        ((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane])) *
        tb.scale);
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
  const long blocks = std::min<long>((n + tokens - 1) / tokens, 1 << 20);
  embed_fwd_kernel<T, VEC><<<(unsigned)blocks, 256, 0, s>>>(
      a, static_cast<T*>(y.data_ptr()), n, width, nvec, (uint32_t)mul, sh,
      (int)tokens);
}

template <typename T, int VEC>
void launch_grad(const GradArgs& a, const at::Tensor& dy, int width,
                 unsigned blocks, hipStream_t s) {
  // even shares of the columns: 768 in two of 384, not 512 and 256
  const int most = kWave * VEC;
  const int parts = (width + most - 1) / most;
  const int cols = ((width + parts - 1) / parts + VEC - 1) / VEC * VEC;
  embed_grad_kernel<T, VEC><<<dim3(blocks, (unsigned)parts), 256, 0, s>>>(
      a, static_cast<const T*>(dy.data_ptr()), width, cols);
  // a row has more than one piece only among more tokens than that
  if (dy.size(0) > kPiece)
    embed_join_kernel<T><<<dim3((unsigned)a.joins, (unsigned)a.n,
                                (unsigned)((width + kWave - 1) / kWave)),
                           256, 0, s>>>(a, width);
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
  TORCH_CHECK(width <= (1 << 21), "embedding: a row is too wide");
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

namespace {

// The buckets of a table of so many rows (log2), and the ids of each: 256
// buckets, more where a bucket's counts would not fit a block's LDS.
struct Buckets {
  int lg;
  long own;
  explicit Buckets(long rows) : lg(0) {
    while ((1l << lg) < rows && (lg < 8 || (rows >> lg) >= kMaxOwn)) ++lg;
    own = std::max<long>((rows + (1l << lg) - 1) >> lg, 1);
  }
  long places() const { return own << lg; }
  long light_blocks() const {
    return (places() + 4 * kLightRows - 1) / (4 * kLightRows);
  }
};

}  // namespace

// Whether the gradient of such a lookup can be taken: what the lookup itself
// has no reason to refuse is refused before it, not in the backward pass.
void embed_check_grad(int64_t n, int64_t width, at::IntArrayRef rows) {
  TORCH_CHECK_VALUE(width <= (1 << 21) && n <= (1 << 30),
                    "embedding_sum: a gradient of ", n, " tokens of ", width,
                    " is too large");
  long blocks = (long)rows.size() * (n / kSlotUnit + 1);
  for (const int64_t r : rows) {
    TORCH_CHECK_VALUE(r >= 0 && r < (1l << (2 * kMaxSplit)),
                      "embedding_sum: a table with a gradient has under 2^22 "
                      "rows, got ", r);
    blocks += Buckets(r).light_blocks();
  }
  // a grid has under 2^32 threads in x
  TORCH_CHECK_VALUE(blocks < (1l << 24),
                    "embedding_sum: too many tokens, or too large tables, for "
                    "a gradient");
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
  embed_check_grad(n, width, rows);
  const long slots = n / kSlotUnit + 1;
  const long joins = n / kPiece + 1;
  std::vector<at::Tensor> hold, out;
  GradArgs a{};
  a.n = (int)nt;
  a.slots = (int)slots;
  a.joins = (int)joins;
  long buckets = 0, light_blocks = 0, most = 1, ints = 0, at[kMaxTables];
  // Tables of few rows first, whatever their order in the call: they have the
  // longest buckets, whose blocks should not begin last.  embed_order of 16384
  // tokens in tables of 30528, 512 and 2 rows: 10.6 to 11.1 us in any order of
  // the call, by the call's own 10.3 to 13.3; the whole gradient of 4096 tokens
  // in them 32 us, in the call's order 35 to 36.5.
  size_t by_rows[kMaxTables];
  for (size_t j = 0; j < nt; ++j) {
    check_ids(ids_in[j], dy, n);
    out.push_back(at::empty({rows[j], width}, dy.options()));
    by_rows[j] = j;
  }
  std::sort(by_rows, by_rows + nt, [&](size_t x, size_t y) {
    return rows[x] != rows[y] ? rows[x] < rows[y] : x < y;
  });
  for (size_t k = 0; k < nt; ++k) {
    const size_t j = by_rows[k];
    GradTable& t = a.t[k];
    t.rows = (int)rows[j];
    const Buckets split(rows[j]);
    const int lg = split.lg;
    most = std::max(most, std::max(split.own, 1l << lg));
    t.own = (int)split.own;
    t.lg = lg;
    t.bucket0 = (int)buckets;
    buckets += 1l << lg;
    t.light0 = (int)light_blocks;
    light_blocks += split.light_blocks();
    if (!ids_in[j].is_contiguous()) hold.push_back(ids_in[j].contiguous());
    t.ids = (ids_in[j].is_contiguous() ? ids_in[j] : hold.back()).data_ptr();
    t.ids64 = ids_in[j].scalar_type() == at::kLong;
    t.scale = (float)scales[j];
    t.out = out[j].data_ptr();
    // all tables' lists in one piece of memory, each from a 16-byte border
    const long g = n > kDirect ? 1l << lg : 0, m = n > kDirect ? n : 0;
    at[k] = ints;
    ints += (g * kChunks + 2 * m + n + g + 1 + split.places() + 1 + slots +
             joins + 3) / 4 * 4;
  }
  if (width == 0) return out;
  if (n == 0) {
    for (auto& o : out) o.zero_();
    return out;
  }
  // the lists, then the pieces' sums
  const auto work = at::empty({ints + (long)nt * slots * width},
                              dy.options().dtype(at::kInt));
  float* part = reinterpret_cast<float*>(work.data_ptr<int>() + ints);
  const bool direct = n <= kDirect;
  for (size_t j = 0; j < nt; ++j) {
    GradTable& t = a.t[j];
    const long g = direct ? 0 : 1l << t.lg, m = direct ? 0 : n;
    t.count = work.data_ptr<int>() + at[j];    // read 16 bytes at a time
    t.loose = reinterpret_cast<int2*>(t.count + g * kChunks);
    t.order = t.count + g * kChunks + 2 * m;
    t.start = t.order + n;
    t.first = t.start + g + 1;
    t.slot_row = t.first + ((long)t.own << t.lg) + 1;
    t.join_row = t.slot_row + slots;
    t.part = part + (long)j * slots * width;
  }
  const long blocks = (long)nt * slots + light_blocks;
  auto s = at::cuda::getCurrentCUDAStream();
  const size_t lds = ((size_t)kSortWaves * (most + 2)) * sizeof(int);
  if (direct) {
    embed_order_kernel<true>
        <<<(unsigned)buckets, kSortThreads, lds, s>>>(a, (int)n);
  } else {
    const long chunk = std::max<long>(
        kSortThreads, (n + kChunks - 1) / kChunks + kSortThreads - 1) /
        kSortThreads * kSortThreads;
    const long chunks = (n + chunk - 1) / chunk;
    const dim3 by_chunk((unsigned)chunks, (unsigned)nt);
    embed_count_kernel<<<by_chunk, kSortThreads, 0, s>>>(a, (int)n, (int)chunk);
    embed_scatter_kernel<<<by_chunk, kSortThreads, lds, s>>>(
        a, (int)n, (int)chunk, (int)chunks);
    embed_order_kernel<false>
        <<<(unsigned)buckets, kSortThreads, lds, s>>>(a, (int)n);
  }
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

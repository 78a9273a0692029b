// Attention inside documents that lie one behind the other, and its
// gradients.
//
//   s_ij = scale q_i . k_j - slope_h |i - j|     i, j of the same document
//   p_ij = exp(s_ij) / sum_j exp(s_ij)           o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i                       D_i = do_i . o_i
//   ds_ij = p_ij (do_i . v_j - D_i)
//   dq_i = scale sum_j ds_ij k_j                 dk_j = scale sum_i ds_ij q_i
//
// Documents are given by their borders (cu_seqlens); a tile begins where its
// document does, so no tile holds two of them, what a document holds (NaN
// too) never reaches another, and only a document's last tile has a mask.
// Tokens in front of the first border and behind the last get zeros.
//
// Every product runs on 32x32x16 matrix instructions with the transposed
// result: in S^T = K Q^T a lane holds one query, so the softmax of a row is
// its lane's own but for one exchange with lane ^ 32, and the registers of
// P^T are at once operand B of O^T = V^T P^T (mfma_tile.h).  The gradient of
// keys and values takes S = Q K^T instead, a lane holding one key.  P is
// rounded to the inputs' type for the second product, as its other operand
// is, and so is ds (in two parts where documents are short, kFine; scaled in
// fp16, kPUp); maxima, sums and all accumulators are fp32.  D takes o in twice
// the bits (a training forward writes what rounding leaves of it): with the
// rounded o alone, gradients are off by up to 1.57 times what rounding the
// exact ones costs (where values have a large part in common by much more), so
// by 1.41.  A pass over 16384 packed tokens takes 185 us instead of 181; with
// that part in a byte, 190.
//
// No atomics: dq comes from a pass over keys, dk and dv from a pass over
// queries, each with its own recomputation of P (two products of seven).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>

#include "mfma_tile.h"

namespace dlx {

namespace {

constexpr int kKeys = 64;             // rows of an LDS tile
constexpr float kLog2e = 1.4426950408889634f;
// Tokens to a document from which blocks have eight waves instead of four,
// which halves what each query (or key) reads but leaves short documents
// waves without rows.  us, four / eight, 16384 tokens in documents of 512,
// 1024, 4096: forward of 12 heads of 64 52 / 50, 88 / 78, 259 / 240; of 8
// heads of 128 52 / 70, 85 / 84, 290 / 269; gradients of those 166 / 224,
// 273 / 269, 919 / 857, of the narrow ones 141 / 176, 231 / 255, 744 / 745,
// which stay with four.
constexpr int kWide = 1024;
// Tokens of a document up to which P and dS are taken in two parts of the
// inputs' type, and tokens of a call up to which they are in all of it (where
// launches, not products, take the time).  In one part, with few terms to even
// out its rounding, it leaves dq and dk off by 1.5 (at worst 2.3) times what
// rounding the exact ones costs, in two by 1.0; in long documents one leaves
// 1.41.  The second part costs 32 x 128 and 16384 packed tokens nothing that
// shows (14 -> 14.7 us of the forward's 32 x 128).
constexpr int kFine = 64, kFineAll = 1024;
constexpr float kLazy = 8.f;          // P stays under 2^8
// fp16 ends at 6e-8.  dS is about gradient / tokens, so gradients of 1e-3 over
// 4096 tokens left dq and dk off by 8 times what rounding the exact ones costs
// (gradients of 1: 1.4), a dS past 65504 was infinite, and of 60000 tokens P
// itself is down there.  So fp16's gradients take P, which is at most 1, times
// 2^14, and dP - D times a power of two (`up`) that each query (key) holds on
// to until one grows past it.  That costs 3 to 7 % (16384 tokens in documents
// of 512, 12 heads of 64, slopes: 194 -> 202 us; 8192 of 16 heads of 128 on
// four: 1235 -> 1316).
constexpr int kPUp = 14;
constexpr float kPDown = 1.f / (1 << kPUp);
constexpr float kUp0 = 0x1p46f;       // where `up` begins: it only falls

__device__ const uint4 g_zero16 = {0, 0, 0, 0};

struct View {                         // [tokens, heads, dim]
  uint16_t* p;
  long token, head;                   // strides, in elements
};

struct AttnArgs {
  View q, k, v, o, dout, dq, dk, dv;
  uint16_t* low;                      // [tokens, heads, dim]: what o leaves
  float* lse;                         // [heads, tokens], base 2
  int fine;                           // tokens: P and dS in two parts
  float* delta;                       // [heads, tokens]
  const int* cu;
  const float* slopes;                // [heads] or none
  float* part;                        // dk, dv: [2, splits, tokens, kv_heads,
                                      // dim] where the walk is split
  int docs, tokens, heads, group, dim, splits;
  float scale;
};

// Border e of the documents with what lies in front of and behind them:
// 0, cu[0], .., cu[docs], tokens.  Clamped, so that no border, whatever the
// caller's array holds, leads out of the tokens.
DLX_DEV int border(const AttnArgs& a, int e) {
  if (e == 0) return 0;
  if (e == a.docs + 2) return a.tokens;
  const int c = a.cu[e - 1];
  return c < 0 ? 0 : c > a.tokens ? a.tokens : c;
}

struct Tile {
  int start, len, row0;               // document, first row of the tile in it
  bool doc;                           // false: in no document
};

// Tile t of ROWS rows.  Document e's tiles are numbered from
// border(e) / ROWS + e, which leaves each at least as many as it has rows
// for; the tiles it does not need are empty (row0 >= len).
template <int ROWS> DLX_DEV Tile find_tile(const AttnArgs& a, int t) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, n = a.docs + 2;         // the document is one of lo..lo+n-1
  Tile x;
  while (true) {
    const int step = (n + kWave - 1) / kWave;
    const int e = lo + lane * step;
    // one border more than there are documents, where a lane is left for it
    const int at = border(a, e < a.docs + 2 ? e : a.docs + 2);
    const uint64_t in = __ballot(lane * step < n && at / ROWS + e <= t);
    int c = __popcll(in);
    c = c < 1 ? 1 : c;
    lo = __builtin_amdgcn_readfirstlane(lo + (c - 1) * step);
    if (step == 1) {
      x.start = __builtin_amdgcn_readlane(at, c - 1);
      x.len = (c < kWave ? __builtin_amdgcn_readlane(at, c)
                         : __builtin_amdgcn_readfirstlane(border(a, lo + 1))) -
              x.start;
      break;
    }
    const int left = n - (c - 1) * step;
    n = left < step ? left : step;
  }
  x.row0 = (t - (x.start / ROWS + lo)) * ROWS;
  x.doc = lo > 0 && lo <= a.docs;
  if (x.row0 < 0) x.row0 = x.len < 0 ? 0 : x.len;
  return x;
}

// Rows row0.. of a document into an LDS tile; rows behind its end repeat the
// last one, chunks behind the head's width are zero.
template <int DP, int NT>
DLX_DEV void load_tile(uint16_t* lds, const uint16_t* base, long stride,
                       int row0, int len, int dim) {
  constexpr int CH = DP / 8;
#pragma unroll
  for (int u = 0; u < kKeys * CH / NT; ++u) {
    const int f = u * NT + threadIdx.x;
    const int row = f / CH;
    const int chunk = (f % CH) ^ swizzle<DP>(row);
    const int r = row0 + row < len ? row0 + row : len - 1;
    const void* src = base + r * stride + chunk * 8;
    if (chunk * 8 >= dim) src = &g_zero16;
    copy16_to_lds(src, lds + f * 8);
  }
}

// Operand B of a wave's 32 rows, from memory.
template <int DP>
DLX_DEV void load_rows(s16x8* f, const uint16_t* row, int dim, int lane) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = (s * 2 + (lane >> 5)) * 8;
    f[s] = c < dim ? *reinterpret_cast<const s16x8*>(row + c) : s16x8{};
  }
}

// A result C[d][row] to row `row`: four d at a time.
template <typename T, int DP>
DLX_DEV void store_rows(uint16_t* row, const f32x16* acc, float by, int dim,
                        int lane) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = b * 32 + g * 8 + (lane >> 5) * 4;
      uint2 x;
      x.x = pack2<T>(acc[b][g * 4] * by, acc[b][g * 4 + 1] * by);
      x.y = pack2<T>(acc[b][g * 4 + 2] * by, acc[b][g * 4 + 3] * by);
      if (d < dim) *reinterpret_cast<uint2*>(row + d) = x;
    }
}

// What store_rows leaves of the same numbers, as numbers of the type.
template <typename T, int DP>
DLX_DEV void store_low(uint16_t* row, const f32x16* acc, float by, int dim,
                       int lane) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = b * 32 + g * 8 + (lane >> 5) * 4;
      float r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = acc[b][g * 4 + e] * by;
        r[e] = x - to_f32<T>(from_f32<T>(x));
      }
      uint2 x;
      x.x = pack2<T>(r[0], r[1]);
      x.y = pack2<T>(r[2], r[3]);
      if (d < dim) *reinterpret_cast<uint2*>(row + d) = x;
    }
}

template <int DP>
DLX_DEV void zero_rows(const View& v, long token, int head, int dim, int lane) {
  uint16_t* row = v.p + token * v.token + head * v.head;
  for (int c = (lane >> 5) * 8; c < dim; c += 16)
    *reinterpret_cast<s16x8*>(row + c) = s16x8{};
}

// register i of a result: its row of 32
DLX_DEV constexpr int reg_row(int i) { return 8 * (i >> 2) + (i & 3); }

// A head's slope in units of the scores before their scale.  A finite one stays
// finite: infinity times a distance of 0 would be NaN, where nothing is taken
// off.
DLX_DEV float slope_of(const AttnArgs& a, int head) {
  const float s = a.slopes[head], x = s / a.scale;
  return isinf(x) && !isinf(s) ? copysignf(3.402823466e38f, s) : x;
}

// What a block of scores begins at: -sl |key - query|, keys k0 + .., queries
// wave_row ..+31, shift = 4 * (lane >> 5) - query.  Where the block lies on
// one side of the diagonal the sign is known, and a register takes one fma.
DLX_DEV f32x16 bias(float sl, int k0, int wave_row, int shift) {
  f32x16 s;
  const float d0 = (float)(k0 + shift);
  if (k0 >= wave_row + 31) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = fmaf(-sl, (float)reg_row(i), -sl * d0);
  } else if (k0 + 31 <= wave_row) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fmaf(sl, (float)reg_row(i), sl * d0);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = -sl * fabsf(d0 + (float)reg_row(i));
  }
  return s;
}

// ---------------------------------------------------------------------------
// forward: a wave owns 32 queries, a block NW waves; keys and values pass in
// tiles of 64, the next one on its way while this one is worked on.
// Bound by exp and the rest of the softmax: of the cycles of a SIMD vector
// instructions take 82 % and matrix instructions, beside them, 41 %.  2 x 8192
// tokens, 12 heads of 64, slopes: 530 us (0.78 PFLOP/s); 16384 packed tokens
// in documents up to 512: 52 us; 8192 tokens of 16 heads of 128: 275 us.
// ---------------------------------------------------------------------------

template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, DP == 64 ? 4 : 2) void doc_attn_fwd_kernel(AttnArgs a) {
  constexpr int NT = NW * 64, ROWS = NW * 32, TS = kKeys * DP;
  __shared__ __attribute__((aligned(16))) uint16_t lds[4 * TS];

  const int tiles = gridDim.x / a.heads;
  const int bid = xcd_block(blockIdx.x, gridDim.x);
  const int head = bid / tiles;
  const Tile tl = find_tile<ROWS>(a, bid - head * tiles);
  if (tl.row0 >= tl.len) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane >> 5;
  const int wave_row = tl.row0 + wid * 32;
  const bool mine = wave_row < tl.len;   // else this wave only moves tiles
  const int qpos = wave_row + (lane & 31);
  const bool real = qpos < tl.len;
  if (!tl.doc) {
    if (real) zero_rows<DP>(a.o, tl.start + qpos, head, a.dim, lane);
    return;
  }
  const int kvh = head / a.group;
  const uint16_t* kb = a.k.p + tl.start * a.k.token + kvh * a.k.head;
  const uint16_t* vb = a.v.p + tl.start * a.v.token + kvh * a.v.head;
  const long token = tl.start + (real ? qpos : tl.len - 1);

  const int nt = (tl.len + kKeys - 1) / kKeys;
  load_tile<DP, NT>(lds, kb, a.k.token, 0, tl.len, a.dim);
  load_tile<DP, NT>(lds + TS, vb, a.v.token, 0, tl.len, a.dim);
  s16x8 qf[DP / 16];
  load_rows<DP>(qf, a.q.p + token * a.q.token + head * a.q.head, a.dim, lane);

  const Frags<DP> fr(lds, lane);
  const float sc = a.scale * kLog2e;
  const float sl = BIAS ? slope_of(a, head) : 0.f;
  // m: what the row's exponents are taken next to; it follows the row's
  // maximum only when that is past it by 2^kLazy, which spares the products
  // their rescaling in nearly every tile.  ms: m, or 0 in a row of -inf.
  float m = -INFINITY, ms = 0.f, l = 0.f;
  f32x16 acc[DP / 32] = {};

  auto body = [&](int t, auto half_, auto fine_) {
    constexpr bool FINE = decltype(fine_)::value;
    constexpr int LK = decltype(half_)::value * 2 * TS, LV = LK + TS;
    uint16_t* nx = lds + (2 * TS - LK);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + 1 < nt) {
      load_tile<DP, NT>(nx, kb, a.k.token, (t + 1) * kKeys, tl.len, a.dim);
      load_tile<DP, NT>(nx + TS, vb, a.v.token, (t + 1) * kKeys, tl.len, a.dim);
    }
    if (!mine) return;
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = BIAS ? bias(sl, t * kKeys + b * 32, wave_row, half * 4 - qpos)
                  : f32x16{};
    }
    // two sums in turn: a product does not wait for the one before it
#pragma unroll
    for (int st = 0; st < DP / 16; ++st)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = mfma32<T>(fr.row(LK + b * 32 * DP, st), qf[st], s[b]);
    if ((t + 1) * kKeys > tl.len) {
      const int k0 = t * kKeys + half * 4;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + b * 32 + reg_row(i) >= tl.len) s[b][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    mx *= sc;
    if (__ballot(mx > m + kLazy)) {
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float mn = fmaxf(m, mx);
      const float by =
          mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      ms = m == -INFINITY ? 0.f : m;
      l *= by;
#pragma unroll
      for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= by;
    }
    unroll<4>([&](auto n) {                     // 16 keys at a time
      constexpr int b = n / 2, st = n % 2;
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(s[b][st * 8 + e] * sc - ms);
        l += p[e];
      }
      const s16x8 pf = pack_step<T>(p);
      s16x8 vf[DP / 32];
      fr.template tr<DP / 32, LV + n * 16 * DP>(vf);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
        acc[db] = mfma32<T>(vf[db], pf, acc[db]);
      if constexpr (FINE) {
        const s16x8 rest = pack_rest<T>(p, pf);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = mfma32<T>(vf[db], rest, acc[db]);
      }
    });
  };
  // two tiles a turn, so that each half of LDS has its own addresses
  auto walk = [&](auto fine) {
    for (int t = 0; t < nt; t += 2) {
      body(t, std::integral_constant<int, 0>{}, fine);
      if (t + 1 < nt) body(t + 1, std::integral_constant<int, 1>{}, fine);
    }
  };
  if (tl.len <= a.fine) walk(std::true_type{});
  else walk(std::false_type{});
  l += __shfl_xor(l, 32, kWave);
  if (!real) return;
  store_rows<T, DP>(a.o.p + token * a.o.token + head * a.o.head, acc, 1.f / l,
                    a.dim, lane);
  if (a.lse) {
    store_low<T, DP>(a.low + (token * a.heads + head) * a.dim, acc, 1.f / l,
                     a.dim, lane);
    if (half == 0) a.lse[(long)head * a.tokens + token] = m + log2f(l);
  }
}

template <typename T> constexpr bool kHalf = std::is_same_v<T, FP16>;

// Whether one of a wave's dP - D, times its `up`, is past 1, and what up and all
// that was summed are multiplied by then to have 2^6 of room again (1 in lanes
// that need none): times a P of at most 2^14 it stays in fp16.  Lanes l and
// l ^ 32 hold one query (key).
DLX_DEV bool lower(const f32x16& dp, float up, float& f) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(dp[i]));
  mx *= up;
  if (!__ballot(mx > 1.f)) return false;
  const uint32_t x = __builtin_bit_cast(uint32_t, mx);
  const auto both = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const uint32_t top = both[0] > both[1] ? both[0] : both[1];  // not negative
  // to 2^-6 .. 2^-5; infinity stays what it is
  f = top > 0x3f800000u && top < 0x7f800000u
          ? __builtin_bit_cast(float, (127u - 6u + 127u - (top >> 23)) << 23)
          : 1.f;
  return true;
}

// What exp2 takes off for P times 2^kPUp and up.
DLX_DEV float scaled(float lse, float up) {
  return lse -
         (float)(kPUp - 127 + (int)(__builtin_bit_cast(uint32_t, up) >> 23));
}

// ---------------------------------------------------------------------------
// gradient of the queries: the forward's walk over the keys, a third product.
// Also writes delta, which the next kernel reads.  The same packed tokens:
// 60 us; the same 16 heads of 128 on four key heads: 370 us, registers leaving
// two waves to a SIMD.
// ---------------------------------------------------------------------------

template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, DP == 64 ? 3 : 2) void doc_attn_dq_kernel(AttnArgs a) {
  constexpr int NT = NW * 64, ROWS = NW * 32, TS = kKeys * DP;
  __shared__ __attribute__((aligned(16))) uint16_t lds[4 * TS];

  const int tiles = gridDim.x / a.heads;
  const int bid = xcd_block(blockIdx.x, gridDim.x);
  const int head = bid / tiles;
  const Tile tl = find_tile<ROWS>(a, bid - head * tiles);
  if (tl.row0 >= tl.len) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane >> 5;
  const int wave_row = tl.row0 + wid * 32;
  const bool mine = wave_row < tl.len;   // else this wave only moves tiles
  const int qpos = wave_row + (lane & 31);
  const bool real = qpos < tl.len;
  if (!tl.doc) {
    if (real) zero_rows<DP>(a.dq, tl.start + qpos, head, a.dim, lane);
    return;
  }
  const int kvh = head / a.group;
  const uint16_t* kb = a.k.p + tl.start * a.k.token + kvh * a.k.head;
  const uint16_t* vb = a.v.p + tl.start * a.v.token + kvh * a.v.head;
  const long token = tl.start + (real ? qpos : tl.len - 1);

  const int nt = (tl.len + kKeys - 1) / kKeys;
  load_tile<DP, NT>(lds, kb, a.k.token, 0, tl.len, a.dim);
  load_tile<DP, NT>(lds + TS, vb, a.v.token, 0, tl.len, a.dim);
  s16x8 qf[DP / 16], gf[DP / 16];
  load_rows<DP>(qf, a.q.p + token * a.q.token + head * a.q.head, a.dim, lane);
  load_rows<DP>(gf, a.dout.p + token * a.dout.token + head * a.dout.head,
                a.dim, lane);
  float delta = 0.f;
  {
    s16x8 of[DP / 16], lf[DP / 16];
    load_rows<DP>(of, a.o.p + token * a.o.token + head * a.o.head, a.dim, lane);
    load_rows<DP>(lf, a.low + (token * a.heads + head) * a.dim, a.dim, lane);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta += to_f32<T>(T{(uint16_t)gf[s][e]}) *
                 (to_f32<T>(T{(uint16_t)of[s][e]}) +
                  to_f32<T>(T{(uint16_t)lf[s][e]}));
    delta += __shfl_xor(delta, 32, kWave);
  }
  if (real && half == 0) a.delta[(long)head * a.tokens + token] = delta;
  const float lse0 = a.lse[(long)head * a.tokens + token];
  float up = kHalf<T> ? kUp0 : 1.f;
  float lse = kHalf<T> ? scaled(lse0, up) : lse0;   // P comes out times both
  const Frags<DP> fr(lds, lane);
  const float sc = a.scale * kLog2e;
  const float sl = BIAS ? slope_of(a, head) : 0.f;
  f32x16 acc[DP / 32] = {};
  f32x16 less;                        // what dP begins at: dP - D for nothing
#pragma unroll
  for (int i = 0; i < 16; ++i) less[i] = -delta;

  auto body = [&](int t, auto half_, auto fine_) {
    constexpr int LK = decltype(half_)::value * 2 * TS, LV = LK + TS;
    constexpr bool FINE = decltype(fine_)::value;
    uint16_t* nx = lds + (2 * TS - LK);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + 1 < nt) {
      load_tile<DP, NT>(nx, kb, a.k.token, (t + 1) * kKeys, tl.len, a.dim);
      load_tile<DP, NT>(nx + TS, vb, a.v.token, (t + 1) * kKeys, tl.len, a.dim);
    }
    if (!mine) return;
    unroll<2>([&](auto b) {
      f32x16 s = BIAS ? bias(sl, t * kKeys + b * 32, wave_row, half * 4 - qpos)
                      : f32x16{};
      f32x16 dp = less;
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        s = mfma32<T>(fr.row(LK + b * 32 * DP, st), qf[st], s);
        dp = mfma32<T>(fr.row(LV + b * 32 * DP, st), gf[st], dp);
      }
      if constexpr (kHalf<T>) {
        float f;
        if (lower(dp, up, f)) {
          up *= f;
          lse = scaled(lse0, up);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db) acc[db] *= f;
        }
      }
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        ds[i] = __builtin_amdgcn_exp2f(s[i] * sc - lse) * dp[i];
      if ((t + 1) * kKeys > tl.len) {
        const int k0 = t * kKeys + b * 32 + half * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + reg_row(i) >= tl.len) ds[i] = 0.f;
      }
      unroll<2>([&](auto st) {
        const s16x8 df = pack_step<T>(&ds[st * 8]);
        s16x8 kf[DP / 32];
        fr.template tr<DP / 32, LK + (b * 2 + st) * 16 * DP>(kf);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = mfma32<T>(kf[db], df, acc[db]);
        if constexpr (FINE) {
          const s16x8 rest = pack_rest<T>(&ds[st * 8], df);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db)
            acc[db] = mfma32<T>(kf[db], rest, acc[db]);
        }
      });
    });
  };
  auto walk = [&](auto fine) {
    for (int t = 0; t < nt; t += 2) {
      body(t, std::integral_constant<int, 0>{}, fine);
      if (t + 1 < nt) body(t + 1, std::integral_constant<int, 1>{}, fine);
    }
  };
  if (tl.len <= a.fine) walk(std::true_type{});
  else walk(std::false_type{});
  if (real)             // of one score p is 1: nothing depends on q or k
    store_rows<T, DP>(a.dq.p + token * a.dq.token + head * a.dq.head, acc,
                      tl.len == 1 ? 0.f
                                  : a.scale * (kHalf<T> ? kPDown : 1.f) / up,
                      a.dim, lane);
}

// ---------------------------------------------------------------------------
// gradients of keys and values: a wave owns 32 keys of one key head; the
// queries of every head that shares it pass in tiles of 64.  Shared heads
// leave few such waves and give each a long walk: then the walk is split, its
// parts' sums stay in fp32 and doc_attn_join_kernel adds them, in their order.
// The same packed tokens: 77 us; the same 16 heads, in
// fp16 (kPUp): 570 us and 23 to join.
// ---------------------------------------------------------------------------

template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, DP == 64 ? 3 : 2) void doc_attn_dkv_kernel(AttnArgs a) {
  constexpr int NT = NW * 64, ROWS = NW * 32, TS = kKeys * DP;
  __shared__ __attribute__((aligned(16))) uint16_t lds[4 * TS];
  __shared__ __attribute__((aligned(16))) float stat[2][2][kKeys];

  const int kv_heads = a.heads / a.group;
  const int tiles = gridDim.x / (kv_heads * a.splits);
  const int bid = xcd_block(blockIdx.x, gridDim.x);
  const int kvh = bid / (tiles * a.splits);
  const int split = (bid - kvh * tiles * a.splits) / tiles;
  const Tile tl = find_tile<ROWS>(a, bid % tiles);
  if (tl.row0 >= tl.len) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane >> 5;
  const bool mine = tl.row0 + wid * 32 < tl.len;
  const int kpos = tl.row0 + wid * 32 + (lane & 31);
  const bool real = kpos < tl.len;
  const long half_part = (long)a.splits * a.tokens * kv_heads * a.dim;
  auto part_row = [&](long t) {
    return a.part + (((long)split * a.tokens + t) * kv_heads + kvh) * a.dim;
  };
  if (!tl.doc) {
    if (real && a.splits > 1) {
      float* row = part_row(tl.start + kpos);
      for (int c = half; c < a.dim; c += 2) row[c] = row[half_part + c] = 0.f;
    } else if (real) {
      zero_rows<DP>(a.dk, tl.start + kpos, kvh, a.dim, lane);
      zero_rows<DP>(a.dv, tl.start + kpos, kvh, a.dim, lane);
    }
    return;
  }
  const long token = tl.start + (real ? kpos : tl.len - 1);
  const int nt = (tl.len + kKeys - 1) / kKeys;
  const int n0 = (int)((long)nt * a.group * split / a.splits);
  const int n1 = (int)((long)nt * a.group * (split + 1) / a.splits);

  const float sc = a.scale * kLog2e, unit = 1.f / sc;

  // tile n of the walk: head kvh * group + n / nt, rows (n % nt) * 64..
  auto stage = [&](int n, uint16_t* at, float (*st)[kKeys]) {
    const int head = kvh * a.group + n / nt;
    const int row0 = (n % nt) * kKeys;
    load_tile<DP, NT>(at, a.q.p + tl.start * a.q.token + head * a.q.head,
                      a.q.token, row0, tl.len, a.dim);
    load_tile<DP, NT>(at + TS,
                      a.dout.p + tl.start * a.dout.token + head * a.dout.head,
                      a.dout.token, row0, tl.len, a.dim);
    if (threadIdx.x < kKeys) {
      // what S and dP begin at; behind the document's end exp2(-inf) is 0
      const int r = row0 + threadIdx.x;
      const long i = (long)head * a.tokens + tl.start + r;
      st[0][threadIdx.x] =
          r < tl.len ? (a.lse[i] - (kHalf<T> ? kPUp : 0)) * -unit : -INFINITY;
      st[1][threadIdx.x] = r < tl.len ? -a.delta[i] : 0.f;
    }
  };
  if (n0 < n1) stage(n0, lds, stat[0]);
  s16x8 kf[DP / 16], vf[DP / 16];
  load_rows<DP>(kf, a.k.p + token * a.k.token + kvh * a.k.head, a.dim, lane);
  load_rows<DP>(vf, a.v.p + token * a.v.token + kvh * a.v.head, a.dim, lane);
  const Frags<DP> fr(lds, lane);
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  float up = kUp0;                      // fp16's

  // REST: what rounding P and dS has left, in a turn of its own over the same
  // tile (in the first one it would need registers that are not there)
  auto turn = [&](int n, auto half_, auto rest_) {
    constexpr int H = decltype(half_)::value;
    constexpr bool REST = decltype(rest_)::value;
    constexpr int LQ = H * 2 * TS, LG = LQ + TS;
    const float (*st_)[kKeys] = stat[H];
    int place = kpos;                  // nothing of the first turn is kept
    if (REST) asm volatile("" : "+v"(place)::"memory");
    const float sl = BIAS ? slope_of(a, kvh * a.group + n / nt) : 0.f;
    unroll<2>([&](auto b) {
      const int q0 = b * 32 + half * 4;
      const float d0 = (float)((n % nt) * kKeys + q0 - place);
      f32x16 s, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const F32x4 ls = *reinterpret_cast<const F32x4*>(&st_[0][q0 + g * 8]);
        const F32x4 de = *reinterpret_cast<const F32x4*>(&st_[1][q0 + g * 8]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[g * 4 + e] = ls.v[e];
          if (BIAS) s[g * 4 + e] -= sl * fabsf(d0 + (float)(g * 8 + e));
          dp[g * 4 + e] = de.v[e];
        }
      }
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        s = mfma32<T>(fr.row(LQ + b * 32 * DP, st), kf[st], s);
        dp = mfma32<T>(fr.row(LG + b * 32 * DP, st), vf[st], dp);
      }
      if constexpr (kHalf<T>) {
        float f;
        // the second turn finds what the first has made room for
        if (!REST && lower(dp, up, f)) {
          up *= f;
#pragma unroll
          for (int db = 0; db < DP / 32; ++db) dk[db] *= f;
        }
      }
      unroll<2>([&](auto st) {
        float p[8], ds[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(s[st * 8 + e] * sc);
          ds[e] = p[e] * dp[st * 8 + e];
          if (kHalf<T>) ds[e] *= up;
        }
        s16x8 pf = pack_step<T>(p), df = pack_step<T>(ds);
        if (REST) {
          pf = pack_rest<T>(p, pf);
          df = pack_rest<T>(ds, df);
        }
        constexpr int at = (b * 2 + st) * 16 * DP;
        unroll<DP / 64>([&](auto h) {           // two operands at a time
          s16x8 f[2];
          fr.template tr<2, LG + at, h * 2>(f);
          dv[h * 2] = mfma32<T>(f[0], pf, dv[h * 2]);
          dv[h * 2 + 1] = mfma32<T>(f[1], pf, dv[h * 2 + 1]);
          fr.template tr<2, LQ + at, h * 2>(f);
          dk[h * 2] = mfma32<T>(f[0], df, dk[h * 2]);
          dk[h * 2 + 1] = mfma32<T>(f[1], df, dk[h * 2 + 1]);
        });
      });
    });
  };
  auto body = [&](int n, auto half_) {
    constexpr int H = decltype(half_)::value;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (n + 1 < n1) stage(n + 1, lds + (1 - H) * 2 * TS, stat[1 - H]);
    if (!mine) return;
    turn(n, half_, std::false_type{});
    if (tl.len <= a.fine) turn(n, half_, std::true_type{});
  };
  for (int n = n0; n < n1; n += 2) {
    body(n, std::integral_constant<int, 0>{});
    if (n + 1 < n1) body(n + 1, std::integral_constant<int, 1>{});
  }
  if (!real) return;
  if (kHalf<T>) {
    const float less = kPDown / up;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
      dk[b] *= less;
      dv[b] *= kPDown;
    }
  }
  if (tl.len == 1) {    // of one score p is 1: nothing depends on q or k
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dk[b] *= 0.f;
  }
  if (a.splits > 1) {
    float* row = part_row(token);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = b * 32 + g * 8 + half * 4;
        if (d >= a.dim) continue;
        *reinterpret_cast<F32x4*>(row + d) =
            F32x4{{dk[b][g * 4], dk[b][g * 4 + 1], dk[b][g * 4 + 2],
                   dk[b][g * 4 + 3]}};
        *reinterpret_cast<F32x4*>(row + half_part + d) =
            F32x4{{dv[b][g * 4], dv[b][g * 4 + 1], dv[b][g * 4 + 2],
                   dv[b][g * 4 + 3]}};
      }
    return;
  }
  store_rows<T, DP>(a.dk.p + token * a.dk.token + kvh * a.dk.head, dk,
                    a.scale, a.dim, lane);
  store_rows<T, DP>(a.dv.p + token * a.dv.token + kvh * a.dv.head, dv, 1.f,
                    a.dim, lane);
}

// The sums of a split walk: eight columns of dk or dv a thread.
template <typename T>
__global__ __launch_bounds__(256) void doc_attn_join_kernel(AttnArgs a) {
  const int kv_heads = a.heads / a.group, chunks = a.dim / 8;
  const long rows = (long)a.tokens * kv_heads, half = rows * chunks;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * half) return;
  const bool is_v = i >= half;
  const long at = is_v ? i - half : i;
  const long row = at / chunks, token = row / kv_heads;
  const int c = (int)(at - row * chunks) * 8;
  const int head = (int)(row - token * kv_heads);
  const long stride = rows * a.dim;
  const float* p =
      a.part + (is_v ? a.splits * stride : 0) + row * a.dim + c;
  float x[8] = {};
  for (int s = 0; s < a.splits; ++s, p += stride)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += p[e];
  const float by = is_v ? 1.f : a.scale;
  const View& v = is_v ? a.dv : a.dk;
  Pack<uint32_t, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y.v[e] = pack2<T>(x[2 * e] * by, x[2 * e + 1] * by);
  *reinterpret_cast<Pack<uint32_t, 4>*>(v.p + token * v.token + head * v.head +
                                        c) = y;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// 16-byte rows at any stride: what the kernels' loads take.
bool loadable(const at::Tensor& t) {
  return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
         t.stride(0) >= 0 && t.stride(1) >= 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// A contiguous tensor that begins off a 16-byte border (cut out of a flat
// buffer) is its own contiguous(): only a copy has a place that fits.
at::Tensor rows(const at::Tensor& t) {
  if (loadable(t)) return t;
  const auto c = t.contiguous();
  return loadable(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}

View view(const at::Tensor& t) {
  return View{static_cast<uint16_t*>(t.data_ptr()), t.stride(0), t.stride(1)};
}

void check_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& cu, const c10::optional<at::Tensor>& slopes,
                  double scale) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3,
              "document_attention: q, k and v are [tokens, heads, dim]");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
              "document_attention: bf16 or fp16 only, got ", q.scalar_type());
  TORCH_CHECK(k.scalar_type() == q.scalar_type() &&
                  v.scalar_type() == q.scalar_type(),
              "document_attention: q, k and v differ in type");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) &&
                  k.size(2) == q.size(2),
              "document_attention: q/k/v shape mismatch");
  TORCH_CHECK(k.size(1) > 0 && q.size(1) % k.size(1) == 0,
              "document_attention: query heads have to be a multiple of key "
              "heads");
  TORCH_CHECK(q.size(2) % 8 == 0 && q.size(2) >= 8 && q.size(2) <= 128,
              "document_attention: the head's width has to be a multiple of 8 "
              "up to 128, got ", q.size(2));
  TORCH_CHECK(q.size(0) < (1l << 30),
              "document_attention: too many tokens");
  TORCH_CHECK(cu.dim() == 1 && cu.numel() >= 1 &&
                  cu.scalar_type() == at::kInt && cu.is_contiguous(),
              "document_attention: cu_seqlens is a contiguous int32 vector");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device() &&
                  cu.device() == q.device(),
              "document_attention: inputs on different devices");
  if (slopes)
    TORCH_CHECK(slopes->scalar_type() == at::kFloat && slopes->dim() == 1 &&
                    slopes->size(0) == q.size(1) && slopes->is_contiguous() &&
                    slopes->device() == q.device(),
                "document_attention: slopes is a float32 vector, one a head");
  TORCH_CHECK(scale >= 1e-30 && scale <= 1e30,
              "document_attention: scale has to lie between 1e-30 and 1e30");
}

void fill(AttnArgs& a, const at::Tensor& q, const at::Tensor& k,
          const at::Tensor& v, const at::Tensor& cu,
          const c10::optional<at::Tensor>& slopes, double scale) {
  a.q = view(q);
  a.k = view(k);
  a.v = view(v);
  a.cu = cu.data_ptr<int>();
  a.slopes = slopes ? slopes->data_ptr<float>() : nullptr;
  a.docs = (int)cu.numel() - 1;
  a.tokens = (int)q.size(0);
  a.heads = (int)q.size(1);
  a.group = (int)(q.size(1) / k.size(1));
  a.dim = (int)q.size(2);
  a.scale = (float)scale;
  a.fine = a.tokens <= kFineAll ? kFineAll : kFine;
}

unsigned blocks_of(const AttnArgs& a, int rows_, int heads) {
  const long n = ((long)a.tokens / rows_ + a.docs + 2) * heads;
  // a grid has under 2^32 threads, two a row
  TORCH_CHECK(n * rows_ < (1l << 31),
              "document_attention: too many tokens or documents");
  return (unsigned)n;
}

enum { kFwd, kDq, kDkv };

template <typename T, int DP, int NW, bool BIAS>
void launch_grad(int which, const AttnArgs& a, hipStream_t s) {
  const unsigned b = blocks_of(
      a, NW * 32, which == kDkv ? a.heads / a.group * a.splits : a.heads);
  if (which == kDq)
    doc_attn_dq_kernel<T, DP, NW, BIAS><<<b, NW * 64, 0, s>>>(a);
  else
    doc_attn_dkv_kernel<T, DP, NW, BIAS><<<b, NW * 64, 0, s>>>(a);
}

template <typename T, int DP, bool BIAS>
void launch_tile(int which, const AttnArgs& a, hipStream_t s) {
  const bool wide = a.tokens / (a.docs < 1 ? 1 : a.docs) >= kWide;
  if (which == kFwd) {
    if (wide)
      doc_attn_fwd_kernel<T, DP, 8, BIAS>
          <<<blocks_of(a, 256, a.heads), 512, 0, s>>>(a);
    else
      doc_attn_fwd_kernel<T, DP, 4, BIAS>
          <<<blocks_of(a, 128, a.heads), 256, 0, s>>>(a);
    return;
  }
  if constexpr (DP == 128) {
    if (wide) return launch_grad<T, DP, 8, BIAS>(which, a, s);
  }
  launch_grad<T, DP, 4, BIAS>(which, a, s);
}

template <typename T>
void launch_type(int which, const AttnArgs& a, hipStream_t s) {
  if (a.dim <= 64)
    a.slopes ? launch_tile<T, 64, true>(which, a, s)
             : launch_tile<T, 64, false>(which, a, s);
  else
    a.slopes ? launch_tile<T, 128, true>(which, a, s)
             : launch_tile<T, 128, false>(which, a, s);
}

void launch(int which, const AttnArgs& a, at::ScalarType t, hipStream_t s) {
  if (t == at::kBFloat16) launch_type<BF16>(which, a, s);
  else launch_type<FP16>(which, a, s);
}

}  // namespace

// q [T,H,D], k and v [T,Hkv,D] (rows at any stride), cu [docs+1] int32
// -> (o [T,H,D], and for the gradients: lse [H,T] fp32, base 2, and what
// rounding leaves of o [T,H,D]; both empty without need_grad)
std::tuple<at::Tensor, at::Tensor, at::Tensor> doc_attn_fwd_impl(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
    const at::Tensor& cu, const c10::optional<at::Tensor>& slopes, double scale,
    bool need_grad) {
  check_inputs(q_in, k_in, v_in, cu, slopes, scale);
  const c10::DeviceGuard guard(q_in.device());
  const auto q = rows(q_in), k = rows(k_in), v = rows(v_in);
  auto o = at::empty(q.sizes(), q.options());
  auto lse = at::empty({need_grad ? q.size(1) : 0, need_grad ? q.size(0) : 0},
                       q.options().dtype(at::kFloat));
  auto low = at::empty({need_grad ? q.size(0) : 0, q.size(1), q.size(2)},
                       q.options());
  if (q.numel() == 0) return {o, lse, low};
  AttnArgs a{};
  fill(a, q, k, v, cu, slopes, scale);
  a.o = view(o);
  a.lse = need_grad ? lse.data_ptr<float>() : nullptr;
  a.low = need_grad ? static_cast<uint16_t*>(low.data_ptr()) : nullptr;
  launch(kFwd, a, q.scalar_type(), at::cuda::getCurrentCUDAStream());
  return {o, lse, low};
}

// dq, dk, dv: written whole, rows at any stride
void doc_attn_bwd_impl(const at::Tensor& dout_in, const at::Tensor& q_in,
                       const at::Tensor& k_in, const at::Tensor& v_in,
                       const at::Tensor& o, const at::Tensor& lse,
                       const at::Tensor& low, const at::Tensor& cu,
                       const c10::optional<at::Tensor>& slopes, double scale,
                       at::Tensor dq, at::Tensor dk, at::Tensor dv) {
  check_inputs(q_in, k_in, v_in, cu, slopes, scale);
  const c10::DeviceGuard guard(q_in.device());
  TORCH_CHECK(dout_in.sizes() == q_in.sizes() &&
                  dout_in.scalar_type() == q_in.scalar_type() &&
                  dout_in.device() == q_in.device(),
              "document_attention: the gradient differs from the output");
  TORCH_CHECK(o.sizes() == q_in.sizes() && o.scalar_type() == q_in.scalar_type()
                  && loadable(o) && lse.numel() == q_in.size(0) * q_in.size(1)
                  && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  low.sizes() == o.sizes() && low.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(low.data_ptr()) % 16 == 0 &&
                  low.scalar_type() == o.scalar_type() &&
                  o.device() == q_in.device() &&
                  lse.device() == q_in.device() &&
                  low.device() == q_in.device(),
              "document_attention: o, lse and low are not the forward's");
  TORCH_CHECK(dq.sizes() == q_in.sizes() && dk.sizes() == k_in.sizes() &&
                  dv.sizes() == k_in.sizes() && loadable(dq) && loadable(dk) &&
                  loadable(dv) && dq.scalar_type() == q_in.scalar_type() &&
                  dk.scalar_type() == q_in.scalar_type() &&
                  dv.scalar_type() == q_in.scalar_type() &&
                  dq.device() == q_in.device() &&
                  dk.device() == q_in.device() && dv.device() == q_in.device(),
              "document_attention: dq, dk, dv do not fit q, k, v");
  if (q_in.numel() == 0) {
    dk.zero_();
    dv.zero_();
    return;
  }
  const auto q = rows(q_in), k = rows(k_in), v = rows(v_in);
  const auto dout = rows(dout_in);
  auto delta = at::empty({q.size(1), q.size(0)}, lse.options());
  AttnArgs a{};
  fill(a, q, k, v, cu, slopes, scale);
  a.o = view(o);
  a.dout = view(dout);
  a.dq = view(dq);
  a.dk = view(dk);
  a.dv = view(dv);
  a.low = static_cast<uint16_t*>(low.data_ptr());
  a.lse = lse.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  const auto s = at::cuda::getCurrentCUDAStream();
  launch(kDq, a, q.scalar_type(), s);
  // a wave owns 32 keys of a key head: the walk over a group's queries is
  // split until there are about four waves to each of the 1024 SIMDs
  const long waves = ((long)a.tokens / 32 + 1) * k.size(1);
  a.splits = 1;
  while (a.splits < a.group && waves * a.splits < 4096) ++a.splits;
  at::Tensor part;
  if (a.splits > 1) {
    part = at::empty({2l * a.splits * k.numel()}, lse.options());
    a.part = part.data_ptr<float>();
  }
  launch(kDkv, a, q.scalar_type(), s);
  if (a.splits > 1) {
    const long n = (k.numel() / 4 + 255) / 256;   // two tensors, 8 a thread
    if (q.scalar_type() == at::kBFloat16)
      doc_attn_join_kernel<BF16><<<(unsigned)n, 256, 0, s>>>(a);
    else
      doc_attn_join_kernel<FP16><<<(unsigned)n, 256, 0, s>>>(a);
  }
}

}  // namespace dlx

// Matrix-instruction tiles of 16-bit elements, shared by document attention
// and Newton-Schulz.
//
// v_mfma_f32_32x32x16, lane l of the 64, h = l >> 5:
//   A[m][k]: m = l & 31, k = 8h + e            (e = 0..7, one 16-byte read)
//   B[k][n]: n = l & 31, k = 8h + e
//   C[m][n]: n = l & 31, m = 8 (i >> 2) + 4h + (i & 3)      (i = 0..15)
// The order of k is free as long as A and B agree.  Taking it as
//   k(e) = 8 (e >> 2) + 4h + (e & 3)
// makes registers 8a..8a+7 of a result C the operand B of step a of a next
// product whose k is C's m: a product's result feeds the next one without
// leaving its lane.  The next product's A, read across its rows, is then two
// transposing reads of four rows each (Frags::tr).
//
// LDS tiles are rows of DP elements in chunks of 8 (16 bytes), chunk c of row
// r stored at place c ^ swizzle(r).  The swizzle is linear in the row's bits
// and chosen so that 8 rows at one chunk fill 128 bytes of banks and 16 rows
// 256 (Frags::row), and 4 rows at four neighbouring chunks fill 256 (Frags::tr).
#pragma once

#include <type_traits>
#include <utility>

#include "seq_common.h"

namespace dlx {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using bf16v8_t = __attribute__((ext_vector_type(8))) __bf16;
using f16v8_t = __attribute__((ext_vector_type(8))) _Float16;
using bf16v2_t = __attribute__((ext_vector_type(2))) __bf16;
using f16v2_t = __attribute__((ext_vector_type(2))) _Float16;
using f32v2_t = __attribute__((ext_vector_type(2))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

typedef __attribute__((address_space(3))) uint32_t lds_word_t;
typedef const __attribute__((address_space(1))) uint32_t glb_word_t;

template <typename T> DLX_DEV f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c);
template <> DLX_DEV f32x16 mfma32<BF16>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16v8_t, a), __builtin_bit_cast(bf16v8_t, b), c, 0, 0,
      0);
}
template <> DLX_DEV f32x16 mfma32<FP16>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(f16v8_t, a), __builtin_bit_cast(f16v8_t, b), c, 0, 0,
      0);
}

// two fp32 to two 16-bit, round to nearest even
template <typename T> DLX_DEV uint32_t pack2(float a, float b);
template <> DLX_DEV uint32_t pack2<BF16>(float a, float b) {
  return __builtin_bit_cast(
      uint32_t, __builtin_convertvector(f32v2_t{a, b}, bf16v2_t));
}
template <> DLX_DEV uint32_t pack2<FP16>(float a, float b) {
  return __builtin_bit_cast(
      uint32_t, __builtin_convertvector(f32v2_t{a, b}, f16v2_t));
}

// registers 8a..8a+7 of a result as the next product's operand B
template <typename T> DLX_DEV s16x8 pack_step(const float* p) {
  return __builtin_bit_cast(
      s16x8, u32x4{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]),
                   pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7])});
}

// what pack_step's rounding leaves of them
template <typename T> DLX_DEV s16x8 pack_rest(const float* p, s16x8 high) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = p[e] - to_f32<T>(T{(uint16_t)high[e]});
  return pack_step<T>(rest);
}

template <int DP> DLX_DEV constexpr int swizzle(int r) {
  if (DP == 32) return ((r >> 2) & 1) | (((r >> 3) ^ (r >> 1)) & 1) << 1;
  if (DP == 64)
    return ((r >> 2) & 1) | ((r ^ (r >> 3)) & 1) << 1 | ((r >> 1) & 1) << 2;
  return ((r >> 2) & 1) | (((r >> 1) ^ (r >> 3)) & 1) << 1 | (r & 1) << 2 |
         ((r >> 1) & 1) << 3;
}

template <int DP> DLX_DEV int tile_at(int row, int chunk) {
  return row * DP + ((chunk ^ swizzle<DP>(row)) << 3);
}

// f(0), f(1), .. with numbers that are known when it is compiled
template <class F, int... I>
DLX_DEV void unroll_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F> DLX_DEV void unroll(F&& f) {
  unroll_(f, std::make_integer_sequence<int, N>{});
}

// Transposing reads, 2 N of them, at byte OFF from each lane's places.  The
// builtin would do, but the compiler cannot tell its reads from the tile that
// copy16_to_lds is filling and waits for that first, at every tile.  The wait
// for the reads themselves is part of the block.
template <int OFF>
DLX_DEV void read_tr2(uint32_t p0, uint32_t p1, s16x4& a, s16x4& b) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %2 offset:%4\n\t"
      "ds_read_b64_tr_b16 %1, %3 offset:%4\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a), "=&v"(b)
      : "v"(p0), "v"(p1), "i"(OFF)
      : "memory");
}

template <int OFF>
DLX_DEV void read_tr4(const uint32_t* p, const uint32_t* q, s16x4* a,
                      s16x4* b) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%8\n\t"
      "ds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
      "ds_read_b64_tr_b16 %2, %6 offset:%8\n\t"
      "ds_read_b64_tr_b16 %3, %7 offset:%8\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(b[0]), "=&v"(a[1]), "=&v"(b[1])
      : "v"(p[0]), "v"(q[0]), "v"(p[1]), "v"(q[1]), "i"(OFF)
      : "memory");
}

template <int OFF>
DLX_DEV void read_tr8(const uint32_t* p, const uint32_t* q, s16x4* a,
                      s16x4* b) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%16\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%16\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
      "ds_read_b64_tr_b16 %4, %12 offset:%16\n\t"
      "ds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
      "ds_read_b64_tr_b16 %6, %14 offset:%16\n\t"
      "ds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(b[0]), "=&v"(a[1]), "=&v"(b[1]), "=&v"(a[2]),
        "=&v"(b[2]), "=&v"(a[3]), "=&v"(b[3])
      : "v"(p[0]), "v"(q[0]), "v"(p[1]), "v"(q[1]), "v"(p[2]), "v"(q[2]),
        "v"(p[3]), "v"(q[3]), "i"(OFF)
      : "memory");
}

// Where a lane's fragments lie in a tile of DP columns.  The swizzle leaves a
// place for each chunk a lane reads; rows are offsets that fit the read
// instruction.
template <int DP> struct Frags {
  const uint16_t* lds;
  int row_[DP / 16];                  // elements from `lds`
  uint32_t lo_[DP / 32], hi_[DP / 32];  // LDS addresses

  // base: what the offsets of row() and tr() are taken from; col0: where
  // tr's block 0 begins, a multiple of 32
  DLX_DEV Frags(const uint16_t* base, int lane, int col0 = 0) : lds(base) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
      row_[s] = tile_at<DP>(lane & 31, s * 2 + (lane >> 5));
    const int row = ((lane >> 5) << 2) + ((lane & 15) >> 2);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
      const int col = col0 + b * 32 + (lane & 16) + ((lane & 3) << 2);
      lo_[b] = address(base + tile_at<DP>(row, col >> 3) + (col & 7));
      hi_[b] = address(base + tile_at<DP>(row + 8, col >> 3) + (col & 7));
    }
  }

  static DLX_DEV uint32_t address(const uint16_t* p) {
    return (uint32_t)(uintptr_t)(
        const __attribute__((address_space(3))) uint16_t*)p;
  }

  // operand A or B of step `step`, k along the rows: rows off / DP ..+31, the
  // first a multiple of 16
  DLX_DEV s16x8 row(int off, int step) const {
    return *reinterpret_cast<const s16x8*>(lds + row_[step] + off);
  }

  // N operands A (or B) whose m (n) runs along the rows, columns col0 + 32
  // (FIRST + n) .., and whose k runs over rows OFF / DP ..+15 (the first a
  // multiple of 16) in the order of pack_step
  // `more`: bytes further on, where an offset would not fit
  template <int N, int OFF, int FIRST = 0>
  DLX_DEV void tr(s16x8* f, uint32_t more = 0) const {
    s16x4 a[N], b[N];
    static_assert(OFF * 2 < 65536 && (N == 1 || N == 2 || N == 4), "");
    uint32_t lo[N], hi[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lo[i] = lo_[FIRST + i] + more;
      hi[i] = hi_[FIRST + i] + more;
    }
    if constexpr (N == 1) read_tr2<OFF * 2>(lo[0], hi[0], a[0], b[0]);
    if constexpr (N == 2) read_tr4<OFF * 2>(lo, hi, a, b);
    if constexpr (N == 4) read_tr8<OFF * 2>(lo, hi, a, b);
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = __builtin_shufflevector(a[i], b[i], 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // tr of block 0 in two tiles, `more` bytes apart, for one wait
  template <int OFF>
  DLX_DEV void tr_both(s16x8* f, uint32_t more) const {
    s16x4 a[2], b[2];
    static_assert(OFF * 2 < 65536, "");
    const uint32_t lo[2] = {lo_[0], lo_[0] + more};
    const uint32_t hi[2] = {hi_[0], hi_[0] + more};
    read_tr4<OFF * 2>(lo, hi, a, b);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      f[i] = __builtin_shufflevector(a[i], b[i], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// 16 bytes a lane from memory to LDS, lanes one behind the other there
DLX_DEV void copy16_to_lds(const void* src, uint16_t* dst) {
  __builtin_amdgcn_global_load_lds((glb_word_t*)src, (lds_word_t*)dst, 16, 0,
                                   0);
}

// The blocks of one stretch of the grid onto one XCD (blocks go round the
// eight XCDs by number), so that neighbours share its L2.
DLX_DEV int xcd_block(int bid, int blocks) {
  const int q = blocks / 8, r = blocks % 8;
  const int xcd = bid % 8, idx = bid / 8;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

}  // namespace dlx

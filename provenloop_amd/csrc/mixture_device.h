// Device pieces of the mixture operators' matrix kernels: matrix instructions
// by type, asynchronous loads into LDS, transposing LDS reads, bounded loads.
//
// Matrix instructions are 16 x 16 outputs over 32 contraction steps. Lane l
// holds row (column) l % 16 of each operand, contraction steps
// (l / 16) * 8 .. + 8, and of the result column l % 16, rows (l / 16) * 4 .. + 4.
#pragma once
#include <type_traits>

#include "mixture.h"

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) bf16_t bf16x8;
typedef __attribute__((ext_vector_type(8))) f16_t f16x8;

template <class T>
struct Vec8;
template <>
struct Vec8<bf16_t> {
  using type = bf16x8;
};
template <>
struct Vec8<f16_t> {
  using type = f16x8;
};
template <class T>
using vec8 = typename Vec8<T>::type;

__device__ inline f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// What lanes read in place of elements outside a matrix.
__device__ const uint4 mix_zero16 = {0, 0, 0, 0};

// A float as a pair of bf16, high + low: 16 bits of its significand, in
// float's exponent range, so that a low-rank factor held in float meets the
// matrix instructions with an error of 2^-17, far below an output's rounding.
__device__ inline void split8(const f32x8& v, bf16x8& hi, bf16x8& lo) {
  for (int i = 0; i < 8; ++i) {
    hi[i] = (bf16_t)v[i];
    lo[i] = (bf16_t)(v[i] - (float)hi[i]);
  }
}

// Infinities and NaN among 16-bit values: all exponent bits set.
template <class T>
constexpr uint32_t exponent_bits() {
  return std::is_same<T, bf16_t>::value ? 0x7f80 : 0x7c00;
}
template <class T>
__device__ inline bool is_finite(T v) {
  return (__builtin_bit_cast(uint16_t, v) & exponent_bits<T>()) != exponent_bits<T>();
}
// Adding the exponent's lowest bit to a full exponent carries into the sign's place.
template <class T>
__device__ inline bool all_finite(const vec8<T>& v) {
  constexpr uint32_t full = exponent_bits<T>(), one = full & -full;
  const uint4 d = __builtin_bit_cast(uint4, v);
  auto carry = [](uint32_t w) { return (w & (full << 16 | full)) + (one << 16 | one); };
  return ((carry(d.x) | carry(d.y) | carry(d.z) | carry(d.w)) & 0x80008000u) == 0;
}

// Whether every value's high part is finite: those from half a step above
// bf16's largest on round to infinity, and the low part would be the infinity
// of the other sign.
__device__ inline bool splits(float v) { return (__float_as_uint(v) & 0x7fffffff) < 0x7f7f8000; }
__device__ inline bool all_split(const f32x8& v) {
  uint32_t most = 0;
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffff);
  return most < 0x7f7f8000;
}

// The same pair for any float: one that rounds to infinity is bf16's largest and
// the rest, infinities and NaN are themselves with no low part.
__device__ inline void split8_any(const f32x8& v, bf16x8& hi, bf16x8& lo) {
  split8(v, hi, lo);
  if (all_split(v)) return;
  for (int i = 0; i < 8; ++i) {
    if (splits(v[i])) continue;
    const bool number = (__float_as_uint(v[i]) & 0x7fffffff) < 0x7f800000;
    if (number) hi[i] = __builtin_bit_cast(bf16_t, (uint16_t)(v[i] < 0 ? 0xff7f : 0x7f7f));
    lo[i] = number ? (bf16_t)(v[i] - (float)hi[i]) : (bf16_t)0.0f;
  }
}

// acc += a * b with b given as floats split in two; an f16 operand is split
// too (11 bits, exact in the pair), a bf16 one needs no low part.
__device__ inline f32x4 mfma_split(bf16x8 a, bf16x8 hi, bf16x8 lo, f32x4 c) { return mfma(a, hi, mfma(a, lo, c)); }
struct SplitF16 {
  bf16x8 hi, lo;
};
__device__ inline bf16x8 widen(bf16x8 v) { return v; }
__device__ inline SplitF16 widen(f16x8 v) {
  f32x8 f;
  for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
  SplitF16 s;
  split8(f, s.hi, s.lo);
  return s;
}
__device__ inline f32x4 mfma_split(const SplitF16& a, bf16x8 hi, bf16x8 lo, f32x4 c) {
  return mfma(a.hi, hi, mfma(a.hi, lo, mfma(a.lo, hi, c)));
}

// The high parts' product alone. Infinities times pairs may be infinities of both
// signs or meet a zero low part; here they are what they are in the product of
// the values themselves.
__device__ inline f32x4 mfma_high(bf16x8 a, bf16x8 hi, f32x4 c) { return mfma(a, hi, c); }
__device__ inline f32x4 mfma_high(const SplitF16& a, bf16x8 hi, f32x4 c) { return mfma(a.hi, hi, c); }

// 8 elements at p of which the first `valid` exist; the rest read as zero.
// whole: all 8 may be read at once at any alignment of an element.
template <class T>
__device__ inline vec8<T> load8(const T* p, int64_t valid) {
  vec8<T> v;
  if (valid >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else {
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? p[i] : (T)0.0f;
  }
  return v;
}

// 16 bytes per lane from global memory to lds + 16 * lane, without a register.
// The compiler does not know of it: the arrived... functions wait for it, and
// the compiler's own waits, which count fewer loads than there are, only wait
// longer. (It keeps nothing of its own in m0 here, which it does not let an asm
// name as written.)
__device__ inline void load_lds16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory");
}
// Every load into LDS of this wavefront has arrived and every LDS access has
// been answered; then the workgroup's barrier.
__device__ inline void arrived_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The same for this wavefront alone: at most N loads into LDS are under way;
// its LDS reads have been answered.
template <int N>
__device__ inline void arrived(void) {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ inline void answered(void) { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ inline uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Rows 0..3 of a 4 x 16 block of 16-bit elements, 8 bytes a lane (lane l of 16:
// row l / 4, columns (l % 4) * 4 .. + 4): lane l receives column l.
__device__ inline s16x4 read_transposed(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// A tile of contraction rows in LDS, `cols` elements each, with 16-byte chunk c
// of row k at c ^ swizzle(k): the 16 rows that a transposing read touches at
// one column then lie in different banks.
template <int COLS>
__device__ inline uint32_t tr_swizzle(uint32_t k) {
  return (2 * ((k & 3) | ((k >> 3) & 1) << 2)) & (COLS / 8 - 1);
}
// Lane's operand for columns col .. + 16, contraction rows k .. + 32.
template <class T, int COLS>
__device__ inline vec8<T> tr_fragment(const char* tile, uint32_t col, uint32_t k, uint32_t lane) {
  const uint32_t row = k + lane / 16 * 8 + lane % 16 / 4, c = col + lane % 4 * 4;
  const char* p = tile + row * (COLS * 2) + ((c / 8) ^ tr_swizzle<COLS>(row)) * 16 + c % 8 * 2;
  // four rows on: the swizzle goes by row bits 0, 1 and 3 and is the same
  const s16x4 a = read_transposed(p), b = read_transposed(p + 4 * COLS * 2);
  return __builtin_bit_cast(vec8<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Workgroup `id` of `total` tiles, neighbours in the tile order kept on one of
// the 8 XCDs (workgroups go to them in turn), whose L2 they then share.
__device__ inline uint32_t xcd_tile(uint32_t id, uint32_t total) {
  const uint32_t q = total / 8, r = total % 8, x = id % 8;
  return x * q + min(x, r) + id / 8;
}

// Where a tile of at most BM rows of one group lies: groups 0 .. E - 1, and
// group E for the slots without one.
struct GroupTile {
  uint32_t group;
  int64_t begin, end;  // slots in sorted order
};
__device__ inline int64_t group_begin(const int32_t* offsets, uint32_t g, uint32_t E, int64_t slots) {
  return g > E ? slots : min(max((int64_t)offsets[g], (int64_t)0), slots);
}
// Tiles of all groups [0, groups); every lane of the calling wavefront gets the answer.
__device__ inline uint32_t count_group_tiles(const int32_t* offsets, uint32_t E, uint32_t groups, int64_t slots,
                                             uint32_t bm, uint32_t lane) {
  uint32_t n = 0;
  for (uint32_t g = lane; g < groups; g += 64) {
    const int64_t c = group_begin(offsets, g + 1, E, slots) - group_begin(offsets, g, E, slots);
    if (c > 0) n += (uint32_t)((c + bm - 1) / bm);
  }
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  return n;
}
__device__ inline GroupTile find_group_tile(const int32_t* offsets, uint32_t E, uint32_t groups, int64_t slots,
                                            uint32_t bm, uint32_t tile, uint32_t lane) {
  GroupTile t{groups, 0, 0};
  uint32_t before = 0;
  for (uint32_t at = 0; at < groups; at += 64) {
    const uint32_t g = at + lane;
    int64_t lo = 0, c = 0;
    if (g < groups) {
      lo = group_begin(offsets, g, E, slots);
      c = group_begin(offsets, g + 1, E, slots) - lo;
    }
    const uint32_t n = c > 0 ? (uint32_t)((c + bm - 1) / bm) : 0;
    uint32_t sum = n;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if ((int)lane >= d) sum += up;
    }
    const uint32_t first = before + sum - n;
    const uint64_t here = __ballot(n && tile >= first && tile < first + n);
    if (here) {
      const int src = __ffsll((unsigned long long)here) - 1;
      t.group = at + src;
      t.begin = __shfl((int)lo, src) + (int64_t)(tile - __shfl(first, src)) * bm;
      t.end = min(t.begin + (int64_t)bm, (int64_t)__shfl((int)(lo + c), src));
      return t;
    }
    before += __shfl(sum, 63);
  }
  return t;
}

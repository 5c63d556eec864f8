// The tile kernel of large matrix products, y = x w^T or y = x w, of ragged
// groups or with low-rank adapters added (see wide.hip).
#pragma once
#include <type_traits>

#include "mixture_device.h"

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

namespace mix {

constexpr int BK = 64;  // contraction steps of one LDS tile: 128 bytes a row

// Waits until at most N of this wavefront's loads into LDS are under way and
// its LDS reads have been answered; then the workgroup's barrier.
template <int N>
__device__ inline void arrived_but(void) {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The low-rank part of a workgroup's tile, y_t += sum_j c_tj P[id_tj] u_tj, as
// further contraction steps: the adapters that the tile's rows use are listed,
// and for 64 of their ranks at a time the rows' coefficients c u (zero where a
// row does not use the adapter) and the adapters' columns are laid in LDS as
// bf16 pairs, high and low, so that u keeps its float's 16 leading bits: one
// more product with the low halves costs little next to the main one, and
// rounding u once to bf16 would be as large an error as rounding y.
//
// A row's zeros meet the columns of adapters that it does not use, so an
// infinity or NaN among those would make NaN of it; and an infinity times the
// two parts of a pair, or an infinite coefficient's parts, are infinities of
// both signs. They are laid as zeros too, and what they add to the rows that do
// use them is made by add_nonfinite.
//
// list_adapters runs under the main product's first loads and leaves in LDS the
// adapters and, for up to KEPT choices, each row's and its coefficients; the
// loads of one set of 64 ranks then go out together. 4096 x 1536 x 1536 with two
// of 8 rank-16 adapters a token takes 37 us, 24.5 without adapters; with the
// lists made after the main product and pieces loaded one by one it took 50.
constexpr uint32_t KEPT = 4;
template <int BM>
struct LowLists {
  uint32_t words[32];  // a bit per adapter: used, and after the listing, whether something of it is left out
  uint32_t count;
  uint16_t list[th::MIX_MAX_EXPERTS];  // those used, rising
  uint32_t id[BM * KEPT];              // rows x choices; ~0: none
  float c[BM * KEPT];
};

template <int BM, int THREADS>
__device__ inline void list_adapters(const MatArgs& a, int64_t m0, int64_t mend, LowLists<BM>& l) {
  const uint32_t lane = threadIdx.x & 63, used = (uint32_t)(mend - m0) * a.kc;
  if (threadIdx.x < 32) l.words[threadIdx.x] = 0;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < used; i += THREADS) {
    const int64_t s = m0 * a.kc + i;
    const uint32_t e = (uint32_t)a.ids[s];
    float c = a.gate ? a.gate[s] : 1.0f;
    if (e < a.E) {
      atomicOr(&l.words[e / 32], 1u << (e % 32));
      if (a.scale) c *= a.scale[e];
    }
    if (a.kc <= KEPT) {
      l.id[i] = e < a.E ? e : ~0u;
      l.c[i] = c;
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const uint32_t word = lane < 32 ? l.words[lane] : 0, own = __popc(word);
    uint32_t sum = own;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if ((int)lane >= d) sum += up;
    }
    uint32_t at = sum - own;
    for (uint32_t w = word; w; w &= w - 1) l.list[at++] = (uint16_t)(lane * 32 + __ffs(w) - 1);
    if (lane == 63) l.count = sum;
  }
  __syncthreads();
  if (threadIdx.x < 32) l.words[threadIdx.x] = 0;
}

// Coefficient of choice `s` of the tile (row x choices + j), which uses adapter e.
template <int BM>
__device__ inline float coefficient(const MatArgs& a, int64_t m0, const LowLists<BM>& l, uint32_t s, uint32_t e) {
  if (a.kc <= KEPT) return l.c[s];
  return (a.gate ? a.gate[m0 * a.kc + s] : 1.0f) * (a.scale ? a.scale[e] : 1.0f);
}
template <int BM>
__device__ inline uint32_t adapter_of(const MatArgs& a, int64_t m0, const LowLists<BM>& l, uint32_t s) {
  return a.kc <= KEPT ? l.id[s] : (uint32_t)a.ids[m0 * a.kc + s];
}

// The products that add_lowrank leaves out, those of infinities and NaN and of
// coefficients that make no finite pair, for a wavefront's TM x 64 outputs: each
// row's own adapters alone, a row at a time in float, through the wavefront's own
// LDS in two halves. -0 where there is none, which changes no sum.
template <class T, int BM, int TM, int TN>
__device__ inline void add_nonfinite(const MatArgs& a, int64_t m0, uint32_t rows, uint32_t row0, uint32_t n0, float* own,
                                     const LowLists<BM>& l, uint32_t lane, f32x4 (&acc)[TN / 16][TM / 16]) {
  static_assert(TN == 64);
  constexpr int SLAB = TM / 2;
  const uint32_t n = min(n0 + lane, a.n - 1);
#pragma unroll
  for (int s0 = 0; s0 < TM; s0 += SLAB) {
#pragma unroll 1
    for (uint32_t i = 0; i < SLAB; ++i) {
      const uint32_t row = __builtin_amdgcn_readfirstlane(row0) + s0 + i;
      float sum = -0.0f;
#pragma unroll 1
      for (uint32_t j = 0; row < rows && j < a.kc; ++j) {
        const uint32_t s = row * a.kc + j, e = __builtin_amdgcn_readfirstlane(adapter_of(a, m0, l, s));
        if (e >= a.E || !(__builtin_amdgcn_readfirstlane(l.words[e / 32]) >> (e % 32) & 1)) continue;
        const T* p = (const T*)a.p + e * a.ldpe + (int64_t)n * a.ldp;
        const float* u = a.u + (m0 * a.kc + s) * a.ru;
        float f = 0, d = 0;  // f: what add_lowrank took for this adapter's coefficient
        for (uint32_t i = 0; i < a.kc; ++i)
          if (adapter_of(a, m0, l, row * a.kc + i) == e) f += coefficient(a, m0, l, row * a.kc + i, e);
        bool any = false;
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < a.r; r0 += 8) {
          const vec8<T> v = load8<T>(p + r0, (int64_t)a.r - r0);
#pragma unroll
          for (uint32_t q = 0; q < 8; ++q) {
            const float x = r0 + q < a.r ? u[r0 + q] : 0.0f;
            if (r0 + q < a.r && !(is_finite(v[q]) && splits(f * x))) {
              d = fmaf(x, (float)v[q], d);
              any = true;
            }
          }
        }
        if (any) sum += coefficient(a, m0, l, s, e) * d;
      }
      own[i * TN + lane] = sum;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int mi = s0 / 16; mi < (s0 + SLAB) / 16; ++mi)
#pragma unroll
      for (int ni = 0; ni < TN / 16; ++ni)
        acc[ni][mi] += *(const f32x4*)&own[(mi * 16 - s0 + lane % 16) * TN + ni * 16 + lane / 16 * 4];
    __builtin_amdgcn_wave_barrier();
  }
}

template <class T, int BM, int BN, int WM, int WN>
__device__ inline void add_lowrank(const MatArgs& a, int64_t m0, int64_t mend, uint32_t n0, char* lds,
                                   LowLists<BM>& l, f32x4 (&acc)[BN / WN / 16][BM / WM / 16]) {
  constexpr int THREADS = 64 * WM * WN, TM = BM / WM, TN = BN / WN;
  constexpr int XI = BM * 8 / THREADS, WI = BN * 8 / THREADS;   // 16-byte pieces of a thread
  constexpr bool PAIR = !std::is_same<T, bf16_t>::value;  // f16 operands are pairs too
  char *xhi = lds, *xlo = xhi + BM * 128, *whi = xlo + BM * 128, *wlo = whi + (PAIR ? BN * 128 : 0);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const uint32_t rows = (uint32_t)(mend - m0);
  const uint32_t each = (a.r + 7) / 8, chunks = l.count * each;  // chunks of 8 ranks
  const uint32_t piece = threadIdx.x % 8;                        // this thread's chunk of a set, in all its rows
  bool odd = false;
  // it leaves something of adapter e out
  auto left_out = [&](uint32_t e) __attribute__((always_inline)) {
    odd = true;
    atomicOr(&l.words[e / 32], 1u << (e % 32));
  };
  for (uint32_t c0 = 0; c0 < chunks; c0 += 8) {
    const uint32_t c = c0 + piece, e = c < chunks ? l.list[c / each] : ~1u, r0 = c % each * 8;
    const bool whole = r0 + 8 <= a.r;
    f32x4 u0[XI], u1[XI];
    float f[XI];
    vec8<T> v[WI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t row = i * (THREADS / 8) + threadIdx.x / 8;
      u0[i] = u1[i] = f32x4{0, 0, 0, 0};
      f[i] = 0;
      uint32_t at = ~0u;
      if (row < rows && c < chunks) {
        for (uint32_t j = 0; j < a.kc; ++j) {  // an adapter chosen twice counts with both coefficients
          const uint32_t s = row * a.kc + j;
          if (adapter_of(a, m0, l, s) != e) continue;
          at = s;
          f[i] += coefficient(a, m0, l, s, e);
        }
      }
      if (at != ~0u) {
        const float* u = a.u + (m0 * a.kc + at) * a.ru + r0;
        if (whole) {
          u0[i] = *(const f32x4*)u;
          u1[i] = *(const f32x4*)(u + 4);
        } else {
          for (uint32_t q = 0; q < 8; ++q)
            if (r0 + q < a.r) (q < 4 ? u0[i] : u1[i])[q % 4] = u[q];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < WI; ++i) {
      const uint32_t n = n0 + i * (THREADS / 8) + threadIdx.x / 8;
      const bool in = c < chunks && n < a.n;
      v[i] = load8<T>(in ? (const T*)a.p + e * a.ldpe + (int64_t)n * a.ldp + r0 : (const T*)&mix_zero16,
                      in ? (int64_t)a.r - r0 : 0);
    }
    __syncthreads();  // the LDS below has been read
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t row = i * (THREADS / 8) + threadIdx.x / 8, at = row * 128 + (piece ^ (row & 7)) * 16;
      f32x8 x;
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = f[i] * (q < 4 ? u0[i] : u1[i])[q % 4];
      if (!all_split(x)) {
        left_out(e);
        for (int q = 0; q < 8; ++q) x[q] = splits(x[q]) ? x[q] : 0.0f;
      }
      bf16x8 hi, lo;
      split8(x, hi, lo);
      *(bf16x8*)(xhi + at) = hi;
      *(bf16x8*)(xlo + at) = lo;
    }
#pragma unroll
    for (int i = 0; i < WI; ++i) {
      const uint32_t row = i * (THREADS / 8) + threadIdx.x / 8, at = row * 128 + (piece ^ (row & 7)) * 16;
      if (!all_finite<T>(v[i])) {
        left_out(e);
        for (int q = 0; q < 8; ++q) v[i][q] = is_finite(v[i][q]) ? v[i][q] : (T)0.0f;
      }
      if constexpr (PAIR) {
        const SplitF16 s = widen(v[i]);
        *(bf16x8*)(whi + at) = s.hi;
        *(bf16x8*)(wlo + at) = s.lo;
      } else {
        *(bf16x8*)(whi + at) = v[i];
      }
    }
    __syncthreads();
    for (uint32_t kk = 0; kk < 2; ++kk) {
      if (c0 + kk * 4 >= chunks) break;
      bf16x8 hi[TM / 16], lo[TM / 16];
#pragma unroll
      for (int mi = 0; mi < TM / 16; ++mi) {
        const uint32_t row = wm * TM + mi * 16 + lane % 16, at = row * 128 + ((kk * 4 + lane / 16) ^ (row & 7)) * 16;
        hi[mi] = *(const bf16x8*)(xhi + at);
        lo[mi] = *(const bf16x8*)(xlo + at);
      }
#pragma unroll
      for (int ni = 0; ni < TN / 16; ++ni) {
        const uint32_t row = wn * TN + ni * 16 + lane % 16, at = row * 128 + ((kk * 4 + lane / 16) ^ (row & 7)) * 16;
        const bf16x8 wf = *(const bf16x8*)(whi + at);
#pragma unroll
        for (int mi = 0; mi < TM / 16; ++mi) acc[ni][mi] = mfma(wf, hi[mi], mfma(wf, lo[mi], acc[ni][mi]));
        if constexpr (PAIR) {
          const bf16x8 wl = *(const bf16x8*)(wlo + at);
#pragma unroll
          for (int mi = 0; mi < TM / 16; ++mi) acc[ni][mi] = mfma(wl, hi[mi], acc[ni][mi]);
        }
      }
    }
  }
  if (__syncthreads_or(odd))
    add_nonfinite<T, BM, TM, TN>(a, m0, rows, wm * TM, n0 + wn * TN, (float*)(lds + wave * (TM * TN * 2)), l, lane, acc);
}
template <class T, int BM, int BN>
constexpr uint32_t lowrank_lds() {
  return 2 * BM * 128 + (std::is_same<T, bf16_t>::value ? 1 : 2) * BN * 128;
}

// LDS: the stages, the low-rank tiles and each wavefront's outputs in turn in
// the same place, then the tile's rows and low-rank lists.
template <class T, int BM, int BN, int S, bool LR>
constexpr uint32_t wide_slots() {
  const uint32_t main = S * (BM + BN) * BK * 2, low = LR ? lowrank_lds<T, BM, BN>() : 0, out = BM * BN * 2;
  return main > low ? (main > out ? main : out) : (low > out ? low : out);
}
template <class T, int BM, int BN, int S, bool LR>
constexpr uint32_t wide_lds() {
  return wide_slots<T, BM, BN, S, LR>() + BM * 4 + (LR ? (uint32_t)sizeof(LowLists<BM>) : 0);
}

// A wavefront's TM x TN outputs to memory. A lane holds 4 neighbouring columns
// of each of its rows, and stores of 8 bytes to 16 rows at once fill a sixteenth
// of what a store can carry, so they go through the wavefront's own TM TN 2
// bytes of LDS and leave as 16 bytes a lane, whole lines of a row. They stream
// past the caches, which the operands need: 16384 x 3584 x 1536 took 187 us with
// streaming stores and 210 without, 4096 x 1536 x 1536 24.5 and 27.7.
struct Out {
  void* y;
  int64_t ld;
  uint32_t n;
  const void* bias;  // null, or a value per column
};
template <class O, class T, int TM, int TN>
__device__ inline void put(const Out& out, f32x4 (&acc)[TN / 16][TM / 16], char* own, const uint32_t* slots,
                           uint32_t m0, uint32_t rows, uint32_t n0, uint32_t lane) {
  constexpr int PER = 16 / sizeof(O), CH = TN / PER;      // values of a 16-byte chunk, chunks of a row
  constexpr int SLAB = TM * 2 / (int)sizeof(O);           // rows that fit
  constexpr int MASK = CH < 16 ? CH - 1 : 15;
  const bool wide = out.ld % PER == 0 && ((uintptr_t)out.y & 15) == 0;
#pragma unroll
  for (int s0 = 0; s0 < TM; s0 += SLAB) {
#pragma unroll
    for (int ni = 0; ni < TN / 16; ++ni) {
      float bias[4] = {0, 0, 0, 0};
      const uint32_t n = n0 + ni * 16 + lane / 16 * 4;
      if (out.bias)
        for (int q = 0; q < 4; ++q)
          if (n + q < out.n) bias[q] = to_float(((const T*)out.bias)[n + q]);
#pragma unroll
      for (int mi = s0 / 16; mi < (s0 + SLAB) / 16; ++mi) {
        const f32x4 v = acc[ni][mi];
        O o[4] = {(O)(v[0] + bias[0]), (O)(v[1] + bias[1]), (O)(v[2] + bias[2]), (O)(v[3] + bias[3])};
        const uint32_t row = mi * 16 - s0 + lane % 16, at = ni * 16 + lane / 16 * 4;
        char* p = own + (row * CH + ((at / PER) ^ (row & MASK))) * 16 + at % PER * sizeof(O);
        __builtin_memcpy(__builtin_assume_aligned(p, 4 * sizeof(O)), o, 4 * sizeof(O));
      }
    }
    __builtin_amdgcn_wave_barrier();  // a wavefront's LDS accesses are answered in order
    for (uint32_t i = lane; i < SLAB * CH; i += 64) {
      const uint32_t row = i / CH, m = m0 + s0 + row, n = n0 + i % CH * PER;
      if (m >= rows || n >= out.n) continue;
      O o[PER];
      __builtin_memcpy(o, __builtin_assume_aligned(own + (row * CH + ((i % CH) ^ (row & MASK))) * 16, 16), 16);
      O* y = (O*)out.y + (int64_t)(slots ? slots[m] : m) * out.ld + n;
      if (wide && n + PER <= out.n) {
        u32x4 v;
        __builtin_memcpy(&v, o, 16);
        if constexpr (std::is_same<O, float>::value) *(u32x4*)y = v;  // a workspace: read again at once
        else __builtin_nontemporal_store(v, (u32x4*)y);
      }
      else
        for (int q = 0; q < PER; ++q)
          if (n + q < out.n) y[q] = o[q];
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// BM x BN outputs per workgroup of WM x WN wavefronts. S tiles of x (BM rows
// of 64 contraction steps) and of w are in LDS or on their way there; a tile's
// two halves of 32 steps pass through registers, the next half being read from
// LDS while the matrix cores work on this one. One barrier a tile: at it, every
// wavefront has the tile's second half in registers, so the tile's place can
// take new loads, and the next tile has arrived. w's tile is BN rows of 64
// steps, or, for y = x w, 64 rows of BN columns read through the transposing
// LDS read.
//
// The matrix cores bound it: 8192 x 8192 x 8192 in bf16 runs at 1452 TFLOP/s in a
// long series (y = x w: 1331), 90 % of what the library's product reaches on the
// card (1621, at the clock the power leaves). 256 x 256 needs 64 KiB a tile, so
// two of them and one workgroup of 8 wavefronts a CU; 4 wavefronts of 128 x 128
// outputs did not fit the registers, 128 x 128 tiles reach 924 in a short series.
// Interleaving LDS reads, loads and products in 8 pieces a half took 8192 x 3584 x
// 3584 from 231 to 215 us. What is left there (164 us in a long series, floor 130)
// is 448 tiles on 256 CUs, two rounds of which the second is three quarters full,
// and 4 us a round of stores.
template <class T, int BM, int BN, int WM, int WN, int S, bool TR, bool LR>
__global__ void __launch_bounds__(64 * WM * WN) wide_kernel(MatArgs a) {
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN;
  constexpr int AJ = BM / 8 / WAVES, BJ = BN / 8 / WAVES;  // 1 KiB loads per wavefront and tile
  constexpr uint32_t STAGE = (BM + BN) * BK * 2;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wm = wave / WN, wn = wave % WN;

  // ---- which rows and columns
  const uint32_t ntiles = (a.n + BN - 1) / BN;
  const bool grouped = a.offsets != nullptr;
  const uint32_t mtiles = grouped ? count_group_tiles(a.offsets, a.E, a.E + 1, a.rows, BM, lane)
                                  : (uint32_t)((a.rows + BM - 1) / BM);
  const uint32_t total = mtiles * ntiles;
  if (blockIdx.x >= total) return;
  // bands of 8 row tiles, column tiles outside, so that both stay in an L2
  const uint32_t tile = xcd_tile(blockIdx.x, total);
  const uint32_t band = tile / (8 * ntiles), in = tile % (8 * ntiles), height = min(8u, mtiles - band * 8);
  const uint32_t mt = band * 8 + in % height, n0 = in / height * BN;
  GroupTile g{0, (int64_t)mt * BM, min((int64_t)(mt + 1) * BM, a.rows)};
  if (grouped) g = find_group_tile(a.offsets, a.E, a.E + 1, a.rows, BM, mt, lane);
  if (g.begin >= g.end) return;
  // the rows of y (slots) of this tile
  uint32_t* slots = (uint32_t*)(lds + wide_slots<T, BM, BN, S, LR>());
  for (uint32_t i = threadIdx.x; i < BM; i += 64 * WAVES) {
    const int64_t at = min(g.begin + i, g.end - 1);
    slots[i] = a.order ? (uint32_t)min((int64_t)(uint32_t)a.order[at], a.rows - 1) : (uint32_t)at;
  }
  __syncthreads();

  f32x4 acc[TN / 16][TM / 16];
  #pragma unroll
  for (int i = 0; i < TN / 16; ++i)
    #pragma unroll
    for (int j = 0; j < TM / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (!grouped || g.group < a.E) {
    const T* w = (const T*)a.w + (grouped ? (int64_t)g.group * a.ldwe : 0);
    const char* zero = (const char*)&mix_zero16;
    // ---- this lane's 16-byte pieces of both tiles
    const T* xp[AJ];
    const T* wp[BJ];
    const uint32_t xk = ((lane % 8) ^ (lane / 8)) * 8;  // chunk of the row: chunk c of row i lies at c ^ (i % 8)
    #pragma unroll
    for (int j = 0; j < AJ; ++j) {
      const uint32_t s = slots[(wave * AJ + j) * 8 + lane / 8];
      xp[j] = (const T*)a.x + (int64_t)(s / a.div) * a.ldx + xk;
    }
    constexpr int ROWC = BN / 8;           // chunks of a row of the transposed tile
    uint32_t wk[TR ? BJ : 1];              // contraction step of each piece of it,
    uint32_t inside = 0;                   // bit j: whether its columns exist
    #pragma unroll
    for (int j = 0; j < BJ; ++j) {
      if constexpr (TR) {
        const uint32_t row = (wave * BJ + j) * (64 / ROWC) + lane / ROWC;
        const uint32_t col = n0 + ((lane % ROWC) ^ tr_swizzle<BN>(row)) * 8;
        wk[j] = row;
        if (col < a.n) inside |= 1u << j;
        wp[j] = w + (int64_t)row * a.ldw + min(col, a.n - 1);
      } else {
        const uint32_t row = min(n0 + (wave * BJ + j) * 8 + lane / 8, a.n - 1);
        wp[j] = w + (int64_t)row * a.ldw + xk;
      }
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + wave * AJ * 1024;
    const uint32_t lds1 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + BM * BK * 2 + wave * BJ * 1024;
    // load j of this wavefront's of a tile
    auto load = [&](int j, uint32_t k0, uint32_t stage) __attribute__((always_inline)) {
      const bool whole = k0 + BK <= a.k;
      if (j < AJ) {
        const void* p = xp[j] + k0;
        if (!whole && k0 + xk >= a.k) p = zero;
        load_lds16(p, lds0 + stage * STAGE + j * 1024);
      } else {
        j -= AJ;
        const void* p;
        if constexpr (TR) {
          p = wp[j] + (int64_t)k0 * a.ldw;
          if ((!whole && k0 + wk[j] >= a.k) || !(inside >> j & 1)) p = zero;
        } else {
          p = wp[j] + k0;
          if (!whole && k0 + xk >= a.k) p = zero;
        }
        load_lds16(p, lds1 + stage * STAGE + j * 1024);
      }
    };
    constexpr int MI = TM / 16, NI = TN / 16, LOADS = AJ + BJ;
    vec8<T> xf[2][MI], wf[2][NI];
    auto read_x = [&](int set, int mi, uint32_t stage, int kk) __attribute__((always_inline)) {
      const uint32_t row = wm * TM + mi * 16 + lane % 16, chunk = kk * 4 + lane / 16;
      xf[set][mi] = *(const vec8<T>*)(lds + stage * STAGE + row * 128 + (chunk ^ (row & 7)) * 16);
    };
    auto read_w = [&](int set, int ni, uint32_t stage, int kk) __attribute__((always_inline)) {
      const char* wt = lds + stage * STAGE + BM * BK * 2;
      if constexpr (TR) {
        wf[set][ni] = tr_fragment<T, BN>(wt, wn * TN + ni * 16, kk * 32, lane);
      } else {
        const uint32_t row = wn * TN + ni * 16 + lane % 16, chunk = kk * 4 + lane / 16;
        wf[set][ni] = *(const vec8<T>*)(wt + row * 128 + (chunk ^ (row & 7)) * 16);
      }
    };
    // Half a tile: products of register set `set`, while the other set is read
    // from (stage, kk) and the loads of the tile at k0 are started. In 8
    // pieces, so that a SIMD's two wavefronts fill each other's gaps.
    auto half = [&](int set, bool reads, uint32_t stage, int kk, bool loads, uint32_t k0, uint32_t to)
        __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (reads)
#pragma unroll
          for (int f = p * (MI + NI) / 8; f < (p + 1) * (MI + NI) / 8; ++f) {
            if (f < NI) read_w(set ^ 1, f, stage, kk);
            else read_x(set ^ 1, f - NI, stage, kk);
          }
        if (loads)
#pragma unroll
          for (int j = p * LOADS / 8; j < (p + 1) * LOADS / 8; ++j) load(j, k0, to);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = p * MI * NI / 8; q < (p + 1) * MI * NI / 8; ++q)
          acc[q / MI][q % MI] = mfma(wf[set][q / MI], xf[set][q % MI], acc[q / MI][q % MI]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const uint32_t tiles = (a.k + BK - 1) / BK;
    for (uint32_t s = 0; s < S; ++s)
      if (s < tiles)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) load(j, s * BK, s);
    LowLists<BM>& lists = *(LowLists<BM>*)(slots + BM);
    if (LR) list_adapters<BM, 64 * WAVES>(a, g.begin, g.end, lists);
    if (tiles >= S) arrived_but<(S - 1) * LOADS>();
    else arrived_but<0>();
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) read_w(0, ni, 0, 0);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) read_x(0, mi, 0, 0);
    uint32_t stage = 0;
    for (uint32_t i = 0; i + S < tiles; ++i) {
      const uint32_t next = stage + 1 == S ? 0 : stage + 1;
      half(0, true, stage, 1, false, 0, 0);
      arrived_but<(S - 2) * LOADS>();  // tile i + 1 is there; the S - 2 after it may still be under way
      half(1, true, next, 0, true, (i + S) * BK, stage);
      stage = next;
    }
    for (uint32_t i = tiles > S ? tiles - S : 0; i < tiles; ++i) {
      const uint32_t next = stage + 1 == S ? 0 : stage + 1;
      half(0, true, stage, 1, false, 0, 0);
      arrived_but<0>();
      half(1, i + 1 < tiles, next, 0, false, 0, 0);
      stage = next;
    }
    if (LR) add_lowrank<T, BM, BN, WM, WN>(a, g.begin, g.end, n0, lds, lists, acc);
  }

  __syncthreads();
  char* own = lds + wave * (TM * TN * 2);
  const uint32_t rows = (uint32_t)(g.end - g.begin);
  const Out out{a.y, a.ldy, a.n, a.bias};
  if (a.y_float) put<float, T, TM, TN>(out, acc, own, slots, wm * TM, rows, n0 + wn * TN, lane);
  else put<T, T, TM, TN>(out, acc, own, slots, wm * TM, rows, n0 + wn * TN, lane);
}

}  // namespace mix

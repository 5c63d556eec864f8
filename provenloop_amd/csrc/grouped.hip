// Matrix products of ragged groups and of the shared projection with its
// low-rank adapters, y = x w^T or x w, on the matrix cores.
#include "mixture_device.h"

namespace {

constexpr int BK = 64;  // contraction steps of one LDS tile: 128 bytes a row

// The low-rank part of one wavefront's TM x TN outputs: one pass per adapter
// that its rows use, u (float) times the adapter's rows, as bf16 pairs.
template <class T, int TM, int TN>
__device__ void add_lowrank(const MatArgs& a, int64_t m0, int64_t mend, uint32_t n0, f32x4 (&acc)[TN / 16][TM / 16],
                            uint32_t lane) {
  constexpr int HALF = TM < 64 ? TM : 64;
  for (int h = 0; h < TM / HALF; ++h) {
    const int64_t row = m0 + h * HALF + lane;
    const bool valid = lane < HALF && row < mend;
    uint32_t done = 0;  // lane i: word i of the adapters dealt with
    for (uint32_t j = 0; j < a.kc; ++j) {
      const uint32_t id = valid ? (uint32_t)a.ids[row * a.kc + j] : ~0u;
      const uint32_t word = __shfl(done, id < a.E ? id >> 5 : 0);
      bool open = id < a.E && !((word >> (id & 31)) & 1);
      uint64_t pending;
      while ((pending = __ballot(open))) {
        const uint32_t e = __builtin_amdgcn_readlane(id, __ffsll((unsigned long long)pending) - 1);
        if (lane == e >> 5) done |= 1u << (e & 31);
        if (id == e) open = false;
        // the row's first choice of this adapter, and its coefficient there
        int at = -1;
        float c = 0;
        if (valid)
          for (uint32_t i = 0; i < a.kc; ++i)
            if ((uint32_t)a.ids[row * a.kc + i] == e) {
              if (at < 0) at = (int)i;
              c += a.gate ? a.gate[row * a.kc + i] : 1.0f;
            }
        if (a.scale) c *= a.scale[e];
        const T* pe = (const T*)a.p + (int64_t)e * a.ldpe;
        for (uint32_t r0 = 0; r0 < a.r; r0 += 32) {
          const int rr = (int)(r0 + lane / 16 * 8);
          const int rv = (int)a.r - rr;
          decltype(widen(vec8<T>())) pf[TN / 16];
          for (int ni = 0; ni < TN / 16; ++ni) {
            const uint32_t n = min(n0 + ni * 16 + lane % 16, a.n - 1);
            pf[ni] = widen(load8<T>(pe + (int64_t)n * a.ldp + (rv > 0 ? rr : 0), rv));
          }
          for (int mi = 0; mi < HALF / 16; ++mi) {
            const int src = mi * 16 + lane % 16;
            const int ju = __shfl(at, src);
            const float cu = __shfl(c, src);
            f32x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
            if (ju >= 0) {
              const float* u = a.u + ((m0 + h * HALF + src) * a.kc + ju) * a.ru + rr;
              for (int i = 0; i < 8; ++i)
                if (i < rv) v[i] = cu * u[i];
            }
            bf16x8 hi, lo;
            split8(v, hi, lo);
            for (int ni = 0; ni < TN / 16; ++ni)
              acc[ni][h * (HALF / 16) + mi] = mfma_split(pf[ni], hi, lo, acc[ni][h * (HALF / 16) + mi]);
          }
        }
      }
    }
  }
}

// BM x BN outputs per workgroup of WM x WN wavefronts. Tiles of x (BM rows of
// 64 contraction steps) and of w in LDS, two of each: one is loaded while the
// other is multiplied. w's tile is BN rows of 64 steps, or, for y = x w, 64
// rows of BN columns read through the transposing LDS read.
template <class T, int BM, int BN, int WM, int WN, bool TR, bool ALIGNED, bool LR>
__global__ void __launch_bounds__(64 * WM * WN) mat_kernel(MatArgs a) {
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
  auto slot_of = [&](int64_t i) {  // sorted position -> row of y
    i = min(i, g.end - 1);
    return a.order ? min((int64_t)(uint32_t)a.order[i], a.rows - 1) : i;
  };

  f32x4 acc[TN / 16][TM / 16];
  for (int i = 0; i < TN / 16; ++i)
    for (int j = 0; j < TM / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (!grouped || g.group < a.E) {
    const T* w = (const T*)a.w + (grouped ? (int64_t)g.group * a.ldwe : 0);
    const char* zero = (const char*)&mix_zero16;
    // ---- this lane's 16-byte pieces of both tiles
    const T* xp[AJ];
    const T* wp[BJ];
    uint32_t xk = (lane % 8) ^ (lane / 8);  // chunk of the row: chunk c of row i lies at c ^ (i % 8)
    xk *= 8;
    for (int j = 0; j < AJ; ++j) {
      const int64_t s = slot_of(g.begin + (wave * AJ + j) * 8 + lane / 8);
      xp[j] = (const T*)a.x + s / a.div * a.ldx + xk;
    }
    constexpr int ROWC = BN / 8;  // chunks of a row of the transposed tile
    uint32_t wk[BJ], wc[BJ];      // contraction step, and columns left, of each piece
    for (int j = 0; j < BJ; ++j) {
      if (TR) {
        const uint32_t row = (wave * BJ + j) * (64 / ROWC) + lane / ROWC;
        const uint32_t col = n0 + ((lane % ROWC) ^ tr_swizzle<BN>(row)) * 8;
        wk[j] = row;
        wc[j] = col < a.n ? a.n - col : 0;
        wp[j] = w + (int64_t)row * a.ldw + min(col, a.n - 1);
      } else {
        const uint32_t row = min(n0 + (wave * BJ + j) * 8 + lane / 8, a.n - 1);
        wk[j] = xk;
        wc[j] = 8;
        wp[j] = w + (int64_t)row * a.ldw + xk;
      }
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));
    vec8<T> rx[ALIGNED ? 1 : AJ], rw[ALIGNED ? 1 : BJ];
    auto fetch = [&](uint32_t k0, uint32_t stage) {
      if constexpr (ALIGNED) {
        const uint32_t base = lds0 + stage * STAGE;
        const bool whole = k0 + BK <= a.k;
        for (int j = 0; j < AJ; ++j) {
          const void* p = xp[j] + k0;
          if (!whole && k0 + xk >= a.k) p = zero;
          load_lds16(p, base + (wave * AJ + j) * 1024);
        }
        for (int j = 0; j < BJ; ++j) {
          const void* p = wp[j] + (TR ? (int64_t)k0 * a.ldw : (int64_t)k0);
          if ((!whole && k0 + wk[j] >= a.k) || (TR && wc[j] == 0)) p = zero;
          load_lds16(p, base + BM * BK * 2 + (wave * BJ + j) * 1024);
        }
      } else {
        for (int j = 0; j < AJ; ++j) {
          const int64_t left = (int64_t)a.k - (k0 + xk);
          rx[j] = load8<T>(left > 0 ? xp[j] + k0 : (const T*)zero, left);
        }
        for (int j = 0; j < BJ; ++j) {
          const int64_t left = (int64_t)a.k - (k0 + wk[j]);
          const T* p = wp[j] + (TR ? (int64_t)k0 * a.ldw : (int64_t)k0);
          const int64_t valid = TR ? (left > 0 ? (int64_t)wc[j] : 0) : left;
          rw[j] = load8<T>(valid > 0 ? p : (const T*)zero, valid);
        }
      }
    };
    auto commit = [&](uint32_t stage) {
      if constexpr (!ALIGNED) {
        char* base = lds + stage * STAGE + lane * 16;
        for (int j = 0; j < AJ; ++j) *(vec8<T>*)(base + (wave * AJ + j) * 1024) = rx[j];
        for (int j = 0; j < BJ; ++j) *(vec8<T>*)(base + BM * BK * 2 + (wave * BJ + j) * 1024) = rw[j];
      }
    };
    fetch(0, 0);
    commit(0);
    uint32_t stage = 0;
    for (uint32_t k0 = 0; k0 < a.k; k0 += BK, stage ^= 1) {
      arrived_barrier();
      const bool more = k0 + BK < a.k;
      if (more) fetch(k0 + BK, stage ^ 1);
      const char* xt = lds + stage * STAGE;
      const char* wt = xt + BM * BK * 2;
      for (int kk = 0; kk < BK / 32; ++kk) {
        vec8<T> xf[TM / 16], wf[TN / 16];
        const uint32_t chunk = kk * 4 + lane / 16;
        for (int mi = 0; mi < TM / 16; ++mi) {
          const uint32_t row = wm * TM + mi * 16 + lane % 16;
          xf[mi] = *(const vec8<T>*)(xt + row * 128 + (chunk ^ (row & 7)) * 16);
        }
        for (int ni = 0; ni < TN / 16; ++ni) {
          if (TR) {
            wf[ni] = tr_fragment<T, BN>(wt, wn * TN + ni * 16, kk * 32, lane);
          } else {
            const uint32_t row = wn * TN + ni * 16 + lane % 16;
            wf[ni] = *(const vec8<T>*)(wt + row * 128 + (chunk ^ (row & 7)) * 16);
          }
        }
        for (int ni = 0; ni < TN / 16; ++ni)
          for (int mi = 0; mi < TM / 16; ++mi) acc[ni][mi] = mfma(wf[ni], xf[mi], acc[ni][mi]);
      }
      if (more) commit(stage ^ 1);
    }
    if (LR) add_lowrank<T, TM, TN>(a, g.begin + wm * TM, g.end, n0 + wn * TN, acc, lane);
  }

  // ---- out: a lane holds 4 neighbouring columns of one row
  for (int mi = 0; mi < TM / 16; ++mi) {
    const int64_t i = g.begin + wm * TM + mi * 16 + lane % 16;
    if (i >= g.end) continue;
    const int64_t s = slot_of(i);
    for (int ni = 0; ni < TN / 16; ++ni) {
      const uint32_t n = n0 + wn * TN + ni * 16 + lane / 16 * 4;
      if (n >= a.n) continue;
      f32x4 v = acc[ni][mi];
      if (a.bias)
        for (int q = 0; q < 4; ++q)
          if (n + q < a.n) v[q] += to_float(((const T*)a.bias)[n + q]);
      if (a.y_float) {
        float* y = (float*)a.y + s * a.ldy + n;
        for (int q = 0; q < 4; ++q)
          if (n + q < a.n) y[q] = v[q];
      } else {
        T* y = (T*)a.y + s * a.ldy + n;
        if (n + 4 <= a.n && a.ldy % 4 == 0) {
          T o[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          *(uint64_t*)y = __builtin_bit_cast(uint64_t, o);
        } else {
          for (int q = 0; q < 4; ++q)
            if (n + q < a.n) y[q] = (T)v[q];
        }
      }
    }
  }
}

template <class T, int BM, int BN, int WM, int WN, bool TR, bool ALIGNED>
hipError_t run_mat(const MatArgs& a, hipStream_t s) {
  const uint64_t groups = a.offsets ? (uint64_t)min((int64_t)a.E + 1, a.rows) : 0;
  const uint64_t tiles = (a.offsets ? a.rows / BM + groups : th::ceil_div(a.rows, BM)) * th::ceil_div(a.n, BN);
  constexpr uint32_t bytes = 2 * (BM + BN) * BK * 2;
  if (a.u) mat_kernel<T, BM, BN, WM, WN, TR, ALIGNED, true><<<(uint32_t)tiles, 64 * WM * WN, bytes, s>>>(a);
  else mat_kernel<T, BM, BN, WM, WN, TR, ALIGNED, false><<<(uint32_t)tiles, 64 * WM * WN, bytes, s>>>(a);
  return hipGetLastError();
}

template <class T>
hipError_t mat_typed(const MatArgs& a, int transposed, hipStream_t s) {
  if (a.aligned)
    return transposed ? run_mat<T, 128, 128, 2, 2, true, true>(a, s) : run_mat<T, 128, 128, 2, 2, false, true>(a, s);
  return transposed ? run_mat<T, 128, 128, 2, 2, true, false>(a, s) : run_mat<T, 128, 128, 2, 2, false, false>(a, s);
}

// ---------------------------------------------------------------- weight gradients
// 128 x 128 outputs of one group: both operands are rows of slots, 64 slots a
// step, read through the transposing LDS read.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) outer_kernel(OuterArgs a) {
  constexpr int BN = 128, JOBS = 4;  // 1 KiB loads (4 slots) per wavefront and tile
  constexpr uint32_t TILE = 64 * BN * 2, STAGE = 2 * TILE;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t nt = (a.n + 127) / 128, kt = (a.k + 127) / 128;
  const uint32_t tile = xcd_tile(blockIdx.x, nt * kt * a.E);
  const uint32_t e = tile / (nt * kt), n0 = tile % (nt * kt) % nt * 128, c0 = tile % (nt * kt) / nt * 128;
  const int64_t begin = group_begin(a.offsets, e, a.E, a.slots), end = group_begin(a.offsets, e + 1, a.E, a.slots);
  const char* zero = (const char*)&mix_zero16;
  f32x4 acc[4][4];
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // this lane's pieces: slot row and 16-byte column chunk of each load
  uint32_t row[JOBS], cn[JOBS], ck[JOBS];
  for (int j = 0; j < JOBS; ++j) {
    row[j] = (wave * JOBS + j) * 4 + lane / 16;
    const uint32_t c = ((lane % 16) ^ tr_swizzle<BN>(row[j])) * 8;
    cn[j] = n0 + c;
    ck[j] = c0 + c;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));
  int64_t slot[JOBS];  // of the step that is fetched next; -1 past the group
  auto look = [&](int64_t s0) {
    for (int j = 0; j < JOBS; ++j) {
      const int64_t i = s0 + row[j];
      slot[j] = i < end ? min((int64_t)(uint32_t)a.order[i], a.slots - 1) : -1;
    }
  };
  vec8<T> rn[JOBS], rk[JOBS];
  auto fetch = [&](uint32_t stage) {
    for (int j = 0; j < JOBS; ++j) {
      const bool inn = slot[j] >= 0 && cn[j] < a.n, ink = slot[j] >= 0 && ck[j] < a.k;
      const T* pn = inn ? (const T*)a.dy + slot[j] * a.lddy + cn[j] : (const T*)zero;
      const T* pk = ink ? (const T*)a.x + slot[j] / a.div * a.ldx + ck[j] : (const T*)zero;
      if constexpr (ALIGNED) {
        load_lds16(pn, lds0 + stage * STAGE + (wave * JOBS + j) * 1024);
        load_lds16(pk, lds0 + stage * STAGE + TILE + (wave * JOBS + j) * 1024);
      } else {
        rn[j] = load8<T>(pn, inn ? a.n - cn[j] : 0);
        rk[j] = load8<T>(pk, ink ? a.k - ck[j] : 0);
      }
    }
  };
  auto commit = [&](uint32_t stage) {
    if constexpr (!ALIGNED)
      for (int j = 0; j < JOBS; ++j) {
        char* p = lds + stage * STAGE + (wave * JOBS + j) * 1024 + lane * 16;
        *(vec8<T>*)p = rn[j];
        *(vec8<T>*)(p + TILE) = rk[j];
      }
  };
  if (begin < end) {
    look(begin);
    fetch(0);
    commit(0);
    look(begin + 64);
  }
  uint32_t stage = 0;
  for (int64_t s0 = begin; s0 < end; s0 += 64, stage ^= 1) {
    arrived_barrier();
    const bool more = s0 + 64 < end;
    if (more) {
      fetch(stage ^ 1);
      look(s0 + 128);
    }
    const char* tn = lds + stage * STAGE;
    const char* tk = tn + TILE;
    for (int kk = 0; kk < 2; ++kk) {
      vec8<T> fn[4], fk[4];
      for (int i = 0; i < 4; ++i) fn[i] = tr_fragment<T, BN>(tn, wave / 2 * 64 + i * 16, kk * 32, lane);
      for (int i = 0; i < 4; ++i) fk[i] = tr_fragment<T, BN>(tk, wave % 2 * 64 + i * 16, kk * 32, lane);
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma(fk[i], fn[j], acc[i][j]);
    }
    if (more) commit(stage ^ 1);
  }
  for (int j = 0; j < 4; ++j) {
    const uint32_t n = n0 + wave / 2 * 64 + j * 16 + lane % 16;
    if (n >= a.n) continue;
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = c0 + wave % 2 * 64 + i * 16 + lane / 16 * 4;
      T* o = (T*)a.out + ((int64_t)e * a.n + n) * a.k + c;
      if (c + 4 <= a.k && a.k % 4 == 0) {
        T v[4] = {(T)acc[i][j][0], (T)acc[i][j][1], (T)acc[i][j][2], (T)acc[i][j][3]};
        *(uint64_t*)o = __builtin_bit_cast(uint64_t, v);
      } else {
        for (int q = 0; q < 4; ++q)
          if (c + q < a.k) o[q] = (T)acc[i][j][q];
      }
    }
  }
}

// ---------------------------------------------------------------- low-rank gradients
// Partial sums over a span of one adapter's slots: 16 MR rows of the low-rank
// factor (float, scaled, as a bf16 pair) by 128 columns of the wide operand.
template <class T, int MR>
__global__ void __launch_bounds__(256) low_outer_kernel(LowOuterArgs a, uint32_t ctiles) {
  constexpr int BN = 128, LD = 72;  // LDS row of 64 slots, padded
  __shared__ __attribute__((aligned(16))) char wide[64 * BN * 2];
  __shared__ __attribute__((aligned(16))) bf16_t low[2][MR * 16 * LD];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c0 = blockIdx.x % ctiles * BN, span = blockIdx.x / ctiles;
  const GroupTile g = find_group_tile(a.offsets, a.E, a.E, a.slots, a.span, span, lane);
  if (g.begin >= g.end) return;
  f32x4 acc[MR][2];
  for (int i = 0; i < MR; ++i) acc[i][0] = acc[i][1] = f32x4{0, 0, 0, 0};
  const float se = a.scale ? a.scale[g.group] : 1.0f;
  for (int64_t s0 = g.begin; s0 < g.end; s0 += 64) {
    __syncthreads();
    for (int j = 0; j < 4; ++j) {
      const uint32_t piece = j * 256 + threadIdx.x, row = piece / 16;
      const uint32_t c = c0 + ((piece % 16) ^ tr_swizzle<BN>(row)) * 8;
      const int64_t i = s0 + row;
      vec8<T> v;
      if (i < g.end && c < a.cols) {
        const int64_t s = min((int64_t)(uint32_t)a.order[i], a.slots - 1);
        const T* p = (const T*)a.wide + s / a.div * a.ldwide + c;
        v = load8<T>(p, a.cols - c);
      } else {
        v = load8<T>((const T*)&mix_zero16, 0);
      }
      *(vec8<T>*)(wide + piece * 16) = v;
    }
    for (uint32_t i = threadIdx.x; i < MR * 16 * 64; i += 256) {
      const uint32_t q = i % (MR * 16), row = i / (MR * 16);
      const int64_t at = s0 + row;
      float v = 0;
      if (at < g.end && q < a.r) {
        const int64_t s = min((int64_t)(uint32_t)a.order[at], a.slots - 1);
        v = a.low[s * a.ru + q] * ((a.gate ? a.gate[s] : 1.0f) * se);
      }
      const bf16_t hi = (bf16_t)v;
      low[0][q * LD + row] = hi;
      low[1][q * LD + row] = (bf16_t)(v - (float)hi);
    }
    __syncthreads();
    for (int kk = 0; kk < 2; ++kk) {
      decltype(widen(vec8<T>())) wf[2];
      for (int i = 0; i < 2; ++i) wf[i] = widen(tr_fragment<T, BN>(wide, wave * 32 + i * 16, kk * 32, lane));
      for (int m = 0; m < MR; ++m) {
        const uint32_t at = (m * 16 + lane % 16) * LD + kk * 32 + lane / 16 * 8;
        const bf16x8 hi = *(const bf16x8*)&low[0][at], lo = *(const bf16x8*)&low[1][at];
        for (int i = 0; i < 2; ++i) acc[m][i] = mfma_split(wf[i], hi, lo, acc[m][i]);
      }
    }
  }
  // a lane: row lane % 16 of the low-rank factor, 4 neighbouring columns
  for (int m = 0; m < MR; ++m)
    for (int i = 0; i < 2; ++i) {
      const uint32_t q = m * 16 + lane % 16, c = c0 + wave * 32 + i * 16 + lane / 16 * 4;
      if (q >= a.r) continue;
      float* o = a.partial + ((int64_t)span * a.r + q) * a.cols + c;
      for (int x = 0; x < 4; ++x)
        if (c + x < a.cols) o[x] = acc[m][i][x];
    }
}

// Adds an adapter's partial sums, in slot order.
template <class T>
__global__ void __launch_bounds__(256) low_sum_kernel(LowOuterArgs a) {
  const uint32_t e = blockIdx.y, lane = threadIdx.x & 63;
  uint32_t first = count_group_tiles(a.offsets, a.E, e, a.slots, a.span, lane);
  const int64_t c = group_begin(a.offsets, e + 1, a.E, a.slots) - group_begin(a.offsets, e, a.E, a.slots);
  const uint32_t n = c > 0 ? (uint32_t)((c + a.span - 1) / a.span) : 0;
  const uint64_t size = (uint64_t)a.r * a.cols;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (uint64_t)gridDim.x * 256) {
    const uint64_t at = a.transposed ? i % a.r * a.cols + i / a.r : i;
    float v = 0;
    for (uint32_t p = 0; p < n; ++p) v += a.partial[(uint64_t)(first + p) * size + at];
    ((T*)a.out)[e * size + i] = (T)v;
  }
}

template <class T>
hipError_t low_outer_typed(const LowOuterArgs& a, hipStream_t s) {
  const uint32_t ctiles = (uint32_t)th::ceil_div(a.cols, 128);
  const uint32_t blocks = ctiles * (uint32_t)th::lowrank_spans(a.slots, a.E, a.span);
  if (blocks) {
    if (a.r <= 16) low_outer_kernel<T, 1><<<blocks, 256, 0, s>>>(a, ctiles);
    else if (a.r <= 32) low_outer_kernel<T, 2><<<blocks, 256, 0, s>>>(a, ctiles);
    else if (a.r <= 64) low_outer_kernel<T, 4><<<blocks, 256, 0, s>>>(a, ctiles);
    else low_outer_kernel<T, 8><<<blocks, 256, 0, s>>>(a, ctiles);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint64_t size = (uint64_t)a.r * a.cols;
  low_sum_kernel<T><<<dim3((uint32_t)min(th::ceil_div(size, 256), (uint64_t)1024), a.E), 256, 0, s>>>(a);
  return hipGetLastError();
}

__global__ void __launch_bounds__(256) transpose_kernel(const uint16_t* in, int64_t ld, int64_t lde, uint16_t* out,
                                                        uint32_t rows, uint32_t cols) {
  __shared__ uint16_t tile[64][66];
  const uint32_t r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, e = blockIdx.z;
  for (uint32_t i = threadIdx.x; i < 64 * 64; i += 256) {
    const uint32_t r = r0 + i / 64, c = c0 + i % 64;
    if (r < rows && c < cols) tile[i / 64][i % 64] = in[e * lde + r * ld + c];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 64 * 64; i += 256) {
    const uint32_t c = c0 + i / 64, r = r0 + i % 64;
    if (r < rows && c < cols) out[((int64_t)e * cols + c) * rows + r] = tile[i % 64][i / 64];
  }
}

template <class T>
__global__ void __launch_bounds__(256) sum_choices_kernel(const float* in, T* out, int64_t tokens, uint32_t k,
                                                          uint32_t n) {
  const int64_t size = tokens * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / n;
    float v = 0;
    for (uint32_t j = 0; j < k; ++j) v += in[(t * k + j) * n + i % n];
    out[i] = (T)v;
  }
}

__global__ void __launch_bounds__(256) gate_grad_kernel(const float* u, const float* v, const int32_t* ids,
                                                        const float* scale, float* out, int64_t slots, uint32_t r,
                                                        uint32_t ru, uint32_t E) {
  const int64_t s = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (s >= slots) return;
  const uint32_t e = (uint32_t)ids[s];
  float d = 0;
  if (e < E) {
    for (uint32_t i = 0; i < r; ++i) d += u[s * ru + i] * v[s * ru + i];
    if (scale) d *= scale[e];
  }
  out[s] = d;
}

}  // namespace

hipError_t launch_mat(MixType type, const MatArgs& a, int transposed, hipStream_t s) {
  if (a.rows == 0 || a.n == 0) return hipSuccess;
  if (a.scan || (!transposed && th::narrow_product(a.rows, a.n, a.offsets ? a.E : 1))) return launch_narrow(type, a, s);
  return type == MIX_BF16 ? mat_typed<bf16_t>(a, transposed, s) : mat_typed<f16_t>(a, transposed, s);
}

hipError_t launch_outer(MixType type, const OuterArgs& a, hipStream_t s) {
  const uint64_t blocks = th::ceil_div(a.n, 128) * th::ceil_div(a.k, 128) * a.E;
  constexpr uint32_t bytes = 2 * 2 * 64 * 128 * 2;
  if (type == MIX_BF16 && a.aligned) outer_kernel<bf16_t, true><<<(uint32_t)blocks, 256, bytes, s>>>(a);
  else if (type == MIX_BF16) outer_kernel<bf16_t, false><<<(uint32_t)blocks, 256, bytes, s>>>(a);
  else if (a.aligned) outer_kernel<f16_t, true><<<(uint32_t)blocks, 256, bytes, s>>>(a);
  else outer_kernel<f16_t, false><<<(uint32_t)blocks, 256, bytes, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_low_outer(MixType type, LowOuterArgs a, hipStream_t s) {
  return type == MIX_BF16 ? low_outer_typed<bf16_t>(a, s) : low_outer_typed<f16_t>(a, s);
}

hipError_t launch_transpose(const void* in, int64_t ld, int64_t lde, void* out, uint32_t E, uint32_t rows,
                            uint32_t cols, hipStream_t s) {
  const dim3 grid((uint32_t)th::ceil_div(rows, 64), (uint32_t)th::ceil_div(cols, 64), E);
  transpose_kernel<<<grid, 256, 0, s>>>((const uint16_t*)in, ld, lde, (uint16_t*)out, rows, cols);
  return hipGetLastError();
}

hipError_t launch_sum_choices(MixType type, const float* in, void* out, int64_t tokens, uint32_t k, uint32_t n,
                              hipStream_t s) {
  const uint64_t size = (uint64_t)tokens * n;
  if (!size) return hipSuccess;
  const uint32_t blocks = (uint32_t)min(th::ceil_div(size, 256), (uint64_t)8192);
  if (type == MIX_BF16) sum_choices_kernel<<<blocks, 256, 0, s>>>(in, (bf16_t*)out, tokens, k, n);
  else sum_choices_kernel<<<blocks, 256, 0, s>>>(in, (f16_t*)out, tokens, k, n);
  return hipGetLastError();
}

hipError_t launch_gate_grad(const float* u, const float* v, const int32_t* ids, const float* scale, float* out,
                            int64_t slots, uint32_t r, uint32_t ru, uint32_t E, hipStream_t s) {
  if (!slots) return hipSuccess;
  gate_grad_kernel<<<(uint32_t)th::ceil_div(slots, 256), 256, 0, s>>>(u, v, ids, scale, out, slots, r, ru, E);
  return hipGetLastError();
}

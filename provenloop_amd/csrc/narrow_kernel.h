// The tile kernel of matrix products with few output tiles (see narrow.hip, and
// narrow4.hip for weights of 4 bits).
#pragma once
#include "four_device.h"

namespace mix {

// low[o] = the low-rank part of output (m0 + (tid + o THREADS) / BN, n0 + (tid +
// o THREADS) % BN) for o in FIRST .. FIRST + OUTS, clamped to the tile's rows and
// the product's columns; these outputs' loads go out together.
template <class T, int FIRST, int OUTS, int THREADS, int BN>
__device__ __forceinline__ void lowrank_part(const MatArgs& a, int64_t m0, int64_t mend, uint32_t n0, float* low) {
  const T* p[OUTS];
  const float* u[OUTS];
  int64_t row[OUTS];
#pragma unroll
  for (int o = 0; o < OUTS; ++o) {
    const uint32_t at = threadIdx.x + (FIRST + o) * THREADS;
    row[o] = min(m0 + at / BN, mend - 1) * a.kc;
    p[o] = (const T*)a.p + (int64_t)min(n0 + at % BN, a.n - 1) * a.ldp;
    low[FIRST + o] = 0;
  }
  for (uint32_t j = 0; j < a.kc; ++j) {
    uint32_t e[OUTS];
    float c[OUTS], d[OUTS];
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      e[o] = (uint32_t)a.ids[row[o] + j];
      c[o] = a.gate ? a.gate[row[o] + j] : 1.0f;
      u[o] = a.u + (row[o] + j) * a.ru;
      d[o] = 0;
    }
    // a slot without an adapter takes part with the first one's values, and its product is dropped
    uint32_t i = 0;
    for (; i + 8 <= a.r; i += 8) {
      vec8<T> v[OUTS];
      f32x4 u0[OUTS], u1[OUTS];
#pragma unroll
      for (int o = 0; o < OUTS; ++o) {
        v[o] = load8<T>(p[o] + (e[o] < a.E ? e[o] : 0) * a.ldpe + i, 8);
        u0[o] = *(const f32x4*)(u[o] + i);
        u1[o] = *(const f32x4*)(u[o] + i + 4);
      }
#pragma unroll
      for (int o = 0; o < OUTS; ++o)
#pragma unroll
        for (int q = 0; q < 8; ++q) d[o] = fmaf((q < 4 ? u0[o] : u1[o])[q % 4], (float)v[o][q], d[o]);
    }
    for (; i < a.r; ++i)
#pragma unroll
      for (int o = 0; o < OUTS; ++o)
        d[o] = fmaf(u[o][i], (float)p[o][(e[o] < a.E ? e[o] : 0) * a.ldpe + i], d[o]);
#pragma unroll
    for (int o = 0; o < OUTS; ++o)
      if (e[o] < a.E) low[FIRST + o] = fmaf(a.scale ? c[o] * a.scale[e[o]] : c[o], d[o], low[FIRST + o]);
  }
}
// Of all OUTS outputs, 4 at a time: what 8 have on the way at once is more than 256
// registers, and a CU then holds one workgroup of 4 wavefronts (64 x 32 tiles of
// 4-bit weights, 3584 -> 3584 with rank 32 and A x: 256 rows 52.8 us and 34.3 with
// 4, 512 rows 97 and 59; with 2 the same as with 4).
template <class T, int OUTS, int THREADS, int BN>
__device__ __forceinline__ void lowrank_at(const MatArgs& a, int64_t m0, int64_t mend, uint32_t n0, float (&low)[OUTS]) {
  static_assert(OUTS <= 4 || OUTS == 8);
  lowrank_part<T, 0, OUTS == 8 ? 4 : OUTS, THREADS, BN>(a, m0, mend, n0, low);
  if constexpr (OUTS == 8) {
    __builtin_amdgcn_sched_barrier(0);
    lowrank_part<T, 4, 4, THREADS, BN>(a, m0, mend, n0, low);
  }
}

// A line of 4-bit weights is 1 KiB of codes, 128 columns of 16 rows or 64 of 32,
// and up to 192 bytes of scales and zeros.
template <int MT, int NT, bool FOUR>
constexpr uint32_t narrow_stage() {
  return FOUR ? 16 * MT * (128 / NT) * 2 + 1024 + 256 : 16 * (MT + NT) * 128;
}
template <int MT, int NT, int WAVES, int S, bool FOUR = false>
constexpr uint32_t narrow_lds() {
  const uint32_t rings = WAVES * S * narrow_stage<MT, NT, FOUR>(), sums = WAVES * 16 * MT * (16 * NT + 4) * 4;
  return rings > sums ? rings : sums;
}

// 16 MT rows by 16 NT columns, WAVES wavefronts, S lines of each row in a ring.
// TR: w is k x n, and a line of it 64 rows of 16 NT values, read through the
// transposing LDS read. FOUR: w has 4 bits, and a lane makes its operands' values
// from the codes of its own lines.
template <class T, int MT, int NT, int WAVES, int S, bool TR, bool ALIGNED, bool LR, bool FOUR = false>
__global__ void __launch_bounds__(64 * WAVES) narrow_kernel(MatArgs a, uint32_t shares) {
  constexpr int BM = 16 * MT, BN = 16 * NT, LD = BN + 4, THREADS = 64 * WAVES;
  constexpr int OUTS = BM * BN / THREADS ? BM * BN / THREADS : 1;
  constexpr int LINE = FOUR ? 128 / NT : 64;       // contraction steps
  constexpr int LOADS = FOUR ? MT * 2 * (LINE / 64) + 2 : 2 * (MT + NT);  // of a line: 8 rows by 64 steps each
  constexpr int FEWEST = LINE / 64 + 2;  // FOUR: of a line of at most 8 rows
  constexpr uint32_t STAGE = narrow_stage<MT, NT, FOUR>();
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  float* red = (float*)lds;                        // WAVES x BM x LD, after the rings
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ntiles = (a.n + BN - 1) / BN;

  // ---- which rows and columns
  const bool scan = !FOUR && a.scan, grouped = a.offsets != nullptr;
  GroupTile g{0, 0, 0};
  uint32_t n0, share = 0;
  int32_t* list = (int32_t*)(lds + narrow_lds<MT, NT, WAVES, S>());  // scan: this group's slots
  uint32_t listed = 0;
  if (scan) {
    // workgroup (column tile, group, share): the group's slots by looking at every slot's
    n0 = blockIdx.x % ntiles * BN;
    g.group = blockIdx.x / ntiles % a.E;
    share = blockIdx.x / ntiles / a.E;
    if (wave == 0) {
      for (int64_t at = 0; at < a.rows; at += 512) {
        uint32_t e[8];
        for (int i = 0; i < 8; ++i) {
          const int64_t s = at + i * 64 + lane;
          e[i] = s < a.rows ? (uint32_t)a.ids[s] : ~0u;
        }
        for (int i = 0; i < 8; ++i) {
          const uint64_t here = __ballot(e[i] == g.group);
          if (e[i] == g.group) list[listed + __popcll(here & ((1ull << lane) - 1))] = (int32_t)(at + i * 64 + lane);
          listed += __popcll(here);
        }
      }
      if (lane == 0) list[th::NARROW_SCAN_SLOTS] = (int32_t)listed;
    }
    __syncthreads();
    listed = (uint32_t)list[th::NARROW_SCAN_SLOTS];
    g.begin = (int64_t)share * BM;
    g.end = listed;
  } else {
    const uint32_t mtiles = grouped ? count_group_tiles(a.offsets, a.E, a.E + 1, a.rows, BM, lane)
                                    : (uint32_t)((a.rows + BM - 1) / BM);
    if (blockIdx.x >= mtiles * ntiles) return;
    // row tiles of one column tile side by side on an XCD, whose L2 then holds the weight's rows once
    const uint32_t tile = xcd_tile(blockIdx.x, mtiles * ntiles);
    const uint32_t mt = tile % mtiles;
    n0 = tile / mtiles * BN;
    g = GroupTile{0, (int64_t)mt * BM, min((int64_t)(mt + 1) * BM, a.rows)};
    if (grouped) g = find_group_tile(a.offsets, a.E, a.E + 1, a.rows, BM, mt, lane);
  }
  auto slot_of = [&](int64_t i) -> int64_t {
    i = min(i, g.end - 1);
    if (scan) return list[i];
    return a.order ? min((int64_t)(uint32_t)a.order[i], a.rows - 1) : i;
  };
  auto row_of = [&](int64_t i) -> int64_t { return (uint32_t)slot_of(i) / a.div; };  // of x: slots are below 2^31
  const bool has = !grouped || g.group < a.E;
  const T* w = (const T*)a.w + (grouped || scan ? (int64_t)g.group * a.ldwe : 0);
  const T* zero = (const T*)&mix_zero16;
  const uint32_t lines = has ? (a.k + LINE - 1) / LINE : 0;
  const uint32_t mine = wave < lines ? (lines - wave + WAVES - 1) / WAVES : 0;  // this wavefront's: wave + i WAVES

  for (int64_t m0 = g.begin; m0 < g.end; m0 += (int64_t)shares * BM) {
    f32x4 acc[NT][MT];
#pragma unroll
    for (int ni = 0; ni < NT; ++ni)
#pragma unroll
      for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = f32x4{0, 0, 0, 0};
    float low[OUTS] = {};
    if constexpr (FOUR) {
      constexpr int STEPS = LINE / 32, SUBS = LINE / 64;
      const th::FourLayout f = a.four.at;
      const uint32_t xk = ((lane % 8) ^ (lane / 8)) * 8;  // chunk c of row i lies at c ^ (i % 8)
      const T* p[2 * MT];
      // only rows that exist are loaded, 8 at a time: with 4-bit weights a tile's x is
      // the larger part. What else lies in their places gives columns of no output.
      const uint32_t rows_left = (uint32_t)min(g.end - m0, (int64_t)BM);
      const bool all_rows = rows_left > BM - 8;
#pragma unroll
      for (int j = 0; j < 2 * MT; ++j) p[j] = (const T*)a.x + row_of(m0 + j * 8 + lane / 8) * a.ldx + xk;
      const uint64_t e = grouped && has ? g.group : 0;
      const uint32_t rows = f.strips * 16;  // of the weights as they are stored
      const uint32_t strip = n0 / 16 + (NT == 2 ? lane / 32 : 0);
      const uint8_t* codes = a.four.codes + e * f.codes() + (uint64_t)strip * f.blocks * 512 + lane % (64 / NT) * 16;
      // lanes 0 .. 7: 8 rows' scales of one step's group each; 8 .. 11: 16 rows' zeros
      const bool of_zeros = lane >= 8;
      const uint32_t piece = of_zeros ? lane % NT : lane % (2 * NT), part = of_zeros ? (lane - 8) / NT : lane / (2 * NT);
      const uint32_t row = n0 + piece * (of_zeros ? 16 : 8);
      const uint8_t* fine = of_zeros ? (a.four.zeros ? a.four.zeros + e * f.scales() + row : nullptr)
                                     : (const uint8_t*)a.four.scales + (e * f.scales() + row) * 2;
      const uint64_t per = (uint64_t)rows * (of_zeros ? 1 : 2);  // bytes of a group
      const bool in_rows = row < rows;
      const uint32_t fine_lanes = a.four.zeros ? 12 : 8;
      const uint32_t turns = __builtin_amdgcn_readfirstlane(mine);
      const char* ring = lds + wave * (S * STAGE);
      const uint32_t base = __builtin_amdgcn_readfirstlane(lds_address(ring));
      auto load = [&](uint32_t i, uint32_t stage) __attribute__((always_inline)) {
        const uint32_t line = wave + i * WAVES, k0 = line * LINE, to = base + stage * STAGE;
        {
          const bool in = NT == 2 ? strip < f.strips : line * 2 + lane / 32 < f.blocks;
          load_lds16(in ? (const void*)(codes + (uint64_t)line * (1024 / NT)) : zero, to + BM * LINE * 2);
        }
#pragma unroll
        for (int h = 0; h < SUBS; ++h)
#pragma unroll
          for (int j = 0; j < 2 * MT; ++j)
            if (j * 8 + lane / 8 < rows_left)
              load_lds16(k0 + h * 64 + xk < a.k ? p[j] + k0 + h * 64 : zero, to + (h * 2 * MT + j) * 1024);
        if (lane < fine_lanes) {
          const uint32_t k = k0 + part * 32;
          const bool in = in_rows && k < f.blocks * 64;
          load_lds16(in ? (const void*)(fine + (k >> f.shift) * per) : zero, to + BM * LINE * 2 + 1024);
        }
      };
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < (int)turns) load(i, i);
      if (LR) lowrank_at<T, OUTS, THREADS, BN>(a, m0, g.end, n0, low);  // while the first lines are on their way
      uint32_t stage = 0;
      for (uint32_t i = 0; i < turns; ++i) {
        if (i + S > turns) arrived<0>();
        else if (all_rows) arrived<(S - 1) * LOADS>();
        else arrived<(S - 1) * FEWEST>();
        const char *xt = ring + stage * STAGE, *ct = xt + BM * LINE * 2, *st = ct + 1024;
        uint2 q[2];
        vec8<T> xf[STEPS][MT];
        T scale[STEPS][NT];
        uint32_t zeros[STEPS][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h) q[h] = *(const uint2*)(ct + h * 512 + lane * 8);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
#pragma unroll
          for (int ni = 0; ni < NT; ++ni) {
            const uint32_t at = (s * NT + ni) * 16 + lane % 16;
            scale[s][ni] = ((const T*)st)[at];
            zeros[s][ni] = a.four.zeros ? ((const uint8_t*)st)[128 + at] : 8;
          }
#pragma unroll
          for (int mi = 0; mi < MT; ++mi) {
            const uint32_t r = mi * 16 + lane % 16, c = s % 2 * 4 + lane / 16;
            xf[s][mi] = *(const vec8<T>*)(xt + s / 2 * (BM * 128) + r * 128 + (c ^ (r & 7)) * 16);
          }
        }
        answered();  // the stage has been read before its place is loaded again
        if (i + S < turns) load(i + S, stage);
        stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int ni = 0; ni < NT; ++ni) {
            const uint2 w = q[NT == 2 ? ni : s / 2];
            const vec8<T> wf = four_values(s % 2 ? w.y : w.x, FourScale<T>(scale[s][ni], zeros[s][ni]));
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = mfma(wf, xf[s][mi], acc[ni][mi]);
          }
      }
    } else if constexpr (ALIGNED) {
      const uint32_t xk = ((lane % 8) ^ (lane / 8)) * 8;  // chunk c of row i lies at c ^ (i % 8)
      constexpr int CH = 2 * NT;                          // chunks of a row of a transposed line
      const T* p[LOADS];
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int jw = j - 2 * MT;
        if (j < 2 * MT) {
          p[j] = (const T*)a.x + row_of(m0 + j * 8 + lane / 8) * a.ldx + xk;
        } else if constexpr (TR) {
          const uint32_t row = jw * (64 / CH) + lane / CH, col = n0 + ((lane % CH) ^ tr_swizzle<BN>(row)) * 8;
          p[j] = col < a.n ? w + (int64_t)row * a.ldw + col : nullptr;
        } else {
          p[j] = w + (int64_t)min(n0 + jw * 8 + lane / 8, a.n - 1) * a.ldw + xk;
        }
      }
      const char* ring = lds + wave * (S * STAGE);
      const uint32_t base = __builtin_amdgcn_readfirstlane(lds_address(ring));
      auto load = [&](uint32_t i, uint32_t stage) __attribute__((always_inline)) {
        const uint32_t k0 = (wave + i * WAVES) * 64;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const T* q;
          if (TR && j >= 2 * MT)
            q = k0 + (j - 2 * MT) * (64 / CH) + lane / CH < a.k && p[j] ? p[j] + (int64_t)k0 * a.ldw : zero;
          else
            q = k0 + xk < a.k ? p[j] + k0 : zero;
          load_lds16(q, base + stage * STAGE + j * 1024);
        }
      };
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < (int)mine) load(i, i);
      if (LR) lowrank_at<T, OUTS, THREADS, BN>(a, m0, g.end, n0, low);  // while the first lines are on their way
      uint32_t stage = 0;
      for (uint32_t i = 0; i < mine; ++i) {
        if (i + S <= mine) arrived<(S - 1) * LOADS>();
        else arrived<0>();
        const char *xt = ring + stage * STAGE, *wt = xt + BM * 128;
        vec8<T> xf[2][MT], wf[2][NT];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const uint32_t c = kk * 4 + lane / 16;
#pragma unroll
          for (int mi = 0; mi < MT; ++mi) {
            const uint32_t r = mi * 16 + lane % 16;
            xf[kk][mi] = *(const vec8<T>*)(xt + r * 128 + (c ^ (r & 7)) * 16);
          }
#pragma unroll
          for (int ni = 0; ni < NT; ++ni) {
            const uint32_t r = ni * 16 + lane % 16;
            if constexpr (TR) wf[kk][ni] = tr_fragment<T, BN>(wt, ni * 16, kk * 32, lane);
            else wf[kk][ni] = *(const vec8<T>*)(wt + r * 128 + (c ^ (r & 7)) * 16);
          }
        }
        answered();  // the stage has been read before its place is loaded again
        if (i + S < mine) load(i + S, stage);
        stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int ni = 0; ni < NT; ++ni)
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = mfma(wf[kk][ni], xf[kk][mi], acc[ni][mi]);
      }
    } else {
      const uint32_t kl = lane / 16 * 16;  // this lane's 16 values of a line
      const T *xp[MT], *wp[NT];
#pragma unroll
      for (int mi = 0; mi < MT; ++mi) xp[mi] = (const T*)a.x + row_of(m0 + mi * 16 + lane % 16) * a.ldx + kl;
#pragma unroll
      for (int ni = 0; ni < NT; ++ni) wp[ni] = w + (int64_t)min(n0 + ni * 16 + lane % 16, a.n - 1) * a.ldw + kl;
      struct Line {
        vec8<T> x[MT][2], w[NT][2];
      };
      auto piece = [&](const T* p, int64_t left) __attribute__((always_inline)) -> vec8<T> {
        return load8<T>(left > 0 ? p : zero, left);
      };
      auto fetch = [&](Line& s, uint32_t i) __attribute__((always_inline)) {
        const uint32_t k0 = (wave + i * WAVES) * 64;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t left = (int64_t)a.k - (k0 + kl + h * 8);
#pragma unroll
          for (int ni = 0; ni < NT; ++ni) s.w[ni][h] = piece(wp[ni] + k0 + h * 8, left);
#pragma unroll
          for (int mi = 0; mi < MT; ++mi) s.x[mi][h] = piece(xp[mi] + k0 + h * 8, left);
        }
      };
      Line s[2];
      if (mine) fetch(s[0], 0);
      if (LR) lowrank_at<T, OUTS, THREADS, BN>(a, m0, g.end, n0, low);
      for (uint32_t i = 0; i < mine; i += 2) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (i + q >= mine) break;
          if (i + q + 1 < mine) fetch(s[q ^ 1], i + q + 1);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int ni = 0; ni < NT; ++ni)
#pragma unroll
              for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = mfma(s[q].w[ni][h], s[q].x[mi][h], acc[ni][mi]);
        }
      }
    }
    __syncthreads();  // every wavefront's ring has been read
#pragma unroll
    for (int ni = 0; ni < NT; ++ni)
#pragma unroll
      for (int mi = 0; mi < MT; ++mi)
        *(f32x4*)&red[(wave * BM + mi * 16 + lane % 16) * LD + ni * 16 + lane / 16 * 4] = acc[ni][mi];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      const uint32_t at = threadIdx.x + o * THREADS, m = at / BN, n = n0 + at % BN;
      const int64_t i = m0 + m;
      if (at >= BM * BN || i >= g.end || n >= a.n) continue;
      float v = 0;
#pragma unroll
      for (int q = 0; q < WAVES; ++q) v += red[(q * BM + m) * LD + at % BN];
      v += low[o];
      if (a.bias) v += to_float(((const T*)a.bias)[n]);
      const int64_t s = slot_of(i);
      if (a.y_float) ((float*)a.y)[s * a.ldy + n] = v;
      else ((T*)a.y)[s * a.ldy + n] = (T)v;
    }
    if (!scan) break;
    __syncthreads();
  }
}

}  // namespace mix

// Matrix products with few output tiles: y = x w^T for decodes, small batches and
// the low-rank factors A x, and y = x w for the gradients of small batches.
//
// What bounds them is the latency of reading w (a decode reads each weight for
// a few rows) and how many CUs take part, not the matrix cores. So a workgroup
// takes a small tile (16 or 32 rows by 16 or 32 columns), and its wavefronts
// split the contraction among them: a wavefront's step is one 128-byte line (64
// values) of every row. Each has a ring of lines of its own in LDS, filled by
// asynchronous loads of whole lines and waited for by that wavefront alone, so
// nothing but the last sum, in LDS and in order, needs a barrier. Measured
// against operands loaded into registers in the matrix instructions' layout
// (16 rows by 64 bytes a load): 32 x 3584 x 3584 6.7 us against 13.2, 250 x 1536
// x 1536 6.7 against 12.3, 8192 x 32 x 3584 10.8 against 16.8; one row of 1536 x
// 1536 2.8 against 4.4.
//
// Operands whose rows do not start on 16 bytes go through registers, 32 bytes a
// lane from (l / 16) * 32 on in a line, two matrix instructions' worth; the
// contraction is then taken in another order, the same for both operands.
//
// The low-rank part of the shared projection is a dot product of `rank` floats
// per output and choice, in ordinary float arithmetic: rows of a small batch
// seldom share an adapter.
#include "mixture_device.h"

namespace {

// low[o] = the low-rank part of output (m0 + (tid + o THREADS) / BN, n0 + (tid +
// o THREADS) % BN), clamped to the tile's rows and the product's columns; the
// outputs' loads go out together.
template <class T, int OUTS, int THREADS, int BN>
__device__ __forceinline__ void lowrank_at(const MatArgs& a, int64_t m0, int64_t mend, uint32_t n0, float (&low)[OUTS]) {
  const T* p[OUTS];
  const float* u[OUTS];
  int64_t row[OUTS];
#pragma unroll
  for (int o = 0; o < OUTS; ++o) {
    const uint32_t at = threadIdx.x + o * THREADS;
    row[o] = min(m0 + at / BN, mend - 1) * a.kc;
    p[o] = (const T*)a.p + (int64_t)min(n0 + at % BN, a.n - 1) * a.ldp;
    low[o] = 0;
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
      if (e[o] < a.E) low[o] = fmaf(a.scale ? c[o] * a.scale[e[o]] : c[o], d[o], low[o]);
  }
}

template <int MT, int NT, int WAVES, int S>
constexpr uint32_t narrow_lds() {
  const uint32_t rings = WAVES * S * 16 * (MT + NT) * 128, sums = WAVES * 16 * MT * (16 * NT + 4) * 4;
  return rings > sums ? rings : sums;
}

// 16 MT rows by 16 NT columns, WAVES wavefronts, S lines of each row in a ring.
// TR: w is k x n, and a line of it 64 rows of 16 NT values, read through the
// transposing LDS read.
template <class T, int MT, int NT, int WAVES, int S, bool TR, bool ALIGNED, bool LR>
__global__ void __launch_bounds__(64 * WAVES) narrow_kernel(MatArgs a, uint32_t shares) {
  constexpr int BM = 16 * MT, BN = 16 * NT, LD = BN + 4, THREADS = 64 * WAVES;
  constexpr int OUTS = BM * BN / THREADS ? BM * BN / THREADS : 1;
  constexpr int LOADS = 2 * (MT + NT);             // of a line of every row, 8 rows each
  constexpr uint32_t STAGE = (BM + BN) * 128;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  float* red = (float*)lds;                        // WAVES x BM x LD, after the rings
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ntiles = (a.n + BN - 1) / BN;

  // ---- which rows and columns
  const bool scan = a.scan, grouped = a.offsets != nullptr;
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
  const bool has = !grouped || g.group < a.E;
  const T* w = (const T*)a.w + (grouped || scan ? (int64_t)g.group * a.ldwe : 0);
  const T* zero = (const T*)&mix_zero16;
  const uint32_t lines = has ? (a.k + 63) / 64 : 0;
  const uint32_t mine = wave < lines ? (lines - wave + WAVES - 1) / WAVES : 0;  // this wavefront's: wave + i WAVES

  for (int64_t m0 = g.begin; m0 < g.end; m0 += (int64_t)shares * BM) {
    f32x4 acc[NT][MT];
#pragma unroll
    for (int ni = 0; ni < NT; ++ni)
#pragma unroll
      for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = f32x4{0, 0, 0, 0};
    float low[OUTS] = {};
    if constexpr (ALIGNED) {
      const uint32_t xk = ((lane % 8) ^ (lane / 8)) * 8;  // chunk c of row i lies at c ^ (i % 8)
      constexpr int CH = 2 * NT;                          // chunks of a row of a transposed line
      const T* p[LOADS];
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int jw = j - 2 * MT;
        if (j < 2 * MT) {
          p[j] = (const T*)a.x + slot_of(m0 + j * 8 + lane / 8) / a.div * a.ldx + xk;
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
      for (int mi = 0; mi < MT; ++mi) xp[mi] = (const T*)a.x + slot_of(m0 + mi * 16 + lane % 16) / a.div * a.ldx + kl;
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

template <class T, int MT, int NT, int WAVES, int S>
hipError_t run(const MatArgs& a, int transposed, hipStream_t s) {
  constexpr uint32_t BM = 16 * MT, BN = 16 * NT, most = narrow_lds<MT, NT, WAVES, S>() + (th::NARROW_SCAN_SLOTS + 1) * 4;
  const uint64_t ntiles = th::ceil_div(a.n, BN);
  uint64_t mtiles = th::ceil_div(a.rows, BM), blocks;
  uint32_t shares = 1;
  if (a.scan) {
    // workgroups of one group: as many as its slots can need, no more than fill the GPU
    shares = (uint32_t)min(mtiles, th::ceil_div(256, ntiles * a.E));
    blocks = ntiles * a.E * shares;
  } else {
    if (a.offsets) mtiles = a.rows / BM + (uint64_t)min((int64_t)a.E + 1, a.rows);
    blocks = mtiles * ntiles;
  }
  const uint32_t bytes = a.scan ? most : narrow_lds<MT, NT, WAVES, S>();
  auto go = [&]<bool TR, bool ALIGNED>() {
    return a.u ? launch<narrow_kernel<T, MT, NT, WAVES, S, TR, ALIGNED, true>, most>(blocks, 64 * WAVES, bytes, s, a, shares)
               : launch<narrow_kernel<T, MT, NT, WAVES, S, TR, ALIGNED, false>, most>(blocks, 64 * WAVES, bytes, s, a, shares);
  };
  if (transposed) return go.template operator()<true, true>();
  return a.aligned ? go.template operator()<false, true>() : go.template operator()<false, false>();
}

template <class T>
hipError_t typed(const MatArgs& a, int transposed, hipStream_t s) {
  switch (th::narrow_tile(a.rows, a.n, a.offsets || a.scan ? a.E : 1)) {
    case th::NARROW_16x16: return run<T, 1, 1, 8, 2>(a, transposed, s);
    case th::NARROW_16x16_MANY: return run<T, 1, 1, 4, 2>(a, transposed, s);
    case th::NARROW_32x16: return run<T, 2, 1, 8, 3>(a, transposed, s);
    default: return run<T, 2, 2, 4, 2>(a, transposed, s);
  }
}

}  // namespace

hipError_t launch_narrow(MixType type, const MatArgs& a, int transposed, hipStream_t s) {
  return type == MIX_BF16 ? typed<bf16_t>(a, transposed, s) : typed<f16_t>(a, transposed, s);
}

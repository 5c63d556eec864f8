// Large matrix products, y = x w^T or y = x w, of ragged groups and of the
// shared projection with its low-rank adapters: which kernel takes which.
#include "wide_kernel.h"

using namespace mix;

namespace {

// wide_kernel's product for operands whose rows do not start on 16 bytes or
// whose widths are not multiples of 8 (grouped products, which have no workspace
// for copies, and small gradients): tiles pass through registers, with loads
// that end at a row's end.
template <class T, int BM, int BN, int WM, int WN, bool TR, bool LR>
__global__ void __launch_bounds__(64 * WM * WN) unaligned_kernel(MatArgs a) {
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
  uint32_t* slots = (uint32_t*)(lds + wide_slots<T, BM, BN, 2, LR>());
  for (uint32_t i = threadIdx.x; i < BM; i += 64 * WAVES) {
    const int64_t at = min(g.begin + i, g.end - 1);
    slots[i] = a.order ? (uint32_t)min((int64_t)(uint32_t)a.order[at], a.rows - 1) : (uint32_t)at;
  }
  __syncthreads();

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
      const uint32_t s = slots[(wave * AJ + j) * 8 + lane / 8];
      xp[j] = (const T*)a.x + (int64_t)(s / a.div) * a.ldx + xk;
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
    vec8<T> rx[AJ], rw[BJ];
    auto fetch = [&](uint32_t k0) {
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
    };
    auto commit = [&](uint32_t stage) {
      char* base = lds + stage * STAGE + lane * 16;
      for (int j = 0; j < AJ; ++j) *(vec8<T>*)(base + (wave * AJ + j) * 1024) = rx[j];
      for (int j = 0; j < BJ; ++j) *(vec8<T>*)(base + BM * BK * 2 + (wave * BJ + j) * 1024) = rw[j];
    };
    fetch(0);
    commit(0);
    LowLists<BM>& lists = *(LowLists<BM>*)(slots + BM);
    if (LR) list_adapters<BM, 64 * WAVES>(a, g.begin, g.end, lists);
    uint32_t stage = 0;
    for (uint32_t k0 = 0; k0 < a.k; k0 += BK, stage ^= 1) {
      __syncthreads();
      const bool more = k0 + BK < a.k;
      if (more) fetch(k0 + BK);
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
    if (LR) add_lowrank<T, BM, BN, WM, WN>(a, g.begin, g.end, n0, lds, lists, acc);
  }

  __syncthreads();
  char* own = lds + wave * (TM * TN * 2);
  const uint32_t rows = (uint32_t)(g.end - g.begin);
  const Out out{a.y, a.ldy, a.n, a.bias};
  if (a.y_float) put<float, T, TM, TN>(out, acc, own, slots, wm * TM, rows, n0 + wn * TN, lane);
  else put<T, T, TM, TN>(out, acc, own, slots, wm * TM, rows, n0 + wn * TN, lane);
}

template <class T, int BM, int BN, int WM, int WN, int S, bool TR, bool LR>
hipError_t run(const MatArgs& a, hipStream_t s) {
  constexpr uint32_t bytes = wide_lds<T, BM, BN, S, LR>();
  const uint64_t groups = a.offsets ? (uint64_t)min((int64_t)a.E + 1, a.rows) : 0;
  const uint64_t tiles = (a.offsets ? a.rows / BM + groups : th::ceil_div(a.rows, BM)) * th::ceil_div(a.n, BN);
  if constexpr (S > 0 && BM * BN > 128 * 128)
    return launch<wide_kernel<T, BM, BN, WM, WN, S, TR, LR>, bytes>(tiles, 64 * WM * WN, bytes, s, a);
  else
    return launch<unaligned_kernel<T, BM, BN, WM, WN, TR, LR>, bytes>(tiles, 64 * WM * WN, bytes, s, a);
}

template <class T, bool TR, bool LR>
hipError_t sized(const MatArgs& a, hipStream_t s) {
  if (!a.aligned) return run<T, 128, 128, 2, 2, 2, TR, LR>(a, s);
  return th::wide_square(a.rows, a.n, a.offsets ? a.E : 1) ? run<T, 256, 256, 2, 4, 2, TR, LR>(a, s)
                                                           : run<T, 256, 128, 4, 2, 3, TR, LR>(a, s);
}

template <class T>
hipError_t typed(const MatArgs& a, int transposed, hipStream_t s) {
  if (transposed) return a.u ? sized<T, true, true>(a, s) : sized<T, true, false>(a, s);
  return a.u ? sized<T, false, true>(a, s) : sized<T, false, false>(a, s);
}

}  // namespace

hipError_t launch_mat(MixType type, const MatArgs& a, int transposed, hipStream_t s) {
  if (a.rows == 0 || a.n == 0) return hipSuccess;
  if (a.scan || ((!transposed || a.aligned) && th::narrow_product(a.rows, a.n, a.k, a.offsets ? a.E : 1)))
    return launch_narrow(type, a, transposed, s);
  return type == MIX_BF16 ? typed<bf16_t>(a, transposed, s) : typed<f16_t>(a, transposed, s);
}

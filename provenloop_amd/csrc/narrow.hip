// Matrix products with few rows of output tiles: y = x w^T for decodes, small
// batches and the low-rank factors A x.
//
// What bounds them is the latency of reading w (a decode reads each weight for
// a few rows) and how many CUs take part, not the matrix cores. So a workgroup
// takes a small tile (16 to 64 rows by 16 or 32 columns), its 8 wavefronts split
// the contraction among them, and operands go straight from memory into
// registers in the matrix instructions' layout, several 128-byte lines of each
// row in flight a wavefront; the wavefronts' sums meet in LDS, added in order.
//
// A wavefront's step is one 128-byte line (64 values) of every row: lane l reads
// 32 bytes of row l % 16 from (l / 16) * 32 on, two matrix instructions' worth.
// The contraction steps are thereby taken in another order than memory's, the
// same for both operands.
//
// The low-rank part of the shared projection is a dot product of `rank` floats
// per output and choice, in ordinary float arithmetic: rows of a small batch
// seldom share an adapter, and the loads run under the weights'.
#include "mixture_device.h"

namespace {

constexpr int WAVES = 8, THREADS = 64 * WAVES;

template <class T>
__device__ __forceinline__ float lowrank_at(const MatArgs& a, int64_t row, uint32_t n) {
  float sum = 0;
  for (uint32_t j = 0; j < a.kc; ++j) {
    const int64_t s = row * a.kc + j;
    const uint32_t e = (uint32_t)a.ids[s];
    if (e >= a.E) continue;
    const T* p = (const T*)a.p + (int64_t)e * a.ldpe + (int64_t)n * a.ldp;
    const float* u = a.u + s * a.ru;
    float d = 0;
    uint32_t i = 0;
    for (; i + 8 <= a.r; i += 8) {
      const vec8<T> v = load8<T>(p + i, 8);
      const f32x4 u0 = *(const f32x4*)(u + i), u1 = *(const f32x4*)(u + i + 4);
      for (int q = 0; q < 4; ++q) d = fmaf(u0[q], (float)v[q], d);
      for (int q = 0; q < 4; ++q) d = fmaf(u1[q], (float)v[q + 4], d);
    }
    for (; i < a.r; ++i) d = fmaf(u[i], (float)p[i], d);
    float c = a.gate ? a.gate[s] : 1.0f;
    if (a.scale) c *= a.scale[e];
    sum = fmaf(c, d, sum);
  }
  return sum;
}

template <class T, int MT, int NT, bool ALIGNED, bool LR>
__global__ void __launch_bounds__(THREADS) narrow_kernel(MatArgs a, uint32_t shares) {
  constexpr int BM = 16 * MT, BN = 16 * NT, LD = BN + 4;
  constexpr int U = MT * NT == 1 ? 4 : MT * NT == 2 ? 3 : MT * NT == 4 ? 2 : 1;  // lines of a row, twice, in registers
  constexpr int OUTS = BM * BN / THREADS ? BM * BN / THREADS : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* red = (float*)lds;                       // WAVES x BM x LD
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ntiles = (a.n + BN - 1) / BN;

  // ---- which rows and columns
  const bool scan = a.scan, grouped = a.offsets != nullptr;
  GroupTile g{0, 0, 0};
  uint32_t n0, share = 0;
  int32_t* list = (int32_t*)(red + WAVES * BM * LD);  // scan: this group's slots
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
  const uint32_t kl = lane / 16 * 16;  // this lane's 16 values of a line
  const uint32_t lines = (a.k + 63) / 64;
  const T* wp[NT];
  for (int ni = 0; ni < NT; ++ni) wp[ni] = w + (int64_t)min(n0 + ni * 16 + lane % 16, a.n - 1) * a.ldw + kl;

  for (int64_t m0 = g.begin; m0 < g.end; m0 += (int64_t)shares * BM) {
    const T* xp[MT];
    for (int mi = 0; mi < MT; ++mi) xp[mi] = (const T*)a.x + slot_of(m0 + mi * 16 + lane % 16) / a.div * a.ldx + kl;
    f32x4 acc[NT][MT];
    for (int ni = 0; ni < NT; ++ni)
      for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = f32x4{0, 0, 0, 0};
    struct Step {
      vec8<T> x[U][MT][2], w[U][NT][2];
    };
    auto piece = [&](const T* p, int64_t left) __attribute__((always_inline)) -> vec8<T> {
      if constexpr (ALIGNED) return *(const vec8<T>*)(left > 0 ? p : zero);
      else return load8<T>(left > 0 ? p : zero, left);
    };
    // a line that ends within the contraction, or is past it, reads zeros there
    auto fetch = [&](Step& s, uint32_t line) __attribute__((always_inline)) {
      for (int q = 0; q < U; ++q) {
        const uint32_t k0 = (line + q * WAVES) * 64;
        if (ALIGNED && k0 + 64 <= a.k) {
          for (int ni = 0; ni < NT; ++ni)
            for (int h = 0; h < 2; ++h) s.w[q][ni][h] = *(const vec8<T>*)(wp[ni] + k0 + h * 8);
          for (int mi = 0; mi < MT; ++mi)
            for (int h = 0; h < 2; ++h) s.x[q][mi][h] = *(const vec8<T>*)(xp[mi] + k0 + h * 8);
        } else {
          for (int h = 0; h < 2; ++h) {
            const int64_t left = (int64_t)a.k - (k0 + kl + h * 8);
            for (int ni = 0; ni < NT; ++ni) s.w[q][ni][h] = piece(wp[ni] + k0 + h * 8, left);
            for (int mi = 0; mi < MT; ++mi) s.x[q][mi][h] = piece(xp[mi] + k0 + h * 8, left);
          }
        }
      }
    };
    auto multiply = [&](const Step& s) __attribute__((always_inline)) {
      for (int q = 0; q < U; ++q)
        for (int h = 0; h < 2; ++h)
          for (int ni = 0; ni < NT; ++ni)
            for (int mi = 0; mi < MT; ++mi) acc[ni][mi] = mfma(s.w[q][ni][h], s.x[q][mi][h], acc[ni][mi]);
    };
    float low[OUTS];
    if (has && wave < lines) {
      Step s0, s1;
      fetch(s0, wave);
      uint32_t line = wave;
      for (;;) {
        line += U * WAVES;
        const bool more = line < lines;
        if (more) fetch(s1, line);
        multiply(s0);
        if (!more) break;
        line += U * WAVES;
        const bool again = line < lines;
        if (again) fetch(s0, line);
        multiply(s1);
        if (!again) break;
      }
    }
    for (int o = 0; o < OUTS; ++o) {
      const uint32_t at = threadIdx.x + o * THREADS;
      const int64_t row = m0 + at / BN;
      low[o] = LR && at < BM * BN && row < g.end && n0 + at % BN < a.n ? lowrank_at<T>(a, row, n0 + at % BN) : 0;
    }
    for (int ni = 0; ni < NT; ++ni)
      for (int mi = 0; mi < MT; ++mi)
        *(f32x4*)&red[(wave * BM + mi * 16 + lane % 16) * LD + ni * 16 + lane / 16 * 4] = acc[ni][mi];
    __syncthreads();
    for (int o = 0; o < OUTS; ++o) {
      const uint32_t at = threadIdx.x + o * THREADS, m = at / BN, n = n0 + at % BN;
      const int64_t i = m0 + m;
      if (at >= BM * BN || i >= g.end || n >= a.n) continue;
      float v = 0;
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

template <class T, int MT, int NT>
hipError_t run(const MatArgs& a, hipStream_t s) {
  constexpr uint32_t BM = 16 * MT, BN = 16 * NT;
  const uint64_t ntiles = th::ceil_div(a.n, BN);
  uint64_t mtiles = th::ceil_div(a.rows, BM), blocks;
  uint32_t shares = 1, bytes = WAVES * BM * (BN + 4) * 4;
  if (a.scan) {
    // workgroups of one group: as many as its slots can need, no more than fill the GPU
    shares = (uint32_t)min(mtiles, th::ceil_div(256, ntiles * a.E));
    blocks = ntiles * a.E * shares;
    bytes += (th::NARROW_SCAN_SLOTS + 1) * 4;
  } else {
    if (a.offsets) mtiles = a.rows / BM + (uint64_t)min((int64_t)a.E + 1, a.rows);
    blocks = mtiles * ntiles;
  }
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(THREADS), bytes, s, a, shares);
    return hipGetLastError();
  };
  if (a.u) return a.aligned ? go(narrow_kernel<T, MT, NT, true, true>) : go(narrow_kernel<T, MT, NT, false, true>);
  return a.aligned ? go(narrow_kernel<T, MT, NT, true, false>) : go(narrow_kernel<T, MT, NT, false, false>);
}

template <class T>
hipError_t typed(const MatArgs& a, hipStream_t s) {
  switch (th::narrow_tile(a.rows, a.n, a.offsets || a.scan ? a.E : 1)) {
    case th::NARROW_16x16: return run<T, 1, 1>(a, s);
    case th::NARROW_32x16: return run<T, 2, 1>(a, s);
    case th::NARROW_32x32: return run<T, 2, 2>(a, s);
    default: return run<T, 4, 2>(a, s);
  }
}

}  // namespace

hipError_t launch_narrow(MixType type, const MatArgs& a, hipStream_t s) {
  return type == MIX_BF16 ? typed<bf16_t>(a, s) : typed<f16_t>(a, s);
}

// Gradients of grouped weights and of low-rank factors: products whose
// contraction runs over a group's slots.
#include "wide_kernel.h"

using namespace mix;

namespace {

// Slots whose rows a workgroup of low_outer_kernel holds in LDS: 64 KiB of the
// wide operand and 16 to 64 KiB of ranks, or, above rank 64, 32 KiB and 64. Up
// to rank 16 that is 80 KiB in all, so that a CU holds two.
constexpr int low_batch(int mr) { return mr <= 4 ? 256 : 128; }

// ---------------------------------------------------------------- weight gradients
// The group that comes n-th by its number of slots, most first (of up to 256;
// further ones in their own order): the long contractions then start first and
// the short ones fill the CUs that the last of them leave.
__device__ uint32_t nth_longest(const int32_t* offsets, uint32_t E, int64_t slots, uint32_t n, uint32_t lane) {
  if (E > 256) return n;
  uint32_t size[4], rank[4] = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t g = c * 64 + lane;
    size[c] = 0;
    if (g < E) {
      const int64_t d = group_begin(offsets, g + 1, E, slots) - group_begin(offsets, g, E, slots);
      size[c] = d > 0 ? (uint32_t)d : 0;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    for (uint32_t l = 0; l < 64 && q * 64 + l < E; ++l) {
      const uint32_t other = __builtin_amdgcn_readlane(size[q], l), g = q * 64 + l;
#pragma unroll
      for (int c = 0; c < 4; ++c) rank[c] += other > size[c] || (other == size[c] && g < c * 64 + lane);
    }
  uint32_t found = n;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint64_t here = __ballot(c * 64 + lane < E && rank[c] == n);
    if (here) found = c * 64 + __ffsll((unsigned long long)here) - 1;
  }
  return found;
}

// B x B outputs of one group, WM x WN wavefronts: both operands are rows of
// slots, 64 slots a tile, read through the transposing LDS read. Two tiles in
// LDS or on their way, a tile's halves passing through registers as in the wide
// products (wide_kernel.h); the slots' numbers are loaded a tile ahead of them.
template <class T, int B, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) outer_kernel(OuterArgs a) {
  constexpr int WAVES = WM * WN, TM = B / WM, TN = B / WN, MI = TM / 16, NI = TN / 16;
  constexpr int JOBS = B / 8 / WAVES;                    // 1 KiB loads of an operand per wavefront and tile
  constexpr int CHUNKS = B / 8, PER = 64 / CHUNKS;       // 16-byte pieces of a row, rows of a load
  constexpr uint32_t TILE = B * 128, STAGE = 2 * TILE;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wm = wave / WN, wn = wave % WN;
  const uint32_t nt = (a.n + B - 1) / B, kt = (a.k + B - 1) / B;
  // every group's tiles in 8 rectangles, one for each XCD, whose L2 then serves each of its rows and columns once; groups
  // differ in their slots, so an XCD must not have a group to itself
  const uint32_t gn = nt >= kt ? 4 : 2, gk = 8 / gn, hn = (nt + gn - 1) / gn, hk = (kt + gk - 1) / gk;
  const uint32_t xcd = blockIdx.x % 8, at8 = blockIdx.x / 8, in = at8 % (hn * hk);
  const uint32_t n0 = (xcd % gn * hn + in % hn) * B, c0 = (xcd / gn * hk + in / hn) * B;
  if (in % hn + xcd % gn * hn >= nt || in / hn + xcd / gn * hk >= kt) return;
  const uint32_t e = nth_longest(a.offsets, a.E, a.slots, at8 / (hn * hk), lane);
  const int64_t begin = group_begin(a.offsets, e, a.E, a.slots), end = group_begin(a.offsets, e + 1, a.E, a.slots);
  const char* zero = (const char*)&mix_zero16;
  f32x4 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  const uint32_t tiles = begin < end ? (uint32_t)((end - begin + 63) / 64) : 0;
  if (tiles) {
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + wave * JOBS * 1024;
    uint32_t slot[JOBS];  // of this lane's rows of the tile that is loaded next, ~0 past the group
    const uint32_t row0 = wave * JOBS * PER + lane / CHUNKS;
    auto look = [&](uint32_t i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < JOBS; ++j) {
        const int64_t at = begin + (int64_t)i * 64 + row0 + j * PER;
        slot[j] = at < end ? (uint32_t)a.order[at] : ~0u;
      }
    };
    // the numbers have arrived here, before any load that would be waited for with them
    auto looked = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < JOBS; ++j) asm volatile("" ::"v"(slot[j]));
    };
    auto load = [&](int j, uint32_t stage) __attribute__((always_inline)) {
      const uint32_t s = slot[j % JOBS];
      const uint32_t c = ((lane % CHUNKS) ^ tr_swizzle<B>(row0 + j % JOBS * PER)) * 8;
      const void* p = zero;
      if (j < JOBS) {
        if (s < (uint64_t)a.slots && n0 + c < a.n) p = (const T*)a.dy + (int64_t)s * a.lddy + (n0 + c);
      } else {
        if (s < (uint64_t)a.slots && c0 + c < a.k) p = (const T*)a.x + (int64_t)(s / a.div) * a.ldx + (c0 + c);
      }
      load_lds16(p, lds0 + stage * STAGE + (j < JOBS ? 0 : TILE) + j % JOBS * 1024);
    };
    vec8<T> fa[2][MI], fb[2][NI];
    auto half = [&](int set, bool reads, uint32_t stage, int kk, bool loads, uint32_t to)
        __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (reads)
#pragma unroll
          for (int f = p * (MI + NI) / 8; f < (p + 1) * (MI + NI) / 8; ++f) {
            const char* at = lds + stage * STAGE;
            if (f < NI) fb[set ^ 1][f] = tr_fragment<T, B>(at + TILE, wn * TN + f * 16, kk * 32, lane);
            else fa[set ^ 1][f - NI] = tr_fragment<T, B>(at, wm * TM + (f - NI) * 16, kk * 32, lane);
          }
        if (loads)
#pragma unroll
          for (int j = p * JOBS / 4; j < (p + 1) * JOBS / 4; ++j) load(j, to);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = p * MI * NI / 8; q < (p + 1) * MI * NI / 8; ++q)
          acc[q / MI][q % MI] = mfma(fb[set][q / MI], fa[set][q % MI], acc[q / MI][q % MI]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    look(0);
    looked();
#pragma unroll
    for (int j = 0; j < 2 * JOBS; ++j) load(j, 0);
    look(1);  // past the end: zeros
    looked();
#pragma unroll
    for (int j = 0; j < 2 * JOBS; ++j) load(j, 1);
    look(2);
    arrived_barrier();
#pragma unroll
    for (int f = 0; f < NI; ++f) fb[0][f] = tr_fragment<T, B>(lds + TILE, wn * TN + f * 16, 0, lane);
#pragma unroll
    for (int f = 0; f < MI; ++f) fa[0][f] = tr_fragment<T, B>(lds, wm * TM + f * 16, 0, lane);
    uint32_t stage = 0;
    for (uint32_t i = 0; i + 2 < tiles; ++i, stage ^= 1) {
      half(0, true, stage, 1, false, 0);
      arrived_barrier();
      looked();
      half(1, true, stage ^ 1, 0, true, stage);
      look(i + 3);
    }
    for (uint32_t i = tiles > 2 ? tiles - 2 : 0; i < tiles; ++i, stage ^= 1) {
      half(0, true, stage, 1, false, 0);
      arrived_barrier();
      half(1, i + 1 < tiles, stage ^ 1, 0, false, 0);
    }
  }
  __syncthreads();
  // rows of the output are dy's columns
  const Out out{(T*)a.out + ((int64_t)e * a.n + n0) * a.k, a.k, a.k, nullptr};
  put<T, T, TM, TN>(out, acc, lds + wave * (TM * TN * 2), nullptr, wm * TM, a.n - n0, c0 + wn * TN, lane);
}

// The same for rows that do not start on 16 bytes or widths that are no
// multiples of 8: 128 x 128 outputs, tiles through registers.
template <class T>
__global__ void __launch_bounds__(256) unaligned_outer_kernel(OuterArgs a) {
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
  int64_t slot[JOBS];  // of the step that is fetched next; -1 past the group
  auto look = [&](int64_t s0) {
    for (int j = 0; j < JOBS; ++j) {
      const int64_t i = s0 + row[j];
      slot[j] = i < end ? min((int64_t)(uint32_t)a.order[i], a.slots - 1) : -1;
    }
  };
  vec8<T> rn[JOBS], rk[JOBS];
  auto fetch = [&]() {
    for (int j = 0; j < JOBS; ++j) {
      const bool inn = slot[j] >= 0 && cn[j] < a.n, ink = slot[j] >= 0 && ck[j] < a.k;
      const T* pn = inn ? (const T*)a.dy + slot[j] * a.lddy + cn[j] : (const T*)zero;
      const T* pk = ink ? (const T*)a.x + slot[j] / a.div * a.ldx + ck[j] : (const T*)zero;
      rn[j] = load8<T>(pn, inn ? a.n - cn[j] : 0);
      rk[j] = load8<T>(pk, ink ? a.k - ck[j] : 0);
    }
  };
  auto commit = [&](uint32_t stage) {
    for (int j = 0; j < JOBS; ++j) {
      char* p = lds + stage * STAGE + (wave * JOBS + j) * 1024 + lane * 16;
      *(vec8<T>*)p = rn[j];
      *(vec8<T>*)(p + TILE) = rk[j];
    }
  };
  if (begin < end) {
    look(begin);
    fetch();
    commit(0);
    look(begin + 64);
  }
  uint32_t stage = 0;
  for (int64_t s0 = begin; s0 < end; s0 += 64, stage ^= 1) {
    __syncthreads();
    const bool more = s0 + 64 < end;
    if (more) {
      fetch();
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
__device__ inline void gate_grad(const GateGradArgs& a, uint32_t block) {
  const int64_t s = (int64_t)block * 256 + threadIdx.x;
  if (s >= a.slots) return;
  const uint32_t e = (uint32_t)a.ids[s];
  float d = 0;
  if (e < a.E) {
    for (uint32_t i = 0; i < a.r; ++i) d += a.u[s * a.ru + i] * a.v[s * a.ru + i];
    if (a.scale) d *= a.scale[e];
  }
  a.out[s] = d;
}

// Partial sums over a span of one adapter's slots: 16 MR rows of the low-rank
// factor (float, scaled, as a bf16 pair) by 128 columns of the wide operand,
// BATCH slots at a time. Few flops and short contractions: what bounds it is the
// chain slot -> row -> product, so a batch's loads all go out together, and the
// CU's other workgroups run meanwhile. Both gradients, and the gate's, share a launch: 8192 slots
// of 8 rank-16 adapters by 1536 columns each way take 17 us (50 MB of gathered
// rows, 10 us at a copy's rate; 26 with one workgroup a CU) and 6 for adding the
// partial sums.
//
// Where a sum is no finite number, the span is taken again with coefficients
// that round to infinity as bf16's largest and the rest, and, if infinities or
// NaN are left, once more by the high parts alone (mfma_high): a span has one
// adapter, so its other sums and other adapters' do not change.
//
// One pass over a span: its 16 MR x 128 partial sums, or, after the first, those
// of them that are no finite numbers yet. Whether there are any of those.
template <class T, int MR, bool ALIGNED, int PASS>
__device__ inline bool low_span(const LowOuterArgs& a, const GroupTile& g, uint32_t span, uint32_t c0, char* lds, uint32_t lane,
                                uint32_t wave) {
  constexpr int BATCH = low_batch(MR), BN = 128, R = 16 * MR;
  constexpr int JOBS = BATCH / 16;  // 1 KiB loads (4 slots) per wavefront and batch
  char *wide = lds, *low[2] = {wide + BATCH * BN * 2, wide + BATCH * BN * 2 + BATCH * R * 2};
  uint32_t* slot = (uint32_t*)low[1];  // until the low-rank rows come there
  const char* zero = (const char*)&mix_zero16;
  f32x4 acc[MR][2];
#pragma unroll
  for (int i = 0; i < MR; ++i) acc[i][0] = acc[i][1] = f32x4{0, 0, 0, 0};
  const float se = a.scale ? a.scale[g.group] : 1.0f;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + wave * JOBS * 1024;
  for (int64_t s0 = g.begin; s0 < g.end; s0 += BATCH) {
    // thread i < BATCH: slot i of the batch, its coefficient and its row of the low-rank factor
    uint32_t s = ~0u;
    float c = 0;
    if (threadIdx.x < BATCH && s0 + threadIdx.x < g.end) {
      s = (uint32_t)a.order[s0 + threadIdx.x];
      if (s >= (uint64_t)a.slots) s = ~0u;
      else c = (a.gate ? a.gate[s] : 1.0f) * se;
    }
    __syncthreads();
    if (threadIdx.x < BATCH) slot[threadIdx.x] = s;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < JOBS; ++j) {
      const uint32_t row = (wave * JOBS + j) * 4 + lane / 16, sr = slot[row];
      const uint32_t col = c0 + ((lane % 16) ^ tr_swizzle<BN>(row)) * 8;
      const bool in = sr != ~0u && col < a.cols;
      const T* p = in ? (const T*)a.wide + (int64_t)(sr / a.div) * a.ldwide + col : (const T*)zero;
      if constexpr (ALIGNED) load_lds16(p, lds0 + j * 1024);
      else *(vec8<T>*)(wide + (wave * JOBS + j) * 1024 + lane * 16) = load8<T>(p, in ? (int64_t)a.cols - col : 0);
    }
    __syncthreads();
    if (threadIdx.x < BATCH) {
      const float* u = a.low + (int64_t)(s == ~0u ? 0 : s) * a.ru;
      const uint32_t limit = s == ~0u ? 0 : a.r;
#pragma unroll
      for (int q = 0; q < R; q += 8) {
        f32x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (q + 8 <= (int)limit) {
          const f32x4 u0 = *(const f32x4*)(u + q), u1 = *(const f32x4*)(u + q + 4);
          for (int x = 0; x < 8; ++x) v[x] = c * (x < 4 ? u0 : u1)[x % 4];
        } else {
          for (int x = 0; x < 8; ++x)
            if (q + x < (int)limit) v[x] = c * u[q + x];
        }
        bf16x8 hi, lo;
        if constexpr (PASS == 0) split8(v, hi, lo);
        else split8_any(v, hi, lo);
        const uint32_t at = threadIdx.x * (R * 2) + ((q / 8) ^ tr_swizzle<R>(threadIdx.x)) * 16;
        *(bf16x8*)(low[0] + at) = hi;
        *(bf16x8*)(low[1] + at) = lo;
      }
    }
    arrived_barrier();
    const uint32_t steps = min((uint32_t)BATCH, (uint32_t)(g.end - s0));
    for (uint32_t k = 0; k < steps; k += 32) {
      decltype(widen(vec8<T>())) wf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) wf[i] = widen(tr_fragment<T, BN>(wide, wave * 32 + i * 16, k, lane));
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const bf16x8 hi = tr_fragment<bf16_t, R>(low[0], m * 16, k, lane);
        const bf16x8 lo = tr_fragment<bf16_t, R>(low[1], m * 16, k, lane);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if constexpr (PASS < 2) acc[m][i] = mfma_split(wf[i], hi, lo, acc[m][i]);
          else acc[m][i] = mfma_high(wf[i], hi, acc[m][i]);
      }
    }
  }
  // a lane: row lane % 16 of the low-rank factor, 4 neighbouring columns
  bool odd = false;
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t q = m * 16 + lane % 16, c = c0 + wave * 32 + i * 16 + lane / 16 * 4;
      if (q >= a.r) continue;
      float* o = a.partial + ((int64_t)span * a.r + q) * a.cols + c;
      if (PASS == 0 && c + 4 <= a.cols && a.cols % 4 == 0) {
        *(f32x4*)o = acc[m][i];
      } else {
        for (int x = 0; x < 4; ++x)
          if (c + x < a.cols && (PASS == 0 || !isfinite(o[x]))) o[x] = acc[m][i][x];
      }
      for (int x = 0; x < 4; ++x) odd |= !isfinite(acc[m][i][x]);
    }
  // (__syncthreads_or would take LDS of its own, and the CU's second workgroup with it)
  uint32_t* flag = (uint32_t*)wide;
  odd = __ballot(odd);
  __syncthreads();
  if (lane == 0) flag[wave] = odd;
  __syncthreads();
  return flag[0] | flag[1] | flag[2] | flag[3];
}

template <class T, int MR, bool ALIGNED>
__global__ void __launch_bounds__(256) low_outer_kernel(LowOuterPair pair) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x >= pair.gate_from) return gate_grad(pair.gate, blockIdx.x - pair.gate_from);
  const bool second = blockIdx.x >= pair.blocks;
  const LowOuterArgs& a = pair.p[second];
  const uint32_t block = blockIdx.x - (second ? pair.blocks : 0), ctiles = (a.cols + 127) / 128;
  const uint32_t c0 = block % ctiles * 128, span = block / ctiles;
  const GroupTile g = find_group_tile(a.offsets, a.E, a.E, a.slots, a.span, span, lane);
  if (g.begin >= g.end) return;
  if (low_span<T, MR, ALIGNED, 0>(a, g, span, c0, lds, lane, wave) &&
      low_span<T, MR, ALIGNED, 1>(a, g, span, c0, lds, lane, wave))
    low_span<T, MR, ALIGNED, 2>(a, g, span, c0, lds, lane, wave);
}

// Adds an adapter's partial sums, in slot order. A thread: 4 columns of a rank,
// or, where the output is transposed, a column of 8 ranks, so that it writes
// 8 or 16 bytes; loads of several partial sums are under way at once.
template <class T>
__global__ void __launch_bounds__(256) low_sum_kernel(LowOuterPair pair) {
  const LowOuterArgs& a = pair.p[blockIdx.z];
  const uint32_t e = blockIdx.y, lane = threadIdx.x & 63;
  if (!a.out) return;
  const uint32_t first = count_group_tiles(a.offsets, a.E, e, a.slots, a.span, lane);
  const int64_t c = group_begin(a.offsets, e + 1, a.E, a.slots) - group_begin(a.offsets, e, a.E, a.slots);
  const uint32_t n = c > 0 ? (uint32_t)((c + a.span - 1) / a.span) : 0;
  const uint64_t size = (uint64_t)a.r * a.cols;
  const float* partial = a.partial + first * size;
  T* out = (T*)a.out + e * size;
  const uint32_t across = a.transposed ? a.cols : (a.cols + 3) / 4, down = a.transposed ? (a.r + 7) / 8 : a.r;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)across * down;
       i += (uint64_t)gridDim.x * 256) {
    const uint32_t x = (uint32_t)(i % across), y = (uint32_t)(i / across);
    if (a.transposed) {
      const uint32_t q0 = y * 8, many = min(8u, a.r - q0);
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      const float* from = partial + (uint64_t)q0 * a.cols + x;
      if (many == 8) {
#pragma unroll 4
        for (uint32_t p = 0; p < n; ++p)
#pragma unroll
          for (uint32_t q = 0; q < 8; ++q) v[q] += from[p * size + (uint64_t)q * a.cols];
      } else {
        for (uint32_t p = 0; p < n; ++p)
          for (uint32_t q = 0; q < many; ++q) v[q] += from[p * size + (uint64_t)q * a.cols];
      }
      T* o = out + (uint64_t)x * a.r + q0;
      if (many == 8 && a.r % 8 == 0) {
        vec8<T> w;
        for (int q = 0; q < 8; ++q) w[q] = (T)v[q];
        *(vec8<T>*)o = w;
      } else {
        for (uint32_t q = 0; q < many; ++q) o[q] = (T)v[q];
      }
    } else if (a.cols % 4 == 0) {
      f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
      for (uint32_t p = 0; p < n; ++p) v += *(const f32x4*)(partial + p * size + (uint64_t)y * a.cols + x * 4);
      const T w[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
      *(uint64_t*)(out + (uint64_t)y * a.cols + x * 4) = __builtin_bit_cast(uint64_t, w);
    } else {
      for (uint32_t q = x * 4; q < min(x * 4 + 4, a.cols); ++q) {
        float v = 0;
        for (uint32_t p = 0; p < n; ++p) v += partial[p * size + (uint64_t)y * a.cols + q];
        out[(uint64_t)y * a.cols + q] = (T)v;
      }
    }
  }
}

template <class T, int MR>
hipError_t run_low(const LowOuterPair& pair, uint64_t blocks, hipStream_t s) {
  constexpr uint32_t bytes = low_batch(MR) * (128 * 2 + 2 * 16 * MR * 2);
  return pair.p[0].aligned && pair.p[1].aligned ? launch<low_outer_kernel<T, MR, true>, bytes>(blocks, 256, bytes, s, pair)
                                                : launch<low_outer_kernel<T, MR, false>, bytes>(blocks, 256, bytes, s, pair);
}

template <class T>
hipError_t low_outer_typed(LowOuterPair pair, hipStream_t s) {
  uint64_t blocks = 0;
  uint32_t rows = 0;
  for (int i = 0; i < 2; ++i) {
    const LowOuterArgs& a = pair.p[i];
    if (i == 1) pair.blocks = (uint32_t)blocks;
    if (!a.out) continue;
    blocks += th::ceil_div(a.cols, 128) * th::lowrank_spans(a.slots, a.E, a.span);
    const uint64_t threads = a.transposed ? a.cols * th::ceil_div(a.r, 8) : a.r * th::ceil_div(a.cols, 4);
    rows = max(rows, (uint32_t)min(th::ceil_div(threads, 256), (uint64_t)1024));
  }
  const LowOuterArgs& a = pair.p[pair.p[0].out ? 0 : 1];
  pair.gate_from = (uint32_t)blocks;
  if (pair.gate.out) blocks += th::ceil_div(pair.gate.slots, 256);
  if (blocks) {
    const hipError_t e = a.r <= 16   ? run_low<T, 1>(pair, blocks, s)
                         : a.r <= 32 ? run_low<T, 2>(pair, blocks, s)
                         : a.r <= 64 ? run_low<T, 4>(pair, blocks, s)
                                     : run_low<T, 8>(pair, blocks, s);
    if (e != hipSuccess) return e;
  }
  low_sum_kernel<T><<<dim3(rows, a.E, 2), 256, 0, s>>>(pair);
  return hipGetLastError();
}

// 64 x 64 pieces of the matrices of up to two stacks.
__global__ void __launch_bounds__(256) transpose_kernel(TransposePair pair) {
  __shared__ uint16_t tile[64][66];
  const bool second = blockIdx.x >= pair.blocks;
  const TransposeArgs& a = pair.p[second];
  const uint32_t block = blockIdx.x - (second ? pair.blocks : 0);
  const uint32_t rt = (a.rows + 63) / 64, ct = (a.cols + 63) / 64;
  const uint32_t r0 = block % rt * 64, c0 = block / rt % ct * 64, e = block / rt / ct;
  const uint32_t h = min(64u, a.rows - r0), w = min(64u, a.cols - c0);
  for (uint32_t i = threadIdx.x; i < h * w; i += 256)
    tile[i / w][i % w] = ((const uint16_t*)a.in)[e * a.lde + (int64_t)(r0 + i / w) * a.ld + c0 + i % w];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < h * w; i += 256)
    ((uint16_t*)a.out)[((int64_t)e * a.cols + c0 + i / h) * a.out_ld + r0 + i % h] = tile[i % h][i / h];
  const uint32_t tail = r0 + 64 >= a.rows ? a.out_ld - a.rows : 0;
  for (uint32_t i = threadIdx.x; i < tail * w; i += 256)
    ((uint16_t*)a.out)[((int64_t)e * a.cols + c0 + i / tail) * a.out_ld + a.rows + i % tail] = 0;
}

// 8 values a thread at a time.
__global__ void __launch_bounds__(256) pad_kernel(PadSet set) {
  const uint32_t which = (blockIdx.x >= set.blocks[0]) + (blockIdx.x >= set.blocks[1]);
  const PadArgs& a = set.p[which];
  const uint32_t first = which ? set.blocks[which - 1] : 0, many = (which < 2 ? set.blocks[which] : gridDim.x) - first;
  const uint32_t chunks = (a.cols + 7) / 8;
  for (uint64_t i = (uint64_t)(blockIdx.x - first) * 256 + threadIdx.x;; i += (uint64_t)many * 256) {
    const uint64_t row = i / chunks;
    if (row >= (uint64_t)a.rows * a.E) return;
    const uint32_t c = (uint32_t)(i % chunks) * 8;
    const bf16_t* p = (const bf16_t*)a.in + (int64_t)(row / a.rows) * a.lde + (int64_t)(row % a.rows) * a.ld + c;
    ((bf16x8*)a.out)[i] = load8<bf16_t>(p, (int64_t)a.cols - c);
  }
}

// A thread: 8 columns of a token, or 1 where rows are no multiple of 8.
template <class T, int W>
__global__ void __launch_bounds__(256) sum_choices_kernel(const float* in, T* out, int64_t tokens, uint32_t k,
                                                          uint32_t n) {
  const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * W;
  if (c >= n) return;
  for (int64_t t = blockIdx.y; t < tokens; t += gridDim.y) {
    const float* p = in + t * k * n + c;
    float v[W] = {};
#pragma unroll 2
    for (uint32_t j = 0; j < k; ++j) {
      float x[W];
      __builtin_memcpy(x, __builtin_assume_aligned(p + (int64_t)j * n, W == 8 ? 16 : 4), sizeof(x));
      for (int q = 0; q < W; ++q) v[q] += x[q];
    }
    T o[W];
    for (int q = 0; q < W; ++q) o[q] = (T)v[q];
    __builtin_memcpy(__builtin_assume_aligned(out + t * n + c, W == 8 ? 16 : 2), o, sizeof(o));
  }
}

__global__ void __launch_bounds__(256) gate_grad_kernel(GateGradArgs a) { gate_grad(a, blockIdx.x); }

}  // namespace

template <class T>
static hipError_t outer_typed(const OuterArgs& a, hipStream_t s) {
  if (!a.aligned) {
    const uint64_t blocks = th::ceil_div(a.n, 128) * th::ceil_div(a.k, 128) * a.E;
    return launch<unaligned_outer_kernel<T>>(blocks, 256, 2 * 2 * 64 * 128 * 2, s, a);
  }
  constexpr uint32_t B = 128;
  const uint64_t nt = th::ceil_div(a.n, B), kt = th::ceil_div(a.k, B), gn = nt >= kt ? 4 : 2, gk = 8 / gn;
  const uint64_t blocks = 8 * th::ceil_div(nt, gn) * th::ceil_div(kt, gk) * a.E;
  return launch<outer_kernel<T, B, 2, 4>>(blocks, 512, 2 * 2 * B * 128, s, a);
}
hipError_t launch_outer(MixType type, const OuterArgs& a, hipStream_t s) {
  return type == MIX_BF16 ? outer_typed<bf16_t>(a, s) : outer_typed<f16_t>(a, s);
}

hipError_t launch_low_outer(MixType type, const LowOuterPair& pair, hipStream_t s) {
  return type == MIX_BF16 ? low_outer_typed<bf16_t>(pair, s) : low_outer_typed<f16_t>(pair, s);
}

hipError_t launch_transpose(TransposePair pair, hipStream_t s) {
  uint64_t blocks = 0;
  for (int i = 0; i < 2; ++i) {
    const TransposeArgs& a = pair.p[i];
    if (i == 1) pair.blocks = (uint32_t)blocks;
    if (a.out) blocks += th::ceil_div(a.rows, 64) * th::ceil_div(a.cols, 64) * a.E;
  }
  return blocks ? launch<transpose_kernel>(blocks, 256, 0, s, pair) : hipSuccess;
}

hipError_t launch_pad(PadSet set, hipStream_t s) {
  uint32_t blocks = 0;
  for (int i = 0; i < 3; ++i) {
    if (i) set.blocks[i - 1] = blocks;
    if (set.p[i].out) blocks += th::pad_blocks(set.p[i].rows, set.p[i].E, set.p[i].cols);
  }
  return blocks ? launch<pad_kernel>(blocks, 256, 0, s, set) : hipSuccess;
}

hipError_t launch_sum_choices(MixType type, const float* in, void* out, int64_t tokens, uint32_t k, uint32_t n,
                              hipStream_t s) {
  if (!tokens) return hipSuccess;
  const bool by8 = n % 8 == 0 && ((uintptr_t)out & 15) == 0;
  const dim3 grid((uint32_t)th::ceil_div(n, by8 ? 2048 : 256), (uint32_t)min(tokens, (int64_t)16384));
  if (type == MIX_BF16 && by8) sum_choices_kernel<bf16_t, 8><<<grid, 256, 0, s>>>(in, (bf16_t*)out, tokens, k, n);
  else if (type == MIX_BF16) sum_choices_kernel<bf16_t, 1><<<grid, 256, 0, s>>>(in, (bf16_t*)out, tokens, k, n);
  else if (by8) sum_choices_kernel<f16_t, 8><<<grid, 256, 0, s>>>(in, (f16_t*)out, tokens, k, n);
  else sum_choices_kernel<f16_t, 1><<<grid, 256, 0, s>>>(in, (f16_t*)out, tokens, k, n);
  return hipGetLastError();
}

hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t s) {
  if (!a.slots) return hipSuccess;
  return launch<gate_grad_kernel>(th::ceil_div(a.slots, 256), 256, 0, s, a);
}

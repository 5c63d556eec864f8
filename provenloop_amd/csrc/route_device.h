// What the gates share: reductions over a token's lanes, and the places of its
// slots (see route.hip).
#pragma once
#include "mixture.h"

namespace mix {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t group_lds(uint32_t E, bool chunks = false) { return ((chunks ? 2 : 1) * WAVES + 1) * (E + 1) * 4; }
constexpr uint32_t MOST = group_lds(th::MIX_MAX_EXPERTS), MOST_CHUNKS = group_lds(th::MIX_MAX_EXPERTS, true);

// The same value from a lane on the other side, of pairs, quads, 8, 16, 32 or
// 64 lanes whose halves each agree on theirs.
template <int D>
__device__ inline uint32_t across(uint32_t v) {
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
  else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  else if constexpr (D == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);  // row_half_mirror
  else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);  // row_mirror
  else return __shfl_xor(v, D);
}
template <int D>
__device__ inline uint64_t across(uint64_t v) {
  return (uint64_t)across<D>((uint32_t)(v >> 32)) << 32 | across<D>((uint32_t)v);
}
template <int G, class C, int D = 1>
__device__ inline C group_max(C v) {
  if constexpr (D < G) {
    const C o = across<D>(v);
    return group_max<G, C, 2 * D>(o > v ? o : v);
  } else {
    return v;
  }
}
template <int G, int D = 1>
__device__ inline float group_sum(float v) {
  if constexpr (D < G) return group_sum<G, 2 * D>(v + __uint_as_float(across<D>(__float_as_uint(v))));
  else return v;
}

template <class T>
__device__ inline bool allowed_at(const RouteArgs& a, int64_t t, uint32_t e, float& l) {
  l = to_float(((const T*)a.logits)[t * a.ld + e]);
  const bool ok = !(l == -INFINITY) && (!a.mask || a.mask[t * a.mask_ld + e]);
  return ok;
}

// Exclusive prefix of n words in LDS by the first wavefront.
__device__ inline void prefix_words(uint32_t* v, uint32_t n) {
  if (threadIdx.x < 64) {
    uint32_t run = 0;
    for (uint32_t at = 0; at < n; at += 64) {
      const uint32_t i = at + threadIdx.x;
      const uint32_t own = i < n ? v[i] : 0;
      uint32_t sum = own;
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(sum, d);
        if ((int)threadIdx.x >= d) sum += up;
      }
      if (i < n) v[i] = run + sum - own;
      run += __shfl(sum, 63);
    }
  }
}

// Positions of the slots [s0, s1) of one workgroup. `base` (LDS, E + 1 words)
// holds where the workgroup's first slot of each expert goes; `counts` (LDS,
// WAVES x (E + 1)). A wavefront ranks its 64 slots by matching the expert's
// bits across its lanes; the wavefronts' counts are summed per expert.
__device__ inline void place_slots(const int32_t* experts, int64_t s0, int64_t s1, uint32_t E, int32_t* order, uint32_t* base,
                            uint32_t* counts) {
  const uint32_t keys = E + 1, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int bits = 32 - __clz(E);
  for (int64_t at = s0; at < s1; at += THREADS) {
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += THREADS) counts[i] = 0;
    __syncthreads();
    const int64_t s = at + threadIdx.x;
    const bool in = s < s1;
    uint32_t key = E;
    if (in) {
      const uint32_t e = (uint32_t)experts[s];
      key = e < E ? e : E;
    }
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((key >> b) & 1);
      same &= (key >> b) & 1 ? set : ~set;
    }
    const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
    if (in && rank == 0) counts[wave * keys + key] = __popcll(same);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < keys; i += THREADS) {
      uint32_t run = base[i];
      for (int w = 0; w < WAVES; ++w) {
        const uint32_t c = counts[w * keys + i];
        counts[w * keys + i] = run;
        run += c;
      }
      base[i] = run;
    }
    __syncthreads();
    if (in) order[counts[wave * keys + key] + rank] = (int32_t)s;
    __syncthreads();
  }
}

// The end of a gate's chunk, whose chosen experts `base` has counted: the counts
// for the launch that places the slots, or, of a single chunk, the slots' places.
__device__ inline void end_chunk(const RouteArgs& a, uint32_t* base, uint32_t* counts) {
  __threadfence_block();
  __syncthreads();
  if (gridDim.x > 1) {
    for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.hist[(size_t)blockIdx.x * (a.E + 1) + i] = base[i];
    return;
  }
  prefix_words(base, a.E + 1);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.offsets[i] = (int32_t)base[i];
  __syncthreads();
  place_slots(a.experts, 0, a.T * a.k, a.E, a.order, base, counts);
}

}  // namespace mix

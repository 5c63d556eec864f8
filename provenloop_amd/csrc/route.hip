// Softmax gate with top-k and the grouping of (token, choice) slots by expert.
//
// Gate: of the experts a token may use (its mask, and a logit above -inf) the
// k largest logits are chosen, ties to the lowest index, and
//   w_j = exp(l_j - max l) / Z,  Z over the chosen or over all allowed experts.
// Sums are in float; the logits decide the choice before any rounding.
//
// Grouping: a stable counting sort of the slots s = t k + j by expert, slots
// without an expert last. Counts and positions are integers, so the result
// does not depend on the order in which workgroups run.
//
// Both read their input once and write 12 bytes a slot; what bounds them is
// the latency of the chain of dependent steps, at small sizes the launch.
// Candidates are single numbers in a lane's registers, sorted once, and lanes
// compare by DPP: 65536 tokens over 64 experts, 8 chosen, take 12.8 us for the
// gate and 10 us for the slots' places. The gate moves 19 MB, 4 us at a copy's
// rate; about 450 instructions a token's lane are some 6 us, and the rest is loads
// that a workgroup's rounds of tokens wait for one after the other.
#include "mixture.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t group_lds(uint32_t E, bool chunks = false) { return ((chunks ? 2 : 1) * WAVES + 1) * (E + 1) * 4; }
constexpr uint32_t MOST = group_lds(th::MIX_MAX_EXPERTS), MOST_CHUNKS = group_lds(th::MIX_MAX_EXPERTS, true);

// A logit as a whole number that orders candidates: its bits made to rise with
// its value (NaN above +inf, as a comparison sort of the framework's users puts
// it; -0 with +0), over the expert's number from the top, so that of equal
// logits the lowest expert is the largest. 0 is kept for "not allowed".
template <class T>
struct Ranked {  // bf16 and f16: 16 bits and 16 bits
  using type = uint32_t;
  static __device__ inline uint32_t of(T v, uint32_t e) {
    uint16_t b = __builtin_bit_cast(uint16_t, v);
    b = b == 0x8000 ? 0 : b;
    const uint32_t key = v != v ? 0xffffu : b & 0x8000 ? 0xffffu & ~b : b | 0x8000u;
    return key << 16 | (0xffffu - e);
  }
  static __device__ inline uint32_t expert(uint32_t c) { return 0xffffu - (c & 0xffffu); }
  static __device__ inline float value(uint32_t c) {
    const uint32_t key = c >> 16;
    const uint16_t b = (uint16_t)(key & 0x8000 ? key ^ 0x8000 : ~key);
    return key == 0xffffu ? NAN : (float)__builtin_bit_cast(T, b);
  }
};
template <>
struct Ranked<float> {
  using type = uint64_t;
  static __device__ inline uint64_t of(float v, uint32_t e) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    const uint32_t key = v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)key << 32 | (0xffffffffu - e);
  }
  static __device__ inline uint32_t expert(uint64_t c) { return 0xffffffffu - (uint32_t)c; }
  static __device__ inline float value(uint64_t c) {
    const uint32_t key = (uint32_t)(c >> 32);
    return key == 0xffffffffu ? NAN : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
  }
};

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
__device__ void prefix_words(uint32_t* v, uint32_t n) {
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
__device__ void place_slots(const int32_t* experts, int64_t s0, int64_t s1, uint32_t E, int32_t* order, uint32_t* base,
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

// base = where this chunk's slots start, per expert, from every chunk's counts
// hist[chunk][key]; offsets written by chunk 0. A wavefront adds up every 16th
// chunk, 64 keys at a time; sums: LDS, 2 WAVES (E + 1) words.
__device__ void chunk_bases(const uint32_t* hist, uint32_t E, uint32_t chunks, uint32_t* base, uint32_t* sums,
                            int32_t* offsets) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, keys = E + 1;
  for (uint32_t key = lane; key < keys; key += 64) {
    uint32_t before = 0, all = 0;
#pragma unroll 8
    for (uint32_t c = wave; c < chunks; c += WAVES) {
      const uint32_t n = hist[(size_t)c * keys + key];
      all += n;
      before += c < blockIdx.x ? n : 0;
    }
    sums[wave * keys + key] = before;
    sums[(WAVES + wave) * keys + key] = all;
  }
  __syncthreads();
  for (uint32_t key = threadIdx.x; key < keys; key += THREADS) {
    uint32_t before = 0, all = 0;
    for (int w = 0; w < WAVES; ++w) {
      before += sums[w * keys + key];
      all += sums[(WAVES + w) * keys + key];
    }
    base[key] = before;
    sums[key] = all;
  }
  __syncthreads();
  prefix_words(sums, keys);
  __syncthreads();
  for (uint32_t key = threadIdx.x; key < keys; key += THREADS) {
    base[key] += sums[key];
    if (blockIdx.x == 0 && key < keys) offsets[key] = (int32_t)sums[key];
  }
  __syncthreads();
}

// One workgroup's tokens [t0, t1): a group of G lanes per token, 8 experts a
// lane in falling order in its registers, and k rounds: the largest of the
// lanes' first candidates is chosen and its lane moves on. Lane j of the group
// keeps choice j. Counts the chosen experts in `base`.
template <class T, int G>
__device__ void choose(const RouteArgs& a, int64_t t0, int64_t t1, uint32_t* base) {
  using R = Ranked<T>;
  using C = typename R::type;
  const uint32_t g = threadIdx.x % G;
  const bool whole = g * 8 + 8 <= a.E && a.vector;
  for (int64_t at = t0; at < t1; at += THREADS / G) {
    const int64_t t = at + threadIdx.x / G;
    if (t >= t1) continue;  // whole groups of G lanes leave together
    const T* row = (const T*)a.logits + t * a.ld + g * 8;
    const uint8_t* mask = a.mask ? a.mask + t * a.mask_ld + g * 8 : nullptr;
    T l[8];
    uint64_t allowed = ~0ull;  // a byte per expert
    if (whole) {
      __builtin_memcpy(l, __builtin_assume_aligned(row, 16), sizeof(l));
      if (mask) __builtin_memcpy(&allowed, __builtin_assume_aligned(mask, 8), 8);
    } else {
      for (uint32_t i = 0; i < 8; ++i) {
        const bool in = g * 8 + i < a.E;
        l[i] = in ? row[i] : (T)0.0f;
        if (!in || (mask && !mask[i])) allowed &= ~(0xffull << (8 * i));
      }
    }
    C c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = (allowed >> (8 * i) & 0xff) && !((float)l[i] == -INFINITY) ? R::of(l[i], g * 8 + i) : 0;
    // Batcher's odd-even merge of 8: 19 exchanges
    auto order = [&](int i, int j) __attribute__((always_inline)) {
      const C hi = c[i] > c[j] ? c[i] : c[j], lo = c[i] > c[j] ? c[j] : c[i];
      c[i] = hi;
      c[j] = lo;
    };
    order(0, 1), order(2, 3), order(4, 5), order(6, 7), order(0, 2), order(1, 3), order(4, 6), order(5, 7);
    order(1, 2), order(5, 6), order(0, 4), order(1, 5), order(2, 6), order(3, 7), order(2, 4), order(3, 5);
    order(1, 2), order(3, 4), order(5, 6);
    const C first = group_max<G>(c[0]);
    const float big = first ? R::value(first) : -INFINITY;
    float z = 0;
    if (!a.normalize) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c[i]) z += expf(R::value(c[i]) - big);
      z = group_sum<G>(z);
    }
    constexpr int KEEP = G >= 32 ? 1 : G >= 4 ? 32 / G : 8;  // choices that one lane can have to keep
    float p[KEEP];
    int32_t e[KEEP];
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      p[r] = 0;
      e[r] = -1;
      if (r * G < (int)a.k) {
        for (uint32_t j = 0; j < G && r * G + j < a.k; ++j) {
          const C best = group_max<G>(c[0]);
          if (c[0] == best) {
#pragma unroll
            for (int i = 0; i < 7; ++i) c[i] = c[i + 1];
            c[7] = 0;
          }
          if (g == j && best) {
            e[r] = (int32_t)R::expert(best);
            p[r] = expf(R::value(best) - big);
          }
        }
      }
    }
    if (a.normalize) {
#pragma unroll
      for (int r = 0; r < KEEP; ++r) z += p[r];
      z = group_sum<G>(z);
    }
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      const uint32_t j = r * G + g;
      if (j < a.k) {
        a.experts[t * a.k + j] = e[r];
        a.weights[t * a.k + j] = e[r] < 0 ? 0.0f : p[r] / z;
        atomicAdd(&base[e[r] < 0 ? a.E : e[r]], 1u);
      }
    }
  }
}

// Chunks of tokens: gate and counts; a single chunk also places its slots.
template <class T, int G>
__global__ void __launch_bounds__(THREADS) route_kernel(RouteArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t *base = lds, *counts = lds + a.E + 1;
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) base[i] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * a.chunk, t1 = min(t0 + (int64_t)a.chunk, a.T);
  choose<T, G>(a, t0, t1, base);
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

// Counts of one chunk of given slots; a single chunk also places them.
__global__ void __launch_bounds__(THREADS) count_kernel(RouteArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t *base = lds, *counts = lds + a.E + 1;
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) base[i] = 0;
  __syncthreads();
  const int64_t s0 = (int64_t)blockIdx.x * a.chunk * a.k, s1 = min(s0 + (int64_t)a.chunk * a.k, a.T * a.k);
  for (int64_t s = s0 + threadIdx.x; s < s1; s += THREADS) {
    const uint32_t e = (uint32_t)a.experts[s];
    atomicAdd(&base[e < a.E ? e : a.E], 1u);
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.hist[(size_t)blockIdx.x * (a.E + 1) + i] = base[i];
    return;
  }
  prefix_words(base, a.E + 1);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.offsets[i] = (int32_t)base[i];
  __syncthreads();
  place_slots(a.experts, s0, s1, a.E, a.order, base, counts);
}

__global__ void __launch_bounds__(THREADS) place_kernel(RouteArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t *base = lds, *counts = lds + a.E + 1;
  chunk_bases(a.hist, a.E, gridDim.x, base, counts, a.offsets);
  const int64_t s0 = (int64_t)blockIdx.x * a.chunk * a.k, s1 = min(s0 + (int64_t)a.chunk * a.k, a.T * a.k);
  place_slots(a.experts, s0, s1, a.E, a.order, base, counts);
}

// dlogits: normalized weights, w_j (dw_j - sum_i w_i dw_i) at the chosen
// experts and 0 elsewhere; full-softmax weights, p_i ([i chosen] dw_i -
// sum_j w_j dw_j), with p from the logits again. A wavefront per token.
template <class T>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a, const float* dweights, T* dlogits) {
  const uint32_t lane = threadIdx.x & 63;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.T; t += (int64_t)gridDim.x * 4) {
    float inner = 0;
    for (uint32_t j = 0; j < a.k; ++j)
      if (a.experts[t * a.k + j] >= 0) inner += a.weights[t * a.k + j] * dweights[t * a.k + j];
    float big = -INFINITY, z = 0;
    if (!a.normalize) {
      for (uint32_t e = lane; e < a.E; e += 64) {
        float l;
        if (allowed_at<T>(a, t, e, l)) big = l != l || big != big ? NAN : fmaxf(big, l);
      }
      for (int d = 32; d; d >>= 1) {
        const float o = __shfl_xor(big, d);
        big = o != o || big != big ? NAN : fmaxf(big, o);
      }
      for (uint32_t e = lane; e < a.E; e += 64) {
        float l;
        if (allowed_at<T>(a, t, e, l)) z += expf(l - big);
      }
      for (int d = 32; d; d >>= 1) z += __shfl_xor(z, d);
    }
    for (uint32_t e = lane; e < a.E; e += 64) {
      float grad = 0, l;
      if (!a.normalize && allowed_at<T>(a, t, e, l)) grad = -(expf(l - big) / z) * inner;
      for (uint32_t j = 0; j < a.k; ++j)
        if (a.experts[t * a.k + j] == (int32_t)e) {
          const float w = a.weights[t * a.k + j], dw = dweights[t * a.k + j];
          grad = a.normalize ? w * (dw - inner) : grad + w * dw;
        }
      dlogits[t * a.E + e] = from_float<T>(grad);
    }
  }
}

template <class T>
hipError_t route_typed(const RouteArgs& a, uint32_t chunks, uint32_t lds, hipStream_t s) {
  if (a.E <= 8) return launch<route_kernel<T, 1>>(chunks, THREADS, lds, s, a);
  if (a.E <= 16) return launch<route_kernel<T, 2>>(chunks, THREADS, lds, s, a);
  if (a.E <= 32) return launch<route_kernel<T, 4>>(chunks, THREADS, lds, s, a);
  if (a.E <= 64) return launch<route_kernel<T, 8>>(chunks, THREADS, lds, s, a);
  if (a.E <= 128) return launch<route_kernel<T, 16>>(chunks, THREADS, lds, s, a);
  if (a.E <= 256) return launch<route_kernel<T, 32>>(chunks, THREADS, lds, s, a);
  return launch<route_kernel<T, 64>>(chunks, THREADS, lds, s, a);
}

hipError_t place(const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  if (chunks == 1) return hipSuccess;
  return launch<place_kernel, MOST_CHUNKS>(chunks, THREADS, group_lds(a.E, true), s, a);
}

}  // namespace

hipError_t launch_route(MixType type, RouteArgs a, hipStream_t s) {
  const uint32_t chunks = (uint32_t)th::group_chunks(a.T, a.k);
  a.chunk = (uint32_t)th::group_chunk_tokens(a.T, a.k);
  const uint32_t size = type == MIX_F32 ? 4 : 2;
  a.vector = (uintptr_t)a.logits % 16 == 0 && (a.T == 1 || a.ld * size % 16 == 0) &&
             (!a.mask || ((uintptr_t)a.mask % 8 == 0 && a.mask_ld % 8 == 0));
  hipError_t e = type == MIX_BF16  ? route_typed<bf16_t>(a, chunks, group_lds(a.E), s)
                 : type == MIX_F16 ? route_typed<f16_t>(a, chunks, group_lds(a.E), s)
                                   : route_typed<float>(a, chunks, group_lds(a.E), s);
  return e != hipSuccess ? e : place(a, chunks, s);
}

hipError_t launch_group(RouteArgs a, hipStream_t s) {
  const uint32_t chunks = (uint32_t)th::group_chunks(a.T, a.k);
  a.chunk = (uint32_t)th::group_chunk_tokens(a.T, a.k);
  const hipError_t e = launch<count_kernel, MOST>(chunks, THREADS, group_lds(a.E), s, a);
  return e != hipSuccess ? e : place(a, chunks, s);
}

hipError_t launch_route_backward(MixType type, const RouteArgs& a, const float* dweights, void* dlogits,
                                 hipStream_t s) {
  const uint32_t blocks = th::loop_blocks(th::ceil_div(a.T, 4));
  if (type == MIX_BF16) return launch<route_backward_kernel<bf16_t>>(blocks, 256, 0, s, a, dweights, (bf16_t*)dlogits);
  if (type == MIX_F16) return launch<route_backward_kernel<f16_t>>(blocks, 256, 0, s, a, dweights, (f16_t*)dlogits);
  return launch<route_backward_kernel<float>>(blocks, 256, 0, s, a, dweights, (float*)dlogits);
}

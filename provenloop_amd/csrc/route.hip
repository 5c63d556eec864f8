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
#include "mixture.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;

__device__ inline uint64_t u64_shfl_xor(uint64_t v, int m) {
  const uint32_t lo = __shfl_xor((uint32_t)v, m), hi = __shfl_xor((uint32_t)(v >> 32), m);
  return (uint64_t)hi << 32 | lo;
}

// Orders logits as whole numbers above 0: NaN above +inf (as a comparison sort
// of the framework's users puts it), -0 with +0. 0 is kept for "not allowed".
__device__ inline uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
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
// hist[key][chunk]; offsets written by chunk 0.
__device__ void chunk_bases(const uint32_t* hist, uint32_t E, uint32_t chunks, uint32_t* base, uint32_t* total,
                            int32_t* offsets) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (uint32_t key = wave; key <= E; key += WAVES) {
    uint32_t before = 0, all = 0;
    for (uint32_t c = lane; c < chunks; c += 64) {
      const uint32_t n = hist[(size_t)key * chunks + c];
      all += n;
      if (c < blockIdx.x) before += n;
    }
    for (int d = 32; d; d >>= 1) {
      before += __shfl_xor(before, d);
      all += __shfl_xor(all, d);
    }
    if (lane == 0) {
      base[key] = before;
      total[key] = all;
    }
  }
  __syncthreads();
  prefix_words(total, E + 1);
  __syncthreads();
  for (uint32_t key = threadIdx.x; key <= E; key += THREADS) {
    base[key] += total[key];
    if (blockIdx.x == 0) offsets[key] = (int32_t)total[key];
  }
  __syncthreads();
}

// One workgroup's tokens [t0, t1): a group of G lanes per token, 8 experts a
// lane, k rounds of a maximum over (logit, lowest index). Counts the chosen
// experts in `base`.
template <class T, int G>
__device__ void choose(const RouteArgs& a, int64_t t0, int64_t t1, uint32_t* base) {
  const uint32_t g = threadIdx.x % G;
  for (int64_t at = t0; at < t1; at += THREADS / G) {
    const int64_t t = at + threadIdx.x / G;
    if (t >= t1) continue;  // whole groups of G lanes leave together
    uint32_t key[8];
    float l[8], big = -INFINITY;
    for (int i = 0; i < 8; ++i) {
      const uint32_t e = g * 8 + i;
      key[i] = 0;
      l[i] = -INFINITY;
      if (e < a.E && allowed_at<T>(a, t, e, l[i])) key[i] = order_key(l[i]);
    }
    float z = 0;
    for (uint32_t j = 0; j < a.k; ++j) {
      uint64_t best = 0;
      for (int i = 0; i < 8; ++i) {
        const uint64_t c = (uint64_t)key[i] << 32 | (0xffffffffu - (g * 8 + i));
        if (key[i] && c > best) best = c;
      }
      for (int d = 1; d < G; d <<= 1) {
        const uint64_t o = u64_shfl_xor(best, d);
        best = o > best ? o : best;
      }
      const int32_t e = best ? (int32_t)(0xffffffffu - (uint32_t)best) : -1;
      float v = -INFINITY;
      for (int i = 0; i < 8; ++i)
        if (e == (int32_t)(g * 8 + i)) {
          v = l[i];
          key[i] = 0;
        }
      // the chosen logit is in one lane of the group; the others hold -inf, and
      // a NaN has to survive the exchange, so it goes by the owner's lane
      if (G > 1) v = __shfl(v, e < 0 ? 0 : (int)((threadIdx.x & 63) / G * G + e / 8));
      if (e < 0) v = -INFINITY;
      if (j == 0) {
        big = v;
        if (!a.normalize) {
          for (int i = 0; i < 8; ++i)  // the keys but the first chosen one's are still whole
            if (key[i]) z += expf(l[i] - big);
          for (int d = 1; d < G; d <<= 1) z += __shfl_xor(z, d);
          if (e >= 0) z += expf(v - big);
        }
      }
      const float p = e < 0 ? 0.0f : expf(v - big);
      if (a.normalize) z += p;
      if (g == 0) {
        a.experts[t * a.k + j] = e;
        a.weights[t * a.k + j] = p;
        atomicAdd(&base[e < 0 ? a.E : e], 1u);
      }
    }
    if (g == 0) {
      for (uint32_t j = 0; j < a.k; ++j) {
        const float p = a.weights[t * a.k + j];
        a.weights[t * a.k + j] = a.experts[t * a.k + j] < 0 ? 0.0f : p / z;
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
    for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.hist[(size_t)i * gridDim.x + blockIdx.x] = base[i];
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
    for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) a.hist[(size_t)i * gridDim.x + blockIdx.x] = base[i];
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
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t lane = threadIdx.x & 63;
  if (t >= a.T) return;
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

template <class T>
hipError_t route_typed(const RouteArgs& a, uint32_t chunks, size_t lds, hipStream_t s) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(chunks), dim3(THREADS), lds, s, a); };
  if (a.E <= 8) go(route_kernel<T, 1>);
  else if (a.E <= 16) go(route_kernel<T, 2>);
  else if (a.E <= 32) go(route_kernel<T, 4>);
  else if (a.E <= 64) go(route_kernel<T, 8>);
  else if (a.E <= 128) go(route_kernel<T, 16>);
  else if (a.E <= 256) go(route_kernel<T, 32>);
  else go(route_kernel<T, 64>);
  return hipGetLastError();
}

size_t group_lds(uint32_t E) { return (size_t)(WAVES + 1) * (E + 1) * 4; }

hipError_t place(const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  if (chunks > 1) place_kernel<<<chunks, THREADS, group_lds(a.E), s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route(MixType type, RouteArgs a, hipStream_t s) {
  const uint32_t chunks = (uint32_t)th::group_chunks(a.T, a.k);
  a.chunk = (uint32_t)th::group_chunk_tokens(a.T, a.k);
  hipError_t e = type == MIX_BF16  ? route_typed<bf16_t>(a, chunks, group_lds(a.E), s)
                 : type == MIX_F16 ? route_typed<f16_t>(a, chunks, group_lds(a.E), s)
                                   : route_typed<float>(a, chunks, group_lds(a.E), s);
  return e != hipSuccess ? e : place(a, chunks, s);
}

hipError_t launch_group(RouteArgs a, hipStream_t s) {
  const uint32_t chunks = (uint32_t)th::group_chunks(a.T, a.k);
  a.chunk = (uint32_t)th::group_chunk_tokens(a.T, a.k);
  count_kernel<<<chunks, THREADS, group_lds(a.E), s>>>(a);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : place(a, chunks, s);
}

hipError_t launch_route_backward(MixType type, const RouteArgs& a, const float* dweights, void* dlogits,
                                 hipStream_t s) {
  const uint32_t blocks = (uint32_t)th::ceil_div(a.T, 4);
  if (type == MIX_BF16) route_backward_kernel<bf16_t><<<blocks, 256, 0, s>>>(a, dweights, (bf16_t*)dlogits);
  else if (type == MIX_F16) route_backward_kernel<f16_t><<<blocks, 256, 0, s>>>(a, dweights, (f16_t*)dlogits);
  else route_backward_kernel<float><<<blocks, 256, 0, s>>>(a, dweights, (float*)dlogits);
  return hipGetLastError();
}

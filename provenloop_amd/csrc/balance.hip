// Gate with balanced choices: scores of a softmax or of sigmoids, a bias that
// takes part in the choice alone, and experts that lie on nodes of which a token
// may use a few.
//
//   s_e = exp(l_e - max l) / sum over the allowed  or  1 / (1 + exp(-l_e))
//   c_e = s_e + bias_e; without a bias, and with a node's value its largest c, the
//         logits themselves, whose order is the scores'
//   value of a node = its largest c, or the sum of its two largest
// Of the nodes the top_nodes of largest value are kept, of their experts the k of
// largest c, ties to the lowest number each, and
//   w_j = scale s_j / (sum of the chosen s, or 1).
//
// A choice by scores is a choice between numbers that were rounded. It is defined
// by s and c in 64 bits. Those cost a token of 256 experts several times the rest
// of its work, so the numbers are first made in float, and only a token two of
// whose decisive numbers are nearer than float's errors can tell apart goes
// through them again in double.
//
// The lanes of a token, its slots' places and what bounds both are route.hip's.
#include "route_device.h"

using namespace mix;

namespace {

// A candidate as a number that orders like (value, lowest expert first), 0 for
// none: the value's bits made to rise with it, NaN above +inf, over the expert's
// number from the top.
template <class V>
struct Candidate;
__device__ inline uint32_t rising(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline uint64_t rising(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v != v ? ~0ull : b >> 63 ? ~b : b | 1ull << 63;
}
template <>
struct Candidate<float> {
  uint64_t v;
  __device__ inline Candidate() : v(0) {}
  __device__ inline Candidate(float c, uint32_t e) : v((uint64_t)rising(c) << 32 | (0xffffffffu - e)) {}
  __device__ inline bool any() const { return v != 0; }
  __device__ inline bool operator>(const Candidate& o) const { return v > o.v; }
  __device__ inline bool operator==(const Candidate& o) const { return v == o.v; }
  __device__ inline uint32_t expert() const { return 0xffffffffu - (uint32_t)v; }
};
template <>
struct Candidate<double> {
  uint64_t v;
  uint32_t low;
  __device__ inline Candidate() : v(0), low(0) {}
  __device__ inline Candidate(double c, uint32_t e) : v(rising(c)), low(0xffffffffu - e) {}
  __device__ inline bool any() const { return v != 0; }
  __device__ inline bool operator>(const Candidate& o) const { return v > o.v || (v == o.v && low > o.low); }
  __device__ inline bool operator==(const Candidate& o) const { return v == o.v && low == o.low; }
  __device__ inline uint32_t expert() const { return 0xffffffffu - low; }
};
template <int D>
__device__ inline Candidate<float> across(const Candidate<float>& c) {
  Candidate<float> o;
  o.v = mix::across<D>(c.v);
  return o;
}
template <int D>
__device__ inline Candidate<double> across(const Candidate<double>& c) {
  Candidate<double> o;
  o.v = mix::across<D>(c.v);
  o.low = mix::across<D>(c.low);
  return o;
}
template <int G, class V, int D = 1>
__device__ inline Candidate<V> largest(const Candidate<V>& c) {
  if constexpr (D < G) {
    const Candidate<V> o = across<D>(c);
    return largest<G, V, 2 * D>(o > c ? o : c);
  } else {
    return c;
  }
}
// Over a token's lanes; NaN if any is.
template <int G, int D = 1>
__device__ inline float most(float v) {
  if constexpr (D < G) {
    const float o = __uint_as_float(mix::across<D>(__float_as_uint(v)));
    return most<G, 2 * D>(o != o || v != v ? NAN : fmaxf(v, o));
  } else {
    return v;
  }
}
template <int G, int D = 1>
__device__ inline double sum(double v) {
  if constexpr (D < G) return sum<G, 2 * D>(v + __longlong_as_double(mix::across<D>((uint64_t)__double_as_longlong(v))));
  else return v;
}
template <int G>
__device__ inline float sum(float v) {
  return group_sum<G>(v);
}

// A token's lanes see what each has laid in LDS; they are in one wavefront, whose
// LDS accesses are answered in order.
__device__ inline void lanes_agree() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}


constexpr int keep(int G) { return G >= 32 ? 1 : G >= 4 ? 32 / G : 8; }  // choices that one lane can have to keep

// A token's logits, 8 a lane, and which of them are allowed.
struct Row {
  float l[8];
  uint32_t allowed;  // a bit each
  float big;         // the largest allowed; NaN if one is
};

// Of a token's experts with numbers c those on the nodes that it may use. own: LDS
// for the numbers.
struct Kept {
  uint32_t allowed;
  float clear;  // by how much the least of the kept nodes is above the best of the others
};
template <int G, class V>
__device__ inline Kept keep_nodes(const RouteArgs& a, uint32_t g, const V (&c)[8], uint32_t allowed, V* own) {
  // a lane takes every G-th node: its value in place of its first expert's c,
  // then whether it is kept
  const uint32_t per = a.E / a.nodes, to_node = (1u << 20) / per + 1;  // e * to_node >> 20 = e / per, for e < 512
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (g * 8 + i < a.E) own[g * 8 + i] = allowed >> i & 1 ? c[i] : (V)-INFINITY;
  lanes_agree();
  for (uint32_t n = g; n < a.nodes; n += G) {
    V one = -INFINITY, two = -INFINITY;
    bool nan = false;
    for (uint32_t i = 0; i < per; ++i) {
      const V v = own[n * per + i];
      nan |= v != v;
      if (v > one) {
        two = one;
        one = v;
      } else if (v > two) {
        two = v;
      }
    }
    if (a.node_best == 2 && two > (V)-INFINITY) one += two;
    own[n * per] = nan ? (V)NAN : one;
  }
  lanes_agree();
  uint32_t kept = 0, at = 0;
  float least = INFINITY, above = -INFINITY;  // of the kept, of the others
  for (uint32_t n = g; n < a.nodes; n += G, ++at) {
    const V mine = own[n * per];
    const Candidate<V> me(mine, n);
    uint32_t before = 0;
    for (uint32_t m = 0; m < a.nodes; ++m) before += Candidate<V>(own[m * per], m) > me;
    if (before < a.top_nodes) {
      kept |= 1u << at;
      least = fminf(least, (float)mine);
    } else {
      above = fmaxf(above, (float)mine);
    }
  }
  lanes_agree();
  at = 0;
  for (uint32_t n = g; n < a.nodes; n += G, ++at) own[n * per] = kept >> at & 1 ? (V)1 : (V)0;
  lanes_agree();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t ex = g * 8 + i;
    if (ex < a.E && own[(ex * to_node >> 20) * per] == (V)0) allowed &= ~(1u << i);
  }
  lanes_agree();  // before the next numbers are laid there
  if constexpr (std::is_same<V, float>::value) {
    above = most<G>(above);
    return Kept{allowed, above > -INFINITY ? -most<G>(-least) - above : INFINITY};
  }
  return Kept{allowed, 0};
}

// The largest key of a token's lanes.
template <int G>
__device__ inline uint32_t most_key(uint32_t v) {
  if constexpr (G > 1) v = max(v, mix::across<1>(v));
  if constexpr (G > 2) v = max(v, mix::across<2>(v));
  if constexpr (G > 4) v = max(v, mix::across<4>(v));
  if constexpr (G > 8) v = max(v, mix::across<8>(v));
  if constexpr (G > 16) {
    const auto o = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(o[0], o[1]);
  }
  if constexpr (G > 32) {
    const auto o = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(o[0], o[1]);
  }
  return v;
}
__device__ inline float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Chooses by scores in float, or returns false where those are too near to tell.
// A candidate is one word: its c made to rise, the lowest 3 bits its place among
// the lane's 8, so that the lane's candidates are put in order by 38 maxima and
// minima; equal c need no order of their own, since they are too near. The rounds
// then take the largest of the lanes' first.
template <int G>
__device__ inline bool pick_near(const RouteArgs& a, const Row& r, uint32_t g, float* own, int32_t (&e)[keep(G)]) {
  constexpr float LOG2E = 1.44269504f;
  float c[8];
  // exp through exp2 of a rounded product: off by |l| 2^-24 of itself, which is
  // below 2^-24 of the score's range since x exp(-x) < 1
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * r.l[i]));
  } else {
    float z = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = r.allowed >> i & 1 ? __builtin_amdgcn_exp2f(LOG2E * (r.l[i] - r.big)) : 0.0f;
      z += c[i];
    }
    z = __builtin_amdgcn_rcpf(group_sum<G>(z));
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] *= z;
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] += g * 8 + i < a.E ? a.bias[g * 8 + i] : 0.0f;
  }
  uint32_t s[8], size = 0, allowed = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!(r.allowed >> i & 1) || c[i] == -INFINITY) continue;
    allowed |= 1u << i;
    size = max(size, __float_as_uint(c[i]) & 0x7fffffffu);
  }
  // How near two decisive numbers may come. A sigmoid is off by up to 2^-22, a
  // softmax's share by 2^-20 (a sum 14 additions deep), a sum with the bias by
  // 2^-24 of its size, and the word leaves 2^-20 of it away; a node's sum of two
  // twice all that, and so does a difference. NaN is near everything.
  float clear = INFINITY;  // the least difference that decides something
  const float near = (a.sigmoid ? 0x1p-20f : 0x1p-18f) + 0x1p-18f * __uint_as_float(most_key<G>(size));

  // the lanes of a node: a power of two of them alone, or 0
  const uint32_t per = a.E / a.nodes, lanes = a.nodes > 1 && per % 8 == 0 && __popc(per) == 1 ? per / 8 : 0;
  if (a.nodes > 1 && !lanes) {
    const Kept k = keep_nodes<G>(a, g, c, allowed, own);
    allowed = k.allowed;
    clear = k.clear;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = allowed >> i & 1 ? (rising(c[i]) & ~7u) | (7 - i) : 0;
  auto order = [&](int i, int j) __attribute__((always_inline)) {
    const uint32_t hi = max(s[i], s[j]), lo = min(s[i], s[j]);
    s[i] = hi;
    s[j] = lo;
  };
  order(0, 1), order(2, 3), order(4, 5), order(6, 7), order(0, 2), order(1, 3), order(4, 6), order(5, 7);
  order(1, 2), order(5, 6), order(0, 4), order(1, 5), order(2, 6), order(3, 7), order(2, 4), order(3, 5);
  order(1, 2), order(3, 4), order(5, 6);

  if (lanes) {
    // a node's two largest by all of its lanes
    float one = s[0] ? key_value(s[0]) : -INFINITY, two = s[1] ? key_value(s[1]) : -INFINITY;
    for (uint32_t d = 1; d < lanes; d *= 2) {
      const float o1 = __shfl_xor(one, d), o2 = __shfl_xor(two, d);
      two = fmaxf(fminf(one, o1), fmaxf(two, o2));
      one = fmaxf(one, o1);
    }
    const float mine = a.node_best == 2 && two > -INFINITY ? one + two : one;
    if (g % lanes == 0) own[g / lanes] = mine;
    lanes_agree();
    uint32_t before = 0;
    for (uint32_t n = 0; n < a.nodes; ++n) before += own[n] > mine || (own[n] == mine && n < g / lanes);
    const bool kept = before < a.top_nodes;
    const float least = -most<G>(kept ? -mine : -INFINITY), above = most<G>(kept ? -INFINITY : mine);
    if (above > -INFINITY) clear = least - above;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = kept ? s[i] : 0;
    lanes_agree();  // before the next numbers are laid there
  }

  const uint32_t lane = threadIdx.x & 63, first_lane = lane & ~(uint32_t)(G - 1);
  float last = INFINITY;
  auto next = [&](int32_t& expert) __attribute__((always_inline)) {
    const uint32_t best = most_key<G>(s[0]);
    uint64_t here = __ballot(s[0] == best) >> first_lane;
    if constexpr (G < 64) here &= (1ull << G) - 1;
    const uint32_t from = G == 1 ? lane : first_lane + __ffsll((unsigned long long)here) - 1;
    const bool out = lane == from;
#pragma unroll
    for (int i = 0; i < 7; ++i) s[i] = out ? s[i + 1] : s[i];
    s[7] = out ? 0 : s[7];
    const float value = key_value(best);
    if (best) {
      clear = fminf(clear, last - value);
      last = value;
    }
    expert = best ? (int32_t)((from - first_lane) * 8 + 7 - (best & 7)) : -1;
  };
#pragma unroll
  for (int q = 0; q < keep(G); ++q) {
    e[q] = -1;
    if (q * G < (int)a.k) {
      for (uint32_t j = 0; j < G && q * G + j < a.k; ++j) {
        int32_t expert;
        next(expert);
        if (g == j) e[q] = expert;
      }
    }
  }
  int32_t expert;
  next(expert);  // the best that is not chosen has to be clearly less
  return clear > near;
}

// Chooses a token's experts: lane j of its G lanes keeps choices j, j + G, ... in
// e. V: the type of the decisive numbers, double for scores, float for logits.
// own: LDS for the token's c, 8 a lane.
template <class V, int G>
__device__ inline void pick(const RouteArgs& a, const Row& r, uint32_t g, V* own, int32_t (&e)[keep(G)]) {
  constexpr bool SCORES = std::is_same<V, double>::value;
  V c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = (V)r.l[i];
  if constexpr (SCORES) {
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = (V)1 / ((V)1 + exp(-c[i]));
    } else {
      V z = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = exp(c[i] - (V)r.big);
        z += r.allowed >> i & 1 ? c[i] : (V)0;
      }
      z = sum<G>(z);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] /= z;
    }
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (g * 8 + i < a.E) c[i] += (V)a.bias[g * 8 + i];
    }
  }
  uint32_t allowed = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if ((r.allowed >> i & 1) && !(c[i] == (V)-INFINITY)) allowed |= 1u << i;

  if (a.nodes > 1) allowed = keep_nodes<G>(a, g, c, allowed, own).allowed;

  // without a bias the experts go by their logits, and only the nodes by scores
  const bool by_scores = SCORES && a.bias;
  Candidate<V> s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (allowed >> i & 1) s[i] = Candidate<V>(by_scores ? c[i] : (V)r.l[i], g * 8 + i);
  // Batcher's odd-even merge of 8: 19 exchanges
  auto order = [&](int i, int j) __attribute__((always_inline)) {
    if (s[j] > s[i]) {
      const Candidate<V> t = s[i];
      s[i] = s[j];
      s[j] = t;
    }
  };
  order(0, 1), order(2, 3), order(4, 5), order(6, 7), order(0, 2), order(1, 3), order(4, 6), order(5, 7);
  order(1, 2), order(5, 6), order(0, 4), order(1, 5), order(2, 6), order(3, 7), order(2, 4), order(3, 5);
  order(1, 2), order(3, 4), order(5, 6);
  // the next largest leaves its lane
  auto next = [&]() __attribute__((always_inline)) {
    const Candidate<V> best = largest<G>(s[0]);
    if (best.any() && s[0] == best) {
#pragma unroll
      for (int i = 0; i < 7; ++i) s[i] = s[i + 1];
      s[7] = Candidate<V>();
    }
    return best;
  };
#pragma unroll
  for (int q = 0; q < keep(G); ++q) {
    e[q] = -1;
    if (q * G < (int)a.k) {
      for (uint32_t j = 0; j < G && q * G + j < a.k; ++j) {
        const Candidate<V> best = next();
        if (g == j && best.any()) e[q] = (int32_t)best.expert();
      }
    }
  }
}

// LDS for the numbers of a wavefront's tokens: a float for each of a lane's 8
// experts, which are taken by one token at a time where it is doubles that they
// have to hold.
constexpr uint32_t space_of_wave(int G) { return G < 64 ? 64 * 8 * 4 : 64 * 8 * 8; }

// One workgroup's tokens [t0, t1): G lanes a token, 8 experts a lane. Counts the
// chosen experts in `base`.
template <class T, int G, bool SCORES>
__device__ void choose_balanced(const RouteArgs& a, int64_t t0, int64_t t1, uint32_t* base, char* space) {
  const uint32_t g = threadIdx.x % G;
  const bool whole = g * 8 + 8 <= a.E && a.vector;
  char* wave_space = space + threadIdx.x / 64 * space_of_wave(G);
  float* own = (float*)wave_space + (threadIdx.x & 63) / G * (G * 8);
  for (int64_t at = t0; at < t1; at += THREADS / G) {
    const int64_t t = at + threadIdx.x / G;
    if (t >= t1) continue;  // whole groups of G lanes leave together
    const T* row = (const T*)a.logits + t * a.ld;
    const uint8_t* mask = a.mask ? a.mask + t * a.mask_ld + g * 8 : nullptr;
    Row r;
    r.allowed = 0;
    T l[8];
    uint64_t in = ~0ull;  // a byte per expert
    if (whole) {
      __builtin_memcpy(l, __builtin_assume_aligned(row + g * 8, 16), sizeof(l));
      if (mask) __builtin_memcpy(&in, __builtin_assume_aligned(mask, 8), 8);
    } else {
      for (uint32_t i = 0; i < 8; ++i) {
        const bool is = g * 8 + i < a.E;
        l[i] = is ? row[g * 8 + i] : (T)0.0f;
        if (!is || (mask && !mask[i])) in &= ~(0xffull << (8 * i));
      }
    }
    r.big = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r.l[i] = (float)l[i];
      if ((in >> (8 * i) & 0xff) && !(r.l[i] == -INFINITY)) {
        r.allowed |= 1u << i;
        r.big = r.l[i] != r.l[i] || r.big != r.big ? NAN : fmaxf(r.big, r.l[i]);
      }
    }
    r.big = most<G>(r.big);

    int32_t e[keep(G)];
    if constexpr (SCORES) {
      const bool sure = pick_near<G>(a, r, g, own, e);
      for (uint64_t left = __ballot(!sure); left;) {  // one token after the other
        const uint32_t first = (uint32_t)(__ffsll((unsigned long long)left) - 1) / G;
        if ((threadIdx.x & 63) / G == first) pick<double, G>(a, r, g, (double*)wave_space, e);
        left &= G == 64 ? 0 : ~(((1ull << (G % 64)) - 1) << (first * G));
      }
    } else {
      pick<float, G>(a, r, g, own, e);
    }

    // scores of the chosen; normalized ones from the largest chosen logit where
    // they are a softmax, or sigmoids so small that they are exp(l)
    float z = 1, p[keep(G)], lc[keep(G)], top = -INFINITY;
#pragma unroll
    for (int q = 0; q < keep(G); ++q) {
      lc[q] = e[q] < 0 ? -INFINITY : (float)row[e[q]];
      top = lc[q] != lc[q] || top != top ? NAN : fmaxf(top, lc[q]);
    }
    top = most<G>(top);
    const bool by_exp = !a.sigmoid || (a.normalize && top < -40.0f);
    const float from = a.normalize ? top : r.big;
    if (a.normalize) {
      z = 0;
    } else if (!a.sigmoid) {
      z = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r.allowed >> i & 1) z += expf(r.l[i] - from);
      z = group_sum<G>(z);
    }
#pragma unroll
    for (int q = 0; q < keep(G); ++q) {
      p[q] = e[q] < 0 ? 0.0f : by_exp ? expf(lc[q] - from) : 1.0f / (1.0f + expf(-lc[q]));
      if (a.normalize) z += p[q];
    }
    if (a.normalize) z = group_sum<G>(z);
#pragma unroll
    for (int q = 0; q < keep(G); ++q) {
      const uint32_t j = q * G + g;
      if (j < a.k) {
        a.experts[t * a.k + j] = e[q];
        a.weights[t * a.k + j] = e[q] < 0 ? 0.0f : a.scale * (p[q] / z);
        atomicAdd(&base[e[q] < 0 ? a.E : e[q]], 1u);
      }
    }
  }
}

constexpr uint32_t space_bytes(int G, uint32_t nodes) { return nodes > 1 ? WAVES * space_of_wave(G) : 0; }

template <class T, int G, bool SCORES>
__global__ void __launch_bounds__(THREADS) balanced_kernel(RouteArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  uint32_t* words = lds + space_bytes(G, a.nodes) / 4;
  uint32_t *base = words, *counts = words + a.E + 1;
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) base[i] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * a.chunk, t1 = min(t0 + (int64_t)a.chunk, a.T);
  choose_balanced<T, G, SCORES>(a, t0, t1, base, (char*)lds);
  end_chunk(a, base, counts);
}

// With p the weights without their scale, P = sum p_i dw_i over the chosen:
//   normalized    softmax  w_j (dw_j - P)             sigmoid  w_j (1 - s_j) (dw_j - P), at the chosen
//   not           softmax  [chosen] w_e dw_e - scale s_e P     sigmoid  w_j (1 - s_j) dw_j
// A wavefront a token.
template <class T>
__global__ void __launch_bounds__(256) balanced_backward_kernel(RouteArgs a, const float* dweights, T* dlogits) {
  const uint32_t lane = threadIdx.x & 63;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.T; t += (int64_t)gridDim.x * 4) {
    float inner = 0;  // scale P
    for (uint32_t j = 0; j < a.k; ++j)
      if (a.experts[t * a.k + j] >= 0) inner += a.weights[t * a.k + j] * dweights[t * a.k + j];
    const bool full = !a.normalize && !a.sigmoid;
    float big = -INFINITY, z = 0;
    if (full) {
      for (uint32_t e = lane; e < a.E; e += 64) {
        float l;
        if (allowed_at<T>(a, t, e, l)) big = l != l || big != big ? NAN : fmaxf(big, l);
      }
      big = most<64>(big);
      for (uint32_t e = lane; e < a.E; e += 64) {
        float l;
        if (allowed_at<T>(a, t, e, l)) z += expf(l - big);
      }
      z = group_sum<64>(z);
    }
    for (uint32_t e = lane; e < a.E; e += 64) {
      float grad = 0, l;
      if (full && allowed_at<T>(a, t, e, l)) grad = -(expf(l - big) / z) * inner;
      for (uint32_t j = 0; j < a.k; ++j) {
        if (a.experts[t * a.k + j] != (int32_t)e) continue;
        const float w = a.weights[t * a.k + j];
        const float d = w * (a.normalize ? dweights[t * a.k + j] - inner / a.scale : dweights[t * a.k + j]);
        if (!a.sigmoid) grad += d;
        else grad += d * (1.0f / (1.0f + expf(to_float(((const T*)a.logits)[t * a.ld + e]))));
      }
      dlogits[t * a.E + e] = from_float<T>(grad);
    }
  }
}

template <class T, int G>
hipError_t sized(const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  constexpr uint32_t most = space_bytes(G, 2) + group_lds(G * 8);
  // the logits decide where they order the experts as their scores do
  const bool scores = a.bias || (a.nodes > 1 && a.node_best == 2);
  const uint32_t lds = space_bytes(G, a.nodes) + group_lds(a.E);
  return scores ? launch<balanced_kernel<T, G, true>, most>(chunks, THREADS, lds, s, a)
                : launch<balanced_kernel<T, G, false>, most>(chunks, THREADS, lds, s, a);
}

template <class T>
hipError_t typed(const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  if (a.E <= 8) return sized<T, 1>(a, chunks, s);
  if (a.E <= 16) return sized<T, 2>(a, chunks, s);
  if (a.E <= 32) return sized<T, 4>(a, chunks, s);
  if (a.E <= 64) return sized<T, 8>(a, chunks, s);
  if (a.E <= 128) return sized<T, 16>(a, chunks, s);
  if (a.E <= 256) return sized<T, 32>(a, chunks, s);
  return sized<T, 64>(a, chunks, s);
}

}  // namespace

hipError_t launch_balanced(MixType type, const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  return type == MIX_BF16 ? typed<bf16_t>(a, chunks, s) : type == MIX_F16 ? typed<f16_t>(a, chunks, s) : typed<float>(a, chunks, s);
}

hipError_t launch_balanced_backward(MixType type, const RouteArgs& a, const float* dweights, void* dlogits,
                                    hipStream_t s) {
  const uint32_t blocks = th::loop_blocks(th::ceil_div(a.T, 4));
  if (type == MIX_BF16) return launch<balanced_backward_kernel<bf16_t>>(blocks, 256, 0, s, a, dweights, (bf16_t*)dlogits);
  if (type == MIX_F16) return launch<balanced_backward_kernel<f16_t>>(blocks, 256, 0, s, a, dweights, (f16_t*)dlogits);
  return launch<balanced_backward_kernel<float>>(blocks, 256, 0, s, a, dweights, (float*)dlogits);
}

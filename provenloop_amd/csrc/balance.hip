// Gate with balanced choices: scores of a softmax or of sigmoids, a bias that
// takes part in the choice alone, and experts that lie on nodes of which a token
// may use a few.
//
//   s_e = exp(l_e - max l) / sum over the allowed  or  1 / (1 + exp(-l_e))
//   c_e = s_e + bias_e; without a bias the logit l_e, whose order is the scores' and
//         which tells apart what scores in 64 bits round to one number
//   value of a node = its largest c, or the sum of its two largest (without a bias,
//                     of its two largest s)
// Of the nodes the top_nodes of largest value are kept, of their experts the k of
// largest c, ties to the lowest number each, and
//   w_j = scale s_j / (sum of the chosen s, or 1).
//
// A choice by scores is a choice between numbers that were rounded. It is defined
// by s and c in 64 bits. Those cost a token of 256 experts several times the rest
// of its work, so its lanes first make the numbers in float, and only a token two
// of whose decisive numbers are nearer than float's errors can tell apart is
// decided again in double, by a whole wavefront, once the workgroup's others are
// done: next to them double's registers would cost the loop that all go through.
//
// Up to 16 lanes take a token, several chunks of 8 experts a lane. Chunks are put in
// order in a lane's registers and merged there and then across the lanes, 8 numbers
// with 8: the fewer lanes a token has, the fewer steps go across lanes, which cost
// most. 65536 tokens of 256 experts on 8 nodes, 8 chosen, bf16 logits, kernel times of
// one trace: 44 us where no two numbers come near, 52 (57 on another card) where a few
// tokens of nearly every workgroup are decided again, and 16 for the launch that places
// their slots; 57 and 67 us a call in a series. A token that is decided again takes 13
// us and more, waiting for one step after the other. Both launches' bytes are 8 us at a
// copy's rate; about 2100 vector instructions a wavefront's 8 tokens are 33 of the 44.
// One token takes 9.3 us of 64 experts and 20 of 256: the chain of its steps.
//
// A workgroup of 16 wavefronts has 128 registers a lane, and the forms for more than
// 128 experts (more than 64 with more than 8 choices) need some more: 28 bytes a lane
// are in scratch for 256 experts and 48 for 512, 44, 260 and 244 for 128, 256 and 512
// with more than 8 choices.
#include "route_device.h"

using namespace mix;

namespace {

// A number's bits made to rise with its value, NaN above +inf, -0 with +0; never 0.
__device__ inline uint32_t rising(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline uint64_t rising(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v != v ? ~0ull : b >> 63 ? ~b : b | 1ull << 63;
}
__device__ inline float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The largest of G lanes' words.
template <int G>
__device__ inline uint32_t most_key(uint32_t v) {
  if constexpr (G > 1) v = max(v, across<1>(v));
  if constexpr (G > 2) v = max(v, across<2>(v));
  if constexpr (G > 4) v = max(v, across<4>(v));
  if constexpr (G > 8) v = max(v, across<8>(v));
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
// The largest of G lanes' numbers; NaN if any is.
template <int G>
__device__ inline float most(float v) {
  return value_of(most_key<G>(rising(v)));
}

// A wavefront's lanes see what each has laid in LDS, whose accesses are answered
// in order.
__device__ inline void lanes_agree() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---------------------------------------------------------------- experts on lanes
// Experts in chunks of 8, a node in chunks of its own (the last one's rest is
// empty). Chunk i of a token's G lanes is the (i / G)-th of lane i % G.
struct Chunks {
  uint32_t per, chunks_per;  // experts and chunks of a node
};
__host__ __device__ inline Chunks chunks_of(uint32_t E, uint32_t nodes) {
  const uint32_t per = E / nodes;
  return Chunks{per, (per + 7) / 8};
}

// What decides: the scores, with a bias or as sums of two, or else the logits.
__device__ inline bool by_scores(const RouteArgs& a) { return a.bias || (a.nodes > 1 && a.node_best == 2); }

// LDS floats of a lane: two of each chunk, one of each node.
constexpr uint32_t lane_space(int C) { return 3 * C; }

// ---------------------------------------------------------------- 8 numbers in falling order
// A candidate is a double: its c, which float's 24 bits leave 29 bits of, and below
// these the expert's number, so that of equal c the lowest expert's is the larger.
// -inf: none; c is not -0, whose expert would be read as another's.
__device__ inline double candidate(float c, uint32_t e) {
  const uint64_t b = (uint64_t)__double_as_longlong((double)c);
  const uint32_t low = c == -INFINITY ? 0 : c < 0 ? e : 511 - e;
  return __longlong_as_double((long long)(b | low));
}
__device__ inline int32_t expert_of(double v) {
  const uint32_t low = (uint32_t)(uint64_t)__double_as_longlong(v) & 511;
  return v == -INFINITY ? -1 : (int32_t)(v < 0 ? low : 511 - low);
}
template <int I, int J>
__device__ inline void order(double (&s)[8]) {
  const double hi = fmax(s[I], s[J]), lo = fmin(s[I], s[J]);
  s[I] = hi;
  s[J] = lo;
}
__device__ inline void sort8(double (&s)[8]) {  // Batcher's odd-even merge
  order<0, 1>(s), order<2, 3>(s), order<4, 5>(s), order<6, 7>(s), order<0, 2>(s), order<1, 3>(s), order<4, 6>(s);
  order<5, 7>(s), order<1, 2>(s), order<5, 6>(s), order<0, 4>(s), order<1, 5>(s), order<2, 6>(s), order<3, 7>(s);
  order<2, 4>(s), order<3, 5>(s), order<1, 2>(s), order<3, 4>(s), order<5, 6>(s);
}
// top = the 8 largest of both; rest: the largest of what was left out, if asked for.
__device__ inline void merge8(double (&top)[8], const double (&s)[8], double& rest, bool ask) {
  if (ask) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rest = fmax(rest, fmin(top[i], s[7 - i]));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) top[i] = fmax(top[i], s[7 - i]);  // falls and rises: three steps put it in order
  order<0, 4>(top), order<1, 5>(top), order<2, 6>(top), order<3, 7>(top);
  order<0, 2>(top), order<1, 3>(top), order<4, 6>(top), order<5, 7>(top);
  order<0, 1>(top), order<2, 3>(top), order<4, 5>(top), order<6, 7>(top);
}
// The 8 largest of G lanes' lists, in all of them.
template <int G>
__device__ inline void merge_lanes(double (&top)[8], double& rest, bool ask) {
#pragma unroll 1
  for (int d = 1; d < G; d *= 2) {
    double s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = __shfl_xor(top[i], d);
    if (ask) rest = fmax(rest, __shfl_xor(rest, d));
    merge8(top, s, rest, ask);
  }
}

// ---------------------------------------------------------------- in float
// c becomes -inf on the nodes that are not kept. Returns by how much the least of
// the kept is above the best of the others. own: the token's LDS.
template <int G, int C>
__device__ inline float keep_nodes(const RouteArgs& a, uint32_t chunks_per, uint32_t g, float (&c)[8 * C], float* own) {
  float* values = own + 2 * G * C;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    float one = -INFINITY, two = -INFINITY;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      two = fmaxf(two, fminf(one, c[8 * i + r]));
      one = fmaxf(one, c[8 * i + r]);
    }
    *(float2*)&own[2 * (i * G + g)] = float2{one, two};
    __builtin_amdgcn_sched_barrier(0);
  }
  lanes_agree();
#pragma unroll 1
  for (uint32_t n = g; n < a.nodes; n += G) {
    float one = -INFINITY, two = -INFINITY;
    for (uint32_t q = n * chunks_per; q < (n + 1) * chunks_per; ++q) {
      const float2 v = *(const float2*)&own[2 * q];
      two = fmaxf(fminf(one, v.x), fmaxf(two, v.y));
      one = fmaxf(one, v.x);
    }
    values[n] = a.node_best == 2 && two > -INFINITY ? one + two : one;
  }
  lanes_agree();
  uint64_t kept = 0;  // a bit for each node
  float least = INFINITY, above = -INFINITY;
#pragma unroll 1
  for (uint32_t at = 0; at < a.nodes; at += G) {  // the same rounds for all lanes, which vote in them
    const uint32_t n = at + g;
    const float mine = n < a.nodes ? values[n] : -INFINITY;
    uint32_t before = n < a.nodes ? 0 : a.nodes;
    for (uint32_t o = 0; o < a.nodes; ++o) {
      const float v = values[o];
      before += v > mine || (v == mine && o < n);
    }
    const bool is = before < a.top_nodes;
    least = is ? fminf(least, mine) : least;
    above = is ? above : fmaxf(above, mine);
    const uint64_t all = __ballot(is) >> ((threadIdx.x & 63) & ~(uint32_t)(G - 1));
    kept |= (all & ((1ull << G) - 1)) << at;
  }
  lanes_agree();  // before the next token's numbers are laid there
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t n = min((i * G + g) / chunks_per, 63u);
#pragma unroll
    for (int r = 0; r < 8; ++r) c[8 * i + r] = kept >> n & 1 ? c[8 * i + r] : -INFINITY;
  }
  above = most<G>(above);
  return above > -INFINITY ? -most<G>(-least) - above : INFINITY;
}

// ---------------------------------------------------------------- in double
// The largest of a wavefront's lanes.
__device__ inline uint64_t most_key64(uint64_t v) {
  auto step = [&](uint64_t o) __attribute__((always_inline)) { v = o > v ? o : v; };
  step(across<1>(v));
  step(across<2>(v));
  step(across<4>(v));
  step(across<8>(v));
  auto swapped = [&](auto lo, auto hi) __attribute__((always_inline)) {
    const uint64_t x = (uint64_t)hi[0] << 32 | lo[0], y = (uint64_t)hi[1] << 32 | lo[1];
    v = x > y ? x : y;
  };
  swapped(__builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false),
          __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false));
  swapped(__builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false),
          __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false));
  return v;
}

// The same choice of one token by a whole wavefront, EACH neighbouring experts a
// lane; d: LDS for 64 EACH doubles. Lane j returns choice j and its logit. A few tokens go through
// it, each once in a while, so what it takes is fetching its code and waiting for
// one step after the other: exps and quotients go side by side (65.4 us against 67.2
// in the case above with one after the other and shuffles through LDS).
template <class T, int EACH>
__device__ inline int32_t pick_exactly(const RouteArgs& a, int64_t t, double* d, float& lc) {
  constexpr int SIDE = EACH < 4 ? EACH : 4;  // exps and quotients side by side
  const uint32_t lane = threadIdx.x & 63, e0 = lane * EACH;
  const bool scores = by_scores(a);
  float l[EACH], b[EACH], big = -INFINITY;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const uint32_t e = min(e0 + i, a.E - 1);
    l[i] = to_float(((const T*)a.logits)[t * a.ld + e]);
    b[i] = a.bias ? a.bias[e] : 0.0f;
    if (e0 + i >= a.E || (a.mask && !a.mask[t * a.mask_ld + e])) l[i] = -INFINITY;
    big = l[i] != l[i] || big != big ? NAN : fmaxf(big, l[i]);
  }
  double c[EACH];
  if (!scores) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) c[i] = l[i];
  } else {
    big = a.sigmoid ? 0.0f : most<64>(big);
#pragma unroll
    for (int i = 0; i < EACH; ++i) d[e0 + i] = a.sigmoid ? -(double)l[i] : (double)l[i] - (double)big;
    double z = 0;
#pragma unroll SIDE
    for (int i = 0; i < EACH; ++i) {
      const double v = exp(d[e0 + i]);
      d[e0 + i] = v;
      z += v;
    }
    if (!a.sigmoid)
#pragma unroll 1
      for (int m = 1; m < 64; m *= 2) z += __shfl_xor(z, m);
#pragma unroll SIDE
    for (int i = 0; i < EACH; ++i) {
      const double v = d[e0 + i];
      d[e0 + i] = (a.sigmoid ? 1.0 : v) / (a.sigmoid ? 1.0 + v : z);
    }
    // a bias of -inf withholds its expert whatever the score, which may be NaN
#pragma unroll
    for (int i = 0; i < EACH; ++i) c[i] = l[i] == -INFINITY || b[i] == -INFINITY ? -INFINITY : d[e0 + i] + (double)b[i];
  }
  if (a.nodes > 1) {
    // a node's value and then whether it is kept are laid in its first expert's place
    const uint32_t per = a.E / a.nodes;
#pragma unroll
    for (int i = 0; i < EACH; ++i) d[e0 + i] = c[i];
    lanes_agree();
#pragma unroll 1
    for (uint32_t n = lane; n < a.nodes; n += 64) {
      double one = -INFINITY, two = -INFINITY;
      bool nan = false;
#pragma unroll 4
      for (uint32_t i = 0; i < per; ++i) {
        const double v = d[n * per + i];
        nan |= v != v;
        two = fmax(two, fmin(one, v));
        one = fmax(one, v);
      }
      if (a.node_best == 2 && two > -INFINITY) one += two;
      d[n * per] = nan ? NAN : one;
    }
    lanes_agree();
    uint32_t is = 0, at = 0;
#pragma unroll 1
    for (uint32_t n = lane; n < a.nodes; n += 64, ++at) {
      const uint64_t mine = rising(d[n * per]);
      uint32_t before = 0;
#pragma unroll 4
      for (uint32_t m = 0; m < a.nodes; ++m) {
        const uint64_t v = rising(d[m * per]);
        before += v > mine || (v == mine && m < n);
      }
      if (before < a.top_nodes) is |= 1u << at;
    }
    lanes_agree();
    at = 0;
#pragma unroll 1
    for (uint32_t n = lane; n < a.nodes; n += 64, ++at) d[n * per] = is >> at & 1;
    lanes_agree();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (e0 + i < a.E && d[(e0 + i) / per * per] == 0) c[i] = -INFINITY;
    lanes_agree();  // before the next token's numbers are laid there
  }
  uint64_t key[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    // without a bias the experts go by their logits, and only the nodes by scores
    key[i] = c[i] == -INFINITY ? 0 : rising(scores && !a.bias ? (double)l[i] : c[i]);
  }
  int32_t chosen = -1;  // of choice number `lane`
#pragma unroll 1
  for (uint32_t j = 0; j < a.k; ++j) {
    uint64_t mine = 0;  // the largest of this lane's, the lowest of equals at `at`
    uint32_t at = 0;
    float own = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      at = key[i] > mine ? i : at;
      own = key[i] > mine ? l[i] : own;
      mine = key[i] > mine ? key[i] : mine;
    }
    const uint64_t best = most_key64(mine);
    if (!best) break;
    const uint32_t from = __ffsll((unsigned long long)__ballot(mine == best)) - 1;
    at = __builtin_amdgcn_readlane(at, from);
    own = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own), from));
    if (lane == j) {
      chosen = (int32_t)(from * EACH + at);
      lc = own;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) key[i] = lane == from && i == (int)at ? 0 : key[i];
  }
  return chosen;
}

// ---------------------------------------------------------------- weights
// The weights of the choices of one token, which its G lanes keep, from their
// logits lc (-inf: none). Normalized ones are taken from the largest chosen logit:
// exp(l - top) of a softmax; of sigmoids, with `from` the largest or 0 if that is less,
// s exp(-from) = exp(l - from) / (1 + exp(l)) for l <= 0, which is a float wherever the
// weight is, though s itself may be none. z_all: sum of exp(l - big) over the allowed,
// of a softmax that is not normalized.
template <int G, int KEEP>
__device__ inline void weigh(const RouteArgs& a, const float (&lc)[KEEP], float big, float z_all, float (&w)[KEEP]) {
  float top = -INFINITY;
  if (a.normalize) {
#pragma unroll
    for (int q = 0; q < KEEP; ++q) top = lc[q] != lc[q] || top != top ? NAN : fmaxf(top, lc[q]);
    top = most<G>(top);
  }
  const float from = !a.sigmoid ? a.normalize ? top : big : a.normalize ? fminf(top, 0.0f) : 0.0f;
  float z = a.normalize ? 0 : a.sigmoid ? 1 : z_all;
#pragma unroll
  for (int q = 0; q < KEEP; ++q) {
    const bool small = lc[q] <= 0;
    const float x = expf(!a.sigmoid || small ? lc[q] - from : -lc[q]);
    const float y = a.sigmoid && from != 0 ? expf(lc[q]) : x;  // of a sigmoid: exp(-|l|)
    w[q] = lc[q] == -INFINITY ? 0.0f : !a.sigmoid ? x : (small ? x : 1.0f) / (1.0f + y);
    if (a.normalize) z += w[q];
  }
  if (a.normalize) z = group_sum<G>(z);
#pragma unroll
  for (int q = 0; q < KEEP; ++q) w[q] = lc[q] == -INFINITY ? 0.0f : a.scale * (w[q] / z);
}

// ---------------------------------------------------------------- tokens
constexpr int32_t UNSURE = INT32_MIN;  // first choice of a token that is to be decided in double

__device__ inline void put(const RouteArgs& a, int64_t t, uint32_t j, int32_t e, float w, uint32_t* base) {
  a.experts[t * a.k + j] = e;
  a.weights[t * a.k + j] = w;
  atomicAdd(&base[e < 0 ? a.E : e], 1u);
}

// One workgroup's tokens [t0, t1): G lanes a token, C chunks a lane, up to P times 8
// choices. Counts the chosen experts in `base`; space: LDS of the lanes; sbias: each
// expert's bias in the chunks' order, 0 without. Says in `unsure` whether a token is.
template <class T, int G, int C, int P>
__device__ void choose_balanced(const RouteArgs& a, int64_t t0, int64_t t1, uint32_t* base, float* space,
                                const float* sbias, float near, uint32_t* unsure) {
  constexpr int W = G < 8 ? G : 8, EACH = 8 / W;  // lanes that keep choices, choices of a pass that each keeps
  constexpr float LOG2E = 1.44269504f;
  const uint32_t g = threadIdx.x % G;
  const Chunks ch = chunks_of(a.E, a.nodes);
  const bool whole = a.vector && ch.per % 8 == 0, scores = by_scores(a);
  float* own = space + threadIdx.x / G * (G * lane_space(C));
  uint32_t first[C], count[C];  // of the lane's chunks: first expert, how many
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t n = (i * G + g) / ch.chunks_per, in = (i * G + g) % ch.chunks_per * 8;
    count[i] = n < a.nodes ? min(ch.per - in, 8u) : 0;
    first[i] = n < a.nodes ? n * ch.per + in : 0;
  }
  // every lane of a wavefront stays in it: past the end, tokens are taken again and not written
  const int64_t rounds = (t1 - t0 + THREADS / G - 1) / (THREADS / G);
  for (int64_t round = 0; round < rounds; ++round) {
    const int64_t here = t0 + round * (THREADS / G) + threadIdx.x / G, t = min(here, t1 - 1);
    const T* row = (const T*)a.logits + t * a.ld;
    const uint8_t* mask = a.mask ? a.mask + t * a.mask_ld : nullptr;
    // nothing that is made from these is kept from token to token
#pragma unroll
    for (int i = 0; i < C; ++i) asm volatile("" : "+v"(first[i]), "+v"(count[i]));
    // the logits, -inf where the expert is not allowed; one chunk after the other
    // here and below: several at once would put more of them into scratch
    float c[8 * C];
    if (whole) {
      T l[8 * C];
#pragma unroll
      for (int i = 0; i < C; ++i) __builtin_memcpy(l + 8 * i, __builtin_assume_aligned(row + first[i], 16), 8 * sizeof(T));
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int r = 0; r < 8; ++r) c[8 * i + r] = count[i] ? (float)l[8 * i + r] : -INFINITY;
      if (mask) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          uint64_t m;
          __builtin_memcpy(&m, __builtin_assume_aligned(mask + first[i], 8), 8);
#pragma unroll
          for (int r = 0; r < 8; ++r) c[8 * i + r] = (m >> (8 * r) & 0xff) ? c[8 * i + r] : -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        uint8_t m[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t e = min(first[i] + r, a.E - 1);
          c[8 * i + r] = (float)row[e];
          m[r] = mask ? mask[e] : 1;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) c[8 * i + r] = r < (int)count[i] && m[r] ? c[8 * i + r] : -INFINITY;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    float big = -INFINITY, z = 0;  // of a softmax
    if (!a.sigmoid) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) {
        big = fmaxf(big, c[i]);
        nan |= c[i] != c[i];
      }
      big = most<G>(nan ? NAN : big);
      if (scores || !a.normalize) {
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) {
          z += c[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(LOG2E * (c[i] - big));
          if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
        }
        z = group_sum<G>(z);
      }
    }
    if (scores) {
      // exp through exp2 of a rounded product: off by |l| 2^-24 of itself, and
      // |x| exp(-|x|) < 1
      const float per_z = __builtin_amdgcn_rcpf(z);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float* b = sbias + 8 * (i * G + g);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float l = c[8 * i + r], x = __builtin_amdgcn_exp2f(a.sigmoid ? -LOG2E * l : LOG2E * (l - big));
          const float v = (a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + x) : x * per_z) + b[r];
          c[8 * i + r] = l == -INFINITY ? -INFINITY : v;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // -0 is 0, and a candidate's sign is its number's; a score is never -0
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) c[i] += 0.0f;
    }
    bool bad = false;  // a NaN or +inf, which the candidates cannot hold: decided in double, also where its bias is -inf
#pragma unroll
    for (int i = 0; i < 8 * C; ++i) bad |= !(c[i] < INFINITY);
    float clear = INFINITY;  // the least difference that decides something
    if (a.nodes > 1) {
      clear = keep_nodes<G, C>(a, ch.chunks_per, g, c, own);
      if (!scores) clear = INFINITY;  // logits are what they are, and ties are in order
    }

    int32_t e[P * EACH];  // -1 also of the passes that k does not reach
#pragma unroll
    for (int q = 0; q < P * EACH; ++q) e[q] = -1;
    double limit = INFINITY;  // the last pass's least
    float last = INFINITY;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (p * 8 >= (int)a.k) break;
      const bool ask = scores && (int)a.k == 8 * (p + 1);
      double top[8], rest = -INFINITY;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        double s[8];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          s[r] = candidate(c[8 * i + r], first[i] + r);
          if (p) s[r] = s[r] < limit ? s[r] : -INFINITY;
        }
        sort8(s);
        if (i == 0) {
#pragma unroll
          for (int r = 0; r < 8; ++r) top[r] = s[r];
        } else {
          merge8(top, s, rest, ask);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      merge_lanes<G>(top, rest, ask);
      __builtin_amdgcn_sched_barrier(0);
      limit = top[7];
      if (scores) {
        float before = last;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float v = (float)top[r];
          if (p * 8 + r <= (int)a.k) clear = fminf(clear, v == -INFINITY ? INFINITY : before - v);
          before = v;
        }
        last = before;
        if (ask && rest > -INFINITY) clear = fminf(clear, before - (float)rest);
      }
#pragma unroll
      for (int q = 0; q < EACH; ++q) {
        double v = top[q * W];
#pragma unroll
        for (int o = 1; o < W; ++o) v = g == o ? top[q * W + o] : v;
        e[p * EACH + q] = g < W && p * 8 + q * W + g < a.k ? expert_of(v) : -1;
      }
    }
    const bool sure = clear > near && !most_key<G>(bad);

    float lc[P * EACH], w[P * EACH];
#pragma unroll
    for (int q = 0; q < P * EACH; ++q) lc[q] = e[q] < 0 ? -INFINITY : (float)row[min((uint32_t)e[q], a.E - 1)];  // a NaN's number may be any
    weigh<G>(a, lc, big, z, w);
    if (here >= t1) continue;
    if (!sure) {
      if (g == 0) {
        a.experts[t * a.k] = UNSURE;
        *unsure = 1;
      }
      continue;
    }
#pragma unroll
    for (int q = 0; q < P * EACH; ++q) {
      const uint32_t j = q * W + g;
      if (g < W && j < a.k) put(a, t, j, e[q], w[q], base);
    }
  }
}

// Those of the tokens that are marked as unsure, each by a wavefront.
template <class T, int EACH>
__device__ void choose_exactly(const RouteArgs& a, int64_t t0, int64_t t1, uint32_t* base, double* d) {
  const uint32_t lane = threadIdx.x & 63, each = (a.E + 63) / 64;
  for (int64_t at = t0 + threadIdx.x / 64; at < t1; at += WAVES * 64) {  // neighbours to different wavefronts
    const int64_t look = at + (int64_t)lane * WAVES;
    uint64_t marked = __ballot(look < t1 && a.experts[look * a.k] == UNSURE);
    for (; marked; marked &= marked - 1) {
      const int64_t t = at + (int64_t)(__ffsll((unsigned long long)marked) - 1) * WAVES;
      float lc[1] = {-INFINITY}, w[1];
      const int32_t e[1] = {pick_exactly<T, EACH>(a, t, d, lc[0])};
      float big = -INFINITY, z = 0;
      const bool full = !a.normalize && !a.sigmoid;
      for (uint32_t i = 0; full && i < each; ++i) {
        const uint32_t x = lane * each + i;
        float l;
        if (x < a.E && allowed_at<T>(a, t, x, l)) big = l != l || big != big ? NAN : fmaxf(big, l);
      }
      if (full) big = most<64>(big);
      for (uint32_t i = 0; full && i < each; ++i) {
        const uint32_t x = lane * each + i;
        float l;
        if (x < a.E && allowed_at<T>(a, t, x, l)) z += expf(l - big);
      }
      weigh<64>(a, lc, big, group_sum<64>(z), w);
      if (lane < a.k) put(a, t, lane, e[0], w[0], base);
    }
  }
}

constexpr int each_of(int G, int C) { return G * C < 8 ? 1 : G * C / 8; }  // experts of a lane of 64
// LDS: the tokens' numbers in float, in whose place a wavefront of each 16 then has
// E doubles of one token, the biases, the counts.
template <int G, int C>
constexpr uint32_t space_bytes() {
  const uint32_t tokens = THREADS * lane_space(C) * 4, exact = WAVES * 64 * each_of(G, C) * 8;
  return tokens > exact ? tokens : exact;
}

template <class T, int G, int C, int P>
__global__ void __launch_bounds__(THREADS) balanced_kernel(RouteArgs a, int near_first) {
  constexpr int EACH = each_of(G, C);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* sbias = (float*)(lds + space_bytes<G, C>());
  uint32_t *base = (uint32_t*)(sbias + 8 * G * C), *counts = base + a.E + 1;
  __shared__ uint32_t unsure, size;
  const int64_t t0 = (int64_t)blockIdx.x * a.chunk, t1 = min(t0 + (int64_t)a.chunk, a.T);
  const Chunks ch = chunks_of(a.E, a.nodes);
  // the first logits are on their way while the biases are laid out
  float ahead = 0;
  if (t0 < t1) ahead = to_float(((const T*)a.logits)[min(t0 + threadIdx.x / G, t1 - 1) * a.ld + min(threadIdx.x % G * 8, a.E - 1)]);
  if (threadIdx.x == 0) unsure = size = 0;
  for (uint32_t i = threadIdx.x; i <= a.E; i += THREADS) base[i] = 0;
  __syncthreads();
  if (a.bias && threadIdx.x < 8 * G * C) {  // whole wavefronts
    const uint32_t n = threadIdx.x / (ch.chunks_per * 8), in = threadIdx.x % (ch.chunks_per * 8);
    const float b = n < a.nodes && in < ch.per ? a.bias[n * ch.per + in] : 0.0f;
    sbias[threadIdx.x] = b;
    const uint32_t most = most_key<G * C < 8 ? 8 * G * C : 64>(b == -INFINITY ? 0 : __float_as_uint(b) & 0x7fffffffu);
    if (threadIdx.x % 64 == 0) atomicMax(&size, most);
  } else if (threadIdx.x < 8 * G * C) {
    sbias[threadIdx.x] = 0;
  }
  __syncthreads();
  asm volatile("" ::"v"(ahead));
  // How near two decisive numbers may come. A sigmoid is off by up to 2^-22, a
  // softmax's share by 2^-22 and by its sum's error, up to 35 additions deep, 2^-18.8
  // of the difference between two shares; a sum with the bias by 2^-24 of its size; a
  // node's sum of two twice all that but the sum's and 2^-24 of its own, and so is a
  // difference. Near a bias that is NaN or infinite is everything, and the more the
  // larger it is: one of -1e4 or less that is to withhold an expert sends every token to
  // be decided in double (65536 tokens as above: 229 us for 64), one of -inf none.
  const float near = !by_scores(a) ? 0 : (a.sigmoid ? 0x1p-20f : 0x1p-18f) + 0x1p-21f * (1 + __uint_as_float(size));
  if (near_first) {
    choose_balanced<T, G, C, P>(a, t0, t1, base, (float*)lds, sbias, near, &unsure);
  } else {
    for (int64_t t = t0 + threadIdx.x; t < t1; t += THREADS) a.experts[t * a.k] = UNSURE;
    unsure = 1;
  }
  __threadfence_block();
  __syncthreads();
  if (unsure) choose_exactly<T, EACH>(a, t0, t1, base, (double*)lds + threadIdx.x / 64 * (64 * EACH));
  end_chunk(a, base, counts);
}

// With p the weights without their scale, P = sum p_i dw_i over the chosen:
//   normalized    softmax  w_j (dw_j - P)             sigmoid  w_j (1 - s_j) (dw_j - P), at the chosen
//   not           softmax  [chosen] w_e dw_e - scale s_e P     sigmoid  w_j (1 - s_j) dw_j
// A wavefront a token. 4099 tokens of 60 experts, 5 chosen, take 6.8 us; 65536 of 256,
// 8 chosen, in bf16 138 us for 70 MB (14 at a copy's rate): every lane reads the
// token's choices, weights and gradients again for each 64 experts.
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

template <class T, int G, int C>
hipError_t sized(const RouteArgs& a, int near_first, uint32_t chunks, hipStream_t s) {
  constexpr uint32_t more = space_bytes<G, C>() + 8 * G * C * 4, most = more + group_lds(8 * G * C);
  const uint32_t lds = more + group_lds(a.E);
  // further choices are further passes over the same numbers
  return a.k <= 8 ? launch<balanced_kernel<T, G, C, 1>, most>(chunks, THREADS, lds, s, a, near_first)
                  : launch<balanced_kernel<T, G, C, 4>, most>(chunks, THREADS, lds, s, a, near_first);
}

template <class T>
hipError_t typed(const RouteArgs& a, uint32_t chunks, hipStream_t s) {
  // chunks of 8 that nodes have for themselves; more than the 64 of 512 experts (nodes
  // of a few experts) are not laid out, and every token is decided in double (65536
  // tokens of 512 experts, 8 chosen: on 64 nodes 187 us, on 128 nodes 764, on 256 2260)
  const uint64_t n = (uint64_t)chunks_of(a.E, a.nodes).chunks_per * a.nodes;
  const int near_first = n <= 64;
  const uint64_t m = near_first ? n : (a.E + 7) / 8;
  if (m <= 1) return sized<T, 1, 1>(a, near_first, chunks, s);
  if (m <= 2) return sized<T, 2, 1>(a, near_first, chunks, s);
  if (m <= 4) return sized<T, 4, 1>(a, near_first, chunks, s);
  if (m <= 8) return sized<T, 8, 1>(a, near_first, chunks, s);
  if (m <= 16) return sized<T, 8, 2>(a, near_first, chunks, s);
  if (m <= 32) return sized<T, 8, 4>(a, near_first, chunks, s);
  return sized<T, 16, 4>(a, near_first, chunks, s);
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

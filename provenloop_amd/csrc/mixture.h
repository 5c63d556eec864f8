// Shared declarations of the plain (unencrypted) mixture-of-adapters operators:
//   route.hip     softmax gate with top-k, grouping of slots by expert
//   narrow.hip    matrix products of few output tiles
//   wide.hip      large ones, of ragged groups or with low-rank adapters added
//   grouped.hip   weight gradients of groups and of low-rank factors
//   mixture.hip   argument checks, workspaces and the C entry points
// They know nothing of a CKKS context: each call runs on the stream it is
// given, in memory its caller owns.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "mixture_rules.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

enum MixType { MIX_BF16 = 1, MIX_F16 = 2, MIX_F32 = 3 };

// A launch of `blocks` workgroups with `lds` bytes, MOST at most where they can
// be more than the 64 KiB that every kernel may have; or none if the workgroups
// are too many for one.
template <auto Kernel, uint32_t MOST = 65536, class... Args>
hipError_t launch(uint64_t blocks, uint32_t threads, uint32_t lds, hipStream_t s, const Args&... args) {
  if (!th::launchable(blocks, threads)) return hipErrorInvalidConfiguration;
  if constexpr (MOST > 65536) {
    const hipError_t ready = th::once_for<Kernel>(
        [] { return hipFuncSetAttribute((const void*)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, MOST); });
    if (ready != hipSuccess) return ready;
  }
  Kernel<<<(uint32_t)blocks, threads, lds, s>>>(args...);
  return hipGetLastError();
}

__device__ inline float to_float(bf16_t v) { return (float)v; }
__device__ inline float to_float(f16_t v) { return (float)v; }
__device__ inline float to_float(float v) { return v; }
template <class T>
__device__ inline T from_float(float v) { return (T)v; }

struct RouteArgs {
  const void* logits;  // T x E, row stride ld
  const uint8_t* mask;  // null, or T x E, row stride mask_ld (0: one row for all)
  int64_t T, ld, mask_ld;
  uint32_t E, k, chunk;
  int normalize, vector;  // vector: 8 logits, and their mask bytes, can be loaded at once
  float* weights;     // T x k
  int32_t* experts;   // T x k (input of launch_group)
  int32_t* order;     // T k
  int32_t* offsets;   // E + 1
  uint32_t* hist;     // chunks x (E + 1), with more than one chunk
};
hipError_t launch_route(MixType type, RouteArgs a, hipStream_t s);
hipError_t launch_group(RouteArgs a, hipStream_t s);
hipError_t launch_route_backward(MixType type, const RouteArgs& a, const float* dweights, void* dlogits,
                                 hipStream_t s);

// Rows of a matrix product. Without groups, row i of `x` gives row i of `y`.
// With them, slot order[i] (offsets[g] <= i < offsets[g + 1]) reads row
// slot / div of x, multiplies by matrix g of w and writes row slot of y; slots
// from offsets[E] on have no matrix, and their rows of y become zero.
struct MatArgs {
  const void* x;
  const void* w;
  void* y;
  const void* bias;   // null, or one value per output column
  const int32_t* order;
  const int32_t* offsets;
  int64_t ldx, ldw, ldwe, ldy;  // elements; ldwe: from matrix to matrix
  int64_t rows;                 // rows of y
  uint32_t n, k, E, div;        // outputs, contraction length
  int y_float;                  // y holds floats (a workspace)
  int aligned;                  // every row of x and w starts on 16 bytes and has a multiple of 8 values, or zeros up to one
  int scan;                     // no order or offsets: a slot's matrix is ids[slot], rows without one are not written
  // low-rank part: y_t += sum_j c_tj P[id_tj] u_tj over the token's choices
  // with P[e] = `p` + e * ldpe, n x r with row stride ldp
  const void* p;
  const float* u;          // slots x ru
  const int32_t* ids;      // T x kc
  const float* gate;       // null, or T x kc
  const float* scale;      // null, or per adapter
  int64_t ldp, ldpe;
  uint32_t r, ru, kc;
};
// w is n x k (transposed = 0: y = x w^T) or k x n (1: y = x w).
hipError_t launch_mat(MixType type, const MatArgs& a, int transposed, hipStream_t s);
hipError_t launch_narrow(MixType type, const MatArgs& a, int transposed, hipStream_t s);  // launch_mat's choice

// out[g] = sum over the slots s of group g of left[s] (outer) right[s / div]:
// n x k per group, with left row s of dy (n values), right row s / div of x (k).
struct OuterArgs {
  const void* dy;
  const void* x;
  void* out;  // E x n x k
  const int32_t* order;
  const int32_t* offsets;
  int64_t lddy, ldx, slots;
  uint32_t n, k, E, div;
  int aligned;
};
hipError_t launch_outer(MixType type, const OuterArgs& a, hipStream_t s);

// The low-rank gradients: out[e] = sum over the slots s of adapter e of
// c_s low[s] (outer) wide[s / div], low: slots x r floats (row stride ru).
// Partial sums of a few hundred slots each in `partial` (lowrank_spans x r x
// cols floats), added in slot order. transposed: out is E x cols x r.
struct LowOuterArgs {
  const float* low;
  const void* wide;
  void* out;
  float* partial;
  const int32_t* order;
  const int32_t* offsets;
  const float* gate;   // null, or per slot
  const float* scale;  // null, or per adapter
  int64_t ldwide, slots;
  uint32_t r, ru, cols, E, div, span;  // span: slots of one partial sum
  int aligned, transposed;
};
// out[s] = scale_e (u_s . v_s)
struct GateGradArgs {
  const float *u, *v;  // slots x ru
  const int32_t* ids;
  const float* scale;  // null, or per adapter
  float* out;
  int64_t slots;
  uint32_t r, ru, E;
};

// Two such sums with the same slots and ranks, and the gate's gradient, in one
// launch; what has no `out` is left out.
struct LowOuterPair {
  LowOuterArgs p[2];
  GateGradArgs gate;
  uint32_t blocks, gate_from;  // workgroups of the first, of both
};
hipError_t launch_low_outer(MixType type, const LowOuterPair& pair, hipStream_t s);

// out (E x cols x rows) = transposes of E matrices of rows x cols; two stacks in
// one launch, one without `out` is left out.
// out_ld: the row stride of `out`, zeros from `rows` on.
struct TransposeArgs {
  const void* in;
  void* out;
  int64_t ld, lde;
  uint32_t E, rows, cols, out_ld;
};
struct TransposePair {
  TransposeArgs p[2];
  uint32_t blocks;  // of the first
};
hipError_t launch_transpose(TransposePair pair, hipStream_t s);
// out = E matrices of rows x cols with rows of a multiple of 8 values, zeros
// beyond cols; up to three stacks in one launch, one without `out` is left out.
struct PadArgs {
  const void* in;
  void* out;
  int64_t ld, lde;
  uint32_t E, cols;
  int64_t rows;
};
struct PadSet {
  PadArgs p[3];
  uint32_t blocks[2];  // up to the second, up to the third
};
hipError_t launch_pad(PadSet set, hipStream_t s);
// out[t] = sum_j in[t k + j], rows of n floats
hipError_t launch_sum_choices(MixType type, const float* in, void* out, int64_t tokens, uint32_t k, uint32_t n,
                              hipStream_t s);
hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t s);

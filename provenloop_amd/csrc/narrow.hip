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
#include "narrow_kernel.h"

using namespace mix;

namespace {

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

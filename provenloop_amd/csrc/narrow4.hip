// Products of few output tiles with 4-bit weights: y = x w^T for decodes and
// small batches, as narrow.hip's of 16-bit ones. A line of a wavefront is 1 KiB of
// codes, contiguous in memory, the rows' values and up to 192 bytes of scales and
// zeros, all by asynchronous loads into the wavefront's ring; a lane then has its
// operands' codes in its own 16 bytes and makes their values in registers.
//
// A quarter of the weights' bytes leaves other things to wait for: x, which every
// column tile reads from L2 again (8 groups of 4 rows, 3584 -> 3584: 24.8 us for 53 MB
// with 16 columns a tile, 21.0 with 32), the 23 instructions a word, and for one row
// the chain of steps before the first load (1536 -> 1536 4.7 us in a series of
// launches, 3584 -> 3584 6.2). More lines in the rings change nothing (16 x 32 with
// 2, 3 and 4: 9.3, 9.3 and 9.4 us at 32 rows of 3584 -> 3584). So a decode has a quarter
// of the memory but not of the time (16 bits / 4, us a call in a series: one row of 1536
// -> 1536 with its adapter 8.1 / 8.2, 32 rows of 3584 -> 3584 15.1 / 13.9, 32 slots of 8
// experts 3584 -> 512 5.9 / 6.9 and 1536 -> 3584 17.8 / 11.6).
#include "narrow_kernel.h"

using namespace mix;

namespace {

template <class T, int MT, int NT, int WAVES, int S>
hipError_t run(const MatArgs& a, hipStream_t s) {
  constexpr uint32_t BM = 16 * MT, BN = 16 * NT, bytes = narrow_lds<MT, NT, WAVES, S, true>();
  uint64_t mtiles = th::ceil_div(a.rows, BM);
  if (a.offsets) mtiles = a.rows / BM + (uint64_t)min((int64_t)a.E + 1, a.rows);
  const uint64_t blocks = mtiles * th::ceil_div(a.n, BN);
  return a.u ? launch<narrow_kernel<T, MT, NT, WAVES, S, false, true, true, true>, bytes>(blocks, 64 * WAVES, bytes, s, a, 1u)
             : launch<narrow_kernel<T, MT, NT, WAVES, S, false, true, false, true>, bytes>(blocks, 64 * WAVES, bytes, s, a, 1u);
}

template <class T>
hipError_t typed(const MatArgs& a, hipStream_t s) {
  switch (th::four_tile(a.rows, a.n, a.offsets ? a.E : 1)) {
    case th::FOUR_16x16: return run<T, 1, 1, 8, 2>(a, s);
    case th::FOUR_16x32: return run<T, 1, 2, 8, 2>(a, s);
    case th::FOUR_32x32_ONCE: return run<T, 2, 2, 8, 2>(a, s);
    case th::FOUR_64x32_ONCE: return run<T, 4, 2, 8, 2>(a, s);
    case th::FOUR_32x32: return run<T, 2, 2, 4, 2>(a, s);
    default: return run<T, 4, 2, 4, 2>(a, s);
  }
}

}  // namespace

hipError_t launch_narrow4(MixType type, const MatArgs& a, hipStream_t s) {
  return type == MIX_BF16 ? typed<bf16_t>(a, s) : typed<f16_t>(a, s);
}

// Products of few output tiles with 4-bit weights: y = x w^T for decodes and
// small batches.
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
  switch (th::narrow_tile(a.rows, a.n, a.offsets ? a.E : 1)) {
    case th::NARROW_16x16: return run<T, 1, 1, 8, 2>(a, s);
    case th::NARROW_16x16_MANY: return run<T, 1, 1, 4, 2>(a, s);
    case th::NARROW_32x16: return run<T, 2, 1, 8, 2>(a, s);
    default: return run<T, 2, 2, 4, 2>(a, s);
  }
}

}  // namespace

hipError_t launch_narrow4(MixType type, const MatArgs& a, hipStream_t s) {
  return type == MIX_BF16 ? typed<bf16_t>(a, s) : typed<f16_t>(a, s);
}

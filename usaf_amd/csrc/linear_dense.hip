// linear_kernel on 16-bit weights: its tiles, and the rule that chooses one.
#include "linear_kernel.h"

namespace usaf {
namespace {
typedef LinShape<2, 4, 4, 2, false, true> D256x256;
typedef LinShape<2, 4, 2, 2, false> D128x256;
typedef LinShape<2, 4, 2, 1, false> D128x128;
typedef LinShape<2, 4, 1, 1, false> D64x128;
typedef LinShape<2, 2, 1, 1, false> D64x64;
typedef LinShape<1, 8, 1, 1, false> D32x256;
typedef LinShape<1, 2, 1, 1, false> D32x64;
}  // namespace

LinPlan plan_linear_dense(const LinArgs& g, int dt, bool gated) {
  LinPlan best;
  consider<D256x256>(best, g, dt, gated);
  consider<D128x256>(best, g, dt, gated);
  consider<D128x128>(best, g, dt, gated);
  consider<D64x128>(best, g, dt, gated);
  consider<D64x64>(best, g, dt, gated);
  consider<D32x256>(best, g, dt, gated);
  consider<D32x64>(best, g, dt, gated);
  return best;
}

void prepare_linear_dense() {
  D256x256::prepare();
  D128x256::prepare();
  D128x128::prepare();
  D64x128::prepare();
  D64x64::prepare();
  D32x256::prepare();
  D32x64::prepare();
}

}  // namespace usaf

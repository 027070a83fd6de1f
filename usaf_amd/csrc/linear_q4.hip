// linear_kernel on 4-bit weights: its tiles, and the rule that chooses one.
#include "linear_kernel.h"

namespace usaf {
namespace {
typedef LinShape<1, 8, 4, 1, true> Q128x256;
typedef LinShape<1, 4, 4, 1, true> Q128x128;
typedef LinShape<1, 4, 2, 1, true> Q64x128;
typedef LinShape<1, 2, 2, 1, true> Q64x64;
typedef LinShape<1, 8, 1, 1, true> Q32x256;
typedef LinShape<1, 2, 1, 1, true> Q32x64;
typedef LinShape<1, 1, 1, 1, true> Q32x32;
}  // namespace

LinPlan plan_linear_q4(const LinArgs& g, int dt, bool gated) {
  LinPlan best;
  consider<Q128x256>(best, g, dt, gated);
  consider<Q128x128>(best, g, dt, gated);
  consider<Q64x128>(best, g, dt, gated);
  consider<Q64x64>(best, g, dt, gated);
  consider<Q32x256>(best, g, dt, gated);
  consider<Q32x64>(best, g, dt, gated);
  consider<Q32x32>(best, g, dt, gated);
  return best;
}

void prepare_linear_q4() {
  Q128x256::prepare();
  Q128x128::prepare();
  Q64x128::prepare();
  Q64x64::prepare();
  Q32x256::prepare();
  Q32x64::prepare();
  Q32x32::prepare();
}

}  // namespace usaf

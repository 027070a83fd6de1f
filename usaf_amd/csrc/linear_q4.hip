// linear_kernel on 4-bit weights: its tiles, and the rule that chooses one: the shortest by a step's and a tile's end's times,
// measured tile by tile (10 ns, bf16; fp16 leaves out the last conversion and is up to 12 % faster).  Steps below 128 x 256 are of
// two, 32-row ones of up to eight blocks of the contraction.
#include "linear_kernel.h"

namespace usaf {
namespace {
typedef LinShape<1, 8, 4, 1, true, 120, 800> Q128x256;
typedef LinShape<1, 4, 4, 1, true, 123, 500> Q128x128;
typedef LinShape<1, 4, 2, 1, true, 93, 370> Q64x128;
typedef LinShape<1, 2, 2, 1, true, 97, 260> Q64x64;
typedef LinShape<1, 8, 1, 1, true, 80, 250> Q32x256;
typedef LinShape<1, 2, 1, 1, true, 81, 150> Q32x64;
typedef LinShape<1, 1, 1, 1, true, 79, 130> Q32x32;
}  // namespace

LinPlan plan_linear_q4(const LinArgs& g, bool gated) {
  LinPlan best;
  consider<Q128x256>(best, g, gated);
  consider<Q128x128>(best, g, gated);
  consider<Q64x128>(best, g, gated);
  consider<Q64x64>(best, g, gated);
  consider<Q32x256>(best, g, gated);
  consider<Q32x64>(best, g, gated);
  consider<Q32x32>(best, g, gated);
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

// linear_kernel on 16-bit weights: its tiles, and the rule that chooses one: the shortest by a step's and a tile's end's times,
// measured tile by tile (10 ns, bf16; the smallest tiles' steps are of two and four blocks of the contraction).
#include "linear_kernel.h"

namespace usaf {
namespace {
typedef LinShape<2, 4, 4, 2, false, 163, 700, true> D256x256;
typedef LinShape<2, 4, 2, 2, false, 90, 450> D128x256;
typedef LinShape<2, 4, 2, 1, false, 56, 350> D128x128;
typedef LinShape<2, 4, 1, 1, false, 33, 250> D64x128;
typedef LinShape<2, 2, 1, 1, false, 40, 250> D64x64;
typedef LinShape<1, 8, 1, 1, false, 41, 250> D32x256;
typedef LinShape<1, 2, 1, 1, false, 75, 200> D32x64;
}  // namespace

LinPlan plan_linear_dense(const LinArgs& g, bool gated) {
  LinPlan best;
  consider<D256x256>(best, g, gated);
  consider<D128x256>(best, g, gated);
  consider<D128x128>(best, g, gated);
  consider<D64x128>(best, g, gated);
  consider<D64x64>(best, g, gated);
  consider<D32x256>(best, g, gated);
  consider<D32x64>(best, g, gated);
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

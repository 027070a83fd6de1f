// linear_kernel on 16-bit operands that are stored with the contraction's index first, for gradients: dx = dy W, dW = dy^T x.
#include "linear_kernel.h"

namespace usaf {
namespace {
template <int TR>
struct Shapes {
  typedef LinTurned<2, 4, 4, 2, TR, 163, 700, true> T256x256;
  typedef LinTurned<2, 4, 2, 2, TR, 90, 450> T128x256;
  typedef LinTurned<2, 4, 2, 1, TR, 56, 350> T128x128;

  static LinPlan plan(const LinArgs& g) {
    LinPlan best;
    consider<T256x256>(best, g, false);
    consider<T128x256>(best, g, false);
    consider<T128x128>(best, g, false);
    return best;
  }
  static void prepare() {
    T256x256::prepare();
    T128x256::prepare();
    T128x128::prepare();
  }
};
}  // namespace

LinPlan plan_linear_turned(const LinArgs& g, bool both) { return both ? Shapes<2>::plan(g) : Shapes<1>::plan(g); }

void prepare_linear_turned() {
  Shapes<1>::prepare();
  Shapes<2>::prepare();
}

}  // namespace usaf

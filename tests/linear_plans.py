"""Sizes that the rules on tiles send to every kernel of the 4-bit product and the gated projection on 256 CUs."""
import ctypes

from usaf_amd import _native as N

ROWS, CODES, FEW, W_TURNED, TURNED = range(5)  # usaf_hip.h's USAF_PLAN_*

# call, rows, N (gated: I), K, checkpoint; kernels of the output, of dx and of a 16-bit weight's gradient: what they read, the
# tile's rows and weight rows, whether the contraction is taken in parts.  Columns and rows end inside tiles and, where a
# kernel takes them, inside 16-byte chunks; contractions run through the ring's stages several times.
CASES = [
    ("gated16", 1, 1377, 1148, "fp8", [(ROWS, 32, 256, False), (ROWS, 64, 128, True), (ROWS, 128, 128, False)]),
    ("gated16", 1, 9320, 2589, None, [(ROWS, 64, 128, False), (ROWS, 32, 256, True), (ROWS, 256, 256, False)]),
    ("gated16", 1, 18988, 1083, None, [(ROWS, 32, 256, False), (ROWS, 64, 128, True), (ROWS, 256, 256, False)]),
    ("gated16", 164, 544, 4904, None, [(ROWS, 32, 64, False), (W_TURNED, 128, 128, False), (ROWS, 128, 256, False)]),
    ("gated16", 165, 14304, 1032, None, [(ROWS, 128, 256, False), (W_TURNED, 128, 256, True), (ROWS, 256, 256, False)]),
    ("gated16", 167, 960, 144, "fp8", [(ROWS, 32, 256, False), (W_TURNED, 128, 128, True), (ROWS, 32, 64, False)]),
    ("gated16", 257, 700, 1000, "fp8", [(ROWS, 32, 256, False), (ROWS, 32, 64, False), (ROWS, 64, 128, False)]),
    ("gated16", 273, 512, 13976, "fp8", [(ROWS, 32, 256, False), (W_TURNED, 128, 256, False), (ROWS, 256, 256, False)]),
    ("gated16", 291, 8768, 5576, None, [(ROWS, 128, 256, False), (W_TURNED, 256, 256, True), (ROWS, 256, 256, False)]),
    ("gated16", 529, 65, 11874, "fp8", [(ROWS, 32, 256, False), (ROWS, 128, 256, False), (ROWS, 32, 256, False)]),
    ("gated16", 669, 12858, 336, "fp8", [(ROWS, 128, 256, False), (ROWS, 128, 256, True), (ROWS, 256, 256, False)]),
    ("gated16", 676, 1787, 522, None, [(ROWS, 128, 128, False), (ROWS, 32, 64, False), (ROWS, 128, 128, False)]),
    ("gated16", 680, 263, 705, None, [(ROWS, 32, 64, False), (ROWS, 64, 64, False), (ROWS, 32, 64, False)]),
    ("gated16", 973, 4590, 536, None, [(ROWS, 256, 256, False), (ROWS, 128, 128, True), (ROWS, 128, 256, False)]),
    ("gated16", 1024, 5988, 264, "fp8", [(ROWS, 256, 256, False), (ROWS, 64, 128, True), (TURNED, 128, 256, False)]),
    ("gated16", 1027, 4100, 1027, None, [(ROWS, 256, 256, False), (ROWS, 64, 128, False), (ROWS, 256, 256, False)]),
    ("gated16", 1088, 12212, 272, "fp8", [(ROWS, 256, 256, False), (ROWS, 128, 128, True), (TURNED, 256, 256, False)]),
    ("gated16", 1152, 68, 5960, "fp8", [(ROWS, 32, 256, False), (ROWS, 128, 256, False), (TURNED, 128, 128, False)]),
    ("gated16", 1864, 512, 4376, "fp8", [(ROWS, 32, 256, False), (W_TURNED, 256, 256, False), (ROWS, 128, 256, False)]),
    ("gated16", 2048, 8192, 2048, None, [(ROWS, 256, 256, False), (W_TURNED, 128, 256, True), (TURNED, 256, 256, False)]),
    ("gated16", 3712, 68, 776, None, [(ROWS, 64, 64, False), (ROWS, 128, 128, False), (TURNED, 128, 128, True)]),
    ("gated16", 4096, 68, 4232, None, [(ROWS, 64, 64, False), (ROWS, 128, 256, False), (TURNED, 128, 256, True)]),
    ("gated16", 9267, 11, 1026, None, [(ROWS, 64, 64, False), (ROWS, 256, 256, False), (ROWS, 32, 64, True)]),
    ("gated16", 16429, 8, 1044, "fp8", [(ROWS, 128, 256, False), (ROWS, 128, 256, False), (ROWS, 64, 128, True)]),
    ("gated16", 32194, 2886, 131, None, [(ROWS, 256, 256, False), (ROWS, 128, 256, False), (ROWS, 256, 256, True)]),
    ("gated16", 32832, 1548, 272, None, [(ROWS, 256, 256, False), (ROWS, 128, 128, False), (TURNED, 256, 256, True)]),
    ("gated16", 33516, 10, 1087, "fp8", [(ROWS, 256, 256, False), (ROWS, 256, 256, False), (ROWS, 64, 128, True)]),
    ("gated4", 1, 11, 1024, None, [(FEW, 16, 16, False), (ROWS, 32, 64, False)]),
    ("gated4", 34, 20, 1024, None, [(CODES, 32, 32, False), (ROWS, 32, 64, False)]),
    ("gated4", 34, 2970, 1024, "fp8", [(CODES, 32, 256, False), (ROWS, 64, 64, True)]),
    ("gated4", 35, 2420, 1024, None, [(CODES, 32, 64, False), (ROWS, 64, 64, True)]),
    ("gated4", 69, 5541, 1024, None, [(CODES, 64, 128, False), (ROWS, 64, 64, True)]),
    ("gated4", 75, 9991, 512, None, [(CODES, 32, 256, False), (ROWS, 64, 64, True)]),
    ("gated4", 97, 2119, 1024, None, [(CODES, 64, 64, False), (ROWS, 64, 64, True)]),
    ("gated4", 140, 14492, 1024, None, [(CODES, 128, 256, False), (ROWS, 64, 128, True)]),
    ("gated4", 145, 7294, 1024, "fp8", [(CODES, 128, 256, False), (ROWS, 64, 128, True)]),
    ("gated4", 1000, 2816, 2048, "fp8", [(ROWS, 128, 256, False), (ROWS, 64, 128, False)]),
    ("gated4", 11443, 71, 1024, None, [(CODES, 128, 128, False), (ROWS, 256, 256, False)]),
    ("q4", 1, 17, 1024, None, [(FEW, 16, 16, False), (ROWS, 32, 64, False)]),
    ("q4", 35, 4318, 1024, None, [(CODES, 32, 64, False), (ROWS, 64, 64, True)]),
    ("q4", 66, 696, 8960, None, [(CODES, 64, 64, True), (ROWS, 64, 128, False)]),
    ("q4", 67, 1144, 9728, None, [(CODES, 32, 32, True), (ROWS, 64, 128, False)]),
    ("q4", 67, 2098, 1024, None, [(CODES, 32, 32, False), (ROWS, 64, 64, True)]),
    ("q4", 68, 12494, 1024, None, [(CODES, 64, 128, False), (ROWS, 64, 64, True)]),
    ("q4", 73, 16723, 512, None, [(CODES, 32, 256, False), (ROWS, 64, 64, True)]),
    ("q4", 100, 4096, 14336, None, [(CODES, 128, 128, True), (ROWS, 64, 128, False)]),
    ("q4", 140, 1683, 8192, None, [(CODES, 128, 128, True), (ROWS, 64, 128, False)]),
    ("q4", 197, 8599, 1024, None, [(CODES, 128, 128, False), (ROWS, 64, 64, True)]),
    ("q4", 220, 18598, 1024, None, [(CODES, 128, 256, False), (ROWS, 64, 128, True)]),
    ("q4", 333, 1411, 1920, None, [(CODES, 32, 64, False), (ROWS, 64, 64, False)]),
    ("q4", 6148, 69, 1024, None, [(CODES, 64, 64, False), (ROWS, 128, 256, False)]),
]


def plans(call, m, n, k, checkpoint):
    """What the library says of them."""
    lib, plan = N.load(), (ctypes.c_int32 * 4)()

    def of(name, *args):
        assert getattr(lib, name)(*args, plan) == N.USAF_OK
        return (*plan[:3], plan[3] > 1)

    if call == "q4":
        return [of("usaf_hip_q4_linear_plan", m, n, k, back) for back in (0, 1)]
    four = call == "gated4"
    out = of("usaf_hip_gated_plan", m, n, k, four, 4 if checkpoint else 0, 0)
    if four:
        return [out, of("usaf_hip_gated_plan", m, n, k, 1, 1, 0)]
    return [out] + [of("usaf_hip_gated_plan", m, n, k, 0, 3, w) for w in (0, 1)]


def kernels(call, checkpoint, plans):
    """The kernels themselves: what leaves a tile belongs to them."""
    ends = "product" if call == "q4" else "blocks" if checkpoint else "activation"
    return {(ends, *plans[0])} | {("product", *p) for p in plans[1:]}

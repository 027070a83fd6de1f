// The product with a 4-bit weight for a few rows, as decoding calls it, and the gated projection of them:
//
//   out[m, n] = dt( sum_k x[m, k] W[n, k] )   or   dt( silu(g) u ),  g, u the sums of W's rows n and N + n
//   W[n, k] = dt(fp16(fp16(q s) + z)), the codec's value bit for bit
//
// A block takes tiles of 16 columns; its eight waves take a tile's pairs of groups (256 of the contraction, a
// 128-byte line of each weight row) in turn and join their sums in order.  Codes are loaded as they lie in memory, eight lanes
// a line, several steps ahead and across tile ends, and turned through the wave's own LDS into the matrix
// instruction's order: a lane has 32 codes of one weight row.  x sits in LDS in the order in which the codes come apart.
//
// Dequantizing: nibbles i and i + 4 of a word become a pair of fp16 by one and-or (1024 + q, or 64 + q for the upper
// nibble of a byte); q s is an fma with -1024 s (-64 s), which rounds the exact product once, where 1024 s is
// finite, and else (a scale of 60 or more, which no model has) a product.  6 1/4 vector instructions a pair in
// bf16, 3 1/4 in fp16, where the general form takes 8 and 5.
#include "linear.h"

namespace usaf {
namespace {

constexpr int QS_WAVES = 8, QS_THREADS = 64 * QS_WAVES;
constexpr int QS_COLS = 16, QS_ROWS = 16;
constexpr int QS_TURN = 2048;                     // bytes of a step's codes of 16 weight rows
constexpr int64_t QS_VALUES = 1 << 15;            // values of x that a block keeps

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, f32x4 c) {
  if constexpr (DT == USAF_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A group's scale and zero in both halves, with what the fma takes off.
struct Group {
  f16x2 s, z, lo, hi;
  bool plain;  // wave-uniform: 1024 s is finite in every lane
  __device__ __forceinline__ explicit Group(uint32_t p) {
    const f16 a = __builtin_bit_cast(f16, (uint16_t)p), b = __builtin_bit_cast(f16, (uint16_t)(p >> 16));
    s = f16x2{a, a};
    z = f16x2{b, b};
    lo = s * f16x2{(f16)-1024.f, (f16)-1024.f};
    hi = s * f16x2{(f16)-64.f, (f16)-64.f};
    plain = __ballot((p & 0x7FFFu) >= 0x5380u) == 0;  // 60
  }
};

// 8 codes of a word -> weights (0, 4), (1, 5), (2, 6), (3, 7).
template <int DT>
__device__ __forceinline__ u32x4 dq8_pairs(uint32_t w, const Group& g) {
#pragma clang fp contract(off)
  const uint32_t w8 = w >> 8;
  const uint32_t t[4] = {(w & 0x000F000Fu) | 0x64006400u, (w & 0x00F000F0u) | 0x54005400u, (w8 & 0x000F000Fu) | 0x64006400u,
                         (w8 & 0x00F000F0u) | 0x54005400u};
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 v = __builtin_bit_cast(f16x2, t[i]);
    f16x2 m;
    if (g.plain) {
      m = __builtin_elementwise_fma(v, g.s, i & 1 ? g.hi : g.lo);
    } else {
      const f16 off = i & 1 ? (f16)-64.f : (f16)-1024.f;
      m = (v + f16x2{off, off}) * g.s;
    }
    const uint32_t h = __builtin_bit_cast(uint32_t, m + g.z);
    o[i] = DT == USAF_BF16 ? h2_to_bf2(h) : h;
  }
  return o;
}

template <int DT, bool GATED>
__global__ __launch_bounds__(QS_THREADS) void q4_small_kernel(const uint16_t* __restrict__ x, int M, int K, int64_t ld,
                                                              const uint8_t* __restrict__ q, const uint32_t* __restrict__ sz,
                                                              int64_t N, uint16_t* __restrict__ out) {
  constexpr int HALVES = GATED ? 2 : 1, AHEAD = GATED ? 2 : 4;
  constexpr int PART = QS_WAVES * HALVES * QS_ROWS * QS_COLS;  // a tile's sums, twice
  extern __shared__ __align__(16) uint8_t lds[];
  float* const part = reinterpret_cast<float*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, quad = lane >> 4;
  uint8_t* const turn = lds + 2 * PART * 4 + wave * (HALVES * QS_TURN);
  uint8_t* const xs = lds + 2 * PART * 4 + QS_WAVES * HALVES * QS_TURN;
  const int row_bytes = 2 * K + 16;  // (rows 16 bytes apart in the banks)
  const int groups = K / 128, steps = (groups + 1) / 2, per = (steps + QS_WAVES - 1) / QS_WAVES;
  const int tiles = (int)((N + QS_COLS - 1) / QS_COLS);

  // the wave's next step to load: its line of the rows that the lane loads, and its row's scales
  int l_tile = blockIdx.x, l_i = 0;
  const uint8_t* l_q[HALVES][2];
  const uint32_t* l_s[HALVES];
  auto open = [&] {  // (past the last tile: that one again, which nobody reads)
    const int64_t n0 = (int64_t)(l_tile < tiles ? l_tile : tiles - 1) * QS_COLS;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t n = n0 + 8 * u + (lane >> 3);
        l_q[h][u] = q + ((n < N ? n : N - 1) + h * N) * (K / 2);
      }
      l_s[h] = sz + ((n0 + r < N ? n0 + r : N - 1) + h * N) * groups;
    }
  };
  u32x4 c[AHEAD][HALVES][2];
  uint32_t sc[AHEAD][HALVES][2];
  auto load = [&](int p) {
    const int step = wave + QS_WAVES * l_i, s = step < steps ? step : steps - 1;
    const int at = s * 128 + 16 * (lane & 7), most = K / 2 - 16;  // (of an odd last group: the row's end again)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
#pragma unroll
      for (int u = 0; u < 2; ++u) c[p][h][u] = *reinterpret_cast<const u32x4*>(l_q[h][u] + (at < most ? at : most));
      sc[p][h][0] = l_s[h][2 * s];
      sc[p][h][1] = l_s[h][2 * s + 1 < groups ? 2 * s + 1 : groups - 1];
    }
    if (++l_i == per) {
      l_i = 0;
      l_tile += gridDim.x;
      open();
    }
  };
  open();
#pragma unroll
  for (int p = 0; p < AHEAD; ++p) load(p);

  const int chunks = K / 8;
  for (int i = tid; i < M * chunks; i += QS_THREADS) {
    const int m = i / chunks, k = i - m * chunks;
    const uint4 v = *reinterpret_cast<const uint4*>(x + m * ld + 8 * k);
    *reinterpret_cast<uint4*>(xs + m * row_bytes + 16 * k) =
        uint4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
              __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
  }
  lds_barrier();

  const uint8_t* const x_row = xs + (r < M ? r : 0) * row_bytes + 64 * quad;
  f32x4 acc[HALVES];
  int tile = blockIdx.x, i = 0, buf = 0;
  while (tile < tiles) {
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      if (tile < tiles) {  // uniform over the block
        if (i == 0)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int s = wave + QS_WAVES * i;
        if (s < steps) {  // wave-uniform
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int row = 8 * u + (lane >> 3);
              *reinterpret_cast<u32x4*>(turn + h * QS_TURN + (lane & 4) * 256 + row * 64 + 16 * ((lane & 3) ^ (row >> 2))) = c[p][h][u];
            }
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (2 * s + g < groups) {  // wave-uniform
              u32x4 xf[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) xf[j] = *reinterpret_cast<const u32x4*>(x_row + (2 * s + g) * 256 + 16 * j);
#pragma unroll
              for (int h = 0; h < HALVES; ++h) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(turn + h * QS_TURN + g * 1024 + r * 64 + 16 * (quad ^ (r >> 2)));
                const Group gr(sc[p][h][g]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[h] = mfma16<DT>(xf[j], dq8_pairs<DT>(w[j], gr), acc[h]);
              }
            }
          }
        }
        load(p);
        if (++i == per) {  // the tile is done: the waves' sums, in order
          float* const mine = part + buf * PART;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[((wave * HALVES + h) * QS_ROWS + 4 * quad + j) * QS_COLS + r] = acc[h][j];
          lds_barrier();
          const int m = tid >> 4;
          const int64_t n = (int64_t)tile * QS_COLS + r;
          if (m < M && n < N) {  // M <= 16
            float sum[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              sum[h] = 0.f;
#pragma unroll
              for (int v = 0; v < QS_WAVES; ++v) sum[h] += mine[((v * HALVES + h) * QS_ROWS + m) * QS_COLS + r];
            }
            store_from_f32<DT>(out, m * N + n, GATED ? silu_fast(sum[0]) * sum[HALVES - 1] : sum[0]);
          }
          buf ^= 1;
          i = 0;
          tile += gridDim.x;
        }
      }
    }
  }
}

size_t lds_bytes(int M, int K, bool gated) {
  const int halves = gated ? 2 : 1;
  return (size_t)2 * QS_WAVES * halves * QS_ROWS * QS_COLS * 4 + QS_WAVES * halves * QS_TURN + (size_t)M * (2 * K + 16);
}

template <int DT, bool GATED>
void prepare_one() {
  static const bool done = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&q4_small_kernel<DT, GATED>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    (void)hipGetLastError();
    return true;
  }();
  (void)done;
}

template <int DT, bool GATED>
void launch(const LinArgs& g, hipStream_t st) {
  prepare_one<DT, GATED>();
  const int64_t tiles = (g.N + QS_COLS - 1) / QS_COLS, most = 2 * (int64_t)device_cu_count();
  q4_small_kernel<DT, GATED><<<(unsigned)(tiles < most ? tiles : most), QS_THREADS, lds_bytes((int)g.M, (int)g.K, GATED), st>>>(
      reinterpret_cast<const uint16_t*>(g.A), (int)g.M, (int)g.K, g.lda / 2, g.W, g.sz, g.N, g.out);
}

}  // namespace

bool q4_small_ok(int64_t M, int64_t K) { return M >= 1 && M <= QS_ROWS && M * K <= QS_VALUES; }

int q4_small(const LinArgs& g, int dt, bool gated, hipStream_t st) {
  if (dt == USAF_BF16) {
    if (gated) launch<USAF_BF16, true>(g, st);
    else launch<USAF_BF16, false>(g, st);
  } else {
    if (gated) launch<USAF_F16, true>(g, st);
    else launch<USAF_F16, false>(g, st);
  }
  return check_launch("q4_small");
}

void prepare_q4_small() {
  prepare_one<USAF_BF16, false>();
  prepare_one<USAF_BF16, true>();
  prepare_one<USAF_F16, false>();
  prepare_one<USAF_F16, true>();
}

}  // namespace usaf

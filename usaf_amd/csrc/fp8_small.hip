// The 8-bit product for a few rows, as decoding calls it: quantization and product in one launch.
//
//   out[m, n] = dt(sum over blocks of 128 of 2^(ea + ew) sum_k a[m, k] w[n, k]),   a, ea = Q(x)
//
// A block takes tiles of 16 columns of out and has all rows; its eight waves take a tile's
// groups of 128 of the contraction in turn and join their sums in order.  The first weights
// are on their way before the block quantizes the rows into LDS, all of them again in every
// block, which takes less than a launch of its own.  The weights stream through
// registers, a tile's behind the last one's sums; both sides' codes become bf16 values, exactly,
// for the 16-bit matrix instruction, whose sums keep fp32's precision.  The weights' way from
// memory bounds it, and for small ones the launch: 8.4 MB 6.1 us, 59 MB 16.6 us (3.5 TB/s), 268 MB 57.5 us
// (4.7 TB/s), one row each.
#include "fp8.h"

namespace usaf {
namespace {

constexpr int S_WAVES = 8, S_THREADS = 64 * S_WAVES;
constexpr int S_COLS = 16;
constexpr int S_AHEAD = 4;       // groups of a wave in flight
constexpr int S_PAD = 16;        // bytes behind a row of codes: 16 rows' words in different banks
// Rows times columns (whole blocks) at most: every block quantizes all rows, which a launch
// of its own is quicker at from some size on.  Measured (us, here / two launches, one behind the other in a
// graph): 1, 4, 8, 16 rows of 2,048 to 4,096 outputs 6.1 / 8.0, 6.9 / 8.3, 7.7 / 8.4, 10.1 / 8.5; 1, 4, 8 rows of 4,096 to
// 14,336 16.6 / 22.5, 17.8 / 22.8, 22.0 / 22.7; one of 14,336 to 4,096 18.1 / 26.5.  The host saves 4 us beside.
constexpr int64_t S_VALUES = 1 << 14;

__device__ __forceinline__ f32x4 mfma16_bf16(const u32x4 a, const u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int DT, int MT>
__global__ __launch_bounds__(S_THREADS) void fp8_small_kernel(const uint16_t* __restrict__ x, int M, int64_t K, int64_t ld,
                                                              bool vec, const uint8_t* __restrict__ w,
                                                              const uint8_t* __restrict__ ws, int64_t N,
                                                              uint16_t* __restrict__ out) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int PART = S_WAVES * MT * 16 * S_COLS;  // a tile's sums, twice
  float* const part = reinterpret_cast<float*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, quad = lane >> 4;
  const int ng = (int)((K + FP8_BLOCK - 1) / FP8_BLOCK), row = ng * FP8_BLOCK + S_PAD, blocks = M * ng;
  uint8_t* const s_q = lds + 2 * PART * 4;  // [M, row]
  uint8_t* const s_e = s_q + M * row;       // [M, ng]
  const int tiles = (int)((N + S_COLS - 1) / S_COLS);

  // the wave's next group to load: of tile l_tile, with the weight row's and scales' places there
  const uint8_t *l_w, *l_s;
  int l_tile = blockIdx.x, l_g = wave;
  auto open = [&] {  // (past the last tile: that one again, multiplied by nothing)
    const int64_t n0 = (int64_t)(l_tile < tiles ? l_tile : tiles - 1) * S_COLS;
    l_w = w + (n0 + r < N ? n0 + r : N - 1) * ((int64_t)ng * FP8_BLOCK) + 32 * quad;
    l_s = ws + n0 / FP8_BLOCK * ng;
  };
  u32x4 b0[S_AHEAD], b1[S_AHEAD];
  int be[S_AHEAD];
  auto load = [&](int p) {
    const int g = l_g < ng ? l_g : ng - 1;
    b0[p] = *reinterpret_cast<const u32x4*>(l_w + (int64_t)g * FP8_BLOCK);
    b1[p] = *reinterpret_cast<const u32x4*>(l_w + (int64_t)g * FP8_BLOCK + 16);
    be[p] = l_s[g];
    l_g += S_WAVES;
    if (l_g - wave >= ng) {  // as many groups for every wave: the tile's steps are ceil(ng / waves)
      l_g = wave;
      l_tile += gridDim.x;
      open();
    }
  };
  open();
#pragma unroll
  for (int p = 0; p < S_AHEAD; ++p) load(p);

  if (vec && K % FP8_BLOCK == 0) {
    constexpr int AT_ONCE = 4;
    for (int i0 = tid >> 4; i0 < blocks; i0 += AT_ONCE * S_THREADS / 16) {
      uint4 q[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int at = i0 + u * S_THREADS / 16, i = at < blocks ? at : blocks - 1, m = i / ng;
        q[u] = *reinterpret_cast<const uint4*>(x + m * ld + (i - m * ng) * FP8_BLOCK + 8 * r);
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * S_THREADS / 16, m = i / ng;
        if (i < blocks) {  // uniform over the 16 lanes
          float v[8];
          unpack8<DT>(q[u], v);
          store_block(v, r, s_q + m * row + (i - m * ng) * FP8_BLOCK + 8 * r, s_e + i);
        }
      }
    }
  } else {
    for (int i = tid >> 4; i < blocks; i += S_THREADS / 16) {
      const int m = i / ng, g = i - m * ng, c = g * FP8_BLOCK + 8 * r;
      const int64_t left = K - c;
      float v[8];
      load8<DT>(x + m * ld + c, vec, left > 8 ? 8 : left < 0 ? 0 : (int)left, v);
      store_block(v, r, s_q + m * row + c, s_e + i);
    }
  }
  lds_barrier();

  const int steps = (ng + S_WAVES - 1) / S_WAVES;
  f32x4 acc[MT];
  int tile = blockIdx.x, step = 0, buf = 0;
  while (tile < tiles) {
#pragma unroll
    for (int p = 0; p < S_AHEAD; ++p) {
      if (tile < tiles) {  // uniform over the block
        if (step == 0)
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int g = wave + S_WAVES * step;
        if (g < ng) {
          u32x4 bf[4];
          values16(b0[p], b1[p], be[p], bf);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int m = 16 * t + r < M ? 16 * t + r : M - 1;
            const u32x4* const a = reinterpret_cast<const u32x4*>(s_q + m * row + g * FP8_BLOCK + 32 * quad);
            u32x4 af[4];
            values16(a[0], a[1], s_e[m * ng + g], af);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t] = mfma16_bf16(af[j], bf[j], acc[t]);
          }
        }
        load(p);
        if (++step == steps) {  // the tile is done: the waves' sums, in order
          float* const mine = part + buf * PART;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[((wave * MT + t) * 16 + 4 * quad + j) * S_COLS + r] = acc[t][j];
          lds_barrier();
          const int m = tid >> 4;
          const int64_t n = (int64_t)tile * S_COLS + r;
          if (m < M && n < N) {  // M <= 32 rows, a thread an output
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < S_WAVES; ++v) sum += mine[(v * MT * 16 + m) * S_COLS + r];
            store_from_f32<DT>(out, m * N + n, sum);
          }
          buf ^= 1;
          step = 0;
          tile += gridDim.x;
        }
      }
    }
  }
}

template <int DT>
void launch(const uint16_t* x, int64_t M, int64_t K, int64_t ld, bool vec, const uint8_t* w, const uint8_t* ws, int64_t N,
            uint16_t* out, hipStream_t st) {
  const int64_t tiles = (N + S_COLS - 1) / S_COLS, most = 2 * (int64_t)device_cu_count();
  const unsigned blocks = (unsigned)(tiles < most ? tiles : most);
  const int64_t ng = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  // at most 53 KiB: two tiles' sums, the codes and the scale bytes
  const size_t lds = (size_t)(2 * S_WAVES * (M > 16 ? 32 : 16) * S_COLS * 4 + M * (ng * FP8_BLOCK + S_PAD + ng));
  if (M <= 16) fp8_small_kernel<DT, 1><<<blocks, S_THREADS, lds, st>>>(x, (int)M, K, ld, vec, w, ws, N, out);
  else fp8_small_kernel<DT, 2><<<blocks, S_THREADS, lds, st>>>(x, (int)M, K, ld, vec, w, ws, N, out);
}

}  // namespace

bool fp8_small_ok(int64_t M, int64_t K) {
  return M >= 1 && M <= 32 && K >= 1 && K <= S_VALUES && M * ((K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK) <= S_VALUES;
}

int fp8_small(const void* x, int dtype, int64_t M, int64_t K, int64_t ld, const uint8_t* w, const uint8_t* w_scale, int64_t N,
              void* out, hipStream_t st) {
  const bool vec = ((uintptr_t)x % 16) == 0 && ld % 8 == 0;
  const uint16_t* const p = reinterpret_cast<const uint16_t*>(x);
  if (dtype == USAF_BF16) launch<USAF_BF16>(p, M, K, ld, vec, w, w_scale, N, reinterpret_cast<uint16_t*>(out), st);
  else launch<USAF_F16>(p, M, K, ld, vec, w, w_scale, N, reinterpret_cast<uint16_t*>(out), st);
  return check_launch("fp8_linear/small");
}

}  // namespace usaf

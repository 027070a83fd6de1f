// The product with a 4-bit weight for a few rows, as decoding calls it, and the gated projection of them:
//
//   out[m, n] = dt( sum_k x[m, k] W[n, k] )   or   dt( silu(g) u ),  g, u the sums of W's rows n and N + n
//   W[n, k] = dt(fp16(fp16(q s) + z)), the codec's value bit for bit
//
// A block takes tiles of 16 columns; its eight waves (gated: four of them for gate, four for up) take a tile's pairs of groups
// (256 of the contraction, a 128-byte line of each weight row) in turn and join their sums in order.  Codes come by LDS DMA,
// whole lines, into a ring of the wave's own, several steps ahead and across tile ends, and leave it in the matrix
// instruction's order: a lane has 32 codes of one weight row.  x sits in LDS in the order in which the codes come apart.
//
// Dequantizing: nibbles i and i + 4 of a word become a pair of fp16 by one and-or (1024 + q, or 64 + q for the upper
// nibble of a byte); q s is an fma with -1024 s (-64 s), which rounds the exact product once, where 1024 s is
// finite, and else (a scale of 60 or more, which no model has) a product.  6 1/4 vector instructions a pair in
// bf16, 3 1/4 in fp16, where the general form takes 8 and 5.
//
// Vector instructions, of which the dequantization is 44 (8 rows, fp16) to 74 % (gated, bf16), fill 54 to 64 % of a SIMD's
// cycles; waves wait for codes or LDS 30 to 38 % of their time, for an issue slot 30 to 39 %: neither the stream of codes nor
// the instructions bound it alone (cold weights, one launch behind the other in a graph, us, bf16 / fp16): 1 x 4,096 x
// 4,096 5.8, 1 x 14,336 x 4,096 13.5 / 11.0 (2.3 / 2.8 TB/s), 8 x 32,000 x 2,048 15.5 / 13.0, gated 1 x 28,672 x 4,096
// 22.6 / 17.1 (2.8 / 3.7 TB/s); 1 x 4,096 x 2,048 4.3: a start, one trip to memory, the sums' meeting.
#include "dma.h"
#include "linear.h"

namespace usaf {
namespace {

constexpr int QS_WAVES = 8, QS_THREADS = 64 * QS_WAVES;
constexpr int QS_COLS = 16, QS_ROWS = 16;
constexpr int QS_STEP = 2048 + 256;               // bytes of a wave's step: 16 weight rows' lines of codes, their scales twice
constexpr int QS_DEPTH = 2;                       // steps of a wave in its ring
// Values of x that a block keeps at most, and for how many a CU has room for a second block.  Measured (us, here / linear_kernel's
// best tile, bf16, one behind the other in a graph): 1, 8, 16 rows of 2,048 to 4,096 outputs 4.3 / 7.4, 5.0 / 7.5, 5.8 / 7.5; 4, 12 of
// 4,096 to 4,096 6.2 / 9.6, 7.5 / 9.6; 3 of 14,336 to 4,096 13.0 / 18.3; with many columns and one block a CU 8 of 4,096 to
// 14,336 17.7 / 17.7, 12 19.2 / 17.4, 16 of 2,048 to 14,336 12.7 / 10.9.
constexpr int64_t QS_VALUES = 3 << 14, QS_TWO = 1 << 14, QS_MANY = 8192;

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, f32x4 c) {
  if constexpr (DT == USAF_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The masks in scalar and the exponents in vector registers, as one and-or takes them.
struct Nibbles {
  uint32_t low = 0x000F000Fu, high = 0x00F000F0u, e_low = 0x64006400u, e_high = 0x54005400u;
  __device__ __forceinline__ Nibbles() {
    asm volatile("" : "+s"(low), "+s"(high));
    asm volatile("" : "+v"(e_low), "+v"(e_high));
  }
};

// 8 codes of a word -> weights (0, 4), (1, 5), (2, 6), (3, 7) of a group with scale s and zero z; FMA: 1024 s is finite, and
// lo, hi are -1024 s, -64 s.
template <int DT, bool FMA>
__device__ __forceinline__ u32x4 dq8_pairs(uint32_t w, const Nibbles& n, f16x2 s, f16x2 z, f16x2 lo, f16x2 hi) {
#pragma clang fp contract(off)
  const uint32_t w8 = w >> 8;
  const uint32_t t[4] = {(w & n.low) | n.e_low, (w & n.high) | n.e_high, (w8 & n.low) | n.e_low, (w8 & n.high) | n.e_high};
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 v = __builtin_bit_cast(f16x2, t[i]);
    f16x2 m;
    if constexpr (FMA) {
      m = __builtin_elementwise_fma(v, s, i & 1 ? hi : lo);
    } else {
      const f16 off = i & 1 ? (f16)-64.f : (f16)-1024.f;
      m = (v + f16x2{off, off}) * s;
    }
    const uint32_t h = __builtin_bit_cast(uint32_t, m + z);
    o[i] = DT == USAF_BF16 ? h2_to_bf2(h) : h;
  }
  return o;
}

template <int DT, bool GATED>
__global__ __launch_bounds__(QS_THREADS) void q4_small_kernel(const uint16_t* __restrict__ x, int M, int K, int64_t ld,
                                                              const uint8_t* __restrict__ q, const uint32_t* __restrict__ sz,
                                                              int64_t N, uint16_t* __restrict__ out) {
  constexpr int WAVES = QS_WAVES / (GATED ? 2 : 1);  // waves of a tile's rows: of gate and of up half of the block's each
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, quad = lane >> 4;
  const int half = wave / WAVES, kw = wave % WAVES;
  uint8_t* const ring = lds + wave * (QS_DEPTH * QS_STEP);
  const uint32_t ring_lds = (uint32_t)(uintptr_t)(lds_void_ptr)ring;
  float* const part = reinterpret_cast<float*>(lds + QS_WAVES * QS_DEPTH * QS_STEP);  // [2, waves, M, 16]
  uint8_t* const xs = reinterpret_cast<uint8_t*>(part + 2 * QS_WAVES * M * QS_COLS);
  const int groups = K / 128, steps = (groups + 1) / 2, per = (steps + WAVES - 1) / WAVES;
  const int tiles = (int)((N + QS_COLS - 1) / QS_COLS);
  const Nibbles nib;
  int blocks = gridDim.x;
  asm volatile("" : "+s"(blocks));  // (held: else it is fetched again at every tile)

  // ---- the wave's loads: uniform places of the tile's first row, 32-bit lane offsets (rows past the last: that one again).
  //      Lane l of code instruction u has chunk l % 8 of row 8 u + l / 8; lanes of the scales' a row's two words
  const int row_q = K / 2;
  const int64_t row_s = 4 * (GATED ? 2 * N : N);  // bytes of a group's words
  const uint8_t *l_q, *l_s;
  uint32_t o_q[2], o_s;
  int l_tile = blockIdx.x, l_i = 0, l_slot = 0;
  auto open = [&] {  // (past the last tile: that one again, which nobody reads)
    const int64_t n0 = (int64_t)(l_tile < tiles ? l_tile : tiles - 1) * QS_COLS;
    const int left = N - 1 - n0 < QS_COLS ? (int)(N - 1 - n0) : QS_COLS;
    l_q = q + (n0 + half * N) * row_q;
    l_s = reinterpret_cast<const uint8_t*>(sz + n0 + half * N);
    const uint32_t most_q = (uint32_t)(left * row_q);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 8 * u + (lane >> 3);
      const uint32_t o = (uint32_t)(row * row_q);
      o_q[u] = (o < most_q ? o : most_q) + 16 * ((lane & 7) ^ g_swz(row));
    }
    o_s = 4 * (uint32_t)(r < left ? r : left);
  };
  auto load = [&] {
    const int step = kw + WAVES * l_i, s = step < steps ? step : steps - 1;
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(ring_lds + l_slot * QS_STEP));
    // an odd last group has half a line: its upper chunks are the lower ones again, the second scale is the first
    const bool odd = 2 * s + 1 == groups;
    const uint8_t* const at_q = uniform(l_q + s * 128);
    const uint8_t* const at_s = uniform(l_s + 2 * s * row_s);
#pragma unroll
    for (int u = 0; u < 2; ++u) g_dma16(at_q, odd ? o_q[u] - 16 * (((lane & 7) ^ g_swz(8 * u + (lane >> 3))) & 4) : o_q[u], to + 1024 * u);
    g_dma4(at_s, o_s + (!odd && (quad & 1) ? (uint32_t)row_s : 0), to + 2048);
    l_slot = l_slot + 1 == QS_DEPTH ? 0 : l_slot + 1;
    if (++l_i == per) {
      l_i = 0;
      l_tile += blocks;
      open();
    }
  };
  // ---- x: by DMA too, ahead of the weights, and turned in place: chunk c of row m at c ^ (m & 15), which spreads 16 rows'
  //      chunks over the banks
  const int chunks = K / 8, all = M * chunks;
  for (int i = wave; i < (all + 63) / 64; i += QS_WAVES) {
    const int d = 64 * i + lane < all ? 64 * i + lane : all - 1, m = d / chunks, c = (d - m * chunks) ^ (m & 15);
    g_dma16(x, (uint32_t)((m * ld + 8 * c) * 2),
            (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(uintptr_t)(lds_void_ptr)xs + 1024 * i)));
  }
  open();
  for (int p = 0; p < QS_DEPTH; ++p) load();
  wait_vmcnt<3 * QS_DEPTH>();
  lds_barrier();
  for (int d = tid; d < all; d += QS_THREADS) {
    uint4* const at = reinterpret_cast<uint4*>(xs) + d;
    const uint4 v = *at;
    *at = uint4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
  }
  lds_barrier();

  const int x_m = r < M ? r : 0;
  const uint8_t* const x_row = xs + x_m * (2 * K);
  uint32_t x_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) x_at[j] = 16 * ((4 * quad + j) ^ x_m);
  int slot = 0, buf = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += blocks) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < per; ++i) {
      wait_vmcnt<3 * (QS_DEPTH - 1)>();  // the step's three DMAs have landed
      const uint8_t* const at = ring + slot * QS_STEP;
      u32x4 w[2];
      uint32_t words[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        w[g] = *reinterpret_cast<const u32x4*>(at + r * 128 + 16 * ((4 * g + quad) ^ g_swz(r)));
        words[g] = *reinterpret_cast<const uint32_t*>(at + 2048 + 4 * (16 * g + r));
      }
      const int s = kw + WAVES * i;
      u32x4 xf[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j)  // (past the last group: that one again)
          xf[g][j] = *reinterpret_cast<const u32x4*>(x_row + (2 * s + g < groups ? 2 * s + g : groups - 1) * 256 + x_at[j]);
      asm volatile("s_waitcnt lgkmcnt(8)" : "+v"(w[0]), "+v"(w[1]), "+v"(words[0]), "+v"(words[1])::"memory");
      load();  // the slot has been read
      slot = slot + 1 == QS_DEPTH ? 0 : slot + 1;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (2 * s + g < groups) {  // wave-uniform
          const f16 a = __builtin_bit_cast(f16, (uint16_t)words[g]), b = __builtin_bit_cast(f16, (uint16_t)(words[g] >> 16));
          const f16x2 s2 = {a, a}, z2 = {b, b}, k1024 = {(f16)-1024.f, (f16)-1024.f}, k64 = {(f16)-64.f, (f16)-64.f};
          if (__ballot((words[g] & 0x7FFFu) >= 0x5380u) == 0) {  // every lane's |s| is below 60
            const f16x2 lo = s2 * k1024, hi = s2 * k64;
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = mfma16<DT>(xf[g][j], dq8_pairs<DT, true>(w[g][j], nib, s2, z2, lo, hi), acc);
          } else {
            asm volatile("");  // (both ways and a choice between their results would take longer)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = mfma16<DT>(xf[g][j], dq8_pairs<DT, false>(w[g][j], nib, s2, z2, s2, s2), acc);
          }
        }
      }
    }
    // the waves' sums, in order
    float* const mine = part + buf * (QS_WAVES * M * QS_COLS);
    buf ^= 1;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * quad + j < M) mine[(wave * M + 4 * quad + j) * QS_COLS + r] = acc[j];
    lds_barrier();
    const int m = tid >> 4;
    const int64_t n = (int64_t)tile * QS_COLS + r;
    if (m < M && n < N) {  // M <= 16
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int v = 0; v < QS_WAVES; ++v) sum[v / WAVES] += mine[(v * M + m) * QS_COLS + r];
      store_from_f32<DT>(out, m * N + n, GATED ? silu_fast(sum[0]) * sum[1] : sum[0]);
    }
  }
  wait_vmcnt<0>();  // no DMA lands in LDS that is someone else's by then
}

size_t lds_bytes(int M, int K) {
  return (size_t)QS_WAVES * QS_DEPTH * QS_STEP + (size_t)2 * QS_WAVES * M * QS_COLS * 4 + ((size_t)M * K * 2 + 1023) / 1024 * 1024;
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
  q4_small_kernel<DT, GATED><<<(unsigned)(tiles < most ? tiles : most), QS_THREADS, lds_bytes((int)g.M, (int)g.K), st>>>(
      reinterpret_cast<const uint16_t*>(g.A), (int)g.M, (int)g.K, g.lda / 2, g.W, g.sz, g.N, g.out);
}

}  // namespace

bool q4_small_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 1 && M <= QS_ROWS && M * K <= (N <= QS_MANY ? QS_VALUES : QS_TWO);
}

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

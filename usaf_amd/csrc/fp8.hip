// The 8-bit block format: codec, and the elementwise steps between its products.
//
// Codes are e4m3 (OCP, "fn"), every block of 128 (activations: 1 x 128 along the
// row; weights: 128 x 128) has one scale 2^e, held as the E8M0 byte e + 127:
//   e = the smallest integer with max|x| 2^-e <= 448,   code = RNE_e4m3(x 2^-e).
// A power of two, because the matrix instruction applies E8M0 scales itself
// (v_mfma_scale_*): the products need no vector instruction for them.  It costs no
// precision against a scale of max / 448: e4m3 is a floating format, the relative
// step of a normal code is the same wherever the block sits, and x 2^-e is exact.
// e is kept within [-120, 120], so that the inverse scale is a normal number:
// blocks below 2^-112 lose their low codes, which no model's values reach.
// A value that is not finite becomes the NaN code 0x7F and takes no part in max|x|:
// its row of a product is NaN, as the row's 16-bit product would be (inf or NaN).
// Values above 248 2^120 = 3.30e38, the last 3 % of bf16's range, round to 2^128, which no product can hold:
// they count as infinite there.
#include "fp8.h"

namespace usaf {
namespace {

constexpr int FB = FP8_BLOCK;

// Rows of 16-bit values -> codes [rows, kp] and scale bytes [rows, sp].  16 lanes a
// block; columns past the row's end are zeros.  n_rows (device, may be null): rows
// from there on are left as they are.
template <int DT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const uint16_t* __restrict__ x, int64_t rows, int64_t cols,
                                                       int64_t ld, bool vec, int nkb, int64_t kp, int sp,
                                                       const int32_t* __restrict__ n_rows, uint8_t* __restrict__ q,
                                                       uint8_t* __restrict__ s) {
  const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane16 = threadIdx.x & 15;
  const int64_t row = i / nkb;
  const int kb = (int)(i - row * nkb);
  if (row >= rows || (n_rows && row >= *n_rows)) return;  // uniform over the 16 lanes
  const int64_t c = (int64_t)kb * FB + 8 * lane16;
  const int64_t left = cols - c;
  float v[8];
  load8<DT>(x + row * ld + c, vec, left > 8 ? 8 : left < 0 ? 0 : (int)left, v);
  store_block(v, lane16, q + row * kp + c, s + row * sp + kb);
}

// The same for aligned rows of a multiple of 512 columns: a wave has four blocks of a row, whose
// scale bytes are one word, R_AHEAD times, whose loads go out together.  Bytes bound it: 8,192 x 4,096, 101 MB,
// 27 us, 3.7 TB/s (one block for each 16 lanes and a byte store for each scale: 29).
constexpr int R_AHEAD = 4;
template <int DT>
__global__ __launch_bounds__(256) void fp8_rows4_kernel(const uint16_t* __restrict__ x, int64_t rows, int64_t ld, int nkw,
                                                        const int32_t* __restrict__ n_rows, uint8_t* __restrict__ q,
                                                        uint8_t* __restrict__ s) {
  const int lane = threadIdx.x & 63;
  const int64_t end = n_rows && *n_rows < rows ? *n_rows : rows;
  int64_t at = (int64_t)blockIdx.x * (4 * R_AHEAD) + (threadIdx.x >> 6), row[R_AHEAD];  // the wave's words
  int kw[R_AHEAD];
  row[0] = at / nkw;
  kw[0] = (int)(at - row[0] * nkw);
  uint4 v[R_AHEAD];
#pragma unroll
  for (int i = 0; i < R_AHEAD; ++i) {
    if (i) {  // four words on
      row[i] = row[i - 1];
      kw[i] = kw[i - 1] + 4;
      while (kw[i] >= nkw) {
        kw[i] -= nkw;
        ++row[i];
      }
    }
    v[i] = *reinterpret_cast<const uint4*>(x + (row[i] < rows ? row[i] : rows - 1) * ld + kw[i] * 512 + 8 * lane);
  }
#pragma unroll
  for (int i = 0; i < R_AHEAD; ++i) {
    if (row[i] >= end) return;  // wave-uniform
    float f[8], m = 0.f;
    unpack8<DT>(v[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(f[j]));
    const int e = e8m0_of(max16(m));
    const float inv = inv_scale(e), a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
    *reinterpret_cast<uint2*>(q + (row[i] * nkw + kw[i]) * 512 + 8 * lane) = uint2{to_codes(a, inv), to_codes(b, inv)};
    const uint32_t word = (uint32_t)__builtin_amdgcn_readlane(e, 0) | (uint32_t)__builtin_amdgcn_readlane(e, 16) << 8 |
                          (uint32_t)__builtin_amdgcn_readlane(e, 32) << 16 | (uint32_t)__builtin_amdgcn_readlane(e, 48) << 24;
    if (lane == 0) *reinterpret_cast<uint32_t*>(s + (row[i] * nkw + kw[i]) * 4) = word;
  }
}

// Weight [E, R, C] -> codes [E, R, kp], scale bytes [E, ceil(R / 128), kp / 128].
// A block of threads takes one 128 x 128 block: 16 lanes a row, 16 rows at a time.
template <int DT>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const void* __restrict__ w, int64_t R, int64_t C, int64_t kp,
                                                         uint8_t* __restrict__ q, uint8_t* __restrict__ s) {
  __shared__ float s_max[4];
  const int64_t nkb = kp / FB, nrb = (R + FB - 1) / FB;
  const int64_t kb = blockIdx.x % nkb, rb = blockIdx.x / nkb % nrb, e = blockIdx.x / nkb / nrb;
  const int64_t c = kb * FB + 8 * (threadIdx.x & 15);
  float v[8][8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = rb * FB + 16 * i + (threadIdx.x >> 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = r < R && c + j < C ? load_as_f32<DT>(w, (e * R + r) * C + c + j) : 0.f;
      m = fmaxf(m, finite_abs(v[i][j]));
    }
  }
  m = max16(m);
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  __syncthreads();
  const int eb = e8m0_of(fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3])));
  const float inv = inv_scale(eb);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = rb * FB + 16 * i + (threadIdx.x >> 4);
    const float a[4] = {v[i][0], v[i][1], v[i][2], v[i][3]}, b[4] = {v[i][4], v[i][5], v[i][6], v[i][7]};
    if (r < R) *reinterpret_cast<uint2*>(q + (e * R + r) * kp + c) = uint2{to_codes(a, inv), to_codes(b, inv)};
  }
  if (threadIdx.x == 0) s[(e * nrb + rb) * nkb + kb] = (uint8_t)eb;
}

template <int DT>
__global__ __launch_bounds__(256) void fp8_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                          int64_t R, int64_t C, int64_t kp, int64_t total,
                                                          void* __restrict__ out) {
  const int64_t nkb = kp / FB, nrb = (R + FB - 1) / FB;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / C, c = i - row * C, e = row / R, r = row - e * R;
    const float v = __builtin_amdgcn_cvt_f32_fp8((int)q[row * kp + c], 0);
    store_from_f32<DT>(out, i, ldexpf(v, (int)s[(e * nrb + r / FB) * nkb + c / FB] - 127));
  }
}

// [R, kp] codes -> [C, rp] codes of the transpose, rows past R as zeros; with the
// scale bytes transposed.  One 128 x 128 block per thread block, through LDS: 402 MB read and written
// in 200 us, 4.0 TB/s, once for a weight.
__global__ __launch_bounds__(256) void fp8_transpose_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                            int64_t R, int64_t C, int64_t kp, int64_t rp,
                                                            uint8_t* __restrict__ qt, uint8_t* __restrict__ st) {
  __shared__ uint32_t tile[FB * 33];  // row of 128 codes and one word of padding
  const int64_t nkb = kp / FB, nrb = rp / FB;
  const int64_t kb = blockIdx.x % nkb, rb = blockIdx.x / nkb % nrb, e = blockIdx.x / nkb / nrb;
  for (int i = threadIdx.x; i < FB * 32; i += 256) {
    const int r = i >> 5, w = i & 31;
    const int64_t row = rb * FB + r;
    tile[r * 33 + w] = row < R ? *reinterpret_cast<const uint32_t*>(q + (e * R + row) * kp + kb * FB + 4 * w) : 0u;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < FB * 32; i += 256) {
    const int c = i >> 5, w = i & 31;  // column c of the block, its rows 4 w .. 4 w + 3
    if (kb * FB + c >= C) continue;
    uint32_t o = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) o |= ((tile[(4 * w + j) * 33 + (c >> 2)] >> (8 * (c & 3))) & 0xFFu) << (8 * j);
    *reinterpret_cast<uint32_t*>(qt + (e * C + kb * FB + c) * rp + rb * FB + 4 * w) = o;
  }
  if (threadIdx.x == 0) st[(e * nkb + kb) * nrb + rb] = s[(e * nrb + rb) * nkb + kb];
}

// gu [S, 2I] -> act = dt(dt(silu(gate)) up) [S, I] (null: not stored), its codes and scale
// bytes, for the slots in use (offsets[E]).  16 lanes a block of 128 columns.  Bytes bound it:
// 32,768 slots of 768, 126 MB, 26 us, 4.8 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void fp8_swiglu_kernel(const uint16_t* __restrict__ gu, int64_t S, int64_t I,
                                                         const int32_t* __restrict__ n_slots, uint16_t* __restrict__ act,
                                                         uint8_t* __restrict__ q, uint8_t* __restrict__ s, int sp) {
  const int nkb = (int)(I / FB);
  const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane16 = threadIdx.x & 15;
  const int64_t m = i / nkb;
  const int kb = (int)(i - m * nkb);
  if (m >= S || m >= *n_slots) return;
  const int64_t c = (int64_t)kb * FB + 8 * lane16;
  float g[8], u[8], a[8];
  load8<DT>(gu + m * 2 * I + c, true, 8, g);
  load8<DT>(gu + m * 2 * I + I + c, true, 8, u);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x2 sg = unpack2<DT>(pack2<DT>(silu_fast(g[2 * j]), silu_fast(g[2 * j + 1])));
    w[j] = pack2<DT>(sg.x * u[2 * j], sg.y * u[2 * j + 1]);
    const f32x2 v = unpack2<DT>(w[j]);
    a[2 * j] = v.x;
    a[2 * j + 1] = v.y;
  }
  if (act) *reinterpret_cast<uint4*>(act + m * I + c) = make_uint4(w[0], w[1], w[2], w[3]);
  store_block(a, lane16, q + m * I + c, s + m * sp + kb);
}

// gu, dact -> dgu [S, 2I] with the roundings of the layer's other grad-input kernels
// (null: not stored), its codes and scale bytes.  Bytes bound it: 32,768 slots of 768, 202 MB, 42
// us, 4.8 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void fp8_swiglu_bwd_kernel(const uint16_t* __restrict__ gu,
                                                             const uint16_t* __restrict__ dact, int64_t S, int64_t I,
                                                             const int32_t* __restrict__ n_slots,
                                                             uint16_t* __restrict__ dgu, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ s, int sp) {
#pragma clang fp contract(off)
  const int nkb = (int)(I / FB);
  const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane16 = threadIdx.x & 15;
  const int64_t m = i / nkb;
  const int kb = (int)(i - m * nkb);
  if (m >= S || m >= *n_slots) return;
  const int64_t c = (int64_t)kb * FB + 8 * lane16;
  float g[8], u[8], d[8], dg[8], du[8];
  load8<DT>(gu + m * 2 * I + c, true, 8, g);
  load8<DT>(gu + m * 2 * I + I + c, true, 8, u);
  load8<DT>(dact + m * I + c, true, 8, d);
  uint32_t wg[4], wu[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float s2[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      s2[b] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g[2 * j + b]));
    const f32x2 sg = unpack2<DT>(pack2<DT>(g[2 * j] * s2[0], g[2 * j + 1] * s2[1]));
    const f32x2 ds = unpack2<DT>(pack2<DT>(d[2 * j] * u[2 * j], d[2 * j + 1] * u[2 * j + 1]));
    wg[j] = pack2<DT>((ds.x * s2[0]) * (1.0f + g[2 * j] * (1.0f - s2[0])),
                      (ds.y * s2[1]) * (1.0f + g[2 * j + 1] * (1.0f - s2[1])));
    wu[j] = pack2<DT>(d[2 * j] * sg.x, d[2 * j + 1] * sg.y);
    const f32x2 a = unpack2<DT>(wg[j]), b = unpack2<DT>(wu[j]);
    dg[2 * j] = a.x;
    dg[2 * j + 1] = a.y;
    du[2 * j] = b.x;
    du[2 * j + 1] = b.y;
  }
  if (dgu) {
    *reinterpret_cast<uint4*>(dgu + m * 2 * I + c) = make_uint4(wg[0], wg[1], wg[2], wg[3]);
    *reinterpret_cast<uint4*>(dgu + m * 2 * I + I + c) = make_uint4(wu[0], wu[1], wu[2], wu[3]);
  }
  store_block(dg, lane16, q + m * 2 * I + c, s + m * sp + kb);
  store_block(du, lane16, q + m * 2 * I + I + c, s + m * sp + nkb + kb);
}

// Backward of the weighted sum, slot m (token t, expert e): dcur = dt(w dout[t]) as codes and
// scale bytes (and, where a sampled or dense weight gradient reads it, in 16 bits), and
// dweights[t, e] = dt(<dout[t], y[m]>).  One block a slot, 16 lanes a block of 128
// columns.  32,768 slots of 2,048: 134 MB of y and as much of dout from the caches in, 67 out, 54 us (with the
// 16-bit dcur written and read again 59 + 47).
template <int DT>
__global__ __launch_bounds__(256) void fp8_combine_bwd_kernel(const uint16_t* __restrict__ dout,
                                                              const uint16_t* __restrict__ y,
                                                              const int32_t* __restrict__ token_idx,
                                                              const float* __restrict__ slot_w,
                                                              const int32_t* __restrict__ offsets, int E, int64_t H,
                                                              int sp, uint16_t* __restrict__ dcur,
                                                              uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                                              uint16_t* __restrict__ dweights) {
#pragma clang fp contract(off)
  __shared__ float s_part[4];
  const int64_t m = blockIdx.x;
  if (m >= offsets[E]) return;  // block-uniform
  const int64_t t = token_idx[m];
  const float wm = slot_w[m];
  const int lane16 = threadIdx.x & 15;
  float part = 0.f;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < H; c += 2048) {  // H % 128 == 0: 16 lanes go together
    float g[8], v[8], d[8];
    load8<DT>(dout + t * H + c, true, 8, g);
    load8<DT>(y + m * H + c, true, 8, v);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pack2<DT>(g[2 * j] * wm, g[2 * j + 1] * wm);
      const f32x2 f = unpack2<DT>(w[j]);
      d[2 * j] = f.x;
      d[2 * j + 1] = f.y;
      part += g[2 * j] * v[2 * j];
      part += g[2 * j + 1] * v[2 * j + 1];
    }
    if (dcur) *reinterpret_cast<uint4*>(dcur + m * H + c) = make_uint4(w[0], w[1], w[2], w[3]);
    store_block(d, lane16, q + m * H + c, s + m * sp + c / FB);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) part += __shfl_xor(part, k, 64);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    int lo = 0, hi = E - 1;  // expert of slot m: the largest e with offsets[e] <= m
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offsets[mid] <= m) lo = mid;
      else hi = mid - 1;
    }
    store_from_f32<DT>(dweights, t * E + lo, s_part[0] + s_part[1] + s_part[2] + s_part[3]);
  }
}

int blocks16(int64_t n, const char* what, unsigned* out) {  // 16 lane groups a block
  const int64_t b = (n + 15) / 16;
  if (b >= ((int64_t)1 << 31)) return set_error(USAF_ERR_INVALID, "%s: too many blocks of 128", what);
  *out = (unsigned)b;
  return USAF_OK;
}

}  // namespace
}  // namespace usaf

using namespace usaf;

extern "C" int64_t usaf_hip_fp8_scale_stride(int64_t cols) {
  if (cols < 0) return -1;
  return ((cols + FP8_BLOCK - 1) / FP8_BLOCK + 3) / 4 * 4;
}

extern "C" int usaf_hip_fp8_quantize_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld,
                                          const int32_t* n_rows, uint8_t* q, uint8_t* s, void* stream) {
  if (rows < 0 || cols < 0 || cols > (int64_t)1 << 30 || ld < cols)
    return set_error(USAF_ERR_INVALID, "fp8_quantize_rows: need 0 <= cols <= ld, cols <= 2^30");
  if (rows == 0 || cols == 0) return clear_error();
  if (!x || !q || !s) return set_error(USAF_ERR_INVALID, "fp8_quantize_rows: null pointer");
  if ((uintptr_t)q % 16 || (uintptr_t)x % 2)
    return set_error(USAF_ERR_INVALID, "fp8_quantize_rows: codes must be 16-byte and values 2-byte aligned");
  const int64_t nkb = (cols + FP8_BLOCK - 1) / FP8_BLOCK;
  const bool vec = ((uintptr_t)x % 16) == 0 && ld % 8 == 0;
  if (rows > ((int64_t)1 << 40) / nkb) return set_error(USAF_ERR_INVALID, "fp8_quantize_rows: too many rows");
  if (dtype != USAF_BF16 && dtype != USAF_F16)
    return set_error(USAF_ERR_INVALID, "fp8_quantize_rows: dtype must be fp16 or bf16");
  const uint16_t* p = reinterpret_cast<const uint16_t*>(x);
  const hipStream_t st = as_stream(stream);
  unsigned blocks;
  if (vec && cols % 512 == 0 && (uintptr_t)s % 4 == 0) {
    if (int rc = blocks16((rows * nkb + R_AHEAD - 1) / R_AHEAD, "fp8_quantize_rows", &blocks)) return rc;
    if (dtype == USAF_BF16) fp8_rows4_kernel<USAF_BF16><<<blocks, 256, 0, st>>>(p, rows, ld, (int)(nkb / 4), n_rows, q, s);
    else fp8_rows4_kernel<USAF_F16><<<blocks, 256, 0, st>>>(p, rows, ld, (int)(nkb / 4), n_rows, q, s);
    return check_launch("fp8_quantize_rows");
  }
  if (int rc = blocks16(rows * nkb, "fp8_quantize_rows", &blocks)) return rc;
  const int sp = (int)usaf_hip_fp8_scale_stride(cols);
  if (dtype == USAF_BF16)
    fp8_rows_kernel<USAF_BF16><<<blocks, 256, 0, st>>>(p, rows, cols, ld, vec, (int)nkb, nkb * FP8_BLOCK, sp, n_rows, q, s);
  else
    fp8_rows_kernel<USAF_F16><<<blocks, 256, 0, st>>>(p, rows, cols, ld, vec, (int)nkb, nkb * FP8_BLOCK, sp, n_rows, q, s);
  return check_launch("fp8_quantize_rows");
}

static int weight_shape(const char* what, int64_t E, int64_t R, int64_t C) {
  if (E < 0 || R < 0 || C < 0 || E > 1 << 20 || R > 1 << 24 || C > 1 << 24)
    return set_error(USAF_ERR_INVALID, "%s: bad shape [%lld, %lld, %lld]", what, (long long)E, (long long)R, (long long)C);
  const int64_t blocks = E * ((R + FP8_BLOCK - 1) / FP8_BLOCK) * ((C + FP8_BLOCK - 1) / FP8_BLOCK);
  if (blocks >= (int64_t)1 << 31) return set_error(USAF_ERR_INVALID, "%s: too many blocks", what);
  return USAF_OK;
}

extern "C" int usaf_hip_fp8_quantize_weight(const void* w, int32_t dtype, int64_t E, int64_t R, int64_t C, uint8_t* q,
                                            uint8_t* s, void* stream) {
  if (int rc = weight_shape("fp8_quantize_weight", E, R, C)) return rc;
  if (E == 0 || R == 0 || C == 0) return clear_error();
  if (!w || !q || !s || (uintptr_t)q % 16)
    return set_error(USAF_ERR_INVALID, "fp8_quantize_weight: null pointer, or codes not 16-byte aligned");
  const int64_t kp = (C + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
  const unsigned blocks = (unsigned)(E * ((R + FP8_BLOCK - 1) / FP8_BLOCK) * (kp / FP8_BLOCK));
  USAF_DISPATCH_DT(dtype, DT, fp8_weight_kernel<DT><<<blocks, 256, 0, as_stream(stream)>>>(w, R, C, kp, q, s));
  return check_launch("fp8_quantize_weight");
}

extern "C" int usaf_hip_fp8_dequantize(const uint8_t* q, const uint8_t* s, int64_t E, int64_t R, int64_t C, void* out,
                                       int32_t out_dtype, void* stream) {
  if (int rc = weight_shape("fp8_dequantize", E, R, C)) return rc;
  const int64_t total = E * R * C;
  if (total == 0) return clear_error();
  if (!q || !s || !out) return set_error(USAF_ERR_INVALID, "fp8_dequantize: null pointer");
  const int64_t kp = (C + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
  const int64_t want = (total + 1023) / 1024;
  const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
  USAF_DISPATCH_DT(out_dtype, DT,
                   fp8_dequant_kernel<DT><<<blocks, 256, 0, as_stream(stream)>>>(q, s, R, C, kp, total, out));
  return check_launch("fp8_dequantize");
}

extern "C" int usaf_hip_fp8_transpose(const uint8_t* q, const uint8_t* s, int64_t E, int64_t R, int64_t C, uint8_t* qt,
                                      uint8_t* st, void* stream) {
  if (int rc = weight_shape("fp8_transpose", E, R, C)) return rc;
  if (E == 0 || R == 0 || C == 0) return clear_error();
  if (!q || !s || !qt || !st || ((uintptr_t)q | (uintptr_t)qt) % 16)
    return set_error(USAF_ERR_INVALID, "fp8_transpose: null pointer, or codes not 16-byte aligned");
  const int64_t kp = (C + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK, rp = (R + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
  const unsigned blocks = (unsigned)(E * (rp / FP8_BLOCK) * (kp / FP8_BLOCK));
  fp8_transpose_kernel<<<blocks, 256, 0, as_stream(stream)>>>(q, s, R, C, kp, rp, qt, st);
  return check_launch("fp8_transpose");
}

static int swiglu_args(const char* what, int64_t S, int64_t I, const void* a, const void* b, const void* c, const void* n,
                       const void* q, const void* s, unsigned* blocks) {
  if (S < 0 || I <= 0 || I % FP8_BLOCK || I > 1 << 24)
    return set_error(USAF_ERR_INVALID, "%s: need S >= 0 and I a positive multiple of 128", what);
  if (S > ((int64_t)1 << 40) / I) return set_error(USAF_ERR_INVALID, "%s: too many slots", what);
  if (S > 0 && (!a || !b || !n || !q || !s)) return set_error(USAF_ERR_INVALID, "%s: null pointer", what);
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)q) % 16)
    return set_error(USAF_ERR_INVALID, "%s: operands must be 16-byte aligned", what);
  return blocks16(S * (I / FP8_BLOCK), what, blocks);
}

extern "C" int usaf_hip_fp8_swiglu(const void* gu, int64_t S, int64_t I, int32_t dtype, const int32_t* n_slots, void* act,
                                   uint8_t* q, uint8_t* s, void* stream) {
  unsigned blocks;
  if (int rc = swiglu_args("fp8_swiglu", S, I, gu, gu, act, n_slots, q, s, &blocks)) return rc;
  if (S == 0) return clear_error();
  const int sp = (int)usaf_hip_fp8_scale_stride(I);
  const uint16_t* g = reinterpret_cast<const uint16_t*>(gu);
  uint16_t* a = reinterpret_cast<uint16_t*>(act);
  if (dtype == USAF_BF16)
    fp8_swiglu_kernel<USAF_BF16><<<blocks, 256, 0, as_stream(stream)>>>(g, S, I, n_slots, a, q, s, sp);
  else if (dtype == USAF_F16)
    fp8_swiglu_kernel<USAF_F16><<<blocks, 256, 0, as_stream(stream)>>>(g, S, I, n_slots, a, q, s, sp);
  else
    return set_error(USAF_ERR_INVALID, "fp8_swiglu: dtype must be fp16 or bf16");
  return check_launch("fp8_swiglu");
}

extern "C" int usaf_hip_fp8_swiglu_bwd(const void* gu, const void* dact, int64_t S, int64_t I, int32_t dtype,
                                       const int32_t* n_slots, void* dgu, uint8_t* q, uint8_t* s, void* stream) {
  unsigned blocks;
  if (int rc = swiglu_args("fp8_swiglu_bwd", S, I, gu, dact, dgu, n_slots, q, s, &blocks)) return rc;
  if (S == 0) return clear_error();
  const int sp = (int)usaf_hip_fp8_scale_stride(2 * I);
  const uint16_t *g = reinterpret_cast<const uint16_t*>(gu), *d = reinterpret_cast<const uint16_t*>(dact);
  uint16_t* o = reinterpret_cast<uint16_t*>(dgu);
  if (dtype == USAF_BF16)
    fp8_swiglu_bwd_kernel<USAF_BF16><<<blocks, 256, 0, as_stream(stream)>>>(g, d, S, I, n_slots, o, q, s, sp);
  else if (dtype == USAF_F16)
    fp8_swiglu_bwd_kernel<USAF_F16><<<blocks, 256, 0, as_stream(stream)>>>(g, d, S, I, n_slots, o, q, s, sp);
  else
    return set_error(USAF_ERR_INVALID, "fp8_swiglu_bwd: dtype must be fp16 or bf16");
  return check_launch("fp8_swiglu_bwd");
}

extern "C" int usaf_hip_fp8_combine_bwd(const void* dout, const void* y, const int32_t* token_idx, const float* slot_w,
                                        const int32_t* offsets, int64_t S, int64_t E, int64_t H, int32_t dtype, void* dcur,
                                        uint8_t* q, uint8_t* s, void* dweights, void* stream) {
  if (S < 0 || S > 0x7FFFFFFF || E < 1 || E > 1024 || H <= 0 || H % FP8_BLOCK || H > 1 << 24)
    return set_error(USAF_ERR_INVALID, "fp8_combine_bwd: need 0 <= S < 2^31, 1 <= E <= 1024 and H a positive multiple of 128");
  if (S == 0) return clear_error();
  if (!dout || !y || !token_idx || !slot_w || !offsets || !q || !s || !dweights)
    return set_error(USAF_ERR_INVALID, "fp8_combine_bwd: null pointer");
  if (((uintptr_t)dout | (uintptr_t)y | (uintptr_t)dcur | (uintptr_t)q) % 16)
    return set_error(USAF_ERR_INVALID, "fp8_combine_bwd: operands must be 16-byte aligned");
  const int sp = (int)usaf_hip_fp8_scale_stride(H);
  const uint16_t *d = reinterpret_cast<const uint16_t*>(dout), *yy = reinterpret_cast<const uint16_t*>(y);
  uint16_t *o = reinterpret_cast<uint16_t*>(dcur), *dw = reinterpret_cast<uint16_t*>(dweights);
  if (dtype == USAF_BF16)
    fp8_combine_bwd_kernel<USAF_BF16><<<(unsigned)S, 256, 0, as_stream(stream)>>>(d, yy, token_idx, slot_w, offsets, (int)E, H,
                                                                                  sp, o, q, s, dw);
  else if (dtype == USAF_F16)
    fp8_combine_bwd_kernel<USAF_F16><<<(unsigned)S, 256, 0, as_stream(stream)>>>(d, yy, token_idx, slot_w, offsets, (int)E, H,
                                                                                 sp, o, q, s, dw);
  else
    return set_error(USAF_ERR_INVALID, "fp8_combine_bwd: dtype must be fp16 or bf16");
  return check_launch("fp8_combine_bwd");
}

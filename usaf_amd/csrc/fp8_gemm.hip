// Product with an 8-bit block-scaled weight, grouped over experts:
//
//   C[m, n] = dt( sum_k A[row(m), k] W_e[n, k] )     (slots m of expert e)
//
// A: e4m3 codes with an E8M0 scale for each 1 x 128, W: for each 128 x 128.  The
// matrix instruction takes both scales (v_mfma_scale_f32_32x32x64_f8f6f4, one byte
// for each row and 32 k): nothing but it touches the codes or the accumulators.
// The weights are its A operand, the slots its B operand, so a lane's accumulator
// holds 4 consecutive columns of one slot.  Codes are padded with zeros to whole
// blocks along k; rows past the last slot or column repeat it and are not stored.
#include "fp8.h"

namespace usaf {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Args {
  const uint8_t* A;        // [.., Kp] codes
  const uint8_t* as;       // [.., sp] scale bytes
  int sp;
  const int32_t* a_rows;   // A row of slot m (nullptr: row m)
  const uint8_t* W;        // [E, N, Kp] codes
  const uint8_t* ws;       // [E, ceil(N / 128), Kp / 128] scale bytes
  int64_t N, Kp;
  const int32_t* offsets;  // [E + 1]; nullptr: one expert, M slots
  int E;
  int64_t M;
  uint16_t* out;           // [M, N]
};

constexpr int GT = 256;  // threads
constexpr int GN = 128;  // columns of a tile

__device__ __forceinline__ int g_swz(int r) { return (r >> 1) & 7; }

__device__ __forceinline__ f32x16 mfma8(const u32x4 a0, const u32x4 a1, const u32x4 b0, const u32x4 b1, f32x16 c, int sa,
                                        int sb) {
  const i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// One tile: 32 MB slots x 128 columns; wave w has columns 32 w + [0, 32).
template <int MB, int DT>
__global__ __launch_bounds__(GT) void fp8_gemm_kernel(const Fp8Args g) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[2][(32 * MB + GN) * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int n_nt = (int)((g.N + GN - 1) / GN);
  const int mt = blockIdx.x / n_nt, nt = blockIdx.x - mt * n_nt;
  int e = 0, valid;
  int64_t m_beg;
  if (g.offsets) {
    GemmArgs o{};
    o.offsets = g.offsets;
    o.E = g.E;
    int mb;
    if (!slot_tile<32 * MB>(o, lane, mt, e, mb, valid)) return;  // block-uniform
    m_beg = mb;
  } else {
    m_beg = (int64_t)mt * 32 * MB;
    const int64_t left = g.M - m_beg;
    valid = left < 32 * MB ? (int)left : 32 * MB;
  }
  const int nkb = (int)(g.Kp / 128);
  const int r8 = tid >> 3, c8 = tid & 7;
  const uint8_t* a_src[MB];
#pragma unroll
  for (int p = 0; p < MB; ++p) {
    const int r = 32 * p + r8;
    const int64_t m = m_beg + (r < valid ? r : valid - 1);
    a_src[p] = g.A + (g.a_rows ? (int64_t)g.a_rows[m] : m) * g.Kp + 16 * c8;
  }
  const uint8_t* w_src[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    int64_t n = (int64_t)nt * GN + 32 * p + r8;
    n = n < g.N ? n : g.N - 1;
    w_src[p] = g.W + ((int64_t)e * g.N + n) * g.Kp + 16 * c8;
  }
  const uint32_t* s_src[MB];  // scale bytes of the lane's slot, a word for 4 blocks
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int r = 32 * i + l32;
    const int64_t m = m_beg + (r < valid ? r : valid - 1);
    s_src[i] = reinterpret_cast<const uint32_t*>(g.as + (g.a_rows ? (int64_t)g.a_rows[m] : m) * g.sp);
  }
  const uint8_t* const ws = g.ws + ((int64_t)e * n_nt + nt) * nkb;

  u32x4 ar[MB], wr[4];
  auto load = [&](int kb) {
#pragma unroll
    for (int p = 0; p < MB; ++p) ar[p] = *reinterpret_cast<const u32x4*>(a_src[p] + (int64_t)kb * 128);
#pragma unroll
    for (int p = 0; p < 4; ++p) wr[p] = *reinterpret_cast<const u32x4*>(w_src[p] + (int64_t)kb * 128);
  };
  auto at = [&](int r, int c) { return r * 128 + 16 * (c ^ g_swz(r)); };
  auto store = [&](uint8_t* b) {
#pragma unroll
    for (int p = 0; p < MB; ++p) *reinterpret_cast<u32x4*>(b + at(32 * p + r8, c8)) = ar[p];
#pragma unroll
    for (int p = 0; p < 4; ++p) *reinterpret_cast<u32x4*>(b + 32 * MB * 128 + at(32 * p + r8, c8)) = wr[p];
  };
  f32x16 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = f32x16{};
  uint32_t sc[MB];

  load(0);
  store(sm[0]);
  __syncthreads();
  for (int kb = 0; kb < nkb; ++kb) {
    if (kb + 1 < nkb) load(kb + 1);
    if ((kb & 3) == 0) {
#pragma unroll
      for (int i = 0; i < MB; ++i) sc[i] = s_src[i][kb >> 2];
    }
    const int sw = ws[kb];
    const uint8_t* const b = sm[kb & 1];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      const int c = 4 * h2 + 2 * half;
      const uint8_t* const w = b + 32 * MB * 128;
      const u32x4 w0 = *reinterpret_cast<const u32x4*>(w + at(32 * wave + l32, c));
      const u32x4 w1 = *reinterpret_cast<const u32x4*>(w + at(32 * wave + l32, c + 1));
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const u32x4 a0 = *reinterpret_cast<const u32x4*>(b + at(32 * i + l32, c));
        const u32x4 a1 = *reinterpret_cast<const u32x4*>(b + at(32 * i + l32, c + 1));
        acc[i] = mfma8(w0, w1, a0, a1, acc[i], sw, (int)sc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) sc[i] >>= 8;
    if (kb + 1 < nkb) store(sm[(kb + 1) & 1]);
    __syncthreads();
  }
  // lane's values 4 q .. 4 q + 3: columns 8 q + 4 half + [0, 4) of slot l32
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    if (32 * i + l32 >= valid) continue;
    uint16_t* const row = g.out + (m_beg + 32 * i + l32) * g.N;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t n = (int64_t)nt * GN + 32 * wave + 8 * q + 4 * half;
      const uint32_t lo = pack2<DT>(acc[i][4 * q], acc[i][4 * q + 1]), hi = pack2<DT>(acc[i][4 * q + 2], acc[i][4 * q + 3]);
      if (g.N % 4 == 0) {
        if (n < g.N) *reinterpret_cast<uint2*>(row + n) = uint2{lo, hi};
      } else {
        const uint16_t v[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < g.N) row[n + j] = v[j];
      }
    }
  }
}

template <int MB>
int launch(const Fp8Args& g, int dt, hipStream_t st) {
  const int64_t tiles = g.offsets ? (g.M < g.E ? g.M : g.E) + g.M / (32 * MB) : (g.M + 32 * MB - 1) / (32 * MB);
  const int64_t blocks = tiles * ((g.N + GN - 1) / GN);
  if (blocks >= (int64_t)1 << 31) return set_error(USAF_ERR_INVALID, "fp8_gemm: too many tiles");
  if (dt == USAF_BF16) fp8_gemm_kernel<MB, USAF_BF16><<<(unsigned)blocks, GT, 0, st>>>(g);
  else fp8_gemm_kernel<MB, USAF_F16><<<(unsigned)blocks, GT, 0, st>>>(g);
  return check_launch("fp8_gemm");
}

}  // namespace
}  // namespace usaf

using namespace usaf;

extern "C" int usaf_hip_fp8_gemm(const uint8_t* a, const uint8_t* a_scale, const int32_t* a_rows, int64_t M,
                                 const uint8_t* w, const uint8_t* w_scale, const int32_t* offsets, int64_t E, int64_t N,
                                 int64_t K, int32_t dtype, void* out, void* stream) {
  if (M < 0 || N < 0 || K < 0 || E < 1 || N > 1 << 24 || K > 1 << 24 || M > 0x7FFFFFFF)
    return set_error(USAF_ERR_INVALID, "fp8_gemm: bad size M=%lld N=%lld K=%lld E=%lld", (long long)M, (long long)N,
                     (long long)K, (long long)E);
  if (dtype != USAF_BF16 && dtype != USAF_F16) return set_error(USAF_ERR_INVALID, "fp8_gemm: dtype must be fp16 or bf16");
  if (M == 0 || N == 0) return clear_error();
  if (K == 0) return set_error(USAF_ERR_INVALID, "fp8_gemm: need K >= 1");
  if (!a || !a_scale || !w || !w_scale || !out) return set_error(USAF_ERR_INVALID, "fp8_gemm: null pointer");
  if (!offsets && E != 1) return set_error(USAF_ERR_INVALID, "fp8_gemm: more than one expert needs offsets");
  if (E > Q_MAX_E) return set_error(USAF_ERR_UNSUPPORTED, "fp8_gemm: at most %d experts", Q_MAX_E);
  if (((uintptr_t)a | (uintptr_t)w) % 16 || (uintptr_t)a_scale % 4 || (uintptr_t)out % 8)
    return set_error(USAF_ERR_INVALID, "fp8_gemm: codes must be 16-byte, the output 8-byte and scales 4-byte aligned");
  Fp8Args g{};
  g.A = a;
  g.as = a_scale;
  g.Kp = (K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
  g.sp = (int)usaf_hip_fp8_scale_stride(K);
  g.a_rows = a_rows;
  g.W = w;
  g.ws = w_scale;
  g.N = N;
  g.offsets = offsets;
  g.E = (int)E;
  g.M = M;
  g.out = reinterpret_cast<uint16_t*>(out);
  hipStream_t st = as_stream(stream);
  const int64_t per = M / E;  // slots of an expert on average
  if (per <= 32) return launch<1>(g, dtype, st);
  if (per <= 64) return launch<2>(g, dtype, st);
  return launch<4>(g, dtype, st);
}

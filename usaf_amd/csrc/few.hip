// A whole MoE layer for 1 to 32 tokens, on 4-bit or 8-bit experts:
//
//   l = x Wr^T, the k largest l (ties: the lowest expert), w = softmax(l) there (renormalised or not)
//   a_e = dt(silu(g) u),  (g, u) = Wgu_e x;   out = dt(sum_e w_e Wd_e a_e)
//
// Three launches, nothing read back to the host, no slot lists: an expert takes the
// tokens in place.  At most 32 tokens, so one 32-row MFMA operand holds them all
// whatever their experts; a lane whose token the expert does not serve loads nothing,
// and its rows of the result are not used.
//
//   few_route    a block a token: logits, selection by rank, weights
//   few_gate_up  a block an (expert in use, 32 columns of a): four waves split the contraction
//   few_down     a block (32 columns of out, a part of the experts in use): its waves take
//                (expert, part of the contraction) items and keep a weighted sum; the last
//                block of a column tile adds the parts in order
//
// Weights are the MFMA's second operand, a lane's accumulators 16 tokens of one weight
// row: the row's scale and zero are one register each.  A group of 128 is multiplied as
// codes, D = sum_k x_k (c_k + offset) with exact small whole numbers as operands, and
//   y += s D + (z - offset s) sum_k x_k           (4-bit; the sum by an MFMA against ones)
//   y += 2^e D                                    (8-bit)
// which takes 7 vector instructions for 8 codes and 64 for a group of a 32 x 32 tile,
// where dequantizing each weight takes 32 for 8 codes.  The weight is the real number
// s q + z: nothing rounds it.
#include "fp8.h"

namespace usaf {
namespace {

constexpr int FT = 32;        // tokens at most
constexpr int F_MAX_E = 256;  // experts
constexpr int F_MAX_K = 16;   // experts of a token
enum { FMT_Q4 = 0, FMT_FP8 = 1 };

struct FewArgs {
  const uint16_t* x;        // [T, H]
  const uint16_t* router;   // [E, H]
  int T, E, k, norm;
  int H, I;
  const uint8_t* gu;        // codes [E, 2I, H]
  const void* gu_s;         // 4-bit: fp16 scale | zero << 16 for each group; 8-bit: E8M0 bytes
  const uint8_t* dn;        // codes [E, H, I]
  const void* dn_s;
  uint16_t* out;            // [T, H]
  // workspace
  int32_t* sel;             // [T, k] experts
  float* wt;                // [T, k] weights
  uint16_t* xp;             // [T, H] x in the fragments' order (4-bit)
  uint16_t* act;            // [experts in use, T, I] in the fragments' order
  float* part;              // [P, T, H] partial sums
  int32_t* done;            // [H / 32] parts of a column tile that have arrived
  int P, KS;                // few_down: parts of the experts, of the contraction
};

// Order of 8 neighbouring values in a fragment of 4-bit codes: a code word's nibbles
// come apart as (0, 4), (1, 5), (2, 6), (3, 7).
template <int FMT>
__device__ __forceinline__ int frag_pos(int c) {
  if constexpr (FMT == FMT_Q4) return (c & ~7) | ((c & 3) << 1) | ((c >> 2) & 1);
  else return c;
}

// ---- routing ---------------------------------------------------------------------

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// A total order of doubles: larger is larger, a NaN below everything.
__device__ __forceinline__ int64_t order_key(double v) {
  if (v != v) return INT64_MIN;
  const int64_t b = __double_as_longlong(v);
  return b < 0 ? -(b & INT64_MAX) : b;  // -0 with 0
}

// Logits in fp32 products of 8, added in 64 bits: which expert is the k-th hangs on
// differences near fp32's own rounding.  1024 threads read the router's weight once
// for a token; a wave has its experts' rows four at a time in flight.
template <int DT, int FMT>
__global__ __launch_bounds__(1024) void few_route_kernel(const FewArgs g) {
  extern __shared__ __attribute__((aligned(16))) uint16_t s_x[];
  __shared__ double s_l[F_MAX_E];
  __shared__ int64_t s_key[F_MAX_E];
  __shared__ float s_p[F_MAX_K];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (t == 0)
    for (int i = tid; i < g.H / 32; i += 1024) g.done[i] = 0;
  for (int i = tid; i < g.H / 8; i += 1024) {
    const uint4 v = *reinterpret_cast<const uint4*>(g.x + (int64_t)t * g.H + 8 * i);
    *reinterpret_cast<uint4*>(s_x + 8 * i) = v;
    if constexpr (FMT == FMT_Q4) {
      const uint4 o = {__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                       __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
      *reinterpret_cast<uint4*>(g.xp + (int64_t)t * g.H + 8 * i) = o;
    }
  }
  __syncthreads();
  for (int e0 = wave; e0 < g.E; e0 += 64) {
    double acc[4] = {0, 0, 0, 0};
    for (int h = 8 * lane; h < g.H; h += 512) {
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = e0 + 16 * j < g.E ? e0 + 16 * j : g.E - 1;
        w[j] = *reinterpret_cast<const uint4*>(g.router + (int64_t)e * g.H + h);
      }
      const uint4 xv = *reinterpret_cast<const uint4*>(s_x + h);
      const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x2 a = unpack2<DT>(xw[q]), b = unpack2<DT>(ww[q]);
          s = fmaf(a.x, b.x, s);
          s = fmaf(a.y, b.y, s);
        }
        acc[j] += (double)s;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double l = wave_sum_d(acc[j]);
      if (lane == 0 && e0 + 16 * j < g.E) {
        s_l[e0 + 16 * j] = l;
        s_key[e0 + 16 * j] = order_key(l);
      }
    }
  }
  __syncthreads();
  // rank of expert tid / 4: how many come before it; its four threads look at a quarter each
  const int e = tid >> 2;
  int rank = 0;
  if (e < g.E) {
    const int64_t mine = s_key[e];
    for (int o = tid & 3; o < g.E; o += 4) {
      const int64_t other = s_key[o];
      rank += other > mine || (other == mine && o < e);
    }
  }
  rank += __shfl_xor(rank, 1, 64);
  rank += __shfl_xor(rank, 2, 64);
  // softmax: every wave has the whole row, in the same order
  double m = -INFINITY;
  for (int o = lane; o < g.E; o += 64) m = s_l[o] > m ? s_l[o] : m;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const double o = __shfl_xor(m, d, 64);
    m = o > m ? o : m;
  }
  float sum = 0.f;
  for (int o = lane; o < g.E; o += 64) sum += expf((float)(s_l[o] - m));
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
  const bool chosen = e < g.E && rank < g.k;
  const float p = chosen ? expf((float)(s_l[e] - m)) : 0.f;
  if (chosen && (tid & 3) == 0) s_p[rank] = p;
  __syncthreads();
  if (chosen && (tid & 3) == 0) {
    float total = sum;
    if (g.norm) {
      total = 0.f;
      for (int i = 0; i < g.k; ++i) total += s_p[i];
      if (sum != sum) total = sum;  // a NaN anywhere in the row
    }
    g.sel[t * g.k + rank] = e;
    g.wt[t * g.k + rank] = p / total;
  }
}

// ---- products --------------------------------------------------------------------

// Which tokens each expert serves, from the selections (ends with a barrier).
__device__ __forceinline__ void token_masks(const FewArgs& g, uint32_t* s_mask, int tid, int threads) {
  for (int i = tid; i < F_MAX_E; i += threads) s_mask[i] = 0;
  __syncthreads();
  for (int i = tid; i < g.T * g.k; i += threads) atomicOr(&s_mask[g.sel[i]], 1u << (i / g.k));
  __syncthreads();
}

// A wave's operands of one group of 128: NU units of 32 weight rows, and the tokens.
template <int NU, int FMT>
struct Group {
  u32x4 c[NU][FMT == FMT_Q4 ? 2 : 4];  // codes: lane (row, half) has k = 64 s + 32 half + [0, 32) of its row
  uint32_t z[NU];                      // scale | zero, or the E8M0 byte
  u32x4 x[8];                          // tokens: lane (token, half), register 4 s + j: k = 64 s + 32 half + 8 j + [0, 8)
};

template <int FMT>
__device__ __forceinline__ int64_t row_bytes(int K) {
  return FMT == FMT_Q4 ? K / 2 : K;
}

template <int NU, int FMT>
__device__ __forceinline__ void load_group(Group<NU, FMT>& b, const uint8_t* const (&w)[NU], const void* const (&s)[NU],
                                           const uint16_t* x, bool live, int gr) {
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    if constexpr (FMT == FMT_Q4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) b.c[u][i] = *reinterpret_cast<const u32x4*>(w[u] + gr * 64 + 32 * i);
      b.z[u] = reinterpret_cast<const uint32_t*>(s[u])[gr];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) b.c[u][i] = *reinterpret_cast<const u32x4*>(w[u] + gr * 128 + 64 * (i >> 1) + 16 * (i & 1));
      b.z[u] = reinterpret_cast<const uint8_t*>(s[u])[gr];
    }
  }
  if (live) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b.x[i] = *reinterpret_cast<const u32x4*>(x + gr * 128 + 64 * (i >> 2) + 8 * (i & 3));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b.x[i] = u32x4{0, 0, 0, 0};
  }
}

// Eight 4-bit codes -> a fragment register: bf16 128 + q, or fp16 q - 8.
template <int DT>
__device__ __forceinline__ u32x4 frag4(uint32_t w) {
  u32x4 o;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t t = (w >> (4 * p)) & 0x000F000Fu;
    if constexpr (DT == USAF_BF16) {
      o[p] = t | 0x43004300u;
    } else {
      const f16x2 c = {(f16)-1032.0f, (f16)-1032.0f};
      o[p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, t | 0x64006400u) + c);
    }
  }
  return o;
}
// Eight 8-bit codes -> a fragment register (exact in both types).
template <int DT>
__device__ __forceinline__ u32x4 frag8(uint32_t a, uint32_t b) {
  u32x4 o;
  if constexpr (DT == USAF_BF16) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  } else {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
  }
  return o;
}

// acc[u] += the group's product: rows are tokens, columns the unit's weight rows.
template <int NU, int FMT, int DT>
__device__ __forceinline__ void mul_group(const Group<NU, FMT>& b, f32x16 (&acc)[NU]) {
  f32x16 xs = f32x16{};
  if constexpr (FMT == FMT_Q4) {
    const uint32_t one = DT == USAF_BF16 ? 0x3F803F80u : 0x3C003C00u;
#pragma unroll
    for (int i = 0; i < 8; ++i) xs = mfma32<DT>(b.x[i], u32x4{one, one, one, one}, xs);
  }
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    f32x16 d = f32x16{};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (FMT == FMT_Q4) d = mfma32<DT>(b.x[i], frag4<DT>(b.c[u][i >> 2][i & 3]), d);
      else d = mfma32<DT>(b.x[i], frag8<DT>(b.c[u][i >> 1][2 * (i & 1)], b.c[u][i >> 1][2 * (i & 1) + 1]), d);
    }
    if constexpr (FMT == FMT_Q4) {
      const float s = f16_bits_to_f32((uint16_t)b.z[u]), z = f16_bits_to_f32((uint16_t)(b.z[u] >> 16));
      const float zo = DT == USAF_BF16 ? fmaf(-128.0f, s, z) : fmaf(8.0f, s, z);
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[u][i] = fmaf(zo, xs[i], fmaf(s, d[i], acc[u][i]));
    } else {
      const float s = __uint_as_float(b.z[u] == 0 ? 0x00400000u : b.z[u] << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[u][i] = fmaf(s, d[i], acc[u][i]);
    }
  }
}

// Groups [g0, g1) of the contraction, the next one's loads in flight.
template <int NU, int FMT, int DT>
__device__ __forceinline__ void mul_range(const uint8_t* const (&w)[NU], const void* const (&s)[NU], const uint16_t* x,
                                          bool live, int g0, int g1, f32x16 (&acc)[NU]) {
  if (g0 >= g1) return;
  Group<NU, FMT> a, b;
  load_group<NU, FMT>(a, w, s, x, live, g0);
  for (int gr = g0;;) {
    if (gr + 1 < g1) load_group<NU, FMT>(b, w, s, x, live, gr + 1);
    __builtin_amdgcn_sched_barrier(0);
    mul_group<NU, FMT, DT>(a, acc);
    if (++gr >= g1) break;
    if (gr + 1 < g1) load_group<NU, FMT>(a, w, s, x, live, gr + 1);
    __builtin_amdgcn_sched_barrier(0);
    mul_group<NU, FMT, DT>(b, acc);
    if (++gr >= g1) break;
  }
}

// Scales of weight row `row` (of an expert with R rows): the first group's.
template <int FMT>
__device__ __forceinline__ const void* row_scales(const void* s, int e, int R, int row, int ng) {
  if constexpr (FMT == FMT_Q4) return reinterpret_cast<const uint32_t*>(s) + ((int64_t)e * R + row) * ng;
  else return reinterpret_cast<const uint8_t*>(s) + ((int64_t)e * ((R + 127) / 128) + row / 128) * ng;
}

constexpr int GU_WAVES = 4, GU_THREADS = 64 * GU_WAVES;

template <int DT, int FMT>
__global__ __launch_bounds__(GU_THREADS, 2) void few_gate_up_kernel(const FewArgs g) {
  __shared__ uint32_t s_mask[F_MAX_E];
  __shared__ int s_cnt[F_MAX_E / 64], s_e;
  __shared__ f32x4 s_red[GU_WAVES][8][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int n_nt = g.I / 32, u = blockIdx.x / n_nt, n0 = (blockIdx.x - u * n_nt) * 32;
  if (tid == 0) s_e = -1;
  token_masks(g, s_mask, tid, GU_THREADS);
  {  // the u-th expert in use
    const bool used = s_mask[tid] != 0;
    const uint64_t bal = __ballot(used);
    if (lane == 0) s_cnt[wave] = __popcll(bal);
    __syncthreads();
    int rank = __popcll(bal & ((1ull << lane) - 1));
    for (int i = 0; i < wave; ++i) rank += s_cnt[i];
    if (used && rank == u) s_e = tid;
    __syncthreads();
  }
  const int e = __builtin_amdgcn_readfirstlane(s_e);
  if (e < 0) return;  // block-uniform
  const uint32_t mask = s_mask[e];
  const int ng = g.H / 128;
  const int64_t rb = row_bytes<FMT>(g.H);
  const int rows[2] = {n0 + l32, g.I + n0 + l32};
  const int lane_off = FMT == FMT_Q4 ? 16 * half : 32 * half;
  const uint8_t* const w[2] = {g.gu + ((int64_t)e * 2 * g.I + rows[0]) * rb + lane_off,
                               g.gu + ((int64_t)e * 2 * g.I + rows[1]) * rb + lane_off};
  const void* const s[2] = {row_scales<FMT>(g.gu_s, e, 2 * g.I, rows[0], ng), row_scales<FMT>(g.gu_s, e, 2 * g.I, rows[1], ng)};
  const uint16_t* const x = (FMT == FMT_Q4 ? g.xp : g.x) + (int64_t)(l32 < g.T ? l32 : 0) * g.H + 32 * half;
  f32x16 acc[2] = {f32x16{}, f32x16{}};
  mul_range<2, FMT, DT>(w, s, x, (mask >> l32) & 1, ng * wave / GU_WAVES, ng * (wave + 1) / GU_WAVES, acc);
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      s_red[wave][4 * v + q][lane] = f32x4{acc[v][4 * q], acc[v][4 * q + 1], acc[v][4 * q + 2], acc[v][4 * q + 3]};
  __syncthreads();
  // wave q finishes tokens 8 q + 4 half + [0, 4) of column n0 + l32
  f32x4 gt = s_red[0][wave][lane], up = s_red[0][4 + wave][lane];
#pragma unroll
  for (int i = 1; i < GU_WAVES; ++i) {
    const f32x4 a = s_red[i][wave][lane], b = s_red[i][4 + wave][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      gt[j] += a[j];
      up[j] += b[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = 8 * wave + 4 * half + j;
    if ((mask >> t) & 1)
      store_from_f32<DT>(g.act, ((int64_t)u * g.T + t) * g.I + frag_pos<FMT>(n0 + l32), silu_fast(gt[j]) * up[j]);
  }
}

constexpr int DN_WAVES = 8, DN_THREADS = 64 * DN_WAVES;

template <int DT, int FMT>
__global__ __launch_bounds__(DN_THREADS, 2) void few_down_kernel(const FewArgs g) {
  __shared__ uint32_t s_mask[F_MAX_E];
  __shared__ uint16_t s_used[F_MAX_E];
  __shared__ int s_cnt[F_MAX_E / 64], s_last;
  __shared__ __attribute__((aligned(16))) float s_w[F_MAX_E * FT];  // weight of (expert, token); later the partial sums
  static_assert(F_MAX_E * FT * 4 >= DN_WAVES * 4 * 64 * 16, "the waves' sums fit the weights' place");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int nt = blockIdx.x / g.P, p = blockIdx.x - nt * g.P, n0 = 32 * nt;
  token_masks(g, s_mask, tid, DN_THREADS);
  for (int i = tid; i < g.T * g.k; i += DN_THREADS) s_w[g.sel[i] * FT + i / g.k] = g.wt[i];
  bool used = false;
  uint64_t bal = 0;
  if (tid < F_MAX_E) {
    used = s_mask[tid] != 0;
    bal = __ballot(used);
    if (lane == 0) s_cnt[wave] = __popcll(bal);
  }
  __syncthreads();
  int total = 0;
  {
    int before = 0;
#pragma unroll
    for (int i = 0; i < F_MAX_E / 64; ++i) {
      if (i == wave) before = total;
      total += s_cnt[i];
    }
    if (used) s_used[before + __popcll(bal & ((1ull << lane) - 1))] = (uint16_t)tid;
  }
  __syncthreads();
  const int u0 = total * p / g.P, u1 = total * (p + 1) / g.P;
  const int ng = g.I / 128, n_items = (u1 - u0) * g.KS;
  const int64_t rb = row_bytes<FMT>(g.I);
  const int lane_off = FMT == FMT_Q4 ? 16 * half : 32 * half;
  f32x16 sum = f32x16{};
  for (int it = wave; it < n_items; it += DN_WAVES) {
    const int u = __builtin_amdgcn_readfirstlane(u0 + it / g.KS), ks = it % g.KS;
    const int e = __builtin_amdgcn_readfirstlane((int)s_used[u]);
    const uint32_t mask = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_mask[e]);
    const uint8_t* const w[1] = {g.dn + ((int64_t)e * g.H + n0 + l32) * rb + lane_off};
    const void* const s[1] = {row_scales<FMT>(g.dn_s, e, g.H, n0 + l32, ng)};
    const bool live = (mask >> l32) & 1;
    const uint16_t* const x = g.act + ((int64_t)u * g.T + (live ? l32 : 0)) * g.I + 32 * half;
    f32x16 y[1] = {f32x16{}};
    mul_range<1, FMT, DT>(w, s, x, live, ng * ks / g.KS, ng * (ks + 1) / g.KS, y);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 wv = *reinterpret_cast<const f32x4*>(&s_w[e * FT + 8 * q + 4 * half]);
      const uint32_t m4 = mask >> (8 * q + 4 * half);
#pragma unroll
      for (int j = 0; j < 4; ++j)  // a row of another token's is not added, not even as 0 times something
        if ((m4 >> j) & 1) sum[4 * q + j] = fmaf(wv[j], y[0][4 * q + j], sum[4 * q + j]);
    }
  }
  __syncthreads();
  f32x4* const red = reinterpret_cast<f32x4*>(s_w);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    red[(wave * 4 + q) * 64 + lane] = f32x4{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]};
  __syncthreads();
  float v[4];
  if (wave < 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.f;
#pragma unroll
    for (int i = 0; i < DN_WAVES; ++i) {
      const f32x4 a = red[(i * 4 + wave) * 64 + lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += a[j];
    }
    // tokens 8 wave + 4 half + [0, 4) of column n0 + l32
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 8 * wave + 4 * half + j;
      if (t >= g.T) continue;
      if (g.P == 1) store_from_f32<DT>(g.out, (int64_t)t * g.H + n0 + l32, v[j]);
      else __hip_atomic_store(&g.part[((int64_t)p * g.T + t) * g.H + n0 + l32], v[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (g.P == 1) return;
  // The parts of a column tile meet at the device's coherence point: stored and loaded at
  // agent scope, which passes the dies' L2s, and counted behind a wait for the stores.  The
  // last block adds them in order, so the sum does not hang on who came last; no block waits for another.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    s_last = __hip_atomic_fetch_add(&g.done[nt], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == g.P - 1;
  __syncthreads();
  if (!s_last) return;
  for (int i = tid; i < g.T * 32; i += DN_THREADS) {
    const int t = i >> 5;
    const int64_t at = (int64_t)t * g.H + n0 + (i & 31);
    float o = 0.f;
    for (int q = 0; q < g.P; ++q)
      o += __hip_atomic_load(&g.part[(int64_t)q * g.T * g.H + at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    store_from_f32<DT>(g.out, at, o);
  }
}

struct FewPlan {
  int64_t in_use, sel, wt, xp, act, part, done, bytes;
  int P, KS;
};

// Sizes, and where each buffer sits in the workspace (16-byte steps).
FewPlan few_plan(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) {
  FewPlan p;
  p.in_use = E < T * k ? E : T * k;
  const int64_t tiles = H / 32, groups = I / 128;
  int64_t parts = 512 / tiles;
  parts = parts < 1 ? 1 : parts > p.in_use ? p.in_use : parts;
  const int64_t per = (p.in_use + parts - 1) / parts;
  int64_t ks = (DN_WAVES + per - 1) / per;
  p.P = (int)parts;
  p.KS = (int)(ks > groups ? groups : ks);
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t b = at; at += (bytes + 15) / 16 * 16; return b; };
  p.sel = take(T * k * 4);
  p.wt = take(T * k * 4);
  p.done = take(tiles * 4);
  p.xp = take(T * H * 2);
  p.act = take(p.in_use * T * I * 2);
  p.part = take(parts > 1 ? parts * T * H * 4 : 0);
  p.bytes = at;
  return p;
}

template <int DT, int FMT>
int launch_few_layer(const FewArgs& g, int64_t in_use, hipStream_t st) {
  few_route_kernel<DT, FMT><<<(unsigned)g.T, 1024, (size_t)g.H * 2, st>>>(g);
  if (int rc = check_launch("moe_few/route")) return rc;
  few_gate_up_kernel<DT, FMT><<<(unsigned)(in_use * (g.I / 32)), GU_THREADS, 0, st>>>(g);
  if (int rc = check_launch("moe_few/gate_up")) return rc;
  few_down_kernel<DT, FMT><<<(unsigned)(g.H / 32 * g.P), DN_THREADS, 0, st>>>(g);
  return check_launch("moe_few/down");
}

int few_sizes(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) {
  if (T < 0 || T > FT) return set_error(USAF_ERR_INVALID, "moe_few: 0 to %d tokens, got %lld", FT, (long long)T);
  if (E < 1 || k < 1 || k > E) return set_error(USAF_ERR_INVALID, "moe_few: need 1 <= top_k <= E");
  if (E > F_MAX_E || k > F_MAX_K)
    return set_error(USAF_ERR_UNSUPPORTED, "moe_few: at most %d experts and top_k %d", F_MAX_E, F_MAX_K);
  if (H < 128 || I < 128 || H % 128 || I % 128 || H > 16384 || I > 65536)
    return set_error(USAF_ERR_UNSUPPORTED, "moe_few: H (<= 16384) and I (<= 65536) must be positive multiples of 128");
  return USAF_OK;
}

}  // namespace
}  // namespace usaf

using namespace usaf;

extern "C" int64_t usaf_hip_moe_few_ws_bytes(int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I) {
  if (few_sizes(T, E, top_k, H, I) != USAF_OK) return -1;
  return T == 0 ? 0 : few_plan(T, E, top_k, H, I).bytes;
}

extern "C" int usaf_hip_moe_few(const void* x, int64_t T, int64_t H, const void* router, int64_t E, int64_t top_k,
                                int32_t norm_topk_prob, int32_t dtype, int64_t I, int32_t eight_bit,
                                const uint8_t* gate_up, const void* gate_up_scale, const uint8_t* down,
                                const void* down_scale, void* out, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = few_sizes(T, E, top_k, H, I)) return rc;
  if (dtype != USAF_BF16 && dtype != USAF_F16) return set_error(USAF_ERR_INVALID, "moe_few: dtype must be fp16 or bf16");
  if (T == 0) return clear_error();
  if (!x || !router || !gate_up || !gate_up_scale || !down || !down_scale || !out || !ws)
    return set_error(USAF_ERR_INVALID, "moe_few: null pointer");
  if (((uintptr_t)x | (uintptr_t)router | (uintptr_t)gate_up | (uintptr_t)down | (uintptr_t)ws) % 16)
    return set_error(USAF_ERR_INVALID, "moe_few: activations, router, codes and workspace must be 16-byte aligned");
  if ((!eight_bit && ((uintptr_t)gate_up_scale | (uintptr_t)down_scale) % 4) || (uintptr_t)out % 2)
    return set_error(USAF_ERR_INVALID, "moe_few: misaligned scales or output");
  const FewPlan p = few_plan(T, E, top_k, H, I);
  if (ws_bytes < p.bytes)
    return set_error(USAF_ERR_INVALID, "moe_few: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)p.bytes);
  FewArgs g{};
  g.x = reinterpret_cast<const uint16_t*>(x);
  g.router = reinterpret_cast<const uint16_t*>(router);
  g.T = (int)T;
  g.E = (int)E;
  g.k = (int)top_k;
  g.norm = norm_topk_prob ? 1 : 0;
  g.H = (int)H;
  g.I = (int)I;
  g.gu = gate_up;
  g.gu_s = gate_up_scale;
  g.dn = down;
  g.dn_s = down_scale;
  g.out = reinterpret_cast<uint16_t*>(out);
  uint8_t* const b = reinterpret_cast<uint8_t*>(ws);
  g.sel = reinterpret_cast<int32_t*>(b + p.sel);
  g.wt = reinterpret_cast<float*>(b + p.wt);
  g.done = reinterpret_cast<int32_t*>(b + p.done);
  g.xp = reinterpret_cast<uint16_t*>(b + p.xp);
  g.act = reinterpret_cast<uint16_t*>(b + p.act);
  g.part = reinterpret_cast<float*>(b + p.part);
  g.P = p.P;
  g.KS = p.KS;
  hipStream_t st = as_stream(stream);
  if (eight_bit)
    return dtype == USAF_BF16 ? launch_few_layer<USAF_BF16, FMT_FP8>(g, p.in_use, st)
                              : launch_few_layer<USAF_F16, FMT_FP8>(g, p.in_use, st);
  return dtype == USAF_BF16 ? launch_few_layer<USAF_BF16, FMT_Q4>(g, p.in_use, st)
                            : launch_few_layer<USAF_F16, FMT_Q4>(g, p.in_use, st);
}
